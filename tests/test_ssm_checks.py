"""Checks of the state-space facade that need no GPU: which tensors of a call may share memory."""
import pytest
import torch


def overlaps(a, b):
    """Whether two views of one buffer share an element, by their element numbers."""
    def elements(t):
        at = torch.tensor([t.storage_offset()])
        for n, s in zip(t.shape, t.stride()):
            at = (at[:, None] + torch.arange(n) * s).reshape(-1)
        return set(at.tolist())
    return bool(elements(a) & elements(b))


@pytest.mark.parametrize("strides,shape,off", [((25, 10), (2, 4, 4), 5), ((25, 10), (3, 5, 4), 5), ((35, 10), (2, 4, 4), 5), ((32, 8), (2, 4, 4), 4),
                                               ((40, 10), (2, 4, 4), 5), ((10, 40), (4, 2, 4), 4), ((10, 25), (2, 2, 4), 5), ((30, 10), (2, 3, 4), 6)])
def test_other_columns_of_the_same_rows_share_nothing(strides, shape, off):
    """Batches may start at any row of the buffer, but where a batch stride is no multiple of the row stride, other columns of one batch are
    the first columns of another."""
    from mockingbird_amd import _lib, ssm
    buf = torch.zeros(400)
    out, x = buf.as_strided(shape, strides + (1,), 0), buf.as_strided(shape, strides + (1,), off)
    if overlaps(out, x):
        with pytest.raises(_lib.MbHipError, match="overlap"):
            ssm._apart("f", out, shape[:2], shape[2], ("x", x))
    elif all(max(strides) % s == 0 for s in strides):  # (apart all the same, but not by a rule on the strides alone: may be refused)
        ssm._apart("f", out, shape[:2], shape[2], ("x", x))
