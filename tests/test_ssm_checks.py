"""Which tensors of a state-space call may share memory, and other refusals of the facade and the library."""
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


@pytest.fixture
def host_calls(lib, monkeypatch):
    """Calls on host tensors, up to what the library refuses."""
    from mockingbird_amd import _lib, ssm
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would be launched on host memory")
    monkeypatch.setattr(ssm, "_inputs", lambda fn, x, **others: 0)
    monkeypatch.setattr(ssm, "_launch", lambda fn, index, call, *args: _lib.check(call(*args, None), fn))


F32 = torch.float32
T, C, K, H, P, N, SLOTS = 6, 32, 4, 2, 16, 8, 7


def arguments():
    """(call, its tensors by name with shape and type)"""
    i32, rows = torch.int32, [T]
    slots = dict(slots=([2], i32))
    seqs = dict(cu_seqlens=([3], i32), has_state=([2], torch.bool), **slots)
    conv = dict(x=(rows + [C], F32), weight=([C, K], F32), bias=([C], F32), state=([SLOTS, K - 1, C], F32))
    scan = dict(x=(rows + [H, P], F32), dt=(rows + [H], F32), A=([H], F32), B=(rows + [1, N], F32), C=(rows + [1, N], F32), D=([H], F32), dt_bias=([H], F32),
                state=([SLOTS, H, P, N], F32))
    many = dict(slots=([T], i32))  # a step has one row for each request
    norm = dict(x=(rows + [C], F32), weight=([C], F32), bias=([C], F32), gate=(rows + [C], F32), residual=(rows + [C], F32), scale=([C], F32),
                next_weight=([C], F32), next_bias=([C], F32))
    padded = {k: ([2, T // 2] + v[0][1:] if v[0][0] == T else v[0], v[1]) for k, v in scan.items()}
    return [("causal_conv1d", {**conv, **seqs}), ("causal_conv1d_step", {**conv, **many}), ("selective_scan", {**scan, **seqs}),
            ("selective_scan", {**padded, **slots, "lengths": ([2], i32)}), ("selective_scan_step", {**scan, **many}), ("block_norm", norm)]


def pairs():
    for i, (name, spec) in enumerate(arguments()):
        for arg in spec:
            yield i, "out", arg
            if name == "block_norm":
                yield i, "residual_out", arg
            elif arg != "state":
                yield i, "state", arg


def place(shape, dtype, buf, at):
    e = torch.empty(0, dtype=dtype).element_size()
    return buf[at:at + torch.Size(shape).numel() * e].view(dtype).view(shape)


def call_with(i, written, arg, behind, shared, device):
    """The call with arg right behind or in front of what it writes, or (shared) four bytes into it."""
    from mockingbird_amd import ssm
    name, spec = arguments()[i]
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device=device)
    kw = {k: torch.zeros(v[0], dtype=v[1], device=device) for k, v in spec.items()}
    if "cu_seqlens" in kw:
        kw["cu_seqlens"].copy_(torch.tensor([0, 2, T]))
    if "slots" in kw:
        kw["slots"].copy_(torch.arange(kw["slots"].numel()))
    if written != "state":
        kw[written] = torch.zeros(spec["x"][0], dtype=F32, device=device)
    if name == "block_norm":
        kw["norm"], kw["next_norm"] = "layer", "rms"
    first, second = (written, arg) if behind else (arg, written)
    for k, at in ((first, 4096), (second, 4096 + kw[first].numel() * kw[first].element_size())):
        if k == second:
            at = (at - 1) // 4 * 4 if shared else (at + 15) // 16 * 16
        kw[k] = place(list(kw[k].shape), kw[k].dtype, buf, at).copy_(kw[k])
    return getattr(ssm, name)(**kw)


@pytest.mark.parametrize("i,written,arg", list(pairs()))
@pytest.mark.parametrize("behind", [True, False])
def test_what_a_call_writes_and_its_arguments_may_not_overlap(host_calls, i, written, arg, behind):
    from mockingbird_amd import _lib
    with pytest.raises(_lib.MbHipError, match="overlaps"):
        call_with(i, written, arg, behind, True, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("i,written,arg", list(pairs()))
@pytest.mark.parametrize("behind", [True, False])
def test_what_a_call_writes_and_its_arguments_may_be_neighbours(cuda, lib, i, written, arg, behind):
    from mockingbird_amd import _lib
    call_with(i, written, arg, behind, False, "cuda")
    with pytest.raises(_lib.MbHipError, match="overlaps"):
        call_with(i, written, arg, behind, True, "cuda")
    torch.cuda.synchronize()


def slot_rows(n, x_row, out_row, device):
    """One token with x and y in rows of the slots' own [taps + 1, channels] buffer."""
    from mockingbird_amd import ssm
    buf = torch.randn(SLOTS, K + 1, C, generator=torch.Generator().manual_seed(n)).to(device)
    was = buf.clone()
    w = torch.ones(C, K, device=device)
    y = ssm.causal_conv1d_step(buf[:n, x_row], buf[:, :K - 1], w, slots=torch.arange(n, dtype=torch.int32, device=device), out=buf[:n, out_row])
    return buf, was, y


def test_a_token_inside_its_own_state_is_refused(host_calls):
    from mockingbird_amd import _lib
    for n in (1, 3, SLOTS):
        with pytest.raises(_lib.MbHipError, match="state overlaps x"):
            slot_rows(n, K - 2, K, "cpu")
        with pytest.raises(_lib.MbHipError, match="out overlaps"):
            slot_rows(n, K - 1, K - 1, "cpu")


@pytest.mark.gpu
def test_slots_with_room_for_the_next_input_and_the_answer(cuda, lib):
    """x and y in further rows of every slot's buffer: other columns of the same rows, however many requests there are."""
    for n in (1, 3, SLOTS):
        buf, was, y = slot_rows(n, K - 1, K, "cuda")
        assert torch.equal(buf[:n, :K - 1], was[:n, 1:K]) and torch.equal(buf[:n, K - 1], was[:n, K - 1]) and torch.equal(buf[n:], was[n:])
        # four products with ones, each sum rounded
        assert (y.double() - was[:n, :K].double().sum(1)).abs().max() <= 4 * 2.0 ** -24 * was[:n, :K].abs().sum(1).max()


def test_forward_mode_tangents_are_seen(lib):
    from torch.autograd import forward_ad
    from mockingbird_amd import _lib, ssm
    x = torch.zeros(3)
    with forward_ad.dual_level():
        ssm._refuse_tangents("f", x=x, bias=None)
        with pytest.raises(_lib.MbHipError, match="bias is a dual tensor"), torch.no_grad():
            ssm._refuse_tangents("f", x=x, bias=forward_ad.make_dual(x, x))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("i,arg", [(i, a) for i, (_, spec) in enumerate(arguments()) for a, (_, dtype) in spec.items() if dtype is F32 and a[:5] != "next_"])
def test_forward_mode_derivatives_are_refused(cuda, lib, i, arg, grad):
    from torch.autograd import forward_ad
    from mockingbird_amd import _lib, ssm
    name, spec = arguments()[i]
    kw = {k: torch.zeros(shape, dtype=dtype, device="cuda") for k, (shape, dtype) in spec.items()}
    if name == "block_norm":
        kw.pop("next_weight"), kw.pop("next_bias")
    if "cu_seqlens" in kw:  # every row belongs to a request: rows of a fresh output that belong to none hold anything
        kw["cu_seqlens"].copy_(torch.tensor([0, 2, T]))
    if "lengths" in kw:
        kw["lengths"].fill_(T // 2)
    if "slots" in kw:
        kw["slots"].copy_(torch.arange(kw["slots"].numel()))
    plain = getattr(ssm, name)(**kw)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert torch.equal(getattr(ssm, name)(**kw), plain)  # other tensors of the program have tangents, these have none
        kw[arg] = forward_ad.make_dual(kw[arg], torch.ones_like(kw[arg]))
        with pytest.raises(_lib.MbHipError, match=f"{arg} is a dual tensor"):
            getattr(ssm, name)(**kw)


def test_launches_beyond_the_hardware_are_refused_by_name(lib):
    """A launch has less than 2^32 threads."""
    from mockingbird_amd import _lib
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would be launched on addresses that are none")
    rows = 1 << 24
    norm = _lib.BlockNormArgs(d_x=1 << 60, d_sum=1 << 61, rows=rows, channels=4096, groups=1, norm=1, dtype=_lib.MB_BF16, res_dtype=_lib.MB_BF16, x_rstride=4096,
                              sum_rstride=4096, eps=1e-5, res_scale=1.0)
    scan = _lib.SelectiveScanArgs(d_x=1 << 56, d_y=1 << 57, d_dt=1 << 58, d_b=1 << 59, d_c=1 << 60, d_a=256, dtype=_lib.MB_BF16, dt_dtype=_lib.MB_BF16, batch=rows, t=1,
                                  heads=2, head_dim=64, groups=1, d_state_dim=64, dt_min=0.0, dt_max=1.0)
    step = _lib.SelectiveScanArgs(d_x=1 << 56, d_y=1 << 57, d_dt=1 << 58, d_b=1 << 59, d_c=1 << 60, d_a=256, d_state=1 << 61, n_slots=rows, dtype=_lib.MB_BF16,
                                  dt_dtype=_lib.MB_BF16, batch=rows, heads=2, head_dim=64, groups=1, d_state_dim=64, dt_min=0.0, dt_max=1.0)
    conv = _lib.CausalConv1dArgs(d_x=1 << 60, d_y=1 << 61, d_w=256, dtype=_lib.MB_BF16, batch=rows, t=1, channels=64, ksize=4)
    conv_step = _lib.CausalConv1dArgs(d_x=1 << 60, d_y=1 << 61, d_w=256, d_state=1 << 62, n_slots=1 << 27, dtype=_lib.MB_BF16, batch=1 << 27, channels=64, ksize=4)
    for name, call in dict(block_norm=lambda: lib.mb_block_norm(norm, None), selective_scan=lambda: lib.mb_selective_scan(scan, None, 0, None),
                           selective_scan_step=lambda: lib.mb_selective_scan_step(step, None), causal_conv1d=lambda: lib.mb_causal_conv1d(conv, None),
                           causal_conv1d_step=lambda: lib.mb_causal_conv1d_step(conv_step, None)).items():
        assert call() == -1, name
        assert "too many" in lib.mb_last_error().decode() and name in lib.mb_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(6))
def test_calls_while_another_device_is_current(cuda, lib, monkeypatch, i):
    """The way that a call takes when its tensors are not on the current device (which is said to be another one here)."""
    from mockingbird_amd import ssm
    name, spec = arguments()[i]
    r = torch.Generator().manual_seed(i)
    kw = {k: torch.randn(shape, generator=r).cuda() if dtype is F32 else torch.ones(shape, dtype=dtype, device="cuda") for k, (shape, dtype) in spec.items()}
    if "cu_seqlens" in kw:
        kw["cu_seqlens"].copy_(torch.tensor([0, 2, T]))
    if "slots" in kw:
        kw["slots"].copy_(torch.arange(kw["slots"].numel()))
    if "lengths" in kw:
        kw["lengths"].fill_(T // 2)
    if "A" in kw:
        kw["A"].abs_().neg_()
    if name == "block_norm":
        kw["norm"], kw["next_norm"] = "layer", "rms"
    other = {k: v.clone() if torch.is_tensor(v) else v for k, v in kw.items()}
    want = getattr(ssm, name)(**kw)
    entered = []

    class Entered(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(ssm, "_device", lambda: torch.cuda.device_count())
    monkeypatch.setattr(torch.cuda, "device", Entered)
    got = getattr(ssm, name)(**other)
    assert entered == [0]
    for a, b in zip(want if isinstance(want, tuple) else (want,), got if isinstance(got, tuple) else (got,)):
        assert torch.equal(a, b)
    if "state" in kw:
        assert torch.equal(kw["state"], other["state"])
