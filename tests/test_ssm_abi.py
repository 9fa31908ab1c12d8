"""The state-space entry points refuse bad arguments before any GPU work (no GPU needed), and their structs match the header."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


def test_struct_layouts(lib, tmp_path):
    from mockingbird_amd import _lib
    src = tmp_path / "sz.c"
    names = [("mb_causal_conv1d_args", _lib.CausalConv1dArgs), ("mb_selective_scan_args", _lib.SelectiveScanArgs), ("mb_block_norm_args", _lib.BlockNormArgs)]
    body = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in m._fields_) for n, m in names)
    src.write_text('#include "mbhip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){' + body + 'return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)])
    want = []
    for _, m in names:
        want += [C.sizeof(m)] + [getattr(m, f).offset for f, _ in m._fields_]
    assert list(map(int, subprocess.check_output([str(exe)], text=True).split())) == want


def conv(**kw):
    from mockingbird_amd import _lib
    a = dict(d_x=256, d_y=256, d_w=256, dtype=_lib.MB_F32, batch=2, t=4, channels=8, ksize=4, x_rstride=8, y_rstride=8)
    a.update(kw)
    return _lib.CausalConv1dArgs(**a)


def scan(**kw):
    from mockingbird_amd import _lib
    a = dict(d_x=256, d_y=256, d_dt=256, d_b=256, d_c=256, d_a=256, dtype=_lib.MB_F32, dt_dtype=_lib.MB_F32, batch=2, t=4, heads=4, head_dim=8,
             groups=2, d_state_dim=8, dt_min=0.0, dt_max=1.0)
    a.update(kw)
    return _lib.SelectiveScanArgs(**a)


def norm(**kw):
    from mockingbird_amd import _lib
    a = dict(d_x=256, d_sum=256, rows=2, channels=8, groups=1, norm=1, dtype=_lib.MB_F32, res_dtype=_lib.MB_F32, eps=1e-5, res_scale=1.0)
    a.update(kw)
    return _lib.BlockNormArgs(**a)


@pytest.mark.parametrize("make,kw,match", [
    (conv, dict(dtype=2), "dtype"), (conv, dict(ksize=1), "ksize"), (conv, dict(ksize=9), "ksize"), (conv, dict(act=2), "act"), (conv, dict(batch=-1), "negative"),
    (conv, dict(d_w=None), "weight"), (conv, dict(d_x=None), "null"), (conv, dict(d_state=256, n_slots=1), "slots"), (conv, dict(d_slots=256), "pool"),
    (conv, dict(d_cu_seqlens=256, d_valid=256), "packed"), (conv, dict(batch=1 << 30, t=1 << 30), "too many"),
    (conv, dict(d_cu_seqlens=256, t=(1 << 31) - 1), "too many"), (scan, dict(t=(1 << 30) + 1), "too many"),
    (scan, dict(dtype=2), "dtype"), (scan, dict(dt_dtype=1), "dt_dtype"), (scan, dict(head_dim=0), "head_dim"), (scan, dict(head_dim=129), "head_dim"),
    (scan, dict(d_state_dim=257), "d_state"), (scan, dict(groups=3), "groups"), (scan, dict(dt_min=2.0), "dt_min"), (scan, dict(dt_min=float("nan")), "dt_min"),
    (scan, dict(d_a=None), "no A"), (scan, dict(d_c=None), "null"), (scan, dict(d_has_state=256), "pool"), (scan, dict(batch=1 << 30, heads=4, t=1 << 30), "too many"),
    (norm, dict(dtype=7), "dtype"), (norm, dict(res_dtype=1), "res_dtype"), (norm, dict(norm=3), "norm"), (norm, dict(gate_act=3), "gate_act"),
    (norm, dict(groups=3), "groups"), (norm, dict(groups=0), "groups"), (norm, dict(norm=0), "nothing"), (norm, dict(next_norm=1), "y comes"),
    (norm, dict(d_sum=None), "y comes"), (norm, dict(rows=1 << 31), "too many"), (norm, dict(d_x=None), "null x")])
def test_bad_arguments_are_refused(lib, make, kw, match):
    a = make(**kw)
    rc = {conv: lambda: lib.mb_causal_conv1d(a, None), scan: lambda: lib.mb_selective_scan(a, None, 0, None), norm: lambda: lib.mb_block_norm(a, None)}[make]()
    assert rc == -1 and match in lib.mb_last_error().decode()


def test_steps_need_a_pool_and_null_structs_are_refused(lib):
    assert lib.mb_causal_conv1d_step(conv(), None) == -1 and b"state pool" in lib.mb_last_error()
    assert lib.mb_selective_scan_step(scan(), None) == -1 and b"state pool" in lib.mb_last_error()
    assert lib.mb_causal_conv1d(None, None) == -1 and lib.mb_selective_scan(None, None, 0, None) == -1 and lib.mb_block_norm(None, None) == -1
    assert lib.mb_selective_scan_workspace_bytes(None) == 0


def test_nothing_to_do_is_no_error(lib):
    assert lib.mb_causal_conv1d(conv(batch=0), None) == 0 and lib.mb_selective_scan(scan(heads=0, groups=1), None, 0, None) == 0
    assert lib.mb_block_norm(norm(rows=0), None) == 0


def test_facade_checks_without_a_gpu(lib):
    from mockingbird_amd import _lib, ssm
    with pytest.raises(_lib.MbHipError, match="no CPU path"):
        ssm.causal_conv1d(torch.zeros(4, 8), torch.zeros(8, 4))
    with pytest.raises(_lib.MbHipError, match="float32, float16 or bfloat16"):
        ssm.block_norm(torch.zeros(4, 8, dtype=torch.int32))
    rows = torch.zeros(6, 10)
    assert ssm._rows("f", "t", rows[:, 2:6], (6,), (4,), torch.float32) == (0, 10)
    with pytest.raises(_lib.MbHipError, match="dense"):
        ssm._rows("f", "t", rows[:, ::2], (6,), (5,), torch.float32)
    ssm._apart("f", rows[:, :4], (6,), 4, ("x", rows[:, 4:8]))  # other columns of the same rows
    with pytest.raises(_lib.MbHipError, match="overlaps x"):
        ssm._apart("f", rows[:, :4], (6,), 4, ("x", rows[:, 3:7]))
    with pytest.raises(_lib.MbHipError, match="each other"):
        ssm._apart("f", rows[:1].expand(6, 10), (6,), 10)
    assert ssm._row_stride("f", "t", torch.zeros(2, 3, 8)[..., :5], torch.Size((2, 3, 5)), torch.float32) == 8
    with pytest.raises(_lib.MbHipError, match="evenly"):
        ssm._row_stride("f", "t", torch.zeros(2, 4, 8)[:, :3], torch.Size((2, 3, 8)), torch.float32)
