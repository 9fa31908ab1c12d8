"""State-space decoder blocks on the MI355X (include/mbhip.h section 8): the short causal convolution, the selective scan -- each for
prompts and for single tokens -- and the norms, gate and residual sum around a block.

    h, u = block_norm(o_prev, residual=h, next_norm="rms", next_weight=w0)            # residual sum, norm of this block
    z, xbc, dt = in_proj(u).split(...)
    xbc = causal_conv1d(xbc, conv_w, conv_b, "silu", cu_seqlens=cu, state=conv_pool, slots=slots, has_state=has)
    y = selective_scan(x, dt, A, B, C, D, dt_bias=b, dt_softplus=True, cu_seqlens=cu, state=pool, slots=slots, has_state=has)
    o = out_proj(block_norm(y.flatten(-2), w1, gate=z, groups=8))                     # the gated norm behind the scan

and, token by token, causal_conv1d_step / selective_scan_step on the same pools.

Activations are float32, float16 or bfloat16 CUDA(HIP) tensors, time-major and dense within a row; rows may be strided (slices of a
projection).  Parameters and scan states are float32.  Packed requests are [rows, ...] with cu_seqlens (int32 [n + 1]), padded ones
[batch, t, ...] with optional lengths (int32 [batch]); both stay on the device.  Rows that belong to no request are left as `out` held them
(a fresh `out` is not initialised there).  state[slots[i]] is request i's state, updated in place; a request whose slot is outside the
pool, or already named by an earlier request of the call, is left out.  has_state[i] == False starts request i from zeros.  What a call writes
shares no memory with its other tensors (other columns of the same rows are fine).

Inference only: a tensor that requires grad is refused while grad mode is on, one with a forward-mode tangent always.  There is no CPU path."""
import ctypes as C

import torch
from torch.autograd import forward_ad

from .. import _lib

_DTYPES = {torch.float32: _lib.MB_F32, torch.float16: _lib.MB_F16, torch.bfloat16: _lib.MB_BF16}
_NORMS = {None: 0, "rms": 1, "layer": 2}
_GATES = {None: 0, "silu": 1, "sigmoid": 2}
_INF = float("inf")
_F32 = torch.float32


def _refuse(what):
    raise _lib.MbHipError(what)


def _inputs(fn, x, **others):
    """x fixes device and type; every other tensor must be on x's device, none may need a gradient.  Returns the device index."""
    try:
        index = x.get_device()  # -1 on the host
        good = index >= 0 and x.dtype in _DTYPES
        grad = torch.is_grad_enabled()
        wanted = grad and x.requires_grad
        for t in others.values():
            if t is not None:
                good = good and t.get_device() == index
                wanted = wanted or (grad and t.requires_grad)
        if good and not wanted:
            if forward_ad._current_level >= 0:  # -1 outside of dual_level()
                _refuse_tangents(fn, x=x, **others)
            return index
    except AttributeError:
        pass
    _refuse_inputs(fn, x, others)


def _refuse_tangents(fn, **tensors):
    """no_grad() does not keep forward-mode derivatives from being asked for; the results would carry none."""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            _refuse(f"{fn} has no derivative: {name} is a dual tensor")


def _refuse_inputs(fn, x, others):
    if not torch.is_tensor(x) or x.dtype not in _DTYPES:
        _refuse(f"{fn}: x must be a float32, float16 or bfloat16 tensor, not {getattr(x, 'dtype', type(x).__name__)}")
    if not x.is_cuda:
        _refuse(f"{fn} needs CUDA(HIP) tensors; there is no CPU path")
    for name, t in others.items():
        if t is None:
            continue
        if not torch.is_tensor(t):
            _refuse(f"{fn}: {name} must be a tensor, not {type(t).__name__}")
        if t.device != x.device:
            _refuse(f"{fn}: {name} is on {t.device}, x on {x.device}")
    for name, t in dict(x=x, **others).items():
        if t is not None and t.requires_grad:
            _refuse(f"{fn} has no backward: {name} requires grad (use torch.no_grad() or detach it)")


def _param(fn, name, t, *shape):
    """fp32, contiguous, of that shape; None stays None."""
    if t is None:
        return None
    if t.dtype is _F32 and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    _refuse(f"{fn}: {name} must be contiguous float32 {list(shape)}, got {t.dtype} {list(t.shape)} with strides {t.stride()}")


def _numbers(fn, name, t, dtype, n):
    """A device list of n row numbers / flags; None stays None."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    _refuse(f"{fn}: {name} must be a contiguous {dtype} tensor of {n}, got {t.dtype} {list(t.shape)}")


def _rows(fn, name, t, lead, tail, dtype):
    """(batch stride, row stride) of a tensor of `lead` rows of `tail`, dense within a row."""
    st, k = t.stride(), len(tail)
    if t.dtype is dtype and t.shape == lead + tail and st[-1] == 1 and (k == 1 or (st[-2] == tail[-1] and (
            k == 2 or st[-3] == tail[-1] * tail[-2]))):
        return (st[0], st[1]) if len(lead) == 2 else (0, st[0])
    if t.dtype is not dtype:
        _refuse(f"{fn}: {name} is {t.dtype}, expected {dtype}")
    if t.shape != lead + tail:
        _refuse(f"{fn}: {name} has shape {list(t.shape)}, expected {list(lead + tail)}")
    dense = 1
    for i in range(len(tail)):
        if tail[-1 - i] != 1 and st[-1 - i] != dense and t.numel():
            _refuse(f"{fn}: {name} must be dense within a row of {list(tail)}; its strides are {st}")
        dense *= tail[-1 - i]
    n = len(lead)
    return (st[0] if n == 2 else 0), st[n - 1]


def _fresh(x, lead, tail, bstride, rstride):
    """A new contiguous output of x's type with its (batch stride, row stride)."""
    return (torch.empty_like(x) if x.is_contiguous() else x.new_empty(lead + tail)), bstride, rstride


def _extent(t):
    """Address range of a tensor, empty tensors have none."""
    n = t.numel()
    if n == 0:
        return 0, 0
    lo = t.data_ptr()
    if not t.is_contiguous():
        n = 1
        for size, stride in zip(t.shape, t.stride()):
            n += (size - 1) * stride
    return lo, lo + t.element_size() * n


def _apart(fn, out, lead, row, *others):
    """An output must not hold a row twice, nor overlap another tensor of the call ((name, tensor) pairs) -- unless both are different columns
    of the same rows.  (The library looks at everything else that a call writes and reads.)"""
    if not out.is_contiguous():
        need = row
        for st, n in sorted((st, n) for st, n in zip(out.stride()[:len(lead)], lead) if n > 1):
            if st < need:
                _refuse(f"{fn}: out's rows overlap each other (strides {out.stride()})")
            need = st * (n - 1) + need
    lo, hi = _extent(out)
    for name, t in others:
        if t is None:
            continue
        a, b = _extent(t)
        if lo < b and a < hi and not _other_columns(out, t, a - lo):
            _refuse(f"{fn}: out overlaps {name}")


def _blocks(t):
    """(bytes of the dense block that a tensor repeats, byte strides of the axes that repeat it)."""
    e, width, front = t.element_size(), 1, []
    for n, st in zip(reversed(t.shape), reversed(t.stride())):
        if n == 1:
            continue
        if not front and st == width:
            width *= n
        else:
            front.append(st * e)
    return width * e, front


def _other_columns(t, u, off):
    """u, `off` bytes behind t, holds other columns of the same rows: both repeat a block at multiples of one row, and the blocks lie apart."""
    (wt, ft), (wu, fu) = _blocks(t), _blocks(u)
    steps = ft + fu
    step = min((st for st in steps if st), default=0)
    if not step or any(st % step for st in steps):  # (a batch that starts inside a row of the others: columns do not tell them apart)
        return False
    off %= step
    return off >= wt and off + wu <= step


# torch.cuda.current_stream(index).cuda_stream and torch.cuda.current_device() without the objects and the start-up check around them (there
# are tensors on the device).  A call of one token is a few microseconds of kernel: what the host spends per call is most of its time.
_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


def _launch(fn, index, call, *args):
    """The call on the current stream of the tensors' device."""
    if index == _device():
        rc = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, fn)


def _requests(fn, lead, cu_seqlens, lengths):
    """(requests, rows per request or in all, cu pointer, lengths pointer)."""
    if len(lead) == 1:
        if cu_seqlens is None:
            _refuse(f"{fn}: packed rows need cu_seqlens (or pass [batch, t, ...])")
        if lengths is not None:
            _refuse(f"{fn}: lengths belong to padded [batch, t, ...] tensors, not to packed rows")
        n = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
        if n < 0:
            _refuse(f"{fn}: cu_seqlens must be one-dimensional with one entry more than there are requests")
        return n, lead[0], _numbers(fn, "cu_seqlens", cu_seqlens, torch.int32, n + 1), None
    if cu_seqlens is not None:
        _refuse(f"{fn}: cu_seqlens belong to packed [rows, ...] tensors, not to padded ones")
    return lead[0], lead[1], None, _numbers(fn, "lengths", lengths, torch.int32, lead[0])


def _pool(fn, state, dtype, inner, batch, slots, has_state):
    """(state pointer, slot stride, slots in the pool, slot pointer, flag pointer)."""
    if state is None:
        if slots is not None or has_state is not None:
            _refuse(f"{fn}: slots and has_state belong to a state pool")
        return None, 0, 0, None, None
    shape = state.shape
    if len(shape) != 1 + len(inner):
        _refuse(f"{fn}: state must have shape [slots, {', '.join(map(str, inner))}], got {list(shape)}")
    n = shape[0]
    stride = _rows(fn, "state", state, (n,), inner, dtype)[1]
    if n > 1 and stride < (inner[0] * inner[1] if len(inner) == 2 else inner[0] * inner[1] * inner[2]):
        _refuse(f"{fn}: state's slots overlap each other (strides {state.stride()})")
    if slots is None and batch > n:
        _refuse(f"{fn}: {batch} requests without slots, but a pool of {n}")
    return (state.data_ptr(), stride, n, None if slots is None else _numbers(fn, "slots", slots, torch.int32, batch),
            None if has_state is None else _numbers(fn, "has_state", has_state, torch.bool, batch))


def _conv_weight(fn, weight, channels):
    if weight is None:
        _refuse(f"{fn}: weight is required")
    if weight.dim() == 3 and weight.shape[1] == 1:  # torch's depthwise layout [channels, 1, taps]
        weight = weight[:, 0]
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        _refuse(f"{fn}: weight must be [channels, taps] or [channels, 1, taps] with 2..8 taps, got {list(weight.shape)}")
    return _param(fn, "weight", weight, channels, weight.shape[1]), weight.shape[1]


def _activation(fn, activation):
    if activation not in (None, "silu"):
        _refuse(f"{fn}: activation must be None or 'silu', not {activation!r}")
    return 0 if activation is None else 1


def causal_conv1d(x, weight, bias=None, activation=None, *, cu_seqlens=None, lengths=None, state=None, slots=None, has_state=None,
                  out=None):
    """Depthwise causal convolution y[t, c] = act(bias[c] + sum_j weight[c, j] * x[t - taps + 1 + j, c]) of packed x [rows, channels] or padded
    x [batch, t, channels]; taps 2..8, activation None or "silu".  state [slots, taps - 1, channels] of x's type holds the last inputs
    of every request, oldest first."""
    fn = "causal_conv1d"
    index = _inputs(fn, x, weight=weight, bias=bias, cu_seqlens=cu_seqlens, lengths=lengths, state=state, slots=slots, has_state=has_state,
                    out=out)
    if x.dim() not in (2, 3):
        _refuse(f"{fn}: x must be [rows, channels] or [batch, t, channels], got {list(x.shape)}")
    lead, c = tuple(x.shape[:-1]), x.shape[-1]
    batch, t, cu, valid = _requests(fn, lead, cu_seqlens, lengths)
    xb, xr = _rows(fn, "x", x, lead, (c,), x.dtype)
    w, k = _conv_weight(fn, weight, c)
    st, st_stride, n_slots, sl, has = _pool(fn, state, x.dtype, (k - 1, c), batch, slots, has_state)
    if out is None:
        out, yb, yr = _fresh(x, lead, (c,), t * c, c)
    else:
        _apart(fn, out, lead, c, ("x", x), ("state", state))
        yb, yr = _rows(fn, "out", out, lead, (c,), x.dtype)
    a = _lib.CausalConv1dArgs(x.data_ptr(), out.data_ptr(), w, _param(fn, "bias", bias, c), st, sl, has, cu, valid, xb, xr, yb, yr,
                              st_stride, _DTYPES[x.dtype], batch, t, c, k, _activation(fn, activation), n_slots)
    _launch(fn, index, _lib.lib().mb_causal_conv1d, C.byref(a))
    return out


def causal_conv1d_step(x, state, weight, bias=None, activation=None, *, slots=None, out=None):
    """One token for each request: x [batch, channels] with the states of causal_conv1d, which move on by one input."""
    fn = "causal_conv1d_step"
    index = _inputs(fn, x, state=state, weight=weight, bias=bias, slots=slots, out=out)
    if x.dim() != 2:
        _refuse(f"{fn}: x must be [batch, channels], got {list(x.shape)}")
    if state is None:
        _refuse(f"{fn} needs a state pool")
    b, c = x.shape
    _, xr = _rows(fn, "x", x, (b,), (c,), x.dtype)
    w, k = _conv_weight(fn, weight, c)
    st, st_stride, n_slots, sl, _ = _pool(fn, state, x.dtype, (k - 1, c), b, slots, None)
    if out is None:
        out, _, yr = _fresh(x, (b,), (c,), 0, c)
    else:
        _apart(fn, out, (b,), c, ("x", x), ("state", state))
        _, yr = _rows(fn, "out", out, (b,), (c,), x.dtype)
    a = _lib.CausalConv1dArgs(x.data_ptr(), out.data_ptr(), w, _param(fn, "bias", bias, c), st, sl, None, None, None, 0, xr, 0, yr,
                              st_stride, _DTYPES[x.dtype], b, 1, c, k, _activation(fn, activation), n_slots)
    _launch(fn, index, _lib.lib().mb_causal_conv1d_step, C.byref(a))
    return out


def _scan_args(fn, step, x, dt, A, B, C_, D, dt_bias, dt_softplus, dt_limit, cu_seqlens, lengths, state, slots, has_state, out):
    index = _inputs(fn, x, dt=dt, A=A, B=B, C=C_, D=D, dt_bias=dt_bias, cu_seqlens=cu_seqlens, lengths=lengths, state=state, slots=slots,
                    has_state=has_state, out=out)
    for name, t in (("dt", dt), ("A", A), ("B", B), ("C", C_)):
        if t is None:
            _refuse(f"{fn}: {name} is required")
    if x.dim() != 3 and (step or x.dim() != 4):
        _refuse(f"{fn}: x must be {'[batch, heads, head_dim]' if step else '[rows, heads, head_dim] or [batch, t, heads, head_dim]'}, "
                f"got {list(x.shape)}")
    lead, (h, p) = tuple(x.shape[:-2]), x.shape[-2:]
    if step:
        if state is None:
            _refuse(f"{fn} needs a state pool")
        batch, t, cu, valid = lead[0], 1, None, None
    else:
        batch, t, cu, valid = _requests(fn, lead, cu_seqlens, lengths)
    if B.dim() != len(lead) + 2:
        _refuse(f"{fn}: B must have x's leading sizes and [groups, d_state], got {list(B.shape)}")
    g, n = B.shape[-2:]
    if not 1 <= p <= 128 or not 1 <= n <= 256:
        _refuse(f"{fn}: head_dim {p} is outside 1..128 or d_state {n} outside 1..256")
    if g < 1 or h % g:
        _refuse(f"{fn}: {h} heads do not divide into {g} groups")
    lo, hi = (-_INF, _INF) if dt_limit is None else map(float, dt_limit)
    if not lo <= hi:
        _refuse(f"{fn}: dt_limit {dt_limit} is no range")
    xb, xr = _rows(fn, "x", x, lead, (h, p), x.dtype)
    db, dr = _rows(fn, "dt", dt, lead, (h,), torch.float32 if dt.dtype is torch.float32 else x.dtype)
    bb, br = _rows(fn, "B", B, lead, (g, n), x.dtype)
    cb, cr = _rows(fn, "C", C_, lead, (g, n), x.dtype)
    st, st_stride, n_slots, sl, has = _pool(fn, state, torch.float32, (h, p, n), batch, slots, has_state)
    if out is None:
        out, yb, yr = _fresh(x, lead, (h, p), t * h * p, h * p)
    else:
        _apart(fn, out, lead, h * p, ("x", x), ("dt", dt), ("B", B), ("C", C_), ("state", state))
        yb, yr = _rows(fn, "out", out, lead, (h, p), x.dtype)
    a = _lib.SelectiveScanArgs(x.data_ptr(), out.data_ptr(), dt.data_ptr(), B.data_ptr(), C_.data_ptr(), _param(fn, "A", A, h),
                               _param(fn, "D", D, h), _param(fn, "dt_bias", dt_bias, h), st, sl, has, cu, valid, xb, xr, yb, yr, db, dr,
                               bb, br, cb, cr, st_stride, _DTYPES[x.dtype], _DTYPES[dt.dtype], batch, t, h, p, g, n, n_slots,
                               1 if dt_softplus else 0, lo, hi)
    return index, a, out


def selective_scan(x, dt, A, B, C, D=None, *, dt_bias=None, dt_softplus=False, dt_limit=None, cu_seqlens=None, lengths=None, state=None,
                   slots=None, has_state=None, out=None):
    """Per head d = clamp(softplus(dt + dt_bias), dt_limit); h = exp(d * A) * h + (d * x) B^T; y = h C + D * x.
    x [rows | batch, t, heads, head_dim], dt [.., heads] (x's type or float32), A, D, dt_bias [heads], B, C [.., groups, d_state] where
    head i reads group i // (heads // groups); state float32 [slots, heads, head_dim, d_state].  head_dim <= 128, d_state <= 256."""
    fn = "selective_scan"
    index, a, out = _scan_args(fn, False, x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, cu_seqlens, lengths, state, slots, has_state,
                               out)
    lib = _lib.lib()
    need = lib.mb_selective_scan_workspace_bytes(a)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    _launch(fn, index, lib.mb_selective_scan, a, _lib.ptr(ws), need)
    return out


def selective_scan_step(x, dt, A, B, C, state, D=None, *, dt_bias=None, dt_softplus=False, dt_limit=None, slots=None, out=None):
    """One token for each request: x [batch, heads, head_dim], dt [batch, heads], B, C [batch, groups, d_state] with the states of
    selective_scan, which move on by one step."""
    fn = "selective_scan_step"
    index, a, out = _scan_args(fn, True, x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, None, None, state, slots, None, out)
    _launch(fn, index, _lib.lib().mb_selective_scan_step, a)
    return out


def _row_stride(fn, name, t, shape, dtype):
    """Row stride of a [..., channels] tensor whose leading axes form one evenly spaced axis of rows."""
    if t.dtype is not dtype:
        _refuse(f"{fn}: {name} is {t.dtype}, expected {dtype}")
    if t.shape != shape:
        _refuse(f"{fn}: {name} has shape {list(t.shape)}, expected {list(shape)}")
    if t.is_contiguous():
        return shape[-1]
    st = t.stride()
    if len(st) == 2 and st[1] == 1 and shape[0] > 1:
        return st[0]
    if shape[-1] > 1 and st[-1] != 1:
        _refuse(f"{fn}: {name} must be dense within a row; its strides are {st}")
    step, rows = None, 1
    for n, s in zip(reversed(shape[:-1]), reversed(st[:-1])):
        if n == 1:
            continue
        if step is None:
            step = s
        elif s != step * rows:
            _refuse(f"{fn}: {name}'s leading axes must form evenly spaced rows; shape {list(shape)}, strides {st}")
        rows *= n
    return shape[-1] if step is None else step


def _same_or_apart(fn, name, out, stride, others):
    """An output is exactly one of the inputs (same address, rows and element size) or overlaps none of them."""
    lo, hi = _extent(out)
    for other, t, other_stride in others:
        a, b = _extent(t)
        if lo >= b or a >= hi:
            continue
        width = out.shape[-1] * out.element_size()
        if out.element_size() == t.element_size() and stride == other_stride:
            off = (a - lo) % (stride * out.element_size()) if stride else 0
            if (lo == a and not other.startswith("*")) or (off >= width and off + width <= stride * out.element_size()):
                continue
        _refuse(f"{fn}: {name} overlaps {other.lstrip('*')}")


def block_norm(x, weight=None, bias=None, *, norm="rms", eps=1e-5, groups=1, gate=None, gate_act="silu", gate_first=True, residual=None,
               scale=None, next_norm=None, next_weight=None, next_bias=None, next_eps=1e-5, out=None, residual_out=None):
    """The seam between two blocks, row by row:
        u = x * gate_act(gate) if gate_first;  v = norm(u) (over each of `groups` parts of the row);  v *= gate_act(gate) if not gate_first;
        s = residual + scale * v;  y = next_norm(s).
    Returns s (x's type, or residual's with one) without next_norm, else (s, y).  norm / next_norm: "rms", "layer" or None; weights and
    biases float32 [channels]; scale a number or float32 [channels]; residual x's type or float32.  out receives y (s without
    next_norm), residual_out receives s; either may be exactly one of the inputs."""
    fn = "block_norm"
    vec = torch.is_tensor(scale)
    index = _inputs(fn, x, weight=weight, bias=bias, gate=gate, residual=residual, scale=scale if vec else None, next_weight=next_weight,
                    next_bias=next_bias, out=out, residual_out=residual_out)
    if norm not in _NORMS or next_norm not in _NORMS:
        _refuse(f"{fn}: norm and next_norm must be 'rms', 'layer' or None, not {norm!r} and {next_norm!r}")
    if gate_act not in _GATES:
        _refuse(f"{fn}: gate_act must be 'silu', 'sigmoid' or None, not {gate_act!r}")
    if x.dim() < 1:
        _refuse(f"{fn}: x must have a channel axis")
    shape, c = x.shape, x.shape[-1]
    if norm is None and (weight is not None or bias is not None):
        _refuse(f"{fn}: weight and bias belong to norm")
    if next_norm is None and (next_weight is not None or next_bias is not None):
        _refuse(f"{fn}: next_weight and next_bias belong to next_norm")
    if not isinstance(groups, int) or not 1 <= groups <= 1024 or c % groups or (norm is None and groups != 1):
        _refuse(f"{fn}: {c} channels in {groups!r} groups (1..1024 equal ones, of the first norm)")
    if norm is None and next_norm is None and residual is None and gate is None:
        _refuse(f"{fn}: nothing to compute")
    dtype = sum_dtype = x.dtype
    xs = _row_stride(fn, "x", x, shape, dtype)
    gs = rs = 0
    if gate is not None:
        gs = _row_stride(fn, "gate", gate, shape, dtype)
    if residual is not None:
        if residual.dtype is _F32:
            sum_dtype = _F32
        rs = _row_stride(fn, "residual", residual, shape, sum_dtype)
    reads = [(name, t, st) for name, t, st in (("x", x, xs), ("gate", gate, gs), ("residual", residual, rs)) if t is not None] \
        if out is not None or residual_out is not None else ()
    if next_norm is None:
        if out is not None and residual_out is not None:
            _refuse(f"{fn}: without next_norm there is one result: out or residual_out")
        total, y = (out if residual_out is None else residual_out), None
    else:
        total, y = residual_out, out
    rows = x.numel() // c if c else 0
    if total is None:
        like = x if residual is None else residual  # of the sum's type
        total, ss = (torch.empty_like(like) if like.is_contiguous() else like.new_empty(shape)), c
    else:
        ss = _row_stride(fn, "residual_out" if next_norm or residual_out is not None else "out", total, shape, sum_dtype)
        if rows > 1 and ss < c:
            _refuse(f"{fn}: the result's rows overlap each other")
        _same_or_apart(fn, "the sum", total, ss, reads)
    ys = 0
    if next_norm is not None:
        if y is None:
            y, ys = (torch.empty_like(x) if x.is_contiguous() else x.new_empty(shape)), c
        else:
            ys = _row_stride(fn, "out", y, shape, dtype)
            if rows > 1 and ys < c:
                _refuse(f"{fn}: out's rows overlap each other")
            _same_or_apart(fn, "out", y, ys, [*reads, ("*the sum", total, ss)])
    a = _lib.BlockNormArgs(x.data_ptr(), None if gate is None else gate.data_ptr(), None if residual is None else residual.data_ptr(),
                           total.data_ptr(), None if y is None else y.data_ptr(), _param(fn, "weight", weight, c),
                           _param(fn, "bias", bias, c), _param(fn, "scale", scale, c) if vec else None,
                           _param(fn, "next_weight", next_weight, c), _param(fn, "next_bias", next_bias, c), rows, xs, gs, rs, ss, ys,
                           _DTYPES[dtype], _DTYPES[sum_dtype], c, groups, _NORMS[norm], _NORMS[next_norm], _GATES[gate_act],
                           1 if gate_first else 0, eps, next_eps, 1.0 if scale is None or vec else float(scale))
    _launch(fn, index, _lib.lib().mb_block_norm, C.byref(a))
    return total if y is None else (total, y)
