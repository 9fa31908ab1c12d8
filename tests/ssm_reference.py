"""The state-space operators in float64 on the CPU, row by row, each with a bound on the rounding error of an fp32 evaluation.

Bounds count half steps u(type): a result that is rounded once to `type` is off by u(type) * |result| (plus half the smallest subnormal);
U = 2^-24 is fp32's.  `slack` counts fp32 roundings, `scale` is the sum of the absolute values of the terms."""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def d64(t):
    return None if t is None else t.detach().cpu().double()


def rounded(value, err, dtype):
    """Bound of a value whose fp32 evaluation is off by err and that is then stored as dtype."""
    return err + HALF[dtype] * (value.abs() + err) + TINY[dtype]


def check(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), (what, "finite in different places")
    ok = torch.isfinite(want)
    over = ((got - want).abs() - bound)[ok]
    assert over.numel() == 0 or over.max() <= 0, (what, "over the bound by", over.max().item(), "bound", bound[ok].max().item())


def sequences(lens, packed, t):
    """[(first row, rows)] on the flattened row axis."""
    out, at = [], 0
    for i, n in enumerate(lens):
        out.append((at if packed else i * t, n))
        at += n
    return out


def silu_bound(v, err):
    """v * sigmoid(v) from a v off by err: the slope is at most 1.1; exp of an argument rounded to fp32 is off by |v| U relative,
    exp, sum, quotient and product by 8 U together, twice that where v_exp / v_rcp (1 ulp each) are used."""
    y = v * torch.sigmoid(v)
    return y, 1.1 * err + y.abs() * (v.abs() + 16) * 2 * U


def conv(x, weight, bias, act, seqs, state=None, slots=None, has_state=None):
    """(y, error of fp32 y, new state) on flattened rows; a slot of None leaves the item out; y rows of no item are NaN."""
    x, w, c = d64(x), d64(weight), x.shape[-1]
    k = w.shape[-1]
    w = w.reshape(c, k)
    b = d64(bias) if bias is not None else torch.zeros(c, dtype=torch.float64)
    y, bound = torch.full_like(x, float("nan")), torch.zeros_like(x)
    new = d64(state)
    for i, (at, n) in enumerate(seqs):
        slot = None
        if state is not None:
            slot = slots[i]
            if slot is None:
                continue
        head = torch.zeros(k - 1, c, dtype=torch.float64)
        if slot is not None and has_state[i]:
            head = d64(state)[slot]
        line = torch.cat([head, x[at:at + n]])
        v = b.expand(n, c).clone()
        s = b.abs().expand(n, c).clone()
        for j in range(k):
            v += w[:, j] * line[j:j + n]
            s += (w[:, j] * line[j:j + n]).abs()
        err = (k + 1) * U * s  # bias and k fused multiply-adds
        if act:
            v, err = silu_bound(v, err)
        y[at:at + n], bound[at:at + n] = v, err
        if slot is not None:
            new[slot] = line[n:]
    return y, bound, new


def scan(x, dt, A, B, C, D, dt_bias, softplus, limit, seqs, state=None, slots=None, has_state=None, planes=2.0 ** -21):
    """(y, error of fp32 y, new state, its error).  Rows are flattened: x [R,H,P], dt [R,H], B, C [R,G,N].

    The error of the state follows the recurrence itself: each step adds 8 fp32 roundings (decay and its exponent's |d A| U, step size,
    products, sums) of the absolute state.  The answer adds one rounding per column and the skip; `planes` is the relative error of
    products taken on split operands (hi + lo of 16-bit halves: 2^-16; three planes or fp32 itself: below 2^-21)."""
    x, dt, A, B, C = (d64(v) for v in (x, dt, A, B, C))
    D = d64(D) if D is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    h_, p, n_ = x.shape[1], x.shape[2], B.shape[2]
    rep = h_ // B.shape[1]
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    d = dt + (d64(dt_bias) if dt_bias is not None else 0.0)
    if softplus:
        d = torch.logaddexp(d, torch.zeros_like(d))
    if limit is not None:
        d = d.clamp(*limit)
    y, yerr = torch.full_like(x, float("nan")), torch.zeros_like(x)
    new = d64(state)
    nerr = None if state is None else torch.zeros_like(new)
    for i, (at, n) in enumerate(seqs):
        slot = None
        if state is not None:
            slot = slots[i]
            if slot is None:
                continue
        h = torch.zeros(h_, p, n_, dtype=torch.float64)
        if slot is not None and has_state[i]:
            h = d64(state)[slot]
        mag, err = h.abs(), torch.zeros_like(h)
        for t in range(at, at + n):
            da = d[t] * A
            decay = torch.exp(da)[:, None, None]
            inp = (d[t][:, None] * x[t])[:, :, None] * B[t][:, None, :]
            h = h * decay + inp
            mag = mag * decay + inp.abs()
            err = err * decay + U * (8 + da.abs())[:, None, None] * mag
            skip = D[:, None] * x[t]
            y[t] = (h * C[t][:, None, :]).sum(-1) + skip
            cabs = C[t].abs()[:, None, :]
            yerr[t] = (cabs * (err + (planes + (n_ + 4) * U) * mag)).sum(-1) + 4 * U * skip.abs() + planes * skip.abs()
        if slot is not None:
            new[slot], nerr[slot] = h, err + 2.0 ** -22 * mag
    return y, yerr, new, nerr


def gate_value(g, act):
    """(value, relative error)"""
    if act == "silu":
        return g * torch.sigmoid(g), (g.abs() + 16) * 2 * U
    if act == "sigmoid":
        return torch.sigmoid(g), (g.abs() + 16) * 2 * U
    return g, torch.zeros_like(g)


def norm_value(v, err, kind, weight, bias, groups, eps):
    """Norm of a v that is off by err (both [rows, channels]).  The mean is off by the mean error and n sum roundings, the centred values
    by that and their own; 1 / deviation by the root mean square of those relative to the deviation, and roundings."""
    if kind is None:
        return v, err
    r, c = v.shape
    n = c // groups
    p, e = v.reshape(r, groups, n), err.reshape(r, groups, n)
    roundings = (n / 64 + 16) * U  # partial sums of at most n / 64 values, then a tree
    if kind == "layer":
        mean = p.mean(-1, keepdim=True)
        e = e + e.mean(-1, keepdim=True) + roundings * p.abs().mean(-1, keepdim=True) + U * (p.abs() + mean.abs())
        p = p - mean
    dev = ((p * p).mean(-1, keepdim=True) + eps).sqrt()
    q = p / dev
    qerr = e / dev + q.abs() * ((e * e).mean(-1, keepdim=True).sqrt() / dev + roundings + 8 * U)
    q, qerr = q.reshape(r, c), qerr.reshape(r, c)
    if weight is not None:
        q, qerr = q * d64(weight), qerr * d64(weight).abs()
    if bias is not None:
        q = q + d64(bias)
        qerr = qerr + U * (q.abs() + d64(bias).abs())
    return q, qerr + 3 * U * q.abs()


def block_norm(x, weight=None, bias=None, norm="rms", eps=1e-5, groups=1, gate=None, gate_act="silu", gate_first=True, residual=None,
               scale=None, next_norm=None, next_weight=None, next_bias=None, next_eps=1e-5):
    """(s, error, y, error); the last two None without next_norm."""
    v = d64(x).reshape(-1, x.shape[-1])
    err = torch.zeros_like(v)

    def gated(v, err):
        g, rel = gate_value(d64(gate).reshape(v.shape), gate_act)
        return v * g, err * g.abs() + (v * g).abs() * (rel + U)

    if gate is not None and gate_first:
        v, err = gated(v, err)
    v, err = norm_value(v, err, norm, weight, bias, groups, eps)
    if gate is not None and not gate_first:
        v, err = gated(v, err)
    s = d64(scale) if torch.is_tensor(scale) else 1.0 if scale is None else scale
    v = v * s
    err = err * abs(s) + 3 * U * v.abs()
    if residual is not None:
        r = d64(residual).reshape(v.shape)
        err = err + U * (v.abs() + r.abs())
        v = v + r
    if next_norm is None:
        return v, err, None, None
    return (v, err) + norm_value(v, err, next_norm, next_weight, next_bias, 1, next_eps)
