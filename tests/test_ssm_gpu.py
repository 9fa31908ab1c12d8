"""The state-space operators (mockingbird_amd.ssm) against float64 on the CPU, with bounds derived in ssm_reference.py."""
import itertools

import pytest
import torch

import ssm_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
NAN = float("nan")


@pytest.fixture(autouse=True)
def _library(cuda, lib):
    pass


def gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *shape, scale=1.0, dtype=F32: (torch.randn(*shape, generator=g) * scale).to(dtype)


def pool_of(n, inner, seqs, r, dtype, order=None):
    """A pool with live slots in odd order, (pool, slots, has_state): the slot of an item without state holds NaN."""
    b = len(seqs)
    slots = order or [(5 * i + 2) % (b + 4) for i in range(b)]
    if order is None and len(set(slots)) != b:
        slots = list(range(b, 0, -1))
    has = [i % 3 != 1 for i in range(b)]
    pool = r(b + 4, *inner, dtype=dtype)
    for s, k in zip(slots, has):
        if not k:
            pool[s] = NAN
    return pool, slots, has


def meta(lens, packed):
    if packed:
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        return dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda()), (cu[-1],), None
    return dict(lengths=torch.tensor(lens, dtype=torch.int32).cuda()), (len(lens), max(lens)), max(lens)


def slot_args(slots, has):
    return dict(slots=torch.tensor(slots, dtype=torch.int32).cuda(), has_state=torch.tensor(has).cuda())


def strided(t, extra, offset):
    """t as a slice of wider rows (inner axes stay dense)."""
    n = t.shape[-1]
    wide = torch.full(t.shape[:-1] + (n + extra,), NAN, dtype=t.dtype, device="cuda")
    wide[..., offset:offset + n] = t.cuda()
    return wide[..., offset:offset + n]


LENGTHS = [[1], [0, 5, 1, 2, 0, 37], [130, 3], [64, 65, 63, 1, 0, 200]]


# ------------------------------------------------------------------------------------------- convolution

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,k,act", [(96, 4, "silu"), (200, 3, None), (37, 2, "silu"), (1, 8, None), (1032, 5, "silu"), (64, 7, "silu")])
@pytest.mark.parametrize("packed", [True, False])
def test_causal_conv1d(dtype, channels, k, act, packed):
    from mockingbird_amd import ssm
    for seed, lens in enumerate(LENGTHS):
        r = gen(seed + channels)
        args, lead, t = meta(lens, packed)
        x, w, b = r(*lead, channels, dtype=dtype), r(channels, k, scale=0.5), r(channels)
        seqs = ref.sequences(lens, packed, t)
        pool, slots, has = pool_of(len(lens), (k - 1, channels), seqs, r, dtype)
        for state in (False, True):
            dpool = pool.cuda() if state else None
            out = torch.full(x.shape, 7.0, dtype=dtype, device="cuda")
            more = dict(state=dpool, **slot_args(slots, has)) if state else {}
            xd = x.cuda() if seed % 2 else strided(x, 24, 16)
            y = ssm.causal_conv1d(xd, w.cuda(), b.cuda() if seed else None, act, out=out, **args, **more)
            assert y is out
            want, err, new = ref.conv(x.reshape(-1, channels), w, b if seed else None, act, seqs, pool if state else None, slots, has)
            rows = torch.isnan(want)[:, 0] if channels and want.numel() else torch.zeros(0, dtype=torch.bool)
            got = y.reshape(-1, channels).cpu()
            assert (got[rows] == 7.0).all(), "rows of no item were written"
            ref.check(got[~rows], want[~rows], ref.rounded(want, err, dtype)[~rows], (lens, state))
            if state:  # inputs are moved, not computed: bit for bit
                keep = torch.ones(pool.shape[0], dtype=torch.bool)
                keep[slots] = False
                assert torch.equal(dpool.cpu()[slots].double(), new[slots])
                assert torch.equal(torch.nan_to_num(dpool.cpu()[keep].float(), nan=9.0), torch.nan_to_num(pool[keep].float(), nan=9.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,channels,k,act", [(1, 64, 4, "silu"), (5, 37, 2, None), (70, 520, 3, "silu"), (3, 8, 8, None), (130, 96, 4, "silu")])
def test_causal_conv1d_step(dtype, batch, channels, k, act):
    from mockingbird_amd import ssm
    r = gen(batch)
    x, w, b = r(batch, channels, dtype=dtype), r(channels, k, scale=0.5), r(channels)
    pool = r(batch + 3, k - 1, channels, dtype=dtype)
    slots = [(i * 7 + 1) % (batch + 3) for i in range(batch)]
    if len(set(slots)) != batch:
        slots = list(range(batch - 1, -1, -1))
    dpool = pool.cuda()
    y = ssm.causal_conv1d_step(strided(x, 8, 8), dpool, w.cuda()[:, None], b.cuda(), act, slots=torch.tensor(slots, dtype=torch.int32).cuda())
    want, err, new = ref.conv(x, w, b, act, [(i, 1) for i in range(batch)], pool, slots, [True] * batch)
    ref.check(y, want, ref.rounded(want, err, dtype))
    assert torch.equal(dpool.cpu().double(), new)


# -------------------------------------------------------------------------------------------------- scan

SHAPES = [  # heads, head_dim, d_state, groups
    (2, 64, 128, 1), (4, 32, 64, 2), (3, 48, 40, 3), (5, 17, 20, 1), (2, 128, 256, 2), (1, 1, 1, 1), (6, 64, 16, 1), (4, 100, 100, 4), (1, 63, 255, 1)]


def scan_inputs(r, lead, h, p, n, g, dtype):
    x, bm, cm = r(*lead, h, p, dtype=dtype), r(*lead, g, n, dtype=dtype), r(*lead, g, n, dtype=dtype)
    dt = r(*lead, h, scale=0.5, dtype=dtype)
    a = -(r(h).abs() * 4 + 0.5)
    bias, skip = r(h) - 3.0, r(h)
    return x, dt, a, bm, cm, skip, bias


# products on split operands: 16-bit types keep two planes (2^-16 relative), fp32 three
PLANES = {F32: 2.0 ** -21, F16: 2.0 ** -15, BF16: 2.0 ** -15}


def flat(t, k):
    return t.reshape(-1, *t.shape[t.dim() - k:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("packed", [True, False])
def test_selective_scan(dtype, shape, packed):
    from mockingbird_amd import ssm
    h, p, n, g = shape
    for seed, lens in enumerate(LENGTHS):
        r = gen(seed + h * p)
        args, lead, t = meta(lens, packed)
        x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
        seqs = ref.sequences(lens, packed, t)
        pool, slots, has = pool_of(len(lens), (h, p, n), seqs, r, F32)
        state = seed != 1
        dpool = pool.cuda() if state else None
        more = dict(state=dpool, **slot_args(slots, has)) if state else {}
        out = torch.full(x.shape, 7.0, dtype=dtype, device="cuda")
        d_skip = skip if seed % 2 == 0 else None
        y = ssm.selective_scan(strided(x.flatten(-2), 24, 16).unflatten(-1, (h, p)), dt.cuda(), a.cuda(), strided(bm.flatten(-2), 9, 3).unflatten(-1, (g, n)),
                               cm.cuda(), None if d_skip is None else skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, out=out, **args, **more)
        want, err, new, nerr = ref.scan(flat(x, 2), flat(dt, 1), a, flat(bm, 2), flat(cm, 2), d_skip, bias, True, None, seqs,
                                        pool if state else None, slots, has, PLANES[dtype])
        got = y.reshape(-1, h, p).cpu()
        rows = torch.isnan(want)[:, 0, 0]
        assert (got[rows] == 7.0).all(), "rows of no item were written"
        ref.check(got[~rows], want[~rows], ref.rounded(want, err, dtype)[~rows], (lens, "y"))
        if state:
            ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs() + ref.TINY[F32], (lens, "state"))
            rest = [i for i in range(pool.shape[0]) if i not in slots]
            assert torch.equal(dpool.cpu()[rest], pool[rest])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[1500], [700, 2, 0, 641], [400] * 3])
def test_selective_scan_long(dtype, lens):
    """Long enough to be split along time when there are few heads, with states that remember the first rows."""
    from mockingbird_amd import ssm
    h, p, n, g = 2, 32, 32, 1
    r = gen(len(lens))
    args, lead, t = meta(lens, True)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
    a, bias = a * 0.05, bias - 2.0
    pool, slots, has = pool_of(len(lens), (h, p, n), lens, r, F32)
    dpool = pool.cuda()
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, state=dpool,
                           **args, **slot_args(slots, has))
    want, err, new, nerr = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, ref.sequences(lens, True, t), pool, slots, has, PLANES[dtype])
    ref.check(y, want, ref.rounded(want, err, dtype))
    ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softplus,limit,dt32", [(False, None, True), (True, (0.01, 0.05), False), (False, (0.0, 100.0), False)])
def test_selective_scan_step_sizes(dtype, softplus, limit, dt32):
    """Without softplus, clamped, in fp32 beside 16-bit activations; strong decays that leave nothing of the state; dt = 0 rows do nothing."""
    from mockingbird_amd import ssm
    h, p, n, g, t = 3, 24, 16, 1, 90
    r = gen(11)
    x, dt, a, bm, cm, skip, _ = scan_inputs(r, (2, t), h, p, n, g, dtype)
    dt = dt.float().abs() * 0.1 if not softplus else dt.float()
    dt[:, 40] = 0.0
    dt[:, 60] = 30.0
    dt = dt.to(F32 if dt32 else dtype)
    pool = r(2, h, p, n)
    dpool = pool.cuda()
    y = ssm.selective_scan(x.cuda(), dt.cuda(), (a * 5).cuda(), bm.cuda(), cm.cuda(), dt_softplus=softplus, dt_limit=limit, state=dpool)
    want, err, new, nerr = ref.scan(flat(x, 2), flat(dt, 1), a * 5, flat(bm, 2), flat(cm, 2), None, None, softplus, limit,
                                    [(0, t), (t, t)], pool, [0, 1], [True] * 2, PLANES[dtype])
    ref.check(flat(y, 2), want, ref.rounded(want, err, dtype))
    ref.check(dpool, new, nerr + ref.HALF[F32] * new.abs() + ref.TINY[F32])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["x", "B", "C", "dt"])
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_selective_scan_stays_causal_around_nan(dtype, what, value):
    """A NaN or infinity in a row changes no row before it (nor another item), and every head that reads it stays non-finite behind it."""
    from mockingbird_amd import ssm
    h, p, n, g, lens = 2, 20, 24, 1, [75, 30]
    r = gen(5)
    args, lead, t = meta(lens, True)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
    bad = dict(x=x, B=bm, C=cm, dt=dt)[what]
    bad[42] = value
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, **args).cpu()
    clean = dict(x=x, B=bm, C=cm, dt=dt)
    clean[what] = bad.clone()
    clean[what][42] = 0.5
    want, err, _, _ = ref.scan(clean["x"], clean["dt"], a, clean["B"], clean["C"], skip, bias, True, None, ref.sequences(lens, True, t),
                               planes=PLANES[dtype])
    bound = ref.rounded(want, err, dtype)
    ref.check(y[:42], want[:42], bound[:42], "before")
    ref.check(y[75:], want[75:], bound[75:], "the next item")
    assert not torch.isfinite(y[42]).any()
    if what == "C":
        ref.check(y[43:75], want[43:75], bound[43:75], "behind")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,shape", [(1, (2, 64, 128, 1)), (3, (3, 48, 40, 3)), (9, (5, 17, 21, 1)), (2, (2, 128, 256, 2)), (70, (4, 32, 64, 2)), (1, (1, 1, 1, 1)), (2, (2, 100, 255, 1)),
                                         (4, (64, 64, 128, 1))])
def test_selective_scan_step(dtype, batch, shape):
    from mockingbird_amd import ssm
    h, p, n, g = shape
    r = gen(batch + p)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, (batch,), h, p, n, g, dtype)
    pool = r(batch + 2, h, p, n)
    slots = list(range(batch, 0, -1))
    dpool = pool.cuda()
    y = ssm.selective_scan_step(strided(x.flatten(-2), 8, 0).unflatten(-1, (h, p)), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), dpool, skip.cuda(),
                                dt_bias=bias.cuda(), dt_softplus=True, slots=torch.tensor(slots, dtype=torch.int32).cuda())
    want, err, new, nerr = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, [(i, 1) for i in range(batch)], pool, slots, [True] * batch)
    ref.check(y, want, ref.rounded(want, err, dtype))
    ref.check(dpool, new, nerr + ref.HALF[F32] * new.abs() + ref.TINY[F32])


# -------------------------------------------------------------------------------------------------- norms

NORMS = [  # norm, groups, gate, gate_first, residual, scale, next_norm
    ("rms", 1, None, True, False, None, None), ("layer", 1, None, True, False, None, None), (None, 1, None, True, True, None, "rms"),
    ("rms", 4, "silu", True, False, None, None), ("rms", 1, "sigmoid", False, True, "vector", "layer"), ("layer", 2, "silu", False, True, 0.3, "rms"),
    (None, 1, "none", True, True, 0.5, "layer"), ("rms", 1, None, True, True, "vector", None), (None, 1, "silu", True, False, None, None),
    ("rms", 4, "silu", True, True, "vector", "rms")]


@pytest.mark.parametrize("dtype,res", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("form", NORMS, ids=lambda f: "-".join(map(str, f)))
def test_block_norm(dtype, res, form):
    from mockingbird_amd import ssm
    norm, groups, gate, first, residual, scale, nxt = form
    for rows, c in [(1, 64), (3, 1024), (5, 36), (2, 4096), (130, 512), (2, 5120), (1, 12000), (7, 100 * 8)]:
        r = gen(rows + c)
        x = r(rows, c, scale=2.0, dtype=dtype) + 0.5
        kw = dict(norm=norm, groups=groups, gate_act=None if gate in (None, "none") else gate, gate_first=first, next_norm=nxt)
        tensors = {}
        if norm:
            tensors.update(weight=r(c) + 1.0, bias=r(c) if norm == "layer" else None)
        if gate:
            tensors["gate"] = r(rows, c, dtype=dtype)
        if residual:
            tensors["residual"] = r(rows, c, scale=3.0, dtype=res)
        if scale:
            tensors["scale"] = r(c) if scale == "vector" else scale
        if nxt:
            tensors.update(next_weight=r(c) + 1.0, next_bias=r(c) if nxt == "layer" else None)
        dev = {k: (strided(v, 40, 8) if k in ("gate",) else v.cuda()) if torch.is_tensor(v) else v for k, v in tensors.items()}
        got = ssm.block_norm(x.cuda(), **dev, **kw)
        s, serr, y, yerr = ref.block_norm(x, **tensors, **kw)
        total = got if nxt is None else got[0]
        sum_type = res if residual else dtype
        assert total.dtype is sum_type
        ref.check(total, s, ref.rounded(s, serr, sum_type), (rows, c, "sum"))
        if nxt:
            ref.check(got[1], y, ref.rounded(y, yerr, dtype), (rows, c, "y"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,c", [(3, 1), (4, 1001), (2, 33), (6, 4099), (1, 70001)])
def test_block_norm_odd_widths(dtype, rows, c):
    from mockingbird_amd import ssm
    r = gen(c)
    x, w, g, res, w2, b2 = r(rows, c, dtype=dtype), r(c), r(rows, c, dtype=dtype), r(rows, c, dtype=dtype), r(c), r(c)
    kw = dict(norm="rms", gate_act="silu", gate_first=True, scale=0.7, next_norm="layer")
    a, y = ssm.block_norm(x.cuda(), w.cuda(), gate=g.cuda(), residual=res.cuda(), next_weight=w2.cuda(), next_bias=b2.cuda(), **kw)
    s, serr, want, err = ref.block_norm(x, w, gate=g, residual=res, next_weight=w2, next_bias=b2, **kw)
    ref.check(a, s, ref.rounded(s, serr, dtype))
    if c > 1:  # one channel: a layer norm's deviation is sqrt(eps), its centred value a rounding
        ref.check(y, want, ref.rounded(want, err, dtype))


def test_block_norm_in_place_and_views():
    """Outputs on the inputs' own buffers, [batch, t, channels] views, a gate row shared by every row (stride 0)."""
    from mockingbird_amd import ssm
    r = gen(3)
    x, h, w, g = r(4, 6, 256, dtype=BF16), r(4, 6, 256), r(256), r(256, dtype=BF16)
    plain = ssm.block_norm(x.cuda(), w.cuda(), gate=g.cuda().expand(4, 6, 256), residual=h.cuda(), next_norm="rms", next_weight=w.cuda())
    xd, hd = x.cuda(), h.cuda()
    s, y = ssm.block_norm(xd, w.cuda(), gate=g.cuda().expand(4, 6, 256), residual=hd, next_norm="rms", next_weight=w.cuda(), out=xd, residual_out=hd)
    assert s is hd and y is xd and torch.equal(s, plain[0]) and torch.equal(y, plain[1])
    want = ref.block_norm(x, w, gate=g.expand(4, 6, 256), residual=h, next_norm="rms", next_weight=w)
    ref.check(s.reshape(-1, 256), want[0], ref.rounded(want[0], want[1], F32))


def test_block_norm_zero_and_extreme_rows():
    """A row of zeros gives zeros (eps keeps the deviation), huge rows do not overflow the statistics' result type for nothing, and a
    NaN stays in its row."""
    from mockingbird_amd import ssm
    x = torch.randn(5, 512, generator=torch.Generator().manual_seed(1))
    x[1], x[2, 7], x[3] = 0.0, NAN, x[3] * 1e15
    y = ssm.block_norm(x.cuda(), norm="rms").cpu()
    s, e, _, _ = ref.block_norm(x)
    good = [0, 1, 3, 4]
    ref.check(y[good], s[good], ref.rounded(s, e, F32)[good])
    assert (y[1] == 0).all() and torch.isnan(y[2]).all()


# ----------------------------------------------------------------------------- slots, streams, graphs, sizes

def block(n_tokens, seed=0, dtype=BF16):
    """One state-space layer's parameters and the pieces of its input projection."""
    d, h, p, n, g, k = 96, 4, 32, 32, 1, 4
    r = gen(seed)
    return dict(h=h, p=p, n=n, g=g, d=d, w_in=r(2 * h * p + 2 * g * n + h, d, scale=d ** -0.5, dtype=dtype).cuda(),
                w_out=r(d, h * p, scale=(h * p) ** -0.5, dtype=dtype).cuda(), conv_w=r(h * p + 2 * g * n, k, scale=0.5).cuda(),
                conv_b=r(h * p + 2 * g * n).cuda(), A=-(r(h).abs() * 2 + 0.5).cuda(), D=r(h).cuda(), dt_bias=(r(h) - 3).cuda(), w0=(r(d) + 1).cuda(),
                w1=(r(h * p) + 1).cuda(), tokens=r(n_tokens, d, scale=2.0).cuda(), k=k)


def run_block(q, res, conv_state, state, slots, cu=None, has=None):
    """Norm, projection, convolution, scan, gated norm, projection, residual sum: prompts with cu, single tokens without."""
    from mockingbird_amd import ssm
    h, p, n, g = q["h"], q["p"], q["n"], q["g"]
    u = ssm.block_norm(res.to(q["w_in"].dtype), q["w0"])
    proj = u @ q["w_in"].t()
    z, xbc, dt = proj.split([h * p, h * p + 2 * g * n, h], -1)
    if cu is None:
        xbc = ssm.causal_conv1d_step(xbc, conv_state, q["conv_w"], q["conv_b"], "silu", slots=slots)
    else:
        xbc = ssm.causal_conv1d(xbc, q["conv_w"], q["conv_b"], "silu", cu_seqlens=cu, state=conv_state, slots=slots, has_state=has)
    x, bm, cm = xbc.split([h * p, g * n, g * n], -1)
    x, bm, cm = x.unflatten(-1, (h, p)), bm.unflatten(-1, (g, n)), cm.unflatten(-1, (g, n))
    if cu is None:
        y = ssm.selective_scan_step(x, dt, q["A"], bm, cm, state, q["D"], dt_bias=q["dt_bias"], dt_softplus=True, slots=slots)
    else:
        y = ssm.selective_scan(x, dt, q["A"], bm, cm, q["D"], dt_bias=q["dt_bias"], dt_softplus=True, cu_seqlens=cu, state=state, slots=slots,
                               has_state=has)
    o = ssm.block_norm(y.flatten(-2), q["w1"], gate=z, groups=4) @ q["w_out"].t()
    return ssm.block_norm(o, norm=None, residual=res, scale=0.5, next_norm="rms", next_weight=q["w0"])


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_block_over_prompts_chunks_and_tokens(dtype):
    """Two requests: whole prompts at once, in two chunks, and a prompt followed by single tokens give the same rows and states."""
    q = block(0, 1, dtype)
    la, lb = 90, 41
    r = gen(9)
    ta, tb = r(la, q["d"], scale=2.0).cuda(), r(lb, q["d"], scale=2.0).cuda()
    c = q["h"] * q["p"] + 2 * q["g"] * q["n"]

    def pools():
        return torch.full((5, q["k"] - 1, c), NAN, dtype=dtype, device="cuda"), torch.full((5, q["h"], q["p"], q["n"]), NAN, device="cuda")

    conv, st = pools()
    slots = i32(3, 1)
    none, some = torch.zeros(2, dtype=torch.bool, device="cuda"), torch.ones(2, dtype=torch.bool, device="cuda")
    whole, _ = run_block(q, torch.cat([ta, tb]), conv, st, slots, i32(0, la, la + lb), none)
    conv2, st2 = pools()
    one, _ = run_block(q, torch.cat([ta[:70], tb[:1]]), conv2, st2, slots, i32(0, 70, 71), none)
    two, _ = run_block(q, torch.cat([ta[70:], tb[1:]]), conv2, st2, slots, i32(0, la - 70, la - 70 + lb - 1), some)
    conv3, st3 = pools()
    rows = [run_block(q, torch.cat([ta[:88], tb[:39]]), conv3, st3, slots, i32(0, 88, 127), none)[0]]
    for i in range(2):
        rows.append(run_block(q, torch.stack([ta[88 + i], tb[39 + i]]), conv3, st3, slots)[0])
    # between two ways through the block lie other groupings of the same sums; in bf16 those move roundings of its intermediate
    # results (four of them behind each other, each half a step of values up to 8 here), in fp32 sums of up to 2 * 90 terms
    tol = 2.0 ** -24 * 256 if dtype is F32 else 4 * 2.0 ** -8
    size = whole.abs().max().item()
    for got, want in [(torch.cat([one[:70], two[:la - 70]]), whole[:la]), (torch.cat([one[70:], two[la - 70:]]), whole[la:]),
                      (rows[0][:88], whole[:88]), (torch.stack([rows[1][0], rows[2][0]]), whole[88:la]),
                      (torch.stack([rows[1][1], rows[2][1]]), whole[la + 39:])]:
        assert (got - want).abs().max().item() <= tol * size
    for s in (st2, st3):
        assert (s[[3, 1]] - st[[3, 1]]).abs().max().item() <= tol * st[[3, 1]].abs().max().item() * 4
    for cv, s in ((conv2, st2), (conv3, st3)):
        assert torch.isnan(s[[0, 2, 4]]).all() and torch.isnan(cv[[0, 2, 4]]).all()


@pytest.mark.parametrize("step", [False, True])
def test_slots_outside_the_pool_and_named_twice(step):
    """A slot outside the pool leaves its request out; of two requests with one slot the first counts."""
    from mockingbird_amd import ssm
    h, p, n, c = 2, 16, 16, 40
    r = gen(2)
    b = 5
    slots = [4, -1, 2, 4, 9]
    ok = [4, None, 2, None, None]
    lead = (b,) if step else (b, 3)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, 1, BF16)
    cx, w = r(*lead, c, dtype=BF16), r(c, 4)
    pool, cpool = r(6, h, p, n), r(6, 3, c, dtype=BF16)
    dp, dc = pool.cuda(), cpool.cuda()
    out, cout = torch.full(x.shape, 7.0, dtype=BF16, device="cuda"), torch.full(cx.shape, 7.0, dtype=BF16, device="cuda")
    if step:
        ssm.causal_conv1d_step(cx.cuda(), dc, w.cuda(), slots=i32(*slots), out=cout)
        ssm.selective_scan_step(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), dp, dt_softplus=True, slots=i32(*slots), out=out)
    else:
        ssm.causal_conv1d(cx.cuda(), w.cuda(), state=dc, slots=i32(*slots), out=cout)
        ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), dt_softplus=True, state=dp, slots=i32(*slots), out=out)
    seqs = [(i, 1) for i in range(b)] if step else ref.sequences([3] * b, False, 3)
    want, err, new, nerr = ref.scan(flat(x, 2), flat(dt, 1), a, flat(bm, 2), flat(cm, 2), None, None, True, None, seqs, pool, ok, [True] * b,
                                    PLANES[BF16])
    live = ~torch.isnan(want)[:, 0, 0]
    got = out.reshape(-1, h, p).cpu()
    ref.check(got[live], want[live], ref.rounded(want, err, BF16)[live])
    assert (got[~live] == 7.0).all()
    ref.check(dp, new, nerr + 2 * ref.HALF[F32] * new.abs())
    want, err, new = ref.conv(flat(cx, 1), w, None, None, seqs, cpool, ok, [True] * b)
    got = cout.reshape(-1, c).cpu()
    ref.check(got[live], want[live], ref.rounded(want, err, BF16)[live])
    assert (got[~live] == 7.0).all() and torch.equal(dc.cpu().double(), new)


def test_empty_calls_and_empty_items_keep_the_states():
    from mockingbird_amd import ssm
    x = torch.zeros(0, 2, 16, dtype=BF16, device="cuda")
    bm = torch.zeros(0, 1, 8, dtype=BF16, device="cuda")
    a = -torch.ones(2, device="cuda")
    pool = torch.randn(3, 2, 16, 8, device="cuda")
    was = pool.clone()
    cx, w = torch.zeros(0, 24, device="cuda"), torch.ones(24, 4, device="cuda")
    cpool = torch.randn(3, 3, 24, device="cuda")
    cwas = cpool.clone()
    has = torch.tensor([True, False], device="cuda")
    for cu in (i32(0), i32(0, 0, 0)):
        sl = dict(slots=i32(*range(1, cu.numel())), has_state=has[:cu.numel() - 1], cu_seqlens=cu)
        assert ssm.selective_scan(x, x[..., 0], a, bm, bm, state=pool, **sl).shape == x.shape
        assert ssm.causal_conv1d(cx, w, state=cpool, **sl).shape == cx.shape
        if cu.numel() == 3:
            was[2], cwas[2] = 0.0, 0.0  # starts from zeros and has no rows
        assert torch.equal(pool, was) and torch.equal(cpool, cwas)
    assert ssm.block_norm(torch.zeros(0, 24, device="cuda")).shape == (0, 24)
    assert ssm.causal_conv1d_step(cx, cpool, w).shape == cx.shape
    assert ssm.selective_scan_step(x, x[..., 0], a, bm, bm, pool).shape == x.shape
    torch.cuda.synchronize()
    assert torch.equal(pool, was) and torch.equal(cpool, cwas)


def test_row_numbers_outside_the_tensors_are_clamped():
    """cu_seqlens and lengths that lead outside the rows stay inside them."""
    from mockingbird_amd import ssm
    x = torch.randn(10, 16, device="cuda")
    w = torch.ones(16, 2, device="cuda")
    whole = ssm.causal_conv1d(x, w, cu_seqlens=i32(0, 10))
    assert torch.equal(ssm.causal_conv1d(x, w, cu_seqlens=i32(-5, 1000)), whole)
    assert torch.equal(ssm.causal_conv1d(x[None], w, lengths=i32(99))[0], whole)
    sx, bm = torch.randn(10, 2, 16, device="cuda"), torch.randn(10, 1, 16, device="cuda")
    args = (sx, sx[..., 0].contiguous(), -torch.ones(2, device="cuda"), bm, bm)
    whole = ssm.selective_scan(*args, dt_softplus=True, cu_seqlens=i32(0, 10))
    assert torch.equal(ssm.selective_scan(*args, dt_softplus=True, cu_seqlens=i32(-5, 1000)), whole)


def test_other_streams_and_graph_replays():
    """A step and a prompt captured into one graph, replayed with eager work of the program between the replays."""
    q = block(64, 4)
    c = q["h"] * q["p"] + 2 * q["g"] * q["n"]
    conv0, st0 = torch.randn(4, 3, c, device="cuda").to(BF16), torch.randn(4, q["h"], q["p"], q["n"], device="cuda")
    tok, prompt = q["tokens"][:2].clone(), q["tokens"][:40].clone()
    slots, cu = i32(2, 0), i32(0, 33, 40)
    has = torch.tensor([True, False], device="cuda")
    conv, st = conv0.clone(), st0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_block(q, prompt, conv, st, slots, cu, has)
        run_block(q, tok, conv, st, slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = run_block(q, prompt, conv, st, slots, cu, has)
        b = run_block(q, tok, conv, st, slots)
    for i in range(3):
        r = gen(20 + i)
        tok.copy_(r(2, q["d"], scale=2.0))
        prompt.copy_(r(40, q["d"], scale=2.0))
        conv.copy_(conv0)
        st.copy_(st0)
        ec, es = conv0.clone(), st0.clone()
        ea, eb = run_block(q, prompt, ec, es, slots, cu, has), run_block(q, tok, ec, es, slots)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((*a, *b, conv, st), (*ea, *eb, ec, es)):
            assert torch.equal(got, want), i


def test_results_do_not_depend_on_the_run():
    from mockingbird_amd import ssm
    r = gen(6)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, (700,), 4, 64, 64, 1, BF16)
    args = [v.cuda() for v in (x, dt, a, bm, cm, skip)]
    outs = [ssm.selective_scan(*args, dt_bias=bias.cuda(), dt_softplus=True, cu_seqlens=i32(0, 500, 700)) for _ in range(4)]
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_offsets_beyond_32_bits():
    """Row strides that put rows more than 2^31 elements apart."""
    from mockingbird_amd import ssm
    wide = 1 << 28
    buf = torch.empty(11 * wide, dtype=BF16, device="cuda")
    rows = buf.view(11, wide)
    x = torch.randn(11, 160, generator=torch.Generator().manual_seed(2)).to(BF16)
    rows[:, :160] = x.cuda()
    far = rows[:, :160]
    w = torch.randn(160, 4, device="cuda")
    assert torch.equal(ssm.causal_conv1d(far, w, cu_seqlens=i32(0, 11)), ssm.causal_conv1d(x.cuda(), w, cu_seqlens=i32(0, 11)))
    assert torch.equal(ssm.block_norm(far), ssm.block_norm(x.cuda()))
    a = -torch.ones(2, device="cuda")

    def scan(v):
        s = v[:, :64].unflatten(-1, (2, 32)), v[:, 150:152], a, v[:, 64:96].unflatten(-1, (1, 32)), v[:, 96:128].unflatten(-1, (1, 32))
        y = ssm.selective_scan(*s, dt_softplus=True, cu_seqlens=i32(0, 11))
        pool = torch.zeros(11, 2, 32, 32, device="cuda")
        return y, ssm.selective_scan_step(*s, pool, dt_softplus=True)

    for got, want in zip(scan(far), scan(x.cuda())):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 64, 64, 1), (4, 128, 128, 2), (2, 64, 256, 1), (6, 64, 128, 1)])
def test_selective_scan_of_whole_tiles(dtype, shape):
    """Head sizes without partial tiles (buffer accesses), over several chunks, split along time, in packed slices and padded batches."""
    from mockingbird_amd import ssm
    h, p, n, g = shape
    for packed, lens in [(True, [700, 0, 1, 333]), (False, [500, 64, 301])]:
        r = gen(h * n + packed)
        args, lead, t = meta(lens, packed)
        x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
        a = a * 0.2
        seqs = ref.sequences(lens, packed, t)
        pool, slots, has = pool_of(len(lens), (h, p, n), seqs, r, F32)
        dpool = pool.cuda()
        row = torch.cat([x.flatten(-2), bm.flatten(-2), cm.flatten(-2)], -1).cuda()  # one projection's output
        d = h * p
        out = torch.full(x.shape, 7.0, dtype=dtype, device="cuda")
        y = ssm.selective_scan(row[..., :d].unflatten(-1, (h, p)), dt.cuda(), a.cuda(), row[..., d:d + g * n].unflatten(-1, (g, n)),
                               row[..., d + g * n:].unflatten(-1, (g, n)), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, state=dpool, out=out,
                               **args, **slot_args(slots, has))
        want, err, new, nerr = ref.scan(flat(x, 2), flat(dt, 1), a, flat(bm, 2), flat(cm, 2), skip, bias, True, None, seqs, pool, slots, has,
                                        PLANES[dtype])
        got = y.reshape(-1, h, p).cpu()
        rows = torch.isnan(want)[:, 0, 0]
        assert (got[rows] == 7.0).all(), "rows of no item were written"
        ref.check(got[~rows], want[~rows], ref.rounded(want, err, dtype)[~rows], (lens, "y"))
        ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs() + ref.TINY[F32], (lens, "state"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [NAN, float("-inf")])
def test_selective_scan_of_whole_tiles_stays_causal(dtype, value):
    """The same around a NaN or infinity in one column of one head: nothing before it, no other column and no other head changes."""
    from mockingbird_amd import ssm
    h, p, n, t = 2, 64, 64, 150
    r = gen(8)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, (t,), h, p, n, 1, dtype)
    clean = x.clone()
    for row, head, col in [(37, 0, 5), (100, 1, 60)]:
        x[row, head, col] = value
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, cu_seqlens=i32(0, t)).cpu()
    want, err, _, _ = ref.scan(clean, dt, a, bm, cm, skip, bias, True, None, [(0, t)], planes=PLANES[dtype])
    bound = ref.rounded(want, err, dtype)
    hit = torch.zeros(t, h, p, dtype=torch.bool)
    hit[37:, 0, 5] = True
    hit[100:, 1, 60] = True
    assert not torch.isfinite(y[hit]).any()
    ref.check(y[~hit], want[~hit], bound[~hit])


def test_a_split_prompt_in_a_graph():
    """The two passes of a long prompt captured, replayed on new inputs between eager calls, in two graphs with pools of their own."""
    from mockingbird_amd import ssm
    h, p, n, t = 2, 64, 64, 900
    x, dt, a, bm, cm, skip, bias = [v.cuda() for v in scan_inputs(gen(1), (t,), h, p, n, 1, BF16)]
    cu, pool0 = i32(0, 600, t), torch.randn(2, h, p, n, device="cuda")

    def call(pool):
        return ssm.selective_scan(x, dt, a, bm, cm, skip, dt_bias=bias, dt_softplus=True, cu_seqlens=cu, state=pool)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(pool0.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        pool = pool0.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call(pool)
        graphs.append((g, pool, y))
    for i in range(3):
        x.copy_(gen(30 + i)(t, h, p, dtype=BF16))
        want_pool = pool0.clone()
        want = call(want_pool)
        for g, pool, y in graphs:
            pool.copy_(pool0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(pool, want_pool)


def test_row_numbers_that_overlap_touch_nothing_else():
    """Items that claim the same rows (which is not allowed) still write only rows and slots of their own tensors."""
    from mockingbird_amd import ssm
    h, p, n, t = 2, 32, 16, 700
    x, dt, a, bm, cm, skip, bias = [v.cuda() for v in scan_inputs(gen(2), (t,), h, p, n, 1, F32)]
    cu = i32(*([0, t] * 6), 0)
    wide = torch.full((t + 64, h, p), 7.0, device="cuda")
    pools = torch.full((14, h, p, n), 3.0, device="cuda")
    ssm.selective_scan(x, dt, a, bm, cm, skip, dt_bias=bias, dt_softplus=True, cu_seqlens=cu, state=pools[1:13], out=wide[:t])
    cx = torch.full((t + 64, 48), 7.0, device="cuda")
    ssm.causal_conv1d(torch.zeros(t, 48, device="cuda"), torch.zeros(48, 4, device="cuda"), cu_seqlens=cu, out=cx[:t])
    torch.cuda.synchronize()
    assert (wide[t:] == 7.0).all() and (cx[t:] == 7.0).all() and (pools[[0, 13]] == 3.0).all()


def test_many_items():
    """More items than a wave sums up at once, most of them short, some empty."""
    from mockingbird_amd import ssm
    lens = [(7 * i) % 11 for i in range(150)] + [300] + [i % 3 for i in range(60)]
    args, lead, t = meta(lens, True)
    h, p, n = 2, 16, 16
    r = gen(3)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, 1, BF16)
    pool, slots, has = pool_of(len(lens), (h, p, n), lens, r, F32)
    dpool = pool.cuda()
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, state=dpool,
                           **args, **slot_args(slots, has))
    seqs = ref.sequences(lens, True, t)
    want, err, new, nerr = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, seqs, pool, slots, has, PLANES[BF16])
    ref.check(y, want, ref.rounded(want, err, BF16))
    ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs() + ref.TINY[F32])
    cx, w = r(*lead, 40, dtype=BF16), r(40, 4)
    cpool, slots, has = pool_of(len(lens), (3, 40), lens, r, BF16)
    dc = cpool.cuda()
    y = ssm.causal_conv1d(cx.cuda(), w.cuda(), state=dc, **args, **slot_args(slots, has))
    want, err, new = ref.conv(cx, w, None, None, seqs, cpool, slots, has)
    ref.check(y, want, ref.rounded(want, err, BF16))
    assert torch.equal(dc.cpu()[slots].double(), new[slots])


def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives what it gives alone."""
    from mockingbird_amd import ssm
    h, p, n, t = 2, 64, 64, 1200
    ins = [[v.cuda() for v in scan_inputs(gen(40 + i), (t,), h, p, n, 1, BF16)] for i in range(2)]
    cu = i32(0, t)

    def call(v):
        x, dt, a, bm, cm, skip, bias = v
        return ssm.selective_scan(x, dt, a, bm, cm, skip, dt_bias=bias, dt_softplus=True, cu_seqlens=cu)

    alone = [call(v) for v in ins]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(ins[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, alone[i]) for y in got[i])


# ---------------------------------------------------------------------------------------------- refusals

def refusals():
    x = torch.zeros(4, 16)
    s, b3 = torch.zeros(4, 2, 8), torch.zeros(4, 1, 8)
    a, dt = torch.zeros(2), torch.zeros(4, 2)
    w, cu = torch.zeros(16, 4), torch.tensor([0, 4], dtype=torch.int32)
    conv = lambda **k: ("causal_conv1d", (k.pop("x", x), k.pop("w", w)), k)  # noqa: E731
    scan = lambda **k: ("selective_scan", (k.pop("x", s), k.pop("dt", dt), k.pop("A", a), k.pop("B", b3), k.pop("C", b3)), k)  # noqa: E731
    norm = lambda **k: ("block_norm", (k.pop("x", x),), k)  # noqa: E731
    return [
        (conv(), "cu_seqlens"), (conv(x=x[None], cu_seqlens=cu), "cu_seqlens"), (conv(cu_seqlens=cu.long()), "int32"),
        (conv(cu_seqlens=cu, w=torch.zeros(16, 9)), "taps"), (conv(cu_seqlens=cu, w=torch.zeros(15, 4)), "weight"),
        (conv(cu_seqlens=cu, w=w.half()), "float32"), (conv(cu_seqlens=cu, activation="relu"), "silu"),
        (conv(cu_seqlens=cu, slots=cu[:1]), "pool"), (conv(cu_seqlens=cu, state=torch.zeros(2, 4, 16)), "state"),
        (conv(cu_seqlens=cu, state=torch.zeros(2, 3, 16).half()), "state"), (conv(cu_seqlens=cu, out=x), "overlap"),
        (conv(cu_seqlens=cu, out=x[:1].expand(4, 16)), "overlap"), (conv(cu_seqlens=cu, x=x.t().contiguous().t()), "dense"),
        (conv(cu_seqlens=cu, x=x.double()), "float32"), (conv(cu_seqlens=cu, bias=torch.zeros(15)), "bias"),
        (conv(x=x[None], lengths=cu), "lengths"), (conv(x=x[None].expand(3, 4, 16), state=torch.zeros(2, 3, 16)), "requests"),
        (conv(cu_seqlens=cu, x=x.clone().requires_grad_()), "backward"),
        (scan(), "cu_seqlens"), (scan(cu_seqlens=cu, B=torch.zeros(4, 3, 8), C=torch.zeros(4, 3, 8)), "groups"),
        (scan(cu_seqlens=cu, x=torch.zeros(4, 2, 129)), "head_dim"), (scan(cu_seqlens=cu, B=torch.zeros(4, 1, 257)), "d_state"),
        (scan(cu_seqlens=cu, C=torch.zeros(4, 1, 9)), "C has shape"), (scan(cu_seqlens=cu, dt=torch.zeros(4, 3)), "dt has shape"),
        (scan(cu_seqlens=cu, dt=dt.half()), "dt is"), (scan(cu_seqlens=cu, A=torch.zeros(3)), "A must"), (scan(cu_seqlens=cu, A=None), "A is required"),
        (scan(cu_seqlens=cu, dt_limit=(1.0, 0.0)), "dt_limit"), (scan(cu_seqlens=cu, state=torch.zeros(2, 2, 8, 9)), "state"),
        (scan(cu_seqlens=cu, out=s), "overlap"), (scan(cu_seqlens=cu, D=torch.zeros(2, 8)), "D must"),
        (scan(cu_seqlens=cu, x=torch.zeros(4, 8, 2).transpose(1, 2)), "dense"),
        (norm(norm="batch"), "norm"), (norm(groups=3), "groups"), (norm(norm=None), "nothing"), (norm(gate=x, gate_act="tanh"), "gate_act"),
        (norm(weight=torch.zeros(15)), "weight"), (norm(next_weight=torch.zeros(16)), "next_weight"), (norm(residual=x.half()), "residual"),
        (norm(residual=x.clone(), next_norm="rms", out=x, residual_out=x), "overlap"), (norm(out=x[:1].expand(4, 16)), "overlap"),
        (norm(norm=None, weight=torch.zeros(16), gate=x), "weight"), (norm(out=x.clone(), residual_out=x.clone()), "one result"),
        (norm(gate=torch.zeros(4, 17)), "gate has shape"), (norm(x=torch.zeros(4, 4, 16)[:, :2]), "evenly"),
    ]


@pytest.mark.parametrize("i", range(len(refusals())))
def test_refusals(i):
    from mockingbird_amd import _lib, ssm
    (name, args, kw), match = refusals()[i]
    up = {}

    def dev(t):  # one device tensor per storage, so that overlaps stay overlaps
        if not torch.is_tensor(t):
            return t
        base = up.setdefault(t.untyped_storage().data_ptr(), torch.empty(0, dtype=torch.uint8, device="cuda").set_(
            t.detach().untyped_storage().cuda()) if t.numel() else t.detach().cuda())
        v = torch.empty(0, dtype=t.dtype, device="cuda").set_(base.untyped_storage(), t.storage_offset(), t.shape, t.stride())
        return v.requires_grad_(t.requires_grad)

    with pytest.raises(_lib.MbHipError, match=match):
        getattr(ssm, name)(*[dev(t) for t in args], **{k: dev(v) for k, v in kw.items()})
    torch.cuda.synchronize()


def test_refusals_of_steps_and_devices():
    from mockingbird_amd import _lib, ssm
    x, w = torch.zeros(3, 16, device="cuda"), torch.zeros(16, 4, device="cuda")
    with pytest.raises(_lib.MbHipError, match="state pool"):
        ssm.causal_conv1d_step(x, None, w)
    with pytest.raises(_lib.MbHipError, match="requests"):
        ssm.causal_conv1d_step(x, torch.zeros(2, 3, 16, device="cuda"), w)
    with pytest.raises(_lib.MbHipError, match="weight is on"):
        ssm.causal_conv1d(x, w.cpu(), cu_seqlens=i32(0, 3))
    with pytest.raises(_lib.MbHipError, match="no CPU path"):
        ssm.block_norm(x.cpu())
    with pytest.raises(_lib.MbHipError, match="weight is required"):
        ssm.causal_conv1d(x, None, cu_seqlens=i32(0, 3))
    s = torch.zeros(3, 2, 8, device="cuda")
    with pytest.raises(_lib.MbHipError, match="B is required"):
        ssm.selective_scan(s, s[..., 0].contiguous(), torch.zeros(2, device="cuda"), None, None, cu_seqlens=i32(0, 3))
    with pytest.raises(_lib.MbHipError, match="dt has shape"):
        ssm.selective_scan(s, torch.zeros((), device="cuda"), torch.zeros(2, device="cuda"), s[:, :1], s[:, :1], cu_seqlens=i32(0, 3))
    with pytest.raises(_lib.MbHipError, match="must be a tensor"):
        ssm.causal_conv1d(x, [1.0], cu_seqlens=i32(0, 3))
    p = torch.zeros(16, device="cuda", requires_grad=True)
    with pytest.raises(_lib.MbHipError, match="backward"):
        ssm.block_norm(x, p)
    with torch.no_grad():
        assert ssm.block_norm(x, p).shape == x.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_selective_scan_repeats_to_the_bit_in_any_order(dtype):
    """Calls of many shapes behind each other in changing orders, on fresh copies of their inputs: what a call gives does not depend on what
    the chip did before it."""
    import random
    from mockingbird_amd import ssm
    rng, r = random.Random(11), gen(11)
    calls = []
    for _ in range(200):
        h, p, n = rng.randint(1, 24), rng.choice([32, 40, 64, 96, 128]), rng.choice([24, 64, 64, 128])
        lens = [rng.randint(1, 130) for _ in range(rng.randint(1, 5))]
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
        x, dt, a, bm, cm, skip, bias = (t.cuda() for t in scan_inputs(r, (sum(lens),), h, p, n, 1, dtype))
        calls.append(((x, dt, a, bm, cm, skip), dict(dt_bias=bias, dt_softplus=True, cu_seqlens=cu)))
    want = [None] * len(calls)
    for turn in range(8):
        order = list(range(len(calls)))
        rng.shuffle(order)
        for i in order:
            args, kw = calls[i]
            got = ssm.selective_scan(*[t.clone() for t in args], **kw)
            if want[i] is None:
                want[i] = got
            assert torch.equal(got, want[i]), (turn, i, list(args[0].shape), list(args[3].shape))
