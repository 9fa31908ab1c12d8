"""selective_scan around infinities, NaN and step sizes whose products leave fp32: every value is the one of the row-by-row recurrence,
an infinity with its sign as well as a NaN."""
import pytest
import torch

import ssm_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _library(cuda, lib):
    pass


def same_values(got, want, bound, what):
    got = got.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN in different places", torch.nonzero(torch.isnan(got) != torch.isnan(want))[:4].tolist())
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), (what, "infinities differ")
    ref.check(got, want, bound, what)


def case(seed, shape, lens, dtype, positive):
    """Inputs, on the host; positive: B and C have one sign, so that an infinite state gives infinite answers and not NaN."""
    from test_ssm_gpu import gen, meta, pool_of, scan_inputs
    r = gen(seed)
    args, lead, t = meta(lens, True)
    h, p, n, g = shape
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
    if positive:
        bm, cm = bm.abs() + 0.125, cm.abs() + 0.125
    pool, slots, has = pool_of(len(lens), (h, p, n), lens, r, F32)
    return dict(x=x, dt=dt, a=a * 0.1, bm=bm, cm=cm, skip=skip, bias=bias, pool=pool, slots=slots, has=has, args=args, seqs=ref.sequences(lens, True, t))


def run_and_check(c, dtype, what, softplus=True):
    from test_ssm_gpu import PLANES, slot_args
    from mockingbird_amd import ssm
    dpool = c["pool"].cuda()
    bias = None if c["bias"] is None else c["bias"].cuda()
    y = ssm.selective_scan(c["x"].cuda(), c["dt"].cuda(), c["a"].cuda(), c["bm"].cuda(), c["cm"].cuda(), c["skip"].cuda(), dt_bias=bias, dt_softplus=softplus,
                           state=dpool, **c["args"], **slot_args(c["slots"], c["has"]))
    want, err, new, nerr = ref.scan(c["x"], c["dt"], c["a"], c["bm"], c["cm"], c["skip"], c["bias"], softplus, None, c["seqs"], c["pool"], c["slots"], c["has"],
                                    PLANES[dtype])
    fine, keep = torch.isfinite(want), torch.isfinite(new)
    err, nerr = torch.where(fine, err, torch.zeros_like(err)), torch.where(keep, nerr, torch.zeros_like(nerr))
    same_values(y, want, ref.rounded(want, err, dtype), (what, "y"))
    at = c["slots"]
    same_values(dpool[at], new[at], nerr[at] + ref.HALF[F32] * new[at].abs() + ref.TINY[F32], (what, "state"))


# one walk over several chunks; split along time, with whole tiles and without
RUNS = [((2, 64, 64, 1), [150, 40]), ((3, 20, 24, 1), [75, 30, 0, 9]), ((2, 64, 64, 1), [700, 90]), ((3, 20, 24, 3), [641])]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("what", ["x", "bm", "cm", "dt", "pool"])
@pytest.mark.parametrize("run", range(len(RUNS)))
@pytest.mark.parametrize("positive", [True, False])
def test_values_behind_an_infinity_or_nan(dtype, value, what, run, positive):
    shape, lens = RUNS[run]
    c = case(run + 10 * positive, shape, lens, dtype, positive)
    if what == "pool":
        c["pool"][c["slots"][0], 1, 5, 7] = value  # item 0 continues from its state
    else:
        t = c[what]
        for row, rest in ((lens[0] // 2 + 3, (0, 5, 7)), (lens[0] - 1, (-1, -1, -1))):
            t[(row,) + rest[:t.dim() - 1]] = value
    run_and_check(c, dtype, (what, value))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("run", range(len(RUNS)))
def test_growing_states(dtype, run):
    """A > 0 for one head: what 64 rows grow by together is beyond fp32, but the state is zero until the last rows of each request."""
    shape, lens = RUNS[run]
    c = case(30 + run, shape, lens, dtype, False)
    c["a"][0], c["bias"] = 2.0, None
    c["dt"] = c["dt"].abs().clamp(0.25, 2.0)
    c["has"] = [False] * len(lens)
    c["bm"][...] = 0.0
    r = torch.Generator().manual_seed(run)
    for at, n in c["seqs"]:
        last = min(n, 7)
        c["bm"][at + n - last:at + n] = torch.randn(last, *c["bm"].shape[1:], generator=r).to(dtype)
    run_and_check(c, dtype, "growth", softplus=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("run", range(len(RUNS)))
def test_states_that_vanish_at_once(dtype, run):
    """A of minus infinity, or so large that its products leave fp32: each row stands for itself, y = (d C.B + D) x."""
    from mockingbird_amd import ssm
    shape, lens = RUNS[run]
    c = case(50 + run, shape, lens, dtype, False)
    for a in (-INF, -3e38):
        c["a"][...] = a
        dt = c["dt"].float().abs() + 2.0
        y = ssm.selective_scan(c["x"].cuda(), dt.cuda(), c["a"].cuda(), c["bm"].cuda(), c["cm"].cuda(), c["skip"].cuda(), **c["args"])
        h = shape[0] // shape[3]
        cb = (c["bm"].double() * c["cm"].double()).sum(-1).repeat_interleave(h, 1)
        size = (c["bm"].double() * c["cm"].double()).abs().sum(-1).repeat_interleave(h, 1)
        x = c["x"].double()
        want = (dt.double() * cb + c["skip"].double())[..., None] * x
        # products and sums of d_state + 2 terms, operands in planes of 2^-15 relative or fp32
        err = (dt.double() * size + c["skip"].double().abs())[..., None] * x.abs() * ((shape[2] + 8) * ref.U + (2.0 ** -15 if dtype is BF16 else 2.0 ** -21))
        same_values(y, want, ref.rounded(want, err, dtype), a)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("what", ["x", "bm", "cm", "dt", "pool"])
@pytest.mark.parametrize("shape", [(2, 64, 64, 1), (3, 20, 24, 1), (1, 5, 3, 1), (2, 16, 130, 2)])
def test_single_tokens_with_an_infinity_or_nan(dtype, value, what, shape):
    from test_ssm_gpu import gen, scan_inputs
    from mockingbird_amd import ssm
    h, p, n, g = shape
    b = 4
    r = gen(n)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, (b,), h, p, n, g, dtype)
    bm, cm, pool = bm.abs() + 0.125, cm.abs() + 0.125, r(b, h, p, n)
    t = dict(x=x, bm=bm, cm=cm, dt=dt, pool=pool)[what]
    t[(1,) + (0,) * (t.dim() - 1)] = value
    t[(2,) + (-1,) * (t.dim() - 1)] = value
    dpool = pool.cuda()
    y = ssm.selective_scan_step(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), dpool, skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True)
    want, err, new, nerr = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, [(i, 1) for i in range(b)], pool, list(range(b)), [True] * b)
    err, nerr = torch.where(torch.isfinite(want), err, torch.zeros_like(err)), torch.where(torch.isfinite(new), nerr, torch.zeros_like(nerr))
    same_values(y, want, ref.rounded(want, err, dtype), (what, "y"))
    same_values(dpool, new, nerr + ref.HALF[F32] * new.abs() + ref.TINY[F32], (what, "state"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("run", [2, 3])
def test_an_infinity_meets_a_decay_of_zero(dtype, run):
    """0 * infinity in a row is NaN, whichever tile the row is in; decays that are zero only together leave the infinity."""
    shape, lens = RUNS[run]
    for gone in (None, lens[0] - 40, lens[0] // 2, 200):
        c = case(70 + run, shape, lens, dtype, True)
        c["a"], c["bias"] = c["a"] * 30 - 2.0, None
        c["dt"] = c["dt"].float().abs() * 0.5 + 0.5  # (16 rows decay by 2^-23 and more, a tile by less than fp32 has)
        c["x"][20, 0, 5] = INF
        if gone is not None:
            c["dt"][gone] = 1e5
        run_and_check(c, dtype, ("zero", gone), softplus=False)
