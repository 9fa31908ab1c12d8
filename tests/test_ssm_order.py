"""selective_scan behind other work: what a call gives on a busy chip is right, not only the same every time."""
import random

import pytest
import torch

import ssm_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _library(cuda, lib):
    pass


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_calls_among_others_are_right(dtype):
    """Small calls of several chunks, among calls of other shapes in changing orders, against float64."""
    from test_ssm_gpu import PLANES, gen, scan_inputs
    from mockingbird_amd import ssm
    rng, r = random.Random(17), gen(17)
    calls, wants = [], []
    for i in range(60):
        h, p, n = rng.randint(1, 6), rng.choice([32, 40, 64, 96, 128]), rng.choice([24, 64, 128])
        lens = [rng.randint(1, 130) for _ in range(rng.randint(1, 3))]
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
        x, dt, a, bm, cm, skip, bias = scan_inputs(r, (sum(lens),), h, p, n, 1, dtype)
        calls.append(([v.cuda() for v in (x, dt, a, bm, cm, skip)], dict(dt_bias=bias.cuda(), dt_softplus=True, cu_seqlens=cu.cuda())))
        if i < 12:
            want, err, _, _ = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, ref.sequences(lens, True, None), planes=PLANES[dtype])
            wants.append((want, ref.rounded(want, err, dtype)))
    for turn in range(30):
        order = list(range(len(calls)))
        rng.shuffle(order)
        got = {i: ssm.selective_scan(*[t.clone() for t in calls[i][0]], **calls[i][1]) for i in order}
        for i, (want, bound) in enumerate(wants):
            ref.check(got[i], want, bound, (turn, i))
