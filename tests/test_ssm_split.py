"""Selective scans that are split along time: what they reserve, and what they compute where split and unsplit requests share a call."""
import pytest
import torch


def workspace(lib, batch, t, packed=True, heads=64, head_dim=64, d_state=128, groups=1, dtype=None):
    from mockingbird_amd import _lib
    a = _lib.SelectiveScanArgs(d_x=256, d_y=256, d_dt=256, d_b=256, d_c=256, d_a=256, dtype=_lib.MB_BF16 if dtype is None else dtype, dt_dtype=_lib.MB_F32,
                               batch=batch, t=t, heads=heads, head_dim=head_dim, groups=groups, d_state_dim=d_state, dt_min=0.0, dt_max=1.0,
                               d_cu_seqlens=256 if packed else None)
    return lib.mb_selective_scan_workspace_bytes(a)


@pytest.mark.parametrize("heads,head_dim,d_state,groups", [(64, 64, 128, 1), (24, 64, 64, 1), (32, 128, 256, 8), (8, 16, 16, 2), (3, 50, 200, 3)])
@pytest.mark.parametrize("t", [400, 1000, 16384, 100000])
def test_the_workspace_goes_by_the_rows_and_not_by_the_requests(lib, heads, head_dim, d_state, groups, t):
    """Only requests longer than a tile need one, and together they have at most the call's rows."""
    one = workspace(lib, 1, t, True, heads, head_dim, d_state, groups)
    for batch in (2, 16, 256, 1024, 4096):
        assert workspace(lib, batch, t, True, heads, head_dim, d_state, groups) <= 2 * one
    state = heads * (head_dim * d_state + 1) * 4
    assert one <= (t // 64 + 1) * state + 512


F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(8, 16, 16, 8), (16, 64, 64, 8)])
@pytest.mark.parametrize("order", [0, 1])
def test_long_and_short_requests_in_one_call(cuda, lib, dtype, shape, order):
    """Enough requests to fill the chip: only those beyond twice the mean length are split, the others walk from and to their states."""
    import ssm_reference as ref
    from test_ssm_gpu import PLANES, gen, meta, pool_of, scan_inputs, slot_args
    from mockingbird_amd import ssm
    h, p, n, g = shape
    lens = [0, 5, 700, 1] + [(7 * i) % 23 for i in range(30)] + [333, 2, 64]
    lens = lens[::-1] if order else lens
    r = gen(h + order)
    args, lead, t = meta(lens, True)
    seqs = ref.sequences(lens, True, t)
    # (the rule: requests x workgroups of a request fill 256 CUs, and the call is longer than five chunks)
    assert workspace(lib, len(lens), lead[0], True, h, p, n, g) > 0 and len(lens) * g >= 256
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, lead, h, p, n, g, dtype)
    a = a * 0.1
    pool, slots, has = pool_of(len(lens), (h, p, n), seqs, r, F32)
    dpool = pool.cuda()
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, state=dpool,
                           **args, **slot_args(slots, has))
    want, err, new, nerr = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, seqs, pool, slots, has, PLANES[dtype])
    ref.check(y, want, ref.rounded(want, err, dtype), "y")
    ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs() + ref.TINY[F32], "state")
    rest = [i for i in range(pool.shape[0]) if i not in slots]
    assert torch.equal(dpool.cpu()[rest], pool[rest])
    # the same call without a pool
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, **args)
    want, err, _, _ = ref.scan(x, dt, a, bm, cm, skip, bias, True, None, seqs, planes=PLANES[dtype])
    ref.check(y, want, ref.rounded(want, err, dtype), "y without states")


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_row_numbers_in_no_order_stay_inside(cuda, lib, seed):
    """Lists of row numbers that overlap, run backwards and lead outside (none of which is allowed) write only rows and slots of their tensors."""
    from test_ssm_gpu import gen, scan_inputs
    from mockingbird_amd import ssm
    h, p, n, t, b = 8, 16, 16, 700, 40
    r = gen(seed)
    x, dt, a, bm, cm, skip, bias = [v.cuda() for v in scan_inputs(r, (t,), h, p, n, 8, F32)]
    cu = torch.randint(-50, t + 50, (b + 1,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
    wide = torch.full((t + 128, h, p), 7.0, device="cuda")
    pools = torch.full((b + 2, h, p, n), 3.0, device="cuda")
    ssm.selective_scan(x, dt, a, bm, cm, skip, dt_bias=bias, dt_softplus=True, cu_seqlens=cu, state=pools[1:b + 1], out=wide[64:t + 64])
    torch.cuda.synchronize()
    assert (wide[:64] == 7.0).all() and (wide[t + 64:] == 7.0).all() and (pools[[0, b + 1]] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,batch,t", [((2, 64, 64, 1), 3, 700), ((3, 20, 24, 3), 2, 641), ((2, 64, 64, 1), 1, 321)])
def test_padded_requests_of_one_length(cuda, lib, dtype, shape, batch, t):
    """[batch, t, ...] without lengths, split along time, with and without states to start from."""
    import ssm_reference as ref
    from test_ssm_gpu import PLANES, flat, gen, pool_of, scan_inputs, slot_args
    from mockingbird_amd import ssm
    h, p, n, g = shape
    assert workspace(lib, batch, t, False, h, p, n, g, {F32: 0, F16: 1, BF16: 3}[dtype]) > 0
    r = gen(t)
    x, dt, a, bm, cm, skip, bias = scan_inputs(r, (batch, t), h, p, n, g, dtype)
    a = a * 0.1
    seqs = ref.sequences([t] * batch, False, t)
    pool, slots, has = pool_of(batch, (h, p, n), seqs, r, F32)
    dpool = pool.cuda()
    y = ssm.selective_scan(x.cuda(), dt.cuda(), a.cuda(), bm.cuda(), cm.cuda(), skip.cuda(), dt_bias=bias.cuda(), dt_softplus=True, state=dpool,
                           **slot_args(slots, has))
    want, err, new, nerr = ref.scan(flat(x, 2), flat(dt, 1), a, flat(bm, 2), flat(cm, 2), skip, bias, True, None, seqs, pool, slots, has, PLANES[dtype])
    ref.check(flat(y, 2), want, ref.rounded(want, err, dtype), "y")
    ref.check(dpool.cpu()[slots], new[slots], nerr[slots] + ref.HALF[F32] * new[slots].abs() + ref.TINY[F32], "state")
