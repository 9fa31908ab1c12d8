"""Measured cases of the state-space block operators (mockingbird_amd.ssm): the short causal convolution, the
selective scan (both for prompts and for single tokens) and the norms / gate / residual around a block.

`own` selects the framework's calls; otherwise `run` computes the same in elementary torch operations in 32 bits.
`exact` states the operators again in 64 bits, in another form (the convolution as one gather over shifted rows, the
scan as its blocked quadratic form, the norms from centred sums).

Layouts: packed prompts [rows, ...] with the requests behind each other, padded batches [batch, t, ...] with lengths,
state pools [slots, ...] that calls update in place through slot numbers."""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # prefill of a serving step: twelve prompts of very different lengths packed behind each other, x|B|C of a wide layer
        dict(name="conv_prompts_bf16", op="conv", dtype="bf16", channels=4352, ksize=4, act=True, packed=True, pool=True,
             lengths="4096,1,733,2048,64,3001,17,1500,2,3000,890,1031"),
        # a padded batch of utterances in the framework's own type, an odd channel count, a 3-tap filter without activation
        dict(name="conv_batch_f32", op="conv", dtype="f32", channels=1290, ksize=3, act=False, packed=False, pool=False,
             lengths="400,377,0,391,212,1,399,105"),
        # one token for each of 48 running requests, half precision
        dict(name="conv_step_f16", op="conv_step", dtype="f16", channels=2304, ksize=4, act=True, batch=48),
        # one long prompt alone: the work has to be split along time
        dict(name="scan_long_bf16", op="scan", dtype="bf16", heads=64, head_dim=64, d_state=128, groups=1, packed=True,
             pool=True, lengths="8192"),
        # packed prompts of a middle layer, eight heads sharing one B / C
        dict(name="scan_prompts_f16", op="scan", dtype="f16", heads=32, head_dim=64, d_state=64, groups=4, packed=True,
             pool=True, lengths="900,3,1777,64,512,1,1203,333,65,127"),
        # a padded batch in fp32 with odd head sizes, no state kept
        dict(name="scan_batch_f32", op="scan", dtype="f32", heads=12, head_dim=48, d_state=40, groups=3, packed=False,
             pool=False, lengths="400,0,211,399,1,307"),
        # one token for each of 128 running requests: the states are read and written once
        dict(name="scan_step_bf16", op="scan_step", dtype="bf16", heads=64, head_dim=64, d_state=128, groups=1, batch=128),
        # one token of one request: latency
        dict(name="scan_step_one_f32", op="scan_step", dtype="f32", heads=24, head_dim=64, d_state=64, groups=1, batch=1),
        # the norm behind a scan: y * silu(z), then an RMS norm over each of 8 groups
        dict(name="norm_gated_bf16", op="norm", dtype="bf16", res="", rows=16384, channels=4096, norm="rms", groups=8,
             gate="silu", gate_first=True, scale="", next_norm=""),
        # between two blocks: norm behind the block, per-channel residual scale, an fp32 residual stream, norm of the next block
        dict(name="norm_sandwich_bf16", op="norm", dtype="bf16", res="f32", rows=8192, channels=2048, norm="rms", groups=1,
             gate="", gate_first=False, scale="vector", next_norm="rms"),
        # layer norms with an odd width and a sigmoid gate behind the norm
        dict(name="norm_layer_f16", op="norm", dtype="f16", res="f16", rows=777, channels=1001, norm="layer", groups=1,
             gate="sigmoid", gate_first=False, scale="scalar", next_norm="layer"),
        # one token between two blocks: latency
        dict(name="norm_one_f32", op="norm", dtype="f32", res="f32", rows=1, channels=1024, norm="", groups=1, gate="",
             gate_first=False, scale="", next_norm="rms"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, total, n):
    """n lengths that sum to about total, one of them possibly empty."""
    w = [rng.random() ** 2 + 1e-3 for _ in range(n)]
    out = [max(1, int(total * v / sum(w))) for v in w]
    if n > 2 and rng.random() < 0.3:
        out[rng.randrange(n)] = 0
    return ",".join(map(str, out))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan_step", "norm", "norm"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "conv":
        c = _log(rng, 96, 4352)
        n = _log(rng, 1, 24)
        total = _log(rng, 8, min(12000, 40000000 // c))
        packed = rng.random() < 0.6
        if not packed:
            total, n = total // 3 + 1, min(n, 8)
        return dict(op=op, dtype=dtype, channels=c, ksize=rng.choice([2, 3, 4, 4, 5]), act=rng.random() < 0.7, packed=packed,
                    pool=rng.random() < 0.7, lengths=_lengths(rng, total, n))
    if op == "conv_step":
        return dict(op=op, dtype=dtype, channels=_log(rng, 96, 4352), ksize=rng.choice([2, 3, 4, 4, 5]), act=rng.random() < 0.7,
                    batch=_log(rng, 1, 256))
    if op in ("scan", "scan_step"):
        p = rng.choice([16, 32, 40, 64, 64, 64, 96, 128])
        n = rng.choice([16, 24, 64, 64, 100, 128, 128, 256])
        g = rng.choice([1, 1, 2, 4])
        h = g * _log(rng, 1, max(1, min(64, 4096 // p) // g))
        if op == "scan_step":
            return dict(op=op, dtype=dtype, heads=h, head_dim=p, d_state=n, groups=g,
                        batch=_log(rng, 1, max(1, min(128, 60000000 // (h * p * n)))))
        b = _log(rng, 1, 12)
        total = _log(rng, 8, max(8, min(6000, 2000000000 // (h * p * n))))
        packed = rng.random() < 0.6
        if not packed:
            total, b = total // 3 + 1, min(b, 6)
        return dict(op=op, dtype=dtype, heads=h, head_dim=p, d_state=n, groups=g, packed=packed, pool=rng.random() < 0.7,
                    lengths=_lengths(rng, total, b))
    g = rng.choice([1, 1, 1, 4, 8])
    c = g * _log(rng, max(8, 96 // g), 6144 // g)
    rows = _log(rng, 1, min(12000, 24000000 // c))
    res = rng.choice(["", "same", "f32"])
    res = dtype if res == "same" else res
    norm = rng.choice(["rms", "rms", "layer", ""])
    gate = rng.choice(["", "silu", "sigmoid", "none"])
    nxt = rng.choice(["rms", "layer"]) if res else ""
    if not (norm or res):
        norm = "rms"
    return dict(op=op, dtype=dtype, res=res, rows=rows, channels=c, norm=norm, groups=g if norm else 1, gate=gate,
                gate_first=bool(gate) and rng.random() < 0.5, scale=rng.choice(["", "scalar", "vector"]) if res else "", next_norm=nxt)


# ------------------------------------------------------------------------------------------------ inputs

def _lens(case):
    return [int(v) for v in case["lengths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    def slots(b):  # live requests sit in any slot of a pool that is a little larger
        return torch.randperm(b + 3, generator=g, device="cuda")[:b].to(torch.int32)

    s = dict(case=case)
    op = case["op"]
    if op == "norm":
        r, c = case["rows"], case["channels"]
        s["x"] = normal(r, c, scale=1.5, dtype=dt)
        if case["norm"]:
            s["weight"] = normal(c, scale=0.1, shift=1.0)
            s["bias"] = normal(c, scale=0.1) if case["norm"] == "layer" else None
        if case["gate"]:  # the gate is a slice of the block's input projection
            s["gate"] = normal(r, c + 64, dtype=dt)[:, :c]
        if case["res"]:
            s["residual"] = normal(r, c, scale=4.0, dtype=_TYPES[case["res"]])
        if case["scale"] == "vector":
            s["scale"] = normal(c, scale=0.1, shift=0.5)
        elif case["scale"] == "scalar":
            s["scale"] = 0.25
        if case["next_norm"]:
            s["next_weight"] = normal(c, scale=0.1, shift=1.0)
            s["next_bias"] = normal(c, scale=0.1) if case["next_norm"] == "layer" else None
        return s
    step = op.endswith("_step")
    lens = [1] * case["batch"] if step else _lens(case)
    b = len(lens)
    if not step:
        starts, at = [], 0
        for i, n in enumerate(lens):
            starts.append(at if case["packed"] else i * max(lens))
            at += n
        s["starts"], s["lens"] = starts, lens
        if case["packed"]:
            s["cu_seqlens"] = torch.tensor([sum(lens[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
            lead = (sum(lens),)
        else:
            s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            lead = (b, max(lens))
    else:
        lead = (b,)
    pool = step or case["pool"]
    if pool:
        s["slots"] = slots(b)
        if not step:
            s["has_state"] = torch.rand(b, generator=g, device="cuda") < 0.5
    if op.startswith("conv"):
        c, k = case["channels"], case["ksize"]
        s["x"] = normal(*lead, c, dtype=dt)
        s["weight"] = uniform(-1, 1, c, k) * k ** -0.5
        s["bias"] = uniform(-0.5, 0.5, c)
        if pool:
            s["state"] = normal(b + 3, k - 1, c, dtype=dt)
        s["out"] = torch.zeros(*lead, c, dtype=dt, device="cuda")
        return s
    h, p, n, grp = case["heads"], case["head_dim"], case["d_state"], case["groups"]
    # x, B and C are slices of one convolution's output
    xbc = normal(*lead, h * p + 2 * grp * n, dtype=dt)
    s["x"] = xbc[..., :h * p].unflatten(-1, (h, p))
    s["B"] = xbc[..., h * p:h * p + grp * n].unflatten(-1, (grp, n))
    s["C"] = xbc[..., h * p + grp * n:].unflatten(-1, (grp, n))
    s["dt"] = normal(*lead, h, scale=0.5, dtype=dt)
    s["A"] = -uniform(1, 16, h)
    step_size = torch.exp(uniform(math.log(1e-3), math.log(0.1), h))
    s["dt_bias"] = step_size + torch.log(-torch.expm1(-step_size))
    s["D"] = normal(h, scale=0.1, shift=1.0)
    if pool:
        s["state"] = normal(b + 3, h, p, n)
    s["out"] = torch.zeros(*lead, h, p, dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------------------------------- plain forms

def _act(v, kind):
    if kind == "silu":
        return v / (1 + torch.exp(-v))
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    return v


def _norm(v, kind, weight, bias, groups, eps):
    if not kind:
        return v
    u = v.view(v.shape[0], groups, -1)
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    u = u.reshape(v.shape) * weight
    return u if bias is None else u + bias


def _plain_norm(s):
    case = s["case"]
    v = s["x"].float()
    gate = _act(s["gate"].float(), case["gate"]) if case["gate"] else None
    if gate is not None and case["gate_first"]:
        v = v * gate
    v = _norm(v, case["norm"], s.get("weight"), s.get("bias"), case["groups"], _EPS)
    if gate is not None and not case["gate_first"]:
        v = v * gate
    if not case["res"]:
        return v.to(s["x"].dtype)
    v = s["residual"].float() + v * s.get("scale", 1.0)
    o = _norm(v, case["next_norm"], s["next_weight"], s["next_bias"], 1, _EPS)
    return v.to(s["residual"].dtype), o.to(s["x"].dtype)


def _plain_conv(s):
    case, x = s["case"], s["x"]
    c, k = case["channels"], case["ksize"]
    flat = x.reshape(-1, c)
    out = torch.zeros(flat.shape[0], c, dtype=x.dtype, device=x.device)
    for i, (at, n) in enumerate(zip(s["starts"], s["lens"])):
        before = torch.zeros(k - 1, c, dtype=x.dtype, device=x.device)
        if "state" in s:
            before = torch.where(s["has_state"][i], s["state"][s["slots"][i].long()], before)
        rows = torch.cat([before, flat[at:at + n]])
        if "state" in s:
            s["state"].index_copy_(0, s["slots"][i:i + 1].long(), rows[n:][None])
        if n:
            v = s["bias"].expand(n, c)
            for j in range(k):
                v = v + s["weight"][:, j] * rows[j:j + n].float()
            out[at:at + n] = _act(v, "silu" if case["act"] else "").to(x.dtype)
    return (out.view_as(x), s["state"]) if "state" in s else out.view_as(x)


def _plain_conv_step(s):
    case, x = s["case"], s["x"]
    k, at = case["ksize"], s["slots"].long()
    rows = torch.cat([s["state"][at], x[:, None]], 1)
    v = s["bias"]
    for j in range(k):
        v = v + s["weight"][:, j] * rows[:, j].float()
    s["state"][at] = rows[:, 1:]
    return _act(v, "silu" if case["act"] else "").to(x.dtype), s["state"]


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _scan_terms(s):
    """Per row of the flattened leading axes, in fp32: decay [rows,H], dt * x [rows,H,P], D * x, B and C [rows,G,1,1,N]."""
    hn, p = s["x"].shape[-2:]
    x = s["x"].reshape(-1, hn, p).float()
    d = _softplus(s["dt"].reshape(-1, hn).float() + s["dt_bias"])
    bm, cm = (v.reshape(-1, v.shape[-2], 1, 1, v.shape[-1]).float() for v in (s["B"], s["C"]))
    return torch.exp(d * s["A"]), d[:, :, None] * x, s["D"][:, None] * x, bm, cm


def _token(h, decay, dx, skip, bm, cm):
    """One token of some requests: h [n,H,P,N] is updated in place; returns y [n,H,P]."""
    n, hn, p, ns = h.shape
    v = h.view(n, bm.shape[1], hn // bm.shape[1], p, ns)
    v.mul_(decay.view(n, v.shape[1], -1, 1, 1)).add_(dx.view(*v.shape[:4], 1) * bm)
    return (v * cm).sum(-1).view(n, hn, p) + skip


def _plain_scan(s):
    x = s["x"]
    hn, p, n = x.shape[-2], x.shape[-1], s["B"].shape[-1]
    lens, starts = s["lens"], s["starts"]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])  # longest first: the requests still running are a prefix
    dev = x.device
    h = torch.zeros(len(lens), hn, p, n, device=dev)
    pick = torch.tensor(order, device=dev)
    if "state" in s:
        at = s["slots"].long()[pick]
        h = torch.where(s["has_state"][pick][:, None, None, None], s["state"][at], h)
    first = torch.tensor([starts[i] for i in order], device=dev)
    terms = _scan_terms(s)
    out = torch.zeros(terms[1].shape, dtype=x.dtype, device=dev)
    for t in range(max(lens)):
        live = sum(1 for i in lens if i > t)
        if live == 1:
            rows = slice(starts[order[0]] + t, starts[order[0]] + t + 1)
        else:
            rows = first[:live] + t
        out[rows] = _token(h[:live], *(v[rows] for v in terms)).to(x.dtype)
    if "state" in s:
        s["state"][at] = h
        return out.view(s["out"].shape), s["state"]
    return out.view(s["out"].shape)


def _plain_scan_step(s):
    at = s["slots"].long()
    h = s["state"][at]
    y = _token(h, *_scan_terms(s))
    s["state"][at] = h
    return y.to(s["x"].dtype), s["state"]


# ---------------------------------------------------------------------------------------------- run, work

def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"norm": _plain_norm, "conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan,
                "scan_step": _plain_scan_step}[op](s)
    from mockingbird_amd import ssm
    if op == "norm":
        return ssm.block_norm(s["x"], s.get("weight"), s.get("bias"), norm=case["norm"] or None, eps=_EPS, groups=case["groups"],
                              gate=s.get("gate"), gate_act=None if case["gate"] in ("", "none") else case["gate"],
                              gate_first=case["gate_first"], residual=s.get("residual"), scale=s.get("scale"),
                              next_norm=case["next_norm"] or None, next_weight=s.get("next_weight"), next_bias=s.get("next_bias"),
                              next_eps=_EPS)
    act = "silu" if case.get("act") else None
    if op == "conv_step":
        return ssm.causal_conv1d_step(s["x"], s["state"], s["weight"], s["bias"], act, slots=s["slots"]), s["state"]
    if op == "scan_step":
        y = ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], s["D"], dt_bias=s["dt_bias"],
                                    dt_softplus=True, slots=s["slots"])
        return y, s["state"]
    seqs = dict(cu_seqlens=s.get("cu_seqlens"), lengths=s.get("lengths"), state=s.get("state"), slots=s.get("slots"),
                has_state=s.get("has_state"), out=s["out"])
    if op == "conv":
        y = ssm.causal_conv1d(s["x"], s["weight"], s["bias"], act, **seqs)
    else:
        y = ssm.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], dt_bias=s["dt_bias"], dt_softplus=True, **seqs)
    return (y, s["state"]) if "state" in s else y


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "": 0}
    e, op = size[case["dtype"]], case["op"]
    if op == "norm":
        r, c = case["rows"], case["channels"]
        moved = r * c * (e + (e if case["gate"] else 0) + 2 * size[case["res"]] + (e if case["next_norm"] or not case["res"] else 0))
        per = 2 + (8 if case["gate"] else 0) + (4 if case["norm"] else 0) + (2 if case["res"] else 0) + (4 if case["next_norm"] else 0)
        return {"bytes": moved + 4 * c * (bool(case["norm"]) + bool(case["next_norm"]) + (case["scale"] == "vector")), "flops": per * r * c}
    step = op.endswith("_step")
    b = case["batch"] if step else len(_lens(case))
    rows = b if step else sum(_lens(case))
    pool = step or case["pool"]
    if op.startswith("conv"):
        c, k = case["channels"], case["ksize"]
        return {"bytes": rows * c * 2 * e + (2 * b * (k - 1) * c * e if pool else 0) + 4 * c * (k + 1),
                "flops": rows * c * (2 * k + (4 if case["act"] else 0))}
    h, p, n, g = case["heads"], case["head_dim"], case["d_state"], case["groups"]
    return {"bytes": rows * (2 * h * p + 2 * g * n + h) * e + (2 * b * h * p * n * 4 if pool else 0) + 12 * h,
            "flops": rows * h * (5 * p * n + 3 * p + 8)}


# -------------------------------------------------------------------------------------- 64-bit definitions

def _exact_norm(s):
    case = s["case"]
    wide = {k: (v.double() if torch.is_tensor(v) else v) for k, v in s.items()}

    def squash(v):
        return torch.sigmoid(v) * (v if case["gate"] == "silu" else 1.0) if case["gate"] in ("silu", "sigmoid") else v

    def normed(v, kind, w, b, groups):
        parts = v.reshape(v.shape[0], groups, v.shape[1] // groups)
        centre = parts.sum(-1, keepdim=True) / parts.shape[-1] if kind == "layer" else 0.0
        power = ((parts - centre) ** 2).sum(-1, keepdim=True) / parts.shape[-1]
        flat = ((parts - centre) * (power + _EPS) ** -0.5).flatten(1)
        return flat * w + (0.0 if b is None else b)

    v = wide["x"]
    if case["gate"] and case["gate_first"]:
        v = squash(wide["gate"]) * v
    if case["norm"]:
        v = normed(v, case["norm"], wide["weight"], wide["bias"], case["groups"])
    if case["gate"] and not case["gate_first"]:
        v = squash(wide["gate"]) * v
    if not case["res"]:
        return v
    v = wide["residual"] + wide.get("scale", 1.0) * v
    return v, normed(v, case["next_norm"], wide["next_weight"], wide["next_bias"], 1)


def _requests(s):
    """(row numbers of the flattened leading axes, slot, keeps its state) of each request."""
    at = s["slots"].tolist() if "slots" in s else None
    if "starts" not in s:
        return [(torch.tensor([i], device="cuda"), at[i], True) for i in range(s["case"]["batch"])]
    keep = s["has_state"].tolist() if "has_state" in s else None
    return [(torch.arange(a, a + n, device="cuda"), at[i] if at else None, keep[i] if keep else False)
            for i, (a, n) in enumerate(zip(s["starts"], s["lens"]))]


def _exact_conv(s):
    case = s["case"]
    c, k = case["channels"], case["ksize"]
    x = s["x"].reshape(-1, c).double()
    y = torch.zeros_like(x)
    state = s["state"].double() if "state" in s else None
    taps = torch.arange(k, device="cuda")
    for rows, slot, keep in _requests(s):
        head = state[slot] if keep else torch.zeros(k - 1, c, dtype=torch.float64, device="cuda")
        line = torch.cat((head, x[rows]), 0)
        for part in torch.arange(len(rows), device="cuda").split(512):
            v = (line[part[:, None] + taps] * s["weight"].double().t()).sum(1) + s["bias"].double()
            y[rows[part]] = v * torch.sigmoid(v) if case["act"] else v
        if state is not None:
            state[slot] = line[len(line) - (k - 1):]
    y = y.reshape(s["x"].shape)
    return y if state is None else (y, state)


def _exact_scan(s):
    case = s["case"]
    h, p, n, g = case["heads"], case["head_dim"], case["d_state"], case["groups"]
    x = s["x"].reshape(-1, h, p).double()
    b, c = s["B"].reshape(-1, g, n).double(), s["C"].reshape(-1, g, n).double()
    raw = s["dt"].reshape(-1, h).double() + s["dt_bias"].double()
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    y = torch.zeros_like(x)
    state = s["state"].double() if "state" in s else None
    for rows, slot, keep in _requests(s):
        carry = state[slot].clone() if keep else torch.zeros(h, p, n, dtype=torch.float64, device="cuda")
        for part in rows.split(96):
            if not len(part):
                continue
            m = len(part)
            run_sum = torch.cumsum(dt[part] * s["A"].double(), 0).t()                       # [h, m]
            gap = run_sum[:, :, None] - run_sum[:, None, :]
            causal = torch.ones(m, m, dtype=torch.bool, device="cuda").tril()
            kernel = torch.where(causal, torch.exp(torch.where(causal, gap, 0.0)), 0.0) * dt[part].t()[:, None, :]
            bh = b[part].permute(1, 0, 2).repeat_interleave(h // g, 0).contiguous()         # [h, m, n]
            ch = c[part].permute(1, 0, 2).repeat_interleave(h // g, 0).contiguous()
            xh = x[part].permute(1, 0, 2).contiguous()                                      # [h, m, p]
            mix = torch.matmul(ch, bh.transpose(1, 2).contiguous()) * kernel
            grown = torch.matmul(ch, carry.transpose(1, 2).contiguous()) * torch.exp(run_sum)[:, :, None]
            y[part] = (torch.matmul(mix, xh) + grown + s["D"].double()[:, None, None] * xh).permute(1, 0, 2)
            tail = torch.exp(run_sum[:, -1:] - run_sum) * dt[part].t()
            carry = carry * torch.exp(run_sum[:, -1])[:, None, None] + torch.matmul((xh * tail[:, :, None]).transpose(1, 2).contiguous(), bh)
        if state is not None:
            state[slot] = carry
    y = y.reshape(s["x"].shape)
    return y if state is None else (y, state)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    return _exact_conv(s) if case["op"].startswith("conv") else _exact_scan(s)


if __name__ == "__main__":
    for one in listed() + [dict(draw(random.Random(i)), name=f"draw {i}") for i in range(6)]:
        print(one["name"], work(one))
