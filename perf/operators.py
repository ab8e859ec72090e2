"""Cases that measure the routed-expert and optimizer operators: what one pass is, its plain form, and its definition in 64 bits.

Operators (``kind`` of a case):

``route``    top-k softmax of a router's logits and, when ``train``, the gradient of the logits
``experts``  samples sorted by expert and back with weights applied; when ``train`` all three gradients
``adamw``    one AdamW step over many tensors with the moments in 8 or 32 bits, optionally clipped by the global norm
``clip``     the global gradient norm over many tensors and the scaling by it

``run`` computes the plain form with elementary torch operations, or calls the framework's operators where ``own`` is true.

The 8-bit moments, as this file decodes and encodes them: blocks of 256 elements of one tensor share a power-of-two scale 2^e
for each moment. The first moment is a sign, 4 exponent and 3 mantissa bits; the second is 5 exponent and 3 mantissa bits. e is
the exponent of the block's largest magnitude once that is rounded up to 3 mantissa bits. A value is rounded to one of its two
neighbours with a 16-bit dither, a hash of (seed, tensor, step, index), so that the expectation of what is stored is the value.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 256                       # elements that share a scale
M_EMIN, V_EMIN = -14, -30         # smallest normal exponents of the two codes, relative to the block's scale
MASK = 0xFFFFFFFF
# 2^32 / golden ratio, and the fractional bits of sqrt(2) and sqrt(3): odd multipliers of the dither's hash
PHI, SQ2, SQ3 = 0x9E3779B1, 0x6A09E667, 0xBB67AE85
BETAS, EPS, LR, DECAY, SEED = (0.9, 0.999), 1e-8, 3e-4, 1e-2, 20

# the taxi-fare MLP: Linear 20-256-128-64-16-1 and four BatchNorms
NYC = "5120,256,32768,128,8192,64,1024,16,16,1,256,256,128,128,64,64,16,16"


def _dlrm(rows):
    """The recommendation model's towers (13-512-128-32 and 384-1024-1024-512-256-1) and one parameter for its 26 tables."""
    return "6656,512,65536,128,4096,32,393216,1024,1048576,1024,524288,512,131072,256,256,1,%d" % (26 * 32 * rows)


def _expert_lens(count, d, h):
    """``count`` two-layer experts d -> h -> d with biases."""
    return ",".join([str(d * h), str(h), str(h * d), str(d)] * count)


def listed():
    return [
        # one sample answered by a trained model with a routed tower: latency
        dict(name="route, one row", kind="route", T=1, E=16, k=1, dtype="float32", renorm=True, masked=0.0, train=False),
        # a training batch of the recommendation benchmark through a 64-expert router
        dict(name="route, batch 2048, train", kind="route", T=2048, E=64, k=2, dtype="float32", renorm=True, masked=0.0, train=True),
        # a wide batch, many small experts, some of them masked for some rows, padding rows with all masked
        dict(name="route, 65536 x 256, train", kind="route", T=65536, E=256, k=8, dtype="bfloat16", renorm=False, masked=0.05, train=True),
        # one sample through the routed tower on the interaction's 384 features
        dict(name="experts, one row", kind="experts", T=1, E=16, k=2, D=384, dtype="float32", capacity=0, dropped=0.0, train=False),
        # a ragged batch with capacity-limited experts (static shapes, so that the step can be captured)
        dict(name="experts, 2047 x 383, capacity", kind="experts", T=2047, E=8, k=2, D=383, dtype="float32", capacity=640, dropped=0.02,
             train=True),
        # a wide bf16 batch without drops
        dict(name="experts, 65536 x 1024", kind="experts", T=65536, E=64, k=2, D=1024, dtype="bfloat16", capacity=0, dropped=0.0, train=True),
        # the taxi model's step, clipped: 18 small tensors, latency
        dict(name="adamw 8, taxi model, clipped", kind="adamw", lens=NYC, dtype="float32", bits=8, clip=0.1),
        # the recommendation model with its tables
        dict(name="adamw 8, 36 M fp32", kind="adamw", lens=_dlrm(40000), dtype="float32", bits=8, clip=0.0),
        # 48 experts in bf16, 192 tensors
        dict(name="adamw 8, 50 M bf16, clipped", kind="adamw", lens=_expert_lens(48, 512, 1023), dtype="bfloat16", bits=8, clip=1.0),
        # the same model as above with moments in 32 bits
        dict(name="adamw 32, 36 M fp32", kind="adamw", lens=_dlrm(40000), dtype="float32", bits=32, clip=0.0),
        # clipping before another optimizer's step: few small tensors, and 64 experts' many large ones
        dict(name="clip, taxi model", kind="clip", lens=NYC, dtype="float32", clip=0.1),
        dict(name="clip, 64 experts fp32", kind="clip", lens=_expert_lens(64, 512, 1024), dtype="float32", clip=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_lens(rng, most):
    count, total = _spread(rng, 1, 200), _spread(rng, 1000, most)
    part = [rng.expovariate(1.0) ** 2 + 1e-6 for _ in range(count)]
    return ",".join(str(max(1, int(total * w / sum(part)))) for w in part)


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "adamw", "adamw", "clip"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind == "route":
        E = _spread(rng, 2, 256)
        return dict(kind=kind, T=_spread(rng, 1, 65536), E=E, k=rng.randint(1, min(8, E)), dtype=dtype, renorm=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.1]), train=rng.random() < 0.7)
    if kind == "experts":
        T, E, k = _spread(rng, 1, 32768), _spread(rng, 2, 256), rng.randint(1, 4)
        capacity = rng.choice([0, max(1, int(1.25 * T * k / E))])
        return dict(kind=kind, T=T, E=E, k=k, D=_spread(rng, 16, 1024), dtype=dtype, capacity=capacity, dropped=rng.choice([0.0, 0.05]),
                    train=rng.random() < 0.7)
    if kind == "adamw":
        return dict(kind=kind, lens=_draw_lens(rng, 36_000_000), dtype=dtype, bits=rng.choice([8, 8, 32]), clip=rng.choice([0.0, 1.0]))
    return dict(kind=kind, lens=_draw_lens(rng, 64_000_000), dtype=dtype, clip=1.0)


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def work(case):
    size = {"float32": 4, "bfloat16": 2}[case.get("dtype", "float32")]
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        both = 2 if case["train"] else 1
        return {"bytes": both * (T * E * size + T * k * 4) + T * k * 4, "flops": both * T * (4 * E + 8 * k)}
    if case["kind"] == "experts":
        T, E, k, D = case["T"], case["E"], case["k"], case["D"]
        n = T * k
        rows = E * case["capacity"] if case["capacity"] else n
        kept = min(rows, n)
        row = D * size
        # ids, weights, position, source; x -> rows; expert outputs -> y; and dy -> dh, dw; drows -> dx
        b = n * 12 + rows * 4 + (T + rows) * row + (kept + T) * row
        if case["train"]:
            b += n * 4 + (T + rows) * row + (kept + T) * row
        return {"bytes": b, "flops": n * D * (2 + (5 if case["train"] else 0))}
    n = sum(_lens(case))
    if case["kind"] == "adamw":
        # parameter and moments read and written, gradient read; 8-bit moments also come back as the bf16 values they stand for
        state = 8 * 2 if case["bits"] == 32 else 2 * 2 + 4 / BLOCK + 4
        return {"bytes": n * (3 * size + state), "flops": n * (16 if case["bits"] == 32 else 40)}
    return {"bytes": n * 2 * size, "flops": 3 * n}


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _segments(case):
    """The layout of many tensors in one flat buffer: each starts at a whole block; [blocks] of a block's tensor and first index."""
    lens = _lens(case)
    blocks = [-(-n // BLOCK) for n in lens]
    first = [0]
    for b in blocks:
        first.append(first[-1] + b)
    lens_t = torch.tensor(lens, device=DEV)
    which = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(blocks, device=DEV))
    base = (torch.arange(first[-1], device=DEV) - torch.tensor(first[:-1], device=DEV)[which]) * BLOCK
    live = base[:, None] + torch.arange(BLOCK, device=DEV) < lens_t[which][:, None]
    return lens, [f * BLOCK for f in first[:-1]], which, base, live


def _views(flat, lens, starts):
    return [flat.view(-1)[s:s + n] for n, s in zip(lens, starts)]


def prepare(case, seed):
    g = _gen(seed)
    dtype = getattr(torch, case["dtype"])
    if case["kind"] == "route":
        T, E = case["T"], case["E"]
        logits = _randn(g, T, E) * 2
        if case["masked"]:
            logits = logits.masked_fill(torch.rand(T, E, generator=g, device=DEV) < case["masked"], -math.inf)
            logits[torch.rand(T, generator=g, device=DEV) < case["masked"] / 4] = -math.inf   # padding rows
        return {"case": case, "logits": logits.to(dtype).requires_grad_(own and case["train"]), "dw": _randn(g, T, case["k"])}
    if case["kind"] == "experts":
        T, E, k, D = case["T"], case["E"], case["k"], case["D"]
        # a router's choices: some experts are liked more than others; k different ones for a row, or none
        liking = _randn(g, E) * 0.5
        ids = torch.argsort(_randn(g, T, E) + liking, dim=1, descending=True)[:, :min(k, E)]
        ids = torch.cat([ids, ids[:, :1].expand(-1, k - ids.shape[1])], 1).int().contiguous()
        if case["dropped"]:
            ids[torch.rand(T, generator=g, device=DEV) < case["dropped"]] = -1
        rows = E * case["capacity"] if case["capacity"] else T * k
        grad = own and case["train"]
        return {"case": case, "ids": ids, "x": _randn(g, T, D).to(dtype).requires_grad_(grad),
                "w": torch.softmax(_randn(g, T, k), 1).requires_grad_(grad),
                "h": _randn(g, rows, D).to(dtype).requires_grad_(grad), "dy": _randn(g, T, D).to(dtype),
                "drows": _randn(g, rows, D).to(dtype)}
    lens, starts, which, base, live = _segments(case)
    shape = live.shape
    # gradients of tensors differ in scale, and of the elements of one tensor too
    spread = torch.exp(_randn(g, len(lens)))[which][:, None] * torch.exp(_randn(g, *shape))
    grad = (_randn(g, *shape) * spread * 1e-3 * live).to(dtype)
    s = {"case": case, "g": grad, "lens": lens, "starts": starts}
    if case["kind"] == "clip":
        if own:
            s["params"] = []
            for v in _views(grad, lens, starts):
                p = torch.nn.Parameter(torch.empty_like(v))
                p.grad = v
                s["params"].append(p)
        return s
    s.update(which=which, base=base, t=11, p=(_randn(g, *shape) * 0.05 * live).to(dtype))
    # moments as the eleven steps before this one leave them
    m = _randn(g, *shape) * spread * 2e-4 * live
    v = torch.square(spread * 1e-3) * (0.5 + torch.rand(shape, generator=g, device=DEV)) * 0.01 * live
    if case["bits"] == 32:
        s.update(m=m, v=v)
    else:
        half = torch.full(shape, 1 << 15, dtype=torch.int64, device=DEV)
        (mc, ms), (vc, vs) = _encode(m.abs(), half, M_EMIN, False), _encode(v, half, V_EMIN, True)
        s.update(m=(mc | (m < 0).long() * 128).to(torch.uint8), v=vc.to(torch.uint8),
                 scales=torch.stack([ms, vs], 1).to(torch.uint8))
    if own:
        from raydp_amd.ops.fused_optim import FusedAdamW
        params = [torch.nn.Parameter(v) for v in _views(s["p"], lens, starts)]
        for p, v in zip(params, _views(grad, lens, starts)):
            p.grad = v
        opt = FusedAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                         max_grad_norm=case["clip"] or None, seed=SEED)
        blocks = [x // BLOCK for x in starts] + [shape[0]]
        for i, (p, em, ev) in enumerate(zip(params, _views(s["m"], lens, starts), _views(s["v"], lens, starts))):
            opt.state[p] = {"step": torch.tensor(float(s["t"]), device=DEV), "exp_avg": em, "exp_avg_sq": ev}
            if case["bits"] == 8:
                opt.state[p]["scales"] = s["scales"][blocks[i]:blocks[i + 1]]
        s["opt"] = opt
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _mix(x):
    """Two rounds of shift and multiply on 32-bit values held in 64."""
    x = x & MASK
    x = ((x ^ (x >> 16)) * SQ2) & MASK
    x = ((x ^ (x >> 15)) * SQ3) & MASK
    return x ^ (x >> 16)


def _dither(which, base, t):
    """32 random bits for every element: low half for the first moment, high half for the second."""
    key = _mix(_mix(SEED + which * PHI) + t)
    idx = base[:, None] + torch.arange(BLOCK, device=base.device)
    return _mix((idx & MASK) * PHI + (idx >> 32) * SQ2 + key[:, None])


def _pow2(e):
    """2^e in 64 bits, exactly."""
    return ((e + 1023) << 52).view(torch.float64)


def _encode(x, rnd16, emin, positive):
    """Codes without sign and biased scale exponents of blocks x >= 0 (32 bits)."""
    top = x.contiguous().view(torch.int32).long().amax(1)
    s = (top + 0xFFFFF) >> 23
    y = x.double() * _pow2(127 - s.clamp(min=1))[:, None]
    f = ((y.view(torch.int64) >> 52) - 1023).clamp(min=emin)
    grid = y * _pow2(3 - f)
    code = ((torch.round(grid * 2.0 ** 20).long() + rnd16 * 16 + 8) >> 20) + 8 * (f - emin)
    if positive:   # what is not zero stays so: it is divided by
        code = torch.where(x > 0, code.clamp(min=1), code)
    return code, s


def _decode(code, s, emin):
    e, man = code >> 3, code & 7
    val = torch.where(e > 0, (8 + man).double() * _pow2((e - 1).clamp(min=0) + emin - 3), man.double() * 2.0 ** (emin - 3))
    return val * _pow2(s.clamp(min=1) - 127)[:, None]


def _plain_route(z, dw, k, renorm, train):
    z32 = z.float()
    top, ids = torch.sort(z32, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    there = top > -math.inf
    peak = torch.where(there[:, :1], top[:, :1], 0.0)
    e = torch.where(there, torch.exp(top - peak), 0.0)
    total = e.sum(1, keepdim=True) if renorm else torch.exp(z32 - peak).sum(1, keepdim=True)
    w = e / torch.where(total > 0, total, 1.0)
    out = {"weights": w, "experts": torch.where(there, ids, -1).int()}
    if train:
        s = (w * dw).sum(1, keepdim=True)
        if renorm:
            dz = torch.zeros_like(z32).scatter(1, ids, w * (dw - s))
        else:
            p = torch.exp(z32 - peak) / torch.where(total > 0, total, 1.0)
            dz = p * (torch.zeros_like(z32).scatter(1, ids, torch.where(there, dw, 0.0)) - s)
        out["dlogits"] = dz.to(z.dtype)
    return out


def _plain_experts(s):
    case, ids, x, w, h, dy, drows = (s[n] for n in ("case", "ids", "x", "w", "h", "dy", "drows"))
    E, C, n, k = case["E"], case["capacity"], ids.numel(), ids.shape[1]
    R = h.shape[0]
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order_key, order = torch.sort(key, stable=True)
    load = torch.zeros(E + 1, dtype=torch.int64, device=DEV).scatter_add(0, key, torch.ones_like(key))
    start = torch.cumsum(load, 0) - load
    every = torch.arange(n, device=DEV)
    rank = torch.zeros_like(key).scatter(0, order, every - start[order_key])
    base = torch.arange(E + 1, device=DEV) * C if C else start
    keep = (key < E) & (rank < C) if C else key < E
    pos = torch.where(keep, base[key] + rank, R)
    source = torch.full((R + 1,), -1, dtype=torch.int64, device=DEV).scatter(0, pos, every)[:R]
    filled, token = (source >= 0)[:, None], source.clamp(min=0) // k
    at = pos.clamp(max=R - 1).view(-1, k)
    kept = keep.view(-1, k)
    hk = h.float()[at] * kept[:, :, None]
    out = {"position": torch.where(keep, pos, -1).view(-1, k).int(), "source": source.int(), "load": load[:E].int(),
           "rows": torch.where(filled, x[token], 0.0), "y": (hk * w[:, :, None]).sum(1).to(x.dtype)}
    if case["train"]:
        dy32 = dy.float()
        out["dh"] = torch.where(filled, w.reshape(-1)[source.clamp(min=0)][:, None] * dy32[token], 0.0).to(x.dtype)
        out["dw"] = (hk * dy32[:, None, :]).sum(2)
        out["dx"] = (drows.float()[at] * kept[:, :, None]).sum(1).to(x.dtype)
    return out


def _plain_clip(g, limit):
    """The norm, and the factor that brings it under the limit. Long sums: 64 bits."""
    norm = torch.sqrt(torch.square(g.double()).sum())
    return norm.float(), (limit / (norm + 1e-6)).clamp(max=1.0).float()


def _plain_adamw(s):
    case, out = s["case"], {}
    s["t"] += 1
    t, (b1, b2) = s["t"], BETAS
    g = s["g"].float()
    if case["clip"]:
        out["norm"], scale = _plain_clip(s["g"], case["clip"])
        g = g * scale
    small = case["bits"] == 8
    if small:
        mc, vc, sc = s["m"].long(), s["v"].long(), s["scales"].long()
        m = (_decode(mc & 127, sc[:, 0], M_EMIN) * (1 - (mc >> 7) * 2)).float()
        v = _decode(vc, sc[:, 1], V_EMIN).float()
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    step = (-LR / (1 - b1 ** t)) * m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** t)) + EPS)
    p = s["p"].float() * (1 - LR * DECAY) + step
    low = s["p"].dtype == torch.bfloat16
    if small or low:
        h = _dither(s["which"], s["base"], t)
    if small:
        # moments decay by 1 - b2 = 0.1 % a step, a fiftieth of a code's spacing: rounded to nearest they would never move
        (mc, ms), (vc, vs) = _encode(m.abs(), h & 0xFFFF, M_EMIN, False), _encode(v, h >> 16, V_EMIN, True)
        s["m"].copy_(mc | (m < 0).long() * 128)
        s["v"].copy_(vc)
        s["scales"].copy_(torch.stack([ms, vs], 1))
        m = (_decode(mc, ms, M_EMIN) * torch.where(m < 0, -1.0, 1.0)).to(torch.bfloat16)   # 4 significant bits: exact
        v = _decode(vc, vs, V_EMIN).to(torch.bfloat16)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if low:        # parameters without a master copy: the same rounding in expectation
        bits = p.view(torch.int32).long() & MASK
        bits = (bits + (((h * SQ2) & MASK) >> 16)) >> 16 << 16
        p = torch.where(bits > 0x7FFFFFFF, bits - (1 << 32), bits).int().view(torch.float32)
    s["p"].copy_(p)
    return dict(out, p=s["p"], m=m, v=v)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        return _own(state)
    if kind == "route":
        return _plain_route(state["logits"], state["dw"], case["k"], case["renorm"], case["train"])
    if kind == "experts":
        return _plain_experts(state)
    if kind == "adamw":
        return _plain_adamw(state)
    norm, scale = _plain_clip(state["g"], case["clip"])
    state["g"].copy_(state["g"].float() * scale)
    return {"norm": norm, "g": state["g"]}


def _own(state):
    case = state["case"]
    if case["kind"] == "route":
        from raydp_amd.ops.expert_ops import route
        w, ids = route(state["logits"], case["k"], renormalize=case["renorm"])
        out = {"weights": w, "experts": ids}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad(w, state["logits"], state["dw"])
        return out
    if case["kind"] == "experts":
        from raydp_amd.ops.expert_ops import combine, dispatch, expert_plan
        plan = expert_plan(state["ids"], case["E"], capacity=case["capacity"] or None)
        rows = dispatch(state["x"], plan)
        y = combine(state["h"], plan, state["w"])
        out = {"position": plan.position, "source": plan.source, "load": plan.load, "rows": rows, "y": y}
        if case["train"]:
            out["dh"], out["dw"] = torch.autograd.grad(y, (state["h"], state["w"]), state["dy"])
            out["dx"], = torch.autograd.grad(rows, state["x"], state["drows"])
        return out
    if case["kind"] == "clip":
        from raydp_amd.ops.fused_optim import clip_grad_norm_
        return {"norm": clip_grad_norm_(state["params"], case["clip"]), "g": state["g"]}
    from raydp_amd.ops.fused_optim import decode_moments
    opt = state["opt"]
    opt.step()
    out = {"norm": opt.grad_norm} if case["clip"] else {}
    m, v = state["m"], state["v"]
    if case["bits"] == 8:
        m, v = decode_moments(m, v, state["scales"], torch.bfloat16)
    return dict(out, p=state["p"], m=m, v=v)


# ------------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    """The first pass on prepare(case, seed), from the definitions, on real numbers held in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(s)
    if kind == "experts":
        return _exact_experts(s)
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if kind == "clip":
        return {"norm": norm, "g": g * min(1.0, case["clip"] / (float(norm) + 1e-6))}
    return _exact_adamw(s, g, norm)


def _exact_route(s):
    case, z = s["case"], s["logits"].detach().double()
    T, E = z.shape
    k, column = case["k"], torch.arange(E, device=DEV)
    left, ids, zs = z.clone(), [], []
    for _ in range(k):                      # the largest that is left, the lowest index where there are several
        best = left.amax(1, keepdim=True)
        i = torch.where(left == best, column, E).amin(1)
        none = best[:, 0] == -math.inf
        ids.append(torch.where(none, -1, i))
        zs.append(best[:, 0])
        left[torch.arange(T, device=DEV), i] = -math.inf
    ids, zs = torch.stack(ids, 1), torch.stack(zs, 1)
    lse = torch.logsumexp(zs if case["renorm"] else z, 1, keepdim=True)
    w = torch.where(ids >= 0, torch.exp(zs - lse), 0.0)
    out = {"weights": w, "experts": ids.int()}
    if case["train"]:
        chosen = (ids[:, :, None] == column).double()
        at = torch.einsum("tk,tke->te", s["dw"].double(), chosen) if T * k * E < 1 << 24 else \
            sum(s["dw"][:, j:j + 1].double() * chosen[:, j] for j in range(k))
        p = torch.where(z > -math.inf, torch.exp(z - lse), 0.0)
        if case["renorm"]:
            p = p * chosen.sum(1)
        out["dlogits"] = p * (at - (p * at).sum(1, keepdim=True))
    return out


def _exact_experts(s):
    case, ids = s["case"], s["ids"].reshape(-1).cpu()
    k, R, C = s["ids"].shape[1], s["h"].shape[0], case["capacity"]
    source, load, at = torch.full((R,), -1, dtype=torch.int64), [], 0
    for e in range(case["E"]):
        mine = torch.nonzero(ids == e).flatten()
        load.append(mine.numel())
        mine = mine[:C] if C else mine
        at = e * C if C else at
        source[at:at + mine.numel()] = mine
        at += mine.numel()
    r = torch.nonzero(source >= 0).flatten()
    position = torch.full((ids.numel(),), -1, dtype=torch.int64)
    position[source[r]] = r
    r, src = r.to(DEV), source[r].to(DEV)
    tok = src // k
    x, w, h, dy, drows = (s[n].detach().double() for n in ("x", "w", "h", "dy", "drows"))
    wr = w.reshape(-1)[src][:, None]
    out = {"position": position.view(-1, k).int(), "source": source.int(), "load": torch.tensor(load, dtype=torch.int32),
           "rows": torch.zeros_like(h).index_copy(0, r, x[tok]), "y": torch.zeros_like(x).index_add(0, tok, wr * h[r])}
    if case["train"]:
        out["dh"] = torch.zeros_like(h).index_copy(0, r, wr * dy[tok])
        out["dw"] = torch.zeros_like(w).view(-1).index_copy(0, src, (h[r] * dy[tok]).sum(1)).view_as(w)
        out["dx"] = torch.zeros_like(x).index_add(0, tok, drows[r])
    return out


def _exact_adamw(s, g, norm):
    case, t, (b1, b2) = s["case"], s["t"] + 1, BETAS
    if case["clip"]:
        g = g * min(1.0, case["clip"] / (float(norm) + 1e-6))
    small = case["bits"] == 8

    def value(code, scale, emin):
        e, man = torch.div(code, 8, rounding_mode="floor").double(), (code % 8).double()
        mag = torch.where(e == 0, man / 8 * 2.0 ** emin, (1 + man / 8) * torch.exp2(e - 1 + emin))
        return mag * torch.exp2(scale.clamp(min=1).double() - 127)[:, None]

    def rounded(x, rnd, emin):
        """|x| to the format's grid: up where the part that is cut off and the dither reach one."""
        top = x.amax(1)
        mant, ex = torch.frexp(top)
        # the largest magnitude, rounded up to 3 mantissa bits, has to fit under 2 * 2^e
        ex = torch.where(torch.ceil(mant * 16) >= 16, ex + 1, ex) - 1
        scale = torch.exp2(ex.double())[:, None]
        y = torch.where(top[:, None] > 0, x / scale, 0.0)
        unit = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=emin).double() - 3)
        cut = y / unit
        up = cut - torch.floor(cut) + (rnd.double() + 0.5) / 65536 >= 1
        return (torch.floor(cut) + up) * unit * scale, unit * scale

    if small:
        m = value(s["m"].long() % 128, s["scales"][:, 0].long(), M_EMIN) * torch.where(s["m"] > 127, -1.0, 1.0)
        v = value(s["v"].long(), s["scales"][:, 1].long(), V_EMIN)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = s["p"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    h = _dither(s["which"], s["base"], t)
    if small:
        m = rounded(m.abs(), h & 0xFFFF, M_EMIN)[0] * torch.sign(m)
        q, unit = rounded(v, h >> 16, V_EMIN)
        v = torch.where((v > 0) & (q == 0), unit, q)
    if case["dtype"] == "bfloat16":
        unit = torch.exp2(torch.frexp(p)[1].double() - 8)
        cut = p.abs() / unit
        up = cut - torch.floor(cut) + (((h * SQ2) & MASK) >> 16).double() / 65536 >= 1
        p = torch.where(p == 0, 0.0, (torch.floor(cut) + up) * unit * torch.sign(p))
    out = {"p": p, "m": m, "v": v}
    return dict(out, norm=norm) if case["clip"] else out
