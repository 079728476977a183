"""The cases the router and the FP8 expert operators are measured at: Router, f8_quantize / f8_dequantize and GroupedMm over
FP8 operands with a scale for each block of 128, in plain torch (`own` false) or through this repository's package (`own`
true)."""
import math
import sys
from pathlib import Path

import torch

own = False

PKG = Path("radiance-exl3_b200").resolve()
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
BLOCK = 128         # values a scale covers: of a row of x, and 128 x 128 of a weight
TOP = 448.0         # e4m3's largest value
LEAST = 2.0 ** -110     # the least maximum a block's scale is made for


def _dense():
    if str(PKG) not in sys.path:
        sys.path.insert(0, str(PKG))
    from exl3b200 import dense
    return dense


def listed():
    """The layer sizes are this repository's: 512 experts of top-10 routing, hidden 2048 and width 512 (64 experts where
    the experts are few), the 2560 / 640 model geometry, the 4096 x 1536 linear; grouped routing over 256 experts."""
    route = {"op": "route", "E": 512, "k": 10, "dtype": "f32", "score": "softmax", "bias": False, "groups": 1, "keep": 1,
             "top": 1, "renorm": True, "scale": 1.0, "sort": True}
    grouped = dict(route, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4, top=2, scale=2.5)
    mm = {"op": "mm", "E": 512, "k": 10, "K": 2048, "N": 512, "act": "silu_mul", "gather": True, "x": "codes", "out": "bf16"}
    return [
        # one token's routing and sort: a launch's latency
        dict(route, name="route T=1 E=512 softmax", T=1),
        # a decode batch: sigmoid scores, a balance bias, four of eight groups; the sort too
        dict(grouped, name="route T=64 E=256 grouped", T=64),
        # a prefill pass's routing and sort, logits as a bf16 router product leaves them
        dict(route, name="route T=2048 E=512 softmax bf16", T=2048, dtype="bf16", renorm=False),
        # a long prompt's routing, for an engine that sorts by itself
        dict(grouped, name="route T=16384 E=256 grouped", T=16384, sort=False),
        # a decode batch's rows into FP8 and back
        {"op": "quant", "name": "f8 rows 64x2048 f16", "rows": 64, "H": 2048, "dtype": "f16", "out": "f16", "pow2": False},
        # the hidden rows of a long pass
        {"op": "quant", "name": "f8 rows 20480x4096 bf16", "rows": 20480, "H": 4096, "dtype": "bf16", "out": "bf16",
         "pow2": False},
        # one token through its ten gate/up matrices, its row quantised in the pass: the weights' bytes
        dict(mm, name="f8 mm T=1 E=512 gate_up", T=1, x="bf16"),
        # a decode batch's down product, the 2560 / 640 geometry, rows already sorted
        dict(mm, name="f8 mm T=64 E=512 down", T=64, K=640, N=2560, act="none", gather=False),
        # a prefill pass of the whole layer: 40 ragged rows an expert
        dict(mm, name="f8 mm T=2048 E=512 gate_up", T=2048, out="f16"),
        # a prefill pass over the 64 experts of one rank, quantised in the pass
        dict(mm, name="f8 mm T=2048 E=64 gate_up", T=2048, E=64, x="bf16"),
        # few large experts: bound by the tensor cores
        dict(mm, name="f8 mm T=4096 E=16 linear", T=4096, E=16, k=4, K=4096, N=1536, act="none"),
        # a shared expert's gate/up: one weight, every row
        dict(mm, name="f8 mm T=4096 E=1 shared", T=4096, E=1, k=1),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["route", "quant", "mm", "mm"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log_int(rng, 16, 512 // groups, rng.choice([1, 8]))
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(16, E // groups * keep))
        return {"op": op, "T": _log_int(rng, 1, 16384), "E": E, "k": k, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "keep": keep,
                "top": rng.choice([1, 2]), "renorm": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
                "sort": rng.random() < 0.5}
    if op == "quant":
        return {"op": op, "rows": _log_int(rng, 1, 20480), "H": _log_int(rng, 128, 4096, rng.choice([16, 128])),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "out": rng.choice(["bf16", "f32"]), "pow2": rng.random() < 0.3}
    while True:
        E, T = _log_int(rng, 1, 512), _log_int(rng, 1, 4096)
        k = min(E, rng.choice([1, 2, 4, 8, 10]))
        K, N = _log_int(rng, 128, 4096, rng.choice([16, 128])), _log_int(rng, 128, 4096, rng.choice([8, 128]))
        act = rng.choice(["none", "silu_mul"])
        wn = N * (2 if act == "silu_mul" else 1)
        # no dearer than the largest listed: its flops, and the prefill layer's weights
        if 2 * T * k * K * wn <= 2.0e11 and E * K * wn <= 1.07e9:
            break
    return {"op": "mm", "T": T, "E": E, "k": k, "K": K, "N": N, "act": act, "gather": rng.random() < 0.5,
            "x": rng.choice(["codes", "codes", "bf16", "f16"]), "out": rng.choice(["bf16", "f16", "f32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """N(0, 1) with a few channels some ten times larger, as hidden states have them."""
    big = 1 + 9 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
    return (torch.randn((rows, cols), generator=g, device="cuda") * big).to(dtype)


def _routing(g, T, E, k):
    """Top-k of log-normally popular experts, one slot in fifty dropped, sorted by expert: sorted_tok (slot index
    t * k + s, -1 past the live count), expert_offset, the fullest expert's rows."""
    logits = torch.randn((T, E), generator=g, device="cuda") + 0.8 * torch.randn(E, generator=g, device="cuda")
    ids = logits.topk(k, dim=1).indices
    ids = torch.where(torch.rand((T, k), generator=g, device="cuda") < 0.02, E, ids).reshape(-1)
    order = torch.sort(ids, stable=True).indices
    count = torch.bincount(ids, minlength=E + 1)[:E]
    offset = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offset[1:] = count.cumsum(0)
    place = torch.arange(T * k, device="cuda")
    return torch.where(place < offset[E], order, -1).to(torch.int32), offset, max(1, int(count.max()))


def _weight_blocks(c):
    """The scale blocks along a weight's rows: gate's and then up's for silu_mul."""
    return -(-c["N"] // BLOCK) * (2 if c["act"] == "silu_mul" else 1)


def _weight(g, c):
    """N(0, 0.02) weights as e4m3 codes with a scale for each 128 x 128 (gate's rows and up's rows in blocks of their own)."""
    E, K, N, halves = c["E"], c["K"], c["N"], 2 if c["act"] == "silu_mul" else 1
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    w = torch.empty((E, halves * N, K), dtype=F8, device="cuda")
    scales = torch.empty((E, halves * nb, kb), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (halves * N * K))            # experts at a time
    for e in range(0, E, step):
        n = min(step, E - e)
        v = torch.zeros((n, halves, nb * BLOCK, kb * BLOCK), dtype=torch.float32, device="cuda")
        v[:, :, :N, :K] = 0.02 * torch.randn((n, halves, N, K), generator=g, device="cuda")
        b = v.view(n, halves, nb, BLOCK, kb, BLOCK)
        s = b.abs().amax((3, 5), keepdim=True) / TOP
        q = (b / s).clamp(-TOP, TOP).view(v.shape)[:, :, :N, :K]
        w[e:e + n] = q.reshape(n, halves * N, K).to(F8)
        scales[e:e + n] = s.reshape(n, halves * nb, kb)
    return w, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    s = dict(case=case)
    d = s["dense"] = _dense() if own else None
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        s["logits"] = (1.5 * torch.randn((T, E), generator=g, device="cuda")
                       + 0.5 * torch.randn(E, generator=g, device="cuda")).to(DT[c["dtype"]])
        s["bias"] = 0.05 * torch.randn(E, generator=g, device="cuda") if c["bias"] else None
        if own:
            ints = dict(dtype=torch.int32, device="cuda")
            s["got"] = {"ids": torch.empty((T, k), **ints), "w": torch.empty((T, k), device="cuda")}
            if c["sort"]:
                s["got"] |= {"sorted_tok": torch.empty(T * k, **ints), "expert_offset": torch.empty(E + 1, **ints)}
            s["plan"] = d.Router(logits=s["logits"], bias=s["bias"], top_k=k, score=c["score"], groups=c["groups"],
                                 keep_groups=c["keep"], group_top=c["top"], renorm=c["renorm"], scale=c["scale"], **s["got"])
    elif c["op"] == "quant":
        s["x"] = _activations(g, c["rows"], c["H"], DT[c["dtype"]])
        if own:
            s["q"], s["qs"] = d.f8_empty(c["rows"], c["H"], device="cuda")
            s["y"] = torch.empty((c["rows"], c["H"]), dtype=DT[c["out"]], device="cuda")
    else:
        T, E, k, K, N = (c[n] for n in ("T", "E", "k", "K", "N"))
        s["tok"], s["offset"], s["most"] = _routing(g, T, E, k)
        rows = T if c["gather"] else T * k
        s["w"], s["ws"] = _weight(g, c)
        if c["x"] == "codes":
            s["x"], s["xs"] = _quantised(_activations(g, rows, K, torch.bfloat16), False)
        else:
            s["x"] = _activations(g, rows, K, DT[c["x"]])
        if own:
            s["y"] = torch.empty((T * k, N), dtype=DT[c["out"]], device="cuda")
            x, xs = d.f8_empty(rows, K, device="cuda")
            if c["x"] == "codes":
                x, xs = x.copy_(s["x"]), xs.copy_(s["xs"])
            s["q"], s["qs"] = x, xs
            s["plan"] = d.GroupedMm(x=x, w=s["w"], x_scales=xs, w_scales=s["ws"], expert_offset=s["offset"],
                                    sorted_tok=s["tok"], top_k=k if c["gather"] else 0, act=c["act"], y=s["y"])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _quantised(x, pow2):
    """x [rows, cols] as e4m3 codes and a scale for each 128 values of a row."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    b = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, BLOCK)
    m = b.abs().amax(-1, keepdim=True).clamp(min=LEAST)
    top = torch.full_like(m, TOP)           # tensors: a Python number's quotient is a product with its rounded reciprocal
    s = m / top
    if pow2:
        s = _pow2_up(s)
        v = b / s
    else:
        v = b * (top / m)
    q = v.clamp(-TOP, TOP).view(rows, -1)[:, :cols].to(F8)
    return q, s[..., 0].contiguous()


def _pow2_up(s):
    """The least power of two from s (normal, 32 bits) on, from its bits."""
    bits = s.view(torch.int32)
    return ((bits + 0x7FFFFF) & 0x7F800000).view(torch.float32)


def _spread(scales, cols):
    return scales.repeat_interleave(BLOCK, -1)[..., :cols]


def _run_route(s):
    c, l = s["case"], s["logits"].double()      # 64 bits: choices between neighbouring scores
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    choice = score + s["bias"].double() if c["bias"] else score
    T, E, G = c["T"], c["E"], c["groups"]
    if G > 1:
        best = torch.sort(choice.view(T, G, -1), dim=2, descending=True).values[..., :c["top"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        live = torch.zeros((T, G), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = choice.masked_fill(~live.repeat_interleave(E // G, 1), -math.inf)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    got = {"ids": ids.to(torch.int32), "w": (w * c["scale"]).float()}
    if c["sort"]:
        flat = ids.reshape(-1)
        got["sorted_tok"] = torch.sort(flat, stable=True).indices.to(torch.int32)
        offset = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        offset[1:] = (flat[:, None] == torch.arange(E, device="cuda")).sum(0).cumsum(0)
        got["expert_offset"] = offset
    return got


def _run_mm(s):
    c = s["case"]
    q, qs = (s["x"], s["xs"]) if c["x"] == "codes" else _quantised(s["x"], False)
    x = q.float() * _spread(qs, c["K"])
    w = s["w"].float()
    halves = 2 if c["act"] == "silu_mul" else 1
    per = _spread(s["ws"], c["K"]).view(c["E"], halves, -1, c["K"]).repeat_interleave(BLOCK, 2)[:, :, :c["N"]]
    w = w * per.reshape(w.shape)
    off = s["offset"].long()
    # every expert's rows padded to the fullest one's
    slot = off[:-1, None] + torch.arange(s["most"], device="cuda")
    live = slot < off[1:, None]
    slot = torch.where(live, slot, 0)
    src = torch.clamp(s["tok"].long()[slot] // c["k"], min=0) if c["gather"] else slot
    z = torch.bmm(x[src], w.transpose(1, 2))
    if c["act"] == "silu_mul":
        z = z[..., :c["N"]] * torch.sigmoid(z[..., :c["N"]]) * z[..., c["N"]:]
    y = torch.zeros((c["T"] * c["k"], c["N"]), device="cuda", dtype=DT[c["out"]])
    y[slot[live]] = z[live].to(y.dtype)
    return y


def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "route":
            return _run_route(s)
        if c["op"] == "quant":
            q, qs = _quantised(s["x"], c["pow2"])
            return {"values": (q.float() * _spread(qs, c["H"])).to(DT[c["out"]]), "scales": qs}
        return _run_mm(s)
    dense, stream = s["dense"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "route":
        s["plan"].run(stream)
        return s["got"]
    if c["op"] == "quant":
        dense.f8_quantize(s["x"], s["q"], s["qs"], pow2=c["pow2"], stream=stream)
        return {"values": dense.f8_dequantize(s["q"], s["qs"], s["y"], stream=stream), "scales": s["qs"]}
    if c["x"] != "codes":
        dense.f8_quantize(s["x"], s["q"], s["qs"], stream=stream)
    s["plan"].run(stream)
    return s["y"]


# ------------------------------------------------------------------------------------------------ work and exact values
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
F8_SIZE = 1 + 4 / BLOCK


def work(case):
    c = case
    if c["op"] == "route":
        b = c["T"] * (c["E"] * SIZE[c["dtype"]] + 8 * c["k"]) + (4 * c["E"] if c["bias"] else 0)
        return {"bytes": b + (4 * c["T"] * c["k"] + 4 * (c["E"] + 1) if c["sort"] else 0), "flops": 4 * c["T"] * c["E"]}
    if c["op"] == "quant":
        n = c["rows"] * c["H"]
        return {"bytes": n * (SIZE[c["dtype"]] + 2 * F8_SIZE + SIZE[c["out"]]), "flops": 4 * n}
    T, E, k, K, N = (c[n] for n in ("T", "E", "k", "K", "N"))
    wn = N * (2 if c["act"] == "silu_mul" else 1)
    live = E * (1 - (1 - k / E) ** T)                      # experts some row reads, popularity aside
    rows = T if c["gather"] else T * k
    x_size = F8_SIZE if c["x"] == "codes" else 2 + 2 * F8_SIZE
    return {"bytes": live * (wn * K + 4 * _weight_blocks(c) * -(-K // BLOCK)) + rows * K * x_size
            + T * k * N * SIZE[c["out"]], "flops": 2 * T * k * K * wn}


def _nearest_e4m3(v):
    """The e4m3 value nearest v (64 bits), ties to the even mantissa, from the exponent and its spacing."""
    a = v.abs()
    _, e = torch.frexp(a)                                   # a = m 2^e, m in [0.5, 1)
    gap = torch.ldexp(torch.ones_like(a), torch.clamp(e - 4, min=-9))
    n = a / gap
    lo = torch.floor(n)
    up = (n - lo > 0.5) | ((n - lo == 0.5) & (lo % 2 == 1))
    return torch.sign(v) * torch.clamp((lo + up) * gap, max=448.0)


def _exact_f8(x, pow2):
    """(values, scales) by the definition: the 32-bit numbers the definition names are rounded to 32 bits, nothing else."""
    rows, cols = x.shape
    b = torch.zeros((rows, -(-cols // 128) * 128), dtype=torch.float64, device="cuda")
    b[:, :cols] = x.double()
    b = b.view(rows, -1, 128)
    m = torch.clamp(b.abs().max(-1, keepdim=True).values, min=2.0 ** -110)
    s = (m / 448).float().double()
    if pow2:
        f, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), torch.where(f == 0.5, e - 1, e))
        v = b / s
    else:
        v = (b * (448 / m).float().double()).float().double()
    return (_nearest_e4m3(v) * s).view(rows, -1)[:, :cols], s[..., 0]


def _exact_route(c, s):
    l, T, E, k, G = s["logits"].double(), c["T"], c["E"], c["k"], c["groups"]
    if c["score"] == "softmax":
        score = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    else:
        score = torch.exp(-torch.log1p(torch.exp(-l)))
    choice = score + (s["bias"].double() if c["bias"] else 0)
    at = torch.arange(E, device="cuda")
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    step = max(1, (1 << 27) // (E * E))
    for t in range(0, T, step):
        v = choice[t:t + step]
        if G > 1:
            by = v.view(v.shape[0], G, -1)
            best, where = by.max(2)
            if c["top"] == 2:
                best = best + by.scatter(2, where[..., None], -math.inf).max(2).values
            ga = torch.arange(G, device="cuda")
            ahead = (best[:, None] > best[..., None]) | ((best[:, None] == best[..., None]) & (ga < ga[:, None]))
            v = torch.where((ahead.sum(2) < c["keep"]).repeat_interleave(E // G, 1), v, -math.inf)
        # an expert's place is the number of those ahead of it
        place = ((v[:, None] > v[..., None]) | ((v[:, None] == v[..., None]) & (at < at[:, None]))).sum(2)
        r, e = torch.nonzero(place < k, as_tuple=True)
        ids[t + r, place[r, e]] = e.to(torch.int32)
    w = score.gather(1, ids.long())
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    got = {"ids": ids, "w": w * c["scale"]}
    if c["sort"]:
        flat = ids.reshape(-1).long()
        count = torch.bincount(flat, minlength=E)
        got["sorted_tok"] = torch.argsort(flat * flat.numel() + torch.arange(flat.numel(), device="cuda")).to(torch.int32)
        got["expert_offset"] = torch.cat((torch.zeros_like(count[:1]), count.cumsum(0))).to(torch.int32)
    return got


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "route":
        return _exact_route(c, s)
    if c["op"] == "quant":
        v, sc = _exact_f8(s["x"], c["pow2"])
        return {"values": v, "scales": sc}
    tok, off, K, N = s["tok"].tolist(), s["offset"].tolist(), c["K"], c["N"]
    if c["x"] == "codes":
        x = s["x"].double() * s["xs"].double()[:, torch.arange(K, device="cuda") // 128]
    else:
        x = _exact_f8(s["x"], False)[0]
    row = torch.arange(s["w"].shape[1], device="cuda")
    block = torch.where(row < N, row // 128, -(-N // 128) + (row - N) // 128)
    col = torch.arange(K, device="cuda") // 128
    y = torch.zeros((c["T"] * c["k"], N), dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        rows = torch.tensor([t // c["k"] for t in tok[a:b]], device="cuda") if c["gather"] else slice(a, b)
        z = x[rows] @ (s["w"][e].double() * s["ws"][e].double()[block][:, col]).T
        if c["act"] == "silu_mul":
            z = z[:, :N] / (1 + torch.exp(-z[:, :N])) * z[:, N:]
        y[a:b] = z
    return y
