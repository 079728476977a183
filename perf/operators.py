"""The cases the dense and MXFP4 expert operators are measured at: block_norm, mx4_quantize / mx4_dequantize and
grouped_mm (f16 / bf16 / MXFP4), in plain torch (`own` false) or through this repository's package (`own` true)."""
import math
import sys
from pathlib import Path

import torch

own = False

PKG = Path("radiance-exl3_b200").resolve()
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32          # values an MXFP4 scale covers


def _dense():
    if str(PKG) not in sys.path:
        sys.path.insert(0, str(PKG))
    from exl3b200 import dense
    return dense


def listed():
    """The layer sizes are this repository's: 512 experts of top-10 routing, hidden 2048 and width 512 (64 experts where
    the experts are few), the 2560 / 640 model geometry, the 4096 x 1536 linear."""
    norm = {"op": "norm", "branch": "f32", "dtype": "bf16", "post": True, "gate": "none", "pre": True, "mx4": False}
    mm = {"op": "mm", "E": 512, "k": 10, "K": 2048, "N": 512, "act": "silu_mul", "gather": True, "dtype": "f16",
          "out": "f16"}
    mx = dict(mm, dtype="mx4", x="bf16", out="bf16")
    return [
        # one token's residual step between two blocks: a launch's latency
        dict(norm, name="norm T=1 H=2048", T=1, H=2048),
        # a prefill pass in f16 with an element gate
        dict(norm, name="norm T=2048 H=2560 gated", T=2048, H=2560, dtype="f16", branch="f16", gate="element"),
        # a long prompt: gated shared branch, the next block's input in bf16 and in MXFP4
        dict(norm, name="norm T=16384 H=4096 mx4", T=16384, H=4096, gate="token", mx4=True),
        # a decode batch's rows into MXFP4 and back
        {"op": "quant", "name": "quant 64x2048 f16", "rows": 64, "H": 2048, "dtype": "f16", "out": "f16"},
        # the hidden rows of a long pass
        {"op": "quant", "name": "quant 20480x4096 bf16", "rows": 20480, "H": 4096, "dtype": "bf16", "out": "bf16"},
        # one token through its ten gate/up matrices: the weights' bytes
        dict(mm, name="mm T=1 E=512 gate_up f16", T=1),
        # a decode batch's down product, the 2560 / 640 geometry, rows already sorted
        dict(mm, name="mm T=64 E=512 down bf16", T=64, K=640, N=2560, act="none", gather=False, dtype="bf16",
             out="bf16"),
        # a prefill pass of the whole layer: 40 ragged rows an expert
        dict(mm, name="mm T=2048 E=512 gate_up f16", T=2048),
        # few large experts: bound by the tensor cores
        dict(mm, name="mm T=4096 E=16 linear bf16", T=4096, E=16, k=4, K=1536, N=4096, act="none", dtype="bf16",
             out="bf16"),
        # one token through its ten MXFP4 gate/up matrices, its row quantised in the pass
        dict(mx, name="mx4 T=1 E=512 gate_up", T=1),
        # a prefill pass over the 64 experts of one rank, quantised in the pass
        dict(mx, name="mx4 T=2048 E=64 gate_up", T=2048, E=64),
        # few large MXFP4 experts, the rows' codes in hand
        dict(mx, name="mx4 T=4096 E=16 linear", T=4096, E=16, k=4, K=4096, N=1536, act="none", x="codes"),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["norm", "quant", "mm", "mx4"])
    if op == "norm":
        mx4 = rng.random() < 0.4
        H = _log_int(rng, 128, 4096, 32 if mx4 else 1 if rng.random() < 0.2 else 8)
        return {"op": op, "T": _log_int(rng, 1, 16384), "H": H, "branch": rng.choice(["f32", "bf16", "f16"]),
                "dtype": rng.choice(["bf16", "f16"]), "post": rng.random() < 0.8,
                "gate": rng.choice(["none", "token", "channel", "element"]), "pre": rng.random() < 0.8 or mx4,
                "mx4": mx4}
    if op == "quant":
        return {"op": op, "rows": _log_int(rng, 1, 20480), "H": _log_int(rng, 32, 4096, 32),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "out": rng.choice(["bf16", "f32"])}
    step = 8 if op == "mm" else 32
    while True:
        E, T = _log_int(rng, 1, 512), _log_int(rng, 1, 4096)
        k = min(E, rng.choice([1, 2, 4, 8, 10]))
        K, N = _log_int(rng, 256, 4096, step), _log_int(rng, 128, 4096, step)
        act = rng.choice(["none", "silu_mul"])
        wn = N * (2 if act == "silu_mul" else 1)
        # no dearer than the largest listed: its flops, the prefill layer's weights, and padded rows that fit the card
        if 2 * T * k * K * wn <= 2.0e11 and E * K * wn <= 1.07e9 and 3072 not in (K, N, wn):
            break
    case = {"op": "mm", "T": T, "E": E, "k": k, "K": K, "N": N, "act": act, "gather": rng.random() < 0.5}
    if op == "mm":
        d = rng.choice(["f16", "bf16"])
        return dict(case, dtype=d, out=d)
    return dict(case, dtype="mx4", x=rng.choice(["bf16", "f16", "codes"]), out=rng.choice(["bf16", "f16"]))


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _activations(g, rows, cols, dtype):
    """N(0, 1) with a few channels some ten times larger, as hidden states have them."""
    big = 1 + 9 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
    return (torch.randn((rows, cols), generator=g, device="cuda") * big).to(dtype)


def _routing(g, T, E, k):
    """Top-k of log-normally popular experts, one slot in fifty dropped, sorted by expert: sorted_tok (slot index
    t * k + s, -1 past the live count), expert_offset."""
    logits = torch.randn((T, E), generator=g, device="cuda") + 0.8 * torch.randn(E, generator=g, device="cuda")
    ids = logits.topk(k, dim=1).indices
    ids = torch.where(torch.rand((T, k), generator=g, device="cuda") < 0.02, E, ids).reshape(-1)
    order = torch.sort(ids, stable=True).indices
    count = torch.bincount(ids, minlength=E + 1)[:E]
    offset = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offset[1:] = count.cumsum(0)
    place = torch.arange(T * k, device="cuda")
    return torch.where(place < offset[E], order, -1).to(torch.int32), offset, max(1, int(count.max()))


def _codes(g, *shape):
    """Random e2m1 codes, two a byte, and the E8M0 scales of blocks of weights around 0.02 (or 1 for rows of x)."""
    return torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, device="cuda", dtype=torch.uint8)


def _scales(g, centre, *shape):
    return torch.randint(centre - 2, centre + 2, (*shape[:-1], shape[-1] // BLOCK), generator=g, device="cuda",
                         dtype=torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if own:
        s["dense"] = _dense()
    if case["op"] == "norm":
        T, H, dt = case["T"], case["H"], DT[case["dtype"]]
        s |= {"branch": _activations(g, T, H, DT[case["branch"]]), "res": _activations(g, T, H, dt),
              "post_w": _randn(g, H, scale=0.1).add_(1).to(dt) if case["post"] else None,
              "pre_w": _randn(g, H, scale=0.1).add_(1).to(dt) if case["pre"] else None,
              "gate": {"none": lambda: None, "token": lambda: _randn(g, T), "channel": lambda: _randn(g, H, dtype=dt),
                       "element": lambda: _randn(g, T, H, dtype=dt)}[case["gate"]](), "res_scale": 0.75, "eps": 1e-6}
        if own:
            s["out"] = torch.empty((T, H), dtype=dt, device="cuda")
            s["y"] = torch.empty((T, H), dtype=dt, device="cuda") if case["pre"] else None
            if case["mx4"]:
                s["q"], s["qs"] = s["dense"].mx4_empty(T, H, device="cuda")
                s["qv"] = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
            s["plan"] = s["dense"].BlockNorm(branch=s["branch"], post_w=s["post_w"], post_eps=s["eps"], gate=s["gate"],
                                           gate_kind=case["gate"], res=s["res"], res_scale=s["res_scale"],
                                           out=s["out"], pre_w=s["pre_w"], pre_eps=s["eps"], y=s["y"],
                                           y_codes=s.get("q"), y_scales=s.get("qs"))
    elif case["op"] == "quant":
        s["x"] = _activations(g, case["rows"], case["H"], DT[case["dtype"]])
        if own:
            s["q"], s["qs"] = s["dense"].mx4_empty(case["rows"], case["H"], device="cuda")
            s["y"] = torch.empty((case["rows"], case["H"]), dtype=DT[case["out"]], device="cuda")
    else:
        T, E, k, K, N = (case[n] for n in ("T", "E", "k", "K", "N"))
        wn = N * (2 if case["act"] == "silu_mul" else 1)
        s["tok"], s["offset"], s["most"] = _routing(g, T, E, k)
        rows = T if case["gather"] else T * k
        if case["dtype"] == "mx4":
            s["w"], s["ws"] = _codes(g, E, wn, K), _scales(g, 120, E, wn, K)
            if case["x"] == "codes":
                s["x"], s["xs"] = _codes(g, rows, K), _scales(g, 126, rows, K)
            else:
                s["x"] = _activations(g, rows, K, DT[case["x"]])
        else:
            s["x"] = _activations(g, rows, K, DT[case["dtype"]])
            s["w"] = torch.empty((E, wn, K), dtype=DT[case["dtype"]], device="cuda").normal_(0, 0.02, generator=g)
        if own:
            s["y"] = torch.empty((T * k, N), dtype=DT[case["out"]], device="cuda")
            x, xs, ws = s["x"], s.get("xs"), s.get("ws")
            if case["dtype"] == "mx4":
                ws = s["dense"].mx4_tile_scales(ws, act=case["act"])
                if xs is None:
                    x, xs = s["q"], s["qs"] = s["dense"].mx4_empty(rows, K, device="cuda")
            s["plan"] = s["dense"].GroupedMm(x=x, w=s["w"], x_scales=xs, w_scales=ws, expert_offset=s["offset"],
                                           sorted_tok=s["tok"], top_k=k if case["gather"] else 0, act=case["act"],
                                           y=s["y"])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _round_e2m1(v):
    """|v| / step rounded half to even on e2m1's grid (0 .5 1 1.5 2 3 4 6), saturating."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.clamp(torch.round(a / step) * step, max=6.0), v)


def _pow2(e):
    """2^e for whole e in [-127, 127], from its bits: a power function may be off by the last one, which moves ties."""
    return torch.where(e < -126, 1 << 22, (e.int() + 127) << 23).int().view(torch.float32)


def _mx4_values(x):
    """The values x takes in MXFP4, in 32 bits."""
    b = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))          # amax = m * 2^e, m in [0.5, 1)
    s = _pow2(torch.clamp(e - 3, min=-127))
    return (_round_e2m1(b / s) * s).reshape(x.shape)


def _decode(codes, scales):
    """The values that e2m1 codes (low nibble first) and their E8M0 scales stand for, in 32 bits."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    n = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1, BLOCK)
    v = grid[n.int()] * _pow2(scales.int() - 127)[..., None]
    return v.reshape(*codes.shape[:-1], -1)


def _rms(v, eps, w):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.float()


def _run_norm(s):
    c, dt = s["case"], DT[s["case"]["dtype"]]
    n = s["branch"].float()
    n = _rms(n, s["eps"], s["post_w"]) if c["post"] else n
    gate = s["gate"].float() if s["gate"] is not None else None
    n = {"none": lambda: n, "token": lambda: n * torch.sigmoid(gate)[:, None], "channel": lambda: n * gate,
         "element": lambda: n * torch.sigmoid(gate)}[c["gate"]]()
    r = s["res"].float() * s["res_scale"] + n
    got = {"out": r.to(dt)}
    if c["pre"]:
        y = _rms(r, s["eps"], s["pre_w"])
        got["y"] = y.to(dt)
        if c["mx4"]:
            got["y_mx4"] = _mx4_values(y).to(torch.bfloat16)
    return got


def _run_mm(s):
    c = s["case"]
    if c["dtype"] == "mx4":
        x = _decode(s["x"], s["xs"]) if c["x"] == "codes" else _mx4_values(s["x"])
        w = _decode(s["w"], s["ws"])
    else:
        x, w = s["x"].float(), s["w"].float()
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
        if c["op"] == "norm":
            return _run_norm(s)
        if c["op"] == "quant":
            return _mx4_values(s["x"]).to(DT[c["out"]])
        return _run_mm(s)
    dense, stream = s["dense"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm":
        s["plan"].run(stream)
        got = {"out": s["out"]}
        if c["pre"]:
            got["y"] = s["y"]
        if c["mx4"]:
            got["y_mx4"] = dense.mx4_dequantize(s["q"], s["qs"], s["qv"], stream)
        return got
    if c["op"] == "quant":
        dense.mx4_quantize(s["x"], s["q"], s["qs"], stream)
        return dense.mx4_dequantize(s["q"], s["qs"], s["y"], stream)
    if "q" in s:
        dense.mx4_quantize(s["x"], s["q"], s["qs"], stream)
    s["plan"].run(stream)
    return s["y"]


# ------------------------------------------------------------------------------------------------ work and exact values
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
MX4 = 0.5 + 1 / BLOCK


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["T"] * c["H"]
        size = SIZE[c["dtype"]]
        b = n * (SIZE[c["branch"]] + 2 * size + (size if c["pre"] else 0) + (size if c["gate"] == "element" else 0))
        b += (c["T"] * 4 if c["gate"] == "token" else 0) + c["H"] * size * (c["post"] + c["pre"])
        return {"bytes": b + (n * (2 * MX4 + 2) if c["mx4"] else 0), "flops": n * (5 + 5 * c["pre"])}
    if c["op"] == "quant":
        n = c["rows"] * c["H"]
        return {"bytes": n * (SIZE[c["dtype"]] + 2 * MX4 + SIZE[c["out"]]), "flops": 4 * n}
    T, E, k, K, N = (c[n] for n in ("T", "E", "k", "K", "N"))
    wn = N * (2 if c["act"] == "silu_mul" else 1)
    live = E * (1 - (1 - k / E) ** T)                      # experts some row reads, popularity aside
    rows = T if c["gather"] else T * k
    w_size = MX4 if c["dtype"] == "mx4" else 2
    x_size = w_size if c.get("x", "codes") == "codes" else 2 + 2 * MX4
    return {"bytes": live * wn * K * w_size + rows * K * x_size + T * k * N * SIZE[c["out"]],
            "flops": 2 * T * k * K * wn}


def _two_to(e):
    return ((e + 1023) << 52).view(torch.float64)


def _exact_mx4(x):
    """MXFP4 by its definition, value by value against the midpoints of the grid, in 64 bits."""
    b = x.double().reshape(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    s = _two_to(torch.clamp((top.view(torch.int64) >> 52) - 1023 - 2, min=-127))     # the exponent field: floor(log2)
    a = b.abs() / s
    # one grid step up for each midpoint passed; a midpoint itself goes to the value with the even mantissa (0, 1, 2, 4)
    v = (0.5 * ((a > .25).double() + (a >= .75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5).double() + (a >= 3.5)
         + 2 * (a > 5).double())
    return (v * b.sign() * s).reshape(x.shape)


def _exact_decode(codes, scales):
    lo, hi = codes.long() & 15, codes.long() >> 4
    n = torch.stack((lo, hi), -1).flatten(-2)
    e, m = (n >> 1) & 3, n & 1
    v = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * _two_to(e - 1))
    return torch.where(n > 7, -v, v) * _two_to(scales.long() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "quant":
        return _exact_mx4(s["x"])
    if c["op"] == "norm":
        n = s["branch"].double()
        if c["post"]:
            n = n / torch.sqrt((n * n).mean(1, keepdim=True) + s["eps"]) * s["post_w"].double()
        if c["gate"] != "none":
            g = s["gate"].double()
            g = g[:, None] if c["gate"] == "token" else g
            n = n * (g if c["gate"] == "channel" else 1 / (1 + torch.exp(-g)))
        r = s["res_scale"] * s["res"].double() + n
        got = {"out": r}
        if c["pre"]:
            got["y"] = r / torch.sqrt((r * r).mean(1, keepdim=True) + s["eps"]) * s["pre_w"].double()
        if c["mx4"]:
            got["y_mx4"] = None      # a step function of y: a value beside a midpoint goes either way with y's last bit
        return got
    tok, off = s["tok"].tolist(), s["offset"].tolist()
    if c["dtype"] != "mx4":
        x = s["x"].double()
    else:
        x = _exact_decode(s["x"], s["xs"]) if c["x"] == "codes" else _exact_mx4(s["x"])
    y = torch.zeros((c["T"] * c["k"], c["N"]), dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        rows = torch.tensor([t // c["k"] for t in tok[a:b]], device="cuda") if c["gather"] else slice(a, b)
        w = _exact_decode(s["w"][e], s["ws"][e]) if c["dtype"] == "mx4" else s["w"][e].double()
        z = x[rows] @ w.T
        if c["act"] == "silu_mul":
            gate, up = z[:, :c["N"]], z[:, c["N"]:]
            z = gate / (1 + torch.exp(-gate)) * up
        y[a:b] = z
    return y
