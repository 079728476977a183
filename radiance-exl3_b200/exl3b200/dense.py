"""dense.py -- experts whose weights are not EXL3 records (f16, bf16, FP8 or MXFP4), the router before them and the norms
around a block, over torch tensors: grouped_mm, router, block_norm and the FP8 and MXFP4 conversions of libexl3b200.so
(include/exl3b200.h).

A GroupedMm, Router or BlockNorm is a plan: it reads its tensors' addresses, shapes and strides once, keeps the tensors alive, and
`run(stream)` enqueues the call on a cudaStream_t (an integer; 0 the legacy default stream). Every entry's default is torch's
current stream. The tensors' contents may change between runs, their addresses may not. A call's tensors share one GPU, which
is the current device when it runs. torch only holds memory here. Tensors that do not fit one another are a ValueError; what
the library refuses is a RuntimeError with its status. MXFP4 rows are two uint8 tensors: codes [rows, cols / 2] and scales
[rows, cols / 32]. FP8 rows: codes of float8_e4m3fn [rows, cols] and f32 scales [rows, ceil(cols / 128)]."""
import ctypes as C

import torch

from .native import BlockNormDesc, ExpertBlockDesc, GroupedMmDesc, Native, RouterDesc

MX4 = 1024 + 0x3B4                      # EXL3B_MX4
F8 = 1024 + 0x3B8                       # EXL3B_F8
DTYPES = {torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
ACTS = {"none": 0, "silu_mul": 1}
SCORES = {"softmax": 0, "sigmoid": 1}
SORT_PAIRS = 2048                       # a sort of up to so many pairs needs no work buffer
GATES = {"none": 0, "token": 1, "channel": 2, "element": 3}

_native = None
_several = True                         # more than one GPU here: with one there is no other that could be current


def native():
    global _native, _several
    if _native is None:
        _native, _several = Native(), torch.cuda.device_count() != 1
    return _native


def _dtype(t):
    dt = DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"f32, f16 or bf16, not {t.dtype}")
    return dt


def _check_current(dev):
    """The library launches on the current device: a call's tensors have to be there."""
    if torch.cuda.current_device() != dev:
        raise ValueError(f"the tensors are on cuda:{dev}, the current device is cuda:{torch.cuda.current_device()}")


def _current_stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _rows(t, name, dev, shape=None, dtype=None):
    """A tensor whose last dimension is dense, on GPU dev (that of the call's first tensor), of this shape and type:
    (address, row pitch in elements)."""
    if t is None:
        raise ValueError(f"{name} is missing")
    have, st = t.shape, t.stride()
    if not (t.get_device() == dev >= 0 and (dtype is None or t.dtype is dtype) and (shape is None or have == shape)
            and (st[-1] == 1 or have[-1] <= 1)):
        what = ("is not on a GPU" if t.get_device() < 0 else f"is on {t.device}, not cuda:{dev}" if t.get_device() != dev else
                f"is {t.dtype}, not {dtype}" if dtype not in (None, t.dtype) else
                f"has shape {tuple(have)}, not {tuple(shape)}" if shape is not None and have != shape else
                "has a strided last dimension")
        raise ValueError(f"{name} {what}")
    if len(st) < 2:
        return t.data_ptr(), 0
    return t.data_ptr(), st[-2] if have[-2] > 1 else max(st[-2], have[-1])


# ------------------------------------------------------------------------------------------------ MXFP4
def mx4_empty(rows, cols, device="cuda"):
    """(codes, scales) for `rows` rows of `cols` values; the scales' rows 16 bytes apart or a multiple, which GroupedMm
    reads fastest."""
    return (torch.empty((rows, cols // 2), dtype=torch.uint8, device=device),
            torch.empty((rows, (cols // 32 + 15) // 16 * 16), dtype=torch.uint8, device=device)[:, :cols // 32])


def mx4_quantize(x, codes, scales, stream=None):
    """x [rows, cols] in f32, f16 or bf16 -> its MXFP4 codes and scales."""
    rows, cols = x.shape
    dev = x.get_device()
    xp, pitch = _rows(x, "x", dev)
    cp, c_pitch = _rows(codes, "codes", dev, (rows, cols // 2), torch.uint8)
    sp, s_pitch = _rows(scales, "scales", dev, (rows, cols // 32), torch.uint8)
    if _several:
        _check_current(dev)
    rc = native().lib.exl3b200_mx4_quantize(xp, _dtype(x), pitch, rows, cols, cp, c_pitch, sp, s_pitch,
                                           _current_stream(dev) if stream is None else stream)
    if rc:
        raise RuntimeError(f"exl3b200_mx4_quantize: status {rc}")
    return codes, scales


def mx4_dequantize(codes, scales, y, stream=None):
    """The values that codes and scales stand for, into y [rows, cols] (f32, f16 or bf16)."""
    rows, cols = y.shape
    dev = y.get_device()
    yp, pitch = _rows(y, "y", dev)
    cp, c_pitch = _rows(codes, "codes", dev, (rows, cols // 2), torch.uint8)
    sp, s_pitch = _rows(scales, "scales", dev, (rows, cols // 32), torch.uint8)
    if _several:
        _check_current(dev)
    rc = native().lib.exl3b200_mx4_dequantize(cp, c_pitch, sp, s_pitch, rows, cols, yp, _dtype(y), pitch,
                                             _current_stream(dev) if stream is None else stream)
    if rc:
        raise RuntimeError(f"exl3b200_mx4_dequantize: status {rc}")
    return y


def mx4_tile_scales(scales, act="none", stream=None):
    """A weight's scales [experts, rows, cols / 32] in the form GroupedMm reads; once, when the weight is loaded."""
    n_expert, rows, blocks = scales.shape
    dev = scales.get_device()
    sp, pitch = _rows(scales, "scales", dev, dtype=torch.uint8)
    if _several:
        _check_current(dev)
    n = native().mx4_tiled_bytes(n_expert, rows, blocks * 32, ACTS[act])
    here = _current_stream(dev)
    if stream is None or stream == here:
        stream, out = here, torch.empty(n, dtype=torch.uint8, device=scales.device)
    else:                               # memory of that stream's: this one's pool may hand out what is still in use here
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, dev) if stream else torch.cuda.default_stream(dev)):
            out = torch.empty(n, dtype=torch.uint8, device=scales.device)
    native().mx4_tile_scales(sp, pitch, scales.stride(0), n_expert, rows, blocks * 32, ACTS[act], out.data_ptr(), stream)
    return out


# ------------------------------------------------------------------------------------------------ FP8
def f8_empty(rows, cols, device="cuda"):
    """(codes, scales) for `rows` rows of `cols` values; the scales' rows 16 bytes apart or a multiple, which GroupedMm
    reads fastest."""
    blocks = (cols + 127) // 128
    return (torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=device),
            torch.empty((rows, (blocks + 3) // 4 * 4), dtype=torch.float32, device=device)[:, :blocks])


def _f8_rows(x, codes, scales, name):
    """Both conversions' checks: x's GPU, type and pitch, (address, pitch) of the codes and of the scales."""
    dev, shape, xs, cs, ss = x.get_device(), x.shape, x.stride(), codes.stride(), scales.stride()
    if (dev == codes.get_device() == scales.get_device() >= 0 and len(xs) == 2 and shape[0] > 1 and codes.shape == shape
            and scales.shape == (shape[0], (shape[1] + 127) // 128) and 1 == xs[1] == cs[1] == ss[1]
            and codes.dtype is torch.float8_e4m3fn and scales.dtype is torch.float32):
        at = codes.data_ptr(), cs[0], scales.data_ptr(), ss[0]      # what _rows finds, in one go: a call costs a microsecond less
        pitch = xs[0]
    else:
        if len(shape) != 2:
            raise ValueError(f"{name} has {len(shape)} dimensions, not 2")
        _, pitch = _rows(x, name, dev)
        at = _rows(codes, "codes", dev, (shape[0], shape[1]), torch.float8_e4m3fn)
        at += _rows(scales, "scales", dev, (shape[0], (shape[1] + 127) // 128), torch.float32)
    if _several:
        _check_current(dev)
    return dev, DTYPES.get(x.dtype) or _dtype(x), pitch, at


def f8_quantize(x, codes, scales, pow2=False, stream=None):
    """x [rows, cols] in f32, f16 or bf16 -> its e4m3 codes and their scales (pow2: powers of two)."""
    dev, dt, pitch, at = _f8_rows(x, codes, scales, "x")
    rc = native().lib.exl3b200_f8_quantize(x.data_ptr(), dt, pitch, *x.shape, *at, pow2,
                                           _current_stream(dev) if stream is None else stream)
    if rc:
        raise RuntimeError(f"exl3b200_f8_quantize: status {rc}")
    return codes, scales


def f8_dequantize(codes, scales, y, stream=None):
    """The values that codes and scales stand for, into y [rows, cols] (f32, f16 or bf16)."""
    dev, dt, pitch, at = _f8_rows(y, codes, scales, "y")
    rc = native().lib.exl3b200_f8_dequantize(*at, *y.shape, y.data_ptr(), dt, pitch,
                                             _current_stream(dev) if stream is None else stream)
    if rc:
        raise RuntimeError(f"exl3b200_f8_dequantize: status {rc}")
    return y


# ------------------------------------------------------------------------------------------------ plans
class _Plan:
    _entry = None

    def _finish(self, desc, dev, *tensors):
        self.desc, self._dev, self._keep = desc, dev, tensors
        self._addr, self._call = C.addressof(desc), getattr(native().lib, self._entry)

    def run(self, stream=None):
        if _several:
            _check_current(self._dev)
        rc = self._call(self._addr, _current_stream(self._dev) if stream is None else stream)
        if rc:
            raise RuntimeError(f"{self._entry}: status {rc}")


class GroupedMm(_Plan):
    """y[i] = x[t(i)] @ w[e(i)].T for the sorted rows i of the routing contract (act "silu_mul": silu of the first half
    of w's rows times the second).

    x [x_rows, n_in] and w [experts, w_rows, n_in] in f16 or bf16; or MXFP4 codes (uint8, half as wide) with x_scales
    [x_rows, n_in / 32] and w_scales from mx4_tile_scales; or FP8 (float8_e4m3fn) with f32 x_scales [x_rows, ceil(n_in / 128)]
    and w_scales [experts, blocks, ceil(n_in / 128)], a block each 128 weight rows (silu_mul: ceil(n_out / 128) blocks of gate
    rows, then as many of up rows), the two scales' product a normal f32 number. y [rows, n_out] in f32, f16 or bf16, or (not
    from FP8) MXFP4 codes with y_scales. expert_offset i32 [experts + 1] (None: one expert); sorted_tok i32 [rows] (None: no
    dropped slot). top_k: row i reads x row sorted_tok[i] // top_k; 0: x is sorted already."""
    _entry = "exl3b200_grouped_mm"

    def __init__(self, *, x, w, y, expert_offset=None, sorted_tok=None, top_k=0, act="none", x_scales=None,
                 w_scales=None, y_scales=None):
        mx, f8, mx_out = w.dtype == torch.uint8, w.dtype == torch.float8_e4m3fn, y.dtype == torch.uint8
        d = GroupedMmDesc()
        per, per_out = 2 if mx else 1, 2 if mx_out else 1
        if x.dtype != w.dtype:
            raise ValueError(f"x is {x.dtype}, w {w.dtype}")
        if (x.dim(), w.dim(), y.dim()) != (2, 3, 2):
            raise ValueError(f"x, w and y have {x.dim()}, {w.dim()} and {y.dim()} dimensions, not 2, 3 and 2")
        dev = x.get_device()
        d.n_expert, d.n_rows, d.x_rows, d.top_k = w.shape[0], y.shape[0], x.shape[0], top_k
        d.n_out, d.n_in, d.act = y.shape[1] * per_out, x.shape[1] * per, ACTS[act]
        d.dtype, d.y_dtype = MX4 if mx else F8 if f8 else _dtype(x), MX4 if mx_out else _dtype(y)
        _rows(w, "w", dev, (d.n_expert, d.n_out * (2 if d.act else 1), x.shape[1]))
        d.x, pitch = _rows(x, "x", dev)
        d.x_pitch = pitch * per
        d.w, pitch = _rows(w, "w", dev)
        d.w_pitch, d.w_expert_pitch = pitch * per, w.stride(0) * per
        d.y, pitch = _rows(y, "y", dev)
        d.y_pitch = pitch * per_out
        if mx:
            d.x_scales, d.x_scales_pitch = _rows(x_scales, "x_scales", dev, (d.x_rows, d.n_in // 32), torch.uint8)
            want = native().mx4_tiled_bytes(d.n_expert, w.shape[1], d.n_in, d.act)
            d.w_scales, _ = _rows(w_scales, "w_scales", dev, (want,), torch.uint8)
        if f8:
            kb = (d.n_in + 127) // 128
            d.x_scales, pitch = _rows(x_scales, "x_scales", dev, (d.x_rows, kb), torch.float32)
            d.x_scales_pitch = pitch * 4
            blocks = (d.n_out + 127) // 128 * (2 if d.act else 1)
            d.w_scales, _ = _rows(w_scales, "w_scales", dev, (d.n_expert, blocks, kb), torch.float32)
            if not w_scales.is_contiguous():
                raise ValueError("w_scales is strided")
        if mx_out:
            d.y_scales, d.y_scales_pitch = _rows(y_scales, "y_scales", dev, (d.n_rows, d.n_out // 32), torch.uint8)
        if expert_offset is not None:
            d.expert_offset, _ = _rows(expert_offset, "expert_offset", dev, (d.n_expert + 1,), torch.int32)
        if sorted_tok is not None:
            d.sorted_tok, _ = _rows(sorted_tok, "sorted_tok", dev, (d.n_rows,), torch.int32)
        self._finish(d, dev, x, w, y, expert_offset, sorted_tok, x_scales, w_scales, y_scales)


class Router(_Plan):
    """Which experts a token goes to: scores ("softmax" or "sigmoid" of logits [tokens, experts]), compared with bias
    [experts] f32 added, the keep_groups best of `groups` groups (by the sum of their group_top best, masked experts left
    out), the top_k best of those -> ids [tokens, top_k] i32 (-1 where none is left) and w [tokens, top_k] f32: the scores
    without the bias, divided by their sum (renorm), times scale. logits in f32, f16 or bf16.

    sorted_tok [tokens * top_k] and expert_offset [local experts + 1] i32 (both or neither): the pairs sorted over the experts
    from expert_base on, as GroupedMm reads them. A plan that sorts more than 2048 pairs has a work buffer: its runs come one
    after another, and one made under graph capture runs on the capturing stream, or on streams that wait for it."""
    _entry = "exl3b200_router"

    def __init__(self, *, logits, top_k, ids, w, score="softmax", bias=None, groups=1, keep_groups=1, group_top=1, renorm=False,
                 scale=1.0, sorted_tok=None, expert_offset=None, expert_base=0):
        d = RouterDesc()
        if logits.dim() != 2:
            raise ValueError(f"logits have {logits.dim()} dimensions, not 2")
        dev = logits.get_device()
        d.n_tok, d.n_expert = logits.shape
        d.top_k, d.score, d.renorm, d.scale = top_k, SCORES[score], renorm, scale
        d.n_group, d.group_keep, d.group_top = groups, keep_groups, group_top
        d.logits, d.logits_pitch = _rows(logits, "logits", dev)
        d.dtype = _dtype(logits)
        if bias is not None:
            d.bias, _ = _rows(bias, "bias", dev, (d.n_expert,), torch.float32)
        for name, t, kind in (("ids", ids, torch.int32), ("w", w, torch.float32)):
            p, _ = _rows(t, name, dev, (d.n_tok, top_k), kind)
            if not t.is_contiguous():
                raise ValueError(f"{name} is strided")
            setattr(d, name, p)
        work = None
        if sorted_tok is not None or expert_offset is not None:
            d.sorted_tok, _ = _rows(sorted_tok, "sorted_tok", dev, (d.n_tok * top_k,), torch.int32)
            d.expert_offset, _ = _rows(expert_offset, "expert_offset", dev, dtype=torch.int32)
            if expert_offset.dim() != 1 or expert_offset.shape[0] < 2:
                raise ValueError(f"expert_offset has shape {tuple(expert_offset.shape)}, not (local experts + 1,)")
            d.n_local, d.expert_base = expert_offset.shape[0] - 1, expert_base
            if d.n_tok * top_k > SORT_PAIRS:
                work = torch.empty(native().scatter_work_bytes(d.n_tok * top_k, d.n_local), dtype=torch.uint8, device=logits.device)
                d.work = work.data_ptr()
                # a run may come on any stream: whatever used the buffer's memory before is done by then. Under capture it is
                # the graph's own memory, in the capturing stream's order
                if not torch.cuda.is_current_stream_capturing():
                    torch.cuda.current_stream(dev).synchronize()
        self._finish(d, dev, logits, bias, ids, w, sorted_tok, expert_offset, work)


class BlockNorm(_Plan):
    """The norm behind a block with its gate and residual scale, and the norm before the next, in one pass:
    r = res_scale * res + g * rmsnorm(branch) * post_w -> out; rmsnorm(r) * pre_w -> y and / or (y_codes, y_scales).
    gate_kind: "none"; "token" (f32 logits [rows]) or "element" (logits [rows, cols]) through a sigmoid; "channel"
    ([cols], as it is). Every tensor but branch and a token gate shares one of f32, f16, bf16."""
    _entry = "exl3b200_block_norm"

    def __init__(self, *, branch=None, post_w=None, post_eps=1e-6, gate=None, gate_kind="none", res=None, res_scale=1.0,
                 out=None, pre_w=None, pre_eps=1e-6, y=None, y_codes=None, y_scales=None):
        d = BlockNormDesc()
        lead = branch if branch is not None else res
        if lead is None:
            raise ValueError("neither branch nor res")
        rows, cols = d.rows, d.cols = lead.shape
        dev = lead.get_device()
        typed = next((t for t in (res, out, y, post_w, pre_w) if t is not None), lead)
        dt = typed.dtype
        d.dtype, d.gate_kind = _dtype(typed), GATES[gate_kind]
        d.res_scale, d.post_eps, d.pre_eps = res_scale, post_eps, pre_eps
        if branch is not None:
            d.branch, d.branch_pitch = _rows(branch, "branch", dev, (rows, cols))
            d.branch_dtype = _dtype(branch)
        for name, t in (("res", res), ("out", out), ("y", y)):
            if t is not None:
                p, pitch = _rows(t, name, dev, (rows, cols), dt)
                setattr(d, name, p)
                setattr(d, name + "_pitch", pitch)
        for name, t in (("post_w", post_w), ("pre_w", pre_w)):
            if t is not None:
                setattr(d, name, _rows(t, name, dev, (cols,), dt)[0])
        if gate is not None:
            shape, want = {"token": ((rows,), torch.float32), "channel": ((cols,), dt),
                           "element": ((rows, cols), dt)}.get(gate_kind, (None, None))
            d.gate, d.gate_pitch = _rows(gate, "gate", dev, shape, want)
        if y_codes is not None:
            d.y_codes, d.y_codes_pitch = _rows(y_codes, "y_codes", dev, (rows, cols // 2), torch.uint8)
        if y_scales is not None:
            d.y_scales, d.y_scales_pitch = _rows(y_scales, "y_scales", dev, (rows, cols // 32), torch.uint8)
        self._finish(d, dev, branch, post_w, gate, res, out, pre_w, y, y_codes, y_scales)


# ------------------------------------------------------------------------------------------------ the block
class ExpertBlock:
    """A residual MoE block over such experts (exl3b200_expert_block_forward): norm, router, the experts' gate / up and down
    products, the gather, and the norm, gate and residual behind it, and the next block's norm.

    router_w [experts, hidden] in f16 or bf16 sets the stream's type, which pre_w, post_w, gate (a scale a channel) and
    next_w [hidden] share. gu_w [experts, 2 width, hidden] and dn_w [experts, hidden, width] are of that type, or uint8
    MXFP4 codes with gu_scales and dn_scales [experts, rows, cols / 32] (tiled here, once), or float8_e4m3fn with f32 gu_scales
    [experts, 2 ceil(width / 128), ceil(hidden / 128)] and dn_scales [experts, ceil(hidden / 128), ceil(width / 128)].

    router: None (softmax over all experts, the top_k), or a dict of Router's score, bias, groups, keep_groups, group_top,
    renorm and scale.

    A block has one work buffer: its forwards run one after another, on one stream or on streams that wait for each other,
    and it is kept until they are done."""

    def __init__(self, *, router_w, gu_w, dn_w, pre_w, post_w=None, gate=None, next_w=None, gu_scales=None, dn_scales=None,
                 top_k, eps=1e-6, res_scale=1.0, max_tokens=2048, router=None):
        E, H = router_w.shape
        dev = self._dev = router_w.get_device()
        mx, f8 = gu_w.dtype == torch.uint8, gu_w.dtype == torch.float8_e4m3fn
        per, dt = 2 if mx else 1, router_w.dtype
        W = dn_w.shape[2] * per
        d = self.desc = ExpertBlockDesc()
        d.n_expert, d.hidden, d.width, d.top_k, d.eps, d.res_scale = E, H, W, top_k, eps, res_scale
        d.dtype, d.weights = _dtype(router_w), MX4 if mx else F8 if f8 else _dtype(gu_w)
        want = torch.uint8 if mx else torch.float8_e4m3fn if f8 else dt
        keep = [router_w, gu_w, dn_w, pre_w, post_w, gate, next_w]
        for name, t, shape, kind in (("router_w", router_w, (E, H), dt), ("gu_w", gu_w, (E, 2 * W, H // per), want),
                                     ("dn_w", dn_w, (E, H, W // per), want), ("pre_w", pre_w, (H,), dt),
                                     ("post_w", post_w, (H,), dt), ("gate", gate, (H,), dt), ("next_w", next_w, (H,), dt)):
            if t is not None:
                if not t.is_contiguous():
                    raise ValueError(f"{name} is strided")
                setattr(d, name, _rows(t, name, dev, shape, kind)[0])
        if mx:
            _rows(gu_scales, "gu_scales", dev, (E, 2 * W, H // 32), torch.uint8)
            _rows(dn_scales, "dn_scales", dev, (E, H, W // 32), torch.uint8)
            keep += [mx4_tile_scales(gu_scales, "silu_mul"), mx4_tile_scales(dn_scales)]
            d.gu_scales, d.dn_scales = keep[-2].data_ptr(), keep[-1].data_ptr()
        if f8:
            h, w = (H + 127) // 128, (W + 127) // 128
            for name, t, shape in (("gu_scales", gu_scales, (E, 2 * w, h)), ("dn_scales", dn_scales, (E, h, w))):
                setattr(d, name, _rows(t, name, dev, shape, torch.float32)[0])
                if not t.is_contiguous():
                    raise ValueError(f"{name} is strided")
            keep += [gu_scales, dn_scales]
        self.router = None
        if router is not None:
            o = {**dict(score="softmax", bias=None, groups=1, keep_groups=1, group_top=1, renorm=False, scale=1.0), **router}
            if len(o) != 7:
                raise ValueError(f"router has {sorted(set(o))}")
            r = self.router = RouterDesc(score=SCORES[o["score"]], n_group=o["groups"], group_keep=o["keep_groups"],
                                         group_top=o["group_top"], renorm=o["renorm"], scale=o["scale"])
            if o["bias"] is not None:
                r.bias, _ = _rows(o["bias"], "bias", dev, (E,), torch.float32)
            keep.append(o["bias"])
        self._keep, self.dtype, self.hidden, self.max_tokens = keep, dt, H, max_tokens
        n = native().expert_block_work_bytes(d, max_tokens)
        self.work = torch.empty(n, dtype=torch.uint8, device=router_w.device)
        self.bufs = native().expert_block_carve(d, max_tokens, self.work.data_ptr(), n)
        # a forward may come on any stream: the tiling is done by then, and whatever used the work buffer's memory before
        torch.cuda.current_stream(dev).synchronize()

    def forward(self, x, out, next_out=None, stream=None):
        """x [T, hidden] through the block into out (which may be x); next_out: the next block's normed input."""
        T = x.shape[0]
        for name, t in (("x", x), ("out", out), ("next_out", next_out)):
            if t is not None:
                _rows(t, name, self._dev, (T, self.hidden), self.dtype)
                if not t.is_contiguous():
                    raise ValueError(f"{name} is strided")
        if _several:
            _check_current(self._dev)
        args = (self.bufs, x.data_ptr(), T, out.data_ptr(), next_out.data_ptr() if next_out is not None else None,
                _current_stream(self._dev) if stream is None else stream)
        if self.router is None:
            native().expert_block_forward(self.desc, *args)
        else:
            native().expert_block_forward_routed(self.desc, self.router, *args)
        return out
