/* exl3b200_expert_block.c -- a residual MoE block over experts that are not EXL3 records, driven from C: block_norm (with
 * MXFP4 output), the router's product, router_scatter, the experts' two grouped products, the gather, and block_norm again
 * into the residual stream. Nothing here allocates or synchronises: one caller block is sized and carved up front, and a
 * forward only enqueues. */
#include "exl3b200.h"

#include <string.h>

static int mis(const void* p, int64_t a) { return (int)((uintptr_t)p % (uintptr_t)a); }
static int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

static int check(const Exl3bExpertBlockDesc* d) {
    if (!d) return RAD_E_INVAL;
    const int mx = d->weights == EXL3B_MX4, step = mx ? 32 : 8;
    if (d->dtype != RAD_F16 && d->dtype != RAD_BF16) return RAD_E_DTYPE;
    if (!mx && d->weights != d->dtype) return RAD_E_DTYPE;
    if (d->n_expert < 8 || d->n_expert % 8 || d->n_expert > 2048 || d->top_k < 1 || d->top_k > 32 ||
        d->top_k > d->n_expert || d->hidden < step || d->hidden % step || d->hidden > 32768 || d->width < step ||
        d->width % step || d->width > 32768)
        return RAD_E_SHAPE;
    if (!d->router_w || !d->gu_w || !d->dn_w || !d->pre_w || (mx && (!d->gu_scales || !d->dn_scales))) return RAD_E_INVAL;
    return RAD_OK;
}

typedef struct Sizes {
    int64_t xn, xq, xs, logits, ids, sorted, offset, scatter, h, hs, rows, branch, gather;
} Sizes;

static Sizes sizes(const Exl3bExpertBlockDesc* d, int64_t T) {
    const int64_t H = d->hidden, W = d->width, P = T * d->top_k, mx = d->weights == EXL3B_MX4;
    Sizes s;
    s.xn = up256(T * H * 2);
    s.xq = mx ? up256(T * H / 2) : 0;
    s.xs = mx ? up256(T * ((H / 32 + 15) / 16 * 16)) : 0;
    s.logits = up256(T * d->n_expert * 4);
    s.ids = up256(P * 4);
    s.sorted = up256(P * 4);
    s.offset = up256((d->n_expert + 1) * 4);
    s.scatter = up256(exl3b200_moe_scatter_work_bytes(P, d->n_expert));
    s.h = up256(mx ? P * W / 2 : P * W * 2);
    s.hs = mx ? up256(P * ((W / 32 + 15) / 16 * 16)) : 0;
    s.rows = up256(P * H * 2);
    s.branch = up256(T * H * 4);
    s.gather = up256(exl3b200_moe_gather_work_bytes(T, d->top_k));
    return s;
}

/* Tokens a pass at most: the pair count and every buffer's size stay far inside 64 bits and the routing's 32. */
static int tokens_ok(const Exl3bExpertBlockDesc* d, int64_t T) { return T >= 1 && T <= (int64_t)(1 << 24) / d->top_k; }

int64_t exl3b200_expert_block_work_bytes(const Exl3bExpertBlockDesc* d, int64_t max_tokens) {
    if (check(d) != RAD_OK || !tokens_ok(d, max_tokens)) return -1;
    const Sizes s = sizes(d, max_tokens);
    return s.xn + s.xq + s.xs + s.logits + 2 * s.ids + s.sorted + s.offset + s.scatter + s.h + s.hs + s.rows + s.branch +
           s.gather + 256;
}

int exl3b200_expert_block_carve(const Exl3bExpertBlockDesc* d, int64_t max_tokens, void* work, int64_t work_bytes,
                                Exl3bExpertBlockBufs* b) {
    if (!b || !work) return RAD_E_INVAL;
    const int64_t need = exl3b200_expert_block_work_bytes(d, max_tokens);
    if (need < 0) return RAD_E_INVAL;
    if (work_bytes < need) return RAD_E_SCRATCH;
    const Sizes s = sizes(d, max_tokens);
    uint8_t* p = (uint8_t*)(((uintptr_t)work + 255) / 256 * 256);
    memset(b, 0, sizeof *b);
    b->max_tokens = max_tokens;
    b->xn = p;                       p += s.xn;
    b->x_codes = s.xq ? p : 0;       p += s.xq;
    b->x_scales = s.xs ? p : 0;      p += s.xs;
    b->logits = (float*)p;           p += s.logits;
    b->ids = (int32_t*)p;            p += s.ids;
    b->w = (float*)p;                p += s.ids;
    b->sorted_tok = (int32_t*)p;     p += s.sorted;
    b->expert_offset = (int32_t*)p;  p += s.offset;
    b->scatter_work = p;             p += s.scatter;
    b->h = p;                        p += s.h;
    b->h_scales = s.hs ? p : 0;      p += s.hs;
    b->y_rows = (uint16_t*)p;        p += s.rows;
    b->branch = (float*)p;           p += s.branch;
    b->gather_work = p;
    return RAD_OK;
}

int exl3b200_expert_block_forward(const Exl3bExpertBlockDesc* d, const Exl3bExpertBlockBufs* b, const void* x, int64_t T,
                                  void* out, void* next, void* stream) {
    int rc = check(d);
    if (rc != RAD_OK) return rc;
    if (!b || T < 0 || T > b->max_tokens) return RAD_E_INVAL;
    if (T == 0) return RAD_OK;
    if (!x || !out || (next && !d->next_w)) return RAD_E_INVAL;
    const int mx = d->weights == EXL3B_MX4;
    /* what the later steps would refuse is refused before the first is enqueued */
    if (mis(out, 2) || mis(next, 2) || mis(d->post_w, 2) || mis(d->gate, 2) || mis(d->next_w, 2) || mis(d->router_w, 16) ||
        mis(d->gu_w, 16) || mis(d->dn_w, 16) || (mx && (mis(d->gu_scales, 16) || mis(d->dn_scales, 16))))
        return RAD_E_ALIGN;
    const int64_t H = d->hidden, W = d->width, P = T * d->top_k;
    const int64_t xs_pitch = (H / 32 + 15) / 16 * 16, hs_pitch = (W / 32 + 15) / 16 * 16;

    /* the block's input, normed (and in MXFP4 for its experts) */
    Exl3bBlockNorm n;
    memset(&n, 0, sizeof n);
    n.rows = T;
    n.cols = H;
    n.dtype = d->dtype;
    n.res_scale = 1.f;
    n.res = x;
    n.res_pitch = H;
    n.pre_w = d->pre_w;
    n.pre_eps = d->eps;
    n.y = b->xn;
    n.y_pitch = H;
    if (mx) {
        n.y_codes = b->x_codes;
        n.y_codes_pitch = H / 2;
        n.y_scales = b->x_scales;
        n.y_scales_pitch = xs_pitch;
    }
    if ((rc = exl3b200_block_norm(&n, stream)) != RAD_OK) return rc;

    /* the router: one group, f32 logits */
    Exl3bGroupedMm m;
    memset(&m, 0, sizeof m);
    m.n_expert = 1;
    m.n_rows = m.x_rows = T;
    m.n_out = d->n_expert;
    m.n_in = H;
    m.dtype = d->dtype;
    m.y_dtype = RAD_F32;
    m.x = b->xn;
    m.x_pitch = m.w_pitch = H;
    m.w = d->router_w;
    m.y = b->logits;
    m.y_pitch = d->n_expert;
    if ((rc = exl3b200_grouped_mm(&m, stream)) != RAD_OK) return rc;
    rc = exl3b200_router_scatter(b->logits, T, d->n_expert, d->top_k, b->ids, b->w, d->n_expert, 0, b->sorted_tok,
                                 b->expert_offset, b->scatter_work, stream);
    if (rc != RAD_OK) return rc;

    /* gate and up, then down, over the sorted rows */
    memset(&m, 0, sizeof m);
    m.n_expert = d->n_expert;
    m.n_rows = P;
    m.n_out = W;
    m.n_in = H;
    m.x_rows = T;
    m.top_k = d->top_k;
    m.dtype = d->weights;
    m.y_dtype = d->weights;
    m.act = EXL3B_ACT_SILU_MUL;
    m.x = mx ? (const void*)b->x_codes : b->xn;
    m.x_pitch = m.w_pitch = H;
    m.x_scales = b->x_scales;
    m.x_scales_pitch = xs_pitch;
    m.w = d->gu_w;
    m.w_expert_pitch = 2 * W * H;
    m.w_scales = d->gu_scales;
    m.sorted_tok = b->sorted_tok;
    m.expert_offset = b->expert_offset;
    m.y = b->h;
    m.y_pitch = W;
    m.y_scales = b->h_scales;
    m.y_scales_pitch = hs_pitch;
    if ((rc = exl3b200_grouped_mm(&m, stream)) != RAD_OK) return rc;
    m.n_out = H;
    m.n_in = W;
    m.x_rows = P;
    m.top_k = 0;
    m.y_dtype = RAD_BF16;             /* what moe_gather reads, an f16 block's rows too: f16's range and more, three bits less */
    m.act = EXL3B_ACT_NONE;
    m.x = b->h;
    m.x_pitch = m.w_pitch = W;
    m.x_scales = b->h_scales;
    m.x_scales_pitch = hs_pitch;
    m.w = d->dn_w;
    m.w_expert_pitch = H * W;
    m.w_scales = d->dn_scales;
    m.y = b->y_rows;
    m.y_pitch = H;
    m.y_scales = 0;
    m.y_scales_pitch = 0;
    if ((rc = exl3b200_grouped_mm(&m, stream)) != RAD_OK) return rc;
    rc = exl3b200_moe_gather(b->y_rows, H, b->sorted_tok, P, b->w, T, d->top_k, H, b->branch, b->gather_work, stream);
    if (rc != RAD_OK) return rc;

    /* behind the block: norm, gate, residual; and the next block's norm */
    memset(&n, 0, sizeof n);
    n.rows = T;
    n.cols = H;
    n.dtype = d->dtype;
    n.branch = b->branch;
    n.branch_pitch = H;
    n.branch_dtype = RAD_F32;
    n.post_w = d->post_w;
    n.post_eps = n.pre_eps = d->eps;
    n.gate = d->gate;
    n.gate_kind = d->gate ? EXL3B_GATE_CHANNEL : EXL3B_GATE_NONE;
    n.res = x;
    n.res_pitch = H;
    n.res_scale = d->res_scale;
    n.out = out;
    n.out_pitch = H;
    if (next) {
        n.pre_w = d->next_w;
        n.y = next;
        n.y_pitch = H;
    }
    return exl3b200_block_norm(&n, stream);
}
