/* exl3b200_dense.c -- the C host side of the dense and MXFP4 expert operators (include/exl3b200.h): the argument checks
 * and the kernels' argument records. Nothing is enqueued on a refusal. */
#include "exl3b200.h"
#include "exl3b200_dense.h"

#include <string.h>

/* exl3b200_norm.cu, exl3b200_gmm.cu, exl3b200_gmm8.cu, exl3b200_moe.cu */
int exl3b_cuda_block_norm(const Exl3bNormOp* p, int dtype, int branch_dtype, int vec, int sm_count,
                          void* stream);
int exl3b_cuda_mx4_quantize(const void* x, int dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* q,
                            int64_t q_pitch, uint8_t* qs, int64_t qs_pitch, void* stream);
int exl3b_cuda_mx4_dequantize(const uint8_t* q, int64_t q_pitch, const uint8_t* qs, int64_t qs_pitch, int64_t rows,
                              int64_t cols, void* y, int dtype, int64_t y_pitch, void* stream);
int exl3b_cuda_mx4_tile(const uint8_t* s, int64_t s_pitch, int64_t e_pitch, int64_t n_expert, int64_t rows, int64_t cols,
                        int act, int64_t n_blk, int64_t n_k, void* out, void* stream);
int exl3b_cuda_gmm(const Exl3bGmmOp* p, int sm_count, void* stream);
int exl3b_cuda_gmm8(const Exl3bGmmOp* p, int sm_count, void* stream);
int exl3b_gmm_max_expert(void);
/* exl3b200_route.cu, exl3b200_f8.cu */
int exl3b_route_fuses(int64_t n_tok, int64_t top_k, int64_t n_local);
int exl3b_cuda_route(const Exl3bRouteOp* p, int dtype, int fused, void* stream);
int exl3b_cuda_f8_quantize(const void* x, int dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* q,
                           int64_t q_pitch, float* s, int64_t s_pitch, int pow2, void* stream);
int exl3b_cuda_f8_dequantize(const uint8_t* q, int64_t q_pitch, const float* s, int64_t s_pitch, int64_t rows, int64_t cols,
                             void* y, int dtype, int64_t y_pitch, void* stream);
int exl3b_cuda_device_info(int* sm_count, int32_t** err_word);

/* Largest sizes taken: rows and columns that 32-bit coordinates hold, norm rows that a block holds in registers. */
static const int64_t kMaxDim = (int64_t)1 << 30;
static const int64_t kMaxNormCols = 32768;
/* A product's n_in: its byte offsets along k, and those of the scales' tiles (1 KB each 256 columns), stay in 32 bits, and
 * the stages of one unit's k (a million at 16 bits) inside the 2 s after which a wait for its sums gives up. */
static const int64_t kMaxIn = (int64_t)1 << 26;

static int is_float(int dt) { return dt == RAD_F32 || dt == RAD_F16 || dt == RAD_BF16; }
static int64_t size_of(int dt) { return dt == RAD_F32 ? 4 : 2; }
static int mis(const void* p, int64_t a) { return (int)((uintptr_t)p % (uintptr_t)a); }
static int rc_of(int rc) { return rc == 0 ? RAD_OK : RAD_E_DEVICE; }

int exl3b200_block_norm(const Exl3bBlockNorm* d, void* stream) {
    if (!d) return RAD_E_INVAL;
    if (d->rows < 0 || d->cols < 1 || d->rows > kMaxDim || d->cols > kMaxNormCols) return RAD_E_SHAPE;
    if (!is_float(d->dtype) || (d->branch && !is_float(d->branch_dtype))) return RAD_E_DTYPE;
    if (d->rows == 0) return RAD_OK;
    if (!d->branch && !d->res) return RAD_E_INVAL;
    if (!d->out && !d->y && !d->y_codes) return RAD_E_INVAL;
    if ((d->post_w || d->gate_kind != EXL3B_GATE_NONE) && !d->branch) return RAD_E_INVAL;
    if ((d->y || d->y_codes) && !d->pre_w) return RAD_E_INVAL;
    if (d->pre_w && !d->y && !d->y_codes) return RAD_E_INVAL;
    if (!d->y_codes != !d->y_scales) return RAD_E_INVAL;
    if (d->gate_kind < EXL3B_GATE_NONE || d->gate_kind > EXL3B_GATE_ELEMENT) return RAD_E_INVAL;
    if ((d->gate_kind != EXL3B_GATE_NONE) != (d->gate != 0)) return RAD_E_INVAL;
    if (!(d->post_eps >= 0.f) || !(d->pre_eps >= 0.f)) return RAD_E_INVAL;
    if ((d->branch && d->branch_pitch < d->cols) || (d->res && d->res_pitch < d->cols) ||
        (d->out && d->out_pitch < d->cols) || (d->y && d->y_pitch < d->cols) ||
        (d->gate_kind == EXL3B_GATE_ELEMENT && d->gate_pitch < d->cols))
        return RAD_E_STRIDE;
    const int64_t es = size_of(d->dtype), bs = size_of(d->branch_dtype);
    if (mis(d->branch, bs) || mis(d->res, es) || mis(d->out, es) || mis(d->y, es) || mis(d->post_w, es) ||
        mis(d->pre_w, es) || mis(d->gate, d->gate_kind == EXL3B_GATE_TOKEN ? 4 : es))
        return RAD_E_ALIGN;
    /* 16-byte vectors of eight values (f32: two) where every address and the width allow them */
    int vec = d->cols % 8 == 0 && !mis(d->branch, 16) && !mis(d->res, 16) && !mis(d->out, 16) && !mis(d->y, 16) &&
              !mis(d->post_w, 16) && !mis(d->pre_w, 16);
    vec = vec && (!d->branch || d->branch_pitch * bs % 16 == 0) && (!d->res || d->res_pitch * es % 16 == 0) &&
          (!d->out || d->out_pitch * es % 16 == 0) && (!d->y || d->y_pitch * es % 16 == 0);
    if (d->gate_kind == EXL3B_GATE_ELEMENT) vec = vec && !mis(d->gate, 16) && d->gate_pitch * es % 16 == 0;
    if (d->gate_kind == EXL3B_GATE_CHANNEL) vec = vec && !mis(d->gate, 16);
    if (d->y_codes) {
        if (d->cols % 32) return RAD_E_SHAPE;
        if (d->y_codes_pitch < d->cols / 2 || d->y_scales_pitch < d->cols / 32) return RAD_E_STRIDE;
        if (!vec || mis(d->y_codes, 4) || d->y_codes_pitch % 4) return RAD_E_ALIGN;
    }
    int sm = 0;
    int32_t* err = 0;
    if (exl3b_cuda_device_info(&sm, &err) != 0) return RAD_E_DEVICE;
    Exl3bNormOp p;
    memset(&p, 0, sizeof p);
    p.rows = d->rows;
    p.cols = d->cols;
    p.branch = d->branch;
    p.branch_pitch = d->branch_pitch;
    p.post_w = d->post_w;
    p.gate = d->gate;
    p.gate_pitch = d->gate_pitch;
    p.gate_kind = d->gate_kind;
    p.res = d->res;
    p.res_pitch = d->res_pitch;
    p.out = d->out;
    p.out_pitch = d->out_pitch;
    p.pre_w = d->pre_w;
    p.y = d->y;
    p.y_pitch = d->y_pitch;
    p.q = d->y_codes;
    p.q_pitch = d->y_codes_pitch;
    p.q_scales = d->y_scales;
    p.qs_pitch = d->y_scales_pitch;
    p.post_eps = d->post_eps;
    p.pre_eps = d->pre_eps;
    p.res_scale = d->res_scale;
    return rc_of(exl3b_cuda_block_norm(&p, d->dtype, d->branch ? d->branch_dtype : d->dtype, vec, sm, stream));
}

static int check_rows(int64_t rows, int64_t cols) {
    return rows < 0 || cols < 32 || cols % 32 || rows > kMaxDim || cols > kMaxDim ? RAD_E_SHAPE : RAD_OK;
}

int exl3b200_mx4_quantize(const void* x, int x_dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* codes,
                          int64_t codes_pitch, uint8_t* scales, int64_t scales_pitch, void* stream) {
    const int rc = check_rows(rows, cols);
    if (rc) return rc;
    if (!is_float(x_dtype)) return RAD_E_DTYPE;
    if (rows == 0) return RAD_OK;
    if (!x || !codes || !scales) return RAD_E_INVAL;
    if (x_pitch < cols || codes_pitch < cols / 2 || scales_pitch < cols / 32) return RAD_E_STRIDE;
    if (mis(x, 16) || x_pitch * size_of(x_dtype) % 16 || mis(codes, 4) || codes_pitch % 4) return RAD_E_ALIGN;
    return rc_of(exl3b_cuda_mx4_quantize(x, x_dtype, x_pitch, rows, cols, codes, codes_pitch, scales, scales_pitch,
                                         stream));
}

int exl3b200_mx4_dequantize(const uint8_t* codes, int64_t codes_pitch, const uint8_t* scales, int64_t scales_pitch,
                            int64_t rows, int64_t cols, void* y, int y_dtype, int64_t y_pitch, void* stream) {
    const int rc = check_rows(rows, cols);
    if (rc) return rc;
    if (!is_float(y_dtype)) return RAD_E_DTYPE;
    if (rows == 0) return RAD_OK;
    if (!y || !codes || !scales) return RAD_E_INVAL;
    if (y_pitch < cols || codes_pitch < cols / 2 || scales_pitch < cols / 32) return RAD_E_STRIDE;
    if (mis(y, 16) || y_pitch * size_of(y_dtype) % 16 || mis(codes, 4) || codes_pitch % 4) return RAD_E_ALIGN;
    return rc_of(exl3b_cuda_mx4_dequantize(codes, codes_pitch, scales, scales_pitch, rows, cols, y, y_dtype, y_pitch,
                                           stream));
}

/* FP8 rows: eight values a lane, 1024 lanes a block of the grid. */
static int check_f8(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 8 || cols % 8 || rows > kMaxDim || cols > kMaxDim) return RAD_E_SHAPE;
    return rows * ((cols + 127) / 128 * 16) > (int64_t)INT32_MAX * 1024 ? RAD_E_SHAPE : RAD_OK;
}

int exl3b200_f8_quantize(const void* x, int x_dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* codes,
                         int64_t codes_pitch, float* scales, int64_t scales_pitch, int pow2, void* stream) {
    const int rc = check_f8(rows, cols);
    if (rc) return rc;
    if (!is_float(x_dtype)) return RAD_E_DTYPE;
    if (rows == 0) return RAD_OK;
    if (!x || !codes || !scales) return RAD_E_INVAL;
    if (x_pitch < cols || codes_pitch < cols || scales_pitch < (cols + 127) / 128) return RAD_E_STRIDE;
    if (mis(x, 16) || x_pitch * size_of(x_dtype) % 16 || mis(codes, 8) || codes_pitch % 8 || mis(scales, 4))
        return RAD_E_ALIGN;
    return rc_of(exl3b_cuda_f8_quantize(x, x_dtype, x_pitch, rows, cols, codes, codes_pitch, scales, scales_pitch, pow2 != 0,
                                        stream));
}

int exl3b200_f8_dequantize(const uint8_t* codes, int64_t codes_pitch, const float* scales, int64_t scales_pitch,
                           int64_t rows, int64_t cols, void* y, int y_dtype, int64_t y_pitch, void* stream) {
    const int rc = check_f8(rows, cols);
    if (rc) return rc;
    if (!is_float(y_dtype)) return RAD_E_DTYPE;
    if (rows == 0) return RAD_OK;
    if (!y || !codes || !scales) return RAD_E_INVAL;
    if (y_pitch < cols || codes_pitch < cols || scales_pitch < (cols + 127) / 128) return RAD_E_STRIDE;
    if (mis(y, 16) || y_pitch * size_of(y_dtype) % 16 || mis(codes, 8) || codes_pitch % 8 || mis(scales, 4))
        return RAD_E_ALIGN;
    return rc_of(exl3b_cuda_f8_dequantize(codes, codes_pitch, scales, scales_pitch, rows, cols, y, y_dtype, y_pitch, stream));
}

/* How many neighbouring experts a lane holds; 2^*shift lanes a group: as many as a power of two of groups leaves each. */
static int64_t lane_experts(const Exl3bRouter* d, int* shift) {
    int s = 5;
    while ((int64_t)d->n_group << s > 32) --s;
    if (shift) *shift = s;
    return (d->n_expert / d->n_group + (1 << s) - 1) >> s;
}

int exl3b_router_check(const Exl3bRouter* d) {
    if (!d) return RAD_E_INVAL;
    if (!is_float(d->dtype)) return RAD_E_DTYPE;
    if ((d->score != EXL3B_SCORE_SOFTMAX && d->score != EXL3B_SCORE_SIGMOID) || !(d->scale - d->scale == 0.f)) return RAD_E_INVAL;
    const int64_t E = d->n_expert, G = d->n_group;
    if (d->n_tok < 0 || E < 1 || E > 2048 || d->top_k < 1 || d->top_k > 32 || d->n_tok > INT32_MAX / d->top_k || G < 1 ||
        G > 32 || E % G || d->group_keep < 1 || d->group_keep > G || d->group_top < 1 || d->group_top > 2 ||
        d->top_k > E / G * d->group_keep)
        return RAD_E_SHAPE;
    if (lane_experts(d, 0) > 64) return RAD_E_SHAPE;
    const int sort = d->expert_offset != 0;
    if (d->n_tok > 0 && sort != (d->sorted_tok != 0)) return RAD_E_INVAL;
    if (sort && (d->n_local < 1 || d->n_local > 16384)) return RAD_E_SHAPE;
    if (sort && d->n_tok * d->top_k > 2048 && !d->work) return RAD_E_INVAL;
    if (d->n_tok > 0 && (!d->logits || !d->ids || !d->w)) return RAD_E_INVAL;
    if (d->n_tok > 0 && d->logits_pitch < E) return RAD_E_STRIDE;
    if (mis(d->logits, size_of(d->dtype)) || mis(d->bias, 4) || mis(d->ids, 4) || mis(d->w, 4) || mis(d->sorted_tok, 4) ||
        mis(d->expert_offset, 4) || (sort && mis(d->work, 4)))
        return RAD_E_ALIGN;
    return RAD_OK;
}

int exl3b200_router(const Exl3bRouter* d, void* stream) {
    const int bad = exl3b_router_check(d);
    if (bad) return bad;
    const int64_t E = d->n_expert, G = d->n_group;
    const int sort = d->expert_offset != 0;
    if (d->n_tok > 0) {
        const int fused = sort && exl3b_route_fuses(d->n_tok, d->top_k, d->n_local);
        int shift = 0;
        const int64_t per = lane_experts(d, &shift);
        Exl3bRouteOp p;
        memset(&p, 0, sizeof p);
        p.n_tok = d->n_tok;
        p.logits = d->logits;
        p.logits_pitch = d->logits_pitch;
        p.bias = d->bias;
        p.score = d->score;
        p.top_k = (int32_t)d->top_k;
        p.renorm = d->renorm != 0;
        p.n_group = d->n_group;
        p.group_keep = d->group_keep;
        p.group_top = d->group_top;
        p.group_size = (int32_t)(E / G);
        p.group_shift = shift;
        p.lane_experts = (int32_t)per;
        const int64_t es = size_of(d->dtype);
        if (E / G % per == 0 && per * es % 16 == 0 && !mis(d->logits, 16) && d->logits_pitch * es % 16 == 0) p.vec |= 1;
        if (E / G % per == 0 && per % 4 == 0 && !mis(d->bias, 16)) p.vec |= 2;
        p.scale = d->scale;
        p.ids = d->ids;
        p.w = d->w;
        p.sorted_tok = d->sorted_tok;
        p.expert_offset = d->expert_offset;
        p.expert_base = d->expert_base;
        p.n_local = (int32_t)d->n_local;
        const int rc = exl3b_cuda_route(&p, d->dtype, fused, stream);
        if (rc || fused) return rc_of(rc);
    }
    if (!sort) return RAD_OK;
    if (d->n_tok == 0)                   /* no pairs: neither array is looked at */
        return exl3b200_moe_scatter(d->expert_offset, 0, d->n_local, 0, d->expert_offset, d->expert_offset, 0, stream);
    return exl3b200_moe_scatter(d->ids, d->n_tok * d->top_k, d->n_local, d->expert_base, d->sorted_tok, d->expert_offset,
                                d->work, stream);
}

/* Blocks of 128 weight rows (silu_mul: 64 gate + 64 up), padded to pairs; 128-column tiles, padded to pairs. */
static int64_t tile_blocks(int64_t rows, int act) {
    const int64_t b = act ? (rows / 2 + 63) / 64 : (rows + 127) / 128;
    return (b + 1) / 2 * 2;
}
static int64_t tile_cols(int64_t cols) { return (cols + 255) / 256 * 2; }

int64_t exl3b200_mx4_tiled_bytes(int64_t n_expert, int64_t rows, int64_t cols, int act) {
    if (n_expert < 1 || n_expert > exl3b_gmm_max_expert() || rows < 1 || check_rows(rows, cols) ||
        (act != EXL3B_ACT_NONE && act != EXL3B_ACT_SILU_MUL) || (act && rows % 2))
        return -1;
    return n_expert * tile_blocks(rows, act) * tile_cols(cols) * 512;
}

int exl3b200_mx4_tile_scales(const uint8_t* scales, int64_t scales_pitch, int64_t expert_pitch, int64_t n_expert,
                             int64_t rows, int64_t cols, int act, void* tiled, void* stream) {
    if (exl3b200_mx4_tiled_bytes(n_expert, rows, cols, act) < 0) return RAD_E_SHAPE;
    if (!scales || !tiled) return RAD_E_INVAL;
    if (scales_pitch < cols / 32 || (n_expert > 1 && expert_pitch < 0)) return RAD_E_STRIDE;
    if (mis(tiled, 16)) return RAD_E_ALIGN;
    return rc_of(exl3b_cuda_mx4_tile(scales, scales_pitch, expert_pitch, n_expert, rows, cols, act,
                                     tile_blocks(rows, act), tile_cols(cols), tiled, stream));
}

int exl3b200_grouped_mm(const Exl3bGroupedMm* d, void* stream) {
    if (!d) return RAD_E_INVAL;
    const int mx = d->dtype == EXL3B_MX4, f8 = d->dtype == EXL3B_F8, mx_out = d->y_dtype == EXL3B_MX4;
    if (!mx && !f8 && d->dtype != RAD_F16 && d->dtype != RAD_BF16) return RAD_E_DTYPE;
    if ((!mx_out || f8) && !is_float(d->y_dtype)) return RAD_E_DTYPE;
    if (d->act != EXL3B_ACT_NONE && d->act != EXL3B_ACT_SILU_MUL) return RAD_E_INVAL;
    if (d->n_expert < 1 || d->n_expert > exl3b_gmm_max_expert() || d->n_rows < 0 || d->n_rows > kMaxDim ||
        d->x_rows < 0 || d->x_rows > kMaxDim || d->top_k < 0 || d->top_k > 4096 || d->n_out < 8 || d->n_out % 8 ||
        d->n_out > kMaxDim / 2 || d->n_in < 8 || d->n_in > kMaxIn || d->n_in % (mx ? 32 : f8 ? 16 : 8) ||
        (mx_out && d->n_out % 32))
        return RAD_E_SHAPE;
    if (d->n_rows == 0) return RAD_OK;
    if (!d->x || !d->w || !d->y || ((mx || f8) && (!d->x_scales || !d->w_scales)) || (mx_out && !d->y_scales)) return RAD_E_INVAL;
    if (!d->expert_offset && d->n_expert != 1) return RAD_E_INVAL;
    if (d->x_rows < 1 || (d->top_k == 0 && d->x_rows < d->n_rows) ||
        (d->top_k > 0 && !d->sorted_tok && d->x_rows < (d->n_rows + d->top_k - 1) / d->top_k))
        return RAD_E_SHAPE;
    const int64_t w_rows = d->act ? 2 * d->n_out : d->n_out, kb = (d->n_in + 127) / 128;
    /* units are counted in 32 bits: a group each 32 rows and an expert, a block each 64 outputs */
    if ((d->n_rows / 32 + d->n_expert + 1) * (d->n_out / 64 + 1) > INT32_MAX) return RAD_E_SHAPE;
    if (d->x_pitch < d->n_in || d->w_pitch < d->n_in || (d->n_expert > 1 && d->w_expert_pitch < w_rows * d->w_pitch) ||
        d->y_pitch < d->n_out || (mx && d->x_scales_pitch < d->n_in / 32) ||
        (f8 && d->x_scales_pitch < kb * 4) || (mx_out && d->y_scales_pitch < d->n_out / 32))
        return RAD_E_STRIDE;
    /* TMA reads rows that start on 16-byte boundaries; stores are 16 bytes (MXFP4 codes: 4) */
    const int64_t xe = mx ? 32 : f8 ? 16 : 8, ye = mx_out ? 8 : 16 / size_of(d->y_dtype);
    if (mis(d->x, 16) || mis(d->w, 16) || d->x_pitch % xe || d->w_pitch % xe ||
        (d->n_expert > 1 && d->w_expert_pitch % xe) || mis(d->y, mx_out ? 4 : 16) || d->y_pitch % ye ||
        (mx && mis(d->w_scales, 16)) || (f8 && (mis(d->x_scales, 4) || d->x_scales_pitch % 4 || mis(d->w_scales, 4))) ||
        mis(d->sorted_tok, 4) || mis(d->expert_offset, 4))
        return RAD_E_ALIGN;
    int sm = 0;
    int32_t* err = 0;
    if (exl3b_cuda_device_info(&sm, &err) != 0) return RAD_E_DEVICE;
    Exl3bGmmOp p;
    memset(&p, 0, sizeof p);
    p.n_rows = d->n_rows;
    p.n_out = d->n_out;
    p.n_in = d->n_in;
    p.w_rows = w_rows;
    p.x_rows = d->x_rows;
    p.n_expert = (int32_t)d->n_expert;
    p.top_k = (int32_t)d->top_k;
    p.slots = exl3b_div(d->top_k > 1 ? (uint32_t)d->top_k : 1);
    p.act = d->act;
    p.y_dtype = d->y_dtype;
    p.x = d->x;
    const int64_t half_bytes = mx ? 1 : f8 ? 2 : 4;
    p.x_pitch_bytes = d->x_pitch * half_bytes / 2;
    p.w = d->w;
    p.w_pitch_bytes = d->w_pitch * half_bytes / 2;
    p.w_expert_bytes = d->n_expert > 1 ? d->w_expert_pitch * half_bytes / 2 : w_rows * p.w_pitch_bytes;
    p.sorted_tok = d->sorted_tok;
    p.expert_offset = d->expert_offset;
    p.y = d->y;
    p.y_pitch = mx_out ? d->y_pitch / 2 : d->y_pitch;
    p.y_scales = d->y_scales;
    p.ys_pitch = d->y_scales_pitch;
    p.x_scales = d->x_scales;
    p.xs_pitch = d->x_scales_pitch;
    p.w_scales = (const uint8_t*)d->w_scales;
    p.ws_blk_bytes = tile_cols(d->n_in) * 512;
    p.ws_expert_bytes = tile_blocks(w_rows, d->act) * p.ws_blk_bytes;
    if (f8) {
        p.ws_blocks = (int32_t)((d->n_out + 127) / 128);
        p.ws_blk_bytes = kb * 4;
        p.ws_expert_bytes = p.ws_blocks * (d->act ? 2 : 1) * p.ws_blk_bytes;
    }
    p.mx4 = mx;
    p.f8 = f8;
    p.bf16 = d->dtype == RAD_BF16;
    p.err = err;
    return rc_of(f8 ? exl3b_cuda_gmm8(&p, sm, stream) : exl3b_cuda_gmm(&p, sm, stream));
}
