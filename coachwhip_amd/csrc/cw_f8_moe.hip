// A MoE layer of experts in 8-bit floats on 8-bit rows (gfx950).
#include <algorithm>

#include "cw_f8.h"
#include "cw_piles.h"

namespace cw {

struct F8MoeLayout {
    size_t ids, w, order, place, offsets, tiles, sort, g, u, hq, hs, dn, total;
};

static F8MoeLayout layout(const cw_f8_moe_desc *d, int T) {
    F8MoeLayout L = {};
    size_t off = 0;
    auto take = [&](size_t &at, size_t bytes) { at = off; off = (off + bytes + 255) & ~(size_t)255; };
    const size_t TK = (size_t)T * d->top_k;
    take(L.ids, TK * 4);
    take(L.w, TK * 4);
    take(L.order, TK * 4);
    take(L.place, TK * 4);
    take(L.offsets, (size_t)(d->n_experts + 1) * 4);
    take(L.tiles, (size_t)pile_tiles_bytes(TK, d->n_experts));
    take(L.sort, cw_sort_picks_workspace_size(TK, d->n_experts));
    take(L.g, TK * (size_t)d->inter * 4);
    take(L.u, TK * (size_t)d->inter * 4);
    take(L.hq, TK * f8_row_bytes(d->inter));
    take(L.hs, TK * f8_blocks(d->inter) * 4);
    take(L.dn, TK * (size_t)d->hidden * 4);
    L.total = off;
    return L;
}

static int check_desc(const cw_f8_moe_desc *d, int T) {
    CW_REQUIRE(d != nullptr, "f8 moe: null descriptor");
    CW_REQUIRE(T >= 0, "f8 moe: negative token count %d", T);
    CW_REQUIRE(d->n_experts > 0 && d->n_experts <= PILE_MAX_EXPERTS, "f8 moe: %d experts (1..%d supported)", d->n_experts, PILE_MAX_EXPERTS);
    CW_REQUIRE(d->top_k > 0 && d->top_k <= 32 && d->top_k <= d->n_experts, "f8 moe: top_k %d for %d experts", d->top_k, d->n_experts);
    CW_REQUIRE(d->hidden > 0 && d->inter > 0, "f8 moe: hidden %d, inter %d", d->hidden, d->inter);
    if (d->hidden > CW_F8_MAX_K || d->inter > CW_F8_MAX_K)
        return set_error(CW_ENOTSUP, "f8 moe: hidden %d, inter %d above %d", d->hidden, d->inter, CW_F8_MAX_K);
    CW_REQUIRE(d->act == CW_ACT_SILU || d->act == CW_ACT_CLAMPED_SWIGLU, "f8 moe: unknown activation %d", d->act);
    // (a launch holds fewer than 2^32 threads)
    const int64_t TK = (int64_t)T * d->top_k, blocks = pile_max_tiles(TK, d->n_experts) * f8_blocks(std::max(d->inter, d->hidden));
    if (TK >= 1 << 28 || blocks >= 1 << 23 || TK * f8_blocks(d->inter) >= 1 << 27)
        return set_error(CW_ENOTSUP, "f8 moe: %d tokens of %d picks, hidden %d, inter %d", T, d->top_k, d->hidden, d->inter);
    for (int m = 0; m < 3; m++) {
        const int64_t need = (m == 2 ? d->hidden : d->inter) * f8_row_bytes(m == 2 ? d->inter : d->hidden);
        CW_REQUIRE(d->w[m] && d->scale[m], "f8 moe: matrix %d is null", m);
        CW_REQUIRE(f8_aligned(d->w[m], 16) && d->slot_stride[m] % 16 == 0, "f8 moe: matrix %d must be 16-byte aligned", m);
        CW_REQUIRE(d->slot_stride[m] >= need, "f8 moe: matrix %d slot stride %lld below its %lld bytes", m, (long long)d->slot_stride[m],
                   (long long)need);
    }
    return CW_OK;
}

}  // namespace cw

using namespace cw;

extern "C" {

size_t cw_f8_moe_workspace_size(const cw_f8_moe_desc *d, int T) {
    if (check_desc(d, T) != CW_OK || T == 0) return 0;
    return layout(d, T).total;
}

int cw_f8_moe_layer(const cw_f8_moe_desc *d, const uint8_t *x, const float *x_scale, const float *logits, int T, int ydtype, void *out,
                    uint32_t *ids_out, float *w_out, void *ws, size_t ws_bytes, cw_stream_t stream) {
    if (int rc = check_desc(d, T)) return rc;
    if (!f8_float_type(ydtype)) return set_error(CW_ENOTSUP, "f8 moe: type %d of out (f32, f16 or bf16)", ydtype);
    if (T == 0) return CW_OK;
    CW_REQUIRE(x && x_scale && logits && out, "f8 moe: null x, scales, logits or out");
    CW_REQUIRE(f8_aligned(x, 16), "f8 moe: codes must be 16-byte aligned");
    const F8MoeLayout L = layout(d, T);
    CW_REQUIRE(ws && ws_bytes >= L.total, "f8 moe: workspace of %zu bytes, %zu needed", ws_bytes, L.total);
    CW_REQUIRE(f8_aligned(ws, 256), "f8 moe: workspace must be 256-byte aligned");
    uint8_t *base = (uint8_t *)ws;
    const int E = d->n_experts, K = d->top_k, H = d->hidden, I = d->inter;
    const int64_t TK = (int64_t)T * K;
    uint32_t *ids = ids_out ? ids_out : (uint32_t *)(base + L.ids);
    float *w = w_out ? w_out : (float *)(base + L.w), *g = (float *)(base + L.g), *u = (float *)(base + L.u), *hs = (float *)(base + L.hs),
          *dn = (float *)(base + L.dn);
    int32_t *order = (int32_t *)(base + L.order), *place = (int32_t *)(base + L.place), *offsets = (int32_t *)(base + L.offsets);
    void *tiles = base + L.tiles;
    uint8_t *hq = base + L.hq;
    if (int rc = cw_route_topk(logits, T, E, K, d->norm, ids, w, stream)) return rc;
    if (int rc = cw_sort_picks(ids, TK, E, order, place, offsets, tiles, base + L.sort, cw_sort_picks_workspace_size(TK, E), stream)) return rc;
    float *gu[2] = {g, u};
    for (int m = 0; m < 2; m++)
        if (int rc = cw_f8_matmul_experts(d->w[m], d->slot_stride[m], d->scale[m], E, I, H, x, x_scale, T, order, K, TK, tiles, d->bias[m], CW_F32,
                                          gu[m], I, stream))
            return rc;
    if (int rc = cw_swiglu_f8(CW_F32, g, u, I, TK, I, d->act, d->alpha, d->limit, hq, hs, stream)) return rc;
    if (int rc = cw_f8_matmul_experts(d->w[2], d->slot_stride[2], d->scale[2], E, H, I, hq, hs, TK, nullptr, K, TK, tiles, d->bias[2], CW_F32, dn, H,
                                      stream))
        return rc;
    return from_piles_f32(ydtype, dn, w, T, K, E, H, place, offsets, out, (hipStream_t)stream);
}

}  // extern "C"
