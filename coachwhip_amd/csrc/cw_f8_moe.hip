// A MoE layer of experts in 8-bit floats on 8-bit rows (gfx950).
#include <algorithm>

#include "cw_f8_tile.h"

namespace cw {

struct F8GateUpArgs {
    const uint8_t *w[2], *x;
    const float *ws[2], *bias[2], *xs;
    int64_t stride[2], m, picks;  // bytes from an expert's matrix to the next; rows of x; positions
    int E, K, I, rb, blocks;      // of a row of x
    Glu glu;
    const void *tiles;
    const int *order;
    uint8_t *hq;  // rows of ceil(I / 128) * 128 codes, and their scales
    float *hs;
};

// Gate and up of a tile of up to 128 positions, 128 columns of both, and their activation as codes: a block holds whole groups of 128 columns of
// its rows, so that the hidden rows leave it as codes and nothing else is written (f32 hidden rows of 2,048 tokens of 4 picks of 2,880 columns: 94 MB
// written and read again). A wave has 32 columns: the largest magnitude of a row's 128 meets in LDS, as do the codes, which leave as whole rows of 128.
template <bool EXACT>
__global__ __launch_bounds__(256, 2) void k_f8_gateup(F8GateUpArgs a, int n_blocks) {
    extern __shared__ __align__(1024) uint8_t lds[];
    constexpr int ROW = 144;  // bytes of a row of codes in LDS (128 and a shift of the banks)
    PileTile tl;
    int nb;
    if (!f8_item_of_block(a.tiles, n_blocks, tl, nb) || tl.expert >= a.E) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = 128 * nb + 32 * wave, n_in = min(n0, a.I - 1);
    F8Operands<2> o;
    o.x = a.x;
    o.xs = a.xs;
    o.m = a.m;
    o.rb = a.rb;
    o.blocks = a.blocks;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        o.w0[i] = a.w[i] + tl.expert * a.stride[i] + (int64_t)n_in * a.rb;
        o.ws0[i] = a.ws[i] + ((int64_t)tl.expert * n_blocks + nb) * a.blocks;
    }
    uint32_t wrow[4];
#pragma unroll
    for (int j = 0; j < 4; j++) wrow[j] = (uint32_t)min(16 * (j & 1) + (lane & 15), a.I - 1 - n_in) * (uint32_t)a.rb + 16 * (lane >> 4);
    f8_by_height(tl.m, [&](auto mb_) __attribute__((always_inline)) {
        constexpr int MB = decltype(mb_)::value;
        f32x4 acc[MB][4];
        auto row_at = [&](int r) __attribute__((always_inline)) { return (int64_t)(a.order[tl.pos0 + min(r, tl.m - 1)] / a.K); };
        const bool odd = f8_stream<MB, 4, 2, EXACT>(lds, o, row_at, wrow, acc);
        const int col = n0 + 4 * (lane >> 4);
        if (__syncthreads_or(odd)) {
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int n = col + 16 * (j & 1);
                    if (n >= a.I) continue;
                    const int64_t row = row_at(16 * mb + (lane & 15));
                    acc[mb][j] = f8_strange_sums(a.x + row * a.rb, a.xs + row, a.m, a.w[j >> 1] + tl.expert * a.stride[j >> 1] + (int64_t)n * a.rb,
                                                 o.ws0[j >> 1], a.rb, min(a.I - n, 4), acc[mb][j]);
                }
        }
        float b[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                b[j][c] = a.bias[j >> 1] ? a.bias[j >> 1][(int64_t)tl.expert * a.I + min(col + 16 * (j & 1) + c, a.I - 1)] : 0.f;
        uint32_t *top = (uint32_t *)(lds + 16 * MB * ROW);  // of each wave
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float h = glu(acc[mb][j][c] + b[j][c], acc[mb][2 + j][c] + b[2 + j][c], a.glu);
                    acc[mb][j][c] = col + 16 * j + c < a.I ? h : 0.f;
                    bits = max_bits(bits, acc[mb][j][c]);
                }
            bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16));
            bits = max(bits, (uint32_t)__shfl_xor((int)bits, 32));
            if (lane < 16) top[wave * 16 * MB + 16 * mb + lane] = bits;
        }
        __syncthreads();
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            const int r = 16 * mb + (lane & 15);
            const F8Group g(max(max(top[r], top[16 * MB + r]), max(top[32 * MB + r], top[48 * MB + r])));
#pragma unroll
            for (int j = 0; j < 2; j++)
                *(uint32_t *)(lds + r * ROW + 32 * wave + 16 * j + 4 * (lane >> 4)) =
                    f8_codes4(g.quotient(acc[mb][j][0]), g.quotient(acc[mb][j][1]), g.quotient(acc[mb][j][2]), g.quotient(acc[mb][j][3]));
            if (wave == 0 && lane < 16 && r < tl.m) a.hs[nb * a.picks + tl.pos0 + r] = g.scale;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * tl.m; i += 256)
            *(i32x4 *)(a.hq + (int64_t)(tl.pos0 + (i >> 3)) * (n_blocks * F8_BLOCK) + nb * F8_BLOCK + 16 * (i & 7)) =
                *(const i32x4 *)(lds + (i >> 3) * ROW + 16 * (i & 7));
    });
}

struct F8MoeLayout {
    size_t ids, w, order, place, offsets, tiles, sort, hq, hs, dn, total;
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
    float *w = w_out ? w_out : (float *)(base + L.w), *hs = (float *)(base + L.hs),
          *dn = (float *)(base + L.dn);
    int32_t *order = (int32_t *)(base + L.order), *place = (int32_t *)(base + L.place), *offsets = (int32_t *)(base + L.offsets);
    void *tiles = base + L.tiles;
    uint8_t *hq = base + L.hq;
    if (int rc = cw_route_topk(logits, T, E, K, d->norm, ids, w, stream)) return rc;
    if (int rc = cw_sort_picks(ids, TK, E, order, place, offsets, tiles, base + L.sort, cw_sort_picks_workspace_size(TK, E), stream)) return rc;
    hipStream_t s = (hipStream_t)stream;
    F8GateUpArgs a = {};
    for (int m = 0; m < 2; m++) {
        a.w[m] = d->w[m];
        a.ws[m] = d->scale[m];
        a.bias[m] = d->bias[m];
        a.stride[m] = d->slot_stride[m];
    }
    a.x = x;
    a.xs = x_scale;
    a.m = T;
    a.picks = TK;
    a.E = E;
    a.K = K;
    a.I = I;
    a.rb = (int)f8_row_bytes(H);
    a.blocks = (int)f8_blocks(H);
    a.glu = glu_of(d->act, d->alpha, d->limit);
    a.tiles = tiles;
    a.order = order;
    a.hq = hq;
    a.hs = hs;
    // bf16's rounding covers what the 8-bit instruction leaves out of gate and up (hidden codes that take their neighbour: 1.1e-3 of a result,
    // beside 1.7e-3); results in f16 and f32 have hidden codes from exact products, those in f32 exact products in down too
    const int blocks = (int)f8_blocks(I);
    const dim3 grid((unsigned)((pile_max_tiles(TK, E) * blocks + 7) / 8 * 8));
    constexpr int LDS = F8Stream<8, 4>::LDS;
    if (ydtype == CW_BF16) hipLaunchKernelGGL(k_f8_gateup<false>, grid, dim3(256), LDS, s, a, blocks);
    else hipLaunchKernelGGL(k_f8_gateup<true>, grid, dim3(256), LDS, s, a, blocks);
    if (int rc = check_launch("k_f8_gateup")) return rc;
    if (int rc = f8_matmul_experts(d->w[2], d->slot_stride[2], d->scale[2], E, H, I, hq, hs, TK, nullptr, K, TK, tiles, d->bias[2], CW_F32, dn, H,
                                   ydtype == CW_F32, s))
        return rc;
    return from_piles_f32(ydtype, dn, w, T, K, E, H, place, offsets, out, s);
}

}  // extern "C"
