// A MoE layer of experts in 8-bit floats on 8-bit rows (gfx950).
#include <algorithm>

#include "cw_f8_tile.h"
#include "cw_f8_rules.h"
#include "cw_i8_rules.h"
#include "cw_mfma.h"

namespace cw {

// ------------------------------------------------------------------------------ a few tokens

struct F8FewArgs {
    const uint8_t *w[3], *x;
    const float *ws[3], *bias[3], *xs, *logits;
    int64_t stride[3];
    int E, K, H, I, T, norm;
    Glu glu;
    int rbh, rbi, ldh;  // bytes of a row of H and of I codes, floats of a hidden row
    uint32_t *ids;
    float *wt, *h;
    void *out;
};

// Gate and up of one pick of a token, 16 columns a block: 16 rows of either matrix against the token's row (in all 16 columns of the
// instruction: its sums cost nothing here, unpacking the codes for the vector unit 1.3 times the bytes' time), the steps of 128
// codes dealt to eight waves, even ones gate, odd ones up, their sums joined in LDS in the waves' order. One wave routes the token for its block, no
// further than this pick; the last pick's first block, which goes all the way, stores the routing. One token of 8 picks of 512 x 2,048: 7.1 us for 16.8 MB, a
// chain of logits, routing, weights, sums; 4 tokens of 4 picks of 2,880 x 2,880, with down: 88 to 96 us, 4.1 to 4.6 TB/s.
template <int PER, int NS, bool EXACT>
__global__ __launch_bounds__(64 * F8_FEW_WAVES, NS > 4 ? 2 : 4) void k_f8_few_gateup(F8FewArgs a) {
    __shared__ uint32_t expert;
    __shared__ float part[F8_FEW_WAVES][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.z, j = blockIdx.y;
    const int n0 = blockIdx.x * 16, blocks = a.rbh / F8_BLOCK, m = wave & 1, at = 16 * (lane >> 4);
    if (wave == 0) {
        uint32_t id;
        float wt;
        wave_route<PER>(a.logits + (int64_t)t * a.E, a.E, j + 1, a.norm, &id, &wt);
        if (blockIdx.x == 0 && j == a.K - 1 && lane < a.K) {
            a.ids[(int64_t)t * a.K + lane] = id;
            a.wt[(int64_t)t * a.K + lane] = wt;
        }
        if (lane == j) expert = id;
    }
    F8Frag<EXACT> x[NS], w[NS];
    float s[NS];
    auto step_of = [&](int i) __attribute__((always_inline)) { return (wave >> 1) + F8_FEW_WAVES / 2 * i; };
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const int step = min(step_of(i), blocks - 1);
        const uint8_t *p = a.x + (int64_t)t * a.rbh + step * F8_BLOCK + at;
        x[i].load(p, p + 64);
        s[i] = a.xs[(int64_t)step * a.T + t];
    }
    __syncthreads();
    const int64_t e = __builtin_amdgcn_readfirstlane((int)expert);
    const uint8_t *row = a.w[m] + e * a.stride[m] + (int64_t)min(n0 + (lane & 15), a.I - 1) * a.rbh + at;
    const float *ws = a.ws[m] + (e * ((a.I + 127) / 128) + n0 / F8_BLOCK) * blocks;
    bool strange = false;
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const int step = min(step_of(i), blocks - 1);
        const uint8_t *p = row + step * F8_BLOCK;
        w[i].load(p, p + 64);
        const float sw = ws[step];
        strange |= f8_strange(s[i]) | f8_strange(sw);
        s[i] = step_of(i) < blocks ? s[i] * sw : 0.f;  // (past the end the last step again, times nothing)
    }
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const f32x4 p = F8Frag<EXACT>::product(w[i], x[i]);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = fmaf(p[c], s[i], acc[c]);
    }
    if ((lane & 15) == 0) *(f32x4 *)&part[wave][4 * (lane >> 4)] = acc;
    strange = __syncthreads_or(strange);
    if (threadIdx.x >= 16 || n0 + threadIdx.x >= a.I) return;
    const int n = n0 + threadIdx.x;
    float v[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v[i] = part[i][threadIdx.x];
#pragma unroll
        for (int q = 2; q < F8_FEW_WAVES; q += 2) v[i] += part[q + i][threadIdx.x];
        if (strange) {
            f32x4 sum = {v[i], 0.f, 0.f, 0.f};
            f8_strange_sums(a.x + (int64_t)t * a.rbh, a.xs + t, a.T, a.w[i] + e * a.stride[i] + (int64_t)n * a.rbh,
                            a.ws[i] + (e * ((a.I + 127) / 128) + n0 / F8_BLOCK) * blocks, a.rbh, 1, sum);
            v[i] = sum[0];
        }
        if (a.bias[i]) v[i] += a.bias[i][e * a.I + n];
    }
    a.h[((int64_t)t * a.K + j) * a.ldh + n] = glu(v[0], v[1], a.glu);
}

// Down and the weighted sum of a token, 16 outputs a block: the block makes the token's K hidden rows codes in LDS (every block of the token does,
// one, two, four or eight waves a row; 32 lanes hold a group of 128 columns), then its waves take the steps of the K rows end to end in turn. The hidden
// rows are asked for before the weights: loads return in order, and the codes are made while the weights come in. One token of 8 picks of 512 x 2,048: 5.7
// us for 8.4 MB, a chain of the hidden rows, their codes, the sums.
template <class T, int NS, bool EXACT>
__global__ __launch_bounds__(64 * F8_FEW_WAVES, NS > 4 ? 2 : 4) void k_f8_few_down(F8FewArgs a) {
    constexpr int NH = NS < 12 ? (NS + 1) / 2 : 6;  // pieces of a hidden row held in registers (the others are read later)
    extern __shared__ __align__(16) uint8_t hq[];  // K rows of rbi codes, then their scales
    __shared__ float wk[32], part[F8_FEW_WAVES][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.y, blocks = a.rbi / F8_BLOCK, steps = a.K * blocks;
    float *hs = (float *)(hq + a.K * a.rbi);
    const int n0 = blockIdx.x * 16, at = 16 * (lane >> 4);
    const int wpp = a.K > 4 ? 1 : a.K > 2 ? 2 : a.K > 1 ? 4 : 8, at0 = 4 * ((wave & (wpp - 1)) * 64 + lane), stride = 256 * wpp;
    const float *h = a.h + (int64_t)t * a.K * a.ldh;
    float hv[NH][4];
    auto fetch_h = [&](int j) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NH; i++) load_row<4>(h + (int64_t)j * a.ldh + at0 + i * stride, a.I - at0 - i * stride, hv[i]);
    };
    fetch_h(min(wave / wpp, a.K - 1));
    const uint32_t *ids = a.ids + (int64_t)t * a.K;
    const float *wt = a.wt + (int64_t)t * a.K;
    auto step_of = [&](int i) __attribute__((always_inline)) { return min(wave + F8_FEW_WAVES * i, steps - 1); };
    auto matrix_of = [&](int pick) __attribute__((always_inline)) { return a.w[2] + (int64_t)ids[pick] * a.stride[2]; };
    auto scales_of = [&](int pick) __attribute__((always_inline)) { return a.ws[2] + ((int64_t)ids[pick] * ((a.H + 127) / 128) + n0 / F8_BLOCK) * blocks; };
    i32x4 w[NS][2];
    float sd[NS];
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const int step = step_of(i), pick = step / blocks, b = step - pick * blocks;
        const uint8_t *p = matrix_of(pick) + (int64_t)min(n0 + (lane & 15), a.H - 1) * a.rbi + b * F8_BLOCK + at;
        w[i][0] = *(const i32x4 *)p;
        w[i][1] = *(const i32x4 *)(p + 64);
        sd[i] = scales_of(pick)[b];
    }
    if (threadIdx.x < a.K) wk[threadIdx.x] = wt[threadIdx.x];
    for (int j0 = 0; j0 < a.K; j0 += F8_FEW_WAVES / wpp) {
        const int j = j0 + wave / wpp;
        const float *row = h + (int64_t)min(j, a.K - 1) * a.ldh;
        if (j0) fetch_h(min(j, a.K - 1));
        if (j >= a.K) continue;
        auto store = [&](int at, const float (&v)[4]) __attribute__((always_inline)) {
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) bits = max_bits(bits, v[i]);
            bits = max16_u(bits);
            bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16));  // (the 32 lanes of a group are all in the row's codes, or none)
            if (at >= a.rbi) return;
            const F8Group g(bits);
            *(uint32_t *)(hq + j * a.rbi + at) = f8_codes4(g.quotient(v[0]), g.quotient(v[1]), g.quotient(v[2]), g.quotient(v[3]));
            if ((lane & 31) == 0) hs[j * blocks + at / F8_BLOCK] = g.scale;
        };
#pragma unroll
        for (int i = 0; i < NH; i++) store(at0 + i * stride, hv[i]);
        for (int o = at0 + NH * stride; o - 4 * lane < a.rbi; o += stride) {
            float v[4];
            load_row<4>(row + o, a.I - o, v);
            store(o, v);
        }
    }
    __syncthreads();
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    bool strange = false;
#pragma unroll
    for (int i = 0; i < NS; i++) {
        if (wave + F8_FEW_WAVES * i >= steps) break;
        const int step = step_of(i), pick = step / blocks;
        const uint8_t *p = hq + step * F8_BLOCK + at;
        F8Frag<EXACT> x, wf;
        x.load(p, p + 64);
        wf.load((const uint8_t *)&w[i][0], (const uint8_t *)&w[i][1]);
        const float sx = hs[step], s = sx * sd[i], wj = wk[pick];
        strange |= f8_strange(sx) | f8_strange(sd[i]);
        const f32x4 v = F8Frag<EXACT>::product(wf, x);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = fmaf(v[c] * s, wj, acc[c]);
    }
    if ((lane & 15) == 0) *(f32x4 *)&part[wave][4 * (lane >> 4)] = acc;
    strange = __syncthreads_or(strange);
    if (threadIdx.x >= 16 || n0 + threadIdx.x >= a.H) return;
    const int n = n0 + threadIdx.x;
    float v = part[0][threadIdx.x];
#pragma unroll
    for (int q = 1; q < F8_FEW_WAVES; q++) v += part[q][threadIdx.x];
    if (strange) {
        v = 0.f;
        for (int j = 0; j < a.K; j++) {
            f32x4 sum;
            f8_strange_sums(hq + j * a.rbi, hs + j * blocks, 1, matrix_of(j) + (int64_t)n * a.rbi, scales_of(j), a.rbi, 1, sum, true);
            v = fmaf(sum[0], wk[j], v);
        }
    }
    if (a.bias[2])
        for (int j = 0; j < a.K; j++) v = fmaf(wk[j], a.bias[2][(int64_t)ids[j] * a.H + n], v);
    ((T *)a.out)[(int64_t)t * a.H + n] = from_f32<T>(v);
}

template <class T, bool EXACT>
static int few_down(const F8FewArgs &a, hipStream_t s) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.H + 15) / 16), a.T), dim3(64 * F8_FEW_WAVES), a.K * (a.rbi + a.rbi / 32), s, a);
        return check_launch("k_f8_few_down");
    };
    const int steps = (a.K * (a.rbi / F8_BLOCK) + F8_FEW_WAVES - 1) / F8_FEW_WAVES;  // of a wave
    return steps <= 1 ? go(k_f8_few_down<T, 1, EXACT>) : steps <= 2 ? go(k_f8_few_down<T, 2, EXACT>) : steps <= 4 ? go(k_f8_few_down<T, 4, EXACT>)
         : steps <= 8 ? go(k_f8_few_down<T, 8, EXACT>) : steps <= 12 ? go(k_f8_few_down<T, 12, EXACT>) : go(k_f8_few_down<T, 16, EXACT>);
}
template <int PER, bool EXACT>
static int few_gateup(const F8FewArgs &a, hipStream_t s) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.I + 15) / 16), a.K, a.T), dim3(64 * F8_FEW_WAVES), 0, s, a);
        return check_launch("k_f8_few_gateup");
    };
    const int steps = (a.rbh / F8_BLOCK + F8_FEW_WAVES / 2 - 1) / (F8_FEW_WAVES / 2);
    return steps <= 2 ? go(k_f8_few_gateup<PER, 2, EXACT>) : steps <= 4 ? go(k_f8_few_gateup<PER, 4, EXACT>) : steps <= 6 ? go(k_f8_few_gateup<PER, 6, EXACT>)
                      : go(k_f8_few_gateup<PER, 8, EXACT>);
}
template <bool EXACT>
static int few_gateup(const F8FewArgs &a, hipStream_t s) {
    const int per = i8_route_width(a.E);
    return per == 4 ? few_gateup<4, EXACT>(a, s) : per == 8 ? few_gateup<8, EXACT>(a, s) : few_gateup<16, EXACT>(a, s);
}

// ------------------------------------------------------------------------------ many tokens

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
// 2,048 tokens of 4 picks over 128 experts of 2,880 x 2,880: 470 to 496 us, 4.3 to 4.5 TB/s of weights (exact products 617); the waves wait for loads 35 % of their cycles and to issue 46 %.
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
                    f8_strange_sums(a.x + row * a.rb, a.xs + row, a.m, a.w[j >> 1] + tl.expert * a.stride[j >> 1] + (int64_t)n * a.rb,
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
    size_t ids, w, h, order, place, offsets, tiles, sort, hq, hs, dn, total;
    bool few;
};

static F8MoeLayout layout(const cw_f8_moe_desc *d, int T) {
    F8MoeLayout L = {};
    size_t off = 0;
    auto take = [&](size_t &at, size_t bytes) { at = off; off = (off + bytes + 255) & ~(size_t)255; };
    const size_t TK = (size_t)T * d->top_k;
    take(L.ids, TK * 4);
    take(L.w, TK * 4);
    L.few = f8_few_tokens(d->n_experts, d->top_k, d->hidden, d->inter, T);
    if (L.few) {
        take(L.h, TK * ((d->inter + 3) & ~3) * 4);
        L.total = off;
        return L;
    }
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
    if (TK >= 1 << 28 || blocks >= 1 << 23)
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
    hipStream_t s = (hipStream_t)stream;
    if (L.few) {
        F8FewArgs a = {};
        for (int m = 0; m < 3; m++) {
            a.w[m] = d->w[m];
            a.stride[m] = d->slot_stride[m];
            a.ws[m] = d->scale[m];
            a.bias[m] = d->bias[m];
        }
        a.x = x;
        a.xs = x_scale;
        a.logits = logits;
        a.E = E;
        a.K = K;
        a.H = H;
        a.I = I;
        a.T = T;
        a.norm = d->norm;
        a.glu = glu_of(d->act, d->alpha, d->limit);
        a.rbh = (int)f8_row_bytes(H);
        a.rbi = (int)f8_row_bytes(I);
        a.ldh = (I + 3) & ~3;
        a.ids = ids;
        a.wt = w;
        a.h = (float *)(base + L.h);
        a.out = out;
        // (as below: results in f16 and f32 from exact products)
        if (int rc = ydtype == CW_BF16 ? few_gateup<false>(a, s) : few_gateup<true>(a, s)) return rc;
        return ydtype == CW_F16 ? few_down<_Float16, true>(a, s) : ydtype == CW_BF16 ? few_down<bf16_t, false>(a, s) : few_down<float, true>(a, s);
    }
    if (int rc = cw_route_topk(logits, T, E, K, d->norm, ids, w, stream)) return rc;
    if (int rc = cw_sort_picks(ids, TK, E, order, place, offsets, tiles, base + L.sort, cw_sort_picks_workspace_size(TK, E), stream)) return rc;
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
    // beside 1.7e-3); results in f16 and f32 have exact products in gate and up, whose codes hang on them, and in down
    const int blocks = (int)f8_blocks(I);
    const dim3 grid((unsigned)((pile_max_tiles(TK, E) * blocks + 7) / 8 * 8));
    constexpr int LDS = F8Stream<8, 4>::LDS;
    if (ydtype == CW_BF16) hipLaunchKernelGGL(k_f8_gateup<false>, grid, dim3(256), LDS, s, a, blocks);
    else hipLaunchKernelGGL(k_f8_gateup<true>, grid, dim3(256), LDS, s, a, blocks);
    if (int rc = check_launch("k_f8_gateup")) return rc;
    if (int rc = f8_matmul_experts(d->w[2], d->slot_stride[2], d->scale[2], E, H, I, hq, hs, TK, nullptr, K, TK, tiles, d->bias[2], CW_F32, dn, H,
                                   ydtype != CW_BF16, s))
        return rc;
    return from_piles_f32(ydtype, dn, w, T, K, E, H, place, offsets, out, s);
}

}  // extern "C"
