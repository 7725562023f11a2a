// A MoE layer of 8-bit integer experts on 8-bit integer rows (gfx950): two kernels for a few tokens, grouped
// matrix products for many.
#include <algorithm>

#include "cw_i8.h"
#include "cw_i8_tile.h"
#include "cw_mfma.h"

namespace cw {

struct I8MoeArgs {
    const uint8_t *w[3];
    int64_t stride[3];
    const float *ws[3], *bias[3];
    const uint8_t *x;
    const float *xs, *logits;
    int E, K, H, I, T, norm, act;
    float alpha, limit;
    int rbh, rbi, ldh;  // bytes of a row of H and of I codes, floats of a hidden row
    uint32_t *ids;
    float *wt, *h;
    void *out;
    // many tokens
    const MfTile *tiles;
    const int *n_tiles, *pile_pick, *pile_tok;
    const uint8_t *hq;
    const float *hs;
    float *dn;
};

__device__ __forceinline__ int dot16(i32x4 a, i32x4 b, int acc) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_sdot4(a[i], b[i], acc, false);
    return acc;
}
__device__ __forceinline__ int wave_sum_i(int v) {
    v += (int)dpp_u<0xB1>((uint32_t)v);
    v += (int)dpp_u<0x4E>((uint32_t)v);
    v += (int)dpp_u<0x141>((uint32_t)v);
    v += (int)dpp_u<0x140>((uint32_t)v);
    return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) + (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}

// ------------------------------------------------------------------------------ a few tokens

// Gate and up of one pick of a token: every wave routes the token itself (its logits are one load), then takes
// R rows of both matrices, lane l the 16 bytes l, l + 64, ... of each row and of x.
template <int PER, int NC, int R>
__global__ __launch_bounds__(256) void k_i8_few_gateup(I8MoeArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.z, j = blockIdx.y;
    const int r0 = (blockIdx.x * 4 + wave) * R;
    uint32_t id;
    float wt;
    wave_route<PER>(a.logits + (int64_t)t * a.E, a.E, a.K, a.norm, &id, &wt);
    if (blockIdx.x == 0 && j == 0 && wave == 0 && lane < a.K) {
        a.ids[(int64_t)t * a.K + lane] = id;
        a.wt[(int64_t)t * a.K + lane] = wt;
    }
    if (r0 >= a.I) return;
    const int64_t e = __builtin_amdgcn_readlane((int)id, j);
    i32x4 x[NC], g[R][NC], u[R][NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int o = 16 * (lane + 64 * c), off = o < a.rbh ? o : 0;  // past the row: any valid bytes, times zeros
        x[c] = load16(a.x + (int64_t)t * a.rbh + off);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t row = (int64_t)min(r0 + r, a.I - 1) * a.rbh + off;
            g[r][c] = load16(a.w[0] + e * a.stride[0] + row);
            u[r][c] = load16(a.w[1] + e * a.stride[1] + row);
        }
        if (o >= a.rbh) x[c] = i32x4{0, 0, 0, 0};
    }
    const float sx = a.xs[t];
#pragma unroll
    for (int r = 0; r < R; r++) {
        int sg = 0, su = 0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            sg = dot16(g[r][c], x[c], sg);
            su = dot16(u[r][c], x[c], su);
        }
        sg = wave_sum_i(sg);
        su = wave_sum_i(su);
        const int64_t n = e * a.I + min(r0 + r, a.I - 1);
        const float gv = fmaf((float)sg, sx * a.ws[0][n], a.bias[0] ? a.bias[0][n] : 0.f);
        const float uv = fmaf((float)su, sx * a.ws[1][n], a.bias[1] ? a.bias[1][n] : 0.f);
        if (lane == 0 && r0 + r < a.I) a.h[((int64_t)t * a.K + j) * a.ldh + r0 + r] = glu(gv, uv, a.act, a.alpha, a.limit);
    }
}

// Down and the weighted sum of a token: the block quantizes the token's K hidden rows into LDS (every block of
// the token does), then each wave sums one output: lane l holds the 16 bytes l, l + 64, ... of the K rows' codes
// laid end to end.
constexpr int FEW_DOWN_WAVES = 8;
template <class T, int NC>
__global__ __launch_bounds__(64 * FEW_DOWN_WAVES) void k_i8_few_down(I8MoeArgs a) {
    extern __shared__ __align__(16) uint8_t hq[];  // K rows of rbi codes
    __shared__ float coef[32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.y, cpr = a.rbi / 16;
    const int row = blockIdx.x * FEW_DOWN_WAVES + wave, rowc = min(row, a.H - 1);
    const uint32_t *ids = a.ids + (int64_t)t * a.K;
    i32x4 w[NC];
    float sd[NC];
    int pick[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int i = min(lane + 64 * c, a.K * cpr - 1);
        pick[c] = i / cpr;
        const int64_t e = ids[pick[c]];
        w[c] = load16(a.w[2] + e * a.stride[2] + (int64_t)rowc * a.rbi + 16 * (i - pick[c] * cpr));
        sd[c] = a.ws[2][e * a.H + rowc];
    }
    float b = 0.f;
    if (a.bias[2] && lane < a.K) b = a.wt[(int64_t)t * a.K + lane] * a.bias[2][(int64_t)ids[lane] * a.H + rowc];
    for (int j = wave; j < a.K; j += FEW_DOWN_WAVES) {
        const float *h = a.h + ((int64_t)t * a.K + j) * a.ldh;
        double m = 0.0;
        for (int c = 4 * lane; c < a.I; c += 256) {
            float v[4];
            load_row<4>(h + c, a.I - c, v);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double y = fabs((double)v[i]);
                m = y <= m ? m : y < INFINITY ? y : INFINITY;
            }
        }
        m = wave_max_d(m);
        const bool some = m > 0.0 && m < INFINITY;
        const double inv = some ? 127.0 / m : 0.0;
        for (int c = 4 * lane; c < a.rbi; c += 256) {
            float v[4];
            load_row<4>(h + c, a.I - c, v);
            *(uint32_t *)(hq + j * a.rbi + c) = some ? codes4(code(v[0], inv), code(v[1], inv), code(v[2], inv), code(v[3], inv)) : 0u;
        }
        if (lane == 0) coef[j] = a.wt[(int64_t)t * a.K + j] * (m < INFINITY ? (float)(m / 127.0) : __int_as_float(0x7fc00000));
    }
    __syncthreads();
    if (row >= a.H) return;
    float acc = b;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int i = lane + 64 * c;
        if (i < a.K * cpr) {
            const int d = dot16(w[c], *(const i32x4 *)(hq + 16 * i), 0);
            acc = fmaf((float)d, coef[pick[c]] * sd[c], acc);
        }
    }
    acc = wave_sum(acc);
    if (lane == 0) ((T *)a.out)[(int64_t)t * a.H + row] = from_f32<T>(acc);
}

// ------------------------------------------------------------------------------ many tokens

constexpr int I8_TILE = 128;  // picks of a tile

// Gate and up of a tile: a wave holds 16 rows of each. Hidden rows in pile order, f32.
template <int MB>
__device__ __forceinline__ void gateup_tile(const I8MoeArgs &a, const MfTile &tl, int n0, uint8_t *lds) {
    constexpr int NB = 1;
    const int lane = threadIdx.x & 63;
    const uint8_t *w0[2];
    uint32_t wrow[2 * NB];
#pragma unroll
    for (int j = 0; j < 2; j++) w0[j] = a.w[j] + (int64_t)tl.expert * a.stride[j];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++) wrow[j] = min(n0 + 16 * (j % NB) + (lane & 15), a.I - 1) * a.rbh + 16 * (lane >> 4);
    i32x4 acc[MB][2 * NB];
    i8_loop<MB, 2 * NB, 2>(lds, a.x, [&](int r) { return (uint32_t)a.pile_tok[tl.pos0 + min(r, tl.m - 1)] * (uint32_t)a.rbh; }, w0, wrow,
                              a.rbh, acc);
    float sw[2 * NB][4], b[2 * NB][4];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t n = (int64_t)tl.expert * a.I + min(n0 + 16 * (j % NB) + 4 * (lane >> 4) + i, a.I - 1);
            sw[j][i] = a.ws[j / NB][n];
            b[j][i] = a.bias[j / NB] ? a.bias[j / NB][n] : 0.f;
        }
    // (all loads before the bounds checks, from clamped places: inside them each would be waited for in turn)
    float sxs[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) sxs[mb] = a.xs[a.pile_tok[tl.pos0 + min(16 * mb + (lane & 15), tl.m - 1)]];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int r = 16 * mb + (lane & 15);
        if (r >= tl.m) continue;
        const int p = tl.pos0 + r;
        const float sx = sxs[mb];
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int n = n0 + 16 * j + 4 * (lane >> 4);
            if (n >= a.I) continue;
            float h[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                h[i] = glu(fmaf((float)acc[mb][j][i], sx * sw[j][i], b[j][i]), fmaf((float)acc[mb][NB + j][i], sx * sw[NB + j][i], b[NB + j][i]),
                           a.act, a.alpha, a.limit);
            store_row<4>(a.h + (int64_t)p * a.ldh + n, a.I - n, h);
        }
    }
}
// Down of a tile: a wave holds 32 rows. One row of H per pick, f32, in pick order.
template <int MB>
__device__ __forceinline__ void down_tile(const I8MoeArgs &a, const MfTile &tl, int n0, uint8_t *lds) {
    constexpr int NW = 2;
    const int lane = threadIdx.x & 63;
    const uint8_t *w0[1] = {a.w[2] + (int64_t)tl.expert * a.stride[2]};
    uint32_t wrow[NW];
#pragma unroll
    for (int j = 0; j < NW; j++) wrow[j] = min(n0 + 16 * j + (lane & 15), a.H - 1) * a.rbi + 16 * (lane >> 4);
    i32x4 acc[MB][NW];
    i8_loop<MB, NW, 1>(lds, a.hq + (int64_t)tl.pos0 * a.rbi, [&](int r) { return (uint32_t)(min(r, tl.m - 1) * a.rbi); }, w0, wrow,
                          a.rbi, acc);
    float sw[NW][4];
#pragma unroll
    for (int j = 0; j < NW; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) sw[j][i] = a.ws[2][(int64_t)tl.expert * a.H + min(n0 + 16 * j + 4 * (lane >> 4) + i, a.H - 1)];
    float sxs[MB];
    int picks[MB];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int p = tl.pos0 + min(16 * mb + (lane & 15), tl.m - 1);
        sxs[mb] = a.hs[p];
        picks[mb] = a.pile_pick[p];
    }
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        if (16 * mb + (lane & 15) >= tl.m) continue;
        const float sx = sxs[mb];
        float *d = a.dn + (int64_t)picks[mb] * a.H;
#pragma unroll
        for (int j = 0; j < NW; j++) {
            const int n = n0 + 16 * j + 4 * (lane >> 4);
            if (n >= a.H) continue;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (float)acc[mb][j][i] * (sx * sw[j][i]);
            store_row<4>(d + n, a.H - n, v);
        }
    }
}

// Blocks go to the eight dies in turn; each die takes a contiguous range of the items (a tile's blocks of W one after
// the other), so that a tile's picks are read by one die and not by all (2,048 tokens over 128 experts of 2,880 x 2,880:
// 2.4 GB fetched for gate and up instead of 2.1).
template <bool DOWN>
__global__ __launch_bounds__(256, 2) void k_i8_moe_tiles(I8MoeArgs a, int n_blocks) {
    extern __shared__ __align__(1024) uint8_t lds[];
    const int total = *a.n_tiles * n_blocks, die = blockIdx.x & 7, at = blockIdx.x >> 3, per = total >> 3, rest = total & 7;
    if (at >= per + (die < rest)) return;
    const int item = __builtin_amdgcn_readfirstlane(die * per + min(die, rest) + at), tile = item / n_blocks, nb = item % n_blocks;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const MfTile tl = a.tiles[tile];
    const int n0 = DOWN ? 128 * nb + 32 * wave : 64 * nb + 16 * wave;
    auto run = [&](auto mb) __attribute__((always_inline)) {
        if constexpr (DOWN) down_tile<decltype(mb)::value>(a, tl, n0, lds);
        else gateup_tile<decltype(mb)::value>(a, tl, n0, lds);
    };
    if (tl.m <= 16) run(Ic<1>{});
    else if (tl.m <= 32) run(Ic<2>{});
    else if (tl.m <= 48) run(Ic<3>{});
    else if (tl.m <= 64) run(Ic<4>{});
    else if (tl.m <= 80) run(Ic<5>{});
    else if (tl.m <= 96) run(Ic<6>{});
    else run(Ic<8>{});
}

// out[t] = sum_j w_j (dn_j + bias), in pick order; a thread per four columns
template <class T>
__global__ __launch_bounds__(256) void k_i8_combine(I8MoeArgs a) {
    const int per = (a.H + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.T * per; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per;
        const int n = 4 * (int)(i - t * per), valid = a.H - n;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < a.K; j++) {
            const int64_t p = t * a.K + j;
            float v[4], b[4] = {0.f, 0.f, 0.f, 0.f};
            load_row<4>(a.dn + p * a.H + n, valid, v);
            if (a.bias[2]) load_row<4>(a.bias[2] + (int64_t)a.ids[p] * a.H + n, valid, b);
            const float w = a.wt[p];
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] = fmaf(w, v[c] + b[c], acc[c]);
        }
        store_row<4>((T *)a.out + t * a.H + n, valid, acc);
    }
}

// ------------------------------------------------------------------------------ the layer

struct I8MoeLayout {
    size_t ids, w, h, tiles, n_tiles, pile_pick, pile_tok, hq, hs, dn, total;
    bool few;
};

static bool few_path(const cw_i8_moe_desc *d, int T) {
    return T <= 8 && i8_row_bytes(d->hidden) <= 4 * 1024 && d->top_k * i8_row_bytes(d->inter) <= 16 * 1024;
}

static I8MoeLayout layout(const cw_i8_moe_desc *d, int T) {
    I8MoeLayout L = {};
    size_t off = 0;
    auto take = [&](size_t &at, size_t bytes) { at = off; off = (off + bytes + 255) & ~(size_t)255; };
    const size_t TK = (size_t)T * d->top_k;
    L.few = few_path(d, T);
    take(L.ids, TK * 4);
    take(L.w, TK * 4);
    take(L.h, TK * ((d->inter + 3) & ~3) * 4);
    if (!L.few) {
        take(L.tiles, (size_t)max_tiles((int)TK, d->n_experts, I8_TILE) * sizeof(MfTile));
        take(L.n_tiles, 4);
        take(L.pile_pick, TK * 4);
        take(L.pile_tok, TK * 4);
        take(L.hq, TK * i8_row_bytes(d->inter));
        take(L.hs, TK * 4);
        take(L.dn, TK * (size_t)d->hidden * 4);
    }
    L.total = off;
    return L;
}

static int check_desc(const cw_i8_moe_desc *d, int T) {
    CW_REQUIRE(d != nullptr, "i8 moe: null descriptor");
    CW_REQUIRE(T >= 0, "i8 moe: negative token count %d", T);
    CW_REQUIRE(d->n_experts > 0 && d->n_experts <= 1024, "i8 moe: %d experts (1..1024 supported)", d->n_experts);
    CW_REQUIRE(d->top_k > 0 && d->top_k <= 32 && d->top_k <= d->n_experts, "i8 moe: top_k %d for %d experts", d->top_k, d->n_experts);
    CW_REQUIRE(d->hidden > 0 && d->inter > 0, "i8 moe: hidden %d, inter %d", d->hidden, d->inter);
    if (d->hidden > CW_I8_MAX_K || d->inter > CW_I8_MAX_K)
        return set_error(CW_ENOTSUP, "i8 moe: hidden %d, inter %d above %d", d->hidden, d->inter, CW_I8_MAX_K);
    CW_REQUIRE(d->act == CW_ACT_SILU || d->act == CW_ACT_CLAMPED_SWIGLU, "i8 moe: unknown activation %d", d->act);
    CW_REQUIRE((int64_t)T * d->top_k < (1ll << 28), "i8 moe: %lld picks", (long long)T * d->top_k);
    for (int m = 0; m < 3; m++) {
        const int64_t need = (m == 2 ? d->hidden : d->inter) * i8_row_bytes(m == 2 ? d->inter : d->hidden);
        CW_REQUIRE(d->w[m] && d->scale[m], "i8 moe: matrix %d is null", m);
        CW_REQUIRE(i8_aligned(d->w[m], 16) && d->slot_stride[m] % 16 == 0, "i8 moe: matrix %d must be 16-byte aligned", m);
        CW_REQUIRE(d->slot_stride[m] >= need, "i8 moe: matrix %d slot stride %lld below its %lld bytes", m, (long long)d->slot_stride[m],
                   (long long)need);
    }
    return CW_OK;
}

template <class T>
static int few_down(const I8MoeArgs &a, hipStream_t s) {
    const int chunks = a.K * (a.rbi / 16);
    const dim3 grid((a.H + FEW_DOWN_WAVES - 1) / FEW_DOWN_WAVES, a.T);
#define CW_DOWN(N) \
    if (chunks <= 64 * N) { \
        hipLaunchKernelGGL((k_i8_few_down<T, N>), grid, dim3(64 * FEW_DOWN_WAVES), a.K * a.rbi, s, a); \
        return check_launch("k_i8_few_down"); \
    }
    CW_DOWN(2) CW_DOWN(4) CW_DOWN(8) CW_DOWN(12) CW_DOWN(16)
#undef CW_DOWN
    return set_error(CW_ENOTSUP, "i8 moe: %d picks' rows of %d", a.K, a.I);
}
template <int PER>
static int few_gateup(const I8MoeArgs &a, hipStream_t s) {
#define CW_GU(N, R) \
    if (a.rbh <= 1024 * N) { \
        hipLaunchKernelGGL((k_i8_few_gateup<PER, N, R>), dim3((a.I + 4 * R - 1) / (4 * R), a.K, a.T), dim3(256), 0, s, a); \
        return check_launch("k_i8_few_gateup"); \
    }
    CW_GU(1, 4) CW_GU(2, 2) CW_GU(3, 2) CW_GU(4, 2)
#undef CW_GU
    return set_error(CW_ENOTSUP, "i8 moe: rows of %d", a.H);
}

static int moe_layer(const cw_i8_moe_desc *d, I8MoeArgs a, int ydtype, const I8MoeLayout &L, uint8_t *base, hipStream_t s) {
    int rc;
    if (L.few) {
        rc = a.E <= 256 ? few_gateup<4>(a, s) : a.E <= 512 ? few_gateup<8>(a, s) : few_gateup<16>(a, s);
        if (rc) return rc;
        return ydtype == CW_F16 ? few_down<_Float16>(a, s) : ydtype == CW_BF16 ? few_down<bf16_t>(a, s) : few_down<float>(a, s);
    }
    const int TK = a.T * a.K, tmax = max_tiles(TK, a.E, I8_TILE);
    if ((rc = cw_route_topk(a.logits, a.T, a.E, a.K, a.norm, a.ids, a.wt, s))) return rc;
    int *pile_pick = (int *)(base + L.pile_pick), *pile_tok = (int *)(base + L.pile_tok), *n_tiles = (int *)(base + L.n_tiles);
    MfTile *tiles = (MfTile *)(base + L.tiles);
    if ((rc = mfma_piles(a.ids, nullptr, TK, a.K, a.E, 0, pile_pick, pile_tok, tiles, n_tiles, s, I8_TILE))) return rc;
    int8_t *hq = (int8_t *)(base + L.hq);
    float *hs = (float *)(base + L.hs);
    a.tiles = tiles;
    a.n_tiles = n_tiles;
    a.pile_pick = pile_pick;
    a.pile_tok = pile_tok;
    a.hq = (const uint8_t *)hq;
    a.hs = hs;
    a.dn = (float *)(base + L.dn);
    const int lds = I8Stage<I8_TILE / 16>::LDS, gu = (a.I + 63) / 64, dn = (a.H + 127) / 128;
    hipLaunchKernelGGL(k_i8_moe_tiles<false>, dim3((unsigned)((tmax * gu + 7) / 8 * 8)), dim3(256), lds, s, a, gu);
    if ((rc = check_launch("k_i8_moe_tiles"))) return rc;
    if ((rc = i8_quantize_f32(a.h, TK, a.I, a.ldh, hq, hs, s))) return rc;
    hipLaunchKernelGGL(k_i8_moe_tiles<true>, dim3((unsigned)((tmax * dn + 7) / 8 * 8)), dim3(256), lds, s, a, dn);
    if ((rc = check_launch("k_i8_moe_tiles"))) return rc;
    const int64_t n = (int64_t)a.T * ((a.H + 3) / 4);
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16));
    if (ydtype == CW_F16) hipLaunchKernelGGL(k_i8_combine<_Float16>, grid, dim3(256), 0, s, a);
    else if (ydtype == CW_BF16) hipLaunchKernelGGL(k_i8_combine<bf16_t>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_i8_combine<float>, grid, dim3(256), 0, s, a);
    return check_launch("k_i8_combine");
}

}  // namespace cw

using namespace cw;

extern "C" {

size_t cw_i8_moe_workspace_size(const cw_i8_moe_desc *d, int T) {
    if (check_desc(d, T) != CW_OK || T == 0) return 0;
    return layout(d, T).total;
}

int cw_i8_moe_layer(const cw_i8_moe_desc *d, const int8_t *x, const float *x_scale, const float *logits, int T, int ydtype, void *out,
                    uint32_t *ids_out, float *w_out, void *ws, size_t ws_bytes, cw_stream_t stream) {
    if (int rc = check_desc(d, T)) return rc;
    if (!i8_float_type(ydtype)) return set_error(CW_ENOTSUP, "i8 moe: type %d of out (f32, f16 or bf16)", ydtype);
    if (T == 0) return CW_OK;
    CW_REQUIRE(x && x_scale && logits && out, "i8 moe: null x, scales, logits or out");
    CW_REQUIRE(i8_aligned(x, 16), "i8 moe: codes must be 16-byte aligned");
    const I8MoeLayout L = layout(d, T);
    CW_REQUIRE(ws && ws_bytes >= L.total, "i8 moe: workspace of %zu bytes, %zu needed", ws_bytes, L.total);
    CW_REQUIRE(i8_aligned(ws, 256), "i8 moe: workspace must be 256-byte aligned");
    uint8_t *base = (uint8_t *)ws;
    I8MoeArgs a = {};
    for (int m = 0; m < 3; m++) {
        a.w[m] = (const uint8_t *)d->w[m];
        a.stride[m] = d->slot_stride[m];
        a.ws[m] = d->scale[m];
        a.bias[m] = d->bias[m];
    }
    a.x = (const uint8_t *)x;
    a.xs = x_scale;
    a.logits = logits;
    a.E = d->n_experts;
    a.K = d->top_k;
    a.H = d->hidden;
    a.I = d->inter;
    a.T = T;
    a.norm = d->norm;
    a.act = d->act;
    a.alpha = d->alpha;
    a.limit = d->limit;
    a.rbh = (int)i8_row_bytes(a.H);
    a.rbi = (int)i8_row_bytes(a.I);
    a.ldh = (a.I + 3) & ~3;
    a.ids = ids_out ? ids_out : (uint32_t *)(base + L.ids);
    a.wt = w_out ? w_out : (float *)(base + L.w);
    a.h = (float *)(base + L.h);
    a.out = out;
    return moe_layer(d, a, ydtype, L, base, (hipStream_t)stream);
}

}  // extern "C"
