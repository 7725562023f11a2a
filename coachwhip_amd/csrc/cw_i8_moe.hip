// A MoE layer of 8-bit integer experts on 8-bit integer rows (gfx950): two kernels for a few tokens, grouped
// matrix products for many.
#include <algorithm>

#include "cw_i8.h"
#include "cw_i8_rules.h"
#include "cw_i8_tile.h"
#include "cw_mfma.h"

namespace cw {

// A tile: m picks of one expert from pile position pos0; the expert has `of` tiles, the first of them tile `first`.
struct I8Tile {
    int expert, pos0, m, first, of;
};

struct I8MoeArgs {
    const uint8_t *w[3];
    int64_t stride[3];
    const float *ws[3], *bias[3];
    const uint8_t *x;
    const float *xs, *logits;
    int E, K, H, I, T, norm;
    Glu glu;
    int rbh, rbi, ldh;  // bytes of a row of H and of I codes, floats of a hidden row
    uint32_t *ids;
    float *wt, *h;
    void *out;
    // many tokens
    const I8Tile *tiles;
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

// Gate and up of one pick of a token, eight waves of R rows of both matrices each: lane l takes the 16 bytes l, l + 64,
// ... of each row and of x. One wave routes the token for its block (every wave for itself: 16,384 times 2,500 cycles
// for 8 tokens of 8 picks), no further than this pick; the last pick's first block, which goes all the way, stores the
// routing.
template <int PER, int NC, int R>
__global__ __launch_bounds__(64 * I8_FEW_WAVES) void k_i8_few_gateup(I8MoeArgs a) {
    __shared__ uint32_t expert;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.z, j = blockIdx.y;
    const int r0 = (blockIdx.x * I8_FEW_WAVES + wave) * R;
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
    i32x4 x[NC], g[R][NC], u[R][NC];
    int off[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int o = 16 * (lane + 64 * c);
        off[c] = o < a.rbh ? o : 0;  // past the row: any valid bytes, times zeros
        x[c] = load16(a.x + (int64_t)t * a.rbh + off[c]);
        if (o >= a.rbh) x[c] = i32x4{0, 0, 0, 0};
    }
    const double sx = a.xs[t];
    __syncthreads();
    if (r0 >= a.I) return;
    const int64_t e = __builtin_amdgcn_readfirstlane((int)expert);
    // lane r < R scales row r0 + r
    const int64_t mine = e * a.I + min(r0 + (lane & (R - 1)), a.I - 1);
    float sw[2], b[2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
        sw[m] = a.ws[m][mine];
        b[m] = a.bias[m] ? a.bias[m][mine] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int row = min(r0 + r, a.I - 1);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            g[r][c] = load16(a.w[0] + e * a.stride[0] + (int64_t)row * a.rbh + off[c]);
            u[r][c] = load16(a.w[1] + e * a.stride[1] + (int64_t)row * a.rbh + off[c]);
        }
    }
    int sum[2] = {0, 0};
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
        sum[0] = lane == r ? sg : sum[0];
        sum[1] = lane == r ? su : sum[1];
    }
    const float h = glu(scaled(sum[0], sx * sw[0], b[0]), scaled(sum[1], sx * sw[1], b[1]), a.glu);
    if (lane < R && r0 + lane < a.I) a.h[((int64_t)t * a.K + j) * a.ldh + r0 + lane] = h;
}

// Down and the weighted sum of a token: the block quantizes the token's K hidden rows into LDS (every block of
// the token does, one, two, four or eight waves a row), then each wave sums R outputs: lane l holds the 16 bytes l,
// l + 64, ... of the K rows' codes laid end to end. The hidden rows are asked for before the weights: loads return in
// order, and the codes are made while the weights come in.
template <class T, int NC, int R>
__global__ __launch_bounds__(64 * I8_FEW_WAVES, NC >= 8 || R == 4 ? 4 : NC == 4 ? 6 : 8) void k_i8_few_down(I8MoeArgs a) {
    constexpr int NH = NC < 12 ? (NC + 1) / 2 : 6;  // pieces of a hidden row held in registers (the others are read twice)
    extern __shared__ __align__(16) uint8_t hq[];  // K rows of rbi codes
    __shared__ float hs[32];
    __shared__ double coef[I8_FEW_WAVES * R][33];
    __shared__ uint32_t top[I8_FEW_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.y, cpr = a.rbi / 16;
    const int row0 = (blockIdx.x * I8_FEW_WAVES + wave) * R;
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
    i32x4 w[R][NC];
    uint32_t picks[(NC + 3) / 4] = {};  // of each chunk, a byte each
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int i = min(lane + 64 * c, a.K * cpr - 1), pick = i / cpr;
        picks[c / 4] |= (uint32_t)pick << (8 * (c % 4));
        const uint8_t *p = a.w[2] + (int64_t)ids[pick] * a.stride[2] + 16 * (i - pick * cpr);
#pragma unroll
        for (int r = 0; r < R; r++) w[r][c] = load16(p + (int64_t)min(row0 + r, a.H - 1) * a.rbi);
    }
    // lane j < K: the pick's weight, the scale of its output channel and its bias
    const int mine = min(lane, a.K - 1);
    const float wj = wt[mine];
    float sd[R], b[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int64_t n = (int64_t)ids[mine] * a.H + min(row0 + r, a.H - 1);
        sd[r] = a.ws[2][n];
        b[r] = a.bias[2] && lane < a.K ? a.bias[2][n] : 0.f;
    }
    for (int j0 = 0; j0 < a.K; j0 += I8_FEW_WAVES / wpp) {
        const int j = j0 + wave / wpp;
        const float *row = h + (int64_t)min(j, a.K - 1) * a.ldh;
        if (j0) fetch_h(min(j, a.K - 1));
        uint32_t bits = 0;
        auto more = [&](const float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; i++) bits = max_bits(bits, v[i]);
        };
#pragma unroll
        for (int i = 0; i < NH; i++) more(hv[i]);
        for (int c = at0 + NH * stride; c < a.I; c += stride) {
            float v[4];
            load_row<4>(row + c, a.I - c, v);
            more(v);
        }
        bits = wave_max_u(bits);
        if (wpp > 1) {
            if (lane == 0) top[wave] = bits;
            __syncthreads();
            for (int o = 1; o < wpp; o++) bits = max(bits, top[wave ^ o]);
            if (j0 + I8_FEW_WAVES / wpp < a.K) __syncthreads();
        }
        if (j >= a.K) continue;
        const bool fine = bits < 0x7F800000u, some = fine && bits;
        const double m = __uint_as_float(bits), inv = some ? 127.0 / m : 0.0;
        auto store = [&](int c, const float (&v)[4]) __attribute__((always_inline)) {
            *(uint32_t *)(hq + j * a.rbi + c) = some ? codes4(code(v[0], inv), code(v[1], inv), code(v[2], inv), code(v[3], inv)) : 0u;
        };
#pragma unroll
        for (int i = 0; i < NH; i++)
            if (at0 + i * stride < a.rbi) store(at0 + i * stride, hv[i]);
        for (int c = at0 + NH * stride; c < a.rbi; c += stride) {
            float v[4];
            load_row<4>(row + c, a.I - c, v);
            store(c, v);
        }
        if (lane == 0 && (wave & (wpp - 1)) == 0) hs[j] = fine ? (float)(m / 127.0) : __int_as_float(0x7fc00000);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++)
        if (lane < a.K) coef[wave * R + r][lane] = (double)wj * sd[r] * hs[lane];  // (read by this wave alone; in 64 bits as in scaled())
    if (row0 >= a.H) return;
    double acc[R];
#pragma unroll
    for (int r = 0; r < R; r++) acc[r] = (double)wj * b[r];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int i = lane + 64 * c;
        if (i < a.K * cpr) {
            const i32x4 x = *(const i32x4 *)(hq + 16 * i);
#pragma unroll
            for (int r = 0; r < R; r++) acc[r] = fma((double)dot16(w[r][c], x, 0), coef[wave * R + r][(picks[c / 4] >> (8 * (c % 4))) & 0xFF], acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const float v = (float)wave_sum_d(acc[r]);
        if (lane == 0 && row0 + r < a.H) ((T *)a.out)[(int64_t)t * a.H + row0 + r] = from_f32<T>(v);
    }
}

// ------------------------------------------------------------------------------ many tokens


// One block: the picks counted by expert in LDS, the experts' places and tiles from a scan, and the picks dealt out
// (their order within a pile does not matter: each pick's outputs are computed by themselves), through LDS up to
// I8_STAGED picks (scattered 4-byte stores from one CU cost a memory transaction each). 8,192 picks 6.2 us, 12,288 8.2, 12,800
// 17.1, 16,384 20.7. PER (a lane's logits) not 0: of up to I8_PLAN_TOKENS tokens, which its waves route first, every 16th token
// each: one launch less (9 tokens over 256 experts 9.8 -> 7 us; with more tokens the routing of a CU to each is faster).
constexpr int I8_STAGED = 12288;
template <int PER>
__global__ __launch_bounds__(1024) void k_i8_plan(I8MoeArgs a, int *pile_pick, int *pile_tok, I8Tile *tiles, int *n_tiles) {
    constexpr bool ROUTE = PER > 0;
    __shared__ int cnt[1024], place[1024], sums[2][16], staged[I8_STAGED];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, picks = a.T * a.K;
    cnt[tid] = 0;
    if constexpr (ROUTE) {
        int *expert = staged;  // (staged[] is filled after the last read of these)
        for (int t = wave; t < a.T; t += 16) {
            uint32_t id;
            float w;
            wave_route<PER>(a.logits + (int64_t)t * a.E, a.E, a.K, a.norm, &id, &w);
            if (lane < a.K) {
                a.ids[t * a.K + lane] = id;
                a.wt[t * a.K + lane] = w;
                expert[t * a.K + lane] = (int)id;
            }
        }
    }
    __syncthreads();
    constexpr int U = ROUTE ? 2 : 8;  // a thread's picks at a time (ROUTE: all of them)
    int e[U];
    auto load = [&](int p0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = min(p0 + 1024 * u + tid, picks - 1);
            e[u] = ROUTE ? staged[p] : (int)a.ids[p];
        }
    };
    for (int p0 = 0; p0 < picks; p0 += 1024 * U) {
        load(p0);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p0 + 1024 * u + tid < picks) atomicAdd(&cnt[e[u]], 1);
    }
    __syncthreads();
    const int c = cnt[tid], tc = (c + I8_TILE - 1) / I8_TILE;
    int ic = c, it = tc;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int uc = __shfl_up(ic, d), ut = __shfl_up(it, d);
        if (lane >= d) {
            ic += uc;
            it += ut;
        }
    }
    if (lane == 63) {
        sums[0][wave] = ic;
        sums[1][wave] = it;
    }
    __syncthreads();
    for (int w = 0; w < wave; w++) {
        ic += sums[0][w];
        it += sums[1][w];
    }
    place[tid] = ic - c;
    // (an expert's picks spread over its tiles evenly, in whole 16s)
    const int rows = tc ? ((c + tc - 1) / tc + 15) / 16 * 16 : 0;
    for (int q = 0; q < tc; q++) tiles[it - tc + q] = I8Tile{tid, ic - c + q * rows, min(rows, c - q * rows), it - tc, tc};
    if (tid == 1023) *n_tiles = it;
    __syncthreads();
    for (int p0 = 0; p0 < picks; p0 += 1024 * U) {
        if (!ROUTE && picks > 1024 * U) load(p0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = p0 + 1024 * u + tid;
            if (p >= picks) continue;
            const int at = atomicAdd(&place[e[u]], 1);
            if (picks <= I8_STAGED) {
                staged[at] = p;
            } else {
                pile_pick[at] = p;
                pile_tok[at] = p / a.K;
            }
        }
    }
    if (picks > I8_STAGED) return;
    __syncthreads();
    for (int at = tid; at < picks; at += 1024) {
        const int p = staged[at];
        pile_pick[at] = p;
        pile_tok[at] = p / a.K;
    }
}
// A wave's sums of gate (acc[i][j], j < NB) and up (acc[i][NB + j]): rows r0 + 16 i of the tile's picks, columns n0 + 16 j
// of the hidden row, which is stored in pile order, f32. (All loads before the bounds checks, from clamped places: inside
// them each would be waited for in turn.)
template <int MB, int NB>
__device__ __forceinline__ void finish_gateup(const I8MoeArgs &a, const I8Tile &tl, int r0, int n0, const i32x4 (&acc)[MB][2 * NB]) {
    const int lane = threadIdx.x & 63;
    float sw[2 * NB][4], b[2 * NB][4], sx[MB];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t n = (int64_t)tl.expert * a.I + min(n0 + 16 * (j % NB) + 4 * (lane >> 4) + i, a.I - 1);
            sw[j][i] = a.ws[j / NB][n];
            b[j][i] = a.bias[j / NB] ? a.bias[j / NB][n] : 0.f;
        }
#pragma unroll
    for (int mb = 0; mb < MB; mb++) sx[mb] = a.xs[a.pile_tok[tl.pos0 + min(r0 + 16 * mb + (lane & 15), tl.m - 1)]];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int r = r0 + 16 * mb + (lane & 15);
        if (r >= tl.m) continue;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int n = n0 + 16 * j + 4 * (lane >> 4);
            if (n >= a.I) continue;
            float h[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                h[i] = glu(scaled(acc[mb][j][i], (double)sx[mb] * sw[j][i], b[j][i]),
                           scaled(acc[mb][NB + j][i], (double)sx[mb] * sw[NB + j][i], b[NB + j][i]), a.glu);
            store_row<4>(a.h + (int64_t)(tl.pos0 + r) * a.ldh + n, a.I - n, h);
        }
    }
}
// The same of down: one row of H per pick, f32, in pick order.
template <int MB, int NW>
__device__ __forceinline__ void finish_down(const I8MoeArgs &a, const I8Tile &tl, int r0, int n0, const i32x4 (&acc)[MB][NW]) {
    const int lane = threadIdx.x & 63;
    float sw[NW][4], sx[MB];
    int picks[MB];
#pragma unroll
    for (int j = 0; j < NW; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) sw[j][i] = a.ws[2][(int64_t)tl.expert * a.H + min(n0 + 16 * j + 4 * (lane >> 4) + i, a.H - 1)];
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        const int p = tl.pos0 + min(r0 + 16 * mb + (lane & 15), tl.m - 1);
        sx[mb] = a.hs[p];
        picks[mb] = a.pile_pick[p];
    }
#pragma unroll
    for (int mb = 0; mb < MB; mb++) {
        if (r0 + 16 * mb + (lane & 15) >= tl.m) continue;
        float *d = a.dn + (int64_t)picks[mb] * a.H;
#pragma unroll
        for (int j = 0; j < NW; j++) {
            const int n = n0 + 16 * j + 4 * (lane >> 4);
            if (n >= a.H) continue;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = scaled(acc[mb][j][i], (double)sx[mb] * sw[j][i], 0.f);
            store_row<4>(d + n, a.H - n, v);
        }
    }
}

// The item of a block: blocks go to the eight dies in turn; each die takes a contiguous range of the items, an expert's
// blocks of W one after the other and its tiles side by side for each, so that an expert's picks and weights are read by
// one die and not by all, the weights once for all its tiles (2,048 tokens over 128 experts of 2,880 x 2,880: 2.2 GB
// fetched for gate and up, 2.4 with the tiles in block order).
__device__ __forceinline__ bool item_of_block(const I8MoeArgs &a, int n_blocks, I8Tile &tl, int &nb) {
    const int total = *a.n_tiles * n_blocks, die = blockIdx.x & 7, at = blockIdx.x >> 3, per = total >> 3, rest = total & 7;
    if (at >= per + (die < rest)) return false;
    const int item = die * per + min(die, rest) + at;
    const I8Tile any = a.tiles[__builtin_amdgcn_readfirstlane(item / n_blocks)];  // a tile of the item's expert
    const int in = item - any.first * n_blocks;
    nb = __builtin_amdgcn_readfirstlane(in / any.of);
    if (any.of == 1) tl = any;
    else tl = a.tiles[__builtin_amdgcn_readfirstlane(any.first + in - nb * any.of)];
    return true;
}

// A wave multiplies a tile's picks with 8 NW rows of gate and of up, or 16 NW of down. 2,048 tokens over 128 experts of
// 2,880 x 2,880: gate and up 492 us, down 257, 4.35 TB/s of weights, beside the f32 rows it writes (gate and up without
// their stores: 411). With many picks an expert its waves wait to issue: 61 % of their cycles over 8 experts of 2,048 x 4,096, at 42 %
// of the integer rate, L2 read at 6.7 TB/s.
template <bool DOWN, int MB, int NW>
__device__ __forceinline__ void stream_tile(const I8MoeArgs &a, const I8Tile &tl, int n0, uint8_t *lds) {
    constexpr int NB = NW / 2;
    const int lane = threadIdx.x & 63, rb = DOWN ? a.rbi : a.rbh;
    uint32_t wrow[NW];
    i32x4 acc[MB][NW];
    if constexpr (DOWN) {
        const uint8_t *w0[1] = {a.w[2] + (int64_t)tl.expert * a.stride[2]};
#pragma unroll
        for (int j = 0; j < NW; j++) wrow[j] = (uint32_t)min(n0 + 16 * j + (lane & 15), a.H - 1) * (uint32_t)rb + 16 * (lane >> 4);
        i8_loop<MB, NW, 1>(lds, a.hq + (int64_t)tl.pos0 * rb, [&](int r) { return (uint32_t)(min(r, tl.m - 1) * rb); }, w0, wrow, rb, acc);
        finish_down<MB, NW>(a, tl, 0, n0, acc);
    } else {
        const uint8_t *w0[2] = {a.w[0] + (int64_t)tl.expert * a.stride[0], a.w[1] + (int64_t)tl.expert * a.stride[1]};
#pragma unroll
        for (int j = 0; j < NW; j++) wrow[j] = (uint32_t)min(n0 + 16 * (j % NB) + (lane & 15), a.I - 1) * (uint32_t)rb + 16 * (lane >> 4);
        i8_loop<MB, NW, 2>(lds, a.x, [&](int r) { return (uint32_t)a.pile_tok[tl.pos0 + min(r, tl.m - 1)] * (uint32_t)rb; }, w0, wrow, rb, acc);
        finish_gateup<MB, NB>(a, tl, 0, n0, acc);
    }
}
template <bool DOWN, int NW>
__global__ __launch_bounds__(256, 2) void k_i8_moe_stream(I8MoeArgs a, int n_blocks) {
    extern __shared__ __align__(1024) uint8_t lds[];
    I8Tile tl;
    int nb;
    if (!item_of_block(a, n_blocks, tl, nb)) return;
    const int n0 = (DOWN ? 16 : 8) * NW * (4 * nb + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    if (tl.m <= 16) stream_tile<DOWN, 1, NW>(a, tl, n0, lds);
    else if (tl.m <= 32) stream_tile<DOWN, 2, NW>(a, tl, n0, lds);
    else if (tl.m <= 48) stream_tile<DOWN, 3, NW>(a, tl, n0, lds);
    else if (tl.m <= 64) stream_tile<DOWN, 4, NW>(a, tl, n0, lds);
    else if (tl.m <= 80) stream_tile<DOWN, 5, NW>(a, tl, n0, lds);
    else if (tl.m <= 96) stream_tile<DOWN, 6, NW>(a, tl, n0, lds);
    else stream_tile<DOWN, 8, NW>(a, tl, n0, lds);
}

// out[t] = sum_j w_j (dn_j + bias), in pick order; a thread per four columns (2,048 tokens of 4 picks, 2,880 columns:
// 106 MB in 23 us, 4.6 TB/s)
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

static I8MoeLayout layout(const cw_i8_moe_desc *d, int T) {
    I8MoeLayout L = {};
    size_t off = 0;
    auto take = [&](size_t &at, size_t bytes) { at = off; off = (off + bytes + 255) & ~(size_t)255; };
    const size_t TK = (size_t)T * d->top_k;
    L.few = i8_few_tokens(d->n_experts, d->top_k, d->hidden, d->inter, T);
    take(L.ids, TK * 4);
    take(L.w, TK * 4);
    take(L.h, TK * ((d->inter + 3) & ~3) * 4);
    if (!L.few) {
        take(L.tiles, (size_t)i8_max_tiles(TK, d->n_experts) * sizeof(I8Tile));
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
    // (a launch holds fewer than 2^32 threads; offsets of rows of x from its start are 32 bits)
    const int64_t blocks = i8_max_tiles((int64_t)T * d->top_k, d->n_experts) * std::max((d->inter + 63) / 64, (d->hidden + 127) / 128);
    if ((int64_t)T * d->top_k >= 1 << 28 || blocks >= 1 << 23 || (int64_t)T * i8_row_bytes(d->hidden) >= 1ll << 32)
        return set_error(CW_ENOTSUP, "i8 moe: %d tokens of %d picks, hidden %d, inter %d", T, d->top_k, d->hidden, d->inter);
    for (int m = 0; m < 3; m++) {
        const int64_t need = (m == 2 ? d->hidden : d->inter) * i8_row_bytes(m == 2 ? d->inter : d->hidden);
        CW_REQUIRE(d->w[m] && d->scale[m], "i8 moe: matrix %d is null", m);
        CW_REQUIRE(i8_aligned(d->w[m], 16) && d->slot_stride[m] % 16 == 0, "i8 moe: matrix %d must be 16-byte aligned", m);
        CW_REQUIRE(d->slot_stride[m] >= need, "i8 moe: matrix %d slot stride %lld below its %lld bytes", m, (long long)d->slot_stride[m],
                   (long long)need);
    }
    return CW_OK;
}

template <class T, int NC>
static int few_down(const I8MoeArgs &a, hipStream_t s) {
    const int r = i8_down_rows(NC, a.H, a.T, (int)resident_blocks(1));
    auto go = [&](auto kernel) {
        const int per = I8_FEW_WAVES * r;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.H + per - 1) / per), a.T), dim3(64 * I8_FEW_WAVES), a.K * a.rbi, s, a);
        return check_launch("k_i8_few_down");
    };
    if constexpr (NC <= 4)
        if (r == 4) return go(k_i8_few_down<T, NC, 4>);
    if constexpr (NC <= 8)
        if (r == 2) return go(k_i8_few_down<T, NC, 2>);
    return go(k_i8_few_down<T, NC, 1>);
}
template <class T>
static int few_down(const I8MoeArgs &a, hipStream_t s) {
    switch (i8_down_pieces(a.K, a.rbi)) {
    case 1: return few_down<T, 1>(a, s);
    case 2: return few_down<T, 2>(a, s);
    case 4: return few_down<T, 4>(a, s);
    case 8: return few_down<T, 8>(a, s);
    case 12: return few_down<T, 12>(a, s);
    default: return few_down<T, 16>(a, s);
    }
}
template <int PER, int NC>
static int few_gateup(const I8MoeArgs &a, hipStream_t s) {
    const int r = i8_gateup_rows(NC, a.I, a.T * a.K, (int)resident_blocks(1));
    auto go = [&](auto kernel) {
        const int per = I8_FEW_WAVES * r;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.I + per - 1) / per), a.K, a.T), dim3(64 * I8_FEW_WAVES), 0, s, a);
        return check_launch("k_i8_few_gateup");
    };
    if constexpr (NC <= 2)
        if (r == 4) return go(k_i8_few_gateup<PER, NC, 4>);
    return r == 2 ? go(k_i8_few_gateup<PER, NC, 2>) : go(k_i8_few_gateup<PER, NC, 1>);
}
template <int PER>
static int few_gateup(const I8MoeArgs &a, hipStream_t s) {
    switch (i8_gateup_pieces(a.rbh)) {
    case 1: return few_gateup<PER, 1>(a, s);
    case 2: return few_gateup<PER, 2>(a, s);
    case 3: return few_gateup<PER, 3>(a, s);
    default: return few_gateup<PER, 4>(a, s);
    }
}

static int moe_layer(const cw_i8_moe_desc *d, I8MoeArgs a, int ydtype, const I8MoeLayout &L, uint8_t *base, hipStream_t s) {
    int rc;
    if (L.few) {
        const int per = i8_route_width(a.E);
        rc = per == 4 ? few_gateup<4>(a, s) : per == 8 ? few_gateup<8>(a, s) : few_gateup<16>(a, s);
        if (rc) return rc;
        return ydtype == CW_F16 ? few_down<_Float16>(a, s) : ydtype == CW_BF16 ? few_down<bf16_t>(a, s) : few_down<float>(a, s);
    }
    const int TK = a.T * a.K, tmax = (int)i8_max_tiles(TK, a.E);
    int *pile_pick = (int *)(base + L.pile_pick), *pile_tok = (int *)(base + L.pile_tok), *n_tiles = (int *)(base + L.n_tiles);
    I8Tile *tiles = (I8Tile *)(base + L.tiles);
    auto plan = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(1), dim3(1024), 0, s, a, pile_pick, pile_tok, tiles, n_tiles);
        return check_launch("k_i8_plan");
    };
    if (a.T <= I8_PLAN_TOKENS) {
        const int per = i8_route_width(a.E);
        rc = per == 4 ? plan(k_i8_plan<4>) : per == 8 ? plan(k_i8_plan<8>) : plan(k_i8_plan<16>);
    } else {
        if ((rc = cw_route_topk(a.logits, a.T, a.E, a.K, a.norm, a.ids, a.wt, s))) return rc;
        rc = plan(k_i8_plan<0>);
    }
    if (rc) return rc;
    int8_t *hq = (int8_t *)(base + L.hq);
    float *hs = (float *)(base + L.hs);
    a.tiles = tiles;
    a.n_tiles = n_tiles;
    a.pile_pick = pile_pick;
    a.pile_tok = pile_tok;
    a.hq = (const uint8_t *)hq;
    a.hs = hs;
    a.dn = (float *)(base + L.dn);
    constexpr int LDS = I8Stage<I8_TILE / 16, 2>::LDS;
    auto product = [&](auto kernel, int nw, bool down) {
        const int cols = (down ? 64 : 32) * nw, blocks = ((down ? a.H : a.I) + cols - 1) / cols;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((tmax * blocks + 7) / 8 * 8)), dim3(256), LDS, s, a, blocks);
        return check_launch("k_i8_moe_stream");
    };
    const bool many = i8_many_picks(a.E, a.K, a.I, a.T, (int)resident_blocks(1));
    rc = many ? product(k_i8_moe_stream<false, 4>, 4, false) : product(k_i8_moe_stream<false, 2>, 2, false);
    if (rc) return rc;
    if ((rc = i8_quantize_f32(a.h, TK, a.I, a.ldh, hq, hs, s))) return rc;
    rc = many ? product(k_i8_moe_stream<true, 4>, 4, true) : product(k_i8_moe_stream<true, 2>, 2, true);
    if (rc) return rc;
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
    a.glu = glu_of(d->act, d->alpha, d->limit);
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
