// Tokens sorted by expert and back, with weights applied, and the gradients of both (gfx950).
#include <atomic>

#include "cw_piles.h"
#include "cw_i8_dev.h"
#include "cw_mfma.h"

namespace cw {

// ------------------------------------------------------------------------------ the sort

struct SortArgs {
    const int *ids;
    int picks, experts;  // expert `experts`: none
    int chunk, bits;     // picks of a block (a multiple of SORT_ROUND); bits of an expert's number
    int *order, *place, *offsets;
    int *n_tiles;
    PileTile *tiles;
    int *counts;  // chunks x (experts + 1), or NULL: every block counts the other chunks itself
};
constexpr int SORT_WAVES = 16, SORT_PER = 8, SORT_ROUND = 64 * SORT_WAVES * SORT_PER;
constexpr int sort_lds(int experts) { return 4 * (PILE_MAX_EXPERTS + 4 + SORT_WAVES * (experts + 1)); }
constexpr int SORT_MAX_LDS = sort_lds(PILE_MAX_EXPERTS);

__device__ __forceinline__ int expert_of(const SortArgs &a, int p) {
    const uint32_t e = (uint32_t)a.ids[p];
    return e < (uint32_t)a.experts ? (int)e : a.experts;
}
// the lanes of the wave whose expert is this lane's (both of `bits` bits); lanes that are not in: none
__device__ __forceinline__ uint64_t same_expert(int e, int bits, bool in) {
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; b++) {
        const bool set = (e >> b) & 1;
        const uint64_t v = __ballot(set);
        m &= set ? v : ~v;
    }
    return m;
}

// counts[chunk][e] of many picks
__global__ __launch_bounds__(1024) void k_pile_counts(SortArgs a) {
    __shared__ int cnt[PILE_MAX_EXPERTS + 1];
    for (int e = threadIdx.x; e <= a.experts; e += 1024) cnt[e] = 0;
    __syncthreads();
    const int p0 = blockIdx.x * a.chunk, p1 = min(a.picks, p0 + a.chunk);
    for (int p = p0 + threadIdx.x; p < p1; p += 1024) atomicAdd(&cnt[expert_of(a, p)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += 1024) a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = cnt[e];
}

// A stable counting sort, a block to a chunk of picks. The block counts all picks by expert, and those before its chunk (integer
// counts: the order of the atomics does not show); a scan over the experts gives each its first position. Then the chunk in
// rounds of 8,192, a wave's picks neighbours: a wave's lanes with the same expert find one another by ballots over the bits of its
// number, a pick's rank is the count of its expert so far in the wave's part plus the lanes before it, and the waves' counts are
// summed in their order. Nothing depends on timing. The first block writes the
// offsets, the blocks in turn the tiles.
__global__ __launch_bounds__(1024) void k_pile_sort(SortArgs a) {
    extern __shared__ int lds[];  // next position of each expert, then the waves' counts of a round
    __shared__ int sums[2][16];
    int *next = lds, *total = lds + (PILE_MAX_EXPERTS + 4), *mine = total;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E1 = a.experts + 1;
    const int c0 = blockIdx.x * a.chunk, c1 = min(a.picks, c0 + a.chunk);
    for (int e = tid; e < E1; e += 1024) next[e] = total[e] = 0;
    __syncthreads();
    if (a.counts) {
        for (int e = tid; e < E1; e += 1024) {
            int before = 0, all = 0;
            for (int c = 0; c < (int)gridDim.x; c++) {
                const int v = a.counts[(int64_t)c * E1 + e];
                before += c < (int)blockIdx.x ? v : 0;
                all += v;
            }
            next[e] = before;
            total[e] = all;
        }
    } else {
        for (int p = tid; p < a.picks; p += 1024) {
            const int e = expert_of(a, p);
            atomicAdd(&total[e], 1);
            if (p < c0) atomicAdd(&next[e], 1);
        }
    }
    __syncthreads();
    // exclusive sums over the experts of their picks and tiles, a thread an expert (expert 1,024, none, by the last thread besides)
    const int c = tid < E1 ? total[tid] : 0, tc = (c + PILE_TILE - 1) / PILE_TILE;
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
    auto place_expert = [&](int e, int from, int count, int first, int tiles) {
        next[e] += from;
        if (blockIdx.x == 0) a.offsets[e] = from;
        // (an expert's picks spread over its tiles evenly, in whole 16s)
        const int rows = tiles ? ((count + tiles - 1) / tiles + 15) / 16 * 16 : 0;
        for (int q = blockIdx.x; q < tiles; q += gridDim.x) a.tiles[first + q] = PileTile{e, from + q * rows, min(rows, count - q * rows), first, tiles};
    };
    if (tid < E1) place_expert(tid, ic - c, c, it - tc, tc);
    if (tid == 1023) {
        if (E1 > 1024) {
            const int count = total[1024], tiles = (count + PILE_TILE - 1) / PILE_TILE;
            place_expert(1024, ic, count, it, tiles);
            it += tiles;
        }
        if (blockIdx.x == 0) *a.n_tiles = it;
    }
    for (int r0 = c0; r0 < c1; r0 += SORT_ROUND) {
        __syncthreads();  // (the totals, and the last round's counts, have been read)
        for (int i = tid; i < SORT_WAVES * E1; i += 1024) mine[i] = 0;
        __syncthreads();
        volatile int *own = mine + wave * E1;  // (a wave's reads and writes of LDS are in order; the compiler keeps them so)
        int e[SORT_PER], rank[SORT_PER];
#pragma unroll
        for (int i = 0; i < SORT_PER; i++) {
            const int p = r0 + 64 * (SORT_PER * wave + i) + lane;
            e[i] = p < c1 ? expert_of(a, p) : -1;
        }
#pragma unroll
        for (int i = 0; i < SORT_PER; i++) {
            const uint64_t m = same_expert(e[i], a.bits, e[i] >= 0);
            if (e[i] >= 0) {
                const uint64_t below = m & ((1ull << lane) - 1);
                const int before = own[e[i]];
                rank[i] = before + __popcll(below);
                if (!below) own[e[i]] = before + __popcll(m);
            }
        }
        __syncthreads();
        for (int x = tid; x < E1; x += 1024) {
            int at = next[x];
            for (int w = 0; w < SORT_WAVES; w++) {
                const int n = mine[w * E1 + x];
                mine[w * E1 + x] = at;
                at += n;
            }
            next[x] = at;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SORT_PER; i++) {
            if (e[i] < 0) continue;
            const int p = r0 + 64 * (SORT_PER * wave + i) + lane, at = own[e[i]] + rank[i];
            a.place[p] = at;
            a.order[at] = p;
        }
    }
}

// ------------------------------------------------------------------------------ the rows

struct PileArgs {
    const void *x, *y;
    int64_t ldx, ldy;
    const int *place, *offsets;
    const float *w;
    int T, K, E, h;
    int per;  // pieces of 8 elements of a row
    void *out;
    float *dw;
};

template <class R>
struct Raw8 {
    R v[8];
};
// 8 elements as they are, at any address of their type; of a row's last piece the `valid` ones
template <class R>
__device__ __forceinline__ Raw8<R> load_raw(const R *p, int valid) {
    Raw8<R> t;
    if (valid >= 8) {
        memcpy(&t, p, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) t.v[i] = i < valid ? p[i] : R(0);
    }
    return t;
}
template <class R>
__device__ __forceinline__ void store_raw(R *p, int valid, const Raw8<R> &t) {
    if (valid >= 8) {
        memcpy(p, &t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < valid) p[i] = t.v[i];
    }
}

// out[place[t][j]] = x[t]: a thread reads a piece of a token once and writes it K times; rows of picks of no expert are zeros
template <class R>
__global__ __launch_bounds__(256) void k_to_piles(PileArgs a) {
    const int here = a.offsets[a.E];
    const int64_t n = (int64_t)a.T * a.per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)((uint64_t)i / (uint32_t)a.per), e = 8 * (int)(i - (int64_t)t * a.per), valid = a.h - e;
        const Raw8<R> v = load_raw((const R *)a.x + t * a.ldx + e, valid);
        const int *at = a.place + (int64_t)t * a.K;
        for (int j = 0; j < a.K; j++) {
            const int pos = at[j];
            store_raw((R *)a.out + (int64_t)pos * a.h + e, valid, pos < here ? v : Raw8<R>{});
        }
    }
}

// out[t] = sum_j w[t][j] y[place[t][j]] (w NULL: 1), in pick order, in f32, rounded once; picks of no expert add nothing, whatever
// their rows hold
template <class T, class O, bool WEIGHTS>
__global__ __launch_bounds__(256) void k_from_piles(PileArgs a) {
    const int here = a.offsets[a.E];
    const int64_t n = (int64_t)a.T * a.per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)((uint64_t)i / (uint32_t)a.per), e = 8 * (int)(i - (int64_t)t * a.per), valid = a.h - e;
        const int64_t p0 = (int64_t)t * a.K;
        float acc[8] = {};
        for (int j = 0; j < a.K; j++) {
            const int pos = a.place[p0 + j];
            if (pos >= here) continue;
            float v[8];
            load_row<8>((const T *)a.y + (int64_t)pos * a.ldy + e, valid, v);
            if constexpr (WEIGHTS) {
                const float w = a.w[p0 + j];
#pragma unroll
                for (int c = 0; c < 8; c++) acc[c] = fmaf(w, v[c], acc[c]);
            } else {
#pragma unroll
                for (int c = 0; c < 8; c++) acc[c] += v[c];
            }
        }
        store_row<8>((O *)a.out + (int64_t)t * a.h + e, valid, acc);
    }
}

// A wave a pick: dy = w x[t] (x: the gradient of the tokens' output) into its position, dw = <x[t], y>. The picks of a token are
// neighbours, so that its row comes from the caches after the first.
template <class T>
__global__ __launch_bounds__(256) void k_from_piles_grad(PileArgs a) {
    const int here = a.offsets[a.E], lane = threadIdx.x & 63;
    const int64_t p = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (p >= (int64_t)a.T * a.K) return;
    const int pos = a.place[p];
    const bool in = pos < here;
    const float w = a.w[p];
    const T *x = (const T *)a.x + p / a.K * a.ldx, *y = (const T *)a.y + (int64_t)pos * a.ldy;
    T *out = (T *)a.out + (int64_t)pos * a.h;
    float dot = 0.f;
    for (int e = 8 * lane; e < a.h; e += 512) {
        float g[8] = {}, v[8];
        const int valid = a.h - e;
        if (in) {
            load_row<8>(x + e, valid, g);
            load_row<8>(y + e, valid, v);
#pragma unroll
            for (int c = 0; c < 8; c++) {
                dot = fmaf(g[c], v[c], dot);
                g[c] *= w;
            }
        }
        store_row<8>(out + e, valid, g);
    }
    dot = wave_sum(dot);
    if (lane == 0) a.dw[p] = dot;
}

static int check_piles(const char *what, int dtype, int64_t T, int K, int E, int64_t h) {
    if (dtype != CW_F32 && dtype != CW_F16 && dtype != CW_BF16) return set_error(CW_ENOTSUP, "%s: type %d (f32, f16 or bf16)", what, dtype);
    CW_REQUIRE(T >= 0 && K > 0 && h > 0 && h < 1ll << 31, "%s: %lld tokens of %d picks, rows of %lld", what, (long long)T, K, (long long)h);
    CW_REQUIRE(E > 0 && E <= PILE_MAX_EXPERTS, "%s: %d experts (1..%d supported)", what, E, PILE_MAX_EXPERTS);
    if (K > 1 << 20 || T >= 1 << 28 || T * K >= 1 << 28) return set_error(CW_ENOTSUP, "%s: %lld tokens of %d picks", what, (long long)T, K);
    return CW_OK;
}
static PileArgs pile_args(const int *place, const int *offsets, int64_t T, int K, int E, int64_t h) {
    PileArgs a = {};
    a.place = place;
    a.offsets = offsets;
    a.T = (int)T;
    a.K = K;
    a.E = E;
    a.h = (int)h;
    a.per = (int)((h + 7) / 8);
    return a;
}
static dim3 piece_grid(const PileArgs &a) { return dim3((unsigned)std::min<int64_t>(((int64_t)a.T * a.per + 255) / 256, 1 << 20)); }

template <class R>
static int to_piles(const PileArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(k_to_piles<R>, piece_grid(a), dim3(256), 0, s, a);
    return check_launch("k_to_piles");
}
template <class T, class O>
static int from_piles(const PileArgs &a, hipStream_t s) {
    if (a.w) hipLaunchKernelGGL((k_from_piles<T, O, true>), piece_grid(a), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_from_piles<T, O, false>), piece_grid(a), dim3(256), 0, s, a);
    return check_launch("k_from_piles");
}
int from_piles_f32(int dtype, const float *rows, const float *w, int64_t T, int K, int E, int64_t h, const int *place, const int *offsets, void *out,
                   hipStream_t s) {
    PileArgs a = pile_args(place, offsets, T, K, E, h);
    a.y = rows;
    a.ldy = h;
    a.w = w;
    a.out = out;
    return dtype == CW_F16 ? from_piles<float, _Float16>(a, s) : dtype == CW_BF16 ? from_piles<float, bf16_t>(a, s) : from_piles<float, float>(a, s);
}
template <class T>
static int from_piles_grad(const PileArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(k_from_piles_grad<T>, dim3((unsigned)(((int64_t)a.T * a.K + 3) / 4)), dim3(256), 0, s, a);
    return check_launch("k_from_piles_grad");
}

// dynamic LDS above 64 KB, opted into once per device
static int sort_allow_lds(int lds) {
    static std::atomic<bool> set[MAX_DEVICES];
    const int dev = current_device();
    if (lds <= 65536 - 512 || set[dev].load(std::memory_order_relaxed)) return CW_OK;
    if (hipFuncSetAttribute((const void *)k_pile_sort, hipFuncAttributeMaxDynamicSharedMemorySize, SORT_MAX_LDS) != hipSuccess)
        return set_error(CW_EHIP, "sort_picks: %d bytes of LDS", lds);
    set[dev].store(true, std::memory_order_relaxed);
    return CW_OK;
}
// chunks of the sort: 8,192 picks each, or more where there would be more than 256 of them
static int sort_chunk(int64_t picks) {
    const int64_t rounds = (picks + SORT_ROUND - 1) / SORT_ROUND;
    return (int)((rounds + 255) / 256 * SORT_ROUND);
}
// Above this the chunks are counted by a launch of their own instead of by every block.
constexpr int64_t SORT_RECOUNT = 1 << 16;
static int64_t sort_chunks(int64_t picks) { return (picks + sort_chunk(picks) - 1) / sort_chunk(picks); }

static int check_sort(int64_t picks, int E) {
    CW_REQUIRE(picks >= 0, "sort_picks: %lld picks", (long long)picks);
    CW_REQUIRE(E > 0 && E <= PILE_MAX_EXPERTS, "sort_picks: %d experts (1..%d supported)", E, PILE_MAX_EXPERTS);
    if (picks >= 1 << 28) return set_error(CW_ENOTSUP, "sort_picks: %lld picks", (long long)picks);
    return CW_OK;
}

}  // namespace cw

using namespace cw;

extern "C" {

int64_t cw_pile_tiles_bytes(int64_t picks, int n_experts) {
    return check_sort(picks, n_experts) ? 0 : pile_tiles_bytes(picks, n_experts);
}
size_t cw_sort_picks_workspace_size(int64_t picks, int n_experts) {
    return check_sort(picks, n_experts) || picks <= SORT_RECOUNT ? 0 : (size_t)(sort_chunks(picks) * (n_experts + 1) * 4);
}

int cw_sort_picks(const uint32_t *ids, int64_t picks, int n_experts, int32_t *order, int32_t *place, int32_t *offsets, void *tiles, void *ws,
                  size_t ws_bytes, cw_stream_t stream) {
    if (int rc = check_sort(picks, n_experts)) return rc;
    CW_REQUIRE(offsets && tiles && (picks == 0 || (ids && order && place)), "sort_picks: null pointer");
    CW_REQUIRE(((uintptr_t)tiles & 15) == 0, "sort_picks: tiles must be 16-byte aligned");
    const size_t need = cw_sort_picks_workspace_size(picks, n_experts);
    CW_REQUIRE(need == 0 || (ws && ws_bytes >= need), "sort_picks: workspace of %zu bytes, %zu needed", ws_bytes, need);
    SortArgs a = {};
    a.ids = (const int *)ids;
    a.picks = (int)picks;
    a.experts = n_experts;
    a.chunk = picks ? sort_chunk(picks) : SORT_ROUND;
    for (a.bits = 1; n_experts >> a.bits; a.bits++) {}
    a.order = order;
    a.place = place;
    a.offsets = offsets;
    a.n_tiles = (int *)tiles;
    a.tiles = (PileTile *)pile_tiles(tiles);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)(picks ? sort_chunks(picks) : 1));
    if (need) {
        a.counts = (int *)ws;
        hipLaunchKernelGGL(k_pile_counts, grid, dim3(1024), 0, s, a);
        if (int rc = check_launch("k_pile_counts")) return rc;
    }
    const int lds = sort_lds(n_experts);
    if (int rc = sort_allow_lds(lds)) return rc;
    hipLaunchKernelGGL(k_pile_sort, grid, dim3(1024), lds, s, a);
    return check_launch("k_pile_sort");
}

int cw_to_piles(int dtype, const void *x, int64_t ldx, int64_t T, int K, int n_experts, int64_t h, const int32_t *place, const int32_t *offsets,
                void *rows, cw_stream_t stream) {
    if (int rc = check_piles("to_piles", dtype, T, K, n_experts, h)) return rc;
    if (T == 0) return CW_OK;
    CW_REQUIRE(x && place && offsets && rows && ldx >= h, "to_piles: null pointer, or rows of %lld %lld apart", (long long)h, (long long)ldx);
    PileArgs a = pile_args(place, offsets, T, K, n_experts, h);
    a.x = x;
    a.ldx = ldx;
    a.out = rows;
    return dtype == CW_F32 ? to_piles<uint32_t>(a, (hipStream_t)stream) : to_piles<uint16_t>(a, (hipStream_t)stream);
}

int cw_from_piles(int dtype, const void *rows, int64_t ldr, const float *w, int64_t T, int K, int n_experts, int64_t h, const int32_t *place,
                  const int32_t *offsets, void *out, cw_stream_t stream) {
    if (int rc = check_piles("from_piles", dtype, T, K, n_experts, h)) return rc;
    if (T == 0) return CW_OK;
    CW_REQUIRE(rows && place && offsets && out && ldr >= h, "from_piles: null pointer, or rows of %lld %lld apart", (long long)h, (long long)ldr);
    PileArgs a = pile_args(place, offsets, T, K, n_experts, h);
    a.y = rows;
    a.ldy = ldr;
    a.w = w;
    a.out = out;
    hipStream_t s = (hipStream_t)stream;
    return dtype == CW_F16 ? from_piles<_Float16, _Float16>(a, s) : dtype == CW_BF16 ? from_piles<bf16_t, bf16_t>(a, s) : from_piles<float, float>(a, s);
}

int cw_from_piles_grad(int dtype, const void *dout, int64_t ldd, const void *rows, int64_t ldr, const float *w, int64_t T, int K, int n_experts,
                       int64_t h, const int32_t *place, const int32_t *offsets, void *drows, float *dw, cw_stream_t stream) {
    if (int rc = check_piles("from_piles_grad", dtype, T, K, n_experts, h)) return rc;
    if (T == 0) return CW_OK;
    CW_REQUIRE(dout && rows && w && place && offsets && drows && dw, "from_piles_grad: null pointer");
    CW_REQUIRE(ldd >= h && ldr >= h, "from_piles_grad: rows of %lld %lld and %lld apart", (long long)h, (long long)ldd, (long long)ldr);
    PileArgs a = pile_args(place, offsets, T, K, n_experts, h);
    a.x = dout;
    a.ldx = ldd;
    a.y = rows;
    a.ldy = ldr;
    a.w = w;
    a.out = drows;
    a.dw = dw;
    hipStream_t s = (hipStream_t)stream;
    return dtype == CW_F16 ? from_piles_grad<_Float16>(a, s) : dtype == CW_BF16 ? from_piles_grad<bf16_t>(a, s) : from_piles_grad<float>(a, s);
}

}  // extern "C"
