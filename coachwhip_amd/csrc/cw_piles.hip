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
    int chunk, bits;     // picks of a block; bits of an expert's number
    int *order, *place, *offsets;
    int *n_tiles;
    PileTile *tiles;
    int *counts;  // of more than one chunk: chunks x (experts + 1)
};
constexpr int SORT_WAVES = 16, SORT_THREADS = 64 * SORT_WAVES;
constexpr int sort_lds(int experts) { return 4 * (PILE_MAX_EXPERTS + 4 + SORT_WAVES * (experts + 1)); }
constexpr int SORT_MAX_LDS = sort_lds(PILE_MAX_EXPERTS);

__device__ __forceinline__ int expert_of(const SortArgs &a, int p) {
    const uint32_t e = (uint32_t)a.ids[p];
    return e < (uint32_t)a.experts ? (int)e : a.experts;
}
// the lanes of the wave whose expert is this lane's, of those that are in
__device__ __forceinline__ uint64_t same_expert(int e, int bits, bool in) {
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; b++) {
        const bool set = (e >> b) & 1;
        const uint64_t v = __ballot(set);
        m &= set ? v : ~v;
    }
    return m;
}

// counts[chunk][e]: a wave adds for each expert once, however many of its lanes have it
__global__ __launch_bounds__(SORT_THREADS) void k_pile_counts(SortArgs a) {
    __shared__ int cnt[PILE_MAX_EXPERTS + 1];
    const int lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e <= a.experts; e += SORT_THREADS) cnt[e] = 0;
    __syncthreads();
    const int p0 = blockIdx.x * a.chunk, p1 = min(a.picks, p0 + a.chunk);
    for (int p = p0 + threadIdx.x; p - lane < p1; p += SORT_THREADS) {
        const int e = p < p1 ? expert_of(a, p) : 0;
        const uint64_t m = same_expert(e, a.bits, p < p1);
        if (p < p1 && !(m & ((1ull << lane) - 1))) atomicAdd(&cnt[e], __popcll(m));
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += SORT_THREADS) a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = cnt[e];
}

// A stable counting sort, a block to a chunk of picks, in rounds of 1,024 PER, a wave's picks neighbours: a wave's lanes with the same
// expert find one another by ballots over the bits of its number, a pick's rank is the count of its expert so far in the wave's
// part plus the lanes before it, and the waves' counts are summed in their order. The experts' first positions come from a scan
// over all picks' counts: this round's where it is all there is, else those of the chunks, of which the ones before this add
// to its own. 65,536 picks of 256 experts: 7.4 us, and 5.0 to count them; 64: 4.8.
// Nothing depends on timing, nor on how the picks are spread. The first block writes the offsets, the blocks in turn the tiles.
template <int PER>
__global__ __launch_bounds__(SORT_THREADS) void k_pile_sort(SortArgs a) {
    extern __shared__ int lds[];  // next position of each expert, then the waves' counts and places of a round
    __shared__ int sums[2][SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E1 = a.experts + 1;
    int *next = lds, *mine = lds + PILE_MAX_EXPERTS + 4;
    volatile int *own = mine + wave * E1;  // (a wave's reads and writes of LDS are in order; the compiler keeps them so)
    const int c0 = blockIdx.x * a.chunk, c1 = min(a.picks, c0 + a.chunk);
    int e[PER], rank[PER];
    auto rank_round = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int p = r0 + 64 * (PER * wave + i) + lane;
            e[i] = p < c1 ? expert_of(a, p) : -1;
        }
        for (int i = tid; i < SORT_WAVES * E1; i += SORT_THREADS) mine[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint64_t m = same_expert(e[i], a.bits, e[i] >= 0);
            if (e[i] < 0) continue;
            const uint64_t below = m & ((1ull << lane) - 1);
            const int before = own[e[i]];
            rank[i] = before + __popcll(below);
            if (!below) own[e[i]] = before + __popcll(m);
        }
        __syncthreads();
    };
    // the waves' counts of expert x become the places of their first picks, from `at` on; the place after the last
    auto place_waves = [&](int x, int at, const int (&n)[SORT_WAVES]) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < SORT_WAVES; w++) {
            mine[w * E1 + x] = at;
            at += n[w];
        }
        next[x] = at;
    };
    auto waves_of = [&](int x, int (&n)[SORT_WAVES]) __attribute__((always_inline)) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; w++) {
            n[w] = mine[w * E1 + x];
            sum += n[w];
        }
        return sum;
    };
    auto write_round = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (e[i] < 0) continue;
            const int p = r0 + 64 * (PER * wave + i) + lane, at = own[e[i]] + rank[i];
            a.place[p] = at;
            a.order[at] = p;
        }
    };
    rank_round(c0);
    // an expert's waves in this round, its picks in all and in the chunks before
    auto count = [&](int x, int (&n)[SORT_WAVES], int &before) __attribute__((always_inline)) {
        int all = waves_of(x, n);
        before = 0;
        if (a.counts) {
            all = 0;
#pragma unroll 8
            for (int c = 0; c < (int)gridDim.x; c++) {
                const int v = a.counts[(int64_t)c * E1 + x];
                before += c < (int)blockIdx.x ? v : 0;
                all += v;
            }
        }
        return all;
    };
    auto settle = [&](int x, int from, int all, int first, int tiles, int before, const int (&n)[SORT_WAVES]) __attribute__((always_inline)) {
        place_waves(x, from + before, n);
        if (blockIdx.x == 0) a.offsets[x] = from;
        // (an expert's picks spread over its tiles evenly, in whole 16s)
        const int rows = tiles ? ((all + tiles - 1) / tiles + 15) / 16 * 16 : 0;
        for (int q = blockIdx.x; q < tiles; q += gridDim.x) a.tiles[first + q] = PileTile{x, from + q * rows, min(rows, all - q * rows), first, tiles};
    };
    // exclusive sums over the experts of their picks and tiles, a thread an expert (number 1,024, none of 1,024, by the last besides)
    int n[SORT_WAVES], before, c = 0;
    if (tid < E1) c = count(tid, n, before);
    const int tc = (c + PILE_TILE - 1) / PILE_TILE;
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
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) {
        ic += w < wave ? sums[0][w] : 0;
        it += w < wave ? sums[1][w] : 0;
    }
    if (tid < E1) settle(tid, ic - c, c, it - tc, tc, before, n);
    if (tid == SORT_THREADS - 1) {
        if (E1 > SORT_THREADS) {
            const int all = count(SORT_THREADS, n, before), tiles = (all + PILE_TILE - 1) / PILE_TILE;
            settle(SORT_THREADS, ic, all, it, tiles, before, n);
            it += tiles;
        }
        if (blockIdx.x == 0) *a.n_tiles = it;
    }
    __syncthreads();
    write_round(c0);
    for (int r0 = c0 + SORT_THREADS * PER; r0 < c1; r0 += SORT_THREADS * PER) {
        __syncthreads();  // (the last round's places have been read)
        rank_round(r0);
        if (tid < E1) {
            waves_of(tid, n);
            place_waves(tid, next[tid], n);
        }
        if (E1 > SORT_THREADS && tid == SORT_THREADS - 1) {
            waves_of(SORT_THREADS, n);
            place_waves(SORT_THREADS, next[SORT_THREADS], n);
        }
        __syncthreads();
        write_round(r0);
    }
}

// ------------------------------------------------------------------------------ the rows

struct PileArgs {
    const void *x, *y;
    int64_t ldx, ldy;
    const int *order, *place, *offsets;  // (order or place)
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

// out[pos] = x[order[pos] / K], zeros at positions of no expert: a thread a piece of a position, in the order in which they are written;
// a token's row comes from the caches after the first of its picks (8,192 tokens of 8 picks, half of no expert, 2,048 bf16 values: 60 us, 5.0
// TB/s; each token's row read once and scattered to its K positions: 83; the same for 4 picks of 4,095 tokens of 2,880, 29 us).
template <class R>
__global__ __launch_bounds__(256) void k_to_piles(PileArgs a) {
    const int here = a.offsets[a.E];
    const int64_t n = (int64_t)a.T * a.K * a.per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int pos = (int)((uint64_t)i / (uint32_t)a.per), e = 8 * (int)(i - (int64_t)pos * a.per), valid = a.h - e;
        Raw8<R> v = {};
        if (pos < here) v = load_raw((const R *)a.x + a.order[pos] / a.K * a.ldx + e, valid);
        store_raw((R *)a.out + (int64_t)pos * a.h + e, valid, v);
    }
}

// out[t] = sum_j w[t][j] y[place[t][j]] (w NULL: 1), in pick order, in f32, rounded once; picks of no expert add nothing, whatever
// their rows hold (8,192 tokens of 8 picks, half of no expert, 2,048 bf16 values: 54 us, 3.1 TB/s, 87 % of the waves'
// cycles waits for the places and then the rows; 31 with the rows in the caches)
template <class T, class O, bool WEIGHTS>
__global__ __launch_bounds__(256) void k_from_piles(PileArgs a) {
    const int here = a.offsets[a.E];
    const int64_t n = (int64_t)a.T * a.per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)((uint64_t)i / (uint32_t)a.per), e = 8 * (int)(i - (int64_t)t * a.per), valid = a.h - e;
        const int64_t p0 = (int64_t)t * a.K;
        float acc[8] = {};
        // four picks at a time, their loads together (a pick of no expert: any row, not used)
        for (int j0 = 0; j0 < a.K; j0 += 4) {
            float v[4][8], w[4];
            int pos[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = min(j0 + u, a.K - 1);
                pos[u] = a.place[p0 + j];
                w[u] = WEIGHTS ? a.w[p0 + j] : 1.f;
                if (j0 + u >= a.K) pos[u] = here;
            }
#pragma unroll
            for (int u = 0; u < 4; u++) load_row<8>((const T *)a.y + (int64_t)min(pos[u], max(here - 1, 0)) * a.ldy + e, valid, v[u]);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (pos[u] < here)
#pragma unroll
                    for (int c = 0; c < 8; c++) acc[c] = fmaf(w[u], v[u][c], acc[c]);
        }
        store_row<8>((O *)a.out + (int64_t)t * a.h + e, valid, acc);
    }
}

// A wave a pick: dy = w x[t] (x: the gradient of the tokens' output) into its position, dw = <x[t], y>. The picks of a token are a
// block's neighbours: its row comes from the caches after the first (4,095 tokens of 4 picks, 2,880 bf16 values: 42 us over sets of inputs in turn, 5.0 TB/s. In a graph on
// one set, which the caches hold in part: 35; a wave a position, whose long rows are then read and written in order: 44; 8,192 of 8, half of no expert, 91 and 88).
template <class T>
__global__ __launch_bounds__(256) void k_from_piles_grad(PileArgs a) {
    const int here = a.offsets[a.E], lane = threadIdx.x & 63;
    for (int64_t p = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); p < (int64_t)a.T * a.K; p += 4 * (int64_t)gridDim.x) {
        const int64_t pos = a.place[p];
        const bool in = pos < here;
        const float w = a.w[p];
        const T *x = (const T *)a.x + p / a.K * a.ldx, *y = (const T *)a.y + pos * a.ldy;
        T *out = (T *)a.out + pos * a.h;
        float dot = 0.f;
        for (uint32_t e = 8 * lane; e < (uint32_t)a.h; e += 512) {  // (a row may have 2^31 - 1 values: the last step passes that)
            float g[8] = {}, v[8];
            const int valid = a.h - (int)e;
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
}

static int check_piles(const char *what, int dtype, int64_t T, int K, int E, int64_t h) {
    if (dtype != CW_F32 && dtype != CW_F16 && dtype != CW_BF16) return set_error(CW_ENOTSUP, "%s: type %d (f32, f16 or bf16)", what, dtype);
    CW_REQUIRE(T >= 0 && K > 0 && h > 0 && h < 1ll << 31, "%s: %lld tokens of %d picks, rows of %lld", what, (long long)T, K, (long long)h);
    CW_REQUIRE(E > 0 && E <= PILE_MAX_EXPERTS, "%s: %d experts (1..%d supported)", what, E, PILE_MAX_EXPERTS);
    if (K > 1 << 20 || T >= 1 << 28 || T * K >= 1 << 28) return set_error(CW_ENOTSUP, "%s: %lld tokens of %d picks", what, (long long)T, K);
    return CW_OK;
}
static PileArgs pile_args(const int *order, const int *place, const int *offsets, int64_t T, int K, int E, int64_t h) {
    PileArgs a = {};
    a.order = order;
    a.place = place;
    a.offsets = offsets;
    a.T = (int)T;
    a.K = K;
    a.E = E;
    a.h = (int)h;
    a.per = (int)((h + 7) / 8);
    return a;
}
// (a launch holds fewer than 2^32 threads)
static dim3 piece_grid(const PileArgs &a, int64_t rows) { return dim3((unsigned)std::min<int64_t>((rows * a.per + 255) / 256, 1 << 22)); }

template <class R>
static int to_piles(const PileArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(k_to_piles<R>, piece_grid(a, (int64_t)a.T * a.K), dim3(256), 0, s, a);
    return check_launch("k_to_piles");
}
template <class T, class O, bool WEIGHTS>
static int from_piles(const PileArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((k_from_piles<T, O, WEIGHTS>), piece_grid(a, a.T), dim3(256), 0, s, a);
    return check_launch("k_from_piles");
}
template <class T>
static int from_piles(const PileArgs &a, hipStream_t s) {
    return a.w ? from_piles<T, T, true>(a, s) : from_piles<T, T, false>(a, s);
}
int from_piles_f32(int dtype, const float *rows, const float *w, int64_t T, int K, int E, int64_t h, const int *place, const int *offsets, void *out,
                   hipStream_t s) {
    PileArgs a = pile_args(nullptr, place, offsets, T, K, E, h);
    a.y = rows;
    a.ldy = h;
    a.w = w;
    a.out = out;
    return dtype == CW_F16 ? from_piles<float, _Float16, true>(a, s) : dtype == CW_BF16 ? from_piles<float, bf16_t, true>(a, s)
                                                                                      : from_piles<float, float, true>(a, s);
}
template <class T>
static int from_piles_grad(const PileArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(k_from_piles_grad<T>, dim3((unsigned)std::min<int64_t>(((int64_t)a.T * a.K + 3) / 4, 1 << 22)), dim3(256), 0, s, a);
    return check_launch("k_from_piles_grad");
}

// Up to 2,048 picks one block sorts, in one round of 1 or 2 picks a thread; more of them in chunks of 2,048 (or of as many as make
// 256 chunks), which a launch of its own counts first (8,192 picks of 256 experts in one block, 8 a thread: 15.2 us in a graph).
constexpr int SORT_CHUNK = 2 * SORT_THREADS, SORT_CHUNKS = 256;
static int64_t sort_chunk(int64_t picks) {
    const int64_t rounds = (picks + SORT_CHUNK - 1) / SORT_CHUNK;
    return std::max<int64_t>(1, (rounds + SORT_CHUNKS - 1) / SORT_CHUNKS) * SORT_CHUNK;
}
static int64_t sort_chunks(int64_t picks) { return std::max<int64_t>(1, (picks + sort_chunk(picks) - 1) / sort_chunk(picks)); }

template <int PER>
static int sort_launch(const SortArgs &a, unsigned chunks, hipStream_t s) {
    // dynamic LDS above 64 KB, opted into once per kernel and device
    static std::atomic<bool> set[MAX_DEVICES];
    const int dev = current_device(), lds = sort_lds(a.experts);
    if (lds > 65536 - 512 && !set[dev].load(std::memory_order_relaxed)) {
        if (hipFuncSetAttribute((const void *)k_pile_sort<PER>, hipFuncAttributeMaxDynamicSharedMemorySize, SORT_MAX_LDS) != hipSuccess)
            return set_error(CW_EHIP, "sort_picks: %d bytes of LDS", lds);
        set[dev].store(true, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(k_pile_sort<PER>, dim3(chunks), dim3(SORT_THREADS), lds, s, a);
    return check_launch("k_pile_sort");
}

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
    return check_sort(picks, n_experts) || picks <= SORT_CHUNK ? 0 : (size_t)(sort_chunks(picks) * (n_experts + 1) * 4);
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
    a.chunk = (int)sort_chunk(picks);
    for (a.bits = 1; n_experts >> a.bits; a.bits++) {}
    a.order = order;
    a.place = place;
    a.offsets = offsets;
    a.n_tiles = (int *)tiles;
    a.tiles = (PileTile *)pile_tiles(tiles);
    hipStream_t s = (hipStream_t)stream;
    const unsigned chunks = (unsigned)sort_chunks(picks);
    if (need) {
        a.counts = (int *)ws;
        hipLaunchKernelGGL(k_pile_counts, dim3(chunks), dim3(SORT_THREADS), 0, s, a);
        if (int rc = check_launch("k_pile_counts")) return rc;
    }
    return picks <= SORT_THREADS ? sort_launch<1>(a, chunks, s) : sort_launch<2>(a, chunks, s);
}

int cw_to_piles(int dtype, const void *x, int64_t ldx, int64_t T, int K, int n_experts, int64_t h, const int32_t *order, const int32_t *offsets,
                void *rows, cw_stream_t stream) {
    if (int rc = check_piles("to_piles", dtype, T, K, n_experts, h)) return rc;
    if (T == 0) return CW_OK;
    CW_REQUIRE(x && order && offsets && rows && ldx >= h, "to_piles: null pointer, or rows of %lld %lld apart", (long long)h, (long long)ldx);
    PileArgs a = pile_args(order, nullptr, offsets, T, K, n_experts, h);
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
    PileArgs a = pile_args(nullptr, place, offsets, T, K, n_experts, h);
    a.y = rows;
    a.ldy = ldr;
    a.w = w;
    a.out = out;
    hipStream_t s = (hipStream_t)stream;
    return dtype == CW_F16 ? from_piles<_Float16>(a, s) : dtype == CW_BF16 ? from_piles<bf16_t>(a, s) : from_piles<float>(a, s);
}

int cw_from_piles_grad(int dtype, const void *dout, int64_t ldd, const void *rows, int64_t ldr, const float *w, int64_t T, int K, int n_experts,
                       int64_t h, const int32_t *place, const int32_t *offsets, void *drows, float *dw, cw_stream_t stream) {
    if (int rc = check_piles("from_piles_grad", dtype, T, K, n_experts, h)) return rc;
    if (T == 0) return CW_OK;
    CW_REQUIRE(dout && rows && w && place && offsets && drows && dw, "from_piles_grad: null pointer");
    CW_REQUIRE(ldd >= h && ldr >= h, "from_piles_grad: rows of %lld %lld and %lld apart", (long long)h, (long long)ldd, (long long)ldr);
    PileArgs a = pile_args(nullptr, place, offsets, T, K, n_experts, h);
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
