// Sums of rows by id: out[v] = scale * sum over positions j with key v of  coef[j] * src[j / per_row]  (coef optional),
// in fp32, rounded once; rows that no position names are zero.  The positions come sorted by key (row_sort.cu), so
// nothing is accumulated in memory, the order of the additions depends on the keys alone, and every row is written once.
//
// The sorted positions are cut into tiles of equal length, whatever the keys' frequencies are (text: one id can hold a
// tenth of all tokens).  A key whose positions lie in one tile is finished there, in the order of its positions; one that
// crosses tiles leaves a partial row per tile, and the join kernel adds those in a fixed order (two interleaved runs,
// then the runs).
#include "kernels.h"
#include "row_ops.cuh"

namespace peer {

namespace {

constexpr int SUM_THREADS = 256;

struct SumParams {
    const uint32_t* keys; const uint32_t* order;   // sorted ids (vocab = none) and their positions
    int64_t n; uint32_t vocab;
    const void* src; int64_t src_stride;           // rows that are added
    const float* coef; uint32_t per_row;           // position j adds coef[j] * row j / per_row
    float scale;
    void* out; int64_t D;
    float* partial;                                // [tiles][2][D]
    int* open_tiles; int* open_count;              // tiles in which an id begins that goes on behind them
    int64_t tiles;
    int row_threads, slabs;                        // threads of a tile, column slabs of row_threads pieces
    int zero_blocks;                               // leading blocks write the rows no position names; 0: the sort has done it
};

// 32-ary search by the warp over a sorted array: number of leading entries (of n, `stride` apart) for which
// below(i) holds.  below() must be true, then false.
template <typename F>
__device__ __forceinline__ int64_t warp_count(int64_t n, const F& below) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = n;                                // below(i) for i < lo, not for i >= hi
    while (lo < hi) {
        const int64_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const unsigned yes = __ballot_sync(FULL_MASK, i < hi && below(i));
        const int k = __popc(yes);                         // the first k samples hold
        const int64_t next_lo = k ? lo + (k - 1) * step + 1 : lo, next_hi = lo + k * step;
        hi = next_hi < hi ? next_hi : hi;
        lo = next_lo;
    }
    return lo;
}

constexpr int ZERO_ROWS = 64;

// rows [first, first + ZERO_ROWS): which of them the sorted keys name, then zeros for the others
template <typename T>
__device__ __forceinline__ void zero_rows(const SumParams& p, int64_t first) {
    __shared__ uint32_t named[ZERO_ROWS / 32];
    if (threadIdx.x < ZERO_ROWS / 32) named[threadIdx.x] = 0u;
    __shared__ int64_t from;
    const int64_t last = first + ZERO_ROWS < p.vocab ? first + ZERO_ROWS : p.vocab;
    if (threadIdx.x < 32) {
        const int64_t at = warp_count(p.n, [&](int64_t i) { return p.keys[i] < static_cast<uint32_t>(first); });
        if (threadIdx.x == 0) from = at;
    }
    __syncthreads();
    // one thread per position of these rows; an id with many positions is met at its first few strides only once per
    // stride, so rows are skipped to by search when a stride brought no new one
    for (int64_t j0 = from; j0 < p.n;) {
        const int64_t j = j0 + threadIdx.x;
        const uint32_t key = j < p.n ? p.keys[j] : p.vocab;
        if (key < last) atomicOr(&named[(key - first) >> 5], 1u << ((key - first) & 31));
        const uint32_t end_key = j0 + blockDim.x - 1 < p.n ? p.keys[j0 + blockDim.x - 1] : p.vocab;
        if (end_key >= last) break;
        // the stride ended inside end_key's positions: go on behind them
        j0 += blockDim.x;
        if (p.keys[j0 < p.n ? j0 : p.n - 1] == end_key)
            j0 += warp_count(p.n - j0, [&](int64_t i) { return p.keys[j0 + i] <= end_key; });
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int V = 16 / sizeof(T);
    const bool vec = p.D % V == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
    for (int64_t v = first + warp; v < last; v += blockDim.x >> 5) {
        if (named[(v - first) >> 5] >> ((v - first) & 31) & 1u) continue;
        T* row = static_cast<T*>(p.out) + v * p.D;
        if (vec) for (int64_t c = lane; c < p.D / V; c += 32) reinterpret_cast<uint4*>(row)[c] = make_uint4(0u, 0u, 0u, 0u);
        else for (int64_t c = lane; c < p.D; c += 32) row[c] = from_f32<T>(0.f);
    }
}

// Blocks behind the zero blocks: tiles of PER sorted positions, row_threads pieces of columns each (several tiles per
// block when rows are short).  Eight rows' pieces are in flight per thread; the additions keep the order of positions.
template <typename T, bool WIDE, int PER, bool COEF>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_kernel(const SumParams p) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N, U = 8;
    __shared__ uint32_t s_key[SUM_THREADS / 8 * PER], s_pos[SUM_THREADS / 8 * PER];
    __shared__ float s_coef[COEF ? SUM_THREADS / 8 * PER : 1];
    grid_wait();                                           // the sort's results
    if (static_cast<int>(blockIdx.x) < p.zero_blocks) {
        for (int64_t r = static_cast<int64_t>(blockIdx.x) * ZERO_ROWS; r < p.vocab; r += static_cast<int64_t>(p.zero_blocks) * ZERO_ROWS) {
            zero_rows<T>(p, r);
            __syncthreads();
        }
        return;
    }
    const int subs = SUM_THREADS / p.row_threads, sub = threadIdx.x / p.row_threads;
    const int64_t job = blockIdx.x - p.zero_blocks, slab = job % p.slabs, tile0 = job / p.slabs * subs;
    for (int i = threadIdx.x; i < subs * PER; i += SUM_THREADS) {
        const int64_t j = tile0 * PER + i;
        s_key[i] = j < p.n ? p.keys[j] : p.vocab;
        const uint32_t at = j < p.n ? p.order[j] : 0u;
        s_pos[i] = COEF ? at / p.per_row : at;
        if constexpr (COEF) s_coef[i] = j < p.n ? p.coef[at] : 0.f;
    }
    __syncthreads();
    const int64_t tile = tile0 + sub, t0 = tile * PER;
    const int64_t c = (slab * p.row_threads + (threadIdx.x - sub * p.row_threads)) * N;
    if (t0 >= p.n || c >= p.D) return;
    const uint32_t* key = s_key + sub * PER;
    const uint32_t* pos = s_pos + sub * PER;
    uint32_t cur = key[0];
    if (cur == p.vocab) return;
    bool open_left = t0 > 0 && p.keys[t0 - 1] == cur;      // the id's positions begin in an earlier tile
    const bool goes_on = t0 + PER < p.n && key[PER - 1] != p.vocab && p.keys[t0 + PER] == key[PER - 1];
    const T* src = static_cast<const T*>(p.src) + c;
    float acc[N];
#pragma unroll
    for (int q = 0; q < N; ++q) acc[q] = 0.f;
    auto flush = [&](bool open_right) {
        if (open_left || open_right) {
            float* dst = p.partial + (tile * 2 + (open_left ? 0 : 1)) * p.D + c;
#pragma unroll
            for (int q = 0; q < N; ++q) dst[q] = acc[q];
            if (!open_left && c == 0) p.open_tiles[atomicAdd(p.open_count, 1)] = static_cast<int>(tile);
        } else {
            float f[N];
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] = acc[q] * p.scale;
            P::store(static_cast<T*>(p.out) + static_cast<int64_t>(cur) * p.D + c, P::encode(f));
        }
    };
    bool done = false;
    for (int j0 = 0; j0 < PER && !done; j0 += U) {
        typename P::Raw raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            raw[u] = key[j0 + u] != p.vocab ? P::load(src + static_cast<int64_t>(pos[j0 + u]) * p.src_stride) : P::zero();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = key[j0 + u];
            if (k != cur && !done) {
                flush(false);
                if (k == p.vocab) { done = true; }
                cur = k;
                open_left = false;
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] = 0.f;
            }
            float f[N];
            P::decode(raw[u], f);
            if constexpr (COEF) {
                const float w = s_coef[sub * PER + j0 + u];
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] = fmaf(w, f[q], acc[q]);
            } else {
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] += f[q];
            }
        }
    }
    if (!done) flush(goes_on);
}

// Sums of the partial rows of ids that cross tiles: jobs are (entry of open_tiles, slab of 128 V columns), two runs of
// partial rows per job.  Most ids end in the next tile, which the first two loads find out; a frequent one (12,000 of
// 131,072 text-like positions) has hundreds of partial rows, eight of which are kept in flight per run (by cp.async: from
// plain loads the compiler makes a chain of one load and its addition after another, four times slower).
constexpr int JOIN_COLUMNS = 128, JOIN_DEPTH = 8;
template <typename T, int V, int PER>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_join_kernel(const SumParams p) {
    __shared__ float second[JOIN_COLUMNS * V];
    __shared__ __align__(16) float ahead[JOIN_DEPTH][SUM_THREADS][V];      // rows on their way, each thread's its own
    const int tx = threadIdx.x & (JOIN_COLUMNS - 1), ty = threadIdx.x / JOIN_COLUMNS;
    const int slabs = static_cast<int>((p.D + JOIN_COLUMNS * V - 1) / (JOIN_COLUMNS * V));
    grid_wait();
    const int64_t jobs = static_cast<int64_t>(*p.open_count) * slabs;
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int64_t tile = p.open_tiles[job / slabs], c = (job % slabs) * JOIN_COLUMNS * V + tx * V;
        const uint32_t cur = p.keys[tile * PER + PER - 1];
        // tiles behind this one whose last position is still cur's, and the one in which cur ends
        auto full = [&](int64_t i) {
            const int64_t e = (tile + 2 + i) * PER;
            return e < p.n && p.keys[e - 1] == cur && p.keys[e] == cur;
        };
        const int64_t more = full(0) ? warp_count(p.tiles - tile - 1, full) + 1 : 1;
        float acc[V];
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] = 0.f;
        if (c < p.D) {
            // run 0: its own row, then every second of those behind it; run 1: the others
            const float* own = p.partial + (tile * 2 + 1) * p.D + c;
            const float* rest = p.partial + (tile + (ty == 0 ? 2 : 1)) * 2 * p.D + c;
            const int count = static_cast<int>(ty == 0 ? more / 2 + 1 : (more + 1) / 2);
            auto fetch = [&](int k) {
                if (k < count) {
                    const float* row = ty == 0 ? (k == 0 ? own : rest + static_cast<int64_t>(k - 1) * 4 * p.D)
                                               : rest + static_cast<int64_t>(k) * 4 * p.D;
                    copy_async<4 * V>(smem_u32(ahead[k % JOIN_DEPTH][threadIdx.x]), row);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            for (int k = 0; k < JOIN_DEPTH - 1; ++k) fetch(k);
            for (int k = 0; k < count; ++k) {
                fetch(k + JOIN_DEPTH - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"(JOIN_DEPTH - 1) : "memory");
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += ahead[k % JOIN_DEPTH][threadIdx.x][q];
            }
        }
        if (ty == 1) {
#pragma unroll
            for (int q = 0; q < V; ++q) second[tx * V + q] = acc[q];
        }
        __syncthreads();
        if (ty == 0 && c < p.D) {
#pragma unroll
            for (int q = 0; q < V; ++q)
                static_cast<T*>(p.out)[static_cast<int64_t>(cur) * p.D + c + q] = from_f32<T>((acc[q] + second[tx * V + q]) * p.scale);
        }
        __syncthreads();
    }
}

int per_tile_for(int64_t n) { return n <= (1 << 15) ? 16 : 64; }

template <typename T, bool WIDE, int PER, bool COEF>
cudaError_t sums_launch(SumParams p, cudaStream_t s) {
    constexpr int N = Piece<T, WIDE>::N;
    const int64_t pieces = p.D / N;
    p.row_threads = 8;
    while (p.row_threads < SUM_THREADS && p.row_threads < pieces) p.row_threads *= 2;
    p.slabs = static_cast<int>((pieces + p.row_threads - 1) / p.row_threads);
    const int subs = SUM_THREADS / p.row_threads;
    const int64_t zb = (static_cast<int64_t>(p.vocab) + ZERO_ROWS - 1) / ZERO_ROWS;
    p.zero_blocks = p.zero_blocks ? static_cast<int>(zb < GRID_SMS * 32 ? zb : GRID_SMS * 32) : 0;
    const int64_t blocks = p.zero_blocks + (p.tiles + subs - 1) / subs * p.slabs;
    cudaError_t e = launch_behind(row_sum_kernel<T, WIDE, PER, COEF>, dim3(static_cast<unsigned>(blocks)), dim3(SUM_THREADS), s, p);
    if (e != cudaSuccess || p.tiles <= 1) return e;
    const int64_t jobs = p.tiles * ((p.D + 511) / 512);
    const dim3 grid(static_cast<unsigned>(jobs < GRID_SMS * 8 ? jobs : GRID_SMS * 8));
    return p.D % 4 == 0 ? launch_behind(row_sum_join_kernel<T, 4, PER>, grid, dim3(SUM_THREADS), s, p)
                        : launch_behind(row_sum_join_kernel<T, 1, PER>, grid, dim3(SUM_THREADS), s, p);
}

template <typename T>
cudaError_t sums_t(const SumParams& p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = p.D % N == 0 && p.src_stride % N == 0 && aligned16(p.src) && aligned16(p.out);
    const bool small = per_tile_for(p.n) == 16;
    if (p.coef) {                                           // the expert tables: always whole 16-byte pieces
        if (!wide) return cudaErrorInvalidValue;
        return small ? sums_launch<T, true, 16, true>(p, s) : sums_launch<T, true, 64, true>(p, s);
    }
    if (small) return wide ? sums_launch<T, true, 16, false>(p, s) : sums_launch<T, false, 16, false>(p, s);
    return wide ? sums_launch<T, true, 64, false>(p, s) : sums_launch<T, false, 64, false>(p, s);
}

}  // namespace

int64_t row_sum_bytes(int64_t n, int64_t D) {
    const int per = per_tile_for(n);
    const int64_t tiles = (n + per - 1) / per;
    return (tiles * 4 + 255) / 256 * 256 + tiles * 2 * D * static_cast<int64_t>(sizeof(float));
}

cudaError_t launch_row_sums(RowSumArgs& a, cudaStream_t s) {
    SumParams p{};
    p.keys = a.keys; p.order = a.order; p.n = a.n; p.vocab = static_cast<uint32_t>(a.vocab);
    p.src = a.src; p.src_stride = a.src_stride; p.coef = a.coef; p.per_row = static_cast<uint32_t>(a.per_row);
    p.scale = a.scale; p.out = a.out; p.D = a.D;
    const int per = per_tile_for(a.n);
    p.tiles = (a.n + per - 1) / per;
    p.open_count = a.counter;
    p.open_tiles = static_cast<int*>(a.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + (p.tiles * 4 + 255) / 256 * 256);
    p.zero_blocks = a.zero ? 1 : 0;
    a.launches = p.tiles > 1 ? 2 : 1;
    if (a.dtype == PEER_DTYPE_F32) return sums_t<float>(p, s);
    if (a.dtype == PEER_DTYPE_BF16) return sums_t<__nv_bfloat16>(p, s);
    if (a.dtype == PEER_DTYPE_F16) return sums_t<__half>(p, s);
    return cudaErrorInvalidValue;
}

}  // namespace peer
