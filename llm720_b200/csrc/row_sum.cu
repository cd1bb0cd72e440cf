// Sums of rows by id: out[v] = scale * sum over positions j with key v of  coef[j] * src[j / per_row]  (coef optional),
// in fp32, rounded once; rows that no position names are zero.  The positions come sorted by key (row_sort.cu), so
// nothing is accumulated in memory, the order of the additions depends on the keys alone, and every row is written once.
//
// The sorted positions are cut into tiles of equal length, whatever the keys' frequencies are (text: one id can hold a
// tenth of all tokens).  A key with no more positions than a tile is finished by the tile in which they begin, in their
// order, wherever they end; one with more leaves a partial row per tile, and the join kernel adds those in a fixed order
// (four interleaved runs, then the runs).
#include <type_traits>

#include "kernels.h"
#include "row_ops.cuh"
#include "row_shift.cuh"

namespace peer {

namespace {

constexpr int SUM_THREADS = 256;

struct SumParams {
    const uint32_t* keys; const uint32_t* order;   // sorted ids (vocab = none) and their positions
    int64_t n; uint32_t vocab;
    const void* src; int64_t src_stride;           // rows that are added
    const void* src_end;                           // behind the last one's last value (not WIDE)
    uint32_t edge, inner;                          // rows [edge, edge + inner) are 16 bytes away from the ends of src (not WIDE)
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

constexpr int ZERO_ROWS = 64, ZERO_SCAN = 2048;

// rows [first, first + ZERO_ROWS): which of them the sorted keys name, then zeros for the others
template <typename T>
__device__ __forceinline__ void zero_rows(const SumParams& p, int64_t first) {
    __shared__ uint32_t named[ZERO_ROWS / 32];
    __shared__ int64_t range[2];                           // the rows' positions
    if (threadIdx.x < ZERO_ROWS / 32) named[threadIdx.x] = 0u;
    const int64_t last = first + ZERO_ROWS < p.vocab ? first + ZERO_ROWS : p.vocab;
    if (threadIdx.x < 64) {
        const uint32_t key = static_cast<uint32_t>(threadIdx.x < 32 ? first : last);
        const int64_t at = warp_count(p.n, [&](int64_t i) { return p.keys[i] < key; });
        if ((threadIdx.x & 31) == 0) range[threadIdx.x >> 5] = at;
    }
    __syncthreads();
    const int64_t from = range[0], to = range[1];
    if (to - from <= ZERO_SCAN) {
        for (int64_t j = from + threadIdx.x; j < to; j += SUM_THREADS) {
            const uint32_t r = p.keys[j] - static_cast<uint32_t>(first);
            atomicOr(&named[r >> 5], 1u << (r & 31));
        }
    } else if (static_cast<int64_t>(threadIdx.x) < last - first) {
        // frequent ids, often next to one another: a search per row instead (65,536 ids in order of their frequency,
        // 64 of which hold half of all positions: this kernel takes 45 us instead of 107)
        const uint32_t key = static_cast<uint32_t>(first) + threadIdx.x;
        int64_t lo = from, hi = to;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.keys[mid] < key) lo = mid + 1;
            else hi = mid;
        }
        if (lo < to && p.keys[lo] == key) atomicOr(&named[threadIdx.x >> 5], 1u << (threadIdx.x & 31));
    }
    __syncthreads();
    constexpr int N = 16 / sizeof(T);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t v = first + warp; v < last; v += blockDim.x >> 5) {
        if (named[(v - first) >> 5] >> ((v - first) & 31) & 1u) continue;
        T* row = static_cast<T*>(p.out) + v * p.D;
        for (int64_t c = lane * N - static_cast<int>(offset16(row) / sizeof(T)); c < p.D; c += 32 * N) store_granule(row, c, p.D, make_uint4(0u, 0u, 0u, 0u));
    }
}

// first index in [lo, hi) that does not lie below (hi if all do)
template <typename F>
__device__ __forceinline__ int first_index(int lo, int hi, const F& below) {
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (below(mid)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Blocks behind the zero blocks: tiles of PER sorted positions, row_threads pieces of columns each (several tiles per
// block when rows are short).  Eight rows' pieces are in flight per thread, four where rows are not whole 16-byte pieces; the
// additions keep the order of positions.  Not WIDE: a thread's columns begin at a granule of the row that it writes, so they
// depend on the id, and are read as two granules and shifted (20,000 ids of 8,000 x 2500 bf16: the gradient takes
// 66 us, 109 value by value).
template <typename T, bool WIDE, int PER, bool COEF>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_kernel(const SumParams p) {
    using P = Piece<T, true>;
    constexpr int N = P::N, U = WIDE ? 8 : 4, MOST = SUM_THREADS / 8 * PER;
    __shared__ uint32_t s_key[MOST + 2 * PER], s_pos[MOST + PER];      // the block's tiles; keys of one tile before, both of one behind
    __shared__ float s_coef[COEF ? MOST + PER : 1];
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
    bool edge = false;                                     // rows within 16 bytes of the ends of src among them
    for (int i = threadIdx.x; i < (subs + 2) * PER; i += SUM_THREADS) {
        const int64_t j = (tile0 - 1) * PER + i;
        s_key[i] = j >= 0 && j < p.n ? p.keys[j] : p.vocab;
        if (i < PER) continue;
        const uint32_t at = j < p.n ? p.order[j] : 0u;
        s_pos[i - PER] = COEF ? at / p.per_row : at;
        if constexpr (COEF) s_coef[i - PER] = j < p.n ? p.coef[at] : 0.f;
        if constexpr (!WIDE) edge |= j < p.n && at - p.edge >= p.inner;
    }
    const bool edges = __syncthreads_or(edge) != 0;        // one block or two of the grid
    const int64_t tile = tile0 + sub, t0 = tile * PER;
    const int64_t c = (slab * p.row_threads + (threadIdx.x - sub * p.row_threads)) * N;
    if (t0 >= p.n || c >= p.D + (WIDE ? 0 : N - 1)) return;
    const uint32_t* key = s_key + (sub + 1) * PER;         // [-PER, 2 PER)
    const uint32_t* pos = s_pos + sub * PER;
    // An id has more than PER positions exactly if its first one and the one PER behind that are both its own.
    uint32_t cur = key[0];
    if (cur == p.vocab) return;
    int j = 0, end = PER;
    bool open_left = false, goes_on = false;               // the id at the tile's begin, at its end has a partial row
    if (t0 > 0 && key[-1] == cur) {
        const int begin = first_index(-PER, 0, [&](int i) { return key[i] < cur; });
        open_left = key[begin + PER] == cur;
        if (!open_left) {                                  // the tile before has it; it ends in front of begin + PER
            j = first_index(0, PER, [&](int i) { return key[i] <= cur; });
            cur = key[j];
        }
    }
    const uint32_t last = key[PER - 1];
    if (last == p.vocab) {
        end = first_index(j, PER, [&](int i) { return key[i] < p.vocab; });
        if (j == end) return;
    } else if (key[PER] == last) {
        const int begin = first_index(0, PER, [&](int i) { return key[i] < last; });
        goes_on = key[begin + PER] == last;
        if (!goes_on) end = first_index(PER, 2 * PER, [&](int i) { return key[i] <= last; });
    }
    const T* src = static_cast<const T*>(p.src);
    T* out = static_cast<T*>(p.out);
    // first of this thread's columns of an id's row
    const uint32_t out_low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out)), row_low = static_cast<uint32_t>(p.D * sizeof(T));
    auto column = [&](uint32_t id) { return WIDE ? c : c - static_cast<int>(((out_low + id * row_low) & 15u) / sizeof(T)); };
    float acc[N];
#pragma unroll
    for (int q = 0; q < N; ++q) acc[q] = 0.f;
    auto flush = [&](bool open_right) {
        const int64_t at = column(cur);
        if (open_left || open_right) {
            float* dst = p.partial + (tile * 2 + (open_left ? 0 : 1)) * p.D + at;
            if constexpr (WIDE) {
#pragma unroll
                for (int q = 0; q < N; q += 4) *reinterpret_cast<float4*>(dst + q) = make_float4(acc[q], acc[q + 1], acc[q + 2], acc[q + 3]);
            } else {
#pragma unroll
                for (int q = 0; q < N; ++q)
                    if (at + q >= 0 && at + q < p.D) dst[q] = acc[q];
            }
            if (!open_left && c == 0) p.open_tiles[atomicAdd(p.open_count, 1)] = static_cast<int>(tile);
        } else {
            float f[N];
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] = acc[q] * p.scale;
            T* row = out + static_cast<int64_t>(cur) * p.D;
            if constexpr (WIDE) P::store(row + at, P::encode(f));
            else store_granule(row, at, p.D, P::encode(f));
        }
    };
    for (; j < end; j += U) {
        std::conditional_t<WIDE, uint4, Granules> raw[U];
        if constexpr (WIDE) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = j + u < end ? P::load(src + static_cast<int64_t>(pos[j + u]) * p.src_stride + c) : P::zero();
        } else if (!edges) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u < end) raw[u] = load_granules(src + static_cast<int64_t>(pos[j + u]) * p.src_stride, column(key[j + u]), p.D);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u < end)
                    raw[u] = load_edge_granules(src + static_cast<int64_t>(pos[j + u]) * p.src_stride, column(key[j + u]), p.D, src, p.src_end);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j + u >= end) break;
            const uint32_t k = key[j + u];
            if (k != cur) {
                flush(false);
                cur = k;
                open_left = false;
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] = 0.f;
            }
            float f[N];
            if constexpr (WIDE) P::decode(raw[u], f);
            else P::decode(shifted(raw[u].lo, raw[u].hi, raw[u].shift), f);
            if constexpr (COEF) {
                const float w = s_coef[sub * PER + j + u];
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] = fmaf(w, f[q], acc[q]);
            } else {
#pragma unroll
                for (int q = 0; q < N; ++q) acc[q] += f[q];
            }
        }
    }
    flush(goes_on);
}

// Sums of the partial rows of ids with more than PER positions: jobs are (entry of open_tiles, slab of 64 V columns), four
// runs of partial rows per job.  Most ids end in the next tile, which the first two loads find out; a frequent one (12,000 of
// 131,072 text-like positions) has hundreds of partial rows, eight of which are kept in flight per run (by cp.async: from
// plain loads the compiler makes a chain of one load and its addition after another, four times slower).  The gradient of
// 131,072 text-like ids of 32,000 x 2048 bf16 takes 150 us with four runs, 156 with two or eight.
constexpr int JOIN_COLUMNS = 64, JOIN_RUNS = SUM_THREADS / JOIN_COLUMNS, JOIN_DEPTH = 8;
template <typename T, int V, int PER>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_join_kernel(const SumParams p) {
    __shared__ __align__(16) float others[JOIN_RUNS - 1][JOIN_COLUMNS][V];
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
            // run r: partial rows r, r + JOIN_RUNS, ... of the id; row 0 is where it begins
            const float* first = p.partial + tile * 2 * p.D + c;
            const int count = more < ty ? 0 : static_cast<int>((more - ty) / JOIN_RUNS) + 1;
            auto fetch = [&](int k) {
                if (k < count) {
                    const int64_t m = static_cast<int64_t>(k) * JOIN_RUNS + ty;
                    copy_async<4 * V>(smem_u32(ahead[k % JOIN_DEPTH][threadIdx.x]), first + (m ? m * 2 : 1) * p.D);
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
        if (ty > 0) {
#pragma unroll
            for (int q = 0; q < V; ++q) others[ty - 1][tx][q] = acc[q];
        }
        __syncthreads();
        if (ty == 0 && c < p.D) {
#pragma unroll
            for (int i = 0; i < JOIN_RUNS - 1; ++i)
#pragma unroll
                for (int q = 0; q < V; ++q) acc[q] += others[i][tx][q];
#pragma unroll
            for (int q = 0; q < V; ++q) static_cast<T*>(p.out)[static_cast<int64_t>(cur) * p.D + c + q] = from_f32<T>(acc[q] * p.scale);
        }
        __syncthreads();
    }
}

int per_tile_for(int64_t n) { return n <= (1 << 15) ? 16 : 64; }

template <typename T, bool WIDE, int PER, bool COEF>
cudaError_t sums_launch(SumParams p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const int64_t pieces = WIDE ? p.D / N : (p.D + 2 * N - 2) / N;      // a row that begins inside a granule: one more
    p.row_threads = 8;
    while (p.row_threads < SUM_THREADS && p.row_threads < pieces) p.row_threads *= 2;
    for (int t = p.row_threads / 2; t >= 32; t /= 2)       // narrower slabs where they leave fewer threads without columns
        if ((pieces + t - 1) / t * t < (pieces + p.row_threads - 1) / p.row_threads * p.row_threads) p.row_threads = t;
    p.slabs = static_cast<int>((pieces + p.row_threads - 1) / p.row_threads);
    const int subs = SUM_THREADS / p.row_threads;
    const int64_t zb = (static_cast<int64_t>(p.vocab) + ZERO_ROWS - 1) / ZERO_ROWS;
    p.zero_blocks = p.zero_blocks ? static_cast<int>(zb < GRID_SMS * 32 ? zb : GRID_SMS * 32) : 0;
    const int64_t blocks = p.zero_blocks + (p.tiles + subs - 1) / subs * p.slabs;
    cudaError_t e = launch_behind(row_sum_kernel<T, WIDE, PER, COEF>, dim3(static_cast<unsigned>(blocks)), dim3(SUM_THREADS), s, p);
    if (e != cudaSuccess || p.tiles <= 1) return e;
    const int64_t jobs = p.tiles * ((p.D + JOIN_COLUMNS * 4 - 1) / (JOIN_COLUMNS * 4));
    const dim3 grid(static_cast<unsigned>(jobs < GRID_SMS * 8 ? jobs : GRID_SMS * 8));
    return p.D % 4 == 0 ? launch_behind(row_sum_join_kernel<T, 4, PER>, grid, dim3(SUM_THREADS), s, p)
                        : launch_behind(row_sum_join_kernel<T, 1, PER>, grid, dim3(SUM_THREADS), s, p);
}

template <typename T>
cudaError_t sums_t(SumParams p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = p.D % N == 0 && p.src_stride % N == 0 && aligned16(p.src) && aligned16(p.out);
    const bool small = per_tile_for(p.n) == 16;
    p.src_end = static_cast<const T*>(p.src) + (p.n - 1) * p.src_stride + p.D;      // one row per position
    const int64_t edge = edge_rows(p.n, p.src_stride * static_cast<int64_t>(sizeof(T)));
    p.edge = static_cast<uint32_t>(edge);
    p.inner = static_cast<uint32_t>(p.n > 2 * edge ? p.n - 2 * edge : 0);
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
