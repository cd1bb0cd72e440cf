// Scaled embedding lookup and its gradient.
//
//   out[t]  = scale * W[id_t]                       (a row of zeros for an id outside the table)
//   dW[v]   = scale * sum over t with id_t = v of dy[t], rounded once; zero for rows no token names
//
// The lookup replaces the nn.Embedding read of the reference's model
// (llm/models/foundation.py:338) and of torch's backward pass to it.  The
// gradient sorts the positions by id (row_sort.cu), then adds each id's rows in
// the order of their positions, in fp32: nothing is accumulated in memory, so
// the sums have one order and every row of dW is written exactly once.
//
// The sorted positions are cut into tiles of equal length, whatever the ids'
// frequencies are (text: one id can hold a tenth of all tokens).  An id whose
// positions lie in one tile is finished there, in the order of its positions;
// one that crosses tiles leaves a partial row per tile, and the join kernel adds
// those in a fixed order (two interleaved runs, then the runs).
#include <cstdio>

#include "kernels.h"
#include "row_ops.cuh"

namespace peer {
void set_global_error(const char* msg);

namespace {

constexpr int SUM_THREADS = 256;

template <typename T, int VEC> struct Load;
template <typename T> struct Load<T, 1> {
    __device__ static __forceinline__ void get(const T* p, float (&f)[1]) { f[0] = to_f32<T>(*p); }
    __device__ static __forceinline__ void put(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};
template <> struct Load<float, 4> {
    __device__ static __forceinline__ void get(const float* p, float (&f)[4]) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    __device__ static __forceinline__ void put(float* p, const float (&f)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <typename T> struct Load<T, 8> {
    __device__ static __forceinline__ void get(const T* p, float (&f)[8]) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = to_f32<T>(e[q]);
    }
    __device__ static __forceinline__ void put(T* p, const float (&f)[8]) {
        uint4 v;
        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q) e[q] = from_f32<T>(f[q]);
        *reinterpret_cast<uint4*>(p) = v;
    }
};

__device__ __forceinline__ int64_t id_at(const void* ids, int id_bytes, int64_t i) {
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// one warp per token
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_kernel(const void* __restrict__ ids, int id_bytes, int64_t n, const T* __restrict__ w,
                                                    int64_t vocab, int64_t D, float scale, T* __restrict__ out,
                                                    unsigned long long* dropped) {
    const int lane = threadIdx.x & 31;
    const int64_t stride = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    for (int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; t < n; t += stride) {
        const int64_t id = id_at(ids, id_bytes, t);
        const bool inside = id >= 0 && id < vocab;
        if (!inside && dropped && lane == 0) atomicAdd(dropped, 1ULL);
        const T* row = w + (inside ? id : 0) * D;
        for (int64_t c = static_cast<int64_t>(lane) * VEC; c < D; c += 32 * VEC) {
            float f[VEC];
            if (inside) {
                Load<T, VEC>::get(row + c, f);
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] *= scale;
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] = 0.f;
            }
            Load<T, VEC>::put(out + t * D + c, f);
        }
    }
}

struct SumParams {
    const uint32_t* keys; const uint32_t* order;   // sorted ids (vocab = none) and their positions
    int64_t n; uint32_t vocab;
    const void* src; int64_t src_stride;           // rows that are added
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
template <typename T, bool WIDE, int PER>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_kernel(const SumParams p) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N, U = 8;
    __shared__ uint32_t s_key[SUM_THREADS / 8 * PER], s_pos[SUM_THREADS / 8 * PER];
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
        s_pos[i] = j < p.n ? p.order[j] : 0u;
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
#pragma unroll
            for (int q = 0; q < N; ++q) acc[q] += f[q];
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

template <typename T>
cudaError_t embed_t(const void* ids, int id_bytes, int64_t n, const void* w, int64_t vocab, int64_t D, float scale, void* out,
                    int64_t* dropped, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t blocks = (n + 7) / 8;
    const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
    const bool vec = D % V == 0 && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    auto* d = reinterpret_cast<unsigned long long*>(dropped);
    if (vec) embed_kernel<T, V><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d);
    else embed_kernel<T, 1><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d);
    return cudaGetLastError();
}

template <typename T, bool WIDE, int PER>
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
    cudaError_t e = launch_behind(row_sum_kernel<T, WIDE, PER>, dim3(static_cast<unsigned>(blocks)), dim3(SUM_THREADS), s, p);
    if (e != cudaSuccess || p.tiles <= 1) return e;
    const int64_t jobs = p.tiles * ((p.D + 511) / 512);
    const dim3 grid(static_cast<unsigned>(jobs < GRID_SMS * 8 ? jobs : GRID_SMS * 8));
    return p.D % 4 == 0 ? launch_behind(row_sum_join_kernel<T, 4, PER>, grid, dim3(SUM_THREADS), s, p)
                        : launch_behind(row_sum_join_kernel<T, 1, PER>, grid, dim3(SUM_THREADS), s, p);
}

template <typename T>
cudaError_t sums_t(const SumParams& p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (p.n == 0) return cudaMemsetAsync(p.out, 0, sizeof(T) * static_cast<size_t>(p.vocab) * static_cast<size_t>(p.D), s);
    const bool wide = p.D % N == 0 && p.src_stride % N == 0 && aligned16(p.src) && aligned16(p.out);
    if (per_tile_for(p.n) == 16) return wide ? sums_launch<T, true, 16>(p, s) : sums_launch<T, false, 16>(p, s);
    return wide ? sums_launch<T, true, 64>(p, s) : sums_launch<T, false, 64>(p, s);
}

int report(const char* name, cudaError_t e) {
    if (e == cudaSuccess) return PEER_OK;
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", name, cudaGetErrorString(e));
    set_global_error(buf);
    return PEER_ERR_CUDA;
}
int refuse(const char* msg) {
    set_global_error(msg);
    return PEER_ERR_INVALID_ARG;
}
constexpr int64_t INDEX_MAX = 0x7ffffffe;

}  // namespace
}  // namespace peer

using namespace peer;

extern "C" int peer_embedding(const void* ids, int32_t id_bytes, int64_t n_ids, const void* weight, int32_t dtype, int64_t vocab,
                              int64_t dim, float scale, void* out, int64_t* dropped, void* stream) {
    if (n_ids < 0 || vocab < 1 || vocab > INDEX_MAX || dim < 1 || dim > PEER_ROW_DIM_MAX)
        return refuse("peer_embedding: n_ids must not be negative, vocab lie in [1, 2^31 - 2], dim in [1, 2^20]");
    if (id_bytes != 4 && id_bytes != 8) return refuse("peer_embedding: ids are int32 or int64");
    if (n_ids == 0) return PEER_OK;
    if (!ids || !weight || !out) return refuse("peer_embedding: null pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_embedding", embed_t<float>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_embedding", embed_t<__nv_bfloat16>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_embedding", embed_t<__half>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    return refuse("peer_embedding: dtype must be F32, BF16 or F16");
}

extern "C" int64_t peer_embedding_workspace(int64_t n_ids, int64_t dim) {
    if (n_ids <= 0 || dim < 1) return 0;
    const int per = per_tile_for(n_ids);
    const int64_t tiles = (n_ids + per - 1) / per;
    return row_sort_bytes(n_ids) + ((tiles + 4) * 4 + 255) / 256 * 256 + tiles * 2 * dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int peer_embedding_backward(const void* ids, int32_t id_bytes, int64_t n_ids, const void* grad, int64_t grad_stride,
                                       int32_t dtype, int64_t vocab, int64_t dim, float scale, int64_t padding_idx,
                                       void* grad_weight, void* workspace, int64_t workspace_bytes, void* stream) {
    if (n_ids < 0 || n_ids > INDEX_MAX || vocab < 1 || vocab > INDEX_MAX || dim < 1 || dim > PEER_ROW_DIM_MAX || grad_stride < 0)
        return refuse("peer_embedding_backward: n_ids and vocab must lie below 2^31 - 1, dim in [1, 2^20]");
    if (id_bytes != 4 && id_bytes != 8) return refuse("peer_embedding_backward: ids are int32 or int64");
    if (dtype != PEER_DTYPE_F32 && dtype != PEER_DTYPE_BF16 && dtype != PEER_DTYPE_F16)
        return refuse("peer_embedding_backward: dtype must be F32, BF16 or F16");
    if (!grad_weight || (n_ids > 0 && (!ids || !grad))) return refuse("peer_embedding_backward: null pointer");
    if (n_ids > 0 && (!workspace || workspace_bytes < peer_embedding_workspace(n_ids, dim)))
        return refuse("peer_embedding_backward: workspace is missing or smaller than peer_embedding_workspace says");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowSortArgs a{};
    a.ids = ids; a.id_bytes = id_bytes; a.n = n_ids; a.vocab = vocab; a.skip = padding_idx;
    SumParams p{};
    p.n = n_ids; p.vocab = static_cast<uint32_t>(vocab); p.src = grad; p.src_stride = grad_stride; p.scale = scale;
    p.out = grad_weight; p.D = dim;
    if (n_ids > 0) {
        const int per = per_tile_for(n_ids);
        p.tiles = (n_ids + per - 1) / per;
        row_sort_layout(a, workspace);
        char* rest = static_cast<char*>(workspace) + row_sort_bytes(n_ids);
        p.open_count = a.counter = reinterpret_cast<int*>(rest);
        p.open_tiles = p.open_count + 4;
        p.partial = reinterpret_cast<float*>(rest + ((p.tiles + 4) * 4 + 255) / 256 * 256);
        a.zero_rows = grad_weight;
        a.row_bytes = dim * (dtype == PEER_DTYPE_F32 ? 4 : 2);
        const cudaError_t e = launch_row_sort(a, s);
        if (e != cudaSuccess) return report("peer_embedding_backward", e);
        p.keys = a.sorted_keys; p.order = a.order;
        p.zero_blocks = a.zeroed ? 0 : 1;
    }
    if (dtype == PEER_DTYPE_F32) return report("peer_embedding_backward", sums_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_embedding_backward", sums_t<__nv_bfloat16>(p, s));
    return report("peer_embedding_backward", sums_t<__half>(p, s));
}
