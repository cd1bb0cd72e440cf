// Scaled embedding lookup and its gradient.
//
//   out[t]  = scale * W[id_t]                       (a row of zeros for an id outside the table)
//   dW[v]   = scale * sum over t with id_t = v of dy[t], rounded once; zero for rows no token names
//
// The lookup replaces the nn.Embedding read of the reference's model
// (llm/models/foundation.py:338) and of torch's backward pass to it.  The
// gradient sorts the positions by id (row_sort.cu), then adds each id's rows
// (row_sum.cu): the sums are fp32 in one order, every row of dW is written once.
#include <cstdio>

#include "kernels.h"
#include "row_ops.cuh"
#include "row_shift.cuh"

namespace peer {
void set_global_error(const char* msg);

namespace {

__device__ __forceinline__ int64_t id_at(const void* ids, int id_bytes, int64_t i) {
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// `group` threads (a warp, or the block when there are few tokens) per token, 16-byte pieces.  Not WIDE: the pieces are the
// granules of the row that is written, read as two granules and shifted (20,000 x 2500 bf16: 37 us, 57 value by value); the
// values in front of the first whole granule and behind the last one are copied by a thread each, and so are those of a piece
// whose granules reach beyond the table.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) embed_kernel(const void* __restrict__ ids, int id_bytes, int64_t n, const T* __restrict__ w,
                                                    int64_t vocab, int64_t D, float scale, T* __restrict__ out,
                                                    unsigned long long* dropped, int group) {
    using P = Piece<T, true>;
    constexpr int N = P::N;
    const int gt = threadIdx.x & (group - 1), per_block = blockDim.x / group;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / group; t < n; t += static_cast<int64_t>(gridDim.x) * per_block) {
        const int64_t id = id_at(ids, id_bytes, t);
        const bool inside = id >= 0 && id < vocab;
        if (!inside && dropped && gt == 0) atomicAdd(dropped, 1ULL);
        const T* row = w + (inside ? id : 0) * D;          // row 0 is read in place of none: no test between the loads
        T* dst = out + t * D;
        int begin = 0, end = static_cast<int>(D);
        uint32_t shift = 0;
        if constexpr (!WIDE) {
            const PieceRange range = piece_range(reinterpret_cast<uintptr_t>(row), reinterpret_cast<uintptr_t>(dst), static_cast<int>(D),
                                                 sizeof(T), reinterpret_cast<uintptr_t>(w), reinterpret_cast<uintptr_t>(w + vocab * D));
            begin = range.begin;
            end = range.end;
            shift = range.shift;
            // fewer than 2 N values at either end: lanes 0 to 15 in front, 16 to 31 behind
            const int c = gt < 16 ? gt : end + gt - 16;
            if (gt < 16 ? gt < begin : c < D && gt < 32) dst[c] = from_f32<T>(inside ? to_f32<T>(row[c]) * scale : 0.f);
        }
#pragma unroll 4
        for (int c = begin + gt * N; c < end; c += group * N) {
            float f[N];
            if constexpr (WIDE) {
                P::decode(P::load(row + c), f);
            } else {
                const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row + c) - shift);
                const uint4 lo = __ldg(at), hi = shift ? __ldg(at + 1) : lo;
                P::decode(shifted(lo, hi, shift), f);
            }
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] = inside ? f[q] * scale : 0.f;
            P::store(dst + c, P::encode(f));
        }
    }
}

template <typename T>
cudaError_t embed_t(const void* ids, int id_bytes, int64_t n, const void* w, int64_t vocab, int64_t D, float scale, void* out,
                    int64_t* dropped, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int group = n < GRID_SMS * 8 ? 256 : 32;          // fewer tokens than a warp each would need to fill the SMs
    const int64_t blocks = (n * group + 255) / 256;
    const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
    const bool vec = D % V == 0 && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    auto* d = reinterpret_cast<unsigned long long*>(dropped);
    if (vec) embed_kernel<T, true><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d, group);
    else embed_kernel<T, false><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d, group);
    return cudaGetLastError();
}

int report(const char* name, cudaError_t e) {
    if (e == cudaSuccess) return PEER_OK;
    cudaGetLastError();                                      // reported here, not by the next launch's check
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", name, cudaGetErrorString(e));
    set_global_error(buf);
    return PEER_ERR_CUDA;
}
int refuse(const char* msg) {
    set_global_error(msg);
    return PEER_ERR_INVALID_ARG;
}
constexpr int64_t INDEX_MAX = PEER_SORT_IDS_MAX;

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
    if ((reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1)) || !aligned_to(weight, dtype) || !aligned_to(out, dtype) ||
        (reinterpret_cast<uintptr_t>(dropped) & 7u))
        return refuse("peer_embedding: a pointer is not aligned to its type");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_embedding", embed_t<float>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_embedding", embed_t<__nv_bfloat16>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_embedding", embed_t<__half>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    return refuse("peer_embedding: dtype must be F32, BF16 or F16");
}

extern "C" int64_t peer_embedding_workspace(int64_t n_ids, int64_t dim) {
    if (n_ids <= 0 || dim < 1) return 0;
    return row_sort_bytes(n_ids) + row_sum_bytes(n_ids, dim);
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
    if ((reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1)) || !aligned_to(grad, dtype) || !aligned_to(grad_weight, dtype) ||
        !aligned16(workspace))
        return refuse("peer_embedding_backward: a pointer is not aligned to its type, or the workspace to 16 bytes");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (n_ids == 0)
        return report("peer_embedding_backward",
                      cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(vocab) * dim * (dtype == PEER_DTYPE_F32 ? 4 : 2), s));
    RowSortArgs a{};
    a.ids = ids; a.id_bytes = id_bytes; a.n = n_ids; a.vocab = vocab; a.skip = padding_idx;
    row_sort_layout(a, workspace);
    a.zero_rows = grad_weight;
    a.row_bytes = dim * (dtype == PEER_DTYPE_F32 ? 4 : 2);
    const cudaError_t e = launch_row_sort(a, s);
    if (e != cudaSuccess) return report("peer_embedding_backward", e);
    RowSumArgs r{};
    r.keys = a.sorted_keys; r.order = a.order; r.n = n_ids; r.vocab = vocab; r.src = grad; r.src_stride = grad_stride;
    r.per_row = 1; r.dtype = dtype; r.scale = scale; r.out = grad_weight; r.D = dim; r.counter = a.counters;
    r.workspace = static_cast<char*>(workspace) + row_sort_bytes(n_ids); r.zero = !a.zeroed;
    return report("peer_embedding_backward", launch_row_sums(r, s));
}
