// Activation checkpoints in 8 bits: rows to row-scaled e4m3 and back
// (the format is defined in row_ops.cuh).  Packing reads 2 (4) bytes and writes
// 1 per value, unpacking the reverse: both are bound by HBM.
#include <cstdio>
#include <type_traits>

#include "kernels.h"
#include "row_ops.cuh"
#include "row_shift.cuh"

namespace peer {
void set_global_error(const char* msg);

namespace {

// any width, any alignment: one block per row, the row read twice (the second time from L1/L2)
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_loop_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int64_t D,
                                                             uint8_t* __restrict__ payload, float* __restrict__ scale) {
    __shared__ float buf[33];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * x_stride;
        uint32_t m = 0u;
        for (int64_t c = threadIdx.x; c < D; c += blockDim.x) m = max(m, finite_abs_bits(to_f32<T>(xr[c])));
        const int e = e4m3_scale_exponent(block_max_u32(m, buf));
        const float inv = exp2_int(-e);
        for (int64_t c = threadIdx.x; c < D; c += blockDim.x)
            payload[r * D + c] = static_cast<uint8_t>(e4m3_pair(e4m3_operand(to_f32<T>(xr[c]), inv), 0.f));
        if (threadIdx.x == 0) scale[r] = exp2_int(e);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) unpack_rows_loop_kernel(const uint8_t* __restrict__ payload, const float* __restrict__ scale,
                                                               int64_t rows, int64_t D, T* __restrict__ out) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float s = scale[r];
        for (int64_t c = threadIdx.x; c < D; c += blockDim.x)
            out[r * D + c] = from_f32<T>(unpacked<T>(e4m3_value(payload[r * D + c]), s));
    }
}

// A group of `warps` warps per row, the row in registers: read once.  Rows are independent, so a group takes one at a
// time and the SM's other groups cover its exchange.
template <typename T, bool WIDE, int NV, bool MULTI>
__global__ void __launch_bounds__(512) pack_rows_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int64_t D,
                                                        uint8_t* __restrict__ payload, float* __restrict__ scale, int warps) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N;
    __shared__ uint32_t part[MULTI ? 2 * MAX_ROW_WARPS : 1];
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = MULTI ? threadIdx.x / threads : threadIdx.x >> 5;
    const int gt = threadIdx.x - group * threads;
    const int groups = blockDim.x / threads;
    const int64_t pieces = D / N;
    int parity = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * groups + group; r < rows; r += static_cast<int64_t>(gridDim.x) * groups) {
        typename P::Raw v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = gt + static_cast<int64_t>(i) * threads;
            v[i] = c < pieces ? P::load(x + r * x_stride + c * N) : P::zero();
        }
        bool odd;
        uint32_t top = warp_top<T, WIDE, NV>(v, odd);
        if constexpr (MULTI) {
            uint32_t* slot = part + parity * MAX_ROW_WARPS + group * warps;
            if (lane == 0) slot[gt >> 5] = top;
            group_sync(group, threads);
            for (int k = 0; k < warps; ++k) top = max(top, slot[k]);
            parity ^= 1;                                   // the next row's exchange leaves these slots alone
        }
        const int e = e4m3_scale_exponent(top);
        const float inv = exp2_int(-e);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = gt + static_cast<int64_t>(i) * threads;
            if (c < pieces) *reinterpret_cast<typename P::Packed*>(payload + r * D + c * N) = pack_piece<T, WIDE>(v[i], inv, odd);
        }
        if (gt == 0) scale[r] = exp2_int(e);
    }
}

// One warp per segment of 8 * 32 pieces of a row.
constexpr int SEGMENT = 8;
template <typename T>
__global__ void __launch_bounds__(256) unpack_rows_kernel(const uint8_t* __restrict__ payload, const float* __restrict__ scale,
                                                          int64_t rows, int64_t D, int segments, T* __restrict__ out) {
    using P = Piece<T, true>;
    constexpr int N = P::N;
    const int lane = threadIdx.x & 31;
    const int64_t pieces = D / N, jobs = rows * segments;
    const int64_t stride = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    for (int64_t j = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; j < jobs; j += stride) {
        const int64_t r = segments == 1 ? j : j / segments;
        const int64_t c0 = (j - r * segments) * SEGMENT * 32 + lane;
        const float s = __ldg(scale + r);
        typename P::Packed v[SEGMENT];
#pragma unroll
        for (int i = 0; i < SEGMENT; ++i)
            if (c0 + i * 32 < pieces) v[i] = P::load_packed(payload + r * D + (c0 + i * 32) * N);
#pragma unroll
        for (int i = 0; i < SEGMENT; ++i)
            if (c0 + i * 32 < pieces) {
                float f[N];
                unpack_piece<T, true>(v[i], s, f);
                P::store(out + r * D + (c0 + i * 32) * N, P::encode(f));
            }
    }
}

// Rows at any address, as granules (row_shift.cuh): a ring of rows per group, a barrier behind a row's arrival and one
// before its bytes leave.  16384 x 2001 bf16: pack 39 us, unpack 26 us, against 64 and 37 one value at a time.
template <typename T, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 2) pack_shift_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int64_t D64,
                                                                     uint8_t* __restrict__ payload, float* __restrict__ scale, int warps) {
    using P = Piece<T, true>;
    constexpr int N = P::N, NV = RING_COLUMNS / N, XB = static_cast<int>(sizeof(typename P::Packed));
    extern __shared__ __align__(16) unsigned char ring_smem[];
    __shared__ uint32_t part[2 * MAX_ROW_WARPS];
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads;
    const int groups = blockDim.x / threads, D = static_cast<int>(D64), bytes = D * static_cast<int>(sizeof(T));
    const int room = row_room(threads * RING_COLUMNS, sizeof(T)), room8 = row_room(threads * RING_COLUMNS, 1);
    const uint32_t slot0 = smem_u32(ring_smem) + group * (STAGES * room + 16 + room8), slot_end = slot0 + STAGES * room;
    const uint32_t out8 = slot_end + 16;
    auto sync = [&]() { if (warps > 1) group_sync(group, threads); else __syncwarp(); };
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int left = first < rows ? static_cast<int>((rows - first + step - 1) / step) : 0, to_fetch = left;
    const T* src = x + first * x_stride;
    const T* cur = src;
    uint32_t slot = slot0, fetch_slot = slot0;
    auto fetch = [&](auto head) {
        if (to_fetch > 0) fetch_row<decltype(head)::value>(fetch_slot, src, bytes, gt, threads, x);
        src += step * x_stride;
        --to_fetch;
        fetch_slot += room;
        if (fetch_slot == slot_end) fetch_slot = slot0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(std::true_type());
    for (int k = 1; k < STAGES - 1; ++k) fetch(std::false_type());
    int parity = 0;
    for (int64_t r = first; left > 0; --left, r += step) {
        fetch(std::false_type());
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        sync();                                             // the other threads' granules
        const uint32_t shift = offset16(cur);
        cur += step * x_stride;
        typename P::Raw v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            v[i] = (gt + i * threads) * N < D ? shared_shifted(slot + (gt + i * threads) * 16, shift) : P::zero();
        slot += room;
        if (slot == slot_end) slot = slot0;
        bool odd;
        uint32_t top = warp_top<T, true, NV>(v, odd);
        if (warps > 1) {
            uint32_t* mine = part + parity * MAX_ROW_WARPS + group * warps;
            if (lane == 0) mine[gt >> 5] = top;
            group_sync(group, threads);
            for (int k = 0; k < warps; ++k) top = max(top, mine[k]);
            parity ^= 1;                                    // the next row's exchange leaves these slots alone
        }
        const int e = e4m3_scale_exponent(top);
        const float inv = exp2_int(-e);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((gt + i * threads) * N < D) store_shared(out8 + (gt + i * threads) * XB, pack_piece<T, true>(v[i], inv, odd));
        sync();
        store_row<uint8_t>(payload + r * D, out8, D, gt, threads);
        if (gt == 0) scale[r] = exp2_int(e);
    }
}

template <typename T, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 2) unpack_shift_kernel(const uint8_t* __restrict__ payload, const float* __restrict__ scale,
                                                                       int64_t rows, int64_t D64, T* __restrict__ out_rows, int warps) {
    using P = Piece<T, true>;
    using X = typename P::Packed;
    constexpr int N = P::N, NV = RING_COLUMNS / N, XB = static_cast<int>(sizeof(X));
    extern __shared__ __align__(16) unsigned char ring_smem[];
    const int threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads;
    const int groups = blockDim.x / threads, D = static_cast<int>(D64), bytes = D * static_cast<int>(sizeof(T));
    const int room = row_room(threads * RING_COLUMNS, sizeof(T)), room8 = row_room(threads * RING_COLUMNS, 1);
    const uint32_t slot0 = smem_u32(ring_smem) + group * (STAGES * room8 + 16 + room), slot_end = slot0 + STAGES * room8;
    const uint32_t out = slot_end + 16;
    auto sync = [&]() { if (warps > 1) group_sync(group, threads); else __syncwarp(); };
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int left = first < rows ? static_cast<int>((rows - first + step - 1) / step) : 0;
    int64_t fetch_row_no = first;
    uint32_t slot = slot0, fetch_slot = slot0;
    auto fetch = [&](auto head) {
        if (fetch_row_no < rows) fetch_row<decltype(head)::value>(fetch_slot, payload + fetch_row_no * D, D, gt, threads, payload);
        fetch_row_no += step;
        fetch_slot += room8;
        if (fetch_slot == slot_end) fetch_slot = slot0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(std::true_type());
    for (int k = 1; k < STAGES - 1; ++k) fetch(std::false_type());
    for (int64_t r = first; left > 0; --left, r += step) {
        const float s = __ldg(scale + r);
        fetch(std::false_type());
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        sync();                                             // the other threads' granules; the last row's results have left
        const uint32_t shift = offset16(payload + r * D);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            if (c * N < D) {
                float f[N];
                unpack_piece<T, true>(shared_unaligned<X>(slot + shift + c * XB), s, f);
                store_shared(out + c * 16, P::encode(f));
            }
        }
        slot += room8;
        if (slot == slot_end) slot = slot0;
        sync();
        store_row<T>(out_rows + r * D, out, bytes, gt, threads);
    }
}

template <typename T, bool WIDE, int NV>
cudaError_t pack_launch(const T* x, int64_t x_stride, int64_t rows, int64_t D, uint8_t* payload, float* scale, const RowShape& h,
                        cudaStream_t s) {
    const int64_t need = (rows + h.groups - 1) / h.groups;
    const unsigned grid = static_cast<unsigned>(need < GRID_SMS * 16 ? need : GRID_SMS * 16), threads = h.warps * h.groups * 32;
    if constexpr (NV < 16) {                                 // sixteen values a thread: rows of nine warps and more
        if (h.warps == 1) {
            pack_rows_kernel<T, WIDE, NV, false><<<grid, threads, 0, s>>>(x, x_stride, rows, D, payload, scale, h.warps);
            return cudaGetLastError();
        }
    }
    if constexpr (!WIDE || NV == 1 || NV == 8) {             // two and four pieces: what brings a row down to one warp
        pack_rows_kernel<T, WIDE, NV, true><<<grid, threads, 0, s>>>(x, x_stride, rows, D, payload, scale, h.warps);
        return cudaGetLastError();
    }
    return cudaErrorInvalidValue;
}

constexpr int64_t SHIFT_ROWS = 1024;      // fewer rows: latency, not the loads' width, decides

template <typename T>
cudaError_t pack_t(const void* xv, int64_t x_stride, int64_t rows, int64_t D, uint8_t* payload, float* scale, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const T* x = static_cast<const T*>(xv);
    const bool wide = D % N == 0 && x_stride % N == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(payload) & (N - 1)) == 0;
    if (!wide && rows >= SHIFT_ROWS && D >= 512 && ring_warps(D) <= MAX_ROW_WARPS &&
        first_row_alone(x, x_stride * static_cast<int64_t>(sizeof(T)), rows)) {      // 32768 x 65: 19 us against 10
        constexpr int STAGES = 4;
        const int warps = ring_warps(D), groups = MAX_ROW_WARPS / warps, columns = warps * 32 * RING_COLUMNS;
        const int smem = groups * (STAGES * row_room(columns, sizeof(T)) + 16 + row_room(columns, 1));
        const cudaError_t e = cudaFuncSetAttribute(pack_shift_kernel<T, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        const int64_t need = (rows + groups - 1) / groups, cap = GRID_SMS * (sizeof(T) == 4 ? 1 : 2);
        pack_shift_kernel<T, STAGES><<<static_cast<unsigned>(need < cap ? need : cap), groups * warps * 32, smem, s>>>(x, x_stride, rows, D, payload, scale, warps);
        return cudaGetLastError();
    }
    const RowShape h = wide ? row_shape(rows, D / N, 1, 8, 8) : narrow_shape(rows, D, 8);
    if (h.warps == 0) {
        const unsigned grid = static_cast<unsigned>(rows < GRID_SMS * 64 ? rows : GRID_SMS * 64);
        pack_rows_loop_kernel<T><<<grid, 256, 0, s>>>(x, x_stride, rows, D, payload, scale);
        return cudaGetLastError();
    }
    if (!wide) return h.nv == 4 ? pack_launch<T, false, 4>(x, x_stride, rows, D, payload, scale, h, s)
                    : h.nv == 8 ? pack_launch<T, false, 8>(x, x_stride, rows, D, payload, scale, h, s)
                                : pack_launch<T, false, 16>(x, x_stride, rows, D, payload, scale, h, s);
    switch (h.nv) {
        case 1: return pack_launch<T, true, 1>(x, x_stride, rows, D, payload, scale, h, s);
        case 2: return pack_launch<T, true, 2>(x, x_stride, rows, D, payload, scale, h, s);
        case 4: return pack_launch<T, true, 4>(x, x_stride, rows, D, payload, scale, h, s);
        default: return pack_launch<T, true, 8>(x, x_stride, rows, D, payload, scale, h, s);
    }
}

template <typename T>
cudaError_t unpack_t(const uint8_t* payload, const float* scale, int64_t rows, int64_t D, void* out, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (D % N == 0 && aligned16(out) && (reinterpret_cast<uintptr_t>(payload) & (N - 1)) == 0) {
        const int segments = static_cast<int>((D / N + SEGMENT * 32 - 1) / (SEGMENT * 32));
        const int64_t blocks = (rows * segments + 7) / 8;
        const unsigned grid = static_cast<unsigned>(blocks < GRID_SMS * 64 ? blocks : GRID_SMS * 64);
        unpack_rows_kernel<T><<<grid, 256, 0, s>>>(payload, scale, rows, D, segments, static_cast<T*>(out));
        return cudaGetLastError();
    }
    if (rows >= SHIFT_ROWS && ring_warps(D) <= MAX_ROW_WARPS && first_row_alone(payload, D, rows)) {
        constexpr int STAGES = 4;
        const int warps = ring_warps(D), groups = MAX_ROW_WARPS / warps, columns = warps * 32 * RING_COLUMNS;
        const int smem = groups * (STAGES * row_room(columns, 1) + 16 + row_room(columns, sizeof(T)));
        const cudaError_t e = cudaFuncSetAttribute(unpack_shift_kernel<T, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        const int64_t need = (rows + groups - 1) / groups, cap = GRID_SMS * 2;
        unpack_shift_kernel<T, STAGES><<<static_cast<unsigned>(need < cap ? need : cap), groups * warps * 32, smem, s>>>(
            payload, scale, rows, D, static_cast<T*>(out), warps);
        return cudaGetLastError();
    }
    const unsigned grid = static_cast<unsigned>(rows < GRID_SMS * 64 ? rows : GRID_SMS * 64);
    unpack_rows_loop_kernel<T><<<grid, 256, 0, s>>>(payload, scale, rows, D, static_cast<T*>(out));
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

}  // namespace
}  // namespace peer

using namespace peer;

extern "C" int peer_pack_rows(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t dim, void* payload,
                              float* scale, void* stream) {
    if (rows < 0 || dim < 1 || dim > PEER_ROW_DIM_MAX || x_stride < 0)
        return refuse("peer_pack_rows: negative row count or stride, or dim outside [1, 2^20]");
    if (rows == 0) return PEER_OK;
    if (!x || !payload || !scale) return refuse("peer_pack_rows: null pointer");
    if (!aligned_to(x, dtype) || !aligned_to(scale, PEER_DTYPE_F32)) return refuse("peer_pack_rows: a pointer is not aligned to its type");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* p = static_cast<uint8_t*>(payload);
    if (dtype == PEER_DTYPE_F32) return report("peer_pack_rows", pack_t<float>(x, x_stride, rows, dim, p, scale, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_pack_rows", pack_t<__nv_bfloat16>(x, x_stride, rows, dim, p, scale, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_pack_rows", pack_t<__half>(x, x_stride, rows, dim, p, scale, s));
    return refuse("peer_pack_rows: dtype must be F32, BF16 or F16");
}

extern "C" int peer_unpack_rows(const void* payload, const float* scale, int32_t dtype, int64_t rows, int64_t dim, void* out,
                                void* stream) {
    if (rows < 0 || dim < 1 || dim > PEER_ROW_DIM_MAX)
        return refuse("peer_unpack_rows: negative row count, or dim outside [1, 2^20]");
    if (rows == 0) return PEER_OK;
    if (!payload || !scale || !out) return refuse("peer_unpack_rows: null pointer");
    if (!aligned_to(out, dtype) || !aligned_to(scale, PEER_DTYPE_F32)) return refuse("peer_unpack_rows: a pointer is not aligned to its type");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint8_t* p = static_cast<const uint8_t*>(payload);
    if (dtype == PEER_DTYPE_F32) return report("peer_unpack_rows", unpack_t<float>(p, scale, rows, dim, out, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_unpack_rows", unpack_t<__nv_bfloat16>(p, scale, rows, dim, out, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_unpack_rows", unpack_t<__half>(p, scale, rows, dim, out, s));
    return refuse("peer_unpack_rows: dtype must be F32, BF16 or F16");
}
