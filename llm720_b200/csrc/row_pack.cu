// Activation checkpoints in 8 bits: rows to row-scaled e4m3 and back
// (the format is defined in row_ops.cuh).  Packing reads 2 (4) bytes and writes
// 1 per value, unpacking the reverse: both are bound by HBM.
#include <cstdio>

#include "kernels.h"
#include "row_ops.cuh"

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

template <typename T>
cudaError_t pack_t(const void* x, int64_t x_stride, int64_t rows, int64_t D, uint8_t* payload, float* scale, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(rows < 148 * 64 ? rows : 148 * 64);
    pack_rows_loop_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(x), x_stride, rows, D, payload, scale);
    return cudaGetLastError();
}

template <typename T>
cudaError_t unpack_t(const uint8_t* payload, const float* scale, int64_t rows, int64_t D, void* out, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(rows < 148 * 64 ? rows : 148 * 64);
    unpack_rows_loop_kernel<T><<<grid, 256, 0, s>>>(payload, scale, rows, D, static_cast<T*>(out));
    return cudaGetLastError();
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

}  // namespace
}  // namespace peer

using namespace peer;

extern "C" int peer_pack_rows(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t dim, void* payload,
                              float* scale, void* stream) {
    if (rows < 0 || dim < 1 || dim > PEER_ROW_DIM_MAX || x_stride < 0)
        return refuse("peer_pack_rows: negative row count or stride, or dim outside [1, 2^20]");
    if (rows == 0) return PEER_OK;
    if (!x || !payload || !scale) return refuse("peer_pack_rows: null pointer");
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint8_t* p = static_cast<const uint8_t*>(payload);
    if (dtype == PEER_DTYPE_F32) return report("peer_unpack_rows", unpack_t<float>(p, scale, rows, dim, out, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_unpack_rows", unpack_t<__nv_bfloat16>(p, scale, rows, dim, out, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_unpack_rows", unpack_t<__half>(p, scale, rows, dim, out, s));
    return refuse("peer_unpack_rows: dtype must be F32, BF16 or F16");
}
