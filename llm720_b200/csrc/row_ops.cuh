// Helpers shared by the row-wise operators (layer norm, 8-bit row packing,
// embedding): the row-scaled e4m3 format and block-wide sums.
#pragma once

#include "common.cuh"

namespace peer {

// ---------------------------------------------------------------------------
// Row-scaled e4m3.  A row is stored as one byte per value and one fp32 scale, the smallest power of two s with
// max|x| / s <= 448 (the format's largest value); the maximum is taken over the row's finite values, s = 1 for a row
// of zeros and s >= 2^-126 so that 1/s is finite.  With a power of two x/s and payload*s are exact, so the only
// rounding is the one to e4m3 (nearest even, at most 2^-4 relative above the format's subnormals), and every
// implementation of the definition gives the same bytes.  It costs no precision against s = max|x|/448, e4m3 being a
// floating-point format, only up to one binade of the 17.8 at the small end.  e4m3 has no infinity: infinite and
// NaN values become NaN.
// ---------------------------------------------------------------------------
constexpr uint32_t F32_INF_BITS = 0x7f800000u;

// |v| as bits, 0 when v is infinite or NaN: the row maximum of these is the bits of the largest finite magnitude
__device__ __forceinline__ uint32_t finite_abs_bits(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < F32_INF_BITS ? b : 0u;
}
// exponent of the scale for a largest magnitude given as bits
__device__ __forceinline__ int e4m3_scale_exponent(uint32_t amax_bits) {
    if (amax_bits == 0u) return 0;
    // 448 = 1.75 * 2^8; a magnitude 1.m * 2^E needs 2^(E-8) when 1.m <= 1.75, else 2^(E-7)
    const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;                          // subnormal fp32 magnitudes end here too
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float e4m3_operand(float v, float inv_scale) {
    return (__float_as_uint(v) & 0x7fffffffu) < F32_INF_BITS ? v * inv_scale : __uint_as_float(0x7fffffffu);
}
// two values, already divided by the scale, to two bytes (a in the low one)
__device__ __forceinline__ uint16_t e4m3_pair(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3_pair_values(uint16_t p) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(p, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float e4m3_value(uint8_t p) { return e4m3_pair_values(p).x; }

// largest finite value of a storage type.  Rounding up in e4m3 can pass it in the topmost binade (65504 -> 65536
// for fp16); what a packed value stands for is clamped there.
template <typename T> __device__ __forceinline__ float max_finite();
template <> __device__ __forceinline__ float max_finite<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float max_finite<__nv_bfloat16>() { return 3.389531390e38f; }
template <> __device__ __forceinline__ float max_finite<__half>() { return 65504.0f; }
template <typename T> __device__ __forceinline__ float unpacked(float payload_value, float scale) {
    const float v = payload_value * scale;
    return fabsf(v) > max_finite<T>() ? copysignf(max_finite<T>(), v) : v;     // NaN stays NaN
}

__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) { return __reduce_max_sync(FULL_MASK, v); }

// Sum of one value per thread over the block; every thread gets the result.  `buf` holds 33 floats.  Ends with the
// buffer free for the next call.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    v = warp_sum(v);
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const float t = warp_sum(lane < warps ? buf[lane] : 0.f);
        if (lane == 0) buf[32] = t;
    }
    __syncthreads();
    const float r = buf[32];
    __syncthreads();
    return r;
}
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, float* buf) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    uint32_t* b = reinterpret_cast<uint32_t*>(buf);
    v = warp_max_u32(v);
    if (lane == 0) b[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const uint32_t t = warp_max_u32(lane < warps ? b[lane] : 0u);
        if (lane == 0) b[32] = t;
    }
    __syncthreads();
    const uint32_t r = b[32];
    __syncthreads();
    return r;
}

// parameter vectors come in the activations' type or in fp32
template <typename T> __device__ __forceinline__ float param_at(const void* p, bool f32, int64_t i) {
    return f32 ? static_cast<const float*>(p)[i] : to_f32<T>(static_cast<const T*>(p)[i]);
}

}  // namespace peer
