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
// A row with such a scale may hold values that need the clamp, 448 * |scale| being above the type's largest.  The limit, 2^7 or
// 2^119, is the largest power of two below that; a caller's own scale may be any number, negative or NaN.
template <typename T> __device__ __forceinline__ bool may_clamp(float scale) {
    return !(fabsf(scale) <= (max_finite<T>() < 1e5f ? 128.f : 6.646139979e35f));
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


// 16, 8 or 4 bytes from global to shared memory, asynchronously
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// shared to global memory, asynchronously: addresses and size multiples of 16 bytes.  The wait covers the calling thread's
// copies and comes before the block ends.
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_s2g_wait() {
    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------
// Pieces of a row: what one thread loads at once.  Wide: 16 bytes (rows whose start, stride and width are multiples
// of 16 bytes); narrow: one value.
// ---------------------------------------------------------------------------
template <typename T, bool WIDE> struct Piece;
template <typename T> struct Piece<T, false> {
    static constexpr int N = 1;
    using Raw = T;
    using Packed = uint8_t;
    __device__ static __forceinline__ Raw zero() { return from_f32<T>(0.f); }
    __device__ static __forceinline__ Raw load(const T* p) { return __ldg(p); }
    __device__ static __forceinline__ void store(T* p, const Raw& r) { *p = r; }
    __device__ static __forceinline__ void decode(const Raw& r, float (&f)[1]) { f[0] = to_f32<T>(r); }
    __device__ static __forceinline__ Raw encode(const float (&f)[1]) { return from_f32<T>(f[0]); }
    __device__ static __forceinline__ Packed load_packed(const uint8_t* p) { return __ldg(p); }
    __device__ static __forceinline__ void decode_packed(const Packed& r, float (&f)[1]) { f[0] = e4m3_value(r); }
    __device__ static __forceinline__ Packed encode_packed(const float (&f)[1]) { return static_cast<uint8_t>(e4m3_pair(f[0], 0.f)); }
};
template <> struct Piece<float, true> {
    static constexpr int N = 4;
    using Raw = uint4;
    using Packed = uint32_t;
    __device__ static __forceinline__ Raw zero() { return make_uint4(0u, 0u, 0u, 0u); }
    __device__ static __forceinline__ Raw load(const float* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ static __forceinline__ void store(float* p, const Raw& r) { *reinterpret_cast<uint4*>(p) = r; }
    __device__ static __forceinline__ void decode(const Raw& r, float (&f)[4]) {
        f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
    }
    __device__ static __forceinline__ Raw encode(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    __device__ static __forceinline__ Packed load_packed(const uint8_t* p) { return __ldg(reinterpret_cast<const uint32_t*>(p)); }
    __device__ static __forceinline__ void decode_packed(const Packed& r, float (&f)[4]) {
        const float2 a = e4m3_pair_values(static_cast<uint16_t>(r)), b = e4m3_pair_values(static_cast<uint16_t>(r >> 16));
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
    __device__ static __forceinline__ Packed encode_packed(const float (&f)[4]) {
        return e4m3_pair(f[0], f[1]) | (static_cast<uint32_t>(e4m3_pair(f[2], f[3])) << 16);
    }
};
template <typename T> struct Piece<T, true> {
    static constexpr int N = 8;
    using Raw = uint4;
    using Packed = uint2;
    __device__ static __forceinline__ Raw zero() { return make_uint4(0u, 0u, 0u, 0u); }
    __device__ static __forceinline__ Raw load(const T* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ static __forceinline__ void store(T* p, const Raw& r) { *reinterpret_cast<uint4*>(p) = r; }
    __device__ static __forceinline__ void decode(const Raw& r, float (&f)[8]) {
        const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = to_f32<T>(e[q]);
    }
    __device__ static __forceinline__ Raw encode(const float (&f)[8]) {
        uint4 r;
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int q = 0; q < 8; ++q) e[q] = from_f32<T>(f[q]);
        return r;
    }
    __device__ static __forceinline__ Packed load_packed(const uint8_t* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }
    __device__ static __forceinline__ void decode_packed(const Packed& r, float (&f)[8]) {
        const uint32_t h[2] = {r.x, r.y};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float2 a = e4m3_pair_values(static_cast<uint16_t>(h[q >> 1] >> (16 * (q & 1))));
            f[2 * q] = a.x;
            f[2 * q + 1] = a.y;
        }
    }
    __device__ static __forceinline__ Packed encode_packed(const float (&f)[8]) {
        return make_uint2(e4m3_pair(f[0], f[1]) | (static_cast<uint32_t>(e4m3_pair(f[2], f[3])) << 16),
                          e4m3_pair(f[4], f[5]) | (static_cast<uint32_t>(e4m3_pair(f[6], f[7])) << 16));
    }
};

// a piece's values from its packed form
template <typename T, bool WIDE>
__device__ __forceinline__ void unpack_piece(const typename Piece<T, WIDE>::Packed& r, float scale, float (&f)[Piece<T, WIDE>::N]) {
    Piece<T, WIDE>::decode_packed(r, f);
    if (may_clamp<T>(scale)) {                              // the same for the whole row
#pragma unroll
        for (int q = 0; q < Piece<T, WIDE>::N; ++q) f[q] = unpacked<T>(f[q], scale);
    } else {
#pragma unroll
        for (int q = 0; q < Piece<T, WIDE>::N; ++q) f[q] *= scale;
    }
}

// Largest magnitude of raw pieces as an unsigned number in the storage type's own bit pattern (two 16-bit lanes per
// word: `join` folds them), which orders like the magnitude itself; at `not_finite` or above it an infinity or NaN was
// among them.  One logic and one maximum instruction per word instead of a conversion per value.
template <typename T> struct Magnitude;
template <> struct Magnitude<float> {
    static constexpr uint32_t not_finite = F32_INF_BITS;
    __device__ static __forceinline__ uint32_t fold(uint32_t m, const float& v) { return max(m, __float_as_uint(v) & 0x7fffffffu); }
    __device__ static __forceinline__ uint32_t fold(uint32_t m, const uint4& v) {
        return max(max(max(m, v.x & 0x7fffffffu), v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
    }
    __device__ static __forceinline__ uint32_t join(uint32_t m) { return m; }
    __device__ static __forceinline__ uint32_t f32_bits(uint32_t m) { return m; }
};
template <typename T> struct Magnitude16 {
    __device__ static __forceinline__ uint32_t fold(uint32_t m, const T& v) { return __vmaxu2(m, *reinterpret_cast<const uint16_t*>(&v) & 0x7fffu); }
    __device__ static __forceinline__ uint32_t fold(uint32_t m, const uint4& v) {
        m = __vmaxu2(m, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu));
        return __vmaxu2(m, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    }
    __device__ static __forceinline__ uint32_t join(uint32_t m) { return max(m & 0xffffu, m >> 16); }
};
template <> struct Magnitude<__nv_bfloat16> : Magnitude16<__nv_bfloat16> {
    static constexpr uint32_t not_finite = 0x7f80u;
    __device__ static __forceinline__ uint32_t f32_bits(uint32_t m) { return m << 16; }
};
template <> struct Magnitude<__half> : Magnitude16<__half> {
    static constexpr uint32_t not_finite = 0x7c00u;
    __device__ static __forceinline__ uint32_t f32_bits(uint32_t m) {
        return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
    }
};
// Largest finite magnitude (fp32 bits) over the warp's pieces; `odd`: the warp holds an infinity or NaN somewhere.
template <typename T, bool WIDE, int NV>
__device__ __forceinline__ uint32_t warp_top(const typename Piece<T, WIDE>::Raw (&x)[NV], bool& odd) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = Magnitude<T>::fold(m, x[i]);
    m = warp_max_u32(Magnitude<T>::join(m));
    odd = m >= Magnitude<T>::not_finite;
    if (!odd) return Magnitude<T>::f32_bits(m);
    m = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[Piece<T, WIDE>::N];
        Piece<T, WIDE>::decode(x[i], f);
#pragma unroll
        for (int q = 0; q < Piece<T, WIDE>::N; ++q) m = max(m, finite_abs_bits(f[q]));
    }
    return warp_max_u32(m);
}
// a piece in 8 bits; infinities and NaN are looked for only where the warp has some
template <typename T, bool WIDE>
__device__ __forceinline__ typename Piece<T, WIDE>::Packed pack_piece(const typename Piece<T, WIDE>::Raw& x, float inv, bool odd) {
    constexpr int N = Piece<T, WIDE>::N;
    float f[N];
    Piece<T, WIDE>::decode(x, f);
    if (odd) {
#pragma unroll
        for (int q = 0; q < N; ++q) f[q] = e4m3_operand(f[q], inv);
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) f[q] *= inv;
    }
    return Piece<T, WIDE>::encode_packed(f);
}

// the same from values decoded before; `x` is looked at only when the warp holds infinities or NaN
template <typename T>
__device__ __forceinline__ typename Piece<T, true>::Packed pack_pairs(const float2 (&v)[Piece<T, true>::N / 2], const uint4& x, float inv, bool odd) {
    constexpr int N = Piece<T, true>::N;
    if (odd) return pack_piece<T, true>(x, inv, true);
    float f[N];
#pragma unroll
    for (int h = 0; h < N / 2; ++h) {
        const float2 s = __fmul2_rn(v[h], make_float2(inv, inv));
        f[2 * h] = s.x;
        f[2 * h + 1] = s.y;
    }
    return Piece<T, true>::encode_packed(f);
}

// Sums of K values (a power of two) over the warp in K - 1 + 5 - log2(K) shuffles: each step halves the values a lane
// carries.  On return lane k * (32 / K) (and its neighbours up to the next) holds the sum of v[k] as the result.
template <int K>
__device__ __forceinline__ float warp_sums(float (&v)[K]) {
    const int lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int half = K / 2; half >= 1; half >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = up ? v[i] : v[i + half];
            const float keep = up ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(FULL_MASK, give, o);
        }
        o >>= 1;
    }
    float r = v[0];
#pragma unroll
    for (; o > 0; o >>= 1) r += __shfl_xor_sync(FULL_MASK, r, o);
    return r;
}

// barrier of one of several row groups of a block (ids 1 .. groups); one group: the block's
__device__ __forceinline__ void group_sync(int group, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}


// ---------------------------------------------------------------------------
// Programmatic dependent launch: a kernel launched with `launch_behind` may be set up while the one before it in the
// stream still runs.  `grid_wait` in it returns when that one has completed and its writes are visible; `grid_release`
// in the earlier kernel says that a block no longer minds.  Saves the 2 us between a kernel and a short one behind it.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
inline cudaError_t launch_behind_smem(void (*kernel)(Params...), dim3 grid, dim3 block, int smem, cudaStream_t s, Args... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
    if (e != cudaSuccess) cudaGetLastError();               // reported here, not by the next launch's check
    return e;
}
template <typename... Params, typename... Args>
inline cudaError_t launch_behind(void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t s, Args... args) {
    return launch_behind_smem(kernel, grid, block, 0, s, args...);
}

// ---------------------------------------------------------------------------
// How a row is spread over threads: `warps` warps per row, `groups` rows' worth of warps per block, nv pieces per
// thread.  warps == 0: the row is longer than MAX_ROW_WARPS warps take.
// ---------------------------------------------------------------------------
constexpr int MAX_ROW_WARPS = 16;
constexpr int GRID_SMS = 148;
struct RowShape { int warps, groups, nv; };

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned_to(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == PEER_DTYPE_F32 ? 3u : 1u)) == 0; }

// Many rows: up to nv_max pieces per thread (doubling from nv_min until one warp takes the row), so that a row needs
// few warps and few exchanges between them.  Fewer than 1024 rows (under seven per SM): nv_min, a row is then spread
// wider and finished sooner.
inline RowShape row_shape(int64_t rows, int64_t pieces, int nv_min, int nv_max, int block_warps) {
    RowShape s{};
    s.nv = nv_min;
    if (rows >= 1024 || pieces > 32 * MAX_ROW_WARPS * nv_min)
        while (s.nv < nv_max && pieces > 32 * s.nv) s.nv *= 2;
    const int64_t warps = (pieces + 32 * s.nv - 1) / (32 * s.nv);
    if (warps > MAX_ROW_WARPS) return s;
    s.warps = static_cast<int>(warps);
    s.groups = block_warps / s.warps < 1 ? 1 : block_warps / s.warps;
    return s;
}

// rows that are not whole 16-byte pieces: one value at a time, 8 per thread (16 spill) unless the row is wider
inline RowShape narrow_shape(int64_t rows, int64_t D, int block_warps) {
    return row_shape(rows, D, 4, D <= 32 * MAX_ROW_WARPS * 8 ? 8 : 16, block_warps);
}

}  // namespace peer
