// Layer norm with its backward pass, for training: the `ln_2` of the
// reference's TransformerBlock (llm/models/foundation.py:118, 196-199) as an
// operator of its own.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), n = (x - m) r, y = n w + b
//   g = dy w,  dx = r (g - mean(g) - n mean(g n)),  dw = sum_rows dy n,  db = sum_rows dy
//
// The backward pass takes x as it was, or from its 8-bit form (row_ops.cuh)
// that the forward pass wrote beside y; m and r are those of the exact x either
// way.  All sums are fp32; the column sums are added in a fixed order (per row
// split, then over the splits), so results do not vary from run to run.
#include <cstdio>
#include <type_traits>

#include "kernels.h"
#include "row_ops.cuh"
#include "row_shift.cuh"

namespace peer {
void set_global_error(const char* msg);

namespace {

struct NormParams {
    const void* x; int64_t x_stride;
    const void* w; const void* b; bool param_f32;
    float eps; int64_t rows, D;
    void* y; float* mean; float* rstd;
    uint8_t* payload; float* scale;
};

struct NormGradParams {
    const void* dy; int64_t dy_stride;
    const void* x; int64_t x_stride;
    const uint8_t* payload; const float* scale;
    const float* mean; const float* rstd;
    const void* w; bool param_f32;
    const void* add;                 // optional [rows, D]: added to dx (the gradient of a residual branch)
    int64_t rows, D;
    void* dx; void* dw; void* db;
    float* partial;                  // [splits][2][D]
    int splits;
};

// ---------------------------------------------------------------------------
// Rows in registers.  A group of `warps` warps owns a row; every thread holds the same NV pieces of columns in every row,
// and one exchange between the group's warps joins their sums.
//
// Forward statistics (here and below): each warp takes the mean of its own columns, rounded, as a center c and sums the
// deviations from it, s = sum(x - c), and their squares, q.  About any one center c0 a warp's n columns then have
//   sum(x - c0) = s + n e =: t,   sum(x - c0)^2 = q + e (s + t),   e = c - c0,
// so one exchange of (c, q, s) gives the row's  mean = c0 + T / D  and  M2 = Q - T^2 / D  with T, Q summed over the warps.  The
// centers cancel: without s the roundings of the warps' means (2^-24 of the mean) would enter M2 times the distance between the
// warps' means (530 fp32 values of 1000 +- 0.5: a deviation off by 250 * 2^-24 and more; the mean, too, is only as good).  c0 is
// the first warp's center, which lies within four deviations of the mean (it holds 1/16 of the columns at least), mostly far less.
// For the 16-bit types s costs no pass: where the mean is large against the deviation the values share their leading bits, a
// warp's sum S of at most 2,048 of them is exact in fp32, and s = S - n c is one fma (zero where n is a power of two, as in rows of
// 512 W columns); elsewhere its rounding is one of the values' magnitude, as everywhere.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void add_part(float c0, float c, float q, float s, float n, float& t_all, float& q_all) {
    const float e = c - c0, t = fmaf(n, e, s);
    t_all += t;
    q_all += fmaf(e, s + t, q);
}
// T, Q about c0 to the mean and M2, which rounding can take below zero and overflow to inf - inf; rows with an infinity or NaN
// have a mean of NaN
__device__ __forceinline__ void finish_stats(float c0, float t, float q, float inv_d, float& mean, float& m2) {
    const float off = t * inv_d, inf = __uint_as_float(F32_INF_BITS);
    mean = c0 + off;
    m2 = fmaf(-t, off, q);
    if (!(m2 >= 0.f)) m2 = fabsf(mean) < inf ? (fabsf(q) < inf ? 0.f : inf) : q;
}
constexpr int MAX_WARPS = MAX_ROW_WARPS;

// any width, any alignment: one block per row
template <typename T>
__global__ void __launch_bounds__(256) norm_loop_kernel(const NormParams p) {
    __shared__ float buf[33];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* xr = static_cast<const T*>(p.x) + r * p.x_stride;
        float s = 0.f;
        uint32_t top = 0u;
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) {
            const float v = to_f32<T>(xr[c]);
            s += v;
            top = max(top, finite_abs_bits(v));
        }
        const float inv_d = 1.f / static_cast<float>(p.D), center = block_sum(s, buf) * inv_d;
        float q = 0.f;
        s = 0.f;
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) {
            const float d = to_f32<T>(xr[c]) - center;
            s += d;
            q = fmaf(d, d, q);
        }
        s = block_sum(s, buf);
        q = block_sum(q, buf);
        float mean, m2;
        finish_stats(center, s, q, inv_d, mean, m2);
        const float rstd = 1.0f / sqrtf(m2 * inv_d + p.eps);
        T* yr = static_cast<T*>(p.y) + r * p.D;
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) {
            float v = (to_f32<T>(xr[c]) - mean) * rstd;
            if (p.w) v *= param_at<T>(p.w, p.param_f32, c);
            if (p.b) v += param_at<T>(p.b, p.param_f32, c);
            yr[c] = from_f32<T>(v);
        }
        if (p.payload) {
            const int e = e4m3_scale_exponent(block_max_u32(top, buf));
            const float inv = exp2_int(-e);
            for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x)
                p.payload[r * p.D + c] = static_cast<uint8_t>(e4m3_pair(e4m3_operand(to_f32<T>(xr[c]), inv), 0.f));
            if (threadIdx.x == 0) p.scale[r] = exp2_int(e);
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
    }
}

template <typename T, int NV, int N>
__device__ __forceinline__ void load_params(const void* p, bool f32, int64_t D, int first, int step, float absent, float (&f)[NV * N]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (first + static_cast<int64_t>(i) * step) * N;
#pragma unroll
        for (int q = 0; q < N; ++q) f[i * N + q] = (p && c < D) ? param_at<T>(p, f32, c + q) : absent;
    }
}

template <typename T, int N>
__device__ __forceinline__ void load_param_piece(const void* p, bool f32, int64_t c, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = param_at<T>(p, f32, c);
    } else if (f32) {
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + q));
            f[q] = v.x; f[q + 1] = v.y; f[q + 2] = v.z; f[q + 3] = v.w;
        }
    } else {
        Piece<T, true>::decode(Piece<T, true>::load(static_cast<const T*>(p) + c), f);
    }
}

// Forward of few rows, of rows too wide for the ring below, and of narrow rows at odd addresses.  A row per group and at
// most 64 values per thread; the parameters come from L1.
template <typename T, bool WIDE, int NV, bool MULTI, bool PACK>
__global__ void __launch_bounds__(512, 2) norm_kernel(const NormParams p, int warps) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N;
    __shared__ float2 part[MULTI ? 2 * MAX_WARPS : 1];     // center and squares of a warp
    __shared__ float part_sum[MULTI ? 2 * MAX_WARPS : 1];
    __shared__ uint32_t part_top[MULTI && PACK ? 2 * MAX_WARPS : 1];
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = MULTI ? threadIdx.x / threads : threadIdx.x >> 5;
    const int gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    const int pieces = static_cast<int>(p.D / N);
    auto columns_of = [&](int wi) {                        // columns held by warp wi of the group
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) n += min(max(pieces - (i * threads + wi * 32), 0), 32);
        return static_cast<float>(n * N);
    };
    const float mine = columns_of(gw), inv_mine = mine > 0.f ? 1.f / mine : 0.f;
    const float inv_d = 1.f / static_cast<float>(p.D);
    int parity = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * groups + group; r < p.rows; r += static_cast<int64_t>(gridDim.x) * groups) {
        const T* xr = static_cast<const T*>(p.x) + r * p.x_stride;
        typename P::Raw x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            x[i] = c < pieces ? P::load(xr + c * N) : P::zero();
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[N];
            P::decode(x[i], f);
#pragma unroll
            for (int q = 0; q < N; ++q) s += f[q];
        }
        bool odd = false;                                   // the warp holds an infinity or NaN of this row
        uint32_t top = 0u;
        if (PACK) top = warp_top<T, WIDE, NV>(x, odd);
        s = warp_sum(s);
        float mean = s * inv_mine, m2 = 0.f;                // the warp's center, deviations from it and their squares
        s = sizeof(T) == 2 ? fmaf(-mine, mean, s) : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (gt + i * threads < pieces) {
                float f[N];
                P::decode(x[i], f);
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float d = f[q] - mean;
                    if (sizeof(T) == 4) s += d;
                    m2 = fmaf(d, d, m2);
                }
            }
        }
        if constexpr (sizeof(T) == 4) s = warp_sum(s);
        m2 = warp_sum(m2);
        if constexpr (!MULTI) {
            finish_stats(mean, s, m2, inv_d, mean, m2);
        } else {
            const int at = parity * MAX_WARPS + group * warps;
            if (lane == 0) {
                part[at + gw] = make_float2(mean, m2);
                part_sum[at + gw] = s;
                if (PACK) part_top[at + gw] = top;
            }
            group_sync(group, threads);
            const float c0 = part[at].x;
            float t = 0.f, q = 0.f;
            for (int k = 0; k < warps; ++k) {
                const float2 v = part[at + k];
                add_part(c0, v.x, v.y, part_sum[at + k], columns_of(k), t, q);
                if (PACK) top = max(top, part_top[at + k]);
            }
            finish_stats(c0, t, q, inv_d, mean, m2);
            parity ^= 1;                                    // the next row's exchange leaves these slots alone
        }
        const float rstd = 1.f / sqrtf(m2 * inv_d + p.eps);
        const int e = PACK ? e4m3_scale_exponent(top) : 0;
        const float inv = exp2_int(-e);
        T* yr = static_cast<T*>(p.y) + r * p.D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            if (c < pieces) {
                float f[N], v[N];
                P::decode(x[i], f);
#pragma unroll
                for (int q = 0; q < N; ++q) f[q] = (f[q] - mean) * rstd;
                if (p.w) {
                    load_param_piece<T, N>(p.w, p.param_f32, c * N, v);
#pragma unroll
                    for (int q = 0; q < N; ++q) f[q] *= v[q];
                }
                if (p.b) {
                    load_param_piece<T, N>(p.b, p.param_f32, c * N, v);
#pragma unroll
                    for (int q = 0; q < N; ++q) f[q] += v[q];
                }
                P::store(yr + c * N, P::encode(f));
                if constexpr (PACK)
                    *reinterpret_cast<typename P::Packed*>(p.payload + r * p.D + c * N) = pack_piece<T, WIDE>(x[i], inv, odd);
            }
        }
        if (gt == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
            if (PACK) p.scale[r] = exp2_int(e);
        }
    }
}

// Backward of few rows and of narrow rows at odd addresses: at most 16 values per thread, so the column sums stay in
// registers until the end.  KEPT: x comes in its 8-bit form.
template <typename T, bool WIDE, int NV, bool MULTI, bool KEPT>
__global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradParams p, int warps) {
    using P = Piece<T, WIDE>;
    using X = typename std::conditional<KEPT, typename P::Packed, typename P::Raw>::type;
    constexpr int N = P::N, E = NV * N;
    __shared__ float2 part[MULTI ? 2 * MAX_WARPS : 1];
    extern __shared__ float columns[];                     // [2][threads * E] when the block has several groups
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = MULTI ? threadIdx.x / threads : threadIdx.x >> 5;
    const int gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    const int pieces = static_cast<int>(p.D / N);
    float w[E], aw[E], ab[E];
    load_params<T, NV, N>(p.w, p.param_f32, p.D, gt, threads, 1.f, w);
#pragma unroll
    for (int q = 0; q < E; ++q) aw[q] = ab[q] = 0.f;
    const float inv_d = 1.f / static_cast<float>(p.D);
    int parity = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * groups + group; r < p.rows; r += static_cast<int64_t>(gridDim.x) * groups) {
        X x[NV];
        typename P::Raw dy[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            const bool in = c < pieces;
            dy[i] = in ? P::load(static_cast<const T*>(p.dy) + r * p.dy_stride + c * N) : P::zero();
            if constexpr (KEPT) x[i] = in ? P::load_packed(p.payload + r * p.D + c * N) : X{};
            else x[i] = in ? P::load(static_cast<const T*>(p.x) + r * p.x_stride + c * N) : P::zero();
        }
        const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r), sc = KEPT ? __ldg(p.scale + r) : 1.f;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[N], d[N];
            if constexpr (KEPT) unpack_piece<T, WIDE>(x[i], sc, f); else P::decode(x[i], f);
            P::decode(dy[i], d);                            // zero where there is no column
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const float n = (f[q] - mean) * rstd, g = d[q] * w[i * N + q];
                s[0] += g;
                s[1] = fmaf(g, n, s[1]);
                aw[i * N + q] = fmaf(d[q], n, aw[i * N + q]);
                ab[i * N + q] += d[q];
            }
        }
        if (!p.dx) continue;
        const float total = warp_sums<2>(s);                // lane 0: the first sum, lane 16: the second
        float m1 = 0.f, m2 = 0.f;
        if constexpr (!MULTI) {
            m1 = __shfl_sync(FULL_MASK, total, 0);
            m2 = __shfl_sync(FULL_MASK, total, 16);
        } else {
            float2* slot = part + parity * MAX_WARPS + group * warps;
            if ((lane & 15) == 0) reinterpret_cast<float*>(slot + gw)[lane >> 4] = total;
            group_sync(group, threads);
            for (int k = 0; k < warps; ++k) {
                const float2 v = slot[k];
                m1 += v.x;
                m2 += v.y;
            }
            parity ^= 1;                                    // the next row's exchange leaves these slots alone
        }
        m1 *= inv_d;
        m2 *= inv_d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            if (c >= pieces) break;
            float f[N], d[N], a[N];
            if constexpr (KEPT) unpack_piece<T, WIDE>(x[i], sc, f); else P::decode(x[i], f);
            P::decode(dy[i], d);
            if (p.add) P::decode(P::load(static_cast<const T*>(p.add) + r * p.D + c * N), a);
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const float n = (f[q] - mean) * rstd;
                f[q] = rstd * (d[q] * w[i * N + q] - m1 - n * m2);
                if (p.add) f[q] += a[q];
            }
            P::store(static_cast<T*>(p.dx) + r * p.D + c * N, P::encode(f));
        }
    }
    if (!p.dw && !p.db) return;
    grid_release();
    // the block's groups add up in order, then the block writes its partial row
    const int wide = threads * E;
    for (int g = 0; g + 1 < groups; ++g) {
        if (group == g) {
#pragma unroll
            for (int q = 0; q < E; ++q) {
                const int at = q * threads + gt;
                columns[at] = aw[q];
                columns[wide + at] = ab[q];
            }
        }
        __syncthreads();
        if (group == g + 1) {
#pragma unroll
            for (int q = 0; q < E; ++q) {
                const int at = q * threads + gt;
                aw[q] += columns[at];
                ab[q] += columns[wide + at];
            }
        }
        __syncthreads();
    }
    if (group == groups - 1) {
        float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (gt + static_cast<int64_t>(i) * threads) * N;
            if (c >= p.D) break;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                out[c + q] = aw[i * N + q];
                out[p.D + c + q] = ab[i * N + q];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Many or wide rows of whole 16-byte pieces.  A group of warps owns a row, 16 columns per thread, the same columns in every row,
// so parameters and column sums stay in registers.  Every thread copies its own pieces of the group's next rows into
// shared memory (cp.async) while it works on the current one; nobody else reads them, so the ring needs no barrier and
// no registers, and what is left in a row's chain is one exchange between the group's warps.
// With the loads covered the instruction count decides: values are decoded once, kept as fp32 pairs across the exchange
// and go through the packed fp32 instructions, two columns each.  The forward pass takes two rows at a time of the 16-bit
// types, whose exchanges cover one another; the backward pass has no registers for two.  One block per SM, whose registers and
// shared memory it takes.  16384 x 2048 bf16: forward 25.4 us (5.3 TB/s), dx 34.3 us (5.9 TB/s), all gradients 38.9 us;
// 4096 x 8192: 26.8, 37.3 and 45.2 us.
// W > 0: the row is exactly W full warps (512 W columns), which turns the addresses of a thread's pieces and the exchange
// into constants; W == 0 takes any other width.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float2 splat(float a) { return make_float2(a, a); }
// 1/sqrt(v): the hardware estimate and one Newton step (relative error below 2^-23); 0, infinite and NaN pass through
__device__ __forceinline__ float inverse_sqrt(float v) {
    const float r = rsqrtf(v);
    return (v > 0.f && v < __uint_as_float(F32_INF_BITS)) ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

template <typename T, int NV, int N>
__device__ __forceinline__ void load_param_pairs(const void* p, bool f32, const bool (&in)[NV], int gt, int threads, float absent,
                                                 float2 (&out)[NV][N / 2]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[N];
#pragma unroll
        for (int q = 0; q < N; ++q) f[q] = absent;
        if (p && in[i]) load_param_piece<T, N>(p, f32, (gt + i * threads) * N, f);
#pragma unroll
        for (int h = 0; h < N / 2; ++h) out[i][h] = make_float2(f[2 * h], f[2 * h + 1]);
    }
}

// Exchange of a group that takes two rows at a time: every warp leaves its part of both rows in 32 slots, and after the
// group's barrier lane 16 u + k of every warp picks up warp k's part of row u, so a few shuffles over half a warp replace
// 2 x warps reads by every thread.
template <int K>
__device__ __forceinline__ void half_warp_sums(float (&v)[K]) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] += __shfl_xor_sync(FULL_MASK, v[i], o);
}

template <typename T, int W, int U, bool PACK, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 1) norm_ring_kernel(const NormParams p, int row_warps) {
    using P = Piece<T, true>;
    constexpr int N = P::N, NV = RING_COLUMNS / N, H = N / 2;
    constexpr int ROW = NV * RING_THREADS * 16, STAGE = U * ROW;      // bytes: [row][piece][thread]
    extern __shared__ __align__(16) unsigned char ring_smem[];
    __shared__ float2 part[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];      // center and squares; U == 2: [parity][group][row][warp]
    __shared__ float part_sum[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];
    __shared__ uint32_t part_top[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];
    __shared__ float held[MAX_WARPS];                       // columns of each of the group's warps
    const int warps = W ? W : row_warps;
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    bool in[NV];
    int mine = 0;
    {
        const int pieces = static_cast<int>(p.D / N);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            in[i] = W || gt + i * threads < pieces;
            mine += min(max(pieces - (i * threads + gw * 32), 0), 32) * N;
        }
    }
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int rows = first < p.rows ? static_cast<int>((p.rows - first + step - 1) / step) : 0;      // of this group
    int to_fetch = rows;
    const T* src = static_cast<const T*>(p.x) + first * p.x_stride + gt * N;      // this thread's pieces of the row fetched next
    const int64_t src_step = step * p.x_stride;
    const uint32_t slot0 = smem_u32(ring_smem) + threadIdx.x * 16, slot_end = slot0 + STAGES * STAGE;
    uint32_t slot = slot0, fetch_slot = slot0;
    auto fetch = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (to_fetch > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (in[i]) copy_async<16>(fetch_slot + u * ROW + i * RING_THREADS * 16, src + i * threads * N);
            }
            src += src_step;
            --to_fetch;
        }
        fetch_slot += STAGE;
        if (fetch_slot == slot_end) fetch_slot = slot0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int k = 0; k < STAGES - 1; ++k) fetch();
    float2 w[NV][H], b[NV][H];                              // loaded while the first rows are on their way
    load_param_pairs<T, NV, N>(p.w, p.param_f32, in, gt, threads, 1.f, w);
    load_param_pairs<T, NV, N>(p.b, p.param_f32, in, gt, threads, 0.f, b);
    if (group == 0 && lane == 0) held[gw] = static_cast<float>(mine);
    __syncthreads();
    const float inv_mine = mine > 0 ? 1.f / static_cast<float>(mine) : 0.f, inv_d = 1.f / static_cast<float>(p.D);
    T* dst = static_cast<T*>(p.y) + first * p.D + gt * N;
    uint8_t* dst8 = p.payload + first * p.D + gt * N;
    const int64_t dst_step = step * p.D;
    int64_t r = first;
    // this row's slots; the next row's leave them alone
    int exchange = U == 2 ? group * 32 : group * warps, other = U == 2 ? 8 * 32 : MAX_WARPS;
    for (; rows > 0; rows -= U) {
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        typename P::Raw raw[U][NV];
        float2 x[U][NV][H];
        float mean[U], m2[U], dev[U];                       // first the warp's center, squares and sum of the deviations from it
        uint32_t top[U];
        bool odd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float2 s2 = splat(0.f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                raw[u][i] = in[i] && u < rows ? shared_at<uint4>(slot + u * ROW + i * RING_THREADS * 16) : P::zero();
                float f[N];
                P::decode(raw[u][i], f);
#pragma unroll
                for (int h = 0; h < H; ++h) { x[u][i][h] = make_float2(f[2 * h], f[2 * h + 1]); s2 = __fadd2_rn(s2, x[u][i][h]); }
            }
            mean[u] = s2.x + s2.y;
            odd[u] = false;
            top[u] = 0u;
            if (PACK) top[u] = warp_top<T, true, NV>(raw[u], odd[u]);
        }
        slot += STAGE;
        if (slot == slot_end) slot = slot0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float sum = warp_sum(mean[u]);
            mean[u] = sum * inv_mine;
            dev[u] = U == 2 && !W ? fmaf(-static_cast<float>(mine), mean[u], sum) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float2 neg = splat(-mean[u]);
            float2 s1 = splat(0.f), s2 = splat(0.f);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i]) {
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const float2 d = __fadd2_rn(x[u][i][h], neg);
                        if (U == 1) s1 = __fadd2_rn(s1, d);
                        s2 = __ffma2_rn(d, d, s2);
                    }
                }
            m2[u] = s2.x + s2.y;
            if (U == 1) dev[u] = s1.x + s1.y;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            m2[u] = warp_sum(m2[u]);
            if (U == 1) dev[u] = warp_sum(dev[u]);
        }
        if (warps == 1) {
#pragma unroll
            for (int u = 0; u < U; ++u) finish_stats(mean[u], dev[u], m2[u], inv_d, mean[u], m2[u]);
        } else if constexpr (U == 2) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (lane == 0) {
                    part[exchange + u * 16 + gw] = make_float2(mean[u], m2[u]);
                    if (!W) part_sum[exchange + u * 16 + gw] = dev[u];
                    if (PACK) part_top[exchange + u * 16 + gw] = top[u];
                }
            }
            group_sync(group, threads);
            const bool has = (lane & 15) < warps;
            const float c0 = part[exchange + (lane & 16)].x;
            float both[2] = {0.f, 0.f}, row_mean, row_m2;
            if (has) {
                const float2 v = part[exchange + lane];
                add_part(c0, v.x, v.y, W ? 0.f : part_sum[exchange + lane], (W ? 32.f * RING_COLUMNS : held[lane & 15]), both[0], both[1]);
            }
            half_warp_sums<2>(both);
            finish_stats(c0, both[0], both[1], inv_d, row_mean, row_m2);
            uint32_t t = PACK && has ? part_top[exchange + lane] : 0u;
            if (PACK) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(FULL_MASK, t, o));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                mean[u] = __shfl_sync(FULL_MASK, row_mean, u * 16);
                m2[u] = __shfl_sync(FULL_MASK, row_m2, u * 16);
                if (PACK) top[u] = __shfl_sync(FULL_MASK, t, u * 16);
            }
            exchange += other;
            other = -other;
        } else {
            if (lane == 0) {
                part[exchange + gw] = make_float2(mean[0], m2[0]);
                part_sum[exchange + gw] = dev[0];
                if (PACK) part_top[exchange + gw] = top[0];
            }
            group_sync(group, threads);
            const float c0 = part[exchange].x;
            float t = 0.f, q = 0.f;
#pragma unroll
            for (int k = 0; k < (W ? W : warps); ++k) {
                const float2 v = part[exchange + k];
                add_part(c0, v.x, v.y, part_sum[exchange + k], W ? 32.f * RING_COLUMNS : held[k], t, q);
                if (PACK) top[0] = max(top[0], part_top[exchange + k]);
            }
            finish_stats(c0, t, q, inv_d, mean[0], m2[0]);
            exchange += other;
            other = -other;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= rows) break;
            const float rstd = inverse_sqrt(m2[u] * inv_d + p.eps);
            const float2 r2 = splat(rstd), minus = splat(-mean[u]);
            const int e = PACK ? e4m3_scale_exponent(top[u]) : 0;
            const float inv = exp2_int(-e);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i]) {
                    float f[N];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const float2 v = __ffma2_rn(__fmul2_rn(__fadd2_rn(x[u][i][h], minus), r2), w[i][h], b[i][h]);
                        f[2 * h] = v.x;
                        f[2 * h + 1] = v.y;
                    }
                    P::store(dst + i * threads * N, P::encode(f));
                    if constexpr (PACK)
                        *reinterpret_cast<typename P::Packed*>(dst8 + i * threads * N) = pack_pairs<T>(x[u][i], raw[u][i], inv, odd[u]);
                }
            dst += dst_step;
            if (PACK) dst8 += dst_step;
            if (gt == 0) {
                if (p.mean) p.mean[r] = mean[u];
                if (p.rstd) p.rstd[r] = rstd;
                if (PACK) p.scale[r] = exp2_int(e);
            }
            r += step;
        }
    }
}

template <typename T, int W, bool KEPT, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 1) norm_grad_ring_kernel(const NormGradParams p, int row_warps) {
    using P = Piece<T, true>;
    using X = typename std::conditional<KEPT, typename P::Packed, uint4>::type;
    constexpr int N = P::N, NV = RING_COLUMNS / N, H = N / 2, XB = static_cast<int>(sizeof(X));
    // bytes of a stage: dy [piece][thread], x [piece][thread], {mean, 1/deviation, scale, -} [warp]
    constexpr int X_AT = NV * RING_THREADS * 16, STAT_AT = X_AT + NV * RING_THREADS * XB, STAGE = STAT_AT + (RING_THREADS / 32) * 16;
    extern __shared__ __align__(16) unsigned char ring_smem[];
    __shared__ float2 part[2 * MAX_WARPS];
    const int warps = W ? W : row_warps;
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    bool in[NV];
    {
        const int pieces = static_cast<int>(p.D / N);
#pragma unroll
        for (int i = 0; i < NV; ++i) in[i] = W || gt + i * threads < pieces;
    }
    const float inv_d = 1.f / static_cast<float>(p.D);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int rows = first < p.rows ? static_cast<int>((p.rows - first + step - 1) / step) : 0;      // of this group
    int to_fetch = rows;
    const T* src_dy = static_cast<const T*>(p.dy) + first * p.dy_stride + gt * N;
    const T* src_x = static_cast<const T*>(p.x) + first * p.x_stride + gt * N;
    const uint8_t* src_8 = p.payload + first * p.D + gt * N;
    // lanes 0, 1 and (KEPT) 2 of every warp bring the row's mean, 1/deviation and scale into the warp's own slots
    const float* src_stat = (lane == 0 ? p.mean : lane == 1 ? p.rstd : p.scale) + first;
    const bool brings = lane < (KEPT ? 3 : 2);
    const int64_t dy_step = step * p.dy_stride, x_step = step * (KEPT ? p.D : p.x_stride);
    const uint32_t base = smem_u32(ring_smem);
    const int dy_at = threadIdx.x * 16, x_at = X_AT + threadIdx.x * XB, stat_at = STAT_AT + (threadIdx.x >> 5) * 16;
    uint32_t slot = base, fetch_slot = base;
    auto fetch = [&]() {
        if (to_fetch > 0) {
            if (brings) copy_async<4>(fetch_slot + stat_at + lane * 4, src_stat);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i]) {
                    copy_async<16>(fetch_slot + dy_at + i * RING_THREADS * 16, src_dy + i * threads * N);
                    if constexpr (KEPT) copy_async<XB>(fetch_slot + x_at + i * RING_THREADS * XB, src_8 + i * threads * N);
                    else copy_async<16>(fetch_slot + x_at + i * RING_THREADS * XB, src_x + i * threads * N);
                }
        }
        src_dy += dy_step;
        if constexpr (KEPT) src_8 += x_step; else src_x += x_step;
        src_stat += step;
        --to_fetch;
        fetch_slot += STAGE;
        if (fetch_slot == base + STAGES * STAGE) fetch_slot = base;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int k = 0; k < STAGES - 1; ++k) fetch();
    float2 w[NV][H], aw[NV][H], ab[NV][H];                  // w loaded while the first rows are on their way
    load_param_pairs<T, NV, N>(p.w, p.param_f32, in, gt, threads, 1.f, w);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) aw[i][h] = ab[i][h] = splat(0.f);
    T* dst = static_cast<T*>(p.dx) + first * p.D + gt * N;
    const T* add = static_cast<const T*>(p.add) + first * p.D + gt * N;
    const int64_t dst_step = step * p.D;
    int exchange = group * warps, other = MAX_WARPS;        // this row's slots; the next row's leave them alone
    for (; rows > 0; --rows) {
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();                                       // the row's statistics came by other lanes
        float mean, rstd, sc;
        {
            const uint4 v = shared_at<uint4>(slot + stat_at);
            mean = __uint_as_float(v.x);
            rstd = __uint_as_float(v.y);
            sc = __uint_as_float(v.z);
        }
        // kept in 8 bits: the scale, a power of two, goes into the factor, unless the row's values may need the clamp
        const bool clamp = KEPT && may_clamp<T>(sc);
        const float2 r2 = splat(rstd), rx = splat(KEPT && !clamp ? rstd * sc : rstd), c2 = splat(-mean * rstd);
        float2 n[NV][H], g[NV][H], s1 = splat(0.f), s2 = splat(0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const X xr = in[i] ? shared_at<X>(slot + x_at + i * RING_THREADS * XB) : X{};
            const uint4 dr = in[i] ? shared_at<uint4>(slot + dy_at + i * RING_THREADS * 16) : P::zero();
            float f[N], d[N];
            if constexpr (KEPT) {
                P::decode_packed(xr, f);
                if (clamp) {
#pragma unroll
                    for (int q = 0; q < N; ++q) f[q] = unpacked<T>(f[q], sc);
                }
            } else {
                P::decode(xr, f);
            }
            P::decode(dr, d);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const float2 dv = make_float2(d[2 * h], d[2 * h + 1]);
                n[i][h] = __ffma2_rn(make_float2(f[2 * h], f[2 * h + 1]), rx, c2);
                g[i][h] = __fmul2_rn(dv, w[i][h]);
                s1 = __fadd2_rn(s1, g[i][h]);
                s2 = __ffma2_rn(g[i][h], n[i][h], s2);
                aw[i][h] = __ffma2_rn(dv, n[i][h], aw[i][h]);
                ab[i][h] = __fadd2_rn(ab[i][h], dv);
            }
        }
        slot += STAGE;
        if (slot == base + STAGES * STAGE) slot = base;
        if (p.dx) {
            float s[2] = {s1.x + s1.y, s2.x + s2.y};
            const float total = warp_sums<2>(s);            // lane 0: the first sum, lane 16: the second
            float m1 = 0.f, m2 = 0.f;
            if (warps == 1) {
                m1 = __shfl_sync(FULL_MASK, total, 0);
                m2 = __shfl_sync(FULL_MASK, total, 16);
            } else {
                if ((lane & 15) == 0) reinterpret_cast<float*>(part + exchange + gw)[lane >> 4] = total;
                group_sync(group, threads);
                if (W == 16 || (W == 0 && warps >= 8)) {    // a warp's part per lane, joined by shuffles
                    const float2 v = (lane & 15) < warps ? part[exchange + (lane & 15)] : splat(0.f);
                    float both[2] = {v.x, v.y};
                    half_warp_sums<2>(both);
                    m1 = both[0];
                    m2 = both[1];
                } else {
#pragma unroll
                    for (int k = 0; k < (W ? W : warps); ++k) {
                        const float2 v = part[exchange + k];
                        m1 += v.x;
                        m2 += v.y;
                    }
                }
                exchange += other;
                other = -other;
            }
            const float scaled = -inv_d * rstd;
            const float2 m1p = splat(m1 * scaled), m2p = splat(m2 * scaled);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i]) {
                    float f[N];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const float2 v = __ffma2_rn(g[i][h], r2, __ffma2_rn(n[i][h], m2p, m1p));
                        f[2 * h] = v.x;
                        f[2 * h + 1] = v.y;
                    }
                    if (p.add) {
                        float o[N];
                        P::decode(P::load(add + i * threads * N), o);
#pragma unroll
                        for (int q = 0; q < N; ++q) f[q] += o[q];
                    }
                    P::store(dst + i * threads * N, P::encode(f));
                }
            dst += dst_step;
            add += dst_step;
        }
        __syncwarp();                                       // before a fetch overwrites a slot another lane may still read
    }
    if (!p.dw && !p.db) return;
    grid_release();
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                        // the ring is free: the groups add up in order through it
    float2* columns = reinterpret_cast<float2*>(ring_smem);      // [2 * NV * H][threads]
    for (int q = 0; q + 1 < groups; ++q) {
        if (group == q) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    columns[(i * H + h) * threads + gt] = aw[i][h];
                    columns[((NV + i) * H + h) * threads + gt] = ab[i][h];
                }
        }
        __syncthreads();
        if (group == q + 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    aw[i][h] = __fadd2_rn(aw[i][h], columns[(i * H + h) * threads + gt]);
                    ab[i][h] = __fadd2_rn(ab[i][h], columns[((NV + i) * H + h) * threads + gt]);
                }
        }
        __syncthreads();
    }
    if (group == groups - 1) {
        float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in[i]) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const int c = (gt + i * threads) * N + 2 * h;
                    *reinterpret_cast<float2*>(out + c) = aw[i][h];
                    *reinterpret_cast<float2*>(out + p.D + c) = ab[i][h];
                }
            }
    }
}

// ---------------------------------------------------------------------------
// The same for rows that are not whole 16-byte pieces at 16-byte addresses (an odd width, an odd stride, a view that
// begins anywhere), brought and stored as the granules that cover them (row_shift.cuh).  A granule is another thread's,
// so a row has a barrier behind its arrival and one before its results leave.  16384 x 2001 bf16: forward 47 us, all
// gradients 64 us, against 172 and 187 us one value at a time.
// ---------------------------------------------------------------------------
// parameters of this thread's columns, `absent` beyond the row's end
template <typename T, int NV, int N>
__device__ __forceinline__ void load_param_values(const void* p, bool f32, int D, int gt, int threads, float absent, float2 (&out)[NV][N / 2]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int c = (gt + i * threads) * N + q;
            f[q] = p && c < D ? param_at<T>(p, f32, c) : absent;
        }
#pragma unroll
        for (int h = 0; h < N / 2; ++h) out[i][h] = make_float2(f[2 * h], f[2 * h + 1]);
    }
}

template <typename T, int U, bool PACK, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 1) norm_shift_kernel(const NormParams p, int warps) {
    using P = Piece<T, true>;
    constexpr int N = P::N, NV = RING_COLUMNS / N, H = N / 2, XB = static_cast<int>(sizeof(typename P::Packed));
    extern __shared__ __align__(16) unsigned char ring_smem[];
    __shared__ float2 part[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];      // center and squares; U == 2: [parity][group][row][warp]
    __shared__ float part_sum[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];
    __shared__ uint32_t part_top[U == 2 ? 2 * 8 * 32 : 2 * MAX_WARPS];
    __shared__ float held[MAX_WARPS];                       // columns of each of the group's warps
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads, D = static_cast<int>(p.D), bytes = D * static_cast<int>(sizeof(T));
    // a group's memory: STAGES times U rows of x, then U times {16 bytes, a row of y}, U times {16 bytes, a row of payload}
    const int room = row_room(threads * RING_COLUMNS, sizeof(T)), room8 = row_room(threads * RING_COLUMNS, 1);
    const uint32_t slot0 = smem_u32(ring_smem) + group * U * ((STAGES + 1) * room + room8 + 32), slot_end = slot0 + STAGES * U * room;
    const uint32_t out = slot_end + 16, out8 = slot_end + U * (room + 16) + 16;
    auto sync = [&]() { if (warps > 1) group_sync(group, threads); else __syncwarp(); };
    int valid[NV], mine = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        valid[i] = min(max(D - (gt + i * threads) * N, 0), N);
        mine += min(max(D - (i * threads + gw * 32) * N, 0), 32 * N);
    }
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int rows = first < p.rows ? static_cast<int>((p.rows - first + step - 1) / step) : 0;      // of this group
    int to_fetch = rows;
    const T* src = static_cast<const T*>(p.x) + first * p.x_stride;
    const T* cur = src;
    const int64_t src_step = step * p.x_stride;
    uint32_t slot = slot0, fetch_slot = slot0;
    auto fetch = [&](auto head) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (to_fetch > 0) fetch_row<decltype(head)::value>(fetch_slot, src, bytes, gt, threads, p.x);
            src += src_step;
            --to_fetch;
            fetch_slot += room;
        }
        if (fetch_slot == slot_end) fetch_slot = slot0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(std::true_type());
    for (int k = 1; k < STAGES - 1; ++k) fetch(std::false_type());
    float2 w[NV][H], b[NV][H];
    load_param_values<T, NV, N>(p.w, p.param_f32, D, gt, threads, 1.f, w);
    load_param_values<T, NV, N>(p.b, p.param_f32, D, gt, threads, 0.f, b);
    if (group == 0 && lane == 0) held[gw] = static_cast<float>(mine);
    __syncthreads();
    const float inv_mine = mine > 0 ? 1.f / static_cast<float>(mine) : 0.f, inv_d = 1.f / static_cast<float>(D);
    int64_t r = first;
    // this row's slots; the next row's leave them alone
    int exchange = U == 2 ? group * 32 : group * warps, other = U == 2 ? 8 * 32 : MAX_WARPS;
    for (; rows > 0; rows -= U) {
        fetch(std::false_type());
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        sync();                                             // the other threads' granules
        typename P::Raw raw[U][NV];
        float2 x[U][NV][H];
        float mean[U], m2[U], dev[U];                       // first the warp's center, squares and sum of the deviations from it
        uint32_t top[U];
        bool odd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t shift = offset16(cur);
            cur += src_step;
            float2 s2 = splat(0.f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                raw[u][i] = valid[i] && u < rows ? shared_shifted(slot + (gt + i * threads) * 16, shift) : P::zero();      // zeros behind the row
                float f[N];
                P::decode(raw[u][i], f);
#pragma unroll
                for (int h = 0; h < H; ++h) { x[u][i][h] = make_float2(f[2 * h], f[2 * h + 1]); s2 = __fadd2_rn(s2, x[u][i][h]); }
            }
            slot += room;
            mean[u] = s2.x + s2.y;
            odd[u] = false;
            top[u] = 0u;
            if (PACK) top[u] = warp_top<T, true, NV>(raw[u], odd[u]);
        }
        if (slot == slot_end) slot = slot0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float sum = warp_sum(mean[u]);
            mean[u] = sum * inv_mine;
            dev[u] = U == 2 ? fmaf(-static_cast<float>(mine), mean[u], sum) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float2 neg = splat(-mean[u]);
            float2 s1 = splat(0.f), s2 = splat(0.f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    float2 d = __fadd2_rn(x[u][i][h], neg);
                    if (valid[i] < N) {                     // the row's last piece, and those behind it
                        if (2 * h >= valid[i]) d.x = 0.f;
                        if (2 * h + 1 >= valid[i]) d.y = 0.f;
                    }
                    if (U == 1) s1 = __fadd2_rn(s1, d);
                    s2 = __ffma2_rn(d, d, s2);
                }
            }
            m2[u] = s2.x + s2.y;
            if (U == 1) dev[u] = s1.x + s1.y;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            m2[u] = warp_sum(m2[u]);
            if (U == 1) dev[u] = warp_sum(dev[u]);
        }
        if (warps == 1) {
#pragma unroll
            for (int u = 0; u < U; ++u) finish_stats(mean[u], dev[u], m2[u], inv_d, mean[u], m2[u]);
        } else if constexpr (U == 2) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (lane == 0) {
                    part[exchange + u * 16 + gw] = make_float2(mean[u], m2[u]);
                    part_sum[exchange + u * 16 + gw] = dev[u];
                    if (PACK) part_top[exchange + u * 16 + gw] = top[u];
                }
            }
            group_sync(group, threads);
            const bool has = (lane & 15) < warps;
            const float c0 = part[exchange + (lane & 16)].x;
            float both[2] = {0.f, 0.f}, row_mean, row_m2;
            if (has) {
                const float2 v = part[exchange + lane];
                add_part(c0, v.x, v.y, part_sum[exchange + lane], held[lane & 15], both[0], both[1]);
            }
            half_warp_sums<2>(both);
            finish_stats(c0, both[0], both[1], inv_d, row_mean, row_m2);
            uint32_t t = PACK && has ? part_top[exchange + lane] : 0u;
            if (PACK) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(FULL_MASK, t, o));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                mean[u] = __shfl_sync(FULL_MASK, row_mean, u * 16);
                m2[u] = __shfl_sync(FULL_MASK, row_m2, u * 16);
                if (PACK) top[u] = __shfl_sync(FULL_MASK, t, u * 16);
            }
            exchange += other;
            other = -other;
        } else {
            if (lane == 0) {
                part[exchange + gw] = make_float2(mean[0], m2[0]);
                part_sum[exchange + gw] = dev[0];
                if (PACK) part_top[exchange + gw] = top[0];
            }
            group_sync(group, threads);
            const float c0 = part[exchange].x;
            float t = 0.f, q = 0.f;
            for (int k = 0; k < warps; ++k) {
                const float2 v = part[exchange + k];
                add_part(c0, v.x, v.y, part_sum[exchange + k], held[k], t, q);
                if (PACK) top[0] = max(top[0], part_top[exchange + k]);
            }
            finish_stats(c0, t, q, inv_d, mean[0], m2[0]);
            exchange += other;
            other = -other;
        }
        float rstd[U];
        int e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            rstd[u] = inverse_sqrt(m2[u] * inv_d + p.eps);
            e[u] = PACK ? e4m3_scale_exponent(top[u]) : 0;
            const float2 r2 = splat(rstd[u]), minus = splat(-mean[u]);
            const float inv = exp2_int(-e[u]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (valid[i]) {
                    float f[N];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const float2 v = __ffma2_rn(__fmul2_rn(__fadd2_rn(x[u][i][h], minus), r2), w[i][h], b[i][h]);
                        f[2 * h] = v.x;
                        f[2 * h + 1] = v.y;
                    }
                    store_shared(out + u * (room + 16) + (gt + i * threads) * 16, P::encode(f));
                    if constexpr (PACK) store_shared(out8 + u * (room8 + 16) + (gt + i * threads) * XB, pack_pairs<T>(x[u][i], raw[u][i], inv, odd[u]));
                }
        }
        sync();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= rows) break;
            store_row<T>(static_cast<T*>(p.y) + r * p.D, out + u * (room + 16), bytes, gt, threads);
            if (PACK) store_row<uint8_t>(p.payload + r * p.D, out8 + u * (room8 + 16), D, gt, threads);
            if (gt == 0) {
                if (p.mean) p.mean[r] = mean[u];
                if (p.rstd) p.rstd[r] = rstd[u];
                if (PACK) p.scale[r] = exp2_int(e[u]);
            }
            r += step;
        }
    }
}

template <typename T, bool KEPT, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, 1) norm_grad_shift_kernel(const NormGradParams p, int warps) {
    using P = Piece<T, true>;
    using X = typename std::conditional<KEPT, typename P::Packed, uint4>::type;
    constexpr int N = P::N, NV = RING_COLUMNS / N, H = N / 2, XB = static_cast<int>(sizeof(X));
    extern __shared__ __align__(16) unsigned char ring_smem[];
    __shared__ float2 part[2 * MAX_WARPS];
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = threadIdx.x / threads, gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads, D = static_cast<int>(p.D), bytes = D * static_cast<int>(sizeof(T));
    const int x_bytes = KEPT ? D : bytes;
    // a group's memory: STAGES of {dy, x or payload, {mean, 1/deviation, scale, -}}, 16 bytes, a row of dx
    const int room = row_room(threads * RING_COLUMNS, sizeof(T)), room_x = row_room(threads * RING_COLUMNS, KEPT ? 1 : sizeof(T));
    const int stage = room + room_x + 16;
    const uint32_t slot0 = smem_u32(ring_smem) + group * (STAGES * stage + 16 + room), slot_end = slot0 + STAGES * stage;
    const uint32_t out = slot_end + 16;
    auto sync = [&]() { if (warps > 1) group_sync(group, threads); else __syncwarp(); };
    bool in[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) in[i] = (gt + i * threads) * N < D;
    const float inv_d = 1.f / static_cast<float>(D);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group, step = static_cast<int64_t>(gridDim.x) * groups;
    int rows = first < p.rows ? static_cast<int>((p.rows - first + step - 1) / step) : 0;      // of this group
    int to_fetch = rows;
    const T* src_dy = static_cast<const T*>(p.dy) + first * p.dy_stride;
    const char* src_x = KEPT ? reinterpret_cast<const char*>(p.payload) + first * p.D
                             : reinterpret_cast<const char*>(static_cast<const T*>(p.x) + first * p.x_stride);
    const float* src_stat = (gt == 0 ? p.mean : gt == 1 ? p.rstd : p.scale) + first;
    const bool brings = gt < (KEPT ? 3 : 2);
    const T* cur_dy = src_dy;
    const char* cur_x = src_x;
    const int64_t dy_step = step * p.dy_stride, x_step = step * (KEPT ? p.D : p.x_stride * static_cast<int64_t>(sizeof(T)));
    uint32_t slot = slot0, fetch_slot = slot0;
    auto fetch = [&](auto head) {
        if (to_fetch > 0) {
            if (brings) copy_async<4>(fetch_slot + room + room_x + gt * 4, src_stat);
            fetch_row<decltype(head)::value>(fetch_slot, src_dy, bytes, gt, threads, p.dy);
            fetch_row<decltype(head)::value>(fetch_slot + room, src_x, x_bytes, gt, threads, KEPT ? static_cast<const void*>(p.payload) : p.x);
        }
        src_dy += dy_step;
        src_x += x_step;
        src_stat += step;
        --to_fetch;
        fetch_slot += stage;
        if (fetch_slot == slot_end) fetch_slot = slot0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(std::true_type());
    for (int k = 1; k < STAGES - 1; ++k) fetch(std::false_type());
    float2 w[NV][H], aw[NV][H], ab[NV][H];
    load_param_values<T, NV, N>(p.w, p.param_f32, D, gt, threads, 1.f, w);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) aw[i][h] = ab[i][h] = splat(0.f);
    int64_t r = first;
    int exchange = group * warps, other = MAX_WARPS;        // this row's slots; the next row's leave them alone
    for (; rows > 0; --rows) {
        fetch(std::false_type());
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        sync();                                             // the other threads' granules
        const uint4 st = shared_at<uint4>(slot + room + room_x);
        const float mean = __uint_as_float(st.x), rstd = __uint_as_float(st.y), sc = KEPT ? __uint_as_float(st.z) : 1.f;
        const bool clamp = KEPT && may_clamp<T>(sc);
        const float2 r2 = splat(rstd), rx = splat(KEPT && !clamp ? rstd * sc : rstd), c2 = splat(-mean * rstd);
        const uint32_t dy_shift = offset16(cur_dy), x_shift = offset16(cur_x);
        cur_dy += dy_step;
        cur_x += x_step;
        float2 n[NV][H], g[NV][H], s1 = splat(0.f), s2 = splat(0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = gt + i * threads;
            float f[N], d[N];
            if constexpr (KEPT) {
                P::decode_packed(in[i] ? shared_unaligned<X>(slot + room + x_shift + c * XB) : X{}, f);
                if (clamp) {
#pragma unroll
                    for (int q = 0; q < N; ++q) f[q] = unpacked<T>(f[q], sc);
                }
            } else {
                P::decode(in[i] ? shared_shifted(slot + room + c * 16, x_shift) : X{}, f);
            }
            P::decode(in[i] ? shared_shifted(slot + c * 16, dy_shift) : P::zero(), d);      // zeros behind the row
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const float2 dv = make_float2(d[2 * h], d[2 * h + 1]);
                n[i][h] = __ffma2_rn(make_float2(f[2 * h], f[2 * h + 1]), rx, c2);
                g[i][h] = __fmul2_rn(dv, w[i][h]);
                s1 = __fadd2_rn(s1, g[i][h]);
                s2 = __ffma2_rn(g[i][h], n[i][h], s2);
                aw[i][h] = __ffma2_rn(dv, n[i][h], aw[i][h]);
                ab[i][h] = __fadd2_rn(ab[i][h], dv);
            }
        }
        slot += stage;
        if (slot == slot_end) slot = slot0;
        if (p.dx) {
            float s[2] = {s1.x + s1.y, s2.x + s2.y};
            const float total = warp_sums<2>(s);            // lane 0: the first sum, lane 16: the second
            float m1 = 0.f, m2 = 0.f;
            if (warps == 1) {
                m1 = __shfl_sync(FULL_MASK, total, 0);
                m2 = __shfl_sync(FULL_MASK, total, 16);
            } else {
                if ((lane & 15) == 0) reinterpret_cast<float*>(part + exchange + gw)[lane >> 4] = total;
                group_sync(group, threads);
                const float2 v = (lane & 15) < warps ? part[exchange + (lane & 15)] : splat(0.f);
                float both[2] = {v.x, v.y};                 // a warp's part per lane, joined by shuffles
                half_warp_sums<2>(both);
                m1 = both[0];
                m2 = both[1];
                exchange += other;
                other = -other;
            }
            const float scaled = -inv_d * rstd;
            const float2 m1p = splat(m1 * scaled), m2p = splat(m2 * scaled);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (in[i]) {
                    float f[N];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const float2 v = __ffma2_rn(g[i][h], r2, __ffma2_rn(n[i][h], m2p, m1p));
                        f[2 * h] = v.x;
                        f[2 * h + 1] = v.y;
                    }
                    store_shared(out + (gt + i * threads) * 16, P::encode(f));
                }
            sync();
            store_row<T>(static_cast<T*>(p.dx) + r * p.D, out, bytes, gt, threads);
        } else {
            sync();                                         // before a fetch overwrites what another thread still reads
        }
        r += step;
    }
    if (!p.dw && !p.db) return;
    grid_release();
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                        // the ring is free: the groups add up in order through it
    float2* columns = reinterpret_cast<float2*>(ring_smem);      // [2 * NV * H][threads]
    for (int q = 0; q + 1 < groups; ++q) {
        if (group == q) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    columns[(i * H + h) * threads + gt] = aw[i][h];
                    columns[((NV + i) * H + h) * threads + gt] = ab[i][h];
                }
        }
        __syncthreads();
        if (group == q + 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    aw[i][h] = __fadd2_rn(aw[i][h], columns[(i * H + h) * threads + gt]);
                    ab[i][h] = __fadd2_rn(ab[i][h], columns[((NV + i) * H + h) * threads + gt]);
                }
        }
        __syncthreads();
    }
    if (group == groups - 1) {
        float* sums = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int c = (gt + i * threads) * N + 2 * h;
                if (c < D) { sums[c] = aw[i][h].x; sums[p.D + c] = ab[i][h].x; }
                if (c + 1 < D) { sums[c + 1] = aw[i][h].y; sums[p.D + c + 1] = ab[i][h].y; }
            }
    }
}

// Backward of rows beyond 8,192 values, and of an empty batch (column sums of zero): dx by a block per row, which reads it
// twice, the second time from L1; the column sums by a pass of their own.  4096 x 12288 bf16: dx 84 us, all gradients
// 138 us (floor 46 us; 238 and 350 us value by value): no ring as below, whose 16 columns per thread end at 8,192.
template <typename T, bool WIDE, bool KEPT>
__device__ __forceinline__ void x_piece(const NormGradParams& p, int64_t r, int64_t c, float scale, float (&f)[Piece<T, WIDE>::N]) {
    using P = Piece<T, WIDE>;
    if constexpr (KEPT) unpack_piece<T, WIDE>(P::load_packed(p.payload + r * p.D + c), scale, f);
    else P::decode(P::load(static_cast<const T*>(p.x) + r * p.x_stride + c), f);
}

template <typename T, bool WIDE, bool KEPT>
__global__ void __launch_bounds__(256) norm_grad_rows_loop_kernel(const NormGradParams p) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N;
    __shared__ float buf[33];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* dyr = static_cast<const T*>(p.dy) + r * p.dy_stride;
        const float mean = p.mean[r], rstd = p.rstd[r], sc = KEPT ? p.scale[r] : 1.f;
        float s1 = 0.f, s2 = 0.f;
        auto piece = [&](int64_t c, float (&g)[N], float (&n)[N]) {      // g = dy w, n = (x - mean) rstd
            P::decode(P::load(dyr + c), g);
            x_piece<T, WIDE, KEPT>(p, r, c, sc, n);
            float w[N];
            if (p.w) {
                load_param_piece<T, N>(p.w, p.param_f32, c, w);
#pragma unroll
                for (int q = 0; q < N; ++q) g[q] *= w[q];
            }
#pragma unroll
            for (int q = 0; q < N; ++q) n[q] = (n[q] - mean) * rstd;
        };
#pragma unroll 4
        for (int64_t c = threadIdx.x * N; c < p.D; c += blockDim.x * N) {
            float g[N], n[N];
            piece(c, g, n);
#pragma unroll
            for (int q = 0; q < N; ++q) { s1 += g[q]; s2 = fmaf(g[q], n[q], s2); }
        }
        s1 = block_sum(s1, buf) / static_cast<float>(p.D);
        s2 = block_sum(s2, buf) / static_cast<float>(p.D);
#pragma unroll 2
        for (int64_t c = threadIdx.x * N; c < p.D; c += blockDim.x * N) {
            float g[N], n[N], a[N];
            piece(c, g, n);
            if (p.add) P::decode(P::load(static_cast<const T*>(p.add) + r * p.D + c), a);
#pragma unroll
            for (int q = 0; q < N; ++q) {
                g[q] = rstd * (g[q] - s1 - n[q] * s2);
                if (p.add) g[q] += a[q];
            }
            P::store(static_cast<T*>(p.dx) + r * p.D + c, P::encode(g));
        }
    }
}

// column sums of one split of the rows: 32 pieces of columns by 8 row lanes per block
template <typename T, bool WIDE, bool KEPT>
__global__ void __launch_bounds__(256) norm_grad_cols_loop_kernel(const NormGradParams p) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N;
    __shared__ float sums[8][2][N][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + tx) * N;
    const int64_t per = (p.rows + p.splits - 1) / p.splits;
    const int64_t r0 = per * blockIdx.y, r1 = r0 + per < p.rows ? r0 + per : p.rows;
    float aw[N], ab[N];
#pragma unroll
    for (int q = 0; q < N; ++q) aw[q] = ab[q] = 0.f;
    if (c < p.D) {
#pragma unroll 4
        for (int64_t r = r0 + ty; r < r1; r += 8) {
            const float mean = p.mean[r], rstd = p.rstd[r];
            float d[N], x[N];
            P::decode(P::load(static_cast<const T*>(p.dy) + r * p.dy_stride + c), d);
            x_piece<T, WIDE, KEPT>(p, r, c, KEPT ? p.scale[r] : 1.f, x);
#pragma unroll
            for (int q = 0; q < N; ++q) { aw[q] = fmaf(d[q], (x[q] - mean) * rstd, aw[q]); ab[q] += d[q]; }
        }
    }
#pragma unroll
    for (int q = 0; q < N; ++q) { sums[ty][0][q][tx] = aw[q]; sums[ty][1][q][tx] = ab[q]; }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N * 32; i += 256) {
        const int which = i / (N * 32), k = i % (N * 32);
        const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 * N + k;
        float t = 0.f;
#pragma unroll
        for (int y = 0; y < 8; ++y) t += sums[y][which][k % N][k / N];
        if (col < p.D) p.partial[(static_cast<int64_t>(blockIdx.y) * 2 + which) * p.D + col] = t;
    }
}

// `splits` partial rows to the gradients: 32 columns by 32 lanes of partials per block, so that a lane's few loads are
// all in flight at once
constexpr int JOIN_LANES = 32;
template <typename T>
__global__ void __launch_bounds__(32 * JOIN_LANES) norm_grad_join_kernel(const NormGradParams p) {
    __shared__ float sw[JOIN_LANES][33], sb[JOIN_LANES][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
    float aw = 0.f, ab = 0.f;
    grid_wait();
    if (c < p.D) {
#pragma unroll
        for (int k = 0; k < (GRID_SMS + JOIN_LANES - 1) / JOIN_LANES; ++k) {
            const int i = ty + k * JOIN_LANES;
            if (i < p.splits) {
                aw += p.partial[static_cast<int64_t>(i) * 2 * p.D + c];
                ab += p.partial[(static_cast<int64_t>(i) * 2 + 1) * p.D + c];
            }
        }
    }
    sw[ty][tx] = aw;
    sb[ty][tx] = ab;
    __syncthreads();
    // warp ty finishes column ty: lane tx holds the partial sum of lane row tx
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + ty;
    aw = warp_sum(sw[tx][ty]);
    ab = warp_sum(sb[tx][ty]);
    if (tx != 0 || col >= p.D) return;
    if (p.dw) { if (p.param_f32) static_cast<float*>(p.dw)[col] = aw; else static_cast<T*>(p.dw)[col] = from_f32<T>(aw); }
    if (p.db) { if (p.param_f32) static_cast<float*>(p.db)[col] = ab; else static_cast<T*>(p.db)[col] = from_f32<T>(ab); }
}

constexpr int MAX_SPLITS = GRID_SMS;       // one block per SM: rows of partial column sums

int splits_for(int64_t rows) {
    const int64_t s = (rows + 63) / 64;
    return static_cast<int>(s < 1 ? 1 : (s > MAX_SPLITS ? MAX_SPLITS : s));
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>(rows < 148 * 64 ? rows : 148 * 64); }

// Ring kernels take many rows, many values, or rows so wide that the others' exchange between sixteen warps costs more than
// the start of a ring.  Measured, rings / others: forward 1000 x 1024 bf16 5.2 / 6.1 us, 512 x 1024 4.7 / 4.2, 128 x 8192
// 5.2 / 10.3, 64 x 8191 7.9 / 18.6; all gradients 256 x 2048 bf16 8.3 / 10.3 us, 256 x 1024 fp32 8.3 / 6.7, 64 x 8192 12.4 / 16.5.
constexpr int64_t RING_ROWS = 1024, RING_DIM = 4096;
constexpr int64_t RING_VALUES = 1000000, RING_GRAD_VALUES = 1 << 19;
bool ring_pays(int64_t rows, int64_t D, int64_t values) { return rows >= RING_ROWS || rows * D >= values || D > RING_DIM; }

// Rows at any address: a warp's 512 columns are too many for narrower ones (32768 x 129 bf16: 23 us forward, 21 us one
// value at a time; 16384 x 2001: 47 and 172); the backward pass needs more rows (1500 x 1001 bf16: 13.4 us, 12.4 one value at a
// time; 1500 x 4099: 29 and 33; 512 x 8191: 27 and 21; 5003 x 1537 fp16: 27 and 41)
constexpr int64_t SHIFT_DIM = 256, SHIFT_GRAD_ROWS = 2048, SHIFT_GRAD_DIM = 2000;
bool shift_grad_pays(int64_t rows, int64_t D) {
    return D > SHIFT_DIM && (rows >= SHIFT_GRAD_ROWS || (rows >= RING_ROWS && D >= SHIFT_GRAD_DIM));
}

// the width a ring kernel is built for: W full warps when the row is exactly that, else 0
inline int ring_width(int64_t D) {
    for (int w = 1; w <= MAX_WARPS; w *= 2)
        if (D == static_cast<int64_t>(w) * 32 * RING_COLUMNS) return w;
    return 0;
}

template <typename T, int W, bool PACK>
cudaError_t norm_ring_width(const NormParams& p, cudaStream_t s) {
    // rows a group takes at a time: two cover one another's exchange (16384 x 2048 bf16 24.7 us instead of 30.8, x 1536 22.6
    // instead of 29.2, 4096 x 8192 26.6 instead of 39); fp32 rows are bound by memory with one
    constexpr int U = sizeof(T) == 4 ? 1 : 2, ROWS = sizeof(T) == 4 ? 4 : 6;      // rows in the ring: 128 KB, 96 KB
    constexpr int SMEM = ROWS * RING_THREADS * RING_COLUMNS * static_cast<int>(sizeof(T));
    const int warps = ring_warps(p.D), groups = MAX_WARPS / warps;
    auto* kernel = norm_ring_kernel<T, W, U, PACK, ROWS / U>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    const int64_t need = (p.rows + groups - 1) / groups;
    kernel<<<static_cast<unsigned>(need < GRID_SMS ? need : GRID_SMS), groups * warps * 32, SMEM, s>>>(p, warps);
    return cudaGetLastError();
}
template <typename T, bool PACK>
cudaError_t norm_ring_launch(const NormParams& p, cudaStream_t s) {
    switch (ring_width(p.D)) {
        case 1: return norm_ring_width<T, 1, PACK>(p, s);
        case 2: return norm_ring_width<T, 2, PACK>(p, s);
        case 4: return norm_ring_width<T, 4, PACK>(p, s);
        case 8: return norm_ring_width<T, 8, PACK>(p, s);
        case 16: return norm_ring_width<T, 16, PACK>(p, s);
        default: return norm_ring_width<T, 0, PACK>(p, s);
    }
}

template <typename T, bool PACK>
cudaError_t norm_shift_launch(const NormParams& p, cudaStream_t s) {
    constexpr int U = sizeof(T) == 4 ? 1 : 2, STAGES = sizeof(T) == 4 ? 3 : 2;      // with the results' rows at most 150 KB
    auto* kernel = norm_shift_kernel<T, U, PACK, STAGES>;
    const int warps = ring_warps(p.D), groups = MAX_WARPS / warps, columns = warps * 32 * RING_COLUMNS;
    const int smem = groups * U * ((STAGES + 1) * row_room(columns, sizeof(T)) + row_room(columns, 1) + 32);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int64_t need = (p.rows + groups - 1) / groups;
    kernel<<<static_cast<unsigned>(need < GRID_SMS ? need : GRID_SMS), groups * warps * 32, smem, s>>>(p, warps);
    return cudaGetLastError();
}

template <typename T, bool WIDE, int NV, bool PACK>
cudaError_t norm_launch(const NormParams& p, const RowShape& h, cudaStream_t s) {
    const int64_t need = (p.rows + h.groups - 1) / h.groups;
    const unsigned grid = static_cast<unsigned>(need < GRID_SMS * 16 ? need : GRID_SMS * 16), threads = h.warps * h.groups * 32;
    if constexpr (!WIDE || NV == 1) {                        // eight pieces a thread: rows of three warps and more
        if (h.warps == 1) {
            norm_kernel<T, WIDE, NV, false, PACK><<<grid, threads, 0, s>>>(p, h.warps);
            return cudaGetLastError();
        }
    }
    norm_kernel<T, WIDE, NV, true, PACK><<<grid, threads, 0, s>>>(p, h.warps);
    return cudaGetLastError();
}

template <typename T, bool PACK>
cudaError_t norm_pack_t(const NormParams& p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = p.D % N == 0 && p.x_stride % N == 0 && aligned16(p.x) && aligned16(p.y) && (!p.w || aligned16(p.w)) &&
                      (!p.b || aligned16(p.b)) && (reinterpret_cast<uintptr_t>(p.payload) & (N - 1)) == 0;
    if (ring_pays(p.rows, p.D, RING_VALUES) && ring_warps(p.D) <= MAX_WARPS) {
        if (wide) return norm_ring_launch<T, PACK>(p, s);
        if (p.D > SHIFT_DIM && first_row_alone(p.x, p.x_stride * static_cast<int64_t>(sizeof(T)), p.rows)) return norm_shift_launch<T, PACK>(p, s);
    }
    const RowShape h = wide ? row_shape(p.rows, p.D / N, 1, 8, 8) : narrow_shape(p.rows, p.D, 8);      // wide: nv is 1 or 8 here
    if (h.warps == 0 || (!wide && p.D > RING_DIM)) {      // the latter: expanded or overlapping rows at an odd address
        norm_loop_kernel<T><<<row_blocks(p.rows), 256, 0, s>>>(p);
        return cudaGetLastError();
    }
    if (!wide) return h.nv == 4 ? norm_launch<T, false, 4, PACK>(p, h, s) : norm_launch<T, false, 8, PACK>(p, h, s);      // up to RING_DIM here
    return h.nv == 1 ? norm_launch<T, true, 1, PACK>(p, h, s) : norm_launch<T, true, 8, PACK>(p, h, s);
}

template <typename T>
cudaError_t norm_t(const NormParams& p, cudaStream_t s) {
    return p.payload ? norm_pack_t<T, true>(p, s) : norm_pack_t<T, false>(p, s);
}

template <typename T, bool WIDE, int NV, bool KEPT>
cudaError_t norm_grad_launch(const NormGradParams& p, const RowShape& h, cudaStream_t s) {
    const unsigned threads = h.warps * h.groups * 32, grid = static_cast<unsigned>(p.splits);
    const size_t smem = h.groups > 1 ? sizeof(float) * 2 * h.warps * 32 * NV * Piece<T, WIDE>::N : 0;
    if constexpr (WIDE ? NV == 1 : NV < 16) {                // sixteen values a thread: rows of five warps and more
        if (h.warps == 1) {
            norm_grad_kernel<T, WIDE, NV, false, KEPT><<<grid, threads, smem, s>>>(p, h.warps);
            return cudaGetLastError();
        }
    }
    norm_grad_kernel<T, WIDE, NV, true, KEPT><<<grid, threads, smem, s>>>(p, h.warps);
    return cudaGetLastError();
}

template <typename T, int W, bool KEPT>
cudaError_t norm_grad_ring_width(NormGradParams& p, cudaStream_t s) {
    constexpr int X = KEPT ? 1 : static_cast<int>(sizeof(T));           // bytes of a kept value
    constexpr int STAGES = sizeof(T) == 4 ? 3 : 6;                       // at most 193 KB
    constexpr int SMEM = STAGES * (RING_THREADS * RING_COLUMNS * (static_cast<int>(sizeof(T)) + X) + RING_THREADS / 2);
    auto* kernel = norm_grad_ring_kernel<T, W, KEPT, STAGES>;
    const int warps = ring_warps(p.D), groups = MAX_WARPS / warps;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    const int64_t need = (p.rows + groups - 1) / groups;
    p.splits = static_cast<int>(need < MAX_SPLITS ? need : MAX_SPLITS);
    kernel<<<p.splits, groups * warps * 32, SMEM, s>>>(p, warps);
    return cudaGetLastError();
}
template <typename T, bool KEPT>
cudaError_t norm_grad_ring_launch(NormGradParams& p, cudaStream_t s) {
    switch (ring_width(p.D)) {
        case 1: return norm_grad_ring_width<T, 1, KEPT>(p, s);
        case 2: return norm_grad_ring_width<T, 2, KEPT>(p, s);
        case 4: return norm_grad_ring_width<T, 4, KEPT>(p, s);
        case 8: return norm_grad_ring_width<T, 8, KEPT>(p, s);
        case 16: return norm_grad_ring_width<T, 16, KEPT>(p, s);
        default: return norm_grad_ring_width<T, 0, KEPT>(p, s);
    }
}

template <typename T, bool KEPT>
cudaError_t norm_grad_shift_launch(NormGradParams& p, cudaStream_t s) {
    constexpr int STAGES = sizeof(T) == 4 ? (KEPT ? 3 : 2) : (KEPT ? 5 : 4);          // at most 170 KB
    auto* kernel = norm_grad_shift_kernel<T, KEPT, STAGES>;
    const int warps = ring_warps(p.D), groups = MAX_WARPS / warps, columns = warps * 32 * RING_COLUMNS;
    const int smem = groups * (STAGES * (row_room(columns, sizeof(T)) + row_room(columns, KEPT ? 1 : sizeof(T)) + 16) + 16 +
                               row_room(columns, sizeof(T)));
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int64_t need = (p.rows + groups - 1) / groups;
    p.splits = static_cast<int>(need < MAX_SPLITS ? need : MAX_SPLITS);
    kernel<<<p.splits, groups * warps * 32, smem, s>>>(p, warps);
    return cudaGetLastError();
}

template <typename T, bool KEPT>
cudaError_t norm_grad_kept_t(NormGradParams p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    bool wide = p.D % N == 0 && p.dy_stride % N == 0 && aligned16(p.dy) && (!p.dx || aligned16(p.dx)) && (!p.add || aligned16(p.add)) &&
                (!p.w || aligned16(p.w));
    wide = wide && (KEPT ? (reinterpret_cast<uintptr_t>(p.payload) & (N - 1)) == 0 : p.x_stride % N == 0 && aligned16(p.x));
    const RowShape h = wide ? row_shape(p.rows, p.D / N, 1, 16 / N, 16) : narrow_shape(p.rows, p.D, 16);      // wide: nv is 1, or 4 of fp32 here
    const bool sums = p.dw || p.db;
    const bool alone = wide || (first_row_alone(p.dy, p.dy_stride * static_cast<int64_t>(sizeof(T)), p.rows) &&
                                (KEPT || first_row_alone(p.x, p.x_stride * static_cast<int64_t>(sizeof(T)), p.rows)));
    if (p.rows > 0 && ring_warps(p.D) <= MAX_WARPS && (wide ? ring_pays(p.rows, p.D, RING_GRAD_VALUES) : alone && !p.add && shift_grad_pays(p.rows, p.D))) {
        const cudaError_t e = wide ? norm_grad_ring_launch<T, KEPT>(p, s) : norm_grad_shift_launch<T, KEPT>(p, s);
        if (e != cudaSuccess) return e;
    } else if (h.warps == 0 || p.rows == 0) {
        p.splits = splits_for(p.rows);
        const int64_t columns = wide ? 32 * N : 32;
        const dim3 grid(static_cast<unsigned>((p.D + columns - 1) / columns), static_cast<unsigned>(p.splits));
        if (p.dx) {
            if (wide) norm_grad_rows_loop_kernel<T, true, KEPT><<<row_blocks(p.rows), 256, 0, s>>>(p);
            else norm_grad_rows_loop_kernel<T, false, KEPT><<<row_blocks(p.rows), 256, 0, s>>>(p);
        }
        if (sums) {
            if (wide) norm_grad_cols_loop_kernel<T, true, KEPT><<<grid, 256, 0, s>>>(p);
            else norm_grad_cols_loop_kernel<T, false, KEPT><<<grid, 256, 0, s>>>(p);
        }
    } else {
        const int64_t need = (p.rows + h.groups - 1) / h.groups;
        p.splits = static_cast<int>(need < MAX_SPLITS ? need : MAX_SPLITS);
        cudaError_t e;
        if (!wide) e = h.nv == 4 ? norm_grad_launch<T, false, 4, KEPT>(p, h, s)
                     : h.nv == 8 ? norm_grad_launch<T, false, 8, KEPT>(p, h, s) : norm_grad_launch<T, false, 16, KEPT>(p, h, s);
        else if constexpr (N == 8) e = norm_grad_launch<T, true, 1, KEPT>(p, h, s);      // up to RING_DIM here
        else e = h.nv == 1 ? norm_grad_launch<T, true, 1, KEPT>(p, h, s) : norm_grad_launch<T, true, 4, KEPT>(p, h, s);
        if (e != cudaSuccess) return e;
    }
    if (sums) return launch_behind(norm_grad_join_kernel<T>, dim3(static_cast<unsigned>((p.D + 31) / 32)), dim3(32 * JOIN_LANES), s, p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t norm_grad_t(const NormGradParams& p, cudaStream_t s) {
    return p.payload ? norm_grad_kept_t<T, true>(p, s) : norm_grad_kept_t<T, false>(p, s);
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
bool act_dtype_ok(int d) { return d == PEER_DTYPE_F32 || d == PEER_DTYPE_BF16 || d == PEER_DTYPE_F16; }

}  // namespace
}  // namespace peer

using namespace peer;

extern "C" int peer_layer_norm(const void* x, int64_t x_stride, int32_t dtype, const void* weight, const void* bias,
                               int32_t param_dtype, float eps, int64_t rows, int64_t dim, void* y, float* mean, float* rstd,
                               void* payload, float* scale, void* stream) {
    if (rows < 0 || dim < 1 || dim > PEER_ROW_DIM_MAX || x_stride < 0)
        return refuse("peer_layer_norm: negative row count or stride, or dim outside [1, 2^20]");
    if (!act_dtype_ok(dtype)) return refuse("peer_layer_norm: dtype must be F32, BF16 or F16");
    if (param_dtype != PEER_DTYPE_F32 && param_dtype != dtype)
        return refuse("peer_layer_norm: the parameters are fp32 or of the activations' dtype");
    if (!(eps >= 0.f)) return refuse("peer_layer_norm: eps must not be negative");
    if ((payload == nullptr) != (scale == nullptr)) return refuse("peer_layer_norm: payload and scale come together");
    if (rows == 0) return PEER_OK;
    if (!x || !y) return refuse("peer_layer_norm: null pointer");
    if (!aligned_to(x, dtype) || !aligned_to(y, dtype) || !aligned_to(weight, param_dtype) || !aligned_to(bias, param_dtype) ||
        !aligned_to(mean, PEER_DTYPE_F32) || !aligned_to(rstd, PEER_DTYPE_F32) || !aligned_to(scale, PEER_DTYPE_F32))
        return refuse("peer_layer_norm: a pointer is not aligned to its type");
    NormParams p{x, x_stride, weight, bias, param_dtype == PEER_DTYPE_F32, eps, rows, dim, y, mean, rstd,
                 static_cast<uint8_t*>(payload), scale};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_layer_norm", norm_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_layer_norm", norm_t<__nv_bfloat16>(p, s));
    return report("peer_layer_norm", norm_t<__half>(p, s));
}

extern "C" int64_t peer_layer_norm_workspace(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 1) return 0;
    const int64_t splits = rows < MAX_SPLITS ? (rows < 1 ? 1 : rows) : MAX_SPLITS;
    return splits * 2 * dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int peer_layer_norm_backward(const void* grad_y, int64_t grad_stride, const void* x, int64_t x_stride,
                                        const void* payload, const float* scale, const float* mean, const float* rstd,
                                        const void* weight, int32_t dtype, int32_t param_dtype, const void* add, int64_t rows,
                                        int64_t dim, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    if (rows < 0 || dim < 1 || dim > PEER_ROW_DIM_MAX || x_stride < 0 || grad_stride < 0)
        return refuse("peer_layer_norm_backward: negative row count or stride, or dim outside [1, 2^20]");
    if (!act_dtype_ok(dtype)) return refuse("peer_layer_norm_backward: dtype must be F32, BF16 or F16");
    if (param_dtype != PEER_DTYPE_F32 && param_dtype != dtype)
        return refuse("peer_layer_norm_backward: the parameters are fp32 or of the activations' dtype");
    if ((payload == nullptr) != (scale == nullptr)) return refuse("peer_layer_norm_backward: payload and scale come together");
    if (rows > 0 && (!grad_y || !mean || !rstd || (!x && !payload)))
        return refuse("peer_layer_norm_backward: grad_y, mean, rstd and x (or its packed form) are required");
    if ((grad_weight || grad_bias) && (!workspace || workspace_bytes < peer_layer_norm_workspace(rows, dim)))
        return refuse("peer_layer_norm_backward: workspace is missing or smaller than peer_layer_norm_workspace says");
    if (!aligned_to(grad_y, dtype) || !aligned_to(x, dtype) || !aligned_to(add, dtype) || !aligned_to(grad_x, dtype) ||
        !aligned_to(weight, param_dtype) || !aligned_to(grad_weight, param_dtype) || !aligned_to(grad_bias, param_dtype) ||
        !aligned_to(mean, PEER_DTYPE_F32) || !aligned_to(rstd, PEER_DTYPE_F32) || !aligned_to(scale, PEER_DTYPE_F32) ||
        !aligned16(workspace))
        return refuse("peer_layer_norm_backward: a pointer is not aligned to its type, or the workspace to 16 bytes");
    if (rows == 0 && !grad_weight && !grad_bias) return PEER_OK;
    NormGradParams p{grad_y, grad_stride, x, x_stride, static_cast<const uint8_t*>(payload), scale, mean, rstd, weight,
                     param_dtype == PEER_DTYPE_F32, add, rows, dim, rows ? grad_x : nullptr, grad_weight, grad_bias,
                     static_cast<float*>(workspace), 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_layer_norm_backward", norm_grad_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_layer_norm_backward", norm_grad_t<__nv_bfloat16>(p, s));
    return report("peer_layer_norm_backward", norm_grad_t<__half>(p, s));
}
