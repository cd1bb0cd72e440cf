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
        const float mean = block_sum(s, buf) / static_cast<float>(p.D);
        float ss = 0.f;
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) { const float d = to_f32<T>(xr[c]) - mean; ss = fmaf(d, d, ss); }
        const float rstd = 1.0f / sqrtf(block_sum(ss, buf) / static_cast<float>(p.D) + p.eps);
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

// x[r, c] of the backward pass, from either form
template <typename T>
__device__ __forceinline__ float kept_x(const NormGradParams& p, int64_t r, int64_t c, float s) {
    return p.payload ? unpacked<T>(e4m3_value(p.payload[r * p.D + c]), s) : to_f32<T>(static_cast<const T*>(p.x)[r * p.x_stride + c]);
}

template <typename T>
__global__ void __launch_bounds__(256) norm_grad_rows_loop_kernel(const NormGradParams p) {
    __shared__ float buf[33];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* dyr = static_cast<const T*>(p.dy) + r * p.dy_stride;
        const float mean = p.mean[r], rstd = p.rstd[r], sc = p.payload ? p.scale[r] : 1.f;
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) {
            const float g = to_f32<T>(dyr[c]) * (p.w ? param_at<T>(p.w, p.param_f32, c) : 1.f);
            s1 += g;
            s2 = fmaf(g, (kept_x<T>(p, r, c, sc) - mean) * rstd, s2);
        }
        s1 = block_sum(s1, buf) / static_cast<float>(p.D);
        s2 = block_sum(s2, buf) / static_cast<float>(p.D);
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) {
            const float g = to_f32<T>(dyr[c]) * (p.w ? param_at<T>(p.w, p.param_f32, c) : 1.f);
            float v = rstd * (g - s1 - (kept_x<T>(p, r, c, sc) - mean) * rstd * s2);
            if (p.add) v += to_f32<T>(static_cast<const T*>(p.add)[r * p.D + c]);
            static_cast<T*>(p.dx)[r * p.D + c] = from_f32<T>(v);
        }
    }
}

// column sums of one split of the rows: 32 columns by 8 row lanes per block
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_cols_loop_kernel(const NormGradParams p) {
    __shared__ float sw[8][33], sb[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
    const int64_t per = (p.rows + p.splits - 1) / p.splits;
    const int64_t r0 = per * blockIdx.y, r1 = r0 + per < p.rows ? r0 + per : p.rows;
    float aw = 0.f, ab = 0.f;
    if (c < p.D)
        for (int64_t r = r0 + ty; r < r1; r += 8) {
            const float d = to_f32<T>(static_cast<const T*>(p.dy)[r * p.dy_stride + c]);
            aw = fmaf(d, (kept_x<T>(p, r, c, p.payload ? p.scale[r] : 1.f) - p.mean[r]) * p.rstd[r], aw);
            ab += d;
        }
    sw[ty][tx] = aw;
    sb[ty][tx] = ab;
    __syncthreads();
    if (ty == 0 && c < p.D) {
        for (int i = 1; i < 8; ++i) { aw += sw[i][tx]; ab += sb[i][tx]; }
        p.partial[(static_cast<int64_t>(blockIdx.y) * 2 + 0) * p.D + c] = aw;
        p.partial[(static_cast<int64_t>(blockIdx.y) * 2 + 1) * p.D + c] = ab;
    }
}

// ---------------------------------------------------------------------------
// Rows of up to 16 values per thread of a 512-thread block: the row stays in registers.
//
// A group of `warps` warps owns a row, every thread the same NV pieces of columns in every row, so the parameters are
// read once per block and the column sums of the backward pass stay in registers until the end.  A group takes U rows
// at a time: U rows' loads are in flight together and one exchange between the group's warps serves all of them.
//
// Forward statistics: each warp computes the mean of its own columns and the sum of squared deviations from that mean,
// and the warps' results are merged with  M2 = sum M2_w + n_w (mean_w - mean)^2,  which loses nothing when the mean is
// large against the deviation and needs one exchange, not two.
// ---------------------------------------------------------------------------
constexpr int MAX_WARPS = MAX_ROW_WARPS;

template <typename T, int NV, int N>
__device__ __forceinline__ void load_params(const void* p, bool f32, int64_t D, int first, int step, float absent, float (&f)[NV * N]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (first + static_cast<int64_t>(i) * step) * N;
#pragma unroll
        for (int q = 0; q < N; ++q) f[i * N + q] = (p && c < D) ? param_at<T>(p, f32, c + q) : absent;
    }
}

template <typename T, bool WIDE, int NV, int U, bool MULTI, bool PACK>
__global__ void __launch_bounds__(512) norm_kernel(const NormParams p, int warps, int ru) {
    using P = Piece<T, WIDE>;
    constexpr int N = P::N, E = NV * N;
    __shared__ float2 part[MULTI ? 2 * MAX_WARPS * U : 1];
    __shared__ uint32_t part_top[MULTI && PACK ? 2 * MAX_WARPS * U : 1];
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = MULTI ? threadIdx.x / threads : threadIdx.x >> 5;
    const int gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    const int64_t pieces = p.D / N;
    float w[E], b[E];
    load_params<T, NV, N>(p.w, p.param_f32, p.D, gt, threads, 1.f, w);
    load_params<T, NV, N>(p.b, p.param_f32, p.D, gt, threads, 0.f, b);
    auto columns_of = [&](int wi) {                        // columns held by warp wi of the group
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t left = pieces - (static_cast<int64_t>(i) * threads + wi * 32);
            n += static_cast<int>(left < 0 ? 0 : (left > 32 ? 32 : left)) * N;
        }
        return static_cast<float>(n);
    };
    const float mine = columns_of(gw), inv_mine = mine > 0.f ? 1.f / mine : 0.f;
    const float inv_d = 1.f / static_cast<float>(p.D);
    int parity = 0;
    for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * groups + group) * ru; r0 < p.rows;
         r0 += static_cast<int64_t>(gridDim.x) * groups * ru) {
        typename P::Raw x[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = gt + static_cast<int64_t>(i) * threads;
                const bool in = u < ru && r0 + u < p.rows && c < pieces;
                x[u][i] = in ? P::load(static_cast<const T*>(p.x) + (r0 + u) * p.x_stride + c * N) : P::zero();
            }
        float s[U], mean[U], rstd[U];
        uint32_t top[U];
        bool odd[U];                                        // the warp holds an infinity or NaN of row u
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[N];
                P::decode(x[u][i], f);
#pragma unroll
                for (int q = 0; q < N; ++q) s[u] += f[q];
            }
            if (PACK) top[u] = warp_top<T, WIDE, NV>(x[u], odd[u]);
        }
        const float wm = warp_sums<U>(s) * inv_mine;        // lane u * (32 / U): this warp's mean of row u
        float m2[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = __shfl_sync(FULL_MASK, wm, u * (32 / U));
            m2[u] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (gt + static_cast<int64_t>(i) * threads < pieces) {
                    float f[N];
                    P::decode(x[u][i], f);
#pragma unroll
                    for (int q = 0; q < N; ++q) { const float d = f[q] - mean[u]; m2[u] = fmaf(d, d, m2[u]); }
                }
            }
        }
        const float wm2 = warp_sums<U>(m2);
        if constexpr (!MULTI) {
#pragma unroll
            for (int u = 0; u < U; ++u) rstd[u] = 1.f / sqrtf(__shfl_sync(FULL_MASK, wm2, u * (32 / U)) * inv_d + p.eps);
        } else {
            float2* slot = part + parity * MAX_WARPS * U + group * warps * U;
            uint32_t* slot_top = part_top + (PACK ? parity * MAX_WARPS * U + group * warps * U : 0);
            if (lane % (32 / U) == 0) slot[gw * U + lane / (32 / U)] = make_float2(wm, wm2);
            if (PACK && lane == 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) slot_top[gw * U + u] = top[u];
            }
            group_sync(group, threads);
#pragma unroll
            for (int u = 0; u < U; ++u) mean[u] = 0.f;
            for (int k = 0; k < warps; ++k) {
                const float n = columns_of(k);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    mean[u] = fmaf(n, slot[k * U + u].x, mean[u]);
                    if (PACK) top[u] = max(top[u], slot_top[k * U + u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) { mean[u] *= inv_d; m2[u] = 0.f; }
            for (int k = 0; k < warps; ++k) {
                const float n = columns_of(k);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float2 v = slot[k * U + u];
                    const float d = v.x - mean[u];
                    m2[u] += fmaf(n * d, d, v.y);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) rstd[u] = 1.f / sqrtf(m2[u] * inv_d + p.eps);
            parity ^= 1;                                    // the next rows' exchange leaves these slots alone
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = r0 + u;
            if (u >= ru || r >= p.rows) break;
            const int e = PACK ? e4m3_scale_exponent(top[u]) : 0;
            const float inv = exp2_int(-e);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = gt + static_cast<int64_t>(i) * threads;
                if (c >= pieces) break;
                float f[N], y[N];
                P::decode(x[u][i], f);
#pragma unroll
                for (int q = 0; q < N; ++q) y[q] = fmaf((f[q] - mean[u]) * rstd[u], w[i * N + q], b[i * N + q]);
                P::store(static_cast<T*>(p.y) + r * p.D + c * N, P::encode(y));
                if constexpr (PACK)
                    *reinterpret_cast<typename P::Packed*>(p.payload + r * p.D + c * N) = pack_piece<T, WIDE>(x[u][i], inv, odd[u]);
            }
            if (gt == 0) {
                if (p.mean) p.mean[r] = mean[u];
                if (p.rstd) p.rstd[r] = rstd[u];
                if (PACK) p.scale[r] = exp2_int(e);
            }
        }
    }
}

// KEPT: x comes in its 8-bit form
template <typename T, bool WIDE, int NV, int U, bool MULTI, bool KEPT>
__global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradParams p, int warps, int ru) {
    using P = Piece<T, WIDE>;
    using X = typename std::conditional<KEPT, typename P::Packed, typename P::Raw>::type;
    constexpr int N = P::N, E = NV * N;
    __shared__ float part[MULTI ? 2 * MAX_WARPS * U * 2 : 1];
    extern __shared__ float columns[];                     // [2][threads * E] when the block has several groups
    const int lane = threadIdx.x & 31, threads = warps * 32;
    const int group = MULTI ? threadIdx.x / threads : threadIdx.x >> 5;
    const int gt = threadIdx.x - group * threads, gw = gt >> 5;
    const int groups = blockDim.x / threads;
    const int64_t pieces = p.D / N;
    float w[E], aw[E], ab[E];
    load_params<T, NV, N>(p.w, p.param_f32, p.D, gt, threads, 1.f, w);
#pragma unroll
    for (int q = 0; q < E; ++q) aw[q] = ab[q] = 0.f;
    const float inv_d = 1.f / static_cast<float>(p.D);
    int parity = 0;
    for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * groups + group) * ru; r0 < p.rows;
         r0 += static_cast<int64_t>(gridDim.x) * groups * ru) {
        X x[U][NV];
        typename P::Raw dy[U][NV];
        float mean[U], rstd[U], sc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = r0 + u;
            const bool row_in = u < ru && r < p.rows;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = gt + static_cast<int64_t>(i) * threads;
                const bool in = row_in && c < pieces;
                dy[u][i] = in ? P::load(static_cast<const T*>(p.dy) + r * p.dy_stride + c * N) : P::zero();
                if constexpr (KEPT) x[u][i] = in ? P::load_packed(p.payload + r * p.D + c * N) : X{};
                else x[u][i] = in ? P::load(static_cast<const T*>(p.x) + r * p.x_stride + c * N) : P::zero();
            }
            mean[u] = row_in ? __ldg(p.mean + r) : 0.f;
            rstd[u] = row_in ? __ldg(p.rstd + r) : 0.f;
            sc[u] = KEPT && row_in ? __ldg(p.scale + r) : 1.f;
        }
        float s[2 * U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[N], d[N];
                if constexpr (KEPT) P::decode_packed(x[u][i], sc[u], f); else P::decode(x[u][i], f);
                P::decode(dy[u][i], d);                     // zero where there is no column or no row
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float n = (f[q] - mean[u]) * rstd[u], g = d[q] * w[i * N + q];
                    s[2 * u] += g;
                    s[2 * u + 1] = fmaf(g, n, s[2 * u + 1]);
                    aw[i * N + q] = fmaf(d[q], n, aw[i * N + q]);
                    ab[i * N + q] += d[q];
                }
            }
        }
        if (!p.dx) continue;
        const float total = warp_sums<2 * U>(s);
        float m1[U], m2[U];
        if constexpr (!MULTI) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                m1[u] = __shfl_sync(FULL_MASK, total, 2 * u * (16 / U)) * inv_d;
                m2[u] = __shfl_sync(FULL_MASK, total, (2 * u + 1) * (16 / U)) * inv_d;
            }
        } else {
            float* slot = part + (parity * MAX_WARPS + group * warps) * U * 2;
            if (lane % (16 / U) == 0) slot[gw * 2 * U + lane / (16 / U)] = total;
            group_sync(group, threads);
#pragma unroll
            for (int u = 0; u < U; ++u) m1[u] = m2[u] = 0.f;
            for (int k = 0; k < warps; ++k)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float2 v = *reinterpret_cast<const float2*>(slot + (k * U + u) * 2);
                    m1[u] += v.x;
                    m2[u] += v.y;
                }
#pragma unroll
            for (int u = 0; u < U; ++u) { m1[u] *= inv_d; m2[u] *= inv_d; }
            parity ^= 1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = r0 + u;
            if (u >= ru || r >= p.rows) break;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = gt + static_cast<int64_t>(i) * threads;
                if (c >= pieces) break;
                float f[N], d[N], a[N];
                if constexpr (KEPT) P::decode_packed(x[u][i], sc[u], f); else P::decode(x[u][i], f);
                P::decode(dy[u][i], d);
                if (p.add) P::decode(P::load(static_cast<const T*>(p.add) + r * p.D + c * N), a);
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float n = (f[q] - mean[u]) * rstd[u];
                    f[q] = rstd[u] * (d[q] * w[i * N + q] - m1[u] - n * m2[u]);
                    if (p.add) f[q] += a[q];
                }
                P::store(static_cast<T*>(p.dx) + r * p.D + c * N, P::encode(f));
            }
        }
    }
    if (!p.dw && !p.db) return;
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

// `splits` partial rows to the gradients: 32 columns by 8 lanes of partials per block
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_join_kernel(const NormGradParams p) {
    __shared__ float sw[8][33], sb[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + tx;
    float aw = 0.f, ab = 0.f;
    if (c < p.D) {
#pragma unroll 4
        for (int i = ty; i < p.splits; i += 8) {
            aw += p.partial[static_cast<int64_t>(i) * 2 * p.D + c];
            ab += p.partial[(static_cast<int64_t>(i) * 2 + 1) * p.D + c];
        }
    }
    sw[ty][tx] = aw;
    sb[ty][tx] = ab;
    __syncthreads();
    if (ty != 0 || c >= p.D) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) { aw += sw[i][tx]; ab += sb[i][tx]; }
    if (p.dw) { if (p.param_f32) static_cast<float*>(p.dw)[c] = aw; else static_cast<T*>(p.dw)[c] = from_f32<T>(aw); }
    if (p.db) { if (p.param_f32) static_cast<float*>(p.db)[c] = ab; else static_cast<T*>(p.db)[c] = from_f32<T>(ab); }
}

constexpr int MAX_SPLITS = GRID_SMS;       // one block per SM: rows of partial column sums

int splits_for(int64_t rows) {
    const int64_t s = (rows + 63) / 64;
    return static_cast<int>(s < 1 ? 1 : (s > MAX_SPLITS ? MAX_SPLITS : s));
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>(rows < 148 * 64 ? rows : 148 * 64); }

template <typename T, bool WIDE, int NV, int U, bool PACK>
cudaError_t norm_launch(const NormParams& p, const RowShape& h, cudaStream_t s) {
    const int64_t need = (p.rows + static_cast<int64_t>(h.groups) * h.u_rows - 1) / (static_cast<int64_t>(h.groups) * h.u_rows);
    const unsigned grid = static_cast<unsigned>(need < 148 * 4 ? need : 148 * 4), threads = h.warps * h.groups * 32;
    if (h.warps > 1) norm_kernel<T, WIDE, NV, U, true, PACK><<<grid, threads, 0, s>>>(p, h.warps, h.u_rows);
    else norm_kernel<T, WIDE, NV, U, false, PACK><<<grid, threads, 0, s>>>(p, h.warps, h.u_rows);
    return cudaGetLastError();
}

template <typename T, bool PACK>
cudaError_t norm_pack_t(const NormParams& p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = p.D % N == 0 && p.x_stride % N == 0 && aligned16(p.x) && aligned16(p.y) &&
                      (reinterpret_cast<uintptr_t>(p.payload) & (N - 1)) == 0;
    const RowShape h = wide ? row_shape(p.rows, p.D / N, 1, 16 / N, 8, 4) : row_shape(p.rows, p.D, 4, 16, 8, 2);
    if (h.warps == 0) {
        norm_loop_kernel<T><<<row_blocks(p.rows), 256, 0, s>>>(p);
        return cudaGetLastError();
    }
    if (!wide) return h.nv == 4 ? norm_launch<T, false, 4, 2, PACK>(p, h, s) : norm_launch<T, false, 16, 2, PACK>(p, h, s);
    if (h.nv == 1) return norm_launch<T, true, 1, 4, PACK>(p, h, s);
    return norm_launch<T, true, 16 / N, 4, PACK>(p, h, s);
}

template <typename T>
cudaError_t norm_t(const NormParams& p, cudaStream_t s) {
    return p.payload ? norm_pack_t<T, true>(p, s) : norm_pack_t<T, false>(p, s);
}

template <typename T, bool WIDE, int NV, int U, bool KEPT>
cudaError_t norm_grad_launch(const NormGradParams& p, const RowShape& h, cudaStream_t s) {
    const unsigned threads = h.warps * h.groups * 32;
    const size_t smem = h.groups > 1 ? sizeof(float) * 2 * h.warps * 32 * NV * Piece<T, WIDE>::N : 0;
    const unsigned grid = static_cast<unsigned>(p.splits);
    if (h.warps > 1) norm_grad_kernel<T, WIDE, NV, U, true, KEPT><<<grid, threads, smem, s>>>(p, h.warps, h.u_rows);
    else norm_grad_kernel<T, WIDE, NV, U, false, KEPT><<<grid, threads, smem, s>>>(p, h.warps, h.u_rows);
    return cudaGetLastError();
}

template <typename T, bool KEPT>
cudaError_t norm_grad_kept_t(NormGradParams p, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    bool wide = p.D % N == 0 && p.dy_stride % N == 0 && aligned16(p.dy) && (!p.dx || aligned16(p.dx)) && (!p.add || aligned16(p.add));
    wide = wide && (KEPT ? (reinterpret_cast<uintptr_t>(p.payload) & (N - 1)) == 0 : p.x_stride % N == 0 && aligned16(p.x));
    const RowShape h = wide ? row_shape(p.rows, p.D / N, 1, 16 / N, 16, 2) : row_shape(p.rows, p.D, 4, 16, 16, 1);
    const bool sums = p.dw || p.db;
    if (h.warps == 0 || p.rows == 0) {
        p.splits = splits_for(p.rows);
        if (p.dx) norm_grad_rows_loop_kernel<T><<<row_blocks(p.rows), 256, 0, s>>>(p);
        if (sums) norm_grad_cols_loop_kernel<T><<<dim3(static_cast<unsigned>((p.D + 31) / 32), static_cast<unsigned>(p.splits)), 256, 0, s>>>(p);
    } else {
        const int64_t need = (p.rows + static_cast<int64_t>(h.groups) * h.u_rows - 1) / (static_cast<int64_t>(h.groups) * h.u_rows);
        p.splits = static_cast<int>(need < MAX_SPLITS ? need : MAX_SPLITS);
        cudaError_t e;
        if (!wide) e = h.nv == 4 ? norm_grad_launch<T, false, 4, 1, KEPT>(p, h, s) : norm_grad_launch<T, false, 16, 1, KEPT>(p, h, s);
        else if (h.nv == 1) e = norm_grad_launch<T, true, 1, 2, KEPT>(p, h, s);
        else e = norm_grad_launch<T, true, 16 / N, 2, KEPT>(p, h, s);
        if (e != cudaSuccess) return e;
    }
    if (sums) norm_grad_join_kernel<T><<<static_cast<unsigned>((p.D + 31) / 32), 256, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t norm_grad_t(const NormGradParams& p, cudaStream_t s) {
    return p.payload ? norm_grad_kept_t<T, true>(p, s) : norm_grad_kept_t<T, false>(p, s);
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
    if (rows == 0 && !grad_weight && !grad_bias) return PEER_OK;
    NormGradParams p{grad_y, grad_stride, x, x_stride, static_cast<const uint8_t*>(payload), scale, mean, rstd, weight,
                     param_dtype == PEER_DTYPE_F32, add, rows, dim, rows ? grad_x : nullptr, grad_weight, grad_bias,
                     static_cast<float*>(workspace), 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_layer_norm_backward", norm_grad_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_layer_norm_backward", norm_grad_t<__nv_bfloat16>(p, s));
    return report("peer_layer_norm_backward", norm_grad_t<__half>(p, s));
}
