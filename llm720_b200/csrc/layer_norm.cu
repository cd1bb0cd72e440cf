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

template <typename T>
__global__ void __launch_bounds__(256) norm_grad_join_kernel(const NormGradParams p) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (c >= p.D) return;
    float aw = 0.f, ab = 0.f;
    for (int i = 0; i < p.splits; ++i) {
        aw += p.partial[(static_cast<int64_t>(i) * 2 + 0) * p.D + c];
        ab += p.partial[(static_cast<int64_t>(i) * 2 + 1) * p.D + c];
    }
    if (p.dw) { if (p.param_f32) static_cast<float*>(p.dw)[c] = aw; else static_cast<T*>(p.dw)[c] = from_f32<T>(aw); }
    if (p.db) { if (p.param_f32) static_cast<float*>(p.db)[c] = ab; else static_cast<T*>(p.db)[c] = from_f32<T>(ab); }
}

int splits_for(int64_t rows) {
    const int64_t s = (rows + 63) / 64;
    return static_cast<int>(s < 1 ? 1 : (s > 128 ? 128 : s));
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>(rows < 148 * 64 ? rows : 148 * 64); }

template <typename T>
cudaError_t norm_t(const NormParams& p, cudaStream_t s) {
    norm_loop_kernel<T><<<row_blocks(p.rows), 256, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t norm_grad_t(const NormGradParams& p, cudaStream_t s) {
    if (p.dx) norm_grad_rows_loop_kernel<T><<<row_blocks(p.rows), 256, 0, s>>>(p);
    if (p.dw || p.db) {
        norm_grad_cols_loop_kernel<T><<<dim3(static_cast<unsigned>((p.D + 31) / 32), static_cast<unsigned>(p.splits)), 256, 0, s>>>(p);
        norm_grad_join_kernel<T><<<static_cast<unsigned>((p.D + 255) / 256), 256, 0, s>>>(p);
    }
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
    return static_cast<int64_t>(splits_for(rows)) * 2 * dim * static_cast<int64_t>(sizeof(float));
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
                     static_cast<float*>(workspace), splits_for(rows)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_layer_norm_backward", norm_grad_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_layer_norm_backward", norm_grad_t<__nv_bfloat16>(p, s));
    return report("peer_layer_norm_backward", norm_grad_t<__half>(p, s));
}
