// feq_layernorm.cu -- layer norm over the last dimension, forward and backward.
//
//   mu = sum_j x_j / D,  v = sum_j (x_j - mu)^2 / D,  r = 1 / sqrt(v + eps),  u = (x - mu) r
//   y  = u w + b
//   gx = r (g w - mean_j(g w) - u mean_j(g w u)),  gw = sum_rows g u,  gb = sum_rows g
//
// Both passes move every element once (forward 2, backward 3 elements per position) and do about
// ten operations on it, so HBM bounds them.  A row is held in registers by a group of `tpr`
// threads (a power of two, within a warp or of whole warps), E elements a thread, so the mean and
// the centred sum of squares are exact two-pass sums over registers and the row is read once.
// A thread owns the same columns for every row of its group, so w and b are read once per
// thread and, backwards, gw and gb are summed in registers over the group's rows; the groups of
// a block join in shared memory and the blocks in a second kernel, all in a fixed order.
// Products that enter the row's sums, and u mean(g w u), are rounded before they are added: in rows of
// two the terms of gx cancel down to eps / v of their size, and a product kept longer on one side only
// would be what is left.
// Rows wider than kMaxWidth go through kernels that stream the row from L2 instead.
#include "feq_token.cuh"

namespace feq {
namespace lnorm {

using namespace token;

constexpr int kBlock = 256;
constexpr int kMaxTpr = 512;
constexpr int kMaxWidth = 16 * kMaxTpr;      // 16 elements a thread
constexpr int kLimitWidth = 1 << 29;         // column arithmetic stays in 32 bits
constexpr int kReduceCols = 32;

struct Args {
    const void *x, *g, *w, *b;
    void *y, *gx;
    float *mean, *rstd;
    float *partial;                           // (blocks, 2, width)
    int64_t rows, x_stride, g_stride;
    int width, tpr, param_f32;
    float eps;
};

// Sum over the `tpr` threads of a group.  tpr > 32: red holds one value per warp of the block and
// each group has a named barrier; `slot` alternates so that one barrier per sum is enough.
__device__ __forceinline__ float group_sum(float v, int tpr, float (*red)[32], int &slot) {
    if (tpr <= 32) return lane_sum(v, tpr);
    v = lane_sum(v, 32);
    const int nw = tpr >> 5, lane = threadIdx.x & 31, group = threadIdx.x / tpr;
    if (lane == 0) red[slot][threadIdx.x >> 5] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
    const float s = lane < nw ? red[slot][group * nw + lane] : 0.0f;
    slot ^= 1;
    return lane_sum(s, 32);
}

// Element e of a thread's row part is column (e / V * tpr + t) * V + e % V.
template <typename T, int V, int E>
__device__ __forceinline__ void load_row(const T *row, int width, int tpr, int t, float (&v)[E]) {
    constexpr int N = E / V;
    Pack<T, V> p[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int c = (i * tpr + t) * V;
        if (c < width) p[i] = *reinterpret_cast<const Pack<T, V> *>(row + c);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int c = (i * tpr + t) * V;
#pragma unroll
        for (int q = 0; q < V; q++) v[i * V + q] = c < width ? to_f32(p[i].v[q]) : 0.0f;
    }
}

template <typename T, int V, int E>
__device__ __forceinline__ void store_row(T *row, int width, int tpr, int t, const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E / V; i++) {
        const int c = (i * tpr + t) * V;
        if (c < width) {
            Pack<T, V> p;
#pragma unroll
            for (int q = 0; q < V; q++) p.v[q] = from_f32<T>(v[i * V + q]);
            *reinterpret_cast<Pack<T, V> *>(row + c) = p;
        }
    }
}

template <typename T, int V, int E>
__device__ __forceinline__ void load_param(const void *p, int is_f32, float otherwise, int width, int tpr, int t,
                                           float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int c = (e / V * tpr + t) * V + e % V;
        v[e] = p && c < width ? param_at<T>(p, is_f32, c) : otherwise;
    }
}

template <typename T, int V, int E>
__global__ void __launch_bounds__(kMaxTpr) forward_kernel(const Args a) {
    __shared__ float red[2][32];
    int slot = 0;
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1);
    const int groups = blockDim.x / tpr;
    float w[E], b[E];
    load_param<T, V, E>(a.w, a.param_f32, 1.0f, a.width, tpr, t, w);
    load_param<T, V, E>(a.b, a.param_f32, 0.0f, a.width, tpr, t, b);
    const float inv = 1.0f / (float)a.width;
    // every thread of a warp makes the same number of rounds: the sums are warp-wide
    const int64_t step = (int64_t)gridDim.x * groups;
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + threadIdx.x / tpr;
        const bool live = r < a.rows;
        const int width = live ? a.width : 0;
        float x[E];
        load_row<T, V, E>(static_cast<const T *>(a.x) + (live ? r * a.x_stride : 0), width, tpr, t, x);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s += x[e];
        const float mu = group_sum(s, tpr, red, slot) * inv;
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = (e / V * tpr + t) * V;
            const float d = c < width ? x[e] - mu : 0.0f;
            x[e] = d;
            q += __fmul_rn(d, d);
        }
        const float rstd = rsqrtf(group_sum(q, tpr, red, slot) * inv + a.eps);
        if (live && t == 0 && a.mean) {
            a.mean[r] = mu;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = x[e] * rstd * w[e] + b[e];
        store_row<T, V, E>(static_cast<T *>(a.y) + (live ? r * (int64_t)a.width : 0), width, tpr, t, x);
    }
}

template <typename T, int V, int E>
__global__ void __launch_bounds__(kMaxTpr) backward_kernel(const Args a) {
    __shared__ float red[2][32];
    extern __shared__ float sums[];           // (2, width): gw and gb of this block
    int slot = 0;
    const int tpr = a.tpr, t = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr;
    const int groups = blockDim.x / tpr;
    float w[E], gw[E], gb[E];
    load_param<T, V, E>(a.w, a.param_f32, 1.0f, a.width, tpr, t, w);
#pragma unroll
    for (int e = 0; e < E; e++) gw[e] = gb[e] = 0.0f;
    const float inv = 1.0f / (float)a.width;
    const int64_t step = (int64_t)gridDim.x * groups;
    for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + group;
        const bool live = r < a.rows;
        const int width = live ? a.width : 0;
        float x[E], g[E];
        load_row<T, V, E>(static_cast<const T *>(a.x) + (live ? r * a.x_stride : 0), width, tpr, t, x);
        load_row<T, V, E>(static_cast<const T *>(a.g) + (live ? r * a.g_stride : 0), width, tpr, t, g);
        const float mu = live ? a.mean[r] : 0.0f, rstd = live ? a.rstd[r] : 0.0f;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = (e / V * tpr + t) * V;
            const float u = c < width ? (x[e] - mu) * rstd : 0.0f;
            gw[e] += g[e] * u;
            gb[e] += g[e];
            x[e] = u;
            g[e] *= w[e];
            s1 += g[e];
            s2 += __fmul_rn(g[e], u);
        }
        s1 = group_sum(s1, tpr, red, slot) * inv;
        s2 = group_sum(s2, tpr, red, slot) * inv;
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = rstd * (g[e] - s1 - __fmul_rn(x[e], s2));
        if (a.gx) store_row<T, V, E>(static_cast<T *>(a.gx) + (live ? r * (int64_t)a.width : 0), width, tpr, t, x);
    }
    if (!a.partial) return;
    // join the groups in their order
    for (int k = 0; k < groups; k++) {
        if (group == k) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int c = (e / V * tpr + t) * V + e % V;
                if (c < a.width) {
                    sums[c] = (k ? sums[c] : 0.0f) + gw[e];
                    sums[a.width + c] = (k ? sums[a.width + c] : 0.0f) + gb[e];
                }
            }
        }
        __syncthreads();
    }
    float *out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
    for (int i = threadIdx.x; i < 2 * a.width; i += blockDim.x) out[i] = sums[i];
}

// gw, gb = the sum of the blocks' partial sums: 32 columns a block, 32 warps over the partials,
// joined in warp order.
template <typename T>
__global__ void __launch_bounds__(1024)
reduce_kernel(const float *__restrict__ partial, int blocks, int width, int param_f32, void *gw, void *gb) {
    __shared__ float sh[32][kReduceCols + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * kReduceCols + lane;        // of 2 * width
    float s = 0.0f;
    if (i < 2 * width)
        for (int k = warp; k < blocks; k += 32) s += partial[(int64_t)k * 2 * width + i];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < 2 * width) {
        float v = 0.0f;
        for (int k = 0; k < 32; k++) v += sh[k][lane];
        if (i < width) {
            if (gw) param_put<T>(gw, param_f32, i, v);
        } else if (gb) {
            param_put<T>(gb, param_f32, i - width, v);
        }
    }
}

// ---- rows wider than kMaxWidth: one block a row, the row streamed once per sum ----
template <typename T>
__global__ void __launch_bounds__(1024) wide_forward_kernel(const Args a) {
    __shared__ float red[2][32];
    int slot = 0;
    const float inv = 1.0f / (float)a.width;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        T *y = static_cast<T *>(a.y) + r * (int64_t)a.width;
        float s = 0.0f, q = 0.0f;
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) s += to_f32(x[c]);
        const float mu = group_sum(s, blockDim.x, red, slot) * inv;
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
            const float d = to_f32(x[c]) - mu;
            q += d * d;
        }
        const float rstd = rsqrtf(group_sum(q, blockDim.x, red, slot) * inv + a.eps);
        if (threadIdx.x == 0 && a.mean) {
            a.mean[r] = mu;
            a.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
            const float u = (to_f32(x[c]) - mu) * rstd;
            y[c] = from_f32<T>(u * (a.w ? param_at<T>(a.w, a.param_f32, c) : 1.0f) +
                               (a.b ? param_at<T>(a.b, a.param_f32, c) : 0.0f));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) wide_backward_kernel(const Args a) {
    __shared__ float red[2][32];
    int slot = 0;
    const float inv = 1.0f / (float)a.width;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        const T *g = static_cast<const T *>(a.g) + r * a.g_stride;
        T *gx = static_cast<T *>(a.gx) + r * (int64_t)a.width;
        const float mu = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
            const float v = to_f32(g[c]) * (a.w ? param_at<T>(a.w, a.param_f32, c) : 1.0f);
            s1 += v;
            s2 += v * ((to_f32(x[c]) - mu) * rstd);
        }
        s1 = group_sum(s1, blockDim.x, red, slot) * inv;
        s2 = group_sum(s2, blockDim.x, red, slot) * inv;
        for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
            const float v = to_f32(g[c]) * (a.w ? param_at<T>(a.w, a.param_f32, c) : 1.0f);
            gx[c] = from_f32<T>(rstd * (v - s1 - (to_f32(x[c]) - mu) * rstd * s2));
        }
    }
}

// The columns of gw and gb over a share of the rows (a thread a column).
template <typename T>
__global__ void __launch_bounds__(kBlock) wide_columns_kernel(const Args a) {
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float g = to_f32(static_cast<const T *>(a.g)[r * a.g_stride + c]);
        sw += g * ((to_f32(static_cast<const T *>(a.x)[r * a.x_stride + c]) - a.mean[r]) * a.rstd[r]);
        sb += g;
    }
    float *out = a.partial + (int64_t)blockIdx.y * 2 * a.width;
    out[c] = sw;
    out[a.width + c] = sb;
}

// Elements a thread: 8 while a row fits one warp that way (more rows in flight, fewer registers),
// else 16.
int elems_per_thread(int width) { return width <= 8 * 32 ? 8 : 16; }

// Blocks of the backward: one wave at two blocks a SM, so that the partial sums stay few.
int64_t backward_blocks(int64_t rows, int width) {
    if (width > kMaxWidth) return min64(max64(rows / 8, 1), 64);
    const int tpr = pow2_ceil((width + elems_per_thread(width) - 1) / elems_per_thread(width));
    const int groups = tpr > kBlock ? 1 : kBlock / tpr;
    return max64(1, min64((rows + groups - 1) / groups, 148 * 2));
}

}  // namespace lnorm
}  // namespace feq

using namespace feq;
using namespace feq::token;

extern "C" size_t feq_layer_norm_bwd_workspace_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return (size_t)lnorm::backward_blocks(rows, width) * 2 * (size_t)width * sizeof(float);
}

extern "C" int feq_layer_norm_fwd(const void *x, int64_t rows, int64_t x_stride, int32_t width, int32_t dtype,
                                  const void *weight, const void *bias, int32_t param_f32, float eps, void *y,
                                  float *mean, float *rstd, feq_stream_t stream) {
    if (rows < 0 || width <= 0 || x_stride < 0 || !dtype_ok(dtype) || !(eps >= 0.0f)) return FEQ_ERR_INVALID_ARGUMENT;
    if (width > lnorm::kLimitWidth) return FEQ_ERR_UNSUPPORTED;
    if (rows == 0) return FEQ_OK;
    if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return FEQ_ERR_INVALID_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    ProfScope prof("layer_norm", s);
    lnorm::Args a = {};
    a.x = x;
    a.w = weight;
    a.b = bias;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.x_stride = x_stride;
    a.width = width;
    a.param_f32 = param_f32 || dtype == FEQ_DTYPE_F32;
    a.eps = eps;
    const size_t es = dtype_bytes(dtype);
    if (width > lnorm::kMaxWidth) {
        const unsigned grid = (unsigned)min64(rows, sm_count() * 2);
        FEQ_TOKEN_TYPE(dtype, lnorm::wide_forward_kernel<T><<<grid, 1024, 0, s>>>(a);)
        FEQ_LAUNCH_CHECK();
        return FEQ_OK;
    }
    const int vec = vector_elems((uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)y | (uint64_t)x_stride * es |
                                     (uint64_t)width * es, es);
    const int elems = lnorm::elems_per_thread(width);
    a.tpr = pow2_ceil((width + elems - 1) / elems);
    const int threads = a.tpr > lnorm::kBlock ? a.tpr : lnorm::kBlock, groups = threads / a.tpr;
    const unsigned grid = (unsigned)min64((rows + groups - 1) / groups, (int64_t)sm_count() * (2048 / threads));
    FEQ_TOKEN_TYPE(dtype, FEQ_TOKEN_VEC(T, vec, if (elems == 8) lnorm::forward_kernel<T, V, 8><<<grid, threads, 0, s>>>(a);
                                        else lnorm::forward_kernel<T, V, 16><<<grid, threads, 0, s>>>(a);))
    FEQ_LAUNCH_CHECK();
    return FEQ_OK;
}

extern "C" int feq_layer_norm_bwd(const void *grad_out, int64_t grad_stride, const void *x, int64_t rows,
                                  int64_t x_stride, int32_t width, int32_t dtype, const void *weight,
                                  int32_t param_f32, const float *mean, const float *rstd, void *grad_x,
                                  void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                                  feq_stream_t stream) {
    if (rows < 0 || width <= 0 || x_stride < 0 || grad_stride < 0 || !dtype_ok(dtype)) return FEQ_ERR_INVALID_ARGUMENT;
    if (width > lnorm::kLimitWidth) return FEQ_ERR_UNSUPPORTED;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool params = grad_weight || grad_bias;
    param_f32 = param_f32 || dtype == FEQ_DTYPE_F32;
    const size_t es = dtype_bytes(dtype);
    if (rows == 0) {                          // an empty sum
        const size_t bytes = (size_t)width * (param_f32 ? 4 : 2);
        if (grad_weight) FEQ_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, bytes, s));
        if (grad_bias) FEQ_CUDA_TRY(cudaMemsetAsync(grad_bias, 0, bytes, s));
        return FEQ_OK;
    }
    if (!x || !grad_out || !mean || !rstd || (!grad_x && !params)) return FEQ_ERR_INVALID_ARGUMENT;
    if (params && (!workspace || workspace_bytes < feq_layer_norm_bwd_workspace_bytes(rows, width)))
        return FEQ_ERR_WORKSPACE;
    ProfScope prof("layer_norm_bwd", s);
    lnorm::Args a = {};
    a.x = x;
    a.g = grad_out;
    a.w = weight;
    a.gx = grad_x;
    a.mean = const_cast<float *>(mean);
    a.rstd = const_cast<float *>(rstd);
    a.partial = params ? static_cast<float *>(workspace) : nullptr;
    a.rows = rows;
    a.x_stride = x_stride;
    a.g_stride = grad_stride;
    a.width = width;
    a.param_f32 = param_f32;
    const int blocks = (int)lnorm::backward_blocks(rows, width);
    if (width > lnorm::kMaxWidth) {
        if (grad_x) {
            const unsigned grid = (unsigned)min64(rows, sm_count() * 2);
            FEQ_TOKEN_TYPE(dtype, lnorm::wide_backward_kernel<T><<<grid, 1024, 0, s>>>(a);)
            FEQ_LAUNCH_CHECK();
        }
        if (params) {
            const dim3 grid((unsigned)((width + lnorm::kBlock - 1) / lnorm::kBlock), (unsigned)blocks);
            FEQ_TOKEN_TYPE(dtype, lnorm::wide_columns_kernel<T><<<grid, lnorm::kBlock, 0, s>>>(a);)
            FEQ_LAUNCH_CHECK();
        }
    } else {
        const int vec = vector_elems((uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)grad_out |
                                         (uint64_t)(uintptr_t)grad_x | (uint64_t)x_stride * es |
                                         (uint64_t)grad_stride * es | (uint64_t)width * es, es);
        const int elems = lnorm::elems_per_thread(width);
        a.tpr = pow2_ceil((width + elems - 1) / elems);
        const int threads = a.tpr > lnorm::kBlock ? a.tpr : lnorm::kBlock;
        const size_t smem = params ? (size_t)width * 2 * sizeof(float) : 0;
        FEQ_TOKEN_TYPE(dtype, FEQ_TOKEN_VEC(T, vec, {
            auto kern = elems == 8 ? lnorm::backward_kernel<T, V, 8> : lnorm::backward_kernel<T, V, 16>;
            if (smem > 40 * 1024)
                FEQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            kern<<<(unsigned)blocks, threads, smem, s>>>(a);
        }))
        FEQ_LAUNCH_CHECK();
    }
    if (params) {
        const unsigned grid = (unsigned)((2 * (int64_t)width + lnorm::kReduceCols - 1) / lnorm::kReduceCols);
        FEQ_TOKEN_TYPE(dtype, lnorm::reduce_kernel<T><<<grid, 1024, 0, s>>>(a.partial, blocks, width, param_f32,
                                                                          grad_weight, grad_bias);)
        FEQ_LAUNCH_CHECK();
    }
    return FEQ_OK;
}
