// feq_expertlin.cu -- the experts' linear maps on rows sorted by expert, forward and backward.
//
//   y[r, p, :]  = W[e(r), irrep(p)] x[r, p, :]  (+ bias[e(r), scalar(p)] on l = 0 components)
//   gx[r, p, :] = W[e(r), irrep(p)]^T gy[r, p, :]
//   gW[e, i]    = sum over rows r of e and components p of irrep i of gy[r, p] x[r, p]^T
//   gb[e, s]    = sum over rows r of e of gy[r, component of scalar s]
//
// Rows of expert e are offsets[e] .. offsets[e + 1); rows from offsets[experts] on belong to none and
// give zeros.  The offsets stay on the device.
#include "feq_token.cuh"

namespace feq {
namespace elin {

using namespace token;

constexpr int kMaxExperts = 512;
constexpr int kT = 64;                        // tile edge

// Components of a row: which weight they use, and which bias (-1: none).
struct Comps {
    int dim, reps, scalars;
    int8_t rep[kMaxDim], scalar[kMaxDim];
};

struct Args {
    const void *x, *w, *b, *gy;               // b in the weights' type
    void *y, *gx, *gw, *gb;
    int64_t rows, x_row, x_comp, gy_row, gy_comp;   // strides in elements; channels are contiguous
    int experts, cin, cout;
    const int32_t *offsets;
};

// offsets as the kernels use them: never decreasing and within the rows.
__device__ __forceinline__ void load_offsets(const Args &a, int32_t *off) {
    if (threadIdx.x == 0) {
        int32_t at = 0;
        for (int e = 0; e <= a.experts; e++) {
            const int32_t v = a.offsets[e];
            if (e > 0) at = v < at ? at : (v > a.rows ? (int32_t)a.rows : v);
            off[e] = at;
        }
    }
    __syncthreads();
}

// Tile `tile` of the row tiles of all experts (each expert's rows in tiles of kT, then the rows
// that belong to none): expert (a.experts for none) and first and last row; false past the end.
__device__ __forceinline__ bool find_tile(const Args &a, const int32_t *off, int tile, int &e, int64_t &r0, int64_t &r1) {
    for (e = 0; e <= a.experts; e++) {
        const int64_t lo = off[e], hi = e == a.experts ? a.rows : off[e + 1];
        const int n = (int)((hi - lo + kT - 1) / kT);
        if (tile < n) {
            r0 = lo + (int64_t)tile * kT;
            r1 = min64(r0 + kT, hi);
            return true;
        }
        tile -= n;
    }
    return false;
}

// C[r, j] = sum_k A[r, k] B[j * bj + k * bk] (+ bias[j]) for one row tile, 64 columns, one component.
template <typename T>
__global__ void __launch_bounds__(256)
rows_kernel(const Args a, const Comps c, const T *A, int64_t a_row, int64_t a_comp, int K, int J, int bj, int bk,
            const T *bias, T *C) {
    __shared__ int32_t off[kMaxExperts + 1];
    __shared__ float As[kT][17], Bs[kT][17];
    load_offsets(a, off);
    int e;
    int64_t r0, r1;
    if (!find_tile(a, off, blockIdx.y, e, r0, r1)) return;
    const int p = blockIdx.z, j0 = blockIdx.x * kT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float acc[4][4] = {};
    if (e < a.experts) {
        const T *B = static_cast<const T *>(a.w) + ((int64_t)e * c.reps + c.rep[p]) * a.cin * a.cout;
        for (int k0 = 0; k0 < K; k0 += 16) {
            for (int i = threadIdx.x; i < kT * 16; i += 256) {
                const int row = i >> 4, k = k0 + (i & 15);
                As[row][i & 15] = r0 + row < r1 && k < K ? to_f32(A[(r0 + row) * a_row + p * a_comp + k]) : 0.0f;
                Bs[row][i & 15] = j0 + row < J && k < K ? to_f32(B[(int64_t)(j0 + row) * bj + (int64_t)k * bk]) : 0.0f;
            }
            __syncthreads();
            for (int k = 0; k < 16; k++)
                for (int u = 0; u < 4; u++)
                    for (int v = 0; v < 4; v++) acc[u][v] += As[ty * 4 + u][k] * Bs[tx * 4 + v][k];
            __syncthreads();
        }
    }
    for (int u = 0; u < 4; u++)
        for (int v = 0; v < 4; v++) {
            const int64_t r = r0 + ty * 4 + u;
            const int j = j0 + tx * 4 + v;
            if (r >= r1 || j >= J) continue;
            float s = acc[u][v];
            if (bias && e < a.experts && c.scalar[p] >= 0)
                s += to_f32(bias[((int64_t)e * c.scalars + c.scalar[p]) * J + j]);
            C[(r * c.dim + p) * J + j] = from_f32<T>(s);
        }
}

// gW of one expert and irrep, a 64 x 64 tile (o, i).
template <typename T>
__global__ void __launch_bounds__(256) weights_kernel(const Args a, const Comps c) {
    __shared__ int32_t off[kMaxExperts + 1];
    __shared__ float Gs[16][kT + 1], Xs[16][kT + 1];
    load_offsets(a, off);
    const int e = blockIdx.z / c.reps, rep = blockIdx.z % c.reps;
    const int o0 = blockIdx.y * kT, i0 = blockIdx.x * kT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const T *x = static_cast<const T *>(a.x), *g = static_cast<const T *>(a.gy);
    float acc[4][4] = {}, total[4][4] = {};
    for (int p = 0; p < c.dim; p++) {
        if (c.rep[p] != rep) continue;
        for (int64_t r0 = off[e]; r0 < off[e + 1]; r0 += 16) {
            for (int i = threadIdx.x; i < kT * 16; i += 256) {
                const int row = i >> 6, col = i & 63;
                const bool live = r0 + row < off[e + 1];
                Gs[row][col] = live && o0 + col < a.cout ? to_f32(g[(r0 + row) * a.gy_row + p * a.gy_comp + o0 + col]) : 0.0f;
                Xs[row][col] = live && i0 + col < a.cin ? to_f32(x[(r0 + row) * a.x_row + p * a.x_comp + i0 + col]) : 0.0f;
            }
            __syncthreads();
            for (int k = 0; k < 16; k++)
                for (int u = 0; u < 4; u++)
                    for (int v = 0; v < 4; v++) acc[u][v] += Gs[k][ty * 4 + u] * Xs[k][tx * 4 + v];
            __syncthreads();
            // sums of at most 256 rows are joined, so that a long sum keeps its last bits
            if (((r0 - off[e]) & 255) == 240 || r0 + 16 >= off[e + 1])
                for (int u = 0; u < 4; u++)
                    for (int v = 0; v < 4; v++) {
                        total[u][v] += acc[u][v];
                        acc[u][v] = 0.0f;
                    }
        }
    }
    T *out = static_cast<T *>(a.gw) + (int64_t)blockIdx.z * a.cin * a.cout;
    for (int u = 0; u < 4; u++)
        for (int v = 0; v < 4; v++)
            if (o0 + ty * 4 + u < a.cout && i0 + tx * 4 + v < a.cin)
                out[(int64_t)(o0 + ty * 4 + u) * a.cin + i0 + tx * 4 + v] = from_f32<T>(total[u][v]);
}

// gb of one expert and scalar: a warp per 32 columns walks the expert's rows.
template <typename T>
__global__ void __launch_bounds__(1024) bias_kernel(const Args a, const Comps c) {
    __shared__ int32_t off[kMaxExperts + 1];
    __shared__ float sh[32][33];
    load_offsets(a, off);
    const int e = blockIdx.y / c.scalars, sc = blockIdx.y % c.scalars;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, o = blockIdx.x * 32 + lane;
    int p = 0;
    while (c.scalar[p] != sc) p++;
    float s = 0.0f;
    if (o < a.cout)
        for (int64_t r = off[e] + warp; r < off[e + 1]; r += 32)
            s += to_f32(static_cast<const T *>(a.gy)[r * a.gy_row + p * a.gy_comp + o]);
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && o < a.cout) {
        float v = 0.0f;
        for (int k = 0; k < 32; k++) v += sh[k][lane];
        static_cast<T *>(a.gb)[(int64_t)blockIdx.y * a.cout + o] = from_f32<T>(v);
    }
}

int build_comps(const int32_t *lvals, int32_t n, Comps *c) {
    if (!lvals || n < 1) return FEQ_ERR_INVALID_ARGUMENT;
    if (n > kMaxIrreps) return FEQ_ERR_UNSUPPORTED;
    c->dim = 0;
    c->reps = n;
    c->scalars = 0;
    for (int i = 0; i < n; i++) {
        if (lvals[i] < 0) return FEQ_ERR_INVALID_ARGUMENT;
        if (lvals[i] > kMaxL || c->dim + 2 * lvals[i] + 1 > kMaxDim) return FEQ_ERR_UNSUPPORTED;
        for (int m = 0; m < 2 * lvals[i] + 1; m++) {
            c->rep[c->dim] = (int8_t)i;
            c->scalar[c->dim++] = (int8_t)(lvals[i] == 0 ? c->scalars : -1);
        }
        c->scalars += lvals[i] == 0;
    }
    return FEQ_OK;
}

int check(int64_t rows, int32_t experts, int32_t cin, int32_t cout, int32_t dtype) {
    if (rows < 0 || experts < 1 || cin < 1 || cout < 1 || !dtype_ok(dtype)) return FEQ_ERR_INVALID_ARGUMENT;
    if (experts > kMaxExperts || rows >= (int64_t)1 << 31) return FEQ_ERR_UNSUPPORTED;
    return FEQ_OK;
}

}  // namespace elin
}  // namespace feq

using namespace feq;
using namespace feq::token;

extern "C" size_t feq_expert_linear_workspace_bytes(const FeqExpertLinearArgs *args, int32_t backward) {
    elin::Comps c = {};
    if (!args || elin::check(args->rows, args->num_experts, args->c_in, args->c_out, args->dtype) != FEQ_OK ||
        elin::build_comps(args->lvals, args->n_lvals, &c) != FEQ_OK)
        return 0;
    return 256;
}

extern "C" int feq_expert_linear_fwd(const FeqExpertLinearArgs *args, void *workspace, size_t workspace_bytes,
                                     feq_stream_t stream) {
    if (!args) return FEQ_ERR_INVALID_ARGUMENT;
    const FeqExpertLinearArgs &q = *args;
    elin::Comps c = {};
    int rc = elin::check(q.rows, q.num_experts, q.c_in, q.c_out, q.dtype);
    if (rc == FEQ_OK) rc = elin::build_comps(q.lvals, q.n_lvals, &c);
    if (rc != FEQ_OK) return rc;
    if (q.rows == 0) return FEQ_OK;
    if (!q.x || !q.weight || !q.offsets || !q.out) return FEQ_ERR_INVALID_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    ProfScope prof("expert_linear", s);
    elin::Args a = {};
    a.w = q.weight;
    a.rows = q.rows;
    a.experts = q.num_experts;
    a.cin = q.c_in;
    a.cout = q.c_out;
    a.offsets = q.offsets;
    const dim3 grid((q.c_out + 63) / 64, (unsigned)((q.rows + 63) / 64 + q.num_experts + 1), c.dim);
    FEQ_TOKEN_TYPE(q.dtype, elin::rows_kernel<T><<<grid, 256, 0, s>>>(
                                a, c, static_cast<const T *>(q.x), q.x_row_stride, q.x_comp_stride, q.c_in, q.c_out,
                                q.c_in, 1, static_cast<const T *>(q.bias), static_cast<T *>(q.out));)
    FEQ_LAUNCH_CHECK();
    return FEQ_OK;
}

extern "C" int feq_expert_linear_bwd(const FeqExpertLinearArgs *args, void *workspace, size_t workspace_bytes,
                                     feq_stream_t stream) {
    if (!args) return FEQ_ERR_INVALID_ARGUMENT;
    const FeqExpertLinearArgs &q = *args;
    elin::Comps c = {};
    int rc = elin::check(q.rows, q.num_experts, q.c_in, q.c_out, q.dtype);
    if (rc == FEQ_OK) rc = elin::build_comps(q.lvals, q.n_lvals, &c);
    if (rc != FEQ_OK) return rc;
    if (!q.offsets || (q.rows && !q.grad_out) || (q.grad_x && !q.weight) || (q.rows && q.grad_weight && !q.x))
        return FEQ_ERR_INVALID_ARGUMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    ProfScope prof("expert_linear_bwd", s);
    elin::Args a = {};
    a.x = q.x;
    a.w = q.weight;
    a.gy = q.grad_out;
    a.gw = q.grad_weight;
    a.gb = q.grad_bias;
    a.rows = q.rows;
    a.x_row = q.x_row_stride;
    a.x_comp = q.x_comp_stride;
    a.gy_row = q.grad_row_stride;
    a.gy_comp = q.grad_comp_stride;
    a.experts = q.num_experts;
    a.cin = q.c_in;
    a.cout = q.c_out;
    a.offsets = q.offsets;
    if (q.grad_x && q.rows) {
        const dim3 grid((q.c_in + 63) / 64, (unsigned)((q.rows + 63) / 64 + q.num_experts + 1), c.dim);
        FEQ_TOKEN_TYPE(q.dtype, elin::rows_kernel<T><<<grid, 256, 0, s>>>(
                                    a, c, static_cast<const T *>(q.grad_out), q.grad_row_stride, q.grad_comp_stride,
                                    q.c_out, q.c_in, 1, q.c_in, nullptr, static_cast<T *>(q.grad_x));)
        FEQ_LAUNCH_CHECK();
    }
    if (q.grad_weight) {
        const dim3 grid((q.c_in + 63) / 64, (q.c_out + 63) / 64, q.num_experts * c.reps);
        FEQ_TOKEN_TYPE(q.dtype, elin::weights_kernel<T><<<grid, 256, 0, s>>>(a, c);)
        FEQ_LAUNCH_CHECK();
    }
    if (q.grad_bias && c.scalars) {
        const dim3 grid((q.c_out + 31) / 32, q.num_experts * c.scalars);
        FEQ_TOKEN_TYPE(q.dtype, elin::bias_kernel<T><<<grid, 1024, 0, s>>>(a, c);)
        FEQ_LAUNCH_CHECK();
    }
    return FEQ_OK;
}
