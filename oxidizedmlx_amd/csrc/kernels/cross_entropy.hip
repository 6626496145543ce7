// cross_entropy.hip — softmax cross entropy of the logits x W^T of an output
// projection, and the gradients of x and W, in pieces of the vocabulary: the
// logits are never held whole.
//
//   z_rv   = sum_k x_rk W_vk
//   lse_r  = log sum_v exp(z_rv)          (running maximum and sum)
//   loss_r = lse_r - z_r,t(r)             (0 for a target outside [0, vocab))
//   dS_rv  = dloss_r (exp(z_rv - lse_r) - [v = t(r)])   (0 for such a target)
//   dx = dS W,  dW = dS^T x
#include "../common.hpp"
#include "../kernels.hpp"
#include "device_math.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace {

using dev::Elem;

constexpr float LOG2E = 1.44269504088896340736f;
// Bytes of one piece's logits.
constexpr int64_t PIECE_BYTES = int64_t(128) << 20;

__device__ inline bool counted(int32_t t, int64_t vocab) { return t >= 0 && t < vocab; }

// Running maximum and sum of a row over one more piece of its logits, and the
// target's logit where the piece holds it; a workgroup per row.
__global__ __launch_bounds__(256) void ce_stats_kernel(const float* __restrict__ z, int64_t rows, int64_t width, int64_t v0,
                                                       const int32_t* __restrict__ targets, float2* __restrict__ stats,
                                                       float* __restrict__ target_z, bool first) {
    __shared__ float2 waves[4];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* p = z + r * width;
        float m = -INFINITY;
        for (int64_t c = threadIdx.x; c < width; c += 256) m = fmaxf(m, p[c]);
        m = dev::wave_max(m);
        float s = 0.0f;
        const float base = m == -INFINITY ? 0.0f : m;
        for (int64_t c = threadIdx.x; c < width; c += 256) s += exp2f((p[c] - base) * LOG2E);
        s = dev::wave_sum(s);
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = make_float2(m, s);
        __syncthreads();
        if (threadIdx.x == 0) {
            float2 a = first ? make_float2(-INFINITY, 0.0f) : stats[r];
            for (int w = 0; w < 4; ++w) {
                const float2 b = waves[w];
                const float mn = fmaxf(a.x, b.x);
                const float mb = mn == -INFINITY ? 0.0f : mn;
                a = make_float2(mn, a.y * exp2f((a.x - mb) * LOG2E) + b.y * exp2f((b.x - mb) * LOG2E));
            }
            stats[r] = a;
            const int64_t t = (int64_t)targets[r] - v0;
            if (t >= 0 && t < width) target_z[r] = p[t];
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void ce_loss_kernel(const float2* __restrict__ stats, const float* __restrict__ target_z,
                                                      const int32_t* __restrict__ targets, int64_t rows, int64_t vocab,
                                                      float* __restrict__ loss, float* __restrict__ lse) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const float2 a = stats[r];
    const float l = a.x + logf(a.y);
    lse[r] = l;
    loss[r] = counted(targets[r], vocab) ? l - target_z[r] : 0.0f;
}

// z becomes dS.
__global__ __launch_bounds__(256) void ce_grad_kernel(float* __restrict__ z, int64_t rows, int64_t width, int64_t v0,
                                                      int64_t vocab, const int32_t* __restrict__ targets,
                                                      const float* __restrict__ lse, const float* __restrict__ dloss) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int32_t t = targets[r];
        const bool on = counted(t, vocab);
        const float l = lse[r], g = dloss[r];
        for (int64_t c = threadIdx.x; c < width; c += 256) {
            const float p = exp2f((z[r * width + c] - l) * LOG2E);
            z[r * width + c] = on ? g * (v0 + c == t ? p - 1.0f : p) : 0.0f;
        }
    }
}

// x as f32, zeros in the rows without a target (whatever they hold must not
// reach dW through a product with 0).
template <int DT>
__global__ __launch_bounds__(256) void ce_rows_kernel(const typename Elem<DT>::type* __restrict__ x, int64_t rows,
                                                      int64_t dim, int64_t vocab, const int32_t* __restrict__ targets,
                                                      float* __restrict__ out) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const bool on = !targets || counted(targets[r], vocab);
        for (int64_t c = threadIdx.x; c < dim; c += 256) out[r * dim + c] = on ? dev::to_f32<DT>(x[r * dim + c]) : 0.0f;
    }
}

// Rows of sum (f32) into dx, zeros where there is no target.
template <int DT>
__global__ __launch_bounds__(256) void ce_out_kernel(const float* __restrict__ sum, int64_t rows, int64_t dim, int64_t vocab,
                                                     const int32_t* __restrict__ targets,
                                                     typename Elem<DT>::type* __restrict__ out) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const bool on = !targets || counted(targets[r], vocab);
        for (int64_t c = threadIdx.x; c < dim; c += 256) out[r * dim + c] = dev::from_f32<DT>(on ? sum[r * dim + c] : 0.0f);
    }
}

__global__ __launch_bounds__(256) void ce_add_kernel(float* __restrict__ acc, const float* __restrict__ v, int64_t n,
                                                     bool first) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        acc[i] = first ? v[i] : acc[i] + v[i];
}

template <typename T>
__global__ __launch_bounds__(256) void ce_zero_kernel(T* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = T(0);
}

unsigned row_grid(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }

// Sub-blocks of one workspace.
struct Carve {
    size_t used = 0;
    size_t take(size_t bytes) {
        const size_t at = used;
        used += (bytes + 255) / 256 * 256;
        return at;
    }
};

int64_t piece_width(int64_t rows, int64_t vocab) {
    const int64_t w = std::max<int64_t>(PIECE_BYTES / 4 / std::max<int64_t>(rows, 1) / 256 * 256, 1024);
    return std::min(w, vocab);
}

template <int DT>
int run_loss(const void* x, const void* w, const int32_t* targets, float* loss, float* lse, int64_t rows, int64_t dim,
             int64_t vocab, hipStream_t s) {
    typedef typename Elem<DT>::type T;
    const int64_t width = piece_width(rows, vocab);
    Carve c;
    const size_t oz = c.take((size_t)rows * width * 4), os = c.take((size_t)rows * 8), ot = c.take((size_t)rows * 4);
    const bool wide = DT == MLXHIP_DTYPE_F32;
    const size_t ox = c.take(wide ? 0 : (size_t)rows * dim * 4), ow = c.take(wide ? 0 : (size_t)width * dim * 4);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    float *z = (float*)(ws + oz), *tz = (float*)(ws + ot);
    float2* stats = (float2*)(ws + os);
    const float* xf = (const float*)x;
    if (!wide) {
        xf = (float*)(ws + ox);
        hipLaunchKernelGGL((ce_rows_kernel<DT>), dim3(row_grid(rows)), dim3(256), 0, s, (const T*)x, rows, dim, vocab,
                           nullptr, (float*)(ws + ox));
        MLXHIP_TRY(launch_check("ce_rows_kernel"));
    }
    for (int64_t v0 = 0; v0 < vocab; v0 += width) {
        const int64_t n = std::min(width, vocab - v0);
        const float* wf = (const float*)w + v0 * dim;
        if (!wide) {
            wf = (float*)(ws + ow);
            hipLaunchKernelGGL((ce_rows_kernel<DT>), dim3(row_grid(n)), dim3(256), 0, s, (const T*)w + v0 * dim, n, dim,
                               vocab, nullptr, (float*)(ws + ow));
            MLXHIP_TRY(launch_check("ce_rows_kernel"));
        }
        MLXHIP_TRY(gemm(MLXHIP_DTYPE_F32, MLXHIP_DTYPE_F32, 0, 1, rows, n, dim, 1, xf, dim, 0, wf, dim, 0, z, n, 0, s));
        hipLaunchKernelGGL(ce_stats_kernel, dim3(row_grid(rows)), dim3(256), 0, s, z, rows, n, v0, targets, stats, tz,
                           v0 == 0);
        MLXHIP_TRY(launch_check("ce_stats_kernel"));
    }
    hipLaunchKernelGGL(ce_loss_kernel, dim3((unsigned)ceil_div(rows, 256)), dim3(256), 0, s, stats, tz, targets, rows, vocab,
                       loss, lse);
    return launch_check("ce_loss_kernel");
}

template <int DT>
int run_grad(const void* x, const void* w, const int32_t* targets, const float* lse, const float* dloss, void* dx,
             void* dw, int64_t rows, int64_t dim, int64_t vocab, hipStream_t s) {
    typedef typename Elem<DT>::type T;
    if (rows == 0) {  // a sum over no rows
        if (!dw) return MLXHIP_OK;
        hipLaunchKernelGGL((ce_zero_kernel<T>), dim3((unsigned)std::min<int64_t>(ceil_div(vocab * dim, 256), 4096)),
                           dim3(256), 0, s, (T*)dw, vocab * dim);
        return launch_check("ce_zero_kernel");
    }
    const int64_t width = piece_width(rows, vocab);
    const bool wide = DT == MLXHIP_DTYPE_F32;
    Carve c;
    const size_t oz = c.take((size_t)rows * width * 4), oa = c.take((size_t)rows * dim * 4),
                 op = c.take((size_t)rows * dim * 4), ox = c.take((size_t)rows * dim * 4),
                 ow = c.take(wide ? 0 : (size_t)width * dim * 4), od = c.take(wide ? 0 : (size_t)width * dim * 4);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    float *z = (float*)(ws + oz), *acc = (float*)(ws + oa), *part = (float*)(ws + op), *xf = (float*)(ws + ox);
    hipLaunchKernelGGL((ce_rows_kernel<DT>), dim3(row_grid(rows)), dim3(256), 0, s, (const T*)x, rows, dim, vocab, targets,
                       xf);
    MLXHIP_TRY(launch_check("ce_rows_kernel"));
    for (int64_t v0 = 0; v0 < vocab; v0 += width) {
        const int64_t n = std::min(width, vocab - v0);
        const float* wf = (const float*)w + v0 * dim;
        if (!wide) {
            wf = (float*)(ws + ow);
            hipLaunchKernelGGL((ce_rows_kernel<DT>), dim3(row_grid(n)), dim3(256), 0, s, (const T*)w + v0 * dim, n, dim,
                               vocab, nullptr, (float*)(ws + ow));
            MLXHIP_TRY(launch_check("ce_rows_kernel"));
        }
        MLXHIP_TRY(gemm(MLXHIP_DTYPE_F32, MLXHIP_DTYPE_F32, 0, 1, rows, n, dim, 1, xf, dim, 0, wf, dim, 0, z, n, 0, s));
        hipLaunchKernelGGL(ce_grad_kernel, dim3(row_grid(rows)), dim3(256), 0, s, z, rows, n, v0, vocab, targets, lse,
                           dloss);
        MLXHIP_TRY(launch_check("ce_grad_kernel"));
        if (dx) {
            MLXHIP_TRY(gemm(MLXHIP_DTYPE_F32, MLXHIP_DTYPE_F32, 0, 0, rows, dim, n, 1, z, n, 0, wf, dim, 0, part, dim, 0, s));
            hipLaunchKernelGGL(ce_add_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(rows * dim, 256), 4096)), dim3(256),
                               0, s, acc, part, rows * dim, v0 == 0);
            MLXHIP_TRY(launch_check("ce_add_kernel"));
        }
        if (dw) {
            float* to = wide ? (float*)dw + v0 * dim : (float*)(ws + od);
            MLXHIP_TRY(gemm(MLXHIP_DTYPE_F32, MLXHIP_DTYPE_F32, 1, 0, n, dim, rows, 1, z, n, 0, xf, dim, 0, to, dim, 0, s));
            if (!wide) {
                hipLaunchKernelGGL((ce_out_kernel<DT>), dim3(row_grid(n)), dim3(256), 0, s, to, n, dim, vocab, nullptr,
                                   (T*)dw + v0 * dim);
                MLXHIP_TRY(launch_check("ce_out_kernel"));
            }
        }
    }
    if (!dx) return MLXHIP_OK;
    hipLaunchKernelGGL((ce_out_kernel<DT>), dim3(row_grid(rows)), dim3(256), 0, s, acc, rows, dim, vocab, targets, (T*)dx);
    return launch_check("ce_out_kernel");
}

}  // namespace

int linear_cross_entropy(int dt, const void* x, const void* w, const int32_t* targets, float* loss, float* lse,
                         int64_t rows, int64_t dim, int64_t vocab, hipStream_t s) {
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) { rc = run_loss<d.value>(x, w, targets, loss, lse, rows, dim, vocab, s); }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

int linear_cross_entropy_vjp(int dt, const void* x, const void* w, const int32_t* targets, const float* lse,
                             const float* dloss, void* dx, void* dw, int64_t rows, int64_t dim, int64_t vocab,
                             hipStream_t s) {
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            rc = run_grad<d.value>(x, w, targets, lse, dloss, dx, dw, rows, dim, vocab, s);
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy gradient: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

}  // namespace mlxhip
