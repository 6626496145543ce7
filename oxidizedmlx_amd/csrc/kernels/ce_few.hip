// ce_few.hip — the linear cross entropy of a few f32 rows (up to 64), which
// reading W (and writing dW) bounds: W goes from memory straight into the f32
// matrix instructions, with no copies and no planes.
//
//   stats: z = x W^T, a wave per 16 entries of the vocabulary; the row maxima and
//          sums of a workgroup's 64 entries, and the targets' logits.
//   ds:    z again, kept as dS^T [vocab][16 NB] (zeros behind the rows).
//   grad:  a wave per 64 columns and slice of the vocabulary: dW = dS^T x of 16
//          entries at a time, and its sums of dx = dS W.
//
// v_mfma_f32_16x16x4_f32: lane l gives row (column) l % 16 of A (B) at k = l / 16
// and holds rows 4 (l / 16) + i of column l % 16 of the result. A lane loads four
// consecutive floats and gives them to four instructions: along K that is a
// permutation of the sum, along the columns of W and x one of the columns, which
// the stores undo.
//
// 8 rows of 1024 over 32000 entries: forward 131 MB of W, floor 27 us; backward
// W twice and dW once.
#include "../common.hpp"
#include "../kernels.hpp"
#include "ce_gemm.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace ce {
namespace {

constexpr int F = MLXHIP_DTYPE_F32;

__device__ inline f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// z[v][r] of the wave's 16 entries from v0 on and NB tiles of 16 rows.
template <int NB>
__device__ inline void few_logits(const FewArgs& g, int64_t v0, int lane, f32x4 (&acc)[NB]) {
    const int i = lane & 15, q = lane >> 4;
    const float* w = g.w + min(v0 + i, g.vocab - 1) * g.dim;
    const float* x[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        x[b] = g.x + min((int64_t)(16 * b + i), g.rows - 1) * g.dim;
        acc[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int64_t whole = g.dim / 16 * 16;
#pragma unroll 8
    for (int64_t k = 0; k < whole; k += 16) {
        float a[4], c[NB][4];
        dev::unpack<F>(dev::Vec16<F>{*reinterpret_cast<const dev::AnyVec<F>*>(w + k + 4 * q)}, a);
#pragma unroll
        for (int b = 0; b < NB; ++b)
            dev::unpack<F>(dev::Vec16<F>{*reinterpret_cast<const dev::AnyVec<F>*>(x[b] + k + 4 * q)}, c[b]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] = mfma4(a[e], c[b][e], acc[b]);
    }
    if (whole < g.dim) {
        float a[4], c[NB][4];
        dev::unpack<F>(dev::load_raw<F>(w, whole + 4 * q, g.dim), a);
#pragma unroll
        for (int b = 0; b < NB; ++b) dev::unpack<F>(dev::load_raw<F>(x[b], whole + 4 * q, g.dim), c[b]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] = mfma4(a[e], c[b][e], acc[b]);
    }
}

template <int NB>
__global__ __launch_bounds__(256) void few_stats_kernel(FewArgs g) {
    __shared__ float red[4][2][16 * NB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * 16;
    f32x4 acc[NB];
    if (v0 < g.vocab) few_logits<NB>(g, v0, lane, acc);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = 16 * b + i;
        float m = -INFINITY, s = 0.0f;
        if (v0 < g.vocab) {
            const int64_t t = r < g.rows ? g.targets[r] - (v0 + 4 * q) : -1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = v0 + 4 * q + e < g.vocab;
                if (in && t == e) g.target_z[r] = acc[b][e];
                // fmaxf would drop a NaN; the sum below keeps it.
                if (in) m = fmaxf(m, acc[b][e]);
            }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v0 + 4 * q + e < g.vocab) s += __builtin_amdgcn_exp2f((acc[b][e] - base) * LOG2E);
        }
        merge(m, s, __shfl_xor(m, 16, 64), __shfl_xor(s, 16, 64));
        merge(m, s, __shfl_xor(m, 32, 64), __shfl_xor(s, 32, 64));
        if (q == 0) {
            red[wave][0][16 * b + i] = m;
            red[wave][1][16 * b + i] = s;
        }
    }
    __syncthreads();
    const int r = threadIdx.x;
    if (r >= 16 * NB || r >= g.rows) return;
    float m = red[0][0][r], s = red[0][1][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) merge(m, s, red[w][0][r], red[w][1][r]);
    g.stats[r * g.stat_tiles + blockIdx.x] = make_float2(m, s);
}

template <int NB>
__global__ __launch_bounds__(256) void few_ds_kernel(FewArgs g) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
    if (v0 >= g.vocab) return;
    f32x4 acc[NB];
    few_logits<NB>(g, v0, lane, acc);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = 16 * b + i;
        const bool on = r < g.rows && counted(g.targets[r], g.vocab);
        const float lse = on ? g.lse[r] : 0.0f, f = on ? g.dloss[r] : 0.0f;
        const int64_t t = on ? g.targets[r] - (v0 + 4 * q) : -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f((acc[b][e] - lse) * LOG2E) - (t == e ? 1.0f : 0.0f);
            if (v0 + 4 * q + e < g.vocab) g.ds[(v0 + 4 * q + e) * (16 * NB) + r] = on ? p * f : 0.0f;
        }
    }
}

template <int NB>
__global__ __launch_bounds__(256) void few_grad_kernel(FewArgs g) {
    constexpr int RP = 16 * NB;
    __shared__ float sums[4][RP][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 64 + 4 * i;  // the lane's four columns
    const int64_t from = ((int64_t)blockIdx.y * 4 + wave) * g.slice, to = min(from + g.slice, g.vocab);
    // x at k = 4 t + q, columns n0 + j; zeros in rows without a target.
    float xr[4 * NB][4];
#pragma unroll
    for (int t = 0; t < 4 * NB; ++t) {
        const int64_t r = 4 * t + q;
#pragma unroll
        for (int j = 0; j < 4; ++j) xr[t][j] = 0.0f;
        if (r < g.rows && counted(g.targets[r], g.vocab) && n0 < g.dim)
            dev::unpack<F>(dev::load_raw<F>(g.x + r * g.dim, n0, g.dim), xr[t]);
    }
    f32x4 dx[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) dx[b][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t v = from; v < to; v += 16) {
        if (g.dx) {
            float w[4][4], a[4][NB];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t at = v + 4 * s + q;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[s][j] = 0.0f;
                if (at < to && n0 < g.dim) dev::unpack<F>(dev::load_raw<F>(g.w + at * g.dim, n0, g.dim), w[s]);
#pragma unroll
                for (int b = 0; b < NB; ++b) a[s][b] = at < to ? g.ds[at * RP + 16 * b + i] : 0.0f;
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) dx[b][j] = mfma4(a[s][b], w[s][j], dx[b][j]);
        }
        if (g.dw) {
            f32x4 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const float* ds = g.ds + min(v + i, g.vocab - 1) * RP + q;
#pragma unroll
            for (int t = 0; t < 4 * NB; ++t) {
                const float a = ds[4 * t];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = mfma4(a, xr[t][j], o[j]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float out[4] = {o[0][e], o[1][e], o[2][e], o[3][e]};
                if (v + 4 * q + e < to && n0 < g.dim) dev::store_vec<F>(g.dw + (v + 4 * q + e) * g.dim, n0, g.dim, out);
            }
        }
    }
    if (!g.dx) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][16 * b + 4 * q + e][4 * i + j] = dx[b][j][e];
    __syncthreads();
    for (int k = threadIdx.x; k < RP * 16; k += 256) {
        const int64_t r = k >> 4, c = 4 * (k & 15), n = (int64_t)blockIdx.x * 64 + c;
        if (r >= g.rows || n >= g.ldx) continue;
        float4 s = *reinterpret_cast<const float4*>(&sums[0][r][c]);
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const float4 o = *reinterpret_cast<const float4*>(&sums[w][r][c]);
            s = make_float4(s.x + o.x, s.y + o.y, s.z + o.z, s.w + o.w);
        }
        *reinterpret_cast<float4*>(g.dx + ((int64_t)blockIdx.y * g.rows + r) * g.ldx + n) = s;
    }
}

template <int NB>
int few(int which, const FewArgs& g, hipStream_t s) {
    const dim3 entries((unsigned)ceil_div(g.vocab, 64));
    if (which == CE_STATS) {
        hipLaunchKernelGGL((few_stats_kernel<NB>), entries, dim3(256), 0, s, g);
        return launch_check("few_stats_kernel");
    }
    if (which == CE_DS) {
        hipLaunchKernelGGL((few_ds_kernel<NB>), entries, dim3(256), 0, s, g);
        return launch_check("few_ds_kernel");
    }
    hipLaunchKernelGGL((few_grad_kernel<NB>), dim3((unsigned)ceil_div(g.dim, 64), (unsigned)g.slices), dim3(256), 0, s, g);
    return launch_check("few_grad_kernel");
}

}  // namespace
}  // namespace ce

int ce_few(int which, const ce::FewArgs& g, hipStream_t s) {
    if (g.rows <= 16) return ce::few<1>(which, g, s);
    if (g.rows <= 32) return ce::few<2>(which, g, s);
    return ce::few<4>(which, g, s);
}

}  // namespace mlxhip
