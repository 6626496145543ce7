// norm_affine.hip — layer norm over the last axis with a weight and a bias,
// and its gradients, for f32, bf16 and f16 rows.
//
//   xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   y  = xh w + b
//   g  = dy w;  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh;  db = sum over rows of dy
//
// The normalisation is the reference's layer_norm (crates/mlx-core/src/
// cpu_kernels.rs:338-363) and its gradient layer_norm_vjp (:403-454), neither
// of which has a weight or bias. All sums, statistics and products are f32;
// a 16-bit result is rounded once, as it is stored.
//
// Rows of up to 16384 columns stay in registers: WPR waves own a row, each
// lane NV 16-byte vectors of it (at most 16 values), so x and dy are read
// once and y or dx written once. The statistics take two exchanges between a
// row's lanes: the mean, then the sums of the deviations d from it, of d^2 and, going
// back, of g and g d as well. The mean of d is what the f32 mean is off by, by its own
// rounding and those of its sum: it is taken off d and out of the other sums, so a
// large mean costs no digits (a row of 3000.7s has deviations of 1e-9, and of 5e-4
// without). Workgroups walk over rows with the weights held in
// registers; going back each lane also keeps its columns' dw and db sums and
// writes them at the end as one partial row per workgroup, which a second
// launch adds up in a fixed order (no atomics: the same bits every time).
// Longer rows are read again from the caches: a launch for the rows'
// statistics, then one over tiles of columns.
//
// Bound by memory, small ones by the launches. 4096 rows of 4096, f32: 27 us forward
// (4.9 TB/s) and 34 back (5.9 TB/s, x and dy partly cached), the fold 4.8; 2048 bf16
// rows of 1024: 4.2, 8.2 and 2.5; 1000 f16 rows of 777: 3.8, 6.0 and 4.8.
#include "../common.hpp"
#include "../kernels.hpp"
#include "device_math.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace {

using dev::Elem;
using dev::load_raw;
using dev::store_vec;
using dev::to_f32;
using dev::unpack;
using dev::Vec16;

constexpr int MAX_COLS = 16384;    // of rows held in registers
constexpr int PARTIALS = 256;      // workgroups, and partial sums, of the gradient
constexpr int LONG_TILE = 1024;    // columns of a workgroup's tile for longer rows

// N sums over the WPR waves of a row; every lane gets them. Two rounds of
// slots alternate, so one barrier per call is enough.
template <int WPR, int N>
__device__ inline void row_sums(float (&v)[N], float* slots, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dev::wave_sum(v[i]);
    if constexpr (WPR > 1) {
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) slots[i * WPR + wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = slots[i * WPR];
#pragma unroll
            for (int w = 1; w < WPR; ++w) s += slots[i * WPR + w];
            v[i] = s;
        }
    }
}

// 1 / sqrt(var + eps) of a row whose deviations have the sum s1, the sum of squares s2
// and the mean off. Squares past f32's range make it 0, whatever the product gives.
__device__ inline float inverse_std(float s1, float s2, float off, float inv, float eps) {
    const float rest = s2 - off * s1, sum = s2 == INFINITY ? s2 : rest < 0.0f ? 0.0f : rest;  // NaN stays
    return 1.0f / sqrtf(sum * inv + eps);
}

// A row's columns in lane t of 64 * WPR: NV vectors, of which every one but the
// last is whole in all lanes (the launch picks NV so). The last begins at the
// row's end less VEC where it would run past it: its elements below `from` belong
// to other lanes too, which hold the same values, and count in no sum. (Loading
// such a row's end element by element: 1023 f16 columns of 16384 rows 22 us
// forward and 58 back; this way 13 and 27.) Rows of fewer than VEC columns end at `to`.
template <int DT, int WPR, int NV>
struct Columns {
    static constexpr int VEC = Elem<DT>::VEC;
    int t, last, from, to;
    __device__ Columns(int lane, int64_t cols) : t(lane) {
        const int c = ((NV - 1) * 64 * WPR + t) * VEC;
        last = min(c, max((int)cols - VEC, 0));
        from = min(c - last, VEC);
        to = min((int)cols, VEC);
    }
    __device__ int at(int j) const { return j < NV - 1 ? (j * 64 * WPR + t) * VEC : last; }
    // Whether element e of vector j counts.
    __device__ bool own(int j, int e) const { return j < NV - 1 || (e >= from && e < to); }
    __device__ void load(const typename Elem<DT>::type* p, Vec16<DT> (&out)[NV]) const {
#pragma unroll
        for (int j = 0; j < NV - 1; ++j) out[j].q = dev::load16<DT>(p + at(j));
        if (to == VEC) out[NV - 1].q = dev::load16<DT>(p + last);
        else out[NV - 1] = load_raw<DT>(p, 0, to);
    }
    __device__ void store(typename Elem<DT>::type* p, int j, const float* v) const {
        if (j < NV - 1 || from < VEC) store_vec<DT>(p, at(j), j < NV - 1 ? at(j) + VEC : last + to, v);
    }
};

template <int DT, int WPR, int NV>
__global__ __launch_bounds__(WPR < 4 ? 256 : 64 * WPR) void affine_fwd_kernel(
    const typename Elem<DT>::type* __restrict__ x, const typename Elem<DT>::type* __restrict__ w,
    const typename Elem<DT>::type* __restrict__ b, typename Elem<DT>::type* __restrict__ y, int64_t rows, int64_t cols,
    float eps) {
    constexpr int VEC = Elem<DT>::VEC, RPB = WPR < 4 ? 4 / WPR : 1;  // rows of a workgroup
    __shared__ float slots[2][RPB][2 * WPR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = wave / WPR, wr = wave % WPR;
    const Columns<DT, WPR, NV> col(wr * 64 + lane, cols);
    const float inv = 1.0f / (float)cols;
    Vec16<DT> wv[NV], bv[NV];
    col.load(w, wv);
    col.load(b, bv);
    for (int64_t r = (int64_t)blockIdx.x * RPB + sub; r < rows; r += (int64_t)gridDim.x * RPB) {
        Vec16<DT> raw[NV];
        col.load(x + r * cols, raw);
        float v[NV * VEC], s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack<DT>(raw[j], v + j * VEC);
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) s[0] += col.own(i / VEC, i % VEC) ? v[i] : 0.0f;
        row_sums<WPR, 1>(s, slots[0][sub], wr, lane);
        const float mean = s[0] / (float)cols;
        float m[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) {
            v[i] -= mean;
            const float d = col.own(i / VEC, i % VEC) ? v[i] : 0.0f;
            m[0] += d;
            m[1] += d * d;
        }
        row_sums<WPR, 2>(m, slots[1][sub], wr, lane);
        const float off = m[0] * inv, rstd = inverse_std(m[0], m[1], off, inv, eps);
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) v[i] -= off;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float wf[VEC], bf[VEC];
            unpack<DT>(wv[j], wf);
            unpack<DT>(bv[j], bf);
#pragma unroll
            for (int e = 0; e < VEC; ++e) wf[e] = v[j * VEC + e] * rstd * wf[e] + bf[e];
            col.store(y + r * cols, j, wf);
        }
    }
}

// dx, and the workgroup's sums of dw (part[2 * blockIdx.x]) and db (the row after).
template <int DT, int WPR, int NV>
__global__ __launch_bounds__(WPR < 4 ? 256 : 64 * WPR) void affine_bwd_kernel(
    const typename Elem<DT>::type* __restrict__ dy, const typename Elem<DT>::type* __restrict__ x,
    const typename Elem<DT>::type* __restrict__ w, typename Elem<DT>::type* __restrict__ dx, float* __restrict__ part,
    int64_t rows, int64_t cols, float eps) {
    constexpr int VEC = Elem<DT>::VEC, RPB = WPR < 4 ? 4 / WPR : 1, EPL = NV * VEC;
    __shared__ float slots[2][RPB][4 * WPR];
    __shared__ float fold[RPB > 1 ? RPB * 64 * EPL : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = wave / WPR, wr = wave % WPR;
    const Columns<DT, WPR, NV> col(wr * 64 + lane, cols);
    const float inv = 1.0f / (float)cols;
    Vec16<DT> wv[NV];
    col.load(w, wv);
    float aw[EPL], ab[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) aw[i] = ab[i] = 0.0f;
    // The next row's loads are in flight while this one is reduced.
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + sub;
    Vec16<DT> xn[NV], gn[NV];
    if (r < rows) {
        col.load(x + r * cols, xn);
        col.load(dy + r * cols, gn);
    }
    for (; r < rows; r += step) {
        Vec16<DT> xr[NV], gr[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            xr[j] = xn[j];
            gr[j] = gn[j];
        }
        if (r + step < rows) {
            col.load(x + (r + step) * cols, xn);
            col.load(dy + (r + step) * cols, gn);
        }
        float v[EPL], g[EPL], s1[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack<DT>(xr[j], v + j * VEC);
#pragma unroll
        for (int i = 0; i < EPL; ++i) s1[0] += col.own(i / VEC, i % VEC) ? v[i] : 0.0f;
        row_sums<WPR, 1>(s1, slots[0][sub], wr, lane);
        const float mean = s1[0] / (float)cols;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float wf[VEC];
            unpack<DT>(gr[j], g + j * VEC);
            unpack<DT>(wv[j], wf);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = j * VEC + e;
                v[i] -= mean;
                ab[i] += g[i];
                const float gw = col.own(j, e) ? g[i] * wf[e] : 0.0f, d = col.own(j, e) ? v[i] : 0.0f;
                s[0] += d;
                s[1] += d * d;
                s[2] += gw;
                s[3] += gw * d;
            }
        }
        row_sums<WPR, 4>(s, slots[1][sub], wr, lane);
        const float off = s[0] * inv, rstd = inverse_std(s[0], s[1], off, inv, eps);
        const float c1 = s[2] * inv, c2 = (s[3] - off * s[2]) * inv * rstd;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float wf[VEC];
            unpack<DT>(wv[j], wf);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = j * VEC + e;
                const float xh = (v[i] - off) * rstd;
                aw[i] += g[i] * xh;
                wf[e] = rstd * (g[i] * wf[e] - c1 - xh * c2);
            }
            col.store(dx + r * cols, j, wf);
        }
    }
    float* out = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float (&a)[EPL] = which ? ab : aw;
        if constexpr (RPB > 1) {
            // The rows' waves of a workgroup add up through LDS.
            __syncthreads();
#pragma unroll
            for (int i = 0; i < EPL; ++i) fold[(sub * EPL + i) * 64 + lane] = a[i];
            __syncthreads();
            if (sub == 0)
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    for (int k = 1; k < RPB; ++k) a[i] += fold[(k * EPL + i) * 64 + lane];
        }
        if (sub == 0)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (col.own(j, e)) out[which * cols + col.at(j) + e] = a[j * VEC + e];
    }
}

// Sums of n partial rows of 2 * cols values into dw and db: 32 columns of a
// workgroup, 32 threads to each, which fold every 32nd row (of 256 partial rows all
// eight loads in flight: by 8 threads the fold waited 9 us for 32 loads in turn; of fewer
// rows, what is no whole eight is loaded one by one: 250 rows of 1554 sums take 4.8 us
// where 256 of 2048 take 2.5) and then each other.
constexpr int FOLD = 32;
template <int DT>
__global__ __launch_bounds__(32 * FOLD) void affine_fold_kernel(const float* __restrict__ part, int64_t n, int64_t cols,
                                                                typename Elem<DT>::type* __restrict__ dw,
                                                                typename Elem<DT>::type* __restrict__ db) {
    __shared__ float sums[FOLD][33];
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    float s = 0.0f;
    if (col < 2 * cols) {
#pragma unroll 8
        for (int64_t i = k; i < n; i += FOLD) s += part[i * 2 * cols + col];
    }
    sums[k][c] = s;
    __syncthreads();
    // Lane c of wave-half k now adds up column k's sums.
    s = sums[c][k];
#pragma unroll
    for (int o = FOLD / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 32);
    const int64_t to = (int64_t)blockIdx.x * 32 + k;
    if (c || to >= 2 * cols) return;
    if (to < cols) dw[to] = dev::from_f32<DT>(s);
    else db[to - cols] = dev::from_f32<DT>(s);
}

// Longer rows: mean, what it is off by, rstd and, with dy, the means of g and g xh (c2) of
// a row per workgroup.
template <int DT, bool GRAD>
__global__ __launch_bounds__(1024) void long_stats_kernel(const typename Elem<DT>::type* __restrict__ dy,
                                                          const typename Elem<DT>::type* __restrict__ x,
                                                          const typename Elem<DT>::type* __restrict__ w,
                                                          float4* __restrict__ stats, float* __restrict__ c2,
                                                          int64_t rows, int64_t cols, float eps) {
    constexpr int VEC = Elem<DT>::VEC;
    __shared__ float slots[2][4 * 16];
    const float inv = 1.0f / (float)cols;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const typename Elem<DT>::type *xr = x + r * cols, *gr = GRAD ? dy + r * cols : nullptr;
        float s1[1] = {0.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < cols; c += 1024 * VEC) {
            float v[VEC];
            unpack<DT>(load_raw<DT>(xr, c, cols), v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s1[0] += v[e];
        }
        row_sums<16, 1>(s1, slots[0], wave, lane);
        const float mean = s1[0] / (float)cols;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < cols; c += 1024 * VEC) {
            float v[VEC], g[VEC], wf[VEC];
            unpack<DT>(load_raw<DT>(xr, c, cols), v);
            if constexpr (GRAD) {
                unpack<DT>(load_raw<DT>(gr, c, cols), g);
                unpack<DT>(load_raw<DT>(w, c, cols), wf);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = c + e < cols ? v[e] - mean : 0.0f;
                s[0] += d;
                s[1] += d * d;
                if constexpr (GRAD) {
                    s[2] += g[e] * wf[e];
                    s[3] += g[e] * wf[e] * d;
                }
            }
        }
        row_sums<16, 4>(s, slots[1], wave, lane);
        if (threadIdx.x == 0) {
            const float off = s[0] * inv, rstd = inverse_std(s[0], s[1], off, inv, eps);
            stats[r] = make_float4(mean, off, rstd, s[2] * inv);
            if constexpr (GRAD) c2[r] = (s[3] - off * s[2]) * inv * rstd;
        }
    }
}

// Longer rows, one tile of columns of every gridDim.y-th row: y, or dx and the
// tile's sums of dw and db over those rows (part, as affine_bwd_kernel's).
template <int DT, bool GRAD>
__global__ __launch_bounds__(LONG_TILE / Elem<DT>::VEC) void long_apply_kernel(
    const typename Elem<DT>::type* __restrict__ dy, const typename Elem<DT>::type* __restrict__ x,
    const typename Elem<DT>::type* __restrict__ w, const typename Elem<DT>::type* __restrict__ b,
    const float4* __restrict__ stats, const float* __restrict__ c2, typename Elem<DT>::type* __restrict__ out,
    float* __restrict__ part, int64_t rows, int64_t cols) {
    constexpr int VEC = Elem<DT>::VEC;
    const int64_t c = (int64_t)blockIdx.x * LONG_TILE + threadIdx.x * VEC;
    if (c >= cols) return;
    float wf[VEC], bf[VEC], aw[VEC], ab[VEC];
    unpack<DT>(load_raw<DT>(w, c, cols), wf);
    if constexpr (!GRAD) unpack<DT>(load_raw<DT>(b, c, cols), bf);
#pragma unroll
    for (int e = 0; e < VEC; ++e) aw[e] = ab[e] = 0.0f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float4 st = stats[r];
        const float k = GRAD ? c2[r] : 0.0f;
        float v[VEC], g[VEC];
        unpack<DT>(load_raw<DT>(x + r * cols, c, cols), v);
        if constexpr (GRAD) unpack<DT>(load_raw<DT>(dy + r * cols, c, cols), g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float xh = (v[e] - st.x - st.y) * st.z;
            if constexpr (GRAD) {
                aw[e] += g[e] * xh;
                ab[e] += g[e];
                v[e] = st.z * (g[e] * wf[e] - st.w - xh * k);
            } else {
                v[e] = xh * wf[e] + bf[e];
            }
        }
        store_vec<DT>(out + r * cols, c, cols, v);
    }
    if constexpr (GRAD) {
        float* p = part + (int64_t)blockIdx.y * 2 * cols;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c + e < cols) {
                p[c + e] = aw[e];
                p[cols + c + e] = ab[e];
            }
    }
}

template <int DT>
struct Args {
    typedef typename Elem<DT>::type T;
    const T *dy, *x, *w, *b;
    T *out, *dw, *db;
    float* part;
    int64_t rows, cols;
    float eps;
    bool grad;
    hipStream_t s;
};

template <int DT, int WPR, int NV>
int launch_registers(const Args<DT>& a, int64_t groups) {
    const int threads = WPR < 4 ? 256 : 64 * WPR;
    if (a.grad) {
        hipLaunchKernelGGL((affine_bwd_kernel<DT, WPR, NV>), dim3((unsigned)groups), dim3(threads), 0, a.s, a.dy, a.x, a.w,
                           a.out, a.part, a.rows, a.cols, a.eps);
        return launch_check("affine_bwd_kernel");
    }
    hipLaunchKernelGGL((affine_fwd_kernel<DT, WPR, NV>), dim3((unsigned)groups), dim3(threads), 0, a.s, a.x, a.w, a.b,
                       a.out, a.rows, a.cols, a.eps);
    return launch_check("affine_fwd_kernel");
}

template <int DT, int WPR>
int launch_waves(const Args<DT>& a, int64_t groups) {
    const int nv = (int)ceil_div(a.cols, 64 * WPR * Elem<DT>::VEC);
    if constexpr (DT == MLXHIP_DTYPE_F32) {
        if (nv == 4) return launch_registers<DT, WPR, 4>(a, groups);
        if (nv == 3) return launch_registers<DT, WPR, 3>(a, groups);
    }
    if (nv == 2) return launch_registers<DT, WPR, 2>(a, groups);
    // Four times the waves start at four times the columns: one vector is
    // left to f32 rows of a single wave and to 16-bit rows.
    if constexpr (DT != MLXHIP_DTYPE_F32 || WPR == 1) return launch_registers<DT, WPR, 1>(a, groups);
    return fail(MLXHIP_ERR_INVALID_ARGUMENT, "layernorm_affine: no kernel for %lld columns", (long long)a.cols);
}

template <int DT>
int run_affine(Args<DT> a) {
    const bool registers = a.cols <= MAX_COLS;
    const int rpb = a.cols <= 1024 ? 4 : 1;  // rows of a workgroup at a time
    // Forward: eight workgroups to a CU at most, so that each has its weights'
    // load to share between rows when there are many.
    int64_t groups = registers ? std::min<int64_t>(ceil_div(a.rows, rpb), a.grad ? PARTIALS : 2048)
                               : std::min<int64_t>(a.rows, 64);
    const size_t part = a.grad ? (size_t)groups * 2 * a.cols * sizeof(float) : 0;
    const size_t stats = registers ? 0 : (size_t)a.rows * (sizeof(float4) + sizeof(float));  // and c2
    char* ws = nullptr;
    if (part + stats) MLXHIP_TRY(stream_workspace(a.s, WS_NORM, part + stats, reinterpret_cast<void**>(&ws)));
    a.part = reinterpret_cast<float*>(ws + stats);
    if (a.rows == 0) {
        // No rows: the fold below writes the zeros of dw and db.
    } else if (!registers) {
        float4* st = reinterpret_cast<float4*>(ws);
        float* c2 = reinterpret_cast<float*>(st + a.rows);
        const dim3 grid((unsigned)ceil_div(a.cols, LONG_TILE), (unsigned)groups);
        const int threads = LONG_TILE / Elem<DT>::VEC;
        const unsigned blocks = (unsigned)std::min<int64_t>(a.rows, 4096);
        if (a.grad) {
            hipLaunchKernelGGL((long_stats_kernel<DT, true>), dim3(blocks), dim3(1024), 0, a.s, a.dy, a.x, a.w, st, c2,
                               a.rows, a.cols, a.eps);
            MLXHIP_TRY(launch_check("long_stats_kernel"));
            hipLaunchKernelGGL((long_apply_kernel<DT, true>), grid, dim3(threads), 0, a.s, a.dy, a.x, a.w, a.b, st,
                               c2, a.out, a.part, a.rows, a.cols);
        } else {
            hipLaunchKernelGGL((long_stats_kernel<DT, false>), dim3(blocks), dim3(1024), 0, a.s, a.dy, a.x, a.w, st, c2,
                               a.rows, a.cols, a.eps);
            MLXHIP_TRY(launch_check("long_stats_kernel"));
            hipLaunchKernelGGL((long_apply_kernel<DT, false>), grid, dim3(threads), 0, a.s, a.dy, a.x, a.w, a.b, st,
                               c2, a.out, a.part, a.rows, a.cols);
        }
        MLXHIP_TRY(launch_check("long_apply_kernel"));
    } else if (a.cols <= 1024) {
        MLXHIP_TRY((launch_waves<DT, 1>(a, groups)));
    } else if (a.cols <= 4096) {
        MLXHIP_TRY((launch_waves<DT, 4>(a, groups)));
    } else {
        MLXHIP_TRY((launch_waves<DT, 16>(a, groups)));
    }
    if (!a.grad) return MLXHIP_OK;
    hipLaunchKernelGGL((affine_fold_kernel<DT>), dim3((unsigned)ceil_div(2 * a.cols, 32)), dim3(32 * FOLD), 0, a.s, a.part, groups,
                       a.cols, a.dw, a.db);
    return launch_check("affine_fold_kernel");
}

int affine(int dt, const void* dy, const void* x, const void* w, const void* b, void* out, void* dw, void* db,
           int64_t rows, int64_t cols, float eps, bool grad, hipStream_t s) {
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            typedef typename Elem<d.value>::type T;
            rc = run_affine<d.value>({(const T*)dy, (const T*)x, (const T*)w, (const T*)b, (T*)out, (T*)dw, (T*)db, nullptr,
                                      rows, cols, eps, grad, s});
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "layernorm_affine: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

}  // namespace

int layernorm_affine(int dt, const void* x, const void* w, const void* b, void* y, int64_t rows, int64_t cols,
                     float eps, hipStream_t s) {
    return affine(dt, nullptr, x, w, b, y, nullptr, nullptr, rows, cols, eps, false, s);
}

int layernorm_affine_vjp(int dt, const void* dy, const void* x, const void* w, void* dx, void* dw, void* db,
                         int64_t rows, int64_t cols, float eps, hipStream_t s) {
    return affine(dt, dy, x, w, nullptr, dx, dw, db, rows, cols, eps, true, s);
}

}  // namespace mlxhip
