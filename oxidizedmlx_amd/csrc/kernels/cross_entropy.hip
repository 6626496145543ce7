// cross_entropy.hip — softmax cross entropy of the logits x W^T of an output
// projection, and the gradients of x and W, in pieces of the vocabulary: the
// logits are never held.
//
//   z_rv   = sum_k x_rk W_vk
//   lse_r  = log sum_v exp(z_rv)
//   loss_r = lse_r - z_r,t(r)             (0 for a target outside [0, vocab))
//   dS_rv  = dloss_r (exp(z_rv - lse_r) - [v = t(r)])   (0 for such a target)
//   dx = dS W,  dW = dS^T x
//
// Forward: one product whose tiles leave each row's maximum and sum over their
// columns (ce_gemm.hpp), and a launch that joins them. Backward, per piece of
// the vocabulary: the product again, stored as dS in two or three bf16 planes, then
// dW of the piece whole and dx's share added to f32 sums, which a last launch
// rounds. At several hundred rows the matrix cores bound the products.
//
// Measured, forward and backward (products and copies; what bounds each product:
// ce_gemm.hpp): bf16 2048 rows of 1024 over 32000 722 - 785 us, 8192 of 2048 over 50257
// 8.4 - 9.2 ms (1.1 - 1.2 PFLOP/s); f32 2048 of 1024 over 32000 2.15 - 2.3 ms, of which the
// copies of W to planes take 55 us (forward, two planes) and 100 (backward, five).
//
// For dW, x is copied once with zeros in the rows without a target (whatever they
// hold must not reach dW through a product with 0) and its rows rounded up to whole
// 16-byte chunks; W is read in place where its rows are such chunks and their
// type is the product's, else copied piece by piece; the same copies split operands
// into planes.
#include "../common.hpp"
#include "../kernels.hpp"
#include "ce_gemm.hpp"
#include "device_math.hpp"
#include "elem.hpp"

#include <algorithm>
#include <atomic>

namespace mlxhip {
namespace {

using ce::Args;
using ce::counted;
using dev::Elem;

constexpr float LN2 = 0.69314718055994530942f;
// Bytes of a piece's dS, and of a copied piece of W; mlxhip_debug_cross_entropy_pieces
// sets others and counts the pieces.
constexpr int64_t PIECE_BYTES = int64_t(512) << 20;
std::atomic<int64_t> g_piece_bytes{PIECE_BYTES}, g_pieces{0};

// 2^e with the largest magnitude m below it (1/2 of it at least); 15 for an m
// that says nothing, so that the factors made from it are 1.
__device__ inline int exponent(float m) { return m > 0.0f && m < INFINITY ? min(max(ilogbf(m) + 1, -100), 128) : 15; }

__device__ inline float finite_abs(float v) { return __builtin_isfinite(v) ? fabsf(v) : 0.0f; }

// v as P planes of type MT, from column c on, `plane` elements apart. A value that is
// not finite is all in the last plane, which meets the other operand's first one
// only: it reaches the product as itself, with the other's sign. A finite value
// that rounds to infinity is cut off instead.
template <int MT, int P>
__device__ inline void store_planes(float (&v)[8], int64_t c, int64_t plane, uint16_t* dst) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        float h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = dev::to_f32<MT>(dev::from_f32<MT>(v[e]));
            if (p + 1 < P) {
                if (MT == MLXHIP_DTYPE_BF16 && __builtin_isinf(h[e]))
                    h[e] = __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
                if (!__builtin_isfinite(v[e])) h[e] = 0.0f;
            }
        }
        dev::store_vec<MT>(dst + p * plane, c, c + 8, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] -= h[e];
    }
}

// Eight columns from c on of a row as f32.
template <int OT>
__device__ inline void load8(const typename Elem<OT>::type* src, int64_t c, int64_t dim, float (&v)[8]) {
    constexpr int VEC = Elem<OT>::VEC;
#pragma unroll
    for (int k = 0; k < 8 / VEC; ++k) dev::unpack<OT>(dev::load_raw<OT>(src, c + k * VEC, dim), v + k * VEC);
}

// src [rows][dim] of 16-bit values as they are into z [rows][dim_p] and, f16 ones times
// dloss and *scale, as planes into g (either may be null): zeros past dim and, where
// targets are given, in the rows without one. 8 columns a thread.
template <int OT>
__global__ __launch_bounds__(1024) void pack_kernel(const typename Elem<OT>::type* __restrict__ src, int64_t rows,
                                                    int64_t dim, int64_t dim_p, const int32_t* __restrict__ targets,
                                                    int64_t vocab, const float* __restrict__ dloss,
                                                    const float* __restrict__ scale, uint16_t* __restrict__ z,
                                                    uint16_t* __restrict__ g) {
    const int64_t chunks = dim_p / 8;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < rows * chunks; i += (int64_t)gridDim.x * 1024) {
        const int64_t r = i / chunks, c = (i - r * chunks) * 8;
        const dev::u32x4 raw = dev::load_raw<OT>(src + r * dim, c, dim).q, none = {0, 0, 0, 0};
        const bool on = !targets || counted(targets[r], vocab);
        const dev::u32x4 q = on ? raw : none;
        if (z) *reinterpret_cast<dev::u32x4*>(z + r * dim_p + c) = q;
        if (OT == MLXHIP_DTYPE_F16 && g) {
            const float f = on ? dloss[r] * *scale : 0.0f;
            float v[8];
            dev::unpack<OT>(dev::Vec16<OT>{q}, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
            store_planes<OT, ce::X_PLANES<OT>>(v, c, rows * dim_p, g + r * dim_p);
        }
    }
}

// The largest finite |dloss x| of each row with a target (0 for the others), a wave to
// a row; and, by one workgroup, from those the power of two that brings them below
// 2^15 (scale[0]) and what undoes it and dS's own (scale[1]).
template <int OT>
__global__ __launch_bounds__(256) void peak_kernel(const typename Elem<OT>::type* __restrict__ x, int64_t rows, int64_t dim,
                                                   const int32_t* __restrict__ targets, int64_t vocab,
                                                   const float* __restrict__ dloss, float* __restrict__ peak) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        float m = 0.0f;
        if (counted(targets[r], vocab))
            for (int64_t c = lane * 8; c < dim; c += 512) {
                float v[8];
                load8<OT>(x + r * dim, c, dim, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
            }
        m = dev::wave_max(m);
        if (lane == 0) peak[r] = finite_abs(m * dloss[r]);
    }
}
__global__ __launch_bounds__(1024) void scale_kernel(const float* __restrict__ peak, int64_t rows, float* __restrict__ scale) {
    __shared__ float waves[16];
    float m = 0.0f;
#pragma unroll 4
    for (int64_t r = threadIdx.x; r < rows; r += 1024) m = fmaxf(m, peak[r]);
    m = dev::wave_max(m);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 16; ++i) m = fmaxf(m, waves[i]);
    const int e = exponent(m);
    scale[0] = ldexpf(1.0f, 15 - e);
    scale[1] = ldexpf(1.0f / ce::DS_F16, e - 15);
}

// As pack_kernel for f32: z is two f16 planes of the row times a power of two made from
// its own largest magnitude (row_scale: what undoes it), so that no row takes digits
// from another; either of z and g may be null. `lanes` (a power of two) to a row: a wave, fewer for short rows.
__global__ __launch_bounds__(256) void pack_rows_kernel(const float* __restrict__ src, int64_t rows, int64_t dim,
                                                        int64_t dim_p, const int32_t* __restrict__ targets, int64_t vocab,
                                                        int lanes, float* __restrict__ row_scale,
                                                        uint16_t* __restrict__ z, uint16_t* __restrict__ g) {
    constexpr int F32 = MLXHIP_DTYPE_F32;
    const int lane = threadIdx.x % lanes, each = 256 / lanes;
    for (int64_t r = (int64_t)blockIdx.x * each + threadIdx.x / lanes; r < rows; r += (int64_t)gridDim.x * each) {
        const float* p = src + r * dim;
        const bool on = !targets || counted(targets[r], vocab);
        float f = 1.0f;
        if (z) {
            float m = 0.0f;
            for (int64_t c = lane * 8; c < dim; c += lanes * 8) {
                float v[8];
                load8<F32>(p, c, dim, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
            }
            for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            const int e2 = exponent(m);
            if (lane == 0) row_scale[r] = ldexpf(1.0f, e2 - 15);
            f = ldexpf(1.0f, 15 - e2);
        }
        for (int64_t c = lane * 8; c < dim_p; c += lanes * 8) {
            float v[8], u[8];
            load8<F32>(p, c, dim, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = on ? v[e] : 0.0f;
                u[e] = v[e] * f;
            }
            if (z) store_planes<MLXHIP_DTYPE_F16, ce::Z_PLANES<F32>>(u, c, rows * dim_p, z + r * dim_p);
            if (g) store_planes<MLXHIP_DTYPE_BF16, ce::X_PLANES<F32>>(v, c, rows * dim_p, g + r * dim_p);
        }
    }
}

// A row's maxima and sums over the tiles joined: 16 rows of a workgroup, 64
// threads to each (16 rows of a tile are a line of stats).
constexpr int JOIN_ROWS = 16, JOIN = 64;
__global__ __launch_bounds__(JOIN_ROWS * JOIN) void loss_kernel(const float2* __restrict__ stats, int64_t tiles,
                                                                const float* __restrict__ target_z,
                                                                const int32_t* __restrict__ targets, int64_t rows,
                                                                int64_t vocab, float* __restrict__ loss,
                                                                float* __restrict__ lse) {
    __shared__ float2 part[JOIN_ROWS][JOIN + 1];
    const int k = threadIdx.x / JOIN_ROWS, c = threadIdx.x % JOIN_ROWS;
    float m = -INFINITY, s = 0.0f;
    if ((int64_t)blockIdx.x * JOIN_ROWS + c < rows) {
        const float2* p = stats + (int64_t)blockIdx.x * JOIN_ROWS + c;
#pragma unroll 4
        for (int64_t t = k; t < tiles; t += JOIN) {
            const float2 a = p[t * rows];
            ce::merge(m, s, a.x, a.y);
        }
    }
    part[c][k] = make_float2(m, s);
    __syncthreads();
    // A wave to each row.
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * JOIN_ROWS + w;
    if (r >= rows) return;
    m = part[w][lane].x;
    s = part[w][lane].y;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ce::merge(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    if (lane) return;
    const float l = m + LN2 * __builtin_amdgcn_logf(s);
    lse[r] = l;
    loss[r] = counted(targets[r], vocab) ? l - target_z[r] : 0.0f;
}

// dx from the f32 sums of its slices of K (f16 operands: times dloss, where the sums are
// of dS without it), zeros where there is no target: 64
// quads of columns of a workgroup, four threads to each, which add up a quarter
// of the slices each and then those, in order.
template <int OT>
__global__ __launch_bounds__(256) void dx_kernel(const float* __restrict__ sums, int splits, int64_t rows, int64_t dim,
                                                 int64_t ld, const int32_t* __restrict__ targets, int64_t vocab,
                                                 const float* __restrict__ dloss,
                                                 typename Elem<OT>::type* __restrict__ dx) {
    __shared__ float4 part[4][64];
    const int64_t quads = ld / 4, n = rows * quads;
    const int q = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int each = (splits + 3) / 4, k0 = g * each, k1 = min(k0 + each, splits);
    for (int64_t base = (int64_t)blockIdx.x * 64; base < n; base += (int64_t)gridDim.x * 64) {
        const int64_t i = base + q, r = i / quads, c = (i - r * quads) * 4;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const bool on = i < n && counted(targets[r], vocab);
        if (on) {
            const float* p = sums + r * ld + c;
#pragma unroll 4
            for (int k = k0; k < k1; ++k) {
                const float4 v = *reinterpret_cast<const float4*>(p + k * (rows * ld));
                a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
            }
        }
        part[g][q] = a;
        __syncthreads();
        if (g == 0 && i < n) {
#pragma unroll
            for (int k = 1; k < 4; ++k) {
                const float4 v = part[k][q];
                a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
            }
            const float f = on && dloss ? dloss[r] : 1.0f, down = dloss ? 1.0f / ce::DS_F16 : 1.0f;
            const float v[4] = {a.x * down * f, a.y * down * f, a.z * down * f, a.w * down * f};
            typename Elem<OT>::type* to = dx + r * dim + c;
            if (c + 4 <= dim) {
                if constexpr (OT == MLXHIP_DTYPE_F32) {
                    dev::store_vec<OT>(to, 0, 4, v);
                } else {
                    typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(2)));
                    *reinterpret_cast<u32x2*>(to) = {gemm16::pack2<OT>(v[0], v[1]), gemm16::pack2<OT>(v[2], v[3])};
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < dim) to[e] = dev::from_f32<OT>(v[e]);
            }
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void lse_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                  const int32_t* __restrict__ targets, const float* __restrict__ loss,
                                                  float* __restrict__ lse, int64_t rows, int64_t dim, int64_t vocab) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const int32_t t = targets[r];
    float z = 0.0f;
    if (counted(t, vocab))
        for (int64_t c = lane; c < dim; c += 64) z = fmaf(x[r * dim + c], w[t * dim + c], z);
    z = dev::wave_sum(z);
    if (lane == 0) lse[r] = loss[r] + z;
}

template <typename T>
__global__ __launch_bounds__(256) void zero_kernel(T* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = T(0);
}

unsigned grid_for(int64_t threads) { return (unsigned)std::min<int64_t>(ceil_div(threads, 256), 8192); }

// Sub-blocks of one workspace.
struct Carve {
    size_t used = 0;
    size_t take(size_t bytes) {
        const size_t at = used;
        used += (bytes + 255) / 256 * 256;
        return at;
    }
};

template <int OT>
struct Op {
    typedef typename Elem<OT>::type T;
    static constexpr int ZP = ce::Z_PLANES<OT>, SP = ce::DS_PLANES<OT>, XP = ce::X_PLANES<OT>, WP = ce::W_PLANES<OT>;
    using ZTiles = ce::Tiling<ZP, ZP>;   // of the logits
    using DXTiles = ce::Tiling<SP, WP>;
    using DWTiles = ce::Tiling<SP, XP>;
    const T *x, *w;
    const int32_t* targets;
    int64_t rows, dim, vocab;
    hipStream_t s;
    int64_t dim_p() const { return ceil_div(dim, 8) * 8; }
    // Whether the logits' product reads a matrix of rows of dim as it is.
    bool in_place(const T* p) const { return ZP == 1 && dim % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }
    // Bytes of n rows' planes.
    size_t bytes(int64_t n, int planes) const { return (size_t)n * dim_p() * planes * 2; }
    // n rows of src into z and g where not null; scale: f32 rows' factors, or of f16
    // operands' dloss x.
    int pack(const T* src, int64_t n, const int32_t* t, const float* dloss, float* scale, uint16_t* z, uint16_t* g) const {
        if constexpr (OT == MLXHIP_DTYPE_F32) {
            int lanes = 1;
            while (lanes < 64 && lanes * 8 < dim) lanes *= 2;
            const int64_t groups = std::min<int64_t>(ceil_div(n, 256 / lanes), 16384);
            hipLaunchKernelGGL(pack_rows_kernel, dim3((unsigned)groups), dim3(256), 0, s, src, n, dim, dim_p(), t, vocab, lanes,
                               scale, z, g);
        } else {
            const int64_t groups = std::min<int64_t>(ceil_div(n * dim_p() / 8, 1024), 2048);
            hipLaunchKernelGGL((pack_kernel<OT>), dim3((unsigned)groups), dim3(1024), 0, s, src, n, dim, dim_p(), t, vocab,
                               dloss, scale, z, g);
        }
        return launch_check("pack_kernel");
    }
    // The scales of f16 operands' dloss x (peak: room for a value a row).
    int scales(const float* dloss, float* peak, float* scale) const {
        const int64_t groups = std::min<int64_t>(ceil_div(rows, 4), 16384);
        hipLaunchKernelGGL((peak_kernel<OT>), dim3((unsigned)groups), dim3(256), 0, s, x, rows, dim, targets, vocab, dloss,
                           peak);
        MLXHIP_TRY(launch_check("peak_kernel"));
        hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(1024), 0, s, peak, rows, scale);
        return launch_check("scale_kernel");
    }
    int product(int which, bool large, const Args& a) const {
        if (OT == MLXHIP_DTYPE_F32) return ce_gemm_f32(which, large, a, s);
        return OT == MLXHIP_DTYPE_BF16 ? ce_gemm_bf16(which, large, a, s) : ce_gemm_f16(which, large, a, s);
    }
    template <class Tiles>
    static int64_t tiles(int64_t m, int64_t n, bool large) {
        typedef typename Tiles::Large L;
        typedef typename Tiles::Small S;
        return large ? ceil_div(m, L::BM) * ceil_div(n, L::BN) : ceil_div(m, S::BM) * ceil_div(n, S::BN);
    }
    // Large tiles where they fill most of the compute units, one each.
    template <class Tiles>
    static bool large(int64_t m, int64_t n) { return tiles<Tiles>(m, n, true) >= 192; }
    // Columns of a piece: with `ds`, dS, and `copied` planes of a copied piece of W within
    // the piece's bytes, offsets within a piece and the count of its tiles within 32 bits.
    int64_t width(bool ds, int copied) const {
        const int64_t bytes = g_piece_bytes.load();
        int64_t w = std::min<int64_t>(vocab, (int64_t(1) << 29) / dim_p());
        w = std::min(w, (int64_t(1) << 43) / rows);
        if (ds) w = std::min(w, bytes / (2 * SP) / rows);
        if (copied) w = std::min(w, bytes / (2 * copied) / dim_p());
        if (w >= vocab) return vocab;
        w = std::max<int64_t>(w / 256 * 256, 256);
        // Pieces of like width: a short last one leaves compute units idle (1105 of
        // 50257 columns: 160 us of small tiles, 60 in proportion).
        return ceil_div(ceil_div(vocab, ceil_div(vocab, w)), 256) * 256;
    }
};

int finish_loss(const float2* stats, int64_t tiles, const float* target_z, const int32_t* targets, int64_t rows,
                int64_t vocab, float* loss, float* lse, hipStream_t s) {
    hipLaunchKernelGGL(loss_kernel, dim3((unsigned)ceil_div(rows, JOIN_ROWS)), dim3(JOIN_ROWS * JOIN), 0, s, stats, tiles,
                       target_z, targets, rows, vocab, loss, lse);
    return launch_check("loss_kernel");
}

// Few rows: W as it is in each product (measured in ce_few.hip).
template <int OT>
ce::FewArgs few_args(const Op<OT>& o) {
    ce::FewArgs g;
    g.x = o.x;
    g.w = o.w;
    g.rows = o.rows;
    g.dim = o.dim;
    g.vocab = o.vocab;
    g.targets = o.targets;
    return g;
}

template <int OT>
int few_loss(const Op<OT>& o, float* loss, float* lse) {
    ce::FewArgs g = few_args(o);
    const int64_t tiles = ce_few_tiles(OT, o.rows, o.vocab);
    Carve c;
    const size_t os = c.take((size_t)tiles * o.rows * sizeof(float2)), oz = c.take((size_t)o.rows * 4);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(o.s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    g.stats = (float2*)(ws + os);
    g.target_z = (float*)(ws + oz);
    MLXHIP_TRY(ce_few_loss(OT, g, o.s));
    return finish_loss(g.stats, tiles, g.target_z, o.targets, o.rows, o.vocab, loss, lse, o.s);
}

template <int OT>
int few_grad(const Op<OT>& o, const float* lse, const float* loss, const float* dloss, typename Elem<OT>::type* dx,
             typename Elem<OT>::type* dw) {
    ce::FewArgs g = few_args(o);
    g.lse = lse;
    g.loss = loss;
    g.dloss = dloss;
    g.dw = dw;
    const bool tiles_z = !ce::few_loss(OT, !o.in_place(o.w), o.rows, o.vocab), copy_x = tiles_z && !o.in_place(o.x);
    // Eight waves to a compute unit, four of a workgroup along the vocabulary.
    g.ldx = ceil_div(o.dim, 4) * 4;
    const int64_t most = std::max<int64_t>(512 / ceil_div(o.dim, 16 * Elem<OT>::VEC), 1);
    g.slice = ceil_div(ceil_div(o.vocab, 4 * most), 16) * 16;
    g.slices = ceil_div(o.vocab, 4 * g.slice);
    Carve c;
    const size_t od = c.take((size_t)o.vocab * ce::few_ds_rows(o.rows) * 4),
                 ox = c.take(dx ? (size_t)g.slices * o.rows * g.ldx * 4 : 0), oxz = c.take(copy_x ? o.bytes(o.rows, 1) : 0);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(o.s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    g.ds = (float*)(ws + od);
    g.dx = dx ? (float*)(ws + ox) : nullptr;
    if (tiles_z) {
        // The loss took z from the tiles.
        g.form_ds = false;
        uint16_t* xz = copy_x ? (uint16_t*)(ws + oxz) : nullptr;
        if (copy_x) MLXHIP_TRY(o.pack(o.x, o.rows, nullptr, nullptr, nullptr, xz, nullptr));
        const int64_t width = o.width(false, 0);
        for (int64_t v0 = 0; v0 < o.vocab; v0 += width) {
            Args z;
            z.a = xz ? xz : (const uint16_t*)o.x;
            z.b = (const uint16_t*)o.w + v0 * o.dim;
            z.lda = z.ldb = z.ka = z.kb = o.dim_p();
            z.m = o.rows;
            z.n = std::min(width, o.vocab - v0);
            z.targets = o.targets;
            z.v0 = v0;
            z.vocab = o.vocab;
            z.lse = lse;
            z.dloss = dloss;
            z.dst = g.ds + v0 * 16;
            MLXHIP_TRY(o.product(ce::CE_DST, Op<OT>::template large<typename Op<OT>::ZTiles>(o.rows, z.n), z));
        }
    }
    MLXHIP_TRY(ce_few_grad(OT, g, o.s));
    if (!dx) return MLXHIP_OK;
    hipLaunchKernelGGL((dx_kernel<OT>), dim3(grid_for(o.rows * g.ldx)), dim3(256), 0, o.s, g.dx,
                       (int)g.slices, o.rows, o.dim, g.ldx, o.targets, o.vocab, nullptr, dx);
    return launch_check("dx_kernel");
}

template <int OT>
int run_loss(const Op<OT>& o, float* loss, float* lse) {
    typedef Op<OT> O;
    const bool copy_x = !o.in_place(o.x), copy_w = !o.in_place(o.w);
    if (ce::few_loss(OT, copy_w, o.rows, o.vocab)) return few_loss(o, loss, lse);
    const int64_t width = o.width(false, copy_w ? O::ZP : 0);
    // One tile size for all pieces, whose widths are multiples of its columns.
    const bool large = O::template large<typename O::ZTiles>(o.rows, o.vocab);
    const int64_t bn = large ? O::ZTiles::Large::BN : O::ZTiles::Small::BN, tiles = ceil_div(o.vocab, bn);
    Carve c;
    const size_t os = c.take((size_t)tiles * o.rows * sizeof(float2)), oz = c.take((size_t)o.rows * 4),
                 ox = c.take(copy_x ? o.bytes(o.rows, O::ZP) : 0), ow = c.take(copy_w ? o.bytes(width, O::ZP) : 0),
                 orow = c.take(O::ZP > 1 ? (size_t)o.rows * 4 : 0),
                 ocol = c.take(O::ZP > 1 ? (size_t)ceil_div(width, 256) * 256 * 4 : 0);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(o.s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    Args a;
    a.a = copy_x ? (uint16_t*)(ws + ox) : (const uint16_t*)o.x;
    a.lda = a.ldb = a.ka = a.kb = o.dim_p();
    a.a_plane = o.rows * o.dim_p();
    a.m = o.rows;
    a.targets = o.targets;
    a.vocab = o.vocab;
    a.target_z = (float*)(ws + oz);
    a.row_scale = (float*)(ws + orow);
    a.col_scale = (float*)(ws + ocol);
    if (copy_x) MLXHIP_TRY(o.pack(o.x, o.rows, nullptr, nullptr, (float*)(ws + orow), (uint16_t*)(ws + ox), nullptr));
    for (int64_t v0 = 0; v0 < o.vocab; v0 += width) {
        g_pieces.fetch_add(1);
        a.n = std::min(width, o.vocab - v0);
        a.b = copy_w ? (uint16_t*)(ws + ow) : (const uint16_t*)o.w + v0 * o.dim;
        a.b_plane = a.n * o.dim_p();
        a.v0 = v0;
        a.stats = (float2*)(ws + os) + v0 / bn * o.rows;
        if (copy_w)
            MLXHIP_TRY(o.pack(o.w + v0 * o.dim, a.n, nullptr, nullptr, (float*)(ws + ocol), (uint16_t*)(ws + ow), nullptr));
        MLXHIP_TRY(o.product(ce::CE_STATS, large, a));
    }
    return finish_loss((const float2*)(ws + os), tiles, a.target_z, o.targets, o.rows, o.vocab, loss, lse, o.s);
}

template <int OT>
int run_grad(const Op<OT>& o, const float* lse, const float* loss, const float* dloss, typename Elem<OT>::type* dx,
             typename Elem<OT>::type* dw) {
    typedef typename Elem<OT>::type T;
    typedef Op<OT> O;
    typedef typename O::DXTiles DX;
    constexpr int ZP = O::ZP, SP = O::SP, XP = O::XP, WP = O::WP;
    constexpr bool F16 = OT == MLXHIP_DTYPE_F16;
    if (o.rows == 0) {  // a sum over no rows
        if (!dw) return MLXHIP_OK;
        hipLaunchKernelGGL((zero_kernel<T>), dim3(grid_for(o.vocab * o.dim)), dim3(256), 0, o.s, dw, o.vocab * o.dim);
        return launch_check("zero_kernel");
    }
    if (ce::few_grad(OT, o.rows, o.vocab)) return few_grad(o, lse, loss, dloss, dx, dw);
    // One plane of x or W serves z and the gradient, but x's then has to be a copy.
    // Rows whose loss ce_few.hip forms take z from there.
    const bool few_z = ce::few_loss(OT, !o.in_place(o.w), o.rows, o.vocab);
    const bool copy_x = XP == 1 ? !few_z || dw : !few_z && !o.in_place(o.x), planes_x = XP > 1 && dw,
               copy_w = !o.in_place(o.w) && (!few_z || (WP == 1 && dx)),
               planes_w = WP > 1 && dx;
    const int64_t width = o.width(true, (copy_w ? ZP : 0) + (planes_w ? WP : 0)), ld = ceil_div(width, 256) * 256,
                  dim_p = o.dim_p();
    // dx: few tiles, so K is cut into slices until every place on the chip has one,
    // of at least 512 each.
    const bool dx_large = O::template tiles<DX>(o.rows, o.dim, true) >= 16;
    const int64_t dx_tiles = O::template tiles<DX>(o.rows, o.dim, dx_large);
    const int64_t room = 256 * (dx_large ? DX::Large::PER_CU : DX::Small::PER_CU);
    const int64_t most = std::max<int64_t>(1, std::min(room / dx_tiles, width / 512));
    const int64_t chunk = ceil_div(ceil_div(width, most), 32) * 32;
    const int splits = (int)ceil_div(width, chunk);
    const int64_t ldx = ceil_div(o.dim, 4) * 4;
    Carve c;
    const size_t ods = c.take((size_t)SP * o.rows * ld * 2), ox = c.take(copy_x ? o.bytes(o.rows, ZP) : 0),
                 oxg = c.take(planes_x ? o.bytes(o.rows, XP) : 0), ow = c.take(copy_w ? o.bytes(width, ZP) : 0),
                 owg = c.take(planes_w ? o.bytes(width, WP) : 0), orow = c.take(ZP > 1 || F16 ? (size_t)o.rows * 4 : 0),
                 osc = c.take(F16 ? 2 * 4 : 0), ocol = c.take(ZP > 1 ? (size_t)ld * 4 : 0), osum = c.take(dx ? (size_t)splits * o.rows * ldx * 4 : 0);
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(o.s, WS_CE, c.used, reinterpret_cast<void**>(&ws)));
    uint16_t *ds = (uint16_t*)(ws + ods), *xz = copy_x ? (uint16_t*)(ws + ox) : nullptr,
             *xg = planes_x ? (uint16_t*)(ws + oxg) : nullptr, *wz = copy_w ? (uint16_t*)(ws + ow) : nullptr,
             *wg = planes_w ? (uint16_t*)(ws + owg) : nullptr;
    float *sums = (float*)(ws + osum), *row_scale = (float*)(ws + orow), *col_scale = (float*)(ws + ocol);
    float* scale = F16 ? (float*)(ws + osc) : row_scale;
    if constexpr (F16)
        if (dw) MLXHIP_TRY(o.scales(dloss, row_scale, scale));
    if (xz || xg) MLXHIP_TRY(o.pack(o.x, o.rows, o.targets, dloss, scale, xz, xg));
    for (int64_t v0 = 0; v0 < o.vocab; v0 += width) {
        g_pieces.fetch_add(1);
        const int64_t n = std::min(width, o.vocab - v0);
        if (wz || wg) MLXHIP_TRY(o.pack(o.w + v0 * o.dim, n, nullptr, nullptr, col_scale, wz, wg));
        Args z;
        z.a = xz ? xz : (const uint16_t*)o.x;
        z.b = wz ? wz : (const uint16_t*)o.w + v0 * o.dim;
        z.lda = z.ldb = z.ka = z.kb = dim_p;
        z.a_plane = o.rows * dim_p;
        z.b_plane = n * dim_p;
        z.m = o.rows;
        z.n = n;
        z.targets = o.targets;
        z.v0 = v0;
        z.vocab = o.vocab;
        z.lse = lse;
        z.loss = loss;
        z.dloss = dloss;
        z.row_scale = row_scale;
        z.col_scale = col_scale;
        z.ds = ds;
        z.ldc = ceil_div(n, 256) * 256;
        if (few_z) {
            ce::FewArgs f = few_args(o);
            f.w = o.w + v0 * o.dim;
            f.vocab = n;
            f.first = v0;
            f.whole = o.vocab;
            f.lse = lse;
            f.loss = loss;
            f.dloss = dloss;
            f.planes = ds;
            f.ldc = z.ldc;
            f.plane = o.rows * z.ldc;
            MLXHIP_TRY(ce_few_planes(OT, f, o.s));
        } else {
            MLXHIP_TRY(o.product(ce::CE_DS, O::template large<typename O::ZTiles>(o.rows, n), z));
        }
        if (dw) {
            Args p;
            p.a = ds;
            p.lda = z.ldc;
            p.a_plane = o.rows * z.ldc;
            p.b = XP > 1 ? xg : xz;
            p.ldb = dim_p;
            p.b_plane = z.a_plane;
            p.ka = p.kb = o.rows;
            p.m = n;
            p.n = o.dim;
            p.dw = dw + v0 * o.dim;
            p.ldc = o.dim;
            p.scale = scale + 1;
            MLXHIP_TRY(o.product(ce::CE_DW, O::template large<typename O::DWTiles>(n, o.dim), p));
        }
        if (dx) {
            Args p;
            p.a = ds;
            p.lda = z.ldc;
            p.a_plane = o.rows * z.ldc;
            p.ka = ceil_div(n, 8) * 8;  // dS holds zeros behind the piece
            p.b = WP > 1 ? wg : z.b;
            p.ldb = dim_p;
            p.b_plane = z.b_plane;
            p.kb = n;
            p.m = o.rows;
            p.n = o.dim;
            // A last piece may have fewer slices; the others keep their sums.
            p.splits = (int)std::min<int64_t>(splits, ceil_div(p.ka, chunk));
            p.k_chunk = chunk;
            p.dx = sums;
            p.ldc = ldx;
            p.add = v0 > 0;
            MLXHIP_TRY(o.product(ce::CE_DX, dx_large, p));
        }
    }
    if (!dx) return MLXHIP_OK;
    hipLaunchKernelGGL((dx_kernel<OT>), dim3(grid_for(o.rows * ldx)), dim3(256), 0, o.s, sums, splits, o.rows, o.dim, ldx,
                       o.targets, o.vocab, F16 ? dloss : nullptr, dx);
    return launch_check("dx_kernel");
}

}  // namespace

int linear_cross_entropy(int dt, const void* x, const void* w, const int32_t* targets, float* loss, float* lse,
                         int64_t rows, int64_t dim, int64_t vocab, hipStream_t s) {
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            typedef typename Elem<d.value>::type T;
            rc = run_loss<d.value>({(const T*)x, (const T*)w, targets, rows, dim, vocab, s}, loss, lse);
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

int64_t linear_cross_entropy_pieces(int64_t piece_bytes) {
    g_piece_bytes.store(piece_bytes > 0 ? piece_bytes : PIECE_BYTES);
    return g_pieces.exchange(0);
}

int linear_cross_entropy_lse(const float* x, const float* w, const int32_t* targets, const float* loss, float* lse,
                             int64_t rows, int64_t dim, int64_t vocab, hipStream_t s) {
    if (rows == 0) return MLXHIP_OK;
    hipLaunchKernelGGL(lse_kernel, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, s, x, w, targets, loss, lse, rows, dim,
                       vocab);
    return launch_check("lse_kernel");
}

int linear_cross_entropy_vjp(int dt, const void* x, const void* w, const int32_t* targets, const float* lse,
                             const float* loss, const float* dloss, void* dx, void* dw, int64_t rows, int64_t dim, int64_t vocab,
                             hipStream_t s) {
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            typedef typename Elem<d.value>::type T;
            rc = run_grad<d.value>({(const T*)x, (const T*)w, targets, rows, dim, vocab, s}, lse, loss, dloss, (T*)dx,
                                   (T*)dw);
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy gradient: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

}  // namespace mlxhip
