// ce_few.hip — the linear cross entropy of a few rows (the loss of up to 128 f32
// rows, or 64 of 16 bits where W's rows are no whole 16-byte chunks; the gradients
// of up to 64 f32 rows, or 16 of 16 bits), which reading W (and writing dW) bounds:
// W goes from memory straight into the matrix instructions (f32 ones but for the
// logits of 16-bit operands), with no copies and no planes; dS stays f32.
//
//   stats: z = x W^T, a wave per 16 or 32 entries of the vocabulary; the row maxima
//          and sums of a workgroup's entries, and the targets' logits.
//   ds:    z again, kept as dS^T [vocab][16 NB] (zeros behind the rows); planes: as
//          CE_DS of ce_gemm.hpp leaves it, for rows whose loss is formed here and whose
//          gradients are not.
//   grad:  a wave per 16 VEC columns (VEC values in 16 bytes) and slice of the
//          vocabulary: dW = dS^T x of 16 entries at a time, and its sums of
//          dx = dS W.
//
// v_mfma_f32_16x16x4_f32: lane l gives row (column) l % 16 of A (B) at k = l / 16
// and holds rows 4 (l / 16) + i of column l % 16 of the result. A lane loads VEC
// consecutive values and gives them to VEC instructions: along K that is a
// permutation of the sum, along the columns of W and x one of the columns, which
// the stores undo.
//
// Measured over 32000 entries of 1024, f32: 8 rows 29 us (stats, 4.6 TB/s), 29 (ds),
// 49 (grad, 5.3 TB/s read and written); 32 rows 42, 38, 69; 64 rows 54 (loss), 159 (gradients).
// On planes (ce_gemm.hpp), whose copies read W twice and write it two and five times,
// the loss of 129 to 256 rows takes 104 - 112 us (128 here: 92; over 50257 of 2044: 350
// and 279) and the gradients of 65 rows 255 (of 2044 over 50257: 900, 64 rows here 540).
// bf16: 8 rows 73 us with the loss, 17 on the tiles 78 (2044 columns over 50257: 279
// for 16, 369 for 17). The loss where the tiles read W in place: 15 us a call there, 21
// here (8 rows of 768 over 32000); where they would copy it (2044 columns over 50257):
// 44 - 83 here, 144 there for 65 rows.
#include "../common.hpp"
#include "../kernels.hpp"
#include "ce_gemm.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace ce {
namespace {

using dev::Elem;

__device__ inline f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// The eight values of a lane at once (k = 8 (l / 16) + 0..7): 16-bit products.
template <int DT>
__device__ inline f32x4 mfma32(const dev::u32x4& a, const dev::u32x4& b, f32x4 c) {
    if constexpr (DT == MLXHIP_DTYPE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gemm16::bf16x8, a),
                                                       __builtin_bit_cast(gemm16::bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gemm16::f16x8, a),
                                                      __builtin_bit_cast(gemm16::f16x8, b), c, 0, 0, 0);
}

// Tiles of 16 entries of a wave: with more rows two, so that a load of x serves
// twice (64 rows of 1024 over 32000: 82 us with one).
template <int NB>
constexpr int TILES = NB == 1 ? 1 : 2;
template <int NB>
constexpr int ENTRIES = 64 * TILES<NB>;  // of a workgroup

// Rows whose elements may begin in the middle of a dword (16-bit types, ODD): the
// 16 bytes from the dword that a vector begins in and the dword behind them (of
// one that begins with its dword: the fourth again, unused), moved together as
// they are used: every dword read holds an element of the row. Loads at such
// addresses take several times as long: 8 rows of 2047 over 50257 took 171 us with them.
template <bool ODD>
struct Loaded {
    dev::u32x4 q;
    uint32_t next[ODD ? 1 : 0];
};
template <int DT, bool ODD>
struct Row {
    typedef typename Elem<DT>::type E;
    const E* p;
    uint32_t shift = 0;  // bits
    __device__ void set(const E* row) {
        p = row;
        if constexpr (ODD) {
            shift = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 2) * 8;
            p -= shift / 16;
        }
    }
    __device__ Loaded<ODD> load(int64_t k) const {
        Loaded<ODD> v;
        if constexpr (ODD) {
            v.q = dev::load16<MLXHIP_DTYPE_F32>(reinterpret_cast<const float*>(p + k));
            v.next[0] = *reinterpret_cast<const uint32_t*>(p + k + 6 + shift / 8);
        } else {
            v.q = dev::load16<DT>(p + k);
        }
        return v;
    }
    __device__ dev::u32x4 join(const Loaded<ODD>& v) const {
        if constexpr (!ODD) return v.q;
        else
            return dev::u32x4{__builtin_amdgcn_alignbit(v.q[1], v.q[0], shift), __builtin_amdgcn_alignbit(v.q[2], v.q[1], shift),
                              __builtin_amdgcn_alignbit(v.q[3], v.q[2], shift),
                              __builtin_amdgcn_alignbit(v.next[0], v.q[3], shift)};
    }
    __device__ dev::u32x4 load_end(int64_t k, int64_t n) const { return dev::load_raw<DT>(p + shift / 16, k, n).q; }
};

template <int T, int NB>
__device__ inline void zero(f32x4 (&a)[T][NB]) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b) a[t][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}
template <int T, int NB>
__device__ inline void add(f32x4 (&to)[T][NB], const f32x4 (&a)[T][NB]) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b) to[t][b] += a[t][b];
}

// z[v][r] of the wave's TILES * 16 entries from v0 on and NB tiles of 16 rows. KB
// blocks along K are loaded at once.
template <int DT, int NB, bool ODD>
__device__ inline void few_logits(const FewArgs& g, int64_t v0, int lane, f32x4 (&acc)[TILES<NB>][NB]) {
    constexpr int KB = NB == 1 ? 6 : NB == 2 ? 4 : 3, T = TILES<NB>, VEC = Elem<DT>::VEC, BLOCK = 4 * VEC;
    typedef typename Elem<DT>::type E;
    const int i = lane & 15, q = lane >> 4;
    Row<DT, ODD> w[T], x[NB];
#pragma unroll
    for (int t = 0; t < T; ++t) w[t].set(static_cast<const E*>(g.w) + min(v0 + 16 * t + i, g.vocab - 1) * g.dim);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        x[b].set(static_cast<const E*>(g.x) + min((int64_t)(16 * b + i), g.rows - 1) * g.dim);
    }
    zero(acc);
    auto step = [&](const dev::u32x4 (&a)[T], const dev::u32x4 (&c)[NB], f32x4 (&to)[T][NB]) {
        if constexpr (DT == MLXHIP_DTYPE_F32) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int t = 0; t < T; ++t)
                        to[t][b] = mfma4(__uint_as_float(a[t][e]), __uint_as_float(c[b][e]), to[t][b]);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int t = 0; t < T; ++t) to[t][b] = mfma32<DT>(a[t], c[b], to[t][b]);
        }
    };
    // Two batches of loads in turn: one on its way while the other is used.
    struct Batch {
        Loaded<ODD> a[KB][T], c[KB][NB];
    } batch[2];
    auto fetch = [&](int64_t n, int steps, Batch& to) {
        const int64_t k = n * BLOCK * KB + VEC * q;
#pragma unroll
        for (int s = 0; s < KB; ++s) {
            if (s >= steps) break;
#pragma unroll
            for (int t = 0; t < T; ++t) to.a[s][t] = w[t].load(k + BLOCK * s);
#pragma unroll
            for (int b = 0; b < NB; ++b) to.c[s][b] = x[b].load(k + BLOCK * s);
        }
    };
    // f32 products are summed batch by batch: four to an instruction, one chain of 2000
    // columns is 500 roundings long and three times as far off as sums of its pieces.
    constexpr bool PIECES = DT == MLXHIP_DTYPE_F32;
    auto use = [&](const Batch& from, int steps) {
        f32x4 part[T][NB];
        zero(part);
#pragma unroll
        for (int s = 0; s < KB; ++s) {
            if (s >= steps) break;
            dev::u32x4 a[T], c[NB];
#pragma unroll
            for (int t = 0; t < T; ++t) a[t] = w[t].join(from.a[s][t]);
#pragma unroll
            for (int b = 0; b < NB; ++b) c[b] = x[b].join(from.c[s][b]);
            if constexpr (PIECES) step(a, c, part);
            else step(a, c, acc);
        }
        if constexpr (PIECES) add(acc, part);
    };
    const int64_t batches = g.dim / (BLOCK * KB);
    if (batches) fetch(0, KB, batch[0]);
    for (int64_t n = 0; n < batches; n += 2) {
        if (n + 1 < batches) fetch(n + 1, KB, batch[1]);
        __builtin_amdgcn_sched_barrier(0);
        use(batch[0], KB);
        if (n + 1 == batches) break;
        if (n + 2 < batches) fetch(n + 2, KB, batch[0]);
        __builtin_amdgcn_sched_barrier(0);
        use(batch[1], KB);
    }
    // The whole blocks that are left, and a last one that is not.
    const int left = (int)(g.dim / BLOCK - batches * KB);
    const int64_t end = g.dim / BLOCK * BLOCK;
    fetch(batches, left, batch[0]);
    dev::u32x4 a[T], c[NB];
    if (end < g.dim) {
#pragma unroll
        for (int t = 0; t < T; ++t) a[t] = w[t].load_end(end + VEC * q, g.dim);
#pragma unroll
        for (int b = 0; b < NB; ++b) c[b] = x[b].load_end(end + VEC * q, g.dim);
    }
    use(batch[0], left);
    if (end < g.dim) step(a, c, acc);
}

// The maxima and sums of z over the T tiles of 16 entries from v0 on of each of the
// workgroup's waves, for NB tiles of 16 rows from r0 on, as entry `tile` of stats.
template <int T, int NB>
__device__ inline void leave_stats(const FewArgs& g, int64_t v0, int64_t r0, int64_t tile, const f32x4 (&acc)[T][NB]) {
    __shared__ float red[4][2][16 * NB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = r0 + 16 * b + i;
        float m = -INFINITY, s = 0.0f;
        if (v0 < g.vocab) {
            const int64_t target = r < g.rows ? g.targets[r] : -1;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t v = v0 + 16 * t + 4 * q + e;
                    if (v < g.vocab && v == target) g.target_z[r] = acc[t][b][e];
                    // fmaxf drops a NaN; the sum below keeps it.
                    if (v < g.vocab) m = fmaxf(m, acc[t][b][e]);
                }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v0 + 16 * t + 4 * q + e < g.vocab) s += __builtin_amdgcn_exp2f((acc[t][b][e] - base) * LOG2E);
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
    if (r >= 16 * NB || r0 + r >= g.rows) return;
    float m = red[0][0][r], s = red[0][1][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) merge(m, s, red[w][0][r], red[w][1][r]);
    g.stats[tile * g.rows + r0 + r] = make_float2(m, s);
}

// p less 1 at the target, there from the loss where that is known (hit).
__device__ inline float p_of(float z, float lse, bool target, bool known, float hit) {
    const float p = __builtin_amdgcn_exp2f((z - lse) * LOG2E);
    return !target ? p : known ? hit : p - 1.0f;
}

// dS^T of the same from z.
template <int T, int NB>
__device__ inline void leave_ds(const FewArgs& g, int64_t v0, const f32x4 (&acc)[T][NB]) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = 16 * b + i;
        const int64_t target = r < g.rows ? g.targets[r] : -1;
        const bool on = target >= 0 && target < g.vocab;
        const float lse = on ? g.lse[r] : 0.0f, f = on ? g.dloss[r] : 0.0f;
        const float hit = on && g.loss ? expm1f(-g.loss[r]) : 0.0f;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t v = v0 + 16 * t + 4 * q + e;
                const float p = p_of(acc[t][b][e], lse, v == target, g.loss, hit);
                if (v < g.vocab) g.ds[v * (16 * NB) + r] = on ? p * f : 0.0f;
            }
    }
}

// dS of the same from z, for NB tiles of 16 rows from r0 on, as CE_DS leaves it; zeros
// behind the entries up to a multiple of 8.
template <int DT, int T, int NB>
__device__ inline void leave_planes(const FewArgs& g, int64_t v0, int64_t r0, const f32x4 (&acc)[T][NB]) {
    constexpr int GT = G_TYPE<DT>, SP = DS_PLANES<DT>;
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = r0 + 16 * b + i;
        if (r >= g.rows) continue;
        const int64_t target = g.targets[r];
        const bool on = target >= 0 && target < g.whole;
        const float hit = on && g.loss ? expm1f(-g.loss[r]) : 0.0f;
        const float lse = on ? g.lse[r] : 0.0f, f = !on ? 0.0f : DT == MLXHIP_DTYPE_F16 ? DS_F16 : g.dloss[r];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int64_t v = v0 + 16 * t + 4 * q;
            if (v >= (g.vocab + 7) / 8 * 8) continue;
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = p_of(acc[t][b][e], lse, g.first + v + e == target, g.loss, hit);
                d[e] = on && v + e < g.vocab ? p * f : 0.0f;
            }
#pragma unroll
            for (int p = 0; p < SP; ++p) {
                *reinterpret_cast<u32x2*>(g.planes + p * g.plane + r * g.ldc + v) =
                    u32x2{gemm16::pack2<GT>(d[0], d[1]), gemm16::pack2<GT>(d[2], d[3])};
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] -= dev::to_f32<GT>(dev::from_f32<GT>(d[e]));
            }
        }
    }
}

template <int DT, int NB, bool ODD>
__global__ __launch_bounds__(256) void few_stats_kernel(FewArgs g) {
    constexpr int T = TILES<NB>;
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 * T;
    f32x4 acc[T][NB];
    if (v0 < g.vocab) few_logits<DT, NB, ODD>(g, v0, threadIdx.x & 63, acc);
    leave_stats<T, NB>(g, v0, 0, blockIdx.x, acc);
}

// f32 rows by 64: x goes through LDS, KC columns at a time, and serves a
// workgroup's four waves of 16 T entries each; W comes straight from memory, a
// chunk ahead. 128 rows of 1024 over 32000: 82 us, 102 TFLOP/s of f32, and 270 for
// 2044 over 50257 (whole calls 92 and 279; 129 rows on planes 104 and 350; a large f32
// product reaches 154 TFLOP/s). 32 entries a wave, 32 columns a chunk, or two or five waves
// to a SIMD: 1 - 15 % slower; 128 rows a workgroup: 64 rows take 97 instead of 57.
constexpr int WIDE_ROWS = 64, WIDE_T = 1, WIDE_ENTRIES = 64 * WIDE_T;
enum Wide { WIDE_STATS, WIDE_DS, WIDE_PLANES };
template <int OUT>
__global__ __launch_bounds__(256, 4) void wide_kernel(FewArgs g, int64_t row_blocks, int64_t tiles) {
    constexpr int NB = WIDE_ROWS / 16, T = WIDE_T, KC = 64, S = KC / 16, PIECES = WIDE_ROWS * KC / 4 / 256;
    constexpr int DT = MLXHIP_DTYPE_F32;
    __shared__ __attribute__((aligned(16))) float xs[2][WIDE_ROWS][KC + 4];  // 16 rows' quads in different banks
    // The row blocks of a tile of entries follow each other on one XCD (every
    // eighth workgroup), whose cache then holds the tile's part of W.
    const int64_t xcd = blockIdx.x % 8, at = blockIdx.x / 8, tile = at / row_blocks * 8 + xcd, r0 = at % row_blocks * WIDE_ROWS;
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int64_t v0 = (tile * 4 + (threadIdx.x >> 6)) * 16 * T;
    const float *w[T], *x = static_cast<const float*>(g.x);
    int32_t xo[PIECES];  // rows * dim fits
#pragma unroll
    for (int t = 0; t < T; ++t) w[t] = static_cast<const float*>(g.w) + min(v0 + 16 * t + i, g.vocab - 1) * g.dim;
    const int px = (threadIdx.x % (KC / 4)) * 4, pr = threadIdx.x / (KC / 4);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
        xo[p] = (int32_t)(min(r0 + pr + p * (1024 / KC), g.rows - 1) * g.dim);
    dev::u32x4 wv[2][T][S], xv[PIECES];
    auto fetch = [&](int64_t k, dev::u32x4 (&to)[T][S]) {
        if (k + KC <= g.dim) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int s = 0; s < S; ++s) to[t][s] = dev::load16<DT>(w[t] + k + 16 * s + 4 * q);
#pragma unroll
            for (int p = 0; p < PIECES; ++p) xv[p] = dev::load16<DT>(x + xo[p] + k + px);
        } else {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int s = 0; s < S; ++s) to[t][s] = dev::load_raw<DT>(w[t], k + 16 * s + 4 * q, g.dim).q;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) xv[p] = dev::load_raw<DT>(x + xo[p], k + px, g.dim).q;
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) *reinterpret_cast<dev::u32x4*>(&xs[buf][pr + p * (1024 / KC)][px]) = xv[p];
        __syncthreads();
    };
    f32x4 acc[T][NB];
    zero(acc);
    auto use = [&](const dev::u32x4 (&a)[T][S], int buf) {
        f32x4 part[T][NB];  // a chunk's sums, as in few_logits
        zero(part);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            dev::u32x4 c[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) c[b] = *reinterpret_cast<const dev::u32x4*>(&xs[buf][16 * b + i][16 * s + 4 * q]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int t = 0; t < T; ++t)
                        part[t][b] = mfma4(__uint_as_float(a[t][s][e]), __uint_as_float(c[b][e]), part[t][b]);
        }
        add(acc, part);
    };
    fetch(0, wv[0]);
    stage(0);
    // A chunk's loads are on their way while the one before it is used; a buffer
    // is written again after a barrier behind its last use.
    for (int64_t k = 0; k < g.dim; k += 2 * KC) {
        if (k + KC < g.dim) fetch(k + KC, wv[1]);
        use(wv[0], 0);
        if (k + KC >= g.dim) break;
        stage(1);
        if (k + 2 * KC < g.dim) fetch(k + 2 * KC, wv[0]);
        use(wv[1], 1);
        if (k + 2 * KC < g.dim) stage(0);
    }
    if constexpr (OUT == WIDE_DS) leave_ds<T, NB>(g, v0, acc);  // of one block of rows
    else if constexpr (OUT == WIDE_PLANES) leave_planes<DT, T, NB>(g, v0, r0, acc);
    else leave_stats<T, NB>(g, v0, r0, tile, acc);
}

template <int DT, int NB, bool ODD>
__global__ __launch_bounds__(256) void few_ds_kernel(FewArgs g) {
    constexpr int T = TILES<NB>;
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 * T;
    if (v0 >= g.vocab) return;
    f32x4 acc[T][NB];
    few_logits<DT, NB, ODD>(g, v0, threadIdx.x & 63, acc);
    leave_ds<T, NB>(g, v0, acc);
}

template <int DT, int NB, bool ODD>
__global__ __launch_bounds__(256) void few_planes_kernel(FewArgs g) {
    constexpr int T = TILES<NB>;
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 * T;
    if (v0 >= g.vocab) return;
    f32x4 acc[T][NB];
    few_logits<DT, NB, ODD>(g, v0, threadIdx.x & 63, acc);
    leave_planes<DT, T, NB>(g, v0, 0, acc);
}

template <int DT, int NB>
__global__ __launch_bounds__(256, 2) void few_grad_kernel(FewArgs g) {
    constexpr int RP = 16 * NB, VEC = Elem<DT>::VEC, COLS = 16 * VEC;
    typedef typename Elem<DT>::type E;
    __shared__ float sums[4][RP][COLS];
    // 64 rows of x leave no registers for two waves to a SIMD (124 us instead of 107):
    // LDS holds them.
    constexpr bool XL = NB == 4;
    __shared__ __attribute__((aligned(16))) float xs[XL ? RP : 1][COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * COLS + VEC * i;  // the lane's columns
    const int64_t from = ((int64_t)blockIdx.y * 4 + wave) * g.slice, to = min(from + g.slice, g.vocab);
    // x at row 16 (t / 4) + 4 q + t % 4 (so that a lane reads four of dS^T's values
    // at once), columns n0 + j; zeros in rows without a target.
    float xr[XL ? 1 : 4 * NB][VEC];
    auto load_x = [&](int64_t r, int64_t n, float* v) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
        if (r < g.rows && counted(g.targets[r], g.vocab) && n < g.dim)
            dev::unpack<DT>(dev::load_raw<DT>(static_cast<const E*>(g.x) + r * g.dim, n, g.dim), v);
    };
    if constexpr (XL) {
        for (int k = threadIdx.x * VEC; k < RP * COLS; k += 256 * VEC) {
            float v[VEC];
            load_x(k / COLS, (int64_t)blockIdx.x * COLS + k % COLS, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) xs[k / COLS][k % COLS + j] = v[j];
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int t = 0; t < 4 * NB; ++t) load_x(16 * (t / 4) + 4 * q + t % 4, n0, xr[t]);
    }
    f32x4 dx[NB][VEC];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dx[b][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // 16 entries' values: one block on its way while the other is used.
    struct Block {
        dev::Vec16<DT> w[4];
        float a[4][NB];
        f32x4 d[NB];
    } block[2];
    auto fetch = [&](int64_t v, Block& to_) {
        if (g.dx) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t at = v + 4 * s + q;
                to_.w[s].q = dev::u32x4{0, 0, 0, 0};
                if (at < to && n0 < g.dim) to_.w[s] = dev::load_raw<DT>(static_cast<const E*>(g.w) + at * g.dim, n0, g.dim);
#pragma unroll
                for (int b = 0; b < NB; ++b) to_.a[s][b] = at < to ? g.ds[at * RP + 16 * b + i] : 0.0f;
            }
        }
        if (g.dw) {
            const float* ds = g.ds + min(v + i, g.vocab - 1) * RP + 4 * q;
#pragma unroll
            for (int b = 0; b < NB; ++b) to_.d[b] = *reinterpret_cast<const f32x4*>(ds + 16 * b);
        }
    };
    auto use = [&](int64_t v, const Block& from_) {
        if (g.dx) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                float wf[VEC];
                dev::unpack<DT>(from_.w[s], wf);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dx[b][j] = mfma4(from_.a[s][b], wf[j], dx[b][j]);
            }
        }
        if (g.dw) {
            f32x4 o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 4 * NB; ++t) {
                const float* x = XL ? &xs[16 * (t / 4) + 4 * q + t % 4][VEC * i] : xr[XL ? 0 : t];
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = mfma4(from_.d[t / 4][t % 4], x[j], o[j]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float out[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) out[j] = o[j][e];
                if (v + 4 * q + e < to && n0 < g.dim)
                    dev::store_vec<DT>(static_cast<E*>(g.dw) + (v + 4 * q + e) * g.dim, n0, g.dim, out);
            }
        }
    };
    if (from < to) fetch(from, block[0]);
    for (int64_t v = from; v < to; v += 32) {
        if (v + 16 < to) fetch(v + 16, block[1]);
        __builtin_amdgcn_sched_barrier(0);
        use(v, block[0]);
        if (v + 16 >= to) break;
        if (v + 32 < to) fetch(v + 32, block[0]);
        __builtin_amdgcn_sched_barrier(0);
        use(v + 16, block[1]);
    }
    if (!g.dx) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][16 * b + 4 * q + e][VEC * i + j] = dx[b][j][e];
    __syncthreads();
    for (int k = threadIdx.x; k < RP * COLS / 4; k += 256) {
        const int64_t r = k / (COLS / 4), c = 4 * (k % (COLS / 4)), n = (int64_t)blockIdx.x * COLS + c;
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

// Whether a row of x or W begins in the middle of a dword.
bool odd_rows(const FewArgs& g) {
    return (reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.w) | (uintptr_t)g.dim * 2) & 2;
}

template <int DT, int NB>
int launch_loss(const FewArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(g.vocab, ENTRIES<NB>));
    if (DT != MLXHIP_DTYPE_F32 && odd_rows(g))
        hipLaunchKernelGGL((few_stats_kernel<DT, NB, DT != MLXHIP_DTYPE_F32>), grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((few_stats_kernel<DT, NB, false>), grid, dim3(256), 0, s, g);
    return launch_check("few_stats_kernel");
}

template <int OUT>
int launch_wide(const FewArgs& g, hipStream_t s) {
    const int64_t blocks = ceil_div(g.rows, WIDE_ROWS), tiles = ceil_div(g.vocab, WIDE_ENTRIES);
    hipLaunchKernelGGL((wide_kernel<OUT>), dim3((unsigned)(ceil_div(tiles, 8) * 8 * blocks)), dim3(256), 0, s, g, blocks, tiles);
    return launch_check("wide_kernel");
}

template <int DT, int NB>
int launch_planes(const FewArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(g.vocab, ENTRIES<NB>));
    if (DT != MLXHIP_DTYPE_F32 && odd_rows(g))
        hipLaunchKernelGGL((few_planes_kernel<DT, NB, DT != MLXHIP_DTYPE_F32>), grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((few_planes_kernel<DT, NB, false>), grid, dim3(256), 0, s, g);
    return launch_check("few_planes_kernel");
}

template <int DT>
int typed_planes(const FewArgs& g, hipStream_t s) {
    if (g.rows <= 16) return launch_planes<DT, 1>(g, s);
    if (g.rows <= 32) return launch_planes<DT, 2>(g, s);
    if constexpr (DT == MLXHIP_DTYPE_F32) return launch_wide<WIDE_PLANES>(g, s);
    else return launch_planes<DT, 4>(g, s);
}

template <int DT>
int typed_loss(const FewArgs& g, hipStream_t s) {
    if (g.rows <= 16) return launch_loss<DT, 1>(g, s);
    if (g.rows <= 32) return launch_loss<DT, 2>(g, s);
    if constexpr (DT == MLXHIP_DTYPE_F32) {
        return launch_wide<WIDE_STATS>(g, s);
    } else {
        return launch_loss<DT, 4>(g, s);
    }
}

template <int DT, int NB>
int launch_grad(const FewArgs& g, hipStream_t s) {
    if constexpr (NB == 4) {
        MLXHIP_TRY(launch_wide<WIDE_DS>(g, s));
    } else if (g.form_ds) {
        const dim3 grid((unsigned)ceil_div(g.vocab, ENTRIES<NB>));
        if (DT != MLXHIP_DTYPE_F32 && odd_rows(g))
            hipLaunchKernelGGL((few_ds_kernel<DT, NB, DT != MLXHIP_DTYPE_F32>), grid, dim3(256), 0, s, g);
        else
            hipLaunchKernelGGL((few_ds_kernel<DT, NB, false>), grid, dim3(256), 0, s, g);
    }
    MLXHIP_TRY(launch_check("few_ds_kernel"));
    hipLaunchKernelGGL((few_grad_kernel<DT, NB>), dim3((unsigned)ceil_div(g.dim, 16 * Elem<DT>::VEC), (unsigned)g.slices),
                       dim3(256), 0, s, g);
    return launch_check("few_grad_kernel");
}

}  // namespace
}  // namespace ce

int64_t ce_few_tiles(int dt, int64_t rows, int64_t vocab) {
    if (rows <= 16) return ceil_div(vocab, ce::ENTRIES<1>);
    if (rows <= 32) return ceil_div(vocab, ce::ENTRIES<2>);
    return ceil_div(vocab, dt == MLXHIP_DTYPE_F32 ? ce::WIDE_ENTRIES : ce::ENTRIES<4>);
}

int ce_few_loss(int dt, const ce::FewArgs& g, hipStream_t s) {
    if (dt == MLXHIP_DTYPE_F32) return ce::typed_loss<MLXHIP_DTYPE_F32>(g, s);
    return dt == MLXHIP_DTYPE_BF16 ? ce::typed_loss<MLXHIP_DTYPE_BF16>(g, s) : ce::typed_loss<MLXHIP_DTYPE_F16>(g, s);
}

int ce_few_planes(int dt, const ce::FewArgs& g, hipStream_t s) {
    if (dt == MLXHIP_DTYPE_F32) return ce::typed_planes<MLXHIP_DTYPE_F32>(g, s);
    return dt == MLXHIP_DTYPE_BF16 ? ce::typed_planes<MLXHIP_DTYPE_BF16>(g, s) : ce::typed_planes<MLXHIP_DTYPE_F16>(g, s);
}

int ce_few_grad(int dt, const ce::FewArgs& g, hipStream_t s) {
    if (dt == MLXHIP_DTYPE_BF16) return ce::launch_grad<MLXHIP_DTYPE_BF16, 1>(g, s);
    if (dt == MLXHIP_DTYPE_F16) return ce::launch_grad<MLXHIP_DTYPE_F16, 1>(g, s);
    if (g.rows <= 16) return ce::launch_grad<MLXHIP_DTYPE_F32, 1>(g, s);
    return g.rows <= 32 ? ce::launch_grad<MLXHIP_DTYPE_F32, 2>(g, s) : ce::launch_grad<MLXHIP_DTYPE_F32, 4>(g, s);
}

}  // namespace mlxhip
