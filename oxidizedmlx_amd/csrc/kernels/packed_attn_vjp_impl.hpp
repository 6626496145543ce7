// packed_attn_vjp_impl.hpp — gradients of attention over packed sequences.
//
// With P = 2^(c S - lse log2 e), D = rowsum(dO o O) (one small kernel writes lse log2 e
// and D as the others read them):
//   dS = P o (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two kernels, so that every sum has one owner and a fixed order: dQ by tiles of query rows
// (S and dO V^T transposed, a query to a lane), dK and dV by tiles of keys (a key to a lane), which
// walk over the group's heads and their tokens. S and dO V^T are formed in both: seven
// products where one kernel with atomic sums of dQ would take five.
//
// Roundings: P and dS to the operands' type for their products, sums in f32. f16 would
// lose dS below 2^-24: each column of dS (a query's in dQ, a key's in dK) has a power of two
// of its own that brings it to about 2^12, changed (with the sum so far) when a later
// tile outgrows it; P is scaled by 2^14. bf16 and f32 have the range.
#pragma once

#include "attn_tile.hpp"
#include "packed_attn.hpp"

namespace mlxhip {
namespace attn {

template <int DT>
constexpr float P_SHIFT = DT == MLXHIP_DTYPE_F16 ? 14.0f : 0.0f;

// 16 lanes to a row (token, head).
template <int DT>
__global__ __launch_bounds__(THREADS) void attn_stats_kernel(BwdArgs a) {
    const int64_t row = (int64_t)blockIdx.x * (THREADS / 16) + threadIdx.x / 16;
    if (row >= (int64_t)a.tokens * a.heads) return;
    const int token = (int)(row / a.heads), head = (int)(row - (int64_t)token * a.heads);
    const int64_t at = token * a.o_stride + (int64_t)head * a.dim;
    typedef typename dev::Elem<DT>::type E;
    constexpr int V = dev::Elem<DT>::VEC;
    float sum = 0.0f;
    for (int d = (threadIdx.x & 15) * V; d < a.dim; d += 16 * V) {
        float o[V], g[V];
        dev::unpack<DT>({*reinterpret_cast<const u32x4*>((const E*)a.o + at + d)}, o);
        dev::unpack<DT>({*reinterpret_cast<const u32x4*>((const E*)a.dout + at + d)}, g);
#pragma unroll
        for (int e = 0; e < V; ++e) sum += o[e] * g[e];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (threadIdx.x & 15) return;
    a.delta[(int64_t)head * a.tokens + token] = sum;
    a.lse2[(int64_t)head * a.tokens + token] = a.lse[row] * LOG2E - P_SHIFT<DT>;
}

// f16: the power of two of a lane's column of dS, and the sums in it.
template <int DT>
struct Column {
    static constexpr bool ON = DT == MLXHIP_DTYPE_F16;
    float by = ON ? 0x1p100f : 1.0f;
    // Brings e (a lane's half of the column's 32 values) to the scale.
    template <int DB>
    __device__ inline void fit(float (&e)[16], f32x16 (&acc)[DB]) {
        if constexpr (ON) {
            float mx = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(e[r]));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const bool over = mx * by > 0x1p15f;
            if (__ballot(over)) {
                const int ex = (int)(__float_as_uint(mx) >> 23) - 127;  // mx > 2^-85: normal
                const float to = over ? __uint_as_float((uint32_t)(12 - ex + 127) << 23) : by;
                const float f = to / by;
                by = to;
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] *= by;
        }
    }
};

// A lane's column of a transposed result (32 x DP values of a wave) to a row of memory.
template <int DT, int DB>
__device__ inline void store_row(typename dev::Elem<DT>::type* to, const f32x16 (&acc)[DB], int h, int dim, float f) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * d + 8 * g + 4 * h;
            if (at >= dim) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[d][4 * g + e] * f;
            if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to + at) = f32x4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<u32x2*>(to + at) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
        }
}

// dQ of a tile of query rows: as the forward kernel, K and V tiles in LDS, the
// rows' Q and dO in registers.
template <int DT, int DP>
__global__ __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS), amdgpu_waves_per_eu(DT == MLXHIP_DTYPE_F32 ? 1 : 2, 2)))
void attn_dq_kernel(BwdArgs a) {
    constexpr int BM = ROW_TILE, BN = DT == MLXHIP_DTYPE_F32 ? 32 : 64, EB = ELEM<DT>;
    constexpr int KB = BN / 32, KS = DP / 16, DB = DP / 32;
    using T = Tile<DT, DP, BN>;
    __shared__ __attribute__((aligned(1024))) char smem_raw[4 * T::BYTES];
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw;
    typedef typename dev::Elem<DT>::type E;

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lin = blockIdx.x;
    const bool per8 = (a.kv_heads & 7) == 0;
    const int item = per8 ? (lin >> 3) % a.row_items : lin / a.kv_heads;
    const int kvh = per8 ? (lin >> 3) / a.row_items * 8 + (lin & 7) : lin % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, a.group, BM, item, &at)) return;
    const int row0 = (at.tiles - 1 - at.tile) * BM, rows = at.tokens * a.group, n = at.tokens;

    const int wrow = row0 + 32 * wave, row = wrow + (lane & 31);
    const bool live = row < rows;
    const int tok = live ? (int)((uint32_t)row / (uint32_t)a.group) : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int lim = !live ? -1 : a.causal ? tok : n - 1;
    const auto last_key = [&](int r) { return a.causal ? min(r, rows - 1) / a.group : n - 1; };
    const int wave_last = last_key(wrow + 31), wave_first = last_key(wrow);
    const int n_tiles = (last_key(row0 + BM - 1) + BN) / BN;

    Frag<DT> q[KS], g[KS];
    const int64_t token = at.first + tok;
    const E* qrow = (const E*)a.q + token * a.q_stride + (int64_t)head * a.dim;
    const E* grow = (const E*)a.dout + token * a.o_stride + (int64_t)head * a.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        q[s] = load_frag<DT>(qrow, lane, s, a.dim, live);
        g[s] = load_frag<DT>(grow, lane, s, a.dim, live);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(q[s]) / 16); ++i) q[s].q[i] ^= a.flip;
    }
    const float lse2 = a.lse2[(int64_t)head * a.tokens + token], delta = a.delta[(int64_t)head * a.tokens + token];

    TileLoader<DT, DP, BN, WAVES, false> loader;
    const uint32_t stride_bytes = (uint32_t)(a.kv_stride * EB);
    loader.init(wave, lane, a.dim, stride_bytes);
    const int64_t off = ((int64_t)at.first * a.kv_stride + (int64_t)kvh * a.dim) * EB;
    const auto issue = [&](const void* p, MLXHIP_LDS char* tile, int j) {
        const int left = max(0, min(n - j * BN, BN));
        const auto rsrc = buffer((const char*)p + off + (int64_t)j * BN * stride_bytes, (uint32_t)left * stride_bytes);
#pragma unroll
        for (int i = 0; i < loader.L; ++i) gemm16::lds_load16(rsrc, tile + (i * WAVES + wave) * 1024, loader.voff[i]);
    };

    RowFrag<DT, DP, BN> rf;
    ColFrag<DT, DP, BN> cf;
    rf.init(lane);
    cf.init(lane);
    f32x16 dq[DB] = {};
    Column<DT> column;
    if (n_tiles > 0) {
        issue(a.k, smem, 0);
        issue(a.v, smem + T::BYTES, 0);
    }
    for (int j = 0; j < n_tiles; ++j) {
        const MLXHIP_LDS char* kt = smem + (j & 1) * 2 * T::BYTES;
        const MLXHIP_LDS char* vt = kt + T::BYTES;
        MLXHIP_LDS char* other = smem + ((j + 1) & 1) * 2 * T::BYTES;
        gemm16::wait_vmcnt<0>();
        gemm16::lds_barrier();
        if (j + 1 < n_tiles) {
            issue(a.k, other, j + 1);
            issue(a.v, other + T::BYTES, j + 1);
        }
        if (wrow >= rows) continue;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int k0 = j * BN + 32 * b;
            if (k0 > wave_last) break;
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                mma<DT>(rf.read(kt, 32 * b, s), q[s], sc);
                mma<DT>(rf.read(vt, 32 * b, s), g[s], dp);
            }
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], a.c, -lse2)) * (dp[r] - delta);
            if (__ballot(k0 + 31 > wave_first || !live)) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + 8 * (r / 4) + 4 * h + r % 4 > lim) e[r] = 0.0f;
            }
            column.fit(e, dq);
            const Frag<DT> ds[2] = {frag_of<DT>(e), frag_of<DT>(e + 8)};
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int s = 0; s < 2; ++s) mma<DT>(cf.read(kt, 32 * b + 16 * s, d), ds[s], dq[d]);
        }
    }
    if (live)
        store_row<DT, DB>((E*)a.dq + token * a.q_stride + (int64_t)head * a.dim, dq, h, a.dim,
                          a.scale / column.by * __builtin_amdgcn_exp2f(-P_SHIFT<DT>));
}

// 64 floats from `first` of p (records: as many bytes as there are) to LDS, lane i the i-th.
__device__ inline void lds_load4(__amdgpu_buffer_rsrc_t rsrc, MLXHIP_LDS char* dst, uint32_t voff) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(m0) : "memory");
}

// dK and dV of a tile of keys, 32 to a wave, over share blockIdx.y of the group's
// heads: the keys' K and V in registers, tiles of a head's Q and dO in LDS with the
// rows' lse and delta.
template <int DT, int DP>
__global__ __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS), amdgpu_waves_per_eu(1, 2)))
void attn_dkdv_kernel(BwdArgs a) {
    constexpr int BR = DT == MLXHIP_DTYPE_F32 ? 32 : 64, EB = ELEM<DT>;
    constexpr int RB = BR / 32, KS = DP / 16, DB = DP / 32;
    using T = Tile<DT, DP, BR>;
    constexpr int STATS = 256, STAGE = 2 * T::BYTES + 2 * STATS;
    __shared__ __attribute__((aligned(1024))) char smem_raw[2 * STAGE];
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw;
    typedef typename dev::Elem<DT>::type E;

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lin = blockIdx.x;
    const bool per8 = (a.kv_heads & 7) == 0;
    const int item = per8 ? (lin >> 3) % a.key_items : lin / a.kv_heads;
    const int kvh = per8 ? (lin >> 3) / a.key_items * 8 + (lin & 7) : lin % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, 1, KEY_TILE, item, &at)) return;
    const int n = at.tokens, tile0 = at.tile * KEY_TILE;
    const int g0 = (int)((int64_t)a.group * blockIdx.y / a.shares), g1 = (int)((int64_t)a.group * (blockIdx.y + 1) / a.shares);
    const int first = a.causal ? tile0 / BR : 0, per = (n + BR - 1) / BR - first, steps = (g1 - g0) * per;

    const int wkey = tile0 + 32 * wave, key = wkey + (lane & 31);
    const bool live = key < n;
    Frag<DT> kf[KS], vf[KS];
    const int64_t kv_at = (at.first + (int64_t)(live ? key : 0)) * a.kv_stride + (int64_t)kvh * a.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kf[s] = load_frag<DT>((const E*)a.k + kv_at, lane, s, a.dim, live);
        vf[s] = load_frag<DT>((const E*)a.v + kv_at, lane, s, a.dim, live);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(kf[s]) / 16); ++i) kf[s].q[i] ^= a.flip;
    }

    TileLoader<DT, DP, BR, WAVES, false> lq, lo;
    const uint32_t q_bytes = (uint32_t)(a.q_stride * EB), o_bytes = (uint32_t)(a.o_stride * EB);
    lq.init(wave, lane, a.dim, q_bytes);
    lo.init(wave, lane, a.dim, o_bytes);
    const auto issue = [&](int i, MLXHIP_LDS char* stage) {
        const int head = kvh * a.group + g0 + i / per, j = first + i % per, left = min(n - j * BR, BR);
        const int64_t token = at.first + (int64_t)j * BR;
        const auto rq = buffer((const char*)a.q + (token * a.q_stride + (int64_t)head * a.dim) * EB, (uint32_t)left * q_bytes);
        const auto ro = buffer((const char*)a.dout + (token * a.o_stride + (int64_t)head * a.dim) * EB, (uint32_t)left * o_bytes);
#pragma unroll
        for (int x = 0; x < lq.L; ++x) {
            gemm16::lds_load16(rq, stage + (x * WAVES + wave) * 1024, lq.voff[x]);
            gemm16::lds_load16(ro, stage + T::BYTES + (x * WAVES + wave) * 1024, lo.voff[x]);
        }
        if (wave < 2) {
            const float* p = (wave ? a.delta : a.lse2) + (int64_t)head * a.tokens + token;
            lds_load4(buffer(p, (uint32_t)left * 4), stage + 2 * T::BYTES + wave * STATS, (uint32_t)lane * 4);
        }
    };

    RowFrag<DT, DP, BR> rf;
    ColFrag<DT, DP, BR> cf;
    rf.init(lane);
    cf.init(lane);
    f32x16 dk[DB] = {}, dv[DB] = {};
    Column<DT> column;
    if (steps > 0) issue(0, smem);
    for (int i = 0; i < steps; ++i) {
        const MLXHIP_LDS char* qt = smem + (i & 1) * STAGE;
        const MLXHIP_LDS char* gt = qt + T::BYTES;
        const MLXHIP_LDS float* stats = (const MLXHIP_LDS float*)(qt + 2 * T::BYTES);
        gemm16::wait_vmcnt<0>();
        gemm16::lds_barrier();
        if (i + 1 < steps) issue(i + 1, smem + ((i + 1) & 1) * STAGE);
        if (wkey >= n) continue;
        const int j = first + i % per;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int r0 = j * BR + 32 * b;
            if (r0 >= n || (a.causal && r0 + 31 < wkey)) continue;
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                mma<DT>(rf.read(qt, 32 * b, s), kf[s], sc);
                mma<DT>(rf.read(gt, 32 * b, s), vf[s], dp);
            }
            float p[16], e[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 lse2 = *(const MLXHIP_LDS f32x4*)(stats + 32 * b + 8 * q + 4 * h);
                const f32x4 delta = *(const MLXHIP_LDS f32x4*)(stats + STATS / 4 + 32 * b + 8 * q + 4 * h);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    p[4 * q + x] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * q + x], a.c, -lse2[x]));
                    e[4 * q + x] = p[4 * q + x] * (dp[4 * q + x] - delta[x]);
                }
            }
            if (a.causal && r0 < wkey + 31) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (r0 + 8 * (r / 4) + 4 * h + r % 4 < key) p[r] = e[r] = 0.0f;
            }
            column.fit(e, dk);
            const Frag<DT> pf[2] = {frag_of<DT>(p), frag_of<DT>(p + 8)}, ds[2] = {frag_of<DT>(e), frag_of<DT>(e + 8)};
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    mma<DT>(cf.read(gt, 32 * b + 16 * s, d), pf[s], dv[d]);
                    mma<DT>(cf.read(qt, 32 * b + 16 * s, d), ds[s], dk[d]);
                }
        }
    }
    if (!live) return;
    const float unshift = __builtin_amdgcn_exp2f(-P_SHIFT<DT>), fk = a.scale / column.by * unshift;
    if (a.shares > 1) {
        const int64_t each = (int64_t)a.tokens * a.kv_heads * a.dim;
        float* to = a.part + 2 * each * blockIdx.y + ((int64_t)(at.first + key) * a.kv_heads + kvh) * a.dim;
        store_row<MLXHIP_DTYPE_F32, DB>(to, dk, h, a.dim, fk);
        store_row<MLXHIP_DTYPE_F32, DB>(to + each, dv, h, a.dim, unshift);
        return;
    }
    store_row<DT, DB>((E*)a.dk + kv_at, dk, h, a.dim, fk);
    store_row<DT, DB>((E*)a.dv + kv_at, dv, h, a.dim, unshift);
}

// The shares of dK and dV summed in order; only the tokens of sequences.
template <int DT>
__global__ __launch_bounds__(THREADS) void attn_dkdv_join_kernel(BwdArgs a) {
    const int quads = a.kv_heads * a.dim / 4;
    const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int64_t token = i / quads;
    if (token >= a.tokens) return;
    bool of_sequence = false;
    for (int s = 0; s < a.n_seqs && !of_sequence; ++s) of_sequence = a.starts[s] <= token && token < a.starts[s + 1];
    if (!of_sequence) return;
    const int64_t each = (int64_t)a.tokens * a.kv_heads * a.dim, at = 4 * (i - token * quads);
    typedef typename dev::Elem<DT>::type E;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float* p = a.part + w * each + 4 * i;
        f32x4 v = *reinterpret_cast<const f32x4*>(p);
        for (int s = 1; s < a.shares; ++s) v += *reinterpret_cast<const f32x4*>(p + 2 * each * s);
        E* to = (E*)(w ? a.dv : a.dk) + token * a.kv_stride + at;
        if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to) = v;
        else *reinterpret_cast<u32x2*>(to) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
    }
}

template <int DT, int DP>
int launch_bwd(const BwdArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(attn_stats_kernel<DT>, dim3((unsigned)ceil_div((int64_t)a.tokens * a.heads, THREADS / 16)), dim3(THREADS),
                       0, s, a);
    MLXHIP_TRY(launch_check("attn_stats_kernel"));
    hipLaunchKernelGGL((attn_dkdv_kernel<DT, DP>), dim3((unsigned)(a.key_items * a.kv_heads), (unsigned)a.shares), dim3(THREADS),
                       0, s, a);
    MLXHIP_TRY(launch_check("attn_dkdv_kernel"));
    if (a.shares > 1) {
        hipLaunchKernelGGL(attn_dkdv_join_kernel<DT>, dim3((unsigned)ceil_div((int64_t)a.tokens * a.kv_heads * a.dim / 4, THREADS)),
                           dim3(THREADS), 0, s, a);
        MLXHIP_TRY(launch_check("attn_dkdv_join_kernel"));
    }
    hipLaunchKernelGGL((attn_dq_kernel<DT, DP>), dim3((unsigned)(a.row_items * a.kv_heads)), dim3(THREADS), 0, s, a);
    return launch_check("attn_dq_kernel");
}

template <int DT>
int bwd(const BwdArgs& a, hipStream_t s) {
    return a.dim > 64 ? launch_bwd<DT, 128>(a, s) : launch_bwd<DT, 64>(a, s);
}

}  // namespace attn
}  // namespace mlxhip
