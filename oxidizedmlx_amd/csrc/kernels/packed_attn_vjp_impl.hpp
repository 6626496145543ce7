// packed_attn_vjp_impl.hpp — gradients of attention over packed sequences.
//
// With P = 2^(c S - lse log2 e), D = rowsum(dO o O):
//   dS = P o (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two kernels, so that every sum has one owner and a fixed order: dQ by tiles of query rows
// (S and dO V^T transposed, a query to a lane; it leaves lse log2 e and D as the other reads
// them), then dK and dV by tiles of keys (a key to a lane), which walk over the group's heads
// and their tokens. S and dO V^T are formed in both: seven products where one kernel
// with atomic sums of dQ would take five.
//
// Roundings: sums are f32; P and dS are rounded to the operands' type for their products, as
// many independent errors as keys or rows, together about the one that a result itself gets (8192 tokens in 6
// sequences, bf16, o and gradients: 2.1e-3 from 64 bits, 1.7e-3 by rounding exact results).
// Rows that see few keys carry most of a causal sequence's gradient (P is about 1 / keys), so
// those that see up to 64 have P and dS in two terms, the second what the first
// rounds off; and D, which the rounding of O moves (by as much as dS itself after a few keys),
// is formed anew for them, as the row's sum of P dP, in a walk before the one over dS.
// f16 would lose dS below 2^-24: each column of dS (a query's in dQ, a key's in dK) has a power of
// two of its own that brings it to about 2^12, changed (with the sum so far) when a later
// tile outgrows it; P is scaled by 2^14. bf16 and f32 have the range.
//
// Bound by the matrix cores, and what their operands wait for: 8192 tokens in 6 sequences, 32 heads on 8 of 128, bf16:
// dQ 228 us (46 % of the cycles busy), dK and dV 363 (37 %): their sums leave one workgroup of
// eight waves to a compute unit, which wait 47 % of their cycles.
#pragma once

#include "attn_tile.hpp"
#include "packed_attn.hpp"

namespace mlxhip {
namespace attn {

template <int DT>
constexpr float P_SHIFT = DT == MLXHIP_DTYPE_F16 ? 14.0f : 0.0f;

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

// dQ of a tile of query rows: as the forward kernel (ROWS: four waves of 32 rows share tiles of K and
// V in LDS; KEYS: four waves have the same 32 rows and every fourth tile), the rows'
// Q and dO in registers.
template <int DT, int DP, bool KEYS>
__global__ __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS),
                          amdgpu_waves_per_eu(DT == MLXHIP_DTYPE_F32 && (KEYS || DP == 128) ? 1 : 2, 2)))
void attn_dq_kernel(BwdArgs a) {
    constexpr int BM = KEYS ? FEW_ROWS : ROW_TILE, BN = KEYS || DT == MLXHIP_DTYPE_F32 ? 32 : 64, EB = ELEM<DT>;
    constexpr int KB = BN / 32, KS = DP / 16, DB = DP / 32, LW = KEYS ? 1 : WAVES;
    using T = Tile<DT, DP, BN>;
    constexpr int TILES = (KEYS ? WAVES : 2) * 2 * T::BYTES, JOIN = KEYS ? WAVES * 32 * DP * 4 : 0;
    __shared__ __attribute__((aligned(1024))) char smem_raw[TILES > JOIN ? TILES : JOIN];
    __shared__ float row_sums[WAVES][32];
    typedef typename dev::Elem<DT>::type E;

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw + (KEYS ? wave * 2 * T::BYTES : 0);
    const int lin = blockIdx.x;
    const bool per8 = (a.kv_heads & 7) == 0;
    const int item = per8 ? (lin >> 3) % a.row_items : lin / a.kv_heads;
    const int kvh = per8 ? (lin >> 3) / a.row_items * 8 + (lin & 7) : lin % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, a.group, BM, item, &at)) return;
    const int row0 = (at.level - 1) * BM, rows = at.tokens * a.group, n = at.tokens;

    const int wrow = row0 + (KEYS ? 0 : 32 * wave), row = wrow + (lane & 31);
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
    const float lse2 = a.lse[token * a.heads + head] * LOG2E - P_SHIFT<DT>;
    float delta = 0.0f;
    {
        const E* orow = (const E*)a.o + token * a.o_stride + (int64_t)head * a.dim;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const Frag<DT> y = load_frag<DT>(orow, lane, s, a.dim, live);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(y) / 16); ++i) {
                float u[dev::Elem<DT>::VEC], w[dev::Elem<DT>::VEC];
                dev::unpack<DT>({y.q[i]}, u);
                dev::unpack<DT>({g[s].q[i]}, w);
#pragma unroll
                for (int e = 0; e < dev::Elem<DT>::VEC; ++e) delta = __builtin_fmaf(u[e], w[e], delta);
            }
        }
        delta += __shfl_xor(delta, 32, 64);
    }

    TileLoader<DT, DP, BN, LW, TILE> loader;
    const uint32_t stride_bytes = (uint32_t)(a.kv_stride * EB);
    loader.init(KEYS ? 0 : wave, lane, a.dim, stride_bytes);
    const int64_t off = ((int64_t)at.first * a.kv_stride + (int64_t)kvh * a.dim) * EB;
    const auto issue = [&](const void* p, MLXHIP_LDS char* tile, int j) {
        loader.rows((const char*)p + off + (int64_t)j * BN * stride_bytes, n - j * BN, stride_bytes, tile, KEYS ? 0 : wave);
    };

    RowFrag<DT, DP, BN> rf;
    ColFrag<DT, DP, BN> cf;
    rf.init(lane);
    cf.init(lane);
    f32x16 dq[DB] = {};
    Column<DT> column;
    enum { PLAIN, ROW_SUM, FINE };
    float sum = 0.0f;  // ROW_SUM: of P (dP - D), 0 were D exact
    // A tile of keys. after_v: what may start once V has been read.
    const auto compute = [&](auto which, const MLXHIP_LDS char* kt, const MLXHIP_LDS char* vt, int first, auto&& after_v) {
        constexpr int KIND = decltype(which)::value;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int k0 = first + 32 * b;
            if (k0 > wave_last) break;
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                mma<DT>(rf.read(kt, 32 * b, s), q[s], sc);
                mma<DT>(rf.read(vt, 32 * b, s), g[s], dp);
            }
            if (b == KB - 1) after_v();
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], a.c, -lse2)) * (dp[r] - delta);
            if (__ballot(k0 + 31 > wave_first || !live)) {
                own_branch();
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + 8 * (r / 4) + 4 * h + r % 4 > lim) e[r] = 0.0f;
            }
            if constexpr (KIND == ROW_SUM) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += e[r];
            } else {
                column.fit(e, dq);
                const Frag<DT> ds[2] = {frag_of<DT>(e), frag_of<DT>(e + 8)};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const Frag<DT> kc = cf.read(kt, 32 * b + 16 * s, d);
                        if constexpr (KIND == FINE) mma<DT>(kc, rest_of<DT>(e + 8 * s, ds[s]), dq[d]);
                        mma<DT>(kc, ds[s], dq[d]);
                    }
                }
            }
        }
    };
    const auto walk = [&](auto which) {
        if constexpr (KEYS) {
            // A wave's own tiles: V of the next one loads during this one's second product.
            MLXHIP_LDS char* kt = smem;
            MLXHIP_LDS char* vt = smem + T::BYTES;
            int j = wave;
            if (j < n_tiles) {
                issue(a.v, vt, j);
                issue(a.k, kt, j);
            }
            for (; j < n_tiles; j += WAVES) {
                gemm16::wait_vmcnt<0>();
                compute(which, kt, vt, j * BN, [&] {
                    __builtin_amdgcn_s_waitcnt(0xC07F);
                    if (j + WAVES < n_tiles) issue(a.v, vt, j + WAVES);
                });
                __builtin_amdgcn_s_waitcnt(0xC07F);
                if (j + WAVES < n_tiles) issue(a.k, kt, j + WAVES);
            }
        } else {
            if (n_tiles > 0) {
                issue(a.k, smem, 0);
                issue(a.v, smem + T::BYTES, 0);
            }
            for (int j = 0; j < n_tiles; ++j) {
                const MLXHIP_LDS char* kt = smem + (j & 1) * 2 * T::BYTES;
                MLXHIP_LDS char* other = smem + ((j + 1) & 1) * 2 * T::BYTES;
                gemm16::wait_vmcnt<0>();
                gemm16::lds_barrier();
                if (j + 1 < n_tiles) {
                    issue(a.k, other, j + 1);
                    issue(a.v, other + T::BYTES, j + 1);
                }
                if (wrow < rows) compute(which, kt, kt + T::BYTES, j * BN, [] {});
            }
        }
    };
    // By the tile's first row, so that none that sees few keys is left out: 128 rows of ungrouped heads
    // are 128 tokens, of which the first 64 see up to 64 keys.
    if (DT != MLXHIP_DTYPE_F32 && last_key(row0) < FINE_KEYS) {
        walk(std::integral_constant<int, ROW_SUM>{});
        sum += __shfl_xor(sum, 32, 64);
        if constexpr (KEYS) {
            if (h == 0) row_sums[wave][lane] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) sum += row_sums[i][lane & 31];
        } else {
            gemm16::lds_barrier();  // the first tiles are loaded again
        }
        delta += sum * __builtin_amdgcn_exp2f(-P_SHIFT<DT>);
        walk(std::integral_constant<int, DT == MLXHIP_DTYPE_F32 ? PLAIN : FINE>{});
    } else {
        walk(std::integral_constant<int, PLAIN>{});
    }
    float f = a.scale / column.by * __builtin_amdgcn_exp2f(-P_SHIFT<DT>);
    if (live && h == 0 && (!KEYS || wave == 0)) {
        a.lse2[(int64_t)head * a.tokens + token] = lse2;
        a.delta[(int64_t)head * a.tokens + token] = -delta;
    }
    if constexpr (KEYS) {
        // The waves' sums joined in order, value by value; wave w then holds every fourth block of the head.
        __syncthreads();
        float* all = reinterpret_cast<float*>(smem_raw);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) all[(wave * DB * 16 + d * 16 + r) * 64 + lane] = dq[d][r] * f;
        __syncthreads();
        E* to = (E*)a.dq + token * a.q_stride + (int64_t)head * a.dim;
        for (int i = wave; i < DB * 4; i += WAVES) {  // registers 4 i .. 4 i + 3
            f32x4 v = {};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v[e] += all[(w * DB * 16 + 4 * i + e) * 64 + lane];
            const int at_d = 32 * (i / 4) + 8 * (i % 4) + 4 * h;
            if (!live || at_d >= a.dim) continue;
            if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to + at_d) = v;
            else *reinterpret_cast<u32x2*>(to + at_d) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
        }
        return;
    }
    if (live) store_row<DT, DB>((E*)a.dq + token * a.q_stride + (int64_t)head * a.dim, dq, h, a.dim, f);
}

// dK and dV of a tile of keys over share blockIdx.y of its walk (the group's heads, their rows): a wave's 32 keys'
// K and V in registers, tiles of a head's Q and dO in LDS with the rows' lse and
// delta. Two groups of four waves (f32 heads of 128, over 256 registers: one) have the same keys, every
// other tile each, and join at the end: a causal sequence's first keys are seen by all its
// rows, and the longest such walk is what the kernel waits for.
template <int DT, int DP>
constexpr int DKDV_GROUPS = DT == MLXHIP_DTYPE_F32 && DP == 128 ? 1 : 2;

template <int DT, int DP>
__global__ __attribute__((amdgpu_flat_work_group_size(THREADS * DKDV_GROUPS<DT, DP>, THREADS * DKDV_GROUPS<DT, DP>),
                          amdgpu_waves_per_eu(DKDV_GROUPS<DT, DP>, 2)))
void attn_dkdv_kernel(BwdArgs a) {
    constexpr int GROUPS = DKDV_GROUPS<DT, DP>, BR = DT == MLXHIP_DTYPE_F32 ? 32 : 64, EB = ELEM<DT>;
    constexpr int RB = BR / 32, KS = DP / 16, DB = DP / 32;
    using T = Tile<DT, DP, BR>;
    constexpr int STATS = 256, STAGE = 2 * T::BYTES + 2 * STATS, JOIN = (GROUPS - 1) * THREADS * 2 * DB * 16 * 4;
    __shared__ __attribute__((aligned(1024))) char smem_raw[GROUPS * 2 * STAGE > JOIN ? GROUPS * 2 * STAGE : JOIN];
    typedef typename dev::Elem<DT>::type E;

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) % WAVES), part = __builtin_amdgcn_readfirstlane((tid >> 6) / WAVES);
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw + part * 2 * STAGE;
    const int lin = blockIdx.x;
    const bool per8 = (a.kv_heads & 7) == 0;
    const int item = per8 ? (lin >> 3) % a.key_items : lin / a.kv_heads;
    const int kvh = per8 ? (lin >> 3) / a.key_items * 8 + (lin & 7) : lin % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, 1, KEY_TILE, item, &at)) return;
    const int n = at.tokens, tile0 = (at.tiles - at.level) * KEY_TILE;
    const int share = blockIdx.y;
    const int first = a.causal ? tile0 / BR : 0, per = (n + BR - 1) / BR - first, all_steps = a.group * per;
    const int step0 = (int)((int64_t)all_steps * share / a.shares), steps = (int)((int64_t)all_steps * (share + 1) / a.shares) - step0;
    const int fine_rows = a.causal ? FINE_KEYS : n <= FINE_KEYS ? n : 0;

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

    // The sums and the keys' rows leave few registers: what goes by the lane is formed anew
    // where it is used. A spilled register in the loop would wait for the loads behind it.
    const auto lane_now = [&] {
        int l = tid;
        asm volatile("" : "+v"(l));
        return l & 63;
    };
    const uint32_t q_bytes = (uint32_t)(a.q_stride * EB), o_bytes = (uint32_t)(a.o_stride * EB);
    const auto issue = [&](int i, MLXHIP_LDS char* stage) {
        const int at_i = step0 + i, g = at_i / per, head = kvh * a.group + g, j = first + at_i - g * per, left = min(n - j * BR, BR);
        const int64_t token = at.first + (int64_t)j * BR;
        const int l = lane_now();
        TileLoader<DT, DP, BR, WAVES, LEAN> lq, lo;
        lq.init(wave, l, a.dim, q_bytes);
        lo.init(wave, l, a.dim, o_bytes);
        lq.rows((const char*)a.q + (token * a.q_stride + (int64_t)head * a.dim) * EB, left, q_bytes, stage, wave);
        lo.rows((const char*)a.dout + (token * a.o_stride + (int64_t)head * a.dim) * EB, left, o_bytes, stage + T::BYTES, wave);
        if (wave < 2) {
            const float* p = (wave ? a.delta : a.lse2) + (int64_t)head * a.tokens + token;
            lds_load4(buffer(p, (uint32_t)left * 4), stage + 2 * T::BYTES + wave * STATS, (uint32_t)l * 4);
        }
    };

    f32x16 dk[DB] = {}, dv[DB] = {};
    Column<DT> column;
    if (part < steps) issue(part, smem);
    for (int at_step = 0; at_step < steps; at_step += GROUPS) {  // all waves as often: they share the barrier
        const int i = at_step + part, odd = at_step / GROUPS & 1;
        const MLXHIP_LDS char* qt = smem + odd * STAGE;
        const MLXHIP_LDS char* gt = qt + T::BYTES;
        const MLXHIP_LDS float* stats = (const MLXHIP_LDS float*)(qt + 2 * T::BYTES);
        gemm16::wait_vmcnt<0>();
        gemm16::lds_barrier();
        if (i + GROUPS < steps) issue(i + GROUPS, smem + (odd ^ 1) * STAGE);
        if (wkey >= n || i >= steps) continue;
        const int j = first + (step0 + i) % per;
        const int b0 = a.causal && j * BR + 31 < wkey ? min((wkey - j * BR) / 32, RB) : 0, b1 = min(RB, (n - j * BR + 31) / 32);
#pragma unroll 1
        for (int b = b0; b < b1; ++b) {  // blocks of 32 rows that see any of the keys
            const int r0 = j * BR + 32 * b;
            const int l = lane_now(), h = l >> 5, key = wkey + (l & 31);
            RowFrag<DT, DP, BR> rf;
            ColFrag<DT, DP, BR> cf;
            rf.init(l);
            cf.init(l);
            f32x16 sc = {}, dp;  // dp starts as -delta
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 delta = *(const MLXHIP_LDS f32x4*)(stats + STATS / 4 + 32 * b + 8 * q + 4 * h);
#pragma unroll
                for (int x = 0; x < 4; ++x) dp[4 * q + x] = delta[x];
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                mma<DT>(rf.read(qt, 32 * b, s), kf[s], sc);
                mma<DT>(rf.read(gt, 32 * b, s), vf[s], dp);
            }
            float p[16], e[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 lse2 = *(const MLXHIP_LDS f32x4*)(stats + 32 * b + 8 * q + 4 * h);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    p[4 * q + x] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * q + x], a.c, -lse2[x]));
                    e[4 * q + x] = p[4 * q + x] * dp[4 * q + x];
                }
            }
            if (a.causal && r0 < wkey + 31) {
                own_branch();
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (r0 + 8 * (r / 4) + 4 * h + r % 4 < key) p[r] = e[r] = 0.0f;
            }
            // dV, then dK: what one needs is gone before the other's is made.
            const bool fine = DT != MLXHIP_DTYPE_F32 && r0 < fine_rows;
            const auto product = [&](const float (&x)[16], const MLXHIP_LDS char* tile, f32x16 (&acc)[DB]) {
                const Frag<DT> f[2] = {frag_of<DT>(x), frag_of<DT>(x + 8)};
                if constexpr (DT != MLXHIP_DTYPE_F32) {
                    if (fine) {
                        const Frag<DT> rest[2] = {rest_of<DT>(x, f[0]), rest_of<DT>(x + 8, f[1])};
#pragma unroll
                        for (int d = 0; d < DB; ++d)
#pragma unroll
                            for (int s = 0; s < 2; ++s) mma<DT>(cf.read(tile, 32 * b + 16 * s, d), rest[s], acc[d]);
                    }
                }
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int s = 0; s < 2; ++s) mma<DT>(cf.read(tile, 32 * b + 16 * s, d), f[s], acc[d]);
            };
            __builtin_amdgcn_sched_barrier(0);
            product(p, gt, dv);
            __builtin_amdgcn_sched_barrier(0);
            column.fit(e, dk);
            product(e, qt, dk);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    const float unshift = __builtin_amdgcn_exp2f(-P_SHIFT<DT>);
    float fk = a.scale / column.by * unshift;
    if constexpr (GROUPS > 1) {
        __syncthreads();
        float* sums = reinterpret_cast<float*>(smem_raw) + (tid & (THREADS - 1));
        constexpr int EACH = 2 * DB * 16 * THREADS;
        if (part > 0) {
            float* to = sums + (part - 1) * EACH;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    to[(d * 16 + r) * THREADS] = dk[d][r] * fk;
                    to[((DB + d) * 16 + r) * THREADS] = dv[d][r];
                }
        }
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dk[d][r] *= fk;
#pragma unroll
                for (int g = 0; g < GROUPS - 1; ++g) {
                    dk[d][r] += sums[g * EACH + (d * 16 + r) * THREADS];
                    dv[d][r] += sums[g * EACH + ((DB + d) * 16 + r) * THREADS];
                }
            }
        fk = 1.0f;
    }
    if (!live) return;
    if (a.shares > 1) {
        const int64_t each = (int64_t)a.tokens * a.kv_heads * a.dim;
        float* to = a.part + 2 * each * share + ((int64_t)(at.first + key) * a.kv_heads + kvh) * a.dim;
        store_row<MLXHIP_DTYPE_F32, DB>(to, dk, h, a.dim, fk);
        store_row<MLXHIP_DTYPE_F32, DB>(to + each, dv, h, a.dim, unshift);
        return;
    }
    store_row<DT, DB>((E*)a.dk + kv_at, dk, h, a.dim, fk);
    store_row<DT, DB>((E*)a.dv + kv_at, dv, h, a.dim, unshift);
}

// The shares of dK and dV summed in order, a wave to a token.
template <int DT>
__global__ __launch_bounds__(THREADS) void attn_dkdv_join_kernel(BwdArgs a) {
    const int token = (int)blockIdx.x * WAVES + threadIdx.x / 64, quads = a.kv_heads * a.dim / 4;
    Place at;
    if (token >= a.tokens || !find_token(a.starts, a.n_seqs, a.tokens, token, &at)) return;
    const int64_t each = (int64_t)a.tokens * a.kv_heads * a.dim;
    typedef typename dev::Elem<DT>::type E;
    for (int i = threadIdx.x & 63; i < 2 * quads; i += 64) {
        const int w = i >= quads, d = 4 * (i - w * quads);
        const float* p = a.part + w * each + (int64_t)token * a.kv_heads * a.dim + d;
        f32x4 x[MAX_SHARES];
#pragma unroll
        for (int s = 0; s < MAX_SHARES; ++s)
            if (s < a.shares) x[s] = *reinterpret_cast<const f32x4*>(p + 2 * each * s);
        f32x4 v = x[0];
#pragma unroll
        for (int s = 1; s < MAX_SHARES; ++s)
            if (s < a.shares) v += x[s];
        E* to = (E*)(w ? a.dv : a.dk) + (int64_t)token * a.kv_stride + d;
        if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to) = v;
        else *reinterpret_cast<u32x2*>(to) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
    }
}

template <int DT, int DP>
int launch_bwd(const BwdArgs& a, hipStream_t s) {
    const dim3 rows((unsigned)(a.row_items * a.kv_heads)), keys((unsigned)(a.key_items * a.kv_heads), (unsigned)a.shares);
    if (a.few_rows) hipLaunchKernelGGL((attn_dq_kernel<DT, DP, true>), rows, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((attn_dq_kernel<DT, DP, false>), rows, dim3(THREADS), 0, s, a);
    MLXHIP_TRY(launch_check("attn_dq_kernel"));
    hipLaunchKernelGGL((attn_dkdv_kernel<DT, DP>), keys, dim3(THREADS * DKDV_GROUPS<DT, DP>), 0, s, a);
    MLXHIP_TRY(launch_check("attn_dkdv_kernel"));
    if (a.shares == 1) return MLXHIP_OK;
    hipLaunchKernelGGL(attn_dkdv_join_kernel<DT>, dim3((unsigned)ceil_div(a.tokens, WAVES)), dim3(THREADS), 0, s, a);
    return launch_check("attn_dkdv_join_kernel");
}

template <int DT>
int bwd(const BwdArgs& a, hipStream_t s) {
    return a.dim > 64 ? launch_bwd<DT, 128>(a, s) : launch_bwd<DT, 64>(a, s);
}

}  // namespace attn
}  // namespace mlxhip
