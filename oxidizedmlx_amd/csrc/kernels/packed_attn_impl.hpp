// packed_attn_impl.hpp — attention of packed sequences with grouped heads, and of new
// tokens over a cache in pages.
//
// For each sequence and K/V head the query rows are the pairs (token, head of the
// group), row = token * group + head, so that a tile of K and V serves the whole group.
// With c = scale log2 e and a row's running maximum m,
//   S^T = K Q^T,  p = 2^(c S - c m),  l += sum p,  O^T += V^T p^T,
// O and l rescaled when m moves: one pass over the keys. The transposed scores put a
// query in a lane, its keys in the lane's registers: the maximum needs one exchange
// between the two halves of a wave, p none before it is the next product's operand.
//
// Roundings: scores, p's sum and O are f32. p is rounded to the operands' type for its
// product (relative 2^-8 or 2^-11 at most each, as many independent ones as keys, beside the one
// that the result itself gets); f16's p is scaled by 2^6, which keeps probabilities
// down to 2^-20 normal. Results are off from 64 bits by 1.8e-3 to 2.3e-3 of their size in
// bf16, 2.5e-4 to 2.9e-4 in f16, where rounding exact ones takes 1.4e-3 to 1.7e-3 and 2.1e-4.
// A maximum moves only once it is passed by 2^8: p stays below 2^14 and most tiles rescale
// nothing. Sums of p v may then pass the range of f32 and bf16 where the result does not (v
// from about 2^120 / keys on): rows that end non-finite are formed again with p times 2^-40,
// parts are joined again in such units.
//
// ROWS: four waves of 32 rows share tiles of 64 keys (f32: 32), two in LDS, the next
// on its way. KEYS, for few rows: the four waves have the same 32 rows and every fourth
// tile of 32 keys each, with LDS of their own and no barrier, and join at the end.
// Where there are few tiles of rows the keys are split over workgroups too; the parts
// (O, m, l in f32) are joined by a second kernel.
//
// Bound: prompts by the matrix cores with softmax's vector work between (32768 tokens, 16 heads on 4 of 128,
// bf16: 4.0 ms, 1.10 PFLOP/s; a large library product 1.33), single tokens by HBM (64 over up to 8192
// positions, 700 MB: 143 us and 6 to join; 2 over 131072, 1.07 GB: 183 and 9), few of them by a
// chain of loads and one wave's products (8 f32 tokens over 144 positions: 10.8 us a call).
#pragma once

#include "attn_tile.hpp"
#include "packed_attn.hpp"

namespace mlxhip {
namespace attn {

__device__ inline int length_of(const PagedArgs& p, int seq) { return __builtin_amdgcn_readfirstlane(max(p.lens[seq], 0)); }
// Of a length's positions those that the table has room for.
__device__ inline int keys_of(const PagedArgs& p, int length) { return (int)min((int64_t)length, p.table_width << p.page_shift); }

// Parts of a sequence: of as many keys as the longest one has in each of the launch's `splits`, so that
// workgroups take about as long whatever their sequence, and MIN_SPAN at least.
__device__ inline int parts_of(const PagedArgs& p, int keys, int splits) {
    if (splits == 1) return 1;
    int most = 0;
    for (int i = threadIdx.x & 63; i < p.n_seqs; i += 64) most = max(most, p.lens[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    most = __builtin_amdgcn_readfirstlane(keys_of(p, most));
    const int span = max(MIN_SPAN, (most + splits - 1) / splits);
    return max(1, (keys + span - 1) / span);
}

template <int DT, int DP, bool KEYS>
struct FwdShape {
    static constexpr int BM = KEYS ? FEW_ROWS : ROW_TILE, BN = KEYS || DT == MLXHIP_DTYPE_F32 ? 32 : 64;
    static constexpr int LW = KEYS ? 1 : WAVES, STAGES = KEYS ? 1 : 2;
    using T = Tile<DT, DP, BN>;
    static constexpr int TILES = (KEYS ? WAVES : 1) * STAGES * 2 * T::BYTES, JOIN = KEYS ? WAVES * 32 * (DP + 3) * 4 : 0;
    static constexpr int LDS = TILES > JOIN ? TILES : JOIN;
};

// A workgroup's tile of rows over its part of the keys. False where a result is not finite: nothing is
// stored then, and the CAREFUL form, which keeps non-finite values of v from rows that do not see them,
// forms it all anew. That form takes tid and lin through registers of their own, so that nothing of
// it is kept while the other runs.
template <int DT, int DP, bool PAGED, bool KEYS, bool CAREFUL>
__device__ __attribute__((always_inline)) inline bool fwd_tile(const FwdArgs& a, char* smem_raw, int tid, int lin) {
    using S = FwdShape<DT, DP, KEYS>;
    constexpr int BM = S::BM, BN = S::BN, LW = S::LW, STAGES = S::STAGES;
    constexpr int KB = BN / 32, KS = DP / 16, DB = DP / 32, EB = ELEM<DT>;
    constexpr int AHEAD = DT == MLXHIP_DTYPE_F32 ? 2 : 4;  // fragments read ahead
    constexpr float SHIFT = DT == MLXHIP_DTYPE_F16 ? 6.0f : 0.0f, MOVE = 8.0f;
    constexpr bool RANGE = DT != MLXHIP_DTYPE_F16;  // v as large as f32's largest
    constexpr float DOWN = 0x1p-40f, DOWN_LOG2 = -40.0f;
    using T = typename S::T;
    typedef typename dev::Elem<DT>::type E;

    const int lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw + (KEYS ? wave * STAGES * 2 * T::BYTES : 0);

    // Workgroups go round the 8 dies: with a multiple of 8 K/V heads each die keeps
    // to its own, whose keys its L2 then holds. Long tiles of a causal sequence first.
    const int per8 = a.kv_heads & 7 ? 1 : 8;
    const int item = per8 == 8 ? (lin >> 3) % a.items : lin / a.kv_heads;
    const int kvh = per8 == 8 ? (lin >> 3) / a.items * 8 + (lin & 7) : lin % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, a.group, BM, item, &at)) return true;
    const int row0 = (at.level - 1) * BM, rows = at.tokens * a.group;
    const int length = PAGED ? length_of(a.pages, at.seq) : at.tokens, keys = PAGED ? keys_of(a.pages, length) : length;
    const int shift = length - at.tokens;  // position of the first new token
    const int parts = PAGED ? parts_of(a.pages, keys, a.splits) : 1, part = PAGED ? blockIdx.y : 0;
    if (part >= parts) return true;

    // This lane's row and the last key it sees.
    const int wrow = row0 + (KEYS ? 0 : 32 * wave), row = wrow + (lane & 31);
    const bool live = row < rows;
    const int tok = (int)((uint32_t)row / (uint32_t)a.group), head = kvh * a.group + (row - tok * a.group);
    const int lim = !live ? -1 : a.causal ? min(tok + shift, keys - 1) : keys - 1;
    const auto last_key = [&](int r) {  // of row r, or of the last row
        return a.causal ? min((min(r, rows - 1)) / a.group + shift, keys - 1) : keys - 1;
    };
    const int wave_last = last_key(wrow + 31), wave_first = last_key(wrow);
    const int n_tiles = max(0, last_key(row0 + BM - 1) + BN) / BN;
    // Divided by the vector unit; in scalar registers, or the walk and its loads go by vector ones.
    const int t0 = __builtin_amdgcn_readfirstlane((int)((int64_t)n_tiles * part / parts));
    const int t1 = __builtin_amdgcn_readfirstlane((int)((int64_t)n_tiles * (part + 1) / parts));

    Frag<DT> q[KS];
    const E* qrow = (const E*)a.q + (int64_t)(at.first + (live ? tok : 0)) * a.q_stride + (int64_t)(live ? head : 0) * a.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        q[s] = load_frag<DT>(qrow, lane, s, a.dim, live);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(q[s]) / 16); ++i) q[s].q[i] ^= a.flip;
    }

    // Loads: a tile's rows one after another in memory, or page by page (an
    // instruction's rows lie in one page: pages hold a multiple of 16).
    TileLoader<DT, DP, BN, LW, PAGED ? PAGES : TILE> loader;
    const uint32_t stride_bytes = (uint32_t)((PAGED ? a.dim : a.kv_stride) * EB);
    loader.init(KEYS ? 0 : wave, lane, a.dim, stride_bytes);
    const char* kbase = (const char*)a.k;
    const char* vbase = (const char*)a.v;
    if constexpr (!PAGED) {
        const int64_t off = ((int64_t)at.first * a.kv_stride + (int64_t)kvh * a.dim) * EB;
        kbase += off;
        vbase += off;
    }
    // Page numbers of 64 pages, one to a lane, read anew where the tiles reach the next 64. The
    // wait is there, or the compiler would wait at every use for all loads under way.
    const int32_t* table = PAGED ? a.pages.table + (int64_t)at.seq * a.pages.table_width : nullptr;
    int window = -64, numbers = -1;
    const auto turn_to = [&](int j) {
        if constexpr (PAGED) {
            const int first = (j * BN >> a.pages.page_shift) & ~63;
            if (first == window) return;
            window = first;
            numbers = (int64_t)first + lane < a.pages.table_width ? table[first + lane] : -1;
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        }
    };
    const auto issue = [&](const char* base, MLXHIP_LDS char* tile, int j) {
        if constexpr (PAGED) {
            loader.paged(base, tile, KEYS ? 0 : wave, [&](int from, uint32_t* bytes) {
                const int r = j * BN + from, left = min(keys - r, 16);
                const int page = __builtin_amdgcn_readlane(numbers, (r >> a.pages.page_shift) & 63);
                const bool ok = left > 0 && page >= 0 && page < a.pages.pages;
                *bytes = ok ? (uint32_t)left * stride_bytes : 0u;
                const int64_t at_row = (((int64_t)(ok ? page : 0) * a.kv_heads + kvh) << a.pages.page_shift) +
                                       (r & ((1 << a.pages.page_shift) - 1));
                return at_row * stride_bytes;
            });
        } else {
            loader.rows(base + (int64_t)j * BN * stride_bytes, keys - j * BN, stride_bytes, tile, KEYS ? 0 : wave);
        }
    };

    RowFrag<DT, DP, BN> kf;
    ColFrag<DT, DP, BN> vf;
    kf.init(lane);
    vf.init(lane);
    f32x16 o[DB] = {};
    float m = -INFINITY, l = 0.0f;
    float down = 1.0f;  // of a row's p in its sums with v (not in l)

    // One tile of keys from k0 on. after_scores: what may start once K has been read; before_v: what V waits for.
    const auto compute = [&](const MLXHIP_LDS char* kt, const MLXHIP_LDS char* vt, int k0, auto&& after_scores,
                             auto&& before_v) {
        f32x16 sc[KB] = {};
        stream<DT, KB * KS, AHEAD>([&](int i) { return kf.read(kt, 32 * (i / KS), i % KS); },
                                   [&](int i, const Frag<DT>& f) { mma<DT>(f, q[i % KS], sc[i / KS]); });
        after_scores();
        const bool masked = k0 + BN - 1 > wave_first || !live;
        const bool any_masked = __ballot(masked) != 0;
        if (any_masked) {
            own_branch();
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + 32 * b + 8 * (r / 4) + 4 * h + r % 4 > lim) sc[b][r] = -INFINITY;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[b][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__ballot(mx > m && !((mx - m) * a.c <= MOVE))) {
            const float to = fmaxf(m, mx);
            const float by = to == m ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * a.c);
            m = to;
            l *= by;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= by;
        }
        const float mc = m == -INFINITY ? 0.0f : m * a.c - SHIFT;
        Frag<DT> p[2 * KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][r], a.c, -mc));
                l += e[r];
                if constexpr (CAREFUL) e[r] *= down;
            }
            p[2 * b] = frag_of<DT>(e);
            p[2 * b + 1] = frag_of<DT>(e + 8);
        }
        before_v();
        if (CAREFUL && any_masked) {
            // p = 0 of a masked key would make NaN of a non-finite v: those are taken out of the
            // product, and what is counted of them among the keys that a row sees makes it NaN.
#pragma unroll 1
            for (int s = 0; s < 2 * KB; ++s) {
                float sees[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = k0 + 16 * s + 8 * (j / 4) + 4 * h + j % 4 <= lim ? 1.0f : 0.0f;
                Frag<DT> ps = p[0];
#pragma unroll
                for (int i = 1; i < 2 * KB; ++i)
                    if (i == s) ps = p[i];
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    Frag<DT> v = vf.read(vt, 16 * s, d);
                    const Frag<DT> bad = take_non_finite<DT>(v);
                    mma<DT>(v, ps, o[d]);
                    f32x16 count = {};
                    mma<DT>(bad, frag_of<DT>(sees), count);
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] = count[r] > 0.0f ? NAN : o[d][r];
                }
            }
        } else {
            stream<DT, DB * 2 * KB, AHEAD>([&](int i) { return vf.read(vt, 16 * (i % (2 * KB)), i / (2 * KB)); },
                                           [&](int i, const Frag<DT>& f) { mma<DT>(f, p[i % (2 * KB)], o[i / (2 * KB)]); });
        }
    };

    const auto walk = [&] {
        if constexpr (KEYS) {
            // K of the next tile loads during this one's softmax and second product, V during
            // the next one's first; a wait leaves the newest loads under way.
            MLXHIP_LDS char* kt = smem;
            MLXHIP_LDS char* vt = smem + T::BYTES;
            constexpr int L = decltype(loader)::L;
            int j = t0 + wave;
            if (j < t1) {
                turn_to(j);
                issue(kbase, kt, j);
                issue(vbase, vt, j);
            }
            for (; j < t1; j += WAVES) {
                const bool more = j + WAVES < t1;
                gemm16::wait_vmcnt<L>();
                compute(
                    kt, vt, j * BN,
                    [&] {
                        __builtin_amdgcn_s_waitcnt(0xC07F);
                        if (more) {
                            turn_to(j + WAVES);
                            issue(kbase, kt, j + WAVES);
                        }
                    },
                    [&] {
                        if (more) gemm16::wait_vmcnt<L>();
                        else gemm16::wait_vmcnt<0>();
                    });
                __builtin_amdgcn_s_waitcnt(0xC07F);
                if (more) issue(vbase, vt, j + WAVES);
            }
        } else {
            if (t0 < t1) {
                turn_to(t0);
                issue(kbase, smem, t0);
                issue(vbase, smem + T::BYTES, t0);
            }
            for (int j = t0; j < t1; ++j) {
                MLXHIP_LDS char* tile = smem + ((j - t0) & 1) * 2 * T::BYTES;
                MLXHIP_LDS char* other = smem + ((j - t0 + 1) & 1) * 2 * T::BYTES;
                gemm16::wait_vmcnt<0>();
                gemm16::lds_barrier();
                if (j + 1 < t1) {
                    turn_to(j + 1);
                    issue(kbase, other, j + 1);
                    issue(vbase, other + T::BYTES, j + 1);
                }
                if (wrow < rows && j * BN <= wave_last) compute(tile, tile + T::BYTES, j * BN, [] {}, [] {});
            }
        }
    };
    // KEYS: what the four waves' sums make together, too.
    const auto finite = [&] {
        float sum = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum = __builtin_fmaf(KEYS && RANGE ? o[d][r] * WAVES : o[d][r], 0.0f, sum);
        return sum == 0.0f;  // NaN is not 0
    };
    if constexpr (!CAREFUL) {
        walk();
        if (__builtin_expect(__syncthreads_or(!finite()) != 0, 0)) return false;
    } else {
        // Rows that are still not finite once more, with p taken down; the others have the same bits again.
#pragma unroll 1
        for (int last = !RANGE;; last = 1) {
            walk();
            const bool bad = !finite();
            if (last || !__syncthreads_or(bad)) break;
            if (__ballot(bad) >> (lane & 31) & 0x100000001ull) down = DOWN;  // either half of the row's values
            window = -64;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = f32x16{};
            m = -INFINITY;
            l = 0.0f;
        }
    }
    const float up = 1.0f / down;
    const auto store = [&] {
        l += __shfl_xor(l, 32, 64);
        float mc = m == -INFINITY ? 0.0f : m * a.c - SHIFT;  // l and o are sums of 2^(c S - mc)
        bool empty = m == -INFINITY && l == 0.0f;            // no key seen (by this wave)
        // A part's base and sum; where o is taken down, in its units.
        const auto store_part = [&](float* to, float base, float sum, float up) {
            to[0] = empty ? -INFINITY : up > 1.0f ? base - DOWN_LOG2 : base;
            to[1] = up > 1.0f ? sum * DOWN : sum;
        };

        if constexpr (KEYS) {
            // Joined through LDS: each wave's o, mc, l for the 32 rows; wave w then sums
            // the four for every fourth part of the head.
            __syncthreads();
            float* all = reinterpret_cast<float*>(smem_raw);
            constexpr int EACH = 32 * (DP + 3);
            float* mine = all + wave * EACH;
            const int r = lane & 31;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[(32 * d + 8 * (i / 4) + 4 * h + i % 4) * 32 + r] = o[d][i];
            if (h == 0) {
                mine[DP * 32 + r] = empty ? -INFINITY : mc;
                mine[(DP + 1) * 32 + r] = l;
                mine[(DP + 2) * 32 + r] = up;
            }
            __syncthreads();
            float top = -INFINITY, w[WAVES], lift = 0.0f;
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                w[i] = all[i * EACH + DP * 32 + r];
                top = w[i] > top || w[i] != w[i] ? w[i] : top;
            }
            empty = top == -INFINITY;
            mc = empty ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                w[i] = w[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w[i] - mc);
                l += w[i] * all[i * EACH + (DP + 1) * 32 + r];
                lift = fmaxf(lift, all[i * EACH + (DP + 2) * 32 + r]);
            }
            // The four sums weighed by what they are divided by in the end; of a part they stay taken down.
            const bool whole = parts == 1;
            const float by = 1.0f / (whole ? l : lift);
#pragma unroll
            for (int i = 0; i < WAVES; ++i) w[i] *= by * all[i * EACH + (DP + 2) * 32 + r];
            // Head values 4 (h + 2 wave + 8 i) .. + 3 of the lane's row.
            for (int d0 = 4 * (h + 2 * wave); d0 < a.dim; d0 += 32) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = 0.0f;
#pragma unroll
                    for (int i = 0; i < WAVES; ++i) v[e] += w[i] * all[i * EACH + (d0 + e) * 32 + r];
                    if (whole && lim < 0) v[e] = 0.0f;
                }
                if (!live) continue;
                if (!PAGED && a.lse && d0 == 0)
                    a.lse[(int64_t)(at.first + tok) * a.heads + head] = lim < 0 ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * LN2;
                if (!whole) {
                    float* to = a.part + ((int64_t)part * a.tokens * a.heads + (int64_t)(at.first + tok) * a.heads + head) * (a.dim + 4);
                    *reinterpret_cast<f32x4*>(to + d0) = f32x4{v[0], v[1], v[2], v[3]};
                    if (d0 == 0) store_part(to + a.dim, mc, l, lift);
                    continue;
                }
                E* to = (E*)a.o + (int64_t)(at.first + tok) * a.o_stride + (int64_t)head * a.dim + d0;
                if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
                else *reinterpret_cast<u32x2*>(to) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
            }
            return;
        }

        if (!live) return;
        if (parts > 1) {
            float* to = a.part + ((int64_t)part * a.tokens * a.heads + (int64_t)(at.first + tok) * a.heads + head) * (a.dim + 4);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int at_d = 32 * d + 8 * g + 4 * h;
                    if (at_d < a.dim) *reinterpret_cast<f32x4*>(to + at_d) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                }
            if (h == 0) store_part(to + a.dim, mc, l, up);
            return;
        }
        if (a.lse && h == 0) a.lse[(int64_t)(at.first + tok) * a.heads + head] = lim < 0 ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * LN2;
        const float inv = 1.0f / l * up;
        E* orow = (E*)a.o + (int64_t)(at.first + tok) * a.o_stride + (int64_t)head * a.dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at_d = 32 * d + 8 * g + 4 * h;
                if (at_d >= a.dim) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = lim < 0 ? 0.0f : o[d][4 * g + e] * inv;
                if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(orow + at_d) = f32x4{v[0], v[1], v[2], v[3]};
                else *reinterpret_cast<u32x2*>(orow + at_d) = u32x2{gemm16::pack2<DT>(v[0], v[1]), gemm16::pack2<DT>(v[2], v[3])};
            }
    };
    store();
    return true;
}

template <int DT, int DP, bool PAGED, bool KEYS>
__global__ __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS), amdgpu_waves_per_eu(KEYS && DP == 128 && DT == MLXHIP_DTYPE_F32 ? 1 : 2, 2)))
void attn_fwd_kernel(FwdArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[FwdShape<DT, DP, KEYS>::LDS];
    int tid = threadIdx.x, lin = blockIdx.x;
    if (__builtin_expect(fwd_tile<DT, DP, PAGED, KEYS, false>(a, smem, tid, lin), 1)) return;
    asm volatile("" : "+v"(tid), "+s"(lin));
    fwd_tile<DT, DP, PAGED, KEYS, true>(a, smem, tid, lin);
}

// The parts of a tile of rows joined, in order: 32 threads to a row, four values each, eight
// rows at a time; a row's parts are read 16 at a time.
template <int DT, int BM>
__global__ __launch_bounds__(THREADS) void attn_join_kernel(FwdArgs a) {
    const int t = threadIdx.x % 32, item = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads;
    Place at;
    if (!find_tile(a.starts, a.n_seqs, a.tokens, a.group, BM, item, &at)) return;
    const int length = length_of(a.pages, at.seq), parts = parts_of(a.pages, keys_of(a.pages, length), a.splits);
    if (parts == 1 || 4 * t >= a.dim) return;
    const int row0 = (at.level - 1) * BM, rows = min(at.tokens * a.group - row0, BM);
    const int64_t step = (int64_t)a.tokens * a.heads * (a.dim + 4);
    typedef typename dev::Elem<DT>::type E;
    for (int r = threadIdx.x / 32; r < rows; r += THREADS / 32) {
        const int tok = (row0 + r) / a.group, head = kvh * a.group + (row0 + r - tok * a.group);
        const float* p = a.part + ((int64_t)(at.first + tok) * a.heads + head) * (a.dim + 4);
        const auto join = [&](float unit) {  // what the sum is counted in
            f32x4 sum = {};
            float top = -INFINITY, l = 0.0f;
            for (int i0 = 0; i0 < parts; i0 += 16) {
                f32x4 x[16];
                float2 ml[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i0 + i < parts) {
                        x[i] = *reinterpret_cast<const f32x4*>(p + (i0 + i) * step + 4 * t);
                        ml[i] = *reinterpret_cast<const float2*>(p + (i0 + i) * step + a.dim);
                    }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i0 + i < parts) {  // -inf: no key seen, or none with a score; 0 times what v made of those
                        const float to = ml[i].x > top || ml[i].x != ml[i].x ? ml[i].x : top;
                        const float u = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - to);
                        const float w = ml[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - to);
                        sum = sum * u + x[i] * (w * unit);
                        l = l * u + ml[i].y * w;
                        top = to;
                    }
            }
            return sum / l;
        };
        f32x4 sum = join(1.0f);
        if constexpr (DT != MLXHIP_DTYPE_F16) {
            const f32x4 zero = sum * 0.0f;
            if (__builtin_expect(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.0f), 0)) sum = join(0x1p-44f) * 0x1p44f;
        }
        const bool none = tok + length - at.tokens < 0;
        if (none) sum = f32x4{};
        E* to = (E*)a.o + (int64_t)(at.first + tok) * a.o_stride + (int64_t)head * a.dim + 4 * t;
        if constexpr (DT == MLXHIP_DTYPE_F32) *reinterpret_cast<f32x4*>(to) = sum;
        else *reinterpret_cast<u32x2*>(to) = u32x2{gemm16::pack2<DT>(sum[0], sum[1]), gemm16::pack2<DT>(sum[2], sum[3])};
    }
}

template <int DT, int DP, bool PAGED, bool KEYS>
int launch_fwd(const FwdArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((attn_fwd_kernel<DT, DP, PAGED, KEYS>), dim3((unsigned)(a.items * a.kv_heads), (unsigned)a.splits),
                       dim3(THREADS), 0, s, a);
    MLXHIP_TRY(launch_check("attn_fwd_kernel"));
    if constexpr (!PAGED) return MLXHIP_OK;
    if (a.splits == 1) return MLXHIP_OK;
    hipLaunchKernelGGL((attn_join_kernel<DT, KEYS ? FEW_ROWS : ROW_TILE>), dim3((unsigned)(a.items * a.kv_heads)), dim3(THREADS), 0, s,
                       a);
    return launch_check("attn_join_kernel");
}

template <int DT>
int fwd(const FwdArgs& a, bool paged, bool keys, hipStream_t s) {
    const bool wide = a.dim > 64;
    if (!paged && keys) return wide ? launch_fwd<DT, 128, false, true>(a, s) : launch_fwd<DT, 64, false, true>(a, s);
    if (!paged) return wide ? launch_fwd<DT, 128, false, false>(a, s) : launch_fwd<DT, 64, false, false>(a, s);
    if (keys) return wide ? launch_fwd<DT, 128, true, true>(a, s) : launch_fwd<DT, 64, true, true>(a, s);
    return wide ? launch_fwd<DT, 128, true, false>(a, s) : launch_fwd<DT, 64, true, false>(a, s);
}

}  // namespace attn
}  // namespace mlxhip
