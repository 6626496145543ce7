// ce_gemm.hpp — the matrix products of the linear cross entropy on the 16-bit
// matrix cores, with the loss's row operations in their epilogues.
//
//   CE_STATS  z = x W^T; per tile and row the maximum and the sum of
//             exp(z - max), and the target's logit: the logits leave the
//             registers only as these.
//   CE_DS     z again; dS = exp(z - lse) - [v = target], times the row's
//             dloss, stored as two 16-bit planes (f32 operands: three).
//   CE_DX     f32 sums of dS W over a slice of K, added to those of the
//             pieces of the vocabulary before.
//   CE_DW     dS^T x, in the operands' type.
//   CE_DST    dS^T of up to 16 rows of 16 bits in f32, for ce_few.hip: z as CE_STATS forms
//             it, or p - 1 of a certain target would be the difference.
//
// A plane is a 16-bit value: hi is the f32 value rounded, the next plane what that
// leaves, rounded. The products run over pairs of planes, those whose places add
// up to the last plane's, smallest first.
//
// z of 16-bit operands takes them as they are. z of f32 operands is formed from
// two f16 planes (22 bits) of x and W, each row of either times a power of two that
// brings its largest magnitude to between 2^14 and 2^15: a value keeps 22 bits
// down to 2^-18 of its row's largest, and what is lost below is 2^-39 of that. The
// three products hi hi + hi lo + lo hi leave out less than 2^-22 of a term. That is
// within what f32 sums of some hundred terms are off by anyway.
//
// The gradients of f32 and bf16 operands take bf16 planes, which have f32's range
// and need no scale, so that a row, a vocabulary entry or a dloss of any size keeps
// its digits beside others far larger: dS^T's rows of improbable words are sums of
// values of 2^-40 and less. f32 operands and their dS are three planes (24 bits, six
// products); bf16 operands are read as they are against two planes of dS (16 bits, two
// products). Those of f16 operands take f16 planes: dS without dloss, times
// 2^15, in two (22 bits, a floor of 2^-40), against W as it is (two products; dloss
// follows in dx's last launch) and against two planes of dloss x on one scale (three
// products), whose floor of 2^-40 of the largest is below an f16 result's own.
// Two f16 planes on one scale each for W, x and dloss took half the time for f32
// gradients and lost all digits of what lies 2^-40 below the largest; dS in one
// plane of the operands' type took half the time for 16-bit ones, whose errors beside
// the results' own rounding were as large as that.
//
// Tiles are fed by direct global->LDS loads, STAGES K tiles
// of 32 deep, with the building blocks and LDS layouts of gemm16_impl.hpp; workgroups
// stay and walk over tiles, the next tile's loads on their way during an epilogue
// that has LDS of its own.
//
// Bound by the matrix cores. 2048 rows of 1024 over 32000 (134 GFLOP a product of one
// pair of planes; a library product of 8192^3 reaches 1.17 PFLOP/s), in a trace: bf16
// stats 147 us, dS 187 (262 MB of its planes stored), dx 238 and dW 235 of two pairs
// each (1.13 PFLOP/s); f32 stats 368, dS 429 of three pairs (393 MB stored), dx 637 and
// dW 646 of six (1.25 PFLOP/s). 1000 rows of 777 over 32003, f16: stats 68, dS 87, dx
// 121 of two pairs, dW 162 of three, 0.6 - 0.92 PFLOP/s: 504 tiles of 256 x 256 on 256
// compute units, of 25 steps of K each, so a workgroup's first loads and last epilogue
// weigh more.
#pragma once

#include "elem.hpp"
#include "gemm16_impl.hpp"

namespace mlxhip {
namespace ce {

using gemm16::BK;
using gemm16::f32x16;
using gemm16::f32x4;
using gemm16::u32x2;
using gemm16::u32x4;

enum Product { CE_STATS = 0, CE_DS = 1, CE_DX = 2, CE_DW = 3, CE_DST = 4 };

constexpr float LOG2E = 1.44269504088896340736f;

// WM x WN waves of TM x TN 32x32 tiles, PA planes of A and PB of B in each of
// STAGES stages.
template <int WM_, int WN_, int TM_, int TN_, int STAGES_, int PA_, int PB_>
struct Cfg {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, STAGES = STAGES_, PA = PA_, PB = PB_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;  // one plane of one stage
    static constexpr int STAGE_BYTES = PA * A_BYTES + PB * B_BYTES;     // A's planes, then B's
    static constexpr int LA = A_BYTES / (THREADS * 16), LB = B_BYTES / (THREADS * 16);  // loads per thread and plane
    static_assert(BM >= 128 && BN >= 128, "MN-contiguous LDS rows need >= 16 chunks for the swizzle");
    static_assert(LA * THREADS * 16 == A_BYTES && LB * THREADS * 16 == B_BYTES, "whole 1 KiB blocks per wave");
    // LDS of the epilogue per wave, and workgroups to a compute unit.
    static constexpr int EPI = PA == 1 ? 4096 : 2048;
    static constexpr int LDS = STAGES * STAGE_BYTES + WAVES * EPI, PER_CU = 160 * 1024 / LDS;
    static_assert(STAGES >= 2 && LDS <= 160 * 1024, "LDS budget");
    static_assert(WN * 2 * BM * 4 <= WAVES * EPI, "row statistics of a tile");
};
// The tiles of a product of PA and PB planes: 256 x 256 or, where each operand has
// several planes, 256 x 128; and 128 x 128 (one plane of B: two workgroups to a
// compute unit).
template <int PA, int PB>
struct Tiling;
template <>
struct Tiling<1, 1> {
    using Large = Cfg<2, 4, 4, 2, 4, 1, 1>;
    using Small = Cfg<2, 2, 2, 2, 4, 1, 1>;
};
template <>
struct Tiling<2, 1> {
    using Large = Cfg<4, 2, 2, 4, 3, 2, 1>;
    using Small = Cfg<2, 2, 2, 2, 3, 2, 1>;
};
template <>
struct Tiling<2, 2> {
    using Large = Cfg<4, 2, 2, 2, 3, 2, 2>;
    using Small = Cfg<2, 4, 2, 1, 4, 2, 2>;
};
template <>
struct Tiling<3, 3> {
    using Large = Cfg<4, 2, 2, 2, 2, 3, 3>;
    using Small = Cfg<2, 4, 2, 1, 3, 3, 3>;
};

// The pairs of planes of a product, smallest first: of PA and PB planes those with
// i + j < PA.
template <int PA, int PB>
struct Pairs {
    int n = 0, a[6] = {}, b[6] = {};
    constexpr Pairs() {
        for (int sum = PA - 1; sum >= 0; --sum)
            for (int i = sum; i >= 0; --i)
                if (sum - i < PB) {
                    a[n] = i;
                    b[n] = sum - i;
                    ++n;
                }
    }
};

// Planes of the operands in the logits' product and their type; of dS, x and W in the
// gradients' and their type.
template <int OT>
constexpr int Z_PLANES = OT == MLXHIP_DTYPE_F32 ? 2 : 1;
template <int OT>
constexpr int Z_TYPE = OT == MLXHIP_DTYPE_F32 ? MLXHIP_DTYPE_F16 : OT;
template <int OT>
constexpr int DS_PLANES = OT == MLXHIP_DTYPE_F32 ? 3 : 2;
template <int OT>
constexpr int X_PLANES = OT == MLXHIP_DTYPE_F32 ? 3 : OT == MLXHIP_DTYPE_F16 ? 2 : 1;
template <int OT>
constexpr int W_PLANES = OT == MLXHIP_DTYPE_F32 ? 3 : 1;
template <int OT>
constexpr int G_TYPE = OT == MLXHIP_DTYPE_F16 ? MLXHIP_DTYPE_F16 : MLXHIP_DTYPE_BF16;
// dS of f16 operands is without dloss and times this.
constexpr float DS_F16 = 0x1p15f;

struct Args {
    // op(A) [m, k], op(B) [k, n]; planes of an operand *_plane elements apart.
    const uint16_t *a = nullptr, *b = nullptr;
    int64_t lda = 0, ldb = 0, a_plane = 0, b_plane = 0;
    int64_t m = 0, n = 0;
    int64_t ka = 0, kb = 0;  // K extent of each operand's memory; zeros beyond
    int tiles_m = 0, tiles_n = 0;
    int splits = 1;          // CE_DX: slices of K, of k_chunk (a multiple of 32) each
    int64_t k_chunk = 0;
    // Of each row of x: its target, and for CE_DS the forward's lse, dloss and, of f32
    // operands, its loss or null (p - 1 of the target is then made from that).
    const int32_t* targets = nullptr;
    int64_t v0 = 0, vocab = 0;  // the piece's first column, the whole vocabulary
    const float *lse = nullptr, *dloss = nullptr, *loss = nullptr;
    float2* stats = nullptr;    // CE_STATS: [tiles of columns][m], from this launch's first tile on
    float* target_z = nullptr;  // CE_STATS: [m]
    uint16_t* ds = nullptr;     // CE_DS: [DS_PLANES][m][ldc]
    float* dst = nullptr;       // CE_DST: [n][16]
    float* dx = nullptr;        // CE_DX: [splits][m][ldc]
    bool add = false;           // CE_DX: add to what is there
    void* dw = nullptr;         // CE_DW: [m][ldc]
    // z of planes: x's row r is row_scale[r] times its planes, W's row v
    // col_scale[v - v0] times its (room for a multiple of 256 columns).
    const float *row_scale = nullptr, *col_scale = nullptr;
    const float* scale = nullptr;  // CE_DW of f16 operands: dW is *scale times the product
    int64_t ldc = 0;
};

// Few rows (ce_few.hip, with what each bound measured): the loss of up to 128 f32
// rows, or 64 of 16 bits where the tiles would need a copy of W; the gradients of up
// to 64 f32 rows, or 16 of 16 bits. Where only the loss is formed there, it leaves dS of
// more rows to the tiles as CE_DS does: z has to be the same in both. What they keep of
// each entry stays within FEW_BYTES (the statistics of its 64th, the row of dS^T), and
// their launches, four work items to an entry and block of 64 rows, within the 2^32
// that a dispatch counts.
constexpr int64_t FEW_BYTES = int64_t(1) << 30, FEW_ENTRIES = int64_t(1) << 29;
inline int64_t few_ds_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
inline bool few_loss(int dt, bool copy_w, int64_t rows, int64_t vocab) {
    return copy_w && rows <= (dt == MLXHIP_DTYPE_F32 ? 128 : 64) && vocab / 64 * rows * 8 <= FEW_BYTES && vocab <= FEW_ENTRIES;
}
inline bool few_grad(int dt, int64_t rows, int64_t vocab) {
    return rows <= (dt == MLXHIP_DTYPE_F32 ? 64 : 16) && vocab * few_ds_rows(rows) * 4 <= FEW_BYTES;
}
struct FewArgs {
    const void *x = nullptr, *w = nullptr;
    int64_t rows = 0, dim = 0, vocab = 0;
    const int32_t* targets = nullptr;
    const float *lse = nullptr, *dloss = nullptr, *loss = nullptr;
    float2* stats = nullptr;    // [ce_few_tiles()][rows]
    float* target_z = nullptr;
    float* ds = nullptr;        // dS^T [vocab][few_ds_rows(rows)]
    bool form_ds = true;        // or it is there
    float* dx = nullptr;        // [slices][rows][ldx] or null
    void* dw = nullptr;         // [vocab][dim] or null
    int64_t ldx = 0, slices = 0, slice = 0;  // of 4 * slice entries each; slice a multiple of 16
    // dS as CE_DS leaves it instead, of the entries `first` on of `whole`: planes of
    // [rows][ldc], `plane` elements apart.
    uint16_t* planes = nullptr;
    int64_t ldc = 0, plane = 0, first = 0, whole = 0;
};

// Max and sum of exp(z - max) of two groups of a row.
__device__ inline void merge(float& m, float& s, float m2, float s2) {
    const float mn = fmaxf(m, m2);
    const float base = mn == -INFINITY ? 0.0f : mn;
    s = s * __builtin_amdgcn_exp2f((m - base) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - base) * LOG2E);
    m = mn;
}

__device__ inline bool counted(int32_t target, int64_t vocab) { return target >= 0 && target < vocab; }

// A target's place from column v on, -1 where it is not among `width` of them.
__device__ inline int column_of(int32_t target, int64_t v, int width) {
    const int64_t c = target - v;
    return c >= 0 && c < width ? (int)c : -1;
}

// A workgroup's tiles: consecutive workgroup ids go to the 8 XCDs in turn, so
// each XCD takes a contiguous range of tiles, which its workgroups share out one
// by one; a range runs through groups of four tile rows.
struct Tiles {
    int at, end, step;
    __device__ inline Tiles(int total) {
        const int xcd = blockIdx.x & 7, per = total >> 3, rest = total & 7;
        const int first = xcd * per + min(xcd, rest);
        at = first + (blockIdx.x >> 3);
        end = first + per + (xcd < rest);
        step = gridDim.x >> 3;
    }
};
struct Tile {
    int64_t m0, n0, k0, ka, kb;
    int split;
};
template <int PRODUCT, class C>
__device__ inline Tile tile_of(const Args& g, int lin) {
    Tile t;
    const int nwg = g.tiles_m * g.tiles_n;
    t.split = PRODUCT == CE_DX ? lin / nwg : 0;
    const int id = lin - t.split * nwg;
    constexpr int GROUP_M = 4;
    const int in_group = GROUP_M * g.tiles_n, first = id / in_group * GROUP_M;
    const int rows = min(g.tiles_m - first, GROUP_M);
    t.m0 = (int64_t)(first + id % in_group % rows) * C::BM;
    t.n0 = (int64_t)(id % in_group / rows) * C::BN;
    t.k0 = PRODUCT == CE_DX ? t.split * g.k_chunk : 0;
    const int64_t most = PRODUCT == CE_DX && g.splits > 1 ? g.k_chunk : INT64_MAX;
    t.ka = min(g.ka - t.k0, most);
    t.kb = min(g.kb - t.k0, most);
    return t;
}

// Descriptor of an operand's part that the tile at row / column r0 (of R) and
// k from k0 on reads. KC: [R][k] in memory, else [k][R] with rows of ld.
template <bool KC, int ROWS, int P>
__device__ inline __amdgpu_buffer_rsrc_t operand(const uint16_t* p, int64_t plane, int64_t ld, int64_t r0, int64_t R,
                                                 int64_t k0, int64_t k) {
    const uint16_t* at = p + (KC ? r0 * ld + k0 : k0 * ld + r0);
    const int64_t rows = min(R - r0, (int64_t)ROWS);
    const int64_t ext = (KC ? (rows - 1) * ld + k : (k - 1) * ld + min((rows + 7) / 8 * 8, ld - r0)) + (P - 1) * plane;
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, (int)(uint32_t)(ext * 2), gemm16::BUF_FLAGS);
}

// Stores the tile of values acc through the wave's LDS region (C::EPI bytes),
// whole row segments at a time: 16-byte vectors at any element alignment where
// they end before column `cap`, single elements up to column n else. 16-byte
// chunks of a region's row are permuted by its place among the rows that share
// 256 bytes' worth of banks. ACC (f32): added to what is there.
template <int CT, class C, bool ACC, bool NT>
__device__ inline void store_tile(const f32x16 (&acc)[C::TM][C::TN], MLXHIP_LDS char* region, typename dev::Elem<CT>::type* out,
                                  int64_t ld, int64_t m, int64_t n, int64_t cap, int64_t row0, int64_t col0, int lane,
                                  bool add) {
    typedef typename dev::Elem<CT>::type T;
    typedef uint32_t any __attribute__((ext_vector_type(4), aligned(2)));  // at any element
    constexpr int TM = C::TM, TN = C::TN, ES = sizeof(T), VEC = 16 / ES;
    constexpr int ROW_BYTES = 32 * TN * ES, CHUNKS = ROW_BYTES / 16, SHARE = CHUNKS >= 16 ? 1 : 16 / CHUNKS;
    constexpr int PASS = C::EPI / ROW_BYTES < 32 ? C::EPI / ROW_BYTES : 32;  // rows staged at a time
    constexpr int ROWS = 64 / CHUNKS;
    static_assert(32 % PASS == 0 && PASS % ROWS == 0, "epilogue passes");
    auto place = [](int r, int chunk) { return r * ROW_BYTES + ((chunk ^ ((r / SHARE) & (CHUNKS - 1))) * 16); };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int h = 0; h < 32 / PASS; ++h) {
            if (PASS == 32 || (lane & 31) / PASS == h) {
                const int r = lane & (PASS - 1);
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int b = (32 * j + 8 * q + 4 * (lane >> 5)) * ES;
                        MLXHIP_LDS char* p = region + place(r, b / 16) + b % 16;
                        const f32x16& a = acc[i][j];
                        if constexpr (ES == 4)
                            *(MLXHIP_LDS f32x4*)p = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                        else
                            *(MLXHIP_LDS u32x2*)p = u32x2{gemm16::pack2<CT>(a[4 * q], a[4 * q + 1]),
                                                          gemm16::pack2<CT>(a[4 * q + 2], a[4 * q + 3])};
                    }
            }
            // Read back by other lanes of the same wave: its LDS accesses complete
            // in order, so only the compiler has to keep them in it.
            asm volatile("" ::: "memory");
#pragma unroll
            for (int rr = 0; rr < PASS; rr += ROWS) {
                const int r = rr + lane / CHUNKS, chunk = lane % CHUNKS;
                u32x4 v = *(const MLXHIP_LDS u32x4*)(region + place(r, chunk));
                const int64_t row = row0 + 32 * i + h * PASS + r, col = col0 + chunk * VEC;
                if (row >= m || col >= n) continue;
                T* dst = out + row * ld + col;
                if (col + VEC <= cap) {
                    if constexpr (ACC) {
                        if (add) {
                            const u32x4 had = *reinterpret_cast<const u32x4*>(dst);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[e] = __float_as_uint(__uint_as_float(had[e]) + __uint_as_float(v[e]));
                        }
                    }
                    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<any*>(dst));
                    else *reinterpret_cast<any*>(dst) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        if (col + e >= n) break;
                        if constexpr (ES == 4) dst[e] = __uint_as_float(v[e]);
                        else dst[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
                    }
                }
            }
            asm volatile("" ::: "memory");
        }
}

// acc's columns times col_scale (from the lane's first column on).
template <int TM, int TN>
__device__ inline void scale_columns(f32x16 (&acc)[TM][TN], const float* col_scale) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 c = *reinterpret_cast<const f32x4*>(col_scale + 32 * j + 8 * q);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] *= c[e];
        }
}

// MT: type of the operands' planes (BF16, F16); OT: type of the operator's operands.
//
// A workgroup runs through its tiles without draining its loads: behind a
// tile's last K tile come the first of the next one, which land while the
// epilogue runs (it has LDS of its own).
template <int PRODUCT, int MT, int OT, class C>
__global__ __attribute__((amdgpu_flat_work_group_size(C::THREADS, C::THREADS), amdgpu_waves_per_eu(2, 2)))
void ce_gemm_kernel(Args g) {
    constexpr bool KCA = PRODUCT != CE_DW, KCB = PRODUCT <= CE_DS || PRODUCT == CE_DST;
    constexpr int STAGES = C::STAGES, TM = C::TM, TN = C::TN, WAVES = C::WAVES, PA = C::PA, PB = C::PB;
    constexpr Pairs<PA, PB> pairs;
    __shared__ __attribute__((aligned(1024))) char smem_raw[STAGES * C::STAGE_BYTES + WAVES * C::EPI];
    MLXHIP_LDS char* smem = (MLXHIP_LDS char*)smem_raw;
    MLXHIP_LDS char* epi = smem + STAGES * C::STAGE_BYTES;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN;
    const uint32_t plane_a = (uint32_t)(g.a_plane * 2), plane_b = (uint32_t)(g.b_plane * 2);
    constexpr int ROWB_A = C::BM * 2, ROWB_B = C::BN * 2;
    gemm16::FragAddr<KCA, TM, ROWB_A> fa;
    gemm16::FragAddr<KCB, TN, ROWB_B> fb;
    fa.init(lane, 32 * TM * wm);
    fb.init(lane, 32 * TN * wn);

    // What is loaded next: K tile `lk` of the tile at `lat` of the list; past
    // the list's end, loads that no chunk is in range of.
    const Tiles list(g.tiles_m * g.tiles_n * (PRODUCT == CE_DX ? g.splits : 1));
    if (list.at >= list.end) return;
    gemm16::Loader<KCA, C::BM, WAVES> la;
    gemm16::Loader<KCB, C::BN, WAVES> lb;
    __amdgpu_buffer_rsrc_t ra, rb;
    int lat = list.at, lk = 0, lnk = 0;
    auto seek = [&] {
        const Tile t = tile_of<PRODUCT, C>(g, lat);
        ra = operand<KCA, C::BM, PA>(g.a, g.a_plane, g.lda, t.m0, g.m, t.k0, t.ka);
        rb = operand<KCB, C::BN, PB>(g.b, g.b_plane, g.ldb, t.n0, g.n, t.k0, t.kb);
        la.init(tid, 0, g.m - t.m0, g.lda, t.ka);
        lb.init(tid, 0, g.n - t.n0, g.ldb, t.kb);
        lk = 0;
        lnk = (int)((max(t.ka, t.kb) + BK - 1) / BK);
    };
    auto next = [&] {
        if (++lk < lnk || lat >= list.end) return;
        lat += list.step;
        if (lat < list.end) seek();
    };
    auto next_k = [&] { return lat < list.end ? lk * BK : INT32_MAX; };
    seek();

    constexpr int LA = C::LA, LB = C::LB, LPT = PA * LA + PB * LB, B0 = PA * C::A_BYTES;
#pragma unroll
    for (int t = 0; t < STAGES; ++t) {
        MLXHIP_LDS char* st = smem + t * C::STAGE_BYTES;
        const int k = next_k();
#pragma unroll
        for (int p = 0; p < PA; ++p) la.issue(ra, st + p * C::A_BYTES, wave, k, (uint32_t)p * plane_a);
#pragma unroll
        for (int p = 0; p < PB; ++p) lb.issue(rb, st + B0 + p * C::B_BYTES, wave, k, (uint32_t)p * plane_b);
        next();
    }
    gemm16::wait_vmcnt<(STAGES - 1) * LPT>();
    gemm16::lds_barrier();

    constexpr int NA = KCA ? TM : 2 * TM, NB = KCB ? TN : 2 * TN, NR = PA * NA + PB * NB;
    u32x4 af[2][PA][TM], bf[2][PB][TN];
    auto read_op = [&](const MLXHIP_LDS char* st, int s, int o) {
        if (o < PA * NA) {
            const int p = o / NA;
            gemm16::read_one<KCA, TM, ROWB_A>(st + p * C::A_BYTES, fa, s, o - p * NA, af[s][p]);
        } else {
            const int ob = o - PA * NA, p = ob / NB;
            gemm16::read_one<KCB, TN, ROWB_B>(st + B0 + p * C::B_BYTES, fb, s, ob - p * NB, bf[s][p]);
        }
    };
#pragma unroll
    for (int o = 0; o < NR; ++o) read_op(smem, 0, o);

    int cur = 0;  // stage of the K tile at hand
    for (int at = list.at; at < list.end; at += list.step) {
        const Tile tile = tile_of<PRODUCT, C>(g, at);
        const int nk = (int)((max(tile.ka, tile.kb) + BK - 1) / BK);
        f32x16 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

        // Per K tile two steps of 16: each step's MFMAs with the next step's LDS
        // reads, and in the second the loads of the K tile STAGES on, between them.
        constexpr int NM = TM * TN, NMI = pairs.n * NM, OPS = NR + LPT;
        for (int kt = 0; kt < nk; ++kt) {
            const MLXHIP_LDS char* st = smem + cur * C::STAGE_BYTES;
#pragma unroll
            for (int q = 0; q < NMI; ++q) {
                const int e = q / NM, t = q % NM;
                gemm16::mfma<MT>(bf[0][pairs.b[e]][t % TN], af[0][pairs.a[e]][t / TN], acc[t / TN][t % TN]);
                constexpr bool ONE = NR <= NMI;  // a read a step, the first ones first
#pragma unroll
                for (int o = ONE ? min(q, NR) : (q * NR) / NMI; o < (ONE ? min(q + 1, NR) : ((q + 1) * NR) / NMI); ++o)
                    read_op(st, 1, o);
                __builtin_amdgcn_sched_barrier(0);
            }
            // The next K tile has landed for every wave (stores of an epilogue in
            // between only make the wait longer); every wave has read this one's
            // stage, which then receives the K tile STAGES on.
            gemm16::wait_vmcnt<(STAGES - 2) * LPT>();
            gemm16::lds_barrier();
            MLXHIP_LDS char* dst = smem + cur * C::STAGE_BYTES;
            cur = cur + 1 == STAGES ? 0 : cur + 1;
            const MLXHIP_LDS char* nx = smem + cur * C::STAGE_BYTES;
            const int kl = next_k();
#pragma unroll
            for (int q = 0; q < NMI; ++q) {
                const int e = q / NM, t = q % NM;
                gemm16::mfma<MT>(bf[1][pairs.b[e]][t % TN], af[1][pairs.a[e]][t / TN], acc[t / TN][t % TN]);
#pragma unroll
                for (int o = (q * OPS) / NMI; o < ((q + 1) * OPS) / NMI; ++o) {
                    if (o < NR) {
                        read_op(nx, 0, o);
                    } else if (o < NR + PA * LA) {
                        const int p = (o - NR) / LA;
                        la.issue_one(ra, dst + p * C::A_BYTES, wave, kl, o - NR - p * LA, (uint32_t)p * plane_a);
                    } else {
                        const int ob = o - NR - PA * LA, p = ob / LB;
                        lb.issue_one(rb, dst + B0 + p * C::B_BYTES, wave, kl, ob - p * LB, (uint32_t)p * plane_b);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            next();
        }

        // acc[i][j][4 q + e] is row 32 i + lane % 32, column 32 j + 8 q +
        // 4 (lane / 32) + e of the wave's part.
        const int64_t m0 = tile.m0, n0 = tile.n0, wrow = m0 + 32 * TM * wm, wcol = n0 + 32 * TN * wn;
        const int64_t row0 = wrow + (lane & 31), col0 = wcol + 4 * (lane >> 5);
        MLXHIP_LDS char* region = epi + wave * C::EPI;
        if constexpr (PRODUCT == CE_STATS) {
            MLXHIP_LDS float* red = (MLXHIP_LDS float*)epi;  // [WN][2][BM]
            const bool edge = n0 + C::BN > g.n;
            if constexpr (PA > 1) scale_columns(acc, g.col_scale + col0);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t r = row0 + 32 * i;
                const float f = PA == 1 || r >= g.m ? 1.0f : g.row_scale[r];
                // The target's logit, from the lane that holds its column.
                const int tc = r < g.m ? column_of(g.targets[r], g.v0 + col0, 32 * TN) : -1;
                const bool mine = tc >= 0 && (tc & 4) == 0 && tc + col0 < g.n;
                if (__ballot(mine)) {
                    float z = 0.0f;
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (tc == 32 * j + 8 * (v >> 2) + (v & 3)) z = acc[i][j][v];
                    if (mine) g.target_z[r] = z * f;
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (col0 + 32 * j + 8 * (v >> 2) + (v & 3) >= g.n) acc[i][j][v] = -INFINITY;
                }
                float mx = acc[i][0][0];
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, acc[i][j][v]);
                // exp(z - mx) as exp2(z log2 e - mb), mb = mx log2 e rounded; what
                // that rounding leaves is put right in the sum.
                const float base = mx == -INFINITY ? 0.0f : mx, up = LOG2E * f;
                const float mb = base * up;
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v) s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][v], up, -mb));
                s *= __builtin_amdgcn_exp2f(__builtin_fmaf(-base, up, mb));
                mx *= f;
                merge(mx, s, __shfl_xor(mx, 32, 64), __shfl_xor(s, 32, 64));
                if (lane < 32) {
                    MLXHIP_LDS float* p = red + 2 * wn * C::BM + 32 * TM * wm + 32 * i + lane;
                    p[0] = mx;
                    p[C::BM] = s;
                }
            }
            gemm16::lds_barrier();
            if (tid < C::BM && m0 + tid < g.m) {
                float2 a = make_float2(red[tid], red[C::BM + tid]);
#pragma unroll
                for (int w = 1; w < C::WN; ++w) merge(a.x, a.y, red[2 * w * C::BM + tid], red[(2 * w + 1) * C::BM + tid]);
                g.stats[n0 / C::BN * g.m + m0 + tid] = a;
            }
        } else if constexpr (PRODUCT == CE_DS || PRODUCT == CE_DST) {
            if constexpr (PA > 1) scale_columns(acc, g.col_scale + col0);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t r = row0 + 32 * i;
                float shift = 0.0f, f = 0.0f, fix = 1.0f, up = LOG2E;
                int tc = -1;
                if (r < g.m) {
                    const int32_t t = g.targets[r];
                    if (counted(t, g.vocab)) {
                        shift = -g.lse[r] * LOG2E;
                        f = OT == MLXHIP_DTYPE_F16 && PRODUCT == CE_DS ? DS_F16 : g.dloss[r];
                        // What the rounding of shift leaves: near a certain target it would be
                        // most of p - 1.
                        fix = __builtin_amdgcn_exp2f(__builtin_fmaf(-g.lse[r], LOG2E, -shift));
                    }
                    if constexpr (PA > 1) up *= g.row_scale[r];
                    tc = column_of(t, g.v0 + col0, 32 * TN);
                }
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        acc[i][j][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][v], up, shift)) * (f * fix);
                if (__ballot(tc >= 0)) {  // some lane holds its row's target
                    const bool known = OT == MLXHIP_DTYPE_F32 && g.loss;
                    const float hit = known && tc >= 0 ? expm1f(-g.loss[r]) * f : 0.0f;
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (tc == 32 * j + 8 * (v >> 2) + (v & 3)) acc[i][j][v] = known ? hit : acc[i][j][v] - f;
                }
                // A row without a target has no dS, whatever x, lse and dloss hold.
                const bool on = r < g.m && counted(g.targets[r], g.vocab);
                if (__ballot(!on)) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v) acc[i][j][v] = on ? acc[i][j][v] : 0.0f;
                }
            }
            if constexpr (PRODUCT == CE_DST) {
                if (row0 < 16) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            const int64_t c = col0 + 32 * j + 8 * (v >> 2) + (v & 3);
                            if (c < g.n) g.dst[c * 16 + row0] = acc[0][j][v];
                        }
                }
                continue;
            }
            if (n0 + C::BN > g.n) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (col0 + 32 * j + 8 * (v >> 2) + (v & 3) >= g.n)
#pragma unroll
                            for (int i = 0; i < TM; ++i) acc[i][j][v] = 0.0f;
            }
            constexpr int GT = G_TYPE<OT>, SP = DS_PLANES<OT>;
#pragma unroll
            for (int p = 0; p < SP; ++p) {
                store_tile<GT, C, false, false>(acc, region, g.ds + p * g.m * g.ldc, g.ldc, g.m, g.ldc, g.ldc, wrow, wcol,
                                                  lane, false);
                if (p + 1 < SP) {
                    // What the plane leaves (exact in f32).
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
#pragma unroll
                            for (int v = 0; v < 16; ++v)
                                acc[i][j][v] -= dev::to_f32<GT>(dev::from_f32<GT>(acc[i][j][v]));
                }
            }
        } else if constexpr (PRODUCT == CE_DW) {
            if constexpr (OT == MLXHIP_DTYPE_F16) {
                const float f = *g.scale;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int v = 0; v < 16; ++v) acc[i][j][v] *= f;
            }
            store_tile<OT, C, false, true>(acc, region, static_cast<typename dev::Elem<OT>::type*>(g.dw), g.ldc, g.m, g.n, g.n,
                                           wrow, wcol, lane, false);
        } else {
            store_tile<MLXHIP_DTYPE_F32, C, true, false>(acc, region, g.dx + tile.split * g.m * g.ldc, g.ldc, g.m, g.n, g.ldc,
                                                         wrow, wcol, lane, g.add);
        }
    }
    // The loads past the last tile write (zeros) to this workgroup's LDS.
    gemm16::wait_vmcnt<0>();
}

template <int PRODUCT, int MT, int OT, class C>
int launch(Args a, hipStream_t s) {
    a.tiles_m = (int)ceil_div(a.m, C::BM);
    a.tiles_n = (int)ceil_div(a.n, C::BN);
    // One workgroup for each place on the chip (a multiple of the 8 XCDs), or
    // for each tile if those are fewer.
    const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n * a.splits;
    const int64_t groups = std::min<int64_t>(ceil_div(tiles, 8) * 8, 256 * C::PER_CU);
    hipLaunchKernelGGL((ce_gemm_kernel<PRODUCT, MT, OT, C>), dim3((unsigned)groups), dim3(C::THREADS), 0, s, a);
    return launch_check("ce_gemm_kernel");
}

// The product's large or small tiles.
template <int PRODUCT, int MT, int OT, int PA, int PB>
int product(bool large, const Args& a, hipStream_t s) {
    return large ? launch<PRODUCT, MT, OT, typename Tiling<PA, PB>::Large>(a, s)
                 : launch<PRODUCT, MT, OT, typename Tiling<PA, PB>::Small>(a, s);
}

template <int OT>
int dispatch(int which, bool large, const Args& a, hipStream_t s) {
    constexpr int ZP = Z_PLANES<OT>, ZT = Z_TYPE<OT>, SP = DS_PLANES<OT>, GT = G_TYPE<OT>;
    switch (which) {
        case CE_STATS: return product<CE_STATS, ZT, OT, ZP, ZP>(large, a, s);
        case CE_DS: return product<CE_DS, ZT, OT, ZP, ZP>(large, a, s);
        case CE_DST:
            if constexpr (OT != MLXHIP_DTYPE_F32) return product<CE_DST, ZT, OT, ZP, ZP>(large, a, s);
            return fail(MLXHIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy: no dS^T of f32 tiles");
        case CE_DX: return product<CE_DX, GT, OT, SP, W_PLANES<OT>>(large, a, s);
        default: return product<CE_DW, GT, OT, SP, X_PLANES<OT>>(large, a, s);
    }
}

}  // namespace ce

// ce_bf16.hip, ce_f16.hip, ce_f32.hip: the products of operands of each type.
int ce_gemm_bf16(int which, bool large, const ce::Args& a, hipStream_t s);
int ce_gemm_f16(int which, bool large, const ce::Args& a, hipStream_t s);
int ce_gemm_f32(int which, bool large, const ce::Args& a, hipStream_t s);
// ce_few.hip
int ce_few_planes(int dt, const ce::FewArgs& g, hipStream_t s);
int ce_few_loss(int dt, const ce::FewArgs& g, hipStream_t s);
int ce_few_grad(int dt, const ce::FewArgs& g, hipStream_t s);
int64_t ce_few_tiles(int dt, int64_t rows, int64_t vocab);  // of the loss's statistics

}  // namespace mlxhip
