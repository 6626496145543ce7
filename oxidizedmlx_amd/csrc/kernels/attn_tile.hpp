// attn_tile.hpp — tiles of attention over packed sequences: rows of a head in LDS,
// the matrix fragments read from them, and which rows a workgroup has.
//
// Every product is 32 x 32 outputs a wave and 16 of the inner index a step:
// v_mfma_f32_32x32x16 for 16-bit operands, eight v_mfma_f32_32x32x2 for f32. Of a
// step's operand a lane (half h = lane / 32) holds eight inner values of row or
// column lane % 32. Which eight is free as long as both operands agree:
//   along a row of LDS     8 h + (0..7): 16-byte reads;
//   against a product's    4 h + (0..3), 8 + 4 h + (0..3): an accumulator's
//   own result             registers 8 s .. 8 s + 7 hold rows 16 s + those.
// So the scores are formed transposed where their rows are what the next product
// sums over, and go from accumulator to operand with no exchange between lanes.
//
// LDS: a row of DP values (head_dim rounded up to 64 or 128, zeros behind), chunk c of 16
// bytes at c ^ swizzle(row). Row reads (lane = row, one chunk) then spread 16
// rows over all banks, and the transposed reads (ds_read_b64_tr_b16: 4 rows x 64
// bytes; f32: 32 values of one row) do too. The swizzle is applied by which
// chunk a lane fetches; loads go straight from memory to LDS, 1 KiB to an instruction,
// and chunks past the head or past the last row are zeros by the buffer's bounds.
#pragma once

#include "elem.hpp"
#include "gemm16_impl.hpp"

namespace mlxhip {
namespace attn {

using gemm16::f32x16;
using gemm16::f32x4;
using gemm16::u32x2;
using gemm16::u32x4;

constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <int DT>
constexpr int ELEM = DT == MLXHIP_DTYPE_F32 ? 4 : 2;

template <int DT>
struct Frag {  // eight inner values
    u32x4 q[DT == MLXHIP_DTYPE_F32 ? 2 : 1];
};

template <int DT>
__device__ inline void mma(const Frag<DT>& a, const Frag<DT>& b, f32x16& acc) {
    if constexpr (DT == MLXHIP_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.q[j / 4][j % 4]), __uint_as_float(b.q[j / 4][j % 4]),
                                                       acc, 0, 0, 0);
    } else {
        gemm16::mfma<DT>(a.q[0], b.q[0], acc);
    }
}

// Registers 8 s .. 8 s + 7 of an accumulator as an operand.
template <int DT>
__device__ inline Frag<DT> frag_of(const float* v) {
    Frag<DT> f;
    if constexpr (DT == MLXHIP_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f.q[j / 4][j % 4] = __float_as_uint(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) f.q[0][j] = gemm16::pack2<DT>(v[2 * j], v[2 * j + 1]);
    }
    return f;
}

// What frag_of rounds off: v less the operand, as another operand.
template <int DT>
__device__ inline Frag<DT> rest_of(const float* v, const Frag<DT>& f) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r[2 * j] = v[2 * j] - dev::to_f32<DT>((uint16_t)f.q[0][j]);
        r[2 * j + 1] = v[2 * j + 1] - dev::to_f32<DT>((uint16_t)(f.q[0][j] >> 16));
    }
    return frag_of<DT>(r);
}

// The non-finite values of f as ones, zeros elsewhere; f is left with zeros in their place.
template <int DT>
__device__ inline Frag<DT> take_non_finite(Frag<DT>& f) {
    Frag<DT> bad;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(f) / 16); ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t ones = 0;
            if constexpr (DT == MLXHIP_DTYPE_F32) {
                const bool b = (f.q[i][j] & 0x7F800000u) == 0x7F800000u;
                ones = b ? 0x3F800000u : 0u;
                f.q[i][j] = b ? 0u : f.q[i][j];
            } else {
                constexpr uint32_t EXP = DT == MLXHIP_DTYPE_BF16 ? 0x7F80u : 0x7C00u, ONE = DT == MLXHIP_DTYPE_BF16 ? 0x3F80u : 0x3C00u;
#pragma unroll
                for (int k = 0; k < 32; k += 16)
                    if ((f.q[i][j] >> k & EXP) == EXP) {
                        ones |= ONE << k;
                        f.q[i][j] &= ~(0xFFFFu << k);
                    }
            }
            bad.q[i][j] = ones;
        }
    return bad;
}

// N products whose operands from LDS are read DEPTH ahead: read(i) gives product i's fragment, use(i, f)
// forms it. Left alone the compiler reads a fragment into the registers of the one before and waits for
// it every time.
template <int DT, int N, int DEPTH, class Read, class Use>
__device__ inline void stream(Read&& read, Use&& use) {
    constexpr int D = DEPTH < N ? DEPTH : N;
    Frag<DT> f[D];
#pragma unroll
    for (int i = 0; i < D; ++i) f[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, f[i % D]);
        if (i + D < N) {
            f[i % D] = read(i + D);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// A tile of ROWS rows of a head in LDS.
template <int DT, int DP, int ROWS>
struct Tile {
    static constexpr int ROWB = DP * ELEM<DT>;       // bytes of a row
    static constexpr int CPR = ROWB / 16;            // its chunks
    static constexpr int RPI = 64 / CPR;             // rows of one load instruction
    static constexpr int BYTES = ROWS * ROWB;
    static constexpr int INSTR = ROWS / RPI;         // load instructions
    static_assert(CPR >= 8 && CPR <= 32 && INSTR >= 1, "row of 128 to 512 bytes");

    __device__ static inline int swizzle(int row) {
        if constexpr (CPR == 8) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);  // two rows to 256 bytes
        else return (row & 3) << 2 | ((row >> 2) & 3);
    }
};

// p and bytes are the same in all lanes; arithmetic on them may have gone through
// vector registers, the descriptor is scalar. A scalar register that the vector unit
// writes takes five cycles to reach a memory instruction: the compiler counts them for its own
// instructions only, and the asm loads below would go by the old descriptor.
__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)((uint64_t)hi << 32 | lo), 0,
                                                                 __builtin_amdgcn_readfirstlane(bytes), gemm16::BUF_FLAGS);
    asm volatile("s_nop 4" : "+s"(r));
    return r;
}

// 16 or 4 bytes per lane from buffer offset voff to LDS at dst + 16 or 4 * lane (M0's wait in front).
__device__ inline void lds_load16(__amdgpu_buffer_rsrc_t rsrc, MLXHIP_LDS char* dst, uint32_t voff) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(m0) : "memory");
}
__device__ inline void lds_load4(__amdgpu_buffer_rsrc_t rsrc, MLXHIP_LDS char* dst, uint32_t voff) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(m0) : "memory");
}

// One wave's loads of a tile that LW waves share. voff: the lane's offset, past any buffer where
// the chunk is past the head.
//   TILE   rows one after another in memory, one descriptor: an offset for each instruction, from
//          the tile's first row.
//   PAGES  16 rows (which lie in one page) to a descriptor, a wave's instructions side by side, so that
//          it has one or two: an offset for each instruction of 16 rows, from the first of them.
//   LEAN   rows one after another, one descriptor: the swizzle comes round after 16 rows, so that one or
//          two offsets, and an addition for each instruction, serve all where registers are short.
enum LoadMode { TILE, PAGES, LEAN };
template <int DT, int DP, int ROWS, int LW, int MODE>
struct TileLoader {
    using T = Tile<DT, DP, ROWS>;
    static constexpr int L = T::INSTR / LW;  // instructions of a wave
    static constexpr int STEP = (MODE == PAGES ? 1 : LW) * T::RPI, PER16 = STEP >= 16 ? 1 : 16 / STEP;
    static constexpr int ROUND = MODE == TILE || L < PER16 ? L : PER16;
    static_assert(L * LW == T::INSTR && (16 % STEP == 0 || STEP % 16 == 0), "whole instructions to a wave");
    // Past any buffer: LEAN's with a row's offset added too, which must not come round (a tile is 2^27
    // bytes at most: strides up to 2^20 elements, 64 rows of 16 bits, 32 of f32).
    static constexpr uint32_t PAST = MODE == LEAN ? 0x80000000u : gemm16::OOB;
    uint32_t voff[ROUND];
    __device__ static inline int instr(int wave, int i) { return MODE == PAGES ? wave * L + i : i * LW + wave; }
    __device__ inline void init(int wave, int lane, int dim, uint32_t stride_bytes) {
#pragma unroll
        for (int i = 0; i < ROUND; ++i) {
            const int row = instr(wave, i) * T::RPI + lane / T::CPR, c = lane % T::CPR ^ T::swizzle(row);
            voff[i] = c * 16 < dim * ELEM<DT> ? (uint32_t)(MODE == TILE ? row : row % 16) * stride_bytes + c * 16 : PAST;
        }
    }
    // TILE, LEAN: `left` rows (1 or more) from p on, stride_bytes apart; zeros behind them.
    __device__ inline void rows(const char* p, int left, uint32_t stride_bytes, MLXHIP_LDS char* tile, int wave) const {
        const __amdgpu_buffer_rsrc_t rsrc = buffer(p, (uint32_t)max(0, min(left, ROWS)) * stride_bytes);
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const uint32_t at = MODE == TILE ? 0 : (uint32_t)(instr(wave, i) * T::RPI & ~15) * stride_bytes;
            lds_load16(rsrc, tile + instr(wave, i) * 1024, voff[i % ROUND] + at);
        }
    }
    // PAGES: at(r, &bytes): where rows r .. r + 15 of the tile lie from p on, and how many bytes of them.
    template <class F>
    __device__ inline void paged(const char* p, MLXHIP_LDS char* tile, int wave, F&& at) const {
        __amdgpu_buffer_rsrc_t rsrc;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            if (i % PER16 == 0) {
                uint32_t bytes;
                const int64_t off = at(instr(wave, i) * T::RPI & ~15, &bytes);
                rsrc = buffer(p + off, bytes);
            }
            lds_load16(rsrc, tile + instr(wave, i) * 1024, voff[i % ROUND]);
        }
    }
};

// Row fragments: lane = row base + lane % 32, inner values 16 s + 8 h + (0..7).
template <int DT, int DP, int ROWS>
struct RowFrag {
    using T = Tile<DT, DP, ROWS>;
    uint32_t row, key;
    __device__ inline void init(int lane) {
        row = (uint32_t)(lane & 31) * T::ROWB;
        key = (uint32_t)(T::swizzle(lane & 31) ^ ((lane >> 5) * (DT == MLXHIP_DTYPE_F32 ? 2 : 1)));
    }
    __device__ inline Frag<DT> read(const MLXHIP_LDS char* tile, int base_row, int s) const {
        Frag<DT> f;
        const MLXHIP_LDS char* p = tile + base_row * T::ROWB + row;
        if constexpr (DT == MLXHIP_DTYPE_F32) {
            f.q[0] = *(const MLXHIP_LDS u32x4*)(p + ((4 * s) ^ key) * 16);
            f.q[1] = *(const MLXHIP_LDS u32x4*)(p + ((4 * s + 1) ^ key) * 16);
        } else {
            f.q[0] = *(const MLXHIP_LDS u32x4*)(p + ((2 * s) ^ key) * 16);
        }
        return f;
    }
};

// Transposed fragments: lane = column 32 b + lane % 32, inner rows base + 4 h + (0..3),
// base + 8 + 4 h + (0..3); base a multiple of 16.
template <int DT, int DP, int ROWS>
struct ColFrag {
    using T = Tile<DT, DP, ROWS>;
    int lane;
    uint32_t at, key;  // 16 bits: the lane's source row and its chunk
    __device__ inline void init(int l) {
        lane = l;
        const int g = l >> 4, t = l & 15;
        at = (uint32_t)((4 * (g >> 1) + (t >> 2)) * T::ROWB + (t & 1) * 8);
        key = (uint32_t)(2 * (g & 1) + ((t >> 1) & 1));
    }
    __device__ inline Frag<DT> read(const MLXHIP_LDS char* tile, int base, int b) const {
        Frag<DT> f;
        const MLXHIP_LDS char* p = tile + base * T::ROWB;
        if constexpr (DT == MLXHIP_DTYPE_F32) {
            const int h = lane >> 5, chunk = 8 * b + ((lane & 31) >> 2);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 8 * (j / 4) + 4 * h + j % 4;
                f.q[j / 4][j % 4] = *(const MLXHIP_LDS uint32_t*)(p + row * T::ROWB + ((chunk ^ T::swizzle(row)) << 4) + (lane & 3) * 4);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * r + 4 * (lane >> 5) + ((lane & 15) >> 2);  // of the source lane
                const uint32_t c = (uint32_t)(4 * b) ^ (key ^ (uint32_t)T::swizzle(row));
                const MLXHIP_LDS char* a = p + 8 * r * T::ROWB + at + c * 16;
                const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MLXHIP_LDS gemm16::i16x4*)a));
                f.q[0][2 * r] = v.x;
                f.q[0][2 * r + 1] = v.y;
            }
        }
        return f;
    }
};

// Row fragment of memory: eight values from element 16 s + 8 h of a row, zeros
// past its end (head_dim is a multiple of 8) or where ok is false.
template <int DT>
__device__ inline Frag<DT> load_frag(const typename dev::Elem<DT>::type* row, int lane, int s, int dim, bool ok) {
    Frag<DT> f;
    const int d = 16 * s + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < (DT == MLXHIP_DTYPE_F32 ? 2 : 1); ++i)
        f.q[i] = ok && d < dim ? *reinterpret_cast<const u32x4*>(row + d + 4 * i) : u32x4{0, 0, 0, 0};
    return f;
}

// Keeps what follows in a branch of its own: made into selects, work for the few tiles that a
// mask cuts would be done for all.
__device__ inline void own_branch() { asm volatile(""); }

// Sum over a wave, the same in all lanes: row shifts and broadcasts, no LDS.
__device__ inline int wave_total(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // within rows of 16 lanes: by 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // a row's last lane to the next row
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the first half's to the second
    return __builtin_amdgcn_readlane(v, 63);
}

// Of sequence `i`: its first token and how many it has. starts is the caller's: what it says is
// brought into [0, tokens], a sequence that ends before it starts has no rows.
__device__ inline int first_of(const int32_t* __restrict__ starts, int tokens, int i) { return min(max(starts[i], 0), tokens); }

// The sequence and the tile in it that work item `item` names, of the sequences' rows
// (tokens times per_token) in tiles of `rows`. Sequences go 64 at a time (a group), the groups' items
// from what lies before them on: a tile for each `rows` rows and one for each sequence with any, which
// is enough, and found without a sum over all lengths. A group's items go down by the number of the
// tile, 1 for each sequence's shortest walk under a causal mask: the longest walks of its sequences come
// first, so that none is left to run alone at the end. A wave together; false past a group's last tile.
struct Place {
    int seq, first, tokens, level, tiles;  // level: 1 .. tiles
};
__device__ inline bool find_tile(const int32_t* __restrict__ starts, int n_seqs, int tokens, int per_token, int rows,
                                 int item, Place* out) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    if (n_seqs > 64) {
        const auto before = [&](int g) {  // rows are fewer than 2^29
            const int first = first_of(starts, tokens, 64 * g);
            return (int)((uint32_t)(first * per_token) / (uint32_t)rows) + min(64 * g, first);
        };
        base = dev::last_group((n_seqs + 63) / 64, [&](int g) { return before(g) <= item; });
        if (base > 0) item -= before(base);
        base *= 64;
    }
    const int i = base + lane;
    int first = 0, n = 0;
    if (i < n_seqs) {
        first = first_of(starts, tokens, i);
        n = max(first_of(starts, tokens, i + 1) - first, 0);
    }
    const int tiles = (int)(((int64_t)n * per_token + rows - 1) / rows);
    const int all = n_seqs == 1 ? __builtin_amdgcn_readfirstlane(tiles) : wave_total(tiles);
    if (item >= all) return false;
    // The highest level that more than `item` tiles reach: those from it on.
    int lo = 1, over = 0;
    if (n_seqs == 1) {
        lo = all - item;
        over = item;
    } else {
        for (int hi = all + 1; hi - lo > 1;) {  // above(lo) > item >= above(hi)
            const int mid = lo + (hi - lo) / 2, above = wave_total(max(0, tiles - mid + 1));
            if (above > item) {
                lo = mid;
            } else {
                hi = mid;
                over = above;
            }
        }
    }
    uint64_t reach = __ballot(tiles >= lo);
    for (int k = item - over; k > 0; --k) reach &= reach - 1;
    const int at = __builtin_ctzll(reach);
    out->seq = base + at;
    out->first = __builtin_amdgcn_readlane(first, at);
    out->tokens = __builtin_amdgcn_readlane(n, at);
    out->tiles = __builtin_amdgcn_readlane(tiles, at);
    out->level = lo;
    return true;
}

// The sequence that a token lies in (first and tokens of it), a wave together.
__device__ inline bool find_token(const int32_t* __restrict__ starts, int n_seqs, int tokens, int token, Place* out) {
    const int lane = threadIdx.x & 63;
    const int base = 64 * dev::last_group((n_seqs + 63) / 64, [&](int g) { return first_of(starts, tokens, 64 * g) <= token; });
    const int i = base + lane;
    int first = 0, n = 0;
    if (i < n_seqs) {
        first = first_of(starts, tokens, i);
        n = max(first_of(starts, tokens, i + 1) - first, 0);
    }
    const uint64_t in = __ballot(token >= first && token - first < n);
    if (!in) return false;
    const int at = __builtin_ctzll(in);
    out->seq = base + at;
    out->first = __builtin_amdgcn_readlane(first, at);
    out->tokens = __builtin_amdgcn_readlane(n, at);
    return true;
}

}  // namespace attn
}  // namespace mlxhip
