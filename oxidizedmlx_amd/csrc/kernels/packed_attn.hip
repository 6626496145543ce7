// packed_attn.hip — which kernels a call of the packed or paged attention takes.
#include "packed_attn.hpp"
#include "elem.hpp"
#include "../common.hpp"

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

namespace mlxhip {
namespace {

// For tests (attention_plan): tiles of few rows or not, and shares, whatever the sizes.
std::atomic<int> forced_few_rows{-1}, forced_shares{0};

// Work items of sequences whose lengths are known on the device only: a tile more for each.
int items_of(int64_t tokens, int64_t per_token, int64_t n_seqs, int64_t rows) {
    return (int)(tokens * per_token / rows + std::min(n_seqs, tokens));
}

uint32_t flip_of(int dtype, float scale) {
    return !(scale < 0) ? 0u : dtype == MLXHIP_DTYPE_F32 ? 0x80000000u : 0x80008000u;
}

// |scale| log2 e; never 0, which a masked score of -inf would not survive (scores
// times the smallest normal number are 0 beside any other).
float factor_of(float scale) { return std::max(std::fabs(scale) * 1.44269504088896340736f, FLT_MIN); }

// Whether a prompt's rows go in tiles of 32 whose keys four waves share out, not in tiles of 128: where
// those would leave compute units without work, or with a causal sequence's longest walks alone at the end,
// which the more tiles make up for the longer the walks are. Tiles of 32 reach about four fifths of the other's
// rate where both fill the card. Forward, us, tiles of 128 / 32:
//   f16: 123 tiles (1537 tokens, 9 heads on 3 of 80) 18.2 / 12.0;
//   bf16, 8 heads of 128: 224 tiles (3500 tokens) 75.6 / 48.1, 288 (4500) 98.7 / 72.7, 376 (6000) 135.9 / 116,
//   304 (4500 in 3 sequences) 57.6 / 40.4; but 320 (8 of 512) 17.5 / 20.5, 408 (1600, 32 heads on 8) 39.4 / 50.3;
//   not causal: 176 (2800) 63.1 / 59.1, but 288 (4500) 123.6 / 139.9;
//   f32: 320 (4 of 512, 16 heads of 64) 50.4 / 36.6, 516 (4096, 16 on 4 of 128) 741 / 642, 632 (10000, 8 of
//   128) 1950 / 1791, 640 (8 of 512, 16 of 64) 68.1 / 66.7; but 752 (6000, 16 on 4 of 128) 1213 / 1322, 776
//   (12288, 8 of 128) 2529 / 2643, 1280 (16 of 512, 16 of 64) 106 / 130; and not causal, which the limit does
//   not look at, 264 (4096, 8 of 128) 541 / 606.
// dQ takes the same tiles. Whole gradients: bf16: 288 (4500) 269 / 227, 376 (6000) 385 / 340; but 320 (8 of 512)
// 52.7 / 56.7, 408 (1600, 32 heads on 8) 150 / 166; f32: 264 (4096, 8 of 128) 1491 / 1133, 520 (8192) 4154 / 4168,
// 640 (8 of 512, 16 of 64) 203 / 200, 1280 (16 of 512) 361 / 388.
bool few_rows(int dtype, int64_t tokens, int64_t group, int64_t n_seqs, int64_t kv_heads, int causal) {
    if (const int forced = forced_few_rows.load(); forced >= 0) return forced;
    const int64_t wgs = items_of(tokens, group, n_seqs, attn::ROW_TILE) * kv_heads;
    if (dtype == MLXHIP_DTYPE_F32) return wgs < 640;
    return wgs < (causal ? std::min<int64_t>(192 + tokens / n_seqs / 12, 480) : 192);
}

template <class F>
int by_dtype(int dtype, F&& f) {
    int rc = MLXHIP_OK;
    with_float_dtype(dtype, [&](auto dt) { rc = f(dt); });
    return rc;
}

}  // namespace

void attention_plan(int few_rows, int shares) {
    forced_few_rows = few_rows;
    forced_shares = std::clamp(shares, 0, attn::MAX_SHARES);
}

int packed_attention(int dtype, const void* q, const void* k, const void* v, const int32_t* starts, void* o, float* lse,
                     int64_t n_seqs, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_stride,
                     int64_t kv_stride, int64_t o_stride, float scale, int causal, hipStream_t s) {
    attn::FwdArgs a{};
    a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse, a.starts = starts;
    a.n_seqs = (int)n_seqs, a.tokens = (int)tokens, a.heads = (int)heads, a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads), a.dim = (int)dim;
    a.q_stride = q_stride, a.kv_stride = kv_stride, a.o_stride = o_stride;
    a.c = factor_of(scale), a.flip = flip_of(dtype, scale);
    a.causal = causal, a.splits = 1;
    const bool keys = few_rows(dtype, tokens, a.group, n_seqs, kv_heads, causal);
    a.items = items_of(tokens, a.group, n_seqs, keys ? attn::FEW_ROWS : attn::ROW_TILE);
    return by_dtype(dtype, [&](auto dt) { return attn::fwd<decltype(dt)::value>(a, false, keys, s); });
}

int packed_attention_vjp(int dtype, const void* q, const void* k, const void* v, const void* o, const void* dout,
                         const float* lse, const int32_t* starts, void* dq, void* dk, void* dv, int64_t n_seqs,
                         int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_stride, int64_t kv_stride,
                         int64_t o_stride, float scale, int causal, hipStream_t s) {
    attn::BwdArgs a{};
    a.q = q, a.k = k, a.v = v, a.o = o, a.dout = dout, a.lse = lse, a.starts = starts;
    a.dq = dq, a.dk = dk, a.dv = dv;
    a.n_seqs = (int)n_seqs, a.tokens = (int)tokens, a.heads = (int)heads, a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads), a.dim = (int)dim;
    a.q_stride = q_stride, a.kv_stride = kv_stride, a.o_stride = o_stride;
    a.c = factor_of(scale), a.scale = scale, a.flip = flip_of(dtype, scale);
    a.causal = causal;
    a.few_rows = few_rows(dtype, tokens, a.group, n_seqs, kv_heads, causal);
    a.row_items = items_of(tokens, a.group, n_seqs, a.few_rows ? attn::FEW_ROWS : attn::ROW_TILE);
    a.key_items = items_of(tokens, 1, n_seqs, attn::KEY_TILE);
    // Few tiles of keys: each one's walk over several workgroups, their sums joined, until there are 512, of
    // three blocks of 32 rows or more on average; where every compute unit has a tile, only of long
    // walks, which end far apart. us, whole and in shares: the kernel of 51 tiles (1537 tokens, 9 heads on 3 of
    // 80, f16) 75 and 29 + 5; steps of 260 tiles (8192 tokens, 16 heads on 4 of 128, bf16) 1750 and 1320;
    // of 320 tiles with walks of 8 blocks (4 x 512 tokens, 16 heads of 64, bf16) 46 and 63, so not there.
    const int64_t wgs = a.key_items * kv_heads, blocks = a.group * (tokens / n_seqs) / (causal ? 64 : 32);
    const int64_t most = wgs < 256 || blocks >= 64 ? ceil_div(512, wgs) : 1;
    a.shares = (int)std::clamp<int64_t>(std::min(most, blocks / 3), 1, attn::MAX_SHARES);
    if (const int forced = forced_shares.load()) a.shares = forced;
    const size_t stats = (((size_t)tokens * heads + 63) & ~size_t(63)) * sizeof(float);
    const size_t part = a.shares > 1 ? (size_t)a.shares * 2 * tokens * kv_heads * dim * sizeof(float) : 0;
    void* ws = nullptr;
    MLXHIP_TRY(stream_workspace(s, WS_PACKED, 2 * stats + part, &ws));
    a.lse2 = (float*)ws, a.delta = (float*)((char*)ws + stats), a.part = (float*)((char*)ws + 2 * stats);
    return by_dtype(dtype, [&](auto dt) { return attn::bwd<decltype(dt)::value>(a, s); });
}

int paged_attention(int dtype, const void* q, const void* k_pages, const void* v_pages, const PagedArgs& pages, void* o,
                    int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_stride, int64_t o_stride,
                    float scale, hipStream_t s) {
    attn::FwdArgs a{};
    a.q = q, a.k = k_pages, a.v = v_pages, a.o = o, a.starts = pages.starts, a.pages = pages;
    a.n_seqs = pages.n_seqs, a.tokens = (int)tokens, a.heads = (int)heads, a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads), a.dim = (int)dim;
    a.q_stride = q_stride, a.o_stride = o_stride;
    a.c = factor_of(scale), a.flip = flip_of(dtype, scale);
    a.causal = 1;
    // Up to 32 rows a sequence on average (single tokens of up to 32 heads to a K/V head, say): one tile of 32 to
    // a sequence. us, tiles of 128 / 32 rows, 16 sequences of up to 8192, 32 heads on 8 of 128: bf16 at 16 rows
    // a sequence 54 / 52, at 32 71 / 56, at 64 84 / 73, at 128 103 / 104; f32 at 32 434 / 171, at 128 698 / 432.
    const bool keys = tokens * a.group <= (int64_t)attn::FEW_ROWS * a.n_seqs;
    a.items = items_of(tokens, a.group, a.n_seqs, keys ? attn::FEW_ROWS : attn::ROW_TILE);
    // The keys over several workgroups. Few rows: until there are 512, one round of two to a compute unit
    // (us: 2 sequences of 131072, f16, 16 tiles: 193, at 1024 199: more parts to join); with 64 tiles and more,
    // whose sequences differ, 1024 (16 of up to 4096, f32, 144 tiles: 100, at 512 110, at 2048 121); 2048
    // where the tiles alone are a round and what is left is to even out (64 of up to 8192, bf16, 576 tiles:
    // 148, at 1024 176). Tiles of rows: 512 for one sequence, whose walks are alike (256 tokens over 32768:
    // 183, at 1100 196, at 1600 220; 2048 over 16384: 500, 522 and 526); for several, 800 where the tiles are
    // less than a round (256 tokens in 4 over up to 32768: 153, at 512 207, at 1600 183; 1024 in 8 over up to
    // 8192: 146, 192 and 150) and 1600 from there on (2000 in 4 over 16384: 632, at 512 and 800 756; over up
    // to 16384: 417, at both 440). Within 256 MiB of parts, and 64 of them at most: what more of them save in the
    // walks the join takes (one sequence of 131072, f16: 8 heads on 1, 39.1, with 32 parts 52.9, 128 38.3, 256
    // 53.1; 16 on 2, 39.2, with 128 46.7; two of them, 16 on 2, 58.1, with 32 54.3, 128 66.9).
    const int64_t most = pages.table_width << pages.page_shift, wgs = std::max<int64_t>((int64_t)a.items * kv_heads, 1);
    const int64_t target = keys                ? (wgs < 64 ? 512 : wgs < 512 ? 1024 : 2048)
                           : pages.n_seqs == 1 ? 512
                           : wgs < 512         ? 800
                                               : 1600;
    int64_t splits = std::min<int64_t>({target / wgs, ceil_div(most, attn::MIN_SPAN), 64});
    const int64_t row = tokens * heads * (dim + 4) * (int64_t)sizeof(float);
    splits = std::min<int64_t>(splits, (int64_t(256) << 20) / std::max<int64_t>(row, 1));
    a.splits = (int)std::max<int64_t>(splits, 1);
    if (a.splits > 1) {
        void* ws = nullptr;
        MLXHIP_TRY(stream_workspace(s, WS_PACKED, (size_t)(a.splits * row), &ws));
        a.part = (float*)ws;
    }
    return by_dtype(dtype, [&](auto dt) { return attn::fwd<decltype(dt)::value>(a, true, keys, s); });
}

}  // namespace mlxhip
