// packed_attn.hpp — arguments of the packed attention's kernels and the functions that
// launch them for one type.
#pragma once

#include "../kernels.hpp"

namespace mlxhip {
namespace attn {

struct FwdArgs {
    const void *q, *k, *v;   // k, v: the K/V rows, or the pages
    void* o;
    float* lse;              // [tokens][heads], or null
    float* part;             // [splits][tokens * heads][dim + 4] (splits > 1): o, its base, its sum
    const int32_t* starts;
    PagedArgs pages;         // paged
    int n_seqs, tokens, heads, kv_heads, group, dim;
    int64_t q_stride, kv_stride, o_stride;
    float c;                 // |scale| log2 e
    uint32_t flip;           // Q's signs turned round (a negative scale)
    int causal, items, splits;
};
template <int DT>
int fwd(const FwdArgs& a, bool paged, bool keys, hipStream_t s);

struct BwdArgs {
    const void *q, *k, *v, *o, *dout;
    const float* lse;        // [tokens][heads]
    float *lse2, *delta;     // [heads][tokens], dQ's kernel for dK and dV's: lse log2 e less the shift of p, -rowsum(dO o O)
    float* part;             // [shares][2][tokens][kv_heads][dim] (shares > 1): dK, dV
    void *dq, *dk, *dv;
    const int32_t* starts;
    int n_seqs, tokens, heads, kv_heads, group, dim;
    int64_t q_stride, kv_stride, o_stride;
    float c, scale;
    uint32_t flip;
    int causal, row_items, key_items, shares;
    bool few_rows;  // rows in tiles of FEW_ROWS
};
template <int DT>
int bwd(const BwdArgs& a, hipStream_t s);

// Rows of a work item: query rows (token, head of the group) and keys.
constexpr int ROW_TILE = 128, FEW_ROWS = 32, KEY_TILE = 128;
constexpr int MAX_SHARES = 16;
// Rows that see up to as many keys get P and dS in two terms in the gradients of 16-bit types.
constexpr int FINE_KEYS = 64;
// Keys that are worth a workgroup of their own.
constexpr int MIN_SPAN = 256;

}  // namespace attn
}  // namespace mlxhip
