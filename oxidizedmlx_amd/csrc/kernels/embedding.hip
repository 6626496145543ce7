// embedding.hip — rows of a weight matrix at integer ids, scaled, and the
// gradient with respect to the weight, for f32, bf16 and f16.
//
//   y_i  = scale * W[id_i]                         (ids clamped to [0, vocab - 1],
//   dW_v = scale * sum over i with id_i = v of dy_i  as embedding_lookup does,
//                                   crates/mlx-core/src/cpu_kernels.rs:317-336)
//
// The lookup copies rows, a wave to each: it is bound by memory (or, for a
// few rows, by the launch).
//
// The gradient adds up the dy rows of equal ids in f32, in the order of the
// positions, and rounds once. Text has words that are a tenth of all tokens
// beside thousands that occur once, so a workgroup per id would wait for its
// one longest sum, and atomics would give other bits every time. Instead the
// positions are sorted by id (a stable radix sort of 8 bits a pass, so equal
// ids stay in the order of their positions) and the sorted list is cut into
// equal shares, one to a wave: a share writes the rows that begin and end in
// it, and leaves the sums of the ids that cross its borders as partial rows,
// which a last launch adds up in the order of the shares. Rows of ids that do
// not occur are zeroed by the launches of the sort, on the compute units that the
// sort leaves idle.
//
// 65536 bf16 rows of 1024 over 50257: lookup 40 us (134 MB written, 3.4 TB/s, and
// as much read, the frequent rows from the caches), two passes of the sort 34 with
// the 103 MB of zeros beside them, sums 51, join 12. 2048 f32 rows over 32000: lookup
// 7.5, sort 20 (its 131 MB of zeros at 6.5 TB/s), sums 6.3, join 5.1.
#include "../common.hpp"
#include "../kernels.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace {

using dev::Elem;
using dev::store_vec;
using dev::u32x4;
using dev::unpack;
using dev::Vec16;

constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int BITS = 8, BINS = 1 << BITS;
// Positions that one workgroup sorts in its LDS (key and position, 8 bytes each:
// 64 KiB; 8192 take 29 us that way and 31 in blocks), and those of a
// workgroup's block in a longer sort.
constexpr int LDS_SORT = 8192;
constexpr int BLOCK_SORT = 2048;
// Blocks whose counts the moving launch adds up itself.
constexpr int SCAN_BLOCKS = 64;
// Shares of the sorted list, about.
constexpr int SHARES = 2048;

// N elements of a row from column c on, N = VEC (16 bytes) or 1, at any element
// alignment. A row's last N columns serve the lanes that would run past its end
// (column_of): two lanes then hold some columns both, with the same values.
template <int DT, int N>
struct Piece {
    std::conditional_t<N == 1, typename Elem<DT>::type, u32x4> q;
};
template <int DT, int N>
__device__ inline Piece<DT, N> load_piece(const typename Elem<DT>::type* p) {
    if constexpr (N == 1) return {*p};
    else return {dev::load16<DT>(p)};
}
template <int DT, int N>
__device__ inline void widen(const Piece<DT, N>& x, float (&v)[N]) {
    if constexpr (N == 1) v[0] = dev::to_f32<DT>(x.q);
    else unpack<DT>(Vec16<DT>{x.q}, v);
}
template <int DT, int N>
__device__ inline void store_piece(typename Elem<DT>::type* p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = dev::from_f32<DT>(v[0]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k += Elem<DT>::VEC) store_vec<DT>(p + k, 0, Elem<DT>::VEC, v + k);
    }
}
template <int N>
__device__ inline int64_t column_of(int64_t unit, int64_t dim) {
    return min(unit * N, dim - N);
}

// A wave copies ROWS rows at a time, all their loads in flight.
template <int DT, int N>
__global__ __launch_bounds__(256) void embed_kernel(const typename Elem<DT>::type* __restrict__ w,
                                                    const int32_t* __restrict__ ids,
                                                    typename Elem<DT>::type* __restrict__ y, int64_t n, int64_t vocab,
                                                    int64_t dim, float scale) {
    constexpr int ROWS = 4;
    const int lane = threadIdx.x & 63;
    for (int64_t i = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS; i < n; i += (int64_t)gridDim.x * 4 * ROWS) {
        int64_t id[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) id[k] = min(max((int64_t)ids[min(i + k, n - 1)], (int64_t)0), vocab - 1);
        for (int64_t u = (int64_t)blockIdx.y * 64 + lane; u * N < dim; u += (int64_t)gridDim.y * 64) {
            const int64_t c = column_of<N>(u, dim);
            Piece<DT, N> raw[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) raw[k] = load_piece<DT, N>(w + id[k] * dim + c);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                if (i + k >= n) break;
                float v[N];
                widen<DT, N>(raw[k], v);
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] *= scale;
                store_piece<DT, N>(y + (i + k) * dim + c, v);
            }
        }
    }
}

// Zeros for part `part` of `parts` of the `bytes` (a multiple of 2) from p, by
// workgroup b of nb.
__device__ inline void zero_fill(char* p, int64_t bytes, int part, int parts, int64_t b, int64_t nb) {
    const int64_t from = bytes / 2 * part / parts * 2, to = bytes / 2 * (part + 1) / parts * 2;
    p += from;
    bytes = to - from;
    const int64_t step = nb * SORT_THREADS;
    // The 16-byte words inside, and the bytes before and after them by pairs.
    const int64_t head = min((int64_t)(-reinterpret_cast<intptr_t>(p) & 15), bytes);
    const int64_t words = (bytes - head) / 16, tail = (bytes - head) % 16;
    uint4* q = reinterpret_cast<uint4*>(p + head);
    for (int64_t i = b * SORT_THREADS + threadIdx.x; i < words; i += step) q[i] = make_uint4(0, 0, 0, 0);
    if (b == 0 && threadIdx.x < 16) {
        const int o = threadIdx.x * 2;
        if (o < head) *reinterpret_cast<uint16_t*>(p + o) = 0;
        if (o < tail) *reinterpret_cast<uint16_t*>(p + head + words * 16 + o) = 0;
    }
}

// Of the 64 lanes' digits: how many lower lanes hold this lane's, how many in
// all, both over the lanes with `in`.
__device__ inline void match(uint32_t digit, bool in, int lane, uint32_t* below, uint32_t* count) {
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const uint64_t ones = __ballot((digit >> b) & 1);
        same &= (digit >> b) & 1 ? ones : ~ones;
    }
    *below = (uint32_t)__popcll(same & ((uint64_t(1) << lane) - 1));
    *count = (uint32_t)__popcll(same);
}

// Where each of a workgroup's elements goes by its digit, stably: wave w owns
// elements [w * steps * 64, (w + 1) * steps * 64), step s of them at lane
// offset s * 64. hist[d * SORT_WAVES + w] counts wave w's digits d and, after
// the scan, is the place of the first of them in the workgroup's order.
template <int STEPS>
__device__ inline void local_ranks(const uint32_t (&digit)[STEPS], int steps, int first, int n, uint32_t* hist,
                                   uint32_t (&rank)[STEPS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < BINS * SORT_WAVES; i += SORT_THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (s >= steps) break;
        const bool in = first + s * 64 + lane < n;
        uint32_t below, count;
        match(digit[s], in, lane, &below, &count);
        // Only this wave touches its counters, and its LDS accesses complete
        // in order: every lane reads before the first lane of a digit writes.
        volatile uint32_t* h = hist + digit[s] * SORT_WAVES + wave;
        const uint32_t had = in ? *h : 0;
        rank[s] = had + below;
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) *h = had + count;
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
}

// Exclusive scan of hist (BINS * SORT_WAVES counters) in place by the
// workgroup, four counters a thread.
__device__ inline void scan_hist(uint32_t* hist, uint32_t* wave_sums) {
    static_assert(BINS * SORT_WAVES == 4 * SORT_THREADS, "four counters a thread");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t v[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = sum;
        sum += hist[threadIdx.x * 4 + i];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
    }
    if (lane == 63) wave_sums[wave] = incl;
    __syncthreads();
    uint32_t base = incl - sum;
    for (int w = 0; w < wave; ++w) base += wave_sums[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) hist[threadIdx.x * 4 + i] = base + v[i];
    __syncthreads();
}

__device__ inline uint32_t clamped(int32_t id, uint32_t vocab) {
    return id < 0 ? 0u : min((uint32_t)id, vocab - 1);
}

// Up to LDS_SORT positions: workgroup 0 sorts them, the others zero dW.
__global__ __launch_bounds__(SORT_THREADS) void sort_small_kernel(const int32_t* __restrict__ ids, int n, uint32_t vocab,
                                                                  int passes, uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ order, char* dw,
                                                                  int64_t dw_bytes) {
    constexpr int STEPS = LDS_SORT / SORT_THREADS;
    __shared__ uint32_t skey[LDS_SORT], spos[LDS_SORT], hist[BINS * SORT_WAVES], wave_sums[SORT_WAVES];
    if (blockIdx.x > 0) {
        zero_fill(dw, dw_bytes, 0, 1, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int steps = (n + SORT_THREADS - 1) / SORT_THREADS, first = wave * steps * 64;
    uint32_t key[STEPS], pos[STEPS], digit[STEPS], rank[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = first + s * 64 + lane;
        key[s] = s < steps && i < n ? clamped(ids[i], vocab) : 0;
        pos[s] = i;
    }
    for (int p = 0; p < passes; ++p) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) digit[s] = (key[s] >> (BITS * p)) & (BINS - 1);
        local_ranks<STEPS>(digit, steps, first, n, hist, rank);
        scan_hist(hist, wave_sums);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s < steps && first + s * 64 + lane < n) {
                const uint32_t to = hist[digit[s] * SORT_WAVES + wave] + rank[s];
                skey[to] = key[s];
                spos[to] = pos[s];
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = first + s * 64 + lane;
            if (s < steps && i < n) {
                key[s] = skey[i];
                pos[s] = spos[i];
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += SORT_THREADS) {
        keys[i] = skey[i];
        order[i] = spos[i];
    }
}

// One pass of a longer sort, in blocks of BLOCK_SORT positions: the blocks'
// counts of each digit (counts[digit * blocks + block]), their scan along the
// blocks (of few blocks: by the launch that follows), and the move to the places
// that follow. The first pass reads the ids. Each of these launches also zeroes
// its part of dW with the workgroups past the blocks.
constexpr int BSTEPS = BLOCK_SORT / SORT_THREADS;

__device__ inline void load_block(const int32_t* ids, const uint32_t* keys, int64_t n, uint32_t vocab, int64_t base,
                                  int64_t left, uint32_t (&key)[BSTEPS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 0; s < BSTEPS; ++s) {
        const int i = wave * BSTEPS * 64 + s * 64 + lane;
        key[s] = i < left ? (ids ? clamped(ids[base + i], vocab) : keys[base + i]) : 0;
    }
}

__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const int32_t* __restrict__ ids,
                                                                  const uint32_t* __restrict__ keys, int64_t n,
                                                                  uint32_t vocab, int shift, int blocks,
                                                                  uint32_t* __restrict__ counts, char* dw,
                                                                  int64_t dw_bytes, int part, int parts) {
    __shared__ uint32_t hist[BINS];
    if ((int)blockIdx.x >= blocks) {
        zero_fill(dw, dw_bytes, part, parts, blockIdx.x - blocks, gridDim.x - blocks);
        return;
    }
    if (threadIdx.x < BINS) hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * BLOCK_SORT, left = min((int64_t)BLOCK_SORT, n - base);
    uint32_t key[BSTEPS];
    load_block(ids, keys, n, vocab, base, left, key);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 0; s < BSTEPS; ++s)
        if (wave * BSTEPS * 64 + s * 64 + lane < left) atomicAdd(&hist[(key[s] >> shift) & (BINS - 1)], 1u);
    __syncthreads();
    if (threadIdx.x < BINS) counts[(int64_t)threadIdx.x * blocks + blockIdx.x] = hist[threadIdx.x];
}

// counts[d][*] becomes its exclusive scan, totals[d] its sum: a wave per digit.
__global__ __launch_bounds__(64) void sort_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals,
                                                       int blocks) {
    uint32_t* c = counts + (int64_t)blockIdx.x * blocks;
    const int lane = threadIdx.x;
    uint32_t base = 0;
    for (int b = 0; b < blocks; b += 64) {
        const uint32_t v = b + lane < blocks ? c[b + lane] : 0;
        uint32_t incl = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(incl, o, 64);
            if (lane >= o) incl += u;
        }
        if (b + lane < blocks) c[b + lane] = base + incl - v;
        base += __shfl(incl, 63, 64);
    }
    if (lane == 0) totals[blockIdx.x] = base;
}

__global__ __launch_bounds__(SORT_THREADS) void sort_move_kernel(const int32_t* __restrict__ ids,
                                                                 const uint32_t* __restrict__ keys,
                                                                 const uint32_t* __restrict__ order, int64_t n,
                                                                 uint32_t vocab, int shift, int blocks,
                                                                 const uint32_t* __restrict__ counts,
                                                                 const uint32_t* __restrict__ totals,
                                                                 uint32_t* __restrict__ keys_out,
                                                                 uint32_t* __restrict__ order_out, char* dw,
                                                                 int64_t dw_bytes, int part, int parts) {
    if ((int)blockIdx.x >= blocks) {
        zero_fill(dw, dw_bytes, part, parts, blockIdx.x - blocks, gridDim.x - blocks);
        return;
    }
    __shared__ uint32_t hist[BINS * SORT_WAVES], wave_sums[SORT_WAVES], start[BINS], total[BINS], before[BINS];
    const int64_t base = (int64_t)blockIdx.x * BLOCK_SORT, left = min((int64_t)BLOCK_SORT, n - base);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t key[BSTEPS], digit[BSTEPS], rank[BSTEPS];
    load_block(ids, keys, n, vocab, base, left, key);
#pragma unroll
    for (int s = 0; s < BSTEPS; ++s) digit[s] = (key[s] >> shift) & (BINS - 1);
    local_ranks<BSTEPS>(digit, BSTEPS, wave * BSTEPS * 64, (int)left, hist, rank);
    scan_hist(hist, wave_sums);
    // Digit d's elements in all blocks, and in those before this one.
    if (threadIdx.x < BINS) {
        const uint32_t* c = counts + (int64_t)threadIdx.x * blocks;
        uint32_t all = 0, mine = 0;
        if (totals) {
            all = totals[threadIdx.x];
            mine = c[blockIdx.x];
        } else {
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) {
                const uint32_t v = c[b];
                all += v;
                if (b < (int)blockIdx.x) mine += v;
            }
        }
        total[threadIdx.x] = all;
        before[threadIdx.x] = mine;
    }
    __syncthreads();
    // Where the block's elements of a digit begin in the whole order, less
    // their place in the block's.
    if (wave == 0) {
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < BINS / 64; ++i) sum += total[lane * (BINS / 64) + i];
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(incl, o, 64);
            if (lane >= o) incl += u;
        }
        uint32_t at = incl - sum;
#pragma unroll
        for (int i = 0; i < BINS / 64; ++i) {
            const int d = lane * (BINS / 64) + i;
            start[d] = at + before[d] - hist[d * SORT_WAVES];
            at += total[d];
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < BSTEPS; ++s) {
        const int i = wave * BSTEPS * 64 + s * 64 + lane;
        if (i < left) {
            const uint32_t to = start[digit[s]] + hist[digit[s] * SORT_WAVES + wave] + rank[s];
            keys_out[to] = key[s];
            order_out[to] = order ? order[base + i] : (uint32_t)(base + i);
        }
    }
}

// A wave's share of the sorted positions and chunk of 64 * N columns. part
// holds two rows of dim sums per share: of the id that began before it, and
// of the one that goes on after it (an id that does both: the first only).
// The lanes hold 64 positions' keys and places, so the rows' addresses come
// from registers and AHEAD rows are loaded at once. 65536 bf16 rows of 1024 with
// ids as frequent as words: 51 us for some 190 MB (rows read, sums and partial
// sums written), 3.7 TB/s, whatever the length of the shares; the join then takes
// 12 us for shares of 32 rows, and some two and four times that for 16 and 8.
template <int DT, int N>
__global__ __launch_bounds__(256) void embed_sum_kernel(const typename Elem<DT>::type* __restrict__ dy,
                                                        const uint32_t* __restrict__ keys,
                                                        const uint32_t* __restrict__ order, int64_t n, int share,
                                                        int64_t shares, int64_t dim, float scale,
                                                        typename Elem<DT>::type* __restrict__ dw,
                                                        float* __restrict__ part) {
    constexpr int AHEAD = 16;
    const int lane = threadIdx.x & 63;
    const int64_t sh = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
    if (sh >= shares) return;
    const int64_t unit = (int64_t)blockIdx.x * 64 + lane, c = column_of<N>(unit, dim);
    const bool in = unit * N < dim;  // other lanes load what the last one does and store nothing
    const int64_t lo = sh * share, hi = min(n, lo + share);
    const typename Elem<DT>::type* from = dy + c;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    // The keys around the share, and its first one.
    const uint32_t before = lo > 0 ? keys[lo - 1] : 0, after = hi < n ? keys[hi] : 0;
    uint32_t cur = __builtin_amdgcn_readfirstlane(keys[lo]);
    bool head = lo > 0 && before == cur;
    auto leave = [&](float* to) {
        if (in) store_piece<MLXHIP_DTYPE_F32, N>(to + c, acc);
    };
    auto flush = [&] {
        if (head) {
            leave(part + 2 * sh * dim);
        } else if (in) {
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] *= scale;
            store_piece<DT, N>(dw + (int64_t)cur * dim + c, acc);
        }
        head = false;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    };
    for (int64_t i0 = lo; i0 < hi; i0 += 64) {
        const int count = (int)min(hi - i0, (int64_t)64);
        const int64_t mine = min(i0 + lane, hi - 1);
        const int key_l = (int)keys[mine], pos_l = (int)order[mine];
        for (int i = 0; i < count; i += AHEAD) {
            Piece<DT, N> raw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (i + a < count)
                    raw[a] = load_piece<DT, N>(from + (int64_t)(uint32_t)__builtin_amdgcn_readlane(pos_l, i + a) * dim);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (i + a >= count) break;
                const uint32_t key = (uint32_t)__builtin_amdgcn_readlane(key_l, i + a);
                if (key != cur) {
                    flush();
                    cur = key;
                }
                float v[N];
                widen<DT, N>(raw[a], v);
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] += v[e];
            }
        }
    }
    if (hi < n && after == cur) leave(part + (2 * sh + (head ? 0 : 1)) * dim);
    else flush();
}

// The ids that go on after a share and began in it: their shares' sums in
// order, 64 columns at a time. A workgroup's four waves have a share each; an
// id that reaches over more than ALONE of them (a frequent word's some hundred)
// is added up by all four, a contiguous part of the shares each.
constexpr int ALONE = 16;
template <int DT>
__global__ __launch_bounds__(256) void embed_join_kernel(const uint32_t* __restrict__ keys, int64_t n, int share,
                                                         int64_t shares, int64_t dim, float scale,
                                                         typename Elem<DT>::type* __restrict__ dw,
                                                         const float* __restrict__ part) {
    __shared__ int64_t runs[4];  // the last share of a wave's id; 0: nothing to add up
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t sh = (int64_t)blockIdx.x * 4 + wave, c = (int64_t)blockIdx.y * 64 + lane;
    int64_t last = 0;
    uint32_t key = 0;
    if (sh + 1 < shares) {
        const int64_t lo = sh * share, hi = lo + share;
        const uint32_t first = keys[lo], before = lo > 0 ? keys[lo - 1] : ~keys[lo], after = keys[hi];
        key = keys[hi - 1];
        if (after == key && (first != key || before != key)) {
            // The last share that the id reaches: 64 of their first keys at a time.
            last = sh + 1;
            for (;;) {
                const int64_t k = last + 1 + lane;
                const uint64_t go = __ballot(k < shares && keys[min(k, shares - 1) * share] == key);
                const int run = ~go ? __builtin_ctzll(~go) : 64;
                last += run;
                if (run < 64) break;
            }
        }
    }
    const bool alone = last - sh <= ALONE;
    if (last && alone && c < dim) {
        float acc = part[(2 * sh + 1) * dim + c];
#pragma unroll 8
        for (int64_t k = sh + 1; k <= last; ++k) acc += part[2 * k * dim + c];
        dw[(int64_t)key * dim + c] = dev::from_f32<DT>(acc * scale);
    }
    if (lane == 0) runs[wave] = alone ? 0 : last;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        const int64_t end = runs[w], from = (int64_t)blockIdx.x * 4 + w;
        if (end == 0) continue;
        const int64_t each = (end - from + 3) / 4, k0 = from + 1 + wave * each, k1 = min(k0 + each, end + 1);
        float acc = 0.0f;
        if (c < dim) {
            if (wave == 0) acc = part[(2 * from + 1) * dim + c];
#pragma unroll 16
            for (int64_t k = k0; k < k1; ++k) acc += part[2 * k * dim + c];
        }
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave == w && c < dim)
            dw[(int64_t)key * dim + c] =
                dev::from_f32<DT>((((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane]) * scale);
        __syncthreads();
    }
}

// Up to 64 positions: one launch, in which a workgroup owns `each` rows of dW. It
// finds the positions of its rows (in order) and their bits among its rows, writes
// zeros to the others, and gives each id's sum to a wave, 64 pieces of columns at a
// time. Against sorting (64 distinct positions and 65, 2000 rows of 1024 f32 values: 4.4
// and 11.8 us) it saves three launches, but one compute unit adds up all positions of
// one id, behind its zeros: 64 of them take 5 us more for rows of 4 KiB, 8 for 8, 17 for
// 16 and 34 for 32, where sorting stays at 13 to 17 in all. So it takes up to 512 KiB
// of dy where dW has up to 32 MiB (64 rows of 8 KiB of one id 13.0 us, sorted 15.2; 32 of
// 16 KiB 15.5 and 15.3, 64 of them 24 and 16). The sort's launches hide behind a larger
// dW's zeros: there half of that dy (131 MB, 64 rows of 4 KiB of one id 20.6, 65 sorted
// 23.8), and none from 192 MiB on (262 MB: 39 distinct either way, 24 of one id 45 and 40).
constexpr int FEW = 64, FEW_ROWS = 4096;  // most rows of a workgroup
inline bool few_positions(int64_t n, int64_t dy_bytes, int64_t dw_bytes) {
    return n <= FEW && dw_bytes <= (192 << 20) && dy_bytes <= (dw_bytes <= (32 << 20) ? 512 << 10 : 256 << 10);
}
template <int DT, int N>
__global__ __launch_bounds__(1024) void embed_few_kernel(const typename Elem<DT>::type* __restrict__ dy,
                                                         const int32_t* __restrict__ ids, int n, int64_t vocab,
                                                         int64_t dim, float scale, int each,
                                                         typename Elem<DT>::type* __restrict__ dw) {
    constexpr int AHEAD = 8;
    __shared__ uint32_t bits[FEW_ROWS / 32], key[FEW], pos[FEW];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t v0 = (int64_t)blockIdx.x * each, v1 = min(v0 + each, vocab);
    if (tid < FEW_ROWS / 32) bits[tid] = 0;
    if (tid < FEW) key[tid] = ~0u;  // behind the workgroup's positions
    __syncthreads();
    if (wave == 0) {
        const int64_t id = lane < n ? (int64_t)clamped(ids[lane], (uint32_t)vocab) : -1;
        const bool mine = id >= v0 && id < v1;
        const uint64_t mask = __ballot(mine);
        if (mine) {
            const int at = (int)__popcll(mask & ((uint64_t(1) << lane) - 1));
            key[at] = (uint32_t)(id - v0);
            pos[at] = (uint32_t)lane;
            atomicOr(&bits[(id - v0) / 32], 1u << ((id - v0) % 32));
        }
        if (lane == 0) count = (int)__popcll(mask);
    }
    __syncthreads();
    const uint32_t units = (uint32_t)((dim + N - 1) / N), all = (uint32_t)(v1 - v0) * units;
    float zeros[N];
#pragma unroll
    for (int e = 0; e < N; ++e) zeros[e] = 0.0f;
    for (uint32_t i = tid; i < all; i += 1024) {
        const uint32_t r = i / units;
        if (!(bits[r / 32] >> (r % 32) & 1)) store_piece<DT, N>(dw + (v0 + r) * dim + column_of<N>(i - r * units, dim), zeros);
    }
    const int chunks = (int)((units + 63) / 64);
    const uint32_t keys = key[lane];
    const int places = (int)pos[lane];  // read by lane: no trip to LDS before a load
    for (int it = wave; it < count * chunks; it += 16) {
        const int entry = it / chunks;
        const uint32_t k = key[entry];
        uint64_t left = __ballot(keys == k);
        if (entry != __builtin_ctzll(left)) continue;  // the id's first position has it
        const uint32_t unit = (uint32_t)(it - entry * chunks) * 64 + lane;
        const int64_t c = column_of<N>(unit, dim);  // lanes behind the row load its end
        float acc[N];
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.0f;
        while (left) {
            Piece<DT, N> raw[AHEAD];
            const int got = min((int)__popcll(left), AHEAD);
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
                if (a < got) {
                    raw[a] = load_piece<DT, N>(dy + (int64_t)__builtin_amdgcn_readlane(places, __builtin_ctzll(left)) * dim + c);
                    left &= left - 1;
                }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (a >= got) break;
                float v[N];
                widen<DT, N>(raw[a], v);
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] += v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] *= scale;
        if (unit < units) store_piece<DT, N>(dw + (v0 + k) * dim + c, acc);
    }
}

// Rows of at least 16 bytes in pieces of that size (N values), others one by one.
template <int DT, int N>
int run_embed(const void* w, const int32_t* ids, void* y, int64_t n, int64_t vocab, int64_t dim, float scale,
              hipStream_t s) {
    typedef typename Elem<DT>::type T;
    // At most 2^30 work-items, which a dispatch counts in 32 bits.
    const int64_t gy = std::min<int64_t>(ceil_div(dim, 64 * N), 64);
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(n, 16), (1 << 22) / gy), (unsigned)gy);
    hipLaunchKernelGGL((embed_kernel<DT, N>), grid, dim3(256), 0, s, (const T*)w, ids, (T*)y, n, vocab, dim, scale);
    return launch_check("embed_kernel");
}

template <int DT, int N>
int run_embed_vjp(const void* dy, const int32_t* ids, void* dw, int64_t n, int64_t vocab, int64_t dim, float scale,
                  hipStream_t s) {
    typedef typename Elem<DT>::type T;
    // 512 workgroups, two to a compute unit; `all` above within 32 bits.
    const int64_t each = std::min<int64_t>(ceil_div(vocab, 512), std::min<int64_t>(FEW_ROWS, (int64_t(1) << 30) / dim));
    const int64_t dw_bytes = vocab * dim * (int64_t)sizeof(T);
    if (n == 0 || few_positions(n, n * dim * (int64_t)sizeof(T), dw_bytes)) {
        hipLaunchKernelGGL((embed_few_kernel<DT, N>), dim3((unsigned)ceil_div(vocab, each)), dim3(1024), 0, s, (const T*)dy,
                           ids, (int)n, vocab, dim, scale, (int)each, (T*)dw);
        return launch_check("embed_few_kernel");
    }
    const int fill = (int)std::min<int64_t>(ceil_div(dw_bytes, 16 * SORT_THREADS), 512);
    const int64_t blocks = n <= LDS_SORT ? 0 : ceil_div(n, BLOCK_SORT);
    // 2048 shares fill the compute units (8 waves each, times the chunks of
    // columns) and leave a frequent id few partial sums to add up.
    const int share = (int)std::max<int64_t>(ceil_div(n, SHARES), 4);
    const int64_t shares = ceil_div(n, share);
    const size_t list = ((size_t)n * 4 + 255) / 256 * 256;
    const size_t sums = (size_t)shares * 2 * dim * sizeof(float);
    const size_t counts = blocks ? ((size_t)BINS * blocks + BINS) * 4 : 0;
    char* ws = nullptr;
    MLXHIP_TRY(stream_workspace(s, WS_EMBED, (blocks ? 4 : 2) * list + sums + counts, reinterpret_cast<void**>(&ws)));
    uint32_t *keys = reinterpret_cast<uint32_t*>(ws), *order = reinterpret_cast<uint32_t*>(ws + list);
    float* part = reinterpret_cast<float*>(ws + (blocks ? 4 : 2) * list);
    int passes = 1;
    while (passes < 4 && (vocab - 1) >> (BITS * passes)) ++passes;
    if (!blocks) {
        hipLaunchKernelGGL(sort_small_kernel, dim3((unsigned)(1 + fill)), dim3(SORT_THREADS), 0, s, ids, (int)n,
                           (uint32_t)vocab, passes, keys, order, (char*)dw, dw_bytes);
        MLXHIP_TRY(launch_check("sort_small_kernel"));
    } else {
        uint32_t *keys2 = reinterpret_cast<uint32_t*>(ws + 2 * list), *order2 = reinterpret_cast<uint32_t*>(ws + 3 * list);
        uint32_t* cnt = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(part) + sums);
        uint32_t* totals = cnt + BINS * blocks;
        for (int p = 0; p < passes; ++p) {
            const int32_t* src = p == 0 ? ids : nullptr;
            hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)(blocks + fill)), dim3(SORT_THREADS), 0, s, src, keys, n,
                               (uint32_t)vocab, BITS * p, (int)blocks, cnt, (char*)dw, dw_bytes, 2 * p, 2 * passes);
            MLXHIP_TRY(launch_check("sort_count_kernel"));
            if (blocks > SCAN_BLOCKS) {
                hipLaunchKernelGGL(sort_scan_kernel, dim3(BINS), dim3(64), 0, s, cnt, totals, (int)blocks);
                MLXHIP_TRY(launch_check("sort_scan_kernel"));
            }
            hipLaunchKernelGGL(sort_move_kernel, dim3((unsigned)(blocks + fill)), dim3(SORT_THREADS), 0, s, src, keys,
                               p == 0 ? nullptr : order, n, (uint32_t)vocab, BITS * p, (int)blocks, cnt,
                               blocks > SCAN_BLOCKS ? totals : nullptr, keys2, order2, (char*)dw, dw_bytes, 2 * p + 1,
                               2 * passes);
            MLXHIP_TRY(launch_check("sort_move_kernel"));
            std::swap(keys, keys2);
            std::swap(order, order2);
        }
    }
    const dim3 grid((unsigned)ceil_div(dim, 64 * N), (unsigned)ceil_div(shares, 4));
    hipLaunchKernelGGL((embed_sum_kernel<DT, N>), grid, dim3(256), 0, s, (const T*)dy, keys, order, n, share, shares, dim,
                       scale, (T*)dw, part);
    MLXHIP_TRY(launch_check("embed_sum_kernel"));
    const dim3 jgrid((unsigned)ceil_div(shares, 4), (unsigned)ceil_div(dim, 64));
    hipLaunchKernelGGL((embed_join_kernel<DT>), jgrid, dim3(256), 0, s, keys, n, share, shares, dim, scale, (T*)dw, part);
    return launch_check("embed_join_kernel");
}

}  // namespace

int embedding_rows(int dt, const void* w, const int32_t* ids, void* y, int64_t n, int64_t vocab, int64_t dim,
                   float scale, hipStream_t s) {
    if (n == 0 || dim == 0) return MLXHIP_OK;
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            constexpr int VEC = Elem<d.value>::VEC;
            rc = dim < VEC ? run_embed<d.value, 1>(w, ids, y, n, vocab, dim, scale, s)
                           : run_embed<d.value, VEC>(w, ids, y, n, vocab, dim, scale, s);
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "embedding: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

int embedding_vjp_rows(int dt, const void* dy, const int32_t* ids, void* dw, int64_t n, int64_t vocab, int64_t dim,
                       float scale, hipStream_t s) {
    if (vocab == 0 || dim == 0) return MLXHIP_OK;
    int rc = MLXHIP_OK;
    if (!with_float_dtype(dt, [&](auto d) {
            constexpr int VEC = Elem<d.value>::VEC;
            rc = dim < VEC ? run_embed_vjp<d.value, 1>(dy, ids, dw, n, vocab, dim, scale, s)
                           : run_embed_vjp<d.value, VEC>(dy, ids, dw, n, vocab, dim, scale, s);
        }))
        return fail(MLXHIP_ERR_INVALID_ARGUMENT, "embedding gradient: dtype %d (f32, bf16 or f16)", dt);
    return rc;
}

}  // namespace mlxhip
