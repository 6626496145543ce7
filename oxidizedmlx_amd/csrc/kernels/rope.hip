// rope.hip — rotary positions of rows [tokens, heads, head_dim] and their
// gradient, the table of frequencies, and the append of new tokens' keys
// (rotated) and values to a cache in pages.
//
// Pair i of a head, at (i, i + rotary/2) or (2i, 2i + 1), turns by the angle
// a = position * f_i:  (u, v) -> m (u cos a - v sin a, v cos a + u sin a).
// The gradient is the transpose: the angle's sign turned round.
//
// Bound by HBM: each value is read and written once, the angles of a token are
// the same for all its heads. A workgroup takes TK tokens, forms their cosines
// and sines once in LDS (a pair to a thread), then streams the heads' rows in
// 16-byte vectors. Angles are products in 64 bits, brought to an eighth of a turn
// there: a position of 10^6 in f32 alone is off by 0.06 of a radian.
// 16384 tokens of 40 heads of 128, bf16, one way: 61 us, 5.5 TB/s, a large copy's rate. An append
// of few tokens is a chain of loads (starts and lengths, the page's number): 64 tokens 7.5 us a call.
#include "../kernels.hpp"
#include "../common.hpp"
#include "elem.hpp"

#include <algorithm>

namespace mlxhip {
namespace {

using dev::Elem;
using dev::Vec16;

constexpr int THREADS = 256;
constexpr int TK = 2;         // tokens of a workgroup (16384 tokens of 40 heads of 128, bf16, both ways: 121 us; 4: 124, 1: 126)
constexpr int APPEND_TK = 4;  // of an append: 4 waves, one to a token

// cos and sin of `turns` whole turns, any size.
__device__ inline float2 cos_sin_turns(double turns) {
    // q quarters and a rest of up to an eighth of a turn either way, whose f32
    // rounding is 2^-27 of a turn at most.
    const double q = rint(turns * 4.0);
    const float rest = (float)(turns - q * 0.25);
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    const int quarter = (int)(q - 4.0 * floor(q * 0.25));
    const float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    // quarters 0..3: (c, s), (-s, c), (-c, -s), (s, -c)
    return {quarter == 1 || quarter == 2 ? -cc : cc, quarter >= 2 ? -ss : ss};
}

constexpr double TURNS = 0.15915494309189533576888;  // 1 / 2 pi

// Vector `u` of a row of a head: the units of the rotated part, then those that
// are copied.
struct Rotation {
    int64_t dim, half;     // elements of a head; pairs
    int rot, units;        // units of the rotated part and of the whole row
    int interleaved;
};
template <int DT>
__host__ __device__ inline Rotation rotation(int64_t dim, int64_t rotary, int interleaved) {
    constexpr int V = Elem<DT>::VEC;
    Rotation r;
    r.dim = dim;
    r.half = rotary / 2;
    r.interleaved = interleaved;
    r.rot = (int)((interleaved ? rotary : r.half) + V - 1) / V;
    r.units = r.rot + (int)((dim - rotary + V - 1) / V);
    return r;
}

template <int DT>
struct Unit {  // as read
    Vec16<DT> a, b;
};
template <int DT>
__device__ inline Unit<DT> load_unit(const Rotation& r, const typename Elem<DT>::type* x, int u) {
    constexpr int V = Elem<DT>::VEC;
    Unit<DT> out;
    if (u >= r.rot) out.a = dev::load_raw<DT>(x + 2 * r.half, (int64_t)(u - r.rot) * V, r.dim - 2 * r.half);
    else if (r.interleaved) out.a = dev::load_raw<DT>(x, (int64_t)u * V, 2 * r.half);
    else {
        out.a = dev::load_raw<DT>(x, (int64_t)u * V, r.half);
        out.b = dev::load_raw<DT>(x + r.half, (int64_t)u * V, r.half);
    }
    return out;
}
// Turns it by the table's (cos, sin) of the token's pairs and stores it.
template <int DT, bool NT = false>
__device__ inline void store_unit(const Rotation& r, typename Elem<DT>::type* y, int u, const Unit<DT>& in,
                                  const float2* cs) {
    constexpr int V = Elem<DT>::VEC;
    float a[V], b[V];
    dev::unpack<DT>(in.a, a);
    if (u >= r.rot) {
        dev::store_vec<DT, NT>(y + 2 * r.half, (int64_t)(u - r.rot) * V, r.dim - 2 * r.half, a);
    } else if (r.interleaved) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float2 t = cs[min((int64_t)(u * V + e) / 2, r.half - 1)];
            const float p = a[e], q = a[e + 1];
            a[e] = p * t.x - q * t.y;
            a[e + 1] = q * t.x + p * t.y;
        }
        dev::store_vec<DT, NT>(y, (int64_t)u * V, 2 * r.half, a);
    } else {
        dev::unpack<DT>(in.b, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 t = cs[min((int64_t)u * V + e, r.half - 1)];
            const float p = a[e], q = b[e];
            a[e] = p * t.x - q * t.y;
            b[e] = q * t.x + p * t.y;
        }
        dev::store_vec<DT, NT>(y, (int64_t)u * V, r.half, a);
        dev::store_vec<DT, NT>(y + r.half, (int64_t)u * V, r.half, b);
    }
}

// x and y may be the same rows: a unit is read before it is written, and by its
// thread alone (what a vector at a part's end holds of its neighbour is not used).
// blockIdx.y takes a share of the heads.
template <int DT, bool NT>
__global__ __launch_bounds__(THREADS) void rope_kernel(const typename Elem<DT>::type* x, const int32_t* positions,
                                                       const double* freqs, typename Elem<DT>::type* y, int64_t tokens,
                                                       int heads, int heads_each, Rotation r, int64_t x_stride,
                                                       int64_t y_stride, float magnitude, float sign) {
    extern __shared__ float2 cs[];  // [TK][half]
    const int64_t t0 = (int64_t)blockIdx.x * TK;
    const int n = (int)min((int64_t)TK, tokens - t0), half = (int)r.half;
    const int h0 = blockIdx.y * heads_each, hn = min(heads_each, heads - h0);
    // A token's heads' units in a row: unit fastest, so that a wave's vectors lie side by side.
    const int per = hn * r.units, all = n * per;
    constexpr int DEPTH = 3;
    Unit<DT> in[DEPTH];
    int tk[DEPTH], h[DEPTH], u[DEPTH];  // token, head and unit of each
    const auto load = [&](int i0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int i = i0 + d * THREADS;
            if (i < all) {
                tk[d] = (int)((uint32_t)i / (uint32_t)per);
                const int rest = i - tk[d] * per;
                h[d] = (int)((uint32_t)rest / (uint32_t)r.units);
                u[d] = rest - h[d] * r.units;
                in[d] = load_unit<DT>(r, x + (t0 + tk[d]) * x_stride + (h0 + h[d]) * r.dim, u[d]);
            }
        }
    };
    load((int)threadIdx.x);  // on its way while the table is formed
    for (int i = (int)threadIdx.x; i < n * half; i += THREADS) {
        const int tk = i / half, p = i - tk * half;
        const float2 c = cos_sin_turns((double)positions[t0 + tk] * freqs[p] * TURNS);
        cs[i] = {magnitude * c.x, magnitude * sign * c.y};
    }
    __syncthreads();
    for (int i0 = (int)threadIdx.x; i0 < all; i0 += DEPTH * THREADS) {
        if (i0 != (int)threadIdx.x) load(i0);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int i = i0 + d * THREADS;
            if (i < all) store_unit<DT, NT>(r, y + (t0 + tk[d]) * y_stride + (h0 + h[d]) * r.dim, u[d], in[d], cs + tk[d] * half);
        }
    }
}

__global__ void rope_frequencies_kernel(double* freqs, int half, double rotary, double base, double factor, double low,
                                        double high, double original) {
    for (int i = (int)threadIdx.x; i < half; i += THREADS) {
        const double f = pow(base, -2.0 * i / rotary);
        double keep = 0.0;
        if (original > 0.0) keep = fmin(fmax((original * f * TURNS - low) / (high - low), 0.0), 1.0);
        freqs[i] = factor == 1.0 ? f : f * (keep + (1.0 - keep) / factor);
    }
}

// ── append to pages ───────────────────────────────────────────────────────

// Where a new token goes: its sequence (of the 64 that it may lie in), its position from the
// sequence's length. page -1: nowhere (no sequence's token, or outside the table or the pages).
struct Place {
    int position, page;
};
__device__ inline Place place_of(int token, const PagedArgs& a) {
    const int lane = threadIdx.x & 63;
    const int base = 64 * dev::last_group((a.n_seqs + 63) / 64, [&](int g) { return a.starts[64 * g] <= token; }), i = base + lane;
    int first = 0, end = 0, length = 0;
    if (i < a.n_seqs) {
        first = a.starts[i];
        end = a.starts[i + 1];
        length = a.lens[i];
    }
    const uint64_t in = __ballot(first >= 0 && token >= first && token < end);
    if (!in) return {0, -1};
    const int at = __builtin_ctzll(in);
    const int64_t position = (int64_t)__builtin_amdgcn_readlane(length, at) - __builtin_amdgcn_readlane(end, at) + token;
    if (position < 0 || position >> a.page_shift >= a.table_width) return {0, -1};
    const int page = a.table[(int64_t)(base + at) * a.table_width + (position >> a.page_shift)];
    return {(int)position, page >= 0 && page < a.pages ? page : -1};
}

template <int DT>
__global__ __launch_bounds__(THREADS) void paged_append_kernel(const typename Elem<DT>::type* k,
                                                               const typename Elem<DT>::type* v, const double* freqs,
                                                               typename Elem<DT>::type* k_pages,
                                                               typename Elem<DT>::type* v_pages, PagedArgs a,
                                                               int64_t tokens, int kv_heads, int64_t kv_stride, Rotation r,
                                                               float magnitude) {
    extern __shared__ float2 cs[];
    __shared__ Place places[APPEND_TK];
    const int64_t t0 = (int64_t)blockIdx.x * APPEND_TK;
    const int n = (int)min((int64_t)APPEND_TK, tokens - t0), half = (int)r.half;
    // Units under way of a thread: more gained nothing. As plain variables in place of arrays of one the
    // bf16 kernel takes 82 registers for 68 (5001 tokens of 7 prompts, f16: 7.8 us for 7.6).
    constexpr int V = Elem<DT>::VEC, DEPTH = 1;
    // A head's units: K's, then V's, which are copied.
    const int per_head = r.units + (int)((r.dim + V - 1) / V), per = kv_heads * per_head, all = n * per;
    Unit<DT> in[DEPTH];
    int tk[DEPTH], h[DEPTH], u[DEPTH];
    const auto load = [&](int i0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int i = i0 + d * THREADS;
            if (i < all) {
                tk[d] = (int)((uint32_t)i / (uint32_t)per);
                const int rest = i - tk[d] * per;
                h[d] = (int)((uint32_t)rest / (uint32_t)per_head);
                u[d] = rest - h[d] * per_head;
                const int64_t from = (t0 + tk[d]) * kv_stride + h[d] * r.dim;
                if (u[d] < r.units) in[d] = load_unit<DT>(r, k + from, u[d]);
                else in[d].a = dev::load_raw<DT>(v + from, (int64_t)(u[d] - r.units) * V, r.dim);
            }
        }
    };
    load((int)threadIdx.x);  // on its way while the places are found
    const int w = (int)threadIdx.x / 64;
    if (w < n) {
        const Place p = place_of((int)(t0 + w), a);
        if (threadIdx.x % 64 == 0) places[w] = p;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < n * half; i += THREADS) {
        const int t = i / half, p = i - t * half;
        const float2 c = cos_sin_turns((double)places[t].position * freqs[p] * TURNS);
        cs[i] = {magnitude * c.x, magnitude * c.y};
    }
    if (half) __syncthreads();
    for (int i0 = (int)threadIdx.x; i0 < all; i0 += DEPTH * THREADS) {
        if (i0 != (int)threadIdx.x) load(i0);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (i0 + d * THREADS >= all) continue;
            const Place p = places[tk[d]];
            if (p.page < 0) continue;
            const int row = p.position & ((1 << a.page_shift) - 1);
            const int64_t to = ((((int64_t)p.page * kv_heads + h[d]) << a.page_shift) + row) * r.dim;
            if (u[d] < r.units) {
                store_unit<DT>(r, k_pages + to, u[d], in[d], cs + tk[d] * half);
            } else {
                float x[V];
                dev::unpack<DT>(in[d].a, x);
                dev::store_vec<DT>(v_pages + to, (int64_t)(u[d] - r.units) * V, r.dim, x);
            }
        }
    }
}

}  // namespace

int rope_frequencies(double* freqs, int64_t rotary, double base, double factor, double low, double high, int64_t original,
                     hipStream_t s) {
    hipLaunchKernelGGL(rope_frequencies_kernel, dim3(1), dim3(THREADS), 0, s, freqs, (int)(rotary / 2), (double)rotary, base,
                       factor, low, high, (double)original);
    return launch_check("rope_frequencies_kernel");
}

int rope_rows(int dtype, const void* x, const int32_t* positions, const double* freqs, void* y, int64_t tokens,
              int64_t heads, int64_t dim, int64_t rotary, int64_t x_stride, int64_t y_stride, int interleaved,
              float magnitude, bool vjp, hipStream_t s) {
    const int64_t groups = ceil_div(tokens, TK);
    // Few tokens: their heads over several workgroups, as long as each keeps a
    // vector for every other thread.
    int64_t each = heads;
    const int64_t vec = dtype == MLXHIP_DTYPE_F32 ? 4 : 8;
    while (each > 1 && groups * ceil_div(heads, each) < 512 && each * ceil_div(dim, vec) * std::min<int64_t>(TK, tokens) > 128)
        each = ceil_div(each, 2);
    const size_t lds = sizeof(float2) * (size_t)(std::min<int64_t>(TK, tokens) * rotary / 2);
    with_float_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        typedef typename Elem<DT>::type E;
        const auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)groups, (unsigned)ceil_div(heads, each)), dim3(THREADS), lds, s, (const E*)x,
                               positions, freqs, (E*)y, tokens, (int)heads, (int)each, rotation<DT>(dim, rotary, interleaved),
                               x_stride, y_stride, magnitude, vjp ? -1.0f : 1.0f);
        };
        // Rows of 64 MiB and more are stored past the caches (16384 tokens of 40 heads of 128,
        // bf16, both ways: 121 us, 130 through them; 6554: 48 and 51); smaller ones stay there for whoever reads
        // them next (4096: 31 and 34).
        if (tokens * heads * dim * (int64_t)sizeof(E) >= (int64_t(64) << 20)) launch(rope_kernel<DT, true>);
        else launch(rope_kernel<DT, false>);
    });
    return launch_check("rope_kernel");
}

int paged_append(int dtype, const void* k, const void* v, void* k_pages, void* v_pages, const PagedArgs& a, int64_t tokens,
                 int64_t kv_heads, int64_t dim, int64_t kv_stride, const double* freqs, int64_t rotary, int interleaved,
                 float magnitude, hipStream_t s) {
    if (!freqs) rotary = 0;
    const size_t lds = sizeof(float2) * (size_t)(std::min<int64_t>(APPEND_TK, tokens) * rotary / 2);
    with_float_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        typedef typename Elem<DT>::type E;
        hipLaunchKernelGGL(paged_append_kernel<DT>, dim3((unsigned)ceil_div(tokens, APPEND_TK)), dim3(THREADS), lds, s, (const E*)k,
                           (const E*)v, freqs, (E*)k_pages, (E*)v_pages, a, tokens, (int)kv_heads, kv_stride,
                           rotation<DT>(dim, rotary, interleaved), magnitude);
    });
    return launch_check("paged_append_kernel");
}

}  // namespace mlxhip
