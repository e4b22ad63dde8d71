// A language model's answer -- a row of logits x over V tokens for every place -- turned into what the Monte Carlo
// path works on (gfx950): the score of given tokens (calc_ml2p), with entropy and the most probable alternatives; the
// gradient of that score; draws with their probability (pick_expand, lib4mc/ProbLib.py:31-43); and the float64 keys
// of whole passwords.  With c = log2(e) / T, m = the row's largest logit, y = (x - m) c <= 0, w = 2^y, Z = sum of w:
//
//   score      -log2 p_t = log2 Z - y_t,   H = log2 Z - (sum of w y) / Z          (bits)
//   gradient   d/dx_i of a * (-log2 p_t) + b * H = (a (p_i - [i = t]) / ln 2 - b p_i (log2 p_i + H)) / T
//   draw       the first token whose running sum of weights exceeds u Z
//   keys       the sum of a password's -log2 p in 64 bits
//
// A row holds 10^2 .. 10^5 numbers that are read once: every kernel here is bound by HBM.  One pass keeps the running
// maximum, the sum scaled to it and the sum of w y in 32 bits (all terms are positive or all negative: no cancellation);
// a change of the maximum scales both.  The smallest finite float stands in for the maximum of a row (or a part of one)
// in which every logit is -inf, so that its weights are 0 and nothing becomes NaN by itself; NaN and +inf logits make
// Z NaN and with it every output of the row.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>

#include "mc_internal.h"
#include "mc_philox.h"

#define HIP_TRY(expr)                                                                        \
    do {                                                                                     \
        hipError_t e_ = (expr);                                                              \
        if (e_ != hipSuccess) {                                                              \
            mc_set_error("%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
            return MC_ERR_HIP;                                                               \
        }                                                                                    \
    } while (0)

namespace {

typedef unsigned long long u64;
typedef unsigned int u32;
typedef long long i64;

constexpr int BLOCK = 256, WAVES = BLOCK / 64;
constexpr float LOWEST = -FLT_MAX;
constexpr double LOG2E = 1.4426950408889634074;
// a step of the maximum beyond 2^-10000 loses everything summed before it: the bound keeps 0 * inf out of the sums
constexpr float FAR = -1e4f;

// A division by the same number for every row, as a multiplication: exact for row numbers below 2^31.
struct Div {
    u32 d, mul, shift;
};

Div make_div(u64 d) {
    Div r{(u32)d, 0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.mul = (u32)((((u64)1 << (31 + r.shift)) + d - 1) / d);
    return r;
}

// Something with a value (or a row of values) for every row, addressed by (row / inner, row % inner); strides in bytes.
struct View {
    const char *p;
    i64 os, is;
};

struct Rows {
    View logits, tokens;
    Div inner;
    u32 rows, vocab, nvec, token_bytes;
    float c;  // log2(e) / T
};

__device__ __forceinline__ const char *at(const View &v, const Div &inner, u32 row) {
    const u32 o = __umulhi(row << 1, inner.mul) >> inner.shift;
    return v.p + (i64)o * v.os + (i64)(row - o * inner.d) * v.is;
}

// A token id as the kernels use it: [0, V), MC_TOKEN_SKIP, or MC_TOKEN_OUTSIDE for everything else.
__device__ __forceinline__ int token_of(const Rows &a, u32 row) {
    const char *p = at(a.tokens, a.inner, row);
    const i64 t = a.token_bytes == 8 ? *(const i64 *)p : (i64) * (const int *)p;
    return t == MC_TOKEN_SKIP ? MC_TOKEN_SKIP : (t >= 0 && t < (i64)a.vocab) ? (int)t : MC_TOKEN_OUTSIDE;
}

// one workgroup a row: a grid of two dimensions, since one holds at most 2^32 work items
constexpr u32 GRID_X = 1u << 20;
__device__ __forceinline__ u32 row_of_block() { return blockIdx.y * GRID_X + blockIdx.x; }
u32 rows_to_blocks(u32 rows, u32 group) { return (u32)(((u64)rows * group + BLOCK - 1) / BLOCK); }
dim3 grid_of(u32 rows) { return rows <= GRID_X ? dim3(rows) : dim3(GRID_X, (rows + GRID_X - 1) / GRID_X); }

template <int DT>
struct Elt;
template <>
struct Elt<MC_LOGITS_F32> {
    static constexpr int BYTES = 4;
    static constexpr u32 NEG_INF = 0xFF800000u;
};
template <>
struct Elt<MC_LOGITS_F16> {
    static constexpr int BYTES = 2;
    static constexpr u32 NEG_INF = 0xFC00FC00u;
};
template <>
struct Elt<MC_LOGITS_BF16> {
    static constexpr int BYTES = 2;
    static constexpr u32 NEG_INF = 0xFF80FF80u;
};

template <int DT>
constexpr int VEC = 16 / Elt<DT>::BYTES;

// 16 bytes of a row; rows begin where they like (an odd number of 2-byte tokens), which the loads take as they are
typedef u32 raw4 __attribute__((ext_vector_type(4)));
typedef raw4 raw4_at2 __attribute__((aligned(2)));

template <int DT>
__device__ __forceinline__ float to_float(u32 word, int half) {
    if constexpr (DT == MC_LOGITS_F32) return __uint_as_float(word);
    if constexpr (DT == MC_LOGITS_BF16) return __uint_as_float(half ? word & 0xFFFF0000u : word << 16);
    if constexpr (DT == MC_LOGITS_F16) {
        const unsigned short h = (unsigned short)(half ? word >> 16 : word);
        return (float)__builtin_bit_cast(_Float16, h);
    }
}

template <int DT>
__device__ __forceinline__ float element(const char *row, u32 i) {
    if constexpr (Elt<DT>::BYTES == 4) return *(const float *)(row + 4 * (u64)i);
    else return to_float<DT>(*(const unsigned short *)(row + 2 * (u64)i), 0);
}

// element j of a vector of raw words
template <int DT>
__device__ __forceinline__ float unpack(const raw4 &q, int j) {
    if constexpr (Elt<DT>::BYTES == 4) return to_float<DT>(q[j], 0);
    else return to_float<DT>(q[j >> 1], j & 1);
}

// vector v of a row; what lies behind the row's end is -inf
template <int DT>
__device__ __forceinline__ raw4 load_vec(const char *row, u32 v, u32 nvec, u32 vocab) {
    constexpr u32 N = VEC<DT>;
    raw4 q = {Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF};
    if ((u64)v * N + N <= vocab) {
        q = *(const raw4_at2 *)(row + (u64)v * 16);
    } else if (v < nvec) {
#pragma unroll
        for (u32 j = 0; j < N; ++j) {
            if (v * N + j < vocab) {
                if constexpr (Elt<DT>::BYTES == 4) {
                    q[j] = *(const u32 *)(row + ((u64)v * N + j) * 4);
                } else {
                    const u32 h = *(const unsigned short *)(row + ((u64)v * N + j) * 2);
                    q[j >> 1] = (j & 1) ? (q[j >> 1] & 0xFFFFu) | (h << 16) : (q[j >> 1] & 0xFFFF0000u) | h;
                }
            }
        }
    }
    return q;
}

// one rounding to the logits' type, to nearest even
template <int DT>
__device__ __forceinline__ u32 pack2(float lo, float hi) {
    if constexpr (DT == MC_LOGITS_BF16)
        return (u32)__builtin_bit_cast(unsigned short, (__bf16)lo) | ((u32)__builtin_bit_cast(unsigned short, (__bf16)hi) << 16);
    else
        return (u32)__builtin_bit_cast(unsigned short, (_Float16)lo) | ((u32)__builtin_bit_cast(unsigned short, (_Float16)hi) << 16);
}

template <int DT>
__device__ __forceinline__ void store_at(char *row, u32 from, u32 vocab, const float *g) {
    constexpr u32 N = VEC<DT>;
    if ((u64)from + N <= vocab) {
        raw4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (Elt<DT>::BYTES == 4) q[j] = __float_as_uint(g[j]);
            else q[j] = pack2<DT>(g[2 * j], g[2 * j + 1]);
        }
        *(raw4_at2 *)(row + (u64)from * Elt<DT>::BYTES) = q;
    } else {
#pragma unroll
        for (u32 j = 0; j < N; ++j) {
            if (from + j < vocab) {
                if constexpr (Elt<DT>::BYTES == 4) *(float *)(row + ((u64)from + j) * 4) = g[j];
                else *(unsigned short *)(row + ((u64)from + j) * 2) = (unsigned short)pack2<DT>(g[j], 0.f);
            }
        }
    }
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// running maximum m (at least the lowest finite float), sum s of 2^((x - m) c) and sum e of the same times its exponent
struct Stat {
    float m, s, e;
};

__device__ __forceinline__ void rescale(Stat &st, float m, float c) {
    const float d = fmaxf((st.m - m) * c, FAR), f = exp2_(d);
    st.e = (st.e + d * st.s) * f;
    st.s *= f;
    st.m = m;
}

__device__ __forceinline__ void merge(Stat &a, Stat b, float c) {
    const float m = fmaxf(a.m, b.m);
    rescale(a, m, c);
    rescale(b, m, c);
    a.s += b.s;
    a.e += b.e;
}

template <int DT>
__device__ __forceinline__ float take(Stat &st, const raw4 &q, float c) {
    constexpr int N = VEC<DT>;
    float x[N], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        x[j] = unpack<DT>(q, j);
        m = fmaxf(m, x[j]);
    }
    rescale(st, fmaxf(st.m, m), c);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float y = (x[j] - st.m) * c, w = exp2_(y);
        st.s += w;
        st.e += w * fmaxf(y, FAR);
    }
    return m;
}

__device__ __forceinline__ Stat wave_stat(Stat st, float c) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        Stat o{__shfl_xor(st.m, d), __shfl_xor(st.s, d), __shfl_xor(st.e, d)};
        // both sides of a pair add in the same order, so that all lanes end with the same bits
        if (threadIdx.x & d) {
            merge(o, st, c);
            st = o;
        } else {
            merge(st, o, c);
        }
    }
    return st;
}

// the whole workgroup's, in every thread
__device__ __forceinline__ Stat block_stat(Stat st, float c) {
    __shared__ Stat part[WAVES];
    st = wave_stat(st, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
    __syncthreads();
    st = part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) merge(st, part[w], c);
    return st;
}

__device__ __forceinline__ u32 block_sum(u32 v) {
    __shared__ u32 part[WAVES];
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += part[w];
    return v;
}

// exclusive prefix sum over the workgroup and the total
template <typename A>
__device__ __forceinline__ A block_scan(A v, A &total) {
    __shared__ A part[WAVES];
    A inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const A o = __shfl_up(inc, d);
        if ((threadIdx.x & 63) >= (u32)d) inc += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = inc;
    __syncthreads();
    A base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < (int)(threadIdx.x >> 6)) base += part[w];
        total += part[w];
    }
    return base + inc - v;
}

__device__ __forceinline__ u32 block_min(u32 v) {
    __shared__ u32 part[WAVES];
#pragma unroll
    for (int d = 32; d; d >>= 1) v = min(v, (u32)__shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v = min(v, part[w]);
    return v;
}

// what a row's statistics say about its token
__device__ __forceinline__ float ml2p_of(int tok, const Stat &st, float x, float c) {
    if (tok == MC_TOKEN_SKIP) return 0.f;
    if (!(st.s == st.s)) return st.s;
    return tok >= 0 && st.s > 0.f ? log2f(st.s) - (x - st.m) * c : INFINITY;
}

__device__ __forceinline__ float entropy_of(int tok, const Stat &st) {
    return tok == MC_TOKEN_SKIP || st.s == 0.f ? 0.f : log2f(st.s) - st.e / st.s;
}

// ---- rows of few tokens: a group of G lanes a row, several rows a wave, the row in registers ---------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}

struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
    __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};

// the same bits in every lane of the group: each step joins two halves that hold one value each
template <int G, typename Op>
__device__ __forceinline__ float group_all(float x, Op op) {
    if constexpr (G >= 2) x = op(x, dpp<0xB1>(x));    // quad_perm 1 0 3 2
    if constexpr (G >= 4) x = op(x, dpp<0x4E>(x));    // quad_perm 2 3 0 1
    if constexpr (G >= 8) x = op(x, dpp<0x141>(x));   // half rows mirrored
    if constexpr (G >= 16) x = op(x, dpp<0x140>(x));  // rows mirrored
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return x;
}

template <int G, typename Op>
__device__ __forceinline__ double group_all(double x, Op op) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) x = op(x, __shfl_xor(x, d));
    return x;
}

// inclusive prefix sum over the lanes of a group
template <int G, typename A>
__device__ __forceinline__ A group_scan(A x) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        const A o = __shfl_up(x, d, G);
        if ((threadIdx.x & (G - 1)) >= (u32)d) x += o;
    }
    return x;
}

constexpr int SUB_NV = 8;  // vectors a lane holds at most

// Vector v of a row, 16 bytes whole: the last one of a row that is no multiple of it reaches back into the one before it.
// `from`: its first element's number; `own`: the first that is not the vector's before it.
template <int DT>
__device__ __forceinline__ raw4 load_sub(const char *row, u32 v, u32 nvec, u32 vocab, u32 &from, u32 &own) {
    constexpr u32 N = VEC<DT>;
    raw4 q = {Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF};
    from = own = v * N;
    if (v < nvec) {
        if (vocab < N) {
            q = load_vec<DT>(row, v, nvec, vocab);
        } else {
            from = min(own, vocab - N);
            q = *(const raw4_at2 *)(row + (u64)from * Elt<DT>::BYTES);
        }
    }
    return q;
}

// the vector with -inf in the places that are another one's
template <int DT>
__device__ __forceinline__ raw4 masked(raw4 q, u32 from, u32 own) {
    if (from == own) return q;
    const u32 n = own - from;
#pragma unroll
    for (u32 w = 0; w < 4; ++w) {
        u32 m;
        if constexpr (Elt<DT>::BYTES == 4) m = w < n ? 0xFFFFFFFFu : 0u;
        else m = (2 * w < n ? 0xFFFFu : 0u) | (2 * w + 1 < n ? 0xFFFF0000u : 0u);
        q[w] = (q[w] & ~m) | (Elt<DT>::NEG_INF & m);
    }
    return q;
}

template <int DT>
struct SubRow {
    raw4 q[SUB_NV];      // as loaded
    u32 from, own;       // of the lane's last vector (the others' are whole)
    u32 nv;              // vectors a lane holds, the same in the whole grid
};

template <int DT, int G>
__device__ __forceinline__ void load_row(SubRow<DT> &r, const char *p, const Rows &a, bool read) {
    const u32 lane = threadIdx.x & (G - 1);
    r.nv = (a.nvec + G - 1) / G;
    r.from = r.own = 0;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        if (i < (int)r.nv) r.q[i] = load_sub<DT>(p, i * G + lane, read ? a.nvec : 0u, a.vocab, r.from, r.own);
    }
}

template <int DT, int G>
__device__ __forceinline__ raw4 vec_of(const SubRow<DT> &r, int i) {
    return i + 1 == (int)r.nv ? masked<DT>(r.q[i], r.from, r.own) : r.q[i];
}

template <int DT, int G, bool ENT>
__device__ __forceinline__ Stat sub_stat(const SubRow<DT> &r, float c) {
    float m = LOWEST;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        if (i < (int)r.nv) {
            const raw4 q = vec_of<DT, G>(r, i);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) m = fmaxf(m, unpack<DT>(q, j));
        }
    }
    m = group_all<G>(m, Max());
    float s = 0.f, e = 0.f;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        if (i < (int)r.nv) {
            const raw4 q = vec_of<DT, G>(r, i);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float y = (unpack<DT>(q, j) - m) * c, w = exp2_(y);
                s += w;
                if (ENT) e += w * fmaxf(y, FAR);
            }
        }
    }
    return Stat{m, group_all<G>(s, Add()), ENT ? group_all<G>(e, Add()) : 0.f};
}

// ---- top alternatives ------------------------------------------------------------------------------------------
// The order is that of the logits themselves (equal logits: the lower index), so it never depends on a rounding.  A
// logit as a word whose unsigned order is the numbers' (both zeros alike):
__device__ __forceinline__ u32 order_of(float x) {
    const u32 b = __float_as_uint(x + 0.0f);
    return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(u32 o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr u32 ORDER_NEG_INF = 0x007FFFFFu;

constexpr int UNROLL = 4;            // vectors of a thread and a chunk
constexpr int CELL_ROWS = 32;        // cells of a thread
constexpr int LIST_CAP = 512, CAND_CAP = 1024;

// A pass over the row keeps, beside its sums, the largest logit of every cell (one thread's vectors of some chunks).  The
// k-th largest of the threads' largest is a lower bound of the k-th largest of all: only the few cells that reach
// it are looked at again.
struct TopShared {
    float cell[CELL_ROWS][BLOCK];
    float tmax[BLOCK];
    u64 cand[CAND_CAP];
    u32 list[LIST_CAP];
    u32 n_list, n_cand;
    float bound;
};

template <int DT>
__device__ __noinline__ u32 count_from(const char *row, u32 nvec, u32 vocab, u32 order) {
    u32 n = 0;
    for (u32 v = threadIdx.x; v < nvec; v += BLOCK) {
        const raw4 q = load_vec<DT>(row, v, nvec, vocab);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) n += order_of(unpack<DT>(q, j)) >= order;
    }
    return block_sum(n);
}

// The k largest when the candidates do not fit (rows of equal logits, orders made to defeat the cells): the k-th
// largest value by bits, unless `bound` is it already; then one pass in order of the index.
template <int DT>
__device__ __noinline__ u32 select_by_bits(TopShared &sh, const char *row, u32 nvec, u32 vocab, u32 k, u32 bound) {
    const u32 valid = count_from<DT>(row, nvec, vocab, ORDER_NEG_INF + 1);
    k = min(k, valid);
    if (k == 0) return 0;
    u32 kth = bound, above = bound >= ORDER_NEG_INF + 1 ? count_from<DT>(row, nvec, vocab, bound + 1) : 0xFFFFFFFFu;
    if (above >= k) {
        kth = 0;
        for (int b = 31; b >= 0; --b) {
            const u32 t = kth | (1u << b);
            if (count_from<DT>(row, nvec, vocab, t) >= k) kth = t;
        }
        above = count_from<DT>(row, nvec, vocab, kth + 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.n_cand = k - above;  // (those above come behind the equal ones, in any order)
    __syncthreads();
    u32 found = 0;
    for (u32 base = 0; base < nvec; base += BLOCK) {
        const u32 v = base + threadIdx.x;
        const raw4 q = load_vec<DT>(row, v, nvec, vocab);
        u32 n = 0;
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) n += order_of(unpack<DT>(q, j)) == kth;
        u32 total, place = found + block_scan(n, total);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) {
            const u32 o = order_of(unpack<DT>(q, j)), i = v * VEC<DT> + j;
            if (o == kth && place < k - above) sh.cand[place] = (u64)o << 32 | (0xFFFFFFFFu - i);
            place += o == kth;
            if (o > kth) sh.cand[atomicAdd(&sh.n_cand, 1u)] = (u64)o << 32 | (0xFFFFFFFFu - i);
        }
        found += total;
    }
    __syncthreads();
    return k;
}

// all candidates of the k largest into sh.cand: their number
template <int DT>
__device__ u32 select(TopShared &sh, const char *row, u32 nvec, u32 vocab, u32 k, float tmax, u32 chunks_per_cell) {
    sh.tmax[threadIdx.x] = tmax;
    if (threadIdx.x == 0) sh.n_list = sh.n_cand = 0;
    __syncthreads();
    u32 rank = 0;
    for (int i = 0; i < BLOCK; ++i) rank += sh.tmax[i] > tmax || (sh.tmax[i] == tmax && i < (int)threadIdx.x);
    if (rank == k - 1) sh.bound = tmax;
    __syncthreads();
    const float bound = sh.bound;
    const u32 cell_vecs = chunks_per_cell * UNROLL;
    for (u32 r = 0; r * cell_vecs * BLOCK < nvec; ++r) {
        const float m = sh.cell[r][threadIdx.x];
        if (m >= bound && m > -INFINITY) {
            const u32 n = atomicAdd(&sh.n_list, 1u);
            if (n < LIST_CAP) sh.list[n] = r * BLOCK + threadIdx.x;
        }
    }
    __syncthreads();
    const u32 n_list = sh.n_list;
    if (n_list <= LIST_CAP) {
        for (u32 i = threadIdx.x; i < n_list * cell_vecs; i += BLOCK) {
            const u32 cell = sh.list[i / cell_vecs], u = i % cell_vecs;
            const u32 v = ((cell / BLOCK) * cell_vecs + u) * BLOCK + cell % BLOCK;
            const raw4 q = load_vec<DT>(row, v, nvec, vocab);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float x = unpack<DT>(q, j);
                if (x >= bound && x > -INFINITY) {
                    const u32 n = atomicAdd(&sh.n_cand, 1u);
                    if (n < CAND_CAP) sh.cand[n] = (u64)order_of(x) << 32 | (0xFFFFFFFFu - (v * VEC<DT> + j));
                }
            }
        }
    }
    __syncthreads();
    const u32 n = sh.n_cand;
    if (n_list <= LIST_CAP && n <= CAND_CAP) return n;
    return select_by_bits<DT>(sh, row, nvec, vocab, k, order_of(bound));
}

// ---- score ---------------------------------------------------------------------------------------------------------
struct ScoreOut {
    float *ml2p, *entropy, *top_ml2p;
    int *top;
    u32 k;
};

template <int DT, bool TOP>
__global__ __launch_bounds__(BLOCK) void k_logits_score(Rows a, ScoreOut out) {
    __shared__ typename std::conditional<TOP, TopShared, int>::type sh;
    const u32 row = row_of_block();
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    if (tok == MC_TOKEN_SKIP) {
        if (threadIdx.x == 0) {
            out.ml2p[row] = 0.f;
            if (out.entropy) out.entropy[row] = 0.f;
        }
        if (TOP && threadIdx.x < out.k) {
            out.top[(u64)row * out.k + threadIdx.x] = MC_TOKEN_SKIP;
            out.top_ml2p[(u64)row * out.k + threadIdx.x] = 0.f;
        }
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const u32 chunks = (a.nvec + BLOCK * UNROLL - 1) / (BLOCK * UNROLL), per_cell = (chunks + CELL_ROWS - 1) / CELL_ROWS;
    Stat st{LOWEST, 0.f, 0.f};
    float cell = -INFINITY, tmax = -INFINITY;
    for (u32 ch = 0; ch < chunks; ++ch) {
        raw4 q[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) q[u] = load_vec<DT>(p, (ch * UNROLL + u) * BLOCK + threadIdx.x, a.nvec, a.vocab);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const float m = take<DT>(st, q[u], a.c);
            if (TOP) cell = fmaxf(cell, m);
        }
        if constexpr (TOP) {
            if ((ch + 1) % per_cell == 0 || ch + 1 == chunks) {
                sh.cell[ch / per_cell][threadIdx.x] = cell;
                tmax = fmaxf(tmax, cell);
                cell = -INFINITY;
            }
        }
    }
    st = block_stat(st, a.c);
    if (threadIdx.x == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (out.entropy) out.entropy[row] = entropy_of(tok, st);
    }
    if constexpr (TOP) {
        const u32 k = out.k;
        int *ids = out.top + (u64)row * k;
        float *vals = out.top_ml2p + (u64)row * k;
        const bool bad = !(st.s == st.s);
        u32 n = 0;
        if (!bad && st.s > 0.f) n = select<DT>(sh, p, a.nvec, a.vocab, k, tmax, per_cell);
        for (u32 i = threadIdx.x; i < n; i += BLOCK) {
            const u64 key = sh.cand[i];
            u32 rank = 0;
            for (u32 j = 0; j < n; ++j) rank += sh.cand[j] > key;
            if (rank < k) {
                const float v = log2f(st.s) - (value_of((u32)(key >> 32)) - st.m) * a.c;
                ids[rank] = v == INFINITY ? MC_TOKEN_OUTSIDE : (int)(0xFFFFFFFFu - (u32)key);
                vals[rank] = v;
            }
        }
        for (u32 i = n + threadIdx.x; i < k; i += BLOCK) {
            ids[i] = MC_TOKEN_OUTSIDE;
            vals[i] = bad ? st.s : INFINITY;
        }
    }
}

// The k largest of a row in registers, one after the other: the largest that comes behind the last one in the order (logit
// descending, index ascending).
template <int DT, int G>
__device__ __forceinline__ void sub_top(const SubRow<DT> &r, const Rows &a, const Stat &st, const ScoreOut &out, u32 row, bool writes, int fill,
                                        float fill_value) {
    const u32 lane = threadIdx.x & (G - 1);
    const float lz = log2f(st.s);
    float last = INFINITY;
    u32 last_i = 0xFFFFFFFFu;
    for (u32 k = 0; k < out.k; ++k) {
        float best = -INFINITY;
        u32 best_i = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < SUB_NV; ++i) {
            if (i < (int)r.nv) {
                const raw4 q = vec_of<DT, G>(r, i);
                const u32 from = i + 1 == (int)r.nv ? r.from : (i * G + lane) * VEC<DT>;
#pragma unroll
                for (int j = 0; j < VEC<DT>; ++j) {
                    const float x = unpack<DT>(q, j);
                    const bool open = x < last || (x == last && from + j > last_i);
                    if (open && x > best) best = x, best_i = from + j;
                }
            }
        }
        const float top = group_all<G>(best, Max());
        u32 at = best == top ? best_i : 0xFFFFFFFFu;
#pragma unroll
        for (int d = 1; d < G; d <<= 1) at = min(at, (u32)__shfl_xor(at, d));
        const float v = lz - (top - st.m) * a.c;
        const bool there = fill == 0 && top > -INFINITY && v < INFINITY;
        if (writes && lane == 0) {
            out.top[(u64)row * out.k + k] = there ? (int)at : fill == 0 ? MC_TOKEN_OUTSIDE : fill;
            out.top_ml2p[(u64)row * out.k + k] = there ? v : fill == 0 ? INFINITY : fill_value;
        }
        last = top;
        last_i = at;
    }
}

template <int DT, int G, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_logits_score_sub(Rows a, ScoreOut out) {
    const u32 row = row_of_block() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows;
    const int tok = there ? token_of(a, row) : MC_TOKEN_SKIP;
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT> r;
    load_row<DT, G>(r, p, a, tok != MC_TOKEN_SKIP);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const Stat st = sub_stat<DT, G, ENT>(r, a.c);
    if (there && lane == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (ENT) out.entropy[row] = entropy_of(tok, st);
    }
    if (out.k) {
        const bool bad = !(st.s == st.s);
        sub_top<DT, G>(r, a, st, out, row, there, tok == MC_TOKEN_SKIP ? MC_TOKEN_SKIP : bad ? MC_TOKEN_OUTSIDE : 0,
                       tok == MC_TOKEN_SKIP ? 0.f : st.s);
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------------
struct GradOut {
    View weights, entropy_weights;  // entropy_weights.p may be null
    float inv_t;
    float *ml2p, *entropy;
    char *grad;
};

template <int DT>
__global__ __launch_bounds__(BLOCK) void k_logits_gradient(Rows a, GradOut out) {
    const u32 row = row_of_block();
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    const char *p = at(a.logits, a.inner, row);
    char *gp = out.grad + (u64)row * a.vocab * Elt<DT>::BYTES;
    Stat st{LOWEST, 0.f, 0.f};
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    if (tok != MC_TOKEN_SKIP) {
        for (u32 base = 0; base < a.nvec; base += BLOCK * UNROLL) {
            raw4 q[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) q[u] = load_vec<DT>(p, base + u * BLOCK + threadIdx.x, a.nvec, a.vocab);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) take<DT>(st, q[u], a.c);
        }
        st = block_stat(st, a.c);
    }
    if (threadIdx.x == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (out.entropy) out.entropy[row] = entropy_of(tok, st);
    }
    const bool none = tok == MC_TOKEN_SKIP || st.s == 0.f;
    const float A = tok >= 0 ? *(const float *)at(out.weights, a.inner, row) * (a.c) : 0.f;
    const float B = out.entropy_weights.p ? *(const float *)at(out.entropy_weights, a.inner, row) * out.inv_t : 0.f;
    const float inv = 1.f / st.s, off = entropy_of(tok, st) - log2f(st.s);
    for (u32 v = threadIdx.x; v < a.nvec; v += BLOCK) {
        float g[VEC<DT>];
        if (none) {
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) g[j] = 0.f;
        } else {
            const raw4 q = load_vec<DT>(p, v, a.nvec, a.vocab);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float y = (unpack<DT>(q, j) - st.m) * a.c, pr = exp2_(y) * inv;
                g[j] = pr * (A - B * (fmaxf(y, FAR) + off));
                if ((int)(v * VEC<DT> + j) == tok) g[j] -= A;
            }
        }
        store_at<DT>(gp, v * VEC<DT>, a.vocab, g);
    }
}

template <int DT, int G, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_logits_gradient_sub(Rows a, GradOut out) {
    const u32 row = row_of_block() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows;
    const int tok = there ? token_of(a, row) : MC_TOKEN_SKIP;
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT> r;
    load_row<DT, G>(r, p, a, tok != MC_TOKEN_SKIP);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const float A = tok >= 0 ? *(const float *)at(out.weights, a.inner, row) * a.c : 0.f;
    const float B = ENT && there ? *(const float *)at(out.entropy_weights, a.inner, row) * out.inv_t : 0.f;
    const Stat st = sub_stat<DT, G, ENT>(r, a.c);
    if (!there) return;
    if (lane == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (ENT) out.entropy[row] = entropy_of(tok, st);
    }
    const bool none = tok == MC_TOKEN_SKIP || st.s == 0.f;
    const float inv = none ? 0.f : 1.f / st.s, off = ENT ? entropy_of(tok, st) - log2f(st.s) : 0.f;
    char *gp = out.grad + (u64)row * a.vocab * Elt<DT>::BYTES;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        if (i < (int)r.nv && i * G + lane < a.nvec) {
            // (a last vector that reaches back computes and stores what the one before it does)
            const u32 from = none || a.vocab < VEC<DT> ? min((i * G + lane) * VEC<DT>, a.vocab < VEC<DT> ? 0u : a.vocab - VEC<DT>)
                             : i + 1 == (int)r.nv ? r.from : (i * G + lane) * VEC<DT>;
            float g[VEC<DT>];
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float y = (unpack<DT>(r.q[i], j) - st.m) * a.c, pr = exp2_(y) * inv;
                g[j] = ENT ? pr * (A - B * (fmaxf(y, FAR) + off)) : pr * A;
                if ((int)(from + j) == tok) g[j] -= A;
                if (none) g[j] = 0.f;
            }
            store_at<DT>(gp, from, a.vocab, g);
        }
    }
}

// ---- draw ----------------------------------------------------------------------------------------------------------
struct DrawArgs {
    const double *uniforms;  // or null: Philox
    u64 seed, first_id;
    u32 draw;
    double t, eps;
    const unsigned char *live;
    int *token;
    float *ml2p;
};

__device__ __forceinline__ double uniform_of(const DrawArgs &d, u32 row) {
    if (d.uniforms) {
        const double u = d.uniforms[row];
        return u > 0. ? u : 0.;
    }
    const u64 id = d.first_id + row;
    u32 o0, o1, o2, o3;
    philox4x32_10((u32)id, (u32)(id >> 32), d.draw >> 1, 0u, (u32)d.seed, (u32)(d.seed >> 32), o0, o1, o2, o3);
    const u32 a = d.draw & 1 ? o2 : o0, b = d.draw & 1 ? o3 : o1;
    return (double)((u64)(a >> 5) << 26 | b >> 6) * 0x1p-53;
}

template <typename A>
__device__ __forceinline__ A weight(float x, float m, float c, double t) {
    if constexpr (sizeof(A) == 4) return exp2_((x - m) * c);
    else return exp(((double)x - (double)m) / t);
}

// The token that u falls on, in sums of type A with the row's maximum known: the first whose running sum exceeds u Z.
// `eps`: how far off a running sum may be, as a share of Z; false when u Z lies nearer than that to either end of the
// token's interval.  0 takes any answer.
template <int DT, typename A>
__device__ bool draw_row(const char *p, const Rows &a, const DrawArgs &d, float m, double u, double eps, u32 &token) {
    A mine = 0;
    for (u32 v = threadIdx.x; v < a.nvec; v += BLOCK) {
        const raw4 q = load_vec<DT>(p, v, a.nvec, a.vocab);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) mine += weight<A>(unpack<DT>(q, j), m, a.c, d.t);
    }
    A total;
    block_scan(mine, total);
    const double z = (double)total, target = u * z;
    double before = 0.;
    u32 last = 0;
    __shared__ u32 hit;
    __shared__ int sure;
    if (threadIdx.x == 0) hit = 0xFFFFFFFFu;
    for (u32 base = 0; base < a.nvec; base += BLOCK) {
        const u32 v = base + threadIdx.x;
        const raw4 q = load_vec<DT>(p, v, a.nvec, a.vocab);
        A w[VEC<DT>], s = 0;
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) {
            w[j] = weight<A>(unpack<DT>(q, j), m, a.c, d.t);
            if (w[j] > 0) last = v * VEC<DT> + j;
            s += w[j];
        }
        A step;
        const double lo = before + (double)block_scan(s, step);
        const u32 first = block_min(lo + (double)s > target ? threadIdx.x : 0xFFFFFFFFu);
        if (first != 0xFFFFFFFFu) {
            if (threadIdx.x == first) {
                double run = lo;
                u32 got = 0xFFFFFFFFu;
                bool ok = false;
#pragma unroll
                for (int j = 0; j < VEC<DT>; ++j) {
                    const double next = run + (double)w[j];
                    if (got == 0xFFFFFFFFu && w[j] > 0 && next > target) {
                        got = v * VEC<DT> + j;
                        ok = target - run >= eps * z && next - target >= eps * z;
                    }
                    run = next;
                }
                if (got == 0xFFFFFFFFu) got = last;  // (the vector's sum exceeds the target, its running sum by a rounding not)
                hit = got;
                sure = ok;
            }
            __syncthreads();
            token = hit;
            return eps == 0. || sure;
        }
        before += (double)step;
    }
    // u Z at or behind the last running sum: the last token with any weight
    token = 0xFFFFFFFFu - block_min(0xFFFFFFFFu - last);
    return eps == 0.;
}

template <int DT>
__global__ __launch_bounds__(BLOCK) void k_logits_draw(Rows a, DrawArgs d) {
    const u32 row = row_of_block();
    if (row >= a.rows) return;
    if (d.live && !d.live[row]) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_SKIP;
            d.ml2p[row] = 0.f;
        }
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    Stat st{LOWEST, 0.f, 0.f};
    for (u32 v = threadIdx.x; v < a.nvec; v += BLOCK) take<DT>(st, load_vec<DT>(p, v, a.nvec, a.vocab), a.c);
    st = block_stat(st, a.c);
    u32 token = 0;
    if (st.s > 0.f) {
        const double u = uniform_of(d, row);
        draw_row<DT, double>(p, a, d, st.m, u, 0., token);
    }
    if (threadIdx.x == 0) {
        d.token[row] = st.s > 0.f ? (int)token : MC_TOKEN_OUTSIDE;
        d.ml2p[row] = st.s > 0.f ? ml2p_of(0, st, element<DT>(p, token), a.c) : st.s == 0.f ? INFINITY : st.s;
    }
}

// draw_row for a group's row in registers: running sums in the order of the index, vector by vector of the lanes
template <int DT, int G, typename A>
__device__ __forceinline__ bool draw_sub(const SubRow<DT> &r, const Rows &a, const DrawArgs &d, float m, double u, double eps, u32 &token) {
    const u32 lane = threadIdx.x & (G - 1);
    A s[SUB_NV], z = 0;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        s[i] = 0;
        if (i < (int)r.nv) {
            const raw4 q = vec_of<DT, G>(r, i);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) s[i] += weight<A>(unpack<DT>(q, j), m, a.c, d.t);
            z += s[i];
        }
    }
    z = group_all<G>(z, Add());
    const double target = u * (double)z;
    // the vector step whose running sum passes the target, or the last one with any weight
    double before = 0., run = 0.;
    A mine = 0;
    raw4 q = r.q[0];
    u32 from = lane * VEC<DT>;
    bool found = false;
#pragma unroll
    for (int i = 0; i < SUB_NV; ++i) {
        if (i < (int)r.nv) {
            const double step = (double)group_all<G>(s[i], Add());
            if (!found && step > 0.) {
                before = run;
                mine = s[i];
                q = vec_of<DT, G>(r, i);
                from = i + 1 == (int)r.nv ? r.from : (i * G + lane) * VEC<DT>;
                found = run + step > target;
            }
            run += step;
        }
    }
    const A inc = group_scan<G>(mine);
    const double lo = before + (double)(inc - mine);
    const u32 shift = threadIdx.x & 63 & ~(G - 1);
    const u64 all = G == 64 ? ~0ull : (1ull << (G & 63)) - 1;
    const u64 passes = (__ballot(before + (double)inc > target) >> shift) & all, some = (__ballot(mine > 0) >> shift) & all;
    // (a sum that passes by a rounding only, or none: the last lane with any weight)
    const bool hit = found && passes;
    const u32 who = hit ? (u32)__ffsll((unsigned long long)passes) - 1 : some ? 63u - (u32)__clzll((long long)some) : 0u;
    double at_lo = lo;
    u32 got = 0xFFFFFFFFu, last = 0;
    bool ok = false;
#pragma unroll
    for (int j = 0; j < VEC<DT>; ++j) {
        const A w = weight<A>(unpack<DT>(q, j), m, a.c, d.t);
        const double next = at_lo + (double)w;
        if (w > 0) {
            last = from + j;
            if (got == 0xFFFFFFFFu && next > target) {
                got = from + j;
                ok = hit && target - at_lo >= eps * (double)z && next - target >= eps * (double)z;
            }
        }
        at_lo = next;
    }
    if (!hit || got == 0xFFFFFFFFu) got = last;
    token = __shfl(got, who, G);
    return __shfl((int)ok, who, G) || eps == 0.;
}

template <int DT, int G>
__global__ __launch_bounds__(BLOCK) void k_logits_draw_sub(Rows a, DrawArgs d) {
    const u32 row = row_of_block() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows, live = there && (!d.live || d.live[row]);
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT> r;
    load_row<DT, G>(r, p, a, live);
    const double u = there ? uniform_of(d, row) : 0.;
    const Stat st = sub_stat<DT, G, false>(r, a.c);
    u32 token = 0;
    bool sure = draw_sub<DT, G, float>(r, a, d, st.m, u, d.eps, token);
    if (!(st.s > 0.f)) sure = true, token = 0;
    if (__ballot(!sure)) {  // (a few rows in a million: the whole wave decides again in 64 bits)
        u32 again;
        draw_sub<DT, G, double>(r, a, d, st.m, u, 0., again);
        if (!sure) token = again;
    }
    if (there && lane == 0) {
        d.token[row] = !live ? MC_TOKEN_SKIP : st.s > 0.f ? (int)token : MC_TOKEN_OUTSIDE;
        d.ml2p[row] = !live ? 0.f : st.s > 0.f ? ml2p_of(0, st, element<DT>(p, token), a.c) : st.s == 0.f ? INFINITY : st.s;
    }
}

// ---- keys ----------------------------------------------------------------------------------------------------------
// one lane a password
__global__ __launch_bounds__(BLOCK) void k_logits_keys(const float *ml2p, const i64 *offsets, const void *lengths, u32 length_bytes,
                                                       u64 count, i64 stride, u64 longest, double *out) {
    for (u64 i = (u64)blockIdx.x * BLOCK + threadIdx.x; i < count; i += (u64)gridDim.x * BLOCK) {
        u64 from = 0, to = 0;
        const float *p = ml2p;
        if (offsets) {
            // (offsets that do not ascend or leave the array name no symbols: nothing is read through them)
            const i64 lo = offsets[i], hi = offsets[i + 1];
            if (lo >= 0 && hi > lo && (u64)hi <= longest) from = (u64)lo, to = (u64)hi;
        } else {
            p += (i64)i * stride;
            const i64 n = length_bytes == 8 ? ((const i64 *)lengths)[i] : length_bytes == 4 ? (i64)((const int *)lengths)[i] : (i64)longest;
            to = n < 0 ? 0 : (u64)n > longest ? longest : (u64)n;
        }
        double s = 0.;
        for (u64 k = from; k < to; ++k) s += (double)p[k];
        out[i] = s == INFINITY ? 1022.0 : s;
    }
}

// A group of lanes a row while a row's vectors fit the registers of 64 lanes (4096 tokens of two bytes), else a workgroup.
constexpr u32 SUB_VECS = 64 * SUB_NV;

#define BY_GROUP(nvec, ...)                              \
    if ((nvec) <= 4 * SUB_NV) { constexpr int G = 4; __VA_ARGS__; }        \
    else if ((nvec) <= 8 * SUB_NV) { constexpr int G = 8; __VA_ARGS__; }   \
    else if ((nvec) <= 16 * SUB_NV) { constexpr int G = 16; __VA_ARGS__; } \
    else if ((nvec) <= 32 * SUB_NV) { constexpr int G = 32; __VA_ARGS__; } \
    else { constexpr int G = 64; __VA_ARGS__; }

// How far off a running sum of weights in 32 bits may be as a share of the whole: the weights' own errors (the exponent's
// three roundings weigh at most 2.1 log2 V of half a step in the sum, the power's own 2) and one half step for each of
// the additions behind each other (a lane's vectors, then the joining of lanes); twice, since the target is such a sum too.
double error_of_sums(const Rows &a) { return 0x1p-24 * 2. * (SUB_NV * 8 + 16 + 8 + 2.1 * std::log2((double)a.vocab)); }

int bad(const char *who, const char *why) {
    mc_set_error("%s: %s", who, why);
    return MC_ERR_ARG;
}

bool one_run(uint64_t inner, int64_t outer_stride, int64_t inner_stride) { return outer_stride == (int64_t)inner * inner_stride; }

// the arguments that every entry point on logits shares
// (`flat`: everything else that a row has lies as one run too)
int rows_of(const char *who, Rows &a, const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
            int64_t outer_stride, int64_t inner_stride, double temperature, bool flat) {
    if (dtype > MC_LOGITS_BF16) return bad(who, "unknown element type");
    if (vocab == 0 || vocab >= (1ull << 31) - 64) return bad(who, "the vocabulary holds 1 .. 2^31 - 65 tokens");
    if (outer >= (1ull << 31) || inner >= (1ull << 31) || outer * inner >= (1ull << 31)) return bad(who, "at most 2^31 - 1 rows");
    if (!(temperature >= 1e-30 && temperature <= 1e30)) return bad(who, "the temperature is a positive number (1e-30 .. 1e30)");
    if (outer * inner && !logits) return bad(who, "no logits");
    const int bytes = dtype == MC_LOGITS_F32 ? 4 : 2;
    if ((uintptr_t)logits % bytes) return bad(who, "logits that are not aligned to their type");
    a.rows = (u32)(outer * inner);
    if (outer > 1 && flat && one_run(inner, outer_stride, inner_stride)) {
        inner *= outer;
        outer = 1;
    }
    a.logits = View{(const char *)logits, outer_stride * bytes, inner_stride * bytes};
    a.inner = make_div(inner ? inner : 1);
    a.vocab = (u32)vocab;
    a.nvec = (u32)((vocab + 16 / bytes - 1) / (16 / bytes));
    a.c = (float)(LOG2E / temperature);
    return MC_OK;
}

int tokens_of(const char *who, Rows &a, const void *tokens, uint32_t token_bytes, int64_t outer_stride, int64_t inner_stride, uint64_t rows) {
    if (token_bytes != 4 && token_bytes != 8) return bad(who, "token ids of 4 or 8 bytes");
    if (rows && !tokens) return bad(who, "no tokens");
    if ((uintptr_t)tokens % token_bytes) return bad(who, "tokens that are not aligned to their type");
    a.token_bytes = token_bytes;
    a.tokens = View{(const char *)tokens, outer_stride * (i64)token_bytes, inner_stride * (i64)token_bytes};
    return MC_OK;
}

}  // namespace

#define BY_TYPE(dtype, ...)                            \
    switch (dtype) {                                    \
        case MC_LOGITS_F32: { constexpr int DT = MC_LOGITS_F32; __VA_ARGS__; break; }   \
        case MC_LOGITS_F16: { constexpr int DT = MC_LOGITS_F16; __VA_ARGS__; break; }   \
        default: { constexpr int DT = MC_LOGITS_BF16; __VA_ARGS__; break; }             \
    }

extern "C" int mc_logits_score(const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
                               int64_t outer_stride, int64_t inner_stride, const void *tokens, uint32_t token_bytes,
                               int64_t token_outer_stride, int64_t token_inner_stride, double temperature, float *out_ml2p,
                               float *out_entropy, uint32_t top, int32_t *out_top, float *out_top_ml2p, void *stream) {
    const char *who = "mc_logits_score";
    Rows a{};
    if (int rc = tokens_of(who, a, tokens, token_bytes, token_outer_stride, token_inner_stride, outer * inner)) return rc;
    if (int rc = rows_of(who, a, logits, dtype, outer, inner, vocab, outer_stride, inner_stride, temperature,
                         one_run(inner, token_outer_stride, token_inner_stride)))
        return rc;
    if (top > MC_LOGITS_MAX_TOP || top > vocab) return bad(who, "top: at most 64 alternatives, and no more than tokens");
    if (a.rows == 0) return MC_OK;
    if (!out_ml2p || (top && (!out_top || !out_top_ml2p))) return bad(who, "no output");
    ScoreOut out{out_ml2p, out_entropy, out_top_ml2p, out_top, top};
    hipStream_t s = (hipStream_t)stream;
    if (a.nvec <= SUB_VECS) {
        BY_TYPE(dtype, BY_GROUP(a.nvec, {
                    if (out_entropy) hipLaunchKernelGGL((k_logits_score_sub<DT, G, true>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, out);
                    else hipLaunchKernelGGL((k_logits_score_sub<DT, G, false>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, out);
                }));
    } else if (top) {
        BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_score<DT, true>), grid_of(a.rows), dim3(BLOCK), 0, s, a, out));
    } else {
        BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_score<DT, false>), grid_of(a.rows), dim3(BLOCK), 0, s, a, out));
    }
    HIP_TRY(hipGetLastError());
    return MC_OK;
}

extern "C" int mc_logits_gradient(const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
                                  int64_t outer_stride, int64_t inner_stride, const void *tokens, uint32_t token_bytes,
                                  int64_t token_outer_stride, int64_t token_inner_stride, double temperature,
                                  const float *weights, int64_t weight_outer_stride, int64_t weight_inner_stride,
                                  const float *entropy_weights, int64_t entropy_outer_stride, int64_t entropy_inner_stride,
                                  float *out_ml2p, float *out_entropy, void *out_grad, void *stream) {
    const char *who = "mc_logits_gradient";
    Rows a{};
    if (int rc = tokens_of(who, a, tokens, token_bytes, token_outer_stride, token_inner_stride, outer * inner)) return rc;
    const bool flat = one_run(inner, token_outer_stride, token_inner_stride) && one_run(inner, weight_outer_stride, weight_inner_stride) &&
                      (!entropy_weights || one_run(inner, entropy_outer_stride, entropy_inner_stride));
    if (int rc = rows_of(who, a, logits, dtype, outer, inner, vocab, outer_stride, inner_stride, temperature, flat)) return rc;
    if (a.rows == 0) return MC_OK;
    if (!weights) return bad(who, "no weights");
    if (!out_ml2p || !out_grad) return bad(who, "no output");
    if ((uintptr_t)out_grad % (dtype == MC_LOGITS_F32 ? 4 : 2)) return bad(who, "a gradient that is not aligned to its type");
    GradOut out{View{(const char *)weights, weight_outer_stride * 4, weight_inner_stride * 4},
                View{(const char *)entropy_weights, entropy_outer_stride * 4, entropy_inner_stride * 4},
                (float)(1.0 / temperature), out_ml2p, out_entropy, (char *)out_grad};
    if (a.nvec <= SUB_VECS) {
        BY_TYPE(dtype, BY_GROUP(a.nvec, {
                    if (entropy_weights) hipLaunchKernelGGL((k_logits_gradient_sub<DT, G, true>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, (hipStream_t)stream, a, out);
                    else hipLaunchKernelGGL((k_logits_gradient_sub<DT, G, false>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, (hipStream_t)stream, a, out);
                }));
    } else BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_gradient<DT>), grid_of(a.rows), dim3(BLOCK), 0, (hipStream_t)stream, a, out));
    HIP_TRY(hipGetLastError());
    return MC_OK;
}

extern "C" int mc_logits_draw(const void *logits, uint32_t dtype, uint64_t rows, uint64_t vocab, int64_t row_stride,
                              double temperature, const double *uniforms, uint64_t seed, uint64_t first_id, uint32_t draw,
                              const uint8_t *live, int32_t *out_token, float *out_ml2p, void *stream) {
    const char *who = "mc_logits_draw";
    Rows a{};
    if (int rc = rows_of(who, a, logits, dtype, 1, rows, vocab, 0, row_stride, temperature, true)) return rc;
    if (a.rows == 0) return MC_OK;
    if (!out_token || !out_ml2p) return bad(who, "no output");
    DrawArgs d{uniforms, seed, first_id, draw, temperature, error_of_sums(a), live, out_token, out_ml2p};
    if (a.nvec <= SUB_VECS) {
        BY_TYPE(dtype, BY_GROUP(a.nvec, hipLaunchKernelGGL((k_logits_draw_sub<DT, G>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, (hipStream_t)stream, a, d)));
    } else BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_draw<DT>), grid_of(a.rows), dim3(BLOCK), 0, (hipStream_t)stream, a, d));
    HIP_TRY(hipGetLastError());
    return MC_OK;
}

extern "C" int mc_logits_keys(const float *ml2p, const int64_t *offsets, const void *lengths, uint32_t length_bytes,
                              uint64_t count, int64_t stride, uint64_t longest, double *out_keys, void *stream) {
    const char *who = "mc_logits_keys";
    if (count >= (1ull << 40)) return bad(who, "too many passwords");
    if (offsets && lengths) return bad(who, "offsets or lengths, not both");
    if (lengths && length_bytes != 4 && length_bytes != 8) return bad(who, "lengths of 4 or 8 bytes");
    if (count == 0) return MC_OK;
    if (!out_keys || (longest && !ml2p)) return bad(who, "null pointer");
    const u64 blocks = (count + BLOCK - 1) / BLOCK;
    hipLaunchKernelGGL(k_logits_keys, dim3((u32)(blocks < 65536 ? blocks : 65536)), dim3(BLOCK), 0, (hipStream_t)stream, ml2p,
                       (const i64 *)offsets, lengths, lengths ? length_bytes : 0u, (u64)count, (i64)stride, (u64)longest, out_keys);
    HIP_TRY(hipGetLastError());
    return MC_OK;
}
