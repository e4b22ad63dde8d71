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
__device__ __forceinline__ void store_vec(char *row, u32 v, u32 vocab, const float *g) {
    constexpr u32 N = VEC<DT>;
    if ((u64)v * N + N <= vocab) {
        raw4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (Elt<DT>::BYTES == 4) q[j] = __float_as_uint(g[j]);
            else q[j] = pack2<DT>(g[2 * j], g[2 * j + 1]);
        }
        *(raw4_at2 *)(row + (u64)v * 16) = q;
    } else {
#pragma unroll
        for (u32 j = 0; j < N; ++j) {
            if ((u64)v * N + j < vocab) {
                if constexpr (Elt<DT>::BYTES == 4) *(float *)(row + ((u64)v * N + j) * 4) = g[j];
                else *(unsigned short *)(row + ((u64)v * N + j) * 2) = (unsigned short)pack2<DT>(g[j], 0.f);
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
        store_vec<DT>(gp, v, a.vocab, g);
    }
}

// ---- draw ----------------------------------------------------------------------------------------------------------
struct DrawArgs {
    const double *uniforms;  // or null: Philox
    u64 seed, first_id;
    u32 draw;
    double t;
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

#define BY_TYPE(dtype, call)                            \
    switch (dtype) {                                    \
        case MC_LOGITS_F32: { constexpr int DT = MC_LOGITS_F32; call; break; }   \
        case MC_LOGITS_F16: { constexpr int DT = MC_LOGITS_F16; call; break; }   \
        default: { constexpr int DT = MC_LOGITS_BF16; call; break; }             \
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
    if (top) {
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
    BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_gradient<DT>), grid_of(a.rows), dim3(BLOCK), 0, (hipStream_t)stream, a, out));
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
    DrawArgs d{uniforms, seed, first_id, draw, temperature, live, out_token, out_ml2p};
    BY_TYPE(dtype, hipLaunchKernelGGL((k_logits_draw<DT>), grid_of(a.rows), dim3(BLOCK), 0, (hipStream_t)stream, a, d));
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
