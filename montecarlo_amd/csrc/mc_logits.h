// What the kernels on logits share (device code; mc_logits_score.hip says what they compute).
//
// With c = log2(e) / T a token's exponent is y = x c - M, where M is the largest logit's m c rounded up to a whole number:
// one multiply-add, one power and the sums an element, and sums under different M are brought together without a rounding.
// (m c itself may be off by a rounding; every use subtracts the same M, so that cancels.)  That holds while |M| <= 2^15.
// Parts of a row whose own maximum lies lower take -2^15 for it; a ROW whose M is beyond is summed again with
// y = (x - m) c (`exact`): a row of the type's lowest value, temperatures near 0.  m says the rest: it is -inf where nothing
// is left (s is 0 then), NaN where the row holds a NaN and +inf where it holds one (s is NaN then).
#pragma once
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>

#include "mc_internal.h"

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

constexpr int BLOCK = 256;
constexpr float LOWEST = -FLT_MAX;
constexpr double LOG2E = 1.4426950408889634074;
constexpr float FAR = 32768.f;

// A division by the same number for every row, as a multiplication: exact for row numbers below 2^31.
struct Div {
    u32 d, mul, shift;
};

// Something with a value (or a row of values) for every row, addressed by (row / inner, row % inner); strides in bytes.
struct View {
    const char *p;
    i64 os, is;
    u32 narrow;  // neither stride is negative or needs more than 32 bits
};

struct Rows {
    View logits, tokens;
    Div inner;
    u32 rows, vocab, nvec, full, token_bytes;  // nvec: vectors of 16 bytes a row; full: those that are whole
    float c;                                   // log2(e) / T
};

__device__ __forceinline__ const char *at(const View &v, const Div &inner, u32 row) {
    const u32 o = __umulhi(row << 1, inner.mul) >> inner.shift, i = row - o * inner.d;
    if (v.narrow) return v.p + ((u64)o * (u32)v.os + (u64)i * (u32)v.is);
    return v.p + (i64)o * v.os + (i64)i * v.is;
}

// A token id as the kernels use it: [0, V), MC_TOKEN_SKIP, or MC_TOKEN_OUTSIDE for everything else.
__device__ __forceinline__ int token_of(const Rows &a, u32 row) {
    const char *p = at(a.tokens, a.inner, row);
    const i64 t = a.token_bytes == 8 ? *(const i64 *)p : (i64) * (const int *)p;
    return t == MC_TOKEN_SKIP ? MC_TOKEN_SKIP : (t >= 0 && t < (i64)a.vocab) ? (int)t : MC_TOKEN_OUTSIDE;
}

// workgroups in a grid of two dimensions, since one holds at most 2^32 work items
constexpr u32 GRID_X = 1u << 20;
__device__ __forceinline__ u32 block_id() { return blockIdx.y * GRID_X + blockIdx.x; }
inline dim3 grid_of(u32 blocks) { return blocks <= GRID_X ? dim3(blocks) : dim3(GRID_X, (blocks + GRID_X - 1) / GRID_X); }

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

template <int DT>
__device__ __forceinline__ raw4 nothing() {
    return raw4{Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF, Elt<DT>::NEG_INF};
}

// A row as vectors: `nvec` of them from p on, the first `full` whole, `vocab` elements in all.  head: 1 where the row's
// first element stays before them, so that vectors of 2-byte elements begin at a multiple of 4 (rows of 50001 tokens, every
// other one odd: score 61 -> 51 us, gradient 125 -> 103 us for 2684 rows).
struct Span {
    const char *p;
    u32 head, vocab, nvec, full;
    float first;  // the head's logit, or -inf
};

// (`read`: false for a row that is skipped, of which nothing is loaded)
template <int DT>
__device__ __forceinline__ Span span_of(const Rows &a, const char *row, bool read) {
    if constexpr (Elt<DT>::BYTES == 2) {
        if ((uintptr_t)row & 2) {
            const u32 n = a.vocab - 1;
            return Span{row + 2, 1, n, (n + VEC<DT> - 1) / VEC<DT>, n / VEC<DT>, read ? element<DT>(row, 0) : -INFINITY};
        }
    }
    return Span{row, 0, a.vocab, a.nvec, a.full, -INFINITY};
}

// vector v of a row; what lies behind the row's end, or in vectors from `end` on, is -inf
template <int DT>
__device__ __forceinline__ raw4 load_vec(const Span &r, u32 v, u32 end) {
    constexpr u32 N = VEC<DT>;
    raw4 q = nothing<DT>();
    if (v < min(end, r.full)) {
        q = *(const raw4_at2 *)(r.p + (u64)v * 16);
    } else if (v < end) {
#pragma unroll
        for (u32 j = 0; j < N; ++j) {
            if (v * N + j < r.vocab) {
                if constexpr (Elt<DT>::BYTES == 4) {
                    q[j] = *(const u32 *)(r.p + ((u64)v * N + j) * 4);
                } else {
                    const u32 h = *(const unsigned short *)(r.p + ((u64)v * N + j) * 2);
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

// The elements from `from` on that the row has room for.  STREAM: past the caches (a row of many tokens fills whole lines by
// itself, and what the gradient does not displace there is read again from there: 200000 tokens 173 -> 137 us; rows of 97
// tokens leave parts of lines to each other and took twice as long that way).
template <int DT, bool STREAM, bool MAY_END = true>
__device__ __forceinline__ void store_at(char *row, u32 from, u32 vocab, const float *g) {
    constexpr u32 N = VEC<DT>;
    if (!MAY_END || (u64)from + N <= vocab) {
        raw4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (Elt<DT>::BYTES == 4) q[j] = __float_as_uint(g[j]);
            else q[j] = pack2<DT>(g[2 * j], g[2 * j + 1]);
        }
        raw4_at2 *p = (raw4_at2 *)(row + (u64)from * Elt<DT>::BYTES);
        if (STREAM) __builtin_nontemporal_store(q, p);
        else *p = q;
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

// the larger of two logits, NaN if one is (an instruction that takes three and, unlike fmaxf's, quiets nothing first)
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// of sums, which are 0, about 1 or more, or NaN: no scaling of the smallest numbers is needed
__device__ __forceinline__ float log2_(float s) { return __builtin_amdgcn_logf(s); }
// 1 / s for a sum other than 0, to about half a step: the instruction's value and one step of Newton's method
__device__ __forceinline__ float inverse(float s) {
    const float r = __builtin_amdgcn_rcpf(s);
    return __builtin_fmaf(__builtin_fmaf(-s, r, 1.f), r, r);
}

// A row's (or a part's) largest logit m, the sum s of 2^y and the sum e of 2^y y; `exact` says how y is meant.
struct Stat {
    float m, s, e;
    bool exact;
};

__device__ __forceinline__ float scaled(float m, float c) { return ceilf(fmaxf(m * c, -FAR)); }

// s 2^d for a whole number d (between -2^16 and 0 in rows whose sums stand; beside a NaN, a +inf or a maximum whose scaled value
// overflows it may be anything, which no conversion to a whole number is defined for: kept within 2^17, NaN included)
__device__ __forceinline__ float times2(float s, float d) { return __builtin_amdgcn_ldexpf(s, (int)__builtin_amdgcn_fmed3f(d, -131072.f, 131072.f)); }

// The exponent (x - m) c of a logit below the largest one, by halves: two logits of 32 bits may lie further apart than their type
// reaches, where the exponent does not (halves of such logits are exact; c is below 2^101).
__device__ __forceinline__ float below(float x, float m, float c) { return __builtin_fmaf(x, 0.5f, -0.5f * m) * (c + c); }

// the exponent of a logit under a row's statistics
struct Expo {
    float m, c, M;
    bool exact;
    __device__ __forceinline__ Expo(const Stat &st, float c_) : m(fmaxf(st.m, LOWEST)), c(c_), M(scaled(st.m, c_)), exact(st.exact) {}
    __device__ __forceinline__ float fast(float x) const { return __builtin_fmaf(x, c, -M); }
    __device__ __forceinline__ float operator()(float x) const { return exact ? below(x, m, c) : fast(x); }
};

// whether a row's fast sums do not stand
__device__ __forceinline__ bool doubtful(float m, float c) { return fabsf(m) < INFINITY && fabsf(m * c) > FAR; }

// A -log2 p or an entropy as it is put.  A token of probability 1 has log2 Z = y but for the roundings of a power and a logarithm,
// which may leave a few 2^-24 on either side of 0; keys are sorted by their bits, where a negative one would come last of all.
__device__ __forceinline__ float at_least_0(float v) { return maximum(v, 0.f); }

// what a row's statistics say about its token
__device__ __forceinline__ float ml2p_of(int tok, const Stat &st, float x, float c) {
    if (tok == MC_TOKEN_SKIP) return 0.f;
    if (!(st.s == st.s)) return st.s;
    return tok >= 0 && st.s > 0.f ? at_least_0(log2_(st.s) - Expo(st, c)(x)) : INFINITY;
}

__device__ __forceinline__ float entropy_of(int tok, const Stat &st) {
    return tok == MC_TOKEN_SKIP || st.s == 0.f ? 0.f : at_least_0(log2_(st.s) - st.e * inverse(st.s));
}

// ---- reductions over groups of lanes and over workgroups ---------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}

struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); }
};
struct Min {
    __device__ __forceinline__ float operator()(float a, float b) const { return __uint_as_float(min(__float_as_uint(a), __float_as_uint(b))); }  // (of words)
};
struct Add {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const {
        return a + b;
    }
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

template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const float lo = dpp<CTRL>(__int_as_float(__double2loint(x))), hi = dpp<CTRL>(__int_as_float(__double2hiint(x)));
    return __hiloint2double(__float_as_int(hi), __float_as_int(lo));
}

template <int G, typename Op>
__device__ __forceinline__ double group_all(double x, Op op) {
    if constexpr (G >= 2) x = op(x, dpp<0xB1>(x));
    if constexpr (G >= 4) x = op(x, dpp<0x4E>(x));
    if constexpr (G >= 8) x = op(x, dpp<0x141>(x));
    if constexpr (G >= 16) x = op(x, dpp<0x140>(x));
    if constexpr (G >= 32) x = op(x, __shfl_xor(x, 16));
    if constexpr (G >= 64) x = op(x, __shfl_xor(x, 32));
    return x;
}

struct AddWords {
    __device__ __forceinline__ float operator()(float a, float b) const { return __uint_as_float(__float_as_uint(a) + __float_as_uint(b)); }
};

template <int G>
__device__ __forceinline__ u32 group_sum(u32 x) {
    return __float_as_uint(group_all<G>(__uint_as_float(x), AddWords()));
}

template <int G>
__device__ __forceinline__ u32 group_min(u32 x) {
    return __float_as_uint(group_all<G>(__uint_as_float(x), Min()));
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

template <int G>
__device__ __forceinline__ float group_scan(float x) {
    const u32 lane = threadIdx.x & (G - 1);
    float o;
    if constexpr (G >= 2) o = dpp<0x111>(x), x += lane >= 1 ? o : 0.f;  // rows shifted by 1, 2, 4, 8
    if constexpr (G >= 4) o = dpp<0x112>(x), x += lane >= 2 ? o : 0.f;
    if constexpr (G >= 8) o = dpp<0x114>(x), x += lane >= 4 ? o : 0.f;
    if constexpr (G >= 16) o = dpp<0x118>(x), x += lane >= 8 ? o : 0.f;
    if constexpr (G >= 32) o = __shfl(x, 15, 32), x += (lane & 31) >= 16 ? o : 0.f;  // (rows do not see each other: the sum of
    if constexpr (G >= 64) o = __shfl(x, 31, 64), x += lane >= 32 ? o : 0.f;         // all before)
    return x;
}

// the lanes of a group joined: the common maximum, the sums scaled to it
template <int G, bool ENT>
__device__ __forceinline__ Stat group_stat(Stat st, float c) {
    const float mine = scaled(st.m, c);
    st.m = group_all<G>(st.m, Max());
    const float d = mine - scaled(st.m, c);
    if (ENT) st.e = group_all<G>(times2(__builtin_fmaf(d, st.s, st.e), d), Add());
    st.s = group_all<G>(times2(st.s, d), Add());
    return st;
}

// the whole workgroup's, in every thread
template <int T, bool ENT>
__device__ __forceinline__ Stat block_stat(Stat st, float c) {
    __shared__ float pm[T / 64], ps[T / 64], pe[T / 64];
    st = group_stat<64, ENT>(st, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        pm[threadIdx.x >> 6] = st.m;
        ps[threadIdx.x >> 6] = st.s;
        if (ENT) pe[threadIdx.x >> 6] = st.e;
    }
    __syncthreads();
    const u32 w = threadIdx.x & (T / 64 - 1);  // (every group of as many lanes as there are waves joins the waves once more)
    return group_stat<T / 64, ENT>(Stat{pm[w], ps[w], ENT ? pe[w] : 0.f, false}, c);
}

template <int T>
__device__ __forceinline__ u32 block_sum(u32 v) {
    __shared__ u32 part[T / 64];
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += part[w];
    return v;
}

// exclusive prefix sum over the workgroup and the total
template <int T, typename A>
__device__ __forceinline__ A block_scan(A v, A &total) {
    __shared__ A part[T / 64];
    const A inc = group_scan<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = inc;
    __syncthreads();
    A base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        if (w < (int)(threadIdx.x >> 6)) base += part[w];
        total += part[w];
    }
    return base + inc - v;
}

template <int N>
__device__ __forceinline__ float pairs(const float *w) {
    if constexpr (N == 1) return w[0];
    else return pairs<N / 2>(w) + pairs<N / 2>(w + N / 2);
}

// ---- rows of few tokens: a group of G lanes a row, several rows a wave, the row in registers ---------------------------------
constexpr u32 SUB_VECS = 64 * 8;  // vectors that 64 lanes hold at most: 4096 tokens of two bytes

// A row in the registers of G lanes, NV vectors each: vector i * G + lane; only a lane's last one may lie behind the row's
// end.  NV = 0: a row shorter than a vector, in one lane's only vector.
template <int DT, int NV>
struct SubRow {
    static constexpr int N = NV ? NV : 1;
    raw4 q[N];           // as loaded
    raw4 last;           // the lane's last vector with -inf in the places that are another vector's
    u32 from;            // its first element's number
};

// The row's last vector is loaded whole, 16 bytes that end where the row does: when the row is no multiple of a vector it
// reaches back into the one before it.
template <int DT, int G, int NV>
__device__ __forceinline__ void load_row(SubRow<DT, NV> &r, const char *p, const Rows &a, bool read) {
    constexpr u32 E = VEC<DT>;
    constexpr int N = SubRow<DT, NV>::N;
    const u32 lane = threadIdx.x & (G - 1), v = (N - 1) * G + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) r.q[i] = nothing<DT>();
    r.from = v * E;
    if (read) {
#pragma unroll
        for (int i = 0; i + 1 < N; ++i) r.q[i] = *(const raw4_at2 *)(p + (u64)(i * G + lane) * 16);
        if (NV == 0) {
            r.q[0] = load_vec<DT>(Span{p, 0, a.vocab, a.nvec, a.full, 0.f}, lane, a.nvec);
        } else if (v < a.nvec) {
            r.from = min(v * E, a.vocab - E);
            r.q[N - 1] = *(const raw4_at2 *)(p + (u64)r.from * Elt<DT>::BYTES);
        }
    }
    r.last = r.q[N - 1];
    const u32 n = v * E - r.from;  // places of the vector before it
    if (n) {
#pragma unroll
        for (u32 w = 0; w < 4; ++w) {
            u32 m;
            if constexpr (Elt<DT>::BYTES == 4) m = w < n ? 0xFFFFFFFFu : 0u;
            else m = (2 * w < n ? 0xFFFFu : 0u) | (2 * w + 1 < n ? 0xFFFF0000u : 0u);
            r.last[w] = (r.last[w] & ~m) | (Elt<DT>::NEG_INF & m);
        }
    }
}

template <int DT, int NV>
__device__ __forceinline__ raw4 vec_of(const SubRow<DT, NV> &r, int i) {
    return i + 1 == SubRow<DT, NV>::N ? r.last : r.q[i];
}

// `a` takes the value of b where `yes` (by words: a choice between vectors becomes one between their addresses, and the row
// goes to memory for it)
__device__ __forceinline__ void choose(raw4 &a, const raw4 &b, bool yes) {
    const u32 m = yes ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int w = 0; w < 4; ++w) a[w] = (a[w] & ~m) | (b[w] & m);
}

// the number of vector i's first element
template <int DT, int G, int NV>
__device__ __forceinline__ u32 from_of(const SubRow<DT, NV> &r, int i) {
    return i + 1 == SubRow<DT, NV>::N ? r.from : (i * G + (threadIdx.x & (G - 1))) * VEC<DT>;
}

// The words of a row as if just loaded: what comes next unpacks them again, where the compiler would keep the numbers of
// all vectors in registers.  For code that seldom runs, and for rows of more than four vectors a lane.
template <int DT, int NV>
__device__ __forceinline__ void forget(SubRow<DT, NV> &r) {
#pragma unroll
    for (int i = 0; i + 1 < SubRow<DT, NV>::N; ++i) asm("" : "+v"(r.q[i]));
    asm("" : "+v"(r.last));
}

template <int DT, int G, bool ENT, bool EXACT, int NV>
__device__ __forceinline__ Stat sub_sums(const SubRow<DT, NV> &r, float m, float c) {
    Stat st{m, 0.f, 0.f, EXACT};
    const Expo y_of(st, c);
#pragma unroll
    for (int i = 0; i < SubRow<DT, NV>::N; ++i) {
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) {
            const float x = unpack<DT>(vec_of(r, i), j), y = EXACT ? below(x, y_of.m, c) : y_of.fast(x), w = exp2_(y);
            st.s += w;
            if (ENT) st.e = __builtin_fmaf(w, fmaxf(y, -FAR), st.e);
        }
    }
    st.s = group_all<G>(st.s, Add());
    if (ENT) st.e = group_all<G>(st.e, Add());
    return st;
}

template <int DT, int G, int NV>
__device__ __forceinline__ float sub_max(const SubRow<DT, NV> &r) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < SubRow<DT, NV>::N; ++i)
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) m = maximum(m, unpack<DT>(vec_of(r, i), j));
    return group_all<G>(m, Max());
}

template <int DT, int G, bool ENT, int NV>
__device__ __forceinline__ Stat sub_stat(SubRow<DT, NV> &r, float c) {
    const float m = sub_max<DT, G>(r);
    if (NV > 4) forget(r);
    Stat st = sub_sums<DT, G, ENT, false>(r, m, c);
    const bool again = doubtful(m, c);
    if (__ballot(again)) {
        forget(r);
        const Stat ex = sub_sums<DT, G, ENT, true>(r, m, c);
        if (again) st = ex;
    }
    return st;
}

// ---- rows of many tokens: workgroups that stream a row or a part of it ---------------------------------------------------
constexpr int UNROLL = 4;  // vectors of a thread in flight

// a chunk joins a thread's running statistics; returns the chunk's largest logit
template <int DT, bool ENT>
__device__ __forceinline__ float take(Stat &st, const raw4 (&q)[UNROLL], float c) {
    constexpr int N = VEC<DT>;
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int j = 0; j < N; ++j) m = maximum(m, unpack<DT>(q[u], j));
    const float old = scaled(st.m, c);
    st.m = maximum(st.m, m);
    const float M = scaled(st.m, c), d = old - M;
    if (ENT) st.e = times2(__builtin_fmaf(d, st.s, st.e), d);
    float s[UNROLL];  // (in pairs, so that few additions follow each other)
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        float w[N], e = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float y = __builtin_fmaf(unpack<DT>(q[u], j), c, -M);
            w[j] = exp2_(y);
            if (ENT) e = __builtin_fmaf(w[j], fmaxf(y, -FAR), e);
        }
        s[u] = pairs<N>(w);
        if (ENT) st.e += e;
    }
    st.s = times2(st.s, d) + pairs<UNROLL>(s);
    return m;
}

// the vectors base + u * STRIDE + lane of a row, as far as they are below `end`
template <int DT, int STRIDE, int U>
__device__ __forceinline__ void load_chunk(raw4 (&q)[U], const Span &r, u32 base, u32 lane, u32 end) {
    if (base + U * STRIDE <= min(end, r.full)) {
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = *(const raw4_at2 *)(r.p + (u64)(base + u * STRIDE + lane) * 16);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = load_vec<DT>(r, base + u * STRIDE + lane, end);
    }
}

// one logit joins a thread's running statistics (-inf changes nothing)
template <bool ENT>
__device__ __forceinline__ void take_one(Stat &st, float x, float c) {
    const float old = scaled(st.m, c);
    st.m = maximum(st.m, x);
    const float M = scaled(st.m, c), d = old - M, y = __builtin_fmaf(x, c, -M), w = exp2_(y);
    if (ENT) st.e = times2(__builtin_fmaf(d, st.s, st.e), d) + w * fmaxf(y, -FAR);
    st.s = times2(st.s, d) + w;
}

// A doubtful row's statistics (every thread of the workgroup calls): m is its largest logit.
template <int DT, int T, bool ENT>
__device__ __forceinline__ Stat exact_stat(const Span &r, float c, float m) {
    Stat st{m, 0.f, 0.f, true};
    const auto add = [&](float x) {
        const float y = below(x, m, c), w = exp2_(y);
        st.s += w;
        st.e += w * fmaxf(y, -FAR);
    };
    if (threadIdx.x == 0) add(r.first);
    for (u32 v = threadIdx.x; v < r.nvec; v += T) {
        const raw4 q = load_vec<DT>(r, v, r.nvec);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) add(unpack<DT>(q, j));
    }
    __shared__ float ps[T / 64], pe[T / 64];
    st.s = group_all<64>(st.s, Add());
    st.e = group_all<64>(st.e, Add());
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        ps[threadIdx.x >> 6] = st.s;
        pe[threadIdx.x >> 6] = st.e;
    }
    __syncthreads();
    const u32 w = threadIdx.x & (T / 64 - 1);
    st.s = group_all<T / 64>(ps[w], Add());
    st.e = group_all<T / 64>(pe[w], Add());
    return st;
}

// ---- host ------------------------------------------------------------------------------------------------------------------
inline int bad(const char *who, const char *why) {
    mc_set_error("%s: %s", who, why);
    return MC_ERR_ARG;
}

inline bool aligned(const void *p, size_t bytes) { return (uintptr_t)p % bytes == 0; }  // (null is)

inline Div make_div(u64 d) {
    Div r{(u32)d, 0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.mul = (u32)((((u64)1 << (31 + r.shift)) + d - 1) / d);
    return r;
}

inline View view_of(const void *p, int64_t outer_stride, int64_t inner_stride, int64_t bytes) {
    const i64 os = outer_stride * bytes, is = inner_stride * bytes;
    return View{(const char *)p, os, is, os >= 0 && is >= 0 && os < (1ll << 32) && is < (1ll << 32)};
}

inline bool one_run(uint64_t inner, int64_t outer_stride, int64_t inner_stride) { return (u64)outer_stride == inner * (u64)inner_stride; }

// the arguments that every entry point on logits shares (`flat`: everything else that a row has lies as one run too)
inline int rows_of(const char *who, Rows &a, const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
                   int64_t outer_stride, int64_t inner_stride, double temperature, bool flat) {
    if (dtype > MC_LOGITS_BF16) return bad(who, "unknown element type");
    if (vocab == 0 || vocab >= (1ull << 31) - 64) return bad(who, "the vocabulary holds 1 .. 2^31 - 65 tokens");
    if (outer >= (1ull << 31) || inner >= (1ull << 31) || outer * inner >= (1ull << 31)) return bad(who, "at most 2^31 - 1 rows");
    if (!(temperature >= 1e-30 && temperature <= 1e30)) return bad(who, "the temperature is a positive number (1e-30 .. 1e30)");
    if (outer * inner && !logits) return bad(who, "no logits");
    const int bytes = dtype == MC_LOGITS_F32 ? 4 : 2;
    if (!aligned(logits, bytes)) return bad(who, "logits that are not aligned to their type");
    a.rows = (u32)(outer * inner);
    if (outer > 1 && flat && one_run(inner, outer_stride, inner_stride)) {
        inner *= outer;
        outer = 1;
    }
    a.logits = view_of(logits, outer_stride, inner_stride, bytes);
    a.inner = make_div(inner ? inner : 1);
    a.vocab = (u32)vocab;
    a.full = (u32)(vocab / (16 / bytes));
    a.nvec = (u32)((vocab + 16 / bytes - 1) / (16 / bytes));
    a.c = (float)(LOG2E / temperature);
    return MC_OK;
}

inline int tokens_of(const char *who, Rows &a, const void *tokens, uint32_t token_bytes, int64_t outer_stride, int64_t inner_stride,
                     uint64_t rows) {
    if (token_bytes != 4 && token_bytes != 8) return bad(who, "token ids of 4 or 8 bytes");
    if (rows && !tokens) return bad(who, "no tokens");
    if (!aligned(tokens, token_bytes)) return bad(who, "tokens that are not aligned to their type");
    a.token_bytes = token_bytes;
    a.tokens = view_of(tokens, outer_stride, inner_stride, token_bytes);
    return MC_OK;
}

inline u32 rows_to_blocks(u32 rows, u32 group) { return (u32)(((u64)rows * group + BLOCK - 1) / BLOCK); }

}  // namespace

#define BY_TYPE(dtype, ...)                                                            \
    switch (dtype) {                                                                   \
        case MC_LOGITS_F32: { constexpr int DT = MC_LOGITS_F32; __VA_ARGS__; break; }  \
        case MC_LOGITS_F16: { constexpr int DT = MC_LOGITS_F16; __VA_ARGS__; break; }  \
        default: { constexpr int DT = MC_LOGITS_BF16; __VA_ARGS__; break; }            \
    }

// How many lanes share a row (G) and how many vectors each of them holds (NV, at most 8).  Many rows: the fewest lanes, since
// what is done once a row and lane costs as much as eight elements; but four at least, since two lanes ask for 32 bytes of a
// row at a time and the loads then take as long as the arithmetic saved (1e6 rows of 97 tokens: 46 us with 4 lanes of 4
// vectors, 48 with 2 of 7).  Few rows (less than a wave for each of the 1024 SIMDs): a lane for each vector, since such a
// launch waits for its loads and its instructions (12 rows of 97 tokens took 15.7 us with 4 lanes, 4.4 with 32).
inline void group_of(u32 rows, u32 vocab, u32 nvec, u32 vec, int &g, int &nv) {
    g = 4, nv = 0;
    if (vocab < vec) return;
    while (nvec > 8u * g) g *= 2;
    if ((u64)rows * g <= 32768) {
        while (g < 64 && nvec > (u32)g) g *= 2;
    }
    nv = (int)((nvec + g - 1) / g);
}

#define BY_LANES(...)                                              \
    switch (g_) {                                                  \
        case 4: { constexpr int G = 4; __VA_ARGS__; break; }       \
        case 8: { constexpr int G = 8; __VA_ARGS__; break; }       \
        case 16: { constexpr int G = 16; __VA_ARGS__; break; }     \
        case 32: { constexpr int G = 32; __VA_ARGS__; break; }     \
        default: { constexpr int G = 64; __VA_ARGS__; break; }     \
    }
// (2 to 4 vectors a lane: the shortest rows and, of few rows, the longest)
#define BY_ENDS(...)                                               \
    if (g_ == 4) { constexpr int G = 4; __VA_ARGS__; }             \
    else { constexpr int G = 64; __VA_ARGS__; }

#define BY_GROUP(a, ...)                                                            \
    {                                                                               \
        int g_, nv_;                                                                \
        group_of((a).rows, (a).vocab, (a).nvec, VEC<DT>, g_, nv_);                  \
        switch (nv_) {                                                              \
            case 0: { constexpr int NV = 0, G = 4; __VA_ARGS__; break; }            \
            case 1: { constexpr int NV = 1; BY_LANES(__VA_ARGS__) break; }          \
            case 2: { constexpr int NV = 2; BY_ENDS(__VA_ARGS__) break; }           \
            case 3: { constexpr int NV = 3; BY_ENDS(__VA_ARGS__) break; }           \
            case 4: { constexpr int NV = 4; BY_ENDS(__VA_ARGS__) break; }           \
            case 5: { constexpr int NV = 5; BY_LANES(__VA_ARGS__) break; }          \
            case 6: { constexpr int NV = 6; BY_LANES(__VA_ARGS__) break; }          \
            case 7: { constexpr int NV = 7; BY_LANES(__VA_ARGS__) break; }          \
            default: { constexpr int NV = 8; BY_LANES(__VA_ARGS__) break; }         \
        }                                                                           \
    }
