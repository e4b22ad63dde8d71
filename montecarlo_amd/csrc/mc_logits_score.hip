// A language model's answer -- a row of logits x over V tokens for every place -- turned into what the Monte Carlo
// path works on (gfx950): the score of given tokens (calc_ml2p), with entropy and the most probable alternatives; the
// gradient of that score (mc_logits_gradient.hip); draws with their probability (pick_expand, lib4mc/ProbLib.py:31-43) and
// the float64 keys of whole passwords (mc_logits_draw.hip).  With c = log2(e) / T, m the row's largest logit,
// y = (x - m) c <= 0, w = 2^y and Z the sum of w:
//
//   score      -log2 p_t = log2 Z - y_t,   H = log2 Z - (sum of w y) / Z          (bits)
//   gradient   d/dx_i of a * (-log2 p_t) + b * H = (a (p_i - [i = t]) / ln 2 - b p_i (log2 p_i + H)) / T
//   draw       the first token whose running sum of weights exceeds u Z
//   keys       the sum of a password's -log2 p in 64 bits
//
// A row holds 10^2 .. 10^5 numbers that are read once: every kernel here is bound by HBM, then by the eight to ten
// operations an element takes.  One pass keeps the running maximum, the sum scaled to it and the sum of w y in 32 bits
// (all terms are positive or all negative: no cancellation); a change of the maximum scales both.
#include "mc_logits.h"

namespace {

struct ScoreOut {
    float *ml2p, *entropy, *top_ml2p;
    int *top;
    u32 k;
};

// The order of alternatives is that of the logits themselves (equal logits: the lower index), so it never depends on a
// rounding.  A logit as a word whose unsigned order is the numbers' (both zeros alike):
__device__ __forceinline__ u32 order_of(float x) {
    const u32 b = __float_as_uint(x + 0.0f);
    return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(u32 o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr u32 ORDER_NEG_INF = 0x007FFFFFu;

// a candidate: larger for a larger logit and, among equals, for a lower index; 0: none
__device__ __forceinline__ u64 key_of(u32 order, u32 index) { return (u64)order << 32 | (0xFFFFFFFFu - index); }
__device__ __forceinline__ u32 index_of(u64 key) { return 0xFFFFFFFFu - (u32)key; }

// one alternative's outputs
__device__ __forceinline__ void put_top(const ScoreOut &out, u32 row, u32 rank, u64 key, const Stat &st, float lz, float c) {
    const float v = at_least_0(lz - Expo(st, c)(value_of((u32)(key >> 32))));
    out.top[(u64)row * out.k + rank] = v < INFINITY ? (int)index_of(key) : MC_TOKEN_OUTSIDE;
    out.top_ml2p[(u64)row * out.k + rank] = v < INFINITY ? v : INFINITY;
}

// ---- rows of few tokens --------------------------------------------------------------------------------------------------
// The k largest of a row in registers, one after the other: the largest that comes behind the last one in the order.
template <int DT, int G, int NV>
__device__ __forceinline__ void top_by_turns(SubRow<DT, NV> &r, const Stat &st, const ScoreOut &out, u32 row, bool writes, float c) {
    const u32 lane = threadIdx.x & (G - 1);
    const float lz = log2_(st.s);
    float last = INFINITY;
    u32 last_i = 0xFFFFFFFFu;
    for (u32 k = 0; k < out.k; ++k) {
        if (NV > 1) forget(r);
        float best = -INFINITY;
        u32 best_i = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < SubRow<DT, NV>::N; ++i) {
            const u32 from = from_of<DT, G>(r, i);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float x = unpack<DT>(vec_of(r, i), j);
                const bool open = x < last || (x == last && from + j > last_i);
                if (open && x > best) best = x, best_i = from + j;
            }
        }
        const float top = group_all<G>(best, Max());
        const u32 at = group_min<G>(best == top ? best_i : 0xFFFFFFFFu);
        if (writes && lane == 0) {
            if (top > -INFINITY) {
                put_top(out, row, k, key_of(order_of(top), at), st, lz, c);
            } else {
                out.top[(u64)row * out.k + k] = MC_TOKEN_OUTSIDE;
                out.top_ml2p[(u64)row * out.k + k] = INFINITY;
            }
        }
        last = top;
        last_i = at;
    }
}

// The k largest of a row in registers at once.  The first 16 bits of the order word that k of the row's vectors' largest (or,
// where these are fewer than 2 k, of its elements) reach, bit by bit; the few elements that reach them go to LDS, and
// each finds its place by counting the larger ones.  (One after the other, 10 of 1000 took 271 us for 67108 rows, 32 took 938.)
// `room`: candidates a row has room for; rows with more (many equal ones) take turns.  The sixteen counts are what bounds it: 2^20
// rows of 97 two-byte tokens take 52 us without alternatives, 155 with 5 and 282 with 10, which count elements (2 k > G N).
template <int DT, int G, int NV>
__device__ __forceinline__ void sub_top(SubRow<DT, NV> &r, const Rows &a, const Stat &st, const ScoreOut &out, u32 row, bool writes, int tok, u64 *room_of_all,
                                        u32 room) {
    constexpr int N = SubRow<DT, NV>::N;
    const u32 lane = threadIdx.x & (G - 1);
    u64 *cand = room_of_all + threadIdx.x / G * room;
    const bool blank = tok == MC_TOKEN_SKIP || !(st.s > 0.f);
    writes = writes && !blank;
    if (blank && row < a.rows) {
        for (u32 i = lane; i < out.k; i += G) {
            out.top[(u64)row * out.k + i] = tok == MC_TOKEN_SKIP ? MC_TOKEN_SKIP : MC_TOKEN_OUTSIDE;
            out.top_ml2p[(u64)row * out.k + i] = tok == MC_TOKEN_SKIP ? 0.f : st.s == st.s ? INFINITY : st.s;
        }
    }
    const bool by_vectors = 2 * out.k <= (u32)(G * N);
    float largest[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        largest[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) largest[i] = maximum(largest[i], unpack<DT>(vec_of(r, i), j));
    }
    u32 bound = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; --bit) {
        const u32 t = bound | (1u << bit);
        const float x = value_of(t);  // (a NaN where no number has these bits: nothing reaches it)
        u32 n = 0;
        if (by_vectors) {
#pragma unroll
            for (int i = 0; i < N; ++i) n += largest[i] >= x;
        } else {
            forget(r);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < VEC<DT>; ++j) n += unpack<DT>(vec_of(r, i), j) >= x;
        }
        if (group_sum<G>(n) >= out.k) bound = t;
    }
    forget(r);
    const float least = bound > ORDER_NEG_INF ? value_of(bound) : LOWEST;
    u32 mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) mine += unpack<DT>(vec_of(r, i), j) >= least;
    const u32 upto = group_scan<G>(mine), n = group_sum<G>(mine);
    const bool fits = n <= room;
    forget(r);
    if (fits && writes) {
        u64 *put = cand + (upto - mine);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const u32 from = from_of<DT, G>(r, i);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float x = unpack<DT>(vec_of(r, i), j);
                if (x >= least) *put++ = key_of(order_of(x), from + j);
            }
        }
    }
    __syncthreads();
    if (fits && writes) {
        const float lz = log2_(st.s);
        for (u32 i = lane; i < n; i += G) {
            const u64 key = cand[i];
            u32 rank = 0;
            for (u32 j = 0; j < n; ++j) rank += cand[j] > key;
            if (rank < out.k) put_top(out, row, rank, key, st, lz, a.c);
        }
        for (u32 i = n + lane; i < out.k; i += G) {
            out.top[(u64)row * out.k + i] = MC_TOKEN_OUTSIDE;
            out.top_ml2p[(u64)row * out.k + i] = INFINITY;
        }
    }
    if (__ballot(writes && !fits)) top_by_turns<DT, G>(r, st, out, row, writes && !fits, a.c);
}

// (Waves a SIMD with alternatives: six while the row's vectors leave the registers for it, else four.  Of five vectors of four-byte
// logits six spill 27 registers inside the loops: 60000 rows of 1200 tokens 484 us.)
template <int DT, int G, int NV, bool ENT, bool TOP>
__global__ __launch_bounds__(BLOCK, !TOP ? 8 : NV > (DT == MC_LOGITS_F32 ? 4 : 5) ? 4 : 6) void k_logits_score_sub(Rows a, ScoreOut out, u32 room) {
    extern __shared__ u64 candidates[];
    const u32 row = block_id() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows;
    const int tok = there ? token_of(a, row) : MC_TOKEN_SKIP;
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT, NV> r;
    load_row<DT, G>(r, p, a, tok != MC_TOKEN_SKIP);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const Stat st = sub_stat<DT, G, ENT>(r, a.c);
    if (there && lane == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (ENT && out.entropy) out.entropy[row] = entropy_of(tok, st);
    }
    if constexpr (TOP) sub_top<DT, G>(r, a, st, out, row, there, tok, candidates, room);
}

// ---- rows of many tokens ---------------------------------------------------------------------------------------------------
constexpr int CELL_ROWS = 16;  // cells of a thread
constexpr u32 LIST_CAP = 256, CAND_CAP = 512;

// A pass over the row keeps, beside its sums, the largest logit of every cell (one thread's vectors of `per_cell` chunks) and of
// every thread.  The k-th largest of n groups of threads is a lower bound of the k-th largest of all (about n ln(n / (n - k))
// logits of a random row reach it): only the cells that do are looked at again.
template <int T>
struct TopShared {
    u32 most[T];             // order words of the threads' largest
    u64 cand[CAND_CAP + 1];  // (and the row's first element)
    u32 list[LIST_CAP];
    u32 n_list, n_cand;
};

// An order word among the wave's N * 64 that at least k of them reach: the least that reaches the k-th's first 16 bits.
template <int N>
__device__ __forceinline__ u32 bound_of(const u32 (&o)[N], u32 k) {
    u32 b = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const u32 t = b | (1u << bit);
        u32 n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += (u32)__popcll(__ballot(o[i] >= t));
        if (n >= k) b = t;
    }
    u32 least = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < N; ++i) least = min(least, o[i] >= b ? o[i] : 0xFFFFFFFFu);
    return group_min<64>(least);
}

// The same for the workgroup's T words in `words`: of 64 (the largest of those 64 apart) while k is small, else of 256.
template <int T>
__device__ __forceinline__ u32 bound_among(const u32 *words, u32 k) {
    u32 o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < T / 64; ++w) o[w % 4] = max(o[w % 4], words[w * 64 + (threadIdx.x & 63)]);
    if (k > 16) return bound_of<4>(o, k);
    const u32 one[1] = {max(max(o[0], o[1]), max(o[2], o[3]))};
    return bound_of<1>(one, k);
}

template <int DT, int T>
__device__ __forceinline__ u32 count_from(const Span &row, u32 v0, u32 v1, u32 order) {
    u32 n = 0;
    for (u32 v = v0 + threadIdx.x; v < v1; v += T) {
        const raw4 q = load_vec<DT>(row, v, v1);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) n += order_of(unpack<DT>(q, j)) >= order;
    }
    return block_sum<T>(n);
}

// The k largest when the candidates do not fit (rows of equal logits, orders made to defeat the cells): the k-th largest
// value by bits, unless `bound` is it already; then one pass in order of the index.
template <int DT, int T>
__device__ __forceinline__ u32 select_by_bits(TopShared<T> &sh, const Span &row, u32 v0, u32 v1, u32 k, u32 bound) {
    u32 kth = bound, above;
    if (bound <= ORDER_NEG_INF) {  // fewer than k lanes hold anything: there may be fewer than k candidates
        k = min(k, count_from<DT, T>(row, v0, v1, ORDER_NEG_INF + 1));
        if (k == 0) return 0;
        above = 0xFFFFFFFFu;
    } else {
        above = count_from<DT, T>(row, v0, v1, bound + 1);
    }
    if (above >= k) {
        kth = 0;
        for (int b = 31; b >= 0; --b) {
            const u32 t = kth | (1u << b);
            if (count_from<DT, T>(row, v0, v1, t) >= k) kth = t;
        }
        above = count_from<DT, T>(row, v0, v1, kth + 1);
    }
    const u32 equal = k - above;
    __syncthreads();
    if (threadIdx.x == 0) sh.n_cand = equal;  // (those above come behind the equal ones, in any order)
    __syncthreads();
    u32 found = 0, base = v0;
    for (; base < v1 && found < equal; base += T) {
        const u32 v = base + threadIdx.x;
        const raw4 q = load_vec<DT>(row, v, v1);
        u32 n = 0;
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) n += order_of(unpack<DT>(q, j)) == kth;
        u32 total, place = found + block_scan<T>(n, total);
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) {
            const u32 o = order_of(unpack<DT>(q, j)), i = row.head + v * VEC<DT> + j;
            if (o == kth && place < equal) sh.cand[place] = key_of(o, i);
            place += o == kth;
            if (o > kth) sh.cand[atomicAdd(&sh.n_cand, 1u)] = key_of(o, i);
        }
        found += total;
    }
    if (above) {
        for (u32 v = base + threadIdx.x; v < v1; v += T) {
            const raw4 q = load_vec<DT>(row, v, v1);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const u32 o = order_of(unpack<DT>(q, j));
                if (o > kth) sh.cand[atomicAdd(&sh.n_cand, 1u)] = key_of(o, row.head + v * VEC<DT> + j);
            }
        }
    }
    __syncthreads();
    return k;
}

// the row's first element is a candidate of its first part
template <int T>
__device__ __forceinline__ u32 add_head(TopShared<T> &sh, const Span &row, u32 v0, u32 n) {
    if (v0 == 0 && row.first > -INFINITY) {
        if (threadIdx.x == 0) sh.cand[n] = key_of(order_of(row.first), 0);
        ++n;
        __syncthreads();
    }
    return n;
}

// candidates for the k largest of vectors v0 .. v1 into sh.cand: their number (sh.most holds the threads' largest)
template <int DT, int T>
__device__ __forceinline__ u32 select(TopShared<T> &sh, const float *cells, const Span &row, u32 v0, u32 v1, u32 k, u32 per_cell) {
    if (threadIdx.x == 0) sh.n_list = sh.n_cand = 0;
    __syncthreads();
    const u32 bound = bound_among<T>(sh.most, k);
    const u32 cell_vecs = per_cell * UNROLL;
    for (u32 r = 0; v0 + r * cell_vecs * T < v1; ++r) {
        const float m = cells[r * T + threadIdx.x];
        if (m > -INFINITY && order_of(m) >= bound) {
            const u32 n = atomicAdd(&sh.n_list, 1u);
            if (n < LIST_CAP) sh.list[n] = r * T + threadIdx.x;
        }
    }
    __syncthreads();
    const u32 n_list = sh.n_list;
    if (n_list <= LIST_CAP) {
        for (u32 i = threadIdx.x; i < n_list * cell_vecs; i += T) {
            const u32 cell = sh.list[i / cell_vecs], u = i % cell_vecs;
            const u32 v = v0 + ((cell / T) * cell_vecs + u) * T + cell % T;
            const raw4 q = load_vec<DT>(row, v, v1);
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float x = unpack<DT>(q, j);
                if (x > -INFINITY && order_of(x) >= bound) {
                    const u32 n = atomicAdd(&sh.n_cand, 1u);
                    if (n < CAND_CAP) sh.cand[n] = key_of(order_of(x), row.head + v * VEC<DT> + j);
                }
            }
        }
    }
    __syncthreads();
    u32 n = sh.n_cand;
    if (n_list > LIST_CAP || n > CAND_CAP) n = select_by_bits<DT, T>(sh, row, v0, v1, k, bound);
    return add_head<T>(sh, row, v0, n);
}

// How the work on a row is cut: 2^shift workgroups of `vecs` vectors, whose statistics (and candidates, by place and part)
// another launch joins.
struct Split {
    u32 shift, vecs;
    float4 *stats;  // [row][part]: m, s, e
    u64 *keys;      // [row][place][part]
    u32 per_cell;   // chunks a cell
};

__device__ __forceinline__ void put_skipped(const ScoreOut &out, u32 row) {
    if (threadIdx.x == 0) {
        out.ml2p[row] = 0.f;
        if (out.entropy) out.entropy[row] = 0.f;
    }
    if (threadIdx.x < out.k) {
        out.top[(u64)row * out.k + threadIdx.x] = MC_TOKEN_SKIP;
        out.top_ml2p[(u64)row * out.k + threadIdx.x] = 0.f;
    }
}

// a row's statistics are known (to all threads): its outputs, with n candidates for the alternatives
template <int T>
__device__ __forceinline__ void put_row(const ScoreOut &out, u32 row, int tok, float x, const Stat &st, float c, const u64 *cand, u32 n) {
    if (threadIdx.x == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, c);
        if (out.entropy) out.entropy[row] = entropy_of(tok, st);
    }
    if (!out.k) return;
    if (!(st.s > 0.f)) n = 0;
    const float lz = log2_(st.s);
    for (u32 i = threadIdx.x; i < n; i += T) {
        const u64 key = cand[i];
        u32 rank = 0;
        for (u32 j = 0; j < n; ++j) rank += cand[j] > key;
        if (rank < out.k) put_top(out, row, rank, key, st, lz, c);
    }
    for (u32 i = n + threadIdx.x; i < out.k; i += T) {
        out.top[(u64)row * out.k + i] = MC_TOKEN_OUTSIDE;
        out.top_ml2p[(u64)row * out.k + i] = st.s == st.s ? INFINITY : st.s;
    }
}

template <int DT, int T, bool ENT, bool TOP, bool PART>
__global__ __launch_bounds__(T, 8) void k_logits_score(Rows a, ScoreOut out, Split sp) {
    __shared__ typename std::conditional<TOP, TopShared<T>, int>::type sh;
    extern __shared__ float cells[];
    const u32 id = block_id(), row = PART ? id >> sp.shift : id, part = PART ? id & ((1u << sp.shift) - 1) : 0;
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    if (tok == MC_TOKEN_SKIP) {
        if (!PART) put_skipped(out, row);
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, true);
    const float x = !PART && tok >= 0 ? element<DT>(p, tok) : 0.f;
    const u32 v0 = PART ? min(part * sp.vecs, r.nvec) : 0, v1 = PART ? min(r.nvec, v0 + sp.vecs) : r.nvec;
    // (cells of as many chunks as the launch's LDS was counted with: a shorter last part, or a row without its first element, may
    // have fewer chunks, and fewer chunks spread anew may need more rows of cells: 17 make 9, 16 make 16)
    const u32 chunks = (v1 - v0 + T * UNROLL - 1) / (T * UNROLL), per_cell = sp.per_cell;
    Stat st{-INFINITY, 0.f, 0.f, false};
    float cell = -INFINITY;
    for (u32 ch = 0, in = 0, cr = 0; ch < chunks; ++ch) {
        raw4 q[UNROLL];
        load_chunk<DT, T>(q, r, v0 + ch * T * UNROLL, threadIdx.x, v1);
        const float m = take<DT, ENT>(st, q, a.c);
        if constexpr (TOP) {
            cell = maximum(cell, m);
            if (++in == per_cell || ch + 1 == chunks) {
                cells[cr++ * T + threadIdx.x] = cell;
                cell = -INFINITY;
                in = 0;
            }
        }
    }
    if constexpr (TOP) sh.most[threadIdx.x] = order_of(st.m);
    if (threadIdx.x == 0 && v0 == 0) take_one<ENT>(st, r.first, a.c);
    st = block_stat<T, ENT>(st, a.c);
    if constexpr (PART) {
        if (threadIdx.x == 0) sp.stats[id] = make_float4(st.m, st.s, st.e, 0.f);
        if constexpr (TOP) {
            // (a part with a NaN or +inf needs none, and NaNs have no place in the order that the selection counts by)
            const u32 n = fabsf(st.m) < INFINITY ? select<DT, T>(sh, cells, r, v0, v1, out.k, per_cell) : 0u;
            u64 *keys = sp.keys + ((u64)row * out.k << sp.shift) + part;
            for (u32 i = threadIdx.x; i < n; i += T) {
                const u64 key = sh.cand[i];
                u32 rank = 0;
                for (u32 j = 0; j < n; ++j) rank += sh.cand[j] > key;
                if (rank < out.k) keys[rank << sp.shift] = key;
            }
            for (u32 i = n + threadIdx.x; i < out.k; i += T) keys[i << sp.shift] = 0;
        }
    } else {
        if (doubtful(st.m, a.c)) st = exact_stat<DT, T, ENT>(r, a.c, st.m);
        u32 n = 0;
        const u64 *cand = nullptr;
        if constexpr (TOP) {
            if (st.s > 0.f) n = select<DT, T>(sh, cells, r, v0, v1, out.k, per_cell);
            cand = sh.cand;
        }
        put_row<T>(out, row, tok, x, st, a.c, cand, n);
    }
}

// the parts of a row joined
template <int DT, bool ENT, bool TOP>
__global__ __launch_bounds__(BLOCK) void k_logits_score_join(Rows a, ScoreOut out, Split sp) {
    constexpr int T = BLOCK;
    __shared__ typename std::conditional<TOP, TopShared<T>, int>::type sh;
    const u32 row = block_id();
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    if (tok == MC_TOKEN_SKIP) {
        put_skipped(out, row);
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, true);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const u32 parts = 1u << sp.shift, lane = threadIdx.x & 63;
    Stat st{-INFINITY, 0.f, 0.f, false};
    if (lane < parts) {
        const float4 f = sp.stats[((u64)row << sp.shift) + lane];
        st = Stat{f.x, f.y, f.z, false};
    }
    st = group_stat<64, ENT>(st, a.c);
    if (doubtful(st.m, a.c)) st = exact_stat<DT, T, ENT>(r, a.c, st.m);
    u32 n = 0;
    const u64 *cand = nullptr;
    if constexpr (TOP) {
        cand = sh.cand;
        if (st.s > 0.f) {
            const u32 total = out.k << sp.shift;
            const u64 *keys = sp.keys + (u64)row * total;
            u32 lm = 0;
            for (u32 i = threadIdx.x; i < total; i += T) lm = max(lm, (u32)(keys[i] >> 32));
            if (threadIdx.x == 0) sh.n_cand = 0;
            sh.most[threadIdx.x] = lm;
            __syncthreads();
            const u32 bound = bound_among<T>(sh.most, out.k);
            for (u32 i = threadIdx.x; i < total; i += T) {
                const u64 key = keys[i];
                if (key && (u32)(key >> 32) >= bound) {
                    const u32 at = atomicAdd(&sh.n_cand, 1u);
                    if (at < CAND_CAP) sh.cand[at] = key;
                }
            }
            __syncthreads();
            n = sh.n_cand;
            if (n > CAND_CAP) n = add_head<T>(sh, r, 0, select_by_bits<DT, T>(sh, r, 0, r.nvec, out.k, bound));
        }
    }
    put_row<T>(out, row, tok, x, st, a.c, cand, n);
}

// Rows of more than 160000 tokens are cut into parts while there are too few to fill the GPU and the parts still hold a chunk
// of 16 KB.  Shorter ones are not: a second launch costs the caller 4 us, what a workgroup of 1024 lanes takes for 10^5 tokens
// (one row of 131072: 11 us a call whole, 15 in parts; of 262144: 17 and 15).
u32 split_shift(u32 rows, u32 vocab, u32 nvec) {
    u32 shift = 0;
    while (vocab > 160000 && shift < 6 && ((u64)rows << shift) < 1024 && (nvec >> (shift + 1)) >= BLOCK * UNROLL) ++shift;
    return shift;
}

// Lanes of a workgroup that has a row to itself: 1024 for the longest rows (2049 rows of 131073 tokens, a third of them
// skipped: 197 us with 256 lanes, 137 with 1024: fewer rows at a time share the load evenly) and where there are few rows;
// else 256, since eight workgroups a compute unit hide each other's phases (8192 rows of 32768 with 10 alternatives: 113 and
// 178 us).  (With alternatives of two-byte rows 1024 lanes leave 6 or 7 registers to scratch.)
constexpr int WIDE = 1024;
bool wide(u32 rows, u32 nvec) { return nvec >= 16384 || (rows <= 256 && nvec >= 2048); }

u32 split_vecs(u32 nvec, u32 shift) {
    const u32 each = (nvec + (1u << shift) - 1) >> shift;
    return (each + BLOCK * UNROLL - 1) / (BLOCK * UNROLL) * (BLOCK * UNROLL);
}

size_t split_bytes(u32 rows, u32 shift, u32 top) { return shift ? ((size_t)rows << shift) * (16 + 8 * (size_t)top) : 0; }

// The cells of workgroups of `threads` lanes over at most `vecs` vectors: chunks a cell, bytes in all.
u32 chunks_of(u32 vecs, u32 threads) { return (vecs + threads * UNROLL - 1) / (threads * UNROLL); }
u32 cell_chunks(u32 vecs, u32 threads) { return (chunks_of(vecs, threads) + CELL_ROWS - 1) / CELL_ROWS; }
size_t cell_bytes(u32 vecs, u32 threads, u32 per_cell) { return (chunks_of(vecs, threads) + per_cell - 1) / per_cell * threads * sizeof(float); }

template <int DT, bool ENT, bool TOP>
void launch(const Rows &a, const ScoreOut &out, Split sp, hipStream_t s) {
    const u32 vecs = sp.shift ? sp.vecs : a.nvec, threads = !sp.shift && wide(a.rows, a.nvec) ? WIDE : BLOCK;
    sp.per_cell = cell_chunks(vecs, threads);
    const size_t cells = TOP ? cell_bytes(vecs, threads, sp.per_cell) : 0;
    if (sp.shift) {
        hipLaunchKernelGGL((k_logits_score<DT, BLOCK, ENT, TOP, true>), grid_of(a.rows << sp.shift), dim3(BLOCK), cells, s, a, out, sp);
        hipLaunchKernelGGL((k_logits_score_join<DT, ENT, TOP>), grid_of(a.rows), dim3(BLOCK), 0, s, a, out, sp);
    } else if (threads == BLOCK) {
        hipLaunchKernelGGL((k_logits_score<DT, BLOCK, ENT, TOP, false>), grid_of(a.rows), dim3(BLOCK), cells, s, a, out, sp);
    } else {
        hipLaunchKernelGGL((k_logits_score<DT, WIDE, ENT, TOP, false>), grid_of(a.rows), dim3(WIDE), cells, s, a, out, sp);
    }
}

}  // namespace

extern "C" size_t mc_logits_score_workspace_bytes(uint32_t dtype, uint64_t rows, uint64_t vocab, uint32_t top) {
    if (dtype > MC_LOGITS_BF16 || rows >= (1ull << 31) || vocab >= (1ull << 31) || top > MC_LOGITS_MAX_TOP) return 0;
    const u64 per = dtype == MC_LOGITS_F32 ? 4 : 8;
    return split_bytes((u32)rows, split_shift((u32)rows, (u32)vocab, (u32)((vocab + per - 1) / per)), top);
}

extern "C" int mc_logits_score(const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
                               int64_t outer_stride, int64_t inner_stride, const void *tokens, uint32_t token_bytes,
                               int64_t token_outer_stride, int64_t token_inner_stride, double temperature, float *out_ml2p,
                               float *out_entropy, uint32_t top, int32_t *out_top, float *out_top_ml2p, void *workspace,
                               size_t workspace_bytes, void *stream) {
    const char *who = "mc_logits_score";
    Rows a{};
    if (int rc = tokens_of(who, a, tokens, token_bytes, token_outer_stride, token_inner_stride, outer * inner)) return rc;
    if (int rc = rows_of(who, a, logits, dtype, outer, inner, vocab, outer_stride, inner_stride, temperature,
                         one_run(inner, token_outer_stride, token_inner_stride)))
        return rc;
    if (top > MC_LOGITS_MAX_TOP || top > vocab) return bad(who, "top: at most 64 alternatives, and no more than tokens");
    if (a.rows == 0) return MC_OK;
    if (!out_ml2p || (top && (!out_top || !out_top_ml2p))) return bad(who, "no output");
    if (!aligned(out_ml2p, 4) || !aligned(out_entropy, 4) || (top && !(aligned(out_top, 4) && aligned(out_top_ml2p, 4))))
        return bad(who, "outputs that are not aligned to their type");
    ScoreOut out{out_ml2p, out_entropy, out_top_ml2p, out_top, top};
    hipStream_t s = (hipStream_t)stream;
    if (a.nvec <= SUB_VECS) {
        const u32 room = 2 * top + 9;  // (odd: the rows of a wave in banks of their own)
        BY_TYPE(dtype, BY_GROUP(a, {
                    if (top) hipLaunchKernelGGL((k_logits_score_sub<DT, G, NV, true, true>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK),
                                                BLOCK / G * room * sizeof(u64), s, a, out, room);
                    else if (out_entropy) hipLaunchKernelGGL((k_logits_score_sub<DT, G, NV, true, false>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, out, 0u);
                    else hipLaunchKernelGGL((k_logits_score_sub<DT, G, NV, false, false>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, out, 0u);
                }));
    } else {
        Split sp{split_shift(a.rows, a.vocab, a.nvec), 0, nullptr, nullptr, 0};
        if (sp.shift) {
            if (!workspace || workspace_bytes < split_bytes(a.rows, sp.shift, top) || !aligned(workspace, 16)) {
                mc_set_error("%s: an aligned workspace of %zu bytes is needed, not %zu", who, split_bytes(a.rows, sp.shift, top), workspace_bytes);
                return MC_ERR_WORKSPACE;
            }
            sp.vecs = split_vecs(a.nvec, sp.shift);
            sp.stats = (float4 *)workspace;
            sp.keys = (u64 *)(sp.stats + ((size_t)a.rows << sp.shift));
        }
        BY_TYPE(dtype, {
            if (top) launch<DT, true, true>(a, out, sp, s);
            else if (out_entropy) launch<DT, true, false>(a, out, sp, s);
            else launch<DT, false, false>(a, out, sp, s);
        });
    }
    HIP_TRY(hipGetLastError());
    return MC_OK;
}
