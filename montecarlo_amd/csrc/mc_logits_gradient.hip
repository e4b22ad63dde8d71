// The gradient of weights * (-log2 p of the given token) + entropy weights * entropy for the logits, with both values
// (formulas: mc_logits_score.hip).  A row is read once and its gradient written once while its vectors fit the registers
// of a group of lanes or of one workgroup of up to 1024 lanes (131072 tokens of two bytes); longer rows, and
// rows too few to fill the GPU, are summed part by part by one launch, joined by a second one (before anything is written, since the
// gradient may take the logits' place) and written by a third.
#include "mc_logits.h"

namespace {

struct GradOut {
    View weights, entropy_weights;  // entropy_weights.p may be null
    float inv_t;
    float *ml2p, *entropy;
    char *grad;
};

// What the elements of a row's gradient need: p (C - B y) - [i = t] A with C = A - B (H - log2 Z); all 0 where there is none.
struct Slope {
    float A, B, C, inv;
    bool none;
    int tok;
};

template <bool ENT>
__device__ __forceinline__ Slope slope_of(const Rows &a, const GradOut &out, u32 row, int tok, const Stat &st) {
    Slope s;
    s.none = tok == MC_TOKEN_SKIP || st.s == 0.f;
    s.A = tok >= 0 && !s.none ? *(const float *)at(out.weights, a.inner, row) * a.c : 0.f;
    s.B = ENT && !s.none ? *(const float *)at(out.entropy_weights, a.inner, row) * out.inv_t : 0.f;
    s.inv = s.none ? 0.f : inverse(st.s);
    s.C = ENT && !s.none ? __builtin_fmaf(st.e * s.inv, s.B, s.A) : s.A;  // (H - log2 Z = -e / Z)
    s.tok = tok;
    return s;
}

template <bool ENT>
__device__ __forceinline__ float slope(float y, const Slope &s) {
    const float p = exp2_(y) * s.inv;
    return ENT ? p * __builtin_fmaf(-s.B, fmaxf(y, -FAR), s.C) : p * s.A;
}

template <int DT, bool ENT, bool EXACT>
__device__ __forceinline__ void slope_vec(const raw4 &q, u32 from, const Slope &s, const Expo &y_of, float *g) {
#pragma unroll
    for (int j = 0; j < VEC<DT>; ++j) {
        const float x = unpack<DT>(q, j);
        g[j] = slope<ENT>(EXACT ? y_of(x) : y_of.fast(x), s);
    }
    const u32 t = (u32)s.tok - from;
    if (t < (u32)VEC<DT>) {
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) g[j] -= t == (u32)j ? s.A : 0.f;
    }
}

// vector v of a row's gradient, which begins at gp
template <int DT, bool ENT>
__device__ __forceinline__ void put_slope(char *gp, const Span &r, u32 v, const raw4 &q, const Slope &s, const Expo &y_of, bool exact) {
    float g[VEC<DT>];
    if (s.none) {
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) g[j] = 0.f;
    } else if (exact) {
        slope_vec<DT, ENT, true>(q, r.head + v * VEC<DT>, s, y_of, g);
    } else {
        slope_vec<DT, ENT, false>(q, r.head + v * VEC<DT>, s, y_of, g);
    }
    store_at<DT, true>(gp + r.head * Elt<DT>::BYTES, v * VEC<DT>, r.vocab, g);
}

// the first element of a row whose vectors begin behind it
template <int DT, bool ENT>
__device__ __forceinline__ void put_head(char *gp, const Span &r, const Slope &s, const Expo &y_of) {
    if (!r.head) return;
    float g = slope<ENT>(y_of(r.first), s);
    if (s.tok == 0) g -= s.A;
    *(unsigned short *)gp = (unsigned short)pack2<DT>(s.none ? 0.f : g, 0.f);
}

template <int DT, int G, int NV, bool ENT>
__global__ __launch_bounds__(BLOCK, 8) void k_logits_gradient_sub(Rows a, GradOut out) {
    const u32 row = block_id() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows;
    const int tok = there ? token_of(a, row) : MC_TOKEN_SKIP;
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT, NV> r;
    load_row<DT, G>(r, p, a, tok != MC_TOKEN_SKIP);
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    const Stat st = sub_stat<DT, G, ENT>(r, a.c);
    if (!there) return;
    if (lane == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (ENT) out.entropy[row] = entropy_of(tok, st);
    }
    const Slope s = slope_of<ENT>(a, out, row, tok, st);
    const Expo y_of(st, a.c);
    char *gp = out.grad + (u64)row * a.vocab * Elt<DT>::BYTES;
#pragma unroll
    for (int i = 0; i < SubRow<DT, NV>::N; ++i) {
        const u32 v = i * G + lane;
        if (i + 1 < SubRow<DT, NV>::N || v < a.nvec) {
            // (a last vector that reaches back computes and stores there what the one before it does)
            const u32 from = NV == 0 ? 0u : i + 1 < NV ? v * VEC<DT> : min(v * VEC<DT>, a.vocab - VEC<DT>);
            float g[VEC<DT>];
            if (st.exact) slope_vec<DT, ENT, true>(r.q[i], from, s, y_of, g);
            else slope_vec<DT, ENT, false>(r.q[i], from, s, y_of, g);
            store_at<DT, false, NV == 0>(gp, from, a.vocab, g);
        }
    }
}

// one workgroup a row, the row in its registers: HELD vectors a lane at most
template <int DT, int T, int HELD, bool ENT>
__global__ __launch_bounds__(T, HELD > 8 ? 4 : 8) void k_logits_gradient_held(Rows a, GradOut out) {
    const u32 row = block_id();
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, tok != MC_TOKEN_SKIP);
    char *gp = out.grad + (u64)row * a.vocab * Elt<DT>::BYTES;
    const u32 nv = (r.nvec + T - 1) / T;
    const float x = tok >= 0 ? element<DT>(p, tok) : 0.f;
    Stat st{-INFINITY, 0.f, 0.f, false};
    raw4 q[HELD];
    if (tok != MC_TOKEN_SKIP) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (i < (int)nv) q[i] = load_vec<DT>(r, i * T + threadIdx.x, r.nvec);
        }
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (i < (int)nv) {
#pragma unroll
                for (int j = 0; j < VEC<DT>; ++j) st.m = maximum(st.m, unpack<DT>(q[i], j));
            }
        }
        const Expo y_of(st, a.c);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            asm("" : "+v"(q[i]));  // (see forget)
            if (i < (int)nv) {
#pragma unroll
                for (int j = 0; j < VEC<DT>; ++j) {
                    const float y = y_of.fast(unpack<DT>(q[i], j)), w = exp2_(y);
                    st.s += w;
                    if (ENT) st.e = __builtin_fmaf(w, fmaxf(y, -FAR), st.e);
                }
            }
        }
        if (threadIdx.x == 0) take_one<ENT>(st, r.first, a.c);
        st = block_stat<T, ENT>(st, a.c);
#pragma unroll
        for (int i = 0; i < HELD; ++i) asm("" : "+v"(q[i]));
        if (doubtful(st.m, a.c)) st = exact_stat<DT, T, ENT>(r, a.c, st.m);
    }
    const Slope s = slope_of<ENT>(a, out, row, tok, st);
    const Expo y_of(st, a.c);
    if (threadIdx.x == 0) {
        out.ml2p[row] = ml2p_of(tok, st, x, a.c);
        if (ENT) out.entropy[row] = entropy_of(tok, st);
        put_head<DT, ENT>(gp, r, s, y_of);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const u32 v = i * T + threadIdx.x;
        if (i < (int)nv && v < r.nvec) put_slope<DT, ENT>(gp, r, v, q[i], s, y_of, st.exact);
    }
}

// 2^shift workgroups of `vecs` vectors a row
struct Split {
    u32 shift, vecs;
    float4 *stats;  // [row][part]: m, s, e
};

template <int DT, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_logits_gradient_sums(Rows a, Split sp) {
    const u32 id = block_id(), row = id >> sp.shift, part = id & ((1u << sp.shift) - 1);
    if (row >= a.rows || token_of(a, row) == MC_TOKEN_SKIP) return;
    const Span r = span_of<DT>(a, at(a.logits, a.inner, row), true);
    const u32 v0 = min(part * sp.vecs, r.nvec), v1 = min(r.nvec, v0 + sp.vecs);
    Stat st{-INFINITY, 0.f, 0.f, false};
    for (u32 v = v0; v < v1; v += BLOCK * UNROLL) {
        raw4 q[UNROLL];
        load_chunk<DT, BLOCK>(q, r, v, threadIdx.x, v1);
        take<DT, ENT>(st, q, a.c);
    }
    if (threadIdx.x == 0 && part == 0) take_one<ENT>(st, r.first, a.c);
    st = block_stat<BLOCK, ENT>(st, a.c);
    if (threadIdx.x == 0) sp.stats[id] = make_float4(st.m, st.s, st.e, 0.f);
}

// A row's statistics joined into its first part's place, and its outputs: before any part of the row is written, since
// the gradient may take the logits' place.
template <int DT, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_logits_gradient_join(Rows a, GradOut out, Split sp) {
    const u32 row = block_id(), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    const char *p = at(a.logits, a.inner, row);
    Stat st{-INFINITY, 0.f, 0.f, false};
    if (tok != MC_TOKEN_SKIP) {
        if (lane < (1u << sp.shift)) {
            const float4 f = sp.stats[((u64)row << sp.shift) + lane];
            st = Stat{f.x, f.y, f.z, false};
        }
        st = group_stat<64, ENT>(st, a.c);
        if (doubtful(st.m, a.c)) st = exact_stat<DT, BLOCK, ENT>(span_of<DT>(a, p, true), a.c, st.m);
    }
    __syncthreads();  // (every wave has read the parts)
    if (threadIdx.x == 0) {
        sp.stats[(u64)row << sp.shift] = make_float4(st.m, st.s, st.e, st.exact ? 1.f : 0.f);
        out.ml2p[row] = ml2p_of(tok, st, tok >= 0 ? element<DT>(p, tok) : 0.f, a.c);
        if (ENT) out.entropy[row] = entropy_of(tok, st);
    }
}

template <int DT, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_logits_gradient_parts(Rows a, GradOut out, Split sp) {
    const u32 id = block_id(), row = id >> sp.shift, part = id & ((1u << sp.shift) - 1);
    if (row >= a.rows) return;
    const int tok = token_of(a, row);
    const Span r = span_of<DT>(a, at(a.logits, a.inner, row), tok != MC_TOKEN_SKIP);
    char *gp = out.grad + (u64)row * a.vocab * Elt<DT>::BYTES;
    const u32 v0 = min(part * sp.vecs, r.nvec), v1 = min(r.nvec, v0 + sp.vecs);
    const float4 f = sp.stats[(u64)row << sp.shift];
    const Stat st{f.x, f.y, f.z, f.w != 0.f};
    const Slope s = slope_of<ENT>(a, out, row, tok, st);
    const Expo y_of(st, a.c);
    if (threadIdx.x == 0 && part == 0) put_head<DT, ENT>(gp, r, s, y_of);
    for (u32 v = v0; v < v1; v += BLOCK * UNROLL) {
        raw4 q[UNROLL];
        if (!s.none) load_chunk<DT, BLOCK>(q, r, v, threadIdx.x, v1);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const u32 mine = v + u * BLOCK + threadIdx.x;
            if (mine < v1) put_slope<DT, ENT>(gp, r, mine, q[u], s, y_of, st.exact);
        }
    }
}

constexpr u32 HELD_VECS = 1024 * 16;  // vectors of a row that one workgroup holds

// Parts where a row is longer than one workgroup holds, and where it is half as long and there are few (one row of 131072
// tokens of two bytes: 18 us either way for a caller who waits for the launches, 18 and 8 us of the GPU).
u32 split_shift(u32 rows, u32 nvec) {
    u32 shift = 0;
    if (nvec > HELD_VECS || (nvec > HELD_VECS / 2 && rows <= 64)) {
        while (shift < 6 && ((u64)rows << shift) < 256 && (nvec >> (shift + 1)) >= BLOCK * UNROLL) ++shift;
        while (shift < 6 && nvec > HELD_VECS && (nvec >> shift) > HELD_VECS / 4) ++shift;
    }
    return shift;
}

size_t split_bytes(u32 rows, u32 shift) { return shift ? ((size_t)rows << shift) * 16 : 0; }

template <int DT, bool ENT>
void launch(const Rows &a, const GradOut &out, const Split &sp, hipStream_t s) {
    const bool few = a.rows <= 256 && a.nvec >= 1024;  // (all the lanes there are for each)
    if (a.nvec <= SUB_VECS) {
        BY_GROUP(a, hipLaunchKernelGGL((k_logits_gradient_sub<DT, G, NV, ENT>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, out));
    } else if (sp.shift) {
        hipLaunchKernelGGL((k_logits_gradient_sums<DT, ENT>), grid_of(a.rows << sp.shift), dim3(BLOCK), 0, s, a, sp);
        hipLaunchKernelGGL((k_logits_gradient_join<DT, ENT>), grid_of(a.rows), dim3(BLOCK), 0, s, a, out, sp);
        hipLaunchKernelGGL((k_logits_gradient_parts<DT, ENT>), grid_of(a.rows << sp.shift), dim3(BLOCK), 0, s, a, out, sp);
    } else if (a.nvec <= 256 * 8 && !few) {
        hipLaunchKernelGGL((k_logits_gradient_held<DT, 256, 8, ENT>), grid_of(a.rows), dim3(256), 0, s, a, out);
    } else if (a.nvec <= 512 * 8 && !few) {
        hipLaunchKernelGGL((k_logits_gradient_held<DT, 512, 8, ENT>), grid_of(a.rows), dim3(512), 0, s, a, out);
    } else if (a.nvec <= 1024 * 8) {
        hipLaunchKernelGGL((k_logits_gradient_held<DT, 1024, 8, ENT>), grid_of(a.rows), dim3(1024), 0, s, a, out);
    } else {
        hipLaunchKernelGGL((k_logits_gradient_held<DT, 1024, 16, ENT>), grid_of(a.rows), dim3(1024), 0, s, a, out);
    }
}

}  // namespace

extern "C" size_t mc_logits_gradient_workspace_bytes(uint32_t dtype, uint64_t rows, uint64_t vocab) {
    if (dtype > MC_LOGITS_BF16 || rows >= (1ull << 31) || vocab >= (1ull << 31)) return 0;
    const u64 per = dtype == MC_LOGITS_F32 ? 4 : 8;
    return split_bytes((u32)rows, split_shift((u32)rows, (u32)((vocab + per - 1) / per)));
}

extern "C" int mc_logits_gradient(const void *logits, uint32_t dtype, uint64_t outer, uint64_t inner, uint64_t vocab,
                                  int64_t outer_stride, int64_t inner_stride, const void *tokens, uint32_t token_bytes,
                                  int64_t token_outer_stride, int64_t token_inner_stride, double temperature,
                                  const float *weights, int64_t weight_outer_stride, int64_t weight_inner_stride,
                                  const float *entropy_weights, int64_t entropy_outer_stride, int64_t entropy_inner_stride,
                                  float *out_ml2p, float *out_entropy, void *out_grad, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    const char *who = "mc_logits_gradient";
    Rows a{};
    if (int rc = tokens_of(who, a, tokens, token_bytes, token_outer_stride, token_inner_stride, outer * inner)) return rc;
    const bool flat = one_run(inner, token_outer_stride, token_inner_stride) && one_run(inner, weight_outer_stride, weight_inner_stride) &&
                      (!entropy_weights || one_run(inner, entropy_outer_stride, entropy_inner_stride));
    if (int rc = rows_of(who, a, logits, dtype, outer, inner, vocab, outer_stride, inner_stride, temperature, flat)) return rc;
    if (a.rows == 0) return MC_OK;
    if (!weights) return bad(who, "no weights");
    if (!out_ml2p || !out_grad || (entropy_weights && !out_entropy)) return bad(who, "no output");
    if (!aligned(out_grad, dtype == MC_LOGITS_F32 ? 4 : 2)) return bad(who, "a gradient that is not aligned to its type");
    if (!aligned(weights, 4) || !aligned(entropy_weights, 4)) return bad(who, "weights that are not aligned to their type");
    if (!aligned(out_ml2p, 4) || (entropy_weights && !aligned(out_entropy, 4))) return bad(who, "outputs that are not aligned to their type");
    GradOut out{view_of(weights, weight_outer_stride, weight_inner_stride, 4),
                view_of(entropy_weights, entropy_outer_stride, entropy_inner_stride, 4),
                (float)(1.0 / temperature), out_ml2p, out_entropy, (char *)out_grad};
    Split sp{split_shift(a.rows, a.nvec), 0, nullptr};
    if (sp.shift) {
        if (!workspace || workspace_bytes < split_bytes(a.rows, sp.shift) || !aligned(workspace, 16)) {
            mc_set_error("%s: an aligned workspace of %zu bytes is needed, not %zu", who, split_bytes(a.rows, sp.shift), workspace_bytes);
            return MC_ERR_WORKSPACE;
        }
        const u32 each = (a.nvec + (1u << sp.shift) - 1) >> sp.shift;
        sp.vecs = (each + BLOCK - 1) / BLOCK * BLOCK;
        sp.stats = (float4 *)workspace;
    }
    BY_TYPE(dtype, {
        if (entropy_weights) launch<DT, true>(a, out, sp, (hipStream_t)stream);
        else launch<DT, false>(a, out, sp, (hipStream_t)stream);
    });
    HIP_TRY(hipGetLastError());
    return MC_OK;
}
