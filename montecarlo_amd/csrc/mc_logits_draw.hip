// Draws from rows of logits by inversion, and the keys of whole passwords (formulas: mc_logits_score.hip).
//
// The draw is defined by running sums in 64 bits.  Sums in 32 bits are known to e = a few parts in 10^6 and leave the token
// open where u Z lies nearer than that to an end of its interval: a share sum of min(p_i, 2 e) of the draws, 0.07 % at V = 97,
// a twelfth at V = 32768 and a fifth at 131072 (logits of deviation 2.5; most where 10^5 are about equally likely).  Rows begin
// with them (seven operations an element; 64 bits take sixteen) and are summed again in 64 bits where they leave the token
// open, but for those that begin with 64 bits (in_64_bits).
// Weights in 64 bits come from a polynomial that is right to 4e-11 (this GPU does them at the rate of 32 bits), and where u Z
// lies within 1e-10 Z of an end (a row in 10^5) the row is summed once more with the library's exponential.  Exponents of
// 64 bits reach far enough that no maximum has to be known first.
#include "mc_logits.h"

#include <algorithm>

#include "mc_philox.h"

namespace {

// 2^y from y c's whole part n (as the low word of n + 1.5 * 2^52) and the rest f in [-1/2, 1/2]: the polynomial of degree 7
// that approximates 2^f best relative to its value (found by exchange of the extremal points; largest error 4.03e-11).
__device__ __forceinline__ double power_of(double n_word, double f) {
    double p = 0x1.fe1786b50da52p-17;
    p = __builtin_fma(p, f, 0x1.446a1fdd54f3ap-13);
    p = __builtin_fma(p, f, 0x1.5d8a7085cddb8p-10);
    p = __builtin_fma(p, f, 0x1.3b29dc40d2ec5p-7);
    p = __builtin_fma(p, f, 0x1.c6b08aaf3156ep-5);
    p = __builtin_fma(p, f, 0x1.ebfbe0a4be886p-3);
    p = __builtin_fma(p, f, 0x1.62e42ff11627ap-1);
    p = __builtin_fma(p, f, 0x1.ffffffffabbccp-1);
    return __hiloint2double(__double2hiint(p) + (int)((u32)__double2loint(n_word) << 20), __double2loint(p));
}

// 2^(x c) for x c in [-1000, 900]; lower ones as 2^-1000: so far below any sum that `good` lets pass that it changes
// nothing.
struct Power {
    double c;
    float lo;
    __device__ __forceinline__ double operator()(float x) const {
        const double v = (double)maximum(x, lo), t = __builtin_fma(v, c, 0x1.8p52);
        return power_of(t, __builtin_fma(v, c, 0x1.8p52 - t));
    }
};

// 2^((x - m) c): for rows whose logits are too far from 0 for Power
struct PowerBelow {
    double c, m;
    __device__ __forceinline__ double operator()(float x) const {
        const double y = fmax(((double)x - m) * c, -1000.), t = y + 0x1.8p52;
        return power_of(t, y - (t - 0x1.8p52));
    }
};
constexpr double MARGIN = 1e-10;

// The draw's own weights: exp((x - m) / T) in 64 bits, m the row's largest logit.
struct Definition {
    double t, m;
    __device__ __forceinline__ double operator()(float x) const { return exp(((double)x - m) / t); }
};

// whether a row with this largest logit suits Power: no exponent too large, not all too small
__device__ __forceinline__ bool good(float m, double c) { return fabs((double)m * c) <= 900.; }

// what a row gives that has no draw: nothing left, or a NaN or +inf
__device__ __forceinline__ bool drawable(float m) { return fabsf(m) < INFINITY; }
__device__ __forceinline__ float no_draw(float m) { return m == -INFINITY ? INFINITY : NAN; }

// -log2 p of a token whose exponent is y, under a sum in 64 bits
__device__ __forceinline__ float ml2p_under(double z, double y) {
    int e;
    const double m = frexp(z, &e);
    return at_least_0((float)(((double)e - y) + (double)log2f((float)m)));
}

// What a row's tokens score under the sums that it began with: a token comes with one value, whether its uniform was
// decided by these sums or, beside the border of an interval, by those of a later pass.
struct Under64 {
    double z, m, c;
    __device__ __forceinline__ float operator()(float x) const { return ml2p_under(z, ((double)x - m) * c); }
};
struct Under32 {
    float lz;  // log2 Z
    Expo y_of;
    __device__ __forceinline__ float operator()(float x) const { return at_least_0(lz - y_of.fast(x)); }
};

struct DrawArgs {
    const double *uniforms;  // or null: Philox
    u64 seed, first_id;
    u32 draw;
    double t, margin;        // margin: how far off the running sums in 32 bits may be, as a share of Z
    Power power;
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

// ---- rows of few tokens --------------------------------------------------------------------------------------------------
// The token of a group's row in registers: running sums in the order of the index, vector step by vector step.  False when
// u Z lies within `margin` Z of an end of the token's interval (0 takes any answer).
template <int DT, int G, typename W, int NV>
__device__ __forceinline__ bool draw_sub(const SubRow<DT, NV> &r, const W &weight, double u, double margin, u32 &token, float &x, double &z) {
    constexpr int N = SubRow<DT, NV>::N;
    double s[N];
    z = 0.;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = 0.;
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) s[i] += weight(unpack<DT>(vec_of(r, i), j));
        z += s[i];
    }
    z = group_all<G>(z, Add());
    const double target = u * z, near = margin * z;
    // the vector step whose running sum passes the target, or the last one with any weight
    double before = 0., run = 0.;
    double mine = 0.;
    raw4 q = vec_of(r, 0);
    u32 from = from_of<DT, G>(r, 0);
    bool found = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double step = group_all<G>(s[i], Add());
        const bool here = !found && step > 0.;
        before = here ? run : before;
        mine = here ? s[i] : mine;
        choose(q, vec_of(r, i), here);
        from = here ? from_of<DT, G>(r, i) : from;
        found = found || (here && run + step > target);
        run += step;
    }
    const double inc = group_scan<G>(mine);
    const u32 shift = threadIdx.x & 63 & ~(G - 1);
    const u64 all = G == 64 ? ~0ull : (1ull << (G & 63)) - 1;
    const u64 passes = (__ballot(before + inc > target) >> shift) & all, some = (__ballot(mine > 0.) >> shift) & all;
    // (a sum that passes by a rounding only, or none: the last lane with any weight)
    const bool hit = found && passes;
    const u32 who = hit ? (u32)__ffsll((unsigned long long)passes) - 1 : some ? 63u - (u32)__clzll((long long)some) : 0u;
    double at_lo = before + (inc - mine);
    u32 got = 0xFFFFFFFFu, last = 0;
    float got_x = 0.f, last_x = 0.f;
    bool ok = false;
#pragma unroll
    for (int j = 0; j < VEC<DT>; ++j) {
        const float e = unpack<DT>(q, j);
        const double w = weight(e);
        const double next = at_lo + w;
        if (w > 0.) {
            last = from + j;
            last_x = e;
            if (got == 0xFFFFFFFFu && next > target) {
                got = from + j;
                got_x = e;
                ok = hit && target - at_lo >= near && next - target >= near;
            }
        }
        at_lo = next;
    }
    if (!hit || got == 0xFFFFFFFFu) got = last, got_x = last_x;
    token = __shfl(got, who, G);
    x = __shfl(got_x, who, G);
    return __shfl((int)ok, who, G) || margin == 0.;
}

// The token in a vector of which u Z lies `t` behind the beginning: running sums ascend, so that its place is the number of
// them at or below t, and the nearest of them says how near an end is.  True if the token is here and none is nearer than `near`.
template <int DT>
__device__ __forceinline__ bool place_of(const raw4 &q, const Expo &y_of, float t, float near, u32 from, u32 &token, float &x) {
    float run = 0.f, off = t;
    u32 place = 0;
#pragma unroll
    for (int j = 0; j < VEC<DT>; ++j) {
        run += exp2_(y_of.fast(unpack<DT>(q, j)));
        place += run <= t;
        off = fminf(off, fabsf(run - t));
    }
    token = from + place;
    u32 word = q[0];
    constexpr u32 PER = VEC<DT> / 4;
#pragma unroll
    for (u32 w = 1; w < 4; ++w) word = place >= w * PER ? q[w] : word;
    x = PER == 1 ? to_float<DT>(word, 0) : to_float<DT>(place & 1 ? word >> 16 : word & 0xFFFFu, 0);
    return off >= near && place < (u32)VEC<DT>;
}

// The same in 32 bits, for the lane that holds the token: true there, and only there, when u Z is at least `margin` Z from both
// ends of the token's interval (nowhere otherwise).
template <int DT, int G, int NV>
__device__ __forceinline__ bool draw_fast(const SubRow<DT, NV> &r, const Expo &y_of, double u, double margin, u32 &token, float &x, float &z) {
    constexpr int N = SubRow<DT, NV>::N;
    float s[N], upto[N], mine = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float w[VEC<DT>];
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) w[j] = exp2_(y_of.fast(unpack<DT>(vec_of(r, i), j)));
        s[i] = pairs<VEC<DT>>(w);
        upto[i] = group_all<G>(s[i], Add());
        if (i) upto[i] += upto[i - 1];
    }
    z = upto[N - 1];
    const float target = (float)(u * (double)z), near = (float)margin * z;
    float before = 0.f;
    raw4 q = vec_of(r, 0);
    u32 from = from_of<DT, G>(r, 0);
    mine = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) {
        const bool past = upto[i - 1] <= target;
        before = past ? upto[i - 1] : before;
        mine = past ? s[i] : mine;
        from = past ? from_of<DT, G>(r, i) : from;
        choose(q, vec_of(r, i), past);
    }
    return place_of<DT>(q, y_of, target - (before + (group_scan<G>(mine) - mine)), near, from, token, x);
}

template <int DT, int G, int NV>
__global__ __launch_bounds__(BLOCK, NV > 5 ? 4 : 6) void k_logits_draw_sub(Rows a, DrawArgs d) {
    const u32 row = block_id() * (BLOCK / G) + threadIdx.x / G, lane = threadIdx.x & (G - 1);
    const bool there = row < a.rows, live = there && (!d.live || d.live[row]);
    const char *p = there ? at(a.logits, a.inner, row) : nullptr;
    SubRow<DT, NV> r;
    load_row<DT, G>(r, p, a, live);
    const double u = there ? uniform_of(d, row) : 0.;
    Stat st{sub_max<DT, G>(r), 0.f, 0.f, false};
    if (NV > 4) forget(r);
    const Expo y_of(st, a.c);
    const float m = st.m;
    u32 token;
    float x;
    if (drawable(m) && live) {  // (a group's lanes agree)
        const bool mine = draw_fast<DT, G>(r, y_of, u, d.margin, token, x, st.s) && !doubtful(m, a.c);
        if (mine) {
            d.token[row] = (int)token;
            d.ml2p[row] = Under32{log2_(st.s), y_of}(x);
        }
        st.exact = group_sum<G>(mine) == 0;  // still open
    } else if (there && lane == 0) {
        d.token[row] = live ? MC_TOKEN_OUTSIDE : MC_TOKEN_SKIP;
        d.ml2p[row] = live ? no_draw(m) : 0.f;
    }
    const bool open = st.exact;
    if (__ballot(open)) {  // the whole wave decides again, in 64 bits
        // (what the row's tokens score under waits in LDS: its registers, across what follows, cost all waves one of seven a SIMD)
        __shared__ float2 sums[BLOCK];
        sums[threadIdx.x] = make_float2(st.s, y_of.M);
        asm volatile("" ::: "memory");
        forget(r);
        double z;
        bool now = draw_sub<DT, G>(r, PowerBelow{d.power.c, (double)m}, u, MARGIN, token, x, z);
        if (__ballot(open && !now)) {  // and again, by the definition
            forget(r);
            u32 again;
            float x_again;
            double z_again;
            draw_sub<DT, G>(r, Definition{d.t, (double)m}, u, 0., again, x_again, z_again);
            if (!now) token = again, x = x_again, z = z_again;
        }
        if (open && lane == 0) {
            d.token[row] = (int)token;
            const float2 sum = sums[threadIdx.x];
            Expo again = y_of;
            again.M = sum.y;
            d.ml2p[row] = doubtful(m, a.c) ? Under64{z, (double)m, d.power.c}(x) : Under32{log2_(sum.x), again}(x);
        }
    }
}

// ---- rows of many tokens ---------------------------------------------------------------------------------------------------
constexpr int WIDE = 512, WIDE_WAVES = WIDE / 64, STEPS = 4;

// The token by the definition's weights, by the whole workgroup: every wave sums a share of the row, and the one whose share
// holds the token (true there) looks for it, first by steps of 4 x 64 tokens.  Where sums that are right to 1e-10 leave it open:
// one row of 131072 in 40000, which took a single wave 1.8 ms.
template <int DT, int T>
__device__ __forceinline__ bool draw_exact(const char *p, const Rows &a, const Definition &weight, double u, u32 &token, float &x) {
    constexpr int WAVES = T / 64;
    constexpr u32 STEP = 4 * 64;
    __shared__ double part[WAVES];
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const auto step_sum = [&](u32 from, u32 to) {
        float e[4];
#pragma unroll
        for (u32 j = 0; j < 4; ++j) e[j] = from + j * 64 + lane < to ? element<DT>(p, from + j * 64 + lane) : -INFINITY;
        double w = 0.;
#pragma unroll 1
        for (u32 j = 0; j < 4; ++j) {
            w += weight(e[0]);
            e[0] = e[1], e[1] = e[2], e[2] = e[3];
        }
        return w;
    };
    const u32 share = (a.vocab / STEP / WAVES + 1) * STEP, i0 = min(wave * share, a.vocab), i1 = min(a.vocab, i0 + share);
    double s = 0.;
#pragma unroll 1
    for (u32 i = i0; i < i1; i += STEP) s += step_sum(i, i1);
    s = group_all<64>(s, Add());
    if (lane == 0) part[wave] = s;
    __syncthreads();
    const double inc = group_scan<64>(lane < (u32)WAVES ? part[lane] : 0.);
    const double target = u * __shfl(inc, 63);
    const u64 passes = __ballot(inc > target);
    const u32 who = passes ? (u32)__ffsll((unsigned long long)passes) - 1 : WAVES - 1;
    if (wave != who) return false;
    double before = who ? __shfl(inc, (int)who - 1) : 0.;
    u32 from = i0;
#pragma unroll 1
    for (; from + STEP < i1; from += STEP) {
        const double next = before + group_all<64>(step_sum(from, i1), Add());
        if (next > target) break;
        before = next;
    }
    token = 0;
    // (the last token with any weight stands in for a target at or behind the last running sum: found from 0 on, if not from here)
    for (bool any = false, again = false; !any && !again; again = from == 0, from = 0, before = 0.) {
#pragma unroll 1
        for (u32 base = from; base < a.vocab; base += 64) {
            const float e = base + lane < a.vocab ? element<DT>(p, base + lane) : -INFINITY;
            const double w = weight(e), upto = before + group_scan<64>(w);
            const u64 over = __ballot(w > 0. && upto > target), some = __ballot(w > 0.);
            if (some) {
                const u32 at = over ? (u32)__ffsll((unsigned long long)over) - 1 : 63u - (u32)__clzll((long long)some);
                token = base + at;
                x = __shfl(e, at);
                any = true;
            }
            if (over) break;
            before = __shfl(upto, 63);
        }
    }
    return true;
}

// The token among vectors v0 .. v1, whose running sums begin at `before`, by one wave: the sums of rounds of STEPS steps of
// 64 vectors.  False when the target lies within `margin` of an end of the token's interval.
template <int DT>
__device__ __forceinline__ bool locate(const Span &r, const PowerBelow &weight, u32 v0, u32 v1, double before, double target, double margin,
                                       u32 &token, float &x) {
    const u32 lane = threadIdx.x & 63;
    if (v0 == 0 && r.head) {
        const double next = before + weight(r.first);
        if (next > target) {
            token = 0;
            x = r.first;
            return next - target >= margin;
        }
        if (target - next < margin) return false;
        before = next;
    }
#pragma unroll 1
    for (u32 base = v0; base < v1; base += 64 * STEPS) {
        raw4 q[STEPS];
        double s[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) q[i] = load_vec<DT>(r, base + i * 64 + lane, v1);
        raw4 mq = q[0];
        double ms = 0.;
        double start = before, run = before;
        u32 step = 0;
        bool found = false;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            s[i] = 0.;
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) s[i] += weight(unpack<DT>(q[i], j));
            const double all = group_all<64>(s[i], Add());
            const bool here = !found && run + all > target;
            choose(mq, q[i], here);
            ms = here ? s[i] : ms;
            start = here ? run : start;
            step = here ? i : step;
            found = found || here;
            run += all;
        }
        if (found) {
            const double minc = group_scan<64>(ms);
            const u64 over = __ballot(start + minc > target);
            const u32 who = over ? (u32)__ffsll((unsigned long long)over) - 1 : 63u;
            double at_lo = start + (minc - ms);
            u32 got = 0;
            float got_x = 0.f;
            bool sure = false;
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float e = unpack<DT>(mq, j);
                const double next = at_lo + weight(e);
                if (!sure && target - at_lo >= margin && next - target >= margin) {
                    sure = true;
                    got = r.head + (base + step * 64 + lane) * VEC<DT> + j;
                    got_x = e;
                }
                at_lo = next;
            }
            token = __shfl(got, who);
            x = __shfl(got_x, who);
            return over && __shfl((int)sure, who);
        }
        before = run;
    }
    return false;
}

// How the work on a row is cut: 2^shift workgroups of `vecs` vectors, whose sums another launch joins.
struct Split {
    u32 shift, vecs;
    float *most;   // [row][part]: the largest logit
    double *sums;  // [row][part][wave]: the waves' shares of the part lie behind each other
};
constexpr int PART_WAVES = BLOCK / 64;

// the wave's sum and largest logit over its share of vectors v0 .. v1
template <int DT, int U, typename W>
__device__ __forceinline__ void sum_vecs(const Span &r, const W &weight, u32 v0, u32 v1, u32 lane, double &s, float &m) {
    s = 0.;
    m = -INFINITY;
    if (v0 == 0 && lane == 0 && r.head) {
        s = weight(r.first);
        m = r.first;
    }
    for (u32 v = v0; v < v1; v += 64 * U) {
        raw4 q[U];
        load_chunk<DT, 64>(q, r, v, lane, v1);
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) {
                const float e = unpack<DT>(q[i], j);
                m = maximum(m, e);
                s += weight(e);
            }
    }
    s = group_all<64>(s, Add());
    m = group_all<64>(m, Max());
}

// the sums of the parts of a row
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_logits_draw_sums(Rows a, DrawArgs d, Split sp) {
    __shared__ float pm[PART_WAVES];
    const u32 id = block_id(), row = id >> sp.shift, part = id & ((1u << sp.shift) - 1), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (row >= a.rows || (d.live && !d.live[row])) return;
    const Span r = span_of<DT>(a, at(a.logits, a.inner, row), true);
    const u32 share = sp.vecs / PART_WAVES, v0 = min(part * sp.vecs + wave * share, r.nvec), v1 = min(r.nvec, v0 + share);
    double s;
    float m;
    sum_vecs<DT, 2>(r, d.power, v0, v1, lane, s, m);
    if (lane == 0) {
        sp.sums[(u64)id * PART_WAVES + wave] = s;
        pm[wave] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < PART_WAVES; ++w) m = maximum(m, pm[w]);
        sp.most[id] = m;
    }
}

// A row of which lane i holds the sum of part i of `share` vectors: its token, by one wave; false where its outputs are still to
// be put.  `within` (if by_shares): the same for the PART_WAVES shares of the lane's part.  (Sums of Power are those of PowerBelow
// for m = 0 but for roundings far below the margin.)  `value`: what a token scores.
template <int DT, typename V>
__device__ __forceinline__ bool put_token(const DrawArgs &d, u32 row, const Span &r, const PowerBelow &weight, double mine, u32 share, double u,
                                          bool by_shares, const double (&within)[PART_WAVES], const V &value) {
    const double inc = group_scan<64>(mine), z = __shfl(inc, 63), target = u * z;
    const u64 passes = __ballot(inc > target);
    if (!passes) return false;
    const u32 part = (u32)__ffsll((unsigned long long)passes) - 1;
    double before = __shfl(inc - mine, part);
    u32 v0 = part * share, v1 = v0 + share;
    if (by_shares) {
        v1 = v0;
        bool found = false;
#pragma unroll
        for (int w = 0; w < PART_WAVES; ++w) {
            const double next = before + __shfl(within[w], part);
            if (!found) v1 = v0 + share / PART_WAVES;
            found = found || next > target;
            if (!found && w + 1 < PART_WAVES) before = next, v0 = v1;
        }
    }
    u32 token = 0;
    float x = 0.f;
    if (!locate<DT>(r, weight, min(v0, r.nvec), min(r.nvec, v1), before, target, MARGIN * z, token, x)) return false;
    if ((threadIdx.x & 63) == 0) {
        d.token[row] = (int)token;
        d.ml2p[row] = value(x);
    }
    return true;
}

// the same by the definition, by the workgroup
template <int DT, int T, typename V>
__device__ __forceinline__ void put_exact(const Rows &a, const DrawArgs &d, u32 row, const char *p, float m, double u, const V &value) {
    u32 token;
    float x = m;
    if (draw_exact<DT, T>(p, a, Definition{d.t, (double)m}, u, token, x) && (threadIdx.x & 63) == 0) {
        d.token[row] = (int)token;
        d.ml2p[row] = value(x);
    }
}

// One workgroup a row, in 64 bits.  Its waves sum a share of it each, and the wave whose share holds the token looks at it again.
template <int DT>
__global__ __launch_bounds__(WIDE, 4) void k_logits_draw(Rows a, DrawArgs d) {
    __shared__ float pm[WIDE_WAVES];
    __shared__ double ps[WIDE_WAVES];
    __shared__ int done;
    const u32 row = block_id(), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (row >= a.rows) return;
    if (d.live && !d.live[row]) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_SKIP;
            d.ml2p[row] = 0.f;
        }
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, true);
    const double u = uniform_of(d, row);
    const u32 share = (r.nvec + WIDE_WAVES - 1) / WIDE_WAVES, v0 = min(wave * share, r.nvec), v1 = min(r.nvec, v0 + share);
    double s;
    float m;
    sum_vecs<DT, UNROLL>(r, d.power, v0, v1, lane, s, m);
    if (lane == 0) {
        pm[wave] = m;
        ps[wave] = s;
    }
    if (threadIdx.x == 0) done = 0;
    __syncthreads();
    m = group_all<WIDE_WAVES>(pm[lane & (WIDE_WAVES - 1)], Max());
    if (!drawable(m)) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_OUTSIDE;
            d.ml2p[row] = no_draw(m);
        }
        return;
    }
    const bool suits = good(m, d.power.c);
    const PowerBelow weight{d.power.c, suits ? 0. : (double)m};
    if (!suits) {
        float unused;
        sum_vecs<DT, UNROLL>(r, weight, v0, v1, lane, s, unused);
        if (lane == 0) ps[wave] = s;  // (nobody has read the first ones)
        __syncthreads();
    }
    const double part_sum = lane < WIDE_WAVES ? ps[lane] : 0., inc = group_scan<64>(part_sum), z = __shfl(inc, 63);
    const u64 passes = __ballot(inc > u * z);
    const Under64 value{z, weight.m, d.power.c};
    if (wave == (passes ? (u32)__ffsll((unsigned long long)passes) - 1 : 0u)) {
        const double none[PART_WAVES] = {};
        if (put_token<DT>(d, row, r, weight, part_sum, share, u, false, none, value)) done = 1;
    }
    __syncthreads();
    if (!done) put_exact<DT, WIDE>(a, d, row, p, m, u, value);
}

// One workgroup a row, in 32 bits first, the row in the registers of T lanes, HELD vectors each at most: what decides it is not
// loaded again (bf16, 16000 rows of 8192 tokens: 115 us when streamed, 70 held; 2600 of 50001: 95 and 84; 4096 of 32768: 80 and 75).  The
// waves' vectors lie behind each other.  (Of eight vectors a lane six waves a SIMD leave 4 to 8 registers to scratch, sixteen at
// four waves none; eight waves a SIMD spill more: 83 us for the last of these.)
template <int DT, int T, int HELD>
__global__ __launch_bounds__(T, HELD > 8 ? 4 : 6) void k_logits_draw_held(Rows a, DrawArgs d) {
    constexpr int WAVES = T / 64;
    __shared__ float pm[WAVES];
    __shared__ double ps[WAVES], under64[WAVES];  // (what the tokens score under: every wave's own copy, in no register meanwhile)
    __shared__ float2 under32[WAVES];
    __shared__ int done;
    const u32 row = block_id(), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (row >= a.rows) return;
    if (d.live && !d.live[row]) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_SKIP;
            d.ml2p[row] = 0.f;
        }
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, true);
    const u32 nv = (r.nvec + T - 1) / T, v0 = wave * nv * 64;
    raw4 q[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        q[i] = nothing<DT>();
        if (i < (int)nv) q[i] = load_vec<DT>(r, v0 + i * 64 + lane, r.nvec);
    }
    const double u = uniform_of(d, row);
    float m = threadIdx.x == 0 ? r.first : -INFINITY;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i < (int)nv) {
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) m = maximum(m, unpack<DT>(q[i], j));
        }
    }
    m = group_all<64>(m, Max());
    const auto sum_of = [&](const raw4 &v, const Expo &y_of) {
        float w[VEC<DT>];
#pragma unroll
        for (int j = 0; j < VEC<DT>; ++j) w[j] = exp2_(y_of.fast(unpack<DT>(v, j)));
        return pairs<VEC<DT>>(w);
    };
    float s[HELD];
    {
        const Expo y_of(Stat{m, 0.f, 0.f, false}, a.c);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            asm("" : "+v"(q[i]));  // (see forget)
            s[i] = i < (int)nv ? sum_of(q[i], y_of) : 0.f;
        }
        const float sum = pairs<HELD>(s) + (threadIdx.x == 0 ? exp2_(y_of.fast(r.first)) : 0.f);
        const double all = group_all<64>((double)sum, Add());  // (lanes and waves in 64 bits: a third fewer rows stay open)
        if (lane == 0) {
            pm[wave] = m;
            ps[wave] = all;
        }
    }
    if (threadIdx.x == 0) done = 0;
    __syncthreads();
    // as many lanes as there are waves hold the waves' sums, each under its own largest logit
    const u32 of = lane & (WAVES - 1);
    const float mine_m = m;
    m = group_all<WAVES>(pm[of], Max());
    if (!drawable(m)) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_OUTSIDE;
            d.ml2p[row] = no_draw(m);
        }
        return;
    }
    if (!doubtful(m, a.c)) {
        const Expo y_of(Stat{m, 0.f, 0.f, false}, a.c);
        const double w = __builtin_ldexp(ps[of], (int)(scaled(pm[of], a.c) - y_of.M)), inc = group_scan<WAVES>(w), z = __shfl(inc, WAVES - 1);
        const double target = u * z;
        if (lane == 0) under32[wave] = make_float2(log2_((float)z), y_of.M);
        const float near = (float)(d.margin * z);
        const u32 part = (u32)__popcll(__ballot(inc <= target) & ((1u << WAVES) - 1));
        if (wave == part) {
            u32 token = 0;
            float x = r.first;
            double run = __shfl(inc - w, part);
            bool here = false, sure = true;  // (here: the row's first element is it)
            if (wave == 0 && r.head) {
                run = exp2_(y_of.fast(r.first));
                here = run > target;
                sure = here ? lane == 0 && run - target >= (double)near : target - run >= (double)near;
            }
            if (!here && sure) {
                const float d2 = scaled(mine_m, a.c) - y_of.M;
                raw4 mq = q[0];
                float mine = 0.f;
                double start = run;
                u32 step = 0;
                bool found = false;
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    if (i < (int)nv) {
                        const float t = times2(s[i], d2);
                        const double upto = run + (double)group_all<64>(t, Add());
                        const bool now = !found && upto > target;
                        mine = now ? t : mine;
                        start = now ? run : start;
                        step = now ? i : step;
                        choose(mq, q[i], now);
                        found = found || now;
                        run = upto;
                    }
                }
                const float t = (float)(target - (start + (double)(group_scan<64>(mine) - mine)));
                sure = found && place_of<DT>(mq, y_of, t, near, r.head + (v0 + step * 64 + lane) * VEC<DT>, token, x);
            }
            if (sure) {
                d.token[row] = (int)token;
                d.ml2p[row] = Under32{log2_((float)z), y_of}(x);
                done = 1;
            }
        }
        __syncthreads();
        if (done) return;
    }
    // in 64 bits
    const PowerBelow weight{d.power.c, (double)m};
    double sum = threadIdx.x == 0 ? weight(r.first) : 0.;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        asm("" : "+v"(q[i]));
        if (i < (int)nv) {
#pragma unroll
            for (int j = 0; j < VEC<DT>; ++j) sum += weight(unpack<DT>(q[i], j));
        }
    }
    sum = group_all<64>(sum, Add());
    __syncthreads();  // (every wave has read the first ones)
    if (lane == 0) ps[wave] = sum;
    __syncthreads();
    const double part_sum = lane < (u32)WAVES ? ps[lane] : 0., inc = group_scan<64>(part_sum), z = __shfl(inc, 63);
    const u64 passes = __ballot(inc > u * z);
    if (lane == 0) under64[wave] = z;
    const auto value = [&](float x) {
        if (doubtful(m, a.c)) return Under64{under64[wave], (double)m, d.power.c}(x);
        Expo y_of(Stat{m, 0.f, 0.f, false}, a.c);
        y_of.M = under32[wave].y;
        return Under32{under32[wave].x, y_of}(x);
    };
    if (wave == (passes ? (u32)__ffsll((unsigned long long)passes) - 1 : 0u)) {
        const double none[PART_WAVES] = {};
        if (put_token<DT>(d, row, r, weight, part_sum, nv * 64, u, false, none, value)) done = 1;
    }
    __syncthreads();
    if (!done) put_exact<DT, T>(a, d, row, p, m, u, value);
}

// The parts of a row joined, by the workgroup's first wave; the others help where it leaves the token open.  (A row whose logits are
// too far from 0 for the parts' sums is summed again by that wave alone: 8 rows of 131072 tokens at T = 0.01 158 us, at T = 1 13.)
template <int DT>
__global__ __launch_bounds__(BLOCK) void k_logits_draw_join(Rows a, DrawArgs d, Split sp) {
    __shared__ int done;
    __shared__ double total;
    const u32 row = block_id(), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    if (d.live && !d.live[row]) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_SKIP;
            d.ml2p[row] = 0.f;
        }
        return;
    }
    const char *p = at(a.logits, a.inner, row);
    const Span r = span_of<DT>(a, p, true);
    const double u = uniform_of(d, row);
    double mine = 0., within[PART_WAVES] = {};
    float m = -INFINITY;
    if (lane < (1u << sp.shift)) {
        const u64 id = ((u64)row << sp.shift) + lane;
        m = sp.most[id];
#pragma unroll
        for (int w = 0; w < PART_WAVES; ++w) mine += within[w] = sp.sums[id * PART_WAVES + w];
    }
    m = group_all<64>(m, Max());
    if (!drawable(m)) {
        if (threadIdx.x == 0) {
            d.token[row] = MC_TOKEN_OUTSIDE;
            d.ml2p[row] = no_draw(m);
        }
        return;
    }
    const bool suits = good(m, d.power.c);
    const PowerBelow weight{d.power.c, suits ? 0. : (double)m};
    if (threadIdx.x < 64) {
        if (!suits) {
            float unused;
            sum_vecs<DT, UNROLL>(r, weight, 0, r.nvec, lane, mine, unused);
            if (lane) mine = 0.;
        }
        const double z = __shfl(group_scan<64>(mine), 63);
        const bool sure = put_token<DT>(d, row, r, weight, mine, suits ? sp.vecs : r.nvec, u, suits, within, Under64{z, weight.m, d.power.c});
        if (lane == 0) {
            done = sure;
            total = z;
        }
    }
    __syncthreads();
    if (!done) put_exact<DT, BLOCK>(a, d, row, p, m, u, Under64{total, weight.m, d.power.c});
}

// Rows begin with 64 bits where 32 would leave too many open: from 128 KB on (of 4-byte logits, which 64 bits keep up with: 2048
// rows of 41000 tokens 89 us, 120 from 32 bits on; 2048 of 20000 52 and 48) or 256 KB (1024 rows of 200000 tokens of two bytes 176 us,
// 210 from 32 bits on; 1024 of 90000 83 and 78).  Few rows do too: they wait for their loads, not for arithmetic, and an open
// row would be summed twice (511 rows of 30000 tokens 21 us, 512 from 32 bits on 26).  Few rows of more than 40000 tokens are cut
// into parts that still hold a chunk of 16 KB; a second launch costs 4 us, which shorter rows take less than.
bool few(u32 rows) { return rows < 512; }
bool in_64_bits(u32 rows, u32 dtype, u32 nvec) { return few(rows) || nvec > (dtype == MC_LOGITS_F32 ? 512u * 16 : 1024u * 16); }
u32 split_shift(u32 rows, u32 vocab, u32 nvec) {
    u32 shift = 0;
    while (few(rows) && vocab > 40000 && shift < 6 && ((u64)rows << shift) < 512 && (nvec >> (shift + 1)) >= BLOCK * UNROLL) ++shift;
    return shift;
}

size_t split_bytes(u32 rows, u32 shift) { return shift ? ((size_t)rows << shift) * (8 * PART_WAVES + 4) : 0; }

// How near u Z may come to an end of a token's interval, as a share of Z, before sums in 32 bits leave the token open, in half
// steps.  The weights: 2 for the power, 1.4 times its exponent for the exponent's two roundings, which the weights' mean
// makes at most log2 V + 1 (they weigh once: what is off in the running sum is off in Z too).  Rows of few tokens: of the
// additions behind each other, in Z and in the running sum 3 in a vector (in pairs), 8 steps, 6 over lanes; 8 in the last vector, 3
// where its parts are joined, 2 for the target.  Rows held by a workgroup: in Z 3 in a vector, 4 over a lane's (in pairs) and 1
// for the row's first element; in the running sum 3 and 6 over lanes, 8 in the last vector, 3 where its parts are joined.
double margin_of(const Rows &a) {
    const double sums = a.nvec <= SUB_VECS ? 2 * (3 + 8 + 6) + 8 + 3 + 2 : (3 + 4 + 1) + (3 + 6) + 8 + 3;
    return 0x1p-24 * (2 + 1.4 * (std::log2((double)a.vocab) + 1) + sums);
}

template <int DT>
void launch_wide(const Rows &a, const DrawArgs &d, hipStream_t s) {
    if (in_64_bits(a.rows, DT, a.nvec)) {
        hipLaunchKernelGGL((k_logits_draw<DT>), grid_of(a.rows), dim3(WIDE), 0, s, a, d);
        return;
    }
    // the fewest lanes that hold the row with six waves a SIMD, then with four
    if (a.nvec <= 256 * 8) hipLaunchKernelGGL((k_logits_draw_held<DT, 256, 8>), grid_of(a.rows), dim3(256), 0, s, a, d);
    else if (a.nvec <= 512 * 8) hipLaunchKernelGGL((k_logits_draw_held<DT, 512, 8>), grid_of(a.rows), dim3(512), 0, s, a, d);
    else if (DT == MC_LOGITS_F32 || a.nvec <= 512 * 16) hipLaunchKernelGGL((k_logits_draw_held<DT, 512, 16>), grid_of(a.rows), dim3(512), 0, s, a, d);
    else if constexpr (DT != MC_LOGITS_F32) hipLaunchKernelGGL((k_logits_draw_held<DT, 1024, 16>), grid_of(a.rows), dim3(1024), 0, s, a, d);
}

// ---- keys ----------------------------------------------------------------------------------------------------------
struct KeyArgs {
    const float *ml2p;
    const i64 *offsets;
    const void *lengths;
    u32 length_bytes;
    u64 count, longest;
    i64 stride;
    double *out;
};

// (not below 0, which rank indexes would put last: the caller's own values of certain tokens may be off by a rounding)
__device__ __forceinline__ double key_of(double sum) { return sum == INFINITY ? 1022.0 : sum <= 0. ? 0. : sum; }

// Password i's values p[0 .. n).  (Offsets that do not ascend or leave the array name none: nothing is read through them.)
__device__ __forceinline__ u64 values_of(const KeyArgs &k, u64 i, u64 &from) {
    from = 0;
    if (k.offsets) {
        const i64 lo = k.offsets[i], hi = k.offsets[i + 1];
        if (lo < 0 || hi <= lo || (u64)hi > k.longest) return 0;
        from = (u64)lo;
        return (u64)(hi - lo);
    }
    from = (u64)((i64)i * k.stride);
    const i64 n = k.length_bytes == 8 ? ((const i64 *)k.lengths)[i] : k.length_bytes == 4 ? (i64)((const int *)k.lengths)[i] : (i64)k.longest;
    return n < 0 ? 0 : (u64)n > k.longest ? k.longest : (u64)n;
}

// a group of G lanes a password
template <int G>
__global__ __launch_bounds__(BLOCK) void k_logits_keys(KeyArgs k) {
    const u32 lane = threadIdx.x & (G - 1);
    const u64 step = (u64)gridDim.x * (BLOCK / G);
    for (u64 first = (u64)blockIdx.x * (BLOCK / G); first < k.count; first += step) {
        const u64 i = first + threadIdx.x / G;
        u64 from = 0;
        const u64 n = i < k.count ? values_of(k, i, from) : 0;
        const float *p = k.ml2p + from;
        double s = 0.;
        for (u64 j = lane; j < n; j += G) s += (double)p[j];
        s = group_all<G>(s, Add());
        if (i < k.count && lane == 0) k.out[i] = key_of(s);
    }
}

// Packed passwords of a few symbols, one lane a password: the workgroup's values lie side by side and go through LDS (a
// lane that reads its own password's from memory touches a line of its own with every load: 71 us for 2e6 passwords of 12
// symbols).  What does not fit the window is read from memory.
constexpr u32 WINDOW = 4096;
typedef float float4_at4 __attribute__((ext_vector_type(4), aligned(4)));
__global__ __launch_bounds__(BLOCK) void k_logits_keys_packed(KeyArgs k) {
    __shared__ __attribute__((aligned(16))) float win[WINDOW];
    for (u64 first = (u64)blockIdx.x * BLOCK; first < k.count; first += (u64)gridDim.x * BLOCK) {
        const u64 last = min(first + BLOCK, k.count), i = first + threadIdx.x;
        const i64 lo = k.offsets[first], hi = k.offsets[last];
        u64 from = 0;
        const u64 m = i < k.count ? values_of(k, i, from) : 0;
        const u64 base = lo >= 0 && (u64)lo <= k.longest ? (u64)lo : 0;
        const u32 n = hi > (i64)base && (u64)hi <= k.longest ? (u32)min((u64)hi - base, (u64)WINDOW) : 0u;
#pragma unroll
        for (u32 u = 0; u < WINDOW / (4 * BLOCK); ++u) {
            const u32 j = (u * BLOCK + threadIdx.x) * 4;
            if (j + 4 <= n) {
                *(float4_at4 *)(win + j) = *(const float4_at4 *)(k.ml2p + base + j);
            } else {
                for (u32 t = j; t < n; ++t) win[t] = k.ml2p[base + t];
            }
        }
        __syncthreads();
        double s = 0.;
        if (from >= base && from + m <= base + n) {
            const float *p = win + (u32)(from - base);
#pragma unroll 4
            for (u32 j = 0; j < (u32)m; ++j) s += (double)p[j];
        } else {
            for (u64 j = 0; j < m; ++j) s += (double)k.ml2p[from + j];
        }
        if (i < k.count) k.out[i] = key_of(s);
        __syncthreads();
    }
}

}  // namespace

extern "C" size_t mc_logits_draw_workspace_bytes(uint32_t dtype, uint64_t rows, uint64_t vocab) {
    if (dtype > MC_LOGITS_BF16 || rows >= (1ull << 31) || vocab >= (1ull << 31)) return 0;
    const u64 per = dtype == MC_LOGITS_F32 ? 4 : 8;
    return split_bytes((u32)rows, split_shift((u32)rows, (u32)vocab, (u32)((vocab + per - 1) / per)));
}

extern "C" int mc_logits_draw(const void *logits, uint32_t dtype, uint64_t rows, uint64_t vocab, int64_t row_stride,
                              double temperature, const double *uniforms, uint64_t seed, uint64_t first_id, uint32_t draw,
                              const uint8_t *live, int32_t *out_token, float *out_ml2p, void *workspace, size_t workspace_bytes,
                              void *stream) {
    const char *who = "mc_logits_draw";
    Rows a{};
    if (int rc = rows_of(who, a, logits, dtype, 1, rows, vocab, 0, row_stride, temperature, true)) return rc;
    if (a.rows == 0) return MC_OK;
    if (!out_token || !out_ml2p) return bad(who, "no output");
    if (!aligned(uniforms, 8)) return bad(who, "uniforms that are not aligned to their type");
    if (!aligned(out_token, 4) || !aligned(out_ml2p, 4)) return bad(who, "outputs that are not aligned to their type");
    hipStream_t s = (hipStream_t)stream;
    const double c = LOG2E / temperature;
    DrawArgs d{uniforms, seed, first_id, draw, temperature, margin_of(a), Power{c, (float)(-1000. / c)}, live, out_token, out_ml2p};
    if (a.nvec <= SUB_VECS) {
        BY_TYPE(dtype, BY_GROUP(a, hipLaunchKernelGGL((k_logits_draw_sub<DT, G, NV>), grid_of(rows_to_blocks(a.rows, G)), dim3(BLOCK), 0, s, a, d)));
    } else {
        Split sp{split_shift(a.rows, a.vocab, a.nvec), 0, nullptr, nullptr};
        if (sp.shift) {
            if (!workspace || workspace_bytes < split_bytes(a.rows, sp.shift) || !aligned(workspace, 16)) {
                mc_set_error("%s: an aligned workspace of %zu bytes is needed, not %zu", who, split_bytes(a.rows, sp.shift), workspace_bytes);
                return MC_ERR_WORKSPACE;
            }
            const u32 each = (a.nvec + (1u << sp.shift) - 1) >> sp.shift;
            sp.vecs = (each + BLOCK - 1) / BLOCK * BLOCK;
            sp.sums = (double *)workspace;
            sp.most = (float *)(sp.sums + ((size_t)a.rows << sp.shift) * PART_WAVES);
            BY_TYPE(dtype, {
                hipLaunchKernelGGL((k_logits_draw_sums<DT>), grid_of(a.rows << sp.shift), dim3(BLOCK), 0, s, a, d, sp);
                hipLaunchKernelGGL((k_logits_draw_join<DT>), grid_of(a.rows), dim3(BLOCK), 0, s, a, d, sp);
            });
        } else {
            BY_TYPE(dtype, launch_wide<DT>(a, d, s));
        }
    }
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
    if (!aligned(ml2p, 4) || !aligned(offsets, 8) || !aligned(lengths, lengths ? length_bytes : 1) || !aligned(out_keys, 8))
        return bad(who, "values, offsets, lengths and keys are aligned to their types");
    const KeyArgs k{ml2p, (const i64 *)offsets, lengths, lengths ? length_bytes : 0u, (u64)count, (u64)longest, (i64)stride, out_keys};
    hipStream_t s = (hipStream_t)stream;
    const u64 usual = offsets ? longest / count : longest;  // symbols of a password, or as many as it may have
    const auto blocks = [&](u64 group) { return dim3((u32)std::min<u64>((count * group + BLOCK - 1) / BLOCK, 1u << 20)); };
    if (offsets && usual <= 64 && count >= 4096) hipLaunchKernelGGL(k_logits_keys_packed, blocks(1), dim3(BLOCK), 0, s, k);
    else if (usual <= 2) hipLaunchKernelGGL(k_logits_keys<1>, blocks(1), dim3(BLOCK), 0, s, k);
    else if (usual <= 8) hipLaunchKernelGGL(k_logits_keys<4>, blocks(4), dim3(BLOCK), 0, s, k);
    else if (usual <= 64) hipLaunchKernelGGL(k_logits_keys<16>, blocks(16), dim3(BLOCK), 0, s, k);
    else hipLaunchKernelGGL(k_logits_keys<64>, blocks(64), dim3(BLOCK), 0, s, k);
    HIP_TRY(hipGetLastError());
    return MC_OK;
}
