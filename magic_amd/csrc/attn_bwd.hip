// Segment attention, backward (magic_attn_bwd).  With D_i = do_i.o_i and p recomputed from lse:
//   dv = p^T do,  dl = p (do.v - D),  ds = scale dl (1 - (c / cap)^2),  dq = ds k,  dk = ds^T q,
//   dslope_h = -sum dl |pos_q - pos_k|.
// Two sweeps, so that every sum has one owner and a fixed order (no atomics): dq with the rows' wavefronts walking the
// keys (three products), dk and dv with the keys' wavefronts walking the rows of all heads that share them (four).
// Seven products instead of the five that one sweep with atomic adds would need.
// Bound like the forward pass.  Twelve graphs of 8,000 nodes, 4 heads of 64, float32: dq 4.33 ms (280 TFLOP/s of its three
// products), dk and dv 4.95 ms (328); bfloat16, 8 heads of 128 over 2, capped, half the keys masked: 1.65 ms (605) and
// 2.60 ms (512: 128 accumulators and both operands' rows leave one wavefront a SIMD, which has nothing to put beside its
// own waits).
#include "attn_common.h"

namespace {

using namespace magic::attn;
using magic::bf16_t;

struct BwdArgs {
    magic_attn a;
    const void *out, *dout;
    int64_t ld_o, hs_o, ld_do, hs_do;
    const double *lse;
    float *lse2;        // [q_heads][n_q] lse rounded down, +inf for rows that see no key (their probabilities become zeros)
    float *rest;        // [q_heads][n_q] 2^(lse2 - lse), what the rounding took: p = 2^(l log2 e - lse2) rest, rest <= 1
    float *delta;       // [q_heads][n_q]
    void *dq, *dk, *dv;
    double *slope_part; // [n_q tiles][q_heads] or NULL
    int64_t items;
    int sub;            // blocks that share a 128-row tile of the table
    bool hold;          // scaled launches: the forward pass's scores may be others (at_most)
    bool make_delta;    // the dq sweep forms lse2 and delta (no pass before it needs them)
    uint32_t sweep_blocks;   // of the dk / dv sweep; blocks behind them: d slope of one head each, from n_slope sums
    int64_t n_slope;
    float *dslopes;
    Prepared pr;
    int q_split;        // ranges of the keys a row tile's sums are cut into (1: they go straight to dq)
    float *part_q;      // [q_split][n_q][q_heads][head_dim]
    double *row_sums;   // [q_split][q_heads][n_q][3] of SlopeSums, where the slopes' gradient is wanted
    int n_split;        // shares of the rows a key tile's sums are cut into (1: they go straight to dk / dv)
    float *part;        // [n_split][dk | dv][n_k][kv_heads][head_dim]
};

// what the forward pass's rounding took from eight results
template <typename T> __device__ __forceinline__ void add_low(const magic_attn &a, int64_t row, int h, int c, float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        if (a.out_lo) {
            Raw<T> r;
            float y[8];
            r.load((const T *)a.out_lo + (row * a.q_heads + h) * a.head_dim + c);
            r.floats(y);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += y[e];
        }
    }
}

__device__ __forceinline__ float round_down(double x) {
    const float f = (float)x;
    if (!((double)f > x)) return f;
    return f > 0.f ? __uint_as_float(__float_as_uint(f) - 1u) : f < 0.f ? __uint_as_float(__float_as_uint(f) + 1u) : -0x1p-149f;
}
__device__ __forceinline__ float rest_of(double lse, float lse2) { return __builtin_amdgcn_exp2f((float)((double)lse2 - lse)); }

// lse2, rest and D of every row: DP / 8 lanes a row and head
template <typename T, int DP> __global__ __launch_bounds__(256) void k_attn_delta(BwdArgs b) {
    constexpr int LPR = DP / 8;
    const magic_attn &a = b.a;
    const int64_t total = a.n_q * a.q_heads;
    const int l = threadIdx.x % LPR, c = 8 * l;
    for (int64_t i = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR; i < total;
         i += (int64_t)gridDim.x * (256 / LPR)) {
        const int64_t row = i / a.q_heads;
        const int h = (int)(i - row * a.q_heads);
        float s = 0.f;
        if (c < a.head_dim) {
            float x[8], y[8];
            const T *o = (const T *)b.out + row * b.ld_o + h * b.hs_o + c, *d = (const T *)b.dout + row * b.ld_do + h * b.hs_do + c;
            Raw<T> ro, rd;
            ro.load(o), rd.load(d);
            ro.floats(x), rd.floats(y);
            add_low<T>(a, row, h, c, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) s += x[e] * y[e];
        }
#pragma unroll
        for (int k = LPR / 2; k > 0; k >>= 1) s += __shfl_xor(s, k, LPR);
        if (l == 0) {
            const double ls = b.lse[(int64_t)h * a.n_q + row];
            const bool none = ls == -INFINITY;
            const float lr = round_down(ls);
            b.lse2[(int64_t)h * a.n_q + row] = none ? INFINITY : lr;
            b.rest[(int64_t)h * a.n_q + row] = none ? 0.f : rest_of(ls, lr);
            b.delta[(int64_t)h * a.n_q + row] = none ? 0.f : s;
        }
    }
}

// Powers of two on the operands of a segment and head (1 unless the mode is scaled) and what undoes them
struct Scales {
    float q = 1.f, k = 1.f, v = 1.f, g = 1.f;
    float s_in, dp_in;
    // heads h .. h + n - 1, which share key head hk, take one kind and one scale
    template <typename M>
    __device__ __forceinline__ bool init(const Ranges &rg, int h, int n, int hk, int seg, const magic_attn &a) {
        if (rg.q) {
            const Range rk = rg.k[hk * rg.n_seg + seg], rv = rg.v[hk * rg.n_seg + seg];
            Range rq = {0u, 0xffffffffu}, rr = rq;
            for (int i = h; i < h + n; ++i) {
                const Range x = rg.q[i * rg.n_seg + seg], y = rg.g[i * rg.n_seg + seg];
                rq.max = max(rq.max, x.max), rq.min = min(rq.min, x.min);
                rr.max = max(rr.max, y.max), rr.min = min(rr.min, y.min);
            }
            if ((range_ok(rq) && range_ok(rk) && range_ok(rv) && range_ok(rr)) != rg.want_safe) return false;
            if constexpr (M::SCALED) q = range_scale(rq), k = range_scale(rk), v = range_scale(rv), g = range_scale(rr);
        }
        s_in = (a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E) * (1.f / q * (1.f / k));
        dp_in = 1.f / v * (1.f / g);
        return true;
    }
};

// Score gradients as operand planes.  In the scaled mode a lane (a column of the product's result) carries a power of
// two `u` that keeps its largest value so far at most 2^14 and its results in units of it; a larger value lowers u and
// the results with it.
struct Running {
    float u = 0.f;   // 0: nothing seen yet
    template <int DB> __device__ __forceinline__ void step(const float (&x)[16], f32x16_t (&acc)[DB]) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[e]));
        m = fmaxf(m, other_half(m));
        const bool grow = m > 0.f && (u == 0.f || m * u > 16384.f);
        if (__any(grow)) {
            int e = 13 + 127 - (int)(__float_as_uint(m) >> 23);                     // brings m to [2^13, 2^14)
            e = e > 120 ? 120 : e < -120 ? -120 : e;
            const float un = grow ? __uint_as_float((uint32_t)(e + 127) << 23) : u;
            const float f = u == 0.f ? 1.f : un / u;
            u = un;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        }
    }
    __device__ __forceinline__ float undo() const { return u == 0.f ? 0.f : 1.f / u; }
};

// d slope of head h: the tiles' sums, fixed tree (a block of up to four wavefronts)
__device__ __forceinline__ void sum_slope(const double *part, int64_t n, int H, int h, float *out, double *red) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += part[i * H + h];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < (int)blockDim.x / 64; ++w) s += red[w];
        out[h] = (float)s;
    }
}

// What a lane knows of its row in the dq sweep
struct RowSide {
    float s_in, dp_in, scale, f_cap, slope;   // f_cap: -scale / (cap log2 e)^2, for scale (1 - tanh^2) from the capped score
    uint32_t pos;
    float lse, delta;
};
// Of the lane's row: sum dl dist, sum dl, sum p dist.  The matrix instructions round their inner sums downwards by about
// 2^-27 of the terms; alike for all keys of a row, this changes no gradient but the slope's, where it meets the mean
// distance with one sign in every row (4e-5 of d slope over 97,000 rows).  sum dl, zero but for such an offset, takes it
// out again.  In double: long sums of both signs.
struct SlopeSums {
    double dl_dist = 0.0, dl = 0.0, pd = 0.0;
};

// No logit is above the row's log-sum.  A float32 one recomputed from other planes than the forward pass took can be (by 2^-22
// of its products' size): with logits of millions its probability would be no fp16 number.  HOLD takes it down to the sum
// (v_minimum3_f32: a NaN stays one) wherever the two passes' planes may differ; elsewhere the scores are the same bits, from
// one order of the products: 4 % of the sweep over the keys.
template <bool HOLD> __device__ __forceinline__ float at_most(float x, float top) {
    return HOLD ? __builtin_elementwise_minimum(x, top) : x;
}

// Scores and do.v of 32 keys by 32 rows -> gradients of the scores (before the scale of dq); km, kp: the keys' masks
// (0 / -inf) and positions, four for every group of registers
template <typename M, bool CAP, bool BIAS, bool MASK>
__device__ __forceinline__ void score_grad(f32x16_t &s, const f32x16_t &dp, const RowSide &c, const Cap<M::N == 1> &cap,
                                           const f32x4_t *km, const i32x4_t *kp, float (&ds)[16], SlopeSums &sums) {
#pragma clang fp contract(off)      // (a logit is rounded once, for its row's maximum and for its probability alike)
    if (CAP) cap_tile(s, cap);
    float t_dsl = 0.f, t_dl = 0.f, t_pd = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        f32x4_t base = {-c.lse, -c.lse, -c.lse, -c.lse};       // -inf for masked keys: their probabilities are zeros
        if (MASK) base += km[2 * g];
        i32x4_t pos;
        if (BIAS) pos = kp[2 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float x = CAP ? s[r] : s[r] * c.s_in, dist;
            const float f = CAP ? fmaf(x * x, c.f_cap, c.scale) : c.scale;
            if (BIAS) {
                dist = dist_of((uint32_t)pos[e], c.pos);
                x = fmaf(-c.slope, dist, x);
            }
            const float pr = __builtin_amdgcn_exp2f(at_most<(M::N > 1)>(x, c.lse) + base[e]);
            const float dl = pr * fmaf(dp[r], c.dp_in, -c.delta);
            if (BIAS) {
                t_dsl = fmaf(dl, dist, t_dsl);
                t_pd = fmaf(pr, dist, t_pd);
                t_dl += dl;
            }
            ds[r] = dl * f;
        }
    }
    if (BIAS) sums.dl_dist += (double)t_dsl, sums.dl += (double)t_dl, sums.pd += (double)t_pd;
}

// The same with the keys in the lanes: probabilities (times 2^14 in the scaled mode) and score gradients, both still without
// the row's `rest`; l, d: minus lse2 and minus D of the rows, qp their positions
template <typename M, bool HOLD, bool CAP, bool BIAS>
__device__ __forceinline__ void prob_grad(f32x16_t &s, const f32x16_t &dp, const RowSide &c, const Cap<M::N == 1> &cap,
                                          const f32x4_t *l, const f32x4_t *d, const i32x4_t *qp, float (&pr)[16], float (&ds)[16]) {
#pragma clang fp contract(off)      // (a logit is rounded once, for its row's maximum and for its probability alike)
    if (CAP) cap_tile(s, cap);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4_t l4 = l[2 * g], d4 = d[2 * g];
        i32x4_t pos;
        if (BIAS) pos = qp[2 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float x = CAP ? s[r] : s[r] * c.s_in;
            const float f = CAP ? fmaf(x * x, c.f_cap, c.scale) : c.scale;
            if (BIAS) x = fmaf(-c.slope, dist_of((uint32_t)pos[e], c.pos), x);
            const float q = __builtin_amdgcn_exp2f(at_most<HOLD>(x, -l4[e]) + l4[e]);
            pr[r] = M::SCALED ? q * 16384.f : q;
            ds[r] = q * fmaf(dp[r], c.dp_in, d4[e]) * f;
        }
    }
}


// WM groups of 32 rows, KG groups of 32 keys of a staged tile: a block of WM * KG wavefronts
template <typename M, int DP, int WM, int KG>
__global__ __launch_bounds__(64 * WM *KG, (DP == 128 && M::N > 1) || (DP >= 64 && KG > 1) ? 1 : 2) void k_attn_dq(BwdArgs p) {
    typedef typename M::T T;
    typedef typename M::vec vec;
    constexpr int NP = M::N, KS = DP / 16, DB = (DP + 31) / 32, BK = 32 * KG, NT = 64 * WM * KG;
    static_assert(KG == 1 || !M::SCALED, "the key groups' sums are joined in one unit");
    typedef Stage<M, DP, BK, NT> stage;
    typedef Tile<M, DP, BK> tile;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16_t *sK = reinterpret_cast<bf16_t *>(smem), *sV = sK + NP * tile::PLANE;
    uint32_t *sPos = reinterpret_cast<uint32_t *>(smem + 2 * tile::BYTES);
    float *sMask = reinterpret_cast<float *>(sPos + BK);

    const magic_attn &a = p.a;
    const int64_t item = xcd_item(blockIdx.x, 16);
    if (item >= p.items) return;
    const int D = a.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int wm = wave % WM, kg = wave / WM;
    const int64_t per_h = (int64_t)a.n_q_tiles * p.sub, tl = item % per_h;
    const int h = (int)(item / per_h % a.q_heads), hk = h / (a.q_heads / a.kv_heads), split = (int)(item / (per_h * a.q_heads));
    const int32_t *t = a.q_tiles + TAB * (tl / p.sub);
    const int first = (int)(tl % p.sub) * 32 * WM, nq = t[1] - first;      // this block's rows of the table's tile
    if (nq <= 0) {
        if (p.slope_part && p.q_split == 1 && tid == 0) p.slope_part[tl * a.q_heads + h] = 0.0;
        return;
    }
    const int64_t q0 = (int64_t)t[0] + first, k0 = t[2];
    const int nk = t[3] > 0 && p.pr.cnt ? p.pr.cnt[t[4]] : t[3];
    const int share = ((nk + BK - 1) / BK + p.q_split - 1) / p.q_split * BK;               // this block's keys
    const int j_beg = (int)min((int64_t)split * share, (int64_t)nk), j_end = min(j_beg + share, nk);
    const int row = wm * 32 + li;
    const bool ok = row < nq;
    const int64_t qr = q0 + (ok ? row : 0);
    const Src<M> K = src_of<M>(a.k, a.ld_k, a.hs_k, p.pr.k, k0, hk, D),
                 V = src_of<M>(a.v, a.ld_v, a.hs_v, p.pr.v, k0, hk, D);
    float ls = INFINITY, rest = 0.f, dl0 = 0.f;
    if (ok) {
        const int64_t at = (int64_t)h * a.n_q + qr;
        if (p.make_delta) {
            const double x = p.lse[at];
            if (x != -INFINITY) ls = round_down(x), rest = rest_of(x, ls);
        } else {
            ls = p.lse2[at], rest = p.rest[at], dl0 = p.delta[at];
        }
    }
    const bool live = ls != INFINITY;

    Scales sc;
    if (!sc.init<M>(p.pr.rg, h, 1, hk, t[4], a)) return;          // the other launch's segment
    vec qf[KS][NP], gf[KS][NP];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * hf, cc = c < D ? c : 0;
        Raw<T> r, g;
        r.load((const T *)a.q + qr * a.ld_q + h * a.hs_q + cc);
        g.load((const T *)p.dout + qr * p.ld_do + h * p.hs_do + cc);
        if (!live || c >= D) r.zero(), g.zero();      // (rows that see no key: nothing of them, NaN included)
        if (p.make_delta) {
            float x[8], y[8];
            Raw<T> o;
            o.load((const T *)p.out + qr * p.ld_o + h * p.hs_o + cc);
            if (!live || c >= D) o.zero();
            o.floats(x), g.floats(y);
            if (live && c < D) add_low<T>(a, qr, h, c, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) dl0 += x[e] * y[e];
        }
        r.planes(qf[ks], sc.q);
        g.planes(gf[ks], sc.g);
    }
    if (p.make_delta) {      // what the dk / dv sweep reads
        dl0 += other_half(dl0);
        if (ok && hf == 0 && kg == 0 && split == 0) {
            const int64_t at = (int64_t)h * a.n_q + qr;
            p.lse2[at] = ls, p.rest[at] = rest, p.delta[at] = dl0;
        }
    }
    const float dp_in = sc.dp_in * rest;         // `rest` once a row: score_grad's probabilities are without it
    dl0 *= rest;
    const bool bias = a.slopes != nullptr;
    const float slope = bias ? a.slopes[h] * LOG2E : 0.f;
    const uint32_t qpos = bias ? flip(a.q_pos[qr]) : 0u;
    const float f_cap = a.cap > 0.f ? -a.scale / a.cap / a.cap * (1.f / (LOG2E * LOG2E)) : 0.f;
    const Cap<M::N == 1> cap(sc.s_in, a.cap);
    Running run;
    SlopeSums sums;
    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

    uint32_t plain = tile::lane_plain(lane) + 64u * kg * tile::W, turned = tile::lane_turned(lane) + 64u * kg * tile::W;
    stage kst, vst;
    kst.init(K, D, tid), vst.init(V, D, tid);
    uint8_t keep[stage::N];
    int pos = 0;             // (taken as loaded: a use here would wait for the whole tile)
    uint8_t mk = 0;
    auto load = [&](int j0) {
        kst.load(K, j0, nk, D, tid);
        vst.load(V, j0, nk, D, tid);
#pragma unroll
        for (int i = 0; i < stage::N; ++i) {
            const int j = j0 + stage::row_of(i, tid);
            keep[i] = j < nk;
            if (!Src<M>::READY && a.key_mask && j < nk) keep[i] = a.key_mask[k0 + j];
        }
        if (tid < BK) {
            const int j = j0 + tid;
            const bool in = j < nk;
            mk = in && a.key_mask ? a.key_mask[k0 + j] : in;
            pos = bias && in ? a.k_pos[k0 + j] : 0;
        }
    };
    if (j_beg < j_end) load(j_beg);
    for (int j0 = j_beg; j0 < j_end; j0 += BK) {
        __syncthreads();
        const bool masked = a.key_mask != nullptr || j0 + BK > nk;
        kst.store(sK, D, tid, masked, [&](int i) { return keep[i] != 0; });
        vst.store(sV, D, tid, masked, [&](int i) { return keep[i] != 0; });
        if (tid < BK) sPos[tid] = flip(pos), sMask[tid] = mk ? 0.f : -INFINITY;
        __syncthreads();
        if (j0 + BK < j_end) load(j0 + BK);
        {
            const int b = kg;
            stay(plain), stay(turned);
            f32x16_t s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                vec f[NP], g[NP];
                tile::frag(sK, plain, 0, ks, f);
                tile::frag(sV, plain, 0, ks, g);
                mma(s, f, qf[ks]);
                mma(dp, g, gf[ks]);
            }
            feed<2 * NP, 2 * PRODUCTS<M>, KS>();
            float ds[16];
            const RowSide rs = {sc.s_in, dp_in, a.scale, f_cap, slope, qpos, ls, dl0};
            const f32x4_t *km = reinterpret_cast<const f32x4_t *>(sMask + 32 * b + 4 * hf);
            const i32x4_t *kp = reinterpret_cast<const i32x4_t *>(sPos + 32 * b + 4 * hf);
            if (a.cap > 0.f) {
                if (bias)
                    masked ? score_grad<M, true, true, true>(s, dp, rs, cap, km, kp, ds, sums) : score_grad<M, true, true, false>(s, dp, rs, cap, km, kp, ds, sums);
                else
                    masked ? score_grad<M, true, false, true>(s, dp, rs, cap, km, kp, ds, sums) : score_grad<M, true, false, false>(s, dp, rs, cap, km, kp, ds, sums);
            } else {
                if (bias)
                    masked ? score_grad<M, false, true, true>(s, dp, rs, cap, km, kp, ds, sums) : score_grad<M, false, true, false>(s, dp, rs, cap, km, kp, ds, sums);
                else
                    masked ? score_grad<M, false, false, true>(s, dp, rs, cap, km, kp, ds, sums) : score_grad<M, false, false, false>(s, dp, rs, cap, km, kp, ds, sums);
            }
            float u = 1.f;
            if constexpr (M::SCALED) {
                run.step<DB>(ds, acc);
                u = run.u;
            }
            // Few keys: dq is the difference of a few large terms, and what rounding takes from the score gradients does not
            // average out (2.5e-3 of the norm over four keys, 1.9e-3 with a second product of the low parts).  Narrow heads
            // (2.6e-3 at worst) take it always: their products are the smaller part of the work.  So do the blocks of 32 rows, which
            // wait more than they compute (3.0e-3 at worst).
            if constexpr (M::N == 1) {
                if (DP <= 32 || KG > 1 || nk <= 64) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = ds[8 * w + e] - (float)(bf16_t)ds[8 * w + e];
                        vec pf[NP];
                        to_planes(x, pf);
#pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            vec f[NP];
                            tile::frag_t(sK, turned, 16 * w, d, f);
                            mma(acc[d], f, pf);
                        }
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = M::SCALED ? ds[8 * w + e] * u : ds[8 * w + e];
                vec pf[NP];
                to_planes(x, pf);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    vec f[NP];
                    tile::frag_t(sK, turned, 16 * w, d, f);
                    mma(acc[d], f, pf);
                }
            }
            feed<2 * NP, PRODUCTS<M>, 2 * DB>();
        }
    }
    if constexpr (KG > 1) {      // the key groups' sums come together through LDS, in group order
        float *so = reinterpret_cast<float *>(smem);
        constexpr int OW = DB * 32 + 1;
#pragma unroll
        for (int g = KG - 1; g >= 1; --g) {
            __syncthreads();
            if (kg == g) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float *q = so + (wm * 32 + li) * OW + 32 * d + 8 * (r >> 2) + 4 * hf + (r & 3);
                        *q = g == KG - 1 ? acc[d][r] : *q + acc[d][r];
                    }
            }
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] += so[(wm * 32 + li) * OW + 32 * d + 8 * (r >> 2) + 4 * hf + (r & 3)];
        }
    }
    sums.pd *= (double)rest;
    const float undo = M::SCALED ? run.undo() * (1.f / sc.k) : 1.f;
    if (p.q_split > 1) {       // (one key group: k_attn_dq_join puts the ranges together)
        if (p.row_sums) {
            double *r = p.row_sums + (((int64_t)split * a.q_heads + h) * a.n_q + qr) * 3;
            const double x = sums.dl_dist + __shfl_xor(sums.dl_dist, 32, 64), y = sums.dl + __shfl_xor(sums.dl, 32, 64),
                         z = sums.pd + __shfl_xor(sums.pd, 32, 64);
            if (ok && hf == 0) r[0] = x, r[1] = y, r[2] = z;
        }
        if (!ok) return;
        float *o = p.part_q + (((int64_t)split * a.n_q + qr) * a.q_heads + h) * D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hf;
                if (c < D)
                    *reinterpret_cast<f32x4_t *>(o + c) =
                        f32x4_t{acc[d][4 * g] * undo, acc[d][4 * g + 1] * undo, acc[d][4 * g + 2] * undo, acc[d][4 * g + 3] * undo};
            }
        return;
    }
    if (ok && kg == 0) {
        T *o = (T *)p.dq + (qr * a.q_heads + h) * D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hf;
                const float x[4] = {acc[d][4 * g] * undo, acc[d][4 * g + 1] * undo, acc[d][4 * g + 2] * undo, acc[d][4 * g + 3] * undo};
                magic::store_vec<T, 4>(o + c, c < D, x);
            }
    }
    if (p.slope_part) {
        __syncthreads();
        double *red = reinterpret_cast<double *>(smem), *sdl = red + WM * KG;
        sdl[wave * 64 + lane] = sums.dl;
        __syncthreads();
        double all = 0.0;                    // sum dl of the lane's row: both halves, all key groups
#pragma unroll
        for (int g = 0; g < KG; ++g) all += sdl[(g * WM + wm) * 64 + li] + sdl[(g * WM + wm) * 64 + li + 32];
        double dsl = all * sums.pd - sums.dl_dist;          // (with this lane's share of sum p dist)
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) dsl += __shfl_xor(dsl, k, 64);
        if (lane == 0) red[wave] = dsl;
        __syncthreads();
        if (tid == 0) {
            double x = 0.0;
#pragma unroll
            for (int w = 0; w < WM * KG; ++w) x += red[w];
            p.slope_part[tl * a.q_heads + h] = x;
        }
    }
}

// dq from the ranges of the keys, in order.  The blocks behind `join_blocks`: the slopes' sums of 256 rows of a head each.
template <typename T> __global__ __launch_bounds__(256) void k_attn_dq_join(BwdArgs p, int join_blocks, int row_blocks) {
    const magic_attn &a = p.a;
    if ((int)blockIdx.x >= join_blocks) {
        __shared__ double red[4];
        const int h = ((int)blockIdx.x - join_blocks) / row_blocks, b = ((int)blockIdx.x - join_blocks) % row_blocks;
        const int64_t row = (int64_t)b * 256 + threadIdx.x;
        double x = 0.0, y = 0.0, z = 0.0;
        if (row < a.n_q)
            for (int s = 0; s < p.q_split; ++s) {
                const double *r = p.row_sums + (((int64_t)s * a.q_heads + h) * a.n_q + row) * 3;
                x += r[0], y += r[1], z += r[2];
            }
        double dsl = y * z - x;
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) dsl += __shfl_xor(dsl, k, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dsl;
        __syncthreads();
        if (threadIdx.x == 0) p.slope_part[(int64_t)b * a.q_heads + h] = red[0] + red[1] + red[2] + red[3];
        return;
    }
    const int64_t plane = a.n_q * a.q_heads * a.head_dim, n4 = plane / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)join_blocks * 256) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.q_split; ++s) x += *reinterpret_cast<const f32x4_t *>(p.part_q + s * plane + 4 * i);
        const float y[4] = {x[0], x[1], x[2], x[3]};
        magic::store_vec<T, 4>((T *)p.dq + 4 * i, true, y);
    }
}

// WM groups of 32 keys, KG groups of 32 NB rows of a staged tile.  The blocks behind the sweep's add up the slopes' sums.
template <typename M, int DP, int WM, int KG, int NB, bool HOLD>
__global__ __launch_bounds__(64 * WM *KG, DP == 128 || (DP >= 64 && KG > 1) ? 1 : 2) void k_attn_dkv(BwdArgs p) {
    typedef typename M::T T;
    typedef typename M::vec vec;
    constexpr int NP = M::N, KS = DP / 16, DB = (DP + 31) / 32, BQ = 32 * KG * NB, NT = 64 * WM * KG;
    static_assert(KG == 1 || !M::SCALED, "the row groups' sums are joined in one unit");
    typedef Stage<M, DP, BQ, NT> stage;
    typedef Tile<M, DP, BQ> tile;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16_t *sQ = reinterpret_cast<bf16_t *>(smem), *sG = sQ + NP * tile::PLANE;
    float *sL = reinterpret_cast<float *>(smem + 2 * tile::BYTES), *sD = sL + BQ, *sZ = sD + BQ;
    uint32_t *sPos = reinterpret_cast<uint32_t *>(sZ + BQ);
    int *sFar = reinterpret_cast<int *>(sPos + BQ);

    const magic_attn &a = p.a;
    if (blockIdx.x >= p.sweep_blocks) {
        sum_slope(p.slope_part, p.n_slope, a.q_heads, blockIdx.x - p.sweep_blocks, p.dslopes, reinterpret_cast<double *>(smem));
        return;
    }
    const int64_t item = xcd_item(blockIdx.x, 16);
    if (item >= p.items) return;
    const int D = a.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int wm = wave % WM, kg = wave / WM;
    const int64_t tiles = (int64_t)a.n_k_tiles * p.sub, tl = item % tiles;
    const int hk = (int)(item / tiles % a.kv_heads), G = a.q_heads / a.kv_heads;
    const int split = (int)(item / (tiles * a.kv_heads));
    const int32_t *t = a.k_tiles + TAB * (tl / p.sub);
    const int first = (int)(tl % p.sub) * 32 * WM;                         // this block's keys of the table's tile
    const int64_t k0 = (int64_t)t[0] + first, q0 = t[2];
    const int nk = (p.pr.cnt ? min(t[1], p.pr.cnt[t[4]] - (t[0] - t[5])) : t[1]) - first, nq = t[3];
    if (nk <= 0) return;                     // (all unmasked keys of the segment are in the tiles before)
    const int col = wm * 32 + li;
    const bool in = col < nk;
    const int64_t kr = p.pr.idx ? p.pr.idx[k0 + (in ? col : 0)] : k0 + (in ? col : 0);
    const bool ok = in && (p.pr.idx || !a.key_mask || a.key_mask[kr]);

    Scales sc;
    if (!sc.init<M>(p.pr.rg, hk * G, G, hk, t[4], a)) return;  // the other launch's segment
    vec kf[KS][NP], vf[KS][NP];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * hf, cc = c < D ? c : 0;
        Raw<T> r, g;
        r.load((const T *)a.k + kr * a.ld_k + hk * a.hs_k + cc);
        g.load((const T *)a.v + kr * a.ld_v + hk * a.hs_v + cc);
        if (!ok || c >= D) r.zero(), g.zero();
        r.planes(kf[ks], sc.k);
        g.planes(vf[ks], sc.v);
    }
    const bool bias = a.slopes != nullptr;
    const uint32_t kpos = bias ? flip(a.k_pos[kr]) : 0u;
    const float f_cap = a.cap > 0.f ? -a.scale / a.cap / a.cap * (1.f / (LOG2E * LOG2E)) : 0.f;
    // Without `rest` a row's probabilities are off by up to |lse2| 2^-23: up to this size it is left out.  (The scaled mode has
    // it in the rows of the gradient.)
    constexpr float FAR = M::N == 1 ? 256.f : 1.f;
    const Cap<M::N == 1> cap(sc.s_in, a.cap);
    Running run;
    f32x16_t gk[DB], gv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) gk[d][r] = 0.f, gv[d][r] = 0.f;

    uint32_t plain = tile::lane_plain(lane), turned = tile::lane_turned(lane);
    stage qst, gst;
    qst.init(src_of<M>(a.q, a.ld_q, a.hs_q, p.pr.q, q0, 0, D), D, tid);
    gst.init(src_of<M>(p.dout, p.ld_do, p.hs_do, p.pr.g, q0, 0, D), D, tid);
    int staged = 0;          // rows of the segment behind the staged tile's first
    float ls = 0.f, rest = 0.f, dl0 = 0.f;
    int pos = 0;             // (all taken as loaded: a use here would wait for the whole tile)
    auto load = [&](int h, int i0) {
        qst.load(src_of<M>(a.q, a.ld_q, a.hs_q, p.pr.q, q0, h, D), i0, nq, D, tid);
        gst.load(src_of<M>(p.dout, p.ld_do, p.hs_do, p.pr.g, q0, h, D), i0, nq, D, tid);
        const int64_t at = (int64_t)h * a.n_q + q0;
        staged = nq - i0;
        if (tid < BQ) {
            const int r = i0 + tid;
            ls = r < nq ? p.lse2[at + r] : INFINITY;
            rest = r < nq ? p.rest[at + r] : 0.f;
            dl0 = r < nq ? p.delta[at + r] : 0.f;
            pos = bias && r < nq ? a.q_pos[q0 + r] : 0;
        }
    };
    // this block's share of the steps (heads that share the key head, tiles of their rows)
    const int per_h = (nq + BQ - 1) / BQ, steps = per_h * G, share = (steps + p.n_split - 1) / p.n_split;
    const int s_beg = min(split * share, steps), s_end = min(s_beg + share, steps);
    int h = hk * G + (per_h > 0 ? s_beg / per_h : 0), it = per_h > 0 ? s_beg % per_h : 0;
    if (s_beg < s_end) load(h, it * BQ);
    for (int st = s_beg; st < s_end; ++st) {
        __syncthreads();
        // (a row that sees no key belongs to a segment without any: its dk and dv are written as zeros whatever it holds)
        const bool part = staged < BQ;
        const int rows = staged;
        qst.store(sQ, D, tid, part, [&](int i) { return stage::row_of(i, tid) < rows; });
        gst.store(sG, D, tid, part, [&](int i) { return stage::row_of(i, tid) < rows; });
        if (tid < BQ) {
            sL[tid] = -ls, sZ[tid] = rest, sD[tid] = M::SCALED ? -dl0 * rest : -dl0, sPos[tid] = flip(pos);
            const bool far = __any(fabsf(ls) > FAR && ls != INFINITY);
            if (lane == 0) sFar[wave] = far;
        }
        const float slope = bias ? a.slopes[h] * LOG2E : 0.f;
        __syncthreads();
        int far = M::SCALED ? 0 : sFar[0];
        if (!M::SCALED && BQ > 64) far |= sFar[1];
        far = __builtin_amdgcn_readfirstlane(far);
        if (++it == per_h) it = 0, ++h;
        if (st + 1 < s_end) load(h, it * BQ);
#pragma unroll 1
        for (int nb = 0; nb < NB; ++nb) {
            const int b = kg * NB + nb;
            stay(plain), stay(turned);
            f32x16_t s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                vec f[NP], g[NP];
                tile::frag(sQ, plain, 32 * b, ks, f);
                tile::frag(sG, plain, 32 * b, ks, g);
                mma_turned(s, f, kf[ks]);
                mma(dp, g, vf[ks]);
            }
            feed<2 * NP, 2 * PRODUCTS<M>, KS>();
            float pr[16], ds[16];
            const RowSide ks = {sc.s_in, sc.dp_in, a.scale, f_cap, slope, kpos, 0.f, 0.f};
            const f32x4_t *l4 = reinterpret_cast<const f32x4_t *>(sL + 32 * b + 4 * hf);
            const f32x4_t *d4 = reinterpret_cast<const f32x4_t *>(sD + 32 * b + 4 * hf);
            const i32x4_t *qp = reinterpret_cast<const i32x4_t *>(sPos + 32 * b + 4 * hf);
            if (a.cap > 0.f)
                bias ? prob_grad<M, HOLD, true, true>(s, dp, ks, cap, l4, d4, qp, pr, ds) : prob_grad<M, HOLD, true, false>(s, dp, ks, cap, l4, d4, qp, pr, ds);
            else
                bias ? prob_grad<M, HOLD, false, true>(s, dp, ks, cap, l4, d4, qp, pr, ds) : prob_grad<M, HOLD, false, false>(s, dp, ks, cap, l4, d4, qp, pr, ds);
            if (!M::SCALED && far) {
                const f32x4_t *z4 = reinterpret_cast<const f32x4_t *>(sZ + 32 * b + 4 * hf);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4_t z = z4[2 * g];
#pragma unroll
                    for (int e = 0; e < 4; ++e) pr[4 * g + e] *= z[e], ds[4 * g + e] *= z[e];
                }
            }
            float u = 1.f;
            if constexpr (M::SCALED) {
                run.step<DB>(ds, gk);
                u = run.u;
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float x[8], y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = pr[8 * w + e], y[e] = M::SCALED ? ds[8 * w + e] * u : ds[8 * w + e];
                vec pf[NP], sf[NP];
                to_planes(x, pf);
                to_planes(y, sf);
                constexpr bool LOW = M::N == 1 && (DP <= 32 || KG > 1);      // low parts too, as in the dq sweep
                vec pl[NP], sl[NP];
                if constexpr (LOW) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] -= (float)(bf16_t)x[e], y[e] -= (float)(bf16_t)y[e];
                    to_planes(x, pl);
                    to_planes(y, sl);
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    vec f[NP];
                    tile::frag_t(sG, turned, 32 * b + 16 * w, d, f);
                    mma(gv[d], f, pf);
                    if constexpr (LOW) mma(gv[d], f, pl);
                    tile::frag_t(sQ, turned, 32 * b + 16 * w, d, f);
                    mma(gk[d], f, sf);
                    if constexpr (LOW) mma(gk[d], f, sl);
                }
            }
            feed<2 * NP, PRODUCTS<M>, 4 * DB>();
        }
    }
    if constexpr (KG > 1) {      // the row groups' sums come together through LDS, in group order
        float *so = reinterpret_cast<float *>(smem);
        constexpr int OW = 2 * DB * 32 + 1;
#pragma unroll
        for (int g = KG - 1; g >= 0; --g) {
            __syncthreads();
            if (kg == g) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float *q = so + (wm * 32 + li) * OW + 64 * d + 8 * (r >> 2) + 4 * hf + (r & 3);
                        if (g < KG - 1) gk[d][r] += q[0], gv[d][r] += q[32];
                        if (g > 0) q[0] = gk[d][r], q[32] = gv[d][r];
                    }
            }
        }
        if (kg != 0) return;
    }
    if (!in) return;
    const float uk = M::SCALED ? run.undo() * (1.f / sc.q) : 1.f, uv = M::SCALED ? 1.f / 16384.f * (1.f / sc.g) : 1.f;
    const int64_t at = (kr * a.kv_heads + hk) * D;
    if (p.n_split > 1) {
        float *pk = p.part + (int64_t)split * 2 * a.n_k * a.kv_heads * D + at, *pv = pk + a.n_k * a.kv_heads * D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hf;
                if (c < D) {
                    f32x4_t x, y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = ok ? gk[d][4 * g + e] * uk : 0.f, y[e] = ok ? gv[d][4 * g + e] * uv : 0.f;
                    *reinterpret_cast<f32x4_t *>(pk + c) = x;
                    *reinterpret_cast<f32x4_t *>(pv + c) = y;
                }
            }
        return;
    }
    T *o_k = (T *)p.dk + at, *o_v = (T *)p.dv + at;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hf;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = ok ? gk[d][4 * g + e] * uk : 0.f, y[e] = ok ? gv[d][4 * g + e] * uv : 0.f;
            magic::store_vec<T, 4>(o_k + c, c < D, x);
            magic::store_vec<T, 4>(o_v + c, c < D, y);
        }
}

// dk and dv from the shares of the rows, in order
template <typename T> __global__ __launch_bounds__(256) void k_attn_dkv_join(BwdArgs p) {
    const int64_t plane = p.a.n_k * p.a.kv_heads * p.a.head_dim, n4 = 2 * plane / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
        // (masked keys: nothing was written for them)
        const int64_t row = (4 * i < plane ? 4 * i : 4 * i - plane) / ((int64_t)p.a.kv_heads * p.a.head_dim);
        if (!p.a.key_mask || p.a.key_mask[row])
        for (int s = 0; s < p.n_split; ++s) x += *reinterpret_cast<const f32x4_t *>(p.part + s * 2 * plane + 4 * i);
        const float y[4] = {x[0], x[1], x[2], x[3]};
        const int64_t e = 4 * i;
        magic::store_vec<T, 4>(e < plane ? (T *)p.dk + e : (T *)p.dv + (e - plane), true, y);
    }
}

// zeros for the masked keys, which no tile of gathered keys holds
template <typename T> __global__ __launch_bounds__(256) void k_attn_dkv_masked(BwdArgs p) {
    const int cpr = p.a.kv_heads * p.a.head_dim / 8;
    const int64_t total = p.a.n_k * cpr;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        if (p.a.key_mask[i / cpr]) continue;
        Raw<T> z;
        z.zero();
        z.store((T *)p.dk + 8 * i);
        z.store((T *)p.dv + 8 * i);
    }
}

// d slope of a head where no dk / dv sweep runs
__global__ __launch_bounds__(256) void k_attn_dslope(const double *part, int64_t n, int H, float *out) {
    __shared__ double red[4];
    sum_slope(part, n, H, blockIdx.x, out, red);
}

template <typename M, int DP, int WM, int KG> int run_dq(BwdArgs &b, hipStream_t st) {
    size_t lds = 2 * Tile<M, DP, 32 * KG>::BYTES + 32 * KG * 8;
    const size_t sums = (size_t)WM * KG * 65 * 8, join = (size_t)32 * WM * ((DP + 31) / 32 * 32 + 1) * 4;
    if (lds < sums) lds = sums;
    if (KG > 1 && lds < join) lds = join;
    if (magic::ensure_dynamic_lds((const void *)k_attn_dq<M, DP, WM, KG>, lds) != MAGIC_OK) return MAGIC_ERR_RUNTIME;
    b.items = (int64_t)b.a.n_q_tiles * b.sub * b.a.q_heads * b.q_split;
    if (xcd_grid(b.items, 16) > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
    MAGIC_LAUNCH(M::SCALED ? "attn_bwd_dq_f16x2" : "attn_bwd_dq", (k_attn_dq<M, DP, WM, KG>), (int)xcd_grid(b.items, 16),
                 64 * WM * KG, lds, st, b);
    return magic::launch_status();
}

template <typename M, int DP, int WM, int KG, int NB, bool HOLD = (M::N > 1)> int run_dkv(BwdArgs &b, int slope_heads, hipStream_t st) {
    constexpr int BQ = 32 * KG * NB;
    size_t lds = 2 * Tile<M, DP, BQ>::BYTES + BQ * 16 + 8;
    const size_t join = (size_t)32 * WM * (2 * ((DP + 31) / 32 * 32) + 1) * 4;
    if (KG > 1 && lds < join) lds = join;
    if (magic::ensure_dynamic_lds((const void *)k_attn_dkv<M, DP, WM, KG, NB, HOLD>, lds) != MAGIC_OK) return MAGIC_ERR_RUNTIME;
    b.items = (int64_t)b.a.n_k_tiles * b.sub * b.a.kv_heads * b.n_split;
    const int64_t grid = xcd_grid(b.items, 16);
    if (grid + slope_heads > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
    b.sweep_blocks = (uint32_t)grid;
    MAGIC_LAUNCH(M::SCALED ? "attn_bwd_dkv_f16x2" : "attn_bwd_dkv", (k_attn_dkv<M, DP, WM, KG, NB, HOLD>), (int)grid + slope_heads,
                 64 * WM * KG, lds, st, b);
    return magic::launch_status();
}

// 32 rows a block where tiles of 128 would leave most of the chip idle: the wavefronts share the rows and deal out the keys
// Heads of more than 32 columns leave a CU room for one such block: one round of them at most.  Four heads, us of both
// sweeps, 32 rows against 128: 64 wide, bfloat16, graphs of 500 nodes, 64 tiles 34 / 48, 80 tiles 52 / 48, one graph of 7,000
// (220) 499 / 367; float32, 64 tiles 59 / 111, forty graphs of 100 (160) 72 / 47; 128 wide, float32, 64 tiles 160 / 174, 80
// tiles 301 / 176.  16 wide: one graph of 7,000 503 / 570 in float32 and 216 / 279 in bfloat16, a hundred graphs of 100
// (400 tiles) 33 / 23.
bool small_side(const magic_attn &a, int64_t blocks) { return blocks <= (a.head_dim <= 32 ? 255 : 64); }

int sub_tiles(const magic_attn &a, int64_t tiles, int heads, int longest) {
    if (!small_side(a, tiles * heads)) return 1;
    const int rows = longest < MAGIC_ATTN_TILE ? longest : MAGIC_ATTN_TILE;
    return rows > 32 ? (rows + 31) / 32 : 1;
}

template <typename M, int DP> int sweeps(BwdArgs &b, bool last, hipStream_t st) {
    const magic_attn full = b.a;
    constexpr int KG = DP == 128 && M::N == 3 ? 2 : 4;      // (three planes of 128 rows and columns would not fit the LDS)
    int rc = MAGIC_OK;
    if (full.n_q > 0 && b.dq) {
        b.a = gathered(&full, b.pr);
        b.sub = sub_tiles(full, full.n_q_tiles, full.q_heads, full.max_q);
        if constexpr (M::SCALED) {
            b.sub = 1;
            rc = run_dq<M, DP, 4, 1>(b, st);
        } else {
            const bool few = b.q_split == 1 && !b.pr.rg.q && small_side(full, (int64_t)full.n_q_tiles * full.q_heads);
            if (!few) b.sub = 1;
            rc = few ? run_dq<M, DP, 1, KG>(b, st) : run_dq<M, DP, 4, 1>(b, st);
        }
        b.n_slope = (int64_t)full.n_q_tiles * b.sub;
        if (rc == MAGIC_OK && last && b.q_split > 1) {
            const int join = magic::stride_grid(full.n_q * full.q_heads * full.head_dim / 4, 256);
            const int rows = b.row_sums ? (int)((full.n_q + 255) / 256) : 0;
            b.n_slope = rows;
            MAGIC_LAUNCH("attn_dq_join", k_attn_dq_join<typename M::T>, join + rows * full.q_heads, 256, 0, st, b, join, rows);
            rc = magic::launch_status();
        }
    }
    b.a = full;                    // (a key's own rows are read where they are)
    if (rc == MAGIC_OK && full.n_k > 0 && b.dk) {
        const int slopes = last && b.slope_part ? full.q_heads : 0;
        b.sub = 1;
        constexpr int NB = DP == 128 && M::N == 1 ? 2 : 1;  // (one more block of rows a step where registers allow it)
        if constexpr (M::SCALED) {
            rc = b.hold ? run_dkv<M, DP, 4, 1, NB, true>(b, slopes, st) : run_dkv<M, DP, 4, 1, NB, false>(b, slopes, st);
        } else {
            const bool few = !b.pr.rg.q && b.n_split == 1 && small_side(full, (int64_t)full.n_k_tiles * full.kv_heads);
            if (few) b.sub = sub_tiles(full, full.n_k_tiles, full.kv_heads, full.max_k);
            rc = few ? run_dkv<M, DP, 1, KG, 1>(b, slopes, st) : run_dkv<M, DP, 4, 1, NB>(b, slopes, st);
        }
    }
    return rc;
}

template <typename M> int sweeps_of(BwdArgs &b, bool last, hipStream_t st) {
    const int D = b.a.head_dim;
    return D <= 16   ? sweeps<M, 16>(b, last, st)
           : D <= 32 ? sweeps<M, 32>(b, last, st)
           : D <= 64 ? sweeps<M, 64>(b, last, st)
                     : sweeps<M, 128>(b, last, st);
}

template <typename T, int DP> int delta(BwdArgs &b, hipStream_t st) {
    const int grid = magic::stride_grid(b.a.n_q * b.a.q_heads, 256 / (DP / 8));
    MAGIC_LAUNCH("attn_bwd_delta", (k_attn_delta<T, DP>), grid, 256, 0, st, b);
    return magic::launch_status();
}
template <typename T> int delta_of(BwdArgs &b, hipStream_t st) {
    const int D = b.a.head_dim;
    return D <= 16 ? delta<T, 16>(b, st) : D <= 32 ? delta<T, 32>(b, st) : D <= 64 ? delta<T, 64>(b, st) : delta<T, 128>(b, st);
}

// Ranges of the keys a row tile is cut into: as below; short calls take 32-row blocks instead.
// One graph, 4 heads of 64, whole against cut: 4,000 nodes 232 / 115 us in float32 and 144 / 75 in bfloat16, 12,000 nodes
// 951 / 815 and 549 / 460 (with the pass that joins them).
int q_splits(const magic_attn *a) {
    const int64_t blocks = (int64_t)a->n_q_tiles * a->q_heads;
    if (blocks <= 0 || (!use_f16(a) && small_side(*a, blocks))) return 1;
    int64_t s = (1536 + blocks - 1) / blocks;
    const int64_t most = ((int64_t)a->max_k + 511) / 512;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

// shares of the rows a key tile is cut into: enough blocks to fill the chip three times over (segments of very different
// lengths leave long ones running alone otherwise), at least 512 (head, row) steps each
int splits(const magic_attn *a) {
    const int64_t blocks = (int64_t)a->n_k_tiles * a->kv_heads;
    if (blocks <= 0) return 1;
    int64_t s = (1536 + blocks - 1) / blocks;
    const int64_t most = ((int64_t)a->max_q * (a->q_heads / a->kv_heads) + 511) / 512;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

}  // namespace

extern "C" {

size_t magic_attn_bwd_workspace_bytes(const magic_attn *a) {
    if (check(a) != MAGIC_OK) return 256;
    const int n = splits(a);
    const size_t part = n > 1 ? (size_t)n * 2 * a->n_k * a->kv_heads * a->head_dim * sizeof(float) : 0;
    const int m = q_splits(a);
    const size_t rows = m > 1 ? (size_t)m * a->n_q * a->q_heads : 0;
    return magic::align_up(part) + magic::align_up(rows * a->head_dim * sizeof(float)) + magic::align_up(rows * 3 * sizeof(double)) + prepare_bytes(a, use_f16(a), true) + 3 * magic::align_up((size_t)a->n_q * a->q_heads * sizeof(float)) +
           magic::align_up((size_t)a->n_q_tiles * 4 * a->q_heads * sizeof(double)) + 256;
}

int magic_attn_bwd(const magic_attn *a, const void *out, int64_t ld_out, int64_t hs_out, const double *lse, const void *d_out,
                   int64_t ld_do, int64_t hs_do, void *dq, void *dk, void *dv, float *d_slopes, void *workspace,
                   size_t workspace_bytes, void *stream_) {
    const int st = check(a);
    if (st != MAGIC_OK) return st;
    hipStream_t stream = (hipStream_t)stream_;
    if (a->n_q > 0 && (!out || !lse || !d_out || (d_slopes && !dq))) return MAGIC_ERR_INVALID_ARG;
    if (!dk != !dv) return MAGIC_ERR_INVALID_ARG;
    if (d_slopes && !a->slopes) return MAGIC_ERR_INVALID_ARG;
    const int per = a->dtype == MAGIC_F32 ? 4 : 8;
    if (((uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) return MAGIC_ERR_INVALID_ARG;
    if (ld_do > MAX_LD) return MAGIC_ERR_UNSUPPORTED;
    if (ld_out < 0 || hs_out < 0 || ld_do < 0 || hs_do < 0 || (ld_out | hs_out | ld_do | hs_do) % per) return MAGIC_ERR_INVALID_ARG;
    BwdArgs b;
    b.a = *a;
    b.out = out, b.dout = d_out, b.ld_o = ld_out, b.hs_o = hs_out, b.ld_do = ld_do, b.hs_do = hs_do;
    b.lse = lse, b.dq = dq, b.dk = dk, b.dv = dv, b.dslopes = d_slopes;
    b.n_slope = 0, b.sub = 1, b.sweep_blocks = 0;
    magic::Arena ar(workspace, workspace_bytes);
    b.delta = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.lse2 = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.rest = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.slope_part = ar.take<double>((size_t)a->n_q_tiles * 4 * a->q_heads);
    const bool f16 = use_f16(a) && a->n_q > 0 && a->n_k > 0;
    b.n_split = dk ? splits(a) : 1;
    b.part = b.n_split > 1 ? ar.take<float>((size_t)b.n_split * 2 * a->n_k * a->kv_heads * a->head_dim) : nullptr;
    b.q_split = dq ? q_splits(a) : 1;
    const size_t q_rows = (size_t)b.q_split * a->n_q * a->q_heads;
    b.part_q = b.q_split > 1 ? ar.take<float>(q_rows * a->head_dim) : nullptr;
    b.row_sums = b.q_split > 1 && d_slopes ? ar.take<double>(q_rows * 3) : nullptr;
    if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
    if (!d_slopes) b.slope_part = nullptr;
    const bool f32 = a->dtype == MAGIC_F32;
    int rc = MAGIC_OK;
    b.hold = !fwd_scores_f16(a);
    b.make_delta = dq && !f16;      // (the planes of the scaled launches are zero where lse2 says so: they need it before)
    if (a->n_q > 0 && !b.make_delta) rc = f32 ? delta_of<float>(b, stream) : delta_of<bf16_t>(b, stream);
    if (rc != MAGIC_OK) return rc;
    if (a->n_q > 0 && a->n_k > 0) {
        const GradRows g = {d_out, ld_do, hs_do, b.lse2, b.rest};
        rc = prepare(a, f16, &g, ar, b.pr, stream);
        if (rc != MAGIC_OK) return rc;
    }
    if (f16) {
        rc = sweeps_of<F16x2>(b, false, stream);
        if (rc != MAGIC_OK) return rc;
        b.pr.rg.want_safe = false;             // the segments whose rows differ too much in size
    }
    rc = f32 ? sweeps_of<F32x3>(b, true, stream) : sweeps_of<BF16>(b, true, stream);
    if (rc != MAGIC_OK) return rc;
    if (b.n_split == 1 && dk && b.pr.idx) {
        const int grid = magic::stride_grid(a->n_k * a->kv_heads * a->head_dim / 8, 256);
        if (f32)
            MAGIC_LAUNCH("attn_dkv_masked", k_attn_dkv_masked<float>, grid, 256, 0, stream, b);
        else
            MAGIC_LAUNCH("attn_dkv_masked", k_attn_dkv_masked<bf16_t>, grid, 256, 0, stream, b);
    }
    if (b.n_split > 1 && a->n_k > 0) {
        const int grid = magic::stride_grid(a->n_k * a->kv_heads * a->head_dim / 2, 256);
        if (f32)
            MAGIC_LAUNCH("attn_dkv_join", k_attn_dkv_join<float>, grid, 256, 0, stream, b);
        else
            MAGIC_LAUNCH("attn_dkv_join", k_attn_dkv_join<bf16_t>, grid, 256, 0, stream, b);
    }
    if (d_slopes && !(dk && a->n_k > 0))
        MAGIC_LAUNCH("attn_bwd_dslope", k_attn_dslope, a->q_heads, 256, 0, stream, b.slope_part, b.n_slope, a->q_heads, d_slopes);
    return magic::launch_status();
}

}  // extern "C"
