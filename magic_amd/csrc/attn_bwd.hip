// Segment attention, backward (magic_attn_bwd).  With D_i = do_i.o_i and p recomputed from lse:
//   dv = p^T do,  dl = p (do.v - D),  ds = scale dl (1 - (c / cap)^2),  dq = ds k,  dk = ds^T q,
//   dslope_h = -sum dl |pos_q - pos_k|.
// Two sweeps, so that every sum has one owner and a fixed order (no atomics): dq with the rows' wavefronts walking the
// keys (three products), dk and dv with the keys' wavefronts walking the rows of all heads that share them (four).
// Seven products instead of the five that one sweep with atomic adds would need.
#include "attn_common.h"

namespace {

using namespace magic::attn;
using magic::bf16_t;
using magic::bf16x8_t;

struct BwdArgs {
    magic_attn a;
    const void *out, *dout;
    int64_t ld_o, hs_o, ld_do, hs_do;
    const float *lse;
    float *lse2;        // [q_heads][n_q] lse in base 2, +inf for rows that see no key (their probabilities become zeros)
    float *delta;       // [q_heads][n_q]
    void *dq, *dk, *dv;
    float *slope_part;  // [n_q tiles][q_heads] or NULL
    int64_t items;
};

// lse2 and D of every row: DP / 8 lanes a row and head
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
#pragma unroll
            for (int e = 0; e < 8; ++e) s += x[e] * y[e];
        }
#pragma unroll
        for (int k = LPR / 2; k > 0; k >>= 1) s += __shfl_xor(s, k, LPR);
        if (l == 0) {
            const float ls = b.lse[(int64_t)h * a.n_q + row];
            const bool none = ls == -INFINITY;
            b.lse2[(int64_t)h * a.n_q + row] = none ? INFINITY : ls * LOG2E;
            b.delta[(int64_t)h * a.n_q + row] = none ? 0.f : s;
        }
    }
}

// p and ds of one 32 x 32 tile in place: s = scores before the scale, dp = do.v; the lane's column carries `cl`-side
// values, the four registers of a group the row-side ones
struct Soft {
    float s_in, s_out, scale, cap;
    __device__ __forceinline__ void init(const magic_attn &a) {
        cap = a.cap, scale = a.scale;
        s_in = cap > 0.f ? a.scale / cap : a.scale * LOG2E, s_out = cap * LOG2E;
    }
};

constexpr int NT = 256, BK = 64;

template <typename T, int DP>
__global__ __launch_bounds__(NT, (DP == 128 && Planes<T>::N == 3) ? 1 : 2) void k_attn_dq(BwdArgs p) {
    constexpr int NP = Planes<T>::N, KS = DP / 16, DB = (DP + 31) / 32;
    typedef Stage<T, DP, BK, NT> stage;
    typedef Tile<T, DP, BK> tile;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16_t *sK = reinterpret_cast<bf16_t *>(smem), *sV = sK + NP * tile::PLANE;
    uint32_t *sPos = reinterpret_cast<uint32_t *>(smem + 2 * tile::BYTES);
    float *sMask = reinterpret_cast<float *>(sPos + BK);

    const magic_attn &a = p.a;
    const int64_t item = xcd_item(blockIdx.x, 16);
    if (item >= p.items) return;
    const int D = a.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int64_t tl = item % a.n_q_tiles;
    const int h = (int)(item / a.n_q_tiles), hk = h / (a.q_heads / a.kv_heads);
    const int32_t *t = a.q_tiles + 4 * tl;
    const int64_t q0 = t[0], k0 = t[2];
    const int nq = t[1], nk = t[3];
    const int row = wave * 32 + li;
    const bool ok = row < nq;
    const int64_t qr = q0 + (ok ? row : 0);
    const T *K = (const T *)a.k + k0 * a.ld_k + hk * a.hs_k, *V = (const T *)a.v + k0 * a.ld_v + hk * a.hs_v;
    const float ls = ok ? p.lse2[(int64_t)h * a.n_q + qr] : INFINITY, dl0 = ok ? p.delta[(int64_t)h * a.n_q + qr] : 0.f;
    const bool live = ls != INFINITY;

    bf16x8_t qf[KS][NP], gf[KS][NP];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * hf, cc = c < D ? c : 0;
        Raw<T> r, g;
        r.load((const T *)a.q + qr * a.ld_q + h * a.hs_q + cc);
        g.load((const T *)p.dout + qr * p.ld_do + h * p.hs_do + cc);
        if (!ok || c >= D) r.zero();
        if (!live || c >= D) g.zero();
        r.planes(qf[ks]);
        g.planes(gf[ks]);
    }
    const bool bias = a.slopes != nullptr;
    const float slope2 = bias ? a.slopes[h] * LOG2E : 0.f;
    const uint32_t qpos = bias ? flip(a.q_pos[qr]) : 0u;
    Soft sf;
    sf.init(a);
    float dsl = 0.f;
    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

    stage kst, vst;
    uint8_t keep[stage::N];
    uint32_t pos = 0;
    float mk = 0.f;
    auto load = [&](int j0) {
        kst.load(K, a.ld_k, j0, nk, D, tid);
        vst.load(V, a.ld_v, j0, nk, D, tid);
#pragma unroll
        for (int i = 0; i < stage::N; ++i) {
            const int j = j0 + stage::row_of(i, tid);
            keep[i] = j < nk;
            if (a.key_mask && j < nk) keep[i] = a.key_mask[k0 + j];
        }
        if (tid < BK) {
            const int j = j0 + tid;
            const bool in = j < nk;
            mk = in && (!a.key_mask || a.key_mask[k0 + (in ? j : 0)]) ? 1.f : 0.f;
            pos = bias && in ? flip(a.k_pos[k0 + j]) : 0u;
        }
    };
    if (nk > 0) load(0);
    for (int j0 = 0; j0 < nk; j0 += BK) {
        __syncthreads();
        kst.store(sK, D, tid, [&](int i, int) { return keep[i] != 0; });
        vst.store(sV, D, tid, [&](int i, int) { return keep[i] != 0; });
        if (tid < BK) sPos[tid] = pos, sMask[tid] = mk;
        const bool masked = a.key_mask != nullptr || j0 + BK > nk;
        __syncthreads();
        if (j0 + BK < nk) load(j0 + BK);
#pragma unroll
        for (int b = 0; b < BK / 32; ++b) {
            f32x16_t s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8_t f[NP], g[NP];
                tile::frag(sK, 32 * b + li, 16 * ks + 8 * hf, f);
                tile::frag(sV, 32 * b + li, 16 * ks + 8 * hf, g);
                mma(s, f, qf[ks]);
                mma(dp, g, gf[ks]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float ds[8];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int jr = 32 * b + 16 * u + 8 * g + 4 * hf;
                    f32x4_t km = {1.f, 1.f, 1.f, 1.f};
                    if (masked) km = *reinterpret_cast<const f32x4_t *>(sMask + jr);
                    i32x4_t kp = {0, 0, 0, 0};
                    if (bias) kp = *reinterpret_cast<const i32x4_t *>(sPos + jr);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 8 * u + 4 * g + e;
                        float x = s[r] * sf.s_in, f = sf.scale, dist = 0.f;
                        if (sf.cap > 0.f) {
                            const float th = tanh_f(x);
                            x = th * sf.s_out;
                            f *= 1.f - th * th;
                        }
                        if (bias) {
                            dist = dist_of((uint32_t)kp[e], qpos);
                            x -= slope2 * dist;
                        }
                        float pr = __builtin_amdgcn_exp2f(x - ls);
                        float dl = pr * (dp[r] - dl0);
                        if (km[e] == 0.f) dl = 0.f;
                        if (bias) dsl -= dl * dist;
                        ds[4 * g + e] = dl * f;
                    }
                }
                bf16x8_t pf[NP];
                to_planes(ds, pf);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8_t f[NP];
                    tile::frag_t(sK, 32 * b + 16 * u, 32 * d, lane, f);
                    mma(acc[d], f, pf);
                }
            }
        }
    }
    if (ok) {
        T *o = (T *)p.dq + (qr * a.q_heads + h) * D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hf;
                const float x[4] = {acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
                magic::store_vec<T, 4>(o + c, c < D, x);
            }
    }
    if (p.slope_part) {
        __syncthreads();
        float *red = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int k = 32; k > 0; k >>= 1) dsl += __shfl_xor(dsl, k, 64);
        if (lane == 0) red[wave] = dsl;
        __syncthreads();
        if (tid == 0) p.slope_part[tl * a.q_heads + h] = (red[0] + red[1]) + (red[2] + red[3]);
    }
}

template <typename T, int DP, int BQ>
__global__ __launch_bounds__(NT, (DP == 128 && Planes<T>::N == 3) ? 1 : 2) void k_attn_dkv(BwdArgs p) {
    constexpr int NP = Planes<T>::N, KS = DP / 16, DB = (DP + 31) / 32;
    typedef Stage<T, DP, BQ, NT> stage;
    typedef Tile<T, DP, BQ> tile;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16_t *sQ = reinterpret_cast<bf16_t *>(smem), *sG = sQ + NP * tile::PLANE;
    float *sL = reinterpret_cast<float *>(smem + 2 * tile::BYTES), *sD = sL + BQ;
    uint32_t *sPos = reinterpret_cast<uint32_t *>(sD + BQ);

    const magic_attn &a = p.a;
    const int64_t item = xcd_item(blockIdx.x, 16);
    if (item >= p.items) return;
    const int D = a.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int64_t tl = item % a.n_k_tiles;
    const int hk = (int)(item / a.n_k_tiles), G = a.q_heads / a.kv_heads;
    const int32_t *t = a.k_tiles + 4 * tl;
    const int64_t k0 = t[0], q0 = t[2];
    const int nk = t[1], nq = t[3];
    const int col = wave * 32 + li;
    const bool in = col < nk;
    const int64_t kr = k0 + (in ? col : 0);
    const bool ok = in && (!a.key_mask || a.key_mask[kr]);

    bf16x8_t kf[KS][NP], vf[KS][NP];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * hf, cc = c < D ? c : 0;
        Raw<T> r, g;
        r.load((const T *)a.k + kr * a.ld_k + hk * a.hs_k + cc);
        g.load((const T *)a.v + kr * a.ld_v + hk * a.hs_v + cc);
        if (!ok || c >= D) r.zero(), g.zero();
        r.planes(kf[ks]);
        g.planes(vf[ks]);
    }
    const bool bias = a.slopes != nullptr;
    const uint32_t kpos = bias ? flip(a.k_pos[kr]) : 0u;
    Soft sf;
    sf.init(a);
    f32x16_t gk[DB], gv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) gk[d][r] = 0.f, gv[d][r] = 0.f;

    stage qst, gst;
    uint8_t keep[stage::N];
    float ls = 0.f, dl0 = 0.f;
    uint32_t pos = 0;
    auto load = [&](int h, int i0) {
        qst.load((const T *)a.q + q0 * a.ld_q + h * a.hs_q, a.ld_q, i0, nq, D, tid);
        gst.load((const T *)p.dout + q0 * p.ld_do + h * p.hs_do, p.ld_do, i0, nq, D, tid);
        const float *l2 = p.lse2 + (int64_t)h * a.n_q + q0;
#pragma unroll
        for (int i = 0; i < stage::N; ++i) {
            const int r = i0 + stage::row_of(i, tid);
            keep[i] = r < nq && l2[r < nq ? r : 0] != INFINITY;
        }
        if (tid < BQ) {
            const int r = i0 + tid;
            ls = r < nq ? l2[r] : INFINITY;
            dl0 = r < nq ? p.delta[(int64_t)h * a.n_q + q0 + r] : 0.f;
            pos = bias && r < nq ? flip(a.q_pos[q0 + r]) : 0u;
        }
    };
    const int per_h = (nq + BQ - 1) / BQ, steps = per_h * G;
    if (steps > 0) load(hk * G, 0);
    int h = hk * G, it = 0;
    for (int st = 0; st < steps; ++st) {
        __syncthreads();
        qst.store(sQ, D, tid, [&](int i, int) { return keep[i] != 0; });
        gst.store(sG, D, tid, [&](int i, int) { return keep[i] != 0; });
        if (tid < BQ) sL[tid] = ls, sD[tid] = dl0, sPos[tid] = pos;
        const float slope2 = bias ? a.slopes[h] * LOG2E : 0.f;
        __syncthreads();
        if (++it == per_h) it = 0, ++h;
        if (st + 1 < steps) load(h, it * BQ);
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
            f32x16_t s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f, dp[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8_t f[NP], g[NP];
                tile::frag(sQ, 32 * b + li, 16 * ks + 8 * hf, f);
                tile::frag(sG, 32 * b + li, 16 * ks + 8 * hf, g);
                mma(s, f, kf[ks]);
                mma(dp, g, vf[ks]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float pr[8], ds[8];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int ir = 32 * b + 16 * u + 8 * g + 4 * hf;
                    const f32x4_t l4 = *reinterpret_cast<const f32x4_t *>(sL + ir);
                    const f32x4_t d4 = *reinterpret_cast<const f32x4_t *>(sD + ir);
                    i32x4_t qp = {0, 0, 0, 0};
                    if (bias) qp = *reinterpret_cast<const i32x4_t *>(sPos + ir);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 8 * u + 4 * g + e;
                        float x = s[r] * sf.s_in, f = sf.scale;
                        if (sf.cap > 0.f) {
                            const float th = tanh_f(x);
                            x = th * sf.s_out;
                            f *= 1.f - th * th;
                        }
                        if (bias) x -= slope2 * dist_of((uint32_t)qp[e], kpos);
                        const float q = __builtin_amdgcn_exp2f(x - l4[e]);
                        pr[4 * g + e] = q;
                        ds[4 * g + e] = q * (dp[r] - d4[e]) * f;
                    }
                }
                bf16x8_t pf[NP], sfr[NP];
                to_planes(pr, pf);
                to_planes(ds, sfr);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    bf16x8_t f[NP];
                    tile::frag_t(sG, 32 * b + 16 * u, 32 * d, lane, f);
                    mma(gv[d], f, pf);
                    tile::frag_t(sQ, 32 * b + 16 * u, 32 * d, lane, f);
                    mma(gk[d], f, sfr);
                }
            }
        }
    }
    if (!in) return;
    T *ok_ = (T *)p.dk + (kr * a.kv_heads + hk) * D, *ov = (T *)p.dv + (kr * a.kv_heads + hk) * D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hf;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = ok ? gk[d][4 * g + e] : 0.f, y[e] = ok ? gv[d][4 * g + e] : 0.f;
            magic::store_vec<T, 4>(ok_ + c, c < D, x);
            magic::store_vec<T, 4>(ov + c, c < D, y);
        }
}

// d slope of a head: the tile sums lane by lane, fixed tree, in double
__global__ __launch_bounds__(64) void k_attn_dslope(const float *part, int n, int H, float *out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 64) s += (double)part[(int64_t)i * H + blockIdx.x];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x == 0) out[blockIdx.x] = (float)s;
}

template <typename T, int DP> int run(BwdArgs &b, hipStream_t st) {
    const magic_attn &a = b.a;
    constexpr int BQ = 64;
    if (a.n_q > 0) {
        const int grid = magic::stride_grid(a.n_q * a.q_heads, 256 / (DP / 8));
        MAGIC_LAUNCH("attn_bwd_delta", (k_attn_delta<T, DP>), grid, 256, 0, st, b);
    }
    if (a.n_q > 0 && b.dq) {
        const size_t lds = 2 * Tile<T, DP, BK>::BYTES + BK * 8;
        if (magic::ensure_dynamic_lds((const void *)k_attn_dq<T, DP>, lds) != MAGIC_OK) return MAGIC_ERR_RUNTIME;
        b.items = (int64_t)a.n_q_tiles * a.q_heads;
        if (xcd_grid(b.items, 16) > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
        MAGIC_LAUNCH("attn_bwd_dq", (k_attn_dq<T, DP>), (int)xcd_grid(b.items, 16), NT, lds, st, b);
    }
    if (a.n_k > 0 && b.dk) {
        const size_t lds = 2 * Tile<T, DP, BQ>::BYTES + BQ * 12;
        if (magic::ensure_dynamic_lds((const void *)k_attn_dkv<T, DP, BQ>, lds) != MAGIC_OK) return MAGIC_ERR_RUNTIME;
        b.items = (int64_t)a.n_k_tiles * a.kv_heads;
        if (xcd_grid(b.items, 16) > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
        MAGIC_LAUNCH("attn_bwd_dkv", (k_attn_dkv<T, DP, BQ>), (int)xcd_grid(b.items, 16), NT, lds, st, b);
    }
    return magic::launch_status();
}

template <typename T> int pick(BwdArgs &b, hipStream_t st) {
    const int D = b.a.head_dim;
    return D <= 16 ? run<T, 16>(b, st) : D <= 32 ? run<T, 32>(b, st) : D <= 64 ? run<T, 64>(b, st) : run<T, 128>(b, st);
}

}  // namespace

extern "C" {

size_t magic_attn_bwd_workspace_bytes(const magic_attn *a) {
    if (check(a) != MAGIC_OK) return 256;
    return 2 * magic::align_up((size_t)a->n_q * a->q_heads * sizeof(float)) +
           magic::align_up((size_t)a->n_q_tiles * a->q_heads * sizeof(float)) + 256;
}

int magic_attn_bwd(const magic_attn *a, const void *out, int64_t ld_out, int64_t hs_out, const float *lse, const void *d_out,
                   int64_t ld_do, int64_t hs_do, void *dq, void *dk, void *dv, float *d_slopes, void *workspace,
                   size_t workspace_bytes, void *stream_) {
    const int st = check(a);
    if (st != MAGIC_OK) return st;
    hipStream_t stream = (hipStream_t)stream_;
    if (a->n_q > 0 && (!out || !lse || !d_out || (d_slopes && !dq))) return MAGIC_ERR_INVALID_ARG;
    if (!dk != !dv || (dk && a->n_k > 0 && (a->n_k_tiles < 1 || !a->k_tiles))) return MAGIC_ERR_INVALID_ARG;
    if (d_slopes && !a->slopes) return MAGIC_ERR_INVALID_ARG;
    const int per = a->dtype == MAGIC_F32 ? 4 : 8;
    if (((uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) return MAGIC_ERR_INVALID_ARG;
    if (ld_out < 0 || hs_out < 0 || ld_do < 0 || hs_do < 0 || (ld_out | hs_out | ld_do | hs_do) % per) return MAGIC_ERR_INVALID_ARG;
    BwdArgs b;
    b.a = *a;
    b.out = out, b.dout = d_out, b.ld_o = ld_out, b.hs_o = hs_out, b.ld_do = ld_do, b.hs_do = hs_do;
    b.lse = lse, b.dq = dq, b.dk = dk, b.dv = dv;
    magic::Arena ar(workspace, workspace_bytes);
    b.delta = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.lse2 = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.slope_part = ar.take<float>((size_t)a->n_q_tiles * a->q_heads);
    if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
    if (!d_slopes) b.slope_part = nullptr;
    const int rc = a->dtype == MAGIC_F32 ? pick<float>(b, stream) : pick<bf16_t>(b, stream);
    if (rc != MAGIC_OK) return rc;
    if (d_slopes)
        MAGIC_LAUNCH("attn_bwd_dslope", k_attn_dslope, a->q_heads, 64, 0, stream, b.slope_part, a->n_q > 0 ? a->n_q_tiles : 0,
                     a->q_heads, d_slopes);
    return magic::launch_status();
}

}  // extern "C"
