// Softmax attention of the rows of a segment over the keys of the same segment (magic_attn_*).
//   s = scale q.k,  c = cap tanh(s / cap) (cap > 0),  l = c - slope_h |pos_q - pos_k|,  p = softmax of l over the
//   unmasked keys,  o = sum p v;   lse = log sum exp(l), -inf for a row that sees no key (o = 0 then).
// Backward, with D_i = do_i.o_i and p recomputed from lse:
//   dv = p^T do,  dl = p (do.v - D),  ds = scale dl (1 - (c / cap)^2),  dq = ds k,  dk = ds^T q,
//   dslope_h = -sum dl |pos_q - pos_k|.
#include "common.h"
#include "lowp.h"

namespace {

constexpr int MAXD = MAGIC_ATTN_MAX_DIM;

struct BwdArgs {
    magic_attn a;
    const void *out, *dout;
    int64_t ld_o, hs_o, ld_do, hs_do;
    const float *lse;
    float *delta;   // [Hq][n_q]
    void *dq, *dk, *dv;
    float *slope_part;  // [n_q tiles][Hq]
    float *dslopes;
};

template <typename T> __device__ __forceinline__ const T *row_of(const void *p, int64_t ld, int64_t hs, int64_t r, int h) {
    return (const T *)p + r * ld + h * hs;
}

// what one lane of a wavefront wrote to LDS is read by another (the wavefront's LDS operations run in order)
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// capped, biased logit; c: the capped score
__device__ __forceinline__ float logit(const magic_attn &a, float dot, int h, int64_t qr, int64_t kr, float &c, float &dist) {
    c = dot * a.scale;
    if (a.cap > 0.f) c = a.cap * tanhf(c / a.cap);
    dist = 0.f;
    float l = c;
    if (a.slopes) {
        const int64_t d = (int64_t)a.q_pos[qr] - a.k_pos[kr];
        dist = (float)(d < 0 ? -d : d);
        l -= a.slopes[h] * dist;
    }
    return l;
}

// wavefront per (row, head): lanes over keys for the scores, over columns for the output
template <typename T> __global__ __launch_bounds__(256) void k_attn_fwd(magic_attn a, T *out, int64_t ld_o, int64_t hs_o, float *lse) {
    __shared__ float sq[4][MAXD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, D = a.head_dim;
    const int32_t *t = a.q_tiles + 4 * (int64_t)blockIdx.x;
    const int64_t q0 = t[0], k0 = t[2];
    const int nq = t[1], nk = t[3], hk = h / (a.q_heads / a.kv_heads);
    for (int i = wave; i < nq; i += 4) {
        const T *q = row_of<T>(a.q, a.ld_q, a.hs_q, q0 + i, h);
        for (int d = lane; d < D; d += 64) sq[wave][d] = (float)q[d];
        wave_lds_sync();
        float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
        for (int j0 = 0; j0 < nk; j0 += 64) {
            const int j = j0 + lane;
            float x = -INFINITY, c, dist;
            if (j < nk && (!a.key_mask || a.key_mask[k0 + j])) {
                const T *k = row_of<T>(a.k, a.ld_k, a.hs_k, k0 + j, hk);
                float s = 0.f;
                for (int d = 0; d < D; ++d) s += sq[wave][d] * (float)k[d];
                x = logit(a, s, h, q0 + i, k0 + j, c, dist);
            }
            const float mx = fmaxf(m, wave_max(x));
            if (mx == -INFINITY) continue;
            const float p = expf(x - mx), f = expf(m - mx);
            l = l * f + wave_sum(p);
            o0 *= f, o1 *= f, m = mx;
            for (int jj = 0; jj < 64 && j0 + jj < nk; ++jj) {
                const float pj = __shfl(p, jj, 64);
                if (pj == 0.f) continue;
                const T *v = row_of<T>(a.v, a.ld_v, a.hs_v, k0 + j0 + jj, hk);
                if (lane < D) o0 += pj * (float)v[lane];
                if (lane + 64 < D) o1 += pj * (float)v[lane + 64];
            }
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
        T *o = out + (q0 + i) * ld_o + h * hs_o;
        if (lane < D) o[lane] = (T)(o0 * inv);
        if (lane + 64 < D) o[lane + 64] = (T)(o1 * inv);
        if (lane == 0) lse[(int64_t)h * a.n_q + q0 + i] = l > 0.f ? m + logf(l) : -INFINITY;
        wave_lds_sync();
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_attn_delta(BwdArgs b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, D = b.a.head_dim;
    for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < b.a.n_q; r += (int64_t)gridDim.x * 4) {
        const T *o = row_of<T>(b.out, b.ld_o, b.hs_o, r, h), *d = row_of<T>(b.dout, b.ld_do, b.hs_do, r, h);
        float s = 0.f;
        for (int i = lane; i < D; i += 64) s += (float)o[i] * (float)d[i];
        s = wave_sum(s);
        if (lane == 0) b.delta[(int64_t)h * b.a.n_q + r] = s;
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_attn_dq(BwdArgs b) {
    __shared__ float sq[4][MAXD], sd[4][MAXD], red[4];
    const magic_attn &a = b.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, D = a.head_dim;
    const int32_t *t = a.q_tiles + 4 * (int64_t)blockIdx.x;
    const int64_t q0 = t[0], k0 = t[2];
    const int nq = t[1], nk = t[3], hk = h / (a.q_heads / a.kv_heads);
    float dsl = 0.f;
    for (int i = wave; i < nq; i += 4) {
        const T *q = row_of<T>(a.q, a.ld_q, a.hs_q, q0 + i, h), *g = row_of<T>(b.dout, b.ld_do, b.hs_do, q0 + i, h);
        for (int d = lane; d < D; d += 64) sq[wave][d] = (float)q[d], sd[wave][d] = (float)g[d];
        wave_lds_sync();
        const float ls = b.lse[(int64_t)h * a.n_q + q0 + i], dl0 = b.delta[(int64_t)h * a.n_q + q0 + i];
        float o0 = 0.f, o1 = 0.f;
        for (int j0 = 0; j0 < nk; j0 += 64) {
            const int j = j0 + lane;
            float ds = 0.f;
            if (j < nk && (!a.key_mask || a.key_mask[k0 + j]) && ls > -INFINITY) {
                const T *k = row_of<T>(a.k, a.ld_k, a.hs_k, k0 + j, hk), *v = row_of<T>(a.v, a.ld_v, a.hs_v, k0 + j, hk);
                float s = 0.f, dp = 0.f, c, dist;
                for (int d = 0; d < D; ++d) s += sq[wave][d] * (float)k[d], dp += sd[wave][d] * (float)v[d];
                const float p = expf(logit(a, s, h, q0 + i, k0 + j, c, dist) - ls);
                const float dl = p * (dp - dl0);
                dsl -= dl * dist;
                ds = dl * a.scale;
                if (a.cap > 0.f) ds *= 1.f - (c / a.cap) * (c / a.cap);
            }
            for (int jj = 0; jj < 64 && j0 + jj < nk; ++jj) {
                const float w = __shfl(ds, jj, 64);
                if (w == 0.f) continue;
                const T *k = row_of<T>(a.k, a.ld_k, a.hs_k, k0 + j0 + jj, hk);
                if (lane < D) o0 += w * (float)k[lane];
                if (lane + 64 < D) o1 += w * (float)k[lane + 64];
            }
        }
        T *o = (T *)b.dq + ((q0 + i) * a.q_heads + h) * D;
        if (lane < D) o[lane] = (T)o0;
        if (lane + 64 < D) o[lane + 64] = (T)o1;
        wave_lds_sync();
    }
    if (b.slope_part) {
        dsl = wave_sum(dsl);
        if (lane == 0) red[wave] = dsl;
        __syncthreads();
        if (threadIdx.x == 0) b.slope_part[(int64_t)blockIdx.x * a.q_heads + h] = (red[0] + red[1]) + (red[2] + red[3]);
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_attn_dkv(BwdArgs b) {
    __shared__ float sk[4][MAXD], sv[4][MAXD];
    const magic_attn &a = b.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hk = blockIdx.y, D = a.head_dim, G = a.q_heads / a.kv_heads;
    const int32_t *t = a.k_tiles + 4 * (int64_t)blockIdx.x;
    const int64_t k0 = t[0], q0 = t[2];
    const int nk = t[1], nq = t[3];
    for (int j = wave; j < nk; j += 4) {
        const T *k = row_of<T>(a.k, a.ld_k, a.hs_k, k0 + j, hk), *v = row_of<T>(a.v, a.ld_v, a.hs_v, k0 + j, hk);
        for (int d = lane; d < D; d += 64) sk[wave][d] = (float)k[d], sv[wave][d] = (float)v[d];
        wave_lds_sync();
        float gk0 = 0.f, gk1 = 0.f, gv0 = 0.f, gv1 = 0.f;
        const bool seen = !a.key_mask || a.key_mask[k0 + j];
        if (seen) {
            for (int h = hk * G; h < hk * G + G; ++h)
                for (int i0 = 0; i0 < nq; i0 += 64) {
                    const int i = i0 + lane;
                    float p = 0.f, ds = 0.f;
                    if (i < nq) {
                        const float ls = b.lse[(int64_t)h * a.n_q + q0 + i];
                        if (ls > -INFINITY) {
                            const T *q = row_of<T>(a.q, a.ld_q, a.hs_q, q0 + i, h), *g = row_of<T>(b.dout, b.ld_do, b.hs_do, q0 + i, h);
                            float s = 0.f, dp = 0.f, c, dist;
                            for (int d = 0; d < D; ++d) s += sk[wave][d] * (float)q[d], dp += sv[wave][d] * (float)g[d];
                            p = expf(logit(a, s, h, q0 + i, k0 + j, c, dist) - ls);
                            ds = p * (dp - b.delta[(int64_t)h * a.n_q + q0 + i]) * a.scale;
                            if (a.cap > 0.f) ds *= 1.f - (c / a.cap) * (c / a.cap);
                        }
                    }
                    for (int ii = 0; ii < 64 && i0 + ii < nq; ++ii) {
                        const float wp = __shfl(p, ii, 64), ws = __shfl(ds, ii, 64);
                        const T *q = row_of<T>(a.q, a.ld_q, a.hs_q, q0 + i0 + ii, h), *g = row_of<T>(b.dout, b.ld_do, b.hs_do, q0 + i0 + ii, h);
                        if (lane < D) gk0 += ws * (float)q[lane], gv0 += wp * (float)g[lane];
                        if (lane + 64 < D) gk1 += ws * (float)q[lane + 64], gv1 += wp * (float)g[lane + 64];
                    }
                }
        }
        T *ok = (T *)b.dk + ((k0 + j) * a.kv_heads + hk) * D, *ov = (T *)b.dv + ((k0 + j) * a.kv_heads + hk) * D;
        if (lane < D) ok[lane] = (T)gk0, ov[lane] = (T)gv0;
        if (lane + 64 < D) ok[lane + 64] = (T)gk1, ov[lane + 64] = (T)gv1;
        wave_lds_sync();
    }
}

// d slope of a head: the tile sums in order, in double
__global__ __launch_bounds__(64) void k_attn_dslope(const float *part, int n, int H, float *out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 64) s += (double)part[(int64_t)i * H + blockIdx.x];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x == 0) out[blockIdx.x] = (float)s;
}

int check(const magic_attn *a) {
    if (!a) return MAGIC_ERR_INVALID_ARG;
    if (a->dtype != MAGIC_F32 && a->dtype != MAGIC_BF16) return MAGIC_ERR_UNSUPPORTED;
    if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->head_dim < 1) return MAGIC_ERR_INVALID_ARG;
    if (a->head_dim > MAXD || a->head_dim % 8 || a->q_heads > 65535) return MAGIC_ERR_UNSUPPORTED;
    if (a->n_q < 0 || a->n_k < 0 || a->n_q > 0x7fffffff || a->n_k > 0x7fffffff) return MAGIC_ERR_INVALID_ARG;
    if (a->n_q_tiles < 0 || a->n_k_tiles < 0) return MAGIC_ERR_INVALID_ARG;
    if (a->n_q > 0 && (!a->q || a->n_q_tiles < 1 || !a->q_tiles)) return MAGIC_ERR_INVALID_ARG;
    if (a->n_k > 0 && (!a->k || !a->v)) return MAGIC_ERR_INVALID_ARG;
    if (a->ld_q < 0 || a->hs_q < 0 || a->ld_k < 0 || a->hs_k < 0 || a->ld_v < 0 || a->hs_v < 0) return MAGIC_ERR_INVALID_ARG;
    if (!(a->cap >= 0.f) || !(a->scale == a->scale)) return MAGIC_ERR_INVALID_ARG;
    if (a->slopes && ((a->n_q > 0 && !a->q_pos) || (a->n_k > 0 && !a->k_pos))) return MAGIC_ERR_INVALID_ARG;
    return MAGIC_OK;
}

}  // namespace

extern "C" {

size_t magic_attn_fwd_workspace_bytes(const magic_attn *a) { return 256; }

int magic_attn_fwd(const magic_attn *a, void *out, int64_t ld_out, int64_t hs_out, float *lse, void *workspace,
                   size_t workspace_bytes, void *stream) {
    const int st = check(a);
    if (st != MAGIC_OK || a->n_q == 0) return st;
    if (!out || !lse) return MAGIC_ERR_INVALID_ARG;
    const dim3 grid(a->n_q_tiles, a->q_heads);
    if (a->dtype == MAGIC_F32)
        MAGIC_LAUNCH("attn_fwd", k_attn_fwd<float>, grid, 256, 0, (hipStream_t)stream, *a, (float *)out, ld_out, hs_out, lse);
    else
        MAGIC_LAUNCH("attn_fwd", k_attn_fwd<magic::bf16_t>, grid, 256, 0, (hipStream_t)stream, *a, (magic::bf16_t *)out, ld_out,
                     hs_out, lse);
    return magic::launch_status();
}

size_t magic_attn_bwd_workspace_bytes(const magic_attn *a) {
    if (check(a) != MAGIC_OK) return 256;
    return magic::align_up((size_t)a->n_q * a->q_heads * sizeof(float)) +
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
    BwdArgs b;
    b.a = *a;
    b.out = out, b.dout = d_out, b.ld_o = ld_out, b.hs_o = hs_out, b.ld_do = ld_do, b.hs_do = hs_do;
    b.lse = lse, b.dq = dq, b.dk = dk, b.dv = dv, b.dslopes = d_slopes;
    magic::Arena ar(workspace, workspace_bytes);
    b.delta = ar.take<float>((size_t)a->n_q * a->q_heads);
    b.slope_part = ar.take<float>((size_t)a->n_q_tiles * a->q_heads);
    if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
    if (!d_slopes) b.slope_part = nullptr;
    const bool f32 = a->dtype == MAGIC_F32;
    if (a->n_q > 0) {
        const dim3 gd(magic::stride_grid(a->n_q, 4, 4096), a->q_heads), gq(a->n_q_tiles, a->q_heads);
        if (f32) {
            MAGIC_LAUNCH("attn_bwd_delta", k_attn_delta<float>, gd, 256, 0, stream, b);
            if (dq) MAGIC_LAUNCH("attn_bwd_dq", k_attn_dq<float>, gq, 256, 0, stream, b);
        } else {
            MAGIC_LAUNCH("attn_bwd_delta", k_attn_delta<magic::bf16_t>, gd, 256, 0, stream, b);
            if (dq) MAGIC_LAUNCH("attn_bwd_dq", k_attn_dq<magic::bf16_t>, gq, 256, 0, stream, b);
        }
    }
    if (dk && a->n_k > 0) {
        const dim3 gk(a->n_k_tiles, a->kv_heads);
        if (f32)
            MAGIC_LAUNCH("attn_bwd_dkv", k_attn_dkv<float>, gk, 256, 0, stream, b);
        else
            MAGIC_LAUNCH("attn_bwd_dkv", k_attn_dkv<magic::bf16_t>, gk, 256, 0, stream, b);
    }
    if (d_slopes)
        MAGIC_LAUNCH("attn_bwd_dslope", k_attn_dslope, a->q_heads, 64, 0, stream, b.slope_part, a->n_q > 0 ? a->n_q_tiles : 0,
                     a->q_heads, d_slopes);
    return magic::launch_status();
}

}  // extern "C"
