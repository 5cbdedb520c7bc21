// RMS norm of every head of the queries and keys with the position rotation, one pass (magic_head_norm_rope_*).
//   r = rsqrt(mean_d x_d^2 + eps),  u = x r w,  pairs (i, i + R/2) of the first R columns turned by the angle
//   pos * base^(-2i/R).   Backward: gu = turn(-angle) dy;  dw += gu x r;  g = gu w;
//   dx = r (g - x r^2 mean_d(g x)).
// HBM-bound: every element is read once and written once (backward: x and dy read, dx written).  A group of GL lanes
// owns one row and walks its heads, so that the sines of a row are formed once and serve all heads: a lane holds the
// chunk of VEC columns at c and its partner at c + R/2.  Angles: pos times the frequency in revolutions as a double,
// reduced to [-1/2, 1/2] before it is rounded to float (position 700,000 times the first frequency is 1e5
// revolutions: in float the angle would be off by 0.05).
#include "common.h"
#include "lowp.h"

namespace {

struct RopeArgs {
    int64_t n;
    int hq, hk, D, half;      // half = R / 2 rotated pairs
    const void *q, *k;
    int64_t ld_q, hs_q, ld_k, hs_k;           // row and head strides, elements
    const float *wq, *wk;
    const int32_t *pos;
    float eps;
    void *yq, *yk;            // forward: [n, h, D] contiguous
    const void *dyq, *dyk;    // backward
    int64_t ld_dyq, hs_dyq, ld_dyk, hs_dyk;
    float *partial;           // backward: [gridDim.x][2][D]
    double freq[64];          // base^(-2i/R) / (2 pi)
};

// item j of a head: j < half / VEC: the pair of chunks at j*VEC and half + j*VEC; above: the plain chunk behind them
template <int VEC> struct Item {
    int a, b;                 // first columns; b < 0: no partner
    bool ok;
};
template <int VEC> __device__ __forceinline__ Item<VEC> item(const RopeArgs &p, int j) {
    const int np = p.half / VEC;
    Item<VEC> it;
    if (j < np) {
        it.a = j * VEC, it.b = p.half + j * VEC, it.ok = true;
    } else {
        it.a = 2 * p.half + (j - np) * VEC, it.b = -1, it.ok = it.a < p.D;
    }
    return it;
}

template <int GL> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, GL);
    return v;
}

template <typename T, int VEC, int GL, int IPL, bool BWD>
__global__ __launch_bounds__(256) void k_head_norm(RopeArgs p) {
    constexpr int RPB = 256 / GL;  // rows of a block
    const int gl = threadIdx.x % GL;
    Item<VEC> it[IPL];
    float w[2][IPL][2][VEC];
    float dw[2][IPL][2][VEC];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        it[i] = item<VEC>(p, gl + i * GL);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float *wp = s ? p.wk : p.wq;
                w[s][i][0][e] = it[i].ok ? wp[it[i].a + e] : 0.f;
                w[s][i][1][e] = it[i].b >= 0 ? wp[it[i].b + e] : 0.f;
                dw[s][i][0][e] = dw[s][i][1][e] = 0.f;
            }
    }
    const float inv_d = 1.f / (float)p.D;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / GL; row < p.n; row += (int64_t)gridDim.x * RPB) {
        float sn[IPL][VEC], cs[IPL][VEC];
        const double ps = (double)p.pos[row];
#pragma unroll
        for (int i = 0; i < IPL; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                double t = it[i].b >= 0 ? ps * p.freq[it[i].a + e] : 0.0;
                t -= rint(t);
                sincospif(2.f * (float)t, &sn[i][e], &cs[i][e]);
            }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int nh = s ? p.hk : p.hq;
            const T *x = (const T *)(s ? p.k : p.q) + row * (s ? p.ld_k : p.ld_q);
            const int64_t hs = s ? p.hs_k : p.hs_q;
            const T *dy = BWD ? (const T *)(s ? p.dyk : p.dyq) + row * (s ? p.ld_dyk : p.ld_dyq) : nullptr;
            const int64_t hsd = s ? p.hs_dyk : p.hs_dyq;
            T *y = (T *)(s ? p.yk : p.yq) + row * nh * p.D;
            for (int h = 0; h < nh; ++h, x += hs, y += p.D) {
                float v[IPL][2][VEC], g[IPL][2][VEC];
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < IPL; ++i) {
                    magic::load_vec<T, VEC>(x + it[i].a, it[i].ok, v[i][0]);
                    magic::load_vec<T, VEC>(x + it[i].b, it[i].b >= 0, v[i][1]);
                    if (BWD) {
                        magic::load_vec<T, VEC>(dy + (int64_t)h * hsd + it[i].a, it[i].ok, g[i][0]);
                        magic::load_vec<T, VEC>(dy + (int64_t)h * hsd + it[i].b, it[i].b >= 0, g[i][1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < IPL; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) ss += v[i][0][e] * v[i][0][e] + v[i][1][e] * v[i][1][e];
                ss = group_sum<GL>(ss);
                const float r = 1.f / sqrtf(ss * inv_d + p.eps);
                if (!BWD) {
#pragma unroll
                    for (int i = 0; i < IPL; ++i) {
                        float o[2][VEC];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float a = v[i][0][e] * r * w[s][i][0][e], b = v[i][1][e] * r * w[s][i][1][e];
                            o[0][e] = a * cs[i][e] - b * sn[i][e];
                            o[1][e] = b * cs[i][e] + a * sn[i][e];
                        }
                        magic::store_vec<T, VEC>(y + it[i].a, it[i].ok, o[0]);
                        magic::store_vec<T, VEC>(y + it[i].b, it[i].b >= 0, o[1]);
                    }
                } else {
                    float dot = 0.f;
#pragma unroll
                    for (int i = 0; i < IPL; ++i)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float a = g[i][0][e] * cs[i][e] + g[i][1][e] * sn[i][e];
                            const float b = g[i][1][e] * cs[i][e] - g[i][0][e] * sn[i][e];
                            dw[s][i][0][e] += a * v[i][0][e] * r;
                            dw[s][i][1][e] += b * v[i][1][e] * r;
                            g[i][0][e] = a * w[s][i][0][e];
                            g[i][1][e] = b * w[s][i][1][e];
                            dot += g[i][0][e] * v[i][0][e] + g[i][1][e] * v[i][1][e];
                        }
                    dot = group_sum<GL>(dot) * inv_d * r * r;
#pragma unroll
                    for (int i = 0; i < IPL; ++i) {
                        float o[2][VEC];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            o[0][e] = r * (g[i][0][e] - v[i][0][e] * dot);
                            o[1][e] = r * (g[i][1][e] - v[i][1][e] * dot);
                        }
                        magic::store_vec<T, VEC>(y + it[i].a, it[i].ok, o[0]);
                        magic::store_vec<T, VEC>(y + it[i].b, it[i].b >= 0, o[1]);
                    }
                }
            }
        }
    }
    if (BWD) {
        // the block's weight gradients: row groups added in order through LDS
        __shared__ float red[2][128];
        for (int t = threadIdx.x; t < 256; t += 256) red[t >> 7][t & 127] = 0.f;
        __syncthreads();
        // lanes of a wavefront that hold the same columns first (fixed tree), then the four wavefronts in order
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < IPL; ++i)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
#pragma unroll
                        for (int o = 32; o >= GL; o >>= 1) dw[s][i][c][e] += __shfl_xor(dw[s][i][c][e], o, 64);
        for (int wv = 0; wv < 4; ++wv) {
            if ((int)(threadIdx.x >> 6) == wv && (threadIdx.x & 63) < GL) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < IPL; ++i)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            if (it[i].ok) red[s][it[i].a + e] += dw[s][i][0][e];
                            if (it[i].b >= 0) red[s][it[i].b + e] += dw[s][i][1][e];
                        }
            }
            __syncthreads();
        }
        for (int t = threadIdx.x; t < 2 * p.D; t += 256)
            p.partial[(int64_t)blockIdx.x * 2 * p.D + t] = red[t / p.D][t % p.D];
    }
}

// column sums of the block partials, in double: wavefront per output column, blocks lane by lane, fixed tree
__global__ __launch_bounds__(64) void k_head_norm_dw(const float *partial, int blocks, int D, float *dwq, float *dwk) {
    const int c = blockIdx.x;
    double s = 0.0;
    for (int b = threadIdx.x; b < blocks; b += 64) s += (double)partial[(int64_t)b * 2 * D + c];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x == 0) {
        if (c < D) dwq[c] = (float)s;
        else dwk[c - D] = (float)s;
    }
}

int rope_blocks(int64_t n, int gl) { return magic::stride_grid(n, 256 / gl, 1024); }

template <typename T, int VEC, int GL, int IPL> int run(const RopeArgs &p, bool bwd, hipStream_t st) {
    const int grid = rope_blocks(p.n, GL);
    if (bwd)
        MAGIC_LAUNCH("head_norm_rope_bwd", (k_head_norm<T, VEC, GL, IPL, true>), grid, 256, 0, st, p);
    else
        MAGIC_LAUNCH("head_norm_rope_fwd", (k_head_norm<T, VEC, GL, IPL, false>), grid, 256, 0, st, p);
    return magic::launch_status();
}

template <typename T, int VEC> int pick(const RopeArgs &p, bool bwd, hipStream_t st, int *gl_out) {
    const int items = p.half / VEC + (p.D - 2 * p.half) / VEC;
    int gl = 4;
    while (gl < items && gl < 64) gl *= 2;
    if (gl_out) {
        *gl_out = gl;
        return MAGIC_OK;
    }
    if (gl < items) return run<T, VEC, 64, 2>(p, bwd, st);  // at most 127 items (one pair, 126 plain columns)
    switch (gl) {
        case 4: return run<T, VEC, 4, 1>(p, bwd, st);
        case 8: return run<T, VEC, 8, 1>(p, bwd, st);
        case 16: return run<T, VEC, 16, 1>(p, bwd, st);
        case 32: return run<T, VEC, 32, 1>(p, bwd, st);
        default: return run<T, VEC, 64, 1>(p, bwd, st);
    }
}

bool mult(const void *p, int64_t ld, int64_t hs, int vec, int size) {
    return (uintptr_t)p % (size_t)(vec * size) == 0 && ld % vec == 0 && hs % vec == 0;
}

// whole chunks of 4 columns wherever strides, widths and addresses allow them, single columns otherwise
int launch(const RopeArgs &p, int dtype, bool bwd, hipStream_t st, int *gl_out = nullptr) {
    const int size = dtype == MAGIC_F32 ? 4 : 2;
    bool v4 = p.half % 4 == 0 && p.D % 4 == 0 && mult(p.q, p.ld_q, p.hs_q, 4, size) && mult(p.k, p.ld_k, p.hs_k, 4, size) &&
              mult(p.yq, 4, 4, 4, size) && mult(p.yk, 4, 4, 4, size);
    if (bwd) v4 = v4 && mult(p.dyq, p.ld_dyq, p.hs_dyq, 4, size) && mult(p.dyk, p.ld_dyk, p.hs_dyk, 4, size);
    if (dtype == MAGIC_F32) return v4 ? pick<float, 4>(p, bwd, st, gl_out) : pick<float, 1>(p, bwd, st, gl_out);
    return v4 ? pick<magic::bf16_t, 4>(p, bwd, st, gl_out) : pick<magic::bf16_t, 1>(p, bwd, st, gl_out);
}

int fill(RopeArgs &p, int64_t n, int hq, int hk, int D, int rot, int dtype, const void *q, int64_t ld_q, int64_t hs_q,
         const void *k, int64_t ld_k, int64_t hs_k, const float *wq, const float *wk, const int32_t *pos, double eps,
         double base) {
    if (n < 0 || hq < 1 || hk < 1 || D < 1 || rot < 0 || rot > D || (rot & 1)) return MAGIC_ERR_INVALID_ARG;
    if (!(eps >= 0.0) || !(base > 0.0)) return MAGIC_ERR_INVALID_ARG;
    if (dtype != MAGIC_F32 && dtype != MAGIC_BF16) return MAGIC_ERR_UNSUPPORTED;
    if (D > MAGIC_ATTN_MAX_DIM) return MAGIC_ERR_UNSUPPORTED;
    if (n == 0) return MAGIC_OK;
    if (!q || !k || !wq || !wk || !pos) return MAGIC_ERR_INVALID_ARG;
    if (ld_q < 0 || hs_q < 0 || ld_k < 0 || hs_k < 0) return MAGIC_ERR_INVALID_ARG;
    p.n = n, p.hq = hq, p.hk = hk, p.D = D, p.half = rot / 2;
    p.q = q, p.k = k, p.ld_q = ld_q, p.hs_q = hs_q, p.ld_k = ld_k, p.hs_k = hs_k;
    p.wq = wq, p.wk = wk, p.pos = pos, p.eps = (float)eps;
    for (int i = 0; i < 64; ++i)
        p.freq[i] = i < p.half ? pow(base, -2.0 * i / rot) * 0.15915494309189533576888376337251 : 0.0;
    return MAGIC_OK;
}

}  // namespace

extern "C" {

int magic_head_norm_rope_fwd(int64_t n_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t rotary_dim,
                             int32_t dtype, const void *q, int64_t ld_q, int64_t hs_q, const void *k, int64_t ld_k,
                             int64_t hs_k, const float *wq, const float *wk, const int32_t *pos, double eps, double base,
                             void *yq, void *yk, void *stream) {
    RopeArgs p = {};
    int st = fill(p, n_rows, q_heads, kv_heads, head_dim, rotary_dim, dtype, q, ld_q, hs_q, k, ld_k, hs_k, wq, wk, pos, eps,
                  base);
    if (st != MAGIC_OK || n_rows == 0) return st;
    if (!yq || !yk) return MAGIC_ERR_INVALID_ARG;
    p.yq = yq, p.yk = yk;
    return launch(p, dtype, false, (hipStream_t)stream);
}

size_t magic_head_norm_rope_bwd_workspace_bytes(int64_t n_rows, int32_t head_dim) {
    if (n_rows < 0 || head_dim < 1) return 256;
    return magic::align_up((size_t)1024 * 2 * head_dim * sizeof(float)) + 256;
}

int magic_head_norm_rope_bwd(int64_t n_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t rotary_dim,
                             int32_t dtype, const void *q, int64_t ld_q, int64_t hs_q, const void *k, int64_t ld_k,
                             int64_t hs_k, const float *wq, const float *wk, const int32_t *pos, double eps, double base,
                             const void *dyq, int64_t ld_dyq, int64_t hs_dyq, const void *dyk, int64_t ld_dyk,
                             int64_t hs_dyk, void *dq, void *dk, float *dwq, float *dwk, void *workspace,
                             size_t workspace_bytes, void *stream_) {
    RopeArgs p = {};
    hipStream_t stream = (hipStream_t)stream_;
    int st = fill(p, n_rows, q_heads, kv_heads, head_dim, rotary_dim, dtype, q, ld_q, hs_q, k, ld_k, hs_k, wq, wk, pos, eps,
                  base);
    if (st != MAGIC_OK) return st;
    if (!dwq || !dwk) return MAGIC_ERR_INVALID_ARG;
    int grid = 0;
    magic::Arena ar(workspace, workspace_bytes);
    p.partial = ar.take<float>((size_t)1024 * 2 * head_dim);
    if (!ar.ok() || !p.partial) return MAGIC_ERR_WORKSPACE;
    if (n_rows > 0) {
        if (!dyq || !dyk || !dq || !dk || ld_dyq < 0 || hs_dyq < 0 || ld_dyk < 0 || hs_dyk < 0) return MAGIC_ERR_INVALID_ARG;
        p.yq = dq, p.yk = dk;
        p.dyq = dyq, p.ld_dyq = ld_dyq, p.hs_dyq = hs_dyq, p.dyk = dyk, p.ld_dyk = ld_dyk, p.hs_dyk = hs_dyk;
        int gl = 0;
        launch(p, dtype, true, stream, &gl);
        grid = rope_blocks(n_rows, gl);
        st = launch(p, dtype, true, stream);
        if (st != MAGIC_OK) return st;
    }
    MAGIC_LAUNCH("head_norm_rope_dw", k_head_norm_dw, 2 * head_dim, 64, 0, stream, p.partial, grid, head_dim, dwq, dwk);
    return magic::launch_status();
}

}  // extern "C"
