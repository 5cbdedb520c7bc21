// RMS norm of every head of the queries and keys with the position rotation, one pass (magic_head_norm_rope_*).
//   r = rsqrt(mean_d x_d^2 + eps),  u = x r w,  pairs (i, i + R/2) of the first R columns turned by the angle
//   pos * base^(-2i/R).   Backward: gu = turn(-angle) dy;  dw += gu x r;  g = gu w;
//   dx = r (g - x r^2 mean_d(g x)).
// HBM-bound: every element is read once and written once (backward: x and dy read, dx written).  A group of GL lanes
// owns one row and walks its heads, so that the sines of a row are formed once and serve all heads: a lane holds the
// chunk of VEC columns at c and its partner at c + R/2.  Angles: pos times the frequency in revolutions as a double,
// reduced to [-1/2, 1/2] before it is rounded to float (position 700,000 times the first frequency is 1e5
// revolutions: in float the angle would be off by 0.05).
// 97,000 rows of 4 + 4 heads of 64, float32: 75 us forward (5.3 TB/s), 131 us backward (4.6); 131,071 rows of 16 + 4 heads
// of 128, bfloat16: 290 and 439 us (4.6 TB/s both).  A large copy reaches 5.0.
#include "common.h"
#include "lowp.h"

namespace {

constexpr int MAX_BLOCKS = 2048;   // of the row sweep

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
    float *partial;           // backward: [2][D][blocks]
    double freq[64];          // base^(-2i/R) / (2 pi)
};

// Item j of a head, two chunks of VEC columns: the rotated pair (j VEC, half + j VEC), or two chunks of the columns behind
// the rotated ones (b < 0: an odd column left alone)
template <int VEC> struct Item {
    int a, b;
    bool ok, turn;
};
template <int VEC> __device__ __forceinline__ Item<VEC> item(const RopeArgs &p, int j) {
    const int np = p.half / VEC, plain = p.D - 2 * p.half, ph = (plain / VEC + 1) / 2;   // chunks in the first plain half
    Item<VEC> it;
    it.turn = j < np;
    if (it.turn) {
        it.a = j * VEC, it.b = p.half + j * VEC, it.ok = true;
    } else {
        const int i = j - np;
        it.ok = i < ph;
        it.a = 2 * p.half + i * VEC, it.b = 2 * p.half + (ph + i) * VEC;
        if (!it.ok || it.b >= p.D) it.b = -1;
    }
    return it;
}

template <int GL> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, GL);
    return v;
}

// A head's chunks as they lie in memory: the next head's are under way while one is worked on
template <typename T, int VEC, bool BWD> struct Chunks {
    typename magic::vec_of<T, VEC>::type x[2], g[2];
    __device__ __forceinline__ void load(const T *xp, const T *gp, const Item<VEC> &it) {
        typedef typename magic::vec_of<T, VEC>::type vt;
        const int a = it.ok ? it.a : 0, b = it.b >= 0 ? it.b : 0;    // (lanes without columns read the first ones)
        x[0] = *reinterpret_cast<const vt *>(xp + a), x[1] = *reinterpret_cast<const vt *>(xp + b);
        if (BWD) g[0] = *reinterpret_cast<const vt *>(gp + a), g[1] = *reinterpret_cast<const vt *>(gp + b);
    }
};

template <typename T, int VEC, int GL, bool BWD>
__global__ __launch_bounds__(256) void k_head_norm(RopeArgs p) {
    constexpr int RPB = 256 / GL;
    const int gl = threadIdx.x % GL;
    const Item<VEC> it = item<VEC>(p, gl);
    float w[2][2][VEC], dw[2][2][VEC];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float *wp = s ? p.wk : p.wq;
            w[s][0][e] = it.ok ? wp[it.a + e] : 0.f;
            w[s][1][e] = it.b >= 0 ? wp[it.b + e] : 0.f;
            dw[s][0][e] = dw[s][1][e] = 0.f;
        }
    const float inv_d = 1.f / (float)p.D;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / GL; row < p.n; row += (int64_t)gridDim.x * RPB) {
        float sn[VEC], cs[VEC];
        const double ps = (double)p.pos[row];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            double t = it.turn ? ps * p.freq[it.a + e] : 0.0;
            t -= rint(t);
            sincospif(2.f * (float)t, &sn[e], &cs[e]);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int nh = s ? p.hk : p.hq;
            const T *x0 = (const T *)(s ? p.k : p.q) + row * (s ? p.ld_k : p.ld_q);
            const int64_t hs = s ? p.hs_k : p.hs_q;
            const T *dy0 = BWD ? (const T *)(s ? p.dyk : p.dyq) + row * (s ? p.ld_dyk : p.ld_dyq) : nullptr;
            const int64_t hsd = s ? p.hs_dyk : p.hs_dyq;
            T *y0 = (T *)(s ? p.yk : p.yq) + row * nh * p.D;
            Chunks<T, VEC, BWD> cur, next;
            next.load(x0, dy0, it);
            for (int h = 0; h < nh; ++h) {
                cur = next;
                const int hn = h + 1 < nh ? h + 1 : h;
                next.load(x0 + hn * hs, BWD ? dy0 + hn * hsd : nullptr, it);
                float v[2][VEC], g[2][VEC];
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    v[0][e] = it.ok ? (float)cur.x[0][e] : 0.f, v[1][e] = it.b >= 0 ? (float)cur.x[1][e] : 0.f;
                    if (BWD) g[0][e] = it.ok ? (float)cur.g[0][e] : 0.f, g[1][e] = it.b >= 0 ? (float)cur.g[1][e] : 0.f;
                    ss += v[0][e] * v[0][e] + v[1][e] * v[1][e];
                }
                ss = group_sum<GL>(ss);
                const float r = 1.f / sqrtf(ss * inv_d + p.eps);
                float dot = 0.f;
                if (BWD) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float a = g[0][e] * cs[e] + g[1][e] * sn[e];
                        const float b = g[1][e] * cs[e] - g[0][e] * sn[e];
                        dw[s][0][e] += a * v[0][e] * r;
                        dw[s][1][e] += b * v[1][e] * r;
                        g[0][e] = a * w[s][0][e];
                        g[1][e] = b * w[s][1][e];
                        dot += g[0][e] * v[0][e] + g[1][e] * v[1][e];
                    }
                    dot = group_sum<GL>(dot) * inv_d * r * r;
                }
                float o[2][VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (BWD) {
                        o[0][e] = r * (g[0][e] - v[0][e] * dot);
                        o[1][e] = r * (g[1][e] - v[1][e] * dot);
                    } else {
                        const float a = v[0][e] * r * w[s][0][e], b = v[1][e] * r * w[s][1][e];
                        o[0][e] = a * cs[e] - b * sn[e];
                        o[1][e] = b * cs[e] + a * sn[e];
                    }
                }
                magic::store_vec<T, VEC>(y0 + h * p.D + it.a, it.ok, o[0]);
                magic::store_vec<T, VEC>(y0 + h * p.D + it.b, it.b >= 0, o[1]);
            }
        }
    }
    if (BWD) {
        // the block's weight gradients: lanes of a wavefront that hold the same columns first (fixed tree), then the four
        // wavefronts in order
        __shared__ float red[2][128];
        red[threadIdx.x >> 7][threadIdx.x & 127] = 0.f;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
#pragma unroll
                        for (int o = 32; o >= GL; o >>= 1) dw[s][c][e] += __shfl_xor(dw[s][c][e], o, 64);
        for (int wv = 0; wv < 4; ++wv) {
            if ((int)(threadIdx.x >> 6) == wv && (threadIdx.x & 63) < GL) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            if (it.ok) red[s][it.a + e] += dw[s][0][e];
                            if (it.b >= 0) red[s][it.b + e] += dw[s][1][e];
                        }
            }
            __syncthreads();
        }
        for (int t = threadIdx.x; t < 2 * p.D; t += 256)
            p.partial[(int64_t)t * gridDim.x + blockIdx.x] = red[t / p.D][t % p.D];
    }
}

// column sums of the block partials, in double: a block per output column, fixed tree
__global__ __launch_bounds__(256) void k_head_norm_dw(const float *partial, int blocks, int D, float *dwq, float *dwk) {
    __shared__ double red[4];
    const int c = blockIdx.x;
    float x[MAX_BLOCKS / 256];
#pragma unroll
    for (int i = 0; i < MAX_BLOCKS / 256; ++i) {
        const int b = threadIdx.x + 256 * i;
        x[i] = b < blocks ? partial[(int64_t)c * blocks + b] : 0.f;
    }
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < MAX_BLOCKS / 256; ++i) s += (double)x[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = (red[0] + red[1]) + (red[2] + red[3]);
        if (c < D) dwq[c] = (float)s;
        else dwk[c - D] = (float)s;
    }
}

int rope_blocks(int64_t n, int gl) { return magic::stride_grid(n, 256 / gl, MAX_BLOCKS); }

template <typename T, int VEC, int GL> int run(const RopeArgs &p, bool bwd, hipStream_t st) {
    const int grid = rope_blocks(p.n, GL);
    if (bwd)
        MAGIC_LAUNCH("head_norm_rope_bwd", (k_head_norm<T, VEC, GL, true>), grid, 256, 0, st, p);
    else
        MAGIC_LAUNCH("head_norm_rope_fwd", (k_head_norm<T, VEC, GL, false>), grid, 256, 0, st, p);
    return magic::launch_status();
}

template <typename T, int VEC> int pick(const RopeArgs &p, bool bwd, hipStream_t st, int *gl_out) {
    const int items = p.half / VEC + ((p.D - 2 * p.half) / VEC + 1) / 2;
    int gl = 4;
    while (gl < items && gl < 64) gl *= 2;
    if (gl_out) {
        *gl_out = gl;
        return MAGIC_OK;
    }
    // (at most 64 items: single columns of heads of 128)
    switch (gl) {
        case 4: return run<T, VEC, 4>(p, bwd, st);
        case 8: return run<T, VEC, 8>(p, bwd, st);
        case 16: return run<T, VEC, 16>(p, bwd, st);
        case 32: return run<T, VEC, 32>(p, bwd, st);
        default: return run<T, VEC, 64>(p, bwd, st);
    }
}

bool mult(const void *p, int64_t ld, int64_t hs, int vec, int size) {
    return (uintptr_t)p % (size_t)(vec * size) == 0 && ld % vec == 0 && hs % vec == 0;
}

bool chunks(const RopeArgs &p, bool bwd, int vec, int size) {
    const bool ok = p.half % vec == 0 && p.D % vec == 0 && mult(p.q, p.ld_q, p.hs_q, vec, size) &&
                    mult(p.k, p.ld_k, p.hs_k, vec, size) && mult(p.yq, vec, vec, vec, size) && mult(p.yk, vec, vec, vec, size);
    return ok && (!bwd || (mult(p.dyq, p.ld_dyq, p.hs_dyq, vec, size) && mult(p.dyk, p.ld_dyk, p.hs_dyk, vec, size)));
}

// chunks of 16 (or 8) bytes wherever strides, widths and addresses allow them, single columns otherwise
int launch(const RopeArgs &p, int dtype, bool bwd, hipStream_t st, int *gl_out = nullptr) {
    if (dtype == MAGIC_F32)
        return chunks(p, bwd, 4, 4) ? pick<float, 4>(p, bwd, st, gl_out) : pick<float, 1>(p, bwd, st, gl_out);
    return chunks(p, bwd, 8, 2)   ? pick<magic::bf16_t, 8>(p, bwd, st, gl_out)
           : chunks(p, bwd, 4, 2) ? pick<magic::bf16_t, 4>(p, bwd, st, gl_out)
                                  : pick<magic::bf16_t, 1>(p, bwd, st, gl_out);
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
    return magic::align_up((size_t)MAX_BLOCKS * 2 * head_dim * sizeof(float)) + 256;
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
    p.partial = ar.take<float>((size_t)MAX_BLOCKS * 2 * head_dim);
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
    MAGIC_LAUNCH("head_norm_rope_dw", k_head_norm_dw, 2 * head_dim, 256, 0, stream, p.partial, grid, head_dim, dwq, dwk);
    return magic::launch_status();
}

}  // extern "C"
