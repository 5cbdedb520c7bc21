// Activations kept for the backward pass in 8 bits (magic_act8_*): blocks of 32 columns of a row share a power-of-two
// scale, x ~ code * 2^(exp - 127) with a signed 8-bit code.
//   e    = floor(log2 amax) - 6, one more where amax 2^-e would round to 128, never below -126
//   code = round_to_nearest_even(x 2^-e), |code| <= 127
// Every step is exact but the one rounding (half a step, 2^(e-1)), so a code does not depend on how it is computed.
// A power of two costs up to one of the eight bits against amax / 127, but code * 2^e has at most seven significant
// bits: it IS a bf16 value, and the weight gradient takes it as ONE plane of a split-bf16 product (three matrix
// instructions instead of six).  exp = 255 marks a block that held an infinity or a NaN: it reads back as NaN, so a
// diverging run is not silently repaired.
#include "common.h"
#include "attn_common.h"
#include "act8.h"

namespace {

using magic::bf16_t;
using magic::bf16x8_t;
using magic::attn::f32x16_t;
using magic::attn::f32x4_t;

using magic::act8::block_exp;
using magic::act8::codes4;
using magic::act8::pow2f;

__device__ __forceinline__ float scale_of(int e) { return e == 255 ? __uint_as_float(0x7fc00000u) : pow2f(e - 127); }

// four floats at any address; the hardware reads and writes them in one access as long as it is a whole float's
typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));

// columns c .. c + 3 of a row of F >= 4, zeros behind the last: the last ones are read with what is before them
__device__ __forceinline__ f32x4_t row_end(const float *p, int c, int F) {
    const int at = min(c, F - 4), s = c - at;
    const f32x4u_t t = *reinterpret_cast<const f32x4u_t *>(p + at);
    f32x4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = s == 0 ? t[e] : 0.f;
#pragma unroll
        for (int k = 1; e + k < 4; ++k) v[e] = s == k ? t[e + k] : v[e];
    }
    return v;
}

// VEC 8: four lanes a block, two float4 each (ODD: rows that are not whole aligned float4s); VEC 1: thirty-two lanes, for
// less than four columns.  U blocks a thread are in flight together.  I: index type of a block (a 64-bit division costs
// as much as the rest).  HBM-bound: 97,000 x 1,024 in 125 us, 4.0 TB/s.
template <int VEC, bool ODD, typename I>
__global__ __launch_bounds__(256) void k_act8_pack(I total, int F, const float *x, int64_t ld_x, int8_t *codes,
                                                   int64_t ld_c, uint8_t *exps, I nb) {
    constexpr int LPB = 32 / VEC, U = 4;
    constexpr I PER = 256 / LPB;
    const int l = threadIdx.x % LPB;
    for (I b0 = (I)blockIdx.x * (U * PER) + threadIdx.x / LPB; b0 < total; b0 += (I)gridDim.x * (U * PER)) {
        float v[U][VEC];
        int64_t at[U];      // code of the first column
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const I b = b0 + u * PER < total ? b0 + u * PER : total - 1;
            const I row = b / nb;
            c[u] = (int)(b - row * nb) * 32 + l * VEC;
            at[u] = (int64_t)row * ld_c + c[u];
            const float *p = x + (int64_t)row * ld_x;
            if constexpr (VEC == 8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool in = c[u] + 4 * h < F;
                    f32x4_t t;
                    if constexpr (ODD)
                        t = row_end(p, c[u] + 4 * h, F);
                    else
                        t = *reinterpret_cast<const f32x4_t *>(p + (in ? c[u] + 4 * h : 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][4 * h + e] = ODD || in ? t[e] : 0.f;
                }
            } else {
                v[u][0] = c[u] < F ? p[c[u]] : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const I b = b0 + u * PER;
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(v[u][e]) & 0x7fffffffu);
#pragma unroll
            for (int o = LPB / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, LPB));
            if (b >= total) continue;          // (whole blocks: the lanes of one agree)
            const int ex = block_exp(m);
            if constexpr (VEC == 8) {
                const uint2 w = make_uint2(codes4(v[u][0], v[u][1], v[u][2], v[u][3], ex),
                                           codes4(v[u][4], v[u][5], v[u][6], v[u][7], ex));
                if (c[u] < ld_c) *reinterpret_cast<uint2 *>(codes + at[u]) = w;
            } else {
                if (c[u] < ld_c) codes[at[u]] = (int8_t)codes4(v[u][0], 0.f, 0.f, 0.f, ex);
            }
            if (l == 0) exps[b] = (uint8_t)ex;
        }
    }
}

// Four columns a thread.  97,000 x 1,024 in 90 us, 5.5 TB/s.
template <bool ODD>
__global__ __launch_bounds__(256) void k_act8_unpack(int64_t n, int F, const int8_t *codes, int64_t ld_c,
                                                     const uint8_t *exps, int nb, float *x, int64_t ld_x) {
    const int fv = (F + 3) / 4;
    const int64_t total = n * fv;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / fv;
        const int c = (int)(i - row * fv) * 4;
        const float s = scale_of(exps[row * nb + c / 32]);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + row * ld_c + c);
        f32x4_t t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (float)(int8_t)(w >> (8 * e)) * s;
        float *q = x + row * ld_x + c;
        if (!ODD) {
            *reinterpret_cast<f32x4_t *>(q) = t;
        } else if (c + 4 <= F) {
            *reinterpret_cast<f32x4u_t *>(q) = t;
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (c + e < F) q[e] = t[e];
        }
    }
}

// dW[M,F] = dY[N,M]^T . Xhat[N,F].  Few operations a byte at the entity-level shapes: a block of four wavefronts owns an output tile as
// large as its registers hold (64 x 192 covers the whole of the THEIA-shaped decoder input: each operand is read once) and
// a strip of the rows.  Steps of 32 rows: dY split into three bf16 planes and the codes turned into their one bf16 value go
// row-major to LDS, where transposed reads deliver eight rows of a column; three 32x32x16 products a tile and 16 rows.  The
// next step's rows are loaded under the products.  The strips' tiles are added in order by k_act8_dw_reduce.  700,000 rows,
// 64 x 192: 114 us, 2.8 TB/s (the split of dY and its LDS traffic beside the loads), and 11 us to add 768 strips.
struct DwArgs {
    int64_t n;
    int M, F, nb;
    const float *dy;
    int64_t ld_dy;
    const int8_t *codes;
    int64_t ld_c;
    const uint8_t *exps;
    float *partial, *dw;
    int strips, mt, ft;   // tiles along M and F
    int64_t rows;         // of a strip, a multiple of STEP
};

constexpr int STEP = 32, NT = 256;

// tile: TM = 64 MB rows of dW (two wavefronts of 32 MB), 64 FB columns (two of 32 FB)
template <int MB, int FB, bool ALIGNED> __global__ __launch_bounds__(NT, MB *FB > 4 ? 2 : 3) void k_act8_dw(DwArgs a) {
    constexpr int TM = 64 * MB, TF = 64 * FB;
    typedef magic::attn::Tile<magic::attn::F32x3, TM, STEP> ytile;
    typedef magic::attn::Tile<magic::attn::BF16, 64, STEP> xtile;        // FB of them side by side
    constexpr int YN = STEP * TM / 8 / NT, XC = STEP * TF / 8, XN = (XC + NT - 1) / NT;
    __shared__ __align__(16) bf16_t sy[3 * ytile::PLANE], sx[FB * xtile::PLANE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int wm = wave & 1, wf = wave >> 1;
    const int m0 = (int)(blockIdx.y / a.ft) * TM, f0 = (int)(blockIdx.y % a.ft) * TF;
    const int64_t r0 = (int64_t)blockIdx.x * a.rows, r1 = min(r0 + a.rows, a.n);
    f32x16_t acc[MB][FB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    float y[YN][8];
    uint64_t x[XN];
    uint8_t ex[XN];
    auto load = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < YN; ++i) {
            const int c = tid + i * NT, col = m0 + (c % (TM / 8)) * 8;
            const int64_t row = min(r + c / (TM / 8), a.n - 1);
            const float *p = a.dy + row * a.ld_dy;
            if (ALIGNED) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p + (col + 4 * h < a.M ? col + 4 * h : 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[i][4 * h + e] = v[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = p[col + e < a.M ? col + e : 0];
            }
        }
#pragma unroll
        for (int i = 0; i < XN; ++i) {
            const int c = min(tid + i * NT, XC - 1), col = f0 + (c % (TF / 8)) * 8;
            const int64_t row = min(r + c / (TF / 8), a.n - 1);
            const int cc = col < a.ld_c ? col : 0;
            x[i] = *reinterpret_cast<const uint64_t *>(a.codes + row * a.ld_c + cc);
            ex[i] = a.exps[row * a.nb + cc / 32];
        }
    };
    auto store = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < YN; ++i) {
            const int c = tid + i * NT, row = c / (TM / 8), col = m0 + (c % (TM / 8)) * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = r + row < r1 && col + e < a.M ? y[i][e] : 0.f;
            bf16x8_t p[3];
            magic::attn::to_planes(v, p);
#pragma unroll
            for (int k = 0; k < 3; ++k)
                *reinterpret_cast<bf16x8_t *>(sy + k * ytile::PLANE + ytile::at(row, c % (TM / 8))) = p[k];
        }
#pragma unroll
        for (int i = 0; i < XN; ++i) {
            const int c = tid + i * NT;
            if (XC % NT != 0 && c >= XC) break;
            const int row = c / (TF / 8), cx = c % (TF / 8);
            const bool ok = r + row < r1 && f0 + cx * 8 < a.ld_c;
            const float s = ok ? scale_of(ex[i]) : 0.f;
            bf16x8_t v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (bf16_t)((float)(int8_t)(x[i] >> (8 * e)) * s);      // (exact)
            *reinterpret_cast<bf16x8_t *>(sx + (cx / 8) * xtile::PLANE + xtile::at(row, cx % 8)) = v;
        }
    };
    const uint32_t ty = ytile::lane_turned(lane), tx = xtile::lane_turned(lane);
    if (r0 < r1) load(r0);
    for (int64_t r = r0; r < r1; r += STEP) {
        __syncthreads();
        store(r);
        __syncthreads();
        if (r + STEP < r1) load(r + STEP);
#pragma unroll
        for (int k = 0; k < STEP / 16; ++k) {
            bf16x8_t fx[FB][1];
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                const int t = wf * FB + j;         // of the tile's 2 FB column blocks of 32
                xtile::frag_t(sx + (t >> 1) * xtile::PLANE, tx ^ (uint32_t)(64 * (t & 1)), 16 * k, 0, fx[j]);
            }
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                bf16x8_t fy[3];
                ytile::frag_t(sy, ty ^ (uint32_t)(64 * (wm * MB)), 16 * k, i, fy);
#pragma unroll
                for (int j = 0; j < FB; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fy[2], fx[j][0], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fy[1], fx[j][0], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fy[0], fx[j][0], acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    float *out = a.partial + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * (TM * TF);
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                out[((wm * MB + i) * 32 + (r & 3) + 8 * (r >> 2) + 4 * hf) * TF + (wf * FB + j) * 32 + li] = acc[i][j][r];
}

// dW from the strips' tiles: 64 consecutive elements a block, its sixteen wavefronts take the strips in turn (strip order
// within each, eight loads in flight) and are added in order
__global__ __launch_bounds__(1024) void k_act8_dw_reduce(DwArgs a, int TM, int TF) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, tile = blockIdx.y, tiles = gridDim.y;
    const int e = blockIdx.x * 64 + lane;
    const int64_t stride = (int64_t)tiles * TM * TF;
    const float *p = a.partial + (int64_t)tile * TM * TF + e;
    float s = 0.f;
    int k = w;
    for (; k + 7 * 16 < a.strips; k += 8 * 16) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = p[(k + 16 * u) * stride];
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; k < a.strips; k += 16) s += p[k * stride];
    red[w][lane] = s;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    const int i = (tile / a.ft) * TM + e / TF, j = (tile % a.ft) * TF + e % TF;
    if (i < a.M && j < a.F) a.dw[(int64_t)i * a.F + j] = s;
}

struct DwPlan {
    int mb, fb, mt, ft, strips;
    int64_t rows;
    size_t floats;
};
// The output tile that reads the least: dY once for every tile column, the codes once for every tile row.
DwPlan plan(int64_t n, int M, int F) {
    static const int cand[][2] = {{1, 1}, {1, 2}, {1, 3}, {2, 2}, {2, 3}, {2, 4}};
    DwPlan p;
    double best = -1.0;
    for (auto &c : cand) {
        const int mt = (M + 64 * c[0] - 1) / (64 * c[0]), ft = (F + 64 * c[1] - 1) / (64 * c[1]);
        const double cost = 4.0 * ft * (mt * 64.0 * c[0]) + 1.03 * mt * (ft * 64.0 * c[1]);
        if (best < 0 || cost < best) best = cost, p.mb = c[0], p.fb = c[1], p.mt = mt, p.ft = ft;
    }
    const int64_t tiles = (int64_t)p.mt * p.ft, tile = (int64_t)p.mb * p.fb * 4096;
    int64_t strips = 768 / tiles;                       // three resident blocks a CU
    const int64_t fit = (64 << 20) / (tiles * tile);    // at most 256 MB of partial tiles
    if (strips > fit) strips = fit;
    if (strips < 1) strips = 1;
    int64_t rows = (n + strips - 1) / strips;
    if (rows < 4 * STEP) rows = 4 * STEP;
    p.rows = (rows + STEP - 1) / STEP * STEP;
    p.strips = (int)((n + p.rows - 1) / p.rows);
    p.floats = (size_t)p.strips * tiles * tile;
    return p;
}

template <int MB, int FB> int run_dw(const DwArgs &a, hipStream_t stream) {
    const dim3 grid(a.strips, a.mt * a.ft);
    if (a.M % 4 == 0 && a.ld_dy % 4 == 0 && (uintptr_t)a.dy % 16 == 0)
        MAGIC_LAUNCH("act8_weight_grad", (k_act8_dw<MB, FB, true>), grid, NT, 0, stream, a);
    else
        MAGIC_LAUNCH("act8_weight_grad", (k_act8_dw<MB, FB, false>), grid, NT, 0, stream, a);
    return magic::launch_status();
}

template <int VEC, bool ODD>
int run_pack(int64_t total, int F, const float *x, int64_t ld_x, int8_t *codes, int64_t ld_c, uint8_t *exps, int nb, hipStream_t st) {
    const int grid = magic::stride_grid(total, VEC == 8 ? 256 : 32);
    if (total < (1 << 30))
        MAGIC_LAUNCH("act8_pack", (k_act8_pack<VEC, ODD, uint32_t>), grid, 256, 0, st, (uint32_t)total, F, x, ld_x, codes, ld_c, exps, (uint32_t)nb);
    else
        MAGIC_LAUNCH("act8_pack", (k_act8_pack<VEC, ODD, int64_t>), grid, 256, 0, st, total, F, x, ld_x, codes, ld_c, exps, (int64_t)nb);
    return magic::launch_status();
}

}  // namespace

extern "C" {

int64_t magic_act8_code_stride(int32_t n_cols) { return n_cols <= 0 ? 0 : ((int64_t)n_cols + 15) / 16 * 16; }

int magic_act8_pack(int64_t n_rows, int32_t n_cols, const float *x, int64_t ld_x, int8_t *codes, uint8_t *exps,
                    void *stream) {
    if (n_rows < 0 || n_cols <= 0) return MAGIC_ERR_INVALID_ARG;
    if (n_rows == 0) return MAGIC_OK;
    if (!x || !codes || !exps || ld_x < n_cols || (uintptr_t)codes % 16) return MAGIC_ERR_INVALID_ARG;
    const int nb = (n_cols + 31) / 32;
    const int64_t ld_c = magic_act8_code_stride(n_cols);
    hipStream_t st = (hipStream_t)stream;
    const int64_t total = n_rows * nb;
    const bool vec = n_cols % 4 == 0 && ld_x % 4 == 0 && (uintptr_t)x % 16 == 0;
    if (n_cols < 4) return run_pack<1, false>(total, n_cols, x, ld_x, codes, ld_c, exps, nb, st);
    return vec ? run_pack<8, false>(total, n_cols, x, ld_x, codes, ld_c, exps, nb, st)
               : run_pack<8, true>(total, n_cols, x, ld_x, codes, ld_c, exps, nb, st);
}

int magic_act8_unpack(int64_t n_rows, int32_t n_cols, const int8_t *codes, const uint8_t *exps, float *x, int64_t ld_x,
                      void *stream) {
    if (n_rows < 0 || n_cols <= 0) return MAGIC_ERR_INVALID_ARG;
    if (n_rows == 0) return MAGIC_OK;
    if (!x || !codes || !exps || ld_x < n_cols || (uintptr_t)codes % 16) return MAGIC_ERR_INVALID_ARG;
    const int nb = (n_cols + 31) / 32;
    const int64_t ld_c = magic_act8_code_stride(n_cols);
    const int grid = magic::stride_grid(n_rows * ((n_cols + 3) / 4), 256, 4096);
    if (n_cols % 4 == 0 && ld_x % 4 == 0 && (uintptr_t)x % 16 == 0)
        MAGIC_LAUNCH("act8_unpack", k_act8_unpack<false>, grid, 256, 0, (hipStream_t)stream, n_rows, n_cols, codes, ld_c, exps, nb, x, ld_x);
    else
        MAGIC_LAUNCH("act8_unpack", k_act8_unpack<true>, grid, 256, 0, (hipStream_t)stream, n_rows, n_cols, codes, ld_c, exps, nb, x, ld_x);
    return magic::launch_status();
}

size_t magic_act8_weight_grad_workspace_bytes(int64_t n_rows, int32_t m, int32_t f) {
    if (n_rows <= 0 || m <= 0 || f <= 0) return 256;
    return magic::align_up(plan(n_rows, m, f).floats * sizeof(float)) + 256;
}

int magic_act8_weight_grad(int64_t n_rows, int32_t m, int32_t f, const float *dy, int64_t ld_dy, const int8_t *codes,
                           const uint8_t *exps, float *dw, void *workspace, size_t workspace_bytes, void *stream_) {
    if (n_rows < 0 || m <= 0 || f <= 0 || !dw) return MAGIC_ERR_INVALID_ARG;
    if (n_rows > 0 && (!dy || !codes || !exps || ld_dy < m || (uintptr_t)codes % 16)) return MAGIC_ERR_INVALID_ARG;
    hipStream_t stream = (hipStream_t)stream_;
    const DwPlan p = plan(n_rows, m, f);
    if ((int64_t)p.mt * p.ft > 65535) return MAGIC_ERR_UNSUPPORTED;
    DwArgs a;
    a.n = n_rows, a.M = m, a.F = f, a.nb = (f + 31) / 32;
    a.dy = dy, a.ld_dy = ld_dy, a.codes = codes, a.ld_c = magic_act8_code_stride(f), a.exps = exps;
    a.dw = dw, a.mt = p.mt, a.ft = p.ft, a.rows = p.rows, a.strips = n_rows > 0 ? p.strips : 0;
    a.partial = nullptr;
    if (n_rows > 0) {
        magic::Arena ar(workspace, workspace_bytes);
        a.partial = ar.take<float>(p.floats);
        if (!ar.ok() || !a.partial) return MAGIC_ERR_WORKSPACE;
        const int st = p.mb == 1 ? (p.fb == 1   ? run_dw<1, 1>(a, stream)
                                    : p.fb == 2 ? run_dw<1, 2>(a, stream)
                                                : run_dw<1, 3>(a, stream))
                                 : (p.fb == 2   ? run_dw<2, 2>(a, stream)
                                    : p.fb == 3 ? run_dw<2, 3>(a, stream)
                                                : run_dw<2, 4>(a, stream));
        if (st != MAGIC_OK) return st;
    }
    const int TM = 64 * p.mb, TF = 64 * p.fb;
    MAGIC_LAUNCH("act8_weight_grad_reduce", k_act8_dw_reduce, dim3(TM * TF / 64, p.mt * p.ft), 1024, 0, stream, a, TM, TF);
    return magic::launch_status();
}

}  // extern "C"
