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
#include "bf16_split.h"

namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// amax of a block (its bits as an unsigned number: magnitudes compare like integers, NaN above infinity) -> stored exponent
__device__ __forceinline__ int block_exp(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255;
    const int k = (int)(amax_bits >> 23);                        // biased exponent, 0 for subnormals and zero
    int e = k - 6;
    if ((amax_bits & 0x7fffffu) >= 0x7f0000u) ++e;               // mantissa >= 127.5 / 64: would round to 128
    return e < 1 ? 1 : e;
}

__device__ __forceinline__ int code_of(float x, int e) {         // e: stored exponent, 1 .. 249
    return (int)rintf(x * pow2f(127 - e));
}

__device__ __forceinline__ float scale_of(int e) { return e == 255 ? __uint_as_float(0x7fc00000u) : pow2f(e - 127); }

// eight lanes of four columns (VEC 4) or thirty-two of one (VEC 1) per block
template <int VEC>
__global__ __launch_bounds__(256) void k_act8_pack(int64_t n, int F, const float *x, int64_t ld_x, int8_t *codes,
                                                   int64_t ld_c, uint8_t *exps, int nb) {
    constexpr int LPB = 32 / VEC;
    const int64_t total = n * nb;
    const int l = threadIdx.x % LPB;
    for (int64_t b = (int64_t)blockIdx.x * (256 / LPB) + threadIdx.x / LPB; b < total;
         b += (int64_t)gridDim.x * (256 / LPB)) {
        const int64_t row = b / nb;
        const int blk = (int)(b - row * nb);
        const int c = blk * 32 + l * VEC;
        float v[VEC];
        uint32_t m = 0;
        if constexpr (VEC == 4) {
            f32x4_t t = c < F ? *reinterpret_cast<const f32x4_t *>(x + row * ld_x + c) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = t[e];
        } else {
            v[0] = c < F ? x[row * ld_x + c] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = LPB / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, LPB));
        const int ex = block_exp(m);
        if constexpr (VEC == 4) {
            uint32_t w = 0;
            if (ex != 255) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w |= ((uint32_t)code_of(v[e], ex) & 0xffu) << (8 * e);
            }
            if (c < ld_c) *reinterpret_cast<uint32_t *>(codes + row * ld_c + c) = w;
        } else {
            if (c < ld_c) codes[row * ld_c + c] = ex == 255 ? (int8_t)0 : (int8_t)code_of(v[0], ex);
        }
        if (l == 0) exps[b] = (uint8_t)ex;
    }
}

template <int VEC>
__global__ __launch_bounds__(256) void k_act8_unpack(int64_t n, int F, const int8_t *codes, int64_t ld_c,
                                                     const uint8_t *exps, int nb, float *x, int64_t ld_x) {
    const int fv = (F + VEC - 1) / VEC;
    const int64_t total = n * fv;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / fv;
        const int c = (int)(i - row * fv) * VEC;
        const float s = scale_of(exps[row * nb + c / 32]);
        if constexpr (VEC == 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + row * ld_c + c);
            f32x4_t t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = (float)(int8_t)(w >> (8 * e)) * s;
            *reinterpret_cast<f32x4_t *>(x + row * ld_x + c) = t;
        } else {
            x[row * ld_x + c] = (float)codes[row * ld_c + c] * s;
        }
    }
}

// dW[M,F] = dY[N,M]^T . Xhat[N,F]: a wavefront owns a 32 x 32 output tile and a strip of rows; three matrix products
// (dY in three bf16 pieces, Xhat in its only one) per 16 rows; the strips are added in order by k_act8_dw_reduce.
struct DwArgs {
    int64_t n;
    int M, F, nb;
    const float *dy;
    int64_t ld_dy;
    const int8_t *codes;
    int64_t ld_c;
    const uint8_t *exps;
    float *partial, *dw;
    int strips, ft;
    int64_t rows;  // of a strip, a multiple of 16
};

__global__ __launch_bounds__(64) void k_act8_dw(DwArgs a) {
    const int lane = threadIdx.x, li = lane & 31, hf = lane >> 5;
    const int m0 = (blockIdx.y / a.ft) * 32, f0 = (blockIdx.y % a.ft) * 32;
    const int64_t r0 = (int64_t)blockIdx.x * a.rows;
    const int64_t r1 = r0 + a.rows < a.n ? r0 + a.rows : a.n;
    const int mc = m0 + li < a.M ? m0 + li : 0, fc = f0 + li < a.F ? f0 + li : 0;
    float16_t acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    for (int64_t r = r0; r < r1; r += 16) {
        float y[8], x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t row = r + 8 * hf + u;
            const int64_t rc = row < a.n ? row : a.n - 1;
            const float dv = a.dy[rc * a.ld_dy + mc];
            const float xv = (float)a.codes[rc * a.ld_c + fc] * scale_of(a.exps[rc * a.nb + f0 / 32]);
            y[u] = row < r1 && m0 + li < a.M ? dv : 0.f;
            x[u] = row < r1 && f0 + li < a.F ? xv : 0.f;
        }
        magic::bf16x8_t y1, y2, y3, xb;
        magic::split8(make_float4(y[0], y[1], y[2], y[3]), make_float4(y[4], y[5], y[6], y[7]), y1, y2, y3);
#pragma unroll
        for (int u = 0; u < 8; ++u) xb[u] = (__bf16)x[u];
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y3, xb, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y2, xb, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y1, xb, acc, 0, 0, 0);
    }
    float *out = a.partial + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * 1024;
#pragma unroll
    for (int r = 0; r < 16; ++r) out[((r & 3) + 8 * (r >> 2) + 4 * hf) * 32 + li] = acc[r];
}

__global__ __launch_bounds__(256) void k_act8_dw_reduce(DwArgs a, int tiles) {
    const int e = blockIdx.x * 256 + threadIdx.x, tile = blockIdx.y;
    const int i = (tile / a.ft) * 32 + (e >> 5), j = (tile % a.ft) * 32 + (e & 31);
    if (i >= a.M || j >= a.F) return;
    float s = 0.f;
    for (int k = 0; k < a.strips; ++k) s += a.partial[((int64_t)k * tiles + tile) * 1024 + e];
    a.dw[(int64_t)i * a.F + j] = s;
}

struct DwPlan {
    int strips, mt, ft;
    int64_t rows;
    size_t floats;
};
DwPlan plan(int64_t n, int M, int F) {
    DwPlan p;
    p.mt = (M + 31) / 32, p.ft = (F + 31) / 32;
    int64_t strips = 4096 / ((int64_t)p.mt * p.ft);
    if (strips < 1) strips = 1;
    int64_t rows = (n + strips - 1) / strips;
    if (rows < 128) rows = 128;
    p.rows = (rows + 15) / 16 * 16;
    p.strips = (int)((n + p.rows - 1) / p.rows);
    p.floats = (size_t)p.strips * p.mt * p.ft * 1024;
    return p;
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
    if (n_cols % 4 == 0 && ld_x % 4 == 0 && (uintptr_t)x % 16 == 0)
        MAGIC_LAUNCH("act8_pack", k_act8_pack<4>, magic::stride_grid(n_rows * nb, 32), 256, 0, (hipStream_t)stream, n_rows,
                     n_cols, x, ld_x, codes, ld_c, exps, nb);
    else
        MAGIC_LAUNCH("act8_pack", k_act8_pack<1>, magic::stride_grid(n_rows * nb, 8), 256, 0, (hipStream_t)stream, n_rows,
                     n_cols, x, ld_x, codes, ld_c, exps, nb);
    return magic::launch_status();
}

int magic_act8_unpack(int64_t n_rows, int32_t n_cols, const int8_t *codes, const uint8_t *exps, float *x, int64_t ld_x,
                      void *stream) {
    if (n_rows < 0 || n_cols <= 0) return MAGIC_ERR_INVALID_ARG;
    if (n_rows == 0) return MAGIC_OK;
    if (!x || !codes || !exps || ld_x < n_cols || (uintptr_t)codes % 16) return MAGIC_ERR_INVALID_ARG;
    const int nb = (n_cols + 31) / 32;
    const int64_t ld_c = magic_act8_code_stride(n_cols);
    if (n_cols % 4 == 0 && ld_x % 4 == 0 && (uintptr_t)x % 16 == 0)
        MAGIC_LAUNCH("act8_unpack", k_act8_unpack<4>, magic::stride_grid(n_rows * (n_cols / 4), 256, 4096), 256, 0,
                     (hipStream_t)stream, n_rows, n_cols, codes, ld_c, exps, nb, x, ld_x);
    else
        MAGIC_LAUNCH("act8_unpack", k_act8_unpack<1>, magic::stride_grid(n_rows * n_cols, 256, 4096), 256, 0,
                     (hipStream_t)stream, n_rows, n_cols, codes, ld_c, exps, nb, x, ld_x);
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
    DwPlan p = plan(n_rows, m, f);
    DwArgs a;
    a.n = n_rows, a.M = m, a.F = f, a.nb = (f + 31) / 32;
    a.dy = dy, a.ld_dy = ld_dy, a.codes = codes, a.ld_c = magic_act8_code_stride(f), a.exps = exps;
    a.dw = dw, a.ft = p.ft, a.rows = p.rows, a.strips = n_rows > 0 ? p.strips : 0;
    a.partial = nullptr;
    const int tiles = p.mt * p.ft;
    if (n_rows > 0) {
        magic::Arena ar(workspace, workspace_bytes);
        a.partial = ar.take<float>(p.floats);
        if (!ar.ok() || !a.partial) return MAGIC_ERR_WORKSPACE;
        MAGIC_LAUNCH("act8_weight_grad", k_act8_dw, dim3(p.strips, tiles), 64, 0, stream, a);
    }
    MAGIC_LAUNCH("act8_weight_grad_reduce", k_act8_dw_reduce, dim3(4, tiles), 256, 0, stream, a, tiles);
    return magic::launch_status();
}

}  // extern "C"
