// Building blocks of the segment-attention kernels (attn_fwd.hip, attn_bwd.hip).
//
// All products run on v_mfma_f32_32x32x16_bf16 and _f16.  float32 operands are split into three bf16 planes and take the six
// leading cross products (bf16_split.h: fp32-grade) or, scaled, into two fp16 planes and three products (F16x2 below);
// bfloat16 operands are one plane and one product.
// Lane l of a wavefront, li = l & 31, hf = l >> 5:
//   A [32 x 16]: row li, columns 8 hf .. + 7        B [16 x 32]: rows 8 hf .. + 7, column li
//   C [32 x 32]: column li, rows 8 (r / 4) + 4 hf + (r & 3), r = 0 .. 15
// The 16 rows of a product's inner dimension may come in any order as long as A and B agree, so the accumulators of one
// product serve as the B operand of the next without leaving their registers: registers 8 s .. 8 s + 7 of a C tile are
// the inner rows {4 hf + j, 8 + 4 hf + j}, j < 4, of its 16-row slice s.  The other operand of that product is the
// transpose of a tile that lies row-major in LDS; ds_read_tr16_b64 delivers it: the 16 lanes of a group name a 4 x 16
// block (lane i: row i / 4, columns 4 (i & 3) .. + 3) and lane i receives column i of it.
#pragma once
#include "common.h"
#include "bf16_split.h"
#include "lowp.h"

namespace magic {
namespace attn {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f;

// How operands become matrix operands (16-bit planes):
//   F32x3  float32 as three bf16 pieces, six products; exact pieces for any magnitude
//   F16x2  float32 times a power of two as two fp16 pieces, three products (hi hi, hi lo, lo hi).  22 bits: with the
//          operand's largest magnitude brought to [2^13, 2^14) a value keeps its error below 2^-22 relative or 2^-39 of
//          that largest magnitude, whichever is more; what the dropped lo lo takes away is below 2^-22 of a product.
//          Serves where the rows' magnitudes lie within 2^14 of each other (`Ranges`); F32x3 serves the rest.
//   BF16   bfloat16, one plane, one product
struct F32x3 {
    typedef float T;
    typedef bf16x8_t vec;
    static constexpr int N = 3;
    static constexpr bool SCALED = false;
};
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
struct F16x2 {
    typedef float T;
    typedef f16x8_t vec;
    static constexpr int N = 2;
    static constexpr bool SCALED = true;
};
struct BF16 {
    typedef bf16_t T;
    typedef bf16x8_t vec;
    static constexpr int N = 1;
    static constexpr bool SCALED = false;
};

__device__ __forceinline__ void split_f16(const float (&x)[8], f16x8_t (&p)[2]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2_t v = {x[2 * j], x[2 * j + 1]};
        const f16x2_t h = __builtin_convertvector(v, f16x2_t);
        f32x2_t r;          // v - h, the half read in place (the compiler converts it first)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(h), "v"(v[0]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(h), "v"(v[1]));
        const f16x2_t l = __builtin_convertvector(r, f16x2_t);
        p[0][2 * j] = h[0], p[0][2 * j + 1] = h[1];
        p[1][2 * j] = l[0], p[1][2 * j + 1] = l[1];
    }
}

// eight float32 values -> operand planes
__device__ __forceinline__ void to_planes(const float (&x)[8], bf16x8_t (&p)[3]) {
    split8(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), p[0], p[1], p[2]);
}
__device__ __forceinline__ void to_planes(const float (&x)[8], f16x8_t (&p)[2]) { split_f16(x, p); }
__device__ __forceinline__ void to_planes(const float (&x)[8], bf16x8_t (&p)[1]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[0][e] = (bf16_t)x[e];
}

// eight consecutive elements of an operand row as they lie in memory
template <typename T> struct Raw;
template <> struct Raw<float> {
    f32x4_t a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = *reinterpret_cast<const f32x4_t *>(p);
        b = *reinterpret_cast<const f32x4_t *>(p + 4);
    }
    __device__ __forceinline__ void store(float *p) const {
        *reinterpret_cast<f32x4_t *>(p) = a;
        *reinterpret_cast<f32x4_t *>(p + 4) = b;
    }
    __device__ __forceinline__ void zero() { a = b = f32x4_t{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void planes(bf16x8_t (&p)[3], float) const {
        split8(make_float4(a[0], a[1], a[2], a[3]), make_float4(b[0], b[1], b[2], b[3]), p[0], p[1], p[2]);
    }
    __device__ __forceinline__ void planes(f16x8_t (&p)[2], float scale) const {
        const float x[8] = {a[0] * scale, a[1] * scale, a[2] * scale, a[3] * scale,
                            b[0] * scale, b[1] * scale, b[2] * scale, b[3] * scale};
        split_f16(x, p);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    }
};
template <> struct Raw<bf16_t> {
    bf16x8_t v;
    __device__ __forceinline__ void load(const bf16_t *p) { v = *reinterpret_cast<const bf16x8_t *>(p); }
    __device__ __forceinline__ void store(bf16_t *p) const { *reinterpret_cast<bf16x8_t *>(p) = v; }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (bf16_t)0.f;
    }
    __device__ __forceinline__ void planes(bf16x8_t (&p)[1], float) const { p[0] = v; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    }
};

struct RawF16 {
    f16x8_t h, l;
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = l[e] = (_Float16)0.f;
    }
    __device__ __forceinline__ void planes(f16x8_t (&p)[2]) const { p[0] = h, p[1] = l; }
};

// Rows of one head that a kernel stages tile by tile.  F16x2 rows come split, scaled and with the rows that take no part
// as zeros, from the pass that prepares them (a tile's rows are staged once for every 128 rows of the other side).
template <typename M> struct Src {
    typedef typename M::T T;
    struct raw : Raw<T> {
        __device__ __forceinline__ void planes(typename M::vec (&p)[M::N]) const { Raw<T>::planes(p, 1.f); }
    };
    static constexpr bool READY = false;
    const T *p;
    int64_t ld;
    __device__ __forceinline__ Src from(int64_t row) const { return {p + row * ld, ld}; }
    __device__ __forceinline__ void load(raw &r, uint32_t off) const {
        r.load(reinterpret_cast<const T *>(reinterpret_cast<const char *>(p) + off * (uint32_t)sizeof(T)));
    }
};
template <> struct Src<F16x2> {
    typedef RawF16 raw;
    static constexpr bool READY = true;
    const _Float16 *p;
    int64_t ld, lo;      // lo: from a high piece to its low one
    __device__ __forceinline__ Src from(int64_t row) const { return {p + row * ld, ld, lo}; }
    __device__ __forceinline__ void load(raw &r, uint32_t off) const {
        const char *b = reinterpret_cast<const char *>(p);
        r.h = *reinterpret_cast<const f16x8_t *>(b + off * 2u);
        r.l = *reinterpret_cast<const f16x8_t *>(b + 2 * lo + off * 2u);
    }
};
// planes of one operand in the workspace: [hi | lo][rows][heads][D]
struct PlaneSet {
    const _Float16 *p;
    int64_t rows;
    int heads;
};
template <typename M>
__device__ __forceinline__ Src<M> src_of(const void *p, int64_t ld, int64_t hs, const PlaneSet &s, int64_t row, int h, int D) {
    if constexpr (M::SCALED)
        return Src<M>{s.p + (row * s.heads + h) * D, (int64_t)s.heads * D, s.rows * s.heads * D};
    else
        return Src<M>{(const typename M::T *)p + row * ld + h * hs, ld};
}

__device__ __forceinline__ void mma(f32x16_t &c, const bf16x8_t (&a)[3], const bf16x8_t (&b)[3]) {
    mfma_split6(c, a[0], a[1], a[2], b[0], b[1], b[2]);
}
__device__ __forceinline__ void mma(f32x16_t &c, const f16x8_t (&a)[2], const f16x8_t (&b)[2]) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16_t &c, const bf16x8_t (&a)[1], const bf16x8_t (&b)[1]) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}

// The same sums in the same order with the operands' parts exchanged: scores of rows by keys come out bit for bit like those
// of keys by rows, and so do the probabilities that the sweeps rebuild from them.
__device__ __forceinline__ void mma_turned(f32x16_t &c, const bf16x8_t (&a)[3], const bf16x8_t (&b)[3]) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ void mma_turned(f32x16_t &c, const f16x8_t (&a)[2], const f16x8_t (&b)[2]) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ void mma_turned(f32x16_t &c, const bf16x8_t (&a)[1], const bf16x8_t (&b)[1]) { mma(c, a, b); }

// Order of a run of matrix instructions and the LDS reads that feed them: STEPS steps of READS reads and MFMAS
// instructions, the reads of AHEAD steps before the first.  (Left alone, the compiler reads, waits and multiplies in turn:
// a trip to the LDS before every product.)
template <int READS, int MFMAS, int STEPS, int AHEAD = 2> __device__ __forceinline__ void feed() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
        if (i + AHEAD < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
}
template <typename M> constexpr int PRODUCTS = M::N == 3 ? 6 : M::N == 2 ? 3 : 1;

// A tile of ROWS operand rows in LDS: planes of [ROWS][W] 16-bit values.  The 16-byte chunks of a row are permuted by its
// number (swz): sixteen rows at one column range, what a plain fragment reads, and four rows at a 64-byte range, what a
// transposed one reads, then lie on different banks (padded rows serve only one of the two: 45 % of the LDS cycles at
// 128 columns were conflicts).
template <typename M, int DP, int ROWS> struct Tile {
    typedef typename M::vec vec;
    static constexpr int NP = M::N;
    static constexpr int W = DP < 32 ? 32 : DP;      // a transposed read covers 32 columns
    static constexpr int PLANE = ROWS * W;
    static constexpr size_t BYTES = (size_t)NP * PLANE * 2;

    static __device__ __forceinline__ int swz(int row) {
        return W == 128  ? ((row & 3) << 2) | ((row >> 2) & 3)
               : W == 64 ? ((row & 2) << 1) | ((row >> 2) & 3)
                         : (row >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * W + (chunk ^ swz(row)) * 8; }

    // A lane's byte offsets: the plain fragment of rows 0 .. 31 at columns 0 .. 15, and the transposed one of rows 0 .. 15 at
    // columns 0 .. 31.  Further columns flip bits of them (a chunk is 16 bytes and a row a power of two), further rows
    // (multiples of 16) and planes are added.
    static __device__ __forceinline__ uint32_t lane_plain(int lane) { return 2u * at(lane & 31, lane >> 5); }
    static __device__ __forceinline__ uint32_t lane_turned(int lane) {
        return 2u * (at(4 * (lane >> 5) + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 4 * (lane & 1));
    }
    // columns 16 ks .. + 15 of rows r0 .. r0 + 31
    static __device__ __forceinline__ void frag(const bf16_t *t, uint32_t plain, int r0, int ks, vec (&f)[NP]) {
        const char *q = reinterpret_cast<const char *>(t) + (plain ^ (uint32_t)(32 * ks));
#pragma unroll
        for (int p = 0; p < NP; ++p) f[p] = *reinterpret_cast<const vec *>(q + 2 * (p * PLANE + r0 * W));
    }
    // transpose of rows r0 .. r0 + 15, columns 32 d .. + 31, inner order as described above
    static __device__ __forceinline__ void frag_t(const bf16_t *t, uint32_t turned, int r0, int d, vec (&f)[NP]) {
        const char *q = reinterpret_cast<const char *>(t) + (turned ^ (uint32_t)(64 * d));
        const char *q8 = reinterpret_cast<const char *>(t) + (turned ^ (uint32_t)(64 * d + 32));
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            typedef __attribute__((address_space(3))) s16x4_t *lds_ptr;
            union {
                s16x4_t s[2];
                vec h;
            } u;
            u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q + 2 * (p * PLANE + r0 * W)));
            u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q8 + 2 * (p * PLANE + (r0 + 8) * W)));
            f[p] = u.h;
        }
    }
};
// Keeps what is formed from x inside the loop: dozens of addresses would be held in registers instead of one flip each
__device__ __forceinline__ void stay(uint32_t &x) { asm volatile("" : "+v"(x)); }

// Staging of a tile by NT threads: rows of DP columns (zeros behind D) in chunks of eight elements.  A chunk's place is a
// 32-bit offset (MAX_LD bounds it) from the tile's first row, which is the same for all threads.
constexpr int64_t MAX_LD = 1 << 22;
constexpr int MAX_HEADS = 8192;               // grids' second dimension
constexpr int64_t MAX_ROWS = 0x7fff0000;      // a tile past the last row still has a 32-bit number
template <typename M, int DP, int ROWS, int NT> struct Stage {
    typedef typename M::T T;
    typedef Tile<M, DP, ROWS> tile;
    static constexpr int CPR = DP / 8;                          // chunks of a row
    static constexpr int TOTAL = ROWS * CPR;
    static constexpr int N = (TOTAL + NT - 1) / NT;
    typename Src<M>::raw r[N];
    uint32_t off[N];

    static __device__ __forceinline__ int chunk(int i, int tid) {
        const int c = tid + i * NT;
        return TOTAL % NT != 0 && c >= TOTAL ? 0 : c;
    }
    static __device__ __forceinline__ int row_of(int i, int tid) { return chunk(i, tid) / CPR; }
    __device__ __forceinline__ void init(const Src<M> &src, int D, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = chunk(i, tid), col = (c % CPR) * 8;
            off[i] = (uint32_t)(c / CPR) * (uint32_t)src.ld + (uint32_t)(col < D ? col : 0);
        }
    }
    // rows row0 .. of an operand of `n` rows (n >= 1): rows past the end are read as the last one
    __device__ __forceinline__ void load(const Src<M> &src, int row0, int n, int D, int tid) {
        if (row0 + ROWS <= n) {
            const Src<M> s = src.from(row0);
#pragma unroll
            for (int i = 0; i < N; ++i) s.load(r[i], off[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = chunk(i, tid), row = row0 + c / CPR, col = (c % CPR) * 8;
                src.from(row < n ? row : n - 1).load(r[i], col < D ? col : 0);
            }
        }
    }
    // some: rows may have to become zeros, those with keep(i) false
    template <typename Keep> __device__ __forceinline__ void store(bf16_t *t, int D, int tid, bool some, Keep keep) {
        if (some) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (!keep(i)) r[i].zero();
        }
        if (D < DP) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((chunk(i, tid) % CPR) * 8 >= D) r[i].zero();
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (TOTAL % NT != 0 && tid + i * NT >= TOTAL) break;
            const int c = tid + i * NT;
            typename M::vec p[tile::NP];
            r[i].planes(p);
#pragma unroll
            for (int k = 0; k < tile::NP; ++k)
                *reinterpret_cast<typename M::vec *>(t + k * tile::PLANE + tile::at(c / CPR, c % CPR)) = p[k];
        }
    }
};

// Logits are formed times log2 e (scale, cap and slopes carry it): a probability is 2^(x - m) with m the row's largest x
// itself, so that x - m is exact where it matters, whatever the logits' size.
// Capped scores of a tile: x[i] = log2 e cap tanh(x[i] f).  Below TANH_SMALL tanh(t) / t is a polynomial in t^2 (equal ripples on
// that range, the first one 1): 4.2e-8 off with four terms, less than a rounding of float32.  (Three terms, 2.9e-6 off, show in the slopes'
// gradients of bfloat16 calls, which are float32.)  Elsewhere tanh is (1 - e) / (1 + e).  A cap is far above most scores:
// the polynomial serves alone where no score of the wavefront leaves its range.  RAW (bfloat16) has f and cap in its coefficients and starts from
// the scores themselves, up to RAW_MAX (their powers stay in range; the scaled modes' scores are far larger).
constexpr float TANH_SMALL = 0.35f, RAW_MAX = 1e5f;
constexpr float K0 = 1.f, K1 = -0.333326638f, K2 = 0.132998258f, K3 = -0.0491485037f;
template <bool RAW> struct Cap {
    float f, cap, lim, c0, c1, c2, c3;
    __device__ __forceinline__ Cap(float f, float cap_e) : f(f), cap(cap_e * LOG2E) {
        lim = RAW ? fminf(TANH_SMALL / fabsf(f), RAW_MAX) : TANH_SMALL;
        if (RAW) {
            const float u = cap * f, f2 = f * f;
            c0 = K0 * u, c1 = K1 * u * f2, c2 = K2 * u * f2 * f2, c3 = K3 * u * f2 * f2 * f2;
            if (!(fabsf(c3) < INFINITY)) lim = -1.f;        // a steep cap: never by these coefficients
        } else {
            c0 = K0 * cap, c1 = K1 * cap, c2 = K2 * cap, c3 = K3 * cap;
        }
    }
    // of a score (RAW) or of a score times f
    __device__ __forceinline__ float poly(float x) const {
        const float z = x * x;
        return x * fmaf(z, fmaf(z, fmaf(z, c3, c2), c1), c0);
    }
};
template <bool RAW> __device__ __forceinline__ void cap_tile(f32x16_t &x, const Cap<RAW> &c) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        if (!RAW) x[r] *= c.f;
        m = fmaxf(m, fabsf(x[r]));
    }
    if (__any(m >= c.lim)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = RAW ? x[r] * c.f : x[r], a = fabsf(t);
            const float e = __builtin_amdgcn_exp2f(-2.f * LOG2E * a);
            float b = copysignf(c.cap * (1.f - e) * __builtin_amdgcn_rcpf(1.f + e), t);
            asm("" : "+v"(b));          // (a select between two values, not a branch around one)
            // (RAW: scores above RAW_MAX may still be small ones of a larger cap)
            const float s = RAW ? c.cap * (t * fmaf(t * t, fmaf(t * t, fmaf(t * t, K3, K2), K1), K0)) : c.poly(x[r]);
            x[r] = a < TANH_SMALL ? s : b;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = c.poly(x[r]);
    }
}

// distance of two positions whose sign bit was flipped (order and differences of the unsigned values are theirs)
__device__ __forceinline__ uint32_t flip(int32_t pos) { return (uint32_t)pos ^ 0x80000000u; }
__device__ __forceinline__ float dist_of(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("v_sad_u32 %0, %1, %2, 0" : "=v"(d) : "v"(a), "v"(b));      // |a - b|
    return (float)d;
}

// log2 of a sum: the hardware's and a step of Newton's method, within 2e-7
__device__ __forceinline__ double log2_of(float l) {
    const float y = __builtin_amdgcn_logf(l);
    return (double)y + (double)(fmaf(l, __builtin_amdgcn_exp2f(-y), -1.f) * LOG2E);
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// Block b of a launch runs on XCD b % 8.  Runs of GS consecutive work items (tiles of one segment and head: they read
// the same keys) go to one XCD, whose L2 then serves all but the first of them; the runs go round the XCDs in order.
__device__ __forceinline__ int64_t xcd_item(int64_t b, int GS) {
    const int64_t x = b & 7, i = b >> 3;
    return ((i / GS) * 8 + x) * GS + i % GS;
}
inline int64_t xcd_grid(int64_t items, int GS) { return (items + 8 * GS - 1) / (8 * GS) * (8 * GS); }

int check(const magic_attn *a);  // argument checks shared by the entry points

// Largest magnitude of an operand and the smallest of its nonzero rows' largest ones, per head and segment, as the bits
// of floats (finite values of the rows that take part; masked keys do not).  F16x2 serves a segment where max / min is
// at most 2^14 in every operand: its absolute error of 2^-39 max is then below 2^-25 of any row's own largest value.
struct Range {
    uint32_t max, min;
};
struct Ranges {
    const Range *q, *k, *v, *g;   // [heads][n_seg], NULL: not used
    int n_seg;
    bool want_safe;               // which segments this launch serves (NULL arrays: all)
};
__device__ __forceinline__ bool range_ok(Range r) {
    // zero operands are fine; else exponents at most 14 apart
    return r.max == 0u || ((r.max >> 23) <= (r.min >> 23) + 14u && (r.min >> 23) > 0u);
}
// power of two that brings the largest magnitude to [2^13, 2^14)
__device__ __forceinline__ float range_scale(Range r) {
    int e = 13 + 127 - (int)(r.max >> 23);       // exponent of the scale
    if (r.max == 0u) e = 0;
    e = e > 120 ? 120 : e;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// What the launches of a call need beside its arguments: for F16x2 the ranges and the planes of the operands they stage; with
// a key mask the unmasked keys of every segment -- idx[first key row of the segment + i] is the row of the i-th, cnt[segment]
// their number.  Masked keys then cost nothing: the staged side walks rows that were gathered (planes, or kc / vc / posc).
struct Prepared {
    Ranges rg = {nullptr, nullptr, nullptr, nullptr, 0, false};
    PlaneSet q = {}, k = {}, v = {}, g = {};
    const int32_t *idx = nullptr, *cnt = nullptr, *posc = nullptr;
    const void *kc = nullptr, *vc = nullptr;
};
// the call with the gathered rows in the place of its keys
inline magic_attn gathered(const magic_attn *a, const Prepared &p) {
    magic_attn g = *a;
    if (!p.idx) return g;
    g.k = p.kc, g.v = p.vc, g.k_pos = p.posc, g.key_mask = nullptr;
    g.ld_k = g.ld_v = (int64_t)a->kv_heads * a->head_dim, g.hs_k = g.hs_v = a->head_dim;
    return g;
}
// The output's gradient, what marks rows that see no key (lse = +inf there) and what lse's rounding took, in backward
struct GradRows {
    const void *g;
    int64_t ld, hs;
    const float *lse, *rest;
};
bool use_f16(const magic_attn *a);                                 // whether F16x2 is tried for a call
bool fwd_scores_f16(const magic_attn *a);                          // whether its forward pass takes the scores that way too, scaled as here
bool use_gather(const magic_attn *a);                              // whether unmasked keys are gathered
size_t prepare_bytes(const magic_attn *a, bool f16, bool backward);   // workspace of prepare
// ranges and planes (k, v, and in backward q and the output's gradient) where f16; unmasked keys
int prepare(const magic_attn *a, bool f16, const GradRows *g, Arena &ar, Prepared &out, hipStream_t stream);
constexpr int TAB = 8;            // int32 words of a tile-table entry

}  // namespace attn
}  // namespace magic
