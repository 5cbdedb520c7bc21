// Softmax attention of the rows of a segment over the keys of the same segment, forward (magic_attn_fwd).
//   s = scale q.k,  c = cap tanh(s / cap) (cap > 0),  l = c - slope_h |pos_q - pos_k|,  p = softmax of l over the
//   unmasked keys,  o = sum p v;   lse = log2 sum exp(l), -inf for a row that sees no key (o = 0 then).  lse is a double:
//   p = 2^(l log2 e - lse), which the backward pass forms again, is off by as much as lse is, for a whole row.
// One pass over the keys with a running maximum and sum per row; scores are formed transposed (keys x rows), so that a
// lane owns ONE row's statistics and the probabilities feed the second product from their registers (attn_common.h).
// Bound by the matrix and the vector units together (beside its 4 D flops a score takes some eleven vector instructions:
// cap, exponential, sums, conversion).  Twelve graphs of 8,000 nodes, 4 heads of 64, float32 with a distance bias: 2.85 ms,
// 283 TFLOP/s; seven graphs of up to 15,001 nodes, 8 bfloat16 heads of 128 over 2, capped, half the keys masked: 1.12 ms,
// 594 TFLOP/s of the unmasked products.  Three rows over 262,147 keys, 16 heads of 128 over 4: 120 us + 13 to join the
// ranges, 4.5 TB/s of keys and values while it sweeps them.
#include "attn_common.h"
#include <cmath>
#include <type_traits>

namespace magic {
namespace attn {

int check(const magic_attn *a) {
    if (!a) return MAGIC_ERR_INVALID_ARG;
    if (a->dtype != MAGIC_F32 && a->dtype != MAGIC_BF16) return MAGIC_ERR_UNSUPPORTED;
    if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->head_dim < 1) return MAGIC_ERR_INVALID_ARG;
    if (a->head_dim > MAGIC_ATTN_MAX_DIM || a->head_dim % 8 || a->q_heads > MAX_HEADS) return MAGIC_ERR_UNSUPPORTED;
    if (a->n_q < 0 || a->n_k < 0 || a->n_q > MAX_ROWS || a->n_k > MAX_ROWS) return MAGIC_ERR_INVALID_ARG;
    if (a->n_q_tiles < 0 || a->n_k_tiles < 0 || a->max_q < 0 || a->max_k < 0 || a->n_seg < 0) return MAGIC_ERR_INVALID_ARG;
    if (a->n_q > 0 && (!a->q || a->n_q_tiles < 1 || !a->q_tiles)) return MAGIC_ERR_INVALID_ARG;
    if (a->n_k > 0 && (!a->k || !a->v || a->n_k_tiles < 1 || !a->k_tiles)) return MAGIC_ERR_INVALID_ARG;
    if (a->ld_q > MAX_LD || a->ld_k > MAX_LD || a->ld_v > MAX_LD || (int64_t)a->q_heads * a->head_dim > MAX_LD) return MAGIC_ERR_UNSUPPORTED;
    if (a->ld_q < 0 || a->hs_q < 0 || a->ld_k < 0 || a->hs_k < 0 || a->ld_v < 0 || a->hs_v < 0) return MAGIC_ERR_INVALID_ARG;
    const int per = a->dtype == MAGIC_F32 ? 4 : 8;   // rows and heads start on 16-byte addresses
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out_lo) & 15) return MAGIC_ERR_INVALID_ARG;
    if ((a->ld_q | a->hs_q | a->ld_k | a->hs_k | a->ld_v | a->hs_v) % per) return MAGIC_ERR_INVALID_ARG;
    // (scale / cap and cap stay normal float32 numbers)
    if (!(a->cap == 0.f || (a->cap >= 1e-3f && a->cap <= 1e30f)) || !(std::fabs(a->scale) <= 1e30f)) return MAGIC_ERR_INVALID_ARG;
    if (a->cap > 0.f && a->scale != 0.f && !(std::fabs(a->scale / a->cap) >= 0x1p-126f)) return MAGIC_ERR_INVALID_ARG;
    if (a->slopes && ((a->n_q > 0 && !a->q_pos) || (a->n_k > 0 && !a->k_pos))) return MAGIC_ERR_INVALID_ARG;
    return MAGIC_OK;
}

namespace {

__global__ __launch_bounds__(256) void k_range_init(Range *r, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) r[i] = Range{0u, 0xffffffffu};
}

struct RangeArgs {
    magic_attn a;
    const void *g;
    int64_t ld_g, hs_g;
    Range *q, *k, *v, *gr;
    int n_seg;
};

// block: a 128-row tile of one head of one operand, sixteen lanes a row.  Finite values only: an infinity or a NaN becomes
// one in the planes whatever the scale.  (max and min do not depend on the order of the atomics.)
__global__ __launch_bounds__(256) void k_range(RangeArgs r) {
    const magic_attn &a = r.a;
    int y = blockIdx.y;
    const float *base;
    int64_t ld, hs;
    Range *out;
    bool key = false;
    if (y < a.q_heads) {
        base = (const float *)a.q, ld = a.ld_q, hs = a.hs_q, out = r.q;
    } else if ((y -= a.q_heads) < a.kv_heads) {
        base = (const float *)a.k, ld = a.ld_k, hs = a.hs_k, out = r.k, key = true;
    } else if ((y -= a.kv_heads) < a.kv_heads) {
        base = (const float *)a.v, ld = a.ld_v, hs = a.hs_v, out = r.v, key = true;
    } else {
        y -= a.kv_heads;
        base = (const float *)r.g, ld = r.ld_g, hs = r.hs_g, out = r.gr;
    }
    if ((int)blockIdx.x >= (key ? a.n_k_tiles : a.n_q_tiles)) return;
    const int32_t *t = (key ? a.k_tiles : a.q_tiles) + TAB * (int64_t)blockIdx.x;
    constexpr int L = 16;                            // lanes of a row: 16 bytes each, twice for more than 64 columns
    const int c = 4 * (threadIdx.x & (L - 1));
    uint32_t mx = 0u, mn = 0xffffffffu;
#pragma unroll 4
    for (int i = threadIdx.x / L; i < MAGIC_ATTN_TILE; i += 256 / L) {
        const bool in = i < t[1];
        const int64_t row = (int64_t)t[0] + (in ? i : 0);
        const float *x = base + row * ld + y * hs;
        const bool use = in && !(key && a.key_mask && !a.key_mask[row]);
        const f32x4_t u = *reinterpret_cast<const f32x4_t *>(x + (c < a.head_dim ? c : 0));
        f32x4_t v = u;
        if (a.head_dim > 64) v = *reinterpret_cast<const f32x4_t *>(x + (c + 64 < a.head_dim ? c + 64 : 0));
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t p = __float_as_uint(u[e]) & 0x7fffffffu, q = __float_as_uint(v[e]) & 0x7fffffffu;
            m = max(m, max(p < 0x7f800000u ? p : 0u, q < 0x7f800000u ? q : 0u));
        }
        m = use ? m : 0u;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, L));
        mx = max(mx, m);
        if (m != 0u) mn = min(mn, m);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
        mn = min(mn, (uint32_t)__shfl_xor((int)mn, o, 64));
    }
    // one pair of atomics a block: the tiles of a segment all meet in one place
    __shared__ uint32_t smx[4], smn[4];
    if ((threadIdx.x & 63) == 0) smx[threadIdx.x >> 6] = mx, smn[threadIdx.x >> 6] = mn;
    __syncthreads();
    if (threadIdx.x == 0) {
        mx = max(max(smx[0], smx[1]), max(smx[2], smx[3])), mn = min(min(smn[0], smn[1]), min(smn[2], smn[3]));
        if (mx == 0u) return;
        Range *d = out + (int64_t)y * r.n_seg + t[4];
        atomicMax(&d->max, mx);
        atomicMin(&d->min, mn);
    }
}

}  // namespace

namespace {

// Unmasked keys of a segment in ascending order; block: a 128-key tile, which first counts the unmasked keys before it
__global__ __launch_bounds__(256) void k_compact(magic_attn a, int32_t *idx, int32_t *cnt) {
    __shared__ int part[4], w[2];
    const int32_t *t = a.k_tiles + TAB * (int64_t)blockIdx.x;
    const int64_t first = t[5], row0 = t[0];
    const int tid = threadIdx.x, lane = tid & 63, before = (int)(row0 - first);
    const uint8_t *m = a.key_mask + first;
    int n = 0;
    // whole words from the first aligned one on, single bytes around them
    const int head = min(before, (int)((16 - ((uintptr_t)m & 15)) & 15)), words = (before - head) / 16;
    if (tid < head) n += m[tid] != 0;
    for (int i = tid; i < words; i += 256) {
        const uint4 v = *reinterpret_cast<const uint4 *>(m + head + 16 * i);
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) n += __popc((((x[e] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[e]) & 0x80808080u);
    }
    const int tail = head + 16 * words + tid;
    if (tail < before) n += m[tail] != 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0) part[tid >> 6] = n;
    const bool in = tid < t[1] && a.key_mask[row0 + (tid < t[1] ? tid : 0)] != 0;     // (t[1] <= 128: two wavefronts)
    const unsigned long long b = __ballot(in);
    if (lane == 0 && tid < 128) w[tid >> 6] = __popcll(b);
    __syncthreads();
    const int base = part[0] + part[1] + part[2] + part[3];
    if (in) idx[first + base + (tid >= 64 ? w[0] : 0) + __popcll(b & ((1ull << lane) - 1ull))] = (int32_t)(row0 + tid);
    if (tid == 0 && row0 + t[1] == first + t[6]) cnt[t[4]] = base + w[0] + w[1];
}

struct GatherArgs {
    magic_attn a;
    const int32_t *idx, *cnt;
    Ranges rg;              // only what the F16x2 launch leaves over, if ranges are given
    void *kc, *vc;
    int32_t *posc;
};
// rows of the unmasked keys side by side; block: 128 of them, one key head (y) of k or v
template <typename T> __global__ __launch_bounds__(256) void k_gather(GatherArgs g) {
    const magic_attn &a = g.a;
    const int32_t *t = a.k_tiles + TAB * (int64_t)blockIdx.x;
    const int local = t[0] - t[5], n = min(t[1], g.cnt[t[4]] - local);
    if (n <= 0) return;
    const int h = blockIdx.y >> 1, G = a.q_heads / a.kv_heads;
    const bool v = blockIdx.y & 1;
    if (blockIdx.y == 0 && a.slopes && threadIdx.x < n) g.posc[t[0] + threadIdx.x] = a.k_pos[g.idx[t[0] + threadIdx.x]];
    if (g.rg.k) {
        bool safe = range_ok(g.rg.k[h * g.rg.n_seg + t[4]]) && range_ok(g.rg.v[h * g.rg.n_seg + t[4]]);
        for (int i = h * G; i < h * G + G; ++i)
            safe = safe && range_ok(g.rg.q[i * g.rg.n_seg + t[4]]) && (!g.rg.g || range_ok(g.rg.g[i * g.rg.n_seg + t[4]]));
        if (safe) return;
    }
    const T *base = (const T *)(v ? a.v : a.k) + h * (v ? a.hs_v : a.hs_k);
    const int64_t ld = v ? a.ld_v : a.ld_k;
    T *out = (T *)(v ? g.vc : g.kc);
    const int cpr = a.head_dim / 8;
    for (int i = threadIdx.x; i < n * cpr; i += 256) {
        const int64_t at = (int64_t)t[0] + i / cpr;
        const int c = (i % cpr) * 8;
        Raw<T> x;
        x.load(base + g.idx[at] * ld + c);
        x.store(out + (at * a.kv_heads + h) * a.head_dim + c);
    }
}

struct SplitArgs {
    magic_attn a;
    GradRows g;
    Ranges rg;
    const int32_t *idx, *cnt;      // unmasked keys, or NULL
    _Float16 *q, *k, *v, *gr;      // hi planes; the lo ones follow
};

// block: a 128-row tile of one head of k, v (then q and the gradient, scaled alike for all heads of a key head)
__global__ __launch_bounds__(256) void k_split(SplitArgs s) {
    const magic_attn &a = s.a;
    const int D = a.head_dim, G = a.q_heads / a.kv_heads;
    int y = blockIdx.y;
    const float *base;
    int64_t ld, hs, rows;
    _Float16 *out;
    bool key = true;
    int heads = a.kv_heads;
    const Range *rg;
    if (y < a.kv_heads) {
        base = (const float *)a.k, ld = a.ld_k, hs = a.hs_k, out = s.k, rg = s.rg.k;
    } else if ((y -= a.kv_heads) < a.kv_heads) {
        base = (const float *)a.v, ld = a.ld_v, hs = a.hs_v, out = s.v, rg = s.rg.v;
    } else if ((y -= a.kv_heads, key = false, heads = a.q_heads, y < a.q_heads)) {
        base = (const float *)a.q, ld = a.ld_q, hs = a.hs_q, out = s.q, rg = s.rg.q;
    } else {
        y -= a.q_heads;
        base = (const float *)s.g.g, ld = s.g.ld, hs = s.g.hs, out = s.gr, rg = s.rg.g;
    }
    rows = key ? a.n_k : a.n_q;
    if ((int)blockIdx.x >= (key ? a.n_k_tiles : a.n_q_tiles)) return;
    const int32_t *t = (key ? a.k_tiles : a.q_tiles) + TAB * (int64_t)blockIdx.x;
    Range r = {0u, 0xffffffffu};
    for (int i = key ? y : y / G * G, e = key ? y + 1 : i + G; i < e; ++i) {
        const Range x = rg[i * s.rg.n_seg + t[4]];
        r.max = max(r.max, x.max);
    }
    const float scale = range_scale(r);
    const int cpr = D / 8, n = (key && s.cnt ? min(t[1], s.cnt[t[4]] - (t[0] - t[5])) : t[1]) * cpr;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int64_t row = (int64_t)t[0] + i / cpr;
        const int c = (i % cpr) * 8;
        Raw<float> x;
        x.load(base + (key && s.idx ? s.idx[row] : row) * ld + y * hs + c);
        const bool use = key || !s.g.lse || s.g.lse[(int64_t)y * a.n_q + row] != INFINITY;
        if (!use) x.zero();
        if (out == s.gr) {           // (a rounding of float32; the sweep over the keys has no registers left for it)
            const float z = s.g.rest[(int64_t)y * a.n_q + row];
            x.a *= z, x.b *= z;
        }
        f16x8_t p[2];
        x.planes(p, scale);
        _Float16 *o = out + (row * heads + y) * D + c;
        *reinterpret_cast<f16x8_t *>(o) = p[0];
        *reinterpret_cast<f16x8_t *>(o + rows * heads * D) = p[1];
    }
}

size_t plane_elems(const magic_attn *a, bool key) {
    return 2 * (size_t)(key ? a->n_k * a->kv_heads : a->n_q * a->q_heads) * a->head_dim;
}
int64_t range_count(const magic_attn *a, bool grad) {
    return ((grad ? 2 : 1) * (int64_t)a->q_heads + 2 * (int64_t)a->kv_heads) * a->n_seg;
}

}  // namespace

// F16x2 needs two passes over the operands first: for float32 calls of enough work to pay for them.  Heads up to 32 wide
// gain less (the softmax takes much of their time) and need longer segments.  us with those passes, three planes against
// two: 64 wide, forward and backward, twenty graphs of 600 nodes 295 / 284, ten of 1,200 483 / 405; 16 wide, forward,
// twenty of 1,500 147 / 141 (half the keys masked: 93 / 109), eight of 3,000 224 / 188 (134 / 135), four of 8,000 827 /
// 608 (450 / 339); forward and backward, eight of 3,000 861 / 752, four of 8,000 2,912 / 2,356.
bool use_f16(const magic_attn *a) { return a->dtype == MAGIC_F32 && a->max_k >= (a->head_dim > 32 ? 512 : 2048) && a->n_seg > 0; }

// Gathering costs two launches and a copy of the unmasked rows, and saves the masked share of everything else
bool use_gather(const magic_attn *a) { return a->key_mask && a->max_k >= 512 && a->n_seg > 0 && a->n_k > 0; }

size_t prepare_bytes(const magic_attn *a, bool f16, bool backward) {
    size_t n = 0;
    if (f16) {
        const size_t k = align_up(plane_elems(a, true) * 2), q = align_up(plane_elems(a, false) * 2);
        n += align_up(range_count(a, backward) * sizeof(Range)) + 2 * k + (backward ? 2 * q : 0);
    }
    if (use_gather(a))
        n += 2 * align_up((size_t)a->n_k * 4) + align_up((size_t)a->n_seg * 4) +
             2 * align_up((size_t)a->n_k * a->kv_heads * a->head_dim * (a->dtype == MAGIC_F32 ? 4 : 2));
    return n;
}

int prepare(const magic_attn *a, bool f16, const GradRows *g, Arena &ar, Prepared &out, hipStream_t stream) {
    int32_t *idx = nullptr, *cnt = nullptr, *posc = nullptr;
    unsigned char *kc = nullptr, *vc = nullptr;
    const int x = a->n_q_tiles > a->n_k_tiles ? a->n_q_tiles : a->n_k_tiles;
    if (use_gather(a)) {
        const size_t rows = (size_t)a->n_k * a->kv_heads * a->head_dim * (a->dtype == MAGIC_F32 ? 4 : 2);
        idx = ar.take<int32_t>(a->n_k), posc = ar.take<int32_t>(a->n_k), cnt = ar.take<int32_t>(a->n_seg);
        kc = ar.take<unsigned char>(rows), vc = ar.take<unsigned char>(rows);
        if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
        out.idx = idx, out.cnt = cnt, out.posc = posc, out.kc = kc, out.vc = vc;
        MAGIC_LAUNCH("attn_compact", k_compact, a->n_k_tiles, 256, 0, stream, *a, idx, cnt);
    }
    if (f16) {
        const int64_t n = range_count(a, g != nullptr);
        Range *r = ar.take<Range>(n);
        SplitArgs s;
        s.a = *a;
        s.g = g ? *g : GradRows{nullptr, 0, 0, nullptr, nullptr};
        s.idx = idx, s.cnt = cnt;
        s.k = ar.take<_Float16>(plane_elems(a, true)), s.v = ar.take<_Float16>(plane_elems(a, true));
        s.q = s.gr = nullptr;
        if (g) s.q = ar.take<_Float16>(plane_elems(a, false)), s.gr = ar.take<_Float16>(plane_elems(a, false));
        if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
        RangeArgs ra;
        ra.a = *a, ra.g = s.g.g, ra.ld_g = s.g.ld, ra.hs_g = s.g.hs, ra.n_seg = a->n_seg;
        ra.q = r, ra.k = r + (int64_t)a->q_heads * a->n_seg, ra.v = ra.k + (int64_t)a->kv_heads * a->n_seg,
        ra.gr = ra.v + (int64_t)a->kv_heads * a->n_seg;
        out.rg = s.rg = Ranges{ra.q, ra.k, ra.v, g ? ra.gr : nullptr, a->n_seg, true};
        out.k = {s.k, a->n_k, a->kv_heads}, out.v = {s.v, a->n_k, a->kv_heads};
        out.q = {s.q, a->n_q, a->q_heads}, out.g = {s.gr, a->n_q, a->q_heads};
        MAGIC_LAUNCH("attn_range_init", k_range_init, magic::stride_grid(n, 256), 256, 0, stream, r, n);
        const int y = a->q_heads * (g ? 2 : 1) + 2 * a->kv_heads, ys = 2 * a->kv_heads + (g ? 2 * a->q_heads : 0);
        if (y > 65535) return MAGIC_ERR_UNSUPPORTED;
        MAGIC_LAUNCH("attn_range", k_range, dim3(x, y), 256, 0, stream, ra);
        MAGIC_LAUNCH("attn_split", k_split, dim3(x, ys), 256, 0, stream, s);
    }
    if (idx) {
        const GatherArgs ga = {*a, idx, cnt, out.rg, kc, vc, posc};
        const dim3 grid(a->n_k_tiles, 2 * a->kv_heads);
        if (2 * a->kv_heads > 65535) return MAGIC_ERR_UNSUPPORTED;
        if (a->dtype == MAGIC_F32)
            MAGIC_LAUNCH("attn_gather", k_gather<float>, grid, 256, 0, stream, ga);
        else
            MAGIC_LAUNCH("attn_gather", k_gather<bf16_t>, grid, 256, 0, stream, ga);
    }
    return magic::launch_status();
}

}  // namespace attn
}  // namespace magic

namespace {

using namespace magic::attn;
using magic::bf16_t;
using magic::bf16x8_t;

struct FwdArgs {
    magic_attn a;
    void *out;
    int64_t ld_o, hs_o;
    double *lse;
    int n_split;          // key ranges of a tile (1: results go straight to out / lse)
    float *part_o;        // [n_split][q_heads][n_q][head_dim], normalised within the range
    double *part_l;       // [n_split][q_heads][n_q], base-2 log of the range's sum
    int cols, rows, gc;   // columns of a block's tile = rows x gc heads of one key head
    int sub;              // blocks that share a 128-row tile of the table
    int n_hb;             // head blocks: q_heads / gc
    int64_t items;
    Prepared pr;
};

__device__ __forceinline__ int h_of(const FwdArgs &p, int hb) { return hb * p.gc; }

// four results of a row and head: rounded, and what the rounding took where it is wanted
template <typename T> __device__ __forceinline__ void store_out(const FwdArgs &p, int64_t row, int64_t h, int c, const float (&x)[4]) {
    magic::store_vec<T, 4>((T *)p.out + row * p.ld_o + h * p.hs_o + c, true, x);
    if constexpr (sizeof(T) == 2) {
        if (p.a.out_lo) {
            float r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = x[e] - (float)(T)x[e];
            magic::store_vec<T, 4>((T *)p.a.out_lo + (row * p.a.q_heads + h) * p.a.head_dim + c, true, r);
        }
    }
}

// WM groups of 32 columns (rows, or rows x heads of one key head), KG groups of KW keys: a block of WM * KG wavefronts
template <typename M, int DP, int WM, int KG, int KW>
__global__ __launch_bounds__(64 * WM *KG, DP == 128 && (M::N > 1 || WM == 1) ? 1 : 2) void k_attn_fwd(FwdArgs p) {
#pragma clang fp contract(off)      // (a logit is rounded once, for its row's maximum and for its probability alike)
    typedef typename M::T T;
    typedef typename M::vec vec;
    constexpr int NP = M::N, KS = DP / 16, DB = (DP + 31) / 32, BK = KG * KW, NT = 64 * WM * KG, KB = KW / 32;
    typedef Stage<M, DP, BK, NT> stage;
    typedef Tile<M, DP, BK> tile;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16_t *sK = reinterpret_cast<bf16_t *>(smem), *sV = sK + NP * tile::PLANE;
    uint32_t *sPos = reinterpret_cast<uint32_t *>(smem + 2 * tile::BYTES);
    uint32_t *sMask = sPos + BK;           // all bits of a key that takes part

    const magic_attn &a = p.a;
    const int64_t item = xcd_item(blockIdx.x, 16);
    if (item >= p.items) return;
    const int D = a.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hf = lane >> 5;
    const int wm = wave % WM, kg = wave / WM;
    const int64_t per_hb = (int64_t)a.n_q_tiles * p.sub;
    const int64_t ts = item % per_hb;
    const int hb = (int)(item / per_hb % p.n_hb), split = (int)(item / (per_hb * p.n_hb));
    const int32_t *t = a.q_tiles + TAB * (ts / p.sub);
    const int nq = t[1] - (int)(ts % p.sub) * p.rows;     // rows left for this block and the ones behind it
    if (nq <= 0) return;
    const int64_t q0 = (int64_t)t[0] + (ts % p.sub) * p.rows, k0 = t[2];
    const int nk = t[3] > 0 && p.pr.cnt ? p.pr.cnt[t[4]] : t[3];
    // this block's range of keys, in whole tiles
    const int tiles = (nk + BK - 1) / BK, per = (tiles + p.n_split - 1) / p.n_split;
    const int t_beg = split * per, t_end = min(t_beg + per, tiles);

    const int col = wm * 32 + li;
    const int row = col / p.gc, h = hb * p.gc + col % p.gc;
    const bool ok = col < p.cols && row < nq && row < p.rows;
    const int hk = hb * p.gc / (a.q_heads / a.kv_heads);
    const Src<M> K = src_of<M>(a.k, a.ld_k, a.hs_k, p.pr.k, k0, hk, a.head_dim),
                 V = src_of<M>(a.v, a.ld_v, a.hs_v, p.pr.v, k0, hk, a.head_dim);

    float sq = 1.f, sk = 1.f, sv = 1.f;
    if (p.pr.rg.q) {
        const Range rq = p.pr.rg.q[h_of(p, hb) * p.pr.rg.n_seg + t[4]], rk = p.pr.rg.k[hk * p.pr.rg.n_seg + t[4]],
                    rv = p.pr.rg.v[hk * p.pr.rg.n_seg + t[4]];
        if ((range_ok(rq) && range_ok(rk) && range_ok(rv)) != p.pr.rg.want_safe) return;   // the other launch's segment
        if constexpr (M::SCALED) sq = range_scale(rq), sk = range_scale(rk), sv = range_scale(rv);
    }
    vec qf[KS][NP];
    {
        const T *q = (const T *)a.q + (q0 + (ok ? row : 0)) * a.ld_q + (ok ? h : hb * p.gc) * a.hs_q;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Raw<T> r;
            const int c = 16 * ks + 8 * hf;
            r.load(q + (c < D ? c : 0));
            if (!ok || c >= D) r.zero();
            r.planes(qf[ks], sq);
        }
    }
    const bool bias = a.slopes != nullptr;
    const float slope = bias ? a.slopes[ok ? h : hb * p.gc] * LOG2E : 0.f;
    const uint32_t qpos = bias ? flip(a.q_pos[q0 + (ok ? row : 0)]) : 0u;
    const float unscale = 1.f / sq * (1.f / sk);
    const float s_in = (a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E) * unscale;
    const Cap<M::N == 1> cap(s_in, a.cap);
    // A probability is formed as 2^(x - unit(m)).  The scaled mode keeps them times 2^14 and adds 14 - m, rounded, at once:
    // alike for a row, so the sum takes it out again.  From FAR on that rounding would be off by 1 and more (2^16 is no
    // fp16 number): there m is taken off first.
    constexpr float P_EXP = M::SCALED ? 14.f : 0.f, FAR = 1048576.f;
    auto unit = [&](float m) { return M::SCALED ? (fabsf(m) >= FAR ? (double)m - 14.0 : -(double)(14.f - m)) : (double)m; };

    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    // Of this lane's keys: the two halves of a wavefront share m, the largest logit so far, and add l at the end.
    float m = -INFINITY, l = 0.f;

    uint32_t plain = tile::lane_plain(lane) + 2u * kg * KW * tile::W, turned = tile::lane_turned(lane) + 2u * kg * KW * tile::W;
    stage kst, vst;
    kst.init(K, D, tid), vst.init(V, D, tid);
    uint8_t keep[stage::N];
    int pos = 0;             // (taken as loaded: a use here would wait for the whole tile)
    uint8_t mk = 0;
    auto load = [&](int tt) {
        const int j0 = tt * BK;
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
    if (t_beg < t_end) load(t_beg);
    for (int tt = t_beg; tt < t_end; ++tt) {
        __syncthreads();  // the reads of the tile before are done
        const bool masked = a.key_mask != nullptr || (tt + 1) * BK > nk;
        kst.store(sK, D, tid, masked, [&](int i) { return keep[i] != 0; });
        vst.store(sV, D, tid, masked, [&](int i) { return keep[i] != 0; });
        if (tid < BK) sPos[tid] = flip(pos), sMask[tid] = mk ? 0xffffffffu : 0u;
        __syncthreads();
        if (tt + 1 < t_end) load(tt + 1);

        stay(plain), stay(turned);
        f32x16_t s[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                vec f[NP];
                tile::frag(sK, plain, 32 * b, ks, f);
                mma(s[b], f, qf[ks]);
            }
        feed<NP * KB, PRODUCTS<M> * KB, KS>();
        // logits; a masked key's is -inf, whatever its score became (0 times an infinity of q)
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            if (a.cap > 0.f) {
                cap_tile(s[b], cap);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] *= s_in;
            }
            if (masked) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const i32x4_t km = *reinterpret_cast<const i32x4_t *>(sMask + kg * KW + 32 * b + 8 * g + 4 * hf);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[b][4 * g + e] = __uint_as_float((__float_as_uint(s[b][4 * g + e]) & (uint32_t)km[e]) | (0xff800000u & ~(uint32_t)km[e]));
                }
            }
            if (bias) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const i32x4_t kp = *reinterpret_cast<const i32x4_t *>(sPos + kg * KW + 32 * b + 8 * g + 4 * hf);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[b][4 * g + e] = fmaf(-slope, dist_of((uint32_t)kp[e], qpos), s[b][4 * g + e]);
                }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        mx = fmaxf(m, fmaxf(mx, other_half(mx)));
        const float ms = mx == -INFINITY ? 0.f : mx;
        float mo = P_EXP - ms;
        const float al = __builtin_amdgcn_exp2f(M::SCALED ? (float)(unit(m) - unit(ms)) : m - ms);
        if (M::SCALED && __any(fabsf(ms) >= FAR)) {
            const bool far = fabsf(ms) >= FAR;
            const float off = far ? ms : 0.f;
            if (far) mo = P_EXP;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] -= off;
        }
        m = mx;
        // The tile's sums are formed by themselves and added once: a long tail of small terms, each below half a unit of
        // the running sum, would otherwise be lost term by term (3e-6 of the result over 8,000 keys with a distance bias).
        // bfloat16 results do not see that: their sums run on, and are scaled where a maximum moves.
        constexpr bool TILE_SUM = M::N > 1;
        if (!TILE_SUM && __any(al != 1.f)) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= al;
        }
        float tsum = 0.f;
        // What rounding takes from bfloat16 probabilities goes through a second product in blocks of 32 columns, which wait for
        // their keys more than they compute: outputs 1.94e-3 -> 1.66e-3 of their norm off, a rounding of the result alone, and
        // three rows over 262,147 keys 120 -> 124 us.  (Tiles of 128 rows: 24 wide 279 -> 323 us, 128 wide 1,095 -> 1,455.)
        constexpr bool LOW = M::N == 1 && KG > 1;
        vec pf[KB * 2][NP], pl[LOW ? KB * 2 : 1][NP];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(s[b][8 * u + e] + mo);
                    tsum += x[e];
                }
                to_planes(x, pf[2 * b + u]);
                if constexpr (LOW) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] -= (float)pf[2 * b + u][0][e];
                    to_planes(x, pl[2 * b + u]);
                }
            }
        l = fmaf(l, al, tsum);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            f32x16_t c = o[d];
            if (TILE_SUM) {
#pragma unroll
                for (int r = 0; r < 16; ++r) c[r] = 0.f;
            }
#pragma unroll
            for (int w = 0; w < KB * 2; ++w) {
                vec f[NP];
                tile::frag_t(sV, turned, 16 * w, d, f);
                if constexpr (LOW) mma(c, f, pl[w]);
                mma(c, f, pf[w]);
            }
            feed<2 * NP, (LOW ? 2 : 1) * PRODUCTS<M>, KB * 2>();
            if (TILE_SUM) {
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] = fmaf(o[d][r], al, c[r]);
            } else {
                o[d] = c;
            }
        }
    }
    l += other_half(l);
    if constexpr (KG > 1) {
        // the key groups' (m, l, o) come together through LDS, in group order
        __syncthreads();
        float *sM = reinterpret_cast<float *>(smem), *sL = sM + KG * 32 * WM, *sO = sL + KG * 32 * WM;
        constexpr int OW = DB * 32 + 1;
        if (hf == 0) sM[(kg * WM + wm) * 32 + li] = m, sL[(kg * WM + wm) * 32 + li] = l;
        __syncthreads();
        float mt = -INFINITY, lt = 0.f;
#pragma unroll
        for (int g = 0; g < KG; ++g) mt = fmaxf(mt, sM[(g * WM + wm) * 32 + li]);
        const float ms = mt == -INFINITY ? 0.f : mt;
#pragma unroll
        for (int g = 0; g < KG; ++g) lt += sL[(g * WM + wm) * 32 + li] * __builtin_amdgcn_exp2f(sM[(g * WM + wm) * 32 + li] - ms);
        const float al = __builtin_amdgcn_exp2f(m - ms);
        for (int g = KG - 1; g >= 1; --g) {
            if (kg == g) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float *q = sO + (wm * 32 + li) * OW + 32 * d + 8 * (r >> 2) + 4 * hf + (r & 3);
                        *q = (g == KG - 1 ? 0.f : *q) + o[d][r] * al;
                    }
            }
            __syncthreads();
        }
        if (kg != 0) return;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                o[d][r] = o[d][r] * al + sO[(wm * 32 + li) * OW + 32 * d + 8 * (r >> 2) + 4 * hf + (r & 3)];
        m = mt, l = lt;
    }
    if (!ok) return;
    // (two factors: l times the scale of tiny values is no float32 number)
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f, unv = 1.f / sv;
    const double ls = m == -INFINITY && l == 0.f ? -INFINITY : unit(m) + P_EXP + log2_of(M::SCALED ? l * 0x1p-14f : l);   // base 2
    if (p.n_split > 1) {
        const int64_t base = ((int64_t)split * a.q_heads + h) * a.n_q + q0 + row;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hf;
                if (c < D)
                    *reinterpret_cast<f32x4_t *>(p.part_o + base * D + c) =
                        f32x4_t{o[d][4 * g] * inv * unv, o[d][4 * g + 1] * inv * unv, o[d][4 * g + 2] * inv * unv, o[d][4 * g + 3] * inv * unv};
            }
        if (hf == 0) p.part_l[base] = ls;
        return;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hf;
            const float x[4] = {o[d][4 * g] * inv * unv, o[d][4 * g + 1] * inv * unv, o[d][4 * g + 2] * inv * unv, o[d][4 * g + 3] * inv * unv};
            if (c < D) store_out<T>(p, q0 + row, h, c, x);
        }
    if (hf == 0) p.lse[(int64_t)h * a.n_q + q0 + row] = ls;
}

// sum over LPR neighbouring lanes, the same in all of them
template <int LPR> __device__ __forceinline__ float lanes_sum(float x) {
    auto add = [](float v, auto ctrl) {
        return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (LPR >= 2) x = add(x, std::integral_constant<int, 0xB1>{});    // lane ^ 1
    if constexpr (LPR >= 4) x = add(x, std::integral_constant<int, 0x4E>{});    // lane ^ 2
    if constexpr (LPR >= 8) x = add(x, std::integral_constant<int, 0x141>{});   // mirrored in eight
    if constexpr (LPR >= 16) x = add(x, std::integral_constant<int, 0x140>{});  // mirrored in sixteen
    if constexpr (LPR >= 32) x += __shfl_xor(x, 16, 64);
    return x;
}

// Few columns (rows x heads of one key head, at most NC): no tiles, no matrix instructions -- the keys and values stream
// through registers once.  LPR lanes hold a key row in 16-byte chunks; every such group walks its own keys with its own
// running maximum, sum and output, four keys at a time with the next four under way; the groups join through LDS.
// A matrix tile would split 64 float32 keys into planes for one column of thirty-two: 75 us against 36 us for twelve rows
// over twelve stored graphs of 8,000 nodes (4 heads of 64; 199 MB, 5.5 TB/s).
template <typename T, int DP, int NC> __global__ __launch_bounds__(256) void k_attn_few(FwdArgs p) {
#pragma clang fp contract(off)      // (a logit is rounded once, for its row's maximum and for its probability alike)
    constexpr int EPL = 16 / (int)sizeof(T), LPR = DP / EPL, GPB = 256 / LPR, U = 4;
    typedef typename magic::vec_of<T, EPL>::type vt;
    __shared__ float sm[GPB][NC], sl[GPB][NC], so[GPB * NC * DP];
    const magic_attn &a = p.a;
    const int64_t item = blockIdx.x;
    const int D = a.head_dim, tid = threadIdx.x, gl = tid % LPR, grp = tid / LPR;
    const int64_t per_hb = (int64_t)a.n_q_tiles * p.sub;
    const int64_t ts = item % per_hb;
    const int hb = (int)(item / per_hb % p.n_hb), split = (int)(item / (per_hb * p.n_hb));
    const int32_t *t = a.q_tiles + TAB * (ts / p.sub);
    const int nq = t[1] - (int)(ts % p.sub) * p.rows;
    if (nq <= 0) return;
    const int64_t q0 = (int64_t)t[0] + (ts % p.sub) * p.rows, k0 = t[2];
    const int nk = t[3], per = (nk + p.n_split - 1) / p.n_split;
    const int beg = min(split * per, nk), end = min(beg + per, nk);
    const int c0 = gl * EPL;
    const bool cin = c0 < D;
    const int hk = hb * p.gc / (a.q_heads / a.kv_heads);
    const T *K = (const T *)a.k + k0 * a.ld_k + hk * a.hs_k + (cin ? c0 : 0), *V = (const T *)a.v + k0 * a.ld_v + hk * a.hs_v + (cin ? c0 : 0);
    const bool bias = a.slopes != nullptr;
    const float scale = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E, cap = a.cap * LOG2E;

    float q[NC][EPL], slope[NC], m[NC], l[NC], o[NC][EPL];
    uint32_t qpos[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int row = c / p.gc, h = hb * p.gc + c % p.gc;
        const bool ok = c < p.cols && row < nq;
        const T *qp = (const T *)a.q + (q0 + (ok ? row : 0)) * a.ld_q + (ok ? h : hb * p.gc) * a.hs_q + (cin ? c0 : 0);
        const vt x = *reinterpret_cast<const vt *>(qp);
#pragma unroll
        for (int e = 0; e < EPL; ++e) q[c][e] = ok && cin ? (float)x[e] : 0.f, o[c][e] = 0.f;
        slope[c] = bias ? a.slopes[ok ? h : hb * p.gc] * LOG2E : 0.f;
        qpos[c] = bias ? flip(a.q_pos[q0 + (ok ? row : 0)]) : 0u;
        m[c] = -INFINITY, l[c] = 0.f;
    }
    vt kn[U], vn[U];
    uint8_t keep[U];
    int pos[U];
    auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * GPB, jc = j < end ? j : end - 1;
            kn[u] = *reinterpret_cast<const vt *>(K + (int64_t)jc * a.ld_k);
            vn[u] = *reinterpret_cast<const vt *>(V + (int64_t)jc * a.ld_v);
            keep[u] = a.key_mask ? a.key_mask[k0 + jc] : 1;
            pos[u] = bias ? a.k_pos[k0 + jc] : 0;
        }
    };
    if (beg < end) load(beg + grp);
    for (int j0 = beg + grp; j0 < end; j0 += U * GPB) {
        vt kc[U], vc[U];
        bool in[U];
        uint32_t kp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) kc[u] = kn[u], vc[u] = vn[u], in[u] = j0 + u * GPB < end && keep[u] != 0, kp[u] = flip(pos[u]);
        load(j0 + U * GPB);
        float kf[U][EPL], vf[U][EPL];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < EPL; ++e) kf[u][e] = cin ? (float)kc[u][e] : 0.f, vf[u][e] = in[u] && cin ? (float)vc[u][e] : 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float x[U], mx = m[c];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < EPL; ++e) d = fmaf(q[c][e], kf[u][e], d);
                x[u] = lanes_sum<LPR>(d) * scale;
            }
            if (a.cap > 0.f) {
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = cap * tanhf(x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (bias) x[u] = fmaf(-slope[c], dist_of(kp[u], qpos[c]), x[u]);
                x[u] = in[u] ? x[u] : -INFINITY;
                mx = fmaxf(mx, x[u]);
            }
            const float ms = mx == -INFINITY ? 0.f : mx, al = __builtin_amdgcn_exp2f(m[c] - ms);
            m[c] = mx;
            float ps = 0.f, acc[EPL];
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] = o[c][e] * al;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float pr = __builtin_amdgcn_exp2f(x[u] - ms);
                ps += pr;
#pragma unroll
                for (int e = 0; e < EPL; ++e) acc[e] = fmaf(pr, vf[u][e], acc[e]);
            }
            l[c] = fmaf(l[c], al, ps);
#pragma unroll
            for (int e = 0; e < EPL; ++e) o[c][e] = acc[e];
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (gl == 0) sm[grp][c] = m[c], sl[grp][c] = l[c];
#pragma unroll
        for (int e = 0; e < EPL; ++e) so[(grp * NC + c) * DP + c0 + e] = o[c][e];
    }
    __syncthreads();
    // a thread per (column, output column): the groups in order
    for (int i = tid; i < NC * DP; i += 256) {
        const int c = i / DP, d = i % DP, row = c / p.gc, h = hb * p.gc + c % p.gc;
        if (c >= p.cols || row >= nq || d >= D) continue;
        float mt = -INFINITY, lt = 0.f, ot = 0.f;
        for (int g = 0; g < GPB; ++g) mt = sm[g][c] > mt || sm[g][c] != sm[g][c] ? sm[g][c] : mt;
        const float ms = mt == -INFINITY ? 0.f : mt;
        for (int g = 0; g < GPB; ++g) {
            const float w = __builtin_amdgcn_exp2f(sm[g][c] - ms);
            lt = fmaf(sl[g][c], w, lt), ot = fmaf(so[(g * NC + c) * DP + d], w, ot);
        }
        const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
        const double ls = mt == -INFINITY && lt == 0.f ? -INFINITY : mt + log2_of(lt);
        if (p.n_split > 1) {
            const int64_t base = ((int64_t)split * a.q_heads + h) * a.n_q + q0 + row;
            p.part_o[base * D + d] = ot * inv;
            if (d == 0) p.part_l[base] = ls;
        } else {
            const float x = ot * inv;
            ((T *)p.out)[(q0 + row) * p.ld_o + h * p.hs_o + d] = (T)x;
            if (sizeof(T) == 2 && a.out_lo) ((T *)a.out_lo)[((q0 + row) * a.q_heads + h) * D + d] = (T)(x - (float)(T)x);
            if (d == 0) p.lse[(int64_t)h * a.n_q + q0 + row] = ls;
        }
    }
}

// The key ranges of a row joined: o = sum_s 2^(l_s - l) o_s.  A block takes a row and head; CPR lanes hold its columns
// and the 256 / CPR lane groups take the ranges in turn, added in group order.
template <typename T, int CPR> __global__ __launch_bounds__(256) void k_attn_join(FwdArgs p) {
    constexpr int NG = 256 / CPR;
    __shared__ float w[256];
    __shared__ double red[256];
    __shared__ f32x4_t so[256];
    const magic_attn &a = p.a;
    const int64_t plane = a.n_q * a.q_heads;
    const int tid = threadIdx.x, g = tid / CPR, c = (tid % CPR) * 4;
    const int64_t hr = blockIdx.x;                  // head * n_q + row
    const double mine = tid < p.n_split ? p.part_l[tid * plane + hr] : -INFINITY;
    red[tid] = mine;
    __syncthreads();
    double m = -INFINITY;                           // (a NaN is the largest of all: it has to reach the result)
    for (int s = 0; s < p.n_split; ++s) m = red[s] > m || red[s] != red[s] ? red[s] : m;
    const double ms = m == -INFINITY ? 0.0 : m;
    w[tid] = __builtin_amdgcn_exp2f((float)(mine - ms));
    __syncthreads();
    float l = 0.f;
    for (int s = 0; s < p.n_split; ++s) l += w[s];
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    if (c < a.head_dim)
        for (int s = g; s < p.n_split; s += NG)
            o += w[s] * *reinterpret_cast<const f32x4_t *>(p.part_o + (s * plane + hr) * a.head_dim + c);
    so[tid] = o;
    __syncthreads();
    if (g != 0 || c >= a.head_dim) return;
    const int n = p.n_split < NG ? p.n_split : NG;
    for (int i = 1; i < n; ++i) o += so[i * CPR + tid];
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    const int64_t h = hr / a.n_q, row = hr - h * a.n_q;
    store_out<T>(p, row, h, c, x);
    if (c == 0) p.lse[hr] = m == -INFINITY ? -INFINITY : ms + log2_of(l);
}

// The same for up to MANY ranges of many rows: a thread holds four columns of a (row, head) and walks its ranges.
// 8,000 rows of 4 heads of 64 in two ranges: 9 us, where a block for every row and head takes 27.
constexpr int MANY = 16;
template <typename T> __global__ __launch_bounds__(256) void k_attn_join_rows(FwdArgs p) {
    const magic_attn &a = p.a;
    const int cpr = a.head_dim / 4;
    const int64_t plane = (int64_t)a.q_heads * a.n_q, total = plane * cpr;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t hr = i / cpr;
        const int c = (int)(i - hr * cpr) * 4;
        double m = -INFINITY;
        for (int s = 0; s < p.n_split; ++s) {
            const double x = p.part_l[s * plane + hr];
            m = x > m || x != x ? x : m;
        }
        const double ms = m == -INFINITY ? 0.0 : m;
        float l = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.n_split; ++s) {
            const float w = __builtin_amdgcn_exp2f((float)(p.part_l[s * plane + hr] - ms));
            l += w;
            o += w * *reinterpret_cast<const f32x4_t *>(p.part_o + (s * plane + hr) * a.head_dim + c);
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        const int64_t h = hr / a.n_q, row = hr - h * a.n_q;
        store_out<T>(p, row, h, c, x);
        if (c == 0) p.lse[hr] = m == -INFINITY ? -INFINITY : ms + log2_of(l);
    }
}

constexpr int FEW = 4;

struct Shape {
    int wm, n_split, cols, rows, gc, sub, n_hb;
    bool f16;
    int64_t items;
};

// Tiles of 128 rows up to which blocks of 32 columns serve better: where those still find the chip empty.  Measured on
// both sides with 4 heads, us of kernels, 32 columns against 128.  float32, 64 wide: four graphs of 500 nodes (64 tiles)
// 33 / 36, one of 2,000 (64) 111 / 94, of 4,000 (128) 295 / 144; 128 wide: one of 128 nodes (4) 27 / 22, of 500 (16)
// 84 / 63.  bfloat16, 64 wide: eight of 500 (128) 15 / 19, one of 4,000 (128) 62 / 59, forty of 100 (160) 16 / 10; 128
// wide: one of 1,000 (32) 33 / 33, of 2,000 (64) 54 / 40.  Up to 32 wide: one of 7,000 (220), float32 213 / 188, bfloat16
// 91 / 110, eight of 500 (128) 16 / 21 and 12 / 15, a hundred of 100 (400) 13 / 10 in bfloat16; float32 by
// two planes, one of 4,000 (128) 78 / 92, half masked 81 / 88, of 5,500 (172) 134 / 150, half masked 134 / 117, of 7,000
// 222 / 183, half masked 222 / 136.
int64_t few_tiles(const magic_attn *a) {
    const bool f32 = a->dtype == MAGIC_F32;
    if (a->head_dim <= 32) return magic::attn::use_f16(a) ? 144 : 255;
    if (a->head_dim <= 64) return f32 ? 48 : 128;
    return f32 ? 0 : 32;
}

// Ranges of keys that fill the rounds of blocks best: `slots` of them run at once (two a CU, one where planes and registers
// fill it), a block takes 1 / ranges of the time, and the fewest ranges within 8 % of the best are taken.  4 heads of 64,
// one graph, us whole against cut: 10,000 nodes (316 tiles) 515 / 396 in three, 12,000 (376) 620 / 534 in four, twenty graphs
// of 700 (480) 83 / 97 in two: stay whole; 128 wide in float32, 10,000 nodes 1,276 / 1,002 in two.
int64_t ranges(int64_t blocks, int64_t slots, int64_t most) {
    int64_t top = 3 * slots / blocks, best = 1;
    if (top > most) top = most;
    if (top > 256) top = 256;
    double least = 1e30;
    for (int64_t n = 1; n <= top; ++n) {
        const double rounds = (double)((blocks * n + slots - 1) / slots) / (double)n;
        if (rounds < least) least = rounds;
    }
    while (best < top && (double)((blocks * best + slots - 1) / slots) > 1.08 * least * (double)best) ++best;
    return best;
}

// How a call is cut: 128 rows of one head a block (wm 4), or 32 (row, head) columns with the keys dealt to its wavefronts
// (wm 1), or up to four columns without matrix instructions (wm 0; not for bfloat16 training, whose backward pass takes the
// scores of the matrix instructions to be the forward pass's); then key ranges until there are enough blocks.
Shape shape_of(const magic_attn *a) {
    Shape s;
    const int G = a->q_heads / a->kv_heads;
    const int64_t big = (int64_t)a->n_q_tiles * a->q_heads;
    s.wm = big > few_tiles(a) && a->max_q > 32 ? 4 : 1;
    if ((int64_t)a->max_q * G <= FEW && !a->out_lo) {
        s.wm = 0, s.gc = G, s.rows = a->max_q > 0 ? a->max_q : 1, s.cols = s.rows * G, s.sub = 1, s.n_hb = a->kv_heads;
        s.f16 = false;
        const int64_t blocks = (int64_t)a->n_q_tiles * s.n_hb, most = (a->max_k + 255) / 256;
        int64_t split = (1024 + blocks - 1) / blocks;
        if (split > most) split = most;
        s.n_split = (int)(split > 256 ? 256 : split < 1 ? 1 : split);
        s.items = blocks * s.n_split;
        return s;
    }
    if (s.wm == 4) {
        s.gc = 1, s.cols = s.rows = 128;
    } else {
        s.gc = G;
        while (s.gc > 32 || G % s.gc) --s.gc;          // heads of a key head that share its tile
        s.rows = 32 / s.gc, s.cols = s.rows * s.gc;
    }
    const int longest = a->max_q < MAGIC_ATTN_TILE ? a->max_q : MAGIC_ATTN_TILE;   // rows of the fullest table entry
    s.sub = (longest + s.rows - 1) / s.rows;
    if (s.sub < 1) s.sub = 1;
    s.n_hb = a->q_heads / s.gc;
    const int64_t blocks = (int64_t)a->n_q_tiles * s.sub * s.n_hb;
    const int64_t most = (a->max_k + 511) / 512;
    int64_t split = 512 / blocks;
    if (s.wm == 4) split = ranges(blocks, a->dtype == MAGIC_F32 && a->head_dim > 64 ? 256 : 512, most);
    if (split > most) split = most;
    if (split > 256) split = 256;
    if (split < 1) split = 1;
    s.n_split = (int)split;
    s.items = blocks * split;
    s.f16 = magic::attn::use_f16(a) && s.wm == 4 && a->n_k > 0;
    return s;
}

}  // namespace

bool magic::attn::fwd_scores_f16(const magic_attn *a) { return a->n_q_tiles > 0 && shape_of(a).f16 && a->q_heads == a->kv_heads; }

namespace {

template <typename M, int DP, int WM, int KG, int KW> int launch(FwdArgs &p, hipStream_t st) {
    typedef Tile<M, DP, KG * KW> tile;
    size_t lds = 2 * tile::BYTES + KG * KW * 8;
    const size_t join = (size_t)KG * 32 * WM * 8 + (size_t)32 * WM * ((DP + 31) / 32 * 32 + 1) * 4;
    if (KG > 1 && join > lds) lds = join;
    if (magic::ensure_dynamic_lds((const void *)k_attn_fwd<M, DP, WM, KG, KW>, lds) != MAGIC_OK) return MAGIC_ERR_RUNTIME;
    const int64_t grid = xcd_grid(p.items, 16);
    if (grid > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
    MAGIC_LAUNCH(M::SCALED ? "attn_fwd_f16x2" : "attn_fwd", (k_attn_fwd<M, DP, WM, KG, KW>), (int)grid, 64 * WM * KG, lds, st, p);
    return magic::launch_status();
}

template <typename M> int run_rows(FwdArgs &p, hipStream_t st) {
    const int D = p.a.head_dim;
    return D <= 16   ? launch<M, 16, 4, 1, 64>(p, st)
           : D <= 32 ? launch<M, 32, 4, 1, 64>(p, st)
           : D <= 64 ? launch<M, 64, 4, 1, 64>(p, st)
                     : launch<M, 128, 4, 1, 64>(p, st);
}

template <typename T, int DP> int run_few(FwdArgs &p, hipStream_t st) {
    if (p.items > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
    if (p.cols == 1)
        MAGIC_LAUNCH("attn_few", (k_attn_few<T, DP, 1>), (int)p.items, 256, 0, st, p);
    else if (p.cols == 2)
        MAGIC_LAUNCH("attn_few", (k_attn_few<T, DP, 2>), (int)p.items, 256, 0, st, p);
    else
        MAGIC_LAUNCH("attn_few", (k_attn_few<T, DP, 4>), (int)p.items, 256, 0, st, p);
    return magic::launch_status();
}

template <typename M> int run(FwdArgs &p, int wm, hipStream_t st) {
    const int D = p.a.head_dim;
    if (wm == 4) return run_rows<M>(p, st);
    if (wm == 0) {
        typedef typename M::T T;
        return D <= 16 ? run_few<T, 16>(p, st) : D <= 32 ? run_few<T, 32>(p, st) : D <= 64 ? run_few<T, 64>(p, st) : run_few<T, 128>(p, st);
    }
    // wavefronts of a block: as many as leave the LDS room for two blocks a CU
    constexpr int KG64 = M::N == 3 ? 2 : 4, KG128 = M::N == 3 ? 1 : 2;
    return D <= 16   ? launch<M, 16, 1, 4, 32>(p, st)
           : D <= 32 ? launch<M, 32, 1, 4, 32>(p, st)
           : D <= 64 ? launch<M, 64, 1, KG64, 32>(p, st)
                     : launch<M, 128, 1, KG128, 32>(p, st);
}

template <typename T> int join(FwdArgs &p, hipStream_t st) {
    const int D = p.a.head_dim;
    if (p.n_split <= MANY) {
        MAGIC_LAUNCH("attn_join", k_attn_join_rows<T>, magic::stride_grid(p.a.n_q * p.a.q_heads * (D / 4), 256, 8192), 256, 0, st, p);
        return magic::launch_status();
    }
    const int64_t grid = p.a.n_q * p.a.q_heads;
    if (grid > 0x7fffffffLL) return MAGIC_ERR_UNSUPPORTED;
    if (D <= 16)
        MAGIC_LAUNCH("attn_join", (k_attn_join<T, 4>), (int)grid, 256, 0, st, p);
    else if (D <= 32)
        MAGIC_LAUNCH("attn_join", (k_attn_join<T, 8>), (int)grid, 256, 0, st, p);
    else if (D <= 64)
        MAGIC_LAUNCH("attn_join", (k_attn_join<T, 16>), (int)grid, 256, 0, st, p);
    else
        MAGIC_LAUNCH("attn_join", (k_attn_join<T, 32>), (int)grid, 256, 0, st, p);
    return magic::launch_status();
}

}  // namespace

extern "C" {

size_t magic_attn_fwd_workspace_bytes(const magic_attn *a) {
    if (check(a) != MAGIC_OK || a->n_q == 0) return 256;
    const Shape s = shape_of(a);
    const size_t rows = s.n_split > 1 ? (size_t)s.n_split * a->q_heads * a->n_q : 0;
    return magic::align_up(rows * a->head_dim * sizeof(float)) + magic::align_up(rows * sizeof(double)) +
           (s.wm == 4 ? magic::attn::prepare_bytes(a, s.f16, false) : 0) + 256;
}

int magic_attn_fwd(const magic_attn *a, void *out, int64_t ld_out, int64_t hs_out, double *lse, void *workspace,
                   size_t workspace_bytes, void *stream) {
    const int st = check(a);
    if (st != MAGIC_OK || a->n_q == 0) return st;
    const int per = a->dtype == MAGIC_F32 ? 4 : 8;
    if (!out || !lse || ((uintptr_t)out & 15) || ld_out < 0 || hs_out < 0 || (ld_out | hs_out) % per) return MAGIC_ERR_INVALID_ARG;
    const Shape s = shape_of(a);
    FwdArgs p;
    p.a = *a;
    p.out = out, p.ld_o = ld_out, p.hs_o = hs_out, p.lse = lse;
    p.n_split = s.n_split, p.cols = s.cols, p.rows = s.rows, p.gc = s.gc, p.sub = s.sub, p.n_hb = s.n_hb, p.items = s.items;
    p.part_o = nullptr, p.part_l = nullptr;
    magic::Arena ar(workspace, workspace_bytes);
    if (s.n_split > 1) {
        const size_t rows = (size_t)s.n_split * a->q_heads * a->n_q;
        p.part_o = ar.take<float>(rows * a->head_dim);
        p.part_l = ar.take<double>(rows);
        if (!ar.ok()) return MAGIC_ERR_WORKSPACE;
    }
    int rc = MAGIC_OK;
    if (s.wm == 4) {
        rc = magic::attn::prepare(a, s.f16, nullptr, ar, p.pr, (hipStream_t)stream);
        if (rc != MAGIC_OK) return rc;
        p.a = magic::attn::gathered(a, p.pr);
        if (s.f16) {
            rc = run_rows<F16x2>(p, (hipStream_t)stream);
            if (rc != MAGIC_OK) return rc;
            p.pr.rg.want_safe = false;         // the segments whose rows differ too much in size
        }
    }
    const bool f32 = a->dtype == MAGIC_F32;
    rc = f32 ? run<F32x3>(p, s.wm, (hipStream_t)stream) : run<BF16>(p, s.wm, (hipStream_t)stream);
    if (rc != MAGIC_OK || s.n_split == 1) return rc;
    return f32 ? join<float>(p, (hipStream_t)stream) : join<magic::bf16_t>(p, (hipStream_t)stream);
}

}  // extern "C"
