// Adam / AdamW over many tensors in one launch (crates/weta-optim/src/lib.rs:210-239, 276-283, which walks the parameter
// list), with its state in 32 or in 8 bits, and the 2-norm of all their gradients.
//
// State layout: tensor i owns the elements [offset_i, offset_i + len_i), offset_i a multiple of 256.
//   32 bits: m[P], v[P] as f32 (P: all offsets' end).
//   8 bits:  codes of m (signed) [P], codes of sqrt(v) (unsigned) [P], then one f32 scale per 256 elements for each.
// Both codes are companded by a square root, m = s sign(c) (c / 127)^2 and sqrt(v) = s (c / 255)^2 with s the largest
// magnitude of the block: the distance between neighbouring values is 2 / c of the value, so the large ones, which
// carry the update, are kept to 0.8 % (m) and 0.4 % (sqrt(v)) and the least one is 6e-5 (1.5e-5) of the largest.
// sqrt(v) rather than v is coded because it has m's range (v's is twice as many decades) and is at hand in the update.
// A second moment that is not zero keeps at least code 1: rounding it to zero would leave m / (0 + eps).
// Compiled with -fmad=false, and approximate functions are corrected to the rounded result wherever it counts: every f32
// rounding is the one written here, so the codes do not depend on the launch's shape, and the 32-bit step gives
// wb_adam_step's bits.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>

#include "adam.cuh"
#include "common.h"
#include "pair.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int BLOCK8 = 256;        // elements that share a scale: one warp, eight per lane
constexpr int CHUNK = 2048;         // elements a thread block takes at a time, all of one tensor
constexpr float M_TOP = 127.f, V_TOP = 255.f;
constexpr float TINY = 7.8886090522101181e-31f;  // 2^-100, the least scale: its reciprocal is still finite

struct Tensor {
    float* theta;
    const float* grad;
    int64_t offset;
    int64_t len;  // negative: -len elements, exempt from weight decay
};

constexpr int HINTS = 128;

// The tensors of one launch, passed by value: nothing to upload, nothing a captured graph could lose.
template <int N>
struct Table {
    int n;
    int shift;
    unsigned int chunks;    // of all tensors together
    uint16_t hint[HINTS + 1];  // the tensor of chunk i << shift
    unsigned int first[N];  // a tensor's first chunk
    Tensor t[N];
};

// The tensor that holds chunk c: the last one whose first chunk is not behind it (tensors of no chunk share their
// successor's first one).  Between two hints few are left to search: every step is a dependent load that the block's first
// load of data waits for.
template <int N>
__device__ __forceinline__ int find_tensor(const Table<N>& tab, unsigned int c) {
    int lo = tab.hint[c >> tab.shift], hi = tab.hint[(c >> tab.shift) + 1];
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ AdamK with_device_scale(AdamK k, const float* scale) {
    if (scale) {
        const float s = *scale;
        k.gscale = k.scale_grad ? k.gscale * s : s;
        k.scale_grad = 1;
    }
    return k;
}

// ---- 32-bit state -------------------------------------------------------------------------------------------

__device__ __forceinline__ void one(float* th, const float* g, float* m, float* v, int i, const AdamK& k) {
    float a = th[i], mi = k.first ? 0.f : m[i], vi = k.first ? 0.f : v[i];
    adam_one(a, g[i], mi, vi, k);
    th[i] = a;
    m[i] = mi;
    v[i] = vi;
}

// A tensor whose pointers are both on 16-byte boundaries takes 128-bit accesses (the state always is); any other, and a
// tensor's last group, goes element by element.
template <int N>
__global__ void __launch_bounds__(THREADS) adam_multi32_kernel(const __grid_constant__ Table<N> tab, float* __restrict__ m, float* __restrict__ v,
                                                               AdamK k0, const float* __restrict__ scale) {
    wb_pdl_enter();
    const int ti = find_tensor(tab, blockIdx.x);
    const Tensor t = tab.t[ti];
    if (!t.grad) return;
    AdamK k = with_device_scale(k0, scale);
    const int64_t len = t.len < 0 ? -t.len : t.len, at = static_cast<int64_t>(blockIdx.x - tab.first[ti]) * CHUNK;
    if (t.len < 0) k.has_wd = 0;
    float *th = t.theta + at, *mp = m + t.offset + at, *vp = v + t.offset + at;
    const float* gp = t.grad + at;
    const int n = static_cast<int>(min(static_cast<int64_t>(CHUNK), len - at));
    if (((reinterpret_cast<uintptr_t>(t.theta) | reinterpret_cast<uintptr_t>(t.grad)) & 15) == 0) {
        constexpr int U = CHUNK / (4 * THREADS);
        float4 a[U], g[U], mi[U], vi[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * THREADS + threadIdx.x) * 4;
            if (i + 4 <= n) {
                a[u] = *reinterpret_cast<const float4*>(th + i);
                g[u] = *reinterpret_cast<const float4*>(gp + i);
                mi[u] = k.first ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(mp + i);
                vi[u] = k.first ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(vp + i);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * THREADS + threadIdx.x) * 4;
            if (i + 4 <= n) {
                adam_one(a[u].x, g[u].x, mi[u].x, vi[u].x, k);
                adam_one(a[u].y, g[u].y, mi[u].y, vi[u].y, k);
                adam_one(a[u].z, g[u].z, mi[u].z, vi[u].z, k);
                adam_one(a[u].w, g[u].w, mi[u].w, vi[u].w, k);
                *reinterpret_cast<float4*>(th + i) = a[u];
                *reinterpret_cast<float4*>(mp + i) = mi[u];
                *reinterpret_cast<float4*>(vp + i) = vi[u];
            }
        }
        const int i = (n & ~3) + static_cast<int>(threadIdx.x);
        if (i < n) one(th, gp, mp, vp, i, k);
    } else {
        for (int i = threadIdx.x; i < n; i += THREADS) one(th, gp, mp, vp, i, k);
    }
}

// ---- 8-bit state --------------------------------------------------------------------------------------------

// A byte as f32 without the conversion unit (16 lanes per clock, which the square roots and the division need): put under
// the exponent of 2^23 it is 2^23 + byte, exactly.  And a value of magnitude under 2^22 plus 1.5 * 2^23 is rounded to the
// nearest integer, ties to even, whose two's complement the low bits then are.
constexpr float BYTE_BASE = 8388608.f, MAGIC = 12582912.f;
__device__ __forceinline__ float based_byte(uint32_t word, int i) { return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7440 + i)); }
__device__ __forceinline__ Pair<float> bytes_of(uint32_t word, int i, float base) {
    return pair(based_byte(word, i), based_byte(word, i + 1)) + pair(-base, -base);
}
// The codes' values; codes of m are signed.
__device__ __forceinline__ Pair<float> m_codes(uint32_t word, int i) { return bytes_of(word ^ 0x80808080u, i, BYTE_BASE + 128.f); }
__device__ __forceinline__ Pair<float> v_codes(uint32_t word, int i) { return bytes_of(word, i, BYTE_BASE); }
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* c) {
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
__device__ __forceinline__ float decode_m(float c, float unit) { return c * fabsf(c) * unit; }
__device__ __forceinline__ float decode_root(float c, float unit) { return c * c * unit; }

// Square root and quotient, correctly rounded, two at a time, for operands far from the ends of the exponent range (the
// caller sends all others to sqrtf and /): an approximation from the function unit, refined, then corrected by its exact
// residual with one fused operation (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", IBM J. Res. Dev. 34, 1990: with 1/d correctly rounded and q within a unit, q + (m - d q) / d rounds to m/d).
// That the root and the reciprocal are correctly rounded is checked for every value of the range they are used in
// (wb_adam_multi_selftest_rounding, which a test calls).
constexpr float LOW_M = 8.6736173798840355e-19f, TOP_M = 1.152921504606847e18f;   // 2^-60 and 2^60
constexpr float LOW_V = 7.8886090522101181e-31f, TOP_V = 1.2089258196146292e24f;  // 2^-100 and 2^80
constexpr float LOW_D = LOW_M, TOP_D = 2.305843009213694e18f;                     // 2^-60 and 2^61
__device__ __forceinline__ Pair<float> root_of(const Pair<float>& v) {
    float a, b, ya, yb;
    unpair(v, a, b);
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(ya) : "f"(a));
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(yb) : "f"(b));
    const Pair<float> y = pair(ya, yb), g = v * y, minus_v = v * pair(-1.f, -1.f), minus_half = y * pair(-0.5f, -0.5f);
    return muladd(muladd(g, g, minus_v), minus_half, g);
}
// 1 / d from -d.
__device__ __forceinline__ Pair<float> reciprocal_of(const Pair<float>& minus_d) {
    float a, b, ya, yb;
    unpair(minus_d, a, b);
    asm("rcp.approx.f32 %0, %1;" : "=f"(ya) : "f"(-a));
    asm("rcp.approx.f32 %0, %1;" : "=f"(yb) : "f"(-b));
    const Pair<float> y = pair(ya, yb);
    return muladd(muladd(minus_d, y, pair(1.f, 1.f)), y, y);
}
// m / d from -d.
__device__ __forceinline__ Pair<float> quotient_of(const Pair<float>& m, const Pair<float>& minus_d) {
    const Pair<float> y = reciprocal_of(minus_d), q = m * y;
    return muladd(muladd(minus_d, q, m), y, q);
}

// The largest and the least of three magnitudes; `largest_or_nan` is NaN if one is.
__device__ __forceinline__ float largest_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float largest(float a, float b, float c) {
    float r;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float least(float a, float b, float c) {
    float r;
    asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The scale of a block from every lane's largest magnitude.  One that is not finite poisons the block: its scale is stored as
// NaN, and every value read from it is NaN.  (The bits of f32 magnitudes order like the values, NaN last.)
__device__ __forceinline__ float block_scale(float lane_max) {
    const unsigned int bits = __reduce_max_sync(0xffffffffu, __float_as_uint(lane_max) & 0x7fffffffu);
    if (bits >= 0x7f800000u) return __int_as_float(0x7fffffff);
    return fmaxf(__uint_as_float(bits), TINY);
}

// Codes of eight values: rint(sqrt(|x| level)), the square root correctly rounded; negative where x is (SIGNED); at least 1
// where x is above 0 (else).  level is top^2 / (largest |x|), so sqrt(|x| level) exceeds top by rounding at most and no code
// does.  The approximate square root's relative error is at most 2^-23 (PTX ISA, sqrt.approx), 2^-15 of at most 256, and moves
// rint's result only next to a half: a lane that comes within 2^-14 of one takes all its roots again (within 2^-11, every
// fourth warp did).  The codes are the results' low bytes.
template <bool SIGNED>
__device__ __forceinline__ void encode(const Pair<float> (&x)[4], float level, uint32_t (&code)[8]) {
    float far = 0.f, low = 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float q0, q1, s0, s1, f0, f1, c0, c1;
        unpair(x[j] * pair(level, level), q0, q1);
        asm("sqrt.approx.f32 %0, %1;" : "=f"(s0) : "f"(fabsf(q0)));
        asm("sqrt.approx.f32 %0, %1;" : "=f"(s1) : "f"(fabsf(q1)));
        if (!SIGNED) low = least(low, s0, s1);
        const Pair<float> s = SIGNED ? pair(copysignf(s0, q0), copysignf(s1, q1)) : pair(s0, s1), r = s + pair(MAGIC, MAGIC);
        unpair(s + muladd(r, pair(-1.f, -1.f), pair(MAGIC, MAGIC)), f0, f1);
        far = largest(far, f0, f1);
        unpair(r, c0, c1);
        code[2 * j] = __float_as_uint(c0);
        code[2 * j + 1] = __float_as_uint(c1);
    }
    if (far > 0.49993896484375f || (!SIGNED && low < 1.f)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float a, b;
            unpair(x[j >> 1], a, b);
            if (j & 1) a = b;
            float s = sqrtf(fabsf(a * level));
            s = SIGNED ? copysignf(s, a) : fmaxf(s, a > 0.f ? 1.f : 0.f);
            code[j] = __float_as_uint(s + MAGIC);
        }
    }
}

// The step's scalars, each twice, so that a packed operation reads both from the constant bank at once.
struct AdamK8 {
    Pair<float> b1, omb1, b2, omb2, minus_inv_sqrt_bc2, minus_eps, minus_step, minus_zero;
    float gscale, decay_mul;  // 1 where there is none: x * 1 is x
    float wd, inv_sqrt_bc2, eps, step;
    int l2;          // weight decay through the gradient
    int eps_normal;  // eps is in [2^-60, 2^60] and inv_sqrt_bc2 at most 2^20
};

// One warp takes a block of 256 elements, a lane the groups of four at 4 lane and 128 + 4 lane.
// Bound by instruction issue (82 % of the slots): 101 M elements in 128 tensors took 562 us with conversions, roots and
// quotients one at a time, 286 us now (251 us are their bytes).  One block per warp and five thread blocks per processor: when
// that took 311 us, four thread blocks took 334 us and six 322 us; two blocks in turn per warp took 378 us.
// That holds where no moment is 0.  A lane that holds one, and every lane of a tensor's last block that is not full, takes
// sqrtf and / for its eight elements and all roots of encode<false> again: the same tensors with nine rows of ten without
// gradient since the first step 478 us, with every tenth gradient 0 579 us, with none at all 494 us.
template <int N, bool FIRST>
__global__ void __launch_bounds__(THREADS, 5) adam_multi8_kernel(const __grid_constant__ Table<N> tab, uint32_t* __restrict__ mc, uint32_t* __restrict__ vc,
                                                              float* __restrict__ ms, float* __restrict__ vs, const __grid_constant__ AdamK8 k8,
                                                              const float* __restrict__ scale) {
    wb_pdl_enter();
    const int ti = find_tensor(tab, blockIdx.x);
    const Tensor t = tab.t[ti];
    if (!t.grad) return;
    const int64_t len = t.len < 0 ? -t.len : t.len;
    const float gscale = scale ? k8.gscale * *scale : k8.gscale, shrink = t.len < 0 ? 1.f : k8.decay_mul;
    const bool aligned = ((reinterpret_cast<uintptr_t>(t.theta) | reinterpret_cast<uintptr_t>(t.grad)) & 15) == 0;
    const int lane = threadIdx.x & 31;
    const int64_t start = static_cast<int64_t>(blockIdx.x - tab.first[ti]) * CHUNK + (threadIdx.x >> 5) * BLOCK8;
    if (start >= len) return;
    const int n = static_cast<int>(min(static_cast<int64_t>(BLOCK8), len - start));
    // x y, rounded whatever is added to it (see rounded_product)
    auto times = [&](const Pair<float>& x, const Pair<float>& y) { return rounded_product(x, y, k8.minus_zero); };
    const int64_t s = t.offset + start, block = s / BLOCK8;
    float* tp = t.theta + start;
    const float* gp = t.grad + start;
    Pair<float> th[4], g[4], mn[4], root[4];  // root: first v
    const bool wide = aligned && n == BLOCK8;
    auto at = [&](int j) { return (j >> 1) * 128 + lane * 4 + 2 * (j & 1); };  // pair j's place in the block
    if (wide) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(tp + at(2 * h)), b = *reinterpret_cast<const ulonglong2*>(gp + at(2 * h));
            th[2 * h].v = a.x;
            th[2 * h + 1].v = a.y;
            g[2 * h].v = b.x;
            g[2 * h + 1].v = b.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = at(j);
            th[j] = pair(e < n ? tp[e] : 0.f, e + 1 < n ? tp[e + 1] : 0.f);
            g[j] = pair(e < n ? gp[e] : 0.f, e + 1 < n ? gp[e + 1] : 0.f);
        }
    }
    uint32_t cm[2], cv[2];
    float um = 0.f, ur = 0.f;
    if (!FIRST) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            cm[h] = mc[s / 4 + h * 32 + lane];
            cv[h] = vc[s / 4 + h * 32 + lane];
        }
        um = ms[block] * (1.f / (M_TOP * M_TOP));
        ur = vs[block] * (1.f / (V_TOP * V_TOP));
    }
    // adam_one's chain without its additions of 0 (they only turn -0 into 0), two elements at a time
    const Pair<float> by = pair(gscale, gscale), keep = pair(shrink, shrink);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = times(g[j], by);
    if (k8.l2 && t.len >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = g[j] + times(th[j], pair(k8.wd, k8.wd));
    }
    float top_m = 0.f, top_v = 0.f, low_m = 1.f, low_v = 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Pair<float> m = times(g[j], k8.omb1), v = times(times(g[j], g[j]), k8.omb2);
        if (!FIRST) {
            float c0, c1;
            unpair(m_codes(cm[j >> 1], 2 * (j & 1)), c0, c1);
            const Pair<float> old = times(pair(c0 * fabsf(c0), c1 * fabsf(c1)), pair(um, um));
            const Pair<float> c = v_codes(cv[j >> 1], 2 * (j & 1)), r = times(times(c, c), pair(ur, ur));
            m = times(old, k8.b1) + m;
            v = times(times(r, r), k8.b2) + v;
        }
        if (n < BLOCK8) {  // behind the tensor's end: the padding, whose codes stay 0
            if (at(j) >= n) m = v = pair(0.f, 0.f);
            else if (at(j) + 1 >= n) {
                float a, b;
                unpair(m, a, b);
                m = pair(a, 0.f);
                unpair(v, a, b);
                v = pair(a, 0.f);
            }
        }
        th[j] = times(th[j], keep);
        mn[j] = m;
        root[j] = v;
        float a, b;
        unpair(m, a, b);
        top_m = largest_or_nan(top_m, a, b);
        low_m = least(low_m, a, b);
        unpair(v, a, b);
        top_v = largest_or_nan(top_v, a, b);
        low_v = least(low_v, a, b);
    }
    // m in [2^-60, 2^60], v in [2^-100, 2^80], eps in [2^-60, 2^60] and 1 / sqrt(1 - beta2^t) at most 2^20: the denominator lies in
    // [2^-60, 2^61] and the quotient in [2^-121, 2^120], so nothing leaves the normal range before the quotient is multiplied
    if (k8.eps_normal && low_m >= LOW_M && low_v >= LOW_V && top_m <= TOP_M && top_v <= TOP_V) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            root[j] = root_of(root[j]);
            th[j] = th[j] + times(quotient_of(mn[j], times(root[j], k8.minus_inv_sqrt_bc2) + k8.minus_eps), k8.minus_step);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float m0, m1, r0, r1, t0, t1;
            unpair(mn[j], m0, m1);
            unpair(root[j], r0, r1);
            unpair(th[j], t0, t1);
            r0 = sqrtf(r0);
            r1 = sqrtf(r1);
            root[j] = pair(r0, r1);
            th[j] = pair(t0 - m0 / (r0 * k8.inv_sqrt_bc2 + k8.eps) * k8.step, t1 - m1 / (r1 * k8.inv_sqrt_bc2 + k8.eps) * k8.step);
        }
    }
    if (wide) {
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<ulonglong2*>(tp + at(2 * h)) = make_ulonglong2(th[2 * h].v, th[2 * h + 1].v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a, b;
            unpair(th[j], a, b);
            if (at(j) < n) tp[at(j)] = a;
            if (at(j) + 1 < n) tp[at(j) + 1] = b;
        }
    }
    // the largest root is the root of the largest v: rounding is monotone
    const float sm = block_scale(top_m), sr = block_scale(sqrtf(top_v));
    uint32_t code[8];
    encode<true>(mn, (M_TOP * M_TOP) / sm, code);
#pragma unroll
    for (int h = 0; h < 2; ++h) mc[s / 4 + h * 32 + lane] = pack_bytes(code + 4 * h);
    encode<false>(root, (V_TOP * V_TOP) / sr, code);
#pragma unroll
    for (int h = 0; h < 2; ++h) vc[s / 4 + h * 32 + lane] = pack_bytes(code + 4 * h);
    if (lane == 0) {
        ms[block] = sm;
        vs[block] = sr;
    }
}

// The values that the 8-bit state stands for, four at a time (the state's length is a multiple of 256).
__global__ void __launch_bounds__(THREADS) adam_multi8_read_kernel(const uint32_t* __restrict__ mc, const uint32_t* __restrict__ vc,
                                                                   const float* __restrict__ ms, const float* __restrict__ vs, float* __restrict__ m,
                                                                   float* __restrict__ v, int64_t groups, int wide) {
    wb_pdl_enter();
    const int64_t q = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
    if (q >= groups) return;
    auto put = [&](float* to, const float (&a)[4]) {
        if (wide) {
            reinterpret_cast<float4*>(to)[q] = make_float4(a[0], a[1], a[2], a[3]);
        } else {
            for (int i = 0; i < 4; ++i) to[4 * q + i] = a[i];
        }
    };
    float a[4];
    if (m) {
        const uint32_t c = mc[q];
        const float unit = ms[q / (BLOCK8 / 4)] * (1.f / (M_TOP * M_TOP));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            unpair(m_codes(c, i), a[i], a[i + 1]);
            a[i] = decode_m(a[i], unit);
            a[i + 1] = decode_m(a[i + 1], unit);
        }
        put(m, a);
    }
    if (v) {
        const uint32_t c = vc[q];
        const float unit = vs[q / (BLOCK8 / 4)] * (1.f / (V_TOP * V_TOP));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            unpair(v_codes(c, i), a[i], a[i + 1]);
            a[i] = decode_root(a[i], unit);
            a[i + 1] = decode_root(a[i + 1], unit);
            a[i] *= a[i];
            a[i + 1] *= a[i + 1];
        }
        put(v, a);
    }
}

// Counts the values of the fast path's range whose root or reciprocal is not the rounded one, quotients of four numerators
// for each denominator, and last all roots and reciprocals that were looked at.
__global__ void __launch_bounds__(THREADS) adam_rounding_selftest_kernel(unsigned long long* bad) {
    const uint32_t stride = gridDim.x * THREADS, first = blockIdx.x * THREADS + threadIdx.x;
    unsigned long long roots = 0, reciprocals = 0, quotients = 0, seen = 0;
    auto differ = [](const Pair<float>& p, float x, float y) {
        float a, b;
        unpair(p, a, b);
        return (__float_as_uint(a) != __float_as_uint(x)) + (__float_as_uint(b) != __float_as_uint(y));
    };
    for (uint32_t i = __float_as_uint(LOW_V) + 2 * first; i <= __float_as_uint(TOP_V); i += 2 * stride) {
        const float a = __uint_as_float(i), b = __uint_as_float(i + 1);
        roots += differ(root_of(pair(a, b)), sqrtf(a), sqrtf(b));
        seen += 2;
    }
    for (uint32_t i = __float_as_uint(LOW_D) + 2 * first; i <= __float_as_uint(TOP_D); i += 2 * stride) {
        const float a = __uint_as_float(i), b = __uint_as_float(i + 1);
        const Pair<float> minus_d = pair(-a, -b);
        reciprocals += differ(reciprocal_of(minus_d), 1.f / a, 1.f / b);
        seen += 2;
        uint32_t h = i * 2654435761u;
        for (int k = 0; k < 4; ++k) {  // numerators of any mantissa and sign, exponents -60 to 59
            h = h * 1664525u + 1013904223u;
            const uint32_t e = (67u + (h >> 8) % 120u) << 23;
            const float m = __uint_as_float((h & 0x807fffffu) | e), n = __uint_as_float(((h * 40503u) & 0x807fffffu) | e);
            quotients += differ(quotient_of(pair(m, n), minus_d), m / a, n / b);
        }
    }
    atomicAdd(bad, roots);
    atomicAdd(bad + 1, reciprocals);
    atomicAdd(bad + 2, quotients);
    atomicAdd(bad + 3, seen);
}

// ---- the norm -----------------------------------------------------------------------------------------------

// Squares of f32 are exact in f64 and neither overflow nor vanish there; sums in f64, each in a fixed order.  Block b of
// this launch takes its share of the chunks, one after the other (so that it looks the first one's tensor up and then walks on),
// and leaves parts[at + b]; the block that arrives last of all launches joins the `total` parts and leaves the counter zero.
template <int N>
__global__ void __launch_bounds__(THREADS) grad_norm_kernel(const __grid_constant__ Table<N> tab, double* __restrict__ parts, int at, int total,
                                                            unsigned int* __restrict__ counter, double max_norm, float* __restrict__ norm,
                                                            float* __restrict__ clip) {
    __shared__ double warp_sum[THREADS / 32];
    __shared__ unsigned int last;
    wb_pdl_enter();
    unsigned int c = static_cast<unsigned int>(static_cast<uint64_t>(tab.chunks) * blockIdx.x / gridDim.x);
    const unsigned int end = static_cast<unsigned int>(static_cast<uint64_t>(tab.chunks) * (blockIdx.x + 1) / gridDim.x);
    double acc = 0.0;
    auto add = [&](float g) {
        const double d = g;
        acc += d * d;
    };
    for (int ti = c < end ? find_tensor(tab, c) : 0; c < end; ++ti) {
        const Tensor& t = tab.t[ti];
        const unsigned int next = ti + 1 < tab.n ? min(tab.first[ti + 1], end) : end;
        if (next <= c) continue;  // a tensor of no chunk
        if (t.grad) {
            const int64_t len = t.len < 0 ? -t.len : t.len;
            const int64_t i0 = static_cast<int64_t>(c - tab.first[ti]) * CHUNK, i1 = min(static_cast<int64_t>(next - tab.first[ti]) * CHUNK, len);
            const float* g = t.grad + i0;
            const int64_t n = i1 - i0, head = min(n, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / 4);
            const int64_t packs = (n - head) / 4;
            if (threadIdx.x < head) add(g[threadIdx.x]);
            const float4* g4 = reinterpret_cast<const float4*>(g + head);
            for (int64_t q0 = threadIdx.x; q0 < packs; q0 += 4 * THREADS) {
                float4 a[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) a[u] = q0 + u * THREADS < packs ? g4[q0 + u * THREADS] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    add(a[u].x);
                    add(a[u].y);
                    add(a[u].z);
                    add(a[u].w);
                }
            }
            const int64_t rest = head + 4 * packs + threadIdx.x;
            if (rest < n) add(g[rest]);
        }
        c = next;
    }
    auto block_sum = [&](double v) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
        __syncthreads();
        double s = 0.0;
        for (int w = 0; w < THREADS / 32; ++w) s += warp_sum[w];
        return s;
    };
    const double mine = block_sum(acc);
    if (threadIdx.x == 0) {
        parts[at + blockIdx.x] = mine;
        __threadfence();
        last = atomicAdd(counter, 1u) == static_cast<unsigned int>(total) - 1u;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    acc = 0.0;
    for (int i = threadIdx.x; i < total; i += THREADS) acc += __ldcg(parts + i);
    const double sum = sqrt(block_sum(acc));
    if (threadIdx.x == 0) {
        *norm = static_cast<float>(sum);
        if (clip) {
            const double f = max_norm / (sum + 1e-6);
            *clip = static_cast<float>(f > 1.0 ? 1.0 : f);  // a NaN stays one
        }
        *counter = 0u;
    }
}

// ---- the handle ---------------------------------------------------------------------------------------------

constexpr int LARGE = 768;  // tensors of a launch at most: 28 KB of arguments (limit: 32,764 bytes)
static_assert(sizeof(Table<LARGE>) + sizeof(AdamK8) + 64 <= 32764, "a launch's parameters");

int64_t padded(int64_t n) { return (n + BLOCK8 - 1) / BLOCK8 * BLOCK8; }
int64_t chunks_of(int64_t len) { return (len + CHUNK - 1) / CHUNK; }

// All tensors' padded length, or -1.
int64_t padded_total(const int64_t* lens, int n) {
    int64_t p = 0;
    for (int i = 0; i < n; ++i) {
        if (lens[i] < 0 || lens[i] > (int64_t(1) << 40) - p) return -1;
        p += padded(lens[i]);
    }
    return p;
}
int64_t bytes_of(int64_t p, int state_bits) { return state_bits == 32 ? 8 * p : 2 * p + 8 * (p / BLOCK8); }

struct Range {
    const char *lo, *hi;
};

}  // namespace

struct WbAdamMulti {
    WbBackend* b = nullptr;
    int bits = 32;
    int64_t padded = 0;
    char* state = nullptr;
    bool grads_set = false;
    std::vector<int64_t> lens, offsets;
    std::vector<Table<LARGE>> launches;   // the tensors in runs of at most LARGE
    std::vector<Range> thetas;            // sorted; then the state
    void* work = nullptr;                 // the norm's counter (16 bytes) and parts
    size_t work_class = 0;
    std::vector<int> norm_grids;
    int norm_parts = 0;
};

namespace {

// Whether [lo, hi) touches a parameter or the state.
bool touches(const WbAdamMulti* h, const void* p, int64_t bytes) {
    const char *lo = static_cast<const char*>(p), *hi = lo + bytes;
    auto it = std::lower_bound(h->thetas.begin(), h->thetas.end(), hi, [](const Range& r, const char* q) { return r.lo < q; });
    return it != h->thetas.begin() && (it - 1)->hi > lo;
}

// The smallest table that holds a launch's tensors, because all arguments are copied with every launch. A call on
// tensors of 64 elements, f32 state, in a stream of calls: 33 tensors 6.5 us with the table of 768, 3.9 us with that
// of 128; 300 tensors 6.4 and 4.8 us (320).
template <int N, class F>
int with_table(const Table<LARGE>& t, int l, F&& launch) {
    if constexpr (N == LARGE) {
        return launch(l, t);
    } else {
        Table<N> s;
        s.n = t.n;
        s.shift = t.shift;
        s.chunks = t.chunks;
        std::copy(t.hint, t.hint + HINTS + 1, s.hint);
        std::copy(t.first, t.first + t.n, s.first);
        std::copy(t.t, t.t + t.n, s.t);
        return launch(l, s);
    }
}

template <class F>
int per_launch(WbAdamMulti* h, F&& launch) {
    for (size_t l = 0; l < h->launches.size(); ++l) {
        const Table<LARGE>& t = h->launches[l];
        const int i = static_cast<int>(l);
        WB_TRY(t.n <= 32    ? with_table<32>(t, i, launch)
               : t.n <= 128 ? with_table<128>(t, i, launch)
               : t.n <= 320 ? with_table<320>(t, i, launch)
                            : with_table<LARGE>(t, i, launch));
    }
    return WB_OK;
}

int create(WbBackend* b, const WbAdamTensor* tensors, int n, int state_bits, void* state, int64_t state_bytes, int keep_state, WbAdamMulti* h) {
    h->b = b;
    h->bits = state_bits;
    h->state = static_cast<char*>(state);
    h->lens.resize(n);
    for (int i = 0; i < n; ++i) h->lens[i] = tensors[i].len;
    h->padded = padded_total(h->lens.data(), n);
    WB_REQUIRE(h->padded >= 0, WB_ERR_INVALID, "wb_adam_multi_create: a length is negative or too large");
    const int64_t need = bytes_of(h->padded, state_bits);
    WB_REQUIRE(need == 0 || (state && state_bytes >= need), WB_ERR_INVALID, "wb_adam_multi_create: the state holds %lld bytes, %lld are needed",
               static_cast<long long>(state ? state_bytes : 0), static_cast<long long>(need));
    WB_REQUIRE(reinterpret_cast<uintptr_t>(state) % 16 == 0, WB_ERR_INVALID, "wb_adam_multi_create: the state is not aligned to 16 bytes");
    for (int i = 0; i < n; ++i) {
        WB_REQUIRE(tensors[i].theta || tensors[i].len == 0, WB_ERR_INVALID, "wb_adam_multi_create: tensor %d is null", i);
        WB_REQUIRE(reinterpret_cast<uintptr_t>(tensors[i].theta) % 4 == 0, WB_ERR_INVALID, "wb_adam_multi_create: tensor %d is not aligned to 4 bytes", i);
        if (tensors[i].len == 0) continue;
        const char* lo = reinterpret_cast<const char*>(tensors[i].theta);
        h->thetas.push_back({lo, lo + 4 * tensors[i].len});
    }
    if (need) h->thetas.push_back({h->state, h->state + need});
    std::sort(h->thetas.begin(), h->thetas.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
    for (size_t i = 1; i < h->thetas.size(); ++i)
        WB_REQUIRE(h->thetas[i - 1].hi <= h->thetas[i].lo, WB_ERR_INVALID, "wb_adam_multi_create: two tensors, or a tensor and the state, overlap");
    int64_t offset = 0;
    for (int i = 0; i < n; ++i) {
        h->offsets.push_back(offset);
        if (h->launches.empty() || h->launches.back().n == LARGE || h->launches.back().chunks + chunks_of(h->lens[i]) > INT32_MAX) {
            h->launches.emplace_back();
            h->launches.back().n = 0;

            h->launches.back().chunks = 0;
        }
        Table<LARGE>& t = h->launches.back();
        t.first[t.n] = t.chunks;
        t.t[t.n] = {tensors[i].theta, nullptr, offset, tensors[i].no_decay ? -h->lens[i] : h->lens[i]};
        t.n++;
        t.chunks += static_cast<unsigned int>(chunks_of(h->lens[i]));
        offset += padded(h->lens[i]);
    }
    for (auto& t : h->launches) {
        t.shift = 0;
        while ((t.chunks >> t.shift) >= HINTS) t.shift++;
        for (int i = 0, k = 0; i <= HINTS; ++i) {
            while (k + 1 < t.n && t.first[k + 1] <= (static_cast<uint64_t>(i) << t.shift)) k++;
            t.hint[i] = static_cast<uint16_t>(k);
        }
        // at least one block: the norm of nothing is still written
        const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(t.chunks, 8 * b->sm_count)));
        h->norm_grids.push_back(grid);
        h->norm_parts += grid;
    }
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    WB_CHECK_CUDA(cudaStreamIsCapturing(b->stream, &capture));
    WB_REQUIRE(capture == cudaStreamCaptureStatusNone, WB_ERR_INVALID, "wb_adam_multi_create: the stream is being captured; a replay would zero the state");
    WB_TRY(wb_arena_alloc(b, 16 + sizeof(double) * static_cast<size_t>(h->norm_parts), &h->work, &h->work_class));
    WB_CHECK_CUDA(cudaMemsetAsync(h->work, 0, 16, b->stream));
    if (need && !keep_state) WB_CHECK_CUDA(cudaMemsetAsync(state, 0, static_cast<size_t>(need), b->stream));
    return WB_OK;
}

}  // namespace

extern "C" int64_t wb_adam_multi_state_bytes(const int64_t* lens, int n, int state_bits) {
    if (!lens || n < 1 || (state_bits != 32 && state_bits != 8)) return -1;
    const int64_t p = padded_total(lens, n);
    return p < 0 ? -1 : bytes_of(p, state_bits);
}

extern "C" int wb_adam_multi_create(WbBackend* b, const WbAdamTensor* tensors, int n, int state_bits, void* state, int64_t state_bytes, int keep_state,
                                    WbAdamMulti** out) {
    WB_REQUIRE(b && tensors && out, WB_ERR_INVALID, "wb_adam_multi_create: null pointer");
    WB_REQUIRE(n >= 1, WB_ERR_INVALID, "wb_adam_multi_create: no tensors");
    WB_REQUIRE(state_bits == 32 || state_bits == 8, WB_ERR_UNSUPPORTED, "wb_adam_multi_create: the state has 32 or 8 bits, not %d", state_bits);
    WbAdamMulti* h = nullptr;
    int status;
    try {
        h = new WbAdamMulti();
        status = create(b, tensors, n, state_bits, state, state_bytes, keep_state, h);
    } catch (const std::exception&) {
        wb_set_error("wb_adam_multi_create: out of host memory");
        status = WB_ERR_OOM;
    }
    if (status != WB_OK) {
        wb_adam_multi_destroy(h);
        return status;
    }
    *out = h;
    return WB_OK;
}

extern "C" int wb_adam_multi_destroy(WbAdamMulti* h) {
    if (!h) return WB_OK;
    if (h->work) wb_arena_free(h->b, h->work, h->work_class);
    delete h;
    return WB_OK;
}

extern "C" int64_t wb_adam_multi_state_len(const WbAdamMulti* h) { return h ? h->padded : -1; }

extern "C" int64_t wb_adam_multi_offset(const WbAdamMulti* h, int index) {
    return h && index >= 0 && index < static_cast<int>(h->offsets.size()) ? h->offsets[index] : -1;
}

extern "C" int wb_adam_multi_set_grads(WbAdamMulti* h, const float* const* grads, int n) {
    WB_REQUIRE(h && grads, WB_ERR_INVALID, "wb_adam_multi_set_grads: null pointer");
    WB_REQUIRE(n == static_cast<int>(h->lens.size()), WB_ERR_INVALID, "wb_adam_multi_set_grads: %d gradients for %zu tensors", n, h->lens.size());
    for (int i = 0; i < n; ++i) {
        if (!grads[i] || h->lens[i] == 0) continue;
        WB_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % 4 == 0, WB_ERR_INVALID, "wb_adam_multi_set_grads: gradient %d is not aligned to 4 bytes", i);
        WB_REQUIRE(!touches(h, grads[i], 4 * h->lens[i]), WB_ERR_INVALID, "wb_adam_multi_set_grads: gradient %d overlaps a parameter or the state", i);
    }
    int i = 0;
    for (auto& t : h->launches)
        for (int k = 0; k < t.n; ++k) t.t[k].grad = grads[i++];
    h->grads_set = true;
    return WB_OK;
}

extern "C" int wb_adam_multi_grad_norm(WbAdamMulti* h, double max_norm, float* norm, float* clip_scale) {
    WB_REQUIRE(h && norm, WB_ERR_INVALID, "wb_adam_multi_grad_norm: null pointer");
    WB_REQUIRE(h->grads_set, WB_ERR_INVALID, "wb_adam_multi_grad_norm: no gradients were set");
    WB_REQUIRE((reinterpret_cast<uintptr_t>(norm) | reinterpret_cast<uintptr_t>(clip_scale)) % 4 == 0 && norm != clip_scale, WB_ERR_INVALID,
               "wb_adam_multi_grad_norm: the two outputs are one, or not aligned to 4 bytes");
    WB_REQUIRE(!touches(h, norm, 4) && !(clip_scale && touches(h, clip_scale, 4)), WB_ERR_INVALID,
               "wb_adam_multi_grad_norm: an output lies in a parameter or the state");
    WB_REQUIRE(!clip_scale || max_norm > 0.0, WB_ERR_INVALID, "wb_adam_multi_grad_norm: the largest norm has to be above 0, got %g", max_norm);
    WbBackend* b = h->b;
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WbProfileScope ps(b, "grad_norm");
    unsigned int* counter = static_cast<unsigned int*>(h->work);
    double* parts = reinterpret_cast<double*>(static_cast<char*>(h->work) + 16);
    int at = 0;
    const int status = per_launch(h, [&](int l, const auto& tab) -> int {
        constexpr int N = sizeof(tab.first) / sizeof(tab.first[0]);
        WB_CHECK_CUDA(wb_launch_pdl(grad_norm_kernel<N>, dim3(h->norm_grids[l]), dim3(THREADS), 0, b->stream, tab, parts, at, h->norm_parts, counter,
                                    max_norm, norm, clip_scale));
        WB_LAUNCH_OK(b);
        at += h->norm_grids[l];
        return WB_OK;
    });
    if (status != WB_OK) (void)cudaMemsetAsync(counter, 0, sizeof(unsigned int), b->stream);  // some blocks of this call will not arrive
    return status;
}

extern "C" int wb_adam_multi_step(WbAdamMulti* h, const WbAdamConfig* cfg, int64_t t, double grad_scale, const float* device_grad_scale) {
    WB_REQUIRE(h && cfg, WB_ERR_INVALID, "wb_adam_multi_step: null pointer");
    WB_REQUIRE(h->grads_set, WB_ERR_INVALID, "wb_adam_multi_step: no gradients were set");
    WB_REQUIRE(reinterpret_cast<uintptr_t>(device_grad_scale) % 4 == 0, WB_ERR_INVALID, "wb_adam_multi_step: the scale is not aligned to 4 bytes");
    WB_REQUIRE(!device_grad_scale || !touches(h, device_grad_scale, 4), WB_ERR_INVALID, "wb_adam_multi_step: the scale lies in a parameter or the state");
    WB_REQUIRE(t >= 1 && t <= INT32_MAX, WB_ERR_INVALID, "wb_adam_multi_step: step counts from 1 to 2^31 - 1");
    WbBackend* b = h->b;
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WbProfileScope ps(b, h->bits == 32 ? "adam_multi" : "adam_multi_8bit");
    const AdamK k = wb_adam_constants(t, cfg->lr, cfg->beta1, cfg->beta2, cfg->eps, cfg->weight_decay, cfg->decoupled, grad_scale);
    AdamK8 k8;
    auto twice = [](float v) {
        uint32_t bits;
        memcpy(&bits, &v, 4);
        return Pair<float>{static_cast<uint64_t>(bits) << 32 | bits};
    };
    k8.b1 = twice(k.b1);
    k8.omb1 = twice(k.omb1);
    k8.b2 = twice(k.b2);
    k8.omb2 = twice(k.omb2);
    k8.minus_inv_sqrt_bc2 = twice(-k.inv_sqrt_bc2);
    k8.minus_eps = twice(-k.eps);
    k8.inv_sqrt_bc2 = k.inv_sqrt_bc2;
    k8.eps = k.eps;
    k8.step = k.step_size;
    k8.eps_normal = k.eps >= LOW_M && k.eps <= TOP_M && k.inv_sqrt_bc2 <= 1048576.f;
    k8.minus_step = twice(-k.step_size);
    k8.minus_zero = twice(-0.f);
    k8.gscale = k.scale_grad ? k.gscale : 1.f;
    k8.decay_mul = k.has_wd && k.decoupled ? k.decay_mul : 1.f;
    k8.wd = k.wd;
    k8.l2 = k.has_wd && !k.decoupled;
    const int64_t p = h->padded;
    return per_launch(h, [&](int, const auto& tab) -> int {
        constexpr int N = sizeof(tab.first) / sizeof(tab.first[0]);
        if (tab.chunks == 0) return WB_OK;
        if (h->bits == 32) {
            float* m = reinterpret_cast<float*>(h->state);
            WB_CHECK_CUDA(wb_launch_pdl(adam_multi32_kernel<N>, dim3(tab.chunks), dim3(THREADS), 0, b->stream, tab, m, m + p, k, device_grad_scale));
        } else {
            float* scales = reinterpret_cast<float*>(h->state + 2 * p);
            WB_CHECK_CUDA(wb_launch_pdl(k.first ? adam_multi8_kernel<N, true> : adam_multi8_kernel<N, false>, dim3(tab.chunks), dim3(THREADS), 0, b->stream, tab, reinterpret_cast<uint32_t*>(h->state),
                                        reinterpret_cast<uint32_t*>(h->state + p), scales, scales + p / BLOCK8, k8, device_grad_scale));
        }
        WB_LAUNCH_OK(b);
        return WB_OK;
    });
}

extern "C" int wb_adam_multi_read_state(WbAdamMulti* h, float* m, float* v) {
    WB_REQUIRE(h && (m || v), WB_ERR_INVALID, "wb_adam_multi_read_state: null pointer");
    if (h->padded == 0) return WB_OK;
    WbBackend* b = h->b;
    const int64_t p = h->padded;
    const char* state = h->state;
    const WbSpan spans[3] = {{state, state + bytes_of(p, h->bits), false},
                             {reinterpret_cast<char*>(m), reinterpret_cast<char*>(m) + (m ? 4 * p : 0), true},
                             {reinterpret_cast<char*>(v), reinterpret_cast<char*>(v) + (v ? 4 * p : 0), true}};
    WB_REQUIRE(!wb_spans_clash(spans, 3), WB_ERR_INVALID, "wb_adam_multi_read_state: the outputs overlap each other or the state");
    WB_REQUIRE((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) % 4 == 0, WB_ERR_INVALID,
               "wb_adam_multi_read_state: an output is not aligned to 4 bytes");
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WbProfileScope ps(b, "adam_multi_read_state");
    if (h->bits == 32) {
        if (m) WB_CHECK_CUDA(cudaMemcpyAsync(m, state, static_cast<size_t>(4 * p), cudaMemcpyDeviceToDevice, b->stream));
        if (v) WB_CHECK_CUDA(cudaMemcpyAsync(v, state + 4 * p, static_cast<size_t>(4 * p), cudaMemcpyDeviceToDevice, b->stream));
        return WB_OK;
    }
    const float* scales = reinterpret_cast<const float*>(state + 2 * p);
    const int64_t groups = p / 4, grid = (groups + THREADS - 1) / THREADS;
    WB_REQUIRE(grid <= INT32_MAX, WB_ERR_INVALID, "wb_adam_multi_read_state: state too large");
    const int wide = ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    WB_CHECK_CUDA(wb_launch_pdl(adam_multi8_read_kernel, dim3(static_cast<unsigned>(grid)), dim3(THREADS), 0, b->stream,
                                reinterpret_cast<const uint32_t*>(state), reinterpret_cast<const uint32_t*>(state + p), scales, scales + p / BLOCK8, m, v,
                                groups, wide));
    WB_LAUNCH_OK(b);
    return WB_OK;
}

extern "C" int wb_adam_multi_selftest_rounding(WbBackend* b, int64_t* wrong) {
    WB_REQUIRE(b && wrong, WB_ERR_INVALID, "wb_adam_multi_selftest_rounding: null pointer");
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    void* counts = nullptr;
    size_t klass = 0;
    WB_TRY(wb_arena_alloc(b, 4 * sizeof(int64_t), &counts, &klass));
    cudaError_t e = cudaMemsetAsync(counts, 0, 4 * sizeof(int64_t), b->stream);
    if (e == cudaSuccess) {
        adam_rounding_selftest_kernel<<<8 * b->sm_count, THREADS, 0, b->stream>>>(static_cast<unsigned long long*>(counts));
        b->launches++;
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) {
        e = cudaMemcpyAsync(wrong, counts, 4 * sizeof(int64_t), cudaMemcpyDeviceToHost, b->stream);
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(b->stream);
    wb_arena_free(b, counts, klass);
    WB_CHECK_CUDA(e);
    return WB_OK;
}
