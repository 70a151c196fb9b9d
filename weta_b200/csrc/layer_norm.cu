// Layer normalisation over the last dims of a strided view, forward and backward
// (crates/weta-nn/src/functional.rs:183-195 and the gradients autograd derives through it):
//   mu = mean_c x,  rstd = 1 / sqrt(mean_c (x - mu)^2 + eps),  xhat = (x - mu) rstd,  y = xhat w + b
//   g = dy w,  dx = rstd (g - mean_c g - xhat mean_c (g xhat)),  dw = sum_r dy xhat,  db = sum_r dy
// The view is taken as [rows, cols]: cols is the product of the normalised dims.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.h"
#include "pair.cuh"

namespace {

constexpr int THREADS = 256;

// Where the elements of a view lie: collapsed outer dims (rows) and collapsed inner dims (columns).
struct RowView {
    int nd_row, nd_col;
    int64_t size_row[WB_MAX_DIMS], st_row[WB_MAX_DIMS], size_col[WB_MAX_DIMS], st_col[WB_MAX_DIMS];
};

__device__ __forceinline__ int64_t offset_of(int64_t i, int nd, const int64_t* size, const int64_t* st) {
    int64_t off = 0;
    for (int d = nd - 1; d > 0; --d) {
        const int64_t q = i / size[d];
        off += (i - q * size[d]) * st[d];
        i = q;
    }
    return off + i * st[0];
}
__device__ __forceinline__ int64_t row_offset(const RowView& v, int64_t row) { return offset_of(row, v.nd_row, v.size_row, v.st_row); }
__device__ __forceinline__ int64_t col_offset(const RowView& v, int64_t col) {
    return v.nd_col == 1 ? col * v.st_col[0] : offset_of(col, v.nd_col, v.size_col, v.st_col);
}

// Sum over the block, returned to every thread; `part` holds one value per warp and may be used again at once.
__device__ __forceinline__ double block_sum(double v, double* part) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) s += part[w];
    return s;
}

// ---- any view: one block per row, the row read from memory once per pass, sums in f64 -------------------

template <class T>
__global__ void __launch_bounds__(THREADS) ln_fwd_any_kernel(const T* __restrict__ x, RowView vx, int64_t rows, int64_t cols, const T* __restrict__ w,
                                                             const T* __restrict__ bias, double eps, T* __restrict__ y, T* __restrict__ mean_out,
                                                             T* __restrict__ rstd_out) {
    __shared__ double part[THREADS / 32];
    wb_pdl_enter();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row_offset(vx, row);
        double s = 0.0;
        for (int64_t c = threadIdx.x; c < cols; c += THREADS) s += static_cast<double>(xr[col_offset(vx, c)]);
        const double mean = block_sum(s, part) / static_cast<double>(cols);
        double q = 0.0;
        for (int64_t c = threadIdx.x; c < cols; c += THREADS) {
            const double d = static_cast<double>(xr[col_offset(vx, c)]) - mean;
            q += d * d;
        }
        const double rstd = 1.0 / sqrt(block_sum(q, part) / static_cast<double>(cols) + eps);
        for (int64_t c = threadIdx.x; c < cols; c += THREADS) {
            double o = (static_cast<double>(xr[col_offset(vx, c)]) - mean) * rstd;
            if (w) o *= static_cast<double>(w[c]);
            if (bias) o += static_cast<double>(bias[c]);
            y[row * cols + c] = static_cast<T>(o);
        }
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = static_cast<T>(mean);
            if (rstd_out) rstd_out[row] = static_cast<T>(rstd);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS) ln_dx_any_kernel(const T* __restrict__ x, RowView vx, const T* __restrict__ dy, RowView vg, int64_t rows,
                                                            int64_t cols, const T* __restrict__ w, const T* __restrict__ mean,
                                                            const T* __restrict__ rstd, T* __restrict__ dx) {
    __shared__ double part[THREADS / 32];
    wb_pdl_enter();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row_offset(vx, row);
        const T* gr = dy + row_offset(vg, row);
        const double mu = mean[row], rs = rstd[row];
        double s = 0.0, p = 0.0;
        for (int64_t c = threadIdx.x; c < cols; c += THREADS) {
            const double g = static_cast<double>(gr[col_offset(vg, c)]) * (w ? static_cast<double>(w[c]) : 1.0);
            s += g;
            p += g * ((static_cast<double>(xr[col_offset(vx, c)]) - mu) * rs);
        }
        s = block_sum(s, part) / static_cast<double>(cols);
        p = block_sum(p, part) / static_cast<double>(cols);
        for (int64_t c = threadIdx.x; c < cols; c += THREADS) {
            const double g = static_cast<double>(gr[col_offset(vg, c)]) * (w ? static_cast<double>(w[c]) : 1.0);
            const double xh = (static_cast<double>(xr[col_offset(vx, c)]) - mu) * rs;
            dx[row * cols + c] = static_cast<T>(rs * (g - s - xh * p));
        }
    }
}

// ---- rows of unit stride ---------------------------------------------------------------------------------
// TPR threads hold one row in registers: vector j of thread t covers columns (j TPR + t) VEC ..., so every access of a
// warp is one contiguous run.  Rows are `pitch` elements apart.

template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

// Sum over the TPR threads of a row, returned to all of them.  Rows of more than a warp meet at the barrier of their
// group (`bar`, at least 1; the block's own where it is one group: a barrier known only at run time reserves all sixteen,
// which let four blocks onto an SM) and join the warps' sums, `part` (2 K warps), in a second tree; two buffers in turn make one
// barrier per sum enough.  `after_barrier` runs there.
struct Nothing {
    __device__ __forceinline__ void operator()() const {}
};
template <class T, int TPR, int G, int K, class F = Nothing>
__device__ __forceinline__ void row_sum(T (&v)[K], T* part, int bar, unsigned int& turn, F&& after_barrier = F()) {
#pragma unroll
    for (int d = (TPR < 32 ? TPR : 32) / 2; d > 0; d >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int lane = threadIdx.x & 31, warp = threadIdx.x % TPR >> 5;
        T* mine = part + (turn & 1) * K * W;
        ++turn;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) mine[k * W + warp] = v[k];
        if constexpr (G == 1) __syncthreads();
        else asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(TPR) : "memory");
        after_barrier();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            T s = mine[k * W + lane % W];
#pragma unroll
            for (int d = W / 2; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            v[k] = s;
        }
    }
}

// s / n, correctly rounded, from y = 1 / n correctly rounded: the quotient's exact residual corrects it (Markstein's theorem, as
// in adam_multi.cu).  The mean of equal values then is that value where their sum is exact, which s y misses by a unit, and a
// division in its place made the forward pass of [8192, 4096] in f64 107 us instead of 83.
template <class T>
__device__ __forceinline__ T divide(T s, T n, T y) {
    const T q = s * y, r = fma(-q, n, s);
    return r == r ? fma(r, y, q) : q;  // the residual of what is not finite is NaN
}

template <int TPR>
constexpr int fwd_threads = TPR < 64 ? 128 : TPR;

template <class T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(fwd_threads<TPR>) ln_fwd_rows_kernel(const T* __restrict__ x, int64_t pitch, int64_t rows, int cols,
                                                                       const T* __restrict__ w, const T* __restrict__ bias, T eps, T inv_cols,
                                                                       T* __restrict__ y, T* __restrict__ mean_out, T* __restrict__ rstd_out) {
    constexpr int G = fwd_threads<TPR> / TPR;
    __shared__ T part[G][TPR > 32 ? 2 * TPR / 32 : 1];
    wb_pdl_enter();
    const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * G + group;
    const bool live = row < rows;  // the other rows of a warp still need this one in their shuffles
    if (TPR >= 32 && !live) return;
    const T* xr = x + row * pitch;
    Pack<T, VEC> a[NV];
    T s[1] = {0};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * VEC;
        if (live && c < cols) a[j] = load_pack<T, VEC>(xr + c);
        else
#pragma unroll
            for (int i = 0; i < VEC; ++i) a[j].v[i] = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[0] += a[j].v[i];
    }
    unsigned int turn = 0;
    row_sum<T, TPR, G, 1>(s, part[group], 1 + group, turn);
    const T mean = divide(s[0], static_cast<T>(cols), inv_cols);
    T q[1] = {0};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const bool in = (j * TPR + t) * VEC < cols;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            a[j].v[i] -= mean;
            if (in) q[0] += a[j].v[i] * a[j].v[i];
        }
    }
    row_sum<T, TPR, G, 1>(q, part[group], 1 + group, turn);
    const T rstd = T(1) / sqrt(q[0] * inv_cols + eps);
    if (!live) return;
    T* yr = y + row * cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * VEC;
        if (c < cols) {
            Pack<T, VEC> o, pw, pb;
            if (w) pw = load_pack<T, VEC>(w + c);
            if (bias) pb = load_pack<T, VEC>(bias + c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                o.v[i] = a[j].v[i] * rstd;
                if (w) o.v[i] *= pw.v[i];
                if (bias) o.v[i] += pb.v[i];
            }
            *reinterpret_cast<Pack<T, VEC>*>(yr + c) = o;
        }
    }
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// ---- rows through a ring in shared memory --------------------------------------------------------------------
// A group of threads walks spans: R rows that follow each other in memory (one row, or a part of it, where they do not).
// The spans ahead are fetched into a ring of two to four slots by one bulk copy for each operand, which costs the group one
// thread's instruction whatever the width.  A bulk copy takes whole 16-byte units; the elements short of a unit at either
// end of a span, and the rows' statistics, are copied beside it one by one (cp.async) by lanes of the group, so nothing
// outside the span is read.
constexpr int MOST_RING = 4;
constexpr uint32_t POLLS = 1u << 26;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(bar)));
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes),
                 "r"(smem_addr(bar))
                 : "memory");
}
template <class T>
__device__ __forceinline__ void copy_one(T* dst, const T* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst)), "l"(src), "n"(sizeof(T)) : "memory");
}
// Bounded: after `limit` polls the backend's flag (pinned host memory, read by wb_layer_norm_check) goes up, later waits give up
// sooner and the kernel runs to its end on what is there.
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t parity, uint32_t& limit, int* gave_up) {
    const uint32_t addr = smem_addr(bar);
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done)
                     : "r"(addr), "r"(parity)
                     : "memory");
        if (done) return;
    }
    limit = POLLS >> 10;
    *reinterpret_cast<volatile int*>(gave_up) = 1;
}

template <class T>
constexpr int UNIT = 16 / static_cast<int>(sizeof(T));  // elements of 16 bytes

template <class T>
__device__ __forceinline__ int misalignment(const T* p) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (UNIT<T> - 1);
}

// How a run of n elements at p splits at 16-byte boundaries: `head` elements, `mid` in whole units, `tail`.  In shared memory
// element i lies at buf[mis + i], so that the whole units stay aligned.
template <class T>
struct Split {
    int mis, head, mid, tail;
    __device__ __forceinline__ Split(const T* p, int n) {
        mis = misalignment(p);
        head = min((UNIT<T> - mis) % UNIT<T>, n);
        mid = (n - head) / UNIT<T> * UNIT<T>;
        tail = n - head - mid;
    }
};

// Fetches a run of n elements into `buf` (the first lane of the warp, after its expect_tx) ...
template <class T>
__device__ __forceinline__ void fetch_units(T* buf, const T* p, const Split<T>& s, uint64_t* bar) {
    if (s.mid) bulk_load(buf + s.mis + s.head, p + s.head, static_cast<uint32_t>(s.mid * sizeof(T)), bar);
}
// ... and its ends, by eight lanes: k = 0 .. 7.
template <class T>
__device__ __forceinline__ void fetch_ends(T* buf, const T* p, int n, int k) {
    const Split<T> s(p, n);
    const int i = k < 4 ? k : s.head + s.mid + k - 4;
    if (k < 4 ? k < s.head : k - 4 < s.tail) copy_one(buf + s.mis + i, p + i);
}

// How rows lie to 16-byte boundaries.  ALIGNED: every row of x, dy and the result starts and ends on one, so no unit is cut.
// The others cut units at the rows' ends.  SHIFTED: the three share each row's misalignment and a slot holds one row; the other
// places of its first and last unit hold the row's mean (x) and zeros (dy), so that xhat and the gradient are 0 there.  MIXED:
// they do not share it; x and dy are read from shared memory element by element, and a cut unit's foreign elements are
// replaced.  ELEMENTS, for rows so short that a span of one row would be all overhead: no units, thread t holds the columns t,
// t + TPR, ... of rows of any misalignment.
enum { ALIGNED, SHIFTED, MIXED, ELEMENTS };

// The small copies of a row of n columns by the lanes of a warp, one each: the ends of x (lanes 0 to 7) and of dy (8 to 15), the
// row's mean into the other places of x's first and last unit (SHIFTED, 16 to 23), its rstd to stats + 32 (24) and its mean to
// the first unit of `stats` (25 on).  Where the misalignment stays the same, so does all of this but the row.
template <class T>
struct SmallCopy {
    bool on = false;
    int to = 0;  // in the slot
    const T* from = nullptr;
};
template <class T, int MODE>
__device__ __forceinline__ SmallCopy<T> small_copy(const T* x, const T* dy, int n, int at_dy, int stats, const T* mean, const T* rstd, int lane) {
    SmallCopy<T> c;
    if constexpr (MODE != ALIGNED) {
        const bool of_g = lane >= 8 && lane < 16, gap = lane >= 16, tail = lane & 4;
        const T* p = of_g ? dy : x;
        const Split<T> s(p, n);
        const int end = s.mis + n, i = lane & 3;
        const int place = i + (gap ? (tail ? end : 0) : s.mis + (tail ? s.head + s.mid : 0));
        c.on = i < (gap ? (MODE == SHIFTED ? (tail ? -end & (UNIT<T> - 1) : s.mis) : 0) : tail ? s.tail : s.head);
        c.to = (of_g ? at_dy : 0) + place;
        c.from = gap ? mean : p + place - s.mis;
    }
    if (lane >= 24) {
        c.on = lane < 25 + UNIT<T>;
        c.to = stats + (lane == 24 ? 32 : lane - 25);
        c.from = lane == 24 ? rstd : mean;
    }
    return c;
}

// Which columns a thread holds.  A row is cut into the 16-byte units of the result's memory: unit u of a row that starts `mis`
// elements behind a boundary holds columns u UNIT - mis ..., so whole units are stored at once whatever the row's length.
// Vector j of thread t is unit u0 + j TPR + t.  A group only walks rows of one misalignment, so its columns stay its own.
template <class T, int TPR, int NV>
struct Columns {
    int mis, u0, cols, t;  // cols: where the columns of this CTA end
    __device__ __forceinline__ int first(int j) const { return (u0 + j * TPR + t) * UNIT<T> - mis; }
    __device__ __forceinline__ bool some(int j) const { return first(j) < cols; }
    __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) + UNIT<T> <= cols; }
    __device__ __forceinline__ bool all_whole() const {
        bool w = true;
#pragma unroll
        for (int j = 0; j < NV; ++j) w &= whole(j);
        return w;
    }
};

struct SpanShape {
    int64_t rows, pitch_x, pitch_g, pitch_ref;
    int cols;   // of a row
    int units;  // 16-byte units of one CTA of the cluster
    int r;      // rows of a span
    int spans;
    int ring;  // slots
    int cap;   // elements of a slot's buffer
    int* gave_up;
};

// A unit from shared memory: one 16-byte load, or (where the operand's rows start at another misalignment than the result's)
// element by element.
template <class T, bool SAME>
__device__ __forceinline__ void load_unit(const T* p, Pair<T> (&v)[UNIT<T> / 2]) {
    if constexpr (SAME) {
        struct alignas(16) Raw {
            Pair<T> v[UNIT<T> / 2];
        };
        const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
        for (int i = 0; i < UNIT<T> / 2; ++i) v[i] = r.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < UNIT<T> / 2; ++i) v[i] = pair(p[2 * i], p[2 * i + 1]);
    }
}
template <class T>
__device__ __forceinline__ void store_unit(T* p, const Pair<T> (&v)[UNIT<T> / 2]) {
    struct alignas(16) Raw {
        Pair<T> v[UNIT<T> / 2];
    } r;
#pragma unroll
    for (int i = 0; i < UNIT<T> / 2; ++i) r.v[i] = v[i];
    *reinterpret_cast<Raw*>(p) = r;
}
// The elements of a unit at columns c, c + 1, ... that lie in the row.
template <class T>
__device__ __forceinline__ void store_part(T* row, int c, int cols, const Pair<T> (&v)[UNIT<T> / 2]) {
#pragma unroll
    for (int i = 0; i < UNIT<T> / 2; ++i) {
        T a, b;
        unpair(v[i], a, b);
        if (c + 2 * i >= 0 && c + 2 * i < cols) row[c + 2 * i] = a;
        if (c + 2 * i + 1 >= 0 && c + 2 * i + 1 < cols) row[c + 2 * i + 1] = b;
    }
}
template <class T>
__device__ __forceinline__ void replace_outside(int c, int cols, const T& with, Pair<T> (&v)[UNIT<T> / 2]) {
#pragma unroll
    for (int i = 0; i < UNIT<T> / 2; ++i) {
        T a, b;
        unpair(v[i], a, b);
        if (c + 2 * i < 0 || c + 2 * i >= cols) a = with;
        if (c + 2 * i + 1 < 0 || c + 2 * i + 1 >= cols) b = with;
        v[i] = pair(a, b);
    }
}

constexpr int SPAN_THREADS = 512;
constexpr int MOST_SHARED = 216 << 10;

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ int cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
    return static_cast<int>(n);
}
// The value at the same place in the shared memory of the cluster's CTA q.
template <class T>
__device__ __forceinline__ T peer_value(const T* p, int q) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(q));
    T v;
    if constexpr (sizeof(T) == 4) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    else asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
    return v;
}

// Adds the CTAs' sums of a row over the cluster: every CTA's to every CTA; two buffers in turn, as in row_sum.
template <class T, int CL, int K>
__device__ __forceinline__ void cluster_sum(T (&s)[K], T (*peers)[CL][2], int rank, unsigned int turn) {
    T(*to)[2] = peers[turn & 1];
    if (threadIdx.x < CL) {
        uint32_t remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(to[rank])), "r"(threadIdx.x));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (sizeof(T) == 4) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote + 4 * k), "f"(s[k]) : "memory");
            else asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote + 8 * k), "d"(s[k]) : "memory");
        }
    }
    cluster_sync();
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = 0;
#pragma unroll
    for (int q = 0; q < CL; ++q)
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] += to[q][k];
}

// Backward.  TPR threads hold a row; narrower rows share a warp.  The weight's and the bias's gradients of a thread's columns
// stay in its registers over all rows it sees; at the end the threads of a column are joined in shared memory and the block
// leaves one row of partials.
template <class T, int TPR, int NV, int MODE>
__global__ void __launch_bounds__(SPAN_THREADS, 1) ln_bwd_span_kernel(const T* __restrict__ x, const T* __restrict__ dy, const SpanShape sh,
                                                                     const T* __restrict__ w, const T* __restrict__ mean,
                                                                     const T* __restrict__ rstd, T inv_cols, const T* ref, T* __restrict__ dx,
                                                                     T* __restrict__ parts, T* __restrict__ dw, T* __restrict__ db) {
    constexpr int N = SPAN_THREADS, GT = TPR < 32 ? 32 : TPR, G = N / GT, SUBS = GT / TPR, U = UNIT<T>, H = U / 2, E = NV * U, LINES = N / TPR;
    constexpr bool HALVES = TPR >= 256;
    static_assert(MODE != ELEMENTS || TPR <= 32, "short rows");
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ T part[G][TPR > 32 ? 4 * TPR / 32 : 1];
    __shared__ uint64_t full[G][MOST_RING];
    __shared__ int line_mis[LINES];
    __shared__ alignas(16) T zeros[U];
    wb_pdl_enter();
    const int group = threadIdx.x / GT, g = threadIdx.x % GT, sub = g / TPR;
    const int slab = static_cast<int>(blockIdx.x), slabs = static_cast<int>(gridDim.x);
    const int groups = slabs * G, first = slab * G + group;
    Columns<T, TPR, NV> col;
    col.t = g % TPR;
    col.u0 = 0;
    col.mis = MODE == ELEMENTS ? 0 : misalignment(ref + (static_cast<int64_t>(first) * sh.r + sub) * sh.pitch_ref);
    col.cols = sh.cols;
    const bool whole = col.all_whole();
    auto column = [&](int j, int e) { return MODE == ELEMENTS ? (j * U + e) * TPR + col.t : col.first(j) + e; };
    // ring slot: a unit of room, x, a unit of room, dy, mean [32], rstd [32]
    const int slot_elems = 2 * sh.cap + 64;
    T* ring = reinterpret_cast<T*>(smem_raw) + group * sh.ring * slot_elems + U;
    if (g < sh.ring) bar_init(&full[group][g]);
    if (threadIdx.x < U) zeros[threadIdx.x] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    if constexpr (MODE == SHIFTED) {  // the ends of each buffer of dy: a unit before and after the first, all from the last on
        for (int k = 0; k < sh.ring && g < 32; ++k) {
            T* buf = ring + k * slot_elems + sh.cap;
            const int e = g < 2 * U ? g - U : max(U, sh.cols - U) + g - 2 * U;
            if (e < sh.cap - U) buf[e] = 0;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }

    Pair<T> wv[NV][H], aw[NV][H], ab[NV][H];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int c = column(j, 2 * i), d = column(j, 2 * i + 1);
            const bool a = c >= 0 && c < sh.cols, b = d >= 0 && d < sh.cols;
            wv[j][i] = pair(a ? (w ? w[c] : T(1)) : T(0), b ? (w ? w[d] : T(1)) : T(0));
            aw[j][i] = ab[j][i] = pair(T(0), T(0));
        }

    // Fetches a span, or the first (x and the small copies) or second (dy) part of it: part 0, 1 or 2.
    auto fetch = [&](int span, int slot, int part) {
        if (g >= 32) return;
        if (span < sh.spans) {
            const int64_t row0 = static_cast<int64_t>(span) * sh.r;
            const int nr = static_cast<int>(min(static_cast<int64_t>(sh.r), sh.rows - row0));
            const int n = nr * sh.cols;
            T* base = ring + slot * slot_elems;
            const T* px = x + row0 * sh.pitch_x;
            const T* pg = dy + row0 * sh.pitch_g;
            if (g == 0) {
                const Split<T> sx(px, n), sg(pg, n);
                if (part != 2) {
                    bar_expect(&full[group][slot], static_cast<uint32_t>((sx.mid + sg.mid) * sizeof(T)));
                    fetch_units(base, px, sx, &full[group][slot]);
                }
                if (part != 1) fetch_units(base + sh.cap, pg, sg, &full[group][slot]);
            }
            if (part != 2) {
                if constexpr (MODE == SHIFTED || MODE == MIXED) {  // spans of one row
                    const SmallCopy<T> c = small_copy<T, MODE>(px, pg, n, sh.cap, 2 * sh.cap - U, mean + row0, rstd + row0, g);
                    if (c.on) copy_one(base + c.to, c.from);
                } else {
                    if (MODE == ELEMENTS && g < 16) fetch_ends(base + (g < 8 ? 0 : sh.cap), g < 8 ? px : pg, n, g & 7);
                    if (g < nr) {
                        copy_one(base + 2 * sh.cap - U + g, mean + row0 + g);
                        copy_one(base + 2 * sh.cap - U + 32 + g, rstd + row0 + g);
                    }
                }
            }
        }
        if (part != 2) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // As many spans as the ring has slots are under way at a time.  A slot is filled again as soon as every thread of the
    // group holds the slot's values in registers: in rows of more than a warp that is at the barrier inside the row's sum.
    // Before that barrier the small copies of the next span have arrived, so that it makes them known, too.
    auto settle = [&](int pending) {
        if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
        else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else asm volatile("cp.async.wait_group 3;" ::: "memory");
    };
    for (int k = 0; k < sh.ring; ++k) fetch(first + k * groups, k, 0);
    settle(sh.ring - 1);
    __syncthreads();

    unsigned int turn = 0;
    uint32_t limit = POLLS, phase = 0;
    int slot = 0;
    for (int span = first; span < sh.spans; span += groups) {
        bar_wait(&full[group][slot], phase, limit, sh.gave_up);
        if (HALVES && span != first) fetch(span + (sh.ring - 1) * groups, slot == 0 ? sh.ring - 1 : slot - 1, 2);
        const int64_t row0 = static_cast<int64_t>(span) * sh.r;
        const int nr = static_cast<int>(min(static_cast<int64_t>(sh.r), sh.rows - row0));
        const T* base = ring + slot * slot_elems;
        // unit j of row r starts at base[off + r cols + (j TPR + t) U]
        const int shift = MODE == ELEMENTS ? 0 : col.t * U - col.mis;
        const T *span_x = base + shift, *span_g = base + sh.cap + shift;
        if (MODE != ALIGNED) {
            span_x += misalignment(x + row0 * sh.pitch_x);
            span_g += misalignment(dy + row0 * sh.pitch_g);
        }
        for (int r0 = 0; r0 < nr; r0 += SUBS) {  // the same number of turns for every lane of a warp
            const bool live = SUBS == 1 || r0 + sub < nr;
            const int r = live ? r0 + sub : r0;
            const T *bx = span_x + r * sh.cols, *bg = span_g + r * sh.cols;
            const T mu = base[2 * sh.cap - U + r], rs = base[2 * sh.cap - U + 32 + r];
            const Pair<T> minus_mu = pair(-mu, -mu), rs2 = pair(rs, rs);
            // xhat is 0 where there is no column: (0 - mu) rs may be infinite, which no weight makes nothing of
            const Pair<T> minus_last = MODE == MIXED || MODE == ELEMENTS || col.some(NV - 1) ? minus_mu : pair(T(0), T(0));
            Pair<T> xh[NV][H], gv[NV][H], s0 = pair(T(0), T(0)), s1 = s0;
            auto take = [&](auto edges) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    Pair<T> up[H];
                    if constexpr (MODE == ELEMENTS) {
#pragma unroll
                        for (int i = 0; i < H; ++i) {
                            const int c = column(j, 2 * i), d = column(j, 2 * i + 1);
                            const bool a = c < sh.cols, b = d < sh.cols;
                            xh[j][i] = pair(a ? bx[c] : mu, b ? bx[d] : mu);
                            up[i] = pair(a ? bg[c] : T(0), b ? bg[d] : T(0));
                        }
                    } else {
                        // a unit behind the row's end (of the last vector only, in a row of its own): zeros, since no weight makes
                        // nothing of an infinity
                        const bool there = j < NV - 1 || col.some(j);
                        load_unit<T, MODE != MIXED>(there ? bx + j * TPR * U : zeros, xh[j]);
                        load_unit<T, MODE != MIXED>(there ? bg + j * TPR * U : zeros, up);
                    }
                    if constexpr (decltype(edges)::value) {  // what is not of this row counts as a mean value without gradient
                        replace_outside(col.first(j), sh.cols, mu, xh[j]);
                        replace_outside(col.first(j), sh.cols, T(0), up);
                    }
#pragma unroll
                    for (int i = 0; i < H; ++i) {
                        xh[j][i] = (xh[j][i] + (j < NV - 1 ? minus_mu : minus_last)) * rs2;
                        gv[j][i] = up[i] * wv[j][i];
                        aw[j][i] = muladd(up[i], xh[j][i], aw[j][i]);
                        ab[j][i] = ab[j][i] + up[i];
                        s0 = s0 + gv[j][i];
                        s1 = muladd(gv[j][i], xh[j][i], s1);
                    }
                }
            };
            if (live) {
                if (MODE != MIXED || whole) take(std::false_type{});
                else take(std::true_type{});
            }
            if (!dx) continue;
            T s[2], lo, hi;
            unpair(s0, lo, hi);
            s[0] = lo + hi;
            unpair(s1, lo, hi);
            s[1] = lo + hi;
            if constexpr (TPR > 32) settle(sh.ring - 2);
            row_sum<T, TPR, G, 2>(s, part[group], 1 + group, turn, [&]() { fetch(span + sh.ring * groups, slot, HALVES ? 1 : 0); });
            const T k0 = -rs * (s[0] * inv_cols), k1 = -rs * (s[1] * inv_cols);
            const Pair<T> k0p = pair(k0, k0), k1p = pair(k1, k1);
            if (live) {
                T* dr = dx + (row0 + r) * sh.cols;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    Pair<T> o[H];
#pragma unroll
                    for (int i = 0; i < H; ++i) o[i] = muladd(gv[j][i], rs2, muladd(xh[j][i], k1p, k0p));
                    if constexpr (MODE == ELEMENTS) {
#pragma unroll
                        for (int i = 0; i < H; ++i) {
                            T a, b;
                            unpair(o[i], a, b);
                            if (column(j, 2 * i) < sh.cols) dr[column(j, 2 * i)] = a;
                            if (column(j, 2 * i + 1) < sh.cols) dr[column(j, 2 * i + 1)] = b;
                        }
                    } else if (MODE == ALIGNED ? j < NV - 1 || col.some(j) : whole || col.whole(j)) store_unit(dr + col.first(j), o);
                    else if (MODE != ALIGNED && (j < NV - 1 || col.some(j))) store_part(dr, col.first(j), sh.cols, o);
                }
            }
        }
        if (GT == 32 || !dx) {
            settle(sh.ring - 2);
            if constexpr (GT == 32) __syncwarp();
            else if constexpr (G == 1) __syncthreads();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GT) : "memory");
            fetch(span + sh.ring * groups, slot, HALVES ? 1 : 0);
        }
        slot = slot == sh.ring - 1 ? 0 : slot + 1;
        phase ^= slot == 0;
    }
    if (!parts) return;
    __syncthreads();
    // one line for each row that the block holds at a time, added up in order
    T* joined = reinterpret_cast<T*>(smem_raw);  // [2][LINES][TPR E], then (a cluster's blocks) the block's sums [2][cols]
    T* sums = joined + 2 * LINES * TPR * E;
    const bool cluster = cluster_size() > 1;
    const int line = threadIdx.x / TPR;
    if (col.t == 0) line_mis[line] = col.mis;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if constexpr (MODE == ELEMENTS) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                T a, b;
                unpair(aw[j][i / 2], a, b);
                joined[line * TPR * E + column(j, i)] = i % 2 ? b : a;
                unpair(ab[j][i / 2], a, b);
                joined[(LINES + line) * TPR * E + column(j, i)] = i % 2 ? b : a;
            }
        } else {
            T* a = joined + line * TPR * E + (j * TPR + col.t) * U;
            store_unit(a, aw[j]);
            store_unit(a + LINES * TPR * E, ab[j]);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < sh.cols; c += N) {
        T sw = 0, sb = 0;
        for (int k = 0; k < LINES; ++k) {
            const T* a = joined + k * TPR * E + c + line_mis[k];
            sw += a[0];
            sb += a[LINES * TPR * E];
        }
        if (cluster) {
            sums[c] = sw;
            sums[sh.cols + c] = sb;
        } else if (slabs == 1) {  // nothing to join
            if (dw) dw[c] = sw;
            if (db) db[c] = sb;
        } else {
            parts[static_cast<int64_t>(slab) * sh.cols + c] = sw;
            parts[static_cast<int64_t>(slabs + slab) * sh.cols + c] = sb;
        }
    }
    if (!cluster) return;
    cluster_sync();  // every block's sums are there; each block adds up its share of the columns, in the blocks' order
    for (int c = slab * N + static_cast<int>(threadIdx.x); c < sh.cols; c += slabs * N) {
        T sw = 0, sb = 0;
        for (int q = 0; q < slabs; ++q) {
            sw += peer_value(sums + c, q);
            sb += peer_value(sums + sh.cols + c, q);
        }
        if (dw) dw[c] = sw;
        if (db) db[c] = sb;
    }
    cluster_sync();  // no block leaves while its sums are read
}

// Backward of rows wider than 512 threads hold: a cluster of CTAs takes the row, each its slice of the columns, and they
// exchange the two sums.  A row goes through two passes over its slot, the first for the sums and the columns' gradients, the
// second for dx; the cluster's barrier for one row is waited for only after the next row's first pass, which hides it.
template <class T, int NV, int CL, int MODE>
__global__ void __launch_bounds__(SPAN_THREADS, 1) ln_bwd_wide_kernel(const T* __restrict__ x, const T* __restrict__ dy, const SpanShape sh,
                                                                     const T* __restrict__ w, const T* __restrict__ mean,
                                                                     const T* __restrict__ rstd, T inv_cols, const T* ref, T* __restrict__ dx,
                                                                     T* __restrict__ parts, T* __restrict__ dw, T* __restrict__ db) {
    constexpr int TPR = SPAN_THREADS, U = UNIT<T>, H = U / 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ T part[4 * TPR / 32];
    __shared__ T peers[2][CL][2];
    __shared__ uint64_t full[MOST_RING];
    __shared__ alignas(16) T zeros[U];
    wb_pdl_enter();
    const int t = threadIdx.x, rank = static_cast<int>(blockIdx.x) % CL, slab = static_cast<int>(blockIdx.x) / CL, slabs = static_cast<int>(gridDim.x) / CL;
    Columns<T, TPR, NV> col;
    col.t = t;
    col.u0 = rank * sh.units;
    col.mis = misalignment(ref + slab * sh.pitch_ref);
    const int from = max(0, col.u0 * U - col.mis), to = min(sh.cols, (col.u0 + sh.units) * U - col.mis);  // this CTA's columns
    col.cols = to;
    const bool whole = col.all_whole();
    const int slot_elems = 2 * sh.cap + 64;  // see ln_bwd_span_kernel
    T* ring = reinterpret_cast<T*>(smem_raw) + U;
    if (t < sh.ring) bar_init(&full[t]);
    if (t < U) zeros[t] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    cluster_sync();
    if constexpr (MODE == SHIFTED) {
        for (int k = 0; k < sh.ring && t < 32; ++k) {
            T* buf = ring + k * slot_elems + sh.cap;
            const int e = t < 2 * U ? t - U : max(U, to - from - U) + t - 2 * U;
            if (e < sh.cap - U) buf[e] = 0;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    Pair<T> wv[NV][H], aw[NV][H], ab[NV][H];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int c = col.first(j) + 2 * i;
            const bool a = c >= from && c < to, b = c + 1 >= from && c + 1 < to;
            wv[j][i] = pair(a ? (w ? w[c] : T(1)) : T(0), b ? (w ? w[c + 1] : T(1)) : T(0));
            aw[j][i] = ab[j][i] = pair(T(0), T(0));
        }
    // One warp asks for the whole units, another copies what is small: their instructions lie between two rows.
    auto row_x = [&](int row) { return x + row * sh.pitch_x + from; };
    auto row_g = [&](int row) { return dy + row * sh.pitch_g + from; };
    auto small_of = [&](int row) { return small_copy<T, MODE>(row_x(row), row_g(row), to - from, sh.cap, 2 * sh.cap - U, mean + row, rstd + row, t & 31); };
    const SmallCopy<T> small = small_of(slab);
    const int64_t small_pitch = (t & 31) < 8 ? sh.pitch_x : (t & 31) < 16 ? sh.pitch_g : 1;
    auto fetch = [&](int row, int slot) {
        if (t >= 64) return;
        if (row < sh.spans) {
            T* base = ring + slot * slot_elems;
            if (t == 0) {
                const T *px = row_x(row), *pg = row_g(row);
                const Split<T> sx(px, to - from), sg(pg, to - from);
                bar_expect(&full[slot], static_cast<uint32_t>((sx.mid + sg.mid) * sizeof(T)));
                fetch_units(base, px, sx, &full[slot]);
                fetch_units(base + sh.cap, pg, sg, &full[slot]);
            } else if (t >= 32) {
                SmallCopy<T> c = small;
                if constexpr (MODE == MIXED) c = small_of(row);
                else c.from += (row - slab) * small_pitch;
                if (c.on) copy_one(base + c.to, c.from);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // xhat and dy of unit j of a row in a slot
    auto load = [&](int row, int slot, int j, T mu, const Pair<T>& minus_mu, const Pair<T>& rs2, Pair<T>(&xh)[H], Pair<T>(&up)[H]) {
        const T* base = ring + slot * slot_elems + col.u0 * U - col.mis - from + (j * TPR + t) * U;
        int mx = 0, mg = 0;
        if (MODE != ALIGNED) {
            mx = misalignment(x + row * sh.pitch_x + from);
            mg = misalignment(dy + row * sh.pitch_g + from);
        }
        // behind the columns: the row's mean and no gradient (see ln_bwd_span_kernel)
        load_unit<T, MODE != MIXED>(col.some(j) ? base + mx : ring + slot * slot_elems + 2 * sh.cap - U, xh);
        load_unit<T, MODE != MIXED>(col.some(j) ? base + sh.cap + mg : zeros, up);
        if (MODE == MIXED && !whole) {
            replace_outside(col.first(j), to, mu, xh);
            replace_outside(col.first(j), to, T(0), up);
        }
#pragma unroll
        for (int i = 0; i < H; ++i) xh[i] = (xh[i] + minus_mu) * rs2;
    };
    for (int k = 0; k < sh.ring; ++k) fetch(slab + k * slabs, k);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    unsigned int turn = 0;
    uint32_t limit = POLLS, phase = 0;
    int slot = 0, before = -1;  // before: the slot of the row whose second pass is due
    for (int row = slab;; row += slabs) {
        const bool more = row < sh.spans;
        T s[2] = {0, 0};
        if (more) {
            bar_wait(&full[slot], phase, limit, sh.gave_up);
            const T mu = ring[slot * slot_elems + 2 * sh.cap - U], rs = ring[slot * slot_elems + 2 * sh.cap - U + 32];
            const Pair<T> minus_mu = pair(-mu, -mu), rs2 = pair(rs, rs);
            Pair<T> s0 = pair(T(0), T(0)), s1 = s0;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                Pair<T> xh[H], up[H];
                load(row, slot, j, mu, minus_mu, rs2, xh, up);
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const Pair<T> gv = up[i] * wv[j][i];
                    aw[j][i] = muladd(up[i], xh[i], aw[j][i]);
                    ab[j][i] = ab[j][i] + up[i];
                    s0 = s0 + gv;
                    s1 = muladd(gv, xh[i], s1);
                }
            }
            T lo, hi;
            unpair(s0, lo, hi);
            s[0] = lo + hi;
            unpair(s1, lo, hi);
            s[1] = lo + hi;
            if (dx) row_sum<T, TPR, 1, 2>(s, part, 1, turn);
        }
        if (dx) {
            T total[2] = {0, 0};
            if (before >= 0) {  // the sums of the row before have arrived: written before the barrier that every thread waits for
                asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
                for (int q = 0; q < CL; ++q) {
                    total[0] += peers[(turn - (more ? 1 : 0)) & 1][q][0];
                    total[1] += peers[(turn - (more ? 1 : 0)) & 1][q][1];
                }
            }
            if (more) {
                if (t < CL) {
                    uint32_t remote;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(peers[turn & 1][rank])), "r"(t));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if constexpr (sizeof(T) == 4) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote + 4 * k), "f"(s[k]) : "memory");
                        else asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote + 8 * k), "d"(s[k]) : "memory");
                    }
                }
                __syncwarp();
                asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            }
            if (before >= 0) {
                const int old = row - slabs;
                const T mu = ring[before * slot_elems + 2 * sh.cap - U], rs = ring[before * slot_elems + 2 * sh.cap - U + 32];
                const Pair<T> minus_mu = pair(-mu, -mu), rs2 = pair(rs, rs);
                const T k0 = -rs * (total[0] * inv_cols), k1 = -rs * (total[1] * inv_cols);
                const Pair<T> k0p = pair(k0, k0), k1p = pair(k1, k1);
                T* dr = dx + static_cast<int64_t>(old) * sh.cols;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    Pair<T> xh[H], up[H], o[H];
                    load(old, before, j, mu, minus_mu, rs2, xh, up);
#pragma unroll
                    for (int i = 0; i < H; ++i) o[i] = muladd(up[i] * wv[j][i], rs2, muladd(xh[i], k1p, k0p));
                    if (whole || col.whole(j)) store_unit(dr + col.first(j), o);
                    else if (MODE != ALIGNED && col.some(j)) store_part(dr, col.first(j), to, o);
                }
            }
        }
        if (!more) break;
        asm volatile("cp.async.wait_group 0;" ::: "memory");  // the next row's small copies, one turn old
        __syncthreads();                                      // ... known to all, and the slot behind is read
        const int done = dx ? before : slot;
        if (done >= 0) fetch(dx ? row + (sh.ring - 1) * slabs : row + sh.ring * slabs, done);
        before = slot;
        slot = slot == sh.ring - 1 ? 0 : slot + 1;
        phase ^= slot == 0;
    }
    if (!parts) return;
    T* to_w = slabs == 1 ? dw : parts + static_cast<int64_t>(slab) * sh.cols;
    T* to_b = slabs == 1 ? db : parts + static_cast<int64_t>(slabs + slab) * sh.cols;
    const bool units = MODE == ALIGNED && ((reinterpret_cast<uintptr_t>(to_w) | reinterpret_cast<uintptr_t>(to_b)) & 15) == 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (units && col.whole(j)) {
            if (to_w) store_unit(to_w + col.first(j), aw[j]);
            if (to_b) store_unit(to_b + col.first(j), ab[j]);
        } else {
            if (to_w) store_part(to_w, col.first(j), to, aw[j]);
            if (to_b) store_part(to_b, col.first(j), to, ab[j]);
        }
    }
}

// Forward of wide rows, through the ring: a block's 512 threads, or those of a cluster, hold the row in registers from its one
// read to its store, with the weight and the bias of their columns beside it, while the next rows arrive.  With 1024 threads
// that load it into registers themselves a row fills the processor, and nothing is under way while it is summed:
// [4096, 12000] 98 us against 69 us, [4096, 16384] 115 against 98 us.
template <class T, int NV, int CL, int MODE>
__global__ void __launch_bounds__(SPAN_THREADS, 1) ln_fwd_span_kernel(const T* __restrict__ x, const SpanShape sh, const T* __restrict__ w,
                                                                     const T* __restrict__ bias, T eps, T inv_cols, T* __restrict__ y,
                                                                     T* __restrict__ mean_out, T* __restrict__ rstd_out) {
    constexpr int TPR = SPAN_THREADS, U = UNIT<T>, H = U / 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ T part[2 * TPR / 32];
    __shared__ T peers[CL > 1 ? 2 : 1][CL][2];
    __shared__ uint64_t full[MOST_RING];
    wb_pdl_enter();
    const int t = threadIdx.x;
    const int rank = CL > 1 ? static_cast<int>(blockIdx.x) % CL : 0;
    const int first = static_cast<int>(blockIdx.x) / CL, groups = static_cast<int>(gridDim.x) / CL;
    Columns<T, TPR, NV> col;
    col.t = t;
    col.u0 = rank * sh.units;
    col.mis = misalignment(y + first * sh.pitch_ref);
    const int from = CL > 1 ? max(0, col.u0 * U - col.mis) : 0;  // this CTA's columns [from, to)
    const int to = CL > 1 ? min(sh.cols, (col.u0 + sh.units) * U - col.mis) : sh.cols;
    col.cols = to;
    const bool whole = col.all_whole();
    T* ring = reinterpret_cast<T*>(smem_raw) + U;  // each slot begins with a unit of room
    if (t < sh.ring) bar_init(&full[t]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    if constexpr (CL > 1) cluster_sync();

    Pair<T> wv[NV][H], bv[NV][H];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int c = col.first(j) + 2 * i;
            const bool a = c >= from && c < to, b = c + 1 >= from && c + 1 < to;
            wv[j][i] = pair(a && w ? w[c] : T(1), b && w ? w[c + 1] : T(1));
            bv[j][i] = pair(a && bias ? bias[c] : T(0), b && bias ? bias[c + 1] : T(0));
        }

    auto fetch = [&](int row, int slot) {
        if (t >= 32) return;
        if (row < sh.spans) {
            const T* px = x + static_cast<int64_t>(row) * sh.pitch_x + from;
            T* base = ring + slot * sh.cap;
            if (t == 0) {
                const Split<T> s(px, to - from);
                bar_expect(&full[slot], static_cast<uint32_t>(s.mid * sizeof(T)));
                fetch_units(base, px, s, &full[slot]);
            }
            if (MODE != ALIGNED && t < 8) fetch_ends(base, px, to - from, t);
        }
        if (MODE != ALIGNED) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // See ln_bwd_span_kernel.
    auto settle = [&](int pending) {
        if (MODE == ALIGNED) return;
        if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
        else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else asm volatile("cp.async.wait_group 3;" ::: "memory");
    };
    for (int k = 0; k < sh.ring; ++k) fetch(first + k * groups, k);
    settle(sh.ring - 1);
    __syncthreads();

    unsigned int turn = 0;
    uint32_t limit = POLLS, phase = 0;
    int slot = 0;
    for (int row = first; row < sh.spans; row += groups) {
        bar_wait(&full[slot], phase, limit, sh.gave_up);
        const T* bx = ring + slot * sh.cap + col.u0 * U - col.mis - from + t * U;
        if (MODE != ALIGNED) bx += misalignment(x + static_cast<int64_t>(row) * sh.pitch_x + from);
        Pair<T> d[NV][H], s2 = pair(T(0), T(0));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            load_unit<T, MODE != MIXED>(bx + (col.some(j) ? j * TPR * U : -t * U), d[j]);
            if (!whole) replace_outside(col.first(j), to, T(0), d[j]);
#pragma unroll
            for (int i = 0; i < H; ++i) s2 = s2 + d[j][i];
        }
        T s[1], lo, hi;
        unpair(s2, lo, hi);
        s[0] = lo + hi;
        settle(sh.ring - 2);
        row_sum<T, TPR, 1, 1>(s, part, 1, turn, [&]() { fetch(row + sh.ring * groups, slot); });
        if constexpr (CL > 1) cluster_sum<T, CL, 1>(s, peers, rank, turn);
        const T mu = divide(s[0], static_cast<T>(sh.cols), inv_cols);
        const Pair<T> minus_mu = pair(-mu, -mu);
        s2 = pair(T(0), T(0));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < H; ++i) d[j][i] = d[j][i] + minus_mu;
            if (!whole) replace_outside(col.first(j), to, T(0), d[j]);
#pragma unroll
            for (int i = 0; i < H; ++i) s2 = muladd(d[j][i], d[j][i], s2);
        }
        unpair(s2, lo, hi);
        s[0] = lo + hi;
        row_sum<T, TPR, 1, 1>(s, part, 1, turn);
        if constexpr (CL > 1) cluster_sum<T, CL, 1>(s, peers, rank, turn);
        const T rs = T(1) / sqrt(s[0] * inv_cols + eps);
        const Pair<T> rs2 = pair(rs, rs);
        T* yr = y + static_cast<int64_t>(row) * sh.cols;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Pair<T> o[H];
#pragma unroll
            for (int i = 0; i < H; ++i) o[i] = muladd(d[j][i] * rs2, wv[j][i], bv[j][i]);
            if (whole || col.whole(j)) store_unit(yr + col.first(j), o);
            else if (MODE != ALIGNED && col.some(j)) store_part(yr, col.first(j), to, o);
        }
        if (t == 0 && rank == 0) {
            if (mean_out) mean_out[row] = mu;
            if (rstd_out) rstd_out[row] = rs;
        }
        slot = slot == sh.ring - 1 ? 0 : slot + 1;
        phase ^= slot == 0;
    }
}

// dw and db of 32 columns over one slab of rows: partials [2][slabs][cols].
template <class T>
__global__ void __launch_bounds__(THREADS) ln_dw_any_kernel(const T* __restrict__ x, RowView vx, const T* __restrict__ dy, RowView vg, int64_t rows,
                                                            int64_t cols, const T* __restrict__ mean, const T* __restrict__ rstd,
                                                            T* __restrict__ parts, int slabs) {
    __shared__ double sw[THREADS / 32][33], sb[THREADS / 32][33];
    wb_pdl_enter();
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    const int64_t first = rows * blockIdx.y / slabs, last = rows * (blockIdx.y + 1) / slabs;
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32; c0 < cols; c0 += static_cast<int64_t>(gridDim.x) * 32) {
        const int64_t c = c0 + lane;
        double aw = 0.0, ab = 0.0;
        if (c < cols) {
            const int64_t ox = col_offset(vx, c), og = col_offset(vg, c);
            for (int64_t row = first + line; row < last; row += THREADS / 32) {
                const double g = dy[row_offset(vg, row) + og];
                aw += g * ((static_cast<double>(x[row_offset(vx, row) + ox]) - mean[row]) * rstd[row]);
                ab += g;
            }
        }
        sw[line][lane] = aw;
        sb[line][lane] = ab;
        __syncthreads();
        if (line == 0 && c < cols) {
            for (int k = 1; k < THREADS / 32; ++k) {
                aw += sw[k][lane];
                ab += sb[k][lane];
            }
            parts[static_cast<int64_t>(blockIdx.y) * cols + c] = static_cast<T>(aw);
            parts[static_cast<int64_t>(slabs + blockIdx.y) * cols + c] = static_cast<T>(ab);
        }
        __syncthreads();
    }
}

// Sums the slabs of both partial arrays: 32 columns per block, LINES lines of threads that take every LINES-th slab, joined in
// order.  A line's loads are all in flight at once (ten: 32 lines reach 320 slabs, eight 80, four 40); 296 slabs by eight lines,
// their loads in turn, took 10 us whatever the size, 148 by eight lines of 20 loads 7.8 us against 4.9 us by 32 (the f64 additions
// are a chain), and 8 slabs of 16384 columns by 32 lines 10 us.
template <class T, int LINES>
__global__ void __launch_bounds__(32 * LINES) ln_dw_join_kernel(const T* __restrict__ parts, int slabs, int64_t cols, T* __restrict__ dw,
                                                                T* __restrict__ db) {
    __shared__ double sum[LINES][33];
    wb_pdl_enter();
    T* out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    double acc = 0.0;
    if (c < cols) {
        const T* p = parts + static_cast<int64_t>(blockIdx.y) * slabs * cols + c;
        constexpr int BATCH = 10;
        for (int k0 = line; k0 < slabs; k0 += LINES * BATCH) {
            T v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int k = k0 + j * LINES;
                v[j] = k < slabs ? p[static_cast<int64_t>(k) * cols] : T(0);
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j) acc += v[j];
        }
    }
    sum[line][lane] = acc;
    __syncthreads();
    if constexpr (LINES == 32) {  // transposed: a warp joins one column
        acc = sum[lane][line];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
        const int64_t to = static_cast<int64_t>(blockIdx.x) * 32 + line;
        if (lane == 0 && to < cols) out[to] = static_cast<T>(acc);
    } else if (line == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < LINES; ++k) acc += sum[k][lane];
        out[c] = static_cast<T>(acc);
    }
}

// ---- host ------------------------------------------------------------------------------------------------

struct Shape {
    int64_t rows = 1, cols = 1;
};

int view_shape(const char* who, const WbView* x, int normalized_dims, Shape* s) {
    WB_REQUIRE(x->dtype == WB_F32 || x->dtype == WB_F64, WB_ERR_UNSUPPORTED, "%s: dtype %d is not a float", who, x->dtype);
    WB_REQUIRE(x->ndim >= 1 && x->ndim <= WB_MAX_DIMS, WB_ERR_INVALID, "%s: a view has 1 to %d dims, got %d", who, WB_MAX_DIMS, x->ndim);
    WB_REQUIRE(normalized_dims >= 1 && normalized_dims <= x->ndim, WB_ERR_INVALID, "%s: can't normalise the last %d of %d dims", who, normalized_dims,
               x->ndim);
    bool empty = false;
    for (int d = 0; d < x->ndim; ++d) {
        WB_REQUIRE(x->shape[d] >= 0, WB_ERR_INVALID, "%s: dim %d has size %lld", who, d, static_cast<long long>(x->shape[d]));
        empty |= x->shape[d] == 0;
    }
    for (int d = 0; d < x->ndim; ++d) {
        int64_t& n = d < x->ndim - normalized_dims ? s->rows : s->cols;
        if (d >= x->ndim - normalized_dims) {
            WB_REQUIRE(x->shape[d] > 0, WB_ERR_INVALID, "%s: the normalised dims hold no element", who);
            WB_REQUIRE(n <= INT32_MAX / x->shape[d], WB_ERR_INVALID, "%s: more than 2^31 - 1 normalised elements", who);
        } else if (empty) {
            n = 0;
            continue;
        } else {
            WB_REQUIRE(n <= (int64_t(1) << 56) / x->shape[d], WB_ERR_INVALID, "%s: shape too large", who);
        }
        n *= x->shape[d];
    }
    WB_REQUIRE(s->rows <= (int64_t(1) << 56) / s->cols, WB_ERR_INVALID, "%s: shape too large", who);
    return WB_OK;
}

RowView row_view(const WbView& v, int normalized_dims) {
    RowView r{};
    for (int part = 0; part < 2; ++part) {
        WbView sub{};
        const int from = part == 0 ? 0 : v.ndim - normalized_dims, to = part == 0 ? v.ndim - normalized_dims : v.ndim;
        sub.ndim = to - from;
        for (int d = from; d < to; ++d) {
            sub.shape[d - from] = v.shape[d];
            sub.stride[d - from] = v.stride[d];
        }
        const WbView* one[1] = {&sub};
        WbIterPlan plan;
        wb_make_plan(one, 1, &plan);
        (part == 0 ? r.nd_row : r.nd_col) = plan.nd;
        for (int d = 0; d < WB_MAX_DIMS; ++d) {
            (part == 0 ? r.size_row : r.size_col)[d] = plan.size[d];
            (part == 0 ? r.st_row : r.st_col)[d] = plan.st[0][d];
        }
    }
    return r;
}

const char* view_data(const WbView& v) { return static_cast<const char*>(v.data) + v.offset * static_cast<int64_t>(wb_dtype_size(v.dtype)); }

// The bytes a view reaches (its strides may be negative).
WbSpan view_span(const WbView& v) {
    const int64_t size = static_cast<int64_t>(wb_dtype_size(v.dtype));
    int64_t lo = 0, hi = 0;
    for (int d = 0; d < v.ndim; ++d) {
        if (v.shape[d] == 0) return {view_data(v), view_data(v), false};
        (v.stride[d] < 0 ? lo : hi) += (v.shape[d] - 1) * v.stride[d];
    }
    return {view_data(v) + lo * size, view_data(v) + (hi + 1) * size, false};
}

struct SpanList {
    WbSpan s[8];
    int n = 0;
    int64_t size;
    bool aligned = true;
    explicit SpanList(int dtype) : size(static_cast<int64_t>(wb_dtype_size(dtype))) {}
    void add(const void* p, int64_t len, bool written) {
        if (!p || len == 0) return;
        aligned &= reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(size) == 0;
        const char* c = static_cast<const char*>(p);
        s[n++] = {c, c + len * size, written};
    }
    void add(const WbView& v) {
        aligned &= reinterpret_cast<uintptr_t>(view_data(v)) % static_cast<uintptr_t>(size) == 0;
        s[n++] = view_span(v);
    }
};

// Rows are summed in at most this many slabs for the weight's gradient (a multiple of four groups of them, see
// launch_spans).
int dw_slabs(int sm_count, int64_t rows) { return static_cast<int>(std::max<int64_t>(4, std::min<int64_t>((rows + 3) / 4 * 4, 2 * sm_count))); }

// Unit stride along the row and one stride, *pitch, from row to row (0 where there is one row).
bool plain_rows(const WbView& v, int normalized_dims, int64_t* pitch) {
    int64_t run = 1;
    int d = v.ndim - 1;
    for (; d >= v.ndim - normalized_dims; --d) {
        if (v.shape[d] == 1) continue;
        if (v.stride[d] != run) return false;
        run *= v.shape[d];
    }
    *pitch = 0;
    bool one = true;
    for (; d >= 0; --d) {
        if (v.shape[d] == 1) continue;
        if (one) *pitch = run = v.stride[d];
        else if (v.stride[d] != run) return false;
        one = false;
        run *= v.shape[d];
    }
    return true;
}

// 16-byte accesses: every row of every operand starts on a 16-byte boundary.
template <class T>
constexpr int wide = 16 / static_cast<int>(sizeof(T));
template <class T>
bool rows_aligned(const void* p, int64_t pitch, int64_t cols) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % wide<T> == 0 && cols % wide<T> == 0;
}

// Calls f with (threads per row, vectors per thread) for rows of `packs` vectors, at most MOST vectors per thread and at most
// THREADS_MOST threads: the fewest threads that hold the row, so that small rows share a block and the reductions stay short.
template <int MOST, int LEAST, int THREADS_MOST, class F>
bool choose_row(int64_t packs, F&& f) {
    auto per = [&](auto tpr) -> bool {
        constexpr int TPR = decltype(tpr)::value;
        if constexpr (TPR < LEAST || TPR > THREADS_MOST) {
            return false;
        } else {
            if (packs > static_cast<int64_t>(TPR) * MOST) return false;
            const int64_t nv = (packs + TPR - 1) / TPR;
            if constexpr (TPR == LEAST) {
                if (nv <= 1) return f(tpr, std::integral_constant<int, 1>{}), true;
                if (nv <= 2) return f(tpr, std::integral_constant<int, 2>{}), true;
                if constexpr (MOST / 4 > 2)
                    if (nv <= MOST / 4) return f(tpr, std::integral_constant<int, MOST / 4>{}), true;
                if constexpr (MOST / 2 > 2)
                    if (nv <= MOST / 2) return f(tpr, std::integral_constant<int, MOST / 2>{}), true;
            }
            if constexpr (MOST >= 4)
                if (nv <= MOST * 3 / 4) return f(tpr, std::integral_constant<int, MOST * 3 / 4>{}), true;
            return f(tpr, std::integral_constant<int, MOST>{}), true;
        }
    };
    return per(std::integral_constant<int, 8>{}) || per(std::integral_constant<int, 16>{}) || per(std::integral_constant<int, 32>{}) ||
           per(std::integral_constant<int, 64>{}) || per(std::integral_constant<int, 128>{}) || per(std::integral_constant<int, 256>{}) ||
           per(std::integral_constant<int, 512>{}) || per(std::integral_constant<int, 1024>{});
}

template <class T>
constexpr int row_elems = 64 / static_cast<int>(sizeof(T));  // elements of a row that a thread holds at most

// MOST elements per thread.  Aligned rows that 512 threads do not hold go to fwd_spans.
template <class T, int VEC, int MOST>
bool fwd_rows(WbBackend* b, const T* x, int64_t pitch, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd, cudaError_t* err) {
    return choose_row<MOST / VEC, 8, VEC == 1 ? 1024 : 512>((s.cols + VEC - 1) / VEC, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, G = fwd_threads<TPR> / TPR;
        const int64_t grid = (s.rows + G - 1) / G;
        *err = wb_launch_pdl(ln_fwd_rows_kernel<T, VEC, TPR, NV>, dim3(static_cast<unsigned>(grid)), dim3(fwd_threads<TPR>), 0, b->stream, x, pitch,
                             s.rows, static_cast<int>(s.cols), w, bias, static_cast<T>(eps), static_cast<T>(1.0 / static_cast<double>(s.cols)), y, mean,
                             rstd);
    });
}

// Rows repeat their misalignment after this many (1, 2 or 4): UNIT / gcd(UNIT, pitch).
template <class T>
int period(int64_t pitch) {
    int p = UNIT<T>;
    while (p > 1 && pitch % 2 == 0) {
        p /= 2;
        pitch /= 2;
    }
    return p;
}
template <class T>
bool same_misalignment(const T* a, int64_t pitch_a, const T* b, int64_t pitch_b, int64_t rows) {
    return (reinterpret_cast<uintptr_t>(a) - reinterpret_cast<uintptr_t>(b)) % 16 == 0 && (rows == 1 || (pitch_a - pitch_b) % UNIT<T> == 0);
}

cudaLaunchAttribute cluster_attribute(unsigned n) {
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = n;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    return a;
}

// Lets a kernel take the shared memory that its launches ask for, once per device.
template <auto KERNEL>
cudaError_t allow_shared(int ordinal) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = ordinal < 64 ? uint64_t(1) << ordinal : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SHARED);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// The backend's flag, made by its first call that waits.  That call may be captured, and other threads may be capturing: the
// allocation needs no stream, so this thread leaves their modes aside for it.
int make_wait_flag(WbBackend* b) {
    std::lock_guard<std::mutex> lock(b->mu);
    if (!b->ln_gave_up) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        WB_CHECK_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable);
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
        WB_CHECK_CUDA(e);
        *static_cast<int*>(p) = 0;
        b->ln_gave_up = static_cast<int*>(p);
    }
    return WB_OK;
}

// The grid of a span kernel: as many groups as the device holds at a time or as there are spans, and a multiple of the
// period, so that a group's rows are all of one misalignment.  Where one block with at most `few` spans per group will do, or
// up to `joint` of them, they leave the sums themselves, the latter as a cluster, and *slabs is 1: that saves the launch that
// joins the partials, about what two more rows in turn take.  Then the launch, as the programmatic dependent of what is
// before it.
template <auto KERNEL, int CL, class... Args>
cudaError_t launch_spans(WbBackend* b, const SpanShape& sh, int groups, size_t smem, int period, int few, int joint, int* slabs, Args... args) {
    cudaError_t e = allow_shared<KERNEL>(b->ordinal);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(CL);
    cfg.blockDim = dim3(SPAN_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = b->stream;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    int64_t most = b->sm_count;
    if (CL > 1) {
        // Clusters that are resident at a time: not every processor group is a multiple of CL processors, and a cluster more than
        // fit runs as a second wave (backward, [2000, 30000] over clusters of 4: 254 us with 37 of them, 150 us with those that fit).
        int fit = 0;
        attr[n++] = cluster_attribute(CL);
        cfg.attrs = attr;
        cfg.numAttrs = n;
        e = cudaOccupancyMaxActiveClusters(&fit, reinterpret_cast<const void*>(KERNEL), &cfg);
        if (e != cudaSuccess) return e;
        most = std::min<int64_t>(std::max(fit, 1), most);
    }
    const int step = std::max(1, period / groups);
    int64_t want = std::min<int64_t>(most, (static_cast<int64_t>(sh.spans) + groups - 1) / groups);
    want = std::min((want + step - 1) / step * step, most / step * step);
    if (step == 1 && sh.spans <= few * groups) want = 1;
    else if (sh.spans <= few * joint * groups) want = std::min<int64_t>(want, joint / step * step);
    want = std::max<int64_t>(want, step);
    cfg.gridDim = dim3(static_cast<unsigned>(want * CL));
    *slabs = static_cast<int>(want);
    if (CL == 1 && want > 1 && want <= joint) {
        attr[n++] = cluster_attribute(static_cast<unsigned>(want));
        *slabs = 1;
    }
    if (wb_pdl_allowed()) {
        attr[n] = cudaLaunchAttribute{};
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, KERNEL, args...);
}

// Rows per span: 32 KB per operand and turn of the block, but no more rows than leave every group a span.
template <class T>
int rows_per_span(const WbBackend* b, const Shape& s, int groups, int subs) {
    const int64_t room = 32768 / static_cast<int64_t>(sizeof(T)) / groups / s.cols, all = static_cast<int64_t>(b->sm_count) * groups, share = (s.rows + all - 1) / all;
    const int64_t r = std::min<int64_t>(std::min<int64_t>(room, share), 32);
    return static_cast<int>(std::max<int64_t>((r + subs - 1) / subs * subs, 1));
}

// Slots of the ring, `slots` bytes each for the whole block.  About 128 KB under way on a processor saturate the memory; with
// more of them some processors' copies wait for others', and since rows are dealt out beforehand the last one decides
// ([16384, 4096]: 123 us with 2 slots of 64 KB, 149 us with 3).  A cluster's exchange takes longer than that covers.
int ring_depth(size_t slots, int cl) {
    const int fit = static_cast<int>(MOST_SHARED / slots);
    return std::max(2, std::min({fit, MOST_RING, cl > 1 ? 3 : static_cast<int>(((128 << 10) + slots / 2) / slots)}));
}

// Threads per row and units per thread for rows of up to `units` units: the fewest threads that hold the row.
// Rows that share a warp have to lie end to end and uncut (`shared`).
template <class F>
bool choose_span(int64_t units, bool shared, F&& f) {
    constexpr int MOST = 4;
    auto per = [&](auto tpr) -> bool {
        constexpr int TPR = decltype(tpr)::value;
        if (units > TPR * MOST || (TPR < 32 && !shared)) return false;
        const int nv = static_cast<int>((units + TPR - 1) / TPR);
        using One = std::integral_constant<int, 1>;
        if constexpr (TPR == 8 || TPR == 32) {
            if (nv <= 1) return f(tpr, One{}), true;
            if (nv <= 2) return f(tpr, std::integral_constant<int, 2>{}), true;
        }
        if (nv <= 3) return f(tpr, std::integral_constant<int, 3>{}), true;
        return f(tpr, std::integral_constant<int, 4>{}), true;
    };
    return per(std::integral_constant<int, 8>{}) || per(std::integral_constant<int, 16>{}) || per(std::integral_constant<int, 32>{}) ||
           per(std::integral_constant<int, 64>{}) || per(std::integral_constant<int, 128>{}) || per(std::integral_constant<int, 256>{}) ||
           per(std::integral_constant<int, 512>{});
}

template <class T>
bool bwd_spans(WbBackend* b, const T* x, int64_t pitch_x, const T* dy, int64_t pitch_g, const Shape& s, const T* w, const T* mean, const T* rstd, T* dx,
               T* parts, T* dw, T* db, int* slabs, cudaError_t* err) {
    const T* ref = dx ? dx : dy;
    const int64_t pitch_ref = s.rows == 1 ? 0 : dx ? s.cols : pitch_g;
    const bool same = same_misalignment<T>(x, pitch_x, ref, pitch_ref, s.rows) && same_misalignment<T>(dy, pitch_g, ref, pitch_ref, s.rows);
    const bool dense = pitch_x == s.cols && pitch_g == s.cols;
    const int per = period<T>(pitch_ref);
    const bool aligned = per == 1 && reinterpret_cast<uintptr_t>(ref) % 16 == 0;
    const int64_t units = (s.cols + UNIT<T> - 1 + (aligned ? 0 : UNIT<T> - 1)) / UNIT<T>;
    const bool cut = !aligned || s.cols % UNIT<T> != 0;
    SpanShape sh;
    sh.gave_up = b->ln_gave_up;
    sh.rows = s.rows;
    sh.cols = static_cast<int>(s.cols);
    sh.pitch_x = pitch_x;
    sh.pitch_g = pitch_g;
    sh.pitch_ref = pitch_ref;
    const T inv_cols = static_cast<T>(1.0 / static_cast<double>(s.cols));
    // a slot's buffer behind a unit of room: the misalignment, the run, what a last unit reads behind it
    auto buffer = [](int64_t run) { return static_cast<int>((run + UNIT<T> - 1) / UNIT<T> * UNIT<T> + 3 * UNIT<T>); };
    auto go = [&](auto tpr, auto nv, auto mode) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, MODE = decltype(mode)::value;
        constexpr int N = SPAN_THREADS, GT = TPR < 32 ? 32 : TPR, G = N / GT, SUBS = GT / TPR;
        sh.units = static_cast<int>(units);
        sh.r = GT == 32 && dense && (MODE == ALIGNED || MODE == ELEMENTS) ? rows_per_span<T>(b, s, G, SUBS) : 1;
        sh.spans = static_cast<int>((s.rows + sh.r - 1) / sh.r);
        sh.cap = buffer(sh.r * s.cols);
        const size_t slots = sizeof(T) * static_cast<size_t>(G) * (2 * sh.cap + 64), join = sizeof(T) * 2 * (N * NV * UNIT<T> + static_cast<size_t>(s.cols));
        sh.ring = ring_depth(slots, 1);
        *err = launch_spans<ln_bwd_span_kernel<T, TPR, NV, MODE>, 1>(b, sh, G, std::max(slots * sh.ring, join), MODE == ELEMENTS ? 1 : per, parts ? 3 : 0,
                                                                    parts ? 8 : 0, slabs, x, dy, sh, w, mean, rstd, inv_cols, ref, dx, parts, dw, db);
    };
    auto go_wide = [&](auto nv, auto cl, auto mode) {
        constexpr int NV = decltype(nv)::value, CL = decltype(cl)::value, MODE = decltype(mode)::value;
        sh.units = static_cast<int>((units + CL - 1) / CL);
        sh.r = 1;
        sh.spans = static_cast<int>(s.rows);
        sh.cap = buffer(static_cast<int64_t>(sh.units) * UNIT<T>);
        const size_t slots = sizeof(T) * (2 * sh.cap + 64);
        sh.ring = 3;
        *err = launch_spans<ln_bwd_wide_kernel<T, NV, CL, MODE>, CL>(b, sh, 1, slots * sh.ring, per, parts ? 2 : 0, 0, slabs, x, dy, sh, w, mean, rstd, inv_cols,
                                                                ref, dx, parts, dw, db);
        return true;
    };
    constexpr int SHORT = 16 * 4 * UNIT<T>;
    if ((cut || !same) && s.cols <= SHORT) {
        const int nv = static_cast<int>((s.cols + (s.cols <= 8 * 4 * UNIT<T> ? 8 : 16) * UNIT<T> - 1) / ((s.cols <= 8 * 4 * UNIT<T> ? 8 : 16) * UNIT<T>));
        using M = std::integral_constant<int, ELEMENTS>;
        using N1 = std::integral_constant<int, 1>;
        using N2 = std::integral_constant<int, 2>;
        using N3 = std::integral_constant<int, 3>;
        using N4 = std::integral_constant<int, 4>;
        using T8 = std::integral_constant<int, 8>;
        using T16 = std::integral_constant<int, 16>;
        if (s.cols <= 8 * 4 * UNIT<T>)
            nv == 1 ? go(T8{}, N1{}, M{}) : nv == 2 ? go(T8{}, N2{}, M{}) : nv == 3 ? go(T8{}, N3{}, M{}) : go(T8{}, N4{}, M{});
        else
            nv == 3 ? go(T16{}, N3{}, M{}) : go(T16{}, N4{}, M{});
        return true;
    }
    const bool done = choose_span(units, dense && !cut && same, [&](auto tpr, auto nv) {
        static_assert(SHORT >= 32 * 2 * UNIT<T>, "rows that two units of a warp hold go by elements where they are cut");
        if constexpr (decltype(tpr)::value > 32 || (decltype(tpr)::value == 32 && decltype(nv)::value > 2)) {
            if (!same) return go(tpr, nv, std::integral_constant<int, MIXED>{});
            if (cut) return go(tpr, nv, std::integral_constant<int, SHIFTED>{});
        }
        go(tpr, nv, std::integral_constant<int, ALIGNED>{});
    });
    if (done) return true;
    auto wide = [&](auto mode) {
        // the fewest units per thread that hold the row: [4000, 9001] 129 us with three, 152 us with four; [4096, 12000] 125
        // and 131 us
        auto over = [&](auto cl) {
            constexpr int CL = decltype(cl)::value;
            if (units <= CL * 3 * SPAN_THREADS) return go_wide(std::integral_constant<int, 3>{}, cl, mode);
            if (units <= CL * 4 * SPAN_THREADS) return go_wide(std::integral_constant<int, 4>{}, cl, mode);
            return false;
        };
        return over(std::integral_constant<int, 2>{}) || over(std::integral_constant<int, 4>{}) || over(std::integral_constant<int, 8>{});
    };
    if (!same) return wide(std::integral_constant<int, MIXED>{});
    return cut ? wide(std::integral_constant<int, SHIFTED>{}) : wide(std::integral_constant<int, ALIGNED>{});
}

template <class T>
bool fwd_spans(WbBackend* b, const T* x, int64_t pitch, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd, cudaError_t* err) {
    const int64_t pitch_ref = s.rows == 1 ? 0 : s.cols;
    const bool same = same_misalignment<T>(x, pitch, y, pitch_ref, s.rows);
    const int per = period<T>(pitch_ref);
    const bool aligned = per == 1 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
    const int64_t units = (s.cols + UNIT<T> - 1 + (aligned ? 0 : UNIT<T> - 1)) / UNIT<T>;
    auto go = [&](auto nv, auto cl, auto mode) {
        constexpr int NV = decltype(nv)::value, CL = decltype(cl)::value;
        SpanShape sh{};
        sh.gave_up = b->ln_gave_up;
        sh.rows = s.rows;
        sh.cols = static_cast<int>(s.cols);
        sh.pitch_x = pitch;
        sh.pitch_ref = pitch_ref;
        sh.units = static_cast<int>((units + CL - 1) / CL);
        sh.r = 1;
        sh.spans = static_cast<int>(s.rows);
        sh.cap = sh.units * UNIT<T> + 4 * UNIT<T>;
        const size_t slots = sizeof(T) * static_cast<size_t>(sh.cap);
        sh.ring = ring_depth(slots, CL);
        int slabs = 0;
        *err = launch_spans<ln_fwd_span_kernel<T, NV, CL, decltype(mode)::value>, CL>(b, sh, 1, slots * sh.ring, per, 0, 0, &slabs, x, sh, w, bias,
                                                                                     static_cast<T>(eps), static_cast<T>(1.0 / static_cast<double>(s.cols)),
                                                                                     y, mean, rstd);
        return true;
    };
    auto wide = [&](auto mode) {
        using A = std::integral_constant<int, 8>;
        if (units <= 2 * 4096) return go(A{}, std::integral_constant<int, 2>{}, mode);
        if (units <= 4 * 4096) return go(A{}, std::integral_constant<int, 4>{}, mode);
        if (units <= 8 * 4096) return go(A{}, std::integral_constant<int, 8>{}, mode);
        return false;
    };
    using One = std::integral_constant<int, 1>;
    if (same && aligned && s.cols % UNIT<T> == 0) {
        using M = std::integral_constant<int, ALIGNED>;
        if (units <= 512 * 6) return go(std::integral_constant<int, 6>{}, One{}, M{});
        if (units <= 512 * 8) return go(std::integral_constant<int, 8>{}, One{}, M{});
        return wide(M{});
    }
    // Rows that are not aligned: element by element up to 16384 columns (ln_fwd_rows_kernel: [4000, 9001] 70 us against 73 us
    // here); f64 behind that row by row from the second-level cache (ln_fwd_any_kernel: [4000, 10001] 244 us against 295 us).
    if constexpr (sizeof(T) == 4) {
        if (units > 4096) return same ? wide(std::integral_constant<int, SHIFTED>{}) : wide(std::integral_constant<int, MIXED>{});
    }
    return false;
}

template <class T>
int fwd_typed(WbBackend* b, const WbView* x, int nd, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    cudaError_t err = cudaSuccess;
    bool done = false;
    int64_t pitch;
    if (plain_rows(*x, nd, &pitch) && s.rows < (1 << 30)) {
        if (s.cols * static_cast<int64_t>(sizeof(T)) > 32768) done = fwd_spans<T>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
        if (done) {
        } else if (rows_aligned<T>(xp, pitch, s.cols) && rows_aligned<T>(y, s.cols, s.cols) &&
                   ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias)) & 15) == 0) {
            done = fwd_rows<T, wide<T>, row_elems<T>>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
        } else if (sizeof(T) == 4 && s.cols <= 1024) {
            // [30000, 1001]: 51 us with up to 16 elements per thread, 42 us with 8; [20000, 3333]: 92 us and 105 us
            done = fwd_rows<T, 1, row_elems<T> / 2>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
        } else {
            done = fwd_rows<T, 1, row_elems<T>>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
        }
    }
    if (!done) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
        err = wb_launch_pdl(ln_fwd_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, row_view(*x, nd), s.rows, s.cols, w, bias, eps, y, mean, rstd);
    }
    WB_CHECK_CUDA(err);
    WB_LAUNCH_OK(b);
    return WB_OK;
}

template <class T>
int bwd_typed(WbBackend* b, const WbView* x, const WbView* dy, int nd, const Shape& s, const T* w, const T* mean, const T* rstd, T* dx, T* dw, T* db,
              T* parts) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    const T* gp = reinterpret_cast<const T*>(view_data(*dy));
    const bool sums = dw || db;
    if (!dx && !sums) return WB_OK;
    cudaError_t err = cudaSuccess;
    bool done = false;
    int slabs = dw_slabs(b->sm_count, s.rows);
    int64_t pitch_x, pitch_g;
    if (plain_rows(*x, nd, &pitch_x) && plain_rows(*dy, nd, &pitch_g) && s.rows < (1 << 30)) {
        done = bwd_spans<T>(b, xp, pitch_x, gp, pitch_g, s, w, mean, rstd, dx, sums ? parts : nullptr, dw, db, &slabs, &err);
        if (done) {
            WB_CHECK_CUDA(err);
            WB_LAUNCH_OK(b);
        }
    }
    RowView vx, vg;
    if (!done) {
        vx = row_view(*x, nd);
        vg = row_view(*dy, nd);
    }
    if (!done && dx) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dx_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, w, mean, rstd, dx));
        WB_LAUNCH_OK(b);
    }
    if (!sums || (done && slabs == 1)) return WB_OK;
    if (!done) {
        const unsigned strips = static_cast<unsigned>(std::min<int64_t>((s.cols + 31) / 32, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dw_any_kernel<T>, dim3(strips, slabs), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, mean, rstd,
                                    parts, slabs));
        WB_LAUNCH_OK(b);
    }
    const dim3 strips(static_cast<unsigned>((s.cols + 31) / 32), 2);
    const T* joined = parts;
    if (slabs <= 40) WB_CHECK_CUDA(wb_launch_pdl(ln_dw_join_kernel<T, 4>, strips, dim3(32 * 4), 0, b->stream, joined, slabs, s.cols, dw, db));
    else if (slabs <= 80) WB_CHECK_CUDA(wb_launch_pdl(ln_dw_join_kernel<T, 8>, strips, dim3(32 * 8), 0, b->stream, joined, slabs, s.cols, dw, db));
    else WB_CHECK_CUDA(wb_launch_pdl(ln_dw_join_kernel<T, 32>, strips, dim3(32 * 32), 0, b->stream, joined, slabs, s.cols, dw, db));
    WB_LAUNCH_OK(b);
    return WB_OK;
}

int64_t bwd_workspace(int sm_count, int64_t rows, int64_t cols, int dtype) {
    if (rows == 0) return 0;
    return 2 * static_cast<int64_t>(dw_slabs(sm_count, rows)) * cols * static_cast<int64_t>(wb_dtype_size(dtype));
}

}  // namespace

// Reads and clears the flag of the backend's bounded waits; waits for the stream.  The exchange loses none that goes up meanwhile.
int wb_layer_norm_check(WbBackend* b) {
    if (!b->ln_gave_up) return WB_OK;  // no call of this backend has waited
    WB_CHECK_CUDA(cudaStreamSynchronize(b->stream));
    if (__atomic_exchange_n(b->ln_gave_up, 0, __ATOMIC_ACQ_REL) == 0) return WB_OK;
    wb_set_error("a layer norm gave up waiting for a bulk copy");
    return WB_ERR_TIMEOUT;
}

// One thread waits, the way the kernels above do, on a barrier that nothing arrives at (no copy is in flight), and gives up.
__global__ void ln_timeout_selftest_kernel(int* gave_up, uint32_t polls) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        bar_init(&bar);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        bar_wait(&bar, 0, polls, gave_up);
    }
}

extern "C" int wb_layer_norm_selftest_timeout(WbBackend* b, int polls) {
    WB_REQUIRE(b && polls > 0 && polls <= (1 << 20), WB_ERR_INVALID, "wb_layer_norm_selftest_timeout: polls must be 1..2^20");
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WB_TRY(make_wait_flag(b));
    ln_timeout_selftest_kernel<<<1, 32, 0, b->stream>>>(b->ln_gave_up, static_cast<uint32_t>(polls));
    WB_LAUNCH_OK(b);
    return WB_OK;
}

// ---- entry points ------------------------------------------------------------------------------------------

extern "C" int wb_layer_norm_fwd(WbBackend* b, const WbView* x, int normalized_dims, const void* weight, const void* bias, double eps, void* y,
                                 void* save_mean, void* save_rstd) {
    WB_REQUIRE(b && x && x->data && y, WB_ERR_INVALID, "wb_layer_norm_fwd: null pointer");
    WB_REQUIRE(eps >= 0.0, WB_ERR_INVALID, "wb_layer_norm_fwd: eps has to be at least 0, got %g", eps);
    Shape s;
    WB_TRY(view_shape("wb_layer_norm_fwd", x, normalized_dims, &s));
    if (s.rows == 0) return WB_OK;
    SpanList spans(x->dtype);
    spans.add(*x);
    spans.add(weight, s.cols, false);
    spans.add(bias, s.cols, false);
    spans.add(y, s.rows * s.cols, true);
    spans.add(save_mean, s.rows, true);
    spans.add(save_rstd, s.rows, true);
    WB_REQUIRE(spans.aligned, WB_ERR_INVALID, "wb_layer_norm_fwd: a pointer is not aligned to its element type");
    WB_REQUIRE(!wb_spans_clash(spans.s, spans.n), WB_ERR_INVALID, "wb_layer_norm_fwd: an output overlaps another operand");
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WB_TRY(make_wait_flag(b));
    WbProfileScope ps(b, "layer_norm");
    if (x->dtype == WB_F32)
        return fwd_typed<float>(b, x, normalized_dims, s, static_cast<const float*>(weight), static_cast<const float*>(bias), eps,
                                static_cast<float*>(y), static_cast<float*>(save_mean), static_cast<float*>(save_rstd));
    return fwd_typed<double>(b, x, normalized_dims, s, static_cast<const double*>(weight), static_cast<const double*>(bias), eps,
                             static_cast<double*>(y), static_cast<double*>(save_mean), static_cast<double*>(save_rstd));
}

extern "C" int64_t wb_layer_norm_bwd_workspace(const WbBackend* b, int64_t rows, int64_t cols, int dtype) {
    if (!b || rows < 0 || cols < 1 || cols > INT32_MAX || (dtype != WB_F32 && dtype != WB_F64)) return -1;
    return bwd_workspace(b->sm_count, rows, cols, dtype);
}

extern "C" int wb_layer_norm_bwd(WbBackend* b, const WbView* x, const WbView* dy, int normalized_dims, const void* weight, const void* save_mean,
                                 const void* save_rstd, void* dx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes) {
    WB_REQUIRE(b && x && x->data && dy && dy->data && save_mean && save_rstd, WB_ERR_INVALID, "wb_layer_norm_bwd: null pointer");
    WB_REQUIRE(x->dtype == dy->dtype, WB_ERR_INVALID, "wb_layer_norm_bwd: dtype mismatch %d and %d", x->dtype, dy->dtype);
    WB_REQUIRE(x->ndim == dy->ndim, WB_ERR_INVALID, "wb_layer_norm_bwd: x and dy must share one shape");
    Shape s;
    WB_TRY(view_shape("wb_layer_norm_bwd", x, normalized_dims, &s));
    for (int d = 0; d < x->ndim; ++d)
        WB_REQUIRE(x->shape[d] == dy->shape[d], WB_ERR_INVALID, "wb_layer_norm_bwd: x and dy must share one shape");
    const int64_t size = static_cast<int64_t>(wb_dtype_size(x->dtype));
    const bool sums = dweight || dbias;
    const int64_t need = sums ? bwd_workspace(b->sm_count, s.rows, s.cols, x->dtype) : 0;
    WB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), WB_ERR_INVALID, "wb_layer_norm_bwd: the workspace holds %lld bytes, %lld are needed",
               static_cast<long long>(workspace ? workspace_bytes : 0), static_cast<long long>(need));
    WB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0 || need == 0, WB_ERR_INVALID, "wb_layer_norm_bwd: the workspace is not aligned to 16 bytes");
    SpanList spans(x->dtype);
    spans.add(*x);
    spans.add(*dy);
    // reads: the statistics and the weight; the workspace's span replaces them in a second list (at most eight fit one)
    spans.add(dx, s.rows * s.cols, true);
    spans.add(dweight, s.cols, true);
    spans.add(dbias, s.cols, true);
    if (need) spans.add(workspace, need / size, true);
    SpanList others(x->dtype);
    others.add(weight, s.cols, false);
    others.add(save_mean, s.rows, false);
    others.add(save_rstd, s.rows, false);
    others.add(dx, s.rows * s.cols, true);
    others.add(dweight, s.cols, true);
    others.add(dbias, s.cols, true);
    if (need) others.add(workspace, need / size, true);
    WB_REQUIRE(spans.aligned && others.aligned, WB_ERR_INVALID, "wb_layer_norm_bwd: a pointer is not aligned to its element type");
    WB_REQUIRE(!wb_spans_clash(spans.s, spans.n) && !wb_spans_clash(others.s, others.n), WB_ERR_INVALID,
               "wb_layer_norm_bwd: an output overlaps another operand");
    WbDeviceGuard dev(b->ordinal);
    WB_CHECK_CUDA(dev.status);
    WB_TRY(make_wait_flag(b));
    WbProfileScope ps(b, "layer_norm_bwd");
    if (s.rows == 0) {  // the sums over no rows
        if (dweight) WB_CHECK_CUDA(cudaMemsetAsync(dweight, 0, static_cast<size_t>(s.cols * size), b->stream));
        if (dbias) WB_CHECK_CUDA(cudaMemsetAsync(dbias, 0, static_cast<size_t>(s.cols * size), b->stream));
        return WB_OK;
    }
    if (x->dtype == WB_F32)
        return bwd_typed<float>(b, x, dy, normalized_dims, s, static_cast<const float*>(weight), static_cast<const float*>(save_mean),
                                static_cast<const float*>(save_rstd), static_cast<float*>(dx), static_cast<float*>(dweight),
                                static_cast<float*>(dbias), static_cast<float*>(workspace));
    return bwd_typed<double>(b, x, dy, normalized_dims, s, static_cast<const double*>(weight), static_cast<const double*>(save_mean),
                             static_cast<const double*>(save_rstd), static_cast<double*>(dx), static_cast<double*>(dweight),
                             static_cast<double*>(dbias), static_cast<double*>(workspace));
}
