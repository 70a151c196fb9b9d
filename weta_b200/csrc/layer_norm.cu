// Layer normalisation over the last dims of a strided view, forward and backward
// (crates/weta-nn/src/functional.rs:183-195 and the gradients autograd derives through it):
//   mu = mean_c x,  rstd = 1 / sqrt(mean_c (x - mu)^2 + eps),  xhat = (x - mu) rstd,  y = xhat w + b
//   g = dy w,  dx = rstd (g - mean_c g - xhat mean_c (g xhat)),  dw = sum_r dy xhat,  db = sum_r dy
// The view is taken as [rows, cols]: cols is the product of the normalised dims.
#include <algorithm>
#include <cmath>

#include "common.h"

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
// group (`bar`, at least 1) and join the warps' sums, `part` (2 K warps), in a second tree; two buffers in turn make one
// barrier per sum enough.
template <class T, int TPR, int K>
__device__ __forceinline__ void row_sum(T (&v)[K], T* part, int bar, unsigned int& turn) {
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
        asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(TPR) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) {
            T s = mine[k * W + lane % W];
#pragma unroll
            for (int d = W / 2; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            v[k] = s;
        }
    }
}

template <int TPR>
constexpr int fwd_threads = TPR < 128 ? 128 : TPR;

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
    row_sum<T, TPR, 1>(s, part[group], 1 + group, turn);
    const T mean = s[0] * inv_cols;
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
    row_sum<T, TPR, 1>(q, part[group], 1 + group, turn);
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

// Backward.  A group of TPR threads walks rows id, id + groups, ...; the rows ahead are fetched by cp.async into a ring of
// DEPTH slots in shared memory.  A thread reads back only what it copied itself, so the ring needs no barrier.  The
// weight's and the bias's gradients of its columns stay in the thread's registers over all its rows; at the end the groups
// of a block are joined in shared memory and the block leaves one row of partials.
constexpr int BWD_THREADS = 256;

__device__ __forceinline__ void async_copy(void* smem, const void* gmem, std::integral_constant<int, 16>) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "l"(gmem) : "memory");
}
__device__ __forceinline__ void async_copy(void* smem, const void* gmem, std::integral_constant<int, 8>) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "l"(gmem) : "memory");
}
__device__ __forceinline__ void async_copy(void* smem, const void* gmem, std::integral_constant<int, 4>) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "l"(gmem) : "memory");
}

template <int TPR>
constexpr int bwd_threads = TPR < BWD_THREADS ? BWD_THREADS : TPR;

template <class T, int VEC, int TPR, int NV, int DEPTH>
__global__ void __launch_bounds__(bwd_threads<TPR>) ln_bwd_rows_kernel(const T* __restrict__ x, int64_t pitch_x, const T* __restrict__ dy, int64_t pitch_g,
                                                                       int64_t rows, int cols, const T* __restrict__ w, const T* __restrict__ mean,
                                                                       const T* __restrict__ rstd, T inv_cols, T* __restrict__ dx,
                                                                       T* __restrict__ parts) {
    constexpr int THREADS_B = bwd_threads<TPR>, G = THREADS_B / TPR, E = NV * VEC;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Pack<T, VEC>* ring = reinterpret_cast<Pack<T, VEC>*>(smem_raw);  // [DEPTH][2][NV][THREADS_B]
    __shared__ T part[G][TPR > 32 ? 4 * TPR / 32 : 1];
    wb_pdl_enter();
    const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * G, first = static_cast<int64_t>(blockIdx.x) * G + group;
    auto slot = [&](int stage, int which, int j) -> Pack<T, VEC>& { return ring[((stage * 2 + which) * NV + j) * THREADS_B + threadIdx.x]; };
    T wv[E], aw[E], ab[E];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = (j * TPR + t) * VEC + i;
            wv[j * VEC + i] = c < cols ? (w ? w[c] : T(1)) : T(0);
            aw[j * VEC + i] = ab[j * VEC + i] = 0;
            // columns behind the row's end: their slots are never copied to and stay 0
            for (int d = 0; d < DEPTH; ++d) slot(d, 0, j).v[i] = slot(d, 1, j).v[i] = 0;
        }
    auto fetch = [&](int64_t row, int stage) {
        if (row < rows) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * TPR + t) * VEC;
                if (c < cols) {
                    async_copy(&slot(stage, 0, j), x + row * pitch_x + c, std::integral_constant<int, sizeof(T) * VEC>{});
                    async_copy(&slot(stage, 1, j), dy + row * pitch_g + c, std::integral_constant<int, sizeof(T) * VEC>{});
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(first + d * groups, d);
    T mu = 0, rs = 0;
    if (first < rows) {
        mu = mean[first];
        rs = rstd[first];
    }
    unsigned int turn = 0;
    int stage = 0;
    // groups narrower than a warp share its shuffles: they all walk as far as the warp's first one
    const int64_t lead = TPR < 32 ? first - group % (32 / (TPR < 32 ? TPR : 32)) : first;
    for (int64_t row = first, at = lead; at < rows; row += groups, at += groups) {
        fetch(row + (DEPTH - 1) * groups, stage == 0 ? DEPTH - 1 : stage - 1);
        T mu_next = 0, rs_next = 0;
        if (row + groups < rows) {
            mu_next = mean[row + groups];
            rs_next = rstd[row + groups];
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        const bool live = TPR >= 32 || row < rows;
        T xh[E], g[E], s[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Pack<T, VEC> px = slot(stage, 0, j), pg = slot(stage, 1, j);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int e = j * VEC + i;
                const T up = live ? pg.v[i] : T(0);
                xh[e] = live ? (px.v[i] - mu) * rs : T(0);  // not live: the slot holds an older row
                aw[e] += up * xh[e];
                ab[e] += up;
                g[e] = up * wv[e];
                s[0] += g[e];
                s[1] += g[e] * xh[e];
            }
        }
        if (dx) {
            row_sum<T, TPR, 2>(s, part[group], 1 + group, turn);
            const T c0 = s[0] * inv_cols, c1 = s[1] * inv_cols;
            if (live) {
                T* dr = dx + row * cols;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = (j * TPR + t) * VEC;
                    Pack<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) o.v[i] = rs * (g[j * VEC + i] - c0 - xh[j * VEC + i] * c1);
                    if (c < cols) *reinterpret_cast<Pack<T, VEC>*>(dr + c) = o;
                }
            }
        }
        mu = mu_next;
        rs = rs_next;
        stage = stage + 1 == DEPTH ? 0 : stage + 1;
    }
    if (!parts) return;
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (G > 1) {  // the groups' sums, in the groups' order
        T* joined = reinterpret_cast<T*>(smem_raw);  // [2][G][TPR E]
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = (j * TPR + t) * VEC + i;
                joined[group * TPR * E + c] = aw[j * VEC + i];
                joined[(G + group) * TPR * E + c] = ab[j * VEC + i];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += THREADS_B) {
            T sw = joined[c], sb = joined[G * TPR * E + c];
            for (int k = 1; k < G; ++k) {
                sw += joined[k * TPR * E + c];
                sb += joined[(G + k) * TPR * E + c];
            }
            parts[static_cast<int64_t>(blockIdx.x) * cols + c] = sw;
            parts[static_cast<int64_t>(gridDim.x + blockIdx.x) * cols + c] = sb;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = (j * TPR + t) * VEC + i;
                if (c < cols) {
                    parts[static_cast<int64_t>(blockIdx.x) * cols + c] = aw[j * VEC + i];
                    parts[static_cast<int64_t>(gridDim.x + blockIdx.x) * cols + c] = ab[j * VEC + i];
                }
            }
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

// Sums the slabs of both partial arrays: 32 columns per block, eight runs of slabs side by side, joined in order.
template <class T>
__global__ void __launch_bounds__(THREADS) ln_dw_join_kernel(const T* __restrict__ parts, int slabs, int64_t cols, T* __restrict__ dw,
                                                             T* __restrict__ db) {
    __shared__ double sum[THREADS / 32][32];
    wb_pdl_enter();
    T* out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    const T* p = parts + static_cast<int64_t>(blockIdx.y) * slabs * cols;
    double acc = 0.0;
    if (c < cols) {
#pragma unroll 8
        for (int k = line; k < slabs; k += THREADS / 32) acc += p[static_cast<int64_t>(k) * cols + c];
    }
    sum[line][lane] = acc;
    __syncthreads();
    if (line == 0 && c < cols) {
        for (int k = 1; k < THREADS / 32; ++k) acc += sum[k][lane];
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

// Rows are summed in at most this many slabs for the weight's gradient.
int dw_slabs(int sm_count, int64_t rows) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, 2 * sm_count))); }

// Unit stride along the row and one stride from row to row.
bool plain_rows(const RowView& v, const Shape& s) { return v.nd_row == 1 && v.nd_col == 1 && (v.st_col[0] == 1 || s.cols == 1); }

// 16-byte accesses: every row of every operand starts on a 16-byte boundary.
template <class T>
constexpr int wide = 16 / static_cast<int>(sizeof(T));
template <class T>
bool rows_aligned(const void* p, int64_t pitch, int64_t cols) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % wide<T> == 0 && cols % wide<T> == 0;
}

// Calls f with (threads per row, vectors per thread) for rows of `packs` vectors, at most MOST vectors per thread: the
// fewest threads that hold the row, so that small rows share a block and the reductions stay short.
template <int MOST, class F>
bool choose_row(int64_t packs, F&& f) {
    auto per = [&](auto tpr) -> bool {
        constexpr int TPR = decltype(tpr)::value;
        if (packs > static_cast<int64_t>(TPR) * MOST) return false;
        const int64_t nv = (packs + TPR - 1) / TPR;
        if constexpr (TPR == 8) {
            if (nv <= 1) return f(tpr, std::integral_constant<int, 1>{}), true;
            if (nv <= 2) return f(tpr, std::integral_constant<int, 2>{}), true;
        }
        if constexpr (TPR == 8 && MOST > 4)
            if (nv <= MOST / 4) return f(tpr, std::integral_constant<int, MOST / 4>{}), true;
        if constexpr (TPR == 8)
            if (nv <= MOST / 2) return f(tpr, std::integral_constant<int, MOST / 2>{}), true;
        if (nv <= MOST * 3 / 4) return f(tpr, std::integral_constant<int, MOST * 3 / 4>{}), true;
        return f(tpr, std::integral_constant<int, MOST>{}), true;
    };
    return per(std::integral_constant<int, 8>{}) || per(std::integral_constant<int, 16>{}) || per(std::integral_constant<int, 32>{}) ||
           per(std::integral_constant<int, 64>{}) || per(std::integral_constant<int, 128>{}) || per(std::integral_constant<int, 256>{}) ||
           per(std::integral_constant<int, 512>{}) || per(std::integral_constant<int, 1024>{});
}

template <class T>
constexpr int row_elems = 64 / static_cast<int>(sizeof(T));  // elements of a row that a thread holds at most

template <class T, int VEC>
bool fwd_rows(WbBackend* b, const T* x, int64_t pitch, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd, cudaError_t* err) {
    return choose_row<row_elems<T> / VEC>((s.cols + VEC - 1) / VEC, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, G = fwd_threads<TPR> / TPR;
        const int64_t grid = (s.rows + G - 1) / G;
        if (grid > INT32_MAX) {
            *err = cudaErrorInvalidConfiguration;
            return;
        }
        *err = wb_launch_pdl(ln_fwd_rows_kernel<T, VEC, TPR, NV>, dim3(static_cast<unsigned>(grid)), dim3(fwd_threads<TPR>), 0, b->stream, x, pitch,
                             s.rows, static_cast<int>(s.cols), w, bias, static_cast<T>(eps), static_cast<T>(1.0 / static_cast<double>(s.cols)), y, mean,
                             rstd);
    });
}

template <class T>
int fwd_typed(WbBackend* b, const WbView* x, int nd, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    const RowView vx = row_view(*x, nd);
    cudaError_t err = cudaSuccess;
    bool done = false;
    if (plain_rows(vx, s)) {
        const int64_t pitch = vx.st_row[0];
        if (rows_aligned<T>(xp, pitch, s.cols) && rows_aligned<T>(y, s.cols, s.cols) &&
            ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias)) & 15) == 0)
            done = fwd_rows<T, wide<T>>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
        else
            done = fwd_rows<T, 1>(b, xp, pitch, s, w, bias, eps, y, mean, rstd, &err);
    }
    if (!done) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
        err = wb_launch_pdl(ln_fwd_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, vx, s.rows, s.cols, w, bias, eps, y, mean, rstd);
    }
    WB_CHECK_CUDA(err);
    WB_LAUNCH_OK(b);
    return WB_OK;
}

template <class T, int VEC>
bool bwd_rows(WbBackend* b, const T* x, int64_t pitch_x, const T* dy, int64_t pitch_g, const Shape& s, const T* w, const T* mean, const T* rstd, T* dx,
              T* parts, int* slabs, cudaError_t* err) {
    return choose_row<row_elems<T> / VEC>((s.cols + VEC - 1) / VEC, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, N = bwd_threads<TPR>, G = N / TPR, DEPTH = TPR > 512 ? 1 : 2;
        constexpr size_t smem = sizeof(T) * 2 * DEPTH * NV * VEC * N;
        static_assert(smem <= 200 * 1024, "ring");
        auto kernel = ln_bwd_rows_kernel<T, VEC, TPR, NV, DEPTH>;
        *err = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (*err != cudaSuccess) return;
        *slabs = static_cast<int>(std::min<int64_t>(dw_slabs(b->sm_count, s.rows), (s.rows + G - 1) / G));
        *err = wb_launch_pdl(kernel, dim3(*slabs), dim3(N), smem, b->stream, x, pitch_x, dy, pitch_g, s.rows, static_cast<int>(s.cols), w, mean, rstd,
                             static_cast<T>(1.0 / static_cast<double>(s.cols)), dx, parts);
    });
}

template <class T>
int bwd_typed(WbBackend* b, const WbView* x, const WbView* dy, int nd, const Shape& s, const T* w, const T* mean, const T* rstd, T* dx, T* dw, T* db,
              T* parts) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    const T* gp = reinterpret_cast<const T*>(view_data(*dy));
    const RowView vx = row_view(*x, nd), vg = row_view(*dy, nd);
    const bool sums = dw || db;
    if (!dx && !sums) return WB_OK;
    cudaError_t err = cudaSuccess;
    bool done = false;
    int slabs = dw_slabs(b->sm_count, s.rows);
    if (plain_rows(vx, s) && plain_rows(vg, s)) {
        const int64_t px = vx.st_row[0], pg = vg.st_row[0];
        T* to = sums ? parts : nullptr;
        if (rows_aligned<T>(xp, px, s.cols) && rows_aligned<T>(gp, pg, s.cols) && rows_aligned<T>(dx, s.cols, s.cols))
            done = bwd_rows<T, wide<T>>(b, xp, px, gp, pg, s, w, mean, rstd, dx, to, &slabs, &err);
        else
            done = bwd_rows<T, 1>(b, xp, px, gp, pg, s, w, mean, rstd, dx, to, &slabs, &err);
        if (done) {
            WB_CHECK_CUDA(err);
            WB_LAUNCH_OK(b);
        }
    }
    if (!done && dx) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dx_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, w, mean, rstd, dx));
        WB_LAUNCH_OK(b);
    }
    if (!sums) return WB_OK;
    if (!done) {
        const unsigned strips = static_cast<unsigned>(std::min<int64_t>((s.cols + 31) / 32, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dw_any_kernel<T>, dim3(strips, slabs), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, mean, rstd,
                                    parts, slabs));
        WB_LAUNCH_OK(b);
    }
    WB_CHECK_CUDA(wb_launch_pdl(ln_dw_join_kernel<T>, dim3(static_cast<unsigned>((s.cols + 31) / 32), 2), dim3(THREADS), 0, b->stream,
                                static_cast<const T*>(parts), slabs, s.cols, dw, db));
    WB_LAUNCH_OK(b);
    return WB_OK;
}

int64_t bwd_workspace(int sm_count, int64_t rows, int64_t cols, int dtype) {
    if (rows == 0) return 0;
    return 2 * static_cast<int64_t>(dw_slabs(sm_count, rows)) * cols * static_cast<int64_t>(wb_dtype_size(dtype));
}

}  // namespace

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
