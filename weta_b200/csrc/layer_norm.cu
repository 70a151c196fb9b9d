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

// Sums the slabs of both partial arrays in order.
template <class T>
__global__ void __launch_bounds__(THREADS) ln_dw_join_kernel(const T* __restrict__ parts, int slabs, int64_t cols, T* __restrict__ dw,
                                                             T* __restrict__ db) {
    wb_pdl_enter();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
    if (c >= cols) return;
    double aw = 0.0, ab = 0.0;
    for (int k = 0; k < slabs; ++k) {
        aw += parts[static_cast<int64_t>(k) * cols + c];
        ab += parts[static_cast<int64_t>(slabs + k) * cols + c];
    }
    if (dw) dw[c] = static_cast<T>(aw);
    if (db) db[c] = static_cast<T>(ab);
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

template <class T>
int fwd_typed(WbBackend* b, const WbView* x, int nd, const Shape& s, const T* w, const T* bias, double eps, T* y, T* mean, T* rstd) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    const RowView vx = row_view(*x, nd);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
    WB_CHECK_CUDA(wb_launch_pdl(ln_fwd_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, vx, s.rows, s.cols, w, bias, eps, y, mean, rstd));
    WB_LAUNCH_OK(b);
    return WB_OK;
}

template <class T>
int bwd_typed(WbBackend* b, const WbView* x, const WbView* dy, int nd, const Shape& s, const T* w, const T* mean, const T* rstd, T* dx, T* dw, T* db,
              T* parts) {
    const T* xp = reinterpret_cast<const T*>(view_data(*x));
    const T* gp = reinterpret_cast<const T*>(view_data(*dy));
    const RowView vx = row_view(*x, nd), vg = row_view(*dy, nd);
    if (dx) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(s.rows, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dx_any_kernel<T>, dim3(grid), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, w, mean, rstd, dx));
        WB_LAUNCH_OK(b);
    }
    if (dw || db) {
        const int slabs = dw_slabs(b->sm_count, s.rows);
        const unsigned strips = static_cast<unsigned>(std::min<int64_t>((s.cols + 31) / 32, 65535));
        WB_CHECK_CUDA(wb_launch_pdl(ln_dw_any_kernel<T>, dim3(strips, slabs), dim3(THREADS), 0, b->stream, xp, vx, gp, vg, s.rows, s.cols, mean, rstd,
                                    parts, slabs));
        WB_LAUNCH_OK(b);
        WB_CHECK_CUDA(wb_launch_pdl(ln_dw_join_kernel<T>, dim3(static_cast<unsigned>((s.cols + THREADS - 1) / THREADS)), dim3(THREADS), 0, b->stream,
                                    static_cast<const T*>(parts), slabs, s.cols, dw, db));
        WB_LAUNCH_OK(b);
    }
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
