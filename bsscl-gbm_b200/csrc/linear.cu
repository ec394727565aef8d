// Device operators for leaf-wise linear models: the softmax cross entropy of
// a linear head with its gradients, products grouped by leaf with theirs, and
// the global norm of many gradients with clipping.  See include/gbm_b200.h.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../include/gbm_b200.h"

namespace {

constexpr int64_t kMaxDim = (1LL << 31) - 513;

int fail(char *errbuf, int32_t errlen, int code, const char *fmt, ...) {
    if (errbuf && errlen > 0) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(errbuf, (size_t)errlen, fmt, ap);
        va_end(ap);
    }
    return code;
}

bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

template <class T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

// ---------------------------------------------------------------------------
// a plain tiled product: c(m, n) = sum_k a(m, k) b(n, k) in 32 bits
// ---------------------------------------------------------------------------

// One operand: element (i, k) at p[i * si + k * sk].
template <class T> struct Mat {
    const T *p;
    int64_t si, sk;
};

// 64 x 64 tile of 256 threads, 4 x 4 products a thread, 16 values of k a
// step.  epi(m, n, sum) is called for every m < M, n < N.
template <class TA, class TB, class Epi>
__device__ void mm_tile(int64_t m0, int64_t n0, int64_t M, int64_t N, int64_t K, Mat<TA> a, Mat<TB> b, Epi epi) {
    __shared__ float sa[16][68], sb[16][68];
    const int tid = threadIdx.x, tm = tid / 16, tn = tid % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 16) {
        for (int e = tid; e < 64 * 16; e += 256) {
            // the thread index runs along the operand's contiguous direction
            int ia = a.sk == 1 ? e / 16 : e % 64, ka = a.sk == 1 ? e % 16 : e / 64;
            int ib = b.sk == 1 ? e / 16 : e % 64, kb = b.sk == 1 ? e % 16 : e / 64;
            sa[ka][ia] = (m0 + ia < M && k0 + ka < K) ? to_f(a.p[(m0 + ia) * a.si + (k0 + ka) * a.sk]) : 0.f;
            sb[kb][ib] = (n0 + ib < N && k0 + kb < K) ? to_f(b.p[(n0 + ib) * b.si + (k0 + kb) * b.sk]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += sa[k][tm * 4 + i] * sb[k][tn * 4 + j];
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            int64_t m = m0 + tm * 4 + i, n = n0 + tn * 4 + j;
            if (m < M && n < N) epi(m, n, acc[i][j]);
        }
}

// ---------------------------------------------------------------------------
// softmax cross entropy
// ---------------------------------------------------------------------------

template <class T>
__global__ void __launch_bounds__(256) k_xent_logits(const T *x, int64_t ldx, const T *w, int64_t ldw, int64_t n,
                                                     int64_t d, int64_t pc, float *l) {
    mm_tile(blockIdx.y * 64LL, blockIdx.x * 64LL, n, pc, d, Mat<T>{x, ldx, 1}, Mat<T>{w, ldw, 1},
            [=](int64_t m, int64_t k, float v) { l[m * pc + k] = v; });
}

// The running maximum and sum of a row over one more piece of its logits:
// with m' = max(m, max l), s' = s exp(m - m') + sum exp(l - m').
__global__ void __launch_bounds__(256) k_xent_fold(const float *l, int64_t pc, int64_t c0, int64_t v,
                                                   const int64_t *target, float *stat_m, float *stat_s,
                                                   float *loss, float *lse, bool first, bool last) {
    const int64_t i = blockIdx.x;
    const float *row = l + i * pc;
    __shared__ float red[8];
    float m = -INFINITY;
    for (int64_t k = threadIdx.x; k < pc; k += 256) m = fmaxf(m, row[k]);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = m;
    __syncthreads();
    for (int k = 0; k < 8; k++) m = fmaxf(m, red[k]);
    float m0 = first ? -INFINITY : stat_m[i];
    m = fmaxf(m, m0);
    float s = 0.f;
    for (int64_t k = threadIdx.x; k < pc; k += 256) s += m == -INFINITY ? (isnan(row[k]) ? row[k] : 0.f) : __expf(row[k] - m);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x) return;
    s = 0.f;
    for (int k = 0; k < 8; k++) s += red[k];
    if (!first && m0 != -INFINITY) s += stat_s[i] * __expf(m0 - m);
    else if (!first) s += stat_s[i];
    stat_m[i] = m;
    stat_s[i] = s;
    const int64_t y = target[i];
    if (first) loss[i] = 0.f;
    if (y >= c0 && y < c0 + pc && y < v) loss[i] = row[y - c0];
    if (last) {
        float z = m + logf(s);
        lse[i] = z;
        loss[i] = (y >= 0 && y < v) ? z - loss[i] : 0.f;
    }
}

__global__ void __launch_bounds__(256) k_xent_g(float *l, int64_t pc, int64_t c0, int64_t v, const int64_t *target,
                                                const float *lse, const float *grad_loss) {
    const int64_t i = blockIdx.x, y = target[i];
    float *row = l + i * pc;
    const bool has = y >= 0 && y < v;
    const float z = lse[i], c = has ? grad_loss[i] : 0.f;
    for (int64_t k = threadIdx.x; k < pc; k += 256)
        row[k] = has ? c * (__expf(row[k] - z) - (c0 + k == y ? 1.f : 0.f)) : 0.f;
}

template <class T>
__global__ void __launch_bounds__(256) k_xent_dx(const float *g, int64_t pc, const T *w, int64_t ldw, int64_t n,
                                                 int64_t d, float *acc, T *dx, int64_t lddx, bool first, bool last,
                                                 const int64_t *target, int64_t v) {
    mm_tile(blockIdx.y * 64LL, blockIdx.x * 64LL, n, d, pc, Mat<float>{g, pc, 1}, Mat<T>{w, 1, ldw},
            [=](int64_t m, int64_t k, float s) {
                if (!first) s += acc[m * d + k];
                if (last)
                    dx[m * lddx + k] = from_f<T>(target[m] >= 0 && target[m] < v ? s : 0.f);
                else
                    acc[m * d + k] = s;
            });
}

// x with the ignored rows as zeros
template <class T> __global__ void k_xent_rows(const T *x, int64_t ldx, int64_t d, const int64_t *target, int64_t v, T *out) {
    const int64_t i = blockIdx.x;
    const bool has = target[i] >= 0 && target[i] < v;
    for (int64_t k = threadIdx.x; k < d; k += blockDim.x) out[i * d + k] = has ? x[i * ldx + k] : from_f<T>(0.f);
}

template <class T>
__global__ void __launch_bounds__(256) k_xent_dw(const float *g, int64_t pc, const T *x, int64_t n, int64_t d, T *dw,
                                                 int64_t lddw) {
    mm_tile(blockIdx.y * 64LL, blockIdx.x * 64LL, pc, d, n, Mat<float>{g, 1, pc}, Mat<T>{x, 1, d},
            [=](int64_t m, int64_t k, float s) { dw[m * lddw + k] = from_f<T>(s); });
}

// classes of one piece: its logits stay under 64 MB
int64_t xent_piece(int64_t n, int64_t v) {
    return std::min(v, std::max<int64_t>(64, (int64_t)(16 << 20) / std::max<int64_t>(n, 1) / 64 * 64));
}

struct XentWs {
    float *l, *m, *s, *acc;
    void *x;
    int64_t bytes;
    XentWs(void *ws, int64_t n, int64_t d, int64_t v, bool grad) {
        char *p = static_cast<char *>(ws), *at = p;
        auto take = [&](int64_t b) {
            char *r = at;
            at += round_up(b, 256);
            return r;
        };
        l = (float *)take(n * xent_piece(n, v) * 4);
        m = (float *)take(n * 4);
        s = (float *)take(n * 4);
        acc = (float *)take(grad ? n * d * 4 : 0);
        x = take(grad ? n * d * 2 : 0);
        bytes = at - p;
    }
};

bool sizes_ok(int64_t n, int64_t d, int64_t v) {
    return n >= 0 && n <= kMaxDim && d >= 1 && d <= kMaxDim && v >= 1 && v <= kMaxDim;
}

dim3 tiles(int64_t m, int64_t n) { return dim3((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64)); }

template <class T>
void xent_forward(const T *x, int64_t ldx, const T *w, int64_t ldw, int64_t n, int64_t d, int64_t v,
                  const int64_t *target, float *loss, float *lse, void *ws, cudaStream_t st) {
    XentWs q(ws, n, d, v, false);
    const int64_t step = xent_piece(n, v);
    for (int64_t c = 0; c < v; c += step) {
        int64_t pc = std::min(step, v - c);
        k_xent_logits<T><<<tiles(n, pc), 256, 0, st>>>(x, ldx, w + c * ldw, ldw, n, d, pc, q.l);
        k_xent_fold<<<(unsigned)n, 256, 0, st>>>(q.l, pc, c, v, target, q.m, q.s, loss, lse, c == 0, c + pc == v);
    }
}

template <class T>
void xent_backward(const T *x, int64_t ldx, const T *w, int64_t ldw, int64_t n, int64_t d, int64_t v,
                   const int64_t *target, const float *lse, const float *grad_loss, T *dx, int64_t lddx, T *dw,
                   int64_t lddw, void *ws, cudaStream_t st) {
    XentWs q(ws, n, d, v, true);
    T *xr = static_cast<T *>(q.x);
    k_xent_rows<T><<<(unsigned)n, 128, 0, st>>>(x, ldx, d, target, v, xr);
    const int64_t step = xent_piece(n, v);
    for (int64_t c = 0; c < v; c += step) {
        int64_t pc = std::min(step, v - c);
        k_xent_logits<T><<<tiles(n, pc), 256, 0, st>>>(x, ldx, w + c * ldw, ldw, n, d, pc, q.l);
        k_xent_g<<<(unsigned)n, 256, 0, st>>>(q.l, pc, c, v, target, lse, grad_loss);
        if (dx)
            k_xent_dx<T><<<tiles(n, d), 256, 0, st>>>(q.l, pc, w + c * ldw, ldw, n, d, q.acc, dx, lddx, c == 0,
                                                      c + pc == v, target, v);
        if (dw) k_xent_dw<T><<<tiles(pc, d), 256, 0, st>>>(q.l, pc, xr, n, d, dw + c * lddw, lddw);
    }
}

// ---------------------------------------------------------------------------
// products grouped by leaf
// ---------------------------------------------------------------------------

// Rows [lo, hi) of leaf g, clamped so that no access leaves the arrays.
__device__ __forceinline__ void leaf_rows(const int32_t *off, int32_t g, int64_t t, int64_t &lo, int64_t &hi) {
    lo = min(max((int64_t)off[g], (int64_t)0), t);
    hi = max(min((int64_t)off[g + 1], t), lo);
}

// y = x w^T (TRANS 0) or dx = dy w (TRANS 1): one leaf per blockIdx.y, its
// row tiles taken in turn.
template <class T, int TRANS>
__global__ void __launch_bounds__(256) k_leaf_rows(const T *x, int64_t ldx, const T *w, const int32_t *off, int64_t t,
                                                   int64_t K, int64_t N, T *y, int64_t ldy) {
    int64_t lo, hi;
    leaf_rows(off, blockIdx.y, t, lo, hi);
    const T *wg = w + (int64_t)blockIdx.y * K * N;
    Mat<T> b = TRANS ? Mat<T>{wg, 1, N} : Mat<T>{wg, K, 1};
    for (int64_t r = blockIdx.z * 64LL; r < hi - lo; r += gridDim.z * 64LL)
        mm_tile(r, blockIdx.x * 64LL, hi - lo, N, K, Mat<T>{x + lo * ldx, ldx, 1}, b,
                [=](int64_t m, int64_t n, float s) { y[(lo + m) * ldy + n] = from_f<T>(s); });
}

template <class T>
__global__ void __launch_bounds__(256) k_leaf_dw(const T *x, int64_t ldx, const T *dy, int64_t lddy, const int32_t *off,
                                                 int64_t t, int64_t din, int64_t dout, T *dw) {
    int64_t lo, hi;
    leaf_rows(off, blockIdx.z, t, lo, hi);
    T *out = dw + (int64_t)blockIdx.z * dout * din;
    for (int64_t m0 = blockIdx.y * 64LL; m0 < dout; m0 += gridDim.y * 64LL)
        mm_tile(m0, blockIdx.x * 64LL, dout, din, hi - lo, Mat<T>{dy + lo * lddy, 1, lddy},
                Mat<T>{x + lo * ldx, 1, ldx}, [=](int64_t m, int64_t n, float s) { out[m * din + n] = from_f<T>(s); });
}

// The rows before the first leaf and behind the last one as zeros.
template <class T> __global__ void k_leaf_rest(const int32_t *off, int32_t groups, int64_t t, int64_t cols, T *y, int64_t ldy) {
    int64_t lo = min(max((int64_t)off[0], (int64_t)0), t), hi = max(min((int64_t)off[groups], t), lo);
    const int64_t rest = lo + (t - hi);
    for (int64_t r = blockIdx.x; r < rest; r += gridDim.x) {
        T *row = y + (r < lo ? r : hi + r - lo) * ldy;
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) row[c] = from_f<T>(0.f);
    }
}

unsigned row_blocks(int64_t t) { return (unsigned)std::min<int64_t>(64, std::max<int64_t>(1, t / 64)); }

template <class T>
void leaf_rows_launch(const T *x, int64_t ldx, const T *w, const int32_t *off, int64_t t, int32_t groups, int64_t K,
                      int64_t N, bool trans, T *y, int64_t ldy, bool zero_rest, cudaStream_t st) {
    dim3 grid((unsigned)((N + 63) / 64), (unsigned)groups, row_blocks(t));
    if (trans)
        k_leaf_rows<T, 1><<<grid, 256, 0, st>>>(x, ldx, w, off, t, K, N, y, ldy);
    else
        k_leaf_rows<T, 0><<<grid, 256, 0, st>>>(x, ldx, w, off, t, K, N, y, ldy);
    if (zero_rest) k_leaf_rest<T><<<256, 256, 0, st>>>(off, groups, t, N, y, ldy);
}

// ---------------------------------------------------------------------------
// norm and clipping
// ---------------------------------------------------------------------------

constexpr uint64_t kClipMagic = 0x47424d434c495031ull;
constexpr int64_t kClipChunk = 1 << 16;   // elements of one work item

struct ClipItem {
    const void *src;
    void *dst;
    int32_t n;
    int32_t dtype;
};
struct ClipPlan {
    uint64_t magic;
    int64_t items;
    // ClipItem[items] follow
};

template <class T> __device__ double sum_sq(const T *p, int n) {
    double s = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        double v = to_f(p[i]);
        s += v * v;
    }
    return s;
}

__global__ void __launch_bounds__(256) k_clip_norm(const ClipItem *items, double *part) {
    ClipItem it = items[blockIdx.x];
    double s = it.dtype == GBM_TYPE_F32    ? sum_sq((const float *)it.src, it.n)
               : it.dtype == GBM_TYPE_BF16 ? sum_sq((const __nv_bfloat16 *)it.src, it.n)
                                           : sum_sq((const __half *)it.src, it.n);
    __shared__ double red[8];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0;
        for (int k = 0; k < 8; k++) s += red[k];
        part[blockIdx.x] = s;
    }
}

__global__ void __launch_bounds__(1024) k_clip_sum(const double *part, int64_t items, double max_norm, float *norm,
                                                   float *scale) {
    __shared__ double red[1024];
    double s = 0;
    for (int64_t i = threadIdx.x; i < items; i += 1024) s += part[i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = 512; o; o >>= 1) {
        if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        double r = sqrt(red[0]), c = max_norm / (r + 1e-6);
        *norm = (float)r;
        *scale = (float)(c > 1.0 ? 1.0 : c);
    }
}

template <class T> __device__ void scale_to(const T *p, T *q, int n, float c) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) q[i] = from_f<T>(to_f(p[i]) * c);
}

__global__ void __launch_bounds__(256) k_clip_scale(const ClipItem *items, const float *scale) {
    ClipItem it = items[blockIdx.x];
    const float c = *scale;
    if (it.dtype == GBM_TYPE_F32)
        scale_to((const float *)it.src, (float *)it.dst, it.n, c);
    else if (it.dtype == GBM_TYPE_BF16)
        scale_to((const __nv_bfloat16 *)it.src, (__nv_bfloat16 *)it.dst, it.n, c);
    else
        scale_to((const __half *)it.src, (__half *)it.dst, it.n, c);
}

int finish(const char *what, char *errbuf, int32_t errlen) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(errbuf, errlen, GBM_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    return GBM_OK;
}

int type_size(int32_t t) { return t == GBM_TYPE_F32 ? 4 : t == GBM_TYPE_BF16 || t == GBM_TYPE_F16 ? 2 : 0; }

}  // namespace

extern "C" {

int64_t gbm_softmax_xent_workspace(int64_t n, int64_t d, int64_t v, int32_t grad) {
    if (!sizes_ok(n, d, v)) return -1;
    return XentWs(nullptr, n, d, v, grad != 0).bytes;
}

static int xent_check(const char *what, const void *x, int64_t ldx, const void *w, int64_t ldw, int32_t dtype,
                      int64_t n, int64_t d, int64_t v, const int64_t *target, const void *ws, int64_t ws_bytes,
                      int32_t grad, char *errbuf, int32_t errlen) {
    if (dtype != GBM_TYPE_BF16 && dtype != GBM_TYPE_F16)
        return fail(errbuf, errlen, GBM_ERR_UNSUPPORTED, "%s: type %d is neither bf16 nor f16", what, dtype);
    if (!sizes_ok(n, d, v))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: sizes n=%lld d=%lld v=%lld out of range", what, (long long)n,
                    (long long)d, (long long)v);
    if (!w || (n && (!x || !target))) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null pointer", what);
    if (ldx < d || ldw < d)
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row strides %lld, %lld below the row's %lld elements", what,
                    (long long)ldx, (long long)ldw, (long long)d);
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(target, 8) || !aligned(ws, 256))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: a pointer is not aligned to its elements (workspace: 256 bytes)", what);
    const int64_t need = gbm_softmax_xent_workspace(n, d, v, grad);
    if (need && (!ws || ws_bytes < need))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes,
                    (long long)need);
    return GBM_OK;
}

int gbm_softmax_xent(const void *x, int64_t ldx, const void *w, int64_t ldw, int32_t dtype, int64_t n, int64_t d,
                     int64_t v, const int64_t *target, float *loss, float *lse, void *ws, int64_t ws_bytes,
                     void *stream, char *errbuf, int32_t errlen) {
    int rc = xent_check("gbm_softmax_xent", x, ldx, w, ldw, dtype, n, d, v, target, ws, ws_bytes, 0, errbuf, errlen);
    if (rc != GBM_OK) return rc;
    if (n && (!loss || !lse || !aligned(loss, 4) || !aligned(lse, 4)))
        return fail(errbuf, errlen, GBM_ERR_ARG, "gbm_softmax_xent: loss or lse is null or not aligned");
    if (!n) return GBM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == GBM_TYPE_BF16)
        xent_forward((const __nv_bfloat16 *)x, ldx, (const __nv_bfloat16 *)w, ldw, n, d, v, target, loss, lse, ws, st);
    else
        xent_forward((const __half *)x, ldx, (const __half *)w, ldw, n, d, v, target, loss, lse, ws, st);
    return finish("gbm_softmax_xent", errbuf, errlen);
}

int gbm_softmax_xent_grad(const void *x, int64_t ldx, const void *w, int64_t ldw, int32_t dtype, int64_t n, int64_t d,
                          int64_t v, const int64_t *target, const float *lse, const float *grad_loss, void *dx,
                          int64_t lddx, void *dw, int64_t lddw, void *ws, int64_t ws_bytes, void *stream,
                          char *errbuf, int32_t errlen) {
    const char *what = "gbm_softmax_xent_grad";
    int rc = xent_check(what, x, ldx, w, ldw, dtype, n, d, v, target, ws, ws_bytes, 1, errbuf, errlen);
    if (rc != GBM_OK) return rc;
    if (!dx && !dw) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: neither dx nor dw", what);
    if (n && (!lse || !grad_loss || !aligned(lse, 4) || !aligned(grad_loss, 4) || !aligned(dx, 2) || !aligned(dw, 2)))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer", what);
    if ((dx && lddx < d) || (dw && lddw < d))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row stride of an output below its row", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!n) {
        if (dw && cudaMemset2DAsync(dw, lddw * 2, 0, d * 2, v, st) != cudaSuccess) return finish(what, errbuf, errlen);
        return GBM_OK;
    }
    if (dtype == GBM_TYPE_BF16)
        xent_backward((const __nv_bfloat16 *)x, ldx, (const __nv_bfloat16 *)w, ldw, n, d, v, target, lse, grad_loss,
                      (__nv_bfloat16 *)dx, lddx, (__nv_bfloat16 *)dw, lddw, ws, st);
    else
        xent_backward((const __half *)x, ldx, (const __half *)w, ldw, n, d, v, target, lse, grad_loss, (__half *)dx,
                      lddx, (__half *)dw, lddw, ws, st);
    return finish(what, errbuf, errlen);
}

int64_t gbm_leaf_linear_workspace(int64_t t, int32_t groups, int64_t din, int64_t dout, int32_t grad) {
    if (!sizes_ok(t, din, dout) || groups < 1 || groups >= 65536) return -1;
    return 0;
}

static int leaf_check(const char *what, const int32_t *offsets, int32_t dtype, int64_t t, int32_t groups, int64_t din,
                      int64_t dout, const void *ws, int64_t ws_bytes, int32_t grad, char *errbuf, int32_t errlen) {
    if (dtype != GBM_TYPE_BF16 && dtype != GBM_TYPE_F16)
        return fail(errbuf, errlen, GBM_ERR_UNSUPPORTED, "%s: type %d is neither bf16 nor f16", what, dtype);
    if (!sizes_ok(t, din, dout) || groups < 1 || groups >= 65536)
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: sizes t=%lld groups=%d din=%lld dout=%lld out of range", what,
                    (long long)t, groups, (long long)din, (long long)dout);
    if (!offsets || !aligned(offsets, 4)) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: offsets null or not aligned", what);
    const int64_t need = gbm_leaf_linear_workspace(t, groups, din, dout, grad);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 256)))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", what,
                    (long long)ws_bytes, (long long)need);
    return GBM_OK;
}

int gbm_leaf_linear(const void *x, int64_t ldx, const void *w, const int32_t *offsets, int32_t dtype, int64_t t,
                    int32_t groups, int64_t din, int64_t dout, void *y, int64_t ldy, int32_t zero_rest, void *ws,
                    int64_t ws_bytes, void *stream, char *errbuf, int32_t errlen) {
    const char *what = "gbm_leaf_linear";
    int rc = leaf_check(what, offsets, dtype, t, groups, din, dout, ws, ws_bytes, 0, errbuf, errlen);
    if (rc != GBM_OK) return rc;
    if (!w || (t && (!x || !y)) || !aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer", what);
    if (ldx < din || ldy < dout) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row stride below its row", what);
    if (!t) return GBM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == GBM_TYPE_BF16)
        leaf_rows_launch((const __nv_bfloat16 *)x, ldx, (const __nv_bfloat16 *)w, offsets, t, groups, din, dout, false,
                         (__nv_bfloat16 *)y, ldy, zero_rest != 0, st);
    else
        leaf_rows_launch((const __half *)x, ldx, (const __half *)w, offsets, t, groups, din, dout, false, (__half *)y,
                         ldy, zero_rest != 0, st);
    return finish(what, errbuf, errlen);
}

int gbm_leaf_linear_grad(const void *x, int64_t ldx, const void *w, const int32_t *offsets, const void *dy,
                         int64_t lddy, int32_t dtype, int64_t t, int32_t groups, int64_t din, int64_t dout, void *dx,
                         int64_t lddx, int32_t zero_rest, void *dw, void *ws, int64_t ws_bytes, void *stream,
                         char *errbuf, int32_t errlen) {
    const char *what = "gbm_leaf_linear_grad";
    int rc = leaf_check(what, offsets, dtype, t, groups, din, dout, ws, ws_bytes, 1, errbuf, errlen);
    if (rc != GBM_OK) return rc;
    if (!dx && !dw) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: neither dx nor dw", what);
    if ((t && !dy) || (dx && !w) || (t && dw && !x) || !aligned(x, 2) || !aligned(w, 2) || !aligned(dy, 2) ||
        !aligned(dx, 2) || !aligned(dw, 2))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer", what);
    if (lddy < dout || (dw && ldx < din) || (dx && lddx < din))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row stride below its row", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (dx && t)
            leaf_rows_launch((const T *)dy, lddy, (const T *)w, offsets, t, groups, dout, din, true, (T *)dx, lddx,
                             zero_rest != 0, st);
        if (dw) {
            dim3 grid((unsigned)((din + 63) / 64), (unsigned)std::min<int64_t>(65535, (dout + 63) / 64), (unsigned)groups);
            k_leaf_dw<T><<<grid, 256, 0, st>>>((const T *)x, ldx, (const T *)dy, lddy, offsets, t, din, dout, (T *)dw);
        }
    };
    if (dtype == GBM_TYPE_BF16)
        go(__nv_bfloat16{});
    else
        go(__half{});
    return finish(what, errbuf, errlen);
}

int64_t gbm_grad_clip_plan_bytes(const int64_t *sizes, int32_t n) {
    if (n < 0 || (n && !sizes)) return -1;
    int64_t items = 0;
    for (int32_t i = 0; i < n; i++) {
        if (sizes[i] < 0 || sizes[i] > (1LL << 46)) return -1;
        items += (sizes[i] + kClipChunk - 1) / kClipChunk;
        if (items > INT32_MAX) return -1;
    }
    return (int64_t)sizeof(ClipPlan) + items * (int64_t)sizeof(ClipItem);
}

int gbm_grad_clip_plan(const void *const *src, void *const *dst, const int64_t *sizes, const int32_t *dtypes,
                       int32_t n, void *plan_host, int64_t plan_bytes, char *errbuf, int32_t errlen) {
    const char *what = "gbm_grad_clip_plan";
    const int64_t need = gbm_grad_clip_plan_bytes(sizes, n);
    if (need < 0 || (n && (!src || !dst || !dtypes)) || !plan_host)
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null pointer or a size out of range", what);
    if (plan_bytes < need)
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: plan of %lld bytes, %lld needed", what, (long long)plan_bytes,
                    (long long)need);
    struct Span {
        uintptr_t lo, hi;
        int32_t i;
        bool dst;
    };
    try {
        std::vector<Span> spans;
        for (int32_t i = 0; i < n; i++) {
            const int b = type_size(dtypes[i]);
            if (!b) return fail(errbuf, errlen, GBM_ERR_UNSUPPORTED, "%s: gradient %d has type %d (f32, bf16 or f16)", what, i, dtypes[i]);
            if (!sizes[i]) continue;
            if (!src[i] || !dst[i] || !aligned(src[i], b) || !aligned(dst[i], b))
                return fail(errbuf, errlen, GBM_ERR_ARG, "%s: gradient %d: null or unaligned pointer", what, i);
            uintptr_t s = (uintptr_t)src[i], d = (uintptr_t)dst[i];
            spans.push_back({d, d + (uintptr_t)sizes[i] * b, i, true});
            if (s != d) spans.push_back({s, s + (uintptr_t)sizes[i] * b, i, false});
        }
        std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
        // the furthest end so far, over all spans and over those written
        uintptr_t any = 0, out = 0;
        for (const Span &s : spans) {
            if (s.lo < out || (s.dst && s.lo < any))
                return fail(errbuf, errlen, GBM_ERR_ARG, "%s: gradient %d overlaps another buffer", what, s.i);
            any = std::max(any, s.hi);
            if (s.dst) out = std::max(out, s.hi);
        }
    } catch (const std::exception &) {
        return fail(errbuf, errlen, GBM_ERR_ALLOC, "%s: out of host memory", what);
    }
    ClipPlan *plan = static_cast<ClipPlan *>(plan_host);
    ClipItem *it = reinterpret_cast<ClipItem *>(plan + 1);
    plan->magic = kClipMagic;
    plan->items = 0;
    for (int32_t i = 0; i < n; i++) {
        const int b = type_size(dtypes[i]);
        for (int64_t at = 0; at < sizes[i]; at += kClipChunk)
            it[plan->items++] = {(const char *)src[i] + at * b, (char *)dst[i] + at * b,
                                 (int32_t)std::min(kClipChunk, sizes[i] - at), dtypes[i]};
    }
    return GBM_OK;
}

int64_t gbm_grad_clip_workspace(const void *plan_host) {
    const ClipPlan *plan = static_cast<const ClipPlan *>(plan_host);
    if (!plan || plan->magic != kClipMagic) return -1;
    return 16 + plan->items * 8;
}

int gbm_grad_clip(const void *plan_host, const void *plan_dev, double max_norm, float *norm, void *ws,
                  int64_t ws_bytes, void *stream, char *errbuf, int32_t errlen) {
    const char *what = "gbm_grad_clip";
    const int64_t need = gbm_grad_clip_workspace(plan_host);
    if (need < 0) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: not a plan of gbm_grad_clip_plan", what);
    if (!plan_dev || !norm || !ws || ws_bytes < need || !aligned(ws, 16) || !aligned(plan_dev, 16) || !aligned(norm, 4))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer, or a workspace below %lld bytes", what, (long long)need);
    if (!(max_norm >= 0)) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: max_norm %g", what, max_norm);
    const int64_t items = static_cast<const ClipPlan *>(plan_host)->items;
    const ClipItem *it = reinterpret_cast<const ClipItem *>(static_cast<const ClipPlan *>(plan_dev) + 1);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float *scale = static_cast<float *>(ws);
    double *part = reinterpret_cast<double *>(static_cast<char *>(ws) + 16);
    if (items) k_clip_norm<<<(unsigned)items, 256, 0, st>>>(it, part);
    k_clip_sum<<<1, 1024, 0, st>>>(part, items, max_norm, norm, scale);
    if (items) k_clip_scale<<<(unsigned)items, 256, 0, st>>>(it, scale);
    return finish(what, errbuf, errlen);
}

int gbm_ops_status(void *stream, char *errbuf, int32_t errlen) {
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return fail(errbuf, errlen, GBM_ERR_CUDA, "gbm_ops_status: %s", cudaGetErrorString(e));
    return GBM_OK;
}

}  // extern "C"
