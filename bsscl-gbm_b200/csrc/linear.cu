// Device operators for leaf-wise linear models: the softmax cross entropy of
// a linear head with its gradients, products grouped by leaf with theirs, and
// the global norm of many gradients with clipping.  See include/gbm_b200.h.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <exception>
#include <type_traits>
#include <vector>

#include "../../include/gbm_b200.h"
#include "linear_tc.cuh"

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
// launches
// ---------------------------------------------------------------------------

int sm_count() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64 && cached[dev].load()) return cached[dev].load();
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64) cached[dev].store(n);
    return n;
}

// A matrix the tensor cores read: rows of `inner` contiguous values, `ld` from
// one to the next, `batch` matrices of `rows` rows.  box: rows a copy brings.
struct View {
    const void *p;
    int64_t inner, rows, ld;
    int64_t batch = 1;
};

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static std::atomic<EncodeFn> cached;
    EncodeFn f = cached.load();
    if (f) return f;
    void *q = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
        return nullptr;
    f = reinterpret_cast<EncodeFn>(q);
    cached.store(f);
    return f;
}

struct Err {
    int code = GBM_OK;
    const char *what = "";
    bool bad() const { return code != GBM_OK; }
};

// The tensor map of boxes of 64 values by `box` rows (128-byte swizzle).
Err encode(CUtensorMap *map, const View &v, bool bf16, int box) {
    EncodeFn f = encode_fn();
    if (!f) return {GBM_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled"};
    cuuint64_t dims[3] = {(cuuint64_t)v.inner, (cuuint64_t)v.rows, (cuuint64_t)v.batch};
    cuuint64_t strides[2] = {(cuuint64_t)v.ld * 2, (cuuint64_t)(v.batch > 1 ? v.ld * v.rows * 2 : v.ld * 2)};
    cuuint32_t boxes[3] = {64, (cuuint32_t)box, 1}, steps[3] = {1, 1, 1};
    CUresult r = f(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(v.p), dims, strides, boxes,
                   steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return {GBM_ERR_CUDA, "cuTensorMapEncodeTiled refused an operand"};
    return {};
}

// A kernel whose set-up may overlap the end of the launch in front of it: each
// of this file's kernels waits for that one itself (tc::depend).
template <class... P, class... A> Err start(void (*kernel)(P...), int64_t blocks, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaError_t c = cudaLaunchKernelEx(&cfg, kernel, P(args)...); c != cudaSuccess) return {GBM_ERR_CUDA, cudaGetErrorString(c)};
    return {};
}

// One launch of the frame: `units` tiles at most, a cluster of two CTAs for
// each, at most one CTA an SM.  views: A and B, for a launch of two products
// twice.
template <class Op> Err launch(const View *views, const Op &op, bool bf16, int64_t units, cudaStream_t st) {
    if (units <= 0) return {};
    if (units > INT_MAX - 1024) return {GBM_ERR_ARG, "more than 2^31 tiles"};
    tc::Maps maps;
    for (int i = 0; i < (Op::kDual ? 4 : 2); i++) {
        const bool mn = i & 1 ? Op::kBMN : Op::kDual ? i == 2 : Op::kAMN;
        Err e = encode(&maps.m[i], views[i], bf16, mn ? 64 : 128);
        if (e.bad()) return e;
    }
    static std::atomic<uint64_t> ready;     // devices whose limit for this kernel is set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return {GBM_ERR_CUDA, "no current CUDA device"};
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(ready.load() & bit)) {
        if (cudaFuncSetAttribute(tc::k_tc<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, tc::kSmem) != cudaSuccess)
            return {GBM_ERR_CUDA, "the device does not have the kernel's shared memory"};
        ready.fetch_or(bit);
    }
    const int64_t clusters = std::min<int64_t>(units, sm_count() / 2);
    if (clusters < 1) return {GBM_ERR_CUDA, "no SMs"};
    return start(tc::k_tc<Op>, 2 * clusters, tc::kThreads, tc::kSmem, st, maps, op, tc::make_idesc(bf16, Op::kBMN));
}

// Whether TMA can read the rows in place: 16-byte boundaries.
bool tma_rows(const void *p, int64_t ld) { return aligned(p, 16) && ld % 8 == 0; }

// Rows of 16-bit values to rows on 16-byte boundaries, zeros behind the last
// column; a row whose target is ignored becomes zeros where `target` is given.
struct PackJob {
    const uint16_t *src;
    int64_t ld, rows, cols;
    uint16_t *dst;
    int64_t ldp;
    bool vec;
    const int64_t *target;
    int64_t v;
    int64_t chunks() const { return rows * (ldp / 8); }
};

// The 16 bytes at (r, c) of a packed copy.
__device__ __forceinline__ void pack_chunk(const PackJob &j, int64_t r, int64_t c) {
    uint4 q = make_uint4(0, 0, 0, 0);
    bool has = true;
    if (j.target) {
        const int64_t y = j.target[r];
        has = y >= 0 && y < j.v;
    }
    if (has) {
        const uint16_t *s = j.src + r * j.ld + c;
        if (j.vec && c + 8 <= j.cols) {
            q = *(const uint4 *)s;
        } else {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 8; e++) h[e] = c + e < j.cols ? s[e] : 0;
            q = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
    }
    *(uint4 *)(j.dst + r * j.ldp + c) = q;
}

// The power of two that takes m to 2^14 .. 2^15: |G| <= |c| (1 + the error of
// p) stays within half precision's 65504, and what its subnormals round away is
// at most 2^-25 / 2^14 = 2^-39 of m.
__device__ __forceinline__ int scale_exponent(float m) { return m > 0.f && m < INFINITY ? min(max(14 - ilogbf(m), -100), 100) : 0; }

// What a call's other launches need first: copies of operands, and the power
// of two that takes the largest |grad_loss| of the rows that count into half
// precision's range (scale[0], its inverse in scale[1]; by the last block).
struct Prep {
    PackJob job[3];
    int jobs = 0;
    const float *grad_loss = nullptr;
    const int64_t *target = nullptr;
    int64_t n = 0, v = 0;
    float *scale = nullptr;
};

__global__ void __launch_bounds__(256) k_prep(const __grid_constant__ Prep p) {
    tc::depend();
    const int work = gridDim.x - (p.scale ? 1 : 0);
    if ((int)blockIdx.x == work) {
        __shared__ float red[8];
        float m = 0.f;
        for (int64_t i = threadIdx.x; i < p.n; i += 256 * 16) {     // 16 rows of a thread on their way at a time
            int64_t y[16];
            float g[16];
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const int64_t r = min(i + 256 * k, p.n - 1);
                y[k] = p.target[r];
                g[k] = p.grad_loss[r];
            }
#pragma unroll
            for (int k = 0; k < 16; k++) m = fmaxf(m, y[k] >= 0 && y[k] < p.v ? fabsf(g[k]) : 0.f);
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = m;
        __syncthreads();
        if (threadIdx.x) return;
        for (int k = 1; k < 8; k++) m = fmaxf(m, red[k]);
        const int e = scale_exponent(m);
        p.scale[0] = ldexpf(1.f, e);
        p.scale[1] = ldexpf(1.f, -e);
        return;
    }
    const int64_t first = blockIdx.x * 256LL + threadIdx.x, step = work * 256LL;
    for (int k = 0; k < p.jobs; k++) {
        const PackJob &j = p.job[k];
        const int64_t per = j.ldp / 8, total = j.rows * per;
        for (int64_t i = first; i < total; i += step) {
            // 32 bits where they do: a 64-bit division costs more than the copy
            const int64_t r = total >> 31 ? i / per : (int64_t)((uint32_t)i / (uint32_t)per), c = (i - r * per) * 8;
            pack_chunk(j, r, c);
        }
    }
}

Err run_prep(const Prep &p, cudaStream_t st) {
    int64_t most = 0;
    for (int k = 0; k < p.jobs; k++) most = std::max(most, p.job[k].chunks());
    if (!p.jobs && !p.scale) return {};
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((most + 255) / 256, sm_count() * 8LL));
    return start(k_prep, blocks + (p.scale ? 1 : 0), 256, 0, st, p);
}

void add_pack(Prep &p, const View &v, void *room, int64_t ldp, const int64_t *target, int64_t classes) {
    p.job[p.jobs++] = {(const uint16_t *)v.p, v.ld, v.rows * v.batch, v.inner, (uint16_t *)room, ldp, tma_rows(v.p, v.ld), target, classes};
}

// `v` itself, or its copy at `room`, which the prep makes.
View readable(Prep &p, View v, void *room) {
    if (tma_rows(v.p, v.ld)) return v;
    const int64_t ldp = round_up(v.inner, 8);
    add_pack(p, v, room, ldp, nullptr, 0);
    v.p = room;
    v.ld = ldp;
    return v;
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------

// The tiles of one dense product, 8 tiles of m beside one another before the
// next tile of n, so that the 74 tiles worked on at a time share their
// operands in L2; `splits` parts of the k axis one behind the other.
struct Dense {
    int m, n;          // extents of the result
    int nkb;           // stages of the whole k axis
    int splits;        // parts of the k axis
    int mt, nt;        // tiles
    int per;           // stages of a part
    int wide;          // columns of a tile
    tc::Div all, band; // tiles in all, in 8 rows of tiles
    Dense() : m(0), n(0), nkb(0), splits(1), mt(0), nt(0), per(0), wide(256) {}
    Dense(int64_t m_, int64_t n_, int64_t k, int splits_ = 1, int laps = 1, int wide_ = 256)
        : m((int)m_), n((int)n_), nkb((int)((k + tc::kBK - 1) / tc::kBK) * laps), splits(splits_), mt((int)((m_ + 255) / 256)), nt((int)((n_ + wide_ - 1) / wide_)),
          per((nkb + splits_ - 1) / splits_), wide(wide_), all((uint32_t)std::min<int64_t>(tiles(), INT_MAX)), band((uint32_t)std::min<int64_t>(8LL * nt, INT_MAX)) {}
    int64_t tiles() const { return (int64_t)mt * nt; }
    int64_t units() const { return tiles() * splits; }
    // A tile's place is found in 32 bits; launch() refuses more units.
    __device__ void place(uint32_t at, tc::Tile &t) const {
        const uint32_t part = splits > 1 ? all(at) : 0, i = at - part * all.d;
        const uint32_t block = band(i), rest = i - block * band.d, tall = min(8u, mt - block * 8);
        const uint32_t tn = tall == 8 ? rest >> 3 : rest / tall, tm = block * 8 + (rest - tn * tall);
        t.m0 = (int)(tm * 256);
        t.n0 = (int)tn * wide;
        t.mend = min(m - t.m0, 256) + t.m0;
        t.nend = min(n - t.n0, wide) + t.n0;
        t.k0 = 0;
        t.q0 = min((int)part * per, nkb);
        t.nkb = min(per, nkb - t.q0);
        t.bz = 0;
        t.tail = 0;
        t.kind = 0;
        t.aux = (int)part;
    }
};

struct DenseIter {
    uint32_t at, step;
    template <class Op> __device__ DenseIter(const Op &, int cid, int ncl) : at(cid), step(ncl) {}
    template <class Op> __device__ bool next(const Op &op, tc::Tile &t) {
        if (at >= (uint32_t)(op.dense.mt * op.dense.nt) * op.dense.splits) return false;
        op.dense.place(at, t);
        at += step;
        return true;
    }
};

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

// With a few rows a product is a read of the weights, which a 256-row tile's
// loads (128 bytes of each of 128 rows at a time) take at 5 TB/s at most.
// Here a warp takes 16 rows of weights as the m16 of mma.m16n8k16 and reads
// 512 bytes of each at a time, straight into the operand's registers: a lane's
// 16 bytes are 8 values of k of one row, and as both operands are read alike,
// it does not matter that the instruction counts these k's in another order.
// 1 row x 1024 against 32768 classes: 16 us with the joining launch (67 MB, 4.2
// TB/s; 256 blocks on 148 SMs, so that some have two and some one), 64 rows
// through 63 leaves of 1024 x 1024 23.2 us (132 MB, 5.7 TB/s).  Two blocks an SM
// leave a thread 128 registers: k_leaf_few spills 24 bytes, k_xent_few with up
// to 8 rows 8.

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// acc[i][h + 2 j] = w row (g + 8 j) . x row (8 i + 2 c + h), for lane 4 g + c;
// wrows <= 16 and xrows <= 8 NT rows exist (others repeat the last one), K is
// a multiple of 8 and rows start on 16-byte boundaries.
template <class T, int NT>
__device__ __forceinline__ void dot_few(const T *w, int64_t ldw, int wrows, const T *x, int64_t ldx, int xrows, int K, float (&acc)[NT][4]) {
    constexpr int kDeep = NT == 1 ? 8 : 4;      // steps of 32 values of k on their way
    const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4 * 8;
    const T *w0 = w + min(g, wrows - 1) * ldw + c, *w1 = w + min(g + 8, wrows - 1) * ldw + c;
    const T *xr[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) {
        xr[i] = x + min(8 * i + g, xrows - 1) * ldx + c;
        acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    }
    const uint4 none = make_uint4(0, 0, 0, 0);
    for (int k0 = 0; k0 < K; k0 += 32 * kDeep) {
        uint4 a[kDeep], b[kDeep], q[NT][kDeep];
#pragma unroll
        for (int u = 0; u < kDeep; u++) {
            const int k = k0 + 32 * u;
            const bool in = k + c < K;
            a[u] = in ? __ldcs((const uint4 *)(w0 + k)) : none;
            b[u] = in ? __ldcs((const uint4 *)(w1 + k)) : none;
#pragma unroll
            for (int i = 0; i < NT; i++) q[i][u] = in ? __ldg((const uint4 *)(xr[i] + k)) : none;
        }
#pragma unroll
        for (int u = 0; u < kDeep; u++)
#pragma unroll
            for (int i = 0; i < NT; i++) {
                mma16(acc[i], a[u].x, b[u].x, a[u].y, b[u].y, q[i][u].x, q[i][u].y, T{});
                mma16(acc[i], a[u].z, b[u].z, a[u].w, b[u].w, q[i][u].z, q[i][u].w, T{});
            }
    }
}

constexpr int kFewBlocks = 2;     // blocks of 8 warps an SM

// ---------------------------------------------------------------------------
// softmax cross entropy
// ---------------------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (m, s) stands for the sum s exp(m) of exponentials, and s alone where m is
// infinite: with no finite m yet s stays 0 (or NaN, if a NaN is among them), a
// logit of +inf makes it +inf.
__device__ __forceinline__ float shift_of(float m) { return fabsf(m) == INFINITY ? 0.f : m; }
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), shift = shift_of(m);
    return make_float2(m, a.y * ex2((a.x - shift) * kLog2e) + b.y * ex2((b.x - shift) * kLog2e));
}

// A row's loss and lse from its sum of exponentials and its target's logit.
__device__ __forceinline__ void xent_row(float2 a, float ly, int64_t y, int64_t v, float &loss, float &lse) {
    const float z = shift_of(a.x) + logf(a.y);
    lse = z;
    loss = y >= 0 && y < v ? z - ly : 0.f;
}

// x w^T, of which each tile leaves the maximum and the sum of exponentials of
// its 256 classes for each row (part [128 classes][row]), and the target's
// logit; or, where one cluster takes all classes of its rows (whole), the
// rows' loss and lse at once.  One lane of the epilogue has one row, so no
// exchange between lanes is needed.
struct XentStats {
    static constexpr bool kAMN = false, kBMN = false, kTail = false, kDual = false;
    static constexpr int laps = 1;
    struct Iter {
        uint32_t at, step, c;
        __device__ Iter(const XentStats &, int cid, int ncl) : at(cid), step(ncl), c(0) {}
        __device__ bool next(const XentStats &op, tc::Tile &t) {
            const Dense &g = op.dense;
            if (!op.whole) {
                if (at >= (uint32_t)(g.mt * g.nt)) return false;
                g.place(at, t);
                at += step;
                return true;
            }
            if (at >= (uint32_t)g.mt) return false;
            t.m0 = (int)at * 256;
            t.n0 = (int)c * 256;
            t.mend = min(g.m - t.m0, 256) + t.m0;
            t.nend = min(g.n - t.n0, 256) + t.n0;
            t.k0 = t.q0 = t.bz = t.tail = t.kind = t.aux = 0;
            t.nkb = g.nkb;
            if (++c == (uint32_t)g.nt) c = 0, at += step;
            return true;
        }
    };
    struct State {
        float m, s, ly;
        int turn;
    };
    Dense dense;
    bool whole;
    const int64_t *target;
    float2 *part;
    float *ly, *loss, *lse;
    template <class S> __device__ void rest(S &, int, int, int) const {}
    __device__ int64_t rows(const tc::Tile &t, const tc::Place &p) const { return t.m0 + p.row < t.mend ? target[t.m0 + p.row] : -1; }
    template <class R> __device__ void epilogue(const tc::Tile &t, const tc::Place &p, int64_t y, State &st, uint32_t addr, R release) const {
        const int row = t.m0 + p.row, c0 = p.first(), left = min(t.nend - t.n0 - c0, p.wide);    // columns of this half that exist
        const bool in = row < t.mend;
        const int64_t off = y - t.n0 - c0;
        const int yc = off >= 0 && off < left ? (int)off : -1;
        const tc::F2 log2e = tc::f2(kLog2e, kLog2e);
        const bool fresh = !whole || t.n0 == 0;
        float m = fresh ? -INFINITY : st.m, s = fresh ? 0.f : st.s, z = fresh ? 0.f : st.ly;
        if (t.mend - t.m0 <= p.row - p.lane || left <= 0) release();      // no rows, or no columns, of this warp's
#pragma unroll 1
        for (int c = 0; c < left && t.mend - t.m0 > p.row - p.lane; c += 32) {
            float v[32];
            tc::tmem_ld32(addr + c, v);
            tc::tmem_wait(v);
            if (c + 32 >= left) release();
            if (__any_sync(~0u, yc >= c && yc < c + 32)) {
#pragma unroll
                for (int i = 0; i < 32; i++) z = yc == c + i ? v[i] : z;
            }
            if (c + 32 > left) {
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (c + i >= left) v[i] = -INFINITY;
            }
            float top[4] = {m, v[29], v[30], v[31]};
#pragma unroll
            for (int i = 0; i < 28; i += 2) top[i / 2 % 4] = tc::max3(top[i / 2 % 4], v[i], v[i + 1]);
            const float mc = fmaxf(tc::max3(top[0], top[1], top[2]), fmaxf(top[3], v[28]));
            const float shift = shift_of(mc), zs = shift * kLog2e;
            const tc::F2 minus = tc::f2(-zs, -zs);
            tc::F2 e[4] = {tc::f2(s * ex2((m - shift) * kLog2e), 0.f), tc::f2(0.f, 0.f), tc::f2(0.f, 0.f), tc::f2(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float a, b;
                tc::f2_out(tc::f2_fma(tc::f2(v[i], v[i + 1]), log2e, minus), a, b);
                e[i / 2 & 3] = tc::f2_add(e[i / 2 & 3], tc::f2(ex2(a), ex2(b)));
            }
            float a, b;
            tc::f2_out(tc::f2_add(tc::f2_add(e[0], e[1]), tc::f2_add(e[2], e[3])), a, b);
            s = a + b;
            m = mc;
        }
        if (!whole) {
            if (yc >= 0) ly[row] = z;
            if (in) part[((int64_t)(t.n0 / dense.wide) * 2 + p.half) * dense.m + row] = make_float2(m, s);
            return;
        }
        st.m = m;
        st.s = s;
        st.ly = z;
        if (t.nend < dense.n) return;
        // The right half's sums through shared memory.  Of four places: the
        // right warp is never four row tiles ahead of the left one, whose
        // release of tensor memory the products two tiles on wait for.
        const int slot = st.turn & 3, phase = st.turn >> 2 & 1;
        st.turn++;
        if (p.half) {
            *(float4 *)(p.staging + slot * 512 + p.lane * 16) = make_float4(m, s, z, 0.f);
            __syncwarp();
            if (p.lane == 0) tc::mbar_arrive(p.swap + 8 * slot);
            return;
        }
        if (!tc::mbar_wait_warp(p.swap + 8 * slot, phase, p.dead)) return;
        const float4 o = *(const float4 *)(p.staging + 4 * 4096 + slot * 512 + p.lane * 16);
        if (!in) return;
        // one of the halves has the target's logit, the other 0
        xent_row(join(make_float2(m, s), make_float2(o.x, o.y)), z + o.z, y, dense.n, loss[row], lse[row]);
    }
};

// lse and loss from the tiles' parts: 8 rows a block, 32 threads a row.
__global__ void __launch_bounds__(256) k_xent_join(const float2 *__restrict__ part, int64_t n, int64_t nt, int64_t v, const int64_t *__restrict__ target,
                                                   const float *__restrict__ ly, float *__restrict__ loss, float *__restrict__ lse) {
    tc::depend();
    __shared__ float2 sh[32][9];
    const int r = threadIdx.x % 8, q = threadIdx.x / 8;
    const int64_t row = blockIdx.x * 8LL + r;
    float2 a = make_float2(-INFINITY, 0.f);
    if (row < n)
        for (int64_t k = q; k < nt; k += 32 * 8) {      // eight parts on their way at a time
            float2 b[8];
#pragma unroll
            for (int j = 0; j < 8; j++) b[j] = k + 32 * j < nt ? part[(k + 32 * j) * n + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int j = 0; j < 8; j++) a = join(a, b[j]);
        }
    sh[q][r] = a;
    __syncthreads();
    for (int o = 16; o; o >>= 1) {
        if (q < o) sh[q][r] = join(sh[q][r], sh[q + o][r]);
        __syncthreads();
    }
    if (q || row >= n) return;
    xent_row(sh[0][r], ly[row], target[row], v, loss[row], lse[row]);
}

// One piece of G: the logits once more, G = c (exp(l - lse) - [k = target])
// times the scale, rounded to the products' type.  With two parts what the
// rounding leaves is rounded too and follows in a second matrix.
template <class T> struct XentG {
    static constexpr bool kAMN = false, kBMN = false, kTail = false, kDual = false;
    static constexpr int laps = 1;
    using Iter = DenseIter;
    Dense dense;
    int64_t c0, v;      // the piece's first class; classes in all
    const int64_t *target;
    const float *lse, *grad_loss, *scale;
    T *g;
    int64_t ldg, part;  // row stride; from the leading to the trailing part (0: one part)
    // where no launch went before that did them: the copy of x with the
    // ignored rows as zeros (rows 0: done) and half precision's scale
    // (find_scale)
    PackJob copy;
    tc::Div per;        // 16-byte pieces of a row
    float *find_scale;
    struct State {
        float scale;
    };
    __device__ void rest(State &st, int warp, int warps, int lane) const {
        st.scale = scale ? *scale : 1.f;
        if (find_scale) {
            float m = 0.f;
#pragma unroll 8
            for (int i = lane; i < dense.m; i += 32) {
                const int64_t y = target[i];
                m = fmaxf(m, y >= 0 && y < v ? fabsf(grad_loss[i]) : 0.f);
            }
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
            const int e = scale_exponent(m);
            st.scale = ldexpf(1.f, e);
            if (warp == 0 && lane == 0) find_scale[0] = st.scale, find_scale[1] = ldexpf(1.f, -e);
        }
        const uint32_t all = (uint32_t)copy.rows * per.d;
#pragma unroll 4
        for (uint32_t i = warp * 32 + lane; i < all; i += warps * 32) {
            const uint32_t r = per(i);
            pack_chunk(copy, r, (i - r * per.d) * 8);
        }
    }
    struct Rows {
        int64_t y;
        float c, z;
    };
    __device__ Rows rows(const tc::Tile &t, const tc::Place &p) const {
        const int row = t.m0 + p.row;
        Rows r{-1, 0.f, 0.f};
        if (row < t.mend) r = {target[row], grad_loss[row], lse[row] * kLog2e};
        return r;
    }
    template <class R> __device__ void epilogue(const tc::Tile &t, const tc::Place &p, Rows r, State &st, uint32_t addr, R release) const {
        const int h0 = p.first();
        const int64_t y = r.y;
        const float c = r.c * st.scale, z = r.z;
        const bool has = y >= 0 && y < v, all = __all_sync(~0u, has);
        const int64_t off = y - c0 - t.n0 - h0;
        const int yc = has && off >= 0 && off < p.wide ? (int)off : -1;
        const int row0 = t.m0 + p.row - p.lane;
        auto value = [&](float (&x)[32], int col) {
            const bool here = __any_sync(~0u, yc >= col && yc < col + 32);
            const tc::F2 log2e = tc::f2(kLog2e, kLog2e), minus = tc::f2(-z, -z), cc = tc::f2(c, c);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float a, b;
                tc::f2_out(tc::f2_fma(tc::f2(x[i], x[i + 1]), log2e, minus), a, b);
                tc::f2_out(tc::f2_mul(tc::f2(ex2(a), ex2(b)), cc), x[i], x[i + 1]);
            }
            if (here) {
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (yc == col + i) x[i] -= c;
            }
            if (!all) {    // whatever an ignored row's features hold
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = has ? x[i] : 0.f;
            }
        };
        T *out = g + (int64_t)row0 * ldg + t.n0 + h0;
        const int rows = t.mend - row0, cols = t.nend - t.n0 - h0;
        if (part) {
            tc::store_parts<T>(p, addr, out, part, ldg, rows, cols, value, release);
        } else {
            tc::store_tile<T>(p, addr, out, ldg, rows, cols, 8, false, value, release);
        }
    }
};

// Where a product's sums go: rounded to out where one launch's one unit has
// all of them (one split, and the last piece), else as f32 sums to acc
// [split][m][ldacc], on top of an earlier piece's (add); a launch of
// k_sum adds the splits up, always in the same order.  (The last of a tile's
// units to arrive, told by a ticket, adding them up instead took 84 us for
// 2 tiles of 32 splits: one warp's serial reads.)
template <class T> struct Sink {
    const int64_t *target;     // rows whose target is ignored are 0 (null: none)
    int64_t v;
    const float *scale;        // scale[1] takes G's scale back (null: 1)
    T *out;
    int64_t ld;
    int width;
    float *acc;
    int64_t ldacc;
    bool add, last;
};

// A tile's sums to their sink; m, splits: of the product they belong to.
template <class T, class R>
__device__ __forceinline__ void sink_tile(const Sink<T> &k, int m, int splits, const tc::Tile &t, const tc::Place &p, uint32_t addr, R release) {
    const int row = t.m0 + p.row, row0 = row - p.lane, h0 = p.first(), cols = t.nend - t.n0 - h0;
    const float scale = k.scale ? k.scale[1] : 1.f;
    bool has = row < t.mend;
    if (k.target && has) {
        const int64_t y = k.target[row];
        has = y >= 0 && y < k.v;
    }
    T *out = k.out + (int64_t)row0 * k.ld + t.n0 + h0;
    const bool one = splits == 1;
    float *q = k.acc ? k.acc + ((int64_t)t.aux * m + row) * k.ldacc + t.n0 + h0 : nullptr;
    // ldacc is a multiple of 64: whole groups of 32 columns fit
    const auto mine = [&](int c) { return row < t.mend && c < cols; };
    if (row0 >= t.mend) {
        release();
        return;
    }
    if (!k.acc || (one && k.last)) {
        tc::store_tile<T>(
            p, addr, out, k.ld, t.mend - row0, cols, k.width, t.nkb == 0,
            [&](float (&x)[32], int c) {
                if (k.acc && k.add && mine(c)) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float4 o = ((const float4 *)(q + c))[i];
                        x[4 * i] += o.x, x[4 * i + 1] += o.y, x[4 * i + 2] += o.z, x[4 * i + 3] += o.w;
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = has ? x[i] * scale : 0.f;
            },
            release);
        return;
    }
#pragma unroll 1
    for (int c = 0; c < p.wide; c += 32) {
        float x[32];
        if (t.nkb) {
            tc::tmem_ld32(addr + c, x);
            tc::tmem_wait(x);
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = 0.f;
        }
        if (c == p.wide - 32) release();
        if (mine(c)) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float4 w = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                float4 *d = (float4 *)(q + c) + i;
                if (k.add) {
                    const float4 o = *d;
                    w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
                }
                *d = w;
            }
        }
    }
}

// out = the splits' sums, scaled back and rounded; ignored rows 0.
struct SumJob {
    const float *acc;
    int64_t ldacc, m, n;
    int splits;
    const float *scale;
    const int64_t *target;
    int64_t v;
    void *out;
    int64_t ld;
    tc::Div per;       // groups of 4 columns of a row
};

template <class T> __global__ void __launch_bounds__(256) k_sum(const __grid_constant__ SumJob a, const __grid_constant__ SumJob b) {
    tc::depend();
    for (int k = 0; k < 2; k++) {
        const SumJob &j = k ? b : a;
        const uint32_t total = (uint32_t)j.m * j.per.d;
        const float c = j.scale ? j.scale[1] : 1.f;
        for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
            const uint32_t r = j.per(i), col = (i - r * j.per.d) * 4;
            const float *p = j.acc + r * j.ldacc + col;
            float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 8
            for (int q = 0; q < j.splits; q++) {
                const float4 o = *(const float4 *)(p + q * j.m * j.ldacc);
                s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
            }
            bool has = true;
            if (j.target) {
                const int64_t y = j.target[r];
                has = y >= 0 && y < j.v;
            }
            const float x[4] = {s.x, s.y, s.z, s.w};
            T *out = (T *)j.out + r * j.ld + col;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (col + e < j.n) out[e] = from_f<T>(has ? x[e] * c : 0.f);
        }
    }
}

// The sums of up to two products of which parts lie in acc.
template <class T> Err run_sum(SumJob a, SumJob b, cudaStream_t st) {
    for (SumJob *j : {&a, &b}) {
        if (!j->m) continue;
        const int64_t per = (j->n + 3) / 4;
        if (j->m * per > INT_MAX - (1 << 20)) return {GBM_ERR_ARG, "split sums of more than 2^31 pieces"};
        j->per = tc::Div((uint32_t)per);
    }
    const int64_t most = std::max(a.m * (int64_t)a.per.d, b.m * (int64_t)b.per.d);
    return start(k_sum<T>, std::min<int64_t>((most + 255) / 256, sm_count() * 8LL), 256, 0, st, a, b);
}

// dx = G w (A K-major) and dw = G^T x (A's m axis contiguous), B's n axis
// contiguous in both, as one pool of tiles: neither alone fills its last wave.
// The product with the longer k axis goes first.
template <class T> struct XentPair {
    static constexpr bool kAMN = false, kBMN = true, kTail = false, kDual = true;
    struct Iter : tc::Snake {
        __device__ Iter(const XentPair &, int cid, int ncl) : tc::Snake(cid, ncl) {}
        __device__ bool next(const XentPair &op, tc::Tile &t) {
            const uint32_t u0 = (uint32_t)(op.dense[0].mt * op.dense[0].nt) * op.dense[0].splits,
                           u1 = (uint32_t)(op.dense[1].mt * op.dense[1].nt) * op.dense[1].splits;
            if (at >= u0 + u1) return false;
            const int kind = op.first ? at < u1 : at >= u0;
            const uint32_t i = op.first ? (kind ? at : at - u1) : (kind ? at - u0 : at);
            op.dense[kind].place(i, t);
            t.kind = kind;
            step();
            return true;
        }
    };
    Dense dense[2];
    Sink<T> sink[2];
    int first, laps;
    template <class S> __device__ void rest(S &, int, int, int) const {}
    using State = tc::None;
    __device__ int rows(const tc::Tile &, const tc::Place &) const { return 0; }
    template <class R> __device__ void epilogue(const tc::Tile &t, const tc::Place &p, int, tc::None &, uint32_t addr, R release) const {
        sink_tile(sink[t.kind], dense[t.kind].m, dense[t.kind].splits, t, p, addr, release);
    }
};

// Time, in stages of 0.27 us, in which 74 clusters work through u0 units of l0
// stages and then u1 units of l1 <= l0, dealt out back and forth: the longest
// cluster's, counting about 8 stages for a unit's start and end.
double chain(int64_t u0, int64_t l0, int64_t u1, int64_t l1) {
    constexpr int64_t kClusters = 74;      // 148 SMs; fixed, so that sizes alone set the workspace
    l0 += 8;
    l1 += 8;
    const int64_t all = (u0 * l0 + u1 * l1 + kClusters - 1) / kClusters, waves = (u0 + u1 + kClusters - 1) / kClusters,
                  r0 = (u0 + kClusters - 1) / kClusters;
    // at least the mean; a cluster of the fullest wave, which holds as many long units as fit
    return (double)std::max(all, std::min(r0, waves) * l0 + (waves - std::min(r0, waves)) * l1);
}

// A stage's time against a 256 x 256 tile's, for results of d columns.
double stage_cost(int64_t d) { return d > 128 ? 1.0 : d > 64 ? 0.5 : 0.3; }

// Parts of both products' k axes (tx tiles of kx stages, tw of kw): those that
// end first.  Split sums cost a launch, some 5 us, and the time the f32 sums
// take to be written and read again (512 KB a tile, 0.08 us at the memory's
// rate: 0.3 of a stage).  cost: a stage's time against that of a 256 x 256
// tile.
void choose_splits(int64_t tx, int64_t kx, int64_t tw, int64_t kw, double cost, int &sx, int &sw) {
    static constexpr int kTry[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
    double least = 1e300;
    for (int a : kTry) {
        if (a > 1 && (a > kx || !tx)) break;
        for (int b : kTry) {
            if (b > 1 && (b > kw || !tw)) break;
            const int64_t la = (kx + a - 1) / a, lb = (kw + b - 1) / b;
            double t = cost * (la >= lb ? chain(tx * a, la, tw * b, lb) : chain(tw * b, lb, tx * a, la));
            t += (a > 1 || b > 1 ? 20 : 0) + (a > 1 ? tx * a * 0.3 * cost : 0) + (b > 1 ? tw * b * 0.3 * cost : 0);
            if (t < least * 0.98) least = t, sx = a, sw = b;
        }
    }
}

// How the gradient's work is cut: pieces of classes whose G takes at most
// 512 MB, and splits of both products' k axes.  Pieces small enough for L2 lose
// more in partly filled waves and in dx's sums, which every piece reads and
// writes again, than they save in memory traffic (16384 x 1024 x 50001: 48 MB
// 8.5 ms, 96 MB 6.9, 256 MB 5.55, 1024 MB 5.38).
struct XentPlan {
    int64_t dp;        // features in packed rows
    int64_t pc;        // classes of a piece, a multiple of 256 unless there is one piece
    int64_t ldg;       // row stride of G
    int64_t ldacc;
    int parts;         // of G: see below
    int pieces, sx, sw;
    int64_t tx, tw;    // tiles
    XentPlan(int64_t n, int64_t d, int64_t v) {
        dp = round_up(d, 8);
        // One tile of rows: the products are bound by memory and launches,
        // and few rounded values of G weigh in a result (with one row a
        // single one), whose rounding does not average out: keep G in two parts.
        // With more rows G is rounded once, as the results are: dx and dw are
        // 1.43 times as far from 64 bits as with two parts (norm-wise 2.4e-3
        // against 1.66e-3 in bf16, 3.0e-4 against 2.1e-4 in half precision).
        // Two parts double the products: one / two parts, us, 999 x 100 x 1501
        // 24 / 30, 8192 x 64 x 1000 28 / 36, 2048 x 256 x 8192 47 / 67,
        // 4096 x 512 x 16384 189 / 343.
        parts = n <= 256 ? 2 : 1;
        constexpr int64_t kMost = 512 << 20;
        pieces = (int)std::min<int64_t>((n * v * 2 * parts + kMost - 1) / kMost, (v + 255) / 256);
        pieces = std::max(pieces, 1);
        pc = pieces > 1 ? std::min(v, round_up((v + pieces - 1) / pieces, 256)) : v;
        pieces = (int)((v + pc - 1) / pc);
        ldg = round_up(pc, 64);
        ldacc = round_up(d, 64);
        const int64_t dt = (d + 255) / 256;
        tx = (n + 255) / 256 * dt;
        tw = (pc + 255) / 256 * dt;
        choose_splits(tx, (pc + 63) / 64 * parts, tw, (n + 63) / 64 * parts, stage_cost(d), sx, sw);
    }
    bool dx_acc() const { return pieces > 1 || sx > 1; }
};

struct Room {
    char *at, *base;
    explicit Room(void *p) : at((char *)p), base((char *)p) {}
    template <class T> T *take(int64_t count) {
        char *r = at;
        at += round_up(count * (int64_t)sizeof(T), 256);
        return (T *)r;
    }
    int64_t bytes() const { return at - base; }
};

// The loss's parts for up to 8 NT rows: a warp takes 16 classes at a time and
// keeps each row's maximum and sum of exponentials over them; part [block][row].
template <class T, int NT>
__global__ void __launch_bounds__(256, kFewBlocks) k_xent_few(const T *x, int64_t ldx, const T *w, int64_t ldw, int n, int d, int v,
                                                             const int64_t *__restrict__ target, float2 *__restrict__ part, float *__restrict__ ly) {
    tc::depend();
    __shared__ float2 red[8][8 * NT];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
    float2 st[NT][2];
    int y[NT][2];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = 8 * i + 2 * c + h;
            const int64_t t = row < n ? target[row] : -1;
            y[i][h] = t >= 0 && t < v ? (int)t : -1;
            st[i][h] = make_float2(-INFINITY, 0.f);
        }
    for (int64_t k0 = (blockIdx.x * 8LL + warp) * 16; k0 < v; k0 += gridDim.x * 128LL) {
        float acc[NT][4];
        dot_few<T, NT>(w + k0 * ldw, ldw, (int)min(v - k0, (int64_t)16), x, ldx, n, d, acc);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int64_t k = k0 + g + 8 * j;
            if (k >= v) continue;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float l = acc[i][h + 2 * j];
                    if (y[i][h] == k) ly[8 * i + 2 * c + h] = l;
                    // a NaN is no maximum, but stays in the sum
                    st[i][h] = join(st[i][h], make_float2(isnan(l) ? -INFINITY : l, isnan(l) ? l : 1.f));
                }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float2 a = st[i][h];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) a = join(a, make_float2(__shfl_xor_sync(~0u, a.x, o), __shfl_xor_sync(~0u, a.y, o)));
            if (g == 0) red[warp][8 * i + 2 * c + h] = a;
        }
    __syncthreads();
    const int row = threadIdx.x;
    if (row >= n) return;
    float2 a = red[0][row];
#pragma unroll
    for (int k = 1; k < 8; k++) a = join(a, red[k][row]);
    part[(int64_t)blockIdx.x * n + row] = a;
}

// Up to this many rows the loss takes k_xent_few.  On the device, tiles / few
// rows, us, at 8, 16 and 24 rows: 1024 features x 32768 classes 23.0 / 16.2,
// 21.5 / 19.1, 22.4 / 23.2; 256 x 16384 8.8 / 5.7, 8.8 / 6.4, 8.8 / 7.6; 2048 x
// 4096 16.8 / 11.4, 15.7 / 17.1, 15.9 / 25.1.
constexpr int kFewRows = 16;
int64_t few_blocks(int64_t v) { return std::min<int64_t>((v + 127) / 128, 148 * kFewBlocks); }

// Columns of the softmax's tiles: 256, or with so few of those that half the
// clusters or more would stay idle 128 or 64, whose epilogues are as much shorter
// (of a tile of two stages the epilogue is the longest part: 3300 clocks of
// the loss's 256 columns, 6000 of G's).
int xent_wide(int64_t n, int64_t v) {
    const int64_t tiles = (n + 255) / 256 * ((v + 255) / 256);
    return tiles <= 18 ? 64 : tiles <= 37 ? 128 : 256;
}

// Whether one cluster takes all classes of its rows: where that takes no
// longer than tiles for all clusters and a second launch that joins their
// parts (about 16 stages' time; a tile 4 stages on top of its own).
bool xent_whole(int64_t n, int64_t d, int64_t v) {
    const int64_t mt = (n + 255) / 256, nt = (v + 255) / 256, k = (d + 63) / 64 + 4;
    return (mt + 73) / 74 * nt * k <= (mt * nt + 73) / 74 * k + 16;
}

struct XentLoss {
    uint16_t *x, *w;
    float2 *part;
    float *ly;
    int64_t bytes;
    XentLoss(void *ws, int64_t n, int64_t d, int64_t v, bool in_place) {
        Room r(ws);
        const int64_t dp = round_up(d, 8);
        x = r.take<uint16_t>(in_place ? 0 : n * dp);
        w = r.take<uint16_t>(in_place ? 0 : v * dp);
        const bool parts = !xent_whole(n, d, v);
        const int64_t wide = xent_wide(n, v);
        part = r.take<float2>(parts ? std::max((v + wide - 1) / wide * 2, few_blocks(v)) * n : 0);
        ly = r.take<float>(parts ? n : 0);
        bytes = r.bytes();
    }
};

struct XentGrad {
    uint16_t *x, *w, *g;
    float *accx, *accw, *scale;
    int64_t bytes;
    XentGrad(void *ws, int64_t n, int64_t d, int64_t v, bool in_place) {
        Room r(ws);
        const XentPlan pl(n, d, v);
        scale = r.take<float>(2);
        x = r.take<uint16_t>(n * pl.dp);
        w = r.take<uint16_t>(in_place ? 0 : v * pl.dp);
        g = r.take<uint16_t>(n * pl.ldg * pl.parts);
        accx = r.take<float>(pl.dx_acc() ? pl.sx * n * pl.ldacc : 0);
        accw = r.take<float>(pl.sw > 1 ? pl.sw * pl.pc * pl.ldacc : 0);
        bytes = r.bytes();
    }
};

// Sizes whose products of two stay far from 64 bits in every count of bytes (and tiles within 31).
bool sizes_ok(int64_t n, int64_t d, int64_t v) {
    constexpr int64_t kMost = 1LL << 46;
    return n >= 0 && n <= kMaxDim && d >= 1 && d <= kMaxDim && v >= 1 && v <= kMaxDim && n * d <= kMost && v * d <= kMost && n * v <= kMost;
}

Err xent_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, bool bf16, int64_t n, int64_t d, int64_t v, const int64_t *target, float *loss,
                 float *lse, void *ws, cudaStream_t st) {
    XentLoss q(ws, n, d, v, tma_rows(x, ldx) && tma_rows(w, ldw));
    Prep prep;
    const View a = readable(prep, {x, d, n, ldx}, q.x), b = readable(prep, {w, d, v, ldw}, q.w);
    Err e = run_prep(prep, st);
    if (e.bad()) return e;
    const bool whole = xent_whole(n, d, v);
    if (!whole && n <= kFewRows && tma_rows(x, ldx) && tma_rows(w, ldw) && d % 8 == 0) {
        const int64_t blocks = few_blocks(v);
        auto run = [&](auto type, auto rows) {
            using T = decltype(type);
            return start(k_xent_few<T, decltype(rows)::value>, blocks, 256, 0, st, (const T *)x, ldx, (const T *)w, ldw, (int)n, (int)d, (int)v, target, q.part,
                         q.ly);
        };
        auto go = [&](auto type) {
            return n <= 8 ? run(type, std::integral_constant<int, 1>{}) : run(type, std::integral_constant<int, 2>{});
        };
        Err f = bf16 ? go(__nv_bfloat16{}) : go(__half{});
        if (f.bad()) return f;
        return start(k_xent_join, (n + 7) / 8, 256, 0, st, q.part, n, blocks, v, target, q.ly, loss, lse);
    }
    const Dense g(n, v, d, 1, 1, whole ? 256 : xent_wide(n, v));
    XentStats op{g, whole, target, q.part, q.ly, loss, lse};
    const View ab[2] = {a, b};
    e = launch(ab, op, bf16, op.whole ? g.mt : g.units(), st);
    if (e.bad() || op.whole) return e;
    return start(k_xent_join, (n + 7) / 8, 256, 0, st, q.part, n, g.nt * 2LL, v, target, q.ly, loss, lse);
}

template <class T>
Err xent_pair(const XentPlan &pl, const XentGrad &q, const View &xs, const View &wp, const float *scale, int64_t n, int64_t d, int64_t v, int64_t c, int64_t pc,
              const int64_t *target, T *dx, int64_t lddx, T *dw, int64_t lddw, cudaStream_t st) {
    const View gv{q.g, pc, n, pl.ldg, pl.parts};
    const View views[4] = {gv, wp, gv, xs};
    XentPair<T> op{};
    if (dx) {
        op.dense[0] = Dense(n, d, pc, pl.sx, pl.parts);
        op.sink[0] = {target, v, scale, dx, lddx, tc::store_width(dx, lddx), pl.dx_acc() ? q.accx : nullptr, pl.ldacc, c > 0, c + pc == v};
    }
    if (dw) {
        T *o = dw + c * lddw;
        op.dense[1] = Dense(pc, d, n, pl.sw, pl.parts);
        op.sink[1] = {nullptr, 0, scale, o, lddw, tc::store_width(o, lddw), pl.sw > 1 ? q.accw : nullptr, pl.ldacc, false, true};
    }
    op.first = op.dense[1].per > op.dense[0].per;
    op.laps = pl.parts;
    Err e = launch(views, op, std::is_same<T, __nv_bfloat16>::value, op.dense[0].units() + op.dense[1].units(), st);
    SumJob a{}, b{};
    if (dx && pl.sx > 1 && c + pc == v) a = {q.accx, pl.ldacc, n, d, pl.sx, scale, target, v, dx, lddx, {}};
    if (dw && pl.sw > 1) b = {q.accw, pl.ldacc, pc, d, pl.sw, scale, nullptr, 0, dw + c * lddw, lddw, {}};
    return e.bad() || !(a.m || b.m) ? e : run_sum<T>(a, b, st);
}

template <class T>
Err xent_backward(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t n, int64_t d, int64_t v, const int64_t *target, const float *lse,
                  const float *grad_loss, T *dx, int64_t lddx, T *dw, int64_t lddw, void *ws, cudaStream_t st) {
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const XentPlan pl(n, d, v);
    const XentGrad q(ws, n, d, v, tma_rows(x, ldx) && tma_rows(w, ldw));
    // rows that count, zeros in the others': an ignored row's features must not reach dw
    const View xs{q.x, d, n, pl.dp}, given{x, d, n, ldx};
    float *scale = bf16 ? nullptr : q.scale;
    View xv = given, wv{w, d, v, ldw};
    PackJob copy{};
    Err e;
    // G's own launch makes the copy under its first products where that is a few
    // 16-byte pieces a thread of its epilogue (9472 x 1024, some 32 of them:
    // G 170 -> 194K clocks, against 7 us for a launch), and finds half
    // precision's scale where a warp reads all rows in about a microsecond
    const int64_t threads = std::min<int64_t>(74, (n + 255) / 256 * ((pl.pc + 255) / 256)) * 2 * tc::kEpiWarps * 32;
    const bool own = tma_rows(x, ldx) && tma_rows(w, ldw) && (bf16 || n <= 1024) && (!dw || n * (pl.dp / 8) <= 4 * threads);
    if (own) {
        if (dw) {
            Prep one;
            add_pack(one, given, q.x, pl.dp, target, v);
            copy = one.job[0];
        }
    } else {
        Prep prep;
        add_pack(prep, given, q.x, pl.dp, target, v);
        xv = xs;
        wv = readable(prep, wv, q.w);
        if (!bf16) prep.grad_loss = grad_loss, prep.target = target, prep.n = n, prep.v = v, prep.scale = q.scale;
        e = run_prep(prep, st);
    }
    T *g = (T *)q.g;
    for (int64_t c = 0; c < v && !e.bad(); c += pl.pc) {
        const int64_t pc = std::min(pl.pc, v - c);
        View wp = wv;
        wp.p = (const char *)wv.p + c * wv.ld * 2;
        wp.rows = pc;
        const bool first = own && c == 0;
        XentG<T> og{Dense(n, pc, d, 1, 1, xent_wide(n, pc)), c, v, target, lse, grad_loss, first ? nullptr : scale, g, pl.ldg, pl.parts > 1 ? n * pl.ldg : 0,
                    first ? copy : PackJob{}, tc::Div((uint32_t)(pl.dp / 8)), first ? scale : nullptr};
        const View xw[2] = {xv, wp};
        e = launch(xw, og, bf16, og.dense.units(), st);
        if (e.bad()) break;
        e = xent_pair<T>(pl, q, xs, wp, scale, n, d, v, c, pc, target, dx, lddx, dw, lddw, st);
    }
    return e;
}

// ---------------------------------------------------------------------------
// products grouped by leaf
// ---------------------------------------------------------------------------

// Rows [lo, hi) of leaf g, clamped so that no access leaves the arrays.
__device__ __forceinline__ void leaf_rows(const int32_t *off, int32_t g, int64_t t, int &lo, int &hi) {
    lo = (int)min(max((int64_t)off[g], (int64_t)0), t);
    hi = (int)max(min((int64_t)off[g + 1], t), (int64_t)lo);
}

struct Leaves {
    const int32_t *off;
    int64_t t;
    int32_t groups;
    int n;              // columns of the result
    int nkb, nt;
    int tall, wide;     // rows and columns of a tile
    tc::Div band;       // tiles in 8 rows of tiles
    Leaves(const int32_t *off_, int64_t t_, int32_t groups_, int64_t k, int64_t n_, int tall_ = 256, int wide_ = 256)
        : off(off_), t(t_), groups(groups_), n((int)n_), nkb((int)((k + tc::kBK - 1) / tc::kBK)), nt((int)((n_ + wide_ - 1) / wide_)), tall(tall_),
          wide(wide_), band((uint32_t)std::min<int64_t>(8LL * nt, INT_MAX)) {}
    // tiles at most: each leaf may end in a part of one
    int64_t units() const { return ((t + tall - 1) / tall + groups) * nt; }
};

// The tiles of all leaves' rows, leaf after leaf.  A warp looks
// through 32 leaves at a time: each lane counts one leaf's tiles.
struct LeafIter {
    uint32_t at, step, base, total, upto;    // tiles before these 32 leaves, in them, in them up to this lane's
    int first, lo, hi, next_lo, next_hi;     // rows of this lane's leaf, and of its one among the next 32
    template <class Op> __device__ LeafIter(const Op &, int cid, int ncl) : at(cid), step(ncl), base(0), total(0), first(-32) {}
    template <class Op> __device__ void fetch(const Op &op, int g) {
        next_lo = next_hi = 0;
        if (g < op.leaves.groups) leaf_rows(op.leaves.off, g, op.leaves.t, next_lo, next_hi);
    }
    template <class Op> __device__ void look(const Op &op) {
        const int lane = threadIdx.x % 32, g = first + lane;
        if (first == 0) fetch(op, g);
        lo = next_lo;
        hi = next_hi;
        fetch(op, g + 32);
        upto = (uint32_t)((hi - lo + op.leaves.tall - 1) / op.leaves.tall) * op.leaves.nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += u;
        }
        total = __shfl_sync(~0u, upto, 31);
    }
    template <class Op> __device__ bool next(const Op &op, tc::Tile &t) {
        while (first < 0 || at >= base + total) {
            base += total;
            first += 32;
            if (first >= op.leaves.groups) return false;
            look(op);
        }
        const uint32_t rel = at - base, nt = op.leaves.nt;
        const int l = __ffs(__ballot_sync(~0u, upto > rel)) - 1;
        const int a = __shfl_sync(~0u, lo, l), b = __shfl_sync(~0u, hi, l);
        const uint32_t end = __shfl_sync(~0u, upto, l), rt = (b - a + op.leaves.tall - 1) / op.leaves.tall, i = rel - (end - rt * nt);
        // 8 row tiles beside one another, as in Dense
        const uint32_t block = op.leaves.band(i), rest = i - block * op.leaves.band.d, tall = min(8u, rt - block * 8);
        const uint32_t tn = tall == 8 ? rest >> 3 : rest / tall, tm = block * 8 + (rest - tn * tall);
        t.m0 = a + (int)tm * op.leaves.tall;
        t.n0 = (int)tn * op.leaves.wide;
        t.mend = min(b - t.m0, op.leaves.tall) + t.m0;
        t.nend = min(op.leaves.n - t.n0, op.leaves.wide) + t.n0;
        t.k0 = t.q0 = 0;
        t.nkb = op.leaves.nkb;
        t.bz = first + l;
        t.tail = 0;
        t.kind = 0;
        t.aux = 0;
        at += step;
        return true;
    }
};

// Zeros in the rows before the first leaf and behind the last one, a warp a row.
template <class T> __device__ void leaf_rest(const Leaves &l, T *out, int64_t ld, int warp, int warps, int lane) {
    const int64_t lo = min(max((int64_t)l.off[0], (int64_t)0), l.t), hi = max(min((int64_t)l.off[l.groups], l.t), lo), rest = lo + (l.t - hi);
    for (int64_t r = warp; r < rest; r += warps) {
        T *row = out + (r < lo ? r : hi + r - lo) * ld;
        for (int64_t c = lane; c < l.n; c += 32) row[c] = from_f<T>(0.f);
    }
}

// One 256 x 256 tile of leaf's rows times its weights.  Rows behind a leaf's last one belong to the next
// leaf: they are computed with this leaf's weights and not stored.
template <class T> struct LeafOut {
    T *out;
    int64_t ld;
    int width, rest;
    template <class R> __device__ void store(const tc::Tile &t, const tc::Place &p, uint32_t addr, R release) const {
        const int row0 = t.m0 + p.row - p.lane, h0 = p.first();
        tc::store_tile<T>(p, addr, out + (int64_t)row0 * ld + t.n0 + h0, ld, t.mend - row0, t.nend - t.n0 - h0, width, false, [](float (&)[32], int) {}, release);
    }
};

// y = x w^T, leaf by leaf.
template <class T> struct LeafRows {
    static constexpr bool kAMN = false, kBMN = false, kTail = false, kDual = false;
    static constexpr int laps = 1;
    using Iter = LeafIter;
    Leaves leaves;
    LeafOut<T> y;
    __device__ void rest(tc::None &, int warp, int warps, int lane) const {
        if (y.rest) leaf_rest(leaves, y.out, y.ld, warp, warps, lane);
    }
    using State = tc::None;
    __device__ int rows(const tc::Tile &, const tc::Place &) const { return 0; }
    template <class R> __device__ void epilogue(const tc::Tile &t, const tc::Place &p, int, tc::None &, uint32_t addr, R release) const { y.store(t, p, addr, release); }
};

// y = x w^T for leaves of a few rows: a warp takes 8 rows of a leaf and 16 of
// its columns at a time.
template <class T> struct LeafFew {
    Leaves leaves;
    LeafOut<T> y;
    const T *x, *w;
    int64_t ldx;
    int din;
};

template <class T> __global__ void __launch_bounds__(256, kFewBlocks) k_leaf_few(const __grid_constant__ LeafFew<T> op) {
    tc::depend();
    const int lane = threadIdx.x % 32, warp = blockIdx.x * 8 + threadIdx.x / 32, warps = gridDim.x * 8, g = lane / 4, c = lane % 4;
    if (op.y.rest) leaf_rest(op.leaves, op.y.out, op.y.ld, warp, warps, lane);
    LeafIter it(op, warp, warps);
    tc::Tile t;
    while (it.next(op, t)) {
        float acc[1][4];
        dot_few<T, 1>(op.w + ((int64_t)t.bz * op.leaves.n + t.n0) * op.din, op.din, t.nend - t.n0, op.x + t.m0 * op.ldx, op.ldx, t.mend - t.m0, op.din, acc);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int row = t.m0 + 2 * c + (k & 1), col = t.n0 + g + k / 2 * 8;
            if (row < t.mend && col < t.nend) op.y.out[(int64_t)row * op.y.ld + col] = from_f<T>(acc[0][k]);
        }
    }
}

// The leaves in order of their rows, longest first, for the tiles of dw.
constexpr int kSortLeaves = 2048;

__global__ void __launch_bounds__(1024) k_leaf_order(const int32_t *__restrict__ off, int32_t groups, int64_t t, int4 *__restrict__ order) {
    tc::depend();
    __shared__ int rows[kSortLeaves];
    for (int g = threadIdx.x; g < groups; g += 1024) {
        int lo, hi;
        leaf_rows(off, g, t, lo, hi);
        rows[g] = hi - lo;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += 1024) {
        const int mine = rows[g];
        int before = 0;
        for (int k = 0; k < groups; k++) before += rows[k] > mine || (rows[k] == mine && k < g);
        int lo, hi;
        leaf_rows(off, g, t, lo, hi);
        order[before] = make_int4(g, lo, hi, 0);
    }
}

// dw = dy^T x and dx = dy w of all leaves as one pool of units: first dw's
// tiles (of one leaf and one part of its rows, the k axis; longest leaf
// first), then dx's, all of the same short k axis.
template <class T> struct LeafPair {
    static constexpr bool kAMN = false, kBMN = true, kTail = true, kDual = true;
    static constexpr int laps = 1;
    struct Iter : tc::Snake {
        LeafIter dx;
        uint32_t per, first;     // units of one leaf's dw, of all leaves'
        int4 leaf;               // the next unit's leaf and rows: loaded one unit ahead
        __device__ Iter(const LeafPair &op, int cid, int ncl) : tc::Snake(cid, ncl), dx(op, 0, 0) {
            per = op.mt * op.nt * op.splits;
            first = op.sink.out ? per * op.leaves.groups : 0;
            look(op);
        }
        __device__ void look(const LeafPair &op) {
            if (at >= first) return;
            const uint32_t k = op.per(at);
            if (op.order) {
                leaf = op.order[k];
            } else {
                leaf.x = (int)k;
                leaf_rows(op.leaves.off, (int)k, op.leaves.t, leaf.y, leaf.z);
            }
        }
        __device__ bool next(const LeafPair &op, tc::Tile &t) {
            if (at >= first) {
                if (!op.dx.out) return false;
                dx.at = at - first;
                step();
                return dx.next(op, t);
            }
            const uint32_t i = at - op.per(at) * per, part = op.splits > 1 ? op.tiles(i) : 0, tile = i - part * op.tiles.d, tm = op.cols(tile),
                           tn = tile - tm * op.nt;
            const int g = leaf.x, lo = leaf.y, hi = leaf.z;
            step();
            look(op);
            const int nkb = (hi - lo + 63) / 64, each = op.splits > 1 ? (nkb + op.splits - 1) / op.splits : nkb, k0 = min((int)part * each, nkb),
                      k1 = min(k0 + each, nkb);
            t.m0 = (int)tm * 256;
            t.n0 = (int)tn * 256;
            t.mend = min(op.dout - t.m0, 256) + t.m0;
            t.nend = min(op.leaves.n - t.n0, 256) + t.n0;
            t.k0 = lo;
            t.q0 = k0;
            t.nkb = k1 - k0;
            t.bz = 0;
            t.kind = 1;
            // behind the last row of all TMA fills zeros
            t.tail = k1 == nkb && hi < op.leaves.t ? (hi - lo) % 64 : 0;
            t.aux = (int)(part * op.leaves.groups + g);
            return true;
        }
    };
    Leaves leaves;         // of dx: its columns are dw's too
    LeafOut<T> dx;         // out null: not wanted
    const int4 *order;     // of the leaves (null: as they are)
    int dout, splits, mt, nt;
    tc::Div per, tiles, cols;    // units of one leaf's dw, its tiles, tiles side by side
    Sink<T> sink;          // of the (groups * dout) x din matrix of all leaves' dw; out null: not wanted
    __device__ void rest(tc::None &, int warp, int warps, int lane) const {
        if (dx.out && dx.rest) leaf_rest(leaves, dx.out, dx.ld, warp, warps, lane);
    }
    using State = tc::None;
    __device__ int rows(const tc::Tile &, const tc::Place &) const { return 0; }
    template <class R> __device__ void epilogue(const tc::Tile &t, const tc::Place &p, int, tc::None &, uint32_t addr, R release) const {
        if (!t.kind) {
            dx.store(t, p, addr, release);
            return;
        }
        // the leaf's tile as one of that matrix
        tc::Tile all = t;
        const int g = t.aux % leaves.groups, base = g * dout;
        all.m0 += base;
        all.mend += base;
        all.aux = t.aux / leaves.groups;
        sink_tile(sink, leaves.groups * dout, splits, all, p, addr, release);
    }
};

// Parts of dw's k axis, as if all leaves were alike.
int leaf_splits(int64_t t, int32_t groups, int64_t din, int64_t dout) {
    int none = 1, s = 1;
    choose_splits(0, 0, (int64_t)groups * ((din + 255) / 256) * ((dout + 255) / 256), (t / groups + 63) / 64, stage_cost(din), none, s);
    return s;
}

struct LeafWs {
    uint16_t *x, *w, *dy;
    float *acc;
    int4 *order;
    int64_t ldacc, bytes;
    LeafWs(void *ws, int64_t t, int32_t groups, int64_t din, int64_t dout, bool grad, bool in_place) {
        Room r(ws);
        const int64_t ip = round_up(din, 8), op = round_up(dout, 8);
        x = r.take<uint16_t>(in_place ? 0 : t * ip);
        w = r.take<uint16_t>(in_place ? 0 : groups * dout * ip);
        dy = r.take<uint16_t>(in_place || !grad ? 0 : t * op);
        ldacc = round_up(din, 64);
        const int s = grad ? leaf_splits(t, groups, din, dout) : 1;
        acc = r.take<float>(s > 1 ? s * groups * dout * ldacc : 0);
        order = r.take<int4>(grad ? groups : 0);
        bytes = r.bytes();
    }
};

template <class T>
Err leaf_forward(const void *x, int64_t ldx, const void *w, const int32_t *off, int64_t t, int32_t groups, int64_t din, int64_t dout, T *y, int64_t ldy,
                 bool zero_rest, void *ws, cudaStream_t st) {
    const LeafWs q(ws, t, groups, din, dout, false, tma_rows(x, ldx) && tma_rows(w, din));
    Prep prep;
    const View a = readable(prep, {x, din, t, ldx}, q.x), b = readable(prep, {w, din, dout, din, groups}, q.w);
    Err e = run_prep(prep, st);
    if (e.bad()) return e;
    // At most 8 rows a leaf on average: bound by reading the weights.  (Row
    // blocks of a leaf that has many more are spread over the warps too.)  On
    // the device, tiles against few rows, us: 63 leaves of 1024 x 1024 30.4 /
    // 26.9 at 8 rows each, 30.6 / 38.1 at 12; 200 of 256 x 256 12.9 / 10.1
    // at 8, 13.2 / 13.0 at 16.
    if (t <= 8LL * groups && din % 8 == 0 && tma_rows(x, ldx) && tma_rows(w, din)) {
        LeafFew<T> few{Leaves(off, t, groups, din, dout, 8, 16), {y, ldy, 1, zero_rest}, (const T *)x, (const T *)w, ldx, (int)din};
        if (few.leaves.units() > INT_MAX - (1 << 20)) return {GBM_ERR_ARG, "more than 2^31 tiles"};
        return start(k_leaf_few<T>, std::min<int64_t>((few.leaves.units() + 7) / 8, sm_count() * kFewBlocks), 256, 0, st, few);
    }
    LeafRows<T> op{Leaves(off, t, groups, din, dout), {y, ldy, tc::store_width(y, ldy), zero_rest}};
    const View views[2] = {a, b};
    // a cluster at least for the rows outside the leaves
    return launch(views, op, std::is_same<T, __nv_bfloat16>::value, op.leaves.units(), st);
}

template <class T>
Err leaf_backward(const void *x, int64_t ldx, const void *w, const int32_t *off, const void *dy, int64_t lddy, int64_t t, int32_t groups, int64_t din,
                  int64_t dout, T *dx, int64_t lddx, bool zero_rest, T *dw, void *ws, cudaStream_t st) {
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const bool in_place = (!dw || tma_rows(x, ldx)) && (!dx || tma_rows(w, din)) && tma_rows(dy, lddy);
    const LeafWs q(ws, t, groups, din, dout, true, in_place);
    if (!t) {
        if (dw && cudaMemsetAsync(dw, 0, (size_t)groups * dout * din * 2, st) != cudaSuccess) return {GBM_ERR_CUDA, "cudaMemsetAsync"};
        return {};
    }
    Prep prep;
    const View g = readable(prep, {dy, dout, t, lddy}, q.dy);
    View a{}, b{};
    if (dx) b = readable(prep, {w, din, dout, din, groups}, q.w);
    if (dw) a = readable(prep, {x, din, t, ldx}, q.x);
    Err e = run_prep(prep, st);
    const int s = leaf_splits(t, groups, din, dout), mt = (int)((dout + 255) / 256), nt = (int)((din + 255) / 256);
    LeafPair<T> op{Leaves(off, t, groups, dout, din), {}, nullptr, (int)dout, s, mt, nt, {}, {}, {}, {}};
    if ((int64_t)mt * nt * s > INT_MAX) return {GBM_ERR_ARG, "more than 2^31 tiles"};
    op.per = tc::Div((uint32_t)(mt * nt * s));
    op.tiles = tc::Div((uint32_t)(mt * nt));
    op.cols = tc::Div((uint32_t)nt);
    int64_t units = 0;
    if (dx) {
        op.dx = {dx, lddx, tc::store_width(dx, lddx), zero_rest};
        units += op.leaves.units();
    }
    if (dw) {
        const int64_t own = (int64_t)groups * s * mt * nt;
        // more units than clusters: their order decides how evenly the
        // clusters end, which is worth a launch (3 us) from some 64 stages (17 us) a cluster on
        if (own > sm_count() / 2 && (t / 64) * mt * nt >= 64LL * 74 && groups > 1 && groups <= kSortLeaves && !e.bad()) {
            e = start(k_leaf_order, 1, 1024, 0, st, off, groups, t, q.order);
            op.order = q.order;
        }
        op.sink = {nullptr, 0, nullptr, dw, din, tc::store_width(dw, din), s > 1 ? q.acc : nullptr, q.ldacc, false, true};
        units += own;
    }
    if (e.bad()) return e;
    const View views[4] = {g, dx ? b : a, g, dw ? a : b};
    e = launch(views, op, bf16, units, st);
    if (e.bad() || !dw || s == 1) return e;
    return run_sum<T>({q.acc, q.ldacc, groups * dout, din, s, nullptr, nullptr, 0, dw, din, {}}, {}, st);
}

// ---------------------------------------------------------------------------
// norm and clipping
// ---------------------------------------------------------------------------

// One cooperative launch: every block sums the squares of its share, the grid
// meets once, every block adds up all blocks' sums in the same order, and
// every block scales its share, the last piece first, while L2 still holds
// it.  Bound by memory: two reads and a write of what L2 does not keep.
// The shares are equal across the gradients' ends: with items of fixed size
// dealt out in turn the slowest block or warp took half as long again as the
// mean (300 ragged bf16 gradients, 30M elements: 41 us).
constexpr uint64_t kClipMagic = 0x47424d434c495031ull;
constexpr int kClipBlocks = 4;                // blocks of 256 threads an SM
constexpr int kClipShares = 148 * kClipBlocks;
constexpr int64_t kClipLeast = 512;           // elements of a share: a thread's 2, so that many small gradients are not read one behind the other

struct ClipItem {
    const void *src;
    void *dst;
    int32_t n;
    int32_t dtype;
};
struct ClipPlan {
    uint64_t magic;
    int64_t items;
    int32_t shares, pad;
    int32_t start[kClipShares + 1];    // each share's first item
    int32_t pad2;
    // ClipItem[items] follow
};
static_assert(sizeof(ClipPlan) % 16 == 0, "");

// The elements of all gradients behind one another, cut into units dealt out to
// the shares in turn: as many units a share as keep a unit within 16384
// elements.  (One run of elements a share leaves the blocks reading 592
// places far apart: 400M f32 888 us against 771.)
struct ClipCut {
    int64_t shares, units, each;      // units of a share, elements of a unit: a multiple of 64 (of 16 bytes whatever the type)
    explicit ClipCut(int64_t total) {
        shares = std::max<int64_t>(1, std::min<int64_t>(kClipShares, total / kClipLeast));
        units = std::max<int64_t>(1, (total + shares * 16384 - 1) / (shares * 16384));
        each = std::max<int64_t>(64, round_up((total + shares * units - 1) / (shares * units), 64));
    }
};

template <class T> __device__ __forceinline__ void square_add(uint4 q, double *s) {
    const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
    for (int k = 0; k < (int)(16 / sizeof(T)); k++) {
        const double v = to_f(e[k]);
        s[k & 3] = fma(v, v, s[k & 3]);
    }
}

// elements before the first 16-byte boundary
template <class T> __device__ __forceinline__ int head_of(const T *p, int n) {
    return min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
}

constexpr int kClipDeep = 4;      // 16-byte loads a thread keeps in flight

template <class T> __device__ void sum_sq(const T *p, int n, double *s) {
    constexpr int kVec = 16 / sizeof(T);
    const int head = head_of(p, n), tid = threadIdx.x;
    const int nv = (n - head) / kVec, rest = head + nv * kVec + tid;
    if (tid < head) {
        const double v = to_f(p[tid]);
        s[0] = fma(v, v, s[0]);
    }
    if (rest < n) {
        const double v = to_f(p[rest]);
        s[1] = fma(v, v, s[1]);
    }
    const uint4 *q = (const uint4 *)(p + head);
    int i = tid;
    for (; i + 256 * (kClipDeep - 1) < nv; i += 256 * kClipDeep) {
        uint4 a[kClipDeep];
#pragma unroll
        for (int k = 0; k < kClipDeep; k++) a[k] = __ldg(q + i + 256 * k);
#pragma unroll
        for (int k = 0; k < kClipDeep; k++) square_add<T>(a[k], s);
    }
    uint4 a[kClipDeep - 1];
#pragma unroll
    for (int k = 0; k < kClipDeep - 1; k++) a[k] = i + 256 * k < nv ? __ldg(q + i + 256 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kClipDeep - 1; k++) square_add<T>(a[k], s);
}

template <class T> __device__ __forceinline__ uint4 scaled(uint4 q, float c) {
    T *e = reinterpret_cast<T *>(&q);
#pragma unroll
    for (int k = 0; k < (int)(16 / sizeof(T)); k++) e[k] = from_f<T>(to_f(e[k]) * c);
    return q;
}

// p and q may be the same: no load goes through the read-only path here
template <class T> __device__ void scale_to(const T *p, T *q, int n, float c) {
    constexpr int kVec = 16 / sizeof(T);
    const int tid = threadIdx.x;
    if ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15) {
        // no common boundary: element by element
        for (int i = tid; i < n; i += 256 * 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = to_f(p[min(i + 256 * k, n - 1)]);
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (i + 256 * k < n) q[i + 256 * k] = from_f<T>(v[k] * c);
        }
        return;
    }
    const int head = head_of(p, n);
    const int nv = (n - head) / kVec, rest = head + nv * kVec + tid;
    if (tid < head) q[tid] = from_f<T>(to_f(p[tid]) * c);
    if (rest < n) q[rest] = from_f<T>(to_f(p[rest]) * c);
    const uint4 *a = (const uint4 *)(p + head);
    uint4 *b = (uint4 *)(q + head);
    int i = tid;
    for (; i + 256 * (kClipDeep - 1) < nv; i += 256 * kClipDeep) {
        uint4 v[kClipDeep];
#pragma unroll
        for (int k = 0; k < kClipDeep; k++) v[k] = a[i + 256 * k];
#pragma unroll
        for (int k = 0; k < kClipDeep; k++) __stcs(b + i + 256 * k, scaled<T>(v[k], c));
    }
    for (; i < nv; i += 256) __stcs(b + i, scaled<T>(a[i], c));
}

// The same in every lane.
__device__ __forceinline__ double warp_sum(double s) {
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    return s;
}

__global__ void __launch_bounds__(256, kClipBlocks) k_clip(const ClipPlan *__restrict__ plan, double max_norm, float *norm, double *part) {
    __shared__ double red[8];
    const ClipItem *items = reinterpret_cast<const ClipItem *>(plan + 1);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, shares = plan->shares;
    for (int b = blockIdx.x; b < shares; b += gridDim.x) {
        double s[4] = {0, 0, 0, 0};
        const int end = plan->start[b + 1];
        int i = plan->start[b];
        ClipItem next = items[min(i, end - 1)];      // a piece's place is on its way while the one before it is read
        for (; i < end; i++) {
            const ClipItem it = next;
            next = items[min(i + 1, end - 1)];
            if (it.dtype == GBM_TYPE_F32)
                sum_sq((const float *)it.src, it.n, s);
            else if (it.dtype == GBM_TYPE_BF16)
                sum_sq((const __nv_bfloat16 *)it.src, it.n, s);
            else
                sum_sq((const __half *)it.src, it.n, s);
        }
        const double w = warp_sum((s[0] + s[1]) + (s[2] + s[3]));
        if (lane == 0) red[warp] = w;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0;
            for (int k = 0; k < 8; k++) t += red[k];
            part[b] = t;
        }
        __syncthreads();
    }
    cooperative_groups::this_grid().sync();
    double t = 0;
    for (int k = threadIdx.x; k < shares; k += 256) t += __ldcg(part + k);
    t = warp_sum(t);
    if (lane == 0) red[warp] = t;
    __syncthreads();
    t = 0;
    for (int k = 0; k < 8; k++) t += red[k];
    const double r = sqrt(t), f = max_norm / (r + 1e-6);
    const float c = (float)(f > 1.0 ? 1.0 : f);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)r;
    for (int b = blockIdx.x; b < shares; b += gridDim.x) {
        const int begin = plan->start[b];
        int i = plan->start[b + 1] - 1;
        ClipItem next = items[max(i, begin)];
        for (; i >= begin; i--) {
            const ClipItem it = next;
            next = items[max(i - 1, begin)];
            if (c == 1.f && it.src == it.dst) continue;
            if (it.dtype == GBM_TYPE_F32)
                scale_to((const float *)it.src, (float *)it.dst, it.n, c);
            else if (it.dtype == GBM_TYPE_BF16)
                scale_to((const __nv_bfloat16 *)it.src, (__nv_bfloat16 *)it.dst, it.n, c);
            else
                scale_to((const __half *)it.src, (__half *)it.dst, it.n, c);
        }
    }
}

// Calls item(gradient, first element, elements, share) for the pieces of all
// gradients, share after share.
template <class F> void clip_items(const int64_t *sizes, int32_t n, F item) {
    std::vector<int64_t> edge(1, 0);
    // each gradient begins on a multiple of 64, so that every piece of it does in its own memory
    for (int32_t i = 0; i < n; i++) edge.push_back(edge.back() + round_up(sizes[i], 64));
    const int64_t total = edge.back();
    const ClipCut cut(total);
    for (int64_t s = 0; s < cut.shares; s++)
        for (int64_t u = 0; u < cut.units; u++) {
            int64_t at = (u * cut.shares + s) * cut.each;
            const int64_t end = std::min(total, at + cut.each);
            if (at >= end) continue;
            size_t i = std::upper_bound(edge.begin(), edge.end(), at) - edge.begin() - 1;
            for (; at < end; i++) {
                const int64_t take = std::min(end, edge[i] + sizes[i]) - at;
                if (take > 0) item((int32_t)i, at - edge[i], take, s);
                at = std::max(at, std::min(end, edge[i + 1]));
            }
        }
}

// A call's answer: each launch has told its own error.  (The thread's last
// error may be that of an earlier call, which has told it.)
int finish(const char *what, const Err &e, char *errbuf, int32_t errlen) {
    if (!e.bad()) return GBM_OK;
    cudaGetLastError();
    return fail(errbuf, errlen, e.code, "%s: %s", what, e.what);
}

int type_size(int32_t t) { return t == GBM_TYPE_F32 ? 4 : t == GBM_TYPE_BF16 || t == GBM_TYPE_F16 ? 2 : 0; }

}  // namespace

extern "C" {

int64_t gbm_softmax_xent_workspace(int64_t n, int64_t d, int64_t v, int32_t grad, int32_t in_place) {
    if (!sizes_ok(n, d, v)) return -1;
    return grad ? XentGrad(nullptr, n, d, v, in_place != 0).bytes : XentLoss(nullptr, n, d, v, in_place != 0).bytes;
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
    const int64_t need = gbm_softmax_xent_workspace(n, d, v, grad, tma_rows(x, ldx) && tma_rows(w, ldw));
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
    Err e = xent_forward(x, ldx, w, ldw, dtype == GBM_TYPE_BF16, n, d, v, target, loss, lse, ws, static_cast<cudaStream_t>(stream));
    return finish("gbm_softmax_xent", e, errbuf, errlen);
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
        const bool ok = !dw || cudaMemset2DAsync(dw, lddw * 2, 0, d * 2, v, st) == cudaSuccess;
        return finish(what, ok ? Err{} : Err{GBM_ERR_CUDA, "cudaMemset2DAsync"}, errbuf, errlen);
    }
    Err e = dtype == GBM_TYPE_BF16
                ? xent_backward(x, ldx, w, ldw, n, d, v, target, lse, grad_loss, (__nv_bfloat16 *)dx, lddx, (__nv_bfloat16 *)dw, lddw, ws, st)
                : xent_backward(x, ldx, w, ldw, n, d, v, target, lse, grad_loss, (__half *)dx, lddx, (__half *)dw, lddw, ws, st);
    return finish(what, e, errbuf, errlen);
}

static bool leaf_ok(int64_t t, int32_t groups, int64_t din, int64_t dout) {
    return sizes_ok(t, din, dout) && groups >= 1 && groups < 65536 && groups * dout <= kMaxDim && groups * dout * din <= 1LL << 46;
}

int64_t gbm_leaf_linear_workspace(int64_t t, int32_t groups, int64_t din, int64_t dout, int32_t grad, int32_t in_place) {
    if (!leaf_ok(t, groups, din, dout)) return -1;
    return LeafWs(nullptr, t, groups, din, dout, grad != 0, in_place != 0).bytes;
}

static int leaf_check(const char *what, const int32_t *offsets, int32_t dtype, int64_t t, int32_t groups, int64_t din,
                      int64_t dout, bool in_place, const void *ws, int64_t ws_bytes, int32_t grad, char *errbuf, int32_t errlen) {
    if (dtype != GBM_TYPE_BF16 && dtype != GBM_TYPE_F16)
        return fail(errbuf, errlen, GBM_ERR_UNSUPPORTED, "%s: type %d is neither bf16 nor f16", what, dtype);
    if (!leaf_ok(t, groups, din, dout))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: sizes t=%lld groups=%d din=%lld dout=%lld out of range", what,
                    (long long)t, groups, (long long)din, (long long)dout);
    if (!offsets || !aligned(offsets, 4)) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: offsets null or not aligned", what);
    const int64_t need = gbm_leaf_linear_workspace(t, groups, din, dout, grad, in_place);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 256)))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", what,
                    (long long)ws_bytes, (long long)need);
    return GBM_OK;
}

int gbm_leaf_linear(const void *x, int64_t ldx, const void *w, const int32_t *offsets, int32_t dtype, int64_t t,
                    int32_t groups, int64_t din, int64_t dout, void *y, int64_t ldy, int32_t zero_rest, void *ws,
                    int64_t ws_bytes, void *stream, char *errbuf, int32_t errlen) {
    const char *what = "gbm_leaf_linear";
    int rc = leaf_check(what, offsets, dtype, t, groups, din, dout, tma_rows(x, ldx) && tma_rows(w, din), ws, ws_bytes, 0, errbuf,
                        errlen);
    if (rc != GBM_OK) return rc;
    if (!w || (t && (!x || !y)) || !aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer", what);
    if (ldx < din || ldy < dout) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row stride below its row", what);
    if (!t) return GBM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Err e = dtype == GBM_TYPE_BF16 ? leaf_forward(x, ldx, w, offsets, t, groups, din, dout, (__nv_bfloat16 *)y, ldy, zero_rest != 0, ws, st)
                                   : leaf_forward(x, ldx, w, offsets, t, groups, din, dout, (__half *)y, ldy, zero_rest != 0, ws, st);
    return finish(what, e, errbuf, errlen);
}

int gbm_leaf_linear_grad(const void *x, int64_t ldx, const void *w, const int32_t *offsets, const void *dy,
                         int64_t lddy, int32_t dtype, int64_t t, int32_t groups, int64_t din, int64_t dout, void *dx,
                         int64_t lddx, int32_t zero_rest, void *dw, void *ws, int64_t ws_bytes, void *stream,
                         char *errbuf, int32_t errlen) {
    const char *what = "gbm_leaf_linear_grad";
    int rc = leaf_check(what, offsets, dtype, t, groups, din, dout,
                        (!dw || tma_rows(x, ldx)) && (!dx || tma_rows(w, din)) && tma_rows(dy, lddy), ws, ws_bytes, 1, errbuf, errlen);
    if (rc != GBM_OK) return rc;
    if (!dx && !dw) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: neither dx nor dw", what);
    if ((t && !dy) || (dx && !w) || (t && dw && !x) || !aligned(x, 2) || !aligned(w, 2) || !aligned(dy, 2) ||
        !aligned(dx, 2) || !aligned(dw, 2))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer", what);
    if (lddy < dout || (dw && ldx < din) || (dx && lddx < din))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: row stride below its row", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Err e = dtype == GBM_TYPE_BF16 ? leaf_backward(x, ldx, w, offsets, dy, lddy, t, groups, din, dout, (__nv_bfloat16 *)dx, lddx, zero_rest != 0,
                                                   (__nv_bfloat16 *)dw, ws, st)
                                   : leaf_backward(x, ldx, w, offsets, dy, lddy, t, groups, din, dout, (__half *)dx, lddx, zero_rest != 0, (__half *)dw, ws, st);
    return finish(what, e, errbuf, errlen);
}

int64_t gbm_grad_clip_plan_bytes(const int64_t *sizes, int32_t n) {
    if (n < 0 || (n && !sizes)) return -1;
    int64_t total = 0, items = 0;
    for (int32_t i = 0; i < n; i++) {
        if (sizes[i] < 0 || sizes[i] > (1LL << 40)) return -1;
        total += sizes[i];
        if (total > (1LL << 40)) return -1;
    }
    try {
        clip_items(sizes, n, [&](int32_t, int64_t, int64_t, int64_t) { items++; });
    } catch (const std::exception &) {
        return -1;
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
    std::memset(plan, 0, sizeof *plan);
    plan->magic = kClipMagic;
    try {
        clip_items(sizes, n, [&](int32_t i, int64_t at, int64_t count, int64_t share) {
            const int b = type_size(dtypes[i]);
            it[plan->items++] = {(const char *)src[i] + at * b, (char *)dst[i] + at * b, (int32_t)count, dtypes[i]};
            plan->shares = (int32_t)share + 1;
            plan->start[share + 1] = (int32_t)plan->items;
        });
    } catch (const std::exception &) {
        plan->magic = 0;
        return fail(errbuf, errlen, GBM_ERR_ALLOC, "%s: out of host memory", what);
    }
    return GBM_OK;
}

int64_t gbm_grad_clip_workspace(const void *plan_host) {
    const ClipPlan *plan = static_cast<const ClipPlan *>(plan_host);
    if (!plan || plan->magic != kClipMagic) return -1;
    return std::max(1, plan->shares) * 8;
}

int gbm_grad_clip(const void *plan_host, const void *plan_dev, double max_norm, float *norm, void *ws,
                  int64_t ws_bytes, void *stream, char *errbuf, int32_t errlen) {
    const char *what = "gbm_grad_clip";
    const int64_t need = gbm_grad_clip_workspace(plan_host);
    if (need < 0) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: not a plan of gbm_grad_clip_plan", what);
    if (!plan_dev || !norm || !ws || ws_bytes < need || !aligned(ws, 16) || !aligned(plan_dev, 16) || !aligned(norm, 4))
        return fail(errbuf, errlen, GBM_ERR_ARG, "%s: null or unaligned pointer, or a workspace below %lld bytes", what, (long long)need);
    if (!(max_norm >= 0)) return fail(errbuf, errlen, GBM_ERR_ARG, "%s: max_norm %g", what, max_norm);
    const int shares = static_cast<const ClipPlan *>(plan_host)->shares;
    const ClipPlan *plan = static_cast<const ClipPlan *>(plan_dev);
    double *part = static_cast<double *>(ws);
    // all blocks are on the device at once
    const int blocks = std::max(1, std::min(shares, sm_count() * kClipBlocks));
    void *args[] = {&plan, &max_norm, &norm, &part};
    cudaError_t e = cudaLaunchCooperativeKernel((const void *)k_clip, dim3((unsigned)blocks), dim3(256), args, 0, static_cast<cudaStream_t>(stream));
    return finish(what, e == cudaSuccess ? Err{} : Err{GBM_ERR_CUDA, cudaGetErrorString(e)}, errbuf, errlen);
}

int gbm_test_ops_expire(int32_t timeout_ms, void *stream, char *errbuf, int32_t errlen) {
    if (timeout_ms < 1 || timeout_ms > 10000) return fail(errbuf, errlen, GBM_ERR_ARG, "gbm_test_ops_expire: %d ms", timeout_ms);
    Err e = start(tc::k_wait, 1, 32, 0, static_cast<cudaStream_t>(stream), timeout_ms * 2000000ll);
    return finish("gbm_test_ops_expire", e, errbuf, errlen);
}

int gbm_test_ops_wait(int32_t timeout_ms, void *stream, char *errbuf, int32_t errlen) {
    const int rc = gbm_test_ops_expire(timeout_ms, stream, errbuf, errlen);
    return rc == GBM_OK ? gbm_ops_status(stream, errbuf, errlen) : rc;
}

int gbm_ops_status(void *stream, char *errbuf, int32_t errlen) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    void *flag = nullptr;
    int late = 0;
    cudaError_t e = cudaGetSymbolAddress(&flag, tc::g_ops_timeout);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess) e = cudaMemcpyAsync(&late, flag, sizeof late, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && late) {
        e = cudaMemsetAsync(flag, 0, sizeof late, st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    if (e != cudaSuccess) return fail(errbuf, errlen, GBM_ERR_CUDA, "gbm_ops_status: %s", cudaGetErrorString(e));
    if (late) return fail(errbuf, errlen, GBM_ERR_TIMEOUT, "gbm_ops_status: a wait inside an operator ran out; its outputs are not valid");
    return GBM_OK;
}

}  // extern "C"
