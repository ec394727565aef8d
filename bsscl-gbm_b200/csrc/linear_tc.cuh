// Matrix products on the fifth-generation tensor cores: one persistent kernel
// frame for the operators of linear.cu, which differ in how a tile is found
// (Op::Iter) and in what happens to its sums (Op::epilogue).
//
// A cluster of two CTAs works on one 256 x 256 tile.  Each CTA keeps 128 rows
// of A and 128 rows of B in shared memory, 64 values of k a stage, fetched
// by TMA with the 128-byte swizzle; one tcgen05.mma of the pair reads both
// halves, so each SM fetches half of B: 32 KB a stage, 64 bytes a
// clock and SM against the 512 clocks of the stage's products.  The sums lie
// in tensor memory (128 lanes x 256 columns in each CTA), twice, so that one
// tile's epilogue runs under the next one's products.  A tile whose result
// has at most 128 or 64 columns multiplies that many, and boxes of which
// no row or column is wanted are not fetched: what lies in their place ends in
// sums that nobody stores.
//
// Warp 0 fetches, warp 1 of the leading CTA issues the products, warps 2..9
// run the epilogue (warp w reads the tensor memory lanes 32 (w % 4) .. +31,
// warps 2..5 the tile's left columns, warps 6..9 its right ones), warp 10
// tells the products' thread of its tiles and puts zeros behind a k axis that
// ends inside a stage.  (Few products wait in the tensor core's queue: looking
// for the next tile, 500 clocks, 1500 among leaves, by the products' own warp
// idled it.)  The thread that
// fetches and the one that issues products are chosen by elect.sync: under a
// plain test of the lane the compiler does not know that one thread runs, and
// the loops took up to 20 % more clocks than the products.
//
// Every wait for a barrier in shared memory is bounded (2 s, and more where it
// lasts for a whole k axis: wait_clocks): when one runs out, the
// kernel notes it in g_ops_timeout, all roles leave their loops, the copies in
// flight get time to land, tensor memory is freed and the kernel returns; the
// launches behind it, whose inputs it did not make, do nothing until the host
// has asked (so that a long run of them does not wait each its own 2 s).  What
// the hardware waits for by itself ends with that: a barrier of the cluster is
// reached by every warp of both CTAs on every path, the launch in front
// (griddepcontrol.wait) ends as this one does, and tcgen05.alloc finds all of
// the pair's tensor memory free, for
// - both CTAs run (the cluster has met) before either allocates, and neither
//   leaves before both have freed: allocating and freeing are operations of
//   the pair on both SMs;
// - the launch in front, whose CTAs may have left these SMs a moment ago, is
//   over altogether, its tensor memory freed;
// - a CTA's shared memory keeps a second one of this frame off its SM.
// (With the allocation before the CTAs had met, under the launch in front, a
// training loop twice did not come back.)
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tc {

constexpr int kThreads = 352;
constexpr int kEpiWarps = 8;
constexpr int kBK = 64;                       // values of k a stage: 128 bytes
constexpr int kABytes = 128 * kBK * 2;        // A of one CTA and stage
constexpr int kStaging = kEpiWarps * 4096;    // 32 rows x 128 bytes a warp
constexpr long long kWaitClocks = 4000000000ll;   // about 2 s
// A wait that may last for whole k axes gets more: 16 times the 512 clocks of a stage's products for each stage.
__device__ __forceinline__ long long wait_clocks(long long stages) { return kWaitClocks + stages * 8192; }

static __device__ int g_ops_timeout;

constexpr int kBN = 256;
constexpr int kTold = 4;                      // tiles the products' thread may know of ahead
constexpr int kStageBytes = kABytes + kBN / 2 * kBK * 2;
constexpr int kStages = (227 * 1024 - kStaging - 2048) / kStageBytes;
constexpr int kSmem = kStages * kStageBytes + kStaging + 2048;   // 1024 of alignment, 1024 of barriers
static_assert(kStages == 6, "");

// ---- shared memory, barriers ------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The word at this address in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ int load_at(uint32_t addr, uint32_t rank) {
    int v;
    asm volatile("{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %1, %2;\n ld.shared::cluster.b32 %0, [r];\n}" : "=r"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}
// Arrive on the same barrier of the cluster's CTA `rank`.  DATA: with writes
// to shared memory that the other side is to see; tensor memory has its own fences.
template <bool DATA> __device__ __forceinline__ void mbar_arrive_at(uint32_t bar, uint32_t rank) {
    if (DATA)
        asm volatile(
            "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n"
            " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n}" ::"r"(bar), "r"(rank)
            : "memory");
    else
        asm volatile(
            "{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %0, %1;\n"
            " mbarrier.arrive.shared::cluster.b64 _, [r];\n}" ::"r"(bar), "r"(rank)
            : "memory");
}
template <bool DATA> __device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if (DATA)
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.b32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            " selp.b32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    return ok;
}
// Waits for the phase of this parity; false when the wait ran out here or in another warp of the CTA.
template <bool DATA = false> __device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *dead, long long limit = kWaitClocks) {
    if (mbar_try<DATA>(bar, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t i = 1;; i++) {
        if (mbar_try<DATA>(bar, parity)) return true;
        if ((i & 31) == 0) {
            if (*dead) return false;
            if (clock64() - t0 > limit) {
                *dead = 1;
                g_ops_timeout = 1;
                return false;
            }
        }
    }
}
// The same for a whole warp, whose lanes all get the same answer.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int *dead, long long limit = kWaitClocks) {
    const bool ok = mbar_wait(bar, parity, dead, limit);
    return __all_sync(~0u, ok);
}
// One thread of a converged warp, known as such to the compiler.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}

// ---- TMA --------------------------------------------------------------------

// A 3-D tile into this CTA's shared memory, its bytes counted on the leading CTA's barrier.
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// The same, counted on this CTA's own barrier.
__device__ __forceinline__ void tma_own(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// ---- tcgen05 ----------------------------------------------------------------

// Shared memory descriptor, 128-byte swizzle.  K-major: rows of 128 bytes (64
// k), groups of 8 rows 1024 bytes apart.  MN-major: rows of 64 values of
// m (or n), one row a k, groups of 8 k 1024 bytes apart, the next 64 values
// of m one box of 64 k (8192 bytes) further on.
template <bool MN> __device__ __forceinline__ uint64_t make_desc(uint32_t addr) {
    constexpr uint64_t lead = MN ? (8192 >> 4) : 1, stride = 1024 >> 4;
    return (uint64_t)((addr & 0x3FFFF) >> 4) | lead << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
// 16 values of k further on, in units of 16 bytes
template <bool MN> constexpr uint64_t kKStep = MN ? (2048 >> 4) : (32 >> 4);

__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// Arrive on this barrier of both CTAs once all products issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: lane l gets row l.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
// Waits for the loads; ties the registers to it so that none is read before.
__device__ __forceinline__ void tmem_wait(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) asm volatile("" : "+f"(v[i]));
}

// Two f32 operations at a time.
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_out(F2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// kind::f16: sums in f32; A and B bf16 (1) or f16 (0); M = 256;
// bit 15 (A's m axis contiguous) and N (from bit 17) are set tile by tile
inline uint32_t make_idesc(bool bf16, bool b_mn) {
    return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10  | (b_mn ? 1u : 0u) << 16 |
           (uint32_t)(256 >> 4) << 24;
}

// A launch may start before the one in front of it has ended (its set-up
// overlaps that one's end); from here on that one's results are there.
__device__ __forceinline__ void depend() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- the frame --------------------------------------------------------------

// One unit of work: C[m0 .. mend) x [n0 .. nend) (256 x 256 at most), the
// stages q0 .. q0 + nkb - 1 of its k axis, which starts at k0 in the maps.
// With two parts of A (batches 0 and 1 of its map: a value's leading and
// trailing bits), the stages take both parts of one block of k in turn.
// tail: rows of k that count in the last stage where the operands go on
// behind the k axis' end (0: the maps end there, TMA fills zeros).
struct Tile {
    int m0, n0, mend, nend;
    // columns multiplied: each CTA brings half of them
    __device__ int cols() const { return nend - n0 > 128 ? 256 : nend - n0 > 64 ? 128 : 64; }
    int k0, q0, nkb;
    int bz;           // B's batch
    int tail;
    int kind;         // which of a launch's two products
    int aux;
};
// Division by a number known on the host: four instructions in place of some
// forty, between two tiles (n, d < 2^31).
struct Div {
    uint32_t d = 1, mul = 0, shift = 0;
    Div() = default;
    Div(uint32_t by) : d(by) {
        // n / d = floor(n (2^(31 + s) / d rounded up) / 2^(31 + s)), s = ceil(log2 d): the rounding adds less than n / 2^(31 + s) <= 1 / d
        while ((1ull << shift) < d) shift++;
        mul = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);
    }
    __device__ uint32_t operator()(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> 31 >> shift); }
};

// The units of cluster c of C: c, 2C - 1 - c, 2C + c, 4C - 1 - c, ... so that of units
// in order of length each cluster gets as many long ones as the others.
struct Snake {
    uint32_t at, up, down;
    __device__ Snake(int c, int n) : at(c), up(2 * (n - 1 - c) + 1), down(2 * c + 1) {}
    __device__ void step() {
        at += up;
        const uint32_t u = up;
        up = down;
        down = u;
    }
};
// The operands' maps: A and B of the first product, A and B of the second.
struct Maps {
    alignas(64) CUtensorMap m[4];
};

// An epilogue that keeps nothing from tile to tile.
struct None {};

// What one epilogue warp knows of its place.
struct Place {
    int sub, half, lane, rank;
    int row;             // row of the tile (0..255) of this lane
    int wide;            // columns of one half
    __device__ int first() const { return half * wide; }
    uint8_t *staging;    // 4096 bytes of this warp's own
    uint32_t swap;       // 4 barriers of the two warps of these rows (left and right columns)
    volatile int *dead;
};

// A place among the stages, and its barriers' parity.
struct Ring {
    static constexpr int N = kStages;
    int s = 0;
    uint32_t ph = 0;
    __device__ void step() {
        if (++s == N) s = 0, ph ^= 1;
    }
    __device__ void skip(int n) {
        const uint32_t to = s + n;
        ph ^= to / N & 1;
        s = to % N;
    }
};

// What one CTA of the pair fetches of a tile: boxes of 64 values of k x 128
// rows, or where the m (n) axis is contiguous 64 of its values x 64 of k.  The
// second CTA may have none of either operand (up to 128 rows and 32 columns).
// It arrives on the leading CTA's barrier of every stage all the same: without
// that the leading one could run a lap of the ring ahead, and the second one's
// wait by parity would take the lap after for the one that it is in.  So no
// stage is full before both have come to it.
struct Boxes {
    int am, bn, a, b;      // first row of A and B, boxes of each
    __device__ static int count(bool mn, int from, int end) { return end <= from ? 0 : mn && end - from > 64 ? 2 : 1; }
    __device__ Boxes(const Tile &t, bool amn, bool bmn, int rank) {
        const int half = t.cols() / 2;
        am = t.m0 + rank * 128;
        bn = t.n0 + rank * half;
        a = count(amn, am, min(t.mend, am + 128));
        b = count(bmn, bn, min(t.nend, bn + half));
    }
    __device__ uint32_t bytes(bool amn, bool bmn) const { return a * (amn ? 8192 : kABytes) + b * (bmn ? 8192 : kABytes); }
};

// One stage of both operands into shared memory at `a`, counted on the
// leading CTA's barrier (PAIR) or this one's.
template <class Op, bool AMN, bool PAIR>
__device__ __forceinline__ void load_stage(const CUtensorMap *maps, uint32_t a, uint32_t bar, const Boxes &x, int at, int az, int bz) {
    auto load = [&](uint32_t dst, const CUtensorMap *m, int x, int y, int z) {
        if (PAIR)
            tma_pair(dst, m, bar, x, y, z);
        else
            tma_own(dst, m, bar, x, y, z);
    };
    const uint32_t b = a + kABytes;
    if (AMN) {
        if (x.a > 0) load(a, maps, x.am, at, az);
        if (x.a > 1) load(a + 8192, maps, x.am + 64, at, az);
    } else if (x.a) {
        load(a, maps, at, x.am, az);
    }
    if (Op::kBMN) {
        if (x.b > 0) load(b, maps + 1, x.bn, at, bz);
        if (x.b > 1) load(b + 8192, maps + 1, x.bn + 64, at, bz);
    } else if (x.b) {
        load(b, maps + 1, at, x.bn, bz);
    }
}

template <class Op, bool AMN>
__device__ __forceinline__ bool fetch(const Op &op, const CUtensorMap *maps, const Tile &t, int n, Ring r, uint32_t stages, uint32_t full, uint32_t empty,
                                      uint32_t rank, volatile int *dead) {
    const Boxes mine(t, AMN, Op::kBMN, (int)rank), other(t, AMN, Op::kBMN, (int)rank ^ 1);
    const uint32_t bytes = mine.bytes(AMN, Op::kBMN) + other.bytes(AMN, Op::kBMN);
    const bool two = op.laps == 2;
    for (int q = t.q0; q < t.q0 + n; q++) {
        if (!mbar_wait(empty + 8 * r.s, r.ph ^ 1, dead)) return false;
        const uint32_t bar = full + 8 * r.s;
        if (rank == 0)
            mbar_expect(bar, bytes);
        else
            mbar_arrive_at<false>(bar, 0);
        load_stage<Op, AMN, true>(maps, stages + r.s * kStageBytes, bar, mine, t.k0 + (two ? q >> 1 : q) * kBK, two ? q & 1 : 0, t.bz);
        r.step();
    }
    return true;
}

template <class Op, bool AMN> __device__ __forceinline__ void multiply_stage(uint32_t d, uint32_t a, uint32_t idesc, bool add) {
    uint64_t da = make_desc<AMN>(a), db = make_desc<Op::kBMN>(a + kABytes);
#pragma unroll
    for (int j = 0; j < kBK / 16; j++) {
        mma_pair(d, da, db, idesc | (uint32_t)AMN << 15, add || j > 0);
        da += kKStep<AMN>;
        db += kKStep<Op::kBMN>;
    }
}

template <class Op, bool AMN>
__device__ __forceinline__ bool multiply(uint32_t d, int n, Ring &r, uint32_t stages, uint32_t full, uint32_t empty, uint32_t idesc, volatile int *dead) {
    for (int k = 0; k < n; k++) {
        if (!mbar_wait(full + 8 * r.s, r.ph, dead)) return false;
        fence_after();
        multiply_stage<Op, AMN>(d, stages + r.s * kStageBytes, idesc, k > 0);
        commit_pair(empty + 8 * r.s);
        r.step();
    }
    return true;
}

template <class Op>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_tc(const __grid_constant__ Maps maps, const __grid_constant__ Op op, const uint32_t idesc) {
    constexpr int kCols = 2 * kBN;      // of tensor memory
    extern __shared__ uint8_t raw[];
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint8_t *staging = base + kStages * kStageBytes;
    uint64_t *bars = (uint64_t *)(staging + kStaging);
    const uint32_t stages = smem_u32(base);
    const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16,
                   fixed = tempty + 16, tailbar = fixed + 8 * kStages;
    const uint32_t swap = tailbar + 8 * kStages, told = swap + 8 * 16, heard = told + 8 * kTold;
    int4 *tiles = (int4 *)(bars + 4 * kStages + 20 + 2 * kTold);     // told: stages, columns, tail, kind
    static_assert((4 * kStages + 20 + 2 * kTold) % 2 == 0, "");
    uint32_t *tmem_slot = (uint32_t *)(tiles + kTold);
    volatile int *dead = (volatile int *)(tmem_slot + 1);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_rank();
    const int cid = blockIdx.x / 2, ncl = gridDim.x / 2;

    if (warp == 0) {
        // a lane a barrier: one lane for all took 400 clocks
        if (lane < (Op::kDual ? 4 : 2)) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.m[lane]) : "memory");
        if (lane < kStages) {
            mbar_init(full + 8 * lane, 2);      // both CTAs' fetching threads
            mbar_init(empty + 8 * lane, 1);
            // one a stage: a CTA ahead of the other by a whole short tile must not count for both
            mbar_init(fixed + 8 * lane, 2);
            mbar_init(tailbar + 8 * lane, 1);
        }
        if (lane < 2) {
            mbar_init(tfull + 8 * lane, 1);
            mbar_init(tempty + 8 * lane, 2 * kEpiWarps);
        }
        if (lane < 16) mbar_init(swap + 8 * lane, 1);
        if (lane < 2 * kTold) mbar_init(told + 8 * lane, 1);
        // whether a launch before this one has run out; the one directly in front may not have ended yet
        if (lane == 0) *dead = *(volatile int *)&g_ops_timeout;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_sync();     // both CTAs run, their barriers stand
    const bool none = load_at(smem_u32((const void *)dead), 0) | load_at(smem_u32((const void *)dead), 1);
    depend();
    if (none) {
        cluster_sync();
        return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        fence_before();
    }
    // both have their tensor memory; the fetching warp, which does not touch it, goes ahead
    cluster_arrive();
    uint32_t tmem = 0;
    if (warp) {
        cluster_wait();
        fence_after();
        tmem = *(volatile uint32_t *)tmem_slot;
    }

    if (warp == 0) {
        // ---- fetch: one thread runs a tile's stages (a stage has 512 clocks)
        Ring r;
        typename Op::Iter it(op, cid, ncl);
        Tile t;
        while (it.next(op, t)) {
            __syncwarp();
            if (elect_one()) {
                const bool tail = Op::kTail && t.tail && t.nkb;
                const int n = t.nkb - tail;
                bool ok = Op::kDual && t.kind == 1 ? fetch<Op, true>(op, maps.m + 2, t, n, r, stages, full, empty, rank, dead)
                                                   : fetch<Op, Op::kAMN>(op, maps.m, t, n, r, stages, full, empty, rank, dead);
                if (ok && tail) {
                    // the last stage's bytes count for warp 10, not for the products
                    Ring q = r;
                    q.skip(n);
                    ok = mbar_wait(empty + 8 * q.s, q.ph ^ 1, dead);
                    if (ok) {
                        const Boxes mine(t, true, Op::kBMN, (int)rank);
                        mbar_expect(tailbar + 8 * q.s, mine.bytes(true, Op::kBMN));
                        mbar_arrive_at<false>(full + 8 * q.s, 0);
                        load_stage<Op, true, false>(Op::kDual ? maps.m + 2 : maps.m, stages + q.s * kStageBytes, tailbar + 8 * q.s, mine,
                                                    t.k0 + (t.q0 + n) * kBK, 0, t.bz);
                    }
                }
            }
            if (__any_sync(~0u, *dead)) break;
            r.skip(t.nkb);
        }
        // every product's end has reached this CTA's barriers before it leaves
        for (int i = 0; i < kStages && mbar_wait_warp(empty + 8 * r.s, r.ph ^ 1, dead); i++) r.step();
        cluster_wait();
    } else if (warp == 1) {
        // ---- products, issued by one thread too
        if (rank == 0 && elect_one()) {
            Ring r;
            uint32_t fixed_ph = 0;
            for (int n = 0;; n++) {
                const int buf = n & 1, slot = n % kTold;
                if (!mbar_wait(told + 8 * slot, n / kTold & 1, dead)) break;
                const int4 t = tiles[slot];
                mbar_arrive(heard + 8 * slot);
                if (t.x < 0) break;
                const bool tail = Op::kTail && t.z, second = Op::kDual && t.w;
                if (!mbar_wait(tempty + 8 * buf, ((n >> 1) & 1) ^ 1, dead)) break;
                fence_after();
                const uint32_t d = tmem + buf * kBN, id = idesc | (uint32_t)(t.y >> 3) << 17;
                if (!(second ? multiply<Op, true>(d, t.x - tail, r, stages, full, empty, id, dead)
                             : multiply<Op, Op::kAMN>(d, t.x - tail, r, stages, full, empty, id, dead)))
                    break;
                if (tail) {
                    if (!mbar_wait(full + 8 * r.s, r.ph, dead) || !mbar_wait<true>(fixed + 8 * r.s, fixed_ph >> r.s & 1, dead)) break;
                    fence_after();
                    multiply_stage<Op, true>(d, stages + r.s * kStageBytes, id, t.x > 1);
                    commit_pair(empty + 8 * r.s);
                    fixed_ph ^= 1u << r.s;
                    r.step();
                }
                commit_pair(tfull + 8 * buf);
            }
        }
    } else if (warp == 2 + kEpiWarps) {
        // ---- tells the products' thread of the next tile, then sees to the
        // current one's last stage where its k axis ends inside it: rows
        // behind the end belong to the next leaf; zeros take their place
        // before the products see them
        Ring r;
        uint32_t ph = 0;
        typename Op::Iter it(op, cid, ncl);
        Tile t, next{};
        int n = 0, longest = 0;     // stages of the longest tile so far: this warp is up to kTold tiles ahead of the products
        auto tell = [&](bool more) {
            longest = max(longest, next.nkb);
            if (rank) return true;
            const int slot = n % kTold;
            if (!mbar_wait_warp(heard + 8 * slot, (n / kTold & 1) ^ 1, dead, wait_clocks(longest))) return false;
            if (lane == 0) {
                tiles[slot] = make_int4(more ? next.nkb : -1, next.cols(), next.tail && next.nkb, next.kind);
                mbar_arrive(told + 8 * slot);
            }
            __syncwarp();
            n++;
            return true;
        };
        bool more = it.next(op, next);
        if (tell(more))
            while (more) {
                t = next;
                more = it.next(op, next);
                if (!tell(more)) break;
                if (!Op::kTail) continue;
                r.skip(t.nkb);
                if (!t.tail || !t.nkb) continue;
                const int s = r.s == 0 ? kStages - 1 : r.s - 1;
                if (!mbar_wait_warp(tailbar + 8 * s, ph >> s & 1, dead, wait_clocks((kTold + 1ll) * longest))) break;
                ph ^= 1u << s;
                uint8_t *st = base + s * kStageBytes;
                for (int box = 0; box < kStageBytes / 8192; box++)
                    for (int i = t.tail * 8 + lane; i < 64 * 8; i += 32) *(uint4 *)(st + box * 8192 + i * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_at<true>(fixed + 8 * s, 0);
            }
    } else {
        // ---- epilogue
        Place p;
        p.sub = warp % 4;
        p.half = (warp - 2) / 4;
        p.lane = lane;
        p.rank = (int)rank;
        p.row = (int)rank * 128 + p.sub * 32 + lane;
        p.staging = staging + (warp - 2) * 4096;
        p.swap = swap + 32 * p.sub;
        p.dead = dead;
        typename Op::State state{};
        // what no tile writes, while the first loads are on their way
        op.rest(state, (warp - 2) + kEpiWarps * (int)blockIdx.x, kEpiWarps * (int)gridDim.x, lane);
        int n = 0;
        typename Op::Iter it(op, cid, ncl);
        Tile t;
        while (it.next(op, t)) {
            const int buf = n & 1;
            const auto rows = op.rows(t, p);     // the rows' scalars, on their way while the products run
            if (!mbar_wait_warp(tfull + 8 * buf, (n >> 1) & 1, dead, wait_clocks(t.nkb))) break;
            n++;
            fence_after();
            p.wide = t.cols() / 2;
            op.epilogue(t, p, rows, state, tmem + buf * kBN + ((uint32_t)(p.sub * 32) << 16) + p.half * p.wide, [&] {
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at<false>(tempty + 8 * buf, 0);
            });
        }
    }
    __syncwarp();
    if (*dead)
        for (int i = 0; i < 1000; i++) __nanosleep(1000);    // copies in flight land meanwhile
    cluster_sync();     // nobody reads tensor memory any more
    fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
    cluster_sync();     // both have freed theirs
}

// A wait that nothing ends, for the test of what a wait that runs out does.
__global__ void k_wait(long long clocks) {
    depend();
    __shared__ uint64_t bar;
    __shared__ int dead;
    if (threadIdx.x == 0) {
        dead = 0;
        mbar_init(smem_u32(&bar), 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) mbar_wait(smem_u32(&bar), 0, &dead, clocks);
}

// ---- epilogues --------------------------------------------------------------

template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}

template <class T> __device__ __forceinline__ float unpack(uint32_t bits);
template <> __device__ __forceinline__ float unpack<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <> __device__ __forceinline__ float unpack<__half>(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }

// Elements of one store that rows at `p`, `ld` apart, allow: 8, 4, 2 or 1.
__host__ __device__ inline int store_width(const void *p, int64_t ld) {
    const uint64_t a = (uint64_t)(uintptr_t)p | (uint64_t)ld * 2;
    return a & 15 ? a & 7 ? a & 3 ? 1 : 2 : 4 : 8;
}

// Rows of 64 columns in a warp's staging memory (16-byte piece i of row r at
// piece i ^ (r % 8)) to out[r * ld + c] for r < rows, c < cols, W elements a
// lane: 64 / W lanes have one row, so that a store of the warp covers runs of
// a row whatever W is (with 8 elements a lane stored one by one, rows of odd
// length took 32 places a store).
template <int W, class V, class T>
__device__ __forceinline__ void store_rows(const uint8_t *staging, int lane, T *out, int64_t ld, int rows, int cols) {
    constexpr int kLanes = 64 / W;      // of a row
#pragma unroll 4
    for (int i = lane; i < 32 * kLanes; i += 32) {
        const int r = i / kLanes, c = i % kLanes * W;
        if (r >= rows || c >= cols) continue;
        const uint8_t *from = staging + r * 128 + ((c / 8 ^ (r & 7)) * 16) + c % 8 * 2;
        T *to = out + (int64_t)r * ld + c;
        if (c + W <= cols) {
            *(V *)to = *(const V *)from;
        } else {
#pragma unroll
            for (int k = 0; k < W - 1; k++)
                if (c + k < cols) ((uint16_t *)to)[k] = ((const uint16_t *)from)[k];
        }
    }
}

// The same sums in two parts: rounded to T at out, and what the rounding left,
// rounded too, at out + part; 32 columns of each at a time.  Rows start on
// 16-byte boundaries.
template <class T, class F, class R>
__device__ __forceinline__ void store_parts(const Place &p, uint32_t addr, T *out, int64_t part, int64_t ld, int rows, int cols, F f, R release) {
    if (rows <= 0) {
        release();
        return;
    }
#pragma unroll 1
    for (int c = 0; c < p.wide; c += 32) {
        __syncwarp();
        float v[32];
        tmem_ld32(addr + c, v);
        tmem_wait(v);
        if (c + 32 >= p.wide) release();
        f(v, c);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float x = v[8 * i + 2 * k], y = v[8 * i + 2 * k + 1];
                a[k] = pack2<T>(x, y);
                b[k] = pack2<T>(x - unpack<T>(a[k] & 0xFFFF), y - unpack<T>(a[k] >> 16));
            }
            *(uint4 *)(p.staging + p.lane * 128 + ((i ^ (p.lane & 7)) * 16)) = make_uint4(a[0], a[1], a[2], a[3]);
            *(uint4 *)(p.staging + p.lane * 128 + (((i + 4) ^ (p.lane & 7)) * 16)) = make_uint4(b[0], b[1], b[2], b[3]);
        }
        __syncwarp();
        const int lim = min(cols, p.wide) - c;
        if (lim <= 0) continue;
#pragma unroll 4
        for (int i = p.lane; i < 32 * 8; i += 32) {
            const int r = i / 8, ch = i % 8, col = ch % 4 * 8;
            if (r >= rows || col >= lim) continue;
            const uint4 q = *(const uint4 *)(p.staging + r * 128 + ((ch ^ (r & 7)) * 16));
            T *to = out + (ch / 4) * part + (int64_t)r * ld + c + col;
            if (col + 8 <= lim) {
                *(uint4 *)to = q;
            } else {
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int k = 0; k < 7; k++)
                    if (col + k < lim) ((uint16_t *)to)[k] = (uint16_t)(w[k / 2] >> (k & 1) * 16);
            }
        }
    }
}

// The sums of this warp's 32 rows, p.wide columns from `addr` on, through f(v,
// col) (32 columns at a time, col from the half's first), rounded to T and
// stored at out[r * ld + c] for r < rows, c < cols: 64 columns at a time pass
// through the warp's staging memory, so that eight lanes store one row's 128
// bytes.  width: store_width of the rows.  empty: no products, the sums are
// 0.  release() hands the tensor memory back once it is read.
template <class T, class F, class R>
__device__ __forceinline__ void store_tile(const Place &p, uint32_t addr, T *out, int64_t ld, int rows, int cols, int width, bool empty, F f, R release) {
    if (rows <= 0) {
        release();
        return;
    }
#pragma unroll 1
    for (int c = 0; c < p.wide; c += 64) {
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
            if (c + h >= p.wide) break;
            float v[32];
            if (empty) {
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = 0.f;
            } else {
                tmem_ld32(addr + c + h, v);
                tmem_wait(v);
            }
            f(v, c + h);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint4 q;
                q.x = pack2<T>(v[8 * i], v[8 * i + 1]);
                q.y = pack2<T>(v[8 * i + 2], v[8 * i + 3]);
                q.z = pack2<T>(v[8 * i + 4], v[8 * i + 5]);
                q.w = pack2<T>(v[8 * i + 6], v[8 * i + 7]);
                *(uint4 *)(p.staging + p.lane * 128 + (((h / 8 + i) ^ (p.lane & 7)) * 16)) = q;
            }
        }
        if (c + 64 >= p.wide) release();
        __syncwarp();
        const int lim = min(cols, p.wide) - c;
        if (lim <= 0) continue;
        if (width == 8)
            store_rows<8, uint4>(p.staging, p.lane, out + c, ld, rows, lim);
        else if (width == 4)
            store_rows<4, uint2>(p.staging, p.lane, out + c, ld, rows, lim);
        else if (width == 2)
            store_rows<2, uint32_t>(p.staging, p.lane, out + c, ld, rows, lim);
        else
            store_rows<1, uint16_t>(p.staging, p.lane, out + c, ld, rows, lim);
    }
}

}  // namespace tc
