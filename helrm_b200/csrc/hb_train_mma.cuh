// hb_train_mma.cuh -- the training operators' matrix product on the
// 5th-generation tensor cores.  Included by hb_train.cu after hb_train.cuh.
//
// D[m][n] = sum_k A(m, k) B(n, k) over tiles of 256 x 256, one tile at a time
// on a pair of SMs (a cluster of two, tcgen05 cta_group::2).  Each SM holds
// half of A's rows and half of B's rows of a 64-deep slice in shared memory:
// 32 KB a slice and SM, which halves the shared-memory traffic a 128 x 256
// tile on one SM would have (96 B a clock written and 96 read, where an SM
// moves 128).  Six slices are in flight, and two accumulators of 256 columns
// fill the tensor memory, so that a tile's epilogue runs under the next
// tile's products.  The grid is persistent: a cluster for every SM pair.
//
// Operands come by TMA with the 128-byte swizzle and may lie either way: rows
// along k ("K-major") or rows along m / n ("MN-major"), so that the gradients
// read dG, dU, Z, X, H and the weights as they are stored.  Rows, columns and
// depth past the end are filled with zeros by the TMA unit.
//
// Warps: 0 TMA, 1 MMA issue (first SM of the pair), 2 tensor memory, 4 on
// epilogue: quadrant warp & 3 of the accumulator's rows, and the columns shared
// out among the warps of a quadrant.
//
// What bounds it: long products the tensor pipe at the clock the power cap
// leaves (gated forward of 8192 x 4096 x 4096 in 341 us, 1.61 PFLOP/s at 1.54
// GHz, the pipe active 90 % of the time; its dX 348 us, its weights' gradients
// 365).  Short ones what does not follow the depth: dG and dU of 4096 x K x 4096
// take 107, 169 and 294 thousand clocks at K = 1024, 2048 and 4096 with GELU, 91,
// 154 and 279 with the identity, so 62 for each 1024 of depth (558 a slice, of
// which the tensor pipe needs 512) and beside that 44 or 29, some 6 or 4 thousand
// a tile and SM pair with launch and tail, that no products hide.  Products of a
// few features their epilogue (the loss's exponentials: 72 % of the
// special-function pipe at 16 features).
//
// Every wait is bounded: when one runs out, the block stops taking work,
// waits for what it has in flight, frees its tensor memory and leaves a word
// in host memory that the next training call on the device reports.
#pragma once
#include <cuda.h>

#include "hb_ptx.cuh"
#include "hb_schedule.hpp"

namespace hb {
namespace train {

constexpr int kRows = 256;     // rows of a tile, 128 on each SM
constexpr int kCols = 256;     // accumulator columns of a tile
constexpr int kDepth = 64;     // slice of k: 128 bytes
constexpr int kStages = 6;
constexpr int kOperand = 128 * kDepth * 2;  // bytes of an operand's slice on one SM
constexpr int kStageOut = 32768;  // staging bytes of the epilogue warps together
constexpr int kBarriers = 2 * kStages + 5;
constexpr int kProductSmem = 2 * kStages * kOperand + kStageOut + 8 * kBarriers + 16;
// Epilogue warps.  The loss's exponentials keep 16 busy (8 warps left the
// special-function pipe at 52% of its rate, the warps waiting for their own
// results); the others need the registers of 8.
__host__ __device__ constexpr int epi_warps(int epi) { return epi == EPI_LSE || epi == EPI_Z ? 16 : 8; }
__host__ __device__ constexpr int product_threads(int epi) { return 128 + 32 * epi_warps(epi); }
// The tensor cores cut a running sum towards zero at every 16-deep step, by half
// a unit in its last place on average: a row's largest logit comes out 0.5e-6 of
// itself short at 512 features, 1.0e-6 at 1024 and would 3.9e-6 at 4096, always
// to the same side.  So a loss over more than kChunk slices (1024 features)
// accumulates that many at a time and adds the parts, rounded to nearest, in its
// epilogue's registers (EPI_LSE_LONG, and EPI_Z_LONG, whose logits have to be the
// forward pass's): what is lost stays at the second figure for any depth, the
// loss within 3.5e-7 of itself (8192 x 4096 x 131072: 1.5e-6 in one sum).
// Reading an accumulator holds the tensor pipe up by some 500 clocks: forward of
// 4096 x 4096 x 18944 579,000 clocks in one sum, 653,000 in parts of 512 features
// (loss within 1.6e-7), half of that difference in parts of 1024.
constexpr int kChunk = 16;
constexpr unsigned long long kWaitNs = 4000000000ull;

enum { K_MAJOR = 0, MN_MAJOR = 1 };

// One product.  A launch of gradients (EPI_OUT) may hold two, which the clusters
// share: those by the input and by the weights have nothing to do with each
// other, and fill the SM pairs' rounds together.  A kernel of its own for that
// (JOBS): what is fixed at compile time for one product costs a long one 7 %.
struct Job {
    CUtensorMap a, a1, b, b1;
    int64_t M, N;
    int tiles_m, tiles_n;  // of one output
    int cols;              // accumulator columns of a tile: 256, or 128 for a narrow output (EPI_OUT)
    int outputs;           // 2: a second product A1 B^T into o1
    int splits;            // the depth in this many parts, each with a partial sum of its own
    int kb, kb1;           // slices of (A, B), and after them of (A1, B1)
    int amaj;              // two jobs: how A lies (B is MN-major)
    const LossPlan *plan;  // not NULL: the rows that take part, known on the device only, are
    int plan_k;            // 0: the rows of the tiles, 1: the depth
    EpiArgs e;
};
template <int JOBS>
struct ProductArgs {
    Job job[JOBS];
    int *error;            // host memory
};

// Bounded wait for a barrier's phase, as tc::mbar_wait, except that a wait of
// ordinary length reads no clock.
__device__ __forceinline__ bool mbar_wait(unsigned a, unsigned parity, volatile int *abort, int *err, int code) {
    if (tc::mbar_try(a, parity)) return true;
    unsigned long long t0 = 0;
    for (unsigned it = 1;; it++) {
        if (tc::mbar_try(a, parity)) return true;
        if (abort && *abort) return false;
        if ((it & 255) == 0) {
            const unsigned long long t = tc::gtimer();
            if (t0 == 0) t0 = t;
            if (t - t0 > kWaitNs) {
                if (abort) *abort = 1;
                atomicOr(err, code);
                return false;
            }
        }
    }
}

namespace ptx {
__device__ __forceinline__ unsigned rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// the address of the pair's first SM for a shared-memory address of this one
__device__ __forceinline__ unsigned of_first(unsigned a) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
    return r;
}
// The accumulator's reads are ordered by the tcgen05 fences; a release at
// cluster scope would wait for this thread's stores to global memory too.
__device__ __forceinline__ void arrive_cluster(unsigned a) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
}
__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Shared-memory matrix descriptor with the 128-byte swizzle.  K-major: rows of
// 128 bytes, groups of 8 rows 1024 bytes apart.  MN-major: panels of 64
// elements (128 bytes) `panel` bytes apart, groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t descriptor(unsigned addr, unsigned panel = 8192) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// arrives on both SMs' barrier once the MMAs issued so far are done
__device__ __forceinline__ void commit_both(unsigned bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((unsigned short)3)
        : "memory");
}
__device__ __forceinline__ void commit_own(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 columns of this warp's 32 accumulator rows
__device__ __forceinline__ void load32(unsigned addr, float (&v)[32]) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Waits for this warp's loads.  The registers pass through, so that nothing
// that reads them can be moved before the wait.
__device__ __forceinline__ void wait32(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                   "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                   "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                   "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void load16(unsigned addr, float (&v)[16]) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void wait16(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                   "+f"(v[15])
                 :
                 : "memory");
}
}  // namespace ptx

// A warp's 32 x 32 block of 16-bit values between registers (a row a lane) and
// global memory, turned in shared memory so that a row's 64 bytes move
// together.  Rows from M and columns from N on are left out.
__device__ __forceinline__ unsigned block_at(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }
template <class T>
__device__ __forceinline__ void store_block(unsigned char *st, const unsigned (&v)[16], T *out, int64_t ld, int64_t m0,
                                            int64_t M, int64_t n0, int64_t N, bool vec, int lane) {
#pragma unroll
    for (int j = 0; j < 4; j++)
        *reinterpret_cast<uint4 *>(st + block_at(lane, j)) =
            make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    __syncwarp();
    unsigned short *o = reinterpret_cast<unsigned short *>(out) + m0 * ld + n0;
    if (vec && m0 + 32 <= M && n0 + 32 <= N) {
        o += (lane >> 2) * ld + (lane & 3) * 8;
        const unsigned char *from = st + block_at(lane >> 2, lane & 3);
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(o + i * 8 * ld) = *reinterpret_cast<const uint4 *>(from + i * 512);
    } else if (ld % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0 && n0 + 32 <= N) {
        // rows on 8-byte boundaries: four of them at a time
        const int rows = M - m0 < 32 ? (int)(M - m0) : 32;
#pragma unroll 4
        for (int r = lane >> 3; r < rows; r += 4)
            *reinterpret_cast<uint2 *>(o + r * ld + (lane & 7) * 4) =
                *reinterpret_cast<const uint2 *>(st + block_at(r, (lane & 7) >> 1) + (lane & 1) * 8);
    } else if (n0 + lane < N) {
        const int rows = M - m0 < 32 ? (int)(M - m0) : 32;
#pragma unroll 4
        for (int r = 0; r < rows; r++)
            o[r * ld + lane] = *reinterpret_cast<const unsigned short *>(st + block_at(r, lane >> 3) + (lane & 7) * 2);
    }
    __syncwarp();
}
template <class T>
__device__ __forceinline__ void load_block(unsigned char *st, unsigned (&v)[16], const T *in, int64_t ld, int64_t m0,
                                           int64_t M, int64_t n0, int64_t N, bool vec, int lane) {
    const unsigned short *p = reinterpret_cast<const unsigned short *>(in) + m0 * ld + n0;
    if (vec && m0 + 32 <= M && n0 + 32 <= N) {
        p += (lane >> 2) * ld + (lane & 3) * 8;
        unsigned char *to = st + block_at(lane >> 2, lane & 3);
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(to + i * 512) = *reinterpret_cast<const uint4 *>(p + i * 8 * ld);
    } else if (ld % 4 == 0 && (reinterpret_cast<uintptr_t>(in) & 7) == 0 && n0 + 32 <= N) {
        const int rows = M - m0 < 32 ? (int)(M - m0) : 32;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = i * 4 + (lane >> 3);
            *reinterpret_cast<uint2 *>(st + block_at(r, (lane & 7) >> 1) + (lane & 1) * 8) =
                r < rows ? *reinterpret_cast<const uint2 *>(p + r * ld + (lane & 7) * 4) : make_uint2(0, 0);
        }
    } else {
#pragma unroll 16
        for (int r = 0; r < 32; r++)
            *reinterpret_cast<unsigned short *>(st + block_at(r, lane >> 3) + (lane & 7) * 2) =
                m0 + r < M && n0 + lane < N ? p[r * ld + lane] : (unsigned short)0;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint4 w = *reinterpret_cast<const uint4 *>(st + block_at(lane, j));
        v[4 * j] = w.x, v[4 * j + 1] = w.y, v[4 * j + 2] = w.z, v[4 * j + 3] = w.w;
    }
    __syncwarp();
}
// The same for 32-bit sums, whose rows are padded to whole vectors.
__device__ __forceinline__ void store_sums(unsigned char *st, const float (&v)[32], float *out, int64_t ld, int64_t m0,
                                           int64_t M, int64_t n0, bool add, int lane) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        *reinterpret_cast<float4 *>(st + lane * 128 + ((j ^ (lane & 7)) << 4)) =
            make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = i * 4 + (lane >> 3), c = lane & 7;
        float4 w = *reinterpret_cast<const float4 *>(st + r * 128 + ((c ^ (r & 7)) << 4));
        const int64_t m = m0 + r, n = n0 + c * 4;
        if (m < M && n < ld) {
            float4 *p = reinterpret_cast<float4 *>(out + m * ld + n);
            if (add) {
                const float4 o = *p;
                w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
            }
            *p = w;
        }
    }
    __syncwarp();
}

template <class T, int AMAJ, int BMAJ, int EPI, int ACT, int JOBS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(product_threads(EPI), 1)
    k_mma_product(const __grid_constant__ ProductArgs<JOBS> p) {
    constexpr bool kDual = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
    constexpr int kWarps = epi_warps(EPI), kSets = kWarps / 8;
    constexpr bool kLse = EPI == EPI_LSE || EPI == EPI_LSE_LONG, kZ = EPI == EPI_Z || EPI == EPI_Z_LONG;
    constexpr bool kLong = EPI == EPI_LSE_LONG || EPI == EPI_Z_LONG, kScaled = EPI == EPI_GATED_BWD && std::is_same<T, __half>::value;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *stage = smem + 2 * kStages * kOperand;
    uint64_t *bars = reinterpret_cast<uint64_t *>(stage + kStageOut);
    const unsigned sA = tc::smem_u32(smem), sB = sA + kStages * kOperand;
    const unsigned full = tc::smem_u32(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages,
                   tempty = tfull + 16, drain = tempty + 16;
    unsigned *s_tmem = reinterpret_cast<unsigned *>(bars + kBarriers);
    int *s_error = reinterpret_cast<int *>(s_tmem + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = ptx::rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) {
            tc::mbar_init(full + 8 * i, 1);
            tc::mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            tc::mbar_init(tfull + 8 * i, 1);
            tc::mbar_init(tempty + 8 * i, 16);  // 8 warps of both SMs
        }
        tc::mbar_init(drain, 1);
        *s_error = 0;
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0 && lane < 4) {
        const Job &j = p.job[0];
        const CUtensorMap *map = lane == 0 ? &j.a : lane == 1 ? &j.b : lane == 2 ? &j.a1 : &j.b1;
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(s_tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc::fence_before();
    __syncthreads();
    ptx::cluster_sync();
    tc::fence_after();
    const unsigned tmem = *s_tmem;
    after_previous();

    constexpr bool kOut = EPI == EPI_OUT, kTwo = JOBS == 2;
    // A job's shape, with the rows that take part.
    struct Shape {
        unsigned tiles_m, tiles, items;
        int kb, depth;
        int64_t M;
    };
    auto shape = [&](const Job &j) {
        Shape h;
        h.tiles_m = j.tiles_m, h.kb = j.kb, h.M = j.M;
        if (j.plan) {
            const int n = j.plan->filled;
            if (j.plan_k)
                h.kb = n / kDepth;
            else
                h.tiles_m = n / kRows, h.M = n;
        }
        h.tiles = h.tiles_m * j.tiles_n;
        h.items = h.tiles * j.splits * j.outputs;
        h.depth = h.kb + j.kb1;
        return h;
    };
    const Shape s0 = shape(p.job[0]);
    Shape s1 = {};
    if (kTwo) s1 = shape(p.job[JOBS - 1]);
    const unsigned cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    auto nth = [&](unsigned k) -> unsigned {
        if (!kTwo) return nth_of_one(k, cluster, clusters, s0.items);
        return nth_of_two(k, cluster, clusters, s0.items, s0.depth / p.job[0].splits + 2, s1.items,
                          s1.depth / p.job[JOBS - 1].splits + 2);
    };
    struct Item {
        int job, out, split, mt, nt, k0, k1;
    };
    auto item = [&](unsigned i) {
        Item t;
        t.job = kTwo && i >= s0.items;
        if (t.job) i -= s0.items;
        const Shape &h = kTwo && t.job ? s1 : s0;
        const Job &j = p.job[kTwo ? t.job : 0];
        t.out = t.split = t.k0 = 0;
        t.k1 = h.depth;
        if (h.items > h.tiles) {
            unsigned q = i / h.tiles;
            i -= q * h.tiles;
            t.out = q / j.splits;
            t.split = q - t.out * j.splits;
            part_of(h.depth, t.split, j.splits, t.k0, t.k1);
        }
        tile_at(i, h.tiles_m, j.tiles_n, t.mt, t.nt);
        return t;
    };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA
        if (lane == 0) {
            int s = 0;
            unsigned ph = 0;
            int64_t loads = 0;
            bool ok = true;
            for (unsigned q = 0, i; ok && (i = nth(q)) != kNoItem; q++) {
                const Item t = item(i);
                const Job &j = p.job[kTwo ? t.job : 0];
                const int cols = kOut ? j.cols : kCols, kb = kTwo && t.job ? s1.kb : s0.kb;
                const bool mn_a = kTwo ? j.amaj == MN_MAJOR : AMAJ == MN_MAJOR;
                const int m = t.mt * kRows + 128 * (int)rank;
                const int n = kDual ? t.nt * 128 : t.nt * cols + cols / 2 * (int)rank;
                for (int k = t.k0; k < t.k1; k++) {
                    if (!mbar_wait(empty + 8 * s, ph ^ 1, s_abort, s_error, 1)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) tc::mbar_arrive_tx(full + 8 * s, 2 * kOperand + 256 * cols / 2);
                    const unsigned bar = ptx::of_first(full + 8 * s);
                    const bool second = k >= kb;
                    const int x = (second ? k - kb : k) * kDepth;
                    const CUtensorMap *ma = second || t.out ? &j.a1 : &j.a;
                    const CUtensorMap *mb = second || (kDual && rank) ? &j.b1 : &j.b;
                    const unsigned da = sA + s * kOperand, db = sB + s * kOperand;
                    if (!mn_a) {
                        ptx::tma_load(da, ma, x, m, bar);
                    } else {
                        ptx::tma_load(da, ma, m, x, bar);
                        ptx::tma_load(da + kOperand / 2, ma, m + 64, x, bar);
                    }
                    if (BMAJ == K_MAJOR) {
                        ptx::tma_load(db, mb, x, n, bar);
                    } else {
                        ptx::tma_load(db, mb, n, x, bar);
                        if (cols > 128) ptx::tma_load(db + kOperand / 2, mb, n + 64, x, bar);
                    }
                    loads++;
                    if (++s == kStages) s = 0, ph ^= 1;
                }
            }
            // this SM stays until the last slices are consumed: their release
            // arrives in its shared memory
            for (int i = 0; ok && i < kStages && i < loads; i++) {
                if (s == 0) ph ^= 1;
                s = s == 0 ? kStages - 1 : s - 1;
                ok = mbar_wait(empty + 8 * s, ph, s_abort, s_error, 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (rank == 0 && lane == 0) {
            // 32-bit sums of bf16 or fp16, 256 rows over the pair
            constexpr unsigned kType = (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) |
                                       ((unsigned)BMAJ << 16) | ((kRows >> 4) << 24);
            // 16 of k: 32 bytes along a row, or 16 rows of 128 bytes
            constexpr unsigned step_b = BMAJ == K_MAJOR ? 32 : 2048;
            int s = 0;
            unsigned ph = 0;
            unsigned n = 0, use = 0;  // items, and accumulators filled
            bool ok = true;
            for (unsigned i; ok && (i = nth(n)) != kNoItem; n++) {
                const Item t = item(i);
                const Job &job = p.job[kTwo ? t.job : 0];
                const bool mn_a = kTwo ? job.amaj == MN_MAJOR : AMAJ == MN_MAJOR;
                const unsigned idesc = kType | ((unsigned)mn_a << 15) | ((unsigned)((kOut ? job.cols : kCols) >> 3) << 17);
                const unsigned step_a = mn_a ? 2048 : 32;
                int k = t.k0;
                do {  // an accumulator's share of the depth: all of it, but for kLong
                    const int k0 = k, k1 = kLong && k + kChunk < t.k1 ? k + kChunk : t.k1;
                    const int buf = (int)(use & 1);
                    if (!mbar_wait(tempty + 8 * buf, (unsigned)((use >> 1) & 1) ^ 1, s_abort, s_error, 2)) {
                        ok = false;
                        break;
                    }
                    use++;
                    tc::fence_after();
                    const unsigned d = tmem + buf * kCols;
                    for (; k < k1; k++) {
                        if (!mbar_wait(full + 8 * s, ph, s_abort, s_error, 2)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after();
                        const uint64_t da = ptx::descriptor(sA + s * kOperand), db = ptx::descriptor(sB + s * kOperand);
#pragma unroll
                        for (int j = 0; j < kDepth / 16; j++)
                            ptx::mma(d, da + ((j * step_a) >> 4), db + ((j * step_b) >> 4), idesc, k > k0 || j > 0);
                        ptx::commit_both(empty + 8 * s);
                        if (++s == kStages) s = 0, ph ^= 1;
                    }
                    if (ok) ptx::commit_both(tfull + 8 * buf);
                } while (kLong && ok && k < t.k1);
            }
            // after a failure too, no MMA is left in flight
            ptx::commit_own(drain);
            mbar_wait(drain, 0, nullptr, s_error, 8);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ epilogue
        // 8 warps take a tile, half of its columns each; 16 are two sets that take alternate tiles (with a quarter of
        // every tile each, what a tile costs beside its logits counted twice)
        const int quad = warp & 3, half = (warp - 4) >> 2 & 1, set = kSets > 1 ? (warp - 4) >> 3 : 0;
        unsigned char *st = stage + (warp - 4) * (kStageOut / kWarps);
        const unsigned bar_empty = ptx::of_first(tempty);
        unsigned cnt = set, use = 0;  // items; with kLong, accumulators read
        float scale = 1.0f;
        if constexpr (kScaled) {
            const EpiArgs &e = p.job[0].e;
            scale = gated_scale(e.range, e.ranges);
            if (blockIdx.x == 0 && threadIdx.x == 128) *e.made = 1.0f / scale;
        }
        // What the loss needs to know of this lane's row, fetched a tile ahead.
        int64_t next_target = -1;
        LossRow next_row = {0.0f, 0.0f, 0.0f, kNoTarget};
        unsigned following = nth(set);
        Item next = {};
        auto fetch = [&] {
            next = item(following);
            if (!kLse && !kZ) return;
            const EpiArgs &e = p.job[0].e;
            const int64_t M = s0.M;
            const int64_t m = (int64_t)next.mt * kRows + 128 * rank + 32 * quad + lane;
            if (kLse) next_target = m < M ? e.target[m] : -1;
            if (kZ && m < M) *reinterpret_cast<float4 *>(&next_row) = reinterpret_cast<const float4 *>(e.rows)[m];
        };
        if (following != kNoItem) fetch();
        while (following != kNoItem) {
            const Item t = next;
            const int64_t target = next_target;
            const LossRow row = next_row;
            const Job &job = p.job[kTwo ? t.job : 0];
            const EpiArgs &e = job.e;
            const int64_t M = kTwo && t.job ? s1.M : s0.M, N = job.N;
            const int buf_use = (int)cnt;
            cnt += kSets;
            following = nth(cnt);
            if (following != kNoItem) fetch();
            const int buf = buf_use & 1;
            const int64_t m0 = (int64_t)t.mt * kRows + 128 * rank + 32 * quad, m = m0 + lane;
            const unsigned acc = tmem + ((unsigned)(32 * quad) << 16) + buf * kCols;
            auto release = [&](int buf) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) ptx::arrive_cluster(bar_empty + 8 * buf);
            };
            // kLong: this warp's 128 columns summed over the parts of the depth
            auto logits = [&](float (&v)[4][32], const Item &t) {
                for (int k = t.k0; k < t.k1; k += kChunk, use++) {
                    const unsigned b = use & 1, from = tmem + ((unsigned)(32 * quad) << 16) + b * kCols + half * 128;
                    if (!__all_sync(0xffffffffu, mbar_wait(tfull + 8 * b, (use >> 1) & 1, s_abort, s_error, 4))) return false;
                    tc::fence_after();
                    if (k == t.k0) {
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            ptx::load32(from + c * 32, v[c]);
                            ptx::wait32(v[c]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            float x[16];
                            ptx::load16(from + c * 16, x);
                            ptx::wait16(x);
#pragma unroll
                            for (int j = 0; j < 16; j++) v[c / 2][c % 2 * 16 + j] += x[j];
                        }
                    }
                    release(b);
                }
                return true;
            };
            if constexpr (!kLong) {
                if (!__all_sync(0xffffffffu, mbar_wait(tfull + 8 * buf, (unsigned)((buf_use >> 1) & 1), s_abort, s_error,
                                                       4)))
                    break;
                tc::fence_after();
            }
            if constexpr (kDual) {
                const int64_t n0 = (int64_t)t.nt * 128;
                T *o0 = static_cast<T *>(e.o0), *o1 = static_cast<T *>(e.o1);
                const bool vec = e.vec & 1, vdh = e.vec & 2;
#pragma unroll 1
                for (int c = 0; c < 2; c++) {
                    const int col = half * 64 + c * 32;
                    float g[32], u[32];
                    unsigned w[16];
                    ptx::load32(acc + col, g);
                    ptx::load32(acc + 128 + col, u);
                    if constexpr (EPI == EPI_GATED_BWD)
                        load_block<T>(st, w, static_cast<const T *>(e.dh), e.lddh, m0, M, n0 + col, N, vdh, lane);
                    ptx::wait32(g);
                    ptx::wait32(u);
                    if (c == 1) release(buf);
                    if constexpr (EPI == EPI_GATED) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            w[j] = pack2<T>(act_f<ACT>(g[2 * j]) * u[2 * j], act_f<ACT>(g[2 * j + 1]) * u[2 * j + 1]);
                        store_block<T>(st, w, o0, e.ldo, m0, M, n0 + col, N, vec, lane);
                    } else {
                        unsigned wu[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            float2 dh = unpack2<T>(w[j]);
                            if constexpr (kScaled) dh.x *= scale, dh.y *= scale;
                            float a0, d0, a1, d1;
                            act_df<ACT>(g[2 * j], a0, d0);
                            act_df<ACT>(g[2 * j + 1], a1, d1);
                            w[j] = pack2<T>(dh.x * u[2 * j] * d0, dh.y * u[2 * j + 1] * d1);
                            wu[j] = pack2<T>(dh.x * a0, dh.y * a1);
                        }
                        store_block<T>(st, w, o0, e.ldo, m0, M, n0 + col, N, vec, lane);
                        store_block<T>(st, wu, o1, e.ldo, m0, M, n0 + col, N, vec, lane);
                    }
                }
            } else if constexpr (kOut) {
                const int cols = job.cols;
                const bool summed = e.acc != nullptr;
                const int64_t n0 = (int64_t)t.nt * cols;
                const float scale = !summed && e.unscale ? *e.unscale : 1.0f;
                const bool nothing = t.k0 == t.k1;  // a part of a depth that turned out short: no product ran
#pragma unroll 1
                for (int c = 0; c < cols / 64; c++) {
                    const int col = half * (cols / 2) + c * 32;
                    float v[32];
                    ptx::load32(acc + col, v);
                    ptx::wait32(v);
                    if (c == cols / 64 - 1) release(buf);
                    if (n0 + col >= N) continue;
                    if (nothing) {
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = 0.0f;
                    }
                    if (!summed) {
                        unsigned w[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = pack2<T>(v[2 * j] * scale, v[2 * j + 1] * scale);
                        store_block<T>(st, w, static_cast<T *>(t.out ? e.o1 : e.o0), e.ldo, m0, M, n0 + col, N,
                                       e.vec & 1, lane);
                    } else {
                        float *o = e.acc + ((int64_t)t.out * job.splits + t.split) * job.M * e.ldo;
                        store_sums(st, v, o, e.ldo, m0, M, n0 + col, !e.first, lane);
                    }
                }
            } else if constexpr (kLse) {
                constexpr int kWide = kCols / 2;  // columns a warp
                const int64_t n0 = (int64_t)t.nt * kCols + half * kWide;
                // columns of the vocabulary here, and which of them is the row's target: looked at once a tile, since
                // few tiles hold a target or the end
                const int wide = (int)(N - n0 < kWide ? N - n0 : kWide);
                const int tg = target >= n0 && target < n0 + wide ? (int)(target - n0) : -1;
                const bool any = __any_sync(0xffffffffu, tg >= 0);
                float top = -INFINITY, sum = 0.0f;
                auto take = [&](float (&v)[32], int c) {
                    if (wide < kWide) {
                        asm volatile("");  // a branch, not 32 selections in every tile
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (c * 32 + j >= wide) v[j] = -INFINITY;
                    }
                    if (any) {
                        asm volatile("");
                        const int at = tg - c * 32;
                        float x = v[0];
#pragma unroll
                        for (int j = 1; j < 32; j++) x = at == j ? v[j] : x;
                        if (at >= 0 && at < 32) e.at[m] = x;
                    }
                    float m0 = max3(top, v[0], v[1]), m1 = v[2];
#pragma unroll
                    for (int j = 3; j < 31; j += 4) {
                        m0 = max3(m0, v[j], v[j + 1]);
                        m1 = max3(m1, v[j + 2], v[j + 3]);
                    }
                    const float mx = max3(m0, m1, v[31]);
                    // a row of minus infinities so far: relative to 0, nothing to add
                    const float ref = mx == -INFINITY ? 0.0f : mx;
                    const uint64_t ref2 = join2(-ref, -ref), log2 = join2(kLog2e, kLog2e);
                    uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float x[4];
                        split2(mul2(add2(join2(v[j], v[j + 1]), ref2), log2), x[0], x[1]);
                        split2(mul2(add2(join2(v[j + 2], v[j + 3]), ref2), log2), x[2], x[3]);
                        sum0 = add2(sum0, join2(ex2(x[0]), ex2(x[1])));
                        sum1 = add2(sum1, join2(ex2(x[2]), ex2(x[3])));
                    }
                    float s0, s1;
                    split2(add2(sum0, sum1), s0, s1);
                    sum = (top == mx ? sum : sum * ex2((top - ref) * kLog2e)) + (s0 + s1);
                    top = mx;
                };
                if constexpr (kLong) {
                    float v[4][32];
                    if (!logits(v, t)) break;
#pragma unroll
                    for (int c = 0; c < kWide / 32; c++) take(v[c], c);
                } else {
#pragma unroll 1
                    for (int c = 0; c < kWide / 32; c++) {
                        float v[32];
                        ptx::load32(acc + half * kWide + c * 32, v);
                        ptx::wait32(v);
                        if (c == kWide / 32 - 1) release(buf);
                        take(v, c);
                    }
                }
                if (m < M) e.part[((int64_t)t.nt * 2 + half) * job.M + m] = make_float2(top, sum);
            } else if constexpr (kZ) {
                constexpr int kWide = kCols / 2;
                const int64_t n0 = (int64_t)t.nt * kCols + half * kWide;
                const int col0 = (int)(e.col0 + n0);
                const bool any = __any_sync(0xffffffffu, row.target >= col0 && row.target < col0 + kWide);
                auto put = [&](float (&v)[32], int c) {
                    if (n0 + c * 32 >= N) return;
                    unsigned w[16];
                    loss_z<T>(v, w, row, col0 + c * 32, 32, any, e.lse, e.src, m);
                    store_block<T>(st, w, static_cast<T *>(e.o0), e.ldo, m0, M, n0 + c * 32, N, e.vec & 1, lane);
                };
                if constexpr (kLong) {
                    float v[4][32];
                    if (!logits(v, t)) break;
#pragma unroll
                    for (int c = 0; c < kWide / 32; c++) put(v[c], c);
                } else {
#pragma unroll 1
                    for (int c = 0; c < kWide / 32; c++) {
                        float v[32];
                        ptx::load32(acc + half * kWide + c * 32, v);
                        ptx::wait32(v);
                        if (c == kWide / 32 - 1) release(buf);
                        put(v, c);
                    }
                }
            }
        }
    }

    // ---------------------------------------------------------------- the end
    __syncwarp();
    if (*s_abort) {
        // a wait ran out: give the copies in flight a millisecond to land
        const unsigned long long t0 = tc::gtimer();
        while (tc::gtimer() - t0 < 1000000ull) {
        }
    }
    tc::fence_before();
    __syncthreads();
    ptx::cluster_sync();
    tc::fence_after();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    if (threadIdx.x == 0 && *s_error) {
        *static_cast<volatile int *>(p.error) = *s_error;
        __threadfence_system();
    }
}

// out[m][n] = 16-bit (scale * sum over the parts of acc[part][m][n]), four
// columns a lane; with pos the sums are those of row pos[m], or none (-1).
// MANY: the 8 warps of a block take every 8th part each and are added up in
// order (148 parts of 1024 x 16: 37 us with a thread going through all of them).
struct JoinArgs {
    const float *acc;
    int parts;
    int64_t rows, M, N, ld;  // rows of a part, rows and columns of the result, pitch of acc
    const float *unscale;    // not NULL: the scale
    const int *pos;
};
template <class T, bool MANY>
__global__ void __launch_bounds__(256) k_join(JoinArgs p, T *out) {
    after_previous();
    __shared__ float4 red[MANY ? 8 : 1][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per = p.ld / 4, i = MANY ? (int64_t)blockIdx.x * 32 + lane : (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (!MANY && i >= p.M * per) return;
    const int64_t m = i / per, c = i - m * per;
    int64_t from = -1;
    if (i < p.M * per) from = p.pos ? p.pos[m] : m;
    float4 s = make_float4(0, 0, 0, 0);
    auto add = [&](const float4 &v) { s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w; };
    if (from >= 0) {
        const float4 *a = reinterpret_cast<const float4 *>(p.acc) + from * per + c;
#pragma unroll 4
        for (int k = MANY ? warp : 0; k < p.parts; k += MANY ? 8 : 1) add(a[k * p.rows * per]);
    }
    if (MANY) {
        red[warp][lane] = s;
        __syncthreads();
        if (warp || i >= p.M * per) return;
        for (int k = 1; k < 8; k++) add(red[k][lane]);
    }
    const int64_t n = c * 4;
    const float scale = p.unscale ? *p.unscale : 1.0f;
    const float v[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
    T *o = out + m * p.N + n;
    if (p.N % 4 == 0 && n < p.N && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < p.N) o[j] = from_f<T>(v[j]);
    }
}

// Matrices with rows on 16-byte boundaries, for the TMA unit: up to four in a
// launch, one for each blockIdx.y, eight elements a thread, read one by one
// (5047 rows of 1001 in 5 us, a launch's latency and 4 TB/s).
struct Repitch {
    const unsigned short *from[4];
    unsigned short *to[4];
    int64_t ld[4], rows[4], cols[4], pitch[4];
};
__global__ void k_repitch(const __grid_constant__ Repitch p) {
    after_previous();
    const int k = blockIdx.y;
    const int64_t per = (p.cols[k] + 7) / 8, n = p.rows[k] * per;  // what lies past a row's end is never read
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / per, c = i % per * 8;
        *reinterpret_cast<uint4 *>(p.to[k] + r * p.pitch[k] + c) = load8(p.from[k] + r * p.ld[k], c, p.cols[k], false);
    }
}

}  // namespace train
}  // namespace hb
