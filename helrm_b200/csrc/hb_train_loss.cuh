// hb_train_loss.cuh -- the loss's gradients for narrow rows (inner <= 64), in
// one kernel.  Included by hb_train.cu after hb_train_mma.cuh.
//
// With few features a logit costs little more than its exponential, and Z,
// written once and read twice, would be most of the traffic: 6 bytes a logit
// against 6 * inner flops.  Here Z stays in shared memory.  A block owns every
// gridDim.x-th group of 128 vocabulary rows and takes the tokens 128 at a time:
//
//   S = H_t W_b^T              128 x 128, in tensor memory (two of them)
//   Z = dloss 2^((S - max) log2(e) - ..) - [target]   16 warps, to shared memory
//   dW_b += Z^T H_t            tensor memory, written out after the last t
//   dH_t += Z W_b              tensor memory, one for each t of the group
//
// One copy of each operand serves both of its uses: Z with a token's 64
// vocabulary entries in a 128-byte row is K-major for dH and MN-major for dW,
// H and W with a row's features in 128 bytes are K-major for S and MN-major for
// dW and dH.  128 columns of tensor memory hold dH for a group of tokens
// (128 / depth tiles, depth the features rounded up to 16); more tokens are
// taken group by group, dW then adding up in 32 bits in global memory, always
// by the same block.  Each block's dH is a partial sum, joined in block order
// afterwards: no atomics, the same bits in every run.
//
// Bounds at 1024 tokens x 1000003 rows x 16: the exponentials, 16 a clock and
// SM, 0.23 ms; operand bytes 64 MB.  It takes 0.44 ms: about 2000 clocks a tile,
// of which the exponentials are 1024 and the sixteen small products 1150, with
// three hand-offs between them.
#pragma once

namespace hb {
namespace train {

constexpr int kNarrow = 64;           // features at most
constexpr int kNarrowGroup = 8;       // token tiles of a group at most
constexpr int kNarrowWarps = 16;      // epilogue warps
constexpr int kNarrowThreads = 96 + 32 * kNarrowWarps;
constexpr int kPanel = 128 * 128;     // bytes of 128 rows of 64 elements
constexpr int kNarrowBars = 2 + 2 * 8 + 4;
constexpr int kNarrowSmem = (kNarrowGroup + 2 + 4) * kPanel + 8 * kNarrowBars + 16;

struct NarrowArgs {
    CUtensorMap h, w;
    int64_t capacity, vocab;  // capacity: rows of h and of a block's partial sums
    int inner, depth, group;  // depth: inner rounded up to 16; group: token tiles of a group
    const LossRow *rows;
    const float2 *lse;
    const int *src;
    const LossPlan *plan;
    void *dw;                 // dense rows
    float *acc_w;             // [vocab][depth] running sums, for several groups
    float *part_h;            // [block][tokens][depth]
    int *error;
};

namespace ptx {
__device__ __forceinline__ void tma_load_own(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_own(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
}  // namespace ptx

template <class T>
__global__ void __launch_bounds__(kNarrowThreads, 1) k_loss_grads_narrow(const __grid_constant__ NarrowArgs p) {
    extern __shared__ __align__(1024) unsigned char smem[];
    const unsigned sH = tc::smem_u32(smem), sW = sH + kNarrowGroup * kPanel, sZ = sW + 2 * kPanel;
    unsigned char *zbuf = smem + (kNarrowGroup + 2) * kPanel;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (kNarrowGroup + 6) * kPanel);
    const unsigned bar = tc::smem_u32(bars);
    const unsigned hfull = bar, dhfull = bar + 8, wfull = bar + 16, wempty = bar + 32, sfull = bar + 48,
                   sempty = bar + 64, zfull = bar + 80, zempty = bar + 96, dwfull = bar + 112, dwempty = bar + 128,
                   dhempty = bar + 144, drain = bar + 152, drain2 = bar + 160;
    unsigned *s_tmem = reinterpret_cast<unsigned *>(bars + kNarrowBars);
    int *s_error = reinterpret_cast<int *>(s_tmem + 1);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        tc::mbar_init(hfull, 1);
        tc::mbar_init(dhfull, 1);
        for (int i = 0; i < 2; i++) {
            tc::mbar_init(wfull + 8 * i, 1);
            tc::mbar_init(wempty + 8 * i, 1);
            tc::mbar_init(sfull + 8 * i, 1);
            tc::mbar_init(sempty + 8 * i, kNarrowWarps / 2);
            tc::mbar_init(zfull + 8 * i, kNarrowWarps / 2);
            tc::mbar_init(zempty + 8 * i, 1);
            tc::mbar_init(dwfull + 8 * i, 1);
            tc::mbar_init(dwempty + 8 * i, kNarrowWarps);
        }
        tc::mbar_init(dhempty, kNarrowWarps);
        tc::mbar_init(drain, 1);
        tc::mbar_init(drain2, 1);
        *s_error = 0;
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(s_tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tmem = *s_tmem;
    after_previous();
    const unsigned tS = tmem, tDW = tmem + 256, tDH = tmem + 384;

    const int token_tiles = max(1, (p.plan->count + 127) / 128), groups = (token_tiles + p.group - 1) / p.group;
    const int blocks_all = (int)((p.vocab + 127) / 128);
    const int mine = (blocks_all - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA
        if (lane == 0) {
            bool ok = true;
            unsigned nw = 0;
            for (int g = 0; ok && g < groups; g++) {
                const int tiles = min(p.group, token_tiles - g * p.group);
                // the group before has read its H
                if (g && !(ok = mbar_wait(dhfull, (unsigned)(g - 1) & 1, s_abort, s_error, 1))) break;
                tc::mbar_arrive_tx(hfull, tiles * kPanel);
                for (int t = 0; t < tiles; t++)
                    ptx::tma_load_own(sH + t * kPanel, &p.h, 0, (g * p.group + t) * 128, hfull);
                for (int b = 0; b < mine; b++, nw++) {
                    const unsigned s = nw & 1;
                    if (!(ok = mbar_wait(wempty + 8 * s, ((nw >> 1) & 1) ^ 1, s_abort, s_error, 1))) break;
                    tc::mbar_arrive_tx(wfull + 8 * s, kPanel);
                    ptx::tma_load_own(sW + s * kPanel, &p.w, 0, ((int)blockIdx.x + b * (int)gridDim.x) * 128,
                                      wfull + 8 * s);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA of the gradients
        if (lane == 0) {
            constexpr unsigned kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr unsigned kBase = (1u << 4) | kType | ((128u >> 4) << 24);
            const unsigned idw = kBase | (1u << 15) | (1u << 16) | ((unsigned)(p.depth >> 3) << 17);  // dW
            const unsigned idh = kBase | (1u << 16) | ((unsigned)(p.depth >> 3) << 17);               // dH
            unsigned n = 0, nb = 0;  // tiles and blocks done
            bool ok = true;
            for (int g = 0; ok && g < groups; g++) {
                const int tiles = min(p.group, token_tiles - g * p.group), all = tiles * mine;
                ok = mbar_wait(hfull, (unsigned)g & 1, s_abort, s_error, 2) &&
                     (g == 0 || mbar_wait(dhempty, (unsigned)(g - 1) & 1, s_abort, s_error, 2));
                int t = 0, b = 0;
                for (int j = 0; ok && j < all; j++, n++) {
                    if (t == 0 &&
                        !(ok = mbar_wait(wfull + 8 * (nb & 1), (nb >> 1) & 1, s_abort, s_error, 2) &&
                               mbar_wait(dwempty + 8 * (nb & 1), ((nb >> 1) & 1) ^ 1, s_abort, s_error, 2)))
                        break;
                    if (!(ok = mbar_wait(zfull + 8 * (n & 1), (n >> 1) & 1, s_abort, s_error, 2))) break;
                    tc::fence_after();
                    const unsigned z = sZ + (n & 1) * 2 * kPanel;
                    // Z MN-major: the vocabulary's two 64-entry panels are kPanel bytes apart
                    const uint64_t za = ptx::descriptor(z, kPanel), hb = ptx::descriptor(sH + t * kPanel);
                    const unsigned dw = tDW + (nb & 1) * 64, dh = tDH + t * p.depth;
#pragma unroll
                    for (int k = 0; k < 8; k++) ptx::mma_own(dw, za + 128 * k, hb + 128 * k, idw, t > 0 || k > 0);
                    const uint64_t zk = ptx::descriptor(z), wb = ptx::descriptor(sW + (nb & 1) * kPanel);
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        ptx::mma_own(dh, zk + (k >> 2) * (kPanel >> 4) + 2 * (k & 3), wb + 128 * k, idh, b > 0 || k > 0);
                    ptx::commit(zempty + 8 * (n & 1));
                    if (++t == tiles) {
                        t = 0;
                        ptx::commit(wempty + 8 * (nb & 1));
                        ptx::commit(dwfull + 8 * (nb & 1));
                        nb++;
                        b++;
                    }
                }
                if (ok) ptx::commit(dhfull);
            }
            ptx::commit(drain);
            mbar_wait(drain, 0, nullptr, s_error, 8);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------ MMA of S
        // A thread of its own: S of a tile to come never waits behind the hand-off of a finished Z (one thread for
        // all three products: 83 us at 1024 x 131072 x 16).
        if (lane == 0) {
            constexpr unsigned kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            const unsigned ids = (1u << 4) | kType | ((128u >> 4) << 24) | ((128u >> 3) << 17);
            const int steps = p.depth / 16;
            unsigned n = 0, nb = 0;
            bool ok = true;
            for (int g = 0; ok && g < groups; g++) {
                const int tiles = min(p.group, token_tiles - g * p.group);
                ok = mbar_wait(hfull, (unsigned)g & 1, s_abort, s_error, 2);
                for (int b = 0; ok && b < mine; b++, nb++) {
                    if (!(ok = mbar_wait(wfull + 8 * (nb & 1), (nb >> 1) & 1, s_abort, s_error, 2))) break;
                    const uint64_t wd = ptx::descriptor(sW + (nb & 1) * kPanel);
                    for (int t = 0; t < tiles; t++, n++) {
                        if (!(ok = mbar_wait(sempty + 8 * (n & 1), ((n >> 1) & 1) ^ 1, s_abort, s_error, 2)))
                            break;
                        tc::fence_after();
                        const uint64_t hd = ptx::descriptor(sH + t * kPanel);
                        for (int k = 0; k < steps; k++)
                            ptx::mma_own(tS + (n & 1) * 128, hd + 2 * k, wd + 2 * k, ids, k > 0);
                        ptx::commit(sfull + 8 * (n & 1));
                    }
                }
            }
            ptx::commit(drain2);
            mbar_wait(drain2, 0, nullptr, s_error, 8);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue
        // Warps 3-10 take the even tiles, 11-18 the odd ones, each of them 64 columns: a warp that took a part of
        // every tile would go through all of a tile's hand-offs within one tile's time (1024 x 131072 x 16: 118 us
        // whether or not the exponentials were computed).
        const int quad = warp & 3, quarter = (warp - 3) >> 2, set = quarter >> 1;
        const unsigned lanes = (unsigned)(32 * quad) << 16;
        const int r = 32 * quad + lane;  // row of a tile
        auto wait_all = [&](unsigned a, unsigned parity) {
            return __all_sync(0xffffffffu, mbar_wait(a, parity, s_abort, s_error, 4));
        };
        const float unscale = p.plan->unscale;
        const bool vec = p.inner % 8 == 0 && (reinterpret_cast<uintptr_t>(p.dw) & 15) == 0;
        auto fetch = [&](int64_t m) {  // the rows that fill up the last tile are there
            LossRow q;
            *reinterpret_cast<float4 *>(&q) = reinterpret_cast<const float4 *>(p.rows)[m];
            return q;
        };
        // dW of the block that was finished last: 16 of its columns a warp
        auto write_dw = [&](unsigned nb, int64_t block, int g) -> bool {
            if (!wait_all(dwfull + 8 * (nb & 1), (nb >> 1) & 1)) return false;
            tc::fence_after();
            const int c0 = quarter * 16;
            if (c0 < p.depth) {
                float v[16];
                ptx::load16(tDW + (nb & 1) * 64 + lanes + c0, v);
                ptx::wait16(v);
                const int64_t row = block * 128 + r;
                if (row < p.vocab) {
                    if (groups > 1) {
                        float4 *a = reinterpret_cast<float4 *>(p.acc_w + row * p.depth + c0);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if (g == 0) {
                                a[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                            } else if (g + 1 < groups) {  // this lane alone adds here: the order is the groups'
                                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(a + k),
                                             "f"(v[4 * k]), "f"(v[4 * k + 1]), "f"(v[4 * k + 2]), "f"(v[4 * k + 3])
                                             : "memory");
                            } else {
                                const float4 o = __ldcg(a + k);
                                v[4 * k] += o.x, v[4 * k + 1] += o.y, v[4 * k + 2] += o.z, v[4 * k + 3] += o.w;
                            }
                        }
                    }
                    if (g + 1 == groups) {
                        unsigned short *o = static_cast<unsigned short *>(p.dw) + row * p.inner;
                        unsigned w[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) w[k] = pack2<T>(v[2 * k] * unscale, v[2 * k + 1] * unscale);
                        store8(o, c0, p.inner, vec, make_uint4(w[0], w[1], w[2], w[3]));
                        store8(o, c0 + 8, p.inner, vec, make_uint4(w[4], w[5], w[6], w[7]));
                    }
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(dwempty + 8 * (nb & 1));
            return true;
        };
        unsigned n = 0, nb = 0;  // tiles and blocks so far; written: blocks whose dW this warp has written
        bool ok = true;
        for (int g = 0; ok && g < groups; g++) {
            const int tiles = min(p.group, token_tiles - g * p.group);
            const int64_t first = (int64_t)g * p.group * 128 + r;
            const unsigned nb0 = nb;  // the group's first block
            unsigned written = nb;
            auto write_until = [&](unsigned end) -> bool {
                for (; written < end; written++)
                    if (!write_dw(written, blockIdx.x + (int64_t)(written - nb0) * gridDim.x, g)) return false;
                return true;
            };
            // this warp's tiles: every other one
            auto tile_after = [&](int &b, int &t, int by) {
                for (t += by; t >= tiles; t -= tiles) b++;
            };
            int b = 0, t = 0;
            tile_after(b, t, (n & 1) != (unsigned)set);
            LossRow next = fetch(first + t * 128);
            const unsigned end = n + tiles * mine;
            for (n += (n & 1) != (unsigned)set; n < end; n += 2) {
                const LossRow row = next;
                const int64_t m = first + t * 128;
                const int col = (blockIdx.x + b * gridDim.x) * 128 + (quarter & 1) * 64;
                const unsigned before = nb0 + b;
                tile_after(b, t, 2);
                next = fetch(first + t * 128);
                if (!(ok = wait_all(sfull + 8 * set, (n >> 1) & 1))) break;
                tc::fence_after();
                const bool any = __any_sync(0xffffffffu, row.target >= col && row.target < col + 64);
                unsigned char *z = zbuf + set * 2 * kPanel + (quarter & 1) * kPanel + r * 128;
#pragma unroll 1
                for (int c = 0; c < 2; c++) {
                    float v[32];
                    unsigned w[16];
                    ptx::load32(tS + set * 128 + lanes + (quarter & 1) * 64 + c * 32, v);
                    ptx::wait32(v);
                    if (c) {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(sempty + 8 * set);
                    }
                    loss_z<T>(v, w, row, col + c * 32, (int)p.vocab - col - c * 32, any, p.lse, p.src, m);
                    // the products that read this buffer two tiles ago
                    if (!c && !(ok = wait_all(zempty + 8 * set, ((n >> 1) & 1) ^ 1))) break;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        *reinterpret_cast<uint4 *>(z + (((c * 4 + j) ^ (r & 7)) << 4)) =
                            make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                }
                if (!ok) break;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(zfull + 8 * set);
                // the blocks before this one, while this one's products run
                if (!(ok = write_until(before))) break;
            }
            n = end;
            nb = nb0 + mine;
            if (ok) ok = write_until(nb);
            if (!ok || !(ok = wait_all(dhfull, (unsigned)g & 1))) break;
            tc::fence_after();
            const int c0 = quarter * 16;
            for (int t = 0; t < tiles; t++) {
                const int64_t m = first + t * 128;
                if (c0 >= p.depth) continue;
                float v[16];
                ptx::load16(tDH + t * p.depth + lanes + c0, v);
                ptx::wait16(v);
                float4 *o = reinterpret_cast<float4 *>(p.part_h + ((int64_t)blockIdx.x * p.capacity + m) * p.depth + c0);
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(dhempty);
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
    tc::fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    if (threadIdx.x == 0 && *s_error) {
        *static_cast<volatile int *>(p.error) = *s_error;
        __threadfence_system();
    }
}

}  // namespace train
}  // namespace hb
