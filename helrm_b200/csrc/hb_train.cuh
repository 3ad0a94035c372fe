// hb_train.cuh -- kernels of the training operators: the gated feed-forward
// block and its gradients, 8-bit activation checkpoints, and softmax cross
// entropy over a vocabulary.  Included by hb_train.cu.
//
// Every matrix product here is one tiled product with an operand layout and
// an epilogue of its own:
//   gated forward    G = X Wg^T, U = X Wu^T (one pass over X), H = act(G) U
//   gated backward   the same two, dG = dH U act'(G), dU = dH act(G); then
//                    dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X
//   loss forward     L = H W^T; max and sum of exponentials of a tile's row
//   loss backward    L again, Z = dloss (exp(L - lse) - [column = target]);
//                    then dH = Z W, dW = Z^T H
// Accumulators and softmax statistics are 32-bit floats.  dG, dU and Z are
// rounded to the 16-bit type once, as operands of the products they enter.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace hb {
namespace train {

template <class T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T> __device__ __forceinline__ unsigned pack2(float lo, float hi);
template <> __device__ __forceinline__ unsigned pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&v);
}
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&v);
}
template <class T> __device__ __forceinline__ float2 unpack2(unsigned v);
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
}

// Every kernel here starts while the one before it in the stream ends: it sets
// itself up, lets the next one do the same, and touches no memory of others
// until all of that one's work is visible.  Kernel pointers carry no
// __restrict__, which would let a load move above the wait.
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// Two 32-bit operations in one instruction, on neighbouring registers; each
// half is rounded as the single operation is.
__device__ __forceinline__ uint64_t join2(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void split2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 1 / (1 + exp(-g)), within a few units of 2^-23: a division takes a slow path
// for small numerators (gated 64 x 432 x 512: 17.8 us with it, 8.1 without)
__device__ __forceinline__ float sigmoid(float g) { return rcp(1.0f + ex2(-kLog2e * g)); }

// The normal distribution function and density: Abramowitz and Stegun 7.1.26,
// erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 x), within
// 1.5e-7, whose exponential the density needs anyway (with erff and a second
// exponential the gated backward pass of 4096 x 1024 x 4096 took 92 us).
__device__ __forceinline__ void normal(float g, float &cdf, float &pdf) {
    const float x = fabsf(g) * 0.70710678118654752f, t = rcp(fmaf(0.3275911f, x, 1.0f));
    const float e = ex2(g * g * (-0.5f * kLog2e));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float q = 0.5f * p * t * e;  // the smaller tail
    cdf = g > 0.0f ? 1.0f - q : q;
    pdf = 0.39894228040143268f * e;
}

// act(g), and with its derivative
template <int ACT>
__device__ __forceinline__ float act_f(float g) {
    if (ACT == HELRM_ACT_RELU) return fmaxf(g, 0.0f) + (g != g ? g : 0.0f);  // NaN stays NaN
    if (ACT == HELRM_ACT_SILU) return g * sigmoid(g);
    if (ACT == HELRM_ACT_GELU) {
        float cdf, pdf;
        normal(g, cdf, pdf);
        return g * cdf;
    }
    return g;
}
template <int ACT>
__device__ __forceinline__ void act_df(float g, float &a, float &d) {
    if (ACT == HELRM_ACT_RELU) {
        a = act_f<ACT>(g);
        d = g > 0.0f ? 1.0f : 0.0f;
    } else if (ACT == HELRM_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        d = s * (1.0f + g * (1.0f - s));
    } else if (ACT == HELRM_ACT_GELU) {
        float cdf, pdf;
        normal(g, cdf, pdf);
        a = g * cdf;
        d = fmaf(g, pdf, cdf);
    } else {
        a = g;
        d = 1.0f;
    }
}

// ---------------------------------------------------------------- products
enum Epi { EPI_GATED, EPI_GATED_BWD, EPI_OUT, EPI_LSE, EPI_LSE_LONG, EPI_Z, EPI_Z_LONG };
struct EpiArgs {
    void *o0 = nullptr, *o1 = nullptr;  // 16-bit outputs
    int64_t ldo = 0;                    // their row pitch, or that of acc
    int vec = 0;                        // 1: outputs fit 16-byte stores, 2: dh fits 16-byte loads
    const void *dh = nullptr;
    int64_t lddh = 0;
    float *acc = nullptr;               // EPI_OUT: 32-bit sums instead, [output][part][row][ldo]
    int first = 1;                      // 0: added to what acc holds
    float2 *part = nullptr;             // EPI_LSE: (max, sum) of each warp's columns, [part][row]
    float *at = nullptr;                // EPI_LSE: the target's logit
    const int64_t *target = nullptr;
    const float2 *lse = nullptr;        // EPI_Z: the row's (maximum, log of the sum relative to it)
    const struct LossRow *rows = nullptr;
    const int *src = nullptr;
    int64_t col0 = 0;                   // EPI_Z: first column of the piece in the vocabulary
    const float *unscale = nullptr;     // EPI_OUT: the operands' scale is undone when a product with them is stored
    const float4 *range = nullptr;      // EPI_GATED_BWD in fp16: what k_gated_range found, a block each,
    int ranges = 0;
    float *made = nullptr;              // and where the scale's inverse goes
};

// 16-bit values col..col+7 of a row as four words; zeros past the end
__device__ __forceinline__ uint4 load8(const unsigned short *row, int64_t col, int64_t cols, bool vec) {
    if (vec && col + 8 <= cols) return *reinterpret_cast<const uint4 *>(row + col);
    unsigned p[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (col + k < cols) p[k >> 1] |= (unsigned)row[col + k] << (16 * (k & 1));
    return make_uint4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store8(unsigned short *row, int64_t col, int64_t cols, bool vec, uint4 v) {
    if (vec && col + 8 <= cols) {
        *reinterpret_cast<uint4 *>(row + col) = v;
        return;
    }
    const unsigned p[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (col + k < cols) row[col + k] = (unsigned short)(p[k >> 1] >> (16 * (k & 1)));
}

// ---------------------------------------------------------------- fp16's range
// dG = dH U act'(G) and dU = dH act(G) enter products whose results fp16 may hold
// where it does not hold them (dH 6e4, U 4, weights of 1e-2), or holds few of
// their bits (dH 1e-5, act(G) 1e-2).  So they are scaled by a power of two that
// brings a bound of both to at least 2^14, below 2^15:
//   max_i (max |dH_i| |x_i|) max(1.13 max_j |wu_j|, max_j |wg_j|)
// with the norms of rows (Cauchy and Schwarz; |act'| <= 1.13, |act(g)| <= |g|).
// Values down to 2^-28 of the bound keep all their bits.  What is not finite, a
// value of dH or a row, has no say.  bf16 has a float's range and no scale.
// The kernel reads what the next one will read: 64 x 432 x 512 21.5 us without it
// and 23.6 with it, 2047 x 1001 x 1500 58.6 and 65.6, 4096 x 1024 x 4096 (58 MB,
// in 15 us) 172 and 187.
constexpr int kRangeBlocks = 2 * 148, kRangeThreads = 512, kRangeWarps = kRangeThreads / 32;
constexpr int kRangeBatch = 2048;  // columns of a warp's eight 16-byte loads a lane
struct GatedRange {
    const unsigned short *dh, *x, *w[2];  // wu, wg; rows on 16-byte boundaries, but for dh's (vec)
    int64_t lddh, ldx, ldw[2], tokens, width, inner;
    bool vec;
    float4 *part;  // a block's: (max |dH_i| |x_i|)^2, then |wu_j|^2 and |wg_j|^2
};
// A lane's share of a row's sum of squares (NORM) or of its largest finite
// magnitude, over every step-th batch from the first on.
template <bool NORM>
__device__ __forceinline__ float range_of(const unsigned short *row, int64_t n, bool vec, int first, int step) {
    const int lane = threadIdx.x & 31;
    float s = 0.0f;
    auto take = [&](unsigned two) {
        const float2 f = unpack2<__half>(two);
        const float a = fabsf(f.x), b = fabsf(f.y);
        s = NORM ? fmaf(f.x, f.x, fmaf(f.y, f.y, s)) : fmaxf(s, fmaxf(a < INFINITY ? a : 0.0f, b < INFINITY ? b : 0.0f));
    };
    for (int64_t b = (int64_t)first * kRangeBatch; b < n; b += (int64_t)step * kRangeBatch) {
        const unsigned short *in = row + b;
        const int m = (int)(n - b < kRangeBatch ? n - b : kRangeBatch);
        if (NORM || vec) {
            const int whole = m / 8 * 8;
            uint4 v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int c = lane * 8 + j * 256;
                v[j] = c < whole ? *reinterpret_cast<const uint4 *>(in + c) : make_uint4(0, 0, 0, 0);
            }
            const unsigned short last = whole + lane < m ? in[whole + lane] : (unsigned short)0;
#pragma unroll
            for (int j = 0; j < 8; j++) take(v[j].x), take(v[j].y), take(v[j].z), take(v[j].w);
            take(last);
        } else {
            for (int c0 = lane; c0 < m; c0 += 256) {
                unsigned short v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = c0 + j * 32 < m ? in[c0 + j * 32] : (unsigned short)0;
#pragma unroll
                for (int j = 0; j < 8; j++) take(v[j]);
            }
        }
    }
    return s;
}
__device__ __forceinline__ float warp_sum(float s) {
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
__device__ __forceinline__ float warp_max(float s) {
    for (int o = 16; o; o >>= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
    return s;
}
__global__ void __launch_bounds__(kRangeThreads) k_gated_range(const __grid_constant__ GatedRange p) {
    after_previous();
    __shared__ float red[kRangeWarps][3];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t warps = (int64_t)gridDim.x * kRangeWarps, mine = (int64_t)blockIdx.x * kRangeWarps + warp;
    float top[3] = {0.0f, 0.0f, 0.0f};
    const bool apart = p.width + p.inner > 8 * kRangeBatch;  // long rows: a token a block
    for (int64_t r = blockIdx.x; apart && r < p.tokens; r += gridDim.x) {
        const float d = warp_max(range_of<false>(p.dh + r * p.lddh, p.width, p.vec, warp, kRangeWarps));
        const float n = warp_sum(range_of<true>(p.x + r * p.ldx, p.inner, true, warp, kRangeWarps));
        if (lane == 0) red[warp][0] = d, red[warp][1] = n;
        __syncthreads();
        const float most = warp_max(lane < kRangeWarps ? red[lane][0] : 0.0f);
        const float norm = warp_sum(lane < kRangeWarps ? red[lane][1] : 0.0f);
        __syncthreads();
        if (norm < INFINITY) top[0] = fmaxf(top[0], most * most * norm);
    }
    // a warp a token or a row of weights
    const int64_t tokens = apart ? 0 : p.tokens;
    for (int64_t i = mine; i < tokens + 2 * p.width; i += warps) {
        if (i < tokens) {
            const float d = range_of<false>(p.dh + i * p.lddh, p.width, p.vec, 0, 1);
            const float n = range_of<true>(p.x + i * p.ldx, p.inner, true, 0, 1);
            const float most = warp_max(d), norm = warp_sum(n);
            if (norm < INFINITY) top[0] = fmaxf(top[0], most * most * norm);
        } else {
            const int64_t j = i - tokens;
            const bool second = j >= p.width;
            const float norm = warp_sum(
                range_of<true>(second ? p.w[1] + (j - p.width) * p.ldw[1] : p.w[0] + j * p.ldw[0], p.inner, true, 0, 1));
            if (norm < INFINITY) (second ? top[2] : top[1]) = fmaxf(second ? top[2] : top[1], norm);
        }
    }
    __syncthreads();
    if (lane == 0)
        for (int k = 0; k < 3; k++) red[warp][k] = top[k];  // the same in every lane
    __syncthreads();
    if (threadIdx.x < 3) {
        float t = 0.0f;
        for (int i = 0; i < kRangeWarps; i++) t = fmaxf(t, red[i][threadIdx.x]);
        reinterpret_cast<float *>(p.part + blockIdx.x)[threadIdx.x] = t;
    }
}
// The scale from what n blocks found, in every lane of a warp.
__device__ __forceinline__ float gated_scale(const float4 *part, int n) {
    float d = 0.0f, u = 0.0f, g = 0.0f;
#pragma unroll
    for (int k = 0; k < (kRangeBlocks + 31) / 32; k++) {  // all loads at once
        const int i = 32 * k + (threadIdx.x & 31);
        const float4 v = i < n ? part[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        d = fmaxf(d, v.x), u = fmaxf(u, v.y), g = fmaxf(g, v.z);
    }
    // 2^-75 to 2^80, or 0
    const float bound = sqrtf(warp_max(d)) * fmaxf(1.13f * sqrtf(warp_max(u)), sqrtf(warp_max(g)));
    return bound > 0.0f ? __uint_as_float((unsigned)(127 + 14 + 127 - (int)(__float_as_uint(bound) >> 23)) << 23) : 1.0f;
}

// ---------------------------------------------------------------- the loss
// The row's (maximum, log of the sum relative to it) and loss from the (max,
// sum) of every tile of the vocabulary.  The pair is kept apart: rounded to one
// 32-bit number, a log-sum-exp of some thousands would be off by 2^-13, and so
// would every probability.
// A block takes 32 rows, its 32 warps every 32nd of the parts.  With more than
// kLossParts of them, blockIdx.y first joins that many each (joined, one a
// block), so that few rows over a large vocabulary are read by enough blocks
// (1024 rows, 7814 parts: 133 us in one pass).
constexpr int kLossParts = 512;
template <bool LAST>
__global__ void __launch_bounds__(1024) k_loss(const float2 *part, int64_t parts,
                                               const float *at, const int64_t *target,
                                               int64_t ignore, int64_t vocab, int64_t M, float *loss,
                                               float2 *lse) {
    after_previous();
    __shared__ float2 red[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t m = (int64_t)blockIdx.x * 32 + lane;
    float top = -INFINITY, s = 0.0f;
    auto join = [&](float2 p) {
        const float mx = fmaxf(top, p.x), ref = mx == -INFINITY ? 0.0f : mx;
        s = (top == mx ? s : s * __expf(top - ref)) + (p.x == mx ? p.y : p.y * __expf(p.x - ref));
        top = mx;
    };
    int64_t from = 0;
    if (!LAST) {
        from = (int64_t)blockIdx.y * kLossParts;
        parts = min(parts, from + kLossParts);
    }
    if (m < M) {
#pragma unroll 4
        for (int64_t i = from + warp; i < parts; i += 32) join(part[i * M + m]);
    }
    red[warp][lane] = make_float2(top, s);
    __syncthreads();
    // a warp a row from here
    const float2 mine = red[lane][warp];
    top = mine.x, s = mine.y;
    for (int o = 16; o; o >>= 1) {
        const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, s, o));
        join(other);
    }
    const int64_t row = (int64_t)blockIdx.x * 32 + warp;
    if (lane || row >= M) return;
    if (!LAST) {
        lse[blockIdx.y * M + row] = make_float2(top, s);
        return;
    }
    const float l = logf(s);
    const int64_t t = target[row];
    lse[row] = make_float2(top, l);
    loss[row] = t == ignore ? 0.0f : t < 0 || t >= vocab ? NAN : top - at[row] + l;
}

// What the gradients' epilogues need to know of a row, in one 16-byte load:
// z = g exp(l - max - x1) = sign(g) 2^((l - max) log2(e) + add).  A row that
// only fills up has target kNoTarget, one whose target is out of range g = NaN.
struct LossRow {
    float max, add, g;
    int target;
};
constexpr int kNoTarget = -2147483647 - 1;

// Rows without a target take no part in the gradients: the others are gathered
// to the front (a third of 777 rows ignored: gradients over 32001 rows of 432
// 91 -> 73 us), so that what an ignored row holds, infinities or NaN, reaches
// nothing.  rows[j], src[j]: the j-th row that takes part and where it came
// from, filled up to a multiple of 256, at least 256; pos[m]: the place of row
// m, or -1.
struct LossPlan {
    int filled;  // rows, with those that fill up
    int count;   // rows that take part
    float unscale;  // what Z is to be multiplied by
};
// Each block goes through all the targets, four a thread at a time, keeps the
// `per` places that are its own, and copies their rows to 16-byte boundaries
// (zeros where they fill up): one launch, where a plan by one block and a copy
// after it took 10 us.
// Z is scaled: the largest |dloss| of a row that takes part becomes 1, for fp16
// 2^15, so that probabilities down to 2^-39 keep a place in that type's range.
// A batch whose rows all weigh the same (a mean) then has its targets' entries
// at a power of two, which 16 bits hold without an error.
struct LossRows {
    const float *dloss;
    const int64_t *target;
    const float2 *lse;
    int64_t ignore, vocab, M;
    const unsigned short *h;
    int64_t ldh, cols;
    bool vec;
    float most;  // what the largest |dloss| becomes
    int per;
    LossRow *rows;
    int *src, *pos;
    LossPlan *plan;
    unsigned short *out;
    int64_t ldo;
};
__global__ void __launch_bounds__(1024) k_loss_rows(LossRows p) {
    after_previous();
    __shared__ float red[32];
    __shared__ int sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float top = 0.0f;
    for (int64_t m = threadIdx.x; m < p.M; m += 1024)
        if (p.target[m] != p.ignore) top = fmaxf(top, fabsf(p.dloss[m]));
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < 32; i++) top = fmaxf(top, red[i]);
    if (!(top > 0.0f && top < INFINITY)) top = p.most;
    top = fminf(fmaxf(top, 1e-30f), 1e30f);  // so that neither factor overflows
    const float scale = p.most / top, unscale = top / p.most;
    const int first = blockIdx.x * p.per, last = first + p.per;
    int base = 0;
    for (int64_t m0 = 0; m0 < p.M; m0 += 4096) {
        int64_t t[4];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t m = m0 + threadIdx.x * 4 + k;
            t[k] = m < p.M ? p.target[m] : p.ignore;
            mine += t[k] != p.ignore;
        }
        int before = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) sums[warp] = before;
        __syncthreads();
        if (warp == 0) {
            int v = sums[lane];
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            sums[lane] = v;
        }
        __syncthreads();
        int j = base + before - mine + (warp ? sums[warp - 1] : 0);
        base += sums[31];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t m = m0 + threadIdx.x * 4 + k;
            if (m >= p.M) break;
            const bool on = t[k] != p.ignore;
            if (blockIdx.x == 0) p.pos[m] = on ? j : -1;
            if (!on) continue;
            if (j >= first && j < last) {
                const bool in = t[k] >= 0 && t[k] < p.vocab;
                const float2 l = p.lse[m];
                LossRow r;
                r.g = in ? p.dloss[m] * scale : NAN;
                r.max = l.x;
                r.add = log2f(fabsf(r.g)) - l.y * kLog2e;
                r.target = in ? (int)t[k] : -1;
                p.rows[j] = r;
                p.src[j] = (int)m;
            }
            j++;
        }
        __syncthreads();
    }
    const int filled = max(256, (base + 255) / 256 * 256), end = min(last, filled);
    for (int j = max(first, base) + threadIdx.x; j < end; j += 1024) {
        p.rows[j] = {0.0f, 0.0f, 0.0f, kNoTarget};
        p.src[j] = -1;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.plan = {filled, base, unscale};
    __syncthreads();
    for (int j = first + warp; j < end; j += 32) {  // a warp a row
        const int64_t m = p.src[j];
#pragma unroll 4
        for (int64_t c = lane * 8; c < p.ldo; c += 256)
            *reinterpret_cast<uint4 *>(p.out + j * p.ldo + c) =
                m < 0 ? make_uint4(0, 0, 0, 0) : load8(p.h + m * p.ldh, c, p.cols, p.vec);
    }
}

// 32 logits of a row, the first of them column `col` of the vocabulary, to Z,
// packed in 16 words.  The target's exp(..) - 1 is formed without cancellation.
// any: whether some row of the warp may have its target here; wide: how many of
// the columns are in the vocabulary (past its end exp(0 - lse) may be infinite,
// and zero times that is no zero in the products).
template <class T>
__device__ __forceinline__ void loss_z(float (&v)[32], unsigned (&w)[16], const LossRow &r, int col, int wide, bool any,
                                       const float2 *lse, const int *src, int64_t m) {
    int at = -1;
    float hot = 0.0f;
    if (any) {
        asm volatile("");  // a branch: not 32 selections for every 32 logits
        if (r.target >= col && r.target < col + 32) at = r.target - col;
        float x = v[0];
#pragma unroll
        for (int j = 1; j < 32; j++) x = at == j ? v[j] : x;
        if (at >= 0) hot = expm1f((x - r.max) - lse[src[m]].y) * fabsf(r.g);
    }
    const uint64_t max2 = join2(-r.max, -r.max), log2 = join2(kLog2e, kLog2e), more2 = join2(r.add, r.add);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        split2(fma2(add2(join2(v[j], v[j + 1]), max2), log2, more2), v[j], v[j + 1]);
        v[j] = ex2(v[j]);
        v[j + 1] = ex2(v[j + 1]);
    }
    if (any) {
        asm volatile("");
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = at == j ? hot : v[j];
    }
    if (wide < 32) {
        asm volatile("");
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = j < wide ? v[j] : 0.0f;
    }
    const unsigned mask = r.target == kNoTarget ? 0u : 0xffffffffu, sign = r.g < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int j = 0; j < 16; j++) w[j] = (pack2<T>(v[2 * j], v[2 * j + 1]) & mask) ^ sign;
}

// ---------------------------------------------------------------- checkpoints
// Eight values a thread and row, four lanes a group.  A block's threads lie
// over whole rows (or over a part of one row) and take kCkptRows of them each,
// so that enough loads are in flight to fill the memory's latency (packing 32768
// x 4096 with 1, 2, 4 and 8 rows a thread: 104, 89, 88 and 121 us).  HBM bounds
// both ways: 407 MB in 74 us (5.5 TB/s) to pack, in 67 us (6.0 TB/s) to read.
constexpr int kCkptThreads = 256, kCkptRows = 4;
struct CkptPlan {
    int64_t rows, cols;
    int chunks;      // of 8 values in a row, groups of 4 (the last ones past the end)
    int per_block;   // chunks of a row that a block takes: a multiple of 4
    int rows_block;  // rows beside each other in a block
    bool vec;        // 16-byte accesses to the 16-bit values
};

template <class T>
__global__ void __launch_bounds__(kCkptThreads) k_pack(const T *x, int64_t ldx, CkptPlan p,
                                                       int8_t *q, uint8_t *ex) {
    after_previous();
    const int r = threadIdx.x / p.per_block, c = blockIdx.y * p.per_block + threadIdx.x % p.per_block;
    const bool on = r < p.rows_block && c < p.chunks;
    uint4 v[kCkptRows];
    int64_t row[kCkptRows];
#pragma unroll
    for (int i = 0; i < kCkptRows; i++) {
        row[i] = ((int64_t)blockIdx.x * kCkptRows + i) * p.rows_block + r;
        v[i] = make_uint4(0, 0, 0, 0);
        if (on && row[i] < p.rows)
            v[i] = load8(reinterpret_cast<const unsigned short *>(x) + row[i] * ldx, (int64_t)c * 8, p.cols, p.vec);
    }
    constexpr bool half = std::is_same<T, __half>::value;
    constexpr int least = half ? 127 - 24 : 1, most = half ? 127 + 10 : 127 + 122;
#pragma unroll
    for (int i = 0; i < kCkptRows; i++) {
        const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        // magnitudes of both 16-bit types are ordered like their bits
        unsigned mx = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                               __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        // a group lies in four neighbouring lanes: per_block and the block's first chunk are multiples of 4
        mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const unsigned top = __float_as_uint(unpack2<T>(max(mx & 0xffffu, mx >> 16)).x);
        // top = f 2^E with 1 <= f < 2; max <= 127 s = (127/64) 2^(e+6)
        int E = (int)(top >> 23) - ((top & 0x7fffffu) > 0x7e0000u ? 5 : 6);  // biased by 127
        E = max(E, least);
        const float inv = __uint_as_float((unsigned)(254 - E) << 23);
        float f[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 t = unpack2<T>(w[k]);
            f[2 * k] = t.x * inv, f[2 * k + 1] = t.y * inv;
        }
        if (__any_sync(0xffffffffu, E == most)) {
            asm volatile("");
#pragma unroll
            for (int k = 0; k < 8; k++)  // 64 s would be past the type's range
                if (E == most) f[k] = fminf(fmaxf(f[k], -63.0f), 63.0f);
        }
        // x / s is exact; adding 1.5 2^23 leaves it rounded, halves to even, in the low byte
        unsigned b[8];
#pragma unroll
        for (int k = 0; k < 8; k++) b[k] = __float_as_uint(f[k] + 12582912.0f);
        uint2 o;
        o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
        if (top >= 0x7f800000u) {
            E = 255;
            o = make_uint2(0, 0);
        }
        if (on && row[i] < p.rows) {
            *reinterpret_cast<uint2 *>(q + (row[i] * p.chunks + c) * 8) = o;
            if ((c & 3) == 0) ex[row[i] * (p.chunks >> 2) + (c >> 2)] = (uint8_t)E;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kCkptThreads) k_unpack(const int8_t *q, const uint8_t *ex,
                                                         CkptPlan p, T *x, int64_t ldx) {
    after_previous();
    const int r = threadIdx.x / p.per_block, c = blockIdx.y * p.per_block + threadIdx.x % p.per_block;
    if (r >= p.rows_block || c >= p.chunks) return;
    uint2 v[kCkptRows];
    unsigned E[kCkptRows];
    int64_t row[kCkptRows];
#pragma unroll
    for (int i = 0; i < kCkptRows; i++) {
        row[i] = ((int64_t)blockIdx.x * kCkptRows + i) * p.rows_block + r;
        if (row[i] < p.rows) {
            v[i] = *reinterpret_cast<const uint2 *>(q + (row[i] * p.chunks + c) * 8);
            E[i] = ex[row[i] * (p.chunks >> 2) + (c >> 2)];
        }
    }
#pragma unroll
    for (int i = 0; i < kCkptRows; i++) {
        if (row[i] >= p.rows) break;
        // a byte b of q as the float 2^23 + (b + 128), less 2^23 + 128
        const float s = E[i] == 255 ? NAN : __uint_as_float(E[i] << 23);
        const unsigned w[2] = {v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u};
        unsigned o[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned lo = __byte_perm(w[k >> 1], 0x4b000000u, k & 1 ? 0x7552 : 0x7550);
            const unsigned hi = __byte_perm(w[k >> 1], 0x4b000000u, k & 1 ? 0x7553 : 0x7551);
            o[k] = pack2<T>((__uint_as_float(lo) - 8388736.0f) * s, (__uint_as_float(hi) - 8388736.0f) * s);
        }
        store8(reinterpret_cast<unsigned short *>(x) + row[i] * ldx, (int64_t)c * 8, p.cols, p.vec,
               make_uint4(o[0], o[1], o[2], o[3]));
    }
}

}  // namespace train
}  // namespace hb
