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

// act(g), and with D its derivative
template <int ACT>
__device__ __forceinline__ float act_f(float g) {
    if (ACT == HELRM_ACT_RELU) return fmaxf(g, 0.0f) + (g != g ? g : 0.0f);  // NaN stays NaN
    if (ACT == HELRM_ACT_SILU) return g / (1.0f + __expf(-g));
    if (ACT == HELRM_ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    return g;
}
template <int ACT>
__device__ __forceinline__ void act_df(float g, float &a, float &d) {
    if (ACT == HELRM_ACT_RELU) {
        a = act_f<ACT>(g);
        d = g > 0.0f ? 1.0f : 0.0f;
    } else if (ACT == HELRM_ACT_SILU) {
        const float s = 1.0f / (1.0f + __expf(-g));
        a = g * s;
        d = s * (1.0f + g * (1.0f - s));
    } else if (ACT == HELRM_ACT_GELU) {
        const float p = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        a = g * p;
        d = p + g * 0.39894228040143268f * __expf(-0.5f * g * g);
    } else {
        a = g;
        d = 1.0f;
    }
}

// ---------------------------------------------------------------- products
enum Epi { EPI_GATED, EPI_GATED_BWD, EPI_STORE, EPI_SUM, EPI_LSE, EPI_Z };
struct EpiArgs {
    void *o0 = nullptr, *o1 = nullptr;  // 16-bit outputs
    int64_t ldo = 0;                    // their row pitch, or that of acc
    int vec = 0;                        // 1: outputs fit 16-byte stores, 2: dh fits 16-byte loads
    const void *dh = nullptr;
    int64_t lddh = 0;
    float *acc = nullptr;               // EPI_SUM: 32-bit sums, [output][part][row][ldo]
    int first = 1;                      // 0: added to what acc holds
    float2 *part = nullptr;             // EPI_LSE: (max, sum) of each [half tile][row]
    float *at = nullptr;                // EPI_LSE: the target's logit
    const int64_t *target = nullptr;
    const float2 *lse = nullptr;        // EPI_Z: the row's (maximum, log of the sum relative to it)
    const float *dloss = nullptr;
    int64_t ignore = 0, col0 = 0;       // first column of the piece in the vocabulary of
    int64_t vocab = 0;                  // this many
    const int *shift = nullptr;         // Z is scaled by 2^shift, undone when the products with it are stored
};

// ---------------------------------------------------------------- the loss
// The row's (maximum, log of the sum relative to it) and loss from the (max,
// sum) of every tile of the vocabulary.  The pair is kept apart: rounded to one
// 32-bit number, a log-sum-exp of some thousands would be off by 2^-13, and so
// would every probability.
// A block takes 32 rows, its 32 warps every 32nd of the parts.
__global__ void __launch_bounds__(1024) k_loss(const float2 *__restrict__ part, int64_t parts,
                                               const float *__restrict__ at, const int64_t *__restrict__ target,
                                               int64_t ignore, int64_t vocab, int64_t M, float *__restrict__ loss,
                                               float2 *__restrict__ lse) {
    __shared__ float2 red[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t m = (int64_t)blockIdx.x * 32 + lane;
    float top = -INFINITY, s = 0.0f;
    auto join = [&](float2 p) {
        const float mx = fmaxf(top, p.x), ref = mx == -INFINITY ? 0.0f : mx;
        s = (top == mx ? s : s * __expf(top - ref)) + (p.x == mx ? p.y : p.y * __expf(p.x - ref));
        top = mx;
    };
    if (m < M) {
#pragma unroll 4
        for (int64_t i = warp; i < parts; i += 32) join(part[i * M + m]);
    }
    red[warp][lane] = make_float2(top, s);
    __syncthreads();
    if (warp || m >= M) return;
    for (int i = 1; i < 32; i++) join(red[i][lane]);
    const float l = logf(s);
    const int64_t t = target[m];
    lse[m] = make_float2(top, l);
    loss[m] = t == ignore ? 0.0f : t < 0 || t >= vocab ? NAN : top - at[m] + l;
}

// fp16 only: the power of two that brings the largest |dloss| of a row that
// takes part to [2^14, 2^15), so that Z keeps the probabilities down to 2^-38.
__global__ void k_loss_shift(const float *__restrict__ dloss, const int64_t *__restrict__ target, int64_t ignore,
                             int64_t M, int *__restrict__ shift) {
    __shared__ float red[32];
    float top = 0.0f;
    for (int64_t m = threadIdx.x; m < M; m += blockDim.x)
        if (target[m] != ignore) top = fmaxf(top, fabsf(dloss[m]));
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (unsigned i = 1; i < blockDim.x / 32; i++) top = fmaxf(top, red[i]);
        *shift = top > 0.0f && top < INFINITY ? max(-100, min(120, 14 - ilogbf(top))) : 0;
    }
}

// ---------------------------------------------------------------- checkpoints
// One warp a group: 32 features, one scale.
template <class T>
__global__ void k_pack(const T *__restrict__ x, int64_t ldx, int64_t M, int64_t K, int8_t *__restrict__ q,
                       uint8_t *__restrict__ ex) {
    const int64_t groups = (K + HELRM_CKPT_GROUP - 1) / HELRM_CKPT_GROUP;
    const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (w >= M * groups) return;
    const int lane = threadIdx.x & 31;
    const int64_t m = w / groups, g = w % groups, k = g * HELRM_CKPT_GROUP + lane;
    const float v = k < K ? to_f(x[m * ldx + k]) : 0.0f;
    const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
    constexpr bool half = sizeof(T) == 2 && std::is_same<T, __half>::value;
    // top = f 2^E with 1 <= f < 2; max <= 127 s = (127/64) 2^(e+6)
    int E = (int)(top >> 23) - ((top & 0x7fffffu) > 0x7e0000u ? 5 : 6);  // biased by 127
    const int least = half ? 127 - 24 : 1, most = half ? 127 + 10 : 127 + 122;
    if (E < least) E = least;
    int r = 0;
    if (top < 0x7f800000u) {
        r = __float2int_rn(v * __uint_as_float((unsigned)(254 - E) << 23));
        if (E == most) r = max(-63, min(63, r));
    } else {
        E = 255;
    }
    q[w * HELRM_CKPT_GROUP + lane] = (int8_t)r;
    if (lane == 0) ex[w] = (uint8_t)E;
}
template <class T>
__global__ void k_unpack(const int8_t *__restrict__ q, const uint8_t *__restrict__ ex, int64_t M, int64_t K,
                         T *__restrict__ x, int64_t ldx) {
    const int64_t groups = (K + HELRM_CKPT_GROUP - 1) / HELRM_CKPT_GROUP;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * K) return;
    const int64_t m = i / K, k = i % K, g = m * groups + k / HELRM_CKPT_GROUP;
    const unsigned E = ex[g];
    x[m * ldx + k] = from_f<T>(E == 255 ? NAN : q[m * groups * HELRM_CKPT_GROUP + k] * __uint_as_float(E << 23));
}

}  // namespace train
}  // namespace hb
