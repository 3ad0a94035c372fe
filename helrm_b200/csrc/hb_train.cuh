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
// A strided operand: element (r, k) at p[r * sr + k * sk].
struct View {
    const void *p;
    int64_t sr, sk;
};
enum Epi { EPI_GATED, EPI_GATED_BWD, EPI_STORE, EPI_LSE, EPI_Z };
struct EpiArgs {
    void *o0 = nullptr, *o1 = nullptr;  // outputs, dense rows of ldo
    int64_t ldo = 0;
    const void *dh = nullptr;
    int64_t lddh = 0;
    float *acc = nullptr;               // EPI_STORE: 32-bit running sum over the pieces
    int first = 1, last = 1;
    float2 *part = nullptr;             // EPI_LSE: (max, sum) of each [tile][row]
    float *at = nullptr;                // EPI_LSE: the target's logit
    const int64_t *target = nullptr;
    const float2 *lse = nullptr;        // EPI_Z: the row's (maximum, log of the sum relative to it)
    const float *dloss = nullptr;
    int64_t ignore = 0, col0 = 0;       // first column of the piece in the vocabulary of
    int64_t vocab = 0;                  // this many
    const int *shift = nullptr;         // Z is scaled by 2^shift, undone in EPI_STORE
};

constexpr int kTile = 64, kStep = 16;

// D[m][n] = sum_k A(m, k) B(n, k) over one 64 x 64 tile, 4 x 4 a thread, the
// operands staged as 32-bit floats.  DUAL: a second product with B1.  SECOND:
// a second pair of operands added to the same sum.
template <class T, int EPI, int ACT, bool DUAL, bool SECOND>
__global__ void __launch_bounds__(256) k_product(View a, View b, View a1, View b1, int64_t M, int64_t N, int64_t K,
                                                 EpiArgs e) {
    __shared__ float sa[kStep][kTile + 4], sb[kStep][kTile + 4], sc[DUAL ? kStep : 1][kTile + 4];
    __shared__ float red[EPI == EPI_LSE ? kTile : 1][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
    float acc[4][4] = {}, acc1[4][4] = {};
    for (int pass = 0; pass < (SECOND ? 2 : 1); pass++) {
        const View va = pass ? a1 : a, vb = pass ? b1 : b;
        for (int64_t k0 = 0; k0 < K; k0 += kStep) {
            for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
                const bool ka = va.sk == 1, kb = vb.sk == 1;
                const int ra = ka ? i / kStep : i % kTile, ca = ka ? i % kStep : i / kTile;
                const int rb = kb ? i / kStep : i % kTile, cb = kb ? i % kStep : i / kTile;
                sa[ca][ra] = m0 + ra < M && k0 + ca < K
                                 ? to_f(static_cast<const T *>(va.p)[(m0 + ra) * va.sr + (k0 + ca) * va.sk])
                                 : 0.0f;
                sb[cb][rb] = n0 + rb < N && k0 + cb < K
                                 ? to_f(static_cast<const T *>(vb.p)[(n0 + rb) * vb.sr + (k0 + cb) * vb.sk])
                                 : 0.0f;
                if (DUAL)
                    sc[cb][rb] = n0 + rb < N && k0 + cb < K
                                     ? to_f(static_cast<const T *>(b1.p)[(n0 + rb) * b1.sr + (k0 + cb) * b1.sk])
                                     : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kStep; k++) {
                float x[4], y[4], z[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = sa[k][ty * 4 + i];
                    y[i] = sb[k][tx * 4 + i];
                    if (DUAL) z[i] = sc[k][tx * 4 + i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
                        if (DUAL) acc1[i][j] = fmaf(x[i], z[j], acc1[i][j]);
                    }
            }
            __syncthreads();
        }
    }
    if (EPI == EPI_LSE) {
        for (int i = 0; i < 4; i++) {
            const int64_t m = m0 + ty * 4 + i;
            float top = -INFINITY;
            for (int j = 0; j < 4; j++)
                if (n0 + tx * 4 + j < N) top = fmaxf(top, acc[i][j]);
            red[ty * 4 + i][tx] = top;
            if (m < M) {
                const int64_t t = e.target[m] - n0 - tx * 4;
                for (int j = 0; j < 4; j++)
                    if (t == j && n0 + tx * 4 + j < N) e.at[m] = acc[i][j];
            }
        }
        __syncthreads();
        for (int i = 0; i < 4; i++) {
            float top = -INFINITY;
            for (int j = 0; j < 16; j++) top = fmaxf(top, red[ty * 4 + i][j]);
            float s = 0.0f;
            for (int j = 0; j < 4; j++)
                if (n0 + tx * 4 + j < N) s += top == -INFINITY && acc[i][j] == top ? 0.0f : __expf(acc[i][j] - top);
            for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const int64_t m = m0 + ty * 4 + i;
            if (tx == 0 && m < M) e.part[blockIdx.y * M + m] = make_float2(top, s);
        }
        return;
    }
    for (int i = 0; i < 4; i++) {
        const int64_t m = m0 + ty * 4 + i;
        if (m >= M) continue;
        int64_t t = -1;
        float g = 0.0f;
        float2 lse = make_float2(0.0f, 0.0f);
        if (EPI == EPI_Z) {
            t = e.target[m];
            if (t != e.ignore) g = e.dloss[m], lse = e.lse[m];
            if (e.shift) g = ldexpf(g, *e.shift);
        }
        for (int j = 0; j < 4; j++) {
            const int64_t n = n0 + tx * 4 + j;
            if (n >= N) continue;
            if (EPI == EPI_GATED) static_cast<T *>(e.o0)[m * e.ldo + n] = from_f<T>(act_f<ACT>(acc[i][j]) * acc1[i][j]);
            if (EPI == EPI_GATED_BWD) {
                const float dh = to_f(static_cast<const T *>(e.dh)[m * e.lddh + n]);
                float v, d;
                act_df<ACT>(acc[i][j], v, d);
                static_cast<T *>(e.o0)[m * e.ldo + n] = from_f<T>(dh * acc1[i][j] * d);
                static_cast<T *>(e.o1)[m * e.ldo + n] = from_f<T>(dh * v);
            }
            if (EPI == EPI_Z) {
                float z = 0.0f;
                if (t != e.ignore) {
                    const float x = acc[i][j] - lse.x - lse.y;
                    z = e.col0 + n == t ? expm1f(x) : __expf(x);
                    z = t < 0 || t >= e.vocab ? NAN : z * g;
                }
                static_cast<T *>(e.o0)[m * e.ldo + n] = from_f<T>(z);
            }
            if (EPI == EPI_STORE) {
                float v = acc[i][j];
                if (!e.first) v += e.acc[m * N + n];
                if (e.last)
                    static_cast<T *>(e.o0)[m * e.ldo + n] = from_f<T>(e.shift ? ldexpf(v, -*e.shift) : v);
                else
                    e.acc[m * N + n] = v;
            }
        }
    }
}

// ---------------------------------------------------------------- the loss
// The row's (maximum, log of the sum relative to it) and loss from the (max,
// sum) of every tile of the vocabulary.  The pair is kept apart: rounded to one
// 32-bit number, a log-sum-exp of some thousands would be off by 2^-13, and so
// would every probability.
__global__ void k_loss(const float2 *__restrict__ part, int64_t tiles, const float *__restrict__ at,
                       const int64_t *__restrict__ target, int64_t ignore, int64_t vocab, int64_t M,
                       float *__restrict__ loss, float2 *__restrict__ lse) {
    const int64_t m = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (m >= M) return;
    float top = -INFINITY;
    for (int64_t i = 0; i < tiles; i++) top = fmaxf(top, part[i * M + m].x);
    float s = 0.0f;
    for (int64_t i = 0; i < tiles; i++) {
        const float2 p = part[i * M + m];
        s += p.x == -INFINITY ? p.y : p.y * __expf(p.x - top);
    }
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
        *shift = top > 0.0f && top < INFINITY ? 14 - ilogbf(top) : 0;
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
