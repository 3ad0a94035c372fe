// hb_train.cu -- the training operators' launches and their extern "C"
// entry points (include/helrm_b200.h).
#include <type_traits>

#include "hb_error.hpp"
#include "hb_kernels.cuh"
#include "hb_train.cuh"

namespace hb {
namespace train {

// Makes `device` current for a call, and the caller's device again after it.
struct DeviceGuard {
    int old = -1;
    explicit DeviceGuard(int device) {
        int n = 0;
        cuda_check(cudaGetDeviceCount(&n), "training call");
        if (device < 0 || device >= n) HB_THROW(HB_EINVAL, "no CUDA device " + std::to_string(device));
        cuda_check(cudaGetDevice(&old), "cudaGetDevice");
        if (old != device)
            cuda_check(cudaSetDevice(device), "cudaSetDevice");
        else
            old = -1;
    }
    ~DeviceGuard() {
        if (old >= 0) cudaSetDevice(old);
    }
};

static void launched(const char *what) {
    count_launches(1);
    cuda_check(cudaGetLastError(), what);
}

static void require(bool ok, const char *msg) {
    if (!ok) HB_THROW(HB_EINVAL, msg);
}

// Hands out pieces of the caller's workspace, or with base NULL only counts.
struct Workspace {
    char *base;
    size_t used = 0;
    template <class T>
    T *take(int64_t n) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};
// true: only the size was asked for
static bool sized(const Workspace &w, size_t *ws_bytes) {
    require(ws_bytes != nullptr, "ws_bytes is NULL");
    if (!w.base) {
        *ws_bytes = w.used;
        return true;
    }
    require(((uintptr_t)w.base & 255) == 0, "the workspace is not 256-byte aligned");
    require(*ws_bytes >= w.used, "the workspace is too small");
    return false;
}

static int64_t pad(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
static unsigned blocks(int64_t n, int64_t per) { return (unsigned)((n + per - 1) / per); }

static void check_sizes(int dtype, int64_t tokens, int64_t inner, int64_t cols) {
    require(dtype == HELRM_FP16 || dtype == HELRM_BF16, "dtype is neither HELRM_FP16 nor HELRM_BF16");
    require(tokens >= 0 && inner >= 1 && cols >= 1, "sizes: tokens >= 0, the others >= 1");
    const int64_t lim = (int64_t)1 << 30;
    require(tokens <= lim && inner <= lim && cols <= lim, "sizes above 2^30");
}
static void check_matrix(const void *p, int64_t ld, int64_t cols, int64_t rows) {
    require(rows == 0 || p != nullptr, "a matrix pointer is NULL");
    require(((uintptr_t)p & 1) == 0, "a matrix pointer is not aligned to its type");
    require(ld >= cols, "a row pitch is below the number of columns");
}

template <class T, int EPI, int ACT, bool DUAL, bool SECOND>
static void product(View a, View b, View a1, View b1, int64_t M, int64_t N, int64_t K, const EpiArgs &e,
                    cudaStream_t s) {
    const dim3 grid(blocks(M, kTile), blocks(N, kTile));
    k_product<T, EPI, ACT, DUAL, SECOND><<<grid, 256, 0, s>>>(a, b, a1, b1, M, N, K, e);
    launched("training product");
}

template <class F>
static void by_dtype(int dtype, F &&f) {
    if (dtype == HELRM_FP16)
        f(__half());
    else
        f(__nv_bfloat16());
}
template <class F>
static void by_act(int act, F &&f) {
    switch (act) {
        case HELRM_ACT_IDENTITY: f(std::integral_constant<int, HELRM_ACT_IDENTITY>()); break;
        case HELRM_ACT_RELU: f(std::integral_constant<int, HELRM_ACT_RELU>()); break;
        case HELRM_ACT_SILU: f(std::integral_constant<int, HELRM_ACT_SILU>()); break;
        case HELRM_ACT_GELU: f(std::integral_constant<int, HELRM_ACT_GELU>()); break;
        default: HB_THROW(HB_EINVAL, "unknown activation");
    }
}

// Columns of a vocabulary piece: Z of a piece takes at most 256 MiB.
static int64_t piece_columns(int64_t tokens, int64_t vocab) {
    const int64_t most = ((int64_t)128 << 20) / (tokens > 0 ? tokens : 1);
    const int64_t c = most < 2048 ? 2048 : most / 256 * 256;
    return c < vocab ? c : vocab;
}

}  // namespace train
}  // namespace hb

using namespace hb;
using namespace hb::train;

HB_API int helrm_GatedForward(int device, int dtype, int act, int64_t tokens, int64_t inner, int64_t width,
                              const void *x, int64_t ldx, const void *wg, int64_t ldg, const void *wu, int64_t ldu,
                              void *h, void *ws, size_t *ws_bytes, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, width);
        check_matrix(x, ldx, inner, tokens);
        check_matrix(wg, ldg, inner, width);
        check_matrix(wu, ldu, inner, width);
        require(tokens == 0 || h != nullptr, "the output pointer is NULL");
        require(act >= 0 && act <= HELRM_ACT_GELU, "unknown activation");
        Workspace w{static_cast<char *>(ws)};
        if (sized(w, ws_bytes) || tokens == 0) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        by_dtype(dtype, [&](auto t) {
            by_act(act, [&](auto a) {
                EpiArgs e;
                e.o0 = h;
                e.ldo = width;
                product<decltype(t), EPI_GATED, decltype(a)::value, true, false>(
                    {x, ldx, 1}, {wg, ldg, 1}, {}, {wu, ldu, 1}, tokens, width, inner, e, s);
            });
        });
    });
}

HB_API int helrm_GatedBackward(int device, int dtype, int act, int64_t tokens, int64_t inner, int64_t width,
                               const void *dh, int64_t lddh, const void *x, int64_t ldx, const int8_t *q,
                               const uint8_t *ex, const void *wg, int64_t ldg, const void *wu, int64_t ldu, void *dx,
                               void *dwg, void *dwu, void *ws, size_t *ws_bytes, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, width);
        check_matrix(dh, lddh, width, tokens);
        if (x)
            check_matrix(x, ldx, inner, tokens);
        else
            require(tokens == 0 || (q && ex && ((uintptr_t)q & 15) == 0), "neither x nor an aligned checkpoint is given");
        check_matrix(wg, ldg, inner, width);
        check_matrix(wu, ldu, inner, width);
        require(dx || dwg || dwu, "no output is asked for");
        require(act >= 0 && act <= HELRM_ACT_GELU, "unknown activation");
        Workspace w{static_cast<char *>(ws)};
        const int64_t ldd = pad(width, 8), ldk = pad(inner, 8);
        uint16_t *dg = w.take<uint16_t>(tokens * ldd), *du = w.take<uint16_t>(tokens * ldd);
        uint16_t *xr = x ? nullptr : w.take<uint16_t>(tokens * ldk);
        if (sized(w, ws_bytes)) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        if (tokens == 0) {
            for (void *p : {dwg, dwu})
                if (p) cuda_check(cudaMemsetAsync(p, 0, (size_t)width * inner * 2, s), "zero gradient");
            return;
        }
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            const void *xp = x;
            int64_t lx = ldx;
            if (!x) {
                k_unpack<T><<<blocks(tokens * inner, 256), 256, 0, s>>>(q, ex, tokens, inner, reinterpret_cast<T *>(xr),
                                                                        ldk);
                launched("read checkpoint");
                xp = xr;
                lx = ldk;
            }
            by_act(act, [&](auto a) {
                EpiArgs e;
                e.o0 = dg;
                e.o1 = du;
                e.ldo = ldd;
                e.dh = dh;
                e.lddh = lddh;
                product<T, EPI_GATED_BWD, decltype(a)::value, true, false>({xp, lx, 1}, {wg, ldg, 1}, {}, {wu, ldu, 1},
                                                                           tokens, width, inner, e, s);
            });
            EpiArgs e;
            e.ldo = inner;
            e.o0 = dx;
            if (dx)
                product<T, EPI_STORE, 0, false, true>({dg, ldd, 1}, {wg, 1, ldg}, {du, ldd, 1}, {wu, 1, ldu}, tokens,
                                                      inner, width, e, s);
            e.o0 = dwg;
            if (dwg)
                product<T, EPI_STORE, 0, false, false>({dg, 1, ldd}, {xp, 1, lx}, {}, {}, width, inner, tokens, e, s);
            e.o0 = dwu;
            if (dwu)
                product<T, EPI_STORE, 0, false, false>({du, 1, ldd}, {xp, 1, lx}, {}, {}, width, inner, tokens, e, s);
        });
    });
}

HB_API int helrm_PackCheckpoint(int device, int dtype, int64_t tokens, int64_t inner, const void *x, int64_t ldx,
                                int8_t *q, uint8_t *ex, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, 1);
        check_matrix(x, ldx, inner, tokens);
        if (tokens == 0) return;
        require(q && ex && ((uintptr_t)q & 15) == 0, "q or e is NULL, or q is not 16-byte aligned");
        DeviceGuard dev(device);
        const int64_t groups = blocks(inner, HELRM_CKPT_GROUP);
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            k_pack<T><<<blocks(tokens * groups * 32, 256), 256, 0, (cudaStream_t)stream>>>(
                static_cast<const T *>(x), ldx, tokens, inner, q, ex);
        });
        launched("pack checkpoint");
    });
}

HB_API int helrm_UnpackCheckpoint(int device, int dtype, int64_t tokens, int64_t inner, const int8_t *q,
                                  const uint8_t *ex, void *x, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, 1);
        if (tokens == 0) return;
        require(q && ex && x && ((uintptr_t)q & 15) == 0, "q, e or x is NULL, or q is not 16-byte aligned");
        DeviceGuard dev(device);
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            k_unpack<T><<<blocks(tokens * inner, 256), 256, 0, (cudaStream_t)stream>>>(q, ex, tokens, inner,
                                                                                      static_cast<T *>(x), inner);
        });
        launched("unpack checkpoint");
    });
}

HB_API int helrm_VocabularyLossForward(int device, int dtype, int64_t tokens, int64_t inner, int64_t vocab,
                                       const void *h, int64_t ldh, const void *wt, int64_t ldw, const int64_t *targets,
                                       int64_t ignore_index, float *loss, float *lse, void *ws, size_t *ws_bytes,
                                       void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, vocab);
        check_matrix(h, ldh, inner, tokens);
        check_matrix(wt, ldw, inner, vocab);
        require(tokens == 0 || (targets && loss && lse), "targets, loss or lse is NULL");
        require(((uintptr_t)lse & 7) == 0, "lse is not 8-byte aligned");
        Workspace w{static_cast<char *>(ws)};
        const int64_t tiles = blocks(vocab, kTile);
        float2 *part = w.take<float2>(tiles * tokens);
        float *at = w.take<float>(tokens);
        if (sized(w, ws_bytes) || tokens == 0) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        by_dtype(dtype, [&](auto t) {
            EpiArgs e;
            e.part = part;
            e.at = at;
            e.target = targets;
            product<decltype(t), EPI_LSE, 0, false, false>({h, ldh, 1}, {wt, ldw, 1}, {}, {}, tokens, vocab, inner, e,
                                                           s);
        });
        k_loss<<<blocks(tokens, 128), 128, 0, s>>>(part, tiles, at, targets, ignore_index, vocab, tokens, loss,
                                                     reinterpret_cast<float2 *>(lse));
        launched("loss");
    });
}

HB_API int helrm_VocabularyLossBackward(int device, int dtype, int64_t tokens, int64_t inner, int64_t vocab,
                                        const float *dloss, const void *h, int64_t ldh, const void *wt, int64_t ldw,
                                        const int64_t *targets, const float *lse, int64_t ignore_index, void *dh,
                                        void *dw, void *ws, size_t *ws_bytes, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, vocab);
        check_matrix(h, ldh, inner, tokens);
        check_matrix(wt, ldw, inner, vocab);
        require(tokens == 0 || (targets && dloss && lse), "dloss, targets or lse is NULL");
        require(((uintptr_t)lse & 7) == 0, "lse is not 8-byte aligned");
        require(dh || dw, "no output is asked for");
        Workspace w{static_cast<char *>(ws)};
        const int64_t cols = piece_columns(tokens, vocab), ldz = pad(cols, 8);
        uint16_t *z = w.take<uint16_t>(tokens * ldz);
        float *acc = w.take<float>(cols < vocab ? tokens * inner : 0);
        int *shift = w.take<int>(dtype == HELRM_FP16 ? 1 : 0);
        if (sized(w, ws_bytes)) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        if (tokens == 0) {
            if (dw) cuda_check(cudaMemsetAsync(dw, 0, (size_t)vocab * inner * 2, s), "zero gradient");
            return;
        }
        const bool scaled = dtype == HELRM_FP16;
        if (scaled) {
            k_loss_shift<<<1, 1024, 0, s>>>(dloss, targets, ignore_index, tokens, shift);
            launched("loss shift");
        }
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            for (int64_t c0 = 0; c0 < vocab; c0 += cols) {
                const int64_t n = vocab - c0 < cols ? vocab - c0 : cols;
                const T *wc = static_cast<const T *>(wt) + c0 * ldw;
                EpiArgs e;
                e.shift = scaled ? shift : nullptr;
                e.o0 = z;
                e.ldo = ldz;
                e.target = targets;
                e.lse = reinterpret_cast<const float2 *>(lse);
                e.dloss = dloss;
                e.ignore = ignore_index;
                e.col0 = c0;
                e.vocab = vocab;
                product<T, EPI_Z, 0, false, false>({h, ldh, 1}, {wc, ldw, 1}, {}, {}, tokens, n, inner, e, s);
                e.ldo = inner;
                e.o0 = static_cast<T *>(dw) + c0 * inner;
                if (dw)
                    product<T, EPI_STORE, 0, false, false>({z, 1, ldz}, {h, 1, ldh}, {}, {}, n, inner, tokens, e, s);
                if (!dh) continue;
                e.o0 = dh;
                e.acc = acc;
                e.first = c0 == 0;
                e.last = c0 + n == vocab;
                product<T, EPI_STORE, 0, false, false>({z, ldz, 1}, {wc, 1, ldw}, {}, {}, tokens, inner, n, e, s);
            }
        });
    });
}
