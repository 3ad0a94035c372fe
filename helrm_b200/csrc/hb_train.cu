// hb_train.cu -- the training operators' launches and their extern "C"
// entry points (include/helrm_b200.h).
#include <atomic>
#include <mutex>
#include <type_traits>
#include <vector>

#include "hb_error.hpp"
#include "hb_kernels.cuh"
#include "hb_train.cuh"
#include "hb_train_mma.cuh"
#include "hb_train_loss.cuh"

namespace hb {
namespace train {

// Makes `device` current for a call, and the caller's device again after it.
struct DeviceGuard {
    int old = -1;
    explicit DeviceGuard(int device) {
        cuda_check(cudaGetDevice(&old), "training call");
        if (old == device) {
            old = -1;
            return;
        }
        int n = 0;
        cuda_check(cudaGetDeviceCount(&n), "training call");
        if (device < 0 || device >= n) {
            old = -1;
            HB_THROW(HB_EINVAL, "no CUDA device " + std::to_string(device));
        }
        cuda_check(cudaSetDevice(device), "cudaSetDevice");
    }
    ~DeviceGuard() {
        if (old >= 0) cudaSetDevice(old);
    }
};

// Launches a kernel that may start before the one in front of it in the stream
// has ended and waits for that itself (after_previous): a checkpointed step of
// nine short kernels 114 -> 94 us.
template <class... P, class... A>
static void start(const char *what, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = s;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    cuda_check(cudaLaunchKernelEx(&c, kernel, P(args)...), what);
    count_launches(1);
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

// ---- the process's state: a word of host memory that a kernel whose wait
// ran out writes, and the driver's tensor-map encoder
struct Runtime {
    int *error = nullptr;
    decltype(&cuTensorMapEncodeTiled) encode = nullptr;
    std::atomic<int> sms[64] = {};
};
static Runtime &runtime() {
    static Runtime r;
    static std::mutex mu;
    static std::atomic<bool> ready{false};
    if (!ready) {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready) {
            // allowed while another thread or this one captures a graph
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            cuda_check(cudaThreadExchangeStreamCaptureMode(&mode), "capture mode");
            void *fn = nullptr;
            cudaDriverEntryPointQueryResult found;
            cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
            if (e == cudaSuccess && !r.error) {
                e = cudaHostAlloc(reinterpret_cast<void **>(&r.error), sizeof(int), cudaHostAllocPortable);
                if (e == cudaSuccess) *r.error = 0;
            }
            cudaThreadExchangeStreamCaptureMode(&mode);
            cuda_check(e, "training set-up");
            if (!fn || found != cudaDriverEntryPointSuccess) HB_THROW(HB_ECUDA, "the driver has no tensor maps");
            r.encode = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
            ready = true;
        }
    }
    if (const int code = *static_cast<volatile int *>(r.error)) {
        *static_cast<volatile int *>(r.error) = 0;
        HB_THROW(HB_ECUDA, "an earlier training call gave up waiting in its kernel (code " + std::to_string(code) +
                               "): its results are not valid");
    }
    return r;
}
static int sm_count() {
    int dev = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    std::atomic<int> &known = runtime().sms[dev & 63];
    int n = known;
    if (!n) {
        cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
        known = n;
    }
    return n;
}

// Raises a kernel's shared-memory limit, once for each kernel and device.
template <auto KERNEL>
static void raise_shared_memory(int bytes) {
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    if (set >> (dev & 63) & 1) return;
    cuda_check(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory");
    set |= (uint64_t)1 << (dev & 63);
}

// A row-major 16-bit matrix.
struct Matrix {
    const void *p = nullptr;
    int64_t rows = 0, cols = 0, ld = 0;
};
// Row pitch of the workspace's matrices: whole 128-byte lines, so that a tile's
// rows touch no line twice (gated forward of 2048 x 1000 x 1536 with rows of
// 2000 bytes 18.3 us, of 2048 bytes 15.0), for narrow rows whole 16 bytes.
static int64_t pitch(int64_t cols) { return pad(cols, cols > 64 ? 64 : 8); }
static bool fits_vectors(const void *p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

// Operands that the TMA unit can read: what lies on 16-byte boundaries as it
// is, anything else copied into the workspace first.
struct Operands {
    Workspace &w;
    struct Copy {
        Matrix from;
        unsigned short *to;
    };
    std::vector<Copy> copies;
    explicit Operands(Workspace &ws) : w(ws) {}
    Matrix fit(Matrix m) {
        if (m.rows <= 1) m.ld = pitch(m.cols);
        if (fits_vectors(m.p, m.ld)) return m;
        const int64_t ld = pitch(m.cols);
        unsigned short *to = w.take<unsigned short>(m.rows * ld);
        copies.push_back({m, to});
        return {to, m.rows, m.cols, ld};
    }
    void copy(cudaStream_t s) const {
        if (copies.empty()) return;
        Repitch p = {};
        int64_t most = 0;
        for (size_t i = 0; i < copies.size(); i++) {
            const Matrix &m = copies[i].from;
            p.from[i] = static_cast<const unsigned short *>(m.p);
            p.to[i] = copies[i].to;
            p.ld[i] = m.ld, p.rows[i] = m.rows, p.cols[i] = m.cols, p.pitch[i] = pitch(m.cols);
            const int64_t n = m.rows * ((m.cols + 7) / 8);
            if (n > most) most = n;
        }
        const unsigned grid = blocks(most, 256) < 8u * 148 ? blocks(most, 256) : 8u * 148;
        start("copy to aligned rows", k_repitch, dim3(grid ? grid : 1, (unsigned)copies.size()), 256, 0, s, p);
    }
};

static CkptPlan ckpt_plan(int64_t rows, int64_t cols, bool vec, dim3 &grid) {
    CkptPlan p;
    p.rows = rows;
    p.cols = cols;
    p.chunks = 4 * (int)blocks(cols, HELRM_CKPT_GROUP);
    p.per_block = p.chunks < kCkptThreads ? p.chunks : kCkptThreads;
    p.rows_block = kCkptThreads / p.per_block;
    p.vec = vec;
    grid = dim3(blocks(rows, (int64_t)p.rows_block * kCkptRows), blocks(p.chunks, p.per_block));
    return p;
}
template <class T>
static void read_checkpoint(const int8_t *q, const uint8_t *ex, int64_t rows, int64_t cols, T *x, int64_t ldx,
                            cudaStream_t s) {
    dim3 grid;
    const CkptPlan p = ckpt_plan(rows, cols, fits_vectors(x, ldx), grid);
    start("read checkpoint", k_unpack<T>, grid, kCkptThreads, 0, s, q, ex, p, x, ldx);
}

static CUtensorMap tensor_map(const Matrix &m, bool bf16, int major) {
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows};
    const cuuint64_t strides[1] = {(cuuint64_t)m.ld * 2};
    const cuuint32_t box[2] = {64, major == K_MAJOR ? 128u : 64u}, steps[2] = {1, 1};
    const CUresult r = runtime().encode(
        &map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(m.p),
        dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) HB_THROW(HB_EINVAL, "no tensor map for a matrix (" + std::to_string((int)r) + ")");
    return map;
}

// One product launch.  a, b (and a1, b1 where used) lie K-major or MN-major:
// a K-major operand has the product's depth in its columns, an MN-major one in
// its rows.
struct Product {
    Matrix a, b, a1, b1;
    int64_t M = 0, N = 0, K = 0, K1 = 0;
    int outputs = 1, splits = 1;
    const LossPlan *plan = nullptr;
    bool plan_k = false;
    EpiArgs e;
    int tile_cols() const { return N <= 128 ? 128 : kCols; }
};
template <class T, int AMAJ, int BMAJ, int EPI, int ACT>
static void launch(const Product &d, cudaStream_t s) {
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr bool dual = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
    ProductArgs p;
    p.a = tensor_map(d.a, bf16, AMAJ);
    p.b = tensor_map(d.b, bf16, BMAJ);
    p.a1 = d.a1.p ? tensor_map(d.a1, bf16, AMAJ) : p.a;
    p.b1 = d.b1.p ? tensor_map(d.b1, bf16, BMAJ) : p.b;
    p.M = d.M;
    p.N = d.N;
    p.tiles_m = (int)blocks(d.M, kRows);
    p.cols = d.tile_cols();
    static_assert(BMAJ == MN_MAJOR || (EPI != EPI_STORE && EPI != EPI_SUM), "a K-major B comes in 256-column tiles");
    p.tiles_n = (int)blocks(d.N, dual ? 128 : EPI == EPI_STORE || EPI == EPI_SUM ? p.cols : kCols);
    p.outputs = d.outputs;
    p.splits = d.splits;
    p.kb = (int)blocks(d.K, kDepth);
    p.kb1 = (int)blocks(d.K1, kDepth);
    p.plan = d.plan;
    p.plan_k = d.plan_k;
    p.e = d.e;
    p.error = runtime().error;
    auto kernel = k_mma_product<T, AMAJ, BMAJ, EPI, ACT>;
    raise_shared_memory<k_mma_product<T, AMAJ, BMAJ, EPI, ACT>>(kProductSmem);
    const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits * p.outputs, pairs = sm_count() / 2;
    require(items < (int64_t)1 << 31, "more than 2^31 tiles in one product");
    start("training product", kernel, dim3((unsigned)(2 * (items < pairs ? items : pairs))), product_threads(EPI),
          kProductSmem, s, p);
}

// Parts of the depth for a product of few tiles: enough to give every SM pair
// one, each at least 4 slices deep, and none below 16 slices, where joining
// costs more than it saves (weight gradients of 512 x 512 x 512, 8 slices: 19.4
// us in two parts, 16.3 in one; its dX, 16 slices: 18.0 in four, 18.5 in two).
static int parts_for(int64_t M, int64_t N, int64_t depth, int outputs) {
    const int64_t tiles = (int64_t)blocks(M, kRows) * blocks(N, kCols) * outputs, slices = blocks(depth, kDepth);
    const int64_t n = 74 / tiles < slices / 4 ? 74 / tiles : slices / 4;
    return n > 1 && slices >= 16 ? (int)n : 1;
}
template <class T>
static void join(const JoinArgs &j, void *out, cudaStream_t s) {
    T *o = static_cast<T *>(out);
    if (j.parts > 8)
        start("join parts", k_join<T, true>, blocks(j.M * (j.ld / 4), 32), 256, 0, s, j, o);
    else
        start("join parts", k_join<T, false>, blocks(j.M * (j.ld / 4), 256), 256, 0, s, j, o);
}
// D = A B^T (+ A1 B1^T), or with outputs = 2 also A1 B^T, as dense 16-bit rows
// at out[0], out[1]; the sums of a split depth are joined in acc.
template <class T, int AMAJ, int BMAJ>
static void product_out(Product d, void *const *out, float *acc, cudaStream_t s) {
    if (d.splits == 1) {
        d.e.o0 = out[0];
        d.e.o1 = d.outputs > 1 ? out[1] : nullptr;
        d.e.ldo = d.N;
        d.e.vec = fits_vectors(out[0], d.N) && (d.outputs == 1 || fits_vectors(out[1], d.N));
        launch<T, AMAJ, BMAJ, EPI_STORE, 0>(d, s);
        return;
    }
    d.e.acc = acc;
    d.e.ldo = pad(d.N, 4);
    launch<T, AMAJ, BMAJ, EPI_SUM, 0>(d, s);
    for (int i = 0; i < d.outputs; i++)
        join<T>({acc + (int64_t)i * d.splits * d.M * d.e.ldo, d.splits, d.M, d.M, d.N, d.e.ldo, d.e.plan, nullptr},
                out[i], s);
}
static int64_t sums(int64_t M, int64_t N, int splits, int outputs) {
    return splits > 1 ? (int64_t)outputs * splits * M * pad(N, 4) : 0;
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

// Whether the loss's gradients come from the kernel that keeps Z in shared
// memory, and its shape.  It wins where every block has whole rounds of
// vocabulary rows to itself and few tokens' dH to write out; the estimates (us)
// are fitted to what both ways measured:
//   tokens x inner x vocab    by pieces   Z in shared memory
//   64 x 16 x 40000               38          22
//   1024 x 16 x 19000             46          36
//   1024 x 64 x 19000             46          57   (149 groups of rows for 148 blocks)
//   8192 x 16 x 32001            352         208
//   8192 x 64 x 19000            260         400
//   8192 x 64 x 131072          1408         901
//   32768 x 64 x 32001          1529        1640   (1.2 GB of partial sums)
struct Narrow {
    bool on = false;
    int depth = 0, group = 0, grid = 0;
};
static Narrow narrow(int64_t tokens, int64_t inner, int64_t vocab) {
    Narrow n;
    if (inner > kNarrow) return n;
    n.depth = (int)pad(inner, 16);
    n.group = 128 / n.depth;
    const int64_t groups = blocks(vocab, 128);
    n.grid = (int)(groups < 148 ? groups : 148);
    const double t = (double)pad(tokens, 128), rows = 128.0 * (double)blocks(groups, 148) * 148;
    const double sums = 4.0 * n.grid * t * n.depth;  // bytes of the blocks' dH
    const double here = 12 + t * rows * (3.4e-7 + 8e-9 * n.depth) + 2 * sums / 5e6;
    const double pieces = 20 + 1.35e-6 * t * (double)vocab;
    n.on = here < pieces && sums <= 512e6;
    return n;
}

// The tensor cores cut a sum's last bits off at every 16-deep step, towards
// zero: a logit comes out short by 1.52e-8 of itself a step on average (a row's
// largest logit by 0.48e-6, 0.97e-6, 1.99e-6, 3.87e-6 at 512, 1024, 2048, 4096
// features, whatever its size, where rounding to nearest would leave 1e-7).
// Multiplying by this takes the loss at 4096 features from 1.5e-6 off to the
// noise of 32 bits; it costs nothing, being part of a multiplication that is
// there.  It is 1 for narrow rows, whose gradients' kernel has no use for it.
static float logit_scale(int64_t inner) {
    return inner <= kNarrow ? 1.0f : (float)(1.0 + 1.52e-8 * (double)blocks(inner, 16));
}

// Columns of a vocabulary piece: Z of a piece takes at most 512 MiB (256 MiB:
// 907 us for 4096 x 128 x 131072 where 704 are reached with 1 GiB, 64 MiB:
// 1140), in whole rounds of the SM pairs for dW where that many fit.
static int64_t piece_columns(int64_t tokens, int64_t vocab) {
    const int64_t most = ((int64_t)256 << 20) / (tokens > 0 ? tokens : 1), round = 74 * kCols;
    int64_t c = most / 256 * 256;
    if (most >= round)
        c = most / round * round;
    else if (most >= round / 2)
        c = round / 2;
    if (c < 2048) c = 2048;
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
        Operands in(w);
        Product d;
        d.a = in.fit({x, tokens, inner, ldx});
        d.b = in.fit({wg, width, inner, ldg});
        d.b1 = in.fit({wu, width, inner, ldu});
        if (sized(w, ws_bytes) || tokens == 0) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        in.copy(s);
        d.M = tokens, d.N = width, d.K = inner;
        d.e.o0 = h;
        d.e.ldo = width;
        d.e.vec = fits_vectors(h, width);
        by_dtype(dtype, [&](auto t) {
            by_act(act, [&](auto a) { launch<decltype(t), K_MAJOR, K_MAJOR, EPI_GATED, decltype(a)::value>(d, s); });
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
            require(inner <= 1 << 26 && (tokens == 0 || (q && ex && ((uintptr_t)q & 15) == 0)),
                    "neither x nor an aligned checkpoint is given");
        check_matrix(wg, ldg, inner, width);
        check_matrix(wu, ldu, inner, width);
        require(dx || dwg || dwu, "no output is asked for");
        require(act >= 0 && act <= HELRM_ACT_GELU, "unknown activation");
        Workspace w{static_cast<char *>(ws)};
        Operands in(w);
        const int64_t ldd = pitch(width);
        uint16_t *dg = w.take<uint16_t>(tokens * ldd), *du = w.take<uint16_t>(tokens * ldd);
        uint16_t *read = x ? nullptr : w.take<uint16_t>(tokens * pitch(inner));
        const Matrix mx = x ? in.fit({x, tokens, inner, ldx}) : Matrix{read, tokens, inner, pitch(inner)};
        const Matrix mg = in.fit({wg, width, inner, ldg}), mu = in.fit({wu, width, inner, ldu});
        const Matrix mdg{dg, tokens, width, ldd}, mdu{du, tokens, width, ldd};
        const int both = dwg && dwu ? 2 : 1;
        const int parts_x = dx ? parts_for(tokens, inner, 2 * width, 1) : 1;
        const int parts_w = dwg || dwu ? parts_for(width, inner, tokens, both) : 1;
        const int64_t sums_x = sums(tokens, inner, parts_x, 1), sums_w = sums(width, inner, parts_w, both);
        float *acc = w.take<float>(sums_x > sums_w ? sums_x : sums_w);
        if (sized(w, ws_bytes)) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        if (tokens == 0) {
            for (void *p : {dwg, dwu})
                if (p) cuda_check(cudaMemsetAsync(p, 0, (size_t)width * inner * 2, s), "zero gradient");
            return;
        }
        in.copy(s);
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            if (!x) read_checkpoint<T>(q, ex, tokens, inner, reinterpret_cast<T *>(read), pitch(inner), s);
            Product d;
            d.a = mx, d.b = mg, d.b1 = mu;
            d.M = tokens, d.N = width, d.K = inner;
            d.e.o0 = dg;
            d.e.o1 = du;
            d.e.ldo = ldd;
            d.e.dh = dh;
            d.e.lddh = lddh;
            d.e.vec = 1 | (fits_vectors(dh, lddh) ? 2 : 0);
            by_act(act, [&](auto a) { launch<T, K_MAJOR, K_MAJOR, EPI_GATED_BWD, decltype(a)::value>(d, s); });
            if (dx) {
                Product g;
                g.a = mdg, g.b = mg, g.a1 = mdu, g.b1 = mu;
                g.M = tokens, g.N = inner, g.K = g.K1 = width;
                g.splits = parts_x;
                product_out<T, K_MAJOR, MN_MAJOR>(g, &dx, acc, s);
            }
            if (dwg || dwu) {
                Product g;
                g.a = dwg ? mdg : mdu, g.a1 = mdu, g.b = mx;
                g.M = width, g.N = inner, g.K = tokens;
                g.outputs = both;
                g.splits = parts_w;
                void *out[2] = {dwg ? dwg : dwu, dwu};
                product_out<T, MN_MAJOR, MN_MAJOR>(g, out, acc, s);
            }
        });
    });
}

HB_API int helrm_PackCheckpoint(int device, int dtype, int64_t tokens, int64_t inner, const void *x, int64_t ldx,
                                int8_t *q, uint8_t *ex, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, 1);
        require(inner <= 1 << 26, "rows of a checkpoint have at most 2^26 features");
        check_matrix(x, ldx, inner, tokens);
        if (tokens == 0) return;
        require(q && ex && ((uintptr_t)q & 15) == 0, "q or e is NULL, or q is not 16-byte aligned");
        DeviceGuard dev(device);
        runtime();
        dim3 grid;
        const CkptPlan p = ckpt_plan(tokens, inner, fits_vectors(x, tokens > 1 ? ldx : pitch(inner)), grid);
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            start("pack checkpoint", k_pack<T>, grid, kCkptThreads, 0, (cudaStream_t)stream, static_cast<const T *>(x), ldx,
                  p, q, ex);
        });
    });
}

HB_API int helrm_UnpackCheckpoint(int device, int dtype, int64_t tokens, int64_t inner, const int8_t *q,
                                  const uint8_t *ex, void *x, void *stream) {
    return guard([&] {
        check_sizes(dtype, tokens, inner, 1);
        require(inner <= 1 << 26, "rows of a checkpoint have at most 2^26 features");
        if (tokens == 0) return;
        require(q && ex && x && ((uintptr_t)q & 15) == 0, "q, e or x is NULL, or q is not 16-byte aligned");
        DeviceGuard dev(device);
        runtime();
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            read_checkpoint<T>(q, ex, tokens, inner, static_cast<T *>(x), inner, (cudaStream_t)stream);
        });
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
        Operands in(w);
        const Matrix mh = in.fit({h, tokens, inner, ldh}), mw = in.fit({wt, vocab, inner, ldw});
        const int64_t parts = 2 * (int64_t)blocks(vocab, kCols);
        const int64_t joined = parts > kLossParts ? blocks(parts, kLossParts) : 0;
        // tokens at a time: their statistics take at most 512 MiB (or those of 4096 tokens)
        const int64_t most = ((int64_t)64 << 20) / (parts + joined) / 256 * 256;
        const int64_t piece = tokens < 4096 || tokens < most ? tokens : most < 4096 ? 4096 : most;
        float2 *part = w.take<float2>(parts * piece), *few = w.take<float2>(joined * piece);
        float *at = w.take<float>(piece);
        if (sized(w, ws_bytes) || tokens == 0) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        in.copy(s);
        for (int64_t m0 = 0; m0 < tokens; m0 += piece) {
            const int64_t n = tokens - m0 < piece ? tokens - m0 : piece;
            Product d;
            d.a = {static_cast<const uint16_t *>(mh.p) + m0 * mh.ld, n, inner, mh.ld};
            d.b = mw;
            d.M = n, d.N = vocab, d.K = inner;
            d.e.part = part;
            d.e.at = at;
            d.e.target = targets + m0;
            d.e.grow = logit_scale(inner);
            by_dtype(dtype, [&](auto t) { launch<decltype(t), K_MAJOR, K_MAJOR, EPI_LSE, 0>(d, s); });
            const float *none = nullptr;
            const int64_t *no_targets = nullptr;
            if (joined)
                start("loss", k_loss<false>, dim3(blocks(n, 32), (unsigned)joined), 1024, 0, s, part, parts, none,
                      no_targets, (int64_t)0, (int64_t)0, n, (float *)nullptr, few);
            start("loss", k_loss<true>, blocks(n, 32), 1024, 0, s, joined ? few : part, joined ? joined : parts, at,
                  targets + m0, ignore_index, vocab, n, loss + m0, reinterpret_cast<float2 *>(lse) + m0);
        }
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
        Operands in(w);
        const Matrix mw = in.fit({wt, vocab, inner, ldw});
        const bool scaled = dtype == HELRM_FP16;
        const int64_t cap = pad(tokens, 256);  // the rows that take part, filled up
        uint16_t *hc = w.take<uint16_t>(cap * pitch(inner));
        const Matrix mh{hc, cap, inner, pitch(inner)};
        LossRow *rows = w.take<LossRow>(cap);
        int *src = w.take<int>(cap), *pos = w.take<int>(tokens);
        LossPlan *plan = w.take<LossPlan>(1);
        auto prepare = [&](cudaStream_t s) {
            in.copy(s);
            LossRows r = {dloss, targets, reinterpret_cast<const float2 *>(lse), ignore_index, vocab, tokens,
                          static_cast<const unsigned short *>(h), ldh, inner, fits_vectors(h, ldh), scaled, 0, rows, src,
                          pos, plan, hc, pitch(inner)};
            // 32 rows a block, or at most 512 blocks
            r.per = (int)(cap > 32 * 512 ? pad(blocks(cap, 512), 32) : 32);
            start("loss rows", k_loss_rows, blocks(cap, r.per), 1024, 0, s, r);
        };
        const Narrow nr = narrow(tokens, inner, vocab);
        if (nr.on) {
            const int groups = (int)blocks(blocks(tokens, 128), nr.group);
            float *part = w.take<float>((int64_t)nr.grid * cap * nr.depth);
            float *acc = w.take<float>(groups > 1 ? vocab * nr.depth : 0);
            void *dws = dw ? dw : w.take<uint16_t>(vocab * inner);
            if (sized(w, ws_bytes)) return;
            DeviceGuard dev(device);
            cudaStream_t s = (cudaStream_t)stream;
            if (tokens == 0) {
                if (dw) cuda_check(cudaMemsetAsync(dw, 0, (size_t)vocab * inner * 2, s), "zero gradient");
                return;
            }
            prepare(s);
            by_dtype(dtype, [&](auto t) {
                typedef decltype(t) T;
                NarrowArgs a;
                a.h = tensor_map(mh, std::is_same<T, __nv_bfloat16>::value, K_MAJOR);
                a.w = tensor_map(mw, std::is_same<T, __nv_bfloat16>::value, K_MAJOR);
                a.capacity = cap, a.vocab = vocab;
                a.inner = (int)inner, a.depth = nr.depth, a.group = nr.group;
                a.rows = rows;
                a.lse = reinterpret_cast<const float2 *>(lse);
                a.src = src;
                a.plan = plan;
                a.dw = dws;
                a.acc_w = acc;
                a.part_h = part;
                a.error = runtime().error;
                raise_shared_memory<k_loss_grads_narrow<T>>(kNarrowSmem);
                start("loss gradients", k_loss_grads_narrow<T>, nr.grid, kNarrowThreads, kNarrowSmem, s, a);
                if (dh) join<T>({part, nr.grid, cap, tokens, inner, nr.depth, plan, pos}, dh, s);
            });
            return;
        }
        const int64_t cols = piece_columns(cap, vocab), ldz = pitch(cols), lda = pad(inner, 4);
        uint16_t *z = w.take<uint16_t>(cap * ldz);
        // dh is a 32-bit sum over the pieces, for each part of a piece's depth, of the rows that take part
        const int parts_h = dh ? parts_for(cap, inner, cols, 1) : 1, parts_w = dw ? parts_for(cols, inner, cap, 1) : 1;
        float *acc = w.take<float>(dh ? parts_h * cap * lda : 0);
        float *acc_w = w.take<float>(sums(cols, inner, parts_w, 1));
        if (sized(w, ws_bytes)) return;
        DeviceGuard dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        if (tokens == 0) {
            if (dw) cuda_check(cudaMemsetAsync(dw, 0, (size_t)vocab * inner * 2, s), "zero gradient");
            return;
        }
        prepare(s);
        by_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            for (int64_t c0 = 0; c0 < vocab; c0 += cols) {
                const int64_t n = vocab - c0 < cols ? vocab - c0 : cols;
                const Matrix mc{static_cast<const T *>(mw.p) + c0 * mw.ld, n, inner, mw.ld}, mz{z, cap, n, ldz};
                Product d;
                d.a = mh, d.b = mc;
                d.M = cap, d.N = n, d.K = inner;
                d.plan = plan;
                d.e.o0 = z;
                d.e.ldo = ldz;
                d.e.vec = 1;
                d.e.rows = rows;
                d.e.src = src;
                d.e.lse = reinterpret_cast<const float2 *>(lse);
                d.e.col0 = c0;
                d.e.grow = logit_scale(inner);
                launch<T, K_MAJOR, K_MAJOR, EPI_Z, 0>(d, s);
                if (dw) {
                    Product g;
                    g.a = mz, g.b = mh;
                    g.M = n, g.N = inner, g.K = cap;
                    g.splits = parts_w;
                    g.plan = plan;
                    g.plan_k = true;
                    g.e.plan = plan;
                    void *out = static_cast<T *>(dw) + c0 * inner;
                    product_out<T, MN_MAJOR, MN_MAJOR>(g, &out, acc_w, s);
                }
                if (dh) {
                    Product g;
                    g.a = mz, g.b = mc;
                    g.M = cap, g.N = inner, g.K = n;
                    g.plan = plan;
                    // the last piece may be too short for every part: those keep their sums
                    g.splits = parts_h < (int)blocks(n, kDepth) ? parts_h : (int)blocks(n, kDepth);
                    g.e.acc = acc;
                    g.e.ldo = lda;
                    g.e.first = c0 == 0;
                    launch<T, K_MAJOR, MN_MAJOR, EPI_SUM, 0>(g, s);
                }
            }
            if (dh) join<T>({acc, parts_h, cap, tokens, inner, lda, plan, pos}, dh, s);
        });
    });
}
