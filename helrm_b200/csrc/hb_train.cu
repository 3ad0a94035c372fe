// hb_train.cu -- the training operators' launches and their extern "C"
// entry points (include/helrm_b200.h).
#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>
#include <utility>
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

// ---- the process's state: for each device a word of host memory that a kernel
// whose wait ran out writes, and the driver's tensor-map encoder
struct Runtime {
    int *errors = nullptr;
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
            if (e == cudaSuccess && !r.errors) {
                e = cudaHostAlloc(reinterpret_cast<void **>(&r.errors), 64 * sizeof(int), cudaHostAllocPortable);
                if (e == cudaSuccess) std::memset(r.errors, 0, 64 * sizeof(int));
            }
            cudaThreadExchangeStreamCaptureMode(&mode);
            cuda_check(e, "training set-up");
            if (!fn || found != cudaDriverEntryPointSuccess) HB_THROW(HB_ECUDA, "the driver has no tensor maps");
            r.encode = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
            ready = true;
        }
    }
    return r;
}
static thread_local int t_device = 0;  // of the call that this thread is in
static int *error_word() { return runtime().errors + (t_device & 63); }
// Reports a kernel of the call's device that gave up waiting, once.
static void report_earlier() {
    int *word = error_word();
    if (!*static_cast<volatile int *>(word)) return;
    if (const int code = __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL))
        HB_THROW(HB_ECUDA, "an earlier training call gave up waiting in its kernel (code " + std::to_string(code) +
                               "): its results are not valid");
}
// Makes a call's device current, and reports what its kernels before this call left.
struct CallDevice {
    DeviceGuard dev;
    explicit CallDevice(int device, bool report = true) : dev(device) {
        t_device = device;
        if (report) report_earlier();
    }
};
static int sm_count() {
    std::atomic<int> &known = runtime().sms[t_device & 63];
    int n = known;
    if (!n) {
        cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, t_device), "SM count");
        known = n;
    }
    return n;
}

// Raises a kernel's shared-memory limit, once for each kernel and device.
template <auto KERNEL>
static void raise_shared_memory(int bytes) {
    static std::atomic<uint64_t> set{0};
    const int dev = t_device;
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

// One product.  a, b (and a1, b1 where used) lie K-major or MN-major: a K-major
// operand has the product's depth in its columns, an MN-major one in its rows.
struct Product {
    Matrix a, b, a1, b1;
    int64_t M = 0, N = 0, K = 0, K1 = 0;
    int amaj = K_MAJOR, outputs = 1, splits = 1;
    const LossPlan *plan = nullptr;
    bool plan_k = false;
    EpiArgs e;
    void *out[2] = {};    // gradients: dense 16-bit rows; with none, acc is the result
    float *acc = nullptr;  // of a split depth
    int cols() const { return N <= 128 ? 128 : kCols; }
    int64_t tiles() const { return (int64_t)blocks(M, kRows) * blocks(N, cols()) * outputs; }
    int64_t slices() const { return (int64_t)blocks(K, kDepth) + blocks(K1, kDepth); }
    int64_t sums() const { return splits > 1 ? (int64_t)outputs * splits * M * pad(N, 4) : 0; }
};
static void fill(Job &j, const Product &d, bool bf16, int amaj, int bmaj, int cols_n) {
    j.a = tensor_map(d.a, bf16, amaj);
    j.b = tensor_map(d.b, bf16, bmaj);
    j.a1 = d.a1.p ? tensor_map(d.a1, bf16, amaj) : j.a;
    j.b1 = d.b1.p ? tensor_map(d.b1, bf16, bmaj) : j.b;
    j.M = d.M;
    j.N = d.N;
    j.tiles_m = (int)blocks(d.M, kRows);
    j.tiles_n = (int)blocks(d.N, cols_n);
    j.cols = d.cols();
    j.outputs = d.outputs;
    j.splits = d.splits;
    j.kb = (int)blocks(d.K, kDepth);
    j.kb1 = (int)blocks(d.K1, kDepth);
    j.amaj = amaj;
    j.plan = d.plan;
    j.plan_k = d.plan_k;
    j.e = d.e;
}
static unsigned product_grid(int64_t items) {
    require(items < (int64_t)1 << 31, "more than 2^31 tiles in one product");
    const int64_t pairs = sm_count() / 2;
    return (unsigned)(2 * (items < pairs ? items : pairs));
}
// The products with both operands K-major.
template <class T, int EPI, int ACT>
static void launch(const Product &d, cudaStream_t s) {
    constexpr int cols_n = EPI == EPI_GATED || EPI == EPI_GATED_BWD ? 128 : kCols;
    ProductArgs<1> p;
    fill(p.job[0], d, std::is_same<T, __nv_bfloat16>::value, K_MAJOR, K_MAJOR, cols_n);
    p.error = error_word();
    raise_shared_memory<k_mma_product<T, K_MAJOR, K_MAJOR, EPI, ACT, 1>>(kProductSmem);
    start("training product", k_mma_product<T, K_MAJOR, K_MAJOR, EPI, ACT, 1>,
          product_grid((int64_t)p.job[0].tiles_m * p.job[0].tiles_n), product_threads(EPI), kProductSmem, s, p);
}

// Parts of the depth of each of a launch's products (two, or one): none whose
// items are no longer than what every SM pair has to do on average, else as
// many as bring them there, each at least 4 slices deep, and none below 16
// slices, where joining costs more than it saves (weight gradients of 512 x 512
// x 512, 8 slices: 19.4 us in two parts, 16.3 in one; its dX, 16 slices: 18.0
// in four, 18.5 in two).
static void split_depths(Product *d, int n) {
    double work = 0;
    for (int i = 0; i < n; i++) work += (double)d[i].tiles() * (double)d[i].slices();
    for (int i = 0; i < n; i++) {
        const int64_t slices = d[i].slices(), most = 74 / d[i].tiles() < slices / 4 ? 74 / d[i].tiles() : slices / 4;
        int64_t parts = (int64_t)((double)slices * 74 / work + 0.3);
        if (parts > most) parts = most;
        d[i].splits = parts > 1 && slices >= 16 ? (int)parts : 1;
    }
}
// Splits the two products' depths, for one launch of both or a launch each:
// true for one.  Rounds are counted in slices, a tile's epilogue as two, a
// launch of its own and a joining as eight each, and the kernel for two as 7 %
// slower.  Measured, together and apart (us): gated gradients of 64 x 432 x 512
// 18 and 24, 1024 x 1024 x 1024 28 and 41, 2047 x 1001 x 1500 58 and 61, 4096 x
// 2048 x 2048 155 and 146; the loss's of 2048 x 256 x 20000 80 and 96, 777 x 432
// x 32001 92 and 99, 4096 x 1024 x 32001 602 and 581.  Where what both read
// outgrows L2 (the last), two orders of reading it at once lose what the rounds
// gain.
static bool together(Product *d) {
    auto length = [](const Product &g) { return (double)(g.slices() / g.splits + 2); };
    auto items = [](const Product &g) { return (double)(g.tiles() * g.splits); };
    Product apart[2] = {d[0], d[1]};
    double separate = 8;
    for (Product &g : apart) {
        split_depths(&g, 1);
        separate += std::ceil(items(g) / 74) * length(g) + (g.splits > 1 ? 8 : 0);
    }
    split_depths(d, 2);
    const int first = length(d[1]) > length(d[0]);
    const Product &a = d[first], &b = d[1 - first];
    const double full = std::floor(items(a) / 74), rest = items(a) - 74 * full, start = full * length(a);
    double joint = d[0].splits > 1 || d[1].splits > 1 ? 8 : 0;
    if (rest == 0) {
        joint += start + std::ceil(items(b) / 74) * length(b);
    } else {
        const double beside = std::ceil(length(a) / length(b)) * (74 - rest);
        if (items(b) <= beside) {
            const double tail = std::ceil(items(b) / (74 - rest)) * length(b);
            joint += start + (tail > length(a) ? tail : length(a));
        } else {
            joint += start + length(a) + std::ceil((items(b) - beside) / 74) * length(b);
        }
    }
    // both read the same A (dG and dU, or Z)
    double bytes = 2.0 * (double)d[0].M * (double)(d[0].K + d[0].K1);
    for (int i = 0; i < 2; i++) bytes += 2.0 * (double)d[i].N * (double)(d[i].K + d[i].K1);
    if (joint * 1.07 < separate && bytes <= 160e6) return true;
    d[0].splits = apart[0].splits;
    d[1].splits = apart[1].splits;
    return false;
}
template <class T>
static void join(const JoinArgs &j, void *out, cudaStream_t s) {
    T *o = static_cast<T *>(out);
    if (j.parts > 8)
        start("join parts", k_join<T, true>, blocks(j.M * (j.ld / 4), 32), 256, 0, s, j, o);
    else
        start("join parts", k_join<T, false>, blocks(j.M * (j.ld / 4), 256), 256, 0, s, j, o);
}
// The gradients' products, B MN-major, two of them in one launch (4096 x 1024 x
// 4096: dX of 64 tiles and the weights' of 128 leave 10 of the 74 SM pairs idle
// in one round and 20 in the other on their own).  D = A B^T (+ A1 B1^T), or with
// outputs = 2 also A1 B^T; the sums of a split depth are joined in acc.
template <class T, int AMAJ, int JOBS>
static void launch_gradients(Product *d, cudaStream_t s) {
    ProductArgs<JOBS> p;
    int64_t items = 0;
    for (int i = 0; i < JOBS; i++) {
        Product &g = d[i];
        if (g.out[0] && g.splits == 1) {
            g.e.o0 = g.out[0];
            g.e.o1 = g.out[1];
            g.e.ldo = g.N;
            g.e.vec = fits_vectors(g.out[0], g.N) && (g.outputs == 1 || fits_vectors(g.out[1], g.N));
        } else {
            g.e.acc = g.acc;
            g.e.ldo = pad(g.N, 4);
        }
        fill(p.job[i], g, std::is_same<T, __nv_bfloat16>::value, g.amaj, MN_MAJOR, g.cols());
        items += g.tiles() * g.splits;
    }
    p.error = error_word();
    raise_shared_memory<k_mma_product<T, AMAJ, MN_MAJOR, EPI_OUT, 0, JOBS>>(kProductSmem);
    start("training product", k_mma_product<T, AMAJ, MN_MAJOR, EPI_OUT, 0, JOBS>, product_grid(items),
          product_threads(EPI_OUT), kProductSmem, s, p);
}
template <class T>
static void gradients(Product *d, int n, cudaStream_t s) {
    if (n == 2) {
        // the longer items first
        if (d[1].slices() / d[1].splits > d[0].slices() / d[0].splits) std::swap(d[0], d[1]);
        launch_gradients<T, K_MAJOR, 2>(d, s);
    } else if (n == 1 && d[0].amaj == K_MAJOR) {
        launch_gradients<T, K_MAJOR, 1>(d, s);
    } else if (n == 1) {
        launch_gradients<T, MN_MAJOR, 1>(d, s);
    }
    for (int i = 0; i < n; i++) {
        const Product &g = d[i];
        for (int k = 0; g.out[0] && g.splits > 1 && k < g.outputs; k++)
            join<T>({g.acc + (int64_t)k * g.splits * g.M * g.e.ldo, g.splits, g.M, g.M, g.N, g.e.ldo, g.e.unscale, nullptr},
                    g.out[k], s);
    }
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

// Columns of a vocabulary piece: Z of a piece takes at most 512 MiB (256 MiB:
// 907 us for 4096 x 128 x 131072 where 704 are reached with 1 GiB, 64 MiB:
// 1140), in whole rounds of the SM pairs for dW where that many fit; 2048 at
// least, which more than 131072 rows fill beyond that.
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
        CallDevice dev(device);
        cudaStream_t s = (cudaStream_t)stream;
        in.copy(s);
        d.M = tokens, d.N = width, d.K = inner;
        d.e.o0 = h;
        d.e.ldo = width;
        d.e.vec = fits_vectors(h, width);
        by_dtype(dtype, [&](auto t) {
            by_act(act, [&](auto a) { launch<decltype(t), EPI_GATED, decltype(a)::value>(d, s); });
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
        require(tokens == 0 || dx || dwg || dwu, "no output is asked for");  // an empty dx has no address
        require(act >= 0 && act <= HELRM_ACT_GELU, "unknown activation");
        Workspace w{static_cast<char *>(ws)};
        Operands in(w);
        const int64_t ldd = pitch(width);
        uint16_t *dg = w.take<uint16_t>(tokens * ldd), *du = w.take<uint16_t>(tokens * ldd);
        uint16_t *read = x ? nullptr : w.take<uint16_t>(tokens * pitch(inner));
        const Matrix mx = x ? in.fit({x, tokens, inner, ldx}) : Matrix{read, tokens, inner, pitch(inner)};
        const Matrix mg = in.fit({wg, width, inner, ldg}), mu = in.fit({wu, width, inner, ldu});
        const Matrix mdg{dg, tokens, width, ldd}, mdu{du, tokens, width, ldd};
        // the depths are split as if all were wanted: an output has the same bits with or without the others
        Product all[2], grads[2];
        Product &gx = all[0], &gw = all[1];
        gx.a = mdg, gx.b = mg, gx.a1 = mdu, gx.b1 = mu;
        gx.M = tokens, gx.N = inner, gx.K = gx.K1 = width;
        gx.out[0] = dx;
        gw.a = dwg ? mdg : mdu, gw.a1 = mdu, gw.b = mx;
        gw.amaj = MN_MAJOR;
        gw.M = width, gw.N = inner, gw.K = tokens;
        gw.outputs = 2;
        gw.out[0] = dwg ? dwg : dwu, gw.out[1] = dwu;
        const bool one = tokens && together(all);
        gw.outputs = dwg && dwu ? 2 : 1;
        const bool scaled = dtype == HELRM_FP16;
        float4 *range = scaled ? w.take<float4>(kRangeBlocks) : nullptr;
        float *unscale = scaled ? w.take<float>(1) : nullptr;
        gx.e.unscale = gw.e.unscale = unscale;
        int n = 0;
        for (Product &g : all) {
            if (!g.out[0]) continue;
            g.acc = w.take<float>(g.sums());
            grads[n++] = g;
        }
        if (sized(w, ws_bytes)) return;
        CallDevice dev(device);
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
            if (scaled) {
                GatedRange r = {static_cast<const unsigned short *>(dh),
                                static_cast<const unsigned short *>(mx.p),
                                {static_cast<const unsigned short *>(mu.p), static_cast<const unsigned short *>(mg.p)},
                                lddh, mx.ld, {mu.ld, mg.ld}, tokens, width, inner,
                                fits_vectors(dh, tokens > 1 ? lddh : pitch(width)), range};
                const int64_t rows = tokens + 2 * width;
                d.e.ranges = blocks(rows, kRangeWarps) < kRangeBlocks ? (int)blocks(rows, kRangeWarps) : kRangeBlocks;
                d.e.range = range;
                d.e.made = unscale;
                start("gradients' range", k_gated_range, d.e.ranges, kRangeThreads, 0, s, r);
            }
            by_act(act, [&](auto a) { launch<T, EPI_GATED_BWD, decltype(a)::value>(d, s); });
            if (one) {
                gradients<T>(grads, n, s);
            } else {
                for (int i = 0; i < n; i++) gradients<T>(grads + i, 1, s);
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
        CallDevice dev(device);
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
        CallDevice dev(device);
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
        CallDevice dev(device);
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
            by_dtype(dtype, [&](auto t) {
                if (inner > kChunk * kDepth)
                    launch<decltype(t), EPI_LSE_LONG, 0>(d, s);
                else
                    launch<decltype(t), EPI_LSE, 0>(d, s);
            });
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
        require(tokens == 0 || dh || dw, "no output is asked for");
        Workspace w{static_cast<char *>(ws)};
        Operands in(w);
        const Matrix mw = in.fit({wt, vocab, inner, ldw});
        const int64_t cap = pad(tokens, 256);  // the rows that take part, filled up
        uint16_t *hc = w.take<uint16_t>(cap * pitch(inner));
        const Matrix mh{hc, cap, inner, pitch(inner)};
        LossRow *rows = w.take<LossRow>(cap);
        int *src = w.take<int>(cap), *pos = w.take<int>(tokens);
        LossPlan *plan = w.take<LossPlan>(1);
        auto prepare = [&](cudaStream_t s) {
            in.copy(s);
            LossRows r = {dloss, targets, reinterpret_cast<const float2 *>(lse), ignore_index, vocab, tokens,
                          static_cast<const unsigned short *>(h), ldh, inner, fits_vectors(h, ldh),
                          dtype == HELRM_FP16 ? 32768.0f : 1.0f, 0, rows, src,
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
            CallDevice dev(device);
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
                a.error = error_word();
                raise_shared_memory<k_loss_grads_narrow<T>>(kNarrowSmem);
                start("loss gradients", k_loss_grads_narrow<T>, nr.grid, kNarrowThreads, kNarrowSmem, s, a);
                if (dh) join<T>({part, nr.grid, cap, tokens, inner, nr.depth, &plan->unscale, pos}, dh, s);
            });
            return;
        }
        const int64_t cols = piece_columns(cap, vocab), ldz = pitch(cols), lda = pad(inner, 4);
        uint16_t *z = w.take<uint16_t>(cap * ldz);
        // the products of the first, largest piece: dh is a 32-bit sum over the pieces, for each part of a piece's
        // depth, of the rows that take part
        Product all[2];
        Product &gh = all[0], &gw = all[1];
        gh.a = {z, cap, cols, ldz};
        gh.M = cap, gh.N = inner, gh.K = cols;
        gw.b = mh;
        gw.amaj = MN_MAJOR;
        gw.M = cols, gw.N = inner, gw.K = cap;
        gw.plan_k = true;
        const bool one = tokens && together(all);
        float *acc = w.take<float>(dh ? gh.splits * cap * lda : 0);
        float *acc_w = w.take<float>(dw ? gw.sums() : 0);
        if (sized(w, ws_bytes)) return;
        CallDevice dev(device);
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
                    if (inner > kChunk * kDepth)
                    launch<T, EPI_Z_LONG, 0>(d, s);
                else
                    launch<T, EPI_Z, 0>(d, s);
                Product piece[2];
                int np = 0;
                if (dh) {
                    Product &g = piece[np++] = gh;
                    g.a = mz, g.b = mc;
                    g.plan = plan;
                    g.K = n;
                    // the last piece may be too short for every part: those keep their sums
                    g.splits = gh.splits < (int)blocks(n, kDepth) ? gh.splits : (int)blocks(n, kDepth);
                    g.acc = acc;
                    g.e.first = c0 == 0;
                }
                if (dw) {
                    Product &g = piece[np++] = gw;
                    g.a = mz;
                    g.plan = plan;
                    g.M = n;
                    g.e.unscale = &plan->unscale;
                    g.out[0] = static_cast<T *>(dw) + c0 * inner;
                    g.acc = acc_w;
                }
                if (one) {
                    gradients<T>(piece, np, s);
                } else {
                    // dW first: Z's last columns, just written, are its last rows
                    for (int i = np - 1; i >= 0; i--) gradients<T>(piece + i, 1, s);
                }
            }
            if (dh) join<T>({acc, gh.splits, cap, tokens, inner, lda, &plan->unscale, pos}, dh, s);
        });
    });
}

HB_API int helrm_TrainingSynchronize(int device, void *stream) {
    return guard([&] {
        CallDevice dev(device, false);
        cuda_check(cudaStreamSynchronize((cudaStream_t)stream), "training call");
        report_earlier();
    });
}
HB_API int helrm_TrainingPostFailure(int device, int code) {
    return guard([&] {
        require(code > 0, "a kernel's code is above 0");
        CallDevice dev(device, false);
        __atomic_store_n(error_word(), code, __ATOMIC_RELEASE);
    });
}
