// C ABI of libqsb200 (declared in include/qsb200.h): argument checks, per-device
// state, dispatch to the kernel files.
#include <cuda.h>  // CUcontext (the driver calls themselves are resolved at run time)
#include <mutex>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/qsb200.h"
#include "qs_kernels.h"
#include "qs_matmul.cuh"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

int cuda_fail(cudaError_t e, const char* what) {
    return fail(QS_ECUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

struct TypeInfo {
    int type, qk, bytes, needs_qw;
};

const TypeInfo kTypes[] = {
    {qs::QS_Q4_0, 32, 18, 0},      {qs::QS_Q2_K, 256, 84, 0},      {qs::QS_Q3_K, 256, 110, 0},
    {qs::QS_Q4_K, 256, 144, 0},    {qs::QS_Q5_K, 256, 176, 0},     {qs::QS_Q6_K, 256, 210, 0},
    {qs::QS_IQ2_XXS, 256, 66, 1},  {qs::QS_IQ2_XS, 256, 74, 1},    {qs::QS_IQ3_XXS, 256, 98, 0},
    {qs::QS_IQ3_S, 256, 110, 0},   {qs::QS_IQ2_S, 256, 82, 1},     {qs::QS_IQ4_XS, 256, 136, 0},
    {qs::QS_Q4_1, 32, 20, 0},      {qs::QS_Q5_0, 32, 22, 0},       {qs::QS_Q5_1, 32, 24, 0},
    {qs::QS_Q8_0, 32, 34, 0},
};

const TypeInfo* find_type(int t) {
    for (const auto& ti : kTypes)
        if (ti.type == t) return &ti;
    return nullptr;
}

bool is_iq(int t) {
    return t == qs::QS_IQ2_XXS || t == qs::QS_IQ2_XS || t == qs::QS_IQ2_S || t == qs::QS_IQ3_XXS || t == qs::QS_IQ3_S;
}

constexpr int kMaxDevices = 64;

struct DeviceState {
    bool ready = false;
    int num_sms = 0;
    qs::IqTables* iq = nullptr;
    unsigned int* fault = nullptr;  // the fault word
    cudaMemPool_t pool = nullptr;  // scratch of qs_tensor_error; keeps its memory between calls
};

std::mutex g_mu[kMaxDevices];  // one per device: devices come up in parallel
DeviceState g_dev[kMaxDevices];

// Caller holds no lock; the device must be current.
int ensure_device(int device, DeviceState** out) {
    if (device < 0 || device >= kMaxDevices) return fail(QS_EINVAL, "device %d out of range", device);
    std::lock_guard<std::mutex> lk(g_mu[device]);
    DeviceState& d = g_dev[device];
    if (!d.ready) {
        cudaError_t e = cudaDeviceGetAttribute(&d.num_sms, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
        e = qs::iq_tables_create(&d.iq);
        if (e != cudaSuccess) return cuda_fail(e, "uploading the lattice codebooks");
        if ((e = qs::fault_word(&d.fault)) != cudaSuccess) return cuda_fail(e, "the fault word's address");
        cudaMemPoolProps props;
        memset(&props, 0, sizeof(props));
        props.allocType = cudaMemAllocationTypePinned;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = device;
        if ((e = cudaMemPoolCreate(&d.pool, &props)) != cudaSuccess) return cuda_fail(e, "cudaMemPoolCreate");
        uint64_t keep = UINT64_MAX;
        if ((e = cudaMemPoolSetAttribute(d.pool, cudaMemPoolAttrReleaseThreshold, &keep)) != cudaSuccess)
            return cuda_fail(e, "cudaMemPoolSetAttribute");
        d.ready = true;
    }
    *out = &d;
    return QS_OK;
}

// The calling thread's current CUDA context, saved when an entry point starts and put back
// when it returns: a call that runs on the device owning its data (cudaSetDevice) must not
// leave that device current for the caller, nor create a context the caller never had.
// The two driver calls are looked up once through the runtime, so the library does not
// link libcuda directly.
struct CtxFns {
    CUresult (*get)(CUcontext*) = nullptr;
    CUresult (*set)(CUcontext) = nullptr;
};

const CtxFns& ctx_fns() {
    static CtxFns f;
    static std::once_flag once;
    std::call_once(once, [] {
        void* g = nullptr;
        void* s = nullptr;
        cudaDriverEntryPointQueryResult q1, q2;
        if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &g, cudaEnableDefault, &q1) == cudaSuccess &&
            cudaGetDriverEntryPoint("cuCtxSetCurrent", &s, cudaEnableDefault, &q2) == cudaSuccess &&
            q1 == cudaDriverEntryPointSuccess && q2 == cudaDriverEntryPointSuccess) {
            f.get = reinterpret_cast<CUresult (*)(CUcontext*)>(g);
            f.set = reinterpret_cast<CUresult (*)(CUcontext)>(s);
        }
    });
    return f;
}

class CurrentContextGuard {
public:
    CurrentContextGuard() {
        const CtxFns& f = ctx_fns();
        ok_ = f.get && f.get(&saved_) == CUDA_SUCCESS;
    }
    ~CurrentContextGuard() {
        if (!ok_) return;
        const CtxFns& f = ctx_fns();
        CUcontext now = nullptr;
        if (f.get(&now) == CUDA_SUCCESS && now != saved_) f.set(saved_);
    }
    CurrentContextGuard(const CurrentContextGuard&) = delete;
    CurrentContextGuard& operator=(const CurrentContextGuard&) = delete;

private:
    CUcontext saved_ = nullptr;
    bool ok_ = false;
};

// `p` must be memory of `device` (or managed memory): a pointer into another GPU's memory
// would otherwise reach the kernel and fault there.
int check_on_device(const void* p, int device, const char* what) {
    cudaPointerAttributes pa;
    cudaError_t e = cudaPointerGetAttributes(&pa, p);
    if (e != cudaSuccess) return cuda_fail(e, "cudaPointerGetAttributes");
    if (pa.type == cudaMemoryTypeManaged) return QS_OK;
    if (pa.type != cudaMemoryTypeDevice) return fail(QS_EINVAL, "%s is not device memory", what);
    if (pa.device != device) return fail(QS_EINVAL, "%s is on device %d, the call runs on device %d", what, pa.device, device);
    return QS_OK;
}

}  // namespace

#define QS_API __attribute__((visibility("default")))

extern "C" {

QS_API int qs_version(void) { return QSB200_VERSION; }

QS_API const char* qs_last_error(void) { return g_err; }

QS_API int qs_type_supported(int ggml_type) { return find_type(ggml_type) != nullptr; }

QS_API int qs_type_needs_qw(int ggml_type) {
    const TypeInfo* ti = find_type(ggml_type);
    return ti ? ti->needs_qw : 0;
}

QS_API int qs_block_info(int ggml_type, int* qk, int* block_bytes) {
    const TypeInfo* ti = find_type(ggml_type);
    if (!ti) return fail(QS_ENOTSUP, "ggml type %d is not supported", ggml_type);
    if (qk) *qk = ti->qk;
    if (block_bytes) *block_bytes = ti->bytes;
    return QS_OK;
}

QS_API int qs_row_bytes(int ggml_type, int64_t k, int64_t* out_bytes) {
    const TypeInfo* ti = find_type(ggml_type);
    if (!ti) return fail(QS_ENOTSUP, "ggml type %d is not supported", ggml_type);
    if (k <= 0 || k % ti->qk) return fail(QS_EINVAL, "row length %lld is not a positive multiple of %d", (long long)k, ti->qk);
    if (out_bytes) *out_bytes = k / ti->qk * ti->bytes;
    return QS_OK;
}

QS_API int qs_init(int device) {
    CurrentContextGuard keep;
    cudaError_t e = cudaSetDevice(device);
    if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    DeviceState* d = nullptr;
    return ensure_device(device, &d);
}

}  // extern "C"

namespace {

// Make the device that owns `p` current (the runtime's current device may belong to
// another runtime instance in the process, e.g. the one torch links) and prepare it.
int device_of(const void* p, const char* what, int* device, DeviceState** st) {
    cudaPointerAttributes pa;
    cudaError_t e = cudaPointerGetAttributes(&pa, p);
    if (e != cudaSuccess) return cuda_fail(e, "cudaPointerGetAttributes");
    if (pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged)
        return fail(QS_EINVAL, "%s is not device memory", what);
    int cur = -1;
    if ((e = cudaGetDevice(&cur)) != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (cur != pa.device && (e = cudaSetDevice(pa.device)) != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    *device = pa.device;
    return ensure_device(pa.device, st);
}

// Checks shared by the decode entry points; fills the kernel call.
int check_decode(int ggml_type, const void* blocks, int64_t blocks_row_bytes, int64_t n_rows, int64_t k,
                 qs::DqCall& c) {
    const TypeInfo* ti = find_type(ggml_type);
    if (!ti) return fail(QS_ENOTSUP, "ggml type %d is not supported", ggml_type);
    if (k <= 0 || k % ti->qk) return fail(QS_EINVAL, "row length %lld is not a positive multiple of %d", (long long)k, ti->qk);
    if (n_rows < 0) return fail(QS_EINVAL, "negative row count");
    const int64_t row_bytes = k / ti->qk * ti->bytes;
    if (blocks_row_bytes < row_bytes)
        return fail(QS_EINVAL, "block row stride %lld < packed row size %lld", (long long)blocks_row_bytes, (long long)row_bytes);
    memset(&c, 0, sizeof(c));
    c.blocks = blocks;
    c.blocks_row_bytes = blocks_row_bytes;
    c.n_rows = n_rows;
    c.k = k;
    return QS_OK;
}

int check_source(const void* x, int x_type, const float* qw) {
    if (x_type != QS_SRC_F32 && x_type != QS_SRC_F16 && x_type != QS_SRC_BF16)
        return fail(QS_EINVAL, "source type %d is not F32/F16/BF16", x_type);
    if (!x) return fail(QS_EINVAL, "null source rows");
    if (((uintptr_t)x & 15) || (qw && ((uintptr_t)qw & 15))) return fail(QS_EINVAL, "x and qw must be 16-byte aligned");
    return QS_OK;
}

}  // namespace

extern "C" {

QS_API int qs_quantize(int ggml_type, const void* src, int src_type, int64_t n_rows, int64_t k, const float* qw,
                void* dst, int64_t dst_row_bytes, void* stream) {
    const TypeInfo* ti = find_type(ggml_type);
    if (!ti) return fail(QS_ENOTSUP, "ggml type %d is not supported", ggml_type);
    if (src_type != QS_SRC_F32 && src_type != QS_SRC_F16 && src_type != QS_SRC_BF16)
        return fail(QS_EINVAL, "source type %d is not F32/F16/BF16", src_type);
    if (k <= 0 || k % ti->qk) return fail(QS_EINVAL, "row length %lld is not a positive multiple of %d", (long long)k, ti->qk);
    if (n_rows < 0) return fail(QS_EINVAL, "negative row count");
    const int64_t row_bytes = k / ti->qk * ti->bytes;
    if (dst_row_bytes < row_bytes) return fail(QS_EINVAL, "dst_row_bytes %lld < packed row size %lld", (long long)dst_row_bytes, (long long)row_bytes);
    if (ti->needs_qw && !qw) return fail(QS_ENOIMAT, "ggml type %d needs importance weights (qw)", ggml_type);
    if (n_rows == 0) return QS_OK;
    if (!src || !dst) return fail(QS_EINVAL, "null src or dst");
    if (((uintptr_t)src & 15) || (qw && ((uintptr_t)qw & 15)))
        return fail(QS_EINVAL, "src and qw must be 16-byte aligned");
    CurrentContextGuard keep;

    // run on the device that owns src (the runtime's current device may belong to another
    // runtime instance in the process, e.g. the one torch links)
    cudaPointerAttributes pa;
    cudaError_t e = cudaPointerGetAttributes(&pa, src);
    if (e != cudaSuccess) return cuda_fail(e, "cudaPointerGetAttributes(src)");
    if (pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged)
        return fail(QS_EINVAL, "src is not device memory");
    const int device = pa.device;
    int cur = -1;
    if ((e = cudaGetDevice(&cur)) != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (cur != device && (e = cudaSetDevice(device)) != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    int rc;
    if ((rc = check_on_device(dst, device, "dst")) || (qw && (rc = check_on_device(qw, device, "qw")))) return rc;
    DeviceState* d = nullptr;
    if ((rc = ensure_device(device, &d))) return rc;

    qs::QuantArgs a;
    a.src = src;
    a.src_type = src_type;
    a.n_rows = n_rows;
    a.k = k;
    a.qw = qw;
    a.dst = static_cast<uint8_t*>(dst);
    a.dst_row_bytes = dst_row_bytes;
    a.row_bytes = row_bytes;
    a.nblk_row = k / ti->qk;
    a.nblk = n_rows * a.nblk_row;
    qs::LaunchCtx ctx{static_cast<cudaStream_t>(stream), device, d->num_sms};
    if (is_iq(ggml_type) && (e = qs::iq_tables_ensure(d->iq, ggml_type)) != cudaSuccess)
        return cuda_fail(e, "building lattice tables");
    e = is_iq(ggml_type)             ? qs::launch_iq(ggml_type, a, ctx, d->iq)
        : qs::is_blk32(ggml_type)    ? qs::launch_blk32(ggml_type, a, ctx)
                                     : qs::launch_kquant(ggml_type, a, ctx);
    if (e != cudaSuccess) return cuda_fail(e, "kernel launch");
    return QS_OK;
}

QS_API int qs_dequantize(int ggml_type, const void* src, int64_t src_row_bytes, int64_t n_rows, int64_t k, float* dst,
                         int64_t dst_row_stride, void* stream) {
    qs::DqCall c;
    int rc = check_decode(ggml_type, src, src_row_bytes, n_rows, k, c);
    if (rc) return rc;
    if (dst_row_stride < k || dst_row_stride % 4) return fail(QS_EINVAL, "dst_row_stride %lld must be >= k and a multiple of 4", (long long)dst_row_stride);
    if (n_rows == 0) return QS_OK;
    if (!src || !dst) return fail(QS_EINVAL, "null src or dst");
    if ((uintptr_t)dst & 15) return fail(QS_EINVAL, "dst must be 16-byte aligned");
    CurrentContextGuard keep;
    int device;
    DeviceState* d;
    if ((rc = device_of(src, "src", &device, &d))) return rc;
    if ((rc = check_on_device(dst, device, "dst"))) return rc;
    c.dst = dst;
    c.dst_stride = dst_row_stride;
    qs::LaunchCtx ctx{static_cast<cudaStream_t>(stream), device, d->num_sms};
    cudaError_t e = qs::launch_dequant(ggml_type, c, ctx, d->iq);
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "dequantize launch");
}

QS_API int qs_block_error(int ggml_type, const void* blocks, int64_t blocks_row_bytes, const void* x, int x_type,
                          int64_t n_rows, int64_t k, const float* qw, double* err, void* stream) {
    qs::DqCall c;
    int rc = check_decode(ggml_type, blocks, blocks_row_bytes, n_rows, k, c);
    if (rc) return rc;
    if (n_rows == 0) return QS_OK;
    if ((rc = check_source(x, x_type, qw))) return rc;
    if (!blocks || !err) return fail(QS_EINVAL, "null blocks or err");
    if ((uintptr_t)err & 7) return fail(QS_EINVAL, "err must be 8-byte aligned");
    CurrentContextGuard keep;
    int device;
    DeviceState* d;
    if ((rc = device_of(blocks, "blocks", &device, &d))) return rc;
    if ((rc = check_on_device(x, device, "x")) || (qw && (rc = check_on_device(qw, device, "qw"))) ||
        (rc = check_on_device(err, device, "err")))
        return rc;
    c.x = x;
    c.x_type = x_type;
    c.qw = qw;
    c.err = err;
    qs::LaunchCtx ctx{static_cast<cudaStream_t>(stream), device, d->num_sms};
    cudaError_t e = qs::launch_block_error(ggml_type, c, ctx, d->iq);
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "block error launch");
}

QS_API int qs_tensor_error(int ggml_type, const void* blocks, int64_t blocks_row_bytes, const void* x, int x_type,
                           int64_t n_rows, int64_t k, const float* qw, double* out, void* stream) {
    qs::DqCall c;
    int rc = check_decode(ggml_type, blocks, blocks_row_bytes, n_rows, k, c);
    if (rc) return rc;
    if (!out) return fail(QS_EINVAL, "null out");
    if ((uintptr_t)out & 7) return fail(QS_EINVAL, "out must be 8-byte aligned");
    if (n_rows > 0) {
        if ((rc = check_source(x, x_type, qw))) return rc;
        if (!blocks) return fail(QS_EINVAL, "null blocks");
    }
    CurrentContextGuard keep;
    int device;
    DeviceState* d;
    if ((rc = device_of(out, "out", &device, &d))) return rc;
    if (n_rows > 0 && ((rc = check_on_device(blocks, device, "blocks")) || (rc = check_on_device(x, device, "x")) ||
                       (qw && (rc = check_on_device(qw, device, "qw")))))
        return rc;
    c.x = x;
    c.x_type = x_type;
    c.qw = qw;
    qs::LaunchCtx ctx{static_cast<cudaStream_t>(stream), device, d->num_sms};
    const int np = qs::dq_partial_count(ggml_type, n_rows, k, ctx);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    void* partial = nullptr;
    cudaError_t e = cudaMallocFromPoolAsync(&partial, (size_t)np * 2 * sizeof(double), d->pool, st);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMallocFromPoolAsync (partial sums)");
    e = qs::launch_tensor_error(ggml_type, c, static_cast<double*>(partial), np, out, ctx, d->iq);
    cudaError_t ef = cudaFreeAsync(partial, st);
    if (e != cudaSuccess) return cuda_fail(e, "tensor error launch");
    return ef == cudaSuccess ? QS_OK : cuda_fail(ef, "cudaFreeAsync (partial sums)");
}

QS_API int qs_device_fault(int device, int* bits) {
    if (!bits) return fail(QS_EINVAL, "null bits");
    CurrentContextGuard keep;
    cudaError_t e = cudaSetDevice(device);
    if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    unsigned int b = 0;
    if ((e = qs::read_fault_bits(&b, true)) != cudaSuccess) return cuda_fail(e, "reading the fault word");
    *bits = (int)b;
    return QS_OK;
}

static_assert(qs::NA_MAX_PARTIALS == QS_NOALLOC_MAX_PARTIALS, "static scratch size and its public constant differ");

QS_API int qs_tensor_error_noalloc(int ggml_type, const void* blocks, int64_t blocks_row_bytes, const void* x,
                                   int x_type, int64_t n_rows, int64_t k, const float* qw, double* out, void* stream) {
    // allocation-free: no ensure_device (it uploads tables and creates a pool), only the
    // static scratch resolved by noalloc_setup
    qs::DqCall c;
    int rc = check_decode(ggml_type, blocks, blocks_row_bytes, n_rows, k, c);
    if (rc) return rc;
    if (!out) return fail(QS_EINVAL, "null out");
    if ((uintptr_t)out & 7) return fail(QS_EINVAL, "out must be 8-byte aligned");
    if (n_rows > 0) {
        if ((rc = check_source(x, x_type, qw))) return rc;
        if (!blocks) return fail(QS_EINVAL, "null blocks");
    }
    CurrentContextGuard keep;
    cudaPointerAttributes pa;
    cudaError_t e = cudaPointerGetAttributes(&pa, out);
    if (e != cudaSuccess) return cuda_fail(e, "cudaPointerGetAttributes");
    if (pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged) return fail(QS_EINVAL, "out is not device memory");
    int cur = -1;
    if ((e = cudaGetDevice(&cur)) != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (cur != pa.device && (e = cudaSetDevice(pa.device)) != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
    if (n_rows > 0 && ((rc = check_on_device(blocks, pa.device, "blocks")) || (rc = check_on_device(x, pa.device, "x")) ||
                       (qw && (rc = check_on_device(qw, pa.device, "qw")))))
        return rc;
    const qs::NoAllocDevice* d = nullptr;
    if ((e = qs::noalloc_setup(pa.device, &d)) != cudaSuccess) return cuda_fail(e, "static scratch set-up");
    c.x = x;
    c.x_type = x_type;
    c.qw = qw;
    qs::LaunchCtx ctx{static_cast<cudaStream_t>(stream), pa.device, d->num_sms};
    const int need = qs::dq_partial_count(ggml_type, n_rows, k, ctx);
    if (need > QS_NOALLOC_MAX_PARTIALS)
        return fail(QS_EINVAL, "launch needs %d partial sums; the static scratch holds %d", need, QS_NOALLOC_MAX_PARTIALS);
    e = qs::launch_tensor_error_noalloc(ggml_type, c, out, ctx, *d);
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "tensor error launch (static scratch)");
}

}  // extern "C"

// ---------------------------------------------------------------------------
// operators on packed blocks: norm into Q8_0, routing, products
// ---------------------------------------------------------------------------
namespace {

bool is_src(int t) { return t == QS_SRC_F32 || t == QS_SRC_F16 || t == QS_SRC_BF16; }
int src_size(int t) { return t == QS_SRC_F32 ? 4 : 2; }
bool aligned(const void* p, int a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }

// Alignment that the product kernels load blocks of a type with: the largest power of two (up
// to 16) that divides the block size and the places of its level bytes.
int block_align(int type) {
    switch (type) {
    case qs::QS_Q4_K: case qs::QS_Q5_K: return 16;
    case qs::QS_Q5_1: case qs::QS_IQ4_XS: return 8;
    case qs::QS_Q4_1: case qs::QS_Q2_K: return 4;
    default: return 2;
    }
}

bool has_min(int type) {
    return type == qs::QS_Q4_1 || type == qs::QS_Q5_1 || type == qs::QS_Q2_K || type == qs::QS_Q4_K || type == qs::QS_Q5_K;
}

// two scales per 32 values
bool two_scales(int type) {
    return type == qs::QS_Q2_K || type == qs::QS_Q3_K || type == qs::QS_Q6_K || type == qs::QS_IQ2_XS || type == qs::QS_IQ2_S;
}

// How a product runs: which kernel, its tile, over how many CTAs a tile's rows are split.
struct MmPlan {
    enum { FEW, MID, TC } kind;
    bool lo;
    int bn, splits;
    int64_t part_off, bytes;  // workspace: laid-out activations, then the slots' results before a sum
};

// slots: output rows before a weighted sum; groups: weight matrices that share them; x_rows:
// activation rows. The number of CTAs is set against a B200's 148 SMs.
MmPlan mm_plan(int type, int64_t n, int64_t k, int64_t slots, int64_t groups, int64_t x_rows, bool experts, bool sum, bool lo) {
    MmPlan p;
    const int64_t avg = (slots + groups - 1) / groups, units = k / 32, stages = (units + 1) / 2;
    // rows that the kernel for few slots can not hold go to the next one
    const bool holds = units * qs::FEW_SLOTS * qs::FEW_UNIT_MAX <= qs::FEW_SMEM_MAX;
    // The tcgen05 kernel from 65 rows on; with experts from an average of 57, where many of them have over 64
    // and so two tiles of 64 (32 of 2048 x 2048, float32 results, Q6_K: 56 rows each 160 / 176 us, 64 rows 231 /
    // 176 us). For bfloat16 results from 33 rows on with superblocks, whose unpacking it does once for all
    // rows (64 rows of 4096 x 14336: Q4_K 57 / 46 us, Q6_K 77 / 59 us; Q4_0 46 / 50 us), but not for small
    // matrices with one scale per 32 values (Q4_K 2048 x 1024: 13.8 / 15.4 us, 4096 x 4096: 21.0 / 20.1 us, 8192 x 4096:
    // 32.8 / 29.2 us; Q6_K 2048 x 1024: 17.7 / 16.5 us).
    const bool early = !lo && find_type(type)->qk == 256 && (experts || two_scales(type) || n * k >= (int64_t)1 << 25);
    const int64_t mid = early ? 32 : experts ? 56 : 64;
    p.kind = (experts ? avg <= 1 : slots <= 4) && holds ? MmPlan::FEW : avg <= mid ? MmPlan::MID : MmPlan::TC;
    p.lo = lo;
    p.bn = avg <= 8 ? 8 : avg <= 16 ? 16 : avg <= 32 ? 32 : p.kind == MmPlan::MID ? 64 : avg <= 128 || lo ? 128 : 256;
    p.splits = 1;
    const int64_t chunks = groups == 1 ? (slots + p.bn - 1) / p.bn : slots / p.bn + (groups < slots ? groups : slots) / 2 + 1;
    const int64_t tiles = (n + 127) / 128 * chunks, ctas = p.kind == MmPlan::MID ? 2 * 148 : 148;
    if (tiles > 0 && tiles < ctas) {
        int64_t s = ctas / tiles;
        if (s > 8) s = 8;                    // a cluster
        if (s > stages / 8) s = stages / 8;  // 512 values each at least
        if (s > 1) {
            const int64_t per = ((stages + s - 1) / s + 3) / 4 * 4;  // whole superblocks
            p.splits = (int)((stages + per - 1) / per);
        }
    }
    const int sums = !has_min(type) ? 0 : type == qs::QS_Q2_K ? 2 : 1;
    int64_t xp = 0;
    if (p.kind == MmPlan::MID) xp = qs::mm_mid_workspace(units, x_rows, sums);
    if (p.kind == MmPlan::TC) xp = qs::mm_tc_workspace(units, qs::max_chunks(experts, slots, groups, p.bn), p.bn, lo, sums);
    p.part_off = (xp + 255) / 256 * 256;
    p.bytes = p.part_off + (sum ? slots * n * 4 : 0);
    return p;
}

// Checks of sizes shared by the products and their workspace queries.
int check_mm(int ggml_type, int64_t n, int64_t k, int64_t rows, int64_t per_token, const TypeInfo** out) {
    const TypeInfo* ti = find_type(ggml_type);
    if (!ti) return fail(QS_ENOTSUP, "ggml type %d is not supported", ggml_type);
    if (k <= 0 || k % ti->qk) return fail(QS_EINVAL, "row length %lld is not a positive multiple of %d", (long long)k, ti->qk);
    if (k > (int64_t)1 << 30) return fail(QS_EINVAL, "row length %lld is over 2^30", (long long)k);
    if (n <= 0 || n > (int64_t)1 << 30) return fail(QS_EINVAL, "weight row count %lld is not in 1 .. 2^30", (long long)n);
    if (rows < 0) return fail(QS_EINVAL, "negative row count");
    // 65535 chunks of 32 slots, and the threads of a weighted sum
    if (rows > (1 << 20) / per_token || rows * per_token * n > (int64_t)1 << 38)
        return fail(QS_EINVAL, "%lld rows of %lld outputs are too many for one call", (long long)(rows * per_token), (long long)n);
    *out = ti;
    return QS_OK;
}

int check_mm_operands(const TypeInfo* ti, const void* w, int64_t w_row_bytes, int64_t k, const void* x, int64_t x_row_bytes, const void* out,
                      int out_type, int64_t out_row_stride, int64_t n) {
    const int64_t row_bytes = k / ti->qk * ti->bytes;
    if (!w || !x || !out) return fail(QS_EINVAL, "null weights, activations or out");
    if (!is_src(out_type)) return fail(QS_EINVAL, "output type %d is not F32/F16/BF16", out_type);
    if (w_row_bytes < row_bytes) return fail(QS_EINVAL, "weight row stride %lld < packed row size %lld", (long long)w_row_bytes, (long long)row_bytes);
    if (x_row_bytes < k / 32 * 34) return fail(QS_EINVAL, "activation row stride %lld < Q8_0 row size %lld", (long long)x_row_bytes, (long long)(k / 32 * 34));
    if (out_row_stride < n) return fail(QS_EINVAL, "out_row_stride %lld < %lld", (long long)out_row_stride, (long long)n);
    const int al = block_align(ti->type);
    if (!aligned(w, al) || w_row_bytes % al) return fail(QS_EINVAL, "weights and their row stride must be multiples of %d bytes for ggml type %d", al, ti->type);
    if (!aligned(out, src_size(out_type))) return fail(QS_EINVAL, "out is not aligned to its elements");
    return QS_OK;
}

int run_mm(int ggml_type, const MmPlan& p, qs::MmArgs& a, int64_t k, int64_t x_rows, int top_k, const float* weights, const int* ids,
           void* workspace, const qs::LaunchCtx& ctx) {
    a.units = (int)(k / 32);
    a.splits = p.splits;
    a.part = weights ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.part_off) : nullptr;
    cudaError_t e = p.kind == MmPlan::FEW   ? qs::launch_mm_few(ggml_type, a, ctx)
                    : p.kind == MmPlan::MID ? qs::launch_mm_mid(ggml_type, a, p.bn, (int)x_rows, workspace, ctx)
                                            : qs::launch_mm_tc(ggml_type, a, p.bn, p.lo, workspace, ctx);
    if (e == cudaSuccess && weights) e = qs::launch_mm_sum(a, top_k, weights, ids, ctx);
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "matmul launch");
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
    if (bytes < need) return fail(QS_EINVAL, "workspace of %lld bytes, %lld are needed", (long long)bytes, (long long)need);
    if (need > 0 && !workspace) return fail(QS_EINVAL, "null workspace");
    if (need > 0 && !aligned(workspace, 16)) return fail(QS_EINVAL, "workspace must be 16-byte aligned");
    return QS_OK;
}

}  // namespace

extern "C" {

QS_API int qs_rms_norm_q8(const void* x, int x_type, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, void* total,
                          int64_t total_row_stride, const float* weight, double eps, int64_t n_rows, int64_t k, void* dst,
                          int64_t dst_row_bytes, void* stream) {
    if (!is_src(x_type)) return fail(QS_EINVAL, "source type %d is not F32/F16/BF16", x_type);
    if (k <= 0 || k % 32 || k > (int64_t)1 << 30) return fail(QS_EINVAL, "row length %lld is not a positive multiple of 32 (up to 2^30)", (long long)k);
    if (n_rows < 0 || n_rows > INT32_MAX) return fail(QS_EINVAL, "row count %lld is not in 0 .. 2^31 - 1", (long long)n_rows);
    if (!(eps > 0.0) || !(eps < 1e300)) return fail(QS_EINVAL, "eps must be positive and finite");
    if (!residual != !total) return fail(QS_EINVAL, "residual and total go together");
    if (dst_row_bytes < k / 32 * 34) return fail(QS_EINVAL, "dst_row_bytes %lld < Q8_0 row size %lld", (long long)dst_row_bytes, (long long)(k / 32 * 34));
    if (x_row_stride < k || (residual && (residual_row_stride < k || total_row_stride < k))) return fail(QS_EINVAL, "a row stride is below the row length");
    if (n_rows == 0) return QS_OK;
    if (!x || !weight || !dst) return fail(QS_EINVAL, "null x, weight or dst");
    const int el = 16 / src_size(x_type);
    if (!aligned(x, 16) || x_row_stride % el || !aligned(weight, 16) ||
        (residual && (!aligned(residual, 16) || !aligned(total, 16) || residual_row_stride % el || total_row_stride % el)))
        return fail(QS_EINVAL, "rows of x, residual and total, and weight, must start on 16-byte boundaries");
    CurrentContextGuard keep;
    int device, rc;
    DeviceState* d;
    if ((rc = device_of(x, "x", &device, &d))) return rc;
    if ((rc = check_on_device(weight, device, "weight")) || (rc = check_on_device(dst, device, "dst")) ||
        (residual && ((rc = check_on_device(residual, device, "residual")) || (rc = check_on_device(total, device, "total")))))
        return rc;
    qs::NormCall c;
    c.x = x;
    c.x_type = x_type;
    c.residual = residual;
    c.total = total;
    c.weight = weight;
    c.eps = eps;
    c.n_rows = n_rows;
    c.k = k;
    c.x_stride = x_row_stride;
    c.residual_stride = residual_row_stride;
    c.total_stride = total_row_stride;
    c.dst = dst;
    c.dst_row_bytes = dst_row_bytes;
    cudaError_t e = qs::launch_rms_norm_q8(c, qs::LaunchCtx{static_cast<cudaStream_t>(stream), device, d->num_sms});
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "rms norm launch");
}

QS_API int qs_route(const void* logits, int logits_type, int64_t logits_row_stride, int64_t n_rows, int n_experts, int top_k, int score,
                    const float* bias, int n_groups, int groups_kept, int group_score, int renormalize, float scale, int32_t* ids,
                    float* weights, void* stream) {
    if (!is_src(logits_type)) return fail(QS_EINVAL, "logits type %d is not F32/F16/BF16", logits_type);
    if (n_experts < 1 || n_experts > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts are not in 1 .. %d", n_experts, QS_MAX_EXPERTS);
    if (score != QS_SCORE_SOFTMAX && score != QS_SCORE_SIGMOID) return fail(QS_EINVAL, "score %d is neither softmax nor sigmoid", score);
    if (group_score != QS_GROUP_MAX && group_score != QS_GROUP_TOP2) return fail(QS_EINVAL, "group score %d is neither max nor top2", group_score);
    if (n_groups < 1 || n_groups > 64 || n_experts % n_groups) return fail(QS_EINVAL, "%d groups do not divide %d experts (at most 64)", n_groups, n_experts);
    if (groups_kept < 1 || groups_kept > n_groups) return fail(QS_EINVAL, "%d of %d groups can not be kept", groups_kept, n_groups);
    if (group_score == QS_GROUP_TOP2 && n_groups > 1 && n_groups == n_experts) return fail(QS_EINVAL, "groups of one expert have no two best");
    const int usable = n_experts / n_groups * groups_kept;
    if (top_k < 1 || top_k > 32 || top_k > usable) return fail(QS_EINVAL, "top_k %d is not in 1 .. %d", top_k, usable < 32 ? usable : 32);
    if (n_rows < 0 || n_rows > INT32_MAX) return fail(QS_EINVAL, "row count %lld is not in 0 .. 2^31 - 1", (long long)n_rows);
    if (logits_row_stride < n_experts) return fail(QS_EINVAL, "logits row stride %lld < %d experts", (long long)logits_row_stride, n_experts);
    if (n_rows == 0) return QS_OK;
    if (!logits || !ids || !weights) return fail(QS_EINVAL, "null logits, ids or weights");
    if (!aligned(logits, src_size(logits_type)) || !aligned(ids, 4) || !aligned(weights, 4) || (bias && !aligned(bias, 4)))
        return fail(QS_EINVAL, "a pointer is not aligned to its elements");
    CurrentContextGuard keep;
    int device, rc;
    DeviceState* d;
    if ((rc = device_of(logits, "logits", &device, &d))) return rc;
    if ((rc = check_on_device(ids, device, "ids")) || (rc = check_on_device(weights, device, "weights")) ||
        (bias && (rc = check_on_device(bias, device, "bias"))))
        return rc;
    qs::RouteCall c;
    c.logits = logits;
    c.logits_type = logits_type;
    c.logits_stride = logits_row_stride;
    c.n_rows = n_rows;
    c.n_experts = n_experts;
    c.top_k = top_k;
    c.n_groups = n_groups;
    c.groups_kept = groups_kept;
    c.sigmoid = score == QS_SCORE_SIGMOID;
    c.group_top2 = group_score == QS_GROUP_TOP2;
    c.renormalize = renormalize != 0;
    c.bias = bias;
    c.scale = scale;
    c.ids = ids;
    c.weights = weights;
    cudaError_t e = qs::launch_route(c, qs::LaunchCtx{static_cast<cudaStream_t>(stream), device, d->num_sms});
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "route launch");
}

QS_API int qs_expert_plan(const int32_t* ids, int64_t n_slots, int n_experts, int32_t* order, int32_t* offsets, void* stream) {
    if (n_experts < 1 || n_experts > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts are not in 1 .. %d", n_experts, QS_MAX_EXPERTS);
    if (n_slots < 0 || n_slots > 1 << 20) return fail(QS_EINVAL, "slot count %lld is not in 0 .. 2^20", (long long)n_slots);
    if (!offsets || (n_slots > 0 && (!ids || !order))) return fail(QS_EINVAL, "null ids, order or offsets");
    if (!aligned(ids, 4) || !aligned(order, 4) || !aligned(offsets, 4)) return fail(QS_EINVAL, "a pointer is not aligned to its elements");
    CurrentContextGuard keep;
    int device, rc;
    DeviceState* d;
    if ((rc = device_of(offsets, "offsets", &device, &d))) return rc;
    if (n_slots > 0 && ((rc = check_on_device(ids, device, "ids")) || (rc = check_on_device(order, device, "order")))) return rc;
    cudaError_t e = qs::launch_expert_plan(ids, (int)n_slots, n_experts, order, offsets, qs::LaunchCtx{static_cast<cudaStream_t>(stream), device, d->num_sms});
    return e == cudaSuccess ? QS_OK : cuda_fail(e, "expert plan launch");
}

QS_API int qs_matmul_workspace(int ggml_type, int64_t n, int64_t k, int64_t n_rows, int out_type, int64_t* bytes) {
    const TypeInfo* ti;
    if (!is_src(out_type)) return fail(QS_EINVAL, "output type %d is not F32/F16/BF16", out_type);
    if (int rc = check_mm(ggml_type, n, k, n_rows, 1, &ti)) return rc;
    if (bytes) *bytes = mm_plan(ggml_type, n, k, n_rows, 1, n_rows, false, false, out_type != QS_SRC_BF16).bytes;
    return QS_OK;
}

QS_API int qs_matmul(int ggml_type, const void* w, int64_t w_row_bytes, int64_t n, int64_t k, const void* x, int64_t x_row_bytes, int64_t n_rows,
                     void* out, int out_type, int64_t out_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    const TypeInfo* ti;
    int rc = check_mm(ggml_type, n, k, n_rows, 1, &ti);
    if (rc) return rc;
    if (n_rows == 0) return QS_OK;
    if ((rc = check_mm_operands(ti, w, w_row_bytes, k, x, x_row_bytes, out, out_type, out_row_stride, n))) return rc;
    const MmPlan p = mm_plan(ggml_type, n, k, n_rows, 1, n_rows, false, false, out_type != QS_SRC_BF16);
    if ((rc = check_workspace(workspace, workspace_bytes, p.bytes))) return rc;
    CurrentContextGuard keep;
    int device;
    DeviceState* d;
    if ((rc = device_of(w, "w", &device, &d))) return rc;
    if ((rc = check_on_device(x, device, "x")) || (rc = check_on_device(out, device, "out")) ||
        (p.bytes && (rc = check_on_device(workspace, device, "workspace"))))
        return rc;
    qs::MmArgs a;
    memset(&a, 0, sizeof(a));
    a.w = static_cast<const uint8_t*>(w);
    a.w_row = w_row_bytes;
    a.x = static_cast<const uint8_t*>(x);
    a.x_row = x_row_bytes;
    a.x_div = 1;
    a.n = (int)n;
    a.slots = (int)n_rows;
    a.out = out;
    a.out_stride = out_row_stride;
    a.out_type = out_type;
    a.kgrid = qs::iq_kgrid(d->iq, ggml_type);
    a.fault = d->fault;
    return run_mm(ggml_type, p, a, k, n_rows, 1, nullptr, nullptr, workspace, qs::LaunchCtx{static_cast<cudaStream_t>(stream), device, d->num_sms});
}

QS_API int qs_matmul_experts_workspace(int ggml_type, int n_experts, int64_t n, int64_t k, int64_t n_tokens, int top_k, int x_per_slot, int sum,
                                       int out_type, int64_t* bytes) {
    const TypeInfo* ti;
    if (!is_src(out_type)) return fail(QS_EINVAL, "output type %d is not F32/F16/BF16", out_type);
    if (n_experts < 1 || n_experts > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts are not in 1 .. %d", n_experts, QS_MAX_EXPERTS);
    if (top_k < 1 || top_k > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts per token are not in 1 .. %d", top_k, QS_MAX_EXPERTS);
    if (int rc = check_mm(ggml_type, n, k, n_tokens, top_k, &ti)) return rc;
    if (bytes) *bytes = mm_plan(ggml_type, n, k, n_tokens * top_k, n_experts, x_per_slot ? n_tokens * top_k : n_tokens, true, sum != 0,
                                out_type != QS_SRC_BF16).bytes;
    return QS_OK;
}

QS_API int qs_matmul_experts(int ggml_type, const void* w, int64_t w_row_bytes, int64_t w_expert_bytes, int n_experts, int64_t n, int64_t k,
                             const void* x, int64_t x_row_bytes, int x_per_slot, const int32_t* ids, const int32_t* order,
                             const int32_t* offsets, int64_t n_tokens, int top_k, const float* weights, void* out, int out_type,
                             int64_t out_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    const TypeInfo* ti;
    int rc;
    if (n_experts < 1 || n_experts > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts are not in 1 .. %d", n_experts, QS_MAX_EXPERTS);
    if (top_k < 1 || top_k > QS_MAX_EXPERTS) return fail(QS_EINVAL, "%d experts per token are not in 1 .. %d", top_k, QS_MAX_EXPERTS);
    if ((rc = check_mm(ggml_type, n, k, n_tokens, top_k, &ti))) return rc;
    if (n_tokens == 0) return QS_OK;
    if ((rc = check_mm_operands(ti, w, w_row_bytes, k, x, x_row_bytes, out, out_type, out_row_stride, n))) return rc;
    if (w_expert_bytes < n * w_row_bytes || w_expert_bytes % block_align(ggml_type))
        return fail(QS_EINVAL, "expert stride %lld must be a multiple of %d and at least %lld", (long long)w_expert_bytes, block_align(ggml_type), (long long)(n * w_row_bytes));
    if (!ids || !order || !offsets) return fail(QS_EINVAL, "null ids, order or offsets");
    if (!aligned(ids, 4) || !aligned(order, 4) || !aligned(offsets, 4) || (weights && !aligned(weights, 4)))
        return fail(QS_EINVAL, "a pointer is not aligned to its elements");
    const int64_t slots = n_tokens * top_k, x_rows = x_per_slot ? slots : n_tokens;
    const MmPlan p = mm_plan(ggml_type, n, k, slots, n_experts, x_rows, true, weights != nullptr, out_type != QS_SRC_BF16);
    if ((rc = check_workspace(workspace, workspace_bytes, p.bytes))) return rc;
    CurrentContextGuard keep;
    int device;
    DeviceState* d;
    if ((rc = device_of(w, "w", &device, &d))) return rc;
    if ((rc = check_on_device(x, device, "x")) || (rc = check_on_device(out, device, "out")) || (rc = check_on_device(ids, device, "ids")) ||
        (rc = check_on_device(order, device, "order")) || (rc = check_on_device(offsets, device, "offsets")) ||
        (weights && (rc = check_on_device(weights, device, "weights"))) || (p.bytes && (rc = check_on_device(workspace, device, "workspace"))))
        return rc;
    qs::MmArgs a;
    memset(&a, 0, sizeof(a));
    a.w = static_cast<const uint8_t*>(w);
    a.w_row = w_row_bytes;
    a.w_exp = w_expert_bytes;
    a.x = static_cast<const uint8_t*>(x);
    a.x_row = x_row_bytes;
    a.x_div = x_per_slot ? 1 : top_k;
    a.n = (int)n;
    a.slots = (int)slots;
    a.order = order;
    a.offsets = offsets;
    a.n_exp = n_experts;
    a.out = out;
    a.out_stride = out_row_stride;
    a.out_type = out_type;
    a.kgrid = qs::iq_kgrid(d->iq, ggml_type);
    a.fault = d->fault;
    return run_mm(ggml_type, p, a, k, x_rows, top_k, weights, ids, workspace,
                  qs::LaunchCtx{static_cast<cudaStream_t>(stream), device, d->num_sms});
}

}  // extern "C"
