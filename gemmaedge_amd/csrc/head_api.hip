// C ABI of the answer head (include/gemmaedge_head.h): handles, argument
// checks and launches. Conventions as in sampler_api.hip.
#include <hip/hip_runtime.h>

#include <cstring>
#include <new>

#include "head_internal.h"

struct ge_head {
    int device;
    ge::head::Capacity cap;
    ge::head::Buffers buf;
};

namespace {

int hip_error(hipError_t e, const char* what) {
    (void)hipGetLastError();  // reported here: the next launch's check shall not find it
    char msg[256];
    ge::plan_fail(msg, sizeof(msg), 0, "%s: %s", what, hipGetErrorString(e));
    return ge::report(GE_ERR_DEVICE, msg);
}

// Switches the calling thread to `device` for the lifetime of the object.
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != device) ok = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() {
        int cur = -1;
        if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
    }
};

int check_tensors(const ge_adamw_tensor* t, int count, int state_bits, int64_t& chunks, char* msg, size_t n) {
    using namespace ge;
    if (count < 0 || (count > 0 && !t)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "count %d or tensors is NULL", count);
    if (state_bits != 8 && state_bits != 32) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "state_bits %d", state_bits);
    chunks = 0;
    for (int i = 0; i < count; ++i) {
        const ge_adamw_tensor& x = t[i];
        if (x.n < 0) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "tensor %d: n %lld", i, static_cast<long long>(x.n));
        if (!head::dtype_ok(x.param_dtype) || !head::dtype_ok(x.grad_dtype))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "tensor %d: dtypes %d and %d", i, x.param_dtype, x.grad_dtype);
        if (x.n == 0) continue;
        if (!x.param || !x.grad || !x.m || !x.v || (state_bits == 8 && (!x.m_scale || !x.v_scale)))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "tensor %d: a pointer is NULL", i);
        const size_t ss = state_bits == 8 ? 1 : 4;
        if (!head::aligned_to(x.param, head::elem_size(x.param_dtype)) || !head::aligned_to(x.grad, head::elem_size(x.grad_dtype)) ||
            !head::aligned_to(x.master, 4) || !head::aligned_to(x.m, ss) || !head::aligned_to(x.v, ss) ||
            !head::aligned_to(x.m_scale, 4) || !head::aligned_to(x.v_scale, 4))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "tensor %d is not aligned to its elements", i);
        const int64_t more = x.n / head::kAdamChunk + (x.n % head::kAdamChunk != 0);
        if (more > INT32_MAX - chunks)
            return plan_fail(msg, n, GE_ERR_CAPACITY, "more than %d chunks of %d elements", INT32_MAX, head::kAdamChunk);
        chunks += more;
    }
    return GE_OK;
}

int64_t table_size(int count, int64_t chunks) {
    return static_cast<int64_t>(count) * static_cast<int64_t>(sizeof(ge::head::AdamTensor)) +
           chunks * static_cast<int64_t>(sizeof(ge::head::AdamChunk));
}

}  // namespace

extern "C" {

int ge_head_create(int device, int max_rows, int max_dim, int max_vocab, int dtype, int train, ge_head** out) {
    char msg[256] = "";
    if (!out) return ge::report(GE_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (const int rc = ge::head::check_create(max_rows, max_dim, max_vocab, dtype, msg, sizeof(msg))) return ge::report(rc, msg);
    int n = 0;
    hipDeviceProp_t prop;
    if (hipGetDeviceCount(&n) != hipSuccess || device < 0 || device >= n ||
        hipGetDeviceProperties(&prop, device) != hipSuccess || std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
        ge::plan_fail(msg, sizeof(msg), 0, "device %d is not a gfx950 device (%d devices)", device, n);
        return ge::report(GE_ERR_NO_DEVICE, msg);
    }
    OnDevice guard(device);
    if (!guard.ok) return ge::report(GE_ERR_DEVICE, "hipSetDevice failed");
    ge_head* h = new (std::nothrow) ge_head{};
    if (!h) return ge::report(GE_ERR_DEVICE, "out of host memory");
    h->device = device;
    h->cap = ge::head::Capacity{max_rows, max_dim, max_vocab, dtype, train != 0, 0, 0, 0, 0, 0, 0, 0};
    ge::head::size_workspace(h->cap);
    hipError_t e = hipSuccess;
    auto alloc = [&](auto*& p, int64_t bytes) {
        if (e == hipSuccess && bytes > 0) e = hipMalloc(reinterpret_cast<void**>(&p), static_cast<size_t>(bytes));
    };
    alloc(h->buf.stats, h->cap.stats);
    alloc(h->buf.row, h->cap.row);
    alloc(h->buf.hpack, h->cap.hpack);
    alloc(h->buf.wpack, h->cap.wpack);
    alloc(h->buf.dlogits, h->cap.dlogits);
    alloc(h->buf.dhidden, h->cap.dhidden);
    alloc(h->buf.norm, h->cap.norm);
    if (e != hipSuccess) {
        ge_head_destroy(h);
        return hip_error(e, "ge_head_create");
    }
    *out = h;
    return GE_OK;
}

void ge_head_destroy(ge_head* h) {
    if (!h) return;
    OnDevice guard(h->device);
    (void)hipFree(h->buf.stats);
    (void)hipFree(h->buf.row);
    (void)hipFree(h->buf.hpack);
    (void)hipFree(h->buf.wpack);
    (void)hipFree(h->buf.dlogits);
    (void)hipFree(h->buf.dhidden);
    (void)hipFree(h->buf.norm);
    delete h;
}

static int norm_call(ge_head* h, void* stream, const ge_norm_args* args, bool backward) {
    char msg[256] = "";
    if (!h || !args) return ge::report(GE_ERR_INVALID_ARG, "head or args is NULL");
    if (const int rc = ge::head::check_norm(h->cap, *args, backward, msg, sizeof(msg))) return ge::report(rc, msg);
    OnDevice guard(h->device);
    if (!guard.ok) return ge::report(GE_ERR_DEVICE, "hipSetDevice failed");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = backward ? ge::head::launch_norm_backward(*args, h->cap.dtype, h->buf, st)
                                  : ge::head::launch_norm(*args, h->cap.dtype, st);
    return e == hipSuccess ? GE_OK : hip_error(e, "launch (norm)");
}

int ge_head_norm(ge_head* h, void* stream, const ge_norm_args* args) { return norm_call(h, stream, args, false); }
int ge_head_norm_backward(ge_head* h, void* stream, const ge_norm_args* args) { return norm_call(h, stream, args, true); }

static int loss_call(ge_head* h, void* stream, const ge_loss_args* args, bool backward) {
    char msg[256] = "";
    if (!h || !args) return ge::report(GE_ERR_INVALID_ARG, "head or args is NULL");
    ge::head::LossPlan plan{};
    if (const int rc = ge::head::check_loss(h->cap, *args, backward, plan, msg, sizeof(msg))) return ge::report(rc, msg);
    OnDevice guard(h->device);
    if (!guard.ok) return ge::report(GE_ERR_DEVICE, "hipSetDevice failed");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = backward ? ge::head::launch_loss_backward(*args, h->cap.dtype, plan, h->buf, st)
                                  : ge::head::launch_loss(*args, h->cap.dtype, plan, h->buf, st);
    return e == hipSuccess ? GE_OK : hip_error(e, "launch (loss)");
}

int ge_head_loss(ge_head* h, void* stream, const ge_loss_args* args) { return loss_call(h, stream, args, false); }
int ge_head_loss_backward(ge_head* h, void* stream, const ge_loss_args* args) { return loss_call(h, stream, args, true); }

int ge_adamw_table_bytes(const ge_adamw_tensor* tensors, int count, int state_bits, int64_t* bytes) {
    char msg[256] = "";
    int64_t chunks = 0;
    if (!bytes) return ge::report(GE_ERR_INVALID_ARG, "bytes is NULL");
    *bytes = 0;
    if (const int rc = check_tensors(tensors, count, state_bits, chunks, msg, sizeof(msg))) return ge::report(rc, msg);
    *bytes = table_size(count, chunks);
    return GE_OK;
}

int ge_adamw_table(const ge_adamw_tensor* tensors, int count, int state_bits, void* table, int64_t bytes) {
    char msg[256] = "";
    int64_t chunks = 0;
    if (const int rc = check_tensors(tensors, count, state_bits, chunks, msg, sizeof(msg))) return ge::report(rc, msg);
    if (bytes != table_size(count, chunks) || (bytes > 0 && (!table || !ge::head::aligned_to(table, 8))))
        return ge::report(GE_ERR_INVALID_ARG, "table is NULL, not aligned to 8 bytes or of another size than ge_adamw_table_bytes gives");
    auto* t = static_cast<ge::head::AdamTensor*>(table);
    auto* c = reinterpret_cast<ge::head::AdamChunk*>(t + count);
    int64_t block = 0;
    for (int i = 0; i < count; ++i) {
        t[i] = ge::head::AdamTensor{tensors[i], block};
        block += tensors[i].n / GE_ADAMW_BLOCK + (tensors[i].n % GE_ADAMW_BLOCK != 0);
        const int64_t chunks_i = tensors[i].n / ge::head::kAdamChunk + (tensors[i].n % ge::head::kAdamChunk != 0);
        for (int64_t k = 0; k < chunks_i; ++k) *c++ = ge::head::AdamChunk{i, static_cast<int32_t>(k)};
    }
    return GE_OK;
}

int ge_adamw_step(void* stream, const ge_adamw_args* args) {
    char msg[256] = "";
    if (!args) return ge::report(GE_ERR_INVALID_ARG, "args is NULL");
    const ge_adamw_args& x = *args;
    const int64_t chunk_bytes = x.table_bytes - static_cast<int64_t>(x.count) * static_cast<int64_t>(sizeof(ge::head::AdamTensor));
    const int64_t chunks = chunk_bytes / static_cast<int64_t>(sizeof(ge::head::AdamChunk));
    if (x.count < 0 || chunk_bytes < 0 || chunk_bytes % static_cast<int64_t>(sizeof(ge::head::AdamChunk)) != 0 || chunks > INT32_MAX ||
        (chunks > 0 && (!x.table || !ge::head::aligned_to(x.table, 16))))
        return ge::report(GE_ERR_INVALID_ARG, "table of another size than its count gives, NULL or not aligned to 16 bytes");
    if (x.state_bits != 8 && x.state_bits != 32) return ge::report(GE_ERR_INVALID_ARG, "state_bits is neither 8 nor 32");
    if (!ge::head::aligned_to(x.device_params, 8)) return ge::report(GE_ERR_INVALID_ARG, "device_params is not aligned to 8 bytes");
    if (!x.device_params)
        if (const int rc = ge::head::check_adamw_params(x.params, msg, sizeof(msg))) return ge::report(rc, msg);
    const hipError_t e = ge::head::launch_adamw(x, chunks, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? GE_OK : hip_error(e, "launch (adamw)");
}

}  // extern "C"
