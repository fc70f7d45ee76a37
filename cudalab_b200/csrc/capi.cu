// C ABI of libcudalab_gemv.so (declarations: include/cudalab_gemv.h).
//
// Plain pointers and sizes only.  This layer owns: the variant registry
// lookup, the pointer/size contract checks that do not need tensor metadata,
// status codes + a per-thread error message, and the native launch-loop timer.
// Tensor-level checks (dims, dtypes, devices, contiguity) are made by the host
// wrapper before the call, in the order of the reference extension.
#include <cuda.h>  // CUcontext / CUresult types; the driver functions come via the runtime
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/cudalab_gemv.h"
#include "gemv_launch.h"
#include "gemv_quantize.h"
#include "kv_layout.cuh"

namespace {

thread_local std::string g_last_error;

int fail(int code, const std::string& msg) {
    g_last_error = msg;
    return code;
}

int cuda_fail(cudaError_t e, const char* what) {
    return fail(CL_ERR_CUDA, std::string(what) + ": " + cudaGetErrorName(e) + " (" +
                                 cudaGetErrorString(e) + ")");
}

const clb::VariantDesc* find(const clb::VariantDesc* table, int n, const char* name) {
    if (name == nullptr) return nullptr;
    for (int i = 0; i < n; ++i)
        if (std::strcmp(table[i].name, name) == 0) return &table[i];
    return nullptr;
}

std::string unknown_msg(const char* op, const clb::VariantDesc* table, int n, const char* name) {
    std::vector<std::string> names;
    for (int i = 0; i < n; ++i)
        if (!table[i].quarantined) names.emplace_back(table[i].name);
    std::sort(names.begin(), names.end());
    std::string s = std::string("unknown ") + op + " variant '" + (name ? name : "(null)") +
                    "'; available: ";
    for (auto& v : names) s += v + " ";
    return s;
}

int list_variants(const clb::VariantDesc* table, int n, int which, char* buf, size_t len,
                  size_t* needed) {
    std::vector<std::string> names;
    for (int i = 0; i < n; ++i) {
        const bool q = table[i].quarantined;
        if (which == CL_VARIANTS_NORMAL && q) continue;
        if (which == CL_VARIANTS_QUARANTINED && !q) continue;
        names.emplace_back(table[i].name);
    }
    std::sort(names.begin(), names.end());
    std::string joined;
    for (size_t i = 0; i < names.size(); ++i) {
        if (i) joined += '\n';
        joined += names[i];
    }
    if (needed) *needed = joined.size() + 1;
    if (which != CL_VARIANTS_NORMAL && which != CL_VARIANTS_ALL && which != CL_VARIANTS_QUARANTINED)
        return fail(CL_ERR_INVALID_ARGUMENT, "list_variants: unknown selector");
    if (buf == nullptr || len < joined.size() + 1)
        return fail(CL_ERR_BUFFER_TOO_SMALL, "list_variants: buffer too small");
    std::memcpy(buf, joined.c_str(), joined.size() + 1);
    return CL_OK;
}

// Shared argument checks.  is_int4 adds the group-size contract K % 128 == 0;
// `scale` may be null only for the dense GEMV (pass its W instead).
int check_args(const char* op, const void* W, const void* scale, const void* x, const void* out,
               int64_t N, int64_t K, bool is_int4) {
    if (N <= 0) return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": N must be > 0");
    if (K <= 0) return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": K must be > 0");
    if (is_int4 && (K % 128) != 0)
        return fail(CL_ERR_INVALID_ARGUMENT,
                    std::string(op) + ": K must be divisible by 128 (group_size=128)");
    if (N > (int64_t)1 << 31)
        return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": N exceeds 2^31 rows");
    if (!W || !scale || !x || !out)
        return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": null device pointer");
    return CL_OK;
}

int run(const clb::VariantDesc* table, int n, const char* op, const char* variant, const void* W,
        const void* scale, const void* x, void* out, int64_t N, int64_t K, void* stream,
        uint32_t flags, bool is_int4) {
    const clb::VariantDesc* v = find(table, n, variant);
    if (!v) return fail(CL_ERR_UNKNOWN_VARIANT, unknown_msg(op, table, n, variant));
    const int rc = check_args(op, W, scale, x, out, N, K, is_int4);
    if (rc != CL_OK) return rc;
    const clb::GemvArgs a{W, scale, x, out, N, K, 1, K, N};
    cudaError_t e = v->fn(a, static_cast<cudaStream_t>(stream), flags);
    if (e != cudaSuccess) return cuda_fail(e, "kernel launch");
    return CL_OK;
}

// Batched: X [M, K] -> Y [M, N], both row-major and contiguous; the
// tensor-core kernels take up to 16 activation rows per launch.
int run_batched(const clb::VariantDesc* table, int n, const char* op, const char* variant,
                const void* W, const void* scale, const void* X, void* Y, int64_t M, int64_t N,
                int64_t K, void* stream, uint32_t flags, bool is_int4) {
    const clb::VariantDesc* v = find(table, n, variant);
    if (!v) return fail(CL_ERR_UNKNOWN_VARIANT, unknown_msg(op, table, n, variant));
    if (M <= 0) return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": M must be > 0");
    const int rc = check_args(op, W, scale, X, Y, N, K, is_int4);
    if (rc != CL_OK) return rc;
    constexpr int64_t kPass = 16;
    for (int64_t m0 = 0; m0 < M; m0 += kPass) {
        const clb::GemvArgs a{W, scale, static_cast<const uint16_t*>(X) + m0 * K,
                              static_cast<uint16_t*>(Y) + m0 * N, N, K,
                              std::min<int64_t>(kPass, M - m0), K, N};
        cudaError_t e = v->fn(a, static_cast<cudaStream_t>(stream), flags);
        if (e != cudaSuccess) return cuda_fail(e, "kernel launch");
    }
    return CL_OK;
}

int timing(const clb::VariantDesc* table, int n, const char* op, const char* variant,
           const void* W, const void* scale, const void* x, void* out, int64_t N, int64_t K,
           int64_t warmup, int64_t n_windows, int64_t lpw, void* stream_v, uint32_t flags,
           double* per_window_us, bool is_int4) {
    const clb::VariantDesc* v = find(table, n, variant);
    if (!v) return fail(CL_ERR_UNKNOWN_VARIANT, unknown_msg(op, table, n, variant));
    if (warmup < 0) return fail(CL_ERR_INVALID_ARGUMENT, "warmup must be >= 0");
    if (n_windows < 1) return fail(CL_ERR_INVALID_ARGUMENT, "n_windows must be >= 1");
    if (lpw < 1) return fail(CL_ERR_INVALID_ARGUMENT, "launches_per_window must be >= 1");
    if (!per_window_us) return fail(CL_ERR_INVALID_ARGUMENT, "per_window_us is null");
    int rc = check_args(op, W, scale, x, out, N, K, is_int4);
    if (rc != CL_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream_v);
    const clb::GemvArgs a{W, scale, x, out, N, K, 1, K, N};
    for (int64_t i = 0; i < warmup; ++i) {
        cudaError_t e = v->fn(a, s, flags);
        if (e != cudaSuccess) return cuda_fail(e, "warmup launch");
    }
    cudaError_t e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail(e, "warmup synchronize");
    cudaEvent_t ev0, ev1;
    if ((e = cudaEventCreate(&ev0)) != cudaSuccess) return cuda_fail(e, "event create");
    if ((e = cudaEventCreate(&ev1)) != cudaSuccess) {
        cudaEventDestroy(ev0);
        return cuda_fail(e, "event create");
    }
    rc = CL_OK;
    for (int64_t w = 0; w < n_windows && rc == CL_OK; ++w) {
        if ((e = cudaEventRecord(ev0, s)) != cudaSuccess) { rc = cuda_fail(e, "event record"); break; }
        for (int64_t i = 0; i < lpw; ++i) {
            e = v->fn(a, s, flags);
            if (e != cudaSuccess) { rc = cuda_fail(e, "timed launch"); break; }
        }
        if (rc != CL_OK) break;
        if ((e = cudaEventRecord(ev1, s)) != cudaSuccess) { rc = cuda_fail(e, "event record"); break; }
        if ((e = cudaEventSynchronize(ev1)) != cudaSuccess) { rc = cuda_fail(e, "event sync"); break; }
        float ms = 0.f;
        if ((e = cudaEventElapsedTime(&ms, ev0, ev1)) != cudaSuccess) { rc = cuda_fail(e, "elapsed"); break; }
        per_window_us[w] = (double)ms * 1e3 / (double)lpw;
    }
    cudaEventDestroy(ev0);
    cudaEventDestroy(ev1);
    return rc;
}

const clb::ShardedVariantDesc* find_sharded(const clb::ShardedVariantDesc* t, int n,
                                             const char* name) {
    if (name == nullptr) return nullptr;
    for (int i = 0; i < n; ++i)
        if (std::strcmp(t[i].name, name) == 0) return &t[i];
    return nullptr;
}

int run_sharded(const clb::ShardedVariantDesc* table, int n, const char* op, const char* variant,
                const void* W, const void* scale, const void* x, int64_t M, void* const* y_peers,
                void* const* flag_peers, int rank, int world, int64_t row0, int64_t N_shard,
                int64_t N_total, int64_t K, void* stream, uint32_t flags, bool is_int4) {
    const std::string o(op);
    const clb::ShardedVariantDesc* v = find_sharded(table, n, variant);
    if (!v) {
        std::string m = "unknown " + o + " sharded variant '" + (variant ? variant : "(null)") +
                        "'; available: ";
        for (int i = 0; i < n; ++i) m += std::string(table[i].name) + " ";
        return fail(CL_ERR_UNKNOWN_VARIANT, m);
    }
    int rc = check_args(op, W, scale, x, y_peers, N_shard, K, is_int4);
    if (rc != CL_OK) return rc;
    if (M < 1 || M > 16)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: M must be in [1, 16]");
    if (world < 1 || world > CL_MAX_PEERS)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: world must be in [1, 8]");
    if (rank < 0 || rank >= world)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: rank out of range");
    if (row0 < 0 || N_total <= 0 || row0 + N_shard > N_total)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: shard rows outside [0, N_total)");
    if (!is_int4 && (K % 64) != 0)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: K must be divisible by 64");
    if ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(x)) & 15u)
        return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: W and x must be 16-byte aligned");
    if (!flag_peers) return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: null flag pointers");
    clb::PeerArgs pa{};
    for (int p = 0; p < world; ++p) {
        if (!y_peers[p] || !y_peers[world + p] || !flag_peers[p])
            return fail(CL_ERR_INVALID_ARGUMENT, o + "_sharded: null peer pointer");
        pa.y[0][p] = y_peers[p];
        pa.y[1][p] = y_peers[world + p];
        pa.flag[p] = static_cast<unsigned*>(flag_peers[p]);
    }
    pa.row0 = row0;
    pa.rank = rank;
    pa.world = world;
    const clb::GemvArgs a{W, scale, x, nullptr, N_shard, K, M, K, N_total};
    cudaError_t e = v->fn(a, pa, static_cast<cudaStream_t>(stream), flags);
    if (e != cudaSuccess) {
        char ctx[160];
        std::snprintf(ctx, sizeof ctx, "sharded kernel launch (rank %d/%d, rows %lld+%lld of %lld, K %lld)",
                      rank, world, (long long)row0, (long long)N_shard, (long long)N_total,
                      (long long)K);
        return cuda_fail(e, ctx);
    }
    return CL_OK;
}

// ---- the fused single-GPU step without an allocated flag block ----
//
// Scratch of cl_int4gemv_fused_noalloc: one flag block (CL_PEER_FLAG_BYTES of
// arrival epochs, CTA ticket and step counter), the only memory besides its
// inputs and outputs that the fused kernel touches.  It is a file-scope
// device array, so it costs no allocation; every GPU that loads the library
// holds these 256 bytes until the process exits.  Host code must not hand
// `g_noalloc_flags` to a kernel: on the host the name stands for a host-side
// copy, so its device address is looked up once per device.
constexpr size_t kNoAllocScratchBytes = 256;
static_assert(kNoAllocScratchBytes >= CL_PEER_FLAG_BYTES, "room for one flag block");
static __device__ __align__(256) unsigned char g_noalloc_flags[kNoAllocScratchBytes];

constexpr int kNoAllocMaxDevices = 64;
std::mutex g_noalloc_mu;
struct NoAllocSlot {
    void* addr = nullptr;
    unsigned long long ctx_id = 0;  // context the address belongs to (0: unknown)
};
NoAllocSlot g_noalloc_slot[kNoAllocMaxDevices];

// Unique id of the calling thread's current CUDA context, 0 when the driver
// cannot tell.  The two driver functions are fetched through the runtime, so
// the library keeps no link-time dependency on the driver library.
unsigned long long current_context_id() {
    using GetCurrent = CUresult (*)(CUcontext*);
    using GetId = CUresult (*)(CUcontext, unsigned long long*);
    static GetCurrent get_current = nullptr;
    static GetId get_id = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            get_current = reinterpret_cast<GetCurrent>(p);
        p = nullptr;
        if (cudaGetDriverEntryPoint("cuCtxGetId", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            get_id = reinterpret_cast<GetId>(p);
    });
    CUcontext ctx = nullptr;
    unsigned long long id = 0;
    if (!get_current || !get_id || get_current(&ctx) != CUDA_SUCCESS || ctx == nullptr ||
        get_id(ctx, &id) != CUDA_SUCCESS)
        return 0;
    return id;
}

// Device address of the flag block on the current device.  Set-up happens on
// the first call per device, with that device current, and again whenever
// the device's current context differs from the one the address was looked
// up in (after a cudaDeviceReset the runtime loads the library's module into
// a new context, at a new address); when the context id cannot be read the
// address is looked up on every call.
int noalloc_flag_block(void** out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "int4gemv_fused_noalloc: cudaGetDevice");
    if (dev < 0 || dev >= kNoAllocMaxDevices)
        return fail(CL_ERR_INVALID_ARGUMENT,
                    "int4gemv_fused_noalloc: device ordinal must be below 64");
    std::lock_guard<std::mutex> lock(g_noalloc_mu);
    NoAllocSlot& slot = g_noalloc_slot[dev];
    const unsigned long long ctx = slot.addr ? current_context_id() : 0;
    if (slot.addr == nullptr || ctx == 0 || ctx != slot.ctx_id) {
        void* p = nullptr;
        e = cudaGetSymbolAddress(&p, g_noalloc_flags);
        if (e != cudaSuccess)
            return cuda_fail(e, "int4gemv_fused_noalloc: cudaGetSymbolAddress(flag block)");
        slot.addr = p;
        slot.ctx_id = current_context_id();  // the lookup made the context current
    }
    *out = slot.addr;
    return CL_OK;
}

}  // namespace

extern "C" {

const char* cl_version(void) { return "cudalab-b200 0.1.0 (sm_100a)"; }

const char* cl_last_error(void) { return g_last_error.c_str(); }

int cl_device_status(int clear, int* status_out) {
    if (!status_out) return fail(CL_ERR_INVALID_ARGUMENT, "status_out is null");
    // one word per translation unit with a status; the first nonzero one is reported
    cudaError_t (*const words[])(int, int*) = {clb::read_device_status,
                                               clb::read_kv_attention_status, clb::read_kv_prefix_status,
                                               clb::read_kv_status,
                                               clb::read_qknorm_rope_status};
    int status = 0;
    for (auto read : words) {
        int v = 0;
        cudaError_t e = read(clear, &v);
        if (e != cudaSuccess) return cuda_fail(e, "read device status");
        if (status == 0) status = v;
    }
    *status_out = status;
    return CL_OK;
}

int cl_set_wait_budget(int64_t cycles, int64_t* previous) {
    const long long prev = clb::set_wait_budget((long long)cycles);
    if (previous) *previous = (int64_t)prev;
    return CL_OK;
}

// ---- INT4 ----
int cl_int4gemv_ex(const char* variant, const uint8_t* W_packed, const void* scale, const void* x,
                   void* out, int64_t N, int64_t K, void* stream, uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = clb::int4_variants(&n);
    return run(t, n, "int4gemv", variant, W_packed, scale, x, out, N, K, stream, flags, true);
}

int cl_int4gemv(const char* variant, const uint8_t* W_packed, const void* scale, const void* x,
                void* out, int64_t N, int64_t K, void* stream) {
    return cl_int4gemv_ex(variant, W_packed, scale, x, out, N, K, stream, 0u);
}

int cl_int4gemv_batched(const char* variant, const uint8_t* W_packed, const void* scale,
                        const void* X, void* Y, int64_t M, int64_t N, int64_t K, void* stream,
                        uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = clb::int4_variants(&n);
    return run_batched(t, n, "int4gemv", variant, W_packed, scale, X, Y, M, N, K, stream, flags,
                       true);
}

int cl_int4gemv_native_timing(const char* variant, const uint8_t* W_packed, const void* scale,
                              const void* x, void* out, int64_t N, int64_t K, int64_t warmup,
                              int64_t n_windows, int64_t launches_per_window, void* stream,
                              uint32_t flags, double* per_window_us) {
    int n = 0;
    const clb::VariantDesc* t = clb::int4_variants(&n);
    return timing(t, n, "int4gemv", variant, W_packed, scale, x, out, N, K, warmup, n_windows,
                  launches_per_window, stream, flags, per_window_us, true);
}

int cl_int4gemv_list_variants(int which, char* buf, size_t buf_len, size_t* needed) {
    int n = 0;
    const clb::VariantDesc* t = clb::int4_variants(&n);
    return list_variants(t, n, which, buf, buf_len, needed);
}

// ---- RMSNorm and the fused RMSNorm -> INT4 GEMV ----
int cl_rmsnorm_f16(const void* X, const void* weight, float eps, void* Y, int64_t M, int64_t H,
                   void* stream, uint32_t flags) {
    if (M <= 0) return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: M must be > 0");
    if (H <= 0) return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: H must be > 0");
    if (H % 8 != 0) return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: H must be a multiple of 8");
    if (H > 3 * ((int64_t)1 << 20))
        return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: H exceeds 3 * 2^20 halves");
    if (M > INT32_MAX) return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: M exceeds 2^31 - 1 rows");
    if (!(eps >= 0.f) || !std::isfinite(eps))
        return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: eps must be finite and >= 0");
    if (!X || !weight || !Y) return fail(CL_ERR_INVALID_ARGUMENT, "rmsnorm: null device pointer");
    cudaError_t e = clb::launch_rmsnorm_f16(X, weight, eps, Y, M, H,
                                            static_cast<cudaStream_t>(stream), flags);
    if (e != cudaSuccess) return cuda_fail(e, "rmsnorm launch");
    return CL_OK;
}

int cl_int4gemv_rmsnorm(const char* variant, const uint8_t* W_packed, const void* scale,
                        const void* X, const void* norm_weight, float eps, void* Y, int64_t M,
                        int64_t N, int64_t K, void* stream, uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = clb::int4_rmsnorm_variants(&n);
    const char* op = "int4gemv_rmsnorm";
    const clb::VariantDesc* v = find(t, n, variant);
    if (!v) return fail(CL_ERR_UNKNOWN_VARIANT, unknown_msg(op, t, n, variant));
    if (M <= 0) return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": M must be > 0");
    const int rc = check_args(op, W_packed, scale, X, Y, N, K, true);
    if (rc != CL_OK) return rc;
    if (!norm_weight) return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": null norm weight");
    if (!(eps >= 0.f) || !std::isfinite(eps))
        return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": eps must be finite and >= 0");
    constexpr int64_t kPass = 16;
    for (int64_t m0 = 0; m0 < M; m0 += kPass) {
        clb::GemvArgs a{W_packed, scale, static_cast<const uint16_t*>(X) + m0 * K,
                        static_cast<uint16_t*>(Y) + m0 * N, N, K,
                        std::min<int64_t>(kPass, M - m0), K, N};
        a.norm_w = norm_weight;
        a.norm_eps = eps;
        cudaError_t e = v->fn(a, static_cast<cudaStream_t>(stream), flags);
        if (e != cudaSuccess) return cuda_fail(e, "kernel launch");
    }
    return CL_OK;
}

// ---- INT8 ----
int cl_qgemv_ex(const char* variant, const int8_t* W_q, const float* scale, const void* x,
                void* out, int64_t N, int64_t K, void* stream, uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = clb::int8_variants(&n);
    return run(t, n, "qgemv", variant, W_q, scale, x, out, N, K, stream, flags, false);
}

int cl_qgemv(const char* variant, const int8_t* W_q, const float* scale, const void* x, void* out,
             int64_t N, int64_t K, void* stream) {
    return cl_qgemv_ex(variant, W_q, scale, x, out, N, K, stream, 0u);
}

int cl_qgemv_batched(const char* variant, const int8_t* W_q, const float* scale, const void* X,
                     void* Y, int64_t M, int64_t N, int64_t K, void* stream, uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = clb::int8_variants(&n);
    return run_batched(t, n, "qgemv", variant, W_q, scale, X, Y, M, N, K, stream, flags, false);
}

int cl_qgemv_native_timing(const char* variant, const int8_t* W_q, const float* scale,
                           const void* x, void* out, int64_t N, int64_t K, int64_t warmup,
                           int64_t n_windows, int64_t launches_per_window, void* stream,
                           uint32_t flags, double* per_window_us) {
    int n = 0;
    const clb::VariantDesc* t = clb::int8_variants(&n);
    return timing(t, n, "qgemv", variant, W_q, scale, x, out, N, K, warmup, n_windows,
                  launches_per_window, stream, flags, per_window_us, false);
}

int cl_qgemv_list_variants(int which, char* buf, size_t buf_len, size_t* needed) {
    int n = 0;
    const clb::VariantDesc* t = clb::int8_variants(&n);
    return list_variants(t, n, which, buf, buf_len, needed);
}

// ---- quantisation ----
static const clb::VariantDesc* gemv_table(int dtype, int* n) {
    if (dtype != CL_DTYPE_F16 && dtype != CL_DTYPE_F32) return nullptr;
    return clb::gemv_variants(dtype, n);
}

int cl_gemv_ex(const char* variant, const void* W, const void* x, void* out, int64_t N, int64_t K,
               int dtype, void* stream, uint32_t flags) {
    int n = 0;
    const clb::VariantDesc* t = gemv_table(dtype, &n);
    if (!t) return fail(CL_ERR_INVALID_ARGUMENT, "gemv: dtype must be CL_DTYPE_F16 or CL_DTYPE_F32");
    return run(t, n, "gemv", variant, W, W, x, out, N, K, stream, flags, false);
}

int cl_gemv(const char* variant, const void* W, const void* x, void* out, int64_t N, int64_t K,
            int dtype, void* stream) {
    return cl_gemv_ex(variant, W, x, out, N, K, dtype, stream, 0u);
}

int cl_gemv_native_timing(const char* variant, const void* W, const void* x, void* out, int64_t N,
                          int64_t K, int dtype, int64_t warmup, int64_t n_windows,
                          int64_t launches_per_window, void* stream, uint32_t flags,
                          double* per_window_us) {
    int n = 0;
    const clb::VariantDesc* t = gemv_table(dtype, &n);
    if (!t) return fail(CL_ERR_INVALID_ARGUMENT, "gemv: dtype must be CL_DTYPE_F16 or CL_DTYPE_F32");
    return timing(t, n, "gemv", variant, W, W, x, out, N, K, warmup, n_windows,
                  launches_per_window, stream, flags, per_window_us, false);
}

int cl_gemv_list_variants(int which, char* buf, size_t buf_len, size_t* needed) {
    int n = 0;
    const clb::VariantDesc* t = clb::gemv_variants(CL_DTYPE_F16, &n);  // same names for fp32
    return list_variants(t, n, which, buf, buf_len, needed);
}

int cl_int4gemv_quantize(const void* W, int64_t N, int64_t K, uint8_t* W_packed, void* scale,
                         void* stream) {
    if (N <= 0 || K <= 0) return fail(CL_ERR_INVALID_ARGUMENT, "int4gemv_quantize: N, K must be > 0");
    if (K % 128 != 0)
        return fail(CL_ERR_INVALID_ARGUMENT,
                    "int4gemv_quantize: K must be divisible by 128 (group_size=128)");
    if (!W || !W_packed || !scale)
        return fail(CL_ERR_INVALID_ARGUMENT, "int4gemv_quantize: null device pointer");
    if (reinterpret_cast<uintptr_t>(W) & 7u)
        return fail(CL_ERR_INVALID_ARGUMENT, "int4gemv_quantize: W must be 8-byte aligned");
    cudaError_t e = clb::launch_int4_quantize(W, N, K, W_packed, scale,
                                              static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "int4gemv_quantize launch");
    return CL_OK;
}

int cl_qgemv_quantize(const void* W, int64_t N, int64_t K, int8_t* W_q, float* scale,
                      void* stream) {
    if (N <= 0 || K <= 0) return fail(CL_ERR_INVALID_ARGUMENT, "qgemv_quantize: N, K must be > 0");
    if (N > ((int64_t)1 << 31) - 1)
        return fail(CL_ERR_INVALID_ARGUMENT, "qgemv_quantize: N exceeds 2^31 - 1 rows");
    if (!W || !W_q || !scale)
        return fail(CL_ERR_INVALID_ARGUMENT, "qgemv_quantize: null device pointer");
    cudaError_t e = clb::launch_int8_quantize(W, N, K, W_q, scale,
                                              static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "qgemv_quantize launch");
    return CL_OK;
}

// ---- peer buffers and the row-sharded GEMV ----
int cl_peer_alloc(size_t bytes, void** ptr, void* ipc_handle) {
    if (!ptr || !ipc_handle || bytes == 0)
        return fail(CL_ERR_INVALID_ARGUMENT, "peer_alloc: null output or zero size");
    static_assert(sizeof(cudaIpcMemHandle_t) == CL_IPC_HANDLE_BYTES, "IPC handle size");
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, bytes);
    if (e != cudaSuccess) return cuda_fail(e, "peer_alloc: cudaMalloc");
    if ((e = cudaMemset(p, 0, bytes)) != cudaSuccess) {
        cudaFree(p);
        return cuda_fail(e, "peer_alloc: cudaMemset");
    }
    cudaIpcMemHandle_t h;
    if ((e = cudaIpcGetMemHandle(&h, p)) != cudaSuccess) {
        cudaFree(p);
        return cuda_fail(e, "peer_alloc: cudaIpcGetMemHandle");
    }
    std::memcpy(ipc_handle, &h, sizeof(h));
    *ptr = p;
    return CL_OK;
}

int cl_peer_open(const void* ipc_handle, void** peer_ptr) {
    if (!ipc_handle || !peer_ptr) return fail(CL_ERR_INVALID_ARGUMENT, "peer_open: null pointer");
    cudaIpcMemHandle_t h;
    std::memcpy(&h, ipc_handle, sizeof(h));
    cudaError_t e = cudaIpcOpenMemHandle(peer_ptr, h, cudaIpcMemLazyEnablePeerAccess);
    if (e != cudaSuccess) return cuda_fail(e, "peer_open: cudaIpcOpenMemHandle");
    return CL_OK;
}

int cl_peer_close(void* peer_ptr) {
    if (!peer_ptr) return fail(CL_ERR_INVALID_ARGUMENT, "peer_close: null pointer");
    cudaError_t e = cudaIpcCloseMemHandle(peer_ptr);
    if (e != cudaSuccess) return cuda_fail(e, "peer_close: cudaIpcCloseMemHandle");
    return CL_OK;
}

int cl_peer_free(void* ptr) {
    if (!ptr) return fail(CL_ERR_INVALID_ARGUMENT, "peer_free: null pointer");
    cudaError_t e = cudaFree(ptr);
    if (e != cudaSuccess) return cuda_fail(e, "peer_free: cudaFree");
    return CL_OK;
}

int cl_int4gemv_sharded(const char* variant, const uint8_t* W_shard, const void* scale_shard,
                        const void* x, int64_t M, void* const* y_peers, void* const* flag_peers,
                        int rank,
                        int world, int64_t row0, int64_t N_shard, int64_t N_total, int64_t K,
                        void* stream, uint32_t flags) {
    int n = 0;
    const clb::ShardedVariantDesc* t = clb::int4_sharded_variants(&n);
    return run_sharded(t, n, "int4gemv", variant, W_shard, scale_shard, x, M, y_peers, flag_peers,
                       rank, world, row0, N_shard, N_total, K, stream, flags, true);
}

int cl_int4gemv_fused_noalloc(const char* variant, const uint8_t* W_packed, const void* scale,
                              const void* x, int64_t M, void* y, int64_t N, int64_t K,
                              void* stream, uint32_t flags) {
    int n = 0;
    const clb::ShardedVariantDesc* t = clb::int4_sharded_variants(&n);
    // Every check of the launch first, so that a rejected call leaves the
    // stream untouched.
    if (!find_sharded(t, n, variant))
        return fail(CL_ERR_UNKNOWN_VARIANT, std::string("int4gemv_fused_noalloc: unknown variant '") +
                                                (variant ? variant : "(null)") + "'");
    int rc = check_args("int4gemv_fused_noalloc", W_packed, scale, x, y, N, K, true);
    if (rc != CL_OK) return rc;
    if (M < 1 || M > 16)
        return fail(CL_ERR_INVALID_ARGUMENT,
                    "int4gemv_fused_noalloc: M must be in [1, 16] (larger batches: call again "
                    "per 16 rows)");
    if ((reinterpret_cast<uintptr_t>(W_packed) | reinterpret_cast<uintptr_t>(x)) & 15u)
        return fail(CL_ERR_INVALID_ARGUMENT,
                    "int4gemv_fused_noalloc: W_packed and x must be 16-byte aligned");
    void* flag = nullptr;
    rc = noalloc_flag_block(&flag);
    if (rc != CL_OK) return rc;
    // The block keeps the previous call's contents: start every call from zero.
    cudaError_t e = cudaMemsetAsync(flag, 0, CL_PEER_FLAG_BYTES, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "int4gemv_fused_noalloc: clearing the flag block");
    void* ys[2] = {y, y};  // one rank: both step parities write the caller's y
    void* fs[1] = {flag};
    return run_sharded(t, n, "int4gemv", variant, W_packed, scale, x, M, ys, fs, 0, 1, 0, N, N, K,
                       stream, flags, true);
}

int cl_qgemv_sharded(const char* variant, const int8_t* W_shard, const float* scale_shard,
                     const void* x, int64_t M, void* const* y_peers, void* const* flag_peers,
                     int rank,
                     int world, int64_t row0, int64_t N_shard, int64_t N_total, int64_t K,
                     void* stream, uint32_t flags) {
    int n = 0;
    const clb::ShardedVariantDesc* t = clb::int8_sharded_variants(&n);
    return run_sharded(t, n, "qgemv", variant, W_shard, scale_shard, x, M, y_peers, flag_peers,
                       rank, world, row0, N_shard, N_total, K, stream, flags, false);
}

// ---- attention of a decode step over a quantised paged cache ----
namespace {

int bad(const char* op, const char* what) {
    return fail(CL_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// 16-bit element type of the descriptor -> the kernels' type, -1 if neither.
int type16(int dtype) {
    return dtype == CL_DTYPE_F16 ? clb::kTypeF16 : dtype == CL_DTYPE_BF16 ? clb::kTypeBf16 : -1;
}

// The cache's format, shared by the cache and the attention calls.
int check_cache(const char* op, int64_t num_pages, int kv_heads, int head_dim, int bits,
                int page_size) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return bad(op, "head_dim must be 64, 128 or 256");
    if (bits != 8 && bits != 4) return bad(op, "bits must be 8 or 4");
    if (kv_heads <= 0 || kv_heads > 65535) return bad(op, "kv_heads must be in [1, 65535]");
    if (num_pages <= 0 || num_pages > INT32_MAX) return bad(op, "num_pages must be in [1, 2^31)");
    if (page_size <= 0 || page_size % clb::kKvBlock != 0 || page_size > (1 << 20))
        return bad(op, "page_size must be a multiple of 16, at most 2^20");
    return CL_OK;
}

int cache_args(const char* op, const void* k, const void* v, const void* pages, const int64_t* slots,
               const cl_kvcache_desc* d, clb::KvCacheArgs* a) {
    if (!d) return bad(op, "null descriptor");
    if (d->tokens < 0) return bad(op, "tokens must be >= 0");
    const int type = type16(d->dtype);
    if (type < 0) return bad(op, "dtype must be CL_DTYPE_F16 or CL_DTYPE_BF16");
    const int rc = check_cache(op, d->num_pages, d->kv_heads, d->head_dim, d->bits, d->page_size);
    if (rc != CL_OK) return rc;
    if (!pages || (d->tokens > 0 && (!k || !v || !slots))) return bad(op, "null device pointer");
    if (misaligned16(pages)) return bad(op, "pages must be 16-byte aligned");
    if (d->tokens > (((int64_t)1 << 31) - 256) / d->kv_heads)
        return bad(op, "too many tokens for one launch");
    *a = clb::KvCacheArgs{const_cast<uint8_t*>(static_cast<const uint8_t*>(pages)), slots,
                          const_cast<void*>(k), const_cast<void*>(v), d->k_token, d->k_head,
                          d->v_token, d->v_head, d->tokens, d->num_pages, d->kv_heads, d->head_dim,
                          d->bits, d->page_size, type};
    return CL_OK;
}

}  // namespace

int cl_qknorm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                   const float* table, const void* positions, void* q_out, void* k_out,
                   const cl_qknorm_rope_desc* d, void* stream) {
    const char* op = "qknorm_rope";
    if (!d) return bad(op, "null descriptor");
    if (d->tokens < 0) return bad(op, "tokens must be >= 0");
    if (d->q_heads <= 0 || d->kv_heads <= 0 || d->q_heads > (1 << 20) || d->kv_heads > (1 << 20))
        return bad(op, "q_heads and kv_heads must be in [1, 2^20]");
    if (d->head_dim <= 0 || d->head_dim % 16 != 0 || d->head_dim > 256)
        return bad(op, "head_dim must be a multiple of 16, at most 256");
    if (d->rotary <= 0 || d->rotary % 16 != 0 || d->rotary > d->head_dim)
        return bad(op, "rotary must be a multiple of 16, at most head_dim");
    const int type = type16(d->dtype);
    if (type < 0) return bad(op, "dtype must be CL_DTYPE_F16 or CL_DTYPE_BF16");
    if (!(d->eps >= 0.f) || !std::isfinite(d->eps)) return bad(op, "eps must be finite and >= 0");
    if ((q_weight == nullptr) != (k_weight == nullptr))
        return bad(op, "q_weight and k_weight must both be given, or neither");
    if (d->table_rows <= 0) return bad(op, "table_rows must be > 0");
    if (d->tokens == 0) return CL_OK;
    if (!q || !k || !table || !positions || !q_out || !k_out) return bad(op, "null device pointer");
    if (misaligned16(table)) return bad(op, "table must be 16-byte aligned");
    if (d->tokens > (((int64_t)1 << 31) - 256) / ((int64_t)d->q_heads + d->kv_heads))
        return bad(op, "too many tokens for one launch");
    const clb::QkRopeArgs a{{q, k},
                            {q_out, k_out},
                            {q_weight, k_weight},
                            {d->q_token, d->k_token},
                            {d->q_head, d->k_head},
                            {d->q_out_token, d->k_out_token},
                            {d->q_out_head, d->k_out_head},
                            {d->q_heads, d->kv_heads},
                            table,
                            d->table_rows,
                            positions,
                            d->positions64,
                            d->tokens,
                            d->head_dim,
                            d->rotary,
                            d->interleaved,
                            type,
                            d->eps};
    cudaError_t e = clb::launch_qknorm_rope(a, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "qknorm_rope launch");
    return CL_OK;
}

int cl_kvcache_write(const void* k, const void* v, uint8_t* pages, const int64_t* slots,
                     const cl_kvcache_desc* d, void* stream) {
    clb::KvCacheArgs a;
    const int rc = cache_args("kvcache_write", k, v, pages, slots, d, &a);
    if (rc != CL_OK) return rc;
    cudaError_t e = clb::launch_kv_write(a, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "kvcache_write launch");
    return CL_OK;
}

int cl_kvcache_read(const uint8_t* pages, const int64_t* slots, void* k, void* v,
                    const cl_kvcache_desc* d, void* stream) {
    clb::KvCacheArgs a;
    const int rc = cache_args("kvcache_read", k, v, pages, slots, d, &a);
    if (rc != CL_OK) return rc;
    cudaError_t e = clb::launch_kv_read(a, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "kvcache_read launch");
    return CL_OK;
}

int cl_kvattention_workspace(size_t* bytes) {
    if (!bytes) return bad("kvattention_workspace", "bytes is null");
    *bytes = clb::kv_attention_workspace();
    return CL_OK;
}

namespace {

// The launch over the prefix: the whole batch as the new tokens of one
// sequence that sees all of it.
clb::KvAttentionArgs prefix_args(const cl_kvattention_desc* d) {
    clb::KvAttentionArgs f{};
    f.q_new = d->new_tokens > 1 ? d->q_new : d->q_batch;
    f.q_head = d->q_head;
    f.num_pages = d->num_pages;
    f.max_pages = d->prefix_page_count;
    f.fixed_length = d->prefix_length;
    f.batch = 1;
    f.new_tokens = d->batch * d->new_tokens;
    f.kv_heads = d->kv_heads;
    f.group = d->q_heads / d->kv_heads;
    f.head_dim = d->head_dim;
    f.bits = d->bits;
    f.page_size = d->page_size;
    f.scale = d->scale;
    return f;
}

int check_attention(const char* op, const cl_kvattention_desc* d) {
    if (!d) return bad(op, "null descriptor");
    if (type16(d->dtype) < 0) return bad(op, "dtype must be CL_DTYPE_F16 or CL_DTYPE_BF16");
    const int rc = check_cache(op, d->num_pages, d->kv_heads, d->head_dim, d->bits, d->page_size);
    if (rc != CL_OK) return rc;
    if (d->batch < 0 || d->batch > 4096) return bad(op, "batch must be in [0, 4096]");
    if (d->new_tokens <= 0 || d->new_tokens > (1 << 20))
        return bad(op, "new_tokens must be in [1, 2^20]");
    if (d->q_heads <= 0 || d->q_heads % d->kv_heads != 0)
        return bad(op, "q_heads must be a multiple of kv_heads");
    if ((int64_t)d->batch * d->new_tokens * d->q_heads > INT32_MAX)
        return bad(op, "more than 2^31 - 1 query rows");
    if (d->window < 0) return bad(op, "window must be >= 0");
    if (!std::isfinite(d->scale)) return bad(op, "scale must be finite");
    if (d->max_pages < 0 || (int64_t)d->max_pages * d->page_size > INT32_MAX)
        return bad(op, "max_pages * page_size exceeds 2^31 - 1 tokens");
    if (d->prefix_length < 0 || d->prefix_page_count < 0) return bad(op, "negative prefix");
    if (d->prefix_length > 0) {
        if (d->window != 0) return bad(op, "a prefix and a window exclude each other");
        if ((int64_t)d->prefix_page_count * d->page_size > INT32_MAX)
            return bad(op, "prefix_page_count * page_size exceeds 2^31 - 1 tokens");
        if ((int64_t)d->prefix_page_count * d->page_size < d->prefix_length)
            return bad(op, "prefix_pages hold fewer than prefix_length tokens");
        if (d->batch > 1 && d->new_tokens > 1 && d->q_batch != d->new_tokens * d->q_new)
            return bad(op, "with a prefix the q rows must be evenly spaced");
    }
    return CL_OK;
}

}  // namespace

int cl_kvattention_prefix_floats(const cl_kvattention_desc* d, size_t* floats) {
    const char* op = "kvattention_prefix_floats";
    if (!floats) return bad(op, "floats is null");
    const int rc = check_attention(op, d);
    if (rc != CL_OK) return rc;
    *floats = 0;
    if (d->prefix_length == 0 || d->batch == 0) return CL_OK;
    const clb::KvAttentionArgs f = prefix_args(d);
    const int parts = clb::kv_prefix_takes(f) ? clb::kv_prefix_parts(f) : 1;
    *floats = (size_t)parts * d->batch * d->new_tokens * d->q_heads * (d->head_dim + 1);
    return CL_OK;
}

int cl_kvattention(const void* q, const uint8_t* pages, const int32_t* page_table,
                   const int32_t* lengths, const int32_t* prefix_pages, void* out, float* lse,
                   float* prefix_scratch, void* workspace, const cl_kvattention_desc* d,
                   void* stream) {
    const char* op = "kvattention";
    const int rc = check_attention(op, d);
    if (rc != CL_OK) return rc;
    if (d->batch == 0) return CL_OK;
    if (!q || !pages || !out || !workspace || !lengths || (d->max_pages > 0 && !page_table))
        return bad(op, "null device pointer");
    if (misaligned16(pages) || misaligned16(out) || misaligned16(workspace))
        return bad(op, "pages, out and workspace must be 16-byte aligned");
    clb::KvAttentionArgs a{};
    a.q = q;
    a.q_batch = d->q_batch;
    a.q_new = d->q_new;
    a.q_head = d->q_head;
    a.pages = pages;
    a.num_pages = d->num_pages;
    a.table = page_table;
    a.table_stride = d->table_stride;
    a.max_pages = d->max_pages;
    a.lengths = lengths;
    a.fixed_length = -1;
    a.batch = d->batch;
    a.new_tokens = d->new_tokens;
    a.kv_heads = d->kv_heads;
    a.group = d->q_heads / d->kv_heads;
    a.head_dim = d->head_dim;
    a.bits = d->bits;
    a.page_size = d->page_size;
    a.type = type16(d->dtype);
    a.causal = 1;
    // a window that holds every length the page table allows is none
    a.window = d->window < (int64_t)d->max_pages * d->page_size ? d->window : 0;
    a.scale = d->scale;
    a.out = out;
    a.lse = lse;
    a.workspace = workspace;
    if (!clb::kv_attention_fits(a))
        return bad(op, "the page tables span too many blocks for one launch");
    if (!clb::kv_attention_tiles_fit(a)) return bad(op, "too many query rows for one launch");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->prefix_length > 0) {
        if (!prefix_pages || !prefix_scratch) return bad(op, "null prefix pointer");
        if (misaligned16(prefix_scratch)) return bad(op, "prefix_scratch must be 16-byte aligned");
        clb::KvAttentionArgs f = prefix_args(d);
        f.q = q;
        f.pages = pages;
        f.table = prefix_pages;
        f.type = a.type;
        f.workspace = workspace;
        if (!clb::kv_attention_fits(f))
            return bad(op, "the prefix spans too many blocks for one launch");
        const bool tensor = clb::kv_prefix_takes(f);
        if (!tensor && !clb::kv_attention_tiles_fit(f))
            return bad(op, "too many query rows for one launch over the prefix");
        a.front_parts = tensor ? clb::kv_prefix_parts(f) : 1;
        a.front_by_tensor_cores = tensor;
        a.front = f.out_f32 = prefix_scratch;
        a.front_lse = f.lse = prefix_scratch + (size_t)a.front_parts * d->batch * d->new_tokens *
                                                   d->q_heads * d->head_dim;
        const cudaError_t e = tensor ? clb::launch_kv_prefix(f, s) : clb::launch_kv_attention(f, s);
        if (e != cudaSuccess) return cuda_fail(e, "kvattention prefix launch");
    }
    const cudaError_t e = clb::launch_kv_attention(a, s);
    if (e != cudaSuccess) return cuda_fail(e, "kvattention launch");
    return CL_OK;
}

}  // extern "C"
