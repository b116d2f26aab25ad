// api.cpp -- the C ABI of libb200attn.so (include/b200attn.h): contexts,
// argument validation with the reference's error wording, workspace
// management and kernel dispatch.  No exception crosses the boundary and no
// call falls back to the CPU.
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <numeric>
#include <string>
#include <vector>

#include "../../include/b200attn.h"
#include "../../include/b200attn_testing.h"
#include "internal.h"

using namespace b2a;

// Counters that are zero between launches, for calls that need more of them than a workspace holds at its
// start (kInlineCounters).  They grow into a new allocation and the old one stays until the context ends,
// since a captured launch goes on counting there.
struct Counters {
    static constexpr int kMost = 48;  // each at least twice the one before
    int* at[kMost] = {};
    int n = 0;
    size_t bytes = 0;  // of the last one
    size_t total = 0;
};

struct b2a_context {
    int device = 0;
    int sm_count = 0;
    std::string last_error;
    size_t ws_limit = 0;  // 0: unlimited
    int* status = nullptr;  // device int[kStatusBufferInts]: error flags, prefill work-item counters
    int* status_host = nullptr;  // pinned int[kStatusWords]: where b2a_check_device_status reads the flags
    // decode workspace: [counters][partials]
    // [counters][slots] (ensure_counted_buffer)
    void* dec_ws = nullptr;
    size_t dec_ws_bytes = 0;
    Counters dec_counters;
    // prefill workspace: rope table + rotated q/k staging
    void* pf_ws = nullptr;
    size_t pf_ws_bytes = 0;
    // float NeoX (cos, sin) table [position][D/2] for positions [0, rope_npos), reused by later
    // calls with the same theta and head dim (rebuilt, on the calling stream, when it does not cover)
    void* rope_tab = nullptr;
    size_t rope_tab_bytes = 0;
    double rope_theta = 0.0;
    int rope_D = 0;
    int rope_npos = 0;
    // attention block: the QKV projection's fp32 rows and the attention output
    void* blk_ws = nullptr;
    size_t blk_ws_bytes = 0;
    // split-K projections: [tile counters][fp32 accumulator], all zero between launches
    void* lin_ws = nullptr;
    size_t lin_ws_bytes = 0;
    // generic-kernel key split: [counters][partial slots]
    void* split_ws = nullptr;
    size_t split_ws_bytes = 0;
    // test hook (b2a_test_inject_wait_timeout): the next tcgen05 attention launch
    // leaves one K/V copy unissued
    bool inject_wait_timeout = false;
    // the inverse frequencies of the last (theta, head dim) a cache call rotated with
    double kv4_inv_freq[kMaxHeadDim / 2] = {};
    double kv4_theta = 0.0;
    int kv4_inv_dim = 0;
    // paged 4-bit cache: [counters][partial slots][plan][q operands][q sums]
    void* kv4_ws = nullptr;
    size_t kv4_ws_bytes = 0;
    Counters kv4_counters;
    // paged cache: [words between blocks][the page operations' lists]
    void* pg_ws = nullptr;
    size_t pg_ws_bytes = 0;
    // b2a_set_decode_early_start: tensor-core decodes launched with programmatic serialisation
    bool decode_early_start = false;
    // test hook (b2a_test_last_attention_kernel): the kernel the last whole-sequence
    // attention launch took
    int last_attention_kernel = 0;
};

namespace {

thread_local std::string g_create_error;

int fail(b2a_context* ctx, int status, const char* fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    if (ctx) ctx->last_error = buf;
    else g_create_error = buf;
    return status;
}

int cuda_fail(b2a_context* ctx, cudaError_t e, const char* what) {
    if (e == cudaErrorMemoryAllocation) return fail(ctx, B2A_EOOM, "%s: %s", what, cudaGetErrorString(e));
    return fail(ctx, B2A_ECUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

// Makes ctx->device current for the duration of a call.
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

bool valid_dtype(int d) { return d == B2A_FLOAT32 || d == B2A_FLOAT16 || d == B2A_BFLOAT16; }
size_t dtype_size(int d) { return d == B2A_FLOAT32 ? 4 : 2; }

size_t workspace_total(const b2a_context* ctx) {
    return ctx->dec_ws_bytes + ctx->pf_ws_bytes + ctx->split_ws_bytes + ctx->blk_ws_bytes + ctx->rope_tab_bytes +
           ctx->lin_ws_bytes + ctx->pg_ws_bytes + ctx->kv4_ws_bytes + ctx->dec_counters.total + ctx->kv4_counters.total;
}

// Whether `more` bytes beside `others` stay within the context's limit.
int check_limit(b2a_context* ctx, size_t more, size_t others, const char* what) {
    if (ctx->ws_limit != 0 && more + others > ctx->ws_limit)
        return fail(ctx, B2A_EOOM, "%s workspace of %zu bytes exceeds the context limit of %zu bytes", what,
                    more + others, ctx->ws_limit);
    return B2A_OK;
}

int ensure_buffer(b2a_context* ctx, void** buf, size_t* have, size_t need, const char* what) {
    if (*have >= need) return B2A_OK;
    const int rc = check_limit(ctx, need, workspace_total(ctx) - *have, what);
    if (rc) return rc;
    if (*buf) {
        cudaFree(*buf);  // implicitly waits for work that may still use it
        *buf = nullptr;
        *have = 0;
    }
    cudaError_t e = cudaMalloc(buf, need);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(ctx, e, what);
    }
    *have = need;
    return B2A_OK;
}

// At least `ints` counters at *at, zeroed (on `stream`, or synchronously with `sync`) when they are new.
int ensure_counters(b2a_context* ctx, Counters& c, size_t ints, const char* what, cudaStream_t stream, bool sync,
                    int** at) {
    const size_t need = (ints * sizeof(int) + 255) / 256 * 256;
    if (c.n == 0 || c.bytes < need) {
        const size_t bytes = std::max(need, 2 * c.bytes);
        const int rc = check_limit(ctx, bytes, workspace_total(ctx), what);
        if (rc) return rc;
        if (c.n == Counters::kMost) return fail(ctx, B2A_EOOM, "%s: the counters grew too often", what);
        void* fresh = nullptr;
        cudaError_t e = cudaMalloc(&fresh, bytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return cuda_fail(ctx, e, what);
        }
        e = sync ? cudaMemset(fresh, 0, bytes) : cudaMemsetAsync(fresh, 0, bytes, stream);
        if (e != cudaSuccess) {
            cudaFree(fresh);
            return cuda_fail(ctx, e, what);
        }
        c.at[c.n++] = static_cast<int*>(fresh);
        c.bytes = bytes;
        c.total += bytes;
    }
    *at = c.at[c.n - 1];
    return B2A_OK;
}

void free_counters(Counters& c) {
    for (int i = 0; i < c.n; ++i) cudaFree(c.at[i]);
}

// Sizes a workspace for slot_bytes at *slots and counters at *counters.  The counters lie before the slots
// (in an allocation of their own a decode step of 24 layers took 0.662 ms instead of 0.655), in a region of
// one size whatever the call: no launch's slots, of a graph captured long ago either, lie where a later
// call of other sizes counts.  Calls that need more counters than that have them in `more` (null: such calls
// do not occur).
constexpr size_t kInlineCounters = 64 << 10;  // bytes
int ensure_counted_buffer(b2a_context* ctx, void** buf, size_t* have, Counters* more, size_t counter_ints,
                          size_t slot_bytes, const char* what, cudaStream_t stream, bool sync, int** counters,
                          void** slots) {
    const bool fresh = kInlineCounters + slot_bytes > *have;
    const int rc = ensure_buffer(ctx, buf, have, kInlineCounters + slot_bytes, what);
    if (rc) return rc;
    if (fresh) {
        const cudaError_t e =
            sync ? cudaMemset(*buf, 0, kInlineCounters) : cudaMemsetAsync(*buf, 0, kInlineCounters, stream);
        if (e != cudaSuccess) return cuda_fail(ctx, e, what);
    }
    *slots = static_cast<char*>(*buf) + kInlineCounters;
    *counters = static_cast<int*>(*buf);
    if (counter_ints * sizeof(int) <= kInlineCounters) return B2A_OK;
    if (!more) return fail(ctx, B2A_ENOTSUP, "%s: too many counters", what);
    return ensure_counters(ctx, *more, counter_ints, what, stream, sync, counters);
}

void inv_freq_table(double theta, int D, double* out) {
    // 1 / theta^(2i/D) in double (INF/decoderonly/DecoderOnlyRotaryEmbedding.java:57-59,
    // INF/gemma/Gemma3ReferenceMath.java:74)
    for (int i = 0; i < D / 2; ++i) out[i] = 1.0 / pow(theta, (2.0 * i) / D);
}

// The context's NeoX table covering positions [0, npos) for (theta, D); built on `stream` when the
// cached one does not cover them.  Calls on other streams must be ordered after this one (the
// same rule as every workspace of a context).
int neox_table(b2a_context* ctx, double theta, int D, int npos, cudaStream_t stream, const float2** out) {
    if (!(ctx->rope_tab != nullptr && ctx->rope_theta == theta && ctx->rope_D == D && ctx->rope_npos >= npos)) {
        const int n = (npos + 255) / 256 * 256;
        const int rc = ensure_buffer(ctx, &ctx->rope_tab, &ctx->rope_tab_bytes, (size_t)n * (D / 2) * sizeof(float2),
                                     "rope table");
        if (rc) return rc;
        double inv[kMaxHeadDim / 2];
        inv_freq_table(theta, D, inv);
        const cudaError_t e =
            launch_rope_table_f32(static_cast<float2*>(ctx->rope_tab), n, D / 2, 0, inv, stream);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "rope table launch");
        ctx->rope_theta = theta;
        ctx->rope_D = D;
        ctx->rope_npos = n;
    }
    *out = static_cast<const float2*>(ctx->rope_tab);
    return B2A_OK;
}

// Whether the tcgen05 kernel converts bf16 operands to fp16 itself instead of a pre-pass that
// writes fp16 copies.  In the kernel two otherwise idle warps convert each staged tile, so every
// work item converts the key/value tiles it reads: for sequences of at most 512 keys (at most two
// work items per head) that is cheaper than the extra launch and the copies' HBM round trip; for
// longer ones the repeated conversion costs more.  (Rotating q and k in the kernel the same way was
// slower at every length measured, so RoPE stays in the pre-pass.)
constexpr int kInKernelPrepMaxSeq = 512;

int check_heads(b2a_context* ctx, int Hq, int Hkv) {
    // DecoderOnlyAttentionLayout constructor (INF/decoderonly/DecoderOnlyAttentionLayout.java:12-22)
    if (Hq <= 0) return fail(ctx, B2A_EINVAL, "numQueryHeads must be positive");
    if (Hkv <= 0) return fail(ctx, B2A_EINVAL, "numKeyValueHeads must be positive");
    if (Hq % Hkv != 0)
        return fail(ctx, B2A_EINVAL, "numQueryHeads must be divisible by numKeyValueHeads for grouped-query attention");
    return B2A_OK;
}

int check_head_dim(b2a_context* ctx, int D) {
    // DecoderOnlyRotaryEmbedding constructor (INF/decoderonly/DecoderOnlyRotaryEmbedding.java:14-16)
    if (D <= 0 || D % 2 != 0) return fail(ctx, B2A_EINVAL, "headDim must be positive and even");
    if (D > kMaxHeadDim) return fail(ctx, B2A_ENOTSUP, "headDim %d exceeds the supported maximum %d", D, kMaxHeadDim);
    return B2A_OK;
}

// Whole-sequence attention: the tcgen05 kernel where its shape rules hold,
// else the warp-MMA kernel (16-bit, head_dim 32..128), else the tiled fp32 kernel
// (fp32, head_dim 64 / 128), else the generic one.
cudaError_t launch_attention(b2a_context* ctx, const AttnParams& p, cudaStream_t s) {
    if (attn_tcgen05_supported(p)) {
        const bool stall = ctx->inject_wait_timeout;
        ctx->inject_wait_timeout = false;
        ctx->last_attention_kernel = B2A_TEST_KERNEL_TCGEN05;
        return launch_attn_tcgen05(p, ctx->status, s, stall);
    }
    if (attn_tc_supported(p)) {
        ctx->last_attention_kernel = B2A_TEST_KERNEL_WARP_MMA;
        return launch_attn_tc(p, s);
    }
    if (attn_f32_supported(p)) {
        ctx->last_attention_kernel = B2A_TEST_KERNEL_F32_TILED;
        return launch_attn_f32(p, s);
    }
    ctx->last_attention_kernel = B2A_TEST_KERNEL_GENERIC;
    // generic kernel: launches too small to fill the GPU split each query block's keys
    // over several CTAs; without room for the split workspace they run unsplit
    size_t part_bytes = 0, counter_ints = 0;
    const int nsplit = attn_simt_split_plan(p, ctx->sm_count, &part_bytes, &counter_ints);
    if (nsplit > 1) {
        int* counters = nullptr;
        void* slots = nullptr;
        if (ensure_counted_buffer(ctx, &ctx->split_ws, &ctx->split_ws_bytes, nullptr, counter_ints,
                                  part_bytes, "attention split workspace", s, false, &counters, &slots) == B2A_OK) {
            const SimtSplit sp{static_cast<float*>(slots), counters, nsplit, kSimtSplitKeys};
            return launch_attn_simt(p, s, &sp);
        }
        ctx->last_error.clear();  // the refused workspace is not an error of this call
    }
    return launch_attn_simt(p, s);
}

int run_decode(b2a_context* ctx, DecodeParams& p, cudaStream_t stream, bool allow_tc) {
    // 16-byte row loads need 16-byte aligned cache bases and row strides
    const bool aligned = ((uintptr_t)p.k_cache % 16 == 0) && ((uintptr_t)p.v_cache % 16 == 0) &&
                         p.stride_b % 8 == 0 && p.stride_h % 8 == 0 && p.stride_pos % 8 == 0;
    p.status = ctx->status;
    if (allow_tc && aligned && decode_tc_supported(p.D, p.cache_dtype)) {
        p.n_hg = (p.G + 7) / 8;
        int target = 0, cap = 0;
        size_t partial_bytes = 0;
        decode_tc_workspace(ctx->device, p.B, p.Hkv, p.n_hg, p.D, p.cache_dtype, &target, &cap, &partial_bytes);
        const int bmax = std::min(p.B, kDecodeMaxBatchPerLaunch);
        const size_t counter_ints = (size_t)bmax * p.Hkv * p.n_hg;
        void* slots = nullptr;
        int rc = ensure_counted_buffer(ctx, &ctx->dec_ws, &ctx->dec_ws_bytes, &ctx->dec_counters, counter_ints,
                                       partial_bytes, "decode workspace", stream, false, &p.counters, &slots);
        if (rc != B2A_OK) return rc;
        p.partials = static_cast<float*>(slots);
        p.target_items = target;
        p.item_capacity = cap;
        p.early_start = ctx->decode_early_start ? 1 : 0;
        const int B = p.B;
        // one launch covers at most kDecodeMaxBatchPerLaunch sequences and a key
        // stream (visible keys plus per-unit overhead keys) below 2^31 (the kernel's int32 prefix)
        const int per_launch = (int)std::min<int64_t>(kDecodeMaxBatchPerLaunch,
                                                      INT32_MAX / ((int64_t)p.max_seq + 1 + kDecodeGapKeysMax));
        for (int b0 = 0; b0 < B; b0 += per_launch) {
            DecodeParams s = p;
            s.B = std::min(per_launch, B - b0);
            const size_t qe = dtype_size(p.q_dtype), oe = dtype_size(p.out_dtype), ce = dtype_size(p.cache_dtype);
            s.q = static_cast<const char*>(p.q) + (size_t)b0 * q_stride_of(p) * qe;
            if (p.k_new) s.k_new = static_cast<const char*>(p.k_new) + (size_t)b0 * kvn_stride_of(p) * qe;
            if (p.v_new) s.v_new = static_cast<const char*>(p.v_new) + (size_t)b0 * kvn_stride_of(p) * qe;
            s.k_cache = static_cast<char*>(p.k_cache) + (size_t)b0 * p.stride_b * ce;
            s.v_cache = static_cast<char*>(p.v_cache) + (size_t)b0 * p.stride_b * ce;
            if (p.ctx_lens) s.ctx_lens = p.ctx_lens + b0;
            s.out = static_cast<char*>(p.out) + (size_t)b0 * p.Hq * p.D * oe;
            cudaError_t e = launch_decode_tc(s, ctx->device, stream);
            if (e != cudaSuccess) return cuda_fail(ctx, e, "decode kernel launch");
        }
        return B2A_OK;
    }
    cudaError_t e = launch_decode_simt(p, stream);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "decode kernel launch");
    return B2A_OK;
}

}  // namespace

namespace b2a {
// Message for b2a_last_error(NULL, ...) from entry points that take no context.
void set_thread_error(const char* msg) { g_create_error = msg ? msg : ""; }
}  // namespace b2a

extern "C" {

B2A_API const char* b2a_status_string(int status) {
    switch (status) {
        case B2A_OK: return "B2A_OK";
        case B2A_EINVAL: return "B2A_EINVAL";
        case B2A_ECUDA: return "B2A_ECUDA";
        case B2A_ENCCL: return "B2A_ENCCL";
        case B2A_ETIMEOUT: return "B2A_ETIMEOUT";
        case B2A_EOOM: return "B2A_EOOM";
        case B2A_ENOTSUP: return "B2A_ENOTSUP";
        case B2A_EDEVICE: return "B2A_EDEVICE";
        default: return "B2A_UNKNOWN";
    }
}

B2A_API int b2a_abi_version(void) { return B2A_ABI_VERSION; }

B2A_API const char* b2a_build_info(void) {
    return "libb200attn sm_100a; CUDA " __DATE__ " " __TIME__;
}

B2A_API int b2a_create(int device, b2a_context** out) {
    if (!out) return fail(nullptr, B2A_EINVAL, "out must not be null");
    *out = nullptr;
    int n = 0;
    cudaError_t e = cudaGetDeviceCount(&n);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(nullptr, B2A_ECUDA, "no CUDA device available: %s", cudaGetErrorString(e));
    }
    if (device < 0 || device >= n) return fail(nullptr, B2A_EINVAL, "device %d out of range [0, %d)", device, n);
    cudaDeviceProp prop;
    e = cudaGetDeviceProperties(&prop, device);
    if (e != cudaSuccess) return fail(nullptr, B2A_ECUDA, "cudaGetDeviceProperties: %s", cudaGetErrorString(e));
    if (prop.major != 10 || prop.minor != 0)
        return fail(nullptr, B2A_ENOTSUP, "device %d is sm_%d%d; this library is built for sm_100a (B200) only",
                    device, prop.major, prop.minor);
    DeviceGuard guard(device);
    if (!guard.ok) return fail(nullptr, B2A_ECUDA, "cudaSetDevice(%d) failed", device);
    b2a_context* ctx = new (std::nothrow) b2a_context();
    if (!ctx) return fail(nullptr, B2A_EOOM, "host allocation failed");
    ctx->device = device;
    ctx->sm_count = prop.multiProcessorCount;
    e = cudaMalloc(&ctx->status, kStatusBufferInts * sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(ctx->status, 0, kStatusBufferInts * sizeof(int));
    if (e == cudaSuccess) e = cudaMallocHost(&ctx->status_host, kStatusWords * sizeof(int));
    if (e != cudaSuccess) {
        if (ctx->status) cudaFree(ctx->status);
        delete ctx;
        cudaGetLastError();
        return fail(nullptr, e == cudaErrorMemoryAllocation ? B2A_EOOM : B2A_ECUDA, "status buffer: %s",
                    cudaGetErrorString(e));
    }
    *out = ctx;
    return B2A_OK;
}

B2A_API int b2a_destroy(b2a_context* ctx) {
    if (!ctx) return B2A_OK;
    {
        DeviceGuard guard(ctx->device);
        if (ctx->status) cudaFree(ctx->status);
        if (ctx->status_host) cudaFreeHost(ctx->status_host);
        if (ctx->dec_ws) cudaFree(ctx->dec_ws);
        if (ctx->pf_ws) cudaFree(ctx->pf_ws);
        if (ctx->split_ws) cudaFree(ctx->split_ws);
        if (ctx->blk_ws) cudaFree(ctx->blk_ws);
        if (ctx->rope_tab) cudaFree(ctx->rope_tab);
        if (ctx->lin_ws) cudaFree(ctx->lin_ws);
        if (ctx->pg_ws) cudaFree(ctx->pg_ws);
        if (ctx->kv4_ws) cudaFree(ctx->kv4_ws);
        free_counters(ctx->dec_counters);
        free_counters(ctx->kv4_counters);
    }
    delete ctx;
    return B2A_OK;
}

B2A_API int b2a_last_error(const b2a_context* ctx, char* buf, size_t n) {
    const std::string& s = ctx ? ctx->last_error : g_create_error;
    if (buf && n > 0) {
        size_t k = std::min(n - 1, s.size());
        memcpy(buf, s.data(), k);
        buf[k] = '\0';
    }
    return (int)s.size();
}

B2A_API int b2a_set_workspace_limit(b2a_context* ctx, size_t bytes) {
    if (!ctx) return B2A_EINVAL;
    ctx->ws_limit = bytes;
    return B2A_OK;
}

B2A_API int b2a_set_decode_early_start(b2a_context* ctx, int enable) {
    if (!ctx) return B2A_EINVAL;
    ctx->decode_early_start = enable != 0;
    return B2A_OK;
}

B2A_API int b2a_workspace_bytes(const b2a_context* ctx, size_t* bytes) {
    if (!ctx || !bytes) return B2A_EINVAL;
    *bytes = workspace_total(ctx);
    return B2A_OK;
}

B2A_API int b2a_reserve_decode(b2a_context* ctx, int max_batch, int num_q_heads, int num_kv_heads, int head_dim) {
    if (!ctx) return B2A_EINVAL;
    int rc = check_heads(ctx, num_q_heads, num_kv_heads);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, head_dim))) return rc;
    if (max_batch <= 0) return fail(ctx, B2A_EINVAL, "max_batch must be positive");
    if (!decode_tc_supported(head_dim, B2A_FLOAT16)) return B2A_OK;  // generic kernel needs no workspace
    DeviceGuard guard(ctx->device);
    const int n_hg = (num_q_heads / num_kv_heads + 7) / 8;
    int target = 0, cap = 0;
    size_t partial_bytes = 0;
    decode_tc_workspace(ctx->device, max_batch, num_kv_heads, n_hg, head_dim, B2A_FLOAT16, &target, &cap,
                        &partial_bytes);
    const size_t counter_ints = (size_t)std::min(max_batch, kDecodeMaxBatchPerLaunch) * num_kv_heads * n_hg;
    int* counters = nullptr;
    void* slots = nullptr;
    return ensure_counted_buffer(ctx, &ctx->dec_ws, &ctx->dec_ws_bytes, &ctx->dec_counters, counter_ints,
                                 partial_bytes, "decode workspace", nullptr, true, &counters, &slots);
}

B2A_API int b2a_test_inject_wait_timeout(b2a_context* ctx) {
    if (!ctx) return B2A_EINVAL;
    ctx->inject_wait_timeout = true;
    return B2A_OK;
}

B2A_API int b2a_test_last_attention_kernel(const b2a_context* ctx) {
    return ctx ? ctx->last_attention_kernel : 0;
}

B2A_API int b2a_check_device_status(b2a_context* ctx, void* stream) {
    if (!ctx) return B2A_EINVAL;
    DeviceGuard guard(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // one stream-ordered copy of the flags into pinned memory, one synchronisation
    cudaError_t e = cudaMemcpyAsync(ctx->status_host, ctx->status, kStatusWords * sizeof(int),
                                    cudaMemcpyDeviceToHost, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "status read");
    e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "stream synchronize");
    const int flags = ctx->status_host[0];
    if (flags == 0) return B2A_OK;
    e = cudaMemsetAsync(ctx->status, 0, kStatusWords * sizeof(int), s);  // ordered before later launches
    if (e != cudaSuccess) return cuda_fail(ctx, e, "status clear");
    std::string msg;
    if (flags & 8) msg += "a bounded device wait ran out (attention pipeline aborted; its outputs are undefined). ";
    if (flags & 1) msg += "a ctx_lens entry was outside [0, max_seq); its outputs are NaN. ";
    if (flags & 2) msg += "decode work items exceeded the workspace capacity. ";
    if (flags & 4) msg += "a bf16 input exceeded the fp16 operand range (|x| > 65504). ";
    if (flags & 16) msg += "a page_table entry that was needed named no page of the pool. ";
    if (flags & 32) msg += "a k or v value was not finite or beyond the 4-bit cache's range; its group holds NaN. ";
    if (flags & 64) msg += "a parents entry was outside [-1, n_seq); its row is unchanged. ";
    // a timed-out pipeline is reported as such; the other flags are failed device-side argument checks
    return fail(ctx, (flags & 8) ? B2A_ETIMEOUT : B2A_EDEVICE, "%s", msg.c_str());
}

// ----------------------------------------------------------------- encoder
B2A_API int b2a_mha(b2a_context* ctx, int in_dtype, int out_dtype, const void* q, const void* k, const void* v,
                    const float* mask, const int32_t* key_lengths, void* y, int B, int H, int S, int D, float scale,
                    int layout, void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!valid_dtype(in_dtype) || !valid_dtype(out_dtype))
        return fail(ctx, B2A_EINVAL, "unsupported element type (in %d, out %d)", in_dtype, out_dtype);
    if (!q || !k || !v || !y) return fail(ctx, B2A_EINVAL, "q, k, v and y tensors must not be null");
    if (mask && key_lengths) return fail(ctx, B2A_EINVAL, "pass either an additive mask or key lengths, not both");
    // DirectMlAttentionKernel constructor (WB/runtime/kernels/DirectMlAttentionKernel.java:109-111)
    if (B <= 0 || H <= 0 || S <= 0 || D <= 0) return fail(ctx, B2A_EINVAL, "batch, heads, seq, headDim must be > 0");
    if (D > kMaxHeadDim || D % 2) return fail(ctx, B2A_ENOTSUP, "headDim %d not supported (even, <= %d)", D, kMaxHeadDim);
    if (layout != B2A_HEAD_MAJOR && layout != B2A_SEQ_MAJOR) return fail(ctx, B2A_EINVAL, "unknown layout %d", layout);
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    DeviceGuard guard(ctx->device);
    AttnParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.in_dtype = in_dtype;
    p.o = y;
    p.out_dtype = out_dtype;
    p.B = B;
    p.S = S;
    p.Hq = H;
    p.Hkv = H;
    p.D = D;
    if (layout == B2A_HEAD_MAJOR) {
        p.q_sb = (int64_t)H * S * D;
        p.q_ss = D;
        p.q_sh = (int64_t)S * D;
    } else {
        p.q_sb = (int64_t)S * H * D;
        p.q_ss = (int64_t)H * D;
        p.q_sh = D;
    }
    p.k_sb = p.q_sb;
    p.k_ss = p.q_ss;
    p.k_sh = p.q_sh;
    p.causal = 0;
    p.window = 0;
    p.mask = mask;
    p.key_len = key_lengths;
    p.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (in_dtype == B2A_BFLOAT16) {
        // short sequences: the tensor-core kernel converts the staged bf16 tiles to fp16 itself
        // (no pre-pass; measured on B200, bf16 B=64 H=12 S=128 D=32: 30.2 vs 36.3 us; S=512 D=64:
        // 56.8 vs 69.0 us; at S=1024 D=128 the pre-pass is faster, 142 vs 151 us)
        AttnParams t = p;
        t.xform = 7;
        if (S <= kInKernelPrepMaxSeq && attn_tcgen05_supported(t)) {
            e = launch_attention(ctx, t, s);
            if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel launch");
            return B2A_OK;
        }
    }
    if (in_dtype == B2A_BFLOAT16) {
        // same operand rule as the prefill: bf16 inputs are multiplied as fp16
        const size_t n = (size_t)B * H * S * D;
        const size_t one = (n * 2 + 255) / 256 * 256;
        int rc = ensure_buffer(ctx, &ctx->pf_ws, &ctx->pf_ws_bytes, 3 * one, "encoder");
        if (rc) return rc;
        char* base = static_cast<char*>(ctx->pf_ws);
        const void* ptrs[] = {q, k, v};
        if (prep_vectorizable(D, (int64_t)n, ptrs, 3)) {  // one launch for the three conversions
            const PrepJob jobs[3] = {PrepJob{q, base, nullptr, H, 0}, PrepJob{k, base + one, nullptr, H, 0},
                                     PrepJob{v, base + 2 * one, nullptr, H, 0}};
            e = launch_prep(jobs, 3, B, S, D, in_dtype, B2A_FLOAT16, 0, B2A_ROPE_NONE, nullptr, nullptr, ctx->status,
                            s);
        } else {
            e = launch_convert(q, in_dtype, base, B2A_FLOAT16, (int64_t)n, ctx->status, s);
            if (e == cudaSuccess) e = launch_convert(k, in_dtype, base + one, B2A_FLOAT16, (int64_t)n, ctx->status, s);
            if (e == cudaSuccess)
                e = launch_convert(v, in_dtype, base + 2 * one, B2A_FLOAT16, (int64_t)n, ctx->status, s);
        }
        if (e != cudaSuccess) return cuda_fail(ctx, e, "conversion kernel launch");
        p.q = base;
        p.k = base + one;
        p.v = base + 2 * one;
        p.in_dtype = B2A_FLOAT16;
    }
    e = launch_attention(ctx, p, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel launch");
    return B2A_OK;
}

// ----------------------------------------------------------------- prefill
B2A_API int b2a_prefill_causal(b2a_context* ctx, int in_dtype, int out_dtype, const void* q, const void* k,
                               const void* v, void* o, int B, int S, int Hq, int Hkv, int D, float scale, int rope_mode,
                               double rope_theta, int pos0, int window, void* k_rot_out, void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!valid_dtype(in_dtype) || !valid_dtype(out_dtype))
        return fail(ctx, B2A_EINVAL, "unsupported element type (in %d, out %d)", in_dtype, out_dtype);
    if (!q || !k || !v || !o) return fail(ctx, B2A_EINVAL, "q, k, v and o must not be null");
    int rc = check_heads(ctx, Hq, Hkv);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, D))) return rc;
    if (B <= 0 || S <= 0) return fail(ctx, B2A_EINVAL, "batch and sequence length must be > 0");
    if (window < 0) return fail(ctx, B2A_EINVAL, "window must not be negative");
    if (pos0 < 0) return fail(ctx, B2A_EINVAL, "pos0 must not be negative");
    if (rope_mode != B2A_ROPE_NONE && rope_mode != B2A_ROPE_NEOX && rope_mode != B2A_ROPE_GEMMA)
        return fail(ctx, B2A_EINVAL, "unknown rope mode %d", rope_mode);
    if (rope_mode != B2A_ROPE_NONE && !(rope_theta > 0.0)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    DeviceGuard guard(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    AttnParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.in_dtype = in_dtype;
    p.o = o;
    p.out_dtype = out_dtype;
    p.B = B;
    p.S = S;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.D = D;
    p.q_sb = (int64_t)S * Hq * D;
    p.q_ss = (int64_t)Hq * D;
    p.q_sh = D;
    p.k_sb = (int64_t)S * Hkv * D;
    p.k_ss = (int64_t)Hkv * D;
    p.k_sh = D;
    p.causal = 1;
    p.window = window;
    p.scale = scale;

    const size_t nq = (size_t)B * S * Hq * D, nk = (size_t)B * S * Hkv * D;
    auto r256 = [](size_t x) { return (x + 255) / 256 * 256; };

    // fp32 inputs (the fp32 kernels) with the NeoX rotation and no rotated-key output: the
    // kernel rotates q and k itself from the context's cached table -- one launch, no pre-pass
    if (in_dtype == B2A_FLOAT32 && rope_mode == B2A_ROPE_NEOX && k_rot_out == nullptr) {
        const float2* tab = nullptr;
        if ((int64_t)pos0 + S > INT32_MAX) return fail(ctx, B2A_EINVAL, "pos0 + S exceeds the position range");
        if ((rc = neox_table(ctx, rope_theta, D, pos0 + S, s, &tab))) return rc;
        p.rope_table = tab;
        p.rope_pos0 = pos0;
        const cudaError_t e = launch_attention(ctx, p, s);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel launch");
        return B2A_OK;
    }

    // bf16 inputs are multiplied as fp16 tensor-core operands: the rotated q/k,
    // P and V then carry 11 significant bits instead of 8, which keeps short
    // causal rows within the 2e-3 tolerance (bf16 -> fp16 is exact inside the
    // fp16 range; values beyond it raise device status bit 2).
    const int cdt = in_dtype == B2A_BFLOAT16 ? B2A_FLOAT16 : in_dtype;
    const size_t ce = dtype_size(cdt);
    const bool rope = rope_mode != B2A_ROPE_NONE;
    const bool conv = cdt != in_dtype;
    // the vectorised pre-pass reads NeoX (cos, sin) rows from the context's cached float table;
    // Gemma's double table (and the row-wise fallback's) is built per call into the workspace
    const bool cached_table = rope_mode == B2A_ROPE_NEOX;
    const size_t table_bytes = rope ? r256((size_t)S * (D / 2) * 16) : 0;
    const size_t q_bytes = (rope || conv) ? r256(nq * ce) : 0;
    const bool k_in_out = rope && !conv && k_rot_out != nullptr;  // rotated keys land in k_rot_out directly
    const size_t k_bytes = ((rope || conv) && !k_in_out) ? r256(nk * ce) : 0;
    const size_t v_bytes = conv ? r256(nk * ce) : 0;
    if (table_bytes + q_bytes + k_bytes + v_bytes > 0) {
        rc = ensure_buffer(ctx, &ctx->pf_ws, &ctx->pf_ws_bytes, table_bytes + q_bytes + k_bytes + v_bytes, "prefill");
        if (rc) return rc;
    }
    char* base = static_cast<char*>(ctx->pf_ws);
    double2* table = reinterpret_cast<double2*>(base);
    void* q_c = base + table_bytes;
    void* k_c = k_in_out ? k_rot_out : base + table_bytes + q_bytes;
    void* v_c = base + table_bytes + q_bytes + k_bytes;
    cudaError_t e = cudaSuccess;
    const void* prep_ptrs[] = {q, k, v, q_c, k_c, v_c, k_rot_out};
    const bool vec_prep = (rope || conv) && prep_vectorizable(D, (int64_t)std::max(nq, nk), prep_ptrs, 7);
    if (vec_prep) {
        // one launch: q and k rotated / converted, v converted (NeoX: from the cached table,
        // else after a table build)
        double inv[kMaxHeadDim / 2] = {};
        if (rope) inv_freq_table(rope_theta, D, inv);
        double2* prep_table = table;
        if (rope && cached_table) {
            const float2* tab = nullptr;
            if ((int64_t)pos0 + S > INT32_MAX) return fail(ctx, B2A_EINVAL, "pos0 + S exceeds the position range");
            if ((rc = neox_table(ctx, rope_theta, D, pos0 + S, s, &tab))) return rc;
            prep_table = reinterpret_cast<double2*>(const_cast<float2*>(tab + (size_t)pos0 * (D / 2)));
        }
        PrepJob jobs[3];
        int nj = 0;
        jobs[nj++] = PrepJob{q, q_c, nullptr, Hq, rope ? 1 : 0};
        jobs[nj++] = PrepJob{k, k_c, (rope && k_rot_out && !k_in_out) ? k_rot_out : nullptr, Hkv, rope ? 1 : 0};
        if (conv) jobs[nj++] = PrepJob{v, v_c, nullptr, Hkv, 0};
        e = launch_prep(jobs, nj, B, S, D, in_dtype, cdt, pos0, rope_mode, inv, prep_table, ctx->status, s,
                        rope && cached_table);
        if (e == cudaSuccess && !rope && k_rot_out)
            e = cudaMemcpyAsync(k_rot_out, k, nk * dtype_size(in_dtype), cudaMemcpyDeviceToDevice, s);
    } else if (rope) {
        double inv[kMaxHeadDim / 2];
        inv_freq_table(rope_theta, D, inv);
        e = launch_rope_rows_with_table(q, in_dtype, q_c, cdt, B, S, Hq, D, p.q_sb, p.q_ss, p.q_sh, p.q_sb, p.q_ss,
                                        p.q_sh, pos0, rope_mode, inv, table, true, ctx->status, s);
        if (e == cudaSuccess)
            e = launch_rope_rows_with_table(k, in_dtype, k_c, cdt, B, S, Hkv, D, p.k_sb, p.k_ss, p.k_sh, p.k_sb,
                                            p.k_ss, p.k_sh, pos0, rope_mode, inv, table, false, ctx->status, s);
        if (e == cudaSuccess && k_rot_out && !k_in_out)  // caller wants rotated keys in its own dtype
            e = launch_rope_rows_with_table(k, in_dtype, k_rot_out, in_dtype, B, S, Hkv, D, p.k_sb, p.k_ss, p.k_sh,
                                            p.k_sb, p.k_ss, p.k_sh, pos0, rope_mode, inv, table, false, nullptr, s);
    } else {
        if (conv) {
            e = launch_convert(q, in_dtype, q_c, cdt, (int64_t)nq, ctx->status, s);
            if (e == cudaSuccess) e = launch_convert(k, in_dtype, k_c, cdt, (int64_t)nk, ctx->status, s);
        }
        if (e == cudaSuccess && k_rot_out)
            e = cudaMemcpyAsync(k_rot_out, k, nk * dtype_size(in_dtype), cudaMemcpyDeviceToDevice, s);
    }
    if (e == cudaSuccess && conv && !vec_prep) e = launch_convert(v, in_dtype, v_c, cdt, (int64_t)nk, ctx->status, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "rope / conversion kernel launch");
    if (rope || conv) {
        p.q = q_c;
        p.k = k_c;
    }
    if (conv) p.v = v_c;
    p.in_dtype = cdt;
    e = launch_attention(ctx, p, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel launch");
    return B2A_OK;
}

// ----------------------------------------------------------------- Gemma prefill
B2A_API int b2a_prefill_gemma(b2a_context* ctx, int in_dtype, int out_dtype, const void* q, const void* k, const void* v,
                              void* o, int B, int S, int Hq, int Hkv, int D, float scale, int rope_mode,
                              double rope_theta, int pos0, int window, const float* q_norm_w, const float* k_norm_w,
                              float norm_eps, void* k_rot_out, void* stream) {
    // Gemma3WarpLayer.forwardPrefillBatched steps 3-4 (INF/gemma/Gemma3WarpLayer.java:395-411): per position QK-norm,
    // RoPE at p, KV append, then one attention over [firstValid(p), p] per position; here the
    // norm + rotation of all positions is one pre-pass and the attention one launch.
    if (!ctx) return B2A_EINVAL;
    if (!valid_dtype(in_dtype) || !valid_dtype(out_dtype))
        return fail(ctx, B2A_EINVAL, "unsupported element type (in %d, out %d)", in_dtype, out_dtype);
    if (!q || !k || !v || !o) return fail(ctx, B2A_EINVAL, "q, k, v and o must not be null");
    int rc = check_heads(ctx, Hq, Hkv);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, D))) return rc;
    if (B <= 0 || S <= 0) return fail(ctx, B2A_EINVAL, "batch and sequence length must be > 0");
    if (window < 0) return fail(ctx, B2A_EINVAL, "window must not be negative");
    if (pos0 < 0) return fail(ctx, B2A_EINVAL, "pos0 must not be negative");
    if (rope_mode != B2A_ROPE_NONE && rope_mode != B2A_ROPE_NEOX && rope_mode != B2A_ROPE_GEMMA)
        return fail(ctx, B2A_EINVAL, "unknown rope mode %d", rope_mode);
    if (rope_mode != B2A_ROPE_NONE && !(rope_theta > 0.0)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    if (!(norm_eps >= 0.f)) return fail(ctx, B2A_EINVAL, "norm eps must not be negative");
    DeviceGuard guard(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    // same operand rule as b2a_prefill_causal: bf16 inputs are multiplied as fp16
    const int cdt = in_dtype == B2A_BFLOAT16 ? B2A_FLOAT16 : in_dtype;
    const size_t ce = dtype_size(cdt);
    const size_t nq = (size_t)B * S * Hq * D, nk = (size_t)B * S * Hkv * D;
    auto r256 = [](size_t x) { return (x + 255) / 256 * 256; };
    const bool rope = rope_mode != B2A_ROPE_NONE;
    const bool conv = cdt != in_dtype;
    const size_t table_bytes = rope ? r256((size_t)S * (D / 2) * 16) : 0;
    const size_t q_bytes = r256(nq * ce), k_bytes = r256(nk * ce), v_bytes = conv ? r256(nk * ce) : 0;
    rc = ensure_buffer(ctx, &ctx->pf_ws, &ctx->pf_ws_bytes, table_bytes + q_bytes + k_bytes + v_bytes, "prefill");
    if (rc) return rc;
    char* base = static_cast<char*>(ctx->pf_ws);
    double2* table = reinterpret_cast<double2*>(base);
    void* q_c = base + table_bytes;
    void* k_c = base + table_bytes + q_bytes;
    void* v_c = conv ? base + table_bytes + q_bytes + k_bytes : const_cast<void*>(v);
    double inv[kMaxHeadDim / 2] = {};
    if (rope) inv_freq_table(rope_theta, D, inv);
    cudaError_t e = launch_norm_rope_rows(q, q_c, nullptr, in_dtype, cdt, B, S, Hq, D, q_norm_w, norm_eps, rope_mode,
                                          pos0, inv, table, true, ctx->status, s);
    if (e == cudaSuccess)
        e = launch_norm_rope_rows(k, k_c, k_rot_out, in_dtype, cdt, B, S, Hkv, D, k_norm_w, norm_eps, rope_mode, pos0,
                                  inv, table, false, ctx->status, s);
    if (e == cudaSuccess && conv) e = launch_convert(v, in_dtype, v_c, cdt, (int64_t)nk, ctx->status, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "norm / rope / conversion kernel launch");

    AttnParams p{};
    p.q = q_c;
    p.k = k_c;
    p.v = v_c;
    p.in_dtype = cdt;
    p.o = o;
    p.out_dtype = out_dtype;
    p.B = B;
    p.S = S;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.D = D;
    p.q_sb = (int64_t)S * Hq * D;
    p.q_ss = (int64_t)Hq * D;
    p.q_sh = D;
    p.k_sb = (int64_t)S * Hkv * D;
    p.k_ss = (int64_t)Hkv * D;
    p.k_sh = D;
    p.causal = 1;
    p.window = window;
    p.scale = scale;
    e = launch_attention(ctx, p, s);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel launch");
    return B2A_OK;
}

// ----------------------------------------------------------------- decode
B2A_API int b2a_decode(b2a_context* ctx, int q_dtype, int cache_dtype, int out_dtype, const void* q_new,
                       const void* k_new, const void* v_new, void* k_cache, void* v_cache, int kv_layout,
                       const int32_t* ctx_lens, int B, int Hq, int Hkv, int D, int max_seq, float scale,
                       int rope_mode, double rope_theta, int window, const float* q_norm_w, const float* k_norm_w,
                       float norm_eps, void* o, void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!valid_dtype(q_dtype) || !valid_dtype(cache_dtype) || !valid_dtype(out_dtype))
        return fail(ctx, B2A_EINVAL, "unsupported element type (q %d, cache %d, out %d)", q_dtype, cache_dtype,
                    out_dtype);
    if (!q_new || !k_new || !v_new || !k_cache || !v_cache || !ctx_lens || !o)
        return fail(ctx, B2A_EINVAL, "q_new, k_new, v_new, caches, ctx_lens and o must not be null");
    int rc = check_heads(ctx, Hq, Hkv);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, D))) return rc;
    if (B <= 0) return fail(ctx, B2A_EINVAL, "batch must be > 0");
    if (max_seq <= 0) return fail(ctx, B2A_EINVAL, "max_seq must be > 0");
    if (window < 0) return fail(ctx, B2A_EINVAL, "window must not be negative");
    if (kv_layout != B2A_KV_HEAD_MAJOR && kv_layout != B2A_KV_POS_MAJOR)
        return fail(ctx, B2A_EINVAL, "unknown kv layout %d", kv_layout);
    if (rope_mode != B2A_ROPE_NONE && rope_mode != B2A_ROPE_NEOX && rope_mode != B2A_ROPE_GEMMA)
        return fail(ctx, B2A_EINVAL, "unknown rope mode %d", rope_mode);
    if (rope_mode != B2A_ROPE_NONE && !(rope_theta > 0.0)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
        return fail(ctx, B2A_EINVAL, "q_norm_w and k_norm_w must be given together");
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    if (q_norm_w && !(norm_eps >= 0.f)) return fail(ctx, B2A_EINVAL, "norm_eps must not be negative");
    DeviceGuard guard(ctx->device);
    DecodeParams p{};
    p.q = q_new;
    p.k_new = k_new;
    p.v_new = v_new;
    p.q_dtype = q_dtype;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.cache_dtype = cache_dtype;
    p.stride_b = (int64_t)Hkv * max_seq * D;
    if (kv_layout == B2A_KV_HEAD_MAJOR) {
        p.stride_h = (int64_t)max_seq * D;
        p.stride_pos = D;
    } else {
        p.stride_h = D;
        p.stride_pos = (int64_t)Hkv * D;
    }
    p.ctx_lens = ctx_lens;
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.D = D;
    p.max_seq = max_seq;
    p.window = window;
    p.first_explicit = -1;
    p.append = 1;
    p.rope_mode = rope_mode;
    p.scale = scale;
    p.q_norm_w = q_norm_w;
    p.k_norm_w = k_norm_w;
    p.norm_eps = norm_eps;
    p.out = o;
    p.out_dtype = out_dtype;
    if (rope_mode != B2A_ROPE_NONE) inv_freq_table(rope_theta, D, p.inv_freq);
    return run_decode(ctx, p, static_cast<cudaStream_t>(stream), true);
}

// ------------------------------------------------- reference GPU contracts
B2A_API int b2a_qwen_rope_and_append(b2a_context* ctx, float* q, const float* k, const float* v, float* k_cache,
                                     float* v_cache, int num_heads, int kv_heads, int head_dim, int pos,
                                     int max_seq_len, float rope_theta, void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!q || !k || !v || !k_cache || !v_cache) return fail(ctx, B2A_EINVAL, "buffers must not be null");
    if (num_heads <= 0 || kv_heads <= 0) return fail(ctx, B2A_EINVAL, "numHeads and kvHeads must be positive");
    int rc = check_head_dim(ctx, head_dim);
    if (rc) return rc;
    if (pos < 0 || pos >= max_seq_len) return fail(ctx, B2A_EINVAL, "pos %d outside [0, maxSeqLen=%d)", pos, max_seq_len);
    if (!(rope_theta > 0.f)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    DeviceGuard guard(ctx->device);
    double inv[kMaxHeadDim / 2];
    inv_freq_table((double)rope_theta, head_dim, inv);
    cudaError_t e = launch_qwen_rope_append(q, k, v, k_cache, v_cache, num_heads, kv_heads, head_dim, pos, max_seq_len,
                                            inv, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "rope_and_append launch");
    return B2A_OK;
}

B2A_API int b2a_qwen_gqa_attention_decode(b2a_context* ctx, const float* q, const float* k_cache, const float* v_cache,
                                          float* attn_out, int num_heads, int kv_heads, int head_dim,
                                          int q_heads_per_kv_head, int seq_len, int max_seq_len, float scale,
                                          void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!q || !k_cache || !v_cache || !attn_out) return fail(ctx, B2A_EINVAL, "buffers must not be null");
    int rc = check_heads(ctx, num_heads, kv_heads);
    if (rc) return rc;
    if (q_heads_per_kv_head != num_heads / kv_heads)
        return fail(ctx, B2A_EINVAL, "qHeadsPerKvHead %d != numHeads / kvHeads = %d", q_heads_per_kv_head,
                    num_heads / kv_heads);
    if ((rc = check_head_dim(ctx, head_dim))) return rc;
    if (seq_len <= 0 || seq_len > max_seq_len)
        return fail(ctx, B2A_EINVAL, "seqLen %d outside [1, maxSeqLen=%d]", seq_len, max_seq_len);
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    DeviceGuard guard(ctx->device);
    DecodeParams p{};
    p.q = q;
    p.q_dtype = B2A_FLOAT32;
    p.k_cache = const_cast<float*>(k_cache);
    p.v_cache = const_cast<float*>(v_cache);
    p.cache_dtype = B2A_FLOAT32;
    p.stride_b = 0;
    p.stride_h = (int64_t)max_seq_len * head_dim;
    p.stride_pos = head_dim;
    p.ctx_lens = nullptr;
    p.pos_scalar = seq_len - 1;
    p.B = 1;
    p.Hq = num_heads;
    p.Hkv = kv_heads;
    p.G = q_heads_per_kv_head;
    p.D = head_dim;
    p.max_seq = max_seq_len;
    p.first_explicit = 0;
    p.append = 0;
    p.scale = scale;
    p.out = attn_out;
    p.out_dtype = B2A_FLOAT32;
    return run_decode(ctx, p, static_cast<cudaStream_t>(stream), false);
}

B2A_API int b2a_qwen_decode_step(b2a_context* ctx, const float* qkv, const float* qkv_bias, float* k_cache,
                                 float* v_cache, float* attn_out, int num_heads, int kv_heads, int head_dim, int pos,
                                 int max_seq_len, float rope_theta, float scale, void* stream) {
    // QwenGpuPipeline.decodeLayerGpuResident steps 1b-3 in one launch
    // (INF/qwen/QwenGpuPipeline.java:647-691): bias add on the fused [Q|K|V] row, RoPE of q and k
    // at pos, k/v append at pos, GQA attention over cache positions [0, pos].
    if (!ctx) return B2A_EINVAL;
    if (!qkv || !k_cache || !v_cache || !attn_out)
        return fail(ctx, B2A_EINVAL, "qkv, caches and attn_out must not be null");
    int rc = check_heads(ctx, num_heads, kv_heads);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, head_dim))) return rc;
    if (pos < 0 || pos >= max_seq_len) return fail(ctx, B2A_EINVAL, "pos %d outside [0, maxSeqLen=%d)", pos, max_seq_len);
    if (!(rope_theta > 0.f)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    DeviceGuard guard(ctx->device);
    const int64_t q_size = (int64_t)num_heads * head_dim, kv_size = (int64_t)kv_heads * head_dim;
    DecodeParams p{};
    p.q = qkv;
    p.k_new = qkv + q_size;
    p.v_new = qkv + q_size + kv_size;
    p.q_dtype = B2A_FLOAT32;
    p.q_seq_stride = p.kv_new_seq_stride = q_size + 2 * kv_size;
    if (qkv_bias) {
        p.q_bias = qkv_bias;
        p.k_bias = qkv_bias + q_size;
        p.v_bias = qkv_bias + q_size + kv_size;
    }
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.cache_dtype = B2A_FLOAT32;
    p.stride_b = 0;
    p.stride_h = (int64_t)max_seq_len * head_dim;
    p.stride_pos = head_dim;
    p.ctx_lens = nullptr;
    p.pos_scalar = pos;
    p.B = 1;
    p.Hq = num_heads;
    p.Hkv = kv_heads;
    p.G = num_heads / kv_heads;
    p.D = head_dim;
    p.max_seq = max_seq_len;
    p.first_explicit = 0;
    p.append = 1;
    p.rope_mode = B2A_ROPE_NEOX;
    inv_freq_table((double)rope_theta, head_dim, p.inv_freq);
    p.scale = scale;
    p.out = attn_out;
    p.out_dtype = B2A_FLOAT32;
    return run_decode(ctx, p, static_cast<cudaStream_t>(stream), false);
}

B2A_API int b2a_gemma_fused_attention_context(b2a_context* ctx, const float* q, const float* keys, const float* values,
                                              float* ctx_out, int num_heads, int groups_per_kv, int head_dim,
                                              int kv_dim, int first_valid, int query_pos, float scale, void* stream) {
    if (!ctx) return B2A_EINVAL;
    if (!q || !keys || !values || !ctx_out) return fail(ctx, B2A_EINVAL, "buffers must not be null");
    // Gemma3WarpFusedAttentionContextKernel.context (INF/gemma/Gemma3WarpFusedAttentionContextKernel.java:111-124)
    if (num_heads <= 0 || groups_per_kv <= 0 || num_heads % groups_per_kv != 0)
        return fail(ctx, B2A_EINVAL, "numHeads must be a multiple of numKvHeads");
    if (head_dim > 256)
        return fail(ctx, B2A_EINVAL, "headDim %d exceeds fused-attention group size 256", head_dim);
    int rc = check_head_dim(ctx, head_dim);
    if (rc) return rc;
    const int n_kv = num_heads / groups_per_kv;
    if (kv_dim < n_kv * head_dim) return fail(ctx, B2A_EINVAL, "kvDim %d < numKvHeads * headDim", kv_dim);
    if (query_pos < 0 || first_valid < 0 || first_valid > query_pos)
        return fail(ctx, B2A_EINVAL, "visible key range [%d, %d] is empty or negative", first_valid, query_pos);
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    DeviceGuard guard(ctx->device);
    DecodeParams p{};
    p.q = q;
    p.q_dtype = B2A_FLOAT32;
    p.k_cache = const_cast<float*>(keys);
    p.v_cache = const_cast<float*>(values);
    p.cache_dtype = B2A_FLOAT32;
    p.stride_b = 0;
    p.stride_h = head_dim;
    p.stride_pos = kv_dim;
    p.ctx_lens = nullptr;
    p.pos_scalar = query_pos;
    p.B = 1;
    p.Hq = num_heads;
    p.Hkv = n_kv;
    p.G = groups_per_kv;
    p.D = head_dim;
    p.max_seq = query_pos + 1;
    p.first_explicit = first_valid;
    p.append = 0;
    p.scale = scale;
    p.out = ctx_out;
    p.out_dtype = B2A_FLOAT32;
    return run_decode(ctx, p, static_cast<cudaStream_t>(stream), false);
}

// ----------------------------------------------------------------- projections
namespace {
// b2a_linear; early: launched with programmatic serialisation (the projections of
// b2a_decode_attention_block under b2a_set_decode_early_start)
int run_linear(b2a_context* ctx, int in_dtype, int out_dtype, const void* x, const void* w, const float* bias,
               const void* residual, void* y, int M, int N, int K, void* stream, bool early) {
    if (!ctx) return B2A_EINVAL;
    if (!x || !w || !y) return fail(ctx, B2A_EINVAL, "x, w and y must not be null");
    if (in_dtype != B2A_FLOAT16 && in_dtype != B2A_BFLOAT16)
        return fail(ctx, B2A_ENOTSUP, "b2a_linear multiplies 16-bit operands (FLOAT16 or BFLOAT16), got %d", in_dtype);
    if (!valid_dtype(out_dtype)) return fail(ctx, B2A_EINVAL, "unsupported output element type %d", out_dtype);
    if (M <= 0 || N <= 0 || K <= 0) return fail(ctx, B2A_EINVAL, "M, N and K must be > 0");
    if (K % 8 != 0) return fail(ctx, B2A_EINVAL, "K must be a multiple of 8 (16-byte rows for the TMA loads)");
    DeviceGuard guard(ctx->device);
    if (!linear_tc_supported(in_dtype, K, K, K, x, w))
        return fail(ctx, B2A_EINVAL, "x and w must be 16-byte aligned");
    LinearArgs a{};
    a.x = x;
    a.ldx = K;
    a.w = w;
    a.ldw = K;
    a.in_dtype = in_dtype;
    a.bias = bias;
    a.residual = residual;
    a.ldr = N;
    a.y = y;
    a.ldy = N;
    a.out_dtype = out_dtype;
    a.M = M;
    a.N = N;
    a.K = K;
    a.ksplit = 1;
    a.early = early ? 1 : 0;
    // launches with too few output tiles to fill the GPU split K over CTAs (without room for the
    // split workspace under the context's limit they run unsplit)
    size_t acc_bytes = 0, counter_ints = 0;
    const int ks = linear_split_plan(M, N, K, ctx->sm_count, &acc_bytes, &counter_ints);
    if (ks > 1) {
        // counters and accumulator: zeroed when new, kept zero by the kernel
        const size_t bytes = (counter_ints * sizeof(int) + acc_bytes + 511) / 256 * 256;
        const bool grow = bytes > ctx->lin_ws_bytes;
        if (ensure_buffer(ctx, &ctx->lin_ws, &ctx->lin_ws_bytes, bytes, "projection split workspace") == B2A_OK) {
            if (grow) {
                const cudaError_t e = cudaMemsetAsync(ctx->lin_ws, 0, bytes, static_cast<cudaStream_t>(stream));
                if (e != cudaSuccess) return cuda_fail(ctx, e, "projection split workspace");
            }
            a.ksplit = ks;
            a.counters = static_cast<int*>(ctx->lin_ws);
            a.acc = reinterpret_cast<float*>(static_cast<char*>(ctx->lin_ws) + (counter_ints * sizeof(int) + 255) / 256 * 256);
        } else {
            ctx->last_error.clear();  // the refused workspace is not an error of this call
        }
    }
    const cudaError_t e = launch_linear_tc(a, ctx->status, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "linear kernel launch");
    return B2A_OK;
}
}  // namespace

B2A_API int b2a_linear(b2a_context* ctx, int in_dtype, int out_dtype, const void* x, const void* w, const float* bias,
                       const void* residual, void* y, int M, int N, int K, void* stream) {
    return run_linear(ctx, in_dtype, out_dtype, x, w, bias, residual, y, M, N, K, stream, false);
}

B2A_API int b2a_decode_attention_block(b2a_context* ctx, int act_dtype, int cache_dtype, const void* x,
                                       const void* w_qkv, const float* b_qkv, void* k_cache, void* v_cache,
                                       int kv_layout, const int32_t* ctx_lens, const void* w_o, const void* residual,
                                       void* y, int B, int hidden, int Hq, int Hkv, int D, int max_seq, float scale,
                                       double rope_theta, int window, void* stream) {
    // Qwen2Runtime.processLayerDecode from the normed input to residual 1
    // (INF/qwen/Qwen2Runtime.java:693-777): QKV projection + bias, RoPE, KV append, GQA
    // attention, O projection + residual, in three launches -- the bias in the QKV GEMM's
    // epilogue, RoPE and the append in the attention's prologue, the residual in the O GEMM's
    // epilogue.
    if (!ctx) return B2A_EINVAL;
    if (!x || !w_qkv || !k_cache || !v_cache || !ctx_lens || !w_o || !y)
        return fail(ctx, B2A_EINVAL, "x, w_qkv, caches, ctx_lens, w_o and y must not be null");
    if (act_dtype != B2A_FLOAT16 && act_dtype != B2A_BFLOAT16)
        return fail(ctx, B2A_ENOTSUP, "activations and weights must be FLOAT16 or BFLOAT16");
    int rc = check_heads(ctx, Hq, Hkv);
    if (rc) return rc;
    if ((rc = check_head_dim(ctx, D))) return rc;
    if (B <= 0 || hidden <= 0 || max_seq <= 0) return fail(ctx, B2A_EINVAL, "B, hidden and max_seq must be > 0");
    if (hidden % 8 != 0 || (Hq * D) % 8 != 0)
        return fail(ctx, B2A_EINVAL, "hidden and Hq*D must be multiples of 8 (16-byte rows for the TMA loads)");
    if (!(rope_theta > 0.0)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    DeviceGuard guard(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int nqkv = (Hq + 2 * Hkv) * D;
    const size_t qkv_bytes = ((size_t)B * nqkv * 4 + 255) / 256 * 256;
    const size_t attn_bytes = (size_t)B * Hq * D * 2;
    rc = ensure_buffer(ctx, &ctx->blk_ws, &ctx->blk_ws_bytes, qkv_bytes + attn_bytes, "attention block");
    if (rc) return rc;
    float* qkv = static_cast<float*>(ctx->blk_ws);
    void* attn = static_cast<char*>(ctx->blk_ws) + qkv_bytes;
    // 1. qkv = x W_qkv^T + b (fp32 rows [Q | K | V], as the reference keeps them)
    if ((rc = run_linear(ctx, act_dtype, B2A_FLOAT32, x, w_qkv, b_qkv, nullptr, qkv, B, nqkv, hidden, stream,
                         ctx->decode_early_start)))
        return rc;
    // 2. RoPE of q and k at ctx_lens[b], k/v append, attention (the decode kernel reads the fused rows)
    DecodeParams p{};
    p.q = qkv;
    p.k_new = qkv + (int64_t)Hq * D;
    p.v_new = qkv + (int64_t)(Hq + Hkv) * D;
    p.q_dtype = B2A_FLOAT32;
    p.q_seq_stride = p.kv_new_seq_stride = nqkv;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.cache_dtype = cache_dtype;
    p.stride_b = (int64_t)Hkv * max_seq * D;
    if (kv_layout == B2A_KV_HEAD_MAJOR) {
        p.stride_h = (int64_t)max_seq * D;
        p.stride_pos = D;
    } else if (kv_layout == B2A_KV_POS_MAJOR) {
        p.stride_h = D;
        p.stride_pos = (int64_t)Hkv * D;
    } else {
        return fail(ctx, B2A_EINVAL, "unknown kv layout %d", kv_layout);
    }
    if (!valid_dtype(cache_dtype)) return fail(ctx, B2A_EINVAL, "unsupported cache element type %d", cache_dtype);
    p.ctx_lens = ctx_lens;
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.D = D;
    p.max_seq = max_seq;
    p.window = window;
    p.first_explicit = -1;
    p.append = 1;
    p.rope_mode = B2A_ROPE_NEOX;
    inv_freq_table(rope_theta, D, p.inv_freq);
    p.scale = scale;
    p.out = attn;
    p.out_dtype = act_dtype;
    if ((rc = run_decode(ctx, p, s, true))) return rc;
    // 3. y = attn W_o^T + residual
    return run_linear(ctx, act_dtype, act_dtype, attn, w_o, nullptr, residual, y, B, hidden, Hq * D, stream,
                      ctx->decode_early_start);
}

// ----------------------------------------------------------------- paged 4-bit cache
namespace {

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Fills the cache part of p from the caller's description.
int check_kv4_cache(b2a_context* ctx, const b2a_kv4_cache* cache, Kv4Params& p) {
    if (!cache || !cache->pages || !cache->page_table)
        return fail(ctx, B2A_EINVAL, "the cache, its pages and its page_table must not be null");
    const int D = cache->head_dim, ps = cache->page_size;
    if (cache->num_kv_heads <= 0) return fail(ctx, B2A_EINVAL, "numKeyValueHeads must be positive");
    if (D != 64 && D != 96 && D != 128 && D != 256)
        return fail(ctx, B2A_ENOTSUP, "the 4-bit cache holds headDim 64, 96, 128 or 256, got %d", D);
    if (ps <= 0 || ps % 16 != 0 || ps > kMaxPageSize)
        return fail(ctx, B2A_EINVAL, "page_size %d is not a multiple of 16 in [16, %d]", ps, kMaxPageSize);
    if (cache->num_pages <= 0 || cache->max_pages <= 0)
        return fail(ctx, B2A_EINVAL, "num_pages and max_pages must be > 0");
    if ((int64_t)cache->max_pages * ps > INT32_MAX)
        return fail(ctx, B2A_EINVAL, "max_pages * page_size exceeds the position range");
    if ((int64_t)cache->num_pages * cache->num_kv_heads * (ps / 16) > INT32_MAX)
        return fail(ctx, B2A_EINVAL, "the pool exceeds 2^31 blocks of 16 positions");
    if (!aligned16(cache->pages)) return fail(ctx, B2A_EINVAL, "the pages must be 16-byte aligned");
    p.pages = static_cast<uint8_t*>(cache->pages);
    p.page_table = cache->page_table;
    p.num_pages = cache->num_pages;
    p.page_size = ps;
    p.max_pages = cache->max_pages;
    p.Hkv = cache->num_kv_heads;
    p.D = D;
    p.status = ctx->status;
    return B2A_OK;
}

int check_kv4_tokens(b2a_context* ctx, int act_dtype, const int32_t* ctx_lens, const int32_t* new_lens, int B, int T,
                     int rope_mode, double rope_theta, float norm_eps, Kv4Params& p) {
    if (act_dtype != B2A_FLOAT16 && act_dtype != B2A_BFLOAT16)
        return fail(ctx, B2A_ENOTSUP, "the 4-bit cache takes FLOAT16 or BFLOAT16 rows, got %d", act_dtype);
    if (!ctx_lens) return fail(ctx, B2A_EINVAL, "ctx_lens must not be null");
    if (B <= 0 || T <= 0) return fail(ctx, B2A_EINVAL, "batch and new tokens must be > 0");
    if ((int64_t)B * T > (1 << 24)) return fail(ctx, B2A_EINVAL, "batch * new tokens exceeds 2^24");
    if (rope_mode != B2A_ROPE_NONE && rope_mode != B2A_ROPE_NEOX && rope_mode != B2A_ROPE_GEMMA)
        return fail(ctx, B2A_EINVAL, "unknown rope mode %d", rope_mode);
    if (rope_mode != B2A_ROPE_NONE && !(rope_theta > 0.0)) return fail(ctx, B2A_EINVAL, "rope theta must be > 0");
    if (!(norm_eps >= 0.f)) return fail(ctx, B2A_EINVAL, "norm_eps must not be negative");
    p.act_dtype = act_dtype;
    p.ctx_lens = ctx_lens;
    p.new_lens = new_lens;
    p.B = B;
    p.T = T;
    p.rope_mode = rope_mode;
    p.norm_eps = norm_eps;
    if (rope_mode != B2A_ROPE_NONE) {
        if (ctx->kv4_theta != rope_theta || ctx->kv4_inv_dim != p.D) {
            inv_freq_table(rope_theta, p.D, ctx->kv4_inv_freq);
            ctx->kv4_theta = rope_theta;
            ctx->kv4_inv_dim = p.D;
        }
        memcpy(p.inv_freq, ctx->kv4_inv_freq, sizeof(double) * (p.D / 2));
    }
    return B2A_OK;
}

int check_kv4_new(b2a_context* ctx, const void* k_new, const void* v_new, int64_t kv_stride, void* k_held,
                  void* v_held, const float* k_norm_w, Kv4Params& p) {
    if (!k_new || !v_new) return fail(ctx, B2A_EINVAL, "k_new and v_new must not be null");
    if (!aligned16(k_new) || !aligned16(v_new) || !aligned16(k_held) || !aligned16(v_held))
        return fail(ctx, B2A_EINVAL, "k_new, v_new, k_held and v_held must be 16-byte aligned");
    const int64_t row = (int64_t)p.Hkv * p.D;
    if (kv_stride == 0) kv_stride = row;
    if (kv_stride < row || kv_stride % 8 != 0)
        return fail(ctx, B2A_EINVAL, "kv_token_stride must be at least Hkv * D and a multiple of 8");
    p.k_new = k_new;
    p.v_new = v_new;
    p.kv_stride = kv_stride;
    p.k_held = k_held;
    p.v_held = v_held;
    p.k_norm_w = k_norm_w;
    return B2A_OK;
}

int check_kv4_query(b2a_context* ctx, const void* q, int64_t q_stride, int Hq, float scale, int window,
                    const float* q_norm_w, void* o, Kv4Params& p) {
    if (!q || !o) return fail(ctx, B2A_EINVAL, "q and o must not be null");
    const int rc = check_heads(ctx, Hq, p.Hkv);
    if (rc) return rc;
    if (!aligned16(q) || !aligned16(o)) return fail(ctx, B2A_EINVAL, "q and o must be 16-byte aligned");
    if (q_stride == 0) q_stride = (int64_t)Hq * p.D;
    if (q_stride < (int64_t)Hq * p.D || q_stride % 8 != 0)
        return fail(ctx, B2A_EINVAL, "q_token_stride must be at least Hq * D and a multiple of 8");
    if ((int64_t)p.B * p.T * Hq > INT32_MAX) return fail(ctx, B2A_EINVAL, "batch * new tokens * heads exceeds 2^31");
    if (window < 0) return fail(ctx, B2A_EINVAL, "window must not be negative");
    if (!(scale == scale) || scale <= 0.f) return fail(ctx, B2A_EINVAL, "scale must be a positive number");
    p.q = q;
    p.q_stride = q_stride;
    p.Hq = Hq;
    p.G = Hq / p.Hkv;
    p.scale = scale;
    p.window = window;
    p.q_norm_w = q_norm_w;
    p.o = o;
    return B2A_OK;
}

// Sequences [b0, b0 + count) of a call.
Kv4Params kv4_slice(const Kv4Params& p, int b0, int count) {
    Kv4Params s = p;
    const int64_t rows = (int64_t)b0 * p.T;
    auto advance = [](const void* x, int64_t elems) {
        return x ? static_cast<char*>(const_cast<void*>(x)) + elems * 2 : nullptr;
    };
    s.B = count;
    s.page_table += (int64_t)b0 * p.max_pages;
    s.ctx_lens += b0;
    if (s.new_lens) s.new_lens += b0;
    s.q = advance(p.q, rows * p.q_stride);
    s.k_new = advance(p.k_new, rows * p.kv_stride);
    s.v_new = advance(p.v_new, rows * p.kv_stride);
    s.k_held = advance(p.k_held, rows * p.Hkv * p.D);
    s.v_held = advance(p.v_held, rows * p.Hkv * p.D);
    s.o = advance(p.o, rows * p.Hq * p.D);
    return s;
}

// Chunks of prompts with bf16 results go to the tcgen05 kernel from this many tokens a sequence on;
// shorter ones, whose 128-row query tiles would stand mostly empty, and fp16 results, which carry q
// and P as two words, take the kernel that reads the codes (2 x 1000 tokens on 3000, 32 / 8 heads of
// 128: 1.6 ms in fp16, 0.16 ms in bf16).  Codes / staged rows, bf16: 4 sequences of 2000 cached, 32 / 8
// heads of 128, 48 tokens 78 / 57 us, 64 tokens 98 / 59 us; 16 of 1000, 14 / 2 of 64, 48 tokens 60 / 55 us,
// 64 tokens 73 / 55 us; where few sequences of long contexts let the staging's and the unsplit tiles' cost
// show, more tokens are needed: 8 of 2000, 4 / 1 of 256, 64 tokens 60 / 74 us, 96 tokens 75 / 74 us; 1 of
// 8000, 32 / 8 of 128, 64 tokens 82 / 127 us, 128 tokens 141 / 129 us.
constexpr int kKv4ChunkTokens = 64;
static_assert(kKv4ChunkTokens >= kKv4StoreTokens, "a chunk's append clears its flag");
constexpr size_t kKv4StageBytes = size_t(1) << 30;  // staged cache rows of one launch (one sequence at least)

bool kv4_chunked(const Kv4Params& p) { return p.act_dtype == B2A_BFLOAT16 && p.T >= kKv4ChunkTokens; }

// A chunk: the append, the operands as fp16 rows (kv4_stage.cu), the tcgen05 kernel, and the rows that
// see a value held as NaN.  kNoRoom: the staged rows did not fit, nothing was launched.
constexpr int kNoRoom = -1;
int run_kv4_chunk(b2a_context* ctx, const Kv4Params& p, cudaStream_t stream) {
    auto r256 = [](size_t x) { return (x + 255) / 256 * 256; };
    const int64_t Sk64 = ((int64_t)p.max_pages * p.page_size + 127) / 128 * 128;
    if (Sk64 > INT32_MAX - 128) return kNoRoom;
    const int Sk = (int)Sk64;
    const size_t kv_seq = (size_t)Sk * p.Hkv * p.D * 2, q_seq = (size_t)p.T * p.Hq * p.D * 2;
    const int per = (int)std::max<size_t>(1, std::min<size_t>(p.B, kKv4StageBytes / (2 * kv_seq + q_seq)));
    const size_t kv_bytes = r256(kv_seq * per), q_bytes = r256(q_seq * per);
    if (ensure_buffer(ctx, &ctx->pf_ws, &ctx->pf_ws_bytes, 2 * kv_bytes + q_bytes, "4-bit cache chunk") != B2A_OK) {
        ctx->last_error.clear();  // the refused workspace is not an error of this call
        return kNoRoom;
    }
    char* base = static_cast<char*>(ctx->pf_ws);
    AttnParams a{};
    a.in_dtype = B2A_FLOAT16;
    a.out_dtype = p.act_dtype;
    a.S = p.T;
    a.Sk = Sk;
    a.room = p.max_pages * p.page_size;  // Sk is whole tiles
    a.Hq = p.Hq;
    a.Hkv = p.Hkv;
    a.D = p.D;
    a.q_sb = (int64_t)p.T * p.Hq * p.D;
    a.q_ss = (int64_t)p.Hq * p.D;
    a.q_sh = p.D;
    a.k_sb = (int64_t)Sk * p.Hkv * p.D;
    a.k_ss = (int64_t)p.Hkv * p.D;
    a.k_sh = p.D;
    a.causal = 1;
    a.window = p.window;
    a.scale = p.scale;
    a.q = base;
    a.k = base + q_bytes;
    a.v = base + q_bytes + kv_bytes;
    a.B = per;
    a.q_pos = p.ctx_lens;
    a.o = p.o;
    if (!attn_tcgen05_supported(a)) return kNoRoom;
    cudaError_t e = cudaSuccess;
    if (p.k_new) {
        Kv4Params s = p;
        s.q = nullptr;
        s.nan_flag = ctx->status + kStatusNanWord;
        e = launch_kv4_prepare(s, ctx->sm_count, stream);
    }
    for (int b0 = 0; e == cudaSuccess && b0 < p.B; b0 += per) {
        Kv4Params s = kv4_slice(p, b0, std::min(per, p.B - b0));
        a.B = s.B;
        a.q_pos = s.ctx_lens;
        a.q_len = s.new_lens;
        a.o = s.o;
        s.nan_flag = ctx->status + kStatusNanWord;
        const bool after_append = p.k_new != nullptr && b0 == 0;  // which has cleared the flag
        if (!after_append) e = cudaMemsetAsync(s.nan_flag, 0, sizeof(int), stream);
        if (e == cudaSuccess)
            e = launch_kv4_stage(s, base, const_cast<void*>(a.k), const_cast<void*>(a.v), Sk, after_append,
                                 ctx->sm_count, stream);
        if (e == cudaSuccess) e = launch_attn_tcgen05(a, ctx->status, stream);
        if (e == cudaSuccess) e = launch_kv4_nan_rows(s, ctx->sm_count, stream);
    }
    if (e != cudaSuccess) return cuda_fail(ctx, e, "4-bit cache chunk launch");
    return B2A_OK;
}

// The preparation (q's operands, the plan, and the append where p has new rows), then the attention,
// at most kKv4MaxBatch sequences and 2^31 blocks of the split's stream at a time.
int run_kv4_attention(b2a_context* ctx, Kv4Params& p, cudaStream_t stream) {
    DeviceGuard guard(ctx->device);
    if (kv4_chunked(p)) {
        const int rc = run_kv4_chunk(ctx, p, stream);
        if (rc != kNoRoom) return rc;
    }
    auto r256 = [](size_t x) { return (x + 255) / 256 * 256; };
    const int64_t seq_blocks = (int64_t)p.max_pages * p.page_size / 16 + 1 + kKv4GapBlocksMax;
    const int per_launch = (int)std::max<int64_t>(1, std::min<int64_t>(kKv4MaxBatch, INT32_MAX / seq_blocks));
    p.split = kv4_attn_split(p, ctx->device);
    if (p.split.n_cta <= 0) return fail(ctx, B2A_ECUDA, "no attention kernel for this device");
    const int B = p.B, most = std::min(B, per_launch);
    const size_t units = (size_t)most * p.split.per_seq;
    const size_t part = r256(p.split.partial_bytes), plan = r256((p.split.n_cta + units) * sizeof(Kv4Piece)), frag = r256(kv4_frag_bytes(p) * most),
                 sums = r256(kv4_sums_bytes(p) * most);
    void* slots = nullptr;
    const int rc = ensure_counted_buffer(ctx, &ctx->kv4_ws, &ctx->kv4_ws_bytes, &ctx->kv4_counters, units,
                                         part + plan + frag + sums, "4-bit cache attention", stream, false,
                                         &p.counters, &slots);
    if (rc) return rc;
    char* at = static_cast<char*>(slots);
    auto take = [&](size_t bytes) {
        char* here = at;
        at += bytes;
        return here;
    };
    p.partials = reinterpret_cast<float*>(take(part));
    p.plan = reinterpret_cast<Kv4Piece*>(take(plan));
    p.q_frag = reinterpret_cast<uint4*>(take(frag));
    p.q_sums = reinterpret_cast<float*>(take(sums));
    cudaError_t e = cudaSuccess;
    for (int b0 = 0; e == cudaSuccess && b0 < B; b0 += per_launch) {
        Kv4Params s = kv4_slice(p, b0, std::min(per_launch, B - b0));
        e = launch_kv4_prepare(s, ctx->sm_count, stream);
        if (e == cudaSuccess) e = launch_kv4_attn(s, ctx->device, stream);
    }
    if (e != cudaSuccess) return cuda_fail(ctx, e, "4-bit cache attention launch");
    return B2A_OK;
}

int check_pool(b2a_context* ctx, const b2a_page_pool* pool, bool with_pages, PagePoolParams& p) {
    if (!pool || !pool->page_table || !pool->ref_counts)
        return fail(ctx, B2A_EINVAL, "the pool, its page_table and its ref_counts must not be null");
    if (pool->n_seq <= 0 || pool->max_pages <= 0 || pool->num_pages <= 0)
        return fail(ctx, B2A_EINVAL, "n_seq, max_pages and num_pages must be > 0");
    if ((int64_t)pool->n_seq * pool->max_pages > INT32_MAX)
        return fail(ctx, B2A_EINVAL, "the page table exceeds 2^31 entries");
    if (with_pages) {
        if (!pool->pages) return fail(ctx, B2A_EINVAL, "the pool's pages must not be null");
        if (pool->n_layers <= 0 || pool->page_bytes <= 0 || pool->page_bytes % 16 != 0 || !aligned16(pool->pages))
            return fail(ctx, B2A_EINVAL, "pages need n_layers > 0, 16-byte alignment and a multiple of 16 bytes");
        if (pool->n_layers > 1 && (pool->layer_stride % 16 != 0 ||
                                   pool->layer_stride < (int64_t)pool->num_pages * pool->page_bytes))
            return fail(ctx, B2A_EINVAL, "layer_stride must be a multiple of 16 and at least num_pages * page_bytes");
    }
    p.page_table = pool->page_table;
    p.n_seq = pool->n_seq;
    p.max_pages = pool->max_pages;
    p.ref_counts = pool->ref_counts;
    p.num_pages = pool->num_pages;
    p.pages = static_cast<uint8_t*>(pool->pages);
    p.n_layers = pool->n_layers;
    p.layer_stride = pool->layer_stride;
    p.page_bytes = pool->page_bytes;
    p.status = ctx->status;
    return B2A_OK;
}

int pages_workspace(b2a_context* ctx, int num_pages, cudaStream_t stream, int** sync, int** ws) {
    void* lists = nullptr;
    const int rc = ensure_counted_buffer(ctx, &ctx->pg_ws, &ctx->pg_ws_bytes, nullptr, kPageSyncInts,
                                         pages_workspace_ints(num_pages) * sizeof(int), "page operations", stream,
                                         false, sync, &lists);
    *ws = static_cast<int*>(lists);
    return rc;
}

}  // namespace

B2A_API size_t b2a_kv4_page_bytes(int num_kv_heads, int head_dim, int page_size) {
    if (num_kv_heads <= 0 || page_size <= 0 || page_size % 16 != 0 || page_size > kMaxPageSize) return 0;
    if (head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 256) return 0;
    return (size_t)num_kv_heads * page_size / 4 * 5 * head_dim;
}

B2A_API int b2a_kv4_append(b2a_context* ctx, const b2a_kv4_cache* cache, int act_dtype, const void* k_new,
                           const void* v_new, int64_t kv_token_stride, const int32_t* ctx_lens,
                           const int32_t* new_lens, int B, int T, int rope_mode, double rope_theta,
                           const float* k_norm_w, float norm_eps, void* k_held, void* v_held, void* stream) {
    if (!ctx) return B2A_EINVAL;
    Kv4Params p{};
    int rc = check_kv4_cache(ctx, cache, p);
    if (!rc) rc = check_kv4_tokens(ctx, act_dtype, ctx_lens, new_lens, B, T, rope_mode, rope_theta, norm_eps, p);
    if (!rc) rc = check_kv4_new(ctx, k_new, v_new, kv_token_stride, k_held, v_held, k_norm_w, p);
    if (rc) return rc;
    DeviceGuard guard(ctx->device);
    const cudaError_t e = launch_kv4_prepare(p, ctx->sm_count, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cache append launch");
    return B2A_OK;
}

B2A_API int b2a_kv4_attention(b2a_context* ctx, const b2a_kv4_cache* cache, int act_dtype, const void* q,
                              int64_t q_token_stride, const int32_t* ctx_lens, const int32_t* new_lens, int B, int T,
                              int Hq, float scale, int rope_mode, double rope_theta, int window,
                              const float* q_norm_w, float norm_eps, void* o, void* stream) {
    if (!ctx) return B2A_EINVAL;
    Kv4Params p{};
    int rc = check_kv4_cache(ctx, cache, p);
    if (!rc) rc = check_kv4_tokens(ctx, act_dtype, ctx_lens, new_lens, B, T, rope_mode, rope_theta, norm_eps, p);
    if (!rc) rc = check_kv4_query(ctx, q, q_token_stride, Hq, scale, window, q_norm_w, o, p);
    if (rc) return rc;
    return run_kv4_attention(ctx, p, static_cast<cudaStream_t>(stream));
}

B2A_API int b2a_kv4_decode(b2a_context* ctx, const b2a_kv4_cache* cache, int act_dtype, const void* q,
                           int64_t q_token_stride, const void* k_new, const void* v_new, int64_t kv_token_stride,
                           const int32_t* ctx_lens, const int32_t* new_lens, int B, int T, int Hq, float scale,
                           int rope_mode, double rope_theta, int window, const float* q_norm_w, const float* k_norm_w,
                           float norm_eps, void* k_held, void* v_held, void* o, void* stream) {
    if (!ctx) return B2A_EINVAL;
    Kv4Params p{};
    int rc = check_kv4_cache(ctx, cache, p);
    if (!rc) rc = check_kv4_tokens(ctx, act_dtype, ctx_lens, new_lens, B, T, rope_mode, rope_theta, norm_eps, p);
    if (!rc) rc = check_kv4_new(ctx, k_new, v_new, kv_token_stride, k_held, v_held, k_norm_w, p);
    if (!rc) rc = check_kv4_query(ctx, q, q_token_stride, Hq, scale, window, q_norm_w, o, p);
    if (rc) return rc;
    if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
        return fail(ctx, B2A_EINVAL, "q_norm_w and k_norm_w must be given together");
    return run_kv4_attention(ctx, p, static_cast<cudaStream_t>(stream));
}

B2A_API int b2a_pages_fork(b2a_context* ctx, const b2a_page_pool* pool, const int32_t* parents, void* stream) {
    if (!ctx) return B2A_EINVAL;
    PagePoolParams p{};
    const int rc = check_pool(ctx, pool, false, p);
    if (rc) return rc;
    if (!parents) return fail(ctx, B2A_EINVAL, "parents must not be null");
    if (p.n_seq > kMaxForkRows) return fail(ctx, B2A_ENOTSUP, "fork takes at most %d rows", kMaxForkRows);
    DeviceGuard guard(ctx->device);
    const cudaError_t e = launch_pages_fork(p, parents, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "page fork launch");
    return B2A_OK;
}

B2A_API int b2a_pages_free(b2a_context* ctx, const b2a_page_pool* pool, const int32_t* keep_from,
                           const int32_t* keep_to, int page_size, void* stream) {
    if (!ctx) return B2A_EINVAL;
    PagePoolParams p{};
    const int rc = check_pool(ctx, pool, false, p);
    if (rc) return rc;
    if (!keep_to) return fail(ctx, B2A_EINVAL, "keep_to must not be null");
    if (page_size <= 0) return fail(ctx, B2A_EINVAL, "page_size must be > 0");
    DeviceGuard guard(ctx->device);
    const cudaError_t e = launch_pages_free(p, keep_from, keep_to, page_size, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "page free launch");
    return B2A_OK;
}

B2A_API int b2a_pages_reserve(b2a_context* ctx, const b2a_page_pool* pool, const int32_t* ctx_lens,
                              const int32_t* new_lens, int page_size, int32_t* counts, void* stream) {
    if (!ctx) return B2A_EINVAL;
    PagePoolParams p{};
    int rc = check_pool(ctx, pool, true, p);
    if (rc) return rc;
    if (!ctx_lens || !new_lens || !counts) return fail(ctx, B2A_EINVAL, "ctx_lens, new_lens and counts must not be null");
    if (page_size <= 0) return fail(ctx, B2A_EINVAL, "page_size must be > 0");
    DeviceGuard guard(ctx->device);
    int *sync = nullptr, *ws = nullptr;
    if ((rc = pages_workspace(ctx, p.num_pages, static_cast<cudaStream_t>(stream), &sync, &ws))) return rc;
    const cudaError_t e = launch_pages_reserve(p, ctx_lens, new_lens, page_size, counts, sync, ws, ctx->sm_count,
                                               static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "page reserve launch");
    return B2A_OK;
}

B2A_API int b2a_pages_compact(b2a_context* ctx, const b2a_page_pool* pool, int32_t* counts, void* stream) {
    if (!ctx) return B2A_EINVAL;
    PagePoolParams p{};
    int rc = check_pool(ctx, pool, true, p);
    if (rc) return rc;
    if (!counts) return fail(ctx, B2A_EINVAL, "counts must not be null");
    DeviceGuard guard(ctx->device);
    int *sync = nullptr, *ws = nullptr;
    if ((rc = pages_workspace(ctx, p.num_pages, static_cast<cudaStream_t>(stream), &sync, &ws))) return rc;
    const cudaError_t e = launch_pages_compact(p, counts, sync, ws, ctx->sm_count, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(ctx, e, "page compact launch");
    return B2A_OK;
}

// ----------------------------------------------------------------- sharding
B2A_API int b2a_partition_units(int n_units, int n_ranks, const int64_t* unit_cost, int32_t* rank_of_unit) {
    if (n_units <= 0 || n_ranks <= 0 || !unit_cost || !rank_of_unit) return B2A_EINVAL;
    if (n_units % n_ranks != 0) return B2A_EINVAL;
    const int cap = n_units / n_ranks;
    std::vector<int> order(n_units);
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return unit_cost[a] > unit_cost[b]; });
    std::vector<int64_t> load(n_ranks, 0);
    std::vector<int> count(n_ranks, 0);
    for (int u : order) {
        int best = -1;
        for (int r = 0; r < n_ranks; ++r) {
            if (count[r] >= cap) continue;
            if (best < 0 || load[r] < load[best]) best = r;
        }
        rank_of_unit[u] = best;
        load[best] += unit_cost[u];
        ++count[best];
    }
    return B2A_OK;
}

}  // extern "C"
