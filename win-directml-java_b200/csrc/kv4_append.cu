// kv4_append.cu -- new K/V rows into the paged 4-bit cache: optional key norm, RoPE, group
// quantisation (kv4.cuh), and the rows as the cache holds them for callers that want the prompt's
// own attention to see the same values.
//
// One warp per (token, kv head, K or V).
#include "kv4.cuh"

namespace b2a {
namespace {

constexpr int kAppendWarps = 4;

template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32) kv4_append_kernel(const __grid_constant__ Kv4Params p) {
    __shared__ float vec_all[kAppendWarps * D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* vec = vec_all + warp * D;
    const int64_t rows = (int64_t)p.B * p.T * p.Hkv * 2;
    const int64_t row = (int64_t)blockIdx.x * kAppendWarps + warp;
    if (row >= rows) return;
    const int is_v = (int)(row & 1);
    const int64_t tok = (row >> 1) / p.Hkv;
    const int kvh = (int)((row >> 1) - tok * p.Hkv);
    const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
    int L, n;
    const bool ok = kv4_lens(p, b, L, n);
    void* held = is_v ? p.v_held : p.k_held;
    const int64_t held_at = (tok * p.Hkv + kvh) * D;
    if (!ok || t >= n) {
        if (!ok && lane == 0) atomicOr(p.status, 1);
        if (held)
            for (int d = lane; d < D; d += 32)
                store_from_float(held, held_at + d, ok ? 0.f : __int_as_float(0x7fc00000), p.act_dtype);
        return;
    }
    const int pos = L + t, key = pos % kKv4Block;
    const void* src = is_v ? p.v_new : p.k_new;
    float x[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
        x[j] = load_as_float(src, tok * p.kv_stride + (int64_t)kvh * D + lane + 32 * j, p.act_dtype);
    if (!is_v) kv4_norm_rope<D>(x, p.k_norm_w, p.norm_eps, p.rope_mode, p.inv_freq, pos, vec, lane);
    int code[D / 32];
    __half2 sz[D / 32];
    if (!kv4_quantise(x, code, sz) && lane == 0) atomicOr(p.status, 32);
    uint8_t* block = kv4_block_ptr(p, b, kvh, pos);
    if (block == nullptr && lane == 0) atomicOr(p.status, 16);
    if (block != nullptr && is_v) block += kv4_off_v(D);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const int d = lane + 32 * j;
        const int up = __shfl_down_sync(0xffffffffu, code[j], 8);
        if (held) store_from_float(held, held_at + d, kv4_value(code[j], sz[j]), p.act_dtype);
        if (block == nullptr) continue;
        if ((lane & 8) == 0) block[is_v ? kv4_v_byte(key, d) : kv4_k_byte(key, d)] = (uint8_t)(code[j] | up << 4);
        if (lane == 0) reinterpret_cast<__half2*>(block + kv4_off_kparam(D))[kv4_param(key, j, D / 32)] = sz[j];
    }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Params& p, cudaStream_t stream) {
    const int64_t rows = (int64_t)p.B * p.T * p.Hkv * 2;
    const unsigned grid = (unsigned)((rows + kAppendWarps - 1) / kAppendWarps);
    switch (p.D) {
        case 64: kv4_append_kernel<64><<<grid, kAppendWarps * 32, 0, stream>>>(p); break;
        case 96: kv4_append_kernel<96><<<grid, kAppendWarps * 32, 0, stream>>>(p); break;
        case 128: kv4_append_kernel<128><<<grid, kAppendWarps * 32, 0, stream>>>(p); break;
        case 256: kv4_append_kernel<256><<<grid, kAppendWarps * 32, 0, stream>>>(p); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace b2a
