// kv4_append.cu -- what comes before the attention over the paged 4-bit cache (kv4.cuh), one launch:
// new K/V rows into the cache (optional key norm, RoPE, group quantisation), the rows as the cache
// holds them for callers that want the prompt's own attention to see the same values, and the
// queries' norm, RoPE and layout as the warp MMA's B operand (kv4_attn.cu).
//
// One warp per query row and per (token, kv head, K or V).  The launch lets the attention kernel
// behind it start at once: that kernel plans and requests its first old blocks meanwhile.
#include "kv4.cuh"

namespace b2a {
namespace {

constexpr int kPrepWarps = 4;

// Query row r = token * G + head of the group, of (sequence b, kv head).  Its element 16 x + 8 j +
// 2 t + e of group y goes to half e of operand word (y, lane 4 (r % 8) + t, 2 x + j) of 8-row tile
// r / 8, as q 2^-E / 16^j with |q 2^-E| < 2^14 (the codes of channels with j = 1 enter the product
// 16 times larger); fp16 activations keep a second word with what the first rounding lost.
// q_sums: sum of the group's operand values 2^-24 per group, then scale log2(e) 2^(E + 24).
template <int D>
__device__ __forceinline__ void prepare_query(const Kv4Params& p, int b, int kvh, int r, float* vec, int lane) {
    constexpr int kGroups = D / 32;
    const int tiles = (p.T * p.G + 7) / 8;
    const int64_t tile = ((int64_t)b * p.Hkv + kvh) * tiles + (r >> 3);
    __half* frag = reinterpret_cast<__half*>(p.q_frag + tile * (kGroups * 32 * 2));
    float* sums = p.q_sums + tile * (kGroups + 1) * 8 + (r & 7);
    const int t = r / p.G, hg = r - t * p.G;
    int L = 0, n = 0;
    const bool ok = kv4_lens(p, b, L, n);
    if (!ok && lane == 0) atomicOr(p.status, 1);
    const int64_t tok = (int64_t)b * p.T + t;
    const int h = kvh * p.G + hg;
    const bool there = t < n;
    if (!there && t < p.T)
        for (int d = lane; d < D; d += 32)
            store_from_float(p.o, (tok * p.Hq + h) * D + d, ok ? 0.f : __int_as_float(0x7fc00000), p.act_dtype);
    float x[kGroups], top = 0.f;
#pragma unroll
    for (int y = 0; y < kGroups; ++y)
        x[y] = there ? load_as_float(p.q, tok * p.q_stride + (int64_t)h * D + lane + 32 * y, p.act_dtype) : 0.f;
    bool fine = true;
    if (there) kv4_norm_rope<D>(x, p.q_norm_w, p.norm_eps, p.rope_mode, p.inv_freq, L + t, vec, lane);
#pragma unroll
    for (int y = 0; y < kGroups; ++y) {
        top = fmaxf(top, fabsf(x[y]));
        fine &= isfinite(x[y]);
    }
    top = warp_max(top);
    fine = __all_sync(0xffffffffu, fine);
    const int E = fine && top > 0.f ? ilogbf(top) - 13 : 0;
    const int j = (lane >> 3) & 1;
    const int word = ((r & 7) * 4 + ((lane & 7) >> 1)) * 4 + 2 * (lane >> 4) + j;
#pragma unroll
    for (int y = 0; y < kGroups; ++y) {
        const float v = fine ? scalbnf(x[y], -E) * (j ? 0.0625f : 1.f) : 0.f;
        const __half hi = __float2half_rn(v);
        const int at = (y * 32 * 4 + word) * 2 + (lane & 1);
        frag[at] = hi;
        float used = __half2float(hi);
        if (p.act_dtype == kF16) {
            const __half lo = __float2half_rn(v - used);
            frag[kGroups * 32 * 4 * 2 + at] = lo;
            used += __half2float(lo);
        }
        const float s = warp_sum(used * (j ? 0x1p-20f : 0x1p-24f));
        if (lane == 0) sums[y * 8] = s;
    }
    if (lane == 0) sums[kGroups * 8] = fine ? scalbnf(p.scale * kLog2e, E + 24) : __int_as_float(0x7fc00000);
}

template <int D>
__device__ __forceinline__ void append_row(const Kv4Params& p, int64_t row, float* vec, int lane) {
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

template <int D>
__global__ void __launch_bounds__(kPrepWarps * 32) kv4_prepare_kernel(const __grid_constant__ Kv4Params p,
                                                                      int64_t q_rows, int64_t kv_rows) {
    __shared__ float vec_all[kPrepWarps * D];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * kPrepWarps + warp;
    if (row < q_rows) {
        const int per = (p.T * p.G + 7) / 8 * 8;  // rows of (sequence, kv head), whole tiles
        const int64_t bk = row / per;
        const int b = (int)(bk / p.Hkv);
        prepare_query<D>(p, b, (int)(bk - (int64_t)b * p.Hkv), (int)(row - bk * per), vec_all + warp * D, lane);
    } else if (row - q_rows < kv_rows) {
        append_row<D>(p, row - q_rows, vec_all + warp * D, lane);
    }
}

}  // namespace

cudaError_t launch_kv4_prepare(const Kv4Params& p, cudaStream_t stream) {
    const int64_t q_rows = p.q ? (int64_t)p.B * p.Hkv * ((p.T * p.G + 7) / 8 * 8) : 0;
    const int64_t kv_rows = p.k_new ? (int64_t)p.B * p.T * p.Hkv * 2 : 0;
    const unsigned grid = (unsigned)((q_rows + kv_rows + kPrepWarps - 1) / kPrepWarps);
    constexpr int kT = kPrepWarps * 32;
    switch (p.D) {
        case 64: kv4_prepare_kernel<64><<<grid, kT, 0, stream>>>(p, q_rows, kv_rows); break;
        case 96: kv4_prepare_kernel<96><<<grid, kT, 0, stream>>>(p, q_rows, kv_rows); break;
        case 128: kv4_prepare_kernel<128><<<grid, kT, 0, stream>>>(p, q_rows, kv_rows); break;
        case 256: kv4_prepare_kernel<256><<<grid, kT, 0, stream>>>(p, q_rows, kv_rows); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace b2a
