// kv4_attn.cu -- attention of the new tokens of each sequence over the paged 4-bit cache (kv4.cuh).
//
// One warp per (token, query head): the row's dot product with each visible key, an online softmax
// in fp32 and the weighted sum of the values, element lane + 32 j of the row in a lane.
#include "kv4.cuh"

namespace b2a {
namespace {

constexpr int kAttnWarps = 4;

template <int D>
__global__ void __launch_bounds__(kAttnWarps * 32) kv4_attn_kernel(const __grid_constant__ Kv4Params p) {
    __shared__ float vec_all[kAttnWarps * D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* vec = vec_all + warp * D;
    const int64_t row = (int64_t)blockIdx.x * kAttnWarps + warp;
    if (row >= (int64_t)p.B * p.T * p.Hq) return;
    const int64_t tok = row / p.Hq;
    const int h = (int)(row - tok * p.Hq), kvh = h / p.G;
    const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
    int L, n;
    const bool ok = kv4_lens(p, b, L, n);
    if (!ok || t >= n) {
        if (!ok && lane == 0) atomicOr(p.status, 1);
        for (int d = lane; d < D; d += 32)
            store_from_float(p.o, row * D + d, ok ? 0.f : __int_as_float(0x7fc00000), p.act_dtype);
        return;
    }
    const int pos = L + t;
    const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    float q[D / 32], acc[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        q[j] = load_as_float(p.q, tok * p.q_stride + (int64_t)h * D + lane + 32 * j, p.act_dtype);
        acc[j] = 0.f;
    }
    kv4_norm_rope<D>(q, p.q_norm_w, p.norm_eps, p.rope_mode, p.inv_freq, pos, vec, lane);
    const float scale_log2 = p.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
    bool bad = false;
    const int shift = (lane & 8) ? 4 : 0, low = lane & ~8;
    for (int key = first; key <= pos; ++key) {
        const uint8_t* block = kv4_block_ptr(p, b, kvh, key);
        if (block == nullptr) {
            bad = true;
            break;
        }
        const int k16 = key % kKv4Block;
        const __half2* kp = reinterpret_cast<const __half2*>(block + kv4_off_kparam(D));
        const __half2* vp = reinterpret_cast<const __half2*>(block + kv4_off_vparam(D));
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int c = (block[kv4_k_byte(k16, low + 32 * j)] >> shift) & 15;
            s += q[j] * kv4_value(c, kp[kv4_param(k16, j, D / 32)]);
        }
        s = warp_sum(s) * scale_log2;
        const float mn = fmaxf(m, s);
        const float keep = exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * keep + w;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int c = (block[kv4_off_v(D) + kv4_v_byte(k16, low + 32 * j)] >> shift) & 15;
            acc[j] = acc[j] * keep + w * kv4_value(c, vp[kv4_param(k16, j, D / 32)]);
        }
    }
    if (bad && lane == 0) atomicOr(p.status, 16);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
        store_from_float(p.o, row * D + lane + 32 * j, bad ? __int_as_float(0x7fc00000) : acc[j] / l, p.act_dtype);
}

}  // namespace

cudaError_t launch_kv4_attn(const Kv4Params& p, cudaStream_t stream) {
    const int64_t rows = (int64_t)p.B * p.T * p.Hq;
    const unsigned grid = (unsigned)((rows + kAttnWarps - 1) / kAttnWarps);
    switch (p.D) {
        case 64: kv4_attn_kernel<64><<<grid, kAttnWarps * 32, 0, stream>>>(p); break;
        case 96: kv4_attn_kernel<96><<<grid, kAttnWarps * 32, 0, stream>>>(p); break;
        case 128: kv4_attn_kernel<128><<<grid, kAttnWarps * 32, 0, stream>>>(p); break;
        case 256: kv4_attn_kernel<256><<<grid, kAttnWarps * 32, 0, stream>>>(p); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace b2a
