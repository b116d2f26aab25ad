// kv4.cuh -- the paged 4-bit KV cache: layout, quantisation and row preparation shared by its
// kernels (kv4_append.cu, kv4_attn.cu).
//
// A layer's pool holds num_pages pages; the slab of (page, kv head) is page_size / 16 blocks of 16
// keys, and a block of 20 D bytes is [K codes 8D][K params 2D][V codes 8D][V params 2D].  A row of
// D values is held in groups of 32:
//     lo, hi = min, max;  s = f16((hi - lo) * f32(1/15));  z = f16(lo)
//     c = clamp(rint((x - z) * (1 / s)), 0, 15), every operation rounded to 32 bits; c = 0 where s = 0
// and stands for s * c + z; a group whose s or z is not finite is held as NaN (s = z = NaN).
//
// The codes lie in the order in which the 16x8x16 warp MMA takes its A operand, so that one 32-bit
// word of a lane holds its eight A elements of a 16 x 16 tile (K: 16 keys x 16 channels; V^T: 16
// channels x 16 keys) and needs no transposition, no shuffle and no shared-memory gather:
//     word (y * 32 + lane) * 2 + x  covers channels 32 y + 16 x .. + 15, lane = 4 g + t
//     K: nibble 2 * (2 e + r) + j = key g + 8 r, channel 8 j + 2 t + e of the tile
//     V: nibble 2 * (2 e + r) + j = key 2 t + e + 8 r, channel 8 j + g of the tile
// Two masks and a shift by 8 give the four f16x2 registers: w & 0x000F000F and w & 0x00F000F0 are
// pairs of f16 subnormals c * 2^-24 and c * 2^-20, exact, which the MMA multiplies exactly; the
// factors 2^24 and 2^20 go into q's elements (K) and into the output rows (V), as powers of two.
// A byte holds codes of one key only, so rows of a block are written independently of each other.
// Params: half2 (s, z) number (g * 2 + r) * (D / 32) + y for key g + 8 r.
#pragma once

#include <math.h>

#include "common.cuh"
#include "internal.h"

namespace b2a {
namespace {

constexpr int kKv4Block = 16;  // keys per block
constexpr int kKv4Group = 32;  // channels per (s, z) pair

__host__ __device__ constexpr int kv4_block_bytes(int D) { return 20 * D; }
__host__ __device__ constexpr int kv4_off_kparam(int D) { return 8 * D; }
__host__ __device__ constexpr int kv4_off_v(int D) { return 10 * D; }
__host__ __device__ constexpr int kv4_off_vparam(int D) { return 18 * D; }

// Byte of a block's code area that holds (key, channels d and d + 8); d's bit 3 is clear.
__device__ __forceinline__ int kv4_k_byte(int key, int d) {
    const int y = d >> 5, x = (d >> 4) & 1, t = (d & 7) >> 1, e = d & 1, g = key & 7, r = key >> 3;
    return ((y * 8 + g) * 4 + t) * 8 + x * 4 + 2 * e + r;
}
__device__ __forceinline__ int kv4_v_byte(int key, int d) {
    const int y = d >> 5, x = (d >> 4) & 1, g = d & 7, t = (key & 7) >> 1, e = key & 1, r = key >> 3;
    return ((y * 8 + g) * 4 + t) * 8 + x * 4 + 2 * e + r;
}
__device__ __forceinline__ int kv4_param(int key, int y, int groups) {
    return ((key & 7) * 2 + (key >> 3)) * groups + y;
}

// Sequence b's cached and new token counts; false (device status bit 0) where they do not fit the
// page table.
__device__ __forceinline__ bool kv4_lens(const Kv4Params& p, int b, int& L, int& n) {
    L = p.ctx_lens[b];
    n = p.new_lens ? p.new_lens[b] : p.T;
    const long long room = (long long)p.max_pages * p.page_size;
    if (L < 0 || n < 0 || n > p.T || (long long)L + n > room) {
        L = n = 0;
        return false;
    }
    return true;
}

// The slab of the block that holds position pos of (b, kv head), or null (status bit 4) where the
// table names no page of the pool.
__device__ __forceinline__ uint8_t* kv4_block_ptr(const Kv4Params& p, int b, int kvh, int pos) {
    const int slot = pos / p.page_size, in = pos - slot * p.page_size;
    const int page = p.page_table[(int64_t)b * p.max_pages + slot];
    if (page < 0 || page >= p.num_pages) return nullptr;
    const int64_t slab = (int64_t)(p.page_size / kKv4Block) * kv4_block_bytes(p.D);
    return p.pages + ((int64_t)page * p.Hkv + kvh) * slab + (int64_t)(in / kKv4Block) * kv4_block_bytes(p.D);
}

__device__ __forceinline__ double kv4_warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Optional zero-centred RMS norm, and RoPE with the position's (cos, sin) cs[0 .. D/2), of a row whose
// element lane + 32 j is x[j]; the whole warp, vec[0..D) is its scratch.  The arithmetic is that of
// b2a_decode's prologue (double sum of squares and angles; NeoX rotates in float, Gemma in double),
// each operation rounded by itself, so that the codes decided on the result are reproducible: exactly
// without rotation; with it, as far as the double sine and cosine, which short appends take one by one
// and prompts from kv4_block_angles, round to the same float.
template <int D>
__device__ __forceinline__ void kv4_norm_rope(float (&x)[D / 32], bool norm, const float (&norm_w)[D / 32], float eps,
                                              int rope_mode, const double2* cs, float* vec, int lane) {
    if (norm) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) ss += (double)x[j] * (double)x[j];
        ss = kv4_warp_sum(ss);
        const float rms = (float)(1.0 / sqrt(__dadd_rn(ss / (double)D, (double)eps)));
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
            x[j] = (float)__dmul_rn((double)__fmul_rn(x[j], rms), __dadd_rn(1.0, (double)norm_w[j]));
    }
    if (rope_mode == 0) return;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) vec[lane + 32 * j] = x[j];
    __syncwarp();
    for (int i = lane; i < D / 2; i += 32) {
        const float a = vec[i], b = vec[i + D / 2];
        const double c = cs[i].x, s = cs[i].y;
        if (rope_mode == 2) {
            vec[i] = (float)__dsub_rn(__dmul_rn((double)a, c), __dmul_rn((double)b, s));
            vec[i + D / 2] = (float)__dadd_rn(__dmul_rn((double)b, c), __dmul_rn((double)a, s));
        } else {
            const float cf = (float)c, sf = (float)s;
            vec[i] = __fsub_rn(__fmul_rn(a, cf), __fmul_rn(b, sf));
            vec[i + D / 2] = __fadd_rn(__fmul_rn(a, sf), __fmul_rn(b, cf));
        }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < D / 32; ++j) x[j] = vec[lane + 32 * j];
    __syncwarp();
}

// Cosines and sines of positions pos0 .. pos0 + 15, in 16-byte units that hold one channel's (cos, sin)
// as doubles (Gemma) or two channels' (cos, cos', sin, sin') as floats (NeoX): of channels 8 k .. + 7 a
// row, unit u lies at [row][u][k], so that neighbouring threads read neighbouring units.  By the
// block's first D / 2 threads: two double sincos each -- the first position and one step -- and a
// complex product per further position (an error of some 2^-50, far below the rounding to float; a
// sincos is about a hundred double instructions).
template <int D>
__device__ __forceinline__ void kv4_block_angles(const Kv4Params& p, int pos0, void* cs, int tid) {
    if (tid >= D / 2) return;
    double s, c, s1, c1;
    sincos((double)pos0 * p.inv_freq[tid], &s, &c);
    sincos(p.inv_freq[tid], &s1, &c1);
#pragma unroll
    for (int row = 0; row < 16; ++row) {
        if (p.rope_mode == 2) {
            static_cast<double2*>(cs)[row * (D / 2) + (tid & 7) * (D / 16) + (tid >> 3)] = make_double2(c, s);
        } else {
            float* at = static_cast<float*>(cs) + (row * (D / 4) + (tid >> 1 & 3) * (D / 16) + (tid >> 3)) * 4 + (tid & 1);
            at[0] = (float)c;
            at[2] = (float)s;
        }
        const double next = c * c1 - s * s1;
        s = s * c1 + c * s1;
        c = next;
    }
}

// Quantises the warp's row: lane + 32 j is element lane of group j.  code[j] in 0..15, sz[j] the
// group's (s, z); true where every group is finite.
template <int N>
__device__ __forceinline__ bool kv4_quantise(const float (&x)[N], int (&code)[N], __half2 (&sz)[N]) {
    bool fine = true;
    float low[N], high[N];
#pragma unroll
    for (int j = 0; j < N; ++j) low[j] = high[j] = x[j];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            low[j] = fminf(low[j], __shfl_xor_sync(0xffffffffu, low[j], o));
            high[j] = fmaxf(high[j], __shfl_xor_sync(0xffffffffu, high[j], o));
        }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float lo = low[j], hi = high[j];
        __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), z = __float2half_rn(lo);
        const float sf = __half2float(s), zf = __half2float(z);
        const bool ok = !__any_sync(0xffffffffu, !isfinite(x[j])) && isfinite(sf) && isfinite(zf);
        const float inv = sf > 0.f ? __fdiv_rn(1.0f, sf) : 0.f;
        const float c = rintf(__fmul_rn(__fsub_rn(x[j], zf), inv));
        code[j] = ok ? (int)fminf(fmaxf(c, 0.f), 15.f) : 0;
        if (!ok) s = z = __ushort_as_half(0x7fff);
        sz[j] = __halves2half2(s, z);
        fine &= ok;
    }
    return fine;
}
__device__ __forceinline__ float kv4_value(int code, __half2 sz) {
    return __fadd_rn(__fmul_rn((float)code, __low2float(sz)), __high2float(sz));
}

}  // namespace
}  // namespace b2a
