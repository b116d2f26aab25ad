// kv4_stage.cu -- operands of the tcgen05 attention kernel for chunks of prompts over the paged 4-bit
// cache (kv4.cuh): q rotated and converted to fp16, the visible cache rows as fp16.
//
// A chunk reads every key of its sequence once per 256 of its tokens and head, so the codes are turned
// into fp16 rows once, by one launch (0.625 D bytes in, 2 D out per row), and the
// tensor-core kernel streams those through TMA; per key and head that is far less than the chunk's
// own multiplications.  Measured for 2 x 1000 tokens of 32 heads of 128 on 2 x 3000 cached ones (8 kv
// heads, 87 MB moved): 27 us, of them 16 behind the append beside which the queries are staged,
// before an attention of 102 us (the whole call: 152 to 177 us on one GPU, the attention's clock moving); its warps wait for loads, half of the issue slots are idle.  Turning
// the blocks before the appended ones while the append runs gained nothing (the GPU is full).
// A value beyond fp16 becomes infinite and raises status bit 2, as bf16 inputs of the other entry
// points do.
#include <type_traits>

#include "kv4.cuh"
#include "sm100.cuh"

namespace b2a {
namespace {

// positions [first, L + n) are seen by some token of the chunk; rows are staged from `first` rounded
// down, to L + n rounded up, to whole tiles of 128 keys
__device__ __forceinline__ int first_seen(const Kv4Params& p, int L) {
    return p.window > 0 ? max(0, L - p.window + 1) : 0;
}

// ---------------------------------------------------------------- q
// A block takes 16 tokens of a sequence and kStageHeads heads, two at a time; a thread holds channels
// 8 k .. + 7 and their partners D / 2 further.  Its sines serve eight heads (32 heads of 128, 2 x
// 1000 tokens: with 2, 4, 8 and 16 the launch takes 31.6, 28.8, 27.5 and 27.7 us).
constexpr int kStageHeads = 8;
template <int D, typename T>
__device__ __forceinline__ void stage_query(const Kv4Params& p, __half* out, int block, int blocks, unsigned char* smem) {
    constexpr int kHalf = D / 16, kThreads = 2 * D;  // chunk pairs of a row; 2 heads x 16 tokens x kHalf threads
    void* const cs = smem;  // [16][D / 2] (cos, sin)
    double* const part = reinterpret_cast<double*>(smem + 16 * (D / 2) * sizeof(double2));
    const int tid = threadIdx.x;
    const int head_blocks = (p.Hq + kStageHeads - 1) / kStageHeads;
    const int head0 = block % head_blocks * kStageHeads, head1 = min(p.Hq, head0 + kStageHeads);
    block /= head_blocks;
    const int b = block / blocks, t0 = (block - b * blocks) * 16;
    int L, n;
    const bool ok = kv4_lens(p, b, L, n);
    if (!ok && tid == 0) atomicOr(p.status, 1);
    const int sub = tid / (kThreads / 2), rest = tid - sub * (kThreads / 2);
    const int row = rest / kHalf, k = rest - row * kHalf;
    const int t = t0 + row;
    const int64_t tok = (int64_t)b * p.T + t;
    const bool there = t < n;
    if (!there && t < p.T) {  // no such token: its outputs are zero, or NaN where the lengths do not fit
        const uint32_t v = ok ? 0u : 0x7fff7fffu;
        for (int h = head0 + sub; h < head1; h += 2) {
            uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (tok * p.Hq + h) * D + 8 * k);
            o[0] = o[kHalf] = make_uint4(v, v, v, v);
        }
    }
    if (t0 >= n) return;
    if (p.rope_mode != 0) kv4_block_angles<D>(p, L + t0, cs, tid);
    __syncthreads();
    float top = 0.f;
    for (int h0 = head0; h0 < head1; h0 += 2) {
        const int h = h0 + sub;
        const bool live = there && h < head1;
        float x[8], y[8];
        uint4 wx = make_uint4(0, 0, 0, 0), wy = wx;
        if (live) {
            const T* src = static_cast<const T*>(p.q) + tok * p.q_stride + (int64_t)h * D + 8 * k;
            wx = *reinterpret_cast<const uint4*>(src);
            wy = *reinterpret_cast<const uint4*>(src + D / 2);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = Elem<T>::to_float(reinterpret_cast<const T*>(&wx)[i]);
            y[i] = Elem<T>::to_float(reinterpret_cast<const T*>(&wy)[i]);
        }
        if (p.q_norm_w) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += (double)x[i] * (double)x[i] + (double)y[i] * (double)y[i];
            part[tid] = ss;
            __syncthreads();
            ss = 0.0;
            for (int i = 0; i < kHalf; ++i) ss += part[tid - k + i];
            __syncthreads();
            const float rms = (float)(1.0 / sqrt(ss / (double)D + (double)p.norm_eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = (float)((double)__fmul_rn(x[i], rms) * (1.0 + (double)p.q_norm_w[8 * k + i]));
                y[i] = (float)((double)__fmul_rn(y[i], rms) * (1.0 + (double)p.q_norm_w[D / 2 + 8 * k + i]));
            }
        }
        if (p.rope_mode == 2) {
            const double2* at = static_cast<const double2*>(cs) + row * (D / 2) + k;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = x[i], e = y[i];
                const double2 c = at[i * kHalf];
                x[i] = (float)((double)a * c.x - (double)e * c.y);
                y[i] = (float)((double)e * c.x + (double)a * c.y);
            }
        } else if (p.rope_mode != 0) {
            const float4* at = static_cast<const float4*>(cs) + row * (D / 4) + k;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 c = at[i / 2 * kHalf];
                const float a0 = x[i], e0 = y[i], a1 = x[i + 1], e1 = y[i + 1];
                x[i] = a0 * c.x - e0 * c.z;
                y[i] = a0 * c.z + e0 * c.x;
                x[i + 1] = a1 * c.y - e1 * c.w;
                y[i + 1] = a1 * c.w + e1 * c.y;
            }
        }
        if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(y[i])));
            __half* dst = out + (tok * p.Hq + h) * D + 8 * k;
            store8(dst, 0, x, kF16);
            store8(dst, D / 2, y, kF16);
        }
    }
    if (top >= 65520.f) atomicOr(p.status, 4);
}

// ---------------------------------------------------------------- cache rows
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4], int t) {  // lane t of four: w[c] of lane c's w[t]
#pragma unroll
    for (int bit = 1; bit <= 2; bit <<= 1)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int lo = bit == 1 ? 2 * i : i;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, t & bit ? w[lo] : w[lo + bit], bit);
            if (t & bit) w[lo] = got;
            else w[lo + bit] = got;
        }
}
// One warp turns one group (32 channels) of a block of 16 positions into fp16 rows.  A lane's two code
// words hold, as the MMA wants them, channel pairs of keys g and g + 8 (K) or key pairs of channels
// (V^T); the latter are transposed 8 x 8 at a time.  s c + z is one f16 FMA on the exact code: rounded
// once.  (Rows written 4 bytes a lane, without the exchange below: 2 us more of 29.)
template <int D>
__device__ __forceinline__ void stage_group(const Kv4Params& p, const uint8_t* src, int y, int pos, int first, int end,
                                            __half* k_row0, __half* v_row0, int64_t row_stride, int lane) {
    constexpr int kGroups = D / 32;
    const int g = lane >> 2, t = lane & 3;
    auto seen = [&](int key) { return src != nullptr && pos + key >= first && pos + key < end; };
    uint32_t code[2][2] = {{0, 0}, {0, 0}}, sz[2][3][2] = {};  // [K or V][..]: key g / 2 t / 2 t + 1, + 8
    if (src != nullptr) {
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
            const uint8_t* at = src + is_v * kv4_off_v(D);
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(at + y * 256 + lane * 8));
            code[is_v][0] = w.x;
            code[is_v][1] = w.y;
            const uint32_t* par = reinterpret_cast<const uint32_t*>(at + kv4_off_kparam(D)) + y;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (!is_v) {
                    sz[0][0][r] = __ldg(par + (g * 2 + r) * kGroups);
                } else {
                    sz[1][1][r] = __ldg(par + (2 * t * 2 + r) * kGroups);
                    sz[1][2][r] = __ldg(par + ((2 * t + 1) * 2 + r) * kGroups);
                }
            }
        }
    }
    auto value = [](uint32_t w, uint32_t s2, uint32_t z2) {
        const uint32_t c = (w & 0x000F000Fu) | 0x64006400u;  // f16x2 1024 + code
        const __half2 x = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), __float2half2_rn(1024.f)),
                                  *reinterpret_cast<const __half2*>(&s2), *reinterpret_cast<const __half2*>(&z2));
        return *reinterpret_cast<const uint32_t*>(&x);
    };
    bool nan = false;
    __half2 top = __float2half2_rn(0.f);  // largest |value|: infinite where one left the fp16 range
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const bool row_seen = seen(g + 8 * r);
        // a key held as NaN scores NaN, which a part of the softmax's exponentials would take for a small
        // number: its rows are marked later too
        nan |= row_seen && (sz[0][0][r] & 0x7fffu) > 0x7c00u;
        const uint32_t ks = __byte_perm(sz[0][0][r], 0, 0x1010), kz = __byte_perm(sz[0][0][r], 0, 0x3232);
        uint32_t vs = __byte_perm(sz[1][1][r], sz[1][2][r], 0x5410), vz = __byte_perm(sz[1][1][r], sz[1][2][r], 0x7632);
        // a value held as NaN counts as zero here; the rows that see it are marked later
        if ((vs & 0x7fffu) > 0x7c00u) {
            nan |= seen(2 * t + 8 * r);
            vs &= 0xffff0000u, vz &= 0xffff0000u;
        }
        if ((vs >> 16 & 0x7fffu) > 0x7c00u) {
            nan |= seen(2 * t + 1 + 8 * r);
            vs &= 0xffffu, vz &= 0xffffu;
        }
        uint32_t k[4], v[4];  // channels 8 c + 2 t, + 1
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            k[c] = value(code[0][c >> 1] >> (8 * r + 4 * (c & 1)), ks, kz);
            v[c] = movmatrix_trans(value(code[1][c >> 1] >> (8 * r + 4 * (c & 1)), vs, vz));
            if (!row_seen) k[c] = v[c] = 0;
            top = __hmax2(top, __hmax2(__habs2(*reinterpret_cast<const __half2*>(&k[c])),
                                       __habs2(*reinterpret_cast<const __half2*>(&v[c]))));
        }
        // the row's four lanes exchange, so that each writes 16 bytes: channels 8 t .. + 7
        quad_transpose(k, t);
        quad_transpose(v, t);
        const int64_t at = (int64_t)(g + 8 * r) * row_stride + 32 * y + 8 * t;
        *reinterpret_cast<uint4*>(k_row0 + at) = make_uint4(k[0], k[1], k[2], k[3]);
        *reinterpret_cast<uint4*>(v_row0 + at) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    const bool big = __hisinf(__low2half(top)) || __hisinf(__high2half(top));
    if (__any_sync(0xffffffffu, big) && lane == 0) atomicOr(p.status, 4);
    if (__any_sync(0xffffffffu, nan) && lane == 0) atomicExch(p.nan_flag, 1);
}

template <int D, typename T>
__global__ void __launch_bounds__(2 * D) kv4_stage_kernel(const __grid_constant__ Kv4Params p, __half* q_out, __half* k_out,
                                                          __half* v_out, int Sk, int q_blocks, int q_total) {
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if ((int)blockIdx.x < q_total) {
        stage_query<D, T>(p, q_out, blockIdx.x, q_blocks, smem);
        return;
    }
    // the append before this launch wrote the new rows' codes; the queries above did not need them
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t row_stride = (int64_t)p.Hkv * D;
    constexpr int kGroups = D / 32, kWarps = 2 * D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t i = (int64_t)(blockIdx.x - q_total) * kWarps + warp;
    const int step = (gridDim.x - q_total) * kWarps;
    for (int b = 0; b < p.B; ++b) {
        int L, n;
        if (!kv4_lens(p, b, L, n) || n == 0) continue;
        const int first = first_seen(p, L), end = L + n;
        const int blk0 = first / 128 * 8, blk1 = min((end + 127) / 128 * 8, Sk / kKv4Block);
        const int per_blk = p.Hkv * kGroups;
        const int64_t count = (int64_t)(blk1 - blk0) * per_blk;
        for (; i < count; i += step) {
            // below 2^31: a group is 2 KB of staged rows
            const unsigned at_blk = (unsigned)i / (unsigned)per_blk, in = (unsigned)i - at_blk * per_blk;
            const int blk = blk0 + (int)at_blk, h = in / kGroups, y = in % kGroups;
            const int pos = blk * kKv4Block;
            const bool seen = pos + kKv4Block > first && pos < end;
            const uint8_t* src = seen ? kv4_block_ptr(p, b, h, pos) : nullptr;
            if (seen && src == nullptr && lane == 0) {
                atomicOr(p.status, 16);
                atomicExch(p.nan_flag, 1);
            }
            const int64_t at = ((int64_t)b * Sk + pos) * row_stride + (int64_t)h * D;
            stage_group<D>(p, src, y, pos, first, end, k_out + at, v_out + at, row_stride, lane);
        }
        i -= count;
    }
}

// Rows that see a value group held as NaN, a key held as NaN, or a page that does not exist: their
// outputs become NaN (the group's channels; all of the row's).  Runs to its end only where the staging
// met one.
__global__ void __launch_bounds__(256) kv4_nan_rows_kernel(const __grid_constant__ Kv4Params p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (__ldcg(p.nan_flag) == 0) return;
    const int D = p.D, groups = D / 32;
    const int64_t rows = (int64_t)p.B * p.T * p.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < rows; row += (int64_t)gridDim.x * 8) {
        const int64_t tok = row / p.Hkv;
        const int kvh = (int)(row - tok * p.Hkv), b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
        int L, n;
        if (!kv4_lens(p, b, L, n) || t >= n) continue;
        const int first = p.window > 0 ? max(0, L + t - p.window + 1) : 0;
        unsigned hit = 0;  // bit per value group, bit 31: the key, or a page that is missing
        for (int key = first + lane; key <= L + t; key += 32) {
            const uint8_t* block = kv4_block_ptr(p, b, kvh, key);
            if (block == nullptr) {
                hit |= 1u << 31;
                continue;
            }
            const __half2* ks = reinterpret_cast<const __half2*>(block + kv4_off_kparam(D));
            const __half2* vs = reinterpret_cast<const __half2*>(block + kv4_off_vparam(D));
            for (int y = 0; y < groups; ++y) {
                const int at = kv4_param(key % kKv4Block, y, groups);
                if (__hisnan(__low2half(ks[at]))) hit |= 1u << 31;
                if (__hisnan(__low2half(vs[at]))) hit |= 1u << y;
            }
        }
        hit = __reduce_or_sync(0xffffffffu, hit);
        if (hit == 0) continue;
        for (int e = lane; e < p.G * D; e += 32) {
            const int d = e % D;
            if (hit >> 31 || (hit >> (d / 32) & 1))
                store_from_float(p.o, (tok * p.Hq + kvh * p.G) * D + e, __int_as_float(0x7fc00000), p.act_dtype);
        }
    }
}

template <int D, typename T>
cudaError_t launch_stage(const Kv4Params& p, __half* q_out, __half* k_out, __half* v_out, int Sk, bool after_append,
                         int sm_count, cudaStream_t stream) {
    const size_t smem = 16 * (D / 2) * sizeof(double2) + 2 * D * sizeof(double);
    auto kern = kv4_stage_kernel<D, T>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    const int q_blocks = (p.T + 15) / 16, q_total = p.B * q_blocks * ((p.Hq + kStageHeads - 1) / kStageHeads);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(q_total + sm_count * 8));
    cfg.blockDim = dim3(2 * D);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    // beside an append that was launched just before: the queries' blocks come first
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = after_append ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, p, q_out, k_out, v_out, Sk, q_blocks, q_total);
}

}  // namespace

cudaError_t launch_kv4_stage(const Kv4Params& p, void* q_out, void* k_out, void* v_out, int Sk, bool after_append,
                             int sm_count, cudaStream_t stream) {
    __half *q = static_cast<__half*>(q_out), *k = static_cast<__half*>(k_out), *v = static_cast<__half*>(v_out);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return p.act_dtype == kF16 ? launch_stage<D, __half>(p, q, k, v, Sk, after_append, sm_count, stream)
                                   : launch_stage<D, __nv_bfloat16>(p, q, k, v, Sk, after_append, sm_count, stream);
    };
    switch (p.D) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 96: return go(std::integral_constant<int, 96>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_kv4_nan_rows(const Kv4Params& p, int sm_count, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sm_count * 2);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_nan_rows_kernel, p);
}

}  // namespace b2a
