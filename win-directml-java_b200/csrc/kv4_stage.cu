// kv4_stage.cu -- operands of the tcgen05 attention kernel for chunks of prompts over the paged 4-bit
// cache (kv4.cuh): q rotated and converted to fp16, the visible cache rows as fp16.
//
// A chunk reads every key of its sequence once per 256 of its tokens and head, so the codes are turned
// into fp16 rows once, by one launch that is bound by HBM (0.625 D bytes in, 2 D out per row), and the
// tensor-core kernel streams those through TMA; per key and head that is far less than the chunk's
// own multiplications.  A value beyond fp16 becomes infinite and raises status bit 2, as bf16 inputs
// of the other entry points do.
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
// A block takes 16 tokens of a sequence and walks the heads two at a time; a thread holds channels
// 8 k .. + 7 and their partners D / 2 further.
template <int D, typename T>
__device__ __forceinline__ void stage_query(const Kv4Params& p, __half* out, int block, int blocks, unsigned char* smem) {
    constexpr int kHalf = D / 16, kThreads = 2 * D;  // chunk pairs of a row; 2 heads x 16 tokens x kHalf threads
    double2* const cs = reinterpret_cast<double2*>(smem);           // [16][D / 2]
    double* const part = reinterpret_cast<double*>(smem + 16 * (D / 2) * sizeof(double2));
    const int tid = threadIdx.x;
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
        for (int h = sub; h < p.Hq; h += 2) {
            uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (tok * p.Hq + h) * D + 8 * k);
            o[0] = o[kHalf] = make_uint4(v, v, v, v);
        }
    }
    if (t0 >= n) return;
    if (p.rope_mode != 0)
        for (int i = tid; i < 16 * (D / 2); i += kThreads) {
            double sn, c;
            sincos((double)(L + t0 + i / (D / 2)) * p.inv_freq[i % (D / 2)], &sn, &c);
            cs[i] = make_double2(c, sn);
        }
    __syncthreads();
    float top = 0.f;
    for (int h0 = 0; h0 < p.Hq; h0 += 2) {
        const int h = h0 + sub;
        const bool live = there && h < p.Hq;
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
        if (p.rope_mode != 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double2 c = cs[row * (D / 2) + 8 * k + i];
                const float a = x[i], e = y[i];
                if (p.rope_mode == 2) {
                    x[i] = (float)((double)a * c.x - (double)e * c.y);
                    y[i] = (float)((double)e * c.x + (double)a * c.y);
                } else {
                    x[i] = a * (float)c.x - e * (float)c.y;
                    y[i] = a * (float)c.y + e * (float)c.x;
                }
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
// One block of 16 positions of one kv head at a time, through shared memory: thread (row, chunk of 8
// channels) gathers its 8 codes' bytes.
template <int D>
__device__ __forceinline__ void stage_block(const Kv4Params& p, const uint8_t* src, int pos, int first, int end, __half* k_row0,
                                            __half* v_row0, int64_t row_stride, int* nan_flag, uint8_t* blk) {
    constexpr int kChunks = D / 8, kThreads = 2 * D, kGroups = D / 32;
    const int tid = threadIdx.x, row = tid / kChunks, k = tid - row * kChunks;
    if (src != nullptr)
        for (int i = tid; i < 20 * D / 16; i += kThreads)
            reinterpret_cast<uint4*>(blk)[i] = reinterpret_cast<const uint4*>(src)[i];
    __syncthreads();
    const bool there = src != nullptr && pos + row >= first && pos + row < end;
    const int y = k >> 2, x16 = (k >> 1) & 1, j = k & 1, g = row & 7, r = row >> 3;
#pragma unroll
    for (int is_v = 0; is_v < 2; ++is_v) {
        uint4 out = make_uint4(0, 0, 0, 0);
        if (there) {
            const uint8_t* code = blk + is_v * kv4_off_v(D);
            const float2 sz = __half22float2(
                reinterpret_cast<const __half2*>(code + kv4_off_kparam(D))[kv4_param(row, y, kGroups)]);
            float v[8];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = is_v ? ((y * 8 + i) * 4 + (g >> 1)) * 8 + x16 * 4 + 2 * (g & 1) + r
                                    : ((y * 8 + g) * 4 + (i >> 1)) * 8 + x16 * 4 + 2 * (i & 1) + r;
                v[i] = fmaf((float)(code[at] >> (4 * j) & 15), sz.x, sz.y);
                top = fmaxf(top, fabsf(v[i]));
            }
            if (top >= 65520.f) atomicOr(p.status, 4);
            if (is_v && !(sz.x == sz.x)) {  // held as NaN: zero here, and the rows that see it are marked later
                *nan_flag = 1;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
            }
            uint32_t* w = &out.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_half2(v[2 * i], v[2 * i + 1]);
        }
        *reinterpret_cast<uint4*>((is_v ? v_row0 : k_row0) + row * row_stride + 8 * k) = out;
    }
    __syncthreads();  // blk is reused
}

template <int D, typename T>
__global__ void __launch_bounds__(2 * D) kv4_stage_kernel(const __grid_constant__ Kv4Params p, __half* q_out, __half* k_out,
                                                          __half* v_out, int Sk, int* nan_flag, int q_blocks,
                                                          int q_total) {
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if ((int)blockIdx.x < q_total) {
        stage_query<D, T>(p, q_out, blockIdx.x, q_blocks, smem);
        return;
    }
    const int64_t row_stride = (int64_t)p.Hkv * D;
    int64_t i = blockIdx.x - q_total;
    const int64_t step = gridDim.x - q_total;
    for (int b = 0; b < p.B; ++b) {
        int L, n;
        if (!kv4_lens(p, b, L, n) || n == 0) continue;
        const int first = first_seen(p, L), end = L + n;
        const int blk0 = first / 128 * 8, blk1 = min((end + 127) / 128 * 8, Sk / kKv4Block);
        const int64_t count = (int64_t)(blk1 - blk0) * p.Hkv;
        for (; i < count; i += step) {
            const int blk = blk0 + (int)(i / p.Hkv), h = (int)(i % p.Hkv), pos = blk * kKv4Block;
            const bool seen = pos + kKv4Block > first && pos < end;
            const uint8_t* src = seen ? kv4_block_ptr(p, b, h, pos) : nullptr;
            if (seen && src == nullptr && threadIdx.x == 0) atomicOr(p.status, 16);
            const int64_t at = ((int64_t)b * Sk + pos) * row_stride + (int64_t)h * D;
            stage_block<D>(p, src, pos, first, end, k_out + at, v_out + at, row_stride, nan_flag, smem);
        }
        i -= count;
    }
}

// Rows that see a value group held as NaN, or a page that does not exist: their outputs become NaN
// (the group's channels; all of the row's).  Runs to its end only where the staging met one.
__global__ void __launch_bounds__(256) kv4_nan_rows_kernel(const __grid_constant__ Kv4Params p, const int* nan_flag) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (*nan_flag == 0 && (*p.status & 16) == 0) return;
    const int D = p.D, groups = D / 32;
    const int64_t rows = (int64_t)p.B * p.T * p.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < rows; row += (int64_t)gridDim.x * 8) {
        const int64_t tok = row / p.Hkv;
        const int kvh = (int)(row - tok * p.Hkv), b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
        int L, n;
        if (!kv4_lens(p, b, L, n) || t >= n) continue;
        const int first = p.window > 0 ? max(0, L + t - p.window + 1) : 0;
        unsigned hit = 0;  // bit per group, bit 31: a page is missing
        for (int key = first + lane; key <= L + t; key += 32) {
            const uint8_t* block = kv4_block_ptr(p, b, kvh, key);
            if (block == nullptr) {
                hit |= 1u << 31;
                continue;
            }
            const __half2* sz = reinterpret_cast<const __half2*>(block + kv4_off_vparam(D));
            for (int y = 0; y < groups; ++y)
                if (__hisnan(__low2half(sz[kv4_param(key % kKv4Block, y, groups)]))) hit |= 1u << y;
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
cudaError_t launch_stage(const Kv4Params& p, __half* q_out, __half* k_out, __half* v_out, int Sk, int* nan_flag,
                         int sm_count, cudaStream_t stream) {
    const size_t q_smem = 16 * (D / 2) * sizeof(double2) + 2 * D * sizeof(double);
    const size_t smem = q_smem > 20 * D ? q_smem : 20 * D;
    auto kern = kv4_stage_kernel<D, T>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    const int q_blocks = (p.T + 15) / 16, q_total = p.B * q_blocks;
    kern<<<q_total + sm_count * 8, 2 * D, smem, stream>>>(p, q_out, k_out, v_out, Sk, nan_flag, q_blocks, q_total);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_stage(const Kv4Params& p, void* q_out, void* k_out, void* v_out, int Sk, int* nan_flag,
                             int sm_count, cudaStream_t stream) {
    __half *q = static_cast<__half*>(q_out), *k = static_cast<__half*>(k_out), *v = static_cast<__half*>(v_out);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return p.act_dtype == kF16 ? launch_stage<D, __half>(p, q, k, v, Sk, nan_flag, sm_count, stream)
                                   : launch_stage<D, __nv_bfloat16>(p, q, k, v, Sk, nan_flag, sm_count, stream);
    };
    switch (p.D) {
        case 64: return go(std::integral_constant<int, 64>{});
        case 96: return go(std::integral_constant<int, 96>{});
        case 128: return go(std::integral_constant<int, 128>{});
        case 256: return go(std::integral_constant<int, 256>{});
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_kv4_nan_rows(const Kv4Params& p, const int* nan_flag, int sm_count, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sm_count * 2);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_nan_rows_kernel, p, nan_flag);
}

}  // namespace b2a
