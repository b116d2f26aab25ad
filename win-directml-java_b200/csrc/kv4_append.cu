// kv4_append.cu -- what comes before the attention over the paged 4-bit cache (kv4.cuh), one launch:
// new K/V rows into the cache (optional key norm, RoPE, group quantisation), the rows as the cache
// holds them for callers that want the prompt's own attention to see the same values, and the
// queries' norm, RoPE and layout as the warp MMA's B operand (kv4_attn.cu).
//
// kv4_prepare_kernel: the first CTAs plan the attention's work; each other one takes rows of one token
// (query heads, key heads, value heads), a warp one row at a time, and computes the token's sines and
// cosines once. It is all latency -- lengths, rows, page table, then a chain of double-precision
// steps -- so every read is requested before the first one is waited for, and the attention kernel
// is launched behind it early, to be resident when it ends.  Measured: 3.8 us for one sequence of a
// small model, 5.1 us for 64, 8.7 us for 256 sequences of head dim 256 with norms and double rotation.
// kv4_store_kernel: prompts. A CTA takes one block of 16 positions and walks kv heads; a thread holds
// 8 channels of four rows (16-byte loads), the block is assembled in shared memory and stored whole.
#include <algorithm>

#include "kv4.cuh"
#include "sm100.cuh"

namespace b2a {
namespace {

constexpr int kPrepWarps = 8;

// Query row r = token * G + head of the group, of (sequence b, kv head).  Its element 16 x + 8 j +
// 2 t + e of group y goes to half e of operand word (y, lane 4 (r % 8) + t, 2 x + j) of 8-row tile
// r / 8, as q 2^-E / 16^j with |q 2^-E| < 2^14 (the codes of channels with j = 1 enter the product
// 16 times larger); fp16 activations keep a second word with what the first rounding lost.
// q_sums: sum of the group's operand values 2^-4 (at most 2^15) per group, then scale log2(e) 2^(E + 24).
template <int D>
__device__ __forceinline__ void prepare_query(const Kv4Params& p, float (&x)[D / 32], const float (&wn)[D / 32],
                                              int64_t tok, int h, int t, const double2* cs, float* vec, int lane) {
    constexpr int kGroups = D / 32;
    const int tiles = (p.T * p.G + 7) / 8;
    const int kvh = h / p.G, r = t * p.G + h - kvh * p.G;
    const int64_t tile = (tok / p.T * p.Hkv + kvh) * tiles + (r >> 3);
    __half* frag = reinterpret_cast<__half*>(p.q_frag + tile * (kGroups * 32 * 2));
    float* sums = p.q_sums + tile * (kGroups + 1) * 8 + (r & 7);
    kv4_norm_rope<D>(x, p.q_norm_w != nullptr, wn, p.norm_eps, p.rope_mode, cs, vec, lane);
    float top = 0.f;
    bool fine = true;
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
    const float up = scalbnf(j ? 0.0625f : 1.f, -E);
    float used[kGroups];
#pragma unroll
    for (int y = 0; y < kGroups; ++y) {
        // -E is at most 149 + 13: in two steps, so that the factor stays finite
        const float v = !fine ? 0.f : (E < -100 ? scalbnf(x[y], -E) * (j ? 0.0625f : 1.f) : x[y] * up);
        const __half hi = __float2half_rn(v);
        const int at = (y * 32 * 4 + word) * 2 + (lane & 1);
        frag[at] = hi;
        used[y] = __half2float(hi);
        if (p.act_dtype == kF16) {
            const __half lo = __float2half_rn(v - used[y]);
            frag[kGroups * 32 * 4 * 2 + at] = lo;
            used[y] += __half2float(lo);
        }
        used[y] *= j ? 1.f : 0x1p-4f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int y = 0; y < kGroups; ++y) used[y] += __shfl_xor_sync(0xffffffffu, used[y], o);
    if (lane == 0) {
#pragma unroll
        for (int y = 0; y < kGroups; ++y) sums[y * 8] = used[y];
        sums[kGroups * 8] = fine ? scalbnf(p.scale * kLog2e, E + 24) : __int_as_float(0x7fc00000);
    }
}

template <int D>
__device__ __forceinline__ void append_row(const Kv4Params& p, float (&x)[D / 32], const float (&wn)[D / 32],
                                           int64_t tok, int kvh, bool is_v, int pos, uint8_t* block, const double2* cs,
                                           float* vec, int lane) {
    void* held = is_v ? p.v_held : p.k_held;
    const int64_t held_at = (tok * p.Hkv + kvh) * D;
    const int key = pos % kKv4Block;
    if (!is_v) kv4_norm_rope<D>(x, p.k_norm_w != nullptr, wn, p.norm_eps, p.rope_mode, cs, vec, lane);
    int code[D / 32];
    __half2 sz[D / 32];
    if (!kv4_quantise(x, code, sz) && lane == 0) atomicOr(p.status, 32);
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

// Spreads the attention's work over its CTAs, in one of two ways:
//  * pieces: every unit is cut into k near-equal pieces of at most P blocks, one piece per CTA.  P is
//    the smallest of three sizes, the guaranteed one, blocks / (CTAs - units), 7/8 and 13/16 of it,
//    that needs no more pieces than there are CTAs.
//  * ranges: the blocks of all units, each followed by `gap` that stand for the fixed cost of a piece,
//    form one stream; CTA c takes its c-th equal range, so it may meet several units.
// Pieces are taken where the largest costs no more than a range with a second piece's fixed cost.
// Every planning block sums the lengths itself and writes the pieces of its 256 CTAs.  The attention
// waits for the plan, so it is written for few steps: 32-bit arithmetic wherever the stream allows.
constexpr int kPrepThreads = kPrepWarps * 32;

__device__ __forceinline__ int seen_blocks(const Kv4Params& p, int L, int n, int& first) {
    first = p.window > 0 ? max(0, L - p.window + 1) / kKv4Block : 0;
    return n > 0 ? (L + n - 1) / kKv4Block + 1 - first : 0;
}
__device__ __forceinline__ int cuts_of(int blocks, float inv) { return max(1, (int)ceilf((float)blocks * inv - 1e-3f)); }

struct PlanShared {
    int prefix[kKv4MaxBatch + 1];  // per unit: pieces, or stream length, of the sequences before
    int ctx[kKv4MaxBatch], fresh[kKv4MaxBatch];
    int sums[6][kPrepWarps];
};

// One piece, with what its CTA's first one tells about the others.
__device__ __forceinline__ void put_piece(Kv4Piece* to, int b, int r, int L, int n, int blk0, int blk1, int n_split,
                                          int my_part, int part0, int part_step) {
    int4* w = reinterpret_cast<int4*>(to);
    w[0] = make_int4(b, r, L, n);
    w[1] = make_int4(blk0, blk1, n_split, my_part);
    *reinterpret_cast<int2*>(&to->part0) = make_int2(part0, part_step);
}

// The pieces of CTA c where the units' stream (prefix sums of weights w per unit, `total` in all) fits Int.
template <typename Int>
__device__ __forceinline__ void emit_pieces(const Kv4Params& p, const PlanShared& sh, int c, Int total, bool pieces) {
    const int n_cta = p.split.n_cta, per_seq = p.split.per_seq;
    const Int R = pieces ? 1 : max((Int)p.split.min_blocks, (total + n_cta - 1) / n_cta);
    Int pos = c * R;
    const Int end = min(total, pos + R);
    int made = 0, before = c;  // pieces so far, the last one's place
    while (pos < end) {
        int lo = 0, hi = p.B - 1;
        while (lo < hi) {  // the last sequence that starts at or before pos
            const int mid = (lo + hi + 1) >> 1;
            if ((Int)sh.prefix[mid] * per_seq <= pos) lo = mid;
            else hi = mid - 1;
        }
        const int b = lo, w = sh.prefix[b + 1] - sh.prefix[b], L = sh.ctx[b], n = sh.fresh[b];
        const Int seq_base = (Int)sh.prefix[b] * per_seq;
        int r = (int)((pos - seq_base) / w), first;
        const int nb = seen_blocks(p, L, n, first);
        if (pieces) {
            const int k = (int)(pos - seq_base) - r * w, each = nb / w, rest = nb - each * w;
            put_piece(p.plan + c, b, r, L, n, first + k * each + k * rest / w, first + (k + 1) * each + (k + 1) * rest / w,
                      w, c, c - k, 1);
            made = 1;
            break;
        }
        // pieces after the first lie from n_cta + their unit's number on: a unit that is not a CTA's
        // first begins inside that CTA's range, so no other CTA's range begins it
        for (; r < per_seq && pos < end; ++r) {
            const Int u_start = seq_base + (Int)r * w, u_end = u_start + nb;
            if (pos >= u_end) {  // in the unit's gap
                pos = u_start + w;
                continue;
            }
            const Int c0 = u_start / R, c1 = (u_end - 1) / R, stop = min(end, u_end);
            const int place = made == 0 ? c : n_cta + b * per_seq + r;
            if (made > 0) p.plan[before].more = place;
            before = place;
            // CTA c's slot is 2 c for the piece its range begins with, 2 c + 1 for one that begins later
            put_piece(p.plan + place, b, r, L, n, first + (int)(pos - u_start), first + (int)(stop - u_start),
                      (int)(c1 - c0) + 1, 2 * c + (pos == c * R ? 0 : 1), 2 * (int)c0 + (u_start != c0 * R ? 1 : 0), 2);
            ++made;
            pos = stop < end ? u_start + w : end;
        }
    }
    p.plan[c].count = made;
}

__device__ __noinline__ void plan_attention(const Kv4Params& p, PlanShared& sh, int block) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_cta = p.split.n_cta, per_seq = p.split.per_seq, gap = p.split.gap;
    auto all_warps = [&](int row) {
        int v = 0;
#pragma unroll
        for (int w = 0; w < kPrepWarps; ++w) v += sh.sums[row][w];
        return v;
    };
    int blocks = 0, seqs = 0, longest = 0, first;
    for (int b = tid; b < p.B; b += kPrepThreads) {
        int L, n;
        if (!kv4_lens(p, b, L, n)) n = 0;
        sh.ctx[b] = L;
        sh.fresh[b] = n;
        const int nb = seen_blocks(p, L, n, first);
        blocks += nb;
        seqs += nb > 0;
        longest = max(longest, nb);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    blocks = __reduce_add_sync(0xffffffffu, blocks);
    seqs = __reduce_add_sync(0xffffffffu, seqs);
    if (lane == 0) {
        sh.sums[3][warp] = blocks;
        sh.sums[4][warp] = seqs;
        sh.sums[5][warp] = longest;
    }
    __syncthreads();
    const float total_f = (float)all_warps(3) * (float)per_seq, units_f = (float)all_warps(4) * (float)per_seq;
    bool pieces = false;
    float inv_p = 0.f;
    if (units_f <= 0.875f * (float)n_cta) {
        const float most = __fdividef(total_f, (float)n_cta - units_f) + 1.f, least = (float)p.split.min_blocks;
        const float size[3] = {fmaxf(least, most), fmaxf(least, most * 0.875f), fmaxf(least, most * 0.8125f)};
        const float inv[3] = {__fdividef(1.f, size[0]), __fdividef(1.f, size[1]), __fdividef(1.f, size[2])};
        int count[3] = {0, 0, 0};
        for (int b = tid; b < p.B; b += kPrepThreads) {
            const int nb = seen_blocks(p, sh.ctx[b], sh.fresh[b], first);
#pragma unroll
            for (int k = 0; k < 3; ++k) count[k] += nb ? cuts_of(nb, inv[k]) : 0;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            count[k] = __reduce_add_sync(0xffffffffu, count[k]);
            if (lane == 0) sh.sums[k][warp] = count[k];
        }
        __syncthreads();
        longest = 0;
#pragma unroll
        for (int w = 0; w < kPrepWarps; ++w) longest = max(longest, sh.sums[5][w]);
        float best = 0.f;
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if ((float)all_warps(k) * (float)per_seq <= (float)n_cta) {
                best = fminf(size[k], (float)longest);
                inv_p = inv[k];
            }
        pieces = best > 0.f && best * (float)n_cta <= total_f + (float)(gap * n_cta);
    }
    // prefix sums, kPrepThreads sequences at a time
    auto weight = [&](int b) {
        const int nb = seen_blocks(p, sh.ctx[b], sh.fresh[b], first);
        return nb == 0 ? 0 : (pieces ? cuts_of(nb, inv_p) : nb + gap);
    };
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPrepThreads) {
        const int b = b0 + tid, w = b < p.B ? weight(b) : 0;
        int incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) sh.sums[0][warp] = incl;
        __syncthreads();
        int at = before;
        for (int k = 0; k < warp; ++k) at += sh.sums[0][k];
        if (b < p.B) sh.prefix[b] = at + incl - w;
        before += all_warps(0);
    }
    if (tid == 0) sh.prefix[p.B] = before;
    __syncthreads();
    const int c = block * kPrepThreads + tid;
    if (c >= n_cta) return;
    const long long total = (long long)before * per_seq;
    if (total + n_cta <= (long long)INT32_MAX) emit_pieces<int>(p, sh, c, (int)total, pieces);
    else emit_pieces<long long>(p, sh, c, total, pieces);
}

// Rows of a token: Hq queries (where p.q), Hkv keys and Hkv values (where `append`); after the
// planning blocks, block (token, chunk) takes rows [chunk * per, (chunk + 1) * per).
template <int D>
__global__ void __launch_bounds__(kPrepThreads) kv4_prepare_kernel(const __grid_constant__ Kv4Params p, int append,
                                                                   int chunks, int per, int plans) {
    constexpr int kGroups = D / 32;
    constexpr size_t kRowBytes = kPrepWarps * D * 4 + D / 2 * sizeof(double2);
    __shared__ __align__(16) unsigned char smem[kRowBytes > sizeof(PlanShared) ? kRowBytes : sizeof(PlanShared)];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x < plans) {
        plan_attention(p, *reinterpret_cast<PlanShared*>(smem), blockIdx.x);
        return;
    }
    double2* const cs = reinterpret_cast<double2*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* const vec = reinterpret_cast<float*>(smem + D / 2 * sizeof(double2)) + warp * D;
    const int block = blockIdx.x - plans;
    const int64_t tok = block / chunks;
    const int chunk = block - (int)tok * chunks;
    const int b = (int)(tok / p.T), t = (int)(tok - (int64_t)b * p.T);
    const int nq = p.q ? p.Hq : 0, rows = nq + (append ? 2 * p.Hkv : 0);
    const int end = min(rows, (chunk + 1) * per);
    int r = chunk * per + warp;
    // every read of the first row is requested before anything waits for one
    uint32_t raw[kGroups];
    float wn[kGroups];
    auto fetch = [&](int row) {
        const bool is_q = row < nq;
        const int i = row - nq;
        const void* src = is_q ? p.q : (i & 1) ? p.v_new : p.k_new;
        const int64_t at = is_q ? tok * p.q_stride + (int64_t)row * D : tok * p.kv_stride + (int64_t)(i >> 1) * D;
        const float* w = is_q ? p.q_norm_w : p.k_norm_w;
#pragma unroll
        for (int y = 0; y < kGroups; ++y) {
            raw[y] = load_raw(src, at + lane + 32 * y, p.act_dtype);
            wn[y] = w ? __ldg(w + lane + 32 * y) : 0.f;
        }
    };
    if (r < end) fetch(r);
    int L, n;
    const bool ok = kv4_lens(p, b, L, n);
    if (!ok && threadIdx.x == 0) atomicOr(p.status, 1);
    const bool there = t < n;
    // the new rows' block of kv head 0; the other heads' follow at one slab's distance
    uint8_t* const block0 = there && append ? kv4_block_ptr(p, b, 0, L + t) : nullptr;
    const int64_t slab = (int64_t)(p.page_size / kKv4Block) * kv4_block_bytes(D);
    if (there && p.rope_mode != 0 && threadIdx.x < D / 2) {
        double sn, c;
        sincos((double)(L + t) * p.inv_freq[threadIdx.x], &sn, &c);
        cs[threadIdx.x] = make_double2(c, sn);
    }
    __syncthreads();
    for (; r < end; r += kPrepWarps) {
        float x[kGroups], w[kGroups];
#pragma unroll
        for (int y = 0; y < kGroups; ++y) {
            x[y] = raw_to_float(raw[y], p.act_dtype);
            w[y] = wn[y];
        }
        if (r + kPrepWarps < end) fetch(r + kPrepWarps);
        const int i = r - nq;
        if (!there) {  // no such token: outputs are zero, or NaN where the lengths do not fit
            const float v = ok ? 0.f : __int_as_float(0x7fc00000);
            void* dst = i < 0 ? p.o : (i & 1) ? p.v_held : p.k_held;
            const int64_t at = i < 0 ? (tok * p.Hq + r) * D : (tok * p.Hkv + (i >> 1)) * D;
            if (dst)
                for (int d = lane; d < D; d += 32) store_from_float(dst, at + d, v, p.act_dtype);
        } else if (i < 0) {
            prepare_query<D>(p, x, w, tok, r, t, cs, vec, lane);
        } else {
            append_row<D>(p, x, w, tok, i >> 1, i & 1, L + t, block0 ? block0 + (i >> 1) * slab : nullptr, cs, vec,
                          lane);
        }
    }
}

// ------------------------------------------------------------------ prompts
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8], __half) {
    const uint32_t* e = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(e + i));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8], __nv_bfloat16) {
    const uint32_t* e = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(e[i] << 16);
        x[2 * i + 1] = __uint_as_float(e[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two floats at once, each rounded by itself: sm_100 issues the pair as one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// The low 16 bits' nibbles into the low nibbles of four bytes.
__device__ __forceinline__ uint32_t spread_nibbles(uint32_t x) {
    x = (x | x << 8) & 0x00FF00FFu;
    return (x | x << 4) & 0x0F0F0F0Fu;
}

// Threads of one (block of 16 positions, kv head): thread (q, k) holds channels 8 k .. + 7 of rows
// 2 q, 2 q + 1, 2 q + 8, 2 q + 9 -- the four keys whose codes share the V words -- so that whole 32-bit
// words are put together in registers.
template <int D>
struct StoreGeo {
    static constexpr int kChunks = D / 8;
    static constexpr int kPerHead = 4 * kChunks;              // threads: 32, 48, 64, 128
    static constexpr int kHeads = D <= 64 ? 8 : (D <= 128 ? 4 : 2);  // heads of a CTA side by side, at most
    static constexpr int kMinHeads = D == 96 ? 2 : 1;         // whole warps
    static constexpr int kMaxThreads = kHeads * kPerHead;
    // per SM: 64 (with norms 80) registers a thread at head dim 96, where 4 CTAs take 220 us instead of 193
    // (with norms 303 instead of 347); else 80.  With 2, 3, 4 and 5 CTAs, 8 x 4096 tokens with held rows, bf16
    // without / fp16 with norms: 16 heads of 64 80, 70, 67, 83 / 106, 95, 95, 112 us; 16 heads of 128 138, 127,
    // 125, 161 / 195, 181, 195, 224 us; 4 heads of 256 84, 75, 79, 98 / 112, 102, 110, 131 us
    static constexpr int ctas(bool norm) { return D == 96 ? (norm ? 4 : 5) : 3; }
    // an operand's 16 rows of the CTA's heads; the pad keeps rows two apart on other banks
    __host__ __device__ static constexpr int pitch(int heads) { return heads * D * 2 + (D == 96 ? 32 : 0); }
    __host__ __device__ static size_t stage_at(int heads) { return 2 * 16 * (size_t)pitch(heads); }
    __host__ __device__ static size_t cs_at(int heads) { return stage_at(heads) + heads * 20 * D; }
    __host__ __device__ static size_t part_at(int heads, int rope_mode) {
        return cs_at(heads) + (rope_mode == 0 ? 0 : 16 * (D / 2) * (rope_mode == 2 ? sizeof(double2) : sizeof(float2)));
    }
    // norms: 1 + weight as doubles, sums of squares [head][row][chunk], the rows' factors
    static size_t smem(int heads, int rope_mode, bool norm) {
        return part_at(heads, rope_mode) + (norm ? D * 8 + heads * 16 * (kChunks * 8 + 4) : 0);
    }
};

// The wait for a round's rows at place `failed` (0: K's, 1: V's) ran out: the parity of the last copy
// asked for at `place`.  K's place has been asked for the next round's rows, where there are `more`, by
// the time V's are waited for.
__host__ __device__ constexpr uint32_t pending_parity(int place, int failed, bool more, uint32_t parity) {
    return place < failed && more ? parity ^ 1u : parity;
}
static_assert(pending_parity(0, 1, true, 0) == 1 && pending_parity(0, 1, true, 1) == 0, "the next round's keys");
static_assert(pending_parity(0, 1, false, 1) == 1 && pending_parity(1, 1, true, 0) == 0, "this round's rows");
static_assert(pending_parity(0, 0, true, 1) == 1 && pending_parity(1, 0, true, 1) == 1, "this round's rows");

// A CTA takes one block of a sequence and heads h0 + group, + groups, ...  Its rows of K, then of V, come
// by bulk copies into a place each, asked for again as soon as the last ones are in registers, so that
// a round's rows travel while the round before is worked on.  A key chunk is rotated with its partner
// chunk D / 2 away, which the thread reads too.  The four threads of a group exchange minima and
// maxima so that each ends with one of the four rows, and computes that row's scale for all.
// Bound by issue and latency rather than by HBM: 8 x 4096 tokens of 32 heads of 96 with held rows (932
// MB) take 193 us back to back, 4.8 TB/s, and 201 to 209 us as one call behind an L2 flush.  What it took: packed float pairs (201 -> 159 million warp instructions),
// the rows' scales shared out (148 million, 261 -> 213 us), conflict-free angles (193 us).  Rows loaded
// into registers ahead instead of by bulk copies: 209 us; 4 and 6 CTAs per SM: 220 and 245 us.
// With key norms the sums of squares and the products with 1 + w are doubles as in b2a_decode: 8 x 4096
// tokens of 16 heads of 128, fp16 with held rows, take 180 us (without norms 123), and 210 us with the
// double-precision rotation (146); the rows' factors computed by every thread: 44 and 51 us more.  32 heads of
// 96, bf16: 322 us, where the partner chunk's norm is computed a second time in doubles.
template <int D, typename T, bool kNorm>
__global__ void __launch_bounds__(StoreGeo<D>::kMaxThreads, StoreGeo<D>::ctas(kNorm))
    kv4_store_kernel(const __grid_constant__ Kv4Params p, int blocks, int chunks, int per) {
    using Gm = StoreGeo<D>;
    constexpr int kChunks = Gm::kChunks, kGroups = D / 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a chunk's query staging may run beside this
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[2];  // K's place, V's place
    const int tid = threadIdx.x, groups = blockDim.x / Gm::kPerHead;
    const int group = tid / Gm::kPerHead, in_group = tid - group * Gm::kPerHead;
    const int q = in_group / kChunks, k = in_group - q * kChunks;
    const int pitch = Gm::pitch(groups);
    uint8_t* const stage = smem + Gm::stage_at(groups) + group * 20 * D;
    void* const cs = smem + Gm::cs_at(groups);  // [16][D / 2] (cos, sin)
    double* const weight = reinterpret_cast<double*>(smem + Gm::part_at(groups, p.rope_mode));
    double* const part = weight + D + group * 16 * kChunks;
    float* const factor = reinterpret_cast<float*>(weight + D + groups * 16 * kChunks) + group * 16;
    const uint32_t bar = smem_u32(full);
    if (p.nan_flag != nullptr && blockIdx.x == 0 && tid == 0) *p.nan_flag = 0;
    const int chunk = blockIdx.x % chunks;
    const int64_t bb = blockIdx.x / chunks;
    const int b = (int)(bb / blocks);
    int L, n;
    const bool ok = kv4_lens(p, b, L, n);
    if (!ok && tid == 0) atomicOr(p.status, 1);
    const int blk = L / kKv4Block + (int)(bb - (int64_t)b * blocks);
    const int t_first = blk * kKv4Block - L;  // token of the block's first position
    if (t_first >= p.T) return;
    const int h_begin = chunk * per, h_end = min(p.Hkv, h_begin + per);
    auto row_of = [&](int i) { return 2 * q + (i & 1) + 8 * (i >> 1); };  // i = e + 2 r
    const int64_t seq_tok = (int64_t)b * p.T;
    for (int i = 0; i < 4; ++i) {  // rows that do not exist
        const int t = t_first + row_of(i);
        if (t < n || t >= p.T) continue;
        const uint32_t v = ok ? 0u : 0x7fff7fffu;
        for (int h = h_begin + group; h < h_end; h += groups) {
            const int64_t at = ((seq_tok + t) * p.Hkv + h) * D + 8 * k;
            if (p.k_held) *reinterpret_cast<uint4*>(static_cast<T*>(p.k_held) + at) = make_uint4(v, v, v, v);
            if (p.v_held) *reinterpret_cast<uint4*>(static_cast<T*>(p.v_held) + at) = make_uint4(v, v, v, v);
        }
    }
    if (t_first >= n) return;  // nothing to store (the whole CTA)
    const int row_first = max(0, -t_first), row_end = min(kKv4Block, n - t_first);  // rows that exist
    const bool full_block = row_end - row_first == kKv4Block;
    auto request = [&](int is_v, int h0) {  // warp 0: a round's rows into their place
        const uint32_t bytes = min(groups, h_end - h0) * D * 2;
        if (tid == 0) mbar_expect_tx(bar + is_v * 8, (row_end - row_first) * bytes);
        __syncwarp();
        if (tid < row_first || tid >= row_end) return;
        const T* src = static_cast<const T*>(is_v ? p.v_new : p.k_new) + (seq_tok + t_first + tid) * p.kv_stride + (int64_t)h0 * D;
        bulk_load(smem_u32(smem) + (is_v * 16 + tid) * pitch, src, bytes, bar + is_v * 8);
    };
    if (tid < 32) {
        if (tid == 0) {
            mbar_init(bar, 1);
            mbar_init(bar + 8, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        request(0, h_begin);
        request(1, h_begin);
    }
    if (p.rope_mode != 0) kv4_block_angles<D>(p, blk * kKv4Block, cs, tid);
    if constexpr (kNorm)
        for (int i = tid; i < D; i += blockDim.x) weight[i] = __dadd_rn(1.0, (double)__ldg(p.k_norm_w + i));
    const bool upper = k >= kChunks / 2;
    const int k2 = upper ? k - kChunks / 2 : k + kChunks / 2, k_low = upper ? k2 : k;
    const int j = k & 1, x16 = (k >> 1) & 1, y = k >> 2;
    __syncthreads();

    uint32_t parity = 0;
    const unsigned char* const mine = smem + 2 * q * pitch + group * D * 2 + k * 16;
    for (int h0 = h_begin; h0 < h_end; h0 += groups, parity ^= 1) {
        const int h = h0 + group;
        const bool live = h < h_end;
        const float2 side = both(upper ? 1.f : -1.f);  // x cos -+ partner sin
        const int64_t held_at = ((seq_tok + t_first + 2 * q) * p.Hkv + h) * D + 8 * k;
        auto exists = [&](int i) { return live && row_of(i) >= row_first && row_of(i) < row_end; };
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
            uint8_t* const dst = stage + (is_v ? kv4_off_v(D) : 0);
            const unsigned char* const from = mine + is_v * 16 * pitch;
            auto row_at = [&](int i) { return from + ((i & 1) + 8 * (i >> 1)) * pitch; };
            const bool came = wait_bounded(bar + is_v * 8, parity);
            if (kNorm && !is_v) {
                for (int i = 0; i < 4; ++i) {
                    double ss = 0.0;
                    if (exists(i)) {
                        float x[8];
                        unpack8(*reinterpret_cast<const uint4*>(row_at(i)), x, T{});
#pragma unroll
                        for (int c = 0; c < 8; ++c) ss += (double)x[c] * (double)x[c];
                    }
                    part[row_of(i) * kChunks + k] = ss;
                }
                __syncthreads();
                if (in_group < 16) {  // a row's factor, once
                    double ss = 0.0;
                    for (int c = 0; c < kChunks; ++c) ss += part[in_group * kChunks + c];
                    factor[in_group] = (float)(1.0 / sqrt(__dadd_rn(ss / (double)D, (double)p.norm_eps)));
                }
                __syncthreads();
            }
            // ---- the rows' values, each thread's minima and maxima: NaN reaches `hi`, infinities both
            float2 x[4][4];
            float lo[4], hi[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row_of(i);
                float v[8];
                unpack8(exists(i) ? *reinterpret_cast<const uint4*>(row_at(i)) : make_uint4(0, 0, 0, 0), v, T{});
                if (!is_v) {
                    [[maybe_unused]] const float rms = kNorm ? factor[row] : 0.f;
                    if constexpr (kNorm) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) v[c] = (float)__dmul_rn((double)__fmul_rn(v[c], rms), weight[8 * k + c]);
                    }
                    if (p.rope_mode != 0) {
                        float z[8];
                        if constexpr (kNorm && D != 96) {  // the partner is a lane of this warp
#pragma unroll
                            for (int c = 0; c < 8; ++c) z[c] = __shfl_xor_sync(0xffffffffu, v[c], kChunks / 2);
                        } else {
                            unpack8(exists(i) ? *reinterpret_cast<const uint4*>(row_at(i) + 16 * (k2 - k)) : make_uint4(0, 0, 0, 0), z, T{});
                            if constexpr (kNorm) {
#pragma unroll
                                for (int c = 0; c < 8; ++c)
                                    z[c] = (float)__dmul_rn((double)__fmul_rn(z[c], rms), weight[8 * k2 + c]);
                            }
                        }
                        if (p.rope_mode == 2) {
                            const double2* a = static_cast<const double2*>(cs) + row * (D / 2) + k_low;
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                const double e = __dmul_rn((double)v[c], a[c * (D / 16)].x), f = __dmul_rn((double)z[c], a[c * (D / 16)].y);
                                v[c] = (float)(upper ? __dadd_rn(e, f) : __dsub_rn(e, f));
                            }
                        } else {
                            const float4* a = static_cast<const float4*>(cs) + row * (D / 4) + k_low;
#pragma unroll
                            for (int c = 0; c < 8; c += 2) {  // times +-1 is exact: the FMA adds or subtracts
                                const float4 ang = a[c / 2 * (D / 16)];
                                const float2 e = mul2(make_float2(v[c], v[c + 1]), make_float2(ang.x, ang.y));
                                const float2 f = mul2(make_float2(z[c], z[c + 1]), make_float2(ang.z, ang.w));
                                const float2 turned = fma2(f, side, e);
                                v[c] = turned.x;
                                v[c + 1] = turned.y;
                            }
                        }
                    }
                }
                lo[i] = min3(min3(v[0], v[1], v[2]), min3(v[3], v[4], v[5]), fminf(v[6], v[7]));
                hi[i] = max_nan(max_nan(v[0], v[1], v[2]), max_nan(v[3], v[4], v[5]), max_nan(v[6], v[7]));
#pragma unroll
                for (int c = 0; c < 4; ++c) x[i][c] = make_float2(v[2 * c], v[2 * c + 1]);
            }
            if (__syncthreads_or(!came)) {  // the wait ran out: nothing more is stored or asked for
                if (tid == 0) atomicOr(p.status, 8);
                for (int place = 0; place < 2; ++place)
                    mbar_drain(bar + place * 8, pending_parity(place, is_v, h0 + groups < h_end, parity));
                return;
            }
            if (tid < 32 && h0 + groups < h_end) request(is_v, h0 + groups);
            // ---- the groups' scales, one row of the four to each of a group's four threads
            uint32_t sz;
            float inv;
            bool outside;
            {
                const bool b1 = k & 2, b0 = k & 1;
                auto other = [&](float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); };
                const float lo0 = fminf(b1 ? lo[2] : lo[0], other(b1 ? lo[0] : lo[2], 2));
                const float lo1 = fminf(b1 ? lo[3] : lo[1], other(b1 ? lo[1] : lo[3], 2));
                const float hi0 = max_nan(b1 ? hi[2] : hi[0], other(b1 ? hi[0] : hi[2], 2));
                const float hi1 = max_nan(b1 ? hi[3] : hi[1], other(b1 ? hi[1] : hi[3], 2));
                const float low = fminf(b0 ? lo1 : lo0, other(b0 ? lo0 : lo1, 1));
                const float high = max_nan(b0 ? hi1 : hi0, other(b0 ? hi0 : hi1, 1));
                __half s = __float2half_rn(__fmul_rn(__fsub_rn(high, low), 1.0f / 15.0f)), z = __float2half_rn(low);
                const float sf = __half2float(s), zf = __half2float(z);
                const bool fine = isfinite(sf) && isfinite(zf);
                inv = sf > 0.f && fine ? __fdiv_rn(1.0f, sf) : 0.f;
                // codes leave 0 .. 15 only where the group's ends do (z and s are rounded: rarely; -0.5 goes to
                // the even 0, but 15.5 to the even 16); a group that is not finite counts as such, and its codes
                // become 0 with the others'
                outside = !(__fmul_rn(__fsub_rn(low, zf), inv) >= -0.5f && __fmul_rn(__fsub_rn(high, zf), inv) < 15.5f);
                if (!fine) {
                    s = z = __ushort_as_half(0x7fff);
                    if (exists(k & 3)) atomicOr(p.status, 32);
                }
                const __half2 both_sz = __halves2half2(s, z);
                sz = *reinterpret_cast<const uint32_t*>(&both_sz);
                reinterpret_cast<uint32_t*>(dst + kv4_off_kparam(D))[kv4_param(row_of(k & 3), y, kGroups)] = sz;
            }
            const bool clamp = __any_sync(0xffffffffu, outside);
            // ---- codes
            uint32_t bytes[4];  // by row, channels 4 j .. + 3 of the chunk pair (k, k ^ 1)
            float invs[4];
            float2 szs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = __shfl_sync(0xffffffffu, sz, i, 4);
                szs[i] = __half22float2(*reinterpret_cast<const __half2*>(&w));
                invs[i] = __shfl_sync(0xffffffffu, inv, i, 4);
#pragma unroll
                for (int c = 0; c < 4; ++c) x[i][c] = mul2(add2(x[i][c], both(-szs[i].y)), both(invs[i]));
            }
            if (clamp) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        x[i][c].x = fminf(fmaxf(x[i][c].x, 0.f), 15.f);
                        x[i][c].y = fminf(fmaxf(x[i][c].y, 0.f), 15.f);
                    }
            }
            T* const held = static_cast<T*>(is_v ? p.v_held : p.k_held);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // to the nearest whole number (ties to even) by 1.5 * 2^23
                float2 code[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) code[c] = add2(add2(x[i][c], both(12582912.f)), both(-12582912.f));
                if (held && exists(i)) {
                    uint4 out;
                    uint32_t* ow = &out.x;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float2 v = fma2(code[c], both(szs[i].x), both(szs[i].y));
                        ow[c] = Elem<T>::pack(v.x, v.y);
                    }
                    *reinterpret_cast<uint4*>(held + held_at + ((i & 1) + 8 * (i >> 1)) * p.Hkv * D) = out;
                }
                // four codes to 16 bits, exactly, as c0 + 16 c1 + 256 c2 + 4096 c3 (sums of whole numbers
                // below 2^24), beside 2^23, whose bits they then are
                uint32_t half[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float2 f = fma2(code[2 * c + 1], both(256.f), code[2 * c]);
                    half[c] = __float_as_uint(fmaf(f.y, 16.f, __fadd_rn(f.x, 8388608.f))) & 0xffffu;
                }
                // thread j keeps channels 4 j .. + 3 of both chunks of the pair
                const uint32_t swap = __shfl_xor_sync(0xffffffffu, j ? half[0] : half[1], 1);
                const uint32_t own = j ? half[1] : half[0];
                bytes[i] = spread_nibbles(j ? swap : own) | spread_nibbles(j ? own : swap) << 4;
            }
            uint32_t* const words = reinterpret_cast<uint32_t*>(dst) + y * 64 + x16;
            if (!is_v) {
                // K words (lane 4 g + t, x16): bytes (e, r) = channels 2 t + e of keys g + 8 r
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int g = 2 * q + e;
                    words[(4 * g + 2 * j) * 2] = __byte_perm(bytes[e], bytes[e + 2], 0x5140);
                    words[(4 * g + 2 * j + 1) * 2] = __byte_perm(bytes[e], bytes[e + 2], 0x7362);
                }
            } else {
                // V words (lane 4 g + t, x16): bytes (e, r) = channel g of keys 2 t + e + 8 r
                const uint32_t a = __byte_perm(bytes[0], bytes[2], 0x5140), c = __byte_perm(bytes[1], bytes[3], 0x5140);
                const uint32_t u = __byte_perm(bytes[0], bytes[2], 0x7362), v = __byte_perm(bytes[1], bytes[3], 0x7362);
                words[(4 * (4 * j + 0) + q) * 2] = __byte_perm(a, c, 0x5410);
                words[(4 * (4 * j + 1) + q) * 2] = __byte_perm(a, c, 0x7632);
                words[(4 * (4 * j + 2) + q) * 2] = __byte_perm(u, v, 0x5410);
                words[(4 * (4 * j + 3) + q) * 2] = __byte_perm(u, v, 0x7632);
            }
        }
        __syncthreads();
        if (live) {
            uint8_t* const block = kv4_block_ptr(p, b, h, blk * kKv4Block);
            if (block == nullptr) {
                if (in_group == 0) atomicOr(p.status, 16);
            } else if (full_block) {
                for (int i = in_group; i < 20 * D / 16; i += Gm::kPerHead)
                    reinterpret_cast<uint4*>(block)[i] = reinterpret_cast<const uint4*>(stage)[i];
            } else {
                // the rows that exist: their bytes of the codes, their params
                auto stored = [&](int key) { return key >= row_first && key < row_end; };
                for (int i = in_group; i < 16 * D; i += Gm::kPerHead) {
                    const bool is_v = i >= 8 * D;
                    const int a = is_v ? i - 8 * D : i;
                    const int r = a & 1, e = (a >> 1) & 1, t = (a >> 3) & 3, g = (a >> 5) & 7;
                    const int at = is_v ? kv4_off_v(D) + a : a;
                    if (stored(is_v ? 2 * t + e + 8 * r : g + 8 * r)) block[at] = stage[at];
                }
                for (int i = in_group; i < 2 * 16 * kGroups; i += Gm::kPerHead) {
                    const int w = i % (16 * kGroups), key = (w / kGroups >> 1) + 8 * (w / kGroups & 1);
                    const int at = (i < 16 * kGroups ? kv4_off_kparam(D) : kv4_off_vparam(D)) + 4 * w;
                    if (stored(key)) *reinterpret_cast<uint32_t*>(block + at) = *reinterpret_cast<const uint32_t*>(stage + at);
                }
            }
        }
        // (the next round writes to the stage behind its first barrier)
    }
}

template <int D, typename T>
cudaError_t launch_store(const Kv4Params& p, int sm_count, cudaStream_t stream) {
    using Gm = StoreGeo<D>;
    const int blocks = (p.T + 2 * kKv4Block - 2) / kKv4Block;  // blocks that T tokens can touch
    const int64_t ctas = (int64_t)p.B * blocks;
    const int heads = std::min(Gm::kHeads, p.Hkv), groups = (heads + Gm::kMinHeads - 1) / Gm::kMinHeads * Gm::kMinHeads;
    // a CTA computes its block's sines once for all its heads: heads are cut only where CTAs are few
    const int rounds = (p.Hkv + groups - 1) / groups;
    const int want = (int)std::min<int64_t>(rounds, std::max<int64_t>(1, 4 * sm_count / ctas));
    const int per = (rounds + want - 1) / want * groups, chunks = (p.Hkv + per - 1) / per;
    const size_t smem = Gm::smem(groups, p.rope_mode, p.k_norm_w != nullptr);
    auto kern = p.k_norm_w ? kv4_store_kernel<D, T, true> : kv4_store_kernel<D, T, false>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    kern<<<(unsigned)(ctas * chunks), groups * Gm::kPerHead, smem, stream>>>(p, blocks, chunks, per);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_prepare(const Kv4Params& p, int sm_count, cudaStream_t stream) {
    int append = p.k_new ? 1 : 0;
    if (append && p.T >= kKv4StoreTokens) {
        const cudaError_t e = p.act_dtype == kF16 ? launch_store<D, __half>(p, sm_count, stream)
                                                  : launch_store<D, __nv_bfloat16>(p, sm_count, stream);
        if (e != cudaSuccess || !p.q) return e;
        append = 0;
    }
    // a row per warp while that leaves the GPU room, else longer runs of rows that share their sines
    const int64_t tokens = (int64_t)p.B * p.T;
    const int plans = p.q ? (p.split.n_cta + kPrepThreads - 1) / kPrepThreads : 0;
    const int rows = (p.q ? p.Hq : 0) + (append ? 2 * p.Hkv : 0);
    const int most = (rows + kPrepWarps - 1) / kPrepWarps;
    const int want = (int)std::max<int64_t>(1, std::min<int64_t>(most, 8 * sm_count / tokens));
    const int per = (rows + want - 1) / want, chunks = (rows + per - 1) / per;
    kv4_prepare_kernel<D><<<(unsigned)(plans + tokens * chunks), kPrepThreads, 0, stream>>>(p, append, chunks, per, plans);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_prepare(const Kv4Params& p, int sm_count, cudaStream_t stream) {
    switch (p.D) {
        case 64: return launch_prepare<64>(p, sm_count, stream);
        case 96: return launch_prepare<96>(p, sm_count, stream);
        case 128: return launch_prepare<128>(p, sm_count, stream);
        case 256: return launch_prepare<256>(p, sm_count, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace b2a
