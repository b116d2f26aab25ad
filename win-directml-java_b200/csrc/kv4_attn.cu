// kv4_attn.cu -- attention of the new tokens of each sequence over the paged 4-bit cache (kv4.cuh).
//
// With codes c, scales s and minima z of group y (32 channels), and keys j <= the query's position,
//     S_j = scale * sum_y ( s_yj * sum_{i in y} q_i c_ij  +  z_yj * sum_{i in y} q_i )
//     o_i = ( sum_j (P_j s_yj) c_ij  +  sum_j P_j z_yj ) / sum_j P_j,   P_j = exp(S_j - max)
// so both products run on the codes themselves: the scale of a key's group multiplies the group's
// score (32 bits) or the probability before it is rounded for the second product, and the minima
// enter through sums.  No value is ever dequantised.
//
// Bound.  A key costs 1.25 D bytes per kv head for G query heads, about 3.2 G flop per byte: HBM,
// provided the instructions per key stay few.  Per 16 keys and 32 channels a warp spends ten integer
// instructions on 2 x 512 codes (two masks and a shift per word; the block layout is the MMA's own
// operand order) and four MMAs of 16 keys (K) or 16 channels (V^T) x 8 query rows.
//
// Work split.  A unit is (sequence, kv head, tile of 8 * kTiles query rows); a query row is (token,
// head of the group), so one cache byte serves every head of its group and every token of a draft.
// The blocks of 16 keys of all units form one stream and every CTA takes an equal range of it
// (stream-K); the pieces of a cut unit meet through partial slots (m, l, O) that the last one to
// finish joins.  Inside a piece each warp walks its own blocks with its own ring of bulk copies: one
// copy of 20 D bytes is a block, its address comes from page-table entries fetched 32 blocks at a
// time, and the warps meet only at the end of the piece.
//
// Softmax.  The running maximum moves only when a score exceeds it by more than 2^8 (in base 2: by
// 8), so a block normally costs no reduction across lanes: probabilities are at most 2^8 and sums
// are exact enough in fp32 whatever the reference point.  The same slow path moves the power of two
// 2^vexp that keeps P s within fp16: s 2^-vexp is at most 2^7, which leaves 2^21 of range below the
// largest weight before fp16 subnormals begin.
#include <mutex>
#include <type_traits>

#include "kv4.cuh"
#include "sm100.cuh"

namespace b2a {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLowest = -1e37f;   // a running maximum before any key: finite, so differences are
constexpr float kSlack = 8.f;       // how far a score may exceed the running maximum (log2)

template <int D, int kTiles, bool kSplitQ>
struct AttnGeo {
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kBlockBytes = kv4_block_bytes(D);
    static constexpr int kStages = D <= 128 ? 4 : 3;
    static constexpr int kRows = 8 * kTiles;
    static constexpr int kCtas = D * kTiles <= 64 ? 4 : (D * kTiles <= 128 ? 3 : 2);  // per SM: the registers' bound
    // fixed cost of a piece in blocks of streaming time, charged to every unit by the split
    static constexpr int kGapBlocks = D <= 64 ? 16 : (D <= 128 ? 8 : 4);
    static constexpr int kMinBlocks = 8;  // smallest range of a CTA: two blocks per warp
    static constexpr size_t kRingBytes = size_t(kWarps) * kStages * kBlockBytes;
    static constexpr size_t kMergeBytes = size_t(kWarps) * kRows * D * 4;
    static constexpr size_t a128(size_t x) { return (x + 127) / 128 * 128; }
    static constexpr size_t oBars = a128(kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes);
    static constexpr size_t oMl = oBars + kWarps * kStages * 8;
    static constexpr size_t oMisc = a128(oMl + size_t(kWarps) * kRows * 2 * 4);
    // q operand words in shared memory: the second (fp16) words always, the first ones where the
    // accumulators leave no registers for them
    static constexpr bool kQShared = D * kTiles >= 256;
    static constexpr size_t kQWords = size_t(kTiles) * kGroups * 32 * 16;
    static constexpr size_t oQ = oMisc + 128;
    static constexpr size_t oQlo = oQ + (kQShared ? kQWords : 0);
    static constexpr size_t oPrefix = oQlo + (kSplitQ ? kQWords : 0);
    static size_t total(int B) { return oPrefix + size_t(3 * B + 1) * 4; }
};

// The blocks of 16 positions that some new token of a sequence sees: how many, and the first.
__device__ __forceinline__ int seq_blocks(const Kv4Params& p, int L, int n, int& lo) {
    lo = p.window > 0 ? max(0, L - p.window + 1) / kKv4Block : 0;
    return n > 0 ? (L + n - 1) / kKv4Block + 1 - lo : 0;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// Bounded wait; false after kWaitNs.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity) {
    if (mbar_test(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (uint32_t i = 1;; ++i) {
        if (mbar_test(bar, parity)) return true;
        if ((i & 255u) == 0 && global_ns() - t0 > kWaitNs) return false;
    }
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t x;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(a));
    return x;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 x;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(a));
    return x;
}
// The A operand of one 16 x 16 tile of codes.
__device__ __forceinline__ void code_frag(uint32_t (&a)[4], uint32_t w) {
    const uint32_t h = w >> 8;
    a[0] = w & 0x000F000Fu;
    a[1] = h & 0x000F000Fu;
    a[2] = w & 0x00F000F0u;
    a[3] = h & 0x00F000F0u;
}
__device__ __forceinline__ float2 half2_f(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }

template <int D, int kTiles, bool kSplitQ>
__global__ void __launch_bounds__(kThreads, AttnGeo<D, kTiles, kSplitQ>::kCtas) kv4_attn_kernel(const __grid_constant__ Kv4Params p) {
    using Gm = AttnGeo<D, kTiles, kSplitQ>;
    constexpr int kGroups = Gm::kGroups, kStages = Gm::kStages, kRows = Gm::kRows;
    extern __shared__ __align__(128) unsigned char smem[];
    float* merge_s = reinterpret_cast<float*>(smem);
    float* ml_s = reinterpret_cast<float*>(smem + Gm::oMl);
    int* misc = reinterpret_cast<int*>(smem + Gm::oMisc);
    int* prefix = reinterpret_cast<int*>(smem + Gm::oPrefix);
    int* ctx_s = prefix + p.B + 1;  // cached and new tokens per sequence, 0 and 0 where they do not fit
    int* new_s = ctx_s + p.B;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kStages * Gm::kBlockBytes;
    const uint32_t bars = smem_u32(smem + Gm::oBars) + warp * kStages * 8;

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) mbar_init(bars + s * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }

    // ---------------------------------------------------------------- plan
    // prefix[b]: stream length (visible blocks and the gap) of the sequences before b, per unit
    {
        const int per = (p.B + kThreads - 1) / kThreads;
        const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
        int run = 0;
        for (int b = b0; b < b1; ++b) {
            int L, n, lo;
            if (!kv4_lens(p, b, L, n)) n = 0;
            ctx_s[b] = L;
            new_s[b] = n;
            const int nb = seq_blocks(p, L, n, lo);
            run += nb ? nb + Gm::kGapBlocks : 0;
        }
        int incl = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) misc[warp] = incl;
        __syncthreads();
        int acc = incl - run;
        for (int w = 0; w < warp; ++w) acc += misc[w];
        for (int b = b0; b < b1; ++b) {
            prefix[b] = acc;
            int lo;
            const int nb = seq_blocks(p, ctx_s[b], new_s[b], lo);
            acc += nb ? nb + Gm::kGapBlocks : 0;
        }
        if (tid == kThreads - 1) prefix[p.B] = acc;
        __syncthreads();
    }
    const int row_tiles = (p.T * p.G + kRows - 1) / kRows;
    const int per_seq = p.Hkv * row_tiles;
    const long long total = (long long)prefix[p.B] * per_seq;
    const long long R = max((long long)Gm::kMinBlocks, (total + gridDim.x - 1) / gridDim.x);
    const int q_tiles = (p.T * p.G + 7) / 8;  // tiles of 8 rows that the preparation laid out
    bool dep_done = false, dead = false;  // dead: a copy of this warp did not arrive in time
    uint32_t it = 0;  // blocks this warp has consumed since the launch began: ring slot and parity

    for (long long pos = (long long)blockIdx.x * R, end = min(total, pos + R); pos < end;) {
        int lo_b = 0, hi_b = p.B - 1;
        while (lo_b < hi_b) {  // the last sequence that starts at or before pos
            const int mid = (lo_b + hi_b + 1) >> 1;
            if ((long long)prefix[mid] * per_seq <= pos) lo_b = mid;
            else hi_b = mid - 1;
        }
        const int b = lo_b;
        const int L = ctx_s[b], n = new_s[b];
        int first_blk;
        const int n_blk = seq_blocks(p, L, n, first_blk);
        const int n_v = n_blk + Gm::kGapBlocks;
        const long long seq_base = (long long)prefix[b] * per_seq;
        const int r = (int)((pos - seq_base) / n_v);
        const long long u_start = seq_base + (long long)r * n_v, u_end = u_start + n_blk;
        if (pos >= u_end) {
            pos = u_start + n_v;
            continue;
        }
        const long long piece_end = min(end, u_end);
        const int kvh = r / row_tiles, rt = r - kvh * row_tiles;
        // tokens of this tile's rows, and the blocks of the piece that they see
        const int t_lo = rt * kRows / p.G, t_hi = min(n - 1, (rt * kRows + kRows - 1) / p.G);
        const int key_lo = p.window > 0 ? max(0, L + t_lo - p.window + 1) : 0, key_hi = L + t_hi;
        const int blk0 = max(first_blk + (int)(pos - u_start), key_lo / kKv4Block);
        const int blk1 = t_lo <= t_hi ? min(first_blk + (int)(piece_end - u_start), key_hi / kKv4Block + 1) : blk0;
        const long long c0 = u_start / R, c1 = (u_end - 1) / R;
        const int n_split = (int)(c1 - c0) + 1;
        const int my_slot = 2 * blockIdx.x + (pos == (long long)blockIdx.x * R ? 0 : 1);
        const int unit = b * per_seq + r;
        pos = piece_end;

        // ------------------------------------------------------------ this warp's blocks
        const int bpp = p.page_size / kKv4Block;
        const int my_n = max(0, (blk1 - blk0 - warp + kWarps - 1) / kWarps);
        bool bad = false;
        auto entry = [&](int i) -> int64_t {  // byte offset of the warp's i-th block, per lane
            if (i >= my_n) return 0;
            const int blk = blk0 + warp + kWarps * i;
            const int slot = blk / bpp, in = blk - slot * bpp;
            const int page = p.page_table[(int64_t)b * p.max_pages + slot];
            if (page < 0 || page >= p.num_pages) {
                bad = true;
                return 0;
            }
            return (((int64_t)page * p.Hkv + kvh) * bpp + in) * Gm::kBlockBytes;
        };
        int64_t cur = entry(lane), nxt = entry(32 + lane);
        auto issue = [&](int i) {  // request the warp's i-th block
            if (i > 0 && (i & 31) == 0) {
                cur = nxt;
                nxt = entry(i + 32 + lane);
            }
            const int64_t off = __shfl_sync(0xffffffffu, cur, i & 31);
            if (lane == 0) {
                const uint32_t s = (it + i) % kStages;
                mbar_expect_tx(bars + s * 8, Gm::kBlockBytes);
                bulk_load(ring + s * Gm::kBlockBytes, p.pages + off, Gm::kBlockBytes, bars + s * 8);
            }
        };
        // Blocks before the first new token's are as the kernel before the preparation left them, so
        // the first ones are requested while the preparation kernel still runs.
        int issued = 0;
        auto fill = [&](int upto) {
            while (!dead && issued < min(upto, my_n)) issue(issued++);
        };
        if (!dep_done) {
            const int old_blk = L / kKv4Block;  // blocks below hold no new token
            int ready = 0;
            while (ready < min(kStages, my_n) && blk0 + warp + kWarps * ready < old_blk) ++ready;
            fill(ready);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            dep_done = true;
        }
        fill(kStages);

        // ------------------------------------------------------------ q operands
        // B operand words of 8-row tile i: per group four words a lane (two 16-channel steps)
        uint32_t qf[kTiles][kGroups][4];
        uint4* const q_s = reinterpret_cast<uint4*>(smem + Gm::oQ) + lane;
        uint4* const qlo_s = reinterpret_cast<uint4*>(smem + Gm::oQlo) + lane;
        float qs[kTiles][kGroups][2], f0[kTiles], f1[kTiles];
        int lim0[kTiles], lim1[kTiles];  // last visible key of rows 2t and 2t + 1
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const int tile8 = rt * kTiles + i;
            const int64_t at = ((int64_t)b * p.Hkv + kvh) * q_tiles + min(tile8, q_tiles - 1);
            const uint4* src = p.q_frag + at * (kGroups * 32 * 2);
            const float* sums = p.q_sums + at * (kGroups + 1) * 8;
#pragma unroll
            for (int y = 0; y < kGroups; ++y) {
                const int word = (i * kGroups + y) * 32;
                if constexpr (!Gm::kQShared) {
                    const uint4 w = src[y * 32 + lane];
                    qf[i][y][0] = w.x, qf[i][y][1] = w.y, qf[i][y][2] = w.z, qf[i][y][3] = w.w;
                } else if (warp == y % kWarps) {
                    q_s[word] = src[y * 32 + lane];
                }
                if (kSplitQ && warp == y % kWarps) qlo_s[word] = src[(kGroups + y) * 32 + lane];
                const float2 s = *reinterpret_cast<const float2*>(sums + y * 8 + 2 * t4);
                qs[i][y][0] = s.x, qs[i][y][1] = s.y;
            }
            const float2 f = *reinterpret_cast<const float2*>(sums + kGroups * 8 + 2 * t4);
            f0[i] = f.x, f1[i] = f.y;
            const int r0 = tile8 * 8 + 2 * t4, tok0 = r0 / p.G, tok1 = (r0 + 1) / p.G;
            lim0[i] = tok0 < n ? L + tok0 : -1;
            lim1[i] = tok1 < n ? L + tok1 : -1;
        }
        if (kSplitQ || Gm::kQShared) __syncthreads();
        // keys [all_lo, all_hi] are visible to every present row of the tile (what an absent row
        // computes is not used, and its q operand is zero)
        const int all_hi = L + t_lo;
        const int all_lo = p.window > 0 ? L + t_hi - p.window + 1 : 0;

        // ------------------------------------------------------------ main loop
        float acc[kTiles][D / 16][4], oz[kTiles][kGroups][2];
        float m0[kTiles], m1[kTiles], l0[kTiles], l1[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) acc[i][k][0] = acc[i][k][1] = acc[i][k][2] = acc[i][k][3] = 0.f;
#pragma unroll
            for (int y = 0; y < kGroups; ++y) oz[i][y][0] = oz[i][y][1] = 0.f;
            m0[i] = m1[i] = kLowest;
            l0[i] = l1[i] = 0.f;
        }
        int vexp = -40;          // P s is multiplied by 2^-vexp
        float vinv = 0x1p40f;    // 2^-vexp

        for (int i = 0; i < my_n && !dead; ++i) {
            const uint32_t slot = (it + i) % kStages;
            if (!wait_bounded(bars + slot * 8, ((it + i) / kStages) & 1)) {
                // report, wait for the others in flight and ask for no more; the outputs are NaN
                if (lane == 0) atomicOr(p.status, 8);
                dead = true;
                for (int k = i + 1; k < issued; ++k)
                    if (!wait_bounded(bars + (it + k) % kStages * 8, ((it + k) / kStages) & 1)) break;
                break;
            }
            const uint32_t base = ring + slot * Gm::kBlockBytes;
            const int key = (blk0 + warp + kWarps * i) * kKv4Block;
            // scores, log2 units, relative to the running maximum
            float s[kTiles][4];
#pragma unroll
            for (int j = 0; j < kTiles; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
            const uint32_t kp = base + kv4_off_kparam(D) + g * (2 * kGroups * 4);
#pragma unroll
            for (int y = 0; y < kGroups; ++y) {
                const uint2 w = lds64(base + y * 256 + lane * 8);
                const float2 pa = half2_f(lds32(kp + y * 4)), pb = half2_f(lds32(kp + (kGroups + y) * 4));
                uint32_t a[4], c[4];
                code_frag(a, w.x);
                code_frag(c, w.y);
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (Gm::kQShared) {
                        const uint4 q = q_s[(j * kGroups + y) * 32];
                        Mma<__half>::run(d, a, q.x, q.y);
                        Mma<__half>::run(d, c, q.z, q.w);
                    } else {
                        Mma<__half>::run(d, a, qf[j][y][0], qf[j][y][1]);
                        Mma<__half>::run(d, c, qf[j][y][2], qf[j][y][3]);
                    }
                    if constexpr (kSplitQ) {
                        const uint4 q = qlo_s[(j * kGroups + y) * 32];
                        Mma<__half>::run(d, a, q.x, q.y);
                        Mma<__half>::run(d, c, q.z, q.w);
                    }
                    s[j][0] += pa.x * d[0] + pa.y * qs[j][y][0];
                    s[j][1] += pa.x * d[1] + pa.y * qs[j][y][1];
                    s[j][2] += pb.x * d[2] + pb.y * qs[j][y][0];
                    s[j][3] += pb.x * d[3] + pb.y * qs[j][y][1];
                }
            }
            const bool whole = key + kKv4Block - 1 <= all_hi && key >= all_lo;
            const int ka = key + g, kb = ka + 8;
            bool seen_a = true, seen_b = true;  // by some row: the block's stale rows hold anything
            float over = -INFINITY;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
                s[j][0] *= f0[j];
                s[j][1] *= f1[j];
                s[j][2] *= f0[j];
                s[j][3] *= f1[j];
                if (!whole) {
                    const int w0 = p.window > 0 ? lim0[j] - p.window : -1, w1 = p.window > 0 ? lim1[j] - p.window : -1;
                    if (ka > lim0[j] || ka <= w0) s[j][0] = -INFINITY;
                    if (ka > lim1[j] || ka <= w1) s[j][1] = -INFINITY;
                    if (kb > lim0[j] || kb <= w0) s[j][2] = -INFINITY;
                    if (kb > lim1[j] || kb <= w1) s[j][3] = -INFINITY;
                }
                over = fmaxf(over, fmaxf(fmaxf(s[j][0], s[j][2]) - m0[j], fmaxf(s[j][1], s[j][3]) - m1[j]));
            }
            if (!whole) {
                seen_a = ka <= key_hi && ka >= key_lo;
                seen_b = kb <= key_hi && kb >= key_lo;
            }
            // this lane's keys' value params: scales 2^-vexp and minima
            float va[kGroups], vb[kGroups], za[kGroups], zb[kGroups], top = 0.f;
            const uint32_t vp = base + kv4_off_vparam(D) + g * (2 * kGroups * 4);
#pragma unroll
            for (int y = 0; y < kGroups; ++y) {
                const float2 pa = half2_f(lds32(vp + y * 4)), pb = half2_f(lds32(vp + (kGroups + y) * 4));
                va[y] = seen_a ? pa.x : 0.f;
                vb[y] = seen_b ? pb.x : 0.f;
                za[y] = seen_a ? pa.y : 0.f;
                zb[y] = seen_b ? pb.y : 0.f;
                top = fmaxf(top, fmaxf(va[y], vb[y]));
            }
            if (__any_sync(0xffffffffu, over > kSlack || top * vinv > 128.f)) {
                // move the reference points: the maxima of the rows and the power of two of P s
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                float vscale = 1.f;
                if (top * vinv > 128.f) {
                    const int e = ilogbf(top) - 6;  // top 2^-e in [2^6, 2^7)
                    vscale = exp2f((float)(vexp - e));
                    vexp = e;
                    vinv = exp2f((float)-e);
                }
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    float a0 = fmaxf(s[j][0], s[j][2]), a1 = fmaxf(s[j][1], s[j][3]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, o));
                        a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, o));
                    }
                    a0 = fmaxf(a0, m0[j]);
                    a1 = fmaxf(a1, m1[j]);
                    const float k0 = fast_exp2(m0[j] - a0), k1 = fast_exp2(m1[j] - a1);
                    m0[j] = a0;
                    m1[j] = a1;
                    l0[j] *= k0;
                    l1[j] *= k1;
#pragma unroll
                    for (int y = 0; y < kGroups; ++y) {
                        oz[j][y][0] *= k0;
                        oz[j][y][1] *= k1;
                    }
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        acc[j][k][0] *= k0 * vscale;
                        acc[j][k][1] *= k1 * vscale;
                        acc[j][k][2] *= k0 * vscale;
                        acc[j][k][3] *= k1 * vscale;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
                s[j][0] = fast_exp2(s[j][0] - m0[j]);
                s[j][1] = fast_exp2(s[j][1] - m1[j]);
                s[j][2] = fast_exp2(s[j][2] - m0[j]);
                s[j][3] = fast_exp2(s[j][3] - m1[j]);
                l0[j] += s[j][0] + s[j][2];
                l1[j] += s[j][1] + s[j][3];
            }
            // kSel: some rows of the tile do not see some of the block's keys, whose params may be NaN:
            // a probability of zero then counts as nothing, not as 0 * NaN
            auto values = [&](auto sel) {
                auto times = [](float pr, float x) { return decltype(sel)::value && pr == 0.f ? 0.f : pr * x; };
#pragma unroll
                for (int y = 0; y < kGroups; ++y) {
                    const uint2 w = lds64(base + kv4_off_v(D) + y * 256 + lane * 8);
                    uint32_t a[4], c[4];
                    code_frag(a, w.x);
                    code_frag(c, w.y);
                    // V^T's tile has the channel as its row: registers in the order (channel g, keys 2t),
                    // (g + 8, 2t), (g, 2t + 8), (g + 8, 2t + 8)
                    const uint32_t av[4] = {a[0], a[2], a[1], a[3]}, cv[4] = {c[0], c[2], c[1], c[3]};
                    const float fa = va[y] * vinv, fb = vb[y] * vinv;
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        oz[j][y][0] += times(s[j][0], za[y]) + times(s[j][2], zb[y]);
                        oz[j][y][1] += times(s[j][1], za[y]) + times(s[j][3], zb[y]);
                        const uint32_t p0 = movmatrix_trans(pack_half2(times(s[j][0], fa), times(s[j][1], fa)));
                        const uint32_t p1 = movmatrix_trans(pack_half2(times(s[j][2], fb), times(s[j][3], fb)));
                        Mma<__half>::run(acc[j][2 * y], av, p0, p1);
                        Mma<__half>::run(acc[j][2 * y + 1], cv, p0, p1);
                    }
                }
            };
            if (!whole && p.T > 1) values(std::true_type{});
            else values(std::false_type{});
            __syncwarp();  // every lane has read the slot
            fill(issued + 1);
        }
        it += my_n;
        bad = __any_sync(0xffffffffu, bad);
        if (bad && lane == 0) atomicOr(p.status, 16);
        __syncthreads();  // all rings idle: merge_s may alias them

        // ------------------------------------------------------------ epilogue
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l0[j] += __shfl_xor_sync(0xffffffffu, l0[j], o);
                l1[j] += __shfl_xor_sync(0xffffffffu, l1[j], o);
#pragma unroll
                for (int y = 0; y < kGroups; ++y) {
                    oz[j][y][0] += __shfl_xor_sync(0xffffffffu, oz[j][y][0], o);
                    oz[j][y][1] += __shfl_xor_sync(0xffffffffu, oz[j][y][1], o);
                }
            }
            // unnormalised O in [d][row] pairs, the row index XOR-swizzled by (d >> 2) & 7 as in
            // decode_tc.cu: pair stores and reads along d are free of bank conflicts
            float* mw = merge_s + (warp * kTiles + j) * 8 * D;
            const float lo = exp2f((float)(vexp + 24)), hi = exp2f((float)(vexp + 20));
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 16 * k + g + 8 * h, x = (d >> 2) & 7;
                    const float u = acc[j][k][2 * h] * (h ? hi : lo) + oz[j][k / 2][0];
                    const float v = acc[j][k][2 * h + 1] * (h ? hi : lo) + oz[j][k / 2][1];
                    *reinterpret_cast<float2*>(mw + d * 8 + ((2 * t4) ^ (x & 6))) =
                        (x & 1) ? make_float2(v, u) : make_float2(u, v);
                }
            }
            if (g == 0) {
                const bool nan = bad || dead;
                float* ml = ml_s + ((warp * kTiles + j) * 8 + 2 * t4) * 2;
                ml[0] = m0[j];
                ml[1] = nan ? __int_as_float(0x7fc00000) : l0[j];
                ml[2] = m1[j];
                ml[3] = nan ? __int_as_float(0x7fc00000) : l1[j];
            }
        }
        __syncthreads();
        float* slot = p.partials + (int64_t)my_slot * kRows * (D + 2);
        if (tid < kRows) {
            float M = kLowest, l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml_s[(w * kRows + tid) * 2]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                float* ml = ml_s + (w * kRows + tid) * 2;
                const float x = fast_exp2(ml[0] - M);
                l += x * ml[1];
                ml[0] = x;
            }
            ml_s[tid * 2 + 1] = l;
            if (n_split > 1) {
                slot[kRows * D + tid] = M;
                slot[kRows * D + kRows + tid] = l;
            }
        }
        __syncthreads();
        const int row0 = rt * kRows;
        auto put = [&](int row, int d, float v) {
            const int q_row = row0 + row, tok = q_row / p.G;
            if (tok < n)
                store_from_float(p.o, (((int64_t)b * p.T + tok) * p.Hq + kvh * p.G + q_row - tok * p.G) * D + d, v,
                                 p.act_dtype);
        };
        for (int e = tid; e < kRows * D; e += kThreads) {
            const int row = e / D, d = e - row * D;
            const float* mw = merge_s + (row >> 3) * 8 * D + d * 8 + ((row & 7) ^ ((d >> 2) & 7));
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) o += ml_s[(w * kRows + row) * 2] * mw[w * kRows * D];
            if (n_split == 1) put(row, d, o / ml_s[row * 2 + 1]);
            else slot[row * D + d] = o;
        }
        if (n_split > 1) {
            __syncthreads();
            int* counter = p.counters + unit;
            if (tid == 0) {
                __threadfence();
                const int last = atomicAdd(counter, 1) == n_split - 1;
                if (last) __threadfence();
                misc[8] = last;
            }
            __syncthreads();
            if (misc[8]) {
                // the last piece of the unit joins the slots, in the order of the pieces
                for (int e = tid; e < kRows * D / 4; e += kThreads) {
                    const int row = e * 4 / D, d = e * 4 - row * D;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    float M = kLowest, l = 0.f;
                    constexpr int kBatch = 4;
                    for (int c = 0; c < n_split; c += kBatch) {
                        float4 ov[kBatch];
                        float mv[kBatch], lv[kBatch];
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            if (c + k >= n_split) break;
                            const long long cc = c0 + c + k;
                            const int sub = (c + k == 0 && u_start != c0 * R) ? 1 : 0;
                            const float* sl = p.partials + (2 * cc + sub) * kRows * (D + 2);
                            ov[k] = __ldcg(reinterpret_cast<const float4*>(sl + row * D + d));
                            mv[k] = __ldcg(sl + kRows * D + row);
                            lv[k] = __ldcg(sl + kRows * D + kRows + row);
                        }
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            if (c + k >= n_split) break;
                            const float Mn = fmaxf(M, mv[k]), x = fast_exp2(M - Mn), y = fast_exp2(mv[k] - Mn);
                            M = Mn;
                            l = l * x + lv[k] * y;
                            o.x = o.x * x + ov[k].x * y;
                            o.y = o.y * x + ov[k].y * y;
                            o.z = o.z * x + ov[k].z * y;
                            o.w = o.w * x + ov[k].w * y;
                        }
                    }
                    put(row, d, o.x / l);
                    put(row, d + 1, o.y / l);
                    put(row, d + 2, o.z / l);
                    put(row, d + 3, o.w / l);
                }
                if (tid == 0) *counter = 0;
            }
        }
        // the next piece's copies (async proxy) follow these generic writes of the ring's memory
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    if (!dep_done) asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct LaunchInfo {
    int grid = 0;
    int occ = 0;
};

// Kernel attributes, set up once for each device (the caller has made `device` current).
template <int D, int kTiles, bool kSplitQ>
LaunchInfo launch_info(int device) {
    constexpr int kMaxDevices = 64;
    static std::once_flag once[kMaxDevices];
    static LaunchInfo info[kMaxDevices];
    if (device < 0 || device >= kMaxDevices) return LaunchInfo{};
    std::call_once(once[device], [device] {
        auto kern = kv4_attn_kernel<D, kTiles, kSplitQ>;
        const size_t smem = AttnGeo<D, kTiles, kSplitQ>::total(kKv4MaxBatch);
        int occ = 0, sms = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, AttnGeo<D, kTiles, kSplitQ>::total(256)) !=
            cudaSuccess)
            return;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return;
        info[device].occ = occ;
        info[device].grid = occ * sms;
    });
    return info[device];
}

// Calls f with the instantiation for (D, rows per sequence and kv head, fp16).
template <typename F>
cudaError_t dispatch(int D, int rows, int act_dtype, F&& f) {
    auto by_type = [&](auto d, auto tiles) {
        return act_dtype == kF16 ? f(d, tiles, std::true_type{}) : f(d, tiles, std::false_type{});
    };
    auto by_rows = [&](auto d) {
        return rows <= 8 ? by_type(d, std::integral_constant<int, 1>{}) : by_type(d, std::integral_constant<int, 2>{});
    };
    switch (D) {
        case 64: return by_rows(std::integral_constant<int, 64>{});
        case 96: return by_rows(std::integral_constant<int, 96>{});
        case 128: return by_rows(std::integral_constant<int, 128>{});
        case 256: return by_type(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
        default: return cudaErrorInvalidValue;
    }
}

// 8-row tiles of q per (sequence, kv head), and the bytes of one tile's operand words.
int q_tiles_of(const Kv4Params& p) { return (p.T * p.G + 7) / 8; }

}  // namespace

size_t kv4_frag_bytes(const Kv4Params& p) {
    return (size_t)q_tiles_of(p) * p.Hkv * (p.D / 32) * 32 * 16 * 2;
}
size_t kv4_sums_bytes(const Kv4Params& p) { return (size_t)q_tiles_of(p) * p.Hkv * (p.D / 32 + 1) * 8 * 4; }

void kv4_attn_workspace(const Kv4Params& p, int device, size_t* partial_bytes, size_t* units_per_seq) {
    const int rows = p.T * p.G;
    *partial_bytes = 0;
    dispatch(p.D, rows, p.act_dtype, [&](auto d, auto tiles, auto split) {
        constexpr int kD = decltype(d)::value, kT = decltype(tiles)::value;
        const LaunchInfo li = launch_info<kD, kT, decltype(split)::value>(device);
        *partial_bytes = (size_t)2 * li.grid * 8 * kT * (kD + 2) * sizeof(float);
        *units_per_seq = (size_t)p.Hkv * ((rows + 8 * kT - 1) / (8 * kT));
        return cudaSuccess;
    });
}

cudaError_t launch_kv4_attn(const Kv4Params& p, int device, cudaStream_t stream) {
    return dispatch(p.D, p.T * p.G, p.act_dtype, [&](auto d, auto tiles, auto split) {
        constexpr int kD = decltype(d)::value, kT = decltype(tiles)::value;
        auto kern = kv4_attn_kernel<kD, kT, decltype(split)::value>;
        const LaunchInfo li = launch_info<kD, kT, decltype(split)::value>(device);
        if (li.grid <= 0) return cudaErrorInvalidConfiguration;
        // launched with programmatic serialisation behind the preparation kernel
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)li.grid);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = AttnGeo<kD, kT, decltype(split)::value>::total(p.B);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kern, p);
    });
}

}  // namespace b2a
