// kv4_attn.cu -- attention of the new tokens of each sequence over the paged 4-bit cache (kv4.cuh).
//
// With codes c, scales s and minima z of group y (32 channels), and keys j <= the query's position,
//     S_j = scale * sum_y ( s_yj * sum_{i in y} q_i c_ij  +  z_yj * sum_{i in y} q_i )
//     o_i = ( sum_j (P_j s_yj) c_ij  +  sum_j P_j z_yj ) / sum_j P_j,   P_j = exp(S_j - max)
// so both products run on the codes themselves: the scale of a key's group multiplies the group's
// score (32 bits) or the probability (the second product's B operand), and the minima enter through
// one more MMA each: z (keys x groups) times the sums of q, and z^T (groups x keys, with rows of
// ones below it, which give sum_j P_j) times P.  No value is ever dequantised.
//
// Bound.  A key costs 1.25 D bytes per kv head for G query heads, about 3.2 G flop per byte: HBM,
// provided the instructions per key stay few.  Per 16 keys and 32 channels a warp spends twenty
// integer instructions on 2 x 512 codes (two masks and a shift per word pair; the block layout is
// the MMA's own operand order) and four MMAs of 16 keys (K) or 16 channels (V^T) x 8 columns.
// Measured at head dim 256, 256 sequences of 16.9 k keys (1.38 GB of codes): 272 us back to back, 5.1
// TB/s (283 to 303 us as one call behind an L2 flush), where copying the rings alone takes 215 us; some 620 warp instructions a block keep 60% of the issue slots
// and 54% of the integer pipe busy, and registers allow three warps a scheduler.  Short work is
// latency: 64 sequences of 4.4 k keys, head dim 64 (45 MB), take 31 us, of them 13 in the loop.
//
// Precision.  q and P are f16 operands.  One rounding of each is far below a bf16 result's own; for
// fp16 results each is carried as two words (hi + lo): with at most four query rows the lo words take
// the columns 4..7 of the same MMAs (kSplit 1, nothing extra to multiply), else a second column tile
// (kSplit 2).  The rounding of P s is corrected exactly: lo = fma(P, s, -hi) + P_lo s.  With one word an
// output errs by up to 2^-12 of what it is made of, s c and z, not of their sum: a value far below
// its group's range has the absolute error of the group's large ones.
//
// The tensor cores add to their fp32 accumulators by truncation, a loss towards zero that grows with
// the number of blocks, and the codes are all positive.  Every second block therefore enters as
// s c + z = -s (15 - c) + z + 15 s: its codes complemented (free, in the masks), its P s negated, so
// that the accumulators stay near the difference of two like sums; 15 sum P s is one more MMA.  The
// sums over minima, scales and P are added to their totals in fp32 outside the MMA.
//
// Work split.  A unit is (sequence, kv head, tile of query rows); a query row is (token, head of the
// group), so one cache byte serves every head of its group and every token of a draft.  The
// preparation kernel spreads the units' blocks of 16 keys over the CTAs (kv4_append.cu: plan); the
// pieces of a cut unit meet through partial slots (m, l, O) that the last one to finish joins.
// Inside a piece each warp walks its own blocks with its own ring of bulk copies: one copy of 20 D
// bytes is a block, its address comes from page-table entries fetched 32 blocks at a time, and the
// warps meet only at the end of the piece.
//
// Softmax.  P is computed against a reference that moves only when a probability would exceed 2^15 /
// s_max (s_max: the largest value scale seen, at least 1), to where the largest is 2^7 / s_max: a
// block normally costs no reduction across lanes, P and P s stay inside fp16 with at least 2^21 of
// range below the largest weight before subnormals begin, and sums are in fp32 throughout.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "kv4.cuh"
#include "sm100.cuh"

namespace b2a {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLowest = -1e37f;  // largest score before any key: finite, so differences are numbers

template <int D_, int kTiles_, int kSplit_, bool kPipelined_ = false>
struct Cfg {
    static constexpr int D = D_;
    static constexpr int kTiles = kTiles_;  // column tiles of 8 in the second product
    static constexpr int kSplit = kSplit_;  // 0: one word, 1: lo words in columns 4..7, 2: in tile 1
    static constexpr int kRows = kSplit == 1 ? 4 : (kSplit == 2 ? 8 : 8 * kTiles);
    static constexpr int kSTiles = kSplit == 2 ? 1 : kTiles;  // column tiles of scores
    static constexpr int kCols = 8 * kSTiles;                 // columns of a warp's merged output
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kBlockBytes = kv4_block_bytes(D);
    static constexpr int kSub = D <= 96 ? 2 : 1;  // blocks per ring stage
    static constexpr int kStages = D <= 96 ? 3 : (D <= 128 ? 4 : 3);
    static constexpr int kStageBytes = kSub * kBlockBytes;
    // Side by side in the loop: the scores of one stage and the second product of the one before.  It
    // takes the registers of a third CTA per SM (dispatch says when that pays).
    static constexpr bool kPipelined = kPipelined_;
    // CTAs per SM, the registers' bound
    static constexpr int kCtas = kPipelined ? 2 : (D <= 64 ? (kTiles == 1 ? 4 : 3) : (kTiles == 1 ? 3 : 2));
    // fixed cost of a piece in blocks of streaming time, charged to every unit by the split
    static constexpr int kGapBlocks = D <= 64 ? 26 : (D <= 96 ? 22 : (D <= 128 ? 20 : 16));
    static constexpr int kMinBlocks = 8;  // smallest piece
    // q's operand words in shared memory where the accumulators leave no registers for them
    static constexpr bool kQShared = D * kTiles > (kPipelined ? 256 : 128);
    // head dim 256: the value params are regrouped in shared memory (their rows lie 128 bytes
    // apart, so that reading pairs of keys directly would meet in the same banks)
    static constexpr bool kRegroup = D >= 256;
    static constexpr size_t a128(size_t x) { return (x + 127) / 128 * 128; }
    static constexpr size_t kRingBytes = size_t(kWarps) * kStages * kStageBytes;
    static constexpr size_t kMergeBytes = size_t(kWarps) * kCols * D * 4;
    static constexpr size_t oBars = a128(kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes);
    static constexpr size_t oMl = oBars + kWarps * kStages * 8;
    static constexpr size_t oMisc = a128(oMl + size_t(kWarps) * kCols * 2 * 4);
    static constexpr size_t kQWords = size_t(kTiles) * kGroups * 32 * 16;
    static constexpr size_t oQ = oMisc + 256;
    static constexpr size_t oPairs = oQ + (kQShared ? kQWords : 0);
    static constexpr size_t kSmem = oPairs + (kRegroup ? kWarps * 512 : 0);
    static_assert(kGapBlocks <= kKv4GapBlocksMax, "host launch split assumes this bound");
    static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

__device__ __forceinline__ uint32_t ld32(const unsigned char* a) { return *reinterpret_cast<const uint32_t*>(a); }
__device__ __forceinline__ uint2 ld64(const unsigned char* a) { return *reinterpret_cast<const uint2*>(a); }
// n consecutive params (4 bytes each), 8- or 16-byte aligned as the layout gives them
template <int N>
__device__ __forceinline__ void ld_params(const unsigned char* a, uint32_t (&x)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(a + i * 4);
            x[i] = w.x, x[i + 1] = w.y, x[i + 2] = w.z, x[i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 w = ld64(a + i * 4);
            x[i] = w.x, x[i + 1] = w.y;
        }
    }
}
// The warp MMA (16 x 8 x 16, f16 operands, fp32 accumulators) without ordering against other code:
// d += a b, and d = a b.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (zero: four registers that hold 0; a constant would be copied into d's registers each time)
struct Zero {
    float r[4];
    __device__ __forceinline__ Zero() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.f32 %0, 0f00000000;" : "=f"(r[i]));
    }
};
__device__ __forceinline__ void mma_set(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const Zero& z) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z.r[0]), "f"(z.r[1]), "f"(z.r[2]),
          "f"(z.r[3]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // movmatrix
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// The A operand of one 16 x 16 tile of codes, or of 15 - codes (kFlip).
template <bool kFlip = false>
__device__ __forceinline__ void code_frag(uint32_t (&a)[4], uint32_t w) {
    const uint32_t h = w >> 8;
    a[0] = (kFlip ? ~w : w) & 0x000F000Fu;
    a[1] = (kFlip ? ~h : h) & 0x000F000Fu;
    a[2] = (kFlip ? ~w : w) & 0x00F000F0u;
    a[3] = (kFlip ? ~h : h) & 0x00F000F0u;
}
__device__ __forceinline__ __half2 h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }
// NaN halves become zero
__device__ __forceinline__ uint32_t no_nan(uint32_t x) {
    if ((x & 0x7fffu) > 0x7c00u) x &= 0xffff0000u;
    if ((x >> 16 & 0x7fffu) > 0x7c00u) x &= 0x0000ffffu;
    return x;
}

template <typename C>
__global__ void __launch_bounds__(kThreads, C::kCtas) kv4_attn_kernel(const __grid_constant__ Kv4Params p) {
    constexpr int D = C::D, kTiles = C::kTiles, kSTiles = C::kSTiles, kSplit = C::kSplit;
    constexpr int kGroups = C::kGroups, kStages = C::kStages, kRows = C::kRows, kSub = C::kSub, kCols = C::kCols;
    constexpr uint32_t kOnes = 0x3C003C00u;  // f16x2 (1, 1)
    extern __shared__ __align__(128) unsigned char smem[];
    float* merge_s = reinterpret_cast<float*>(smem);
    float* ml_s = reinterpret_cast<float*>(smem + C::oMl);
    int* misc = reinterpret_cast<int*>(smem + C::oMisc);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t4 = lane & 3;
    unsigned char* const ring = smem + warp * kStages * C::kStageBytes;
    const uint32_t ring_at = smem_u32(ring), bars = smem_u32(smem + C::oBars) + warp * kStages * 8;
    unsigned char* const pairs = smem + C::oPairs + warp * 512;

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; ++s) mbar_init(bars + s * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }

    const int all_rows = p.T * p.G;
    const int row_tiles = (all_rows + kRows - 1) / kRows;
    const int q_tiles = (all_rows + 7) / 8;  // tiles of 8 rows that the preparation laid out
    bool dead = false;  // a copy of this warp did not arrive in time
    int slot = 0;       // this warp's next stage: its place in the ring and its barrier's parity
    uint32_t phase = 0;

    // the preparation kernel made the plan, the q operands and the new rows' blocks
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Kv4Piece* piece = p.plan + blockIdx.x;
    for (int left = -1; left != 0; --left) {
        const int4 w0 = reinterpret_cast<const int4*>(piece)[0], w1 = reinterpret_cast<const int4*>(piece)[1],
                   w2 = reinterpret_cast<const int4*>(piece)[2];
        if (left < 0) left = w2.z;
        if (left == 0) break;
        piece = p.plan + w2.w;  // the next one, where there is one
        const int b = w0.x, r = w0.y, L = w0.z, n = w0.w;
        const int n_split = w1.z, my_part = w1.w, part0 = w2.x, part_step = w2.y;
        const int kvh = r / row_tiles, rt = r - kvh * row_tiles;
        // tokens of this tile's rows, and the blocks of the piece that they see
        const int t_lo = rt * kRows / p.G, t_hi = min(n - 1, (rt * kRows + kRows - 1) / p.G);
        const int key_lo = p.window > 0 ? max(0, L + t_lo - p.window + 1) : 0;
        const int blk0 = max(w1.x, key_lo / kKv4Block);
        const int blk1 = t_lo <= t_hi ? min(w1.y, (L + t_hi) / kKv4Block + 1) : blk0;
        const int key_hi = min(L + t_hi, blk1 * kKv4Block - 1);  // last key that some row takes from this piece
        const int unit = b * p.Hkv * row_tiles + r;

        // ------------------------------------------------------------ this warp's stages
        // stage i holds blocks blk0 + (warp + 4 i) kSub + 0 .. kSub - 1 (those below blk1)
        const int bpp = p.page_size / kKv4Block;
        const int my_n = max(0, ((blk1 - blk0 + kSub - 1) / kSub - warp + kWarps - 1) / kWarps);
        bool bad = false;
        auto entry = [&](int x) {  // place in the pool, in blocks, of the warp's x-th block, per lane; -1: none
            const int blk = blk0 + (warp + kWarps * (x / kSub)) * kSub + x % kSub;
            if (x / kSub >= my_n || blk >= blk1) return -1;
            const int slot = blk / bpp, in = blk - slot * bpp;
            const int page = p.page_table[(int64_t)b * p.max_pages + slot];
            if (page < 0 || page >= p.num_pages) {
                bad = true;
                return 0;
            }
            return (page * p.Hkv + kvh) * bpp + in;
        };
        int cur = entry(lane), nxt = entry(32 + lane);
        auto issue = [&](int i, int to) {  // request the warp's i-th stage into ring slot `to`
            const int x = i * kSub;
            if (x > 0 && (x & 31) == 0) {
                cur = nxt;
                nxt = entry(x + 32 + lane);
            }
            int off[kSub];
#pragma unroll
            for (int u = 0; u < kSub; ++u) off[u] = __shfl_sync(0xffffffffu, cur, (x & 31) + u);
            if (lane == 0) {
                uint32_t bytes = 0;
#pragma unroll
                for (int u = 0; u < kSub; ++u) bytes += off[u] >= 0 ? C::kBlockBytes : 0;
                mbar_expect_tx(bars + to * 8, bytes);
#pragma unroll
                for (int u = 0; u < kSub; ++u)
                    if (off[u] >= 0)
                        bulk_load(ring_at + to * C::kStageBytes + u * C::kBlockBytes,
                                  p.pages + (int64_t)off[u] * C::kBlockBytes, C::kBlockBytes, bars + to * 8);
            }
        };
        int issued = 0;
        auto fill = [&](int upto) {  // the first stages, into the slots from `slot` on
            for (; !dead && issued < min(upto, my_n); ++issued)
                issue(issued, slot + issued < kStages ? slot + issued : slot + issued - kStages);
        };
        // ------------------------------------------------------------ q operands
        // B operand words per column tile and group: four a lane (two 16-channel steps), column g
        uint32_t qf[kTiles][kGroups][4], qz[kSTiles][2];
        float f[kSTiles][2];   // log2 units per score unit, columns 2t and 2t + 1
        int lim[kSTiles][2];   // last key that the columns' rows see in this piece
        uint4* const q_s = reinterpret_cast<uint4*>(smem + C::oQ) + lane;
        auto row_of = [&](int tile, int col) { return rt * kRows + (kSplit == 1 ? (col & 3) : tile * 8 + col); };
        const int64_t head = (int64_t)b * p.Hkv + kvh;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            const int row = row_of(kSplit == 2 ? 0 : j, g);
            const bool there = row < all_rows && row / p.G < n;
            const int64_t at = head * q_tiles + (there ? row >> 3 : 0);
            const bool lo_word = kSplit == 1 ? g >= 4 : (kSplit == 2 && j == 1);
            const uint4* src = p.q_frag + (at * 2 + (lo_word ? 1 : 0)) * (kGroups * 32) + (row & 7) * 4 + t4;
#pragma unroll
            for (int y = 0; y < kGroups; ++y) {
                if (C::kQShared && warp != y % kWarps) continue;
                uint4 w = make_uint4(0, 0, 0, 0);
                if (there) w = src[y * 32];
                if constexpr (C::kQShared) q_s[(j * kGroups + y) * 32] = w;
                else qf[j][y][0] = w.x, qf[j][y][1] = w.y, qf[j][y][2] = w.z, qf[j][y][3] = w.w;
            }
            if (j < kSTiles) {
                // the groups' sums of q, two halves each (k = group and k = 8 + group): 2^20 times as large as
                // the products with the codes, so that the second half is no subnormal and keeps its bits
                float s0 = 0.f, s1 = 0.f;
                const float* sums = p.q_sums + at * (kGroups + 1) * 8;
                if (there && !lo_word && 2 * t4 < kGroups) s0 = sums[2 * t4 * 8 + (row & 7)];
                if (there && !lo_word && 2 * t4 + 1 < kGroups) s1 = sums[(2 * t4 + 1) * 8 + (row & 7)];
                const __half2 hi = __floats2half2_rn(s0, s1);
                qz[j][0] = u32(hi);
                qz[j][1] = pack_half2(s0 - __low2float(hi), s1 - __high2float(hi));
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int rc = row_of(j, 2 * t4 + c), tok = rc / p.G;
                    const bool in = rc < all_rows && tok < n;
                    f[j][c] = in ? p.q_sums[(head * q_tiles + (rc >> 3)) * (kGroups + 1) * 8 + kGroups * 8 + (rc & 7)] : 0.f;
                    lim[j][c] = in ? min(L + tok, key_hi) : -1;
                }
            }
        }
        // requested after q's operands: the page-table entries arrive meanwhile
        fill(kStages);
        if (C::kQShared) __syncthreads();
        // keys [all_lo, all_hi] are seen by every present row of the tile (what an absent row
        // computes is not used, and its q operand is zero)
        const int all_hi = min(L + t_lo, key_hi);
        const int all_lo = p.window > 0 ? L + t_hi - p.window + 1 : 0;

        // ------------------------------------------------------------ main loop
        float acc[kTiles][D / 16][4], zl[kTiles][4];  // zl: sum P z of group g (2), sum P (2)
        float ps[kTiles][2];                          // sum P s of group g over the complemented blocks
        float ref[kSTiles][2], top[kSTiles][2];       // reference point of P, largest score
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) acc[j][k][0] = acc[j][k][1] = acc[j][k][2] = acc[j][k][3] = 0.f;
            zl[j][0] = zl[j][1] = zl[j][2] = zl[j][3] = ps[j][0] = ps[j][1] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < kSTiles; ++j) {
            ref[j][0] = ref[j][1] = 0.f;
            top[j][0] = top[j][1] = kLowest;
        }
        bool fresh = true;  // some present row has seen no key yet: its reference is still to be set
        float s_log = 0.f;                                 // log2 of the bound on the value scales
        __half2 s_bound = __float2half2_rn(1.f);

        const Zero zero;
        // What a stage carries from its softmax to its second product.
        // sv[u][h][y]: scales of keys 2t + 8h and 2t + 8h + 1, group y
        // zv, gv: minima and scales of these keys in group g, the A operands of their sums
        // ph, pl: P of keys 0..7 and 8..15 of the block as B operands (lo words where kept)
        [[maybe_unused]] uint32_t sv[kSub][2][C::kRegroup ? 1 : kGroups];
        uint32_t zv[kSub][2], gv[kSub][2], ph[kSub][kSTiles][2];
        [[maybe_unused]] uint32_t pl[kSub][kSplit ? kSTiles : 1][2];
        float x[kSub][kSTiles][4];  // scores, then their distance from the reference

        auto scores = [&](const unsigned char* stage) {
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const unsigned char* const base = stage + u * C::kBlockBytes;
                const unsigned char* const kp = base + kv4_off_kparam(D) + g * (2 * kGroups * 4);
                uint32_t kw[2 * kGroups];  // params of keys g and g + 8
                ld_params(kp, kw);
                // minima of the groups whose sums this lane's k columns hold
                constexpr int kPairs = (kGroups + 1) / 2;
                const int y0 = 2 * (t4 % kPairs), y1 = min(y0 + 1, kGroups - 1);
                const uint32_t za = high_halves(ld32(kp + y0 * 4), ld32(kp + y1 * 4));
                const uint32_t zb = high_halves(ld32(kp + (kGroups + y0) * 4), ld32(kp + (kGroups + y1) * 4));
                const uint32_t zf[4] = {za, zb, za, zb};
#pragma unroll
                for (int j = 0; j < kSTiles; ++j) {
                    mma_set(x[u][j], zf, qz[j][0], qz[j][1], zero);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][j][e] *= 0x1p-20f;
                }
#pragma unroll
                for (int y = 0; y < kGroups; ++y) {
                    const uint2 w = ld64(base + y * 256 + lane * 8);
                    uint32_t a[4], c[4];
                    code_frag(a, w.x);
                    code_frag(c, w.y);
                    const float sa = __low2float(h2(kw[y])), sb = __low2float(h2(kw[kGroups + y]));
                    float d[kSTiles][4];
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        uint4 q;
                        if constexpr (C::kQShared) q = q_s[(j * kGroups + y) * 32];
                        else q = make_uint4(qf[j][y][0], qf[j][y][1], qf[j][y][2], qf[j][y][3]);
                        float(&dj)[4] = d[kSplit == 2 ? 0 : j];
                        if (kSplit != 2 || j == 0) mma_set(dj, a, q.x, q.y, zero);
                        else mma_add(dj, a, q.x, q.y);
                        mma_add(dj, c, q.z, q.w);
                    }
#pragma unroll
                    for (int j = 0; j < kSTiles; ++j) {
                        x[u][j][0] += sa * d[j][0];
                        x[u][j][1] += sa * d[j][1];
                        x[u][j][2] += sb * d[j][2];
                        x[u][j][3] += sb * d[j][3];
                    }
                }
            }
        };

        auto softmax = [&](const unsigned char* stage, int i) {
            const int key0 = (blk0 + (warp + kWarps * i) * kSub) * kKv4Block;
            const bool whole = key0 + kSub * kKv4Block - 1 <= all_hi && key0 >= all_lo;
            float over = -INFINITY;
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int ka = key0 + u * kKv4Block + g, kb = ka + 8;
#pragma unroll
                for (int j = 0; j < kSTiles; ++j) {
                    if constexpr (kSplit == 1) {  // hi and lo columns: lanes t and t ^ 2
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][j][e] += __shfl_xor_sync(0xffffffffu, x[u][j][e], 2);
                    }
                    x[u][j][0] = fmaf(x[u][j][0], f[j][0], -ref[j][0]);
                    x[u][j][1] = fmaf(x[u][j][1], f[j][1], -ref[j][1]);
                    x[u][j][2] = fmaf(x[u][j][2], f[j][0], -ref[j][0]);
                    x[u][j][3] = fmaf(x[u][j][3], f[j][1], -ref[j][1]);
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = e < 2 ? ka : kb, hi = lim[j][e & 1];
                            // lim is cut at the piece's end: the window counts from the row's own position
                            const int own = L + row_of(j, 2 * t4 + (e & 1)) / p.G;
                            if (key > hi || (p.window > 0 && key <= own - p.window)) x[u][j][e] = -INFINITY;
                        }
                    }
                    over = fmaxf(over, fmaxf(fmaxf(x[u][j][0], x[u][j][2]), fmaxf(x[u][j][1], x[u][j][3])));
                }
            }

            // ---------------------------------------------------- value params
            __half2 s_top = __float2half2_rn(0.f);
            auto regroup = [&](int u, bool clean) {  // head dim 256: pairs of keys side by side, in shared memory
                uint32_t w[4];  // key (lane >> 2) + 8 ((lane >> 1) & 1), groups 4 (lane & 1) + 0 .. 3
                ld_params(stage + u * C::kBlockBytes + kv4_off_vparam(D) + lane * 16, w);
                if (!whole) {
                    const int key = key0 + u * kKv4Block + g + 8 * ((lane >> 1) & 1);
                    if (key < key_lo || key > key_hi) w[0] = w[1] = w[2] = w[3] = 0;
                }
                if (clean) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = no_nan(w[e]);
                }
                const bool odd = g & 1;
                const uint32_t r0 = __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[2], 4);
                const uint32_t r1 = __shfl_xor_sync(0xffffffffu, odd ? w[1] : w[3], 4);
                // the even key's lane makes groups 4 (lane & 1) + 0, 1, the odd one's + 2, 3
                const uint32_t e0 = odd ? r0 : w[0], e1 = odd ? r1 : w[1], o0 = odd ? w[2] : r0, o1 = odd ? w[3] : r1;
                const uint32_t s0 = low_halves(e0, o0), s1 = low_halves(e1, o1);
                s_top = __hmax2_nan(s_top, __hmax2_nan(h2(s0), h2(s1)));
                __syncwarp();  // every lane has read what was there
                uint32_t* const at = reinterpret_cast<uint32_t*>(pairs) + (4 * (lane & 1) + 2 * odd) * 8 + (g >> 1) * 2 +
                                     ((lane >> 1) & 1);
                at[0] = s0;
                at[8] = s1;
                at[64] = high_halves(e0, o0);
                at[72] = high_halves(e1, o1);
                __syncwarp();
                const uint2 z = ld64(pairs + 256 + (g * 4 + t4) * 8);
                zv[u][0] = z.x;
                zv[u][1] = z.y;
                const uint2 sg = ld64(pairs + (g * 4 + t4) * 8);
                gv[u][0] = sg.x;
                gv[u][1] = sg.y;
            };
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                if constexpr (C::kRegroup) {
                    regroup(u, false);
                } else {
                    const unsigned char* const vp = stage + u * C::kBlockBytes + kv4_off_vparam(D);
                    uint32_t wa[2 * kGroups], wb[2 * kGroups];  // keys 2t, 2t + 1 (and + 8)
                    ld_params(vp + 2 * t4 * (2 * kGroups * 4), wa);
                    ld_params(vp + (2 * t4 + 1) * (2 * kGroups * 4), wb);
                    const unsigned char* const gz = vp + (2 * t4 * 2 * kGroups + min(g, kGroups - 1)) * 4;
                    const uint32_t w0 = ld32(gz), w1 = ld32(gz + 2 * kGroups * 4);
                    const uint32_t w2 = ld32(gz + kGroups * 4), w3 = ld32(gz + 3 * kGroups * 4);
                    uint32_t z0 = high_halves(w0, w1), z1 = high_halves(w2, w3);
                    uint32_t g0 = low_halves(w0, w1), g1 = low_halves(w2, w3);
                    uint32_t m0 = 0xffffffffu, m1 = 0xffffffffu;
                    if (!whole) {
                        const int key = key0 + u * kKv4Block + 2 * t4;
                        auto in = [&](int k) { return k >= key_lo && k <= key_hi; };
                        m0 = (in(key) ? 0xffffu : 0u) | (in(key + 1) ? 0xffff0000u : 0u);
                        m1 = (in(key + 8) ? 0xffffu : 0u) | (in(key + 9) ? 0xffff0000u : 0u);
                        z0 &= m0;
                        z1 &= m1;
                        g0 &= m0;
                        g1 &= m1;
                    }
#pragma unroll
                    for (int y = 0; y < kGroups; ++y) {
                        sv[u][0][y] = low_halves(wa[y], wb[y]);
                        sv[u][1][y] = low_halves(wa[kGroups + y], wb[kGroups + y]);
                        if (!whole) {
                            sv[u][0][y] &= m0;
                            sv[u][1][y] &= m1;
                        }
                        s_top = __hmax2_nan(s_top, __hmax2_nan(h2(sv[u][0][y]), h2(sv[u][1][y])));
                    }
                    zv[u][0] = z0;
                    zv[u][1] = z1;
                    gv[u][0] = g0;
                    gv[u][1] = g1;
                }
            }

            // ---------------------------------------------------- rarely: move the reference point
            if (fresh || __any_sync(0xffffffffu, over > 15.f - s_log || !__hble2(s_top, s_bound))) {
                float sm = fmaxf(__low2float(s_top), __high2float(s_top));
                sm = warp_max(__hisnan(__low2half(s_top)) || __hisnan(__high2half(s_top)) ? INFINITY : sm);
                if (isinf(sm)) {
                    // A seen key holds NaN in some group of its value: the group is NaN for the rows
                    // that see the key, and counts as zero in the products, whose columns share it.
#pragma unroll
                    for (int u = 0; u < kSub; ++u) {
                        const unsigned char* const vp = stage + u * C::kBlockBytes + kv4_off_vparam(D) + g * (2 * kGroups * 4);
#pragma unroll
                        for (int y = 0; y < kGroups; ++y) {
                            const bool na = (ld32(vp + y * 4) & 0x7fffu) > 0x7c00u;
                            const bool nb = (ld32(vp + (kGroups + y) * 4) & 0x7fffu) > 0x7c00u;
#pragma unroll
                            for (int j = 0; j < kSTiles; ++j) {
                                unsigned hit = 0;  // bit per column
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if ((e < 2 ? na : nb) && x[u][j][e] != -INFINITY) hit |= 1u << (2 * t4 + (e & 1));
                                hit = __reduce_or_sync(0xffffffffu, hit);
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (hit >> (2 * t4 + (e & 1)) & 1) acc[j][2 * y][e] = acc[j][2 * y + 1][e] = nan_f();
                            }
                        }
                        if constexpr (C::kRegroup) {
                            s_top = __float2half2_rn(0.f);
                            regroup(u, true);
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                zv[u][h] = no_nan(zv[u][h]);
                                gv[u][h] = no_nan(gv[u][h]);
#pragma unroll
                                for (int y = 0; y < kGroups; ++y) sv[u][h][y] = no_nan(sv[u][h][y]);
                            }
                        }
                    }
                    if constexpr (!C::kRegroup) {
                        s_top = __float2half2_rn(0.f);
#pragma unroll
                        for (int u = 0; u < kSub; ++u)
#pragma unroll
                            for (int y = 0; y < kGroups; ++y)
                                s_top = __hmax2(s_top, __hmax2(h2(sv[u][0][y]), h2(sv[u][1][y])));
                    }
                    sm = warp_max(fmaxf(__low2float(s_top), __high2float(s_top)));
                }
                if (sm > __low2float(s_bound)) {  // the next power of two, at most 2^12 (2^16 / 15)
                    s_log = (float)(ilogbf(sm) + 1);
                    s_bound = __float2half2_rn(exp2f(s_log));
                }
                bool unset = false;
#pragma unroll
                for (int j = 0; j < kSTiles; ++j) {
                    float keep[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float m = -INFINITY;
#pragma unroll
                        for (int u = 0; u < kSub; ++u) m = fmaxf(m, fmaxf(x[u][j][c], x[u][j][c + 2]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        const float was = top[j][c];
                        top[j][c] = fmaxf(was, m + ref[j][c]);
                        const float to = top[j][c] == kLowest ? 0.f : top[j][c] - 7.f + s_log, shift = ref[j][c] - to;
                        keep[c] = was == kLowest ? 0.f : fast_exp2(shift);
                        ref[j][c] = to;
                        unset |= top[j][c] == kLowest && lim[j][c] >= 0;
#pragma unroll
                        for (int u = 0; u < kSub; ++u) {
                            x[u][j][c] += shift;
                            x[u][j][c + 2] += shift;
                        }
                    }
                    constexpr int kBoth = kSplit == 2 ? 2 : 1;  // tile 1 holds the same columns' lo words
#pragma unroll
                    for (int e = 0; e < kBoth; ++e) {
                        const int jt = kSplit == 2 ? e : j;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            acc[jt][k][0] *= keep[0];
                            acc[jt][k][1] *= keep[1];
                            acc[jt][k][2] *= keep[0];
                            acc[jt][k][3] *= keep[1];
                        }
                        zl[jt][0] *= keep[0];
                        zl[jt][1] *= keep[1];
                        zl[jt][2] *= keep[0];
                        zl[jt][3] *= keep[1];
                        ps[jt][0] *= keep[0];
                        ps[jt][1] *= keep[1];
                    }
                }
                fresh = __any_sync(0xffffffffu, unset);
            }

#pragma unroll
            for (int u = 0; u < kSub; ++u) {
#pragma unroll
                for (int j = 0; j < kSTiles; ++j) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p0 = fast_exp2(x[u][j][2 * h]), p1 = fast_exp2(x[u][j][2 * h + 1]);
                        const __half2 hi = __floats2half2_rn(p0, p1);
                        ph[u][j][h] = transpose8(u32(hi));
                        if constexpr (kSplit != 0)
                            pl[u][j][h] = transpose8(pack_half2(p0 - __low2float(hi), p1 - __high2float(hi)));
                    }
                }
            }
        };

        // acc += [codes] [P s], zl, ps: block u of the stage, complemented or not
        auto second_product = [&](const unsigned char* stage, auto block, auto complemented) {
            constexpr int u = decltype(block)::value;
            constexpr bool flip = decltype(complemented)::value;
            constexpr uint32_t flip_sign = flip ? 0x80008000u : 0u;
                // zl += [z^T; 1] P, and for a complemented block ps += s^T P
                uint32_t pz[kTiles][2];
#pragma unroll
                for (int j = 0; j < kTiles; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (kSplit == 0) pz[j][h] = ph[u][j][h];
                        else if constexpr (kSplit == 1) pz[j][h] = g >= 4 ? pl[u][0][h] : ph[u][0][h];
                        else pz[j][h] = j ? pl[u][0][h] : ph[u][0][h];
                    }
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    const uint32_t zf[4] = {zv[u][0], kOnes, zv[u][1], kOnes};
                    float d[4];
                    mma_set(d, zf, pz[j][0], pz[j][1], zero);
#pragma unroll
                    for (int e = 0; e < 4; ++e) zl[j][e] += d[e];
                    if constexpr (flip) {
                        const uint32_t gf[4] = {gv[u][0], 0u, gv[u][1], 0u};
                        float c[4];
                        mma_set(c, gf, pz[j][0], pz[j][1], zero);
                        ps[j][0] += c[0];
                        ps[j][1] += c[1];
                    }
                }
                [[maybe_unused]] uint32_t pa[2], pb[2];  // kSplit 1: the lo columns' words (the first negated), zero in the others
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < kSTiles; ++j) {
                        ph[u][j][h] ^= flip_sign;
                        if constexpr (kSplit != 0) pl[u][j][h] ^= flip_sign;
                    }
                    if constexpr (kSplit == 1) {
                        pa[h] = g >= 4 ? ph[u][0][h] ^ 0x80008000u : 0u;
                        pb[h] = g >= 4 ? pl[u][0][h] : 0u;
                    }
                }
#pragma unroll
                for (int y = 0; y < kGroups; ++y) {
                    const uint2 w = ld64(stage + u * C::kBlockBytes + kv4_off_v(D) + y * 256 + lane * 8);
                    uint32_t a[4], c[4];
                    code_frag<flip>(a, w.x);
                    code_frag<flip>(c, w.y);
                    // V^T's tile has the channel as its row: registers in the order (channel g, keys 2t),
                    // (g + 8, 2t), (g, 2t + 8), (g + 8, 2t + 8)
                    const uint32_t av[4] = {a[0], a[2], a[1], a[3]}, cv[4] = {c[0], c[2], c[1], c[3]};
                    uint32_t s[2];
                    if constexpr (C::kRegroup) {
                        const uint2 sp = ld64(pairs + (y * 4 + t4) * 8);
                        s[0] = sp.x;
                        s[1] = sp.y;
                    } else {
                        s[0] = sv[u][0][y];
                        s[1] = sv[u][1][y];
                    }
                    uint32_t bf[kTiles][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const __half2 sc = h2(s[h]);
                        if constexpr (kSplit == 0) {
#pragma unroll
                            for (int j = 0; j < kTiles; ++j) bf[j][h] = u32(__hmul2(h2(ph[u][j][h]), sc));
                        } else if constexpr (kSplit == 1) {
                            const __half2 hi = __hmul2(h2(pa[h]), sc);  // lo columns: minus what the hi column holds
                            bf[0][h] = u32(__hfma2(h2(pb[h]), sc, __hfma2(h2(ph[u][0][h]), sc, hi)));
                        } else {
                            const __half2 hi = __hmul2(h2(ph[u][0][h]), sc);
                            bf[0][h] = u32(hi);
                            bf[1][h] = u32(__hfma2(h2(pl[u][0][h]), sc, __hfma2(h2(ph[u][0][h]), sc, __hneg2(hi))));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        mma_add(acc[j][2 * y], av, bf[j][0], bf[j][1]);
                        mma_add(acc[j][2 * y + 1], cv, bf[j][0], bf[j][1]);
                    }
                }
        };
        auto second_products = [&](const unsigned char* stage, auto odd) {
            if constexpr (kSub == 2) {
                second_product(stage, std::integral_constant<int, 0>{}, std::false_type{});
                second_product(stage, std::integral_constant<int, 1>{}, std::true_type{});
            } else {
                second_product(stage, std::integral_constant<int, 0>{}, odd);
            }
        };

        auto arrived = [&](int at, uint32_t parity, int i) {  // stage i, in ring slot `at`
            if (wait_bounded(bars + at * 8, parity)) return true;
            // report, wait for the others in flight and ask for no more; the outputs are NaN
            if (lane == 0) atomicOr(p.status, 8);
            dead = true;
            for (int k = 1; k < kStages && i + k < my_n; ++k) {
                const bool wrap = at + k >= kStages;
                if (!wait_bounded(bars + (wrap ? at + k - kStages : at + k) * 8, parity ^ (wrap ? 1u : 0u))) break;
            }
            return false;
        };
        auto release = [&](int i, int at, uint32_t parity) {  // stage i is used; go on to ring slot `at`
            __syncwarp();  // every lane has read the stage
            if (!dead && i + kStages < my_n) issue(i + kStages, slot);
            slot = at;
            phase = parity;
        };
        auto step = [&](int i, auto odd) {
            const unsigned char* const stage = ring + slot * C::kStageBytes;
            const int at = slot + 1 == kStages ? 0 : slot + 1;
            const uint32_t parity = at ? phase : phase ^ 1u;
            if constexpr (C::kPipelined) {  // stage i, whose P is known, with the scores of stage i + 1
                const unsigned char* const after = ring + at * C::kStageBytes;
                const bool more = i + 1 < my_n;
                if (more && arrived(at, parity, i + 1)) {
                    scores(after);
                    second_products(stage, odd);
                } else {
                    second_products(stage, odd);
                }
                release(i, at, parity);
                if (more && !dead) softmax(after, i + 1);
            } else {
                if (!arrived(slot, phase, i)) return;
                scores(stage);
                softmax(stage, i);
                second_products(stage, odd);
                release(i, at, parity);
            }
        };
        if constexpr (C::kPipelined) {
            if (my_n > 0 && !dead && arrived(slot, phase, 0)) {
                scores(ring + slot * C::kStageBytes);
                softmax(ring + slot * C::kStageBytes, 0);
            }
        }
        if constexpr (kSub == 2) {
            for (int i = 0; i < my_n && !dead; ++i) step(i, std::false_type{});
        } else {
            for (int i = 0; i < my_n && !dead; i += 2) {
                step(i, std::false_type{});
                if (i + 1 < my_n && !dead) step(i + 1, std::true_type{});
            }
        }
        bad = __any_sync(0xffffffffu, bad);
        if (bad && lane == 0) atomicOr(p.status, 16);
        __syncthreads();  // all rings idle: merge_s may alias them

        // ------------------------------------------------------------ epilogue
#pragma unroll
        for (int j = 0; j < kSTiles; ++j) {
            // unnormalised O in [d][column] pairs, the column index XOR-swizzled by (d >> 2) & 7 as in
            // decode_tc.cu: pair stores and reads along d are free of bank conflicts
            float* mw = merge_s + (warp * kSTiles + j) * 8 * D;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                float z0 = fmaf(15.f, ps[j][0], zl[j][0]), z1 = fmaf(15.f, ps[j][1], zl[j][1]);
                if constexpr (kSplit == 2) {
                    z0 += fmaf(15.f, ps[1][0], zl[1][0]);
                    z1 += fmaf(15.f, ps[1][1], zl[1][1]);
                }
                z0 = __shfl_sync(0xffffffffu, z0, (k / 2) * 4 + t4);
                z1 = __shfl_sync(0xffffffffu, z1, (k / 2) * 4 + t4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = 16 * k + g + 8 * h, sw = (d >> 2) & 7;
                    float u = acc[j][k][2 * h], v = acc[j][k][2 * h + 1];
                    if constexpr (kSplit == 2) {
                        u += acc[1][k][2 * h];
                        v += acc[1][k][2 * h + 1];
                    }
                    u = fmaf(u, h ? 0x1p20f : 0x1p24f, z0);
                    v = fmaf(v, h ? 0x1p20f : 0x1p24f, z1);
                    *reinterpret_cast<float2*>(mw + d * 8 + ((2 * t4) ^ (sw & 6))) =
                        (sw & 1) ? make_float2(v, u) : make_float2(u, v);
                }
            }
            if (g == 0) {
                float* ml = ml_s + ((warp * kSTiles + j) * 8 + 2 * t4) * 2;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float l = zl[j][2 + c];
                    if constexpr (kSplit == 2) l += zl[1][2 + c];
                    ml[2 * c] = top[j][c] == kLowest ? kLowest : ref[j][c];
                    ml[2 * c + 1] = bad || dead ? nan_f() : l;
                }
            }
        }
        __syncthreads();
        float* slot = p.partials + (int64_t)my_part * kRows * (D + 2);
        if (tid < kRows) {
            float M = kLowest, l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml_s[(w * kCols + tid) * 2]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                float* ml = ml_s + (w * kCols + tid) * 2;
                const float k = fast_exp2(ml[0] - M);
                l += k * (kSplit == 1 ? ml[1] + ml[9] : ml[1]);  // columns 4 further on hold the lo words
                ml[0] = k;
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
            if (q_row < all_rows && tok < n)
                store_from_float(p.o, (((int64_t)b * p.T + tok) * p.Hq + kvh * p.G + q_row - tok * p.G) * D + d, v,
                                 p.act_dtype);
        };
        for (int e = tid; e < kRows * D; e += kThreads) {
            const int row = e / D, d = e - row * D, sw = (d >> 2) & 7;
            const float* mw = merge_s + (row >> 3) * 8 * D + d * 8;
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                float v = mw[w * kCols * D + ((row & 7) ^ sw)];
                if constexpr (kSplit == 1) v += mw[w * kCols * D + ((row + 4) ^ sw)];
                o += ml_s[(w * kCols + row) * 2] * v;
            }
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
                misc[0] = last;
            }
            __syncthreads();
            if (misc[0]) {
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
                            // the pieces after the first begin their CTAs' ranges
                            const int part = c + k == 0 ? part0 : (part_step == 1 ? part0 : part0 & ~1) + part_step * (c + k);
                            const float* sl = p.partials + (int64_t)part * kRows * (D + 2);
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
}

struct LaunchInfo {
    int grid = 0;
    int sms = 0;
};

// Kernel attributes, set up once for each device (the caller has made `device` current).
template <typename C>
LaunchInfo launch_info(int device) {
    constexpr int kMaxDevices = 64;
    static std::once_flag once[kMaxDevices];
    static LaunchInfo info[kMaxDevices];
    if (device < 0 || device >= kMaxDevices) return LaunchInfo{};
    std::call_once(once[device], [device] {
        auto kern = kv4_attn_kernel<C>;
        int occ = 0, sms = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem) !=
            cudaSuccess)
            return;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, C::kSmem) != cudaSuccess) return;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return;
        info[device].grid = occ * sms;
        info[device].sms = sms;
    });
    return info[device];
}

// Calls f with the instantiation for (D, query rows per sequence and kv head, element type).
//  * fp16 results carry q and P as two words.
//  * bf16 ones take 16 columns where there are as many rows (a cache byte then serves twice as many),
//    except at head dim 256, whose accumulators fill the registers with 8.
//  * Pipelined at head dim 256 where a CTA has few blocks to walk and one warp's own speed counts (256
//    sequences over a 512-key window, 33 blocks each: 30.9 -> 26.8 us); long contexts want the third CTA
//    (the same sequences over 17 k keys: 299 pipelined, 275 us not).  What a CTA has is bounded by the
//    window, else by the table's capacity: the lengths are on the device, so short contexts in a wide table
//    take the form for long ones.  With 16 columns always: the third CTA does not fit anyway
//    (5-token drafts at head dim 64: 20.6 -> 19.3 us); at head dim 64 with two-word operands never (64
//    sequences of 4 k keys: 34 pipelined, 31 us not).
constexpr int kPipelineBlocks = 128;

bool few_blocks(const Kv4Params& p, int device) {
    const int64_t keys = std::min<int64_t>(p.window > 0 ? (int64_t)p.window + p.T : INT32_MAX,
                                           (int64_t)p.max_pages * p.page_size);
    const int64_t units = (int64_t)p.B * p.Hkv * ((p.T * p.G + 7) / 8);
    // (the pipelined variant has two CTAs per SM)
    return units * (keys / kKv4Block) <= (int64_t)kPipelineBlocks * 2 * launch_info<Cfg<256, 1, 1, true>>(device).sms;
}

// few: few_blocks of the whole call, of which p may be a part.
template <typename F>
cudaError_t dispatch(const Kv4Params& p, bool few, F&& f) {
    const int rows = p.T * p.G;
    auto by_rows = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if constexpr (D == 256) {
            if (p.act_dtype == kF16) {
                if (rows > 4) return f(Cfg<D, 2, 2, true>{});
                return few ? f(Cfg<D, 1, 1, true>{}) : f(Cfg<D, 1, 1, false>{});
            }
            return few ? f(Cfg<D, 1, 0, true>{}) : f(Cfg<D, 1, 0, false>{});
        } else {
            if (p.act_dtype == kF16) return rows <= 4 ? f(Cfg<D, 1, 1>{}) : f(Cfg<D, 2, 2>{});
            return rows > 8 ? f(Cfg<D, 2, 0, true>{}) : f(Cfg<D, 1, 0>{});
        }
    };
    switch (p.D) {
        case 64: return by_rows(std::integral_constant<int, 64>{});
        case 96: return by_rows(std::integral_constant<int, 96>{});
        case 128: return by_rows(std::integral_constant<int, 128>{});
        case 256: return by_rows(std::integral_constant<int, 256>{});
        default: return cudaErrorInvalidValue;
    }
}

// 8-row tiles of q per (sequence, kv head).
int q_tiles_of(const Kv4Params& p) { return (p.T * p.G + 7) / 8; }

}  // namespace

size_t kv4_frag_bytes(const Kv4Params& p) {
    return (size_t)q_tiles_of(p) * p.Hkv * (p.D / 32) * 32 * 16 * 2;
}
size_t kv4_sums_bytes(const Kv4Params& p) { return (size_t)q_tiles_of(p) * p.Hkv * (p.D / 32 + 1) * 8 * 4; }

Kv4Split kv4_attn_split(const Kv4Params& p, int device) {
    Kv4Split split{};
    split.few = few_blocks(p, device);
    dispatch(p, split.few, [&](auto cfg) {
        using C = decltype(cfg);
        split.n_cta = launch_info<C>(device).grid;
        split.per_seq = p.Hkv * ((p.T * p.G + C::kRows - 1) / C::kRows);
        split.gap = C::kGapBlocks;
        split.min_blocks = C::kMinBlocks;
        split.partial_bytes = (size_t)2 * split.n_cta * C::kRows * (C::D + 2) * sizeof(float);
        return cudaSuccess;
    });
    return split;
}

cudaError_t launch_kv4_attn(const Kv4Params& p, int device, cudaStream_t stream) {
    return dispatch(p, p.split.few, [&](auto cfg) {
        using C = decltype(cfg);
        const LaunchInfo li = launch_info<C>(device);
        if (li.grid <= 0) return cudaErrorInvalidConfiguration;
        // launched with programmatic serialisation behind the preparation kernel
        cudaLaunchConfig_t launch = {};
        launch.gridDim = dim3((unsigned)li.grid);
        launch.blockDim = dim3(kThreads);
        launch.dynamicSmemBytes = C::kSmem;
        launch.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        launch.attrs = attr;
        launch.numAttrs = 1;
        return cudaLaunchKernelEx(&launch, kv4_attn_kernel<C>, p);
    });
}

}  // namespace b2a
