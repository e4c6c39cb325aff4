// Attention of prompts and chunks over the 8-bit cache on the fifth-generation tensor cores: heads of up to 128 channels in steps of 16,
// bfloat16 queries, causal, with an optional window.  (Layout and codes: e4m3.cuh.)
//
// One block per (two tiles of 128 query rows, key/value head, sequence).  A query row is a (token, head of the group) pair, heads
// innermost, so that the heads that share keys share their pages too and a short run of queries still fills a tile.  Per page:
//   codes -> half   four warps read the page's codes, a page ahead, turn them into halves, which is exact, and leave them in
//                   shared memory as swizzled tiles: keys [row][channel], values [channel][row], both K-major as the cache has them;
//   S  = Q K^T      tcgen05.mma 128 x 64 x head size, operands in shared memory, S in tensor memory; queries are scaled by a
//                   power of two a row to fill half's range, so that rounding bfloat16 to half loses nothing that counts;
//   P  = softmax    four warps a tile, a thread a row, scores straight from tensor memory; P goes back there as halves;
//   O += P V        tcgen05.mma 128 x head size x 64, A = P from tensor memory, O stays there.
// Scales.  A page's key scale multiplies its scores.  Its value scale 2^v cannot multiply O, which adds up over pages, and
// must not squeeze P's range either: it goes into the exponent.  With x_j = score_j + v_j (in powers of two) and M the running
// maximum of x, P_j = 2^(x_j - M) and O = sum P_j code_j.  The sum is l = sum P_j 2^(w - v_j) = sum 2^(score_j - M + w), w the
// largest v of the block's pages, and O 2^w / l the result.  Where v_j is so far below w that P_j could be 0 while its probability is
// not (a block of zeros among others, for one), v_j counts as w - 96 and the codes are made smaller for it.
// M is raised only when a step's sum of P exceeds 2^15, so P, times 2^7 besides, stays below half's largest number.  From |M| = 2^20 on
// M's own rounding counts, and v_j would get lost in it: M is also kept as the score and the v that it came of, and scores, rounded
// as that one was, are compared with it apart from the v.  So rows of one score have one probability, however large it is.
// Where that makes fewer blocks than multiprocessors, several share a pair of tiles' pages and leave their results to a joining kernel.
// No one unit bounds it: of the 2,500 cycles that a step of both tiles takes, the exponentials fill 1,024 (over a whole call their unit is
// 32 to 42 % busy) and the products 660 (64 channels) to 1,350 (128); the rest is warps waiting for one another's results, 400 to 540
// of it the softmax's for its scores.  Measured on a B200: 2,048 tokens, 32 heads of 64: 54.5 us; 512 tokens behind 7,680,
// 2 sequences, 8 kv heads of 128 under 32: 166 us, 0.83 of what the same kernel for a bfloat16 cache takes in the second case and
// 1.2 of it in the first, where the blocks' begins count.  Steps on the way there, in the second case: 128 rows a block, two threads
// a row 257; issuing from warps of their own 180; codes straight to registers instead of through shared memory 177; two
// threads a row again, with 24 warps, 195.  Every wait is bounded (status word as in the products).
#include "e4m3.cuh"
#include "tcgen05_attention.cuh"
#include <type_traits>

namespace {
constexpr int BQ = 128;                                  // query rows of a tile; a block has two
constexpr int BK = kPageTokens;                          // rows of the cache a step: a page, which has one scale
// Warps: 0-3 and 4-7 the tiles' softmax; 8, 9 convert keys, 10, 11 values; 12, 13 issue the tiles' scores, 14, 15 their
// P V (sixteen: 128 registers).  A warp's waits stand behind the products it has issued, so one warp that issued all of them
// saw every answer hundreds of cycles late: 3,600 cycles a page where the softmax takes 1,900.
constexpr int kKeyWarps = 2, kValueWarps = 2, kScoreWarp = 12, kOutputWarp = 14;
constexpr int kThreads = 512;
constexpr int kLeastSteps = 8;                           // of a block, where several share a tile pair's
constexpr int kTmemCols = 512, kTileCols = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 7.0f, kMostSum = 32768.0f;
constexpr int kMostApart = 96;                           // powers of two that a block's value scales span at most

// HD: 64 or 128, what a tile has room for; heads of fewer channels (kExact false; multiples of 16) fill a part of it, and the products
// take no more than that part.
template <int HD> struct Shape {
    static constexpr int kQBytes = BQ * HD * 2, kTileBytes = BK * HD * 2;
    static constexpr int kOffK = 2 * kQBytes, kOffV = kOffK + 2 * kTileBytes, kOffM = kOffV + 2 * kTileBytes, kOffBar = kOffM + 2 * BQ * 8;
    static constexpr int kSmemBytes = kOffBar + 256;
    static constexpr int kColO = BK, kColP = BK + HD;    // of a tile's tensor memory: S, O, two of P
    static_assert(BK + HD + BK <= kTileCols, "tensor memory");
};

// kind::f16, half operands, both K-major, float sums.
__host__ __device__ constexpr uint32_t f16_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

struct PromptArgs {
    const bf16* q;
    int ldq;
    bf16* out;
    int ldo;
    const int* cu_seqlens;
    const int* slots;
    const int* start_pos;
    int n_heads, group;
    float scale;
    int window;
    float2* stats;               // [token][head]: s, M's score, and c, or null: a row's probability is 2^(score - s + c)
    int splits;                  // blocks that share a tile pair's pages
    float* part_o;               // [token][head][split][channel]: their results, where there are several,
    float2* part_stats;          // [token][head][split]: and statistics; s is -infinity where the split saw no row
};

__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Wait for a phase, the warp asleep meanwhile (up to some 10 us at a time): a block of thirteen warps that poll instead spends half
// of its issue slots on it.  Bounded like mbar_wait.
template <bool kTest>
__device__ __forceinline__ bool mbar_sleep(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (unsigned i = 0; i < (kTest ? 64u : 1u << 18); ++i) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
                     "selp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity), "r"(10000u) : "memory");
        if (done) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(&g_status, 1);
    return false;
}
// Two phases at once: their answers are asked for side by side.
template <bool kTest>
__device__ __forceinline__ bool mbar_sleep_both(uint32_t bar, uint32_t parity, uint32_t other, uint32_t other_parity, volatile int* abort_flag) {
    for (unsigned i = 0; i < (kTest ? 64u : 1u << 18); ++i) {
        uint32_t done;
        asm volatile("{\n.reg .pred p, q;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %5;\n"
                     "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4, %5;\nand.pred p, p, q;\n"
                     "selp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity), "r"(other), "r"(other_parity), "r"(10000u) : "memory");
        if (done) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(&g_status, 1);
    return false;
}
// 16 codes as 16 halves: two chunks of a swizzled row, the second first where `turned` is odd (lanes whose tiles' blocks share
// banks then store to different ones).
__device__ __forceinline__ void store_halves(uint32_t row_at, int chunk, int swizzle, const uint4& u, int turned = 0) {
    const uint32_t a[4] = {e4m3_pair_f16(u.x), e4m3_pair_f16(u.x >> 16), e4m3_pair_f16(u.y), e4m3_pair_f16(u.y >> 16)};
    const uint32_t b[4] = {e4m3_pair_f16(u.z), e4m3_pair_f16(u.z >> 16), e4m3_pair_f16(u.w), e4m3_pair_f16(u.w >> 16)};
    const uint32_t first = row_at + (((chunk + turned) ^ swizzle) << 4), second = row_at + (((chunk + 1 - turned) ^ swizzle) << 4);
    store_shared16(first, turned ? b[0] : a[0], turned ? b[1] : a[1], turned ? b[2] : a[2], turned ? b[3] : a[3]);
    store_shared16(second, turned ? a[0] : b[0], turned ? a[1] : b[1], turned ? a[2] : b[2], turned ? a[3] : b[3]);
}
// Sixteen codes times a power of two below 1, rounded to codes.  (Next to a block 2^96 times larger, what is lost is little.)
__device__ __forceinline__ uint32_t smaller_codes(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) r |= (uint32_t)e4m3_code(e4m3_value((uint8_t)(w >> (8 * e))) * ratio) << (8 * e);
    return r;
}
__device__ __noinline__ uint4 smaller_codes(uint4 u, float ratio) {
    return make_uint4(smaller_codes(u.x, ratio), smaller_codes(u.y, ratio), smaller_codes(u.z, ratio), smaller_codes(u.w, ratio));
}
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two floats at a time.
__device__ __forceinline__ uint64_t two(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float first_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float second_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Products and commits issued by one lane of a warp that runs its loop as a whole: with the loop inside one lane's branch the
// descriptors do not stay in the warp's uniform registers, and a step's products took some 60 cycles each to issue.
__device__ __forceinline__ void warp_umma_ss(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void warp_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, e;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void warp_umma_commit(uint32_t bar) {
    asm volatile("{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar) : "memory");
}

// grid: (kv heads, sequences, pairs of tiles of query rows), the longest first.
template <int HD, bool kExact, bool kTest>
__global__ void __launch_bounds__(kThreads, 1)
attention_e4m3_prompt_kernel(const PromptArgs a, const E4M3Pages kv) {
    using S = Shape<HD>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int h = blockIdx.x, b = blockIdx.y, hd = kExact ? HD : kv.hd;
    const int place = gridDim.z - 1 - blockIdx.z, split = place % a.splits;
    const int row_begin = place / a.splits * 2 * BQ;
    const int q_begin = a.cu_seqlens[b];
    const int q_len = a.cu_seqlens[b + 1] - q_begin;
    const int n_rows = q_len * a.group;
    if (row_begin >= n_rows) {                                   // before any barrier or tensor memory
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0) chain_wait();     // (one block waits whatever there is to do, so that a grid
        return;                                                  // of nothing is not complete before the kernel it stands behind)
    }
    const uint32_t base = smem_addr(smem);
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicExch(&g_status, 2);
        return;
    }
    const uint32_t bars = base + S::kOffBar;
    // by tile: queries there, scores read; by tile and the step's parity: scores there, P there, P V done; by parity: key and
    // value tiles there and free
    auto q_full = [&](int t) { return bars + 8u * t; };
    auto s_free = [&](int t) { return bars + 16u + 8u * t; };
    auto s_full = [&](int t) { return bars + 32u + 8u * t; };
    auto p_full = [&](int t, int i) { return bars + 48u + 16u * t + 8u * (i & 1); };
    auto pv_done = [&](int t, int i) { return bars + 80u + 16u * t + 8u * (i & 1); };
    auto k_full = [&](int i) { return bars + 112u + 8u * (i & 1); };
    auto k_free = [&](int i) { return bars + 128u + 8u * (i & 1); };
    auto v_full = [&](int i) { return bars + 144u + 8u * (i & 1); };
    auto v_free = [&](int i) { return bars + 160u + 8u * (i & 1); };
    auto phase = [](int i) { return ((uint32_t)i >> 1) & 1u; };  // of step i's barriers that go by parity
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::kOffBar + 192);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffBar + 200);
    volatile int* odd_flag = reinterpret_cast<volatile int*>(smem + S::kOffBar + 204);   // a NaN code in a page not all rows see whole

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = a.slots[b];
    const int start = a.start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    const int* table = kv.block_table + (size_t)slot * kv.table_stride;
    const int n_tiles = n_rows - row_begin > BQ ? 2 : 1;
    const int first_at = start + row_begin / a.group;            // cache row of the block's first query, and of its last
    const int last_at = start + (min(row_begin + 2 * BQ, n_rows) - 1) / a.group;
    int j_lo = (a.window > 0 ? max(0, first_at - a.window + 1) : 0) / kPageTokens;
    int steps_last = last_at / kPageTokens - j_lo + 1;           // of the last tile; an earlier one may see less
    int steps_first = n_tiles == 2 ? (start + (row_begin + BQ - 1) / a.group) / kPageTokens - j_lo + 1 : steps_last;
    if (a.splits > 1) {                                          // this block's share of them
        const int share = max(kLeastSteps, (steps_last + a.splits - 1) / a.splits);
        j_lo += split * share;
        steps_first = min(max(steps_first - split * share, 0), share);
        steps_last = min(steps_last - split * share, share);
        if (steps_last <= 0) {                                   // nothing left for it
            chain_wait();
            if (threadIdx.x < 2 * BQ && row_begin + (int)threadIdx.x < n_rows) {
                const int row = row_begin + threadIdx.x;
                a.part_stats[((size_t)(q_begin + row / a.group) * a.n_heads + h * a.group + row % a.group) * a.splits + split] = make_float2(-INFINITY, 0.f);
            }
            return;
        }
    }
    auto page_not_whole = [&](int j) {                           // a page that not every query of the block sees whole
        return j * kPageTokens + kPageTokens - 1 > first_at || (a.window > 0 && j * kPageTokens <= last_at - a.window);
    };

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full(t), 4);
            mbar_init(s_free(t), 4);
            mbar_init(s_full(t), 1);
            for (int i = 0; i < 2; ++i) { mbar_init(p_full(t, i), 4); mbar_init(pv_done(t, i), 1); }
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full(i), kKeyWarps);
            mbar_init(k_free(i), n_tiles);
            mbar_init(v_full(i), kValueWarps);
            mbar_init(v_free(i), n_tiles);
        }
        *abort_flag = 0;
        *odd_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::);
    }
    if (warp == kScoreWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(smem_addr(tmem_holder)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
    const uint32_t tmem = *tmem_holder;
    chain_wait();                                                // queries and the newest rows come from the kernel before
    chain_release();
    // (a wait's answer is the whole warp's before anything is issued: an elected lane waits for all)
    auto all_wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_sleep<kTest>(bar, parity, abort_flag)); };

    // 2^(w - kMostApart), w the largest value scale's logarithm among the block's pages: smaller ones are raised to it.  (A warp's
    // answer; the scales are powers of two from 2^-126 on.)
    auto least_value_scale = [&]() {
        uint32_t top = 0;
#pragma unroll 4
        for (int i = lane; i < steps_last; i += 32)
            top = max(top, __float_as_uint(kv.scales[(size_t)table[j_lo + i] * kv.scale_stride + kv.n_kv + h]));
        top = __reduce_max_sync(0xffffffffu, top);
        return __uint_as_float(max(top, (uint32_t)(kMostApart + 1) << 23) - ((uint32_t)kMostApart << 23));
    };

    // ---- codes to halves: two warps the keys, two the values
    auto convert = [&](auto of_values, const int t) {
        constexpr bool values = decltype(of_values)::value;
        constexpr int threads = 32 * (values ? kValueWarps : kKeyWarps), mine = (BK * HD / 16 + threads - 1) / threads;
        const int pieces = BK * hd / 16, row_pieces = hd / 16;   // of 16 codes in a step's keys (or values), in a key
        const int total = start + q_len;                         // rows that exist after this step
        // The codes come straight to registers, a step ahead of their use (through shared memory, several steps ahead, they
        // cost it the traffic that the products want).  Page numbers are read 32 steps at a time.
        int pages = 0;                                           // lane l: page of step (fetched / 32 * 32 + l)
        const uint8_t* source = (values ? kv.v : kv.k) + (size_t)h * kPageTokens * hd + t * 16;
        const long long stride = values ? kv.v_stride : kv.k_stride;
        uint4 u[mine];
        const float v_least = values ? least_value_scale() : 0.f;
        float v_scales = 1.f;                                    // lane l: of step (i / 32 * 32 + l)
        auto fetch = [&](int i) {
            if ((i & 31) == 0) pages = i + lane < steps_last ? table[j_lo + i + lane] : 0;
            const uint8_t* at = source + (size_t)__shfl_sync(0xffffffffu, pages, i & 31) * stride;
#pragma unroll
            for (int m = 0; m < mine; ++m)
                if (t + threads * m < pieces) u[m] = *reinterpret_cast<const uint4*>(at + threads * m * 16);
        };
        fetch(0);
        for (int i = 0; i < steps_last; ++i) {
            const int j = j_lo + i;
            if (values && page_not_whole(j)) {
                // Rows nobody has written yet become zeros; so do NaN codes, which P's zeros would not silence: who does see them
                // gets them back at the end.
#pragma unroll
                for (int m = 0; m < mine; ++m) {
                    const int at = j * kPageTokens + (t + threads * m) % 4 * 16;                // rows at .. at + 15
                    uint32_t w[4] = {u[m].x, u[m].y, u[m].z, u[m].w};
                    uint32_t found = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int there = min(max(total - at - 4 * c, 0), 4);                   // rows of this word that exist
                        w[c] &= there == 4 ? 0xffffffffu : (1u << (8 * there)) - 1u;
                        const uint32_t nan = nan_codes(w[c]);
                        found |= nan;
                        w[c] &= ~nan;
                    }
                    if (found && t + threads * m < pieces) *odd_flag = 1;
                    u[m] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            if (values) {
                if ((i & 31) == 0 && i + lane < steps_last) v_scales = kv.scales[(size_t)table[j + lane] * kv.scale_stride + kv.n_kv + h];
                const float v_scale = __shfl_sync(0xffffffffu, v_scales, i & 31);
                if (v_scale < v_least) {                         // counted as larger than they are: the codes make up for it
#pragma unroll
                    for (int m = 0; m < mine; ++m) u[m] = smaller_codes(u[m], v_scale * pow2_inverse(v_least));
                }
            }
            if (i >= 2 && !all_wait(values ? v_free(i) : k_free(i), phase(i - 2))) break;
            const uint32_t tile = base + (values ? S::kOffV : S::kOffK) + (i & 1) * S::kTileBytes;
#pragma unroll
            for (int m = 0; m < mine; ++m) {
                const int id = t + threads * m;
                if (id >= pieces) continue;
                if (values) store_halves(tile + id / 4 * 128, id % 4 * 2, id / 4 & 7, u[m]);
                else {
                    const int row = id / row_pieces, piece = id - row * row_pieces;
                    store_halves(tile + piece / 4 * (BK * 128) + row * 128, piece % 4 * 2, row & 7, u[m], piece / 4);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0 && !Waits<kTest>::kSkipCopies) mbar_arrive(values ? v_full(i) : k_full(i));
            if (i + 1 < steps_last) fetch(i + 1);
        }
    };
    if (warp >= 8 + kKeyWarps && warp < kScoreWarp) {
        convert(std::true_type(), (int)threadIdx.x - 32 * (8 + kKeyWarps));
    } else if (warp >= 8 && warp < kScoreWarp) {
        convert(std::false_type(), (int)threadIdx.x - 32 * 8);
    } else if (warp >= kScoreWarp) {
        // ------------------------------------------------------------ products: a warp a tile for the scores, another for P V.
        // A tile that sees fewer pages than the block's last one lets the rest of its tiles' places go as they come.
        const int t = (warp - kScoreWarp) & 1;
        const int n_steps = t == n_tiles - 1 ? steps_last : steps_first;
        if (t >= n_tiles) {
        } else if (warp < kOutputWarp) {
            constexpr uint32_t idesc = f16_idesc(BQ, BK);
            const uint64_t dq = umma_desc(base + t * S::kQBytes), k_desc = umma_desc(base + S::kOffK);
            bool ok = all_wait(q_full(t), 0);
            for (int i = 0; i < steps_last && ok; ++i) {
                ok = all_wait(k_full(i), phase(i));
                if (!ok) break;
                if (i >= n_steps) {
                    if (lane == 0) mbar_arrive(k_free(i));
                    continue;
                }
                if (i > 0) ok = all_wait(s_free(t), (uint32_t)(i - 1) & 1u);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                const uint64_t dk = k_desc + (uint64_t)((i & 1) * (S::kTileBytes >> 4));
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    if (kExact || kk < hd / 16) warp_umma_ss(tmem + t * kTileCols, dq + (kk / 4) * (BQ * 128 >> 4) + 2 * (kk % 4), dk + (kk / 4) * (BK * 128 >> 4) + 2 * (kk % 4), idesc,
                                 kk > 0 ? 1u : 0u);
                warp_umma_commit(s_full(t));
                warp_umma_commit(k_free(i));
            }
        } else {
            const uint32_t idesc = f16_idesc(BQ, hd);
            const uint64_t v_desc = umma_desc(base + S::kOffV);
            bool ok = true;
            for (int i = 0; i < steps_last && ok; ++i) {
                ok = all_wait(v_full(i), phase(i));
                if (!ok) break;
                if (i >= n_steps) {
                    if (lane == 0) mbar_arrive(v_free(i));
                    continue;
                }
                ok = all_wait(p_full(t, i), phase(i));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                const uint64_t dv = v_desc + (uint64_t)((i & 1) * (S::kTileBytes >> 4));
                const uint32_t p_at = tmem + t * kTileCols + S::kColP + 32 * (i & 1);
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) warp_umma_ts(tmem + t * kTileCols + S::kColO, p_at + 8 * kk, dv + 2 * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
                warp_umma_commit(pv_done(t, i));
                warp_umma_commit(v_free(i));
            }
        }
    } else if (warp / 4 < n_tiles) {
        // ------------------------------------------------------------ softmax and output: a thread a query row
        const unsigned full = 0xffffffffu;
        const int tt = warp >> 2, r = (warp & 3) * 32 + lane;
        const int row0 = row_begin + tt * BQ, n_steps = tt == n_tiles - 1 ? steps_last : steps_first;
        const bool real = row0 + r < n_rows;
        const int token = (row0 + (real ? r : 0)) / a.group, head = h * a.group + (row0 + (real ? r : 0)) % a.group;
        const int pos = start + token;                            // the query's own cache row
        const uint32_t tile_at = tmem + tt * kTileCols + ((uint32_t)((warp & 3) * 32) << 16);
        float factor;                                             // a raw score times this and the page's key scale: powers of two
        {
            const bf16* src = a.q + (size_t)(q_begin + token) * a.ldq + (size_t)head * hd;
            uint4 u[HD / 8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                u[c] = real && (kExact || 8 * c < hd) ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = fabsf(__uint_as_float(w[e] << 16)), hi = fabsf(__uint_as_float(w[e] & 0xffff0000u));
                    most = fmaxf(most, fmaxf(finite_f32(lo) ? lo : 0.f, finite_f32(hi) ? hi : 0.f));
                }
            }
            // the largest channel comes to lie in [2^14, 2^15); a negative scale turns the queries round
            const int e = (int)(__float_as_uint(most) >> 23);
            const int up = e == 0 ? 0 : min(14 - (e - 127), 100);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23) * (a.scale < 0.f ? -1.f : 1.f);
            factor = fmaxf(fabsf(a.scale) * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23), 1e-37f);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
                uint32_t o[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const __half2 hh = __floats2half2_rn(__uint_as_float(w[x] << 16) * f, __uint_as_float(w[x] & 0xffff0000u) * f);
                    o[x] = *reinterpret_cast<const uint32_t*>(&hh);
                }
                store_shared16(base + tt * S::kQBytes + (c / 8) * (BQ * 128) + r * 128 + (((c % 8) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(tt));
        }
        const float v_least = least_value_scale();
        const uint32_t top_bits = __float_as_uint(v_least) + ((uint32_t)(kMostApart + 127) << 23);             // 1 / s = top_bits - bits of s, times 2^w
        // scales, 32 steps at a time: lane l has those of step (i / 32 * 32 + l)
        float k_scales = 0.f, v_scales = 1.f;
        float m_run = -INFINITY, l_run = 0.f;
        // What M is the sum of, score and v, touched only where M is raised or large.  In registers where there is room (prompt of
        // 2,048 tokens, 32 heads of 64: 54.4 us, else 55.9), else in shared memory (chunks of 512, 128 channels: 166 us, else 175).
        float2 registers;
        float2* made_of = HD == 64 ? &registers : reinterpret_cast<float2*>(smem + S::kOffM) + tt * BQ + r;
        *made_of = make_float2(-INFINITY, 0.f);
        uint32_t sv[BK];
        bool ok = true;
        for (int i = 0; i < n_steps; ++i) {
            const int key0 = (j_lo + i) * kPageTokens;
            if ((i & 31) == 0 && i + lane < n_steps) {
                const float* at = kv.scales + (size_t)table[j_lo + i + lane] * kv.scale_stride + h;
                k_scales = at[0];
                v_scales = fmaxf(at[kv.n_kv], v_least);
            }
            // the step's scores; and the P of two steps ago has been read
            ok = i < 2 ? all_wait(s_full(tt), (uint32_t)i & 1u)
                       : (bool)__all_sync(full, mbar_sleep_both<kTest>(s_full(tt), (uint32_t)i & 1u, pv_done(tt, i), phase(i - 2), abort_flag));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
            tmem_ld32(tile_at, sv);
            tmem_ld32(tile_at + 32, sv + 32);
            const float sl = fmaxf(factor * __shfl_sync(full, k_scales, i & 31), 1e-37f);       // (not 0, which would make NaN of masked scores)
            const float v_scale = __shfl_sync(full, v_scales, i & 31);
            const float add = (float)((int)(__float_as_uint(v_scale) >> 23) - 127);             // log2 of the value scale
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free(tt));              // the scores are in registers: the tile takes the next step's
            if (!(key0 + BK - 1 <= pos && (a.window <= 0 || key0 > pos - a.window))) {
                const int hi = pos - key0, lo = a.window > 0 ? pos - a.window - key0 : -1;       // columns lo + 1 .. hi are seen
#pragma unroll
                for (int c = 0; c < BK; ++c)
                    if (c > hi || c <= lo) sv[c] = __float_as_uint(-INFINITY);
            }
            // P against the maximum so far, without looking for the step's own: if none of the 64 exceeds 2^15 no sum of
            // them does that half could not hold.  Only where the sum does -- and for a row that has seen nothing yet -- is
            // the maximum found and the step done again.
            uint32_t pw[BK / 2];
            uint64_t sum;
            auto exponentials = [&](float mult, float shift) {
                const uint64_t sl2 = two(mult, mult), shift2 = two(shift, shift);
                uint64_t sums[4] = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < BK; c += 8) {
                    uint64_t x[4];
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = fma2(two(__uint_as_float(sv[c + 2 * e]), __uint_as_float(sv[c + 2 * e + 1])), sl2, shift2);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { p[2 * e] = exp2_in_order(first_of(x[e])); p[2 * e + 1] = exp2_in_order(second_of(x[e])); }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sums[e] = add2(sums[e], two(p[2 * e], p[2 * e + 1]));
                        const __half2 hh = __floats2half2_rn(p[2 * e], p[2 * e + 1]);
                        pw[c / 2 + e] = *reinterpret_cast<const uint32_t*>(&hh);
                    }
                }
                sum = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
            };
            const bool careful = __any_sync(full, fabsf(m_run) > kLargeScore);       // (-infinity: a row that has seen nothing)
            if (!careful) exponentials(sl, add - m_run + kPShift);
            if (careful || __any_sync(full, first_of(sum) + second_of(sum) > kMostSum)) {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < BK; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sv[c + e]), __uint_as_float(sv[c + 4 + e]));
                const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), m_step = fmaf(top, sl, add), score = __fmul_rn(top, sl);
                const bool apart = fabsf(m_run) > kLargeScore || fabsf(m_step) > kLargeScore;
                float up = m_step - m_run;                        // how much larger this step's is
                if (apart) up = (score - made_of->x) + (add - made_of->y);
                float corr = 1.0f;
                if (up > 0.f) {
                    corr = fast_exp2(-up);                        // 0 for a row that has seen nothing
                    m_run = m_step;
                    *made_of = make_float2(score, add);
                    l_run *= corr;
                }
                if (i > 0) {                                      // O may only be touched between products
                    ok = all_wait(pv_done(tt, i - 1), phase(i - 1));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
#pragma unroll 1
                    for (int part = 0; part < hd / 8; ++part) {
                        uint32_t ov[8];
                        tmem_ld8(tile_at + S::kColO + 8 * part, ov);
                        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                        for (int d = 0; d < 8; ++d) ov[d] = __float_as_uint(__uint_as_float(ov[d]) * corr);
                        tmem_st8(tile_at + S::kColO + 8 * part, ov);
                    }
                }
                const float m_use = m_run == -INFINITY ? 0.f : m_run;
                float mult = sl, shift = add - m_use + kPShift;
                if (__any_sync(full, fabsf(m_use) > kLargeScore)) {
                    const float from = made_of->x == -INFINITY ? 0.f : made_of->x, apart_by = add - made_of->y;
#pragma unroll
                    for (int c = 0; c < BK; ++c) sv[c] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(sv[c]), sl), from) + apart_by);
                    mult = 1.0f;
                    shift = kPShift;
                }
                exponentials(mult, shift);
            }
            l_run = fmaf(first_of(sum) + second_of(sum), __uint_as_float(top_bits - __float_as_uint(v_scale)), l_run);
            tmem_st32(tile_at + S::kColP + 32 * (i & 1), pw);
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(tt, i));
        }
        if (ok && n_steps > 0) ok = all_wait(pv_done(tt, n_steps - 1), phase(n_steps - 1));
        if (ok) {
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
            const float inv = 1.0f / l_run, unit = __uint_as_float(__float_as_uint(v_least) + ((uint32_t)kMostApart << 23));    // 2^w
            // P = 2^(score - s + v_j - v + 7), v that of M, and the probability is P 2^(w - v_j) / l
            const float2 stat = make_float2(made_of->x, (float)((int)(__float_as_uint(unit) >> 23) - 127) + kPShift - made_of->y - log2f(l_run));
            const size_t at = (size_t)(q_begin + token) * a.n_heads + head;
            const bool in_parts = a.splits > 1;
            if (real && in_parts) a.part_stats[at * a.splits + split] = stat;
            else if (real && a.stats) a.stats[at] = stat;
            float* part = in_parts ? a.part_o + (at * a.splits + split) * hd : nullptr;
            bf16* dst = a.out + (size_t)(q_begin + token) * a.ldo + (size_t)head * hd;
            const bool odd = *odd_flag != 0;
#pragma unroll 1
            for (int c = 0; 32 * c < hd && n_steps > 0; ++c) {
                tmem_ld32(tile_at + S::kColO + 32 * c, sv);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                if (odd && real) {
                    // NaN codes of rows that this query sees, in pages where they were taken out
                    for (int j = j_lo; j < j_lo + n_steps; ++j) {
                        if (!page_not_whole(j)) continue;
                        const uint8_t* vp = kv.v + (size_t)table[j] * kv.v_stride + ((size_t)h * hd + 32 * c) * kPageTokens;
                        const int lo = a.window > 0 ? max(0, pos - a.window + 1 - j * kPageTokens) : 0, hi = min(pos - j * kPageTokens, kPageTokens - 1);
                        for (int row = lo; row <= hi; ++row)
#pragma unroll
                            for (int d = 0; d < 32; ++d)
                                if ((kExact || 32 * c + d < hd) && (vp[d * kPageTokens + row] & 0x7f) == 0x7f) sv[d] = 0x7fc00000u;
                    }
                }
                if (real && in_parts) {
#pragma unroll
                    for (int piece = 0; piece < 8; ++piece) {
                        if (!kExact && 32 * c + 4 * piece >= hd) break;
                        float o4[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) o4[x] = __uint_as_float(sv[4 * piece + x]) * inv * unit;
                        *reinterpret_cast<float4*>(part + 32 * c + 4 * piece) = make_float4(o4[0], o4[1], o4[2], o4[3]);
                    }
                } else if (real) {
#pragma unroll
                    for (int piece = 0; piece < 4; ++piece) {
                        if (!kExact && 32 * c + 8 * piece >= hd) break;
                        uint32_t o4[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const __nv_bfloat162 hh = __floats2bfloat162_rn(__uint_as_float(sv[8 * piece + 2 * x]) * inv * unit, __uint_as_float(sv[8 * piece + 2 * x + 1]) * inv * unit);
                            o4[x] = *reinterpret_cast<const uint32_t*>(&hh);
                        }
                        *reinterpret_cast<uint4*>(dst + 32 * c + 8 * piece) = make_uint4(o4[0], o4[1], o4[2], o4[3]);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    if (warp == kScoreWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols));
    }
}

// Joins the blocks that shared a tile pair's pages: their results, each with the mass 2^(s - c) that its statistics say, relative to
// the largest.  s and c are subtracted apart: next to a large s c would be lost.
__global__ void __launch_bounds__(256)
e4m3_prompt_join_kernel(const PromptArgs a, int B, int N, int hd) {
    chain_release();
    chain_wait();
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int lanes = hd / 4, d = (int)(id % lanes) * 4;         // four channels a thread
    const long long row = id / lanes;
    const int token = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    if (token >= N || token < a.cu_seqlens[0] || token >= a.cu_seqlens[B]) return;
    const float2* stats = a.part_stats + row * a.splits;
    const float* o = a.part_o + row * a.splits * hd + d;
    float2 top = make_float2(-INFINITY, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float2 st = stats[s];
        if (st.x != -INFINITY && !(st.x - st.y <= top.x - top.y)) top = st;
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float mass = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float2 st = stats[s];
        const float4 v = *reinterpret_cast<const float4*>(o + (size_t)s * hd);
        if (st.x == -INFINITY) continue;
        const float f = fast_exp2(min_or_nan((st.x - top.x) - (st.y - top.y), 64.f));     // (above 0 only as far as the choice was rounded)
        mass += f;
        acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
    }
    const float inv = 1.0f / mass;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(a.out + (size_t)token * a.ldo + (size_t)head * hd + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    if (a.stats && d == 0) a.stats[row] = make_float2(top.x, top.y - log2f(mass));
}

template <int HD, bool kExact, bool kTest>
int launch(const PromptArgs& a, const E4M3Pages& kv, int B, int max_q_len, cudaStream_t stream) {
    static bool allowed[kMaxDevices] = {};
    const int set = allow_shared((const void*)attention_e4m3_prompt_kernel<HD, kExact, kTest>, Shape<HD>::kSmemBytes, allowed);
    if (set != 0) return set;
    const long long rows = (long long)max_q_len * a.group;
    return launch_chained(attention_e4m3_prompt_kernel<HD, kExact, kTest>, dim3(kv.n_kv, B, (unsigned)((rows + 2 * BQ - 1) / (2 * BQ) * a.splits)), dim3(kThreads),
                          (size_t)Shape<HD>::kSmemBytes, stream, a, kv);
}
// ============================================================== gathered weights of prompts and chunks
// weight_j += sum over the queries that see row j, of all heads of the group, of 2^(score - s + c), s and c the query's
// statistics that the attention left.  The products again, the other way round: one block per (128 rows of the cache, query
// head, sequence), the rows as the tile's rows, so that a thread owns a row and its sum:
//   K      converted once to bfloat16 into shared memory, S = K Q^T by tcgen05.mma 128 x 128 x head size.  Not the codes but the keys
//          they stand for, 2^-32 of them (exact: bfloat16 has float's range): queries come as they are, and the codes' products with
//          the largest of them, before the key scale makes them small, left float's range;
//   Q      128 tokens of one head at a time by tensor copies through a ring, as they are (bfloat16);
//   sums   four warps, S from tensor memory, c - s one number a query: one multiply-add, one exponential and one add a
//          score.  Tiles with a query whose |s| is large take a form of their own, in which a score that may be s is s (score_slack).
//          No unit is full (exponentials 42 % of theirs, issue slots 43 %):
//          a sub-partition has one such warp a block, two in all, which reads 32 columns, waits for them, and adds.
// A block a head of the group leaves its sums beside the others', and a second kernel adds them in the heads' order (a block for
// all heads: one block's 48 tiles were the time of all, 95 us of 147 for prompts of 200 to 1,500 tokens).  So a weight does
// not depend on what else runs.
constexpr int kWeightCols = 256;
constexpr int kWeightThreads = 192;                      // sums 0-3, copies 4, products 5
template <int HD> struct WeightShape {
    static constexpr int kStages = HD == 64 ? 3 : 2;
    static constexpr int kTileBytes = 128 * HD * 2;      // 128 rows of keys, or of queries
    static constexpr int kOffQ = kTileBytes, kOffY = kOffQ + kStages * kTileBytes, kOffC = kOffY + 2 * 128 * 4, kOffBar = kOffC + 2 * 128 * 8;
    static constexpr int kSmemBytes = kOffBar + 256;
};

// What a block's codes are multiplied with there: 2^-32 times its scale 2^k, and 2^-100 at least, so that codes of 2^-9 are still
// normal numbers.
__device__ __forceinline__ float key_factor(float k_scale) {
    return __int_as_float(max((int)(__float_as_uint(k_scale) & 0x7f800000u) - (32 << 23), 27 << 23));
}
// Four codes times a power of two as four bfloat16.
__device__ __forceinline__ void bf16_of_codes(uint32_t w, float times, uint32_t& lo, uint32_t& hi) {
    const uint32_t a = e4m3_pair_f16(w), b = e4m3_pair_f16(w >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    const __nv_bfloat162 p = __floats2bfloat162_rn(x.x * times, x.y * times), r = __floats2bfloat162_rn(y.x * times, y.y * times);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&r);
}

// parts: [sequence][query head][part_rows]; rows behind part_rows (a sequence that has outgrown the plan) are done for all heads
// by the block of the group's first.
template <int HD, bool kExact, bool kTest>
__global__ void __launch_bounds__(kWeightThreads, 2)
e4m3_weights_kernel(const __grid_constant__ CUtensorMap map_q, const PromptArgs a, const E4M3Pages kv, float* __restrict__ parts, int part_rows) {
    using S = WeightShape<HD>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int h = blockIdx.y / a.group, g0 = blockIdx.y % a.group, b = blockIdx.z, hd = kExact ? HD : kv.hd;
    const int q_begin = a.cu_seqlens[b];
    const int q_len = a.cu_seqlens[b + 1] - q_begin;
    const int slot = a.slots[b];
    const int start = a.start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    if (q_len <= 0 || (int)blockIdx.x * 128 >= start + q_len) {
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0) chain_wait();     // as above
        return;
    }
    const uint32_t base = smem_addr(smem);
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicExch(&g_status, 2);
        return;
    }
    const uint32_t bars = base + S::kOffBar;
    const uint32_t k_full = bars;
    auto q_full = [&](int s) { return bars + 8u + 8u * s; };
    auto q_free = [&](int s) { return bars + 32u + 8u * s; };
    auto s_full = [&](int s) { return bars + 56u + 8u * s; };
    auto s_free = [&](int s) { return bars + 72u + 8u * s; };
    auto y_full = [&](int s) { return bars + 88u + 8u * s; };
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::kOffBar + 128);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffBar + 136);
    volatile int* large_tile = reinterpret_cast<volatile int*>(smem + S::kOffBar + 144);     // by buffer: 1 + the last tile with a large |s|
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int* table = kv.block_table + (size_t)slot * kv.table_stride;
    if (threadIdx.x == 0) {
        mbar_init(k_full, 4);
        for (int s = 0; s < S::kStages; ++s) { mbar_init(q_full(s), 1); mbar_init(q_free(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(s_full(s), 1); mbar_init(s_free(s), 4); mbar_init(y_full(s), 4); large_tile[s] = 0; }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::);
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(smem_addr(tmem_holder)), "r"(kWeightCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
    const uint32_t tmem = *tmem_holder;
    chain_wait();
    chain_release();

    // the tokens that see any of rows 128 kt .. 128 kt + 127: [t_lo, t_hi), cut into tiles for each of this block's heads
    struct Span { int t_lo, t_hi, per_head, heads; };
    auto span_of = [&](int kt) {
        Span s;
        s.heads = kt * 128 < part_rows ? 1 : g0 == 0 ? a.group : 0;
        s.t_lo = max(0, kt * 128 - start);
        s.t_hi = a.window > 0 ? min((long long)q_len, (long long)kt * 128 + 127 + a.window - start) : q_len;
        s.per_head = s.t_hi > s.t_lo && s.heads > 0 ? (s.t_hi - s.t_lo + 127) / 128 : 0;
        return s;
    };
    int n = 0;                                                   // tiles so far, of all turns
    if (warp == 4) {
        if (lane == 0) {
            bool ok = true;
            for (int kt = blockIdx.x; kt * 128 < start + q_len && ok; kt += gridDim.x) {
                const Span sp = span_of(kt);
                for (int i = 0; i < sp.per_head * sp.heads; ++i, ++n) {
                    const int s = n % S::kStages;
                    ok = mbar_sleep<kTest>(q_free(s), (((uint32_t)n / S::kStages) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    mbar_expect_tx(q_full(s), S::kTileBytes);
                    for (int hh = 0; hh < HD / 64; ++hh)
                        tma_load_2d<kTest>(base + S::kOffQ + s * S::kTileBytes + hh * (128 * 128), &map_q, (h * a.group + g0 + i / sp.per_head) * hd + 64 * hh,
                                           q_begin + sp.t_lo + i % sp.per_head * 128, q_full(s));
                }
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc(128, 128, 0);
            bool ok = true;
            for (int kt = blockIdx.x, turn = 0; kt * 128 < start + q_len && ok; kt += gridDim.x) {
                const Span sp = span_of(kt);
                if (sp.per_head == 0) continue;                  // (rows that no query sees: no role takes a turn for them)
                ok = mbar_sleep<kTest>(k_full, (uint32_t)turn++ & 1u, abort_flag);
                for (int i = 0; i < sp.per_head * sp.heads && ok; ++i, ++n) {
                    const int s = n % S::kStages, buf = n & 1;
                    ok = mbar_sleep<kTest>(q_full(s), ((uint32_t)n / S::kStages) & 1u, abort_flag) &&
                         mbar_sleep<kTest>(s_free(buf), (((uint32_t)n >> 1) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                    const uint32_t qbase = base + S::kOffQ + s * S::kTileBytes;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {              // (a copy of a head's queries may hold the next one's behind them)
                        if (!kExact && kk >= hd / 16) break;
                        const uint64_t dk = umma_desc(base + (kk / 4) * (128 * 128)) + 2 * (kk % 4);
                        const uint64_t dq = umma_desc(qbase + (kk / 4) * (128 * 128)) + 2 * (kk % 4);
                        umma_ss(tmem + 128 * buf, dk, dq, idesc, kk > 0 ? 1u : 0u);
                    }
                    umma_commit(q_free(s));
                    umma_commit(s_full(buf));
                }
            }
        }
    } else {
        const unsigned full = 0xffffffffu;
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        float* y = reinterpret_cast<float*>(smem + S::kOffY);                           // by buffer and column: c - s,
        float2* apart = reinterpret_cast<float2*>(smem + S::kOffC);                     // and s and c
        const int r = threadIdx.x;                               // row of the tile; also a column of the next tile's statistics
        bool ok = true;
        for (int kt = blockIdx.x; kt * 128 < start + q_len && ok; kt += gridDim.x) {
            const Span sp = span_of(kt);
            const int tiles = sp.per_head * sp.heads;
            const int row = kt * 128 + r;
            const bool there = row < start + q_len, in_parts = kt * 128 < part_rows;
            float* part = parts + ((size_t)b * a.n_heads + blockIdx.y) * part_rows + row;
            if (tiles == 0) {
                if (in_parts) *part = 0.f;
                continue;
            }
            // ---- the tile's keys (all products of the turn before are complete: this warp has seen the last one's barrier)
            const bool both = (kt * 2 + 1) * kPageTokens < start + q_len;                       // the tile's second page exists too
            const size_t pages[2] = {(size_t)table[kt * 2], both ? (size_t)table[kt * 2 + 1] : 0};
            const float k_scales[2] = {kv.scales[pages[0] * kv.scale_stride + h], both ? kv.scales[pages[1] * kv.scale_stride + h] : 0.f};
            uint4 u[HD / 16];
#pragma unroll
            for (int m = 0; m < HD / 16; ++m) {                  // (all asked for before the first is waited for)
                u[m] = make_uint4(0, 0, 0, 0);
                if (!kExact && m >= hd / 16) continue;
                const int id = r + 128 * m, key = id / (hd / 16), piece = id - key * (hd / 16);
                if (key < kPageTokens || both)
                    u[m] = *reinterpret_cast<const uint4*>(kv.k + (key < kPageTokens ? pages[0] : pages[1]) * kv.k_stride +
                                                           ((size_t)h * kPageTokens + key % 64) * hd + piece * 16);
            }
            const float times[2] = {key_factor(k_scales[0]), key_factor(k_scales[1])};
#pragma unroll
            for (int m = 0; m < HD / 16; ++m) {
                if (!kExact && m >= hd / 16) break;
                const int id = r + 128 * m, key = id / (hd / 16), piece = id - key * (hd / 16);
                uint32_t o[8];
                bf16_of_codes(u[m].x, key < kPageTokens ? times[0] : times[1], o[0], o[1]);
                bf16_of_codes(u[m].y, key < kPageTokens ? times[0] : times[1], o[2], o[3]);
                bf16_of_codes(u[m].z, key < kPageTokens ? times[0] : times[1], o[4], o[5]);
                bf16_of_codes(u[m].w, key < kPageTokens ? times[0] : times[1], o[6], o[7]);
                const uint32_t at = base + (piece / 4) * (128 * 128) + key * 128;
                store_shared16(at + (((piece % 4 * 2) ^ (key & 7)) << 4), o[0], o[1], o[2], o[3]);
                store_shared16(at + (((piece % 4 * 2 + 1) ^ (key & 7)) << 4), o[4], o[5], o[6], o[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full);
            const size_t page = r < kPageTokens ? pages[0] : pages[1];
            const float k_scale = r < kPageTokens ? k_scales[0] : k_scales[1];
            const float f = there ? a.scale * kLog2e * (k_scale * pow2_inverse(key_factor(k_scale))) : 0.f;
            auto statistic = [&](int i) {                        // of tile i's column r
                const int token = sp.t_lo + i % sp.per_head * 128 + r;
                if (i >= tiles || token >= sp.t_hi) return make_float2(0.f, 0.f);
                return a.stats[(size_t)(q_begin + token) * a.n_heads + h * a.group + g0 + i / sp.per_head];
            };
            float2 mine = statistic(0);
            float total = 0.f;
            for (int i = 0; i < tiles; ++i, ++n) {
                const int buf = n & 1;
                y[128 * buf + r] = mine.y - mine.x;
                apart[128 * buf + r] = mine;
                if (fabsf(mine.x) > kLargeScore) large_tile[buf] = n + 1;
                __syncwarp();
                if (lane == 0) mbar_arrive(y_full(buf));
                mine = statistic(i + 1);
                ok = __all_sync(full, mbar_sleep<kTest>(y_full(buf), ((uint32_t)n >> 1) & 1u, abort_flag) &&
                                          mbar_sleep<kTest>(s_full(buf), ((uint32_t)n >> 1) & 1u, abort_flag));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                const int t0 = sp.t_lo + i % sp.per_head * 128;
                // columns [lo, hi) of the tile are tokens that see this row
                const int lo = max(row - start - t0, 0);
                const long long past = min((long long)sp.t_hi, a.window > 0 ? (long long)row + a.window - start : (long long)sp.t_hi) - t0;
                const int hi = (int)min(past, 128LL);
                const bool whole = __all_sync(full, lo == 0 && hi == 128);
                const float* yt = y + 128 * buf;
                const float4* at = reinterpret_cast<const float4*>(apart + 128 * buf);
                uint64_t sum[2] = {0, 0};
                auto add_up = [&](auto masked, auto large) {
                    const uint64_t f2 = two(f, f);
#pragma unroll 1
                    for (int c = 0; c < 128; c += 32) {
                        uint32_t sv[32];
                        tmem_ld32(tmem + 128 * buf + lane_off + c, sv);
                        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 y4 = *reinterpret_cast<const float4*>(yt + c + e);
                            uint64_t x[2] = {fma2(two(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), f2, two(y4.x, y4.y)),
                                             fma2(two(__uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3])), f2, two(y4.z, y4.w))};
                            if constexpr (decltype(large)::value) {
                                auto exponent = [&](uint32_t score, float s, float own) {
                                    const float d = fmaf(__uint_as_float(score), f, -s);
                                    return own + (fabsf(d) <= score_slack(s) ? 0.f : d);
                                };
                                const float4 a = at[(c + e) / 2], b = at[(c + e) / 2 + 1];
                                x[0] = two(exponent(sv[e], a.x, a.y), exponent(sv[e + 1], a.z, a.w));
                                x[1] = two(exponent(sv[e + 2], b.x, b.y), exponent(sv[e + 3], b.z, b.w));
                            }
                            // (no probability is above 1: the bound is for what scores' roundings leave)
                            float p[4] = {fast_exp2(min_or_nan(first_of(x[0]), 0.f)), fast_exp2(min_or_nan(second_of(x[0]), 0.f)),
                                          fast_exp2(min_or_nan(first_of(x[1]), 0.f)), fast_exp2(min_or_nan(second_of(x[1]), 0.f))};
                            if constexpr (decltype(masked)::value) {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (c + e + i < lo || c + e + i >= hi) p[i] = 0.f;
                            }
                            sum[0] = add2(sum[0], two(p[0], p[1]));
                            sum[1] = add2(sum[1], two(p[2], p[3]));
                        }
                    }
                };
                if (large_tile[buf] == n + 1) add_up(std::true_type(), std::true_type());
                else if (whole) add_up(std::false_type(), std::false_type());
                else add_up(std::true_type(), std::false_type());
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free(buf));
                sum[0] = add2(sum[0], sum[1]);
                total += first_of(sum[0]) + second_of(sum[0]);
            }
            if (ok && in_parts) *part = total;
            else if (ok && there) kv.weights[page * kv.weight_stride + (size_t)h * kPageTokens + row % kPageTokens] += total;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    if (warp == 5) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kWeightCols));
    }
}

// The heads' parts added up, in the heads' order.
__global__ void __launch_bounds__(256)
e4m3_weights_sum_kernel(const PromptArgs a, const E4M3Pages kv, const float* __restrict__ parts, int part_rows) {
    chain_release();
    chain_wait();
    const int row = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int slot = a.slots[b], q_len = a.cu_seqlens[b + 1] - a.cu_seqlens[b];
    const int start = a.start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    if (q_len <= 0 || row >= part_rows || row >= start + q_len) return;
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) sum += parts[((size_t)b * a.n_heads + h * a.group + g) * part_rows + row];
    const size_t page = kv.block_table[(size_t)slot * kv.table_stride + row / kPageTokens];
    kv.weights[page * kv.weight_stride + (size_t)h * kPageTokens + row % kPageTokens] += sum;
}

template <int HD, bool kExact, bool kTest>
int launch_weights(const PromptArgs& a, const E4M3Pages& kv, const CUtensorMap& map_q, int B, int max_kv_len, float* parts, cudaStream_t stream) {
    static bool allowed[kMaxDevices] = {};
    const int set = allow_shared((const void*)e4m3_weights_kernel<HD, kExact, kTest>, WeightShape<HD>::kSmemBytes, allowed);
    if (set != 0) return set;
    const int part_rows = (max_kv_len + 127) / 128 * 128;
    const int st = launch_behind(e4m3_weights_kernel<HD, kExact, kTest>, dim3(part_rows / 128, a.n_heads, B), dim3(kWeightThreads),
                                  (size_t)WeightShape<HD>::kSmemBytes, stream, map_q, a, kv, parts, part_rows);
    if (st != 0) return st;
    return launch_behind(e4m3_weights_sum_kernel, dim3((part_rows + 255) / 256, kv.n_kv, B), dim3(256), 0, stream, a, kv, (const float*)parts, part_rows);
}
}  // namespace

GTG_API int gtg_attention_e4m3_tcgen05_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

// Heads of a multiple of 16 channels up to 128; bfloat16 rows of q and out on 16-byte boundaries.  splits: blocks that share the pages of
// 256 query rows.  scratch, in floats, on a 16-byte boundary: with several splits N n_heads splits (hd + 2); where the pages have
// weights, which then gather what their rows get, 2 N n_heads and n_heads B times max_kv_len rounded up to 128 more; else null.
GTG_API int gtg_attention_e4m3_tcgen05(const void* q, int ldq, void* out, int ldo, const E4M3Pages* pages, const int* cu_seqlens,
                                       const int* slots, const int* start_pos, int B, int max_q_len, int max_kv_len, int N, int n_heads,
                                       float scale, int window, int splits, float* scratch, cudaStream_t stream) {
    if (B <= 0 || max_q_len <= 0 || N <= 0) return 0;
    const E4M3Pages kv = *pages;
    const int n_kv = kv.n_kv, hd = kv.hd;
    float* weights = kv.weights;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || window < 0 || max_kv_len <= 0 || splits < 1 || ((weights || splits > 1) && !scratch)) return kErrBadArgument;
    if (n_heads > 65535) return kErrUnsupported;
    if (hd % 16 || hd > 128 || ldq % 8 || ldo % 8 || (uintptr_t)q % 16 || (uintptr_t)out % 16) return kErrUnsupported;
    if (B > 65535 || ((long long)max_q_len * (n_heads / n_kv) + BQ - 1) / BQ > 65535 / splits) return kErrUnsupported;
    PromptArgs a = {};
    a.q = (const bf16*)q; a.ldq = ldq; a.out = (bf16*)out; a.ldo = ldo;
    a.cu_seqlens = cu_seqlens; a.slots = slots; a.start_pos = start_pos;
    a.n_heads = n_heads; a.group = n_heads / n_kv; a.scale = scale; a.window = window;
    // scratch: results and statistics of splits, statistics, weights by head
    const size_t rows = (size_t)N * n_heads;
    a.splits = splits;
    a.part_o = scratch;
    a.part_stats = (float2*)(scratch + (splits > 1 ? rows * splits * hd : 0));
    a.stats = weights ? a.part_stats + (splits > 1 ? rows * splits : 0) : nullptr;
    float* parts = weights ? (float*)(a.stats + rows) : nullptr;
    const bool test = g_test_waits;
#define GTG_LAUNCH(WHAT, HD, EXACT, ...) (test ? WHAT<HD, EXACT, true>(__VA_ARGS__) : WHAT<HD, EXACT, false>(__VA_ARGS__))
#define GTG_BY_SIZE(WHAT, ...) (hd == 64 ? GTG_LAUNCH(WHAT, 64, true, __VA_ARGS__) : hd == 128 ? GTG_LAUNCH(WHAT, 128, true, __VA_ARGS__) \
                                : hd < 64 ? GTG_LAUNCH(WHAT, 64, false, __VA_ARGS__) : GTG_LAUNCH(WHAT, 128, false, __VA_ARGS__))
    int st = GTG_BY_SIZE(launch, a, kv, B, max_q_len, stream);
    if (st == 0 && splits > 1)
        st = launch_behind(e4m3_prompt_join_kernel, dim3((unsigned)((rows * (hd / 4) + 255) / 256)), dim3(256), 0, stream, a, B, N, hd);
    if (st != 0 || !weights) return st;
    CUtensorMap map_q;
    const int mt = make_map(&map_q, q, N, n_heads * hd, ldq, 128);
    if (mt != 0) return mt;
    return GTG_BY_SIZE(launch_weights, a, kv, map_q, B, max_kv_len, parts, stream);
#undef GTG_BY_SIZE
#undef GTG_LAUNCH
}

// For the test of the give-up path: while set, launches take the kTest form, in which the conversion's warps never say that a
// tile is there, so that every wait runs out after a thousand polls.  Clears the status word.
GTG_API int gtg_attention_e4m3_tcgen05_test_hooks(int test_waits) {
    const int zero = 0;
    cudaError_t e = cudaDeviceSynchronize();
    g_test_waits = test_waits != 0;
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    return (int)e;
}
