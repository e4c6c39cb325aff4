// Attention of few queries a sequence over the 8-bit cache: decode steps, and steps of a few tokens (up to kFewColumns
// queries -- tokens times the heads of a group -- a key/value head).
//
// What bounds it is reading the cache: 2 * head size bytes a row, each used for a few multiply-adds.  So the codes go
// from memory to the tensor cores as they are, once, and everything else is arranged around the order in which they lie.
//
//   * Both products multiply codes with codes: the cache's rows (or, in the second, its channels) are the M = 16 rows of an
//     e4m3 product, S^T = K Q^T and O^T = V^T P^T, and nothing of the cache is converted.  (A form that turned every pair of
//     codes into halves spent more than half of its instructions on that.)
//   * The other operand is split into codes that add up to it, each with columns of its own.  A bfloat16 query has 8 significant
//     bits, two codes of 4: q 2^a = hi + lo / 16, exact down to 2^-13 of the row's largest channel and off by at most 2^-21 of
//     it below.  A probability, times 2^8 and rounded to half (11 bits, half a step 2^-11), is three codes:
//     p1 + p2 / 16 + p3 / 256.  The products of codes are exact and are summed in float, so no other rounding enters.
//   * A lane's operand fragment of 16 rows x 32 channels is four words of four codes of two rows.  Which channel is which k
//     index of the product is free as long as keys and queries agree, so a lane takes 16 neighbouring channels of its row
//     (one 16-byte piece: the fragments of two k steps), and 8 of V^T, whose rows are channels and whose columns are the cache's
//     rows.  The rows of the score tiles are dealt so that the scores come out where the second product wants them
//     (tile_row); one 8 x 8 transpose of 16-bit pairs then makes four probabilities' codes the word of a fragment.
//   * Scores, maxima, sums and outputs are float.  The scales of a page's block multiply a score and a page's output sums
//     once: an exact product.
//   * A warp works by itself: it copies half pages (32 rows of keys and of values) ahead of itself into places of its own in
//     shared memory (cp.async) and has its own running maximum and sum.  Half pages, because 10 to 12 warps an SM then find
//     room: with whole pages six did, and each waited for itself (64 sequences of 130 to 2,300 rows, 8 kv heads of 128: 57.9 us
//     where this form took 52.4 before the steps below).  All warps share the pages of all sequences evenly (few_place).
//   * What is left beside the reading is each warp's begin -- where its stretch lies, page numbers, queries, each a wait
//     for memory -- and the joining kernel, whose waits are the same and which therefore finds its place while the first one
//     still runs, reads all parts of a query at once and, where weights are gathered, turns the scores, kept in float, into
//     probabilities now that every query's maximum and sum are known.
// Measured on a B200, both kernels: 8 sequences of 8,192 rows, 32 heads of 64: 52.0 us for 268 MB of codes (5.2 TB/s; a plain
// copy moves 6.5); the ragged batch above: 37.5 us for 165 MB; 8 of 4,000 with weights, 8 kv heads of 64: 16.5 us for 33 MB; one
// of 2,251, 32 heads of 64: 8.9 us, all of it waits.
#pragma once
#include "mma_helpers.cuh"
#include "e4m3.cuh"
#include <algorithm>

namespace {
constexpr float kLog2e = 1.4426950408889634f;
// Where a query's channels are multiplied with codes in float: kept smaller, so that the products of the largest ones do not
// leave float's range before the key scale is in.
constexpr float kUp = 4294967296.0f, kDown = 1.0f / kUp;
constexpr int kFewWarps = 2, kFewThreads = 32 * kFewWarps;
constexpr int kFewColumns = 32;          // queries a key/value head that these kernels take
constexpr int kStepRows = 32;            // cache rows a warp takes at a time: half a page
constexpr float kPShift = 8.0f;          // probabilities are held times 2^8

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// D = A(16 x 32, row) B(32 x 8, col) (+ D): e4m3 operands, float sums.
__device__ __forceinline__ void mma_e4m3_16832_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_e4m3_16832(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t codes_of_f16(__half2 x) {                  // two codes in the low 16 bits
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
    return r;
}
__device__ __forceinline__ __half2 f16_of_codes(uint32_t c) {
    const uint32_t r = e4m3_pair_f16(c);
    return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
}

// Cache row within its step of row r (0..15) of score tile j: the rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a tile are four
// neighbouring rows, those of the word that lane t has of a row of V^T.
__device__ __forceinline__ int tile_row(int j, int r) { return ((r & 7) >> 1) * 8 + 4 * j + (r & 1) + (r >> 3) * 2; }
// A transposed word holds the codes of the rows 2 t, 2 t + 8, 2 t + 1, 2 t + 9.
__device__ __forceinline__ uint32_t in_row_order(uint32_t w) { return __byte_perm(w, 0, 0x3120); }
// Where a row stands among the kept scores of a query and step: a lane's four side by side.
__device__ __forceinline__ int score_place(int row) {
    return (((row >> 3) * 2 + (row & 1)) << 2) + ((row >> 2) & 1) * 2 + ((row >> 1) & 1);
}

template <int HD> struct Few {
    static constexpr int PIECE = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;     // bytes of a key row a lane takes at a time
    static constexpr int PIECES = HD / (4 * PIECE);
    static constexpr int WORDS = HD / 16;                                      // of a key row a lane has
    static constexpr int STEPS = (WORDS + 1) / 2;                              // of 32 channels
    static constexpr int TILES = HD / 16;                                      // of 16 channels
    static constexpr int PAGE_BYTES = kPageTokens * HD;                        // a page's keys (or values) of one head
    static constexpr int HALF_BYTES = kStepRows * HD;                          // a step's
    // rows of 128 bytes: where two neighbours would share banks, the odd ones lie with their halves exchanged
    static constexpr int SWAP = HD == 128 ? 1 : 0;
    static constexpr int STAGES = 2;                                           // three: one sequence of 2,251 rows 8.9 -> 9.3 us
    static constexpr int RING = kFewWarps * STAGES * 2 * HALF_BYTES;
};

struct FewArgs {
    const bf16* q;
    int ldq, wide, chained;      // wide: rows of q begin on 16 bytes; chained: the kernel before this one may still run
    bf16* out;
    int ldo;
    const int* cu_seqlens;
    const int* slots;
    const int* start_pos;
    int B, n_heads, group;
    float scale;
    int window;
    int columns;                 // max_q_len * group: queries of the longest run
    int tiles;                   // of 4 NT queries in them
    int workers;                 // warps that share the line
    float* part_o;               // [worker + unit][4 NT][HD]
    float* part_ml;              // [worker + unit][4 NT][2]
    float* scores;               // [b][kv head][column][score_pages][64] or null
    int score_pages;
};

// The rows of a sequence that its queries see, in steps, and where they lie on the line of all.
struct FewSeq {
    int begin, first, n_new, start, p_first, p_last, slot;
    __device__ __forceinline__ int steps() const { return n_new > 0 ? p_last - p_first + 1 : 0; }
};
__device__ __forceinline__ FewSeq few_seq(const FewArgs& a, const E4M3Pages& kv, int b) {
    FewSeq s;
    s.begin = 0;
    s.first = a.cu_seqlens[b];
    s.n_new = a.cu_seqlens[b + 1] - s.first;
    s.slot = a.slots[b];
    s.start = a.start_pos[b] - (kv.dropped ? kv.dropped[s.slot] : 0);
    s.p_first = (a.window > 0 ? max(0, s.start - a.window + 1) : 0) / kStepRows;
    s.p_last = (s.start + s.n_new - 1) / kStepRows;
    return s;
}
// All steps of all units -- a unit is a (sequence, kv head, tile of queries) -- lie on one line: sequence by sequence, unit by
// unit, step by step.  Every worker takes an equal stretch of it, so all finish together whatever the lengths are, and
// whatever a plan was made for.  A unit's begin costs a worker queries, a page number and a result: kUnitCost empty steps
// before its first stand for that (none: 43.5 us where
// two take 39.2, 64 sequences of 130 to 2,300 rows, 8 kv heads of 128).  Called by whole warps, which look at 32 sequences at a time, at the first 64 once:
// the steps a worker takes, where worker's stretch begins, and the sequence that this (BY_WORKER) falls into, b = -1 behind
// the line's end; or sequence `which`.
constexpr int kSeenOnce = 2, kUnitCost = 2, kLeastSteps = 2;
__device__ __forceinline__ int on_line(int steps) { return steps > 0 ? steps + kUnitCost : 0; }
struct FewPlace { int per, from, b; FewSeq seq; };
template <bool BY_WORKER>
__device__ __forceinline__ FewPlace few_place(const FewArgs& a, const E4M3Pages& kv, int units, int which) {
    const int lane = threadIdx.x & 31;
    FewSeq seen[kSeenOnce];
    auto at = [&](int b) {                                                      // (no branch: the reads of several do not wait for each other)
        FewSeq s = few_seq(a, kv, min(b, a.B - 1));
        if (b >= a.B) s.n_new = 0;
        return s;
    };
    int total = 0;
#pragma unroll
    for (int x = 0; x < kSeenOnce; ++x) seen[x] = at(32 * x + lane);
#pragma unroll
    for (int x = 0; x < kSeenOnce; ++x) total += __reduce_add_sync(0xffffffffu, on_line(seen[x].steps()));
    for (int b0 = 32 * kSeenOnce; b0 < a.B; b0 += 32) total += __reduce_add_sync(0xffffffffu, on_line(at(b0 + lane).steps()));
    FewPlace p;
    // (shorter stretches would cost more in joining than they save)
    p.per = max(kLeastSteps, (int)(((unsigned)total * units + a.workers - 1) / a.workers));
    p.from = BY_WORKER ? which * p.per : 0;
    p.b = -1;
    int begin = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        FewSeq s = seen[0];
#pragma unroll
        for (int x = 1; x < kSeenOnce; ++x)
            if (b0 == 32 * x) s = seen[x];
        if (b0 >= 32 * kSeenOnce) s = at(b0 + lane);
        const int mine = on_line(s.steps());
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        s.begin = begin + (incl - mine) * units;
        const unsigned past = __ballot_sync(0xffffffffu, BY_WORKER ? begin + incl * units > p.from : b0 + lane == which);
        if (past) {
            const int who = __ffs(past) - 1;
            p.b = b0 + who;
            p.seq.begin = __shfl_sync(0xffffffffu, s.begin, who);
            p.seq.first = __shfl_sync(0xffffffffu, s.first, who);
            p.seq.n_new = __shfl_sync(0xffffffffu, s.n_new, who);
            p.seq.start = __shfl_sync(0xffffffffu, s.start, who);
            p.seq.p_first = __shfl_sync(0xffffffffu, s.p_first, who);
            p.seq.p_last = __shfl_sync(0xffffffffu, s.p_last, who);
            p.seq.slot = __shfl_sync(0xffffffffu, s.slot, who);
            break;
        }
        begin += __shfl_sync(0xffffffffu, incl, 31) * units;
    }
    return p;
}

// A warp a worker; NT tiles of four queries a unit.
template <int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, NT == 4 || (NT == 2 && HD > 80) ? 4 : HD <= 64 ? 6 : 5)
few_queries_kernel(const FewArgs a, const E4M3Pages kv) {
    using F = Few<HD>;
    constexpr int W = F::WORDS;
    chain_release();
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int worker = blockIdx.x * kFewWarps + warp;
    const int units = kv.n_kv * a.tiles;                                        // of a sequence
    const uint32_t ring = smem_u32(smem) + warp * F::STAGES * 2 * F::HALF_BYTES;
    const unsigned char* ring_at = smem + warp * F::STAGES * 2 * F::HALF_BYTES;

    // ---- this worker's stretch of the line
    const FewPlace place = few_place<true>(a, kv, units, worker);
    if (place.b < 0) {
        chain_wait();
        return;
    }
    FewSeq span = place.seq;
    int b = place.b, left = place.per, offset = place.from - span.begin;        // steps still to do; from the sequence's begin
    bool waited = false;
    while (left > 0) {
        const int n_steps = span.steps(), n_line = on_line(n_steps);
        const int in_b = n_steps > 0 ? offset / n_line : units;                 // unit within the sequence
        if (in_b >= units) {
            if (++b == a.B) break;
            span = few_seq(a, kv, b);
            offset = 0;
            continue;
        }
        const int from = offset - in_b * n_line, mine = min(left, n_line - from);
        left -= mine;
        offset += mine;
        const int skip = max(from - kUnitCost, 0), n_mine = max(from + mine - kUnitCost, 0) - skip;
        if (n_mine == 0) continue;
        const int h = in_b / a.tiles, c0 = in_b % a.tiles * 4 * NT;
        const int n_columns = min(span.n_new * a.group, a.columns);
        if (c0 >= n_columns) continue;                                          // a shorter run of queries than the longest
        const int p_begin = span.p_first + skip;
        const int* table = kv.block_table + (size_t)span.slot * kv.table_stride;
        const uint8_t* kh = kv.k + (size_t)h * F::PAGE_BYTES + lane * 16;
        const uint8_t* vh = kv.v + (size_t)h * F::PAGE_BYTES + lane / 2 * kPageTokens + lane % 2 * 16;

        int ahead_pages = lane < n_mine ? table[(p_begin + lane) / 2] : 0;      // lane i: page of step (ahead / 32 * 32 + i) of the stretch
        auto load = [&](int i) {
            if (i > 0 && (i & 31) == 0) ahead_pages = i + lane < n_mine ? table[(p_begin + i + lane) / 2] : 0;
            const size_t page = __shfl_sync(0xffffffffu, ahead_pages, i & 31);
            const int odd = (p_begin + i) & 1;
            const uint32_t dst = ring + (i % F::STAGES) * 2 * F::HALF_BYTES + lane * 16;
            const uint8_t* ks = kh + page * kv.k_stride + odd * F::HALF_BYTES;
            const uint8_t* vs = vh + page * kv.v_stride + odd * kStepRows;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                copy_async16((F::SWAP ? dst ^ (lane << 3 & 64) : dst) + c * 512, ks + c * 512);           // bit 3 of the lane: the row's parity
                copy_async16(dst + F::HALF_BYTES + c * 512, vs + c * 16 * kPageTokens);
            }
        };
        int ahead = 0;
        __syncwarp();                                                           // the stretch before has been read
        if (!waited) {
            // Pages before the newest were complete before the kernel that stores this step's rows began (it lets its successor
            // begin only after its own wait), so their copies may start while it runs; the pages that take new rows may not.
            if (a.chained) {
#pragma unroll
                for (int s = 0; s < F::STAGES - 1; ++s)
                    if (ahead == s && s < n_mine && p_begin + s < span.start / kPageTokens * 2) load(ahead++);
            }
            chain_wait();
            waited = true;
        }
        // ---- queries: column g of a tile is query g / 2, its high codes (even g) or its low ones
        uint32_t qf[NT][2 * F::STEPS];
        float factor[NT];                                                           // of query t4: what a score is multiplied with
        int seen_to[NT];                                                            // the last row query t4 sees; -1: no such query
        uint32_t x[NT][HD / 8];                                                     // two channels each
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int c = c0 + nt * 4 + (g >> 1);
            const bool real = c < n_columns;
            const bf16* src = a.q + (size_t)(span.first + (real ? c / a.group : 0)) * a.ldq + (size_t)(h * a.group + (real ? c % a.group : 0)) * HD +
                              t4 * F::PIECE;
#pragma unroll
            for (int pc = 0; pc < F::PIECES; ++pc) {
                uint32_t* to = x[nt] + pc * F::PIECE / 2;
                const bf16* from = src + pc * 4 * F::PIECE;
                if (a.wide) {
                    if constexpr (F::PIECE == 4) {
                        const uint2 u = *reinterpret_cast<const uint2*>(from);
                        to[0] = u.x; to[1] = u.y;
                    } else {
#pragma unroll
                        for (int i = 0; i < F::PIECE / 8; ++i) {
                            const uint4 u = reinterpret_cast<const uint4*>(from)[i];
                            to[4 * i] = u.x; to[4 * i + 1] = u.y; to[4 * i + 2] = u.z; to[4 * i + 3] = u.w;
                        }
                    }
                } else {
                    const uint16_t* each = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
                    for (int i = 0; i < F::PIECE / 2; ++i) to[i] = each[2 * i] | (uint32_t)each[2 * i + 1] << 16;
                }
            }
            if (!real) {
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) x[nt][i] = 0;
            }
        }
#pragma unroll
        for (int s = 0; s < F::STAGES - 1; ++s) {
            if (ahead == s && s < n_mine) load(ahead++);
            cp_async_commit();
        }
        float k_scales = 0.f, v_scales = 0.f;                                       // lane i: of step (i / 32 * 32 + i) of the stretch
        auto load_scales = [&](int pages) {
            const float* s = kv.scales + (size_t)pages * kv.scale_stride + h;
            k_scales = s[0];
            v_scales = s[kv.n_kv];
        };
        if (lane < n_mine) load_scales(ahead_pages);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t most = 0;                                                      // the largest magnitude, as bits
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) most = __vmaxu2(most, x[nt][i] & 0x7fff7fffu);
            most = max(most & 0xffffu, most >> 16);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // the largest channel comes to lie in [128, 256)
            const int e = (int)(most >> 7), up = e == 0 ? 0 : min(7 - (e - 127), 100);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            const float back = a.scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23);
            factor[nt] = __shfl_sync(0xffffffffu, back, 8 * t4);
            const int cq = c0 + nt * 4 + t4;
            seen_to[nt] = cq < n_columns ? span.start + cq / a.group : -1;
            const bool whole = e < 255;                                             // else the scores are NaN, whatever its other channels are
            uint32_t pair[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {                                      // (8 bits in a half's 11: exact down to 2^-22 of the largest)
                const __half2 y = __floats2half2_rn(__uint_as_float(x[nt][i] << 16) * f, __uint_as_float(x[nt][i] & 0xffff0000u) * f);
                const uint32_t hi = codes_of_f16(y);
                const uint32_t lo = codes_of_f16(__hmul2(__hsub2(y, f16_of_codes(hi)), __floats2half2_rn(16.f, 16.f)));
                pair[i] = !whole ? 0x7f7fu : g & 1 ? lo : hi;
            }
#pragma unroll
            for (int s = 0; s < W; ++s) qf[nt][s] = pair[2 * s] | pair[2 * s + 1] << 16;
            if (W & 1) qf[nt][2 * F::STEPS - 1] = 0;
        }
        const int least_to = span.start + c0 / a.group;
        const int most_to = span.start + min(n_columns - 1, c0 + 4 * NT - 1) / a.group;
        float m[NT], l[NT], o[F::TILES][NT][2];                                     // of query t4; o: channels 16 i + g and + 8
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = -INFINITY;
            l[nt] = 0.f;
#pragma unroll
            for (int i = 0; i < F::TILES; ++i) o[i][nt][0] = o[i][nt][1] = 0.f;
        }

        for (int i = 0; i < n_mine; ++i) {
            const int p = p_begin + i;
            if (i > 0 && (i & 31) == 0 && i + lane < n_mine) load_scales(table[(p + lane) / 2]);
            const float k_scale = __shfl_sync(0xffffffffu, k_scales, i & 31), v_scale = __shfl_sync(0xffffffffu, v_scales, i & 31);
            cp_async_wait<F::STAGES - 2>();
            __syncwarp();                                                           // page i is there, page i - 1 has been read
            const unsigned char* stage = ring_at + i % F::STAGES * 2 * F::HALF_BYTES;
            if (ahead < n_mine) load(ahead++);                                      // where page i - 1 was
            cp_async_commit();
            // (queries that do not exist are zeros and see what they like)
            const bool all_seen = p * kStepRows + kStepRows - 1 <= least_to && (a.window <= 0 || p * kStepRows > most_to - a.window);
            // ---- scores of the step's 32 rows: of query t4, rows g and g + 8 of each tile
            float s[2][NT][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[2][2 * F::STEPS];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int pc = 0; pc < F::PIECES; ++pc) {
                        const unsigned char* at = stage + tile_row(j, g + 8 * r) * HD + (F::SWAP ? pc ^ (g & 1) : pc) * 4 * F::PIECE + t4 * F::PIECE;
                        if constexpr (F::PIECE == 16) {
                            const uint4 u = *reinterpret_cast<const uint4*>(at);
                            w[r][4 * pc] = u.x; w[r][4 * pc + 1] = u.y; w[r][4 * pc + 2] = u.z; w[r][4 * pc + 3] = u.w;
                        } else if constexpr (F::PIECE == 8) {
                            const uint2 u = *reinterpret_cast<const uint2*>(at);
                            w[r][2 * pc] = u.x; w[r][2 * pc + 1] = u.y;
                        } else {
                            w[r][pc] = *reinterpret_cast<const uint32_t*>(at);
                        }
                    }
                    if (W & 1) w[r][2 * F::STEPS - 1] = 0;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float c[4];
                    mma_e4m3_16832_first(c, w[0][0], w[1][0], w[0][1], w[1][1], qf[nt][0], qf[nt][1]);
#pragma unroll
                    for (int k = 1; k < F::STEPS; ++k)
                        mma_e4m3_16832(c, w[0][2 * k], w[1][2 * k], w[0][2 * k + 1], w[1][2 * k + 1], qf[nt][2 * k], qf[nt][2 * k + 1]);
                    const float f = factor[nt] * k_scale;
                    s[j][nt][0] = fmaf(c[1], 0.0625f, c[0]) * f;
                    s[j][nt][1] = fmaf(c[3], 0.0625f, c[2]) * f;
                }
            }
            if (!all_seen) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int to = seen_to[nt], from = a.window > 0 ? to - a.window : -1;              // rows from + 1 .. to
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = p * kStepRows + tile_row(j, g + 8 * r);
                            if (row > to || row <= from) s[j][nt][r] = -INFINITY;
                        }
                }
            }
            if (a.scores && p < 2 * a.score_pages) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int c = c0 + nt * 4 + t4;
                    if (c < n_columns) {
                        float* at = a.scores + (((size_t)b * kv.n_kv + h) * a.columns + c) * a.score_pages * kPageTokens + (size_t)p * kStepRows + g * 4;
                        *reinterpret_cast<float4*>(at) = make_float4(s[0][nt][0], s[0][nt][1], s[1][nt][0], s[1][nt][1]);
                    }
                }
            }
            // ---- running maximum and sum; probabilities' codes as the second product's right operand: columns (query, p1 | p2)
            //      in pf, and in ph the p3 of two tiles (of one, and nothing)
            constexpr int NH = (NT + 1) / 2;
            float corr[NT];
            uint32_t pf[2][NT], ph[2][NH];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float mx = fmaxf(fmaxf(s[0][nt][0], s[0][nt][1]), fmaxf(s[1][nt][0], s[1][nt][1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float now = fmaxf(m[nt], mx);
                const float use = now == -INFINITY ? 0.f : now;
                corr[nt] = exp2_fast(m[nt] - use);
                m[nt] = now;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = exp2_fast(s[j][nt][0] - use + kPShift), p1 = exp2_fast(s[j][nt][1] - use + kPShift);
                    sum += p0 + p1;
                    const __half2 sixteen = __floats2half2_rn(16.f, 16.f);
                    __half2 rest = __floats2half2_rn(p0, p1);
                    const uint32_t c1 = codes_of_f16(rest);
                    rest = __hmul2(__hsub2(rest, f16_of_codes(c1)), sixteen);
                    const uint32_t c2 = codes_of_f16(rest);
                    rest = __hmul2(__hsub2(rest, f16_of_codes(c2)), sixteen);
                    const uint32_t c3 = codes_of_f16(rest);
                    pf[j][nt] = in_row_order(transpose_8x8(c1 | c2 << 16));
                    ph[j][nt / 2] = nt & 1 ? ph[j][nt / 2] | c3 << 16 : c3;
                    if ((nt & 1) || nt == NT - 1) ph[j][nt / 2] = in_row_order(transpose_8x8(ph[j][nt / 2]));
                }
                l[nt] = l[nt] * corr[nt] + sum;
            }
            // ---- O^T += V^T P^T, 16 channels at a time
            bool odd = false;                                                       // a NaN code in a step that not every query sees whole
#pragma unroll
            for (int ct = 0; ct < F::TILES; ++ct) {
                uint32_t w[2][2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint2 u = *reinterpret_cast<const uint2*>(stage + F::HALF_BYTES + (16 * ct + 8 * r + g) * kStepRows + t4 * 8);
                    w[r][0] = u.x; w[r][1] = u.y;
                }
                if (!all_seen) {
                    // A row that a query does not see has probability 0 there; its values may still be the NaN code, which
                    // 0 does not silence.  They are taken out here and given back below to the queries that do see them.
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t nan = __vcmpeq4(w[r][j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                            odd |= nan != 0;
                            w[r][j] &= ~nan;
                        }
                }
                float u[NH][4];
#pragma unroll
                for (int nh = 0; nh < NH; ++nh) mma_e4m3_16832_first(u[nh], w[0][0], w[1][0], w[0][1], w[1][1], ph[0][nh], ph[1][nh]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float t[4];
                    mma_e4m3_16832_first(t, w[0][0], w[1][0], w[0][1], w[1][1], pf[0][nt], pf[1][nt]);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        o[ct][nt][r] = fmaf(o[ct][nt][r], corr[nt],
                                            fmaf(u[nt / 2][2 * r + (nt & 1)], 0.00390625f, fmaf(t[2 * r + 1], 0.0625f, t[2 * r])) * v_scale);
                }
            }
            if (__any_sync(0xffffffffu, odd)) {
                // how many NaN codes of rows it sees a query meets in each channel: ones (code 0x38) for the codes, ones for the rows seen
                uint32_t seen[2][NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t pair = 0;
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int to = seen_to[nt], row = p * kStepRows + tile_row(j, g + 8 * r);
                            if (row <= to && (a.window <= 0 || row > to - a.window)) pair |= 0x38u << (8 * r);
                        }
                        seen[j][nt] = in_row_order(transpose_8x8(pair));
                    }
#pragma unroll
                for (int ct = 0; ct < F::TILES; ++ct) {
                    uint32_t w[2][2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint2 u = *reinterpret_cast<const uint2*>(stage + F::HALF_BYTES + (16 * ct + 8 * r + g) * kStepRows + t4 * 8);
                        w[r][0] = u.x; w[r][1] = u.y;
#pragma unroll
                        for (int j = 0; j < 2; ++j) w[r][j] = __vcmpeq4(w[r][j] & 0x7f7f7f7fu, 0x7f7f7f7fu) & 0x38383838u;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float t[4];
                        mma_e4m3_16832_first(t, w[0][0], w[1][0], w[0][1], w[1][1], seen[0][nt], seen[1][nt]);
                        if (t[0] > 0.f) o[ct][nt][0] = __uint_as_float(0x7fc00000u);
                        if (t[2] > 0.f) o[ct][nt][1] = __uint_as_float(0x7fc00000u);
                    }
                }
            }
        }
        cp_async_wait<0>();

        // ---- the whole of its pages: the unit's result; else a part of it, for the joining kernel
        const bool whole = n_mine == n_steps;
        const size_t part = ((size_t)worker + (size_t)b * units + in_b) * 4 * NT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float sum = l[nt];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int c = nt * 4 + t4;
            if (c0 + c >= n_columns) continue;
            if (g == 0 && (!whole || a.scores)) {
                a.part_ml[(part + c) * 2] = m[nt];
                a.part_ml[(part + c) * 2 + 1] = sum;
            }
            const float inverse = 1.0f / sum;
            bf16* out = a.out + (size_t)(span.first + (c0 + c) / a.group) * a.ldo + (size_t)(h * a.group + (c0 + c) % a.group) * HD;
#pragma unroll
            for (int ct = 0; ct < F::TILES; ++ct)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (whole) out[16 * ct + 8 * r + g] = __float2bfloat16_rn(o[ct][nt][r] * inverse);
                    else a.part_o[(part + c) * HD + 16 * ct + 8 * r + g] = o[ct][nt][r];
                }
        }
    }
    if (!waited) chain_wait();
}

// Joins the parts (blocks x < join_blocks: some queries of one (sequence, kv head)) and, where weights are gathered, adds to
// them (the other blocks, four pages at a time).  Both are a few short reads that wait for one another, so the parts of a
// query are spread over all threads that its channels leave.
constexpr int kJoinThreads = 256, kJoinBlocks = 4;                             // blocks an SM

template <int HD> struct Join {
    static constexpr int LANES = HD / 4;                                        // threads of a query's channels
    static constexpr int ROWS = kJoinThreads / LANES;
    __host__ __device__ static int share(int columns) { return columns >= ROWS ? 1 : ROWS / columns; }    // rows that share a query's parts
    __host__ __device__ static int columns_each(int columns) { return ROWS / share(columns); }
};

template <int HD, int NT>
__global__ void __launch_bounds__(kJoinThreads, kJoinBlocks)
few_join_kernel(const FewArgs a, const E4M3Pages kv, int join_blocks) {
    using J = Join<HD>;
    chain_release();
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const FewPlace place = few_place<false>(a, kv, kv.n_kv * a.tiles, b);       // (of what the kernel before this one only reads, too)
    const FewSeq span = place.seq;
    const int per = place.per, n_columns = min(span.n_new * a.group, a.columns), n_line = on_line(span.steps());
    chain_wait();
    if (n_columns <= 0) return;
    const size_t unit = (size_t)(b * kv.n_kv + h) * a.tiles;
    auto part_of = [&](int worker, int c) { return ((size_t)worker + unit + c / (4 * NT)) * 4 * NT + c % (4 * NT); };
    // the workers that share the steps of query c: first and last
    auto first_worker = [&](int c) { return (span.begin + (h * a.tiles + c / (4 * NT)) * n_line + kUnitCost) / per; };
    auto last_worker = [&](int c) { return (span.begin + (h * a.tiles + c / (4 * NT) + 1) * n_line - 1) / per; };
    // a running maximum and sum, and another part's: what each of the two is multiplied with
    auto join = [](float& M, float m, float& mine, float& theirs) {
        const float now = fmaxf(M, m), use = now == -INFINITY ? 0.f : now;
        mine = exp2_fast(M - use);
        theirs = exp2_fast(m - use);
        M = now;
    };
    if ((int)blockIdx.x < join_blocks) {
        __shared__ float4 sums[J::ROWS * J::LANES];
        __shared__ float2 stats[J::ROWS];
        const int share = J::share(a.columns), row = tid / J::LANES, d = tid % J::LANES * 4;
        const int c = blockIdx.x * J::columns_each(a.columns) + row / share;
        const bool mine = row / share < J::columns_each(a.columns) && c < n_columns;
        const int w0 = mine ? first_worker(c) : 0, w1 = mine ? last_worker(c) : 0;                        // w0 == w1: it is not in parts
        if (w0 < w1) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float M = -INFINITY, L = 0.f, f, g;
            constexpr int kAtOnce = 4;                                              // reads in flight
            for (int w = w0 + row % share; w <= w1; w += kAtOnce * share) {
                float2 ml[kAtOnce];
                float4 o[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const bool there = w + i * share <= w1;
                    const size_t at = part_of(there ? w + i * share : w, c);
                    ml[i] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
                    o[i] = *reinterpret_cast<const float4*>(a.part_o + at * HD + d);
                    if (!there) {
                        ml[i] = make_float2(-INFINITY, 0.f);
                        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    join(M, ml[i].x, f, g);
                    L = fmaf(g, ml[i].y, L * f);
                    acc.x = fmaf(g, o[i].x, acc.x * f); acc.y = fmaf(g, o[i].y, acc.y * f);
                    acc.z = fmaf(g, o[i].z, acc.z * f); acc.w = fmaf(g, o[i].w, acc.w * f);
                }
            }
            sums[tid] = acc;
            if (d == 0) stats[row] = make_float2(M, L);
        }
        __syncthreads();
        if (w0 < w1 && row % share == 0) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float M = -INFINITY, L = 0.f;
            for (int i = 0; i < share; ++i) M = fmaxf(M, stats[row + i].x);
            const float use = M == -INFINITY ? 0.f : M;
#pragma unroll 4
            for (int i = 0; i < share; ++i) {
                const float4 o = sums[tid + i * J::LANES];
                const float f = exp2_fast(stats[row + i].x - use);
                L = fmaf(f, stats[row + i].y, L);
                acc.x = fmaf(f, o.x, acc.x); acc.y = fmaf(f, o.y, acc.y); acc.z = fmaf(f, o.z, acc.z); acc.w = fmaf(f, o.w, acc.w);
            }
            const float inverse = 1.0f / L;
            bf16* out = a.out + (size_t)(span.first + c / a.group) * a.ldo + (size_t)(h * a.group + c % a.group) * HD + d;
            out[0] = __float2bfloat16_rn(acc.x * inverse);
            out[1] = __float2bfloat16_rn(acc.y * inverse);
            out[2] = __float2bfloat16_rn(acc.z * inverse);
            out[3] = __float2bfloat16_rn(acc.w * inverse);
        }
        return;
    }
    __shared__ float top[kFewColumns], inverse[kFewColumns];
    for (int c = tid >> 5; c < n_columns; c += kJoinThreads / 32) {             // a warp a query: its maximum and sum over the parts
        const int w0 = first_worker(c), w1 = last_worker(c);
        float M = -INFINITY, L = 0.f, f, g;
        for (int w = w0 + (tid & 31); w <= w1; w += 32) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + part_of(w, c) * 2);
            join(M, ml.x, f, g);
            L = fmaf(g, ml.y, L * f);
        }
        const float all = warp_max(M), use = all == -INFINITY ? 0.f : all;
        L = warp_sum(exp2_fast(M - use) * L);
        if ((tid & 31) == 0) { top[c] = use; inverse[c] = 1.0f / L; }
    }
    __syncthreads();
    const int* table = kv.block_table + (size_t)span.slot * kv.table_stride;
    const int stride = ((int)gridDim.x - join_blocks) * (kJoinThreads / kPageTokens);
    for (int p = span.p_first / 2 + ((int)blockIdx.x - join_blocks) * (kJoinThreads / kPageTokens) + tid / kPageTokens; p <= span.p_last / 2; p += stride) {
        const int t = tid % kPageTokens, row = p * kPageTokens + t;
        if (row < span.p_first * kStepRows || row >= span.start + span.n_new) continue;                   // seen by no query
        const size_t page = table[p];
        float sum = 0.f;
        if (p < a.score_pages) {
            const float* at = a.scores + (((size_t)b * kv.n_kv + h) * a.columns * a.score_pages + p) * kPageTokens + t / kStepRows * kStepRows + score_place(t % kStepRows);
            for (int c = 0; c < n_columns; ++c) {
                const float s = at[(size_t)c * a.score_pages * kPageTokens];
                sum += s == -INFINITY ? 0.f : exp2_fast(s - top[c] + kPShift) * inverse[c];               // (not seen: not NaN either)
            }
        } else {                                                                // a sequence that has outgrown the plan: score the row again
            const uint8_t* kr = kv.k + page * kv.k_stride + ((size_t)h * kPageTokens + t) * HD;
            const float k_scale = kv.scales[page * kv.scale_stride + h] * a.scale * kLog2e;
            for (int c = 0; c < n_columns; ++c) {
                const int to = span.start + c / a.group;
                if (row > to || (a.window > 0 && row <= to - a.window)) continue;
                const bf16* qr = a.q + (size_t)(span.first + c / a.group) * a.ldq + (size_t)(h * a.group + c % a.group) * HD;
                float s = 0.f;
                for (int d = 0; d < HD; ++d) s = fmaf(__bfloat162float(qr[d]) * kDown, e4m3_value(kr[d]), s);
                sum += exp2_fast(min_or_nan(s * k_scale * kUp - top[c] + score_slack(top[c]), 0.f) + kPShift) * inverse[c];
            }
        }
        kv.weights[page * kv.weight_stride + h * kPageTokens + t] += sum;
    }
}

bool few_takes(int dtype, int max_q_len, int n_heads, int n_kv, int hd) {
    return dtype == 1 && hd % 16 == 0 && hd <= 128 && (long long)max_q_len * (n_heads / n_kv) <= kFewColumns;
}

// Tiles of four queries a unit has.
int few_tiles(int columns) { return columns <= 4 ? 1 : columns <= 8 ? 2 : 4; }
// The line is counted in 32 bits: no table of this width holds more steps than that.
bool few_counts(int B, int max_q_len, int n_heads, int n_kv, int table_width) {
    const int columns = max_q_len * (n_heads / n_kv), each = 4 * few_tiles(columns);
    return (double)B * n_kv * ((columns + each - 1) / each) * ((double)table_width * (kPageTokens / kStepRows) + 1 + kUnitCost) < 1 << 30;
}

// How many warps run at once, and the scratch they need.
struct FewPlan {
    int columns, nt, tiles, workers, score_pages;
    long long part_o, part_ml, scores;                                          // floats, each a multiple of 4
    long long floats() const { return part_o + part_ml + scores; }
};

// Warps of this kernel that the current device runs at once (asked once a device).
template <int HD, int NT>
int few_workers() {
    static int cached[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kFewWarps;
    if (cached[dev] == 0) {
        int blocks = 0, sms = 0;
        if (cudaFuncSetAttribute(few_queries_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<HD>::RING) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, few_queries_kernel<HD, NT>, kFewThreads, Few<HD>::RING) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || blocks < 1) {
            (void)cudaGetLastError();
            return kFewWarps;
        }
        cached[dev] = blocks * sms * kFewWarps;
    }
    return cached[dev];
}

template <int HD>
FewPlan few_plan_for(int B, int max_q_len, int n_heads, int n_kv, int max_kv_len, int weigh) {
    FewPlan plan;
    plan.columns = max_q_len * (n_heads / n_kv);
    plan.nt = few_tiles(plan.columns);
    plan.tiles = (plan.columns + 4 * plan.nt - 1) / (4 * plan.nt);
    plan.workers = plan.nt == 4 ? few_workers<HD, 4>() : plan.nt == 2 ? few_workers<HD, 2>() : few_workers<HD, 1>();
    plan.score_pages = weigh ? (max_kv_len + kPageTokens - 1) / kPageTokens : 0;
    const long long parts = ((long long)plan.workers + (long long)B * n_kv * plan.tiles) * 4 * plan.nt;
    plan.part_o = parts * HD;
    plan.part_ml = parts * 2;
    plan.scores = (long long)B * n_kv * plan.columns * plan.score_pages * kPageTokens;
    return plan;
}

template <int HD, int NT>
int launch_few_tiles(const FewArgs& a, const E4M3Pages& kv, cudaStream_t stream) {
    const int st = launch_early(a.chained != 0, few_queries_kernel<HD, NT>, dim3(a.workers / kFewWarps), dim3(kFewThreads), Few<HD>::RING,
                                stream, a, kv);
    if (st != 0) return st;
    const int join = (a.columns + Join<HD>::columns_each(a.columns) - 1) / Join<HD>::columns_each(a.columns);
    // no more blocks than run at once: each begins with the same few reads, and a second turn would wait for them again
    const int pages = a.score_pages ? std::max(1, std::min((a.score_pages * kPageTokens + kJoinThreads - 1) / kJoinThreads,
                                                           kJoinBlocks * 148 / (kv.n_kv * a.B) - join)) : 0;
    return launch_behind(few_join_kernel<HD, NT>, dim3(join + pages, kv.n_kv, a.B), dim3(kJoinThreads), 0, stream, a, kv, join);
}

template <int HD>
int launch_few(FewArgs a, const E4M3Pages& kv, const FewPlan& plan, float* scratch, cudaStream_t stream) {
    a.columns = plan.columns;
    a.tiles = plan.tiles;
    a.workers = plan.workers;
    a.score_pages = plan.score_pages;
    a.part_o = scratch;
    a.part_ml = a.part_o + plan.part_o;
    a.scores = plan.scores ? a.part_ml + plan.part_ml : nullptr;
    return plan.nt == 4 ? launch_few_tiles<HD, 4>(a, kv, stream)
         : plan.nt == 2 ? launch_few_tiles<HD, 2>(a, kv, stream) : launch_few_tiles<HD, 1>(a, kv, stream);
}
}  // namespace
