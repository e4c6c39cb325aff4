// Attention of few queries a sequence over the 8-bit cache: decode steps, and steps of a few tokens (up to kFewColumns query
// rows -- tokens times the heads of a group -- a key/value head).
//
// What bounds it is reading the cache: 2 * head size bytes a row, each used for a few multiply-adds.  So the cache goes
// from memory to registers once, and everything else is arranged around the order in which it lies there.
//
//   * The keys are the rows of the products (M = 16 rows of the cache, N = 8 queries): S^T = K Q^T, O^T = V^T P^T.  With the
//     queries as rows, 16 of them would be multiplied where a group has one to eight.
//   * A lane's operand fragment of 16 rows x 16 channels is four codes of two rows.  Which channel is which k index of the
//     product is free as long as keys and queries agree, so a lane takes 16 neighbouring channels of its row (one 16-byte piece:
//     the fragments of four k steps), and the same of V^T, whose rows are channels and whose 64 columns are the page's rows.
//     The rows of the score tiles are dealt so that the scores come out where the second product wants them: row r of
//     tile j is cache row 16 (r/2 mod 4) + 4 j + 2 (r / 8) + r mod 2, and a lane's 16 values columns are 16 t4 .. 16 t4 + 15.
//   * Codes become pairs of halves in one instruction a pair, exactly (e4m3 is a subset of half).  Queries are scaled by a
//     power of two a row to fill half's range, so that rounding bfloat16 to half loses nothing that counts; probabilities are
//     kept times 2^14 for the same reason.  Scores, maxima, sums and outputs are float.  The scales of a page's block
//     multiply a score and a page's output sums once: an exact product.
//   * Every warp copies whole pages ahead of itself (cp.async into a place in shared memory that only the lane that copies
//     reads, so nothing is waited for but the copies), four warps to a block take turns with the pages, blocks share a
//     sequence's pages (split), and a second kernel joins the parts -- and, where weights are gathered, turns the scores, kept
//     in float, into probabilities now that every row's maximum and sum are known.
#pragma once
#include "mma_helpers.cuh"
#include "e4m3.cuh"

namespace {
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFewThreads = 128, kFewWarps = 4;
constexpr int kFewColumns = 32;          // query rows a key/value head that these kernels take
constexpr float kPShift = 14.0f;         // probabilities are held times 2^14

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// D += A(16 x 16, row) B(16 x 8, col): half operands, float sums.
__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES));
}

// Cache row within its page of row r (0..15) of score tile j.
__device__ __forceinline__ int tile_row(int j, int r) { return ((r & 7) >> 1) * 16 + 4 * j + (r >> 3) * 2 + (r & 1); }
// Where a page's row stands among a query's 64 kept scores: a lane's eight side by side.
__device__ __forceinline__ int score_place(int row) {
    return (((row >> 4) * 2 + (row & 1)) << 3) + ((row & 15) >> 2) * 2 + ((row >> 1) & 1);
}

template <int HD> struct Few {
    static constexpr int PIECE = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;     // bytes of a key row a lane takes at a time
    static constexpr int PIECES = HD / (4 * PIECE);
    static constexpr int STEPS = HD / 16;
    static constexpr int HALF_BYTES = 64 * HD;                                 // a page's keys (or values) of one head
    static constexpr int STAGES = HD <= 64 ? 3 : 2;
    static constexpr int RING = kFewWarps * STAGES * 2 * HALF_BYTES;
    static constexpr int smem(int nt) {
        const int merge = kFewWarps * 8 * nt * (HD + 2) * 4;
        return RING > merge ? RING : merge;
    }
};

struct FewArgs {
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
    int n_splits, chunk_pages;
    int columns;                 // max_q_len * group: query rows of the longest sequence
    float* part_o;               // [b][kv head][split][column][HD]
    float* part_ml;              // [b][kv head][split][column][2]
    float* scores;               // [b][kv head][column][score_pages][64] or null
    int score_pages;
};

// The rows of sequence b that a step's queries see, in pages, and how they are shared out.
struct FewSpan {
    int first, n_new, start, p_first, p_last, my_splits, per_split;
};
__device__ __forceinline__ FewSpan few_span(const FewArgs& a, const E4M3Pages& kv, int b) {
    FewSpan s;
    s.first = a.cu_seqlens[b];
    s.n_new = a.cu_seqlens[b + 1] - s.first;
    s.start = a.start_pos[b] - (kv.dropped ? kv.dropped[a.slots[b]] : 0);
    s.p_first = (a.window > 0 ? max(0, s.start - a.window + 1) : 0) / kPageTokens;
    s.p_last = (s.start + s.n_new - 1) / kPageTokens;
    const int pages = s.p_last - s.p_first + 1;
    s.my_splits = max(1, min(a.n_splits, (pages + a.chunk_pages - 1) / a.chunk_pages));
    s.per_split = (pages + s.my_splits - 1) / s.my_splits;
    return s;
}

// grid (splits, kv heads x column tiles, sequences); a column is a (token, head of the group) pair, 8 NT of them a block.
template <int HD, int NT>
__global__ void __launch_bounds__(kFewThreads)
few_queries_kernel(const FewArgs a, const E4M3Pages kv) {
    using F = Few<HD>;
    chain_release();
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int b = blockIdx.z, split = blockIdx.x;
    const int tiles = (a.columns + 8 * NT - 1) / (8 * NT);
    const int h = blockIdx.y / tiles, c0 = (blockIdx.y % tiles) * 8 * NT;
    const FewSpan span = few_span(a, kv, b);
    const int n_columns = span.n_new * a.group;
    if (c0 >= n_columns) return;
    const int p_begin = span.p_first + split * span.per_split;
    const int p_end = split < span.my_splits ? min(span.p_last + 1, p_begin + span.per_split) : p_begin;
    const size_t part = (((size_t)b * kv.n_kv + h) * a.n_splits + split) * a.columns + c0;
    if (p_begin >= p_end) return;                                               // the joining kernel knows which splits have pages
    const int* table = kv.block_table + (size_t)a.slots[b] * kv.table_stride;
    const uint32_t ring = smem_u32(smem) + warp * F::STAGES * 2 * F::HALF_BYTES;
    const int n_mine = (p_end - p_begin - warp + kFewWarps - 1) / kFewWarps;    // pages p_begin + warp + 4 i
    const uint8_t* kh = kv.k + (size_t)h * F::HALF_BYTES;
    const uint8_t* vh = kv.v + (size_t)h * F::HALF_BYTES;

    int ahead_pages = 0;                                                        // lane i: the page of the warp's (ahead / 32 * 32 + i)-th
    auto load = [&](int i) {
        if ((i & 31) == 0) ahead_pages = i + lane < n_mine ? table[p_begin + warp + kFewWarps * (i + lane)] : 0;
        const size_t page = __shfl_sync(0xffffffffu, ahead_pages, i & 31);
        const uint32_t dst = ring + (i % F::STAGES) * 2 * F::HALF_BYTES;
        const uint8_t* ks = kh + page * kv.k_stride + tile_row(0, g) * HD + t4 * F::PIECE;
        const uint8_t* vs = vh + page * kv.v_stride + g * kPageTokens + t4 * 16;
#pragma unroll
        for (int r = 0; r < 8; ++r)                                             // tile r / 2, rows g (even r) and g + 8
#pragma unroll
            for (int p = 0; p < F::PIECES; ++p)
                copy_async<F::PIECE>(dst + ((r * F::PIECES + p) * 32 + lane) * F::PIECE, ks + 2 * r * HD + p * 4 * F::PIECE);
#pragma unroll
        for (int i8 = 0; i8 < HD / 8; ++i8) copy_async<16>(dst + F::HALF_BYTES + (i8 * 32 + lane) * 16, vs + i8 * 8 * kPageTokens);
    };
    // Pages before the newest were complete before the kernel that stores this step's rows began (it lets its successor begin
    // only after its own wait), so their copies may start while it runs; the pages that take new rows may not.
    const int p_new = span.start / kPageTokens;
    int ahead = 0;
#pragma unroll
    for (int s = 0; s < F::STAGES - 1; ++s) {
        if (ahead == s && s < n_mine && p_begin + warp + kFewWarps * s < p_new) load(ahead++);
    }
    chain_wait();
#pragma unroll
    for (int s = 0; s < F::STAGES - 1; ++s) {
        if (ahead == s && s < n_mine) load(ahead++);
        cp_async_commit();
    }

    // ---- queries: column g of each tile of 8, a lane's channels of each piece; scaled to fill half's range
    uint32_t qf[NT][F::STEPS][2];
    float q_factor[NT];                                                         // of column g: what a score is multiplied with
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int c = c0 + nt * 8 + g;
        const bool real = c < n_columns;
        const bf16* src = a.q + (size_t)(span.first + (real ? c / a.group : 0)) * a.ldq + (size_t)(h * a.group + (real ? c % a.group : 0)) * HD;
        float x[F::STEPS][4];
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < F::STEPS; ++s) {
            const int d = s / (F::PIECE / 4) * 4 * F::PIECE + t4 * F::PIECE + s % (F::PIECE / 4) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[s][e] = real ? __bfloat162float(src[d + e]) : 0.f;
                most = fmaxf(most, fabsf(x[s][e]));
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^(14 - exponent of the largest): within what a float's exponent can say; 1 for rows of zeros and of infinities
        const int e = (int)(__float_as_uint(most) >> 23);
        const int up = (e == 0 || e == 255) ? 0 : min(max(14 - (e - 127), -100), 100);
        const float f = __uint_as_float((uint32_t)(127 + up) << 23);
        q_factor[nt] = a.scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int s = 0; s < F::STEPS; ++s) {
            qf[nt][s][0] = pack_f16(x[s][0] * f, x[s][1] * f);
            qf[nt][s][1] = pack_f16(x[s][2] * f, x[s][3] * f);
        }
    }
    // the two columns a lane has in score tiles: 2 t4 and 2 t4 + 1
    float factor[NT][2], m[NT][2], l[NT][2];
    int seen_to[NT][2];                                                         // last row a column sees; -1: no such column
    int least_to = 0x7fffffff, most_to = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            factor[nt][e] = __shfl_sync(0xffffffffu, q_factor[nt], (2 * t4 + e) * 4);
            const int c = c0 + nt * 8 + 2 * t4 + e;
            seen_to[nt][e] = c < n_columns ? span.start + c / a.group : -1;
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
        }
    least_to = span.start + c0 / a.group;
    most_to = span.start + min(n_columns - 1, c0 + 8 * NT - 1) / a.group;
    float o[F::STEPS][NT][4];
#pragma unroll
    for (int i = 0; i < F::STEPS; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;

    float k_scales = 0.f, v_scales = 0.f;                                       // lane i: of the warp's (i / 32 * 32 + i)-th page
    for (int i = 0; i < n_mine; ++i) {
        const int p = p_begin + warp + kFewWarps * i;
        if ((i & 31) == 0 && i + lane < n_mine) {
            const float* s = kv.scales + (size_t)table[p + kFewWarps * lane] * kv.scale_stride + h;
            k_scales = s[0];
            v_scales = s[kv.n_kv];
        }
        const float k_scale = __shfl_sync(0xffffffffu, k_scales, i & 31), v_scale = __shfl_sync(0xffffffffu, v_scales, i & 31);
        cp_async_wait<F::STAGES - 2>();
        if (ahead < n_mine) load(ahead++);                                      // where page i - 1 was
        cp_async_commit();
        const unsigned char* stage = smem + (warp * F::STAGES + i % F::STAGES) * 2 * F::HALF_BYTES;
        // ---- scores of the page's 64 rows
        float s[4][NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w[2][F::STEPS];                                            // four codes a k step of rows g and g + 8
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int pc = 0; pc < F::PIECES; ++pc) {
                    const unsigned char* at = stage + (((2 * j + r) * F::PIECES + pc) * 32 + lane) * F::PIECE;
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
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][nt][e] = 0.f;
#pragma unroll
            for (int k = 0; k < F::STEPS; ++k) {
                const uint32_t f[4] = {e4m3_pair_f16(w[0][k]), e4m3_pair_f16(w[1][k]), e4m3_pair_f16(w[0][k] >> 16), e4m3_pair_f16(w[1][k] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[j][nt], f, qf[nt][k][0], qf[nt][k][1]);
            }
        }
        const bool all_seen = p * kPageTokens + kPageTokens - 1 <= least_to && (a.window <= 0 || p * kPageTokens > most_to - a.window) &&
                              c0 + 8 * NT <= n_columns;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = factor[nt][e] * k_scale;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[j][nt][e] *= f;
                    s[j][nt][2 + e] *= f;
                }
                if (!all_seen) {
                    const int to = seen_to[nt][e], from = a.window > 0 ? to - a.window : -1;       // rows from + 1 .. to
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = p * kPageTokens + tile_row(j, g + 8 * r);
                            if (row > to || row <= from) s[j][nt][2 * r + e] = -INFINITY;
                        }
                }
            }
        if (a.scores && p < a.score_pages) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = c0 + nt * 8 + 2 * t4 + e;
                    if (c < n_columns) {
                        float4* at = reinterpret_cast<float4*>(a.scores + ((((size_t)b * kv.n_kv + h) * a.columns + c) * a.score_pages + p) * kPageTokens + g * 8);
                        at[0] = make_float4(s[0][nt][e], s[0][nt][2 + e], s[1][nt][e], s[1][nt][2 + e]);
                        at[1] = make_float4(s[2][nt][e], s[2][nt][2 + e], s[3][nt][e], s[3][nt][2 + e]);
                    }
                }
        }
        // ---- running maximum and sum; probabilities as the second product's right operand
        float corr[NT][2];
        uint32_t pf[4][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(fmaxf(fmaxf(s[0][nt][e], s[0][nt][2 + e]), fmaxf(s[1][nt][e], s[1][nt][2 + e])),
                                 fmaxf(fmaxf(s[2][nt][e], s[2][nt][2 + e]), fmaxf(s[3][nt][e], s[3][nt][2 + e])));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float now = fmaxf(m[nt][e], mx);
                const float use = now == -INFINITY ? 0.f : now;
                corr[nt][e] = exp2_fast(m[nt][e] - use);
                m[nt][e] = now;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[j][nt][e] = exp2_fast(s[j][nt][e] - use + kPShift);
                    s[j][nt][2 + e] = exp2_fast(s[j][nt][2 + e] - use + kPShift);
                    sum += s[j][nt][e] + s[j][nt][2 + e];
                }
                l[nt][e] = l[nt][e] * corr[nt][e] + sum;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                pf[j][nt][0] = transpose_8x8(pack_f16(s[j][nt][0], s[j][nt][1]));
                pf[j][nt][1] = transpose_8x8(pack_f16(s[j][nt][2], s[j][nt][3]));
            }
        }
        // ---- O^T += V^T P^T, 16 channels at a time
        bool odd = false;                                                       // a NaN code in a page that not every column sees whole
#pragma unroll
        for (int i8 = 0; i8 < F::STEPS; ++i8) {
            uint32_t w[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint4 u = *reinterpret_cast<const uint4*>(stage + F::HALF_BYTES + ((2 * i8 + r) * 32 + lane) * 16);
                w[r][0] = u.x; w[r][1] = u.y; w[r][2] = u.z; w[r][3] = u.w;
            }
            if (!all_seen) {
                // A row that a column does not see has probability 0 there; its values may still be the NaN code, which
                // 0 does not silence.  They are taken out here and given back below to the columns that do see them.
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t nan = __vcmpeq4(w[r][j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        odd |= nan != 0;
                        w[r][j] &= ~nan;
                    }
            }
            float t[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) t[nt][0] = t[nt][1] = t[nt][2] = t[nt][3] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t f[4] = {e4m3_pair_f16(w[0][j]), e4m3_pair_f16(w[1][j]), e4m3_pair_f16(w[0][j] >> 16), e4m3_pair_f16(w[1][j] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_16816(t[nt], f, pf[j][nt][0], pf[j][nt][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i8][nt][e] = fmaf(o[i8][nt][e], corr[nt][e & 1], t[nt][e] * v_scale);
        }
        if (__any_sync(0xffffffffu, odd)) {
            // how many NaN codes of rows it sees a column meets in each channel: ones for the codes, ones for the rows seen
            uint32_t seen[4][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float v[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int to = seen_to[nt][e], row = p * kPageTokens + tile_row(j, g + 8 * r);
                            v[e] = row <= to && (a.window <= 0 || row > to - a.window) ? 1.f : 0.f;
                        }
                        seen[j][nt][r] = transpose_8x8(pack_f16(v[0], v[1]));
                    }
#pragma unroll
            for (int i8 = 0; i8 < F::STEPS; ++i8) {
                uint32_t w[2][4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint4 u = *reinterpret_cast<const uint4*>(stage + F::HALF_BYTES + ((2 * i8 + r) * 32 + lane) * 16);
                    w[r][0] = u.x; w[r][1] = u.y; w[r][2] = u.z; w[r][3] = u.w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[r][j] = __vcmpeq4(w[r][j] & 0x7f7f7f7fu, 0x7f7f7f7fu) & 0x38383838u;   // 0x38: 1.0
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t f[4] = {e4m3_pair_f16(w[0][j]), e4m3_pair_f16(w[1][j]), e4m3_pair_f16(w[0][j] >> 16), e4m3_pair_f16(w[1][j] >> 16)};
                        mma_f16_16816(t, f, seen[j][nt][0], seen[j][nt][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (t[e] > 0.f) o[i8][nt][e] = __uint_as_float(0x7fc00000u);
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();                                                            // the ring becomes the place where the warps meet

    // ---- the four warps' shares joined in their order
    float* mo = reinterpret_cast<float*>(smem);                                 // [warp][column][HD]
    float* ml = mo + kFewWarps * 8 * NT * HD;                                   // [warp][column][2]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[nt][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int c = warp * 8 * NT + nt * 8 + 2 * t4 + e;
            if (g == 0) { ml[2 * c] = m[nt][e]; ml[2 * c + 1] = sum; }
#pragma unroll
            for (int i8 = 0; i8 < F::STEPS; ++i8) {
                mo[c * HD + 16 * i8 + g] = o[i8][nt][e];
                mo[c * HD + 16 * i8 + g + 8] = o[i8][nt][2 + e];
            }
        }
    __syncthreads();
    const int n_here = min(8 * NT, n_columns - c0);
    for (int idx = tid; idx < n_here * HD; idx += kFewThreads) {
        const int c = idx / HD, d = idx % HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, ml[2 * (w * 8 * NT + c)]);
        const float use = M == -INFINITY ? 0.f : M;
        float acc = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float f = exp2_fast(ml[2 * (w * 8 * NT + c)] - use);
            acc += f * mo[(w * 8 * NT + c) * HD + d];
            L += f * ml[2 * (w * 8 * NT + c) + 1];
        }
        if (a.n_splits == 1) {
            const int col = c0 + c;
            a.out[(size_t)(span.first + col / a.group) * a.ldo + (size_t)(h * a.group + col % a.group) * HD + d] = __float2bfloat16_rn(acc / L);
        } else {
            a.part_o[(part + c) * HD + d] = acc;
        }
        if (d == 0 && a.part_ml) { a.part_ml[(part + c) * 2] = M; a.part_ml[(part + c) * 2 + 1] = L; }
    }
}

// Joins the splits (blocks x < join_blocks: columns of one (sequence, kv head)) and, where weights are gathered, adds to
// them (the other blocks, four pages at a time).
constexpr int kJoinThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kJoinThreads)
few_join_kernel(const FewArgs a, const E4M3Pages kv, int join_blocks) {
    chain_release();
    chain_wait();
    __shared__ float top[kFewColumns], inverse[kFewColumns];
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const FewSpan span = few_span(a, kv, b);
    const int n_columns = span.n_new * a.group;
    if (n_columns <= 0) return;
    const int used = (span.p_last - span.p_first + span.per_split) / span.per_split;    // splits that have pages
    const size_t base = ((size_t)b * kv.n_kv + h) * a.n_splits * a.columns;
    for (int c = tid >> 5; c < n_columns; c += kJoinThreads / 32) {             // a warp a column: its maximum and sum over the splits
        float M = -INFINITY, L = 0.f;
        for (int s = tid & 31; s < used; s += 32) M = fmaxf(M, a.part_ml[(base + (size_t)s * a.columns + c) * 2]);
        M = warp_max(M);
        const float use = M == -INFINITY ? 0.f : M;
        for (int s = tid & 31; s < used; s += 32) {
            const float* ml = a.part_ml + (base + (size_t)s * a.columns + c) * 2;
            L += exp2_fast(ml[0] - use) * ml[1];
        }
        L = warp_sum(L);
        if ((tid & 31) == 0) { top[c] = use; inverse[c] = 1.0f / L; }
    }
    __syncthreads();
    if ((int)blockIdx.x < join_blocks) {
        for (int idx = blockIdx.x * kJoinThreads + tid; idx < n_columns * HD; idx += join_blocks * kJoinThreads) {
            const int c = idx / HD, d = idx % HD;
            float acc = 0.f;
            for (int s = 0; s < used; ++s) {
                const size_t at = base + (size_t)s * a.columns + c;
                acc += exp2_fast(a.part_ml[at * 2] - top[c]) * a.part_o[at * HD + d];
            }
            a.out[(size_t)(span.first + c / a.group) * a.ldo + (size_t)(h * a.group + c % a.group) * HD + d] = __float2bfloat16_rn(acc * inverse[c]);
        }
        return;
    }
    const int* table = kv.block_table + (size_t)a.slots[b] * kv.table_stride;
    const int stride = ((int)gridDim.x - join_blocks) * (kJoinThreads / kPageTokens);
    for (int p = span.p_first + ((int)blockIdx.x - join_blocks) * (kJoinThreads / kPageTokens) + tid / kPageTokens; p <= span.p_last; p += stride) {
        const int t = tid % kPageTokens, row = p * kPageTokens + t;
        if (row >= span.start + span.n_new) continue;
        const size_t page = table[p];
        float sum = 0.f;
        if (p < a.score_pages) {
            const float* at = a.scores + (((size_t)b * kv.n_kv + h) * a.columns * a.score_pages + p) * kPageTokens + score_place(t);
            for (int c = 0; c < n_columns; ++c)
                sum += exp2_fast(at[(size_t)c * a.score_pages * kPageTokens] - top[c] + kPShift) * inverse[c];
        } else {                                                                // a sequence that has outgrown the plan: score the row again
            const uint8_t* kr = kv.k + page * kv.k_stride + ((size_t)h * kPageTokens + t) * HD;
            const float k_scale = kv.scales[page * kv.scale_stride + h] * a.scale * kLog2e;
            for (int c = 0; c < n_columns; ++c) {
                const int to = span.start + c / a.group;
                if (row > to || (a.window > 0 && row <= to - a.window)) continue;
                const bf16* qr = a.q + (size_t)(span.first + c / a.group) * a.ldq + (size_t)(h * a.group + c % a.group) * HD;
                float s = 0.f;
                for (int d = 0; d < HD; ++d) s = fmaf(__bfloat162float(qr[d]), e4m3_value(kr[d]), s);
                sum += exp2_fast(s * k_scale - top[c] + kPShift) * inverse[c];
            }
        }
        kv.weights[page * kv.weight_stride + h * kPageTokens + t] += sum;
    }
}

// How the pages are shared out: pages a split takes, splits of the longest sequence, pages whose scores are kept.
struct FewPlan {
    int n_splits, chunk_pages, columns, score_pages;
    long long part_o, part_ml, scores;                                          // floats of scratch, each a multiple of 4
    long long floats() const { return part_o + part_ml + scores; }
};

template <int HD>
int few_blocks_per_sm() {
    static int cached = 0;
    if (cached == 0) {
        int n = 0;
        if (cudaFuncSetAttribute(few_queries_kernel<HD, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<HD>::smem(1)) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, few_queries_kernel<HD, 1>, kFewThreads, Few<HD>::smem(1)) != cudaSuccess || n < 1) {
            (void)cudaGetLastError();
            n = 1;
        }
        cached = n;
    }
    return cached;
}

bool few_takes(int dtype, int max_q_len, int n_heads, int n_kv, int hd) {
    return dtype == 1 && hd % 16 == 0 && hd <= 128 && (long long)max_q_len * (n_heads / n_kv) <= kFewColumns;
}

template <int HD>
FewPlan few_plan_for(int B, int max_q_len, int n_heads, int n_kv, int max_kv_len, long long total_kv_len, int window, int weigh) {
    FewPlan plan;
    plan.columns = max_q_len * (n_heads / n_kv);
    const long long max_pages_all = (max_kv_len + kPageTokens - 1) / kPageTokens;
    long long max_pages = max_pages_all;
    if (window > 0) max_pages = min(max_pages, (long long)(window + max_q_len + kPageTokens - 2) / kPageTokens + 1);
    if (total_kv_len <= 0) total_kv_len = (long long)B * max_kv_len;
    const long long total_pages = max((long long)B, min(total_kv_len / kPageTokens + B, max_pages * B));
    const int nt = plan.columns > 8 ? 2 : 1;
    const long long units = (long long)n_kv * ((plan.columns + 8 * nt - 1) / (8 * nt));
    // enough blocks to fill the device about GTG_FEW_WAVES times over, none of less than four pages (a page a warp)
    const long long slots = 148LL * few_blocks_per_sm<HD>();
#ifndef GTG_FEW_WAVES
#define GTG_FEW_WAVES 2
#endif
    long long chunk = (total_pages * units + GTG_FEW_WAVES * slots - 1) / (GTG_FEW_WAVES * slots);
    chunk = max(chunk, 4LL);
    chunk = min(chunk, max_pages);
    long long splits = (max_pages + chunk - 1) / chunk;
    splits = min(splits, 256LL);
    plan.chunk_pages = (int)((max_pages + splits - 1) / splits);
    plan.n_splits = (int)splits;
    plan.score_pages = weigh ? (int)max_pages_all : 0;
    const long long parts = (long long)B * n_kv * splits * plan.columns;
    plan.part_o = splits > 1 ? parts * HD : 0;
    plan.part_ml = splits > 1 || weigh ? (parts * 2 + 3) / 4 * 4 : 0;
    plan.scores = (long long)B * n_kv * plan.columns * plan.score_pages * kPageTokens;
    return plan;
}

template <int HD, int NT>
int launch_few_tiles(const FewArgs& a, const E4M3Pages& kv, int B, cudaStream_t stream) {
    static bool configured = false;
    constexpr int smem = Few<HD>::smem(NT);
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(few_queries_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    const int tiles = (a.columns + 8 * NT - 1) / (8 * NT);
    return launch_chained(few_queries_kernel<HD, NT>, dim3(a.n_splits, kv.n_kv * tiles, B), dim3(kFewThreads), smem, stream, a, kv);
}

template <int HD>
int launch_few(FewArgs a, const E4M3Pages& kv, const FewPlan& plan, int B, float* scratch, cudaStream_t stream) {
    a.n_splits = plan.n_splits;
    a.chunk_pages = plan.chunk_pages;
    a.columns = plan.columns;
    a.score_pages = plan.score_pages;
    a.part_o = plan.part_o ? scratch : nullptr;
    a.part_ml = plan.part_ml ? scratch + plan.part_o : nullptr;
    a.scores = plan.scores ? scratch + plan.part_o + plan.part_ml : nullptr;
    const int st = plan.columns > 8 ? launch_few_tiles<HD, 2>(a, kv, B, stream) : launch_few_tiles<HD, 1>(a, kv, B, stream);
    if (st != 0 || plan.part_ml == 0) return st;
    const int join = plan.n_splits > 1 ? (plan.columns * HD + kJoinThreads - 1) / kJoinThreads : 0;
    const int pages = plan.score_pages ? (plan.score_pages * kPageTokens + kJoinThreads - 1) / kJoinThreads : 0;
    return launch_chained(few_join_kernel<HD>, dim3(join + pages, kv.n_kv, B), dim3(kJoinThreads), 0, stream, a, kv, join);
}
}  // namespace
