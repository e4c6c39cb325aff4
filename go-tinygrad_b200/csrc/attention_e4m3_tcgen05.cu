// Attention of prompts and chunks over the 8-bit cache on the fifth-generation tensor cores: heads of 64 or 128 channels,
// bfloat16 queries, causal, with an optional window.  (Layout and codes: e4m3.cuh.)
//
// One block per (128 query rows, key/value head, sequence).  A query row is a (token, head of the group) pair, heads
// innermost, so that the heads that share keys share their pages too and a short run of queries still fills a tile.  Per step of BK
// rows of the cache (two pages for heads of 64 channels, one for 128):
//   codes -> half   three warps fetch the step's codes (asynchronous copies, two or three steps ahead), turn them into halves,
//                   which is exact, and leave them in shared memory as swizzled tiles: keys [row][channel], values
//                   [channel][row], both K-major as the cache has them;
//   S  = Q K^T      tcgen05.mma 128 x BK x head size, operands in shared memory, S in tensor memory; queries are scaled by a
//                   power of two a row to fill half's range, so that rounding bfloat16 to half loses nothing that counts;
//   P  = softmax    four warps, a thread a row, scores straight from tensor memory; P goes back there as halves;
//   O += P V        tcgen05.mma 128 x head size x BK, A = P from tensor memory, O stays there.
// Scales.  A page's key scale multiplies its scores.  Its value scale 2^v cannot multiply O, which adds up over pages, and
// must not squeeze P's range either: it goes into the exponent.  With x_j = score_j + v_j (in powers of two) and M the running
// maximum of x, P_j = 2^(x_j - M), O = sum P_j code_j and the sum is l = sum P_j 2^(-v_j): O / l is the result, whatever the
// scales (as long as two blocks of values that both count are not 2^100 apart).  M is raised only when a step's maximum exceeds it
// by 2^8; P, times 2^7 besides, then stays below half's largest number.
// What bounds it: for 128 channels the two products (the conversion's 1.5 operations a pair of codes and its stores run beside
// them), for 64 the exponentials, one a score at 16 a cycle.  Every wait is bounded (status word as in the products).
#include "e4m3.cuh"
#include "tcgen05_attention.cuh"

namespace {
constexpr int BQ = 128;
constexpr int kConvWarps = 3;
constexpr int kThreads = 32 * (5 + kConvWarps);          // softmax 0-3, products 4, conversion 5-7
constexpr int kTmemCols = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaiseBy = 8.0f, kPShift = 7.0f;
// Registers: the softmax's warps hold a step's scores, the others little; 168 + 88 is twice the 128 a thread is launched with.
constexpr int kSoftmaxRegs = 168, kOtherRegs = 88;

template <int HD> struct Shape {
    static constexpr int kPages = HD == 64 ? 2 : 1;      // of a step
    static constexpr int BK = 64 * kPages;
    static constexpr int kStages = 2;                    // key tiles; one value tile: it is wanted a softmax later
    static constexpr int kRaw = HD == 64 ? 3 : 2;        // steps of codes on their way
    static constexpr int kQBytes = BQ * HD * 2, kTileBytes = BK * HD * 2;
    static constexpr int kOffK = kQBytes, kOffV = kOffK + kStages * kTileBytes, kOffRaw = kOffV + kTileBytes;
    static constexpr int kRawBytes = BK * HD;            // a step's codes of keys (or of values)
    static constexpr int kOffBar = kOffRaw + kRaw * 2 * kRawBytes;
    static constexpr int kSmemBytes = kOffBar + 256;
    static constexpr int kColO = BK, kColP = BK + HD;
    static_assert(BK + HD + BK / 2 <= kTmemCols, "tensor memory");
    static constexpr int kPieces = BK * HD / 16;         // of 16 codes in a step's keys (or values): 512
    static constexpr int kMine = (kPieces + 32 * kConvWarps - 1) / (32 * kConvWarps);
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
    float2* stats;               // [token][head]: what a score (in powers of two) is compared with, and the sum; or null
};

__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
    return u;
}
// 16-byte copy global -> shared; `bytes` = 0 fills the destination with zeros.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 16 codes as 16 halves: two chunks of a swizzled row.
__device__ __forceinline__ void store_halves(uint32_t row_at, int chunk, int swizzle, const uint4& u) {
    store_shared16(row_at + ((chunk ^ swizzle) << 4), e4m3_pair_f16(u.x), e4m3_pair_f16(u.x >> 16), e4m3_pair_f16(u.y), e4m3_pair_f16(u.y >> 16));
    store_shared16(row_at + (((chunk + 1) ^ swizzle) << 4), e4m3_pair_f16(u.z), e4m3_pair_f16(u.z >> 16), e4m3_pair_f16(u.w), e4m3_pair_f16(u.w >> 16));
}
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// grid: (kv heads, sequences, tiles of query rows), the longest tiles first.
template <int HD, bool kTest>
__global__ void __launch_bounds__(kThreads, 2)
attention_e4m3_prompt_kernel(const PromptArgs a, const E4M3Pages kv) {
    using S = Shape<HD>;
    constexpr int BK = S::BK;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int h = blockIdx.x, b = blockIdx.y;
    const int tile = gridDim.z - 1 - blockIdx.z;
    const int q_begin = a.cu_seqlens[b];
    const int q_len = a.cu_seqlens[b + 1] - q_begin;
    const int n_rows = q_len * a.group;
    if (tile * BQ >= n_rows) return;                             // before any barrier or tensor memory
    const uint32_t base = smem_addr(smem);
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicExch(&g_status, 2);
        return;
    }
    const uint32_t bars = base + S::kOffBar;
    const uint32_t q_full = bars, s_full = bars + 8, s_free = bars + 16, p_full = bars + 24, pv_done = bars + 32;
    auto k_full = [&](int s) { return bars + 40u + 8u * s; };
    auto k_free = [&](int s) { return bars + 56u + 8u * s; };
    const uint32_t v_full = bars + 72, v_free = bars + 80;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::kOffBar + 128);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffBar + 136);
    volatile int* odd_flag = reinterpret_cast<volatile int*>(smem + S::kOffBar + 140);   // a NaN code in a page not all rows see whole

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = a.slots[b];
    const int start = a.start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    const int* table = kv.block_table + (size_t)slot * kv.table_stride;
    const int row0 = tile * BQ;
    const int rows_here = min(BQ, n_rows - row0);
    const int first_at = start + row0 / a.group;                 // cache row of the tile's first query, and of its last
    const int last_at = start + (row0 + rows_here - 1) / a.group;
    const int k_min = a.window > 0 ? max(0, first_at - a.window + 1) : 0;
    const int j_lo = k_min / kPageTokens, j_hi = last_at / kPageTokens;
    const int n_steps = (j_hi - j_lo + S::kPages) / S::kPages;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4);
        mbar_init(s_full, 1);
        mbar_init(s_free, 4);
        mbar_init(p_full, 4);
        mbar_init(pv_done, 1);
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(k_full(s), kConvWarps);
            mbar_init(k_free(s), 1);
        }
        mbar_init(v_full, kConvWarps);
        mbar_init(v_free, 1);
        *abort_flag = 0;
        *odd_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::);
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(smem_addr(tmem_holder)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
    const uint32_t tmem_s = *tmem_holder, tmem_o = tmem_s + S::kColO, tmem_p = tmem_s + S::kColP;
    chain_wait();                                                // queries and the newest rows come from the kernel before
    chain_release();

    if (warp >= 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (warp >= 5) {
            // ------------------------------------------------------------ codes to halves
            const int t = threadIdx.x - 5 * 32;
            const int total = start + q_len;                     // rows that exist after this step
            auto page_of = [&](int i, int pg) { const int j = j_lo + S::kPages * i + pg; return j <= j_hi ? j : -1; };
            // The codes come by asynchronous copies, kRaw steps ahead, each 16-byte piece to a place that only the lane that will
            // convert it reads: nothing is waited for but a lane's own copies.  Page numbers are read a step earlier still.
            int page_k[S::kPages], page_v[S::kPages];            // of the next step to be asked for: page or -1
            auto look_up = [&](int i, int* page) {
#pragma unroll
                for (int pg = 0; pg < S::kPages; ++pg) {
                    const int j = page_of(i, pg);
                    page[pg] = j >= 0 ? table[j] : -1;
                }
            };
            auto slot_of = [&](int i, int values, int id) { return base + S::kOffRaw + ((i % S::kRaw) * 2 + values) * S::kRawBytes + id * 16; };
            auto ask = [&](int i, int values, int* page) {
                if (i < n_steps) {
#pragma unroll
                    for (int m = 0; m < S::kMine; ++m) {
                        const int id = t + 32 * kConvWarps * m;
                        if (id < S::kPieces) {
                            const int pg = id / (S::kPieces / S::kPages), in = id % (S::kPieces / S::kPages), p = S::kPages == 1 || pg == 0 ? page[0] : page[S::kPages - 1];
                            const uint8_t* at = values ? kv.v + (size_t)max(p, 0) * kv.v_stride : kv.k + (size_t)max(p, 0) * kv.k_stride;
                            // a page behind the last: zeros, which no row sees
                            copy_async16(slot_of(i, values, id), at + (size_t)h * kPageTokens * HD + in * 16, p >= 0 ? 16 : 0);
                        }
                    }
                    look_up(i + 1, page);
                }
                asm volatile("cp.async.commit_group;\n" ::);
            };
            look_up(0, page_k);
            look_up(0, page_v);
            for (int i = 0; i < S::kRaw; ++i) { ask(i, 0, page_k); ask(i, 1, page_v); }
            for (int i = 0; i < n_steps; ++i) {
                const int s = i % S::kStages;
                asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S::kRaw - 1));
                if (!__all_sync(0xffffffffu, mbar_wait<kTest>(k_free(s), (((uint32_t)i / S::kStages) & 1u) ^ 1u, abort_flag))) break;
                const uint32_t kt = base + S::kOffK + s * S::kTileBytes;
#pragma unroll
                for (int m = 0; m < S::kMine; ++m) {
                    const int id = t + 32 * kConvWarps * m;
                    if (id < S::kPieces) {
                        const int row = id / (HD / 16), piece = id % (HD / 16);
                        store_halves(kt + (piece / 4) * (BK * 128) + row * 128, piece % 4 * 2, row & 7, load_shared16(slot_of(i, 0, id)));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0 && !Waits<kTest>::kSkipCopies) mbar_arrive(k_full(s));
                ask(i + S::kRaw, 0, page_k);
                asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S::kRaw - 1));
                if (!__all_sync(0xffffffffu, mbar_wait<kTest>(v_free, ((uint32_t)i & 1u) ^ 1u, abort_flag))) break;
                const uint32_t vt = base + S::kOffV;
#pragma unroll
                for (int m = 0; m < S::kMine; ++m) {
                    const int id = t + 32 * kConvWarps * m;
                    if (id < S::kPieces) {
                        uint4 v = load_shared16(slot_of(i, 1, id));
                        const int pg = id / (HD * 4), channel = id / 4 % HD, piece = id % 4;
                        const int j = page_of(i, pg), at = j * kPageTokens + piece * 16;       // rows at .. at + 15
                        if (j >= 0 && (j * kPageTokens + kPageTokens - 1 > first_at || (a.window > 0 && j * kPageTokens <= last_at - a.window))) {
                            // A page that not every query sees whole.  Rows nobody has written yet become zeros; so do NaN codes, which
                            // P's zeros would not silence: who does see them gets them back at the end.
                            uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            uint32_t found = 0;
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int there = min(max(total - at - 4 * c, 0), 4);           // rows of this word that exist
                                w[c] &= there == 4 ? 0xffffffffu : (1u << (8 * there)) - 1u;
                                const uint32_t nan = nan_codes(w[c]);
                                found |= nan;
                                w[c] &= ~nan;
                            }
                            if (found) *odd_flag = 1;
                            v = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        store_halves(vt + pg * (HD * 128) + channel * 128, piece * 2, channel & 7, v);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0 && !Waits<kTest>::kSkipCopies) mbar_arrive(v_full);
                ask(i + S::kRaw, 1, page_v);
            }
            asm volatile("cp.async.wait_group 0;\n" ::);
        } else if (lane == 0) {
            // ------------------------------------------------------------ products
            const uint32_t idesc_s = f16_idesc(BQ, BK), idesc_pv = f16_idesc(BQ, HD);
            bool ok = mbar_wait<kTest>(q_full, 0, abort_flag);
            auto issue_s = [&](int i) {
                const int s = i % S::kStages;
                if (!mbar_wait<kTest>(k_full(s), ((uint32_t)i / S::kStages) & 1u, abort_flag)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                const uint32_t kbase = base + S::kOffK + s * S::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint64_t dq = umma_desc(base + (kk / 4) * (BQ * 128)) + 2 * (kk % 4);
                    const uint64_t dk = umma_desc(kbase + (kk / 4) * (BK * 128)) + 2 * (kk % 4);
                    umma_ss(tmem_s, dq, dk, idesc_s, kk > 0 ? 1u : 0u);
                }
                umma_commit(k_free(s));
                umma_commit(s_full);
                return true;
            };
            if (ok) ok = issue_s(0);
            for (int i = 0; i < n_steps && ok; ++i) {
                if (i + 1 < n_steps) {
                    ok = mbar_wait<kTest>(s_free, (uint32_t)i & 1u, abort_flag) && issue_s(i + 1);
                    if (!ok) break;
                }
                ok = mbar_wait<kTest>(v_full, (uint32_t)i & 1u, abort_flag) &&
                     mbar_wait<kTest>(p_full, (uint32_t)i & 1u, abort_flag);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) {
                    const uint64_t dv = umma_desc(base + S::kOffV + (kk / 4) * (HD * 128)) + 2 * (kk % 4);
                    umma_ts(tmem_o, tmem_p + 8 * kk, dv, idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
                }
                umma_commit(v_free);
                umma_commit(pv_done);
            }
        }
    } else {
        // ------------------------------------------------------------ softmax and output: a thread a query row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        const unsigned full = 0xffffffffu;
        const int r = warp * 32 + lane;
        const bool real = r < rows_here;
        const int token = (row0 + (real ? r : 0)) / a.group, head = h * a.group + (row0 + (real ? r : 0)) % a.group;
        const int pos = start + token;                            // the query's own cache row
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        float factor;                                             // a raw score times this and the page's key scale: powers of two
        {
            const bf16* src = a.q + (size_t)(q_begin + token) * a.ldq + (size_t)head * HD;
            uint4 u[HD / 8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                u[c] = real ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = fabsf(__uint_as_float(w[e] << 16)), hi = fabsf(__uint_as_float(w[e] & 0xffff0000u));
                    most = fmaxf(most, fmaxf(finite_f32(lo) ? lo : 0.f, finite_f32(hi) ? hi : 0.f));
                }
            }
            // the largest channel comes to lie in [2^14, 2^15); a negative scale turns the queries round
            const int e = (int)(__float_as_uint(most) >> 23);
            const int up = e == 0 ? 0 : min(max(14 - (e - 127), -100), 100);
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
                store_shared16(base + (c / 8) * (BQ * 128) + r * 128 + (((c % 8) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        // scales of the step's pages, read a step ahead
        float k_next[S::kPages], v_next[S::kPages];
        auto fetch_scales = [&](int i) {
#pragma unroll
            for (int pg = 0; pg < S::kPages; ++pg) {
                const int j = j_lo + S::kPages * i + pg;
                const float* at = kv.scales + (size_t)table[j <= j_hi ? j : j_hi] * kv.scale_stride + h;
                k_next[pg] = at[0];
                v_next[pg] = at[kv.n_kv];
            }
        };
        fetch_scales(0);
        float m_run = -INFINITY, l_run = 0.f;
        uint32_t sv[BK];
        bool ok = true;
        for (int i = 0; i < n_steps; ++i) {
            const int key0 = (j_lo + S::kPages * i) * kPageTokens;
            float sl[S::kPages], add[S::kPages], back[S::kPages];
#pragma unroll
            for (int pg = 0; pg < S::kPages; ++pg) {
                sl[pg] = factor * k_next[pg];
                add[pg] = (float)((int)(__float_as_uint(v_next[pg]) >> 23) - 127);   // log2 of the value scale
                back[pg] = pow2_inverse(v_next[pg]);
            }
            if (i + 1 < n_steps) fetch_scales(i + 1);
            ok = __all_sync(full, mbar_wait<kTest>(s_full, (uint32_t)i & 1u, abort_flag));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
#pragma unroll
            for (int c = 0; c < BK / 32; ++c) tmem_ld32(tmem_s + lane_off + 32 * c, sv + 32 * c);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free);
            const bool all_visible = key0 + BK - 1 <= pos && (a.window <= 0 || key0 > pos - a.window);
            if (!all_visible) {
#pragma unroll
                for (int c = 0; c < BK; ++c) {
                    const int key = key0 + c;
                    if (key > pos || (a.window > 0 && key <= pos - a.window)) sv[c] = __float_as_uint(-INFINITY);
                }
            }
            float m_step = -INFINITY;
#pragma unroll
            for (int pg = 0; pg < S::kPages; ++pg) {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(sv[64 * pg + c + e]));
                m_step = fmaxf(m_step, fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), sl[pg], add[pg]));
            }
            if (i == 0) {
                m_run = m_step;
            } else {
                const bool raise = m_step > m_run + kRaiseBy;    // also: the first visible row of a query
                if (__any_sync(full, raise)) {
                    ok = __all_sync(full, mbar_wait<kTest>(pv_done, (uint32_t)(i - 1) & 1u, abort_flag));
                    if (!ok) break;
                    float corr = 1.0f;
                    if (raise) {
                        corr = fast_exp2(m_run - m_step);
                        m_run = m_step;
                        l_run *= corr;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                    uint32_t ov[8];
#pragma unroll 1
                    for (int part = 0; part < HD / 8; ++part) {
                        tmem_ld8(tmem_o + lane_off + 8 * part, ov);
                        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                        for (int d = 0; d < 8; ++d) ov[d] = __float_as_uint(__uint_as_float(ov[d]) * corr);
                        tmem_st8(tmem_o + lane_off + 8 * part, ov);
                    }
                }
            }
            const float m_use = (m_run == -INFINITY ? 0.f : m_run) - kPShift;
#pragma unroll
            for (int pg = 0; pg < S::kPages; ++pg) {
                const float shift = add[pg] - m_use;
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int c = 32 * pg; c < 32 * pg + 32; c += 4) {    // scores 2c .. 2c + 7 become words c .. c + 3
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = fmaf(__uint_as_float(sv[2 * c + e]), sl[pg], shift);
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = exp2_in_order(p[e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        l0 += p[2 * e];
                        l1 += p[2 * e + 1];
                        const __half2 hh = __floats2half2_rn(p[2 * e], p[2 * e + 1]);
                        sv[c + e] = *reinterpret_cast<const uint32_t*>(&hh);
                    }
                }
                l_run = fmaf(l0 + l1, back[pg], l_run);
            }
            if (i > 0) {
                ok = __all_sync(full, mbar_wait<kTest>(pv_done, (uint32_t)(i - 1) & 1u, abort_flag));
                if (!ok) break;
            }
#pragma unroll
            for (int c = 0; c < BK / 64; ++c) tmem_st32(tmem_p + lane_off + 32 * c, sv + 32 * c);
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        if (ok) ok = __all_sync(full, mbar_wait<kTest>(pv_done, (uint32_t)(n_steps - 1) & 1u, abort_flag));
        if (ok) {
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
            const float inv = 1.0f / l_run;
            if (a.stats && real) a.stats[(size_t)(q_begin + token) * a.n_heads + head] = make_float2((m_run == -INFINITY ? 0.f : m_run) - kPShift, l_run);
            bf16* dst = a.out + (size_t)(q_begin + token) * a.ldo + (size_t)head * HD;
            const bool odd = *odd_flag != 0;
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                tmem_ld32(tmem_o + lane_off + 32 * c, sv);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                if (odd && real) {
                    // NaN codes of rows that this query sees, in pages where they were taken out
                    for (int j = j_lo; j <= j_hi; ++j) {
                        if (!(j * kPageTokens + kPageTokens - 1 > first_at || (a.window > 0 && j * kPageTokens <= last_at - a.window))) continue;
                        const uint8_t* vp = kv.v + (size_t)table[j] * kv.v_stride + ((size_t)h * HD + 32 * c) * kPageTokens;
                        const int lo = a.window > 0 ? max(0, pos - a.window + 1 - j * kPageTokens) : 0, hi = min(pos - j * kPageTokens, kPageTokens - 1);
                        for (int tt = lo; tt <= hi; ++tt)
#pragma unroll
                            for (int d = 0; d < 32; ++d)
                                if ((vp[d * kPageTokens + tt] & 0x7f) == 0x7f) sv[d] = 0x7fc00000u;
                    }
                }
                if (real) {
#pragma unroll
                    for (int piece = 0; piece < 4; ++piece) {
                        uint32_t o4[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const __nv_bfloat162 hh = __floats2bfloat162_rn(__uint_as_float(sv[8 * piece + 2 * x]) * inv, __uint_as_float(sv[8 * piece + 2 * x + 1]) * inv);
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
    if (warp == 4) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_s), "r"(kTmemCols));
    }
}

template <int HD, bool kTest>
int launch(const PromptArgs& a, const E4M3Pages& kv, int B, int max_q_len, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(attention_e4m3_prompt_kernel<HD, kTest>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmemBytes);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    const long long rows = (long long)max_q_len * a.group;
    return launch_chained(attention_e4m3_prompt_kernel<HD, kTest>, dim3(kv.n_kv, B, (unsigned)((rows + BQ - 1) / BQ)), dim3(kThreads),
                          (size_t)Shape<HD>::kSmemBytes, stream, a, kv);
}
// ============================================================== gathered weights of prompts and chunks
// weight_j += sum over the queries that see row j, of all heads of the group, of 2^(score - x) / l, x and l the query's
// statistics that the attention left.  The products again, the other way round: one block per (128 rows of the cache, key/value
// head, sequence), the rows as the tile's rows, so that a thread owns a row and its sum:
//   K      converted once to bfloat16 (exact) into shared memory, S = K Q^T by tcgen05.mma 128 x 128 x head size;
//   Q      128 tokens of one head at a time by tensor copies through a ring, as they are (bfloat16);
//   sums   four warps, S from tensor memory, 1 / l folded into the exponent: one multiply-add, one exponential and one add a
//          score.  The exponentials bound it (16 a cycle).
// Nothing is shared between blocks, so a weight does not depend on what else runs.
constexpr int kWeightThreads = 192;                      // sums 0-3, copies 4, products 5
template <int HD> struct WeightShape {
    static constexpr int kStages = HD == 64 ? 3 : 2;
    static constexpr int kTileBytes = 128 * HD * 2;      // 128 rows of keys, or of queries
    static constexpr int kOffQ = kTileBytes, kOffY = kOffQ + kStages * kTileBytes, kOffBar = kOffY + 2 * 128 * 4;
    static constexpr int kSmemBytes = kOffBar + 256;
};

// Four codes as four bfloat16.
__device__ __forceinline__ void bf16_of_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t a = e4m3_pair_f16(w), b = e4m3_pair_f16(w >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    const __nv_bfloat162 p = __floats2bfloat162_rn(x.x, x.y), r = __floats2bfloat162_rn(y.x, y.y);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&r);
}

template <int HD, bool kTest>
__global__ void __launch_bounds__(kWeightThreads, 2)
e4m3_weights_kernel(const __grid_constant__ CUtensorMap map_q, const PromptArgs a, const E4M3Pages kv) {
    using S = WeightShape<HD>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int h = blockIdx.y, b = blockIdx.z;
    const int q_begin = a.cu_seqlens[b];
    const int q_len = a.cu_seqlens[b + 1] - q_begin;
    const int slot = a.slots[b];
    const int start = a.start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    if (q_len <= 0 || (int)blockIdx.x * 128 >= start + q_len) return;
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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int* table = kv.block_table + (size_t)slot * kv.table_stride;
    if (threadIdx.x == 0) {
        mbar_init(k_full, 4);
        for (int s = 0; s < S::kStages; ++s) { mbar_init(q_full(s), 1); mbar_init(q_free(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(s_full(s), 1); mbar_init(s_free(s), 4); mbar_init(y_full(s), 4); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::);
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(smem_addr(tmem_holder)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
    const uint32_t tmem = *tmem_holder;
    chain_wait();
    chain_release();

    // the tokens that see any of rows 128 kt .. 128 kt + 127: [t_lo, t_hi), cut into tiles for each head of the group
    struct Span { int t_lo, t_hi, per_head; };
    auto span_of = [&](int kt) {
        Span s;
        s.t_lo = max(0, kt * 128 - start);
        s.t_hi = a.window > 0 ? min((long long)q_len, (long long)kt * 128 + 127 + a.window - start) : q_len;
        s.per_head = s.t_hi > s.t_lo ? (s.t_hi - s.t_lo + 127) / 128 : 0;
        return s;
    };
    int n = 0;                                                   // tiles so far, of all turns
    if (warp == 4) {
        if (lane == 0) {
            bool ok = true;
            for (int kt = blockIdx.x; kt * 128 < start + q_len && ok; kt += gridDim.x) {
                const Span sp = span_of(kt);
                for (int i = 0; i < sp.per_head * a.group; ++i, ++n) {
                    const int s = n % S::kStages;
                    ok = mbar_wait<kTest>(q_free(s), (((uint32_t)n / S::kStages) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    mbar_expect_tx(q_full(s), S::kTileBytes);
                    for (int hh = 0; hh < HD / 64; ++hh)
                        tma_load_2d<kTest>(base + S::kOffQ + s * S::kTileBytes + hh * (128 * 128), &map_q, (h * a.group + i / sp.per_head) * HD + 64 * hh,
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
                ok = mbar_wait<kTest>(k_full, (uint32_t)turn++ & 1u, abort_flag);
                for (int i = 0; i < sp.per_head * a.group && ok; ++i, ++n) {
                    const int s = n % S::kStages, buf = n & 1;
                    ok = mbar_wait<kTest>(q_full(s), ((uint32_t)n / S::kStages) & 1u, abort_flag) &&
                         mbar_wait<kTest>(s_free(buf), (((uint32_t)n >> 1) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                    const uint32_t qbase = base + S::kOffQ + s * S::kTileBytes;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
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
        float* y = reinterpret_cast<float*>(smem + S::kOffY);
        const int r = threadIdx.x;                               // row of the tile; also a column of the next tile's statistics
        bool ok = true;
        for (int kt = blockIdx.x; kt * 128 < start + q_len && ok; kt += gridDim.x) {
            const Span sp = span_of(kt);
            const int tiles = sp.per_head * a.group;
            if (tiles == 0) continue;
            const int row = kt * 128 + r;
            const bool there = row < start + q_len;
            // ---- the tile's keys (all products of the turn before are complete: this warp has seen the last one's barrier)
#pragma unroll
            for (int m = 0; m < HD / 16; ++m) {
                const int id = r + 128 * m, key = id / (HD / 16), piece = id % (HD / 16);
                const int j = kt * 2 + key / 64;
                uint4 u = make_uint4(0, 0, 0, 0);
                if (j * kPageTokens < start + q_len)
                    u = *reinterpret_cast<const uint4*>(kv.k + (size_t)table[j] * kv.k_stride + ((size_t)h * kPageTokens + key % 64) * HD + piece * 16);
                uint32_t o[8];
                bf16_of_codes(u.x, o[0], o[1]);
                bf16_of_codes(u.y, o[2], o[3]);
                bf16_of_codes(u.z, o[4], o[5]);
                bf16_of_codes(u.w, o[6], o[7]);
                const uint32_t at = base + (piece / 4) * (128 * 128) + key * 128;
                store_shared16(at + (((piece % 4 * 2) ^ (key & 7)) << 4), o[0], o[1], o[2], o[3]);
                store_shared16(at + (((piece % 4 * 2 + 1) ^ (key & 7)) << 4), o[4], o[5], o[6], o[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full);
            const size_t page = there ? table[row / kPageTokens] : 0;
            const float f = there ? a.scale * kLog2e * kv.scales[page * kv.scale_stride + h] : 0.f;
            auto statistic = [&](int i) {                        // of tile i's column r: what takes a score to its probability's exponent
                const int token = sp.t_lo + i % sp.per_head * 128 + r;
                if (i >= tiles || token >= sp.t_hi) return 0.f;
                const float2 st = a.stats[(size_t)(q_begin + token) * a.n_heads + h * a.group + i / sp.per_head];
                return -(st.x + log2f(st.y));
            };
            float mine = statistic(0), total = 0.f;
            for (int i = 0; i < tiles; ++i, ++n) {
                const int buf = n & 1;
                y[128 * buf + r] = mine;
                __syncwarp();
                if (lane == 0) mbar_arrive(y_full(buf));
                mine = statistic(i + 1);
                ok = __all_sync(full, mbar_wait<kTest>(y_full(buf), ((uint32_t)n >> 1) & 1u, abort_flag) &&
                                          mbar_wait<kTest>(s_full(buf), ((uint32_t)n >> 1) & 1u, abort_flag));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
                const int t0 = sp.t_lo + i % sp.per_head * 128;
                // columns [lo, hi) of the tile are tokens that see this row
                const int lo = max(row - start - t0, 0);
                const long long past = min((long long)sp.t_hi, a.window > 0 ? (long long)row + a.window - start : (long long)sp.t_hi) - t0;
                const int hi = (int)min(past, 128LL);
                const bool whole = __all_sync(full, lo == 0 && hi == 128);
                const float* yt = y + 128 * buf;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    uint32_t sv[32];
                    tmem_ld32(tmem + 128 * buf + lane_off + c, sv);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 s4 = *reinterpret_cast<const float4*>(yt + c + e);
                        const float ys[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float p = fast_exp2(fmaf(__uint_as_float(sv[e + x]), f, ys[x]));
                            sum[x] += whole || (c + e + x >= lo && c + e + x < hi) ? p : 0.f;
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free(buf));
                total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (ok && there) kv.weights[page * kv.weight_stride + (size_t)h * kPageTokens + row % kPageTokens] += total;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::);
    __syncthreads();
    if (warp == 5) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols));
    }
}

template <int HD, bool kTest>
int launch_weights(const PromptArgs& a, const E4M3Pages& kv, const CUtensorMap& map_q, int B, int max_kv_len, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(e4m3_weights_kernel<HD, kTest>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightShape<HD>::kSmemBytes);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    return launch_chained(e4m3_weights_kernel<HD, kTest>, dim3((max_kv_len + 127) / 128, kv.n_kv, B), dim3(kWeightThreads),
                          (size_t)WeightShape<HD>::kSmemBytes, stream, map_q, a, kv);
}
}  // namespace

GTG_API int gtg_attention_e4m3_tcgen05_status() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

// Heads of 64 or 128 channels, bfloat16 rows of q and out on 16-byte boundaries.  weights (or null) gather what the rows get;
// stats: float2 [N][n_heads] of scratch for that.
GTG_API int gtg_attention_e4m3_tcgen05(const void* q, int ldq, void* out, int ldo, void* k, long long k_stride, void* v, long long v_stride,
                                       float* scales, long long scale_stride, float* weights, long long weight_stride, const int* block_table,
                                       int table_stride, const int* dropped, const int* cu_seqlens, const int* slots, const int* start_pos, int B,
                                       int max_q_len, int max_kv_len, int N, int n_heads, int n_kv, int hd, float scale, int window, float* stats,
                                       cudaStream_t stream) {
    if (B <= 0 || max_q_len <= 0 || N <= 0) return 0;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || window < 0 || max_kv_len <= 0 || (weights && !stats)) return kErrBadArgument;
    if (n_kv > 65535) return kErrUnsupported;
    if ((hd != 64 && hd != 128) || ldq % 8 || ldo % 8 || (uintptr_t)q % 16 || (uintptr_t)out % 16) return kErrUnsupported;
    if (B > 65535 || ((long long)max_q_len * (n_heads / n_kv) + BQ - 1) / BQ > 65535) return kErrUnsupported;
    const E4M3Pages kv = {(uint8_t*)k, (uint8_t*)v, k_stride, v_stride, scales, scale_stride, weights, weight_stride, block_table, table_stride, dropped, n_kv, hd};
    PromptArgs a = {};
    a.q = (const bf16*)q; a.ldq = ldq; a.out = (bf16*)out; a.ldo = ldo;
    a.cu_seqlens = cu_seqlens; a.slots = slots; a.start_pos = start_pos;
    a.n_heads = n_heads; a.group = n_heads / n_kv; a.scale = scale; a.window = window;
    a.stats = weights ? (float2*)stats : nullptr;
    const bool test = g_test_waits;
    const int st = hd == 64 ? (test ? launch<64, true>(a, kv, B, max_q_len, stream) : launch<64, false>(a, kv, B, max_q_len, stream))
                            : (test ? launch<128, true>(a, kv, B, max_q_len, stream) : launch<128, false>(a, kv, B, max_q_len, stream));
    if (st != 0 || !weights) return st;
    CUtensorMap map_q;
    const int mt = make_map(&map_q, q, N, n_heads * hd, ldq, 128);
    if (mt != 0) return mt;
    return hd == 64 ? (test ? launch_weights<64, true>(a, kv, map_q, B, max_kv_len, stream) : launch_weights<64, false>(a, kv, map_q, B, max_kv_len, stream))
                    : (test ? launch_weights<128, true>(a, kv, map_q, B, max_kv_len, stream) : launch_weights<128, false>(a, kv, map_q, B, max_kv_len, stream));
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
