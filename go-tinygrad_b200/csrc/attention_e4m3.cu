// Attention over the 8-bit key/value cache (layout and codes: e4m3.cuh).
//
// o = sum_j p_j v_j with p = softmax_j(scale q . k_j) over the rows j of the sequence up to the query's own (within a window,
// where there is one).  Where the cache gathers weights, row j's weight grows by the sum of p_j over the step's queries and
// the query heads of its key/value head.
//
//   few_queries:      bfloat16, heads of up to 128 channels in steps of 16, few queries a sequence (attention_e4m3_few.cuh);
//   attention_rows:   any head size and type, a block or several per (token, query head); scores, softmax and sums in float.
//   row_weights:      the weights, once every row's maximum and sum are known: a block per (cache page, head, sequence).
#include "attention_e4m3_few.cuh"

namespace {

// ============================================================== any head size, float or bfloat16
constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxChannels = 256;

// 32 rows at a time a warp: a lane scores one row and then adds up the channels lane, lane + 32, ... of all 32.  Few tokens over
// long sequences are cut into `splits` blocks each, whose parts (maximum, sum, outputs) rows_join_kernel joins in their order.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
attention_rows_kernel(const T* __restrict__ q, int ldq, T* __restrict__ out, int ldo, const E4M3Pages kv, const int* __restrict__ cu_seqlens,
                      const int* __restrict__ slots, const int* __restrict__ start_pos, int B, int n_heads, float scale, int window,
                      float2* __restrict__ stats, float* __restrict__ parts) {
    chain_release();
    chain_wait();
    __shared__ float qs[kMaxChannels];
    __shared__ float ps[kRowWarps][32];
    __shared__ float wm[kRowWarps], wl[kRowWarps];
    __shared__ float wo[kRowWarps][kMaxChannels];
    const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (token < cu_seqlens[0] || token >= cu_seqlens[B]) return;
    int b = 0;
    for (int lo = 0, hi = B; lo < hi;) {                                        // the last sequence that begins at or before the token
        const int mid = (lo + hi) >> 1;
        if (cu_seqlens[mid] <= token) { b = mid; lo = mid + 1; } else hi = mid;
    }
    const int slot = slots[b], hd = kv.hd, h = head / (n_heads / kv.n_kv);
    const int* table = kv.block_table + (size_t)slot * kv.table_stride;
    const int row = start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0) + token - cu_seqlens[b];
    const int first = window > 0 ? max(0, row - window + 1) : 0;
    for (int d = tid; d < hd; d += kRowThreads) qs[d] = to_f32(q[(size_t)token * ldq + head * hd + d]) * kDown * scale;
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    float o[kMaxChannels / 32];
#pragma unroll
    for (int i = 0; i < kMaxChannels / 32; ++i) o[i] = 0.f;
    for (int c = first / 32 + blockIdx.z * kRowWarps + warp; c * 32 <= row; c += kRowWarps * gridDim.z) {
        const size_t page = table[c / (kPageTokens / 32)];
        const int t0 = c % (kPageTokens / 32) * 32, t = t0 + lane, j = c * 32 + lane;
        const float k_scale = kv.scales[page * kv.scale_stride + h], v_scale = kv.scales[page * kv.scale_stride + kv.n_kv + h];
        const uint8_t* kr = kv.k + page * kv.k_stride + ((size_t)h * kPageTokens + t) * hd;
        const bool seen = j >= first && j <= row;
        float s = 0.f;
        if (seen) {
            if (hd % 16 == 0) {
                for (int d = 0; d < hd; d += 16) {
                    const uint4 u = *reinterpret_cast<const uint4*>(kr + d);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t pair = e4m3_pair_f16(w[e >> 1] >> (16 * (e & 1)));
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
                        s = fmaf(qs[d + 2 * e], f.x, s);
                        s = fmaf(qs[d + 2 * e + 1], f.y, s);
                    }
                }
            } else {
                for (int d = 0; d < hd; ++d) s = fmaf(qs[d], e4m3_value(kr[d]), s);
            }
        }
        s = seen ? s * k_scale * kUp : -INFINITY;
        const float m_new = fmaxf(m, warp_max(s));
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float p = seen ? expf(s - m_use) : 0.f, corr = expf(m - m_use);
        m = m_new;
        l = l * corr + p;
        __syncwarp();
        ps[warp][lane] = p * v_scale;
        __syncwarp();
        // rows that no query of this token sees may hold anything (a row nobody has written yet: the NaN code)
        const int from = max(first - c * 32, 0), to = min(row - c * 32, 31);
        const uint8_t* vr = kv.v + page * kv.v_stride + (size_t)h * hd * kPageTokens + t0;
#pragma unroll
        for (int i = 0; i < kMaxChannels / 32; ++i) {
            const int d = lane + 32 * i;
            if (d >= hd) break;
            const uint4 u[2] = {*reinterpret_cast<const uint4*>(vr + d * kPageTokens), *reinterpret_cast<const uint4*>(vr + d * kPageTokens + 16)};
            const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
            float acc = o[i] * corr;
            if (from == 0 && to == 31) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t pair = e4m3_pair_f16(w[e >> 1] >> (16 * (e & 1)));
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
                    acc = fmaf(ps[warp][2 * e], f.x, acc);
                    acc = fmaf(ps[warp][2 * e + 1], f.y, acc);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (e >= from && e <= to) acc = fmaf(ps[warp][e], e4m3_value((uint8_t)(w[e >> 2] >> (8 * (e & 3)))), acc);
            }
            o[i] = acc;
        }
    }
    l = warp_sum(l);
    if (lane == 0) { wm[warp] = m; wl[warp] = l; }
#pragma unroll
    for (int i = 0; i < kMaxChannels / 32; ++i)
        if (lane + 32 * i < hd) wo[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float M = wm[0];
    for (int w = 1; w < kRowWarps; ++w) M = fmaxf(M, wm[w]);
    const float M_use = M == -INFINITY ? 0.f : M;
    float f[kRowWarps], L = 0.f;
    for (int w = 0; w < kRowWarps; ++w) { f[w] = expf(wm[w] - M_use); L += f[w] * wl[w]; }
    float* part = gridDim.z > 1 ? parts + (((size_t)token * n_heads + head) * gridDim.z + blockIdx.z) * (hd + 2) : nullptr;
    if (part && tid == 0) { part[0] = M; part[1] = L; }
    for (int d = tid; d < hd; d += kRowThreads) {
        float acc = 0.f;
        for (int w = 0; w < kRowWarps; ++w) acc += f[w] * wo[w][d];
        if (part) part[2 + d] = acc;
        else out[(size_t)token * ldo + head * hd + d] = from_f32<T>(acc / L);
    }
    if (stats && !part && tid == 0) stats[(size_t)token * n_heads + head] = make_float2(M_use, L);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
rows_join_kernel(const float* __restrict__ parts, int splits, T* __restrict__ out, int ldo, const int* __restrict__ cu_seqlens, int B, int n_heads,
                 int hd, float2* __restrict__ stats) {
    chain_release();
    chain_wait();
    const int token = blockIdx.x, head = blockIdx.y;
    if (token < cu_seqlens[0] || token >= cu_seqlens[B]) return;
    const float* part = parts + ((size_t)token * n_heads + head) * splits * (hd + 2);
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, part[(size_t)s * (hd + 2)]);
    const float M_use = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < splits; ++s) L += expf(part[(size_t)s * (hd + 2)] - M_use) * part[(size_t)s * (hd + 2) + 1];
    for (int d = threadIdx.x; d < hd; d += kRowThreads) {
        float acc = 0.f;
        for (int s = 0; s < splits; ++s) acc += expf(part[(size_t)s * (hd + 2)] - M_use) * part[(size_t)s * (hd + 2) + 2 + d];
        out[(size_t)token * ldo + head * hd + d] = from_f32<T>(acc / L);
    }
    if (stats && threadIdx.x == 0) stats[(size_t)token * n_heads + head] = make_float2(M_use, L);
}

// A block per (page of the sequence, key/value head, sequence): 64 rows by two halves of the (query, head) pairs that may
// see them; the halves are added in order, so the sum does not depend on what else runs.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
row_weights_kernel(const T* __restrict__ q, int ldq, const E4M3Pages kv, const int* __restrict__ cu_seqlens, const int* __restrict__ slots,
                   const int* __restrict__ start_pos, int n_heads, float scale, int window, const float2* __restrict__ stats) {
    chain_release();
    chain_wait();
    constexpr int kAtOnce = 8;
    extern __shared__ float row_smem[];
    const int hd = kv.hd, ld = hd + 1;
    float* ks = row_smem;                                                           // [64][hd + 1]
    float* qs = ks + kPageTokens * ld;                                          // [kAtOnce][hd]
    __shared__ float2 st[kAtOnce];
    __shared__ float half_sum[kPageTokens];
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int first = cu_seqlens[b], n_new = cu_seqlens[b + 1] - first, slot = slots[b];
    if (n_new <= 0) return;
    const int start = start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    const int group = n_heads / kv.n_kv, t = tid & 63, part = tid >> 6;
    for (int block = blockIdx.x; block * kPageTokens < start + n_new; block += gridDim.x) {
        const size_t page = kv.block_table[(size_t)slot * kv.table_stride + block];
        const uint8_t* kr = kv.k + page * kv.k_stride + (size_t)h * kPageTokens * hd;
        __syncthreads();
        for (int i = tid; i < kPageTokens * hd; i += kRowThreads) ks[i / hd * ld + i % hd] = e4m3_value(kr[i]);
        const float k_scale = kv.scales[page * kv.scale_stride + h];
        const int row = block * kPageTokens + t;
        const int from = max(0, block * kPageTokens - start);                   // queries before that one see none of these rows
        const int pairs = (n_new - from) * group;
        float sum = 0.f;
        for (int p0 = 0; p0 < pairs; p0 += kAtOnce) {
            __syncthreads();
            const int here = min(kAtOnce, pairs - p0);
            for (int i = tid; i < here * hd; i += kRowThreads) {
                const int pair = p0 + i / hd;
                qs[i] = to_f32(q[(size_t)(first + from + pair / group) * ldq + (h * group + pair % group) * hd + i % hd]) * kDown * scale;
            }
            if (tid < here) st[tid] = stats[(size_t)(first + from + (p0 + tid) / group) * n_heads + h * group + (p0 + tid) % group];
            __syncthreads();
            for (int i = part; i < here; i += 2) {
                const int at = start + from + (p0 + i) / group;
                if (row > at || (window > 0 && row <= at - window)) continue;
                float s = 0.f;                                                  // the very score that the attention took its maximum of
                for (int d = 0; d < hd; ++d) s = fmaf(qs[i * hd + d], ks[t * ld + d], s);
                sum += expf(s * k_scale * kUp - st[i].x) / st[i].y;
            }
        }
        if (part) half_sum[t] = sum;
        __syncthreads();
        if (!part && row < start + n_new) {
            float* w = kv.weights + page * kv.weight_stride + h * kPageTokens + t;
            *w += sum + half_sum[t];
        }
    }
}

template <typename T>
int launch_row_weights(const void* q, int ldq, const E4M3Pages& kv, const int* cu_seqlens, const int* slots, const int* start_pos, int B,
                       int max_kv_len, int n_heads, float scale, int window, const float2* stats, cudaStream_t stream) {
    auto bytes = [](int hd) { return ((size_t)kPageTokens * (hd + 1) + 8 * (size_t)hd) * sizeof(float); };
    const size_t smem = bytes(kv.hd);
    static bool allowed[kMaxDevices] = {};
    const int set = allow_shared((const void*)row_weights_kernel<T>, bytes(kMaxChannels), allowed);
    if (set != 0) return set;
    return launch_behind(row_weights_kernel<T>, dim3((max_kv_len + kPageTokens - 1) / kPageTokens, kv.n_kv, B), dim3(kRowThreads), smem, stream,
                          (const T*)q, ldq, kv, cu_seqlens, slots, start_pos, n_heads, scale, window, stats);
}

// Blocks a (token, query head) has: as many as make four a multiprocessor, of 512 rows and more (float, 8 heads of 64 over 16,000 rows:
// 19.5 us where one block each takes 190; over 1,100: 13.9 and 17.6).
int rows_splits(int N, int n_heads, int max_kv_len, int window) {
    const long long seen = window > 0 ? std::min(window, max_kv_len) : max_kv_len;
    return (int)std::max(1LL, std::min(4LL * 148 / ((long long)N * n_heads), seen / 512));
}
long long rows_floats(int N, int n_heads, int hd, int splits, bool weigh) {
    return (weigh ? 2LL * N * n_heads : 0) + (splits > 1 ? (long long)N * n_heads * splits * (hd + 2) : 0);
}

template <typename T>
int launch_rows(const void* q, int ldq, void* out, int ldo, const E4M3Pages& kv, const int* cu_seqlens, const int* slots, const int* start_pos,
                int B, int max_kv_len, int N, int n_heads, float scale, int window, float* scratch, cudaStream_t stream) {
    float2* stats = kv.weights ? (float2*)scratch : nullptr;
    const int splits = rows_splits(N, n_heads, max_kv_len, window);
    float* parts = splits > 1 ? scratch + (kv.weights ? 2LL * N * n_heads : 0) : nullptr;
    int st = launch_chained(attention_rows_kernel<T>, dim3(N, n_heads, splits), dim3(kRowThreads), 0, stream, (const T*)q, ldq, (T*)out, ldo, kv,
                            cu_seqlens, slots, start_pos, B, n_heads, scale, window, stats, parts);
    if (st == 0 && splits > 1)
        st = launch_behind(rows_join_kernel<T>, dim3(N, n_heads), dim3(kRowThreads), 0, stream, (const float*)parts, splits, (T*)out, ldo, cu_seqlens, B,
                           n_heads, kv.hd, stats);
    if (st != 0 || !kv.weights) return st;
    return launch_row_weights<T>(q, ldq, kv, cu_seqlens, slots, start_pos, B, max_kv_len, n_heads, scale, window, stats, stream);
}
}  // namespace

static FewPlan few_plan(int B, int max_q_len, int n_heads, int n_kv, int hd, int max_kv_len, int weigh) {
#define GTG_FEW(HD) case HD: return few_plan_for<HD>(B, max_q_len, n_heads, n_kv, max_kv_len, weigh);
    switch (hd) { GTG_FEW(16) GTG_FEW(32) GTG_FEW(48) GTG_FEW(64) GTG_FEW(80) GTG_FEW(96) GTG_FEW(112) default: GTG_FEW(128) }
#undef GTG_FEW
}

// Floats of scratch that gtg_attention_e4m3 needs for the same numbers.
GTG_API long long gtg_attention_e4m3_scratch_floats(int dtype, int B, int N, int max_q_len, int n_heads, int n_kv, int hd, int max_kv_len,
                                                    int window, int weigh) {
    if (B <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || max_q_len <= 0 || max_kv_len <= 0) return 0;
    const long long rows = rows_floats(N, n_heads, hd, rows_splits(std::max(N, 1), n_heads, max_kv_len, window), weigh != 0);
    if (few_takes(dtype, max_q_len, n_heads, n_kv, hd))
        return std::max(few_plan(B, max_q_len, n_heads, n_kv, hd, max_kv_len, weigh).floats(), rows);
    return rows;
}

// dtype: of q and out (0 float, 1 bfloat16).  max_kv_len: rows of the longest sequence after this step; it decides how the work is cut
// and how many blocks look for weights.
GTG_API int gtg_attention_e4m3(int dtype, const void* q, int ldq, void* out, int ldo, const E4M3Pages* pages, const int* cu_seqlens,
                               const int* slots, const int* start_pos, int B, int max_q_len, int max_kv_len, int N, int n_heads,
                               float scale, int window, float* scratch, cudaStream_t stream) {
    if (B <= 0 || N <= 0 || max_q_len <= 0) return 0;
    const E4M3Pages kv = *pages;
    const int n_kv = kv.n_kv, hd = kv.hd;
    float* weights = kv.weights;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || hd <= 0 || max_kv_len <= 0 || window < 0) return kErrBadArgument;
    if (hd > kMaxChannels || B > 65535 || n_heads > 65535) return kErrUnsupported;
    if (few_takes(dtype, max_q_len, n_heads, n_kv, hd) && few_counts(B, max_q_len, n_heads, n_kv, kv.table_stride)) {
        const FewPlan plan = few_plan(B, max_q_len, n_heads, n_kv, hd, max_kv_len, weights != nullptr);
        if (plan.floats() && !scratch) return kErrBadArgument;
        FewArgs a = {};
        a.q = (const bf16*)q; a.ldq = ldq; a.wide = (uintptr_t)q % 16 == 0 && ldq % 8 == 0; a.chained = g_chained_launch; a.out = (bf16*)out; a.ldo = ldo;
        a.cu_seqlens = cu_seqlens; a.slots = slots; a.start_pos = start_pos;
        a.B = B; a.n_heads = n_heads; a.group = n_heads / n_kv; a.scale = scale; a.window = window;
#define GTG_FEW(HD) case HD: return launch_few<HD>(a, kv, plan, scratch, stream);
        switch (hd) { GTG_FEW(16) GTG_FEW(32) GTG_FEW(48) GTG_FEW(64) GTG_FEW(80) GTG_FEW(96) GTG_FEW(112) GTG_FEW(128) }
#undef GTG_FEW
    }
    if (rows_floats(N, n_heads, hd, rows_splits(N, n_heads, max_kv_len, window), weights != nullptr) && !scratch) return kErrBadArgument;
    if (dtype == 0) return launch_rows<float>(q, ldq, out, ldo, kv, cu_seqlens, slots, start_pos, B, max_kv_len, N, n_heads, scale, window, scratch, stream);
    return launch_rows<bf16>(q, ldq, out, ldo, kv, cu_seqlens, slots, start_pos, B, max_kv_len, N, n_heads, scale, window, scratch, stream);
}
