// Writing and compacting the 8-bit key/value cache (layout and codes: e4m3.cuh).
//
//   kv_store:  rotates a step's queries and keys and stores its keys and values, block by block;
//   kv_evict:  keeps a sequence's newest rows and the heaviest of the others, in place.
#include "e4m3.cuh"

namespace {

// ============================================================== storing a step's keys and values
constexpr int kStoreThreads = 128;

// One token's row of the projection: query heads, key heads, value heads of hd channels each.
template <typename T>
struct StoreInput {
    const T* qkv;
    int ld;
    const float2* cos_sin;     // [N][rot/2], or null: nothing is rotated
    int n_heads, n_kv, hd, rot, interleaved;
    int v_offset;              // columns from a token's first key head to the head its value is read from
};

// Channel d of a head at `row`, rotated: pairs (i, i + rot/2) or (2i, 2i + 1) of the first `rot` channels,
// (a, b) -> (a cos - b sin, a sin + b cos), every product and sum rounded to float.
template <typename T>
__device__ __forceinline__ float rotated(const T* __restrict__ row, const float2* __restrict__ cs, int d, int rot, int interleaved) {
    const float x = to_f32(row[d]);
    if (cs == nullptr || d >= rot) return x;
    const int half = rot >> 1;
    const int i = interleaved ? d >> 1 : (d < half ? d : d - half);
    const bool first = interleaved ? !(d & 1) : d < half;
    const float y = to_f32(row[interleaved ? d ^ 1 : (first ? d + half : d - half)]);
    const float2 c = cs[i];
    return first ? __fsub_rn(__fmul_rn(x, c.x), __fmul_rn(y, c.y)) : __fadd_rn(__fmul_rn(y, c.y), __fmul_rn(x, c.x));
}

// Blocks [0, blocks_kv): (sequence, key/value head, plane, touched cache block); the rest rotate query rows.
template <typename T>
__global__ void __launch_bounds__(kStoreThreads)
kv_store_kernel(const StoreInput<T> in, const E4M3Pages kv, const int* __restrict__ cu_seqlens, const int* __restrict__ slots,
                const int* __restrict__ start_pos, int blocks_per_seq, long long blocks_kv, int N, T* __restrict__ q_out, int ldq) {
    chain_wait();
    chain_release();                  // only now: what comes next may read older pages at once (all before this kernel is complete)
    __shared__ float scratch[33];
    const int tid = threadIdx.x;
    if ((long long)blockIdx.x >= blocks_kv) {
        const int token = (int)((long long)blockIdx.x - blocks_kv);
        const T* row = in.qkv + (size_t)token * in.ld;
        const float2* cs = in.cos_sin ? in.cos_sin + (size_t)token * (in.rot >> 1) : nullptr;
        for (int i = tid; i < in.n_heads * in.hd; i += kStoreThreads) {
            const int h = i / in.hd, d = i - h * in.hd;
            q_out[(size_t)token * ldq + i] = from_f32<T>(rotated(row + h * in.hd, cs, d, in.rot, in.interleaved));
        }
        return;
    }
    int id = blockIdx.x;
    const int j = id % blocks_per_seq; id /= blocks_per_seq;
    const int plane = id & 1; id >>= 1;
    const int h = id % kv.n_kv, b = id / kv.n_kv;
    const int first = cu_seqlens[b], n_new = cu_seqlens[b + 1] - first;
    if (n_new <= 0) return;
    const int slot = slots[b];
    const int start = start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);     // row of the step's first token
    const int block = start / kPageTokens + j;
    const int lo = max(start - block * kPageTokens, 0);                        // the block's rows [lo, hi) are new
    const int hi = min(start + n_new - block * kPageTokens, kPageTokens);
    if (hi <= lo) return;
    const size_t page = kv.block_table[(size_t)slot * kv.table_stride + block];
    const int rows = hi - lo, hd = kv.hd;
    const int token0 = first + block * kPageTokens + lo - start;
    const int column = (in.n_heads + h) * hd + (plane ? in.v_offset : 0);
    auto value = [&](int r, int d) {                                            // of new row r, channel d
        const size_t token = token0 + r;
        const T* row = in.qkv + token * in.ld + column;
        if (plane) return to_f32(row[d]);
        return rotated(row, in.cos_sin ? in.cos_sin + token * (in.rot >> 1) : nullptr, d, in.rot, in.interleaved);
    };
    float most = 0.f;
    for (int i = tid; i < rows * hd; i += kStoreThreads) {
        const float x = fabsf(value(i / hd, i % hd));
        if (finite_f32(x)) most = fmaxf(most, x);
    }
    most = warp_max(most);
    if ((tid & 31) == 0) scratch[tid >> 5] = most;
    __syncthreads();
    most = fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
    float* scale_at = kv.scales + page * kv.scale_stride + plane * kv.n_kv + h;
    float scale = e4m3_needed_scale(most);
    uint8_t* codes = plane ? kv.v + page * kv.v_stride + (size_t)h * kPageTokens * hd : kv.k + page * kv.k_stride + (size_t)h * kPageTokens * hd;
    auto at = [&](int r, int d) -> uint8_t& { return plane ? codes[d * kPageTokens + r] : codes[r * hd + d]; };
    if (lo > 0) {
        const float before = *scale_at;
        if (before >= scale) {
            scale = before;
        } else {
            const float ratio = before * pow2_inverse(scale);
            for (int i = tid; i < lo * hd; i += kStoreThreads) {
                uint8_t& c = plane ? codes[(i / lo) * kPageTokens + i % lo] : codes[i];
                c = e4m3_code(e4m3_value(c) * ratio);
            }
        }
    }
    const float inverse = pow2_inverse(scale);
    for (int i = tid; i < rows * hd; i += kStoreThreads) at(lo + i / hd, i % hd) = e4m3_code(value(i / hd, i % hd) * inverse);
    __syncthreads();                                                            // every thread has read the old scale
    if (tid == 0) *scale_at = scale;
    if (plane == 0 && kv.weights)
        for (int r = tid; r < rows; r += kStoreThreads) kv.weights[page * kv.weight_stride + h * kPageTokens + lo + r] = 0.f;
}

// ============================================================== eviction
constexpr int kEvictThreads = 256;

// A float's bits in an order that unsigned comparison keeps (the larger float the larger number, NaN above all).
__device__ __forceinline__ uint32_t ordered_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);                                // -0 becomes 0
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix sum over the block of small counts; *total: their sum.
__device__ __forceinline__ int block_prefix(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kEvictThreads / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return before + incl - v;
}

// A block per (key/value head, sequence, entry).  Entries are entry_stride_* apart.
struct EvictStrides { long long k, v, scales, weights; };

__global__ void __launch_bounds__(kEvictThreads)
kv_evict_kernel(const E4M3Pages pages, const EvictStrides strides, int* __restrict__ dropped, const int* __restrict__ slots,
                const int* __restrict__ lengths, int budget, int recent, int* __restrict__ kept_out) {
    extern __shared__ uint8_t tile[];                                           // 64 rows x hd codes
    __shared__ int histogram[256];
    __shared__ int warp_sums[kEvictThreads / 32];
    __shared__ float warp_most[kEvictThreads / 32];
    __shared__ int choice[2];
    const int h = blockIdx.x, b = blockIdx.y, entry = blockIdx.z, tid = threadIdx.x;
    const int length = lengths[b], slot = slots[b], hd = pages.hd;
    int* kept = kept_out + (((size_t)entry * gridDim.y + b) * pages.n_kv + h) * budget;
    if (length <= budget) {
        for (int i = tid; i < budget; i += kEvictThreads) kept[i] = i < length ? i : -1;
        return;
    }
    if (h == 0 && entry == 0 && tid == 0 && dropped) dropped[slot] += length - budget;
    const int* table = pages.block_table + (size_t)slot * pages.table_stride;
    uint8_t* kc = pages.k + entry * strides.k + (size_t)h * kPageTokens * hd;
    uint8_t* vc = pages.v + entry * strides.v + (size_t)h * kPageTokens * hd;
    float* scales = pages.scales + entry * strides.scales + h;
    float* weights = pages.weights + entry * strides.weights + h * kPageTokens;
    auto weight_of = [&](int i) { return ordered_bits(weights[(size_t)table[i / kPageTokens] * pages.weight_stride + i % kPageTokens]); };
    const int n = length - recent, need = budget - recent;

    // ---- the need-th largest of the first n weights, eight bits a pass from the top
    uint32_t threshold = 0;
    int left = need;                                                            // still to be found among those that share the prefix
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            histogram[tid] = 0;
            __syncthreads();
            const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int i = tid; i < n; i += kEvictThreads) {
                const uint32_t u = weight_of(i);
                if ((u & above) == (threshold & above)) atomicAdd(&histogram[(u >> shift) & 255u], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int digit = 255, more = 0;
                while (digit > 0 && more + histogram[digit] < left) more += histogram[digit--];
                choice[0] = digit;
                choice[1] = more;
            }
            __syncthreads();
            threshold |= (uint32_t)choice[0] << shift;
            left -= choice[1];
            __syncthreads();
        }
    }
    // ---- the rows that stay, in order: all above the threshold, the first `left` of those equal to it, the newest
    int equal_before = 0, kept_before = 0;
    for (int i0 = 0; i0 < n && need > 0; i0 += kEvictThreads) {
        const int i = i0 + tid;
        const uint32_t u = i < n ? weight_of(i) : 0u;
        const bool equal = i < n && u == threshold;
        int total;
        const int rank = equal_before + block_prefix(equal ? 1 : 0, warp_sums, &total);
        equal_before += total;
        const bool stays = i < n && (u > threshold || (equal && rank < left));
        const int place = kept_before + block_prefix(stays ? 1 : 0, warp_sums, &total);
        kept_before += total;
        if (stays) kept[place] = i;
    }
    for (int i = tid; i < recent; i += kEvictThreads) kept[need + i] = n + i;
    __threadfence_block();
    __syncthreads();

    // ---- block by block to the front.  Row r of the result comes from a row at or behind r, so what a block overwrites
    //      no later block reads, neither its codes nor its scale.
    for (int to = 0; to * kPageTokens < budget; ++to) {
        const int rows = min(kPageTokens, budget - to * kPageTokens);
        const int* source = kept + to * kPageTokens;
        const bool moves = tid < rows && source[tid] != to * kPageTokens + tid;
        if (!__syncthreads_or(moves)) continue;
        const size_t page = table[to];
        float gathered = 0.f;
        if (tid < rows) gathered = weights[(size_t)table[source[tid] / kPageTokens] * pages.weight_stride + source[tid] % kPageTokens];
        for (int plane = 0; plane < 2; ++plane) {
            float most = 0.f;
            for (int i = tid; i < rows * hd; i += kEvictThreads) {
                const int r = plane ? i % rows : i / hd, d = plane ? i / rows : i % hd;
                const size_t p = table[source[r] / kPageTokens];
                const int t = source[r] % kPageTokens;
                const uint8_t c = plane ? vc[p * pages.v_stride + d * kPageTokens + t] : kc[p * pages.k_stride + t * hd + d];
                tile[r * hd + d] = c;
                const float x = fabsf(e4m3_value(c) * scales[p * pages.scale_stride + plane * pages.n_kv]);
                if (finite_f32(x)) most = fmaxf(most, x);
            }
            most = warp_max(most);
            if ((tid & 31) == 0) warp_most[tid >> 5] = most;
            __syncthreads();
            most = warp_most[0];
            for (int w = 1; w < kEvictThreads / 32; ++w) most = fmaxf(most, warp_most[w]);
            const float scale = e4m3_needed_scale(most), inverse = pow2_inverse(scale);
            for (int i = tid; i < rows * hd; i += kEvictThreads) {
                const int r = plane ? i % rows : i / hd, d = plane ? i / rows : i % hd;
                const float was = scales[(size_t)table[source[r] / kPageTokens] * pages.scale_stride + plane * pages.n_kv];
                const uint8_t c = e4m3_code(e4m3_value(tile[r * hd + d]) * was * inverse);
                if (plane) vc[page * pages.v_stride + d * kPageTokens + r] = c;
                else kc[page * pages.k_stride + r * hd + d] = c;
            }
            __syncthreads();
            if (tid == 0) scales[page * pages.scale_stride + plane * pages.n_kv] = scale;
        }
        if (tid < rows) weights[page * pages.weight_stride + tid] = gathered;
        __syncthreads();
    }
}

template <typename T>
int launch_store(const StoreInput<T>& in, const E4M3Pages& kv, const int* cu_seqlens, const int* slots, const int* start_pos,
                 int B, int max_q_len, int N, int store, void* q_out, int ldq, cudaStream_t stream) {
    const int per_seq = (max_q_len + kPageTokens - 2) / kPageTokens + 1;
    const long long blocks_kv = store ? (long long)B * kv.n_kv * 2 * per_seq : 0;
    const long long blocks = blocks_kv + (q_out ? N : 0);
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL) return kErrUnsupported;
    return launch_chained(kv_store_kernel<T>, dim3((unsigned)blocks), dim3(kStoreThreads), 0, stream, in, kv, cu_seqlens, slots, start_pos,
                          per_seq, blocks_kv, N, (T*)q_out, ldq);
}
}  // namespace

// qkv: [N][ld] of the compute type (dtype 0 float, 1 bfloat16): n_heads query heads, n_kv key heads and, unless values_from_keys,
// n_kv value heads.  cos_sin: float [N][rot/2][2] or null.  store 0: queries only (another run's cache is read).
GTG_API int gtg_kv_store_e4m3(int dtype, const void* qkv, int ld, const float* cos_sin, int n_heads, int n_kv, int hd, int rot, int interleaved,
                              int values_from_keys, int store, void* k, long long k_stride, void* v, long long v_stride, float* scales,
                              long long scale_stride, float* weights, long long weight_stride, const int* block_table, int table_stride,
                              const int* dropped, const int* cu_seqlens, const int* slots, const int* start_pos, int B, int max_q_len, int N,
                              void* q_out, int ldq, cudaStream_t stream) {
    if (B <= 0 || N <= 0 || max_q_len <= 0) return 0;
    if (n_heads < 0 || n_kv < 0 || hd <= 0 || rot < 0 || rot % 2 || rot > hd) return kErrBadArgument;
    const E4M3Pages kv = {(uint8_t*)k, (uint8_t*)v, k_stride, v_stride, scales, scale_stride, weights, weight_stride, block_table, table_stride,
                          dropped, n_kv, hd};
    const int v_offset = values_from_keys ? 0 : n_kv * hd;
    if (dtype == 0) {
        const StoreInput<float> in = {(const float*)qkv, ld, (const float2*)cos_sin, n_heads, n_kv, hd, rot, interleaved, v_offset};
        return launch_store(in, kv, cu_seqlens, slots, start_pos, B, max_q_len, N, store, q_out, ldq, stream);
    }
    const StoreInput<bf16> in = {(const bf16*)qkv, ld, (const float2*)cos_sin, n_heads, n_kv, hd, rot, interleaved, v_offset};
    return launch_store(in, kv, cu_seqlens, slots, start_pos, B, max_q_len, N, store, q_out, ldq, stream);
}

// lengths[b]: rows that the sequence in slots[b] holds.  kept: [entries][B][n_kv][budget].
GTG_API int gtg_kv_evict_e4m3(int entries, void* k, long long k_entry, long long k_stride, void* v, long long v_entry, long long v_stride,
                              float* scales, long long scale_entry, long long scale_stride, float* weights, long long weight_entry,
                              long long weight_stride, const int* block_table, int table_stride, int* dropped, int n_kv, int hd, const int* slots,
                              const int* lengths, int B, int budget, int recent, int* kept, cudaStream_t stream) {
    if (B <= 0 || entries <= 0) return 0;
    if (budget <= 0 || recent < 0 || recent > budget || n_kv <= 0 || hd <= 0 || !weights || !kept) return kErrBadArgument;
    if (B > 65535 || entries > 65535) return kErrUnsupported;
    const size_t smem = (size_t)kPageTokens * hd;
    if (smem > 40 * 1024) return kErrUnsupported;
    const E4M3Pages pages = {(uint8_t*)k, (uint8_t*)v, k_stride, v_stride, scales, scale_stride, weights, weight_stride, block_table, table_stride,
                             nullptr, n_kv, hd};
    const EvictStrides strides = {k_entry, v_entry, scale_entry, weight_entry};
    kv_evict_kernel<<<dim3(n_kv, B, entries), kEvictThreads, smem, stream>>>(pages, strides, dropped, slots, lengths, budget, recent, kept);
    return launch_status();
}
