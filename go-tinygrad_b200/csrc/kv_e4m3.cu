// Writing and compacting the 8-bit key/value cache (layout and codes: e4m3.cuh).
//
//   kv_store:  rotates a step's queries and keys and stores its keys and values, block by block;
//   kv_evict:  keeps a sequence's newest rows and the heaviest of the others, in place.
#include "mma_helpers.cuh"
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
                const int* __restrict__ lengths, int max_length, int budget, int recent, int* __restrict__ kept_out) {
    extern __shared__ uint8_t tile[];                                           // 64 rows x hd codes
    __shared__ int histogram[256];
    __shared__ int warp_sums[kEvictThreads / 32];
    __shared__ float warp_most[kEvictThreads / 32];
    __shared__ int choice[2];
    const int h = blockIdx.x, b = blockIdx.y, entry = blockIdx.z, tid = threadIdx.x;
    const int length = lengths[b], slot = slots[b], hd = pages.hd;
    int* kept = kept_out + (((size_t)entry * gridDim.y + b) * pages.n_kv + h) * budget;
    if (length <= budget || length > max_length) {
        for (int i = tid; i < budget; i += kEvictThreads) kept[i] = i < length && length <= budget ? i : -1;
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

// ---- the same for heads of a multiple of 16 channels, with the sequence's weights, pages and scales in shared memory.
// Choosing: the weights are read once; the need-th largest is found eight bits a pass (equal digits of a warp counted by one
// lane, the digit found by one warp), then every warp places a stretch of the rows by itself, after one exchange of counts.
// Moving: four warps move the keys and four the values, tile by tile of 64 rows from the first that changes, the next codes on
// their way while a tile is worked on (what a tile overwrites no later one reads).  The rows of the values are innermost, so
// a value tile is gathered out of whole pages in shared memory, each copied there once: a thread has the same four rows of
// the tile in several channels, and a word of four codes comes out of the four words that hold them by three byte permutations.
// What bounds it is instructions: 24 entries x 3 sequences of 2,000 rows x 32 heads of 64 take 256 us on a B200 with 71 % of the issue
// slots busy; the 680 MB that reach memory (blocks of which nothing moves are left alone) would take 106.  Eight warps, each with
// twice the channels that sixteen have, because much of a tile's work is the same for all its channels (an earlier form: 440 us with
// sixteen, 337 with eight; eight cost 2 us of 17 where there are fewer blocks than multiprocessors).
constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32, kPlaneThreads = kMoveThreads / 2;
constexpr int kStaged = 4;                 // value pages in shared memory: two that a tile is gathered from, two on their way
template <int HD> struct Move {
    static constexpr int MINE = (4 * HD + kPlaneThreads - 1) / kPlaneThreads;    // 16-byte pieces of a page a thread has
    static constexpr int V_PAGE = HD * kPageTokens;
    static constexpr int V_BYTES = kStaged * V_PAGE;
};

template <int PLANE> __device__ __forceinline__ void plane_sync() { asm volatile("bar.sync %0, %1;\n" ::"n"(1 + PLANE), "n"(kPlaneThreads) : "memory"); }

// Two codes times a power of two each, as halves.  Below 2^-24, half's least, every code becomes zero all the same.  Above 2^17 every
// code is zero: that factor takes the smallest, 2^-9, to 2^8, and 2^18 would take it beyond the 448 that the new scale was made
// for.  Half holds powers up to 2^15: where a factor is FAR above that, the rest is multiplied in a second time.  (Asked once a tile:
// asked at every word, the large eviction named below took 287 us instead of 251.)
constexpr float kLeastHalf = 5.9604645e-8f, kMostHalf = 32768.f;
template <bool FAR>
__device__ __forceinline__ __half2 times_ratio(uint32_t two_codes, float a, float b) {
    const uint32_t h = e4m3_pair_f16(two_codes);
    __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h),
                        __floats2half2_rn(fminf(fmaxf(a, kLeastHalf), kMostHalf), fminf(fmaxf(b, kLeastHalf), kMostHalf)));
    if constexpr (FAR)
        x = __hmul2(x, __floats2half2_rn(fminf(fmaxf(a * (1.f / kMostHalf), 1.f), 4.f), fminf(fmaxf(b * (1.f / kMostHalf), 1.f), 4.f)));
    return x;
}
__device__ __forceinline__ uint32_t pair_codes(__half2 x) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
    return r;
}
// Four codes times a power of two each.
template <bool FAR>
__device__ __forceinline__ uint32_t times_ratios(uint32_t w, float a, float b, float c, float d) {
    return pair_codes(times_ratio<FAR>(w, a, b)) | pair_codes(times_ratio<FAR>(w >> 16, c, d)) << 16;
}
// Each byte's |code| + 1, or 0 for NaN: the even bytes of a word and the odd ones, as 16-bit numbers that maxima are taken of.
__device__ __forceinline__ uint32_t even_sizes(uint32_t w) { return ((w & 0x007f007fu) + 0x00010001u) & 0x007f007fu; }
__device__ __forceinline__ uint32_t odd_sizes(uint32_t w) { return even_sizes(w >> 8); }
__device__ __forceinline__ float size_value(uint32_t size) { return e4m3_value((uint8_t)(max(size, 1u) - 1u)); }

template <int HD>
__global__ void __launch_bounds__(kMoveThreads, 1024 / kMoveThreads)
kv_evict_move_kernel(const E4M3Pages pages, const EvictStrides strides, int* __restrict__ dropped, const int* __restrict__ slots,
                     const int* __restrict__ lengths, int max_length, int budget, int recent, int* __restrict__ kept_out) {
    using M = Move<HD>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int histogram[256];
    __shared__ int greater[kMoveWarps], equal[kMoveWarps];
    __shared__ float warp_most[2 * kMoveWarps];
    __shared__ int choice[2], first_gone;
    const int h = blockIdx.x, b = blockIdx.y, entry = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int length = lengths[b], slot = slots[b];
    int* kept_at = kept_out + (((size_t)entry * gridDim.y + b) * pages.n_kv + h) * budget;
    if (length <= budget || length > max_length) {
        for (int i = tid; i < budget; i += kMoveThreads) kept_at[i] = i < length && length <= budget ? i : -1;
        return;
    }
    if (h == 0 && entry == 0 && tid == 0 && dropped) dropped[slot] += length - budget;
    const int max_pages = (max_length + kPageTokens - 1) / kPageTokens, n_pages = (length + kPageTokens - 1) / kPageTokens;
    unsigned char* staged = smem;                                               // value pages
    float* w = reinterpret_cast<float*>(smem + M::V_BYTES);                     // [max_pages * 64]
    int* kept = reinterpret_cast<int*>(w + max_pages * kPageTokens);            // [budget rounded up to 64]
    int* page_id = kept + (budget + 63) / 64 * 64;                              // [max_pages]
    float* page_scale = reinterpret_cast<float*>(page_id + max_pages);          // [2][max_pages]
    const int* table = pages.block_table + (size_t)slot * pages.table_stride;
    uint8_t* kc = pages.k + entry * strides.k + (size_t)h * kPageTokens * HD;
    uint8_t* vc = pages.v + entry * strides.v + (size_t)h * kPageTokens * HD;
    float* scales = pages.scales + entry * strides.scales + h;
    float* weights = pages.weights + entry * strides.weights + h * kPageTokens;
    for (int i = tid; i < n_pages * (kPageTokens / 4); i += kMoveThreads) {
        const int p = i / (kPageTokens / 4), page = table[p];
        reinterpret_cast<float4*>(w)[i] = reinterpret_cast<const float4*>(weights + (size_t)page * pages.weight_stride)[i % (kPageTokens / 4)];
        if (i % (kPageTokens / 4) == 0) page_id[p] = page;
        if (i % (kPageTokens / 4) < 2) page_scale[i % 2 * max_pages + p] = scales[(size_t)page * pages.scale_stride + i % 2 * pages.n_kv];
    }
    if (tid < 256) histogram[tid] = 0;
    if (tid == 0) first_gone = 0x7fffffff;
    __syncthreads();
    const int n = length - recent, need = budget - recent;

    // ---- the need-th largest of the first n weights
    uint32_t threshold = 0;
    int left = need;
    for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
        const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int i0 = warp * 32; i0 < n; i0 += kMoveThreads) {
            const uint32_t u = i0 + lane < n ? ordered_bits(w[i0 + lane]) : 0u;
            const bool counts = i0 + lane < n && (u & above) == (threshold & above);
            const int digit = counts ? (int)((u >> shift) & 255u) : 256;
            const unsigned like = __match_any_sync(0xffffffffu, digit);
            if (counts && lane == __ffs(like) - 1) atomicAdd(&histogram[digit], __popc(like));
        }
        __syncthreads();
        if (warp == 0) {                                                        // lane l: digits 255 - 8 l down to 248 - 8 l
            int mine[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += mine[e] = histogram[255 - 8 * lane - e];
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            const unsigned enough = __ballot_sync(0xffffffffu, incl >= left);
            if (lane == __ffs(enough) - 1) {
                int more = incl - sum, digit = 255 - 8 * lane;
                bool found = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    found = found || more + mine[e] >= left;
                    if (!found) { more += mine[e]; --digit; }
                }
                choice[0] = digit;
                choice[1] = more;
            }
        }
        __syncthreads();
        threshold |= (uint32_t)choice[0] << shift;
        left -= choice[1];
        if (tid < 256) histogram[tid] = 0;
        __syncthreads();
    }
    // ---- the rows that stay, in order
    {
        const int stretch = (n + kMoveThreads - 1) / kMoveThreads * 32;         // of a warp
        const int begin = min(n, warp * stretch), end = min(n, begin + stretch);
        int more = 0, same = 0;
        for (int i0 = begin; i0 < end; i0 += 32) {
            const uint32_t u = i0 + lane < end ? ordered_bits(w[i0 + lane]) : 0u;
            more += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && u > threshold));
            same += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && u == threshold));
        }
        if (lane == 0) { greater[warp] = more; equal[warp] = same; }
        __syncthreads();
        int place = 0, rank = 0;
        for (int x = 0; x < warp; ++x) { place += greater[x]; rank += equal[x]; }
        const int taken = need > 0 ? left : 0;                                  // of those equal to the threshold
        place += min(taken, rank);
        int gone = 0x7fffffff;
        for (int i0 = begin; i0 < end; i0 += 32) {
            const uint32_t u = i0 + lane < end ? ordered_bits(w[i0 + lane]) : 0u;
            const bool even = i0 + lane < end && u == threshold;
            const unsigned evens = __ballot_sync(0xffffffffu, even), below = (1u << lane) - 1u;
            const bool stays = need > 0 && i0 + lane < end && (u > threshold || (even && rank + __popc(evens & below) < taken));
            const unsigned all = __ballot_sync(0xffffffffu, stays);
            if (stays) kept[place + __popc(all & below)] = i0 + lane;
            if (gone == 0x7fffffff) {
                const unsigned lost = __ballot_sync(0xffffffffu, i0 + lane < end && !stays);
                if (lost) gone = i0 + __ffs(lost) - 1;
            }
            place += __popc(all);
            rank += __popc(evens);
        }
        if (lane == 0 && gone != 0x7fffffff) atomicMin(&first_gone, gone);
        for (int i = tid; i < recent; i += kMoveThreads) kept[need + i] = n + i;
    }
    __syncthreads();
    for (int i = tid; i < budget; i += kMoveThreads) kept_at[i] = kept[i];
    const int tiles = (budget + kPageTokens - 1) / kPageTokens;
    const int first_tile = first_gone < budget ? first_gone / kPageTokens : tiles;        // all rows before it stay where they are
    for (int r = first_tile * kPageTokens + tid; r < budget; r += kMoveThreads)
        weights[(size_t)page_id[r / kPageTokens] * pages.weight_stride + r % kPageTokens] = w[kept[r]];

    // ---- tiles to the front
    const int plane = tid / kPlaneThreads, t = tid % kPlaneThreads;
    const float* old_scale = page_scale + plane * max_pages;
    uint4 ahead[M::MINE];                                                       // of the next key tile
    auto rows_of = [&](int to) { return min(kPageTokens, budget - to * kPageTokens); };
    // the largest of a tile's values, in all threads of a plane; tiles take turns with two places
    auto block_most = [&](float most, int to, auto sync) {
        most = warp_max(most);
        float* at = warp_most + (to & 1) * kMoveWarps + plane * (kMoveWarps / 2);
        if (lane == 0) at[warp % (kMoveWarps / 2)] = most;
        sync();
        most = 0.f;
#pragma unroll
        for (int x = 0; x < kMoveWarps / 2; ++x) most = fmaxf(most, at[x]);
        return most;
    };
    if (plane == 0) {
        auto fetch = [&](int to) {
#pragma unroll
            for (int m = 0; m < M::MINE; ++m) {
                const int id = t + kPlaneThreads * m, r = id / (HD / 16);
                if (r < rows_of(to)) {
                    const int src = kept[to * kPageTokens + r];
                    ahead[m] = *reinterpret_cast<const uint4*>(kc + (size_t)page_id[src / kPageTokens] * pages.k_stride + src % kPageTokens * HD + id % (HD / 16) * 16);
                }
            }
        };
        if (first_tile < tiles) fetch(first_tile);
        for (int to = first_tile; to < tiles; ++to) {
            const int rows = rows_of(to);
            const int* source = kept + to * kPageTokens;
            uint4 mine[M::MINE];
            float was[M::MINE], most = 0.f;
#pragma unroll
            for (int m = 0; m < M::MINE; ++m) {
                const int r = (t + kPlaneThreads * m) / (HD / 16);
                mine[m] = ahead[m];
                if (r < rows) {
                    was[m] = old_scale[source[r] / kPageTokens];
                    const uint32_t even = __vmaxu2(__vmaxu2(even_sizes(mine[m].x), even_sizes(mine[m].y)), __vmaxu2(even_sizes(mine[m].z), even_sizes(mine[m].w)));
                    const uint32_t odd = __vmaxu2(__vmaxu2(odd_sizes(mine[m].x), odd_sizes(mine[m].y)), __vmaxu2(odd_sizes(mine[m].z), odd_sizes(mine[m].w)));
                    const uint32_t both = __vmaxu2(even, odd);
                    most = fmaxf(most, size_value(max(both & 0xffffu, both >> 16)) * was[m]);
                }
            }
            const float scale = e4m3_needed_scale(block_most(most, to, plane_sync<0>)), inverse = pow2_inverse(scale);
            if (to + 1 < tiles) fetch(to + 1);
            uint8_t* at = kc + (size_t)page_id[to] * pages.k_stride;
#pragma unroll
            for (int m = 0; m < M::MINE; ++m) {
                const int id = t + kPlaneThreads * m;
                if (id / (HD / 16) >= rows) continue;
                uint32_t word[4] = {mine[m].x, mine[m].y, mine[m].z, mine[m].w};
                const float ratio = was[m] * inverse;
                if (ratio > kMostHalf) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) word[x] = times_ratios<true>(word[x], ratio, ratio, ratio, ratio);
                } else if (ratio != 1.f) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) word[x] = times_ratios<false>(word[x], ratio, ratio, ratio, ratio);
                }
                *reinterpret_cast<uint4*>(at + id * 16) = make_uint4(word[0], word[1], word[2], word[3]);
            }
            if (t == 0) scales[(size_t)page_id[to] * pages.scale_stride] = scale;
        }
        return;
    }
    if (first_tile >= tiles) return;
    constexpr int APART = kPlaneThreads / 16, CHANNELS = HD / APART;            // channels of a thread: t / 16 + APART i
    const int r0 = t % 16 * 4;                                                  // its rows of a tile: r0 .. r0 + 3
    const int last_page = kept[budget - 1] / kPageTokens;
    int issued = kept[first_tile * kPageTokens] / kPageTokens, there = issued;  // pages below: on their way; there for all threads
    auto issue = [&]() {
        const uint8_t* from = vc + (size_t)page_id[issued] * pages.v_stride;
        const uint32_t to = smem_u32(staged) + issued % kStaged * M::V_PAGE;
#pragma unroll
        for (int m = 0; m < M::MINE; ++m) {
            const int id = t + kPlaneThreads * m;
            if (id < 4 * HD) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + id * 16), "l"(from + id * 16));
        }
        cp_async_commit();
        ++issued;
    };
    for (int to = first_tile; to < tiles; ++to) {
        const int rows = rows_of(to);
        int src[4];
        float was[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            src[e] = r0 + e < rows ? kept[to * kPageTokens + r0 + e] : -1;
            was[e] = old_scale[max(src[e], 0) / kPageTokens];
        }
        uint32_t word[CHANNELS] = {}, even = 0, odd = 0;
        const int page_end = kept[to * kPageTokens + rows - 1] / kPageTokens;
        for (int p = kept[to * kPageTokens] / kPageTokens; p <= page_end; p += 2) {
            // pages p and p + 1.  Those before have been read by all when a barrier has passed since: this one, or the last
            // tile's; so pages up to p + 3 may take their places.
            const int need = min(p + 1, page_end);
            if (need >= there) {
                if (issued < p) {                                               // pages between of which no row stays
                    cp_async_wait<0>();                                         // (a copy under way could land on one's that takes its place)
                    issued = p;
                }
                while (issued <= need) issue();
                if (issued - 1 - need >= 2) cp_async_wait<2>();
                else if (issued - 1 - need == 1) cp_async_wait<1>();
                else cp_async_wait<0>();
                plane_sync<1>();
                there = need + 1;
            }
            while (issued <= min(p + 3, last_page)) issue();
            uint32_t offset[4], mask = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = src[e] / kPageTokens;
                const bool here = src[e] >= 0 && x >= p && x <= p + 1;
                offset[e] = here ? x % kStaged * M::V_PAGE + src[e] % kPageTokens / 4 * 4 : 0;
                mask |= here ? 0xffu << (8 * e) : 0u;
            }
            const uint32_t low = (src[0] & 3) | (4 + (src[1] & 3)) << 4, high = (src[2] & 3) | (4 + (src[3] & 3)) << 4;
#pragma unroll
            for (int i = 0; i < CHANNELS; ++i) {
                const unsigned char* at = staged + (t / 16 + APART * i) * kPageTokens;
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(at + offset[e]);
                word[i] |= __byte_perm(__byte_perm(w[0], w[1], low), __byte_perm(w[2], w[3], high), 0x5410) & mask;
            }
        }
#pragma unroll
        for (int i = 0; i < CHANNELS; ++i) {
            even = __vmaxu2(even, even_sizes(word[i]));
            odd = __vmaxu2(odd, odd_sizes(word[i]));
        }
        const float most = fmaxf(fmaxf(size_value(even & 0xffffu) * was[0], size_value(odd & 0xffffu) * was[1]),
                                 fmaxf(size_value(even >> 16) * was[2], size_value(odd >> 16) * was[3]));
        const float scale = e4m3_needed_scale(block_most(most, to, plane_sync<1>)), inverse = pow2_inverse(scale);
        const bool same = was[0] == scale && was[1] == scale && was[2] == scale && was[3] == scale;
        if (fmaxf(fmaxf(was[0], was[1]), fmaxf(was[2], was[3])) * inverse > kMostHalf) {
#pragma unroll
            for (int i = 0; i < CHANNELS; ++i)
                word[i] = times_ratios<true>(word[i], was[0] * inverse, was[1] * inverse, was[2] * inverse, was[3] * inverse);
        } else if (!same) {
#pragma unroll
            for (int i = 0; i < CHANNELS; ++i)
                word[i] = times_ratios<false>(word[i], was[0] * inverse, was[1] * inverse, was[2] * inverse, was[3] * inverse);
        }
        uint8_t* at = vc + (size_t)page_id[to] * pages.v_stride + r0;
#pragma unroll
        for (int i = 0; i < CHANNELS; ++i) {
            uint8_t* row = at + (t / 16 + APART * i) * kPageTokens;
            if (r0 + 4 <= rows) *reinterpret_cast<uint32_t*>(row) = word[i];
            else
                for (int e = 0; r0 + e < rows; ++e) row[e] = (uint8_t)(word[i] >> (8 * e));
        }
        if (t == 0) scales[(size_t)page_id[to] * pages.scale_stride + pages.n_kv] = scale;
    }
    cp_async_wait<0>();
}

constexpr size_t kMoveBytes = 200 * 1024;   // what that kernel takes at most; longer sequences take the general one
size_t move_bytes(int hd, int max_length, int budget) {
    const size_t max_pages = (max_length + kPageTokens - 1) / kPageTokens;
    return kStaged * (size_t)hd * kPageTokens + max_pages * kPageTokens * 4 + (size_t)(budget + 63) / 64 * 64 * 4 + max_pages * 12;
}
template <int HD>
int launch_move(const E4M3Pages& pages, const EvictStrides& strides, int* dropped, const int* slots, const int* lengths, int max_length, int budget,
                int recent, int* kept, int B, int entries, cudaStream_t stream) {
    const size_t smem = move_bytes(HD, max_length, budget);
    static bool allowed[kMaxDevices] = {};
    const int st = allow_shared((const void*)kv_evict_move_kernel<HD>, kMoveBytes, allowed);
    if (st != 0) return st;
    kv_evict_move_kernel<HD><<<dim3(pages.n_kv, B, entries), kMoveThreads, smem, stream>>>(pages, strides, dropped, slots, lengths, max_length, budget,
                                                                                          recent, kept);
    return launch_status();
}

// ---- storing, for heads of a multiple of 16 channels whose rows lie on 16-byte boundaries.  A block of the cache is read once,
// 16 channels a thread (two runs of 8 that the rotation pairs), kept in registers while the block's largest value is
// found, and written in pieces of 16 or 8 bytes; values go through shared memory, since their rows are innermost in the cache.
// Query rows are rotated by blocks of their own, the angles of 16 channels read once for several heads.
// What bounds it: its reads wait for memory, in 32 warps a multiprocessor (four blocks: 26.6 us where three take 29.6 and five 28.3, the
// prompts named below; their bytes take 16.8), and turning and rounding take half of all issue slots, so codes are made two at
// a time and only a thread that has met a number that is not finite looks at each.
constexpr int kRowsThreads = 256;

__device__ __forceinline__ void load8(const bf16* p, float* x) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const float* p, float* x) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void store8(bf16* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
// Unit u of a head: two runs of 8 channels, starting at *a and *b.  Half-split pairs: run u and its partner; else neighbours.
__device__ __forceinline__ void runs_of(int u, int rot, int interleaved, int* a, int* b) {
    if (!interleaved && u < rot / 16) { *a = 8 * u; *b = *a + rot / 2; }
    else { *a = 16 * u; *b = *a + 8; }
}
// What turns a unit: for half-split pairs 8 angles, for neighbours 4 and 4; (1, 0) where nothing turns.
__device__ __forceinline__ void angles_of(int u, int rot, int interleaved, const float2* __restrict__ cs, float2* t) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = 8 * u + e;                                                // also of the pair (16 u + 2 e, 16 u + 2 e + 1)
        t[e] = 2 * i < rot ? cs[i] : make_float2(1.f, 0.f);
    }
}
__device__ __forceinline__ void turn(float& x, float& y, float2 c) {
    const float a = __fsub_rn(__fmul_rn(x, c.x), __fmul_rn(y, c.y));
    y = __fadd_rn(__fmul_rn(x, c.y), __fmul_rn(y, c.x));
    x = a;
}
__device__ __forceinline__ void turn_unit(int u, int rot, int interleaved, const float2* t, float* x) {   // x: run a, run b
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (16 * u + 2 * e < rot) turn(x[2 * e], x[2 * e + 1], t[e]);
    } else if (u < rot / 16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) turn(x[e], x[8 + e], t[e]);
    }
}
// Four codes; odd: of numbers that may not be finite.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, bool odd) {
    if (!odd) {
        unsigned short lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
        return lo | (uint32_t)hi << 16;
    }
    return e4m3_code(a) | (uint32_t)e4m3_code(b) << 8 | (uint32_t)e4m3_code(c) << 16 | (uint32_t)e4m3_code(d) << 24;
}
// A word's bytes below `n` times a power of two; the others as they are.
__device__ __forceinline__ uint32_t rescaled_bytes(uint32_t w, int n, float ratio) {
    if (n <= 0) return w;
    const uint32_t mask = n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
    const uint32_t r = times_ratios<false>(w, ratio, ratio, ratio, ratio);      // (a scale only grows here)
    return (r & mask) | (w & ~mask);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kRowsThreads, 4)
kv_store_rows_kernel(const StoreInput<T> in, const E4M3Pages kv, const int* __restrict__ cu_seqlens, const int* __restrict__ slots,
                     const int* __restrict__ start_pos, int blocks_per_seq, int blocks_kv, int N, int heads_each, T* __restrict__ q_out, int ldq) {
    constexpr int UNITS = HD / 16;                                              // of a row
    constexpr int K_MINE = (64 * UNITS + kRowsThreads - 1) / kRowsThreads;
    constexpr int V_RUNS = HD / 8, V_MINE = (16 * V_RUNS + kRowsThreads - 1) / kRowsThreads;
    __shared__ float warp_most[kRowsThreads / 32];
    __shared__ uint32_t turned[HD * 16];                                        // a value block: [channel][16 words of 4 rows]
    chain_wait();
    chain_release();                  // only now: what comes next may read older pages at once (all before this kernel is complete)
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= blocks_kv) {
        // ---- queries: a thread a unit of a token, heads_each heads
        const int id = ((int)blockIdx.x - blocks_kv) * kRowsThreads + tid;
        const int groups = (in.n_heads + heads_each - 1) / heads_each;
        const int u = id % UNITS, rest = id / UNITS, group = rest % groups, token = rest / groups;
        if (token >= N) return;
        float2 t[8];
        angles_of(u, in.rot, in.interleaved, in.cos_sin + (size_t)token * (in.rot >> 1), t);
        int a, b;
        runs_of(u, in.rot, in.interleaved, &a, &b);
        const int h1 = min(in.n_heads, (group + 1) * heads_each);
#pragma unroll 4
        for (int h = group * heads_each; h < h1; ++h) {
            float x[16];
            const T* row = in.qkv + (size_t)token * in.ld + h * HD;
            load8(row + a, x);
            load8(row + b, x + 8);
            turn_unit(u, in.rot, in.interleaved, t, x);
            T* to = q_out + (size_t)token * ldq + h * HD;
            store8(to + a, x);
            store8(to + b, x + 8);
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
    const int start = start_pos[b] - (kv.dropped ? kv.dropped[slot] : 0);
    const int block = start / kPageTokens + j;
    const int lo = max(start - block * kPageTokens, 0), hi = min(start + n_new - block * kPageTokens, kPageTokens);
    if (hi <= lo) return;                                                       // rows [lo, hi) of the block are new
    const size_t page = kv.block_table[(size_t)slot * kv.table_stride + block];
    const int token0 = first + block * kPageTokens - start;                     // of row 0
    const T* column = in.qkv + (in.n_heads + h) * HD + (plane ? in.v_offset : 0);
    float x[K_MINE > 2 * V_MINE ? K_MINE : 2 * V_MINE][16];                     // keys: a unit each; values: rows 0, 1 and 2, 3 of a run
    if (plane == 0) {
#pragma unroll
        for (int m = 0; m < K_MINE; ++m) {
            const int unit = tid + kRowsThreads * m, r = lo + unit / UNITS, u = unit % UNITS;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[m][e] = 0.f;
            if (r < hi) {
                int a, c;
                runs_of(u, in.rot, in.interleaved, &a, &c);
                const T* row = column + (size_t)(token0 + r) * in.ld;
                load8(row + a, x[m]);
                load8(row + c, x[m] + 8);
                float2 t[8];
                angles_of(u, in.rot, in.interleaved, in.cos_sin + (size_t)(token0 + r) * (in.rot >> 1), t);
                turn_unit(u, in.rot, in.interleaved, t, x[m]);
            }
        }
    } else {
#pragma unroll
        for (int m = 0; m < V_MINE; ++m) {
            const int unit = tid + kRowsThreads * m, r0 = unit / V_RUNS * 4, run = unit % V_RUNS;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float* at = x[2 * m + i / 2] + i % 2 * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) at[e] = 0.f;
                if (r0 + i >= lo && r0 + i < hi) load8(column + (size_t)(token0 + r0 + i) * in.ld + 8 * run, at);
            }
        }
    }
    constexpr int MINE = K_MINE > 2 * V_MINE ? K_MINE : 2 * V_MINE;
    uint32_t top = 0;                                                           // the largest magnitude's bits: from 0x7f800000 on not finite
#pragma unroll
    for (int m = 0; m < MINE; ++m)
        if (m < (plane ? 2 * V_MINE : K_MINE)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[m][e]) & 0x7fffffffu);
        }
    const bool odd = top >= 0x7f800000u;
    float most = __uint_as_float(top);
    if (odd) {
        most = 0.f;
#pragma unroll
        for (int m = 0; m < MINE; ++m)
            if (m < (plane ? 2 * V_MINE : K_MINE)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) most = fmaxf(most, finite_f32(x[m][e]) ? fabsf(x[m][e]) : 0.f);
            }
    }
    most = warp_max(most);
    if ((tid & 31) == 0) warp_most[tid >> 5] = most;
    float* scale_at = kv.scales + page * kv.scale_stride + plane * kv.n_kv + h;
    const float before = lo > 0 ? *scale_at : 0.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowsThreads / 32; ++w) most = fmaxf(most, warp_most[w]);
    float scale = e4m3_needed_scale(most);
    uint8_t* codes = plane ? kv.v + page * kv.v_stride + (size_t)h * kPageTokens * HD : kv.k + page * kv.k_stride + (size_t)h * kPageTokens * HD;
    if (lo > 0) {
        if (before >= scale) {
            scale = before;
        } else {                                                                // older rows' codes under the larger scale
            const float ratio = before * pow2_inverse(scale);
            if (plane == 0) {
                for (int i = tid; i < lo * UNITS; i += kRowsThreads) {
                    uint4* at = reinterpret_cast<uint4*>(codes) + i;
                    const uint4 u = *at;
                    *at = make_uint4(rescaled_bytes(u.x, 4, ratio), rescaled_bytes(u.y, 4, ratio), rescaled_bytes(u.z, 4, ratio), rescaled_bytes(u.w, 4, ratio));
                }
            } else {
                for (int i = tid; i < 4 * HD; i += kRowsThreads) {
                    const int n = lo - i % 4 * 16;                              // older rows of this piece
                    if (n <= 0) continue;
                    uint4* at = reinterpret_cast<uint4*>(codes) + i;
                    const uint4 u = *at;
                    *at = make_uint4(rescaled_bytes(u.x, n, ratio), rescaled_bytes(u.y, n - 4, ratio), rescaled_bytes(u.z, n - 8, ratio),
                                     rescaled_bytes(u.w, n - 12, ratio));
                }
                __syncthreads();                                                // pieces that hold older and new rows are written again
            }
        }
    }
    const float inverse = pow2_inverse(scale);
    if (plane == 0) {
#pragma unroll
        for (int m = 0; m < K_MINE; ++m) {
            const int unit = tid + kRowsThreads * m, r = lo + unit / UNITS, u = unit % UNITS;
            if (r >= hi) continue;
            int a, c;
            runs_of(u, in.rot, in.interleaved, &a, &c);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[m][e] *= inverse;
            *reinterpret_cast<uint2*>(codes + r * HD + a) = make_uint2(codes4(x[m][0], x[m][1], x[m][2], x[m][3], odd), codes4(x[m][4], x[m][5], x[m][6], x[m][7], odd));
            *reinterpret_cast<uint2*>(codes + r * HD + c) = make_uint2(codes4(x[m][8], x[m][9], x[m][10], x[m][11], odd), codes4(x[m][12], x[m][13], x[m][14], x[m][15], odd));
        }
        if (kv.weights)
            for (int r = lo + tid; r < hi; r += kRowsThreads) kv.weights[page * kv.weight_stride + h * kPageTokens + r] = 0.f;
    } else {
#pragma unroll
        for (int m = 0; m < V_MINE; ++m) {
            const int unit = tid + kRowsThreads * m, r4 = unit / V_RUNS, run = unit % V_RUNS;
            if (r4 >= 16) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e)                                         // (the place is turned so that lanes of a run fall into different banks)
                turned[(8 * run + e) * 16 + (r4 ^ (run & 15))] = codes4(x[2 * m][e] * inverse, x[2 * m][8 + e] * inverse, x[2 * m + 1][e] * inverse, x[2 * m + 1][8 + e] * inverse, odd);
        }
        __syncthreads();
        for (int i = tid; i < 4 * HD; i += kRowsThreads) {
            const int channel = i / 4, r0 = i % 4 * 16;
            if (r0 >= hi || r0 + 16 <= lo) continue;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = turned[channel * 16 + ((i % 4 * 4 + e) ^ ((channel >> 3) & 15))];
            uint8_t* at = codes + channel * kPageTokens + r0;
            if (r0 >= lo && r0 + 16 <= hi) {
                *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (r0 + e >= lo && r0 + e < hi) at[e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
            }
        }
    }
    if (tid == 0) *scale_at = scale;                                            // (every thread has read it before the first barrier)
}

template <typename T>
bool rows_take(const StoreInput<T>& in, const void* q_out, int ldq) {
    constexpr int per16 = 16 / sizeof(T);
    return in.hd % 16 == 0 && in.hd <= 128 && (in.interleaved || in.rot % 16 == 0) && (in.cos_sin == nullptr || in.rot > 0) && in.ld % per16 == 0 &&
           (uintptr_t)in.qkv % 16 == 0 && (!q_out || (ldq % per16 == 0 && (uintptr_t)q_out % 16 == 0));
}
template <typename T, int HD>
int launch_store_rows(const StoreInput<T>& in, const E4M3Pages& kv, const int* cu_seqlens, const int* slots, const int* start_pos, int per_seq,
                      long long blocks_kv, int N, void* q_out, int ldq, cudaStream_t stream) {
    // heads a thread turns with the same angles: four (26.6 us at 4,696 tokens of 32 + 16 heads of 128; one: 27.9, eight: 26.6)
    // once that leaves a thousand threads a multiprocessor
    const int heads_each = (long long)N * (HD / 16) * in.n_heads >= 4LL * 148 * 1024 ? 4 : 1;
    const long long threads = q_out ? (long long)N * ((in.n_heads + heads_each - 1) / heads_each) * (HD / 16) : 0;
    const long long blocks = blocks_kv + (threads + kRowsThreads - 1) / kRowsThreads;
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL || threads > 0x7fffffffLL) return kErrUnsupported;
    return launch_chained(kv_store_rows_kernel<T, HD>, dim3((unsigned)blocks), dim3(kRowsThreads), 0, stream, in, kv, cu_seqlens, slots, start_pos,
                          per_seq, (int)blocks_kv, N, heads_each, (T*)q_out, ldq);
}

template <typename T>
int launch_store(const StoreInput<T>& in, const E4M3Pages& kv, const int* cu_seqlens, const int* slots, const int* start_pos,
                 int B, int max_q_len, int N, int store, void* q_out, int ldq, cudaStream_t stream) {
    const int per_seq = (max_q_len + kPageTokens - 2) / kPageTokens + 1;
    const long long blocks_kv = store ? (long long)B * kv.n_kv * 2 * per_seq : 0;
    if (rows_take(in, q_out, ldq) && blocks_kv < 0x7fffffffLL) {
#define GTG_ROWS(HD) case HD: return launch_store_rows<T, HD>(in, kv, cu_seqlens, slots, start_pos, per_seq, blocks_kv, N, q_out, ldq, stream);
        switch (in.hd) { GTG_ROWS(16) GTG_ROWS(32) GTG_ROWS(48) GTG_ROWS(64) GTG_ROWS(80) GTG_ROWS(96) GTG_ROWS(112) GTG_ROWS(128) }
#undef GTG_ROWS
    }
    const long long blocks = blocks_kv + (q_out ? N : 0);
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL) return kErrUnsupported;
    return launch_chained(kv_store_kernel<T>, dim3((unsigned)blocks), dim3(kStoreThreads), 0, stream, in, kv, cu_seqlens, slots, start_pos,
                          per_seq, blocks_kv, N, (T*)q_out, ldq);
}
}  // namespace

// qkv: [N][ld] of the compute type (dtype 0 float, 1 bfloat16): n_heads query heads, n_kv key heads and, unless values_from_keys,
// n_kv value heads.  cos_sin: float [N][rot/2][2] or null.  store 0: queries only (another run's cache is read).
GTG_API int gtg_kv_store_e4m3(int dtype, const void* qkv, int ld, const float* cos_sin, int n_heads, int rot, int interleaved,
                              int values_from_keys, int store, const E4M3Pages* pages, const int* cu_seqlens, const int* slots,
                              const int* start_pos, int B, int max_q_len, int N, void* q_out, int ldq, cudaStream_t stream) {
    if (B <= 0 || N <= 0 || max_q_len <= 0) return 0;
    const E4M3Pages kv = *pages;
    const int n_kv = kv.n_kv, hd = kv.hd;
    if (n_heads < 0 || n_kv < 0 || hd <= 0 || rot < 0 || rot % 2 || rot > hd) return kErrBadArgument;
    const int v_offset = values_from_keys ? 0 : n_kv * hd;
    if (dtype == 0) {
        const StoreInput<float> in = {(const float*)qkv, ld, (const float2*)cos_sin, n_heads, n_kv, hd, rot, interleaved, v_offset};
        return launch_store(in, kv, cu_seqlens, slots, start_pos, B, max_q_len, N, store, q_out, ldq, stream);
    }
    const StoreInput<bf16> in = {(const bf16*)qkv, ld, (const float2*)cos_sin, n_heads, n_kv, hd, rot, interleaved, v_offset};
    return launch_store(in, kv, cu_seqlens, slots, start_pos, B, max_q_len, N, store, q_out, ldq, stream);
}

// lengths[b]: rows that the sequence in slots[b] holds.  kept: [entries][B][n_kv][budget].
GTG_API int gtg_kv_evict_e4m3(int entries, const E4M3Pages* first, long long k_entry, long long v_entry, long long scale_entry,
                              long long weight_entry, const int* slots, const int* lengths, int B, int max_length, int budget, int recent,
                              int* kept, cudaStream_t stream) {
    if (B <= 0 || entries <= 0) return 0;
    E4M3Pages pages = *first;                                                   // of entry 0
    int* dropped = const_cast<int*>(pages.dropped);
    pages.dropped = nullptr;
    const int n_kv = pages.n_kv, hd = pages.hd;
    if (budget <= 0 || recent < 0 || recent > budget || n_kv <= 0 || hd <= 0 || !pages.weights || !kept) return kErrBadArgument;
    if (B > 65535 || entries > 65535) return kErrUnsupported;
    const size_t smem = (size_t)kPageTokens * hd;
    if (smem > 40 * 1024) return kErrUnsupported;
    const EvictStrides strides = {k_entry, v_entry, scale_entry, weight_entry};
    // sequences whose weights fit in shared memory, heads of a multiple of 16 channels; else the general form
    if (hd % 16 == 0 && hd <= 128 && move_bytes(hd, max_length, budget) <= kMoveBytes) {
#define GTG_MOVE(HD) case HD: return launch_move<HD>(pages, strides, dropped, slots, lengths, max_length, budget, recent, kept, B, entries, stream);
        switch (hd) { GTG_MOVE(16) GTG_MOVE(32) GTG_MOVE(48) GTG_MOVE(64) GTG_MOVE(80) GTG_MOVE(96) GTG_MOVE(112) GTG_MOVE(128) }
#undef GTG_MOVE
    }
    kv_evict_kernel<<<dim3(n_kv, B, entries), kEvictThreads, smem, stream>>>(pages, strides, dropped, slots, lengths, max_length, budget, recent, kept);
    return launch_status();
}
