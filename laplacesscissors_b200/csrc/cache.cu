// Paged key/value cache held in 4 bits: appending to it, reading it back, attention over
// it, and the bookkeeping of its pages (lsx_cache_* of include/lsx.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <limits>

#include "cache.cuh"
#include "device_common.cuh"
#include "lsx_internal.h"

namespace lsx {
namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
    return static_cast<float>(x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// Launches `kernel` so that its prologue may overlap the end of the kernel before it.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t s,
                             Args... args) {
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}

// ---- rows of a call ------------------------------------------------------------
struct SequenceRows {
    int table;   // row of the tables, -1 when the list names none
    int first;   // its first row of the call
    int count;   // its rows
    int length;  // its positions, those of the rows last
};

__device__ __forceinline__ SequenceRows sequence_rows(const CacheView& c, const CacheRows& r, uint32_t b) {
    SequenceRows s;
    s.table = r.sequences ? r.sequences[b] : (int)b;
    if ((uint32_t)s.table >= c.table_rows) s.table = -1;
    s.first = (int)b;
    s.count = 1;
    if (r.starts) {  // what the list names beyond the call's rows is not touched
        const int rows = (int)r.rows, first = min(max(r.starts[b], 0), rows);
        s.first = first;
        s.count = max(min(r.starts[b + 1], rows) - first, 0);
    }
    s.length = s.table < 0 ? 0 : max(c.lengths[s.table], 0);
    return s;
}

// The sequence that row `row` belongs to, by bisection of the ascending starts: the last
// one that starts at or before it.  A row outside every sequence gives one whose rows
// end before it.
__device__ __forceinline__ uint32_t sequence_of(const CacheRows& r, uint32_t row) {
    if (!r.starts) return row;
    uint32_t low = 0, high = r.count;  // starts[low] <= row < starts[high]
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (r.starts[middle] <= (int)row)
            low = middle;
        else
            high = middle;
    }
    return low;
}

// The cell of `position` for head `head`, or NULL where the table names no page of the pool.
__device__ __forceinline__ uint8_t* cell_of(const CacheView& c, int table, uint32_t position, uint32_t head) {
    const uint32_t slot = position / c.page_size;
    if (table < 0 || slot >= c.table_width) return nullptr;
    const uint32_t page = (uint32_t)c.tables[(size_t)table * c.table_width + slot];
    if (page >= c.page_count) return nullptr;
    const uint32_t cells = c.page_size / kCellTokens;
    return c.pages + (((size_t)page * c.kv_heads + head) * cells + position % c.page_size / kCellTokens) *
                         cell_bytes((int)c.dim);
}

// ---- append and read -----------------------------------------------------------
// The level 0..15 of x in a group with zero z and step s (inv = 1 / s, 0 for s = 0):
// (x - z) / s rounded to nearest, ties to even, exactly.  The f32 quotient is off by less
// than 15 * 3 * 2^-24, so only where it lies next to a tie the quotient is formed in 64
// bits, which hold x - z of any f32 x that is not lost beside z.
__device__ __forceinline__ uint32_t level_of(float x, float z, float s, float inv) {
    const float t = (x - z) * inv;
    float n = rintf(t);
    if (fabsf(t - n) > 0.4999f && s > 0.f) n = (float)rint(((double)x - (double)z) / (double)s);
    return (uint32_t)(int)fminf(fmaxf(n, 0.f), 15.f);
}

// One warp a (row, head, key or value): lane l holds two elements of each group of 64, the
// two that share a byte.
template <typename T>
__global__ void __launch_bounds__(128) append_kernel(const T* k, const T* v, size_t k_row, size_t k_head, size_t v_row,
                                                     size_t v_head, CacheView c, CacheRows r) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + warp;
    const uint32_t row = (uint32_t)(unit / (2 * c.kv_heads)), head = (uint32_t)(unit % (2 * c.kv_heads)) >> 1;
    const bool value = unit & 1;
    if (row >= r.rows) return;
    const SequenceRows s = sequence_rows(c, r, sequence_of(r, row));
    const int position = s.length - s.count + (int)row - s.first;
    if ((int)row >= s.first + s.count || (int)row < s.first || position < 0) return;
    uint8_t* cell = cell_of(c, s.table, (uint32_t)position, head);
    if (!cell) return;
    const T* x = value ? v + row * v_row + head * v_head : k + row * k_row + head * k_head;
    const int t = position % kCellTokens, dim = (int)c.dim;
    for (int g = 0; g < dim / kCacheGroup; ++g) {
        const int d0 = g * 64 + (value ? (int)lane / 8 * 16 + (int)lane % 8 : 2 * (int)lane);
        const int d1 = d0 + (value ? 8 : 1);
        const float a = to_f32(x[d0]), b = to_f32(x[d1]);
        float low = fminf(a, b), high = fmaxf(a, b);
        bool finite = isfinite(a) && isfinite(b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        finite = __all_sync(0xffffffffu, finite);
        __half zero = __float2half_rn(low + 0.f);
        __half step = __float2half_rn(fmaxf(__fdiv_rn(high - __half2float(zero), 15.f), 0.f));
        const float z = __half2float(zero), s32 = __half2float(step);
        finite = finite && isfinite(z) && isfinite(s32);
        uint32_t byte = 0;
        if (finite) {
            const float inv = s32 > 0.f ? __fdiv_rn(1.f, s32) : 0.f;
            byte = level_of(a, z, s32, inv) | level_of(b, z, s32, inv) << 4;
        } else {
            zero = step = __ushort_as_half(0x7e00);
        }
        cell[value ? value_byte(dim, t, d0) : key_byte(t, d0)] = (uint8_t)byte;
        if (lane == 0) {
            __half* at = reinterpret_cast<__half*>(cell + (value ? cell_value_steps(dim) : cell_key_steps(dim)) +
                                                   step_byte(t, g));
            at[0] = step;
            at[2] = zero;
        }
    }
}

// One warp a (row, head, key or value), as in append_kernel.
template <typename T>
__global__ void __launch_bounds__(128) read_kernel(CacheView c, CacheRows r, T* k, T* v) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + warp;
    const uint32_t row = (uint32_t)(unit / (2 * c.kv_heads)), head = (uint32_t)(unit % (2 * c.kv_heads)) >> 1;
    const bool value = unit & 1;
    if (row >= r.rows) return;
    const SequenceRows s = sequence_rows(c, r, sequence_of(r, row));
    const int position = s.length - s.count + (int)row - s.first;
    if ((int)row >= s.first + s.count || (int)row < s.first) return;
    const int dim = (int)c.dim;
    T* out = (value ? v : k) + ((size_t)row * c.kv_heads + head) * dim;
    const uint8_t* cell = position < 0 ? nullptr : cell_of(c, s.table, (uint32_t)position, head);
    const int t = position % kCellTokens;
    for (int g = 0; g < dim / kCacheGroup; ++g) {
        const int d0 = g * 64 + (value ? (int)lane / 8 * 16 + (int)lane % 8 : 2 * (int)lane);
        const int d1 = d0 + (value ? 8 : 1);
        float a = position < 0 && s.table >= 0 ? 0.f : std::numeric_limits<float>::quiet_NaN(), b = a;
        if (cell) {
            const uint32_t byte = cell[value ? value_byte(dim, t, d0) : key_byte(t, d0)];
            const __half* at = reinterpret_cast<const __half*>(
                cell + (value ? cell_value_steps(dim) : cell_key_steps(dim)) + step_byte(t, g));
            const float step = __half2float(at[0]), zero = __half2float(at[2]);
            a = fmaf(step, (float)(byte & 15), zero);
            b = fmaf(step, (float)(byte >> 4), zero);
        }
        out[d0] = from_f32<T>(a);
        out[d1] = from_f32<T>(b);
    }
}

// ---- attention -----------------------------------------------------------------
// One block a (row, query head): 128 positions at a time, a score a thread, then an
// element of the output a thread, with the running maximum and sum of the softmax.
template <typename T>
__global__ void __launch_bounds__(128) attention_kernel(const T* q, size_t q_row, size_t q_head, CacheView c,
                                                        CacheRows r, uint32_t q_heads, float scale, T* out,
                                                        size_t out_row, size_t out_head) {
    const uint32_t row = blockIdx.x / q_heads, h = blockIdx.x % q_heads, head = h / (q_heads / c.kv_heads);
    const int dim = (int)c.dim, groups = dim / kCacheGroup;
    __shared__ float query[kMaxCacheDim], weight[128];
    __shared__ float reduce[4];
    const SequenceRows s = sequence_rows(c, r, sequence_of(r, row));
    if ((int)row >= s.first + s.count || (int)row < s.first) return;
    const int seen = s.length - s.count + (int)row - s.first + 1;
    T* o = out + row * out_row + h * out_head;
    for (int d = threadIdx.x; d < dim; d += 128) query[d] = to_f32(q[row * q_row + h * q_head + d]) * scale;
    float most = -INFINITY, sum = 0.f, sums[2] = {0.f, 0.f};
    const float nan = std::numeric_limits<float>::quiet_NaN();
    __syncthreads();
    for (int first = 0; first < seen; first += 128) {
        const int position = first + (int)threadIdx.x, t = position % kCellTokens;
        float score = -INFINITY;
        if (position < seen) {
            const uint8_t* cell = cell_of(c, s.table, (uint32_t)position, head);
            score = cell ? 0.f : nan;
            for (int g = 0; cell && g < groups; ++g) {
                const __half* at = reinterpret_cast<const __half*>(cell + cell_key_steps(dim) + step_byte(t, g));
                float dot = 0.f, plain = 0.f;
                for (int d = g * 64; d < g * 64 + 64; d += 2) {
                    const uint32_t byte = cell[key_byte(t, d)];
                    dot = fmaf(query[d], (float)(byte & 15), dot);
                    dot = fmaf(query[d + 1], (float)(byte >> 4), dot);
                    plain += query[d] + query[d + 1];
                }
                score += __half2float(at[0]) * dot + __half2float(at[2]) * plain;
            }
        }
        float top = score;
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        if (threadIdx.x % 32 == 0) reduce[threadIdx.x / 32] = top;
        __syncthreads();
        const float now = fmaxf(fmaxf(fmaxf(reduce[0], reduce[1]), fmaxf(reduce[2], reduce[3])), most);
        const float against = now == -INFINITY ? 0.f : now;
        weight[threadIdx.x] = position < seen ? expf(score - against) : 0.f;
        const float keep = expf(most - against);
        most = now;
        sum *= keep;
        for (int i = 0; i < 2; ++i) sums[i] *= keep;
        __syncthreads();
        for (int k = 0; k < 128 && first + k < seen; ++k) {
            const float w = weight[k];
            const uint8_t* cell = cell_of(c, s.table, (uint32_t)(first + k), head);
            sum += w;
            for (int i = 0, d = threadIdx.x; d < dim; d += 128, ++i) {
                float x = nan;
                if (cell) {
                    const int u = (first + k) % kCellTokens;
                    const __half* at = reinterpret_cast<const __half*>(cell + cell_value_steps(dim) + step_byte(u, d / 64));
                    const uint32_t byte = cell[value_byte(dim, u, d / 16 * 16 + d % 8)];
                    x = fmaf(__half2float(at[0]), (float)(d % 16 < 8 ? byte & 15 : byte >> 4), __half2float(at[2]));
                }
                sums[i] = fmaf(w, x, sums[i]);
            }
        }
        __syncthreads();
    }
    for (int i = 0, d = threadIdx.x; d < dim; d += 128, ++i)
        o[d] = from_f32<T>(s.table < 0 ? nan : seen > 0 ? sums[i] / sum : 0.f);
}

// ---- pages ---------------------------------------------------------------------
// Sum of `mine` over the threads before this one of a block of 1024, and over all of it.
// Every thread of the block calls it; `parts` holds 32 words.
__device__ __forceinline__ long long block_prefix(long long mine, long long* parts, long long* total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long below = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += below;
    }
    __syncthreads();  // the words may still be read from the call before
    if (lane == 31) parts[warp] = sum;
    __syncthreads();
    long long part = parts[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long below = __shfl_up_sync(0xffffffffu, part, o);
        if (lane >= o) part += below;
    }
    *total = __shfl_sync(0xffffffffu, part, 31);
    const long long before = __shfl_sync(0xffffffffu, part, (warp + 31) % 32);
    return sum - mine + (warp ? before : 0);
}

// Hands the lowest free pages to take(rank, page), rank 0 .. wanted - 1 in ascending
// order of the pages, and returns how many there were.  A block of 1024 threads.
template <typename Take>
__device__ long long take_free_pages(const int32_t* refs, uint32_t page_count, long long wanted, long long* parts,
                                     const Take& take) {
    long long found = 0;
    for (uint64_t base = 0; base < page_count && found < wanted; base += 4096) {
        bool open[4];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t page = base + threadIdx.x * 4 + i;
            open[i] = page < page_count && refs[page] <= 0;
            mine += open[i];
        }
        long long total, rank = found + block_prefix(mine, parts, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!open[i]) continue;
            if (rank < wanted) take(rank, (int)(base + threadIdx.x * 4 + i));
            ++rank;
        }
        found += total;
    }
    return min(found, wanted);
}

// Whether an earlier entry of the list names the same sequence.
__device__ __forceinline__ bool named_before(const int* list, int i) {
    for (int k = 0; k < i; ++k)
        if (list[k] == list[i]) return true;
    return false;
}

// lsx_cache_reserve_device.  One block: entry i of the list is thread i's.
__global__ void __launch_bounds__(1024) reserve_kernel(int32_t* tables, uint32_t table_rows, uint32_t width,
                                                       int32_t* lengths, int32_t* refs, uint32_t page_count,
                                                       uint32_t page_size, const int32_t* sequences,
                                                       const int32_t* counts, uint32_t n, int32_t* missing) {
    __shared__ int list[kMaxListed];
    __shared__ long long starts[kMaxListed + 1];
    __shared__ long long parts[32];
    const int i = (int)threadIdx.x;
    list[i] = i < (int)n ? sequences[i] : -1;
    __syncthreads();
    const int s = list[i];
    const bool valid = i < (int)n && (uint32_t)s < table_rows && !named_before(list, i);
    const long long before = valid ? max(lengths[s], 0) : 0, after = before + (valid ? max(counts[i], 0) : 0);
    const long long held = (before + page_size - 1) / page_size, needed = (after + page_size - 1) / page_size;
    long long beyond, total;
    block_prefix(max(needed - (long long)width, 0ll), parts, &beyond);
    starts[i] = block_prefix(needed - held, parts, &total);
    if (i == 0) starts[kMaxListed] = total;
    __syncthreads();
    if (beyond > 0) {  // a row of the tables is too short: nothing changes
        if (i == 0) *missing = (int)min(beyond, (long long)INT32_MAX);
        return;
    }
    const long long found = take_free_pages(refs, page_count, total, parts, [&](long long rank, int page) {
        int low = 0, high = kMaxListed;  // starts[low] <= rank < starts[high]
        while (high - low > 1) {
            const int middle = (low + high) / 2;
            if (starts[middle] <= rank)
                low = middle;
            else
                high = middle;
        }
        const long long slot = ((long long)max(lengths[list[low]], 0) + page_size - 1) / page_size + rank - starts[low];
        tables[(size_t)list[low] * width + slot] = page;
        refs[page] = 1;
    });
    __syncthreads();
    if (found < total) {  // too few: what was taken is given back
        for (long long k = 0; valid && k < needed - held && starts[i] + k < found; ++k) {
            int32_t* at = tables + (size_t)s * width + held + k;
            refs[*at] = 0;
            *at = -1;
        }
        if (i == 0) *missing = (int)min(total - found, (long long)INT32_MAX);
        return;
    }
    if (valid) lengths[s] = (int)after;
    if (i == 0) *missing = 0;
}

// lsx_cache_fork_device's bookkeeping.  One block: entry i of the lists is thread i's;
// pairs[i] is the partly filled page that child i takes a copy of, and the copy.
__global__ void __launch_bounds__(1024) fork_kernel(int32_t* tables, uint32_t table_rows, uint32_t width,
                                                    int32_t* lengths, int32_t* refs, uint32_t page_count,
                                                    uint32_t page_size, const int32_t* parents, const int32_t* children,
                                                    uint32_t n, int32_t* pairs, int32_t* missing) {
    pdl_launch_dependents();
    __shared__ int list[kMaxListed], source[kMaxListed], length[kMaxListed], fresh[kMaxListed];
    __shared__ long long parts[32];
    const int i = (int)threadIdx.x;
    list[i] = i < (int)n ? children[i] : -1;
    __syncthreads();
    const int child = list[i], parent = i < (int)n ? parents[i] : -1;
    bool valid = (uint32_t)child < table_rows && (uint32_t)parent < table_rows && lengths[child] <= 0 &&
                 !named_before(list, i);
    const long long held = valid ? max(lengths[parent], 0) : 0;
    valid = held > 0 && held <= (long long)width * page_size;
    source[i] = valid ? parent : -1;
    length[i] = (int)held;
    const bool part = valid && held % page_size;
    long long total;
    const long long rank = block_prefix(part, parts, &total);
    const long long found = take_free_pages(refs, page_count, total, parts, [&](long long k, int page) { fresh[k] = page; });
    __syncthreads();
    if (i < (int)n) pairs[2 * i] = pairs[2 * i + 1] = -1;
    if (i == 0) *missing = (int)(total - found);
    if (found < total) return;
    if (part) {
        const size_t slot = (size_t)(held / page_size);
        const int page = tables[(size_t)parent * width + slot], copy = fresh[rank];
        tables[(size_t)child * width + slot] = copy;
        refs[copy] = 1;
        pairs[2 * i] = page;
        pairs[2 * i + 1] = copy;
    }
    if (valid) lengths[child] = (int)held;
    __syncthreads();  // the fresh pages are counted before shared ones
    // the parents' whole pages, a warp an entry: an empty child is nobody's parent here
    for (int k = (int)threadIdx.x / 32; k < (int)n; k += 32) {
        if (source[k] < 0) continue;
        const int32_t* from = tables + (size_t)source[k] * width;
        int32_t* to = tables + (size_t)list[k] * width;
        for (int w = (int)threadIdx.x % 32; w < length[k] / (int)page_size; w += 32) {
            const int page = from[w];
            to[w] = page;
            if ((uint32_t)page < page_count) atomicAdd(refs + page, 1);
        }
    }
}

// lsx_cache_free_device.  A block an entry of the list; only the first that names a
// sequence frees it.
__global__ void __launch_bounds__(256) free_kernel(int32_t* tables, uint32_t table_rows, uint32_t width,
                                                   int32_t* lengths, int32_t* refs, uint32_t page_count,
                                                   uint32_t page_size, const int32_t* sequences) {
    const int s = sequences[blockIdx.x];
    if ((uint32_t)s >= table_rows) return;
    bool earlier = false;
    for (uint32_t k = threadIdx.x; k < blockIdx.x; k += 256) earlier |= sequences[k] == s;
    if (__syncthreads_or(earlier)) return;
    const long long held = max(lengths[s], 0);
    const long long pages = min((held + page_size - 1) / page_size, (long long)width);
    for (long long w = threadIdx.x; w < pages; w += 256) {
        const int page = tables[(size_t)s * width + w];
        tables[(size_t)s * width + w] = -1;
        if ((uint32_t)page < page_count) atomicSub(refs + page, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) lengths[s] = 0;
}

// The bookkeeping of lsx_cache_compact_device: `to_of[p]` is where page p of the upper
// part goes, pairs lists what moves (moved of them), refs_out the counts afterwards.
__global__ void __launch_bounds__(1024) compact_kernel(const int32_t* refs, uint32_t page_count, int32_t* refs_out,
                                                       int32_t* to_of, int32_t* pairs, int32_t* moved) {
    pdl_launch_dependents();
    __shared__ long long parts[32];
    long long live = 0, mine = 0;
    for (uint64_t page = threadIdx.x; page < page_count; page += 1024) mine += refs[page] > 0;
    block_prefix(mine, parts, &live);
    // the k-th free page below `live` is the destination of the k-th live page from there on:
    // all of the former come first in the scan
    long long holes = 0, movers = 0;
    for (uint64_t base = 0; base < page_count; base += 1024) {
        const uint64_t page = base + threadIdx.x;
        const int held = page < page_count ? refs[page] : 0;
        const bool low = (long long)page < live, hole = page < page_count && low && held <= 0, mover = !low && held > 0;
        long long some_holes, some_movers;
        const long long h = holes + block_prefix(hole, parts, &some_holes);
        const long long m = movers + block_prefix(mover, parts, &some_movers);
        if (hole) pairs[2 * h + 1] = (int)page;
        __syncthreads();  // the holes of this piece, for its movers
        if (mover) {
            const int to = pairs[2 * m + 1];
            pairs[2 * m] = (int)page;
            to_of[page] = to;
            refs_out[to] = held;
        }
        if (page < page_count) {
            if (!low) refs_out[page] = 0;
            if (!low && !mover) to_of[page] = (int)page;
            if (low && !hole) refs_out[page] = held;
        }
        holes += some_holes;
        movers += some_movers;
    }
    if (threadIdx.x == 0) {
        moved[0] = (int)movers;
        moved[1] = (int)live;
    }
}

// Copies page pairs[i][0] to page pairs[i][1] in every layer, `count` of them (*moved
// where it is given); a pair that names no page of the pool is passed over.  With `tables`
// the entries of a compacted cache follow their pages.
constexpr int kCopyThreads = 256, kCopyVectors = 8;

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(uint8_t* pool, uint32_t layers, size_t layer_bytes,
                                                                  size_t page_bytes, uint32_t page_count,
                                                                  const int32_t* pairs, uint32_t count,
                                                                  const int32_t* moved, const int32_t* tables,
                                                                  int32_t* tables_out, uint64_t entries,
                                                                  const int32_t* to_of) {
    pdl_wait();
    if (moved) count = min((uint32_t)max(*moved, 0), count);
    constexpr uint32_t kPiece = kCopyThreads * kCopyVectors;
    const uint32_t vectors = (uint32_t)(page_bytes / 16), pieces = (vectors + kPiece - 1) / kPiece;
    const uint64_t work = (uint64_t)count * layers * pieces;
    for (uint64_t item = blockIdx.x; item < work; item += gridDim.x) {
        const uint32_t piece = (uint32_t)(item % pieces);
        const uint64_t page = item / pieces;
        const uint32_t layer = (uint32_t)(page % layers), pair = (uint32_t)(page / layers);
        const uint32_t from = (uint32_t)pairs[2 * pair], to = (uint32_t)pairs[2 * pair + 1];
        if (from >= page_count || to >= page_count) continue;
        const uint4* in = reinterpret_cast<const uint4*>(pool + layer * layer_bytes + from * page_bytes);
        uint4* out = reinterpret_cast<uint4*>(pool + layer * layer_bytes + to * page_bytes);
        const uint32_t first = piece * kPiece + threadIdx.x;
        uint4 held[kCopyVectors];
#pragma unroll
        for (int i = 0; i < kCopyVectors; ++i)
            if (first + i * kCopyThreads < vectors) held[i] = in[first + i * kCopyThreads];
#pragma unroll
        for (int i = 0; i < kCopyVectors; ++i)
            if (first + i * kCopyThreads < vectors) out[first + i * kCopyThreads] = held[i];
    }
    if (!tables) return;
    const uint32_t live = (uint32_t)moved[1];
    for (uint64_t e = (uint64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < entries;
         e += (uint64_t)gridDim.x * kCopyThreads) {
        const int page = tables[e];
        tables_out[e] = (uint32_t)page >= live && (uint32_t)page < page_count ? to_of[page] : page;
    }
}

// ---- checks --------------------------------------------------------------------
int check_view(const lsx_cache_view* view, CacheView* out) {
    LSX_ENSURE(view && view->pages && view->tables && view->lengths, "invalid argument");
    LSX_ENSURE(view->head_dim > 0 && view->head_dim <= (size_t)kMaxCacheDim && view->head_dim % kCacheGroup == 0,
               "the cache holds heads of 64, 128, 192 or 256 elements");
    LSX_ENSURE(view->page_size > 0 && view->page_size % kCellTokens == 0 && view->page_size <= 65536,
               "a page holds a multiple of 16 positions, at most 65536");
    LSX_ENSURE(view->kv_heads > 0 && view->kv_heads <= 65536, "check the number of key heads");
    LSX_ENSURE(view->page_count > 0 && view->page_count <= INT32_MAX && view->table_rows <= INT32_MAX &&
                   view->table_width > 0 && view->table_width <= INT32_MAX / view->page_size,
               "check the numbers of pages, sequences and pages per sequence");
    LSX_ENSURE(reinterpret_cast<uintptr_t>(view->pages) % 16 == 0, "the pages are not aligned to 16 bytes");
    *out = CacheView{(uint8_t*)view->pages, view->tables, view->lengths, (uint32_t)view->page_count,
                     (uint32_t)view->page_size, (uint32_t)view->kv_heads, (uint32_t)view->head_dim,
                     (uint32_t)view->table_rows, (uint32_t)view->table_width};
    return LSX_OK;
}

int check_rows(const lsx_cache_rows* rows, const CacheView& view, CacheRows* out) {
    LSX_ENSURE(rows, "invalid argument");
    LSX_ENSURE(rows->rows > 0 && rows->rows <= (size_t)1 << 26 && rows->sequences <= (size_t)1 << 20 && rows->sequences > 0,
               "check the numbers of rows and sequences");
    LSX_ENSURE(rows->list || rows->sequences <= view.table_rows, "more sequences than the tables have rows");
    LSX_ENSURE(rows->starts || rows->rows == rows->sequences, "without starts each sequence has one row");
    *out = CacheRows{rows->list, rows->starts, (uint32_t)rows->sequences, (uint32_t)rows->rows};
    return LSX_OK;
}

bool known_kind(lsx_dtype kind) { return kind == LSX_F32 || kind == LSX_F16 || kind == LSX_BF16; }

// Rows of heads: `row` and `head` elements from one to the next, each head contiguous.
int check_heads(const void* data, lsx_dtype kind, size_t rows, size_t heads, size_t dim, size_t row, size_t head,
                const char* what) {
    LSX_ENSURE(data, "invalid argument");
    LSX_ENSURE(known_kind(kind), "unknown dtype");
    LSX_ENSURE(reinterpret_cast<uintptr_t>(data) % dtype_bytes(kind) == 0, std::string(what) + " not aligned to the type");
    LSX_ENSURE(row <= (size_t)1 << 40 && head <= (size_t)1 << 40, std::string(what) + ": check the strides");
    (void)rows, (void)heads, (void)dim;
    return LSX_OK;
}

int check_tables(const int32_t* tables, size_t rows, size_t width, const int32_t* lengths, const int32_t* refs,
                 size_t page_count, size_t page_size) {
    LSX_ENSURE(tables && lengths && refs, "invalid argument");
    LSX_ENSURE(page_size > 0 && page_size <= 65536, "a page holds 1..=65536 positions");
    LSX_ENSURE(page_count > 0 && page_count <= INT32_MAX && rows > 0 && rows <= INT32_MAX && width > 0 &&
                   width <= INT32_MAX / page_size,
               "check the numbers of pages, sequences and pages per sequence");
    return LSX_OK;
}

int check_pool(const lsx_cache_pool* pool) {
    LSX_ENSURE(pool && pool->data, "invalid argument");
    LSX_ENSURE(pool->layers > 0 && pool->layers <= 65536 && pool->page_count > 0 && pool->page_count <= INT32_MAX,
               "check the numbers of layers and pages");
    LSX_ENSURE(pool->page_bytes > 0 && pool->page_bytes % 16 == 0 && pool->page_bytes <= (size_t)1 << 32 &&
                   pool->layer_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(pool->data) % 16 == 0,
               "pages are multiples of 16 bytes, aligned to 16");
    LSX_ENSURE(pool->layers == 1 || pool->layer_bytes / pool->page_bytes >= pool->page_count, "layers must not overlap");
    return LSX_OK;
}

template <typename F>
int by_kind(lsx_dtype kind, const F& f) {
    if (kind == LSX_F32) return f(float{});
    if (kind == LSX_F16) return f(__half{});
    return f(__nv_bfloat16{});
}

cudaError_t launch_copy(lsx_ctx* ctx, cudaStream_t s, const lsx_cache_pool& pool, const int32_t* pairs, size_t count,
                        const int32_t* moved, const int32_t* tables, int32_t* tables_out, size_t entries,
                        const int32_t* to_of) {
    const size_t pieces = (pool.page_bytes / 16 + kCopyThreads * kCopyVectors - 1) / (kCopyThreads * kCopyVectors);
    const size_t work = std::max(count * pool.layers * pieces, (entries + kCopyThreads - 1) / kCopyThreads);
    const unsigned blocks = (unsigned)std::min<size_t>(work, (size_t)ctx->sm_count * 6);
    return launch_dependent(copy_pages_kernel, blocks, kCopyThreads, 0, s, (uint8_t*)pool.data, (uint32_t)pool.layers,
                            pool.layer_bytes, pool.page_bytes, (uint32_t)pool.page_count, pairs, (uint32_t)count, moved,
                            tables, tables_out, (uint64_t)entries, to_of);
}

}  // namespace
}  // namespace lsx

using namespace lsx;

// The context's device made current and the stream of the call.
#define LSX_CACHE_SCOPE()                                                   \
    LSX_ENSURE(ctx, "context is NULL");                                     \
    const cudaStream_t on = stream ? (cudaStream_t)stream : ctx->stream;    \
    DeviceScope scope(ctx->device);                                         \
    LSX_CUDA(scope.status, "select device")

extern "C" {

size_t lsx_cache_page_bytes(size_t kv_heads, size_t page_size, size_t head_dim) {
    return kv_heads * (page_size / kCellTokens) * (size_t)cell_bytes((int)head_dim);
}

int lsx_cache_append_device(lsx_ctx* ctx, const lsx_cache_view* view, const lsx_cache_rows* rows, const void* k,
                            const void* v, lsx_dtype kind, size_t k_row, size_t k_head, size_t v_row, size_t v_head,
                            void* stream) {
    CacheView c;
    CacheRows r;
    LSX_TRY(check_view(view, &c));
    LSX_TRY(check_rows(rows, c, &r));
    LSX_TRY(check_heads(k, kind, r.rows, c.kv_heads, c.dim, k_row, k_head, "keys"));
    LSX_TRY(check_heads(v, kind, r.rows, c.kv_heads, c.dim, v_row, v_head, "values"));
    LSX_CACHE_SCOPE();
    const uint64_t units = (uint64_t)r.rows * c.kv_heads * 2;
    LSX_ENSURE(units <= (uint64_t)INT32_MAX * 4, "too many rows and heads");
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        append_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, on>>>((const T*)k, (const T*)v, k_row, k_head, v_row,
                                                                      v_head, c, r);
        LSX_CUDA(cudaGetLastError(), "cache append");
        return (int)LSX_OK;
    });
}

int lsx_cache_read_device(lsx_ctx* ctx, const lsx_cache_view* view, const lsx_cache_rows* rows, lsx_dtype kind,
                          void* k_out, void* v_out, void* stream) {
    CacheView c;
    CacheRows r;
    LSX_TRY(check_view(view, &c));
    LSX_TRY(check_rows(rows, c, &r));
    LSX_TRY(check_heads(k_out, kind, r.rows, c.kv_heads, c.dim, 0, 0, "keys"));
    LSX_TRY(check_heads(v_out, kind, r.rows, c.kv_heads, c.dim, 0, 0, "values"));
    LSX_CACHE_SCOPE();
    const uint64_t units = (uint64_t)r.rows * c.kv_heads * 2;
    LSX_ENSURE(units <= (uint64_t)INT32_MAX * 4, "too many rows and heads");
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        read_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, on>>>(c, r, (T*)k_out, (T*)v_out);
        LSX_CUDA(cudaGetLastError(), "cache read");
        return (int)LSX_OK;
    });
}

size_t lsx_cache_attention_workspace_bytes(lsx_ctx* ctx, size_t head_dim) {
    (void)ctx, (void)head_dim;
    return 16;
}

int lsx_cache_attention_device(lsx_ctx* ctx, const lsx_cache_view* view, const lsx_cache_rows* rows, const void* q,
                               lsx_dtype kind, size_t q_heads, size_t q_row, size_t q_head, double scale, void* out,
                               size_t out_row, size_t out_head, void* workspace, size_t workspace_bytes, void* stream) {
    CacheView c;
    CacheRows r;
    LSX_TRY(check_view(view, &c));
    LSX_TRY(check_rows(rows, c, &r));
    LSX_ENSURE(q_heads > 0 && q_heads <= 65536 && q_heads % c.kv_heads == 0, "query heads are a multiple of key heads");
    LSX_TRY(check_heads(q, kind, r.rows, q_heads, c.dim, q_row, q_head, "queries"));
    LSX_TRY(check_heads(out, kind, r.rows, q_heads, c.dim, out_row, out_head, "output"));
    LSX_ENSURE(scale == scale && scale < 1e30 && scale > -1e30, "check the scale");
    LSX_CACHE_SCOPE();
    LSX_ENSURE(workspace && workspace_bytes >= lsx_cache_attention_workspace_bytes(ctx, c.dim), "workspace too small");
    LSX_ENSURE((uint64_t)r.rows * q_heads <= INT32_MAX, "too many rows and heads");
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        attention_kernel<T><<<(unsigned)(r.rows * q_heads), 128, 0, on>>>((const T*)q, q_row, q_head, c, r,
                                                                         (uint32_t)q_heads, (float)scale, (T*)out,
                                                                         out_row, out_head);
        LSX_CUDA(cudaGetLastError(), "cache attention");
        return (int)LSX_OK;
    });
}

int lsx_cache_reserve_device(lsx_ctx* ctx, int32_t* tables, size_t table_rows, size_t table_width, int32_t* lengths,
                             int32_t* refs, size_t page_count, size_t page_size, const int32_t* sequences,
                             const int32_t* counts, size_t n, int32_t* missing, void* stream) {
    LSX_TRY(check_tables(tables, table_rows, table_width, lengths, refs, page_count, page_size));
    LSX_ENSURE(sequences && counts && missing, "invalid argument");
    LSX_ENSURE(n > 0 && n <= (size_t)kMaxListed, "a call extends 1..=1024 sequences");
    LSX_CACHE_SCOPE();
    reserve_kernel<<<1, 1024, 0, on>>>(tables, (uint32_t)table_rows, (uint32_t)table_width, lengths, refs,
                                       (uint32_t)page_count, (uint32_t)page_size, sequences, counts, (uint32_t)n, missing);
    LSX_CUDA(cudaGetLastError(), "cache reserve");
    return LSX_OK;
}

int lsx_cache_fork_device(lsx_ctx* ctx, const lsx_cache_pool* pool, int32_t* tables, size_t table_rows,
                          size_t table_width, int32_t* lengths, int32_t* refs, size_t page_size, const int32_t* parents,
                          const int32_t* children, size_t n, int32_t* pairs, int32_t* missing, void* stream) {
    LSX_TRY(check_pool(pool));
    LSX_TRY(check_tables(tables, table_rows, table_width, lengths, refs, pool->page_count, page_size));
    LSX_ENSURE(parents && children && pairs && missing, "invalid argument");
    LSX_ENSURE(n > 0 && n <= (size_t)kMaxListed, "a call forks 1..=1024 sequences");
    LSX_CACHE_SCOPE();
    fork_kernel<<<1, 1024, 0, on>>>(tables, (uint32_t)table_rows, (uint32_t)table_width, lengths, refs,
                                    (uint32_t)pool->page_count, (uint32_t)page_size, parents, children, (uint32_t)n,
                                    pairs, missing);
    LSX_CUDA(cudaGetLastError(), "cache fork");
    LSX_CUDA(launch_copy(ctx, on, *pool, pairs, n, nullptr, nullptr, nullptr, 0, nullptr), "cache fork");
    return LSX_OK;
}

int lsx_cache_free_device(lsx_ctx* ctx, int32_t* tables, size_t table_rows, size_t table_width, int32_t* lengths,
                          int32_t* refs, size_t page_count, size_t page_size, const int32_t* sequences, size_t n,
                          void* stream) {
    LSX_TRY(check_tables(tables, table_rows, table_width, lengths, refs, page_count, page_size));
    LSX_ENSURE(sequences && n > 0 && n <= (size_t)1 << 20, "name 1..=2^20 sequences");
    LSX_CACHE_SCOPE();
    free_kernel<<<(unsigned)n, 256, 0, on>>>(tables, (uint32_t)table_rows, (uint32_t)table_width, lengths, refs,
                                             (uint32_t)page_count, (uint32_t)page_size, sequences);
    LSX_CUDA(cudaGetLastError(), "cache free");
    return LSX_OK;
}

size_t lsx_cache_compact_workspace_bytes(size_t page_count) { return page_count * 12 + 16; }

int lsx_cache_compact_device(lsx_ctx* ctx, const lsx_cache_pool* pool, const int32_t* tables, size_t table_rows,
                             size_t table_width, const int32_t* refs, int32_t* tables_out, int32_t* refs_out,
                             void* workspace, size_t workspace_bytes, void* stream) {
    LSX_TRY(check_pool(pool));
    LSX_ENSURE(tables && refs && tables_out && refs_out && workspace, "invalid argument");
    LSX_ENSURE(table_rows > 0 && table_rows <= INT32_MAX && table_width > 0 && table_width <= INT32_MAX,
               "check the numbers of sequences and pages per sequence");
    LSX_ENSURE(workspace_bytes >= lsx_cache_compact_workspace_bytes(pool->page_count) &&
                   reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "workspace too small or not aligned to 16 bytes");
    LSX_CACHE_SCOPE();
    int32_t* moved = (int32_t*)workspace;
    int32_t* pairs = moved + 4;
    int32_t* to_of = pairs + 2 * pool->page_count;
    compact_kernel<<<1, 1024, 0, on>>>(refs, (uint32_t)pool->page_count, refs_out, to_of, pairs, moved);
    LSX_CUDA(cudaGetLastError(), "cache compact");
    LSX_CUDA(launch_copy(ctx, on, *pool, pairs, pool->page_count, moved, tables, tables_out, table_rows * table_width, to_of),
             "cache compact");
    return LSX_OK;
}

int lsx_cache_copy_device(lsx_ctx* ctx, const lsx_cache_pool* pool, const int32_t* pairs, size_t n, void* stream) {
    LSX_TRY(check_pool(pool));
    LSX_ENSURE(pairs && n > 0 && n <= INT32_MAX, "name 1..=2^31 - 1 pairs");
    LSX_CACHE_SCOPE();
    LSX_CUDA(launch_copy(ctx, on, *pool, pairs, n, nullptr, nullptr, nullptr, 0, nullptr), "cache copy");
    return LSX_OK;
}

}  // extern "C"
