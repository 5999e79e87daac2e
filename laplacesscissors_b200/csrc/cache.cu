// Paged key/value cache held in 4 bits: appending to it, reading it back, attention over
// it, and the bookkeeping of its pages (lsx_cache_* of include/lsx.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <limits>
#include <type_traits>

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
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 blocks, unsigned threads, size_t smem, cudaStream_t s,
                             Args... args) {
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = blocks;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}

// ---- rows of a call ------------------------------------------------------------
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
// Levels.  (x - z) / s is rounded to nearest, ties to even, exactly.  Its f32 value `about` (inv = 1 / s, 0 for s = 0;
// clamped to 0..15) is off by less than 15 * 3 * 2^-24, so it decides unless it lies within 2^-16 of a tie; f16 and
// bf16 elements lie on one in a thousand cases.
constexpr float kRound = 0x1.8p23f;  // an f32 plus this has its integer in the last bits
__device__ __forceinline__ float about_level(float x, float z, float inv) { return fminf(fmaxf((x - z) * inv, 0.f), 15.f); }

// The level next to a tie k + 1/2, by the sign of (x - z) - (k + 1/2) s: x - z is a + low exactly (Knuth's sum of
// two), (k + 1/2) s has 16 bits, and its difference from the close a is exact and, unless it is 0, above low.
__device__ __forceinline__ float tied_level(float x, float z, float s, float about) {
    const float k = floorf(about), a = x - z, b = a - x, low = (x - (a - b)) + (-z - b);
    const float side = fmaf(-(k + 0.5f), s, a) + low;
    return side > 0.f || (side == 0.f && ((int)k & 1)) ? k + 1.f : k;
}
__device__ __forceinline__ uint32_t level_of(float x, float z, float s, float inv) {
    const float about = about_level(x, z, inv);
    float level = about + kRound;
    if (fabsf(about - (level - kRound)) > 0.5f - 0x1p-16f) level = tied_level(x, z, s, about) + kRound;
    return __float_as_uint(level) & 15;
}

// The extremes of a group; NaN where one of its elements is.
__device__ __forceinline__ void extremes(const float (&x)[64], float& low, float& high) {
    low = high = x[0];
#pragma unroll
    for (int e = 1; e < 64; ++e) {
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(low) : "f"(x[e]));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(high) : "f"(x[e]));
    }
}
template <typename T2, typename T>
__device__ __forceinline__ void extremes_of_pairs(const T (&x)[64], float& low, float& high) {
    T2 least = *reinterpret_cast<const T2*>(x), most = least;
#pragma unroll
    for (int e = 2; e < 64; e += 2) {
        least = __hmin2_nan(least, *reinterpret_cast<const T2*>(x + e));
        most = __hmax2_nan(most, *reinterpret_cast<const T2*>(x + e));
    }
    low = to_f32(__hmin_nan(least.x, least.y));
    high = to_f32(__hmax_nan(most.x, most.y));
}
__device__ __forceinline__ void extremes(const __half (&x)[64], float& low, float& high) { extremes_of_pairs<__half2>(x, low, high); }
__device__ __forceinline__ void extremes(const __nv_bfloat16 (&x)[64], float& low, float& high) {
    extremes_of_pairs<__nv_bfloat162>(x, low, high);
}

// A group's zero and step from its extremes, and 1 / step; false where they cannot be held.
__device__ __forceinline__ bool group_steps(float low, float high, bool finite, __half& zero, __half& step, float& inv) {
    zero = __float2half_rn(low + 0.f);
    step = __float2half_rn(fmaxf(__fdiv_rn(high - __half2float(zero), 15.f), 0.f));
    const float s = __half2float(step);
    finite = finite && isfinite(__half2float(zero)) && isfinite(s);
    if (!finite) zero = step = __ushort_as_half(0x7e00);
    inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    return finite;
}

// A row's place: its cell for `head`, or NULL where it has none.
struct RowPlace {
    uint8_t* cell;
    int position;  // negative before the sequence's first
    int after;     // rows of the sequence from this one on, 0 for a row of no sequence
    bool first;    // it is the sequence's first row of the call
    int table;
};
__device__ __forceinline__ RowPlace row_place(const CacheView& c, const CacheRows& r, uint32_t row, uint32_t head) {
    const SequenceRows s = sequence_rows(c, r, sequence_of(r, row));
    RowPlace p;
    p.after = (int)row < s.first ? 0 : max(s.first + s.count - (int)row, 0);
    p.position = s.length - p.after;
    p.first = (int)row == s.first;
    p.table = s.table;
    p.cell = p.after > 0 && p.position >= 0 ? cell_of(c, s.table, (uint32_t)p.position, head) : nullptr;
    return p;
}

// Few rows a sequence: one warp a (row, head, key or value); lane l holds two elements of each group of 64, the
// two that share a byte, and the group's extremes meet by shuffles.
template <typename T>
__global__ void __launch_bounds__(128) append_rows_kernel(const T* k, const T* v, size_t k_row, size_t k_head,
                                                          size_t v_row, size_t v_head, CacheView c, CacheRows r) {
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + warp;
    const uint32_t row = (uint32_t)(unit / (2 * c.kv_heads)), head = (uint32_t)(unit % (2 * c.kv_heads)) >> 1;
    const bool value = unit & 1;
    if (row >= r.rows) return;
    const RowPlace p = row_place(c, r, row, head);
    if (!p.cell) return;
    uint8_t* cell = p.cell;
    const T* x = value ? v + row * v_row + head * v_head : k + row * k_row + head * k_head;
    const int t = p.position % kCellTokens, dim = (int)c.dim;
    for (int g = 0; g < dim / kCacheGroup; ++g) {
        const int d0 = g * 64 + (value ? (int)lane / 8 * 16 + (int)lane % 8 : 2 * (int)lane);
        const int d1 = d0 + (value ? 8 : 1);
        const float a = to_f32(x[d0]), b = to_f32(x[d1]);
        float low = fminf(a, b), high = fmaxf(a, b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        __half zero, step;
        float inv;
        uint32_t byte = 0;
        if (group_steps(low, high, __all_sync(0xffffffffu, isfinite(a) && isfinite(b)), zero, step, inv)) {
            const float z = __half2float(zero), s = __half2float(step);
            byte = level_of(a, z, s, inv) | level_of(b, z, s, inv) << 4;
        }
        cell[value ? value_byte(dim, t, d0) : key_byte(t, d0)] = (uint8_t)byte;
        if (lane == 0) {
            __half* at = reinterpret_cast<__half*>(cell + (value ? cell_value_steps(dim) : cell_key_steps(dim)) + step_byte(t, g));
            at[0] = step;
            at[2] = zero;
        }
    }
}

// Many rows a sequence: a warp a group of 64 elements for a (sixteen rows of the call, head), and those cells
// whose first new position is among the rows.  A lane takes a position's group of keys or values whole,
// sixteen positions side by side, so that nothing is exchanged; a cell that is new throughout is put
// together in shared memory and written in one go.
constexpr int kCellWarps = 4;

template <int GROUPS>
constexpr int kAppendUnits = GROUPS == 1 ? 4 : GROUPS == 2 ? 2 : 1;  // (rows, head)s of a block

static_assert(kAppendUnits<2> <= 2 && kAppendUnits<3> == 1 && kAppendUnits<4> == 1, "two barriers");

template <typename T, int GROUPS>
__global__ void __launch_bounds__(32 * GROUPS * kAppendUnits<GROUPS>) append_cells_kernel(
    const T* k, const T* v, size_t k_row, size_t k_head, size_t v_row, size_t v_head, bool wide, CacheView c, CacheRows r) {
    constexpr int D = 64 * GROUPS, kEach = 16 / sizeof(T), kUnits = kAppendUnits<GROUPS>;
    __shared__ __align__(16) uint8_t cells[kUnits][cell_bytes(D)];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = (int)threadIdx.x / 32, lane = (int)threadIdx.x % 32, i = warp % GROUPS;
    const uint64_t unit = (uint64_t)blockIdx.x * kUnits + warp / GROUPS;
    uint8_t* shared_cell = cells[warp / GROUPS];
    // The unit's warps.  Barriers named by a register count as all sixteen, which leaves four blocks an SM
    // (30000 rows of 8 x 128 in bf16: 67 us, 80 with four blocks).
    const auto meet = [&] {
        if constexpr (GROUPS == 1)
            __syncwarp();
        else if (kUnits == 1 || warp / GROUPS == 0)
            asm volatile("bar.sync 1, %0;" ::"n"(32 * GROUPS) : "memory");
        else
            asm volatile("bar.sync 2, %0;" ::"n"(32 * GROUPS) : "memory");
    };
    const uint32_t first = (uint32_t)(unit / c.kv_heads) * kCellTokens, head = (uint32_t)(unit % c.kv_heads);
    if (first >= r.rows) return;
    RowPlace mine = {};
    if (lane < kCellTokens && first + lane < r.rows) mine = row_place(c, r, first + lane, head);
    // a cell begins here, or the sequence's rows begin inside it (those before position 0 have none)
    unsigned begins = __ballot_sync(0xffffffffu, mine.cell && (mine.first || mine.position % kCellTokens == 0));
    // sixteen lanes a group of the keys, then of the values
    const int part = 2 * i + lane / 16, g = part % GROUPS, n = lane % 16;
    const bool value = part >= GROUPS;
    for (; begins; begins &= begins - 1) {
        const int at = __ffs(begins) - 1;
        const uint32_t row = first + at;
        uint8_t* cell = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)mine.cell, at));
        const int t = __shfl_sync(0xffffffffu, mine.position, at) % kCellTokens + n;
        const int count = min(kCellTokens + n - t, __shfl_sync(0xffffffffu, mine.after, at));
        uint8_t* to = count == kCellTokens ? shared_cell : cell;
        if (n < count) {
            const T* x = (value ? v + (row + n) * v_row + head * v_head : k + (row + n) * k_row + head * k_head) + 64 * g;
            __align__(16) T raw[64];
            if (wide) {
#pragma unroll
                for (int e = 0; e < 64 / kEach; ++e)
                    *reinterpret_cast<uint4*>(raw + e * kEach) = *reinterpret_cast<const uint4*>(x + e * kEach);
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) raw[e] = x[e];
            }
            float low, high;
            extremes(raw, low, high);
            __half zero, step;
            float inv;
            group_steps(low, high, isfinite(low) && isfinite(high), zero, step, inv);  // a zero that is NaN makes all levels 0
            const float z = __half2float(zero), s = __half2float(step);
            uint8_t* part_of = to + (value ? value_byte(D, t, 64 * g) : key_byte(t, 64 * g));
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // sixteen elements: a lane of the keys' layout, a word of the values'
                uint32_t level[16];
#pragma unroll
                for (int m = 0; m < 16; ++m) level[m] = level_of(to_f32(raw[16 * e + m]), z, s, inv);
                if (value) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) part_of[4 * e + 64 * m] = (uint8_t)(level[m] | level[m + 8] << 4);
                } else {
                    uint32_t words[2] = {0, 0};
#pragma unroll
                    for (int m = 0; m < 16; ++m) words[m / 8] |= level[m] << 4 * (m % 8);
                    *reinterpret_cast<uint2*>(part_of + 16 * e) = make_uint2(words[0], words[1]);
                }
            }
            __half* steps = reinterpret_cast<__half*>(to + (value ? cell_value_steps(D) : cell_key_steps(D)) + step_byte(t, g));
            steps[0] = step;
            steps[2] = zero;
        }
        if (count == kCellTokens) {
            meet();
#pragma unroll
            for (int e = i * 32 + lane; e < cell_bytes(D) / 16; e += 32 * GROUPS)
                reinterpret_cast<uint4*>(cell)[e] = reinterpret_cast<const uint4*>(shared_cell)[e];
            meet();
        }
    }
}

// Elements 4 e .. 4 e + 3 of a position's key or value, from a cell.
__device__ __forceinline__ float4 read_four(const uint8_t* cell, int dim, int t, int d, bool value) {
    const __half* at = reinterpret_cast<const __half*>(cell + (value ? cell_value_steps(dim) : cell_key_steps(dim)) + step_byte(t, d / 64));
    const float s = __half2float(at[0]), z = __half2float(at[2]);
    uint32_t n[4];
    if (value) {
        const int at_byte = value_byte(dim, t, d / 16 * 16 + d % 8), shift = d % 16 < 8 ? 0 : 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = cell[at_byte + i * 64] >> shift & 15;
    } else {
        const uint32_t two = *reinterpret_cast<const uint16_t*>(cell + key_byte(t, d));
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = two >> 4 * i & 15;
    }
    return make_float4(fmaf(s, (float)n[0], z), fmaf(s, (float)n[1], z), fmaf(s, (float)n[2], z), fmaf(s, (float)n[3], z));
}

template <typename T>
__device__ __forceinline__ void store_four(T* to, float4 x) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(to) = x;
    } else {
        __align__(8) T out[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
        *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(out);
    }
}

// One warp a (row, head, key or value), four elements a lane at a time.
template <typename T>
__global__ void __launch_bounds__(128) read_rows_kernel(CacheView c, CacheRows r, T* k, T* v) {
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + warp;
    const uint32_t row = (uint32_t)(unit / (2 * c.kv_heads)), head = (uint32_t)(unit % (2 * c.kv_heads)) >> 1;
    const bool value = unit & 1;
    if (row >= r.rows) return;
    const RowPlace p = row_place(c, r, row, head);
    if (p.after == 0) return;
    const int dim = (int)c.dim;
    T* out = (value ? v : k) + ((size_t)row * c.kv_heads + head) * dim;
    const float none = p.position < 0 && p.table >= 0 ? 0.f : std::numeric_limits<float>::quiet_NaN();
    for (int d = 4 * (int)lane; d < dim; d += 128)
        store_four(out + d, p.cell ? read_four(p.cell, dim, p.position % kCellTokens, d, value) : make_float4(none, none, none, none));
}

// One warp a (sixteen rows of the call, head): each of their cells comes into shared memory in one go.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(32 * kCellWarps) read_cells_kernel(CacheView c, CacheRows r, T* k, T* v) {
    constexpr int D = 64 * GROUPS;
    __shared__ __align__(16) uint8_t cells[kCellWarps][cell_bytes(D)];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = (int)threadIdx.x / 32, lane = (int)threadIdx.x % 32;
    const uint64_t unit = (uint64_t)blockIdx.x * kCellWarps + warp;
    const uint32_t first = (uint32_t)(unit / c.kv_heads) * kCellTokens, head = (uint32_t)(unit % c.kv_heads);
    if (first >= r.rows) return;
    RowPlace mine = {};
    if (lane < kCellTokens && first + lane < r.rows) mine = row_place(c, r, first + lane, head);
    // the rows in runs of one cell: a run ends where the cell changes
    const unsigned long long cell_here = mine.after > 0 ? (unsigned long long)mine.cell : 1;  // 1: a row of no sequence
    const unsigned long long cell_before = __shfl_up_sync(0xffffffffu, cell_here, 1);
    unsigned begins = __ballot_sync(0xffffffffu, lane < kCellTokens && (lane == 0 || cell_here != cell_before || mine.first));
    const float nan = std::numeric_limits<float>::quiet_NaN();
    while (begins) {
        const int at = __ffs(begins) - 1;
        begins &= begins - 1;
        const int end = begins ? __ffs(begins) - 1 : kCellTokens;
        const unsigned long long which = __shfl_sync(0xffffffffu, cell_here, at);
        if (which == 1) continue;
        const uint4* from = reinterpret_cast<const uint4*>(which);
        if (from) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < (cell_bytes(D) / 16 + 31) / 32; ++e)
                if (e * 32 + lane < cell_bytes(D) / 16) reinterpret_cast<uint4*>(cells[warp])[e * 32 + lane] = from[e * 32 + lane];
            __syncwarp();
        }
        for (int n = at; n < end; ++n) {
            const int position = __shfl_sync(0xffffffffu, mine.position, n), table = __shfl_sync(0xffffffffu, mine.table, n);
            const float none = position < 0 && table >= 0 ? 0.f : nan;
            const size_t to = ((size_t)(first + n) * c.kv_heads + head) * D;
#pragma unroll
            for (int value = 0; value < 2; ++value)
                for (int d = 4 * lane; d < D; d += 128)
                    store_four((value ? v : k) + to + d, from ? read_four(cells[warp], D, position % kCellTokens, d, value)
                                                              : make_float4(none, none, none, none));
        }
    }
}

// ---- attention -----------------------------------------------------------------
// Formulas.  With n, s, z a key's levels, steps and zeros, q . k = sum over its groups of
// s (n . q) + z (1 . q), and with those of the values out = (sum over positions of p s n +
// p z) / sum p.  The products n . q and (p s) n are matrix products on the tensor cores
// (m16n8k16, f16 in, f32 sums) whose operand n needs no arithmetic: a level in bits 0-3 or
// 4-7 of an f16 is the subnormal n 2^-24 or n 2^-20, exactly, so a word of eight levels
// gives its four operand registers by one shift and four masks; what is over in the
// powers of two goes into q (2^-4 for the second kind) and the scaling behind the sum.  The
// cache is the instructions' 16-row operand (positions of the keys, elements of the
// values) and the call's rows are its 8 columns, so that few rows leave little unused.
//
// Rounding.  A query row is scaled by a power of two to below 2^14 and held as f16, which
// holds f16 and bf16 queries exactly down to 2^-38 of the row's largest element, 2^-34 where they meet levels in
// bits 4-7, or for f32 (LOW) as f16 high and low parts: 22 bits, and none below 2^-39 of the row's largest.
// A score stays in the products' units and its difference from the row's reference takes the scale and the powers of
// two: taken by the scores they would round away what a score of 2^31 and more has over the next, and pass what f32 holds (1% of
// the time).
//
// A weight p is taken against that reference, and p s times a unit of its row and group is held the same two ways: 11 bits are
// half a step of an f16 result, twice 11 those of f32.  The unit keeps that product below 2^15; where it might pass (or a
// weight 2^20) the reference becomes the row's largest score and the unit leaves 2^7 for the largest product that the row
// has met in the group, so that 2^-21 of that still has 11 bits, and 2^-10 of it 22, whatever the other groups' steps are and
// whatever steps positions of little weight have.  (With one reference for all groups, a group whose steps are 1e-8 of the
// other's was 7.0e-3 of its size off in f32, now 4.9e-7.)  Steady sequences move it about once.  It costs registers and code: with the
// scores' differences 16 x 4113 positions in f32 take 37.7 instead of 34.6 us, parts of prompts in bf16 1144 instead of 1089, up to
// 6 rows of heads of 256 78.7 instead of 70.1.
//
// Everything else is f32, and exp2 by the hardware (2^-22 of a weight).  The sum of p s n and that of p z
// are often large beside what is left of them, and the tensor cores cut what they add to a sum:
// f32 calls take n - 8 and z + 8 s instead, whose sums are as small as the result (16 x 4113
// positions: 4.5e-7 of the result's size off, 1.8e-5 without).
//
// The low parts of f32 are products of their own.  Where a tile has four rows at most (HALF) they
// take the columns that would be left unused, four further on, and the halves are added by one
// exchange: half the products (16 x 4113 positions: 34.5 us instead of 37.1, before the units).
//
// Work.  The pairs of cells (32 positions of one head) that the rows of a call see, in the
// order of sequence, head, tile of rows and position, are cut into equal runs, one a block;
// the first and last tile of a run may be shared with neighbours, whose parts
// attention_merge_kernel adds up in a fixed order.  So any mix of lengths fills the card,
// the workspace goes by the number of blocks, and nothing needs the lengths on the host.
// A warp streams every fourth pair of the run through its own ring in shared memory by bulk
// copies, with its own softmax; the warps' sums meet at a tile's end.
//
// Positions of a table row up to which tiles are not shared.
constexpr int kWholeTokens = 512;
constexpr int kAttentionWarps = 4, kAttentionThreads = 32 * kAttentionWarps;

// Floats of a row's part: its sums, its reference, the sum of its weights and its scores' factor.
constexpr int part_row(int dim) { return dim + 4; }
// The reference of a row that has seen nothing: below all scores, which are below 2^45 (heads of 256 elements, steps and
// zeros below 2^16, levels below 2^4, queries below 2^14), and still a number when it is taken from one.
constexpr float kNoReference = -0x1p100f;

// GROUPS: of 64 elements; NT: eights of a tile's rows; LOW: f32; HALF: four rows, the low parts beside them.
template <int GROUPS, int NT, bool LOW, bool HALF>
struct AttentionShape {
    static constexpr int kDim = 64 * GROUPS, kPart = part_row(kDim), kRows = HALF ? 4 : 8 * NT, kCell = cell_bytes(kDim), kStage = 2 * kCell;
    // registers a thread: the sums and the queries, beside 75 and more for the rest; where those are not left the
    // queries go to shared memory.  Blocks of an SM, measured in us (three, four): one row of 128, 131072 positions,
    // 39.3 and 42.7; parts of prompts in heads of 64 526 and 440; (two, three) one row of 256, 62 and 87.
    static constexpr int kLoad = NT * GROUPS, kHeld = (LOW && !HALF ? 32 : 24) * kLoad;
    static constexpr int kBlocksPerSm = kHeld <= 24 || (NT == 2 && kHeld <= 48) ? 4 : kHeld <= 96 && GROUPS < 4 && (NT == 1 || LOW) ? 3 : 2;
    static constexpr bool kSharedQuery = kHeld > 180;
    static constexpr int kQuery = kSharedQuery ? kLoad * 4 * 32 * (LOW && !HALF ? 16 : 8) : 0;
    static constexpr int kPlain = kSharedQuery ? kAttentionWarps * kLoad * 4 * 8 : 0;
    static constexpr int kRoom = (228 * 1024 / kBlocksPerSm - 1400 - kQuery - kPlain) / (kAttentionWarps * kStage);
    static constexpr int kStages = kRoom > 6 ? 6 : kRoom;
    static constexpr int kAtOnce = GROUPS <= 2 && (NT == 1 || !LOW) ? 2 : 1;  // cells whose products are under way at the same time
    static constexpr int kRing = kAttentionWarps * kStages * kStage;
    static constexpr int kParts = kAttentionWarps * kRows * kPart * 4;  // the warps' sums, in the ring's memory
    static constexpr int kAside = kAttentionWarps * NT * (4 * GROUPS + 1) * 32;  // sums put aside, four floats each
    static constexpr int kBars = kAttentionWarps * kStages * 8;
    static constexpr int kShared = (kRing > kParts ? kRing : kParts) + kPlain + kQuery + kBars;
    static_assert(kStages >= 2 && kBlocksPerSm * (kShared + 1200) <= 228 * 1024, "shared memory");
};

struct AttentionCall {
    const void* q;
    void* out;
    size_t q_row, q_head, out_row, out_head;
    uint32_t group;            // query heads a key head
    uint32_t tokens, subs;     // rows of a tile: `tokens` positions' (a power of two) heads, or a part of one position's
    uint32_t used;             // of the tile's rows, those that hold any
    float scale;               // times log2 e
    bool wide;                 // queries lie to 16 bytes
    bool whole;                // tiles are not shared
    int* shares;               // [blocks] parts of the tile that a block starts and others finish, 0 where there is none
    int4* tails;               // [blocks] that tile's first row, key head, part of it, and positions
    float* parts;              // [2 blocks][used][part_row(dim)]
    float4* aside;             // [warps][rows / 8][dim / 16 + 1][32]: sums that a thread puts aside
};

// c += a b, and c = a b.
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Two f32 in one register pair, for the instructions that take both: the values of rows 2 j and 2 j + 1.
struct Two {
    unsigned long long bits;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return d;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
    return d;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
    return d;
}

__device__ __forceinline__ Two both(Two a) { return a; }
// The same held as bf16, in one register.
struct PackedTwo {
    uint32_t bits;
    __device__ __forceinline__ PackedTwo() {}
    __device__ __forceinline__ PackedTwo(float a, float b) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
        bits = *reinterpret_cast<const uint32_t*>(&x);
    }
};
__device__ __forceinline__ Two both(PackedTwo a) { return Two(__uint_as_float(a.bits << 16), __uint_as_float(a.bits & 0xffff0000u)); }

__device__ __forceinline__ uint32_t pack_f16(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
// Over the threads of equal lane % 4.
__device__ __forceinline__ float across_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 4);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    return x + __shfl_xor_sync(0xffffffffu, x, 16);
}
__device__ __forceinline__ float across_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
// Two levels of a word as f16, those in bits 0-3 (ODD: 4-7) of its halves: times 2^-24 (2^-20) as subnormals, or
// CENTRED: less 8, from 1024 + n (64 + n), whose last bits the level fills.
template <bool ODD, bool CENTRED>
__device__ __forceinline__ uint32_t levels_f16(uint32_t word) {
    const uint32_t bits = word & (ODD ? 0x00f000f0u : 0x000f000fu);
    if constexpr (!CENTRED) {
        return bits;
    } else {
        uint32_t x;
        asm("add.f16x2 %0, %1, %2;" : "=r"(x) : "r"(bits | (ODD ? 0x54005400u : 0x64006400u)), "r"(ODD ? 0xd480d480u : 0xe408e408u));
        return x;
    }
}

// An 8 x 8 matrix of f16, two neighbours of row lane / 4 a thread, transposed.
__device__ __forceinline__ uint32_t transpose_f16(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Sixteen consecutive elements of a query as they lie in memory, four bytes of them a word.
// Reduced to the largest magnitude's bits as f32 (above those of infinity for a NaN), and pairs
// of them scaled to f16.
template <typename T>
struct Query16 {
    static constexpr int kWords = 4 * (int)sizeof(T);
    uint32_t word[kWords];

    __device__ __forceinline__ void load(const T* x, bool wide) {  // wide: at a 16-byte boundary
        if (wide) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 raw = reinterpret_cast<const uint4*>(x)[i];
                word[4 * i] = raw.x, word[4 * i + 1] = raw.y, word[4 * i + 2] = raw.z, word[4 * i + 3] = raw.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) word[i] = reinterpret_cast<const uint32_t*>(x)[i];
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
            for (int i = 0; i < kWords; ++i) word[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) word[i] = 0;
    }
    // The larger of `most` and the magnitudes, as bits: those of an f32, or two 16-bit values side by side.
    __device__ __forceinline__ uint32_t most(uint32_t top) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4)
                top = max(top, word[i] & 0x7fffffffu);
            else
                top = __vmaxu2(top, word[i] & 0x7fff7fffu);
        }
        return top;
    }
    static __device__ __forceinline__ uint32_t most_f32(uint32_t top) {
        if constexpr (sizeof(T) == 4) return top;
        const uint32_t half = max(top & 0xffffu, top >> 16);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return half << 16;
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)half)));
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word[i]);
        const uint32_t bits = i % 2 ? word[i / 2] >> 16 : word[i / 2] & 0xffffu;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(bits << 16);
        return __half2float(__ushort_as_half((unsigned short)bits));
    }
};

// 2^power for power in -126 .. 127.
__device__ __forceinline__ float pow2(int power) { return __int_as_float((power + 127) << 23); }

// A part of a tile that a block works on.
struct TilePart {
    int first, last;   // pairs, of
    int pairs;         // those of the tile; 0 behind the run's last part
    int row;           // first row of the call
    int positions;     // that the rows stand for
    int least, seen;   // what the first row sees; what the last sees and the table covers
    int head, sub;     // key head, and which part of its query heads
    int table;         // row of the tables, -1 for none
};

template <typename T, int GROUPS, int NT, bool LOW, bool HALF>
__global__ void __launch_bounds__(kAttentionThreads, (AttentionShape<GROUPS, NT, LOW, HALF>::kBlocksPerSm))
    attention_kernel(CacheView c, CacheRows r, AttentionCall call) {
    using Shape = AttentionShape<GROUPS, NT, LOW, HALF>;
    constexpr bool BOTH = LOW && !HALF;  // low parts by products of their own
    // What 11 bits leave of p s acts on n; taken from the sum of p z eight times, it acts on n - 8.  Where the
    // result has 11 bits too that shows (60 sequences of 5000 positions, f16: 2.4e-4 of the result's size off,
    // 2.2e-4 with it, 2.1e-4 by the result's own rounding; 46.1 us, 45.4 without), not in the 8 of bf16.
    constexpr bool kCentred = std::is_same<T, __half>::value;
    static_assert(!HALF || (LOW && NT == 1), "four rows");
    constexpr int D = Shape::kDim, kStages = Shape::kStages;
    constexpr float kMostUnit = 0x1p100f, kRoom = 0x1p7f;
    // Units of two rows; one register each where there are many (up to 6 rows a sequence of heads of 256, bf16: 72 us, 75 in two).
    using Units = std::conditional_t<(NT * GROUPS > 4), PackedTwo, Two>;
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ TilePart part;
    __shared__ long long scan[kAttentionWarps], found[2];
    const int warp = (int)threadIdx.x / 32, lane = (int)threadIdx.x % 32, quad = lane / 4, j = lane % 4;
    const float nan = std::numeric_limits<float>::quiet_NaN();
    uint8_t* ring = shared + warp * kStages * Shape::kStage;
    float* warp_sums = reinterpret_cast<float*>(shared);
    uint2* queries = reinterpret_cast<uint2*>(shared + Shape::kShared - Shape::kBars - Shape::kQuery);
    float2* warp_plain = reinterpret_cast<float2*>(shared + Shape::kShared - Shape::kBars - Shape::kQuery - Shape::kPlain) +
                         warp * Shape::kPlain / (8 * kAttentionWarps) + j;
    uint64_t* bars = reinterpret_cast<uint64_t*>(shared + Shape::kShared - Shape::kBars) + warp * kStages;
    const int tokens = (int)call.tokens;
    const uint32_t tiles_of = c.kv_heads * call.subs;
    if (lane == 0)
        for (int i = 0; i < kStages; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
    pdl_launch_dependents();
    pdl_wait();

    const int covered = (int)min((long long)c.table_width * c.page_size, (long long)INT32_MAX);  // positions of a table row

    // ---- the block's run: each thread takes some of the sequences
    const uint32_t each = (r.count + kAttentionThreads - 1) / kAttentionThreads;
    const uint32_t mine_first = min(threadIdx.x * each, r.count), mine_end = min(mine_first + each, r.count);
    long long mine = 0;
    for (uint32_t b = mine_first; b < mine_end; ++b) mine += sequence_cost(sequence_rows(c, r, b), tokens) * tiles_of;
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long below = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += below;
    }
    if (lane == 31) scan[warp] = before;
    __syncthreads();
    long long total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w < kAttentionWarps; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    const long long shares = total + gridDim.x - 1;
    const long long run = max(shares >> 32 ? shares / gridDim.x : (long long)((uint32_t)shares / gridDim.x), (long long)kLeastRun);
    Run left;
    left.at = run * blockIdx.x;
    left.end = min(left.at + run, total);
    if (threadIdx.x == 0) call.shares[blockIdx.x] = 0;
    if (left.at >= left.end) return;
    if (mine > 0 && before <= left.at && left.at < before + mine) {
        for (uint32_t n = mine_first; n < mine_end; ++n) {
            const long long cost = sequence_cost(sequence_rows(c, r, n), tokens) * tiles_of;
            if (left.at < before + cost) {
                found[0] = n;
                found[1] = left.at - before;
                break;
            }
            before += cost;
        }
    }
    __syncthreads();
    left.sequence = (uint32_t)found[0];
    left.offset = found[1];

    // The first warp finds the next part of a tile in the run.
    const auto next_part = [&] {
        TilePart next;
        next.pairs = 0;
        while (left.at < left.end) {
            const SequenceRows s = sequence_rows(c, r, left.sequence);
            RunTile tile;
            if (!next_tile(left, s, tokens, tiles_of, call.whole, tile)) continue;
            const int base = s.length - s.count, tile_end = min(s.count, (tile.k + 1) * tokens);
            next.first = tile.first;
            next.last = tile.last;
            next.pairs = tile.pairs;
            next.row = s.first + tile.k * tokens;
            next.positions = tile_end - tile.k * tokens;
            next.least = base + tile.k * tokens + 1;
            next.seen = min(base + tile_end, covered);
            next.head = (int)(call.subs == 1 ? tile.head : tile.head / call.subs);
            next.sub = (int)(call.subs == 1 ? 0 : tile.head % call.subs);
            next.table = s.table;
            break;
        }
        if (lane == 0) part = next;
    };
    int stage = 0, into = 0;  // the ring's next stage to take and to fill
    uint32_t phase = 0;       // that the barriers of this turn of the ring complete
    bool dead = false;        // a copy did not arrive in time
    const uint32_t per_page = c.page_size / kCellTokens;
    const bool together = per_page % 2 == 0;  // both cells of a pair lie in one page, one behind the other
    const size_t page_bytes = (size_t)c.kv_heads * per_page * Shape::kCell;

    for (;;) {
        if (warp == 0) next_part();
        fence_proxy_async_shared();  // the ring held sums and queries,
        __syncthreads();             // which all threads have read
        const int first = part.first, last = part.last, least = part.least, seen = part.seen, pairs = part.pairs;
        const int head = part.head, sub = part.sub;
        if (pairs == 0) return;
        // row i of the tile: head sub * rows + i of the one position, or head i % group of position i / group
        const auto place = [&](int i, int& token, int& h) {
            token = call.subs > 1 ? 0 : i / (int)call.group;
            h = call.subs > 1 ? sub * Shape::kRows + i : i % (int)call.group;
            return h < (int)call.group && token < part.positions;
        };

        // ---- the queries are on their way while the first copies are looked up
        Query16<T> raw[NT][GROUPS];
        int sees[NT];  // positions that the thread's row sees
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            int token, h;
            const bool row = place(HALF ? quad % 4 : 8 * t + quad, token, h);
            sees[t] = row ? least + token : 0;
            const T* x = static_cast<const T*>(call.q) + (size_t)(part.row + token) * call.q_row +
                         (size_t)(head * (int)call.group + h) * call.q_head + 16 * j;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                if (row)
                    raw[t][g].load(x + 64 * g, call.wide);
                else
                    raw[t][g].clear();
            }
        }

        // ---- the stream of pairs: warp w takes pairs first + w, first + w + 4, ..
        const int stop = min(last, seen <= 0 ? 0 : ((seen - 1) >> 5) + 1);  // pairs beyond hold nothing
        const int mine_pairs = max(0, (stop - first - warp + kAttentionWarps - 1) / kAttentionWarps);
        const int32_t* table = c.tables + (size_t)max(part.table, 0) * c.table_width;
        const uint32_t seen_cells = seen <= 0 ? 0 : ((seen - 1) >> 4) + 1;
        const uint8_t* head_cells = c.pages + (size_t)head * per_page * Shape::kCell;
        // Each lane looks up one of the next 32 pairs and copies it when a stage is free.
        const uint8_t* from[2] = {nullptr, nullptr};
        uint32_t absent[2] = {0, 0};  // of the 32, those whose first or second cell has no page
        const auto look_up = [&](int n) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (u == 1 && together) {
                    absent[1] = absent[0];
                    break;
                }
                const uint32_t cell = 2u * (uint32_t)(first + warp + n * kAttentionWarps) + u;
                from[u] = nullptr;
                if (n < mine_pairs && cell < seen_cells) {
                    const uint32_t slot = cell / per_page, page = (uint32_t)table[slot];
                    if (page < c.page_count) from[u] = head_cells + page * page_bytes + (cell - slot * per_page) * Shape::kCell;
                }
                absent[u] = ~__ballot_sync(0xffffffffu, from[u] != nullptr);
            }
        };
        look_up(lane);
        int issued = 0;
        uint32_t gone = 0;  // two bits a stage: cells without a page
        const auto issue = [&] {
            if (issued >= mine_pairs || dead) return;
            const int turn = issued & 31;
            gone = (gone & ~(3u << 2 * into)) | (absent[0] >> turn & 1u) << 2 * into | (absent[1] >> turn & 1u) << (2 * into + 1);
            if (lane == turn) {
                uint8_t* to = ring + into * Shape::kStage;
                if (together && from[0]) {
                    mbar_expect_tx(bars + into, Shape::kStage);
                    bulk_load(to, from[0], Shape::kStage, bars + into);
                } else if (!from[0] && !from[1]) {
                    mbar_arrive(bars + into);
                } else {
                    mbar_expect_tx(bars + into, from[0] && from[1] ? Shape::kStage : Shape::kCell);
                    if (from[0]) bulk_load(to, from[0], Shape::kCell, bars + into);
                    if (from[1]) bulk_load(to + Shape::kCell, from[1], Shape::kCell, bars + into);
                }
            }
            into = into + 1 == kStages ? 0 : into + 1;
            if ((++issued & 31) == 0) look_up(issued + lane);
        };
#pragma unroll 1
        for (int n = 0; n < kStages - 1; ++n) issue();

        // ---- queries as the products' columns: the thread's rows of the results are 2 j and 2 j + 1 of each eight
        uint32_t query[Shape::kSharedQuery ? 1 : NT * GROUPS * 4][BOTH ? 4 : 2];
        float factor[NT][2];
        Two plain_of[Shape::kSharedQuery ? 1 : NT][GROUPS];
        const auto plain = [&](int n, int g) -> Two {
            if constexpr (Shape::kSharedQuery) {
                const float2 x = warp_plain[(n * GROUPS + g) * 4];
                return Two(x.x, x.y);
            } else {
                return plain_of[n][g];
            }
        };
        int limit[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint32_t top = 0;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) top = raw[t][g].most(top);
            top = Query16<T>::most_f32(top);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const bool fine = top < 0x7f800000u;
            // 2^power takes the largest into 2^13 .. 2^14
            const int power = fine && top ? 13 - max((int)(top >> 23) - 127, -100) : 0;
            // a row that is not finite gives NaN; the scale's sign goes to the queries, its size into the scores' differences
            const float up = fine ? copysignf(pow2(power), call.scale) : nan;
            const float of_row = fminf(fabsf(call.scale) * pow2(LOW ? -power : 12 - power) * (LOW ? 1.f : 0x1p12f), std::numeric_limits<float>::max());
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int holder = (HALF ? (2 * j + i) % 4 : 2 * j + i) * 4;
                factor[t][i] = __shfl_sync(0xffffffffu, of_row, holder);
                limit[t][i] = __shfl_sync(0xffffffffu, sees[t], holder);
            }
            // word w (8 elements), step e: elements e, e + 4 and e + 2, e + 6; as subnormals the odd ones' levels are 16 times as large
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                float ones[4];  // the levels' factor of the zeros: the sum of the queries, with all levels 1
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float by = e && !LOW ? up * 0.0625f : up;
                        const auto value = [&](int i) { return fine ? raw[t][g].value(8 * w + e + i) * by : nan; };
                        const float y0 = value(0), y4 = value(4), y2 = value(2), y6 = value(6);
                        const int f = (t * GROUPS + g) * 4 + w * 2 + e;
                        const uint32_t one = LOW ? 0x3c003c00u : e ? 0x00100010u : 0x00010001u, a[4] = {one, one, one, one};
                        uint32_t x0 = pack_f16(y0, y4), x1 = pack_f16(y2, y6), l0 = 0, l1 = 0;
                        if (LOW) {
                            const float2 h0 = unpack_f16(x0), h1 = unpack_f16(x1);
                            l0 = pack_f16(y0 - h0.x, y4 - h0.y);
                            l1 = pack_f16(y2 - h1.x, y6 - h1.y);
                        }
                        if (HALF && quad >= 4) x0 = l0, x1 = l1;
                        if (w + e == 0)
                            mma_f16_first(ones, a, x0, x1);
                        else
                            mma_f16(ones, a, x0, x1);
                        if (BOTH) mma_f16(ones, a, l0, l1);
                        if constexpr (Shape::kSharedQuery) {
                            if (warp == f % kAttentionWarps) {
                                uint2* at = queries + f * (BOTH ? 2 : 1) * 32 + lane;
                                at[0] = make_uint2(x0, x1);
                                if constexpr (BOTH) at[32] = make_uint2(l0, l1);
                            }
                        } else {
                            query[f][0] = x0, query[f][1] = x1;
                            if constexpr (BOTH) query[f][2] = l0, query[f][3] = l1;
                        }
                    }
                if (HALF)
                    for (int i = 0; i < 2; ++i) ones[i] += __shfl_xor_sync(0xffffffffu, ones[i], 2);
                if constexpr (Shape::kSharedQuery) {
                    if (quad == 0) warp_plain[(t * GROUPS + g) * 4] = make_float2(ones[0], ones[1]);
                } else {
                    plain_of[t][g] = Two(ones[0], ones[1]);
                }
            }
        }
        if constexpr (Shape::kSharedQuery) __syncthreads();

        float out[NT][4 * GROUPS][4], reference[NT][2];
        Two sum[NT], zeros[NT][GROUPS];
        Units unit[NT][GROUPS], eighth[kCentred ? NT : 1][GROUPS];  // and 8 over it
        float most_unit[GROUPS];  // the largest unit of a group among the thread's rows
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) most_unit[g] = kMostUnit;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int n = 0; n < 4 * GROUPS; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) out[t][n][i] = 0.f;
            reference[t][0] = reference[t][1] = kNoReference;
            sum[t] = Two(0.f);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                zeros[t][g] = Two(0.f);
                unit[t][g] = Units(kMostUnit, kMostUnit);
                if constexpr (kCentred) eighth[t][g] = Units(8.f / kMostUnit, 8.f / kMostUnit);
            }
        }

        const uint32_t pick = quad & 1 ? 0x7632u : 0x5410u;  // a thread's position among two: its step and zero

        // kAtOnce cells at `held`, the first of them at position `start`.  EDGE: some row does not see all of
        // their positions, or one is missing (bits of `none`).
        const auto take = [&](auto edge_tag, const uint8_t* held, int start, uint32_t none) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            constexpr int U = Shape::kAtOnce;
            const int position = start + quad;  // the thread's positions: this and every eighth on
            const auto there = [&](int u, int i) { return position + 16 * u + 8 * i < seen && !(none >> u & 1); };
            const auto blind = [&](int u, int i, int n, int row) {
                return !there(u, i) || position + 16 * u + 8 * i >= limit[n][row];
            };
            // n . q [row 2 j, 2 j + 1 of position, of position + 8]; steps over all cells and groups in turn, so that
            // no product waits for the one before
            float dot[U][GROUPS][NT][4];
            uint4 words[U][GROUPS];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
                    words[u][g] = *reinterpret_cast<const uint4*>(held + u * Shape::kCell + (g * 32 + lane) * 16);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int half = 0; half < (BOTH ? 2 : 1); ++half)
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int g = 0; g < GROUPS; ++g) {
                                const uint32_t low = w ? words[u][g].y : words[u][g].x, high = w ? words[u][g].w : words[u][g].z;
                                const uint32_t a[4] = {e ? levels_f16<true, LOW>(low) : levels_f16<false, LOW>(low),
                                                       e ? levels_f16<true, LOW>(high) : levels_f16<false, LOW>(high),
                                                       e ? levels_f16<true, LOW>(low >> 8) : levels_f16<false, LOW>(low >> 8),
                                                       e ? levels_f16<true, LOW>(high >> 8) : levels_f16<false, LOW>(high >> 8)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    const int f = (n * GROUPS + g) * 4 + w * 2 + e;
                                    uint32_t b0, b1;
                                    if constexpr (Shape::kSharedQuery) {
                                        const uint2 x = queries[(f * (BOTH ? 2 : 1) + half) * 32 + lane];
                                        b0 = x.x, b1 = x.y;
                                    } else {
                                        b0 = query[f][2 * half], b1 = query[f][2 * half + 1];
                                    }
                                    if (w + e + half == 0)
                                        mma_f16_first(dot[u][g][n], a, b0, b1);
                                    else
                                        mma_f16(dot[u][g][n], a, b0, b1);
                                }
                            }
                }
            // then cell by cell, while the products of the next one are under way
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // scores, whose differences `factor` takes to powers of two, and the values' steps and zeros
                Two score[NT][2];  // of position, of position + 8
                __half2 values[GROUPS][2];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const uint8_t* steps_of = held + u * Shape::kCell + g * 64 + quad / 2 * 16;
                    const uint4 raw = *reinterpret_cast<const uint4*>(steps_of + cell_key_steps(D));
                    const float2 sz0 = unpack_f16(__byte_perm(raw.x, raw.y, pick)), sz1 = unpack_f16(__byte_perm(raw.z, raw.w, pick));
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float2 sz = i ? sz1 : sz0;
                            if (LOW) sz.y = fmaf(8.f, sz.x, sz.y);  // s (n - 8) + (z + 8 s)
                            float (&d)[4] = dot[u][g][n];
                            if (HALF) {  // the high and low parts' columns lie four apart
                                d[2 * i] += __shfl_xor_sync(0xffffffffu, d[2 * i], 2);
                                d[2 * i + 1] += __shfl_xor_sync(0xffffffffu, d[2 * i + 1], 2);
                            }
                            const Two zero = g ? fma(Two(sz.y), plain(n, g), score[n][i]) : Two(sz.y) * plain(n, g);
                            score[n][i] = fma(Two(sz.x), Two(d[2 * i], d[2 * i + 1]), zero);
                        }
                    const uint4 more = *reinterpret_cast<const uint4*>(steps_of + cell_value_steps(D));
                    uint32_t sz[2] = {__byte_perm(more.x, more.y, pick), __byte_perm(more.z, more.w, pick)};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (EDGE && !there(u, i)) sz[i] = 0;  // what no row sees may hold anything
                        values[g][i] = *reinterpret_cast<__half2*>(&sz[i]);
                    }
                }
                // weights; `largest`: the most that a weight of 1 times a step and a unit may be here
                float weight[NT][4], most = 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i % 2 == 0) {
                            const Two against(-reference[n][0], -reference[n][1]);
                            ((score[n][i / 2] + against) * Two(factor[n][0], factor[n][1])).get(weight[n][i], weight[n][i + 1]);
                        }
                        weight[n][i] = exp2_approx(weight[n][i]);
                        if (EDGE && blind(u, i / 2, n, i % 2)) weight[n][i] = 0.f;
                        most = fmaxf(most, weight[n][i]);
                    }
                float largest = 0x1p-5f;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) largest = fmaxf(largest, most_unit[g] * __low2float(__hmax2(values[g][0], values[g][1])));
                if (__any_sync(0xffffffffu, !(most * largest < 0x1p15f))) {
                    // a row's largest weight so far becomes 1, and its products with the group's steps kRoom at most
                    float top[NT][2], keep[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            top[n][i] = -INFINITY;
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                float rows[2];
                                score[n][m].get(rows[0], rows[1]);
                                if (!EDGE || !blind(u, m, n, i)) top[n][i] = fmaxf(top[n][i], rows[i]);
                            }
                        }
#pragma unroll
                    for (int o = 4; o < 32; o *= 2)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 2; ++i) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], o));
                    __nv_bfloat162 here[NT][GROUPS];  // of both rows: units need no more than bf16 holds
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float next = fmaxf(reference[n][i], top[n][i]);
                            keep[n][i] = exp2_approx((reference[n][i] - next) * factor[n][i]);
                            reference[n][i] = next;
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                float rows[2], &w = weight[n][2 * m + i];
                                score[n][m].get(rows[0], rows[1]);
                                w = exp2_approx((rows[i] - next) * factor[n][i]);
                                if (EDGE && blind(u, m, n, i)) w = 0.f;
                            }
                        }
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g) {
                            const float s[2] = {__low2float(values[g][0]), __low2float(values[g][1])};
                            here[n][g] = __floats2bfloat162_rn(fmaxf(weight[n][0] * s[0], weight[n][2] * s[1]), fmaxf(weight[n][1] * s[0], weight[n][3] * s[1]));
                        }
                    }
#pragma unroll
                    for (int o = 4; o < 32; o *= 2)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int g = 0; g < GROUPS; ++g) here[n][g] = __hmax2(here[n][g], __shfl_xor_sync(0xffffffffu, here[n][g], o));
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) most_unit[g] = 0.f;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        sum[n] = sum[n] * Two(keep[n][0], keep[n][1]);
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g) {
                            const float2 product = __bfloat1622float2(here[n][g]);
                            float was[2], now[2], by[2];
                            both(unit[n][g]).get(was[0], was[1]);
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                now[i] = fminf(fminf(__fdividef(was[i], keep[n][i]), kMostUnit), __fdividef(kRoom, i ? product.y : product.x));
                            unit[n][g] = Units(now[0], now[1]);
                            both(unit[n][g]).get(now[0], now[1]);
                            if constexpr (kCentred) eighth[n][g] = Units(__fdividef(8.f, now[0]), __fdividef(8.f, now[1]));
                            most_unit[g] = fmaxf(most_unit[g], fmaxf(now[0], now[1]));
#pragma unroll
                            for (int i = 0; i < 2; ++i) by[i] = keep[n][i] * __fdividef(now[i], was[i]);
#pragma unroll
                            for (int m = 4 * g; m < 4 * g + 4; ++m)
#pragma unroll
                                for (int i = 0; i < 4; ++i) out[n][m][i] *= by[i % 2];
                            zeros[n][g] = zeros[n][g] * Two(keep[n][0], keep[n][1]);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) sum[n] = sum[n] + (Two(weight[n][0], weight[n][1]) + Two(weight[n][2], weight[n][3]));
                const uint8_t* cell = held + u * Shape::kCell;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    float2 sz[2] = {__half22float2(values[g][0]), __half22float2(values[g][1])};
                    if (LOW) sz[0].y = fmaf(8.f, sz[0].x, sz[0].y), sz[1].y = fmaf(8.f, sz[1].x, sz[1].y);
                    uint32_t p0[NT], p1[NT], l0[NT], l1[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t low[2];
                        const Two units = both(unit[n][g]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const Two w(weight[n][2 * i], weight[n][2 * i + 1]);
                            float x[2];
                            (w * units * Two(__low2float(values[g][i]))).get(x[0], x[1]);
                            if (EDGE) {  // a position that a row does not see adds nothing, whatever it holds
                                const bool skip[2] = {blind(u, i, n, 0), blind(u, i, n, 1)};
                                if (skip[0]) x[0] = 0.f;
                                if (skip[1]) x[1] = 0.f;
                                zeros[n][g] = fma(w, Two(skip[0] ? 0.f : sz[i].y, skip[1] ? 0.f : sz[i].y), zeros[n][g]);
                            } else {
                                zeros[n][g] = fma(w, Two(sz[i].y), zeros[n][g]);
                            }
                            uint32_t& high = i ? p1[n] : p0[n];
                            high = pack_f16(x[0], x[1]);
                            if constexpr (LOW || kCentred) {  // what the rounding leaves
                                const float2 as = unpack_f16(high);
                                if constexpr (LOW)
                                    low[i] = pack_f16(x[0] - as.x, x[1] - as.y);
                                else
                                    zeros[n][g] = fma(both(eighth[n][g]), Two(x[0], x[1]) + Two(-as.x, -as.y), zeros[n][g]);
                            }
                        }
                        if constexpr (BOTH) l0[n] = transpose_f16(low[0]), l1[n] = transpose_f16(low[1]);
                        if constexpr (HALF)
                            if (j >= 2) p0[n] = low[0], p1[n] = low[1];
                        p0[n] = transpose_f16(p0[n]);
                        p1[n] = transpose_f16(p1[n]);
                    }
                    const uint4 held_words = *reinterpret_cast<const uint4*>(cell + cell_values(D) + (g * 32 + lane) * 16);
                    const uint32_t word[4] = {held_words.x, held_words.y, held_words.z, held_words.w};
#pragma unroll
                    for (int half = 0; half < (BOTH ? 2 : 1); ++half)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t a[4] = {levels_f16<false, LOW>(word[w]), levels_f16<true, LOW>(word[w]),
                                                   levels_f16<false, LOW>(word[w] >> 8), levels_f16<true, LOW>(word[w] >> 8)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(out[n][g * 4 + w], a, half ? l0[n] : p0[n], half ? l1[n] : p1[n]);
                        }
                }
            }
        };

        // The tensor cores cut what they add to a sum, half a unit of its last place a time, so that long sums drift.
        // They are put aside in the workspace, a thread's own, and go on from 0; at the end (!away) they are added.
        constexpr int kPutAside = LOW ? 32 : 128;  // pairs: 2^-24 x 2 x 64, or 2^-24 x 256, of the sum
        const auto put_aside = [&](bool more, bool away) {  // more: something was put aside before
            float4* mine = call.aside + ((size_t)blockIdx.x * kAttentionWarps + warp) * (NT * (4 * GROUPS + 1) * 32) + lane;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float4* of = mine + t * (4 * GROUPS + 1) * 32;
                float keep[2] = {0.f, 0.f};
                if (more) {  // the references that it was taken against
                    const float4 against = of[4 * GROUPS * 32];
                    keep[0] = exp2_approx((against.x - reference[t][0]) * factor[t][0]), keep[1] = exp2_approx((against.y - reference[t][1]) * factor[t][1]);
                }
#pragma unroll
                for (int m = 0; m < 4 * GROUPS; ++m) {
                    float(&x)[4] = out[t][m];
                    float units[2];
                    both(unit[t][m / 4]).get(units[0], units[1]);
                    if (more) {
                        const float4 y = of[m * 32];
                        const float by[2] = {keep[0] * units[0], keep[1] * units[1]};
                        x[0] = fmaf(y.x, by[0], x[0]), x[1] = fmaf(y.y, by[1], x[1]);
                        x[2] = fmaf(y.z, by[0], x[2]), x[3] = fmaf(y.w, by[1], x[3]);
                    }
                    if (away) {
                        const float by[2] = {1.f / units[0], 1.f / units[1]};
                        of[m * 32] = make_float4(x[0] * by[0], x[1] * by[1], x[2] * by[0], x[3] * by[1]);
                        x[0] = x[1] = x[2] = x[3] = 0.f;
                    }
                }
                if (away) of[4 * GROUPS * 32] = make_float4(reference[t][0], reference[t][1], 0.f, 0.f);
            }
        };

#pragma unroll 1
        for (int n = 0; n < mine_pairs; ++n) {
            __syncwarp();
            issue();
            const int pair = first + warp + n * kAttentionWarps;
            const uint8_t* held = ring + stage * Shape::kStage;
            const uint32_t none = gone >> 2 * stage & 3;
            const bool late = dead || !mbar_wait_bounded(bars + stage, phase);
            if (++stage == kStages) stage = 0, phase ^= 1;
            if (__any_sync(0xffffffffu, late)) {
                dead = true;
                while (++n < issued) {  // what is in flight lands first
                    mbar_wait_bounded(bars + stage, phase);
                    if (++stage == kStages) stage = 0, phase ^= 1;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) sum[t] = Two(nan);
                break;
            }
            if (none || pair >= least >> 5) {  // some row does not see all of the pair's positions
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float gone_of[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int sees = min(limit[t][i], seen);  // a missing cell among what the row sees
                        gone_of[i] = (none & 1 && pair * kPairTokens < sees) || (none & 2 && pair * kPairTokens + kCellTokens < sees) ? nan : 0.f;
                    }
                    sum[t] = sum[t] + Two(gone_of[0], gone_of[1]);
                }
#pragma unroll 1
                for (int u = 0; u < 2; u += Shape::kAtOnce)
                    take(std::true_type{}, held + u * Shape::kCell, pair * kPairTokens + u * kCellTokens, none >> u);
            } else {
#pragma unroll 1
                for (int u = 0; u < 2; u += Shape::kAtOnce)
                    take(std::false_type{}, held + u * Shape::kCell, pair * kPairTokens + u * kCellTokens, 0);
            }
            if ((n + 1) % kPutAside == 0 || (n + 1 == mine_pairs && mine_pairs > kPutAside)) put_aside(n >= kPutAside, n + 1 < mine_pairs);
        }
        // rows that see positions which no table entry covers, or whose sequence has no table
#pragma unroll
        for (int t = 0; t < NT; ++t)
            sum[t] = sum[t] + Two(part.table < 0 || limit[t][0] > covered ? nan : 0.f, part.table < 0 || limit[t][1] > covered ? nan : 0.f);

        // ---- the warps' sums
        __syncthreads();  // the rings are drained
        float* mine_sums = warp_sums + warp * Shape::kRows * Shape::kPart;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float* row = mine_sums + (8 * t + (HALF ? (2 * j + i) % 4 : 2 * j + i)) * Shape::kPart;
                const bool mine = !HALF || j < 2;  // the others hold the same rows
                float sums[2], units[2];
                sum[t].get(sums[0], sums[1]);
                const float l = across_sum(sums[i]);
                if (quad == 0 && mine) row[D] = reference[t][i], row[D + 1] = l, row[D + 2] = factor[t][i];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    float of_rows[2];
                    both(unit[t][g]).get(units[0], units[1]);
                    const float by = 1.f / units[i];
                    zeros[t][g].get(of_rows[0], of_rows[1]);
                    const float z = across_sum(of_rows[i]);
#pragma unroll
                    for (int m = 4 * g; m < 4 * g + 4; ++m) {
                        float x = out[t][m][i], y = out[t][m][2 + i];
                        if (HALF) {
                            x += __shfl_xor_sync(0xffffffffu, x, 2);
                            y += __shfl_xor_sync(0xffffffffu, y, 2);
                        }
                        if (!mine) continue;
                        row[16 * m + quad] = fmaf(x, LOW ? by : by * 0x1p24f, z);
                        row[16 * m + 8 + quad] = fmaf(y, LOW ? by : by * 0x1p20f, z);
                    }
                }
            }
        __syncthreads();
        const bool whole = first == 0 && last == pairs;
        float* to_add = call.parts + ((size_t)blockIdx.x * 2 + (first == 0)) * call.used * Shape::kPart;
        for (int i = warp; i < (int)call.used; i += kAttentionWarps) {
            int token, h;
            if (!place(i, token, h)) continue;
            const float factor_of = warp_sums[i * Shape::kPart + D + 2];
            float top = kNoReference, l = 0.f, weight[kAttentionWarps];
#pragma unroll
            for (int w = 0; w < kAttentionWarps; ++w) top = fmaxf(top, warp_sums[(w * Shape::kRows + i) * Shape::kPart + D]);
#pragma unroll
            for (int w = 0; w < kAttentionWarps; ++w) {
                const float* row = warp_sums + (w * Shape::kRows + i) * Shape::kPart;
                weight[w] = exp2_approx((row[D] - top) * factor_of);
                l += weight[w] * row[D + 1];
            }
            const float inverse = l == 0.f ? 0.f : 1.f / l;
            T* to = static_cast<T*>(call.out) + (size_t)(part.row + token) * call.out_row +
                    (size_t)(head * (int)call.group + h) * call.out_head;
            for (int d = lane; d < D; d += 32) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < kAttentionWarps; ++w) x = fmaf(weight[w], warp_sums[(w * Shape::kRows + i) * Shape::kPart + d], x);
                if (whole)
                    to[d] = from_f32<T>(x * inverse);
                else
                    to_add[(size_t)i * Shape::kPart + d] = x;
            }
            if (!whole && lane == 0) *reinterpret_cast<float4*>(to_add + (size_t)i * Shape::kPart + D) = make_float4(top, l, factor_of, 0.f);
        }
        if (first == 0 && !whole && threadIdx.x == 0) {
            call.shares[blockIdx.x] = 1 + (int)((pairs - last + run - 1) / run);
            call.tails[blockIdx.x] = make_int4(part.row, head, sub, part.positions);
        }
        __syncthreads();  // the part and the sums are read
    }
}

// Adds up the parts of the tiles that a block of attention_kernel started and others
// finished, in a fixed order.  Each block lists those tiles (few blocks that read all marks
// start sooner than one for each block before them) and takes some, `most` rows at a time;
// its sixteen warps share the rows and their parts out.
constexpr int kMergeWarps = 16;

template <typename T, int GROUPS>
__global__ void __launch_bounds__(32 * kMergeWarps) attention_merge_kernel(AttentionCall call, int rows, int most, int blocks) {
    constexpr int D = 64 * GROUPS, kRow = part_row(D), kEach = D / 32, kAhead = 4;
    extern __shared__ int started[];  // [blocks] those that started a shared tile
    __shared__ int counts[kMergeWarps];
    __shared__ float2 about_warp[kMergeWarps];  // reference and sum of the weights
    __shared__ float factors[kMergeWarps];
    __shared__ float sums[kMergeWarps][D];
    const int warp = (int)threadIdx.x / 32, lane = (int)threadIdx.x % 32;
    pdl_launch_dependents();
    pdl_wait();
    int tiles = 0;
    for (int base = 0; base < blocks; base += 32 * kMergeWarps) {
        const int block = base + (int)threadIdx.x;
        const unsigned votes = __ballot_sync(0xffffffffu, block < blocks && call.shares[block] > 0);
        if (lane == 0) counts[warp] = __popc(votes);
        __syncthreads();
        int before = tiles;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) {
            if (w < warp) before += counts[w];
            tiles += counts[w];
        }
        if (votes >> lane & 1) started[before + __popc(votes & ((1u << lane) - 1))] = block;
        __syncthreads();
    }
    const int pieces = ((int)call.used + most - 1) / most;
    for (int item = (int)blockIdx.x; item < tiles * pieces; item += (int)gridDim.x) {
        const int block = started[item / pieces], first_row = item % pieces * most;
        const int count = call.shares[block], used = min((int)call.used - first_row, most), per_row = kMergeWarps / used;
        const int4 tail = call.tails[block];
        const int mine = warp / per_row, i = first_row + mine;
        // (the first part's; all have the same)
        const float factor = call.parts[((size_t)(block * 2 + 1) * call.used + min(i, (int)call.used - 1)) * kRow + D + 2];
        float top = kNoReference, l = 0.f, x[kEach] = {};
        for (int n = mine < used ? warp % per_row : count; n < count; n += kAhead * per_row) {  // all loads ahead of their use
            float2 about[kAhead];
            float row[kAhead][kEach];
#pragma unroll
            for (int m = 0; m < kAhead; ++m) {
                about[m] = make_float2(kNoReference, 0.f);
#pragma unroll
                for (int e = 0; e < kEach; ++e) row[m][e] = 0.f;
                const int from = n + m * per_row;
                if (from < count) {
                    const float* p = call.parts + (((size_t)(block + from) * 2 + (from == 0)) * call.used + i) * kRow;
                    about[m] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
                    for (int e = 0; e < kEach; ++e) row[m][e] = p[e * 32 + lane];
                }
            }
            const float now = fmaxf(top, fmaxf(fmaxf(about[0].x, about[1].x), fmaxf(about[2].x, about[3].x)));
            const float keep = exp2_approx((top - now) * factor);
            top = now;
            l *= keep;
#pragma unroll
            for (int e = 0; e < kEach; ++e) x[e] *= keep;
#pragma unroll
            for (int m = 0; m < kAhead; ++m) {
                const float weight = exp2_approx((about[m].x - now) * factor);
                l = fmaf(about[m].y, weight, l);
#pragma unroll
                for (int e = 0; e < kEach; ++e) x[e] = fmaf(row[m][e], weight, x[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) sums[warp][e * 32 + lane] = x[e];
        if (lane == 0) about_warp[warp] = make_float2(top, l), factors[warp] = factor;
        __syncthreads();
        for (int d = (int)threadIdx.x; d < used * D; d += 32 * kMergeWarps) {
            const int row = d / D, first = row * per_row, k = first_row + row;
            const int token = call.subs > 1 ? 0 : k / (int)call.group;
            const int h = call.subs > 1 ? tail.z * rows + k : k % (int)call.group;
            if (h >= (int)call.group || token >= tail.w) continue;
            top = kNoReference, l = 0.f;
            for (int w = first; w < first + per_row; ++w) top = fmaxf(top, about_warp[w].x);
            float y = 0.f;
            for (int w = first; w < first + per_row; ++w) {
                const float weight = exp2_approx((about_warp[w].x - top) * factors[first]);
                l = fmaf(about_warp[w].y, weight, l);
                y = fmaf(sums[w][d % D], weight, y);
            }
            T* to = static_cast<T*>(call.out) + (size_t)(tail.x + token) * call.out_row + (size_t)(tail.y * (int)call.group + h) * call.out_head;
            to[d % D] = from_f32<T>(l == 0.f ? 0.f : y / l);
        }
        __syncthreads();
    }
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

// How many entries of a row of the tables name pages, `held` of them at least: those of a sequence that was shortened
// go on behind its end.
__device__ __forceinline__ long long pages_in(const int32_t* row, uint32_t width, uint32_t page_count, long long held) {
    const auto none = [&](long long slot) { return slot >= width || (uint32_t)row[slot] >= page_count; };
    if (none(held)) return held;
    long long low = held, high = width;  // an entry that names one, and one that does not
    for (long long step = 1; high - low > 1; step *= 2) {  // at twice the distance while there are pages, then by halves
        const long long middle = min(low + step, (low + high) / 2);
        if (none(middle)) {
            high = middle;
            step = 1;
        } else {
            low = middle;
        }
    }
    return high;
}

// lsx_cache_reserve_device.  One block: entry i of the list is thread i's.
__global__ void __launch_bounds__(1024) reserve_kernel(int32_t* tables, uint32_t table_rows, uint32_t width,
                                                       int32_t* lengths, int32_t* refs, uint32_t page_count,
                                                       uint32_t page_size, const int32_t* sequences,
                                                       const int32_t* counts, uint32_t n, int32_t* missing) {
    __shared__ int list[kMaxListed];
    __shared__ long long starts[kMaxListed + 1], firsts[kMaxListed];
    __shared__ long long parts[32];
    const int i = (int)threadIdx.x;
    list[i] = i < (int)n ? sequences[i] : -1;
    __syncthreads();
    const int s = list[i];
    const bool valid = i < (int)n && (uint32_t)s < table_rows && !named_before(list, i);
    const long long before = valid ? max(lengths[s], 0) : 0, after = before + (valid ? max(counts[i], 0) : 0);
    const long long needed = (after + page_size - 1) / page_size;
    long long held = (before + page_size - 1) / page_size, beyond, total;
    if (valid) held = pages_in(tables + (size_t)s * width, width, page_count, held);
    block_prefix(max(needed - (long long)width, 0ll), parts, &beyond);
    starts[i] = block_prefix(max(needed - held, 0ll), parts, &total);
    firsts[i] = held;
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
        tables[(size_t)list[low] * width + firsts[low] + rank - starts[low]] = page;
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
                 (uint32_t)tables[(size_t)child * width] >= page_count && !named_before(list, i);
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
    for (long long base = 0; base < width; base += 256) {  // and those behind the end, which go on without a gap
        const long long w = base + threadIdx.x;
        const int page = w < width ? tables[(size_t)s * width + w] : -1;
        const bool some = (uint32_t)page < page_count;
        if (w < pages || some) {
            tables[(size_t)s * width + w] = -1;
            if (some) atomicSub(refs + page, 1);
        }
        if (!__syncthreads_or(base + 256 < pages || (some && threadIdx.x == 255))) break;
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
    LSX_ENSURE((uint64_t)rows->rows * view.kv_heads <= (uint64_t)1 << 31, "a call takes 2^31 rows of heads at most");
    LSX_ENSURE(rows->list || rows->sequences <= view.table_rows, "more sequences than the tables have rows");
    LSX_ENSURE(rows->starts || rows->rows == rows->sequences, "without starts each sequence has one row");
    *out = CacheRows{rows->list, rows->starts, (uint32_t)rows->sequences, (uint32_t)rows->rows};
    return LSX_OK;
}

bool known_kind(lsx_dtype kind) { return kind == LSX_F32 || kind == LSX_F16 || kind == LSX_BF16; }

// Rows of heads: `row` and `head` elements from one to the next, each head contiguous.
int check_heads(const void* data, lsx_dtype kind, size_t row, size_t head, const char* what) {
    LSX_ENSURE(data, "invalid argument");
    LSX_ENSURE(known_kind(kind), "unknown dtype");
    LSX_ENSURE(reinterpret_cast<uintptr_t>(data) % dtype_bytes(kind) == 0, std::string(what) + " not aligned to the type");
    LSX_ENSURE(row <= (size_t)1 << 40 && head <= (size_t)1 << 40, std::string(what) + ": check the strides");
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
    return launch_dependent(copy_pages_kernel, dim3(blocks), kCopyThreads, 0, s, (uint8_t*)pool.data, (uint32_t)pool.layers,
                            pool.layer_bytes, pool.page_bytes, (uint32_t)pool.page_count, pairs, (uint32_t)count, moved,
                            tables, tables_out, (uint64_t)entries, to_of);
}

// Whether cells are taken whole: where the call has many heads of rows, and a sequence has several on average.
// (Appended in bf16, 8 x 128, by rows and by cells: 100 in one sequence 2.9 and 8.4 us, 16 of 16 5.4 and 8.8, 128
// of 8 11.5 and 9.5, 5 of 2500 101 and 30; 128 of 4 7.4 and 15.1.)
bool by_cells(const CacheView& c, const CacheRows& r) {
    return (uint64_t)r.rows * c.kv_heads >= 8192 && r.rows >= 8 * (uint64_t)r.count;
}

unsigned cell_blocks(const CacheView& c, const CacheRows& r, unsigned units) {
    return (unsigned)(((uint64_t)(r.rows + kCellTokens - 1) / kCellTokens * c.kv_heads + units - 1) / units);
}

template <typename T>
cudaError_t launch_append(cudaStream_t s, const T* k, const T* v, size_t k_row, size_t k_head, size_t v_row, size_t v_head,
                          bool wide, const CacheView& c, const CacheRows& r) {
    const auto cells = [&](auto kernel, unsigned groups, unsigned units) {
        return launch_dependent(kernel, dim3(cell_blocks(c, r, units)), 32 * groups * units, 0, s, k, v, k_row, k_head, v_row, v_head,
                                wide, c, r);
    };
    if (!by_cells(c, r))
        return launch_dependent(append_rows_kernel<T>, dim3((unsigned)(((uint64_t)r.rows * c.kv_heads * 2 + 3) / 4)), 128, 0, s, k, v,
                                k_row, k_head, v_row, v_head, c, r);
    switch (c.dim / kCacheGroup) {
    case 1: return cells(append_cells_kernel<T, 1>, 1, kAppendUnits<1>);
    case 2: return cells(append_cells_kernel<T, 2>, 2, kAppendUnits<2>);
    case 3: return cells(append_cells_kernel<T, 3>, 3, kAppendUnits<3>);
    default: return cells(append_cells_kernel<T, 4>, 4, kAppendUnits<4>);
    }
}

template <typename T>
cudaError_t launch_read(cudaStream_t s, T* k, T* v, const CacheView& c, const CacheRows& r) {
    const auto cells = [&](auto kernel) {
        return launch_dependent(kernel, dim3(cell_blocks(c, r, kCellWarps)), 32 * kCellWarps, 0, s, c, r, k, v);
    };
    if (!by_cells(c, r))
        return launch_dependent(read_rows_kernel<T>, dim3((unsigned)(((uint64_t)r.rows * c.kv_heads * 2 + 3) / 4)), 128, 0, s, c, r, k, v);
    switch (c.dim / kCacheGroup) {
    case 1: return cells(read_cells_kernel<T, 1>);
    case 2: return cells(read_cells_kernel<T, 2>);
    case 3: return cells(read_cells_kernel<T, 3>);
    default: return cells(read_cells_kernel<T, 4>);
    }
}

// attention_kernel's workspace: two parts of a tile a block that the card holds, and what the block starts.
template <int GROUPS, int NT, bool LOW, bool HALF = false>
size_t attention_bytes(int sm_count) {
    using Shape = AttentionShape<GROUPS, NT, LOW, HALF>;
    return (size_t)sm_count * Shape::kBlocksPerSm * (20 + 2 * Shape::kRows * Shape::kPart * 4 + Shape::kAside * 16);
}

template <int GROUPS>
size_t attention_bytes(int sm_count) {
    return std::max({attention_bytes<GROUPS, 1, false>(sm_count), attention_bytes<GROUPS, 2, false>(sm_count),
                     attention_bytes<GROUPS, 1, true>(sm_count), attention_bytes<GROUPS, 2, true>(sm_count),
                     attention_bytes<GROUPS, 1, true, true>(sm_count)});
}

size_t attention_workspace(int sm_count, size_t dim) {
    switch (dim / kCacheGroup) {
    case 1: return attention_bytes<1>(sm_count);
    case 2: return attention_bytes<2>(sm_count);
    case 3: return attention_bytes<3>(sm_count);
    default: return attention_bytes<4>(sm_count);
    }
}

template <typename T, int GROUPS, int NT, bool HALF = false>
cudaError_t launch_tiles(int sm_count, cudaStream_t s, const CacheView& c, const CacheRows& r, AttentionCall call,
                         void* workspace) {
    constexpr bool kLow = std::is_same<T, float>::value;
    using Shape = AttentionShape<GROUPS, NT, kLow, HALF>;
    const auto kernel = attention_kernel<T, GROUPS, NT, kLow, HALF>;
    const unsigned blocks = (unsigned)(sm_count * Shape::kBlocksPerSm);
    call.tokens = 1;
    while (call.tokens * 2 * call.group <= (uint32_t)Shape::kRows) call.tokens *= 2;
    call.subs = (call.group + Shape::kRows - 1) / Shape::kRows;
    call.used = std::min<uint32_t>(Shape::kRows, call.tokens * call.group);
    // Where a row of the tables covers few positions nothing is gained by sharing a tile, and the second launch is
    // left out (one sequence of 9 positions: 8.3 us with it, 5.9 without).
    call.whole = (uint64_t)c.table_width * c.page_size <= kWholeTokens;
    call.tails = static_cast<int4*>(workspace);
    call.aside = reinterpret_cast<float4*>(call.tails + blocks);
    call.parts = reinterpret_cast<float*>(call.aside + (size_t)blocks * Shape::kAside);
    call.shares = reinterpret_cast<int*>(call.parts + (size_t)blocks * 2 * Shape::kRows * Shape::kPart);
    static std::atomic<uint64_t> allowed{0};  // devices that know the kernel's shared memory
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status == cudaSuccess && (device >= 64 || !(allowed.load(std::memory_order_acquire) >> device & 1))) {
        status = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kShared);
        if (status == cudaSuccess && device < 64) allowed.fetch_or(1ull << device, std::memory_order_release);
    }
    if (status != cudaSuccess) return status;
    status = launch_dependent(kernel, dim3(blocks), kAttentionThreads, Shape::kShared, s, c, r, call);
    if (status != cudaSuccess) return status;
    if (call.whole) return cudaSuccess;
    // rows that a block takes at a time: with few tiles each has many parts, for all warps of a block
    const uint64_t tiles = ((uint64_t)r.rows / call.tokens + r.count) * c.kv_heads * call.subs;  // at most
    const unsigned most = tiles * kMergeWarps <= blocks ? 1 : 4, pieces = (call.used + most - 1) / most;
    return launch_dependent(attention_merge_kernel<T, GROUPS>, dim3((unsigned)std::min<uint64_t>(tiles * pieces, 2 * (unsigned)sm_count)),
                            32 * kMergeWarps, blocks * 4, s, call, Shape::kRows, (int)most, (int)blocks);
}

// Rows of a tile by the rows that a sequence and key head has on average.  The time goes by the tiles' rows, used or
// not (12 sequences of 6001 positions, bf16, 8 x 128, 20 rows: 68 us in tiles of 16 and 112 of 64; parts of prompts 1089 us in
// tiles of 16, 1421 of 8), and a step of eight rows or fewer by what it reads.
template <typename T, int GROUPS>
cudaError_t launch_attention(int sm_count, cudaStream_t s, const CacheView& c, const CacheRows& r,
                             const AttentionCall& call, void* workspace) {
    const uint64_t rows = (uint64_t)((r.rows + r.count - 1) / r.count) * call.group;
    if (rows > 8) return launch_tiles<T, GROUPS, 2>(sm_count, s, c, r, call, workspace);
    if constexpr (std::is_same<T, float>::value)
        if (rows <= 4) return launch_tiles<T, GROUPS, 1, true>(sm_count, s, c, r, call, workspace);
    return launch_tiles<T, GROUPS, 1>(sm_count, s, c, r, call, workspace);
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
    LSX_TRY(check_heads(k, kind, k_row, k_head, "keys"));
    LSX_TRY(check_heads(v, kind, v_row, v_head, "values"));
    LSX_CACHE_SCOPE();
    const size_t e = dtype_bytes(kind);
    const bool wide = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                      (k_row | k_head | v_row | v_head) * e % 16 == 0;
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        LSX_CUDA(launch_append<T>(on, (const T*)k, (const T*)v, k_row, k_head, v_row, v_head, wide, c, r), "cache append");
        return (int)LSX_OK;
    });
}

int lsx_cache_read_device(lsx_ctx* ctx, const lsx_cache_view* view, const lsx_cache_rows* rows, lsx_dtype kind,
                          void* k_out, void* v_out, void* stream) {
    CacheView c;
    CacheRows r;
    LSX_TRY(check_view(view, &c));
    LSX_TRY(check_rows(rows, c, &r));
    LSX_TRY(check_heads(k_out, kind, 0, 0, "keys"));
    LSX_TRY(check_heads(v_out, kind, 0, 0, "values"));
    LSX_CACHE_SCOPE();
    LSX_ENSURE((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0, "outputs are not aligned to 16 bytes");
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        LSX_CUDA(launch_read<T>(on, (T*)k_out, (T*)v_out, c, r), "cache read");
        return (int)LSX_OK;
    });
}

size_t lsx_cache_attention_workspace_bytes(lsx_ctx* ctx, size_t head_dim) {
    return ctx ? attention_workspace(ctx->sm_count, head_dim) : 0;
}

int lsx_cache_attention_device(lsx_ctx* ctx, const lsx_cache_view* view, const lsx_cache_rows* rows, const void* q,
                               lsx_dtype kind, size_t q_heads, size_t q_row, size_t q_head, double scale, void* out,
                               size_t out_row, size_t out_head, void* workspace, size_t workspace_bytes, void* stream) {
    CacheView c;
    CacheRows r;
    LSX_TRY(check_view(view, &c));
    LSX_TRY(check_rows(rows, c, &r));
    LSX_ENSURE(q_heads > 0 && q_heads <= 65536 && q_heads % c.kv_heads == 0, "query heads are a multiple of key heads");
    LSX_TRY(check_heads(q, kind, q_row, q_head, "queries"));
    LSX_TRY(check_heads(out, kind, out_row, out_head, "output"));
    LSX_ENSURE(scale == scale && scale < 1e30 && scale > -1e30, "check the scale");
    LSX_CACHE_SCOPE();
    LSX_ENSURE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                   workspace_bytes >= attention_workspace(ctx->sm_count, c.dim),
               "workspace too small or not aligned to 16 bytes");
    AttentionCall call = {};
    call.q = q;
    call.out = out;
    call.q_row = q_row;
    call.q_head = q_head;
    call.out_row = out_row;
    call.out_head = out_head;
    call.group = (uint32_t)(q_heads / c.kv_heads);
    call.scale = (float)(scale * 1.4426950408889634);
    const size_t e = dtype_bytes(kind);
    call.wide = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_row * e % 16 == 0 && q_head * e % 16 == 0;
    return by_kind(kind, [&](auto type) {
        using T = decltype(type);
        cudaError_t status;
        switch (c.dim / kCacheGroup) {
        case 1: status = launch_attention<T, 1>(ctx->sm_count, on, c, r, call, workspace); break;
        case 2: status = launch_attention<T, 2>(ctx->sm_count, on, c, r, call, workspace); break;
        case 3: status = launch_attention<T, 3>(ctx->sm_count, on, c, r, call, workspace); break;
        default: status = launch_attention<T, 4>(ctx->sm_count, on, c, r, call, workspace); break;
        }
        LSX_CUDA(status, "cache attention");
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
    LSX_ENSURE(sequences && n > 0 && n <= (size_t)kMaxFreed, "name 1..=65536 sequences");
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
