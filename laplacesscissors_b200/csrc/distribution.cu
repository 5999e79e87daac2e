// Operators on rows of logits: log probabilities of given tokens with the entropy and
// the top alternatives, distillation from a teacher's top logits, and the gradients
// of both with respect to the logits.
//
// Per row z[0..V) at temperature T, with m = max z and s = ln sum_i exp((z_i - m) / T),
// the probabilities are q_i = exp((z_i - m) / T - s).  The sums are one pass over the row,
// a gradient is one more; HBM traffic bounds both where there is work enough, one
// exponential per element (16 per clock and SM) comes next, and few short rows cost the
// chain of their steps (load, sum, select, put together), about 5 us.
//
// Differences are formed before they are scaled: y = (z - r) * (log2 e / T) against a
// reference r that is itself one of the logits, so the lowest value of a type, -inf
// masks and logits far from zero all give the exponent their difference has.  Sums are
// f32 against the row's maximum, in an order that the sizes, the rows' alignment to 16 bytes
// and the number of SMs decide, so results repeat bit for bit for the same call; what small
// differences are made of (a list's mass, a loss) is f64.  A 16-bit gradient is rounded
// once, when it is stored.
//
// Measured on B200 (6552 GB/s measured copy, a pass among others): log probabilities with 8
// alternatives of 2048 x 151936 f32 191 us (99% of the copy's rate), with 20 of one row
// 9.8 us, with 50 of 777 x 50257 f16 33 us (36%: the rows of an SM select at the same
// time); their gradient, 2048 x 151936 bf16, 190 us (100%); a loss of 512 x 151936 f32 with 20
// listed tokens 58 us (82%); loss and gradient of 2048 x 151936 bf16 with 64 277 us (69%: most
// of a row is read twice); a gradient from saved statistics, 1000 x 50257 f16, 38 us (81%).
// These are short runs at 1965 MHz.  Seconds of the largest calls meet the card's 1 kW: the
// first of them takes 204 us at 1540 MHz, the fused step 311 at 1670.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <string>
#include <type_traits>

#include "device_common.cuh"
#include "distribution.cuh"
#include "lsx_internal.h"

namespace lsx {
namespace {

constexpr int kRowThreads = 256;     // 5 or 6 such blocks on an SM: 512 or 1024 threads overlap a row's steps less
constexpr int kPieceThreads = 128;   // of the gradient kernels
constexpr int kListCap = 2048;       // candidate keys of one selection
// Loss and gradient in one kernel take a slice twice.  From kStagedVectors on it passes
// through shared memory (Stage): kStagedBlocks blocks of kStagedThreads threads on an SM,
// kPlaces chunks of kChunk vectors a thread, 36 KB.  Of 2048 x 151936 bf16, 1000 x 50257 f16:
// 285 and 57 us so, 299 and 62 with 5 blocks of chunks of 2, 304 and 69 with 3 blocks of 384,
// 308 and 56 with 8 of 128.  100 x 32000 f32 (slices of 2000): 12.7 us staged, 16.1 not;
// shorter ones are alike.
// Rows are halved until a slice is at most kAgainVectors (two blocks for a row of 151936 bf16),
// so that what does not stay in shared memory can stay in L2: 2048 of these rows whole 306 us,
// halved 285, in quarters 356.  Slices are longer where a row would take more than kMaxCluster
// blocks, and where one halving less saves a second wave (launch_distill).
constexpr int kStagedThreads = 256;
constexpr int kStagedBlocks = 4;
constexpr int kPlaces = 3;
constexpr int kChunk = 3;
constexpr int kAgainVectors = 10000;
constexpr int kStagedVectors = 1024;
// Slices of the gradient kernels: 1200, 2048 and 3000 vectors measured 201, 190 and 196 us on
// 2048 x 151936 bf16.
constexpr int kPieceVectors = 2048;
// Rows shorter than this are distilled by blocks of 128 threads, which leaves more of them on
// an SM: 1084 x 396 f32 7.1 us against 12.3.
constexpr int kBriefVectors = 512;
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) below this are zero in f32 with room to spare; the bound keeps
// 0 * y finite for masked elements.
constexpr float kLowestExponent = -1e4f;
// A thread's reference is moved up once a logit lies this many powers of two above it.
constexpr float kSlack = 20.f;

// What only the temperature decides.
struct Scale {
    float L;        // log2 e / T
    float inverse;  // 1 / T
    float slack;    // kSlack powers of two as a difference of logits
    explicit Scale(double temperature)
        : L((float)(1.4426950408889634 / temperature)), inverse((float)(1.0 / temperature)), slack(kSlack / L) {}
    // (a - b) / T.  The lowest value of f32 or bf16 is further from large logits than f32 reaches,
    // which halves are not (exponents need no such care: theirs is 0 long before).
    __device__ __forceinline__ float between(float a, float b) const {
        return fmaf(0.5f, a, -0.5f * b) * (2.f * inverse);
    }
};

// ---- 16 bytes of logits ------------------------------------------------------
template <typename E>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void unpack(uint4 w, float* v) {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float top(uint4 w) {
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)),
                     fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
    static __device__ __forceinline__ float one(float x) { return x; }
    static __device__ __forceinline__ float store(float x) { return x; }
};
template <>
struct Vec<__half> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void unpack(uint4 w, float* v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ float top(uint4 w) {
        const __half2* h = reinterpret_cast<const __half2*>(&w);
        const __half2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(a), __high2float(a));
    }
    static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half store(float x) { return __float2half_rn(x); }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void unpack(uint4 w, float* v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    static __device__ __forceinline__ float top(uint4 w) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
        const __nv_bfloat162 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(a), __high2float(a));
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 store(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 w;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(p)
                 : "memory");
    return w;
}

__device__ __forceinline__ float exp2_fast(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}
// max(y, bound) that keeps a NaN.
__device__ __forceinline__ float max_nan(float y, float bound) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(y), "f"(bound));
    return r;
}

// ---- a row as 16-byte vectors ------------------------------------------------
// Rows may start at any element.  Vector j holds elements j * n - lead .. + n - 1;
// vectors [full0, full1) lie inside the row, at most one ragged vector stands at
// either end and is read element by element.
template <typename E>
struct Row {
    const E* base;  // 16-byte aligned address at or before the row
    int lead;       // elements between base and the row
    int vocab;
    int full0, full1;
    bool head, last;

    __device__ __forceinline__ Row(const E* row, int vocab_) : vocab(vocab_) {
        constexpr int n = Vec<E>::n;
        lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
        base = row - lead;
        head = lead != 0;
        full0 = head ? 1 : 0;
        const uint32_t reach = (uint32_t)lead + (uint32_t)vocab;
        const int end = (int)(reach / n);
        last = reach % n != 0 && end >= full0;
        full1 = end > full0 ? end : full0;
    }
    // the element that vector j starts with (rows have at most 2^30)
    __device__ __forceinline__ int first(int j) const { return j * Vec<E>::n - lead; }
    __device__ __forceinline__ uint4 full(int j) const { return load16(base + (long long)j * Vec<E>::n); }
    __device__ __forceinline__ void ragged(int j, float* v) const {
#pragma unroll
        for (int e = 0; e < Vec<E>::n; ++e) {
            const int i = first(j) + e;
            v[e] = i >= 0 && i < vocab ? Vec<E>::one(base[(long long)j * Vec<E>::n + e]) : -INFINITY;
        }
    }
};

// One block's share of a row that `parts` blocks divide.
struct Slice {
    int lo, hi;      // full vectors
    int begin, end;  // elements, the ragged ends included
    bool head, last;
    template <typename E>
    __device__ __forceinline__ Slice(const Row<E>& row, int part, int parts) {
        const uint32_t full = (uint32_t)(row.full1 - row.full0), step = (full + (uint32_t)parts - 1) / (uint32_t)parts;
        lo = row.full0 + (int)min((uint32_t)part * step, full);
        hi = row.full0 + (int)min((uint32_t)(part + 1) * step, full);
        head = row.head && part == 0;
        last = row.last && part == parts - 1;
        begin = part == 0 ? 0 : row.first(lo);
        end = part == parts - 1 ? row.vocab : row.first(hi);
    }
};

// ---- marked tokens -----------------------------------------------------------
// The tokens a row lists, and a bitmap over vector numbers (modulo its size) that tells the
// streaming loop which vectors hold one.  One word covers 32 consecutive vectors, which is
// what a warp holds.  Such vectors are put aside and summed without the listed elements
// once the row has streamed.
constexpr int kMarkWords = 512;
constexpr int kAside = 256;
struct Marks {
    alignas(16) uint32_t ids[kMaxSlots];  // kUnusedToken in unused slots
    uint32_t bits[kMarkWords];
    alignas(16) uint4 aside[kAside];
    int aside_at[kAside];
    short in_order[kAside];
    int asides;
};

__device__ __forceinline__ bool marked(const Marks& M, int j) {
    return (M.bits[((uint32_t)j >> 5) & (kMarkWords - 1)] >> (j & 31)) & 1u;
}

// Sets the listed elements of vector j to -inf.
template <typename E>
__device__ __forceinline__ void strike(const Marks& M, int count, const Row<E>& row, int j, float* v) {
    const uint32_t first = (uint32_t)row.first(j);
#pragma unroll 4
    for (int i = 0; i < count; i += 4) {
        const uint4 ids = *reinterpret_cast<const uint4*>(&M.ids[i]);
        const uint32_t at[4] = {ids.x - first, ids.y - first, ids.z - first, ids.w - first};
        // (an unused slot, -1, can only fall before a row's first element)
        if (min(min(at[0], at[1]), min(at[2], at[3])) >= (uint32_t)Vec<E>::n) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < Vec<E>::n; ++e) v[e] = at[q] == (uint32_t)e ? -INFINITY : v[e];
    }
}

// Whether an earlier slot names this slot's token; `ids` 16-byte aligned, kMaxSlots of them.
__device__ __forceinline__ bool named_before(const uint32_t* ids, int slot) {
    const uint32_t id = ids[slot];
    bool seen = false;
#pragma unroll 4
    for (int j = 0; j < slot; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(&ids[j]);
        seen |= o.x == id | (o.y == id & j + 1 < slot) | (o.z == id & j + 2 < slot) | (o.w == id & j + 3 < slot);
    }
    return seen;
}

// ---- running sums of a softmax ---------------------------------------------------
// Sums over several elements, against one of them.
struct Sums {
    float m, S, W;
    // The same sums against M >= m.
    __device__ __forceinline__ void rebase(float M, float L) {
        if (S == 0.f) return;
        const float shift = (m - M) * L;
        const float f = exp2_fast(shift);
        W = f == 0.f ? 0.f : f * fmaf(shift, S, W);
        S = f == 0.f && S == S ? 0.f : f * S;
    }
};

// S = sum 2^y and W = sum 2^y y over the elements seen (in two halves), y against the
// reference r; S == 0 exactly while only -inf has been seen.  m is the largest element,
// `at` the first vector that holds it and `second` the largest element of the others.
// Without kRanked only S and m.
template <bool kRanked>
struct Running {
    float r = 0.f, limit = -INFINITY, m = -INFINITY, second = -INFINITY;
    float2 S2 = {0.f, 0.f}, W2 = {0.f, 0.f};
    int at = -1;
    __device__ __forceinline__ void rise(float top, const Scale& k) {
        if (S2.x + S2.y != 0.f) {
            const float shift = (r - top) * k.L;
            const float f = exp2_fast(shift);
            const bool none = f == 0.f;
            if (kRanked) {
                W2.x = none ? 0.f : f * fmaf(shift, S2.x, W2.x);
                W2.y = none ? 0.f : f * fmaf(shift, S2.y, W2.y);
            }
            S2.x *= f;
            S2.y *= f;
        }
        r = top;
        limit = top + k.slack;
    }
    template <int n>
    __device__ __forceinline__ void add(const float* v, float top, int j, const Scale& k) {
        if (kRanked) {
            second = fmaxf(second, fminf(m, top));
            at = top > m ? j : at;
        }
        m = fmaxf(m, top);
        if (top > limit) rise(top, k);
        const float2 back = {-r, -r}, scale = {k.L, k.L};
#pragma unroll
        for (int e = 0; e < n; e += 2) {
            float2 y = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), back), scale);
            if (kRanked) {  // 0 * y stays 0
                y.x = max_nan(y.x, kLowestExponent);
                y.y = max_nan(y.y, kLowestExponent);
            }
            const float2 p = {exp2_fast(y.x), exp2_fast(y.y)};
            S2 = __fadd2_rn(S2, p);
            if (kRanked) W2 = __ffma2_rn(p, y, W2);
        }
    }
    __device__ __forceinline__ Sums sums() const { return {r, S2.x + S2.y, W2.x + W2.y}; }
};

// A warp's sums, each lane's against its own reference x.m; `top` is a lane's largest element.
__device__ __forceinline__ Sums warp_sums(Sums x, float top, float L) {
    float M = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    x.rebase(M, L);
    return {M, warp_allsum(x.S), warp_allsum(x.W)};
}

// The block's sums, in every thread.  `scratch` holds one entry per warp and is free
// again after the caller's next block barrier.
template <bool kRanked>
__device__ __forceinline__ Sums block_sums(const Running<kRanked>& a, float L, Sums* scratch) {
    Sums x = warp_sums(a.sums(), a.m, L);
    const int lane = threadIdx.x & 31;
    if (lane == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = lane < (int)(blockDim.x >> 5) ? scratch[lane] : Sums{-INFINITY, 0.f, 0.f};
    return warp_sums(x, x.m, L);
}

// `stage` is a Stage or nullptr; `begun` is called once, when the first loads are on their way.
template <typename E, bool kExclude, bool kRanked, typename S, typename F>
__device__ __forceinline__ void stream_slice(const Row<E>& row, const Slice& part, Marks* M, int count, const Scale& k,
                                             Running<kRanked>& acc, const S& stage, F&& begun) {
    constexpr int n = Vec<E>::n;
    constexpr bool kStaged = !std::is_same_v<S, std::nullptr_t>;
    auto add = [&](const float* v, int j) {
        float top = v[0];
#pragma unroll
        for (int e = 1; e < n; ++e) top = fmaxf(top, v[e]);
        acc.template add<n>(v, top, j, k);
    };
    auto take = [&](int j, uint4 w) {
        float v[n];
        if (kExclude && marked(*M, j)) {
            const int slot = atomicAdd(&M->asides, 1);
            if (slot < kAside) {
                M->aside[slot] = w;
                M->aside_at[slot] = j;
            }
            return;
        }
        Vec<E>::unpack(w, v);
        acc.template add<n>(v, Vec<E>::top(w), j, k);
    };
    auto take_ragged = [&](int j) {
        float v[n];
        row.ragged(j, v);
        if (kExclude) strike(*M, count, row, j, v);
        add(v, j);
    };
    const int tid = threadIdx.x, T = blockDim.x;
    if constexpr (kStaged) {
        stage.begin();
        begun();
        if (part.head && tid == 0) take_ragged(0);
        stage.read(take);
        if (part.last && tid == T - 1) take_ragged(row.full1);
        return;
    }
    int j = part.lo + tid;
    uint4 w[kUnroll];
    bool whole = j + (kUnroll - 1) * T < part.hi;
    if (whole) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = row.full(j + u * T);
    }
    begun();
    // every thread meets its vectors in ascending order
    if (part.head && tid == 0) {
        acc.at = 0;
        take_ragged(0);
    } else if (j < part.hi) {
        acc.at = j;
    } else if (part.last && tid == T - 1) {
        acc.at = row.full1;
    }
    while (whole) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) take(j + u * T, w[u]);
        j += kUnroll * T;
        whole = j + (kUnroll - 1) * T < part.hi;
        if (whole) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) w[u] = row.full(j + u * T);
        }
    }
    for (; j < part.hi; j += T) take(j, row.full(j));
    if (part.last && tid == T - 1) take_ragged(row.full1);
}

// ---- staged slices ----------------------------------------------------------------------
// Copies of 16 bytes into shared memory that the copying thread alone waits for.  `keep`
// marks what is read from global memory once more.
__device__ __forceinline__ void copy16(uint4* shared, const void* global, bool keep) {
    uint64_t kept, passing;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(kept));
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(passing));
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(shared)),
                 "l"(global), "l"(keep ? kept : passing)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until at most n of the thread's groups are under way.
template <int n>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

// A slice that is taken twice, in chunks of kChunk vectors a thread, each thread for itself.
// Three places in shared memory hold a chunk each: the first chunk stays in the first, the
// others pass through the second and third in turn, where the last two stay.  So three
// chunks are read from global memory once, the others twice.
template <typename E, int T>
struct Stage {
    uint4* places;
    const Row<E>& row;
    int first, hi, chunks;
    __device__ __forceinline__ Stage(uint4* shared, const Row<E>& row_, const Slice& part)
        : places(shared + threadIdx.x), row(row_), first(part.lo + (int)threadIdx.x), hi(part.hi) {
        chunks = first < hi ? (hi - first + T * kChunk - 1) / (T * kChunk) : 0;
    }
    __device__ __forceinline__ static int place(int chunk) { return chunk == 0 ? 0 : 1 + ((chunk - 1) & 1); }
    // Every chunk but a thread's last is whole and needs no bounds (2048 x 151936 bf16 277 us
    // against 285).
    template <typename F>
    __device__ __forceinline__ void vectors(int chunk, F&& f) const {
        const int j = first + chunk * kChunk * T;
        if (j + (kChunk - 1) * T < hi) {
#pragma unroll
            for (int u = 0; u < kChunk; ++u) f(j + u * T, u);
        } else if (chunk < chunks) {
#pragma unroll
            for (int u = 0; u < kChunk; ++u)
                if (j + u * T < hi) f(j + u * T, u);
        }
    }
    // one group of copies, empty past the last chunk
    __device__ __forceinline__ void start(int chunk, int at, bool keep) const {
        vectors(chunk, [&](int j, int u) {
            copy16(places + (at * kChunk + u) * T, row.base + (long long)j * Vec<E>::n, keep);
        });
        copies_commit();
    }
    template <typename F>
    __device__ __forceinline__ void each(int chunk, int at, F&& take) const {
        uint4 w[kChunk];
#pragma unroll
        for (int u = 0; u < kChunk; ++u) w[u] = places[(at * kChunk + u) * T];
        vectors(chunk, [&](int j, int u) { take(j, w[u]); });
    }
    __device__ __forceinline__ bool passes(int chunk) const { return chunk > 0 && chunk < chunks - 2; }
    __device__ __forceinline__ void begin() const {
        for (int c = 0; c < kPlaces; ++c) start(c, c, passes(c));
    }
    template <typename F>
    __device__ __forceinline__ void read(F&& take) const {
        for (int c = 0; c < chunks; ++c) {
            if (c == 0) {
                copies_wait<2>();
                each(0, 0, take);
            } else {
                copies_wait<1>();
                each(c, place(c), take);
                start(c + 2, place(c), passes(c + 2));
            }
        }
        copies_wait<0>();
    }
    template <typename F>
    __device__ __forceinline__ void read_again(F&& take) const {
        const int again = chunks - kPlaces;  // chunks 1 to `again` come from global memory
        if (again <= 0) {
            for (int c = 0; c < chunks; ++c) each(c, c, take);
            return;
        }
        const int second = place(chunks - 2), third = place(chunks - 1);
        auto next = [&](int chunk, int at) { start(chunk <= again ? chunk : chunks, at, false); };
        each(0, 0, take);
        next(1, 0);
        each(chunks - 2, second, take);
        next(2, second);
        each(chunks - 1, third, take);
        next(3, third);
        int turn = 0;
        for (int c = 1; c <= again; ++c) {
            copies_wait<2>();
            const int at = turn == 0 ? 0 : turn == 1 ? second : third;
            each(c, at, take);
            next(c + 3, at);
            turn = turn == 2 ? 0 : turn + 1;
        }
    }
};

// The vectors put aside, without their listed elements: thread t takes the one of t-th
// lowest number, whatever order they came in, so that sums repeat.  Where there are more
// than were kept (bitmap words shared by many vectors of a long row) every thread reads its
// own again.  After a block barrier.
template <typename E>
__device__ void add_asides(Marks& M, int count, const Row<E>& row, const Slice& part, const Scale& k,
                           Running<false>& acc) {
    constexpr int n = Vec<E>::n;
    const int tid = threadIdx.x, T = blockDim.x, asides = M.asides;
    auto take = [&](int j, uint4 w) {
        float v[n];
        Vec<E>::unpack(w, v);
        strike(M, count, row, j, v);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < n; ++e) top = fmaxf(top, v[e]);
        acc.template add<n>(v, top, 0, k);
    };
    if (asides > kAside) {
        for (int j = part.lo + tid; j < part.hi; j += T)
            if (marked(M, j)) take(j, row.full(j));
        return;
    }
    for (int i = tid; i < asides; i += T) {
        int rank = 0;
        for (int o = 0; o < asides; ++o) rank += M.aside_at[o] < M.aside_at[i];
        M.in_order[rank] = (short)i;
    }
    __syncthreads();
    for (int i = tid; i < asides; i += T) take(M.aside_at[M.in_order[i]], M.aside[M.in_order[i]]);
}

// Where one token holds nearly all the mass, 1 + rest in f32 keeps little of the rest, and
// ln(1 + rest) and the entropy are all rest.  For such sums one warp adds up the vectors of
// the thread that met the maximum once more, leaving the maximum out; the other threads'
// sums hold nothing of it.
constexpr float kPeaked = 1.0625f;

template <typename E>
__device__ Sums sum_without_maximum(const Row<E>& row, const Slice& part, int owner, float m, float L) {
    constexpr int n = Vec<E>::n;
    float s = 0.f, w = 0.f;
    auto take = [&](const float* v) {
#pragma unroll
        for (int e = 0; e < n; ++e) {
            if (v[e] == m) continue;
            const float y = max_nan((v[e] - m) * L, kLowestExponent);
            const float p = exp2_fast(y);
            s += p;
            w = fmaf(p, y, w);
        }
    };
    const int lane = threadIdx.x & 31, T = blockDim.x;
    float v[n];
    for (int j = part.lo + owner + lane * T; j < part.hi; j += 32 * T) {
        Vec<E>::unpack(row.full(j), v);
        take(v);
    }
    if (lane == 0 && part.head && owner == 0) {
        row.ragged(0, v);
        take(v);
    }
    if (lane == 0 && part.last && owner == T - 1) {
        row.ragged(row.full1, v);
        take(v);
    }
    return {m, warp_allsum(s), warp_allsum(w)};
}

// A block's share of a row's sums as the blocks of a cluster exchange it: the largest
// element counted as 1 and the rest apart.
struct Partial {
    float m, rest, W;
    int any;  // 0: nothing but -inf
};

template <typename E>
__device__ Partial slice_sums(const Row<E>& row, const Slice& part, const Running<true>& acc, const Scale& k,
                              Sums* scratch, int* owner) {
    const Sums x = block_sums(acc, k.L, scratch);
    Partial p{x.m, x.S - 1.f, x.W, x.S != 0.f};
    if (x.S != 0.f && x.S < kPeaked) {  // the maximum is unique
        if (acc.m == x.m) *owner = threadIdx.x;
        __syncthreads();
        Running<true> others = acc;
        if ((int)threadIdx.x == *owner) {
            others = Running<true>();
            others.m = x.m;
        }
        if (threadIdx.x < 32) {
            const Sums again = sum_without_maximum(row, part, *owner, x.m, k.L);
            scratch[32] = again;
        }
        const Sums rest = block_sums(others, k.L, scratch);
        __syncthreads();
        p.rest = rest.S + scratch[32].S;
        p.W = rest.W + scratch[32].W;
    }
    return p;
}

// The row's sums from its blocks' shares, a share to a lane; by whole warps.
__device__ __forceinline__ Partial combine(const Partial* shares, int count, float L) {
    const int lane = threadIdx.x & 31;
    const Partial mine = lane < count ? shares[lane] : Partial{-INFINITY, -1.f, 0.f, 0};
    float m = mine.any ? mine.m : -INFINITY;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    // the first share that holds the maximum counts it as 1
    const uint32_t holders = __ballot_sync(0xffffffffu, mine.any && mine.m == m);
    const bool holder = lane == __ffs(holders) - 1;
    Sums x{m, 0.f, 0.f};
    if (mine.any && !holder) {
        x = {mine.m, 1.f + mine.rest, mine.W};
        x.rebase(m, L);
    } else if (holder) {
        x = {m, mine.rest, mine.W};
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        x.S += __shfl_xor_sync(0xffffffffu, x.S, o);
        x.W += __shfl_xor_sync(0xffffffffu, x.W, o);
    }
    return {m, __shfl_sync(0xffffffffu, x.S, 0), __shfl_sync(0xffffffffu, x.W, 0),
            __any_sync(0xffffffffu, mine.any)};
}

// ---- thread-block clusters --------------------------------------------------------------
__device__ __forceinline__ int cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return (int)n;
}
__device__ __forceinline__ int cluster_rank() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
    return (int)n;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// `local`, a shared-memory address of this block, in block `rank` of the cluster.
template <typename V>
__device__ __forceinline__ V* in_block(V* local, int rank) {
    uint64_t p;
    asm("mapa.u64 %0, %1, %2;" : "=l"(p) : "l"(reinterpret_cast<uint64_t>(local)), "r"(rank));
    return reinterpret_cast<V*>(p);
}

// ---- top alternatives --------------------------------------------------------------
// One 64-bit key orders (logit descending, id ascending): NaN above every number,
// -0 equal to 0.
__device__ __forceinline__ unsigned long long order_key(float z, uint32_t id) {
    const uint32_t v = z != z ? 0xffffffffu : total_order_key(z + 0.f);
    return ((unsigned long long)v << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t key_id(unsigned long long k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ float key_logit(unsigned long long k) { return total_order_value((uint32_t)(k >> 32)); }

constexpr int kFewerCap = 512;
constexpr int kMaxCluster = 8;     // the portable size

struct Selection {
    alignas(16) unsigned long long keys[kListCap];
    alignas(16) unsigned long long fewer[kFewerCap];
    alignas(16) unsigned long long group[kRowThreads / 4];
    unsigned long long best[kMaxSlots];
    unsigned long long bound;
    uint32_t most, least;
    int count;
};

// A bound for the `top`-th largest of the keys that the threads hold, one each (0 for none;
// the others distinct): at least `top` keys reach it.  0 where there are fewer.  Resets
// P.count.  Ends with the block synchronised.
//
// Few of many are bounded by the `top`-th largest of the largest keys of groups of four
// threads, which share the comparisons of their group's key (one row of 151936, 20
// alternatives: 9.8 us against 10.7 by bisection).
__device__ unsigned long long group_bound(Selection& P, unsigned long long mine, int top) {
    const int tid = threadIdx.x, groups = blockDim.x >> 2;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
        mine = other > mine ? other : mine;
    }
    if ((tid & 3) == 0) P.group[tid >> 2] = mine;
    if (tid == 0) {
        P.bound = 0ull;
        P.count = 0;
    }
    __syncthreads();
    int above = 0;
#pragma unroll 4
    for (int i = 2 * (tid & 3); i < groups; i += 8) {
        const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(&P.group[i]);
        above += (pair.x > mine) + (pair.y > mine);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (above == top - 1 && mine != 0ull) P.bound = mine;
    __syncthreads();
    return P.bound;
}

// More, and few of few (`holders` threads have a key), are bounded by bisection: the largest
// value found that `top` keys reach.  It ends once hardly more than `top` reach it, which
// takes about eight counts; keys that differ in their low bits only (ties) take more, never
// more than 64 (29 rows of 5036, 93 alternatives: 11.5 us against 16.7 by groups).
__device__ unsigned long long key_bound(Selection& P, unsigned long long mine, int top, int holders) {
    if (top * 10 <= holders) return group_bound(P, mine, top);
    const uint32_t high = (uint32_t)(mine >> 32);
    const uint32_t most = __reduce_max_sync(0xffffffffu, high);
    const uint32_t least = __reduce_min_sync(0xffffffffu, mine ? high : ~0u);
    if (threadIdx.x == 0) {
        P.most = 0u;
        P.least = ~0u;
        P.count = 0;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        atomicMax(&P.most, most);
        atomicMin(&P.least, least);
    }
    if (__syncthreads_count(mine != 0ull) < top) return 0ull;
    // at least `top` keys reach lo, fewer than `top` reach hi
    unsigned long long lo = (unsigned long long)P.least << 32;
    unsigned long long hi = ((unsigned long long)P.most << 32 | 0xffffffffull) + 1ull;
    if (hi == 0ull) hi = ~0ull;  // (keys of NaN; 2^64 - 1 itself is token 0's, never short of the bound)
    const int enough = top + top / 4 + 4;
    while (hi - lo > 1ull) {
        const unsigned long long mid = lo + ((hi - lo) >> 1);
        const int reach = __syncthreads_count(mine >= mid);
        if (reach < top) {
            hi = mid;
        } else {
            lo = mid;
            if (reach <= enough) break;
        }
    }
    return lo;
}

// The `top` largest of keys[0..n) (distinct) in descending order into P.best; `keys` has
// room for one more.  Four threads share the comparisons of a key.  Starts and ends with
// the block synchronised.
__device__ void rank_all(Selection& P, unsigned long long* keys, int n, int top) {
    if (threadIdx.x == 0 && (n & 1)) keys[n] = 0ull;
    __syncthreads();
    const int part = threadIdx.x & 3;
    for (int base = 0; base < n; base += blockDim.x >> 2) {
        const int i = base + (threadIdx.x >> 2);
        const unsigned long long key = i < n ? keys[i] : 0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = 2 * part; j < n; j += 8) {
            const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(&keys[j]);
            rank += (pair.x > key) + (pair.y > key);
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (part == 0 && i < n && rank < top) P.best[rank] = key;
    }
    __syncthreads();
}

// rank_all for any n: a long list (ties of a masked row, rows in order) is first cut to the
// keys above a bound, since ranking takes n^2 comparisons.
__device__ void rank_keys(Selection& P, unsigned long long* keys, int n, int top) {
    if (n <= kFewerCap / 2) {
        rank_all(P, keys, n, top);
        return;
    }
    __syncthreads();
    unsigned long long mine = 0ull;
    for (int i = threadIdx.x; i < n; i += blockDim.x) mine = keys[i] > mine ? keys[i] : mine;
    const unsigned long long bound = key_bound(P, mine, top, n < (int)blockDim.x ? n : (int)blockDim.x);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const unsigned long long key = keys[i];
        if (key < bound) continue;
        const int pos = atomicAdd(&P.count, 1);
        if (pos < kFewerCap) P.fewer[pos] = key;
    }
    __syncthreads();
    const int count = P.count;
    if (count < kFewerCap)
        rank_all(P, P.fewer, count, top);
    else
        rank_all(P, keys, n, top);
}

// The `top` largest of `parts` descending lists of `top` keys each.  Every list's
// ceil(top / parts)-th key is at or above the smallest of these, so `top` keys are, and the
// others cannot be among them.
__device__ void rank_lists(Selection& P, const unsigned long long* lists, int parts, int top) {
    const int each = (top + parts - 1) / parts;
    if (threadIdx.x == 0) P.count = 0;
    unsigned long long bound = lists[each - 1];
    for (int i = 1; i < parts; ++i) {
        const unsigned long long key = lists[i * top + each - 1];
        bound = key < bound ? key : bound;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < parts * top; i += blockDim.x) {
        const unsigned long long key = lists[i];
        if (key >= bound) P.keys[atomicAdd(&P.count, 1)] = key;
    }
    __syncthreads();
    rank_keys(P, P.keys, P.count, top);
}

// The `top` best tokens of elements [begin, end) of a row, piece by piece: what beats the
// worst kept key joins the list, which is then cut to its best `top`.  Exact for any row.
template <typename E>
__device__ void select_by_pieces(Selection& P, const E* z, int begin, int end, int top, int cap) {
    int have = 0;
    const int piece = cap - kMaxSlots - 1;
    __syncthreads();
    for (int start = begin; start < end; start += piece) {
        if (threadIdx.x == 0) P.count = have;
        __syncthreads();
        const unsigned long long worst = have == top ? P.keys[top - 1] : 0ull;
        const int stop = end - start < piece ? end : start + piece;
        for (int i = start + threadIdx.x; i < stop; i += blockDim.x) {
            const unsigned long long key = order_key(Vec<E>::one(z[i]), (uint32_t)i);
            if (key > worst) P.keys[atomicAdd(&P.count, 1)] = key;
        }
        __syncthreads();
        const int n = P.count;
        if (n > have) {
            rank_keys(P, P.keys, n, top);
            have = n < top ? n : top;
            for (int i = threadIdx.x; i < have; i += blockDim.x) P.keys[i] = P.best[i];
        }
        __syncthreads();
    }
}

// Slices that are ranked whole: the shortest ones, and short ones with hardly a vector for
// each alternative.
template <typename E>
__device__ __forceinline__ bool ranked_whole(const Slice& part, int top) {
    const int tokens = part.end - part.begin;
    return tokens <= 96 || (tokens <= 256 && top * 4 > (part.hi - part.lo) * 3);
}

// The best tokens of a slice from what the threads met while they summed it.  A thread's
// key is its best vector, ordered by (largest logit, lower vector number first); a bound
// that `top` of these keys reach lies below the `top`-th best element.  So only elements at
// or above it are candidates, about T ln(1 / (1 - top / T)) of them where the tokens lie at
// random over T threads.  They are read again (from L2) at the threads' best vectors, and
// in all their vectors only for threads that have a second one to offer.  More candidates
// than the list holds are left to select_by_pieces.
template <typename E>
__device__ void select_by_threads(Selection& P, const Row<E>& row, const Slice& part, const E* z, int top,
                                  const Running<true>& acc, int cap) {
    constexpr int n = Vec<E>::n;
    const int tid = threadIdx.x, lane = tid & 31, T = blockDim.x;
    const unsigned long long mine =
        acc.at < 0 ? 0ull : ((unsigned long long)total_order_key(acc.m + 0.f) << 32) | (0xffffffffu - (uint32_t)acc.at);
    const int vectors = part.hi - part.lo;
    const unsigned long long bound = key_bound(P, mine, top, vectors < T ? vectors : T);
    const uint32_t level = (uint32_t)(bound >> 32);
    const uint32_t bound_at = 0xffffffffu - (uint32_t)bound;  // (a bisected bound may lie past the last vector)
    // the bound's logit; without a bound everything passes
    const float level_logit = bound ? total_order_value(level) : -INFINITY;
    auto offer_vector = [&](int j) {
        float v[n];
        if (j >= row.full0 && j < row.full1) {
            const uint4 w = row.full(j);
            if (Vec<E>::top(w) < level_logit) return;
            Vec<E>::unpack(w, v);
        } else {
            row.ragged(j, v);
        }
#pragma unroll
        for (int e = 0; e < n; ++e) {
            if (v[e] < level_logit) continue;
            const int i = row.first(j) + e;
            const bool tie = bound && total_order_key(v[e] + 0.f) == level;
            if ((!tie || (uint32_t)j <= bound_at) && i >= 0 && i < row.vocab) {
                const int pos = atomicAdd(&P.count, 1);
                if (pos < cap) P.keys[pos] = order_key(v[e], (uint32_t)i);
            }
        }
    };
    const bool in = mine != 0ull && mine >= bound;
    // a second vector counts where its largest logit beats the bound's, or equals it at a
    // vector number up to the bound's
    const uint32_t second = total_order_key(acc.second + 0.f);
    const bool more = vectors - tid + (part.head && tid == 0) + (part.last && tid == T - 1) > 1;
    uint32_t again = __ballot_sync(0xffffffffu, in && more && second >= level);
    if (in) offer_vector(acc.at);
    // lanes for the vectors of one such thread, and as many threads at a time as that leaves
    int per = 32;
    while (per > 1 && (per >> 1) * T >= vectors) per >>= 1;
    while (again) {
        const int which = lane / per;
        uint32_t rest = again;
        for (int i = 0; i < which && rest; ++i) rest &= rest - 1;
        const int from = rest ? __ffs(rest) - 1 : 0, who = (tid & ~31) + from;
        const int skip = __shfl_sync(0xffffffffu, acc.at, from);
        const bool tie = __shfl_sync(0xffffffffu, second, from) == level;
        if (rest) {
            const int end = bound && tie && bound_at < (uint32_t)part.hi ? (int)bound_at + 1 : part.hi;
            for (int j = part.lo + who + (lane & (per - 1)) * T; j < end; j += per * T)
                if (j != skip) offer_vector(j);
            if ((lane & (per - 1)) == 0 && part.head && who == 0 && skip != 0) offer_vector(0);
            if ((lane & (per - 1)) == 0 && part.last && who == T - 1 && skip != row.full1) offer_vector(row.full1);
        }
        __syncwarp();
        for (int i = 0; i < 32 / per && again; ++i) again &= again - 1;
    }
    __syncthreads();
    const int count = P.count;
    if (count >= cap)
        select_by_pieces<E>(P, z, part.begin, part.end, top, cap);
    else
        rank_keys(P, P.keys, count, top);
}

// ---- token_logprobs ------------------------------------------------------------------
// One cluster of blocks per row (one block where there are rows enough): the blocks sum
// and rank their slices and send sums and best keys to the first one's shared memory,
// which puts them together and writes the row's results.  Its 22.6 KB of shared memory leave
// nine blocks of 128 threads on an SM (a bound of ten only took registers: 3000 x 4000 f16 with
// 20 alternatives 29.4 us, 26.6 so; 3000 x 500 bf16 with 100 76.9 and 77.4).
template <typename E, int T>
__global__ void __launch_bounds__(T, T <= 128 ? 9 : T <= 192 ? 7 : T <= 224 ? 6 : 5) token_logprobs_kernel(
    const E* __restrict__ logits, int vocab, size_t stride, const Scale k, const uint32_t* __restrict__ tokens,
    int token_count, int top, LogprobOutputs out) {
    __shared__ Sums scratch[33];
    __shared__ Partial shares[kMaxCluster];
    __shared__ Selection selection;
    __shared__ int owner;
    const int parts = cluster_size(), part = cluster_rank();
    if (parts > 1) cluster_arrive();  // waited for before the first store into another block
    const size_t r = blockIdx.x / (uint32_t)parts;
    const E* z = logits + r * stride;
    // the given token's logit is on its way while the row streams
    uint32_t token = kUnusedToken;
    float given = 0.f;
    const bool asked = part == 0 && out.logprob && (int)threadIdx.x < token_count;
    if (asked) {
        token = tokens[r * token_count + threadIdx.x];
        if (token < (uint32_t)vocab) given = Vec<E>::one(z[token]);
    }
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    Running<true> acc;
    stream_slice<E, false>(row, slice, nullptr, 0, k, acc, nullptr, []() {});
    Partial sums = slice_sums(row, slice, acc, k, scratch, &owner);
    // clusters keep the upper half of the list for the blocks' best keys
    const int cap = parts > 1 ? kListCap / 2 : kListCap;
    if (top > 0) {
        if (ranked_whole<E>(slice, top)) {
            for (int i = threadIdx.x; i < slice.end - slice.begin; i += T)
                selection.keys[i] = order_key(Vec<E>::one(z[slice.begin + i]), (uint32_t)(slice.begin + i));
            rank_all(selection, selection.keys, slice.end - slice.begin, top);
        } else if (!sums.any) {  // nothing but -inf: the lowest ids
            for (int i = threadIdx.x; i < top; i += T) selection.best[i] = order_key(-INFINITY, slice.begin + i);
            __syncthreads();
        } else if (sums.rest == sums.rest)
            select_by_threads<E>(selection, row, slice, z, top, acc, cap);
        else  // NaN or +inf here: NaN leads the order and the threads' maxima pass over it
            select_by_pieces<E>(selection, z, slice.begin, slice.end, top, cap);
    }
    if (parts > 1) {
        cluster_wait();
        if (threadIdx.x == 0) *in_block(&shares[part], 0) = sums;
        for (int i = threadIdx.x; i < top; i += T)
            *in_block(&selection.keys[kListCap / 2 + part * top + i], 0) = selection.best[i];
        cluster_arrive();
        cluster_wait();
        if (part != 0) return;
        sums = combine(shares, parts, k.L);
        if (top > 0) rank_lists(selection, selection.keys + kListCap / 2, parts, top);
    }
    const bool empty = !sums.any;  // every logit is -inf
    const float m = sums.m, log_sum = empty ? 0.f : log1pf(sums.rest);
    auto logprob = [&](float x) { return empty ? -INFINITY : k.between(x, m) - log_sum; };
    if (threadIdx.x == 0) {
        if (out.entropy) out.entropy[r] = empty ? 0.f : log_sum - sums.W / (1.f + sums.rest) * kLn2;
        if (out.stats) {
            out.stats[2 * r] = m;
            out.stats[2 * r + 1] = log_sum;
        }
    }
    if (asked)
        out.logprob[r * token_count + threadIdx.x] =
            token == kUnusedToken ? 0.f : token < (uint32_t)vocab ? logprob(given) : NAN;
    for (int i = threadIdx.x; i < top; i += T) {
        const float x = key_logit(selection.best[i]);
        if (out.top_ids) out.top_ids[r * top + i] = key_id(selection.best[i]);
        if (out.top_logits) out.top_logits[r * top + i] = x;
        if (out.top_logprobs) out.top_logprobs[r * top + i] = logprob(x);
    }
}

// ---- gradients ---------------------------------------------------------------------------
// What the unlisted elements of a row's gradient need: with y = (z - m) L - offset an
// element gets 2^y (a + b y).  Listed ones are written over them afterwards.
struct Dense {
    float m, offset, a, b;
};
// The gradient of a row without any token: 0 for every element (z - 0 = -inf).
__device__ __forceinline__ Dense dense_zero() { return {0.f, 0.f, 0.f, 0.f}; }

template <int n, bool kLinear>
__device__ __forceinline__ void dense_vector(float* v, const Dense& d, float L) {
    const float2 back = {-d.m, -d.m}, scale = {L, L}, offset = {-d.offset, -d.offset}, a = {d.a, d.a}, b = {d.b, d.b};
#pragma unroll
    for (int e = 0; e < n; e += 2) {
        float2 y = __ffma2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), back), scale, offset);
        if (kLinear) {  // 0 * y stays 0
            y.x = max_nan(y.x, kLowestExponent);
            y.y = max_nan(y.y, kLowestExponent);
        }
        const float2 p = {exp2_fast(y.x), exp2_fast(y.y)};
        const float2 g = __fmul2_rn(p, kLinear ? __ffma2_rn(b, y, a) : a);
        v[e] = g.x;
        v[e + 1] = g.y;
    }
}

__device__ __forceinline__ void store16(void* p, uint4 w) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                 : "memory");
}

// The dense gradient of a slice into `out` (the row's first element) by T threads.  `out`
// may be the row.  An `out` of another alignment to 16 bytes than the row is stored element by
// element (1000 x 50257 f16: 137 us instead of 38).  `ready` gives the coefficients, once, after the first loads are on their
// way.  `stage` is the one that stream_slice read through, or nullptr.
template <typename E, bool kLinear, typename S, typename F>
__device__ __forceinline__ void write_dense(const Row<E>& row, const Slice& part, E* out, float L, int tid, int T,
                                            const S& stage, F&& ready) {
    constexpr int n = Vec<E>::n;
    // the output row may lie at another alignment than the logits
    const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == (uintptr_t)(row.lead * sizeof(E));
    E* base = out - row.lead;
    Dense d;
    auto put = [&](int j, uint4 w) {
        float v[n];
        Vec<E>::unpack(w, v);
        dense_vector<n, kLinear>(v, d, L);
        if (same) {
            store16(base + (long long)j * n, Vec<E>::pack(v));
        } else {
#pragma unroll
            for (int e = 0; e < n; ++e) base[(long long)j * n + e] = Vec<E>::store(v[e]);
        }
    };
    auto put_ragged = [&](int j) {
        float v[n];
        row.ragged(j, v);
        dense_vector<n, kLinear>(v, d, L);
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const int i = row.first(j) + e;
            if (i >= 0 && i < row.vocab) out[i] = Vec<E>::store(v[e]);
        }
    };
    if constexpr (!std::is_same_v<S, std::nullptr_t>) {
        d = ready();
        stage.read_again(put);
        if (part.head && tid == 0) put_ragged(0);
        if (part.last && tid == T - 1) put_ragged(row.full1);
        return;
    }
    int j = part.lo + tid;
    uint4 w[kUnroll];
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (from + u * T < part.hi) w[u] = row.full(from + u * T);
    };
    fetch(j);
    d = ready();
    while (j < part.hi) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (j + u * T < part.hi) put(j + u * T, w[u]);
        j += kUnroll * T;
        fetch(j);
    }
    if (part.head && tid == 0) put_ragged(0);
    if (part.last && tid == T - 1) put_ragged(row.full1);
}

// `parts` blocks share a row; none waits for another.
template <typename E>
__global__ void __launch_bounds__(kPieceThreads, 1024 / kPieceThreads) logprobs_gradient_kernel(
    const E* logits, int vocab, size_t stride, const Scale k, int parts, const uint32_t* __restrict__ tokens,
    int token_count, const float* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ logprob_gradient, const float* __restrict__ entropy_gradient, E* gradient,
    size_t gradient_stride) {
    __shared__ uint32_t ids[kMaxSlots];
    __shared__ float given[kMaxSlots];
    const size_t r = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts), tid = threadIdx.x;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    const float m = stats[2 * r], log_sum = stats[2 * r + 1];
    const float h = entropy_gradient ? entropy_gradient[r] : 0.f, H = entropy ? entropy[r] : 0.f;
    // a slot to a thread; the listed logits are read before anything is written
    uint32_t id = kUnusedToken;
    float logit = 0.f;
    if (tid < token_count) {
        id = tokens[r * token_count + tid];
        ids[tid] = id;
        // NaN for a token outside the vocabulary goes through the sum into the whole row
        given[tid] = id == kUnusedToken ? 0.f : id < (uint32_t)vocab ? logprob_gradient[r * token_count + tid] : NAN;
        if (id < (uint32_t)vocab && (int)id >= slice.begin && (int)id < slice.end) logit = Vec<E>::one(z[id]);
    }
    const bool empty = m == -INFINITY && log_sum == 0.f;
    float total = 0.f;
    Dense d;
    auto ready = [&]() {
        __syncthreads();
        for (int i = 0; i < token_count; ++i) total += given[i];
        d = dense_zero();
        if (!empty) {
            d.m = m;
            d.offset = log_sum * kLog2E;
            d.b = -h * kLn2 * k.inverse;
            d.a = -(total + (h != 0.f ? h * H : 0.f)) * k.inverse;
        } else if (total != total) {
            d.a = NAN;
        }
        return d;
    };
    E* out = gradient + r * gradient_stride;
    if (h != 0.f)
        write_dense<E, true>(row, slice, out, k.L, tid, kPieceThreads, nullptr, ready);
    else
        write_dense<E, false>(row, slice, out, k.L, tid, kPieceThreads, nullptr, ready);
    __syncthreads();
    if (id >= (uint32_t)vocab || (int)id < slice.begin || (int)id >= slice.end) return;
    // a token named several times adds up at its first slot
    float own = 0.f;
    for (int i = 0; i < token_count; ++i) {
        if (ids[i] != id) continue;
        if (i < tid) return;
        own += given[i];
    }
    const float y = max_nan(fmaf(logit - d.m, k.L, -d.offset), kLowestExponent), log_q = y * kLn2;
    // own (1 - q) apart from the other tokens' share: own - q own loses a confident token's gradient
    const float g = -expm1f(log_q) * own - exp2_fast(y) * (total - own + (h != 0.f ? h * (H + log_q) : 0.f));
    out[id] = Vec<E>::store(empty ? total * 0.f : g * k.inverse);
}

// ---- distillation --------------------------------------------------------------------------
// The listed tokens' side of a row is summed in 64 bits, a slot to a thread: at most
// kMaxSlots numbers, of which 1 - sum p is next to 0 for a confident teacher.
constexpr int kListWarps = kMaxSlots / 32;

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// max, NaN passed over
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ln p of a slot up to the list's normalisation: against the teacher's statistics where
// they are given, else against `top`, the list's largest logit.  -inf for an unused slot and
// for a teacher's row without tokens, which asks for nothing.
__device__ __forceinline__ double teacher_log(float value, const float* saved, float top, double inverse) {
    if (value == -INFINITY) return -INFINITY;
    if (!saved) return ((double)value - (double)top) * inverse;
    return saved[0] == -INFINITY && saved[1] == 0.f ? -INFINITY
                                                    : ((double)value - (double)saved[0]) * inverse - (double)saved[1];
}

// The teacher's mass outside its list, from the list's (0 without statistics).
__device__ __forceinline__ double teacher_rest(double mass, const float* saved) {
    if (!saved || (saved[0] == -INFINITY && saved[1] == 0.f)) return 0.0;
    return mass < 1.0 ? 1.0 - mass : (mass >= 1.0 ? 0.0 : mass);
}

// The tokens outside the list are one outcome where the student's share q_r of them is more
// than 0 in 64 bits (2^-1074 and up): below that they are masked, with -inf or a type's lowest
// value.  Neither the loss nor the gradient needs q_r itself: ln q_r is a difference of
// logarithms and q_i / q_r an exponential of one, both in range however small q_r is.
constexpr float kSmallestLogShare = -744.44007f;

// What a row's gradient needs beside its list: listed elements get q a - value, q against
// `offset`; the others are exponentiated against their own sum: 2^y = q_i / q_r stays in
// range and (P q_r - p_r) is the whole coefficient, however small q_r is.
struct DistillRow {
    Dense dense;
    float m, offset, a;
    bool empty;
};
__device__ __forceinline__ DistillRow distill_row(float m, float log_sum, float log_rest, float mass, float rest,
                                                  bool empty, bool bad, float scale) {
    const float log_share = log_rest - log_sum;
    const bool tail = log_share >= kSmallestLogShare;
    if (tail) mass = (float)((double)mass + (double)rest);
    if (bad) mass = NAN;
    DistillRow g;
    g.m = m;
    g.offset = log_sum * kLog2E;
    g.a = scale * mass;
    g.empty = empty;
    g.dense = dense_zero();
    if (bad) g.dense.a = NAN;
    if (!empty) {
        g.dense.m = m;
        g.dense.offset = tail ? log_rest * kLog2E : g.offset;
        g.dense.a = scale * (tail ? fmaf(mass, expf(log_share), -rest) : mass);
    }
    return g;
}
// The gradient at a listed token with the student's logit and the teacher's w p / T.
__device__ __forceinline__ float listed_gradient(const DistillRow& g, float logit, float value, float L) {
    const float y = max_nan(fmaf(logit - g.m, L, -g.offset), kLowestExponent);
    return g.empty ? 0.f * g.a : fmaf(exp2_fast(y), g.a, -value);
}

// Loss and statistics of rows that stream through registers, without their listed
// elements, which have their own sums; with kGradient the row is then read again for its
// gradient.  A cluster of blocks shares a row: they exchange their sums (with kGradient
// each takes the list for itself, else the first one).
//
// With the gradient a slice is taken twice, and the rows in flight outlive L2 in part only.
// 2048 x 151936 bf16 with 64 listed tokens: 333 us with plain loads both times, 298 through
// shared memory, 285 with L2 told which chunks return, 277 with bounds for the last chunk only.
// Whole rows in shared memory, by clusters of 8, move in lockstep: 315 us.  Passes over
// groups of rows that fit L2 (16 to 100 MB): 438 to 719 us, each pair of launches adds its
// ramps.
template <typename E, bool kTail, bool kGradient, int T, bool kStaged>
__global__ void __launch_bounds__(T, kStaged ? kStagedBlocks : 6 * kRowThreads / T) distill_kernel(
    const E* logits, int vocab, size_t stride, const Scale k, double inverse, TeacherRows teacher,
    const float* __restrict__ weights, float* loss, float* stats, E* gradient, size_t gradient_stride) {
    __shared__ Sums scratch[33];
    __shared__ Sums shares[kMaxCluster];
    __shared__ Marks marks;
    __shared__ float tops[kListWarps], highs[kListWarps];
    __shared__ double masses[kListWarps], insides[kListWarps], crosses[kListWarps];
    __shared__ int bad;
    extern __shared__ uint4 places[];
    const int parts = cluster_size(), part = cluster_rank(), tid = threadIdx.x;
    if (parts > 1) cluster_arrive();  // waited for before the first store into another block
    const size_t r = blockIdx.x / (uint32_t)parts;
    const int count = (int)teacher.slots;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    const auto stage = [&]() {
        if constexpr (kStaged)
            return Stage<E, T>(places, row, slice);
        else
            return nullptr;
    }();
    const float* saved = kTail ? teacher.stats + 2 * r : nullptr;
    const bool lists = kGradient || part == 0;
    uint32_t id = kUnusedToken;
    float value = -INFINITY, logit = -INFINITY;
    if (tid < count) {
        id = teacher.ids[r * count + tid];
        if (lists) value = teacher.logits[r * count + tid];
    }
    bool kept = false;
    Running<false> acc;
    stream_slice<E, true>(row, slice, &marks, count, k, acc, stage, [&]() {
        for (int i = tid; i < kMarkWords; i += T) marks.bits[i] = 0;
        if (tid == 0) marks.asides = bad = 0;
        if (tid < kMaxSlots) marks.ids[tid] = id < (uint32_t)vocab ? id : kUnusedToken;
        __syncthreads();
        if (id != kUnusedToken && id >= (uint32_t)vocab) bad = 1;
        kept = id < (uint32_t)vocab && !named_before(marks.ids, tid);
        if (kept) {
            const uint32_t j = (id + (uint32_t)row.lead) / Vec<E>::n;
            atomicOr(&marks.bits[(j >> 5) & (kMarkWords - 1)], 1u << (j & 31));
            if (lists) logit = Vec<E>::one(z[id]);
        } else {
            value = -INFINITY;
        }
        __syncthreads();
    });
    if (lists && tid < kMaxSlots) {
        const float top = warp_max(value), high = warp_max(logit);
        if ((tid & 31) == 0) {
            tops[tid >> 5] = top;
            highs[tid >> 5] = high;
        }
    }
    __syncthreads();
    add_asides(marks, count, row, slice, k, acc);
    float top = -INFINITY, high = -INFINITY;
    double p = 0.0;
    if (lists) {
#pragma unroll
        for (int w = 0; w < kListWarps; ++w) {
            top = fmaxf(top, tops[w]);
            high = fmaxf(high, highs[w]);
        }
        if (tid < kMaxSlots) {
            const double log_p = teacher_log(value, saved, top, inverse);
            p = log_p == -INFINITY ? 0.0 : exp(log_p);
            const double log_q = logit == -INFINITY ? -INFINITY : ((double)logit - (double)high) * inverse;
            const double mass = warp_sum_f64(p);
            const double inside = warp_sum_f64(log_q == -INFINITY ? 0.0 : exp(log_q));
            const double cross = part == 0 ? warp_sum_f64(p != 0.0 ? p * (log_p - log_q) : 0.0) : 0.0;
            if ((tid & 31) == 0) {
                masses[tid >> 5] = mass;
                insides[tid >> 5] = inside;
                crosses[tid >> 5] = cross;
            }
        }
    }
    Sums rest = block_sums(acc, k.L, scratch);
    if (parts > 1) {
        cluster_wait();
        if (tid < (kGradient ? parts : 1)) *in_block(&shares[part], tid) = rest;
        cluster_arrive();
    }
    // the row from its blocks' sums and its list's, in every thread that asks
    double mass = 0.0, p_rest = 0.0;
    float m = 0.f, log_sum = 0.f, log_rest = -INFINITY;
    bool empty = false;
    auto put_together = [&]() {
        if (parts > 1) {
            rest = shares[0];
            for (int i = 1; i < parts; ++i) rest.m = fmaxf(rest.m, shares[i].m);
            rest.S = 0.f;
            for (int i = 0; i < parts; ++i) {
                Sums x = shares[i];
                x.rebase(rest.m, k.L);
                rest.S += x.S;
            }
        }
        double inside = 0.0;
#pragma unroll
        for (int w = 0; w < kListWarps; ++w) {
            mass += masses[w];
            inside += insides[w];
        }
        p_rest = teacher_rest(mass, saved);
        // both shares around the larger maximum; sum - 1 apart, since ln(sum) may be all of it
        m = fmaxf(rest.m, high);
        const bool some = rest.S != 0.f, listed = inside != 0.0;
        empty = !some && !listed;
        const float below = some ? k.between(rest.m, m) : -INFINITY;
        const float outside = some ? rest.S * expf(below) : 0.f;
        const float over = high == m ? (float)(inside - 1.0) + outside
                                     : (listed ? (float)inside * expf((high - m) * k.inverse) : 0.f) + (outside - 1.f);
        log_sum = empty ? 0.f : log1pf(over);
        // (without a listed token that the student holds both sums are one: q_r is 1, and exactly)
        if (kTail && some) log_rest = listed ? logf(rest.S) + below : log_sum;
    };
    // By the first warp.  The loss may be a small difference of logarithms: they are taken
    // in 64 bits, one to a lane, so that the row waits for one of each function.
    auto write_row = [&]() {
        double inside = 0.0, cross = 0.0;
#pragma unroll
        for (int w = 0; w < kListWarps; ++w) {
            inside += insides[w];
            cross += crosses[w];
        }
        const bool some = rest.S != 0.f;
        const double down = some ? ((double)rest.m - (double)m) * inverse : -INFINITY;
        const double up = inside == 0.0 ? -INFINITY : ((double)high - (double)m) * inverse;
        const double factor = exp(tid == 0 ? down : up);
        const double outside = some ? (double)rest.S * __shfl_sync(0xffffffffu, factor, 0) : 0.0;
        const double listed = inside == 0.0 ? 0.0 : inside * __shfl_sync(0xffffffffu, factor, 1);
        const double log_of = log(tid == 0 ? listed + outside : tid == 1 ? mass : tid == 2 ? p_rest : (double)rest.S);
        const double log_all = empty ? 0.0 : __shfl_sync(0xffffffffu, log_of, 0);
        const double log_mass = __shfl_sync(0xffffffffu, log_of, 1), log_p = __shfl_sync(0xffffffffu, log_of, 2);
        const double log_S = __shfl_sync(0xffffffffu, log_of, 3);
        if (tid != 0) return;
        double x = mass;
        if (!kTail && x != 0.0) {  // normalised over the list
            cross = cross / x - log_mass;
            x = x == x ? 1.0 : x;
        }
        double value = x == 0.0            ? 0.0
                       : cross == INFINITY ? INFINITY
                                           : cross + x * (((double)m - (double)high) * inverse + log_all);
        if (kTail && p_rest > 0.0 && log_rest - log_sum >= kSmallestLogShare)
            value += p_rest * (log_p - log_S - down + log_all);
        if (loss) loss[r] = bad || x != x || log_sum != log_sum ? NAN : (float)value;
        if (stats) {
            stats[3 * r] = m;
            stats[3 * r + 1] = log_sum;
            stats[3 * r + 2] = log_rest;
        }
    };
    if (!kGradient) {
        if (parts > 1) cluster_wait();
        if (part != 0 || tid >= 32) return;
        put_together();
        write_row();
        return;
    }
    const double weight = weights ? (double)weights[r] * inverse : inverse;
    DistillRow g;
    E* out = gradient + r * gradient_stride;
    write_dense<E, false>(row, slice, out, k.L, tid, T, stage, [&]() {
        if (parts > 1) cluster_wait();
        put_together();
        const float P = kTail ? (float)mass : mass == 0.0 ? 0.f : mass == mass ? 1.f : NAN;
        g = distill_row(m, log_sum, log_rest, P, (float)p_rest, empty, bad, (float)weight);
        return g.dense;
    });
    __syncthreads();
    if (kept && (int)id >= slice.begin && (int)id < slice.end) {
        const double share = kTail || mass == 0.0 ? weight : weight / mass;
        out[id] = Vec<E>::store(listed_gradient(g, logit, (float)(share * p), k.L));
    }
    if (part == 0 && tid < 32) write_row();
}

// The gradient from saved statistics; `parts` blocks share a row, none waits for another.
// Without the teacher's statistics P is 1 and the unlisted elements do not wait for the
// list's sums.
template <typename E, bool kTail>
__global__ void __launch_bounds__(kPieceThreads, 1024 / kPieceThreads) distill_gradient_kernel(
    const E* logits, int vocab, size_t stride, const Scale k, double inverse, int parts, TeacherRows teacher,
    const float* __restrict__ stats, const float* __restrict__ weights, E* gradient, size_t gradient_stride) {
    static_assert(kPieceThreads == kMaxSlots, "a slot to a thread");
    __shared__ __align__(16) uint32_t ids[kMaxSlots];
    __shared__ double sums[kListWarps];
    __shared__ float tops[kListWarps];
    const size_t r = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts), count = (int)teacher.slots, tid = threadIdx.x;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    const float* saved = kTail ? teacher.stats + 2 * r : nullptr;
    const float weight = weights[r], scale = weight * k.inverse;
    // a slot to a thread; the listed logits are read before anything is written
    uint32_t id = kUnusedToken;
    float value = -INFINITY, logit = -INFINITY;
    if (tid < count) {
        id = teacher.ids[r * count + tid];
        value = teacher.logits[r * count + tid];
    }
    const bool here = id < (uint32_t)vocab && (int)id >= slice.begin && (int)id < slice.end;
    if (here) logit = Vec<E>::one(z[id]);
    double p = 0.0;
    bool kept = false;
    DistillRow g;
    auto list_mass = [&]() {  // in every thread
        const double part_sum = warp_sum_f64(p);
        if ((tid & 31) == 0) sums[tid >> 5] = part_sum;
        __syncthreads();
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < kListWarps; ++w) all += sums[w];
        return all;
    };
    E* out = gradient + r * gradient_stride;
    write_dense<E, false>(row, slice, out, k.L, tid, kPieceThreads, nullptr, [&]() {
        ids[tid] = id < (uint32_t)vocab ? id : kUnusedToken;
        const bool bad = __syncthreads_or(id != kUnusedToken && id >= (uint32_t)vocab) != 0;
        kept = id < (uint32_t)vocab && !named_before(ids, tid);
        if (!kept) value = -INFINITY;
        float top = 0.f, mass, rest = 0.f;
        if (!kTail) {
            top = warp_max(value != value ? INFINITY : value);
            if ((tid & 31) == 0) tops[tid >> 5] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kListWarps; ++w) top = fmaxf(top, tops[w]);
            mass = top == -INFINITY ? 0.f : top == INFINITY ? NAN : 1.f;
        }
        const double log_p = teacher_log(value, saved, top, inverse);
        p = log_p == -INFINITY ? 0.0 : exp(log_p);
        if (kTail) {
            const double all = list_mass();
            rest = (float)teacher_rest(all, saved);
            mass = (float)all;
        }
        const float m = stats[3 * r], log_sum = stats[3 * r + 1], log_rest = kTail ? stats[3 * r + 2] : -INFINITY;
        g = distill_row(m, log_sum, log_rest, mass, rest, m == -INFINITY && log_sum == 0.f, bad, scale);
        return g.dense;
    });
    double share = (double)weight * inverse;
    if (!kTail) {
        const double all = list_mass();
        if (all != 0.0) share /= all;
    }
    __syncthreads();
    if (kept && here) out[id] = Vec<E>::store(listed_gradient(g, logit, (float)(share * p), k.L));
}

template <typename F>
cudaError_t by_kind(lsx_dtype kind, F&& f) {
    switch (kind) {
    case LSX_F32: return f((const float*)nullptr);
    case LSX_F16: return f((const __half*)nullptr);
    default: return f((const __nv_bfloat16*)nullptr);
    }
}

// How many blocks share a row: as many as leave `resident` blocks to an SM, while each keeps
// `least` vectors.  4 measured best where nothing is read twice (512 x 151936 f32, 20 listed
// tokens: 58 us at 4, 70 at 8, 66 at 16).
int row_parts(int sm_count, size_t rows, size_t vectors, int least, int resident) {
    int parts = 1;
    while (parts < kMaxCluster && rows * parts * 2 <= (size_t)sm_count * resident &&
           vectors / (parts * 2) >= (size_t)least)
        parts *= 2;
    return parts;
}

template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kernel)(Params...), size_t rows, int parts, int threads, size_t shared,
                            cudaStream_t s, Args... args) {
    if (rows * parts > 2147483647ull) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * parts));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Blocks that share a row in the kernels whose blocks do not wait for one another: slices
// of about kPieceVectors, more where there are few rows.
int row_pieces(int sm_count, size_t rows, size_t vectors) {
    size_t parts = vectors / kPieceVectors + 1;
    while (rows * parts * 2 <= (size_t)sm_count * 8 && vectors / (parts * 2) >= (size_t)kPieceThreads) parts *= 2;
    return (int)parts;
}

}  // namespace

cudaError_t launch_token_logprobs(cudaStream_t s, int sm_count, const LogitRows& z, const uint32_t* tokens,
                                  size_t token_count, size_t alternatives, const LogprobOutputs& out) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        const size_t vectors = z.vocab / Vec<E>::n;
        const Scale k(z.temperature);
        auto launch = [&](auto threads, int parts) {
            constexpr int T = decltype(threads)::value;
            return launch_clusters(token_logprobs_kernel<E, T>, z.rows, parts, T, 0, s, (const E*)z.data, (int)z.vocab,
                                   z.stride, k, tokens, (int)token_count, (int)alternatives, out);
        };
        // few alternatives of a short row: smaller blocks leave more rows on an SM (750 x 253 f32
        // with 8: 7.6 us against 12.1)
        if (vectors < 1024 && (alternatives <= 24 || vectors <= 128))
            return launch(std::integral_constant<int, 128>(), 1);
        // Rows that just miss being resident all at once get narrower blocks instead of a second
        // wave (780 x 128256 f32 with 20 alternatives 74 us in blocks of 224, 89 of 256; 1000 x
        // 32000 bf16 with 8 22 us in blocks of 192, 25 of 256).  With more waves the widest are
        // the fastest (2048 x 151936 f32 with 8: 191 us of 256, 205 of 224).
        const size_t blocks = z.rows, sms = (size_t)sm_count;
        if (blocks > sms * 5 && blocks <= sms * 6) return launch(std::integral_constant<int, 224>(), 1);
        if (blocks > sms * 6 && blocks <= sms * 7) return launch(std::integral_constant<int, 192>(), 1);
        // A row is shared in slices of 1024 vectors or more, and from 4096 on: under that the
        // cluster's exchange costs more than the shorter slice saves (a row of 32000 bf16 with 20
        // alternatives 8.5 us whole, 10.1 halved; 64 rows of 8000 f32 7.9 whole, 9.7 in eighths; a
        // row of 16384 f32 4.1 in quarters, 4.7 halved).
        const int parts = vectors < 4096 ? 1 : row_parts(sm_count, z.rows, vectors, 1024, 4);
        return launch(std::integral_constant<int, 256>(), parts);
    });
}

cudaError_t launch_logprobs_gradient(cudaStream_t s, int sm_count, const LogitRows& z, const uint32_t* tokens,
                                     size_t token_count, const float* stats, const float* entropy,
                                     const float* logprob_gradient, const float* entropy_gradient, void* gradient,
                                     size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        const int parts = row_pieces(sm_count, z.rows, z.vocab / Vec<E>::n);
        if (z.rows * parts > 2147483647ull) return cudaErrorInvalidConfiguration;
        logprobs_gradient_kernel<E><<<(unsigned)(z.rows * parts), kPieceThreads, 0, s>>>(
            (const E*)z.data, (int)z.vocab, z.stride, Scale(z.temperature), parts, tokens, (int)token_count, stats,
            entropy, logprob_gradient, entropy_gradient, (E*)gradient, gradient_stride);
        return cudaGetLastError();
    });
}

cudaError_t launch_distill(cudaStream_t s, int sm_count, const LogitRows& z, const TeacherRows& teacher,
                           const float* weights, float* loss, float* stats, void* gradient, size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        const size_t vectors = z.vocab / Vec<E>::n;
        // With the gradient 3 blocks an SM are faster than 4, and slices of 256 no faster than of
        // 1024 (148 x 151936 bf16 32 us against 40; 60 x 50257 f16 14 us against 16).
        int parts = gradient ? row_parts(sm_count, z.rows, vectors, 1024, 3)
                             : row_parts(sm_count, z.rows, vectors, kRowThreads, 4);
        if (gradient && vectors / parts > (size_t)kAgainVectors) {
            while (parts < kMaxCluster && vectors / parts > (size_t)kAgainVectors) parts *= 2;
            // hardly more blocks than the SMs hold would leave them a second wave for a few (400 x
            // 151936 bf16: 73 us halved, 67 whole; 500 rows of them 80 halved, 86 whole)
            const size_t blocks = z.rows * parts, held = (size_t)sm_count * kStagedBlocks;
            if (blocks > held && blocks * 2 <= held * 3) parts /= 2;
        }
        auto pick = [&](auto threads) {
            constexpr int T = decltype(threads)::value;
            if (gradient)
                return teacher.stats ? distill_kernel<E, true, true, T, false> : distill_kernel<E, false, true, T, false>;
            return teacher.stats ? distill_kernel<E, true, false, T, false> : distill_kernel<E, false, false, T, false>;
        };
        const bool brief = vectors < (size_t)kBriefVectors;
        const bool staged = gradient && vectors / parts >= (size_t)kStagedVectors;
        auto kernel =
            brief ? pick(std::integral_constant<int, 128>()) : pick(std::integral_constant<int, kRowThreads>());
        if (staged)
            kernel = teacher.stats ? distill_kernel<E, true, true, kStagedThreads, true>
                                   : distill_kernel<E, false, true, kStagedThreads, true>;
        const int threads = staged ? kStagedThreads : brief ? 128 : kRowThreads;
        const size_t shared = staged ? (size_t)kPlaces * kChunk * kStagedThreads * sizeof(uint4) : 0;
        return launch_clusters(kernel, z.rows, parts, threads, shared, s, (const E*)z.data, (int)z.vocab, z.stride,
                               Scale(z.temperature), 1.0 / z.temperature, teacher, weights, loss, stats, (E*)gradient,
                               gradient_stride);
    });
}

cudaError_t launch_distill_gradient(cudaStream_t s, int sm_count, const LogitRows& z, const TeacherRows& teacher,
                                    const float* stats, const float* weights, void* gradient, size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        const int parts = row_pieces(sm_count, z.rows, z.vocab / Vec<E>::n);
        if (z.rows * parts > 2147483647ull) return cudaErrorInvalidConfiguration;
        auto kernel = teacher.stats ? distill_gradient_kernel<E, true> : distill_gradient_kernel<E, false>;
        kernel<<<(unsigned)(z.rows * parts), kPieceThreads, 0, s>>>(
            (const E*)z.data, (int)z.vocab, z.stride, Scale(z.temperature), 1.0 / z.temperature, parts, teacher, stats,
            weights, (E*)gradient, gradient_stride);
        return cudaGetLastError();
    });
}

// The checks every entry shares.
int check_rows(const LogitRows& z) {
    LSX_ENSURE(z.data, "invalid argument");
    LSX_ENSURE(z.kind == LSX_F32 || z.kind == LSX_F16 || z.kind == LSX_BF16, "unknown storage kind");
    LSX_ENSURE(z.rows > 0 && z.rows <= (size_t)1 << 27, "check the row count");
    LSX_ENSURE(z.vocab > 0 && z.vocab <= (size_t)1 << 30, "check the vocabulary size");
    LSX_ENSURE(z.stride >= z.vocab && z.stride <= (size_t)1 << 32, "rows of logits must not overlap");
    LSX_ENSURE(reinterpret_cast<uintptr_t>(z.data) % dtype_bytes(z.kind) == 0, "logits are not aligned to their type");
    LSX_ENSURE(z.temperature >= 1e-6 && z.temperature <= 1e6, "the temperature must be in 1e-6..=1e6");
    return LSX_OK;
}

// A gradient of the logits' kind: the logits' own rows (in place), or memory of its own.
int check_gradient(const LogitRows& z, const void* gradient, size_t stride) {
    LSX_ENSURE(gradient, "invalid argument");
    LSX_ENSURE(stride >= z.vocab && stride <= (size_t)1 << 32, "rows of the gradient must not overlap");
    const size_t e = dtype_bytes(z.kind);
    const uintptr_t a = reinterpret_cast<uintptr_t>(z.data), b = reinterpret_cast<uintptr_t>(gradient);
    LSX_ENSURE(b % e == 0, "the gradient is not aligned to its type");
    if (a == b && stride == z.stride) return LSX_OK;
    const uintptr_t a_end = a + ((z.rows - 1) * z.stride + z.vocab) * e;
    const uintptr_t b_end = b + ((z.rows - 1) * stride + z.vocab) * e;
    if (a_end <= b || b_end <= a) return LSX_OK;
    // two column blocks of one buffer
    if (stride == z.stride) {
        const size_t gap = (a < b ? b - a : a - b) / e % stride;
        if (gap >= z.vocab && stride - gap >= z.vocab) return LSX_OK;
    }
    return fail(LSX_E_ARGUMENT, "the gradient overlaps the logits without being them");
}

int check_teacher(const TeacherRows& t) {
    LSX_ENSURE(t.ids && t.logits, "invalid argument");
    LSX_ENSURE(t.slots > 0 && t.slots <= (size_t)kMaxSlots, "the teacher lists 1..=128 tokens a row");
    return LSX_OK;
}

}  // namespace lsx

using namespace lsx;

extern "C" {

int lsx_token_logprobs_device(lsx_ctx* ctx, const void* logits, lsx_dtype kind, size_t rows, size_t vocab,
                              size_t stride, double temperature, const uint32_t* tokens, size_t token_count,
                              size_t alternatives, float* logprob_out, float* entropy_out, float* stats_out,
                              uint32_t* top_ids_out, float* top_logits_out, float* top_logprobs_out, void* stream) {
    const LogitRows z{logits, kind, rows, vocab, stride, temperature};
    LSX_TRY(check_rows(z));
    LSX_ENSURE(token_count <= (size_t)kMaxSlots, "a row names at most 128 tokens");
    LSX_ENSURE((token_count > 0) == (tokens != nullptr) && (tokens || !logprob_out),
               "give the tokens, their count and an output together");
    LSX_ENSURE(alternatives <= (size_t)kMaxSlots && alternatives <= vocab,
               "the alternatives are at most 128 and at most the vocabulary");
    LSX_ENSURE(alternatives > 0 || (!top_ids_out && !top_logits_out && !top_logprobs_out),
               "alternatives need a count");
    LSX_ENSURE(ctx, "context is NULL");
    const cudaStream_t on = stream ? (cudaStream_t)stream : ctx->stream;
    DeviceScope scope(ctx->device);
    LSX_CUDA(scope.status, "select device");
    if (!top_ids_out && !top_logits_out && !top_logprobs_out) alternatives = 0;
    const LogprobOutputs out{logprob_out, entropy_out, stats_out, top_ids_out, top_logits_out, top_logprobs_out};
    LSX_CUDA(launch_token_logprobs(on, ctx->sm_count, z, tokens, token_count, alternatives, out),
             "token log probabilities");
    return LSX_OK;
}

int lsx_token_logprobs_backward_device(lsx_ctx* ctx, const void* logits, lsx_dtype kind, size_t rows, size_t vocab,
                                       size_t stride, double temperature, const uint32_t* tokens, size_t token_count,
                                       const float* stats, const float* entropy, const float* logprob_gradient,
                                       const float* entropy_gradient, void* gradient_out, size_t gradient_stride,
                                       void* stream) {
    const LogitRows z{logits, kind, rows, vocab, stride, temperature};
    LSX_TRY(check_rows(z));
    LSX_TRY(check_gradient(z, gradient_out, gradient_stride));
    LSX_ENSURE(stats, "invalid argument");
    LSX_ENSURE(token_count <= (size_t)kMaxSlots, "a row names at most 128 tokens");
    LSX_ENSURE((token_count > 0) == (tokens != nullptr) && (tokens != nullptr) == (logprob_gradient != nullptr),
               "give the tokens, their count and their gradients together");
    LSX_ENSURE((entropy != nullptr) == (entropy_gradient != nullptr), "give the entropy and its gradient together");
    LSX_ENSURE(ctx, "context is NULL");
    const cudaStream_t on = stream ? (cudaStream_t)stream : ctx->stream;
    DeviceScope scope(ctx->device);
    LSX_CUDA(scope.status, "select device");
    LSX_CUDA(launch_logprobs_gradient(on, ctx->sm_count, z, tokens, token_count, stats, entropy,
                                      logprob_gradient, entropy_gradient, gradient_out, gradient_stride),
             "token log probabilities' gradient");
    return LSX_OK;
}

int lsx_distill_device(lsx_ctx* ctx, const void* logits, lsx_dtype kind, size_t rows, size_t vocab, size_t stride,
                       double temperature, const uint32_t* teacher_ids, const float* teacher_logits,
                       size_t teacher_count, const float* teacher_stats, const float* weights, float* loss_out,
                       float* stats_out, void* gradient_out, size_t gradient_stride, void* stream) {
    const LogitRows z{logits, kind, rows, vocab, stride, temperature};
    const TeacherRows teacher{teacher_ids, teacher_logits, teacher_stats, teacher_count};
    LSX_TRY(check_rows(z));
    LSX_TRY(check_teacher(teacher));
    if (gradient_out) LSX_TRY(check_gradient(z, gradient_out, gradient_stride));
    LSX_ENSURE(gradient_out || !weights, "weights scale the gradient only");
    LSX_ENSURE(ctx, "context is NULL");
    const cudaStream_t on = stream ? (cudaStream_t)stream : ctx->stream;
    DeviceScope scope(ctx->device);
    LSX_CUDA(scope.status, "select device");
    LSX_CUDA(launch_distill(on, ctx->sm_count, z, teacher, weights, loss_out, stats_out, gradient_out,
                            gradient_stride),
             "distillation");
    return LSX_OK;
}

int lsx_distill_backward_device(lsx_ctx* ctx, const void* logits, lsx_dtype kind, size_t rows, size_t vocab,
                                size_t stride, double temperature, const uint32_t* teacher_ids,
                                const float* teacher_logits, size_t teacher_count, const float* teacher_stats,
                                const float* stats, const float* loss_gradient, void* gradient_out,
                                size_t gradient_stride, void* stream) {
    const LogitRows z{logits, kind, rows, vocab, stride, temperature};
    const TeacherRows teacher{teacher_ids, teacher_logits, teacher_stats, teacher_count};
    LSX_TRY(check_rows(z));
    LSX_TRY(check_teacher(teacher));
    LSX_TRY(check_gradient(z, gradient_out, gradient_stride));
    LSX_ENSURE(stats && loss_gradient, "invalid argument");
    LSX_ENSURE(ctx, "context is NULL");
    const cudaStream_t on = stream ? (cudaStream_t)stream : ctx->stream;
    DeviceScope scope(ctx->device);
    LSX_CUDA(scope.status, "select device");
    LSX_CUDA(launch_distill_gradient(on, ctx->sm_count, z, teacher, stats, loss_gradient, gradient_out,
                                     gradient_stride),
             "distillation gradient");
    return LSX_OK;
}

}  // extern "C"
