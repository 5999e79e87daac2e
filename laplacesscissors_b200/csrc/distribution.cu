// Operators on rows of logits: log probabilities of given tokens with the entropy and
// the top alternatives, distillation from a teacher's top logits, and the gradients
// of both with respect to the logits.
//
// Per row z[0..V) at temperature T, with m = max z and s = ln sum_i exp((z_i - m) / T),
// the probabilities are q_i = exp((z_i - m) / T - s).  Every operator is one pass over
// the row (two for a loss with its gradient): HBM traffic bounds it, and one exponential
// per element (MUFU) comes next.
//
// Differences are formed before they are scaled: y = (z - r) * (log2 e / T) against a
// reference r that is itself one of the logits, so the lowest value of a type, -inf
// masks and logits far from zero all give the exponent their difference has.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <cstdlib>
#include <cstdio>
#include <type_traits>

#include "device_common.cuh"
#include "distribution.cuh"
#include "lsx_internal.h"

namespace lsx {
namespace {

constexpr int kRowThreads = 256;
constexpr int kPieceThreads = 128;   // of the gradient kernels
constexpr int kListCap = 2048;     // candidate keys of one selection
constexpr int kMarkWords = 512;    // 32-bit words of the bitmap of marked vectors
constexpr int kStepShared = 8448;        // what the step kernel holds beside its slice, the system's share included
constexpr int kPlainShared = 36 << 10;   // dynamic shared memory that needs no opt-in beside the kernels' own
constexpr int kStagedTarget = 40 << 10;  // a slice kept in shared memory: 4 blocks on an SM
constexpr int kStagedMost = 200 << 10;   // and at most
constexpr int kPieceVectors = 2048;      // a slice of the gradient kernels
constexpr int kUnroll = 4;         // 16-byte loads in flight per thread
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
        const int end = (int)(((long long)lead + vocab) / n);
        last = ((long long)lead + vocab) % n != 0 && end >= full0;
        full1 = end > full0 ? end : full0;
    }
    __device__ __forceinline__ long long first(int j) const { return (long long)j * Vec<E>::n - lead; }
    __device__ __forceinline__ uint4 full(int j) const { return load16(base + (long long)j * Vec<E>::n); }
    __device__ __forceinline__ void ragged(int j, float* v) const {
#pragma unroll
        for (int e = 0; e < Vec<E>::n; ++e) {
            const long long i = first(j) + e;
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
        const long long full = row.full1 - row.full0;
        lo = row.full0 + (int)(full * part / parts);
        hi = row.full0 + (int)(full * (part + 1) / parts);
        head = row.head && part == 0;
        last = row.last && part == parts - 1;
        begin = part == 0 ? 0 : (int)row.first(lo);
        end = part == parts - 1 ? row.vocab : (int)row.first(hi);
    }
};

// ---- marked tokens -----------------------------------------------------------
// The tokens a row lists, sorted; a bitmap over vector numbers (modulo its size) tells
// the streaming loop which vectors to look up.  One word covers 32 consecutive vectors,
// which is what a warp holds.
struct Marks {
    uint32_t raw[kMaxSlots];
    uint32_t ids[kMaxSlots];
    int count;
    uint32_t bits[kMarkWords];
};

// Reads one row's token list and sorts it; ends with the block synchronised.
template <typename E>
__device__ void build_marks(Marks& M, const uint32_t* list, int slots, const Row<E>& row) {
    const int tid = threadIdx.x;
    for (int i = tid; i < kMarkWords; i += blockDim.x) M.bits[i] = 0;
    if (tid == 0) M.count = 0;
    __syncthreads();
    for (int i = tid; i < slots; i += blockDim.x) {
        const uint32_t id = list[i] < (uint32_t)row.vocab ? list[i] : kUnusedToken;
        M.raw[i] = id;
        if (id != kUnusedToken) {
            atomicAdd(&M.count, 1);
            const uint32_t j = (uint32_t)(((long long)id + row.lead) / Vec<E>::n);
            atomicOr(&M.bits[(j >> 5) & (kMarkWords - 1)], 1u << (j & 31));
        }
    }
    __syncthreads();
    for (int slot = tid; slot < slots; slot += blockDim.x) {
        const uint32_t id = M.raw[slot];
        int rank = 0;
        for (int j = 0; j < slots; ++j) rank += M.raw[j] < id || (M.raw[j] == id && j < slot);
        if (id != kUnusedToken) M.ids[rank] = id;
    }
    __syncthreads();
}

__device__ __forceinline__ bool marked(const Marks& M, int j) {
    return (M.bits[((uint32_t)j >> 5) & (kMarkWords - 1)] >> (j & 31)) & 1u;
}

// First position of `ids` holding a token >= first.
__device__ __forceinline__ int mark_position(const Marks& M, long long first) {
    int lo = 0, hi = M.count;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((long long)M.ids[mid] < first)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
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

template <typename E, bool kExclude, bool kRanked>
__device__ __forceinline__ void stream_slice(const Row<E>& row, const Slice& part, const Marks* M, const Scale& k,
                                             Running<kRanked>& acc) {
    constexpr int n = Vec<E>::n;
    auto exclude = [&](int j, float* v) {
        int pos = mark_position(*M, row.first(j));
#pragma unroll
        for (int e = 0; e < n; ++e)
            while (pos < M->count && (long long)M->ids[pos] == row.first(j) + e) {
                v[e] = -INFINITY;
                ++pos;
            }
    };
    auto take = [&](int j, uint4 w) {
        float v[n];
        Vec<E>::unpack(w, v);
        float top = Vec<E>::top(w);
        if (kExclude && marked(*M, j)) {
            exclude(j, v);
            top = v[0];
#pragma unroll
            for (int e = 1; e < n; ++e) top = fmaxf(top, v[e]);
        }
        acc.template add<n>(v, top, j, k);
    };
    auto take_ragged = [&](int j) {
        float v[n];
        row.ragged(j, v);
        if (kExclude) exclude(j, v);
        float top = v[0];
#pragma unroll
        for (int e = 1; e < n; ++e) top = fmaxf(top, v[e]);
        acc.template add<n>(v, top, j, k);
    };
    const int tid = threadIdx.x, T = blockDim.x;
    int j = part.lo + tid;
    // every thread meets its vectors in ascending order
    if (part.head && tid == 0) {
        acc.at = 0;
        take_ragged(0);
    } else if (j < part.hi) {
        acc.at = j;
    } else if (part.last && tid == T - 1) {
        acc.at = row.full1;
    }
    for (; j + (kUnroll - 1) * T < part.hi; j += kUnroll * T) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = row.full(j + u * T);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) take(j + u * T, w[u]);
    }
    for (; j < part.hi; j += T) take(j, row.full(j));
    if (part.last && tid == T - 1) take_ragged(row.full1);
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
    for (long long j = (long long)part.lo + owner + (long long)lane * T; j < part.hi; j += 32ll * T) {
        Vec<E>::unpack(row.full((int)j), v);
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
__device__ Partial slice_sums(const Row<E>& row, const Slice& part, const Running<true>& acc, const Scale& k, Sums* scratch,
                              int* owner) {
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
            // (a thread's own element at x.m, if any, went with the owner's sums)
            scratch[32] = again;
        }
        const Sums rest = block_sums(others, k.L, scratch);
        __syncthreads();
        p.rest = rest.S + scratch[32].S;
        p.W = rest.W + scratch[32].W;
    }
    return p;
}

// The row's sums from its blocks' shares.
__device__ __forceinline__ Partial combine(const Partial* parts, int count, float L) {
    Partial t = parts[0];
    if (count == 1) return t;
    int first = 0;
    for (int i = 1; i < count; ++i)
        if (parts[i].any && (!t.any || parts[i].m > t.m)) {
            t = parts[i];
            first = i;
        }
    for (int i = 0; i < count; ++i) {
        if (i == first || !parts[i].any) continue;
        Sums x{parts[i].m, 1.f + parts[i].rest, parts[i].W};
        x.rebase(t.m, L);
        t.rest += x.S;
        t.W += x.W;
    }
    return t;
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

constexpr int kMaxGroups = 256;
constexpr int kFewerCap = 512;
constexpr int kMaxCluster = 8;     // the portable size

struct Selection {
    alignas(16) unsigned long long keys[kListCap];
    alignas(16) unsigned long long fewer[kFewerCap];
    alignas(16) unsigned long long group[kMaxGroups];
    unsigned long long best[kMaxSlots];
    unsigned long long threshold;
    int count;
};

// A bound for the `top`-th largest of keys that the threads hold: groups of threads take
// their largest (`mine`, 0 for none), and the `top`-th largest of the groups' is returned (0
// where there are not as many).  Distinct keys; `top` of all the keys are at or above the
// bound.  Resets P.count.  Ends with the block synchronised.
__device__ unsigned long long group_bound(Selection& P, unsigned long long mine, int top) {
    const int tid = threadIdx.x, T = blockDim.x;
    // groups as wide as leave 2.5 groups per wanted key
    const int wide = top * 10 <= T ? 4 : top * 5 <= T ? 2 : 1, groups = T / wide;
    for (int o = 1; o < wide; o <<= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
        mine = other > mine ? other : mine;
    }
    if (tid % wide == 0) P.group[tid / wide] = mine;
    if (tid == 0) {
        P.threshold = 0ull;
        P.count = 0;
    }
    __syncthreads();
    // a group's threads share the comparisons of its key
    int above = 0;
#pragma unroll 4
    for (int i = 2 * (tid % wide); i < groups; i += 2 * wide) {
        const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(&P.group[i]);
        above += (pair.x > mine) + (pair.y > mine);
    }
    for (int o = 1; o < wide; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (above == top - 1 && mine != 0ull) P.threshold = mine;
    __syncthreads();
    return P.threshold;
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
    const unsigned long long bound = group_bound(P, mine, top);
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

// The best tokens of a slice from what the threads met while they summed it.  A thread's
// key is its best vector, ordered by (largest logit, lower vector number first); the bound
// from groups of threads lies below the `top`-th best element, since `top` elements, one in
// each better group, are at least as good.  So only elements at or above it are candidates,
// about G ln(1 / (1 - top / G)) of them where the tokens lie at random over G groups.  They
// are read again (from L2) at the threads' best vectors, and in all their vectors only for
// threads that have a second one to offer.  More candidates than the list holds are left
// to select_by_pieces.
template <typename E>
__device__ void select_by_threads(Selection& P, const Row<E>& row, const Slice& part, const E* z, int top,
                                  const Running<true>& acc, int cap) {
    constexpr int n = Vec<E>::n;
    const int tid = threadIdx.x, lane = tid & 31, T = blockDim.x;
    const unsigned long long mine =
        acc.at < 0 ? 0ull : ((unsigned long long)total_order_key(acc.m + 0.f) << 32) | (0xffffffffu - (uint32_t)acc.at);
    const unsigned long long bound = group_bound(P, mine, top);
    auto offer = [&](int j, const float* v) {
        const uint32_t low = 0xffffffffu - (uint32_t)j;
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const long long i = row.first(j) + e;
            const unsigned long long key = ((unsigned long long)total_order_key(v[e] + 0.f) << 32) | low;
            if (key >= bound && i >= 0 && i < row.vocab) {
                const int pos = atomicAdd(&P.count, 1);
                if (pos < cap) P.keys[pos] = order_key(v[e], (uint32_t)i);
            }
        }
    };
    auto offer_vector = [&](int j) {
        float v[n];
        if (j >= row.full0 && j < row.full1)
            Vec<E>::unpack(row.full(j), v);
        else
            row.ragged(j, v);
        offer(j, v);
    };
    const bool in = mine != 0ull && mine >= bound;
    // a second vector counts where its largest logit beats the bound's, or equals it at a
    // vector number up to the bound's
    const uint32_t level = (uint32_t)(bound >> 32), second = total_order_key(acc.second + 0.f);
    const long long bound_at = (long long)(0xffffffffu - (uint32_t)bound);
    uint32_t again = __ballot_sync(0xffffffffu, in && second >= level);
    if (in) offer_vector(acc.at);
    for (; again; again &= again - 1) {
        const int from = __ffs(again) - 1, who = (tid & ~31) + from;
        const int skip = __shfl_sync(0xffffffffu, acc.at, from);
        const bool tie = __shfl_sync(0xffffffffu, second, from) == level;
        const long long end = tie && bound_at + 1 < part.hi ? bound_at + 1 : part.hi;
        for (long long j = (long long)part.lo + who + (long long)lane * T; j < end; j += 32ll * T)
            if (j != skip) offer_vector((int)j);
        if (lane == 0 && part.head && who == 0 && skip != 0) offer_vector(0);
        if (lane == 0 && part.last && who == T - 1 && skip != row.full1) offer_vector(row.full1);
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
// which puts them together and writes the row's results.
template <typename E, int T>
__global__ void __launch_bounds__(T, 1280 / T) token_logprobs_kernel(const E* __restrict__ logits, int vocab, size_t stride,
                                                          const Scale k, const uint32_t* __restrict__ tokens,
                                                          int token_count, int top, LogprobOutputs out) {
    __shared__ Sums scratch[33];
    __shared__ Partial shares[kMaxCluster];
    __shared__ Selection selection;
    __shared__ int owner;
    const int parts = cluster_size(), part = cluster_rank();
    if (parts > 1) cluster_arrive();  // waited for before the first store into another block
    const size_t r = blockIdx.x / parts;
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
    stream_slice<E, false>(row, slice, nullptr, k, acc);
    Partial sums = slice_sums(row, slice, acc, k, scratch, &owner);
    // clusters keep the upper half of the list for the blocks' best keys
    const int cap = parts > 1 ? kListCap / 2 : kListCap;
    if (top > 0) {
        if (!sums.any) {  // nothing but -inf: the lowest ids
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
        if (top > 0) rank_keys(selection, selection.keys + kListCap / 2, parts * top, top);
    }
    const bool empty = !sums.any;  // every logit is -inf
    const float m = sums.m, log_sum = empty ? 0.f : log1pf(sums.rest);
    auto logprob = [&](float x) { return empty ? -INFINITY : (x - m) * k.inverse - log_sum; };
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

// ---- lists of tokens -------------------------------------------------------------------------
// One row's listed tokens.
struct List {
    uint32_t ids[kMaxSlots];  // kUnusedToken but in the first slot that names a token
    float logit[kMaxSlots];   // the row's logit of that token, else -inf
    float value[kMaxSlots];   // what the operator keeps with the slot
    int bad;                 // some slot names a token outside the vocabulary
};

// Reads a row's list and the logits it names in [begin, end), by the first warp (slot
// lane + 32 q).
template <typename E>
__device__ void read_list(List& list, const uint32_t* ids, int count, const E* z, int vocab, int begin, int end) {
    constexpr int kPer = kMaxSlots / 32;
    const int lane = threadIdx.x & 31;
    uint32_t id[kPer];
    bool bad = false;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const int i = lane + 32 * q;
        id[q] = i < count ? ids[i] : kUnusedToken;
    }
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (32 * q >= count) break;
        const int i = lane + 32 * q;
        const bool used = id[q] < (uint32_t)vocab;
        const float logit = used && (int)id[q] >= begin && (int)id[q] < end ? Vec<E>::one(z[id[q]]) : -INFINITY;
        bad |= !used && id[q] != kUnusedToken;
        // the same token in an earlier slot: of these 32, or of the 32s before
        bool again = (__match_any_sync(0xffffffffu, id[q]) & ((1u << lane) - 1)) != 0;
#pragma unroll
        for (int p = 0; p < q; ++p)
#pragma unroll 8
            for (int from = 0; from < 32; ++from) again |= __shfl_sync(0xffffffffu, id[p], from) == id[q];
        if (i < count) {
            list.ids[i] = used && !again ? id[q] : kUnusedToken;
            list.logit[i] = used && !again ? logit : -INFINITY;
            list.value[i] = 0.f;
        }
    }
    const bool any = __any_sync(0xffffffffu, bad);
    if (lane == 0) list.bad = any;
    __syncwarp();
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
    asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}

// The dense gradient of a slice into `out` (the row's first element): vectors from
// `staged` (slot j - lo) or, where it is null, from the row itself, by T threads.  `out` may
// be the row.  `ready` gives the coefficients, once, after the first loads are on their way.
template <typename E, bool kLinear, typename F>
__device__ __forceinline__ void write_dense(const Row<E>& row, const Slice& part, const uint4* staged, E* out, float L,
                                            int tid, int T, F&& ready) {
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
            const long long i = row.first(j) + e;
            if (i >= 0 && i < row.vocab) out[i] = Vec<E>::store(v[e]);
        }
    };
    int j = part.lo + tid;
    if (staged) {
        d = ready();
        for (; j < part.hi; j += T) put(j, staged[j - part.lo]);
    } else {
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
    const size_t r = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - r * parts), tid = threadIdx.x;
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
        write_dense<E, true>(row, slice, nullptr, out, k.L, tid, kPieceThreads, ready);
    else
        write_dense<E, false>(row, slice, nullptr, out, k.L, tid, kPieceThreads, ready);
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
// The listed tokens' side of one row in 64 bits, by one warp: sums over at most kMaxSlots
// numbers, of which 1 - sum p is next to 0 for a confident teacher.
struct Listed {
    double mass;   // sum of p
    double rest;   // the teacher's mass outside the list (0 without its statistics)
    double log_rest;
    float m;       // the largest listed logit of the student
    double inside; // sum exp((z - m) / T) over the listed tokens
    double cross;  // sum p (ln p - (z - m) / T)
};

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

// By the warp that read the list.  Also leaves scale * p in list.value.
template <bool kStudent>
__device__ Listed listed_sums(List& list, double* work, const float* values, const float* stats, int count,
                              double inverse, double scale) {
    const int lane = threadIdx.x & 31;
    Listed t{0.0, 0.0, 0.0, -INFINITY, 0.0, 0.0};
    float top = -INFINITY;
    for (int i = lane; i < count; i += 32) {
        const float value = list.ids[i] != kUnusedToken ? values[i] : -INFINITY;
        list.value[i] = value;
        top = fmaxf(top, value);
        if (kStudent) t.m = fmaxf(t.m, list.logit[i]);
    }
    if (kStudent) t.m = warp_max(t.m);
    double shift, norm = 0.0;
    bool none = false;  // the teacher's row holds no token: it asks for nothing
    if (stats) {
        none = stats[0] == -INFINITY && stats[1] == 0.f;
        shift = none ? 0.0 : (double)stats[0];
        norm = (double)stats[1];
    } else {
        top = warp_max(top);
        shift = top == -INFINITY ? 0.0 : (double)top;
    }
    for (int i = lane; i < count; i += 32) {
        const double log_p = ((double)list.value[i] - shift) * inverse - norm, p = exp(log_p);
        t.mass += p;
        if (kStudent) {
            const float z = list.logit[i];
            const double log_q = z == -INFINITY ? -INFINITY : ((double)z - (double)t.m) * inverse;
            t.inside += exp(log_q);
            work[i] = p != 0.0 ? log_p - log_q : 0.0;
        }
        work[kMaxSlots + i] = p;
    }
    t.mass = warp_sum_f64(t.mass);
    if (kStudent) t.inside = warp_sum_f64(t.inside);
    double share = 1.0;
    norm = 0.0;
    if (stats) {
        if (!none) t.rest = t.mass < 1.0 ? 1.0 - t.mass : (t.mass >= 1.0 ? 0.0 : t.mass);
        t.log_rest = log(t.rest);
    } else if (t.mass != 0.0) {  // normalised over the list
        share = 1.0 / t.mass;
        norm = log(t.mass);
        t.mass = t.mass == t.mass ? 1.0 : t.mass;
    }
    for (int i = lane; i < count; i += 32) {
        const double p = work[kMaxSlots + i] * share;
        list.value[i] = (float)(scale * p);
        if (kStudent && p != 0.0) t.cross += p * (work[i] - norm);
    }
    if (kStudent) t.cross = warp_sum_f64(t.cross);
    __syncwarp();
    return t;
}

// The tokens outside the list are one outcome only where the student's share of them is
// a normal f32 number (2^-126 and up).
constexpr float kSmallestLogShare = -87.33654475f;

// What the gradient of one row needs beside its list: listed elements get q a - value, q
// against `offset`.
struct DistillRow {
    Dense dense;
    float m, offset, a;
    bool zero;
};

// The tokens outside the list are exponentiated against their own sum: 2^y = q_i / q_r
// stays in range and (P q_r - p_r) is the whole coefficient, however small q_r is.
__device__ __forceinline__ DistillRow distill_row(const Listed& t, float m, float log_sum, float log_rest, bool empty,
                                                  bool bad, float scale) {
    const float log_share = log_rest - log_sum;
    const bool tail = log_share >= kSmallestLogShare;
    const float rest = (float)t.rest, mass = (float)(tail ? t.mass + t.rest : t.mass);
    DistillRow g;
    g.m = m;
    g.offset = log_sum * kLog2E;
    g.a = bad ? NAN : scale * mass;
    g.zero = empty;
    g.dense.m = g.m;
    g.dense.offset = tail ? log_rest * kLog2E : g.offset;
    g.dense.a = bad ? NAN : scale * (tail ? fmaf(mass, expf(log_share), -rest) : mass);
    g.dense.b = 0.f;
    if (empty) g.dense = dense_zero();
    return g;
}

// Writes a slice's listed elements over its dense gradient.  After a block barrier.
template <typename E>
__device__ __forceinline__ void write_listed(const List& list, int count, const Slice& slice, const DistillRow& g,
                                             float L, E* out, int tid) {
    if (tid >= count) return;
    const int id = (int)list.ids[tid];  // (an unused slot's is negative)
    if (id < slice.begin || id >= slice.end) return;
    const float y = max_nan(fmaf(list.logit[tid] - g.m, L, -g.offset), kLowestExponent);
    out[id] = Vec<E>::store(g.zero ? 0.f : fmaf(exp2_fast(y), g.a, -list.value[tid]));
}

__device__ __forceinline__ void copy16_async(void* shared, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(shared)), "l"(global) : "memory");
}

// A row's statistics from its listed tokens' and its other tokens' sums: both shares around
// the larger maximum, and sum - 1 apart, since ln(sum) may be all of it.
struct RowSums {
    float m, log_sum, log_rest;
    bool empty;
};
__device__ __forceinline__ RowSums row_sums(const Listed& t, const Sums& rest, const Scale& k, bool tail) {
    RowSums x;
    x.m = fmaxf(rest.m, t.m);
    const bool some = rest.S != 0.f, listed = t.inside != 0.0;
    const float below = some ? (rest.m - x.m) * k.inverse : -INFINITY;
    const float outside = some ? rest.S * expf(below) : 0.f;
    const float over = t.m == x.m ? (float)(t.inside - 1.0) + outside
                                  : (listed ? (float)t.inside * expf((t.m - x.m) * k.inverse) : 0.f) + (outside - 1.f);
    x.empty = !some && !listed;
    x.log_sum = x.empty ? 0.f : log1pf(over);
    x.log_rest = tail && some ? logf(rest.S) + below : -INFINITY;
    return x;
}

// Loss and statistics of a row; by one thread.
__device__ __forceinline__ void write_row(const Listed& t, const RowSums& x, double inverse, bool tail, bool bad,
                                          size_t r, float* loss, float* stats) {
    if (loss) {
        double value = t.mass == 0.0         ? 0.0
                       : t.cross == INFINITY ? INFINITY
                                             : t.cross + t.mass * (((double)x.m - (double)t.m) * inverse + x.log_sum);
        if (tail && t.rest > 0.0 && x.log_rest - x.log_sum >= kSmallestLogShare)
            value += t.rest * (t.log_rest - x.log_rest + x.log_sum);
        loss[r] = bad || t.mass != t.mass || x.log_sum != x.log_sum ? NAN : (float)value;
    }
    if (stats) {
        stats[3 * r] = x.m;
        stats[3 * r + 1] = x.log_sum;
        stats[3 * r + 2] = x.log_rest;
    }
}

// The row's sums over its unlisted tokens from the blocks' shares, in every thread.
__device__ __forceinline__ Sums combine_rest(const Sums* shares, int parts, float L) {
    Sums rest = shares[0];
    for (int i = 1; i < parts; ++i) rest.m = fmaxf(rest.m, shares[i].m);
    rest.S = 0.f;
    for (int i = 0; i < parts; ++i) {
        Sums x = shares[i];
        x.rebase(rest.m, L);
        rest.S += x.S;
    }
    return rest;
}

// Loss and gradient of whole batches: clusters of blocks take row after row.  Each block
// holds its slice of the row in shared memory, so the row is read once: the listed tokens
// are struck out there (their share is summed by itself, in 64 bits), the rest is summed,
// the blocks exchange their sums, and the gradient is formed from the same copy.
// The first block's first warp works a row ahead: it reads the list, gathers its logits
// and forms its sums (a chain of dependent loads and 64-bit functions as long as a
// slice's work) while the other warps take the current row.  One cluster barrier per row
// publishes both the blocks' sums and the list sent during the row before.
constexpr int kOthers = kRowThreads - 32;  // the threads that take the slice
__device__ __forceinline__ void others_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kOthers) : "memory"); }

struct StepRow {  // what the first block sends for a row
    List list;
    Listed sums;
    float scale;
};

template <typename E, bool kTail>
__global__ void __launch_bounds__(kRowThreads, 5) distill_step_kernel(
    const E* logits, int rows, int vocab, size_t stride, const Scale k, double inverse, TeacherRows teacher,
    const float* __restrict__ weights, float* loss, float* stats, E* gradient, size_t gradient_stride) {
    constexpr int n = Vec<E>::n;
    extern __shared__ __align__(16) uint4 staged[];
    __shared__ StepRow ready[2];
    __shared__ Sums shares[2][kMaxCluster];
    __shared__ Sums scratch[kOthers / 32];
    __shared__ DistillRow grow;
    const int parts = cluster_size(), part = cluster_rank(), tid = threadIdx.x;
    const int clusters = gridDim.x / parts, first = blockIdx.x / parts;
    const int count = (int)teacher.slots;

    if (tid < 32) {
        __shared__ StepRow ahead;
        __shared__ double work[2 * kMaxSlots];
        auto prepare = [&](int r) {
            const E* z = logits + (size_t)r * stride;
            const double scale = (weights ? (double)weights[r] : 1.0) * inverse;
            read_list(ahead.list, teacher.ids + (size_t)r * count, count, z, vocab, 0, vocab);
            const Listed t = listed_sums<true>(ahead.list, work, teacher.logits + (size_t)r * count,
                                               kTail ? teacher.stats + 2 * (size_t)r : nullptr, count, inverse, scale);
            if (tid == 0) {
                ahead.sums = t;
                ahead.scale = (float)scale;
            }
            __syncwarp();
        };
        auto send = [&](int to_buffer) {
            for (int to = 0; to < parts; ++to) {
                StepRow* there = in_block(&ready[to_buffer], to);
                for (int i = tid; i < count; i += 32) {
                    there->list.ids[i] = ahead.list.ids[i];
                    there->list.logit[i] = ahead.list.logit[i];
                    there->list.value[i] = ahead.list.value[i];
                }
                if (tid == 0) {
                    there->list.bad = ahead.list.bad;
                    there->sums = ahead.sums;
                    there->scale = ahead.scale;
                }
            }
            __syncwarp();
        };
        cluster_arrive();  // every block of the cluster runs from here on
        if (part == 0 && first < rows) prepare(first);
        cluster_wait();
        if (part == 0 && first < rows) send(0);
        int buffer = 0;
        for (int r = first; r < rows; r += clusters, buffer ^= 1) {
            cluster_arrive();
            const bool more = part == 0 && r + clusters < rows;
            if (more) prepare(r + clusters);
            // after this no block reads what the row before last left in the other buffer
            cluster_wait();
            if (more) send(buffer ^ 1);
        }
        return;
    }

    const int lane = tid - 32;
    cluster_arrive();
    cluster_wait();
    int buffer = 0;
    for (int r = first; r < rows; r += clusters, buffer ^= 1) {
        const Row<E> row(logits + (size_t)r * stride, vocab);
        const Slice slice(row, part, parts);
        const int full = slice.hi - slice.lo;
        const E* from = row.base + (long long)slice.lo * n;
        for (int i = lane; i < full; i += kOthers) copy16_async(&staged[i], from + (long long)i * n);
        const uint32_t id = lane < count ? teacher.ids[(size_t)r * count + lane] : kUnusedToken;
        // the ragged ends follow, -inf beyond the row
        if (slice.head && lane == 0) {
            float v[n];
            row.ragged(0, v);
            staged[full] = Vec<E>::pack(v);
        }
        if (slice.last && lane == kOthers - 1) {
            float v[n];
            row.ragged(row.full1, v);
            staged[full + 1] = Vec<E>::pack(v);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        others_barrier();
        if (id < (uint32_t)vocab && (int)id >= slice.begin && (int)id < slice.end) {
            const uint32_t at = id + row.lead;
            const int j = (int)(at / n);
            const int slot = j < row.full0 ? full : j >= row.full1 ? full + 1 : j - slice.lo;
            reinterpret_cast<E*>(&staged[slot])[at % n] = Vec<E>::store(-INFINITY);
        }
        others_barrier();
        Running<false> acc;
        auto take = [&](int i) {
            const uint4 w = staged[i];
            float v[n];
            Vec<E>::unpack(w, v);
            acc.template add<n>(v, Vec<E>::top(w), i, k);
        };
        for (int i = lane; i < full; i += kOthers) take(i);
        if (slice.head && lane == 0) take(full);
        if (slice.last && lane == kOthers - 1) take(full + 1);
        const Sums mine = warp_sums(acc.sums(), acc.m, k.L);
        if ((lane & 31) == 0) scratch[lane >> 5] = mine;
        others_barrier();
        if (lane < 32) {
            const Sums x = lane < kOthers / 32 ? scratch[lane] : Sums{-INFINITY, 0.f, 0.f};
            const Sums sums = warp_sums(x, x.m, k.L);
            if (lane < parts) *in_block(&shares[buffer][part], lane) = sums;
        }
        cluster_arrive();
        cluster_wait();
        const StepRow& given = ready[buffer];
        // the coefficients by one warp, loss and statistics by another
        if (lane == 0 || (lane == 32 && part == 0)) {
            const RowSums x = row_sums(given.sums, combine_rest(shares[buffer], parts, k.L), k, kTail);
            if (lane == 0)
                grow = distill_row(given.sums, x.m, x.log_sum, x.log_rest, x.empty, given.list.bad, given.scale);
            else
                write_row(given.sums, x, inverse, kTail, given.list.bad, r, loss, stats);
        }
        E* out = gradient + (size_t)r * gradient_stride;
        others_barrier();
        write_dense<E, false>(row, slice, staged, out, k.L, lane, kOthers, [&]() { return grow.dense; });
        others_barrier();
        write_listed(given.list, count, slice, grow, k.L, out, lane);
    }
}

// Loss and statistics of rows that stream through registers, a bitmap of marked vectors
// telling the sum which elements to leave out; the gradient too of rows too long for
// shared memory, which are then read twice.  A cluster of blocks shares a row.
template <typename E, bool kTail>
__global__ void __launch_bounds__(kRowThreads, 4) distill_kernel(
    const E* logits, int vocab, size_t stride, const Scale k, double inverse, TeacherRows teacher,
    const float* __restrict__ weights, float* loss, float* stats, E* gradient, size_t gradient_stride) {
    __shared__ Sums scratch[33];
    __shared__ List list;
    __shared__ double work[2 * kMaxSlots];
    __shared__ Listed listed;
    __shared__ DistillRow grow;
    __shared__ Sums shares[kMaxCluster];
    __shared__ Marks marks;
    const int parts = cluster_size(), part = cluster_rank(), tid = threadIdx.x;
    if (parts > 1) cluster_arrive();  // waited for before the first store into another block
    const size_t r = blockIdx.x / parts;
    const int count = (int)teacher.slots;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    const double scale = (weights ? (double)weights[r] : 1.0) * inverse;
    build_marks(marks, teacher.ids + r * count, count, row);
    if (tid < 32 && (part == 0 || gradient)) {
        read_list(list, teacher.ids + r * count, count, z, vocab, 0, vocab);
        const Listed t = listed_sums<true>(list, work, teacher.logits + r * count,
                                           kTail ? teacher.stats + 2 * r : nullptr, count, inverse, scale);
        if (tid == 0) listed = t;
    }
    Running<false> acc;
    stream_slice<E, true>(row, slice, &marks, k, acc);
    Sums rest = block_sums(acc, k.L, scratch);
    if (parts > 1) {
        cluster_wait();
        if (tid < parts) *in_block(&shares[part], tid) = rest;
        cluster_arrive();
        cluster_wait();
        rest = combine_rest(shares, parts, k.L);
    }
    if (tid == 0 && (part == 0 || gradient)) {
        const RowSums x = row_sums(listed, rest, k, kTail);
        grow = distill_row(listed, x.m, x.log_sum, x.log_rest, x.empty, list.bad, (float)scale);
        if (part == 0) write_row(listed, x, inverse, kTail, list.bad, r, loss, stats);
    }
    if (!gradient) return;
    E* out = gradient + r * gradient_stride;
    write_dense<E, false>(row, slice, nullptr, out, k.L, tid, kRowThreads, [&]() {
        __syncthreads();
        return grow.dense;
    });
    __syncthreads();
    write_listed(list, count, slice, grow, k.L, out, tid);
}

// The gradient from saved statistics; `parts` blocks share a row, none waits for another.
template <typename E, bool kTail>
__global__ void __launch_bounds__(kPieceThreads, 1024 / kPieceThreads) distill_gradient_kernel(
    const E* logits, int vocab, size_t stride, const Scale k, double inverse, int parts, TeacherRows teacher,
    const float* __restrict__ stats, const float* __restrict__ weights, E* gradient, size_t gradient_stride) {
    __shared__ List list;
    __shared__ double work[2 * kMaxSlots];
    __shared__ DistillRow grow;
    const size_t r = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - r * parts), count = (int)teacher.slots;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const Slice slice(row, part, parts);
    E* out = gradient + r * gradient_stride;
    write_dense<E, false>(row, slice, nullptr, out, k.L, (int)threadIdx.x, kPieceThreads, [&]() {
        if (threadIdx.x < 32) {
            const double scale = (double)weights[r] * inverse;
            const float m = stats[3 * r], log_sum = stats[3 * r + 1], log_rest = kTail ? stats[3 * r + 2] : -INFINITY;
            // (another block may be writing over the rest of the row)
            read_list(list, teacher.ids + r * count, count, z, vocab, slice.begin, slice.end);
            const Listed t = listed_sums<false>(list, work, teacher.logits + r * count,
                                                kTail ? teacher.stats + 2 * r : nullptr, count, inverse, scale);
            if (threadIdx.x == 0)
                grow = distill_row(t, m, log_sum, log_rest, m == -INFINITY && log_sum == 0.f, list.bad, (float)scale);
        }
        __syncthreads();
        return grow.dense;
    });
    __syncthreads();
    write_listed(list, count, slice, grow, k.L, out, (int)threadIdx.x);
}

template <typename F>
cudaError_t by_kind(lsx_dtype kind, F&& f) {
    switch (kind) {
    case LSX_F32: return f((const float*)nullptr);
    case LSX_F16: return f((const __half*)nullptr);
    default: return f((const __nv_bfloat16*)nullptr);
    }
}


// How many blocks share a row: as many as fill the GPU, while each keeps a full pass of
// its threads.
int row_parts(int sm_count, size_t rows, size_t vectors, int threads, int resident) {
    int parts = 1;
    while (parts < kMaxCluster && rows * parts * 2 <= (size_t)sm_count * resident &&
           vectors / (parts * 2) >= (size_t)threads)
        parts *= 2;
    return parts;
}

template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kernel)(Params...), size_t rows, int parts, int threads, size_t shared,
                            cudaStream_t s, Args... args) {
    if (shared > (size_t)kPlainShared) {
        const cudaError_t e =
            cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
        if (e != cudaSuccess) return e;
    }
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

// Lowers *clusters to what the current device holds at a time: their blocks have to lie in
// one GPC, so this is less than its SMs' room suggests.  Asked once per kernel and shape.
template <typename... Params>
cudaError_t resident_clusters(void (*kernel)(Params...), int parts, int threads, size_t shared, size_t* clusters) {
    static std::mutex guard;
    static std::map<std::tuple<const void*, int, size_t, int>, int> known;
    int device = 0, most = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const std::lock_guard<std::mutex> lock(guard);
    const auto key = std::make_tuple((const void*)kernel, parts, shared, device);
    const auto found = known.find(key);
    if (found != known.end()) {
        most = found->second;
    } else {
        if (shared > (size_t)kPlainShared) {
            e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
            if (e != cudaSuccess) return e;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)parts);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = shared;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {(unsigned)parts, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
        if (e != cudaSuccess) return e;
        if (getenv("LSX_SHOW")) fprintf(stderr, "parts %d shared %zu clusters %d\n", parts, shared, most);
        known[key] = most;
    }
    if (most > 0 && *clusters > (size_t)most) *clusters = (size_t)most;
    return cudaSuccess;
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
        if (vectors < 1024)
            return launch_clusters(token_logprobs_kernel<E, 128>, z.rows, 1, 128, 0, s, (const E*)z.data, (int)z.vocab,
                                   z.stride, k, tokens, (int)token_count, (int)alternatives, out);
        return launch_clusters(token_logprobs_kernel<E, 256>, z.rows, row_parts(sm_count, z.rows, vectors, 256, 4), 256,
                               0, s, (const E*)z.data, (int)z.vocab, z.stride, k, tokens, (int)token_count,
                               (int)alternatives, out);
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
        const Scale k(z.temperature);
        const double inverse = 1.0 / z.temperature;
        int parts = row_parts(sm_count, z.rows, vectors, kRowThreads, 4);
        auto staged = [&](int p) { return ((vectors + p - 1) / p + 3) * 16; };
        if (gradient) {
            while (parts < kMaxCluster && staged(parts) > (size_t)kStagedTarget) parts *= 2;
            const size_t shared = staged(parts);
            if (shared <= (size_t)kStagedMost) {
                const auto kernel = teacher.stats ? distill_step_kernel<E, true> : distill_step_kernel<E, false>;
                size_t clusters = z.rows;
                const cudaError_t e = resident_clusters(kernel, parts, kRowThreads, shared, &clusters);
                if (e != cudaSuccess) return e;
                return launch_clusters(kernel, clusters, parts, kRowThreads, shared, s, (const E*)z.data, (int)z.rows,
                                       (int)z.vocab, z.stride, k, inverse, teacher, weights, loss, stats, (E*)gradient,
                                       gradient_stride);
            }
        }
        return launch_clusters(teacher.stats ? distill_kernel<E, true> : distill_kernel<E, false>, z.rows, parts,
                               kRowThreads, 0, s, (const E*)z.data, (int)z.vocab, z.stride, k, inverse, teacher, weights,
                               loss, stats, (E*)gradient, gradient_stride);
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
    const uintptr_t a_end = a + ((z.rows - 1) * z.stride + z.vocab) * e, b_end = b + ((z.rows - 1) * stride + z.vocab) * e;
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
                                       const float* entropy_gradient, void* gradient_out, size_t gradient_stride, void* stream) {
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
