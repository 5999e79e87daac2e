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

#include <string>
#include <type_traits>

#include "device_common.cuh"
#include "distribution.cuh"
#include "lsx_internal.h"

namespace lsx {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kListCap = 2048;     // candidate keys of one selection
constexpr int kMarkWords = 512;    // 32-bit words of the bitmap of marked vectors
constexpr int kUnroll = 4;         // 16-byte loads in flight per thread
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents (base 2) below this are zero in f32 with room to spare; the bound keeps
// 0 * y finite for masked elements.
constexpr float kLowestExponent = -1e4f;
// A thread's reference is moved up once a logit lies this many powers of two above it.
constexpr float kSlack = 20.f;

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

// ---- marked tokens -----------------------------------------------------------
// The tokens a row lists, sorted, each with a value; a bitmap over vector numbers
// (modulo its size) tells the streaming loop which vectors to look up.  One word
// covers 32 consecutive vectors, which is what a warp holds.
struct Marks {
    uint32_t raw[kMaxSlots];
    uint32_t ids[kMaxSlots];
    float value[kMaxSlots];
    int slot_rank[kMaxSlots];  // position of each slot in `ids`; -1 unused, -2 - rank for a repeated token
    int count;
    int bad;  // some slot names a token outside the vocabulary
    uint32_t bits[kMarkWords];
};

// Reads one row's token list and sorts it (four threads per slot count the smaller
// ids); ends with the block synchronised.
template <typename E>
__device__ void build_marks(Marks& M, const uint32_t* list, int slots, const Row<E>& row) {
    const int tid = threadIdx.x;
    for (int i = tid; i < kMarkWords; i += blockDim.x) M.bits[i] = 0;
    if (tid == 0) M.count = M.bad = 0;
    __syncthreads();
    for (int i = tid; i < slots; i += blockDim.x) {
        uint32_t id = list[i];
        if (id != kUnusedToken && id >= (uint32_t)row.vocab) {
            M.bad = 1;
            id = kUnusedToken;
        }
        M.raw[i] = id;
        if (id != kUnusedToken) {
            atomicAdd(&M.count, 1);
            const uint32_t j = (uint32_t)(((long long)id + row.lead) / Vec<E>::n);
            atomicOr(&M.bits[(j >> 5) & (kMarkWords - 1)], 1u << (j & 31));
        }
    }
    __syncthreads();
    for (int base = 0; base < slots * 4; base += blockDim.x) {
        const int slot = (base + tid) >> 2, part = tid & 3;
        const uint32_t id = slot < slots ? M.raw[slot] : 0;
        int less = 0, same = 0;
        if (slot < slots)
            for (int j = part; j < slots; j += 4) {
                const uint32_t other = M.raw[j];
                less += other < id;
                same += other == id && j < slot;
            }
        less += __shfl_xor_sync(0xffffffffu, less, 1);
        less += __shfl_xor_sync(0xffffffffu, less, 2);
        same += __shfl_xor_sync(0xffffffffu, same, 1);
        same += __shfl_xor_sync(0xffffffffu, same, 2);
        if (slot < slots && part == 0) {
            const int rank = less + same;
            if (id != kUnusedToken) M.ids[rank] = id;
            M.slot_rank[slot] = id == kUnusedToken ? -1 : same ? -2 - rank : rank;
        }
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

// ---- block reductions ----------------------------------------------------------
struct BlockScratch {
    float f[3][32];
};
__device__ __forceinline__ float block_max(float v, float* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = fmaxf(v, scratch[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = warp_allsum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += scratch[w];
    return v;
}

// ---- running sums of a softmax ---------------------------------------------------
// S = sum 2^y and W = sum 2^y y over the elements seen, y against the reference r;
// S == 0 exactly while only -inf has been seen.
// With kRanked also the first vector holding the largest element, and the largest
// element of the other vectors.
template <bool kWeighted, bool kRanked = false>
struct Running {
    float r = 0.f, limit = -INFINITY, S = 0.f, W = 0.f, m = -INFINITY;
    float second = -INFINITY;
    int at = -1;
    __device__ __forceinline__ void rise(float top, float L, float slack) {
        if (S != 0.f) {
            const float shift = (r - top) * L;
            const float f = exp2_fast(shift);
            if (kWeighted) W = f > 0.f ? f * fmaf(shift, S, W) : (f == 0.f ? 0.f : f);
            S *= f;
        }
        r = top;
        limit = top + slack;
    }
    template <int n>
    __device__ __forceinline__ void add(const float* v, int j, float L, float slack) {
        float top = v[0];
#pragma unroll
        for (int e = 1; e < n; ++e) top = fmaxf(top, v[e]);
        if (kRanked) {
            second = fmaxf(second, fminf(m, top));
            at = top > m ? j : at;
        }
        m = fmaxf(m, top);
        if (top > limit) rise(top, L, slack);
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const float y = max_nan((v[e] - r) * L, kLowestExponent);
            const float p = exp2_fast(y);
            S += p;
            if (kWeighted) W = fmaf(p, y, W);
        }
    }
    // Moves the sums to the reference R >= every element seen.
    __device__ __forceinline__ void rebase(float R, float L) {
        if (S == 0.f) return;
        const float shift = (r - R) * L;
        const float f = exp2_fast(shift);
        if (kWeighted) W = f > 0.f ? f * fmaf(shift, S, W) : (f == 0.f ? 0.f : f);
        S = f == 0.f && S == S ? 0.f : f * S;
        r = R;
    }
};

template <typename E, bool kExclude, bool kWeighted, bool kRanked>
__device__ __forceinline__ void stream_row(const Row<E>& row, const Marks* M, float L, float slack,
                                           Running<kWeighted, kRanked>& acc) {
    constexpr int n = Vec<E>::n;
    auto take = [&](int j, float* v) {
        if (kExclude && marked(*M, j)) {
            int pos = mark_position(*M, row.first(j));
#pragma unroll
            for (int e = 0; e < n; ++e)
                while (pos < M->count && (long long)M->ids[pos] == row.first(j) + e) {
                    v[e] = -INFINITY;
                    ++pos;
                }
        }
        acc.template add<n>(v, j, L, slack);
    };
    const int tid = threadIdx.x, T = blockDim.x;
    int j = row.full0 + tid;
    // every thread meets its vectors in ascending order
    if (row.head && tid == 0) {
        float v[n];
        row.ragged(0, v);
        acc.at = 0;
        take(0, v);
    } else if (j < row.full1) {
        acc.at = j;
    } else if (row.last && tid == T - 1) {
        acc.at = row.full1;
    }
    for (; j + (kUnroll - 1) * T < row.full1; j += kUnroll * T) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = row.full(j + u * T);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float v[n];
            Vec<E>::unpack(w[u], v);
            take(j + u * T, v);
        }
    }
    for (; j < row.full1; j += T) {
        float v[n];
        Vec<E>::unpack(row.full(j), v);
        take(j, v);
    }
    if (row.last && tid == T - 1) {
        float v[n];
        row.ragged(row.full1, v);
        take(row.full1, v);
    }
}

// Where one token holds nearly all the mass, 1 + rest in f32 keeps little of the rest, and
// ln(1 + rest) and the entropy are all rest.  For such rows one warp sums the vectors of
// the thread that met the maximum `m` once more, leaving the maximum out; the other
// threads' sums hold nothing of it.  Returns the sums over that thread's other elements.
constexpr float kPeaked = 1.0625f;

template <typename E>
__device__ void sum_without_maximum(const Row<E>& row, int owner, float m, float L, float& S, float& W) {
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
    for (long long j = (long long)row.full0 + owner + (long long)lane * T; j < row.full1; j += 32ll * T) {
        Vec<E>::unpack(row.full((int)j), v);
        take(v);
    }
    if (lane == 0 && row.head && owner == 0) {
        row.ragged(0, v);
        take(v);
    }
    if (lane == 0 && row.last && owner == T - 1) {
        row.ragged(row.full1, v);
        take(v);
    }
    S = warp_allsum(s);
    W = warp_allsum(w);
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

struct Selection {
    alignas(16) unsigned long long keys[kListCap];
    alignas(16) unsigned long long group[kMaxGroups];
    unsigned long long best[kMaxSlots];
    unsigned long long threshold;
    int rescan[kRowThreads];
    int count, rescans;
};

// The `top` largest of keys[0..n) (all distinct), in descending order, into best and
// to the front of keys; returns how many there are.  Ends with the block synchronised.
__device__ int rank_keys(Selection& P, int n, int top) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const unsigned long long key = P.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += P.keys[j] > key;
        if (rank < top) P.best[rank] = key;
    }
    __syncthreads();
    const int have = n < top ? n : top;
    for (int i = threadIdx.x; i < have; i += blockDim.x) P.keys[i] = P.best[i];
    __syncthreads();
    return have;
}

// The row's `top` best tokens, piece by piece: what beats the worst kept key joins the
// list, which is then cut to its best `top`.  Exact for any row.
template <typename E>
__device__ int select_by_pieces(Selection& P, const E* z, int vocab, int top) {
    int have = 0;
    const int piece = kListCap - kMaxSlots;
    for (int start = 0; start < vocab; start += piece) {
        if (threadIdx.x == 0) P.count = have;
        __syncthreads();
        const unsigned long long worst = have == top ? P.keys[top - 1] : 0ull;
        const int end = vocab - start < piece ? vocab : start + piece;
        for (int i = start + threadIdx.x; i < end; i += blockDim.x) {
            const unsigned long long key = order_key(Vec<E>::one(z[i]), (uint32_t)i);
            if (key > worst) P.keys[atomicAdd(&P.count, 1)] = key;
        }
        __syncthreads();
        const int n = P.count;
        if (n > have) have = rank_keys(P, n, top);
        __syncthreads();
    }
    return have;
}

// The row's `top` best tokens from what the threads met while they summed it.  The
// threads form groups; the `top`-th best of the groups' best vectors, ordered by (its
// largest logit, lower vector number first), bounds the row's `top`-th best element from
// below: `top` elements, one in each better group, are at least as good.  So only elements
// at or above that bound are candidates: about G ln(1 / (1 - top / G)) of them where the
// tokens lie at random over G groups.  They are read again (from L2) at the threads' best vectors, and in
// all vectors only of threads that have a second one to offer.  More candidates than the
// list holds (rows in order) are left to select_by_pieces.
template <typename E>
__device__ void select_by_threads(Selection& P, const Row<E>& row, const E* z, int top, float m, float second, int at) {
    constexpr int n = Vec<E>::n;
    const int tid = threadIdx.x, lane = tid & 31, T = blockDim.x;
    const int wide = top > 64 ? 2 : 4, groups = T / wide;
    const unsigned long long mine =
        at < 0 ? 0ull : ((unsigned long long)total_order_key(m + 0.f) << 32) | (0xffffffffu - (uint32_t)at);
    unsigned long long best = mine;
    for (int o = 1; o < wide; o <<= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (tid % wide == 0) P.group[tid / wide] = best;
    if (tid == 0) {
        P.threshold = 0ull;
        P.count = P.rescans = 0;
    }
    __syncthreads();
    if (tid < groups) {
        const unsigned long long key = P.group[tid];
        int above = 0;
        for (int i = 0; i < groups; i += 2) {
            const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(&P.group[i]);
            above += (pair.x > key) + (pair.y > key);
        }
        if (above == top - 1 && key != 0ull) P.threshold = key;
    }
    __syncthreads();
    const unsigned long long threshold = P.threshold;
    auto offer = [&](int j, const float* v) {
        const uint32_t low = 0xffffffffu - (uint32_t)j;
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const long long i = row.first(j) + e;
            const unsigned long long key = ((unsigned long long)total_order_key(v[e] + 0.f) << 32) | low;
            if (key >= threshold && i >= 0 && i < row.vocab) {
                const int pos = atomicAdd(&P.count, 1);
                if (pos < kListCap) P.keys[pos] = order_key(v[e], (uint32_t)i);
            }
        }
    };
    auto read = [&](int j, float* v) {
        if (j >= row.full0 && j < row.full1)
            Vec<E>::unpack(row.full(j), v);
        else
            row.ragged(j, v);
    };
    if (mine != 0ull && mine >= threshold) {
        float v[n];
        read(at, v);
        offer(at, v);
        if (total_order_key(second + 0.f) >= (uint32_t)(threshold >> 32)) P.rescan[atomicAdd(&P.rescans, 1)] = tid;
    }
    // the best vector of a rescanned thread was offered by the thread itself
    __shared__ int offered[kRowThreads];
    offered[tid] = at;
    __syncthreads();
    const int rescans = P.rescans;
    for (int q = tid >> 5; q < rescans; q += T >> 5) {
        const int who = P.rescan[q], skip = offered[who];
        float v[n];
        for (int j = row.full0 + who + lane * T; j < row.full1; j += 32 * T)
            if (j != skip) {
                read(j, v);
                offer(j, v);
            }
        if (lane == 0 && row.head && who == 0 && skip != 0) {
            row.ragged(0, v);
            offer(0, v);
        }
        if (lane == 0 && row.last && who == T - 1 && skip != row.full1) {
            row.ragged(row.full1, v);
            offer(row.full1, v);
        }
    }
    __syncthreads();
    if (P.count > kListCap) {
        select_by_pieces<E>(P, z, row.vocab, top);
        return;
    }
    rank_keys(P, P.count, top);
}

// ---- token_logprobs ------------------------------------------------------------------
template <typename E>
__global__ void __launch_bounds__(kRowThreads) token_logprobs_kernel(
    const E* __restrict__ logits, int vocab, size_t stride, double temperature, const uint32_t* __restrict__ tokens,
    int token_count, int top, LogprobOutputs out) {
    __shared__ BlockScratch scratch;
    __shared__ Selection selection;
    __shared__ int owner;
    const size_t r = blockIdx.x;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    const float L = (float)(1.4426950408889634 / temperature), slack = kSlack / L;
    Running<true, true> acc;
    stream_row<E, false>(row, nullptr, L, slack, acc);
    const float m = block_max(acc.m, scratch.f[0]);
    acc.rebase(m, L);
    float S = block_sum(acc.S, scratch.f[1]);
    float W = block_sum(acc.W, scratch.f[2]);
    const bool empty = S == 0.f;  // every logit is -inf
    float log_sum = empty ? 0.f : logf(S);
    if (!empty && S < kPeaked) {  // the maximum is unique
        if (acc.m == m) owner = threadIdx.x;
        __syncthreads();
        float s = 0.f, w = 0.f;
        if (threadIdx.x < 32) sum_without_maximum(row, owner, m, L, s, w);
        const bool mine = (int)threadIdx.x == owner;
        s = (mine ? 0.f : acc.S) + (threadIdx.x == 0 ? s : 0.f);
        w = (mine ? 0.f : acc.W) + (threadIdx.x == 0 ? w : 0.f);
        s = block_sum(s, scratch.f[0]);
        W = block_sum(w, scratch.f[1]);
        S = 1.f + s;
        log_sum = log1pf(s);
    }
    const float inverse = (float)(1.0 / temperature);
    auto logprob = [&](float x) { return empty && x == x ? -INFINITY : (x - m) * inverse - log_sum; };
    if (threadIdx.x == 0) {
        if (out.entropy) out.entropy[r] = empty ? 0.f : log_sum - W / S * kLn2;
        if (out.stats) {
            out.stats[2 * r] = m;
            out.stats[2 * r + 1] = log_sum;
        }
    }
    if (out.logprob)
        for (int i = threadIdx.x; i < token_count; i += blockDim.x) {
            const uint32_t t = tokens[r * token_count + i];
            out.logprob[r * token_count + i] =
                t == kUnusedToken ? 0.f : t < (uint32_t)vocab ? logprob(Vec<E>::one(z[t])) : NAN;
        }
    if (top > 0) {
        if (S == S)
            select_by_threads<E>(selection, row, z, top, acc.m, acc.second, acc.at);
        else  // NaN or +inf in the row: NaN leads the order and the threads' maxima pass over it
            select_by_pieces<E>(selection, z, vocab, top);
        for (int i = threadIdx.x; i < top; i += blockDim.x) {
            const uint32_t id = key_id(selection.best[i]);
            const float x = key_logit(selection.best[i]);
            if (out.top_ids) out.top_ids[r * top + i] = id;
            if (out.top_logits) out.top_logits[r * top + i] = x;
            if (out.top_logprobs) out.top_logprobs[r * top + i] = logprob(x);
        }
    }
}

// ---- gradients ---------------------------------------------------------------------------
// What the gradient of one row needs: with y = (z - m) L - log2_sum an element gets
// 2^y (a + b y); a marked one, against its own log2_marked, 2^y (a_marked + b y) + its
// value.  `zero` rows get 0.
struct GradientRow {
    float m, log2_sum, a, b, log2_marked, a_marked;
    bool zero;
};

template <typename E>
__device__ __forceinline__ void gradient_vector(const Marks& M, const Row<E>& row, const GradientRow& g, float L, int j,
                                                float* v) {
    constexpr int n = Vec<E>::n;
    const bool look = marked(M, j);
    int pos = look ? mark_position(M, row.first(j)) : 0;
#pragma unroll
    for (int e = 0; e < n; ++e) {
        float a = g.a, offset = g.log2_sum, add = 0.f;
        if (look)
            while (pos < M.count && (long long)M.ids[pos] == row.first(j) + e) {
                add += M.value[pos];
                a = g.a_marked;
                offset = g.log2_marked;
                ++pos;
            }
        const float y = max_nan(fmaf(v[e] - g.m, L, -offset), kLowestExponent);
        v[e] = g.zero ? 0.f : fmaf(exp2_fast(y), fmaf(g.b, y, a), add);
    }
}

// Vectors [lo, hi) of the full ones, and the ragged ends where asked for.
template <typename E>
__device__ void write_gradient(const Marks& M, const Row<E>& row, E* out, const GradientRow& g, float L,
                               int lo, int hi, bool head, bool last) {
    constexpr int n = Vec<E>::n;
    const int tid = threadIdx.x, T = blockDim.x;
    // the output row may lie at another alignment than the logits
    const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == (uintptr_t)(row.lead * sizeof(E));
    E* base = out - row.lead;
    auto put = [&](int j, const float* v) {
        if (same) {
            *reinterpret_cast<uint4*>(base + (long long)j * n) = Vec<E>::pack(v);
        } else {
#pragma unroll
            for (int e = 0; e < n; ++e) base[(long long)j * n + e] = Vec<E>::store(v[e]);
        }
    };
    auto put_ragged = [&](int j) {
        float v[n];
        row.ragged(j, v);
        gradient_vector(M, row, g, L, j, v);
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const long long i = row.first(j) + e;
            if (i >= 0 && i < row.vocab) out[i] = Vec<E>::store(v[e]);
        }
    };
    int j = lo + tid;
    for (; j + (kUnroll - 1) * T < hi; j += kUnroll * T) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = row.full(j + u * T);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float v[n];
            Vec<E>::unpack(w[u], v);
            gradient_vector(M, row, g, L, j + u * T, v);
            put(j + u * T, v);
        }
    }
    for (; j < hi; j += T) {
        float v[n];
        Vec<E>::unpack(row.full(j), v);
        gradient_vector(M, row, g, L, j, v);
        put(j, v);
    }
    if (head && row.head && tid == 0) put_ragged(0);
    if (last && row.last && tid == T - 1) put_ragged(row.full1);
}

template <typename E>
__global__ void __launch_bounds__(kRowThreads) logprobs_gradient_kernel(
    const E* logits, int vocab, size_t stride, double temperature, const uint32_t* __restrict__ tokens, int token_count,
    const float* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ logprob_gradient,
    const float* __restrict__ entropy_gradient, E* gradient, size_t gradient_stride) {
    __shared__ Marks marks;
    __shared__ float total;
    const size_t r = blockIdx.x;
    const Row<E> row(logits + r * stride, vocab);
    build_marks(marks, tokens + r * token_count, token_count, row);
    const float inverse = (float)(1.0 / temperature);
    if (threadIdx.x < 32) {
        float sum = 0.f;
        for (int i = threadIdx.x; i < token_count; i += 32) {
            const int rank = marks.slot_rank[i];
            if (rank == -1) continue;
            const float v = logprob_gradient[r * token_count + i];
            marks.value[rank >= 0 ? rank : -2 - rank] = v * inverse;
            sum += v;
        }
        sum = warp_allsum(sum);
        if (threadIdx.x == 0) total = marks.bad ? NAN : sum;
    }
    __syncthreads();
    const float L = (float)(1.4426950408889634 / temperature);
    const float h = entropy_gradient ? entropy_gradient[r] : 0.f;
    GradientRow g;
    g.m = stats[2 * r];
    g.log2_sum = stats[2 * r + 1] * kLog2E;
    g.a = -(total + (h != 0.f ? h * entropy[r] : 0.f)) * inverse;
    g.b = -h * kLn2 * inverse;
    g.a_marked = g.a;
    g.log2_marked = g.log2_sum;
    g.zero = g.m == -INFINITY && stats[2 * r + 1] == 0.f;
    write_gradient(marks, row, gradient + r * gradient_stride, g, L, row.full0, row.full1, true, true);
}

// ---- distillation --------------------------------------------------------------------------
// The teacher's side of one row, by one warp, in 64 bits (its sums run over at most
// kMaxSlots numbers, and 1 - sum p is next to 0 for a confident teacher).
struct TeacherSums {
    double mass;  // sum of the listed p
    double rest;  // the teacher's mass outside the list (0 without its statistics)
};

struct TeacherSlots {
    double log_p[kMaxSlots];
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_max_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ TeacherSums teacher_row(const Marks& M, TeacherSlots& slots, const float* values, const float* stats,
                                   int count, double temperature) {
    const int lane = threadIdx.x & 31;
    double top = -INFINITY;
    for (int i = lane; i < count; i += 32)
        if (M.slot_rank[i] >= 0) top = fmax(top, (double)values[i]);
    top = warp_max_f64(top);
    double norm = 0.0, shift = top == -INFINITY ? 0.0 : top;
    if (stats) {
        shift = (double)stats[0];
        norm = (double)stats[1];
    } else {
        double sum = 0.0;
        for (int i = lane; i < count; i += 32)
            if (M.slot_rank[i] >= 0) sum += exp(((double)values[i] - shift) / temperature);
        sum = warp_sum_f64(sum);
        norm = sum > 0.0 ? log(sum) : (sum == 0.0 ? 0.0 : sum);
    }
    double mass = 0.0;
    for (int i = lane; i < count; i += 32) {
        const double log_p =
            M.slot_rank[i] >= 0 ? ((double)values[i] - shift) / temperature - norm : -INFINITY;
        slots.log_p[i] = log_p;
        mass += exp(log_p);
    }
    mass = warp_sum_f64(mass);
    __syncwarp();
    return {mass, stats ? (mass < 1.0 ? 1.0 - mass : (mass >= 1.0 ? 0.0 : mass)) : 0.0};
}

// The tokens outside the list are one outcome only where the student's share of them is
// a normal f32 number (2^-126 and up).
constexpr double kSmallestLogShare = -87.3365447505531;

// The gradient's coefficients from the sums; also fills the marked values.  The tokens
// outside the list are exponentiated against their own sum: 2^y = q_i / q_r stays in range
// and (P q_r - p_r) is the whole coefficient, however small q_r is.
__device__ GradientRow distill_gradient_row(Marks& M, const TeacherSlots& slots, const TeacherSums& t, int count,
                                            float m, double log_sum, double log_rest, bool zero, float weight,
                                            double temperature) {
    const double scale = (double)weight / temperature;
    const double log_share = log_rest - log_sum;
    const bool tail = log_share >= kSmallestLogShare;
    const double mass = t.mass + (tail ? t.rest : 0.0);
    for (int i = threadIdx.x & 31; i < count; i += 32) {
        const int rank = M.slot_rank[i];
        if (rank == -1) continue;
        M.value[rank >= 0 ? rank : -2 - rank] = rank >= 0 ? (float)(-scale * exp(slots.log_p[i])) : 0.f;
    }
    GradientRow g;
    g.m = m;
    g.log2_marked = (float)(log_sum * 1.4426950408889634);
    g.a_marked = M.bad ? NAN : (float)(scale * mass);
    g.log2_sum = tail ? (float)(log_rest * 1.4426950408889634) : g.log2_marked;
    g.a = M.bad ? NAN : (float)(scale * (tail ? mass * exp(log_share) - t.rest : mass));
    g.b = 0.f;
    g.zero = zero;
    return g;
}

// kStream: sums the row (loss, and optionally the gradient); otherwise the statistics
// are given and only the gradient is written.
template <typename E, bool kTail, bool kStream>
__global__ void __launch_bounds__(kRowThreads) distill_kernel(
    const E* logits, int vocab, size_t stride, double temperature, TeacherRows teacher,
    const float* __restrict__ weights, float* loss, float* stats, E* gradient, size_t gradient_stride) {
    __shared__ BlockScratch scratch;
    __shared__ Marks marks;
    __shared__ TeacherSlots slots;
    __shared__ GradientRow grow;
    __shared__ float listed[kMaxSlots];
    const size_t r = blockIdx.x;
    const int count = (int)teacher.slots;
    const E* z = logits + r * stride;
    const Row<E> row(z, vocab);
    build_marks(marks, teacher.ids + r * count, count, row);
    const double T = temperature;
    const float L = (float)(1.4426950408889634 / T), slack = kSlack / L;
    float m_rest = -INFINITY, S = 0.f;
    if (kStream) {
        for (int i = threadIdx.x; i < count; i += blockDim.x)
            listed[i] = marks.slot_rank[i] >= 0 ? Vec<E>::one(z[marks.raw[i]]) : -INFINITY;
        Running<false> acc;
        stream_row<E, true>(row, &marks, L, slack, acc);
        m_rest = block_max(acc.m, scratch.f[0]);
        acc.rebase(m_rest, L);
        S = block_sum(acc.S, scratch.f[1]);
    }
    if (threadIdx.x < 32) {
        const TeacherSums t = teacher_row(marks, slots, teacher.logits + r * count,
                                          kTail ? teacher.stats + 2 * r : nullptr, count, T);
        double m, log_sum, log_rest = -INFINITY;
        bool empty;
        if (kStream) {
            // the listed tokens' mass in f64, and the rest's around its own maximum
            double top = -INFINITY, inside = 0.0;
            bool nan = false;
            for (int i = threadIdx.x; i < count; i += 32) {
                top = fmax(top, (double)listed[i]);
                nan |= listed[i] != listed[i];
            }
            m = fmax((double)m_rest, warp_max_f64(top));
            for (int i = threadIdx.x; i < count; i += 32)
                if (marks.slot_rank[i] >= 0 && listed[i] != -INFINITY) inside += exp(((double)listed[i] - m) / T);
            inside = warp_sum_f64(inside);
            const double rest = S == 0.f ? 0.0 : (double)S * exp(((double)m_rest - m) / T);
            const double sum = __any_sync(0xffffffffu, nan) ? NAN : inside + rest;
            if (kTail) log_rest = S == 0.f ? -INFINITY : log((double)S) + ((double)m_rest - m) / T;
            empty = sum == 0.0;
            log_sum = empty ? 0.0 : log(sum);
            double part = 0.0;
            for (int i = threadIdx.x; i < count; i += 32) {
                const double log_p = slots.log_p[i], p = exp(log_p);
                if (p == 0.0) continue;
                const double log_q = empty ? -INFINITY : ((double)listed[i] - m) / T - log_sum;
                part += p * (log_p - log_q);
            }
            part = warp_sum_f64(part);
            if (kTail && t.rest > 0.0 && log_rest - log_sum >= kSmallestLogShare) part += t.rest * (log(t.rest) - log_rest + log_sum);
            if (threadIdx.x == 0) {
                if (loss) loss[r] = marks.bad || t.mass != t.mass || log_sum != log_sum ? NAN : (float)part;
                if (stats) {
                    stats[3 * r] = (float)m;
                    stats[3 * r + 1] = (float)log_sum;
                    stats[3 * r + 2] = (float)log_rest;
                }
            }
        } else {
            m = (double)stats[3 * r];
            log_sum = (double)stats[3 * r + 1];
            log_rest = (double)stats[3 * r + 2];
            empty = m == -INFINITY && log_sum == 0.0;
        }
        if (gradient) {
            const GradientRow g = distill_gradient_row(marks, slots, t, count, (float)m, log_sum, log_rest, empty,
                                                       weights ? weights[r] : 1.f, T);
            if (threadIdx.x == 0) grow = g;
        }
    }
    if (!gradient) return;
    __syncthreads();
    write_gradient(marks, row, gradient + r * gradient_stride, grow, L, row.full0, row.full1, true, true);
}

template <typename F>
cudaError_t by_kind(lsx_dtype kind, F&& f) {
    switch (kind) {
    case LSX_F32: return f((const float*)nullptr);
    case LSX_F16: return f((const __half*)nullptr);
    default: return f((const __nv_bfloat16*)nullptr);
    }
}

}  // namespace

cudaError_t launch_token_logprobs(cudaStream_t s, int, const LogitRows& z, const uint32_t* tokens, size_t token_count,
                                  size_t alternatives, const LogprobOutputs& out) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        token_logprobs_kernel<E><<<(unsigned)z.rows, kRowThreads, 0, s>>>(
            (const E*)z.data, (int)z.vocab, z.stride, z.temperature, tokens, (int)token_count, (int)alternatives, out);
        return cudaGetLastError();
    });
}

cudaError_t launch_logprobs_gradient(cudaStream_t s, int, const LogitRows& z, const uint32_t* tokens,
                                     size_t token_count, const float* stats, const float* entropy,
                                     const float* logprob_gradient, const float* entropy_gradient, void* gradient,
                                     size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        logprobs_gradient_kernel<E><<<(unsigned)z.rows, kRowThreads, 0, s>>>(
            (const E*)z.data, (int)z.vocab, z.stride, z.temperature, tokens, (int)token_count, stats, entropy,
            logprob_gradient, entropy_gradient, (E*)gradient, gradient_stride);
        return cudaGetLastError();
    });
}

cudaError_t launch_distill(cudaStream_t s, int, const LogitRows& z, const TeacherRows& teacher, const float* weights,
                           float* loss, float* stats, void* gradient, size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        auto kernel = teacher.stats ? distill_kernel<E, true, true> : distill_kernel<E, false, true>;
        kernel<<<(unsigned)z.rows, kRowThreads, 0, s>>>((const E*)z.data, (int)z.vocab, z.stride, z.temperature,
                                                        teacher, weights, loss, stats, (E*)gradient, gradient_stride);
        return cudaGetLastError();
    });
}

cudaError_t launch_distill_gradient(cudaStream_t s, int, const LogitRows& z, const TeacherRows& teacher,
                                    const float* stats, const float* weights, void* gradient, size_t gradient_stride) {
    return by_kind(z.kind, [&](auto* e) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(e)>>;
        auto kernel = teacher.stats ? distill_kernel<E, true, false> : distill_kernel<E, false, false>;
        kernel<<<(unsigned)z.rows, kRowThreads, 0, s>>>((const E*)z.data, (int)z.vocab, z.stride, z.temperature,
                                                        teacher, weights, nullptr, const_cast<float*>(stats),
                                                        (E*)gradient, gradient_stride);
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
