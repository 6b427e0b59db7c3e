// Log probabilities of given tokens, the entropy of every row's distribution and its most likely tokens, in one pass over the
// logits:
//
//   m = max x, Z = sum e^(x - m), log p(t) = x_t - m - ln Z, H = ln Z - sum e^(x - m) (x - m) / Z
//
// A row is one cluster of 1, 2, 4 or 8 blocks (few rows are cut so that they still fill the GPU). Every thread keeps the largest
// logit so far, where it stands, and the two sums relative to it, of differences x - m, so that large logits cost no digits.
// The sum leaves the largest logit's own 1 out: ln Z is log1p of what is left, and a row whose first token has nearly all the
// weight keeps the digits of its small numbers. Sums over threads and blocks are taken in double and in a fixed order: the
// same inputs give the same bits.
//
// The k most likely (ties: the lowest index): a thread's largest logit is a 64-bit key (value, lowest index first), a group of 1 to
// 8 threads has the largest of its threads' keys, of which there are 256 to 32, at least 2 k. All that is among the block's k
// largest lies with the groups whose keys are among the k largest, and is no smaller than the smallest of these. Those groups'
// logits are read again, what reaches the bound is ranked by counting, and the blocks' lists are ranked the same way in the
// first block, where everything a block has meets.
//
// Over many rows the logits' bytes are what bounds it: 4,095 rows of 65,536 float32 logits take 162 us, 6,630 GB/s (in bfloat16
// 151 us: there the instructions a logit do). Of few rows, the chain of a block's reductions: 8.5 us for one row of 65,536 with its
// twenty best, 11 us for 64 of 50,257 with five.
#include "common.cuh"
#include "tcgen05.cuh"

#include <cstring>

namespace celeg_b200 {

constexpr int kLpThreads = 256;
constexpr int kLpMaxTop = 128;
constexpr int kLpPool = 1024;              // candidates of a block that are ranked at once
constexpr int kLpMaxBlocks = 8;            // of a cluster
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpFloor = -1.0e4f;        // differences below it count as it: e^-10000 is 0 in float32 and stays 0 times it

struct LogprobParams {
    const void* logits;
    long long row_stride;
    int rows, vocab, top;
    const int* tokens;             // [rows] or null
    float* logprobs;               // [rows] or null
    float* entropy;                // [rows] or null
    float* top_logprobs;           // [rows, top]
    int* top_tokens;               // [rows, top]
};

typedef unsigned long long LpKey;

// Larger logits have larger keys, equal ones by the lower index; -0 counts as 0 and NaN is below everything.
__device__ __forceinline__ LpKey lp_key(float x, int index) {
    const unsigned bits = __float_as_uint(x + 0.0f);
    const unsigned order = x != x ? 1u : (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
    return ((LpKey)order << 32) | (unsigned)(0x7fffffff - index);
}
__device__ __forceinline__ int lp_index(LpKey key) { return 0x7fffffff - (int)(unsigned)(key & 0xffffffffu); }
__device__ __forceinline__ float lp_value(LpKey key) {
    const unsigned order = (unsigned)(key >> 32);
    return order == 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
constexpr unsigned kLpOrderOfMinusInf = 0x007fffffu;        // the upper half of -inf's key, above NaN's, below all numbers'

__device__ __forceinline__ float lp_exp(float difference) {       // of a difference <= 0
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(difference * kLpLog2e));
    return e;
}

// x - m, not below kLpFloor; NaN stays NaN.
__device__ __forceinline__ float lp_difference(float x, float m) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x - m), "f"(kLpFloor));
    return d;
}

template <typename A> struct LpVector;
template <> struct LpVector<float> {
    static constexpr int kSize = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ void load(const float* p, float* x) { unpack(__ldcs(reinterpret_cast<const uint4*>(p)), x); }
};
template <> struct LpVector<__nv_bfloat16> {
    static constexpr int kSize = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* x) { unpack(__ldcs(reinterpret_cast<const uint4*>(p)), x); }
    static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// What a block reads of its row: whole vectors [first, first + count), of which thread t has first + t, first + t + 256, ...;
// and, in the cluster's last block, the `edge` single logits before the first and behind the last whole vector, thread t's the t-th.
template <typename A>
struct LpShare {
    static constexpr int V = LpVector<A>::kSize;
    const A* row;
    int head, vectors, vocab;          // logits before the first whole vector, whole vectors of the row
    int first, count, edge;
    __device__ __forceinline__ LpShare(const LogprobParams& p, long long at, int rank, int blocks) {
        row = static_cast<const A*>(p.logits) + at * p.row_stride;
        vocab = p.vocab;
        const int past = (int)(((unsigned long long)row & 15) / sizeof(A));
        head = min(past ? V - past : 0, vocab);
        vectors = (vocab - head) / V;
        const int per = (vectors + blocks - 1) / blocks;
        first = min(rank * per, vectors);
        count = min(per, vectors - first);
        edge = rank == blocks - 1 ? vocab - vectors * V : 0;
    }
    __device__ __forceinline__ int vector_index(int i) const { return head + (first + i) * V; }      // of the block's i-th vector
    __device__ __forceinline__ int edge_index(int i) const { return i < head ? i : vectors * V + i; }
};

// Of a thread's logits so far: the largest m, the sum z of e^(x - m) over all but one that is the largest (over all while none
// has exceeded the lowest finite number, which m starts from), the sum s of e^(x - m) (x - m), each in two halves that run side by
// side, and the index where m stood first.
struct LpSums {
    float m;
    unsigned long long z, s;
    int index;                     // -1: m has not been exceeded
};

// `index_of(e)`: where x[e] stands, rising with e. Where a lane of the warp has a larger logit (nearly always one of 32 has, in the
// tens of times that a thread comes here), only what goes with the larger one is done apart: the sums are brought to it, and
// its own place among x counts as far below. The exponentials are common to all lanes.
template <int N, typename IndexOf>
__device__ __forceinline__ void lp_add(LpSums& a, float (&x)[N], IndexOf index_of) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > a.m) {
        const float d = lp_difference(a.m, top), f = lp_exp(d), own = a.index >= 0 ? 1.0f : 0.0f;
        const unsigned long long all = add_f32x2(a.z, pack_f32x2(own, 0.0f)), f2 = pack_f32x2(f, f);
        a.s = mul_f32x2(f2, fma_f32x2(pack_f32x2(d, d), all, a.s));
        a.z = mul_f32x2(f2, all);
        a.m = top;
        int first = 0;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) first = x[i] == top ? i : first;
        a.index = index_of(first);
        const float far_below = top - fmaxf(-kLpFloor, 0.01f * fabsf(top));      // (far enough for any top; -inf is met below)
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i == first ? far_below : x[i];
    }
    const float m = a.m;
    if (N % 2 == 0) {
        const unsigned long long minus = pack_f32x2(-m, -m), log2e = pack_f32x2(kLpLog2e, kLpLog2e);
        unsigned long long z = a.z, s = a.s;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const unsigned long long d = add_f32x2(pack_f32x2(x[i], x[i + 1]), minus);
            float t0, t1, e0, e1;
            unpack_f32x2(mul_f32x2(d, log2e), t0, t1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t1));
            const unsigned long long e = pack_f32x2(e0, e1);
            z = add_f32x2(z, e);
            s = fma_f32x2(e, d, s);
        }
        float s0, s1;
        unpack_f32x2(s, s0, s1);
        if (s0 + s1 == s0 + s1) {
            a.z = z;
            a.s = s;
            return;
        }
    }
    // Differences cut off: a weight of 0 times a difference of -inf (a masked logit) is NaN above. (With the cut in the common
    // path, two more instructions a logit, 4,095 rows of 65,536 took 208 us instead of 180; rows masked all over take 260.)
    float z[2], s[2];
    unpack_f32x2(a.z, z[0], z[1]);
    unpack_f32x2(a.s, s[0], s[1]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = lp_difference(x[i], m), e = lp_exp(d);
        z[i % 2] += e;
        s[i % 2] = fmaf(e, d, s[i % 2]);
    }
    a.z = pack_f32x2(z[0], z[1]);
    a.s = pack_f32x2(s[0], s[1]);
}

struct LpShared {
    LpKey keys[kLpThreads];                    // the groups' largest
    LpKey pool[kLpPool];
    LpKey list[kLpMaxTop];                     // of this block
    LpKey lists[kLpMaxBlocks * kLpMaxTop];     // of the cluster's blocks, in the first one
    double z[kLpMaxBlocks], s[kLpMaxBlocks];
    float m[kLpMaxBlocks];
    LpKey largest[kLpMaxBlocks];
    double warp_z[8], warp_s[8];
    LpKey warp_key[8];
    float warp_m[8];
    int selected[kLpMaxTop];
    int pooled;
    float row_max, log_z;
    LpKey bound;
};

__device__ __forceinline__ LpKey lp_key_max(LpKey key, int from = 16) {
    for (int lanes = from; lanes > 0; lanes >>= 1) {
        const LpKey other = __shfl_xor_sync(0xffffffffu, key, lanes);
        key = other > key ? other : key;
    }
    return key;
}

__device__ __forceinline__ double lp_warp_sum(double v) {
#pragma unroll
    for (int lanes = 16; lanes > 0; lanes >>= 1) v += __shfl_xor_sync(0xffffffffu, v, lanes);
    return v;
}

// How many of `keys` (`count` of them, a multiple of 2) are above `key`.
__device__ __forceinline__ int lp_rank(const LpKey* keys, int count, LpKey key) {
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < count; i += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + i);
        rank += (two.x > key) + (two.y > key);
    }
    return rank;
}

// The logits of `chosen` groups of 2^shift threads, read again by all threads: visit(index, value).
template <typename A, typename Visit>
__device__ __forceinline__ void lp_reread(const LpShared& sh, const LpShare<A>& share, int chosen, int shift, Visit visit) {
    constexpr int V = LpVector<A>::kSize;
    const int rounds = (share.count + kLpThreads - 1) / kLpThreads, per_group = rounds << shift;
    for (int item0 = threadIdx.x; item0 < chosen * per_group; item0 += 4 * kLpThreads) {
        float x[4][V];
        int index[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int item = item0 + u * kLpThreads, group = item / per_group, rest = item % per_group;
            index[u] = -1;
            if (item >= chosen * per_group) continue;
            const int i = (sh.selected[group] << shift) + (rest & ((1 << shift) - 1)) + (rest >> shift) * kLpThreads;
            if (i >= share.count) continue;
            index[u] = share.vector_index(i);
            LpVector<A>::load(share.row + index[u], x[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (index[u] < 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) visit(index[u] + e, x[u][e]);
        }
    }
    for (int item = threadIdx.x; item < chosen << shift; item += kLpThreads) {
        const int owner = (sh.selected[item >> shift] << shift) + (item & ((1 << shift) - 1));
        if (owner < share.edge) {
            const int index = share.edge_index(owner);
            visit(index, to_float(share.row[index]));
        }
    }
}

// The `top` largest of the block's logits into sh.list, largest first; 0 where there are fewer.
template <typename A>
__device__ __forceinline__ void lp_block_top(LpShared& sh, const LpShare<A>& share, const LpKey mine, const int top) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // 32 groups of 8 threads for up to 16, ..., 256 of one for more than 64
    const int shift = top <= 16 ? 3 : top <= 32 ? 2 : top <= 64 ? 1 : 0, groups = kLpThreads >> shift;
    const LpKey group_key = shift > 0 ? lp_key_max(mine, 1 << (shift - 1)) : mine;
    if ((tid & ((1 << shift) - 1)) == 0) sh.keys[tid >> shift] = group_key;
    if (tid == 0) sh.pooled = 0;
    if (tid < top) sh.list[tid] = 0;
    __syncthreads();
    bool chosen_one = false;
    LpKey key = 0;
    int rank = 0;
    if (tid < groups) {
        key = sh.keys[tid];
        rank = lp_rank(sh.keys, groups, key);
        // (keys of groups without logits are 0 and rank behind all others; they have nothing to read)
        chosen_one = rank < top && key != 0;
        if (chosen_one) sh.selected[rank] = tid;
    }
    const int chosen = __syncthreads_count(chosen_one);
    if (chosen_one && rank == chosen - 1) sh.bound = key;
    __syncthreads();
    if (chosen == 0) return;
    const LpKey bound = chosen == top ? sh.bound : 0;
    lp_reread<A>(sh, share, chosen, shift, [&](int index, float x) {
        const LpKey k = lp_key(x, index);
        if (k >= bound) {
            const int at = atomicAdd(&sh.pooled, 1);
            if (at < kLpPool) sh.pool[at] = k;
        }
    });
    __syncthreads();
    const int pooled = sh.pooled;
    if (pooled <= kLpPool) {
        if (tid == 0 && (pooled & 1)) sh.pool[pooled] = 0;
        __syncthreads();
        for (int i = tid; i < pooled; i += kLpThreads) {
            const LpKey k = sh.pool[i];
            const int above = lp_rank(sh.pool, (pooled + 1) & ~1, k);
            if (above < top) sh.list[above] = k;
        }
        __syncthreads();
        return;
    }
    // More than the pool holds (large logits at a stride that gives them to a few threads): one after the other, each the
    // largest below the one before.
    LpKey before = ~0ull;
    for (int n = 0; n < top; ++n) {
        LpKey best = 0;
        lp_reread<A>(sh, share, chosen, shift, [&](int index, float x) {
            const LpKey k = lp_key(x, index);
            if (k < before && k > best) best = k;
        });
        best = lp_key_max(best);
        if (lane == 0) sh.warp_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLpThreads / 32; ++w) best = sh.warp_key[w] > best ? sh.warp_key[w] : best;
        before = best;
        if (tid == 0) sh.list[n] = best;
        __syncthreads();
    }
}

__device__ __forceinline__ unsigned lp_first_block(const void* shared) {       // the same place in the cluster's first block
    unsigned address;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(address) : "r"((unsigned)__cvta_generic_to_shared(shared)));
    return address;
}
__device__ __forceinline__ void lp_give(unsigned address, unsigned long long value) {
    asm volatile("st.shared::cluster.b64 [%0], %1;\n" ::"r"(address), "l"(value) : "memory");
}

template <typename A>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobParams p, const int blocks) {
    // a thread has four vectors under way, and takes 16 logits at a time
    constexpr int V = LpVector<A>::kSize, kUnits = 4, kAtOnce = 16 / V;
    __shared__ __align__(16) LpShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % blocks;
    const long long at = blockIdx.x / blocks;
    chain_release();
    chain_wait();
    const LpShare<A> share(p, at, rank, blocks);
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");

    // ---- the pass over the logits
    LpSums mine = {-3.402823466e38f, 0ull, 0ull, -1};
    {
        uint4 next[kUnits];
        auto load = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) next[u] = __ldcs(reinterpret_cast<const uint4*>(share.row + share.vector_index(i0 + u * kLpThreads)));
        };
        const int whole = share.count - (kUnits - 1) * kLpThreads;      // i0 below it: all units are there
        int i0 = tid;
        if (i0 < whole) load(i0);
        for (; i0 < whole; i0 += kUnits * kLpThreads) {
            uint4 now[kUnits];
#pragma unroll
            for (int u = 0; u < kUnits; ++u) now[u] = next[u];
            if (i0 + kUnits * kLpThreads < whole) load(i0 + kUnits * kLpThreads);
#pragma unroll
            for (int u0 = 0; u0 < kUnits; u0 += kAtOnce) {
                float x[16];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) LpVector<A>::unpack(now[u0 + u], x + u * V);
                lp_add(mine, x, [&](int e) { return share.vector_index(i0 + (u0 + e / V) * kLpThreads) + e % V; });
            }
        }
        for (; i0 < share.count; i0 += kLpThreads) {
            float x[V];
            LpVector<A>::load(share.row + share.vector_index(i0), x);
            lp_add(mine, x, [&](int e) { return share.vector_index(i0) + e; });
        }
    }
    if (tid < share.edge) {
        const int index = share.edge_index(tid);
        float x[1] = {to_float(share.row[index])};
        if (x[0] == mine.m && index < mine.index) mine.index = index;      // (as large, and before all whole vectors)
        lp_add(mine, x, [&](int) { return index; });
    }
    LpKey key = mine.index >= 0 ? lp_key(mine.m, mine.index) : 0;
    if (mine.index < 0 && (tid < share.count || tid < share.edge)) {
        // nothing above the lowest finite number: -inf, NaN or that number
        for (int i = tid; i < share.count; i += kLpThreads) {
            float x[V];
            LpVector<A>::load(share.row + share.vector_index(i), x);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const LpKey k = lp_key(x[e], share.vector_index(i) + e);
                key = k > key ? k : key;
            }
        }
        if (tid < share.edge) {
            const LpKey k = lp_key(to_float(share.row[share.edge_index(tid)]), share.edge_index(tid));
            key = k > key ? k : key;
        }
    }

    // ---- the block's largest logit, and its sums relative to it, without that logit
    LpKey block_best;
    {
        const LpKey best = lp_key_max(key);
        float m = warp_max(mine.m);
        if (lane == 0) {
            sh.warp_key[warp] = best;
            sh.warp_m[warp] = m;
        }
        __syncthreads();
        block_best = sh.warp_key[0];
        for (int w = 1; w < kLpThreads / 32; ++w) block_best = sh.warp_key[w] > block_best ? sh.warp_key[w] : block_best;
        for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, sh.warp_m[w]);
        // a thread's largest is a 1 of its own sum unless it is the block's (while nothing exceeded the start, it is in the sum)
        const float own = mine.index >= 0 ? 1.0f : 0.0f;
        float z0, z1, s0, s1;
        unpack_f32x2(mine.z, z0, z1);
        unpack_f32x2(mine.s, s0, s1);
        const float z_sum = z0 + z1;
        float z = z_sum + own;
        if (key == block_best && key >> 32 > kLpOrderOfMinusInf) z = mine.index >= 0 ? z_sum : z_sum - 1.0f;
        const float d = lp_difference(mine.m, m), f = expf(d);
        const double wz = lp_warp_sum((double)(z * f)), ws = lp_warp_sum((double)(f * fmaf(d, z, s0 + s1)));
        if (lane == 0) {
            sh.warp_z[warp] = wz;
            sh.warp_s[warp] = ws;
        }
        // (another block's shared memory may be written once that block has begun)
        if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            double tz = 0.0, ts = 0.0;
            for (int w = 0; w < kLpThreads / 32; ++w) tz += sh.warp_z[w], ts += sh.warp_s[w];
            lp_give(lp_first_block(&sh.z[rank]), (unsigned long long)__double_as_longlong(tz));
            lp_give(lp_first_block(&sh.s[rank]), (unsigned long long)__double_as_longlong(ts));
            lp_give(lp_first_block(&sh.largest[rank]), block_best);
            asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(lp_first_block(&sh.m[rank])), "f"(m) : "memory");
        }
    }
    if (p.top > 1) {
        lp_block_top<A>(sh, share, key, p.top);
        if (tid < p.top) lp_give(lp_first_block(&sh.lists[rank * p.top + tid]), sh.list[tid]);
    }
    if (blocks > 1)
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    else
        __syncthreads();
    if (rank != 0) return;

    // ---- the first block puts the row together
    if (warp == 0) {
        const bool one = lane < blocks;
        const LpKey own = one ? sh.largest[lane] : 0, largest = lp_key_max(own);
        const float own_m = one ? sh.m[lane] : -3.402823466e38f, m = warp_max(own_m);
        // a block's largest is a 1 of its own sum, unless it is the row's
        const double z_own = one ? sh.z[lane] + (own != largest && own >> 32 > kLpOrderOfMinusInf ? 1.0 : 0.0) : 0.0;
        const float d = lp_difference(own_m, m), f = expf(d);
        const double z = lp_warp_sum(z_own * f), s = lp_warp_sum(one ? f * (sh.s[lane] + d * z_own) : 0.0);
        if (lane == 0) {
            // a row without a logit above -inf has no distribution, nor has one with a logit of inf
            const bool none = (unsigned)(largest >> 32) <= kLpOrderOfMinusInf || m == INFINITY;
            const float log_z = none ? __uint_as_float(0x7fc00000u) : log1pf((float)z);
            if (p.entropy) p.entropy[at] = log_z - (float)(s / (1.0 + z));
            if (p.logprobs) {
                const int token = p.tokens[at];
                const bool inside = token >= 0 && token < p.vocab;
                p.logprobs[at] = inside ? to_float(share.row[token]) - m - log_z : __uint_as_float(0x7fc00000u);
            }
            sh.row_max = m;
            sh.log_z = log_z;
            if (p.top == 1) {
                p.top_tokens[at] = lp_index(largest);
                p.top_logprobs[at] = lp_value(largest) - m - log_z;
            }
        }
    }
    if (p.top <= 1) return;
    __syncthreads();
    const float log_z = sh.log_z, m = sh.row_max;
    const int entries = blocks * p.top;
    for (int i = tid; i < entries; i += kLpThreads) {
        const LpKey k = sh.lists[i];
        if (k == 0) continue;
        int above = i % p.top;                          // (its own list is in order)
        if (blocks > 1 && entries <= 256 && entries % 2 == 0) {
            above = lp_rank(sh.lists, entries, k);
        } else if (blocks > 1) {
            for (int b = 0; b < blocks; ++b) {
                if (b == i / p.top) continue;
                // how many of another list are above it: lists fall
                int low = 0, high = p.top;
                while (low < high) {
                    const int middle = (low + high) / 2;
                    if (sh.lists[b * p.top + middle] > k) low = middle + 1; else high = middle;
                }
                above += low;
            }
        }
        if (above >= p.top) continue;
        p.top_tokens[at * p.top + above] = lp_index(k);
        p.top_logprobs[at * p.top + above] = lp_value(k) - m - log_z;
    }
}

template <typename A>
static int launch_logprobs(const LogprobParams& p, int blocks, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((long long)p.rows * blocks));
    config.blockDim = dim3(kLpThreads);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = chaining_enabled() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {(unsigned)blocks, 1, 1};
    config.attrs = attributes;
    config.numAttrs = blocks > 1 ? 2 : 1;
    const cudaError_t status = cudaLaunchKernelEx(&config, token_logprobs_kernel<A>, p, blocks);
    CELEG_REQUIRE(status == cudaSuccess, "token_logprobs: %s", cudaGetErrorString(status));
    return check_launch("token_logprobs");
}

}  // namespace celeg_b200

using namespace celeg_b200;

// One record. logits: [rows, vocab] float32 or bfloat16, row_stride elements from row to row. tokens [rows] or null (no logprobs
// then); entropy [rows] or null; top_logprobs and top_tokens [rows, top].
CELEG_API int celeg_token_logprobs(const void* record) {
    struct {
        const void* logits;
        const int* tokens;
        float *logprobs, *entropy, *top_logprobs;
        int* top_tokens;
        cudaStream_t stream;
        long long row_stride;
        int rows, vocab, top, act_dtype;
    } a;
    static_assert(sizeof(a) == 80, "the record that kernels.py packs");
    memcpy(&a, record, sizeof(a));
    const int rows = a.rows, vocab = a.vocab, top = a.top, act_dtype = a.act_dtype;
    const long long row_stride = a.row_stride;
    cudaStream_t stream = a.stream;
    CELEG_REQUIRE(rows >= 0 && vocab > 0 && vocab < (1 << 30) && (rows <= 1 || row_stride >= vocab),
                  "token_logprobs: invalid sizes rows=%d vocab=%d row_stride=%lld", rows, vocab, row_stride);
    CELEG_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= vocab && (top == 0 || (a.top_logprobs && a.top_tokens)),
                  "token_logprobs: %d alternatives (at most %d and the vocabulary of %d)", top, kLpMaxTop, vocab);
    CELEG_REQUIRE(!a.logprobs || a.tokens, "token_logprobs: log probabilities of no tokens");
    CELEG_REQUIRE(act_dtype == kFloat32 || act_dtype == kBFloat16, "token_logprobs: unknown dtype code %d", act_dtype);
    CELEG_REQUIRE(((size_t)a.logits & (act_dtype == kFloat32 ? 3 : 1)) == 0, "token_logprobs: logits at %p", a.logits);
    if (rows == 0) return 0;
    LogprobParams p = {};
    p.logits = a.logits;
    p.row_stride = row_stride;
    p.rows = rows;
    p.vocab = vocab;
    p.top = top;
    p.tokens = a.tokens;
    p.logprobs = a.logprobs;
    p.entropy = a.entropy;
    p.top_logprobs = a.top_logprobs;
    p.top_tokens = a.top_tokens;
    // few rows: up to eight blocks a row, as long as a block has 4,096 logits and the blocks fit on the GPU together
    int blocks = 1;
    while (blocks < kLpMaxBlocks && (long long)rows * blocks * 2 <= 592 && vocab / (blocks * 2) >= 4096) blocks *= 2;
    CELEG_REQUIRE((long long)rows * blocks <= 0x7fffffffll, "token_logprobs: %d rows exceed one launch", rows);
    return act_dtype == kFloat32 ? launch_logprobs<float>(p, blocks, stream) : launch_logprobs<__nv_bfloat16>(p, blocks, stream);
}
