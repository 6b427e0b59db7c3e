// Log probabilities of given tokens, the entropy of every row's distribution and its most likely tokens, in one pass over the
// logits:
//
//   m = max x, Z = sum e^(x - m), log p(t) = x_t - m - ln Z, H = ln Z - sum e^(x - m) (x - m) / Z
//
// A row is one cluster of 1, 2, 4 or 8 blocks (few rows are cut so that they still fill the GPU); every thread keeps a running
// maximum with the two sums relative to it and, in float32 arithmetic on differences x - m, loses nothing to large logits. The
// blocks' sums meet in the first block's shared memory, added up in double in a fixed order: the same inputs give the same bits.
// ln Z is taken as log1p of the sum without the largest logit's own 1, which is why that logit's thread is summed
// again without it: a row whose first token has nearly all the weight keeps the digits of its small numbers.
//
// The k most likely (ties: the lowest index): a thread's largest logit is a 64-bit key (value, lowest index first); all that
// is among the block's k largest lies with the threads whose keys are among the k largest keys, and is no smaller than the
// smallest of these. Those threads' logits (a few hundred of them) are read again, what reaches the bound is ranked by
// counting, and the blocks' lists are ranked the same way in the first block.
#include "common.cuh"

#include <cooperative_groups.h>

namespace celeg_b200 {

constexpr int kLpThreads = 256;
constexpr int kLpMaxTop = 128;
constexpr int kLpPool = 1024;              // candidates of a block that are ranked at once
constexpr int kLpMaxBlocks = 8;            // of a cluster
constexpr int kLpUnits = 4;                // vectors a thread reads together
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
    static __device__ __forceinline__ void load(const float* p, float* x) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
};
template <> struct LpVector<__nv_bfloat16> {
    static constexpr int kSize = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* x) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
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

struct LpSums { float m, z, s; };      // maximum, sum of e^(x - m), sum of e^(x - m) (x - m)

template <int N>
__device__ __forceinline__ bool lp_add(LpSums& a, const float* x) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    const bool grown = top > a.m;
    if (grown) {
        const float d = lp_difference(a.m, top), f = lp_exp(d);
        a.s = f * fmaf(d, a.z, a.s);
        a.z *= f;
        a.m = top;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = lp_difference(x[i], a.m), e = lp_exp(d);
        a.z += e;
        a.s = fmaf(e, d, a.s);
    }
    return grown;
}

struct LpShared {
    LpKey keys[kLpThreads];                    // every thread's largest
    LpKey pool[kLpPool];
    LpKey lists[kLpMaxBlocks][kLpMaxTop];      // of the cluster's blocks (the first block's copy is the one used)
    double z[kLpMaxBlocks], s[kLpMaxBlocks];
    float m[kLpMaxBlocks];
    LpKey largest[kLpMaxBlocks];
    double warp_z[8], warp_s[8];
    LpKey warp_key[8];
    float warp_m[8];
    int selected[kLpThreads];
    int pooled, nan_seen;
    float row_max;
    LpKey bound;
};

__device__ __forceinline__ LpKey lp_key_max(LpKey key) {
#pragma unroll
    for (int lanes = 16; lanes > 0; lanes >>= 1) {
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

// A warp reads the logits of thread `owner` again: visit(index, value).
template <typename A, typename Visit>
__device__ __forceinline__ void lp_reread(const LpShare<A>& share, int owner, int lane, Visit visit) {
    constexpr int V = LpVector<A>::kSize;
    for (int i = owner + lane * kLpThreads; i < share.count; i += 32 * kLpThreads) {
        float x[V];
        const int index = share.vector_index(i);
        LpVector<A>::load(share.row + index, x);
#pragma unroll
        for (int e = 0; e < V; ++e) visit(index + e, x[e]);
    }
    if (lane == 0 && owner < share.edge) {
        const int index = share.edge_index(owner);
        visit(index, to_float(share.row[index]));
    }
}

// The `top` largest of the block's logits into `list`, largest first; 0 where there are fewer.
template <typename A>
__device__ __forceinline__ void lp_block_top(LpShared& sh, const LpShare<A>& share, const LpKey mine, const int top, LpKey* list) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    sh.keys[tid] = mine;
    if (tid == 0) sh.pooled = 0;
    if (tid < top) list[tid] = 0;
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < kLpThreads; i += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.keys[i]);
        rank += (two.x > mine) + (two.y > mine);
    }
    // (keys of threads without logits are 0 and rank behind all others; they have nothing to read)
    if (rank < top && mine != 0) sh.selected[rank] = tid;
    if (rank >= top || mine == 0) rank = -1;
    const int chosen = __syncthreads_count(rank >= 0);
    if (rank == chosen - 1 && chosen > 0) sh.bound = mine;
    __syncthreads();
    if (chosen == 0) return;
    LpKey bound = chosen == top ? sh.bound : 0;
    for (int w = warp; w < chosen; w += kLpThreads / 32)
        lp_reread<A>(share, sh.selected[w], lane, [&](int index, float x) {
            const LpKey key = lp_key(x, index);
            if (key >= bound) {
                const int at = atomicAdd(&sh.pooled, 1);
                if (at < kLpPool) sh.pool[at] = key;
            }
        });
    __syncthreads();
    const int pooled = sh.pooled;
    if (pooled <= kLpPool) {
        for (int i = tid; i < pooled; i += kLpThreads) {
            const LpKey key = sh.pool[i];
            int above = 0;
            for (int j = 0; j < pooled; ++j) above += sh.pool[j] > key;
            if (above < top) list[above] = key;
        }
        __syncthreads();
        return;
    }
    // More than the pool holds (large logits at a stride that gives them to a few threads): one after the other, each the
    // largest below the one before.
    LpKey before = ~0ull;
    for (int n = 0; n < top; ++n) {
        LpKey best = 0;
        for (int w = warp; w < chosen; w += kLpThreads / 32)
            lp_reread<A>(share, sh.selected[w], lane, [&](int index, float x) {
                const LpKey key = lp_key(x, index);
                if (key < before && key > best) best = key;
            });
        best = lp_key_max(best);
        if (lane == 0) sh.warp_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLpThreads / 32; ++w) best = sh.warp_key[w] > best ? sh.warp_key[w] : best;
        before = best;
        if (tid == 0) list[n] = best;
        __syncthreads();
    }
}

template <typename A>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p, const int blocks) {
    namespace cg = cooperative_groups;
    constexpr int V = LpVector<A>::kSize;
    __shared__ __align__(16) LpShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % blocks;
    const long long at = blockIdx.x / blocks;
    const LpShare<A> share(p, at, rank, blocks);
    if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");

    // ---- the pass over the logits
    LpSums mine = {-3.402823466e38f, 0.0f, 0.0f};
    int top_vector = -1;                        // the first vector group in which the thread's maximum stood
    for (int i0 = tid; i0 < share.count; i0 += kLpUnits * kLpThreads) {
        float x[kLpUnits * V];
        if (i0 + (kLpUnits - 1) * kLpThreads < share.count) {
#pragma unroll
            for (int u = 0; u < kLpUnits; ++u) LpVector<A>::load(share.row + share.vector_index(i0 + u * kLpThreads), x + u * V);
            if (lp_add<kLpUnits * V>(mine, x)) top_vector = i0;
        } else {
            for (int i = i0; i < share.count; i += kLpThreads) {
                LpVector<A>::load(share.row + share.vector_index(i), x);
                if (lp_add<V>(mine, x)) top_vector = i0;
            }
        }
    }
    bool top_edge = false;
    if (tid < share.edge) {
        const float x = to_float(share.row[share.edge_index(tid)]);
        top_edge = lp_add<1>(mine, &x);
    }
    // the thread's key: the lowest index at which its maximum stands
    LpKey key = 0;
    {
        int index = 0x7fffffff;
        if (top_vector >= 0)
            for (int u = kLpUnits - 1; u >= 0; --u) {
                const int i = top_vector + u * kLpThreads;
                if (i >= share.count) continue;
                float x[V];
                LpVector<A>::load(share.row + share.vector_index(i), x);
#pragma unroll
                for (int e = V - 1; e >= 0; --e)
                    if (x[e] == mine.m) index = share.vector_index(i) + e;
            }
        if (tid < share.edge) {
            const int e = share.edge_index(tid);
            if (top_edge || (to_float(share.row[e]) == mine.m && e < index)) index = e;
        }
        if (index != 0x7fffffff) {
            key = lp_key(mine.m, index);
        } else if (tid < share.count || tid < share.edge) {
            // nothing above the lowest finite number: the thread's lowest index stands for its logits (-inf, NaN or that number)
            key = 1;
        }
    }
    if (key == 1) {
        LpKey best = 0;
        for (int i = tid; i < share.count; i += kLpThreads) {
            float x[V];
            LpVector<A>::load(share.row + share.vector_index(i), x);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const LpKey k = lp_key(x[e], share.vector_index(i) + e);
                best = k > best ? k : best;
            }
        }
        if (tid < share.edge) {
            const LpKey k = lp_key(to_float(share.row[share.edge_index(tid)]), share.edge_index(tid));
            best = k > best ? k : best;
        }
        key = best;
    }

    // ---- the block's largest logit, and its sums relative to it
    {
        const LpKey best = lp_key_max(key);
        if (lane == 0) sh.warp_key[warp] = best;
        __syncthreads();
        LpKey block_best = sh.warp_key[0];
        for (int w = 1; w < kLpThreads / 32; ++w) block_best = sh.warp_key[w] > block_best ? sh.warp_key[w] : block_best;
        float m = mine.m;
        m = warp_max(m);
        if (lane == 0) sh.warp_m[warp] = m;
        __syncthreads();
        for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, sh.warp_m[w]);
        float z = mine.z, s = mine.s;
        if (key == block_best) z = s = 0.0f;           // (summed again below, without the largest itself)
        const float d = lp_difference(mine.m, m), f = expf(d);
        const double wz = lp_warp_sum((double)z * f), ws = lp_warp_sum((double)(f * fmaf(d, z, s)));
        if (lane == 0) {
            sh.warp_z[warp] = wz;
            sh.warp_s[warp] = ws;
        }
        if (key == block_best) sh.selected[0] = tid;
        // (another block's shared memory may be written once that block has begun)
        if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        __syncthreads();
        if (warp == 0) {
            const int skip = lp_index(block_best);
            float rz = 0.0f, rs = 0.0f;
            if (block_best != 0)
                lp_reread<A>(share, sh.selected[0], lane, [&](int index, float x) {
                    if (index == skip && x == m) return;
                    const float dx = lp_difference(x, m), e = lp_exp(dx);
                    rz += e;
                    rs = fmaf(e, dx, rs);
                });
            double tz = lp_warp_sum((double)rz), ts = lp_warp_sum((double)rs);
            if (lane == 0) {
                for (int w = 0; w < kLpThreads / 32; ++w) tz += sh.warp_z[w], ts += sh.warp_s[w];
                // (without the largest: its 1 is added where the blocks meet)
                cg::cluster_group cluster = cg::this_cluster();
                LpShared* first = blocks > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
                first->z[rank] = tz;
                first->s[rank] = ts;
                first->m[rank] = m;
                first->largest[rank] = block_best;
            }
        }
        __syncthreads();
    }
    if (p.top > 0) {
        lp_block_top<A>(sh, share, key, p.top, sh.lists[blocks > 1 ? kLpMaxBlocks - 1 : 0]);
    }
    if (blocks > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        // (the lists of all blocks go to the first one; its own list lies at its last place until then)
        if (p.top > 0) {
            LpKey* to = cluster.map_shared_rank(&sh, 0)->pool + rank * kLpMaxTop;
            const LpKey value = tid < p.top ? sh.lists[kLpMaxBlocks - 1][tid] : 0;
            if (tid < p.top) to[tid] = value;
        }
        cluster.sync();
        if (rank != 0) return;
    }

    // ---- the first block puts the row together
    if (tid == 0) {
        float m = sh.m[0];
        LpKey largest = sh.largest[0];
        for (int b = 1; b < blocks; ++b) {
            m = fmaxf(m, sh.m[b]);
            largest = sh.largest[b] > largest ? sh.largest[b] : largest;
        }
        double z = 0.0, s = 0.0;
        for (int b = 0; b < blocks; ++b) {
            // a block's largest is a 1 of its own sum, unless it is the row's largest
            const double own = sh.largest[b] == largest ? 0.0 : (sh.largest[b] >> 32 > 0x007fffffu ? 1.0 : 0.0);
            const double d = (double)lp_difference(sh.m[b], m), f = exp(d), bz = sh.z[b] + own;
            z += bz * f;
            s += f * (sh.s[b] + d * bz);
        }
        // a row without a logit above -inf has no distribution, nor has one with a logit of inf
        const bool none = (unsigned)(largest >> 32) <= 0x007fffffu || m == INFINITY;
        const double log_z = none ? nan("") : log1p(z);
        if (p.entropy) p.entropy[at] = (float)(log_z - s / (1.0 + z));
        if (p.logprobs) {
            const int token = p.tokens[at];
            const bool inside = token >= 0 && token < p.vocab;
            p.logprobs[at] = inside ? (float)((double)to_float(share.row[token]) - (double)m - log_z) : nanf("");
        }
        sh.row_max = m;
        sh.z[0] = log_z;
    }
    if (p.top == 0) return;
    __syncthreads();
    const double log_z = sh.z[0];
    const float m = sh.row_max;
    const LpKey* lists = blocks > 1 ? sh.pool : sh.lists[0];
    for (int i = tid; i < blocks * p.top; i += kLpThreads) {
        const LpKey k = lists[(i / p.top) * kLpMaxTop + i % p.top];
        if (k == 0) continue;
        int above = i % p.top;                          // (its own list is in order)
        if (blocks > 1)
            for (int b = 0; b < blocks; ++b) {
                if (b == i / p.top) continue;
                // how many of another list are above it: lists fall
                int low = 0, high = p.top;
                while (low < high) {
                    const int middle = (low + high) / 2;
                    if (lists[b * kLpMaxTop + middle] > k) low = middle + 1; else high = middle;
                }
                above += low;
            }
        if (above >= p.top) continue;
        const int index = lp_index(k);
        p.top_tokens[at * p.top + above] = index;
        p.top_logprobs[at * p.top + above] = (float)((double)to_float(share.row[index]) - (double)m - log_z);
    }
}

template <typename A>
static int launch_logprobs(const LogprobParams& p, int blocks, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((long long)p.rows * blocks));
    config.blockDim = dim3(kLpThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = blocks;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = blocks > 1 ? 1 : 0;
    const cudaError_t status = cudaLaunchKernelEx(&config, token_logprobs_kernel<A>, p, blocks);
    CELEG_REQUIRE(status == cudaSuccess, "token_logprobs: %s", cudaGetErrorString(status));
    return check_launch("token_logprobs");
}

}  // namespace celeg_b200

using namespace celeg_b200;

// logits: [rows, vocab] float32 or bfloat16, row_stride elements from row to row. tokens [rows] or null (no logprobs then);
// entropy [rows] or null; top_logprobs and top_tokens [rows, top].
CELEG_API int celeg_token_logprobs(const void* logits, long long row_stride, int rows, int vocab, const int* tokens,
                                   float* logprobs, float* entropy, float* top_logprobs, int* top_tokens, int top,
                                   int act_dtype, cudaStream_t stream) {
    CELEG_REQUIRE(rows >= 0 && vocab > 0 && vocab < (1 << 30) && (rows <= 1 || row_stride >= vocab),
                  "token_logprobs: invalid sizes rows=%d vocab=%d row_stride=%lld", rows, vocab, row_stride);
    CELEG_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= vocab && (top == 0 || (top_logprobs && top_tokens)),
                  "token_logprobs: %d alternatives (at most %d and the vocabulary of %d)", top, kLpMaxTop, vocab);
    CELEG_REQUIRE(!logprobs || tokens, "token_logprobs: log probabilities of no tokens");
    CELEG_REQUIRE(act_dtype == kFloat32 || act_dtype == kBFloat16, "token_logprobs: unknown dtype code %d", act_dtype);
    CELEG_REQUIRE(((size_t)logits & (act_dtype == kFloat32 ? 3 : 1)) == 0, "token_logprobs: logits at %p", logits);
    if (rows == 0) return 0;
    LogprobParams p = {};
    p.logits = logits;
    p.row_stride = row_stride;
    p.rows = rows;
    p.vocab = vocab;
    p.top = top;
    p.tokens = tokens;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.top_logprobs = top_logprobs;
    p.top_tokens = top_tokens;
    // few rows: up to eight blocks a row, as long as a block has 4,096 logits and the blocks fit on the GPU together
    int blocks = 1;
    while (blocks < kLpMaxBlocks && (long long)rows * blocks * 2 <= 592 && vocab / (blocks * 2) >= 4096) blocks *= 2;
    CELEG_REQUIRE((long long)rows * blocks <= 0x7fffffffll, "token_logprobs: %d rows exceed one launch", rows);
    return act_dtype == kFloat32 ? launch_logprobs<float>(p, blocks, stream) : launch_logprobs<__nv_bfloat16>(p, blocks, stream);
}
