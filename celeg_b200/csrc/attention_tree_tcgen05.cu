// Attention of a tree of drafted tokens over the paged cache on the fifth-generation tensor cores: bfloat16, head sizes that are
// multiples of 8 up to 256, pages of any size (see attention_tree.cuh for the operator).
//
//   grid = (row tiles x pieces of the keys, kv heads, spans). A row is a (node, query head of the group) of one kv head, so that
//   a key is read once for a whole group and tree; keys come in blocks of 64, a piece is a run of whole blocks.
//   Fourteen warps, one block an SM. Two teams, each of a warp that issues its products (tcgen05.mma: S = Q K^T, and O += P V
//   with P from tensor memory and V as it lies in the cache) and four warps of softmax, a thread a row. A row tile has 128
//   rows and the teams take its even and odd blocks of keys, with outputs, maxima and sums of their own; or, where there are
//   more rows, 256 rows, a team 128 of them, and every block of keys serves both teams. (Above a head size of 128 the outputs of
//   one team fill the tensor memory: the first team works alone.) A team's S and P exist twice, so that its
//   products run while its softmax is busy with another block. A step of the softmax is a chain of waits around its
//   exponentials, which the two teams hide from one another.
//   Four warps copy K and V: rows of 16-byte pieces by cp.async, written in the layout with the 128-byte swizzle that the
//   products want. (By TMA, a box a page, a page of 16 positions x 64 took 110 cycles whoever asked for it, 880 cycles for a
//   block of 16 KiB of K and V; these copies take 320, and at 6.9 TB/s the memory gives an SM a block in 660.) What holds no key
//   of the span arrives as zeros.
//   At the end the teams' results meet in shared memory, and those of up to eight pieces of the keys, which are a cluster, in
//   one another's; more pieces go through scratch and a second launch.
//
// What bounds it: where blocks of keys are many, the softmax. An SM takes 16 exponentials a cycle, 512 cycles for 128 rows x 64
// keys, and the step of a team (scores from tensor memory, scaling, exponentials, packing, weights to tensor memory) is a chain
// that two teams cover to 850 cycles. Four trees of 64 nodes on 32 heads of 64 behind 65,536 positions: 239 us, 575 TFLOP/s,
// 2.3 TB/s, the special-function pipe at 59 % and the tensor pipe at 29 % of their rates. Where they are few, the chain from the launch to the last store, about 9 us: one tree of 13 nodes behind 601 positions
// 9.7 us. Eight trees of up to 32 nodes behind 1,161 to 4,096 positions, in clusters of two: 27 us, as long as the longest takes.
// (Times in a graph, inputs in turn.)
//
// Blocks of keys before the tree are seen whole by every row and need no mask. In the others a row's mask is 64 bits, cut from
// its words of ancestors; a value that is not finite is taken out there and added to the rows that do see it at the end (a weight
// of zero times it would reach the others).
//
// The weights are rounded to bfloat16 for their product with V (the denominator adds them up before): 2^-8 of each at most, at random.
// Warps without rows take no exponentials.
#include "attention_tree.cuh"
#include "attention_tree_tcgen05.h"
#include "tcgen05.cuh"

#include <atomic>

namespace celeg_b200 {

constexpr int kTtCopyWarps = 4;           // a pair of them brings every other block
constexpr int kTtSoftmaxFirst = kTtCopyWarps + 2;
constexpr int kTtThreads = 32 * (kTtSoftmaxFirst + 8);
constexpr int kTtM = 128;                 // rows of a team
constexpr int kTtN = 64;                  // keys per block
constexpr int kTtMaxCluster = 8;          // pieces of the keys that meet in shared memory
constexpr unsigned kTtTmemColumns = 512;

// D: the head size padded to 64, 128 or 256. Rows lie in shared memory in parts of 64 numbers (a swizzled row is 128 bytes).
template <int D, bool PAIRED>
struct TtLayout {
    static constexpr int kHalves = D / 64;
    static constexpr unsigned kQHalf = kTtM * 128, kKvHalf = kTtN * 128;
    static constexpr unsigned kQBytes = kHalves * kQHalf;       // 16 or 32 KiB a team
    static constexpr unsigned kKvBytes = kHalves * kKvHalf;     // 8 or 16 KiB each for a block's K and V
    static constexpr bool kAlone = D == 256;                    // one team
    static constexpr int kStages = D == 64 ? 12 : kAlone ? 2 : PAIRED ? 5 : 6;
    static constexpr unsigned kAllQ = PAIRED ? 2 * kQBytes : kQBytes;
    static constexpr unsigned kSmemBytes = kAllQ + kStages * 2 * kKvBytes + 1024;      // 193 to 225 KiB
    // what meets at the end lies where queries and keys were: rows of results (16-byte pieces of eight rows in different banks),
    // 128 a team and one more of every part, their maxima and sums, the rows' (token, query head) numbers
    static constexpr int kPitch = D + 4, kMeetRows = (kAlone ? 1 : 2) * (kTtM + kTtMaxCluster);
    static constexpr unsigned kStatsAt = kMeetRows * kPitch * 4, kUnitsAt = kStatsAt + kMeetRows * 8;
    static_assert(kUnitsAt + 2 * kTtM * 4 + 1024 <= kSmemBytes, "the results meet where queries and keys were");
    // Tensor memory of a team: scores of its even and odd blocks at columns 0 and 64, O from 128 on, the weights behind O at a
    // head size of 64 and over the scores they were made of above.
    static constexpr unsigned kTeamColumns = kAlone ? 0 : 256, kOColumn = 2 * kTtN;
    static constexpr bool kOverScores = D > 64;
    static __device__ __forceinline__ unsigned p_column(int n) {
        return kOverScores ? (unsigned)((n & 1) * kTtN) : 2 * kTtN + D + (unsigned)((n & 1) * (kTtN / 2));
    }
};

__device__ __forceinline__ unsigned pack_bf16_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The place that `address` is in block `rank`'s shared memory, or in this block's own.
__device__ __forceinline__ unsigned peer_address(unsigned address, unsigned rank, bool other) {
    unsigned peer;
    if (other)
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(peer) : "r"(address), "r"(rank));
    else
        asm volatile("{\n\t.reg .u32 own;\n\tmov.u32 own, %%cluster_ctarank;\n\tmapa.shared::cluster.u32 %0, %1, own;\n\t}\n" : "=r"(peer) : "r"(address));
    return peer;
}
__device__ __forceinline__ void store_2(unsigned peer, float a, float b) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};\n" ::"r"(peer), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void store_4(unsigned peer, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(peer), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}

// The keys key_base .. key_base + 63 that a row sees, a bit each.
__device__ __forceinline__ unsigned long long tree_visible(const TreeParams& p, const TreeSpan& s, const unsigned* mask, int position,
                                                           int key_base) {
    const int cached = s.context - key_base;                    // bits below it are cached places
    unsigned long long seen = 0;
    if (cached > 0) {
        seen = cached >= 64 ? ~0ull : (1ull << cached) - 1;
        if (p.window) {
            const long long first = (long long)position - p.window + 1 - key_base;
            if (first > 0) seen &= first >= 64 ? 0ull : ~0ull << first;
        }
    }
    if (cached < 64) {
        const int from = cached > 0 ? 0 : -cached;              // the first node of the block
        unsigned long long nodes = 0;
        if (from < s.nodes) {
            const int word = from >> 5, shift = from & 31;
            unsigned w[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) w[i] = word + i < p.words ? __ldg(mask + word + i) : 0u;
            nodes = (unsigned long long)__funnelshift_r(w[0], w[1], shift) | ((unsigned long long)__funnelshift_r(w[1], w[2], shift) << 32);
            if (s.nodes - from < 64) nodes &= (1ull << (s.nodes - from)) - 1;
            if (p.window)
                for (unsigned long long left = nodes; left; left &= left - 1) {
                    const int j = __ffsll((long long)left) - 1;
                    if ((long long)p.positions[s.begin + from + j] <= (long long)position - p.window) nodes &= ~(1ull << j);
                }
        }
        seen |= cached > 0 ? nodes << cached : nodes;
    }
    return seen;
}

__device__ __forceinline__ bool not_finite(unsigned bf16_bits) { return (bf16_bits & 0x7f80u) == 0x7f80u; }

// 32 scores of a row to their weights relative to `base` (scores times `to_log2`), packed in pairs of bfloat16; returns the sum
// of the weights. LARGEST: finds the largest of these scores and the 32 behind them on the way.
template <bool LARGEST>
__device__ __forceinline__ float tree_weights(const float* sc, unsigned long long scale2, unsigned long long neg_base2, unsigned (&packed)[16],
                                              float& largest) {
    unsigned long long sums[4] = {0ull, 0ull, 0ull, 0ull};      // (0.0f, 0.0f) each
    float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j2 = 0; j2 < 16; ++j2) {
        float x0, x1, a, b;
        if (LARGEST) {
            tops[0] = max3_f32(tops[0], sc[2 * j2], sc[2 * j2 + 1]);
            tops[1] = max3_f32(tops[1], sc[32 + 2 * j2], sc[32 + 2 * j2 + 1]);
        }
        unpack_f32x2(fma_f32x2(pack_f32x2(sc[2 * j2], sc[2 * j2 + 1]), scale2, neg_base2), x0, x1);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(x0));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(x1));
        sums[j2 & 3] = add_f32x2(sums[j2 & 3], pack_f32x2(a, b));
        packed[j2] = pack_bf16_pair(a, b);                      // (key 2 j2 in the lower half)
    }
    if (LARGEST) largest = fmaxf(tops[0], tops[1]);
    float s0, s1;
    unpack_f32x2(add_f32x2(add_f32x2(sums[0], sums[1]), add_f32x2(sums[2], sums[3])), s0, s1);
    return s0 + s1;
}

// PAIRED: row tiles of 256 rows, a team a half of them, every block of keys for both; otherwise of 128 rows, a team every other block.
template <int D, bool PAIRED>
__global__ void __launch_bounds__(kTtThreads, 1) attention_tree_tcgen05_kernel(const TreeParams p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    using L = TtLayout<D, PAIRED>;
    constexpr int kStages = L::kStages, kTileRows = PAIRED ? 2 * kTtM : kTtM;
    __shared__ __align__(8) unsigned long long kv_full[kStages], kv_empty[kStages], q_full[2], s_full[2][2], p_full[2][2], o_full[2][2];
    __shared__ unsigned tmem_base_slot;
    __shared__ int lowest_s, highest_s, bad_values;

    // (the warp's number comes from a shuffle so that what follows from it is known to be the same in all lanes: descriptors and
    // addresses of the products are then made once, in uniform registers)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int span = blockIdx.z, kvh = blockIdx.y;
    const int row0 = (blockIdx.x / p.splits) * kTileRows, split = blockIdx.x % p.splits;
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&kv_full[i]), 64);
            mbar_init(smem_u32(&kv_empty[i]), PAIRED ? 2 : 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_u32(&q_full[t]), 128);
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(&s_full[t][b]), 1);
                mbar_init(smem_u32(&p_full[t][b]), 128);
                mbar_init(smem_u32(&o_full[t][b]), 1);
            }
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        lowest_s = 0x7fffffff;
        highest_s = -0x7fffffff - 1;
        bad_values = 0;
    }
    if (warp == kTtCopyWarps) tmem_alloc(smem_u32(&tmem_base_slot), kTtTmemColumns);
    chain_release();
    chain_wait();                                               // (what comes before this line may run under the kernel before)
    const TreeSpan s = tree_span(p, span);
    const int rows = min(s.nodes * p.group - row0, kTileRows);  // (of a whole cluster alike)
    const int d = p.head_dim;

    const bool softmax = warp >= kTtSoftmaxFirst;
    const int team = softmax ? (warp - kTtSoftmaxFirst) >> 2 : warp < kTtCopyWarps ? warp >> 1 : warp - kTtCopyWarps;
    // a softmax thread's row; a warp may touch the 32 lanes of tensor memory that its number gives
    const int lane_row = (warp & 3) * 32 + lane, row = lane_row + (PAIRED ? team * kTtM : 0);
    const bool live = softmax && row < rows;
    const int node = rows > 0 ? s.begin + (row0 + min(row, rows - 1)) / p.group : 0;
    const int head = rows > 0 ? kvh * p.group + (row0 + min(row, rows - 1)) % p.group : 0;
    constexpr int kQueryPieces = PAIRED ? D / 8 : D / 16;       // 16-byte pieces of its query a thread brings: a row, or half of one
    uint4 query[kQueryPieces];                                  // (under way while the block sets up)
    if (softmax) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + (size_t)node * p.q_row_stride + (size_t)head * d);
#pragma unroll
        for (int c0 = 0; c0 < kQueryPieces; ++c0) {
            const int c = PAIRED ? c0 : team * kQueryPieces + c0;
            query[c0] = live && 8 * c < d ? __ldg(q + c) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const int position = p.window && rows > 0 ? p.positions[node] : 0;
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const unsigned tmem_base = tmem_base_slot;
    if (rows <= 0) {
        if (warp == kTtCopyWarps) tmem_dealloc(tmem_base, kTtTmemColumns);
        return;
    }
    if (p.window) {
        if (live) {
            atomicMin(&lowest_s, position);
            atomicMax(&highest_s, position);
        }
        __syncthreads();
    }
    const int first_key = p.window ? tree_first_place(p, s, lowest_s) : 0;
    const int last_key = s.context + s.nodes - 1;
    // blocks below `edge` or with places from the context's end on have keys that some rows see and others do not
    const int edge = p.window ? tree_first_place(p, s, highest_s) : 0;
    const int all_begin = first_key / kTtN, all_end = last_key / kTtN + 1;
    const int per_split = (all_end - all_begin + p.splits - 1) / p.splits;
    const int block_begin = all_begin + split * per_split;
    const int blocks = max(0, min(per_split, all_end - block_begin));
    // the team's n-th block is the piece's block kStride n + kFirst
    constexpr int kStride = PAIRED || L::kAlone ? 1 : 2;
    const int first_block = kStride == 1 ? 0 : team;
    const int mine = PAIRED ? blocks : L::kAlone ? (team == 0 ? blocks : 0) : (blocks + 1 - team) / 2;
    const bool idle = PAIRED && team * kTtM >= rows;            // (a team without rows still gives its share of the stages back)

    const unsigned smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const unsigned q_addr = smem_base + (PAIRED ? team * L::kQBytes : 0);
    const unsigned k_addr = smem_base + L::kAllQ, v_addr = k_addr + kStages * L::kKvBytes;
    const unsigned* mask = p.ancestors + (size_t)node * p.words;
    const unsigned team_base = tmem_base + (unsigned)team * L::kTeamColumns;
    const unsigned row_base = team_base + ((unsigned)((warp & 3) * 32) << 16);

    int error = 0;
    float used_max = -INFINITY, run_sum = 0.0f;
    auto wait = [&](unsigned long long& bar, int parity) {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), (unsigned)parity)) != 0;
    };
    if (warp < kTtCopyWarps) {
        // ------------------------------------------------------------------------------ K and V, block by block
        // A pair of warps brings every other block: a thread has one 16-byte piece of every eighth row of K and of V.
        const int pair = warp >> 1, thread = tid & 63;
        const int piece = thread & 7, row_in_8 = thread >> 3;
        const unsigned to = (unsigned)row_in_8 * 128u + (unsigned)((piece ^ row_in_8) << 4);
        const int* table = p.block_table + (size_t)span * p.table_stride;
        const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(p.k_cache) + piece * 8 + (size_t)kvh * p.page_tokens * d;
        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v_cache) + piece * 8 + (size_t)kvh * p.page_tokens * d;
        bool ok = true;
        auto begin_block = [&](int i) {                         // its stage is free
            return i < kStages || wait(kv_empty[i % kStages], ((i / kStages) - 1) & 1);
        };
        auto end_block = [&](int i) {                           // the barrier counts this thread when its copies so far have landed
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(&kv_full[i % kStages])) : "memory");
        };
        // one piece of a row of K and of V (of both halves of it), or zeros
        auto copy = [&](unsigned k_to, unsigned v_to, const __nv_bfloat16* k_from, const __nv_bfloat16* v_from, bool there) {
#pragma unroll
            for (int half = 0; half < L::kHalves; ++half) {
                const bool some = there && half * 64 + piece * 8 < d;
                const unsigned bytes = some ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(k_to + half * L::kKvHalf), "l"(some ? k_from + half * 64 : k), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(v_to + half * L::kKvHalf), "l"(some ? v_from + half * 64 : v), "r"(bytes) : "memory");
            }
        };
        if (p.page_shift >= 3) {
            // Pages of a power of two positions, eight at least: eight rows of a block are consecutive in a page. The table is
            // read 32 entries at a time, a lane each, and a round ahead: an entry a block would be a round trip to the L2 a
            // block. (With an address of its own for every row the instructions of the copies were what bounded the kernel.)
            const int first_page = block_begin * kTtN >> p.page_shift, last_page = last_key >> p.page_shift, in_page = p.page_tokens - 1;
            auto entries = [&](int round) -> int {
                const int logical = first_page + round * 32 + lane;
                return logical <= last_page && logical < p.table_columns ? table[logical] : -1;
            };
            const unsigned stride = (unsigned)p.page_stride;    // (fits: see tree_tcgen05_takes)
            int held = entries(0), ahead = entries(1), round = 0;
            for (int i = pair; i < blocks; i += 2) {
                const int key_base = (block_begin + i) * kTtN, index = (key_base >> p.page_shift) - first_page;
                if (index >> 5 != round) {
                    held = ahead;
                    ahead = entries(++round + 1);
                }
                ok = begin_block(i);
                if (!ok) break;
                const unsigned stage_at = (unsigned)(i % kStages) * L::kKvBytes + to, k_to = k_addr + stage_at, v_to = v_addr + stage_at;
                const int pages = max(1, kTtN >> p.page_shift);
                const bool good = (unsigned)(lane - (index & 31)) >= (unsigned)pages || (unsigned)held < (unsigned)p.pages;
                if (__all_sync(0xffffffffu, good) && key_base >= first_key && key_base + kTtN - 1 <= last_key) {
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const unsigned page = (unsigned)__shfl_sync(0xffffffffu, held, index + (u * 8 >> p.page_shift));
                        const size_t offset = (size_t)page * stride + (unsigned)((((key_base + u * 8) & in_page) + row_in_8) * d);
                        copy(k_to + u * 1024u, v_to + u * 1024u, k + offset, v + offset, true);
                    }
                } else {
                    for (int u = 0; u < 8; ++u) {
                        const int key = key_base + u * 8 + row_in_8;
                        const int page = __shfl_sync(0xffffffffu, held, index + (u * 8 >> p.page_shift));
                        const bool wanted = key >= first_key && key <= last_key, there = wanted && (unsigned)page < (unsigned)p.pages;
                        if (wanted && !there) atomicExch(p.error_flag, 2);
                        const size_t offset = there ? (size_t)(unsigned)page * stride + (unsigned)((key & in_page) * d) : 0;
                        copy(k_to + u * 1024u, v_to + u * 1024u, k + offset, v + offset, there);
                    }
                }
                end_block(i);
            }
        } else {
            // any other pages: a lane looks up two of a block's 64 keys, a block of its pair ahead
            auto look_up = [&](int i, int u) -> int {
                const int key = (block_begin + i) * kTtN + u * 32 + lane;
                if (i >= blocks || key < first_key || key > last_key) return -2;
                const int logical = key / p.page_tokens;
                return logical < p.table_columns ? table[logical] : -1;
            };
            int page[2] = {look_up(pair, 0), look_up(pair, 1)};
            for (int i = pair; i < blocks; i += 2) {
                long long offsets[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int key = (block_begin + i) * kTtN + u * 32 + lane;
                    offsets[u] = -1;
                    if (page[u] >= 0 && page[u] < p.pages) offsets[u] = (long long)page[u] * p.page_stride + (long long)(key % p.page_tokens) * d;
                    else if (page[u] != -2) atomicExch(p.error_flag, 2);
                    page[u] = look_up(i + 2, u);
                }
                ok = begin_block(i);
                if (!ok) break;
                const unsigned stage_at = (unsigned)(i % kStages) * L::kKvBytes + to;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const long long offset = __shfl_sync(0xffffffffu, offsets[u >> 2], (u & 3) * 8 + row_in_8);
                    const long long from = offset >= 0 ? offset : 0;
                    copy(k_addr + stage_at + u * 1024u, v_addr + stage_at + u * 1024u, k + from, v + from, offset >= 0);
                }
                end_block(i);
            }
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        if (!ok) error = 61;
    } else if (!softmax) {
        // ------------------------------------------------------------------------------------ a team's products
        // The whole warp waits, one elected lane issues.
        constexpr unsigned idesc_s = instruction_descriptor(kTtM, kTtN);
        constexpr unsigned idesc_o = instruction_descriptor_b_mn(kTtM, 64);        // (64 columns of O at a time)
        const unsigned long long desc_q = smem_descriptor(q_addr);
        // S of the team's n-th block, as soon as its keys are there. (The softmax has read the buffer's last content: P of block
        // n - 1 was complete before this point. Where P lies over the scores, its product must be done as well.)
        auto scores = [&](int n) -> bool {
            const int i = kStride * n + first_block, stage = i % kStages;
            if (!wait(kv_full[stage], (i / kStages) & 1)) return false;
            if (L::kOverScores && n >= 2 && !wait(o_full[team][n & 1], ((n - 2) >> 1) & 1)) return false;
            // (the copies wrote through the generic proxy, the products read through the asynchronous one)
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            tcgen05_fence_after();
            const unsigned long long desc_k = smem_descriptor(k_addr + stage * L::kKvBytes);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / kUmmaK; ++kk) {
                    const unsigned long long half = kk >> 2, part = 2 * (kk & 3);
                    umma_bf16(team_base + (unsigned)((n & 1) * kTtN), desc_q + half * (L::kQHalf >> 4) + part,
                              desc_k + half * (L::kKvHalf >> 4) + part, idesc_s, kk > 0 ? 1u : 0u);
                }
                umma_commit(smem_u32(&s_full[team][n & 1]));
            }
            __syncwarp();
            return true;
        };
        if (idle) {
            for (int n = 0; n < mine; ++n) {
                if (!wait(kv_full[n % kStages], (n / kStages) & 1)) {
                    error = 63;
                    break;
                }
                if (elect_one()) mbar_arrive_one(smem_u32(&kv_empty[n % kStages]));
                __syncwarp();
            }
        } else if (mine > 0) {
            if (!wait(q_full[PAIRED ? team : 0], 0) || (!PAIRED && !wait(q_full[1], 0))) error = 62;
            if (!error && !scores(0)) error = 63;
            for (int n = 0; n < mine && !error; ++n) {
                if (n + 1 < mine && !scores(n + 1)) {
                    error = 63;
                    break;
                }
                const int stage = (kStride * n + first_block) % kStages;
                if (!wait(p_full[team][n & 1], (n >> 1) & 1)) {
                    error = 64;
                    break;
                }
                tcgen05_fence_after();
                const unsigned long long desc_v = smem_descriptor(v_addr + stage * L::kKvBytes);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kTtN / kUmmaK; ++kk) {
#pragma unroll
                        for (int half = 0; half < L::kHalves; ++half)
                            umma_bf16_a_tmem(team_base + L::kOColumn + half * 64, team_base + L::p_column(n) + (unsigned)(kk * 8),
                                             desc_v + (unsigned long long)(half * (L::kKvHalf >> 4) + kk * 128), idesc_o, (n > 0 || kk > 0) ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&kv_empty[stage]));
                    umma_commit(smem_u32(&o_full[team][n & 1]));
                }
                __syncwarp();
            }
        }
    } else {
        // ------------------------------------------------------------------------------------- softmax
        // the rows' queries into shared memory in the products' layout: 128-byte rows, 16-byte pieces exchanged by the row's low bits
#pragma unroll
        for (int c0 = 0; c0 < kQueryPieces; ++c0) {
            const int c = PAIRED ? c0 : team * kQueryPieces + c0;
            const unsigned to = q_addr + (unsigned)(c >> 3) * L::kQHalf + (unsigned)lane_row * 128u + (unsigned)(((c & 7) ^ (lane_row & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(query[c0].x), "r"(query[c0].y), "r"(query[c0].z), "r"(query[c0].w)
                         : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        mbar_arrive_one(smem_u32(&q_full[team]));
        const bool warp_live = (row & ~31) < rows;
        const float to_log2 = p.cap_out > 0.0f ? 1.4426950408889634f : p.scale * 1.4426950408889634f;      // (capped scores come scaled)
        const unsigned long long scale2 = pack_f32x2(to_log2, to_log2);
        const unsigned o_taddr = row_base + L::kOColumn;
        bool ok = true;
        // `used_max` (raw scores times to_log2) is the maximum that P and the sum are relative to; it follows the true one only
        // when that has grown by more than kSlack, so that O in tensor memory is rescaled rarely.
        constexpr float kSlack = 8.0f;
        for (int n = 0; n < mine && !idle; ++n) {
            const int i = kStride * n + first_block, stage = i % kStages;
            ok = wait(s_full[team][n & 1], (n >> 1) & 1);
            if (!ok) break;
            tcgen05_fence_after();
            const int key_base = (block_begin + i) * kTtN;
            const bool partial = key_base + kTtN > s.context || key_base < edge;
            unsigned packed[16];
            if (!warp_live) {
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[j] = 0u;
                tmem_store_16(row_base + L::p_column(n), packed);
                tmem_store_16(row_base + L::p_column(n) + 16u, packed);
            } else {
                float sc[kTtN];
                {
                    unsigned lo[32], hi[32];
                    tmem_load_32_issue(row_base + (unsigned)((n & 1) * kTtN), lo);
                    tmem_load_32_issue(row_base + (unsigned)((n & 1) * kTtN + 32), hi);
                    tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        sc[j] = __uint_as_float(lo[j]);
                        sc[32 + j] = __uint_as_float(hi[j]);
                    }
                }
                if (p.cap_out > 0.0f) {
#pragma unroll
                    for (int j = 0; j < kTtN; ++j) sc[j] = p.cap_out * quick_tanh(sc[j] * p.cap_in);
                }
                if (partial) {
                    const unsigned long long seen = tree_visible(p, s, mask, position, key_base);
                    const unsigned lo = (unsigned)seen, hi = (unsigned)(seen >> 32);
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        sc[j] = (lo >> j) & 1u ? sc[j] : -INFINITY;
                        sc[32 + j] = (hi >> j) & 1u ? sc[32 + j] : -INFINITY;
                    }
                }
                // The weights are taken relative to the maximum of the blocks before, while this block's is found: waiting for it first
                // cost 350 cycles a step. Where it turns out larger by more than kSlack, which is rare behind a row's first blocks, O
                // and the sum are rescaled and the weights taken once more. (The warp's rows are asked before the second half's
                // exponentials, which hide the answer: 256 rows x 64 keys take an SM 895 ns, 971 with the question at the end. Asking
                // for the next block's scores there as well, or four teams of which each waits more, took 1,026 and 1,077.)
                bool settled = __any_sync(0xffffffffu, used_max == -INFINITY);
                float largest = -INFINITY, sum = 0.0f;
                if (settled) {
#pragma unroll
                    for (int j = 0; j < kTtN; j += 2) largest = max3_f32(largest, sc[j], sc[j + 1]);
                }
                bool raise = settled;
                while (true) {
                    if (raise) {
                        const float new_max = fmaxf(used_max, largest * to_log2);
                        const bool grown = new_max > used_max + kSlack;      // (-inf + slack = -inf)
                        if (n > 0 && __any_sync(0xffffffffu, grown)) {
                            ok = wait(o_full[team][(n - 1) & 1], ((n - 1) >> 1) & 1);
                            if (!ok) break;
                            tcgen05_fence_after();
                            const float factor = !grown ? 1.0f : (used_max == -INFINITY ? 0.0f : exp2f(used_max - new_max));
                            const unsigned long long factor2 = pack_f32x2(factor, factor);
#pragma unroll
                            for (int c0 = 0; c0 < D; c0 += 16) {
                                unsigned part[16];
                                tmem_load_16_issue(o_taddr + (unsigned)c0, part);
                                tmem_load_wait();
#pragma unroll
                                for (int j = 0; j < 16; j += 2) {
                                    float a, b;
                                    unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(part[j]), __uint_as_float(part[j + 1])), factor2), a, b);
                                    part[j] = __float_as_uint(a);
                                    part[j + 1] = __float_as_uint(b);
                                }
                                tmem_store_16(o_taddr + (unsigned)c0, part);
                            }
                            run_sum *= factor;
                        }
                        if (grown || used_max == -INFINITY) used_max = new_max;
                    }
                    const float base = used_max == -INFINITY ? 0.0f : used_max;
                    const unsigned long long neg_base2 = pack_f32x2(-base, -base);
                    sum = tree_weights<true>(sc, scale2, neg_base2, packed, largest);
                    raise = !settled && __any_sync(0xffffffffu, largest * to_log2 > used_max + kSlack);
                    settled = true;
                    if (raise) continue;
                    tmem_store_16(row_base + L::p_column(n), packed);
                    sum += tree_weights<false>(sc + 32, scale2, neg_base2, packed, largest);
                    tmem_store_16(row_base + L::p_column(n) + 16u, packed);
                    break;
                }
                if (!ok) break;
                run_sum += sum;
            }
            tmem_store_wait();
            if (partial) {
                // values that are not finite are taken out: two threads a row
                ok = wait(kv_full[stage], (i / kStages) & 1);
                if (!ok) break;
                bool found = false;
#pragma unroll
                for (int half = 0; half < L::kHalves; ++half)
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        const unsigned at = v_addr + stage * L::kKvBytes + half * L::kKvHalf + (unsigned)(lane_row * 64 + c);
                        unsigned w[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
                        bool change = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool low = not_finite(w[e] & 0xffffu), high = not_finite(w[e] >> 16);
                            change |= low | high;
                            w[e] = (low ? 0u : w[e] & 0xffffu) | (high ? 0u : w[e] & 0xffff0000u);
                        }
                        if (change) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        found |= change;
                    }
                if (found) bad_values = 1;
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            }
            tcgen05_fence_before();
            mbar_arrive_one(smem_u32(&p_full[team][n & 1]));
        }
        if (ok && mine > 0 && !idle) ok = wait(o_full[team][(mine - 1) & 1], ((mine - 1) >> 1) & 1);
        if (!ok) error = 65;
    }
    if (error) atomicExch(p.error_flag, error);

    // ---- what the teams have, of all pieces of the keys, meets in shared memory, where queries and keys were: every block of the
    // cluster owns some of the rows, and everybody writes a row's part (outputs, maximum, sum) to its owner
    const bool across = p.splits > 1 && p.part_o == nullptr;    // the pieces of the keys are a cluster
    const int pieces = across ? p.splits : 1, parts = kStride == 1 ? pieces : 2 * pieces;
    const int row_first = across ? split * rows / p.splits : 0, count = (across ? (split + 1) * rows / p.splits : rows) - row_first;
    const int most = (rows + pieces - 1) / pieces;              // rows of an owner
    tcgen05_fence_before();
    __syncthreads();                                            // (every product of the block is done, every copy has landed)
    if (across) cluster_sync();
    tcgen05_fence_after();
    const unsigned stats_at = smem_base + L::kStatsAt;          // [part][most] pairs; outputs before: [part][most][kPitch]
    if (softmax && !idle && !(L::kAlone && team == 1)) {
        const int owner = across ? ((row + 1) * p.splits - 1) / rows : 0;
        const int slot = (kStride == 1 ? (across ? split : 0) : (across ? 2 * split : 0) + team) * most + row - (across ? owner * rows / p.splits : 0);
        const unsigned stats_to = peer_address(stats_at + (unsigned)slot * 8u, owner, across && live);
        const unsigned to = peer_address(smem_base + (unsigned)(slot * L::kPitch) * 4u, owner, across && live);
        if (live) store_2(stats_to, used_max, run_sum);
        const bool bad = bad_values != 0;
        if (mine > 0) {
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                unsigned o[32];
                __syncwarp();                                   // (a load from tensor memory wants the whole warp)
                tmem_load_32_issue(row_base + L::kOColumn + (unsigned)c0, o);
                tmem_load_wait();
                if (!live) continue;
                if (bad) {
                    const int* table = p.block_table + (size_t)span * p.table_stride;
                    for (int i = first_block; i < blocks; i += kStride) {
                        const int key_base = (block_begin + i) * kTtN;
                        if (key_base + kTtN <= s.context && key_base >= edge) continue;
                        for (unsigned long long seen = tree_visible(p, s, mask, position, key_base); seen; seen &= seen - 1) {
                            const int key = key_base + __ffsll((long long)seen) - 1;
                            const int logical = key / p.page_tokens;
                            const int page = logical < p.table_columns ? table[logical] : -1;
                            if (page < 0 || page >= p.pages) continue;
                            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v_cache) + (long long)page * p.page_stride +
                                                     ((long long)kvh * p.page_tokens + key % p.page_tokens) * d + c0;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const float x = c0 + j < d ? __bfloat162float(v[j]) : 0.0f;
                                if (!isfinite(x)) o[j] = __float_as_uint(__uint_as_float(o[j]) + x);
                            }
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 32; c += 4) store_4(to + (unsigned)(c0 + c) * 4u, o[c], o[c + 1], o[c + 2], o[c + 3]);
            }
            __syncwarp();
        }
    }
    tcgen05_fence_before();
    if (across)
        cluster_sync();
    else
        __syncthreads();
    if (warp == kTtCopyWarps) tmem_dealloc(tmem_base, kTtTmemColumns);
    // The owner's rows: first the parts' maxima and sums become their factors, a thread a row, then the outputs are added up, eight
    // columns at a time, the parts in order. (Loops short in instructions: this runs once a block, and fetching what it takes for
    // the first time costs more than running it.)
    unsigned char* meeting = smem_raw + (smem_base - smem_u32(smem_raw));
    const float* meet = reinterpret_cast<const float*>(meeting);
    float2* row_stats = reinterpret_cast<float2*>(meeting + L::kStatsAt);
    int* unit_s = reinterpret_cast<int*>(meeting + L::kUnitsAt);
    if (tid < count) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
        for (int part = 0; part < parts; ++part) top = fmaxf(top, row_stats[part * most + tid].x);
#pragma unroll 1
        for (int part = 0; part < parts; ++part) {
            const float2 stats = row_stats[part * most + tid];
            // (a part without a maximum has a sum of 0, or of NaN where it saw NaN alone: maxima leave that out, rows must not)
            const float factor = stats.x == -INFINITY ? stats.y : fast_exp2(stats.x - top);
            sum = fmaf(stats.y, factor, sum);
            row_stats[part * most + tid].x = factor;
        }
        const int of_row = row0 + row_first + tid, of_head = kvh * p.group + of_row % p.group;
        const int unit = (s.begin + of_row / p.group) * p.q_heads + of_head;      // (fits: see tree_tcgen05_takes)
        unit_s[tid] = unit;
        float inv = 1.0f;
        if (p.part_o) {
            *reinterpret_cast<float2*>(p.part_ml + ((size_t)unit * p.splits + split) * 2) = make_float2(top, sum);
        } else {
            if (p.sinks && top != -INFINITY) sum += fast_exp2(p.sinks[of_head] * 1.4426950408889634f - top);
            inv = top == -INFINITY ? sum : 1.0f / sum;
        }
#pragma unroll 1
        for (int part = 0; part < parts; ++part) row_stats[part * most + tid].y = inv;
    }
    __syncthreads();
#pragma unroll 1
    for (int item = tid; item < count * (D / 8); item += kTtThreads) {
        const int r = item / (D / 8), c = item % (D / 8) * 8;
        if (c >= d) continue;
        float4 lo = make_float4(0.0f, 0.0f, 0.0f, 0.0f), hi = lo;
#pragma unroll 2
        for (int part = 0; part < parts; ++part) {
            const float factor = row_stats[part * most + r].x;
            if (factor == 0.0f) continue;                       // (a part without keys of the row has left nothing)
            const float4* at = reinterpret_cast<const float4*>(meet + (part * most + r) * L::kPitch + c);
            const float4 x = at[0], y = at[1];
            lo = make_float4(fmaf(x.x, factor, lo.x), fmaf(x.y, factor, lo.y), fmaf(x.z, factor, lo.z), fmaf(x.w, factor, lo.w));
            hi = make_float4(fmaf(y.x, factor, hi.x), fmaf(y.y, factor, hi.y), fmaf(y.z, factor, hi.z), fmaf(y.w, factor, hi.w));
        }
        const float inv = row_stats[r].y;
        const size_t unit = unit_s[r];
        if (p.part_o) {
            float4* to = reinterpret_cast<float4*>(p.part_o + (unit * p.splits + split) * d + c);
            to[0] = lo;
            to[1] = hi;
        } else {
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + unit * d + c) =
                make_uint4(pack_bf16_pair(lo.x * inv, lo.y * inv), pack_bf16_pair(lo.z * inv, lo.w * inv),
                           pack_bf16_pair(hi.x * inv, hi.y * inv), pack_bf16_pair(hi.z * inv, hi.w * inv));
        }
    }
}

bool tree_tcgen05_takes(const TreeParams& p) {
    // (page strides and (token, query head) numbers of 32 bits)
    return p.head_dim % 8 == 0 && p.head_dim <= 256 && p.page_stride < (1ll << 32) && (long long)p.tokens * p.q_heads < (1ll << 31) && p.page_stride % 8 == 0 && p.q_row_stride % 8 == 0 && p.scale > 0.0f &&
           (((size_t)p.q | (size_t)p.k_cache | (size_t)p.v_cache | (size_t)p.out | (size_t)p.part_o) & 15) == 0;
}

// Two teams' rows a tile where one tile of 128 does not hold them: the same keys would be read for every tile.
static bool tree_paired(const TreeParams& p) { return p.head_dim <= 128 && p.max_nodes * p.group > kTtM; }

// The kernel may have its shared memory: said once a device (a call of its own costs a small launch a tenth of its time).
template <int D, bool PAIRED>
static cudaError_t allow_shared_memory() {
    static std::atomic<unsigned long long> said;
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess || (device < 64 && (said.load(std::memory_order_relaxed) >> device & 1))) return status;
    status = cudaFuncSetAttribute(attention_tree_tcgen05_kernel<D, PAIRED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)TtLayout<D, PAIRED>::kSmemBytes);
    if (status == cudaSuccess && device < 64) said.fetch_or(1ull << device, std::memory_order_relaxed);
    return status;
}

template <int D, bool PAIRED>
static cudaError_t tree_config(cudaLaunchConfig_t& config, cudaLaunchAttribute (&attributes)[2], int cluster) {
    constexpr unsigned smem = TtLayout<D, PAIRED>::kSmemBytes;
    const cudaError_t status = allow_shared_memory<D, PAIRED>();
    config.blockDim = dim3(kTtThreads);
    config.dynamicSmemBytes = smem;
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = chaining_enabled() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return status;
}

// How many clusters of `size` blocks the device runs at a time (a cluster wants SMs of one group: 148 SMs hold fewer than
// 148 / size). Asked once; any device of this kind answers alike.
template <int D, bool PAIRED>
static int clusters_at_once(int size) {
    static std::atomic<int> known[kTtMaxCluster + 1];
    int count = known[size].load(std::memory_order_relaxed);
    if (count == 0) {
        cudaLaunchConfig_t config = {};
        cudaLaunchAttribute attributes[2];
        config.gridDim = dim3(size, 1, 1);
        if (tree_config<D, PAIRED>(config, attributes, size) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&count, attention_tree_tcgen05_kernel<D, PAIRED>, &config) != cudaSuccess || count <= 0) {
            cudaGetLastError();
            count = 148 / size;
        }
        known[size].store(count, std::memory_order_relaxed);
    }
    return count;
}

template <int D, bool PAIRED>
static TreeTile tree_tile() {
    TreeTile tile = {PAIRED ? 2 * kTtM : kTtM, 148, 14, kTtMaxCluster, {0}};
    for (int size = 2; size <= kTtMaxCluster; ++size) tile.problems_at_once[size] = clusters_at_once<D, PAIRED>(size);
    return tile;
}

TreeTile tree_tcgen05_tile(const TreeParams& p) {
    if (p.head_dim <= 64) return tree_paired(p) ? tree_tile<64, true>() : tree_tile<64, false>();
    if (p.head_dim <= 128) return tree_paired(p) ? tree_tile<128, true>() : tree_tile<128, false>();
    return tree_tile<256, false>();
}

template <int D, bool PAIRED>
static int launch_tree(const TreeParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attributes[2];
    cudaError_t status = tree_config<D, PAIRED>(config, attributes, p.part_o ? 1 : p.splits);
    CELEG_REQUIRE(status == cudaSuccess, "attention_tree: %s", cudaGetErrorString(status));
    const int tile = PAIRED ? 2 * kTtM : kTtM, tiles = (p.max_nodes * p.group + tile - 1) / tile;
    config.gridDim = dim3(tiles * p.splits, p.kv_heads, p.spans);
    config.stream = stream;
    status = cudaLaunchKernelEx(&config, attention_tree_tcgen05_kernel<D, PAIRED>, p);
    CELEG_REQUIRE(status == cudaSuccess, "attention_tree: %s", cudaGetErrorString(status));
    return check_launch("attention_tree");
}

int launch_tree_tcgen05(const TreeParams& p, cudaStream_t stream) {
    if (p.head_dim <= 64) return tree_paired(p) ? launch_tree<64, true>(p, stream) : launch_tree<64, false>(p, stream);
    if (p.head_dim <= 128) return tree_paired(p) ? launch_tree<128, true>(p, stream) : launch_tree<128, false>(p, stream);
    return launch_tree<256, false>(p, stream);
}

}  // namespace celeg_b200
