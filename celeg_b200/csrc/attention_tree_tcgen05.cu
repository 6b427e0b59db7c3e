// Attention of a tree of drafted tokens over the paged cache on the fifth-generation tensor cores, bfloat16, head sizes D of 64
// and 128, pages of 8, 16, 32 or 64 positions that lie side by side (see attention_tree.cuh for the operator):
//
//   grid = (row tiles x pieces of the keys, kv heads, spans). A row tile is 128 rows (node, query head of the group) of one kv
//   head, so that a key is read once for a whole group and tree; the pieces are of whole blocks of 64 keys.
//   Six warps. Warp 0 brings a block's K and V page by page through the block table by TMA (128-byte swizzle, a lane a copy,
//   pages looked up a block ahead) into a ring of stages; warp 1 issues S = Q K^T and O += P V (tcgen05.mma, P from tensor
//   memory, V as it lies in the cache); warps 2 to 5 are the softmax, a thread a row. S and P exist twice, so that the products
//   of one block run while the softmax is busy with the next. Two blocks an SM (81 or 97 KiB of shared memory, 256 columns of
//   tensor memory) hide one another's waits.
//   The rows of Q are gathered by the softmax threads themselves (a head here, a node there) and written in the layout that
//   TMA gives the keys.
//
// Blocks of keys before the tree are seen whole by every row and need no mask. In the others a row's mask is 64 bits, cut from
// its words of ancestors; values that no row sees are overwritten with zeros, and a value that is not finite is taken out and
// added to the rows that do see it at the end (a weight of zero times it would reach the others).
//
// The weights are rounded to bfloat16 for their product with V; the denominator adds up the rounded ones, so that the outputs
// are exact averages of what was multiplied. Rows beyond the span's and warps without rows take no exponentials.
#include "attention_tree.cuh"
#include "attention_tree_tcgen05.h"
#include "ring_drain.h"
#include "tcgen05.cuh"

namespace celeg_b200 {

constexpr int kTtThreads = 192;
constexpr int kTtM = 128;                 // rows per tile
constexpr int kTtN = 64;                  // keys per block

template <int D>
struct TtLayout {
    static constexpr int kHalves = D / 64;
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr unsigned kQHalf = kTtM * 128, kKvHalf = kTtN * 128;
    static constexpr unsigned kQBytes = kHalves * kQHalf;       // 16 or 32 KiB
    static constexpr unsigned kKvBytes = kHalves * kKvHalf;     // 8 or 16 KiB each for a block's K and V
    static constexpr unsigned kSmemBytes = kQBytes + kStages * 2 * kKvBytes + 1024;
    // Tensor memory: S of even and odd blocks at columns 0 and 64, O from 128 on; P behind O at a head size of 64, over the
    // scores it is made of at 128.
    static constexpr unsigned kOColumn = 2 * kTtN;
    static constexpr bool kOverScores = D == 128;
    static __device__ __forceinline__ unsigned p_column(int i) {
        return kOverScores ? (unsigned)((i & 1) * kTtN) : 2 * kTtN + D + (unsigned)((i & 1) * (kTtN / 2));
    }
};
constexpr unsigned kTtTmemColumns = 256;

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

template <int D>
__global__ void __launch_bounds__(kTtThreads)
attention_tree_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeParams p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    using L = TtLayout<D>;
    constexpr int kStages = L::kStages;
    __shared__ __align__(8) unsigned long long kv_full[kStages], kv_empty[kStages], q_full, s_full[2], p_full[2], o_full[2];
    __shared__ unsigned tmem_base_slot;
    __shared__ int lowest_s, highest_s, bad_values;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int span = blockIdx.z, kvh = blockIdx.y;
    const int tiles = (p.max_nodes * p.group + kTtM - 1) / kTtM;
    const int row0 = (blockIdx.x % tiles) * kTtM, split = blockIdx.x / tiles;
    const TreeSpan s = tree_span(p, span);
    const int rows = min(s.nodes * p.group - row0, kTtM);
    if (rows <= 0) return;                                      // (the whole block, before anything is taken)

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&kv_full[i]), 1);
            mbar_init(smem_u32(&kv_empty[i]), 1);
        }
        mbar_init(smem_u32(&q_full), 128);
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&s_full[b]), 1);
            mbar_init(smem_u32(&p_full[b]), 128);
            mbar_init(smem_u32(&o_full[b]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        lowest_s = 0x7fffffff;
        highest_s = -0x7fffffff - 1;
        bad_values = 0;
    }
    if (warp == 0) tmem_alloc(smem_u32(&tmem_base_slot), kTtTmemColumns);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const unsigned tmem_base = tmem_base_slot;

    // a softmax thread's row
    const int row = (warp & 3) * 32 + lane;                     // (of warps 2 to 5: the TMEM lane)
    const bool live = warp >= 2 && row < rows;
    const int node = s.begin + (row0 + min(row, rows - 1)) / p.group;
    const int head = kvh * p.group + (row0 + min(row, rows - 1)) % p.group;
    int position = 0;
    if (p.window) {
        position = p.positions[node];
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

    const unsigned smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const unsigned q_addr = smem_base;
    const unsigned k_addr = q_addr + L::kQBytes, v_addr = k_addr + kStages * L::kKvBytes;

    int error = 0;
    if (warp == 0) {
        // ------------------------------------------------------------------------------------ producer
        const int* table = p.block_table + (size_t)span * p.table_stride;
        const int pages_per_block = kTtN / p.page_tokens;                          // 1 to 8
        const int pieces = 2 * L::kHalves * pages_per_block;                       // K and V, halves of a row
        static_assert(2 * L::kHalves * 8 <= 32, "a lane brings one piece");
        auto lookup = [&](int kb, int piece) -> int {
            const int key0 = kb * kTtN + (piece / (2 * L::kHalves)) * p.page_tokens;
            if (piece >= pieces || kb >= block_begin + blocks || key0 > last_key || key0 + p.page_tokens <= first_key) return 0;
            const int logical = key0 / p.page_tokens;
            const int page = logical < p.table_stride ? table[logical] : -1;
            if (page < 0 || page >= p.pages) {
                atomicExch(p.error_flag, 2);
                return 0;                                                          // (keys nobody may see, or reported: any page will do)
            }
            return page;
        };
        int page = lookup(block_begin, lane);
        int brought = 0;
        bool ok = true;
        for (int i = 0; i < blocks && ok; ++i) {
            const int mine = page;
            page = lookup(block_begin + i + 1, lane);
            const int stage = i % kStages;
            const unsigned bar = smem_u32(&kv_full[stage]);
            int got = 1;
            if (lane == 0) {
                if (i >= kStages && !mbar_wait_suspended(smem_u32(&kv_empty[stage]), ((i / kStages) - 1) & 1)) got = 0;
                if (got) mbar_expect_tx(bar, 2 * L::kKvBytes);
            }
            ok = __shfl_sync(0xffffffffu, got, 0) != 0;
            if (ok && lane < pieces) {
                const int pg = lane / (2 * L::kHalves), side = lane % 2, half = (lane / 2) % L::kHalves;
                const unsigned to = (side ? v_addr : k_addr) + stage * L::kKvBytes + half * L::kKvHalf + pg * (unsigned)p.page_tokens * 128u;
                tma_load_2d(to, side ? &map_v : &map_k, bar, half * 64, (mine * p.kv_heads + kvh) * p.page_tokens);
            }
            brought += ok;
        }
        if (lane == 0) {
            if (!ok) error = 61;
            // whichever role gives up: the block does not end before its copies have landed
            drain_ring(max(0, brought - kStages), brought, kStages,
                       [&](int stage, unsigned parity) { mbar_wait_suspended(smem_u32(&kv_full[stage]), parity); });
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------------------------- MMA issuer
        constexpr unsigned idesc_s = instruction_descriptor(kTtM, kTtN);
        constexpr unsigned idesc_o = instruction_descriptor_b_mn(kTtM, 64);        // (64 columns of O at a time)
        const unsigned long long desc_q = smem_descriptor(q_addr);
        auto wait = [&](unsigned long long& bar, int parity) {
            return __all_sync(0xffffffffu, mbar_wait_suspended(smem_u32(&bar), (unsigned)parity)) != 0;
        };
        auto scores = [&](int i) -> bool {
            const int stage = i % kStages;
            if (!wait(kv_full[stage], (i / kStages) & 1)) return false;
            if (L::kOverScores && i >= 2 && !wait(o_full[i & 1], ((i - 2) >> 1) & 1)) return false;
            tcgen05_fence_after();
            const unsigned long long desc_k = smem_descriptor(k_addr + stage * L::kKvBytes);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / kUmmaK; ++kk) {
                    const unsigned long long half = kk >> 2, part = 2 * (kk & 3);
                    umma_bf16(tmem_base + (unsigned)((i & 1) * kTtN), desc_q + half * (L::kQHalf >> 4) + part,
                              desc_k + half * (L::kKvHalf >> 4) + part, idesc_s, kk > 0 ? 1u : 0u);
                }
                umma_commit(smem_u32(&s_full[i & 1]));
            }
            __syncwarp();
            return true;
        };
        if (blocks > 0) {
            if (!wait(q_full, 0)) error = 62;
            if (!error && !scores(0)) error = 63;
        }
        for (int i = 0; i < blocks && !error; ++i) {
            // (the scores of the next block: the softmax has read that buffer, P of block i - 1 was complete before this point)
            if (i + 1 < blocks && !scores(i + 1)) {
                error = 63;
                break;
            }
            const int stage = i % kStages;
            if (!wait(p_full[i & 1], (i >> 1) & 1)) {
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
                        umma_bf16_a_tmem(tmem_base + L::kOColumn + half * 64, tmem_base + L::p_column(i) + (unsigned)(kk * 8),
                                         desc_v + (unsigned long long)(half * (L::kKvHalf >> 4) + kk * 128), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
                }
                umma_commit(smem_u32(&kv_empty[stage]));
                umma_commit(smem_u32(&o_full[i & 1]));
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------------------------- softmax
        // the row's query into shared memory as TMA would lay it: 128-byte rows, 16-byte pieces exchanged by the row's low bits
        {
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + (size_t)node * p.q_row_stride + (size_t)head * D;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(q) + c) : make_uint4(0u, 0u, 0u, 0u);
                const unsigned to = q_addr + (unsigned)(c >> 3) * L::kQHalf + (unsigned)row * 128u + (unsigned)(((c & 7) ^ (row & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            mbar_arrive_one(smem_u32(&q_full));
        }
        const unsigned lane_base = tmem_base + ((unsigned)((warp & 3) * 32) << 16);
        const unsigned* mask = p.ancestors + (size_t)node * p.words;
        const bool warp_live = (warp & 3) * 32 < rows;
        const float scale_log2 = p.scale * 1.4426950408889634f;
        const float to_log2 = p.cap_out > 0.0f ? 1.4426950408889634f : scale_log2;      // (capped scores come scaled)
        const unsigned long long scale2 = pack_f32x2(to_log2, to_log2);
        // `used_max` (raw scores times to_log2) is the maximum that P and the sum are relative to; it follows the true one only
        // when that has grown by more than kSlack, so that O in tensor memory is rescaled rarely.
        constexpr float kSlack = 8.0f;
        float used_max = -INFINITY, run_sum = 0.0f;
        bool ok = true;
        const unsigned o_taddr = lane_base + L::kOColumn;
        for (int i = 0; i < blocks; ++i) {
            ok = ok && mbar_wait(smem_u32(&s_full[i & 1]), (i >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tcgen05_fence_after();
            const int key_base = (block_begin + i) * kTtN;
            unsigned p_packed[kTtN / 2];
            if (!warp_live) {
#pragma unroll
                for (int j = 0; j < kTtN / 2; ++j) p_packed[j] = 0u;
            } else {
                float sc[kTtN];
                {
                    unsigned lo[32], hi[32];
                    tmem_load_32_issue(lane_base + (unsigned)((i & 1) * kTtN), lo);
                    tmem_load_32_issue(lane_base + (unsigned)((i & 1) * kTtN + 32), hi);
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
                if (key_base + kTtN > s.context || key_base < edge) {
                    const unsigned long long seen = tree_visible(p, s, mask, position, key_base);
                    const unsigned lo = (unsigned)seen, hi = (unsigned)(seen >> 32);
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        sc[j] = (lo >> j) & 1u ? sc[j] : -INFINITY;
                        sc[32 + j] = (hi >> j) & 1u ? sc[32 + j] : -INFINITY;
                    }
                }
                float part_max[4];
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                    float m = max3_f32(sc[16 * c4], sc[16 * c4 + 1], sc[16 * c4 + 2]);
#pragma unroll
                    for (int j = 3; j < 15; j += 2) m = max3_f32(m, sc[16 * c4 + j], sc[16 * c4 + j + 1]);
                    part_max[c4] = fmaxf(m, sc[16 * c4 + 15]);
                }
                // (a negative scale turns the order round: the largest is then found among the scaled ones)
                float block_max = fmaxf(max3_f32(part_max[0], part_max[1], part_max[2]), part_max[3]) * to_log2;
                if (to_log2 <= 0.0f) {
                    block_max = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kTtN; ++j) block_max = sc[j] == -INFINITY ? block_max : fmaxf(block_max, sc[j] * to_log2);
                }
                if (i == 0) {
                    used_max = block_max;
                } else {
                    const float new_max = fmaxf(used_max, block_max);
                    const bool grown = new_max > used_max + kSlack;          // (-inf + slack = -inf)
                    if (__any_sync(0xffffffffu, grown)) {
                        ok = mbar_wait(smem_u32(&o_full[(i - 1) & 1]), ((i - 1) >> 1) & 1);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const float factor = !grown ? 1.0f : (used_max == -INFINITY ? 0.0f : exp2f(used_max - new_max));
                        const unsigned long long factor2 = pack_f32x2(factor, factor);
#pragma unroll
                        for (int c0 = 0; c0 < D; c0 += 32) {
                            unsigned part[32];
                            tmem_load_32_issue(o_taddr + (unsigned)c0, part);
                            tmem_load_wait();
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                float a, b;
                                unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(part[j]), __uint_as_float(part[j + 1])), factor2), a, b);
                                part[j] = __float_as_uint(a);
                                part[j + 1] = __float_as_uint(b);
                            }
                            tmem_store_32(o_taddr + (unsigned)c0, part);
                        }
                        tmem_store_wait();
                        run_sum *= factor;
                        if (grown) used_max = new_max;
                    }
                }
                const float safe_max = used_max == -INFINITY ? 0.0f : used_max;
                const unsigned long long neg_max2 = pack_f32x2(-safe_max, -safe_max);
                unsigned long long part_sum[4] = {0ull, 0ull, 0ull, 0ull};          // (0.0f, 0.0f) each
                const bool turned = to_log2 <= 0.0f;
#pragma unroll
                for (int j2 = 0; j2 < kTtN / 2; ++j2) {
                    float x0, x1, a, b;
                    unpack_f32x2(fma_f32x2(pack_f32x2(sc[2 * j2], sc[2 * j2 + 1]), scale2, neg_max2), x0, x1);
                    if (turned) {
                        x0 = sc[2 * j2] == -INFINITY ? -INFINITY : x0;
                        x1 = sc[2 * j2 + 1] == -INFINITY ? -INFINITY : x1;
                    }
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(x0));
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(x1));
                    const __nv_bfloat162 pair = __floats2bfloat162_rn(a, b);          // key 2 j2 in the lower half
                    const unsigned packed = *reinterpret_cast<const unsigned*>(&pair);
                    p_packed[j2] = packed;
                    part_sum[j2 & 3] = add_f32x2(part_sum[j2 & 3], pack_f32x2(__uint_as_float(packed << 16), __uint_as_float(packed & 0xffff0000u)));
                }
                float s0, s1;
                unpack_f32x2(add_f32x2(add_f32x2(part_sum[0], part_sum[1]), add_f32x2(part_sum[2], part_sum[3])), s0, s1);
                run_sum += s0 + s1;
            }
            // (K and V of a block came together: its scores being there, its values are)
            if (key_base + kTtN > s.context || key_base < edge) {
                const int stage = i % kStages;
                ok = mbar_wait(smem_u32(&kv_full[stage]), (i / kStages) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // values of places that hold no key of this span become zeros, as do those that are not finite: two threads a row
                const int key = key_base + row / 2;
                const bool none = key < first_key || key > last_key;
                bool found = false;
#pragma unroll
                for (int half = 0; half < L::kHalves; ++half)
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        const unsigned at = v_addr + stage * L::kKvBytes + half * L::kKvHalf + (unsigned)(row * 64 + c);
                        unsigned w[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
                        bool change = none;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool low = none || not_finite(w[e] & 0xffffu), high = none || not_finite(w[e] >> 16);
                            change |= low | high;
                            w[e] = (low ? 0u : w[e] & 0xffffu) | (high ? 0u : w[e] & 0xffff0000u);
                        }
                        if (change) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        found |= change && !none;
                    }
                if (found) bad_values = 1;
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            }
            tmem_store_32(lane_base + L::p_column(i), p_packed);
            tmem_store_wait();
            tcgen05_fence_before();
            mbar_arrive_one(smem_u32(&p_full[i & 1]));
        }
        if (ok && blocks > 0) {
            ok = mbar_wait(smem_u32(&o_full[(blocks - 1) & 1]), ((blocks - 1) >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) tcgen05_fence_after();
        }
        if (!ok) {
            if (lane == 0) atomicExch(p.error_flag, 65);
        } else {
            const size_t unit = (size_t)node * p.q_heads + head;
            float inv = 1.0f;
            if (p.splits > 1) {
                if (live) {
                    p.part_ml[(unit * p.splits + split) * 2] = used_max;
                    p.part_ml[(unit * p.splits + split) * 2 + 1] = run_sum;
                }
            } else {
                const float sink_part = (p.sinks && used_max != -INFINITY) ? exp2f(p.sinks[head] * 1.4426950408889634f - used_max) : 0.0f;
                inv = used_max == -INFINITY ? 0.0f : 1.0f / (run_sum + sink_part);
            }
            // every softmax thread has passed its last look at the values (o_full came after all of their arrivals)
            const bool bad = *reinterpret_cast<volatile int*>(&bad_values) != 0;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 32) {
                unsigned o[32];
                __syncwarp();
                if (blocks > 0) {
                    tmem_load_32_issue(o_taddr + (unsigned)c0, o);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0u;
                }
                if (!live) continue;
                if (bad) {
                    for (int i = 0; i < blocks; ++i) {
                        const int key_base = (block_begin + i) * kTtN;
                        if (key_base + kTtN <= s.context && key_base >= edge) continue;
                        const int* table = p.block_table + (size_t)span * p.table_stride;
                        for (unsigned long long seen = tree_visible(p, s, mask, position, key_base); seen; seen &= seen - 1) {
                            const int key = key_base + __ffsll((long long)seen) - 1;
                            const int logical = key / p.page_tokens;
                            const int page = logical < p.table_stride ? table[logical] : -1;
                            if (page < 0 || page >= p.pages) continue;
                            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v_cache) + (long long)page * p.page_stride +
                                                     ((long long)kvh * p.page_tokens + key % p.page_tokens) * D + c0;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const float x = __bfloat162float(v[j]);
                                if (!isfinite(x)) o[j] = __float_as_uint(__uint_as_float(o[j]) + x);
                            }
                        }
                    }
                }
                if (p.splits > 1) {
                    float* dst = p.part_o + (unit * p.splits + split) * D + c0;
                    if (used_max != -INFINITY) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(dst + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                    }
                } else {
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + unit * D + c0;
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        uint4 packed;
                        __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
                        for (int e2 = 0; e2 < 4; ++e2)
                            h2[e2] = __floats2bfloat162_rn(__uint_as_float(o[c + 2 * e2]) * inv, __uint_as_float(o[c + 2 * e2 + 1]) * inv);
                        *reinterpret_cast<uint4*>(dst + c) = packed;
                    }
                }
            }
            __syncwarp();
        }
    }
    if (error) atomicExch(p.error_flag, error);
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, kTtTmemColumns);
}

bool tree_tcgen05_takes(const TreeParams& p) {
    return (p.head_dim == 64 || p.head_dim == 128) && p.page_tokens >= 8 && p.page_tokens % 8 == 0 && kTtN % p.page_tokens == 0 &&
           p.page_stride == (long long)p.kv_heads * p.page_tokens * p.head_dim && p.q_row_stride % 8 == 0 &&
           (((size_t)p.q | (size_t)p.k_cache | (size_t)p.v_cache | (size_t)p.out) & 15) == 0 && ((size_t)p.part_o & 15) == 0 &&
           (long long)p.pages * p.kv_heads * p.page_tokens < (1ll << 31);
}

int tree_tcgen05_rows() { return kTtM; }

int launch_tree_tcgen05(const TreeParams& p, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    const long long cache_rows = (long long)p.pages * p.kv_heads * p.page_tokens;
    if (!tensor_map_for(p.k_cache, cache_rows, p.head_dim, p.head_dim, p.page_tokens, &map_k)) return -2;
    if (!tensor_map_for(p.v_cache, cache_rows, p.head_dim, p.head_dim, p.page_tokens, &map_v)) return -2;
    auto kernel = p.head_dim == 64 ? attention_tree_tcgen05_kernel<64> : attention_tree_tcgen05_kernel<128>;
    const unsigned smem = p.head_dim == 64 ? TtLayout<64>::kSmemBytes : TtLayout<128>::kSmemBytes;
    const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    CELEG_REQUIRE(status == cudaSuccess, "attention_tree: %s", cudaGetErrorString(status));
    const int tiles = (p.max_nodes * p.group + kTtM - 1) / kTtM;
    kernel<<<dim3(tiles * p.splits, p.kv_heads, p.spans), kTtThreads, smem, stream>>>(map_k, map_v, p);
    return check_launch("attention_tree");
}

}  // namespace celeg_b200
