// Attention of a tree of drafted tokens over the paged cache (see attention_tree.cuh): the general kernel, the join of split
// keys, and the entry point that chooses.
//
// The general kernel takes float32 and bfloat16, any head size up to 256 and any page size. Everything is float32: a block has
// 32 rows (node, query head of a group) of one kv head and walks its keys 64 at a time. 128 threads: for the scores a thread
// has 4 rows x 4 keys, for the weighted sum 4 rows x 4 columns of every 64, operands from shared memory four numbers at a
// time, products packed two an instruction (neighbouring numbers of a score's sum, neighbouring columns of an output). (With 8
// rows a thread an operand serves twice as many products, but a step's instructions, which come once a step, no longer
// arrive as fast as they run: two requests of 24 nodes x 1,500 positions in float32 took 51 us, 36 with 4.)
// Keys and values come as they are stored, by asynchronous copies where rows are whole 16-byte pieces: of bfloat16 the next tile
// under this one's products, of float32 one tile at a time, which leaves room for twice as many blocks an SM (eight requests of
// 32 nodes x 4,096 positions in two pieces: 256 us, 378 with two tiles).
// Instructions and what waits between a tile's two products bound it: 21 TFLOP/s, of the 72 that its units have, where there are
// eight requests of up to 32 nodes x 4,096 positions on 32 heads of 64 (194 us); two of up to 24 behind 1,500 take 37 us, of which
// the join's launch is a part.
#include "attention_tree.cuh"
#include "attention_tree_tcgen05.h"
#include "tcgen05.cuh"

#include <cstring>
#include <type_traits>

namespace celeg_b200 {

constexpr int kSimtThreads = 128;
constexpr int kSimtRows = 32;
constexpr int kSimtKeys = 64;

// Shared memory of a block, in the order of the members. Rows of keys are 16-byte pieces, neighbours in different banks.
template <typename A, int COLUMNS>
struct SimtLayout {
    static constexpr int kWidth = 64 * COLUMNS;                           // a row's numbers, padded
    static constexpr int kPitch = kWidth + 16 / (int)sizeof(A);
    static constexpr int kQPitch = kWidth + 4, kWeightPitch = kSimtKeys + 4;
    static constexpr int kStages = sizeof(A) == 4 ? 1 : 2;
    static constexpr size_t kStageBytes = (size_t)kSimtKeys * (kPitch + kWidth) * sizeof(A);
    static constexpr size_t kQAt = kStages * kStageBytes, kWeightsAt = kQAt + (size_t)kSimtRows * kQPitch * 4;
    static constexpr size_t kOffsetsAt = kWeightsAt + (size_t)kSimtRows * kWeightPitch * 4, kPositionsAt = kOffsetsAt + 3 * kSimtKeys * 8;
    static constexpr size_t kBytes = kPositionsAt + 3 * kSimtKeys * 4;
};

template <typename A>
__device__ __forceinline__ float4 load_four(const A* p);
template <>
__device__ __forceinline__ float4 load_four<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load_four<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 raw = *reinterpret_cast<const uint2*>(p);
    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}

// COLUMNS: columns of the output in units of 64 (head_dim <= 64 * COLUMNS). PIECES: rows are whole 16-byte pieces on 16-byte
// addresses.
template <typename A, int COLUMNS, bool PIECES>
__global__ void __launch_bounds__(kSimtThreads) attention_tree_simt_kernel(const TreeParams p) {
    extern __shared__ __align__(16) unsigned char simt_smem[];
    using L = SimtLayout<A, COLUMNS>;
    constexpr int RT = kSimtRows / 8;                                                    // rows a thread
    float* q_s = reinterpret_cast<float*>(simt_smem + L::kQAt);                          // [rows][kQPitch]
    float* w_s = reinterpret_cast<float*>(simt_smem + L::kWeightsAt);                    // [rows][kWeightPitch]
    long long* offset_s = reinterpret_cast<long long*>(simt_smem + L::kOffsetsAt);       // [3][keys], -1: no such key
    int* position_s = reinterpret_cast<int*>(simt_smem + L::kPositionsAt);               // [3][keys]
    __shared__ int lowest_s;

    const int tid = threadIdx.x, kx = tid & 15, ry = tid >> 4, d = p.head_dim;
    const int span = blockIdx.z, split = blockIdx.x;
    const int tiles = (p.max_nodes * p.group + kSimtRows - 1) / kSimtRows;
    const int kvh = blockIdx.y / tiles, row0 = (blockIdx.y % tiles) * kSimtRows;
    chain_release();
    chain_wait();
    const TreeSpan s = tree_span(p, span);
    const int rows = s.nodes * p.group;
    if (row0 >= rows) return;
    const int* table = p.block_table + (size_t)span * p.table_stride;
    const A* q = static_cast<const A*>(p.q);
    const A* k = static_cast<const A*>(p.k_cache);
    const A* v = static_cast<const A*>(p.v_cache);

    // the keys of this block: from the first that any of its rows sees, in `splits` pieces of whole tiles
    if (tid == 0) lowest_s = 0x7fffffff;
    __syncthreads();
    if (p.window && tid < kSimtRows && row0 + tid < rows) atomicMin(&lowest_s, p.positions[s.begin + (row0 + tid) / p.group]);
    for (int i = tid; i < kSimtRows * L::kWidth; i += kSimtThreads) {
        const int r = i / L::kWidth, c = i % L::kWidth, row = row0 + r;
        q_s[r * L::kQPitch + c] = row < rows && c < d
            ? to_float(q[(size_t)(s.begin + row / p.group) * p.q_row_stride + (size_t)(kvh * p.group + row % p.group) * d + c]) : 0.0f;
    }
    if (d % 4 != 0) {       // (what a row's last four numbers reach past its end: zeros, for good)
        for (int i = tid; i < L::kStages * kSimtKeys; i += kSimtThreads) {
            A* stage = reinterpret_cast<A*>(simt_smem + (i / kSimtKeys) * L::kStageBytes);
            for (int c = d; c < (d + 3) / 4 * 4; ++c) stage[(i % kSimtKeys) * L::kPitch + c] = from_float<A>(0.0f);
        }
    }
    __syncthreads();
    const int first = p.window ? tree_first_place(p, s, lowest_s) : 0, last = s.context + s.nodes;
    const int per_split = ((last - first + p.splits - 1) / p.splits + kSimtKeys - 1) / kSimtKeys * kSimtKeys;
    const long long from = (long long)first + (long long)split * per_split;
    const int end = (int)min((long long)last, from + per_split);
    const int key_first = (int)min(from, (long long)last), count = end > key_first ? (end - key_first + kSimtKeys - 1) / kSimtKeys : 0;

    int node_position[RT];
    const unsigned* mask[RT];
    float run_max[RT], run_sum[RT];
    unsigned long long acc[RT][COLUMNS][2];                // columns in pairs
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int node = s.begin + min(row0 + ry * RT + i, rows - 1) / p.group;
        node_position[i] = p.window ? p.positions[node] : 0;
        mask[i] = p.ancestors + (size_t)node * p.words;
        run_max[i] = -INFINITY;
        run_sum[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < COLUMNS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[i][j][e] = 0ull;
    }

    // where the keys of tile n lie, and their positions
    auto look_up = [&](int n) {
        if (tid >= kSimtKeys || n >= count) return;
        const int place = key_first + n * kSimtKeys + tid;
        long long offset = -1;
        int position = place;
        if (place < end) {
            const int page = tree_page(p, table, place);
            if (page >= 0) offset = (long long)page * p.page_stride + ((long long)kvh * p.page_tokens + place % p.page_tokens) * d;
            if (p.window && place >= s.context) position = p.positions[s.begin + place - s.context];
        }
        offset_s[n % 3 * kSimtKeys + tid] = offset;
        position_s[n % 3 * kSimtKeys + tid] = position;
    };
    auto bring = [&](int n) {
        unsigned char* stage = simt_smem + (n % L::kStages) * L::kStageBytes;
        A* k_s = reinterpret_cast<A*>(stage);
        A* v_s = k_s + kSimtKeys * L::kPitch;
        if (PIECES) {
            constexpr int kPiece = 16 / (int)sizeof(A), kPerRow = L::kWidth / kPiece, kRowsATurn = kSimtThreads / kPerRow;
            const int c = tid % kPerRow * kPiece, r0 = tid / kPerRow;
#pragma unroll 8
            for (int u = 0; u < kSimtKeys / kRowsATurn; ++u) {
                const int r = r0 + u * kRowsATurn;
                const long long offset = offset_s[n % 3 * kSimtKeys + r];
                const bool there = offset >= 0 && c < d;
                const long long at = there ? offset + c : 0;
                const unsigned bytes = there ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(k_s + r * L::kPitch + c)), "l"(k + at), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(v_s + r * L::kWidth + c)), "l"(v + at), "r"(bytes) : "memory");
            }
        } else {
            for (int i = tid; i < kSimtKeys * L::kWidth; i += kSimtThreads) {
                const int r = i / L::kWidth, c = i % L::kWidth;
                if (c >= d) continue;
                const long long offset = offset_s[n % 3 * kSimtKeys + r];
                k_s[r * L::kPitch + c] = offset >= 0 ? k[offset + c] : from_float<A>(0.0f);
                v_s[r * L::kWidth + c] = offset >= 0 ? v[offset + c] : from_float<A>(0.0f);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };

    look_up(0);
    look_up(1);
    __syncthreads();
    if (L::kStages > 1 && count > 0) bring(0);
    for (int n = 0; n < count; ++n) {
        if (L::kStages > 1) {
            if (n + 1 < count) bring(n + 1);
            look_up(n + 2);
            if (n + 1 < count) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            else asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        } else {
            bring(n);
            look_up(n + 2);
            asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        }
        const int key0 = key_first + n * kSimtKeys, held = min(kSimtKeys, end - key0);
        const long long* offsets = offset_s + n % 3 * kSimtKeys;
        const int* key_positions = position_s + n % 3 * kSimtKeys;
        const A* k_s = reinterpret_cast<const A*>(simt_smem + (n % L::kStages) * L::kStageBytes);
        const A* v_s = k_s + kSimtKeys * L::kPitch;
        // every row sees every key of the tile, unless the tile reaches into the tree, the window's edge or a missing page
        const bool whole = __syncthreads_and(p.window == 0 && key0 + kSimtKeys <= s.context && (tid >= kSimtKeys || offsets[tid] >= 0));

        unsigned long long score2[RT][4];                  // the sums over even and odd numbers
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) score2[i][j] = 0ull;
#pragma unroll 2
        for (int c = 0; c < d; c += 4) {
            float4 a[RT], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = load_four<A>(k_s + (kx + 16 * j) * L::kPitch + c);
#pragma unroll
            for (int i = 0; i < RT; ++i) a[i] = *reinterpret_cast<const float4*>(q_s + (ry * RT + i) * L::kQPitch + c);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) score2[i][j] = fma_f32x2(pack_f32x2(a[i].x, a[i].y), pack_f32x2(b[j].x, b[j].y), score2[i][j]);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) score2[i][j] = fma_f32x2(pack_f32x2(a[i].z, a[i].w), pack_f32x2(b[j].z, b[j].w), score2[i][j]);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            float score[4];
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float even, odd;
                unpack_f32x2(score2[i][j], even, odd);
                float x = even + odd;
                x = p.cap_out > 0.0f ? p.cap_out * tanhf(x * p.cap_in) : x * p.scale;
                const int at = kx + 16 * j;
                if (!whole && (offsets[at] < 0 || !tree_sees(p, s, mask[i], node_position[i], key0 + at, key_positions[at]))) x = -INFINITY;
                score[j] = x;
                top = fmaxf(top, x);
            }
#pragma unroll
            for (int lanes = 8; lanes > 0; lanes >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, lanes));
            const float new_max = fmaxf(run_max[i], top);
            const float base_max = new_max == -INFINITY ? 0.0f : new_max;
            const float factor = expf(run_max[i] - base_max);            // (-inf - 0: 0, of sums that are 0)
            run_max[i] = new_max;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = expf(score[j] - base_max);
                w_s[(ry * RT + i) * L::kWeightPitch + kx + 16 * j] = w;
                sum += w;
            }
            run_sum[i] = run_sum[i] * factor + sum;                      // (this lane's share of the row)
            const unsigned long long factor2 = pack_f32x2(factor, factor);
#pragma unroll
            for (int j = 0; j < COLUMNS; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[i][j][e] = mul_f32x2(acc[i][j][e], factor2);
        }
        __syncwarp();                        // (a warp's 8 rows of weights are read by this warp alone)
        // `masked`: a weight of 0 is a key that the row does not see, whose value, whatever it is, must not reach it
        auto add_up = [&](auto masked) {
#pragma unroll 2
            for (int t = 0; t < held; t += 4) {
                float4 w[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) w[i] = *reinterpret_cast<const float4*>(w_s + (ry * RT + i) * L::kWeightPitch + t);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float4 x[COLUMNS];
#pragma unroll
                    for (int j = 0; j < COLUMNS; ++j) x[j] = load_four<A>(v_s + (t + e) * L::kWidth + j * 64 + kx * 4);
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        const float weight = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
                        if (decltype(masked)::value && weight == 0.0f) continue;
                        const unsigned long long both = pack_f32x2(weight, weight);
#pragma unroll
                        for (int j = 0; j < COLUMNS; ++j) {
                            acc[i][j][0] = fma_f32x2(both, pack_f32x2(x[j].x, x[j].y), acc[i][j][0]);
                            acc[i][j][1] = fma_f32x2(both, pack_f32x2(x[j].z, x[j].w), acc[i][j][1]);
                        }
                    }
                }
            }
        };
        if (whole) add_up(std::false_type()); else add_up(std::true_type());
        __syncthreads();
    }

#pragma unroll
    for (int i = 0; i < RT; ++i) {
        float sum = run_sum[i];
#pragma unroll
        for (int lanes = 8; lanes > 0; lanes >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, lanes);
        const int row = row0 + ry * RT + i;
        if (row >= rows) continue;
        const int head = kvh * p.group + row % p.group;
        const size_t unit = (size_t)(s.begin + row / p.group) * p.q_heads + head;
        if (p.splits > 1) {
            if (kx == 0) {
                p.part_ml[(unit * p.splits + split) * 2] = run_max[i] * 1.4426950408889634f;
                p.part_ml[(unit * p.splits + split) * 2 + 1] = sum;
            }
            if (run_max[i] == -INFINITY && sum == 0.0f) continue;       // (no key; a sum of NaN: scores of NaN, which maxima leave out)
        }
        float inv = 1.0f;
        if (p.splits == 1) {
            if (p.sinks && sum > 0.0f) sum += expf(p.sinks[head] - run_max[i]);
            inv = run_max[i] == -INFINITY ? sum : 1.0f / sum;           // (0, or NaN)
        }
#pragma unroll
        for (int j = 0; j < COLUMNS; ++j) {
            float o[4];
            unpack_f32x2(acc[i][j][0], o[0], o[1]);
            unpack_f32x2(acc[i][j][1], o[2], o[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = j * 64 + kx * 4 + e;
                if (c >= d) continue;
                if (p.splits > 1)
                    p.part_o[(unit * p.splits + split) * d + c] = o[e];
                else
                    static_cast<A*>(p.out)[unit * d + c] = from_float<A>(o[e] * inv);
            }
        }
    }
}

// Joins the pieces of a row's keys: a warp a (token, query head), the pieces in order. Rows of no span, and of spans that the pieces'
// blocks refused, which have left nothing in scratch, stay as they were: a lane asks about every 32nd span, as those blocks did, while
// the maxima are under way (0.1 us of 37 with two spans).
template <typename A>
__global__ void __launch_bounds__(256) attention_tree_join_kernel(const TreeParams p) {
    chain_wait();
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, d = p.head_dim;
    if (unit >= (long long)p.tokens * p.q_heads) return;
    const int token = (int)(unit / p.q_heads);
    // a lane has the factors of two pieces (64 at most); the outputs of four pieces are asked for together
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + unit * p.splits;
    const float2 none = make_float2(-INFINITY, 0.0f);
    const float2 low = lane < p.splits ? ml[lane] : none, high = lane + 32 < p.splits ? ml[lane + 32] : none;
    bool there = false;
    for (int i = 0; i < p.spans && !there; i += 32) {
        TreeSpan s = {0, 0, 0};
        if (i + lane < p.spans) s = tree_span(p, i + lane, false);
        there = __any_sync(0xffffffffu, token >= s.begin && token - s.begin < s.nodes);
    }
    if (!there) return;
    const float top = warp_max(fmaxf(low.x, high.x));
    // (a piece without a maximum has a sum of 0, or of NaN where it saw NaN alone)
    const float low_factor = low.x == -INFINITY ? low.y : exp2f(low.x - top), high_factor = high.x == -INFINITY ? high.y : exp2f(high.x - top);
    float total = warp_sum(low.y * low_factor + high.y * high_factor);
    if (p.sinks && top != -INFINITY) total += exp2f(p.sinks[unit % p.q_heads] * 1.4426950408889634f - top);
    const float inv = top == -INFINITY ? total : 1.0f / total;
    for (int c = lane; c < d + lane; c += 32) {        // (every lane comes to every exchange)
        float sum = 0.0f;
        for (int i0 = 0; i0 < p.splits; i0 += 4) {
            float factor[4], x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u;
                factor[u] = __shfl_sync(0xffffffffu, i < 32 ? low_factor : high_factor, i & 31);
                x[u] = i < p.splits && c < d && factor[u] != 0.0f ? p.part_o[(unit * p.splits + i) * d + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) sum = i0 + u < p.splits ? fmaf(x[u], factor[u], sum) : sum;
        }
        if (c < d) static_cast<A*>(p.out)[unit * d + c] = from_float<A>(sum * inv);
    }
}

template <typename A, int COLUMNS, bool PIECES>
static int launch_simt_columns(const TreeParams& p, cudaStream_t stream) {
    auto kernel = attention_tree_simt_kernel<A, COLUMNS, PIECES>;
    constexpr size_t smem = SimtLayout<A, COLUMNS>::kBytes;
    static_assert(smem <= 227 * 1024, "a block's shared memory");
    if (smem > 40 * 1024) {
        const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        CELEG_REQUIRE(status == cudaSuccess, "attention_tree: %s", cudaGetErrorString(status));
    }
    const int tiles = (p.max_nodes * p.group + kSimtRows - 1) / kSimtRows;
    launch_chained(kernel, dim3(p.splits, p.kv_heads * tiles, p.spans), dim3(kSimtThreads), smem, stream, p);
    return check_launch("attention_tree");
}

template <typename A, bool PIECES>
static int launch_simt(const TreeParams& p, cudaStream_t stream) {
    if (p.head_dim <= 64) return launch_simt_columns<A, 1, PIECES>(p, stream);
    if (p.head_dim <= 128) return launch_simt_columns<A, 2, PIECES>(p, stream);
    return launch_simt_columns<A, 4, PIECES>(p, stream);
}

template <typename A>
static int launch_join(const TreeParams& p, cudaStream_t stream) {
    const long long units = (long long)p.tokens * p.q_heads;
    launch_chained(attention_tree_join_kernel<A>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, stream, p);
    return check_launch("attention_tree (join)");
}

// Into how many pieces the keys are cut on the tensor cores, one block an SM. `problems`: (row tile, kv head, span)s; `steps`: tiles of keys of the longest. A round
// of blocks costs its tiles and some `ends` more for a block's beginning and end. Up to `cluster` pieces meet in a cluster,
// which costs little, but a cluster wants neighbouring SMs; more pieces, as many as scratch holds, want a second launch.
static int tree_splits_tcgen05(long long problems, const TreeTile& tile, long long steps, long long room) {
    long long best = 1, least = 0;
    for (long long splits = 1; splits <= 64 && splits <= steps && (splits <= tile.cluster || splits <= room); ++splits) {
        const long long at_once = splits <= tile.cluster ? tile.problems_at_once[splits] : 0;
        const long long rounds = at_once > 0 ? (problems + at_once - 1) / at_once : (problems * splits + tile.blocks - 1) / tile.blocks;
        const long long joining = splits == 1 ? 0 : splits <= tile.cluster ? 4 : 8;
        const long long cost = 4 * (rounds * ((steps + splits - 1) / splits + tile.ends) + joining) + splits;
        if (splits == 1 || cost < least) best = splits, least = cost;
    }
    return (int)best;
}

// ... and for the general kernel, whose blocks, several an SM, follow one another as they end: all blocks' tiles, with `ends` more a
// block, spread over the places, and the last block's behind them; a join costs about as much as a tile. (Eight requests of 32 nodes
// behind up to 4,096 positions, float32, heads of 64: 196 us in the 9 pieces that it takes, 206 in 12, 220 in 16, 247 in 24; 8 heads
// of 256: 329, 379, 415, 497; two requests of 24 behind 1,500: 39 us in 9, 37 in the 12 that it takes, 40 in 16, 47 in 24.)
static int tree_splits_simt(long long problems, int head_dim, long long steps, long long room) {
    const double places = head_dim <= 64 ? 592 : head_dim <= 128 ? 296 : 148, ends = 3;
    long long best = 1;
    double least = 0;
    for (long long splits = 1; splits <= 64 && splits <= steps && (splits == 1 || splits <= room); ++splits) {
        const double cost = (double)problems * (steps + splits * ends) / places + (double)((steps + splits - 1) / splits) + ends + (splits > 1 ? 1 : 0);
        if (splits == 1 || cost < least) best = splits, least = cost;
    }
    return (int)best;
}

}  // namespace celeg_b200

using namespace celeg_b200;

// The arguments of the entry point, one record. q: [tokens, q_row_stride] with head h at columns h * head_dim; caches: one
// layer's [pages, kv_heads, page_tokens, head_dim], page_stride elements from page to page; span_begin [spans + 1],
// span_context [spans], ancestors [tokens, words] (words of 32 bits), block_table [spans, table_columns], rows table_stride apart; sinks [q_heads] or
// null; out [tokens, q_heads * head_dim]. max_nodes: no span has more nodes (error 4 else); max_keys: about as many keys as the
// longest span has, which only the number of pieces follows. scratch: float32, any number of elements; the keys are cut into
// no more pieces than it holds where these do not meet in a cluster.
struct TreeArguments {
    const void *q;
    void* out;
    const void *k_cache, *v_cache;
    const int *positions, *span_begin, *span_context, *ancestors, *block_table;
    const float* sinks;
    float* scratch;
    int* error_flag;
    cudaStream_t stream;
    long long q_row_stride, page_stride, scratch_elements;
    int pages, words, table_stride, tokens, spans, max_nodes, max_keys, q_heads, kv_heads, head_dim, page_tokens, window, act_dtype;
    float scale, softcap;
    int table_columns;
};
static_assert(sizeof(TreeArguments) == 192, "the record that kernels.py packs");

CELEG_API int celeg_attention_tree(const void* record) {
    TreeArguments a;
    memcpy(&a, record, sizeof(a));
    const int tokens = a.tokens, spans = a.spans, max_nodes = a.max_nodes, max_keys = a.max_keys, q_heads = a.q_heads, kv_heads = a.kv_heads;
    const int head_dim = a.head_dim, page_tokens = a.page_tokens, words = a.words, window = a.window, act_dtype = a.act_dtype;
    const long long page_stride = a.page_stride;
    const float scale = a.scale, softcap = a.softcap;
    // (scratch is used from a 16-byte address on)
    const long long skipped = (long long)((16 - ((size_t)a.scratch & 15)) & 15) / 4;
    float* scratch = a.scratch && a.scratch_elements > skipped ? a.scratch + skipped : nullptr;
    const long long scratch_elements = scratch ? a.scratch_elements - skipped : 0;
    cudaStream_t stream = a.stream;
    CELEG_REQUIRE(tokens >= 0 && spans >= 0 && q_heads > 0 && kv_heads > 0 && head_dim > 0 && page_tokens > 0 && max_keys >= 0,
                  "attention_tree: invalid sizes tokens=%d spans=%d q_heads=%d kv_heads=%d head_dim=%d page_tokens=%d", tokens,
                  spans, q_heads, kv_heads, head_dim, page_tokens);
    CELEG_REQUIRE(q_heads % kv_heads == 0, "attention_tree: %d query heads are not a multiple of %d kv heads", q_heads, kv_heads);
    CELEG_REQUIRE(head_dim <= 256, "attention_tree: a head size of %d exceeds 256", head_dim);
    CELEG_REQUIRE(max_nodes >= 1 && max_nodes <= kTreeMaxNodes && words >= (max_nodes + 31) / 32,
                  "attention_tree: trees of up to %d nodes (at most %d) need masks of %d words, got %d", max_nodes, kTreeMaxNodes,
                  (max_nodes + 31) / 32, words);
    CELEG_REQUIRE(window >= 0 && softcap >= 0.0f && a.error_flag, "attention_tree: window %d, softcap %g, error_flag %p", window,
                  softcap, (void*)a.error_flag);
    CELEG_REQUIRE(act_dtype == kFloat32 || act_dtype == kBFloat16, "attention_tree: unknown dtype code %d", act_dtype);
    CELEG_REQUIRE(a.table_stride >= 0 && a.table_columns >= 0, "attention_tree: a table of %d columns, rows %d apart", a.table_columns, a.table_stride);
    if (tokens == 0 || spans == 0) return 0;
    const int group = q_heads / kv_heads;
    const long long tiles = ((long long)max_nodes * group + 31) / 32;
    CELEG_REQUIRE(spans <= 65535 && kv_heads * tiles <= 65535 && (long long)max_nodes * group <= 1 << 24,
                  "attention_tree: %d spans of %d nodes on %d heads exceed one launch", spans, max_nodes, q_heads);
    TreeParams p = {};
    p.q = a.q;
    p.q_row_stride = a.q_row_stride;
    p.out = a.out;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.page_stride = page_stride;
    p.pages = a.pages;
    p.positions = a.positions;
    p.span_begin = a.span_begin;
    p.span_context = a.span_context;
    p.ancestors = reinterpret_cast<const unsigned*>(a.ancestors);
    p.words = words;
    p.block_table = a.block_table;
    p.table_stride = a.table_stride;
    p.table_columns = a.table_columns;
    p.tokens = tokens;
    p.spans = spans;
    p.max_nodes = max_nodes;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.group = group;
    p.head_dim = head_dim;
    p.page_tokens = page_tokens;
    p.window = window;
    p.page_shift = -1;
    for (int shift = 0; shift < 31; ++shift)
        if (page_tokens == 1 << shift) p.page_shift = shift;
    p.scale = scale;
    p.sinks = a.sinks;
    p.cap_in = softcap > 0.0f ? scale / softcap : 0.0f;
    p.cap_out = softcap;
    p.error_flag = a.error_flag;
    const long long units = (long long)tokens * q_heads;
    p.part_o = scratch;
    const bool tensor_cores = act_dtype == kBFloat16 && tree_tcgen05_takes(p);
    const size_t size = act_dtype == kFloat32 ? 4 : 2;
    const bool pieces = head_dim * size % 16 == 0 && page_stride * size % 16 == 0 && (((size_t)a.k_cache | (size_t)a.v_cache) & 15) == 0;
    const long long reach = window > 0 && (long long)window + max_nodes < max_keys ? (long long)window + max_nodes : max_keys;
    const long long steps = (reach + 63) / 64, room = scratch ? (scratch_elements - 1) / (units * (head_dim + 2)) : 0;
    const long long heads = (long long)spans * kv_heads, rows = (long long)max_nodes * group;
    if (tensor_cores) {
        const TreeTile tile = tree_tcgen05_tile(p);
        p.splits = tree_splits_tcgen05(heads * ((rows + tile.rows - 1) / tile.rows), tile, steps, room);
        if (p.splits <= tile.cluster) p.part_o = nullptr;
    } else {
        p.splits = tree_splits_simt(heads * ((rows + kSimtRows - 1) / kSimtRows), head_dim, steps, room);
        if (p.splits == 1) p.part_o = nullptr;
    }
    p.part_ml = p.part_o ? scratch + (units * p.splits * head_dim + 1) / 2 * 2 : nullptr;      // (read as pairs)
    int code;
    if (tensor_cores)
        code = launch_tree_tcgen05(p, stream);
    else if (act_dtype == kFloat32)
        code = pieces ? launch_simt<float, true>(p, stream) : launch_simt<float, false>(p, stream);
    else
        code = pieces ? launch_simt<__nv_bfloat16, true>(p, stream) : launch_simt<__nv_bfloat16, false>(p, stream);
    if (code != 0 || !p.part_o) return code;
    return act_dtype == kFloat32 ? launch_join<float>(p, stream) : launch_join<__nv_bfloat16>(p, stream);
}
