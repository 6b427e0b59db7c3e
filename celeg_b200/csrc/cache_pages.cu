// What moves inside the paged cache without a model step: whole pages or their first positions into other pages (a request
// that is forked, beams that are reordered), and the accepted path of a tree of drafted tokens to the places behind the
// cached ones. Both take all layers of a group in one launch, keys and values together, and move bytes: any element type.
//
// Caches: [layers, pages, kv_heads, page_tokens, row], a row being the bytes of one head at one position.
#include "common.cuh"

#include <cstdlib>
#include <cstring>

namespace celeg_b200 {

struct CacheSide {
    unsigned char* base;               // null: nothing is cached on this side
    long long layer_stride, page_stride;      // bytes
    int row;                           // bytes
};

struct PageMove { int from, to, rows; };

// The moves travel as a kernel argument: the host knows them, and nothing has to be staged.
template <int N>
struct PageMoves {
    PageMove move[N];
};

constexpr int kFewMoves = 32, kManyMoves = 1024;

// One (move, layer) a block in x, keys or values in y. V: what a thread moves at a time; four of them are under way. A page of 16
// positions x 8 heads x 64 is 16 KiB, a pass of 256 threads: every block asks for all that it moves at once. 768 pages in sixteen
// layers, keys and values (805 MB read and written together), take 125 us, 6,440 GB/s, what a copy reaches here; a fork's one
// page in six layers 1.9 us, a launch.
template <typename V, int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageMoves<N> moves, const int layers, const CacheSide k,
                                                         const CacheSide v, const int kv_heads, const int page_tokens) {
    const CacheSide& side = blockIdx.y ? v : k;
    const PageMove m = moves.move[blockIdx.x / layers];
    unsigned char* layer = side.base + (blockIdx.x % layers) * side.layer_stride;
    const unsigned char* from = layer + m.from * side.page_stride;
    unsigned char* to = layer + m.to * side.page_stride;
    const int head_bytes = page_tokens * side.row;
    const int per_head = (m.rows == page_tokens ? kv_heads * head_bytes : m.rows * side.row) / (int)sizeof(V);
    const int heads = m.rows == page_tokens ? 1 : kv_heads;
    const int total = heads * per_head;
    for (int i0 = threadIdx.x; i0 < total; i0 += 4 * 256) {
        V value[4];
        long long at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 256;
            if (i >= total) continue;
            at[u] = (long long)(i / per_head) * head_bytes + (long long)(i % per_head) * (int)sizeof(V);
            value[u] = *reinterpret_cast<const V*>(from + at[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * 256 < total) *reinterpret_cast<V*>(to + at[u]) = value[u];
    }
}

template <typename V, int N>
static void launch_copy(const PageMove* list, int count, int layers, const CacheSide& k, const CacheSide& v, int kv_heads,
                        int page_tokens, cudaStream_t stream) {
    PageMoves<N> moves;
    for (int i = 0; i < count; ++i) moves.move[i] = list[i];
    // (only keys, or only values: the side that is there)
    const CacheSide& first = k.base ? k : v;
    copy_pages_kernel<V, N><<<dim3((unsigned)(count * layers), k.base && v.base ? 2 : 1), 256, 0, stream>>>(moves, layers, first, v, kv_heads,
                                                                                                         page_tokens);
}

// The size of a piece that every row, page and layer of both caches is a multiple of, from an address that is one too.
static int piece_bytes(const CacheSide& k, const CacheSide& v) {
    unsigned long long bits = 16;
    for (const CacheSide* side : {&k, &v})
        if (side->base) bits |= (unsigned long long)side->base | (unsigned long long)side->layer_stride |
                                (unsigned long long)side->page_stride | (unsigned long long)side->row;
    for (int bytes = 16; bytes > 2; bytes /= 2)
        if ((bits & (bytes - 1)) == 0) return bytes;
    return 2;
}

// The first move that writes a page which another move writes, or reads one which another move writes; -1: none, -2: no memory.
// A table of the written pages, open addressing, at most half full; the usual lists' on the stack.
static int clashing_move(const PageMove* list, int count) {
    constexpr int kOnStack = 4096;
    int on_stack[kOnStack];
    long long size = 16;
    while (size < 2ll * count) size *= 2;
    int* table = size <= kOnStack ? on_stack : static_cast<int*>(malloc((size_t)size * sizeof(int)));
    if (!table) return -2;
    const unsigned mask = (unsigned)(size - 1);
    for (long long i = 0; i < size; ++i) table[i] = -1;
    int clash = -1;
    auto place = [&](int page) {
        unsigned at = ((unsigned)page * 2654435761u) >> 7 & mask;
        while (table[at] >= 0 && table[at] != page) at = (at + 1) & mask;
        return at;
    };
    for (int i = 0; i < count && clash < 0; ++i) {
        const unsigned at = place(list[i].to);
        if (table[at] >= 0) clash = i;
        table[at] = list[i].to;
    }
    for (int i = 0; i < count && clash < 0; ++i)
        if (list[i].from != list[i].to && table[place(list[i].from)] >= 0) clash = i;
    if (table != on_stack) free(table);
    return clash;
}

// ------------------------------------------------------------------------------------------------ accepted drafts
constexpr int kKeepThreads = 256;
constexpr int kKeepMaxNodes = 256;

struct KeepParams {
    CacheSide k, v;
    const int* parents;            // [tokens], within the span; -1: the root, node 0
    const int* tokens;             // [tokens]
    const int* chosen;             // [tokens]: what the model continues each node with
    const int* span_begin;
    const int* span_context;
    const int* block_table;        // [spans, table_columns], rows table_stride apart
    int table_stride, table_columns, pages, token_count, layers, kv_heads, page_tokens, max_nodes;
    int* path;                     // [spans, max_nodes], -1 behind the accepted nodes
    int* accepted;                 // [spans]
    int* next_token;               // [spans], -1 for a span without nodes
    int* error_flag;
};

// A block in y is a span, blocks in x share its columns: a thread owns a piece of a row (one layer, keys or values, one head)
// and moves it for the whole path, in order. Path nodes rise and node n of the path is n or later, so that a row is read
// before its place is written, within the thread that does both; no row is another thread's.
// Every block walks the tree for itself, one warp with up to eight nodes a lane: a step is a ballot of "child of the current node with the
// chosen token" over each 32 nodes, the lowest wins. The chain of reads, span, tree, table, rows, is what bounds it: 3.8 us for one
// request in six layers, 5.1 us for 64 of 32 drafts in sixteen (8.4 MB, 1.3 us at the memory's rate).
template <typename V>
__global__ void __launch_bounds__(kKeepThreads) keep_drafts_kernel(const KeepParams p) {
    __shared__ int path_s[kKeepMaxNodes];
    __shared__ long long from_s[kKeepMaxNodes][2], to_s[kKeepMaxNodes][2];      // byte offsets of the moved rows, keys and values
    __shared__ int accepted_s, moved_s;
    const int span = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int begin = p.span_begin[span], nodes = p.span_begin[span + 1] - begin, context = p.span_context[span];
    if (begin < 0 || nodes < 0 || begin > p.token_count - nodes || nodes > p.max_nodes || context < 0 ||
        context > 0x7fffffff - kKeepMaxNodes) {
        if (blockIdx.x == 0) {
            for (int n = tid; n < p.max_nodes; n += kKeepThreads) p.path[(size_t)span * p.max_nodes + n] = -1;
            if (tid == 0) {
                p.accepted[span] = 0;
                p.next_token[span] = -1;
                atomicExch(p.error_flag, 4);
            }
        }
        return;
    }
    if (tid < 32) {
        int parent[kKeepMaxNodes / 32], token[kKeepMaxNodes / 32];
#pragma unroll
        for (int w = 0; w < kKeepMaxNodes / 32; ++w) {
            const int node = w * 32 + lane;
            parent[w] = node < nodes ? p.parents[begin + node] : -1;
            token[w] = node < nodes ? p.tokens[begin + node] : 0;
        }
        int current = 0, count = 0, next = -1;
        while (current < nodes) {
            if (lane == 0) path_s[count] = current;
            ++count;
            next = p.chosen[begin + current];
            int child = nodes;
#pragma unroll
            for (int w = kKeepMaxNodes / 32 - 1; w >= 0; --w) {
                const int node = w * 32 + lane;
                const unsigned fits = __ballot_sync(0xffffffffu, node > current && node < nodes && parent[w] == current && token[w] == next);
                if (fits) child = w * 32 + __ffs(fits) - 1;
            }
            current = child;
        }
        __syncwarp();
        if (blockIdx.x == 0) {
            for (int n = lane; n < p.max_nodes; n += 32) p.path[(size_t)span * p.max_nodes + n] = n < count ? path_s[n] : -1;
            if (lane == 0) {
                p.accepted[span] = count;
                p.next_token[span] = next;
            }
        }
        if (lane == 0) accepted_s = count;
    }
    __syncthreads();
    // the rows that move: all from the first node that is not in its place already (behind a gap all are)
    const int accepted = accepted_s;
    if (tid == 0) {
        int n = 0;
        while (n < accepted && path_s[n] == n) ++n;
        moved_s = n;
    }
    __syncthreads();
    const int first = moved_s;
    const int* table = p.block_table + (size_t)span * p.table_stride;
    for (int n = first + tid; n < accepted; n += kKeepThreads) {
        const int place[2] = {context + path_s[n], context + n};
        long long at[2][2];
        bool found = true;
        for (int e = 0; e < 2; ++e) {
            const int logical = place[e] / p.page_tokens;
            const int page = logical < p.table_columns ? table[logical] : -1;
            found = found && page >= 0 && page < p.pages;
            at[e][0] = page * p.k.page_stride + (long long)(place[e] % p.page_tokens) * p.k.row;
            at[e][1] = page * p.v.page_stride + (long long)(place[e] % p.page_tokens) * p.v.row;
        }
        if (!found) atomicExch(p.error_flag, 1);
        for (int side = 0; side < 2; ++side) {
            from_s[n][side] = found ? at[0][side] : -1;
            to_s[n][side] = at[1][side];
        }
    }
    __syncthreads();
    const int k_pieces = p.k.base ? p.k.row / (int)sizeof(V) : 0, v_pieces = p.v.base ? p.v.row / (int)sizeof(V) : 0;
    const long long per_layer = (long long)p.kv_heads * (k_pieces + v_pieces);
    const long long column = (long long)blockIdx.x * kKeepThreads + tid;
    if (column >= per_layer * p.layers) return;
    const long long layer = column / per_layer;
    long long rest = column % per_layer;
    const int side = rest >= (long long)p.kv_heads * k_pieces;
    if (side) rest -= (long long)p.kv_heads * k_pieces;
    const CacheSide& cache = side ? p.v : p.k;
    const int pieces = side ? v_pieces : k_pieces;
    unsigned char* base = cache.base + layer * cache.layer_stride + (rest / pieces) * p.page_tokens * (long long)cache.row +
                          (rest % pieces) * (int)sizeof(V);
    for (int n0 = first; n0 < accepted; n0 += 8) {
        V value[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (n0 + u < accepted && from_s[n0 + u][side] >= 0) value[u] = *reinterpret_cast<const V*>(base + from_s[n0 + u][side]);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (n0 + u < accepted && from_s[n0 + u][side] >= 0) *reinterpret_cast<V*>(base + to_s[n0 + u][side]) = value[u];
    }
}

template <typename V>
static void launch_keep(const KeepParams& p, int spans, cudaStream_t stream) {
    const long long columns = (long long)p.layers * p.kv_heads * ((p.k.base ? p.k.row : 0) + (p.v.base ? p.v.row : 0)) / (long long)sizeof(V);
    const unsigned blocks = (unsigned)((columns + kKeepThreads - 1) / kKeepThreads);
    keep_drafts_kernel<V><<<dim3(blocks > 0 ? blocks : 1, spans), kKeepThreads, 0, stream>>>(p);
}

}  // namespace celeg_b200

using namespace celeg_b200;

static CacheSide cache_side(void* base, long long layer_stride, long long page_stride, int dim, int element_bytes) {
    return {dim > 0 ? (unsigned char*)base : nullptr, layer_stride * element_bytes, page_stride * element_bytes, dim * element_bytes};
}

// Both entry points take one record. Of the caches: k, v [layers, pages, kv_heads, page_tokens, k_dim or v_dim]; strides in
// elements of keys' layers and pages and of values' layers and pages, the last three sizes contiguous; sizes k_dim, v_dim,
// layers, pages, kv_heads, page_tokens, bytes of an element; a dimension of 0: nothing is kept on that side.

// moves: `count` triples (from, to, rows) in host memory: the first `rows` positions of page `to` become those of page `from`, in
// every layer. No page may be written twice, nor written and read (a page onto itself aside): the moves run at the same time.
CELEG_API int celeg_copy_pages(const void* record) {
    struct { void *k, *v; const int* moves; cudaStream_t stream; long long strides[4]; int sizes[7], count; } a;
    static_assert(sizeof(a) == 96, "the record that kernels.py packs");
    memcpy(&a, record, sizeof(a));
    const int k_dim = a.sizes[0], v_dim = a.sizes[1], layers = a.sizes[2], pages = a.sizes[3], kv_heads = a.sizes[4];
    const int page_tokens = a.sizes[5], element_bytes = a.sizes[6], count = a.count;
    const int* moves = a.moves;
    cudaStream_t stream = a.stream;
    CELEG_REQUIRE(layers > 0 && pages > 0 && kv_heads > 0 && page_tokens > 0 && k_dim >= 0 && v_dim >= 0 && count >= 0 &&
                      (element_bytes == 2 || element_bytes == 4),
                  "copy_pages: invalid sizes layers=%d pages=%d kv_heads=%d page_tokens=%d dims %d / %d count=%d element %d", layers,
                  pages, kv_heads, page_tokens, k_dim, v_dim, count, element_bytes);
    const CacheSide ks = cache_side(a.k, a.strides[0], a.strides[1], k_dim, element_bytes);
    const CacheSide vs = cache_side(a.v, a.strides[2], a.strides[3], v_dim, element_bytes);
    CELEG_REQUIRE(layers <= (1 << 30) / kManyMoves && (long long)kv_heads * page_tokens * (k_dim > v_dim ? k_dim : v_dim) * element_bytes < (1ll << 31),
                  "copy_pages: %d layers of pages of %d x %d x %d elements are too large", layers, kv_heads, page_tokens,
                  k_dim > v_dim ? k_dim : v_dim);
    const PageMove* list = reinterpret_cast<const PageMove*>(moves);
    for (int i = 0; i < count; ++i)
        CELEG_REQUIRE(list[i].from >= 0 && list[i].from < pages && list[i].to >= 0 && list[i].to < pages && list[i].rows >= 0 &&
                          list[i].rows <= page_tokens,
                      "copy_pages: move %d (page %d to %d, %d positions) is outside %d pages of %d", i, list[i].from, list[i].to,
                      list[i].rows, pages, page_tokens);
    if (count == 0 || (!ks.base && !vs.base)) return 0;
    const int clash = clashing_move(list, count);
    CELEG_REQUIRE(clash != -2, "copy_pages: no memory to check %d moves", count);
    CELEG_REQUIRE(clash < 0, "copy_pages: move %d (page %d to %d) writes a page that another one writes, or reads one that another one writes",
                  clash, list[clash < 0 ? 0 : clash].from, list[clash < 0 ? 0 : clash].to);
    const int piece = piece_bytes(ks, vs);
    for (int done = 0; done < count;) {
        const int now = count - done > kManyMoves ? kManyMoves : count - done;
#define CELEG_COPY(V)                                                                                                    \
    (now <= kFewMoves ? launch_copy<V, kFewMoves>(list + done, now, layers, ks, vs, kv_heads, page_tokens, stream)        \
                      : launch_copy<V, kManyMoves>(list + done, now, layers, ks, vs, kv_heads, page_tokens, stream))
        if (piece == 16) CELEG_COPY(uint4);
        else if (piece == 8) CELEG_COPY(uint2);
        else if (piece == 4) CELEG_COPY(unsigned);
        else CELEG_COPY(unsigned short);
#undef CELEG_COPY
        done += now;
    }
    return check_launch("copy_pages");
}

// The accepted path of every span's tree: from node 0 on, the lowest child of the path's last node whose token is what the
// model chose there. Rows at places context + path[n] move to context + n in every layer, keys and values.
CELEG_API int celeg_keep_drafts(const void* record) {
    struct {
        void *k, *v;
        const int *parents, *tokens, *chosen, *span_begin, *span_context, *block_table;
        int *path, *accepted, *next_token, *error_flag;
        cudaStream_t stream;
        long long strides[4];
        int sizes[7], token_count, table_stride, spans, max_nodes, table_columns;
    } a;
    static_assert(sizeof(a) == 184, "the record that kernels.py packs");
    memcpy(&a, record, sizeof(a));
    const int k_dim = a.sizes[0], v_dim = a.sizes[1], layers = a.sizes[2], pages = a.sizes[3], kv_heads = a.sizes[4];
    const int page_tokens = a.sizes[5], element_bytes = a.sizes[6], token_count = a.token_count, spans = a.spans, max_nodes = a.max_nodes;
    cudaStream_t stream = a.stream;
    CELEG_REQUIRE(layers > 0 && pages > 0 && kv_heads > 0 && page_tokens > 0 && k_dim >= 0 && v_dim >= 0 && token_count >= 0 &&
                      (element_bytes == 2 || element_bytes == 4),
                  "keep_drafts: invalid sizes layers=%d pages=%d kv_heads=%d page_tokens=%d dims %d / %d element %d", layers, pages,
                  kv_heads, page_tokens, k_dim, v_dim, element_bytes);
    CELEG_REQUIRE(spans >= 0 && spans <= 65535 && max_nodes >= 1 && max_nodes <= kKeepMaxNodes && a.error_flag,
                  "keep_drafts: %d spans of up to %d nodes (at most 65535 and %d)", spans, max_nodes, kKeepMaxNodes);
    CELEG_REQUIRE(a.table_stride >= 0 && a.table_columns >= 0, "keep_drafts: a table of %d columns, rows %d apart", a.table_columns,
                  a.table_stride);
    if (spans == 0) return 0;
    KeepParams p = {};
    p.k = cache_side(a.k, a.strides[0], a.strides[1], k_dim, element_bytes);
    p.v = cache_side(a.v, a.strides[2], a.strides[3], v_dim, element_bytes);
    p.parents = a.parents;
    p.tokens = a.tokens;
    p.chosen = a.chosen;
    p.span_begin = a.span_begin;
    p.span_context = a.span_context;
    p.block_table = a.block_table;
    p.table_stride = a.table_stride;
    p.table_columns = a.table_columns;
    p.pages = pages;
    p.token_count = token_count;
    p.layers = layers;
    p.kv_heads = kv_heads;
    p.page_tokens = page_tokens;
    p.max_nodes = max_nodes;
    p.path = a.path;
    p.accepted = a.accepted;
    p.next_token = a.next_token;
    p.error_flag = a.error_flag;
    const int piece = piece_bytes(p.k, p.v);
    if (piece == 16) launch_keep<uint4>(p, spans, stream);
    else if (piece == 8) launch_keep<uint2>(p, spans, stream);
    else if (piece == 4) launch_keep<unsigned>(p, spans, stream);
    else launch_keep<unsigned short>(p, spans, stream);
    return check_launch("keep_drafts");
}
