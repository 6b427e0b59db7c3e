// The tree attention on tcgen05 as attention_tree.cu sees it.
#pragma once

#include "attention_tree.cuh"

namespace celeg_b200 {

// Whether the sizes, strides and addresses of `p` fit it.
bool tree_tcgen05_takes(const TreeParams& p);
// What the choice of the pieces goes by.
struct TreeTile {
    int rows;                      // of a tile
    int blocks;                    // that the GPU runs at a time
    int ends;                      // a block's beginning and end, in tiles of keys
    int cluster;                   // so many pieces of the keys meet without scratch (at most 8),
    int problems_at_once[9];       // and so many (tile, kv head, span)s cut into that many pieces run at a time; 0: blocks / pieces
};
TreeTile tree_tcgen05_tile(const TreeParams& p);
// p.splits pieces of the keys, which meet in scratch if p.part_o is given (and are joined by a launch that follows) and in a
// cluster if not; 0 or a negative code with the library's error text.
int launch_tree_tcgen05(const TreeParams& p, cudaStream_t stream);

}  // namespace celeg_b200
