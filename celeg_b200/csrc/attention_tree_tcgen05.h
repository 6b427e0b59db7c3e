// The tree attention on tcgen05 as attention_tree.cu sees it.
#pragma once

#include "attention_tree.cuh"

namespace celeg_b200 {

// Whether the sizes, strides and addresses of `p` fit it.
bool tree_tcgen05_takes(const TreeParams& p);
// Rows of one of its tiles.
int tree_tcgen05_rows();
// p.splits pieces of the keys; 0 or a negative code with the library's error text.
int launch_tree_tcgen05(const TreeParams& p, cudaStream_t stream);

}  // namespace celeg_b200
