"""B200-native SBNet block ops: reduce_mask, sparse_gather, sparse_scatter[_var], and layer norm and the gated feed-forward
block over the rows of a block stack (sm_100a CUDA behind a C ABI)."""
