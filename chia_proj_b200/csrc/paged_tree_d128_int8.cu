// The kernels for trees of drafted tokens of head size 128 over an int8 cache.
#include "paged_split_sm100.cuh"
#include "paged_tiled_sm100.cuh"

CHIA_INSTANTIATE_SPLIT_TREE(128, chia::CACHE_INT8)
CHIA_INSTANTIATE_TILED_TREE(128, chia::CACHE_INT8)
