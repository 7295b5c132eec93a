// The split kernels of head size 128 over an int8 cache.
#include "paged_split_sm100.cuh"

CHIA_INSTANTIATE_SPLIT(128, chia::CACHE_INT8)
