// The split kernels of head size 64 over an e4m3 cache.
#include "paged_split_sm100.cuh"

CHIA_INSTANTIATE_SPLIT(64, chia::CACHE_E4M3)
