// The tiled kernels of head size 128 over an e4m3 cache.
#include "paged_tiled_sm100.cuh"

CHIA_INSTANTIATE_TILED(128, chia::CACHE_E4M3)
