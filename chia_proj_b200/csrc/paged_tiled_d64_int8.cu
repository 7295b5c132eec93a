// The tiled kernels of head size 64 over an int8 cache.
#include "paged_tiled_sm100.cuh"

CHIA_INSTANTIATE_TILED(64, chia::CACHE_INT8)
