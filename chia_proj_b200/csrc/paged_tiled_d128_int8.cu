// The tiled kernels of head size 128 over an int8 cache.
#include "paged_tiled_sm100.cuh"

CHIA_INSTANTIATE_TILED(128, chia::CACHE_INT8)
