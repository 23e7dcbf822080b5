// tensor_map.cuh — TMA tensor maps shared by the tensor-core kernels.
#pragma once
#include <cuda.h>

#include "moe_common.cuh"

namespace moe {

// A tiled tensor map of 16-bit values with SWIZZLE_128B and zero fill (rank <= 5; strides in bytes, rank - 1 of
// them). Defined in expert_gemm_tc.cu.
moe_status encode_tmap_sw128(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                             const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

}  // namespace moe
