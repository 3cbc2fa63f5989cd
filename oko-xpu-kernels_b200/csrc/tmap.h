// Tensor maps for the TMA unit (tmap.cu).
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace xpuint8 {

// 2-D tensor map: `inner` contiguous elements per row, `outer` rows, row
// stride `ld` bytes, swizzled boxes of box_inner x box_outer elements; false with the
// error recorded where the encoder refuses it
bool make_map(CUtensorMap *m, const void *base, uint64_t inner, uint64_t outer, uint64_t ld,
              uint32_t box_inner, uint32_t box_outer,
              CUtensorMapDataType dtype = CU_TENSOR_MAP_DATA_TYPE_UINT8,
              CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B);

}  // namespace xpuint8
