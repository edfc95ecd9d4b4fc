// Host helpers shared by the translation units of the library.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace xf {
// printf-style setter of the calling thread's last-error text (read by xf_last_error_string()).
void set_error(const char* fmt, ...);
const char* last_error();
// Tensor map of a row-major [d2][d1][d0] array with boxes of b0 x b1 x 1 elements; elements outside the
// array load as zero.  False, with the error text set, if the driver refuses it.
bool encode_3d(CUtensorMap* tm, CUtensorMapDataType dt, const void* base, uint64_t d0, uint64_t d1,
               uint64_t d2, uint64_t stride1_bytes, uint64_t stride2_bytes, uint32_t b0, uint32_t b1,
               CUtensorMapSwizzle sw);
}  // namespace xf
