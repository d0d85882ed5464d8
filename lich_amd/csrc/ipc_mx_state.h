// ipc_mx_state.h - reading a state kept in 8 bits (microscaled int8) in a GEMM.
//
// Codes [rows][row bytes], scales [ceil(n / 128)][rows][4] (ipc_mx.h).  A value is
// its code times a power of two: exact in fp32, and in bf16, whose 8 significant
// bits hold any code.
#pragma once

#include "ipc_mx_device.h"

namespace ipc {
namespace mx {

// Four values of row r from column n on (n a multiple of 4).
__device__ __forceinline__ void state4(const uint8_t* codes, long long row_bytes, const uint8_t* scales,
                                       long long rows, int r, int n, float (&o)[4]) {
  const unsigned q = *reinterpret_cast<const unsigned*>(codes + r * row_bytes + n);
  const float unit = int8_scale(scales[((n >> 7) * rows + r) * 4 + ((n >> 5) & 3)]);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (float)sext8(q, i) * unit;
}

}  // namespace mx
}  // namespace ipc
