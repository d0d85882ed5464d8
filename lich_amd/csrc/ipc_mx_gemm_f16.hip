// ipc_mx_gemm_f16.hip - products of microscaled fp4 matrices, f16 tensors in the epilogue.
#include "ipc_mx_gemm.h"

namespace ipc {

hipError_t launch_mx_product_f16(const MxProblem& p, hipStream_t s) { return mx::run_storage<f16>(p, s); }

}  // namespace ipc
