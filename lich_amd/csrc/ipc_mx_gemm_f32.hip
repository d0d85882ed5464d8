// ipc_mx_gemm_f32.hip - products of microscaled fp4 matrices, float tensors in the epilogue.
#include "ipc_mx_gemm.h"

namespace ipc {

hipError_t launch_mx_product_f32(const MxProblem& p, hipStream_t s) { return mx::run_storage<float>(p, s); }

}  // namespace ipc
