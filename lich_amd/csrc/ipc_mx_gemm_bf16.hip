// ipc_mx_gemm_bf16.hip - products of microscaled fp4 matrices, bf16 tensors in the epilogue.
#include "ipc_mx_gemm.h"

namespace ipc {

hipError_t launch_mx_product_bf16(const MxProblem& p, hipStream_t s) { return mx::run_storage<bf16>(p, s); }

}  // namespace ipc
