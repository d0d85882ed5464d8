// ipc_ckpt_gemm.hip - the backward pass of a state kept in 8 bits as 16-bit products.
#include "ipc_ckpt_gemm.h"

namespace ipc {
namespace {

template <typename OT>
hipError_t run(int mode, const CkptProblem& p, int act, hipStream_t s) {
  if (mode == CKPT_WEIGHT) return mx::run_ckpt<OT, CKPT_WEIGHT, ACT_IDENTITY>(p, s);
  switch (act) {
    case ACT_RELU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_RELU>(p, s);
    case ACT_TANH: return mx::run_ckpt<OT, CKPT_GRAD, ACT_TANH>(p, s);
    case ACT_SIGMOID: return mx::run_ckpt<OT, CKPT_GRAD, ACT_SIGMOID>(p, s);
    case ACT_SILU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_SILU>(p, s);
    case ACT_GELU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_GELU>(p, s);
    default: return mx::run_ckpt<OT, CKPT_GRAD, ACT_IDENTITY>(p, s);
  }
}

}  // namespace

hipError_t launch_ckpt_gemm(int mode, const CkptProblem& p, int operand, int act, hipStream_t s) {
  return operand == DT_F16 ? run<f16>(mode, p, act, s) : run<bf16>(mode, p, act, s);
}

}  // namespace ipc
