// ipc_ckpt_gemm32.hip - the backward pass of a state kept in 8 bits on fp32 operands.
#include "ipc_ckpt_gemm32.h"

namespace ipc {
namespace {

template <int SRC>
hipError_t run(const CkptProblem& p, int act, hipStream_t s) {
  switch (act) {
    case ACT_RELU: return mx::run_ckpt32<SRC, ACT_RELU>(p, s);
    case ACT_TANH: return mx::run_ckpt32<SRC, ACT_TANH>(p, s);
    case ACT_SIGMOID: return mx::run_ckpt32<SRC, ACT_SIGMOID>(p, s);
    case ACT_SILU: return mx::run_ckpt32<SRC, ACT_SILU>(p, s);
    case ACT_GELU: return mx::run_ckpt32<SRC, ACT_GELU>(p, s);
    default: return mx::run_ckpt32<SRC, ACT_IDENTITY>(p, s);
  }
}

}  // namespace

hipError_t launch_ckpt_gemm32(int mode, const CkptProblem& p, int act, hipStream_t s) {
  if (mode == CKPT_GRAD) return run<mx::ROWS32>(p, act, s);
  if (p.b) return mx::run_ckpt32<mx::WIDE32, ACT_IDENTITY>(p, s);
  return run<mx::CODES32>(p, act, s);
}

}  // namespace ipc
