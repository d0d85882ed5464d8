// ipc_ckpt_weight.hip - weight update from a state kept in 8 bits:
// W += alpha E f(X)^T (layout WGT, B the packed state).
#include "ipc_chunk_kernel.h"
#include "ipc_gemm_kernel.h"

namespace ipc {
namespace {

template <typename ST, typename OT>
hipError_t run(const GemmProblem& p, int tile, hipStream_t s) {
  if (tile >= TILE_CHUNK_16) return chunk::run_chunks<ST, OT, LAYOUT_WGT, 1, true>(&p, 1, tile, s);
  return run_tiles<ST, OT, LAYOUT_WGT, 1, true>(&p, 1, tile, s);
}

}  // namespace

hipError_t launch_ckpt_weight(const GemmProblem& p, int storage, int operand, int tile, hipStream_t s) {
  if (storage == DT_F32) {
    if (operand == DT_F32) return run<float, float>(p, tile, s);
    if (operand == DT_F16) return run<float, f16>(p, tile, s);
    return run<float, bf16>(p, tile, s);
  }
  if (storage == DT_F16) return run<f16, f16>(p, tile, s);
  return run<bf16, bf16>(p, tile, s);
}

}  // namespace ipc
