// ipc_ckpt_dma.hip - the weight update from a state kept in 8 bits on the LDS-DMA
// kernel (ipc_dma_gemm.h, 16-bit storage), where the caller lends no workspace: its
// loader widens 8 codes and their scale where the 16-bit kernel widens 8 values.
// Tile configurations and waves are those of the 16-bit kernel (ipc_s16_tiles.h).
#include "ipc_dma_gemm.h"

namespace ipc {
namespace {

template <typename OT>
struct ForType {
  template <int ACT>
  struct Run {
    static hipError_t run(const WideProblem* p, int cfg, hipStream_t s) {
      return cfg == 3 ? dma::Cfg<OT, S16_WEIGHT8, 1, ACT, true, 256, 256, 2, 2, 4>::launch(p, 1, s)
                      : dma::Cfg<OT, S16_WEIGHT8, 1, ACT, true, 256, 128, 3, 4, 2>::launch(p, 1, s);
    }
  };
};

}  // namespace

hipError_t launch_s16_weight8(const WideProblem& p, int operand, int act, int cfg, hipStream_t s) {
  if (operand == DT_F16) return dma::by_act<ForType<f16>::Run>(act, &p, cfg, s);
  return dma::by_act<ForType<bf16>::Run>(act, &p, cfg, s);
}

}  // namespace ipc
