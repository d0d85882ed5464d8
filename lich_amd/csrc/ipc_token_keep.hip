// ipc_token_keep.hip - logits' statistics, and the exponentials of a whole vocabulary that is one piece.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, bool SPLIT>
hipError_t run(const TokenGemm& p, int tile, hipStream_t s) {
  if constexpr (!SPLIT) {
    if (tile == TILE_256) return token::run_tile<OT, SPLIT, TOKEN_KEEP, false, 256, 256, 2, 4>(p, s);
  }
  if (tile == TILE_128) return token::run_tile<OT, SPLIT, TOKEN_KEEP, false, 128, 128, 2, 2, SPLIT ? 3 : 4>(p, s);
  if (tile == TILE_128_64) return token::run_tile<OT, SPLIT, TOKEN_KEEP, false, 128, 64, 2, 2, SPLIT ? 4 : 6>(p, s);
  return token::run_narrow<OT, SPLIT, TOKEN_KEEP, false, 2, 2>(p, s);
}

}  // namespace

hipError_t launch_token_keep(const TokenGemm& p, int storage, int tile, hipStream_t s) {
  if (storage == 0) return run<bf16, true>(p, tile, s);
  return storage == 1 ? run<f16, false>(p, tile, s) : run<bf16, false>(p, tile, s);
}

}  // namespace ipc
