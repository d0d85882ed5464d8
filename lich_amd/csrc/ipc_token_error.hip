// ipc_token_error.hip - errors of a piece of the vocabulary, its logits formed again.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, int TERMS>
hipError_t run(const TokenGemm& p, int tile, hipStream_t s) {
  if constexpr (TERMS == 1) {
    if (tile == TILE_256) return token::run_tile<OT, TERMS, TOKEN_ERROR, 1, 256, 256, 2, 4>(p, s);
  }
  if (tile == TILE_128) return token::run_tile<OT, TERMS, TOKEN_ERROR, 1, 128, 128, 2, 2, TERMS == 3 ? 3 : 4>(p, s);
  if (tile == TILE_128_64) return token::run_tile<OT, TERMS, TOKEN_ERROR, 1, 128, 64, 2, 2, TERMS == 3 ? 4 : 6>(p, s);
  return token::run_narrow<OT, TERMS, TOKEN_ERROR, 1, 2, 2>(p, s);
}

}  // namespace

hipError_t launch_token_error(const TokenGemm& p, int storage, int tile, hipStream_t s) {
  if (storage == 0) return run<bf16, 3>(p, tile, s);
  return storage == 1 ? run<f16, 1>(p, tile, s) : run<bf16, 1>(p, tile, s);
}

}  // namespace ipc
