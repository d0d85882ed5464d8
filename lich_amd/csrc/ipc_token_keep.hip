// ipc_token_keep.hip - logits' statistics, and the exponentials of a whole vocabulary that is one piece.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, int TERMS, int WAYS>
hipError_t run(const TokenGemm& p, int tile, hipStream_t s) {
  constexpr int M = WAYS == 2 ? 4 : 2, N = WAYS == 2 ? 1 : 2;  // (all terms in one wave)
  if constexpr (WAYS == 3) {
    if (tile == TILE_128_64) return token::run_tile<OT, TERMS, TOKEN_KEEP, WAYS, 128, 96, 2, 1, 5>(p, s);
    return token::run_tile<OT, TERMS, TOKEN_KEEP, WAYS, 64, 96, 2, 1, 8>(p, s);
  } else {
    if constexpr (TERMS == 1) {
      if (tile == TILE_256) return token::run_tile<OT, TERMS, TOKEN_KEEP, WAYS, 256, 256, 2, 4>(p, s);
    }
    if (tile == TILE_128) return token::run_tile<OT, TERMS, TOKEN_KEEP, WAYS, 128, 128, 2, 2, TERMS == 3 ? 3 : 4>(p, s);
    if (tile == TILE_128_64) return token::run_tile<OT, TERMS, TOKEN_KEEP, WAYS, 128, 64, M, N, TERMS == 3 ? 4 : 6>(p, s);
    return token::run_narrow<OT, TERMS, TOKEN_KEEP, WAYS, 2, N>(p, s);
  }
}

}  // namespace

hipError_t launch_token_keep(const TokenGemm& p, int storage, int tile, int ways, hipStream_t s) {
  if (!token_ways(storage, ways, true)) return hipErrorInvalidValue;
  if (storage == 0) return run<bf16, 3, 1>(p, tile, s);
  if (storage == 1) return ways == 2 ? run<f16, 1, 2>(p, tile, s) : run<f16, 1, 1>(p, tile, s);
  return ways == 3 ? run<bf16, 1, 3>(p, tile, s) : run<bf16, 1, 1>(p, tile, s);
}

}  // namespace ipc
