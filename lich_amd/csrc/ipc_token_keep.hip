// ipc_token_keep.hip - logits' statistics, and the exponentials of a whole vocabulary that is one piece.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, int TERMS, bool TWO>
hipError_t run(const TokenGemm& p, int tile, hipStream_t s) {
  constexpr int M = TWO ? 4 : 2, N = TWO ? 1 : 2;  // (two terms: both in one wave)
  if constexpr (TERMS == 1) {
    if (tile == TILE_256) return token::run_tile<OT, TERMS, TOKEN_KEEP, TWO, 256, 256, 2, 4>(p, s);
  }
  if (tile == TILE_128) return token::run_tile<OT, TERMS, TOKEN_KEEP, TWO, 128, 128, 2, 2, TERMS == 3 ? 3 : 4>(p, s);
  if (tile == TILE_128_64) return token::run_tile<OT, TERMS, TOKEN_KEEP, TWO, 128, 64, M, N, TERMS == 3 ? 4 : 6>(p, s);
  return token::run_narrow<OT, TERMS, TOKEN_KEEP, TWO, 2, N>(p, s);
}

}  // namespace

hipError_t launch_token_keep(const TokenGemm& p, int storage, int tile, bool two, hipStream_t s) {
  if (storage == 0) return run<bf16, 3, false>(p, tile, s);
  if (two) return storage == 1 ? run<f16, 1, true>(p, tile, s) : run<bf16, 1, true>(p, tile, s);
  return storage == 1 ? run<f16, 1, false>(p, tile, s) : run<bf16, 1, false>(p, tile, s);
}

}  // namespace ipc
