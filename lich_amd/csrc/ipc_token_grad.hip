// ipc_token_grad.hip - the state's gradient from a piece's errors, the vocabulary cut into slices.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

// Two terms of the errors, side by side: tiles of as many different columns, but for the widest.
template <typename OT>
hipError_t grad_of_two(const TokenGemm& p, int tile, hipStream_t s) {
  if (tile == 256) return token::run_tile<OT, 1, TOKEN_GRAD, 2, 256, 256, 2, 2>(p, s);
  if (tile == 128 && p.N > 64) return token::run_tile<OT, 1, TOKEN_GRAD, 2, 128, 256, 2, 2>(p, s);
  if (tile == 128) return token::run_tile<OT, 1, TOKEN_GRAD, 2, 128, 128, 2, 2>(p, s);
  return token::run_tile<OT, 1, TOKEN_GRAD, 2, 64, 128, 2, 2, 6>(p, s);
}

template <typename OT, int TERMS>
hipError_t grad(const TokenGemm& p, int tile, hipStream_t s) {
  if constexpr (TERMS == 1) {
    if (tile == 256) return token::run_tile<OT, TERMS, TOKEN_GRAD, 1, 256, 256, 2, 2>(p, s);
  }
  if (tile >= 128 && p.N > 64) return token::run_tile<OT, TERMS, TOKEN_GRAD, 1, 128, 128, 2, 2, TERMS == 3 ? 3 : 4>(p, s);
  if (tile == 128) return token::run_tile<OT, TERMS, TOKEN_GRAD, 1, 128, 64, 2, 2, TERMS == 3 ? 4 : 6>(p, s);
  return token::run_narrow<OT, TERMS, TOKEN_GRAD, 1, 2, 2>(p, s);
}

}  // namespace

hipError_t launch_token_grad(const TokenGemm& p, int storage, int tile, int ways, hipStream_t s) {
  if (p.slices < 1 || p.slices > p.K / 32) return hipErrorInvalidValue;  // (a slice without a stage has no first one to load)
  if (ways != 1 && (ways != 2 || storage == 0)) return hipErrorInvalidValue;
  if (ways == 2) return storage == 1 ? grad_of_two<f16>(p, tile, s) : grad_of_two<bf16>(p, tile, s);
  if (storage == 0) return grad<bf16, 3>(p, tile, s);
  return storage == 1 ? grad<f16, 1>(p, tile, s) : grad<bf16, 1>(p, tile, s);
}

}  // namespace ipc
