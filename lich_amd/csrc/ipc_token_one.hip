// ipc_token_one.hip - logits, losses and errors of a vocabulary that one tile holds, in one launch.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

// (all terms of f(X) in one wave, as for the logits of a longer vocabulary)
template <typename OT, int TERMS, int WAYS>
hipError_t run(const TokenGemm& p, hipStream_t s) {
  constexpr int BN = WAYS == 3 ? 96 : 64, N = WAYS == 1 ? 2 : 1;
  if (p.M > 64) return token::run_tile<OT, TERMS, TOKEN_ONE, WAYS, 128, BN, WAYS == 2 ? 4 : 2, N, TERMS == 3 ? 4 : WAYS == 3 ? 5 : 6>(p, s);
  return token::run_tile<OT, TERMS, TOKEN_ONE, WAYS, 64, BN, 2, N, TERMS == 3 ? 6 : 8>(p, s);
}

}  // namespace

hipError_t launch_token_one(const TokenGemm& p, int storage, int ways, hipStream_t s) {
  if (ways != (storage == 0 ? 1 : storage == 1 ? 2 : 3)) return hipErrorInvalidValue;
  if (storage == 0) return run<bf16, 3, 1>(p, s);
  return storage == 1 ? run<f16, 1, 2>(p, s) : run<bf16, 1, 3>(p, s);
}

}  // namespace ipc
