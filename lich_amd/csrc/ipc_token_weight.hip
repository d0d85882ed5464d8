// ipc_token_weight.hip - W += alpha e f(X)^T for a piece of the vocabulary.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, bool SPLIT>
hipError_t weight(const TokenGemm& p, hipStream_t s) {
  auto tiles = [&](long long e) { return ((p.M + e - 1) / e) * ((p.N + e - 1) / e); };
  if (tiles(256) >= 160) return token::run_tile<OT, SPLIT, TOKEN_WEIGHT, false, 256, 256, 2, 4>(p, s);
  if (tiles(128) > 128) return token::run_tile<OT, SPLIT, TOKEN_WEIGHT, false, 128, 128, 2, 2>(p, s);
  return token::run_tile<OT, SPLIT, TOKEN_WEIGHT, false, 64, 64, 2, 2>(p, s);
}

}  // namespace

hipError_t launch_token_weight(const TokenGemm& p, int storage, hipStream_t s) {
  if (storage == 0) return weight<bf16, true>(p, s);
  return storage == 1 ? weight<f16, false>(p, s) : weight<bf16, false>(p, s);
}

}  // namespace ipc
