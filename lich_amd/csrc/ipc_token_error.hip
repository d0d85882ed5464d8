// ipc_token_error.hip - errors of a piece of the vocabulary.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <int MODE, typename OT, bool SPLIT>
hipError_t run(const TokenGemm& p, int bm, hipStream_t s) {
  if (bm == 256) return token::run_tile<OT, SPLIT, MODE, 256, 256, 2, 2>(p, s);
  if (bm == 128 && p.N > 64) return token::run_tile<OT, SPLIT, MODE, 128, 128, 2, 2>(p, s);
  if (bm == 128) return token::run_tile<OT, SPLIT, MODE, 128, 64, 2, 2>(p, s);
  return token::run_tile<OT, SPLIT, MODE, 64, 64, 2, 2>(p, s);
}

template <int MODE>
hipError_t by_type(const TokenGemm& p, int storage, int bm, hipStream_t s) {
  if (storage == 0) return run<MODE, bf16, true>(p, bm, s);
  return storage == 1 ? run<MODE, f16, false>(p, bm, s) : run<MODE, bf16, false>(p, bm, s);
}

}  // namespace

hipError_t launch_token_error(const TokenGemm& p, int storage, int bm, hipStream_t s) {
  return by_type<TOKEN_ERROR>(p, storage, bm, s);
}

}  // namespace ipc
