// ipc_token_tail.hip - the last two products of a small update, which neither wait for each other (the
// gradient takes W's copy) nor fill the CUs, in one launch.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

template <typename OT, int GT, int UT, typename WT>
__global__ void __launch_bounds__(256) token_tail_kernel(const TokenGemm g, const TokenGemm u, unsigned first) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (blockIdx.x < first) token::product_tile<OT, GT, TOKEN_STATE, 1, 64, 64, 2, 2, GT == 3 ? 6 : 8, WT>(g, smem, blockIdx.x, first);
  else token::product_tile<OT, UT, TOKEN_WEIGHT, 1, 64, 64, 2, 2, UT == 3 ? 6 : 4, WT>(u, smem, blockIdx.x - first, gridDim.x - first);
}

template <typename OT, int GT, int UT, typename WT>
hipError_t run(const TokenGemm& g, const TokenGemm& u, hipStream_t s) {
  constexpr int a = token::tile_lds<GT, TOKEN_STATE, 1, 64, 64, 2, 2, GT == 3 ? 6 : 8>(), b = token::tile_lds<UT, TOKEN_WEIGHT, 1, 64, 64, 2, 2, UT == 3 ? 6 : 4>();
  constexpr int smem = a > b ? a : b;
  const void* fn = reinterpret_cast<const void*>(&token_tail_kernel<OT, GT, UT, WT>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  TokenGemm p = g, q = u;
  unsigned first = (unsigned)(((p.M + 63LL) / 64) * ((p.N + 63LL) / 64));
  void* args[] = {&p, &q, &first};
  return hipLaunchKernel(fn, dim3(first + (unsigned)(((q.M + 63LL) / 64) * ((q.N + 63LL) / 64))), dim3(256), args, smem, s);
}

}  // namespace

hipError_t launch_token_tail(const TokenGemm& g, const TokenGemm& u, int storage, hipStream_t s) {
  if (storage == 0) return run<bf16, 3, 3, float>(g, u, s);
  return storage == 1 ? run<f16, 1, 2, f16>(g, u, s) : run<bf16, 1, 3, bf16>(g, u, s);
}

}  // namespace ipc
