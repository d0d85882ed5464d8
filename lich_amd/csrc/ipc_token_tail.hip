// ipc_token_tail.hip - the last two products of a small update, which neither wait for each other (the
// gradient takes W's copy) nor fill the CUs, in one launch.  W's product of a long batch, few tiles
// of many steps, is cut into slices, added in order by a launch of their own.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

// The gradient's tile: 64 columns, in 16 bits (GT = 1) with two terms of the errors side by side.
template <int GT> constexpr int kWays = GT == 1 ? 2 : 1;
template <int GT> constexpr int kWide = 64 * kWays<GT>;
template <int GT> constexpr int kStages = GT == 3 ? 6 : 8;

// CUT: W's product as slices (of the form of TOKEN_GRAD: both read A by rows of the contraction)
template <typename OT, int GT, int UT, bool CUT, typename WT>
__global__ void __launch_bounds__(256) token_tail_kernel(const TokenGemm g, const TokenGemm u, unsigned first) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int UM = CUT ? TOKEN_GRAD : TOKEN_WEIGHT;
  if (blockIdx.x < first) token::product_tile<OT, GT, TOKEN_STATE, kWays<GT>, 64, kWide<GT>, 2, 2, kStages<GT>, WT>(g, smem, blockIdx.x, first);
  else token::product_tile<OT, UT, UM, 1, 64, 64, 2, 2, UT == 3 ? 6 : 4, WT>(u, smem, blockIdx.x - first, gridDim.x - first);
}

template <typename OT, int GT, int UT, bool CUT, typename WT>
hipError_t products(const TokenGemm& g, const TokenGemm& u, hipStream_t s) {
  constexpr int a = token::tile_lds<GT, TOKEN_STATE, kWays<GT>, 64, kWide<GT>, 2, 2, kStages<GT>>(), b = token::tile_lds<UT, TOKEN_WEIGHT, 1, 64, 64, 2, 2, UT == 3 ? 6 : 4>();
  constexpr int smem = a > b ? a : b;
  const void* fn = reinterpret_cast<const void*>(&token_tail_kernel<OT, GT, UT, CUT, WT>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  TokenGemm p = g, q = u;
  unsigned first = (unsigned)(((p.M + 63LL) / 64) * ((p.N + 63LL) / 64));
  void* args[] = {&p, &q, &first};
  return hipLaunchKernel(fn, dim3(first + (unsigned)(((q.M + 63LL) / 64) * ((q.N + 63LL) / 64) * q.slices)), dim3(256), args, smem, s);
}

template <typename WT>
__global__ void __launch_bounds__(256) token_add_kernel(WT* w, const float* part, long long count, int slices, float alpha) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  const float old = to_f32(w[at]);
  float sum = 0.0f;
#pragma unroll 8
  for (int s = 0; s < slices; ++s) sum += part[s * count + at];
  w[at] = cvt<WT>(old + alpha * sum);
}

template <typename OT, int GT, int UT, typename WT>
hipError_t run(const TokenGemm& g, const TokenGemm& u, float* part, hipStream_t s) {
  if (u.slices == 1) return products<OT, GT, UT, false, WT>(g, u, s);
  TokenGemm q = u;
  q.out = part; q.add = 0;
  const hipError_t e = products<OT, GT, UT, true, WT>(g, q, s);
  if (e != hipSuccess) return e;
  const long long count = (long long)u.M * u.N;
  hipLaunchKernelGGL((token_add_kernel<WT>), dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, static_cast<WT*>(u.out), part, count,
                     u.slices, u.scal);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_token_tail(const TokenGemm& g, const TokenGemm& u, float* part, int storage, hipStream_t s) {
  if (storage == 0) return run<bf16, 3, 3, float>(g, u, part, s);
  return storage == 1 ? run<f16, 1, 2, f16>(g, u, part, s) : run<bf16, 1, 3, bf16>(g, u, part, s);
}

}  // namespace ipc
