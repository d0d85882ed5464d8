// ipc_token_weight.hip - W += alpha e f(X)^T for a piece of the vocabulary, and the last step
// of the state's gradient.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

inline unsigned finish_blocks(const TokenFinish& f) { return (unsigned)((long long)token_fix_rows(f.D, f.vec) * ((f.B + 63) / 64)); }

// A band of rows of 64 columns: 256 threads, each W consecutive columns of a row (W: 4 where
// rows allow it, else 1).  The slices are added in order.
template <typename ST, int W>
__device__ __forceinline__ void finish_band(const TokenFinish& p, float* red, int block) {
  constexpr int LANES = 64 / W, ROWS = 256 / LANES;
  const int tiles_n = (p.B + 63) / 64, band = block / tiles_n, c = threadIdx.x % LANES * W, r = threadIdx.x / LANES;
  const int n = block % tiles_n * 64 + c, d = band * ROWS + r;
  const long long count = (long long)p.D * p.B, at = (long long)d * p.B + n;
  float fix[W] = {};
  if (n < p.B && d < p.D) {
    float x[W], sum[W] = {};
    ST o[W];
    if constexpr (W == 4) load4(static_cast<const ST*>(p.x) + at, x);
    else x[0] = to_f32(static_cast<const ST*>(p.x)[at]);
#pragma unroll 8
    for (int s = 0; s < p.slices; ++s) {
      float v[W];
      if constexpr (W == 4) load4(p.part + s * count + at, v);
      else v[0] = p.part[s * count + at];
#pragma unroll
      for (int i = 0; i < W; ++i) sum[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const long long id = p.targets[n + i];
      const bool real = id >= 0 && id < p.V;
      sum[i] *= p.scale;
      o[i] = cvt<ST>(real ? act_df(p.act, x[i]) * sum[i] : 0.0f);
      if (p.fixes && real) {
        const float f = act_f(p.act, x[i]);
        fix[i] = sum[i] * (f - to_f32(cvt<ST>(f)));
      }
    }
    typedef ST V __attribute__((ext_vector_type(W)));
    V v;
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = o[i];
    *reinterpret_cast<V*>(static_cast<ST*>(p.g) + at) = v;
  }
  if (!p.fixes) return;
#pragma unroll
  for (int i = 0; i < W; ++i) red[r * 64 + c + i] = fix[i];
  __syncthreads();
  if (threadIdx.x >= 64 || block % tiles_n * 64 + (int)threadIdx.x >= p.B) return;
  float all = red[threadIdx.x];
#pragma unroll
  for (int i = 1; i < ROWS; ++i) all += red[i * 64 + threadIdx.x];
  p.fixes[(long long)band * p.B + block % tiles_n * 64 + threadIdx.x] = all;
}
template <typename ST>
__device__ __forceinline__ void finish(const TokenFinish& p, float* red, int block) {
  if (p.vec) finish_band<ST, 4>(p, red, block);
  else finish_band<ST, 1>(p, red, block);
}

template <typename ST>
__global__ void __launch_bounds__(256) token_finish_kernel(const TokenFinish p) {
  __shared__ float red[16 * 64];
  finish<ST>(p, red, blockIdx.x);
}

// Workgroups 0 .. first - 1: the gradient's last step; the others: W.
template <typename OT, int TERMS, int E, int ST, typename WT>
__global__ void __launch_bounds__(256) token_weight_finish_kernel(const TokenGemm p, const TokenFinish f, unsigned first) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (blockIdx.x < first) {
    finish<WT>(f, reinterpret_cast<float*>(smem), blockIdx.x);
    return;
  }
  token::product_tile<OT, TERMS, TOKEN_WEIGHT, 1, E, E, 2, 2, ST, WT>(p, smem, blockIdx.x - first, gridDim.x - first);
}

// With the gradient's last step, if there is one (its 256 threads are those of a workgroup here).
template <typename OT, int TERMS, int E, int ST, typename WT>
hipError_t weight_finish(const TokenGemm& p, const TokenFinish* f, hipStream_t s) {
  if (!f) return token::run_tile<OT, TERMS, TOKEN_WEIGHT, 1, E, E, 2, 2, ST, WT>(p, s);
  constexpr int smem = token::tile_lds<TERMS, TOKEN_WEIGHT, 1, E, E, 2, 2, ST>();
  const void* fn = reinterpret_cast<const void*>(&token_weight_finish_kernel<OT, TERMS, E, ST, WT>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  TokenGemm q = p;
  TokenFinish g = *f;
  unsigned first = finish_blocks(g);
  void* args[] = {&q, &g, &first};
  return hipLaunchKernel(fn, dim3(first + (unsigned)(((p.M + E - 1LL) / E) * ((p.N + E - 1LL) / E))), dim3(256), args, smem, s);
}

template <typename OT, int TERMS, typename WT>
hipError_t weight(const TokenGemm& p, const TokenFinish* f, int storage, hipStream_t s) {
  auto tiles = [&](long long e) { return ((p.M + e - 1) / e) * ((p.N + e - 1) / e); };
  const bool large = TERMS == 1 && tiles(256) >= 160;
  // (many of the last step's workgroups would wait for LDS that they do not use: us, in one launch / two, fp32
  // 4000 x 4000 x 512 343 / 339, bf16 20000 x 128 x 256 63 / 69)
  if (f && (large || finish_blocks(*f) > 512)) {
    const hipError_t e = launch_token_finish(*f, storage, s);
    if (e != hipSuccess) return e;
    f = nullptr;
  }
  if constexpr (TERMS == 1) {
    if (large) return token::run_tile<OT, TERMS, TOKEN_WEIGHT, 1, 256, 256, 2, 4>(p, s);
  }
  // (narrow tiles where wide ones are mostly padding and a product is a few steps: us, 128 / 64 wide, fp32 10007 x 515 x 77
  // 73 / 70, 50000 x 64 x 16 62 / 54; where they are not, 32000 x 4096 x 4 241 / 265)
  const int wide = (p.N + 127) / 128 * 128, narrow = (p.N + 63) / 64 * 64;
  if (tiles(128) > 128 && !(wide - wide / 16 > narrow && (p.K <= 128 || p.N <= 64))) return weight_finish<OT, TERMS, 128, TERMS == 3 ? 3 : 4, WT>(p, f, s);
  if constexpr (TERMS == 3) {
    if (tiles(64) > 256) return weight_finish<OT, TERMS, 64, 3, WT>(p, f, s);
  }
  return weight_finish<OT, TERMS, 64, TERMS == 3 ? 6 : 8 / TERMS, WT>(p, f, s);
}

}  // namespace

hipError_t launch_token_finish(const TokenFinish& p, int storage, hipStream_t s) {
  const dim3 grid(finish_blocks(p)), block(256);
  if (storage == 0) hipLaunchKernelGGL((token_finish_kernel<float>), grid, block, 0, s, p);
  else if (storage == 1) hipLaunchKernelGGL((token_finish_kernel<f16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((token_finish_kernel<bf16>), grid, block, 0, s, p);
  return hipGetLastError();
}

hipError_t launch_token_weight(const TokenGemm& p, const TokenFinish* f, int storage, int terms, hipStream_t s) {
  if (storage == 0) return weight<bf16, 3, float>(p, f, storage, s);
  if (storage == 1) return terms == 2 ? weight<f16, 2, f16>(p, f, storage, s) : weight<f16, 1, f16>(p, f, storage, s);
  return terms == 3 ? weight<bf16, 3, bf16>(p, f, storage, s) : weight<bf16, 1, bf16>(p, f, storage, s);
}

}  // namespace ipc
