// ipc_mx_predict.hip - OUT = W4 f(X): 4-bit weights, few samples (gfx950).
//
// Bound by the bytes of W4 (0.53 a weight) and, below a few MB of them, by one
// memory latency, so the waves of a workgroup share 16 rows of W and split the
// contraction by groups of 128, each streaming its part of W straight into
// registers: lane (r = lane % 16, g = lane / 16) holds block g of row r, 16 bytes
// and one scale byte, which the scaled conversions widen exactly to bf16.
//
// f(X) is evaluated once per workgroup and element and carried as a sum of bf16
// terms, 3 for fp32 states and 2 for 16-bit ones (errors of 2^-25 and 2^-17), each
// a matrix product of its own (v_mfma_f32_16x16x32_bf16): with W exact, the
// result is that of an fp32 product.  The matrix units stay idle most of the
// time, so the extra terms cost nothing that is waited for.
//
// The k order within a group is free as long as both operands agree: product j
// of a group takes values 8 j .. 8 j + 7 of every lane's own block.
#include <algorithm>

#include "ipc_launch.h"
#include "ipc_mx_device.h"

namespace ipc {
namespace {

constexpr int MAX_WAVES = 16;
constexpr int XLD = MX_GROUP + 8;  // bf16 values per sample row of a staged group

// NT: 16-sample tiles; NP: samples a staging pass covers, a power of two >= the
// samples of the block (16 NT from 16 on), so that consecutive lanes take
// consecutive samples of a k-row.
template <typename ST, int NT, int NP>
__global__ void __launch_bounds__(MAX_WAVES * 64) mx_predict_kernel(const MxPredict p) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = p.M, K = p.K, B = p.B, G = mx_groups(K);
  const int m0 = blockIdx.x * 16, b0 = blockIdx.y * 16 * NT, nb = B - b0 < 16 * NT ? B - b0 : 16 * NT;
  const int r = lane & 15, g = lane >> 4;
  const int m = m0 + r < M ? m0 + r : M - 1;  // rows past the end: never stored
  bf16* xs = reinterpret_cast<bf16*>(smem) + (size_t)wave * TERMS * NP * XLD;  // [term][sample][k], the wave's own
  const uint8_t* wr = p.w + (long long)m * G * 64 + g * 16;
  const ST* x = reinterpret_cast<const ST*>(p.x) + b0;

  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // a group's codes, scales and states; the next group's loads go out before this one's products
  constexpr int XI = 2 * NP;  // staged values per lane
  constexpr int KPI = 64 / NP;  // k-rows per staging step
  const int sn = lane % NP, sk = lane / NP;
  mx::u32x4 wn;
  unsigned sn_;
  float xn[XI];
  auto fetch = [&](int kg) {
    wn = *reinterpret_cast<const mx::u32x4*>(wr + (long long)kg * 64);
    sn_ = p.ws[(long long)kg * M + m];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int k = kg * MX_GROUP + i * KPI + sk;
      xn[i] = k < K && sn < nb ? to_f32(x[(long long)k * B + sn]) : 0.0f;
    }
  };
  if (wave < G) fetch(wave);
  for (int kg = wave; kg < G; kg += waves) {
    const mx::u32x4 w = wn;
    const unsigned sb = (sn_ >> (8 * g)) & 255u;
    float f[XI];
#pragma unroll
    for (int i = 0; i < XI; ++i) f[i] = xn[i];
    const int kbase = kg * MX_GROUP;
    if (kg + waves < G) fetch(kg + waves);
    activate<XI>(p.act, f);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's LDS accesses complete in order)
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      float v = kbase + i * KPI + sk < K ? f[i] : 0.0f;  // past the contraction: zero, whatever f(0) is
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        const bf16 h = cvt<bf16>(v);
        xs[(t * NP + sn) * XLD + i * KPI + sk] = h;
        v = __builtin_isfinite(to_f32(h)) ? v - to_f32(h) : 0.0f;  // (an infinity has no rest)
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const float scale = __builtin_bit_cast(float, (sb == 255u ? 0x7fc00000u : sb << 23));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      bf16x8 a;
      const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 0);
      const bf16x2 a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 1);
      const bf16x2 a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 2);
      const bf16x2 a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 3);
      a[0] = a0[0]; a[1] = a0[1]; a[2] = a1[0]; a[3] = a1[1];
      a[4] = a2[0]; a[5] = a2[1]; a[6] = a3[0]; a[7] = a3[1];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < TERMS; ++u) {
          const int n = t * 16 + r < NP ? t * 16 + r : NP - 1;  // (columns past the samples: never stored)
          const bf16x8 b = *reinterpret_cast<const bf16x8*>(&xs[(u * NP + n) * XLD + g * 32 + j * 8]);
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc[t], 0, 0, 0);
        }
    }
  }
  // partial tiles [wave][16 rows][16 NT + 1 columns], over the staged states
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  constexpr int LD = 16 * NT + 1;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) part[(wave * 16 + 4 * g + q) * LD + t * 16 + r] = acc[t][q];
  __syncthreads();
  ST* out = reinterpret_cast<ST*>(p.out);
  for (int i = tid; i < 16 * nb; i += blockDim.x) {
    const int row = i / nb, n = i % nb;
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += part[(w * 16 + row) * LD + n];
    if (m0 + row < M) out[(long long)(m0 + row) * B + b0 + n] = cvt<ST>(s);
  }
}

template <typename ST, int NT, int NP>
hipError_t run(const MxPredict& p, hipStream_t s) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2;
  constexpr int WAVE_BYTES = std::max(TERMS * NP * XLD * 2, 16 * (16 * NT + 1) * 4);
  constexpr int MOST = std::min(MAX_WAVES, 160 * 1024 / WAVE_BYTES);
  const void* fn = reinterpret_cast<const void*>(&mx_predict_kernel<ST, NT, NP>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, MOST * WAVE_BYTES);
  if (e != hipSuccess) return e;
  const int waves = std::min(mx_groups(p.K), MOST);
  MxPredict q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((p.M + 15) / 16, (p.B + 16 * NT - 1) / (16 * NT)), dim3(waves * 64), args,
                         (size_t)waves * WAVE_BYTES, s);
}

template <typename ST>
hipError_t run_samples(const MxPredict& p, hipStream_t s) {
  if (p.B == 1) return run<ST, 1, 1>(p, s);
  if (p.B <= 4) return run<ST, 1, 4>(p, s);
  if (p.B <= 16) return run<ST, 1, 16>(p, s);
  return run<ST, 2, 32>(p, s);
}

}  // namespace

hipError_t launch_mx_predict(const MxPredict& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return run_samples<float>(p, s);
  if (storage == DT_F16) return run_samples<f16>(p, s);
  return run_samples<bf16>(p, s);
}

}  // namespace ipc
