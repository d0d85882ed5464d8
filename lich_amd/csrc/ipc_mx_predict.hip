// ipc_mx_predict.hip - OUT = W4 f(X): 4-bit weights, few samples (gfx950).
//
// Bound by the bytes of W4 (0.53 a weight) and, below a few MB of them, by one
// memory latency, so the waves of a workgroup share 16 rows of W and split the
// contraction by groups of 128, each streaming its part of W straight into
// registers: lane (r = lane % 16, g = lane / 16) holds block g of row r, 16 bytes
// and one scale byte, which the scaled conversions widen exactly to bf16.
//
// f(X) is evaluated once per workgroup and element and carried as a sum of bf16
// terms, each a matrix product of its own (v_mfma_f32_16x16x32_bf16), with W exact:
// 3 terms for fp32 states (errors of 2^-25 of f(X): the result is that of an fp32
// product), 2 for 16-bit ones (2^-17, a 64th of fp16's own rounding and a 512th of
// bf16's).  The matrix units stay idle most of the time, so the extra terms cost
// nothing that is waited for.
//
// The k order within a group is free as long as both operands agree: product j
// of a group takes values 8 j .. 8 j + 7 of every lane's own block.
//
// Two forms.  Without a workspace each workgroup evaluates f of every element it
// needs (all of X, K x 16 samples at a time): nothing for one sample, most of the
// time for many.  With one, f(X) is evaluated once, in a launch of its own, into its
// terms in the order the operand's lanes hold them: [samples / RB][group][term]
// [product j][sample of RB][block g][8 values], RB = 16 samples or all of fewer, so
// that a load of 64 lanes is one run of 1 KB (in [sample][k] order it touched 32
// cache lines: 1000 x 4096, 12 samples, 12.2 us).
#include <algorithm>

#include "ipc_launch.h"
#include "ipc_mx_device.h"

namespace ipc {
namespace {

constexpr int MAX_WAVES = 16;
constexpr int XLD = MX_GROUP + 8;  // bf16 values per sample row of a staged group

// Eight weights of a block, widened.
__device__ __forceinline__ bf16x8 widen8(unsigned w, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2 a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bf16x8{a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]};
}

// Term t of v, which keeps the rest.  The first one is finite, since a finite fp32 value
// may round past the largest bf16; an infinity or NaN is the second, and has no rest.
__device__ __forceinline__ bf16 take_term(int t, float& v) {
  constexpr float MOST = 0x1.fep127f;
  const bf16 h = cvt<bf16>(t == 0 ? __builtin_amdgcn_fmed3f(v, -MOST, MOST) : v);
  v = t == 0 || __builtin_isfinite(to_f32(h)) ? v - to_f32(h) : 0.0f;
  return h;
}

// The form without a workspace: RM tiles of 16 rows and 16 samples per workgroup.
// NP: samples a staging pass covers, 16 or the power of two >= B below it, so that
// consecutive lanes take consecutive samples of a k-row.
template <typename ST, int RM, int NP>
__global__ void __launch_bounds__(MAX_WAVES * 64) mx_predict_kernel(const MxPredict p) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2, LD = 17;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = p.M, K = p.K, B = p.B, G = mx_groups(K);
  const int m0 = blockIdx.x * 16 * RM, b0 = blockIdx.y * 16, nb = B - b0 < 16 ? B - b0 : 16;
  const int r = lane & 15, g = lane >> 4;
  int m[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) m[i] = m0 + i * 16 + r < M ? m0 + i * 16 + r : M - 1;  // rows past the end: never stored
  bf16* xs = reinterpret_cast<bf16*>(smem) + (size_t)wave * TERMS * NP * XLD;  // [term][sample][k], the wave's own
  const ST* x = reinterpret_cast<const ST*>(p.x) + b0;

  f32x4 acc[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // a group's codes, scales and states; the next group's loads go out before this one's products
  constexpr int XI = 2 * NP;    // staged values per lane
  constexpr int KPI = 64 / NP;  // k-rows per staging step
  const int sn = lane % NP, sk = lane / NP;
  mx::u32x4 w[RM];
  unsigned sw[RM];
  ST xn[XI];  // (as loaded: widened here they would be waited for here)
  auto fetch = [&](int kg) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      w[i] = *reinterpret_cast<const mx::u32x4*>(p.w + ((long long)m[i] * G + kg) * 64 + g * 16);
      sw[i] = p.ws[(long long)kg * M + m[i]];
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int k = kg * MX_GROUP + i * KPI + sk;
      xn[i] = (ST)0.0f;
      if (k < K && sn < nb) xn[i] = x[(long long)k * B + sn];
    }
  };
  fetch(wave);
  for (int kg = wave; kg < G; kg += waves) {
    mx::u32x4 cw[RM];
    float scale[RM], f[XI];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      cw[i] = w[i];
      const unsigned sb = (sw[i] >> (8 * g)) & 255u;
      scale[i] = __builtin_bit_cast(float, (sb == 255u ? 0x7fc00000u : sb << 23));
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) f[i] = to_f32(xn[i]);
    if (kg + waves < G) fetch(kg + waves);
    activate<XI>(p.act, f);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's LDS accesses complete in order)
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      float v = kg * MX_GROUP + i * KPI + sk < K ? f[i] : 0.0f;  // past the contraction: zero, whatever f(0) is
#pragma unroll
      for (int t = 0; t < TERMS; ++t) xs[(t * NP + sn) * XLD + i * KPI + sk] = take_term(t, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 b[TERMS];
#pragma unroll
      for (int u = 0; u < TERMS; ++u)  // (columns past the samples: never stored)
        b[u] = *reinterpret_cast<const bf16x8*>(&xs[(u * NP + (r < NP ? r : NP - 1)) * XLD + g * 32 + j * 8]);
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const bf16x8 a = widen8(cw[i][j], scale[i]);
#pragma unroll
        for (int u = 0; u < TERMS; ++u) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[u], acc[i], 0, 0, 0);
      }
    }
  }
  // partial tiles [wave][16 RM rows][17], over the staged states
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) part[((wave * RM + i) * 16 + 4 * g + q) * LD + r] = acc[i][q];
  __syncthreads();
  ST* out = reinterpret_cast<ST*>(p.out);
  for (int i = tid; i < 16 * RM * nb; i += blockDim.x) {
    const int row = i / nb, n = i % nb;
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += part[(w * RM * 16 + row) * LD + n];
    if (m0 + row < M) out[(long long)(m0 + row) * B + b0 + n] = cvt<ST>(s);
  }
}

// f(X) [K][B] into its bf16 terms, zero past K: 8 values of a sample per thread,
// samples fastest (coalesced reads).
template <typename ST>
__global__ void __launch_bounds__(256) mx_terms_kernel(const ST* __restrict__ x, bf16* __restrict__ out, int K, int B,
                                                       int groups, int act) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int n = (int)(i % B), k = (int)(i / B) * 8, kg = k / MX_GROUP, g = k / 32 & 3, j = k / 8 & 3;
  if (kg >= groups) return;
  float v[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = k + q < K ? to_f32(x[(long long)(k + q) * B + n]) : 0.0f;
  activate<8>(act, v);
  const int rb = B < 16 ? B : 16;
  bf16* to = out + (((((long long)(n / rb) * groups + kg) * TERMS * 4 + j) * rb + n % rb) * 4 + g) * 8;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    bf16x8 h;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (k + q >= K) v[q] = 0.0f;  // past the contraction: zero, whatever f(0) is
      h[q] = take_term(t, v[q]);
    }
    *reinterpret_cast<bf16x8*>(to + (long long)t * 4 * rb * 32) = h;
  }
}

// RM tiles of 16 rows and 16 samples per workgroup, its waves splitting the
// contraction; a group's loads are all issued before its first product.
template <typename ST, int RM>
__global__ void __launch_bounds__(MAX_WAVES * 64) mx_predict_terms_kernel(const MxPredict p) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2, LD = 17;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = p.M, B = p.B, G = mx_groups(p.K);
  const int m0 = blockIdx.x * 16 * RM, b0 = blockIdx.y * 16, nb = B - b0 < 16 ? B - b0 : 16;
  const int r = lane & 15, g = lane >> 4, rb = B < 16 ? B : 16;
  int m[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) m[i] = m0 + i * 16 + r < M ? m0 + i * 16 + r : M - 1;  // rows past the end: never stored
  // (nor samples: of a block of fewer than 16 the last one again, of a last partial block what is there)
  const bf16* xr = reinterpret_cast<const bf16*>(p.terms) + (long long)blockIdx.y * G * TERMS * 4 * rb * 32 +
                   ((r < rb ? r : rb - 1) * 4 + g) * 8;
  f32x4 acc[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  mx::u32x4 w[RM];
  unsigned sw[RM];
  auto weights = [&](int kg) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      w[i] = *reinterpret_cast<const mx::u32x4*>(p.w + ((long long)m[i] * G + kg) * 64 + g * 16);
      sw[i] = p.ws[(long long)kg * M + m[i]];
    }
  };
  weights(wave);
  for (int kg = wave; kg < G; kg += waves) {
    bf16x8 b[4][TERMS];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int u = 0; u < TERMS; ++u)
        b[j][u] = *reinterpret_cast<const bf16x8*>(xr + (((long long)kg * TERMS + u) * 4 + j) * rb * 32);
    mx::u32x4 cw[RM];
    float scale[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      cw[i] = w[i];
      const unsigned sb = (sw[i] >> (8 * g)) & 255u;
      scale[i] = __builtin_bit_cast(float, (sb == 255u ? 0x7fc00000u : sb << 23));
    }
    weights(kg + waves < G ? kg + waves : kg);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const bf16x8 a = widen8(cw[i][j], scale[i]);
#pragma unroll
        for (int u = 0; u < TERMS; ++u) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[j][u], acc[i], 0, 0, 0);
      }
  }
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) part[((wave * RM + i) * 16 + 4 * g + q) * LD + r] = acc[i][q];
  __syncthreads();
  ST* out = reinterpret_cast<ST*>(p.out);
  for (int i = tid; i < 16 * RM * 16; i += blockDim.x) {
    const int row = i / 16, n = i % 16;
    if (m0 + row >= M || n >= nb) continue;
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += part[(w * RM * 16 + row) * LD + n];
    out[(long long)(m0 + row) * B + b0 + n] = cvt<ST>(s);
  }
}

template <typename ST, int RM, int NP>
hipError_t run(const MxPredict& p, hipStream_t s) {
  constexpr int TERMS = sizeof(ST) == 4 ? 3 : 2;
  constexpr int WAVE_BYTES = std::max(TERMS * NP * XLD * 2, RM * 16 * 17 * 4);
  constexpr int MOST = std::min(MAX_WAVES, 160 * 1024 / WAVE_BYTES);
  const void* fn = reinterpret_cast<const void*>(&mx_predict_kernel<ST, RM, NP>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, MOST * WAVE_BYTES);
  if (e != hipSuccess) return e;
  const int waves = std::min(mx_groups(p.K), MOST);
  MxPredict q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((p.M + 16 * RM - 1) / (16 * RM), (p.B + 15) / 16), dim3(waves * 64), args,
                         (size_t)waves * WAVE_BYTES, s);
}

template <typename ST, int RM>
hipError_t run_terms(const MxPredict& p, hipStream_t s) {
  constexpr int WAVE_BYTES = RM * 16 * 17 * 4;
  const void* fn = reinterpret_cast<const void*>(&mx_predict_terms_kernel<ST, RM>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, MAX_WAVES * WAVE_BYTES);
  if (e != hipSuccess) return e;
  const int waves = std::min(mx_groups(p.K), MAX_WAVES);
  MxPredict q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((p.M + 16 * RM - 1) / (16 * RM), (p.B + 15) / 16), dim3(waves * 64), args,
                         (size_t)waves * WAVE_BYTES, s);
}

template <typename ST>
hipError_t run_samples(const MxPredict& p, hipStream_t s) {
  if (p.terms) {
    const int G = mx_groups(p.K);
    const long long items = (long long)G * (MX_GROUP / 8) * p.B;
    hipLaunchKernelGGL(mx_terms_kernel<ST>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s,
                       static_cast<const ST*>(p.x), static_cast<bf16*>(p.terms), p.K, p.B, G, p.act);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const long long tiles = ((p.M + 15LL) / 16) * ((p.B + 15LL) / 16);
    return tiles >= 1024 ? run_terms<ST, 4>(p, s) : tiles >= 512 ? run_terms<ST, 2>(p, s) : run_terms<ST, 1>(p, s);
  }
  if (p.B == 1) return p.M >= 8192 ? run<ST, 2, 1>(p, s) : run<ST, 1, 1>(p, s);
  if (p.B <= 4) return p.M >= 8192 ? run<ST, 2, 4>(p, s) : run<ST, 1, 4>(p, s);
  return run<ST, 1, 16>(p, s);
}

}  // namespace

hipError_t launch_mx_predict(const MxPredict& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return run_samples<float>(p, s);
  if (storage == DT_F16) return run_samples<f16>(p, s);
  return run_samples<bf16>(p, s);
}

}  // namespace ipc
