// ipc_ckpt_gemm.hip - the backward pass of a state kept in 8 bits as 16-bit products.
#include "ipc_ckpt_gemm.h"

namespace ipc {
namespace {

template <typename OT>
hipError_t run(int mode, const CkptProblem& p, int act, hipStream_t s) {
  if (mode == CKPT_WEIGHT) return mx::run_ckpt<OT, CKPT_WEIGHT, ACT_IDENTITY>(p, s);
  switch (act) {
    case ACT_RELU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_RELU>(p, s);
    case ACT_TANH: return mx::run_ckpt<OT, CKPT_GRAD, ACT_TANH>(p, s);
    case ACT_SIGMOID: return mx::run_ckpt<OT, CKPT_GRAD, ACT_SIGMOID>(p, s);
    case ACT_SILU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_SILU>(p, s);
    case ACT_GELU: return mx::run_ckpt<OT, CKPT_GRAD, ACT_GELU>(p, s);
    default: return mx::run_ckpt<OT, CKPT_GRAD, ACT_IDENTITY>(p, s);
  }
}

__global__ void __launch_bounds__(256) ckpt_pad_kernel(const mx::PadJob a, const mx::PadJob b, unsigned blocks_a) {
  typedef mx::Run<bf16, 8> Run8;
  const mx::PadJob& j = blockIdx.x < blocks_a ? a : b;
  const unsigned first = (blockIdx.x < blocks_a ? blockIdx.x : blockIdx.x - blocks_a) * mx::PAD_CHUNKS + threadIdx.x;
  const unsigned per = (unsigned)j.ld / 8, n = (unsigned)j.n;
  uint4 v[4];
  unsigned at[4];  // chunk of dst
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    at[u] = first + u * 256;
    const unsigned r = at[u] / per, c = (at[u] - r * per) * 8;
    v[u] = make_uint4(0, 0, 0, 0);
    if (r >= (unsigned)j.rows) {
      at[u] = ~0u;
      continue;
    }
    const unsigned short* p = j.src + (long long)r * n + c;
    if (c + 8 <= n) {
      v[u] = __builtin_bit_cast(uint4, reinterpret_cast<const Run8::U*>(p)->v);
    } else {
      unsigned short h[8] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < n) h[i] = p[i];
      v[u] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (at[u] != ~0u) *reinterpret_cast<uint4*>(j.dst + (long long)at[u] * 8) = v[u];
}

}  // namespace

hipError_t launch_ckpt_pad(const void* a, void* pa, int rows_a, int na, int lda, const void* b, void* pb, int rows_b,
                           int nb, int ldb, hipStream_t s) {
  auto job = [](const void* src, void* dst, int rows, int n, int ld) {
    return mx::PadJob{static_cast<const unsigned short*>(src), static_cast<unsigned short*>(dst), rows, n, ld};
  };
  const mx::PadJob ja = job(a, pa, a ? rows_a : 0, na, lda), jb = job(b, pb, b ? rows_b : 0, nb, ldb);
  const long long ba = mx::pad_blocks(ja), blocks = ba + mx::pad_blocks(jb);
  hipLaunchKernelGGL(ckpt_pad_kernel, dim3((unsigned)blocks), dim3(256), 0, s, ja, jb, (unsigned)ba);
  return hipGetLastError();
}

hipError_t launch_ckpt_gemm(int mode, const CkptProblem& p, int operand, int act, hipStream_t s) {
  return operand == DT_F16 ? run<f16>(mode, p, act, s) : run<bf16>(mode, p, act, s);
}

}  // namespace ipc
