// ipc_token_small.hip - softmax cross entropy of a small output layer in one workgroup.
//
// The image nets' output (10 classes, 64 features, 128 samples) is 250 thousand
// multiplications: the launches of the general path, five of 4 us each, are all of its time.  Here
// W, f(X) and the errors stay in LDS in fp32 and one workgroup takes every step, in 11.3 us (fp32),
// bound by the latency of each step's LDS reads and of the first loads:
//
//   z[v][b] = sum_d W[v][d] f[d][b]        4 words of a column a thread
//   loss, e = onehot - softmax(z)          a column by `lanes` neighbouring lanes
//   G[d][b] = f'(x) sum_v W[v][d] e[v][b]  4 features of a column a thread
//   W[v][d] += alpha sum_b e[v][b] f[d][b] a thread each, 4 samples a read
//
// Sums run in order; nothing is rounded below fp32 but the results.  Rows of f and e hold
// B + 4 floats (up to a multiple of 4), so that 16-byte reads down a column of rows spread
// over the banks.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

constexpr int kThreads = 1024;
constexpr int kLds = 150 * 1024;
constexpr int kItems = 2;

inline __host__ __device__ int small_row(int n) { return (n + 3) / 4 * 4 + 4; }
inline long long small_lds(int V, int D, int B) { return 4LL * ((long long)D * small_row(B) + (long long)(V + 3) / 4 * 4 * small_row(D) + (long long)V * small_row(B)); }

template <typename ST, int ACT>
__global__ void __launch_bounds__(kThreads) token_small_kernel(const TokenProblem p, int lanes) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int V = p.V, D = p.D, B = p.B, RB = small_row(B), RD = small_row(D), V4 = (V + 3) / 4 * 4, tid = threadIdx.x;
  float* f = reinterpret_cast<float*>(smem);  // [D][RB]
  float* w = f + D * RB;                      // [V4][RD]
  float* e = w + V4 * RD;                     // [V][RB]
  const ST* x = static_cast<const ST*>(p.x);
  ST* W = static_cast<ST*>(p.w);
  // an item of X is 4 features of a sample, kItems of them (and W's first values) are in flight at a time;
  // (every path once: the code comes from memory too, and its length is felt)
  const int items = (D + 3) / 4 * B;
  auto item = [&](int i, int& d, int& b) {
    const int q = i / B;
    d = q * 4;
    b = i - q * B;
  };
  auto x_at = [&](int i, float (&o)[4], bool& real) {
    int d, b;
    item(i, d, b);
    const long long id = p.targets[b];
    real = id >= 0 && id < V;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = to_f32(x[(d + q < D ? d + q : d) * B + b]);
  };
  auto w_at = [&](int i) {
    const int v = i / RD, d = i - v * RD;
    return v < V && d < D ? to_f32(W[v * D + d]) : 0.0f;
  };
  const float w0 = tid < V4 * RD ? w_at(tid) : 0.0f;
#pragma unroll 1
  for (int i0 = tid; i0 < items; i0 += kItems * kThreads) {
    float o[kItems][4];
    bool real[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u)
      if (i0 + u * kThreads < items) x_at(i0 + u * kThreads, o[u], real[u]);
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      int d, b;
      item(i0 + u * kThreads, d, b);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (d + q < D) f[(d + q) * RB + b] = real[u] ? act_t<ACT>(o[u][q]) : 0.0f;
    }
  }
  if (tid < V4 * RD) w[tid] = w0;
#pragma unroll 1
  for (int i = tid + kThreads; i < V4 * RD; i += kThreads) w[i] = w_at(i);
  const int pad = RB - B;  // columns of zeros behind f's and e's
#pragma unroll 1
  for (int i = tid; i < D * pad; i += kThreads) f[i / pad * RB + B + i % pad] = 0.0f;
#pragma unroll 1
  for (int i = tid; i < V * pad; i += kThreads) e[i / pad * RB + B + i % pad] = 0.0f;
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < V4 / 4 * B; i += kThreads) {
    const int v = i / B * 4, b = i % B;
    float z[4] = {};
    int d = 0;
#pragma unroll 4
    for (; d + 4 <= D; d += 4) {
      const float g[4] = {f[d * RB + b], f[(d + 1) * RB + b], f[(d + 2) * RB + b], f[(d + 3) * RB + b]};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 u = *reinterpret_cast<const float4*>(w + (v + q) * RD + d);
        z[q] += u.x * g[0]; z[q] += u.y * g[1]; z[q] += u.z * g[2]; z[q] += u.w * g[3];
      }
    }
#pragma unroll 1
    for (; d < D; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) z[q] += w[(v + q) * RD + d] * f[d * RB + b];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (v + q < V) e[(v + q) * RB + b] = z[q];
  }
  __syncthreads();
#pragma unroll 1
  for (int b0 = 0; b0 < B; b0 += kThreads / lanes) {
    const int b = b0 + tid / lanes, l = tid % lanes;
    const long long id = b < B ? p.targets[b] : -1;
    const bool real = id >= 0 && id < V;
    float top = -__builtin_inff(), sum = 0.0f;
    if (real)
#pragma unroll 1
      for (int v = l; v < V; v += lanes) top = __builtin_fmaxf(top, e[v * RB + b]);
    for (int o = 1; o < lanes; o <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    const float from = top == -__builtin_inff() ? 0.0f : top;
    if (real)
#pragma unroll 1
      for (int v = l; v < V; v += lanes) sum += expf(e[v * RB + b] - from);
    for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor(sum, o);
    const float loss = real ? logf(sum) + (top - e[(int)id * RB + b]) : 0.0f;
    if (b < B && l == 0) p.loss[b] = loss;
    if (!p.g || b >= B) continue;
    const float share = 1.0f / sum;
    // (the target's own lane reads its logit above before it is changed here: the lanes of a
    // column run together)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
    for (int v = l; v < V; v += lanes)
      e[v * RB + b] = !real ? 0.0f : v == id ? -expm1f(-loss) : -expf(e[v * RB + b] - from) * share;
  }
  if (!p.g) return;
  __syncthreads();
  ST* G = static_cast<ST*>(p.g);
#pragma unroll 1
  for (int i = tid; i < items; i += kThreads) {
    float o[4], g[4] = {};
    bool real;
    int d, b;
    x_at(i, o, real);
    item(i, d, b);
#pragma unroll 2
    for (int v = 0; v < V; ++v) {
      const float4 u = *reinterpret_cast<const float4*>(w + v * RD + d);
      const float s = e[v * RB + b];
      g[0] += u.x * s; g[1] += u.y * s; g[2] += u.z * s; g[3] += u.w * s;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (d + q < D) G[(d + q) * B + b] = cvt<ST>(real ? dact_t<ACT>(o[q]) * g[q] : 0.0f);
  }
#pragma unroll 1
  for (int i = tid; i < V * D; i += kThreads) {
    const int v = i / D, d = i - v * D;
    const float4 *a = reinterpret_cast<const float4*>(e + v * RB), *c = reinterpret_cast<const float4*>(f + d * RB);
    float sum = 0.0f;
#pragma unroll 4
    for (int b = 0; b < (B + 3) / 4; ++b) {
      const float4 s = a[b], t = c[b];
      sum += s.x * t.x; sum += s.y * t.y; sum += s.z * t.z; sum += s.w * t.w;
    }
    W[i] = cvt<ST>(w[v * RD + d] + p.alpha * sum);
  }
}

}  // namespace

// One workgroup is slow at anything long: the steps that its threads take one after the other are
// counted.  us, in one / in the launches of the general path, fp32: 10 x 64 x 128 (V, D, B; 82
// steps) 11.3 / 21.6; 64 x 64 x 64 (152) 18 / 23.6; 10 x 256 x 100 (225) 30.6 / 26; 1844 x 4 x 1 (1877) 76 / 22.
bool token_small(int V, int D, int B) {
  constexpr long long most = 1 << 14;
  if ((long long)V * D > most || (long long)D * B > most || (long long)V * B > most || small_lds(V, D, B) > kLds) return false;
  auto rounds = [](long long items) { return (items + kThreads - 1) / kThreads; };
  const long long logits = rounds((V + 3LL) / 4 * B) * ((D + 3) / 4), gradient = rounds((D + 3LL) / 4 * B) * V,
                  update = rounds((long long)V * D) * ((B + 3) / 4), fill = rounds((long long)V * (D + 4)) + 2 * rounds((D + 3LL) / 4 * B);
  return logits + gradient + update + fill <= 192;
}

template <typename ST, int ACT>
hipError_t run_small(const TokenProblem& p, hipStream_t s) {
  const void* fn = reinterpret_cast<const void*>(&token_small_kernel<ST, ACT>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e != hipSuccess) return e;
  int lanes = 1;
  while (lanes < 64 && lanes * 2 * p.B <= kThreads && lanes * 4 <= p.V) lanes *= 2;
  TokenProblem q = p;
  void* args[] = {&q, &lanes};
  return hipLaunchKernel(fn, dim3(1), dim3(kThreads), args, (size_t)small_lds(p.V, p.D, p.B), s);
}

template <typename ST>
hipError_t small_by_act(const TokenProblem& p, hipStream_t s) {
  switch (p.act) {
    case ACT_RELU: return run_small<ST, ACT_RELU>(p, s);
    case ACT_TANH: return run_small<ST, ACT_TANH>(p, s);
    case ACT_SIGMOID: return run_small<ST, ACT_SIGMOID>(p, s);
    case ACT_SILU: return run_small<ST, ACT_SILU>(p, s);
    case ACT_GELU: return run_small<ST, ACT_GELU>(p, s);
    default: return run_small<ST, ACT_IDENTITY>(p, s);
  }
}

hipError_t launch_token_small(const TokenProblem& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return small_by_act<float>(p, s);
  return storage == DT_F16 ? small_by_act<f16>(p, s) : small_by_act<bf16>(p, s);
}

}  // namespace ipc
