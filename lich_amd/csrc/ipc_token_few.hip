// ipc_token_few.hip - softmax cross entropy of a few samples (up to 8, in 16 bits 4): W is read as it lies and
// passed through the vector units, every product and sum in fp32.
//
//   z[v][b] = sum_d W[v][d] f[b][d], loss, e = onehot - softmax(z)
//   G[d][b] = f'(x) sum_v W[v][d] e[v][b],  W[v][d] += alpha sum_b e[v][b] f[b][d]
//
// A matrix product of few columns is bound by W's bytes, so what counts is how often they pass and
// how many launches stand beside them: once for the loss (logits and each workgroup's
// largest and sum, then these joined), twice read and once written for the update, whose
// second pass takes the gradient's share of a row of W before it writes the new row.
// 32000 x 4096 bf16, one sample: logits 41.7 us (6.3 TB/s), the loss 55 in all with W cold; update
// 134, where three passes of W take 154 at a copy's rate (part of W is still in the cache).
#include <algorithm>

#include "ipc_token_gemm.h"

namespace ipc {
namespace {

constexpr int kMost = 8;                     // samples
constexpr int kLds = 144 * 1024;             // of f(X)
constexpr long long kLogits = 1LL << 30;     // bytes of the update's logits
constexpr int kWaves = 16;                   // logits: waves of a workgroup, one a CU
template <int TB> constexpr int kRows = TB == 1 ? 8 : TB == kMost ? 2 : 4;  // and rows of a wave at a time
constexpr int kStep = 128, kWaves2 = 4, kRows2 = 4;  // second pass: rows whose errors are held, waves, rows of a wave at a time

inline int few_samples(int B) { return B <= 1 ? 1 : B <= 2 ? 2 : B <= 4 ? 4 : kMost; }

struct Few {
  int V, D, Dp, B, act, parts, slices, rows;  // Dp: f's rows in LDS; rows: of a slice
  const void* x;
  void* w;
  const long long* targets;
  float* loss;
  void* g;
  float alpha;
  float2* part;   // [parts][B] largest logit and sum of exponentials
  float* logit;   // [B] of the target
  float* z;       // [V][TB], or nullptr: the loss alone
  float* grad;    // [slices][D][B]
};

// 16 bytes of a row, which starts on a value's own alignment.  Of a row's values past the last whole
// piece a lane has the row's last 16 bytes, and leaves alone what others have of them.
template <typename ST> constexpr int PER = 16 / sizeof(ST);
template <typename ST> struct __attribute__((packed, aligned(sizeof(ST)))) Sixteen { ST v[PER<ST>]; };
template <typename ST>
__device__ __forceinline__ Sixteen<ST> get(const ST* from) { return *reinterpret_cast<const Sixteen<ST>*>(from); }

__device__ __forceinline__ bool is_real(const Few& p, int b) {
  const long long id = b < p.B ? p.targets[b] : -1;
  return id >= 0 && id < p.V;
}

__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float top = __builtin_fmaxf(a.x, b.x), none = -__builtin_inff();
  return make_float2(top, (a.x == none ? a.y : a.y * expf(a.x - top)) + (b.x == none ? b.y : b.y * expf(b.x - top)));
}

// ------------------------------------------------------------------ logits
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, i, CTRL, 0xf, 0xf, true));
}
// N sums over the lanes, N = 8 or 16: lane l has that of index l / (64 / N).  Each exchange, between lanes
// 32, 16, 8 (and 4) apart, halves the sums that a lane keeps; the rest sums one.  All but the
// first two stay within 16 lanes: rotated by 8, mirrored in eights, and fours permuted.
template <int N>
__device__ __forceinline__ float sum_lanes(float (&v)[N], int lane) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + N / 2]), false, false);
    v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + N / 4]), false, false);
    v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int i = 0; i < N / 8; ++i) v[i] = (lane & 8 ? v[i + N / 8] : v[i]) + moved<0x128>(lane & 8 ? v[i] : v[i + N / 8]);
  if constexpr (N == 16) v[0] = (lane & 4 ? v[1] : v[0]) + moved<0x141>(lane & 4 ? v[0] : v[1]);
  else v[0] += moved<0x141>(v[0]);
  v[0] += moved<0x4e>(v[0]);
  return v[0] + moved<0xb1>(v[0]);
}

template <typename ST, int TB>
__global__ void __launch_bounds__(kWaves * 64) token_few_logits_kernel(const Few p) {
  constexpr int P = PER<ST>, R = kRows<TB>, N = R * TB;  // N: sums of a wave
  extern __shared__ __align__(16) float f[];  // [TB][Dp]
  __shared__ float2 red[kWaves][TB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int whole = p.D / P * P;
  {
    const int b = tid % TB;
    const bool real = is_real(p, b);
    const ST* x = static_cast<const ST*>(p.x);
#pragma unroll 1
    for (int i = tid; i < TB * p.Dp; i += kWaves * 64) {  // (its last P values: the row's last, zeros for those of whole pieces)
      const int j = i / TB, d = j < whole ? j : p.D - P + (j - whole);
      f[b * p.Dp + j] = real && (j < whole || d >= whole) ? act_f(p.act, to_f32(x[(long long)d * p.B + b])) : 0.0f;
    }
  }
  __syncthreads();
  // after the sums' exchange a lane has that of row `row` and sample `b`
  constexpr int BITS = N == 8 ? 3 : 4;
  const int own = lane >> (6 - BITS), row = own / TB, b = own % TB;
  const bool first = (lane & ((64 >> BITS) - 1)) == 0;
  const long long id = b < p.B ? p.targets[b] : -1;
  float2 all = make_float2(-__builtin_inff(), 0.0f);
  const ST* w = static_cast<const ST*>(p.w);
  const int stride = gridDim.x * kWaves * R;
  for (long long r0 = (blockIdx.x * kWaves + wave) * R; r0 < p.V; r0 += stride) {
    const ST* rows[R];
#pragma unroll
    for (int i = 0; i < R; ++i) rows[i] = w + (r0 + i < p.V ? r0 + i : p.V - 1LL) * p.D;
    float v[N] = {};
#pragma unroll 1
    for (int d = lane * P; d < p.D; d += 64 * P) {
      Sixteen<ST> in[R];
#pragma unroll
      for (int i = 0; i < R; ++i) in[i] = get(rows[i] + (d < whole ? d : p.D - P));
      if (d >= whole) {  // (what whole pieces have is no number here: 0 times infinity)
#pragma unroll
        for (int q = 0; q < P - 1; ++q)
          if (q < P - (p.D - whole)) {
#pragma unroll
            for (int i = 0; i < R; ++i) in[i].v[q] = cvt<ST>(0.0f);
          }
      }
#pragma unroll
      for (int s = 0; s < TB; ++s) {
        float4 g[P / 4];
#pragma unroll
        for (int q = 0; q < P / 4; ++q) g[q] = *reinterpret_cast<const float4*>(f + s * p.Dp + d + q * 4);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int q = 0; q < P / 4; ++q) {
            float& sum = v[i * TB + s];
            sum += to_f32(in[i].v[q * 4]) * g[q].x; sum += to_f32(in[i].v[q * 4 + 1]) * g[q].y;
            sum += to_f32(in[i].v[q * 4 + 2]) * g[q].z; sum += to_f32(in[i].v[q * 4 + 3]) * g[q].w;
          }
      }
    }
    const float z = sum_lanes<N>(v, lane);
    const long long at = r0 + row;
    if (at < p.V) {
      if (first && p.z) p.z[at * TB + b] = z;
      if (first && id == at) p.logit[b] = z;
      const float top = __builtin_fmaxf(all.x, z);
      if (top != -__builtin_inff() || z != z)  // (-inf: no share; NaN: goes on into the sum)
        all = make_float2(top, (all.x == -__builtin_inff() ? all.y : all.y * expf(all.x - top)) + expf(z - top));
    }
  }
  // lanes of a sample (each sum once), then waves
  for (int o = 32; o >= (64 >> BITS) * TB; o >>= 1) all = join(all, make_float2(__shfl_xor(all.x, o), __shfl_xor(all.y, o)));
  if (first && row == 0) red[wave][b] = all;
  __syncthreads();
  if (tid < p.B) {
    float2 v = red[0][tid];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v = join(v, red[i][tid]);
    p.part[(long long)blockIdx.x * p.B + tid] = v;
  }
}

// A workgroup's join of all parts: of each sample its largest logit, 1 / sum and loss.
template <int TB, int THREADS>
__device__ __forceinline__ void join_parts(const Few& p, float2 (&red)[THREADS], float (&loss)[TB]) {
  const int tid = threadIdx.x, b = tid % TB;
  float2 v = make_float2(-__builtin_inff(), 0.0f);
  if (b < p.B)
#pragma unroll 4
    for (int i = tid / TB; i < p.parts; i += THREADS / TB) v = join(v, p.part[(long long)i * p.B + b]);
  red[tid] = v;
  for (int o = THREADS / 2; o >= TB; o >>= 1) {
    __syncthreads();
    if (tid < o) red[tid] = v = join(v, red[tid + o]);
  }
  if (tid < TB) {
    loss[tid] = is_real(p, tid) ? logf(v.y) + (v.x - p.logit[tid]) : 0.0f;
    red[tid].y = 1.0f / v.y;
  }
  __syncthreads();
}

template <int TB>
__global__ void __launch_bounds__(512) token_few_loss_kernel(const Few p) {
  __shared__ float2 red[512];
  __shared__ float loss[TB];
  join_parts<TB, 512>(p, red, loss);
  if (threadIdx.x < p.B) p.loss[threadIdx.x] = loss[threadIdx.x];
}

// -------------------------------------------------------------------- update
// A workgroup has 64 PER columns of a slice of the rows.
template <typename ST, int TB>
__global__ void __launch_bounds__(kWaves2 * 64) token_few_update_kernel(const Few p) {
  constexpr int P = PER<ST>, T = kWaves2 * 64;
  extern __shared__ __align__(16) float sums[];  // f(X) [TB][64 P]; at the end [kWaves2 - 1][P * TB][64]
  __shared__ float2 norm[T];
  __shared__ float loss[TB];
  __shared__ float e[kStep * TB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (p.D + 64 * P - 1) / (64 * P), d0 = blockIdx.x % blocks * 64 * P, slice = blockIdx.x / blocks;
  const long long begin = (long long)slice * p.rows, end = begin + p.rows < p.V ? begin + p.rows : p.V;
  const int b = tid % TB;
  const long long id = b < p.B ? p.targets[b] : -1;
  const bool real = is_real(p, b);
  const ST* x = static_cast<const ST*>(p.x);
#pragma unroll 1
  for (int i = tid; i < TB * 64 * P; i += T) {
    const int d = d0 + i / TB;
    sums[b * 64 * P + i / TB] = real && d < p.D ? p.alpha * act_f(p.act, to_f32(x[(long long)d * p.B + b])) : 0.0f;
  }
  // this lane's columns: at + skip .. at + P - 1
  const int d = d0 + lane * P, at = d + P <= p.D ? d : p.D - P, skip = d - at;  // (skip >= P: none)
  join_parts<TB, T>(p, norm, loss);
  if (blockIdx.x == 0 && tid < p.B) p.loss[tid] = loss[tid];
  const float2 st = norm[b];
  float f[TB][P], g[TB][P] = {};
#pragma unroll
  for (int s = 0; s < TB; ++s)
#pragma unroll
    for (int q = 0; q < P; ++q) f[s][q] = q >= skip ? sums[s * 64 * P + lane * P + q - skip] : 0.0f;
  ST* w = static_cast<ST*>(p.w) + at;
  for (long long r0 = begin; r0 < end; r0 += kStep) {
    const int many = end - r0 < kStep ? (int)(end - r0) : kStep;
    __syncthreads();
    for (int i = tid; i < many * TB; i += T) {
      const float z = p.z[r0 * TB + i];
      e[i] = !real ? 0.0f : r0 + i / TB == id ? token::target_error(loss[b], 1.0f) : -expf(z - st.x) * st.y;
    }
    __syncthreads();
    if (skip >= P) continue;
    for (int i0 = wave * kRows2; i0 < many; i0 += kWaves2 * kRows2) {
      Sixteen<ST> in[kRows2];
#pragma unroll
      for (int i = 0; i < kRows2; ++i) in[i] = get(w + (r0 + (i0 + i < many ? i0 + i : many - 1)) * p.D);
#pragma unroll
      for (int i = 0; i < kRows2; ++i) {
        if (i0 + i >= many) break;
        float more[P] = {};
#pragma unroll
        for (int s = 0; s < TB; ++s) {
          const float of = e[(i0 + i) * TB + s];
#pragma unroll
          for (int q = 0; q < P; ++q) {
            g[s][q] += to_f32(in[i].v[q]) * of;
            more[q] += of * f[s][q];
          }
        }
        Sixteen<ST> o;
#pragma unroll
        for (int q = 0; q < P; ++q) o.v[q] = cvt<ST>(to_f32(in[i].v[q]) + more[q]);
        ST* to = w + (r0 + i0 + i) * p.D;
        if (skip == 0) {
          *reinterpret_cast<Sixteen<ST>*>(to) = o;
        } else {
#pragma unroll
          for (int q = 1; q < P; ++q)
            if (q >= skip) to[q] = o.v[q];
        }
      }
    }
  }
  // the waves' sums, in order
  __syncthreads();
  if (wave > 0) {
#pragma unroll
    for (int s = 0; s < TB; ++s)
#pragma unroll
      for (int q = 0; q < P; ++q) sums[((wave - 1) * P * TB + s * P + q) * 64 + lane] = g[s][q];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int s = 0; s < TB; ++s) {
    if (s >= p.B) break;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      float v = g[s][q];
#pragma unroll
      for (int i = 0; i < kWaves2 - 1; ++i) v += sums[(i * P * TB + s * P + q) * 64 + lane];
      if (q >= skip) p.grad[((long long)slice * p.D + at + q) * p.B + s] = v;
    }
  }
}

// G = f'(X) times the slices' sums, in order: 16 values a workgroup, 16 threads each.
template <typename ST>
__global__ void __launch_bounds__(256) token_few_finish_kernel(const Few p) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const long long at = (long long)blockIdx.x * 16 + c, count = (long long)p.D * p.B;
  float sum = 0.0f;
  if (at < count)
#pragma unroll 8
    for (int s = r; s < p.slices; s += 16) sum += p.grad[s * count + at];
  red[r][c] = sum;
  __syncthreads();
  if (r != 0 || at >= count) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += red[i][c];
  const float x = to_f32(static_cast<const ST*>(p.x)[at]);
  static_cast<ST*>(p.g)[at] = is_real(p, (int)(at % p.B)) ? cvt<ST>(act_df(p.act, x) * sum) : cvt<ST>(0.0f);
}

struct FewPlan {
  int Dp, parts, blocks, slices, rows;
  long long part, logit, z, grad, bytes;
};
FewPlan plan_few(int V, int D, int B, int storage, bool update) {
  auto up = [](long long v, long long m) { return (v + m - 1) / m * m; };
  FewPlan o;
  const int TB = few_samples(B), per = storage == DT_F32 ? 4 : 8;
  o.Dp = (int)up(D, per);
  const int rows = kWaves * (TB == 1 ? kRows<1> : TB == kMost ? kRows<kMost> : kRows<2>);
  o.parts = (int)std::min<long long>((V + rows - 1LL) / rows, 256);
  o.blocks = (D + 64 * per - 1) / (64 * per);
  o.slices = (int)std::max<long long>(1, std::min<long long>(512 / o.blocks, (V + 31LL) / 32));
  o.rows = (int)up((V + o.slices - 1LL) / o.slices, kWaves2 * kRows2);
  o.slices = (int)((V + (long long)o.rows - 1) / o.rows);
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long here = at;
    at += up(bytes, 256);
    return here;
  };
  o.part = take(8LL * o.parts * B);
  o.logit = take(4LL * B);
  o.z = update ? take(4LL * V * TB) : 0;
  o.grad = update ? take(4LL * o.slices * D * B) : 0;
  o.bytes = at;
  return o;
}

template <typename ST, int TB>
hipError_t run(const TokenProblem& t, int storage, hipStream_t s) {
  const FewPlan o = plan_few(t.V, t.D, t.B, storage, t.g != nullptr);
  unsigned char* ws = t.workspace;
  Few p{t.V, t.D, o.Dp, t.B, t.act, o.parts, o.slices, o.rows, t.x, t.w, t.targets, t.loss, t.g, t.alpha,
        reinterpret_cast<float2*>(ws + o.part), reinterpret_cast<float*>(ws + o.logit),
        t.g ? reinterpret_cast<float*>(ws + o.z) : nullptr, reinterpret_cast<float*>(ws + o.grad)};
  const void* fn = reinterpret_cast<const void*>(&token_few_logits_kernel<ST, TB>);
  static const hipError_t set = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (set != hipSuccess) return set;
  void* args[] = {&p};
  hipError_t e = hipLaunchKernel(fn, dim3((unsigned)o.parts), dim3(kWaves * 64), args, (size_t)4 * TB * o.Dp, s);
  if (e != hipSuccess) return e;
  if (!t.g) {
    hipLaunchKernelGGL((token_few_loss_kernel<TB>), dim3(1), dim3(512), 0, s, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((token_few_update_kernel<ST, TB>), dim3((unsigned)(o.blocks * o.slices)), dim3(kWaves2 * 64),
                     kWaves2 * PER<ST> * TB * 64 * 4, s, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((token_few_finish_kernel<ST>), dim3((unsigned)(((long long)t.D * t.B + 15) / 16)), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename ST>
hipError_t by_samples(const TokenProblem& t, int storage, hipStream_t s) {
  switch (few_samples(t.B)) {
    case 1: return run<ST, 1>(t, storage, s);
    case 2: return run<ST, 2>(t, storage, s);
    case 4: return run<ST, 4>(t, storage, s);
    default:
      if constexpr (std::is_same<ST, float>::value) return run<ST, kMost>(t, storage, s);
      return hipErrorInvalidValue;  // (never)
  }
}

}  // namespace

// us, here / by the general path's matrix products: update 50000 x 1025 x 3 (V, D, B) bf16 79 / 148, 32000 x 4096 x 1 bf16
// 141 / 252, 50000 x 4000 x 8 fp32 506 / 1900; loss 50000 x 512 x 1 bf16 15.6 / 20.7, 50000 x 64 x 1 fp32 10.8 / 31.  In 16 bits
// more samples cost the vector units more than the launches: 500 x 512 x 3 fp16 20 / 17, 50000 x 512 x 8 80 / 58.
bool token_few(int V, int D, int B, int storage) {
  const int most = storage == DT_F32 ? kMost : (long long)V * D >= 1 << 22 ? 4 : 2;
  return B <= most && D >= 8 && 4LL * few_samples(B) * (D + 7) <= kLds && 4LL * few_samples(B) * V <= kLogits;
}

long long token_few_workspace_bytes(int V, int D, int B, int storage, bool update) { return plan_few(V, D, B, storage, update).bytes; }

hipError_t launch_token_few(const TokenProblem& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return by_samples<float>(p, storage, s);
  return storage == DT_F16 ? by_samples<f16>(p, storage, s) : by_samples<bf16>(p, storage, s);
}

}  // namespace ipc
