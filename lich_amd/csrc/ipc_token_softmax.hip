// ipc_token_softmax.hip - softmax cross entropy over a vocabulary in pieces, the logits
// never kept: the products of ipc_token_gemm.h and what stands between them.
//
//   z = W f(X), loss_b = log sum_v exp z[v][b] - z[t_b][b], e = onehot - softmax(z),
//   G = f'(X) W^T e, W += alpha e f(X)^T
//
// 1. f(X) once, in both orders and in the operand type, padded places' columns zero
//    whatever they hold (so that nothing of them reaches W).
// 2. Every piece of the vocabulary: the largest logit and sum of exponentials of each wave's
//    rows.
// 3. A column's parts joined: its loss, largest logit and 1 / sum (with one piece, by step 4; a vocabulary
//    that one tile holds: steps 2 to 4 are one).
// 4. Every piece: its errors in 16 bits (fp32: three terms), its share of W^T e, and its
//    rows of W, which nothing reads any more.
// 5. The shares added in order, times f'(X) (small: in the launch that updates W).
// A small output layer has ipc_token_small.hip, a few samples ipc_token_few.hip.
//
// Errors: a vocabulary whose errors fit one piece (1 GiB) has its exponentials kept there by step
// 2, relative to their part's largest, and scaled in place: three products.  A
// larger one forms its logits again piece by piece: four.  Scaling moves 4 bytes an
// error where forming it takes 2 D operations: it is cheaper from D of a few hundred on, and
// not much dearer below.  Kept in fp16 times 2^15: 2^-12 of the value, down to 2^-29 of the
// part's largest, and so finer than the error's own rounding except where both are fp16's.
//
// In 16 bits errors and, but for identity and relu, f(X) do not fit the operand type.  What
// the results lose by it, and what is done:
//   * G is rounded to the type itself, but a target's error, rounded once, would be off by as much for the whole
//     column, and half of its values would be next to the right ones.  Small updates multiply two terms of the errors
//     (2^-16, 2^-22) with W; large ones add the target's row of W times what rounding left of its error to G's sums.
//   * the loss is fp32 and would be off by the logits' rounding, 2^-9 (2^-12).  The loss alone
//     takes f(X) in two terms (small calls in bf16: three), all in one tile, so that W is read once.
//   * W: a sum that is 2^-9 off rounds a weight in a few hundred of a target's row the other
//     way, and the next loss differs by 1e-5 .. 1e-3.
//   Small updates (TOKEN_FINE_ERRORS, TOKEN_FINE_WORK: launches, not products, are their time) have f(X) and e in
//   two terms, three in bf16, and the exponentials in fp32: all of it is good to 2^-22 and better.  Large ones
//   correct the loss to first order by the gradient that they have, loss -= sum_d (W^T e)_d (f - rounded
//   f)_d (left: half the variance of the logits' rounding, 3e-6 of a loss for bf16 logits of deviation
//   3), and make the errors at the targets, the ones near 1, good in fp32 (token_hot_kernel; left in the next
//   loss: up to 2e-5 in bf16, 3e-6 in fp16, most with few words).  Other errors are probabilities, each rounded
//   once: where a net gives one of them most of a column, that column of G is off by up to its rounding.
#include "ipc_token_gemm.h"

namespace ipc {
namespace {

// ------------------------------------------------------------------ f(X)
// F [f_terms][D][Bk] and FT [T][B][Dp] of X [D][B] in the operand type (T terms), zeros past
// the ends and in padded columns.
struct States {
  int D, B, V, Dp, Bk, f_terms;
  const void* x;
  const long long* targets;
  unsigned short* f;  // its first f_terms terms, or nullptr
  unsigned short* ft;
};

// v as the operand's bits; of a sum of terms (`again`), what is left of it.  The first
// term of a finite value stays finite; an infinite one's others are 0.
template <typename OT>
__device__ __forceinline__ unsigned short term(float& v, bool again) {
  OT o = cvt<OT>(v);
  if (again) {
    const bool inf = __builtin_isinf(v);
    if (!inf && __builtin_isinf(to_f32(o)))
      o = __builtin_bit_cast(OT, (unsigned short)((v > 0.0f ? 0u : 0x8000u) | (std::is_same<OT, bf16>::value ? 0x7f7fu : 0x7bffu)));
    v = inf ? 0.0f : v - to_f32(o);
  }
  return __builtin_bit_cast(unsigned short, o);
}
// The same of f(X) in fp32, cut off towards zero (eight bits a term, so three are all 24): a value's terms have its
// sign, those with nothing left too (2^-126), so that an infinite weight's products with them are all the
// infinity that its product with the value is.  What the three products left out come to grows from 6e-9 of a logit to
// 1.8e-8, where the fp32 sums of the others are 1e-7 off.
__device__ __forceinline__ unsigned short inner_term(float& v) {
  if (v != v) return __builtin_bit_cast(unsigned short, cvt<bf16>(v));
  const unsigned bits = __builtin_bit_cast(unsigned, v) & 0xffff0000u;
  if (v != 0.0f) {
    const float left = v - __builtin_bit_cast(float, bits);
    v = __builtin_fabsf(left) >= 0x1p-126f ? left : __builtin_copysignf(0x1p-126f, v);  // (of infinity NaN is left)
  }
  return (unsigned short)(bits >> 16);
}

template <typename ST, typename OT, int TERMS, int ACT>
__device__ __forceinline__ void lay_states(const States& p, int block) {
  __shared__ unsigned short tile[32][34];
  const int tiles_n = p.Bk / 32, d0 = block / tiles_n * 32, n0 = block % tiles_n * 32;
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = n0 + c;
  const long long id = n < p.B ? p.targets[n] : -1;
  const bool real = id >= 0 && id < p.V;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = d0 + i * 8 + r;
    v[i] = n < p.B && d < p.D ? to_f32(static_cast<const ST*>(p.x)[(long long)d * p.B + n]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = real && d0 + i * 8 + r < p.D ? act_t<ACT>(v[i]) : 0.0f;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    if (t > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = d0 + i * 8 + r;
      unsigned short h;
      if constexpr (std::is_same<ST, float>::value) h = inner_term(v[i]);
      else h = term<OT>(v[i], TERMS > 1);
      tile[i * 8 + r][c] = h;
      if (p.f && t < p.f_terms && d < p.D) p.f[((long long)t * p.D + d) * p.Bk + n] = h;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = n0 + i * 8 + r;
      if (row < p.B) p.ft[((long long)t * p.B + row) * p.Dp + d0 + c] = tile[c][i * 8 + r];
    }
  }
}

// ------------------------------------------------------------------ W
// Rows of W as TERMS matrices of the operand type with rows of Dp, zeros past the ends.
struct Rows {
  int rows, padded, D, Dp;
  const void* w;
  unsigned short* out;
};
template <typename ST, typename OT, int TERMS>
__device__ __forceinline__ void lay_rows(const Rows& p, unsigned block) {
  const long long at = ((long long)block * 256 + threadIdx.x) * 4, count = (long long)p.padded * p.Dp;
  if (at >= count) return;
  const int r = (int)(at / p.Dp), d = (int)(at - (long long)r * p.Dp);
  const ST* from = static_cast<const ST*>(p.w) + (long long)r * p.D + d;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = r < p.rows && d + i < p.D ? to_f32(from[i]) : 0.0f;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    unsigned short h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = term<OT>(v[i], TERMS > 1);
    *reinterpret_cast<uint2*>(p.out + t * count + at) = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
  }
}

// Workgroups 0 .. states - 1: f(X); the others: rows of W.
template <typename ST, typename OT, int TERMS, int ACT>
__global__ void __launch_bounds__(256) token_lay_kernel(const States x, const Rows w, unsigned states) {
  if (blockIdx.x < states) lay_states<ST, OT, TERMS, ACT>(x, blockIdx.x);
  else lay_rows<ST, OT, std::is_same<ST, float>::value ? 3 : 1>(w, blockIdx.x - states);  // (whatever terms f(X) has)
}

// ---------------------------------------------------------------- a column's tiles
struct Columns {
  int B, V, tiles;
  const float2* part;  // [tiles][B]
  const float* logit;  // of the target
  const long long* targets;
  float* loss;
  float2* norm;
};
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float top = __builtin_fmaxf(a.x, b.x), none = -__builtin_inff();
  return make_float2(top, (a.x == none ? a.y : a.y * expf(a.x - top)) + (b.x == none ? b.y : b.y * expf(b.x - top)));
}
// `across` columns a workgroup (a power of two, 16 at most), 1024 / across threads each
__global__ void __launch_bounds__(1024) token_columns_kernel(const Columns p, int across) {
  __shared__ float2 red[1024];
  const int c = threadIdx.x & (across - 1), each = 1024 / across, g = threadIdx.x / across, n = blockIdx.x * across + c;
  float2 v = make_float2(-__builtin_inff(), 0.0f);
  if (n < p.B)
    for (int t = g; t < p.tiles; t += each) v = join(v, p.part[(long long)t * p.B + n]);
  red[threadIdx.x] = v;
  for (int o = each / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (g < o) red[threadIdx.x] = v = join(v, red[threadIdx.x + o * across]);
  }
  if (g != 0 || n >= p.B) return;
  const long long id = p.targets[n];
  p.loss[n] = id >= 0 && id < p.V ? logf(v.y) + (v.x - p.logit[n]) : 0.0f;
  p.norm[n] = make_float2(v.x, 1.0f / v.y);
}

// ---------------------------------------------------------------- the loss
// loss -= the fixes, in order; 16 columns a workgroup, 16 threads each.  (Not below 0, where to first order it may
// be once logits of a thousand and more are off by some.)
__global__ void __launch_bounds__(256) token_fix_kernel(const float* fixes, int rows, int B, float* loss) {
  __shared__ float red[16][16];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
  float sum = 0.0f;
  if (n < B)
#pragma unroll 8
    for (int i = g; i < rows; i += 16) sum += fixes[(long long)i * B + n];
  red[g][c] = sum;
  __syncthreads();
  if (g != 0 || n >= B) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += red[i][c];
  sum = loss[n] - sum;
  loss[n] = sum < 0.0f ? 0.0f : sum;
}

// ------------------------------------------------------------------ errors
// Kept exponentials into errors, in place, or from fp32 into two or three terms: a column (a row of ET, up
// to Vp) a workgroup, which joins the column's parts itself, up to TOKEN_ERROR_RUN values; of longer
// ones 2048 values, their columns joined before.  Zeros past the ends and in padded rows, up
// to Bk.  us, joining here / before: V = 10007, B = 77 fp32 9.6 / 4.7 + 5.4; V = 32000, B = 1024
// bf16 34.8 / 6.3 + 27.0; V = 128000, B = 2048 341 / 14.6 + 226.
struct Errors {
  int V, B, Vp, Bk, unit, units;
  const void* kept;     // [Bk][Vp]
  unsigned short* et;
  const float2* part;   // [units][B]
  const float* logit;
  float* loss;
  const float2* norm;
  const long long* targets;
  float scale;
};
template <typename OT, int TERMS, bool JOIN>
__global__ void __launch_bounds__(256) token_errors_kernel(const Errors p) {
  __shared__ float2 red[4];
  const int runs = JOIN ? 1 : (p.Vp + 2047) / 2048, n = blockIdx.x / runs, tid = threadIdx.x;
  const int first = blockIdx.x % runs * 2048, last = JOIN ? p.Vp : min(first + 2048, p.Vp);
  const long long id = n < p.B ? p.targets[n] : -1;
  const bool real = id >= 0 && id < p.V;  // (the same for the whole workgroup)
  float2 all = make_float2(-__builtin_inff(), 0.0f);  // y: 1 / sum
  float loss = 0.0f;
  if constexpr (JOIN) {
    if (real) {
      for (int t = tid; t < p.units; t += 256) all = join(all, p.part[(long long)t * p.B + n]);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) all = join(all, make_float2(__shfl_xor(all.x, o), __shfl_xor(all.y, o)));
      if ((tid & 63) == 0) red[tid >> 6] = all;
      __syncthreads();
      all = join(join(red[0], red[1]), join(red[2], red[3]));
      loss = logf(all.y) + (all.x - p.logit[n]);
      all.y = 1.0f / all.y;
    }
    if (tid == 0 && n < p.B) p.loss[n] = loss;
  } else if (real) {
    all = p.norm[n];
    loss = p.loss[n];
  }
  const float norm = -p.scale * all.y;
  for (int v = first + tid * 8; v < last; v += 256 * 8) {
    const long long place = (long long)n * p.Vp + v;
    float e[8] = {};
    if (real && v < p.V) {
      const float part = p.part[(long long)(v / p.unit) * p.B + n].x;
      const float share = norm * (part == -__builtin_inff() ? 0.0f : expf(part - all.x));
      if constexpr (TERMS == 1) {
        const f16x8 h = *reinterpret_cast<const f16x8*>(static_cast<const unsigned short*>(p.kept) + place);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (float)h[i] * (1.0f / 32768.0f) * share;
      } else {
        const float4* k = reinterpret_cast<const float4*>(static_cast<const float*>(p.kept) + place);
        const float4 a = k[0], b = k[1];
        e[0] = a.x; e[1] = a.y; e[2] = a.z; e[3] = a.w; e[4] = b.x; e[5] = b.y; e[6] = b.z; e[7] = b.w;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] *= share;
      }
      if (v + 8 > p.V) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v + i >= p.V) e[i] = 0.0f;
      }
      if (id >= v && id < v + 8) {
        const float own = token::target_error(loss, p.scale);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (id == v + i) e[i] = own;
      }
    }
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      unsigned short h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = term<OT>(e[i], TERMS > 1);
      *reinterpret_cast<uint4*>(p.et + (long long)t * p.Bk * p.Vp + place) =
          make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
    }
  }
}

// ---------------------------------------------------------------- targets' rows
// What rounding e and f to 16 bits leaves out of the sum e f^T where e is near 1, at the
// targets: hot[p][d] = sum over the columns n of sorted positions p .. of one target of
// (e - rounded e) rounded f + e (f - rounded f), for the first position p of each target.
// (Elsewhere e is a probability, whose rounding counts as little.  Without this a weight in a
// few hundred of a target's row rounds the other way, and the next loss differs by 1e-5 .. 1e-3.)
// A workgroup has 256 features of a position: HOT_GROUPS waves take every so many-th column.  (Words
// are not drawn evenly: the commonest has a tenth of the columns.  128000 words, 2048 samples of 2048 features,
// fp16: 26 us; with G's part 33.)
constexpr int HOT_GROUPS = 4;
struct Hot {
  int B, D, Dp;
  const int* order;
  const int* key;
  const unsigned short* ft;  // [TWO ? 2 : 1][B][Dp]
  const float* loss;
  float* hot;                // [B][Dp]
  float scale;
};

// And out of W^T e: rest[d][n] = (e - rounded e) W[t_n][d], 64 features by 64 columns a workgroup, turned in LDS.
struct Rest {
  int V, D, B;
  const void* w;
  const long long* targets;
  const float* loss;
  float* rest;  // [D][B]
  float scale;
};
template <typename OT>
__device__ __forceinline__ void rest_of_targets(const Rest& p, int block) {
  constexpr int WAVES = HOT_GROUPS, EACH = 64 / WAVES;
  __shared__ float tile[64][65], left[64];
  const int tiles_d = (p.D + 63) / 64, d0 = block % tiles_d * 64, n0 = block / tiles_d * 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const OT* w = static_cast<const OT*>(p.w) + (d0 + lane < p.D ? d0 + lane : 0);
  // a wave has 16 columns, a lane of it the target and error of one
  const int mine = n0 + wave * EACH + (lane & (EACH - 1));
  long long id = mine < p.B ? p.targets[mine] : -1;
  if (id >= p.V) id = -1;
  const int row = (int)id;
  if (lane < EACH) {
    const float e = id < 0 ? 0.0f : token::target_error(p.loss[mine], p.scale);
    left[wave * EACH + lane] = e - to_f32(cvt<OT>(e));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  OT v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int r = __builtin_amdgcn_readlane(row, i);
    v[i] = w[(long long)(r < 0 ? 0 : r) * p.D];
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i)  // (a padded column: none, whatever its row would hold)
    tile[wave * EACH + i][lane] = __builtin_amdgcn_readlane(row, i) < 0 ? 0.0f : to_f32(v[i]) * left[wave * EACH + i];
  __syncthreads();
  if (n0 + lane >= p.B) return;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int d = wave * EACH + i;
    if (d0 + d < p.D) p.rest[(long long)(d0 + d) * p.B + n0 + lane] = tile[lane][d];
  }
}

// Workgroups 0 .. first - 1: G's part; the others: W's.
template <typename OT, bool TWO>
__global__ void __launch_bounds__(HOT_GROUPS * 64) token_hot_kernel(const Hot p, const Rest q, unsigned first) {
  if (blockIdx.x < first) {
    rest_of_targets<OT>(q, blockIdx.x);
    return;
  }
  __shared__ float4 red[HOT_GROUPS][64];
  const int slabs = (p.Dp + 255) / 256, block = blockIdx.x - first, at = block / slabs, lane = threadIdx.x & 63;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = block % slabs * 256 + lane * 4;
  const int id = p.key[at];
  if (id < 0 || (at > 0 && p.key[at - 1] == id)) return;
  float sum[4] = {};
  const OT* ft = reinterpret_cast<const OT*>(p.ft) + (d < p.Dp ? d : 0);
  for (int i = at;; i += 64) {
    // 64 columns of this target, fewer at its end: a lane each for their places and errors
    const unsigned long long other = __ballot(p.key[i + lane < p.B ? i + lane : p.B] != id);
    const int many = other ? __ffsll(other) - 1 : 64, mine = lane < many ? p.order[i + lane] : 0;
    const float e = token::target_error(p.loss[mine], p.scale), left = e - to_f32(cvt<OT>(e));
#pragma unroll 8
    for (int c = group; c < many; c += HOT_GROUPS) {
      const long long n = __builtin_amdgcn_readlane(mine, c);
      const float all = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), c));
      const float rest = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(left), c));
      float f[4], g[4] = {};
      load4(ft + n * p.Dp, f);
      if constexpr (TWO) load4(ft + (p.B + n) * p.Dp, g);
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] += TWO ? rest * f[q] + all * g[q] : rest * f[q];
    }
    if (other) break;
  }
  red[group][lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
  __syncthreads();
  if (group != 0 || d >= p.Dp) return;
  float4 all = red[0][lane];
#pragma unroll
  for (int g = 1; g < HOT_GROUPS; ++g) {
    all.x += red[g][lane].x; all.y += red[g][lane].y; all.z += red[g][lane].z; all.w += red[g][lane].w;
  }
  *reinterpret_cast<float4*>(p.hot + (long long)at * p.Dp + d) = all;
}

template <typename ST, typename OT, int TERMS, int ACT>
hipError_t run(const TokenProblem& p, int storage, hipStream_t s) {
  const bool update = p.g != nullptr;
  TokenPlan o;
  if (!plan_token(p.V, p.D, p.B, storage, p.act, update, o)) return hipErrorInvalidValue;
  unsigned char* ws = p.workspace;
  auto at = [&](long long offset) { return reinterpret_cast<unsigned short*>(ws + offset); };
  const States st{p.D, p.B, p.V, o.Dp, o.Bk, o.f_terms, p.x, p.targets, update ? at(o.f) : nullptr, at(o.ft)};
  const unsigned state_tiles = (unsigned)((long long)(o.Dp / 32) * (o.Bk / 32));
  hipError_t e = hipSuccess;
  auto rows_of = [&](int first) { return std::min(o.rows, p.V - first); };
  // the piece's rows of W where they are laid out, and (states: workgroups) f(X)
  auto lay_out = [&](int first, unsigned states) {
    const int rows = rows_of(first), padded = (rows + 31) / 32 * 32;
    const Rows r{rows, padded, p.D, o.Dp, static_cast<const ST*>(p.w) + (long long)first * p.D, at(o.ws)};
    const long long fours = o.copy ? (long long)padded * o.Dp / 4 : 0;
    const dim3 grid(states + (unsigned)((fours + 255) / 256)), block(256);
    if (o.ft_terms == 2) hipLaunchKernelGGL((token_lay_kernel<ST, OT, TERMS == 1 ? 2 : TERMS, ACT>), grid, block, 0, s, st, r, states);
    else if (o.ft_terms == 3) hipLaunchKernelGGL((token_lay_kernel<ST, OT, std::is_same<OT, bf16>::value ? 3 : TERMS, ACT>), grid, block, 0, s, st, r, states);
    else hipLaunchKernelGGL((token_lay_kernel<ST, OT, TERMS, ACT>), grid, block, 0, s, st, r, states);
    if (e == hipSuccess) e = hipGetLastError();
  };
  // the piece's rows of W, as an operand of the products
  auto weights = [&](int first, TokenGemm& q, bool lay) {
    const int rows = rows_of(first), padded = (rows + 31) / 32 * 32;
    const ST* w = static_cast<const ST*>(p.w) + (long long)first * p.D;
    if (!o.copy) {
      q.a = w; q.lda = p.D; q.a_bytes = (long long)rows * p.D * 2; q.a_term = 0;
      return;
    }
    if (lay) lay_out(first, 0);
    q.a = at(o.ws); q.lda = o.Dp;
    q.a_term = (unsigned)(padded * o.Dp * 2);
    q.a_bytes = (long long)TERMS * padded * o.Dp * 2;
  };
  auto logits = [&](int first, bool lay) {
    TokenGemm q{};
    weights(first, q, lay);
    q.M = rows_of(first); q.N = p.B; q.K = o.copy ? o.Dp : p.D;
    q.b = at(o.ft); q.ldb = o.Dp; q.b_term = (unsigned)(p.B * o.Dp * 2); q.b_bytes = (long long)o.ft_terms * p.B * o.Dp * 2;
    q.targets = p.targets; q.first = first; q.V = p.V;
    q.target_logit = reinterpret_cast<float*>(ws + o.logit);
    return q;
  };
  float2* part = reinterpret_cast<float2*>(ws + o.stats);
  // fp16: errors below its smallest normal number matter (1 / V), so they are kept times 2^10
  const float scale = storage == DT_F16 ? 1024.0f : 1.0f;
  lay_out(0, state_tiles);
  if (e != hipSuccess) return e;
  for (int first = 0; first < p.V && e == hipSuccess; first += o.rows) {
    TokenGemm q = logits(first, first > 0);
    if (e != hipSuccess) return e;
    q.out = part + (long long)(first / o.unit) * p.B;
    if (o.one) {
      q.scal = scale;
      if (update) {
        q.out = at(o.et); q.out_ld = o.Vp; q.out_rows = o.Bk; q.out_term = (long long)o.Bk * o.Vp;
      }
      q.target_logit = p.loss;
      e = launch_token_one(q, storage, o.ways, s);
    } else if (o.keep) {
      q.kept = ws + o.kept; q.out_ld = o.Vp; q.out_rows = o.Bk;
      e = launch_token_keep(q, storage, o.tile, o.ways, s);
    } else {
      e = launch_token_stats(q, storage, o.tile, o.ways, s);
    }
  }
  if (e != hipSuccess) return e;
  const int units = (p.V + o.unit - 1) / o.unit;
  const bool joined = o.keep && o.Vp <= TOKEN_ERROR_RUN;  // with the errors
  if (!joined && !o.one) {
    const Columns c{p.B, p.V, units, part, reinterpret_cast<const float*>(ws + o.logit), p.targets, p.loss,
                    reinterpret_cast<float2*>(ws + o.norm)};
    int across = 16;
    while (across > 1 && across / 2 >= p.B) across /= 2;
    hipLaunchKernelGGL(token_columns_kernel, dim3((unsigned)((p.B + across - 1) / across)), dim3(1024), 0, s, c, across);
    e = hipGetLastError();
  }
  if (!update || e != hipSuccess) return e;

  float* fixes = o.fix ? reinterpret_cast<float*>(ws + o.fixes) : nullptr;
  const int vec_state = p.B % 4 == 0 && reinterpret_cast<uintptr_t>(p.x) % (4 * sizeof(ST)) == 0 &&
                        reinterpret_cast<uintptr_t>(p.g) % (4 * sizeof(ST)) == 0;
  const TokenFinish finish{p.D, p.B, p.V, o.slices + (o.mend ? 1 : 0), p.act, reinterpret_cast<const float*>(ws + o.part), p.x, p.targets, p.g,
                           1.0f / scale, fixes, vec_state};
  auto make_good = [&] {  // once the losses are known
    int *order = reinterpret_cast<int*>(ws + o.order), *key = reinterpret_cast<int*>(ws + o.key);
    e = launch_sort_places(p.targets, p.B, p.V, order, key, reinterpret_cast<int*>(ws + o.slot), s);
    if (e != hipSuccess) return;
    const Hot h{p.B, p.D, o.Dp, order, key, at(o.ft), p.loss, reinterpret_cast<float*>(ws + o.hot), scale};
    // (the slice behind the products')
    const Rest r{p.V, p.D, p.B, p.w, p.targets, p.loss, reinterpret_cast<float*>(ws + o.part) + (long long)o.slices * p.D * p.B, scale};
    const unsigned rests = (unsigned)token_rest_blocks(p.D, p.B);
    const dim3 grid(rests + (unsigned)token_hot_blocks(o.Dp, p.B)), block(HOT_GROUPS * 64);
    if (o.ft_terms == 2) hipLaunchKernelGGL((token_hot_kernel<OT, true>), grid, block, 0, s, h, r, rests);
    else hipLaunchKernelGGL((token_hot_kernel<OT, false>), grid, block, 0, s, h, r, rests);
    e = hipGetLastError();
  };
  for (int first = 0; first < p.V; first += o.rows) {
    const int rows = rows_of(first), Vp = (rows + 31) / 32 * 32;
    if (o.keep && !o.one) {
      const Errors er{p.V, p.B, Vp, o.Bk, o.unit, units, ws + o.kept, at(o.et), part, reinterpret_cast<const float*>(ws + o.logit),
                      p.loss, reinterpret_cast<const float2*>(ws + o.norm), p.targets, scale};
      const dim3 grid((unsigned)token_error_blocks(o.Bk, Vp));
      constexpr int MORE = std::is_same<OT, bf16>::value ? 3 : 2;
      if (o.e_terms == 1 && joined) hipLaunchKernelGGL((token_errors_kernel<OT, TERMS, true>), grid, dim3(256), 0, s, er);
      else if (o.e_terms == 1) hipLaunchKernelGGL((token_errors_kernel<OT, TERMS, false>), grid, dim3(256), 0, s, er);
      else if (joined) hipLaunchKernelGGL((token_errors_kernel<OT, MORE, true>), grid, dim3(256), 0, s, er);
      else hipLaunchKernelGGL((token_errors_kernel<OT, MORE, false>), grid, dim3(256), 0, s, er);
      e = hipGetLastError();
    } else if (!o.keep) {
      TokenGemm q = logits(first, o.rows < p.V);  // (one piece: its rows are laid out already)
      if (e != hipSuccess) return e;
      q.stats = reinterpret_cast<const float2*>(ws + o.norm);
      q.out = at(o.et); q.out_ld = Vp; q.out_rows = o.Bk; q.out_term = (long long)o.Bk * Vp; q.scal = scale; q.loss = p.loss;
      e = launch_token_error(q, storage, o.tile, s);
    }
    if (e == hipSuccess && o.mend && first == 0) make_good();
    if (e != hipSuccess) return e;
    TokenGemm g{};
    weights(first, g, false);
    g.M = p.D; g.N = p.B; g.K = Vp;
    g.b = at(o.et); g.ldb = Vp; g.b_term = (unsigned)((long long)o.Bk * Vp * 2); g.b_bytes = (long long)o.e_terms * o.Bk * Vp * 2;
    g.slices = token_piece_slices(o, rows); g.out = ws + o.part; g.add = first > 0;
    if (!o.tail) e = launch_token_grad(g, storage, o.grad_tile, o.grad_ways, s);
    if (e != hipSuccess) return e;
    TokenGemm u{};
    u.a = at(o.et); u.lda = Vp; u.a_term = g.b_term; u.a_bytes = (long long)o.e_terms * o.Bk * Vp * 2;
    u.b = at(o.f); u.ldb = o.Bk; u.b_term = (unsigned)(p.D * o.Bk * 2); u.b_bytes = (long long)o.f_terms * p.D * o.Bk * 2;
    u.M = rows; u.N = p.D; u.K = o.Bk;
    u.out = static_cast<ST*>(p.w) + (long long)first * p.D;
    u.vec = p.D % 4 == 0 && reinterpret_cast<uintptr_t>(p.w) % (4 * sizeof(ST)) == 0;
    u.scal = p.alpha / scale;
    if (o.tail) {
      g.out = p.g; g.x = p.x; g.act = p.act; g.targets = p.targets; g.V = p.V; g.scal = 1.0f / scale;
      u.slices = o.cut;
      return launch_token_tail(g, u, reinterpret_cast<float*>(ws + o.part), storage, s);
    }
    if (o.mend) {
      u.slot = reinterpret_cast<const int*>(ws + o.slot) + first;
      u.hot = reinterpret_cast<const float*>(ws + o.hot);
      u.hot_ld = o.Dp;
    }
    e = launch_token_weight(u, first + rows == p.V ? &finish : nullptr, storage, o.f_terms, s);
    if (e != hipSuccess) return e;
  }
  if (!fixes) return e;
  hipLaunchKernelGGL(token_fix_kernel, dim3((unsigned)((p.B + 15) / 16)), dim3(256), 0, s, fixes, token_fix_rows(p.D, vec_state), p.B, p.loss);
  return hipGetLastError();
}

template <typename ST, typename OT, int TERMS>
hipError_t by_act(const TokenProblem& p, int storage, hipStream_t s) {
  switch (p.act) {
    case ACT_RELU: return run<ST, OT, TERMS, ACT_RELU>(p, storage, s);
    case ACT_TANH: return run<ST, OT, TERMS, ACT_TANH>(p, storage, s);
    case ACT_SIGMOID: return run<ST, OT, TERMS, ACT_SIGMOID>(p, storage, s);
    case ACT_SILU: return run<ST, OT, TERMS, ACT_SILU>(p, storage, s);
    case ACT_GELU: return run<ST, OT, TERMS, ACT_GELU>(p, storage, s);
    default: return run<ST, OT, TERMS, ACT_IDENTITY>(p, storage, s);
  }
}

}  // namespace

long long token_workspace_bytes(int V, int D, int B, int storage, int act, bool update) {
  if (token_few(V, D, B, storage)) return token_few_workspace_bytes(V, D, B, storage, update);
  TokenPlan o;
  return plan_token(V, D, B, storage, act, update, o) ? o.bytes : 0;
}

hipError_t launch_token(const TokenProblem& p, int storage, hipStream_t s) {
  if (token_small(p.V, p.D, p.B)) return launch_token_small(p, storage, s);
  if (token_few(p.V, p.D, p.B, storage)) return launch_token_few(p, storage, s);
  if (storage == DT_F32) return by_act<float, bf16, 3>(p, storage, s);
  return storage == DT_F16 ? by_act<f16, f16, 1>(p, storage, s) : by_act<bf16, bf16, 1>(p, storage, s);
}

}  // namespace ipc
