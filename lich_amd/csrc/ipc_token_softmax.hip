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
// 3. A column's parts joined: its loss, largest logit and 1 / sum.
// 4. Every piece: its errors in 16 bits (fp32: three terms), its share of W^T e, and its
//    rows of W, which nothing reads any more.
// 5. The shares added in order, times f'(X).
//
// Errors: a vocabulary whose errors fit one piece (1 GiB) has its exponentials kept there by step
// 2, relative to their part's largest, and scaled in place: three products.  A
// larger one forms its logits again piece by piece: four.  Scaling moves 4 bytes an
// error where forming it takes 2 D operations: it is cheaper from D of a few hundred on, and
// not much dearer below.  Kept in fp16 times 2^15: 2^-12 of the value, down to 2^-29 of the
// part's largest, and so finer than the error's own rounding except where both are fp16's.
//
// f(X) in 16 bits, where it is not exact there (all but identity and relu): the loss, which is
// fp32, would be off by the logits' 2^-9 (2^-12).  The loss alone takes f(X) in two terms, both
// in one tile, so that W is read once.  The update corrects it to first order instead,
// by the gradient that it has: loss -= sum_d (W^T e)_d (f - rounded f)_d; what is left
// is half the variance of the logits' rounding, 3e-6 of a loss for bf16 logits of deviation 3.
#include <algorithm>

#include "ipc_token_gemm.h"

namespace ipc {
namespace {

constexpr long long kPieceBytes = 1LL << 30;  // of a piece's errors, and of its rows of W where those are laid out
constexpr long long kOperand = (1LL << 31) - 1;

struct Plan {
  int terms, Dp, Bk;
  bool copy;          // W laid out per piece: fp32, or 16-bit rows of an odd length
  bool two;           // the loss alone: f(X) in two terms
  bool fix;           // the update: the loss corrected
  bool keep;          // one piece, its exponentials kept
  int rows, Vp;       // of a piece (the last may have fewer), ET's row length
  int tile, unit;     // of the logits
  int grad_tile, slices;
  long long f, ft, et, kept, ws, part, stats, logit, norm, fixes, bytes;  // offsets in the workspace
};

bool make_plan(int V, int D, int B, int storage, int act, bool update, Plan& o) {
  auto up = [](long long v, long long m) { return (v + m - 1) / m * m; };
  o = Plan{};
  o.terms = storage == DT_F32 ? 3 : 1;
  if (D > (1 << 26) || B > (1 << 26)) return false;
  o.Dp = (int)up(D, 32);
  o.Bk = (int)up(B, 32);
  o.copy = storage == DT_F32 || D % 2 != 0;
  const bool inexact = storage != DT_F32 && act != ACT_IDENTITY && act != ACT_RELU;
  o.two = inexact && !update;
  o.fix = inexact && update;
  const long long state = (long long)o.terms * o.Dp * o.Bk * 2;
  if (state * (o.two ? 2 : 1) > kOperand) return false;
  const long long row_w = 2LL * (o.copy ? o.terms * o.Dp : D), row_e = update ? 2LL * o.terms * o.Bk : 1;
  long long rows = std::min((o.copy ? kPieceBytes : kOperand) / row_w, kPieceBytes / row_e) / 256 * 256;
  if (rows < 256) rows = 256;
  if (rows * std::max(row_w, row_e) > kOperand && std::min<long long>(rows, up(V, 32)) * std::max(row_w, row_e) > kOperand) return false;
  o.rows = (int)std::min<long long>(rows, V);
  o.Vp = (int)up(o.rows, 32);
  o.keep = update && o.rows == V && (storage != DT_F32 || (long long)o.Bk * o.Vp * 10 <= kPieceBytes);
  auto tiles = [&](long long m, long long n, long long e) { return ((m + e - 1) / e) * ((n + e - 1) / e); };
  const long long columns = o.two ? 2LL * B : B;
  if (columns <= 64) o.tile = o.rows >= 32768 ? TILE_128_64 : TILE_64;
  else o.tile = tiles(o.rows, columns, 256) >= 192 ? TILE_256 : tiles(o.rows, columns, 128) > 128 ? TILE_128 : TILE_64;
  o.unit = token_unit(o.tile, o.two);
  o.grad_tile = D >= 256 && B >= 256 ? 256 : D > 64 ? 128 : 64;
  const long long gt = o.grad_tile == 256 ? tiles(D, B, 256)
                       : o.grad_tile == 128 ? (D + 127LL) / 128 * (B > 64 ? (B + 127LL) / 128 : 1) : tiles(D, B, 64);
  const long long stages = (long long)(o.terms == 3 ? token::PRODUCTS : 1) * (o.Vp / 32);
  o.slices = (int)std::max<long long>(1, std::min({256 / gt, stages / 8, 64LL}));
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long here = at;
    at += up(bytes, 256);
    return here;
  };
  o.ft = take(o.two ? 2 * state : state);
  o.logit = take(4LL * B);
  o.norm = take(8LL * B);
  o.stats = take(8LL * B * (((long long)V + o.unit - 1) / o.unit));
  if (o.copy) o.ws = take((long long)o.terms * o.Vp * o.Dp * 2);
  if (update) {
    o.f = take(state);
    o.et = take((long long)o.terms * o.Bk * o.Vp * 2);
    o.part = take(4LL * o.slices * D * B);
    o.kept = storage != DT_F32 ? o.et : o.keep ? take(4LL * o.Bk * o.Vp) : 0;
    o.fixes = o.fix ? take(4LL * B * ((D + 31) / 32)) : 0;
  }
  o.bytes = at;
  return true;
}

// ------------------------------------------------------------------ f(X)
// F [T][D][Bk] and FT [T][B][Dp] of X [D][B] in the operand type (T terms), zeros past
// the ends and in padded columns.
struct States {
  int D, B, V, Dp, Bk;
  const void* x;
  const long long* targets;
  unsigned short* f;  // or nullptr
  unsigned short* ft;
};

// v as the operand's bits; of a sum of terms (`again`), what is left of it.  The first
// term stays finite, of infinities too (the largest, and nothing left): the products of an
// infinity with the other operand's terms, of either sign, would make a NaN of it.
template <typename OT>
__device__ __forceinline__ unsigned short term(float& v, bool again) {
  OT o = cvt<OT>(v);
  if (again) {
    const bool inf = __builtin_isinf(v);
    if (__builtin_isinf(to_f32(o)))
      o = __builtin_bit_cast(OT, (unsigned short)((v > 0.0f ? 0u : 0x8000u) | (std::is_same<OT, bf16>::value ? 0x7f7fu : 0x7bffu)));
    v = inf ? 0.0f : v - to_f32(o);
  }
  return __builtin_bit_cast(unsigned short, o);
}

template <typename ST, typename OT, int TERMS, int ACT>
__global__ void __launch_bounds__(256) token_states_kernel(const States p) {
  // (TERMS 2: the loss alone, whose second term is what the first leaves of f(X))
  __shared__ unsigned short tile[64][66];
  const int tiles_n = (p.Bk + 63) / 64, d0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
  const int tid = threadIdx.x, c = tid & 63, n = n0 + c;
  const long long id = n < p.B ? p.targets[n] : -1;
  const bool real = id >= 0 && id < p.V;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = d0 + i * 4 + (tid >> 6);
    v[i] = real && d < p.D ? act_t<ACT>(to_f32(static_cast<const ST*>(p.x)[(long long)d * p.B + n])) : 0.0f;
  }
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = i * 4 + (tid >> 6), d = d0 + r;
      const unsigned short h = term<OT>(v[i], TERMS > 1);
      tile[r][c] = h;
      if (p.f && d < p.D && n < p.Bk) p.f[((long long)t * p.D + d) * p.Bk + n] = h;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = i * 4 + (tid >> 6), row = n0 + r, d = d0 + c;
      if (row < p.B && d < p.Dp) p.ft[((long long)t * p.B + row) * p.Dp + d] = tile[c][r];
    }
    __syncthreads();
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
__global__ void __launch_bounds__(256) token_rows_kernel(const Rows p) {
  const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4, count = (long long)p.padded * p.Dp;
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
// 16 columns a workgroup, 64 threads each
__global__ void __launch_bounds__(1024) token_columns_kernel(const Columns p) {
  __shared__ float2 red[64][16];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
  float2 v = make_float2(-__builtin_inff(), 0.0f);
  if (n < p.B)
    for (int t = g; t < p.tiles; t += 64) v = join(v, p.part[(long long)t * p.B + n]);
  red[g][c] = v;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    __syncthreads();
    if (g < o) red[g][c] = v = join(v, red[g + o][c]);
  }
  if (g != 0 || n >= p.B) return;
  const long long id = p.targets[n];
  p.loss[n] = id >= 0 && id < p.V ? logf(v.y) + (v.x - p.logit[n]) : 0.0f;
  p.norm[n] = make_float2(v.x, 1.0f / v.y);
}

// ------------------------------------------------------------------ G
struct Grad {
  int D, B, V, slices;
  const float* part;  // [slices][D][B]
  const void* x;
  const long long* targets;
  void* g;
  float scale;
  float* fixes;       // [(D + 31) / 32][B], or nullptr
};
// 32 rows of 64 columns a workgroup
template <typename ST, int ACT>
__global__ void __launch_bounds__(256) token_gradient_kernel(const Grad p) {
  __shared__ float red[4][64];
  const int tiles_n = (p.B + 63) / 64, d0 = blockIdx.x / tiles_n * 32, c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int n = blockIdx.x % tiles_n * 64 + c;
  const long long count = (long long)p.D * p.B;
  const long long id = n < p.B ? p.targets[n] : -1;
  const bool real = id >= 0 && id < p.V;
  float fix = 0.0f;
  if (n < p.B) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i * 4 + r;
      if (d >= p.D) break;
      const long long at = (long long)d * p.B + n;
      float sum = 0.0f;
#pragma unroll 4
      for (int s = 0; s < p.slices; ++s) sum += p.part[s * count + at];
      const float x = to_f32(static_cast<const ST*>(p.x)[at]);
      sum *= p.scale;
      static_cast<ST*>(p.g)[at] = cvt<ST>(real ? dact_t<ACT>(x) * sum : 0.0f);
      if (p.fixes && real) {
        const float f = act_t<ACT>(x);
        fix += sum * (f - to_f32(cvt<ST>(f)));
      }
    }
  }
  if (!p.fixes) return;
  red[r][c] = fix;
  __syncthreads();
  if (r == 0 && n < p.B) p.fixes[(long long)(d0 / 32) * p.B + n] = red[0][c] + red[1][c] + red[2][c] + red[3][c];
}

// loss -= the fixes, in order; 16 columns a workgroup, 16 threads each
__global__ void __launch_bounds__(256) token_fix_kernel(const float* fixes, int rows, int B, float* loss) {
  __shared__ float red[16][16];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
  float sum = 0.0f;
  if (n < B)
    for (int i = g; i < rows; i += 16) sum += fixes[(long long)i * B + n];
  red[g][c] = sum;
  __syncthreads();
  if (g != 0 || n >= B) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += red[i][c];
  loss[n] -= sum;
}

// ------------------------------------------------------------------ errors
// Kept exponentials into errors, in place (fp32: into three terms).  Eight of a row a thread;
// its columns up to Vp and rows up to Bk, zeros past the ends and in padded rows.
struct Errors {
  int V, B, Vp, Bk, unit;
  const void* kept;   // [Bk][Vp]
  unsigned short* et;
  const float2* part;
  const float2* norm;
  const float* loss;
  const long long* targets;
  float scale;
};
template <typename OT, int TERMS>
__global__ void __launch_bounds__(256) token_errors_kernel(const Errors p) {
  const int per = p.Vp / 8;
  const unsigned at = blockIdx.x * 256u + threadIdx.x, n = at / (unsigned)per;
  const int v = (int)(at - n * (unsigned)per) * 8;
  if (n >= (unsigned)p.Bk) return;
  const long long place = (long long)n * p.Vp + v;
  const long long id = n < (unsigned)p.B ? p.targets[n] : -1;
  float e[8] = {};
  if (id >= 0 && id < p.V && v < p.V) {
    const float2 norm = p.norm[n];
    const float part = p.part[(long long)(v / p.unit) * p.B + n].x;
    const float share = -p.scale * norm.y * (part == -__builtin_inff() ? 0.0f : expf(part - norm.x));
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
      const float own = -expm1f(-p.loss[n]) * p.scale;  // 1 - p without its cancellation
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

template <typename ST, typename OT, int TERMS, int ACT>
hipError_t run(const TokenProblem& p, int storage, hipStream_t s) {
  const bool update = p.g != nullptr;
  Plan o;
  if (!make_plan(p.V, p.D, p.B, storage, p.act, update, o)) return hipErrorInvalidValue;
  unsigned char* ws = p.workspace;
  auto at = [&](long long offset) { return reinterpret_cast<unsigned short*>(ws + offset); };
  const States st{p.D, p.B, p.V, o.Dp, o.Bk, p.x, p.targets, update ? at(o.f) : nullptr, at(o.ft)};
  const unsigned state_tiles = (unsigned)((o.Dp + 63LL) / 64 * ((o.Bk + 63LL) / 64));
  constexpr bool inexact = TERMS == 1 && ACT != ACT_IDENTITY && ACT != ACT_RELU;
  if (inexact && !update) hipLaunchKernelGGL((token_states_kernel<ST, OT, inexact ? 2 : TERMS, ACT>), dim3(state_tiles), dim3(256), 0, s, st);
  else hipLaunchKernelGGL((token_states_kernel<ST, OT, TERMS, ACT>), dim3(state_tiles), dim3(256), 0, s, st);

  hipError_t e = hipGetLastError();
  auto rows_of = [&](int first) { return std::min(o.rows, p.V - first); };
  // the piece's rows of W, as an operand of the products
  auto weights = [&](int first, TokenGemm& q, bool lay) {
    const int rows = rows_of(first), padded = (rows + 31) / 32 * 32;
    const ST* w = static_cast<const ST*>(p.w) + (long long)first * p.D;
    if (!o.copy) {
      q.a = w; q.lda = p.D; q.a_bytes = (long long)rows * p.D * 2; q.a_term = 0;
      return;
    }
    if (lay) {
      const Rows r{rows, padded, p.D, o.Dp, w, at(o.ws)};
      const long long fours = (long long)padded * o.Dp / 4;
      hipLaunchKernelGGL((token_rows_kernel<ST, OT, TERMS>), dim3((unsigned)((fours + 255) / 256)), dim3(256), 0, s, r);
      if (e == hipSuccess) e = hipGetLastError();
    }
    q.a = at(o.ws); q.lda = o.Dp;
    q.a_term = (unsigned)(padded * o.Dp * 2);
    q.a_bytes = (long long)TERMS * padded * o.Dp * 2;
  };
  auto logits = [&](int first, bool lay) {
    TokenGemm q{};
    weights(first, q, lay);
    q.M = rows_of(first); q.N = p.B; q.K = o.copy ? o.Dp : p.D;
    q.b = at(o.ft); q.ldb = o.Dp; q.b_term = (unsigned)(p.B * o.Dp * 2); q.b_bytes = (long long)(o.two ? 2 : TERMS) * p.B * o.Dp * 2;
    q.targets = p.targets; q.first = first; q.V = p.V;
    q.target_logit = reinterpret_cast<float*>(ws + o.logit);
    return q;
  };
  float2* part = reinterpret_cast<float2*>(ws + o.stats);
  for (int first = 0; first < p.V && e == hipSuccess; first += o.rows) {
    TokenGemm q = logits(first, true);
    if (e != hipSuccess) return e;
    q.out = part + (long long)(first / o.unit) * p.B;
    if (o.keep) {
      q.kept = ws + o.kept; q.out_ld = o.Vp; q.out_rows = o.Bk;
      e = launch_token_keep(q, storage, o.tile, s);
    } else {
      e = launch_token_stats(q, storage, o.tile, o.two, s);
    }
  }
  if (e != hipSuccess) return e;
  const Columns c{p.B, p.V, (p.V + o.unit - 1) / o.unit, part, reinterpret_cast<const float*>(ws + o.logit), p.targets, p.loss,
                  reinterpret_cast<float2*>(ws + o.norm)};
  hipLaunchKernelGGL(token_columns_kernel, dim3((unsigned)((p.B + 15) / 16)), dim3(1024), 0, s, c);
  e = hipGetLastError();
  if (!update || e != hipSuccess) return e;

  // fp16: errors below its smallest normal number matter (1 / V), so they are kept times 2^10
  const float scale = storage == DT_F16 ? 1024.0f : 1.0f;
  for (int first = 0; first < p.V; first += o.rows) {
    const int rows = rows_of(first), Vp = (rows + 31) / 32 * 32;
    if (o.keep) {
      const Errors er{p.V, p.B, Vp, o.Bk, o.unit, ws + o.kept, at(o.et), part, reinterpret_cast<const float2*>(ws + o.norm),
                      p.loss, p.targets, scale};
      const long long eights = (long long)o.Bk * Vp / 8;
      hipLaunchKernelGGL((token_errors_kernel<OT, TERMS>), dim3((unsigned)((eights + 255) / 256)), dim3(256), 0, s, er);
      e = hipGetLastError();
    } else {
      TokenGemm q = logits(first, o.rows < p.V);  // (one piece: its rows are laid out already)
      if (e != hipSuccess) return e;
      q.stats = reinterpret_cast<const float2*>(ws + o.norm);
      q.out = at(o.et); q.out_ld = Vp; q.out_rows = o.Bk; q.out_term = (long long)o.Bk * Vp; q.scal = scale;
      e = launch_token_error(q, storage, o.tile, s);
    }
    if (e != hipSuccess) return e;
    TokenGemm g{};
    weights(first, g, false);
    g.M = p.D; g.N = p.B; g.K = Vp;
    g.b = at(o.et); g.ldb = Vp; g.b_term = (unsigned)((long long)o.Bk * Vp * 2); g.b_bytes = (long long)TERMS * o.Bk * Vp * 2;
    g.slices = o.slices; g.out = ws + o.part; g.add = first > 0;
    e = launch_token_grad(g, storage, o.grad_tile, s);
    if (e != hipSuccess) return e;
    TokenGemm u{};
    u.a = at(o.et); u.lda = Vp; u.a_term = g.b_term; u.a_bytes = g.b_bytes;
    u.b = at(o.f); u.ldb = o.Bk; u.b_term = (unsigned)(p.D * o.Bk * 2); u.b_bytes = (long long)TERMS * p.D * o.Bk * 2;
    u.M = rows; u.N = p.D; u.K = o.Bk;
    u.out = static_cast<ST*>(p.w) + (long long)first * p.D;
    u.vec = p.D % 4 == 0 && reinterpret_cast<uintptr_t>(p.w) % (4 * sizeof(ST)) == 0;
    u.scal = p.alpha / scale;
    e = launch_token_weight(u, storage, s);
    if (e != hipSuccess) return e;
  }
  float* fixes = o.fix ? reinterpret_cast<float*>(ws + o.fixes) : nullptr;
  const Grad gr{p.D, p.B, p.V, o.slices, reinterpret_cast<const float*>(ws + o.part), p.x, p.targets, p.g, 1.0f / scale, fixes};
  const int bands = (p.D + 31) / 32;
  hipLaunchKernelGGL((token_gradient_kernel<ST, ACT>), dim3((unsigned)((long long)bands * ((p.B + 63) / 64))), dim3(256), 0, s, gr);
  e = hipGetLastError();
  if (!fixes || e != hipSuccess) return e;
  hipLaunchKernelGGL(token_fix_kernel, dim3((unsigned)((p.B + 15) / 16)), dim3(256), 0, s, fixes, bands, p.B, p.loss);
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
  Plan o;
  return make_plan(V, D, B, storage, act, update, o) ? o.bytes : 0;
}

hipError_t launch_token(const TokenProblem& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return by_act<float, bf16, 3>(p, storage, s);
  return storage == DT_F16 ? by_act<f16, f16, 1>(p, storage, s) : by_act<bf16, bf16, 1>(p, storage, s);
}

}  // namespace ipc
