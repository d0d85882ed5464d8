// ipc_token_gemm.h - the matrix products of a softmax over tokens (gfx950).
//
//   TOKEN_STATS   Z[v][n] = sum_d W[v][d] F[d][n], of which only each tile's largest value and
//                 sum of exponentials a column are kept, and the target's logit
//   TOKEN_KEEP    that, and the exponentials, as KEPT[n][v] relative to their wave's largest
//   TOKEN_ERROR   the same products again; e = onehot - softmax(Z), rounded to the operand
//                 type and stored transposed, ET[n][v]
//   TOKEN_ONE     a vocabulary within one tile: losses and errors (as many terms as f(X) has; none where
//                 the output has no rows) at once
//   TOKEN_GRAD    P[d][n] = sum_v W[v][d] e[v][n]     (a slice of the vocabulary a workgroup)
//   TOKEN_STATE   that of a whole vocabulary, times f'(X): the state's gradient
//   TOKEN_WEIGHT  W[v][d] += alpha sum_n e[v][n] F[d][n]
//
// v_mfma_f32_32x32x16 tiles in the pipeline of ipc_ckpt_gemm.h: three to eight stages of 32 k filled by
// LDS-DMA loads, one barrier a stage, loads and the next fragments' reads between the
// products.  B is k-contiguous in every product (F^T, ET, F lie as that asks); A is for
// the first three (W), and k-rows read transposed for the others (W, ET), so that one
// copy of W and one of the errors serve both products they appear in.
//
// fp32 tensors: every operand is the sum of three bf16 terms (24 bits, the type's own), and a
// product the six term products above 2^-24 of it (2^-22 with f(X), whose terms are cut off), smallest first, from one stage that holds
// all terms.  Six times the 16-bit work, but the fp32 matrix instruction takes sixteen.
//
// What they reach (fp16, 128000 words, 2048 features, 2048 samples, 1.07 PFLOP each; a library's
// products of these sizes 804, 1369 and 804 us): TOKEN_KEEP 1070 us, TOKEN_GRAD 890, TOKEN_WEIGHT 1050.
// The main loop of a 256 x 256 tile runs at 1.17 PFLOP/s, 0.92 us a stage; beside it stand
// 9 us a tile of first loads and epilogue, which the LDS that a tile fills leaves no second
// workgroup to cover (256 x 128 tiles of three stages, two a CU: TOKEN_WEIGHT 1130-1170).  Matrix
// units are busy 63, 81 and 66 % of the CUs' cycles, and power holds them: over zeros the whole
// update takes 2650 us, not 3190.
//
// The accumulators of the first three lie with a column n a lane (and rows v in its
// registers), so that a column's maximum and sum are the lane's own business up to one
// exchange between the halves of a wave and one between waves; the others' with four
// consecutive columns a lane, for the shared tile epilogue.
#pragma once

#include "ipc_ckpt_gemm.h"
#include "ipc_token.h"
#include "ipc_token_plan.h"

namespace ipc {

enum { TOKEN_STATS = 0, TOKEN_KEEP = 1, TOKEN_ERROR = 2, TOKEN_GRAD = 3, TOKEN_WEIGHT = 4, TOKEN_ONE = 5, TOKEN_STATE = 6 };

// One product.  Rows start at multiples of 4 bytes; a and b with all their terms lie
// below 2^31 bytes.
struct TokenGemm {
  int M, N, K;                     // K: of one term; A k-contiguous: of any length, else a multiple of 32
  const void* a; long long lda;    // elements
  const void* b; long long ldb;
  long long a_bytes, b_bytes;      // buffers' ends (loads past them give 0)
  unsigned a_term, b_term;         // bytes from one term to the next
  int slices;                      // GRAD (and WEIGHT, see launch_token_tail): of the contraction, a stage of 32 each at least
  void* out;                       // STATS, KEEP: float2 [units][N]; ERROR: ET; GRAD: [slices][M][N] fp32; WEIGHT: W
  void* kept;                      // KEEP: exponentials times 2^15 in fp16 (fp32: in fp32), layout of ET
  long long out_ld, out_term;      // KEEP, ERROR: elements
  int out_rows;                    // of ET, N up to a multiple of 32
  int add;                         // GRAD: out holds sums already
  int vec;                         // WEIGHT: out allows 4-element accesses
  float scal;                      // WEIGHT: alpha; ERROR, ONE: the errors' scale; STATE: 1 / that
  const void* x; int act;          // STATE: of its type and layout, G's
  // STATS, KEEP, ERROR, ONE, STATE (targets and V)
  const long long* targets; int first, V;  // first: of the piece's rows
  float* target_logit;             // ONE: the losses
  const float* loss;               // ERROR
  const int* slot;                 // WEIGHT, or nullptr: of each row, its row in hot (-1: none), which the sum begins with
  const float* hot; int hot_ld;
  const float2* stats;             // ERROR: of each column, largest logit and 1 / sum of exp(z - largest)
};
// storage: 0 (three bf16 terms), 1, 2
// ways: terms of f(X), as many as token_ways has (ONE: 1, 2, 3 by storage); more than one: the exponentials kept in fp32
hipError_t launch_token_stats(const TokenGemm& p, int storage, int tile, int ways, hipStream_t s);
hipError_t launch_token_keep(const TokenGemm& p, int storage, int tile, int ways, hipStream_t s);
// M at most TOKEN_ONE_ROWS
hipError_t launch_token_one(const TokenGemm& p, int storage, int ways, hipStream_t s);
hipError_t launch_token_error(const TokenGemm& p, int storage, int tile, hipStream_t s);
// ways: terms of the errors, 1 or (16 bits) 2
hipError_t launch_token_grad(const TokenGemm& p, int storage, int tile, int ways, hipStream_t s);

// The state's gradient from its slices, G = f'(X) sum, zeros in padded columns, and what
// the loss is off by for f(X)'s rounding (fixes: [token_fix_rows][B], or nullptr).
struct TokenFinish {
  int D, B, V, slices, act;
  const float* part;  // [slices][D][B]
  const void* x;
  const long long* targets;
  void* g;
  float scale;
  float* fixes;
  int vec;            // x and g allow 4-element accesses
};
hipError_t launch_token_finish(const TokenFinish& p, int storage, hipStream_t s);
// W's update, and (f) the gradient's last step, which needs no more than that does: in one
// launch where both are small.
// terms: of both operands in 16-bit storage, 1, 2 (fp16) or 3 (bf16)
hipError_t launch_token_weight(const TokenGemm& p, const TokenFinish* f, int storage, int terms, hipStream_t s);
// The state's gradient (g, TOKEN_STATE; in 16 bits with two terms of the errors) from W's copy and W's update (u) in one launch.  u.slices > 1: u's
// contraction cut into as many, whose sums ([slices][M][N] at part) a second launch adds to W.
hipError_t launch_token_tail(const TokenGemm& g, const TokenGemm& u, float* part, int storage, hipStream_t s);

namespace token {

using namespace mx;

// a and b terms of the products of three terms each, smallest first (of two terms: the last three)
constexpr int PRODUCTS = 6, TERM_A[PRODUCTS] = {2, 1, 0, 1, 0, 0}, TERM_B[PRODUCTS] = {0, 1, 2, 0, 1, 0};

// (three terms of bf16 are fp32's, but where a launcher says otherwise)
template <typename OT, int TERMS>
using storage_of = typename std::conditional<TERMS == 3, float, OT>::type;

template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
  // the hardware exponential's relative error grows with |x| by 2^-24 a unit; 16-bit results do not see it
  if constexpr (EXACT) return expf(x);
  return __builtin_amdgcn_exp2f(x * 1.44269504f);
}

// The error at the target, 1 - p, without its cancellation.
__device__ __forceinline__ float target_error(float loss, float scale) { return -expm1f(-loss) * scale; }

// Workgroup `block` of `blocks` of a product.
// WT: the type of W, which TOKEN_WEIGHT writes, and of the state.
template <typename OT, int TERMS, int MODE, int WAYS, int BM, int BN, int WGM, int WGN, int ST, typename WT>
__device__ __forceinline__ void product_tile(const TokenGemm& p, unsigned char* smem, int block, int blocks) {
  using MF = Mfma32<OT>;
  typedef typename MF::operand V;
  constexpr bool MN = MODE == TOKEN_GRAD || MODE == TOKEN_WEIGHT || MODE == TOKEN_STATE, COLUMNS = !MN;
  constexpr int NW = WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, RM = WTM / 32, RN = WTN / 32;
  constexpr int RNC = RN / WAYS, BNC = BN / WAYS, WTC = WTN / WAYS;  // blocks and columns of different n
  constexpr bool SPLIT = TERMS == 3, FINE = SPLIT || ((MODE == TOKEN_KEEP || MODE == TOKEN_ONE) && WAYS > 1);  // FINE: kept in fp32
  constexpr int A_BYTES = BM * 64, B_BYTES = BN * 64, STAGE = TERMS * (A_BYTES + B_BYTES);
  static_assert(WAYS == 1 || (MODE != TOKEN_ERROR && MODE != TOKEN_WEIGHT && TERMS == 1 && RN % WAYS == 0), "terms of B");
  constexpr int IA = A_BYTES / 1024 / NW, IB = B_BYTES / 1024 / NW, LPS = TERMS * (IA + IB);  // LDS-DMA loads per wave and stage
  static_assert(IA * 1024 * NW == A_BYTES && IB * 1024 * NW == B_BYTES, "tile / waves");

  // consecutive tiles per XCD, in supertiles of 8 x 4 (as in mx_tile_kernel); slices outermost
  const int tn = (p.N + BNC - 1) / BNC, tm = (p.M + BM - 1) / BM;
  const int b = block, per = blocks >> 3, rem = blocks & 7, xcd = b & 7;
  const int t0 = xcd * per + (xcd < rem ? xcd : rem) + (b >> 3);
  const int slice = MODE == TOKEN_GRAD ? t0 / (tm * tn) : 0, t = t0 - slice * tm * tn;
  const int band = t / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, w8 = t - band * 8 * tn;
  const int cs = w8 / (rows * 4), cols = tn - cs * 4 < 4 ? tn - cs * 4 : 4, w2 = w8 - cs * rows * 4;
  const int m0 = (band * 8 + w2 / cols) * BM, n0 = (cs * 4 + w2 % cols) * BNC;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WGN, wn = w % WGN, lr = lane & 31, lk = lane >> 5;
  const int M = p.M, N = p.N, K = p.K, GS = (K + 31) / 32, tail = K - (GS - 1) * 32;
  // stages of this workgroup: begin .. end - 1
  const int begin = MODE == TOKEN_GRAD ? (int)((long long)GS * slice / p.slices) : 0;
  const int end = MODE == TOKEN_GRAD ? (int)((long long)GS * (slice + 1) / p.slices) : GS;
  const int G = end - begin;

  const Rsrc ga(p.a, (unsigned)p.a_bytes), gb(p.b, (unsigned)p.b_bytes);
  const i32x4 wa = rsrc_words(p.a, (unsigned)p.a_bytes), wb = rsrc_words(p.b, (unsigned)p.b_bytes);
  // byte offset of this lane's 16 bytes of LDS-DMA instruction q of an operand
  auto source = [&](bool mn, int q, int edge, int e0, int lim, long long ld) -> unsigned {
    const int slot = (q * NW + w) * 64 + lane;
    if (mn) {  // columns past the end: the last ones again or the next row's, never stored
      const int cpr = edge / 8, r = slot / cpr, c = (slot % cpr) ^ (edge == 64 ? (r & 2) << 1 : (r & 3) << 2);
      const int col = e0 + c * 8 < (int)ld ? e0 + c * 8 : (int)ld - 2;
      return (unsigned)(r * ld + col) * 2u;
    }
    const int r = slot >> 2, c = (slot & 3) ^ ((r >> 2) & 3), row = e0 + r < lim ? e0 + r : lim - 1;
    return (unsigned)(row * ld) * 2u + (unsigned)c * 16u;
  };
  // (WAYS > 1: the first of as many parts of a wave's columns holds B's leading term, the
  // others, the same columns, the next ones)
  auto source_ways = [&](int q) -> unsigned {
    const int slot = (q * NW + w) * 64 + lane, r = slot >> 2, c = (slot & 3) ^ ((r >> 2) & 3);
    const int of = r / WTN, at = r % WTN, n = n0 + of * WTC + at % WTC;
    return at / WTC * p.b_term + (unsigned)((n < N ? n : N - 1) * p.ldb) * 2u + (unsigned)c * 16u;
  };
  unsigned oa[IA], ob[IB];
#pragma unroll
  for (int q = 0; q < IA; ++q) oa[q] = source(MN, q, BM, m0, M, p.lda);
#pragma unroll
  for (int q = 0; q < IB; ++q) ob[q] = WAYS > 1 ? source_ways(q) : source(false, q, BN, n0, N, p.ldb);
  const unsigned step_a = MN ? (unsigned)p.lda * 64u : 64u;  // of a stage
  // load q of a stage: uniform offsets sa, sb; the terms of A, then those of B
  auto load = [&](int q, unsigned char* st, unsigned sa, unsigned sb) {
    const bool of_a = q < TERMS * IA;
    const int r = of_a ? q : q - TERMS * IA, each = of_a ? IA : IB, term = r / each, i = r % each;
    unsigned char* at = st + (of_a ? term * A_BYTES : TERMS * A_BYTES + term * B_BYTES) + (i * NW + w) * 1024;
    const unsigned v = of_a ? oa[of_a ? i : 0] : ob[of_a ? 0 : i], o = of_a ? sa + term * p.a_term : sb + term * p.b_term;
    if constexpr (MN) to_lds16_unseen(of_a ? wa : wb, at, v, o);
    else (of_a ? ga : gb).to_lds16(at, v, o);
  };
  // uniform offsets of stage kt (past the end: of the last, so that every step counts the
  // same).  A k-contiguous A may end inside a stage: that one comes first, and what it has
  // no k for is cleared.
  unsigned sa, sb;
  auto seek = [&](int kt) {
    const int g = begin + (kt < G ? kt : G - 1);
    const int k = MN || SPLIT ? g : g == 0 ? GS - 1 : g - 1;
    sa = (unsigned)k * step_a;
    sb = (unsigned)k * 64u;
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
  // TOKEN_WEIGHT: what the targets' rows begin with.  Asked for ahead of the operands, used
  // once those are on their way.
  constexpr bool HOT = MODE == TOKEN_WEIGHT && TERMS == 1;
  int slot[HOT ? RM : 1];
  if constexpr (HOT) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int m = m0 + wm * WTM + i * 32 + lr;
      slot[i] = p.slot && m < M ? p.slot[m] : -1;
    }
  }

  // fragments of 16 k (half s of a stage): row / column lr of a 32-wide block, k 8 lk .. + 7
  const int g4 = lane >> 4, li = lane & 15;
  const int tr_row = 8 * (g4 >> 1) + (li >> 2), tr_low = 2 * (g4 & 1) + ((li & 3) >> 1);
  auto straight = [&](const unsigned char* blk, int e, int s) -> V {
    return *reinterpret_cast<const V*>(blk + (e + lr) * 64 + ((((s * 2) | lk) ^ ((lr >> 2) & 3)) << 4));
  };
  auto turned = [&](const unsigned char* blk, int rowb, int e, int s) -> V {
    const int chunk = (((e >> 5) ^ (rowb == 128 ? li >> 3 : li >> 2)) << 2) | tr_low;
    const unsigned char* p0 = blk + (s * 16 + tr_row) * rowb + (chunk << 4) + (li & 1) * 8;
    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0));
    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0 + 4 * rowb));
    return __builtin_bit_cast(V, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  V fa[2][TERMS][RM], fb[2][TERMS][RN];
  // part r of a half stage's fragments
  auto fetch = [&](int r, const unsigned char* st, int s, int set) {
    const int term = r / (RM + RN), i = r % (RM + RN);
    if (i < RN) {
      fb[set][term][i < RN ? i : 0] = straight(st + TERMS * A_BYTES + term * B_BYTES, wn * WTN + i * 32, s);
    } else {
      const unsigned char* blk = st + term * A_BYTES;
      const int e = wm * WTM + (i - RN) * 32;
      if constexpr (MN) fa[set][term][i < RN ? 0 : i - RN] = turned(blk, BM * 2, e, s);
      else fa[set][term][i < RN ? 0 : i - RN] = straight(blk, e, s);
    }
  };

#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    seek(s);
#pragma unroll
    for (int q = 0; q < LPS; ++q) load(q, smem + s * STAGE, sa, sb);
  }
  if constexpr (HOT) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      if (slot[i] >= 0) {
        const float* row = p.hot + (long long)slot[i] * p.hot_ld;
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn * WTN + j * 32 + 8 * q + 4 * lk;
            const float4 v = *reinterpret_cast<const float4*>(row + (n < p.hot_ld ? n : 0));
            acc[i][j][4 * q] = v.x; acc[i][j][4 * q + 1] = v.y; acc[i][j][4 * q + 2] = v.z; acc[i][j][4 * q + 3] = v.w;
          }
      }
    }
    // (a wait that the compiler knows of: it would else wait for these loads in every step)
    __builtin_amdgcn_s_waitcnt(vm_wait<0>());
  }
  wait_loads<(ST - 2) * LPS>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (!SPLIT && !MN && tail < 32) {
    unsigned short* h = reinterpret_cast<unsigned short*>(smem);
    for (int i = tid; i < BM * 32; i += NW * 64)
      if (((i & 31) ^ (((i >> 7) & 3) << 3)) >= tail) h[i] = 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int r = 0; r < TERMS * (RM + RN); ++r) fetch(r, smem, 0, 0);

  // half a step: the products of set S; the fragments of the next 16 k (half S ^ 1 of
  // `next`) and half of a later stage's loads between them
  auto half = [&](auto SV, const unsigned char* next, unsigned char* fill) {
    constexpr int S = decltype(SV)::value, O = S ^ 1;
    constexpr int L0 = S == 0 ? 0 : (LPS + 1) / 2, L1 = S == 0 ? (LPS + 1) / 2 : LPS;
    constexpr int EACH = RM * RN, FIRST = TERMS == 3 ? 0 : TERMS == 2 ? 3 : 5, NM = (PRODUCTS - FIRST) * EACH, NR = TERMS * (RM + RN);
#pragma unroll
    for (int q = 0; q < NM; ++q) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * NM / NR == q) fetch(r, next, O, O);
#pragma unroll
      for (int l = L0; l < L1; ++l)
        if ((l - L0) * NM / (L1 - L0) == q) load(l, fill, sa, sb);
      const int i = q % EACH / RN, j = q % RN;
      const V a = fa[S][TERM_A[FIRST + q / EACH]][i], b = fb[S][TERM_B[FIRST + q / EACH]][j];
      acc[i][j] = COLUMNS ? MF::run(a, b, acc[i][j]) : MF::run(b, a, acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int at = 0;  // place of stage kt
#pragma unroll 1
  for (int kt = 0; kt < G; ++kt) {
    // stage kt + 1 of this wave has landed (later ones may be in flight), then everybody's;
    // everybody is done with stage kt - 1, whose place the last one loaded takes
    wait_loads<(ST - 3) * LPS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    seek(kt + ST - 1);
    unsigned char* here = smem + at * STAGE;
    unsigned char* fill = smem + (at == 0 ? ST - 1 : at - 1) * STAGE;
    at = at + 1 == ST ? 0 : at + 1;
    half(std::integral_constant<int, 0>{}, here, fill);
    half(std::integral_constant<int, 1>{}, smem + at * STAGE, fill);
  }
  wait_loads<0>();  // no load may land in the epilogue's LDS

  // Rows past the last.  (The limit is made anew each time: the compiler would keep a
  // mask of every row, thousands of scalar registers.)
  auto mask_rows = [&](int j, float with) {
    int left = M - m0 - wm * WTM - 4 * lk;
    asm("" : "+v"(left));
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int q = 0; q < 16; ++q)
        if (i * 32 + 8 * (q >> 2) + (q & 3) >= left) acc[i][j][q] = with;
  };
  // Block column j of the accumulators, columns n across the lanes, as rows n of a matrix with
  // v along its rows, through this wave's part of the LDS.  FORM 0: errors in the operand
  // type (fp32: three terms; ONE: as many as f(X) has); 1: exponentials in fp16 times 2^15; 2: in fp32.  Rows and
  // columns past the ends, up to the matrix's own, hold what the accumulators do there.
  auto store_columns = [&](auto form, int j) {
    constexpr int FORM = decltype(form)::value;
    typedef typename std::conditional<FORM == 2, float, unsigned short>::type U;
    constexpr int LD = WTM + (FORM == 2 ? 4 : 8), PARTS = FORM != 0 ? 1 : SPLIT ? 3 : WAYS, PER = 16 / sizeof(U);
    U* es = reinterpret_cast<U*>(smem) + w * 32 * LD;
    U* out = static_cast<U*>(FORM == 0 ? p.out : p.kept);
#pragma unroll
    for (int term = 0; term < PARTS; ++term) {
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; q += 4) {
          U h[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float v = acc[i][j][q + u];
            if constexpr (FORM == 0) {
              const OT o = cvt<OT>(v);
              h[u] = __builtin_bit_cast(unsigned short, o);
              if (PARTS > 1) acc[i][j][q + u] = v - to_f32(o);  // exact; NaN stays
            } else if constexpr (FORM == 1) {
              h[u] = __builtin_bit_cast(unsigned short, cvt<f16>(v * 32768.0f));
            } else {
              h[u] = v;
            }
          }
          typedef U U4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<U4*>(es + lr * LD + i * 32 + 2 * q + 4 * lk) = U4{h[0], h[1], h[2], h[3]};
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      constexpr int LPR = WTM / PER, RPP = 64 / LPR, PASSES = 32 / RPP;  // lanes a row, rows a pass
#pragma unroll
      for (int u = 0; u < PASSES; ++u) {
        const int r = u * RPP + lane / LPR, c = lane % LPR * PER;
        const uint4 v = *reinterpret_cast<const uint4*>(es + r * LD + c);
        const long long row = n0 + wn * WTC + j * 32 + r;
        const int col = m0 + wm * WTM + c;
        if (row < p.out_rows && col < p.out_ld) *reinterpret_cast<uint4*>(out + term * p.out_term + row * p.out_ld + col) = v;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };
  if constexpr (WAYS > 1) {
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < RNC; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) {  // (an infinite weight times the rest, of either sign, is no matter)
          float rest = acc[i][j + RNC][q];
          if constexpr (WAYS == 3) rest += acc[i][j + 2 * RNC][q];
          acc[i][j][q] += __builtin_isinf(acc[i][j][q]) ? 0.0f : rest;
        }
  }
  if constexpr (MODE == TOKEN_STATS || MODE == TOKEN_KEEP) {
    if constexpr (MODE == TOKEN_KEEP) __syncthreads();
    const int mw = m0 + wm * WTM;
#pragma unroll
    for (int j = 0; j < RNC; ++j) {
      const int n = n0 + wn * WTC + j * 32 + lr;
      if (m0 + BM > M) mask_rows(j, -__builtin_inff());
      // the target's place among this lane's rows of the column
      const long long to = (n < N ? p.targets[n] : -1) - p.first - mw;
      const int own = (int)to - 4 * lk;
      const bool hit = to >= 0 && to < WTM && to < M - mw && (own & 4) == 0;
      if (__any(hit)) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int q = 0; q < 16; ++q) z = own == i * 32 + 8 * (q >> 2) + (q & 3) ? acc[i][j][q] : z;
        if (hit) p.target_logit[n] = z;
      }
      float top = acc[0][j][0], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) top = __builtin_fmaxf(top, acc[i][j][q]);
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -__builtin_inff() ? 0.0f : top;  // (a column of -inf: no sum, and no NaN)
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          acc[i][j][q] = exp_of<FINE>(acc[i][j][q] - from);
          sum += acc[i][j][q];
        }
      sum += __shfl_xor(sum, 32);
      if (lk == 0 && n < N && mw < M) static_cast<float2*>(p.out)[(long long)(mw / WTM) * N + n] = make_float2(top, sum);
      if constexpr (MODE == TOKEN_KEEP) store_columns(std::integral_constant<int, FINE ? 2 : 1>{}, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if constexpr (MODE == TOKEN_ONE) {
    // of each column the largest logit and sum of a wave's rows, and its target's logit
    float2* stat = reinterpret_cast<float2*>(smem + NW * 32 * (WTM + 8) * 2);  // [WGM][BNC]
    float* own_logit = reinterpret_cast<float*>(stat + WGM * BNC);
    __syncthreads();
    const int mw = m0 + wm * WTM;
#pragma unroll
    for (int j = 0; j < RNC; ++j) {
      const int c = wn * WTC + j * 32 + lr, n = n0 + c;
      if (m0 + BM > M) mask_rows(j, -__builtin_inff());
      const long long to = (n < N ? p.targets[n] : -1) - mw;
      const int own = (int)to - 4 * lk;
      if (to >= 0 && to < WTM && to < M - mw && (own & 4) == 0) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int q = 0; q < 16; ++q) z = own == i * 32 + 8 * (q >> 2) + (q & 3) ? acc[i][j][q] : z;
        own_logit[c] = z;
      }
      float top = acc[0][j][0], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) top = __builtin_fmaxf(top, acc[i][j][q]);
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          acc[i][j][q] = exp_of<true>(acc[i][j][q] - from);
          sum += acc[i][j][q];
        }
      sum += __shfl_xor(sum, 32);
      if (lk == 0) stat[wm * BNC + c] = make_float2(top, sum);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RNC; ++j) {
      const int c = wn * WTC + j * 32 + lr, n = n0 + c;
      const long long id = n < N ? p.targets[n] : -1, to = id - mw;
      const bool real = id >= 0 && id < p.V;
      const int own = (int)to - 4 * lk;
      const bool hit = real && to >= 0 && to < WTM && (own & 4) == 0;
      float top = stat[c].x, sum = 0.0f;
#pragma unroll
      for (int i = 1; i < WGM; ++i) top = __builtin_fmaxf(top, stat[i * BNC + c].x);
      float of_wave = 0.0f;
#pragma unroll
      for (int i = 0; i < WGM; ++i) {
        const float2 part = stat[i * BNC + c];
        const float by = part.x == -__builtin_inff() ? 0.0f : expf(part.x - top);
        sum += part.x == -__builtin_inff() ? part.y : part.y * by;
        if (i == wm) of_wave = by;
      }
      const float loss = real ? logf(sum) + (top - own_logit[c]) : 0.0f, share = -of_wave / sum * p.scal;
      if (wm == 0 && lk == 0 && n < N) p.target_logit[n] = loss;
      const float at_target = target_error(loss, p.scal);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float v = real ? acc[i][j][q] * share : 0.0f;
          acc[i][j][q] = hit && own == i * 32 + 8 * (q >> 2) + (q & 3) ? at_target : v;
        }
      if (m0 + BM > M) mask_rows(j, 0.0f);
      store_columns(std::integral_constant<int, 0>{}, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if constexpr (MODE == TOKEN_ERROR) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RN; ++j) {
      const int n = n0 + wn * WTN + j * 32 + lr, mw = m0 + wm * WTM;
      const long long id = n < N ? p.targets[n] : -1, to = id - p.first - mw;
      const bool real = id >= 0 && id < p.V;
      const int own = (int)to - 4 * lk;
      const bool hit = real && to >= 0 && to < WTM && (own & 4) == 0;
      const float2 st = real ? p.stats[n] : make_float2(0.0f, 0.0f);
      const float share = -st.y * p.scal, at_target = real ? target_error(p.loss[n], p.scal) : 0.0f;
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[i][j][q] = real ? exp_of<SPLIT>(acc[i][j][q] - st.x) * share : 0.0f;
      if (__any(hit)) {
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int q = 0; q < 16; ++q)
            acc[i][j][q] = hit && own == i * 32 + 8 * (q >> 2) + (q & 3) ? at_target : acc[i][j][q];
      }
      if (m0 + BM > M) mask_rows(j, 0.0f);
      store_columns(std::integral_constant<int, 0>{}, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else if constexpr (MODE == TOKEN_STATE) {
    static_assert(RM == 1 && RNC == 1, "a block a wave");
    __syncthreads();
    float* es = reinterpret_cast<float*>(smem) + w * 32 * 36;
#pragma unroll
    for (int q = 0; q < 16; q += 4)
      *reinterpret_cast<float4*>(es + lr * 36 + 2 * q + 4 * lk) = make_float4(acc[0][0][q], acc[0][0][q + 1], acc[0][0][q + 2], acc[0][0][q + 3]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int n = n0 + wn * WTC + lr;
    const long long id = n < N ? p.targets[n] : -1;
    const bool real = id >= 0 && id < p.V;
#pragma unroll 1
    for (int r = lk; r < 32; r += 2) {
      const int d = m0 + wm * WTM + r;
      if (d >= M || n >= N) continue;
      const long long here = (long long)d * N + n;
      const float v = act_df(p.act, to_f32(static_cast<const WT*>(p.x)[here])) * (es[r * 36 + lr] * p.scal);
      static_cast<WT*>(p.out)[here] = cvt<WT>(real ? v : 0.0f);
    }
  } else {
    typedef typename std::conditional<MODE == TOKEN_GRAD, float, WT>::type TT;
    MxProblem e{};
    e.M = M; e.N = N; e.scal = MODE == TOKEN_GRAD ? 1.0f : p.scal;
    e.out = MODE == TOKEN_GRAD ? static_cast<float*>(p.out) + (long long)slice * M * N : p.out;
    float* es = reinterpret_cast<float*>(smem) + w * 32 * (WTC + 4);
    const int mw = m0 + wm * WTM, nw = n0 + wn * WTC;
    f32x16 sum[RM][RNC];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < RNC; ++j) sum[i][j] = acc[i][j];
    if (MODE == TOKEN_GRAD && !p.add) tile_epilogue<TT, KIND_FWD, ACT_IDENTITY, true, RM, RNC>(e, sum, es, mw, nw);
    else if (MODE == TOKEN_GRAD || p.vec) tile_epilogue<TT, KIND_WEIGHT, ACT_IDENTITY, true, RM, RNC>(e, sum, es, mw, nw);
    else tile_epilogue<TT, KIND_WEIGHT, ACT_IDENTITY, false, RM, RNC>(e, sum, es, mw, nw);
  }
}

template <typename OT, int TERMS, int MODE, int WAYS, int BM, int BN, int WGM, int WGN, int ST, typename WT>
__global__ void __launch_bounds__(WGM * WGN * 64) token_gemm_kernel(const TokenGemm p) {
  extern __shared__ __align__(16) unsigned char smem[];
  product_tile<OT, TERMS, MODE, WAYS, BM, BN, WGM, WGN, ST, WT>(p, smem, blockIdx.x, gridDim.x);
}

template <int TERMS, int MODE, int WAYS, int BM, int BN, int WGM, int WGN, int ST>
constexpr int tile_lds() {
  constexpr int NW = WGM * WGN, ring = ST * TERMS * (BM + BN) * 64;
  constexpr int epi = MODE == TOKEN_STATS ? 0
                      : MODE == TOKEN_STATE ? NW * 32 * 36 * 4
                      : MODE == TOKEN_ONE ? NW * 32 * (BM / WGM + 8) * 2 + (WGM * 8 + 4) * (BN / WAYS)
                      : MODE == TOKEN_ERROR || (MODE == TOKEN_KEEP && TERMS == 1 && WAYS == 1) ? NW * 32 * (BM / WGM + 8) * 2
                      : MODE == TOKEN_KEEP ? NW * 32 * (BM / WGM + 4) * 4 : NW * 32 * (BN / WGN + 4) * 4;
  return epi > ring ? epi : ring;
}

template <typename OT, int TERMS, int MODE, int WAYS, int BM, int BN, int WGM, int WGN, int ST = 4, typename WT = storage_of<OT, TERMS>>
hipError_t run_tile(const TokenGemm& p, hipStream_t s) {
  constexpr int smem = tile_lds<TERMS, MODE, WAYS, BM, BN, WGM, WGN, ST>();
  static_assert(smem <= 160 * 1024, "LDS");
  const void* fn = reinterpret_cast<const void*>(&token_gemm_kernel<OT, TERMS, MODE, WAYS, BM, BN, WGM, WGN, ST, WT>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  constexpr int BNC = BN / WAYS;
  const long long tiles = ((p.M + BM - 1LL) / BM) * ((p.N + BNC - 1LL) / BNC) * (MODE == TOKEN_GRAD ? p.slices : 1);
  TokenGemm q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)tiles), dim3(WGM * WGN * 64), args, smem, s);
}

// 64 x 64 tiles: as many stages as leave two workgroups a CU (fp32: one, or two of three stages
// where there are more workgroups than CUs), since a step of few workgroups is as long as
// a load takes over the stages in flight.
template <typename OT, int TERMS, int MODE, int WAYS, int WGM, int WGN, typename WT = storage_of<OT, TERMS>>
hipError_t run_narrow(const TokenGemm& p, hipStream_t s) {
  constexpr int BNC = 64 / WAYS;
  const long long tiles = ((p.M + 63LL) / 64) * ((p.N + BNC - 1LL) / BNC) * (MODE == TOKEN_GRAD ? p.slices : 1);
  if constexpr (TERMS == 3) {
    if (tiles > 256) return run_tile<OT, TERMS, MODE, WAYS, 64, 64, WGM, WGN, 3, WT>(p, s);
  }
  return run_tile<OT, TERMS, MODE, WAYS, 64, 64, WGM, WGN, TERMS == 3 ? 6 : 8 / TERMS, WT>(p, s);
}

}  // namespace token
}  // namespace ipc
