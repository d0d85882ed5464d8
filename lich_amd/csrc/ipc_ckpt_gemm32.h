// ipc_ckpt_gemm32.h - the backward pass of a state kept in 8 bits on fp32 operands (gfx950).
//
//   CKPT_GRAD     G[m][n] = f'(X)[m][n] sum_k A[k][m] B[k][n]   A = W_lower, B = E_lower
//   CKPT_WEIGHT   W[m][n] += alpha sum_k A[m][k] f(X)[n][k]      A = E
//
// v_mfma_f32_32x32x2_f32: 64 cycles for 2 k of a 32 x 32 block, so that one wave a
// SIMD keeps the matrix units busy if it never waits.  Stages of 16 k (eight
// products of a block) go to LDS by LDS-DMA loads, four stages a ring, and a
// stage's fragments are read between the products of the one before.
//
//   * The order of the contraction is free: lane half lk of product j takes k = 8 lk + j
//     of k-contiguous rows (two 16-byte reads a fragment, the 8 codes of X in one of 8
//     bytes) and k = 2 j + lk of k-rows (4-byte reads: nothing to transpose).
//   * Loads take 16 bytes a lane from any multiple of 4 bytes (rows of any length);
//     where a row ends inside one they bring the next row's first values, which no
//     stored output reads.
//   * The operands' last 1 .. 16 k come first, as stage 0, whose offsets are the
//     lanes' own; loads past the operand's end give 0; what the stage has no k
//     for is cleared in LDS before anything is read.  The loop knows whole stages inside
//     the operands only.
//   * CODES32 keeps X in 8 bits up to the fragment and evaluates f there, in every row
//     of tiles; WIDE32 reads f(X) widened once into a workspace.
//   * WK = 4: four waves share a 32 x 32 tile, each a ring of its own and every fourth
//     stage, no barrier between them; their sums are added in wave order.
//
// LDS: chunk c (4 floats) of k-contiguous row r at c ^ ((r >> 2) & 3) (16 rows of a
// fragment read touch every bank once); column c of k-row r at c ^ 32 (r & 1) (the two
// k of a product from different banks).
//
// MI355X: 4096 x 4096, contraction 1024: gradient 265 us, weight update 258 (133
// TFLOP/s; a plain fp32 matrix product of 8192^3 runs at 154) and 8 for widening; from
// codes 280 (relu), 457 (silu).
#pragma once

#include "ipc_ckpt_gemm.h"

namespace ipc {
namespace mx {

// 4 bytes a lane, as to_lds16_unseen.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds4_unseen(i32x4 rsrc, unsigned char* lds, unsigned v, unsigned s) {
  const unsigned at = (unsigned)(unsigned long long)(lds_void*)lds;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(at), "v"(v), "s"(rsrc), "s"(s)
               : "memory", "m0");
}
#pragma clang diagnostic pop

constexpr int K32 = 16;  // k of a stage

enum { ROWS32, CODES32, WIDE32 };  // CKPT_GRAD; CKPT_WEIGHT from codes; from f(X) in fp32

template <int SRC, int BM, int BN, int GW>
constexpr int stage32_bytes() { return BM * K32 * 4 + (SRC == CODES32 ? BN * K32 + GW * 256 : BN * K32 * 4); }
template <int SRC, int BM, int BN, int WGM, int WGN, int WK>
constexpr int smem32() {
  constexpr int st = STAGES * WK * stage32_bytes<SRC, BM, BN, WGM * WGN>();
  constexpr int epi = WK == 1 ? WGM * WGN * 32 * (BN / WGN + 4) * 4 : WK * BM * (BN + 4) * 4;
  return st > epi ? st : epi;
}

template <int SRC, int ACT, int BM, int BN, int WGM, int WGN, int WK>
__global__ void __launch_bounds__(WGM * WGN * WK * 64) ckpt_gemm32_kernel(const CkptProblem p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr bool MN = SRC == ROWS32, CODES = SRC == CODES32;
  constexpr int GW = WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, RM = WTM / 32, RN = WTN / 32;
  constexpr int A_BYTES = BM * K32 * 4, STAGE = stage32_bytes<SRC, BM, BN, GW>(), S_AT = A_BYTES + BN * K32;
  constexpr int IA = A_BYTES / 1024 / GW, IB = CODES ? BN * K32 / 256 / GW : BN * K32 * 4 / 1024 / GW;
  constexpr int IS = CODES ? 1 : 0, LPS = IA + IB + IS;  // a wave's loads of a stage
  static_assert(IA * 1024 * GW == A_BYTES && IB * (CODES ? 256 : 1024) * GW == BN * K32 * (CODES ? 1 : 4), "tile / waves");
  static_assert(GW == 1 || WK == 1, "the groups of a tile share no barrier");

  // consecutive tiles per XCD, in supertiles of 8 x 4 (as in mx_tile_kernel)
  const int tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
  const int b = blockIdx.x, per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = b & 7;
  const int t = xcd * per + (xcd < rem ? xcd : rem) + (b >> 3);
  const int band = t / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, w8 = t - band * 8 * tn;
  const int cs = w8 / (rows * 4), cols = tn - cs * 4 < 4 ? tn - cs * 4 : 4, w2 = w8 - cs * rows * 4;
  const int m0 = (band * 8 + w2 / cols) * BM, n0 = (cs * 4 + w2 % cols) * BN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w = wave % GW, wk = wave / GW;  // wave of its group, group
  const int wm = w / WGN, wn = w % WGN, lr = lane & 31, lk = lane >> 5;
  const int M = p.M, N = p.N, K = p.K, G = (K + K32 - 1) / K32, tail = K - (G - 1) * K32;
  const int H = wk < G ? (G - wk + WK - 1) / WK : 0;  // steps of a group: stages wk, wk + WK, ...
  unsigned char* ring = smem + wk * STAGES * STAGE;
  auto place = [&](int kt) -> unsigned char* { return ring + (kt & (STAGES - 1)) * STAGE; };
  // first k of a stage; past the end: of the last, so that every step counts the same
  auto k_of = [&](int g) { return g == 0 || G == 1 ? K - tail : ((g < G ? g : G - 1) - 1) * K32; };

  // (the host: operands below 2^31 bytes)
  const long long lda = p.lda, ldb = p.ldb;
  const i32x4 ra = rsrc_words(p.a, (unsigned)((MN ? (long long)K : (long long)M) * lda * 4));
  const i32x4 rb = CODES ? rsrc_words(p.x, (unsigned)((long long)N * p.x_row)) : rsrc_words(p.b, (unsigned)((MN ? (long long)K : (long long)N) * ldb * 4));
  const i32x4 rs = rsrc_words(p.xs, (unsigned)mx_groups(K) * (unsigned)N * 4u);
  // byte offset of this lane's 16 bytes of load q of an fp32 operand, `have` k-rows in the stage
  auto source = [&](int q, int edge, int e0, int lim, long long ld, int have) -> unsigned {
    const int at = ((q * GW + w) * 64 + lane) * 4;
    if constexpr (MN) {  // columns past the end: the last ones again or the next row's, never stored
      const int r = at / edge, c = e0 + ((at % edge) ^ (edge > 32 ? (r & 1) << 5 : 0));
      return (unsigned)((r < have ? r : have - 1) * ld + (c < lim ? c : lim - 1)) * 4u;
    } else {
      const int r = at / K32, k = (at % K32) ^ (((r >> 2) & 3) << 2), row = e0 + r < lim ? e0 + r : lim - 1;
      return (unsigned)(row * ld + k) * 4u;
    }
  };
  unsigned oa[IA], ob[IB], os = 0;
#pragma unroll
  for (int q = 0; q < IA; ++q) oa[q] = source(q, BM, m0, M, lda, K32);
#pragma unroll
  for (int q = 0; q < IB; ++q) {
    if constexpr (CODES) {  // 4 codes of a row; rows are padded to 32
      const int at = (q * GW + w) * 64 + lane, row = n0 + (at >> 2) < N ? n0 + (at >> 2) : N - 1;
      ob[q] = (unsigned)row * (unsigned)p.x_row + (unsigned)(at & 3) * 4u;
    } else {
      ob[q] = source(q, BN, n0, N, ldb, K32);
    }
  }
  if constexpr (CODES) {
    const int row = n0 + wn * WTN + (lane & (WTN < 64 ? WTN - 1 : 63));
    os = (unsigned)(row < N ? row : N - 1) * 4u;
  }
  const unsigned step_a = MN ? (unsigned)lda * 4u : 4u, step_b = MN ? (unsigned)ldb * 4u : CODES ? 1u : 4u;
  // load q of the stage of first k `k`, from offsets va, vb, vs and the uniform sa, sb
  auto load = [&](int q, int k, unsigned char* st, unsigned va, unsigned sa, unsigned vb, unsigned sb, unsigned vs) {
    if (q < IA) to_lds16_unseen(ra, st + (q * GW + w) * 1024, va, sa);
    else if (q >= IA + IB) to_lds4_unseen(rs, st + S_AT + w * 256, vs, (unsigned)(k >> 7) * (unsigned)N * 4u);
    else if (CODES) to_lds4_unseen(rb, st + A_BYTES + ((q - IA) * GW + w) * 256, vb, sb);
    else to_lds16_unseen(rb, st + A_BYTES + ((q - IA) * GW + w) * 1024, vb, sb);
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  struct Fragments {
    float a[RM][8], b[CODES ? 1 : RN][8];
    uint2 codes[CODES ? RN : 1];
    unsigned unit[CODES ? RN : 1];
  };
  // part r of a stage's fragments: one LDS read
  constexpr int PER = MN ? 8 : 2, READS = PER * (RM + RN);
  auto fetch = [&](int r, const unsigned char* st, Fragments& f) {
    const int blk = r / PER, h = r % PER, i = blk < RM ? blk : 0, j = blk < RM ? 0 : blk - RM;
    if constexpr (MN) {
      const int edge = blk < RM ? BM : BN, e = blk < RM ? wm * WTM + i * 32 : wn * WTN + j * 32;
      const float* at = reinterpret_cast<const float*>(blk < RM ? st : st + A_BYTES) + lk * edge +
                        ((e + lr) ^ (edge > 32 ? lk << 5 : 0));
      (blk < RM ? f.a[i] : f.b[j])[h] = at[2 * h * edge];
    } else if (blk < RM || !CODES) {
      const unsigned char* row = (blk < RM ? st + (wm * WTM + i * 32 + lr) * 64 : st + A_BYTES + (wn * WTN + j * 32 + lr) * 64);
      const float4 v = *reinterpret_cast<const float4*>(row + (((2 * lk + h) ^ ((lr >> 2) & 3)) << 4));
      float* o = (blk < RM ? f.a[i] : f.b[CODES ? 0 : j]) + 4 * h;
      o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    } else if (h == 0) {
      f.codes[CODES ? j : 0] = *reinterpret_cast<const uint2*>(st + A_BYTES + (wn * WTN + j * 32 + lr) * K32 + 8 * lk);
    } else {
      f.unit[CODES ? j : 0] = *reinterpret_cast<const unsigned*>(st + S_AT + w * 256 + (j * 32 + lr) * 4);
    }
  };

  // prologue: all stages of the ring but one.  The operands' last k are stage 0.
  const unsigned last_a = (unsigned)(K - tail) * step_a, last_b = (unsigned)(K - tail) * step_b;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    const int g = s * WK + wk;
    const bool first = g == 0 || G == 1;
    const unsigned k = (unsigned)k_of(g);
#pragma unroll
    for (int q = 0; q < LPS; ++q) {
      const bool of_a = q < IA, of_b = q >= IA && q < IA + IB;
      const int qb = of_b ? q - IA : 0;
      unsigned va = of_a ? oa[of_a ? q : 0] : 0u, vb = ob[qb];
      if (first) {
        if (of_a) va = (MN ? source(q, BM, m0, M, lda, tail) : va) + last_a;
        if (of_b) vb = (MN ? source(qb, BN, n0, N, ldb, tail) : vb) + last_b;
      }
      load(q, (int)k, place(s), va, first ? 0u : k * step_a, vb, first ? 0u : k * step_b, os);
    }
  }
  if (G == 1) {  // (no other stage: its loads take the operands' first values)
#pragma unroll
    for (int q = 0; q < IA; ++q) oa[q] = 0;
#pragma unroll
    for (int q = 0; q < IB; ++q) ob[q] = 0;
  }
  wait_loads<2 * LPS>();
  if constexpr (GW > 1) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (tail < K32) {  // clear what stage 0 has no k for
    if (wk == 0) {
      float* a = reinterpret_cast<float*>(ring);
      const int at = w * 64 + lane;
      if constexpr (MN) {
        float* o = reinterpret_cast<float*>(ring + A_BYTES);
        for (int i = tail * BM + at; i < K32 * BM; i += GW * 64) a[i] = 0.0f;
        for (int i = tail * BN + at; i < K32 * BN; i += GW * 64) o[i] = 0.0f;
      } else {
        for (int i = at; i < K32 * BM; i += GW * 64)
          if (((i & (K32 - 1)) ^ (((i >> 6) & 3) << 2)) >= tail) a[i] = 0.0f;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (GW > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  Fragments f0, f1;
#pragma unroll
  for (int r = 0; r < READS; ++r) fetch(r, place(0), f0);

  auto step = [&](int kt, Fragments& cur, Fragments& next) {
    // stage kt + 1 of this wave has landed (later ones may be in flight), then everybody's;
    // everybody is done with stage kt - 1, whose place the refill takes
    wait_loads<LPS>();
    if constexpr (GW > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int g = kt * WK + wk, k3 = G == 1 ? 0 : k_of(g + (STAGES - 1) * WK);
    unsigned char* fill = place(kt + STAGES - 1);
    const unsigned char* after = place(kt + 1);
    float x[RN][8];
    if constexpr (CODES) {
      const int shift = ((k_of(g) >> 5) & 3) * 8;
#pragma unroll
      for (int j = 0; j < RN; ++j) {
        const float unit = int8_scale((cur.unit[CODES ? j : 0] >> shift) & 255u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[j][i] = act_t<ACT>((float)sext8(i < 4 ? cur.codes[CODES ? j : 0].x : cur.codes[CODES ? j : 0].y, i & 3) * unit);
      }
    }
    constexpr int NP = 8 * RM * RN;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * NP / READS == q) fetch(r, after, next);
#pragma unroll
      for (int l = 0; l < LPS; ++l)
        if (l * NP / LPS == q)
          load(l, k3, fill, oa[l < IA ? l : 0], (unsigned)k3 * step_a, ob[l >= IA && l - IA < IB ? l - IA : 0],
               (unsigned)k3 * step_b, os);
      const int kk = q / (RM * RN), i = q / RN % RM, j = q % RN;
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(CODES ? x[j][kk] : cur.b[CODES ? 0 : j][kk], cur.a[i][kk], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll 1
  for (int kt = 0; kt < H;) {
    step(kt++, f0, f1);
    if (kt >= H) break;
    step(kt++, f1, f0);
  }
  wait_loads<0>();  // no load may land in the epilogue's tile

  MxProblem e{};
  e.M = M; e.N = N; e.out = p.out; e.scal = p.alpha;
  e.aux = p.x; e.as = static_cast<const uint32_t*>(p.xs); e.groups = p.x_row;
  constexpr int KIND = MN ? KIND_GRAD8 : KIND_WEIGHT;
  constexpr int EACT = MN ? ACT : ACT_IDENTITY;
  if constexpr (WK == 1) {
    float* es = reinterpret_cast<float*>(smem) + w * 32 * (WTN + 4);
    if (p.vec) tile_epilogue<float, KIND, EACT, true, RM, RN>(e, acc, es, m0 + wm * WTM, n0 + wn * WTN);
    else tile_epilogue<float, KIND, EACT, false, RM, RN>(e, acc, es, m0 + wm * WTM, n0 + wn * WTN);
  } else {
    e.vec = p.vec;
    joined_epilogue<float, KIND, EACT, BM, BN, WK, RM, RN>(e, acc, smem, wk, wm * WTM, wn * WTN, m0, n0);
  }
}

template <int SRC, int ACT, int BM, int BN, int WGM, int WGN, int WK>
hipError_t run_tile32(const CkptProblem& p, hipStream_t s) {
  constexpr int smem = smem32<SRC, BM, BN, WGM, WGN, WK>();
  static_assert(smem <= 160 * 1024, "LDS");
  const void* fn = reinterpret_cast<const void*>(&ckpt_gemm32_kernel<SRC, ACT, BM, BN, WGM, WGN, WK>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  const long long tiles = ((p.M + BM - 1LL) / BM) * ((p.N + BN - 1LL) / BN);
  CkptProblem q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)tiles), dim3(WGM * WGN * WK * 64), args, smem, s);
}

// The tile: 32 x 32 with the contraction split where 64 x 64 ones do not outnumber the
// CUs, 128 x 128 from three a CU.  MI355X, us, 128 / 64 / 32 wide, gradient, then weight
// update from f(X) (out rows x columns x contraction):
//   1531 x 300 x 1000     73 / 26.5 / 14.8   70 / 25.8 / 14.3   (120 tiles of 64 x 64)
//   1024 x 1024 x 1024    74 / 27.7 / 24.9   70 / 26.6 / 24.6   (256)
//   1000 x 1531 x 300     29 / 16.9 / 19.1   26 / 15.9 / 18.0   (384)
//   2048 x 1024 x 1024    73 / 42 / 45       70 / 41 / 45       (512)
//   3200 x 2048 x 1024   134 / 122 / 128    129 / 121 / 126     (400 of 128 x 128)
//   4096 x 4096 x 1024   265 / 276 / 323    258 / 276 / 325     (1024)
template <int SRC, int ACT>
hipError_t run_ckpt32(const CkptProblem& p, hipStream_t s) {
  auto tiles = [&](long long e) { return ((p.M + e - 1) / e) * ((p.N + e - 1) / e); };
  if (tiles(64) <= 256) return run_tile32<SRC, ACT, 32, 32, 1, 1, 4>(p, s);
  if (tiles(128) >= 768) return run_tile32<SRC, ACT, 128, 128, 2, 2, 1>(p, s);
  return run_tile32<SRC, ACT, 64, 64, 2, 2, 1>(p, s);
}

}  // namespace mx
}  // namespace ipc
