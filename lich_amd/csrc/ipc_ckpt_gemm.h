// ipc_ckpt_gemm.h - the backward pass of a state kept in 8 bits as 16-bit products (gfx950).
//
//   CKPT_GRAD     G[m][n] = f'(X)[m][n] sum_k A[k][m] B[k][n]   A = W_lower, B = E_lower
//   CKPT_WEIGHT   W[m][n] += alpha sum_k A[m][k] B[n][k]         A = E, B = f(X) widened
//
// v_mfma_f32_32x32x16 tiles in the pipeline of the 4-bit product's tile kernel
// (ipc_mx_gemm.h): four stages of LDS filled by LDS-DMA loads, here of 32 k (64
// bytes of a k-contiguous row, or 32 k-rows of a tile's columns), one barrier a
// stage, the loads spread between the products, the next fragments read while the
// current products run.  A 16-bit product does a quarter of the fp4 one's work per
// byte in the same time, so the same tile keeps the matrix units as busy.
//
//   * loads take 16 bytes a lane from any multiple of 4 bytes; where a row ends inside one
//     they bring the next row's first values, which no stored output reads.  The last
//     1 .. 32 k come first, as a stage whose rest is cleared before anything is read.
//     Rows of an odd length are laid out once in a workspace (ckpt_pad_kernel);
//   * k-contiguous rows: chunk c (16 bytes) of row r at c ^ ((r >> 2) & 3), fragments
//     are 16-byte reads;
//   * k-rows (CKPT_GRAD): chunk c of k-row r at c ^ ((r & 3) << 2) (64 columns: ^ ((r & 2)
//     << 1)), fragments come from
//     two transposing reads (ds_read_b64_tr_b16), the operands are never transposed in
//     memory.
//
// B is f(X8) rounded once to the operand type, the matrix instruction's: W's error against
// 64 bits, 4096 x 4096, B = 1024, bf16, tanh, 2.0e-3 of its norm, 1.7e-3 with f in fp32 (W's
// own rounding); identity and relu of 8-bit codes are exact in bf16.  A second
// term would double the products.
//
// Reading the packed state in the weight update's own loader instead (codes to
// registers, widened a step or two later, stored to the stage) was slower than
// widening it once into a workspace at every size: 4096 x 4096, B = 1024, relu 59 us
// against 40 and 5 for the widening.
#pragma once

#include "ipc_mx_gemm.h"

namespace ipc {

namespace mx {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 16 bytes a lane from byte offset v + s of a buffer into 64 consecutive places of
// the LDS, unknown to the compiler: it would wait for every such load in flight
// before each transposing read, whose address it cannot tell from theirs (the state
// gradient's main loop then ran four times as long).  There is no register to wait
// for; every wait is one of the kernel's own.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds16_unseen(i32x4 rsrc, unsigned char* lds, unsigned v, unsigned s) {
  const unsigned at = (unsigned)(unsigned long long)(lds_void*)lds;
  // (m0 holds the place; a wait state lies between its write and its use.  Named as
  // clobbered, so that the compiler sets it anew for an instruction of its own that reads
  // it; it warns of any reserved register there.)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(at), "v"(v), "s"(rsrc), "s"(s)
               : "memory", "m0");
}
#pragma clang diagnostic pop
// The buffer resource of `bytes` bytes at `base`, as words.
__device__ __forceinline__ i32x4 rsrc_words(const void* base, unsigned bytes) {
  const unsigned long long a = reinterpret_cast<unsigned long long>(base);
  return i32x4{(int)(unsigned)a, (int)(unsigned)(a >> 32 & 0xffffu), (int)bytes, 0x00020000};
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The epilogue where WK groups of waves split a tile's contraction: their sums meet in
// LDS and are added in the groups' order, every wave finishes some rows of the tile.
template <typename ST, int KIND, int ACT, int BM, int BN, int WK, int RM, int RN>
__device__ __forceinline__ void joined_epilogue(const MxProblem& p, const f32x16 (&acc)[RM][RN], unsigned char* smem, int wk,
                                                int mw, int nw, int m0, int n0) {
  constexpr int LD = BN + 4, LANES = BN / 4, THREADS = (BM / 32 / RM) * (BN / 32 / RN) * WK * 64;
  constexpr int PASS = THREADS / LANES, PASSES = BM / PASS;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lk = lane >> 5;
  const int er = tid / LANES, ec = tid % LANES * 4, n = n0 + ec, left = p.N - n;
  float in[PASSES][4];
  ST* out = static_cast<ST*>(p.out);
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int m = m0 + u * PASS + er;
#pragma unroll
    for (int i = 0; i < 4; ++i) in[u][i] = 0.0f;
    if (m >= p.M || left <= 0) continue;
    if constexpr (KIND == KIND_GRAD8) {
      const unsigned q = *reinterpret_cast<const unsigned*>(static_cast<const uint8_t*>(p.aux) + (long long)m * p.groups + n);
      const float unit = int8_scale(reinterpret_cast<const uint8_t*>(p.as)[((long long)(n >> 7) * p.M + m) * 4 + ((n >> 5) & 3)]);
#pragma unroll
      for (int i = 0; i < 4; ++i) in[u][i] = (float)sext8(q, i) * unit;
    } else {
      get4(out + (long long)m * p.N + n, p.vec != 0, left, in[u]);
    }
  }
  float* part = reinterpret_cast<float*>(smem);
  __syncthreads();  // every wave is done with its ring
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; q += 4)
        *reinterpret_cast<float4*>(part + (wk * BM + mw + i * 32 + lr) * LD + nw + j * 32 + 2 * q + 4 * lk) =
            make_float4(acc[i][j][q], acc[i][j][q + 1], acc[i][j][q + 2], acc[i][j][q + 3]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int m = m0 + u * PASS + er;
    if (m >= p.M || left <= 0) continue;
    float c[4] = {}, none[4] = {}, o[4];
#pragma unroll
    for (int v = 0; v < WK; ++v) {
      const float4 t4 = *reinterpret_cast<const float4*>(part + (v * BM + u * PASS + er) * LD + ec);
      c[0] += t4.x; c[1] += t4.y; c[2] += t4.z; c[3] += t4.w;
    }
    finish4<KIND, ACT>(c, in[u], none, p.scal, o);
    put4(out + (long long)m * p.N + n, p.vec != 0, left, o);
  }
}

template <typename OT, int MODE, int ACT, int BM, int BN, int WGM, int WGN, int WK>
__global__ void __launch_bounds__(WGM * WGN * WK * 64) ckpt_gemm_kernel(const CkptProblem p) {
  extern __shared__ __align__(16) unsigned char smem[];
  using MF = Mfma32<OT>;
  typedef typename MF::operand V;
  constexpr bool MN = MODE == CKPT_GRAD;
  constexpr int NW = WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, RM = WTM / 32, RN = WTN / 32;
  constexpr int A_BYTES = BM * 64, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES;
  constexpr int IA = A_BYTES / 1024 / NW, IB = B_BYTES / 1024 / NW, LPS = IA + IB;  // LDS-DMA loads per wave and stage
  static_assert(IA * 1024 * NW == A_BYTES && IB * 1024 * NW == B_BYTES, "tile / waves");

  // consecutive tiles per XCD, in supertiles of 8 x 4 (as in mx_tile_kernel)
  const int tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
  const int b = blockIdx.x, per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = b & 7;
  const int t = xcd * per + (xcd < rem ? xcd : rem) + (b >> 3);
  const int band = t / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, w8 = t - band * 8 * tn;
  const int cs = w8 / (rows * 4), cols = tn - cs * 4 < 4 ? tn - cs * 4 : 4, w2 = w8 - cs * rows * 4;
  const int m0 = (band * 8 + w2 / cols) * BM, n0 = (cs * 4 + w2 % cols) * BN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w = wave % NW, wk = wave / NW;  // wave of its group, group
  const int wm = w / WGN, wn = w % WGN, lr = lane & 31, lk = lane >> 5;
  unsigned char* ring = smem + wk * STAGES * STAGE;
  // (the host: operands below 2^31 bytes, rows that start at multiples of 4)
  const int M = p.M, N = p.N, K = p.K, G = (K + 31) / 32, tail = K - (G - 1) * 32;

  const Rsrc ga(p.a, (unsigned)((MN ? (long long)p.K : (long long)M) * p.lda * 2));
  const Rsrc gb(p.b, (unsigned)((MN ? (long long)p.K : (long long)N) * p.ldb * 2));
  const i32x4 wa = rsrc_words(p.a, (unsigned)((long long)p.K * p.lda * 2)), wb = rsrc_words(p.b, (unsigned)((long long)p.K * p.ldb * 2));
  // byte offset of this lane's 16 bytes of LDS-DMA instruction q of an operand, `have` k-rows in the stage
  auto source = [&](int q, int edge, int e0, int lim, long long ld, int have) -> unsigned {
    const int slot = (q * NW + w) * 64 + lane;
    if constexpr (MN) {  // columns past the end: the last ones again or the next row's, never stored
      const int cpr = edge / 8, r = slot / cpr, c = (slot % cpr) ^ (edge == 64 ? (r & 2) << 1 : (r & 3) << 2);
      const int col = e0 + c * 8 < (int)ld ? e0 + c * 8 : (int)ld - 2;
      return (unsigned)((r < have ? r : have - 1) * ld + col) * 2u;
    } else {
      const int r = slot >> 2, c = (slot & 3) ^ ((r >> 2) & 3), row = e0 + r < lim ? e0 + r : lim - 1;
      return (unsigned)(row * ld) * 2u + (unsigned)c * 16u;
    }
  };
  unsigned oa[IA], ob[IB];
#pragma unroll
  for (int q = 0; q < IA; ++q) oa[q] = source(q, BM, m0, M, p.lda, 32);
#pragma unroll
  for (int q = 0; q < IB; ++q) ob[q] = source(q, BN, n0, N, p.ldb, 32);
  const unsigned step_a = MN ? (unsigned)p.lda * 2u : 2u, step_b = MN ? (unsigned)p.ldb * 2u : 2u;
  // load q of a stage: lane offset v, uniform offsets sa, sb
  auto load = [&](int q, unsigned char* st, unsigned v, unsigned sa, unsigned sb) {
    unsigned char* at = q < IA ? st + (q * NW + w) * 1024 : st + A_BYTES + ((q - IA) * NW + w) * 1024;
    if constexpr (MN) to_lds16_unseen(q < IA ? wa : wb, at, v, q < IA ? sa : sb);
    else (q < IA ? ga : gb).to_lds16(at, v, q < IA ? sa : sb);
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  // fragments of 16 k (half s of a stage): row / column lr of a 32-wide block, k 8 lk .. + 7
  const int g4 = lane >> 4, li = lane & 15;
  const int tr_row = 8 * (g4 >> 1) + (li >> 2), tr_low = 2 * (g4 & 1) + ((li & 3) >> 1);
  auto fragment = [&](const unsigned char* blk, int rowb, int e, int s) -> V {
    if constexpr (MN) {
      const int chunk = (((e >> 5) ^ (rowb == 128 ? li >> 3 : li >> 2)) << 2) | tr_low;
      const unsigned char* p0 = blk + (s * 16 + tr_row) * rowb + (chunk << 4) + (li & 1) * 8;
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p0 + 4 * rowb));
      return __builtin_bit_cast(V, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const V*>(blk + (e + lr) * 64 + ((((s * 2) | lk) ^ ((lr >> 2) & 3)) << 4));
    }
  };
  V fa[2][RM], fb[2][RN];
  auto stage = [&](int kt) -> unsigned char* { return ring + (kt & (STAGES - 1)) * STAGE; };

  // prologue: stages 0 .. 2.  The last 1 .. 32 k are stage 0; what a load there has past
  // the operand's end is 0, as it is where a whole stage's last row is shorter than a load.
  if (G == 1) {  // (no other stage: its loads take the operands' first values)
#pragma unroll
    for (int q = 0; q < IA; ++q) oa[q] = 0;
#pragma unroll
    for (int q = 0; q < IB; ++q) ob[q] = 0;
  }
  // first k of the group's stage kt (not stage 0); past the end: of the last, so that every step counts the same
  auto k_of = [&](int kt) {
    const int g = kt * WK + wk;
    return (unsigned)(G == 1 ? 0 : (g < G ? g : G - 1) - 1) * 32u;
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    const bool first = s * WK + wk == 0;
    const unsigned k = first ? 0u : k_of(s), last = (unsigned)(K - tail);
#pragma unroll
    for (int q = 0; q < LPS; ++q) {
      unsigned v = q < IA ? oa[q < IA ? q : 0] : ob[q < IA ? 0 : q - IA];
      if (first) v = q < IA ? source(q, BM, m0, M, p.lda, tail) + last * step_a : source(q - IA, BN, n0, N, p.ldb, tail) + last * step_b;
      load(q, stage(s), v, k * step_a, k * step_b);
    }
  }
  wait_loads<2 * LPS>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (tail < 32) {  // clear what stage 0 has no k for
    const int at = w * 64 + lane;
    uint4* o = reinterpret_cast<uint4*>(ring);
    if (wk > 0) {
    } else if constexpr (MN) {
      for (int i = tail * (BM / 8) + at; i < 32 * (BM / 8); i += NW * 64) o[i] = make_uint4(0, 0, 0, 0);
      for (int i = tail * (BN / 8) + at; i < 32 * (BN / 8); i += NW * 64) o[A_BYTES / 16 + i] = make_uint4(0, 0, 0, 0);
    } else {  // of E (f(X) has values there)
      unsigned short* h = reinterpret_cast<unsigned short*>(ring);
      for (int i = at; i < BM * 32; i += NW * 64)
        if (((i & 31) ^ (((i >> 7) & 3) << 3)) >= tail) h[i] = 0;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int j = 0; j < RN; ++j) fb[0][j] = fragment(stage(0) + A_BYTES, BN * 2, wn * WTN + j * 32, 0);
#pragma unroll
  for (int i = 0; i < RM; ++i) fa[0][i] = fragment(stage(0), BM * 2, wm * WTM + i * 32, 0);

  // half a step: the products of set S; the fragments of the next 16 k (half S ^ 1 of
  // `next`) and half of stage kt + 3's loads between them
  auto half = [&](auto SV, const unsigned char* next, int kt) {
    constexpr int S = decltype(SV)::value, O = S ^ 1;
    constexpr int L0 = S == 0 ? 0 : (LPS + 1) / 2, L1 = S == 0 ? (LPS + 1) / 2 : LPS;
    constexpr int NM = RM * RN, NR = RM + RN;
    const unsigned k3 = k_of(kt + 3);
#pragma unroll
    for (int q = 0; q < NM; ++q) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * NM / NR == q) {
          if (r < RN) fb[O][r < RN ? r : 0] = fragment(next + A_BYTES, BN * 2, wn * WTN + r * 32, O);
          else fa[O][r < RN ? 0 : r - RN] = fragment(next, BM * 2, wm * WTM + (r - RN) * 32, O);
        }
#pragma unroll
      for (int l = L0; l < L1; ++l)
        if ((l - L0) * NM / (L1 - L0) == q)
          load(l, stage(kt + 3), l < IA ? oa[l < IA ? l : 0] : ob[l < IA ? 0 : l - IA], k3 * step_a, k3 * step_b);
      const int i = q / RN, j = q % RN;
      if (WK == 1 || kt * WK + wk < G) acc[i][j] = MF::run(fb[S][j], fa[S][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll 1
  for (int kt = 0; kt < (G + WK - 1) / WK; ++kt) {
    // stage kt + 1 of this wave has landed (kt + 2 may be in flight), then everybody's;
    // everybody is done with stage kt - 1, which kt + 3 takes
    wait_loads<LPS>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    half(std::integral_constant<int, 0>{}, stage(kt), kt);
    half(std::integral_constant<int, 1>{}, stage(kt + 1), kt);
  }
  wait_loads<0>();  // no load may land in the epilogue's tile

  MxProblem e{};
  e.M = M; e.N = N; e.out = p.out; e.scal = p.alpha;
  e.aux = p.x; e.as = static_cast<const uint32_t*>(p.xs); e.groups = p.x_row;
  constexpr int KIND = MODE == CKPT_GRAD ? KIND_GRAD8 : KIND_WEIGHT;
  constexpr int EACT = MODE == CKPT_GRAD ? ACT : ACT_IDENTITY;
  if constexpr (WK > 1) {
    e.vec = p.vec;
    joined_epilogue<OT, KIND, EACT, BM, BN, WK, RM, RN>(e, acc, smem, wk, wm * WTM, wn * WTN, m0, n0);
    return;
  }
  float* es = reinterpret_cast<float*>(smem) + w * 32 * (WTN + 4);
  if (p.vec) tile_epilogue<OT, KIND, EACT, true, RM, RN>(e, acc, es, m0 + wm * WTM, n0 + wn * WTN);
  else tile_epilogue<OT, KIND, EACT, false, RM, RN>(e, acc, es, m0 + wm * WTM, n0 + wn * WTN);
}

// Up to two matrices of 16-bit values with their rows padded with zeros to ld, a
// multiple of 8: one pass, 16 bytes a lane, four loads in flight.
struct PadJob {
  const unsigned short* src;
  unsigned short* dst;
  int rows, n, ld;
};
constexpr int PAD_CHUNKS = 4 * 256;  // of a workgroup
inline long long pad_blocks(const PadJob& j) { return (j.rows * (long long)(j.ld / 8) + PAD_CHUNKS - 1) / PAD_CHUNKS; }

template <typename OT, int MODE, int ACT, int BM, int BN, int WGM, int WGN, int WK = 1>
hipError_t run_ckpt_tile(const CkptProblem& p, hipStream_t s) {
  constexpr int epi = WK == 1 ? WGM * WGN * 32 * (BN / WGN + 4) * 4 : WK * BM * (BN + 4) * 4;
  constexpr int st = WK * STAGES * (BM + BN) * 64, smem = epi > st ? epi : st;
  static_assert(smem <= 160 * 1024, "LDS");
  const void* fn = reinterpret_cast<const void*>(&ckpt_gemm_kernel<OT, MODE, ACT, BM, BN, WGM, WGN, WK>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  const long long tiles = ((p.M + BM - 1LL) / BM) * ((p.N + BN - 1LL) / BN);
  CkptProblem q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)tiles), dim3(WGM * WGN * WK * 64), args, smem, s);
}

// The tile: the largest that gives the 256 CUs about one each; where 64 x 64 ones do not
// outnumber the CUs and the contraction is long, four groups of waves split it (a CU
// then has 96 KB of loads in flight instead of 24).  MI355X, bf16, us, 256 / 128 / 64 / 64
// wide and split, gradient, then weight update (out rows x columns x contraction):
//   128 x 128 x 4096     86 / 30 / 20 / 13        71 / 28 / 16.4 / 12.0
//   512 x 512 x 512      28 / 10.2 / 6.0 / 5.9    16 / 7.1 / 6.1 / 6.5
//   1024 x 1024 x 1024   37 / 13.3 / 8.4 / 7.6    24 / 10.4 / 7.0 / 7.5
//   1024 x 1024 x 4096   88 / 37 / 30 / 18        75 / 35 / 28 / 20     (256 tiles of 64 x 64)
//   2048 x 1024 x 1024   38 / 14.3 / 11.3 / 14.1  25 / 11.1 / 10.4 / 13.6
//   2048 x 2048 x 2048   56 / 25.7 / 31.5 / 40    43 / 23.8 / 41 / 40   (256 of 128 x 128)
//   3200 x 3200 x 2048   58 / 55 / 68             48 / 59 / 92          (169 of 256 x 256)
//   8192 x 2048 x 8192   205 / 235                203 / 295             (256)
template <typename OT, int MODE, int ACT>
hipError_t run_ckpt(const CkptProblem& p, hipStream_t s) {
  auto tiles = [&](long long e) { return ((p.M + e - 1) / e) * ((p.N + e - 1) / e); };
  if (tiles(256) >= (MODE == CKPT_GRAD ? 224 : 160)) return run_ckpt_tile<OT, MODE, ACT, 256, 256, 2, 2>(p, s);
  if (tiles(128) > 128) return run_ckpt_tile<OT, MODE, ACT, 128, 128, 2, 2>(p, s);
  if (tiles(64) <= 256 && p.K > 1024) return run_ckpt_tile<OT, MODE, ACT, 64, 64, 2, 2, 4>(p, s);
  return run_ckpt_tile<OT, MODE, ACT, 64, 64, 2, 2>(p, s);
}

}  // namespace mx
}  // namespace ipc
