// ipc_mx_gemm.h - products of two microscaled fp4 matrices (gfx950).
//
// C[m][n] = sum_k A[m][k] B[n][k] for packed A and B (ipc_mx.h: both have the
// contraction contiguous), on the scaled matrix instruction
// v_mfma_scale_f32_32x32x64_f8f6f4, which takes 32 codes (16 bytes) and the
// scale byte of one block per lane and accumulates in fp32: the operands are
// never expanded.  It runs at four times the 16-bit rate on a quarter of the
// bytes, so a tile's k-loop needs the same LDS and cache traffic per cycle as a
// 16-bit one, and the epilogue, whose tensors keep 16 or 32 bits, weighs four
// times as much.
//
// The first operand of the instruction is B (n), the second A (m): result
// register q of lane (lr = lane % 32, lk = lane / 32) is then row m = lr and
// column n = 8 (q / 4) + 4 lk + q % 4, four consecutive columns per lane.
#pragma once

#include <type_traits>

#include "ipc_launch.h"
#include "ipc_mx_device.h"

namespace ipc {
namespace mx {

typedef __attribute__((address_space(3))) void lds_void;

// A buffer of `bytes` bytes: per-lane byte offsets of 32 bits plus a uniform one;
// loads past the end give 0, dword by dword, the uniform offset counted (gfx950: lane
// offset 0, uniform 64, 72 bytes: two dwords of the 16 bytes, then zeros).
struct Rsrc {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Rsrc(const void* base, unsigned bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000)) {}
  // 16 or 4 bytes a lane from offset v + s into 64 consecutive places of the LDS
  __device__ __forceinline__ void to_lds16(unsigned char* lds, unsigned v, unsigned s) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, v, s, 0, 0);
  }
  __device__ __forceinline__ void to_lds4(unsigned char* lds, unsigned v, unsigned s) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 4, v, s, 0, 0);
  }
};

// s_waitcnt vmcnt(N) alone (N below 64), as a builtin's operand
template <int N>
constexpr int vm_wait() { return 0x0f70 | (N & 15) | ((N >> 4) << 14); }

__device__ __forceinline__ i32x8 operand(i32x4 v) {
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// acc += B A^T over 64 k: byte S of the scale dwords sb, sa.
template <int S>
__device__ __forceinline__ f32x16 mma(i32x4 b, unsigned sb, i32x4 a, unsigned sa, f32x16 acc) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b), operand(a), acc, 4, 4, S, (int)sb, S, (int)sa);
}

// Four consecutive elements of a row (`left` of them in range).
template <typename ST>
__device__ __forceinline__ void get4(const ST* p, bool vec, int left, float (&o)[4]) {
  if (vec && left >= 4) {
    load4(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
}
template <typename ST>
__device__ __forceinline__ void put4(ST* p, bool vec, int left, const float (&v)[4]) {
  typedef ST V __attribute__((ext_vector_type(4)));
  V w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = cvt<ST>(v[i]);
  if (vec && left >= 4) {
    *reinterpret_cast<V*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = w[i];
  }
}

// An epilogue of the 16-bit products in ipc_ckpt_gemm.h: G = f'(X) C, X kept in 8 bits
// (aux its codes, as its scales, groups the bytes of its rows).
constexpr int KIND_GRAD8 = 100;

// The epilogue of four elements, in fp32, each operation rounded on its own and
// the result rounded once to the storage type.  in: X_lower (PRED), X (INFER),
// W (WEIGHT); e: E (INFER).
template <int KIND, int ACT>
__device__ __forceinline__ void finish4(const float (&c)[4], const float (&in)[4], const float (&e)[4], float scal,
                                        float (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma clang fp contract(off)
    if (KIND == KIND_GRAD8) o[i] = dact_t<ACT>(in[i]) * c[i];
    else if (KIND == KIND_PRED) o[i] = in[i] - c[i];
    else if (KIND == KIND_FWD) o[i] = c[i];
    else if (KIND == KIND_INFER) o[i] = in[i] + scal * (-e[i] + dact_t<ACT>(in[i]) * c[i]);
    else o[i] = in[i] + scal * c[i];
  }
}
template <typename ST, int KIND>
__device__ __forceinline__ void inputs4(const MxProblem& p, int m, int n, float (&in)[4], float (&e)[4]) {
  const long long o = (long long)m * p.N + n;
  const int left = p.N - n;
  const ST* out = reinterpret_cast<const ST*>(p.out);
  const ST* aux = reinterpret_cast<const ST*>(p.aux);
  if (KIND == KIND_PRED) get4(aux + o, p.vec != 0, left, in);
  if (KIND == KIND_INFER || KIND == KIND_WEIGHT) get4(out + o, p.vec != 0, left, in);
  if (KIND == KIND_INFER) get4(aux + o, p.vec != 0, left, e);
}

// ------------------------------------------------------------- direct kernel
// The fewest output tiles: a workgroup's waves share one 32 x 32 tile and split its
// contraction by groups of 128; operands go from memory straight into
// registers, LOOK groups' loads in flight, and the waves' partial tiles are
// added through LDS in wave order (the bits depend on the number of waves,
// which the host takes from K alone).
constexpr int DIRECT_WAVES = 8;
template <typename ST, int KIND, int ACT>
__global__ void __launch_bounds__(DIRECT_WAVES * 64) mx_direct_kernel(const MxProblem p) {
  constexpr int LOOK = 4, LD = 36;
  __shared__ __align__(16) float part[DIRECT_WAVES][32 * LD];
  const int tn = (p.N + 31) >> 5;
  const int m0 = blockIdx.x / tn * 32, n0 = blockIdx.x % tn * 32;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lk = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int M = p.M, N = p.N, G = p.groups;
  const int m = m0 + lr < M ? m0 + lr : M - 1, n = n0 + lr < N ? n0 + lr : N - 1;  // rows past the end: never stored
  const uint8_t* pa = p.a + (long long)m * G * 64 + lk * 32;
  const uint8_t* pb = p.b + (long long)n * G * 64 + lk * 32;

  // the epilogue's inputs, ahead of the products (threads of the first 4 waves: 4 columns each)
  const int er = tid >> 3, ec = (tid & 7) * 4;
  float in[4], e[4], c[4], o[4];
  const bool mine = tid < 256 && m0 + er < M && n0 + ec < N;
  if (mine) inputs4<ST, KIND>(p, m0 + er, n0 + ec, in, e);

  f32x16 acc;
#pragma unroll
  for (int q = 0; q < 16; ++q) acc[q] = 0.0f;
  // the wave's groups g = wave, wave + waves, ...; half-wave lk takes blocks 2 lk and 2 lk + 1 of each
  for (int g0 = wave; g0 < G; g0 += waves * LOOK) {
    i32x4 a[LOOK][2], b[LOOK][2];
    unsigned sa[LOOK], sb[LOOK];
#pragma unroll
    for (int u = 0; u < LOOK; ++u) {
      const int g = g0 + u * waves < G ? g0 + u * waves : g0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        a[u][h] = *reinterpret_cast<const i32x4*>(pa + (long long)g * 64 + h * 16);
        b[u][h] = *reinterpret_cast<const i32x4*>(pb + (long long)g * 64 + h * 16);
      }
      sa[u] = p.as[(long long)g * M + m] >> (lk * 16);
      sb[u] = p.bs[(long long)g * N + n] >> (lk * 16);
    }
#pragma unroll
    for (int u = 0; u < LOOK; ++u) {
      if (g0 + u * waves >= G) break;
      acc = mma<0>(b[u][0], sb[u], a[u][0], sa[u], acc);
      acc = mma<1>(b[u][1], sb[u], a[u][1], sa[u], acc);
    }
  }
#pragma unroll
  for (int q = 0; q < 16; q += 4)
    *reinterpret_cast<float4*>(&part[wave][lr * LD + 2 * q + 4 * lk]) =
        make_float4(acc[q], acc[q + 1], acc[q + 2], acc[q + 3]);
  __syncthreads();
  if (!mine) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = part[0][er * LD + ec + i];
  for (int w = 1; w < waves; ++w) {
    const float4 t = *reinterpret_cast<const float4*>(&part[w][er * LD + ec]);
    c[0] += t.x; c[1] += t.y; c[2] += t.z; c[3] += t.w;
  }
  finish4<KIND, ACT>(c, in, e, p.scal, o);
  put4(reinterpret_cast<ST*>(p.out) + (long long)(m0 + er) * N + n0 + ec, p.vec != 0, N - n0 - ec, o);
}

// --------------------------------------------------------------- tile kernel
// BM x BN output tile per workgroup, k-steps of one group (128 values: 64 bytes
// of a row and one scale dword), four stages of LDS:
//
//   * codes and scales move HBM -> LDS with LDS-DMA loads (16 and 4 bytes a lane);
//     chunk c (16 bytes = one block) of row r lies at chunk c ^ ((r >> 2) & 3), so
//     that the 16 lanes of a fragment read, 16 consecutive rows, touch every bank
//     once;
//   * step t waits for stage t + 1, then one barrier publishes everybody's, then it
//     refills the stage everybody finished with step t - 1 (t + 3), its loads spread
//     between the products: issued in one go they hold up the wave, which is alone
//     on its SIMD, for as long as the memory pipeline takes them;
//   * the fragments of the next 64 k, at the end of a step those of stage t + 1, are
//     read while the current products run, so no read is waited for.
constexpr int STAGES = 4;
template <int BM, int BN>
constexpr int stage_bytes() { return (BM + BN) * (64 + 4); }
template <int BM, int BN, int WGM, int WGN>
constexpr int tile_smem() {
  constexpr int epi = WGM * WGN * 32 * (BN / WGN + 4) * 4, st = STAGES * stage_bytes<BM, BN>();
  return epi > st ? epi : st;
}

// The epilogue's inputs of 4 columns as loaded: raw dwords, widened when used.
template <typename ST, bool VEC> struct Raw4 { unsigned v[sizeof(ST) == 4 ? 4 : VEC ? 2 : 3]; };

// Rows of a tensor from a uniform element offset `first` on, behind a buffer
// resource that ends with the tensor's last row (mx_rows_bytes): 32-bit offsets, loads
// past the end give 0 or the rest of the last dword, stores past it store nothing.
// Buffer accesses need dwords only, so fp32
// rows of any length are read 16 bytes at a time; VEC: 16-bit rows whose length
// and base are multiples of 4 elements.  Other 16-bit rows are read as the three
// dwords around their 4 elements and shifted, and stored element by element.
// A row's last group may read into the next row (or 0 at the end): values that
// are not stored.
template <typename ST, bool VEC>
struct Rows {
  static constexpr unsigned ES = sizeof(ST), NO = 0xfffffff0u;
  typedef unsigned U2 __attribute__((ext_vector_type(2)));
  typedef unsigned U3 __attribute__((ext_vector_type(3)));
  __amdgpu_buffer_rsrc_t r;
  unsigned mis;  // bytes from the resource's start to element `first` (0 or 2)
  __device__ __forceinline__ Rows(const void* base, long long first, long long end, bool store = false) {
    const unsigned long long at = reinterpret_cast<unsigned long long>(static_cast<const ST*>(base) + first);
    mis = !VEC && ES == 2 ? (unsigned)(at & 2) : 0u;
    const long long bytes = mx_rows_bytes(first, end, ES, mis, store);
    r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(at - mis), (short)0,
                                          (int)(unsigned)(bytes < 0xffffff00LL ? bytes : 0xffffff00LL), 0x00020000);
  }
  // the 4 columns at element `at`, the first `left` of them in range
  __device__ __forceinline__ void get(unsigned at, int left, Raw4<ST, VEC>& o) const {
    const unsigned off = left > 0 ? at * ES + mis : NO;
    if constexpr (ES == 4) {
      const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
      o.v[0] = v[0]; o.v[1] = v[1]; o.v[2] = v[2]; o.v[3] = v[3];
    } else if constexpr (VEC) {
      const U2 v = __builtin_bit_cast(U2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
      o.v[0] = v[0]; o.v[1] = v[1];
    } else {
      const U3 v = __builtin_bit_cast(U3, __builtin_amdgcn_raw_buffer_load_b96(r, off & ~3u, 0, 0));
      o.v[0] = v[0]; o.v[1] = v[1]; o.v[2] = v[2];
    }
  }
  __device__ __forceinline__ void widen(const Raw4<ST, VEC>& q, unsigned at, float (&o)[4]) const {
    if constexpr (ES == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(float, q.v[i]);
    } else {
      const unsigned sh = VEC ? 0u : ((at * ES + mis) & 2u) * 8u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unsigned d = q.v[i];
        if constexpr (!VEC) d = __builtin_amdgcn_alignbit(q.v[i + 1], q.v[i], sh);
        o[2 * i] = h2f(d & 0xffffu, (ST*)nullptr);
        o[2 * i + 1] = h2f(d >> 16, (ST*)nullptr);
      }
    }
  }
  __device__ __forceinline__ void put(unsigned at, int left, const float (&v)[4]) const {
    if constexpr (ES == 4) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, v[i]);
      __builtin_amdgcn_raw_buffer_store_b128(w, r, left >= 4 ? at * ES : NO, 0, 0);
      if (left > 0 && left < 4) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
          __builtin_amdgcn_raw_buffer_store_b32(w[i], r, i < left ? (at + i) * ES : NO, 0, 0);
      }
    } else {
      unsigned short h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __builtin_bit_cast(unsigned short, cvt<ST>(v[i]));
      if constexpr (VEC) {
        const U2 w = {h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16};
        __builtin_amdgcn_raw_buffer_store_b64(w, r, left > 0 ? at * ES : NO, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_buffer_store_b16(h[i], r, i < left ? (at + i) * ES + mis : NO, 0, 0);
      }
    }
  }
};

// The wave's RM x RN blocks (first row mw, first column nw), 32 rows at a time
// through its own part of the LDS (rows of 32 RN + 4 floats: the four-column
// stores and reads of 16 lanes touch every bank once), then walked row by row, so
// that every global access is a run of 4-column groups.  The next 16 rows' inputs
// are in flight while these are finished.
template <typename ST, int KIND, int ACT, bool VEC, int RM, int RN>
__device__ __forceinline__ void tile_epilogue(const MxProblem& p, const f32x16 (&acc)[RM][RN], float* es, int mw, int nw) {
  constexpr int WTN = 32 * RN, LDE = WTN + 4, LPR = WTN / 4, RPP = 64 / LPR, PASSES = 16 / RPP;
  constexpr bool IN = KIND != KIND_FWD, E = KIND == KIND_INFER;
  const int lane = threadIdx.x & 63, lr = lane & 31, lk = lane >> 5;
  const int er = lane / LPR, ec = (lane % LPR) * 4, left = p.N - (nw + ec);
  const long long N = p.N, end = (long long)p.M * N;
  const unsigned at = (unsigned)er * (unsigned)p.N + (unsigned)ec;
  Raw4<ST, VEC> in[2][IN ? PASSES : 1], e[2][E ? PASSES : 1];
  auto fetch = [&](int v, int set) {  // 16 rows
    const long long first = (mw + v * 16) * N + nw;
    if constexpr (KIND == KIND_GRAD8) {  // four codes and their block's scale byte
      const int row = p.groups, n = nw + ec;
      const uint8_t* at8 = static_cast<const uint8_t*>(p.aux) + (long long)(mw + v * 16) * row;
      const Rsrc codes(at8, mw + v * 16 < p.M ? (unsigned)min((p.M - (long long)(mw + v * 16)) * row, 0xffffff00LL) : 0u);
      const Rsrc scales(p.as, (unsigned)mx_groups(p.N) * (unsigned)p.M * 4u);
#pragma unroll
      for (int u = 0; u < PASSES; ++u) {
        const int r = u * RPP + er, m = mw + v * 16 + r;
        in[set][u].v[0] = __builtin_amdgcn_raw_buffer_load_b32(codes.r, left > 0 ? (unsigned)(r * row + n) : 0xfffffff0u, 0, 0);
        in[set][u].v[1] = __builtin_amdgcn_raw_buffer_load_b8(
            scales.r, left > 0 && m < p.M ? ((unsigned)(n >> 7) * (unsigned)p.M + (unsigned)m) * 4u + ((n >> 5) & 3) : 0xfffffff0u, 0, 0);
      }
      return;
    }
    if constexpr (IN) {
      const Rows<ST, VEC> src(KIND == KIND_PRED ? p.aux : p.out, first, end);
#pragma unroll
      for (int u = 0; u < PASSES; ++u) src.get(at + (unsigned)(u * RPP) * (unsigned)p.N, left, in[set][IN ? u : 0]);
    }
    if constexpr (E) {
      const Rows<ST, VEC> src(p.aux, first, end);
#pragma unroll
      for (int u = 0; u < PASSES; ++u) src.get(at + (unsigned)(u * RPP) * (unsigned)p.N, left, e[set][E ? u : 0]);
    }
  };
  fetch(0, 0);
  __syncthreads();  // every wave is done with the stages
#pragma unroll
  for (int v = 0; v < 2 * RM; ++v) {
    const int i = v >> 1, set = v & 1;
    if (v + 1 < 2 * RM) fetch(v + 1, set ^ 1);
    if (set == 0) {
#pragma unroll
      for (int j = 0; j < RN; ++j)
#pragma unroll
        for (int q = 0; q < 16; q += 4)
          *reinterpret_cast<float4*>(es + lr * LDE + j * 32 + 2 * q + 4 * lk) =
              make_float4(acc[i][j][q], acc[i][j][q + 1], acc[i][j][q + 2], acc[i][j][q + 3]);
    }
    // (the wave's own LDS accesses complete in order; the fence keeps the compiler from reordering them)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const long long first = (mw + v * 16) * N + nw;
    const Rows<ST, VEC> dst(p.out, first, end, true);
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
      const float4 t4 = *reinterpret_cast<const float4*>(es + (set * 16 + u * RPP + er) * LDE + ec);
      const float c[4] = {t4.x, t4.y, t4.z, t4.w};
      float o[4], x[4], ev[4];
      const unsigned here = at + (unsigned)(u * RPP) * (unsigned)p.N;
      if constexpr (KIND == KIND_GRAD8) {
        const float unit = int8_scale(in[set][u].v[1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = (float)sext8(in[set][u].v[0], q) * unit;
      } else if constexpr (IN) Rows<ST, VEC>(KIND == KIND_PRED ? p.aux : p.out, first, end).widen(in[set][IN ? u : 0], here, x);
      if constexpr (E) Rows<ST, VEC>(p.aux, first, end).widen(e[set][E ? u : 0], here, ev);
      finish4<KIND, ACT>(c, x, ev, p.scal, o);
      dst.put(here, left, o);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <typename ST, int KIND, int ACT, int BM, int BN, int WGM, int WGN>
__global__ void __launch_bounds__(WGM * WGN * 64) mx_tile_kernel(const MxProblem p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int NW = WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, RM = WTM / 32, RN = WTN / 32;
  // LDS-DMA instructions per wave and stage: 16 rows of codes, 64 rows' scales each
  constexpr int IA = BM / 16 / NW, IB = BN / 16 / NW, CS = (BM + BN) / 64, IS = (CS + NW - 1) / NW;
  constexpr int LPS = IA + IB + IS;
  constexpr int STAGE = stage_bytes<BM, BN>(), A_BYTES = BM * 64, B_BYTES = BN * 64;
  static_assert(IA * 16 * NW == BM && IB * 16 * NW == BN && BM % 64 == 0 && BN % 64 == 0 && RM >= 1 && RN >= 1, "tile / waves");

  // workgroup b runs on XCD b % 8: consecutive tiles per XCD, in supertiles of 8 x 4:
  // the 32 tiles an XCD runs at once read 8 row blocks of A and 4 of B
  const int tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
  const int b = blockIdx.x, per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = b & 7;
  const int t = xcd * per + (xcd < rem ? xcd : rem) + (b >> 3);
  const int band = t / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, w8 = t - band * 8 * tn;
  const int cs = w8 / (rows * 4), cols = tn - cs * 4 < 4 ? tn - cs * 4 : 4, w2 = w8 - cs * rows * 4;
  const int m0 = (band * 8 + w2 / cols) * BM, n0 = (cs * 4 + w2 % cols) * BN;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WGN, wn = w % WGN, lr = lane & 31, lk = lane >> 5;
  const int M = p.M, N = p.N, G = p.groups;
  const unsigned rb = (unsigned)G * 64u;  // bytes of a packed row (codes of a matrix: below 2^30 bytes)

  // LDS-DMA sources: instruction q of this wave fills rows (q NW + w) 16 .. + 15 of the
  // stage's codes, then 64 consecutive scale dwords of A or B (rows past the end: the
  // last row again, never stored)
  const Rsrc ga(p.a, (unsigned)M * rb), gb(p.b, (unsigned)N * rb);
  const Rsrc gas(p.as, (unsigned)M * (unsigned)G * 4u), gbs(p.bs, (unsigned)N * (unsigned)G * 4u);
  const int dr = lane >> 2, dc = ((lane & 3) ^ ((dr >> 2) & 3)) * 16;
  unsigned oa[IA], ob[IB];
#pragma unroll
  for (int q = 0; q < IA; ++q) {
    const int m = m0 + (q * NW + w) * 16 + dr;
    oa[q] = (unsigned)(m < M ? m : M - 1) * rb + (unsigned)dc;
  }
#pragma unroll
  for (int q = 0; q < IB; ++q) {
    const int n = n0 + (q * NW + w) * 16 + dr;
    ob[q] = (unsigned)(n < N ? n : N - 1) * rb + (unsigned)dc;
  }
  unsigned os[IS];
#pragma unroll
  for (int q = 0; q < IS; ++q) {
    const int c = min(q * NW + w, CS - 1), r = c < BM / 64 ? m0 + c * 64 + lane : n0 + (c - BM / 64) * 64 + lane;
    os[q] = (unsigned)min(r, (c < BM / 64 ? M : N) - 1) * 4u;
  }
  auto load = [&](int q, int kt, unsigned char* st) {
    if (q < IA) {
      ga.to_lds16(st + (q * NW + w) * 1024, oa[q < IA ? q : 0], (unsigned)kt * 64u);
    } else if (q < IA + IB) {
      gb.to_lds16(st + A_BYTES + ((q - IA) * NW + w) * 1024, ob[q - IA < IB && q >= IA ? q - IA : 0], (unsigned)kt * 64u);
    } else {
      const int c = min((q - IA - IB) * NW + w, CS - 1);  // uniform; a spare wave repeats the last
      unsigned char* to = st + A_BYTES + B_BYTES + c * 256;
      const unsigned from = os[q >= IA + IB ? q - IA - IB : 0];
      if (c < BM / 64) gas.to_lds4(to, from, (unsigned)kt * (unsigned)M * 4u);
      else gbs.to_lds4(to, from, (unsigned)kt * (unsigned)N * 4u);
    }
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  // fragments of 64 k: chunk 2 s + lk of the lane's rows; scale byte 2 s + lk
  const int sw = (lr >> 2) & 3;
  const unsigned fa0 = (unsigned)((wm * WTM + lr) * 64), fb0 = (unsigned)(A_BYTES + (wn * WTN + lr) * 64);
  const unsigned fs0 = (unsigned)(A_BYTES + B_BYTES + (wm * WTM + lr) * 4);
  const unsigned gs0 = (unsigned)(A_BYTES + B_BYTES + BM * 4 + (wn * WTN + lr) * 4);
  i32x4 fa[2][RM], fb[2][RN];
  unsigned sa[2][RM], sb[2][RN];
  auto read_a = [&](const unsigned char* st, int s, int i, i32x4& o) {
    o = *reinterpret_cast<const i32x4*>(st + fa0 + i * 2048 + ((((s * 2) | lk) ^ sw) << 4));
  };
  auto read_b = [&](const unsigned char* st, int s, int j, i32x4& o) {
    o = *reinterpret_cast<const i32x4*>(st + fb0 + j * 2048 + ((((s * 2) | lk) ^ sw) << 4));
  };
  auto read_scales = [&](const unsigned char* st, unsigned (&a)[RM], unsigned (&bq)[RN]) {
#pragma unroll
    for (int i = 0; i < RM; ++i) a[i] = *reinterpret_cast<const unsigned*>(st + fs0 + i * 128) >> (8 * lk);
#pragma unroll
    for (int j = 0; j < RN; ++j) bq[j] = *reinterpret_cast<const unsigned*>(st + gs0 + j * 128) >> (8 * lk);
  };
  auto stage = [&](int kt) -> unsigned char* { return smem + (kt & (STAGES - 1)) * STAGE; };

  // prologue: stages 0 .. 2; the loads of a stage are always issued, past the last group those of the last again,
  // so that the counts below hold for every step
  auto group = [&](int kt) { return kt < G ? kt : G - 1; };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
#pragma unroll
    for (int q = 0; q < LPS; ++q) load(q, group(s), stage(s));
  __builtin_amdgcn_s_waitcnt(vm_wait<2 * LPS>());
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < RN; ++j) read_b(stage(0), 0, j, fb[0][j]);
#pragma unroll
  for (int i = 0; i < RM; ++i) read_a(stage(0), 0, i, fa[0][i]);
  read_scales(stage(0), sa[0], sb[0]);

  // one half of a step: products of the 64 k in set S; the fragments of the next 64 k
  // (k-half S ^ 1 of stage `next`) and half of the refill's loads between them
  auto half = [&](auto SV, auto PV, const unsigned char* next, int kt, unsigned char* fill) {
    constexpr int S = decltype(SV)::value, O = S ^ 1, P = decltype(PV)::value;
    constexpr int L0 = S == 0 ? 0 : (LPS + 1) / 2, L1 = S == 0 ? (LPS + 1) / 2 : LPS;
    constexpr int NM = RM * RN, NR = RM + RN;
    if constexpr (S == 1) read_scales(next, sa[P ^ 1], sb[P ^ 1]);
#pragma unroll
    for (int q = 0; q < NM; ++q) {
      // (spread evenly: read r before product r NM / NR, load l before product l NM / (L1 - L0))
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * NM / NR == q) {
          if (r < RN) read_b(next, O, r < RN ? r : 0, fb[O][r < RN ? r : 0]);
          else read_a(next, O, r < RN ? 0 : r - RN, fa[O][r < RN ? 0 : r - RN]);
        }
#pragma unroll
      for (int l = L0; l < L1; ++l)
        if ((l - L0) * NM / (L1 - L0) == q) load(l, kt, fill);
      const int i = q / RN, j = q % RN;
      acc[i][j] = mma<2 * S>(fb[S][j], sb[P][j], fa[S][i], sa[P][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  typedef std::integral_constant<int, 0> C0;
  typedef std::integral_constant<int, 1> C1;
  auto step = [&](auto PV, int kt) {
    // stage kt + 1 of this wave has landed (kt + 2 may be in flight), then everybody's;
    // everybody is done with stage kt - 1, which kt + 3 takes
    __builtin_amdgcn_s_waitcnt(vm_wait<LPS>());
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    unsigned char* fill = stage(kt + 3);
    half(C0{}, PV, stage(kt), group(kt + 3), fill);
    half(C1{}, PV, stage(kt + 1), group(kt + 3), fill);
  };
  int kt = 0;
#pragma unroll 1
  for (; kt + 1 < G; kt += 2) {
    step(C0{}, kt);
    step(C1{}, kt + 1);
  }
  if (kt < G) step(C0{}, kt);
  __builtin_amdgcn_s_waitcnt(vm_wait<0>());  // no load may land in the epilogue's tile

  float* es = reinterpret_cast<float*>(smem) + w * 32 * (WTN + 4);
  if (p.vec) tile_epilogue<ST, KIND, ACT, true, RM, RN>(p, acc, es, m0 + wm * WTM, n0 + wn * WTN);
  else tile_epilogue<ST, KIND, ACT, false, RM, RN>(p, acc, es, m0 + wm * WTM, n0 + wn * WTN);
}

// ------------------------------------------------------------------ launches
template <typename ST, int KIND, int ACT, int BM, int BN, int WGM, int WGN>
hipError_t run_tile(const MxProblem& p, hipStream_t s) {
  constexpr int smem = tile_smem<BM, BN, WGM, WGN>();
  static_assert(smem <= 160 * 1024, "LDS");
  const void* fn = reinterpret_cast<const void*>(&mx_tile_kernel<ST, KIND, ACT, BM, BN, WGM, WGN>);
  static const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  const long long tiles = ((p.M + BM - 1LL) / BM) * ((p.N + BN - 1LL) / BN);
  MxProblem q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)tiles), dim3(WGM * WGN * 64), args, smem, s);
}

// Which kernel: the largest tile that fills the 256 CUs about once, the direct
// kernel for the fewest.  MI355X, bf16 forward, us, 256 / 128 / 64 wide tiles / direct:
//   512 x 4096 x 512   (256 tiles of 32 x 32)    23.2 /  9.6 /  6.5 /  6.1
//   1000 x 1531 x 300  (320)                     12.7 /  5.7 /  4.0 /  7.1
//   1024 x 4096 x 1024 (64 of 128 x 128)         23.3 /  9.9 /  7.1 / 17.6
//   2048 x 8192 x 1024 (128)                     41.5 / 22.1 / 21.5 / 64.6
//   2048 x 4096 x 2048 (256)                     24.8 / 13.5 / 21.2 / 62.3
//   2560 x 4096 x 2560 (100 of 256 x 256)        26.6 / 23.3 / 36.4
//   3000 x 2048 x 3000 (144)                     18.9 / 20.5 / 27.2
//   3584 x 4096 x 3584 (196)                     32.9 / 45.9 / 65.6
template <typename ST, int KIND, int ACT>
hipError_t run_product(const MxProblem& p, hipStream_t s) {
  auto tiles = [&](long long e) { return ((p.M + e - 1) / e) * ((p.N + e - 1) / e); };
  if (tiles(32) <= 256) {
    const int waves = p.groups < 4 ? 4 : p.groups < DIRECT_WAVES ? p.groups : DIRECT_WAVES;
    hipLaunchKernelGGL((mx_direct_kernel<ST, KIND, ACT>), dim3((unsigned)tiles(32)), dim3(waves * 64), 0, s, p);
    return hipGetLastError();
  }
  if (tiles(256) >= 136) return run_tile<ST, KIND, ACT, 256, 256, 2, 2>(p, s);
  if (tiles(128) > 128) return run_tile<ST, KIND, ACT, 128, 128, 2, 2>(p, s);
  return run_tile<ST, KIND, ACT, 64, 64, 2, 2>(p, s);
}

template <typename ST>
hipError_t run_storage(const MxProblem& p, hipStream_t s) {
  switch (p.kind) {
    case KIND_PRED: return run_product<ST, KIND_PRED, ACT_IDENTITY>(p, s);
    case KIND_FWD: return run_product<ST, KIND_FWD, ACT_IDENTITY>(p, s);
    case KIND_WEIGHT: return run_product<ST, KIND_WEIGHT, ACT_IDENTITY>(p, s);
    default: break;
  }
  switch (p.act) {
    case ACT_RELU: return run_product<ST, KIND_INFER, ACT_RELU>(p, s);
    case ACT_TANH: return run_product<ST, KIND_INFER, ACT_TANH>(p, s);
    case ACT_SIGMOID: return run_product<ST, KIND_INFER, ACT_SIGMOID>(p, s);
    case ACT_SILU: return run_product<ST, KIND_INFER, ACT_SILU>(p, s);
    case ACT_GELU: return run_product<ST, KIND_INFER, ACT_GELU>(p, s);
    default: return run_product<ST, KIND_INFER, ACT_IDENTITY>(p, s);
  }
}

}  // namespace mx
}  // namespace ipc
