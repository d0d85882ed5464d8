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
// loads whose offset is past the end give 0.
struct Rsrc {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Rsrc(const void* base, unsigned bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000)) {}
  __device__ __forceinline__ void to_lds(unsigned char* lds, unsigned v, unsigned s) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, v, s, 0, 0);
  }
  __device__ __forceinline__ unsigned load(unsigned v, unsigned s) const {
    return __builtin_amdgcn_raw_buffer_load_b32(r, v, s, 0);
  }
};

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

// The epilogue of four elements, in fp32, each operation rounded on its own and
// the result rounded once to the storage type.  in: X_lower (PRED), X (INFER),
// W (WEIGHT); e: E (INFER).
template <int KIND, int ACT>
__device__ __forceinline__ void finish4(const float (&c)[4], const float (&in)[4], const float (&e)[4], float scal,
                                        float (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma clang fp contract(off)
    if (KIND == KIND_PRED) o[i] = in[i] - c[i];
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
// Few output tiles: a workgroup's waves share one 32 x 32 tile and split its
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
// BM x BN output tile per workgroup, k-steps of 256 (128 bytes of a row):
// both operands move HBM -> LDS with 16-byte LDS-DMA loads, two stages; chunk
// c (16 bytes = one block) of row r lies at chunk c ^ ((r >> 1) & 7), so that
// the 16 lanes of a fragment read, 16 consecutive rows, touch every bank once.
// Half-wave lk takes blocks 4 lk .. 4 lk + 3 of a k-step, one per instruction:
// their scales are the four bytes of one dword, loaded straight into a
// register (32 consecutive dwords a half-wave) one step ahead.
//
// A contraction of an odd number of 128-groups ends in half a step: its upper
// half-wave reads the lower half's chunks again, with scale bytes of 0: 2^-127
// on both sides of every product, which vanishes in fp32.
template <int BM, int BN>
constexpr int stage_bytes() { return (BM + BN) * 128; }
template <int BM, int BN, int WGM, int WGN>
constexpr int tile_smem() {
  constexpr int epi = WGM * WGN * 32 * (BN / WGN + 4) * 4, st = 2 * stage_bytes<BM, BN>();
  return epi > st ? epi : st;
}

template <typename ST, int KIND, int ACT, int BM, int BN, int WGM, int WGN>
__global__ void __launch_bounds__(WGM * WGN * 64) mx_tile_kernel(const MxProblem p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int NW = WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, RM = WTM / 32, RN = WTN / 32;
  constexpr int IA = BM / 8 / NW, IB = BN / 8 / NW;  // LDS-DMA instructions (8 rows each) per wave and step
  constexpr int STAGE = stage_bytes<BM, BN>();
  static_assert(IA * 8 * NW == BM && IB * 8 * NW == BN && RM >= 1 && RN >= 1, "tile / waves");

  // workgroup b runs on XCD b % 8: consecutive tiles per XCD, which share rows of A
  const int tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
  const int b = blockIdx.x, per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = b & 7;
  const int t = xcd * per + (xcd < rem ? xcd : rem) + (b >> 3);
  // supertiles of 8 x 4: the 32 tiles an XCD runs at once read 8 row blocks of A and 4 of B
  const int band = t / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, w8 = t - band * 8 * tn;
  const int cs = w8 / (rows * 4), cols = tn - cs * 4 < 4 ? tn - cs * 4 : 4, w2 = w8 - cs * rows * 4;
  const int m0 = (band * 8 + w2 / cols) * BM, n0 = (cs * 4 + w2 % cols) * BN;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WGN, wn = w % WGN, lr = lane & 31, lk = lane >> 5;
  const int M = p.M, N = p.N, G = p.groups, steps = (G + 1) >> 1;
  const unsigned rb = (unsigned)G * 64u;  // bytes of a packed row (codes of a matrix: below 2^30 bytes)

  // LDS-DMA sources: instruction q of this wave fills rows (q NW + w) 8 .. + 7
  unsigned oa[IA], ob[IB], half[2] = {0u, 0u};
#pragma unroll
  for (int q = 0; q < (IA > IB ? IA : IB); ++q) {
    const int r = (q * NW + w) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
    if (q < IA) oa[q] = (unsigned)(m0 + r < M ? m0 + r : M - 1) * rb + (unsigned)c * 16u;
    if (q < IB) ob[q] = (unsigned)(n0 + r < N ? n0 + r : N - 1) * rb + (unsigned)c * 16u;
    if (q < 2) half[q] = c >= 4 ? 64u : 0u;  // (parity of the block's index alone decides c)
  }
  // (buffer loads: a 32-bit offset per lane, the step's as a scalar; the host keeps codes below 2^30 bytes)
  const Rsrc ga(p.a, (unsigned)M * rb), gb(p.b, (unsigned)N * rb);
  const Rsrc gas(p.as, (unsigned)M * (unsigned)G * 4u), gbs(p.bs, (unsigned)N * (unsigned)G * 4u);
  auto issue = [&](int kt, unsigned char* st) {
    // half a step: chunks 4 .. 7 read chunks 0 .. 3 again
    const bool cut = 2 * kt + 1 >= G;
    const unsigned back[2] = {cut ? half[0] : 0u, cut ? half[1] : 0u};
#pragma unroll
    for (int q = 0; q < IA; ++q) ga.to_lds(st + (q * NW + w) * 1024, oa[q] - back[q & 1], (unsigned)kt * 128u);
#pragma unroll
    for (int q = 0; q < IB; ++q) gb.to_lds(st + BM * 128 + (q * NW + w) * 1024, ob[q] - back[q & 1], (unsigned)kt * 128u);
  };
  // scale dwords of this lane's rows at group 2 kt + lk (0 past the end)
  unsigned ra[RM], rn[RN];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int m = m0 + wm * WTM + i * 32 + lr;
    ra[i] = (unsigned)(m < M ? m : M - 1) * 4u + (unsigned)(lk * M) * 4u;
  }
#pragma unroll
  for (int j = 0; j < RN; ++j) {
    const int n = n0 + wn * WTN + j * 32 + lr;
    rn[j] = (unsigned)(n < N ? n : N - 1) * 4u + (unsigned)(lk * N) * 4u;
  }
  auto scales = [&](int kt, unsigned (&sa)[RM], unsigned (&sb)[RN]) {
    const unsigned past = 2 * kt + lk < G ? 0u : 0x80000000u;  // past the last group: beyond the buffer, 0
#pragma unroll
    for (int i = 0; i < RM; ++i) sa[i] = gas.load(ra[i] | past, (unsigned)(2 * kt * M) * 4u);
#pragma unroll
    for (int j = 0; j < RN; ++j) sb[j] = gbs.load(rn[j] | past, (unsigned)(2 * kt * N) * 4u);
  };

  f32x16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;

  const int sw = (lr >> 1) & 7;
  auto frag = [&](const unsigned char* blk, int row0, int s) -> i32x4 {
    return *reinterpret_cast<const i32x4*>(blk + (row0 + lr) * 128 + (((lk * 4 + s) ^ sw) << 4));
  };
  unsigned sa[RM], sb[RN], na[RM], nb[RN];
  scales(0, sa, sb);
  issue(0, smem);
#pragma unroll 1
  for (int kt = 0; kt < steps; ++kt) {
    // this wave's loads of step kt have landed; the barrier says so of everybody's, and
    // that everybody is done with the other stage
    // (vmcnt 0, as a builtin: the compiler then knows that the scales are there too)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // (scales first: they are waited for at the end of this step, the codes at the start of the next)
    scales(kt + 1, na, nb);
    if (kt + 1 < steps) issue(kt + 1, smem + ((kt + 1) & 1) * STAGE);
    const unsigned char* sta = smem + (kt & 1) * STAGE;
    const unsigned char* stb = sta + BM * 128;
    i32x4 fa[2][RM], fb[2][RN];
#pragma unroll
    for (int j = 0; j < RN; ++j) fb[0][j] = frag(stb, wn * WTN + j * 32, 0);
#pragma unroll
    for (int i = 0; i < RM; ++i) fa[0][i] = frag(sta, wm * WTM + i * 32, 0);
    __builtin_amdgcn_sched_barrier(0);
    auto slice = [&](auto SV) {
      constexpr int S = decltype(SV)::value, cur = S & 1, nxt = cur ^ 1;
      if constexpr (S < 3) {
#pragma unroll
        for (int j = 0; j < RN; ++j) fb[nxt][j] = frag(stb, wn * WTN + j * 32, S + 1);
#pragma unroll
        for (int i = 0; i < RM; ++i) fa[nxt][i] = frag(sta, wm * WTM + i * 32, S + 1);
      }
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = mma<S>(fb[cur][j], sb[j], fa[cur][i], sa[i], acc[i][j]);
      if constexpr (S < 3) {
        // one LDS read between consecutive products, as far as the reads go
#pragma unroll
        for (int q = 0; q < RM * RN; ++q) {
          if (q < RM + RN) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    slice(std::integral_constant<int, 0>{});
    slice(std::integral_constant<int, 1>{});
    slice(std::integral_constant<int, 2>{});
    slice(std::integral_constant<int, 3>{});
#pragma unroll
    for (int i = 0; i < RM; ++i) sa[i] = na[i];
#pragma unroll
    for (int j = 0; j < RN; ++j) sb[j] = nb[j];
  }

  // Epilogue, 32 rows of the wave's tile at a time through its own part of the
  // LDS: rows of WTN + 4 floats (16 rows a column of banks apart), then walked
  // row by row, so that every global access is a run of 4-column groups.
  __syncthreads();
  constexpr int LDE = WTN + 4, LPR = WTN / 4, RPP = 64 / LPR, PASSES = 32 / RPP;
  float* es = reinterpret_cast<float*>(smem) + w * 32 * LDE;
  const int er = lane / LPR, ec = (lane % LPR) * 4, n = n0 + wn * WTN + ec;
#pragma unroll 1
  for (int i = 0; i < RM; ++i) {
    const int mb = m0 + wm * WTM + i * 32;
    float in[PASSES][4], e[PASSES][4];
#pragma unroll
    for (int u = 0; u < PASSES; ++u)
      if (mb + u * RPP + er < M && n < N) inputs4<ST, KIND>(p, mb + u * RPP + er, n, in[u], e[u]);
#pragma unroll
    for (int ii = 0; ii < RM; ++ii)
      if (ii == i) {
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
          for (int q = 0; q < 16; q += 4)
            *reinterpret_cast<float4*>(es + lr * LDE + j * 32 + 2 * q + 4 * lk) =
                make_float4(acc[ii][j][q], acc[ii][j][q + 1], acc[ii][j][q + 2], acc[ii][j][q + 3]);
      }
    // (the wave's own LDS accesses complete in order; the fence keeps the compiler from reordering them)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
      const int m = mb + u * RPP + er;
      const float4 t4 = *reinterpret_cast<const float4*>(es + (u * RPP + er) * LDE + ec);
      const float c[4] = {t4.x, t4.y, t4.z, t4.w};
      float o[4];
      if (m < M && n < N) {
        finish4<KIND, ACT>(c, in[u], e[u], p.scal, o);
        put4(reinterpret_cast<ST*>(p.out) + (long long)m * N + n, p.vec != 0, N - n, o);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
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

template <typename ST, int KIND, int ACT>
hipError_t run_product(const MxProblem& p, hipStream_t s) {
  const long long t256 = ((p.M + 255LL) / 256) * ((p.N + 255LL) / 256), t128 = ((p.M + 127LL) / 128) * ((p.N + 127LL) / 128);
  if (t256 >= 192) return run_tile<ST, KIND, ACT, 256, 256, 2, 2>(p, s);
  if (t128 >= 64) return run_tile<ST, KIND, ACT, 128, 128, 2, 2>(p, s);
  const long long tiles = ((p.M + 31LL) / 32) * ((p.N + 31LL) / 32);
  const int waves = p.groups < 4 ? 4 : p.groups < DIRECT_WAVES ? p.groups : DIRECT_WAVES;
  hipLaunchKernelGGL((mx_direct_kernel<ST, KIND, ACT>), dim3((unsigned)tiles), dim3(waves * 64), 0, s, p);
  return hipGetLastError();
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
