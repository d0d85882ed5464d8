// ipc_mx_quant.hip - matrices into microscaled storage and back (gfx950).
//
// Both directions are one pass over the data, bound by HBM: each value is read
// once and each code and scale written once.
#include "ipc_launch.h"
#include "ipc_mx_device.h"

namespace ipc {
namespace {

constexpr int TILE_ROWS = 64;  // packed rows a workgroup of the row kernels takes, 128 values of each

// Packed rows are the rows of x.  16 lanes take the 128 values of a row, 8 each
// (16-byte loads), 4 lanes a block: its largest magnitude comes from two
// exchanges within a quad.  The workgroup's 64 rows go through in 4 passes
// whose loads are issued together.
template <typename ST, int FMT>
__global__ void __launch_bounds__(256) mx_quant_rows_kernel(const ST* __restrict__ x, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, int R, int C,
                                                            int row_bytes, int groups, int act) {
  const int kg = blockIdx.x % groups, r0 = blockIdx.x / groups * TILE_ROWS;
  const int tid = threadIdx.x, sub = tid & 15, c = kg * MX_GROUP + sub * 8;
  constexpr int PASSES = TILE_ROWS / 16;
  float v[PASSES][8];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * 16 + (tid >> 4);
    const ST* p = x + (long long)r * C + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
    if (r < R && c + 8 <= C) {
      mx::load8(p, v[u]);
    } else if (r < R) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) v[u][i] = to_f32(p[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * 16 + (tid >> 4);
    activate<8>(act, v[u]);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i >= C) v[u][i] = 0.0f;  // (f(0) need not be 0: padding stays zero)
      m = max(m, mx::abs_bits(v[u][i]));
    }
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad lanes 1 0 3 2
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));  // quad lanes 2 3 0 1
    if (r >= R) continue;
    const unsigned s = mx::scale_byte<FMT>(m);
    uint8_t* row = codes + (long long)r * row_bytes;
    if constexpr (FMT == MX_FP4) {
      *reinterpret_cast<unsigned*>(row + c / 2) = mx::fp4_codes8(v[u], s);
    } else if (c < row_bytes) {
      uint2 q;
      q.x = mx::int8_codes4(v[u][0], v[u][1], v[u][2], v[u][3], s);
      q.y = mx::int8_codes4(v[u][4], v[u][5], v[u][6], v[u][7], s);
      *reinterpret_cast<uint2*>(row + c) = q;
    }
    if ((sub & 3) == 0) scales[((long long)kg * R + r) * 4 + (sub >> 2)] = (uint8_t)s;
  }
}

// Packed rows are the columns of x [K][N].  A workgroup stages 128 k-rows of 64
// dwords (64 fp32 or 128 16-bit columns) in LDS with 16-byte loads; then each
// thread owns a dword column and one of the four blocks: its 32 values are in
// its registers, so the block's scale needs no exchange, and its codes are 16
// (fp4) or 32 bytes of a packed row, the four blocks of a row side by side.
// Dword w of k-row k lies at w + 16 * (k / 32) (mod 64): a wave reads 16 dwords
// of each of the 4 blocks from 64 different banks.
template <typename ST, int FMT>
__global__ void __launch_bounds__(256) mx_quant_cols_kernel(const ST* __restrict__ x, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, int K, int N,
                                                            int row_bytes, int groups, int act) {
  constexpr int VPD = 4 / sizeof(ST);  // columns per dword
  constexpr int COLS = 64 * VPD, VEC = 16 / sizeof(ST);
  __shared__ __align__(16) unsigned tile[MX_GROUP * 64];
  const int kg = blockIdx.x % groups, n0 = blockIdx.x / groups * COLS, k0 = kg * MX_GROUP;
  const int tid = threadIdx.x;
  {
    typedef typename mx::Run<ST, VEC>::V V;
    const int j = tid & 15, n = n0 + j * VEC;
    V v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = k0 + u * 16 + (tid >> 4);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = (ST)0.0f;
      const ST* p = x + (long long)k * N + n;
      if (k < K && n + VEC <= N) {
        v[u] = reinterpret_cast<const typename mx::Run<ST, VEC>::U*>(p)->v;
      } else if (k < K) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (n + i < N) v[u][i] = p[i];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = u * 16 + (tid >> 4);
      *reinterpret_cast<V*>(&tile[k * 64 + ((j * 4 + 16 * (k >> 5)) & 63)]) = v[u];
    }
  }
  __syncthreads();
  const int w = tid >> 2, blk = tid & 3;
  unsigned d[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) d[i] = tile[(blk * 32 + i) * 64 + ((w + 16 * blk) & 63)];
  const int left = K - k0 - blk * 32;  // values of this block
#pragma unroll
  for (int c = 0; c < VPD; ++c) {
    const int n = n0 + w * VPD + c;
    if (n >= N) break;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if constexpr (VPD == 1) v[i] = __builtin_bit_cast(float, d[i]);
      else v[i] = h2f(c == 0 ? d[i] & 0xffffu : d[i] >> 16, (ST*)nullptr);
    }
    activate<32>(act, v);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i >= left) v[i] = 0.0f;
      m = max(m, mx::abs_bits(v[i]));
    }
    const unsigned s = mx::scale_byte<FMT>(m);
    scales[((long long)kg * N + n) * 4 + blk] = (uint8_t)s;
    uint8_t* row = codes + (long long)n * row_bytes;
    if constexpr (FMT == MX_FP4) {
      unsigned q[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float (&t)[8] = *reinterpret_cast<const float (*)[8]>(&v[h * 8]);
        q[h] = mx::fp4_codes8(t, s);
      }
      *reinterpret_cast<uint4*>(row + kg * 64 + blk * 16) = make_uint4(q[0], q[1], q[2], q[3]);
    } else if (k0 + blk * 32 < row_bytes) {
      unsigned q[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) q[h] = mx::int8_codes4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3], s);
      uint4* o = reinterpret_cast<uint4*>(row + k0 + blk * 32);
      o[0] = make_uint4(q[0], q[1], q[2], q[3]);
      o[1] = make_uint4(q[4], q[5], q[6], q[7]);
    }
  }
}

// f of packed rows into out [R][C], 8 values a lane as in mx_quant_rows_kernel.
template <typename ST, int FMT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, ST* __restrict__ out,
                                                         int R, int C, int row_bytes, int groups, int act) {
  const int kg = blockIdx.x % groups, r0 = blockIdx.x / groups * TILE_ROWS;
  const int tid = threadIdx.x, sub = tid & 15, c = kg * MX_GROUP + sub * 8;
  if (c >= C) return;
  constexpr int PASSES = TILE_ROWS / 16;
  uint2 q[PASSES];
  unsigned s[PASSES];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * 16 + (tid >> 4);
    q[u] = make_uint2(0, 0);
    s[u] = 0;
    if (r < R) {
      const uint8_t* row = codes + (long long)r * row_bytes;
      if constexpr (FMT == MX_FP4) q[u].x = *reinterpret_cast<const unsigned*>(row + c / 2);
      else q[u] = *reinterpret_cast<const uint2*>(row + c);
      s[u] = scales[((long long)kg * R + r) * 4 + (sub >> 2)];
    }
  }
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * 16 + (tid >> 4);
    if (r >= R) continue;
    float v[8];
    const float unit = mx::int8_scale(s[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (FMT == MX_FP4) v[i] = mx::fp4_value(q[u].x >> (4 * i) & 15u, s[u]);
      else v[i] = (float)mx::sext8(i < 4 ? q[u].x : q[u].y, i & 3) * unit;
    }
    activate<8>(act, v);
    ST* p = out + (long long)r * C + c;
    if (c + 8 <= C) {
      mx::store8(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) p[i] = cvt<ST>(v[i]);
    }
  }
}

template <typename ST, int FMT>
hipError_t quantize(const void* x, void* codes, void* scales, int R, int C, int axis, int act, hipStream_t s) {
  const int rows = axis == 1 ? R : C, n = axis == 1 ? C : R;
  const int groups = mx_groups(n), per = axis == 1 ? TILE_ROWS : 256 / (int)sizeof(ST);
  const long long blocks = (long long)groups * ((rows + (long long)per - 1) / per);
  const int row_bytes = (int)mx_row_bytes(FMT, n);
  if (axis == 1)
    hipLaunchKernelGGL((mx_quant_rows_kernel<ST, FMT>), dim3((unsigned)blocks), dim3(256), 0, s,
                       static_cast<const ST*>(x), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), R, C,
                       row_bytes, groups, act);
  else
    hipLaunchKernelGGL((mx_quant_cols_kernel<ST, FMT>), dim3((unsigned)blocks), dim3(256), 0, s,
                       static_cast<const ST*>(x), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), R, C,
                       row_bytes, groups, act);
  return hipGetLastError();
}

template <typename ST, int FMT>
hipError_t dequantize(const void* codes, const void* scales, void* out, int R, int C, int act, hipStream_t s) {
  const int groups = mx_groups(C);
  const long long blocks = (long long)groups * ((R + (long long)TILE_ROWS - 1) / TILE_ROWS);
  hipLaunchKernelGGL((mx_dequant_kernel<ST, FMT>), dim3((unsigned)blocks), dim3(256), 0, s,
                     static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<ST*>(out), R,
                     C, (int)mx_row_bytes(FMT, C), groups, act);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantize(const void* x, void* codes, void* scales, int R, int C, int axis, int format,
                              int storage, int act, hipStream_t s) {
  const bool four = format == MX_FP4;
  switch (storage) {
    case DT_F32:
      return four ? quantize<float, MX_FP4>(x, codes, scales, R, C, axis, act, s)
                  : quantize<float, MX_INT8>(x, codes, scales, R, C, axis, act, s);
    case DT_F16:
      return four ? quantize<f16, MX_FP4>(x, codes, scales, R, C, axis, act, s)
                  : quantize<f16, MX_INT8>(x, codes, scales, R, C, axis, act, s);
    default:
      return four ? quantize<bf16, MX_FP4>(x, codes, scales, R, C, axis, act, s)
                  : quantize<bf16, MX_INT8>(x, codes, scales, R, C, axis, act, s);
  }
}

hipError_t launch_mx_dequantize(const void* codes, const void* scales, void* out, int R, int C, int format,
                                int storage, int act, hipStream_t s) {
  const bool four = format == MX_FP4;
  switch (storage) {
    case DT_F32:
      return four ? dequantize<float, MX_FP4>(codes, scales, out, R, C, act, s)
                  : dequantize<float, MX_INT8>(codes, scales, out, R, C, act, s);
    case DT_F16:
      return four ? dequantize<f16, MX_FP4>(codes, scales, out, R, C, act, s)
                  : dequantize<f16, MX_INT8>(codes, scales, out, R, C, act, s);
    default:
      return four ? dequantize<bf16, MX_FP4>(codes, scales, out, R, C, act, s)
                  : dequantize<bf16, MX_INT8>(codes, scales, out, R, C, act, s);
  }
}

}  // namespace ipc
