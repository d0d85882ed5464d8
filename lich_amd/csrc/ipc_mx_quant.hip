// ipc_mx_quant.hip - matrices into microscaled storage and back (gfx950).
//
// Both directions are one pass over the data, bound by HBM: each value is read
// once and each code and scale written once.  MI355X, fp32, 4096 x 4096, fp4: columns
// 18.6 us from memory (76 MB, 4.1 TB/s; a copy runs at 5.2), 14.3 from the caches, back
// 12.8; bf16, 4096 x 1024, int8: rows 4.0 us, back 3.5 (13 MB, 3-4 TB/s, launches
// included; one of a few KB takes 2.7-2.9).
#include "ipc_launch.h"
#include "ipc_mx_device.h"

namespace ipc {
namespace {

// The row kernels: a workgroup takes 256 values (two groups, so that the fp4
// codes it stores are whole 128-byte lines) of a few rows, a lane EPL consecutive
// ones (16 bytes), in one pass or four whose loads are issued together.
constexpr int WIDTH = 2 * MX_GROUP;
template <typename ST> constexpr int EPL = 16 / (int)sizeof(ST);           // values per lane
template <typename ST> constexpr int ROW_LANES = WIDTH / EPL<ST>;          // lanes per row
template <typename ST> constexpr int PASS_ROWS = 256 / ROW_LANES<ST>;      // rows per pass
template <typename ST, int PASSES> constexpr int TILE_ROWS = PASSES * PASS_ROWS<ST>;  // rows per workgroup

// Packed rows are the rows of x.  A block's lanes (4, or 8 of fp32) sit side by
// side: its largest magnitude comes from exchanges within them.
template <typename ST, int FMT, int PASSES>
__global__ void __launch_bounds__(256) mx_quant_rows_kernel(const ST* __restrict__ x, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, int R, int C,
                                                            int row_bytes, int spans, int act) {
  constexpr int E = EPL<ST>;
  const int c = blockIdx.x % spans * WIDTH + threadIdx.x % ROW_LANES<ST> * E;
  const int r0 = blockIdx.x / spans * TILE_ROWS<ST, PASSES> + threadIdx.x / ROW_LANES<ST>;
  const int groups = mx_groups(C), kg = c / MX_GROUP;
  float v[PASSES][E];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * PASS_ROWS<ST>;
    const ST* p = x + (long long)r * C + c;
#pragma unroll
    for (int i = 0; i < E; ++i) v[u][i] = 0.0f;
    if (mx_run_inside(R - r, C, c, E)) {  // (past the row's end: the next rows' values, cleared below)
      mx::load_run<ST, E>(p, v[u]);
    } else if (r < R) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (c + i < C) v[u][i] = to_f32(p[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int r = r0 + u * PASS_ROWS<ST>;
    activate<E>(act, v[u]);
    if (c + E > C) {  // (f(0) need not be 0: padding stays zero)
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (c + i >= C) v[u][i] = 0.0f;
    }
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) m = max(m, mx::abs_bits(v[u][i]));
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));   // quad lanes 1 0 3 2
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));   // quad lanes 2 3 0 1
    if (E == 4) m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));  // lanes 7 .. 0 of 8
    if (r >= R || kg >= groups) continue;
    const unsigned s = mx::scale_byte<FMT>(m);
    uint8_t* row = codes + (long long)r * row_bytes;
    if constexpr (FMT == MX_FP4) {
      if constexpr (E == 8) *reinterpret_cast<unsigned*>(row + c / 2) = mx::fp4_codes<8>(v[u], s);
      else *reinterpret_cast<unsigned short*>(row + c / 2) = (unsigned short)mx::fp4_codes<4>(v[u], s);
    } else if (c < row_bytes) {
      unsigned q[E / 4];
#pragma unroll
      for (int h = 0; h < E / 4; ++h)
        q[h] = mx::int8_codes4(v[u][4 * h], v[u][4 * h + 1], v[u][4 * h + 2], v[u][4 * h + 3], s);
      if constexpr (E == 8) *reinterpret_cast<uint2*>(row + c) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<unsigned*>(row + c) = q[0];
    }
    if (c % MX_BLOCK == 0) scales[((long long)kg * R + r) * 4 + (c / MX_BLOCK & 3)] = (uint8_t)s;
  }
}

// Packed rows are the columns of x [K][N].  A workgroup stages 128 k-rows of 32
// dwords (128 bytes of a row: 32 fp32 or 64 16-bit columns) in LDS with 16-byte
// loads; then each thread owns a dword column and one of the eight half blocks, the
// other half in the neighbouring lane: 8 (fp4) or 16 bytes of a packed row, the eight of
// a row side by side.  Dword w of k-row k (half block b = k / 16) lies in row k ^ (b & 1) at
// w + 8 (b / 2) (mod 32): a wave reads 8 dwords of each of the 8 from 64 different
// banks.  Whole blocks a thread (no exchange, half as many workgroups, twice the LDS) were
// slower but for the largest, us from memory, half / whole: fp4, fp32 784 x 128 2.7 / 4.6,
// 4096 x 4096 18.6 / 20.5, bf16 4096 x 1024 5.4 / 5.9, 8192 x 2048 11.8 / 13.1, 8192 x 8192 42.5 /
// 40.9; from the caches that one 27.8 / 32.5, and int8 35 / 42.
template <typename ST, int FMT>
__global__ void __launch_bounds__(256) mx_quant_cols_kernel(const ST* __restrict__ x, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, int K, int N,
                                                            int row_bytes, int tiles, int act) {
  constexpr int VPD = 4 / sizeof(ST);  // columns per dword
  constexpr int COLS = 32 * VPD, VEC = 16 / sizeof(ST);
  constexpr int V = MX_BLOCK / 2, LOADS = MX_GROUP / 32;  // values of a thread's run, its 16-byte loads
  __shared__ __align__(16) unsigned tile[MX_GROUP * 32];
  const int n0 = blockIdx.x % tiles * COLS, k0 = blockIdx.x / tiles * MX_GROUP;  // (whole rows at once)
  const int tid = threadIdx.x;
  {
    typedef typename mx::Run<ST, VEC>::V Vec;
    const int j = tid & 7, n = n0 + j * VEC;
    Vec v[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int k = k0 + u * 32 + (tid >> 3);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = (ST)0.0f;
      const ST* p = x + (long long)k * N + n;
      if (mx_run_inside(K - k, N, n, VEC)) {  // (past the row's end: the next rows' values, never stored)
        v[u] = reinterpret_cast<const typename mx::Run<ST, VEC>::U*>(p)->v;
      } else if (k < K) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (n + i < N) v[u][i] = p[i];
      }
    }
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int k = u * 32 + (tid >> 3), run = k / V;
      *reinterpret_cast<Vec*>(&tile[(k ^ (run & 1)) * 32 + ((j * 4 + 8 * (run >> 1)) & 31)]) = v[u];
    }
  }
  __syncthreads();
  const int w = tid >> 3, run = tid & 7;
  const int k = k0 + run * V, left = K - k;  // the run's first k; values of it
  unsigned d[V];
  const unsigned* at = &tile[run * V * 32 + ((w + 8 * (run >> 1)) & 31)];
  const unsigned *even = at + (run & 1) * 32, *odd = at - (run & 1) * 32;  // rows i and i ^ 1
#pragma unroll
  for (int i = 0; i < V; ++i) d[i] = (i & 1 ? odd : even)[i * 32];
  const int kg = k0 / MX_GROUP;
#pragma unroll
  for (int c = 0; c < VPD; ++c) {
    const int n = n0 + w * VPD + c;
    if (n >= N) break;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (VPD == 1) v[i] = __builtin_bit_cast(float, d[i]);
      else v[i] = h2f(c == 0 ? d[i] & 0xffffu : d[i] >> 16, (ST*)nullptr);
    }
    activate<V>(act, v);
    if (left < V) {  // (f(0) need not be 0: padding stays zero)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i >= left) v[i] = 0.0f;
    }
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, mx::abs_bits(v[i]));
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad lanes 1 0 3 2
    const unsigned s = mx::scale_byte<FMT>(m);
    if (!(run & 1)) scales[((long long)kg * N + n) * 4 + (k / MX_BLOCK & 3)] = (uint8_t)s;
    uint8_t* row = codes + (long long)n * row_bytes;
    if constexpr (FMT == MX_FP4) {
      const unsigned lo = mx::fp4_codes<8>(*reinterpret_cast<const float (*)[8]>(&v[0]), s);
      const unsigned hi = mx::fp4_codes<8>(*reinterpret_cast<const float (*)[8]>(&v[8]), s);
      *reinterpret_cast<uint2*>(row + k / 2) = make_uint2(lo, hi);
    } else if (k < row_bytes) {
      unsigned q[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) q[h] = mx::int8_codes4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3], s);
      *reinterpret_cast<uint4*>(row + k) = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
}

// f of packed rows into out [R][C], lanes as in mx_quant_rows_kernel.
template <typename ST, int FMT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, ST* __restrict__ out,
                                                         int R, int C, int row_bytes, int spans, int act) {
  constexpr int E = EPL<ST>;
  const int c = blockIdx.x % spans * WIDTH + threadIdx.x % ROW_LANES<ST> * E;
  const int r = blockIdx.x / spans * PASS_ROWS<ST> + threadIdx.x / ROW_LANES<ST>;
  if (c >= C || r >= R) return;
  const uint8_t* row = codes + (long long)r * row_bytes;
  const unsigned s = scales[((long long)(c / MX_GROUP) * R + r) * 4 + (c / MX_BLOCK & 3)];
  float v[E];
  if constexpr (FMT == MX_FP4) {
    unsigned q;
    if constexpr (E == 8) q = *reinterpret_cast<const unsigned*>(row + c / 2);
    else q = *reinterpret_cast<const unsigned short*>(row + c / 2);
    mx::fp4_values<E>(q, s, v);
  } else {
    unsigned q[E / 4];
    if constexpr (E == 8) {
      const uint2 t = *reinterpret_cast<const uint2*>(row + c);
      q[0] = t.x; q[1] = t.y;
    } else {
      q[0] = *reinterpret_cast<const unsigned*>(row + c);
    }
    const float unit = mx::int8_scale(s);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)mx::sext8(q[i / 4], i & 3) * unit;
  }
  activate<E>(act, v);
  ST* p = out + (long long)r * C + c;
  if (c + E <= C) {
    mx::store_run<ST, E>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (c + i < C) p[i] = cvt<ST>(v[i]);
  }
}

// Four passes a workgroup for large fp32 matrices, else one: shorter code, which small
// calls spend their time to fetch, and more workgroups.  MI355X, us, one / four: fp32 fp4
// 784 x 128 2.9 / 3.3, 2048 x 1024 3.2 / 3.3, 4096 x 2048 7.4 / 6.0; bf16 int8 784 x 128 2.9 /
// 5.0, 4096 x 1024 4.0 / 4.8, 8192 x 8192 33 / 39.
template <typename ST, int FMT>
hipError_t quantize(const void* x, void* codes, void* scales, int R, int C, int axis, int act, hipStream_t s) {
  const int rows = axis == 1 ? R : C, n = axis == 1 ? C : R;
  const int spans = axis == 0 ? mx_groups(n) : (mx_groups(n) + 1) / 2;
  const long long four = (rows + TILE_ROWS<ST, 4> - 1LL) / TILE_ROWS<ST, 4>;
  const bool passes = sizeof(ST) == 4 && four * spans >= 1024;
  const long long tiles = axis == 0 ? (rows * (long long)sizeof(ST) + 127) / 128
                          : passes  ? four : (rows + TILE_ROWS<ST, 1> - 1LL) / TILE_ROWS<ST, 1>;
  const long long blocks = spans * tiles;
  const int row_bytes = (int)mx_row_bytes(FMT, n);
  auto kernel = axis == 0 ? mx_quant_cols_kernel<ST, FMT> : mx_quant_rows_kernel<ST, FMT, 1>;
  if constexpr (sizeof(ST) == 4) {
    if (axis == 1 && passes) kernel = mx_quant_rows_kernel<ST, FMT, 4>;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, s, static_cast<const ST*>(x),
                     static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), R, C, row_bytes,
                     axis == 1 ? spans : (int)tiles, act);
  return hipGetLastError();
}

template <typename ST, int FMT>
hipError_t dequantize(const void* codes, const void* scales, void* out, int R, int C, int act, hipStream_t s) {
  const int spans = (mx_groups(C) + 1) / 2;
  const long long blocks = spans * ((R + PASS_ROWS<ST> - 1LL) / PASS_ROWS<ST>);
  hipLaunchKernelGGL((mx_dequant_kernel<ST, FMT>), dim3((unsigned)blocks), dim3(256), 0, s,
                     static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<ST*>(out), R, C,
                     (int)mx_row_bytes(FMT, C), spans, act);
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
