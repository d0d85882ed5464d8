// ipc_mx.h - microscaled storage (OCP MX): layout, host structs and launchers.
//
// A packed matrix holds `rows` rows of `n` values, blocks of 32 consecutive
// values of a row sharing one power-of-two scale 2^(s - 127), s the block's
// scale byte (E8M0; 255 = the block holds an infinity or NaN and reads as NaN):
//
//   fp4   E2M1 elements 0 0.5 1 1.5 2 3 4 6 and their negatives, two a byte, the
//         lower value in the lower half; rows padded with zeros to a multiple of
//         128 values: codes [rows][mx_row_values / 2]
//   int8  value = code * 2^(s - 133), codes -127 .. 127; rows padded to a
//         multiple of 32 values: codes [rows][mx_row_values]
//   scales [ceil(n / 128)][rows][4] bytes: the four blocks of 128 values of a row
//         in one dword, the rows' dwords contiguous, so that the 32 rows a matrix
//         instruction takes come from one or two cache lines.
//
// The scale of a block follows its largest magnitude once that is rounded to
// the element's precision (so that no element exceeds the largest code by more
// than its own rounding): fp4 amax < 7 * 2^(s-127), int8 amax < 2 * 2^(s-127); at
// the top of the float range it stays finite and the elements saturate.
// Elements round to nearest, ties to the even code.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ipc {

enum { MX_FP4 = 0, MX_INT8 = 1 };
constexpr int MX_BLOCK = 32, MX_GROUP = 128;  // values per scale, per scale dword

// Values of a packed row of n, padding included.
inline long long mx_row_values(int format, int n) {
  const int unit = format == MX_FP4 ? MX_GROUP : MX_BLOCK;
  return ((long long)n + unit - 1) / unit * unit;
}
inline long long mx_row_bytes(int format, int n) {
  return format == MX_FP4 ? mx_row_values(format, n) / 2 : mx_row_values(format, n);
}
__host__ __device__ inline int mx_groups(int n) { return (int)(((long long)n + MX_GROUP - 1) / MX_GROUP); }
// Whether `run` values from column c of a row lie inside a matrix whose rows of n end
// `rows_left` rows from this one on (this one counted; 0 or less: none).  A row's end may
// be read past, into the rows after it: of narrow ones a run takes several.
__host__ __device__ inline bool mx_run_inside(int rows_left, int n, int c, int run) {
  return rows_left > 0 && c < n && (c + run <= n || rows_left * (long long)n >= c + run);
}

// Bytes of the buffer from `mis` bytes before element `first` of a tensor to its end,
// element `end`.  Loads take whole dwords (16-bit rows of any length), so their limit is
// rounded up to the one that holds the last element.  A store's is exact: it is all that
// keeps rows past the tensor's last one from the memory behind it.
__host__ __device__ inline long long mx_rows_bytes(long long first, long long end, int element, unsigned mis, bool store) {
  const long long bytes = end <= first ? 0 : (end - first) * element + mis;
  return store ? bytes : (bytes + 3) & ~3LL;
}

// Whether a tile epilogue's offsets from the first of 16 rows of N elements, rows past the
// tensor's last one and a tile's columns included, fit 32 bits: past them such a row's
// stores would come round to the tensor's start.
inline bool mx_rows_fit(long long N, int element) { return (15 * N + 256) * element < (1LL << 32); }

// axis 1: rows of x [R][C] are the packed rows; axis 0: its columns.
hipError_t launch_mx_quantize(const void* x, void* codes, void* scales, int R, int C, int axis, int format,
                              int storage, int act, hipStream_t s);
hipError_t launch_mx_dequantize(const void* codes, const void* scales, void* out, int R, int C, int format,
                                int storage, int act, hipStream_t s);  // f applied

// C[M][N] = sum over k of A4[m][k] B4[n][k], both fp4 with rows of `groups`
// groups of 128 values, and the epilogue of a kernel family (GemmKind).
struct MxProblem {
  int kind, act;
  int M, N, groups;
  const uint8_t* a; const uint32_t* as;  // codes [M][groups * 64], scales [groups][M]
  const uint8_t* b; const uint32_t* bs;  // codes [N][groups * 64], scales [groups][N]
  void* out;                             // [M][N]: E, OUT (written), X, W (updated)
  const void* aux;                       // [M][N]: X_lower (PRED), E (INFER)
  float scal;                            // gamma (INFER), alpha (WEIGHT)
  int vec;                               // out / aux allow 4-element accesses
};
hipError_t launch_mx_product(const MxProblem& p, int storage, hipStream_t s);
// per storage type, one translation unit each
hipError_t launch_mx_product_f32(const MxProblem& p, hipStream_t s);
hipError_t launch_mx_product_f16(const MxProblem& p, hipStream_t s);
hipError_t launch_mx_product_bf16(const MxProblem& p, hipStream_t s);

// OUT [M][B] = W4 f(X), X [K][B].
struct MxPredict {
  int M, K, B, act;
  const void* x;
  const uint8_t* w; const uint32_t* ws;
  void* out;
  void* terms;  // workspace of mx_predict_terms_bytes bytes for f(X), or nullptr
};
inline long long mx_predict_terms_bytes(int K, int B, int storage) {
  const long long rows = B < 16 ? B : (B + 15LL) / 16 * 16;
  return (storage == 0 ? 3LL : 2LL) * rows * mx_groups(K) * MX_GROUP * 2;
}
hipError_t launch_mx_predict(const MxPredict& p, int storage, hipStream_t s);

// The backward pass of a state kept in 8 bits as 16-bit products (ipc_ckpt_gemm.h):
// rows that start at multiples of 4 bytes (an even lda and ldb), operands below
// 2^31 bytes; CKPT_WEIGHT: rows of b readable and finite up to a multiple of 32.
struct CkptProblem {
  int M, N, K;
  const void* a; long long lda;  // elements
  const void* b; long long ldb;
  const void* x;                 // codes, scales and row bytes of X (CKPT_GRAD: [M][N])
  const void* xs;
  int x_row;
  void* out;                     // [M][N]
  float alpha;
  int vec;                       // out allows 4-element accesses
};
enum { CKPT_GRAD = 0, CKPT_WEIGHT = 1 };
hipError_t launch_ckpt_gemm(int mode, const CkptProblem& p, int operand, int act, hipStream_t s);
// Rows of two 16-bit matrices (nullptr: none) padded with zeros from na, nb to lda, ldb
// values, multiples of 8.
hipError_t launch_ckpt_pad(const void* a, void* pa, int rows_a, int na, int lda, const void* b, void* pb, int rows_b,
                           int nb, int ldb, hipStream_t s);
// On fp32 operands (ipc_ckpt_gemm32.h): rows of any length, operands below 2^31 bytes.
// CKPT_WEIGHT: b = f(X) in fp32, or nullptr: X from its codes x, xs, x_row.
hipError_t launch_ckpt_gemm32(int mode, const CkptProblem& p, int act, hipStream_t s);

}  // namespace ipc
