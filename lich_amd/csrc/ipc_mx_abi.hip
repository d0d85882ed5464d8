// ipc_mx_abi.hip - extern "C" entry points of the microscaled operators
// (declared in include/ipc_hip.h), with the argument checks of ipc_abi.hip:
// everything is refused on the host, before any HIP call.
#include "ipc_abi_check.h"
#include "ipc_launch.h"
#include "ipc_mx.h"

using namespace ipc;
using namespace ipc::abi;

namespace {

int check_format(int format) {
  if (format != IPC_MX_FP4 && format != IPC_MX_INT8) return fail(IPC_ERR_DTYPE, "unknown microscaled format %d", format);
  return ok();
}

// A packed matrix, padding included, stays below 2^31 values (32-bit offsets of
// its codes and scales in the kernels).
int check_packed(long long rows, int n, int format) {
  if (rows < 1 || n < 1) return fail(IPC_ERR_SHAPE, "dimensions must be >= 1 (%lld rows of %d)", rows, n);
  if (rows * mx_groups(n) * MX_GROUP > kMaxElems)
    return fail(IPC_ERR_SHAPE, "packed matrix too large (%lld rows of %d values, padded to a multiple of %d)", rows, n, MX_GROUP);
  return ok();
}

int check_codes(const void* codes, const void* scales, const char* name) {
  if (!codes || !scales) return fail(IPC_ERR_NULL, "%s is NULL", name);
  if (!al16(codes) || reinterpret_cast<uintptr_t>(scales) % 4)
    return fail(IPC_ERR_ALIGN, "%s needs codes aligned to 16 bytes and scales aligned to 4", name);
  return ok();
}

// Bytes of caller workspace that ipc_mx_predict uses: for f(X) evaluated once, which
// pays for its launch from five samples on.  MI355X, bf16, us, without / with: 64 x
// 784 8 samples 6.3 / 6.0; 4096 x 4096 8 relu 13.8 / 8.8, 64 51 / 14.7; 8192 x 8192 4 relu
// 12.1 / 15.0, gelu 16.2 / 15.3, 8 48 / 15.8, 64 191 / 40 (fp32 states the same way).
long long predict_workspace_need(int K, int B, int storage) {
  return B > 4 ? mx_predict_terms_bytes(K, B, storage) : 0;
}

constexpr int kPredictMost = 16 * 65535;  // 16 samples per grid row

int product(int kind, const void* a, const void* as, const char* a_name, const void* b, const void* bs,
            const char* b_name, void* out, const char* out_name, const void* aux, const char* aux_name, int M, int N,
            int K, float scal, int storage, int act, void* stream, const char* what) {
  TRY(check_dtypes(storage, storage));
  TRY(check_act(act));
  TRY(check_dims(M, K, N, 1));
  TRY(check_packed(M, K, IPC_MX_FP4));
  TRY(check_packed(N, K, IPC_MX_FP4));
  TRY(check_codes(a, as, a_name));
  TRY(check_codes(b, bs, b_name));
  const int es = elem_size(storage);
  TRY(check_ptr(out, out_name, es));
  if (aux_name) TRY(check_ptr(aux, aux_name, es));
  MxProblem p{};
  p.kind = kind; p.act = act;
  p.M = M; p.N = N; p.groups = mx_groups(K);
  p.a = static_cast<const uint8_t*>(a); p.as = static_cast<const uint32_t*>(as);
  p.b = static_cast<const uint8_t*>(b); p.bs = static_cast<const uint32_t*>(bs);
  p.out = out; p.aux = aux; p.scal = scal;
  p.vec = vec_ok(out, N, es) && (!aux || vec_ok(aux, N, es));
  return launch_rc(launch_mx_product(p, storage, (hipStream_t)stream), what);
}

}  // namespace

extern "C" {

long long ipc_mx_code_bytes(int rows, int n, int format) {
  if (check_format(format) != IPC_OK || check_packed(rows, n, format) != IPC_OK) return 0;
  return (long long)rows * mx_row_bytes(format, n);
}

long long ipc_mx_scale_bytes(int rows, int n) {
  if (check_packed(rows, n, IPC_MX_FP4) != IPC_OK) return 0;
  return (long long)rows * mx_groups(n) * 4;
}

int ipc_mx_quantize(const void* x, void* codes, void* scales, int R, int C, int axis, int format, int storage,
                    int act, void* stream) {
  TRY(check_dtypes(storage, storage));
  TRY(check_format(format));
  TRY(check_act(act));
  if (axis != 0 && axis != 1) return fail(IPC_ERR_CONFIG, "axis must be 0 or 1 (got %d)", axis);
  TRY(check_packed(axis == 1 ? R : C, axis == 1 ? C : R, format));
  TRY(check_ptr(x, "x", elem_size(storage)));
  TRY(check_codes(codes, scales, "the packed matrix"));
  return launch_rc(launch_mx_quantize(x, codes, scales, R, C, axis, format, storage, act, (hipStream_t)stream),
                   "ipc_mx_quantize");
}

int ipc_mx_dequantize(const void* codes, const void* scales, void* out, int R, int C, int format, int storage,
                      void* stream) {
  TRY(check_dtypes(storage, storage));
  TRY(check_format(format));
  TRY(check_packed(R, C, format));
  TRY(check_codes(codes, scales, "the packed matrix"));
  TRY(check_ptr(out, "out", elem_size(storage)));
  return launch_rc(launch_mx_dequantize(codes, scales, out, R, C, format, storage, IPC_ACT_IDENTITY, (hipStream_t)stream),
                   "ipc_mx_dequantize");
}

int ipc_mx_pred_err(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales,
                    const void* x_lower, void* e, int M, int K, int B, int storage, void* stream) {
  return product(KIND_PRED, w_codes, w_scales, "w", x_codes, x_scales, "x_upper", e, "e", x_lower, "x_lower", M, B, K,
                 0.0f, storage, IPC_ACT_IDENTITY, stream, "ipc_mx_pred_err");
}

int ipc_mx_forward(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out,
                   int M, int K, int B, int storage, void* stream) {
  return product(KIND_FWD, w_codes, w_scales, "w", x_codes, x_scales, "x_upper", out, "out", nullptr, nullptr, M, B, K,
                 0.0f, storage, IPC_ACT_IDENTITY, stream, "ipc_mx_forward");
}

int ipc_mx_infer_update(void* x, const void* e, const void* wt_codes, const void* wt_scales, const void* et_codes,
                        const void* et_scales, int M, int K, int B, float gamma, int storage, int act, void* stream) {
  return product(KIND_INFER, wt_codes, wt_scales, "w_lower", et_codes, et_scales, "e_lower", x, "x", e, "e", M, B, K,
                 gamma, storage, act, stream, "ipc_mx_infer_update");
}

int ipc_mx_weight_update(void* w, const void* e_codes, const void* e_scales, const void* a_codes,
                         const void* a_scales, int M, int K, int B, float alpha, int storage, void* stream) {
  return product(KIND_WEIGHT, e_codes, e_scales, "e", a_codes, a_scales, "x_upper", w, "w", nullptr, nullptr, M, K, B,
                 alpha, storage, IPC_ACT_IDENTITY, stream, "ipc_mx_weight_update");
}

long long ipc_mx_predict_workspace_bytes(int K, int B, int storage) {
  if (K < 1 || B < 1 || B > kPredictMost || storage < IPC_DT_F32 || storage > IPC_DT_BF16) return 0;
  return predict_workspace_need(K, B, storage);
}

int ipc_mx_predict(const void* x, const void* w_codes, const void* w_scales, void* out, int M, int K, int B,
                   int storage, int act, void* workspace, long long workspace_bytes, void* stream) {
  TRY(check_workspace(workspace, workspace_bytes));
  TRY(check_dtypes(storage, storage));
  TRY(check_act(act));
  TRY(check_dims(M, K, B, 1));
  TRY(check_packed(M, K, IPC_MX_FP4));
  if (B > kPredictMost) return fail(IPC_ERR_SHAPE, "ipc_mx_predict takes at most %d samples (got %d)", kPredictMost, B);
  TRY(check_ptr(x, "x", elem_size(storage)));
  TRY(check_codes(w_codes, w_scales, "w"));
  TRY(check_ptr(out, "out", elem_size(storage)));
  MxPredict p{};
  p.M = M; p.K = K; p.B = B; p.act = act;
  p.x = x; p.out = out;
  p.w = static_cast<const uint8_t*>(w_codes); p.ws = static_cast<const uint32_t*>(w_scales);
  const long long need = predict_workspace_need(K, B, storage);
  p.terms = need > 0 && workspace && workspace_bytes >= need ? workspace : nullptr;
  return launch_rc(launch_mx_predict(p, storage, (hipStream_t)stream), "ipc_mx_predict");
}

}  // extern "C"

namespace ipc {

hipError_t launch_mx_product(const MxProblem& p, int storage, hipStream_t s) {
  if (storage == DT_F32) return launch_mx_product_f32(p, s);
  if (storage == DT_F16) return launch_mx_product_f16(p, s);
  return launch_mx_product_bf16(p, s);
}

}  // namespace ipc
