// ipc_abi_check.h - argument checks shared by the entry points of the C ABI.
//
// Each returns IPC_OK or a negative code with the calling thread's message set
// (ipc_last_error); all of them run on the host before any HIP call.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

#include "../../include/ipc_hip.h"

namespace ipc {
namespace abi {

// Sets the thread's message and returns `code` (ipc_abi.hip).
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

inline int ok() { return IPC_OK; }

constexpr long long kMaxElems = (1LL << 31) - 1;  // per-matrix element count (32-bit tile indices)

inline int elem_size(int dt) { return dt == IPC_DT_F32 ? 4 : 2; }

inline int check_dtypes(int storage, int operand) {
  if (storage < IPC_DT_F32 || storage > IPC_DT_BF16)
    return fail(IPC_ERR_DTYPE, "unknown storage dtype %d", storage);
  if (operand < IPC_DT_F32 || operand > IPC_DT_BF16)
    return fail(IPC_ERR_DTYPE, "unknown operand dtype %d", operand);
  if (storage != IPC_DT_F32 && operand != storage)
    return fail(IPC_ERR_DTYPE, "16-bit storage (%d) requires operand dtype == storage (got %d)",
                storage, operand);
  return ok();
}

inline int check_act(int act) {
  if (act < IPC_ACT_IDENTITY || act > IPC_ACT_GELU)
    return fail(IPC_ERR_ACT, "unknown activation %d", act);
  return ok();
}

inline int check_dims(int M, int K, int B, int groups) {
  if (M < 1 || K < 1 || B < 1 || groups < 1)
    return fail(IPC_ERR_SHAPE, "dimensions must be >= 1 (M=%d K=%d B=%d groups=%d)", M, K, B, groups);
  if ((long long)M * K > kMaxElems || (long long)M * B > kMaxElems || (long long)K * B > kMaxElems)
    return fail(IPC_ERR_SHAPE, "matrix too large (M=%d K=%d B=%d)", M, K, B);
  return ok();
}

inline int check_ptr(const void* p, const char* name, int esize) {
  if (!p) return fail(IPC_ERR_NULL, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % esize)
    return fail(IPC_ERR_ALIGN, "%s is not aligned to its %d-byte element", name, esize);
  return ok();
}

#define TRY(x)                  \
  do {                          \
    const int _rc = (x);        \
    if (_rc != IPC_OK) return _rc; \
  } while (0)

// 4-element vector loads need the contiguous length and the base aligned to 4 elements.
inline int vec_ok(const void* p, long long contiguous, int esize) {
  return (contiguous % 4 == 0) && (reinterpret_cast<uintptr_t>(p) % (4 * esize) == 0);
}

inline int launch_rc(hipError_t err, const char* what) {
  if (err != hipSuccess) return fail(IPC_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(err));
  return ok();
}

inline bool al16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }
inline bool al8(const void* q) { return q == nullptr || reinterpret_cast<uintptr_t>(q) % 8 == 0; }


inline int check_workspace(const void* workspace, long long ws_bytes) {
  if (ws_bytes < 0) return fail(IPC_ERR_SHAPE, "workspace_bytes must be >= 0");
  if (workspace && reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(IPC_ERR_ALIGN, "workspace must be 16-byte aligned");
  return ok();
}

}  // namespace abi
}  // namespace ipc
