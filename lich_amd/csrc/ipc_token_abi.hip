// ipc_token_abi.hip - extern "C" entry points of the operators over tokens (declared in
// include/ipc_hip.h), with the argument checks of ipc_abi.hip: everything is
// refused on the host, before any HIP call.
#include "ipc_abi_check.h"
#include "ipc_launch.h"
#include "ipc_token.h"

using namespace ipc;
using namespace ipc::abi;

namespace {

int check_embedding(int V, int D, int C, int B, int storage) {
  TRY(check_dtypes(storage, storage));
  if (V < 1 || D < 1 || C < 1 || B < 1)
    return fail(IPC_ERR_SHAPE, "dimensions must be >= 1 (V=%d D=%d C=%d B=%d)", V, D, C, B);
  if ((long long)V * D > kMaxElems || (long long)C * B > kMaxElems || (long long)C * B * D > kMaxElems)
    return fail(IPC_ERR_SHAPE, "table or state too large (V=%d D=%d C=%d B=%d)", V, D, C, B);
  if (!embed_fits(V, D, C, B, elem_size(storage)))
    return fail(IPC_ERR_SHAPE, "too large for a launch (V=%d D=%d C=%d B=%d)", V, D, C, B);
  return ok();
}

// A lent workspace of `need` bytes.
int check_lent(const void* workspace, long long bytes, long long need) {
  TRY(check_workspace(workspace, bytes));
  if (need > 0 && !workspace) return fail(IPC_ERR_NULL, "workspace is NULL (%lld bytes needed)", need);
  if (bytes < need) return fail(IPC_ERR_SHAPE, "workspace of %lld bytes, %lld needed", bytes, need);
  return ok();
}

int check_token(const void* x, const void* w, const void* targets, const void* loss, int V, int D, int B, int storage,
                int act, bool update) {
  TRY(check_dtypes(storage, storage));
  TRY(check_act(act));
  TRY(check_dims(V, D, B, 1));
  if (token_workspace_bytes(V, D, B, storage, act, update) == 0)
    return fail(IPC_ERR_SHAPE, "too large (V=%d D=%d B=%d)", V, D, B);
  TRY(check_ptr(x, "x", elem_size(storage)));
  TRY(check_ptr(w, "w", elem_size(storage)));
  if (storage != IPC_DT_F32 && D % 2 == 0 && reinterpret_cast<uintptr_t>(w) % 4)
    return fail(IPC_ERR_ALIGN, "w with rows of an even length needs 4-byte alignment");
  TRY(check_ptr(targets, "targets", 8));
  TRY(check_ptr(loss, "loss", 4));
  return ok();
}

}  // namespace

extern "C" {

int ipc_embedding(const long long* ids, const void* table, void* x, int V, int D, int C, int B, float scale, int storage,
                  void* stream) {
  TRY(check_embedding(V, D, C, B, storage));
  const int es = elem_size(storage);
  TRY(check_ptr(ids, "ids", 8));
  TRY(check_ptr(table, "table", es));
  TRY(check_ptr(x, "x", es));
  EmbedProblem p{};
  p.V = V; p.D = D; p.C = C; p.B = B;
  p.ids = ids; p.table = table; p.x = x; p.scale = scale;
  p.vec_d = vec_ok(table, D, es);
  p.vec_b = vec_ok(x, B == 1 ? D : B, es);
  return launch_rc(launch_embedding(p, storage, (hipStream_t)stream), "ipc_embedding");
}

long long ipc_embedding_update_workspace_bytes(int V, int D, int C, int B, int storage) {
  if (check_embedding(V, D, C, B, storage) != IPC_OK) return 0;
  return embed_layout(D, C, B, elem_size(storage)).bytes;
}

int ipc_embedding_update(void* table, const long long* ids, const void* g, int V, int D, int C, int B, float alpha,
                         int storage, void* workspace, long long workspace_bytes, void* stream) {
  TRY(check_embedding(V, D, C, B, storage));
  const int es = elem_size(storage);
  TRY(check_ptr(table, "table", es));
  TRY(check_ptr(ids, "ids", 8));
  TRY(check_ptr(g, "g", es));
  const EmbedLayout l = embed_layout(D, C, B, es);
  TRY(check_lent(workspace, workspace_bytes, l.bytes));
  EmbedUpdate p{};
  p.V = V; p.D = D; p.C = C; p.B = B;
  p.table = table; p.ids = ids; p.g = g; p.alpha = alpha;
  p.vec_d = vec_ok(table, D, es);
  p.vec_b = vec_ok(g, B, es);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  if (l.bytes > 0) {
    p.order = reinterpret_cast<int*>(ws + l.order);
    p.key = reinterpret_cast<int*>(ws + l.key);
    p.rows = ws + l.rows;
    p.part = reinterpret_cast<float*>(ws + l.part);
  }
  return launch_rc(launch_embedding_update(p, storage, (hipStream_t)stream), "ipc_embedding_update");
}

int ipc_dropout(const void* x, const long long* rng, void* out, int M, int B, int dropped, int site, int storage,
                void* stream) {
  TRY(check_dtypes(storage, storage));
  TRY(check_dims(M, 1, B, 1));
  if (dropped < 0 || dropped > 65535) return fail(IPC_ERR_CONFIG, "dropped must be 0 .. 65535 (got %d)", dropped);
  const int es = elem_size(storage);
  TRY(check_ptr(x, "x", es));
  TRY(check_ptr(rng, "rng", 8));
  TRY(check_ptr(out, "out", es));
  DropoutProblem p{};
  p.n = (long long)M * B;
  p.x = x; p.rng = rng; p.out = out;
  p.dropped = (unsigned)dropped; p.site = (unsigned)site;
  p.vec = al16(x) && al16(out);
  return launch_rc(launch_dropout(p, storage, (hipStream_t)stream), "ipc_dropout");
}

long long ipc_token_loss_workspace_bytes(int V, int D, int B, int storage, int act) {
  if (check_dtypes(storage, storage) != IPC_OK || check_act(act) != IPC_OK || check_dims(V, D, B, 1) != IPC_OK) return 0;
  return token_workspace_bytes(V, D, B, storage, act, false);
}

long long ipc_token_update_workspace_bytes(int V, int D, int B, int storage, int act) {
  if (check_dtypes(storage, storage) != IPC_OK || check_act(act) != IPC_OK || check_dims(V, D, B, 1) != IPC_OK) return 0;
  return token_workspace_bytes(V, D, B, storage, act, true);
}

int ipc_token_loss(const void* x, const void* w, const long long* targets, float* loss, int V, int D, int B, int storage,
                   int act, void* workspace, long long workspace_bytes, void* stream) {
  TRY(check_token(x, w, targets, loss, V, D, B, storage, act, false));
  TRY(check_lent(workspace, workspace_bytes, token_workspace_bytes(V, D, B, storage, act, false)));
  TokenProblem p{};
  p.V = V; p.D = D; p.B = B; p.act = act;
  p.x = x; p.w = const_cast<void*>(w); p.targets = targets; p.loss = loss;
  p.workspace = static_cast<unsigned char*>(workspace);
  return launch_rc(launch_token(p, storage, (hipStream_t)stream), "ipc_token_loss");
}

int ipc_token_update(const void* x, void* w, const long long* targets, float* loss, void* g, int V, int D, int B,
                     float alpha, int storage, int act, void* workspace, long long workspace_bytes, void* stream) {
  TRY(check_token(x, w, targets, loss, V, D, B, storage, act, true));
  TRY(check_ptr(g, "g", elem_size(storage)));
  TRY(check_lent(workspace, workspace_bytes, token_workspace_bytes(V, D, B, storage, act, true)));
  TokenProblem p{};
  p.V = V; p.D = D; p.B = B; p.act = act;
  p.x = x; p.w = w; p.targets = targets; p.loss = loss; p.g = g; p.alpha = alpha;
  p.workspace = static_cast<unsigned char*>(workspace);
  return launch_rc(launch_token(p, storage, (hipStream_t)stream), "ipc_token_update");
}

}  // extern "C"
