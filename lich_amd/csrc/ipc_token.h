// ipc_token.h - nets over tokens: layouts, host structs and launchers.
//
//   embedding         X[c D + d][b] = scale TABLE[ids[c][b]][d]
//   embedding update  TABLE[v][d] += alpha sum of G[c D + d][b] over the places (c, b) of v
//   dropout           OUT = m X / (1 - p), m from a counter-based generator
//   token loss        loss[b] = log sum_v exp z[v] - z[t_b], z = W f(X) column b
//   token update      that, e = onehot - softmax(z), G = f'(X) W^T e, W += alpha e f(X)^T
//
// States are [features][batch], weights [out][in], ids and targets 64-bit.  An id or
// target outside 0 .. V - 1 is a padded place.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ipc {

// ------------------------------------------------------------------ embedding
struct EmbedProblem {
  int V, D, C, B;
  const long long* ids;  // [C][B]
  const void* table;     // [V][D]
  void* x;               // [C D][B]
  float scale;
  int vec_d, vec_b;      // rows of the table / of x allow 4-element accesses
};
hipError_t launch_embedding(const EmbedProblem& p, int storage, hipStream_t s);

// Places are sorted by id, ties in their order; their rows of G, transposed once, are then
// summed in runs of EMBED_RUN places, and sums that cross a run's end joined: in order, or by up to four groups of
// threads that have a part of the runs each.  The order is the same every time.
constexpr int EMBED_RUN = 16;
// From so many places on (below, one launch finds the places of an id itself).
constexpr int EMBED_SORTED = 513;
struct EmbedUpdate {
  int V, D, C, B;
  void* table;
  const long long* ids;
  const void* g;         // [C D][B]
  float alpha;
  int vec_d, vec_b;
  // workspace (from EMBED_SORTED places on)
  int* order;            // [N] place of each sorted position
  int* key;              // [N + 1] its id; -1 from the first position without one on
  void* rows;            // [N][D] G transposed
  float* part;           // [runs][2][D] sums of ids that cross a run's start / end
};
struct EmbedLayout {
  long long order, key, rows, part, bytes;
};
inline EmbedLayout embed_layout(int D, int C, int B, int element) {
  auto up = [](long long v) { return (v + 255) & ~255LL; };
  const long long n = (long long)C * B, runs = (n + EMBED_RUN - 1) / EMBED_RUN;
  EmbedLayout l{};
  l.key = up(n * 4);
  l.rows = l.key + up((n + 1) * 4);
  l.part = l.rows + up(n * D * element);
  l.bytes = n < EMBED_SORTED ? 0 : l.part + up(runs * 2 * D * 4);
  return l;
}
// Ids of a range of the sort, at most 512: a workgroup for each 32 places, up to one a CU.  (Few ids each:
// a wave places the ids that it meets among 64 places one after the other; 8192 places of 64
// ids in one range: 56 us, in 64: 11.  But few workgroups for few places: 1505 places of 1531
// ids, 256 ranges 10.6 us, 24 6.2.)
inline int sort_range(int V, int N) {
  const int most = N < 64 ? 1 : N / 32 < 256 ? N / 32 : 256, r = (V + most - 1LL) / most < 512 ? (int)((V + most - 1LL) / most) : 512;
  return r;
}
// Samples of a block that the sort's launch turns (by 64 features).
constexpr int embed_turn(int element) { return element == 4 ? 128 : 256; }
// Workgroups of the lookup: of 256 threads each for a block of samples by features of a place.
inline long long embed_blocks(int D, int C, int B) {
  const int bt = B == 1 ? 1 : B <= 4 ? 4 : B <= 16 ? 16 : 64, dt = bt == 1 ? 1024 : 4096 / bt;
  return (long long)C * ((B + bt - 1LL) / bt) * ((D + dt - 1LL) / dt);
}
// Whether the calls' launches stay below 2^32 work-items.
inline bool embed_fits(int V, int D, int C, int B, int element) {
  constexpr long long most = (1LL << 32) - 1;
  const long long n = (long long)C * B;
  if (256 * embed_blocks(D, C, B) > most) return false;
  if (n < EMBED_SORTED) return true;
  const int range = sort_range(V, (int)n), turn = embed_turn(element);
  const long long sorts = ((long long)V + range - 1) / range + (long long)C * ((B + turn - 1LL) / turn) * ((D + 63LL) / 64);
  return 1024 * sorts <= most && 256 * ((n + EMBED_RUN - 1) / EMBED_RUN) <= most;
}
hipError_t launch_embedding_update(const EmbedUpdate& p, int storage, hipStream_t s);
// Places of N ids sorted by id, ties in their order: order [N], key [N + 1] as in EmbedUpdate; slot
// [V]: the first sorted position of each id, -1 of those that do not occur.
hipError_t launch_sort_places(const long long* ids, int N, int V, int* order, int* key, int* slot, hipStream_t s);

// -------------------------------------------------------------------- dropout
struct DropoutProblem {
  long long n;
  const void* x;
  const long long* rng;  // seed, step
  void* out;
  unsigned dropped;      // of 65536
  unsigned site;
  int vec;               // x and out on 16 bytes
};
hipError_t launch_dropout(const DropoutProblem& p, int storage, hipStream_t s);

// -------------------------------------------------------------------- softmax
struct TokenProblem {
  int V, D, B;
  const void* x;             // [D][B]
  void* w;                   // [V][D]
  const long long* targets;  // [B]
  float* loss;               // [B]
  void* g;                   // [D][B], or nullptr: the loss alone
  float alpha;
  int act;
  unsigned char* workspace;
};
// 0: sizes that the kernels do not take
long long token_workspace_bytes(int V, int D, int B, int storage, int act, bool update);
hipError_t launch_token(const TokenProblem& p, int storage, hipStream_t s);
// A few samples, W as it lies.
bool token_few(int V, int D, int B, int storage);
long long token_few_workspace_bytes(int V, int D, int B, int storage, bool update);
hipError_t launch_token_few(const TokenProblem& p, int storage, hipStream_t s);
// A small one in one workgroup, without a workspace.
bool token_small(int V, int D, int B);
hipError_t launch_token_small(const TokenProblem& p, int storage, hipStream_t s);

}  // namespace ipc
