// ipc_token_embed.hip - rows of a learnt table as a net's input state, and their update.
//
//   X[c D + d][b] = scale TABLE[ids[c][b]][d]
//   TABLE[v][d] += alpha sum over the places (c, b) of v of G[c D + d][b]
//
// Both move bytes and little else.  The table has a token's features next to each
// other, a state has the samples there, so a block of 64 samples by 64 features turns
// in LDS and both sides see runs of 128 bytes (16-bit).  512 features of 8 x 1024 places,
// bf16: 5.7 us, 2.1 TB/s of 12 MB that need be moved, 2.3 of it the launch.
//
// The update sorts the places by id, so that every sum has one owner and one order
// (atomics would add in any), in three launches: sort, with G transposed beside it (12.5 us; the
// sort alone 8.6, each of 256 workgroups reading all 8192 ids), sums of 16 places (6.5), sums that
// cross those (4.6).  Together 23 us for 8192 places of 512 features in bf16, where 15 MB
// take 3: launches and the waits for memory between dependent steps.  Of 8 and 64 places: 4.9 and 5.0 us, of 512 8.5, in
// one launch (embed_few_kernel); of 520 15.2.
#include "ipc_device.h"
#include "ipc_token.h"

namespace ipc {
namespace {

template <typename ST> struct Four { ST v[4]; };

template <typename ST>
__device__ __forceinline__ void store4(ST* p, const ST (&v)[4]) {
  typedef ST V __attribute__((ext_vector_type(4)));
  *reinterpret_cast<V*>(p) = V{v[0], v[1], v[2], v[3]};
}

// BT samples x DT features of one context place.
template <typename ST, int BT>
__global__ void __launch_bounds__(256) embed_kernel(const EmbedProblem p) {
  constexpr int DT = BT == 1 ? 1024 : 4096 / BT, LD = DT + (BT == 1 ? 0 : 2);
  __shared__ ST tile[BT * LD];
  const int tiles_d = (p.D + DT - 1) / DT, tiles_b = (p.B + BT - 1) / BT;
  const int td = blockIdx.x % tiles_d, tb = blockIdx.x / tiles_d % tiles_b, c = blockIdx.x / tiles_d / tiles_b;
  const int d0 = td * DT, b0 = tb * BT, tid = threadIdx.x;
  const ST* table = static_cast<const ST*>(p.table);
  ST* x = static_cast<ST*>(p.x);
  // every id, then every row's part, then the rest: two waits for memory in all
  constexpr int EACH = BT * DT / 1024;
  long long id[EACH];
  Four<ST> v[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int b = b0 + (e * 256 + tid) / (DT / 4);
    id[e] = b < p.B ? p.ids[(long long)c * p.B + b] : -1;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int d = d0 + (e * 256 + tid) % (DT / 4) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[e].v[i] = cvt<ST>(0.0f);
    if (id[e] < 0 || id[e] >= p.V || d >= p.D) continue;
    const ST* from = table + id[e] * p.D + d;
    if (p.vec_d) {
      v[e] = *reinterpret_cast<const Four<ST>*>(__builtin_assume_aligned(from, 4 * sizeof(ST)));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < p.D) v[e].v[i] = from[i];
    }
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int u = e * 256 + tid, r = u / (DT / 4), d = d0 + u % (DT / 4) * 4;
    const bool real = id[e] >= 0 && id[e] < p.V;
    ST o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = real ? cvt<ST>(to_f32(v[e].v[i]) * p.scale) : cvt<ST>(0.0f);
    if constexpr (BT == 1) {  // (one sample: X is as long as the row)
      if (d >= p.D) continue;
      ST* to = x + (long long)c * p.D + d;
      if (p.vec_d && p.vec_b) {
        store4(to, o);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < p.D) to[i] = o[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[r * LD + (d - d0) + i] = o[i];
    }
  }
  if constexpr (BT > 1) {
    __syncthreads();
    for (int u = tid; u < BT * DT / 4; u += 256) {
      const int r = u % (BT / 4) * 4, d = u / (BT / 4), b = b0 + r;
      if (b >= p.B || d0 + d >= p.D) continue;
      ST o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = tile[(r + i) * LD + d];
      ST* to = x + ((long long)c * p.D + d0 + d) * p.B + b;
      if (p.vec_b) {
        store4(to, o);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (b + i < p.B) to[i] = o[i];
      }
    }
  }
}

// ------------------------------------------------------------------ update
// Few places: a workgroup for each place and slab of features.  The first place of an id
// sums all of its places in order, the others have nothing to do.
template <typename ST>
__global__ void __launch_bounds__(256) embed_few_kernel(const EmbedUpdate p) {
  __shared__ int same[EMBED_SORTED];
  __shared__ int count, earlier;
  const int N = p.C * p.B, slabs = (p.D + 255) / 256, n = blockIdx.x / slabs, tid = threadIdx.x;
  const int d = blockIdx.x % slabs * 256 + tid;
  const long long id = p.ids[n];
  if (id < 0 || id >= p.V) return;
  if (tid == 0) earlier = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 256)
    if (p.ids[i] == id) earlier = 1;
  __syncthreads();
  if (earlier) return;
  if (tid < 64) {  // one wave lists the places in order
    int at = 0;
    for (int i = n; i < N; i += 64) {
      const bool hit = i + tid < N && p.ids[i + tid < N ? i + tid : N - 1] == id;
      const unsigned long long m = __ballot(hit);
      if (hit) same[at + __popcll(m & ((1ull << tid) - 1))] = i + tid;
      at += __popcll(m);
    }
    if (tid == 0) count = at;
  }
  __syncthreads();
  if (d >= p.D) return;
  const ST* g = static_cast<const ST*>(p.g);
  ST* t = static_cast<ST*>(p.table) + id * p.D + d;
  const float old = to_f32(*t);
  float sum = 0.0f;
  const int many = count;
#pragma unroll 4
  for (int i = 0; i < many; ++i) {
    const int at = same[i], c = at / p.B, b = at - c * p.B;
    sum += to_f32(g[((long long)c * p.D + d) * p.B + b]);
  }
  *t = cvt<ST>(old + p.alpha * sum);
}

// Workgroups 0 .. ranges - 1: each owns a range of ids, reads all places in order twice and
// writes its own, sorted, behind those of smaller ids (which it counts on the way, so
// that no workgroup waits for another).  Each of the sixteen waves has a sixteenth of the
// places, so that an id's places keep their order; up to 8192 places stay in its registers
// between the two readings.  The other workgroups transpose G.
constexpr int SORT_WAVES = 16, SORT_HELD = 8;

// A block of G, 64 features by TURN samples, so that each thread has several loads in flight.
template <typename ST> constexpr int TURN = embed_turn(sizeof(ST));
template <typename ST, bool VEC>
__device__ void transpose_rows(const EmbedUpdate& p, int block, ST* tile) {
  constexpr int W = TURN<ST>, LD = W + 2, EACH = 64 * W / 4 / (SORT_WAVES * 64);
  const int tiles_d = (p.D + 63) / 64, tiles_b = (p.B + W - 1) / W;
  const int td = block % tiles_d, tb = block / tiles_d % tiles_b, c = block / tiles_d / tiles_b;
  const int d0 = td * 64, b0 = tb * W;
  const ST* g = static_cast<const ST*>(p.g);
  ST* rows = static_cast<ST*>(p.rows);
  ST v[EACH][4];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int u = e * SORT_WAVES * 64 + threadIdx.x, d = u / (W / 4), b = u % (W / 4) * 4;
    if (d0 + d >= p.D || b0 + b >= p.B) continue;
    const ST* from = g + ((long long)c * p.D + d0 + d) * p.B + b0 + b;
    if constexpr (VEC) {
      const Four<ST> f = *reinterpret_cast<const Four<ST>*>(__builtin_assume_aligned(from, 4 * sizeof(ST)));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e][i] = f.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e][i] = b0 + b + i < p.B ? from[i] : cvt<ST>(0.0f);
    }
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int u = e * SORT_WAVES * 64 + threadIdx.x, d = u / (W / 4), b = u % (W / 4) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[d * LD + b + i] = v[e][i];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int u = e * SORT_WAVES * 64 + threadIdx.x, b = u >> 4, d = (u & 15) * 4;
    if (b0 + b >= p.B || d0 + d >= p.D) continue;
    ST o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = tile[(d + i) * LD + b];
    ST* to = rows + ((long long)c * p.B + b0 + b) * p.D + d0 + d;
    if constexpr (VEC) {  // (rows starts on 256 bytes)
      store4(to, o);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d0 + d + i < p.D) to[i] = o[i];
    }
  }
}

// Range `block` of `ranges`; lds: SORT_WAVES * range.
__device__ __forceinline__ void sort_places(const long long* ids, int N, int V, int* order, int* key, int* slot, int* lds, int block,
                                            int ranges, int range) {
  __shared__ int before[SORT_WAVES], sums[SORT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = ((N + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
  const int first = wave * per, last = first + per < N ? first + per : N;
  const long long lo = (long long)block * range;
  const long long hi = lo + range < V ? lo + range : V;
  int* mine = lds + wave * range;
  for (int i = tid; i < SORT_WAVES * range; i += SORT_WAVES * 64) lds[i] = 0;
  __syncthreads();
  int less = 0;
  // 64 SORT_HELD places from i0 on: ids relative to the range, -1 below it or padded, `range` or more above
  unsigned held[SORT_HELD];
  auto fetch = [&](int i0, bool count) {
    long long id[SORT_HELD];
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) {
      const int i = i0 + u * 64 + lane;
      id[u] = i < last ? ids[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) {
      const bool in = id[u] >= lo && id[u] < hi;
      held[u] = in ? (unsigned)(id[u] - lo) : ~0u;
      if (count) {
        less += id[u] >= 0 && id[u] < lo;
        if (in) atomicAdd(&mine[held[u]], 1);  // (a count: the order does not matter)
      }
    }
  };
  for (int i0 = first; i0 < last; i0 += 64 * SORT_HELD) fetch(i0, true);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) less += __shfl_xor(less, o);
  if (lane == 0) before[wave] = less;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) base += before[w];
  // where each id's places of each wave start: ids in order, then waves
  for (int r0 = 0; r0 < range; r0 += SORT_WAVES * 64) {
    const int r = r0 + tid;
    int total = 0;
    if (r < range)
      for (int w = 0; w < SORT_WAVES; ++w) total += lds[w * range + r];
    int scan = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int at = base + scan - total;
    for (int w = 0; w < SORT_WAVES; ++w) {
      if (w < wave) at += sums[w];
      base += sums[w];
    }
    if (slot && r < range && lo + r < V) slot[lo + r] = total > 0 ? at : -1;
    if (r < range)
      for (int w = 0; w < SORT_WAVES; ++w) {
        const int n = lds[w * range + r];
        lds[w * range + r] = at;
        at += n;
      }
    __syncthreads();
  }
  if (block == ranges - 1)  // behind the last place with an id
    for (int i = base + tid; i <= N; i += SORT_WAVES * 64) key[i] = -1;
  for (int i0 = first; i0 < last; i0 += 64 * SORT_HELD) {
    if (last - first > 64 * SORT_HELD) fetch(i0, false);
    unsigned many = 0;  // bit u: the u-th 64 have some in the range
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) many |= __any(held[u] != ~0u) ? 1u << u : 0u;
#pragma unroll 1
    for (; many; many &= many - 1) {
      const int u = __ffs(many) - 1;
      unsigned own = held[0];
#pragma unroll
      for (int q = 1; q < SORT_HELD; ++q) own = u == q ? held[q] : own;
      unsigned long long left = __ballot(own != ~0u);
      while (left) {  // one id after the other, its places in lane order
        const unsigned which = __builtin_amdgcn_readlane(own, __ffsll((unsigned long long)left) - 1);
        const unsigned long long same = __ballot(own == which);
        const int at = mine[which];
        if (own == which) {
          const int to = at + __popcll(same & ((1ull << lane) - 1));
          order[to] = i0 + u * 64 + lane;
          key[to] = (int)(lo + which);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane == 0) mine[which] = at + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        left &= ~same;
      }
    }
  }
}

template <typename ST, bool VEC>
__global__ void __launch_bounds__(SORT_WAVES * 64) embed_sort_kernel(const EmbedUpdate p, int ranges, int range) {
  extern __shared__ __align__(16) int lds[];
  if ((int)blockIdx.x >= ranges) transpose_rows<ST, VEC>(p, blockIdx.x - ranges, reinterpret_cast<ST*>(lds));
  else sort_places(p.ids, p.C * p.B, p.V, p.order, p.key, nullptr, lds, blockIdx.x, ranges, range);
}

__global__ void __launch_bounds__(SORT_WAVES * 64) sort_places_kernel(const long long* ids, int N, int V, int* order, int* key, int* slot,
                                                                      int ranges, int range) {
  extern __shared__ __align__(16) int lds[];
  sort_places(ids, N, V, order, key, slot, lds, blockIdx.x, ranges, range);
}

// A run of EMBED_RUN sorted places, 4 features a thread.  Ids that begin and end in the
// run are finished here; a sum that came over the run's start goes to part[run][0], one
// that goes on past its end to part[run][1].
// W features a thread: 4 where rows and the table are aligned for it, else 1.  Values stay as they
// lie until used, so that many rows can be in flight.
template <typename ST, int W> struct alignas(W * sizeof(ST)) Piece { ST v[W]; };
template <int W, typename ST>
__device__ __forceinline__ Piece<ST, W> get_piece(const ST* from) { return *reinterpret_cast<const Piece<ST, W>*>(from); }
template <int W, typename ST>
__device__ __forceinline__ void put_piece(ST* to, const float (&v)[W]) {
  Piece<ST, W> o;
#pragma unroll
  for (int q = 0; q < W; ++q) o.v[q] = cvt<ST>(v[q]);
  *reinterpret_cast<Piece<ST, W>*>(to) = o;
}
template <int W, typename ST>
__device__ __forceinline__ void add_to_piece(ST* to, const Piece<ST, W>& old, float alpha, const float (&sum)[W]) {
  float v[W];
#pragma unroll
  for (int q = 0; q < W; ++q) v[q] = to_f32(old.v[q]) + alpha * sum[q];
  put_piece<W>(to, v);
}

template <typename ST, int W>
__global__ void __launch_bounds__(256) embed_run_kernel(const EmbedUpdate p) {
  const int run = blockIdx.x, N = p.C * p.B, lane = threadIdx.x & 63;
  // (threads past the last feature go along with the first: their lanes hold places too)
  const int mine = (blockIdx.y * blockDim.x + threadIdx.x) * W, d = mine < p.D ? mine : 0, first = run * EMBED_RUN;
  // lane i: the id of the place before the run's i-th, and the i-th's row of G
  const int at = first - 1 + lane;
  const int keys = at >= 0 && at <= N ? p.key[at] : -1;
  const int orders = lane < EMBED_RUN && first + lane < N ? p.order[first + lane] : 0;
  auto key = [&](int i) { return __builtin_amdgcn_readlane(keys, i + 1); };
  if (key(0) < 0) return;
  const ST* rows = static_cast<const ST*>(p.rows) + d;
  ST* table = static_cast<ST*>(p.table) + d;
  // every row of G and of the table, none stored before all are read (a place without an id: any row)
  Piece<ST, W> v[EMBED_RUN], old[EMBED_RUN];
#pragma unroll
  for (int u = 0; u < EMBED_RUN; ++u) {
    const int id = key(u);
    v[u] = get_piece<W>(rows + (long long)(id < 0 ? 0 : __builtin_amdgcn_readlane(orders, u)) * p.D);
    old[u] = get_piece<W>(table + (long long)(id < 0 ? 0 : id) * p.D);
  }
  bool over = key(-1) == key(0);  // its sum came over the start
  float sum[W] = {};
#pragma unroll
  for (int u = 0; u < EMBED_RUN; ++u) {
    const int id = key(u);
    if (id < 0) return;
#pragma unroll
    for (int q = 0; q < W; ++q) sum[q] += to_f32(v[u].v[q]);
    const bool on = key(u + 1) == id;
    if (on && u + 1 < EMBED_RUN) continue;
    // the run's first and ended, or its last and not: a part
    if (mine >= p.D) {
    } else if (over || on) put_piece<W>(p.part + ((long long)run * 2 + (over ? 0 : 1)) * p.D + d, sum);
    else add_to_piece<W>(table + (long long)id * p.D, old[u], p.alpha, sum);
    over = false;
#pragma unroll
    for (int q = 0; q < W; ++q) sum[q] = 0.0f;
  }
}

// Sums that cross runs' ends, joined by the run they begin in.  `across` threads have its
// features; where these are few, as many groups of them as fit 256 threads each add a part of the
// runs (a word in a quarter of 20840 places goes over 325: 14.1 -> 5.8 us).
template <typename ST, int W>
__global__ void __launch_bounds__(256) embed_join_kernel(const EmbedUpdate p, int across) {
  __shared__ Piece<float, W> red[256];
  const int run = blockIdx.x, N = p.C * p.B, runs = (N + EMBED_RUN - 1) / EMBED_RUN;
  const int group = threadIdx.x / across, groups = blockDim.x / across;
  const int d = (blockIdx.y * across + threadIdx.x % across) * W, lane = threadIdx.x & 63;
  const int first = run * EMBED_RUN, end = first + EMBED_RUN;
  if (end >= N) return;
  const int id = p.key[end - 1];
  if (id < 0 || p.key[end] != id) return;
  if (first > 0 && p.key[first] == id && p.key[first - 1] == id) return;  // it began earlier
  int more = 0;  // runs it goes on into
  for (int r = run + 1;; r += 64) {
    const unsigned long long other = __ballot(r + lane >= runs || p.key[(long long)(r + lane < runs ? r + lane : 0) * EMBED_RUN] != id);
    more += other ? __ffsll(other) - 1 : 64;
    if (other) break;
  }
  const bool mine = d < p.D;
  ST* row = static_cast<ST*>(p.table) + (long long)id * p.D + (mine ? d : 0);
  const Piece<ST, W> old = get_piece<W>(row);
  float sum[W] = {};
  const float* from = p.part + ((long long)run * 2 + 1) * p.D + (mine ? d : 0);
  const int last = (int)((more + 1LL) * (group + 1) / groups);
#pragma unroll 8
  for (int r = (int)((more + 1LL) * group / groups); r < last; ++r) {
    // (its own second sum, then the later runs' first ones: 1, 3, 5, ... rows on)
    const Piece<float, W> v = get_piece<W>(from + (r == 0 ? 0 : 2 * r - 1) * (long long)p.D);
#pragma unroll
    for (int q = 0; q < W; ++q) sum[q] += v.v[q];
  }
  if (groups > 1) {
#pragma unroll
    for (int q = 0; q < W; ++q) red[threadIdx.x].v[q] = sum[q];
    __syncthreads();
    for (int g = 1; g < groups; ++g)
#pragma unroll
      for (int q = 0; q < W; ++q) sum[q] += group == 0 ? red[g * across + threadIdx.x].v[q] : 0.0f;
  }
  if (mine && group == 0) add_to_piece<W>(row, old, p.alpha, sum);
}

template <typename ST, int W>
hipError_t run_sums(const EmbedUpdate& p, hipStream_t s) {
  const int N = p.C * p.B, lanes = (p.D + W - 1) / W, threads = lanes >= 256 ? 256 : (lanes + 63) / 64 * 64;
  const dim3 grid((unsigned)((N + EMBED_RUN - 1) / EMBED_RUN), (unsigned)((lanes + threads - 1) / threads));
  hipLaunchKernelGGL((embed_run_kernel<ST, W>), grid, dim3(threads), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((embed_join_kernel<ST, W>), grid, dim3(256 / threads * threads), 0, s, p, threads);
  return hipGetLastError();
}

template <typename ST>
hipError_t run_embed(const EmbedProblem& p, hipStream_t s) {
  const dim3 grid((unsigned)embed_blocks(p.D, p.C, p.B)), block(256);
  if (p.B == 1) hipLaunchKernelGGL((embed_kernel<ST, 1>), grid, block, 0, s, p);
  else if (p.B <= 4) hipLaunchKernelGGL((embed_kernel<ST, 4>), grid, block, 0, s, p);
  else if (p.B <= 16) hipLaunchKernelGGL((embed_kernel<ST, 16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((embed_kernel<ST, 64>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <typename ST>
hipError_t run_update(const EmbedUpdate& p, hipStream_t s) {
  const int N = p.C * p.B;
  if (N < EMBED_SORTED) {
    hipLaunchKernelGGL((embed_few_kernel<ST>), dim3((unsigned)(N * (long long)((p.D + 255) / 256))), dim3(256), 0, s, p);
    return hipGetLastError();
  }
  const int range = sort_range(p.V, N), ranges = (int)(((long long)p.V + range - 1) / range);
  const long long turns = (long long)p.C * ((p.B + TURN<ST> - 1) / TURN<ST>) * ((p.D + 63) / 64);
  const int turn_lds = 64 * (TURN<ST> + 2) * (int)sizeof(ST), sort_lds = SORT_WAVES * range * 4;
  const dim3 grid((unsigned)(ranges + turns)), block(SORT_WAVES * 64);
  const int lds = turn_lds > sort_lds ? turn_lds : sort_lds;
  if (p.vec_b && p.D % 4 == 0) hipLaunchKernelGGL((embed_sort_kernel<ST, true>), grid, block, lds, s, p, ranges, range);
  else hipLaunchKernelGGL((embed_sort_kernel<ST, false>), grid, block, lds, s, p, ranges, range);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return p.vec_d ? run_sums<ST, 4>(p, s) : run_sums<ST, 1>(p, s);
}

}  // namespace

hipError_t launch_embedding(const EmbedProblem& p, int storage, hipStream_t s) {
  if (storage == 0) return run_embed<float>(p, s);
  return storage == 1 ? run_embed<f16>(p, s) : run_embed<bf16>(p, s);
}

hipError_t launch_sort_places(const long long* ids, int N, int V, int* order, int* key, int* slot, hipStream_t s) {
  const int range = sort_range(V, N), ranges = (int)(((long long)V + range - 1) / range);
  hipLaunchKernelGGL(sort_places_kernel, dim3((unsigned)ranges), dim3(SORT_WAVES * 64), SORT_WAVES * range * 4, s, ids, N, V, order, key, slot,
                     ranges, range);
  return hipGetLastError();
}

hipError_t launch_embedding_update(const EmbedUpdate& p, int storage, hipStream_t s) {
  if (storage == 0) return run_update<float>(p, s);
  return storage == 1 ? run_update<f16>(p, s) : run_update<bf16>(p, s);
}

}  // namespace ipc
