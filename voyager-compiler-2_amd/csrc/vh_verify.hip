// The choice among drafted tokens from given random numbers: which nodes of a
// tree are kept, and the token after them.
//
// A node's children are tried in order against what is left of the target's
// row.  Where children were chosen, a rejected token loses its probability;
// where they were sampled, rest = max(rest - mass * draft, 0), which after any
// number of rejections is max(target - c * draft, 0) with c the sum of the
// masses so far, so a row needs no buffer, only c.
//
// The token after the kept nodes is found in two passes over one row: sums of
// 4096 entries each, over many workgroups, then the one piece in which the
// running sum passes r times the whole.  Sums are float64 in a fixed order:
// 24-bit terms add exactly down to 2^-29 of the whole.
//
// Bound by latency: a row of 128,000 is 512 KB, 0.1 us of the card's
// bandwidth, behind the walk's three dependent reads and two launches (three
// where a draft's probabilities may have to be summed during the walk).
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace {

constexpr int THREADS = 256;
constexpr int WALK_THREADS = 1024;
constexpr int PIECE = 4096;
constexpr int MAX_PIECES = 1024;
constexpr int MAX_NODES = VH_TREE_MAX_NODES;

struct Row {  // how far a sequence's walk came
  int32_t last, count;
  double c, c_before;  // the rest after the last rejection, and before it
};

struct VerifyArgs {
  const float *target, *draft;
  int64_t target_sb, target_sn, draft_sb, draft_sn;
  const int32_t* parents;
  const int64_t* tokens;
  const float *u, *r;
  int nodes, pieces;
  int64_t vocab;
  int64_t* told;
  int32_t *path, *count;
  Row* rows;
  double2* sums;  // [batch, pieces]: of the rest, and of the rest before the last rejection
};

struct Nodes {
  int32_t parent[MAX_NODES];  // -1: not a child
  int32_t token[MAX_NODES];   // -1: outside the vocabulary
  float p[MAX_NODES], q[MAX_NODES];
  int32_t next[MAX_NODES];    // the child taken
};

template <bool DRAFT>
VH_DEV void load_nodes(const VerifyArgs& a, int64_t b, Nodes& s, int threads) {
  for (int n = threadIdx.x; n < a.nodes; n += threads) {
    int up = a.parents[b * a.nodes + n];
    const int64_t x = a.tokens[b * a.nodes + n];
    if (n == 0 || up < 0 || up >= n) up = -1;
    const bool in = up >= 0 && x >= 0 && x < a.vocab;
    s.parent[n] = up;
    s.token[n] = in ? (int32_t)x : -1;
    s.p[n] = in ? a.target[b * a.target_sb + up * a.target_sn + x] : 0.0f;
    if constexpr (DRAFT) s.q[n] = in ? a.draft[b * a.draft_sb + up * a.draft_sn + x] : 0.0f;
    s.next[n] = a.nodes;
  }
  __syncthreads();
}

// One thread writes node `n`, the i-th kept, and its token.
VH_DEV void tell(const VerifyArgs& a, int64_t b, const Nodes& s, int i, int n) {
  a.path[b * a.nodes + i] = n;
  if (i > 0) a.told[b * a.nodes + i - 1] = a.tokens[b * a.nodes + n];
}
// The unused rest of the outputs; the last token's place is written by k_verify_pick.
VH_DEV void tell_none(const VerifyArgs& a, int64_t b, int count, int threads) {
  for (int i = threadIdx.x; i < a.nodes; i += threads) {
    if (i >= count) {
      a.path[b * a.nodes + i] = -1;
      a.told[b * a.nodes + i] = -1;
    }
  }
  if (threadIdx.x == 0) a.count[b] = count;
}

// Sums over the workgroup in a fixed order; every thread gets them.
template <int N>
VH_DEV double2 block_sum(double2 v, double2* s_part) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    v.x += __shfl_xor(v.x, d);
    v.y += __shfl_xor(v.y, d);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  double2 t = s_part[0];
#pragma unroll
  for (int w = 1; w < N / 64; ++w) {
    t.x += s_part[w].x;
    t.y += s_part[w].y;
  }
  return t;
}

// Sampled children: whether one is taken depends on the mass that its
// rejected siblings left, a sum over the row.  A sum is taken only before a
// second sibling is tried: a chain needs none.
__global__ void __launch_bounds__(WALK_THREADS) k_verify_walk(VerifyArgs a) {
  __shared__ Nodes s;
  __shared__ double2 s_part[WALK_THREADS / 64];
  const int64_t b = blockIdx.x;
  load_nodes<true>(a, b, s, WALK_THREADS);
  int cur = 0, count = 1;
  double c = 0.0, mass = 1.0;
  bool rejected = false;
  if (threadIdx.x == 0) tell(a, b, s, 0, 0);
  for (int n = 1; n < a.nodes; ++n) {
    if (s.parent[n] != cur) continue;
    if (rejected) {
      const float* p = a.target + b * a.target_sb + cur * a.target_sn;
      const float* q = a.draft + b * a.draft_sb + cur * a.draft_sn;
      const double more = c + mass;
      double2 v = {0.0, 0.0};
      for (int64_t x = threadIdx.x; x < a.vocab; x += WALK_THREADS) v.x += fmax((double)p[x] - more * (double)q[x], 0.0);
      const double left = block_sum<WALK_THREADS>(v, s_part).x;
      if (left > 0.0) {
        c = more;
        mass = left;
      }
    }
    const double q = s.q[n], rest = fmax((double)s.p[n] - c * q, 0.0);
    if ((double)a.u[b * a.nodes + n] * mass * q < rest) {
      if (threadIdx.x == 0) tell(a, b, s, count, n);
      ++count;
      cur = n;
      c = 0.0;
      mass = 1.0;
      rejected = false;
    } else {
      rejected = true;
    }
  }
  tell_none(a, b, count, WALK_THREADS);
  if (threadIdx.x == 0) a.rows[b] = Row{cur, count, rejected ? c + mass : c, c};
}

// Chosen children: what a node's earlier siblings leave is a sum over them, so
// each node is tested by its own thread as if they had all been rejected; the
// first that passes is its parent's choice.  Returns the last kept node.
VH_DEV int walk_chosen(const VerifyArgs& a, int64_t b, Nodes& s, bool teller) {
  load_nodes<false>(a, b, s, THREADS);
  for (int n = threadIdx.x; n < a.nodes; n += THREADS) {
    const int up = s.parent[n], x = s.token[n];
    if (up < 0 || x < 0) continue;
    bool again = false;
    for (int k = 1; k < n; ++k) again |= s.parent[k] == up && s.token[k] == x;
    if (again) s.p[n] = 0.0f;  // an earlier sibling's token: nothing is left of it
  }
  __syncthreads();
  for (int n = threadIdx.x; n < a.nodes; n += THREADS) {
    const int up = s.parent[n];
    if (up < 0) continue;
    double mass = 1.0;
    for (int k = 1; k < n; ++k)
      if (s.parent[k] == up) mass = fmax(mass - (double)s.p[k], 0.0);
    if ((double)a.u[b * a.nodes + n] * mass < (double)s.p[n]) atomicMin(&s.next[up], n);
  }
  __syncthreads();
  int cur = 0, count = 1;
  if (teller && threadIdx.x == 0) tell(a, b, s, 0, 0);
  while (s.next[cur] < a.nodes) {
    cur = s.next[cur];
    if (teller && threadIdx.x == 0) tell(a, b, s, count, cur);
    ++count;
  }
  if (teller) {
    tell_none(a, b, count, THREADS);
    if (threadIdx.x == 0) a.rows[b] = Row{cur, count, 0.0, 0.0};
  }
  return cur;
}

// What is left of entries [first, first + PIECE) of a row, entry i at w(i): by
// the draft's probabilities, or without the tokens whose bits are set.
template <bool DRAFT>
struct Rest {
  const float *p, *q;
  const uint32_t* gone;
  double c, c_before;
  __device__ __forceinline__ double2 operator()(int64_t first, int i) const {
    const double x = p[first + i];
    if constexpr (DRAFT) {
      const double y = q[first + i];
      return double2{c > 0.0 ? fmax(x - c * y, 0.0) : x, c_before > 0.0 ? fmax(x - c_before * y, 0.0) : x};
    } else {
      return double2{gone[i >> 5] >> (i & 31) & 1 ? 0.0 : x, 0.0};
    }
  }
};

// Marks the tokens of `last`'s children that fall into the piece.
VH_DEV void mark_gone(const VerifyArgs& a, int64_t b, int last, int64_t first, uint32_t* gone) {
  for (int i = threadIdx.x; i < PIECE / 32; i += THREADS) gone[i] = 0u;
  __syncthreads();
  for (int n = threadIdx.x; n < a.nodes; n += THREADS) {
    const int64_t x = a.tokens[b * a.nodes + n] - first;
    if (n > last && a.parents[b * a.nodes + n] == last && x >= 0 && x < PIECE) atomicOr(&gone[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
}

template <bool DRAFT>
VH_DEV Rest<DRAFT> rest_of(const VerifyArgs& a, int64_t b, int last, const uint32_t* gone, const Row& row) {
  return Rest<DRAFT>{a.target + b * a.target_sb + last * a.target_sn,
                     DRAFT ? a.draft + b * a.draft_sb + last * a.draft_sn : nullptr, gone, row.c, row.c_before};
}

template <bool DRAFT>
__global__ void __launch_bounds__(THREADS) k_verify_sums(VerifyArgs a) {
  __shared__ Nodes s;
  __shared__ uint32_t s_gone[PIECE / 32];
  __shared__ double2 s_part[THREADS / 64];
  const int64_t b = blockIdx.y, first = (int64_t)blockIdx.x * PIECE;
  Row row{0, 0, 0.0, 0.0};
  int last;
  if constexpr (DRAFT) {
    row = a.rows[b];
    last = row.last;
  } else {
    last = walk_chosen(a, b, s, blockIdx.x == 0);
    mark_gone(a, b, last, first, s_gone);
  }
  const Rest<DRAFT> rest = rest_of<DRAFT>(a, b, last, s_gone, row);
  const int n = (int)(a.vocab - first < PIECE ? a.vocab - first : PIECE);
  double2 v = {0.0, 0.0};
#pragma unroll 16
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const double2 x = rest(first, i);
    v.x += x.x;
    v.y += x.y;
  }
  v = block_sum<THREADS>(v, s_part);
  if (threadIdx.x == 0) a.sums[b * a.pieces + blockIdx.x] = v;
}

template <bool DRAFT>
__global__ void __launch_bounds__(THREADS) k_verify_pick(VerifyArgs a) {
  __shared__ double s_sum[MAX_PIECES];
  __shared__ double s_w[PIECE];
  __shared__ double s_wave[THREADS / 64];
  __shared__ uint32_t s_gone[PIECE / 32];
  __shared__ int s_first, s_last;
  const int64_t b = blockIdx.x;
  const Row row = a.rows[b];
  bool before = false;  // the last rejection left nothing: the rest is as it was
  if constexpr (DRAFT) {
    double all = 0.0;
    for (int i = 0; i < a.pieces; ++i) all += a.sums[b * a.pieces + i].x;
    before = !(all > 0.0);
  }
  for (int i = threadIdx.x; i < a.pieces; i += THREADS) {
    const double2 v = a.sums[b * a.pieces + i];
    s_sum[i] = before ? v.y : v.x;
  }
  if (threadIdx.x == 0) {
    s_first = PIECE;
    s_last = -1;
  }
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < a.pieces; ++i) total += s_sum[i];
  const double bar = (double)a.r[b] * total;
  // the piece in which the running sum passes the bar, or the last with anything in it
  int piece = -1;
  double base = 0.0, run = 0.0;
  for (int i = 0; i < a.pieces; ++i) {
    const double v = s_sum[i];
    if (v > 0.0) {
      piece = i;
      base = run;
    }
    run += v;
    if (run > bar) break;
  }
  int64_t* out = a.told + b * a.nodes + row.count - 1;
  if (piece < 0 || total != total) {  // no distribution: the end of it, or its start where it holds a NaN
    if (threadIdx.x == 0) *out = total != total ? 0 : a.vocab - 1;
    return;
  }
  const int64_t first = (int64_t)piece * PIECE;
  const int n = (int)(a.vocab - first < PIECE ? a.vocab - first : PIECE);
  if constexpr (!DRAFT) mark_gone(a, b, row.last, first, s_gone);
  const Rest<DRAFT> rest = rest_of<DRAFT>(a, b, row.last, s_gone, row);
#pragma unroll 16
  for (int i = threadIdx.x; i < PIECE; i += THREADS) {
    const double2 x = i < n ? rest(first, i) : double2{0.0, 0.0};
    s_w[i] = before ? x.y : x.x;
  }
  __syncthreads();
  constexpr int PER = PIECE / THREADS;
  double mine = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine += s_w[threadIdx.x * PER + i];
  // the sums of the threads before this one
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double up = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double y = __shfl_up(up, d);
    if (lane >= d) up += y;
  }
  if (lane == 63) s_wave[wave] = up;
  __syncthreads();
  double at = base + (up - mine);
  for (int w = 0; w < wave; ++w) at += s_wave[w];
  int hit = PIECE, any = -1;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const double w = s_w[threadIdx.x * PER + i];
    at += w;
    if (w > 0.0) {
      any = threadIdx.x * PER + i;
      if (at > bar && hit == PIECE) hit = any;
    }
  }
  if (hit < PIECE) atomicMin(&s_first, hit);
  if (any >= 0) atomicMax(&s_last, any);
  __syncthreads();
  // none where a rounding put the piece's own sum on the other side of the bar
  if (threadIdx.x == 0) *out = first + (s_first < PIECE ? s_first : s_last);
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" int64_t vh_verify_workspace_bytes(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0) return 0;
  return align16(batch * (int64_t)sizeof(Row)) + batch * ((vocab + PIECE - 1) / PIECE) * (int64_t)sizeof(double2);
}

extern "C" int vh_verify(const float* target, int64_t target_sb, int64_t target_sn, const float* draft, int64_t draft_sb,
                         int64_t draft_sn, const int32_t* parents, const int64_t* tokens, const float* u, const float* r,
                         int64_t batch, int32_t nodes, int64_t vocab, int64_t* told, int32_t* path, int32_t* count,
                         void* work, int64_t work_bytes, vh_stream_t stream) {
  VH_REQUIRE(batch >= 0 && batch < 65536, "vh_verify: at most 65535 sequences");
  VH_REQUIRE(nodes >= 1 && nodes <= MAX_NODES, "vh_verify: 1 to %d nodes (got %d)", MAX_NODES, nodes);
  VH_REQUIRE(vocab >= 1 && vocab <= (int64_t)PIECE * MAX_PIECES, "vh_verify: a vocabulary of 1 to %lld",
             (long long)PIECE * MAX_PIECES);
  if (batch == 0) return VH_OK;
  VH_REQUIRE(target && parents && tokens && u && r && told && path && count, "vh_verify: null argument");
  VH_REQUIRE(work && (uintptr_t)work % 16 == 0 && work_bytes >= vh_verify_workspace_bytes(batch, vocab),
             "vh_verify: needs %lld bytes of aligned workspace", (long long)vh_verify_workspace_bytes(batch, vocab));
  VerifyArgs a{target, draft, target_sb, target_sn, draft_sb, draft_sn, parents, tokens, u, r, nodes,
               (int)((vocab + PIECE - 1) / PIECE), vocab, told, path, count, (Row*)work,
               (double2*)((char*)work + align16(batch * (int64_t)sizeof(Row)))};
  hipStream_t s = vh::as_stream(stream);
  const dim3 rows((unsigned)batch), pieces((unsigned)a.pieces, (unsigned)batch);
  if (draft) {
    hipLaunchKernelGGL(k_verify_walk, rows, dim3(WALK_THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_sums<true>, pieces, dim3(THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_pick<true>, rows, dim3(THREADS), 0, s, a);
  } else {
    hipLaunchKernelGGL(k_verify_sums<false>, pieces, dim3(THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_pick<false>, rows, dim3(THREADS), 0, s, a);
  }
  return vh::check_launch("vh_verify");
}
