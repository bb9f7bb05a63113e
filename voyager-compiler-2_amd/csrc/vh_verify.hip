// The choice among drafted tokens from given random numbers: which nodes of a
// tree are kept, and the token after them.
//
// A node's children are tried in order against what is left of the target's
// row.  Where children were chosen, a rejected token loses its probability;
// where they were sampled, rest = max(rest - mass * draft, 0), which after any
// number of rejections is max(target - c * draft, 0) with c the sum of the
// masses so far, so a row needs no buffer, only c.
//
// Chosen children may take everything out of a row: the last one taken out is
// then put back, so that no token of probability 0 is told.
//
// The token after the kept nodes is found in two passes over one row: sums of
// 4096 entries each, over many workgroups, then the one piece in which the
// running sum passes r times the whole.  Sums are float64 in a fixed order:
// 24-bit terms add exactly down to 2^-29 of the whole.
//
// Bound by latency: a row of 128,000 is 512 KB, 0.1 us of the card's
// bandwidth, behind the walk's dependent reads and two launches (three where a
// draft's probabilities may have to be summed during the walk).  32 trees of 31
// chosen tokens, 128,000 entries a row (16.4 MB): 9.3 us for the walk with the
// sums and 6.4 for the pick; five sampled tokens, 32,000 entries: 2.4 for the
// walk, 3.8 for the sums, 6.4 for the pick.  Sampled siblings cost more: each that
// is tried after a rejection has its row summed first, by the one workgroup of its
// sequence: about 24 us a sum at 128,000 entries (1 MB), 5 at 32,000.  Trees of
// three sampled children a node, 128,000 entries: one sequence 13 us where no
// second sibling is tried and 61 with two sums, 32 sequences 59 as drawn.
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace {

constexpr int THREADS = 256;
constexpr int WALK_THREADS = 1024;
constexpr int PICK_THREADS = 1024;
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

struct Nodes {  // in LDS; up to a multiple of four, the rest no children
  alignas(16) int32_t parent[MAX_NODES];  // -1: not a child
  alignas(16) int32_t token[MAX_NODES];   // -1: outside the vocabulary
  alignas(16) float p[MAX_NODES];
  float q[MAX_NODES], u[MAX_NODES];
  int32_t next[MAX_NODES];    // the child taken
};

template <bool DRAFT>
VH_DEV void load_nodes(const VerifyArgs& a, int64_t b, Nodes& s, int threads) {
  for (int n = threadIdx.x; n < (a.nodes + 3) / 4 * 4; n += threads) {
    const bool real = n > 0 && n < a.nodes;
    const int64_t at = b * a.nodes + (real ? n : 0);
    int up = a.parents[at];
    const int64_t x = a.tokens[at];
    s.u[n] = a.u[at];
    if (!real || up < 0 || up >= n) up = -1;
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

// What rejections leave of a probability: max(p - c q, 0), and NaN where that is
// one, so that a row which holds a NaN has no sum, with a rejection or without.
VH_DEV double left_of(double p, double c, double q) {
  const double x = p - c * q;
  return x <= 0.0 ? 0.0 : x;
}

// The sum over the workgroup in a fixed order; every thread gets it.
template <int N>
VH_DEV double block_sum(double v, double* s_part) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = s_part[0];
#pragma unroll
  for (int w = 1; w < N / 64; ++w) t += s_part[w];
  return t;
}

// Sampled children: whether one is taken depends on the mass that its
// rejected siblings left, a sum over the row.  A sum is taken only before a
// second sibling is tried: a chain needs none.
__global__ void __launch_bounds__(WALK_THREADS) k_verify_walk(VerifyArgs a) {
  __shared__ Nodes s;
  __shared__ double s_part[WALK_THREADS / 64];
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
      double v = 0.0;
#pragma unroll 8
      for (int64_t x = threadIdx.x; x < a.vocab; x += WALK_THREADS) v += left_of(p[x], more, q[x]);
      const double left = block_sum<WALK_THREADS>(v, s_part);
      if (left > 0.0) {
        c = more;
        mass = left;
      }
    }
    const double q = s.q[n], rest = left_of(s.p[n], c, q);
    if ((double)s.u[n] * mass * q < rest) {
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
    bool again = false;
#pragma unroll 4
    for (int k = 0; k < n; k += 4) {
      const int4 ups = *(const int4*)&s.parent[k], xs = *(const int4*)&s.token[k];
      again |= (ups.x == up && xs.x == x) || (ups.y == up && xs.y == x && k + 1 < n) ||
               (ups.z == up && xs.z == x && k + 2 < n) || (ups.w == up && xs.w == x && k + 3 < n);
    }
    if (again) s.p[n] = 0.0f;  // an earlier sibling's token: nothing is left of it
  }
  __syncthreads();
  for (int n = threadIdx.x; n < a.nodes; n += THREADS) {
    const int up = s.parent[n];
    double mass = 1.0;
#pragma unroll 4
    for (int k = 0; k < n; k += 4) {
      const int4 ups = *(const int4*)&s.parent[k];
      const float4 ps = *(const float4*)&s.p[k];
      mass = fmax(mass - (ups.x == up ? (double)ps.x : 0.0), 0.0);
      mass = fmax(mass - (ups.y == up && k + 1 < n ? (double)ps.y : 0.0), 0.0);
      mass = fmax(mass - (ups.z == up && k + 2 < n ? (double)ps.z : 0.0), 0.0);
      mass = fmax(mass - (ups.w == up && k + 3 < n ? (double)ps.w : 0.0), 0.0);
    }
    if (up >= 0 && (double)s.u[n] * mass < (double)s.p[n]) atomicMin(&s.next[up], n);
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
  // entry first + i, 0 from entry n on (read at the last: a read under a
  // condition would be waited for before the next)
  __device__ __forceinline__ double2 operator()(int64_t first, int i, int n) const {
    const int at = i < n ? i : n - 1;
    const float x0 = p[first + at];
    const double x = i < n ? x0 : 0.0f;
    if constexpr (DRAFT) {
      const float y0 = q[first + at];
      const double y = i < n ? y0 : 0.0f;
      return double2{c > 0.0 ? left_of(x, c, y) : x, c_before > 0.0 ? left_of(x, c_before, y) : x};
    } else {
      return double2{gone[i >> 5] >> (i & 31) & 1 ? 0.0 : x, 0.0};
    }
  }
};

template <bool DRAFT>
VH_DEV Rest<DRAFT> rest_of(const VerifyArgs& a, int64_t b, int last, const uint32_t* gone, const Row& row) {
  return Rest<DRAFT>{a.target + b * a.target_sb + last * a.target_sn,
                     DRAFT ? a.draft + b * a.draft_sb + last * a.draft_sn : nullptr, gone, row.c, row.c_before};
}

template <bool DRAFT>
__global__ void __launch_bounds__(THREADS) k_verify_sums(VerifyArgs a) {
  __shared__ Nodes s;
  __shared__ uint32_t s_gone[PIECE / 32];
  __shared__ double s_part[THREADS / 64];
  const int64_t b = blockIdx.y, first = (int64_t)blockIdx.x * PIECE;
  Row row{0, 0, 0.0, 0.0};
  int last;
  if constexpr (DRAFT) {
    row = a.rows[b];
    last = row.last;
  } else {
    last = walk_chosen(a, b, s, blockIdx.x == 0);
    for (int i = threadIdx.x; i < PIECE / 32; i += THREADS) s_gone[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < a.nodes; i += THREADS) {
      const int64_t x = s.token[i] - first;
      if (s.parent[i] == last && x >= 0 && x < PIECE) atomicOr(&s_gone[x >> 5], 1u << (x & 31));
    }
    __syncthreads();
  }
  const Rest<DRAFT> rest = rest_of<DRAFT>(a, b, last, s_gone, row);
  const int n = (int)(a.vocab - first < PIECE ? a.vocab - first : PIECE);
  double2 v = {0.0, 0.0};
#pragma unroll
  for (int k = 0; k < PIECE / THREADS; ++k) {
    const double2 x = rest(first, k * THREADS + threadIdx.x, n);
    v.x += x.x;
    v.y += x.y;
  }
  v.x = block_sum<THREADS>(v.x, s_part);
  if constexpr (DRAFT) v.y = block_sum<THREADS>(v.y, s_part);
  if (threadIdx.x == 0) a.sums[b * a.pieces + blockIdx.x] = v;
}

// The sum of the threads up to this one, and of all.
VH_DEV double block_scan(double v, double* s_wave, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
#pragma unroll
  for (int w = 0; w < PICK_THREADS / 64; ++w) {
    if (w == wave) before = all;
    all += s_wave[w];
  }
  return before + v;
}

// The first thread of the workgroup whose `hit` is true, or else the last
// whose `any` is, or else -1; s_pick has two places a wave.
VH_DEV int pick(bool hit, bool any, int* s_pick) {
  constexpr int W = PICK_THREADS / 64;
  const uint64_t h = __ballot(hit), y = __ballot(any);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s_pick[wave] = h ? wave * 64 + __ffsll((unsigned long long)h) - 1 : PICK_THREADS;
    s_pick[W + wave] = y ? wave * 64 + 63 - __clzll((long long)y) : -1;
  }
  __syncthreads();
  int first = PICK_THREADS, last = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    first = min(first, s_pick[w]);
    last = max(last, s_pick[W + w]);
  }
  return first < PICK_THREADS ? first : last;
}

// One thread a piece finds the piece, then one thread four entries the entry.
template <bool DRAFT>
__global__ void __launch_bounds__(PICK_THREADS) k_verify_pick(VerifyArgs a) {
  static_assert(MAX_PIECES <= PICK_THREADS && PIECE == 4 * PICK_THREADS, "one thread a piece, or four entries");
  __shared__ double s_wave[PICK_THREADS / 64];
  __shared__ double s_base;
  __shared__ uint32_t s_gone[PIECE / 32];
  __shared__ int s_pick[2 * PICK_THREADS / 64];
  const int64_t b = blockIdx.x;
  const Row row = a.rows[b];
  const double r = a.r[b];
  const bool held = threadIdx.x < a.pieces;
  const double2 sums = held ? a.sums[b * a.pieces + threadIdx.x] : double2{0.0, 0.0};
  // the tokens of the last node's children
  int64_t gone[MAX_NODES / PICK_THREADS];
  if constexpr (!DRAFT) {
#pragma unroll
    for (int k = 0; k < MAX_NODES / PICK_THREADS; ++k) {
      const int n = k * PICK_THREADS + threadIdx.x;
      gone[k] = n < a.nodes && n > row.last && a.parents[b * a.nodes + n] == row.last ? a.tokens[b * a.nodes + n] : -1;
    }
    for (int i = threadIdx.x; i < PIECE / 32; i += PICK_THREADS) s_gone[i] = 0u;
  }
  double total, v = sums.x;
  double upto = block_scan(v, s_wave, total);
  bool before = false;
  if (DRAFT && !(total > 0.0)) {  // the last rejection left nothing: the rest is as it was
    before = true;
    v = sums.y;
    upto = block_scan(v, s_wave, total);
  }
  const double bar = r * total;
  int64_t* out = a.told + b * a.nodes + row.count - 1;
  // the piece in which the running sum passes the bar, or the last with anything in it
  const int piece = pick(v > 0.0 && upto > bar, v > 0.0, s_pick);
  if constexpr (!DRAFT) {
    static_assert(MAX_NODES == PICK_THREADS, "a thread a node");
    if (piece < 0 && total == 0.0) {  // the children took everything out: the last one taken out is put back
      const int64_t x = gone[0];
      bool out_last = x >= 0 && x < a.vocab && a.target[b * a.target_sb + row.last * a.target_sn + x] > 0.0f;
      for (int n = row.last + 1; out_last && n < (int)threadIdx.x; ++n)  // not where an earlier sibling had
        out_last = a.parents[b * a.nodes + n] != row.last || a.tokens[b * a.nodes + n] != x;
      const int node = pick(false, out_last, s_pick);
      if (node >= 0) {
        if (threadIdx.x == node) *out = x;
        return;
      }
    }
  }
  if (piece < 0 || total != total) {  // no distribution: the end of it, or its start where it holds a NaN
    if (threadIdx.x == 0) *out = total != total ? 0 : a.vocab - 1;
    return;
  }
  if (threadIdx.x == piece) s_base = upto - v;
  const int64_t first = (int64_t)piece * PIECE;
  const int n = (int)(a.vocab - first < PIECE ? a.vocab - first : PIECE);
  if constexpr (!DRAFT) {
#pragma unroll
    for (int k = 0; k < MAX_NODES / PICK_THREADS; ++k) {
      const int64_t x = gone[k] - first;
      if (gone[k] >= 0 && x >= 0 && x < PIECE) atomicOr(&s_gone[x >> 5], 1u << (x & 31));
    }
  }
  __syncthreads();
  const Rest<DRAFT> rest = rest_of<DRAFT>(a, b, row.last, s_gone, row);
  double w[4], mine = 0.0, whole;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double2 x = rest(first, threadIdx.x * 4 + i, n);
    w[i] = before ? x.y : x.x;
    mine += w[i];
  }
  const double base = s_base;
  double at = base + (block_scan(mine, s_wave, whole) - mine);
  int hit = 4, any = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    at += w[i];
    if (w[i] > 0.0) {
      any = i;
      if (at > bar && hit == 4) hit = i;
    }
  }
  // none where a rounding put the piece's own sum on the other side of the bar: the last of all
  const int at_thread = pick(hit < 4, any >= 0, s_pick);
  if (threadIdx.x == at_thread) *out = first + threadIdx.x * 4 + (hit < 4 ? hit : any);
}

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" int64_t vh_verify_workspace_bytes(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0) return 0;
  return align16(batch * (int64_t)sizeof(Row)) + batch * ((vocab + PIECE - 1) / PIECE) * (int64_t)sizeof(double2);
}

extern "C" int vh_verify(const vh_verify_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  VH_REQUIRE(d, "vh_verify: null descriptor");
  VH_REQUIRE(d->batch >= 0 && d->batch < 65536, "vh_verify: at most 65535 sequences");
  VH_REQUIRE(d->nodes >= 1 && d->nodes <= MAX_NODES, "vh_verify: 1 to %d nodes (got %lld)", MAX_NODES, (long long)d->nodes);
  VH_REQUIRE(d->vocab >= 1 && d->vocab <= (int64_t)PIECE * MAX_PIECES, "vh_verify: a vocabulary of 1 to %lld",
             (long long)PIECE * MAX_PIECES);
  if (d->batch == 0) return VH_OK;
  VH_REQUIRE(d->target && d->parents && d->tokens && d->u && d->r && d->told && d->path && d->count,
             "vh_verify: null argument");
  const int64_t need = vh_verify_workspace_bytes(d->batch, d->vocab);
  VH_REQUIRE(work && (uintptr_t)work % 16 == 0 && work_bytes >= need, "vh_verify: needs %lld bytes of aligned workspace",
             (long long)need);
  VerifyArgs a{d->target, d->draft, d->target_sb, d->target_sn, d->draft_sb, d->draft_sn, d->parents, d->tokens, d->u, d->r,
               (int)d->nodes, (int)((d->vocab + PIECE - 1) / PIECE), d->vocab, d->told, d->path, d->count, (Row*)work,
               (double2*)((char*)work + align16(d->batch * (int64_t)sizeof(Row)))};
  hipStream_t s = vh::as_stream(stream);
  const dim3 rows((unsigned)d->batch), pieces((unsigned)a.pieces, (unsigned)d->batch);
  if (d->draft) {
    hipLaunchKernelGGL(k_verify_walk, rows, dim3(WALK_THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_sums<true>, pieces, dim3(THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_pick<true>, rows, dim3(PICK_THREADS), 0, s, a);
  } else {
    hipLaunchKernelGGL(k_verify_sums<false>, pieces, dim3(THREADS), 0, s, a);
    hipLaunchKernelGGL(k_verify_pick<false>, rows, dim3(PICK_THREADS), 0, s, a);
  }
  return vh::check_launch("vh_verify");
}
