// Log probabilities of given tokens, with the entropy and the best alternatives.
//
// Of a row x of logits, with m = max x, l = sum exp(x - m) and e = sum
// exp(x - m) (x - m):
//
//   lse = m + log l,  logprob = x[token] - lse,  entropy = log l - e / l
//
// and the `top` largest entries, of equal ones the first.  Back, for gradients
// g of the log probability, h of the entropy and t_k of the alternatives:
//
//   dx_j = g [j = token] + sum_k t_k [j = index_k] - p_j (g + sum_k t_k + h (x_j - lse + entropy))
//
// Forward, a workgroup holds a piece of a row in registers, all loads in
// flight at once: the maximum is known before the first exponential, so
// every logit is read once and takes one exponential.  Rows longer than a
// piece, and few rows, are several pieces, joined by a second kernel.  The
// best are found among the registers as well: what does not reach a bound
// that `top` entries reach is left out, and the rest is ranked.
//
// Bound: with alternatives, and rows for the whole card, what finds them beside the
// exponentials (4001 rows of 32,000 in float16 with the best one: 62 us, 4.2 TB/s);
// without, memory (2048 rows of 128,000 in bfloat16: 107 us, 4.9 TB/s, and 141 behind a
// backward pass, whose writes are on their way to memory; back, read and
// written, 162 us, 6.5 TB/s, part of it in the last cache); for few rows the latency
// of two launches (32 rows of 128,000 with twenty: 11 + 4 us).
//
// Sums are float32.  Exponents are differences x - m, so that entries of the
// type's lowest value, or a row of them, stay in range.
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64;
constexpr int JOIN_THREADS = 256;
constexpr int MAX_TOP = VH_SCORE_MAX_TOP;
constexpr int MAX_PIECES = 64;
constexpr int CANDIDATES = 1024;  // of a piece, that are ranked
constexpr int BACK_THREADS = 256, BACK_VECTORS = 4;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;
constexpr float INF = __builtin_inff();
constexpr float FAR = -1e4f;  // a difference whose power is 0

typedef unsigned long long okey;  // orders entries: by value, then the lowest index first; 0: none

struct Args {
  const void* x;
  int64_t x_st, batch_st, vocab, rows;
  uint32_t batch_rows;  // rows of which lie x_st apart; 0: all
  const int64_t* tokens;
  int64_t piece;  // entries of a piece
  int pieces, top;
  float *logprob, *entropy;
  float2* stats;  // a row's maximum and the logarithm of its sum
  float* top_logprob;
  int64_t* top_token;
  float* part;     // [rows, pieces, 3]: maximum, sum, sum of exponents of two; NULL: a row is one piece
  okey* part_top;  // [rows, pieces, top]
  const float *g_logprob, *g_entropy, *g_top;
  void* grad;
  uint32_t chunks;
};

template <typename T>
VH_DEV const T* logits_of(const Args& a, int64_t row) {
  if (a.batch_rows == 0) return (const T*)a.x + row * a.x_st;
  const uint32_t batch = (uint32_t)row / a.batch_rows;
  return (const T*)a.x + batch * a.batch_st + ((uint32_t)row - batch * a.batch_rows) * a.x_st;
}

VH_DEV float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // keeps a NaN
VH_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Rises with the value, +0 and -0 alike, a NaN above all; 0 is no entry's.
VH_DEV uint32_t rank_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
VH_DEV float value_of(uint32_t r) {
  return r == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(r & 0x80000000u ? r ^ 0x80000000u : ~r);
}
VH_DEV okey key_of(uint32_t rank, uint32_t index) { return (okey)rank << 32 | (uint32_t)~index; }

// Entries [at, at + 16 bytes) of a row, with -inf past its end: 16 bytes at
// any alignment of the type, which the hardware takes.  What would pass the
// row's end is read from there on down, and moved by `shift16`.
template <typename T>
VH_DEV uint4 load16(const T* x, int at, int end) {
  uint4 v;
  __builtin_memcpy(&v, x + min(at, end - 16 / (int)sizeof(T)), 16);
  return v;
}
template <typename T>
VH_DEV uint4 shift16(uint4 v, int at, int end) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr uint32_t NONE = __is_same(T, float) ? 0xff800000u : __is_same(T, _Float16) ? 0xfc00fc00u : 0xff80ff80u;
  const int gone = (at - (end - VEC)) * (int)sizeof(T);  // bytes of entries before `at`
  if (gone > 0) {
    if (gone >= 16) v = make_uint4(NONE, NONE, NONE, NONE);
    if (gone & 8) v = make_uint4(v.z, v.w, NONE, NONE);
    if (gone & 4) v = make_uint4(v.y, v.z, v.w, NONE);
    if (gone & 2) v = make_uint4(v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16 | NONE << 16);
  }
  return v;
}
// A row shorter than that.
template <typename T>
VH_DEV uint4 load_short(const T* x, int end) {
  T e[16 / sizeof(T)];
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(T); ++j) e[j] = j < end ? x[j] : (T)-INF;
  uint4 v;
  __builtin_memcpy(&v, e, 16);
  return v;
}
// Entry j of 16 bytes, and what its power's exponent of two is.
template <typename T>
VH_DEV float entry(uint4 v, int j) {
  T e[16 / sizeof(T)];
  __builtin_memcpy(e, &v, 16);
  return (float)e[j];
}
// The compiler would keep what it converts once for all later uses: twice the
// registers, and half the workgroups.  This hides that the values are the same.
VH_DEV uint4 convert_again(uint4 v) {
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
  return v;
}
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// The largest of 16 bytes' entries; float16 ones two at a time, which bfloat16 has no instruction for.
template <typename T>
VH_DEV float largest_entry(uint4 v) {
  if constexpr (__is_same(T, _Float16)) {
    const auto two = [](uint32_t w) { return __builtin_bit_cast(f16x2, w); };
    const f16x2 a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(two(v.x), two(v.y)),
                                                  __builtin_elementwise_maximum(two(v.z), two(v.w)));
    return maximum((float)a[0], (float)a[1]);
  } else {
    float m = entry<T>(v, 0);
#pragma unroll
    for (int j = 1; j < 16 / (int)sizeof(T); ++j) m = maximum(m, entry<T>(v, j));
    return m;
  }
}
VH_DEV float exponent(float x, float m) { return fmaxf(x - m, FAR) * LOG2E; }  // an entry of -inf has no part

VH_DEV float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// A row's results.  One without a finite entry, or with +inf or NaN, has none.
VH_DEV float2 write_row(const Args& a, int64_t row, int64_t token, float x, float m, float l, float e) {
  const float nan = __builtin_nanf("");
  const bool good = m > -INF && m < INF;
  const float log2l = log2f(l);
  const float2 s = good ? make_float2(m, log2l * LN2) : make_float2(nan, nan);
  a.logprob[row] = token < a.vocab ? x - s.x - s.y : nan;
  a.entropy[row] = good ? fmaxf((log2l - e / l) * LN2, 0.0f) : nan;
  if (a.stats) a.stats[row] = s;
  return s;
}
VH_DEV void write_top(const Args& a, int64_t row, float2 s, int at, okey key) {
  a.top_logprob[row * a.top + at] = value_of((uint32_t)(key >> 32)) - s.x - s.y;
  a.top_token[row * a.top + at] = (uint32_t)~(uint32_t)key;
}
template <int N>
VH_DEV void write_padding(const Args& a, int64_t row) {
  if (threadIdx.x == 0) {
    a.logprob[row] = a.entropy[row] = 0.0f;
    if (a.stats) a.stats[row] = make_float2(0.0f, 0.0f);
  }
  for (int i = threadIdx.x; i < a.top; i += N) {
    a.top_logprob[row * a.top + i] = 0.0f;
    a.top_token[row * a.top + i] = -1;
  }
}

// The m-th largest of a wave's ranks, found bit by bit.
VH_DEV uint32_t largest(uint32_t mine, int m) {
  uint32_t bound = 0u;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = bound | 1u << bit;
    if (__popcll(__ballot(mine >= t)) >= m) bound = t;
  }
  return bound;
}

// Of G groups, each with at least t entries that reach a bound of its own,
// the m-th largest bound is reached by m t entries: by `top`, with these.
struct Share {
  int t, m;
};
VH_DEV Share share_of(int top, int groups) {
  const int t = (top + groups - 1) / groups;
  return Share{t, (top + t - 1) / t};
}

// The `top` largest of n keys, in order, with 0 for those that are not there.
template <int N>
VH_DEV void rank_keys(const okey* keys, int n, int top, okey* best) {
  for (int i = threadIdx.x; i < top; i += N) best[i] = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += N) {
    const okey mine = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < top) best[above] = mine;
  }
  __syncthreads();
}

// How many of the workgroup's threads' counts there are together.
VH_DEV int count_all(int n, int* s_n) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_n[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) n += s_n[w];
  return n;
}

// NV vectors of 16 bytes a thread.  TOP: with alternatives.  Three workgroups a CU, for
// which the compiler spills some registers of these (4001 rows of 32,000 in bfloat16
// with twenty: 102 us with two, 90 with three; in float16 with one 72 and 69).
template <typename T, int NV, bool TOP>
__global__ void __launch_bounds__(THREADS, 6) k_score(Args a) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float s_f[3][WAVES];
  __shared__ uint32_t s_bound[WAVES];
  __shared__ int s_n[WAVES];
  __shared__ uint32_t s_count;
  __shared__ float2 s_stats;
  __shared__ okey s_key[CANDIDATES], s_best[MAX_TOP];
  const int64_t row = blockIdx.x / (uint32_t)a.pieces;
  const int piece = (int)(blockIdx.x - row * a.pieces);
  const int64_t token = a.tokens[row];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (token < 0) {
    if (piece == 0) write_padding<THREADS>(a, row);
    return;
  }
  const T* x = logits_of<T>(a, row);
  const int begin = (int)(piece * a.piece), end = (int)(begin + a.piece < a.vocab ? begin + a.piece : a.vocab);
  const int first = begin + threadIdx.x * VEC;
  uint4 v[NV];  // as they are held: converted where they are used
  if (end >= VEC) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load16<T>(x, first + i * THREADS * VEC, end);
    const int whole = (end - begin) / (THREADS * VEC);  // rounds of vectors that lie in the row
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i >= whole) v[i] = shift16<T>(v[i], first + i * THREADS * VEC, end);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load_short<T>(x, i == 0 && threadIdx.x == 0 ? end : 0);
  }
  float m = -INF, most[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    most[i] = largest_entry<T>(v[i]);
    m = maximum(m, most[i]);
  }
  const float lane_most = m;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = maximum(m, __shfl_xor(m, d));
  if (lane == 0) s_f[0][wave] = m;
  if (threadIdx.x == 0) s_count = 0u;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = maximum(m, s_f[0][w]);
  const float ref = m > -INF && m < INF ? m : 0.0f;
  // (x - m) log2(e) is one operation less as x log2(e) - m log2(e) (2048 rows of 128,000
  // in bfloat16: 110 and 102 us): what the second product's rounding leaves out, `off`,
  // is in all exponents alike, and is taken out of their sums.  Maxima that are too far for
  // that, and could overflow, are subtracted first.
  const bool near = __is_same(T, _Float16) || fabsf(ref) < 65536.0f;
  const float folded = ref * LOG2E, off = near ? __builtin_fmaf(ref, LOG2E, -folded) : 0.0f;
  float l = 0.0f, e = 0.0f;
  const auto sums = [&](auto power) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 w = convert_again(v[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = power(entry<T>(w, j)), p = exp2_fast(d);
        l += p;
        e = __builtin_fmaf(p, d, e);
      }
    }
  };
  if (near) sums([&](float x) { return fmaxf(__builtin_fmaf(x, LOG2E, -folded), FAR); });
  else sums([&](float x) { return exponent(x, ref); });
  l = wave_sum(l);
  e = wave_sum(e);
  if (lane == 0) {
    s_f[1][wave] = l;
    s_f[2][wave] = e;
  }
  if constexpr (TOP) {
    // the t-th largest of the lanes' maxima of a wave: as many of its entries reach that
    const uint32_t bound = largest(rank_of(lane_most), share_of(a.top, WAVES).t);
    if (lane == 0) s_bound[wave] = bound;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = e = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      l += s_f[1][w];
      e += s_f[2][w];
    }
    const float by = exp2f(-off);  // d = (x - m) log2(e) + off: sums of 2^(d - off), and of its products with d - off
    e = (e - off * l) * by;
    l *= by;
    if (a.part) {
      float* part = a.part + (row * a.pieces + piece) * 3;
      part[0] = m;
      part[1] = l;
      part[2] = e;
    } else {
      s_stats = write_row(a, row, token, token < a.vocab ? (float)x[token] : 0.0f, m, l, e);
    }
  }
  if constexpr (!TOP) return;
  // every entry's rank and index, once more
  const auto each = [&](float least, auto f) {  // of vectors that reach `least`, or hold a NaN
    int from = first;
    asm volatile("" : "+v"(from));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (most[i] < least) continue;
      const uint4 w = convert_again(v[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        f(rank_of(entry<T>(w, j)), (uint32_t)(from + i * THREADS * VEC + j));
      }
    }
  };
  uint32_t bound = 0u;  // the m-th largest of the waves'
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    int reach = 0;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) reach += s_bound[u] >= s_bound[w];
    if (reach >= share_of(a.top, WAVES).m) bound = umax32(bound, s_bound[w]);
  }
  // The last index of entries at the bound that count: what stands in for entries
  // past the end is -inf, as low as an entry can be, and so at the bound at most.
  uint32_t upto = (uint32_t)end - 1u;
  // Entries that reach the bound; where ties make them too many, the bound is
  // made the top-th largest value itself, and of those at it the first are taken.
  for (int again = 0; again < 2; ++again) {
    each(value_of(bound), [&](uint32_t r, uint32_t at) {
      if (r > bound || (r == bound && at <= upto)) {
        const uint32_t n = atomicAdd(&s_count, 1u);  // in any order: they are ranked below
        if (n < CANDIDATES) s_key[n] = key_of(r, at);
      }
    });
    __syncthreads();
    if (again || s_count <= CANDIDATES) break;
    bound = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = bound | 1u << bit;
      int n = 0;
      each(-INF, [&](uint32_t r, uint32_t) { n += r >= t; });
      if (count_all(n, s_n) >= a.top) bound = t;
    }
    int above = 0;
    each(-INF, [&](uint32_t r, uint32_t) { above += r > bound; });
    const int need = a.top - count_all(above, s_n);
    upto = 0u;  // the largest index that fewer than `need` ties come before
    for (int bit = 30; bit >= 0; --bit) {
      const uint32_t t = upto | 1u << bit;
      int n = 0;
      each(-INF, [&](uint32_t r, uint32_t at) { n += r == bound && at < t; });
      if (count_all(n, s_n) < need) upto = t;
    }
    upto = min(upto, (uint32_t)end - 1u);
    if (threadIdx.x == 0) s_count = 0u;
    __syncthreads();
  }
  const int n = (int)s_count;
  if (a.part) {
    rank_keys<THREADS>(s_key, n, a.top, s_best);
    for (int i = threadIdx.x; i < a.top; i += THREADS) a.part_top[(row * a.pieces + piece) * a.top + i] = s_best[i];
  } else {
    rank_keys<THREADS>(s_key, n, a.top, s_best);
    for (int i = threadIdx.x; i < a.top; i += THREADS) write_top(a, row, s_stats, i, s_best[i]);
  }
}

// A row's pieces joined.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) k_score_join(Args a) {
  __shared__ float2 s_stats;
  __shared__ uint32_t s_count;
  __shared__ okey s_bound;
  __shared__ okey s_key[MAX_PIECES * MAX_TOP], s_best[MAX_TOP];
  const int64_t row = blockIdx.x;
  const int64_t token = a.tokens[row];
  if (token < 0) return;
  const okey* lists = a.part_top + row * a.pieces * a.top;
  const int listed = a.pieces * a.top;
  const okey early = (int)threadIdx.x < listed ? lists[threadIdx.x] : 0ull;  // on its way while the rest is found
  if (threadIdx.x < 64) {
    const int p = threadIdx.x;
    const float* part = a.part + (row * a.pieces + (p < a.pieces ? p : 0)) * 3;
    const float mine = p < a.pieces ? part[0] : -INF;
    const float x = token < a.vocab ? (float)logits_of<T>(a, row)[token] : 0.0f;
    float to = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) to = maximum(to, __shfl_xor(to, d));
    const bool in = mine > -INF && p < a.pieces;
    const float by = in ? exponent(mine, to) : 0.0f, f = in ? exp2_fast(by) : 0.0f;
    const float l = wave_sum(in ? part[1] * f : 0.0f);
    const float e = wave_sum(in ? __builtin_fmaf(part[1], by, part[2]) * f : 0.0f);
    if (a.top > 0) {  // lists are in order: t keys of one reach its t-th
      const Share by = share_of(a.top, a.pieces);
      const uint32_t reach = largest(p < a.pieces ? (uint32_t)(lists[p * a.top + by.t - 1] >> 32) : 0u, by.m);
      if (p == 0) s_bound = reach > 0u ? (okey)reach << 32 : 1ull;
    }
    if (p == 0) {
      s_stats = write_row(a, row, token, x, to, l, e);
      s_count = 0u;
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  const okey bound = s_bound;
  for (int i = threadIdx.x; i < listed; i += JOIN_THREADS) {
    const okey key = i < JOIN_THREADS ? early : lists[i];
    if (key >= bound) s_key[atomicAdd(&s_count, 1u)] = key;
  }
  __syncthreads();
  rank_keys<JOIN_THREADS>(s_key, (int)s_count, a.top, s_best);
  for (int i = threadIdx.x; i < a.top; i += JOIN_THREADS) write_top(a, row, s_stats, i, s_best[i]);
}

// Entries of the gradient that single entries' gradients are added to, in
// the order in which they are given: the token's, then the alternatives'.
template <typename T>
__global__ void __launch_bounds__(BACK_THREADS) k_score_back(Args a) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ uint32_t s_at[MAX_TOP + 1];
  __shared__ float s_add[MAX_TOP + 1];
  __shared__ int s_n;
  __shared__ float s_sum;
  const int64_t row = blockIdx.x / a.chunks;
  const int begin = (int)(blockIdx.x - row * a.chunks) * (BACK_THREADS * BACK_VECTORS * VEC);
  const int end = begin + BACK_THREADS * BACK_VECTORS * VEC < a.vocab ? begin + BACK_THREADS * BACK_VECTORS * VEC : (int)a.vocab;
  const int64_t token = a.tokens[row];
  const T* x = logits_of<T>(a, row);
  T* out = (T*)a.grad + row * a.vocab;
  const float gp = token < 0 || !a.g_logprob ? 0.0f : token < a.vocab ? a.g_logprob[row] : __builtin_nanf("");
  if (threadIdx.x < 64) {
    const int k = threadIdx.x;
    const bool some = a.g_top && token >= 0 && k < a.top;
    const float t = some ? a.g_top[row * a.top + k] : 0.0f;
    const int64_t at = some ? a.top_token[row * a.top + k] : -1;
    const bool first = k == 0 && gp != 0.0f && token >= begin && token < end;
    const bool in = some && at >= begin && at < end;
    const uint64_t before = __ballot(in) & ((1ull << k) - 1ull);
    const int shift = __shfl(first ? 1 : 0, 0);
    if (first) {
      s_at[0] = (uint32_t)token;
      s_add[0] = gp;
    }
    if (in) {
      s_at[shift + __popcll(before)] = (uint32_t)at;
      s_add[shift + __popcll(before)] = t;
    }
    const int n = shift + __popcll(__ballot(in));
    const float sum = wave_sum(t);
    if (k == 0) {
      s_n = n;
      s_sum = sum + gp;
    }
  }
  __syncthreads();
  const float2 st = a.stats[row];
  const float h = a.g_entropy && token >= 0 ? a.g_entropy[row] : 0.0f;
  const float c0 = h == 0.0f ? s_sum : __builtin_fmaf(h, a.entropy[row], s_sum);
  const int n = s_n;
#pragma unroll
  for (int i = 0; i < BACK_VECTORS; ++i) {
    const int at = begin + (i * BACK_THREADS + (int)threadIdx.x) * VEC;
    if (at >= end) break;
    const bool whole = at + VEC <= end;
    float v[VEC];
    if (token < 0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
    } else {
      const uint4 raw = a.vocab < VEC ? load_short<T>(x, end) : shift16<T>(load16<T>(x, at, end), at, end);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float y = entry<T>(raw, j), d = fmaxf(y - st.x, FAR) - st.y;
        const float nan = y != y || st.x != st.x ? __builtin_nanf("") : 0.0f;  // fmaxf loses it
        v[j] = nan - exp2_fast(d * LOG2E) * __builtin_fmaf(h, d, c0);
      }
      for (int k = 0; k < n; ++k) {
        const uint32_t j0 = s_at[k] - (uint32_t)at;
        if (j0 < (uint32_t)VEC) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[j] += (uint32_t)j == j0 ? s_add[k] : 0.0f;
        }
      }
    }
    if (whole) {
      T e[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = (T)v[j];
      __builtin_memcpy(out + at, e, 16);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (at + j < end) out[at + j] = (T)v[j];
    }
  }
}

// How rows fall into pieces.  A piece of 8 vectors a thread keeps the joining
// small; where rows are few, smaller pieces fill the card: until there are 256.
// (us in a graph at 1, 256 and 1024: 1 row of 128,000 in bfloat16 with twenty 17.5,
// 12.0, 12.0; 32 rows 19.7, 15.0, 16.6; 300 rows of 32,000 with five 15.5, 14.9, 19.3.)
struct Plan {
  int nv, pieces;
  int64_t piece;
};
Plan plan_of(const vh_score_desc* d) {
  const int vec = d->dtype == VH_F32 ? 4 : 8;
  Plan p{8, 1, 0};
  const auto pieces = [&](int nv) { return (d->vocab + (int64_t)nv * vec * THREADS - 1) / ((int64_t)nv * vec * THREADS); };
  // the fewest vectors that hold a row, or its pieces; then fewer where the card is not full
  while (p.nv > 1 && pieces(p.nv / 2) == pieces(p.nv)) p.nv /= 2;
  while (p.nv > 1 && d->rows * pieces(p.nv) < 256 && pieces(p.nv / 2) <= MAX_PIECES) p.nv /= 2;
  p.pieces = (int)pieces(p.nv);
  p.piece = ((d->vocab + p.pieces - 1) / p.pieces + vec - 1) / vec * vec;
  return p;
}

int check(const vh_score_desc* d, const char* what) {
  VH_REQUIRE(d, "%s: null descriptor", what);
  VH_REQUIRE(vh::is_float_dtype(d->dtype), "%s: dtype must be bfloat16, float16 or float32", what);
  VH_REQUIRE(d->rows >= 0 && d->rows < VH_SCORE_MAX_ROWS, "%s: at most %d rows", what, VH_SCORE_MAX_ROWS - 1);
  VH_REQUIRE(d->vocab > 0 && d->vocab <= VH_SCORE_MAX_VOCAB, "%s: a vocabulary of 1 to %d", what, VH_SCORE_MAX_VOCAB);
  VH_REQUIRE(d->top >= 0 && d->top <= MAX_TOP && d->top <= d->vocab, "%s: at most %d alternatives, and no more than the vocabulary",
             what, MAX_TOP);
  return VH_OK;
}

int64_t part_bytes(const vh_score_desc* d, const Plan& p) {  // of the keys: 8 bytes each
  return p.pieces > 1 ? d->rows * p.pieces * (8ll * d->top + 12) : 0;
}

Args args_of(const vh_score_desc* d, int64_t batch_rows, int64_t batch_st) {
  Args a{};
  a.x = d->logits;
  a.x_st = d->logits_st;
  a.batch_rows = batch_rows < d->rows ? (uint32_t)batch_rows : 0u;
  a.batch_st = batch_st;
  a.vocab = d->vocab;
  a.rows = d->rows;
  a.tokens = d->tokens;
  a.top = d->top;
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.stats = (float2*)d->stats;
  a.top_logprob = d->top_logprob;
  a.top_token = d->top_token;
  a.g_logprob = d->g_logprob;
  a.g_entropy = d->g_entropy;
  a.g_top = d->g_top;
  a.grad = d->grad;
  return a;
}

template <typename T, int NV>
void launch_of(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * a.pieces));
  if (a.top > 0) hipLaunchKernelGGL((k_score<T, NV, true>), grid, dim3(THREADS), 0, s, a);
  else hipLaunchKernelGGL((k_score<T, NV, false>), grid, dim3(THREADS), 0, s, a);
}
template <typename T>
void launch(const Args& a, const Plan& p, hipStream_t s) {
  if (p.nv == 1) launch_of<T, 1>(a, s);
  else if (p.nv == 2) launch_of<T, 2>(a, s);
  else if (p.nv == 4) launch_of<T, 4>(a, s);
  else launch_of<T, 8>(a, s);
  if (a.pieces > 1) hipLaunchKernelGGL((k_score_join<T>), dim3((unsigned)a.rows), dim3(JOIN_THREADS), 0, s, a);
}

int forward(const vh_score_desc* d, int64_t batch_rows, int64_t batch_st, void* work, int64_t work_bytes, vh_stream_t stream,
            const char* what) {
  if (d->rows == 0) return VH_OK;
  VH_REQUIRE(d->logits && d->tokens && d->logprob && d->entropy && (d->top == 0 || (d->top_logprob && d->top_token)),
             "%s: null argument", what);
  const Plan p = plan_of(d);
  // a launch has fewer than 2^32 threads
  VH_REQUIRE(d->rows * p.pieces < VH_SCORE_MAX_ROWS, "%s: too many rows of such a vocabulary", what);
  const int64_t need = part_bytes(d, p);
  VH_REQUIRE(need == 0 || (work && work_bytes >= need && (uintptr_t)work % 16 == 0),
             "%s: needs %lld bytes of aligned workspace", what, (long long)need);
  Args a = args_of(d, batch_rows, batch_st);
  a.piece = p.piece;
  a.pieces = p.pieces;
  if (need > 0) {
    a.part_top = (okey*)work;
    a.part = (float*)(a.part_top + d->rows * p.pieces * d->top);
  }
  hipStream_t s = vh::as_stream(stream);
  if (d->dtype == VH_BF16) launch<__bf16>(a, p, s);
  else if (d->dtype == VH_F16) launch<_Float16>(a, p, s);
  else launch<float>(a, p, s);
  return vh::check_launch(what);
}

int backward(const vh_score_desc* d, int64_t batch_rows, int64_t batch_st, vh_stream_t stream, const char* what) {
  if (d->rows == 0) return VH_OK;
  VH_REQUIRE(d->logits && d->tokens && d->entropy && d->stats && d->grad && (!d->g_top || d->top == 0 || d->top_token),
             "%s: null argument", what);
  Args a = args_of(d, batch_rows, batch_st);
  const int64_t each = (int64_t)BACK_THREADS * BACK_VECTORS * (d->dtype == VH_F32 ? 4 : 8);
  a.chunks = (uint32_t)((d->vocab + each - 1) / each);
  const int64_t blocks = d->rows * a.chunks;
  VH_REQUIRE(blocks < (1ll << 24), "%s: too many rows of such a vocabulary", what);  // as above
  const dim3 grid((unsigned)blocks);
  hipStream_t s = vh::as_stream(stream);
  if (d->dtype == VH_BF16) hipLaunchKernelGGL(k_score_back<__bf16>, grid, dim3(BACK_THREADS), 0, s, a);
  else if (d->dtype == VH_F16) hipLaunchKernelGGL(k_score_back<_Float16>, grid, dim3(BACK_THREADS), 0, s, a);
  else hipLaunchKernelGGL(k_score_back<float>, grid, dim3(BACK_THREADS), 0, s, a);
  return vh::check_launch(what);
}

int check_batches(const vh_score_batched_desc* d, const char* what) {
  VH_REQUIRE(d, "%s: null descriptor", what);
  if (int e = check(&d->score, what)) return e;
  VH_REQUIRE(d->batch_rows > 0, "%s: batches of one row at least", what);
  return VH_OK;
}

}  // namespace

extern "C" int64_t vh_score_workspace_bytes(const vh_score_desc* d) {
  if (check(d, "vh_score_workspace_bytes")) return -1;
  return d->rows == 0 ? 0 : part_bytes(d, plan_of(d));
}

extern "C" int vh_score(const vh_score_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  if (int e = check(d, "vh_score")) return e;
  return forward(d, d->rows, 0, work, work_bytes, stream, "vh_score");
}

extern "C" int vh_score_backward(const vh_score_desc* d, vh_stream_t stream) {
  if (int e = check(d, "vh_score_backward")) return e;
  return backward(d, d->rows, 0, stream, "vh_score_backward");
}

extern "C" int vh_score_batched(const vh_score_batched_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  if (int e = check_batches(d, "vh_score_batched")) return e;
  return forward(&d->score, d->batch_rows, d->batch_st, work, work_bytes, stream, "vh_score_batched");
}

extern "C" int vh_score_batched_backward(const vh_score_batched_desc* d, vh_stream_t stream) {
  if (int e = check_batches(d, "vh_score_batched_backward")) return e;
  return backward(&d->score, d->batch_rows, d->batch_st, stream, "vh_score_batched_backward");
}
