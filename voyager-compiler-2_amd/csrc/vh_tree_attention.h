// Attention of a tree of tokens over a paged cache.
//
// Node n of a sequence sees the sequence's `context` cached positions and the
// nodes on its way from the root, itself last, which are cached at positions
// context, context + 1, ...  For each of its heads
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),
//   lse = log sum_j exp(s_j)
//
// in one pass over the keys with the running maximum and sum of the softmax.
//
// The rows of one key head are its query heads at every node (row = node *
// group + head in the group), so a key is read once for all of them.  A wave
// holds 16 * NT rows as the B operand of the matrix instructions and walks
// steps of 32 keys: S^T = K Q^T leaves a lane with eight scores of one row,
// which are, rounded to 16 bits, its share of the B operand of O^T = V^T P^T,
// with no exchange between lanes (the order of keys inside a product is free,
// so V is taken in the order that S^T comes out).  Keys and values go from
// the cache to registers: a lane's share of K is contiguous, and its share of
// V, 8 keys by D / 16 channels, is transposed with byte permutes.
//
// Codes are exact in float16 (int8 as integers, E4M3 as they are), so the
// products of S are exact.  bfloat16 queries over codes are scaled by a power
// of two per row into float16; what falls under its least value is under 2^-38
// of the row's largest channel.  A key's scale multiplies its score, a value's
// scale its probability, which goes into the second product in two 16-bit parts.
//
// Two kernels.  k_tree is for few rows (a token or two of a grouped head),
// where the cache's bytes bound it: each wave takes its own keys straight from
// the cache to registers, and the four waves of a workgroup are joined through
// LDS.  k_tree_wide is for many rows, where converting codes and the softmax
// bound it: a workgroup converts each step's keys and values to 16 bits once,
// into LDS in the order of the matrix instructions' operands, for all of its
// rows.
//
// Keys are shared out by their number, which the device alone knows: every
// workgroup works out from the contexts into how many splits each sequence
// falls (a split of all sequences' keys over about `share` workgroups a row
// block), and k_tree_merge joins them.
#pragma once

#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"
#include "vh_paged.h"

namespace tree {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int WAVES = 4;
constexpr int STEP = 32;  // keys a wave takes at a time
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

struct Args {
  vh_cache c;
  const void* q;
  int64_t q_sb, q_st, q_sh;
  const int32_t* table;
  int64_t table_st;
  const int32_t* context;
  const uint64_t* masks;  // [batch, nodes, words], or NULL: each node sees those before it
  void* o;
  float* lse;                  // or NULL
  float *part_o, *part_ml;     // of the splits, or NULL: each sequence is one
  FastDiv group_div, page_div; // page_div: by 16-key tiles a page
  float scale;                 // times log2(e)
  int q_bf16, q_wide, words, batch, nodes, heads, group, rows, row_blocks, block_rows;
  int table_pages;
  uint32_t share, fill;        // workgroups that a row block's keys are shared out to at most; that fill the card
  uint32_t units;              // most splits of all sequences together
};

// The keys that rows [row0, row0 + block_rows) of sequence b can see: up to
// their last node.  0 where the sequence does not fit its pages.
VH_DEV bool fits(const Args& a, int ctx) {
  return ctx >= 0 && (int64_t)ctx + a.nodes <= (int64_t)a.table_pages * a.c.page;
}
VH_DEV int visible(const Args& a, int ctx, int row0) {
  const int last = row0 + a.block_rows < a.rows ? row0 + a.block_rows : a.rows;
  return fits(a, ctx) ? ctx + (int)fast_div((uint32_t)(last - 1), a.group_div) + 1 : 0;
}

// How the sequences fall into splits of `chunk` pieces of PIECE keys: the least
// with which all pieces make no more than `share` splits and a rest a sequence,
// and four where that still makes `fill`, so that a wave has steps to ask ahead
// in and a split's results are few beside its keys (8 sequences of 8192, heads
// of 256, two tokens: 42 us at one piece a split, 37 at three; one token over
// 4096 each: 28 and 22).  Every lane of a
// wave calls these together; a lane holds a sequence.
constexpr int PIECE = 128, CHUNK = 4;
constexpr uint32_t CHUNK_MOST = 0x7fffffffu / PIECE;  // more pieces than a sequence has; its keys are an int
VH_DEV uint32_t pieces(const Args& a, int b) {
  const int ctx = b < a.batch ? a.context[b] : -1;
  return fits(a, ctx) && b < a.batch ? ((uint32_t)ctx + a.nodes + PIECE - 1) / PIECE : 0u;
}
VH_DEV uint32_t chunk_of(const Args& a) {
  const int lane = threadIdx.x & 63;
  uint32_t all = 0u;
  if (a.batch == 1) {
    all = pieces(a, 0);
  } else {
    for (int b0 = 0; b0 < a.batch; b0 += 64) all += pieces(a, b0 + lane);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += (uint32_t)__shfl_xor((int)all, d);
  }
  all = (uint32_t)__builtin_amdgcn_readfirstlane((int)all);
  if (all == 0u) return 1u;
  const uint32_t least = all / a.share + (all % a.share ? 1u : 0u);
  return least >= CHUNK ? min(least, CHUNK_MOST) : max(least, min((uint32_t)CHUNK, (all + a.fill - 1) / a.fill));
}
VH_DEV uint32_t splits_of(uint32_t piece, uint32_t chunk) { return piece <= chunk ? 1u : (piece + chunk - 1) / chunk; }

// The sequence and split of `unit`; b < 0 past the last.
struct Span {
  int b;
  uint32_t split, chunk;
};
VH_DEV Span span_of(const Args& a, uint32_t unit) {
  Span s{-1, 0u, chunk_of(a)};
  if (a.batch == 1) {  // the scan over sequences is a microsecond of a lone token's
    if (unit < splits_of(pieces(a, 0), s.chunk)) {
      s.b = 0;
      s.split = unit;
    }
    return s;
  }
  const int lane = threadIdx.x & 63;
  uint32_t before = 0u;
  for (int b0 = 0; b0 < a.batch && s.b < 0; b0 += 64) {
    const uint32_t n = b0 + lane < a.batch ? splits_of(pieces(a, b0 + lane), s.chunk) : 0u;
    uint32_t upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t y = (uint32_t)__shfl_up((int)upto, d);
      upto += lane >= d ? y : 0u;
    }
    const uint64_t past = __ballot(before + upto > unit);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      s.b = b0 + at;
      s.split = unit - before - (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), at);
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.split = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.split);
  return s;
}

VH_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four E4M3 codes, or two pairs of int8 codes + 128, as float16.
VH_DEV uint32_t int8_pair(uint32_t spread) {  // bytes 0 and 2 hold the codes
  const f16x2 h = __builtin_bit_cast(f16x2, spread | 0x64006400u);  // 1024 + code + 128
  return __builtin_bit_cast(uint32_t, h - f16x2{(_Float16)1152.0f, (_Float16)1152.0f});
}
VH_DEV uint32_t e4m3_pair(uint32_t w, bool hi) {
  const f16x2 h = hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true)
                     : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false);
  return __builtin_bit_cast(uint32_t, h);
}

// Four codes as float16, in order.
template <int FMT>
VH_DEV uint2 codes4(uint32_t w) {
  if constexpr (FMT == CACHE_E4M3) return make_uint2(e4m3_pair(w, false), e4m3_pair(w, true));
  else return make_uint2(int8_pair(__builtin_amdgcn_perm(0u, w, 0x0c010c00u)), int8_pair(__builtin_amdgcn_perm(0u, w, 0x0c030c02u)));
}

// Element e of four rows, side by side in 16 bits: a column of the transposed
// values.  A row's dword holds four codes or two 16-bit values.
template <int FMT>
VH_DEV uint2 turn4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, int e) {
  if constexpr (FMT == CACHE_E4M3) {  // the converter takes its codes side by side
    const uint32_t two = e < 2 ? 0x05010400u : 0x07030602u;
    const uint32_t lo = __builtin_amdgcn_perm(r1, r0, two), hi = __builtin_amdgcn_perm(r3, r2, two);
    return codes4<FMT>(__builtin_amdgcn_perm(hi, lo, e & 1 ? 0x07060302u : 0x05040100u));
  } else if constexpr (FMT == CACHE_INT8) {
    const uint32_t sel = 0x0c040c00u + e * 0x00010001u;
    return make_uint2(int8_pair(__builtin_amdgcn_perm(r1, r0, sel)), int8_pair(__builtin_amdgcn_perm(r3, r2, sel)));
  } else {
    const uint32_t sel = e ? 0x07060302u : 0x05040100u;
    return make_uint2(__builtin_amdgcn_perm(r1, r0, sel), __builtin_amdgcn_perm(r3, r2, sel));
  }
}

template <int FMT>
VH_DEV f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  if constexpr (FMT == CACHE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two float32 values to packed 16-bit ones, half to even.
template <int FMT>
VH_DEV uint32_t pack2(float x, float y) {
  const f32x2 v = {x, y};
  if constexpr (FMT == CACHE_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int FMT>
VH_DEV f32x2 unpack2(uint32_t w) {
  if constexpr (FMT == CACHE_BF16) return f32x2{bf2f(w & 0xffffu), bf2f(w >> 16)};
  else return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
}

// The 16-bit halves of w that are infinite or NaN, as a mask of their bits.
template <int FMT>
VH_DEV uint32_t nonfinite(uint32_t w) {
  const uint32_t e = FMT == CACHE_BF16 ? 0x7f80u : 0x7c00u;
  return ((w & e) == e ? 0xffffu : 0u) | (((w >> 16) & e) == e ? 0xffff0000u : 0u);
}

// sum, and NaN where a half of w is infinite or NaN: w times zero added.
template <int FMT>
VH_DEV float times_zero(uint32_t w, float sum) {
  if constexpr (FMT == CACHE_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0u), sum, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0u), sum, false);
}

// Over the four lanes that hold a row, 16 apart, by register swaps: rows of
// 16 lanes, then halves of the wave.
VH_DEV float max_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
VH_DEV float sum_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The queries of NT tiles of 16 rows from row0 on as the B operand: column r is
// a row, k the lane's share of D as `chan(s)` says (8 channels from there on).
template <int NT, int KS, typename F>
VH_DEV void load_queries(const Args& a, int b, int h, int row0, uint4 (&Q)[NT][KS], int (&node)[NT], F chan) {
  const int r = threadIdx.x & 15;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 16 * nt + r;
    const int at = row < a.rows ? row : a.rows - 1;
    node[nt] = (int)fast_div((uint32_t)at, a.group_div);
    const int head = h * a.group + at - node[nt] * a.group;
    const uint16_t* q = (const uint16_t*)a.q + b * a.q_sb + node[nt] * a.q_st + head * a.q_sh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = chan(s);
      if (a.q_wide) {
        Q[nt][s] = *(const uint4*)(q + c);
      } else {
        Q[nt][s] = make_uint4(q[c] | (uint32_t)q[c + 1] << 16, q[c + 2] | (uint32_t)q[c + 3] << 16,
                              q[c + 4] | (uint32_t)q[c + 5] << 16, q[c + 6] | (uint32_t)q[c + 7] << 16);
      }
    }
  }
}

// Queries over codes become float16, scaled by a power of two a row; `fac`
// takes it out of the row's products, with the softmax's scale.
template <int NT, int KS, bool TO_F16>
VH_DEV void convert_queries(const Args& a, uint4 (&Q)[NT][KS], float (&fac)[NT]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    fac[nt] = a.scale;
    if (TO_F16 && a.q_bf16) {
      uint32_t key = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t w[4] = {Q[nt][s].x, Q[nt][s].y, Q[nt][s].z, Q[nt][s].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) key = umax32(key, umax32((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
      }
      key = umax32(key, (uint32_t)__shfl_xor((int)key, 16));
      key = umax32(key, (uint32_t)__shfl_xor((int)key, 32));
      // the largest channel to [2^14, 2^15); a row with an infinity or NaN stays as it is
      int e = (int)(key >> 23) - 127;
      e = e > 127 ? 14 : e < -100 ? -100 : e;
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
      fac[nt] *= __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t w[4] = {Q[nt][s].x, Q[nt][s].y, Q[nt][s].z, Q[nt][s].w};
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = pack2<CACHE_F16>(bf2f(w[i] & 0xffffu) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
        Q[nt][s] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
}

// y, or x where c, for values of one structure: as a choice the compiler would
// choose between their addresses, and keep the structure in memory.
template <typename T>
VH_DEV T either(bool c, T x, T y) {
  return y ^ ((x ^ y) & -(T)c);
}

// Two 16-key tiles of the cache: where their rows lie and how many exist.
struct Step {
  int64_t row[2];
  int live[2];
};

// Finds the tiles of keys [key0, key0 + 32) that lie under `end`.  A wave holds
// 64 entries of its table, one a lane, so that a step's pages need no load.
struct Finder {
  const int32_t* table;
  FastDiv page_div;
  int64_t page_rows, head_rows;
  uint32_t pages, page, last;  // last: the table's last entry
  uint32_t first;              // of the entries held
  int held, end;
  int bad;  // a page was not there: nothing of it is seen

  // from key `begin` on, under `end`
  __device__ __forceinline__ Finder(const Args& a, int b, int h, int begin, int end_)
      : table(a.table + (int64_t)b * a.table_st), page_div(a.page_div), page_rows((int64_t)a.c.kv_heads * a.c.page),
        head_rows((int64_t)h * a.c.page), pages((uint32_t)a.c.pages), page((uint32_t)a.c.page),
        last((uint32_t)a.table_pages - 1u), first(0u), held(0), end(end_), bad(0) {
    if (begin < end) hold(fast_div((uint32_t)begin >> 4, page_div));
  }
  __device__ __forceinline__ void hold(uint32_t from) {
    first = from;
    const uint32_t at = from + (threadIdx.x & 63);
    held = table[at < last ? at : last];
  }
  __device__ __forceinline__ Step operator()(int key0) {
    Step st;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int left = end - (key0 + 16 * t);
      // a tile past the end is read where a key lies, and not seen
      const uint32_t tile = (uint32_t)(left > 0 ? key0 + 16 * t : end - 1) >> 4;
      const uint32_t pg = fast_div(tile, page_div);
      if (pg - first >= 64u) hold(pg);
      const int id = __builtin_amdgcn_readlane(held, (int)(pg - first));
      const bool there = (uint32_t)id < pages;
      bad |= there ? 0 : 1;
      st.live[t] = !there || left < 0 ? 0 : left < 16 ? left : 16;
      st.row[t] = (there ? id : 0) * page_rows + head_rows + (tile * 16 - pg * page);
    }
    return st;
  }
};

// The keys of a step that the lane's rows see, as bits 4 t + i.
template <int NT>
VH_DEV void see(const Args& a, int b, int ctx, int key0, const int (&live)[2], const int (&node)[NT], uint32_t (&seen)[NT]) {
  const int g = (threadIdx.x & 63) >> 4;
  const int n0 = key0 - ctx;  // the first key's node, if it is one
  const uint32_t there = ((1u << live[0]) - 1u) | ((1u << live[1]) - 1u) << 16;
  uint32_t window[NT];  // bit j: key key0 + j
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) window[nt] = 0xffffffffu;
  if (n0 > -STEP) {
    if (a.masks) {
      const int sh = n0 < 0 ? 0 : n0 & 63, w = n0 < 0 ? 0 : n0 >> 6;
      uint64_t lo[NT], hi[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t* m = a.masks + ((int64_t)b * a.nodes + node[nt]) * a.words;
        lo[nt] = m[w < a.words ? w : a.words - 1];
        hi[nt] = m[w + 1 < a.words ? w + 1 : a.words - 1];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t l = w < a.words ? lo[nt] : 0ull, h = w + 1 < a.words ? hi[nt] : 0ull;
        const uint32_t x = (uint32_t)(l >> sh | (sh ? h << (64 - sh) : 0ull));
        window[nt] = n0 < 0 ? x << -n0 | ((1u << -n0) - 1u) : x;
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int last = node[nt] - n0;
        window[nt] = last < 0 ? 0u : last >= STEP - 1 ? 0xffffffffu : (2u << last) - 1u;
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const uint32_t x = (window[nt] & there) >> (4 * g);
    seen[nt] = (x & 0xfu) | (x >> 12 & 0xf0u);
  }
}

// A step's softmax is in two forms.  S: products of key 16 t + 4 g + i and row
// 16 nt + r; ks, vs: the keys' scales; m, l: a row's reference (its maximum, or
// under it) and a lane's part of its sum; top: over codes, the largest probability times value scale that
// the row has seen.
//
// The operand of the second product is p * vs in the unit of its row, a power
// of two by `top`.  Only keys that the row sees count: what another branch, a
// node that pads or an old row behind the sequence holds does not move it.
//
// The sum takes a probability in float32, the operand rounds it to float16,
// whose least is 2^-24: the largest operand is placed under 2^PLACE, so that one
// of 2^-34 of it still counts (at 1, 32768 keys of 2^-26 beside one were in the
// sum and not in the product, half of a result).  Over codes the unit does it;
// float16 values have the reference of the softmax, m, that far under the maximum.
// bfloat16 has the range of float32 and needs no place: there the maximum is put
// at 2^-20, so that sums of probabilities times values near the type's largest
// stay finite, as their result is.
//
// In the quick form, for a step that every row sees, nothing moves: the
// probabilities are taken against the reference as it is, and the step is given
// up (true) where an operand passes 2^5 times its place or where a row has no
// reference yet.  It needs no maximum over lanes, and its loop holds no branch
// that writes the accumulators (with one, the compiler keeps two copies of them).
// After the first steps the maximum seldom rises by five binades.
constexpr int PLACE = 10;
template <int FMT>
constexpr float operand_most() { return FMT == CACHE_BF16 ? 0x1p-15f : 0x1p15f; }
// What lies between a row's maximum and its reference, in binades.
template <int FMT>
constexpr float reference_under() { return FMT == CACHE_F16 ? 10.0f : FMT == CACHE_BF16 ? -20.0f : 0.0f; }
// Bounds on a probability and on a value scale in a row's unit, so that no sum
// and no product of the quick form passes float32.
constexpr float QUICK_MOST = 0x1p100f;

VH_DEV float unit_of(float top) {  // top / 2^PLACE, up to the next power of two; 2^-126 at least
  constexpr uint32_t LEAST = (uint32_t)PLACE << 23;
  const uint32_t e = __float_as_uint(top) & 0x7f800000u;
  return __uint_as_float((e < LEAST ? LEAST : e) - LEAST + 0x00800000u);
}
// A row's sum brought to [1/2, 1) by a power of two, which the reference takes
// and by which the accumulators are to be multiplied: they then are no larger
// than the largest value.
VH_DEV float bring(float& L, float& M) {
  const int e = __builtin_amdgcn_frexp_expf(L);
  L = __builtin_amdgcn_ldexpf(L, -e);
  M += (float)e;
  return __builtin_amdgcn_ldexpf(1.0f, -e);
}

VH_DEV float inverse_unit(float top) { return __uint_as_float(0x7f000000u - __float_as_uint(unit_of(top))); }

template <int FMT, int NT>
VH_DEV bool quick(const f32x4 (&S)[2][NT], const f32x4 (&ks)[2], const f32x4 (&vs)[2], const float (&fac)[NT],
                  const float (&m)[NT], const float (&top)[NT], f32x4 (&p)[2][NT]) {
  constexpr bool BYTE = FMT == CACHE_E4M3 || FMT == CACHE_INT8;
  bool far = false;
  float high = 0.0f;
  if constexpr (BYTE) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      high = fmaxf(fmaxf(high, vs[t][0]), vs[t][1]);
      high = fmaxf(fmaxf(high, vs[t][2]), vs[t][3]);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float inv = BYTE ? inverse_unit(top[nt]) : 1.0f;
    float most = 0.0f, operand = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[t][nt][i] = exp2_fast(fmaf(S[t][nt][i], BYTE ? ks[t][i] * fac[nt] : fac[nt], -m[nt]));
      most = fmaxf(fmaxf(most, p[t][nt][0]), p[t][nt][1]);
      most = fmaxf(fmaxf(most, p[t][nt][2]), p[t][nt][3]);
      if constexpr (BYTE) {
        const f32x4 w = vs[t] * inv;
        operand = fmaxf(fmaxf(operand, p[t][nt][0] * w[0]), p[t][nt][1] * w[1]);
        operand = fmaxf(fmaxf(operand, p[t][nt][2] * w[2]), p[t][nt][3] * w[3]);
      }
    }
    far |= m[nt] == -__builtin_inff();
    if constexpr (BYTE) far |= operand > operand_most<FMT>() || most > QUICK_MOST || high * inv > QUICK_MOST;
    else far |= most > operand_most<FMT>();
  }
  return far;
}

// The other form: any step, with the maxima and the unit
// moved to where they belong.  seen: the keys that the rows see.  S becomes the
// probabilities.
template <int FMT, int CT, int NT>
VH_DEV void careful(f32x4 (&S)[2][NT], const f32x4 (&ks)[2], const f32x4 (&vs)[2], const float (&fac)[NT],
                    const uint32_t (&seen)[NT], float (&m)[NT], float (&l)[NT], float (&top)[NT], f32x4 (&acc)[CT][NT]) {
  constexpr bool BYTE = FMT == CACHE_E4M3 || FMT == CACHE_INT8;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float v = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = S[t][nt][i] * (BYTE ? ks[t][i] * fac[nt] : fac[nt]);
          S[t][nt][i] = seen[nt] >> (4 * t + i) & 1 ? x : -__builtin_inff();
          v = fmaxf(v, S[t][nt][i]);
        }
    const float to = fmaxf(m[nt], max_rows(v) - reference_under<FMT>());
    const float alpha = m[nt] == -__builtin_inff() ? 0.0f : exp2_fast(m[nt] - to);
    m[nt] = to;
    l[nt] *= alpha;
    const float ref = to == -__builtin_inff() ? 0.0f : to;
    float most = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S[t][nt][i] = exp2_fast(S[t][nt][i] - ref);
          // a scale that is not seen may be anything
          if (BYTE) most = fmaxf(most, seen[nt] >> (4 * t + i) & 1 ? S[t][nt][i] * vs[t][i] : 0.0f);
        }
    float down = alpha;
    if constexpr (BYTE) {
      const float was = unit_of(top[nt]);
      top[nt] = fmaxf(top[nt] * alpha, max_rows(most));
      down = alpha * was * inverse_unit(top[nt]);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c][nt] *= down;
  }
}

// The probabilities as the B operand of the second product (k = 4 t + i), times
// the value scales in the rows' units: in two 16-bit parts, as one would round
// them by 2^-12 of float16 or 2^-9 of bfloat16, which a result in 16 bits shows.
template <int FMT, bool MASKED, int NT>
VH_DEV void operands(const f32x4 (&p)[2][NT], const f32x4 (&vs)[2], const float (&top)[NT], const uint32_t (&seen)[NT],
                     float (&l)[NT], uint4 (&P)[NT], uint4 (&Plo)[NT]) {
  constexpr bool BYTE = FMT == CACHE_E4M3 || FMT == CACHE_INT8;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float inv = BYTE ? inverse_unit(top[nt]) : 1.0f;
    uint32_t w[4], u[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float p0 = p[t][nt][i], p1 = p[t][nt][i + 1];
        l[nt] += p0 + p1;
        if constexpr (BYTE) {
          if constexpr (MASKED) {  // the scale last: a large one in the unit of small ones would not be finite
            p0 = seen[nt] >> (4 * t + i) & 1 ? p0 * vs[t][i] * inv : 0.0f;
            p1 = seen[nt] >> (4 * t + i + 1) & 1 ? p1 * vs[t][i + 1] * inv : 0.0f;
          } else {
            p0 *= vs[t][i] * inv;
            p1 *= vs[t][i + 1] * inv;
          }
        }
        w[2 * t + i / 2] = pack2<FMT>(p0, p1);
        const f32x2 hi = unpack2<FMT>(w[2 * t + i / 2]);
        u[2 * t + i / 2] = pack2<FMT>(p0 - hi[0], p1 - hi[1]);
      }
    P[nt] = make_uint4(w[0], w[1], w[2], w[3]);
    Plo[nt] = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// Values of a step that are not finite, which were left out of the product
// (they would reach rows that do not see them as 0 * inf, and infinities times
// the low part of a probability are NaN), added to the rows that see them.
// p: the probabilities; chan(c, i): the channel of row 4 g + i of channel tile c.
template <int FMT, int CT, int NT, typename F>
VH_DEV void add_nonfinite(const Args& a, const Step& st, const f32x4 (&p)[2][NT], const uint32_t (&seen)[NT],
                          f32x4 (&acc)[CT][NT], F chan) {
  const int r = threadIdx.x & 15;
  for (int k = 0; k < STEP; ++k) {
    const int t = k >> 4, at = k & 15;
    const uint16_t* v = (const uint16_t*)a.c.v + (either(t != 0, st.row[1], st.row[0]) + at) * a.c.dim;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((at & 3) == i) mine = t ? p[1][nt][i] : p[0][nt][i];
      const int from = (at >> 2) * 16 + r;
      const float w = __shfl(mine, from);
      const bool ok = (uint32_t)__shfl((int)seen[nt], from) >> (4 * t + (at & 3)) & 1;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = v[chan(c, i)];
          if (ok && nonfinite<FMT>(x) & 0xffffu) acc[c][nt][i] += w * unpack2<FMT>(x)[0];
        }
    }
  }
}

// Whether a NaN is among the results of a wave's rows whose scores are numbers:
// then it comes from the values.
template <int CT, int NT>
VH_DEV bool nan_among(const f32x4 (&acc)[CT][NT], const float (&l)[NT]) {
  bool nan = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float sum = sum_rows(l[nt]);
    bool mine = false;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine |= acc[c][nt][i] != acc[c][nt][i];
    nan |= mine && sum == sum;
  }
  return nan;
}

template <int CT, int NT>
VH_DEV void start(float (&m)[NT], float (&l)[NT], float (&top)[NT], f32x4 (&acc)[CT][NT]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -__builtin_inff();
    l[nt] = top[nt] = 0.0f;
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}

// Four values of a row: to the splits' results, or divided and rounded to the output.
VH_DEV void put4(const Args& a, float* part, uint16_t* out, float inv, float x0, float x1, float x2, float x3) {
  if (part) *(f32x4*)part = f32x4{x0, x1, x2, x3};
  else *(uint2*)out = a.q_bf16 ? make_uint2(pack2<CACHE_BF16>(x0 * inv, x1 * inv), pack2<CACHE_BF16>(x2 * inv, x3 * inv))
                               : make_uint2(pack2<CACHE_F16>(x0 * inv, x1 * inv), pack2<CACHE_F16>(x2 * inv, x3 * inv));
}

// Where a row's results go, and its maximum and sum (g: the lane's group).
struct Place {
  float* part;
  uint16_t* out;
  float inv;
};
VH_DEV Place place(const Args& a, int b, int h, uint32_t unit, int row, int node, float M, float L, int g) {
  Place p{};
  if (a.part_o) {
    const int64_t at = ((int64_t)unit * a.c.kv_heads + h) * a.rows + row;
    if (g == 0) *(float2*)(a.part_ml + 2 * at) = make_float2(M, L);
    p.part = a.part_o + at * a.c.dim;
  } else {
    const int64_t at = ((int64_t)b * a.nodes + node) * a.heads + h * a.group + row - node * a.group;
    if (a.lse && g == 0) a.lse[at] = L == 0.0f ? -__builtin_inff() : (M + log2f(L)) * LN2;
    p.out = (uint16_t*)a.o + at * a.c.dim;
    p.inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees nothing is zero
  }
  return p;
}

// A node without itself among its ancestors pads its tree, and sees no context either.
VH_DEV bool pads(const Args& a, int b, int node) {
  return a.masks && !(a.masks[((int64_t)b * a.nodes + node) * a.words + (node >> 6)] >> (node & 63) & 1);
}

// Workgroups of row blocks that share keys are 8 apart: on one XCD, and L2.
struct Block {
  uint32_t unit;
  int h, row0;
};
VH_DEV Block block_of(const Args& a) {
  const uint32_t per = 8u * a.row_blocks, group = blockIdx.x / per, in = blockIdx.x - group * per;
  const uint32_t combo = group * 8 + in % 8;
  const uint32_t unit = combo / a.c.kv_heads;
  return Block{unit, (int)(combo - unit * a.c.kv_heads), (int)(in / 8) * a.block_rows};
}

// Waves of a SIMD that the registers are shared out for: two at least, so that
// accumulators stay where vector instructions reach them (under 256 registers
// a wave), three where a wave's 16 rows of 8-bit keys leave room.
constexpr int waves_of(int d, int fmt, int nt) {
  return nt > 1 || d > 128 ? 2 : fmt == CACHE_E4M3 || fmt == CACHE_INT8 || d == 64 ? 3 : 2;
}

// Few rows.  Each of the four waves takes steps of its own keys, straight from
// the cache to the registers that the matrix instructions read, and asks for
// the next step's as soon as this one's are used; LDS joins the waves' results
// once, at the end.
//
// Bound by the cache's bytes: 32 tokens, one a sequence, over 2048 to 8192
// cached ones, 8 int8 key heads of 128 and 32 query heads (353 MB): 76-82 us,
// 4.3-4.6 TB/s, as fast as this card's memory is read by a plain sum.  In
// bfloat16, all of 8192 (1.07 GB): 201 us with the joining, 5.3 TB/s.  One token
// over 4096 (8.7 MB): 8.8 us, the latency of table, keys, values and joining.
template <int D, int FMT, int NT>
__global__ void __launch_bounds__(WAVES * 64, waves_of(D, FMT, NT)) k_tree(Args a) {
  constexpr bool BYTE = FMT == CACHE_E4M3 || FMT == CACHE_INT8;
  constexpr int ESZ = BYTE ? 1 : 2;
  constexpr int KS = D / 32;                        // matrix instructions along D
  constexpr int KQ = D * ESZ / 64;                  // 16-byte loads of a lane's share of a key tile
  constexpr int CT = D / 16;                        // channel tiles
  constexpr int CPL = CT * ESZ > 16 ? 16 / ESZ : CT;  // channels a lane loads at once
  constexpr int VB = CT / CPL;                      // loads of a value row
  constexpr int VW = CPL * ESZ / 4;                 // dwords of one
  __shared__ f32x4 s_o[2][CT * NT * 64];
  __shared__ float s_m[WAVES][16 * NT], s_l[WAVES][16 * NT];

  const Block blk = block_of(a);
  if (blk.unit >= a.units) return;
  const Span span = span_of(a, blk.unit);
  if (span.b < 0) return;
  const int b = span.b, h = blk.h, row0 = blk.row0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int ctx = __builtin_amdgcn_readfirstlane(a.context[b]);
  const int total = visible(a, ctx, row0);
  if (!fits(a, ctx) && threadIdx.x == 0) atomicOr(a.c.flag, VH_CACHE_ERR_CONTEXT);
  const int begin = (int)(span.split * span.chunk * PIECE);
  const int end = total - begin < (int)(span.chunk * PIECE) ? total : begin + (int)(span.chunk * PIECE);

  uint4 Q[NT][KS];
  float fac[NT];  // of a row's products, in powers of two
  int node[NT];
  load_queries(a, b, h, row0, Q, node, [&](int s) { return BYTE ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; });

  f32x4 acc[CT][NT];
  float m[NT], l[NT], top[NT];
  start(m, l, top, acc);
  Finder find(a, b, h, begin, end);

  uint4 kr[2][KQ];
  uint32_t vr[2][4][VB][VW];
  f32x4 ks[2], vs[2];
  // A lane's part of a tile's rows: keys at r, channels from 16 g bytes on;
  // values at 4 g + i, channels from r CPL on.
  const uint32_t k_lane = (uint32_t)r * (D * ESZ) + g * 16, v_lane = (uint32_t)(4 * g) * (D * ESZ) + r * (CPL * ESZ);
  auto load_k = [&](const Step& st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* kp = (const uint8_t*)a.c.k + st.row[t] * (D * ESZ);
#pragma unroll
      for (int j = 0; j < KQ; ++j) kr[t][j] = *(const uint4*)(kp + k_lane + 64 * j);
      if constexpr (BYTE) ks[t] = *(const f32x4*)(a.c.k_scale + st.row[t] + 4 * g);
    }
  };
  auto load_v = [&](const Step& st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* vp = (const uint8_t*)a.c.v + st.row[t] * (D * ESZ);
      if constexpr (BYTE) vs[t] = *(const f32x4*)(a.c.v_scale + st.row[t] + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < VB; ++w) {
          const uint8_t* at = vp + v_lane + i * (D * ESZ) + w * (16 * CPL * ESZ);
          if constexpr (VW == 4) {
            const uint4 x = *(const uint4*)at;
            vr[t][i][w][0] = x.x; vr[t][i][w][1] = x.y; vr[t][i][w][2] = x.z; vr[t][i][w][3] = x.w;
          } else if constexpr (VW == 2) {
            const uint2 x = *(const uint2*)at;
            vr[t][i][w][0] = x.x; vr[t][i][w][1] = x.y;
          } else {
            vr[t][i][w][0] = *(const uint32_t*)at;
          }
        }
    }
  };

  auto products = [&](f32x4 (&S)[2][NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) S[t][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 A;
        if constexpr (BYTE) {
          const uint4 x = kr[t][s >> 1];
          const uint2 lo = codes4<FMT>(s & 1 ? x.z : x.x), hi = codes4<FMT>(s & 1 ? x.w : x.y);
          A = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          A = kr[t][s];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[t][nt] = mfma<FMT>(A, Q[nt][s], S[t][nt]);
      }
    }
  };
  // O^T += V^T P^T: A's row r of channel tile c is channel (c / CPL) 16 CPL + r CPL + c % CPL
  auto add = [&](const uint4 (&P)[NT], const uint4 (&Plo)[NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < VB; ++w)
#pragma unroll
      for (int d = 0; d < VW; ++d)
#pragma unroll
        for (int e = 0; e < 4 / ESZ; ++e) {
          const uint2 lo = turn4<FMT>(vr[0][0][w][d], vr[0][1][w][d], vr[0][2][w][d], vr[0][3][w][d], e);
          const uint2 hi = turn4<FMT>(vr[1][0][w][d], vr[1][1][w][d], vr[1][2][w][d], vr[1][3][w][d], e);
          const uint4 A = make_uint4(lo.x, lo.y, hi.x, hi.y);
          const int c = w * CPL + (4 / ESZ) * d + e;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[c][nt] = mfma<FMT>(A, P[nt], acc[c][nt]);
            acc[c][nt] = mfma<FMT>(A, Plo[nt], acc[c][nt]);
          }
        }
  };

  int key0 = begin + wave * STEP;
  if (key0 < end) {
    const int whole = end < ctx ? end : ctx;
    // the step after this; after the last it is asked for again, and not waited for
    auto after = [&]() { return key0 + WAVES * STEP < end ? key0 + WAVES * STEP : key0; };
    Step st = find(key0);
    load_k(st);
    load_v(st);
    convert_queries<NT, KS, BYTE>(a, Q, fac);
    do {
      const Step next = find(after());
      {
        f32x4 S[2][NT];
        uint32_t seen[NT];
        uint4 P[NT], Plo[NT];
        products(S);
        see<NT>(a, b, ctx, key0, st.live, node, seen);
        careful<FMT>(S, ks, vs, fac, seen, m, l, top, acc);
        operands<FMT, true>(S, vs, top, seen, l, P, Plo);
        if constexpr (!BYTE) {
          uint32_t any = 0u;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < VB; ++w)
#pragma unroll
                for (int d = 0; d < VW; ++d) {
                  const uint32_t bits = nonfinite<FMT>(vr[t][i][w][d]);
                  any |= bits;
                  vr[t][i][w][d] &= ~bits;
                }
          if (__any(any != 0u))
            add_nonfinite<FMT>(a, st, S, seen, acc, [&](int c, int i) { return (c / CPL) * 16 * CPL + (4 * g + i) * CPL + c % CPL; });
        }
        add(P, Plo);
      }
      load_k(next);
      load_v(next);
      st = next;
      key0 += WAVES * STEP;
      // the next step's keys and values are asked for as soon as this step's registers are free
      while (key0 + STEP <= whole && st.live[0] + st.live[1] == STEP) {
        const Step next = find(after());
        f32x4 S[2][NT], p[2][NT];
        uint4 P[NT], Plo[NT];
        const uint32_t all[NT] = {};
        products(S);
        const f32x4 k1[2] = {ks[0], ks[1]};
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        bool far = quick<FMT>(S, k1, vs, fac, m, top, p);
        if constexpr (!BYTE) {  // an infinity times the low part of a probability would be NaN
          float odd[2] = {0.0f, 0.0f};
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < VB; ++w)
#pragma unroll
                for (int d = 0; d < VW; ++d) odd[t] = times_zero<FMT>(vr[t][i][w][d], odd[t]);
          far |= odd[0] != odd[0] || odd[1] != odd[1];
        }
        if (__any(far)) {
          load_k(st);  // once more, seldom
          break;
        }
        operands<FMT, false>(p, vs, top, all, l, P, Plo);
        add(P, Plo);
        __builtin_amdgcn_sched_barrier(0);
        load_v(next);
        st = next;
        key0 += WAVES * STEP;
      }
    } while (key0 < end);
  }
  if (find.bad && lane == 0) atomicOr(a.c.flag, VH_CACHE_ERR_PAGE);

  // the waves joined: waves 2 and 3 onto 0 and 1, then 1 onto 0
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] = sum_rows(l[nt]);
    if (g == 0) {
      s_m[wave][16 * nt + r] = m[nt];
      s_l[wave][16 * nt + r] = l[nt];
    }
  }
  __syncthreads();
  float L[NT], M[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    M[nt] = -__builtin_inff();
    L[nt] = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M[nt] = fmaxf(M[nt], s_m[w][16 * nt + r]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float mw = s_m[w][16 * nt + r];
      L[nt] += s_l[w][16 * nt + r] * (mw == -__builtin_inff() ? 1.0f : exp2_fast(mw - M[nt]));
    }
    float f = (m[nt] == -__builtin_inff() ? 1.0f : exp2_fast(m[nt] - M[nt])) * (BYTE ? unit_of(top[nt]) : 1.0f);
    f *= bring(L[nt], M[nt]);
    const bool none = pads(a, b, node[nt]);
    if (none) {
      M[nt] = -__builtin_inff();
      L[nt] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c][nt] = none ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[c][nt] * f;
  }
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    if (half == 1) __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s_o[wave - half][(c * NT + nt) * 64 + lane] = acc[c][nt];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[c][nt] += s_o[wave][(c * NT + nt) * 64 + lane];
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 16 * nt + r;
    if (row >= a.rows) continue;
    const Place p = place(a, b, h, blk.unit, row, node[nt], M[nt], L[nt], g);
#pragma unroll
    for (int w = 0; w < VB; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < CPL; c += 4) {
          const int at = w * 16 * CPL + (4 * g + i) * CPL + c, t = w * CPL + c;
          put4(a, p.part ? p.part + at : nullptr, p.out + at, p.inv, acc[t][nt][i], acc[t + 1][nt][i], acc[t + 2][nt][i],
               acc[t + 3][nt][i]);
        }
  }
}

// Many rows.  RW waves of 16 NT rows each share the keys of a step, and 4 / RW
// groups of them take their own tile of 32 keys of it.
//
// A step's second product is done in the next step, so that its matrix
// instructions run while that step's softmax does (they are issued in turn),
// and its values are converted into LDS a step later than its keys: step i
// converts keys i + 1 and values i, reads keys i and values i - 1, and asks
// for keys i + 2 and values i + 1.  One barrier a step, two halves of LDS.
//
// In LDS a lane's operand is 16 bytes at its number: keys [tile][s][lane],
// values [channel tile][lane], where row r of channel tile c is channel
// 64 (c / 4) + 4 r + c % 4 (a thread converts four channels of four keys, and
// writes half an operand of each).
//
// 8 trees of 64 nodes over 1024 to 4096 cached tokens, 8 E4M3 key heads of 128
// and 32 query heads (56 MB, 24 GFLOP): 75 us, 0.31 PFLOP/s (65 with
// probabilities in one part, two tiles a step).  No unit is full: a third of the
// CUs' cycles go to the start, the end and splits of different lengths, and of
// the rest the vector instructions take a half, the matrix instructions three
// tenths and LDS a fifth, with two waves a SIMD to fill each other's waits.  2 of
// 13 nodes over 8192 to 32768 in float16 (218 MB): 49 us, 4.5 TB/s.
template <int D>
constexpr int wide_nt() { return D <= 128 ? 2 : 1; }

template <int D, int FMT, int RW>
__global__ void __launch_bounds__(WAVES * 64, 2) k_tree_wide(Args a) {
  constexpr bool BYTE = FMT == CACHE_E4M3 || FMT == CACHE_INT8;
  constexpr int ESZ = BYTE ? 1 : 2;
  constexpr int NT = wide_nt<D>();
  constexpr int TILES = WAVES / RW, KEYS = STEP * TILES;
  constexpr int KS = D / 32, CT = D / 16;
  constexpr int KB = D / 8 * ESZ / 4;  // dwords of a thread's share of 32 keys: D / 8 channels of one
  constexpr int QUADS = D / 4, VP = QUADS > 32 ? QUADS / 32 : 1;  // passes of a thread over 32 keys' values
  constexpr int SLOTS = 32 * D / 8;                               // operands of 32 keys, keys or values
  struct Stage {
    uint4 k[TILES][SLOTS], v[TILES][SLOTS];
    f32x4 scale[BYTE ? TILES : 1][2][8];  // of keys, of values
  };
  static_assert(sizeof(Stage) * 2 >= (size_t)(TILES - 1) * RW * CT * NT * 64 * 16, "results reuse the stages");
  __shared__ Stage s_stage[2];
  __shared__ int s_nan;
  __shared__ float s_m[RW][16 * NT], s_l[RW][16 * NT];

  const Block blk = block_of(a);
  if (blk.unit >= a.units) return;
  const Span span = span_of(a, blk.unit);
  if (span.b < 0) return;
  const int b = span.b, h = blk.h;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int rw = wave % RW, tile = TILES > 1 ? wave / RW : 0;
  const int row0 = blk.row0 + rw * (16 * NT);
  const int ctx = __builtin_amdgcn_readfirstlane(a.context[b]);
  const int total = visible(a, ctx, blk.row0);
  if (!fits(a, ctx) && tid == 0) atomicOr(a.c.flag, VH_CACHE_ERR_CONTEXT);
  const int begin = (int)(span.split * span.chunk * PIECE);
  const int end = total - begin < (int)(span.chunk * PIECE) ? total : begin + (int)(span.chunk * PIECE);

  uint4 Q[NT][KS];
  float fac[NT];
  int node[NT];
  load_queries(a, b, h, row0, Q, node, [&](int s) { return 32 * s + 8 * g; });

  f32x4 acc[CT][NT];
  float m[NT], l[NT], top[NT];
  start(m, l, top, acc);
  Finder find(a, b, h, begin, end);

  // a thread's part in the conversion
  const int k_r = tid & 15, k_chan = (tid >> 4 & 7) * (D / 8);  // of 16-key tile wave / 2: neighbours write side by side
  const int quad = tid % QUADS, v_tg = tid / QUADS;             // of 16-key tile v_tg / 4, keys 4 (v_tg % 4) on
  uint32_t kr[TILES][KB];
  uint32_t vr[TILES][VP][4][ESZ];
  float sr = 0.0f;  // the first waves: a key's or a value's scale, one a lane
  struct Steps {
    Step s[TILES];
  };
  auto find_all = [&](int key0) __attribute__((always_inline)) {
    Steps x;
#pragma unroll
    for (int w = 0; w < TILES; ++w) x.s[w] = find(key0 + STEP * w);
    return x;
  };
  auto ask_k = [&](const Steps& x) __attribute__((always_inline)) {
    if constexpr (BYTE) {
      if (wave < TILES) {
        static_assert(TILES <= 2, "a choice of two");
        const int64_t row_0 = either(wave != 0, x.s[TILES - 1].row[0], x.s[0].row[0]);
        const int64_t row_1 = either(wave != 0, x.s[TILES - 1].row[1], x.s[0].row[1]);
        sr = (lane & 32 ? a.c.v_scale : a.c.k_scale)[either((lane & 16) != 0, row_1, row_0) + r];
      }
    }
#pragma unroll
    for (int w = 0; w < TILES; ++w) {
      const int64_t row = either(wave < 2, x.s[w].row[0], x.s[w].row[1]);
      const uint8_t* kp = (const uint8_t*)a.c.k + row * (D * ESZ) + (uint32_t)(k_r * (D * ESZ) + k_chan * ESZ);
      if constexpr (KB == 2) {
        const uint2 y = *(const uint2*)kp;
        kr[w][0] = y.x; kr[w][1] = y.y;
      } else {
#pragma unroll
        for (int j = 0; j < KB; j += 4) {
          const uint4 y = *(const uint4*)(kp + 4 * j);
          kr[w][j] = y.x; kr[w][j + 1] = y.y; kr[w][j + 2] = y.z; kr[w][j + 3] = y.w;
        }
      }
    }
  };
  auto ask_v = [&](const Steps& x) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < TILES; ++w)
#pragma unroll
      for (int u = 0; u < VP; ++u) {
        const int tg = VP > 1 ? v_tg + 4 * u : v_tg & 7;  // heads of 64: the upper threads read, and write nothing
        const int t = __builtin_amdgcn_readfirstlane(tg >> 2);
        const int64_t row = either(t != 0, x.s[w].row[1], x.s[w].row[0]);
        const uint8_t* vp = (const uint8_t*)a.c.v + row * (D * ESZ) + (uint32_t)(4 * (tg & 3) * (D * ESZ) + quad * 4 * ESZ);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (BYTE) {
            vr[w][u][i][0] = *(const uint32_t*)(vp + i * D);
          } else {
            const uint2 y = *(const uint2*)(vp + i * (D * 2));
            vr[w][u][i][0] = y.x; vr[w][u][i][1] = y.y;
          }
        }
      }
  };
  auto convert_k = [&](Stage& to) __attribute__((always_inline)) {
    if constexpr (BYTE) {
      if (wave < TILES) ((float*)to.scale[wave])[lane] = sr;
    }
#pragma unroll
    for (int w = 0; w < TILES; ++w)
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {  // eight channels each
        uint4 x;
        if constexpr (BYTE) {
          const uint2 lo = codes4<FMT>(kr[w][2 * j]), hi = codes4<FMT>(kr[w][2 * j + 1]);
          x = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          x = make_uint4(kr[w][4 * j], kr[w][4 * j + 1], kr[w][4 * j + 2], kr[w][4 * j + 3]);
        }
        const int c = k_chan + 8 * j;
        to.k[w][((wave >> 1) * KS + (c >> 5)) * 64 + ((c >> 3) & 3) * 16 + k_r] = x;
      }
  };
  // `masked`: values that are not finite are left out (add_nonfinite adds them)
  auto convert_v = [&](Stage& to, bool masked) __attribute__((always_inline)) {
    if constexpr (!BYTE) {
      if (masked) {
#pragma unroll
        for (int w = 0; w < TILES; ++w)
#pragma unroll
          for (int u = 0; u < VP; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int d = 0; d < ESZ; ++d) vr[w][u][i][d] &= ~nonfinite<FMT>(vr[w][u][i][d]);
      }
    }
#pragma unroll
    for (int w = 0; w < TILES; ++w)
#pragma unroll
      for (int u = 0; u < VP; ++u) {
        const int tg = v_tg + 4 * u;
        if (D == 64 && tg >= 8) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = BYTE ? 0 : e >> 1;
          const uint2 x = turn4<FMT>(vr[w][u][0][d], vr[w][u][1][d], vr[w][u][2][d], vr[w][u][3][d], BYTE ? e : e & 1);
          ((uint2*)&to.v[w][((quad >> 4) * 4 + e) * 64 + (tg & 3) * 16 + (quad & 15)])[tg >> 2] = x;
        }
      }
  };

  uint4 P[NT], Plo[NT];  // the last step's probabilities
  auto products = [&](const Stage& in, f32x4 (&S)[2][NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) S[t][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint4 A = in.k[tile][(t * KS + s) * 64 + lane];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[t][nt] = mfma<FMT>(A, Q[nt][s], S[t][nt]);
      }
    }
  };
  auto scales = [&](const Stage& in, f32x4 (&ks)[2], f32x4 (&vs)[2]) __attribute__((always_inline)) {
    if constexpr (BYTE) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ks[t] = in.scale[tile][0][4 * t + g];
        vs[t] = in.scale[tile][1][4 * t + g];
      }
    }
  };
  auto add = [&](const Stage& in) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const uint4 A = in.v[tile][c * 64 + lane];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        acc[c][nt] = mfma<FMT>(A, P[nt], acc[c][nt]);
        acc[c][nt] = mfma<FMT>(A, Plo[nt], acc[c][nt]);
      }
    }
  };

  // The keys; `quickly`: with quick steps, whose products leave no value out.  An
  // infinity among 16-bit ones may then have become NaN, and a workgroup whose
  // sums hold one takes its keys once more without (a test of the values as they
  // are converted would reach the other waves a step late).
  auto pass = [&](auto quickly) __attribute__((always_inline)) {
    constexpr bool QUICKLY = decltype(quickly)::value;
    const int whole = end < ctx ? end : ctx;
    // a step of the workgroup whose every key every row sees
    auto plain = [&](int key, const Steps& x) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < TILES; ++w) n += x.s[w].live[0] + x.s[w].live[1];
      return QUICKLY && key + KEYS <= whole && n == KEYS;
    };
    // after the last step it is asked for again, and not used
    auto after = [&](int key) { return key + KEYS < end ? key + KEYS : key; };
    int key0 = begin, half = 0;
    Steps now = find_all(key0), next = find_all(after(key0)), later = next;
    bool is_plain = plain(key0, now);
    ask_k(now);
    convert_queries<NT, KS, BYTE>(a, Q, fac);
    convert_k(s_stage[0]);
    ask_k(next);
    ask_v(now);
    __syncthreads();
    bool fed = false, pending = false;
    // the step's part in the pipeline
    auto feed = [&]() __attribute__((always_inline)) {
      convert_k(s_stage[half ^ 1]);
      convert_v(s_stage[half], !is_plain);
      later = find_all(after(after(key0)));
      ask_k(later);
      ask_v(next);
    };
    auto advance = [&]() __attribute__((always_inline)) {
      __syncthreads();
      half ^= 1;
      key0 += KEYS;
      now = next;
      next = later;
      is_plain = plain(key0, now);
    };
    do {
      if (!fed) feed();
      if (pending) add(s_stage[half ^ 1]);
      {
        const Stage& in = s_stage[half];
        f32x4 S[2][NT], ks[2], vs[2];
        uint32_t seen[NT];
        Step st;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          st.row[t] = either(tile != 0, now.s[TILES - 1].row[t], now.s[0].row[t]);
          st.live[t] = either(tile != 0, now.s[TILES - 1].live[t], now.s[0].live[t]);
        }
        products(in, S);
        scales(in, ks, vs);
        see<NT>(a, b, ctx, key0 + STEP * tile, st.live, node, seen);
        careful<FMT>(S, ks, vs, fac, seen, m, l, top, acc);
        operands<FMT, true>(S, vs, top, seen, l, P, Plo);
        if constexpr (!BYTE) {
          if (!is_plain) {
            uint32_t any = 0u;
            const uint16_t* v =
                (const uint16_t*)a.c.v + (either((lane & 32) != 0, st.row[1], st.row[0]) + r) * D + (lane >> 4 & 1) * (D / 2);
#pragma unroll 4
            for (int c = 0; c < D / 2; c += 8) {
              const uint4 x = *(const uint4*)(v + c);
              any |= nonfinite<FMT>(x.x) | nonfinite<FMT>(x.y) | nonfinite<FMT>(x.z) | nonfinite<FMT>(x.w);
            }
            if (__any(any != 0u))
              add_nonfinite<FMT>(a, st, S, seen, acc, [&](int c, int i) { return 64 * (c / 4) + 4 * (4 * g + i) + c % 4; });
          }
        }
      }
      fed = false;
      pending = true;
      advance();
      while (QUICKLY && key0 < end && is_plain) {
        feed();
        // The quick form of the softmax, written out so that nothing waits:
        // operands are read AHEAD of their products, and the last step's second
        // products are issued between this step's softmax, two scores at a time.
        // A step is given up as in the other kernel; a lane's sum stands for its terms.
        constexpr int AHEAD = 4, TN = 2;  // TN: 16-key tiles
        constexpr int KF = KS * TN, HALVES = TN * NT * 2;
        const Stage& in = s_stage[half];
        const Stage& old = s_stage[half ^ 1];
        f32x4 S[TN][NT];
        uint32_t w[TN][NT][2], u[TN][NT][2];
        f32x4 ks[2], vs[2], vn;  // vn: in the unit of a row
        float sum[NT], inv[NT], high = 0.0f, operand = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sum[nt] = 0.0f;
          inv[nt] = BYTE ? inverse_unit(top[nt]) : 1.0f;
#pragma unroll
          for (int t = 0; t < TN; ++t) S[t][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        auto key_at = [&](int n) __attribute__((always_inline)) {  // along D first: tiles' sums do not wait for each other
          const int t = n % TN, s = n / TN;
          return in.k[tile][(t * KS + s) * 64 + lane];
        };
        auto value_at = [&](int n) __attribute__((always_inline)) { return old.v[tile][n * 64 + lane]; };
        auto scale_at = [&](int t) __attribute__((always_inline)) {
          if constexpr (BYTE) {
            ks[t] = in.scale[tile][0][4 * t + g];
            vs[t] = in.scale[tile][1][4 * t + g];
          }
        };
        auto scores2 = [&](int n) __attribute__((always_inline)) {
          const int t = n / (2 * NT), nt = n / 2 % NT, i = n % 2 * 2;
          if (BYTE && n % (2 * NT) == 0) {
            high = fmaxf(fmaxf(high, vs[t][0]), vs[t][1]);
            high = fmaxf(fmaxf(high, vs[t][2]), vs[t][3]);
            if (t + 1 < TN) scale_at(t + 1);
          }
          if (BYTE && i == 0) vn = vs[t] * inv[nt];
          const float f0 = BYTE ? ks[t][i] * fac[nt] : fac[nt], f1 = BYTE ? ks[t][i + 1] * fac[nt] : fac[nt];
          float p0 = exp2_fast(fmaf(S[t][nt][i], f0, -m[nt])), p1 = exp2_fast(fmaf(S[t][nt][i + 1], f1, -m[nt]));
          sum[nt] += p0 + p1;
          if constexpr (BYTE) {
            p0 *= vn[i];
            p1 *= vn[i + 1];
            operand = fmaxf(fmaxf(operand, p0), p1);
          }
          w[t][nt][n % 2] = pack2<FMT>(p0, p1);
          const f32x2 hi = unpack2<FMT>(w[t][nt][n % 2]);
          u[t][nt][n % 2] = pack2<FMT>(p0 - hi[0], p1 - hi[1]);
          // here, between the products: the compiler would leave them for after the loop's exit
          asm volatile("" : "+v"(u[t][nt][n % 2]), "+v"(w[t][nt][n % 2]), "+v"(sum[nt]));
        };
        uint4 f[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) f[n] = key_at(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < KF; ++n) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) S[n % TN][nt] = mfma<FMT>(f[n % AHEAD], Q[nt][n / TN], S[n % TN][nt]);
          f[n % AHEAD] = n + AHEAD < KF ? key_at(n + AHEAD) : value_at(n + AHEAD - KF);
          if (n + AHEAD == KF) scale_at(0);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[c][nt] = mfma<FMT>(f[(KF + c) % AHEAD], P[nt], acc[c][nt]);
            acc[c][nt] = mfma<FMT>(f[(KF + c) % AHEAD], Plo[nt], acc[c][nt]);
          }
          if (c + AHEAD < CT) f[(KF + c) % AHEAD] = value_at(c + AHEAD);
#pragma unroll
          for (int x = c * HALVES / CT; x < (c + 1) * HALVES / CT; ++x) scores2(x);
          __builtin_amdgcn_sched_barrier(0);
        }
        bool far = BYTE && operand > operand_most<FMT>();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          far |= sum[nt] > (BYTE ? QUICK_MOST : operand_most<FMT>()) || m[nt] == -__builtin_inff();
          if constexpr (BYTE) far |= high * inv[nt] > QUICK_MOST;
        }
        pending = false;
        if (__any(far)) {
          fed = true;
          break;
        }
        pending = true;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          l[nt] += sum[nt];
          P[nt] = make_uint4(w[0][nt][0], w[0][nt][1], w[1][nt][0], w[1][nt][1]);
          Plo[nt] = make_uint4(u[0][nt][0], u[0][nt][1], u[1][nt][0], u[1][nt][1]);
        }
        advance();
      }
    } while (key0 < end);
    add(s_stage[half ^ 1]);
  };
  if (begin < end) {
    if (!BYTE && tid == 0) s_nan = 0;
    pass(std::true_type());
    if constexpr (!BYTE) {
      if (nan_among(acc, l)) s_nan = 1;
    }
    if constexpr (!BYTE || TILES > 1) __syncthreads();  // the stages are free
    if constexpr (!BYTE) {
      if (s_nan) {
        start(m, l, top, acc);
        pass(std::false_type());
        if constexpr (TILES > 1) __syncthreads();
      }
    }
  }
  if (find.bad && lane == 0) atomicOr(a.c.flag, VH_CACHE_ERR_PAGE);

  float M[NT], L[NT], unit[NT];  // unit: of the accumulators
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    L[nt] = sum_rows(l[nt]);
    M[nt] = m[nt];
    unit[nt] = bring(L[nt], M[nt]) * (BYTE ? unit_of(top[nt]) : 1.0f);
  }
  if constexpr (TILES > 1) {  // the second group of keys onto the first
    if (tile == 1 && g == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s_m[rw][16 * nt + r] = M[nt];
        s_l[rw][16 * nt + r] = L[nt];
      }
    }
    f32x4* s_o = (f32x4*)s_stage + rw * (CT * NT * 64);
    if (tile == 1) {
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s_o[(c * NT + nt) * 64 + lane] = acc[c][nt] * unit[nt];
    }
    __syncthreads();
    if (tile == 1) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float m1 = s_m[rw][16 * nt + r], to = fmaxf(M[nt], m1) + 1.0f;  // room for two
      const float f0 = M[nt] == -__builtin_inff() ? 1.0f : exp2_fast(M[nt] - to);
      const float f1 = m1 == -__builtin_inff() ? 1.0f : exp2_fast(m1 - to);
      M[nt] = to;
      L[nt] = L[nt] * f0 + s_l[rw][16 * nt + r] * f1;
      const float f = f0 * unit[nt];
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[c][nt] = acc[c][nt] * f + s_o[(c * NT + nt) * 64 + lane] * f1;
    }
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[c][nt] *= unit[nt];
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 16 * nt + r;
    if (row >= a.rows) continue;
    const bool none = pads(a, b, node[nt]);
    if (none) {
      M[nt] = -__builtin_inff();
      L[nt] = 0.0f;
    }
    const Place p = place(a, b, h, blk.unit, row, node[nt], M[nt], L[nt], g);
#pragma unroll
    for (int w = 0; w < CT / 4; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 64 * w + 16 * g + 4 * i, t = 4 * w;
        const f32x4 x = {acc[t][nt][i], acc[t + 1][nt][i], acc[t + 2][nt][i], acc[t + 3][nt][i]};
        put4(a, p.part ? p.part + at : nullptr, p.out + at, p.inv, none ? 0.0f : x[0], none ? 0.0f : x[1],
             none ? 0.0f : x[2], none ? 0.0f : x[3]);
      }
  }
}

// How a kernel of head size D is started: k_tree with NT tiles of rows a wave,
// or k_tree_wide with RW waves of rows.
template <int D>
int launch(const Args& a, bool wide, int n, hipStream_t s);

#define VH_TREE_FORMATS(KERNEL, N)                                                                    \
  switch (a.c.fmt) {                                                                                  \
    case CACHE_E4M3: hipLaunchKernelGGL((KERNEL<D, CACHE_E4M3, N>), grid, block, 0, s, a); break;     \
    case CACHE_INT8: hipLaunchKernelGGL((KERNEL<D, CACHE_INT8, N>), grid, block, 0, s, a); break;     \
    case CACHE_F16: hipLaunchKernelGGL((KERNEL<D, CACHE_F16, N>), grid, block, 0, s, a); break;       \
    default: hipLaunchKernelGGL((KERNEL<D, CACHE_BF16, N>), grid, block, 0, s, a); break;             \
  }

template <int D>
int launch_d(const Args& a, bool wide, int n, hipStream_t s) {
  const int64_t combos = (int64_t)a.units * a.c.kv_heads;
  const dim3 grid((unsigned)((combos + 7) / 8 * 8 * a.row_blocks)), block(WAVES * 64);
  if (wide) {
    if constexpr (D <= 128) {
      if (n == 2) {
        VH_TREE_FORMATS(k_tree_wide, 2)
      } else {
        VH_TREE_FORMATS(k_tree_wide, 4)
      }
    } else {
      VH_TREE_FORMATS(k_tree_wide, 4)
    }
  } else if constexpr (D <= 128) {
    if (n == 1) {
      VH_TREE_FORMATS(k_tree, 1)
    } else {
      VH_TREE_FORMATS(k_tree, 2)
    }
  } else {
    VH_TREE_FORMATS(k_tree, 1)
  }
  return vh::check_launch("vh_tree_attention");
}

}  // namespace tree
