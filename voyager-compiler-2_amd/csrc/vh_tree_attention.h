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
// scale its probability.
//
// The four waves of a workgroup take turns along the keys of a split and are
// joined through LDS; splits are joined by k_tree_merge.
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
  float* lse;                // or NULL
  float *part_o, *part_ml;   // splits > 1
  FastDiv group_div, page_div;  // page_div: by 16-key tiles a page
  float scale;               // times log2(e)
  int q_bf16, q_wide, words, batch, nodes, heads, group, rows, row_blocks, block_rows;
  int table_pages, chunk, splits;
};

// The keys that rows [row0, row0 + block_rows) of sequence b can see: up to
// their last node.  0 where the sequence does not fit its pages.
VH_DEV int visible(const Args& a, int ctx, int row0) {
  const int last = row0 + a.block_rows < a.rows ? row0 + a.block_rows : a.rows;
  if (ctx < 0 || (int64_t)ctx + a.nodes > (int64_t)a.table_pages * a.c.page) return 0;
  return ctx + (int)fast_div((uint32_t)(last - 1), a.group_div) + 1;
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

// The other side of a branch that scales the accumulators: no instructions,
// but a definition of its own, so that both sides keep them in place (without
// it the compiler copies all of them before each such branch).
template <int CT, int NT>
VH_DEV void stay(f32x4 (&acc)[CT][NT]) {
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) asm volatile("" : "+v"(acc[c][nt]));
}

// Waves of a SIMD that the registers are shared out for: two at least, so that
// accumulators stay where vector instructions reach them (under 256 registers
// a wave), three where a wave's 16 rows of 8-bit keys leave room.
constexpr int waves_of(int d, int fmt, int nt) {
  return nt > 1 || d > 128 ? 2 : fmt == CACHE_E4M3 || fmt == CACHE_INT8 || d == 64 ? 3 : 2;
}

template <int D, int FMT, int NT, bool SPLIT>
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

  // Row blocks that share keys are 8 workgroups apart: on one XCD, and L2.
  const int pairs = a.batch * a.c.kv_heads;
  const int combo = (blockIdx.x / (8 * a.row_blocks)) * 8 + blockIdx.x % 8;
  const int row0 = (int)(blockIdx.x / 8 % a.row_blocks) * (16 * NT);
  if (combo >= a.splits * pairs) return;
  const int split = combo / pairs, pair = combo % pairs;
  const int b = pair / a.c.kv_heads, h = pair % a.c.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int ctx = __builtin_amdgcn_readfirstlane(a.context[b]);
  const int total = visible(a, ctx, row0);
  if (total == 0 && split == 0 && threadIdx.x == 0) atomicOr(a.c.flag, VH_CACHE_ERR_CONTEXT);
  const int begin = split * a.chunk;
  if (begin >= total && a.splits > 1) return;
  const int end = begin + a.chunk < total ? begin + a.chunk : total;
  // read through the scalar cache: its waits are apart from those for keys and values
  const auto* table = (const __attribute__((address_space(4))) int32_t*)(a.table + (int64_t)b * a.table_st);

  // the queries, as the B operand: column r is a row, k the lane's share of D
  uint4 Q[NT][KS];
  float fac[NT];  // of a row's products, in powers of two
  int node[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 16 * nt + r;
    const bool in = row < a.rows;
    const int at = in ? row : a.rows - 1;
    node[nt] = (int)fast_div((uint32_t)at, a.group_div);
    const int head = h * a.group + at - node[nt] * a.group;
    const uint16_t* q = (const uint16_t*)a.q + b * a.q_sb + node[nt] * a.q_st + head * a.q_sh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = BYTE ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
      if (a.q_wide) {
        Q[nt][s] = *(const uint4*)(q + c);
      } else {
        Q[nt][s] = make_uint4(q[c] | (uint32_t)q[c + 1] << 16, q[c + 2] | (uint32_t)q[c + 3] << 16,
                              q[c + 4] | (uint32_t)q[c + 5] << 16, q[c + 6] | (uint32_t)q[c + 7] << 16);
      }
    }
    fac[nt] = a.scale;
    if (BYTE && a.q_bf16) {
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

  f32x4 acc[CT][NT];
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -__builtin_inff();
    l[nt] = 0.0f;
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float T = 0x1p-126f;  // the accumulators' unit: a power of two over the value scales so far
  bool bad_page = false;

  uint4 kr[2][KQ];
  uint32_t vr[2][4][VB][VW];
  f32x4 ks[2], vs[2];
  // A lane's part of a tile's rows: keys at r, channels from 16 g bytes on;
  // values at 4 g + i, channels from r CPL on.
  const uint32_t k_lane = (uint32_t)r * (D * ESZ) + g * 16, v_lane = (uint32_t)(4 * g) * (D * ESZ) + r * (CPL * ESZ);

  // Where a step's two tiles lie, and how many of their keys exist.
  struct Step {
    int64_t row[2];
    int live[2];
  };
  const int64_t page_rows = (int64_t)a.c.kv_heads * a.c.page, head_rows = (int64_t)h * a.c.page;
  const uint32_t pages = (uint32_t)a.c.pages;
  auto find = [&](int key0) __attribute__((always_inline)) {
    Step st;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int left = end - (key0 + 16 * t);
      const uint32_t tile = ((uint32_t)key0 >> 4) + (left > 0 ? t : 0);
      const uint32_t pg = fast_div(tile, a.page_div);
      const int id = table[pg];
      const bool there = (uint32_t)id < pages;  // if not, nothing of it is seen
      bad_page |= !there;
      st.live[t] = !there || left < 0 ? 0 : left < 16 ? left : 16;
      st.row[t] = (there ? id : 0) * page_rows + head_rows + (tile * 16 - pg * (uint32_t)a.c.page);
    }
    return st;
  };
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

  // One step of 32 keys; `st` is it, `next` the one whose keys and values are
  // asked for as soon as this step's registers are free.
  auto step = [&](auto is_masked, int key0, const Step& st, const Step& next) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(is_masked)::value;
    // scores: S[t][nt][i] of key 16 t + 4 g + i and row 16 nt + r
    f32x4 S[2][NT];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) S[t][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 A;
        if constexpr (BYTE) {
          const uint4 x = kr[t][s >> 1];
          const uint32_t w0 = s & 1 ? x.z : x.x, w1 = s & 1 ? x.w : x.y;
          if constexpr (FMT == CACHE_E4M3) {
            A = make_uint4(e4m3_pair(w0, false), e4m3_pair(w0, true), e4m3_pair(w1, false), e4m3_pair(w1, true));
          } else {
            A = make_uint4(int8_pair(__builtin_amdgcn_perm(0u, w0, 0x0c010c00u)),
                           int8_pair(__builtin_amdgcn_perm(0u, w0, 0x0c030c02u)),
                           int8_pair(__builtin_amdgcn_perm(0u, w1, 0x0c010c00u)),
                           int8_pair(__builtin_amdgcn_perm(0u, w1, 0x0c030c02u)));
          }
        } else {
          A = kr[t][s];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[t][nt] = mfma<FMT>(A, Q[nt][s], S[t][nt]);
      }
      if constexpr (BYTE) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[t][nt] *= ks[t];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(next);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t seen[NT];  // the lane's keys (bit 4 t + i) that its row sees
    if constexpr (MASKED) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        seen[nt] = 0u;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 4 * g + i, n = key0 + 16 * t + at - ctx;  // n: the key's node, if it is one
            bool ok = at < st.live[t];
            if (ok && n >= 0) {
              if (a.masks) ok = n < a.nodes && (a.masks[((int64_t)b * a.nodes + node[nt]) * a.words + (n >> 6)] >> (n & 63) & 1);
              else ok = n <= node[nt];
            }
            seen[nt] |= ok ? 1u << (4 * t + i) : 0u;
            S[t][nt][i] = ok ? S[t][nt][i] : -__builtin_inff();
          }
      }
    }

    // the running maximum; it moves only when a score is 2^8 over it, so that
    // the accumulators are seldom scaled (probabilities then reach 2^8)
    float mx[NT];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float v = fmaxf(S[0][nt][0], S[0][nt][1]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = t ? 0 : 2; i < 4; i += 2) v = fmaxf(fmaxf(v, S[t][nt][i]), S[t][nt][i + 1]);
      mx[nt] = max_rows(v) * fac[nt];
      grow |= mx[nt] > m[nt] + 8.0f;
    }
    if (__any(grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float to = fmaxf(m[nt], mx[nt]);
        const float alpha = m[nt] == -__builtin_inff() ? 0.0f : exp2_fast(m[nt] - to);
        m[nt] = to;
        l[nt] *= alpha;
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c][nt] *= alpha;
      }
    } else {
      stay(acc);
    }
    f32x4 vn[2];
    if constexpr (BYTE) {
      float top = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) top = fmaxf(fmaxf(top, vs[t][i]), vs[t][i + 1]);
      top = fminf(max_rows(top), 0x1p125f);  // the next power of two stays finite
      top = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(top)));
      if (top > T) {
        const float to = __uint_as_float((__float_as_uint(top) & 0x7f800000u) + 0x00800000u);
        const float down = T * __uint_as_float(0x7f000000u - __float_as_uint(to));  // T / to, both powers of two
        T = to;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < CT; ++c) acc[c][nt] *= down;
      } else {
        stay(acc);
      }
      const float inv = __uint_as_float(0x7f000000u - __float_as_uint(T));  // 1 / T
#pragma unroll
      for (int t = 0; t < 2; ++t) vn[t] = vs[t] * inv;
    }

    // probabilities: the B operand of the second product, k = 4 t + i
    uint4 P[NT], Plo[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float ref = m[nt] == -__builtin_inff() ? 0.0f : m[nt];
      uint32_t w[4], u[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float p0 = exp2_fast(fmaf(S[t][nt][i], fac[nt], -ref)), p1 = exp2_fast(fmaf(S[t][nt][i + 1], fac[nt], -ref));
          l[nt] += p0 + p1;
          if constexpr (BYTE) {
            p0 *= vn[t][i];
            p1 *= vn[t][i + 1];
            if constexpr (MASKED) {  // a scale there may be anything
              p0 = seen[nt] >> (4 * t + i) & 1 ? p0 : 0.0f;
              p1 = seen[nt] >> (4 * t + i + 1) & 1 ? p1 : 0.0f;
            }
          }
          w[2 * t + i / 2] = pack2<FMT>(p0, p1);
          if constexpr (SPLIT) {
            const f32x2 hi = unpack2<FMT>(w[2 * t + i / 2]);
            u[2 * t + i / 2] = pack2<FMT>(p0 - hi[0], p1 - hi[1]);
          }
          if constexpr (!BYTE && MASKED) {
            S[t][nt][i] = p0;
            S[t][nt][i + 1] = p1;
          }
        }
      P[nt] = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (SPLIT) Plo[nt] = make_uint4(u[0], u[1], u[2], u[3]);
    }

    // Values that are not finite would reach rows that do not see them as 0 *
    // inf: in steps with a mask they are taken out and added to the rows that do.
    if constexpr (!BYTE && MASKED) {
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
      if (__any(any != 0u)) {
        for (int k = 0; k < STEP; ++k) {
          const int t = k >> 4, at = k & 15;
          const uint16_t* v = (const uint16_t*)a.c.v + ((t ? st.row[1] : st.row[0]) + at) * D;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float mine = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((at & 3) == i) mine = t ? S[1][nt][i] : S[0][nt][i];
            const int from = (at >> 2) * 16 + r;
            const float p = __shfl(mine, from);
            const bool ok = (uint32_t)__shfl((int)seen[nt], from) >> (4 * t + (at & 3)) & 1;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t x = v[(c / CPL) * 16 * CPL + (4 * g + i) * CPL + c % CPL];
                if (ok && nonfinite<FMT>(x) & 0xffffu) acc[c][nt][i] += p * unpack2<FMT>(x)[0];
              }
          }
        }
      }
    }

    // O^T += V^T P^T: A's row r of channel tile c is channel (c / CPL) 16 CPL + r CPL + c % CPL
#pragma unroll
    for (int w = 0; w < VB; ++w)
#pragma unroll
      for (int d = 0; d < VW; ++d)
#pragma unroll
        for (int e = 0; e < 4 / ESZ; ++e) {
          uint4 A;
          if constexpr (FMT == CACHE_E4M3) {
            // four keys' bytes of a channel side by side, as the converter takes them
            uint32_t x[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t s2 = e < 2 ? 0x05010400u : 0x07030602u;
              const uint32_t lo = __builtin_amdgcn_perm(vr[t][1][w][d], vr[t][0][w][d], s2);
              const uint32_t hi = __builtin_amdgcn_perm(vr[t][3][w][d], vr[t][2][w][d], s2);
              x[t] = __builtin_amdgcn_perm(hi, lo, e & 1 ? 0x07060302u : 0x05040100u);
            }
            A = make_uint4(e4m3_pair(x[0], false), e4m3_pair(x[0], true), e4m3_pair(x[1], false), e4m3_pair(x[1], true));
          } else if constexpr (FMT == CACHE_INT8) {
            const uint32_t sel = 0x0c040c00u + e * 0x00010001u;  // byte e of two keys
            A = make_uint4(int8_pair(__builtin_amdgcn_perm(vr[0][1][w][d], vr[0][0][w][d], sel)),
                           int8_pair(__builtin_amdgcn_perm(vr[0][3][w][d], vr[0][2][w][d], sel)),
                           int8_pair(__builtin_amdgcn_perm(vr[1][1][w][d], vr[1][0][w][d], sel)),
                           int8_pair(__builtin_amdgcn_perm(vr[1][3][w][d], vr[1][2][w][d], sel)));
          } else {
            const uint32_t sel = e ? 0x07060302u : 0x05040100u;
            A = make_uint4(__builtin_amdgcn_perm(vr[0][1][w][d], vr[0][0][w][d], sel),
                           __builtin_amdgcn_perm(vr[0][3][w][d], vr[0][2][w][d], sel),
                           __builtin_amdgcn_perm(vr[1][1][w][d], vr[1][0][w][d], sel),
                           __builtin_amdgcn_perm(vr[1][3][w][d], vr[1][2][w][d], sel));
          }
          const int c = w * CPL + (4 / ESZ) * d + e;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[c][nt] = mfma<FMT>(A, P[nt], acc[c][nt]);
            if constexpr (SPLIT) acc[c][nt] = mfma<FMT>(A, Plo[nt], acc[c][nt]);
          }
        }
    __builtin_amdgcn_sched_barrier(0);
    load_v(next);
  };

  int key0 = begin + wave * STEP;
  if (key0 < end) {
    Step st = find(key0);
    load_k(st);
    load_v(st);
    // Steps that every row sees, then the rest: two loops, so that neither's
    // loads are moved ahead of the other's use of the registers.  After the
    // last step it is asked for again, and not waited for.
    const int whole = end < ctx ? end : ctx;
    auto turn = [&](auto is_masked) __attribute__((always_inline)) {
      const Step next = find(key0 + WAVES * STEP < end ? key0 + WAVES * STEP : key0);
      step(is_masked, key0, st, next);
      st = next;
      key0 += WAVES * STEP;
    };
    auto plain = [&]() { return key0 + STEP <= whole && st.live[0] + st.live[1] == STEP; };
    if (plain()) {
      do turn(std::false_type());
      while (plain());
    }
    if (key0 < end) {
      do turn(std::true_type());
      while (key0 < end);
    }
  }
  if (bad_page && lane == 0) atomicOr(a.c.flag, VH_CACHE_ERR_PAGE);

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
    const float f = (m[nt] == -__builtin_inff() ? 1.0f : exp2_fast(m[nt] - M[nt])) * (BYTE ? T : 1.0f);
    // a node without itself among its ancestors pads its tree, and sees no context either
    const bool pads = a.masks && !(a.masks[((int64_t)b * a.nodes + node[nt]) * a.words + (node[nt] >> 6)] >> (node[nt] & 63) & 1);
    if (pads) {
      M[nt] = -__builtin_inff();
      L[nt] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c][nt] = pads ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[c][nt] * f;
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
    if (a.splits > 1) {
      const int64_t at = ((int64_t)pair * a.splits + split) * a.rows + row;
      if (g == 0) *(float2*)(a.part_ml + 2 * at) = make_float2(M[nt], L[nt]);
#pragma unroll
      for (int w = 0; w < VB; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* o = a.part_o + at * D + w * 16 * CPL + (4 * g + i) * CPL;
#pragma unroll
          for (int c = 0; c < CPL; c += 4)
            *(f32x4*)(o + c) = f32x4{acc[w * CPL + c][nt][i], acc[w * CPL + c + 1][nt][i], acc[w * CPL + c + 2][nt][i],
                                     acc[w * CPL + c + 3][nt][i]};
        }
    } else {
      // a row that sees nothing is zero
      const float inv = L[nt] == 0.0f ? 0.0f : 1.0f / L[nt];
      const int64_t at = ((int64_t)b * a.nodes + node[nt]) * a.heads + h * a.group + row - node[nt] * a.group;
      if (a.lse && g == 0) a.lse[at] = L[nt] == 0.0f ? -__builtin_inff() : (M[nt] + log2f(L[nt])) * LN2;
#pragma unroll
      for (int w = 0; w < VB; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint16_t* o = (uint16_t*)a.o + at * D + w * 16 * CPL + (4 * g + i) * CPL;
#pragma unroll
          for (int c = 0; c < CPL; c += 4) {
            const float x0 = acc[w * CPL + c][nt][i] * inv, x1 = acc[w * CPL + c + 1][nt][i] * inv;
            const float x2 = acc[w * CPL + c + 2][nt][i] * inv, x3 = acc[w * CPL + c + 3][nt][i] * inv;
            *(uint2*)(o + c) = a.q_bf16 ? make_uint2(pack2<CACHE_BF16>(x0, x1), pack2<CACHE_BF16>(x2, x3))
                                        : make_uint2(pack2<CACHE_F16>(x0, x1), pack2<CACHE_F16>(x2, x3));
          }
        }
    }
  }
}

// How a kernel of head size D is started.
template <int D>
int launch(const Args& a, int nt, hipStream_t s);

template <int D, int NT>
void launch_nt(const Args& a, dim3 grid, hipStream_t s) {
  // float16 results are four times finer than float16 probabilities allow once
  // (an error of its own size would join the result's rounding), and bfloat16
  // values need bfloat16 probabilities: both take them in two parts.
  const dim3 block(WAVES * 64);
  switch (a.c.fmt) {
    case CACHE_E4M3:
      if (a.q_bf16) hipLaunchKernelGGL((k_tree<D, CACHE_E4M3, NT, false>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((k_tree<D, CACHE_E4M3, NT, true>), grid, block, 0, s, a);
      break;
    case CACHE_INT8:
      if (a.q_bf16) hipLaunchKernelGGL((k_tree<D, CACHE_INT8, NT, false>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((k_tree<D, CACHE_INT8, NT, true>), grid, block, 0, s, a);
      break;
    case CACHE_F16: hipLaunchKernelGGL((k_tree<D, CACHE_F16, NT, true>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((k_tree<D, CACHE_BF16, NT, true>), grid, block, 0, s, a); break;
  }
}

template <int D>
int launch_d(const Args& a, int nt, hipStream_t s) {
  const int64_t combos = (int64_t)a.splits * a.batch * a.c.kv_heads;
  const dim3 grid((unsigned)((combos + 7) / 8 * 8 * a.row_blocks));
  if (nt == 1) launch_nt<D, 1>(a, grid, s);
  else if constexpr (D <= 128) launch_nt<D, 2>(a, grid, s);
  return vh::check_launch("vh_tree_attention");
}

}  // namespace tree
