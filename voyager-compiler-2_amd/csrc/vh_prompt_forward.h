// The forward pass of packed causal attention: vh_prompt.h says how.
//
// Bound by vector instructions (an exponential, a scaling, a sum and half a
// conversion a score) beside the products, at two waves a SIMD: a prompt of 4096,
// 32 + 8 heads of 128 in bfloat16, 150-165 us, 830-915 TFLOP/s (a large library
// product reaches 1200); of 8192 550-635 us.  No bank conflicts in LDS.
#pragma once

#include "vh_prompt.h"

namespace prompt {

constexpr int KEYS = 64;  // of a tile
// Keys that a wave takes at a time: 64 where the registers hold their scores
// beside four waves of a SIMD, or fewer waves share one (a prompt of 4096, 32 + 8
// heads of 128: 173 us by 32, 165 by 64; 64 prompts, 16 heads of 64: 21 and 23).
constexpr int sub_of(int d) { return d == 64 ? 32 : 64; }

// A weight's exponent is its score less a reference that lies under the row's
// largest score by at most `SLACK`, so that sums are rarely scaled, and moved
// by `LIFT`: float16 weights then reach down to 2^-35 of the largest, and
// bfloat16 ones, whose range is float32's, stay so small that neither their sum
// nor a product with the largest values overflows over 2^24 keys (and products
// with values under 2^-94 may underflow).
template <bool BF>
struct Range {
  static constexpr float SLACK = BF ? 8.0f : 4.0f, LIFT = BF ? -32.0f : 11.0f;
};

// Adds to 32 channels of a wave's rows what infinite and NaN values of 16 keys
// give: weights of the keys that hold one in a channel, by products with ones.
template <bool BF>
VH_DEV void add_nonfinite(uint4 v, uint4 weights, f32x16& acc) {
  constexpr uint32_t ONE = BF ? 0x3f80u : 0x3c00u, INFINITE = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int kind = 0; kind < 3; ++kind) {
    const auto ones = [&](uint32_t w) {
      uint32_t out = 0u;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x = (w >> (16 * half)) & 0xffffu;
        const bool is = kind == 0 ? x == INFINITE : kind == 1 ? x == (INFINITE | 0x8000u) : (x & 0x7fffu) > INFINITE;
        out |= (is ? ONE : 0u) << (16 * half);
      }
      return out;
    };
    f32x16 some = {};
    some = mfma<BF>(make_uint4(ones(v.x), ones(v.y), ones(v.z), ones(v.w)), weights, some);
    const float what = kind == 0 ? __builtin_inff() : kind == 1 ? -__builtin_inff() : __builtin_nanf("");
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += some[r] > 0.0f ? what : 0.0f;
  }
}

template <int D, bool BF, bool CAREFUL>
struct Forward {
  static constexpr int SUB = sub_of(D);
  f32x16 acc[D / 32];
  // a row's reference, and of its sum, and of its sum of rounded weights, the half that is this lane's
  float ref, sum, rounded;

  // SUB keys from key0 on, row `at` of the tile.  masked: some are not seen by some rows.
  __device__ __forceinline__ void step(const uint4 (&q)[D / 16], const char* k, const char* v, int at, int key0, int row, int first, bool masked, float scale) {
    const int half = (threadIdx.x & 63) >> 5;
    f32x16 s[SUB / 32];
#pragma unroll
    for (int t = 0; t < SUB / 32; ++t) {
      s[t] = f32x16{};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s[t] = mfma<BF>(rows_operand<D>(k, at + 32 * t, i), q[i], s[t]);
    }
    if (masked) {
#pragma unroll
      for (int t = 0; t < SUB / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = key0 + 32 * t + result_row(r) + 4 * half;
          s[t][r] = key >= first && key <= row ? s[t][r] : -__builtin_inff();
        }
    }
    float most = s[0][0];
#pragma unroll
    for (int t = 0; t < SUB / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, s[t][r]);
    most = max_halves(most) * scale;
    const bool over = most > ref + Range<BF>::SLACK;
    if (__any(over)) {
      const float to = over ? most : ref, by = ref == -__builtin_inff() ? 1.0f : exp2_fast(ref - to);
      ref = to;
      sum *= by;
      rounded *= by;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] *= by;
    }
    const float less = (ref == -__builtin_inff() ? 0.0f : ref) - Range<BF>::LIFT;
    uint4 p[SUB / 16];
    float part[SUB / 32][4];
#pragma unroll
    for (int t = 0; t < SUB / 32; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = exp2_fast(__builtin_fmaf(s[t][r], scale, -less));
        if (r < 4) part[t][r] = s[t][r];
        else part[t][r & 3] += s[t][r];  // four sums, so that one addition does not wait for the one before
      }
      sum += (part[t][0] + part[t][1]) + (part[t][2] + part[t][3]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        p[2 * t + i] = make_uint4(pack2<BF>(s[t][8 * i], s[t][8 * i + 1]), pack2<BF>(s[t][8 * i + 2], s[t][8 * i + 3]),
                                  pack2<BF>(s[t][8 * i + 4], s[t][8 * i + 5]), pack2<BF>(s[t][8 * i + 6], s[t][8 * i + 7]));
    }
#pragma unroll
    for (int i = 0; i < SUB / 16; ++i) rounded = add_pairs<BF>(p[i].x, add_pairs<BF>(p[i].y, add_pairs<BF>(p[i].z, add_pairs<BF>(p[i].w, rounded))));
#pragma unroll
    for (int i = 0; i < SUB / 16; ++i)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 x = turned_operand<D>(v, at + 16 * i, c);
        if constexpr (CAREFUL) {
          // what all rows see is as it is
          acc[c] = mfma<BF>(masked ? finite_part<BF>(x) : x, p[i], acc[c]);
          if (masked) add_nonfinite<BF>(x, p[i], acc[c]);
        } else {
          acc[c] = mfma<BF>(x, p[i], acc[c]);
        }
      }
  }
};

// A workgroup's rows of one head.  True where a row may have got an infinity
// or NaN that it does not see.
template <int D, bool BF, int HALVES, bool CAREFUL>
VH_DEV bool prompt_block(const Args& a, char* lds) {
  constexpr int BYTES = KEYS * D * 2;  // of a tile: two of keys, two of values
  const int turn = Halves<D, HALVES>::half();
  char* tiles = lds + turn * 4 * BYTES;
  const int rank = blockIdx.x / a.heads, spread = blockIdx.x - rank * a.heads;
  // heads of a group lie `kv_heads` workgroups apart: on one die where those are a multiple of 8
  const int kv = spread % a.kv_heads, head = kv * a.group + spread / a.kv_heads;
  const int row0 = a.order[rank] * BLOCK, wave = __builtin_amdgcn_readfirstlane(threadIdx.x % THREADS / 64), lane = threadIdx.x & 63;
  const int wave0 = row0 + 32 * wave, row = wave0 + (lane & 31);
  const bool in = row < a.tokens;
  const int first = in ? a.first[row] : row + 1;
  const int wave_first = __builtin_amdgcn_readlane(first, 0), wave_last_first = __builtin_amdgcn_readlane(first, 31);
  const int begin = a.first[row0], end = min(row0 + BLOCK, a.tokens);
  uint4 q[D / 16];
  load_columns<D>(a.q, head, wave0, a.tokens, q);
  Loader<D, KEYS> kl, vl;
  kl.init(a.k, kv);
  vl.init(a.v, kv);
  const float scale = a.scale * LOG2E;
  Forward<D, BF, CAREFUL> f;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) f.acc[c] = f32x16{};
  f.ref = -__builtin_inff();
  f.sum = f.rounded = 0.0f;
  const int first_key = begin + turn * KEYS;
  if (first_key < end) {
    kl.load(tiles, first_key, a.tokens);
    vl.load(tiles + 2 * BYTES, first_key, a.tokens);
  }
  int at = 0;
  for (int key0 = first_key; key0 - turn * KEYS < end; key0 += HALVES * KEYS, at ^= 1) {
    arrived();
    if (key0 + HALVES * KEYS < end) {
      kl.load(tiles + (at ^ 1) * BYTES, key0 + HALVES * KEYS, a.tokens);
      vl.load(tiles + (2 + (at ^ 1)) * BYTES, key0 + HALVES * KEYS, a.tokens);
    }
    if (HALVES > 1 && key0 >= end) continue;
    const char *k = tiles + at * BYTES, *v = tiles + (2 + at) * BYTES;
#pragma unroll
    for (int sub = 0; sub < KEYS; sub += sub_of(D)) {
      constexpr int SUB = sub_of(D);
      const int key = key0 + sub;
      if (key >= wave0 + 32 || key + SUB <= wave_first) continue;
      f.step(q, k, v, sub, key, row, first, key + SUB > wave0 + 1 || key < wave_last_first, scale);
    }
  }
  if constexpr (HALVES > 1) {
    constexpr int N = D / 2 + 3;
    __syncthreads();
    float* to = lane_slot(lds, N);
    if (turn > 0) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(16 * c + r) * 64] = f.acc[c][r];
      to[(N - 3) * 64] = f.ref;
      to[(N - 2) * 64] = f.sum;
      to[(N - 1) * 64] = f.rounded;
    }
    __syncthreads();
    if (turn > 0) return false;
    const float other = to[(N - 3) * 64], most = fmaxf(f.ref, other);
    const float mine = f.ref == -__builtin_inff() ? 1.0f : exp2_fast(f.ref - most);  // of nothing: 0 times 1
    const float by = other == -__builtin_inff() ? 1.0f : exp2_fast(other - most);
    f.ref = most;
    f.sum = f.sum * mine + to[(N - 2) * 64] * by;
    f.rounded = f.rounded * mine + to[(N - 1) * 64] * by;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) f.acc[c][r] = f.acc[c][r] * mine + to[(16 * c + r) * 64] * by;
  }
  f.sum = sum_halves(f.sum);
  f.rounded = sum_halves(f.rounded);
  // Divided by the sum of the rounded weights, a row whose weight is one key's has
  // none of its rounding, in its result as in the gradients' D.
  const float by = f.rounded == 0.0f ? 0.0f : 1.0f / f.rounded;
  // back, long sequences' rows read what is left out of theirs
  void* low = a.o_low && !covers(a, short_run(a, row0), row0) ? a.o_low : nullptr;
  store_columns<D, D, BF>(a.o, low, a.heads, head, row, in, 0, f.acc, by);
  if (in && lane < 32) {
    const bool none = f.sum == 0.0f;
    const float less = f.ref - Range<BF>::LIFT, log2_sum = log2f(f.sum), lse = none ? -__builtin_inff() : (less + log2_sum) * LN2;
    a.lse[(int64_t)row * a.heads + head] = lse;
    if (a.rest) a.rest[(int64_t)head * a.tokens + row] = weights_lift(BF) - (none ? 0.0f : (less - log2_units(lse)) + log2_sum);
  }
  // a row whose sum is not finite sees something that is not
  return !CAREFUL && in && f.sum < __builtin_inff() && any_nonfinite(f.acc);
}

// A masked key's weight is 0, but 0 times an infinity or NaN is not: a block
// into whose rows such a value may have come is done once more, with these
// values apart.
template <int D, bool BF, int HALVES>
__global__ void __launch_bounds__(HALVES* THREADS, waves_of(D)) k_prompt(Args a) {
  __shared__ __attribute__((aligned(16))) char s_tiles[HALVES * 4 * KEYS * D * 2];
  const bool apart = prompt_block<D, BF, HALVES, false>(a, s_tiles);
  if (__syncthreads_or(apart)) prompt_block<D, BF, HALVES, true>(a, s_tiles);
}

template <int D, bool BF>
void forward_of(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.tokens + BLOCK - 1) / BLOCK * a.heads));
  if constexpr (D <= 128) {
    if (in_halves(a, waves_of(D))) {
      hipLaunchKernelGGL((k_prompt<D, BF, 2>), grid, dim3(2 * THREADS), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((k_prompt<D, BF, 1>), grid, dim3(THREADS), 0, s, a);
}

template <int D>
int forward(const Args& a, bool bf16, hipStream_t s) {
  if (bf16) forward_of<D, true>(a, s);
  else forward_of<D, false>(a, s);
  return vh::check_launch("vh_prompt_attention");
}

}  // namespace prompt
