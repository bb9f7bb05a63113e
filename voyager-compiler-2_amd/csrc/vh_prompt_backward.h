// The backward pass of packed causal attention: vh_prompt.h says how.
//
// A pass over blocks of rows, which finds D_i and gives dq, and one over blocks
// of keys for dk and dv.  Scores and dP are formed in both: five products become
// seven, but every sum has one owner and one order, and nothing is added up in
// memory.
//
// 8192 rows, 32 + 8 heads of 128 in bfloat16, one sequence: dq 735-755 us, dk and dv
// 1170-1240 us (1110 and 910 TFLOP/s of the products made); six documents of 8192 rows
// 280-290, 420-455 and 12 us of joining.  Both are bound by the matrix units and the
// vector instructions between their products, at two waves a SIMD.
#pragma once

#include "vh_prompt.h"

namespace prompt {

constexpr int DK_ROWS = 32;                      // of a tile of the keys' pass
constexpr int STATS = 512;                       // bytes of its rows' numbers
// Tiles of an item at least, but for a block's last: its sums are written and
// read, 128 KB a head of 128.
constexpr int LEAST = 2 * BLOCK / DK_ROWS;

VH_DEV int sum_before(int x, int* s_sum, int& all) {  // over the first THREADS
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int upto = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    upto += lane >= d ? y : 0;
  }
  __syncthreads();
  if (lane == 63 && wave < WAVES) s_sum[wave] = upto;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? s_sum[w] : 0;
    all += s_sum[w];
  }
  return before + upto - x;
}
constexpr int ITEM_BYTES = MOST_CUT * 6 + 16;  // of LDS
// The items of the keys' pass.  A block's work is the tiles of rows that see
// it; an item is `size` tiles, the most that a workgroup has to take for the card
// to be done in one go, or what a block has left.  The largest come first, of
// equal ones the first: an item's place is the number of those before it.
// `groups` workgroups share the blocks.  (us of the keys' pass by whole blocks, and
// by items and of joining them: six documents of 8192 rows, 32 + 8 heads of 128,
// 1255, 396 + 11; three of 5001, 16 + 4 heads of 64, 733, 120 + 10.)
VH_DEV void prompt_items(const Args& a, int group, int groups, char* lds) {
  const int thread = threadIdx.x < THREADS ? threadIdx.x : MOST_CUT;  // a second half has no block
  int *s_sum = (int*)lds, *s_tiles = s_sum + WAVES;
  uint16_t* s_pieces = (uint16_t*)(s_tiles + MOST_CUT);
  const int blocks = (a.tokens + BLOCK - 1) / BLOCK;
  int sum = 0, all;
  for (int b = thread; b < blocks; b += THREADS) {
    const int key0 = b * BLOCK;
    s_tiles[b] = (max(a.past[min(key0 + BLOCK, a.tokens) - 1] - key0, 0) + DK_ROWS - 1) / DK_ROWS;
    sum += s_tiles[b];
  }
  sum_before(sum, s_sum, all);
  const int size = max((all + a.share - 1) / a.share, LEAST);
  for (int b = thread; b < blocks; b += THREADS) s_pieces[b] = (uint16_t)max((s_tiles[b] + size - 1) / size, 1);
  __syncthreads();
  // a thread has consecutive blocks: the slots before them
  const int each = (blocks + THREADS - 1) / THREADS, b0 = min(thread * each, blocks), b1 = min(b0 + each, blocks);
  int items = 0, slots = 0;
  for (int b = b0; b < b1; ++b) {
    items += s_pieces[b];
    slots += s_pieces[b] > 1 ? s_pieces[b] : 0;
  }
  sum_before(items, s_sum, all);
  int unused, slot = sum_before(slots, s_sum, unused);
  for (int b = b0; b < b1; ++b) {
    const int n = s_pieces[b], key0 = b * BLOCK, end = key0 + s_tiles[b] * DK_ROWS, first = slot;
    slot += n > 1 ? n : 0;
    if (b % groups != group) continue;
    a.joins[b] = make_int2(first, n);
    const int last = s_tiles[b] - (n - 1) * size;  // of its items, which is not a whole one
    int whole_at = 0, last_at = 0;
    for (int c = 0; c < blocks; ++c) {
      const int whole = s_pieces[c] - 1, rest = s_tiles[c] - whole * size;
      whole_at += c < b ? whole + (rest == size) : 0;
      last_at += (size > last || c < b ? whole : 0) + (rest > last || (c < b && rest == last) ? 1 : 0);
    }
    for (int i = 0; i < n; ++i) {
      const int row0 = key0 + i * size * DK_ROWS;
      // the last one comes after its block's others also where it is as long
      const int at = i < n - 1 ? whole_at + i : last_at + (last == size ? n - 1 : 0);
      a.items[at] = make_int4(b, row0, i < n - 1 ? row0 + size * DK_ROWS : end, n > 1 ? first + i : -1);
    }
  }
  if (group == 0)
    for (int i = all + (int)threadIdx.x; i < a.item_count; i += blockDim.x) a.items[i] = make_int4(-1, 0, 0, -1);
}

// Sixteen weights, or their gradients, rounded: the operand of two products.
template <bool BF>
VH_DEV void pack16(const f32x16& s, uint4 (&p)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    p[i] = make_uint4(pack2<BF>(s[8 * i], s[8 * i + 1]), pack2<BF>(s[8 * i + 2], s[8 * i + 3]),
                      pack2<BF>(s[8 * i + 4], s[8 * i + 5]), pack2<BF>(s[8 * i + 6], s[8 * i + 7]));
}

// What that left out.
template <bool BF>
VH_DEV void rest16(const f32x16& s, const uint4 (&p)[2], uint4 (&low)[2]) {
  f32x16 rest;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 u = unpack2<BF>(w[j]);
      rest[8 * i + 2 * j] = s[8 * i + 2 * j] - u[0];
      rest[8 * i + 2 * j + 1] = s[8 * i + 2 * j + 1] - u[1];
    }
  }
  pack16<BF>(rest, low);
}

// float16 has no room for the gradients of weights as they come.  They are
// multiplied by a power of two, a column's own: the largest of its gradients
// so far lies at 2^11 to 2^15, so that a gradient goes down to 2^-36 of it.
// Weights, at most 1, are lifted by 2^15.
template <bool BF>
struct Lift {
  static constexpr float LOG = weights_lift(BF), BACK = BF ? 1.0f : 0x1p-15f, FIRST = BF ? 1.0f : 0x1p100f;
};
template <bool BF, int N>
VH_DEV void lift(f32x16& ds, float& up, f32x16 (&acc)[N]) {
  if constexpr (!BF) {
    float most = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(ds[r]));
    most = max_halves(most);
    const bool over = most * up > 0x1p15f;
    if (__any(over)) {
      const int e = (int)(__float_as_uint(most) >> 23);
      const float to = over ? __uint_as_float((uint32_t)min(max(265 - e, 1), 227) << 23) : up, by = to / up;
      up = to;
#pragma unroll
      for (int c = 0; c < N; ++c) acc[c] *= by;
    }
    ds *= up;
  }
}

// The rows of long sequences have many keys, whose weights' rounding averages out:
// their gradients are off by 1.34 to 1.62 times a result's own rounding.  Those of short
// ones (under VH_PROMPT_SHORT rows) have few, down to two: a weight's rounding is seen
// in a gradient, and twice in D, which is a sum over the output, that has it as well.
// They take D as a sum over the weights instead, and weights and their gradients in
// two parts of 16 bits, each with a product of its own: 1.00 times the rounding.  A
// block with rows of such sequences does so in the tiles in which they meet their
// keys, whatever else it holds (two loops: a choice in the loop costs registers, and
// spills in both cases).  The second parts take 6 to 12% of the two kernels' time (us of dq,
// and of dk and dv, without and with them: 32 sequences of 256, 32 + 8 heads of 128,
// 104 + 78 and 109 + 91; 20 of 400, heads of 64, 82 + 70 and 86 + 84; 64 of 125,
// 16 + 16 heads of 64, 40 + 41 and 42 + 45), and D by the keys two fifths of dq's
// products: too much for long rows.
// ------------------------------------------------------------------ dq
constexpr int DQ_KEYS = 64;  // of a tile; a wave takes 32 at a time

template <int D, bool BF, int HALVES, bool CAREFUL>
VH_DEV bool prompt_dq_block(const Args& a, int id, char* lds) {
  constexpr int BYTES = DQ_KEYS * D * 2;
  const int turn = Halves<D, HALVES>::half();
  char* tiles = lds + turn * 4 * BYTES;
  const int rank = id / a.heads, spread = id - rank * a.heads;
  const int kv = spread % a.kv_heads, head = kv * a.group + spread / a.kv_heads;
  const int row0 = a.order[rank] * BLOCK, wave = __builtin_amdgcn_readfirstlane(threadIdx.x % THREADS / 64), lane = threadIdx.x & 63;
  const int wave0 = row0 + 32 * wave, row = wave0 + (lane & 31), half = lane >> 5;
  const bool in = row < a.tokens;
  const int first = in ? a.first[row] : row + 1;
  const int wave_first = __builtin_amdgcn_readlane(first, 0), wave_last_first = __builtin_amdgcn_readlane(first, 31);
  const int begin = a.first[row0], end = min(row0 + BLOCK, a.tokens);
  uint4 q[D / 16], go[D / 16];
  load_columns<D>(a.q, head, wave0, a.tokens, q);
  load_columns<D>(a.go, head, wave0, a.tokens, go);
  // D, and lse log2(e), which is inf where a row sees nothing, so that its weights are 0: for the keys' pass as well
  const float natural = in ? a.lse[(int64_t)row * a.heads + head] : -__builtin_inff();
  const float lse = natural == -__builtin_inff() ? __builtin_inff() : log2_units(natural);
  // weights are off together by what lse leaves out, and dq is a sum over them
  const float unit = in ? exp2_fast(a.rest[(int64_t)head * a.tokens + row] - Lift<BF>::LOG) : 1.0f;
  Loader<D, DQ_KEYS> kl, vl;
  kl.init(a.k, kv);
  vl.init(a.v, kv);
  const float scale = a.scale * LOG2E;
  const Run of = short_run(a, row0);
  float dot = 0.0f;
  if (!covers(a, of, row0)) {
    uint4 o[D / 16];
    const Tensor out{a.o, (int64_t)a.heads * D, D}, low{a.o_low, (int64_t)a.heads * D, D};
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      load_columns<D>(part == 0 ? out : low, head, wave0, a.tokens, o);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const uint32_t xs[4] = {o[s].x, o[s].y, o[s].z, o[s].w}, ys[4] = {go[s].x, go[s].y, go[s].z, go[s].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2 u = part == 0 ? unpack2<BF>(xs[i]) : unpack2<true>(xs[i]), v = unpack2<BF>(ys[i]);
          dot = __builtin_fmaf(u[0], v[0], dot);
          dot = __builtin_fmaf(u[1], v[1], dot);
        }
      }
    }
    dot = sum_halves(dot);
  }
  if (of.some()) {
    // D as sum P dP, by the short sequences' keys once more (each half of a workgroup by
    // all of them), and over sum P, as the weights of far scores are off together by
    // what lse in 32 bits is.
    float by_weights = 0.0f, all = 0.0f;
    for (int key0 = of.from; key0 < end; key0 += DQ_KEYS) {
      if (key0 > of.from) __syncthreads();
      kl.load(tiles, key0, a.tokens);
      vl.load(tiles + 2 * BYTES, key0, a.tokens);
      arrived();
#pragma unroll
      for (int sub = 0; sub < DQ_KEYS; sub += 32) {
        const int key = key0 + sub;
        if (key >= wave0 + 32 || key + 32 <= wave_first) continue;
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) s = mfma<BF>(rows_operand<D>(tiles, sub, i), q[i], s);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) dp = mfma<BF>(rows_operand<D>(tiles + 2 * BYTES, sub, i), go[i], dp);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = key + result_row(r) + 4 * half;
          const float p = j >= first && j <= row ? exp2_fast(__builtin_fmaf(s[r], scale, -lse)) : 0.0f;
          all += p;
          by_weights += p > 0.0f ? p * dp[r] : 0.0f;
        }
      }
    }
    by_weights = sum_halves(by_weights);
    all = sum_halves(all);
    if (row >= of.from && row < of.to) dot = all == 0.0f ? by_weights : by_weights / all;
    __syncthreads();  // the tiles are loaded over next
  }
  if (in && turn == 0) {
    float* to = a.rows + (int64_t)head * 2 * a.tokens + row;
    if (half == 0) to[0] = lse;
    else to[a.tokens] = dot;
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc[c] = f32x16{};
  float up = Lift<BF>::FIRST;
  // the tiles before the short sequences' keys, and the rest, which take two parts: two loops
  const int parted = of.some() ? begin + max(of.from - begin, 0) / DQ_KEYS * DQ_KEYS : end;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const bool two = part > 0;
    const int from = two ? parted : begin, to = two ? end : parted;
    if (two) __syncthreads();  // the tiles are loaded over next
    const int first_key = from + turn * DQ_KEYS;
    if (first_key < to) {
      kl.load(tiles, first_key, a.tokens);
      vl.load(tiles + 2 * BYTES, first_key, a.tokens);
    }
    int at = 0;
    for (int key0 = first_key; key0 - turn * DQ_KEYS < to; key0 += HALVES * DQ_KEYS, at ^= 1) {
      arrived();
      if (key0 + HALVES * DQ_KEYS < to) {
        kl.load(tiles + (at ^ 1) * BYTES, key0 + HALVES * DQ_KEYS, a.tokens);
        vl.load(tiles + (2 + (at ^ 1)) * BYTES, key0 + HALVES * DQ_KEYS, a.tokens);
      }
      if (HALVES > 1 && key0 >= to) continue;
      const char *k = tiles + at * BYTES, *v = tiles + (2 + at) * BYTES;
#pragma unroll
      for (int sub = 0; sub < DQ_KEYS; sub += 32) {
        const int key = key0 + sub;
        if (key >= wave0 + 32 || key + 32 <= wave_first) continue;
        const bool masked = key + 32 > wave0 + 1 || key < wave_last_first;
        f32x16 s = {}, ds = {};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) s = mfma<BF>(rows_operand<D>(k, sub, i), q[i], s);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) ds = mfma<BF>(rows_operand<D>(v, sub, i), go[i], ds);
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = exp2_fast(__builtin_fmaf(s[r], scale, -lse)) * (ds[r] - dot);
        uint32_t bad = 0u;
        if (CAREFUL && masked) bad = bad_rows<D, BF>(k, sub) >> (4 * half);
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = key + result_row(r) + 4 * half;
            // a key that holds an infinity or NaN is left out of the product: it makes its rows NaN
            const float seen = CAREFUL && (bad >> result_row(r) & 1u) ? __builtin_nanf("") : ds[r];
            ds[r] = j >= first && j <= row ? seen : 0.0f;
          }
        }
        lift<BF>(ds, up, acc);
        uint4 p[2], low[2];
        pack16<BF>(ds, p);
        if (two) rest16<BF>(ds, p, low);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint4 x = turned_operand<D>(k, sub + 16 * i, c);
            if (CAREFUL && masked) x = finite_part<BF>(x);
            acc[c] = mfma<BF>(x, p[i], acc[c]);
            if (two) acc[c] = mfma<BF>(x, low[i], acc[c]);
          }
      }
    }
  }
  if constexpr (HALVES > 1) {
    constexpr int N = D / 2 + 1;
    __syncthreads();
    float* to = lane_slot(lds, N);
    if (turn > 0) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(16 * c + r) * 64] = acc[c][r];
      to[(N - 1) * 64] = up;
    }
    __syncthreads();
    if (turn > 0) return false;
    const float mine = 1.0f / up, by = 1.0f / to[(N - 1) * 64];
    up = 1.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[c][r] = acc[c][r] * mine + to[(16 * c + r) * 64] * by;
  }
  store_columns<D, D, BF>(a.gq, nullptr, a.heads, head, row, in, 0, acc, a.scale / up * unit);
  return !CAREFUL && in && any_nonfinite(acc);
}

template <int D, bool BF, int HALVES>
__global__ void __launch_bounds__(HALVES* THREADS, back_waves_of(D)) k_prompt_dq(Args a, int item_groups) {
  __shared__ __attribute__((aligned(16))) char s_tiles[HALVES * 4 * DQ_KEYS * D * 2];
  static_assert(sizeof(s_tiles) >= ITEM_BYTES, "the items' lists");
  const int id = (int)blockIdx.x - item_groups;
  if (id < 0) {
    prompt_items(a, blockIdx.x, item_groups, s_tiles);
    return;
  }
  const bool apart = prompt_dq_block<D, BF, HALVES, false>(a, id, s_tiles);
  if (__syncthreads_or(apart)) prompt_dq_block<D, BF, HALVES, true>(a, id, s_tiles);
}

// ------------------------------------------------------------- dk and dv
// A wave's 32 keys, `C` channels of dk and dv from channel 32 c0 on, over a
// chunk of the rows that see them.  The scores' products contract over all D: K
// of the wave's keys stays in registers, and V where they hold both; heads of
// 128 have the block's V in LDS.
template <int D, int C, bool BF, bool CAREFUL>
VH_DEV bool prompt_dk_block(const Args& a, const int4& item, char* tiles) {
  constexpr int BYTES = DK_ROWS * D * 2, PARTS = D / C;
  constexpr bool V_LDS = D == 128;
  const int spread = blockIdx.x % (a.kv_heads * PARTS);
  const int kv = spread % a.kv_heads, c0 = spread / a.kv_heads * (C / 32);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int key0 = item.x * BLOCK, begin = item.y, end = item.z;
  const int wave0 = key0 + 32 * wave, key = wave0 + (lane & 31), half = lane >> 5;
  const bool in = key < a.tokens;
  const int past = in ? a.past[key] : key;  // the row after the last that sees the key
  const int wave_past = __builtin_amdgcn_readlane(past, 0), wave_last_past = __builtin_amdgcn_readlane(past, 31);
  char *s_rows = tiles + 4 * BYTES, *s_v = s_rows + 2 * STATS;  // lse, D and the rest of lse of a tile's rows; V
  uint4 k[D / 16], v[V_LDS ? 1 : D / 16];
  load_columns<D>(a.k, kv, wave0, a.tokens, k);
  if constexpr (!V_LDS) load_columns<D>(a.v, kv, wave0, a.tokens, v);
  const float scale = a.scale * LOG2E;
  f32x16 dk[C / 32], dv[C / 32];
#pragma unroll
  for (int c = 0; c < C / 32; ++c) dk[c] = dv[c] = f32x16{};
  float up = Lift<BF>::FIRST;
  if constexpr (V_LDS) {
    if (end > begin) {  // nothing is left on its way to LDS by a workgroup that ends
      Loader<D, BLOCK> vl;
      vl.init(a.v, kv);
      vl.load(s_v, key0, a.tokens);
    }
  }
  // the tiles of short sequences' rows, which take two parts, and the rest: two loops
  const int parted = min(begin + (max(short_run(a, key0).to - begin, 0) + DK_ROWS - 1) / DK_ROWS * DK_ROWS, end);
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const bool two = part == 0;
    const int from = two ? begin : parted, to = two ? parted : end;
    if (!two) __syncthreads();  // the tiles are loaded over next
    Loader<D, DK_ROWS> ql, gl;
    const int rounds = to > from ? (to - from + DK_ROWS - 1) / DK_ROWS : 0, all = rounds * a.group;
    int next_head = kv * a.group, next_row = from;
    ql.init(a.q, next_head);
    gl.init(a.go, next_head);
    const auto load_next = [&](int at) __attribute__((always_inline)) {
      ql.load(tiles + at * BYTES, next_row, a.tokens);
      gl.load(tiles + (2 + at) * BYTES, next_row, a.tokens);
      if (wave == 0) {
        const i32x4 r = buffer_of((const char*)(a.rows + (int64_t)next_head * 2 * a.tokens), a.tokens * 8);
        load_to_lds<4>(r, ((lane >> 5) * a.tokens + next_row + (lane & 31)) * 4,
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(s_rows + at * STATS)));
      }
      if (wave == 1) {
        const i32x4 r = buffer_of((const char*)(a.rest + (int64_t)next_head * a.tokens), a.tokens * 4);
        load_to_lds<4>(r, (next_row + lane) * 4, (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(s_rows + at * STATS + 256)));
      }
      next_row += DK_ROWS;
      if (next_row >= to) {
        next_row = from;
        ++next_head;
        ql.base += a.q.sh * 2;
        gl.base += a.go.sh * 2;
      }
    };
    if (all > 0) load_next(0);
    int at = 0, row0 = from;
    for (int n = 0; n < all; ++n, at ^= 1) {
      arrived();
      if (n + 1 < all) load_next(at ^ 1);
      const int first_row = row0;
      row0 = row0 + DK_ROWS >= to ? from : row0 + DK_ROWS;
      if (first_row + DK_ROWS <= wave0 || first_row >= wave_last_past) continue;
      const bool masked = first_row < wave0 + 31 || first_row + DK_ROWS > wave_past;
      const char *q = tiles + at * BYTES, *go = tiles + (2 + at) * BYTES;
      const float* stats = (const float*)(s_rows + at * STATS) + 4 * half;
      f32x16 s = {};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s = mfma<BF>(rows_operand<D>(q, 0, i), k[i], s);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_fast(__builtin_fmaf(s[r], scale, -stats[result_row(r)]) + stats[64 + result_row(r)]);
      uint32_t bad_go = 0u, bad_q = 0u;
      if (CAREFUL && masked) {
        bad_go = bad_rows<D, BF>(go, 0) >> (4 * half);
        bad_q = bad_rows<D, BF>(q, 0) >> (4 * half);
      }
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = first_row + result_row(r) + 4 * half;
          s[r] = row >= key && row < past ? s[r] : 0.0f;
        }
      }
      f32x16 w = s;
      if (CAREFUL && masked) {  // a row that holds an infinity or NaN is left out of the products: it makes the keys that it sees NaN
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = first_row + result_row(r) + 4 * half;
          if ((bad_go >> result_row(r) & 1u) && row >= key && row < past) w[r] = __builtin_nanf("");
        }
      }
      {
        uint4 p[2], low[2];
        pack16<BF>(w, p);
        if (two) rest16<BF>(w, p, low);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < C / 32; ++c) {
            uint4 x = turned_operand<D>(go, 16 * i, c0 + c);
            if (CAREFUL && masked) x = finite_part<BF>(x);
            dv[c] = mfma<BF>(x, p[i], dv[c]);
            if (two) dv[c] = mfma<BF>(x, low[i], dv[c]);
          }
      }
      f32x16 ds = {};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint4 of_v;
        if constexpr (V_LDS) of_v = rows_operand<D>(s_v, 32 * wave, i);
        else of_v = v[i];
        ds = mfma<BF>(rows_operand<D>(go, 0, i), of_v, ds);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = s[r] * (ds[r] - stats[32 + result_row(r)]);
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = first_row + result_row(r) + 4 * half;
          const float seen = CAREFUL && (bad_q >> result_row(r) & 1u) ? __builtin_nanf("") : ds[r];
          ds[r] = row >= key && row < past ? seen : 0.0f;
        }
      }
      lift<BF>(ds, up, dk);
      {
        uint4 p[2], low[2];
        pack16<BF>(ds, p);
        if (two) rest16<BF>(ds, p, low);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < C / 32; ++c) {
            uint4 x = turned_operand<D>(q, 16 * i, c0 + c);
            if (CAREFUL && masked) x = finite_part<BF>(x);
            dk[c] = mfma<BF>(x, p[i], dk[c]);
            if (two) dk[c] = mfma<BF>(x, low[i], dk[c]);
          }
      }
    }
  }
  const float k_by = a.scale / up * Lift<BF>::BACK, v_by = Lift<BF>::BACK;
  if (item.w < 0) {
    store_columns<D, C, BF>(a.gk, nullptr, a.kv_heads, kv, key, in, c0, dk, k_by);
    store_columns<D, C, BF>(a.gv, nullptr, a.kv_heads, kv, key, in, c0, dv, v_by);
  } else {
    float* to = a.part + ((int64_t)item.w * a.kv_heads + kv) * (2 * BLOCK * D) + (key - key0) * D + 32 * c0 + 4 * half;
#pragma unroll
    for (int c = 0; c < C / 32; ++c)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        *(float4*)(to + 32 * c + result_row(r)) = make_float4(dk[c][r] * k_by, dk[c][r + 1] * k_by, dk[c][r + 2] * k_by, dk[c][r + 3] * k_by);
        *(float4*)(to + BLOCK * D + 32 * c + result_row(r)) =
            make_float4(dv[c][r] * v_by, dv[c][r + 1] * v_by, dv[c][r + 2] * v_by, dv[c][r + 3] * v_by);
      }
  }
  return !CAREFUL && in && (any_nonfinite(dk) || any_nonfinite(dv));
}

template <int D, int C, bool BF>
__global__ void __launch_bounds__(THREADS, back_waves_of(D)) k_prompt_dk(Args a) {
  __shared__ __attribute__((aligned(16))) char s_tiles[4 * DK_ROWS * D * 2 + 2 * STATS + (D == 128 ? BLOCK * D * 2 : 0)];
  const int rank = blockIdx.x / (a.kv_heads * (D / C));
  int4 item = make_int4(0, 0, 0, -1);
  if (a.items) {
    item = a.items[rank];
    if (item.x < 0) return;
  } else {
    item.x = a.order[rank];
    item.y = item.x * BLOCK;
    item.z = a.past[min(item.y + BLOCK, a.tokens) - 1];
  }
  const bool apart = prompt_dk_block<D, C, BF, false>(a, item, s_tiles);
  if (__syncthreads_or(apart)) prompt_dk_block<D, C, BF, true>(a, item, s_tiles);
}

// The sums of a block's items joined, in their order: a thread has 4 channels
// of a key.
template <int D, bool BF>
__global__ void __launch_bounds__(THREADS) k_prompt_join(Args a) {
  const int block = blockIdx.x / a.kv_heads, kv = blockIdx.x - block * a.kv_heads;
  const int2 join = a.joins[block];
  if (join.y <= 1) return;
  const float* part = a.part + ((int64_t)join.x * a.kv_heads + kv) * (2 * BLOCK * D);
  const int64_t apart = (int64_t)a.kv_heads * (2 * BLOCK * D);
  const int i = blockIdx.y * THREADS + threadIdx.x, which = i / (BLOCK * D / 4), at = (i - which * (BLOCK * D / 4)) * 4;
  const int key = block * BLOCK + at / D;
  if (key >= a.tokens) return;
  float4 sum = *(const float4*)(part + i * 4);
  for (int c = 1; c < join.y; ++c) {
    const float4 x = *(const float4*)(part + c * apart + i * 4);
    sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
  }
  *(uint2*)((uint16_t*)(which ? a.gv : a.gk) + ((int64_t)key * a.kv_heads + kv) * D + at % D) =
      make_uint2(pack2<BF>(sum.x, sum.y), pack2<BF>(sum.z, sum.w));
}

template <int D, bool BF>
void backward_of(Args a, const int32_t* q_order, const int32_t* k_order, hipStream_t s) {
  constexpr int C = key_channels_of(D);
  const unsigned blocks = (unsigned)((a.tokens + BLOCK - 1) / BLOCK), groups = a.items ? (blocks + 63) / 64 : 0;
  a.order = q_order;
  const dim3 grid(blocks * a.heads + groups);
  const dim3 k_grid((a.items ? a.item_count : blocks) * a.kv_heads * (D / C));
  bool halves = false;
  if constexpr (D <= 128) {
    halves = in_halves(a, back_waves_of(D));
    if (halves) hipLaunchKernelGGL((k_prompt_dq<D, BF, 2>), grid, dim3(2 * THREADS), 0, s, a, (int)groups);
  }
  if (!halves) hipLaunchKernelGGL((k_prompt_dq<D, BF, 1>), grid, dim3(THREADS), 0, s, a, (int)groups);
  a.order = k_order;
  hipLaunchKernelGGL((k_prompt_dk<D, C, BF>), k_grid, dim3(THREADS), 0, s, a);
  if (a.items) hipLaunchKernelGGL((k_prompt_join<D, BF>), dim3(blocks * a.kv_heads, 2 * BLOCK * D / 4 / THREADS), dim3(THREADS), 0, s, a);
}

template <int D>
int backward(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s) {
  if (bf16) backward_of<D, true>(a, q_order, k_order, s);
  else backward_of<D, false>(a, q_order, k_order, s);
  return vh::check_launch("vh_prompt_attention_backward");
}

}  // namespace prompt
