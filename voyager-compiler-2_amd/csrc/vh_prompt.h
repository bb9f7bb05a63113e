// Causal attention of packed sequences with grouped heads, forward and backward.
//
// Row i of a sequence that begins at row first(i) sees the keys first(i) ... i:
//
//   s_ij = scale * q_i . k_j,  o_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij),
//   lse_i = log sum_j exp(s_ij)
//
// and back, with D_i = do_i . o_i, P = exp(s - lse) and dS = P (do v^T - D),
//
//   dv = P^T do,  dq = scale dS k,  dk = scale dS^T q,
//
// dk and dv summed over the query heads of a group.
//
// Rows are cut into blocks of 128 without regard to where sequences begin:
// short sequences share a block, the grid goes by the number of rows alone,
// and a row's keys are told by first(i), which rises with i.  A plan made
// once for a batch holds first(i), the row after the last that sees key j, and
// the blocks in the order of their work, the most first, so that the card
// ends together.
//
// A wave holds 32 rows (of the keys' pass 32 keys) as columns of the matrix
// instructions: S^T = K Q^T leaves a lane with 16 scores of one row, so a row's
// maximum is one exchange between two lanes, and these scores, rounded to 16
// bits, are the lane's share of the operand of the next product (O^T = V^T P^T;
// the order of keys inside a product is free, and V is taken in the order in
// which S^T comes out).  Tiles of keys (of rows, in the keys' pass) go from
// memory to LDS without registers between, the next while one is used.  A tile
// is stored by rows; where a product contracts over its rows, it is read
// transposed by the LDS's own transposing reads.  16-byte pieces of a row are
// permuted by its number so that both kinds of reads spread over all banks.
#pragma once

#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace prompt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int THREADS = 256, WAVES = 4;  // that share a tile
constexpr int BLOCK = VH_PROMPT_BLOCK;  // rows of a workgroup, 32 a wave
// Waves of a SIMD that the registers are held to, forward and back.
constexpr int waves_of(int d) { return d == 64 ? 4 : d == 128 ? 2 : 1; }
constexpr int back_waves_of(int d) { return d == 64 ? 3 : d == 128 ? 2 : 1; }
constexpr int MOST_CUT = 4096;  // blocks of keys, times the workgroups of each, that are cut into items
// Channels of a workgroup's dk and dv.
constexpr int key_channels_of(int d) { return d <= 128 ? d : 128; }
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

struct Tensor {
  const void* p;
  int64_t st, sh;  // strides of token and head, in elements
};

struct Args {
  Tensor q, k, v, go;
  const int32_t *first, *past, *order;  // of rows, keys, and of this pass's blocks
  void *o, *o_low, *gq, *gk, *gv;
  float* lse;         // [tokens, heads]
  float* rest;        // for the backward pass: [heads, tokens], what a weight's exponent, less lse, takes more
  float* rows;        // backward: [heads, 2, tokens], lse log2(e) and D
  // backward, where key blocks are cut into items:
  int4* items;        // [item_count]: block (-1: none), first row, row after the last, slot of its sums (-1: they are the result)
  int2* joins;        // [blocks]: first slot, and slots
  float* part;        // [slots, kv_heads, dk and dv, 128 keys, dim]
  int item_count, share;
  float scale;
  int tokens, sequences, heads, kv_heads, group;
};

// lse in units of log2, as the backward pass takes it from the natural one.
// Rounded in 32 bits it is off by what, for far scores, is seen in the weights
// (2^-10 of them at 2^13): `rest` is what is missing, and the lift of weights (Lift).
VH_DEV float log2_units(float lse) {
#pragma clang fp contract(off)
  return lse * LOG2E;
}
constexpr float weights_lift(bool bf16) { return bf16 ? 0.0f : 15.0f; }

// Where blocks are few for the card, or one is long beside them, two halves of
// a workgroup take a block's tiles in turn, and join through LDS: the longest
// block takes half the time.
template <int D, int HALVES>
struct Halves {
  static constexpr int WIDTH = HALVES * THREADS;
  __device__ __forceinline__ static int half() { return HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / THREADS); }
};
// One register of every lane of a wave, beside those of its other registers.
VH_DEV float* lane_slot(char* lds, int n) {
  return (float*)lds + (threadIdx.x % THREADS / 64 * n) * 64 + (threadIdx.x & 63);
}

// The element type's conversions and products.
template <bool BF>
VH_DEV uint32_t pack2(float x, float y) {
  const f32x2 v = {x, y};
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <bool BF>
VH_DEV f32x2 unpack2(uint32_t w) {
  if constexpr (BF) return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  else return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
}
// sum and both halves of w.
template <bool BF>
VH_DEV float add_pairs(uint32_t w, float sum) {
  if constexpr (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
}
template <bool BF>
VH_DEV f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
VH_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The 16-bit halves of w that are infinite or NaN, as a mask of their bits.
template <bool BF>
VH_DEV uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | (((w >> 16) & E) == E ? 0xffff0000u : 0u);
}

// The two lanes that hold a row, 32 apart.
VH_DEV float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
VH_DEV float sum_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A tile of ROWS rows of D channels in LDS.  Of a row, the 16-byte piece c is
// stored at place c ^ turn(row): 32 rows' pieces c, and 4 rows' 4 pieces from
// a multiple of 4 on, lie in different banks (a row of 64 channels is half of
// the banks' width, two are side by side).
template <int D>
struct Tile {
  static constexpr int PIECES = D / 8;  // of a row
  VH_DEV int turn(int row) {
    const int line = D == 64 ? row >> 1 : row;
    return D == 64 ? (line & 1) << 2 | ((line >> 1) & 3) : (line & 3) << 2 | ((line >> 2) & 3);
  }
  VH_DEV int place(int row, int piece) { return (row * PIECES + (piece ^ turn(row))) * 16; }  // in bytes
};

typedef __attribute__((address_space(3))) char lds_char;

// Operand A of a tile's 32 rows from row0 on, channels 16 s ...: a lane's row is
// lane % 32, its channels 16 s + 8 (lane / 32) ... + 7.
template <int D>
VH_DEV uint4 rows_operand(const char* tile, int row0, int s) {
  const int lane = threadIdx.x & 63;
  return *(const uint4*)(tile + Tile<D>::place(row0 + (lane & 31), 2 * s + (lane >> 5)));
}

// Operand A of the transpose: a lane's row is channel 32 c + lane % 32, its
// columns the tile's rows row0 + 4 (lane / 32) ... + 3 and 8 further, which
// are those of which a product over the tile's rows leaves it the results.
template <int D>
VH_DEV uint4 turned_operand(const char* tile, int row0, int c) {
  const int lane = threadIdx.x & 63, l = lane & 15;
  const int channel = 32 * c + 16 * ((lane >> 4) & 1) + 4 * (l & 3);
  const int row = row0 + 4 * (lane >> 5) + (l >> 2);
  const auto read = [&](int r) {
    const char* p = tile + Tile<D>::place(r, channel >> 3) + (channel & 4) * 2;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_char*)p);
  };
  const s16x4 a = read(row), b = read(row + 8);
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  return make_uint4(x.x, x.y, y.x, y.y);
}

// Loads ROWS rows of a tensor's head from row0 on into a tile, straight to
// LDS; rows past `rows` are zero.  Every thread of the workgroup calls it, and
// waits (`arrived`) before it reads (of a workgroup of two halves, every thread
// of a half).  The load is written out, as the compiler
// would wait for it before any read of LDS; it has no register for a result.
typedef int i32x4 __attribute__((ext_vector_type(4)));
VH_DEV i32x4 buffer_of(const char* p, int bytes) {
  const uint64_t at = (uint64_t)p;
  return i32x4{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
               __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
VH_DEV uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(const lds_char*)p; }
template <int BYTES>
VH_DEV void load_to_lds(i32x4 buffer, int offset, uint32_t to) {
  // M0 carries the LDS address, an operand, so that the compiler knows what it holds;
  // its write is one wait state before the load that uses it
  if constexpr (BYTES == 16)
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(buffer), "{m0}"(to) : "memory");
  else
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(offset), "s"(buffer), "{m0}"(to) : "memory");
}
// All loads of the workgroup have arrived, and all reads of what is loaded over next are done.
VH_DEV void arrived() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), which the compiler counts by as well
  __syncthreads();
}

template <int D, int ROWS>
struct Loader {
  static constexpr int EACH = ROWS * D * 2 / (16 * THREADS);  // 16-byte pieces a thread
  static constexpr int APART = THREADS / Tile<D>::PIECES;     // rows between them
  static constexpr int TURNS = APART % 16 ? 16 / APART : 1;   // after which their places in a row come again
  int offset[TURNS];                                          // of a thread's pieces, in bytes
  const char* base;
  int64_t step;  // bytes of a row
  uint32_t wave_at;  // of a wave's pieces in a tile, in bytes
  __device__ __forceinline__ void init(const Tensor& t, int head) {
    const int thread = threadIdx.x % THREADS;
    wave_at = (uint32_t)__builtin_amdgcn_readfirstlane(thread / 64 * 1024);
    base = (const char*)t.p + head * t.sh * 2;
    step = t.st * 2;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int row = i * APART + thread / Tile<D>::PIECES;
      offset[i] = row * (int)step + (((thread % Tile<D>::PIECES) ^ Tile<D>::turn(row)) * 16);
    }
  }
  __device__ __forceinline__ void load(const char* tile, int row0, int rows) const {
    const int n = rows - row0 < ROWS ? rows - row0 : ROWS;  // that there are
    const i32x4 r = buffer_of(base + row0 * step, n > 0 ? (int)((n - 1) * step) + D * 2 : 0);
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(tile)) + wave_at;
    int apart = (int)step * (APART * TURNS);
    asm volatile("" : "+s"(apart));  // sums are formed here, not kept
#pragma unroll
    for (int i = 0; i < EACH; ++i) load_to_lds<16>(r, offset[i % TURNS] + i / TURNS * apart, to + i * THREADS * 16);
  }
};

// A wave's 32 rows from row0 on as operand B, straight from memory; rows past
// `rows` are the last one's again.
template <int D>
VH_DEV void load_columns(const Tensor& t, int head, int row0, int rows, uint4 (&to)[D / 16]) {
  const int lane = threadIdx.x & 63, row = min(row0 + (lane & 31), rows - 1);
  const uint16_t* p = (const uint16_t*)t.p + row * t.st + head * t.sh + 8 * (lane >> 5);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) to[s] = *(const uint4*)(p + 16 * s);
}

// Row of a product's result r, of a lane's 16: 8 (r / 4) + r % 4, and 4 more in the upper half.
VH_DEV constexpr int result_row(int r) { return 8 * (r >> 2) + (r & 3); }

// A wave's 32 columns of C / 32 results, times `by`, to channels 32 c0 ... of
// rows of a contiguous tensor; what the rounding leaves out to `low`, if wanted.
template <int D, int C, bool BF>
VH_DEV void store_columns(void* o, void* low, int heads, int head, int row, bool in, int c0, const f32x16 (&acc)[C / 32], float by) {
  if (!in) return;
  const int64_t at = ((int64_t)row * heads + head) * D + 32 * c0 + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
  for (int c = 0; c < C / 32; ++c)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const float x[4] = {acc[c][r] * by, acc[c][r + 1] * by, acc[c][r + 2] * by, acc[c][r + 3] * by};
      const uint2 w = make_uint2(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]));
      *(uint2*)((uint16_t*)o + at + 32 * c + result_row(r)) = w;
      if (low) {
        const f32x2 u = unpack2<BF>(w.x), v = unpack2<BF>(w.y);
        *(uint2*)((uint16_t*)low + at + 32 * c + result_row(r)) =
            make_uint2(pack2<true>(x[0] - u[0], x[1] - u[1]), pack2<true>(x[2] - v[0], x[3] - v[1]));
      }
    }
}

// Whether any of a lane's results is infinite or NaN.
template <int N>
VH_DEV bool any_nonfinite(const f32x16 (&acc)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) m = __builtin_elementwise_maximum(m, fabsf(acc[c][r]));
  return !(m < __builtin_inff());
}

// Operand A without its infinities and NaNs.
template <bool BF>
VH_DEV uint4 finite_part(uint4 v) {
  return make_uint4(v.x & ~nonfinite<BF>(v.x), v.y & ~nonfinite<BF>(v.y), v.z & ~nonfinite<BF>(v.z), v.w & ~nonfinite<BF>(v.w));
}

// Of 32 rows of a tile, those that hold an infinity or NaN, as bits.
template <int D, bool BF>
VH_DEV uint32_t bad_rows(const char* tile, int row0) {
  const int lane = threadIdx.x & 63;
  uint32_t bad = 0u;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint4 v = rows_operand<D>(tile, row0, s);
    bad |= nonfinite<BF>(v.x) | nonfinite<BF>(v.y) | nonfinite<BF>(v.z) | nonfinite<BF>(v.w);
  }
  const uint64_t all = __ballot(bad != 0u);
  return (uint32_t)all | (uint32_t)(all >> 32);
}

// Whether two halves of a workgroup share a block: where one wave of workgroups
// holds all blocks, so that the longest is the pass, and sequences are long by
// their mean, empty ones among them, as the host knows no more of them.
// (us by one and by two, 16 + 4 heads: a prompt of 6000, heads of 64, 150 and 111,
// of 3000, heads of 128, 85 and 64; four of 775 44 and 36; 16 of 250 22 and 27.
// 32 + 8 heads of 128, 4096: 164 and 176.)
inline bool in_halves(const Args& a, int waves) {
  const int64_t blocks = (a.tokens + BLOCK - 1) / BLOCK;
  return blocks * a.heads <= 256 * waves && a.tokens >= (int64_t)VH_PROMPT_SHORT * a.sequences;
}

// The rows of the sequences of fewer than VH_PROMPT_SHORT rows that a block of rows
// has rows of, whose gradients take more care: from the first of the first to the
// last of the last.  Only the block's first and last sequence can be longer, so
// they lie one after another, with rows that pad at the end at most.
struct Run {
  int from, to;
  __device__ __forceinline__ bool some() const { return to > from; }
};
VH_DEV Run short_run(const Args& a, int row0) {
  const int end = min(row0 + BLOCK, a.tokens);
  const int first = a.first[row0], past = a.past[row0], last_first = a.first[end - 1], last_past = a.past[end - 1];
  if (first > row0) return Run{0, 0};  // all pad
  int from = first;
  if (past - first >= VH_PROMPT_SHORT) {
    // the next one, if there is one, is short, or long and the rest of the block
    if (past >= end || a.first[past] > past || a.past[past] - past >= VH_PROMPT_SHORT) return Run{0, 0};
    from = past;
  }
  const bool pads = last_first >= end;
  return Run{from, pads ? end : last_past - last_first < VH_PROMPT_SHORT ? last_past : last_first};
}
// Whether these are all of the block's rows.
VH_DEV bool covers(const Args& a, const Run& run, int row0) { return run.from <= row0 && run.to >= min(row0 + BLOCK, a.tokens); }

template <int D>
int forward(const Args& a, bool bf16, hipStream_t s);
template <int D>
int backward(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s);

}  // namespace prompt
