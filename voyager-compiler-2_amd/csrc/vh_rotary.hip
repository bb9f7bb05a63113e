// Rotary positions of queries and keys: every pair (x0, x1) of a head turned
// by the angle pos * frequency of its pair, in one launch for both tensors.
//
//   y0 = f * (x0 cos - x1 sin),  y1 = f * (x1 cos + x0 sin)
//
// The gradient is the same turn the other way (sin -> -sin).  Channels past
// the rotated part are copied.
//
// The angle is formed in float64 as turns (position times turns per position,
// then the fraction): at position 1e6 a float32 product is off by 0.06 turns,
// the float64 one by less than 1e-9.  Sine and cosine are taken of the fraction,
// once per token and pair, and shared by all heads through LDS: for 16-bit
// values in float32 (off by less than 2^-22, where a result rounds by 2^-12 or
// more), for float32 ones in float64, rounded once with the factor.
//
// Bound by memory: 4 bytes moved per bfloat16 value, 3 operations.  32 + 8
// heads of 128 in bfloat16: 8192 tokens (168 MB read and written) 29-33 us,
// 5.1-5.8 TB/s with part of it in the last cache; a single token 2.5 us, its
// loads' and the launch's latency.  5001 tokens of 16 + 4 heads of 128 in
// float32, half of each turned (102 MB): 17.3 us.
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_DIM = 512;
constexpr int ROPE_TOKENS = 4;  // tokens of a workgroup when there are many

struct RopeTensor {
  const void* x;
  void* y;
  int64_t sb, st, sh;  // input strides: batch, token, head (channels are dense)
};

struct RopeArgs {
  RopeTensor q, k;
  const void* pos;
  int64_t pos_sb, pos_st;
  const double* turns;  // [rotary / 2] turns per position
  int64_t tokens;       // tokens of a sequence
  int64_t rows;         // batch * tokens
  FastDiv heads_div;    // by nq + nk
  int nq, nk, dim, rotary, units, pos64;
  float factor;  // of cosine and sine
  float sign;    // of sine: -1 turns back
};

// 16 bytes (VEC values) or one value at element `at`.
template <typename T, int VEC>
VH_DEV void rope_load(const void* p, int64_t at, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = (float)((const T*)p)[at];
  } else {
    const uint4 v = *(const uint4*)((const T*)p + at);
    T e[VEC];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = (float)e[i];
  }
}

template <typename T, int VEC>
VH_DEV void rope_store(void* p, int64_t at, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    ((T*)p)[at] = (T)x[0];
  } else {
    T e[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = (T)x[i];
    uint4 v;
    __builtin_memcpy(&v, e, 16);
    *(uint4*)((T*)p + at) = v;
  }
}

// A unit is 2 * VEC values of a head: VEC pairs of the rotated part, or as
// many values to copy.  Consecutive threads take consecutive units of a head,
// then the next head, then the next token.
template <typename T, int VEC, bool INTERLEAVED, int TOKENS>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope(RopeArgs a) {
  __shared__ float2 s_cs[TOKENS * (ROPE_MAX_DIM / 2)];
  const int half = a.rotary / 2;
  const int64_t row0 = (int64_t)blockIdx.x * TOKENS;
  const int rows = (int)(a.rows - row0 < TOKENS ? a.rows - row0 : TOKENS);
  for (int i = threadIdx.x; i < rows * half; i += ROPE_THREADS) {
    const int t = i / half, j = i - t * half;
    const int64_t b = (row0 + t) / a.tokens, n = (row0 + t) - b * a.tokens;
    const int64_t at = b * a.pos_sb + n * a.pos_st;
    const int64_t p = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
    const double turn = (double)p * a.turns[j];
    if constexpr (sizeof(T) == 4) {
      double s, c;
      sincospi(2.0 * (turn - rint(turn)), &s, &c);
      s_cs[t * half + j] = make_float2((float)(c * a.factor), (float)(s * a.factor * a.sign));
    } else {
      float s, c;
      sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
      s_cs[t * half + j] = make_float2(c * a.factor, s * a.factor * a.sign);
    }
  }
  __syncthreads();
  const int heads = a.nq + a.nk;
  const int per = ROPE_THREADS / a.units;  // heads in flight
  const int u = threadIdx.x % a.units, lane_head = threadIdx.x / a.units;
  if (lane_head >= per) return;
  const int step = per * gridDim.y;
  for (int i = lane_head + per * blockIdx.y; i < rows * heads; i += step) {
    const int t = TOKENS == 1 ? 0 : (int)fast_div((uint32_t)i, a.heads_div);
    const int h = i - t * heads;
    const int64_t row = row0 + t, b = row / a.tokens, n = row - b * a.tokens;
    const bool key = h >= a.nq;
    const int hh = key ? h - a.nq : h;
    const void* x = key ? a.k.x : a.q.x;
    void* y = key ? a.k.y : a.q.y;
    const int64_t in = key ? b * a.k.sb + n * a.k.st + hh * a.k.sh : b * a.q.sb + n * a.q.st + hh * a.q.sh;
    const int64_t out = (row * (key ? a.nk : a.nq) + hh) * a.dim;
    float x0[VEC], x1[VEC], y0[VEC], y1[VEC];
    const bool turned = u * 2 * VEC < a.rotary;
    // a pair's first and second values: apart by half the rotated part, or side by side
    const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
    const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
    rope_load<T, VEC>(x, in + c0, x0);
    rope_load<T, VEC>(x, in + c1, x1);
    if (!turned) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        y0[j] = x0[j];
        y1[j] = x1[j];
      }
    } else {
      const float2* cs = s_cs + t * half + u * VEC;
      if constexpr (INTERLEAVED) {
        float z[2 * VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          z[j] = x0[j];
          z[VEC + j] = x1[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 w = cs[j];
          const float e = z[2 * j], o = z[2 * j + 1];
          z[2 * j] = e * w.x - o * w.y;
          z[2 * j + 1] = o * w.x + e * w.y;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          y0[j] = z[j];
          y1[j] = z[VEC + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 w = cs[j];
          y0[j] = x0[j] * w.x - x1[j] * w.y;
          y1[j] = x1[j] * w.x + x0[j] * w.y;
        }
      }
    }
    rope_store<T, VEC>(y, out + c0, y0);
    rope_store<T, VEC>(y, out + c1, y1);
  }
}

template <typename T, int VEC>
void rope_launch(const RopeArgs& a, bool interleaved, hipStream_t s) {
  const int heads = a.nq + a.nk;
  // Many tokens: four a workgroup share the launch's cost, and fill it where
  // heads are few.  Fewer: one each, its heads over several workgroups, so that
  // a token's load and store are one trip each.  (us with four and with one;
  // 32 + 8 heads of 128: 64 tokens 5.6 and 3.1, 1024 6.8 and 5.7, 2048 9.4 and
  // 9.2, 8192 28.1 and 28.9; 8 + 1 heads: 1024 4.1 and 3.6, 16384 14.8 and 21.6.)
  if (a.rows >= 2048) {
    const dim3 grid((unsigned)((a.rows + ROPE_TOKENS - 1) / ROPE_TOKENS));
    if (interleaved) hipLaunchKernelGGL((k_rope<T, VEC, true, ROPE_TOKENS>), grid, dim3(ROPE_THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_rope<T, VEC, false, ROPE_TOKENS>), grid, dim3(ROPE_THREADS), 0, s, a);
  } else {
    const int per = ROPE_THREADS / a.units;
    const dim3 grid((unsigned)a.rows, (unsigned)((heads + per - 1) / per));
    if (interleaved) hipLaunchKernelGGL((k_rope<T, VEC, true, 1>), grid, dim3(ROPE_THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_rope<T, VEC, false, 1>), grid, dim3(ROPE_THREADS), 0, s, a);
  }
}

// Whether 16-byte accesses of VEC values are aligned in this tensor; if not,
// values are taken one by one.
bool rope_aligned(const RopeTensor& t, int vec) {
  return (uintptr_t)t.x % 16 == 0 && (uintptr_t)t.y % 16 == 0 && t.sb % vec == 0 && t.st % vec == 0 && t.sh % vec == 0;
}

template <typename T>
void rope_dispatch(RopeArgs& a, bool interleaved, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = a.dim % (2 * VEC) == 0 && a.rotary % (2 * VEC) == 0 && rope_aligned(a.q, VEC) && rope_aligned(a.k, VEC);
  a.units = a.dim / (wide ? 2 * VEC : 2);
  if (wide) rope_launch<T, VEC>(a, interleaved, s);
  else rope_launch<T, 1>(a, interleaved, s);
}

}  // namespace

extern "C" int vh_rope(const vh_rope_desc* d, vh_stream_t stream) {
  VH_REQUIRE(d, "vh_rope: null descriptor");
  VH_REQUIRE(vh::is_float_dtype(d->dtype), "vh_rope: dtype must be bfloat16, float16 or float32");
  VH_REQUIRE(d->batch >= 0 && d->tokens >= 0 && d->heads >= 0 && d->kv_heads >= 0, "vh_rope: negative size");
  VH_REQUIRE(d->dim > 0 && d->dim <= ROPE_MAX_DIM && d->dim % 2 == 0, "vh_rope: dim must be even and at most %d (got %d)",
             ROPE_MAX_DIM, d->dim);
  VH_REQUIRE(d->rotary > 0 && d->rotary <= d->dim && d->rotary % 2 == 0,
             "vh_rope: the rotated part must be even and at most dim");
  VH_REQUIRE(d->pos_bits == 32 || d->pos_bits == 64, "vh_rope: positions of 32 or 64 bits");
  VH_REQUIRE(d->batch < (1ll << 31) && d->tokens < (1ll << 31), "vh_rope: too many rows");
  const int64_t rows = d->batch * d->tokens;
  if (rows == 0 || d->heads + (int64_t)d->kv_heads == 0) return VH_OK;
  VH_REQUIRE(rows < (1ll << 31) && (int64_t)d->heads + d->kv_heads < (1 << 20), "vh_rope: too many rows or heads");
  VH_REQUIRE((d->heads == 0 || (d->q && d->q_out)) && (d->kv_heads == 0 || (d->k && d->k_out)) && d->pos && d->turns,
             "vh_rope: null argument");
  const RopeTensor q{d->q, d->q_out, d->q_sb, d->q_st, d->q_sh}, k{d->k, d->k_out, d->k_sb, d->k_st, d->k_sh};
  // a tensor without heads is never read: the other one's stands for it
  RopeArgs a{d->heads ? q : k, d->kv_heads ? k : q, d->pos, d->pos_sb, d->pos_st, d->turns, d->tokens, rows,
             make_fast_div((uint32_t)(d->heads + d->kv_heads)), d->heads, d->kv_heads, d->dim, d->rotary, 0,
             d->pos_bits == 64, d->factor, d->inverse ? -1.0f : 1.0f};
  hipStream_t s = vh::as_stream(stream);
  if (d->dtype == VH_BF16) rope_dispatch<__bf16>(a, d->interleaved != 0, s);
  else if (d->dtype == VH_F16) rope_dispatch<_Float16>(a, d->interleaved != 0, s);
  else rope_dispatch<float>(a, d->interleaved != 0, s);
  return vh::check_launch("vh_rope");
}
