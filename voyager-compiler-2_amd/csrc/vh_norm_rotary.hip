// Norms of queries and keys a head, and their rotary positions, in one pass.
//
//   r = (mean x^2 + eps)^-1/2,  y = R(pos) (w x r)
//
// with R the turn of every pair by its position's angle (vh_rope) and w a
// weight a channel.  Back, with g = R^T dy and b = w g:
//
//   dw = sum over tokens and heads of g x r,  dx = r (b - x r mean(b x r))
//
// A head's channels lie with a group of 2^n lanes, so its squares are summed
// by exchanges inside the group and its values are read once.  Squares, sums
// and products are float32, results are rounded once.  The weights' gradient
// is summed in a fixed order: each lane over the heads that it takes, in float32
// (ten of 8192 tokens of 32 + 8 heads of 128); the lanes of a workgroup through LDS and
// the workgroups by a second kernel in float64, as sums of many equal terms in
// float32 are off by up to half their number.
//
// Bound by memory.  8192 tokens of 32 + 8 heads of 128 in bfloat16: forward (168
// MB) 30 us, 5.5 TB/s; back (252 MB) 50 us, 5.0 TB/s, and 5 us for the weights'
// sums.  A single token 3.6 us, its loads' and the launch's latency.
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_DIM = 512;
constexpr int TOKENS = 4;      // tokens of a workgroup when there are many
// Workgroups that share out the tokens of a backward pass: four a CU, whose sums
// of the weights' gradients are then 2 MB.
constexpr int BACK_GROUPS = 1024;
// At most, one way and the other, of a launch, which has fewer than 2^32 threads; they take turns beyond.
constexpr int64_t MOST_GROUPS = 1 << 22, MOST_HEAD_GROUPS = 1 << 15;

struct Tensor {
  const void* x;
  void* y;        // or NULL
  const void* g;  // backward: the result's gradient
  int64_t sb, st, sh, gb, gt, gh;
  const void* w;
};

struct Args {
  Tensor q, k;
  const void* pos;
  int64_t pos_sb, pos_st;
  const double* turns;
  int64_t tokens, rows;
  FastDiv heads_div;
  double* part;  // backward: [workgroups, 2, dim] sums of the weights' gradients, or NULL
  int nq, nk, dim, rotary, units, lanes, pos64, w32;
  float factor, eps;
};

template <typename T, int VEC>
VH_DEV void load(const void* p, int64_t at, float* x) {
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
VH_DEV void store(void* p, int64_t at, const float* x) {
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

// The pairs of a unit's 2 * VEC values turned: the first and second values of
// a pair are z[j] and z[VEC + j], or side by side.
template <int VEC, bool INTERLEAVED>
VH_DEV void turn(float* z, const float2* cs, float sign) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float& a = z[INTERLEAVED ? 2 * j : j];
    float& b = z[INTERLEAVED ? 2 * j + 1 : VEC + j];
    const float c = cs[j].x, s = cs[j].y * sign, x0 = a, x1 = b;
    a = x0 * c - x1 * s;
    b = x1 * c + x0 * s;
  }
}

VH_DEV float sum_lanes(float v, int lanes) {
  for (int d = 1; d < lanes; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// A unit is 2 * VEC values of a head, as vh_rope has them; a lane holds UN.
template <typename T, int VEC, int UN, bool INTERLEAVED, int TOK, bool BACK>
__global__ void __launch_bounds__(THREADS) k_norm_rope(Args a) {
  __shared__ float2 s_cs[TOK * (MAX_DIM / 2)];
  __shared__ float s_w[2][MAX_DIM];
  constexpr int V = 2 * VEC * UN;
  float sum[BACK ? 2 : 1][V];  // of the weights' gradients, queries' and keys'
  if constexpr (BACK) {
#pragma unroll
    for (int i = 0; i < V; ++i) sum[0][i] = sum[1][i] = 0.0f;
  }
  const int half = a.rotary / 2, heads = a.nq + a.nk;
  const int lane = threadIdx.x % a.lanes, lane_head = threadIdx.x / a.lanes, per = THREADS / a.lanes;
  for (int i = threadIdx.x; i < 2 * a.dim; i += THREADS) {
    const int key = i >= a.dim, c = i - key * a.dim;
    const void* w = key ? a.k.w : a.q.w;
    s_w[key][c] = a.w32 ? ((const float*)w)[c] : (float)((const T*)w)[c];
  }
  for (int64_t row0 = (int64_t)blockIdx.x * TOK; row0 < a.rows; row0 += (int64_t)gridDim.x * TOK) {
    const int rows = (int)(a.rows - row0 < TOK ? a.rows - row0 : TOK);
    __syncthreads();  // the last tokens' angles are read
    for (int i = threadIdx.x; i < rows * half; i += THREADS) {
      const int t = i / half, j = i - t * half;
      const int64_t b = (row0 + t) / a.tokens, n = (row0 + t) - b * a.tokens;
      const int64_t at = b * a.pos_sb + n * a.pos_st;
      const int64_t p = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
      const double turns = (double)p * a.turns[j];
      if constexpr (sizeof(T) == 4) {
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        s_cs[t * half + j] = make_float2((float)(c * a.factor), (float)(s * a.factor));
      } else {
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        s_cs[t * half + j] = make_float2(c * a.factor, s * a.factor);
      }
    }
    __syncthreads();
    const int step = per * gridDim.y;
    for (int i = lane_head + per * blockIdx.y; i < rows * heads; i += step) {
      const int t = TOK == 1 ? 0 : (int)fast_div((uint32_t)i, a.heads_div);
      const int h = i - t * heads;
      const int64_t row = row0 + t, b = row / a.tokens, n = row - b * a.tokens;
      const bool key = h >= a.nq;
      const int hh = key ? h - a.nq : h;
      const Tensor& in = key ? a.k : a.q;
      const int64_t x_at = b * in.sb + n * in.st + hh * in.sh;
      const int64_t out = (row * (key ? a.nk : a.nq) + hh) * a.dim;
      const float* w = s_w[key];
      float x[V], g[BACK ? V : 1];
      float squares = 0.0f;
#pragma unroll
      for (int n2 = 0; n2 < UN; ++n2) {
        const int u = lane + n2 * a.lanes;
        float* z = x + n2 * 2 * VEC;
        if (u < a.units) {
          const bool turned = u * 2 * VEC < a.rotary;
          const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
          const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
          load<T, VEC>(in.x, x_at + c0, z);
          load<T, VEC>(in.x, x_at + c1, z + VEC);
          if constexpr (BACK) {
            const int64_t g_at = b * in.gb + n * in.gt + hh * in.gh;
            load<T, VEC>(in.g, g_at + c0, g + n2 * 2 * VEC);
            load<T, VEC>(in.g, g_at + c1, g + n2 * 2 * VEC + VEC);
          }
#pragma unroll
          for (int j = 0; j < 2 * VEC; ++j) squares += z[j] * z[j];
        }
      }
      squares = sum_lanes(squares, a.lanes);
      const float r = 1.0f / sqrtf(squares / (float)a.dim + a.eps);
      if constexpr (!BACK) {
#pragma unroll
        for (int n2 = 0; n2 < UN; ++n2) {
          const int u = lane + n2 * a.lanes;
          float* z = x + n2 * 2 * VEC;
          if (u < a.units) {
            const bool turned = u * 2 * VEC < a.rotary;
            const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
            const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              z[j] *= r * w[c0 + j];
              z[VEC + j] *= r * w[c1 + j];
            }
            if (turned) turn<VEC, INTERLEAVED>(z, s_cs + t * half + u * VEC, 1.0f);
            store<T, VEC>(in.y, out + c0, z);
            store<T, VEC>(in.y, out + c1, z + VEC);
          }
        }
      } else {
        float dot = 0.0f;  // b . x r
#pragma unroll
        for (int n2 = 0; n2 < UN; ++n2) {
          const int u = lane + n2 * a.lanes;
          float *z = x + n2 * 2 * VEC, *gz = g + n2 * 2 * VEC;
          if (u < a.units) {
            const bool turned = u * 2 * VEC < a.rotary;
            const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
            const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
            if (turned) turn<VEC, INTERLEAVED>(gz, s_cs + t * half + u * VEC, -1.0f);
#pragma unroll
            for (int j = 0; j < 2 * VEC; ++j) {
              z[j] *= r;
              const float d = gz[j] * z[j];
              if (key) sum[1][n2 * 2 * VEC + j] += d;
              else sum[0][n2 * 2 * VEC + j] += d;
              gz[j] *= w[(j < VEC ? c0 : c1 - VEC) + j];
              dot += gz[j] * z[j];
            }
          }
        }
        dot = sum_lanes(dot, a.lanes) / (float)a.dim;
        if (in.y) {
#pragma unroll
          for (int n2 = 0; n2 < UN; ++n2) {
            const int u = lane + n2 * a.lanes;
            float *z = x + n2 * 2 * VEC, *gz = g + n2 * 2 * VEC;
            if (u < a.units) {
              const bool turned = u * 2 * VEC < a.rotary;
              const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
              const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
#pragma unroll
              for (int j = 0; j < 2 * VEC; ++j) gz[j] = r * (gz[j] - z[j] * dot);
              store<T, VEC>(in.y, out + c0, gz);
              store<T, VEC>(in.y, out + c1, gz + VEC);
            }
          }
        }
      }
    }
  }
  if constexpr (BACK) {
    if (!a.part) return;
    // [per, dim] of one tensor at a time: 256 threads hold V values each
    __shared__ float s_sum[THREADS * V];
    double* to = a.part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.dim;
#pragma unroll
    for (int key = 0; key < 2; ++key) {
      __syncthreads();
#pragma unroll
      for (int n2 = 0; n2 < UN; ++n2) {
        const int u = lane + n2 * a.lanes;
        if (u < a.units) {
          const bool turned = u * 2 * VEC < a.rotary;
          const int c0 = !turned || INTERLEAVED ? u * 2 * VEC : u * VEC;
          const int c1 = !turned || INTERLEAVED ? c0 + VEC : c0 + half;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            s_sum[lane_head * a.dim + c0 + j] = sum[key][n2 * 2 * VEC + j];
            s_sum[lane_head * a.dim + c1 + j] = sum[key][n2 * 2 * VEC + VEC + j];
          }
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.dim; c += THREADS) {
        double all = 0.0;
        for (int p = 0; p < per; ++p) all += (double)s_sum[p * a.dim + c];
        to[key * a.dim + c] = all;
      }
    }
  }
}

// The workgroups' sums joined: 16 columns a workgroup, 16 threads a column.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_weights(const double* part, int parts, int dim, T* gq, T* gk) {
  __shared__ double s_sum[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  double sum = 0.0;
  if (col < 2 * dim) {
#pragma unroll 8
    for (int p = r; p < parts; p += 16) sum += part[(int64_t)p * 2 * dim + col];
  }
  s_sum[r][c] = sum;
  __syncthreads();
  if (r > 0 || col >= 2 * dim) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += s_sum[i][c];
  T* to = col < dim ? gq : gk;
  if (to) to[col < dim ? col : col - dim] = (T)(float)sum;
}

struct Plan {
  dim3 grid;
  bool many;
  int units, lanes;
  bool wide;
};

bool aligned(const void* p, int64_t sb, int64_t st, int64_t sh, int vec) {
  return (uintptr_t)p % 16 == 0 && sb % vec == 0 && st % vec == 0 && sh % vec == 0;
}

Plan plan_of(const vh_norm_rope_desc* d, bool back) {
  Plan p;
  const vh_rope_desc& r = d->rope;
  const int vec = r.dtype == VH_F32 ? 4 : 8;
  p.wide = r.dim % (2 * vec) == 0 && r.rotary % (2 * vec) == 0;
  if (r.heads) p.wide = p.wide && aligned(r.q, r.q_sb, r.q_st, r.q_sh, vec) && (uintptr_t)r.q_out % 16 == 0 &&
                        (!back || aligned(d->gq, d->gq_sb, d->gq_st, d->gq_sh, vec));
  if (r.kv_heads) p.wide = p.wide && aligned(r.k, r.k_sb, r.k_st, r.k_sh, vec) && (uintptr_t)r.k_out % 16 == 0 &&
                           (!back || aligned(d->gk, d->gk_sb, d->gk_st, d->gk_sh, vec));
  p.units = r.dim / (p.wide ? 2 * vec : 2);
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 64) p.lanes *= 2;
  const int64_t rows = r.batch * r.tokens;
  const int heads = r.heads + r.kv_heads, per = THREADS / p.lanes;
  p.many = rows >= 2048;  // as vh_rope, where both sides' times are
  int64_t x = p.many ? (rows + TOKENS - 1) / TOKENS : rows;
  int64_t y = p.many ? 1 : (heads + per - 1) / per;
  if (back && x * y > BACK_GROUPS) {
    y = y < BACK_GROUPS ? y : BACK_GROUPS;
    x = BACK_GROUPS / y;
  } else if (x * y > MOST_GROUPS || y > MOST_HEAD_GROUPS) {
    y = y < MOST_HEAD_GROUPS ? y : MOST_HEAD_GROUPS;
    x = x < MOST_GROUPS / y ? x : MOST_GROUPS / y;
  }
  p.grid = dim3((unsigned)x, (unsigned)y);
  return p;
}

template <typename T, int VEC, int UN, bool BACK>
void launch(const Args& a, const Plan& p, bool interleaved, hipStream_t s) {
  if (p.many) {
    if (interleaved) hipLaunchKernelGGL((k_norm_rope<T, VEC, UN, true, TOKENS, BACK>), p.grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_norm_rope<T, VEC, UN, false, TOKENS, BACK>), p.grid, dim3(THREADS), 0, s, a);
  } else {
    if (interleaved) hipLaunchKernelGGL((k_norm_rope<T, VEC, UN, true, 1, BACK>), p.grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((k_norm_rope<T, VEC, UN, false, 1, BACK>), p.grid, dim3(THREADS), 0, s, a);
  }
}

template <typename T, bool BACK>
void dispatch(const Args& a, const Plan& p, bool interleaved, hipStream_t s) {
  if (p.wide) launch<T, 16 / sizeof(T), 1, BACK>(a, p, interleaved, s);
  else launch<T, 1, 4, BACK>(a, p, interleaved, s);
}

int check(const vh_norm_rope_desc* d, const char* what) {
  VH_REQUIRE(d, "%s: null descriptor", what);
  const vh_rope_desc& r = d->rope;
  VH_REQUIRE(vh::is_float_dtype(r.dtype), "%s: dtype must be bfloat16, float16 or float32", what);
  VH_REQUIRE(d->weight_dtype == VH_F32 || d->weight_dtype == r.dtype, "%s: weights of float32 or the values' dtype", what);
  VH_REQUIRE(r.batch >= 0 && r.tokens >= 0 && r.heads >= 0 && r.kv_heads >= 0, "%s: negative size", what);
  VH_REQUIRE(r.dim > 0 && r.dim <= MAX_DIM && r.dim % 2 == 0, "%s: dim must be even and at most %d (got %d)", what, MAX_DIM, r.dim);
  VH_REQUIRE(r.rotary > 0 && r.rotary <= r.dim && r.rotary % 2 == 0, "%s: the rotated part must be even and at most dim", what);
  VH_REQUIRE(r.pos_bits == 32 || r.pos_bits == 64, "%s: positions of 32 or 64 bits", what);
  VH_REQUIRE(d->eps > 0.0f && d->eps < __builtin_inff(), "%s: eps must be positive", what);
  VH_REQUIRE(r.batch < (1ll << 31) && r.tokens < (1ll << 31) && r.batch * r.tokens < (1ll << 31) &&
                 (int64_t)r.heads + r.kv_heads < (1 << 20),
             "%s: too many rows or heads", what);
  return VH_OK;
}

bool nothing(const vh_rope_desc& r) { return r.batch * r.tokens == 0 || r.heads + r.kv_heads == 0; }

Args args_of(const vh_norm_rope_desc* d, const Plan& p) {
  const vh_rope_desc& r = d->rope;
  const Tensor q{r.q, r.q_out, d->gq, r.q_sb, r.q_st, r.q_sh, d->gq_sb, d->gq_st, d->gq_sh, d->q_weight};
  const Tensor k{r.k, r.k_out, d->gk, r.k_sb, r.k_st, r.k_sh, d->gk_sb, d->gk_st, d->gk_sh, d->k_weight};
  // a tensor without heads is never read, but for its weights: the other one's stand for it
  return Args{r.heads ? q : k, r.kv_heads ? k : q, r.pos, r.pos_sb, r.pos_st, r.turns, r.tokens, r.batch * r.tokens,
              make_fast_div((uint32_t)(r.heads + r.kv_heads)), nullptr, r.heads, r.kv_heads, r.dim, r.rotary, p.units,
              p.lanes, r.pos_bits == 64, d->weight_dtype == VH_F32, r.factor, d->eps};
}

}  // namespace

extern "C" int vh_norm_rope(const vh_norm_rope_desc* d, vh_stream_t stream) {
  if (int e = check(d, "vh_norm_rope")) return e;
  const vh_rope_desc& r = d->rope;
  if (nothing(r)) return VH_OK;
  VH_REQUIRE((r.heads == 0 || (r.q && r.q_out && d->q_weight)) && (r.kv_heads == 0 || (r.k && r.k_out && d->k_weight)) &&
                 r.pos && r.turns,
             "vh_norm_rope: null argument");
  const Plan p = plan_of(d, false);
  const Args a = args_of(d, p);
  hipStream_t s = vh::as_stream(stream);
  if (r.dtype == VH_BF16) dispatch<__bf16, false>(a, p, r.interleaved != 0, s);
  else if (r.dtype == VH_F16) dispatch<_Float16, false>(a, p, r.interleaved != 0, s);
  else dispatch<float, false>(a, p, r.interleaved != 0, s);
  return vh::check_launch("vh_norm_rope");
}

extern "C" int64_t vh_norm_rope_workspace_bytes(const vh_norm_rope_desc* d) {
  if (check(d, "vh_norm_rope_workspace_bytes")) return -1;
  if (nothing(d->rope)) return 0;
  return (int64_t)BACK_GROUPS * 2 * d->rope.dim * (int64_t)sizeof(double);
}

extern "C" int vh_norm_rope_backward(const vh_norm_rope_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  if (int e = check(d, "vh_norm_rope_backward")) return e;
  const vh_rope_desc& r = d->rope;
  if (nothing(r)) return VH_OK;
  VH_REQUIRE((r.heads == 0 || (r.q && d->gq && d->q_weight)) && (r.kv_heads == 0 || (r.k && d->gk && d->k_weight)) && r.pos &&
                 r.turns,
             "vh_norm_rope_backward: null argument");
  const bool weights = d->gq_weight || d->gk_weight;
  const int64_t need = (int64_t)BACK_GROUPS * 2 * r.dim * (int64_t)sizeof(double);
  VH_REQUIRE(!weights || (work && work_bytes >= need && (uintptr_t)work % 16 == 0),
             "vh_norm_rope_backward: needs %lld bytes of aligned workspace", (long long)need);
  const Plan p = plan_of(d, true);
  Args a = args_of(d, p);
  a.part = weights ? (double*)work : nullptr;
  hipStream_t s = vh::as_stream(stream);
  if (r.dtype == VH_BF16) dispatch<__bf16, true>(a, p, r.interleaved != 0, s);
  else if (r.dtype == VH_F16) dispatch<_Float16, true>(a, p, r.interleaved != 0, s);
  else dispatch<float, true>(a, p, r.interleaved != 0, s);
  if (weights) {
    const dim3 grid((unsigned)((2 * r.dim + 15) / 16));
    const int parts = (int)(p.grid.x * p.grid.y);
    void *gq = r.heads ? d->gq_weight : nullptr, *gk = r.kv_heads ? d->gk_weight : nullptr;
    if (d->weight_dtype == VH_F32) hipLaunchKernelGGL(k_norm_weights<float>, grid, dim3(256), 0, s, a.part, parts, r.dim, (float*)gq, (float*)gk);
    else if (d->weight_dtype == VH_BF16) hipLaunchKernelGGL(k_norm_weights<__bf16>, grid, dim3(256), 0, s, a.part, parts, r.dim, (__bf16*)gq, (__bf16*)gk);
    else hipLaunchKernelGGL(k_norm_weights<_Float16>, grid, dim3(256), 0, s, a.part, parts, r.dim, (_Float16*)gq, (_Float16*)gk);
  }
  return vh::check_launch("vh_norm_rope_backward");
}
