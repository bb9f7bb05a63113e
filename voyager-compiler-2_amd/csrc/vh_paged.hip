// A cache of keys and values in pages: rows quantized as they are written
// (one float32 scale a row of a head), read back, and moved.
//
//   scale = amax / most,  code = round(x * (most / amax)),  x' = code * scale
//
// with most 448 (E4M3, rounded by the hardware converter, half to even) or
// 127 (int8), amax at least 2^-100, and every quotient and product rounded to
// float32 once.  A row that holds an infinity or NaN gets the scale NaN, so it
// reads back as NaN everywhere and no code has to stand for it.
//
// Bound by memory: a value is read once in 16 bits and written once in 8, or
// the reverse.  8 heads of 128, E4M3, 32768 tokens in a shuffled order of
// slots: written in 42-43 us (204 MB, 4.8 TB/s), read back in 30.7 (204 MB,
// the codes still in the last cache); 4001 tokens, int8, 8.0 and 6.0 us
// (25 MB each); 8 tokens 3.2 and 3.0 us, one load's and one store's latency.
// Held in 16 bits: 32768 tokens 40.7 and 41.3 us (268 MB each way, 6.5 TB/s with
// part of it in the last cache), 4001 tokens 5.4 and 5.8, 8 tokens 2.4.
#include <hip/hip_runtime.h>

#include "vh_device.h"
#include "vh_host.h"
#include "vh_paged.h"

namespace {

constexpr int PAGED_THREADS = 256;
constexpr float AMAX_LEAST = 0x1p-100f;

struct PagedArgs {
  vh_cache c;
  const void *k, *v;   // write: the input rows
  void *k_out, *v_out; // read: the output rows
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t* slots;
  int64_t n;
  FastDiv page_div;
  int chunks;  // of 8 values a row
};

// Where slot `s` of head `h` begins, in rows of the cache.
VH_DEV int64_t paged_row(const PagedArgs& a, int64_t s, int h) {
  const uint32_t page = fast_div((uint32_t)s, a.page_div);
  return ((int64_t)page * a.c.kv_heads + h) * a.c.page + ((uint32_t)s - page * (uint32_t)a.c.page);
}

// Eight values of a row; wide where 16-byte accesses are aligned.
template <typename T, bool WIDE>
VH_DEV void load8(const void* p, int64_t at, float (&x)[8]) {
  T e[8];
  if constexpr (WIDE) {
    const uint4 v = *(const uint4*)((const T*)p + at);
    __builtin_memcpy(e, &v, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = ((const T*)p)[at + i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)e[i];
}

template <typename T>
VH_DEV void store8(void* p, int64_t at, const float (&x)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = (T)x[i];
  uint4 v;
  __builtin_memcpy(&v, e, 16);
  *(uint4*)((T*)p + at) = v;
}

// The codes of eight values, and their row's scale.  `group` lanes hold a row.
template <int FMT>
VH_DEV uint2 paged_encode(const float (&x)[8], int group, float& scale) {
  uint32_t key = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) key = umax32(key, amax_key(x[i]));
  key = group_umax_rt(key, group);
  const bool bad = key >= 0x7f800000u;
  const float amax = fmaxf(__uint_as_float(key), AMAX_LEAST);
  const float most = FMT == CACHE_E4M3 ? 448.0f : 127.0f;
  const float inv = most / amax;
  scale = bad ? __builtin_nanf("") : amax / most;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = bad ? 0.0f : fminf(fmaxf(x[i] * inv, -most), most);
    const uint32_t b = FMT == CACHE_E4M3 ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu
                                         : (uint32_t)((int)rintf(y) + 128);
    w[i >> 2] |= b << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

template <int FMT>
VH_DEV void paged_decode(uint2 c, float scale, float (&x)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = (w[i >> 2] >> (8 * (i & 3))) & 0xffu;
    x[i] = (FMT == CACHE_E4M3 ? __builtin_amdgcn_cvt_f32_fp8((int)b, 0) : (float)((int)b - 128)) * scale;
  }
}

// A workgroup takes consecutive tokens of one head; `group` lanes a token (a
// power of two, so that a row's maximum stays inside it), 8 values a lane, its
// key and its value.  Heads are the fastest index of the grid: the rows of a
// token are read by workgroups that run together.  A lane reads 16 bytes and
// writes 8, so a wave covers whole rows on both sides, and the row's maximum is
// a few exchanges between neighbours, without LDS.
template <typename T, int FMT, bool WIDE>
__global__ void __launch_bounds__(PAGED_THREADS) k_paged_write(PagedArgs a, int group) {
  const int h = blockIdx.x % a.c.kv_heads;
  const int64_t tok = (int64_t)(blockIdx.x / a.c.kv_heads) * (PAGED_THREADS / group) + threadIdx.x / group;
  const int chunk = threadIdx.x % group;
  const bool in = tok < a.n && chunk < a.chunks;
  float k[8] = {}, v[8] = {};
  int64_t slot = -1;
  if (in) {
    slot = a.slots[tok];
    load8<T, WIDE>(a.k, tok * a.k_st + h * a.k_sh + chunk * 8, k);
    load8<T, WIDE>(a.v, tok * a.v_st + h * a.v_sh + chunk * 8, v);
  }
  if (slot >= a.c.slots) {
    atomicOr(a.c.flag, VH_CACHE_ERR_SLOT);
    slot = -1;
  }
  if constexpr (FMT == CACHE_F16 || FMT == CACHE_BF16) {
    if (slot < 0) return;
    const int64_t at = paged_row(a, slot, h) * a.c.dim + chunk * 8;
    store8<T>(a.c.k, at, k);
    store8<T>(a.c.v, at, v);
  } else {
    float ks, vs;
    const uint2 kc = paged_encode<FMT>(k, group, ks), vc = paged_encode<FMT>(v, group, vs);
    if (slot < 0) return;
    const int64_t row = paged_row(a, slot, h);
    *(uint2*)((uint8_t*)a.c.k + row * a.c.dim + chunk * 8) = kc;
    *(uint2*)((uint8_t*)a.c.v + row * a.c.dim + chunk * 8) = vc;
    if (chunk == 0) {
      a.c.k_scale[row] = ks;
      a.c.v_scale[row] = vs;
    }
  }
}

// The reverse; tokens without a slot read as zeros.
template <typename T, int FMT>
__global__ void __launch_bounds__(PAGED_THREADS) k_paged_read(PagedArgs a, int group) {
  const int h = blockIdx.x % a.c.kv_heads;
  const int64_t tok = (int64_t)(blockIdx.x / a.c.kv_heads) * (PAGED_THREADS / group) + threadIdx.x / group;
  const int chunk = threadIdx.x % group;
  if (tok >= a.n || chunk >= a.chunks) return;
  int64_t slot = a.slots[tok];
  if (slot >= a.c.slots) {
    atomicOr(a.c.flag, VH_CACHE_ERR_SLOT);
    slot = -1;
  }
  float k[8] = {}, v[8] = {};
  if (slot >= 0) {
    const int64_t row = paged_row(a, slot, h), at = row * a.c.dim + chunk * 8;
    if constexpr (FMT == CACHE_F16 || FMT == CACHE_BF16) {
      load8<T, true>(a.c.k, at, k);
      load8<T, true>(a.c.v, at, v);
    } else {
      paged_decode<FMT>(*(const uint2*)((const uint8_t*)a.c.k + at), a.c.k_scale[row], k);
      paged_decode<FMT>(*(const uint2*)((const uint8_t*)a.c.v + at), a.c.v_scale[row], v);
    }
  }
  const int64_t out = (tok * a.c.kv_heads + h) * a.c.dim + chunk * 8;
  store8<T>(a.k_out, out, k);
  store8<T>(a.v_out, out, v);
}

// Moves the rows of the kept nodes of each sequence, path[1], path[2], ... of
// the tree at the sequence's end, to the positions 1, 2, ... there.  A path
// rises, so path[i] >= i: a row is only ever written over rows already moved
// or not kept.  Each thread owns one 8-byte column of a head's rows (or the
// scales) and moves it node by node in order, so nothing else orders the
// moves.  One workgroup per sequence and head.
//
// Bound by latency: path, table and row are three trips in a row for each node.
// 32 sequences, 8 E4M3 heads of 128: 4.7 us with 4 nodes kept (0.4 MB), 11.8 with
// 12; 8 sequences with 20 kept 18.9; one sequence with 4 3.5.
struct KeepArgs {
  vh_cache c;
  const int32_t *table, *context, *path, *count;
  int64_t table_st, path_st;
  int nodes, table_pages;
};

VH_DEV int64_t keep_row(const KeepArgs& a, const int32_t* table, int64_t pos, int h) {
  const int64_t e = pos / a.c.page;
  if (pos < 0 || e >= a.table_pages) return -1;
  const int page = table[e];
  if (page < 0 || page >= a.c.pages) return -1;
  return ((int64_t)page * a.c.kv_heads + h) * a.c.page + pos % a.c.page;
}

__global__ void __launch_bounds__(PAGED_THREADS) k_paged_keep(KeepArgs a) {
  const int h = blockIdx.x;
  const int64_t b = blockIdx.y;
  const int bytes = a.c.fmt == CACHE_E4M3 || a.c.fmt == CACHE_INT8 ? 1 : 2;
  const int cols = a.c.dim * bytes / 8;
  const int32_t* table = a.table + b * a.table_st;
  const int32_t* path = a.path + b * a.path_st;
  const int64_t ctx = a.context[b];
  const int count = a.count[b] < a.nodes ? a.count[b] : a.nodes;
  int last = 0;
  for (int i = 1; i < count; ++i) {
    const int node = path[i];
    const int64_t from = node > last && node < a.nodes ? keep_row(a, table, ctx + node, h) : -1;
    const int64_t to = keep_row(a, table, ctx + i, h);
    if (from < 0 || to < 0) {
      if (threadIdx.x == 0) atomicOr(a.c.flag, VH_CACHE_ERR_PAGE);
      return;
    }
    last = node;
    if (node == i) continue;
    for (int c = threadIdx.x; c < 2 * cols; c += PAGED_THREADS) {
      uint2* base = (uint2*)(c < cols ? a.c.k : a.c.v);
      const int col = c < cols ? c : c - cols;
      base[to * cols + col] = base[from * cols + col];
    }
    if (bytes == 1 && threadIdx.x < 2) {
      float* s = threadIdx.x ? a.c.v_scale : a.c.k_scale;
      s[to] = s[from];
    }
  }
}

int group_of(int chunks) {
  int g = 1;
  while (g < chunks) g *= 2;
  return g;
}

template <typename T, int FMT>
void paged_write(const PagedArgs& a, int group, dim3 grid, bool wide, hipStream_t s) {
  if (wide) hipLaunchKernelGGL((k_paged_write<T, FMT, true>), grid, dim3(PAGED_THREADS), 0, s, a, group);
  else hipLaunchKernelGGL((k_paged_write<T, FMT, false>), grid, dim3(PAGED_THREADS), 0, s, a, group);
}

// Calls f with the kernel's value type and format.
template <typename F>
void paged_types(int fmt, int dtype, F f) {
  if (fmt == CACHE_E4M3) {
    if (dtype == VH_BF16) f(__bf16(), std::integral_constant<int, CACHE_E4M3>());
    else f(_Float16(), std::integral_constant<int, CACHE_E4M3>());
  } else if (fmt == CACHE_INT8) {
    if (dtype == VH_BF16) f(__bf16(), std::integral_constant<int, CACHE_INT8>());
    else f(_Float16(), std::integral_constant<int, CACHE_INT8>());
  } else if (fmt == CACHE_F16) {
    f(_Float16(), std::integral_constant<int, CACHE_F16>());
  } else {
    f(__bf16(), std::integral_constant<int, CACHE_BF16>());
  }
}

int paged_dtype_check(const vh_cache* c, int dtype, const char* what) {
  VH_REQUIRE(dtype == VH_BF16 || dtype == VH_F16, "%s: dtype must be bfloat16 or float16", what);
  VH_REQUIRE(c->fmt != CACHE_F16 || dtype == VH_F16, "%s: a float16 cache holds float16 rows", what);
  VH_REQUIRE(c->fmt != CACHE_BF16 || dtype == VH_BF16, "%s: a bfloat16 cache holds bfloat16 rows", what);
  return VH_OK;
}

}  // namespace

int vh_cache_check(const vh_cache* c, const char* what) {
  VH_REQUIRE(c, "%s: null cache", what);
  VH_REQUIRE(c->fmt >= CACHE_E4M3 && c->fmt <= CACHE_BF16, "%s: unknown cache format %d", what, c->fmt);
  VH_REQUIRE(c->k && c->v && c->flag, "%s: null cache buffer", what);
  VH_REQUIRE(c->fmt == CACHE_F16 || c->fmt == CACHE_BF16 || (c->k_scale && c->v_scale), "%s: null cache scales", what);
  VH_REQUIRE((uintptr_t)c->k % 16 == 0 && (uintptr_t)c->v % 16 == 0, "%s: misaligned cache", what);
  VH_REQUIRE(c->pages > 0 && c->page > 0 && c->kv_heads > 0, "%s: empty cache", what);
  VH_REQUIRE(c->dim > 0 && c->dim % 8 == 0 && c->dim <= 512, "%s: a cache's dim must be a multiple of 8, at most 512", what);
  VH_REQUIRE(c->slots == c->pages * c->page && c->slots < (1ll << 31), "%s: a cache of fewer than 2^31 slots", what);
  VH_REQUIRE(c->kv_heads < (1 << 16), "%s: too many heads", what);
  return VH_OK;
}

extern "C" int vh_paged_write(const vh_cache* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                              int64_t v_sh, int32_t dtype, const int64_t* slots, int64_t n, vh_stream_t stream) {
  if (int e = vh_cache_check(cache, "vh_paged_write")) return e;
  if (int e = paged_dtype_check(cache, dtype, "vh_paged_write")) return e;
  VH_REQUIRE(n >= 0 && n < (1ll << 31), "vh_paged_write: bad number of tokens");
  if (n == 0) return VH_OK;
  VH_REQUIRE(k && v && slots, "vh_paged_write: null argument");
  PagedArgs a{*cache, k, v, nullptr, nullptr, k_st, k_sh, v_st, v_sh, slots, n, make_fast_div((uint32_t)cache->page),
              cache->dim / 8};
  const int group = group_of(a.chunks), per = PAGED_THREADS / group;
  const int64_t blocks = (n + per - 1) / per * cache->kv_heads;
  VH_REQUIRE(blocks < (1ll << 31), "vh_paged_write: too many rows");
  const bool wide = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 &&
                    v_sh % 8 == 0;
  paged_types(cache->fmt, dtype, [&](auto t, auto f) {
    paged_write<decltype(t), decltype(f)::value>(a, group, dim3((unsigned)blocks), wide, vh::as_stream(stream));
  });
  return vh::check_launch("vh_paged_write");
}

extern "C" int vh_paged_read(const vh_cache* cache, void* k, void* v, int32_t dtype, const int64_t* slots, int64_t n,
                             vh_stream_t stream) {
  if (int e = vh_cache_check(cache, "vh_paged_read")) return e;
  if (int e = paged_dtype_check(cache, dtype, "vh_paged_read")) return e;
  VH_REQUIRE(n >= 0 && n < (1ll << 31), "vh_paged_read: bad number of tokens");
  if (n == 0) return VH_OK;
  VH_REQUIRE(k && v && slots, "vh_paged_read: null argument");
  VH_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "vh_paged_read: misaligned output");
  PagedArgs a{*cache, nullptr, nullptr, k, v, 0, 0, 0, 0, slots, n, make_fast_div((uint32_t)cache->page), cache->dim / 8};
  const int group = group_of(a.chunks), per = PAGED_THREADS / group;
  const int64_t blocks = (n + per - 1) / per * cache->kv_heads;
  VH_REQUIRE(blocks < (1ll << 31), "vh_paged_read: too many rows");
  paged_types(cache->fmt, dtype, [&](auto t, auto f) {
    hipLaunchKernelGGL((k_paged_read<decltype(t), decltype(f)::value>), dim3((unsigned)blocks), dim3(PAGED_THREADS), 0,
                       vh::as_stream(stream), a, group);
  });
  return vh::check_launch("vh_paged_read");
}

extern "C" int vh_paged_keep(const vh_cache* cache, const int32_t* table, int64_t table_st, int32_t table_pages,
                             const int32_t* context, const int32_t* path, int64_t path_st, const int32_t* count,
                             int64_t batch, int32_t nodes, vh_stream_t stream) {
  if (int e = vh_cache_check(cache, "vh_paged_keep")) return e;
  VH_REQUIRE(batch >= 0 && batch < 65536 && nodes >= 0 && table_pages >= 0, "vh_paged_keep: bad size");
  if (batch == 0 || nodes < 2) return VH_OK;
  VH_REQUIRE(table && context && path && count, "vh_paged_keep: null argument");
  KeepArgs a{*cache, table, context, path, count, table_st, path_st, nodes, table_pages};
  hipLaunchKernelGGL(k_paged_keep, dim3((unsigned)cache->kv_heads, (unsigned)batch), dim3(PAGED_THREADS), 0,
                     vh::as_stream(stream), a);
  return vh::check_launch("vh_paged_keep");
}
