// Trees of tokens: the ancestors of their nodes, and the entry point of their
// attention, with the kernel that joins its splits.
#include "vh_tree_attention.h"

namespace tree {
template <>
int launch<64>(const Args& a, bool wide, int n, hipStream_t s);
template <>
int launch<128>(const Args& a, bool wide, int n, hipStream_t s);
template <>
int launch<256>(const Args& a, bool wide, int n, hipStream_t s);
}  // namespace tree

namespace {

using tree::Args;
using tree::f32x4;

constexpr int MASK_THREADS = 256;
constexpr int MAX_NODES = VH_TREE_MAX_NODES;

// One workgroup a tree, one thread a word of a node's mask: it walks up from
// the node and sets the bits that fall into its word.  Parents come before
// their children, so every step goes down in number and the walk ends.
__global__ void __launch_bounds__(MASK_THREADS) k_tree_masks(const int32_t* parents, int nodes, int words, uint64_t* masks,
                                                             int32_t* flag) {
  __shared__ int32_t s_parent[MAX_NODES];
  const int32_t* p = parents + (int64_t)blockIdx.x * nodes;
  uint64_t* out = masks + (int64_t)blockIdx.x * nodes * words;
  for (int n = threadIdx.x; n < nodes; n += MASK_THREADS) s_parent[n] = p[n];
  __syncthreads();
  bool bad = s_parent[0] >= 0;
  for (int i = threadIdx.x; i < nodes * words; i += MASK_THREADS) {
    const int w = i % words;
    uint64_t mask = 0ull;
    int n = i / words;
    while (n > 0) {
      if (n >> 6 == w) mask |= 1ull << (n & 63);
      const int up = s_parent[n];
      bad |= up >= n;
      n = up < n ? up : -1;
    }
    if (n == 0 && w == 0) mask |= 1ull;
    out[i] = n == 0 ? mask : 0ull;  // a node that pads, or under one that does
  }
  if (bad) atomicOr(flag, VH_CACHE_ERR_PARENT);
}

// The number of a sequence's splits and of those before them.  Every lane of
// a wave calls it together, each with a sequence of its own.
struct Splits {
  uint32_t before, n;
};
VH_DEV Splits splits_before(const Args& a, int b) {
  Splits s{0u, 1u};
  const uint32_t chunk = tree::chunk_of(a);
  if (a.batch == 1) return Splits{0u, tree::splits_of(tree::pieces(a, 0), chunk)};
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const uint32_t n = b0 + lane < a.batch ? tree::splits_of(tree::pieces(a, b0 + lane), chunk) : 0u;
    uint32_t upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t y = (uint32_t)__shfl_up((int)upto, d);
      upto += lane >= d ? y : 0u;
    }
    const int at = b - b0 < 0 ? 0 : b - b0 > 63 ? 63 : b - b0;
    const uint32_t mine = (uint32_t)__shfl((int)n, at), sum = (uint32_t)__shfl((int)upto, at);
    if (b >= b0 + 64) s.before += sum;
    else if (b >= b0) s = Splits{s.before + sum - mine, mine};
  }
  return s;
}

// The splits of a row joined: D / 4 lanes hold the row's channels, `GROUPS`
// of them take turns along the splits.
template <int D, int GROUPS>
__global__ void __launch_bounds__(256) k_tree_merge(Args a) {
  constexpr int LANES = D / 4, ROWS = 256 / (LANES * GROUPS);
  __shared__ f32x4 s_o[GROUPS > 1 ? 256 : 1];
  __shared__ float2 s_ml[GROUPS > 1 ? GROUPS : 1];
  const int group = GROUPS > 1 ? threadIdx.x / LANES : 0;
  const int64_t id = (int64_t)blockIdx.x * ROWS + (GROUPS > 1 ? 0 : threadIdx.x / LANES);
  const int c = threadIdx.x % LANES * 4;
  const int pairs = a.batch * a.c.kv_heads;
  const bool in = id < (int64_t)pairs * a.rows;  // a wave's lanes go on together: they share out the sequences
  const int pair = in ? (int)(id / a.rows) : 0, row = in ? (int)(id - (int64_t)pair * a.rows) : 0;
  const int b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
  const Splits sp = splits_before(a, b);
  const int splits = (int)sp.n;
  const int64_t step = (int64_t)a.c.kv_heads * a.rows, at = ((int64_t)sp.before * a.c.kv_heads + h) * a.rows + row;
  if (!in) return;
  // splits' sums are under 1 and their results no larger than the largest value:
  // so is what is joined, with the reference this far over the largest one
  const float room = splits > 1 ? (float)(32 - __clz(splits - 1)) : 0.0f;
  float M = -__builtin_inff(), L = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  // four splits at a time, so that their reads overlap
  for (int s0 = group; s0 < splits; s0 += 4 * GROUPS) {
    float2 ml[4];
    f32x4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = s0 + k * GROUPS;
      const int64_t p = at + (s < splits ? s : s0) * step;
      ml[k] = *(const float2*)(a.part_ml + 2 * p);
      x[k] = *(const f32x4*)(a.part_o + p * D + c);
      if (s >= splits) {
        ml[k] = make_float2(-__builtin_inff(), 0.0f);
        x[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    const float to = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)) + room, M);
    const float keep = M == -__builtin_inff() ? 1.0f : tree::exp2_fast(M - to);
    M = to;
    L *= keep;
    o *= keep;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = ml[k].x == -__builtin_inff() ? 1.0f : tree::exp2_fast(ml[k].x - M);
      L += ml[k].y * w;
      o += x[k] * w;
    }
  }
  if constexpr (GROUPS > 1) {
    s_o[threadIdx.x] = o;
    if (c == 0) s_ml[group] = make_float2(M, L);
    __syncthreads();
    if (group > 0) return;
    M = -__builtin_inff();
    L = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) M = fmaxf(M, s_ml[k].x);
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      const float w = s_ml[k].x == -__builtin_inff() ? 1.0f : tree::exp2_fast(s_ml[k].x - M);
      L += s_ml[k].y * w;
      o += s_o[k * LANES + threadIdx.x] * w;
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees nothing is zero
  const int node = (int)fast_div((uint32_t)row, a.group_div);
  const int64_t out = ((int64_t)b * a.nodes + node) * a.heads + h * a.group + row - node * a.group;
  if (a.lse && c == 0) a.lse[out] = L == 0.0f ? -__builtin_inff() : (M + log2f(L)) * tree::LN2;
  o *= inv;
  *(uint2*)((uint16_t*)a.o + out * D + c) =
      a.q_bf16 ? make_uint2(tree::pack2<CACHE_BF16>(o[0], o[1]), tree::pack2<CACHE_BF16>(o[2], o[3]))
               : make_uint2(tree::pack2<CACHE_F16>(o[0], o[1]), tree::pack2<CACHE_F16>(o[2], o[3]));
}

// Many splits a sequence and few rows: a workgroup a row, whose groups share the
// splits.  Else as many rows as fit one: rows alone fill the card then.  (us of
// attention and joining, by the first and the second: 32 rows of 32 splits 10.5
// and 14.2, 512 of 64 24.1 and 27.0, 832 of 32 69 and 68; 4096 of 8 46.8 and
// 39.3, 16384 of 4 or 5 110 and 86.)  Joining these 16384 rows reads 42 MB in
// 10.4 us, the most of it from the last cache.
template <int D>
void merge(const Args& a, hipStream_t s) {
  constexpr int ALL = 1024 / D;  // groups of lanes in a workgroup
  const int64_t rows = (int64_t)a.batch * a.c.kv_heads * a.rows;
  if (a.units >= 8 * (uint32_t)a.batch && rows <= 1024) hipLaunchKernelGGL((k_tree_merge<D, ALL>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_tree_merge<D, 1>), dim3((unsigned)((rows + ALL - 1) / ALL)), dim3(256), 0, s, a);
}

struct Plan {
  bool wide;
  int n, block_rows, row_blocks;  // n: tiles of 16 rows a wave, or waves of rows
  uint32_t share, fill, units;
  int64_t part;  // rows of partial results
};

// The shape of the launch.  Up to 32 rows of a key head (16 of heads of 256)
// a wave holds them all and takes its own keys; more share converted keys.  (us
// by the first and the second, 4 sequences of 8192 over 8 key heads of 128,
// E4M3: 8 rows 22.4 and 34.6, 32 rows 30.6 and 36.4, 40 rows 43.7 and 36.8; 4
// heads of 256: 16 rows 24.3 and 32.8, 32 rows 31.5 and 35.3, but with 16
// sequences 92 and 83, and of 16-bit keys 165 and 114.)
Plan plan_of(const vh_tree_desc* d) {
  Plan p;
  const int64_t rows = (int64_t)d->nodes * (d->heads / d->cache.kv_heads);
  const bool small = d->cache.dim <= 128;
  p.wide = rows > (small ? 32 : 16);
  if (p.wide) {
    p.n = small && rows <= 64 ? 2 : 4;
    p.block_rows = 16 * (small ? 2 : 1) * p.n;
  } else {
    p.n = small && rows > 16 ? 2 : 1;
    p.block_rows = 16 * p.n;
  }
  p.row_blocks = (int)((rows + p.block_rows - 1) / p.block_rows);
  const int64_t keys = (int64_t)d->table_pages * d->cache.page;
  const int64_t most = (keys + tree::PIECE - 1) / tree::PIECE;  // splits of a sequence, a piece each
  const int64_t blocks = (int64_t)d->cache.kv_heads * p.row_blocks;
  // Two workgroups a CU hold their registers where rows are many, and each more
  // share costs its rows' partial results twice; single tokens' keys fill the
  // card best at six, whose results are few.  (8 trees of 64 over 4096: 103 us at
  // 1024, 90 at 512, 101 at 256; 32 tokens over 2048 to 8192: 94 us at 512, 89 at 1536.)
  const int64_t slots = d->workgroups > 0 ? d->workgroups : p.wide ? 512 : 1536;
  int64_t share = slots / blocks;
  if (share < 1) share = 1;
  if (share > most * d->batch) share = most * d->batch > 0 ? most * d->batch : 1;
  p.share = (uint32_t)share;
  const int64_t fill = 256 / blocks;
  p.fill = (uint32_t)(d->workgroups > 0 || fill > share ? share : fill > 1 ? fill : 1);
  // one share: every sequence is one split, and its results are final
  int64_t units = share == 1 ? d->batch : share + d->batch;
  if (units > most * d->batch && most > 0) units = most * d->batch;
  p.units = (uint32_t)units;
  p.part = units > d->batch ? units * d->cache.kv_heads * rows : 0;
  return p;
}

int desc_check(const vh_tree_desc* d, const char* what) {
  VH_REQUIRE(d, "%s: null descriptor", what);
  const vh_cache& c = d->cache;
  if (int e = vh_cache_check(&c, what)) return e;
  VH_REQUIRE(d->dtype == VH_BF16 || d->dtype == VH_F16, "%s: queries must be bfloat16 or float16", what);
  VH_REQUIRE(c.fmt != CACHE_F16 || d->dtype == VH_F16, "%s: float16 queries for a float16 cache", what);
  VH_REQUIRE(c.fmt != CACHE_BF16 || d->dtype == VH_BF16, "%s: bfloat16 queries for a bfloat16 cache", what);
  VH_REQUIRE(c.dim == 64 || c.dim == 128 || c.dim == 256, "%s: heads of 64, 128 or 256 (got %d)", what, c.dim);
  VH_REQUIRE(c.page % 16 == 0, "%s: pages of a multiple of 16 tokens (got %d)", what, c.page);
  VH_REQUIRE(d->batch >= 0 && d->nodes >= 0 && d->table_pages >= 0, "%s: negative size", what);
  VH_REQUIRE(d->heads > 0 && d->heads % c.kv_heads == 0, "%s: query heads must be a multiple of the cache's", what);
  VH_REQUIRE((int64_t)d->nodes * (d->heads / c.kv_heads) < (1 << 24), "%s: too many rows", what);
  VH_REQUIRE((int64_t)d->table_pages * c.page < (1ll << 31) - 4096, "%s: too many pages", what);
  VH_REQUIRE((int64_t)d->batch * c.kv_heads < (1 << 20), "%s: too many sequences", what);
  VH_REQUIRE(d->batch * (((int64_t)d->table_pages * c.page + tree::PIECE - 1) / tree::PIECE) < (1ll << 32),
             "%s: too many keys", what);
  VH_REQUIRE(!d->masks || d->nodes <= MAX_NODES, "%s: at most %d nodes", what, MAX_NODES);
  VH_REQUIRE(d->scale > 0.0f && d->scale < __builtin_inff(), "%s: the scale must be positive", what);
  VH_REQUIRE(d->workgroups >= 0 && d->workgroups <= (1 << 20), "%s: bad number of workgroups", what);
  return VH_OK;
}

}  // namespace

extern "C" int vh_tree_masks(const int32_t* parents, int64_t batch, int32_t nodes, uint64_t* masks, int32_t* flag,
                             vh_stream_t stream) {
  VH_REQUIRE(batch >= 0 && batch < (1ll << 31) && nodes >= 0 && nodes <= MAX_NODES,
             "vh_tree_masks: at most %d nodes (got %d)", MAX_NODES, nodes);
  if (batch == 0 || nodes == 0) return VH_OK;
  VH_REQUIRE(parents && masks && flag, "vh_tree_masks: null argument");
  hipLaunchKernelGGL(k_tree_masks, dim3((unsigned)batch), dim3(MASK_THREADS), 0, vh::as_stream(stream), parents, nodes,
                     (nodes + 63) / 64, masks, flag);
  return vh::check_launch("vh_tree_masks");
}

extern "C" int64_t vh_tree_attention_workspace_bytes(const vh_tree_desc* d) {
  if (desc_check(d, "vh_tree_attention_workspace_bytes")) return -1;
  if (d->batch == 0 || d->nodes == 0) return 0;
  return plan_of(d).part * (int64_t)sizeof(float) * (d->cache.dim + 2);
}

extern "C" int vh_tree_attention(const vh_tree_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  if (int e = desc_check(d, "vh_tree_attention")) return e;
  if (d->batch == 0 || d->nodes == 0) return VH_OK;
  VH_REQUIRE(d->q && d->context && d->o && (d->table || d->table_pages == 0), "vh_tree_attention: null argument");
  VH_REQUIRE((uintptr_t)d->o % 16 == 0, "vh_tree_attention: misaligned output");
  const Plan p = plan_of(d);
  const int64_t need = p.part * (int64_t)sizeof(float) * (d->cache.dim + 2);
  VH_REQUIRE(need == 0 || (work && work_bytes >= need && (uintptr_t)work % 16 == 0),
             "vh_tree_attention: needs %lld bytes of aligned workspace", (long long)need);
  const int group = d->heads / d->cache.kv_heads;
  Args a{};
  a.c = d->cache;
  a.q = d->q;
  a.q_sb = d->q_sb;
  a.q_st = d->q_st;
  a.q_sh = d->q_sh;
  a.table = d->table;
  a.table_st = d->table_st;
  a.context = d->context;
  a.masks = d->masks;
  a.o = d->o;
  a.lse = d->lse;
  if (p.part > 0) {
    a.part_o = (float*)work;
    a.part_ml = a.part_o + p.part * d->cache.dim;
  }
  a.group_div = make_fast_div((uint32_t)group);
  a.page_div = make_fast_div((uint32_t)(d->cache.page / 16));
  a.scale = d->scale * tree::LOG2E;
  a.q_bf16 = d->dtype == VH_BF16;
  a.q_wide = (uintptr_t)d->q % 16 == 0 && d->q_sb % 8 == 0 && d->q_st % 8 == 0 && d->q_sh % 8 == 0;
  a.words = (d->nodes + 63) / 64;
  a.batch = d->batch;
  a.nodes = d->nodes;
  a.heads = d->heads;
  a.group = group;
  a.rows = d->nodes * group;
  a.row_blocks = p.row_blocks;
  a.block_rows = p.block_rows;
  a.table_pages = d->table_pages;
  a.share = p.share;
  a.fill = p.fill;
  a.units = p.units;
  VH_REQUIRE(((int64_t)p.units * a.c.kv_heads + 7) / 8 * 8 * a.row_blocks < (1ll << 31) &&
                 (int64_t)a.batch * a.c.kv_heads * a.rows < (1ll << 31),
             "vh_tree_attention: too many workgroups");
  hipStream_t s = vh::as_stream(stream);
  const int rc = d->cache.dim == 64 ? tree::launch<64>(a, p.wide, p.n, s)
                 : d->cache.dim == 128 ? tree::launch<128>(a, p.wide, p.n, s)
                                       : tree::launch<256>(a, p.wide, p.n, s);
  if (rc != VH_OK || p.part == 0) return rc;
  if (d->cache.dim == 64) merge<64>(a, s);
  else if (d->cache.dim == 128) merge<128>(a, s);
  else merge<256>(a, s);
  return vh::check_launch("vh_tree_attention");
}
