// The plan of a packed batch, and the entry points of its attention.
#include "vh_prompt.h"

#include <algorithm>

namespace prompt {
template <>
int forward<64>(const Args& a, bool bf16, hipStream_t s);
template <>
int forward<128>(const Args& a, bool bf16, hipStream_t s);
template <>
int forward<256>(const Args& a, bool bf16, hipStream_t s);
template <>
int backward<64>(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s);
template <>
int backward<128>(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s);
template <>
int backward<256>(const Args& a, bool bf16, const int32_t* q_order, const int32_t* k_order, hipStream_t s);
}  // namespace prompt

namespace {

using prompt::Args;
using prompt::BLOCK;
using prompt::THREADS;

int64_t blocks_of(int64_t tokens) { return (tokens + BLOCK - 1) / BLOCK; }

// The plan: first [tokens], past [tokens], the blocks of rows in order, the
// blocks of keys in order.  A row that pads sees no key and is seen by none:
// first is the row after it, past itself, so that both rise with the row.
__global__ void __launch_bounds__(THREADS) k_packing(const int32_t* offsets, int64_t sequences, int tokens, int32_t* first,
                                                     int32_t* past, int32_t* flag) {
  int bad = 0;
  for (int64_t s = threadIdx.x; s <= sequences; s += THREADS) {
    const int at = offsets[s], before = s > 0 ? offsets[s - 1] : 0;
    bad |= at < before || at > tokens || (s == 0 && at != 0);
  }
  bad = __syncthreads_or(bad);
  if (bad && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(flag, VH_PACKING_ERR_OFFSETS);
  const int i = blockIdx.x * THREADS + threadIdx.x;
  if (i >= tokens) return;
  int from = i + 1, to = i;
  if (!bad && i < offsets[sequences]) {
    int64_t lo = 0, hi = sequences;  // offsets[lo] <= i < offsets[hi]
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (offsets[mid] <= i) lo = mid;
      else hi = mid;
    }
    from = offsets[lo];
    to = offsets[hi];
  }
  first[i] = from;
  past[i] = to;
}

// The blocks by their work, the most first, of equal ones the first first: a
// block's place is the number of those before it.
__global__ void __launch_bounds__(THREADS) k_packing_order(const int32_t* first, const int32_t* past, int tokens, int blocks,
                                                           int32_t* q_order, int32_t* k_order) {
  __shared__ int s_work[2][THREADS];
  const auto work = [&](int b, int& q, int& k) {
    const int row0 = b * BLOCK, end = min(row0 + BLOCK, tokens);
    q = max(end - first[row0], 0);
    k = max(past[end - 1] - row0, 0);
  };
  const int b = blockIdx.x * THREADS + threadIdx.x;
  int q = 0, k = 0, q_at = 0, k_at = 0;
  if (b < blocks) work(b, q, k);
  for (int c0 = 0; c0 < blocks; c0 += THREADS) {
    __syncthreads();
    if (c0 + (int)threadIdx.x < blocks) work(c0 + threadIdx.x, s_work[0][threadIdx.x], s_work[1][threadIdx.x]);
    __syncthreads();
    const int n = min(THREADS, blocks - c0);
    for (int i = 0; i < n; ++i) {
      q_at += s_work[0][i] > q || (s_work[0][i] == q && c0 + i < b);
      k_at += s_work[1][i] > k || (s_work[1][i] == k && c0 + i < b);
    }
  }
  if (b >= blocks) return;
  q_order[q_at] = b;
  k_order[k_at] = b;
}

bool rows_aligned(const void* p, int64_t st, int64_t sh) {
  return (uintptr_t)p % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && st >= 0 && sh >= 0;
}

// A tile's last row is found by a 31-bit number of bytes.
constexpr int64_t MOST_STRIDE = (1ll << 30) / 128;

int check(const vh_prompt_desc* d, const char* what) {
  VH_REQUIRE(d, "%s: null descriptor", what);
  VH_REQUIRE(d->dtype == VH_BF16 || d->dtype == VH_F16, "%s: values must be bfloat16 or float16", what);
  VH_REQUIRE(d->dim == 64 || d->dim == 128 || d->dim == 256, "%s: heads of 64, 128 or 256 (got %d)", what, d->dim);
  VH_REQUIRE(d->tokens >= 0 && d->tokens < VH_PROMPT_MAX_TOKENS, "%s: at most %d tokens", what, VH_PROMPT_MAX_TOKENS - 1);
  VH_REQUIRE(d->kv_heads > 0 && d->heads > 0 && d->heads % d->kv_heads == 0, "%s: query heads must be a multiple of the keys'", what);
  // a launch has fewer than 2^32 threads
  VH_REQUIRE((blocks_of(d->tokens) + 1) * d->heads < (1ll << 23), "%s: too many heads for as many tokens", what);
  VH_REQUIRE(d->sequences >= 0, "%s: negative size", what);
  VH_REQUIRE(d->scale > 0.0f && d->scale < __builtin_inff(), "%s: the scale must be positive", what);
  VH_REQUIRE(d->q_st < MOST_STRIDE && d->k_st < MOST_STRIDE && d->v_st < MOST_STRIDE && d->go_st < MOST_STRIDE,
             "%s: tokens lie too far apart", what);
  return VH_OK;
}

int check_inputs(const vh_prompt_desc* d, const char* what) {
  VH_REQUIRE(d->q && d->k && d->v && d->plan && d->o && d->lse, "%s: null argument", what);
  VH_REQUIRE(rows_aligned(d->q, d->q_st, d->q_sh) && rows_aligned(d->k, d->k_st, d->k_sh) && rows_aligned(d->v, d->v_st, d->v_sh) &&
                 ((uintptr_t)d->o | (uintptr_t)d->o_low) % 16 == 0,
             "%s: rows must be aligned to 16 bytes", what);
  return VH_OK;
}

Args args_of(const vh_prompt_desc* d) {
  Args a{};
  a.q = {d->q, d->q_st, d->q_sh};
  a.k = {d->k, d->k_st, d->k_sh};
  a.v = {d->v, d->v_st, d->v_sh};
  a.go = {d->go, d->go_st, d->go_sh};
  a.first = d->plan;
  a.past = d->plan + d->tokens;
  a.order = d->plan + 2 * d->tokens;
  a.o = d->o;
  a.o_low = d->o_low;
  a.gq = d->gq;
  a.gk = d->gk;
  a.gv = d->gv;
  a.lse = d->lse;
  a.rest = d->o_low ? d->lse + d->tokens * d->heads : nullptr;
  a.scale = d->scale;
  a.tokens = (int)d->tokens;
  a.sequences = d->sequences;
  a.heads = d->heads;
  a.kv_heads = d->kv_heads;
  a.group = d->heads / d->kv_heads;
  return a;
}

// Where the passes over blocks of keys are few for the card, or one long, they
// are cut into items of equal work, whose number's bound goes by the sizes
// alone; the device knows the work.
struct Back {
  int64_t rows, items, joins, slots, part;  // bytes, but for the slots
  int item_count, share;
};
Back back_of(const vh_prompt_desc* d) {
  const int64_t blocks = blocks_of(d->tokens), each = (int64_t)d->kv_heads * (d->dim / prompt::key_channels_of(d->dim));
  Back b{};
  b.rows = (d->tokens * d->heads * 2 * (int64_t)sizeof(float) + 15) / 16 * 16;
  if (blocks == 0 || blocks * each > prompt::MOST_CUT) return b;
  // the workgroups that the card holds at once, for each of those that share an item
  const int64_t share = (256 * prompt::back_waves_of(d->dim) + each - 1) / each;
  b.share = (int)share;
  b.item_count = (int)(blocks + share + 1);
  // a block in more than one item has at most twice the items that its work is,
  // and an item at least the rows of two blocks
  b.slots = std::min({blocks + share, 2 * share, (blocks + 1) * (blocks + 1) / 4});
  b.items = b.item_count * (int64_t)sizeof(int4);
  b.joins = (blocks * (int64_t)sizeof(int2) + 15) / 16 * 16;
  b.part = b.slots * d->kv_heads * 2 * BLOCK * d->dim * (int64_t)sizeof(float);
  return b;
}

int64_t workspace(const vh_prompt_desc* d) {
  const Back b = back_of(d);
  return b.rows + b.items + b.joins + b.part;
}

}  // namespace

extern "C" int64_t vh_packing_ints(int64_t tokens) {
  return tokens < 0 || tokens >= VH_PROMPT_MAX_TOKENS ? -1 : 2 * (tokens + blocks_of(tokens));
}

extern "C" int vh_packing(const int32_t* offsets, int64_t sequences, int64_t tokens, int32_t* plan, int32_t* flag,
                          vh_stream_t stream) {
  VH_REQUIRE(tokens >= 0 && tokens < VH_PROMPT_MAX_TOKENS, "vh_packing: at most %d tokens", VH_PROMPT_MAX_TOKENS - 1);
  // every workgroup reads them all
  VH_REQUIRE(sequences >= 0 && sequences < VH_PACKING_MAX_SEQUENCES, "vh_packing: at most %d sequences", VH_PACKING_MAX_SEQUENCES - 1);
  VH_REQUIRE(offsets && flag && (plan || tokens == 0), "vh_packing: null argument");
  hipStream_t s = vh::as_stream(stream);
  int32_t *first = plan, *past = plan + tokens, *order = plan + 2 * tokens;
  const int blocks = (int)blocks_of(tokens);
  const unsigned grid = (unsigned)((tokens + THREADS - 1) / THREADS);
  hipLaunchKernelGGL(k_packing, dim3(grid ? grid : 1), dim3(THREADS), 0, s, offsets, sequences, (int)tokens, first, past, flag);
  if (blocks > 0)
    hipLaunchKernelGGL(k_packing_order, dim3((unsigned)((blocks + THREADS - 1) / THREADS)), dim3(THREADS), 0, s, first, past,
                       (int)tokens, blocks, order, order + blocks);
  return vh::check_launch("vh_packing");
}

extern "C" int vh_prompt_attention(const vh_prompt_desc* d, vh_stream_t stream) {
  if (int e = check(d, "vh_prompt_attention")) return e;
  if (d->tokens == 0) return VH_OK;
  if (int e = check_inputs(d, "vh_prompt_attention")) return e;
  const Args a = args_of(d);
  hipStream_t s = vh::as_stream(stream);
  const bool bf16 = d->dtype == VH_BF16;
  return d->dim == 64 ? prompt::forward<64>(a, bf16, s) : d->dim == 128 ? prompt::forward<128>(a, bf16, s) : prompt::forward<256>(a, bf16, s);
}

extern "C" int64_t vh_prompt_attention_workspace_bytes(const vh_prompt_desc* d) {
  if (check(d, "vh_prompt_attention_workspace_bytes")) return -1;
  return workspace(d);
}

extern "C" int vh_prompt_attention_backward(const vh_prompt_desc* d, void* work, int64_t work_bytes, vh_stream_t stream) {
  if (int e = check(d, "vh_prompt_attention_backward")) return e;
  if (d->tokens == 0) return VH_OK;
  if (int e = check_inputs(d, "vh_prompt_attention_backward")) return e;
  VH_REQUIRE(d->go && d->o_low && d->gq && d->gk && d->gv, "vh_prompt_attention_backward: null argument");
  VH_REQUIRE(rows_aligned(d->go, d->go_st, d->go_sh) && ((uintptr_t)d->gq | (uintptr_t)d->gk | (uintptr_t)d->gv) % 16 == 0,
             "vh_prompt_attention_backward: rows must be aligned to 16 bytes");
  VH_REQUIRE(work && work_bytes >= workspace(d) && (uintptr_t)work % 16 == 0,
             "vh_prompt_attention_backward: needs %lld bytes of aligned workspace", (long long)workspace(d));
  Args a = args_of(d);
  const Back b = back_of(d);
  char* at = (char*)work;
  a.rows = (float*)at;
  if (b.item_count > 0) {
    a.items = (int4*)(at += b.rows);
    a.joins = (int2*)(at += b.items);
    a.part = (float*)(at += b.joins);
    a.item_count = b.item_count;
    a.share = b.share;
  }
  hipStream_t s = vh::as_stream(stream);
  const bool bf16 = d->dtype == VH_BF16;
  const int32_t *q = a.order, *k = a.order + blocks_of(d->tokens);
  return d->dim == 64 ? prompt::backward<64>(a, bf16, q, k, s)
         : d->dim == 128 ? prompt::backward<128>(a, bf16, q, k, s)
                         : prompt::backward<256>(a, bf16, q, k, s);
}
