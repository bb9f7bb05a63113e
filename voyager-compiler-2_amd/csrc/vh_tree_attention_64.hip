// Attention of a tree of tokens over a paged cache, heads of 64.
#include "vh_tree_attention.h"

namespace tree {
template <>
int launch<64>(const Args& a, bool wide, int n, hipStream_t s) {
  return launch_d<64>(a, wide, n, s);
}
}  // namespace tree
