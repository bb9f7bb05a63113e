// Attention of a tree of tokens over a paged cache, heads of 256.
#include "vh_tree_attention.h"

namespace tree {
template <>
int launch<256>(const Args& a, bool wide, int n, hipStream_t s) {
  return launch_d<256>(a, wide, n, s);
}
}  // namespace tree
