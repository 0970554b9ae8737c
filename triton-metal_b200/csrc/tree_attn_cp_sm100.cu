// Attention of a tree of drafted tokens and of single tokens: the cp.async form,
// for pages too small for TMA boxes of 64 keys.
#include "tree_attn_kernel.cuh"

namespace b2 {
namespace tree {

void launch_tree_cp(const Params& p, int D, bool f16, bool pair, cudaStream_t st) {
  const Maps none = {};
  const bool cap = p.softcap.log2 > 0.f;
#define B2_TOKEN(HD, FMT)                                                                      \
  do {                                                                                         \
    if (cap) launch<HD, FMT, false, true, true, false>(none, p, st);                           \
    else launch<HD, FMT, false, false, true, false>(none, p, st);                              \
  } while (0)
  if (p.slopes) {  // single tokens with a bias
    if (D == 128 && f16) B2_TOKEN(128, fa::kF16);
    else if (D == 128) B2_TOKEN(128, fa::kBF16);
    else if (f16) B2_TOKEN(64, fa::kF16);
    else B2_TOKEN(64, fa::kBF16);
    return;
  }
#undef B2_TOKEN
#define B2_TREE(HD, FMT)                                                                       \
  do {                                                                                         \
    if (pair && cap) launch<HD, FMT, true, true, false, false>(none, p, st);                   \
    else if (pair) launch<HD, FMT, true, false, false, false>(none, p, st);                    \
    else if (cap) launch<HD, FMT, false, true, false, false>(none, p, st);                     \
    else launch<HD, FMT, false, false, false, false>(none, p, st);                             \
  } while (0)
  if (D == 128 && f16) B2_TREE(128, fa::kF16);
  else if (D == 128) B2_TREE(128, fa::kBF16);
  else if (f16) B2_TREE(64, fa::kF16);
  else B2_TREE(64, fa::kBF16);
#undef B2_TREE
}

}  // namespace tree
}  // namespace b2
