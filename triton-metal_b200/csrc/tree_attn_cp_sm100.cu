// Attention of a tree of drafted tokens and of single tokens: the cp.async form,
// for page sizes that are no multiple of 8 and for tensors that no tensor map
// describes.
#include "tree_attn_kernel.cuh"

namespace b2 {
namespace tree {

void launch_cp(const Maps& m, const Params& p, int D, bool f16, bool pair, cudaStream_t st) {
  launch_form<false>(m, p, D, f16, pair, st);
}

}  // namespace tree
}  // namespace b2
