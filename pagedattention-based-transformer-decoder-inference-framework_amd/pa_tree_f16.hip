// pa_tree over f16 pools.
#include "pa_tree_impl.hpp"

hipError_t llm::launch_tree_f16(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return launch_tree_parts<LLM_F16>(a, D, tiles, grid, st);
}
