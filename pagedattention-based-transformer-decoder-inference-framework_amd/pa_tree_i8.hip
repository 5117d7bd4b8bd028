// pa_tree over i8 pools.
#include "pa_tree_impl.hpp"

hipError_t llm::launch_tree_i8(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return launch_tree_parts<LLM_I8>(a, D, tiles, grid, st);
}
