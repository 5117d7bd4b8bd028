// pa_tree over e4m3 pools.
#include "pa_tree_impl.hpp"

hipError_t llm::launch_tree_e4m3(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return launch_tree_parts<LLM_E4M3>(a, D, tiles, grid, st);
}
