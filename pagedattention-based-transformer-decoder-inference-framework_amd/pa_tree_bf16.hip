// pa_tree over bf16 pools.
#include "pa_tree_impl.hpp"

hipError_t llm::launch_tree_bf16(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return launch_tree_parts<LLM_BF16>(a, D, tiles, grid, st);
}
