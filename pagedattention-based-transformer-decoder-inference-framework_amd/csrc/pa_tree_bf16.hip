// pa_tree over bf16 pools: fp16 queries are two parts of bf16, fp32 ones three.
#include "pa_tree_impl.hpp"

hipError_t llm::launch_tree_bf16(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return a.dtype == LLM_BF16  ? launch_tree_dim<LLM_BF16, 1>(a, D, tiles, grid, st)
         : a.dtype == LLM_F16 ? launch_tree_dim<LLM_BF16, 2>(a, D, tiles, grid, st)
                              : launch_tree_dim<LLM_BF16, 3>(a, D, tiles, grid, st);
}
