// pa_tree: checks, the split of long rows over workgroups, and their merge.
#include "pa_tree.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace llm {
namespace {

constexpr int kMergeThreads = 256;
constexpr int kWaveRows = 2048;

// A row's parts, relative to the largest of their maxima: `LANES` threads a row, D / 4 of which
// hold its dims, the others the same of every (4 LANES / D)th part.  A wave a row where there are
// rows enough to fill the card, else a workgroup a row.
template <int D, int LANES>
__global__ __launch_bounds__(kMergeThreads) void pa_tree_merge_kernel(TreeArgs a) {
  constexpr int PER = D / 4, WAYS = LANES / PER, ROWS = kMergeThreads / LANES;
  __shared__ f32x4 s_x[ROWS][WAYS][PER];
  __shared__ float s_sum[ROWS][WAYS];
  const int mine = threadIdx.x / LANES, d = threadIdx.x % PER, way = threadIdx.x % LANES / PER;
  const long long row = (long long)blockIdx.x * ROWS + mine;
  const long long token = row / a.H;
  const int h = (int)(row - token * a.H), b = (int)(token / a.N), i = (int)(token - (long long)b * a.N);
  bool live = row < (long long)a.B * a.N * a.H;
  float sum = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const TreeRow tr = tree_row(a, b);
    live = i < tr.n;
    const int parts = live ? max((tr.L + tr.split_len - 1) / tr.split_len, 1) : 0;
    const float* ml = a.ml + (size_t)row * a.nsplit * 2;
    const f32x4* acc = reinterpret_cast<const f32x4*>(a.acc + (size_t)row * a.nsplit * D) + d;
    float M = kNegSentinel;
    for (int s = lane_id(); s < parts; s += 64) M = fmaxf(M, ml[2 * s]);
    M = wave_max(M);
#pragma unroll 4
    for (int s = way; s < parts; s += WAYS) {
      const float weight = __builtin_amdgcn_exp2f(ml[2 * s] - M);
      sum = fmaf(ml[2 * s + 1], weight, sum);
      x += acc[(size_t)s * PER] * weight;
    }
  }
  if constexpr (WAYS > 1) {
    s_x[mine][way][d] = x;
    if (d == 0) s_sum[mine][way] = sum;
    __syncthreads();
    if (way > 0) return;
    for (int v = 1; v < WAYS; ++v) {
      x += s_x[mine][v][d];
      sum += s_sum[mine][v];
    }
  }
  if (!live) return;
  x *= 1.f / (sum + 1e-6f);
  const size_t at = (size_t)token * a.out_stride + (size_t)h * D + 4 * d;
  if (a.dtype == LLM_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = x;
  } else if (a.dtype == LLM_F16) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4*>(static_cast<_Float16*>(a.out) + at) = __builtin_convertvector(x, h4);
  } else {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<b4*>(static_cast<__bf16*>(a.out) + at) = __builtin_convertvector(x, b4);
  }
}

template <int D>
hipError_t launch_merge(const TreeArgs& a, hipStream_t st) {
  const long long rows = (long long)a.B * a.N * a.H;
  if (rows >= kWaveRows)
    hipLaunchKernelGGL((pa_tree_merge_kernel<D, 64>), dim3((unsigned)((rows + 3) / 4)), dim3(kMergeThreads), 0, st, a);
  else
    hipLaunchKernelGGL((pa_tree_merge_kernel<D, kMergeThreads>), dim3((unsigned)rows), dim3(kMergeThreads), 0, st, a);
  return hipGetLastError();
}

struct TreePlan {
  int tiles;  // row tiles of a workgroup
  int row_groups, nsplit, split_keys, waves;
};

// Splits of equal length, as many as fill the card once: two workgroups a CU, one where heads of 256
// leave registers for one (16 heads x 63 rows over 32768 e4m3 tokens, us: 256 workgroups 61, 512 54,
// 1024 65; 8 x 16 heads of 256 over 4000 int8 tokens 256 31, 512 38); half as many again where the rows
// of a batch take long turns, as T is the longest one's (16 x 2 heads x 168 over up to 4096: 47 -> 38).  A split has a fixed cost
// of some 5 us and its parts' way through memory: none below 256 keys, 128 where a turn takes
// four waves' tiles (4 x 80 rows over 1000 tokens 19, by 256 keys 23), and none of one tile's rows up
// to 512 tokens (12 heads x 8 over 300 tokens 7.4, in two splits 9.6).  Where the rows alone fill
// the card the parts are there against uneven rows: 2048 keys (64 x 16 heads over up to 8192 int8
// tokens: whole rows 257 us, 4096 keys 245, 2048 233, 1024 240).
//
// One tile's rows of 64 to 511 pairs of long rows take workgroups of 8 waves, half as many splits
// (4 x 16 heads over up to 8192 fp16 tokens 36.6 -> 32.7 us, 16 x 12 of 64 over 2048 int8, 8 tokens
// each, 19.6 -> 16.4, no merge); others 4 (12 heads over 1200 int8 tokens 11.7, by 8 waves 12.2; 64 x
// 16 heads over 500 20.2 and 26.2).
TreePlan tree_plan(const pa_kv_view& kv, int dtype, int B, int N, int H, int T) {
  TreePlan p;
  const int rows = N * (H / kv.num_heads);
  p.tiles = tree_tiles(kv.head_dim, tree_parts(kv.kv_dtype, dtype), rows);
  p.row_groups = (rows + 16 * p.tiles - 1) / (16 * p.tiles);
  const long long room = (long long)kv.max_tiles * kv.page_size;
  const long long keys = std::max(1LL, std::min((long long)T + N, room));
  const long long base = (long long)B * kv.num_heads * p.row_groups;
  const bool one = p.tiles == 1;
  p.waves = one && base >= 64 && base < 512 && keys > 512 ? tree_most_waves(kv.head_dim) : 4;
  const long long fill = kv.head_dim == 256 || p.waves == 8 ? 256 : one || B == 1 ? 512 : 768;
  const long long least = base >= fill ? 2048 : one ? (keys <= 512 ? 512 : 256) : 128;
  const long long want = base >= fill ? keys : fill / base;
  long long per = std::max(least, (keys + want - 1) / want);
  per = (per + kTreeStep - 1) / kTreeStep * kTreeStep;
  p.split_keys = (int)std::min(per, 1LL << 30);
  // (a launch has less than 2^32 threads)
  p.nsplit = (int)std::min({(keys + per - 1) / per, 1024LL, (1LL << 23) / ((long long)B * kv.num_heads)});
  p.nsplit = std::max(p.nsplit, 1);
  return p;
}

bool tree_sizes(const pa_kv_view& kv, int B, int N, int H, int T) {
  return B > 0 && B <= 65535 && N > 0 && N <= 1024 && H > 0 && T >= 0 && kv.num_heads > 0 &&
         H % kv.num_heads == 0 && H / kv.num_heads <= 64 && kv.max_tiles > 0 && kv.page_size > 0 &&
         (long long)B * kv.num_heads <= INT32_MAX / 256 && (long long)B * N * H <= INT32_MAX / 256;
}

}  // namespace
}  // namespace llm

using namespace llm;

extern "C" size_t pa_tree_workspace_bytes(const pa_kv_view* kv, int B, int N, int H, int T) {
  if (!kv || !tree_sizes(*kv, B, N, H, T)) return 0;
  size_t most = 0;  // over the types of q
  for (int dtype : {LLM_F32, LLM_F16, LLM_BF16}) {
    const TreePlan p = tree_plan(*kv, dtype, B, N, H, T);
    if (p.nsplit > 1) most = std::max(most, (size_t)B * N * H * p.nsplit * (kv->head_dim + 2) * sizeof(float));
  }
  return most;
}

extern "C" int pa_tree(const pa_kv_view* kv, const pa_kv_scales* scales, const void* q, long long q_stride,
                       void* out, long long out_stride, int dtype, const int32_t* beam_ids,
                       const int32_t* context_lens, const uint32_t* tree_mask, const int32_t* tree_lens, int B,
                       int N, int H, int D, int T, float sm_scale, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (const int rc = check_paged_view("pa_tree", kv, scales)) return rc;
  LLM_REQUIRE(B >= 0 && N >= 0 && H > 0 && D > 0 && T >= 0, "pa_tree: bad B/N/H/D/T");
  LLM_REQUIRE(kv->head_dim == D, "pa_tree: D != kv->head_dim");
  LLM_REQUIRE(H % kv->num_heads == 0, "pa_tree: H must be a multiple of kv->num_heads");
  LLM_REQUIRE(value_size(dtype) > 0, "pa_tree: dtype must be LLM_F32, LLM_F16 or LLM_BF16");
  LLM_REQUIRE(std::isfinite(sm_scale * kLog2e), "pa_tree: sm_scale must be finite");
  LLM_REQUIRE(kv->kv_dtype == LLM_I8 || (kv->kv_dtype == LLM_E4M3) == (scales != nullptr),
              "pa_tree: LLM_E4M3 pools need scales, 16-bit ones have none");
  if (D != 64 && D != 128 && D != 256)
    return fail(LLM_ERR_UNSUPPORTED, "pa_tree: head_dim must be 64, 128 or 256");
  if (kv->page_size % 16 != 0)
    return fail(LLM_ERR_UNSUPPORTED, "pa_tree: page_size must be a multiple of 16");
  if (B == 0 || N == 0) return LLM_OK;
  if (!tree_sizes(*kv, B, N, H, T))
    return fail(LLM_ERR_UNSUPPORTED, "pa_tree: B <= 65535, N <= 1024, H / num_heads <= 64, "
                                     "B * num_heads and B * N * H below 2^23");
  LLM_REQUIRE(q && out, "pa_tree: q/out NULL");
  const int es = value_size(dtype);
  if (q_stride == 0) q_stride = (long long)H * D;
  if (out_stride == 0) out_stride = (long long)H * D;
  LLM_REQUIRE(q_stride >= (long long)H * D && out_stride >= (long long)H * D && q_stride * es % 16 == 0 &&
                  out_stride * es % 16 == 0 && aligned16(q) && aligned16(out),
              "pa_tree: rows of q and out must be 16-byte aligned, strides 0 or >= H * D");
  const TreePlan p = tree_plan(*kv, dtype, B, N, H, T);
  LLM_REQUIRE(p.nsplit == 1 || (workspace && aligned16(workspace) &&
                                workspace_bytes >= pa_tree_workspace_bytes(kv, B, N, H, T)),
              "pa_tree: workspace NULL, not 16-byte aligned or below pa_tree_workspace_bytes");
  TreeArgs a{};
  a.q = q;
  a.out = out;
  a.dtype = dtype;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.k_pool = static_cast<const uint8_t*>(kv->k_pool);
  a.v_pool = static_cast<const uint8_t*>(kv->v_pool);
  if (scales) {
    a.k_scale = scales->k_scale;
    a.v_scale = scales->v_scale;
    a.scale_stride = scales->page_stride ? (size_t)scales->page_stride : (size_t)kv->page_size;
  }
  a.page_stride = paged_stride(*kv);
  a.table = kv->page_table;
  a.num_pages = kv->num_pages;
  a.num_beams = kv->num_beams;
  a.kv_heads = kv->num_heads;
  a.max_tiles = kv->max_tiles;
  a.page_size = kv->page_size;
  a.beam_ids = beam_ids;
  a.context_lens = context_lens;
  a.tree_lens = tree_lens;
  a.mask = tree_mask;
  a.mask_words = (N + 31) / 32;
  a.B = B;
  a.N = N;
  a.H = H;
  a.G = H / kv->num_heads;
  a.T = T;
  a.scale2 = sm_scale * kLog2e;
  a.nsplit = p.nsplit;
  a.split_keys = p.split_keys;
  a.waves = p.waves;
  a.acc = static_cast<float*>(workspace);
  a.ml = a.acc + (size_t)B * N * H * p.nsplit * D;
  const hipStream_t st = as_stream(stream);
  const int pairs = B * kv->num_heads;
  const dim3 grid = p.tiles == 1 ? dim3(pairs, p.nsplit) : dim3(pairs * p.nsplit, p.row_groups);
  hipError_t e = kv->kv_dtype == LLM_F16    ? launch_tree_f16(a, D, p.tiles, grid, st)
                 : kv->kv_dtype == LLM_BF16 ? launch_tree_bf16(a, D, p.tiles, grid, st)
                 : kv->kv_dtype == LLM_I8   ? launch_tree_i8(a, D, p.tiles, grid, st)
                                            : launch_tree_e4m3(a, D, p.tiles, grid, st);
  LLM_HIP_RET(e);
  if (p.nsplit > 1) {
    LLM_HIP_RET(D == 64 ? launch_merge<64>(a, st) : D == 128 ? launch_merge<128>(a, st) : launch_merge<256>(a, st));
  }
  return LLM_OK;
}
