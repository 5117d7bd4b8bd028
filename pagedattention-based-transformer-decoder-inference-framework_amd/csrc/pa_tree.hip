// pa_tree: checks, the split of long rows over workgroups, and their merge.
#include "pa_tree.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace llm {
namespace {

constexpr int kMergeThreads = 256;
// From this many rows on a wave joins each, four to a workgroup (5376 rows of 128 in 11 parts: 8.5 -> 6.1 us); fewer
// rows would leave CUs empty: a workgroup each, its waves over the splits.
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

// Splits of one tile's rows: of equal length, as many as fill the card once, two workgroups of 4 waves a CU,
// one of 8, or where heads of 256 leave registers for one (8 x 16 heads of 256 over 4000 int8
// tokens, us: 256 workgroups 31, 512 38).  A split has a fixed cost of some 5 us and its parts' way
// through memory: none below 256 keys, and none up to 512 tokens (12 heads x 8 over 300 tokens 7.4, in two
// splits 9.6).  Where the rows alone fill the card the parts are there against uneven rows: 2048
// keys (64 x 16 heads over up to 8192 int8 tokens: whole rows 257, 4096 keys 245, 2048 233, 1024 240).
// 64 to 511 pairs of long rows take 8 waves, half as many splits (4 x 16 heads over up to 8192 fp16
// tokens 36.6 -> 32.7, 16 x 12 of 64 over 2048 int8, 8 tokens each, 19.6 -> 16.4, no merge); others 4 (12
// heads over 1200 int8 tokens 11.7, by 8 waves 12.2; 64 x 16 heads over 500 20.2 and 26.2).
void plan_one_tile(TreePlan& p, const pa_kv_view& kv, long long base, long long keys) {
  p.waves = base >= 64 && base < 512 && keys > 512 ? tree_most_waves(kv.head_dim) : 4;
  const long long fill = kv.head_dim == 256 || p.waves == 8 ? 256 : 512;
  const long long least = base >= fill ? 2048 : keys <= 512 ? 512 : 256;
  const long long want = base >= fill ? keys : fill / base;
  p.split_keys = (int)std::max(least, (keys + want - 1) / want);
}

// Splits of more tiles, whose turns are long: the length for which one or two rounds of workgroups, or
// whole rows, are priced least.  In us, as measured: a workgroup 8 and a turn of its KW blocks 2 (1.4 with
// one tile a wave, 3.5 of heads of 256), 0.65 of it with a CU to itself and up to that with every place taken;
// two a CU, three of heads of 64 in 8 bits with more than 64 rows; a merge 4.5, and every part's way through
// memory.  The plan does not know the rows' lengths.  From 4 rows on it prices two batches, one whose rows are
// all as long as T and one whose rows have 0.6 of it on average, each relative to its own best, the uneven one,
// which is what a server has, twice.  (us, even | uneven: 4 x 16 x 63 rows over 8192 int8 tokens in 13 parts, as the
// uneven batch alone has it, 73 | 63, in 8 65 | 62; 64 x 4 x 40 over 2048 fp16 in 3 74 | 47, in 2 62 | 42;
// 6 x 8 x 48 over 3000 fp16 in 12 38 | 27, in 8 31 | 27; 8 x 8 x 128 over 4096 fp16 in 11 76 | 51, in 7 63 | 57; 4 x 2 x
// 2048 over 1024 bf16 in 6 71 | 80, in 4 66 | 62; 32 x 8 x 63 of 64 over 6000 int8 in 3 119 | 96, in 2 105 | 102.  Left
// as the uneven batch has it: 16 x 2 x 168 over 4096 bf16 in 11 58 | 40, in 7 47 | 44.)
void plan_tiles(TreePlan& p, const pa_kv_view& kv, int parts, int B, int N, int H, long long base, long long keys) {
  const int D = kv.head_dim, mt = tree_wave_tiles(D, parts);
  const int turn_keys = kTreeKeys * (mt == 2 && p.tiles == 4 ? 2 : 1);
  const double turn = D == 256 ? 3.5 : mt == 2 ? 2.0 : 1.4;
  const double slots = D == 256 ? 256 : D == 64 && paged_elem_size(kv.kv_dtype) == 1 && p.tiles == 8 ? 768 : 512;
  const double part = (double)B * N * H * (D + 2) * 8 / 1.2e7;
  // rows of `share` of the longest row's splits (and of a last one that is not full, 0.25 more)
  auto price = [&](long long per, double share) {
    const double m = (double)((keys + per - 1) / per);
    const double groups = base * (share < 1 ? std::min(m, share * m + 0.25) : m);
    const double turns = (double)std::min(per, keys) / turn_keys * turn;
    const double full = std::floor(groups / slots), rest = groups / slots - full;
    return full * (8 + turns) + (rest > 0 ? 8 + turns * (0.65 + 0.35 * std::max(2 * rest - 1, 0.0)) : 0) +
           (m > 1 ? 4.5 + part * share * m : 0);
  };
  constexpr double kShares[2] = {1.0, 0.6}, kWeights[2] = {1.0, 2.0};
  const int batches = B >= 4 ? 2 : 1;
  long long pers[5];
  int n = 0;
  for (int rounds = 0; rounds <= 2; ++rounds)
    for (int i = 0; i < (rounds ? batches : 1); ++i) {
      const long long want = rounds ? std::max(1LL, (long long)(rounds * slots / (kShares[i] * base))) : 1;
      pers[n++] = std::max(128LL, ((keys + want - 1) / want + kTreeStep - 1) / kTreeStep * kTreeStep);
    }
  double best[2], least = 0;
  for (int i = 0; i < batches; ++i) {
    best[i] = price(pers[0], kShares[i]);
    for (int c = 1; c < n; ++c) best[i] = std::min(best[i], price(pers[c], kShares[i]));
  }
  for (int c = 0; c < n; ++c) {
    double cost = 0;
    for (int i = 0; i < batches; ++i) cost += kWeights[i] * price(pers[c], kShares[i]) / best[i];
    if (c && cost >= least) continue;
    least = cost;
    p.split_keys = (int)std::min(pers[c], 1LL << 30);
  }
}

TreePlan tree_plan(const pa_kv_view& kv, int dtype, int B, int N, int H, int T) {
  TreePlan p;
  const int rows = N * (H / kv.num_heads), parts = tree_parts(kv.kv_dtype, dtype);
  p.tiles = tree_tiles(kv.head_dim, parts, rows);
  p.row_groups = (rows + 16 * p.tiles - 1) / (16 * p.tiles);
  p.waves = 4;
  const long long room = (long long)kv.max_tiles * kv.page_size;
  const long long keys = std::max(1LL, std::min((long long)T + N, room));
  const long long base = (long long)B * kv.num_heads * p.row_groups;
  if (p.tiles == 1)
    plan_one_tile(p, kv, base, keys);
  else
    plan_tiles(p, kv, parts, B, N, H, base, keys);
  p.split_keys = (p.split_keys + kTreeStep - 1) / kTreeStep * kTreeStep;
  // (a launch has less than 2^32 threads)
  const long long most = std::min(1024LL, (1LL << 23) / ((long long)B * kv.num_heads));
  p.nsplit = (int)std::max(1LL, std::min((keys + p.split_keys - 1) / p.split_keys, most));
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
