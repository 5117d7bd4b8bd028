// K and V of a batch's tokens quantised into pages, and read back (kv_quant_write,
// kv_quant_read; the layout is in llm_decoder.h).
//
// A row is one token of one head, D elements.  LPR lanes hold it, 8 elements each: the
// largest magnitude goes round them in log2(LPR) exchanges, everything else is the lane's
// own.  A thread takes its 8 elements of K and of V, so that they share one look-up and two
// loads are in flight.  A workgroup's rows are TJ consecutive tokens (a power of two, up to
// 16) of as many heads as fill it: tokens lie beside each other in a page, so what it writes
// are whole lines, and a single token's heads lie beside each other in k and v.
//
// Codes are those of exact arithmetic.  c x in fp32, c = fp32(largest / a), is off by two
// roundings, 2^-23 of itself, which matters where it is that near the border between two codes:
// there the question is asked in fp64, where largest |x| and border * a are exact (24 + 9 bits).
// About one element in ten thousand asks.
//
// Bound by the bytes where there are many rows (4 x 4096 tokens of 16 heads of 128 from fp16 to int8
// and back: written 45 us, read 40; 171 MB each way at the rate of a copy are 35), by the chain
// of lens, table and stores where there are few (64 single tokens of 16 heads: 4.3 and 3.1 us).
#include "common.hpp"
#include "paged_rows.hpp"

#include <algorithm>

namespace llm {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;  // elements of a lane

struct QuantArgs {
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;
  size_t page_stride, scale_stride;
  const int32_t* table;
  int num_pages, num_beams, num_heads, max_tiles, page_size, D;
  const void *k, *v;  // kv_quant_read writes them
  long long token_stride;
  const int32_t *beam_ids, *starts, *lens;
  int B, N;
  int tj_log, head_groups;  // a workgroup's tokens (log2), groups of heads
};

template <typename T>
__device__ __forceinline__ void load8(const void* base, long long at, float (&x)[kPer]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    typedef T V __attribute__((ext_vector_type(8)));
    const V a = *reinterpret_cast<const V*>(static_cast<const T*>(base) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  }
}

template <typename T>
__device__ __forceinline__ void store8(void* base, long long at, const float (&x)[kPer]) {
  if constexpr (sizeof(T) == 4) {
    f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + at);
    p[0] = f32x4{x[0], x[1], x[2], x[3]};
    p[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    typedef T V __attribute__((ext_vector_type(8)));
    V a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (T)x[i];
    *reinterpret_cast<V*>(static_cast<T*>(base) + at) = a;
  }
}

template <int KVT>
constexpr float largest_of() {
  return KVT == LLM_I8 ? 127.f : 448.f;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

// The code of |y| <= border or above, y = largest x / a in exact arithmetic: `low` and `low` + 1
// are the codes of magnitudes around the border, halves go to the even one.
__device__ __forceinline__ int exact_code(float x, float a, float largest, int low, double border) {
  const double at = (double)largest * fabs((double)x), edge = border * (double)a;
  return at > edge || (at == edge && (low & 1)) ? low + 1 : low;
}

// 8 codes of 8 elements (as 8 bytes) and the row's scale; every lane of the row calls it.
template <int KVT>
__device__ __forceinline__ u32x2 quantise(float (&x)[kPer], int lpr, float& scale) {
  constexpr float largest = largest_of<KVT>();
  uint32_t top = 0;  // of the magnitudes' bits: an infinity is above every number, a NaN above it
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  // (mirrors of 8 and 16 lanes: their halves hold the same by then)
  if (lpr >= 2) top = max(top, (uint32_t)mov_lanes<0xB1>((int)top));
  if (lpr >= 4) top = max(top, (uint32_t)mov_lanes<0x4E>((int)top));
  if (lpr >= 8) top = max(top, (uint32_t)mov_lanes<0x141>((int)top));
  if (lpr >= 16) top = max(top, (uint32_t)mov_lanes<0x140>((int)top));
  if (lpr >= 32) {
    const LanePair p = with_lane16(__builtin_bit_cast(float, top));
    top = max(__builtin_bit_cast(uint32_t, p.a), __builtin_bit_cast(uint32_t, p.b));
  }
  const bool finite = top < 0x7f800000u;
  float a = __builtin_bit_cast(float, top);
  scale = finite ? a / largest : __builtin_nanf("");
  if (a < 0x1p-60f) {  // (largest / a stays a number; what it is times is exact)
    a *= 0x1p80f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] *= 0x1p80f;
  }
  if (!finite || a == 0.f) return u32x2{0u, 0u};
  const float c = largest / a;
  u32x2 w = {0u, 0u};
  if constexpr (KVT == LLM_I8) {
    float far = 0.f;
    int code[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float y = x[i] * c, q = rintf(y);
      far = fmaxf(far, fabsf(y - q));
      code[i] = (int)q;
    }
    if (far > 0.5f - 0x1p-14f) {  // (y is off by 127 * 2^-23 at most)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float y = fabsf(x[i] * c);
        if (fabsf(y - rintf(y)) <= 0.5f - 0x1p-14f) continue;
        const int low = (int)y, mag = exact_code(x[i], a, largest, low, low + 0.5);
        code[i] = x[i] < 0.f ? -mag : mag;
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i / 4] |= (uint32_t)(code[i] & 0xff) << (8 * (i % 4));
  } else {
    u32x2 up;  // the codes of a little more: others where y is near a border
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y[4], z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = x[4 * i + e] * c;
        y[e] = t * (1.f - 0x1p-21f);
        z[e] = t * (1.f + 0x1p-21f);
      }
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
      up[i] = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false), true);
    }
    if (w[0] != up[0] || w[1] != up[1]) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int sh = 8 * (i % 4);
        const uint32_t low = w[i / 4] >> sh & 0x7fu, high = up[i / 4] >> sh & 0x7fu;
        if (low == high) continue;
        const double border = 0.5 * ((double)e4m3_value(low) + (double)e4m3_value(high));
        const uint32_t code = exact_code(x[i], a, largest, (int)low, border);
        w[i / 4] = (w[i / 4] & ~(0x7fu << sh)) | code << sh;
      }
    }
  }
  return w;
}

struct Place {
  bool value_there;  // k and v have this element
  bool token;  // ... and the row this token
  bool page;   // ... and it has a page
  size_t at;   // bytes into a pool
  size_t scale;
  long long value;  // elements into k and v
};

// This thread's token, and its lane among the row's.
__device__ __forceinline__ Place place_of(const QuantArgs& a, int lpr_log, bool write) {
  const int row = threadIdx.x >> lpr_log, lane = threadIdx.x & ((1 << lpr_log) - 1);
  const int rows_log = 8 - lpr_log;  // of the workgroup's kThreads
  const int b = blockIdx.y;
  const int tile = blockIdx.x / a.head_groups, hg = blockIdx.x - tile * a.head_groups;
  const int j = (tile << a.tj_log) + (row & ((1 << a.tj_log) - 1));
  const int h = (hg << (rows_log - a.tj_log)) + (row >> a.tj_log);
  const int n = a.lens ? min(a.lens[b], a.N) : a.N;
  const int beam = a.beam_ids ? a.beam_ids[b] : b;
  const int start = a.starts[b];
  Place p;
  p.value_there = j < a.N && h < a.num_heads && lane * kPer < a.D;
  p.token = p.value_there && j < n;
  p.value = ((long long)b * a.N + j) * a.token_stride + (long long)h * a.D + lane * kPer;
  p.page = false;
  p.at = p.scale = 0;
  const long long pos = (long long)start + j;
  if (p.token && pos >= 0 && pos < (long long)a.max_tiles * a.page_size && beam >= 0 && beam < a.num_beams) {
    const int t = (int)pos / a.page_size, slot = (int)pos - t * a.page_size;
    const int page = a.table[((size_t)beam * a.num_heads + h) * a.max_tiles + t];
    p.page = page >= 0 && page < a.num_pages;
    p.at = (size_t)page * a.page_stride + (size_t)slot * a.D + lane * kPer;
    p.scale = (size_t)page * a.scale_stride + slot;
  }
  if (write && a.beam_ids) {
    // a later row of the same beam that has this position keeps its token
    for (int i = b + 1; i < a.B; i += 64) {
      const int o = i + (threadIdx.x & 63);
      if (!__any(o < a.B && a.beam_ids[min(o, a.B - 1)] == beam)) continue;
      for (int r = i; r < min(i + 64, a.B); ++r) {
        if (a.beam_ids[r] != beam) continue;
        const long long d = pos - a.starts[r];
        if (d >= 0 && d < (a.lens ? min(a.lens[r], a.N) : a.N)) p.page = false;
      }
    }
  }
  return p;
}

template <typename T, int KVT>
__global__ __launch_bounds__(kThreads) void kv_quant_write_kernel(QuantArgs a, int lpr_log) {
  const Place p = place_of(a, lpr_log, true);
  float k[kPer] = {}, v[kPer] = {};
  if (p.value_there) {  // (they do not wait for lens)
    load8<T>(a.k, p.value, k);
    load8<T>(a.v, p.value, v);
  }
  float ks, vs;
  const u32x2 kc = quantise<KVT>(k, 1 << lpr_log, ks), vc = quantise<KVT>(v, 1 << lpr_log, vs);
  if (!p.page) return;
  *reinterpret_cast<u32x2*>(a.k_pool + p.at) = kc;
  *reinterpret_cast<u32x2*>(a.v_pool + p.at) = vc;
  if ((threadIdx.x & ((1 << lpr_log) - 1)) == 0) {
    a.k_scale[p.scale] = ks;
    a.v_scale[p.scale] = vs;
  }
}

template <int KVT>
__device__ __forceinline__ void values(u32x2 w, float scale, float (&x)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t byte = w[i / 4] >> (8 * (i % 4)) & 0xff;
    x[i] = scale * (KVT == LLM_I8 ? (float)(int8_t)byte : e4m3_value(byte));
  }
}

template <typename T, int KVT>
__global__ __launch_bounds__(kThreads) void kv_quant_read_kernel(QuantArgs a, int lpr_log) {
  const Place p = place_of(a, lpr_log, false);
  if (!p.token) return;
  float k[kPer] = {}, v[kPer] = {};
  if (p.page) {
    values<KVT>(*reinterpret_cast<const u32x2*>(a.k_pool + p.at), a.k_scale[p.scale], k);
    values<KVT>(*reinterpret_cast<const u32x2*>(a.v_pool + p.at), a.v_scale[p.scale], v);
  }
  store8<T>(const_cast<void*>(a.k), p.value, k);
  store8<T>(const_cast<void*>(a.v), p.value, v);
}

template <typename T, int KVT>
hipError_t launch_quant(const QuantArgs& a, int lpr_log, dim3 grid, bool write, hipStream_t st) {
  hipLaunchKernelGGL((write ? kv_quant_write_kernel<T, KVT> : kv_quant_read_kernel<T, KVT>), grid,
                     dim3(kThreads), 0, st, a, lpr_log);
  return hipGetLastError();
}

int log2_up(int n) {  // the least l with 2^l >= n
  int l = 0;
  while (1 << l < n) ++l;
  return l;
}

int quant(const char* name, const pa_kv_view* kv, const pa_kv_scales* scales, const void* k, const void* v,
          int dtype, long long token_stride, const int32_t* beam_ids, const int32_t* starts,
          const int32_t* lens, int B, int N, bool write, hipStream_t st) {
  const std::string who = std::string(name) + ": ";
  LLM_REQUIRE(B >= 0 && B <= 65535 && N >= 0, who + "bad B/N (0 <= B <= 65535, N >= 0)");
  LLM_REQUIRE(scales, who + "scales are NULL");
  if (const int rc = check_paged_view(name, kv, scales)) return rc;
  LLM_REQUIRE(kv->kv_dtype == LLM_I8 || kv->kv_dtype == LLM_E4M3,
              who + "kv_dtype must be LLM_I8 or LLM_E4M3");
  const int es = value_size(dtype), D = kv->head_dim, H = kv->num_heads;
  LLM_REQUIRE(es > 0, who + "dtype must be LLM_F32, LLM_F16 or LLM_BF16");
  if (D % kPer != 0 || D > 256)
    return fail(LLM_ERR_UNSUPPORTED, who + "head_dim must be a multiple of 8 up to 256");
  if (B == 0 || N == 0) return LLM_OK;
  LLM_REQUIRE(k && v && starts, who + "NULL pointer");
  if (token_stride == 0) token_stride = (long long)H * D;
  LLM_REQUIRE(token_stride >= (long long)H * D && token_stride * es % 16 == 0 && aligned16(k) && aligned16(v),
              who + "k and v must be 16-byte aligned, token_stride 0 or >= H * D and a multiple of 16 bytes");
  const int lpr_log = log2_up(D / kPer), rows_log = 8 - lpr_log;
  QuantArgs a{};
  a.k_pool = static_cast<uint8_t*>(const_cast<void*>(kv->k_pool));
  a.v_pool = static_cast<uint8_t*>(const_cast<void*>(kv->v_pool));
  a.k_scale = scales->k_scale;
  a.v_scale = scales->v_scale;
  a.page_stride = paged_stride(*kv);
  a.scale_stride = scales->page_stride ? (size_t)scales->page_stride : (size_t)kv->page_size;
  a.table = kv->page_table;
  a.num_pages = kv->num_pages;
  a.num_beams = kv->num_beams;
  a.num_heads = H;
  a.max_tiles = kv->max_tiles;
  a.page_size = kv->page_size;
  a.D = D;
  a.k = k;
  a.v = v;
  a.token_stride = token_stride;
  a.beam_ids = beam_ids;
  a.starts = starts;
  a.lens = lens;
  a.B = B;
  a.N = N;
  a.tj_log = std::min({rows_log, 4, log2_up(std::min(N, 16))});
  const int heads = 1 << (rows_log - a.tj_log);
  a.head_groups = (H + heads - 1) / heads;
  const long long groups = (((long long)N + (1 << a.tj_log) - 1) >> a.tj_log) * a.head_groups;
  LLM_REQUIRE(groups < (1LL << 32) / kThreads, who + "too many tokens in one call");  // (threads of a launch)
  const dim3 grid((unsigned)groups, B);
  const bool i8 = kv->kv_dtype == LLM_I8;
  hipError_t e;
  if (dtype == LLM_F32)
    e = i8 ? launch_quant<float, LLM_I8>(a, lpr_log, grid, write, st)
           : launch_quant<float, LLM_E4M3>(a, lpr_log, grid, write, st);
  else if (dtype == LLM_F16)
    e = i8 ? launch_quant<_Float16, LLM_I8>(a, lpr_log, grid, write, st)
           : launch_quant<_Float16, LLM_E4M3>(a, lpr_log, grid, write, st);
  else
    e = i8 ? launch_quant<__bf16, LLM_I8>(a, lpr_log, grid, write, st)
           : launch_quant<__bf16, LLM_E4M3>(a, lpr_log, grid, write, st);
  LLM_HIP_RET(e);
  return LLM_OK;
}

}  // namespace
}  // namespace llm

using namespace llm;

extern "C" int kv_quant_write(const pa_kv_view* kv, const pa_kv_scales* scales, const void* k, const void* v,
                              int dtype, long long token_stride, const int32_t* beam_ids,
                              const int32_t* starts, const int32_t* lens, int B, int N, void* stream) {
  return quant("kv_quant_write", kv, scales, k, v, dtype, token_stride, beam_ids, starts, lens, B, N, true,
               as_stream(stream));
}

extern "C" int kv_quant_read(const pa_kv_view* kv, const pa_kv_scales* scales, void* k, void* v, int dtype,
                             long long token_stride, const int32_t* beam_ids, const int32_t* starts,
                             const int32_t* lens, int B, int N, void* stream) {
  return quant("kv_quant_read", kv, scales, k, v, dtype, token_stride, beam_ids, starts, lens, B, N, false,
               as_stream(stream));
}
