// Penalties for repeated tokens, biases and grammar masks on logits (logits_adjust; the
// formula is in llm_decoder.h).
//
// A workgroup takes a chunk of one row's vocabulary.  It counts the row's history in LDS, a
// word for each token of the chunk (bit 31: in the prompt, below it the times behind the
// prompt; whole numbers, so that the order of the additions does not count), and then
// streams its logits through once, 16 bytes a lane.  A second word holds the last bias
// entry of the token, as its place in the list + 1.  History and biases are read by every
// chunk of the row, from L2.
#include "common.hpp"
#include "paged_rows.hpp"

#include <algorithm>
#include <climits>

namespace llm {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;

struct AdjustArgs {
  const void* x;
  void* out;
  int V, chunk;
  long long stride;
  logits_rules r;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void logits_adjust_kernel(AdjustArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(VEC)));
  extern __shared__ uint32_t lds[];
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + (size_t)row * a.stride;
  T* out = static_cast<T*>(a.out) + (size_t)row * a.stride;
  // Chunks begin at 16 bytes of the row's own: `lead` tokens lie ahead of the first such place.
  const int lead = (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
  const int lo = blockIdx.x == 0 ? 0 : lead + (int)blockIdx.x * a.chunk - VEC;
  const int hi = min(lead + ((int)blockIdx.x + 1) * a.chunk - VEC, a.V);
  const int n = hi - lo;
  if (n <= 0) return;
  const logits_rules& r = a.r;
  const bool counts = r.history, biases = r.bias_ids, masks = r.allowed;
  uint32_t* met = lds;
  uint32_t* entry = lds + (counts ? a.chunk : 0);
  uint32_t* allow = entry + (biases ? a.chunk : 0);  // words of tokens lo / 32 * 32 ..
  if (counts)
    for (int i = tid; i < n; i += kThreads) met[i] = 0;
  if (biases)
    for (int i = tid; i < n; i += kThreads) entry[i] = 0;
  const int mask = masks ? (r.allowed_rows ? r.allowed_rows[row] : row) : -1;
  const bool masked = mask >= 0 && mask < r.num_masks;
  if (masked) {
    const int words = (a.V + 31) / 32, w0 = lo / 32, w1 = (hi + 31) / 32;
    for (int i = w0 + tid; i < w1; i += kThreads) allow[i - w0] = r.allowed[(size_t)mask * words + i];
  }
  __syncthreads();
  if (counts) {
    const int32_t* ids = r.history + (size_t)row * r.history_stride;
    const int len = r.history_lens ? clamp_int(r.history_lens[row], 0, r.history_len) : r.history_len;
    const int prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
    for (int i = tid; i < len; i += kThreads) {
      const uint32_t at = (uint32_t)ids[i] - (uint32_t)lo;
      if (at < (uint32_t)n) {
        if (i < prompt)
          atomicOr(&met[at], kPrompt);
        else
          atomicAdd(&met[at], 1u);
      }
    }
  }
  if (biases) {
    const int32_t* ids = r.bias_ids + (size_t)row * r.bias_stride;
    for (int i = tid; i < r.bias_len; i += kThreads) {
      const uint32_t at = (uint32_t)ids[i] - (uint32_t)lo;
      if (at < (uint32_t)n) atomicMax(&entry[at], (uint32_t)i + 1u);
    }
  }
  __syncthreads();
  const float rep = r.repetition ? r.repetition[row] : 1.f, freq = r.frequency ? r.frequency[row] : 0.f,
              pres = r.presence ? r.presence[row] : 0.f;
  const float* bias = r.bias + (biases ? (size_t)row * r.bias_stride : 0);
  auto one = [&](int i, float v) -> float {  // token lo + i
    if (counts && met[i]) {
      v = v > 0.f ? v / rep : v * rep;
      const float c = (float)(met[i] & ~kPrompt);
      if (c > 0.f) v -= freq * c + pres;
    }
    if (biases && entry[i]) v += bias[entry[i] - 1];
    if (masked && !(allow[(lo + i) / 32 - lo / 32] >> ((lo + i) & 31) & 1u)) v = -INFINITY;
    return v;
  };
  // ahead of the first 16-byte place (the first chunk alone), then whole ones, then the rest
  const int head = blockIdx.x == 0 ? min(lead, n) : 0;
  const int whole = head + (n - head) / VEC * VEC;
  if (tid < head) out[tid] = (T)one(tid, (float)x[tid]);
  if ((uintptr_t)(out + head) % 16 == (uintptr_t)(x + head) % 16) {
    for (int i = head + tid * VEC; i < whole; i += kThreads * VEC) {
      Vec v = *reinterpret_cast<const Vec*>(x + lo + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = (T)one(i + e, (float)v[e]);
      *reinterpret_cast<Vec*>(out + lo + i) = v;
    }
  } else {
    for (int i = head + tid; i < whole; i += kThreads) out[lo + i] = (T)one(i, (float)x[lo + i]);
  }
  if (whole + tid < n) out[lo + whole + tid] = (T)one(whole + tid, (float)x[lo + whole + tid]);
}

// Tokens of a workgroup: as many as their words fit 32 KiB of LDS, fewer where the rows are
// few, so that they reach more CUs.
int chunk_of(int rows, int V, bool biases) {
  int chunk = biases ? 4096 : 8192;
  while (chunk > 1024 && (long long)rows * ((V + chunk - 1) / chunk) < 512) chunk /= 2;
  return chunk;
}

template <typename T>
hipError_t launch_adjust(const AdjustArgs& a, int rows, hipStream_t st) {
  const size_t words = (size_t)a.chunk * ((a.r.history ? 1 : 0) + (a.r.bias_ids ? 1 : 0)) +
                       (a.r.allowed ? a.chunk / 32 + 2 : 0);
  // (the first chunk is up to VEC shorter than the others, a row's last place up to lead + VEC later)
  const int chunks = (int)(((long long)a.V + 16 + a.chunk - 1) / a.chunk);
  hipLaunchKernelGGL(logits_adjust_kernel<T>, dim3(chunks, rows), dim3(kThreads), words * 4, st, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace llm

using namespace llm;

extern "C" int logits_adjust(const void* logits, void* out, int dtype, int rows, int V, long long stride,
                             const logits_rules* rules, void* stream) {
  LLM_REQUIRE(rows >= 0 && rows <= 65535 && V > 0 && V <= 1 << 30,
              "logits_adjust: bad shape (0 <= rows <= 65535, 0 < V <= 2^30)");
  LLM_REQUIRE(value_size(dtype) > 0, "logits_adjust: dtype must be LLM_F32, LLM_F16 or LLM_BF16");
  LLM_REQUIRE(rules, "logits_adjust: rules are NULL");
  if (rows == 0) return LLM_OK;
  LLM_REQUIRE(logits && out, "logits_adjust: NULL pointer");
  if (stride == 0) stride = V;
  LLM_REQUIRE(stride >= V, "logits_adjust: stride must be 0 or >= V");
  LLM_REQUIRE((uintptr_t)logits % value_size(dtype) == 0 && (uintptr_t)out % value_size(dtype) == 0,
              "logits_adjust: logits and out must be aligned to their elements");
  const logits_rules& r = *rules;
  LLM_REQUIRE(!r.history || (r.history_len >= 0 && (r.history_stride == 0 || r.history_stride >= r.history_len)),
              "logits_adjust: bad history_len / history_stride");
  LLM_REQUIRE(r.history || (!r.repetition && !r.frequency && !r.presence),
              "logits_adjust: penalties need a history");
  LLM_REQUIRE(!r.bias_ids == !r.bias, "logits_adjust: bias_ids and bias go together");
  LLM_REQUIRE(!r.bias_ids || (r.bias_len >= 0 && (r.bias_stride == 0 || r.bias_stride >= r.bias_len)),
              "logits_adjust: bad bias_len / bias_stride");
  LLM_REQUIRE(!r.allowed || r.num_masks > 0, "logits_adjust: num_masks must be positive");
  LLM_REQUIRE(!r.allowed || r.allowed_rows || r.num_masks >= rows,
              "logits_adjust: without allowed_rows every row needs a mask of its own");
  AdjustArgs a{logits, out, V, chunk_of(rows, V, r.bias_ids), stride, r};
  hipError_t e;
  if (dtype == LLM_F32)
    e = launch_adjust<float>(a, rows, as_stream(stream));
  else if (dtype == LLM_F16)
    e = launch_adjust<_Float16>(a, rows, as_stream(stream));
  else
    e = launch_adjust<__bf16>(a, rows, as_stream(stream));
  LLM_HIP_RET(e);
  return LLM_OK;
}
