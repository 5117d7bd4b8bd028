// Penalties for repeated tokens, biases and grammar masks on logits (logits_adjust; the
// formula is in llm_decoder.h).
//
// A workgroup takes a chunk of one row's vocabulary: its logits go into registers first, 16 bytes
// a load, and while they come it counts the row's history in LDS, a word for each token of the
// chunk (bit 31: in the prompt, below it the times behind the prompt; whole numbers, so that
// the order of the additions does not count).  A second word holds the last bias entry of the
// token, as its place in the list + 1.  History and biases are read by every chunk of the row,
// from L2, kIds loads of a thread at a time: they are what a short chunk waits for (256 rows of 50,257
// bf16 with history 500 and biases, by 1, 2, 4, 8 and 16 at a time: 18.6, 18.0, 18.5, 20.2 and 23.8 us; 64
// rows of fp32 with history 4096: 13.5, 12.3, 12.0, 11.9 and 12.4).
#include "common.hpp"
#include "paged_rows.hpp"

#include <algorithm>

namespace llm {
namespace {

constexpr int kThreads = 256;
constexpr int kIds = 4;
constexpr int kMostIds = 1 << 30;  // (places in a list and the steps behind it stay in 32 bits)
constexpr uint32_t kPrompt = 0x80000000u;

struct AdjustArgs {
  const void* x;
  void* out;
  int V;
  long long stride;
  logits_rules r;
};

// Tokens of 16 bytes, and of a chunk of U loads a thread.
template <typename T>
constexpr int vec_of() {
  return 16 / sizeof(T);
}
template <typename T, int U>
constexpr int chunk_of() {
  return kThreads * vec_of<T>() * U;
}

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void logits_adjust_kernel(AdjustArgs a) {
  constexpr int VEC = vec_of<T>(), CHUNK = chunk_of<T, U>();
  typedef T Vec __attribute__((ext_vector_type(VEC)));
  extern __shared__ __align__(16) uint32_t lds[];
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + (size_t)row * a.stride;
  T* out = static_cast<T*>(a.out) + (size_t)row * a.stride;
  // Chunks begin at 16 bytes of the row's own; the first one has up to VEC - 1 tokens ahead of such a place.
  const int lead = (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
  const int head = blockIdx.x == 0 ? min(lead, a.V) : 0;
  const int lo = blockIdx.x == 0 ? 0 : lead + (int)blockIdx.x * CHUNK - VEC;
  const int n = min(lead + ((int)blockIdx.x + 1) * CHUNK - VEC, a.V) - lo;
  if (n <= 0) return;
  const int whole = head + (n - head) / VEC * VEC;
  const logits_rules& r = a.r;
  const bool counts = r.history, biases = r.bias_ids;
  const int mask = !r.allowed ? -1 : r.allowed_rows ? r.allowed_rows[row] : row;
  const bool masked = mask >= 0 && mask < r.num_masks;
  const int words = (a.V + 31) / 32;
  const uint32_t* allow = masked ? r.allowed + (size_t)mask * words : nullptr;

  Vec v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int i = head + (k * kThreads + tid) * VEC;
    if (i < whole) v[k] = *reinterpret_cast<const Vec*>(x + lo + i);
  }
  // token lo + i at pad + i, so that VEC of them are 16 bytes' multiples there too
  const int pad = (VEC - head) % VEC;
  uint32_t* met = lds;
  uint32_t* entry = lds + (counts ? CHUNK : 0);
  const u32x4 none = {0u, 0u, 0u, 0u};
  if (counts)
    for (int i = tid * 4; i < CHUNK; i += kThreads * 4) *reinterpret_cast<u32x4*>(met + i) = none;
  if (biases)
    for (int i = tid * 4; i < CHUNK; i += kThreads * 4) *reinterpret_cast<u32x4*>(entry + i) = none;
  __syncthreads();
  // f(place in the chunk, place in the list) for the ids of a list that lie in the chunk
  auto scan = [&](const int32_t* ids, int len, auto f) {
    for (int i = tid; i < len; i += kThreads * kIds) {
      int32_t id[kIds];
#pragma unroll
      for (int k = 0; k < kIds; ++k) id[k] = i + k * kThreads < len ? ids[i + k * kThreads] : -1;
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        const uint32_t at = (uint32_t)id[k] - (uint32_t)lo;  // (lo + n <= 2^30: negative ids lie behind)
        if (at < (uint32_t)n) f(pad + at, i + k * kThreads);
      }
    }
  };
  if (counts) {
    const int len = r.history_lens ? clamp_int(r.history_lens[row], 0, r.history_len) : r.history_len;
    const int prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
    scan(r.history + (size_t)row * r.history_stride, len, [&](uint32_t at, int i) {
      if (i < prompt)
        atomicOr(&met[at], kPrompt);
      else
        atomicAdd(&met[at], 1u);
    });
  }
  if (biases)
    scan(r.bias_ids + (size_t)row * r.bias_stride, r.bias_len,
         [&](uint32_t at, int i) { atomicMax(&entry[at], (uint32_t)i + 1u); });
  __syncthreads();
  const float rep = r.repetition ? r.repetition[row] : 1.f, freq = r.frequency ? r.frequency[row] : 0.f,
              pres = r.presence ? r.presence[row] : 0.f;
  const float* bias = r.bias + (biases ? (size_t)row * r.bias_stride : 0);
  auto one = [&](float y, uint32_t m, uint32_t e, bool ok) -> float {
    if (m) {
      y = y > 0.f ? y / rep : y * rep;
      const float c = (float)(m & ~kPrompt);
      if (c > 0.f) y -= freq * c + pres;
    }
    if (e) y += bias[e - 1];
    return ok ? y : -INFINITY;
  };
  auto single = [&](int i) {  // a token ahead of the whole 16 bytes, or behind them
    const int t = lo + i;
    out[t] = (T)one((float)x[t], counts ? met[pad + i] : 0u, biases ? entry[pad + i] : 0u,
                    !masked || (allow[t >> 5] >> (t & 31) & 1u));
  };
  if (tid < head) single(tid);
  const bool lined = (uintptr_t)out % 16 == (uintptr_t)x % 16;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int i = head + (k * kThreads + tid) * VEC;
    if (i >= whole) break;
    const int t = lo + i;
    uint32_t bits = 0xffffffffu;
    if (masked) {
      const int at = t >> 5;
      const uint64_t two = (uint64_t)allow[min(at + 1, words - 1)] << 32 | allow[at];
      bits = (uint32_t)(two >> (t & 31));
    }
#pragma unroll
    for (int q = 0; q < VEC; q += 4) {
      const u32x4 m = counts ? *reinterpret_cast<const u32x4*>(met + pad + i + q) : none;
      const u32x4 e = biases ? *reinterpret_cast<const u32x4*>(entry + pad + i + q) : none;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[k][q + j] = (T)one((float)v[k][q + j], m[j], e[j], bits >> (q + j) & 1u);
    }
    if (lined) {
      *reinterpret_cast<Vec*>(out + t) = v[k];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[t + e] = v[k][e];
    }
  }
  if (whole + tid < n) single(whole + tid);
}

template <typename T, int U>
hipError_t launch_chunks(const AdjustArgs& a, int rows, hipStream_t st) {
  constexpr int CHUNK = chunk_of<T, U>();
  const size_t words = (size_t)CHUNK * ((a.r.history ? 1 : 0) + (a.r.bias_ids ? 1 : 0));
  // (the first chunk is up to VEC shorter than the others, a row's last place up to lead + VEC later)
  const int chunks = (int)(((long long)a.V + 16 + CHUNK - 1) / CHUNK);
  hipLaunchKernelGGL((logits_adjust_kernel<T, U>), dim3(chunks, rows), dim3(kThreads), words * 4, st, a);
  return hipGetLastError();
}

// Two loads a thread where that leaves 1024 workgroups, the lists being read once for more tokens
// (64 rows of 50,257 fp32 tokens, history 4096: 12.0 us, by one load 13.4; 336 of 32,768 bf16
// 15.6 and 15.7), one where the rows are few (one row of 50,257: 3.1, by two 3.5) or both lists take LDS
// from 16-bit rows, whose chunks are twice as long (256 of 50,257 bf16 with biases: 18.5, by two 23.0).
// An empty launch is 2 us of these, which are between the host's events (a profiler's clock has 12.0 and 16.4
// for the first two); the bytes alone are 5.5, 9.6 and 10.8 at the rate of a copy.
template <typename T>
hipError_t launch_adjust(const AdjustArgs& a, int rows, hipStream_t st) {
  constexpr int CHUNK = chunk_of<T, 2>();
  const bool crowded = sizeof(T) == 2 && a.r.history && a.r.bias_ids;
  return !crowded && (long long)rows * ((a.V + CHUNK - 1) / CHUNK) >= 1024 ? launch_chunks<T, 2>(a, rows, st)
                                                                           : launch_chunks<T, 1>(a, rows, st);
}

// Whether rows of V elements of `size` bytes at x and, elsewhere, at out share any: row by row, or one row of
// the one with another of the other.
bool rows_overlap(const void* x, const void* out, int size, int rows, int V, long long stride) {
  const __int128 apart = (__int128)(intptr_t)out - (intptr_t)x, step = (__int128)stride * size;
  const __int128 extent = step * (rows - 1) + (__int128)V * size;
  if (apart == 0 || apart >= extent || -apart >= extent) return false;
  const __int128 behind = (apart % step + step) % step;  // out's rows lie this far behind the next one of x
  return behind < (__int128)V * size || step - behind < (__int128)V * size;
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
  LLM_REQUIRE(!rows_overlap(logits, out, value_size(dtype), rows, V, stride),
              "logits_adjust: out must be the logits or not overlap them");
  const logits_rules& r = *rules;
  LLM_REQUIRE(!r.history || (r.history_len >= 0 && r.history_len <= kMostIds && (r.history_stride == 0 || r.history_stride >= r.history_len)),
              "logits_adjust: bad history_len / history_stride");
  LLM_REQUIRE(r.history || (!r.repetition && !r.frequency && !r.presence),
              "logits_adjust: penalties need a history");
  LLM_REQUIRE(!r.bias_ids == !r.bias, "logits_adjust: bias_ids and bias go together");
  LLM_REQUIRE(!r.bias_ids || (r.bias_len >= 0 && r.bias_len <= kMostIds && (r.bias_stride == 0 || r.bias_stride >= r.bias_len)),
              "logits_adjust: bad bias_len / bias_stride");
  LLM_REQUIRE(!r.allowed || r.num_masks > 0, "logits_adjust: num_masks must be positive");
  LLM_REQUIRE(!r.allowed || r.allowed_rows || r.num_masks >= rows,
              "logits_adjust: without allowed_rows every row needs a mask of its own");
  AdjustArgs a{logits, out, V, stride, r};
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
