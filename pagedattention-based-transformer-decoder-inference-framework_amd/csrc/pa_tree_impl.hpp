// The kernel of pa_tree.hpp, for the files that build it for one type of pool each.
#pragma once

#include <type_traits>

#include "pa_tree.hpp"

namespace llm {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Operands of 16 bits, as the products of one pool type take them.
template <bool BF>
struct Half {  // fp16
  // Probabilities enter times kP; a maximum moves when it grew by more than kGrow (log2 units), so
  // that they stay below 2^15: half of fp16's smallest step, 2^-25, is 2^-35 of the row's largest at most.
  static constexpr float kP = 2048.f;
  static constexpr float kGrow = 4.f;
  static constexpr uint32_t kOne = 0x3c00u;
  static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2));
  }
  static __device__ __forceinline__ f32x2 values(uint32_t w) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return f32x2{(float)h[0], (float)h[1]};
  }
};
template <>
struct Half<true> {  // bf16
  static constexpr float kP = 1.f;
  static constexpr float kGrow = 8.f;
  static constexpr uint32_t kOne = 0x3f80u;
  static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
  }
  static __device__ __forceinline__ f32x2 values(uint32_t w) {
    return f32x2{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
  }
};

// x, y as `PARTS` pairs of halves, each what the ones before it leave.
template <typename Hf, int PARTS>
__device__ __forceinline__ void split_parts(float x, float y, uint32_t (&w)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    w[i] = Hf::pair(x, y);
    if (i + 1 < PARTS) {
      asm("" : "+v"(w[i]));  // (the compiler would convert a second time for what is left)
      const f32x2 v = Hf::values(w[i]);
      x -= v[0];
      y -= v[1];
    }
  }
}

// Two 8-bit codes of a register (its low or high half) as fp16.
template <int KVT, bool HIGH>
__device__ __forceinline__ uint32_t two_codes(uint32_t w) {
  if constexpr (KVT == LLM_I8) {  // w ^ 0x80808080 before
    const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w, HIGH ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - f16x2{1152.f, 1152.f});
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HIGH));
  }
}

// One byte of two registers each, as two halves of bf16 (exact: codes have 8 bits at most).
__device__ __forceinline__ uint32_t two_bytes(uint32_t a, uint32_t b, int byte) {
  return Half<true>::pair((float)(int8_t)(a >> 8 * byte), (float)(int8_t)(b >> 8 * byte));
}
template <bool HIGH>
__device__ __forceinline__ uint32_t two_e4m3(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HIGH));
}

template <int KVT>
struct Raw {
  static constexpr bool QUANT = KVT == LLM_I8 || KVT == LLM_E4M3;
  static constexpr int ES = QUANT ? 1 : 2;
};

// An element of a pool that is not a number, as its own bits.
template <int KVT>
struct Unusable;
template <>
struct Unusable<LLM_F16> {
  static constexpr uint32_t kInf = 0x7c00u;
};
template <>
struct Unusable<LLM_BF16> {
  static constexpr uint32_t kInf = 0x7f80u;
};
template <>
struct Unusable<LLM_E4M3> {  // NaN alone
  static constexpr uint32_t kInf = 0x7fu;
};
// The elements of w with 0 in the place of infinities and NaNs.
template <int KVT>
__device__ __forceinline__ uint32_t usable(uint32_t w) {
  constexpr int BITS = KVT == LLM_E4M3 ? 8 : 16;
  constexpr uint32_t kInf = Unusable<KVT>::kInf, kAll = (1u << BITS) - 1u;
  uint32_t kept = 0;
#pragma unroll
  for (int s = 0; s < 32; s += BITS)
    if ((w >> s & kInf) != kInf) kept |= w & kAll << s;
  return kept;
}

// NQ, NP: parts of a query, of a probability; KW: waves that share the keys of the same rows, the others
// have rows of their own; MT: row tiles of a wave.
template <int KVT, int D, int NQ, int NP, int WAVES, int KW, int MT>
__global__ __launch_bounds__(64 * WAVES, D <= 128 ? 8 / WAVES : 1) void pa_tree_kernel(TreeArgs a) {
  constexpr bool QUANT = Raw<KVT>::QUANT;
  constexpr int ES = Raw<KVT>::ES, ROWB = D * ES;
  using Hf = Half<KVT == LLM_BF16>;           // of scores' products
  using Pf = Half<KVT == LLM_BF16 || QUANT>;  // of values'
  constexpr int NK = D / 32;          // steps of 32 dims of q.k
  constexpr int NKL = ROWB / 64;      // 16-byte loads of a key tile
  constexpr int ND = D / 16;          // tiles of the output, dims of a lane's keys
  constexpr int NV = ND * ES / 4;     // registers of them
  constexpr int RW = WAVES / KW;      // waves with rows of their own
  constexpr bool STAGED = KW < WAVES;  // keys shared by waves come through LDS
  constexpr bool AHEAD = ROWB < 512;  // a block ahead of the one in work fits the registers
  constexpr int CPR = ROWB / 16;      // 16-byte chunks of a key's row
  constexpr int kBlock = 2 * kTreeKeys * ROWB, kStage = KW * kBlock;  // bytes of a block's K and V, of KW blocks'
  static_assert(STAGED || MT == 1, "what is loaded ahead leaves no room for more tiles");
  // Loads into LDS reach its first 64 KiB: as many stages as fit there, with their scales behind them.
  constexpr int kScales = QUANT ? WAVES * 256 : 0;  // a wave's own 64: of K, of V
  constexpr int STAGES = !STAGED ? 1 : 65536 / (kStage + kScales) < 8 ? 65536 / (kStage + kScales) : 8;
  static_assert(!STAGED || STAGES >= 2, "a stage ahead");
  constexpr int kSums = WAVES * 16 * (D + 4) * 4, kLoads = STAGED ? STAGES * (kStage + kScales) : 0;
  __shared__ __align__(16) uint8_t s_mem[kLoads > kSums + WAVES * 128 ? kLoads : kSums + WAVES * 128];
  // behind the last block: the waves' sums
  float(*s_acc)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(s_mem);
  float(*s_ml)[16][2] = reinterpret_cast<float(*)[16][2]>(s_mem + kSums);

  const int lane = lane_id(), g = lane >> 4, c = lane & 15;
  const int w = wave_id_uniform(), kw = w % KW, rw = w / KW;
  // Workgroups go round the XCDs.  Staged, a pair's splits lie beside each other, so that a long row's are
  // dealt out over all of them (16 x 2 pairs of 168 rows, 11 splits 46.7 -> 39.5 us); else the pairs do,
  // which are many (64 x 16 pairs by splits 249 us, by pairs 241).
  const int pair = STAGED ? blockIdx.x / a.nsplit : blockIdx.x;
  const int split = STAGED ? blockIdx.x - pair * a.nsplit : blockIdx.y;
  const int b = pair / a.kv_heads, kvh = pair - b * a.kv_heads;
  const TreeRow tr = tree_row(a, b);
  const int first = (STAGED ? blockIdx.y : 0) * 16 * RW * MT, all_rows = tr.n * a.G;
  // the wave's tiles: rows row_of(t) .. + 15, of which the row has rows_of(t)
  auto row_of = [&](int t) { return first + 16 * (rw + RW * t); };
  auto rows_of = [&](int t) { return all_rows - row_of(t); };
  const int lo = split * tr.split_len;
  if (first >= all_rows || (split > 0 && lo >= tr.L)) return;
  const int hi = min(lo + tr.split_len, tr.L);
  const int beam = a.beam_ids ? a.beam_ids[b] : b;
  const bool has_beam = beam >= 0 && beam < a.num_beams;
  const int32_t* pt = a.table + ((size_t)(has_beam ? beam : 0) * a.kv_heads + kvh) * a.max_tiles;
  const int blocks = (hi - lo + kTreeKeys - 1) / kTreeKeys;

  // Lane i: where 16 keys lie, of the 64 halves from block `from` on: this wave's own blocks, or,
  // staged, all.
  constexpr int LOOKED = STAGED ? 32 / KW : 32;  // turns of a look-up
  bool found;
  uint64_t at_pool, at_scale;  // bytes into the pools, into the scales (of page 0 where there is none: masked)
  auto look_up = [&](int key) {
    const int tile = key / a.page_size, slot = key - tile * a.page_size;
    const int p = has_beam && key < hi ? pt[tile] : -1;
    found = p >= 0 && p < a.num_pages;
    const uint64_t page = found ? p : 0;
    at_pool = page * a.page_stride + (uint32_t)slot * ROWB;
    at_scale = (page * a.scale_stride + (uint32_t)slot) * 4;
  };
  auto lane64 = [](uint64_t x, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
  };
  auto look_up_from = [&](int i) {
    look_up(STAGED ? lo + i * KW * kTreeKeys + 16 * lane
                   : lo + ((i + (lane >> 1)) * KW + kw) * kTreeKeys + 16 * (lane & 1));
  };
  // ... the lane of half u of block `block` of turn i
  auto half_of = [&](int i, int block, int u) {
    return STAGED ? (i % LOOKED * KW + block) * 2 + u : (2 * i + u) & 63;
  };

  // a block's operands as they are in memory
  struct Block {
    u32x4 k[2][NKL];
    uint32_t v[2][4][NV];
    f32x4 ks[2], vs[2];
    uint32_t here;  // bit u: its u-th 16 keys have a page
  };
  auto load = [&](Block& x, int i) {  // this wave's i-th block
    x.here = (uint32_t)(__ballot(found) >> half_of(i, 0, 0)) & 3u;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint64_t base = lane64(at_pool, half_of(i, 0, u));
      const uint8_t *kp = a.k_pool + base, *vp = a.v_pool + base;
      if constexpr (QUANT) {
        if (a.k_scale) {
          const uint64_t at = lane64(at_scale, half_of(i, 0, u));
          const float* ks = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.k_scale) + at);
          const float* vs = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.v_scale) + at);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x.ks[u][r] = ks[4 * g + r];
            x.vs[u][r] = vs[4 * g + r];
          }
        } else {
          x.ks[u] = x.vs[u] = f32x4{1.f, 1.f, 1.f, 1.f};
        }
      }
#pragma unroll
      for (int l = 0; l < NKL; ++l)
        x.k[u][l] = *reinterpret_cast<const u32x4*>(kp + (uint32_t)(c * ROWB + 64 * l + 16 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint8_t* at = vp + (uint32_t)((4 * g + r) * ROWB + c * ND * ES);
        if constexpr (NV == 1) {
          x.v[u][r][0] = *reinterpret_cast<const uint32_t*>(at);
        } else if constexpr (NV == 2) {
          const u32x2 y = *reinterpret_cast<const u32x2*>(at);
          x.v[u][r][0] = y[0], x.v[u][r][1] = y[1];
        } else {
#pragma unroll
          for (int o = 0; o < NV; o += 4) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(at + 4 * o);
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[u][r][o + e] = y[e];
          }
        }
      }
    }
  };
  // Staged: the KW blocks of turn i into LDS, each K's 32 rows and then V's, 1 KiB an instruction
  // and lane l's 16 bytes at 16 l of it.  The chunks of a row are exchanged by the key's number, so
  // that 16 keys' chunks of one column lie in 16 different places of a bank's line.
  auto exchange = [](int key) {
    return CPR == 4    ? key >> 2 & 3
           : CPR == 8  ? key >> 1 & 7
           : CPR == 16 ? (key << 1 | key >> 3) & 15
                       : key & 15;
  };
  auto stage = [&](int i, int slot) {  // (slot: i % STAGES)
#pragma unroll
    for (int j = 0; j < kStage / 1024 / WAVES; ++j) {
      const int at = j * WAVES + w;               // of the instructions
      const int block = at / (kBlock / 1024);
      const int row = at * (1024 / ROWB) % kTreeKeys;  // its first
      const uint8_t* pool = at % (kBlock / 1024) < kBlock / 2048 ? a.k_pool : a.v_pool;
      const int key = (row & 15) + lane / CPR;
      load_to_lds(pool + lane64(at_pool, half_of(i, block, row >> 4)) +
                      (uint32_t)(key * ROWB + 16 * (lane % CPR ^ exchange(key))),
                  s_mem + slot * kStage + at * 1024);
    }
    if constexpr (QUANT) {  // this wave's block, lane l: of key l % 32
      const uint64_t s0 = lane64(at_scale, half_of(i, kw, 0)), s1 = lane64(at_scale, half_of(i, kw, 1));
      // (without scales anything, so that a stage has the same number of loads)
      const uint8_t* src = a.k_pool;
      if (a.k_scale)
        src = reinterpret_cast<const uint8_t*>(lane < 32 ? a.k_scale : a.v_scale) + (lane & 16 ? s1 : s0) + 4 * c;
      load_to_lds_dword(src, s_mem + STAGES * kStage + slot * kScales + w * 256);
    }
  };
  auto fetch = [&](Block& x, int slot) {  // this wave's block of the turn
    const uint8_t* k = s_mem + slot * kStage + kw * kBlock;
    const uint8_t* v = k + kBlock / 2;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int l = 0; l < NKL; ++l)
        x.k[u][l] = *reinterpret_cast<const u32x4*>(k + (16 * u + c) * ROWB + 16 * ((4 * l + g) ^ exchange(c)));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 4 * g + r;
        const uint8_t* row = v + (16 * u + key) * ROWB;
        if constexpr (NV < 4) {
          const uint8_t* at = row + 16 * (c * NV / 4 ^ exchange(key)) + c * NV % 4 * 4;
          if constexpr (NV == 1) {
            x.v[u][r][0] = *reinterpret_cast<const uint32_t*>(at);
          } else {
            const u32x2 y = *reinterpret_cast<const u32x2*>(at);
            x.v[u][r][0] = y[0], x.v[u][r][1] = y[1];
          }
        } else {
#pragma unroll
          for (int o = 0; o < NV; o += 4) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(row + 16 * ((c * NV + o) / 4 ^ exchange(key)));
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[u][r][o + e] = y[e];
          }
        }
      }
      if constexpr (QUANT) {
        const float* s = reinterpret_cast<const float*>(s_mem + STAGES * kStage + slot * kScales + w * 256) +
                         16 * u + 4 * g;
        const f32x4 one = {1.f, 1.f, 1.f, 1.f};
        x.ks[u] = a.k_scale ? *reinterpret_cast<const f32x4*>(s) : one;
        x.vs[u] = a.k_scale ? *reinterpret_cast<const f32x4*>(s + 32) : one;
      }
    }
  };

  // Queries: lane (g, c) holds row c's dims, those of the 16 bytes of K that it loads.
  u32x4 q[MT][NQ][NK];
  float qf[MT];  // what its scores are multiplied by, in log2 units: > 0, so that -infinity stays what it is
  int tok[MT];
  auto queries = [&] {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = c < rows_of(t) ? row_of(t) + c : 0;  // (no row: the first one's, not put out)
      tok[t] = row / a.G;
      const int h = kvh * a.G + row - tok[t] * a.G;
      const size_t at = ((size_t)b * a.N + tok[t]) * a.q_stride + (size_t)h * D;
      qf[t] = fmaxf(fabsf(a.scale2), 1e-37f);
      float x[NK][8];
      float most = 0.f;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const int d = ES == 1 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g;
        if (a.dtype == LLM_F32) {
          const float* p = static_cast<const float*>(a.q) + at + d;
          const f32x4 y = *reinterpret_cast<const f32x4*>(p), z = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[kk][e] = y[e], x[kk][4 + e] = z[e];
        } else {
          const u32x4 y = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x2 z = a.dtype == LLM_F16 ? Half<false>::values(y[e]) : Half<true>::values(y[e]);
            x[kk][2 * e] = z[0], x[kk][2 * e + 1] = z[1];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[kk][e]));
      }
      float up = a.scale2 < 0.f ? -1.f : 1.f;  // a scale's sign goes with the queries
      if constexpr (KVT != LLM_BF16) {
        int e = 0;
        (void)frexpf(rows_max(most), &e);  // most < 2^e
        e = clamp_int(e, -100, 128);
        up *= ldexpf(1.f, 14 - e);
        qf[t] = fmaxf(qf[t] * ldexpf(1.f, e - 14), 1e-37f);
      }
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[kk][i] *= up;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t part[NQ];
          split_parts<Hf, NQ>(x[kk][2 * i], x[kk][2 * i + 1], part);
#pragma unroll
          for (int p = 0; p < NQ; ++p) q[t][p][kk][i] = part[p];
        }
    }
  };

  f32x4 o[MT][ND];
  // what p is relative to (a whole number), the maximum (m + kLift < top + 1, top <= m + kRise), the sum
  float m[MT], top[MT], l[MT];
  // Weights of quantised values, p times the value's scale, enter the products in bf16 and so have all of fp32's
  // range: scales have any size, and what a row does not see or weigh must not take the others' bits.  p is 2^kLift
  // of a probability, so that scales up to kHuge leave fp32's normal numbers at neither end.  At a larger one
  // the row's weights are looked at; a row with one above 2^100 is in units of its own from then on.
  constexpr int kLift = QUANT ? 40 : 0;
  constexpr float kRise = (float)kLift + Pf::kGrow, kHuge = 0x1p50f;
  float per_unit[MT];    // <= 1
  bool units = false;    // one of them is not 1
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    m[t] = top[t] = kNegSentinel;
    l[t] = 0.f;
    per_unit[t] = 1.f;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) o[t][dd] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Keys key0 .. key0 + 31 that a drafted token sees, as far as its mask says.
  auto visible = [&](int token, int key0) -> uint32_t {
    const int j0 = key0 - tr.C;  // drafted token of the first key
    if (j0 <= -32) return 0xffffffffu;
    if (!a.mask) {
      const int k = token - j0;  // the last key it sees
      return k >= 31 ? 0xffffffffu : k < 0 ? 0u : (2u << k) - 1u;
    }
    const uint32_t* mask = a.mask + ((size_t)b * a.N + token) * a.mask_words;
    if (j0 < 0) return mask[0] << -j0 | ((1u << -j0) - 1u);
    const int at = j0 >> 5, sh = j0 & 31;
    const uint32_t w0 = at < a.mask_words ? mask[at] : 0u;
    const uint32_t w1 = at + 1 < a.mask_words ? mask[at + 1] : 0u;
    return sh ? w0 >> sh | w1 << (32 - sh) : w0;
  };
  // ... and those of them that anyone may: with a page, ahead of the row's end.
  auto present_of = [&](uint32_t here, int key0) -> uint32_t {
    uint32_t present = 0xffffffffu;
    if (!(here & 1u)) present &= 0xffff0000u;
    if (!(here & 2u)) present &= 0x0000ffffu;
    if (tr.L - key0 < 32) present &= (1u << (tr.L - key0)) - 1u;
    return present;
  };
  bool unusable = false;  // a drafted token's V or its scale has held infinities or NaNs

  auto attend = [&](Block& x, int i) {
    const int key0 = lo + (i * KW + kw) * kTreeKeys;
    const bool special = key0 + kTreeKeys > tr.C || x.here != 3u;
    uint32_t present = 0xffffffffu;
    if (special) {
      present = present_of(x.here, key0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool ok = present >> (16 * u + 4 * g + r) & 1u;
#pragma unroll
          for (int e = 0; e < NV; ++e) x.v[u][r][e] = ok ? x.v[u][r][e] : 0u;
          if constexpr (QUANT) x.vs[u][r] = ok ? x.vs[u][r] : 0.f;
        }
      if constexpr (KVT != LLM_I8)
        if (key0 + kTreeKeys > tr.C) {
          bool all = true;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int e = 0; e < NV; ++e) {
                const uint32_t kept = usable<KVT>(x.v[u][r][e]);
                all &= kept == x.v[u][r][e];
                x.v[u][r][e] = kept;
              }
          unusable |= !all;
        }
      if constexpr (QUANT)
        if (key0 + kTreeKeys > tr.C) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool ok = fabsf(x.vs[u][r]) < INFINITY;
              unusable |= !ok;
              x.vs[u][r] = ok ? x.vs[u][r] : 0.f;
            }
        }
    }
    const bool more = MT > 1 && rows_of(MT - 1) > 0;  // (a second tile without rows is left out)
    f32x4 s[MT][2];
    {
      u32x4 kf[2][NK];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          if constexpr (QUANT) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t y = x.k[u][kk / 2][2 * (kk & 1) + e] ^ (KVT == LLM_I8 ? 0x80808080u : 0u);
              kf[u][kk][2 * e] = two_codes<KVT, false>(y);
              kf[u][kk][2 * e + 1] = two_codes<KVT, true>(y);
            }
          } else {
            kf[u][kk] = x.k[u][kk];
          }
        }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && !more) break;
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < NQ; ++p)
#pragma unroll
          for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[t][u] = Hf::dot(kf[u][kk], q[t][p][kk], s[t][u]);
      }
    }
    if constexpr (QUANT) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && !more) break;
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] *= x.ks[u];
      }
    }
    if (special) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const uint32_t seen = present & visible(tok[t], key0);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!(seen >> (16 * u + 4 * g + r) & 1u)) s[t][u][r] = -INFINITY;
      }
    }
    bool grown = false;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t > 0 && !more) break;
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, s[t][u][r]);
      top[t] = fmaxf(top[t], rows_max(most) * qf[t]);
      grown |= top[t] > m[t] + kRise;
    }
    float largest = 0.f;  // scale
    if constexpr (QUANT) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) largest = fmaxf(largest, fabsf(x.vs[u][r]));
      grown |= largest > kHuge;
    }
    if (__any(grown)) {  // few blocks: sums move to the new maxima
      const bool huge = QUANT && (units || __any(largest > kHuge));
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && !more) break;
        const float next = ceilf(top[t]) - (float)kLift;
        const int rise = (int)fmaxf(m[t] - next, -1000.f);  // (<= 0; from the sentinel far below)
        const float corr = ldexpf(1.f, rise);
        l[t] *= corr;
        m[t] = next;
        float down = corr;
        if constexpr (QUANT)
          if (huge) {
            float weight = -1000.f;  // log2, rounded up
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float f = fabsf(x.vs[u][r]);
                if (f > 0.f && f < INFINITY)
                  weight = fmaxf(weight, fmaf(s[t][u][r], qf[t], -m[t]) + __builtin_amdgcn_frexp_expf(f));
                asm volatile("" : "+v"(weight));  // (one after the other: the registers are full)
              }
            const int was = 1 - __builtin_amdgcn_frexp_expf(per_unit[t]) + rise;
            const int to = max(max(was, 0), (int)ceilf(rows_max(weight)) - 100);
            down = ldexpf(1.f, was - to);
            per_unit[t] = ldexpf(1.f, -to);
          }
#pragma unroll
        for (int dd = 0; dd < ND; ++dd) o[t][dd] *= down;
      }
      if (huge) units = __any(per_unit[0] != 1.f || per_unit[MT - 1] != 1.f);
    }
    f32x4 p[MT][2];
    if constexpr (QUANT) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && !more) break;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[t][u][r] = __builtin_amdgcn_exp2f(fmaf(s[t][u][r], qf[t], -m[t]));
            l[t] += p[t][u][r];
          }
      }
      if (units) {  // (ahead of the scale, whose product with a probability may be no fp32 number)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) p[t][u] *= per_unit[t];
      }
    }
    u32x4 ph[MT][NP];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t > 0 && !more) break;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 2 * hf + e;
            if constexpr (QUANT) {
              w[e] = p[t][u][r] * x.vs[u][r];
            } else {
              w[e] = __builtin_amdgcn_exp2f(fmaf(s[t][u][r], qf[t], -m[t]));
              l[t] += w[e];
              w[e] *= Pf::kP;
            }
          }
          uint32_t part[NP];
          split_parts<Pf, NP>(w[0], w[1], part);
#pragma unroll
          for (int i = 0; i < NP; ++i) ph[t][i][2 * u + hf] = part[i];
        }
    }
    // V^T: the 8 keys' dims exchanged to 8 keys of one dim, a register of each at a time.
    constexpr int DIMS = 4 / ES;
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      u32x4 vf[DIMS];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // keys 2 hf, 2 hf + 1 of the four
          const uint32_t v0 = x.v[u][2 * hf][e], v1 = x.v[u][2 * hf + 1][e];
          if constexpr (KVT == LLM_I8) {
#pragma unroll
            for (int d = 0; d < 4; ++d) vf[d][2 * u + hf] = two_bytes(v0, v1, d);
          } else if constexpr (KVT == LLM_E4M3) {
            const uint32_t lo2 = __builtin_amdgcn_perm(v1, v0, 0x05010400u);
            const uint32_t hi2 = __builtin_amdgcn_perm(v1, v0, 0x07030602u);
            vf[0][2 * u + hf] = two_e4m3<false>(lo2);
            vf[1][2 * u + hf] = two_e4m3<true>(lo2);
            vf[2][2 * u + hf] = two_e4m3<false>(hi2);
            vf[3][2 * u + hf] = two_e4m3<true>(hi2);
          } else {
            vf[0][2 * u + hf] = __builtin_amdgcn_perm(v1, v0, 0x05040100u);
            vf[1][2 * u + hf] = __builtin_amdgcn_perm(v1, v0, 0x07060302u);
          }
        }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && !more) break;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int d = 0; d < DIMS; ++d) o[t][DIMS * e + d] = Pf::dot(vf[d], ph[t][i], o[t][DIMS * e + d]);
      }
    }
  };

  // Turns; staged, waves without rows, or without a block in the last one, take their part in the loads.
  const int mine = STAGED ? (blocks + KW - 1) / KW
                          : blocks > kw ? (blocks - kw + KW - 1) / KW : 0;
  if (mine > 0) {
    look_up_from(0);
    Block x;
    if constexpr (STAGED) {
      constexpr int LOADS = kStage / 1024 / WAVES + (QUANT ? 1 : 0);  // of a wave and stage
      uint64_t there = 0, before = 0;  // the halves looked up last, and those before, that have a page
      auto start = [&](int i, int slot) {
        if (i % LOOKED == 0) {
          if (i) look_up_from(i);
          before = there;
          there = __ballot(found);
        }
        stage(i, slot);
      };
      const int ahead = min(STAGES - 1, mine);
      for (int i = 0; i < ahead; ++i) start(i, i);
      queries();  // (while the first blocks come)
      int slot = 0, next = STAGES - 1;
      for (int i = 0; i < mine; ++i) {
        if (i + STAGES - 1 <= mine)
          wait_lds_loads<LOADS*(STAGES - 2)>();
        else
          wait_lds_loads();
        barrier_only();  // block i has landed, block i - 1 is read out
        const int last = min(i + STAGES - 1, mine - 1);
        if (i + STAGES - 1 < mine) start(last, next);
        if (rows_of(0) > 0 && i * KW + kw < blocks) {
          x.here = (uint32_t)((last / LOOKED == i / LOOKED ? there : before) >> half_of(i, kw, 0)) & 3u;
          fetch(x, slot);
          attend(x, i);
        }
        next = slot;
        slot = slot + 1 == STAGES ? 0 : slot + 1;
      }
      __syncthreads();  // the sums take the blocks' place
    } else if constexpr (AHEAD) {
      Block y;
      load(x, 0);
      queries();
      for (int i = 0; i < mine; i += 2) {
        if (i + 1 < mine) load(y, i + 1);
        attend(x, i);
        if (i + 1 >= mine) break;
        if (i + 2 < mine) {
          if (((i + 2) & 31) == 0) look_up_from(i + 2);
          load(x, i + 2);
        }
        attend(y, i + 1);
      }
    } else {
      queries();
      for (int i = 0; i < mine; ++i) {
        if (i && (i & 31) == 0) look_up_from(i);
        load(x, i);
        attend(x, i);
      }
    }
  }
  if (__any(unusable)) {
    // The rows that see them get what the products left out: sums of ones count them.
    for (int i = max((tr.C - lo) / (KW * kTreeKeys) - 1, 0); i < mine; ++i) {
      const int key0 = lo + (i * KW + kw) * kTreeKeys;
      if (key0 + kTreeKeys <= tr.C || key0 >= hi) continue;
      look_up(key0 + 16 * (lane & 1));
      const uint32_t present = present_of((uint32_t)__ballot(found) & 3u, key0);
      u32x4 one[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const uint32_t seen = present & visible(tok[t], key0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t two = seen >> (16 * (e / 2) + 4 * g + 2 * (e % 2));
          one[t][e] = (two & 1u ? Hf::kOne : 0u) | (two & 2u ? Hf::kOne << 16 : 0u);
        }
      }
#pragma unroll
      for (int dd = 0; dd < ND; ++dd) {
        u32x4 plus, minus;  // +infinity or NaN, -infinity or NaN
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          plus[e] = minus[e] = 0;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int u = e / 2, key = 4 * g + 2 * (e % 2) + s;
            if (!(present >> (16 * u + key) & 1u)) continue;
            const uint8_t* at = a.v_pool + lane64(at_pool, u) + (uint32_t)(key * ROWB + (c * ND + dd) * ES);
            const uint32_t x = ES == 1 ? *at : *reinterpret_cast<const uint16_t*>(at);
            constexpr uint32_t kSign = ES == 1 ? 0x80u : 0x8000u;
            bool bad = false, nan = false, minus_of = (x & kSign) != 0;
            if constexpr (KVT != LLM_I8) {
              constexpr uint32_t kInf = Unusable<KVT>::kInf;
              bad = (x & kInf) == kInf, nan = ES == 1 ? bad : (x & (kSign - 1u)) > kInf;
            }
            if constexpr (QUANT)
              if (a.v_scale) {
                const float f = *reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.v_scale) +
                                                                lane64(at_scale, u) + 4 * key);
                bad |= !(fabsf(f) < INFINITY);
                nan |= f != f || !(KVT == LLM_I8 ? x : x & (kSign - 1u));  // (infinity times 0)
                minus_of ^= f < 0.f;
              }
            if (bad && (nan || !minus_of)) plus[e] |= Hf::kOne << 16 * s;
            if (bad && (nan || minus_of)) minus[e] |= Hf::kOne << 16 * s;
          }
        }
        const f32x4 none = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const f32x4 up = Hf::dot(plus, one[t], none), down = Hf::dot(minus, one[t], none);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            o[t][dd][r] += (up[r] > 0.f ? INFINITY : 0.f) - (down[r] > 0.f ? INFINITY : 0.f);
        }
      }
    }
  }

  // The sums of a tile's waves, relative to the largest maximum of the row.
  // a row, ND of its dims; the first 256 threads take a tile, the others the next
  const int rr = threadIdx.x >> 4 & 15, part = threadIdx.x & 15, mine_of = threadIdx.x >> 8;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const float back = __builtin_amdgcn_exp2f(m[t] - top[t]);
    const float sum = add(with_lane32(add(with_lane16(l[t] * back))));
    const float f = ldexpf(back * (1.f / Pf::kP), 1 - __builtin_amdgcn_frexp_expf(per_unit[t]));
    if (t) __syncthreads();  // the tiles before are read
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int dd = 0; dd < ND; dd += 4)
        *reinterpret_cast<f32x4*>(&s_acc[w][c][(4 * g + r) * ND + dd]) =
            f32x4{o[t][dd][r] * f, o[t][dd + 1][r] * f, o[t][dd + 2][r] * f, o[t][dd + 3][r] * f};
    if (g == 0) {
      s_ml[w][c][0] = top[t];
      s_ml[w][c][1] = sum;
    }
    __syncthreads();
#pragma unroll 1  // (a launch finds its code in no cache)
    for (int pair_of = 0; pair_of < RW; pair_of += WAVES / 4) {
      const int tile = pair_of + mine_of;
      const int row = first + 16 * (tile + RW * t) + rr;
      if (tile >= RW || row >= all_rows) break;
      float M = kNegSentinel;
#pragma unroll
      for (int v = tile * KW; v < tile * KW + KW; ++v) M = fmaxf(M, s_ml[v][rr][0]);
      float all = 0.f, r[ND] = {};
#pragma unroll
      for (int v = tile * KW; v < tile * KW + KW; ++v) {
        const float weight = __builtin_amdgcn_exp2f(s_ml[v][rr][0] - M);
        all = fmaf(s_ml[v][rr][1], weight, all);
#pragma unroll
        for (int e = 0; e < ND; ++e) r[e] = fmaf(s_acc[v][rr][part * ND + e], weight, r[e]);
      }
      const int token = row / a.G, h = kvh * a.G + row - token * a.G;
      if (a.nsplit > 1) {
        const size_t at = (((size_t)b * a.N + token) * a.H + h) * a.nsplit + split;
#pragma unroll
        for (int e = 0; e < ND; e += 4)
          *reinterpret_cast<f32x4*>(a.acc + at * D + part * ND + e) = f32x4{r[e], r[e + 1], r[e + 2], r[e + 3]};
        if (part == 0) {
          a.ml[2 * at] = M;
          a.ml[2 * at + 1] = all;
        }
      } else {
        const float inv = 1.f / (all + 1e-6f);
        const size_t at = ((size_t)b * a.N + token) * a.out_stride + (size_t)h * D + part * ND;
#pragma unroll
        for (int e = 0; e < ND; e += 4) {
          const f32x4 y = f32x4{r[e], r[e + 1], r[e + 2], r[e + 3]} * inv;
          if (a.dtype == LLM_F32)
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at + e) = y;
          else
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at + e) =
                a.dtype == LLM_F16 ? u32x2{Half<false>::pair(y[0], y[1]), Half<false>::pair(y[2], y[3])}
                                   : u32x2{Half<true>::pair(y[0], y[1]), Half<true>::pair(y[2], y[3])};
        }
      }
    }
  }
}

// tiles: row tiles of a workgroup (tree_tiles).
template <int KVT, int D, int NQ, int NP>
hipError_t launch_tree_tiles(const TreeArgs& a, int tiles, dim3 grid, hipStream_t st) {
  constexpr int MT = tree_wave_tiles(D, NQ), MOST = tree_most_waves(D);
  if (tiles == 1 && a.waves == MOST)
    hipLaunchKernelGGL((pa_tree_kernel<KVT, D, NQ, NP, MOST, MOST, 1>), grid, dim3(64 * MOST), 0, st, a);
  else if (tiles == 1)
    hipLaunchKernelGGL((pa_tree_kernel<KVT, D, NQ, NP, 4, 4, 1>), grid, dim3(256), 0, st, a);
  else if (tiles == 4 * MT)
    hipLaunchKernelGGL((pa_tree_kernel<KVT, D, NQ, NP, 4, 1, MT>), grid, dim3(256), 0, st, a);
  else if constexpr (MT == 2)
    hipLaunchKernelGGL((pa_tree_kernel<KVT, D, NQ, NP, 4, 2, MT>), grid, dim3(256), 0, st, a);
  else
    return hipErrorInvalidValue;
  return hipGetLastError();
}

template <int KVT, int NQ, int NP>
hipError_t launch_tree_dim(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return D == 64    ? launch_tree_tiles<KVT, 64, NQ, NP>(a, tiles, grid, st)
         : D == 128 ? launch_tree_tiles<KVT, 128, NQ, NP>(a, tiles, grid, st)
                    : launch_tree_tiles<KVT, 256, NQ, NP>(a, tiles, grid, st);
}

// Weights are two parts of 11 bits over fp16 pools, of 8 else and then three for fp32 results (two are off
// by 2^-17, eight times what fp32 sums of the products are).  One of fp16 for results in bf16, whose own
// rounding is by up to 2^-8, would be off by 2^-11 of every weight, which shows where values cancel: 1e-4
// beside a result of 4e-5.  fp16 pools' parts drop what is below 2^-35 of the row's largest weight; a third
// one in bf16, values too, would keep it (fp32 results, 26 x 4 x 228 rows of 64 over up to 8000 tokens: 161 -> 202
// us; one row of 128 32.5 -> 34).
template <int KVT>
hipError_t launch_tree_parts(const TreeArgs& a, int D, int tiles, dim3 grid, hipStream_t st) {
  return a.dtype == LLM_F32   ? launch_tree_dim<KVT, tree_parts(KVT, LLM_F32), KVT == LLM_F16 ? 2 : 3>(a, D, tiles, grid, st)
         : a.dtype == LLM_F16 ? launch_tree_dim<KVT, tree_parts(KVT, LLM_F16), 2>(a, D, tiles, grid, st)
                              : launch_tree_dim<KVT, tree_parts(KVT, LLM_BF16), 2>(a, D, tiles, grid, st);
}

}  // namespace
}  // namespace llm
