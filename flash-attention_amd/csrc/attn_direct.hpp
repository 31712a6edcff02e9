// One wave's step of attention with K and V taken straight from memory into matrix operands: 32 keys (or 64)
// against 16 query rows, no LDS.  The building block of the decoding kernel, where K and V are
// read once and never shared between waves.
//
// Mathematics, per query (column) q and key j, in the exp2 domain (c = softmax_scale * log2 e):
//   s_j = c * k_j . q,   m' = max(m, max_j s_j),   p_j = 2^(s_j - m'),
//   l  <- l * 2^(m - m') + sum_j p_j,   o <- o * 2^(m - m') + sum_j p_j v_j.
// Both products are transposed (S^T = K Q^T, O^T = V^T P^T), so that a lane owns one query column: maximum, sum
// and rescale are per-lane scalars, joined over the four lanes of a query by two permlane swaps.
//
// Fragments of v_mfma_f32_16x16x32 (lane: n = lane & 15, g = lane >> 4):
//   A (16 x 32): row n, k = 8g + j.   B (32 x 16): k = 8g + j, column n.   C/D: column n, rows 4g + i.
//   S^T:  A = K[key n][16-byte chunk 4 ks + g], as one 128-bit load (64 bytes of each of 16 rows per instruction);
//         B = Q with the same chunk.  The lane ends up with keys 4g + i of its query.
//   P^T:  element j < 4 of a 32-key block is key 4g + j of its first 16 keys, j >= 4 key 4g + j - 4 of its last
//         16: the two S^T tiles converted in place, no lane movement.
//   O^T:  A = V^T with that key order.  A lane loads E = D / 16 consecutive columns of each of its 8 keys (whole
//         rows per 16 lanes) and transposes the 8 x E block in registers (E * 4 v_perm_b32): row n of A number e
//         is column E n + e.  O^T tile e then holds columns E (4g + i) + e: E consecutive ones over e.
// Where K and V come from memory for one use (decoding), P is kept as a sum of two 16-bit values, p = hi + lo with
// |lo| <= 2^-8 p (bf16) or 2^-11 p (fp16), and both are multiplied: the second product costs matrix cycles that a kernel
// bound by memory has to spare, and the result carries the rounding of the output alone.  For prompts P is rounded once.
// fp16 has no bits below 2^-24, and a long tail behind one leading key consists of small weights: they are raised by 2^15
// (the largest, 1, stays below 65504) before they are rounded, which keeps them down to 2^-39 of the largest.  bfloat16
// reaches as far as fp32, and the sum of a few values near its end does not fit fp32: its weights are lowered by 2^31,
// one for each of the 2^30 positions that there may be.  The sums of products carry that factor until they are divided by
// l, which does not.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "serving_index.hpp"

namespace flash_hip {
namespace direct {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr int kHalf = 0;      // IEEE binary16 operands
constexpr int kBfloat = 1;    // bfloat16 operands
constexpr float kMinusInf = -__builtin_huge_valf();
template <int EK>
constexpr float kRaise = EK == kHalf ? 0x1p15f : 0x1p-31f;  // of the weights in the second product

// N 32-bit words, as loaded
template <int N>
struct Words;
template <>
struct Words<1> {
  typedef uint32_t type;
};
template <>
struct Words<2> {
  typedef u32x2 type;
};
template <>
struct Words<4> {
  typedef u32x4 type;
};
__device__ __forceinline__ uint32_t word(uint32_t x, int) { return x; }
__device__ __forceinline__ uint32_t word(const u32x2& x, int i) { return x[i]; }
__device__ __forceinline__ uint32_t word(const u32x4& x, int i) { return x[i]; }

template <int EK>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (EK == kBfloat) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
}

// two floats to packed 16-bit values, round to nearest even, and back
template <int EK>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 x = {lo, hi};
  if constexpr (EK == kBfloat) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, b16x2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, h16x2));
}
template <int EK>
__device__ __forceinline__ f32x2 unpack2(uint32_t w) {
  if constexpr (EK == kBfloat) return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  return __builtin_convertvector(__builtin_bit_cast(h16x2, w), f32x2);
}

// Four e4m3 values (a word) to four 16-bit values (two words).  Exact: both 16-bit types hold every e4m3 value.
template <int EK>
__device__ __forceinline__ u32x2 from_e4m3(uint32_t w) {
  if constexpr (EK == kBfloat) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
  }
}

// maximum / sum over the four lanes (g = 0..3) that share a query, in all four, on the vector ALU; always joined in
// the same order
__device__ __forceinline__ float quad_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t m = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto t = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t m = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// inclusive sum over the 64 lanes of a wave, by the vector ALU's own lane shifts (within rows of 16 lanes, then the last
// lane of a row into the next, and lane 31 into the upper half)
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, true);
  return x;
}

// D: head dim rounded up to 64 or 128; CACHE8: K and V are e4m3; NS: 32-key blocks per step
template <int D, int EK, bool CACHE8, int NS>
struct Step {
  static constexpr int kKS = D / 32;             // k-steps of a score tile
  static constexpr int kE = D / 16;              // columns of V per lane
  static constexpr int kKeys = 32 * NS;          // keys per step
  static constexpr int kElem = CACHE8 ? 1 : 2;   // bytes of a K or V element
  static constexpr int kKLoads = CACHE8 ? kKS / 2 : kKS;     // 16-byte loads of a lane per K tile
  typedef typename Words<kE * kElem / 4>::type VWord;        // kE elements of V

  // K and V of one step, as loaded: [16-key tile], [32-key block][key]
  typedef u32x4 KBlock[2 * NS][kKLoads];
  typedef VWord VBlock[NS][8];

  struct State {
    f32x4 o[kE];
    float m, l;  // l: this lane's keys only
  };

  static __device__ __forceinline__ void clear(State& st) {
#pragma unroll
    for (int e = 0; e < kE; ++e) st.o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m = kMinusInf;
    st.l = 0.f;
  }

  static __device__ __forceinline__ int column(int ks, int g) { return k_column(CACHE8, ks, g); }
  // element (of a row) where load i of a lane's K begins
  static __device__ __forceinline__ int load_column(int i, int g) { return CACHE8 ? column(2 * i, g) : column(i, g); }
  // key of the step that lane group g multiplies as element j of block s
  static __device__ __forceinline__ int v_key(int s, int g, int j) { return 32 * s + 4 * g + (j < 4 ? j : 12 + j); }

  static __device__ __forceinline__ u32x4 k_operand(const u32x4 (&k)[kKLoads], int ks) {
    if constexpr (CACHE8) {
      const u32x2 a = from_e4m3<EK>(k[ks / 2][2 * (ks & 1)]), b = from_e4m3<EK>(k[ks / 2][2 * (ks & 1) + 1]);
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      return k[ks];
    }
  }

  static __device__ __forceinline__ bool not_finite(uint32_t half) {
    constexpr uint32_t kExponent = EK == kBfloat ? 0x7f80u : 0x7c00u;
    return (half & kExponent) == kExponent;
  }
  static __device__ __forceinline__ void drop_not_finite(uint32_t (&r)[8][kE / 2]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int w = 0; w < kE / 2; ++w) {
        if (not_finite(r[j][w])) r[j][w] &= 0xffff0000u;
        if (not_finite(r[j][w] >> 16)) r[j][w] &= 0x0000ffffu;
      }
    }
  }

  // Bits of block n's keys, shifted so that bits 0..3 and 16..19 are the lane group's (the asm keeps the masked path, which
  // few steps take, from being worked into the others)
  static __device__ __forceinline__ uint32_t lane_bits(uint64_t valid, int n, int g) {
    uint32_t mine = (uint32_t)(valid >> (32 * n)) >> (4 * g);
    asm volatile("" : "+v"(mine));
    return mine;
  }

  // Scores of the step's keys, the running maximum and sum, and the weights for the second product.
  // `c`: softmax scale * log2 e (and what a unit of an 8-bit K stands for).  `valid`: bit i: key i of the step exists
  // (wave-uniform).  LIMIT: the lane's query sees the first `limit` keys of the step only (fewer than one: none).
  struct Weights {
    u32x4 hi[NS], lo[NS];
    float p[2 * NS][4];  // before they were rounded (LIMIT only)
  };
  template <bool LIMIT>
  static __device__ __forceinline__ void weigh(State& st, Weights& w, const KBlock& k, const u32x4 (&qf)[kKS], uint64_t valid, float c,
                                               int lane, int limit = kKeys) {
    const int g = lane >> 4;
    constexpr uint64_t kAll = NS == 1 ? 0xffffffffull : ~0ull;
    f32x4 s[2 * NS];
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const u32x4 a = k_operand(k[t], ks);
        s[t] = mfma<EK>(a, qf[ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[t]);
      }
    }
    const bool cut = LIMIT && __builtin_amdgcn_ballot_w64(limit < kKeys) != 0;
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) s[t] *= c;
    if (valid != kAll) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const uint32_t mine = lane_bits(valid, n, g);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((mine >> (16 * t + i)) & 1)) s[2 * n + t][i] = kMinusInf;
          }
        }
      }
    }
    if constexpr (LIMIT) {
      if (cut) {
#pragma unroll
        for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (16 * t + 4 * g + i >= limit) s[t][i] = kMinusInf;
          }
        }
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
    }
    const float m_new = fmaxf(st.m, quad_max(mx));
    // nothing visible so far: any finite reference will do (every p is 0)
    const float ref = m_new == kMinusInf ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(st.m - ref);
    st.m = m_new;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
        sum += s[t][i];
        s[t][i] *= kRaise<EK>;
        if constexpr (LIMIT) w.p[t][i] = s[t][i];
      }
    }
    st.l = st.l * alpha + sum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
      for (int e = 0; e < kE; ++e) st.o[e] *= alpha;
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[2 * n + i / 2][2 * (i & 1)], y = s[2 * n + i / 2][2 * (i & 1) + 1];
        w.hi[n][i] = pack2<EK>(x, y);
        if constexpr (!LIMIT) {
          const f32x2 back = unpack2<EK>(w.hi[n][i]);
          w.lo[n][i] = pack2<EK>(x - back[0], y - back[1]);
        }
      }
    }
  }

  // What lies in the place of a key that does not exist may be NaN or infinite, and its weight 0 would not help
  static __device__ __forceinline__ void clear_missing(VBlock& v, uint64_t valid, int lane) {
    constexpr uint64_t kAll = NS == 1 ? 0xffffffffull : ~0ull;
    if (valid == kAll) return;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const uint32_t mine = lane_bits(valid, n, lane >> 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!((mine >> (j < 4 ? j : 12 + j)) & 1)) v[n][j] = VWord{};
      }
    }
  }

  // the lane's 8 keys x kE columns of a block as 16-bit words [key][column pair]
  static __device__ __forceinline__ void v_words(uint32_t (&r)[8][kE / 2], const VWord (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int i = 0; i < (CACHE8 ? kE / 4 : kE / 2); ++i) {
        if constexpr (CACHE8) {
          const u32x2 y = from_e4m3<EK>(word(v[j], i));
          r[j][2 * i] = y[0];
          r[j][2 * i + 1] = y[1];
        } else {
          r[j][i] = word(v[j], i);
        }
      }
    }
  }
  template <bool HIGH, bool LOW>
  static __device__ __forceinline__ void multiply(State& st, const Weights& w, int n, const uint32_t (&r)[8][kE / 2]) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __builtin_amdgcn_perm(r[2 * i + 1][e / 2], r[2 * i][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
      }
      if constexpr (HIGH) st.o[e] = mfma<EK>(a, w.hi[n], st.o[e]);
      if constexpr (LOW) st.o[e] = mfma<EK>(a, w.lo[n], st.o[e]);
    }
  }

  // o += p v with both parts of p.  An infinite v turns into NaN this way (its product with the low part, of either sign
  // or zero); CAREFUL multiplies the low part with finite values only.
  template <bool CAREFUL>
  static __device__ __forceinline__ void accumulate(State& st, const Weights& w, const VBlock& v) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      uint32_t r[8][kE / 2];
      v_words(r, v[n]);
      if constexpr (CAREFUL) {
        multiply<true, false>(st, w, n, r);
        drop_not_finite(r);
        multiply<false, true>(st, w, n, r);
      } else {
        multiply<true, true>(st, w, n, r);
      }
    }
  }
  // whether a sum of this wave is NaN
  static __device__ __forceinline__ bool holds_nan(const State& st) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= st.o[e][i] != st.o[e][i];
    }
    return __builtin_amdgcn_ballot_w64(any) != 0;
  }

  // o += p v, p rounded once, for keys that some of the 16 queries see and others do not: 0 * infinity in the product
  // would reach those that do not.  Such values go around it, to the queries that see them only.
  static __device__ __forceinline__ void accumulate_limited(State& st, const Weights& w, const VBlock& v, int lane, int limit) {
    const int n16 = lane & 15, g = lane >> 4;
    const bool cut = __builtin_amdgcn_ballot_w64(limit < kKeys) != 0;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      uint32_t r[8][kE / 2];
      v_words(r, v[n]);
      if (cut) {
        uint32_t odd = 0;  // bit j: this lane's part of key j is not finite throughout
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int i = 0; i < kE / 2; ++i) {
            if (not_finite(r[j][i]) || not_finite(r[j][i] >> 16)) odd |= 1u << j;
          }
        }
        if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint64_t lanes = __builtin_amdgcn_ballot_w64((odd >> j) & 1);
#pragma unroll 1
            for (int from = 0; from < 4; ++from) {
              if (((lanes >> (16 * from)) & 0xffffu) == 0) continue;
              const float p = __shfl(w.p[2 * n + j / 4][j % 4], n16 + 16 * from);
              const bool sees = v_key(n, from, j) < limit;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int c = 0; c < kE / 2; ++c) {
                  const uint32_t x = (uint32_t)__shfl((int)r[j][c], 16 * from + 4 * g + i);
                  const f32x2 y = unpack2<EK>(x);
                  if (sees && not_finite(x)) st.o[2 * c][i] += p * y[0];
                  if (sees && not_finite(x >> 16)) st.o[2 * c + 1][i] += p * y[1];
                }
              }
            }
          }
          drop_not_finite(r);
        }
      }
      multiply<true, false>(st, w, n, r);
    }
  }
};

}  // namespace direct
}  // namespace flash_hip
