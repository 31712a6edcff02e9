// One wave's step of attention with K and V taken straight from memory into matrix operands: 32 keys (or 64)
// against NQ blocks of 16 query rows, no LDS.  The building block of the decoding kernel, where K and V are
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
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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

// D: head dim rounded up to 64 or 128; CACHE8: K and V are e4m3; NS: 32-key blocks per step; NQ: 16-query blocks
template <int D, int EK, bool CACHE8, int NS, int NQ>
struct Step {
  static constexpr int kKS = D / 32;             // k-steps of a score tile
  static constexpr int kE = D / 16;              // columns of V per lane
  static constexpr int kKeys = 32 * NS;          // keys per step
  static constexpr int kElem = CACHE8 ? 1 : 2;   // bytes of a K or V element
  typedef typename Words<2 * kElem>::type KWord;             // 8 elements of K
  typedef typename Words<kE * kElem / 4>::type VWord;        // kE elements of V

  // K and V of one step, as loaded
  struct Block {
    KWord k[2 * NS][kKS];
    VWord v[NS][8];
    uint64_t valid;  // bit i: key i of the step exists (wave-uniform)
  };
  struct State {
    f32x4 o[NQ][kE];
    float m[NQ], l[NQ];  // l: this lane's keys only
  };

  static __device__ __forceinline__ void clear(State& st) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int e = 0; e < kE; ++e) st.o[q][e] = f32x4{0.f, 0.f, 0.f, 0.f};
      st.m[q] = kMinusInf;
      st.l[q] = 0.f;
    }
  }

  // key of the step that lane group g multiplies as element j of sub-block s
  static __device__ __forceinline__ int v_key(int s, int g, int j) {
    return 32 * s + 4 * g + (j < 4 ? j : 12 + j);
  }

  static __device__ __forceinline__ u32x4 k_operand(const KWord& w) {
    if constexpr (CACHE8) {
      const u32x2 a = from_e4m3<EK>(word(w, 0)), b = from_e4m3<EK>(word(w, 1));
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      return w;
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

  // `c`: softmax scale * log2 e (and what a unit of an 8-bit K stands for).
  // LIMIT: the lane's query sees the first `limit` keys of the step only (fewer than one: none).
  template <bool LIMIT = false>
  static __device__ __forceinline__ void run(State& st, const Block& b, const u32x4 (&qf)[NQ][kKS], float c, int lane,
                                             int limit = kKeys) {
    static_assert(!LIMIT || NQ == 1, "one limit per lane");
    const int n16 = lane & 15, g = lane >> 4;
    constexpr uint64_t kAll = NS == 1 ? 0xffffffffull : ~0ull;
    const bool whole = b.valid == kAll;
    const bool cut = LIMIT && __builtin_amdgcn_ballot_w64(limit < kKeys) != 0;
    float pr[LIMIT ? 2 * NS : 1][4];  // probabilities, for the values that take the way around the matrix product
    u32x4 ph[NQ][NS], pl[NQ][NS];
    {
      f32x4 s[NQ][2 * NS];
#pragma unroll
      for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
        for (int ks = 0; ks < kKS; ++ks) {
          const u32x4 a = k_operand(b.k[t][ks]);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            s[q][t] = mfma<EK>(a, qf[q][ks], ks == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[q][t]);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int t = 0; t < 2 * NS; ++t) s[q][t] *= c;
        if (!whole) {
#pragma unroll
          for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (!((b.valid >> (16 * t + 4 * g + i)) & 1)) s[q][t][i] = kMinusInf;
            }
          }
        }
        if constexpr (LIMIT) {
          if (cut) {
#pragma unroll
            for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (16 * t + 4 * g + i >= limit) s[q][t][i] = kMinusInf;
              }
            }
          }
        }
        float mx = s[q][0][0];
#pragma unroll
        for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[q][t][i]);
        }
        const float m_new = fmaxf(st.m[q], quad_max(mx));
        // nothing visible so far: any finite reference will do (every p is 0)
        const float ref = m_new == kMinusInf ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(st.m[q] - ref);
        st.m[q] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * NS; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[q][t][i] = __builtin_amdgcn_exp2f(s[q][t][i] - ref);
            sum += s[q][t][i];
            if constexpr (LIMIT) pr[t][i] = s[q][t][i];
          }
        }
        st.l[q] = st.l[q] * alpha + sum;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
          for (int e = 0; e < kE; ++e) st.o[q][e] *= alpha;
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float x = s[q][2 * n + w / 2][2 * (w & 1)], y = s[q][2 * n + w / 2][2 * (w & 1) + 1];
            const uint32_t hi = pack2<EK>(x, y);
            ph[q][n][w] = hi;
            if constexpr (!LIMIT) {
              const f32x2 back = unpack2<EK>(hi);
              pl[q][n][w] = pack2<EK>(x - back[0], y - back[1]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      // the lane's 8 keys x kE columns as 16-bit words [key][column pair]
      uint32_t r[8][kE / 2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // a key that does not exist has p = 0, but what lies in its place may be NaN or infinite
        const bool there = whole || ((b.valid >> v_key(n, g, j)) & 1);
#pragma unroll
        for (int w = 0; w < (CACHE8 ? kE / 4 : kE / 2); ++w) {
          const uint32_t x = there ? word(b.v[n][j], w) : 0u;
          if constexpr (CACHE8) {
            const u32x2 y = from_e4m3<EK>(x);
            r[j][2 * w] = y[0];
            r[j][2 * w + 1] = y[1];
          } else {
            r[j][w] = x;
          }
        }
      }
      if constexpr (LIMIT) {
        // A key that some of the 16 queries see and others do not: 0 * infinity in the product would reach
        // those that do not.  Such values go around it, to the queries that see them only.  (Only steps with a
        // limit inside look, and these are few: 3 % of the work at 2048 keys.)
        if (cut) {
          uint32_t odd = 0;  // bit j: this lane's part of key j is not finite throughout
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int w = 0; w < kE / 2; ++w) {
              if (not_finite(r[j][w]) || not_finite(r[j][w] >> 16)) odd |= 1u << j;
            }
          }
          if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint64_t lanes = __builtin_amdgcn_ballot_w64((odd >> j) & 1);
#pragma unroll 1
              for (int from = 0; from < 4; ++from) {
                if (((lanes >> (16 * from)) & 0xffffu) == 0) continue;
                const float p = __shfl(pr[2 * n + j / 4][j % 4], n16 + 16 * from);
                const bool sees = v_key(n, from, j) < limit;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                  for (int w = 0; w < kE / 2; ++w) {
                    const uint32_t x = (uint32_t)__shfl((int)r[j][w], 16 * from + 4 * g + i);
                    const f32x2 v = unpack2<EK>(x);
                    if (sees && not_finite(x)) st.o[0][2 * w][i] += p * v[0];
                    if (sees && not_finite(x >> 16)) st.o[0][2 * w + 1][i] += p * v[1];
                  }
                }
              }
            }
            drop_not_finite(r);
          }
        }
      }
      // An infinite v: its product with the low part of p (of either sign, or zero) would make NaN of it.  The low part
      // multiplies finite values only.
      bool both = true;
      if constexpr (!LIMIT) {
        uint16x2 top = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int w = 0; w < kE / 2; ++w) {
            top = __builtin_elementwise_max(top, __builtin_bit_cast(uint16x2, r[j][w] & 0x7fff7fffu));
          }
        }
        constexpr uint16_t kInfinity = EK == kBfloat ? 0x7f80 : 0x7c00;
        both = __builtin_amdgcn_ballot_w64(top[0] >= kInfinity || top[1] >= kInfinity) == 0;
      }
      auto multiply = [&](auto high, auto low) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          u32x4 a;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            a[w] = __builtin_amdgcn_perm(r[2 * w + 1][e / 2], r[2 * w][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
          }
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if constexpr (decltype(high)::value) st.o[q][e] = mfma<EK>(a, ph[q][n], st.o[q][e]);
            if constexpr (decltype(low)::value) st.o[q][e] = mfma<EK>(a, pl[q][n], st.o[q][e]);
          }
        }
      };
      constexpr std::true_type yes{};
      constexpr std::false_type no{};
      if constexpr (LIMIT) {
        multiply(yes, no);
      } else if (both) {
        multiply(yes, yes);
      } else {
        multiply(yes, no);
        drop_not_finite(r);
        multiply(no, yes);
      }
    }
  }
};

}  // namespace direct
}  // namespace flash_hip
