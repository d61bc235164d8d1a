// Device code shared by the attention kernels (attention.hip, packed_attention.hip, cached_attention.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels/flex_tile.h"

namespace cinn_hip_kernels {
namespace attention {

using flex::bf16x8;
using flex::f16x8;
using flex::f32x16;
using flex::f32x4;
using flex::LoadAny;
using flex::s16x4;
using flex::u32x4;

// [b][h][t][d] in any order of the first three: d is contiguous
struct Rows {
  const void* base;
  int64_t batch, head, row;  // strides in elements
};

template <typename T>
__device__ __forceinline__ const char* HeadOf(const Rows& r, int b, int h) {
  return static_cast<const char*>(r.base) + (b * r.batch + h * r.head) * (int64_t)sizeof(T);
}

// exp(|scale| (s - m)); the scale's sign has gone into the query (a scale of 0 too: there the query is zero and the
// factor 1, since 0 * -inf of a maximum not yet found or of a masked key is no number).  Full accuracy for fp32; v_exp_f32 (2^-22 or so) of one
// fused multiply-add where the result is rounded to 16 bits anyway.  -inf for m (no finite score so far) must not make
// -inf - -inf of scores.
template <typename T>
struct Exp {
  float c;
  __device__ __forceinline__ explicit Exp(float scale) : c(scale == 0.0f ? 1.0f : fabsf(scale) * 1.4426950408889634f) {}
  __device__ __forceinline__ float Base(float m) const { return m == -__builtin_inff() ? 0.0f : m * c; }
  __device__ __forceinline__ float operator()(float s, float base) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -base)); }
};
template <>
struct Exp<float> {
  float c;
  __device__ __forceinline__ explicit Exp(float scale) : c(scale == 0.0f ? 1.0f : fabsf(scale)) {}
  __device__ __forceinline__ float Base(float m) const { return m == -__builtin_inff() ? 0.0f : m; }
  __device__ __forceinline__ float operator()(float s, float base) const { return expf((s - base) * c); }
};

// Base for probabilities that matrix cores take in T: fp16 ones are held times 2^7, since below 2^-14 its places are 2^-24 for
// all, and many keys of little weight would be rounded away together.  With maxima that lag by 2^8 at most they stay below
// 2^15, and are off by 2^-32 of the largest or by half a step, whichever is more.
template <typename T>
__device__ __forceinline__ float HeldBase(const Exp<T>& ex, float m) {
  return __is_same(T, _Float16) ? ex.Base(m) - 7.0f : ex.Base(m);
}

// a chunk of the query, negated where the scale is negative, zero where it is zero
template <typename T>
__device__ __forceinline__ u32x4 Signed(u32x4 v, float scale) {
  if (scale == 0.0f) return u32x4{0, 0, 0, 0};
  return scale < 0.0f ? v ^ (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : v;
}

template <typename T>
struct Mma;
template <>
struct Mma<_Float16> {
  typedef f16x8 vec8;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  typedef bf16x8 vec8;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {  // four MFMAs of two k each: element e of the lane's chunk is k = e of its half of the wavefront
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
};

// How [keys][d] tiles lie in LDS: KAt(row, c) is where chunk c of a key's row starts, VAt(row, c) of a value's.
template <typename T, int D>
struct Shape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NC   = D * (int)sizeof(T) / 16;  // 16-byte chunks per row
  static constexpr int DT   = (D + 31) / 32;            // 32-row results of O^T
};

// Rows of floats apart, for tiles that are stored from registers.  K rows are read 16 bytes per lane, rows over lanes: an odd
// number of 16-byte chunks.  V rows, read as single floats: rows four apart fall into different quarters of the banks.
template <int D>
struct Padded : Shape<float, D> {
  using Shape<float, D>::NC, Shape<float, D>::DT, Shape<float, D>::F32;
  static constexpr int K_PITCH = NC * 16 + 16;
  static constexpr int V_PITCH = DT * 128 + 32;
  static __device__ __forceinline__ int KAt(int row, int c) { return row * K_PITCH + c * 16; }
  static __device__ __forceinline__ int VAt(int row, int c) { return row * V_PITCH + c * 16; }
};

// Rows behind one another, for tiles that loads write to LDS directly, 64 chunks in order per instruction; the chunks of a row
// change places instead.  K: eight rows' neighbouring chunks, which LDS serves together, lie in different sixteenths of the
// banks' 256 bytes.  V at VAt: four rows' 64 bytes in different quarters.
template <typename T, int D>
struct Dense : Shape<T, D> {
  using Shape<T, D>::NC, Shape<T, D>::DT, Shape<T, D>::F32;
  static constexpr int BYTES = 32 * NC * 16;  // a tile of 32 keys or values
  static constexpr bool POW2 = (NC & (NC - 1)) == 0;
  static __device__ __forceinline__ int Turn(int c, int by) { return POW2 ? c ^ by : (c + by >= NC ? c + by - NC : c + by); }
  static __device__ __forceinline__ int Back(int c, int by) { return POW2 ? c ^ by : (c < by ? c - by + NC : c - by); }
  static __device__ __forceinline__ int RowTurn(int row) {
    return NC % 16 == 0 ? 2 * (row & 7) : NC % 8 == 0 ? 2 * ((row >> 1) & 3) : 2 * ((row >> 2) & 1);
  }
  // four rows' 64 bytes, which a transposing read of 32 columns takes together, in different quarters
  static __device__ __forceinline__ int WideTurn(int row) {
    static_assert(!F32);
    return NC == 16 ? 4 * (row & 3) : NC == 8 ? 4 * ((row >> 1) & 1) : 0;
  }
  static __device__ __forceinline__ int KTurn(int row) {
    return NC % 16 == 0 ? row & 15 : NC % 8 == 0 ? (row >> 1) & 7 : (row >> 2) & 3;
  }
  static __device__ __forceinline__ int At(int row, int c) { return (row * NC + Turn(c, RowTurn(row))) * 16; }
  static __device__ __forceinline__ int KAt(int row, int c) { return (row * NC + Turn(c, KTurn(row))) * 16; }
  static __device__ __forceinline__ int VAt(int row, int c) { return (row * NC + Turn(c, WideTurn(row))) * 16; }
};

// the bits of a word of 32 keys below `count`
__device__ __forceinline__ unsigned Below(int count) { return count >= 32 ? ~0u : count <= 0 ? 0u : (1u << count) - 1; }

// registers that hold a lane's sixteen probabilities
template <typename T>
struct Held {
  static constexpr int COUNT = 2;
  typedef T type __attribute__((ext_vector_type(8)));
};
template <>
struct Held<float> {
  static constexpr int COUNT = 1;
  typedef f32x16 type;
};

// 32 queries of a wavefront, a lane of either half holding one: S^T = K Q^T leaves the lane 16 scores of its query, register
// r of key 8 (r / 4) + 4 half + r % 4, and O^T = V^T P^T sixteen sums of each 32 elements of d in the same order.
template <typename T, int D, class Layout>
struct Queries {
  typedef Layout L;
  u32x4 q[L::NC / 2];  // chunks 2 i + half of the query's row
  float m, l;          // l: of this lane's keys only
  f32x16 o[L::DT];

  __device__ __forceinline__ void Start(const char* row, int chunks, int half, float scale) {
#pragma unroll
    for (int i = 0; i < L::NC / 2; ++i) {
      q[i] = u32x4{0, 0, 0, 0};
      if (2 * i + half < chunks) q[i] = Signed<T>(LoadAny<T>(row + (2 * i + half) * 16), scale);
    }
    m = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (int t = 0; t < L::DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = 0.0f;
  }

  // scores of 32 keys whose rows lie at `tile`
  __device__ __forceinline__ f32x16 Scores(const char* tile, int lane) const {
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < L::NC / 2; ++i)
      s = Mma<T>::mma(*reinterpret_cast<const u32x4*>(tile + L::KAt(lane & 31, 2 * i + (lane >> 5))), q[i], s);
    return s;
  }

  // scores of keys that the lane's query does not attend to count nothing
  static __device__ __forceinline__ void Mask(f32x16& s, unsigned word, int lane) {
    word >>= 4 * (lane >> 5);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!((word >> (8 * (r >> 2) + (r & 3))) & 1)) s[r] = -__builtin_inff();
  }

  // Scores become probabilities against a running maximum.  What has been summed is rescaled only when a score exceeds it by
  // more than a factor of 2^8 (fp32, whose exponent is natural: e^8), and only then do the lanes of a query agree on a new
  // one: probabilities up to 256 (2981) lose nothing in either type, and after the first tiles few maxima grow that much.
  static __device__ __forceinline__ float Top(const f32x16& s) {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    return top;
  }
  __device__ __forceinline__ void Grow(float top, const Exp<T>& ex) {
    if (__ballot((top - m) * ex.c > 8.0f)) {
      top = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float keep = ex(m, ex.Base(top));
      l *= keep;
#pragma unroll
      for (int t = 0; t < L::DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= keep;
      m = top;
    }
  }
  // The probabilities of 32 keys as the matrix cores take them: 16-bit ones are rounded, which costs half a step of the type
  // as the result's own rounding does (fp16 ones far below the largest: HeldBase); fp32 operands split in two would take twice
  // the MFMAs.  They are summed before (in twos by dot products with ones: half the instructions, and 3% slower over 16384 keys).
  struct Probabilities {
    typename Held<T>::type g[Held<T>::COUNT];
    __device__ __forceinline__ float At(int r) const {  // of register r, which is known after unrolling
      if constexpr (L::F32) {
        return g[0][r];
      } else {
        return (float)g[r / 8][r % 8];
      }
    }
  };
  __device__ __forceinline__ Probabilities Soften(f32x16 s, const Exp<T>& ex) {
    const float base = HeldBase(ex, m);
    Probabilities p;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = ex(s[r], base);
#pragma unroll
    for (int r = 0; r < 16; ++r) l += s[r];
    if constexpr (L::F32) {
      p.g[0] = s;
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) p.g[r / 8][r % 8] = (T)s[r];
    }
    return p;
  }

  // sums of 32 keys' values
  __device__ __forceinline__ void Add(const Probabilities& p, const char* tile, int lane) {
    const int half = lane >> 5;
    if constexpr (L::F32) {
#pragma unroll
      for (int t = 0; t < L::DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 8 * (r >> 2) + 4 * half + (r & 3);
          const float v = *reinterpret_cast<const float*>(tile + L::VAt(key, t * 8 + (lane & 31) / 4) + (lane & 3) * 4);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p.g[0][r], o[t], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int t = 0; t < L::DT; ++t) {
          // four keys x sixteen d per group of 16 lanes, transposed on the way
          s16x4 part[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const char* at = tile + L::VAt(16 * g + 8 * u + 4 * half + ((lane & 15) >> 2), 4 * t + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) +
                             (lane & 1) * 8;
            part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)at);
          }
          o[t] = Mma<T>::mma(__builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7)),
                             __builtin_bit_cast(u32x4, p.g[g]), o[t]);
        }
      }
    }
  }

  // whether one of the 32 keys' values is infinite or no number
  static __device__ __forceinline__ bool Unbounded(const char* tile, int chunks, int lane) {
    constexpr unsigned kExponent = L::F32 ? 0x7f800000u : sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    bool found = false;
#pragma unroll
    for (int i = 0; i < L::NC / 2; ++i) {
      const int at = i * 64 + lane;
      if (at % L::NC >= chunks) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(tile + L::VAt(at / L::NC, at % L::NC));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        found |= (v[e] & kExponent) == kExponent;
        if (!L::F32) found |= (v[e] >> 16 & kExponent) == kExponent;
      }
    }
    return __ballot(found) != 0;
  }

  // Add for values among which are infinities or NaN, where a probability of zero by the mask must not make 0 * inf: key
  // by key, only where the query attends to it
  __device__ __forceinline__ void AddChosen(const Probabilities& p, unsigned word, const char* tile, int lane) {
    const int half = lane >> 5;
    f32x16 all;
#pragma unroll
    for (int r = 0; r < 16; ++r) all[r] = p.At(r);
#pragma unroll 1
    for (int at = 0; at < 32; ++at) {
      const int owner = at >> 4, reg = at & 15, key = 8 * (reg >> 2) + 4 * owner + (reg & 3);
      float mine = all[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mine = reg == r ? all[r] : mine;
      const float other = __shfl_xor(mine, 32), prob = half == owner ? mine : other;
      const bool chosen = (word >> key) & 1;
#pragma unroll
      for (int t = 0; t < L::DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int byte = (32 * t + 8 * (r >> 2) + 4 * half + (r & 3)) * (int)sizeof(T);
          if (byte >= L::NC * 16) continue;  // the last 32 elements of a D that is no multiple of 32
          const float v = (float)*reinterpret_cast<const T*>(tile + L::VAt(key, byte >> 4) + (byte & 15));
          o[t][r]       = chosen ? __builtin_fmaf(prob, v, o[t][r]) : o[t][r];
        }
    }
  }

  // one step: 32 keys of which the lane's query attends to those in `word`
  __device__ __forceinline__ void Step(const char* k_tile, const char* v_tile, unsigned word, int chunks, const Exp<T>& ex, int lane) {
    f32x16 s = Scores(k_tile, lane);
    const bool masked = __ballot(word != ~0u) != 0;
    if (masked) Mask(s, word, lane);
    Grow(Top(s), ex);
    const Probabilities p = Soften(s, ex);
    if (masked && Unbounded(v_tile, chunks, lane)) {
      AddChosen(p, word, v_tile, lane);
    } else {
      Add(p, v_tile, lane);
    }
  }

  // what another wavefront has of the same queries, [register][lane]
  static constexpr int kRegisters = L::DT * 16 + 2;
  __device__ __forceinline__ void Hand(float* to, int lane) const {
#pragma unroll
    for (int t = 0; t < L::DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) to[(t * 16 + r) * 64 + lane] = o[t][r];
    to[(kRegisters - 2) * 64 + lane] = m;
    to[(kRegisters - 1) * 64 + lane] = l;
  }
  __device__ __forceinline__ void Join(const float* from, const Exp<T>& ex, int lane) {
    const float m2 = from[(kRegisters - 2) * 64 + lane], top = fmaxf(m, m2), base = ex.Base(top);
    const float keep = ex(m, base), add = ex(m2, base);
    l = l * keep + from[(kRegisters - 1) * 64 + lane] * add;
#pragma unroll
    for (int t = 0; t < L::DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = o[t][r] * keep + from[(t * 16 + r) * 64 + lane] * add;
    m = top;
  }

  // o times `factor` to the query's row of the result
  __device__ __forceinline__ void Store(char* row, int d, float factor, int half) const {
#pragma unroll
    for (int t = 0; t < L::DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = t * 32 + 8 * i + 4 * half;
        T four[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = (T)(o[t][4 * i + e] * factor);
        if (at < d) __builtin_memcpy(row + at * sizeof(T), four, sizeof(four));
      }
  }
};

// 16 x PT queries of a wavefront against 32 keys at a time, where there are few: S^T = K Q^T by MFMAs of 16 keys x 16 pairs, a
// lane holding the scores of pair lane % 16 (+ 16 per pair tile) for the keys 16 h + 4 (lane / 16) + r, which is, as it lies, the
// second operand of O^T = V^T P^T.
template <typename T, int D, int PT>
struct FewPairs {
  typedef Dense<T, D> L;
  static constexpr bool F32 = L::F32;
  static constexpr int STEPS = L::NC / 4, DT = D / 16;
  u32x4 q[PT][STEPS];
  float m[PT], l[PT];  // l: of this lane's keys only
  f32x4 o[PT][DT];     // d = 16 t + 4 (lane / 16) + r

  // the chunk of a row that a lane multiplies in step i: halves of a wavefront take neighbouring ones, whose place in LDS
  // differs in the lowest bit
  static __device__ __forceinline__ int ChunkOf(int i, int lane) { return 4 * i + 2 * ((lane >> 4) & 1) + (lane >> 5); }

  __device__ __forceinline__ void Start(int tile, const char* row, int chunks, int lane, float scale) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      q[tile][i] = u32x4{0, 0, 0, 0};
      if (ChunkOf(i, lane) < chunks) q[tile][i] = Signed<T>(LoadAny<T>(row + ChunkOf(i, lane) * 16), scale);
    }
    m[tile] = -__builtin_inff(), l[tile] = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[tile][t] = f32x4{0, 0, 0, 0};
  }
  static __device__ __forceinline__ f32x4 Multiply(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F32) {
      const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
      return c;
    } else {
      typedef typename cinn_hip_kernels::flex::Half16<T> H;
      return H::mfma(__builtin_bit_cast(typename H::vec8, a), __builtin_bit_cast(typename H::vec8, b), c);
    }
  }
  __device__ __forceinline__ void Scores(f32x4 (&s)[PT][2], const char* tile, int lane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < PT; ++n) s[n][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(tile + L::KAt(16 * h + (lane & 15), ChunkOf(i, lane)));
#pragma unroll
        for (int n = 0; n < PT; ++n) s[n][h] = Multiply(k, q[n][i], s[n][h]);
      }
    }
  }
  static __device__ __forceinline__ void Mask(f32x4 (&s)[2], unsigned word, int lane) {
    word >>= 4 * (lane >> 4);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((word >> (16 * h + r)) & 1)) s[h][r] = -__builtin_inff();
  }
  // as Queries::Soften
  __device__ __forceinline__ void Soften(int tile, f32x4 (&s)[2], const Exp<T>& ex) {
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e >> 2][e & 3]);
    if (__ballot((top - m[tile]) * ex.c > 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(m[tile], fmaxf(top, __shfl_xor(top, 32)));
      const float keep = ex(m[tile], ex.Base(top));
      l[tile] *= keep;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[tile][t] *= keep;
      m[tile] = top;
    }
    const float base = HeldBase(ex, m[tile]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e >> 2][e & 3] = ex(s[e >> 2][e & 3], base);
      l[tile] += s[e >> 2][e & 3];
    }
  }
  // 16-bit probabilities round on their way into the matrix cores, as in Queries::Add
  __device__ __forceinline__ void Add(const f32x4 (&s)[PT][2], const char* tile, int lane) {
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = 16 * (e >> 2) + 4 * (lane >> 4) + (e & 3);
          const float v = *reinterpret_cast<const float*>(tile + L::At(key, 4 * t + ((lane & 15) >> 2)) + (lane & 3) * 4);
#pragma unroll
          for (int n = 0; n < PT; ++n) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[n][e >> 2][e & 3], o[n][t], 0, 0, 0);
        }
    } else {
      typedef T vec8 __attribute__((ext_vector_type(8)));
      vec8 pr[PT];
#pragma unroll
      for (int n = 0; n < PT; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) pr[n][e] = (T)s[n][e >> 2][e & 3];
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        s16x4 part[2];  // four keys x sixteen d per group of 16 lanes, transposed on the way
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const char* at = tile + L::At(16 * h + 4 * (lane >> 4) + ((lane & 15) >> 2), 2 * t + ((lane & 3) >> 1)) + (lane & 1) * 8;
          part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)at);
        }
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int n = 0; n < PT; ++n) o[n][t] = Multiply(v, __builtin_bit_cast(u32x4, pr[n]), o[n][t]);
      }
    }
  }
  // as Queries::Unbounded and Queries::AddChosen
  static __device__ __forceinline__ bool Unbounded(const char* tile, int lane) {
    constexpr unsigned kExponent = F32 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    bool found = false;
#pragma unroll
    for (int i = 0; i < L::NC / 2; ++i) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(tile + (i * 64 + lane) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        found |= (v[e] & kExponent) == kExponent;
        if (!F32) found |= (v[e] >> 16 & kExponent) == kExponent;
      }
    }
    return __ballot(found) != 0;
  }
  __device__ __forceinline__ void AddChosen(const f32x4 (&s)[PT][2], const unsigned (&word)[PT], const char* tile, int lane) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      const int reg = (key >> 4) * 4 + (key & 3), owner = (key & 15) >> 2;
#pragma unroll
      for (int n = 0; n < PT; ++n) {
        float prob = s[n][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) prob = reg == e ? s[n][e >> 2][e & 3] : prob;
        prob = __shfl((float)(T)prob, owner * 16 + (lane & 15));
        const bool chosen = (word[n] >> key) & 1;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int byte = (16 * t + 4 * (lane >> 4) + r) * (int)sizeof(T);
            const float v  = (float)*reinterpret_cast<const T*>(tile + L::At(key, byte >> 4) + (byte & 15));
            o[n][t][r]     = chosen ? __builtin_fmaf(prob, v, o[n][t][r]) : o[n][t][r];
          }
      }
    }
  }

  __device__ __forceinline__ void Store(int tile, char* row, int d, float factor, int lane) const {
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int at = 16 * t + 4 * (lane >> 4);
      T four[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) four[r] = (T)(o[tile][t][r] * factor);
      if (at < d) __builtin_memcpy(row + at * sizeof(T), four, sizeof(four));
    }
  }

  // what another wavefront has of one pair tile, [register][lane]
  static constexpr int kRegisters = DT * 4 + 2;
  __device__ __forceinline__ void Hand(int tile, float* to, int lane) const {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) to[(t * 4 + r) * 64 + lane] = o[tile][t][r];
    to[(kRegisters - 2) * 64 + lane] = m[tile];
    to[(kRegisters - 1) * 64 + lane] = l[tile];
  }
};

// v / d for 0 <= v < 2^31 and 1 <= d < 2^31, by a product: m = ceil(2^(31 + s) / d) with 2^s >= d is below 2^32 and off by less
// than d / 2^(31 + s), so v m / 2^(31 + s) is off by less than 1 / d
struct Divisor {
  unsigned multiplier;
  int shift, value;
  __host__ Divisor(int d = 1) : shift(0), value(d) {
    while ((int64_t{1} << shift) < d) ++shift;
    multiplier = (unsigned)(((uint64_t{1} << (31 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ int operator()(int v) const { return (int)((uint64_t)(unsigned)v * multiplier >> (31 + shift)); }
};

// zeros for rows and chunks that are none
__device__ const u32x4 kZeros[32] = {};

// Loads from memory straight to LDS: 16 bytes (4 bytes) a lane, written at LDS address `to` + 16 (4) * lane.  Inline assembly,
// so that the compiler does not track them: tracked, it would wait for all of them before every LDS read.
__device__ __forceinline__ void CopyToLds16(const void* from, unsigned to) {
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory");
}
// from a base that the wavefront shares and a lane's offset
__device__ __forceinline__ void CopyToLds16(const void* base, unsigned off, unsigned to) {
  to = __builtin_amdgcn_readfirstlane(to);
  const uint64_t at = (uint64_t)base;
  base = (const void*)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(at >> 32)) << 32 |
                       (unsigned)__builtin_amdgcn_readfirstlane((unsigned)at));
  // by way of a scalar copy: a vector memory instruction may not read a scalar register right behind a vector instruction, a
  // readlane or a reload among them, that wrote it
  uint64_t copy;
  asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0" : "=&s"(copy) : "s"(to), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void CopyToLds4(const void* from, unsigned to) {
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ unsigned LdsAddress(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// all but the last N of this wavefront's vector memory instructions have landed
template <int N>
__device__ __forceinline__ void WaitForAllBut() {
  static_assert(N < 64);
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
}

}  // namespace attention
}  // namespace cinn_hip_kernels
