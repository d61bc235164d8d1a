// Rotary positions for gfx950: y = magnitude R(p f) x on the first `heads` heads of [tokens][total_heads][d], fp16 / bf16 /
// fp32; pair i of a head, (x_2i, x_2i+1) or (x_i, x_i+r/2), is turned by the position times
//   f_i = theta^(-2i/r), scaled: f / factor, or where original_length is given
//   f (g + (1 - g) / factor), g = clamp((original_length f / 2 pi - low) / (high - low), 0, 1);
// elements from r on are copied.  The transpose (the gradient of x) turns the other way.
//
// Bound by memory: every rotated head is read once and written once, out of and into whatever surrounds it.  Angles: p f in
// turns is a 64-bit product whose fraction is taken before it is rounded to 32 bits (in 32 bits a position of 10^6 would be
// off by 0.06), then sincospi; a thread keeps those of its pairs for two heads.  Measured: 8191 tokens, 40 of 48 heads x 128
// in bf16, 168 MB: 34 us out of memory, 4.9 TB/s, where a copy of as much moves 5.3, and 27 us where the last-level cache holds
// them; 16 tokens 4.7 to 5.6 us, of which a launch is about 4.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "cinn_hip_runtime.h"
#include "runtime/hip_check.h"

namespace {

constexpr int kMostPairs = 256;

// f_i / 2 pi, in the kernel's argument segment: the smallest ones count down to 2^-53 of a turn
struct Turns {
  double v[kMostPairs];
};

struct RotaryParams {
  const char* x;
  const void* positions;
  char* y;
  int wide;                       // positions of 64 bits
  int heads, total_heads, d;
  int pairs;                      // r / 2
  int pair_units, units;          // threads per head: those that turn pairs, and all
  int64_t threads;                // tokens x head groups x units
  int head_groups, heads_each;
  float magnitude;
  int transposed;
};

template <typename T, int V>
struct Chunk {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> Load(const char* p) {
  Chunk<T, V> c;
  __builtin_memcpy(&c, __builtin_assume_aligned(p, sizeof(T)), sizeof(c));
  return c;
}
template <typename T, int V>
__device__ __forceinline__ void Store(char* p, const Chunk<T, V>& c) {
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &c, sizeof(c));
}

// A thread takes V pairs (halves) or V / 2 (neighbours) of a token, or V elements behind the rotated ones, in heads_each
// heads.
template <typename T, int V, bool NEIGHBOURS>
__global__ void __launch_bounds__(256)
rotary_kernel(RotaryParams p, Turns turns) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.threads) return;
  const int unit = (int)(id % p.units);
  const int64_t rest = id / p.units;
  const int first = (int)(rest % p.head_groups) * p.heads_each, last = min(first + p.heads_each, p.heads);
  const int64_t token = rest / p.head_groups;
  const int64_t head_bytes = (int64_t)p.d * sizeof(T);
  const char* x = p.x + (token * p.total_heads + first) * head_bytes;
  char* y       = p.y + (token * p.heads + first) * head_bytes;

  if (unit >= p.pair_units) {
    const int from   = 2 * p.pairs + (unit - p.pair_units) * V;
    const int64_t at = (int64_t)from * sizeof(T);
    if (from + V > p.d) {
      for (int h = first; h < last; ++h, x += head_bytes, y += head_bytes)
        for (int e = 0; e < p.d - from; ++e) reinterpret_cast<T*>(y + at)[e] = reinterpret_cast<const T*>(x + at)[e];
      return;
    }
#pragma unroll 4
    for (int h = first; h < last; ++h, x += head_bytes, y += head_bytes) Store<T, V>(y + at, Load<T, V>(x + at));
    return;
  }
  constexpr int N = NEIGHBOURS ? V / 2 : V;  // pairs
  const double position = p.wide ? (double)static_cast<const int64_t*>(p.positions)[token] : (double)static_cast<const int*>(p.positions)[token];
  float c[N], s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double t = position * turns.v[unit * N + i];
    sincospif(2.0f * (float)(t - rint(t)), &s[i], &c[i]);
    c[i] *= p.magnitude;
    s[i] *= p.transposed ? -p.magnitude : p.magnitude;
  }
  const int64_t at = (int64_t)unit * V * sizeof(T), half = (int64_t)p.pairs * sizeof(T);
#pragma unroll 4
  for (int h = first; h < last; ++h, x += head_bytes, y += head_bytes) {
    if constexpr (NEIGHBOURS) {
      Chunk<T, V> a = Load<T, V>(x + at);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = (float)a.e[2 * i], v = (float)a.e[2 * i + 1];
        a.e[2 * i]     = (T)(u * c[i] - v * s[i]);
        a.e[2 * i + 1] = (T)(v * c[i] + u * s[i]);
      }
      Store<T, V>(y + at, a);
    } else {
      Chunk<T, V> a = Load<T, V>(x + at), b = Load<T, V>(x + at + half);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = (float)a.e[i], v = (float)b.e[i];
        a.e[i] = (T)(u * c[i] - v * s[i]);
        b.e[i] = (T)(v * c[i] + u * s[i]);
      }
      Store<T, V>(y + at, a);
      Store<T, V>(y + at + half, b);
    }
  }
}

template <typename T, int V>
void Launch(RotaryParams p, const Turns& turns, int64_t tokens, bool neighbours, hipStream_t stream) {
  p.pair_units = neighbours ? 2 * p.pairs / V : p.pairs / V;
  p.units      = p.pair_units + (p.d - 2 * p.pairs + V - 1) / V;
  // us with 1 | 2 | 4 | 8 heads a thread: 8191 tokens x 40 heads x 128 in bf16 out of memory 40.1 | 34.9 | 36.4 | 36.6, out of the
  // last-level cache 33.6 | 27.5 | 28.1 | 28.9; 16384 x 40 x 64 in fp16 out of memory 39.6 | 34.9 | 36.7 | 38.7; 512 tokens 5.5 | 5.4 |
  // 5.3 | 6.2, 16 tokens 5.1 | 5.5 | 5.6 | 5.6, 1111 x 12 x 80 in fp32 4.8 | 5.1 | 5.2 | 5.7
  p.heads_each  = 2;
  p.head_groups = (p.heads + p.heads_each - 1) / p.heads_each;
  p.threads     = tokens * p.head_groups * p.units;
  const dim3 grid((unsigned)((p.threads + 255) / 256));
  if (neighbours) {
    if constexpr (V >= 2) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(256), 0, stream, p, turns);
  } else {
    hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(256), 0, stream, p, turns);
  }
}

// the widest access that divides what is turned
template <typename T>
void LaunchWide(const RotaryParams& p, const Turns& turns, int64_t tokens, bool neighbours, hipStream_t stream) {
  constexpr int kWide = 16 / (int)sizeof(T);
  const int run = neighbours ? 2 * p.pairs : p.pairs;
  if (run % kWide == 0) {
    Launch<T, kWide>(p, turns, tokens, neighbours, stream);
  } else if (sizeof(T) == 2 && run % 4 == 0) {
    Launch<T, 4>(p, turns, tokens, neighbours, stream);
  } else if (run % 2 == 0) {
    Launch<T, 2>(p, turns, tokens, neighbours, stream);
  } else {
    Launch<T, 1>(p, turns, tokens, neighbours, stream);
  }
}

cinn_buffer_t* BufferArg(void* v_args, int index) {
  auto* args = static_cast<cinn_pod_value_t*>(v_args);
  CINN_RT_CHECK(args[index].type_code_ == CINN_POD_BUFFER_P, "rotary_embedding: argument %d is not a buffer", index);
  auto* b = static_cast<cinn_buffer_t*>(args[index].value_.v_handle);
  CINN_RT_CHECK(b && b->memory, "rotary_embedding: argument %d has no device memory", index);
  return b;
}

}  // namespace

extern "C" void cinn_call_hip_rotary_embedding(void* v_args, int num_args, int tokens, int heads, int total_heads, int d, int rotary_dim,
                                               int interleaved, int transposed, double theta, double factor, int original_length,
                                               double low, double high, double magnitude, void* stream) {
  CINN_HIP_CLEAR_STALE_ERROR();
  CINN_RT_CHECK(num_args == 3, "rotary_embedding: x, positions and y");
  CINN_RT_CHECK(tokens >= 0 && heads >= 0 && total_heads >= heads && d > 0, "rotary_embedding: %d tokens, %d of %d heads, %d elements each",
                tokens, heads, total_heads, d);
  CINN_RT_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= d && rotary_dim <= 2 * kMostPairs,
                "rotary_embedding: %d of %d elements in pairs (at most %d)", rotary_dim, d, 2 * kMostPairs);
  CINN_RT_CHECK(theta > 0 && factor > 0 && original_length >= 0 && (original_length == 0 || high > low), "rotary_embedding: scaling");
  CINN_RT_CHECK((int64_t)tokens * total_heads * d < INT_MAX, "rotary_embedding: tensor too large");
  if ((int64_t)tokens * heads == 0) return;
  const cinn_buffer_t *x = BufferArg(v_args, 0), *at = BufferArg(v_args, 1), *y = BufferArg(v_args, 2);
  const bool f32 = x->type.code == cinn_type_float && x->type.bits == 32;
  const bool f16 = x->type.code == cinn_type_float && x->type.bits == 16;
  CINN_RT_CHECK(f32 || f16 || (x->type.code == cinn_type_bfloat && x->type.bits == 16), "rotary_embedding: fp16 / bf16 / fp32 only");
  CINN_RT_CHECK(y->type.code == x->type.code && y->type.bits == x->type.bits, "rotary_embedding: x and y of different types");
  CINN_RT_CHECK(at->type.code == cinn_type_int && (at->type.bits == 32 || at->type.bits == 64), "rotary_embedding: positions are int32 or int64");
  Turns turns = {};
  const double two_pi = 6.283185307179586;
  for (int i = 0; i < rotary_dim / 2; ++i) {
    double f = std::pow(theta, -2.0 * i / rotary_dim);
    if (original_length > 0) {
      const double keep = std::min(1.0, std::max(0.0, (original_length * f / two_pi - low) / (high - low)));
      f *= keep + (1.0 - keep) / factor;
    } else {
      f /= factor;
    }
    turns.v[i] = f / two_pi;
  }
  RotaryParams p = {};
  p.x = reinterpret_cast<const char*>(x->memory), p.positions = at->memory, p.y = reinterpret_cast<char*>(y->memory);
  p.wide = at->type.bits == 64, p.heads = heads, p.total_heads = total_heads, p.d = d, p.pairs = rotary_dim / 2;
  p.magnitude = (float)magnitude, p.transposed = transposed;
  auto s = static_cast<hipStream_t>(stream);
  if (f32) {
    LaunchWide<float>(p, turns, tokens, interleaved != 0, s);
  } else if (f16) {
    LaunchWide<_Float16>(p, turns, tokens, interleaved != 0, s);
  } else {
    LaunchWide<__bf16>(p, turns, tokens, interleaved != 0, s);
  }
  CINN_HIP_CALL(hipGetLastError());
}
