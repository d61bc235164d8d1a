// Causal attention over packed prompts for gfx950: sequence s holds rows offsets[s] .. offsets[s + 1] of [tokens][heads][d]
// operands, query head h reads key head h / group, and row t attends to its sequence's rows up to t:
//   O = softmax(scale Q K^T, masked) V,
// fp16 / bf16 / fp32, scores and sums in fp32.
//
// A block takes one key head and a run of its (query, head of the group) pairs, in that order: the group's heads share
// every key that is read, and the keys that the run's queries do not all attend to are few.  The lengths are data: the grid
// covers the most tiles that sequences of so many rows can have, and a block finds its own among the offsets.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "cinn_hip_runtime.h"
#include "kernels/attention_tile.h"
#include "runtime/hip_check.h"

namespace {

using namespace cinn_hip_kernels::attention;

struct PackedParams {
  Rows q, k, v, o;  // of the first head in use; batch unused
  const int* offsets;
  int sequences, tokens, kv_heads, d, tiles;
  Divisor group;
  float scale;
};

// a sequence's rows and the tile of its pairs, or with count 0 the how many-th of the `more` blocks behind the last tile
struct Found {
  int first, count, tile, more;
};

// Offsets out of order or range find rows in range all the same.
struct Sequence {
  int first, count, tiles;
};
__device__ __forceinline__ Sequence SequenceOf(const PackedParams& p, int s, int tile_pairs) {
  if (s >= p.sequences) return {0, 0, 0};
  const int first = min(max(p.offsets[s], 0), p.tokens), count = max(min(p.offsets[s + 1], p.tokens) - first, 0);
  return {first, count, (count * p.group.value + tile_pairs - 1) / tile_pairs};
}

// The tile of block `tile`, by every wavefront for itself.  Later tiles of a sequence have more keys and come first, of few
// sequences across all: how many tiles lie at t or further back in their sequences, for 64 values of t at a time, tells the
// largest t that the block's number falls under.  us, sequence by sequence | across: fp16 12 heads x 64, 8 x 512 rows 17.9 | 15.9,
// 16 x 512 24.1 | 20.9, 24 x 512 35.5 | 29.3; bf16 32 heads over 8 x 128, 8192 rows in 4 sequences of up to 4000 154 | 154, 16 of
// up to 1000 42.8 | 43.7, 24 41.8 | 44.4, 64 of up to 250 42.5 | 50.9: the count takes a step for every sequence.
__device__ __forceinline__ Found Find(const PackedParams& p, int tile, int tile_pairs) {
  const int lane = threadIdx.x & 63;
  if (p.sequences <= 16) {
    const Sequence mine = SequenceOf(p, lane, tile_pairs);
    int t = 0, after = 0;  // after: how many lie further back than t
    while (true) {
      int behind = 0;
      for (int s = 0; s < p.sequences; s += 4)  // lanes behind the last sequence have none
#pragma unroll
        for (int i = 0; i < 4; ++i) behind += max(__builtin_amdgcn_readlane(mine.tiles, s + i) - (t + lane), 0);
      if (t == 0) {
        const int all = __builtin_amdgcn_readlane(behind, 0);
        if (tile >= all) return {0, 0, tile - all, p.tiles - all};
      }
      const int last = 63 - __clzll(__ballot(behind > tile));  // lane 0's are more than `tile`
      t += last;
      if (last == 63) continue;
      after = __builtin_amdgcn_readlane(behind, last + 1);
      break;
    }
    const unsigned long long with = __ballot(mine.tiles > t);
    const int rank = __popcll(with & ((1ull << lane) - 1));
    const int at   = __ffsll(__ballot(mine.tiles > t && rank == tile - after)) - 1;
    return {__builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.count, at), t, 0};
  }
  int before = 0;
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    const Sequence mine = SequenceOf(p, s0 + lane, tile_pairs);
    int sum = mine.tiles;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int up = __shfl_up(sum, x);
      if (lane >= x) sum += up;
    }
    const unsigned long long behind = __ballot(before + sum > tile);
    if (behind) {
      const int at = __ffsll(behind) - 1;
      const int tiles = __builtin_amdgcn_readlane(mine.tiles, at), here = tile - (before + __builtin_amdgcn_readlane(sum, at) - tiles);
      return {__builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.count, at), tiles - 1 - here, 0};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {0, 0, tile - before, p.tiles - before};
}

// zeros to the rows of no sequence
template <typename T>
__device__ void ClearRest(const PackedParams& p, int head, int index, int blocks) {
  const int chunks = p.d * (int)sizeof(T) / 16, group = p.group.value;
  const int lead = min(max(p.offsets[0], 0), p.tokens), end = max(lead, min(p.offsets[p.sequences], p.tokens));
  const int64_t total = (int64_t)(lead + p.tokens - end) * group * chunks;
  for (int64_t i = (int64_t)index * blockDim.x + threadIdx.x; i < total; i += (int64_t)blocks * blockDim.x) {
    const int chunk = (int)(i % chunks), pair = (int)(i / chunks), at = pair / group;
    char* row = const_cast<char*>(HeadOf<T>(p.o, 0, head * group + pair % group)) + (at < lead ? at : at - lead + end) * p.o.row * (int64_t)sizeof(T);
    const u32x4 zero = {0, 0, 0, 0};
    __builtin_memcpy(__builtin_assume_aligned(row + chunk * 16, sizeof(T)), &zero, 16);
  }
}

// 16-bit types: WQ x 32 pairs, KG wavefronts for each 32 that take the steps of 32 keys in turn, tiles of 32 STEPS keys in a
// ring of four in LDS that loads fill directly, one barrier per tile.  A wavefront multiplies the next 32 keys by its queries
// while it takes the exponentials of the last scores: the matrix cores and the vector unit work side by side, within a wavefront
// and, two of them to a SIMD, across.  Rows behind the last key are rows of the tensor all the same; nothing attends to them.
// Bound by matrix cores and vector units together for long prompts, 53 and 50 % of whose cycles are taken: one of 16384 rows, 32 heads
// over 8 x 128 in bf16, 2.00 to 2.06 ms, 1.1 PFLOP/s of the 1.25 that a product of 8192^3 reaches; 11 prompts of 8191 rows together
// 201 to 208 us; 8 x 512 rows, 12 x 64 in fp16, 15.7 us, a chain of eight tiles for the last queries, wavefronts waiting in 56 % of
// their cycles.  Tiles that went through registers took 3.2 ms, 334 and 26 us.
template <typename T, int D, int WQ, int KG, int STEPS>
__global__ void __launch_bounds__(64 * WQ * KG, 2)
packed_attention_ring_kernel(PackedParams p) {
  typedef Dense<T, D> L;
  typedef Queries<T, D, L> Q;
  constexpr int KT = 32 * STEPS, NC = L::NC, STAGE = 2 * STEPS * L::BYTES, STAGES = 4;
  constexpr int LOADS = STEPS * NC, N = (LOADS + WQ * KG - 1) / (WQ * KG);  // for a tile, its values behind its keys, and a wavefront's
  constexpr int MEET = (KG - 1) * WQ * 64 * Q::kRegisters * 4;
  static_assert(STEPS % KG == 0 && (STAGES - 3) * N < 64);
  __shared__ __attribute__((aligned(256))) char lds[STAGES * STAGE > MEET ? STAGES * STAGE : MEET];

  const int head = blockIdx.x % p.kv_heads;
  const Found at = Find(p, blockIdx.x / p.kv_heads, 32 * WQ);
  if (at.count == 0) {
    ClearRest<T>(p, head, at.tile, at.more);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / WQ, wq = wave % WQ;
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = at.count * p.group.value;
  const int pair0 = (at.tile * WQ + wq) * 32;
  const int pair = min(pair0 + (lane & 31), pairs - 1);
  const int query = p.group(pair), my_head = head * p.group.value + pair - query * p.group.value;
  const int first_query = p.group(min(pair0, pairs - 1)), last_query = pair0 < pairs ? p.group(min(pair0 + 31, pairs - 1)) : -1;
  const int keys = p.group(min((at.tile + 1) * WQ * 32, pairs) - 1) + 1;
  const int tiles = (keys + KT - 1) / KT, my_steps = __builtin_amdgcn_readfirstlane(last_query >= 0 ? last_query / 32 + 1 : 0);

  const int64_t k_row = p.k.row * sizeof(T), v_row = p.v.row * sizeof(T);
  const char* k_base = HeadOf<T>(p.k, 0, head) + at.first * k_row;
  const char* v_base = HeadOf<T>(p.v, 0, head) + at.first * v_row;
  const unsigned lds_at = LdsAddress(lds);
  // where this lane's chunk of each load lies in a tile; LDS holds the chunks in order, memory gives them turned
  unsigned off[N];
  bool none[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int load = min(wave * N + i, LOADS - 1), slot = load % (LOADS / 2) * 64 + lane, row = slot / NC;
    const bool values = load >= LOADS / 2;
    const int c = L::Back(slot % NC, values ? L::WideTurn(row) : L::KTurn(row));
    off[i]  = row * (int)(values ? v_row : k_row) + c * 16;
    none[i] = c >= chunks;
  }
  auto request = [&](int tile) {
    const unsigned to = lds_at + tile % STAGES * STAGE;
    const int beyond  = at.first + (tile + 1) * KT - p.tokens;  // rows of the tile that are not the tensor's: its last one instead
    const char *k_tile = k_base + (int64_t)tile * KT * k_row, *v_tile = v_base + (int64_t)tile * KT * v_row;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int load = min(wave * N + i, LOADS - 1);
      const bool values = load >= LOADS / 2;
      const char* from  = values ? v_tile : k_tile;
      if (chunks == NC && beyond <= 0) {
        CopyToLds16(from, off[i], to + load * 1024);
      } else {
        const int row  = (load % (LOADS / 2) * 64 + lane) / NC;
        const int back = max(row - (KT - 1 - beyond), 0) * (int)(values ? v_row : k_row);
        CopyToLds16(none[i] ? reinterpret_cast<const char*>(kZeros) : from + (int)(off[i] - back), to + load * 1024);
      }
    }
  };
  auto keys_of = [&](int step) { return lds + step / STEPS % STAGES * STAGE + step % STEPS * L::BYTES; };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    if (i < tiles) request(i);
  Q rows;
  rows.Start(HeadOf<T>(p.q, 0, my_head) + (at.first + query) * p.q.row * (int64_t)sizeof(T), chunks, half, p.scale);
  const Exp<T> ex(p.scale);
  WaitForAllBut<0>();  // the queries are the last that was asked for
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // before the first step of a tile: it has landed, and everybody is done with the one before the last
  auto turn = [&](int step) {
    if (step % STEPS != 0 || step >= tiles * STEPS) return;
    const int tile = step / STEPS;
    if (tile + 1 < tiles) {
      WaitForAllBut<N>();
    } else {
      WaitForAllBut<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (tile + STAGES - 2 < tiles) request(tile + STAGES - 2);
  };
  f32x16 s  = rows.Scores(keys_of(kg), lane);
  float top = Q::Top(s);
  int step  = kg;
  // steps of keys that all of the wavefront's queries attend to
  const int plain_steps = __builtin_amdgcn_readfirstlane(last_query >= 0 ? (first_query + 1) / 32 : 0);
  auto open = [&] {  // the step's scores are complete
    if (step >= plain_steps) {
      Q::Mask(s, Below(query + 1 - step * 32), lane);
      top = Q::Top(s);
    }
    rows.Grow(top, ex);
  };
  auto values_of = [&](int n) { return keys_of(n) + STEPS * L::BYTES; };
  if constexpr (WQ == 8) {
    // without the branches of the loop below, where the code's length does not count
#pragma unroll 1
    for (; step < plain_steps; step += KG) {
      rows.Grow(top, ex);
      turn(step - kg + KG);
      const typename Q::Probabilities mine = rows.Soften(s, ex);
      s = rows.Scores(keys_of(step + KG), lane);
      rows.Add(mine, values_of(step), lane);
      top = Q::Top(s);
    }
  }
#pragma unroll 1
  for (; step < tiles * STEPS; step += KG) {
    if (step < my_steps) open();
    turn(step - kg + KG);
    if (step >= my_steps) continue;
    if (step >= plain_steps && Q::Unbounded(values_of(step), chunks, lane)) break;
    const typename Q::Probabilities mine = rows.Soften(s, ex);
    s = rows.Scores(keys_of(step + KG), lane);
    rows.Add(mine, values_of(step), lane);
    top = Q::Top(s);
  }
  // from the first step on whose values a mask alone does not keep out; it has been opened
#pragma unroll 1
  for (bool opened = true; step < tiles * STEPS; step += KG, opened = false) {
    if (!opened) {
      if (step < my_steps) open();
      turn(step - kg + KG);
    }
    if (step >= my_steps) continue;
    rows.AddChosen(rows.Soften(s, ex), Below(query + 1 - step * 32), values_of(step), lane);
    s   = rows.Scores(keys_of(step + KG), lane);
    top = Q::Top(s);
  }
  if constexpr (KG > 1) {
    __syncthreads();
    float* meet = reinterpret_cast<float*>(lds);
    if (kg > 0) rows.Hand(meet + ((kg - 1) * WQ + wq) * Q::kRegisters * 64, lane);
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int g = 1; g < KG; ++g) rows.Join(meet + ((g - 1) * WQ + wq) * Q::kRegisters * 64, ex, lane);
  }
  const float sum = rows.l + __shfl_xor(rows.l, 32);
  if (pair0 + (lane & 31) >= pairs) return;
  char* out = const_cast<char*>(HeadOf<T>(p.o, 0, my_head)) + (at.first + query) * p.o.row * (int64_t)sizeof(T);
  rows.Store(out, p.d, 1.0f / sum, half);
}

// The same with 16 pairs a wavefront, for few pairs and for fp32: shorter chains of MFMAs and exponentials per step, and
// twice the wavefronts, where latency counts.  5 prompts of 17 to 100 rows, 8 heads over 2 x 80 in fp32, 16.7 us on 40 blocks, bound by
// a wavefront's latencies with nothing beside it: 44% of its cycles wait for memory, LDS and barriers, 23% for instructions that
// may not issue yet, 33% issue.
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2)
packed_attention_few_kernel(PackedParams p) {
  typedef FewPairs<T, D, 1> Q;
  typedef Dense<T, D> L;
  constexpr int NC = L::NC, STAGE = 2 * L::BYTES, STAGES = 4, LOADS = NC, N = (LOADS + WAVES - 1) / WAVES;  // the last is asked for again
  __shared__ __attribute__((aligned(256))) char lds[STAGES * STAGE];
  const int head = blockIdx.x % p.kv_heads;
  const Found at = Find(p, blockIdx.x / p.kv_heads, 16 * WAVES);
  if (at.count == 0) {
    ClearRest<T>(p, head, at.tile, at.more);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = p.d * (int)sizeof(T) / 16, group = p.group.value, pairs = at.count * group;
  const int pair0 = (at.tile * WAVES + wave) * 16;
  const int first_query = p.group(min(pair0, pairs - 1));
  const int last_query  = pair0 < pairs ? p.group(min(pair0 + 15, pairs - 1)) : -1;
  const int keys  = p.group(min((at.tile + 1) * WAVES * 16, pairs) - 1) + 1;
  const int steps = (keys + 31) / 32, my_steps = __builtin_amdgcn_readfirstlane(last_query >= 0 ? last_query / 32 + 1 : 0);
  const int plain_steps = __builtin_amdgcn_readfirstlane(last_query >= 0 ? (first_query + 1) / 32 : 0);

  const int64_t k_row = p.k.row * sizeof(T), v_row = p.v.row * sizeof(T);
  const char* k_base = HeadOf<T>(p.k, 0, head) + at.first * k_row;
  const char* v_base = HeadOf<T>(p.v, 0, head) + at.first * v_row;
  const unsigned lds_at = LdsAddress(lds);
  unsigned off[N];
  bool none[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int load = min(wave * N + i, LOADS - 1), slot = load % (LOADS / 2) * 64 + lane, row = slot / NC;
    const bool values = load >= LOADS / 2;
    const int c = L::Back(slot % NC, values ? L::RowTurn(row) : L::KTurn(row));
    off[i]  = row * (int)(values ? v_row : k_row) + c * 16;
    none[i] = c >= chunks;
  }
  auto request = [&](int step) {
    const unsigned to = lds_at + step % STAGES * STAGE;
    const int beyond  = at.first + (step + 1) * 32 - p.tokens;  // as in the other kernel
    const char *k_tile = k_base + (int64_t)step * 32 * k_row, *v_tile = v_base + (int64_t)step * 32 * v_row;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int load = min(wave * N + i, LOADS - 1);
      const bool values = load >= LOADS / 2;
      const char* from  = values ? v_tile : k_tile;
      if (chunks == NC && beyond <= 0) {
        CopyToLds16(from, off[i], to + load * 1024);
      } else {
        const int row  = (load % (LOADS / 2) * 64 + lane) / NC;
        const int back = max(row - (31 - beyond), 0) * (int)(values ? v_row : k_row);
        CopyToLds16(none[i] ? reinterpret_cast<const char*>(kZeros) : from + (int)(off[i] - back), to + load * 1024);
      }
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1 && i < steps; ++i) request(i);
  Q rows;
  const int pair = min(pair0 + (lane & 15), pairs - 1), query = p.group(pair), my_head = head * group + pair - query * group;
  rows.Start(0, HeadOf<T>(p.q, 0, my_head) + (at.first + query) * p.q.row * (int64_t)sizeof(T), chunks, lane, p.scale);
  const Exp<T> ex(p.scale);
  WaitForAllBut<0>();  // the queries are the last that was asked for
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // before a step's scores: its keys and values have landed, and everybody is done with those two before it
  auto turn = [&](int step) {
    if (step >= steps) return;
    if (step + 1 < steps) {
      WaitForAllBut<N>();
    } else {
      WaitForAllBut<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (step + STAGES - 2 < steps) request(step + STAGES - 2);
  };
  f32x4 s[1][2];
  unsigned word[1];
  auto keys_of   = [&](int n) { return lds + n % STAGES * STAGE; };
  auto values_of = [&](int n) { return keys_of(n) + L::BYTES; };
  int step = 0;
  auto open = [&] {  // the step's scores are complete
    word[0] = Below(query + 1 - step * 32);
    if (step >= plain_steps) Q::Mask(s[0], word[0], lane);
  };
  rows.Scores(s, keys_of(0), lane);
#pragma unroll 1
  for (; step < steps; ++step) {
    if (step < my_steps) open();
    turn(step + 1);
    if (step >= my_steps) continue;
    if (step >= plain_steps && Q::Unbounded(values_of(step), lane)) break;
    rows.Soften(0, s[0], ex);
    const f32x4 mine[1][2] = {{s[0][0], s[0][1]}};
    rows.Scores(s, keys_of(step + 1), lane);
    rows.Add(mine, values_of(step), lane);
  }
  // from the first step on whose values a mask alone does not keep out; it has been opened
#pragma unroll 1
  for (bool opened = true; step < steps; ++step, opened = false) {
    if (!opened) {
      if (step < my_steps) open();
      turn(step + 1);
    }
    if (step >= my_steps) continue;
    rows.Soften(0, s[0], ex);
    rows.AddChosen(s, word, values_of(step), lane);
    rows.Scores(s, keys_of(step + 1), lane);
  }
  float sum = rows.l[0] + __shfl_xor(rows.l[0], 16);
  sum += __shfl_xor(sum, 32);
  if (pair0 + (lane & 15) >= pairs) return;
  rows.Store(0, const_cast<char*>(HeadOf<T>(p.o, 0, my_head)) + (at.first + query) * p.o.row * (int64_t)sizeof(T), p.d, 1.0f / sum, lane);
}

template <typename T, int D, int WQ, int KG, int STEPS>
void LaunchRing(PackedParams p, hipStream_t stream) {
  p.tiles = (int)((int64_t)p.tokens * p.group.value / (32 * WQ)) + p.sequences + 1;
  hipLaunchKernelGGL((packed_attention_ring_kernel<T, D, WQ, KG, STEPS>), dim3((unsigned)p.tiles * p.kv_heads), dim3(64 * WQ * KG), 0, stream, p);
}

template <typename T, int D>
void LaunchTiles(PackedParams p, hipStream_t stream) {
  // Blocks of 128 pairs: how full the GPU is, whatever the lengths.  us, few | ring of 4 x 2 | 4 x 1 | 8 x 1 wavefronts, the
  // choice in brackets.  bf16 32 heads over 8 x 128, one prompt of 64 [7.2] | 10.2 | 9.1 | 10.7, 256 [11.7] | 13.5 | 13.7 |
  // 16.2, 1024 31.9 | [28.4] | 34.0 | 39.6, 2048 74.7 | [59.4] | 64.1 | 70.9, 4096 - | - | 152 | [144], 16384 - | - | 2100 |
  // [1995]; 11 ragged prompts of 8191 330 | 264 | 201 | [201].  The wavefronts of a block wait for the one with the last
  // queries, with one head a key head 256 queries apart, which costs where prompts are not long.  4 x 1 | 8 x 1 by heads a key
  // head, 1, 2, 3, 4, 8: fp16 12 heads x 64, 8 x 1024 32.6 | 34.5, 30.5 | 31.6, 29.9 | 30.7, 29.7 | 30.4, -; 8 x 2048 83 | 81, 81 | 76,
  // 81 | 75, 81 | 76, -; bf16 32 or 33 x 128, one of 4096 159 | 151, 152 | 146, 160 | 161, 152 | 144, 153 | 146, ragged 215 | 222, 201 |
  // 202, 227 | 216, 201 | 201, 202 | 200: within 8% of each other, the lengths, which the host does not know, counting as much.
  const int64_t blocks = (int64_t)p.tokens * p.group.value / 128 * p.kv_heads;
  if constexpr (sizeof(T) == 2) {
    if (blocks > 512) return p.group.value >= 4 ? LaunchRing<T, D, 8, 1, 2>(p, stream) : LaunchRing<T, D, 4, 1, 1>(p, stream);
    if (blocks > 128) return LaunchRing<T, D, 4, 2, 2>(p, stream);
  }
  constexpr int kPairs = 64;
  p.tiles = (int)((int64_t)p.tokens * p.group.value / kPairs) + p.sequences + 1;
  hipLaunchKernelGGL((packed_attention_few_kernel<T, D, kPairs / 16>), dim3((unsigned)p.tiles * p.kv_heads), dim3(kPairs * 4), 0, stream, p);
}

template <typename T>
void Launch(const PackedParams& p, hipStream_t stream) {
  if (p.d <= 32) {
    LaunchTiles<T, 32>(p, stream);
  } else if (p.d <= 64) {
    LaunchTiles<T, 64>(p, stream);
  } else if (p.d <= 96) {
    LaunchTiles<T, 96>(p, stream);
  } else {
    LaunchTiles<T, 128>(p, stream);
  }
}

cinn_buffer_t* BufferArg(void* v_args, int index) {
  auto* args = static_cast<cinn_pod_value_t*>(v_args);
  CINN_RT_CHECK(args[index].type_code_ == CINN_POD_BUFFER_P, "packed_attention: argument %d is not a buffer", index);
  auto* b = static_cast<cinn_buffer_t*>(args[index].value_.v_handle);
  CINN_RT_CHECK(b && b->memory, "packed_attention: argument %d has no device memory", index);
  return b;
}

}  // namespace

extern "C" void cinn_call_hip_packed_attention(void* v_args, int num_args, float scale, int tokens, int sequences, int heads, int kv_heads,
                                               int d, int operands, int q_heads, int q_head, int k_heads, int k_head, int v_heads,
                                               int v_head, void* stream) {
  CINN_HIP_CLEAR_STALE_ERROR();
  CINN_RT_CHECK(tokens >= 0 && sequences >= 0, "packed_attention: negative extent");
  CINN_RT_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "packed_attention: %d heads, %d key heads", heads, kv_heads);
  CINN_RT_CHECK(d > 0 && d <= 128, "packed_attention: %d elements per row (at most 128)", d);
  CINN_RT_CHECK(q_head >= 0 && k_head >= 0 && v_head >= 0 && q_head + heads <= q_heads && k_head + kv_heads <= k_heads && v_head + kv_heads <= v_heads,
                "packed_attention: heads outside their tensors");
  if (tokens == 0) return;
  const cinn_buffer_t* out = BufferArg(v_args, num_args - 1);
  const bool f32 = out->type.code == cinn_type_float && out->type.bits == 32;
  const bool f16 = out->type.code == cinn_type_float && out->type.bits == 16;
  CINN_RT_CHECK(f32 || f16 || (out->type.code == cinn_type_bfloat && out->type.bits == 16), "packed_attention: fp16 / bf16 / fp32 only");
  CINN_RT_CHECK(d % (f32 ? 4 : 8) == 0, "packed_attention: rows of %d elements are no whole number of 16-byte chunks", d);
  const int64_t row = (int64_t)d * std::max(std::max(q_heads, k_heads), v_heads);
  CINN_RT_CHECK(tokens * row < INT_MAX, "packed_attention: tensor too large");
  CINN_RT_CHECK(row * (f32 ? 4 : 2) <= 1 << 25, "packed_attention: rows of more than 32 MiB");  // a tile's offsets have 32 bits
  auto input = [&](int slot) {
    const int at = (operands >> (4 * slot)) & 15;
    CINN_RT_CHECK(at < num_args - 1, "packed_attention: operand %d is argument %d of %d", slot, at, num_args);
    return BufferArg(v_args, at);
  };
  auto rows = [&](int slot, int total, int first) {
    const cinn_buffer_t* b = input(slot);
    CINN_RT_CHECK(b->type.code == out->type.code && b->type.bits == out->type.bits, "packed_attention: operands of different types");
    CINN_RT_CHECK(reinterpret_cast<uintptr_t>(b->memory) % 16 == 0, "packed_attention: operand %d is not aligned to 16 bytes", slot);
    return Rows{b->memory + (int64_t)first * d * (f32 ? 4 : 2), 0, d, (int64_t)total * d};
  };
  PackedParams p;
  p.q = rows(0, q_heads, q_head), p.k = rows(1, k_heads, k_head), p.v = rows(2, v_heads, v_head);
  p.o = Rows{out->memory, 0, d, (int64_t)heads * d};
  const cinn_buffer_t* offsets = input(3);
  CINN_RT_CHECK(offsets->type.code == cinn_type_int && offsets->type.bits == 32, "packed_attention: offsets are int32");
  p.offsets = reinterpret_cast<const int*>(offsets->memory);
  p.sequences = sequences, p.tokens = tokens, p.kv_heads = kv_heads, p.d = d, p.tiles = 0, p.group = Divisor(heads / kv_heads), p.scale = scale;
  // blocks of up to 512 threads
  CINN_RT_CHECK(((int64_t)tokens * p.group.value / 32 + sequences + 1) * kv_heads < 1 << 23, "packed_attention: too many rows or sequences");
  auto s = static_cast<hipStream_t>(stream);
  if (f32) {
    Launch<float>(p, s);
  } else if (f16) {
    Launch<_Float16>(p, s);
  } else {
    Launch<__bf16>(p, s);
  }
  CINN_HIP_CALL(hipGetLastError());
}
