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
#include <cstdlib>

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

// Every wavefront by itself, 64 sequences at a time.  Offsets out of order or range find rows in range all the same.
__device__ __forceinline__ Found Find(const PackedParams& p, int tile, int tile_pairs) {
  const int lane = threadIdx.x & 63;
  int before     = 0;
  for (int s0 = 0; s0 < p.sequences; s0 += 64) {
    int first = 0, count = 0;
    if (s0 + lane < p.sequences) {
      first = min(max(p.offsets[s0 + lane], 0), p.tokens);
      count = max(min(p.offsets[s0 + lane + 1], p.tokens) - first, 0);
    }
    const int tiles = (count * p.group.value + tile_pairs - 1) / tile_pairs;
    int sum = tiles;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int up = __shfl_up(sum, x);
      if (lane >= x) sum += up;
    }
    const unsigned long long behind = __ballot(before + sum > tile);
    if (behind) {
      const int at = __ffsll(behind) - 1;
      const int all = __builtin_amdgcn_readlane(tiles, at), here = tile - (before + __builtin_amdgcn_readlane(sum, at) - all);
      return {__builtin_amdgcn_readlane(first, at), __builtin_amdgcn_readlane(count, at), all - 1 - here, 0};  // the longest first
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

// D: d rounded up to an instance; WQ x 32 pairs per block, KG groups of wavefronts that take the tiles' keys in turn
template <typename T, int D, int WQ, int KG>
__global__ void __launch_bounds__(64 * WQ * KG, 2)
packed_attention_kernel(PackedParams p) {
  typedef Queries<T, D> Q;
  typedef Padded<T, D> L;
  constexpr int THREADS = 64 * WQ * KG, KT = 32 * KG, NC = L::NC;
  constexpr int V_AT = KT * L::K_PITCH, STAGE = V_AT + KT * L::V_PITCH;
  constexpr int MEET = (KG - 1) * WQ * 64 * Q::kRegisters * 4;
  __shared__ __attribute__((aligned(256))) char lds[2 * STAGE > MEET ? 2 * STAGE : MEET];

  // consecutive blocks, which are on different XCDs, take different key heads
  const int head = blockIdx.x % p.kv_heads;
  const Found at = Find(p, blockIdx.x / p.kv_heads, 32 * WQ);
  if (at.count == 0) {
    ClearRest<T>(p, head, at.tile, at.more);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / WQ, wq = wave % WQ;
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = at.count * p.group.value;
  const int pair0 = (at.tile * WQ + wq) * 32;  // of this wavefront
  const int pair = min(pair0 + (lane & 31), pairs - 1);
  const int query = p.group(pair), my_head = head * p.group.value + pair - query * p.group.value;
  const int first_query = p.group(min(pair0, pairs - 1)), last_query = pair0 < pairs ? p.group(min(pair0 + 31, pairs - 1)) : -1;
  const int keys = p.group(min((at.tile + 1) * WQ * 32, pairs) - 1) + 1;

  const int64_t k_row = p.k.row * sizeof(T), v_row = p.v.row * sizeof(T);
  const char* k_base = HeadOf<T>(p.k, 0, head) + at.first * k_row;
  const char* v_base = HeadOf<T>(p.v, 0, head) + at.first * v_row;
  constexpr int N = (KT * NC + THREADS - 1) / THREADS;
  u32x4 kr[N], vr[N];
  auto load = [&](int key0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (tid + i * THREADS) % NC, row = (tid + i * THREADS) / NC, key = key0 + row;
      kr[i] = vr[i] = u32x4{0, 0, 0, 0};
      if (key < keys && c < chunks && row < KT) {
        kr[i] = LoadAny<T>(k_base + key * k_row + c * 16);
        vr[i] = LoadAny<T>(v_base + key * v_row + c * 16);
      }
    }
  };
  auto store = [&](char* stage) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (tid + i * THREADS) % NC, row = (tid + i * THREADS) / NC;
      if (KT * NC % THREADS == 0 || row < KT) {
        *reinterpret_cast<u32x4*>(stage + row * L::K_PITCH + c * 16)        = kr[i];
        *reinterpret_cast<u32x4*>(stage + V_AT + row * L::V_PITCH + c * 16) = vr[i];
      }
    }
  };

  load(0);
  Q rows;
  rows.Start(HeadOf<T>(p.q, 0, my_head) + (at.first + query) * p.q.row * (int64_t)sizeof(T), chunks, half, p.scale);
  const Exp<T> ex(p.scale);
  store(lds);
  __syncthreads();
  const int tiles = (keys + KT - 1) / KT;
#pragma unroll 1
  for (int kt = 0; kt < tiles; ++kt) {
    const char* cur = lds + (kt & 1) * STAGE;
    if (kt + 1 < tiles) load((kt + 1) * KT);
    const int key0 = kt * KT + kg * 32;
    if (key0 <= last_query) {
      const unsigned word = key0 + 31 <= first_query ? ~0u : Below(query + 1 - key0);
      rows.Step(cur + kg * 32 * L::K_PITCH, cur + V_AT + kg * 32 * L::V_PITCH, word, chunks, ex, lane);
    }
    if (kt + 1 < tiles) {
      store(lds + ((kt + 1) & 1) * STAGE);
      __syncthreads();
    }
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
  // both halves of the wavefront hold this pair
  const float sum = rows.l + __shfl_xor(rows.l, 32);
  if (pair0 + (lane & 31) >= pairs) return;
  char* out = const_cast<char*>(HeadOf<T>(p.o, 0, my_head)) + (at.first + query) * p.o.row * (int64_t)sizeof(T);
  rows.Store(out, p.d, 1.0f / sum, half);
}

// 16-bit types: WQ x 32 pairs, KG wavefronts for each 32 that take the steps of 32 keys in turn, tiles of 32 STEPS keys in a
// ring of four in LDS that loads fill directly, one barrier per tile.  A wavefront multiplies the next 32 keys by its queries while it takes the exponentials of the last
// scores: the matrix cores and the vector unit work side by side, within a wavefront and, two of them to a SIMD, across.
// Rows behind the last key are rows of the tensor all the same; nothing attends to them.
template <typename T, int D, int WQ, int KG, int STEPS>
__global__ void __launch_bounds__(64 * WQ * KG, 2)
packed_attention_ring_kernel(PackedParams p) {
  typedef Dense<T, D> L;
  typedef Queries<T, D, L> Q;
  constexpr int KT = 32 * STEPS, NC = L::NC, STAGE = 2 * STEPS * L::BYTES, STAGES = 4;
  constexpr int N  = STEPS * NC / (WQ * KG);  // loads of a wavefront for a tile, whose values lie behind its keys
  constexpr int MEET = (KG - 1) * WQ * 64 * Q::kRegisters * 4;
  static_assert(N * WQ * KG == STEPS * NC && STEPS % KG == 0 && 2 * N < 64);
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
    const int load = wave * N + i;
    const bool values = load >= STEPS * NC / 2;
    const int slot = (values ? load - STEPS * NC / 2 : load) * 64 + lane, row = slot / NC;
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
      const int load = wave * N + i;
      const bool values = load >= STEPS * NC / 2;
      const char* from  = values ? v_tile : k_tile;
      if (chunks == NC && beyond <= 0) {
        CopyToLds16(from, off[i], to + load * 1024);
      } else {
        const int row  = ((values ? load - STEPS * NC / 2 : load) * 64 + lane) / NC;
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

template <typename T, int D, int WQ, int KG>
void LaunchBlocks(PackedParams p, hipStream_t stream) {
  p.tiles = (int)((int64_t)p.tokens * p.group.value / (32 * WQ)) + p.sequences + 1;
  hipLaunchKernelGGL((packed_attention_kernel<T, D, WQ, KG>), dim3((unsigned)p.tiles * p.kv_heads), dim3(64 * WQ * KG), 0, stream, p);
}

template <typename T, int D, int WQ, int KG, int STEPS>
void LaunchRing(PackedParams p, hipStream_t stream) {
  p.tiles = (int)((int64_t)p.tokens * p.group.value / (32 * WQ)) + p.sequences + 1;
  hipLaunchKernelGGL((packed_attention_ring_kernel<T, D, WQ, KG, STEPS>), dim3((unsigned)p.tiles * p.kv_heads), dim3(64 * WQ * KG), 0, stream, p);
}

template <typename T, int D>
void LaunchTiles(const PackedParams& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    static const char* pick = getenv("PICK");
    const int which = pick ? atoi(pick) : 0;
    if (which == 0) return LaunchRing<T, D, 8, 1, 2>(p, stream);
    if (which == 2) return LaunchRing<T, D, 4, 1, 1>(p, stream);
    if (which == 3) return LaunchRing<T, D, 4, 2, 2>(p, stream);
  }
  // blocks of few pairs where there are few
  const int64_t pairs = (int64_t)p.tokens * p.group.value * p.kv_heads;
  if (pairs >= 256 * 128) {
    LaunchBlocks<T, D, 4, 2>(p, stream);
  } else {
    LaunchBlocks<T, D, 1, 2>(p, stream);
  }
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
  CINN_RT_CHECK((int64_t)tokens * d * std::max(std::max(q_heads, k_heads), v_heads) < INT_MAX, "packed_attention: tensor too large");
  auto input = [&](int slot) {
    const int at = (operands >> (4 * slot)) & 15;
    CINN_RT_CHECK(at < num_args - 1, "packed_attention: operand %d is argument %d of %d", slot, at, num_args);
    return BufferArg(v_args, at);
  };
  auto rows = [&](int slot, int total, int first) {
    const cinn_buffer_t* b = input(slot);
    CINN_RT_CHECK(b->type.code == out->type.code && b->type.bits == out->type.bits, "packed_attention: operands of different types");
    return Rows{b->memory + (int64_t)first * d * (f32 ? 4 : 2), 0, d, (int64_t)total * d};
  };
  PackedParams p;
  p.q = rows(0, q_heads, q_head), p.k = rows(1, k_heads, k_head), p.v = rows(2, v_heads, v_head);
  p.o = Rows{out->memory, 0, d, (int64_t)heads * d};
  const cinn_buffer_t* offsets = input(3);
  CINN_RT_CHECK(offsets->type.code == cinn_type_int && offsets->type.bits == 32, "packed_attention: offsets are int32");
  p.offsets = reinterpret_cast<const int*>(offsets->memory);
  p.sequences = sequences, p.tokens = tokens, p.kv_heads = kv_heads, p.d = d, p.tiles = 0, p.group = Divisor(heads / kv_heads), p.scale = scale;
  CINN_RT_CHECK(((int64_t)tokens * p.group.value / 32 + sequences + 1) * kv_heads < INT_MAX, "packed_attention: too many tiles");
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
