// Attention of a few new tokens per sequence over a paged cache and each other for gfx950, fp16 / bf16 / fp32: decode steps (one
// token), chains and trees of drafted ones.  O = softmax(scale Q K^T, masked) V per sequence and head, query head h reading
// key head h / group.
//
// Bound by one read of the cache: a block takes the (token, head of the group) pairs of one key head together, so that
// every key and value row is read once for all of them, and works through a run of key tiles.  The lengths are data: all
// tiles of all sequences and key heads form one list that the blocks divide evenly, whatever the lengths are.  A block that
// has all tiles of a unit (key head, run of pairs) writes its result; the others leave their sums, maxima and totals in
// scratch and a second kernel joins them, in order.
//
// The new tokens are the last keys of a sequence.  Which of them a token attends to is a word of 64 bits, found from the
// parents by doubling: six rounds of every token taking its pointer's word and pointer.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "cinn_hip_runtime.h"
#include "kernels/attention_tile.h"
#include "runtime/hip_check.h"
#include "runtime/scratch.h"

namespace {

using namespace cinn_hip_kernels::attention;

struct CachedParams {
  Rows q, k, v, o;  // of the new tokens and the first head in use
  const char *k_pages, *v_pages;
  int64_t page, row, head;  // strides of the pages in elements
  const int *table, *lengths, *parents;
  int batch, tokens, kv_heads, d, pages, columns;
  Divisor page_rows, group;
  int units;    // of a sequence: key heads x runs of pairs
  int blocks;   // that divide the list of tiles; 0: every block has a unit
  float* parts;
  float scale;
};

__device__ __forceinline__ int LengthOf(const CachedParams& p, int b) {
  return min(max(p.lengths[b], 0), p.columns * p.page_rows.value);
}

// Where item `item` of the list of all tiles lies: its sequence, that one's rows in the cache and first item.  With item < 0
// only the items are counted.  By every wavefront for itself, 64 sequences at a time.
struct Place {
  int b, length;
  int64_t first, count;
};
__device__ __forceinline__ Place Find(const CachedParams& p, int64_t item, int keys_per_tile) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int length = b0 + lane < p.batch ? LengthOf(p, b0 + lane) : 0;
    const int64_t mine = b0 + lane < p.batch ? (int64_t)((length + p.tokens + keys_per_tile - 1) / keys_per_tile) * p.units : 0;
    int64_t sum = mine;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int64_t up = __shfl_up((long long)sum, x);
      if (lane >= x) sum += up;
    }
    const unsigned long long behind = item < 0 ? 0 : __ballot(before + sum > item);
    if (behind) {
      const int at = __ffsll(behind) - 1;
      return {b0 + at, __shfl(length, at), before + __shfl((long long)(sum - mine), at), __shfl((long long)mine, at)};
    }
    before += __shfl((long long)sum, 63);
  }
  return {0, 0, 0, before};
}

// which new tokens token `token` (of this lane) attends to, itself among them; none: it is no token
__device__ __forceinline__ unsigned long long SeenBy(const CachedParams& p, int b, int token) {
  if (!p.parents) return ~0ull >> (63 - token);
  const int lane = threadIdx.x & 63;
  const int parent = lane < p.tokens ? p.parents[(int64_t)b * p.tokens + lane] : -2;
  const bool real = parent >= -1 && parent < lane;
  unsigned long long word = real ? 1ull << lane : 0;
  int pointer = real ? parent : -1;
#pragma unroll
  for (int round = 0; round < 6; ++round) {
    const unsigned long long theirs = __shfl(word, max(pointer, 0));
    const int next = __shfl(pointer, max(pointer, 0));
    if (pointer >= 0) word |= theirs, pointer = next;
  }
  return __shfl(word, token);
}

// D: d rounded up to an instance; WQ x 32 pairs per block, KG groups of wavefronts that take the tiles' keys in turn
template <typename T, int D, int WQ, int KG>
__global__ void __launch_bounds__(64 * WQ * KG)
cached_attention_kernel(CachedParams p) {
  typedef Queries<T, D> Q;
  typedef Layout<T, D> L;
  constexpr int THREADS = 64 * WQ * KG, KT = 32 * KG, NC = L::NC;
  constexpr int V_AT = KT * L::K_PITCH, HOLDS_AT = V_AT + KT * L::V_PITCH, STAGE = HOLDS_AT + KT;
  constexpr int MEET = (KG - 1) * WQ * 64 * Q::kRegisters * 4;
  __shared__ __attribute__((aligned(256))) char lds[2 * STAGE > MEET ? 2 * STAGE : MEET];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / WQ, wq = wave % WQ;
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = p.tokens * p.group.value;
  const Exp<T> ex(p.scale);

  int64_t at, end;  // this block's items
  Place place;
  if (p.blocks > 0) {
    // no more blocks than items: every block that the second kernel looks at has some
    const int64_t total = Find(p, -1, KT).count, blocks = min((int64_t)p.blocks, total);
    if (blockIdx.x >= blocks) return;
    at = total * blockIdx.x / blocks, end = total * (blockIdx.x + 1) / blocks;
    place = Find(p, at, KT);
  } else {
    const int b = blockIdx.x / p.units, length = LengthOf(p, b), tiles = (length + p.tokens + KT - 1) / KT;
    at = (int64_t)(blockIdx.x % p.units) * tiles, end = at + tiles;
    place = {b, length, 0, (int64_t)tiles * p.units};
  }
#pragma unroll 1
  while (at < end) {
    if (at >= place.first + place.count) place = Find(p, at, KT);
    const int b = place.b, length = place.length, keys = length + p.tokens, tiles = (keys + KT - 1) / KT;
    const int64_t inside = at - place.first;
    const int unit = (int)(inside / tiles), tile0 = (int)(inside - (int64_t)unit * tiles);
    const int tile1 = (int)min((int64_t)tiles, tile0 + end - at);
    const int head = unit % p.kv_heads, pair0 = (unit / p.kv_heads * WQ + wq) * 32;
    const int pair = min(pair0 + (lane & 31), pairs - 1), token = p.group(pair), my_head = head * p.group.value + pair - token * p.group.value;
    const unsigned long long seen = SeenBy(p, b, token);

    const char* k_new = HeadOf<T>(p.k, b, head);
    const char* v_new = HeadOf<T>(p.v, b, head);
    const int* table  = p.table + (int64_t)b * p.columns;
    constexpr int N = (KT * NC + THREADS - 1) / THREADS;
    u32x4 kr[N], vr[N];
    bool holds[N];
    auto load = [&](int key0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (tid + i * THREADS) % NC, row = (tid + i * THREADS) / NC, key = key0 + row;
        kr[i] = vr[i] = u32x4{0, 0, 0, 0};
        holds[i]      = false;
        if (key >= keys || row >= KT) continue;
        const char *k_row, *v_row;
        if (key < length) {
          const int column = p.page_rows(key), page = table[column];
          if (page < 0 || page >= p.pages) continue;
          const int64_t off = (page * p.page + (key - column * p.page_rows.value) * p.row + head * p.head) * (int64_t)sizeof(T);
          k_row = p.k_pages + off, v_row = p.v_pages + off;
        } else {
          k_row = k_new + (key - length) * p.k.row * (int64_t)sizeof(T), v_row = v_new + (key - length) * p.v.row * (int64_t)sizeof(T);
        }
        holds[i] = true;
        if (c < chunks) kr[i] = LoadAny<T>(k_row + c * 16), vr[i] = LoadAny<T>(v_row + c * 16);
      }
    };
    auto store = [&](char* stage) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (tid + i * THREADS) % NC, row = (tid + i * THREADS) / NC;
        if (KT * NC % THREADS == 0 || row < KT) {
          *reinterpret_cast<u32x4*>(stage + row * L::K_PITCH + c * 16)        = kr[i];
          *reinterpret_cast<u32x4*>(stage + V_AT + row * L::V_PITCH + c * 16) = vr[i];
          if (c == 0) stage[HOLDS_AT + row] = holds[i];
        }
      }
    };

    load(tile0 * KT);
    Q rows;
    rows.Start(HeadOf<T>(p.q, b, my_head) + token * p.q.row * (int64_t)sizeof(T), chunks, half, p.scale);
    store(lds);
    __syncthreads();
#pragma unroll 1
    for (int kt = tile0; kt < tile1; ++kt) {
      const char* cur = lds + ((kt - tile0) & 1) * STAGE;
      if (kt + 1 < tile1) load((kt + 1) * KT);
      const int key0 = kt * KT + kg * 32, j0 = key0 - length;
      if (key0 < keys && pair0 < pairs) {
        unsigned word = j0 >= 0 ? (unsigned)(seen >> min(j0, 63)) : j0 <= -32 ? ~0u : (unsigned)(seen << -j0) | Below(-j0);
        word &= (unsigned)__ballot(cur[HOLDS_AT + kg * 32 + (lane & 31)] != 0);
        if (seen == 0) word = 0;
        rows.Step(cur + kg * 32 * L::K_PITCH, cur + V_AT + kg * 32 * L::V_PITCH, word, chunks, ex, lane);
      }
      if (kt + 1 < tile1) {
        store(lds + ((kt + 1 - tile0) & 1) * STAGE);
        __syncthreads();
      }
    }
    if constexpr (KG > 1) {
      __syncthreads();
      float* meet = reinterpret_cast<float*>(lds);
      if (kg > 0) rows.Hand(meet + ((kg - 1) * WQ + wq) * Q::kRegisters * 64, lane);
      __syncthreads();
      if (kg == 0) {
#pragma unroll
        for (int g = 1; g < KG; ++g) rows.Join(meet + ((g - 1) * WQ + wq) * Q::kRegisters * 64, ex, lane);
      }
    }
    __syncthreads();  // the next unit's tiles may overwrite what was read here
    if (kg == 0) {
      // both halves of the wavefront hold this pair
      rows.l += __shfl_xor(rows.l, 32);
      if (tile0 == 0 && tile1 == tiles) {
        if (pair0 + (lane & 31) < pairs) {
          char* out = const_cast<char*>(HeadOf<T>(p.o, b, my_head)) + token * p.o.row * (int64_t)sizeof(T);
          rows.Store(out, p.d, seen == 0 ? 0.0f : 1.0f / rows.l, half);
        }
      } else {
        // a block has at most one run that begins inside a unit, and one that ends inside
        if (seen == 0) rows.l = -1.0f;
        rows.Hand(p.parts + ((int64_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * WQ + wq) * Q::kRegisters * 64, lane);
      }
    }
    at += tile1 - tile0;
  }
}

// Units whose tiles several blocks had: a wavefront takes 4 of the 16 registers of each 32 elements of d, of 32 pairs.
template <typename T, int D, int WQ, int KG>
__global__ void __launch_bounds__(64)
cached_attention_join_kernel(CachedParams p) {
  typedef Queries<T, D> Q;
  typedef Layout<T, D> L;
  constexpr int KT = 32 * KG, QUARTERS = L::DT * 4;
  const int lane = threadIdx.x, quarter = blockIdx.x % QUARTERS, wq = blockIdx.x / QUARTERS % WQ, which = blockIdx.x / QUARTERS / WQ;
  const int b = which / p.units, unit = which % p.units, pairs = p.tokens * p.group.value;
  const int pair = (unit / p.kv_heads * WQ + wq) * 32 + (lane & 31);
  if ((unit / p.kv_heads * WQ + wq) * 32 >= pairs || quarter * 8 >= p.d) return;
  int64_t total = 0, first = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int64_t mine = 0;
    if (b0 + lane < p.batch) mine = (int64_t)((LengthOf(p, b0 + lane) + p.tokens + KT - 1) / KT) * p.units;
    int64_t before = b0 + lane < b ? mine : 0;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) mine += __shfl_xor((long long)mine, x), before += __shfl_xor((long long)before, x);
    total += mine, first += before;
  }
  const int tiles = (LengthOf(p, b) + p.tokens + KT - 1) / KT;
  first += (int64_t)unit * tiles;
  const int64_t blocks = min((int64_t)p.blocks, total);
  const int block0 = (int)(((first + 1) * blocks - 1) / total), block1 = (int)(((first + tiles) * blocks - 1) / total);
  if (block0 == block1) return;  // that block has written the result
  auto part = [&](int block) {
    return p.parts + ((int64_t)(2 * block + (block == block0 ? 1 : 0)) * WQ + wq) * Q::kRegisters * 64 + lane;
  };
  const Exp<T> ex(p.scale);
  float top = -__builtin_inff();
#pragma unroll 4
  for (int i = block0; i <= block1; ++i) top = fmaxf(top, part(i)[(Q::kRegisters - 2) * 64]);
  const float base = ex.Base(top);
  float sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = block0; i <= block1; ++i) {
    const float* from = part(i);
    const float f     = ex(from[(Q::kRegisters - 2) * 64], base);
    sum               = __builtin_fmaf(from[(Q::kRegisters - 1) * 64], f, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(from[(quarter * 4 + e) * 64], f, o[e]);
  }
  const bool token_is_none = part(block0)[(Q::kRegisters - 1) * 64] < 0.0f;
  if (pair >= pairs) return;
  const int token = p.group(pair), my_head = unit % p.kv_heads * p.group.value + pair - token * p.group.value;
  const int at = quarter / 4 * 32 + quarter % 4 * 8 + 4 * (lane >> 5);
  T four[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) four[e] = (T)(token_is_none ? 0.0f : o[e] / sum);
  char* out = const_cast<char*>(HeadOf<T>(p.o, b, my_head)) + (token * p.o.row + at) * (int64_t)sizeof(T);
  if (at < p.d) __builtin_memcpy(out, four, sizeof(four));
}

template <typename T, int D, int WQ, int KG>
void LaunchBlocks(CachedParams p, hipStream_t stream) {
  constexpr int KT = 32 * KG, kMostBlocks = 256;
  const int pairs  = p.tokens * p.group.value;
  p.units          = p.kv_heads * ((pairs + 32 * WQ - 1) / (32 * WQ));
  const int units  = p.batch * p.units;
  const int64_t most_tiles = ((int64_t)p.columns * p.page_rows.value + p.tokens + KT - 1) / KT;
  p.blocks = 0;
  if (most_tiles > 4) {
    const int blocks   = (int)std::min<int64_t>(kMostBlocks, units * most_tiles);
    const size_t bytes = (size_t)2 * blocks * WQ * Queries<T, D>::kRegisters * 64 * sizeof(float);
    if (bytes <= cinn_hip_kernels::ScratchLimit(cinn_hip_kernels::ScratchKind::kSplitK, stream)) {
      p.blocks = blocks;
      p.parts  = static_cast<float*>(cinn_hip_kernels::Scratch(cinn_hip_kernels::ScratchKind::kSplitK, bytes, stream));
    }
  }
  hipLaunchKernelGGL((cached_attention_kernel<T, D, WQ, KG>), dim3((unsigned)(p.blocks > 0 ? p.blocks : units)), dim3(64 * WQ * KG), 0, stream, p);
  if (p.blocks > 0)
    hipLaunchKernelGGL((cached_attention_join_kernel<T, D, WQ, KG>), dim3((unsigned)(units * WQ * Layout<T, D>::DT * 4)), dim3(64), 0, stream, p);
}

template <typename T, int D>
void LaunchTiles(const CachedParams& p, hipStream_t stream) {
  const int pairs = p.tokens * p.group.value;
  if (pairs <= 32) {
    LaunchBlocks<T, D, 1, sizeof(T) == 4 ? 2 : 4>(p, stream);
  } else {
    LaunchBlocks<T, D, 4, 2>(p, stream);
  }
}

template <typename T>
void Launch(const CachedParams& p, hipStream_t stream) {
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
  CINN_RT_CHECK(args[index].type_code_ == CINN_POD_BUFFER_P, "cached_attention: argument %d is not a buffer", index);
  auto* b = static_cast<cinn_buffer_t*>(args[index].value_.v_handle);
  CINN_RT_CHECK(b && b->memory, "cached_attention: argument %d has no device memory", index);
  return b;
}

}  // namespace

extern "C" void cinn_call_hip_cached_attention(void* v_args, int num_args, float scale, int batch, int tokens, int heads, int kv_heads, int d,
                                               int pages, int page_rows, int page_layout, int columns, int operands, int q_heads, int q_head,
                                               int k_heads, int k_head, int v_heads, int v_head, void* stream) {
  CINN_HIP_CLEAR_STALE_ERROR();
  CINN_RT_CHECK(batch >= 0 && tokens >= 0 && tokens <= 64, "cached_attention: %d sequences, %d new tokens each (at most 64)", batch, tokens);
  CINN_RT_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "cached_attention: %d heads, %d key heads", heads, kv_heads);
  CINN_RT_CHECK(d > 0 && d <= 128, "cached_attention: %d elements per row (at most 128)", d);
  CINN_RT_CHECK(pages > 0 && page_rows > 0 && columns > 0 && (int64_t)columns * page_rows < (1 << 30) && (page_layout == 0 || page_layout == 1),
                "cached_attention: %d pages of %d rows, %d in a sequence, layout %d", pages, page_rows, columns, page_layout);
  CINN_RT_CHECK(q_head >= 0 && k_head >= 0 && v_head >= 0 && q_head + heads <= q_heads && k_head + kv_heads <= k_heads && v_head + kv_heads <= v_heads,
                "cached_attention: heads outside their tensors");
  if ((int64_t)batch * tokens == 0) return;
  const cinn_buffer_t* out = BufferArg(v_args, num_args - 1);
  const bool f32 = out->type.code == cinn_type_float && out->type.bits == 32;
  const bool f16 = out->type.code == cinn_type_float && out->type.bits == 16;
  CINN_RT_CHECK(f32 || f16 || (out->type.code == cinn_type_bfloat && out->type.bits == 16), "cached_attention: fp16 / bf16 / fp32 only");
  CINN_RT_CHECK(d % (f32 ? 4 : 8) == 0, "cached_attention: rows of %d elements are no whole number of 16-byte chunks", d);
  CINN_RT_CHECK((int64_t)batch * tokens * d * std::max(std::max(q_heads, k_heads), v_heads) < INT_MAX && (int64_t)batch * columns < INT_MAX &&
                    (int64_t)pages * page_rows * kv_heads * d < ((int64_t)1 << 40),
                "cached_attention: tensor too large");
  auto input = [&](int slot) {
    const int at = ((unsigned)operands >> (4 * slot)) & 15;
    CINN_RT_CHECK(at < num_args - 1, "cached_attention: operand %d is argument %d of %d", slot, at, num_args);
    return BufferArg(v_args, at);
  };
  auto typed = [&](int slot) {
    const cinn_buffer_t* b = input(slot);
    CINN_RT_CHECK(b->type.code == out->type.code && b->type.bits == out->type.bits, "cached_attention: operands of different types");
    return b->memory;
  };
  auto whole = [&](int slot) {
    const cinn_buffer_t* b = input(slot);
    CINN_RT_CHECK(b->type.code == cinn_type_int && b->type.bits == 32, "cached_attention: table, lengths and parents are int32");
    return reinterpret_cast<const int*>(b->memory);
  };
  auto rows = [&](const uint8_t* memory, int total, int first) {
    return Rows{memory + (int64_t)first * d * (f32 ? 4 : 2), (int64_t)tokens * total * d, d, (int64_t)total * d};
  };
  CachedParams p = {};
  p.q = rows(typed(0), q_heads, q_head), p.k = rows(typed(1), k_heads, k_head), p.v = rows(typed(2), v_heads, v_head);
  p.o       = rows(out->memory, heads, 0);
  p.k_pages = reinterpret_cast<const char*>(typed(3)), p.v_pages = reinterpret_cast<const char*>(typed(4));
  p.page = (int64_t)page_rows * kv_heads * d;
  p.row  = page_layout == 0 ? (int64_t)kv_heads * d : d;
  p.head = page_layout == 0 ? d : (int64_t)page_rows * d;
  p.table = whole(5), p.lengths = whole(6), p.parents = ((unsigned)operands >> 28) == 15 ? nullptr : whole(7);
  p.batch = batch, p.tokens = tokens, p.kv_heads = kv_heads, p.d = d, p.pages = pages, p.columns = columns;
  p.page_rows = Divisor(page_rows), p.group = Divisor(heads / kv_heads), p.scale = scale;
  CINN_RT_CHECK((int64_t)batch * heads * tokens < (1 << 24), "cached_attention: too many rows");
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
