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

// What a block's change of units costs beside its tiles, in tiles: every unit has that many empty items in front, so that the
// blocks with many short sequences have fewer of them.  us without | with one: bf16 48 sequences of 100 to 16000 rows, 32 heads
// over 8 x 128, 178 | 153, of 100 to 4000 58 | 45, 8 trees of 48 tokens 68 | 66; with two or three 159 and 161 instead of 157.
constexpr int kEmpty = 1;

// what lane `lane` has, in scalar registers
__device__ __forceinline__ int64_t OfLane(int64_t v, int lane) {
  return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readlane((unsigned)((uint64_t)v >> 32), lane) << 32 |
                   (unsigned)__builtin_amdgcn_readlane((unsigned)v, lane));
}

// Which sequence item `item` of the list of all tiles belongs to, and that one's first item; with item < 0 how many items there
// are.  By every wavefront for itself, 64 sequences at a time.
struct Place {
  int b;
  int64_t first;
};
__device__ __forceinline__ Place Find(const CachedParams& p, int64_t item, int keys_per_tile) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int length = b0 + lane < p.batch ? LengthOf(p, b0 + lane) : 0;
    const int64_t mine = b0 + lane < p.batch ? (int64_t)((length + p.tokens + keys_per_tile - 1) / keys_per_tile + kEmpty) * p.units : 0;
    int64_t sum = mine;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int64_t up = __shfl_up((long long)sum, x);
      if (lane >= x) sum += up;
    }
    const unsigned long long behind = item < 0 ? 0 : __ballot(before + sum > item);
    if (behind) {
      const int at = __ffsll(behind) - 1;
      return {b0 + at, before + OfLane(sum - mine, at)};
    }
    before += OfLane(sum, 63);
  }
  return {0, before};
}

// A block's share of the list: runs of tiles tile0 .. tile1 - 1 of the `tiles` of a unit, one after the other.
struct Share {
  int b, unit, length, tiles, tile0, tile1;
  int next, item;  // the unit and the item of it that the next run begins with
  int64_t left;    // items
  __device__ __forceinline__ Share(const CachedParams& p, int keys_per_tile) {
    if (p.blocks > 0) {
      // no more blocks than items: every block that the second kernel looks at has some
      const int64_t total = Find(p, -1, keys_per_tile).first, blocks = min((int64_t)p.blocks, total);
      left = 0;
      if (blockIdx.x >= blocks) return;
      const int64_t at  = total * blockIdx.x / blocks;
      const Place place = Find(p, at, keys_per_tile);
      left = total * (blockIdx.x + 1) / blocks - at;
      Open(p, place.b, keys_per_tile);
      next = (int)((at - place.first) / (tiles + kEmpty));
      item = (int)(at - place.first - (int64_t)next * (tiles + kEmpty));
    } else {
      Open(p, blockIdx.x / p.units, keys_per_tile);
      next = blockIdx.x % p.units, item = 0, left = tiles + kEmpty;
    }
  }
  __device__ __forceinline__ void Open(const CachedParams& p, int sequence, int keys_per_tile) {
    b = sequence, length = LengthOf(p, sequence), tiles = (length + p.tokens + keys_per_tile - 1) / keys_per_tile;
  }
  __device__ __forceinline__ bool Next(const CachedParams& p, int keys_per_tile) {
    while (left > 0) {
      if (next == p.units) Open(p, b + 1, keys_per_tile), next = 0;
      const int end = (int)min((int64_t)tiles + kEmpty, item + left);
      tile0 = max(item - kEmpty, 0), tile1 = end - kEmpty, unit = next++;
      left -= end - item, item = 0;
      if (tile0 < tile1) return true;
    }
    return false;
  }
};

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

// What becomes of a run of a unit's tiles: the result where it is all of them, otherwise a part for the second kernel.  A
// block has at most one run that begins inside a unit, and one that ends inside.
template <typename T, int D, class Q>
__device__ __forceinline__ void Finish(const CachedParams& p, Q& rows, int b, int head, int pair0, int lane, bool begins, bool ends, int runs,
                                       int run, unsigned long long seen) {
  rows.l += __shfl_xor(rows.l, 32);  // both halves of the wavefront hold the pair
  if (begins && ends) {
    const int pair = pair0 + (lane & 31), token = p.group(pair), group = p.group.value;
    if (pair >= p.tokens * group) return;
    char* out = const_cast<char*>(HeadOf<T>(p.o, b, head * group + pair - token * group)) + token * p.o.row * (int64_t)sizeof(T);
    rows.Store(out, p.d, seen == 0 ? 0.0f : 1.0f / rows.l, lane >> 5);
  } else {
    if (seen == 0) rows.l = -1.0f;
    rows.Hand(p.parts + ((int64_t)(2 * blockIdx.x + (begins ? 1 : 0)) * runs + run) * Q::kRegisters * 64, lane);
  }
}

// More than 32 pairs in fp32: 4 x 32 pairs per block, two wavefronts for each 32 that take the tiles' keys in turn, tiles of 64
// keys through registers into two buffers in LDS.  D: d rounded up to an instance.  8 trees of 48 tokens over 2000 to 5000 rows, 32 heads
// over 8 x 128, 410 us; the products alone would take 144.
template <int D>
__global__ void __launch_bounds__(512)
cached_attention_float_kernel(CachedParams p) {
  typedef float T;
  typedef Padded<D> L;
  typedef Queries<T, D, L> Q;
  constexpr int WQ = 4, KG = 2, THREADS = 64 * WQ * KG, KT = 32 * KG, NC = L::NC;
  constexpr int V_AT = KT * L::K_PITCH, HOLDS_AT = V_AT + KT * L::V_PITCH, STAGE = HOLDS_AT + KT;
  constexpr int MEET = WQ * 64 * Q::kRegisters * 4;
  __shared__ __attribute__((aligned(256))) char lds[2 * STAGE > MEET ? 2 * STAGE : MEET];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / WQ, wq = wave % WQ;
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = p.tokens * p.group.value;
  const Exp<T> ex(p.scale);

  Share share(p, KT);
#pragma unroll 1
  while (share.Next(p, KT)) {
    const int b = share.b, unit = share.unit, length = share.length, keys = length + p.tokens;
    const int tiles = share.tiles, tile0 = share.tile0, tile1 = share.tile1;
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
    __syncthreads();
    float* meet = reinterpret_cast<float*>(lds) + wq * Q::kRegisters * 64;
    if (kg > 0) rows.Hand(meet, lane);
    __syncthreads();
    if (kg == 0) rows.Join(meet, ex, lane);
    __syncthreads();  // the next unit's tiles may overwrite what was read here
    if (kg == 0) Finish<T, D>(p, rows, b, head, pair0, lane, tile0 == 0, tile1 == tiles, WQ, wq, seen);
  }
}

// At most 16 PT pairs, bound by the cache's bytes: a wavefront streams 32 keys of every tile through buffers of its own in LDS,
// STAGES deep for keys and for values, that loads fill directly, and meets the others at the end of a unit only.  The next keys
// are requested as soon as the scores are there, the next values when they are summed.  Which pages the rows lie in comes the same way, STAGES
// tiles ahead of them: every wavefront's loads land in order, so that one count tells what has.  Measured: 48 sequences of 100 to
// 16000 bf16 rows, 32 heads over 8 x 128, 154 us, 5.0 TB/s; one of 100003 fp32 rows, 16 over 4 x 96, 72 us, 4.3 TB/s (96 KiB of
// loads in flight on a CU, less while their scores are taken); 8 of 511 fp16 rows, 12 x 64, 7.3 us, of which a launch is 4.
// Wavefronts with tiles shared through registers took 567, 345 and 23.
template <typename T, int D, int PT, int WAVES, int STAGES>
__global__ void __launch_bounds__(64 * WAVES, (WAVES + 3) / 4)
cached_attention_few_kernel(CachedParams p) {
  typedef FewPairs<T, D, PT> Q;
  typedef Dense<T, D> L;
  static_assert(STAGES == 1 || STAGES == 2);
  constexpr int KT = 32 * WAVES, NC = L::NC, N = NC / 2;  // N: loads for a tile of keys or of values
  constexpr int RPL = 64 / NC;                            // rows per load, where that is a whole number
  constexpr int IDS = 4 * STAGES, IDS_AT = STAGES * 2 * L::BYTES, ROWS_AT = IDS_AT + IDS * 256, WAVE = ROWS_AT + STAGES * 32 * 16;
  constexpr int MEET = WAVES * PT * 64 * Q::kRegisters * 4;
  __shared__ __attribute__((aligned(256))) char lds[WAVES * WAVE > MEET ? WAVES * WAVE : MEET];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = p.tokens * p.group.value;
  const Exp<T> ex(p.scale);
  char* mine = lds + wave * WAVE;
  const unsigned mine_at = LdsAddress(mine);
  // rows of whole loads in one page: a load has one base
  const bool even_rows = L::POW2 && chunks == NC && p.page_rows.value % (L::POW2 ? RPL : 1) == 0;
  const int row_bytes  = (int)(p.row * sizeof(T));
  constexpr int TURNS  = NC == 32 ? 8 : NC == 16 ? 4 : NC == 8 ? 2 : 1;  // places of a row's chunks repeat with every TURNS loads
  int k_off[TURNS], v_off[TURNS];
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    k_off[j] = lane / NC * row_bytes + L::Back(lane % NC, L::KTurn(j * RPL + lane / NC)) * 16;
    v_off[j] = lane / NC * row_bytes + L::Back(lane % NC, L::RowTurn(j * RPL + lane / NC)) * 16;
  }

  Share share(p, KT);
#pragma unroll 1
  while (share.Next(p, KT)) {
    const int b = share.b, head = share.unit, length = share.length, keys = length + p.tokens;
    const int tiles = share.tiles, tile0 = share.tile0, tile1 = share.tile1, last = tile1 - 1;
    const char* k_new = HeadOf<T>(p.k, b, head);
    const char* v_new = HeadOf<T>(p.v, b, head);
    const int* table  = p.table + (int64_t)b * p.columns;

    auto request_pages = [&](int kt) {
      const int key = min(kt * KT + wave * 32 + (lane & 31), max(length - 1, 0));
      CopyToLds4(table + p.page_rows(key), mine_at + IDS_AT + kt % IDS * 256);
    };
    // where a tile's rows lie: the offset in the pages of the lane's key's row, or with a key that is none or new among the 32
    // the rows' addresses in LDS
    int64_t off[STAGES];
    unsigned holds[STAGES];  // which of the 32 keys are some
    bool plain[STAGES];
    struct Two { const char *k, *v; };
    auto place_rows = [&](int kt, int stage) {
      const int key = kt * KT + wave * 32 + (lane & 31);
      const int page = *reinterpret_cast<const int*>(mine + IDS_AT + kt % IDS * 256 + (lane & 31) * 4);
      const bool good = key < length && page >= 0 && page < p.pages;
      const int64_t offset = good ? (page * p.page + (key - p.page_rows(key) * p.page_rows.value) * p.row + head * p.head) * (int64_t)sizeof(T) : 0;
      const unsigned word = (unsigned)__ballot(good || (key >= length && key < keys));
      const bool straight = even_rows && __ballot(good) == ~0ull;
#pragma unroll
      for (int s = 0; s < STAGES; ++s)
        if (stage == s) off[s] = offset, holds[s] = word, plain[s] = straight;
      if (!straight) {
        Two row = {reinterpret_cast<const char*>(kZeros), reinterpret_cast<const char*>(kZeros)};
        if (good) row = {p.k_pages + offset, p.v_pages + offset};
        if (key >= length && key < keys)
          row = {k_new + (key - length) * p.k.row * (int64_t)sizeof(T), v_new + (key - length) * p.v.row * (int64_t)sizeof(T)};
        if (lane < 32) reinterpret_cast<Two*>(mine + ROWS_AT)[stage * 32 + lane] = row;
      }
    };
    auto request = [&](int stage, bool values) {
      const unsigned to = mine_at + (2 * stage + values) * L::BYTES;
      bool straight = plain[0];
      int64_t offset = off[0];
#pragma unroll
      for (int s = 1; s < STAGES; ++s)
        if (stage == s) straight = plain[s], offset = off[s];
      if (straight) {
        const char* pages = values ? p.v_pages : p.k_pages;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const unsigned low = __builtin_amdgcn_readlane((unsigned)offset, j * RPL % 32);
          const unsigned high = __builtin_amdgcn_readlane((unsigned)(offset >> 32), j * RPL % 32);
          CopyToLds16(pages + (int64_t)((uint64_t)high << 32 | low), (unsigned)(values ? v_off : k_off)[j % TURNS], to + j * 1024);
        }
      } else {
        const Two* rows = reinterpret_cast<const Two*>(mine + ROWS_AT) + stage * 32;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int slot = j * 64 + lane, row = slot / NC, c = L::Back(slot % NC, values ? L::RowTurn(row) : L::KTurn(row));
          const char* from = values ? rows[row].v : rows[row].k;
          CopyToLds16(c < chunks ? from + c * 16 : reinterpret_cast<const char*>(kZeros), to + j * 1024);
        }
      }
    };

#pragma unroll
    for (int i = 0; i < STAGES; ++i) request_pages(min(tile0 + i, last));
    Q rows;
    unsigned long long seen[PT];
#pragma unroll
    for (int n = 0; n < PT; ++n) {
      const int pair = min(n * 16 + (lane & 15), pairs - 1), token = p.group(pair), my_head = head * p.group.value + pair - token * p.group.value;
      rows.Start(n, HeadOf<T>(p.q, b, my_head) + token * p.q.row * (int64_t)sizeof(T), chunks, lane, p.scale);
      seen[n] = SeenBy(p, b, token);
    }
    WaitForAllBut<0>();
#pragma unroll
    for (int i = 0; i < STAGES; ++i) {
      if (tile0 + i > last) break;
      request_pages(min(tile0 + STAGES + i, last));
      place_rows(tile0 + i, i);
      request(i, false);
      request(i, true);
    }
    int stage = 0;
#pragma unroll 1
    for (int kt = tile0; kt < tile1; ++kt) {
      const bool more = kt + STAGES <= last;
      const int behind = min(last - kt, STAGES - 1);  // tiles that are on their way behind this one
      const char* cur = mine + stage * 2 * L::BYTES;
      if (STAGES > 1 && behind == 1) {
        WaitForAllBut<N + (STAGES > 1 ? 1 : 0) * (2 * N + 1)>();
      } else {
        WaitForAllBut<N>();
      }
      asm volatile("" ::: "memory");
      f32x4 s[PT][2];
      rows.Scores(s, cur, lane);
      unsigned some = holds[0];
#pragma unroll
      for (int n = 1; n < STAGES; ++n) some = stage == n ? holds[n] : some;
      if (more) {
        __builtin_amdgcn_s_waitcnt(0xC07F);  // the keys have been read
        request_pages(min(kt + 2 * STAGES, last));
        place_rows(kt + STAGES, stage);
        request(stage, false);
      }
      const int j0 = kt * KT + wave * 32 - length;
      unsigned word[PT];
      bool masked = false;
#pragma unroll
      for (int n = 0; n < PT; ++n) {
        word[n] = some & (j0 >= 0 ? j0 < 64 ? (unsigned)(seen[n] >> j0) : 0u : j0 <= -32 ? ~0u : (unsigned)(seen[n] << -j0) | Below(-j0));
        if (seen[n] == 0) word[n] = 0;
        masked |= __ballot(word[n] != ~0u) != 0;
      }
#pragma unroll
      for (int n = 0; n < PT; ++n) {
        if (masked) Q::Mask(s[n], word[n], lane);
        rows.Soften(n, s[n], ex);
      }
      if (more) {
        if (STAGES > 1 && behind == 1) {
          WaitForAllBut<N + 1 + (STAGES > 1 ? 1 : 0) * (2 * N + 1)>();
        } else {
          WaitForAllBut<N + 1>();
        }
      } else if (STAGES > 1 && behind == 1) {
        WaitForAllBut<(STAGES > 1 ? 1 : 0) * (2 * N + 1)>();
      } else {
        WaitForAllBut<0>();
      }
      asm volatile("" ::: "memory");
      if (masked && Q::Unbounded(cur + L::BYTES, lane)) {
        rows.AddChosen(s, word, cur + L::BYTES, lane);
      } else {
        rows.Add(s, cur + L::BYTES, lane);
      }
      if (more) {
        __builtin_amdgcn_s_waitcnt(0xC07F);  // the values have been read
        request(stage, true);
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    // the wavefronts' sums of the same pairs: each adds up a share of them
    __syncthreads();
    float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int n = 0; n < PT; ++n) {
      rows.l[n] += __shfl_xor(rows.l[n], 16);
      rows.l[n] += __shfl_xor(rows.l[n], 32);
      rows.Hand(n, meet + (wave * PT + n) * Q::kRegisters * 64, lane);
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
#pragma unroll
    for (int n = 0; n < PT; ++n) {
      const float* from = meet + n * Q::kRegisters * 64 + lane;
      constexpr int EACH = PT * Q::kRegisters * 64;
      float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, from[w * EACH + (Q::kRegisters - 2) * 64]);
      const float base = ex.Base(top);
      float f[WAVES];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        f[w] = ex(from[w * EACH + (Q::kRegisters - 2) * 64], base);
        sum  = __builtin_fmaf(from[w * EACH + (Q::kRegisters - 1) * 64], f[w], sum);
      }
      const int pair = n * 16 + (lane & 15), token = p.group(min(pair, pairs - 1));
      const int my_head = head * p.group.value + min(pair, pairs - 1) - token * p.group.value;
      char* out = const_cast<char*>(HeadOf<T>(p.o, b, my_head)) + token * p.o.row * (int64_t)sizeof(T);
      float* part = p.parts + ((int64_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * PT + n) * Q::kRegisters * 64 + lane;
      for (int t = wave; t < Q::DT; t += WAVES) {
        float four[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          four[r] = 0.0f;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) four[r] = __builtin_fmaf(from[w * EACH + (t * 4 + r) * 64], f[w], four[r]);
        }
        if (whole) {
          const int to = 16 * t + 4 * (lane >> 4);
          T rounded[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) rounded[r] = (T)(seen[n] == 0 ? 0.0f : four[r] / sum);
          if (pair < pairs && to < p.d) __builtin_memcpy(out + to * sizeof(T), rounded, sizeof(rounded));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) part[(t * 4 + r) * 64] = four[r];
        }
      }
      if (!whole && wave == 0) {
        part[(Q::kRegisters - 2) * 64] = top;
        part[(Q::kRegisters - 1) * 64] = seen[n] == 0 ? -1.0f : sum;
      }
    }
    __syncthreads();  // the next unit's tiles may overwrite what was read here
  }
}

// More pairs, 16-bit types: WQ x 32 pairs, KG wavefronts for each 32 that take the steps of 32 keys in turn, tiles of 64 keys in
// a ring of four in LDS that loads fill directly, one barrier per tile; the next scores' MFMAs run beside the exponentials.
// Page numbers come two tiles ahead of the rows; every wavefront places all 64 rows, a lane each, and requests its share.
// 2.4 us a tile of 64 keys x 192 pairs x 128, whose products alone are 0.9 where a vector unit has two of the six wavefronts, and the
// beginning and end of a block's run, 14 us; wavefronts wait in half of their cycles, matrix cores are busy in 18% and vector units
// in 29%.  8 trees of 48 tokens over 2000 to 5000 bf16 rows, 32 heads over 8 x 128, 62 us; tiles through registers took 113.
template <typename T, int D, int WQ, int KG>
__global__ void __launch_bounds__(64 * WQ * KG, 2)
cached_attention_ring_kernel(CachedParams p) {
  typedef Dense<T, D> L;
  typedef Queries<T, D, L> Q;
  constexpr int STEPS = 2, KT = 32 * STEPS, NC = L::NC, STAGE = 2 * STEPS * L::BYTES, STAGES = 4, WAVES = WQ * KG;
  constexpr int LOADS = STEPS * NC, N = (LOADS + WAVES - 1) / WAVES;  // for a tile, and a wavefront's; the last is asked for again
  constexpr int RPL   = L::POW2 ? 64 / NC : 1;                        // rows per load, where that is a whole number
  constexpr int IDS_AT = STAGES * STAGE, HOLDS_AT = IDS_AT + 8 * 256, ROWS_AT = HOLDS_AT + 64, ALL = ROWS_AT + WAVES * KT * 16;
  constexpr int MEET   = (KG - 1) * WQ * 64 * Q::kRegisters * 4;
  static_assert(2 * (N + 1) < 64 && (KG == 1 || KG == STEPS));
  __shared__ __attribute__((aligned(256))) char lds[ALL > MEET ? ALL : MEET];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave / WQ, wq = wave % WQ;
  const int chunks = p.d * (int)sizeof(T) / 16, pairs = p.tokens * p.group.value;
  const Exp<T> ex(p.scale);
  const unsigned lds_at = LdsAddress(lds);
  const bool even_rows  = L::POW2 && chunks == NC && p.page_rows.value % RPL == 0;  // a load has one base
  unsigned lane_off[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int load = min(wave * N + i, LOADS - 1), slot = load % (LOADS / 2) * 64 + lane, row = slot / NC;
    lane_off[i]    = lane / NC * (int)(p.row * sizeof(T)) + L::Back(slot % NC, load >= LOADS / 2 ? L::WideTurn(row) : L::KTurn(row)) * 16;
  }

  Share share(p, KT);
#pragma unroll 1
  while (share.Next(p, KT)) {
    const int b = share.b, unit = share.unit, length = share.length, keys = length + p.tokens;
    const int tiles = share.tiles, tile0 = share.tile0, tile1 = share.tile1;
    const int head = unit % p.kv_heads, pair0 = (unit / p.kv_heads * WQ + wq) * 32;
    const int pair = min(pair0 + (lane & 31), pairs - 1), token = p.group(pair), my_head = head * p.group.value + pair - token * p.group.value;
    const char* k_new = HeadOf<T>(p.k, b, head);
    const char* v_new = HeadOf<T>(p.v, b, head);
    const int* table  = p.table + (int64_t)b * p.columns;

    auto request_pages = [&](int tile) {
      const int key = min(min(tile, tile1 - 1) * KT + lane, max(length - 1, 0));
      CopyToLds4(table + p.page_rows(key), lds_at + IDS_AT + tile % 8 * 256);
    };
    int clean = tile1;  // the first tile with a row of the cache that is none
    struct Two { const char *k, *v; };
    auto request = [&](int tile) {
      const int key  = tile * KT + lane;
      const int page = *reinterpret_cast<const int*>(lds + IDS_AT + tile % 8 * 256 + lane * 4);
      const bool good = key < length && page >= 0 && page < p.pages;
      const int64_t offset = good ? (page * p.page + (key - p.page_rows(key) * p.page_rows.value) * p.row + head * p.head) * (int64_t)sizeof(T) : 0;
      const unsigned long long word = __ballot(good || (key >= length && key < keys));
      // every wavefront finds and writes the same
      *reinterpret_cast<unsigned long long*>(lds + HOLDS_AT + tile % 8 * 8) = word;
      if (__ballot(key < length && !good) != 0) clean = min(clean, tile);
      const unsigned to = lds_at + tile % STAGES * STAGE;
      if (even_rows && __ballot(good) == ~0ull) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int load = min(wave * N + i, LOADS - 1), row = load % (LOADS / 2) * RPL;
          const unsigned low = __builtin_amdgcn_readlane((unsigned)offset, row);
          const unsigned high = __builtin_amdgcn_readlane((unsigned)(offset >> 32), row);
          CopyToLds16((load >= LOADS / 2 ? p.v_pages : p.k_pages) + (int64_t)((uint64_t)high << 32 | low), lane_off[i], to + load * 1024);
        }
      } else {
        // the rows' addresses by way of LDS
        Two row = {reinterpret_cast<const char*>(kZeros), reinterpret_cast<const char*>(kZeros)};
        if (good) row = {p.k_pages + offset, p.v_pages + offset};
        if (key >= length && key < keys)
          row = {k_new + (key - length) * p.k.row * (int64_t)sizeof(T), v_new + (key - length) * p.v.row * (int64_t)sizeof(T)};
        Two* rows = reinterpret_cast<Two*>(lds + ROWS_AT + wave * KT * 16);
        rows[lane] = row;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int load = min(wave * N + i, LOADS - 1), slot = load % (LOADS / 2) * 64 + lane, r = slot / NC;
          const bool values = load >= LOADS / 2;
          const int c = L::Back(slot % NC, values ? L::WideTurn(r) : L::KTurn(r));
          const char* from = values ? rows[r].v : rows[r].k;
          CopyToLds16(c < chunks ? from + c * 16 : reinterpret_cast<const char*>(kZeros), to + load * 1024);
        }
      }
    };
    auto keys_of = [&](int step) { return lds + step / STEPS % STAGES * STAGE + step % STEPS * L::BYTES; };
    auto values_of = [&](int step) { return keys_of(step) + STEPS * L::BYTES; };

    // page numbers, parents and queries in one wait, then the rows
#pragma unroll 1
    for (int i = 0; i < STAGES; ++i) request_pages(tile0 + i);
    Q rows;
    rows.Start(HeadOf<T>(p.q, b, my_head) + token * p.q.row * (int64_t)sizeof(T), chunks, lane >> 5, p.scale);
    const unsigned long long seen = SeenBy(p, b, token);
    WaitForAllBut<0>();
#pragma unroll 1
    for (int i = 0; i < STAGES - 1 && tile0 + i < tile1; ++i) {
      if (i == 2) request_pages(tile0 + STAGES);
      request(tile0 + i);
    }
    if (tile1 - tile0 > 2) {
      WaitForAllBut<2 * N + 1>();
    } else {
      WaitForAllBut<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // before the first step of a tile: it has landed, and everybody is done with the one before the last
    auto turn = [&](int step) {
      if (step % STEPS != 0 || step >= tile1 * STEPS) return;
      const int tile = step / STEPS;
      if (tile + 1 < tile1) {
        WaitForAllBut<N + 1>();
      } else {
        WaitForAllBut<0>();
      }
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (tile + STAGES - 2 < tile1) {
        request_pages(tile + STAGES);
        request(tile + STAGES - 2);
      }
    };
    int step  = tile0 * STEPS + kg;
    f32x16 s  = rows.Scores(keys_of(step), lane);
    float top = Q::Top(s);
    // steps of cached keys only, for pairs that are tokens
    const int plain_steps = pair0 < pairs && __ballot(seen == 0) == 0 ? length / 32 : 0, steps = tile1 * STEPS;
    const int my_steps    = pair0 < pairs ? min(steps, (keys + 31) / 32) : 0;
    auto word_of = [&](int n) {
      const int j0  = n * 32 - length;
      unsigned word = j0 >= 0 ? (unsigned)(seen >> min(j0, 63)) : j0 <= -32 ? ~0u : (unsigned)(seen << -j0) | Below(-j0);
      word &= *reinterpret_cast<const unsigned*>(lds + HOLDS_AT + n / STEPS % 8 * 8 + n % STEPS * 4);
      return seen == 0 ? 0u : word;
    };
    auto open = [&] {  // the step's scores are complete
      if (step >= min(plain_steps, clean * STEPS)) {
        Q::Mask(s, word_of(step), lane);
        top = Q::Top(s);
      }
      rows.Grow(top, ex);
    };
#pragma unroll 1
    for (; step < steps; step += KG) {
      if (step < my_steps) open();
      turn(step - kg + KG);
      if (step >= my_steps) continue;
      if (step >= min(plain_steps, clean * STEPS) && Q::Unbounded(values_of(step), chunks, lane)) break;
      const typename Q::Probabilities mine = rows.Soften(s, ex);
      s = rows.Scores(keys_of(step + KG), lane);
      rows.Add(mine, values_of(step), lane);
      top = Q::Top(s);
    }
    // from the first step on whose values a mask alone does not keep out; it has been opened
#pragma unroll 1
    for (bool opened = true; step < steps; step += KG, opened = false) {
      if (!opened) {
        if (step < my_steps) open();
        turn(step - kg + KG);
      }
      if (step >= my_steps) continue;
      rows.AddChosen(rows.Soften(s, ex), word_of(step), values_of(step), lane);
      s   = rows.Scores(keys_of(step + KG), lane);
      top = Q::Top(s);
    }
    __syncthreads();
    if constexpr (KG > 1) {
      float* meet = reinterpret_cast<float*>(lds);
      if (kg > 0) rows.Hand(meet + ((kg - 1) * WQ + wq) * Q::kRegisters * 64, lane);
      __syncthreads();
      if (kg == 0) {
#pragma unroll
        for (int g = 1; g < KG; ++g) rows.Join(meet + ((g - 1) * WQ + wq) * Q::kRegisters * 64, ex, lane);
      }
      __syncthreads();  // the next unit's tiles may overwrite what was read here
    }
    if (kg == 0) Finish<T, D>(p, rows, b, head, pair0, lane, tile0 == 0, tile1 == tiles, WQ, wq, seen);
  }
}

// Units whose tiles several blocks had: a wavefront takes four registers of the lanes of TILE pairs, four consecutive elements
// of d; SHARED: the eight of a block take the same ones, and a share of the parts each.  RUNS: of TILE pairs in a unit.
template <typename T, int D, int TILE, int RUNS, bool SHARED>
__global__ void __launch_bounds__(SHARED ? 512 : 256)
cached_attention_join_kernel(CachedParams p, int keys_per_tile) {
  constexpr int GROUPS = 64 / TILE, QUADS = D / 4 / GROUPS, REGISTERS = QUADS * 4 + 2;  // lanes of one pair, fours of registers
  constexpr int WAVES = SHARED ? 8 : 1;
  __shared__ float shares[WAVES][6][64];
  const int lane = threadIdx.x & 63, wave = SHARED ? threadIdx.x >> 6 : 0;
  const int mine = SHARED ? blockIdx.x : blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int quad = mine % QUADS, run = mine / QUADS % RUNS, which = mine / QUADS / RUNS;
  if (which >= p.batch * p.units) return;
  const int b = which / p.units, unit = which % p.units, pairs = p.tokens * p.group.value;
  const int pair0 = (unit / p.kv_heads * RUNS + run) * TILE, pair = pair0 + lane % TILE;
  if (pair0 >= pairs || quad * 4 * GROUPS >= p.d) return;
  int64_t total = 0, first = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int64_t mine = 0;
    if (b0 + lane < p.batch) mine = (int64_t)((LengthOf(p, b0 + lane) + p.tokens + keys_per_tile - 1) / keys_per_tile + kEmpty) * p.units;
    int64_t before = b0 + lane < b ? mine : 0;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) mine += __shfl_xor((long long)mine, x), before += __shfl_xor((long long)before, x);
    total += mine, first += before;
  }
  const int tiles = (LengthOf(p, b) + p.tokens + keys_per_tile - 1) / keys_per_tile;
  first += (int64_t)unit * (tiles + kEmpty) + kEmpty;
  const int64_t blocks = min((int64_t)p.blocks, total);
  const int block0 = (int)(((first + 1) * blocks - 1) / total), block1 = (int)(((first + tiles) * blocks - 1) / total);
  if (block0 == block1) return;  // that block has written the result
  const Exp<T> ex(p.scale);
  float top = -__builtin_inff(), sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  bool token_is_none = false;
  constexpr int AT_ONCE = 4;
  for (int i0 = block0 + wave * AT_ONCE; i0 <= block1; i0 += WAVES * AT_ONCE) {
    float m[AT_ONCE], l[AT_ONCE], v[AT_ONCE][4];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = min(i0 + u, block1);
      const float* from = p.parts + ((int64_t)(2 * i + (i == block0 ? 1 : 0)) * RUNS + run) * REGISTERS * 64 + lane;
      m[u] = from[(REGISTERS - 2) * 64], l[u] = from[(REGISTERS - 1) * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[u][e] = from[(quad * 4 + e) * 64];
    }
    float grown = top;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) grown = fmaxf(grown, m[u]);
    const float base = ex.Base(grown), keep = ex(top, base);
    top = grown, sum *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= keep;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (i0 + u > block1) continue;
      token_is_none |= l[u] < 0.0f;
      const float f = ex(m[u], base);
      sum           = __builtin_fmaf(l[u], f, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[u][e], f, o[e]);
    }
  }
  if constexpr (SHARED) {
    shares[wave][0][lane] = top, shares[wave][1][lane] = token_is_none ? -1.0f : sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) shares[wave][2 + e][lane] = o[e];
    __syncthreads();
    if (wave > 0) return;
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, shares[w][0][lane]);
    const float base = ex.Base(top);
    sum = 0.0f, o[0] = o[1] = o[2] = o[3] = 0.0f;
    for (int w = 0; w < WAVES; ++w) {
      const float f = ex(shares[w][0][lane], base);
      token_is_none |= shares[w][1][lane] < 0.0f;
      sum = __builtin_fmaf(shares[w][1][lane], f, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(shares[w][2 + e][lane], f, o[e]);
    }
  }
  if (pair >= pairs) return;
  const int token = p.group(pair), my_head = unit % p.kv_heads * p.group.value + pair - token * p.group.value;
  const int at = (quad * GROUPS + lane / TILE) * 4;
  T four[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) four[e] = (T)(token_is_none ? 0.0f : o[e] / sum);
  char* out = const_cast<char*>(HeadOf<T>(p.o, b, my_head)) + (token * p.o.row + at) * (int64_t)sizeof(T);
  if (at < p.d) __builtin_memcpy(out, four, sizeof(four));
}

// Blocks that divide the list of tiles of `keys_per_tile` keys, or one per unit of `runs` x `tile` pairs.  Dividing costs the
// second kernel, the parts and a beginning more per block, about six tiles, and gains less the more units there are.  us, fp16
// 12 heads x 64, one token, tiles of 256 keys, divided | not, all sequences of that length (of 64 rows to that length): 1 sequence
// of 1400 14.0 | 12.7, 2000 13.6 | 15.3, 6000 14.0 | 34.6; 8 of 1400 17.0 | 13.3 (13.9 | 12.7), 2000 20.6 | 15.8 (14.4 | 15.2), 2800
// 23.1 | 19.7 (14.8 | 19.0), 6000 36.7 | 35.1 (23.3 | 34.7); 16 of 2800 33.1 | 28.2 (17.0 | 18.9), 6000 61.0 | 53.8 (25.4 | 35.4).
// Tiles of 64 keys, bf16, 48 tokens x 32 heads over 8 x 128: 1 of 250 24.8 | 26.7, 600 27.8 | 41.1, 8 of 250 30.1 | 27.4, 600
// 32.9 | 42.0.  One block per CU: their wavefronts and buffers leave room for no other.
// The lengths are the GPU's, so the table's width stands for them, and short caches in wide tables pay for being divided: 8 of 511
// rows 7.2 in tables for up to 2048 rows, 13.0 for 8192 and 131072; 1 of 511 7.0 and 11.5; 8 of 2000 15.5 and 20.2.
template <int D>
int Divide(CachedParams& p, int tile, int runs, int keys_per_tile, hipStream_t stream) {
  constexpr int kMostBlocks = 256;
  const int pairs  = p.tokens * p.group.value;
  p.units          = p.kv_heads * ((pairs + tile * runs - 1) / (tile * runs));
  const int units  = p.batch * p.units;
  const int64_t most_tiles = ((int64_t)p.columns * p.page_rows.value + p.tokens + keys_per_tile - 1) / keys_per_tile;
  p.blocks = 0;
  if (most_tiles > 6 + std::min(units, 192) / 32) {
    const int blocks   = (int)std::min<int64_t>(kMostBlocks, units * most_tiles);
    const size_t bytes = (size_t)2 * blocks * runs * (D * tile / 64 + 2) * 64 * sizeof(float);
    if (bytes <= cinn_hip_kernels::ScratchLimit(cinn_hip_kernels::ScratchKind::kSplitK, stream)) {
      p.blocks = blocks;
      p.parts  = static_cast<float*>(cinn_hip_kernels::Scratch(cinn_hip_kernels::ScratchKind::kSplitK, bytes, stream));
    }
  }
  return p.blocks > 0 ? p.blocks : units;
}

template <typename T, int D, int TILE, int RUNS>
void LaunchJoin(const CachedParams& p, int keys_per_tile, hipStream_t stream) {
  if (p.blocks == 0) return;
  const int units = p.batch * p.units, wavefronts = units * RUNS * (D * TILE / 256);
  // parts of a unit, four a wavefront at a time.  The whole call, us, by eight wavefronts | one: one sequence of 100003 fp32 rows 74 |
  // 85, 30000 33 | 46, one tree of 16 tokens 21.0 | 26.9, of 48 28.9 | 32.0; with eight from two parts on 8 trees of 48 64 | 78
  if (p.blocks / units >= 8) {
    hipLaunchKernelGGL((cached_attention_join_kernel<T, D, TILE, RUNS, true>), dim3((unsigned)wavefronts), dim3(512), 0, stream, p, keys_per_tile);
  } else {
    hipLaunchKernelGGL((cached_attention_join_kernel<T, D, TILE, RUNS, false>), dim3((unsigned)((wavefronts + 3) / 4)), dim3(256), 0, stream, p,
                       keys_per_tile);
  }
}

template <typename T, int D, int PT>
void LaunchFew(CachedParams p, hipStream_t stream) {
  // The buffers of eight wavefronts in 128 KiB of LDS; of four, which have twice the registers, where a tile, or the queries and
  // sums of 32 pairs, need more than 256: 32 pairs a unit, 8 sequences of 2000 to 5000 bf16 rows, 8 key heads: d 128 40 us
  // (eight: 57), d 96 37.4 us (39.3).
  constexpr int kTile = 2 * Dense<T, D>::BYTES, kWaves = kTile * PT > 16384 ? 4 : 8, kDeep = 128 * 1024 / kWaves / kTile;
  constexpr int kStages = kDeep > 2 ? 2 : kDeep;
  const int blocks = Divide<D>(p, 16, PT, 32 * kWaves, stream);
  hipLaunchKernelGGL((cached_attention_few_kernel<T, D, PT, kWaves, kStages>), dim3((unsigned)blocks), dim3(64 * kWaves), 0, stream, p);
  LaunchJoin<T, D, 16, PT>(p, 32 * kWaves, stream);
}

template <typename T, int D, int WQ, int KG>
void LaunchRing(CachedParams p, hipStream_t stream) {
  const int blocks = Divide<D>(p, 32, WQ, 64, stream);
  hipLaunchKernelGGL((cached_attention_ring_kernel<T, D, WQ, KG>), dim3((unsigned)blocks), dim3(64 * WQ * KG), 0, stream, p);
  LaunchJoin<T, D, 32, WQ>(p, 64, stream);
}

template <typename T, int D>
void LaunchTiles(CachedParams p, hipStream_t stream) {
  // The fewest wavefronts that hold the pairs.  us, bf16 8 sequences of 2000 to 5000 rows, 8 key heads x 128: 32 pairs few 39.7,
  // ring of 2 x 2 48.5.  The choices among rings are worth 1% or nothing, the smaller | the larger in turn: 2 x 2 | 4 x 2 with 36, 48,
  // 64 pairs 45.0 | 45.0, 44.5 | 44.4, 44.7 | 44.6; 6 x 1 | 8 x 1 with 144, 160, 192 pairs 60.1 | 60.4, 60.2 | 60.6, 61.9 | 62.3.
  const int pairs = p.tokens * p.group.value;
  if (pairs <= 16) {
    LaunchFew<T, D, 1>(p, stream);
  } else if (pairs <= 32) {
    LaunchFew<T, D, 2>(p, stream);
  } else if constexpr (sizeof(T) == 4) {
    const int blocks = Divide<D>(p, 32, 4, 64, stream);
    hipLaunchKernelGGL((cached_attention_float_kernel<D>), dim3((unsigned)blocks), dim3(512), 0, stream, p);
    LaunchJoin<T, D, 32, 4>(p, 64, stream);
  } else if (pairs <= 64) {
    LaunchRing<T, D, 2, 2>(p, stream);
  } else if (pairs <= 128) {
    LaunchRing<T, D, 4, 2>(p, stream);
  } else if ((pairs + 191) / 192 * 6 < (pairs + 255) / 256 * 8) {
    LaunchRing<T, D, 6, 1>(p, stream);
  } else {
    LaunchRing<T, D, 8, 1>(p, stream);
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
  const int64_t row = (int64_t)d * std::max(std::max(q_heads, k_heads), v_heads);
  CINN_RT_CHECK(row * (f32 ? 4 : 2) <= 1 << 25, "cached_attention: rows of more than 32 MiB");  // a load's offsets have 32 bits
  CINN_RT_CHECK((int64_t)batch * heads * tokens < 1 << 22, "cached_attention: too many rows");  // blocks of up to 512 threads
  CINN_RT_CHECK((int64_t)batch * tokens * row < INT_MAX && (int64_t)batch * columns < INT_MAX && (int64_t)pages * page_rows * kv_heads * d < (int64_t)1 << 40,
                "cached_attention: tensor too large");
  auto input = [&](int slot) {
    const int at = ((unsigned)operands >> (4 * slot)) & 15;
    CINN_RT_CHECK(at < num_args - 1, "cached_attention: operand %d is argument %d of %d", slot, at, num_args);
    return BufferArg(v_args, at);
  };
  auto typed = [&](int slot) {
    const cinn_buffer_t* b = input(slot);
    CINN_RT_CHECK(b->type.code == out->type.code && b->type.bits == out->type.bits, "cached_attention: operands of different types");
    CINN_RT_CHECK(reinterpret_cast<uintptr_t>(b->memory) % 16 == 0, "cached_attention: operand %d is not aligned to 16 bytes", slot);
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
