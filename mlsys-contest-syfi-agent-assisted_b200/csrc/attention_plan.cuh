// How the attention kernels share out a call's work: every CTA works it out for itself from the sequences' lengths, which the host
// does not know.
//
// A unit is (sequence, row tile, key head): up to ROWS of the sequence's count * group rows (token major, the query heads of the
// key head side by side), over the tiles of TILE positions that any of them sees.  All units' tiles, in the order sequence, row
// tile, head, tile, are one line that is cut into equal pieces, one per CTA; so a piece has at most a unit's end, some whole
// units and a unit's beginning, whatever the lengths are.  In front of a unit's tiles the line has EXTRA places that stand for
// what a unit costs besides its tiles.  Units of at most NARROW rows go through two tiles in the time of one: to the line their tiles
// are twice as long.  A unit that lies in one piece is finished there.  Else each of its CTAs leaves a partial
// result, and the one that comes last (a counter per unit) adds them up, in the order of the pieces.
#pragma once
#include "kv_internal.h"

namespace syfi {

constexpr int kPlanRound = 128;     // sequences whose tiles are summed at a time
constexpr int kFewRowTiles = 4;     // of a sequence that one thread sums up

struct PlanShared {
  long long sum[kPlanRound];        // places of each sequence of the round, then their inclusive prefix sums
  int many[kPlanRound / 32];        // of every 32 of them, whether one has more than kFewRowTiles row tiles
  int start_b, start_rt, start_head, start_place;   // place: EXTRA + tile
  int last;                         // the ticket says that this CTA is the unit's last
};

struct Span {
  int first, tiles;                 // tiles of positions; at least one
};

template <int TILE, int ROWS, int EXTRA, int NARROW = 0>
struct Plan {
  const KvBatch& batch;
  int heads, group, window;

  __device__ int row_tiles(const KvSequence& s) const { return (s.count * group + ROWS - 1) / ROWS; }
  // positions [low, high] that the row tile's rows see
  __device__ Span span(const KvSequence& s, int rt) const {
    const int row0 = rt * ROWS, row1 = min(s.count * group, row0 + ROWS) - 1;
    const int base = s.length - s.count, high = base + row1 / group;
    const int low = window > 0 ? max(base + row0 / group - window + 1, 0) : 0;
    const int tile = row1 - row0 < NARROW ? 2 * TILE : TILE;
    return high < low ? Span{0, 1} : Span{low / tile, high / tile - low / tile + 1};
  }
  __device__ long long tiles_of_warp(const KvSequence& s, int lane) const {     // a head's places of all row tiles; whole warp
    const int n = s.count > 0 ? row_tiles(s) : 0;
    long long sum = 0;
    for (int rt = lane; rt < n; rt += 32) sum += EXTRA + span(s, rt).tiles;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
  }

  // Sums a round of sequences into sh.sum (inclusive); whole block, ends with a barrier.  A thread has a sequence, as long as that has few row
  // tiles; those of more are each summed by a warp together, all warps in turn.  (A warp for every sequence took 3 to 5 us of a short call.  Those
  // of many row tiles left to the warp whose threads have them: 32 prompts of 300 tokens 158 us instead of 147, 300 of them 658 instead of 605.)
  __device__ void sum_round(PlanShared& sh, int round) const {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    for (int first = warp * 32; first < kPlanRound; first += warps * 32) {
      const int b = round * kPlanRound + first + lane;
      KvSequence s = {0, 0, 0};
      if (b < batch.batch) s = kv_sequence(batch, b);
      const int n = s.count > 0 ? row_tiles(s) : 0;
      long long sum = 0;
      for (int rt = 0; rt < n && n <= kFewRowTiles; ++rt) sum += EXTRA + span(s, rt).tiles;
      sh.sum[first + lane] = n > kFewRowTiles ? -1 : sum;
      const int many = __any_sync(0xffffffffu, n > kFewRowTiles);
      if (lane == 0) sh.many[first / 32] = many;
    }
    __syncthreads();
    int many = 0;
#pragma unroll
    for (int i = 0; i < kPlanRound / 32; ++i) many |= sh.many[i];
    if (many) {
      for (int i = warp; i < kPlanRound; i += warps) {
        if (sh.sum[i] >= 0) continue;
        const long long all = tiles_of_warp(kv_sequence(batch, round * kPlanRound + i), lane);
        if (lane == 0) sh.sum[i] = all;
      }
      __syncthreads();
    }
    if (warp == 0) {
      long long mine[kPlanRound / 32], sum = 0;
#pragma unroll
      for (int j = 0; j < kPlanRound / 32; ++j) mine[j] = sum += sh.sum[lane * (kPlanRound / 32) + j];
      long long incl = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
#pragma unroll
      for (int j = 0; j < kPlanRound / 32; ++j) sh.sum[lane * (kPlanRound / 32) + j] = mine[j] + incl - sum;
    }
    __syncthreads();
  }

  // The line's length; whole block.
  __device__ long long total(PlanShared& sh) const {
    long long sum = 0;
    for (int round = 0; round * kPlanRound < batch.batch; ++round) {
      if (round > 0) __syncthreads();
      sum_round(sh, round);
      sum += sh.sum[kPlanRound - 1];
    }
    return sum * heads;
  }

  // Where place `at` of the line lies, into sh.start_*; whole block, ends with a barrier.  Behind total(), whose last round is
  // still in sh.sum.
  __device__ void locate(PlanShared& sh, long long at) const {
    const int rounds = (batch.batch + kPlanRound - 1) / kPlanRound, lane = threadIdx.x % 32;
    long long before = 0;            // tiles of the rounds in front
    int round = 0;
    if (rounds > 1) __syncthreads(); // every thread has read total()'s last sum
    while (true) {
      if (rounds > 1) sum_round(sh, round);
      const long long in_round = sh.sum[kPlanRound - 1] * heads;
      if (at < before + in_round || round + 1 == rounds) break;
      before += in_round;
      ++round;
      __syncthreads();
    }
    if (threadIdx.x < 32) {
      const long long offset = at - before;
      int b = 0;                     // the sequence: as many of the round's as end at or before the offset
      for (int i = lane; i < kPlanRound; i += 32) b += sh.sum[i] * heads <= offset;
      b = min(__reduce_add_sync(0xffffffffu, b), kPlanRound - 1);
      long long left = offset - (b > 0 ? sh.sum[b - 1] * heads : 0);
      const KvSequence s = kv_sequence(batch, min(round * kPlanRound + b, batch.batch - 1));
      const int n = row_tiles(s);
      for (int base = 0; base < n; base += 32) {
        const int mine = base + lane < n ? EXTRA + span(s, base + lane).tiles : 0;
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += up;
        }
        const long long all = static_cast<long long>(__shfl_sync(0xffffffffu, incl, 31)) * heads;
        if (left < all) {
          const long long from = static_cast<long long>(incl - mine) * heads;
          if (left >= from && left < from + static_cast<long long>(mine) * heads) {
            const int o = static_cast<int>(left - from);
            sh.start_b = round * kPlanRound + b;
            sh.start_rt = base + lane;
            sh.start_head = o / mine;
            sh.start_place = o % mine;
          }
          break;
        }
        left -= all;
      }
    }
    __syncthreads();
  }
};

// A walk over the tiles of a piece of the line.  The same in every thread of a block.
template <int TILE, int ROWS, int EXTRA, int NARROW = 0>
struct Cursor {
  int b, rt, head, tile;             // tile of the unit, counted from 0
  int left;                          // places of the piece from this tile on; none: the walk is over
  KvSequence s;
  Span span;
  int row_tiles;

  __device__ void start(const Plan<TILE, ROWS, EXTRA, NARROW>& plan, const PlanShared& sh, int places) {
    b = sh.start_b;
    rt = sh.start_rt;
    head = sh.start_head;
    s = kv_sequence(plan.batch, b);
    row_tiles = plan.row_tiles(s);
    span = plan.span(s, rt);
    const int skipped = max(EXTRA - sh.start_place, 0);
    tile = sh.start_place + skipped - EXTRA;
    left = places - skipped;
  }
  // To the next unit, if the piece has any of its tiles.
  __device__ void next_unit(const Plan<TILE, ROWS, EXTRA, NARROW>& plan) {
    left -= EXTRA;
    if (left <= 0) return;
    tile = 0;
    if (++head < plan.heads) return;
    head = 0;
    if (++rt >= row_tiles) {
      rt = 0;
      do {
        if (++b >= plan.batch.batch) {
          left = 0;
          return;
        }
        s = kv_sequence(plan.batch, b);
      } while (s.count == 0);
      row_tiles = plan.row_tiles(s);
    }
    span = plan.span(s, rt);
  }
  // `n` tiles of the unit on; behind its last to the next unit.
  __device__ void advance(const Plan<TILE, ROWS, EXTRA, NARROW>& plan, int n) {
    tile += n;
    left -= n;
    if (tile == span.tiles && left > 0) next_unit(plan);
  }
  __device__ int tiles_here() const { return min(span.tiles - tile, left); }      // of the unit, in this piece
  __device__ int rows(int group) const { return min(s.count * group - rt * ROWS, ROWS); }
};

// The pieces of a line of `total` places cut among `ctas` CTAs.
__device__ __forceinline__ long long piece_start(long long total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int piece_of(long long total, int ctas, long long at) {
  int c = static_cast<int>(at * ctas / total);       // piece_start(c) <= at, and at most one too low
  while (c + 1 < ctas && piece_start(total, ctas, c + 1) <= at) ++c;
  return c;
}

}  // namespace syfi
