"""How the attention kernels share out a call's work, run on the host: csrc/attention_plan.cuh compiled as C++ with the threads of a
block as contexts that a scheduler switches at shuffles and barriers.  One warp is always the last to run, so a value that another
warp overwrites without a barrier in between is overwritten before that warp reads it.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, build, piece, source

HARNESS = r"""
using namespace syfi;
static std::vector<int32_t> lens, starts;
static KvBatch batch;
static int heads, group, window_size, grid;
static unsigned cta;
static PlanShared shared;
static std::vector<long long> totals;
static std::vector<std::tuple<int, int, int, int>> found;
static std::map<std::tuple<int, int, int, int>, int> covered;   // (sequence, row tile, head, tile) -> times
static int bad;

template <int TILE, int ROWS, int EXTRA, int NARROW>
static void kernel() {
  const Plan<TILE, ROWS, EXTRA, NARROW> plan = {batch, heads, group, window_size};
  const long long total = plan.total(shared);
  totals[threadIdx.x] = total;
  const int ctas = static_cast<int>(min(static_cast<long long>(grid), total));
  if (static_cast<int>(cta) >= ctas) return;
  const long long w0 = piece_start(total, ctas, cta), w1 = piece_start(total, ctas, cta + 1);
  plan.locate(shared, w0);
  found[threadIdx.x] = std::make_tuple(shared.start_b, shared.start_rt, shared.start_head, shared.start_place);
  if (threadIdx.x != 0) return;
  Cursor<TILE, ROWS, EXTRA, NARROW> at;
  at.start(plan, shared, static_cast<int>(w1 - w0));
  while (at.left > 0) {
    const int n = at.tiles_here();
    for (int i = 0; i < n; ++i) ++covered[std::make_tuple(at.b, at.rt, at.head, at.tile + i)];
    at.advance(plan, n);
  }
}

template <int TILE, int ROWS, int EXTRA, int NARROW>
static void check(unsigned block) {
  covered.clear();
  long long want = 0;
  std::map<std::tuple<int, int, int, int>, int> all;
  const Plan<TILE, ROWS, EXTRA, NARROW> plan = {batch, heads, group, window_size};
  for (int b = 0; b < batch.batch; ++b) {
    const KvSequence s = kv_sequence(batch, b);
    for (int rt = 0; s.count > 0 && rt < plan.row_tiles(s); ++rt)
      for (int h = 0; h < heads; ++h) {
        const int tiles = plan.span(s, rt).tiles;
        want += EXTRA + tiles;
        for (int t = 0; t < tiles; ++t) all[std::make_tuple(b, rt, h, t)] = 1;
      }
  }
  for (cta = 0; cta < static_cast<unsigned>(grid); ++cta) {
    totals.assign(block, -1);
    found.assign(block, std::make_tuple(-1, -1, -1, -1));
    shared = PlanShared{};
    run_block(block, kernel<TILE, ROWS, EXTRA, NARROW>, (cta + 1) % (block / 32));
    for (unsigned i = 0; i < block; ++i)
      if (totals[i] != want || found[i] != found[0]) {
        if (++bad < 5) printf("tiles of %d: CTA %u, thread %u: a line of %lld places where it has %lld\n", TILE, cta, i, totals[i], want);
      }
  }
  if (covered != all) {
    ++bad;
    printf("tiles of %d: %zu tiles covered, %zu to do\n", TILE, covered.size(), all.size());
  }
}

int main(int argc, char** argv) {
  const int n = atoi(argv[1]), kind = atoi(argv[2]);
  heads = 2;
  group = 4;
  window_size = kind == 2 ? 100 : 0;
  grid = 7;
  unsigned seed = 1;
  auto random = [&](int m) { seed = seed * 1664525u + 1013904223u; return static_cast<int>((seed >> 8) % m); };
  starts.push_back(0);
  for (int b = 0; b < n; ++b) {
    const int count = kind == 0 ? 1 : random(5) == 0 ? 0 : b == n / 2 ? 300 : 1 + random(3);   // some sequences have no new token, one has many
    lens.push_back(count + random(b % 9 == 0 ? 2000 : 200));
    starts.push_back(starts.back() + count);
  }
  batch = {nullptr, lens.data(), starts.data(), n, 40, starts.back()};
  check<64, 8, 1, 0>(128);
  check<64, 16, 1, 0>(128);
  check<128, 256, 4, 128>(768);
  return bad != 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    plan = source("attention_plan.cuh").replace("#pragma once", "").replace('#include "kv_internal.h"', "")
    of_a_call = piece(source("kv_internal.h"), "struct KvBatch {", "kv_sequence(const KvBatch& a, int b) {") + piece(
        source("kv_internal.h").split("kv_sequence(const KvBatch& a, int b) {")[1], "\n", "\n}\n")
    return build(tmp_path_factory.mktemp("plan"), EMULATOR + "namespace syfi {\nconstexpr int kKvPage = 64;\n" + of_a_call + "}\n" + plan + HARNESS)


@pytest.mark.parametrize("sequences", [1, 40, 127, 128, 129, 256, 257, 300])
@pytest.mark.parametrize("kind", [0, 1, 2], ids=["decoding", "mixed", "window"])
def test_every_thread_sees_the_same_line_and_every_tile_is_done_once(sequences, kind, program):
    done = subprocess.run([program, str(sequences), str(kind)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout
