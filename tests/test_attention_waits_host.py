"""The chunk kernel's planning thread on the host, which is its clock: it gives up when no tile was finished for the limit, however long
the hardware suspends a look at a barrier, and never while tiles are.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, ROLE_SHIM, build, piece, role, source

BEFORE = r"""
using namespace syfi;
struct AttentionArgs { KvBatch batch; int group, window; };
"""

HARNESS = r"""
static const int kTokens = 3000;               // 12 row tiles: more segments than the ring has places
static int32_t lens[] = {kTokens}, starts[] = {0, kTokens};
static AttentionArgs a = {{nullptr, lens, starts, 1, 64, kTokens}, 1, 0};
static const ChunkPlan plan = {a.batch, 1, 1, 0};
static PlanShared s_plan;
static ChunkShared sh;
static long long limit, total, every;
static int freed, described;
static void mbar_arrive(uint64_t*) { ++described; }
static bool world() {                          // a tile every so many clocks, five to a segment; none from `freed` segments on, or all done
  static long long next = every;
  if (every > 0 && clocks >= next && !sh.done) {
    next = clocks + every;
    ++sh.tiles_done;
    if (sh.tiles_done % 5 == 0) ++sh.segment_empty[freed++ % kSegmentRing];
    if (sh.tiles_done == 5 * 20) sh.done = 1;
  }
  return true;
}
int main(int, char** argv) {
  limit = atoll(argv[1]);
  look_clocks = atoll(argv[2]);
  every = atoll(argv[3]);
  total = plan.row_tiles(kv_sequence(a.batch, 0)) * kChunkExtra;
  for (int rt = 0; rt < plan.row_tiles(kv_sequence(a.batch, 0)); ++rt) total += plan.span(kv_sequence(a.batch, 0), rt).tiles;
  run_block(32, [] { if (threadIdx.x == 0) plan_role(a, plan, s_plan, sh, static_cast<int>(total), total, total, 1, limit); }, 0, world);
  printf("code %d after %lld clocks, %u tiles, %d segments\n", static_cast<int>(sh.abort_code), clocks, static_cast<unsigned>(sh.tiles_done), described);
  if (every > 0) return sh.abort_code != 0 || !sh.done || described != 13;
  return sh.abort_code != kStatusChunkTimeout || clocks < limit || clocks > limit + 3 * look_clocks + 1000;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    chunk, internal = source("paged_attention_chunk.cu"), source("kv_internal.h")
    plan = source("attention_plan.cuh").replace("#pragma once", "").replace('#include "kv_internal.h"', "")
    of_a_call = piece(internal, "struct KvBatch {", "kv_sequence(const KvBatch& a, int b) {") + piece(internal.split("kv_sequence(const KvBatch& a, int b) {")[1], "\n", "\n}\n")
    pieces = [piece(chunk, "using ChunkPlan", ";\n"), piece(chunk, "using ChunkCursor", ";\n"), piece(source("attention_common.cuh"), "struct Parts {", "\n};\n"),
              piece(chunk, "struct Watch {", "\n};\n"), piece(chunk, "__device__ __forceinline__ void plan_role(", "\n}\n")]
    return build(tmp_path_factory.mktemp("waits"), EMULATOR + ROLE_SHIM + of_a_call + plan + BEFORE + role() + "\n" + "\n".join(pieces) + HARNESS)


@pytest.mark.parametrize("limit", [1, 1000, 1 << 20, 1 << 32])
@pytest.mark.parametrize("look", [20, 1000, 100003])
def test_it_gives_up_when_the_time_is_over(limit, look, program):
    if limit // look > 1 << 23:
        pytest.skip("too many looks for a test")
    done = subprocess.run([program, str(limit), str(look), "0"], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("look", [20, 1000])
def test_it_waits_for_tiles_however_long_they_take_together(look, program):
    done = subprocess.run([program, "100000", str(look), "90000"], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout
