"""The plan of the attention calls (csrc/attention_plan.cuh) on the host as the kernels over the 4-bit cache use it, and for batches in which many
sequences have many row tiles.  See test_attention_plan_host.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, build, piece, source
from test_attention_plan_host import HARNESS

MAIN = r"""
int main(int, char** argv) {
  const int n = atoi(argv[1]), kind = atoi(argv[2]);
  heads = kind == 4 ? 1 : 2;
  group = kind == 4 ? 64 : 4;
  window_size = kind == 2 ? 100 : 0;
  grid = 5;
  unsigned seed = 1;
  auto random = [&](int m) { seed = seed * 1664525u + 1013904223u; return static_cast<int>((seed >> 8) % m); };
  starts.push_back(0);
  for (int b = 0; b < n; ++b) {                // decoding; chunks, also with a window; prompts; a chunk here and there
    const int count = kind == 0 ? 1 : kind == 3 ? 330 + random(40) : kind == 4 ? (b % 5 == 2 ? 100 : 1) : random(5) == 0 ? 0 : 1 + random(90);
    lens.push_back(count + (kind == 3 ? 0 : random(b % 9 == 0 ? 2000 : 200)));
    starts.push_back(starts.back() + count);
  }
  batch = {nullptr, lens.data(), starts.data(), n, 40, starts.back()};
  check<64, 8, 6, 0>(128);
  check<64, 16, 6, 0>(128);
  // Sequences of many row tiles are the work of all warps: of n in one round none has many more than its share.  (A call looks at a round once or
  // twice, and there are several rounds of 128.)
  summed.assign(32, 0);
  check<128, 256, 5, 0>(512);
  int most = 0, all = 0;
  for (int s : summed) {
    most = max(most, s);
    all += s;
  }
  printf("%d sequences summed by warps, %d by one\n", all, most);
  if (kind == 3 && most * 16 > all + 16 * grid * 2 * ((n + 127) / 128)) ++bad;
  return bad != 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    plan = source("attention_plan.cuh").replace("#pragma once", "").replace('#include "kv_internal.h"', "")
    start = "long long tiles_of_warp(const KvSequence& s, int lane) const {"
    assert start in plan
    plan = plan.replace(start, start + " if (lane == 0) ++summed[threadIdx.x / 32];")
    plan = plan.replace("namespace syfi {", "namespace syfi {\nstatic std::vector<int> summed(32);", 1)
    of_a_call = piece(source("kv_internal.h"), "struct KvBatch {", "kv_sequence(const KvBatch& a, int b) {") + piece(
        source("kv_internal.h").split("kv_sequence(const KvBatch& a, int b) {")[1], "\n", "\n}\n")
    return build(tmp_path_factory.mktemp("plan4"), EMULATOR + "namespace syfi {\nconstexpr int kKvPage = 64;\n" + of_a_call + "}\n" + plan + HARNESS.split("int main(")[0] + MAIN)


def test_the_kernels_use_these_plans():
    """Tiles, rows and extra places as the sources have them."""
    few, many = source("kv4_attention.cu"), source("kv4_attention_chunk.cu")
    assert "constexpr int kDecodeExtra = 6;" in few and "Plan<kKvPage, kRows, kDecodeExtra>" in few and "kRows = 8 * NT" in few
    assert "constexpr int kChunkExtra = 5;" in many and "using ChunkPlan = Plan<kTile, kChunkRows, kChunkExtra>;" in many
    assert "constexpr int kTile = 128;" in many and "constexpr int kChunkRows = 256;" in many and "constexpr int kChunkThreads = 512;" in many


@pytest.mark.parametrize("sequences", [1, 33, 127, 128, 129, 257])
@pytest.mark.parametrize("kind", range(5), ids=["decoding", "chunks", "window", "prompts", "one key head"])
def test_every_tile_is_done_once_and_all_warps_share_long_sequences(sequences, kind, program):
    done = subprocess.run([program, str(sequences), str(kind)], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout
