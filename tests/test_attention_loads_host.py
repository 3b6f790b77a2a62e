"""The chunk kernel's loading thread on the host when another role gives up: roles that failed still arrive at barriers, which frees
stages whose copies may be on their way.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, ROLE_SHIM, build, piece, role, source

BEFORE = r"""
struct CUtensorMap {};
template <typename T> static T __ldg(const T* p) { return *p; }
static uint64_t l2_policy_evict_normal() { return 0; }
static int asked;                            // copies
static void mbar_arrive_expect_tx(uint64_t*, uint32_t) {}
static void bulk_load(void*, const void*, uint32_t, uint64_t*, uint64_t) { ++asked; }
static void tma_load_4d(void*, const CUtensorMap*, uint64_t*, int, int, int, int, uint64_t) { ++asked; }
struct AttentionArgs { KvCache cache; KvBatch batch; };
"""

HARNESS = r"""
template <int D>
struct World {
  static inline ChunkShared sh;
  static inline uint8_t smem[ChunkShape<D>::kSmem];
  static inline int32_t table[64];
  static inline AttentionArgs a;
  static inline int described, freed, asked_then = -1, fail_after;
  static bool step() {                       // frees stages in turn; at some point a role gives up, and stages are freed all the same
    if (!described) {
      Segment& g = sh.segment[0];
      g.tiles = 30;
      g.any_high = 30 * kTile - 1;
      ++sh.segment_full[0];
      ++sh.segment_full[1];                  // (its tiles are 0: the piece's end)
      described = 1;
      return true;
    }
    if (freed == fail_after) {
      sh.abort_code = kStatusChunkTimeout;
      asked_then = asked;
    }
    const int i = freed++;
    ++sh.scale_empty[i % kScaleStages];
    ++sh.k_empty[i % ChunkShape<D>::kKStages];
    ++sh.v_empty[i % ChunkShape<D>::kVStages];
    return i < 100;
  }
  static int run(int n) {
    fail_after = n;
    a.cache = {smem, 1 << 16, 64, 2, 1};
    a.batch = {table, nullptr, nullptr, 1, 64, 1};
    run_block(32, [] { if (threadIdx.x == 0) load_role<D>(CUtensorMap(), a, sh, smem); }, 0, step);
    printf("%d copies, %d of them before the failure\n", asked, asked_then);
    return asked_then < 0 ? asked != 30 * 8 : asked != asked_then;
  }
};
static void mbar_arrive(uint64_t*) {}
int main(int, char** argv) { return atoi(argv[1]) == 64 ? World<64>::run(atoi(argv[2])) : World<128>::run(atoi(argv[2])); }
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    cache = piece(source("kv_internal.h"), "// A cache in device memory.", "  int batch, max_pages, tokens;\n};\n")
    return build(tmp_path_factory.mktemp("loads"), EMULATOR + ROLE_SHIM + cache + BEFORE + role("load_role") + HARNESS)


@pytest.mark.parametrize("fail_after", [0, 1, 2, 3, 7, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_no_copy_is_asked_for_behind_a_failure(dim, fail_after, program):
    done = subprocess.run([program, str(dim), str(fail_after)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout
