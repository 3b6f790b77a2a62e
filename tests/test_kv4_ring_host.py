"""The decoding kernel's ring of pages over the 4-bit cache on the host: which warp asks for which page into which stage, walks that change
warps, and waits that run out (csrc/kv4_attention.cu).  The kernel's own text, with copies that land in any order and one warp always the
last to run; every warp must find its pages, untouched until it is done with them.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, ROLE_SHIM, build, piece, source

BEFORE = r"""
#include <set>
#include <type_traits>
template <typename T> static T __ldg(const T* p) { return *p; }
static int __all_sync(unsigned, int p) { int all = 1; for (long long x : exchange(p)) all &= x != 0; return all; }
static uint64_t l2_policy_evict_first() { return 0; }
static long long looked() { clocks += 20; stop(AT_LOOK); return clocks; }
#define clock64 looked
struct AttentionArgs { KvCache cache; KvBatch batch; int group, window; };
// A barrier of the block beside warps that look at barriers in memory.
static unsigned arrived, meetings;
static void meet() {
  const unsigned before = meetings;
  if (++arrived == blockDim.x) {
    arrived = 0;
    ++meetings;
  }
  while (meetings == before) stop(AT_LOOK);
}
#define __syncthreads meet

// Copies on their way; `world` lands one of them, whichever, unless it is stalled.
struct Copy { uint8_t* to; const uint8_t* from; uint64_t* bar; };
static std::vector<Copy> pending;
static std::map<uint64_t*, int> open_bytes;
static int landings, stall_after;            // no copy lands between `stall_after` and the wait for what is on its way
static bool draining;
static unsigned seed = 1;
static int bad, consumed;
static void wrong(const char* what) { if (++bad < 6) printf("%s\n", what); }
static int rnd(int m) { seed = seed * 1664525u + 1013904223u; return static_cast<int>((seed >> 8) % m); }
static void mbar_arrive(uint64_t* bar) { ++*bar; }
static void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  if (open_bytes[bar] != 0) wrong("a stage is asked for while its last copies are on their way");
  open_bytes[bar] = bytes;
}
static int copy_bytes;
static void bulk_load(void* to, const void* from, uint32_t bytes, uint64_t* bar, uint64_t) {
  copy_bytes = bytes;
  pending.push_back({static_cast<uint8_t*>(to), static_cast<const uint8_t*>(from), bar});
}
static bool world() {
  static int idle, seen;
  idle = consumed == seen && pending.empty() ? idle + 1 : 0;
  seen = consumed;
  if (idle > 100000) return false;             // everybody waits
  if (pending.empty() || (stall_after >= 0 && landings >= stall_after && !draining)) return true;
  const int i = rnd(static_cast<int>(pending.size()));
  const Copy c = pending[i];
  pending.erase(pending.begin() + i);
  memcpy(c.to, &c.from, sizeof(c.from));       // the page's content: where it came from
  ++landings;
  if ((open_bytes[c.bar] -= copy_bytes) == 0) ++*c.bar;
  return true;
}
static void mbar_wait_landed(uint64_t* bar, uint32_t parity) {
  draining = true;
  while ((*bar & 1) == parity) stop(AT_LOOK);
}
static void atomicExch(int* to, int v) { *to = v; }
"""

HARNESS = r"""
static AttentionArgs a;
static int grid, cta, status;
static long long wait_limit;
static std::map<std::tuple<int, int, int, int>, int> covered;
static std::set<std::tuple<int, int, int, int>> spoilt;      // pages of a segment whose sums are NaN

template <int D, int NT>
struct Run {
  using Shape = Decode4Shape<D, NT>;
  using Walk = Cursor<kKvPage, Shape::kRows, kDecodeExtra>;
  using Block = Kv4Block<D>;
  static constexpr int kRows = Shape::kRows, kStages = Shape::kStages;
  static inline DecodeShared<D, NT> sh;
  alignas(16) static inline uint8_t smem[Shape::kSmem];
  static inline bool nan_of[kWarps];
  static void kernel() {
    float* const s_merge = reinterpret_cast<float*>(smem + kStages * Shape::kStageBytes);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const Plan<kKvPage, kRows, kDecodeExtra> plan = {a.batch, a.cache.heads, a.group, a.window};
    const long long total = plan.total(sh.plan);
    const int ctas = static_cast<int>(min(static_cast<long long>(grid), total));
    if (cta >= ctas) return;
    const long long w0 = piece_start(total, ctas, cta), w1 = piece_start(total, ctas, cta + 1);
    if (tid < kStages) sh.holds[tid] = -1;
    if (tid == 0) sh.failed = 0;
    plan.locate(sh.plan, w0);
    @SETUP@
    float l[NT][2] = {}, n[NT][2] = {};
    while (use.left > 0) {
      const int tiles = use.tiles_here();
      for (int t = 0; t < NT; ++t) l[t][0] = l[t][1] = 0.0f;
      const int begin = (warp - page0) & (kWarps - 1);
      for (int tile = begin; tile < tiles; tile += kWarps) {
        @WAIT@
        const int entry_here = a.batch.block_table[use.b * a.batch.max_pages + use.span.first + use.tile + tile];
        const bool there = entry_here >= 0 && entry_here < a.cache.num_pages;
        for (int look = 0; look < 3; ++look) {         // as long as the warp works on the page
          if (sh.there[stage] != there) wrong("a page is taken for there, or for missing");
          for (int kind = 0; there && kind < 2; ++kind) {
            const uint8_t* from;
            memcpy(&from, smem + stage * Shape::kStageBytes + kind * Block::kBytes, sizeof(from));
            if (from != kv4_block<D>(a.cache, entry_here, kind, use.head)) wrong("another page than this warp's");
          }
          if (look < 2) stop(AT_LOOK);
        }
        if (lane == 0) {
          ++covered[std::make_tuple(use.b, use.rt, use.head, use.tile + tile)];
          ++consumed;
        }
        @ASK@
      }
      page0 += tiles;
      if (lane == 0) nan_of[warp] = l[0][0] != l[0][0];
      __syncthreads();
      if (tid == 0 && (nan_of[0] || nan_of[1] || nan_of[2] || nan_of[3]))
        for (int tile = 0; tile < tiles; ++tile) spoilt.insert(std::make_tuple(use.b, use.rt, use.head, use.tile + tile));
      __syncthreads();
      use.advance(plan, tiles);
    }
    @END@
  }

  static int main(int sequences, int kind, int stall) {
    std::vector<int32_t> lens, starts = {0};
    for (int b = 0; b < sequences; ++b) {
      const int count = rnd(6) == 0 ? 0 : kind == 1 ? 1 + rnd(9) : 1;
      lens.push_back(count + (rnd(4) == 0 ? rnd(3000) : rnd(300)));
      starts.push_back(starts.back() + count);
    }
    const int width = 60;
    std::vector<int32_t> table(sequences * width);
    for (int32_t& e : table) e = rnd(8) == 0 ? -1 : rnd(500);
    a.cache = {nullptr, 1 << 20, 450, 2, 3};             // (addresses are only compared)
    a.batch = {table.data(), lens.data(), starts.data(), sequences, width, starts.back()};
    a.group = 4;
    a.window = kind == 2 ? 150 : 0;
    wait_limit = stall >= 0 ? 50000 : 1ll << 60;
    std::map<std::tuple<int, int, int, int>, int> all;
    const Plan<kKvPage, kRows, kDecodeExtra> plan = {a.batch, a.cache.heads, a.group, a.window};
    for (int b = 0; b < sequences; ++b) {
      const KvSequence s = kv_sequence(a.batch, b);
      for (int rt = 0; s.count > 0 && rt < plan.row_tiles(s); ++rt)
        for (int h = 0; h < a.cache.heads; ++h)
          for (int t = 0; t < plan.span(s, rt).tiles; ++t) all[std::make_tuple(b, rt, h, t)] = 1;
    }
    for (grid = 1; grid <= 6; grid += 5)
      for (int last = 0; last < kWarps; ++last) {
        covered.clear();
        spoilt.clear();
        int failures = 0;
        for (cta = 0; cta < grid; ++cta) {
          memset(static_cast<void*>(&sh), 0, sizeof(sh));
          pending.clear();
          open_bytes.clear();
          landings = status = 0;
          draining = false;
          stall_after = stall;
          run_block(32 * kWarps, kernel, (last + cta) % kWarps, world);
          if (!pending.empty() && stall < 0) wrong("copies on their way that nobody takes");
          if (!pending.empty() && stall >= 0) wrong("copies on their way into memory that is given back");
          failures += status != 0;
        }
        for (auto& [page, times] : covered)
          if (times != 1 || !all.count(page)) wrong("a page is done twice, or is none");
        if (stall < 0 && (covered.size() != all.size() || failures || !spoilt.empty())) wrong("pages are left out");
        for (auto& [page, one] : all)
          if (!covered.count(page) && !spoilt.count(page)) wrong("a page is left out and its rows are not NaN");
        if (stall >= 0 && covered.size() != all.size() && !failures) wrong("pages are left out and nobody says so");
      }
    printf("%d stages, %zu pages, %d taken, %d wrong\n", kStages, all.size(), consumed, bad);
    return bad != 0;
  }
};

int main(int, char** argv) {
  const int dim = atoi(argv[1]), nt = atoi(argv[2]), sequences = atoi(argv[3]), kind = atoi(argv[4]), stall = atoi(argv[5]);
  seed = sequences * 100 + kind;
  if (dim == 128) return nt == 1 ? Run<128, 1>::main(sequences, kind, stall) : Run<128, 2>::main(sequences, kind, stall);
  return nt == 1 ? Run<64, 1>::main(sequences, kind, stall) : Run<64, 2>::main(sequences, kind, stall);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    kernel, layout, internal = source("kv4_attention.cu"), source("kv4_internal.h"), source("kv_internal.h")
    plan = source("attention_plan.cuh").replace("#pragma once", "").replace('#include "kv_internal.h"', "")
    cache = piece(internal, "// A cache in device memory.", "};\n")
    of_a_call = piece(internal, "struct KvBatch {", "kv_sequence(const KvBatch& a, int b) {") + piece(internal.split("kv_sequence(const KvBatch& a, int b) {")[1], "\n", "\n}\n")
    blocks = piece(layout, "constexpr int kKv4Group", "template <int D>\nstruct Kv4Block {") + piece(layout.split("struct Kv4Block {")[1], "\n", "\n};\n") + piece(
        layout, "template <int D>\n__device__ __forceinline__ uint8_t* kv4_block", "\n}\n")
    constants = [piece(kernel, "constexpr int %s" % name, ";") for name in ("kDecodeExtra", "kWarps", "kStatusTimeout")]
    structs = [piece(kernel, "template <int D, int NT>\nstruct Decode4Shape", "\n};\n"), piece(kernel, "struct LoadWalk {", "\n};\n"),
               piece(kernel, "template <int D, int NT>\nstruct DecodeShared", "\n};\n"), piece(kernel, "__device__ __forceinline__ bool landed", "\n}\n")]
    harness = HARNESS.replace("@SETUP@", piece(kernel, "  Walk use;\n", "\"a stage for every warp's page\");"))
    harness = harness.replace("@WAIT@", piece(kernel, "if (lost || !__all_sync", "break;\n      }\n"))
    harness = harness.replace("@ASK@", piece(kernel, "__syncwarp();\n      ask(stage, page0 + tile + kStages);", "parity ^= 1u;\n      }\n"))
    harness = harness.replace("@END@", piece(kernel, "if (sh.failed != 0) {", "\n  }\n").replace("atomicExch(status", "atomicExch(&status"))
    text = EMULATOR + ROLE_SHIM + "namespace syfi {\nconstexpr int kKvPageHere = 64;\n" + cache + of_a_call + blocks + "}\n" + plan + "using namespace syfi;\n" + BEFORE
    return build(tmp_path_factory.mktemp("ring"), text + "\n".join(constants + structs) + harness)


@pytest.mark.parametrize("sequences", [1, 7, 40])
@pytest.mark.parametrize("kind", [0, 1, 2], ids=["decoding", "several rows", "window"])
@pytest.mark.parametrize("dim,nt", [(128, 1), (128, 2), (64, 1), (64, 2)], ids=["6 stages", "9 stages", "12 stages", "12 stages of 16 rows"])
def test_every_warp_finds_its_pages(dim, nt, kind, sequences, program):
    done = subprocess.run([program, str(dim), str(nt), str(sequences), str(kind), "-1"], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("stall", [0, 1, 2, 7, 20, 61])
@pytest.mark.parametrize("dim,nt", [(128, 1), (128, 2), (64, 1)], ids=["6 stages", "9 stages", "12 stages"])
def test_waits_that_run_out_spoil_their_rows_and_leave_no_copy_behind(dim, nt, stall, program):
    """From one copy on none lands until somebody waits for all of them."""
    done = subprocess.run([program, str(dim), str(nt), "7", "1", str(stall)], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout
