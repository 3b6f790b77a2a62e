"""The converting warps of the chunk kernel over the 4-bit cache on the host (csrc/kv4_attention_chunk.cu): rows asked for a tile ahead and table
entries two, over the ends of segments; stages that are written only once they are free; and roles that give up.  The kernel's own text, with
one warp always the last to run and the other roles at random.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, ROLE_SHIM, build, piece, source

BEFORE = r"""
struct float2 { float x, y; };
static float2 make_float2(float x, float y) { return {x, y}; }
struct int2 { int x, y; };
static float __uint_as_float(unsigned u) { return __int_as_float(static_cast<int>(u)); }
static unsigned __reduce_min_sync(unsigned, unsigned v) { long long m = v; for (long long x : exchange(v)) m = std::min(m, x); return static_cast<unsigned>(m); }
template <typename T> static T __ldg(const T* p) { return *p; }
struct AttentionArgs { KvCache cache; KvBatch batch; };
static unsigned seed = 1;
static int bad, rows_asked;
static void wrong(const char* what) { if (++bad < 6) printf("%s\n", what); }
static int rnd(int m) { seed = seed * 1664525u + 1013904223u; return static_cast<int>((seed >> 8) % m); }
// The converting warps' barrier, which tells all whether any gave true.
static unsigned arrived, meetings;
static bool any_now, any_then;
static bool meet(bool p) {
  const unsigned before = meetings;
  any_now |= p;
  if (++arrived == blockDim.x) {
    any_then = any_now;
    any_now = false;
    arrived = 0;
    ++meetings;
  }
  while (meetings == before) stop(AT_LOOK);
  return any_then;
}
static void named_bar_sync(int, int) { meet(false); }
static bool converters_any(bool p) { return meet(p); }
// Barriers in memory: arrivals that complete a phase.
static std::map<uint64_t*, int> needs, got;
static void mbar_arrive(uint64_t* bar) {
  if (++got[bar] == needs[bar]) {
    got[bar] = 0;
    ++*bar;
  }
}
static uint32_t smem_u32(const void*) { return 0; }
static std::map<uint32_t, const uint8_t*> content;      // of a row in shared memory: where it came from
static void st_shared_16(uint32_t at, uint32_t, uint32_t, uint32_t, uint32_t) { content[at] = nullptr; }
static bool known_block(const uint8_t* block);
static void (*on_ask)();
template <int D>
struct RawRow {
  const uint8_t* from = nullptr;
  uint32_t groups[D / 64] = {};
  float scale = 0.0f;
  void ask(const uint8_t* block, int at) {
    if (!known_block(block)) wrong("a row outside the cache is asked for");
    ++rows_asked;
    on_ask();
    from = block + at;
    scale = 1.0f + (reinterpret_cast<uintptr_t>(from) % 9973);
  }
  void put(uint32_t to) const { content[to] = from; }
};
"""

HARNESS = r"""
static AttentionArgs a;
static bool known_block(const uint8_t* block) {
  const long long at = block - a.cache.base;
  return at >= 0 && at < a.cache.num_pages * a.cache.page_stride;
}

template <int D>
struct World {
  using Shape = ChunkShape<D>;
  static constexpr int kStages = Shape::kStages;
  struct Tile { int b, tile, head; bool any_low_high[kTile], all; int any_low, any_high; };
  static inline ChunkShared sh;
  alignas(16) static inline uint8_t smem[Shape::kSmem];
  static inline std::vector<Segment> segments;
  static inline std::vector<Tile> tiles;
  static inline int described, keys, values, scales, fail_after, fail_at_row, asked, steps;
  static int entry(const Tile& x, int t) {
    const int page = 2 * x.tile + t / kKvPage;
    const bool any = page < a.batch.max_pages && page * kKvPage <= x.any_high && (page + 1) * kKvPage > x.any_low;
    const int e = any ? a.batch.block_table[x.b * a.batch.max_pages + page] : -1;
    return e >= 0 && e < a.cache.num_pages ? e : -1;
  }
  static const uint8_t* row(const Tile& x, int t, int kind) { return kv4_block<D>(a.cache, entry(x, t), kind, x.head) + t % kKvPage; }
  static uint32_t place(int base, int stage, int t) { return base + stage * Shape::kTileBytes + t * 128 + (t & 7) * 16; }
  static bool seen(const Tile& x, int t) { return x.tile * kTile + t >= x.any_low && x.tile * kTile + t <= x.any_high; }
  static bool step() {                       // the other roles
    if (++steps > 100000) return false;             // everybody waits
    if (fail_after >= 0 && steps > fail_after) sh.abort_code = kStatusTimeout;
    if (sh.abort_code != 0) return true;     // nothing is freed any more
    const int what = rnd(4);
    if (what == 0 && described < static_cast<int>(segments.size()) && described - static_cast<int>(sh.segment_empty[described % kSegmentRing]) * kSegmentRing < kSegmentRing) {
      sh.segment[described % kSegmentRing] = segments[described];
      ++sh.segment_full[described++ % kSegmentRing];
    }
    if (what == 1 && keys < static_cast<int>(tiles.size()) && static_cast<int>(sh.k_full[keys % kStages]) > keys / kStages) {
      for (int t = 0; t < kTile; ++t)
        if (entry(tiles[keys], t) >= 0 && content[place(Shape::kK, keys % kStages, t)] != row(tiles[keys], t, 0)) wrong("other keys than the tile's");
      ++sh.k_empty[keys++ % kStages];
    }
    if (what == 2 && values < static_cast<int>(tiles.size()) && static_cast<int>(sh.v_full[values % kStages]) > values / kStages) {
      const Tile& x = tiles[values];
      for (int t = 0; t < kTile; ++t)
        if (content[place(Shape::kV, values % kStages, t)] != (entry(x, t) >= 0 && seen(x, t) ? row(x, t, 1) : nullptr)) wrong("other values than the tile's");
      ++sh.v_empty[values++ % kStages];
    }
    if (what == 3 && scales < static_cast<int>(tiles.size()) && static_cast<int>(sh.scale_full[scales % kScaleStages]) > scales / kScaleStages) {
      const Tile& x = tiles[scales];
      const float* at = reinterpret_cast<const float*>(smem + Shape::kScales) + scales % kScaleStages * 2 * kTile;
      for (int t = 0; t < kTile; ++t) {
        const bool there = entry(x, t) >= 0;
        if (at[t] != (there ? 1.0f + (reinterpret_cast<uintptr_t>(row(x, t, 0)) % 9973) : 0.0f)) wrong("other key scales than the tile's");
        if (at[kTile + t] != (there && seen(x, t) ? 1.0f + (reinterpret_cast<uintptr_t>(row(x, t, 1)) % 9973) : 1.0f)) wrong("other value scales than the tile's");
      }
      if ((sh.flags[scales % kScaleStages] & 3) != (entry(x, 0) >= 0 ? 1 : 0) + (entry(x, kKvPage) >= 0 ? 2 : 0)) wrong("other pages are there");
      ++sh.scale_empty[scales++ % kScaleStages];
    }
    return true;
  }
  static int run(int count, int fail, int fail_row) {
    on_ask = [] { if (fail_at_row >= 0 && asked++ >= fail_at_row) sh.abort_code = kStatusTimeout; };    // (in between whatever the warps do)
    std::vector<int32_t> table(3 * 30);
    for (int32_t& e : table) e = rnd(6) == 0 ? -1 : rnd(50);
    a.cache = {nullptr, 1 << 20, 45, 2, 3};          // (addresses are only compared)
    a.batch = {table.data(), nullptr, nullptr, 3, 30, 0};
    for (int last = 0; last < 4; ++last) {
      segments.clear();
      tiles.clear();
      for (int i = 0; i < count; ++i) {
        Segment g = {};
        g.b = rnd(3);
        g.head = rnd(3);
        g.tile0 = rnd(12);
        g.tiles = 1 + rnd(rnd(3) == 0 ? 1 : 4);
        g.any_low = rnd(3) == 0 ? g.tile0 * kTile + rnd(kTile) : 0;
        g.any_high = (g.tile0 + g.tiles) * kTile - 1 - rnd(kTile);
        g.all_low = g.any_low + rnd(40);
        g.all_high = g.any_high - rnd(40);
        segments.push_back(g);
        for (int j = 0; j < g.tiles; ++j) {
          Tile x = {};
          x.b = g.b;
          x.tile = g.tile0 + j;
          x.head = g.head;
          x.any_low = g.any_low;
          x.any_high = g.any_high;
          tiles.push_back(x);
        }
      }
      segments.push_back(Segment{});           // the piece's end
      memset(static_cast<void*>(&sh), 0, sizeof(sh));
      content.clear();
      needs.clear();
      got.clear();
      for (int i = 0; i < kSegmentRing; ++i) needs[&sh.segment_empty[i]] = 4;
      for (int i = 0; i < 4; ++i) needs[&sh.k_full[i]] = needs[&sh.v_full[i]] = 4;
      for (int i = 0; i < kScaleStages; ++i) needs[&sh.scale_full[i]] = 1;
      described = keys = values = scales = steps = 0;
      fail_after = fail;
      fail_at_row = fail_row;
      asked = 0;
      run_block(128, [] { convert_role<D>(a, sh, smem); }, last, step);
      while (sh.abort_code == 0 && (keys < static_cast<int>(tiles.size()) || values < static_cast<int>(tiles.size()) || scales < static_cast<int>(tiles.size())) && step()) {}
      if (fail < 0 && fail_row < 0 && (keys != static_cast<int>(tiles.size()) || values != keys || scales != keys)) wrong("tiles are left out");
    }
    printf("%zu tiles, %d rows asked for, %d wrong\n", tiles.size(), rows_asked, bad);
    return bad != 0;
  }
};

int main(int, char** argv) {
  const int count = atoi(argv[2]), fail = atoi(argv[3]), fail_row = atoi(argv[4]);
  seed = count * 1000 + fail + fail_row + 7;
  return atoi(argv[1]) == 64 ? World<64>::run(count, fail, fail_row) : World<128>::run(count, fail, fail_row);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    chunk, layout, internal = source("kv4_attention_chunk.cu"), source("kv4_internal.h"), source("kv_internal.h")
    cache = piece(internal, "// A cache in device memory.", "  int batch, max_pages, tokens;\n};\n")
    blocks = piece(layout, "constexpr int kKv4Group", "template <int D>\nstruct Kv4Block {") + piece(layout.split("struct Kv4Block {")[1], "\n", "\n};\n") + piece(
        layout, "template <int D>\n__device__ __forceinline__ uint8_t* kv4_block", "\n}\n")
    constants = [piece(chunk, "constexpr %s" % name, ";") for name in ("int kTile ", "int kScaleStages", "int kStatusTimeout", "int kSoftmaxWarps", "float kNear")]
    parts = [piece(chunk, "template <int D>\nstruct ChunkShape", "\n};\n"), piece(chunk, "struct Segment {", "\n};\n"), piece(chunk, "constexpr int kSegmentRing", "\n\n"),
             piece(chunk, "struct ChunkShared {", "\n};\n"), piece(chunk, "__device__ __forceinline__ bool wait_for", "\n}\n"),
             piece(chunk, "__device__ __forceinline__ void wait_whole_warp", "}\n"), piece(chunk, "template <int N>\nstruct Ring {", "\n};\n"),
             piece(chunk, "template <int D>\n__device__ __forceinline__ void convert_role(", "\n}\n")]
    return build(tmp_path_factory.mktemp("convert"), "\n".join([EMULATOR + ROLE_SHIM + cache + blocks + BEFORE, *constants, *parts, HARNESS]))


@pytest.mark.parametrize("segments", [0, 1, 2, 5, 25])
@pytest.mark.parametrize("dim", [64, 128])
def test_every_tile_has_its_rows(dim, segments, program):
    done = subprocess.run([program, str(dim), str(segments), "-1", "-1"], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("fail_after", [0, 1, 5, 30, 100, 333, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_all_four_warps_leave_when_a_role_gives_up(dim, fail_after, program):
    done = subprocess.run([program, str(dim), "25", str(fail_after), "-1"], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("row", [0, 100, 128, 200, 256, 300, 1000, 1111, 1500, 2000])
@pytest.mark.parametrize("dim", [64, 128])
def test_all_four_warps_leave_when_a_role_gives_up_while_they_work(dim, row, program):
    done = subprocess.run([program, str(dim), "25", "-1", str(row)], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout
