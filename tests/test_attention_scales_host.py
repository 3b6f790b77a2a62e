"""The chunk kernel's scale warp on the host, with copies that land in the order that is worst for it: scales as early as the kernel's
rings allow, values as late.  Shared memory is full of NaN bytes before, as an earlier kernel may leave it.  No GPU needed."""
import shutil
import subprocess

import pytest

from host_block import EMULATOR, ROLE_SHIM, build, role

HARNESS = r"""
template <int D>
struct World {
  using Shape = ChunkShape<D>;
  static constexpr int kTiles = 12;
  alignas(1024) static inline uint8_t smem[Shape::kSmem];
  static inline ChunkShared sh;
  static inline int scales, values, cleaned, described, bad, masked_from;
  static float* scale_of(int t) { return reinterpret_cast<float*>(smem + Shape::kScales) + t % kScaleStages * 2 * kTile; }
  static uint8_t* value_of(int t) { return smem + Shape::kV + t % Shape::kVStages * Shape::kTileBytes; }
  static bool step() {
    if (described < 2) {                       // the segment, then the end of the piece
      Segment& g = sh.segment[described];
      g = Segment{};
      g.tiles = described == 0 ? kTiles : 0;
      g.any_high = kTiles * kTile - 1;
      g.all_high = masked_from * kTile - 1;
      ++sh.segment_full[described++];
    } else if (scales < kTiles && (scales < kScaleStages || (cleaned > scales - kScaleStages && values > scales - kScaleStages - 1)) &&
               values >= scales - Shape::kVStages) {
      for (int i = 0; i < 2 * kTile; ++i) scale_of(scales)[i] = 1.0f;
      sh.there[scales % kScaleStages] = 3;
      ++sh.scale_full[scales++ % kScaleStages];
    } else if (values < kTiles && cleaned >= values - Shape::kVStages + 1) {
      memset(value_of(values), 0x38, Shape::kTileBytes);
      value_of(values)[swizzled<D>(values, 0)] = 0x7f;       // position t of tile t is a NaN
      ++sh.v_full[values++ % Shape::kVStages];
    } else {
      return false;
    }
    return true;
  }
  static void clean() {                        // the scale warp hands tile `cleaned` over
    for (int i = 0; i < kTile; ++i) {
      const bool taken_out = __float_as_int(scale_of(cleaned)[i]) == kNoValue;
      if (taken_out != (cleaned >= masked_from && i == cleaned) && ++bad < 5) printf("tile %d, position %d: %s\n", cleaned, i, taken_out ? "taken out" : "left in");
    }
    ++cleaned;
  }
  static int run() {
    memset(smem, 0x7f, sizeof(smem));
    sh = ChunkShared{};
    run_block(32, [] { scale_role<D>(sh, smem); }, 0, step);
    if (cleaned != kTiles) { printf("%d tiles\n", cleaned); ++bad; }
    return bad != 0;
  }
};
static void mbar_arrive(uint64_t* bar) {
  auto mine = [&](auto world) {
    for (uint64_t& b : world.sh.scale_clean)
      if (bar == &b) world.clean();
  };
  mine(World<64>{});
  mine(World<128>{});
}
int main(int, char** argv) {
  World<64>::masked_from = World<128>::masked_from = atoi(argv[2]);
  return atoi(argv[1]) == 64 ? World<64>::run() : World<128>::run();
}
"""

@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    return build(tmp_path_factory.mktemp("scales"), EMULATOR + ROLE_SHIM + role("scale_role") + "\n" + HARNESS)


@pytest.mark.parametrize("masked_from", range(13))
@pytest.mark.parametrize("dim", [64, 128])
def test_values_are_looked_at_when_they_have_landed(dim, masked_from, program):
    done = subprocess.run([program, str(dim), str(masked_from)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout
