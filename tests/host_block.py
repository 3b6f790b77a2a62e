"""Device functions of the kernels on the host: C++ text with the threads of a block as contexts, which a scheduler switches where they
wait for one another, and helpers that take pieces of a source file and compile them behind it."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlsys-contest-syfi-agent-assisted_b200", "csrc")

EMULATOR = r"""
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>
#include <algorithm>
#include <map>
#include <tuple>
#include <vector>
#define __device__
#define __forceinline__ inline
struct Dim { unsigned x; };
static Dim threadIdx, blockDim;
static int min(int a, int b) { return a < b ? a : b; }
static int max(int a, int b) { return a > b ? a : b; }
static unsigned max(unsigned a, unsigned b) { return a > b ? a : b; }
static long long min(long long a, long long b) { return a < b ? a : b; }

enum { READY, AT_SHUFFLE, AT_BARRIER, AT_LOOK, DONE };     // AT_LOOK: a look at a barrier in memory that found it closed
struct Thread { ucontext_t context; std::vector<char> stack; int state; long long given; };
static std::vector<Thread> threads;
static ucontext_t scheduler;
static std::vector<std::vector<long long>> handed;   // of each warp: what its lanes gave at the last shuffle
static void stop(int state) {
  Thread& t = threads[threadIdx.x];
  const unsigned me = threadIdx.x;
  t.state = state;
  swapcontext(&t.context, &scheduler);
  threadIdx.x = me;
}
static const std::vector<long long>& exchange(long long v) {
  threads[threadIdx.x].given = v;
  stop(AT_SHUFFLE);
  return handed[threadIdx.x / 32];
}
static void __syncthreads() { stop(AT_BARRIER); }
static void __syncwarp() { exchange(0); }
template <typename T> T __shfl_xor_sync(unsigned, T v, int d) { return static_cast<T>(exchange(v)[(threadIdx.x % 32) ^ d]); }
template <typename T> T __shfl_up_sync(unsigned, T v, int d) { const int l = threadIdx.x % 32; return static_cast<T>(exchange(v)[l >= d ? l - d : l]); }
template <typename T> T __shfl_sync(unsigned, T v, int l) { return static_cast<T>(exchange(v)[l]); }
static int __reduce_add_sync(unsigned, int v) { long long s = 0; for (long long x : exchange(v)) s += x; return static_cast<int>(s); }
static unsigned __reduce_max_sync(unsigned, unsigned v) { long long m = 0; for (long long x : exchange(v)) m = std::max(m, x); return static_cast<unsigned>(m); }
static int __any_sync(unsigned, int p) { int any = 0; for (long long x : exchange(p)) any |= x != 0; return any; }

static void (*body)();
static void entry() { body(); threads[threadIdx.x].state = DONE; swapcontext(&threads[threadIdx.x].context, &scheduler); }
// Runs f in n threads.  The warp `last_warp` runs only when no other can; when none can, `world` is asked to go on (false: it cannot).
static void run_block(unsigned n, void (*f)(), unsigned last_warp, bool (*world)() = nullptr) {
  body = f;
  blockDim.x = n;
  threads.assign(n, Thread{});
  handed.assign(n / 32, std::vector<long long>(32));
  for (Thread& t : threads) {
    t.stack.resize(1 << 16);
    getcontext(&t.context);
    t.context.uc_stack.ss_sp = t.stack.data();
    t.context.uc_stack.ss_size = t.stack.size();
    t.context.uc_link = nullptr;
    makecontext(&t.context, entry, 0);
  }
  auto run_warp = [&](unsigned w) {
    bool moved = false;
    for (unsigned i = w * 32; i < w * 32 + 32; ++i)
      if (threads[i].state == READY) {
        threadIdx.x = i;
        swapcontext(&scheduler, &threads[i].context);
        moved = true;
      }
    bool all = true;
    for (unsigned i = w * 32; i < w * 32 + 32; ++i) all &= threads[i].state == AT_SHUFFLE;
    if (all) {
      for (unsigned i = 0; i < 32; ++i) handed[w][i] = threads[w * 32 + i].given;
      for (unsigned i = 0; i < 32; ++i) threads[w * 32 + i].state = READY;
    }
    return moved;
  };
  while (true) {
    bool moved = false;
    for (unsigned w = 0; w < n / 32; ++w)
      if (w != last_warp) moved |= run_warp(w);
    if (moved) continue;
    if (run_warp(last_warp)) continue;
    bool barrier = true, done = true, look = false;
    for (Thread& t : threads) {
      barrier &= t.state == AT_BARRIER;
      done &= t.state == DONE;
      look |= t.state == AT_LOOK;
    }
    if (done) return;
    if (!barrier && !(look && world && world())) { printf("threads wait for what does not come\n"); exit(2); }
    for (Thread& t : threads)
      if (t.state == AT_BARRIER || t.state == AT_LOOK) t.state = READY;
  }
}
"""


def source(name):
    return open(os.path.join(CSRC, name)).read()


def piece(text, first, last):
    """From `first` up to and with the next `last`."""
    found = re.search(re.escape(first) + ".*?" + re.escape(last), text, flags=re.S)
    assert found, first
    return found.group(0)


def build(folder, text):
    """The path of the compiled program."""
    path, out = folder / "host.cpp", folder / "host"
    path.write_text(text)
    done = subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-o", str(out), str(path)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-3000:]
    return str(out)


# What the chunk kernel's roles need around them: types, casts, and barriers in memory whose word counts the phases that are over.
ROLE_SHIM = r"""
struct float4 { float x, y, z, w; };
struct uint4 { uint32_t x, y, z, w; };
static float __int_as_float(int i) { float f; memcpy(&f, &i, 4); return f; }
static int __float_as_int(float f) { int i; memcpy(&i, &f, 4); return i; }
static unsigned __float_as_uint(float f) { return static_cast<unsigned>(__float_as_int(f)); }
static float ex2(float x) { return exp2f(x); }
static void fence_proxy_async_smem() {}
static void mbar_arrive(uint64_t* bar);
static long long clocks, look_clocks;           // now, and what a look takes that finds a barrier closed
static long long clock64() { return clocks; }
static void __nanosleep(unsigned n) { clocks += 2 * n; stop(AT_LOOK); }
static bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  if ((*bar & 1) != parity) return true;
  clocks += look_clocks;
  stop(AT_LOOK);                               // (the hardware waits a while, too)
  return (*bar & 1) != parity;
}
constexpr int kKvPage = 64;
"""


def role(*names):
    """The chunk kernel's shared memory, its waits and the functions `names`, as C++ for the host."""
    chunk, common = source("paged_attention_chunk.cu"), source("attention_common.cuh")
    constants = [line for line in piece(chunk, "constexpr int kTile = 128;", "template <int D>").splitlines() if line.startswith("constexpr")]
    return "\n".join([
        piece(common, "template <int D>\n__device__ __forceinline__ int swizzled", "\n}\n"), *constants, piece(chunk, "template <int D>\nstruct ChunkShape", "\n};\n"),
        piece(chunk, "struct Segment {", "\n};\n"), piece(chunk, "constexpr int kSegmentRing", "\n\n"), piece(chunk, "struct ChunkShared {", "\n};\n"),
        piece(chunk, "__device__ __forceinline__ int tile_exponent", "\n}\n"), piece(chunk, "__device__ __forceinline__ bool wait_for", "// ------"),
        *(piece(chunk, "template <int D>\n__device__ __forceinline__ void %s(" % name, "\n}\n") for name in names)])
