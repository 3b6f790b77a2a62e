"""The scratch buffers of streams and captured graphs on the host, with a CUDA runtime that only keeps books: whose memory a call gets, and
that no memory which a live graph uses is freed or given to anybody else.  No GPU needed."""
import random
import shutil
import subprocess

import pytest

from host_block import build, source

SHIM = r"""
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <atomic>
#include <map>
#include <mutex>
#include <new>
#include <set>
#include <type_traits>
#include <vector>
#define CUDART_CB
typedef int CUresult, cudaError_t, CUtensorMap, CUtensorMapDataType, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill;
typedef uint32_t cuuint32_t;
typedef uint64_t cuuint64_t;
enum { CUDA_SUCCESS = 0, cudaSuccess = 0, cudaEnableDefault = 0, cudaStreamNonBlocking = 0 };
enum CUstreamCaptureStatus { CU_STREAM_CAPTURE_STATUS_NONE, CU_STREAM_CAPTURE_STATUS_ACTIVE };
enum cudaStreamCaptureStatus { cudaStreamCaptureStatusNone, cudaStreamCaptureStatusActive };
enum cudaDriverEntryPointQueryResult { cudaDriverEntryPointSuccess };
enum cudaStreamCaptureMode { cudaStreamCaptureModeRelaxed };
enum { cudaUserObjectNoDestructorSync = 1, cudaGraphUserObjectMove = 1 };
struct Object { void* self; void (*destroy)(void*); };
typedef Object* cudaUserObject_t;
struct Graph { unsigned long long id; std::vector<Object*> objects; };
typedef Graph* cudaGraph_t;
struct Stream { unsigned long long id; Graph* capturing; };
typedef Stream *CUstream, *cudaStream_t;
static std::set<void*> alive;
static long long waits;
static int cudaMalloc(void** p, size_t n) { *p = malloc(n); alive.insert(*p); return 0; }
static int cudaFree(void* p) { alive.erase(p); return 0; }        // (not given back, so that no address comes twice)
static int cudaDeviceSynchronize() { ++waits; return 0; }
static int cudaStreamCreateWithFlags(cudaStream_t*, int) { return 0; }
static int cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) { memset(p, v, n); return 0; }
static int cudaStreamSynchronize(cudaStream_t) { return 0; }
static int cudaStreamDestroy(cudaStream_t) { return 0; }
static int cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode*) { return 0; }
static int is_capturing(CUstream s, CUstreamCaptureStatus* status) { *status = s->capturing ? CU_STREAM_CAPTURE_STATUS_ACTIVE : CU_STREAM_CAPTURE_STATUS_NONE; return 0; }
static int stream_id(CUstream s, unsigned long long* id) { *id = s->id; return 0; }
static int cudaGetDriverEntryPoint(const char* name, void** p, int, cudaDriverEntryPointQueryResult* q) {
  *p = strstr(name, "Capturing") ? reinterpret_cast<void*>(is_capturing) : strstr(name, "GetId") ? reinterpret_cast<void*>(stream_id) : nullptr;
  *q = cudaDriverEntryPointSuccess;
  return 0;
}
static int cudaStreamGetCaptureInfo_v2(cudaStream_t s, cudaStreamCaptureStatus* status, unsigned long long* id, cudaGraph_t* graph, void*, void*) {
  *status = cudaStreamCaptureStatusActive;
  *id = s->capturing->id;
  *graph = s->capturing;
  return 0;
}
static int cudaUserObjectCreate(cudaUserObject_t* o, void* self, void (*destroy)(void*), int, int) { *o = new Object{self, destroy}; return 0; }
static int cudaUserObjectRelease(cudaUserObject_t o, int) { o->destroy(o->self); return 0; }
static int cudaGraphRetainUserObject(cudaGraph_t g, cudaUserObject_t o, int, int) { g->objects.push_back(o); return 0; }
namespace syfi {
static int set_last_error(int code, const char* what) { printf("error: %s\n", what); return code; }
}
"""

HARNESS = r"""
using namespace syfi;
int main(int argc, char** argv) {
  // commands: e STREAM SIZE: a call; c STREAM GRAPH SIZE: a call that is captured; d GRAPH: the graph is destroyed; n STREAM: the stream is another one
  static ScratchPool pool;
  std::map<int, Stream> streams;
  std::map<int, Graph> graphs;
  std::map<void*, int> used;                   // memory of live graphs
  std::map<void*, long long> size;
  unsigned long long next_id = 1;
  char op;
  int bad = 0, stream, graph;
  long long bytes, held = 0;
  while (scanf(" %c", &op) == 1) {
    if (op == 'd') {
      if (scanf("%d", &graph) != 1) return 3;
      for (Object* o : graphs[graph].objects) o->destroy(o->self);
      for (auto it = used.begin(); it != used.end();) it = it->second == graph ? used.erase(it) : std::next(it);
      graphs.erase(graph);
      continue;
    }
    if (scanf("%d", &stream) != 1) return 3;
    if (!streams.count(stream) || op == 'n') streams[stream] = {next_id++, nullptr};
    if (op == 'n') continue;
    if (op == 'c') {
      if (scanf("%d", &graph) != 1) return 3;
      if (!graphs.count(graph)) graphs[graph].id = next_id++;
      streams[stream].capturing = &graphs[graph];
    }
    if (scanf("%lld", &bytes) != 1) return 3;
    const long long waited = waits;
    int rc = 0;
    auto* s = pool.get(&streams[stream], bytes, 16, 2, &rc);
    streams[stream].capturing = nullptr;
    if (!s || !s->memory || static_cast<long long>(s->bytes) < bytes || !alive.count(s->memory)) { ++bad; printf("%c: no buffer\n", op); continue; }
    if (op == 'c' && waits != waited) { ++bad; printf("a capture waits for the device\n"); }
    if (used.count(s->memory) && !(op == 'c' && used[s->memory] == graph)) { ++bad; printf("%c %d: the buffer of graph %d\n", op, stream, used[s->memory]); }
    if (op == 'c') used[s->memory] = graph;
    for (auto& u : used)
      if (!alive.count(u.first)) { ++bad; printf("%c %d: graph %d's buffer is freed\n", op, stream, u.second); }
  }
  printf("%zu buffers\n", alive.size());
  return bad != 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    text = "\n".join(line for line in source("stream_scratch.h").splitlines() if not line.startswith("#"))
    return build(tmp_path_factory.mktemp("scratch"), SHIM + text + HARNESS)


def _run(program, commands):
    done = subprocess.run([program], input="\n".join(commands), capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout[:2000]
    return int(done.stdout.split()[-2])


def test_streams_keep_their_buffers_and_the_ninth_takes_one_over(program):
    assert _run(program, ["e %d 100" % (i % 8) for i in range(40)]) == 8
    assert _run(program, ["e %d 100" % i for i in range(20)]) == 8


def test_a_call_on_a_capturing_stream_never_frees_a_graphs_buffer(program):
    """Eight streams have captured small calls, then large ones come on the same streams."""
    _run(program, ["c %d %d 100" % (i, i) for i in range(8)] + ["e %d 4000" % i for i in range(8)])
    _run(program, ["e %d 100" % i for i in range(8)] + ["c %d %d 100" % (i, i) for i in range(8)] + ["e %d 4000" % i for i in range(12)])


def test_captures_of_growing_size_on_few_streams(program):
    _run(program, ["c %d %d %d" % (s, 10 * s + size, 100 * size) for s in range(3) for size in (1, 2, 8)] + ["c 9 99 800", "c 9 98 100"])


def test_graphs_captured_on_one_stream_have_a_buffer_each_and_give_it_back(program):
    assert _run(program, [c for g in range(30) for c in ("c 0 %d 100" % g, "c 0 %d 100" % g, "d %d" % g)]) == 1
    assert _run(program, ["c 0 %d 100" % g for g in range(5)] + ["d %d" % g for g in range(5)] + ["c 1 %d 100" % g for g in range(10, 15)]) == 5


def test_a_streams_handle_that_comes_again_is_another_stream(program):
    _run(program, ["c 0 1 100", "n 0", "e 0 100", "c 0 2 100", "n 0", "c 0 3 100", "e 0 200"])


@pytest.mark.parametrize("seed", range(10))
def test_any_order(seed, program):
    rng, graphs, commands = random.Random(seed), [], []
    for step in range(400):
        kind = rng.random()
        if kind < 0.5:
            commands.append("e %d %d" % (rng.randrange(12), rng.choice([100, 200, 4000])))
        elif kind < 0.8 or not graphs:
            graph = rng.choice(graphs) if graphs and rng.random() < 0.3 else 1000 + step
            if graph not in graphs:
                graphs.append(graph)
            commands.append("c %d %d %d" % (rng.randrange(12), graph, rng.choice([100, 200, 4000])))
        elif kind < 0.95:
            commands.append("d %d" % graphs.pop(rng.randrange(len(graphs))))
        else:
            commands.append("n %d" % rng.randrange(12))
    _run(program, commands)
