"""Scratch buffers of streams and captured graphs on the GPU: replays beside calls and beside each other give each call's own result.
Needs a B200."""
import gc
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def kv():
    return importlib.import_module("oracle.kv_oracle")


def _inputs(kv, q_len, kv_lens, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [(n + 63) // 64 for n in kv_lens]
    cache = kv.random_cache(sum(need), 2, 2, 128, seed, DEV)
    table = torch.zeros(len(kv_lens), max(need), dtype=torch.int32, device=DEV)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n, dtype=torch.int32, device=DEV)
    q = torch.randn(q_len * len(kv_lens), 8, 128, generator=g, device=DEV).to(torch.bfloat16)
    starts = torch.arange(len(kv_lens) + 1, dtype=torch.int32, device=DEV) * q_len
    return q, cache, table, torch.tensor(kv_lens, dtype=torch.int32, device=DEV), starts


def _attention(pkg, inputs):
    out = torch.empty_like(inputs[0])
    return out, lambda: pkg.run_paged_attention(*inputs, out)


def _indexer(pkg, lens, seed):
    from oracle import dsa_oracle
    inputs = tuple(t.to(DEV) for t in dsa_oracle.make_inputs(lens, seed=seed))
    out = torch.empty(len(lens), 2048, dtype=torch.int32, device=DEV)
    return out, lambda: pkg.run_dsa_topk_indexer(*inputs, out)


def _captured(call, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


def _jobs(pkg, kv, op, n):
    """(output, call) of n small calls that differ, and of one that needs a larger buffer."""
    if op == "attention":
        return [_attention(pkg, _inputs(kv, 1, [3000 + 500 * i, 20000], i)) for i in range(n)], _attention(pkg, _inputs(kv, 300, [2000, 900], 77))
    return [_indexer(pkg, [9000 + 64 * i, 700], i) for i in range(n)], _indexer(pkg, [60000, 20000, 900], 77)


@pytest.mark.parametrize("op", ["attention", "indexer"])
def test_graphs_outlive_larger_calls_on_their_streams(op, pkg, kv):
    """Ten streams capture a small call each; larger calls follow on the same streams, then the graphs are replayed beside them."""
    small, (large_out, large) = _jobs(pkg, kv, op, 10)
    want = []
    for out, call in small:
        call()
        want.append(out.clone())
    large()
    large_want = large_out.clone()
    streams = [torch.cuda.Stream() for _ in small]
    graphs = [_captured(call, s) for (_, call), s in zip(small, streams)]
    for s in streams:
        with torch.cuda.stream(s):
            large()
    torch.cuda.synchronize()
    for _ in range(5):
        for out, _ in small:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        large()
        torch.cuda.synchronize()
        assert torch.equal(large_out, large_want)
        for (out, _), w in zip(small, want):
            assert torch.equal(out, w)


@pytest.mark.parametrize("op", ["attention", "indexer"])
def test_graphs_captured_on_one_stream_run_side_by_side(op, pkg, kv):
    small, _ = _jobs(pkg, kv, op, 6)
    want = []
    for out, call in small:
        call()
        want.append(out.clone())
    capturing = torch.cuda.Stream()
    graphs = [_captured(call, capturing) for _, call in small]
    streams = [torch.cuda.Stream() for _ in small]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (out, _), w in zip(small, want):
        assert torch.equal(out, w)


@pytest.mark.parametrize("op", ["attention", "indexer"])
def test_a_graphs_buffer_is_used_again_when_the_graph_is_gone(op, pkg, kv):
    """Capturing again and again takes no more memory."""
    _, (out, call) = _jobs(pkg, kv, op, 1)
    call()
    want = out.clone()
    free = []
    for _ in range(12):
        graph = _captured(call, torch.cuda.Stream())
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        graph.reset()
        del graph
        gc.collect()
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info(0)[0])
    assert free[-1] >= free[4], free


def test_branches_of_one_graph_have_buffers_of_their_own(pkg, kv):
    small, (large_out, large) = _jobs(pkg, kv, "attention", 3)
    calls = [call for _, call in small] + [large]
    outs = [out for out, _ in small] + [large_out]
    want = []
    for out, call in zip(outs, calls):
        call()
        want.append(out.clone())
    main, sides = torch.cuda.Stream(), [torch.cuda.Stream() for _ in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        for s, call in zip(sides, calls):
            s.wait_stream(main)
            with torch.cuda.stream(s):
                call()
                call()
        for s in sides:
            main.wait_stream(s)
    for _ in range(10):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
