"""Workspaces of captured launches: graphs of one stream replayed at once, beside plain launches, made and dropped."""
import gc

import numpy as np
import pytest
import torch

from tessera_b200 import capi
from test_many_rows_gpu import Delta, Tree

pytestmark = pytest.mark.gpu


class Call:
    """A typed call that needs a workspace, with buffers of its own."""

    def __init__(self, what, seed):
        self.lib, self.what = capi.load_library(), what
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
        if what == "delta":
            t = self.t = Delta(500, 2, 8, 128, 64, seed=seed)
            self.ins = [up(x) for x in (t.s, t.k, t.v, t.q, t.alpha, t.beta)]
            self.outs = [torch.zeros(t.v.shape, device="cuda"), torch.zeros(t.s.shape, device="cuda")]
        else:
            t = self.t = Tree("fp8" if what == "tree" else "f32", 16, 4000, 12, 2, 128, seed=seed)
            self.ins = [None if x is None else up(x) for x in (t.q, t.k, t.v, t.ks, t.vs, t.parents)]
            self.outs = [torch.zeros(t.q.shape, device="cuda")]

    def call(self, stream):
        a, o, t = [None if x is None else x.data_ptr() for x in self.ins], [x.data_ptr() for x in self.outs], self.t
        if self.what == "delta":
            s, k, v, q, alpha, beta = a
            rc = self.lib.tsr_delta_chunk_heads(s, k, v, q, o[0], alpha, beta, o[1], t.heads, t.k_heads, t.dk, t.dv, t.rows, 0, 0, stream.cuda_stream)
        elif self.what == "tree":
            rc = self.lib.tsr_attention_tree(4, *a, *o, t.m, t.n, t.heads, t.kv_heads, t.d, 0, 0, stream.cuda_stream)
        else:  # causal, in chunks of keys
            rc = self.lib.tsr_attention(0, *a[:5], *o, t.m, t.n + t.m, t.heads, t.kv_heads, t.d, t.n, 0, 0, 1, stream.cuda_stream)
        assert rc == 0

    def clear(self):
        for x in self.outs:
            x.fill_(7.0)

    def results(self):
        return [x.cpu().numpy() for x in self.outs]


def captured(call, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call.call(stream)
    return graph


def alike(call, want):
    return all(np.array_equal(a, b) for a, b in zip(call.results(), want))


WHAT = ["delta", "tree", "attention"]


@pytest.mark.parametrize("what", WHAT)
def test_graphs_of_one_stream_replayed_at_once(what):
    stream, calls = torch.cuda.Stream(), [Call(what, s) for s in (1, 2, 3)]
    torch.cuda.synchronize()
    for c in calls:
        c.call(stream)
    torch.cuda.synchronize()
    want = [c.results() for c in calls]
    graphs = [captured(c, stream) for c in calls[:2]]
    for c in calls:
        c.clear()
    torch.cuda.synchronize()
    others = [torch.cuda.Stream() for _ in graphs]
    for _ in range(100):
        for g, s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
        calls[2].call(stream)  # and a plain launch on the stream they were captured on
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert alike(c, w)


@pytest.mark.parametrize("what", WHAT)
def test_two_calls_of_one_capture(what):
    stream, calls = torch.cuda.Stream(), [Call(what, s) for s in (4, 5)]
    torch.cuda.synchronize()
    for c in calls:
        c.call(stream)
    torch.cuda.synchronize()
    want = [c.results() for c in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for c in calls:
            c.call(stream)
    for c in calls:
        c.clear()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert alike(c, w)


def test_buffers_of_dropped_graphs_serve_later_ones():
    stream, call = torch.cuda.Stream(), Call("delta", 6)
    torch.cuda.synchronize()
    call.call(stream)
    torch.cuda.synchronize()
    want, free = call.results(), []
    for _ in range(30):
        graph = captured(call, stream)
        call.clear()
        graph.replay()
        torch.cuda.synchronize()
        assert alike(call, want)
        del graph
        gc.collect()
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    assert free[5] - free[-1] < 8 << 20  # (a buffer is 8 MB and more)


def test_prompts_that_grow():
    """What a stream keeps after prompts of one to 64 chunks of rows: not much more than the largest needs."""
    heads, k_heads, d, rows = 48, 16, 128, 64 * 32
    new = lambda *shape: torch.full(shape, 0.01, device="cuda")
    s, k, v, gates, o = new(heads, d, d), new(rows, k_heads, d), new(rows, heads, d), new(rows, heads), new(rows, heads, d)
    stream, lib = torch.cuda.Stream(), capi.load_library()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for n in range(20, rows + 1, 60):
        assert lib.tsr_delta_chunk_heads(s.data_ptr(), k.data_ptr(), v.data_ptr(), k.data_ptr(), o.data_ptr(), gates.data_ptr(), gates.data_ptr(),
                                         s.data_ptr(), heads, k_heads, d, d, n, 0, 0, stream.cuda_stream) == 0
    torch.cuda.synchronize()
    chunk = k_heads * 2 * 32 * 4 * d + heads * (32 * 4 * d + 32 * 4 * 32 + 32 * d * 4 + 1024)  # keys and queries; W, P, u, factors
    assert free - torch.cuda.mem_get_info()[0] < 64 * chunk * 1.75
