"""The steps of many rows as a program runs them: one after another (launch by launch, queued, replayed as a graph), through the
typed calls on streams of their own, captured, and on pointers that are aligned to four bytes only."""
import numpy as np
import pytest
import torch

from tessera_b200 import capi
from test_many_rows_gpu import KINDS, SUFFIX, U, Delta, Norm, Tree, check_logprob, decode, logprob_reference, near_rows, near_whole, run, tree_reference

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one step of a model over drafted rows

class Step:
    """A verification step of m drafted rows over n cached ones: queries and keys normalised, rotated and appended, attention
    over the tree, the delta rule over the accepted chain, the rows' log probabilities."""

    def __init__(self, backend, kind, seed=0):
        g = np.random.default_rng(seed)
        self.backend, self.kind, self.m, self.n = backend, kind, 9, 40
        self.norm, self.tree, self.delta = Norm(9, 6, 2, 128, 64, seed), Tree(kind, 9, 40, 6, 2, 128, seed=seed), Delta(9, 2, 4, 64, 32, seed)
        self.logits, self.targets = (2 * g.standard_normal((9, 5003))).astype(np.float32), g.integers(0, 5003, 9).astype(np.uint32)
        up, t, d = backend.upload, self.norm, self.delta
        self.inputs = [up(t.q), up(t.k), up(t.v), up(t.q_w), up(t.k_w), up(t.pos)]
        self.q_out, self.out = backend.AllocateBuffer(t.q.nbytes), backend.AllocateBuffer(t.q.nbytes)
        self.caches = [up(self.tree.k), up(self.tree.v)]
        self.scales = [up(self.tree.ks), up(self.tree.vs)] if self.tree.ks is not None else []
        self.parents = up(self.tree.parents)
        self.d_in = [up(x) for x in (d.s, d.k, d.v, d.q, d.alpha, d.beta)]
        self.d_out = [backend.AllocateBuffer(d.v.nbytes), backend.AllocateBuffer(d.s.nbytes)]
        self.l_in = [up(self.logits), up(self.targets)]
        self.l_out = [backend.AllocateBuffer(9 * 4 * k) for k in (1, 1, 5, 5)]

    def issue(self):
        b, t, d, f16 = self.backend, self.tree, self.delta, int(self.kind == "f16")
        q, k, v, q_w, k_w, pos = self.inputs
        run(b, "qk_norm_rope_append" + SUFFIX[self.kind], [q, k, v, q_w, k_w, pos, self.q_out, *self.caches, *self.scales],
            self.norm.scalars() + [self.n] + ([] if self.scales else [f16]))
        run(b, "attention_tree" + SUFFIX[self.kind], [self.q_out, *self.caches, *self.scales, self.parents, self.out],
            [self.m, self.n, 6, 2, 128, 0, 0] + ([] if self.scales else [f16]))
        s, dk, dv, dq, alpha, beta = self.d_in
        run(b, "delta_chunk_heads", [s, dk, dv, dq, self.d_out[0], alpha, beta, self.d_out[1]], [d.heads, d.k_heads, d.dk, d.dv, d.rows, 0, 0])
        run(b, "logprob_rows", [*self.l_in, *self.l_out], [9, 5003, 5, 0])

    def results(self):
        b, t, d = self.backend, self.tree, self.delta
        return [b.download(self.q_out, np.float32, t.q.size), b.download(self.out, np.float32, t.q.size), b.download(self.d_out[0], np.float32, d.v.size),
                b.download(self.d_out[1], np.float32, d.s.size), *(b.download(x, dt, 9 * k) for x, dt, k in zip(self.l_out, "ffIf", (1, 1, 5, 5)))]

    def caches_now(self):
        t = self.tree
        kept = [self.backend.download(x, np.uint8, y.nbytes).view(y.dtype).reshape(y.shape) for x, y in zip(self.caches, (t.k, t.v))]
        scales = [self.backend.download(x, np.float32, t.n + t.m) for x in self.scales] or [None, None]
        return [decode(self.kind, x, s, 256).reshape(-1, 2, 128) for x, s in zip(kept, scales)]

    def check(self, got):
        q, out, o, s, given, _, ids, tops = got
        want_q, size = self.norm.want("q")
        assert np.all(np.abs(q.reshape(want_q.shape) - want_q) <= 16 * U * size)
        k, v = self.caches_now()  # of what was written, the attention
        assert near_rows(out.reshape(9, 6, 128), tree_reference(q.reshape(9, 6, 128), k, v, self.tree.parents, self.n, 3, 0))
        o_want, s_want = self.delta.want()
        assert near_whole(o.reshape(o_want.shape), o_want) and near_whole(s.reshape(s_want.shape), s_want)
        r = logprob_reference(self.logits, self.targets, 5)
        assert np.array_equal(ids.reshape(9, 5), r[2])
        for a, w in ((given, r[0]), (tops.reshape(9, 5), r[3])):  # sums of 10 exponentials a thread, arguments of up to 16
            assert np.all(np.abs(a - w) <= U * (5003 / 512 + 64 + 6 * 16) + 2 * U * np.abs(w))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("deferred", [0, 1, 2])
def test_a_step_of_drafted_rows(backend, kind, deferred):
    step = Step(backend, kind, seed=50)
    step.issue()
    first = step.results()
    step.check(first)
    backend.SetDeferred(deferred)
    try:
        for rep in range(4):  # (queued, the later passes replay what an earlier one captured)
            graphs0 = backend.LaunchStats()[2]
            for _ in range(3):  # (as the layers of a model: a graph is made of eight launches at least)
                step.issue()
            backend.Synchronize()
            graphs1 = backend.LaunchStats()[2]
            again = step.results()
            assert all(np.array_equal(a, b) for a, b in zip(first, again))
        assert (graphs1 - graphs0 == 1) == (deferred == 1)
    finally:
        backend.SetDeferred(0)
    step.check(again)


# ------------------------------------------------------------------ the delta rule's widths

@pytest.mark.parametrize("shape", [(40, 16, 48, 128, 128), (40, 8, 64, 64, 128), (70, 4, 80, 128, 128), (70, 2, 10, 128, 48), (45, 1, 8, 64, 176), (600, 16, 16, 64, 16),
                                   (33, 3, 15, 128, 32), (1, 16, 48, 128, 128)], ids=lambda s: "x".join(map(str, s)))
def test_delta_rule_of_many_heads(backend, shape):
    """Scans of 32, 48 and 64 columns a CTA, one to eight value heads a key head, more chunks than SMs."""
    t = Delta(*shape, seed=sum(shape))
    o, s = t.launch(backend)
    o_want, s_want = t.want()
    assert near_whole(o, o_want) and near_whole(s, s_want)


@pytest.mark.parametrize("heads", [8, 2, 6, 4])
def test_delta_rule_after_another_number_of_heads(backend, heads):
    """Fewer, then more value heads a key head: each call has the shared memory that it needs."""
    t = Delta(5, 2, heads, 128, 16, seed=heads)
    assert near_whole(t.launch(backend)[0], t.want()[0])


# ------------------------------------------------------------------ the typed calls

def shifted(x, by):
    """x on the device, `by` bytes off a 256-byte boundary."""
    x = torch.from_numpy(np.ascontiguousarray(x))
    raw = torch.full((x.numel() * x.element_size() + by,), 0x55, dtype=torch.uint8, device="cuda")
    raw[by:] = x.reshape(-1).view(torch.uint8).cuda() if x.numel() else raw[by:]
    return raw


class Typed:
    """One typed call with its inputs, outputs and reference; `by`: how far off a boundary every pointer is."""

    def __init__(self, what, kind="f32", by=0, seed=0):
        self.what, self.kind, self.by, self.lib = what, kind, by, capi.load_library()
        if what == "tree":
            t = self.t = Tree(kind, 11, 70, 6, 2, 128, seed=seed)
            self.ins = [t.q, t.k, t.v, t.ks, t.vs, t.parents]
            outs = [t.q]
        elif what == "norm":
            t = self.t = Norm(11, 6, 2, 128, 64, seed=seed)
            self.ins = [t.q, t.k, t.q_w, t.k_w]
            outs = [t.q, t.k]
        elif what == "delta":
            t = self.t = Delta(75, 2, 4, 64, 48, seed=seed)
            self.ins = [t.s, t.k, t.v, t.q, t.alpha, t.beta]
            outs = [t.v, t.s]
        else:
            g = np.random.default_rng(seed)
            self.x, self.targets = (3 * g.standard_normal((5, 4099))).astype(np.float32), g.integers(0, 4099, 5).astype(np.uint32)
            self.ins = [self.x, self.targets]
            outs = [self.x[:, 0], self.x[:, 0], self.x[:, :7], self.x[:, :7]]
        self.sizes = [(x.shape, np.uint32 if what == "logprob" and i == 2 else np.float32) for i, x in enumerate(outs)]
        self.ins = [x if x is None else shifted(x, by) for x in self.ins]
        self.outs = [shifted(np.full(x.shape, 7.0, np.float32), by) for x in outs]
        self.pos = torch.from_numpy(self.t.pos.astype(np.int64)).cuda() if what == "norm" else None

    def pointer(self, x):
        return None if x is None else x.data_ptr() + self.by

    def call(self, stream=None):
        a, o = [self.pointer(x) for x in self.ins], [self.pointer(x) for x in self.outs]
        st = (stream or torch.cuda.current_stream()).cuda_stream
        t = getattr(self, "t", None)
        if self.what == "tree":
            fmt = {"f32": 0, "f16": 1, "q8": 2, "q4": 3, "fp8": 4}[self.kind]
            return self.lib.tsr_attention_tree(fmt, *a, *o, t.m, t.n, t.heads, t.kv_heads, t.d, 0, 0, st)
        if self.what == "norm":
            return self.lib.tsr_qk_norm_rope(*a, self.pos.data_ptr(), *o, t.rows, t.heads, t.kv_heads, t.d, t.rope_dim, t.theta, *t.sections, t.eps, st)
        if self.what == "delta":
            s, k, v, q, alpha, beta = a
            return self.lib.tsr_delta_chunk_heads(s, k, v, q, o[0], alpha, beta, o[1], t.heads, t.k_heads, t.dk, t.dv, t.rows, 0, 0, st)
        return self.lib.tsr_logprob_rows(*a, *o, 5, 4099, 7, 0, st)

    def clear(self):
        for x in self.outs:
            x.fill_(0x55)

    def results(self):
        return [x[self.by:].cpu().numpy().view(dt).reshape(shape).copy() for x, (shape, dt) in zip(self.outs, self.sizes)]

    def check(self, got):
        if self.what == "tree":
            assert near_rows(got[0], self.t.want())
        elif self.what == "norm":
            for y, which in zip(got, "qk"):
                want, size = self.t.want(which)
                assert np.all(np.abs(y - want) <= 16 * U * size)
        elif self.what == "delta":
            assert all(near_whole(y, r) for y, r in zip(got, self.t.want()))
        else:
            r = logprob_reference(self.x, self.targets, 7)
            assert np.array_equal(got[2], r[2])
            tol = U * (4099 / 512 + 64 + 6 * 30)
            for y, w in ((got[0], r[0]), (got[3], r[3])):
                assert np.all(np.abs(y - w) <= tol + 2 * U * np.abs(w))
            assert np.all(np.abs(got[1] - r[1]) <= tol * 32)


CALLS = [("tree", k) for k in KINDS] + [("norm", "f32"), ("delta", "f32"), ("logprob", "f32")]


@pytest.mark.parametrize("what,kind", CALLS)
@pytest.mark.parametrize("by", [0, 4, 8])
def test_typed_calls_on_any_alignment(backend, what, kind, by):
    c = Typed(what, kind, by, seed=60)
    assert c.call() == 0
    torch.cuda.synchronize()
    got = c.results()
    c.check(got)
    for x in c.outs:
        assert bool((x[:by] == 0x55).all())


@pytest.mark.parametrize("what,kind", CALLS)
def test_typed_calls_captured_and_replayed(backend, what, kind):
    stream = torch.cuda.Stream()
    a = Typed(what, kind, seed=61)
    with torch.cuda.stream(stream):
        assert a.call(stream) == 0  # (the workspace of this stream)
    torch.cuda.synchronize()
    want = a.results()
    a.check(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert a.call(stream) == 0
    for _ in range(3):
        a.clear()
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(x, y) for x, y in zip(a.results(), want))


@pytest.mark.parametrize("what,kind", [("delta", "f32"), ("tree", "f16")])
def test_two_graphs_share_a_stream_s_workspace(backend, what, kind):
    """Two captured calls of one stream, replayed in turn, and one of a smaller size between them."""
    stream = torch.cuda.Stream()
    calls = [Typed(what, kind, seed=s) for s in (62, 63)]
    for c in calls:
        assert c.call(stream) == 0
    torch.cuda.synchronize()
    want = [c.results() for c in calls]
    graphs = []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            assert c.call(stream) == 0
    for c in calls:
        c.clear()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(3):
            for g in graphs:
                g.replay()
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert all(np.array_equal(x, y) for x, y in zip(c.results(), w))


@pytest.mark.parametrize("what,kind", CALLS)
def test_two_streams_at_once(backend, what, kind):
    calls = [Typed(what, kind, seed=s) for s in (64, 65)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            assert c.call(s) == 0
    torch.cuda.synchronize()
    for c in calls:
        c.check(c.results())


def test_a_capture_before_the_first_call_is_refused(backend):
    """A workspace cannot grow in a capture: the call says so, and the capture goes on."""
    stream = torch.cuda.Stream()
    c, x = Typed("delta", seed=66), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert c.call(stream) == int(capi.StatusCode.UnsupportedFeature)
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 4


# ------------------------------------------------------------------ the attention's scales

@pytest.mark.parametrize("kind", ["q8", "q4", "fp8"])
@pytest.mark.parametrize("spread", [4, 30])
def test_tree_over_scales_far_apart(backend, kind, spread):
    """Value rows 2^(2 spread) apart, and key rows whose scales are 0."""
    t = Tree(kind, 6, 200, 6, 2, 128, seed=70)
    t.vs *= np.exp2(np.random.default_rng(71).integers(-spread, spread + 1, t.vs.shape)).astype(np.float32)
    t.ks[10:20] = 0.0
    t.vs[30:35] = 0.0
    assert near_rows(t.launch(backend), t.want(), 4e-5)  # (the largest rows need not be those of the largest weights)


# ------------------------------------------------------------------ log probabilities of few tokens

@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 511, 513])
def test_logprob_of_small_vocabularies(backend, vocab):
    x = np.random.default_rng(vocab).standard_normal((3, vocab)).astype(np.float32)
    check_logprob(backend, x, np.array([0, vocab - 1, vocab], np.uint32), min(32, vocab))


@pytest.mark.parametrize("what", ["random", "rising", "falling", "equal", "steps", "late", "lowest"])
@pytest.mark.parametrize("top_k", [1, 32])
def test_logprob_of_many_rows_of_many_tiles(backend, what, top_k):
    """More rows than the machine has room for two CTAs of: a CTA walks over the whole row, the list fills on the way."""
    rows, vocab = 150, 50001 if what == "steps" else 50000
    g = np.random.default_rng(80)
    x = g.standard_normal((rows, vocab)).astype(np.float32)
    if what in ("rising", "falling"):
        x = np.sort(x, 1)[:, ::1 if what == "rising" else -1].copy()
    elif what == "equal":
        x[:] = 0.25
    elif what == "steps":
        x = np.round(x)
    elif what == "late":  # a flood after a long calm
        x[:, 30000:] += 20.0
        x[::2, 45000:] += np.linspace(0, 5, vocab - 45000, dtype=np.float32)
    elif what == "lowest":
        x[:, 9000:40000] = np.finfo(np.float32).min
    check_logprob(backend, x, g.integers(0, vocab, rows).astype(np.uint32), top_k)


def test_a_state_carried_from_call_to_call(backend):
    """Prompts in pieces, the state in place, nothing waiting in between: as with a wait after every piece."""
    stream, lib, t = torch.cuda.Stream(), capi.load_library(), Delta(8 * 45, 2, 6, 128, 64, seed=90)
    x = {n: torch.from_numpy(getattr(t, n)).cuda() for n in ("k", "v", "q", "alpha", "beta", "s")}
    found = []
    for wait in (False, True):
        s, o = x["s"].clone(), torch.zeros_like(x["v"])
        torch.cuda.synchronize()
        for at in range(0, t.rows, 45):
            k, v, q, alpha, beta = (x[n][at:at + 45].data_ptr() for n in ("k", "v", "q", "alpha", "beta"))
            assert lib.tsr_delta_chunk_heads(s.data_ptr(), k, v, q, o[at:].data_ptr(), alpha, beta, s.data_ptr(), 6, 2, 128, 64, 45, 0, 0, stream.cuda_stream) == 0
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        found.append((o.cpu().numpy(), s.cpu().numpy()))
    assert all(np.array_equal(a, b) for a, b in zip(*found))
    assert all(near_whole(y, r) for y, r in zip(found[0], t.want()))


@pytest.mark.parametrize("kind", ["f32", "fp8"])
def test_tree_captured_before_the_first_call(backend, kind):
    """Without a workspace the keys are not cut into chunks: the same rows but for roundings."""
    stream, c = torch.cuda.Stream(), Typed("tree", kind, seed=91)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert c.call(stream) == 0
    c.clear()
    graph.replay()
    torch.cuda.synchronize()
    c.check(c.results())
