"""The tree attention where values, scales and scores are at the ends of their ranges."""
import numpy as np
import pytest
import torch

from tessera_b200 import capi
from test_many_rows_gpu import Tree, near_rows

pytestmark = pytest.mark.gpu

FORMAT = {"f32": 0, "f16": 1, "q8": 2, "q4": 3, "fp8": 4}


class Timed:
    """A typed call on the current stream; its time (us) as the smallest of several."""

    def __init__(self, t):
        self.t, self.lib = t, capi.load_library()
        up = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()
        self.ins = [up(x) for x in (t.q, t.k, t.v, t.ks, t.vs, t.parents)]
        self.out = torch.zeros(t.q.shape, device="cuda")

    def call(self):
        t = self.t
        assert self.lib.tsr_attention_tree(FORMAT[t.kind], *(None if x is None else x.data_ptr() for x in self.ins), self.out.data_ptr(), t.m, t.n, t.heads,
                                           t.kv_heads, t.d, 0, t.window, torch.cuda.current_stream().cuda_stream) == 0

    def time(self):
        self.call()
        best = 1e30
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            self.call()
            b.record()
            b.synchronize()
            best = min(best, 1e3 * a.elapsed_time(b))
        return best


@pytest.mark.parametrize("kind", ["f32", "q8"])
def test_a_cleared_cache_costs_no_more(kind):
    """Equal scores and values of zero (or scales of zero): no row is found not finite and computed again key by key, which takes
    ten times as long and more."""
    t = Tree(kind, 8, 4096, 24, 4, 256, seed=1)
    usual = Timed(t).time()
    t.k[:], t.v[:] = 0, 0
    if t.ks is not None:
        t.ks[:], t.vs[:] = 0, 0
    cleared = Timed(t)
    assert cleared.time() < 3 * usual
    assert bool((cleared.out == 0).all())


@pytest.mark.parametrize("kind", ["f32", "q8"])
def test_a_row_of_zeros_costs_no_more(kind):
    """One value row of zeros in every tile."""
    t = Tree(kind, 8, 4096, 24, 4, 256, seed=3)
    usual = Timed(t).time()
    t.v[5::64] = 0
    if t.vs is not None:
        t.vs[5::64] = 0
    some = Timed(t)
    assert some.time() < 3 * usual
    assert near_rows(some.out.cpu().numpy(), t.want())


@pytest.mark.parametrize("kind", ["f32", "q8"])
def test_tiles_of_zero_values_among_others(kind):
    t = Tree(kind, 8, 700, 12, 2, 128, seed=2)
    t.q[:4] = 0.0
    zero = t.vs if t.vs is not None else t.v
    zero[64:192] = 0.0
    zero[300:310] = 0.0
    y = Timed(t)
    y.call()
    assert near_rows(y.out.cpu().numpy(), t.want())
