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


@pytest.mark.parametrize("kind,exponent", [("f32", 80), ("f32", 92), ("q8", 92), ("q4", 92), ("fp8", 92)])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_keys_and_small_queries(kind, exponent, sign):
    """Products of query and key are ordinary numbers, key by key in 32 bits as well; here all scores of a row are of one sign."""
    t = Tree(kind, 5, 300, 12, 2, 128, seed=4)
    t.q = np.abs(t.q).clip(0.3, 3.0)
    lift = np.float32(2.0 ** exponent)
    if t.ks is None:
        t.k = np.abs(t.k) * sign
        t.k[::3] *= lift
        t.k[1::3] *= lift * 2
        t.k[2::3] *= lift / 2
    else:
        codes = t.k.view(np.int8)
        if kind == "q8":
            t.k = (np.abs(codes.astype(np.int16)).clip(0, 127) * sign).astype(np.int8).view(np.uint8)
        elif kind == "q4":
            nibble = 3 if sign > 0 else 13
            t.k = np.where(np.arange(t.k.size).reshape(t.k.shape) % 5 < 3, nibble, nibble << 4).astype(np.uint8)
        else:
            t.k = (t.k & 0x7F) | (0x80 if sign < 0 else 0)
            t.k = t.k.astype(np.uint8)
        t.ks = (t.ks * lift).astype(np.float32)
    t.q = (t.q / lift / 16).astype(np.float32)
    assert np.all(np.abs(t.q) > 2.0 ** -126)
    y = Timed(t)
    y.call()
    # scores of either size: a weight's error is that of a score of up to 16, 16 2^-24 sqrt(128) / 8 and less
    assert near_rows(y.out.cpu().numpy(), t.want(), 4e-5)


@pytest.mark.parametrize("kind", ["f32", "q8", "q4", "fp8"])
@pytest.mark.parametrize("exponent", [100, 112, -100, -110])
def test_values_at_the_ends_of_their_range(kind, exponent):
    t = Tree(kind, 9, 200, 12, 2, 128, seed=6)
    lift = np.float32(2.0 ** exponent)
    if t.vs is None:
        t.v *= lift
    else:
        t.vs *= lift
    y = Timed(t)
    y.call()
    assert near_rows(y.out.cpu().numpy(), t.want())


@pytest.mark.parametrize("kind,n", [("f32", 1_300_003), ("fp8", 4_500_003)])
@pytest.mark.parametrize("window", [0, 2000])
def test_a_cache_beyond_32_bits_of_bytes(kind, n, window):
    """Zero rows but for a few near and far, whose weights stand out: scores of 0 and values of 0 have a closed form."""
    m, heads, kv_heads, d, cols = 3, 24, 4, 256, 1024
    g = torch.Generator(device="cuda").manual_seed(7)
    dtype = torch.float32 if kind == "f32" else torch.float8_e4m3fn
    k, v = (torch.zeros(n + m, cols, dtype=dtype, device="cuda") for _ in range(2))
    scale = None if kind == "f32" else torch.full((n + m,), 0.25, device="cuda")
    assert k.numel() * k.element_size() > 2 ** 32
    far = [5, n // 2, n - 1500, n - 1, *range(n, n + m)]
    rows = [torch.randint(-7, 8, (2, cols), device="cuda", generator=g).float() for _ in far]
    for j, (a, b) in zip(far, rows):
        k[j], v[j] = a.to(dtype), b.to(dtype)
    q = 2 * torch.randn(m, heads, d, device="cuda", generator=g) * (1.0 if kind == "f32" else 4.0)
    parents, out = torch.arange(m, device="cuda", dtype=torch.int32) - 1, torch.zeros(m, heads, d, device="cuda")
    s = None if scale is None else scale.data_ptr()
    assert capi.load_library().tsr_attention_tree(FORMAT[kind], q.data_ptr(), k.data_ptr(), v.data_ptr(), s, s, parents.data_ptr(), out.data_ptr(), m, n, heads,
                                                  kv_heads, d, 0, window, torch.cuda.current_stream().cuda_stream) == 0
    unit, want = 1.0 if scale is None else 0.25, np.zeros((m, heads, d))
    for i in range(m):
        first = n + i + 1 - window if window else 0
        seen = [x for j, x in zip(far, rows) if first <= j <= n + i]
        keys, values = (unit * torch.stack([x[c] for x in seen]).double().view(-1, kv_heads, d).cpu().numpy() for c in (0, 1))
        for h in range(heads):
            scores = keys[:, h // 6] @ q[i, h].double().cpu().numpy() / np.sqrt(d)
            top = max(0.0, scores.max())
            w = np.exp(scores - top)
            want[i, h] = w @ values[:, h // 6] / (w.sum() + (n + i + 1 - first - len(seen)) * np.exp(-top))
    assert near_rows(out.cpu().numpy(), want, 1e-4)  # (scores of up to 40)
