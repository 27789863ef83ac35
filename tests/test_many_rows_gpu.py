"""The steps of many rows on the GPU (ids attention_tree*, qk_norm_rope*, delta_chunk_heads, logprob_rows) against plain
numpy in 64 bits.  A rounding to fp32 is off by at most 2^-24 of the value, to binary16 by 2^-11, to E4M3 by 2^-4."""
import numpy as np
import pytest
import torch

from tessera_b200 import capi
from tessera_b200.backend import KernelLaunch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KINDS = ("f32", "f16", "q8", "q4", "fp8")
SUFFIX = {"f32": "", "f16": "", "q8": "_q8", "q4": "_q4", "fp8": "_fp8"}
LIMIT = {"q8": 127.0, "q4": 7.0, "fp8": 448.0}


def bits(x):
    return int(np.float32(x).view(np.uint32))


def run(backend, name, buffers, scalars):
    backend.LaunchKernel(backend.LoadKernel(name), KernelLaunch(buffers=buffers, scalars=scalars))


def e4m3_values():
    return torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()


def encode(kind, x):
    """Rows of a cache in its format: (bytes, scales or None)."""
    if kind == "f32":
        return x.astype(np.float32), None
    if kind == "f16":
        return x.astype(np.float16), None
    scale = (np.abs(x).max(1) / LIMIT[kind]).astype(np.float32)
    y = x / scale[:, None]
    if kind == "fp8":
        return torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), scale
    c = np.rint(y).astype(np.int8).view(np.uint8)
    return (c if kind == "q8" else (c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4)).copy(), scale


def decode(kind, codes, scale, cols):
    """The values rows of a cache stand for, in 64 bits."""
    if kind in ("f32", "f16"):
        return codes.astype(np.float64).reshape(-1, cols)
    if kind == "fp8":
        v = e4m3_values()[codes]
    elif kind == "q8":
        v = codes.view(np.int8).astype(np.float64)
    else:
        low, high = ((codes << 4).view(np.int8) >> 4), (codes.view(np.int8) >> 4)
        v = np.stack([low, high], -1).astype(np.float64)
    return v.reshape(-1, cols) * scale.astype(np.float64)[:, None]


# ------------------------------------------------------------------ attention over a tree

def sees(parents, n, i, window):
    """The cache rows that row i of a tree sees, or None for a row that is not used."""
    path, at = [], i
    while 0 <= at and -1 <= parents[at] < at:
        path.append(n + at)
        at = parents[at]
    if at != -1:
        return None
    keys = list(range(n)) + path[::-1]
    return keys[-window:] if window else keys


def tree_reference(q, k, v, parents, n, group, window):
    m, heads, d = q.shape
    out = np.zeros((m, heads, d))
    for i in range(m):
        keys = sees(parents, n, i, window)
        if keys is None:
            continue
        for h in range(heads):
            s = k[keys, h // group] @ q[i, h].astype(np.float64) / np.sqrt(d)
            w = np.exp(s - s.max())
            out[i, h] = w @ v[keys, h // group] / w.sum()
    return out


def make_tree(g, m, shape):
    p = np.arange(m) - 1
    if shape != "chain":
        p = np.maximum(p - g.integers(0, 1 + np.minimum(np.arange(m), 7)), -1)
    if shape == "holes":  # unused rows among the others, and rows below them
        p[g.random(m) < 0.25] = -2
        p[m // 2] = m  # a row behind it
    return p.astype(np.int32)


class Tree:
    def __init__(self, kind, m, n, heads, kv_heads, d, window=0, shape="bushy", seed=0, row_base=0):
        g = np.random.default_rng(seed)
        self.__dict__.update(kind=kind, m=m, n=n, heads=heads, kv_heads=kv_heads, d=d, window=window, row_base=row_base)
        self.q = (1.5 * g.standard_normal((m, heads, d))).astype(np.float32)
        self.k, self.ks = encode(kind, g.standard_normal((n + m, kv_heads * d)))
        self.v, self.vs = encode(kind, g.standard_normal((n + m, kv_heads * d)))
        self.parents = make_tree(g, m, shape)

    def launch(self, backend, q=None, out=None):
        rows = self.row_base + self.m
        if q is None:
            full = np.full((rows, self.heads, self.d), 7.0, np.float32)
            full[self.row_base:] = self.q
            q = backend.upload(full)
        out = out or backend.upload(np.full((rows, self.heads, self.d), 7.0, np.float32))
        scales = [backend.upload(self.ks), backend.upload(self.vs)] if self.ks is not None else []
        sc = [self.m, self.n, self.heads, self.kv_heads, self.d, self.row_base, self.window]
        run(backend, "attention_tree" + SUFFIX[self.kind],
            [q, backend.upload(self.k), backend.upload(self.v), *scales, backend.upload(self.parents), out],
            sc if scales else sc + [int(self.kind == "f16")])
        return backend.download(out, np.float32, rows * self.heads * self.d).reshape(rows, self.heads, self.d)

    def want(self):
        cols = self.kv_heads * self.d
        k, v = (decode(self.kind, x, s, cols).reshape(-1, self.kv_heads, self.d) for x, s in ((self.k, self.ks), (self.v, self.vs)))
        return tree_reference(self.q, k, v, self.parents, self.n, self.heads // self.kv_heads, self.window)


def near_rows(y, r, tol=2e-5):
    """Of every (row, head) by itself.  A score's error is about sqrt(head_dim) 2^-24 of the largest products' sum (scores
    up to 6: 6e-6), a weight's the same relative to it, and the weights of a row are normalised: 2e-5 of the largest output."""
    y, r = y.reshape(-1, y.shape[-1]).astype(np.float64), r.reshape(-1, r.shape[-1])
    return bool(np.all(np.isfinite(y)) and np.all(np.abs(y - r).max(1) <= tol * np.abs(r).max(1)))


TREES = [  # m, n, heads, kv_heads, head_dim, window, shape
    (1, 0, 4, 2, 128, 0, "chain"), (1, 1, 8, 1, 256, 0, "bushy"), (3, 0, 6, 1, 256, 0, "bushy"), (7, 63, 24, 4, 256, 0, "bushy"),
    (16, 64, 6, 6, 128, 0, "bushy"), (16, 500, 24, 4, 256, 0, "holes"), (33, 129, 14, 2, 128, 0, "holes"), (40, 200, 5, 1, 256, 50, "bushy"),
    (64, 1000, 16, 2, 128, 0, "chain"), (20, 30, 8, 2, 128, 5, "chain"), (9, 700, 6, 2, 256, 1, "holes"), (70, 10, 3, 1, 128, 64, "holes"),
    (200, 77, 4, 2, 128, 0, "bushy"), (256, 3, 2, 2, 256, 0, "chain"), (2, 5000, 24, 4, 256, 0, "bushy"), (12, 2500, 7, 1, 128, 0, "bushy"),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", TREES, ids=lambda s: "x".join(map(str, s)))
def test_tree_rows_see_their_path(backend, kind, shape):
    t = Tree(kind, *shape[:5], window=shape[5], shape=shape[6], seed=sum(shape[:5]), row_base=2 if shape[0] % 2 else 0)
    y, r = t.launch(backend), t.want()
    assert near_rows(y[t.row_base:], r)
    assert np.all(y[:t.row_base] == 7.0)
    unused = np.array([sees(t.parents, t.n, i, t.window) is None for i in range(t.m)])
    assert np.all(y[t.row_base:][unused] == 0.0)


@pytest.mark.parametrize("kind", KINDS)
def test_a_tree_without_a_used_row(backend, kind):
    t = Tree(kind, 5, 100, 8, 2, 128)
    t.parents[:] = (-2, 5, 0, 1, 2)
    assert np.all(t.launch(backend) == 0.0)


@pytest.mark.parametrize("kind", ["f32", "f16", "fp8"])
def test_what_a_row_does_not_see_may_be_anything(backend, kind):
    """NaN and infinities in rows of the tree off the path, and in past rows outside the window."""
    t = Tree(kind, 24, 90, 12, 2, 128, window=40, shape="bushy", seed=3)
    t.parents[12:] = -2
    want = t.want()
    bad = {"f32": np.float32(np.nan), "f16": np.float16(np.inf), "fp8": 0x7F}[kind]
    for x in (t.k, t.v):
        x[:90 - 40] = bad
        x[90 + 12:] = bad
    if t.ks is not None:
        t.ks[90 + 12:] = np.inf
        t.vs[:50] = np.nan
    assert near_rows(t.launch(backend), want)
    # a sibling's row: seen by itself and by what hangs from it alone
    t = Tree(kind, 8, 50, 4, 2, 128, seed=4)
    t.parents[:] = (-1, -1, 0, 1, 2, 3, 4, 0)
    want = t.want()
    t.v[50 + 3] = bad
    y = t.launch(backend)
    assert np.all(np.isnan(y[[3, 5]]) | np.isinf(y[[3, 5]]))
    assert near_rows(np.delete(y, (3, 5), 0), np.delete(want, (3, 5), 0))


def test_tree_over_large_and_small_values(backend):
    """Value rows of very different sizes, scores that leave one key, equal keys."""
    t = Tree("f32", 10, 300, 6, 2, 128, seed=5)
    t.v *= np.exp2(np.random.default_rng(6).integers(-20, 20, t.v.shape[0])).astype(np.float32)[:, None]
    t.q[3] *= 40.0
    t.k[:, :128] = t.k[0, :128]
    assert near_rows(t.launch(backend), t.want(), 1e-4)  # (scores of 240: 40 times the error of a weight above)


def test_tree_in_place_and_long(backend):
    """The result over the queries, and more keys than a CTA takes at a time."""
    t = Tree("fp8", 16, 9000, 24, 4, 256, seed=7)
    buf = backend.upload(t.q)
    assert near_rows(t.launch(backend, q=buf, out=buf), t.want())


def test_a_chain_is_causal_attention(backend):
    """A tree without branches against the causal id, whose row i sees keys up to n + i."""
    for kind in ("f32", "fp8"):
        t = Tree(kind, 12, 333, 24, 4, 256, shape="chain", seed=8)
        y = t.launch(backend)
        out = backend.AllocateBuffer(y.nbytes)
        if kind == "f32":
            run(backend, "attention", [backend.upload(t.q), backend.upload(t.k), backend.upload(t.v), out], [12, 345, 24, 4, 256, 333, 0, 0, 0, 1])
        else:
            run(backend, "attention_fp8", [backend.upload(x) for x in (t.q, t.k, t.v, t.ks, t.vs)] + [out], [12, 345, 24, 4, 256, 333, 0, 0, 2])
        assert near_rows(y, backend.download(out, np.float32, y.size).reshape(y.shape).astype(np.float64))


# ------------------------------------------------------------------ norms, rotation, append

def norm_rope_reference(x, w, pos, rope_dim, theta, sections, eps):
    y = x.astype(np.float64)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    half = rope_dim // 2
    axis = np.full(half, 2)
    axis[:sections[0] + sections[1]] = 1
    axis[:sections[0]] = 0
    angle = pos[:, axis].astype(np.float64) * np.float64(np.float32(theta)) ** (-np.arange(half) / half)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = y[..., :half], y[..., half:rope_dim]
    size = np.abs(y)  # what the roundings of an output are relative to
    size[..., :half] = size[..., half:rope_dim] = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, a * s + b * c, y[..., rope_dim:]], -1), size


class Norm:
    # heads, kv_heads, head_dim, rope_dim
    def __init__(self, rows, heads, kv_heads, d, rope_dim, seed=0):
        g = np.random.default_rng(seed)
        self.__dict__.update(rows=rows, heads=heads, kv_heads=kv_heads, d=d, rope_dim=rope_dim, theta=1e6, eps=1e-6)
        self.q, self.k, self.v = (g.standard_normal((rows, h, d)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
        self.q_w, self.k_w = (1.0 + 0.2 * g.standard_normal((2, d))).astype(np.float32)
        self.pos = g.integers(0, 300000, (rows, 3)).astype(np.uint64)
        pairs = rope_dim // 2
        self.sections = (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)

    def want(self, which):
        x, w = (self.q, self.q_w) if which == "q" else (self.k, self.k_w)
        return norm_rope_reference(x, w, self.pos, self.rope_dim, self.theta, self.sections, self.eps)

    def scalars(self):
        return [self.rows, self.heads, self.kv_heads, self.d, self.rope_dim, bits(self.theta), *self.sections, bits(self.eps)]


# a head's squares: eight a lane and five exchanges, half of whose error the root leaves; root, quotients, two products, the
# factors of the rotation, its products and their sum: 16 roundings
NORM_TOL = 16 * U
NORMS = [(1, 1, 1, 64, 64), (1, 24, 4, 256, 64), (5, 8, 2, 128, 128), (3, 6, 3, 96, 32), (2, 5, 1, 34, 18), (200, 24, 4, 256, 64), (7, 16, 16, 250, 100)]


@pytest.mark.parametrize("shape", NORMS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_and_rotation(backend, shape, in_place):
    t = Norm(*shape, seed=sum(shape))
    q, k = backend.upload(t.q), backend.upload(t.k)
    qo, ko = (q, k) if in_place else (backend.AllocateBuffer(t.q.nbytes), backend.AllocateBuffer(t.k.nbytes))
    run(backend, "qk_norm_rope", [q, k, backend.upload(t.q_w), backend.upload(t.k_w), backend.upload(t.pos), qo, ko], t.scalars())
    for buf, which, x in ((qo, "q", t.q), (ko, "k", t.k)):
        want, size = t.want(which)
        y = backend.download(buf, np.float32, x.size).reshape(x.shape)
        assert np.all(np.abs(y - want) <= NORM_TOL * size)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", NORMS[:4] + NORMS[5:6], ids=lambda s: "x".join(map(str, s)))
def test_norm_rotation_and_append(backend, kind, shape):
    t = Norm(*shape, seed=1 + sum(shape))
    cols, at, spare = t.kv_heads * t.d, 3, 2
    row_bytes = {"f32": 4 * cols, "f16": 2 * cols, "q8": cols, "q4": cols // 2, "fp8": cols}[kind]
    total = at + t.rows + spare
    caches = [backend.upload(np.full(total * row_bytes, 0x5A, np.uint8)) for _ in range(2)]
    scales = [backend.upload(np.full(total, 5.0, np.float32)) for _ in range(2)] if kind in LIMIT else []
    k, qo = backend.upload(t.k), backend.AllocateBuffer(t.q.nbytes)
    run(backend, "qk_norm_rope_append" + SUFFIX[kind],
        [backend.upload(t.q), k, backend.upload(t.v), backend.upload(t.q_w), backend.upload(t.k_w), backend.upload(t.pos), qo, *caches, *scales],
        t.scalars() + [at] + ([] if scales else [int(kind == "f16")]))
    want, size = t.want("q")
    assert np.all(np.abs(backend.download(qo, np.float32, t.q.size).reshape(t.q.shape) - want) <= NORM_TOL * size)
    assert np.array_equal(backend.download(k, np.float32, t.k.size).reshape(t.k.shape), t.k)
    k_want, k_size = t.want("k")
    for x, (r, err) in enumerate(((k_want.reshape(t.rows, cols), NORM_TOL * k_size.reshape(t.rows, cols)), (t.v.reshape(t.rows, cols).astype(np.float64), 0.0))):
        raw = backend.download(caches[x], np.uint8, total * row_bytes).reshape(total, row_bytes)
        assert np.all(raw[:at] == 0x5A) and np.all(raw[at + t.rows:] == 0x5A)
        rows = raw[at:at + t.rows]
        if kind == "f32":
            assert np.all(np.abs(rows.view(np.float32) - r) <= err)
        elif kind == "f16":
            assert np.all(np.abs(rows.view(np.float16).astype(np.float64) - r) <= 2.0 ** -11 * np.abs(r) + 2.0 ** -25 + 1.01 * err)
        else:
            s = backend.download(scales[x], np.float32, total)
            assert np.all(s[:at] == 5.0) and np.all(s[at + t.rows:] == 5.0)
            s = s[at:at + t.rows].astype(np.float64)
            exact = np.abs(r).max(1) / LIMIT[kind]
            assert np.all(np.abs(s - exact) <= (2 * U) * exact + np.max(err, initial=0.0) / LIMIT[kind])
            y = decode(kind, rows.copy(), s.astype(np.float32), cols)
            # half a step: of the integers one scale / 2; of E4M3 2^-4 of the value, and its codes below 2^-6 have steps of 2^-9,
            # the last of which the reference rounds down
            step = s[:, None] * 0.5 if kind != "fp8" else np.abs(r) * 2.0 ** -4 + s[:, None] * 2.0 ** -9
            assert np.all(np.abs(y - r) <= step * (1 + 1e-5) + 4 * U * np.abs(r) + err)


def test_append_equals_the_steps_it_stands_for(backend):
    """rmsnorm, mrope, quantize_q8 of a token's keys against the append: codes off by one at most where a value is next to
    the border between two codes."""
    t = Norm(9, 6, 2, 128, 64, seed=30)
    k, pos, w = backend.upload(t.k), backend.upload(t.pos), backend.upload(t.k_w)
    run(backend, "rmsnorm", [k, w, k], [18, 128, bits(t.eps)])
    run(backend, "mrope", [k, pos], [9, 2, 128, 64, bits(t.theta), *t.sections])
    codes, scale = backend.AllocateBuffer(9 * 256), backend.AllocateBuffer(36)
    run(backend, "quantize_q8", [k, codes, scale], [9, 256])
    caches = [backend.AllocateBuffer(9 * 256) for _ in range(2)]
    scales = [backend.AllocateBuffer(36) for _ in range(2)]
    run(backend, "qk_norm_rope_append_q8", [backend.upload(t.q), backend.upload(t.k), backend.upload(t.v), backend.upload(t.q_w), w, pos,
                                            backend.AllocateBuffer(t.q.nbytes), *caches, *scales], t.scalars() + [0])
    a, b = (backend.download(x, np.int8, 9 * 256).astype(int) for x in (codes, caches[0]))
    assert np.abs(a - b).max() <= 1 and np.mean(a != b) < 0.01
    sa, sb = backend.download(scale, np.float32, 9), backend.download(scales[0], np.float32, 9)
    assert np.all(np.abs(sa - sb) <= 2 * NORM_TOL * sa)


# ------------------------------------------------------------------ the delta rule in chunks

def delta_reference(s, k, v, q, alpha, beta):
    rows, heads, _ = v.shape
    s = s.astype(np.float64).copy()
    k, q = (np.tile(x.astype(np.float64), (1, heads // x.shape[1], 1)) for x in (k, q))
    out = np.zeros(v.shape)
    for t in range(rows):
        s *= alpha[t].astype(np.float64)[:, None, None]
        c = beta[t].astype(np.float64)[:, None] * (v[t] - np.einsum("hkv,hk->hv", s, k[t]))
        s += k[t][:, :, None] * c[:, None, :]
        out[t] = np.einsum("hkv,hk->hv", s, q[t])
    return out, s


class Delta:
    def __init__(self, rows, k_heads, heads, dk, dv, seed=0, alike=0.5):
        g = np.random.default_rng(seed)
        self.__dict__.update(rows=rows, k_heads=k_heads, heads=heads, dk=dk, dv=dv)

        def unit(x):
            return (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6)).astype(np.float32)

        common = g.standard_normal((k_heads, dk))
        self.k, self.q = unit(g.standard_normal((rows, k_heads, dk)) + alike * common), unit(g.standard_normal((rows, k_heads, dk)))
        self.v = g.standard_normal((rows, heads, dv)).astype(np.float32)
        self.alpha = np.exp(-np.exp(g.uniform(-6, 1, (rows, heads)))).astype(np.float32)
        self.beta = (1 / (1 + np.exp(-g.standard_normal((rows, heads))))).astype(np.float32)
        self.s = (0.3 * g.standard_normal((heads, dk, dv))).astype(np.float32)

    def launch(self, backend, in_place=False, sbase=0, abase=0, want_code=None):
        def based(x, base):
            return backend.upload(np.concatenate([np.full(base, 9.0, np.float32), x.reshape(-1)]))
        s = based(self.s, sbase)
        s_out = s if in_place else backend.upload(np.full(sbase + self.s.size, 9.0, np.float32))
        o = backend.AllocateBuffer(self.v.nbytes)
        run(backend, "delta_chunk_heads", [s, backend.upload(self.k), backend.upload(self.v), backend.upload(self.q), o, based(self.alpha, abase),
                                           based(self.beta, abase), s_out], [self.heads, self.k_heads, self.dk, self.dv, self.rows, sbase, abase])
        state = backend.download(s_out, np.float32, sbase + self.s.size)
        assert np.all(state[:sbase] == 9.0)
        return backend.download(o, np.float32, self.v.size).reshape(self.v.shape), state[sbase:].reshape(self.s.shape)

    def want(self):
        return delta_reference(self.s, self.k, self.v, self.q, self.alpha, self.beta)


def near_whole(y, r, tol=2e-5):
    """Of the largest magnitude.  An operand's two terms are off by 2^-22, a sum over dk by about sqrt(dk) 2^-24 of its terms, and
    with beta |k|^2 <= 1 an error of a row fades over the next: tens of 2^-22."""
    return bool(np.all(np.isfinite(y)) and np.abs(y - r).max() <= tol * np.abs(r).max())


@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 16), (2, 2, 4, 128, 128), (31, 1, 2, 128, 64), (32, 2, 2, 64, 80), (33, 4, 12, 128, 128), (64, 1, 9, 128, 16),
                                   (100, 2, 6, 64, 64), (300, 2, 2, 128, 144)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("in_place", [False, True])
def test_delta_rule_in_chunks(backend, shape, in_place):
    t = Delta(*shape, seed=sum(shape))
    o, s = t.launch(backend, in_place, sbase=48 if in_place else 0, abase=5 if in_place else 0)
    o_want, s_want = t.want()
    assert near_whole(o, o_want) and near_whole(s, s_want)


def test_delta_rule_extremes(backend):
    """Decays of 0 and 1, corrections of 0 and 1, equal keys, keys and values of very different sizes, an empty state."""
    t = Delta(70, 2, 4, 128, 32, seed=40)
    t.alpha[3], t.alpha[40:44], t.beta[10:20], t.beta[50] = 0.0, 1.0, 0.0, 1.0
    t.k[20:30] = t.k[20]
    t.k[45] = 0.0
    t.v *= np.exp2(np.random.default_rng(41).integers(-8, 8, (70, 1, 1))).astype(np.float32)
    t.s[1] = 0.0
    t.s[2] *= 1e-20
    o, s = t.launch(backend)
    o_want, s_want = t.want()
    assert near_whole(o, o_want) and near_whole(s, s_want)


def test_delta_rule_equals_the_row_form(backend):
    t = Delta(77, 4, 8, 128, 128, seed=42)
    o, s = t.launch(backend)
    k, q = (np.tile(x, (1, 2, 1)) for x in (t.k, t.q))
    state, out = backend.upload(t.s), backend.AllocateBuffer(t.v.nbytes)
    run(backend, "delta_step_heads", [state, backend.upload(k), backend.upload(t.v), backend.upload(q), out, backend.upload(t.alpha), backend.upload(t.beta)],
        [8, 128, 128, 77, 0, 0, 0])
    assert near_whole(o, backend.download(out, np.float32, o.size).reshape(o.shape).astype(np.float64))
    assert near_whole(s, backend.download(state, np.float32, s.size).reshape(s.shape).astype(np.float64))


def test_delta_rule_of_a_long_prompt(backend):
    """More rows than one pair of launches takes."""
    t = Delta(4096 + 70, 1, 1, 64, 16, seed=43)
    o, s = t.launch(backend)
    o_want, s_want = t.want()
    assert near_whole(o, o_want) and near_whole(s, s_want)


# ------------------------------------------------------------------ log probabilities

def logprob_reference(x, targets, top_k):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        y = x - np.where(np.isfinite(top), top, 0.0)
        e = np.exp(y)
        total = e.sum(1, keepdims=True)
        logp = y - np.log(total)
        entropy = np.log(total)[:, 0] - np.where(e > 0, e * y, 0.0).sum(1) / total[:, 0]
    entropy[total[:, 0] == 0] = 0.0
    logp[total[:, 0] == 0] = -np.inf
    order = np.argsort(-(x + 0.0), 1, kind="stable")[:, :top_k]
    given = np.array([logp[r, t] if t < x.shape[1] else -np.inf for r, t in enumerate(targets)])
    return given, entropy, order, np.take_along_axis(logp, order, 1)


def launch_logprob(backend, x, targets, top_k, row_base=0):
    rows, vocab = x.shape[0] - row_base, x.shape[1]
    bufs = [backend.AllocateBuffer(max(4, n * 4)) for n in (rows, rows, rows * top_k, rows * top_k)]
    run(backend, "logprob_rows", [backend.upload(x), backend.upload(targets), *bufs], [rows, vocab, top_k, row_base])
    given, entropy = (backend.download(b, np.float32, rows) for b in bufs[:2])
    if top_k == 0:
        return given, entropy, None, None
    return given, entropy, backend.download(bufs[2], np.uint32, rows * top_k).reshape(rows, top_k), backend.download(bufs[3], np.float32, rows * top_k).reshape(rows, top_k)


def check_logprob(backend, x, targets, top_k, row_base=0):
    y = launch_logprob(backend, x, targets, top_k, row_base)
    x = x[row_base:]
    r = logprob_reference(x, targets, top_k)
    # sums of up to vocab / 512 exponentials a thread and of the threads, each off by an argument's rounding (2^-24 of x - max)
    # and two units of its own; the difference x - max, the logarithm and the last difference
    far = np.ptp(np.where(np.isfinite(x) & (np.abs(x) < 1e30), x, 0.0), axis=1)
    tol = U * (x.shape[1] / 512 + 64 + 6 * far)

    def near(a, b, t):
        fine = np.isfinite(b)
        return np.array_equal(a[~fine], b[~fine].astype(np.float32), equal_nan=True) and np.all(np.abs(a[fine] - b[fine]) <= np.broadcast_to(t, b.shape)[fine] + 2 * U * np.abs(b[fine]))

    assert near(y[0], r[0], tol)
    assert near(y[1], r[1], tol * (2 + far))
    if top_k:
        assert np.array_equal(y[2], r[2])
        assert near(y[3], r[3], tol[:, None])


@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (1, 5, 3), (3, 32, 32), (2, 33, 1), (1, 1000, 20), (5, 4099, 7), (2, 8192, 32), (1, 8193, 5), (7, 20001, 32),
                                              (1, 151936, 20), (40, 30000, 0), (300, 5000, 4), (3, 151937, 32)])
def test_logprob_rows(backend, rows, vocab, top_k):
    g = np.random.default_rng(rows + vocab)
    base = rows % 2
    x = (3 * g.standard_normal((base + rows, vocab))).astype(np.float32)
    check_logprob(backend, x, g.integers(0, vocab, rows).astype(np.uint32), top_k, base)


@pytest.mark.parametrize("vocab", [50, 9000, 40001, 151936])
@pytest.mark.parametrize("what", ["equal", "rising", "falling", "steps", "signed zeros", "few left", "one left", "lowest", "far apart"])
def test_logprob_of_rows_that_are_not_random(backend, what, vocab):
    g = np.random.default_rng(vocab)
    x = g.standard_normal((2, vocab)).astype(np.float32)
    if what == "equal":
        x[:] = 1.5
    elif what == "rising":
        x[:] = np.linspace(-5, 5, vocab, dtype=np.float32)
    elif what == "falling":
        x[:] = np.linspace(5, -5, vocab, dtype=np.float32)
    elif what == "steps":
        x = np.round(x * 2) / 2
    elif what == "signed zeros":
        x = np.where(g.random(x.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
    elif what == "few left":  # fewer than top_k
        keep = g.permutation(vocab)[:6]
        y = np.full_like(x, -np.inf)
        y[:, keep] = x[:, keep]
        x = y
    elif what == "one left":
        x[0], x[1] = -np.inf, -np.inf
        x[0, vocab - 1] = 3.0
    elif what == "lowest":  # masked by the type's lowest value
        x = np.where(g.random(x.shape) < 0.9, np.finfo(np.float32).min, x)
        x[1] = np.finfo(np.float32).min
    else:
        x *= 1e4
    check_logprob(backend, x, np.array([vocab - 1, vocab], np.uint32), 10)


def test_logprob_of_rows_with_nan_and_infinity(backend):
    x = np.random.default_rng(1).standard_normal((3, 3000)).astype(np.float32)
    x[0, 7], x[1, 2999] = np.nan, np.inf
    given, entropy, ids, tops = launch_logprob(backend, x, np.array([1, 2, 3], np.uint32), 4)
    assert np.isnan(given[:2]).all() and np.isnan(entropy[:2]).all() and np.isnan(tops[:2]).all()
    assert ids[1, 0] == 2999 and np.array_equal(ids[0], np.argsort(-np.where(np.isnan(x[0]), -np.inf, x[0]), kind="stable")[:4])
    assert np.isfinite(given[2]) and np.isfinite(tops[2]).all()


def test_logprob_agrees_with_top_k_rows(backend):
    x = np.random.default_rng(2).standard_normal((4, 5001)).astype(np.float32)
    buf, ids, vals = backend.upload(x), backend.AllocateBuffer(4 * 8 * 4), backend.AllocateBuffer(4 * 8 * 4)
    run(backend, "top_k_rows", [buf, ids, vals], [4, 5001, 8, 0])
    assert np.array_equal(launch_logprob(backend, x, np.zeros(4, np.uint32), 8)[2], backend.download(ids, np.uint32, 32).reshape(4, 8))


# ------------------------------------------------------------------ refusals

def test_refusals(backend):
    buf, other = backend.AllocateBuffer(1 << 20), [backend.AllocateBuffer(1 << 20) for _ in range(12)]
    bad, not_served = capi.StatusCode.InvalidArgument, capi.StatusCode.UnsupportedFeature
    th, e = bits(1e6), bits(1e-6)
    norm = [2, 4, 2, 64, 32, th, 6, 5, 5, e]
    cases = [
        ("attention_tree", other[:5], [4, 16, 4, 2, 64, 0, 0, 0], not_served),
        ("attention_tree", other[:5], [257, 16, 4, 2, 128, 0, 0, 0], not_served),
        ("attention_tree", other[:5], [4, 16, 18, 2, 128, 0, 0, 0], not_served),
        ("attention_tree", other[:5], [0, 16, 4, 2, 128, 0, 0, 0], bad),
        ("attention_tree", other[:5], [4, 16, 5, 2, 128, 0, 0, 0], bad),
        ("attention_tree", other[:5], [4, 1 << 20, 4, 2, 128, 0, 0, 0], bad),
        ("attention_tree", other[:4], [4, 16, 4, 2, 128, 0, 0, 0], bad),
        ("attention_tree_q8", other[:7], [4, 8190, 4, 1, 128, 0, 0], bad),
        ("qk_norm_rope", other[:7], [2, 4, 2, 258, 32, th, 6, 5, 5, e], not_served),
        ("qk_norm_rope", other[:7], [2, 4, 2, 64, 66, th, 6, 5, 5, e], bad),
        ("qk_norm_rope", other[:7], [2, 4, 2, 64, 32, th, 6, 6, 5, e], bad),
        ("qk_norm_rope", other[:7], [2, 4, 2, 64, 32, bits(-1.0), 6, 5, 5, e], bad),
        ("qk_norm_rope", other[:7], [2, 4, 2, 64, 32, th, 6, 5, 5, bits(-1.0)], bad),
        ("qk_norm_rope", other[:7], [0] + norm[1:], bad),
        ("qk_norm_rope", [buf, other[0], other[1], other[2], other[3], other[0], other[4]], norm, bad),   # queries over keys
        ("qk_norm_rope_append", [*other[:7], buf, buf], norm + [0, 0], bad),                              # k and v rows alike
        ("qk_norm_rope_append", other[:9], norm + [2047, 0], bad),
        ("qk_norm_rope_append_q4", other[:11], [2, 4, 1, 34, 32, th, 6, 5, 5, e, 0], bad),
        ("qk_norm_rope_append_q8", other[:11], [1, 4, 40, 256, 32, th, 6, 5, 5, e, 0], not_served),
        ("delta_chunk_heads", other[:8], [4, 2, 96, 64, 5, 0, 0], not_served),
        ("delta_chunk_heads", other[:8], [4, 2, 64, 24, 5, 0, 0], not_served),
        ("delta_chunk_heads", other[:8], [4, 3, 64, 32, 5, 0, 0], bad),
        ("delta_chunk_heads", other[:8], [4, 2, 64, 32, 0, 0, 0], bad),
        ("delta_chunk_heads", other[:8], [4, 2, 64, 32, 5, 1 << 18, 0], bad),
        ("delta_chunk_heads", [*other[:4], buf, *other[4:6], buf], [4, 2, 64, 32, 5, 0, 0], bad),         # outputs over the state
        ("logprob_rows", other[:6], [1, 100, 33, 0], bad),
        ("logprob_rows", other[:6], [0, 100, 3, 0], bad),
        ("logprob_rows", other[:6], [3, 100000, 3, 0], bad),
    ]
    for deferred in (0, 1):
        backend.SetDeferred(deferred)
        try:
            for name, buffers, scalars, code in cases:
                with pytest.raises(capi.StatusError) as err:
                    run(backend, name, buffers, scalars)
                assert err.value.code == code, (name, scalars)
        finally:
            backend.SetDeferred(0)
    backend.Synchronize()
