"""The operators of a step over many rows (a prompt's chunk, a tree of drafted tokens), each in its plain form and as the
library's call.

Where `own` is false, `run` computes the operator with elementary torch operations; where it is true, it calls the typed
launchers of the C ABI on torch's current stream, as a host that keeps its own buffers does.  `exact` gives the same from
the definition in 64 bits.  Shapes are those of `tessera_b200.workload` and of `perf/cases.py` (24 query heads over 4 kv
heads of 256, 16 key heads and 48 value heads of 128, a vocabulary of 151936) and of other grouped layouts.

Operators (`case["op"]`):
  tree     attention of the rows of a drafted tree over the key / value cache: the past, the row's ancestors, itself
  norm     per-head norms of queries and keys, their rotation to each row's position, the k and v rows into the cache
  delta    the gated delta rule over many rows, from a given state to a new one
  logprob  log probabilities of given tokens, the rows' entropy and their likeliest tokens
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
THETA, SECTIONS = 1e7, (11, 11, 10)
KV_CODE = {"f32": 0, "f16": 1, "q8": 2, "q4": 3, "fp8": 4}
KV_BYTES = {"f32": 4.0, "f16": 2.0, "q8": 1.0, "q4": 0.5, "fp8": 1.0}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # sixteen drafted tokens behind a short conversation: the smallest verification, where latency counts
        dict(name="tree_small", op="tree", kv="fp8", m=16, n=512, heads=24, kv_heads=4, head_dim=256, window=0, shape="bushy"),
        # a wide tree over a binary16 cache of another layout, some rows of a fixed-size tree unused
        dict(name="tree_f16", op="tree", kv="f16", m=61, n=4000, heads=16, kv_heads=2, head_dim=128, window=0, shape="padded"),
        # eight rows over the fp32 cache the engine starts with
        dict(name="tree_f32", op="tree", kv="f32", m=8, n=4096, heads=24, kv_heads=4, head_dim=256, window=0, shape="bushy"),
        # a large tree far into a long conversation
        dict(name="tree_long", op="tree", kv="fp8", m=64, n=32768, heads=24, kv_heads=4, head_dim=256, window=0, shape="bushy"),
        # the norms, rotation and cache append of a verification and of a prompt's chunk
        dict(name="norm_verify", op="norm", kv="fp8", rows=16, first=4096, heads=24, kv_heads=4, head_dim=256, rope_dim=64),
        dict(name="norm_prefill", op="norm", kv="f16", rows=512, first=0, heads=24, kv_heads=4, head_dim=256, rope_dim=64),
        # linear attention of a chain of drafted tokens, of a prompt's chunk, of a long prompt at once
        dict(name="delta_verify", op="delta", rows=33, k_heads=16, heads=48, dk=128, dv=128),
        dict(name="delta_prefill", op="delta", rows=512, k_heads=16, heads=48, dk=128, dv=128),
        dict(name="delta_long", op="delta", rows=2048, k_heads=16, heads=32, dk=128, dv=128),
        # the likeliest twenty of a decoded token, a verified tree's rows, a scored prompt under a grammar's mask
        dict(name="logprob_token", op="logprob", rows=1, vocab=151936, top_k=20, masked=False),
        dict(name="logprob_verify", op="logprob", rows=16, vocab=151936, top_k=8, masked=False),
        dict(name="logprob_prompt", op="logprob", rows=256, vocab=151936, top_k=20, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "norm", "delta", "logprob"])
    if op == "tree":
        head_dim, kv_heads, group = rng.choice([128, 256]), rng.choice([1, 2, 4, 8]), rng.randint(1, 8)
        while kv_heads * group > 32:
            kv_heads //= 2
        heads, m = kv_heads * group, _log(rng, 1, 256)
        most = int(64 * 32768 * 24 * 256 / (m * heads * head_dim))
        n = _log(rng, 1, max(1, min(32768, most) - m))
        return dict(op=op, kv=rng.choice(list(KV_CODE)), m=m, n=n, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    window=rng.choice([0, 0, 0, max(1, n // 3)]), shape=rng.choice(["bushy", "chain", "padded"]))
    if op == "norm":
        head_dim, kv_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8])
        return dict(op=op, kv=rng.choice(["f32", "f16", "fp8"]), rows=_log(rng, 1, 512), first=rng.randint(0, 4096), heads=kv_heads * rng.randint(1, 6),
                    kv_heads=kv_heads, head_dim=head_dim, rope_dim=rng.choice([64, head_dim]))
    if op == "delta":
        k_heads = rng.choice([4, 8, 16])
        return dict(op=op, rows=_log(rng, 1, 1024), k_heads=k_heads, heads=k_heads * rng.randint(1, 3), dk=128, dv=rng.choice([64, 128]))
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 151936), top_k=rng.randint(1, 32), masked=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

class Random:
    """Seeded tensors on the GPU, one generator for a case."""

    def __init__(self, seed):
        self.seed = int(seed)
        self.g = torch.Generator(device="cuda").manual_seed(self.seed * 7919 + 29)

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.g)

    def uniform(self, lo, hi, *shape):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=self.g)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=self.g)

    def cache(self, kv, rows, cols):
        """(rows of a cache in its format, their scales) for normal values."""
        x = self.normal(rows, cols)
        if kv in ("f32", "f16"):
            return x.half() if kv == "f16" else x, None
        scale = x.abs().amax(1) / {"q8": 127.0, "q4": 7.0, "fp8": 448.0}[kv]
        y = x / scale[:, None]
        if kv == "fp8":
            return y.to(torch.float8_e4m3fn).view(torch.uint8), scale
        c = y.round().to(torch.int8).view(torch.uint8)
        return (c if kv == "q8" else (c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4)).contiguous(), scale


def _parents(case, seed):
    """A drafted tree: -1 for a child of the last past row, -2 for a row that is not used."""
    m, g = case["m"], np.random.default_rng(seed)
    p = np.arange(m) - 1
    if case["shape"] != "chain":  # most rows hang from one of the rows just drafted
        p = np.maximum(p - g.integers(0, 1 + np.minimum(np.arange(m), 7)), -1)
    if case["shape"] == "padded":
        p[m - m // 8:] = -2
    return p.astype(np.int32)


def prepare(case, seed):
    r = Random(seed)
    s = dict(_INPUTS[case["op"]](case, r), case=case)
    s["pointers"] = {name: t.data_ptr() for name, t in s.items() if isinstance(t, torch.Tensor)}
    s["stream"] = torch.cuda.current_stream().cuda_stream
    return s


def _tree_inputs(c, r):
    rows, cols = c["n"] + c["m"], c["kv_heads"] * c["head_dim"]
    s = dict(q=1.5 * r.normal(c["m"], c["heads"], c["head_dim"]), parents=torch.from_numpy(_parents(c, r.seed)).cuda(),
             out=torch.empty(c["m"], c["heads"], c["head_dim"], device="cuda"))
    for name in ("k", "v"):
        s[name], s[name + "_scale"] = r.cache(c["kv"], rows, cols)
    return s


def _norm_inputs(c, r):
    rows, d, kv = c["rows"], c["head_dim"], c["kv"]
    cols = c["kv_heads"] * d
    s = dict(q=r.normal(rows, c["heads"], d), k=r.normal(rows, c["kv_heads"], d), v=r.normal(rows, c["kv_heads"], d),
             q_w=1.0 + 0.1 * r.normal(d), k_w=1.0 + 0.1 * r.normal(d), q_out=torch.empty(rows, c["heads"], d, device="cuda"))
    t = int(r.ints(0, 100000, 1)) + torch.arange(rows, device="cuda")
    s["pos"] = torch.stack([t, t + r.ints(0, 8, rows), t + r.ints(0, 8, rows)], 1).contiguous()
    s["axis"] = torch.tensor([i for i, pairs in enumerate(_sections(c)) for _ in range(pairs)], device="cuda")  # of each pair
    kind = {"f32": torch.float32, "f16": torch.float16, "fp8": torch.float8_e4m3fn}[kv]
    for name in ("k", "v"):
        s[name + "_cache"] = torch.zeros(c["first"] + rows, cols, device="cuda").to(kind)
        s[name + "_scale"] = torch.zeros(c["first"] + rows, device="cuda") if kv == "fp8" else None
    return s


def _delta_inputs(c, r):
    rows, kh, h, dk, dv = c["rows"], c["k_heads"], c["heads"], c["dk"], c["dv"]

    def unit(x):
        return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)

    common = r.normal(kh, dk)  # keys of a head resemble one another
    return dict(s=0.3 * r.normal(h, dk, dv), k=unit(r.normal(rows, kh, dk) + 0.5 * common), q=unit(r.normal(rows, kh, dk)) / math.sqrt(dk),
                v=r.normal(rows, h, dv), alpha=torch.exp(-torch.exp(r.uniform(-6.0, 0.0, rows, h))), beta=torch.sigmoid(r.normal(rows, h)),
                o=torch.empty(rows, h, dv, device="cuda"), s_out=torch.empty(h, dk, dv, device="cuda"))


def _logprob_inputs(c, r):
    rows, vocab, k = c["rows"], c["vocab"], c["top_k"]
    logits = 2.5 * r.normal(rows, vocab)
    top = logits.argmax(1)
    targets = torch.where(r.ints(0, 2, rows) == 0, top, r.ints(0, vocab, rows)).to(torch.int32)
    if c["masked"]:  # tokens that a grammar does not allow
        logits = logits.masked_fill(r.ints(0, 2, rows, vocab) == 0, -math.inf)
    return dict(logits=logits, targets=targets, logprob=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                top_ids=torch.empty(rows, k, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(rows, k, device="cuda"))


_INPUTS = dict(tree=_tree_inputs, norm=_norm_inputs, delta=_delta_inputs, logprob=_logprob_inputs)


# ------------------------------------------------------------------ a pass

def run(state):
    if own:
        _CALL[state["case"]["op"]](_library(), state["case"], state, state["pointers"], state["stream"])
        return _OUTPUTS[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state["case"], state)


def exact(case, seed):
    return _EXACT[case["op"]](case, _INPUTS[case["op"]](case, Random(seed)))


def work(case):
    return _WORK[case["op"]](case)


_LIBRARY = None


def _library():
    global _LIBRARY
    if _LIBRARY is None:
        from tessera_b200 import capi
        _LIBRARY = capi.load_library()
    return _LIBRARY


def _ok(status):
    if status != 0:
        raise RuntimeError("status %d" % status)


# ------------------------------------------------------------------ tree

def _call_tree(lib, c, s, p, stream):
    _ok(lib.tsr_attention_tree(KV_CODE[c["kv"]], p["q"], p["k"], p["v"], p.get("k_scale"), p.get("v_scale"), p["parents"], p["out"],
                               c["m"], c["n"], c["heads"], c["kv_heads"], c["head_dim"], 0, c["window"], stream))


def _values(kv, x, scale, dtype):
    """The values a cache stands for."""
    if kv in ("f32", "f16"):
        return x.to(dtype)
    if kv == "fp8":
        x = x.view(torch.float8_e4m3fn)
    elif kv == "q8":
        x = x.view(torch.int8)
    else:
        x = torch.stack([(x << 4).view(torch.int8) >> 4, x.view(torch.int8) >> 4], 2).flatten(1)
    return x.to(dtype) * scale.to(dtype)[:, None]


def _plain_tree(c, s):
    m, n, kvh, d = c["m"], c["n"], c["kv_heads"], c["head_dim"]
    group = c["heads"] // kvh
    parents, rows = s["parents"], torch.arange(m, device="cuda")
    used = (parents >= -1) & (parents < rows)
    # ancestors: the closure of "is the parent of", by squaring; a row below one that is not used is not used either
    reach = ((parents[:, None] == rows) & used[:, None]) | (rows[:, None] == rows)
    for _ in range(m.bit_length()):
        reach = (reach.float() @ reach.float()) > 0
    used = ~(reach & ~used).any(1)
    depth = reach.sum(1)  # rows of its path, itself included
    see = torch.cat([torch.ones(m, n, dtype=torch.bool, device="cuda"), reach], 1) & used[:, None]
    if c["window"]:
        behind = torch.cat([depth[:, None] + (n - 1 - torch.arange(n, device="cuda")), depth[:, None] - depth], 1)
        see &= behind < c["window"]
    k, v = (_values(c["kv"], s[x], s[x + "_scale"], torch.float32).view(n + m, kvh, d).transpose(0, 1) for x in ("k", "v"))
    q = s["q"].view(m, kvh, group, d).permute(1, 2, 0, 3).reshape(kvh, group * m, d)
    scores = (q @ k.transpose(1, 2) / math.sqrt(d)).view(kvh, group, m, n + m).masked_fill_(~see, -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp_min(-3e38)
    w = scores.exp_()
    total = w.sum(-1, keepdim=True)
    out = (w.view(kvh, group * m, n + m) @ v).view(kvh, group, m, d) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(2, 0, 1, 3).reshape(m, c["heads"], d)


def _exact_tree(c, s):
    m, n, kvh, d, window = c["m"], c["n"], c["kv_heads"], c["head_dim"], c["window"]
    group, parents = c["heads"] // kvh, s["parents"].tolist()
    k, v = (_values(c["kv"], s[x], s[x + "_scale"], torch.float64).view(n + m, kvh, d).permute(1, 2, 0).contiguous() for x in ("k", "v"))
    out = torch.zeros(m, c["heads"], d, dtype=torch.float64, device="cuda")
    for i in range(m):
        path, at = [], i
        while 0 <= at and -1 <= parents[at] < at:
            path.append(at)
            at = parents[at]
        if at != -1:  # the row, or one above it, is not used
            continue
        path = path[:window] if window else path
        past = min(n, window - len(path)) if window else n
        keys = torch.tensor(path, device="cuda") + n
        ki, vi = (torch.cat([x[:, :, n - past:n], x[:, :, keys]], 2) for x in (k, v))
        scores = torch.einsum("kgd,kdn->kgn", s["q"][i].double().view(kvh, group, d), ki) / math.sqrt(d)
        out[i] = torch.einsum("kgn,kdn->kgd", torch.softmax(scores, -1), vi).reshape(c["heads"], d)
    return out


def _work_tree(c):
    rows, cols = c["n"] + c["m"], c["kv_heads"] * c["head_dim"]
    seen = min(rows, c["window"] + c["m"]) if c["window"] else rows
    scales = 8.0 * seen if c["kv"] in ("q8", "q4", "fp8") else 0.0
    pairs = c["m"] * c["heads"]
    return dict(bytes=2.0 * KV_BYTES[c["kv"]] * seen * cols + scales + 8.0 * pairs * c["head_dim"] + 4.0 * c["m"],
                flops=4.0 * pairs * c["head_dim"] * min(c["n"] + 1, c["window"] or c["n"] + 1))


# ------------------------------------------------------------------ norm

def _call_norm(lib, c, s, p, stream):
    _ok(lib.tsr_qk_norm_rope_append(KV_CODE[c["kv"]], p["q"], p["k"], p["v"], p["q_w"], p["k_w"], p["pos"], p["q_out"], p["k_cache"], p["v_cache"],
                                    p.get("k_scale"), p.get("v_scale"), c["rows"], c["first"], c["heads"], c["kv_heads"], c["head_dim"],
                                    c["rope_dim"], THETA, *_sections(c), EPS, stream))


def _sections(c):
    """Pairs that turn with a row's time, height and width."""
    pairs = c["rope_dim"] // 2
    t, h = pairs * SECTIONS[0] // sum(SECTIONS), pairs * SECTIONS[1] // sum(SECTIONS)
    return t, h, pairs - t - h


def _plain_norm(c, s):
    pairs, first = c["rope_dim"] // 2, c["first"]
    freq = torch.exp(torch.arange(pairs, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / c["rope_dim"]))
    angle = s["pos"].double()[:, s["axis"]] * freq  # 64 bits: positions go far
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., 2 * pairs:]], -1)

    out = [turned(s["q"], s["q_w"])]
    for name, x in (("k", turned(s["k"], s["k_w"])), ("v", s["v"])):
        x, cache, scale = x.flatten(1), s[name + "_cache"], s[name + "_scale"]
        if scale is not None:
            unit = (x.abs().amax(1) / torch.full_like(x[:, 0], 448.0)).clamp_min(1.0 / (448.0 * 512.0))
            scale[first:] = unit
            x = (x / unit[:, None]).clamp(-448.0, 448.0)
        cache[first:] = x.to(cache.dtype)
        out += [cache, scale]
    return [x for x in out if x is not None]


def _norm_outputs(s):
    return [s[x] for x in ("q_out", "k_cache", "k_scale", "v_cache", "v_scale") if s[x] is not None]


def _exact_norm(c, s):
    rows, half, first = c["rows"], c["rope_dim"] // 2, c["first"]
    t, h, _ = _sections(c)
    axis = np.array([0] * t + [1] * h + [2] * (half - t - h))
    angle = s["pos"].cpu().numpy()[:, axis].astype(np.float64) * np.float64(np.float32(THETA)) ** (-np.arange(half) / half)
    turn = torch.polar(torch.ones(rows, 1, half, dtype=torch.float64), torch.from_numpy(angle)[:, None]).cuda()

    def turned(x, w):
        y = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)

    out = [turned(s["q"], s["q_w"])]
    for name, x in (("k", turned(s["k"], s["k_w"]).flatten(1)), ("v", s["v"].double().flatten(1))):
        if c["kv"] == "fp8":
            unit = x.abs().amax(1).div(448.0).clamp_min(1.0 / (448.0 * 512.0))
            blank = torch.zeros(first, dtype=torch.float64, device="cuda")
            out += [torch.cat([blank[:, None].expand(-1, x.shape[1]), x / unit[:, None]]), torch.cat([blank, unit])]
        else:
            out.append(torch.cat([torch.zeros(first, x.shape[1], dtype=torch.float64, device="cuda"), x]))
    return out


def _work_norm(c):
    q, kv = c["rows"] * c["heads"] * c["head_dim"], c["rows"] * c["kv_heads"] * c["head_dim"]
    scales = 8.0 * c["rows"] if c["kv"] == "fp8" else 0.0
    return dict(bytes=8.0 * q + 8.0 * kv + 2.0 * KV_BYTES[c["kv"]] * kv + scales + 24.0 * c["rows"] + 8.0 * c["head_dim"], flops=8.0 * (q + kv))


# ------------------------------------------------------------------ delta

def _call_delta(lib, c, s, p, stream):
    _ok(lib.tsr_delta_chunk_heads(p["s"], p["k"], p["v"], p["q"], p["o"], p["alpha"], p["beta"], p["s_out"], c["heads"], c["k_heads"], c["dk"], c["dv"],
                                  c["rows"], 0, 0, stream))


def _plain_delta(c, s):
    """The rule itself, row by row; value head h reads key head h % k_heads."""
    state, factor, out = s["s"], c["heads"] // c["k_heads"], []
    k, q = s["k"].repeat(1, factor, 1), s["q"].repeat(1, factor, 1)
    for kt, qt, vt, at, bt in zip(k[..., None], q[..., None], s["v"], s["alpha"][..., None], s["beta"][..., None]):
        state = state * at[..., None]
        state = state + kt * (bt * (vt - (state * kt).sum(1)))[:, None]
        out.append((state * qt).sum(1))
    return torch.stack(out), state


def _exact_delta(c, s):
    """All rows at once: the system that the corrections of the rows solve, heads in turn."""
    rows, kh = c["rows"], c["k_heads"]
    out, states = [], []
    g = torch.cumsum(torch.log(s["alpha"].double()), 0)
    eye = torch.eye(rows, dtype=torch.float64, device="cuda")
    for h in range(c["heads"]):
        k, q, v = s["k"][:, h % kh].double(), s["q"][:, h % kh].double(), s["v"][:, h].double()
        s0, b, gh = s["s"][h].double(), s["beta"][:, h].double()[:, None], g[:, h]
        ratio = torch.tril(torch.exp(torch.tril(gh[:, None] - gh)))
        u = torch.linalg.solve_triangular(eye + b * torch.tril(k @ k.t() * ratio, -1), b * (v - torch.exp(gh)[:, None] * (k @ s0)),
                                          upper=False, unitriangular=True)
        out.append(torch.exp(gh)[:, None] * (q @ s0) + (q @ k.t() * ratio) @ u)
        states.append(torch.exp(gh[-1]) * s0 + (k * ratio[-1][:, None]).t() @ u)
    return torch.stack(out, 1), torch.stack(states)


def _work_delta(c):
    rows, state = c["rows"], c["heads"] * c["dk"] * c["dv"]
    return dict(bytes=4.0 * (2 * rows * c["k_heads"] * c["dk"] + 2 * rows * c["heads"] * c["dv"] + 2 * rows * c["heads"] + 2 * state),
                flops=7.0 * rows * state)


# ------------------------------------------------------------------ logprob

def _call_logprob(lib, c, s, p, stream):
    _ok(lib.tsr_logprob_rows(p["logits"], p["targets"], p["logprob"], p["entropy"], p["top_ids"], p["top_logprobs"], c["rows"], c["vocab"], c["top_k"],
                             0, stream))


def _plain_logprob(c, s):
    x = s["logits"]
    y = x - x.amax(1, keepdim=True)
    e = y.exp()
    total = e.sum(1, keepdim=True)
    logp = y - total.log()
    entropy = total.log()[:, 0] - (e * y.clamp_min(-3e38)).sum(1) / total[:, 0]
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c["top_k"]]  # stable: of equal logits the lowest index first
    given = torch.gather(logp, 1, s["targets"].long()[:, None])[:, 0]
    return given, entropy, order.to(torch.int32), torch.gather(logp, 1, order)


def _exact_logprob(c, s):
    given, entropy, ids, tops = [], [], [], []
    for x, t in zip(s["logits"], s["targets"].long()):
        x = x.double()
        z = torch.logsumexp(x, 0)
        some = x[x > -math.inf] - z
        given.append(x[t] - z)
        entropy.append(-(some.exp() * some).sum())
        order = torch.sort(x, descending=True, stable=True)[1][:c["top_k"]]
        ids.append(order)
        tops.append(x[order] - z)
    return torch.stack(given), torch.stack(entropy), torch.stack(ids).to(torch.int32), torch.stack(tops)


def _work_logprob(c):
    n = c["rows"] * c["vocab"]
    return dict(bytes=4.0 * n + c["rows"] * (12.0 + 8.0 * c["top_k"]), flops=5.0 * n)


_CALL = dict(tree=_call_tree, norm=_call_norm, delta=_call_delta, logprob=_call_logprob)
_OUTPUTS = dict(tree=lambda s: s["out"], norm=_norm_outputs, delta=lambda s: (s["o"], s["s_out"]),
                logprob=lambda s: (s["logprob"], s["entropy"], s["top_ids"], s["top_logprobs"]))
_PLAIN = dict(tree=_plain_tree, norm=_plain_norm, delta=_plain_delta, logprob=_plain_logprob)
_EXACT = dict(tree=_exact_tree, norm=_exact_norm, delta=_exact_delta, logprob=_exact_logprob)
_WORK = dict(tree=_work_tree, norm=_work_norm, delta=_work_delta, logprob=_work_logprob)
