"""Launches that start under the end of the one before them: a projection copies its weights ahead of its wait, so what wrote
them has to be over by then, whatever lies between on the stream."""
import numpy as np
import pytest
import torch

from tessera_b200 import capi

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM = 4, 4, 256
COLS = KV_HEADS * DIM


class Append:
    """FP8 rows of keys and values appended to a cache, whose codes and scales are then the weights of a one-row projection."""

    def __init__(self, rows=512, sets=4):
        g = np.random.default_rng(5)
        self.rows = rows
        self.lib = capi.load_library()
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
        self.q = up(g.standard_normal((self.rows, HEADS, DIM)).astype(np.float32))
        self.k, self.v = (up(g.standard_normal((sets, self.rows, COLS)).astype(np.float32)) for _ in range(2))
        self.w = up(np.ones(DIM, np.float32))
        self.pos = up(np.repeat(np.arange(self.rows)[:, None], 3, 1).astype(np.int64))
        self.a = up(g.standard_normal(COLS).astype(np.float32))
        self.logits, self.target = up(g.standard_normal((1, 5000)).astype(np.float32)), up(np.zeros(1, np.int32))
        new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device="cuda")
        self.q_out = new(self.rows, HEADS, DIM)
        self.caches, self.scales = [new(self.rows, COLS, dtype=torch.uint8) for _ in range(2)], [new(self.rows) for _ in range(2)]
        self.found = [new(1), new(1), new(1, 4, dtype=torch.int32), new(1, 4)]

    def append(self, i, st):
        p = lambda x: x.data_ptr()
        return self.lib.tsr_qk_norm_rope_append(4, p(self.q), p(self.k[i]), p(self.v[i]), p(self.w), p(self.w), p(self.pos), p(self.q_out),
                                                *map(p, self.caches), *map(p, self.scales), self.rows, 0, HEADS, KV_HEADS, DIM, 64, 1e6, 11, 11, 10, 1e-6, st)

    def project(self, which, out, st):
        return self.lib.tsr_gemm_fp8(self.a.data_ptr(), self.caches[which].data_ptr(), self.scales[which].data_ptr(), out.data_ptr(), 1, self.rows, COLS, st)

    def logprobs(self, st):
        return self.lib.tsr_logprob_rows(self.logits.data_ptr(), self.target.data_ptr(), *(x.data_ptr() for x in self.found), 1, 5000, 4, 0, st)

    def passes(self, count, which, between, wait, others=()):
        stream, out = torch.cuda.Stream(), torch.zeros(count, self.rows, device="cuda")
        part, total = torch.ones(2, 64, device="cuda"), torch.zeros(64, device="cuda")
        torch.cuda.synchronize()
        for i in range(count):
            assert self.append(i % len(self.k), stream.cuda_stream) == 0
            if wait:
                stream.synchronize()
            if between:
                assert self.logprobs(stream.cuda_stream) == 0
            for other in others:
                assert self.lib.tsr_gemm_vec_reduce(part.data_ptr(), total.data_ptr(), 64, 2, other.cuda_stream) == 0
            assert self.project(which, out[i], stream.cuda_stream) == 0
        torch.cuda.synchronize()
        return out.cpu().numpy()


@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
def test_a_projection_over_rows_just_appended(which):
    t = Append()
    want = t.passes(4, which, False, True)
    assert np.isfinite(want).all() and not np.array_equal(want[0], want[1])
    assert np.array_equal(t.passes(400, which, False, False), np.tile(want, (100, 1)))


@pytest.mark.parametrize("which", [0, 1], ids=["keys", "values"])
def test_a_projection_one_launch_after_the_append(which):
    """The launch between them starts under the append, the projection under the launch between, but not under both."""
    t = Append()
    want = t.passes(4, which, False, True)
    assert np.array_equal(t.passes(400, which, True, False), np.tile(want, (100, 1)))


def test_launches_on_many_other_streams_in_between():
    """More streams than the record has places for: the one that waits there is pushed out of it."""
    t = Append(rows=16384, sets=2)
    want = t.passes(2, 0, False, True)
    others = [torch.cuda.Stream() for _ in range(24)]
    assert np.array_equal(t.passes(40, 0, False, False, others), np.tile(want, (20, 1)))
