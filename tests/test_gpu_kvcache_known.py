"""The attention over paged caches by every schedule, type and width, on inputs whose results are known (kv_known.py): a key that is lost
or taken twice, in whatever wave, share or join, is in plain sight."""
import math

import pytest
import torch

import kv_known as K
from test_gpu_kvcache_exact import cache_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = K.shapes()


def attended(s, k, v, q):
    """The shape's call over one set of pages that all of its sequences share: results, logarithms, lengths."""
    cache, row = cache_of(k, v, s.page, s.dtype)
    table = torch.full((len(s.lengths), s.columns), -7, dtype=torch.int32, device=DEV)
    table[:, :row.shape[1]] = row
    lens = torch.tensor(s.lengths, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q.to(DEV), table, lens, scale=1.0, return_lse=True)
    again, lse2 = cache.attend(q.to(DEV), table, lens, scale=1.0, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "two calls differ"
    cache.check()
    return out.cpu(), lse.cpu()


@pytest.mark.parametrize("s", SHAPES, ids=repr)
def test_counts(s):
    """All scores zero: each result a count of keys over the length, exactly."""
    n = max(s.lengths)
    v = K.counting_values(n, s.heads, s.width)
    q = torch.randn((len(s.lengths), s.heads * s.group, s.width), generator=torch.Generator().manual_seed(n)).to(s.q_dtype)
    out, lse = attended(s, torch.zeros_like(v), v, q)
    for b, length in enumerate(s.lengths):
        if length == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        want, total = K.counted(v, length, s.q_dtype)
        assert torch.equal(out[b].reshape(s.heads, s.group, s.width), want[:, None].expand(-1, s.group, -1)), (b, length)
        # the logarithm of a whole number, a step or two of 2^-24 off: one key more or less is a 40000th
        assert float((lse[b].double() - math.log(length)).abs().max()) <= 2.0 ** -22 * max(1.0, math.log(length)), (b, length)


@pytest.mark.parametrize("s", SHAPES, ids=repr)
def test_peaks(s):
    """One key of every 32 scores 20 with the queries of its column: each of them, in each query's row, where it belongs."""
    n = max(s.lengths)
    k, v, at = K.peaked(n, s.heads, s.width, s.dtype)
    q, columns = K.peak_queries(len(s.lengths), s.heads, s.group, s.width, s.q_dtype)
    out, lse = attended(s, k, v, q)
    worst = 0.0
    for b, length in enumerate(s.lengths):
        if length:
            want, allowed = K.peak_results(v, at, length, columns[b], s.q_dtype, s.depth())
            got = out[b].double().reshape(s.heads, s.group, s.width)
            worst = max(worst, float(((got - want).abs() / allowed).max()))
            total = torch.where(at[:length, None] == columns[b][None], math.exp(K.PEAK), 1.0).double().sum(0).log()
            assert float((lse[b].double().reshape(s.heads, s.group) - total).abs().max()) <= 2.0 ** -24 * (2 * (1.5 * (K.PEAK + 8) + 16) + s.depth() + 4 * 31)
    assert worst <= 1.0, worst
