"""Tensors that are more, or something else, than their memory says: refused rather than read as plain ones; and what the calls write is
known to autograd."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_kvcache_host import ROWS, Q, TABLE, host_cache, i32, pages
from whisper_timestamped import PagedKVCache
from whisper_timestamped._lib import WtError

POS = i32(0, 1, 2)


def calls(x, q):
    """One call for each place where x (rows) or q (queries) may stand, on a cache that takes plain tensors."""
    c = host_cache()
    return [lambda: c.append(x, ROWS, TABLE, POS), lambda: c.append(ROWS, x, TABLE, POS), lambda: c.gather(TABLE, POS, out=(x, pages(3, 2, 64))),
            lambda: c.gather(TABLE, POS, out=(pages(3, 2, 64), x)), lambda: c.attend(q, TABLE, POS), lambda: c.attend(Q, TABLE, POS, out=q)]


def test_forward_mode_tangents_are_refused():
    """A dual tensor's tangent would be dropped."""
    with fwd.dual_level():
        x, q = fwd.make_dual(pages(3, 2, 64), pages(3, 2, 64)), fwd.make_dual(pages(3, 4, 64), pages(3, 4, 64))
        for f in calls(x, q):
            with pytest.raises(WtError, match="tangent"):
                f()
        with pytest.raises(WtError, match="tangent"):
            PagedKVCache(fwd.make_dual(pages(4, 2, 16, 64), pages(4, 2, 16, 64)), pages(4, 2, 16, 64))


def negated(*shape):
    """A view whose values are the negatives of its memory."""
    t = torch._neg_view(pages(*shape))
    assert t.is_neg()
    return t


def test_lazily_negated_tensors_are_refused():
    for f in calls(negated(3, 2, 64), negated(3, 4, 64)):
        with pytest.raises(WtError, match="negated"):
            f()
    with pytest.raises(WtError, match="negated"):
        PagedKVCache(negated(4, 2, 16, 64), pages(4, 2, 16, 64))
