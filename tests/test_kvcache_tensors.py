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


def test_tensors_without_memory_are_refused():
    zero = torch._efficientzerotensor((3, 2, 64), dtype=torch.float16)
    with pytest.raises(WtError, match="memory"):
        host_cache().append(zero, ROWS, TABLE, POS)
    freed = pages(3, 2, 64)
    freed.untyped_storage().resize_(0)
    for f in (lambda: host_cache().append(freed, ROWS, TABLE, POS), lambda: host_cache().gather(TABLE, POS, out=(freed, ROWS))):
        with pytest.raises(WtError, match="memory"):
            f()
    cut = i32(*range(64))[:3]
    cut.untyped_storage().resize_(8)
    with pytest.raises(WtError, match="positions: not all of it has memory"):
        host_cache().append(ROWS, ROWS, TABLE, cut)
    short = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    short.untyped_storage().resize_(1000)
    with pytest.raises(WtError, match="memory"):
        PagedKVCache(short, pages(4, 2, 16, 64))


@pytest.mark.parametrize("which", range(4))
def test_a_cache_whose_memory_was_resized(which):
    """The cache holds its memory, but cannot keep it from being resized: its calls are refused then."""
    from whisper_timestamped import kvcache
    from test_kvcache_host import E4M3
    parts = [pages(4, 2, 16, 64, dtype=E4M3) for _ in range(2)] + [pages(4, 2, 16, dtype=torch.uint8) for _ in range(2)]
    cache = object.__new__(PagedKVCache)
    cache._calls = kvcache._calls()
    cache._handle, cache.error = cache._calls.make(*parts, True)
    with pytest.raises(WtError, match="only run on the GPU"):
        cache.append(ROWS, ROWS, TABLE, POS)
    parts[which].untyped_storage().resize_(64)
    for f in (lambda: cache.append(ROWS, ROWS, TABLE, POS), lambda: cache.gather(TABLE, POS), lambda: cache.attend(Q, TABLE, POS),
              lambda: cache.attend_workspace(4, TABLE)):
        with pytest.raises(WtError, match="resized"):
            f()
