"""The paged cache's refusals: what is wrong with a call is said before anything reaches the GPU."""
import ctypes

import pytest
import torch

from whisper_timestamped import PagedKVCache, _lib
from whisper_timestamped._lib import WtError

E4M3 = torch.float8_e4m3fn


def pages(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("k,v,ke,ve,said", [
    (pages(4, 2, 16), pages(4, 2, 16), None, None, "4-dimensional"),
    (pages(4, 2, 16, 64, dtype=torch.float64), pages(4, 2, 16, 64, dtype=torch.float64), None, None, "4-dimensional"),
    (pages(4, 2, 16, 80), pages(4, 2, 16, 80), None, None, "head_dim"),
    (pages(0, 2, 16, 64), pages(0, 2, 16, 64), None, None, "nothing is empty"),
    (pages(4, 2, 64, 16).transpose(2, 3)[..., :32], pages(4, 2, 16, 32), None, None, "contiguous"),
    (pages(4, 2, 16, 65)[..., :64], pages(4, 2, 16, 64), None, None, "16-byte"),
    (pages(4, 2, 16, 72)[..., 1:65], pages(4, 2, 16, 64), None, None, "16-byte"),
    (pages(1, 2, 16, 64).expand(4, 2, 16, 64), pages(4, 2, 16, 64), None, None, "overlap"),
    (pages(4, 2, 16, 64), pages(4, 2, 8, 64), None, None, "differ"),
    (pages(4, 2, 16, 64), pages(4, 2, 16, 64, dtype=torch.bfloat16), None, None, "differ"),
    (pages(4, 2, 16, 64), pages(4, 2, 16, 64), pages(4, 2, 16, dtype=torch.uint8), None, "another has none"),
    (pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3), None, None, "has exponents"),
    (pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 15, dtype=torch.uint8), pages(4, 2, 16, dtype=torch.uint8), "k_exp"),
    (pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, dtype=torch.uint8), pages(4, 2, 16), "v_exp"),
    (pages(4, 2, 16, 64), pages(4, 2, 16, 64), None, None, "GPU"),
])
def test_construction(k, v, ke, ve, said):
    with pytest.raises(WtError, match=said):
        PagedKVCache(k, v, ke, ve)


def test_the_same_memory_twice():
    k = pages(4, 2, 16, 64)
    with pytest.raises(WtError, match="same memory"):
        PagedKVCache(k, k)


# The C entries check on the host before they launch: made-up addresses never reach the device.
A = 1 << 20


def desc(**kw):
    d = dict(k=A, v=2 * A, k_exp=None, v_exp=None, k_page_stride=2048, k_head_stride=1024, k_slot_stride=64, v_page_stride=2048, v_head_stride=1024,
             v_slot_stride=64, n_pages=4, n_heads=2, page_size=16, head_dim=64, dtype=_lib.WT_DTYPE_F16, reserved=0, error=None)
    return _lib.KvCache(**dict(d, **kw))


def append(c=None, **kw):
    a = dict(k=A, v=A, dtype=1, k_row=128, k_head=64, v_row=128, v_head=64, n_rows=1, table=A, stride=4, n_seqs=2, width=4, seq=None, pos=A, st=None)
    a.update(kw)
    return _lib.load().wt_kv_append(ctypes.byref(c or desc()), *a.values())


def gather(c=None, **kw):
    a = dict(k=A, v=2 * A, dtype=1, n_rows=1, table=A, stride=4, n_seqs=2, width=4, seq=None, pos=A, st=None)
    a.update(kw)
    return _lib.load().wt_kv_gather(ctypes.byref(c or desc()), *a.values())


def attend(c=None, **kw):
    a = dict(q=A, dtype=1, q_row=256, q_head=64, n_seqs=2, n_q_heads=4, scale=1.0, table=A, stride=4, width=4, lengths=A, out=A, o_row=256, o_head=64,
             lse=None, ws=None, ws_bytes=0, st=None)
    a.update(kw)
    return _lib.load().wt_kv_attend(ctypes.byref(c or desc()), *a.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(n_pages=0), dict(n_heads=0), dict(page_size=0), dict(reserved=1), dict(dtype=4), dict(dtype=0), dict(k=A + 8),
              dict(k_exp=A), dict(dtype=3), dict(k_slot_stride=65), dict(v_head_stride=-64), dict(head_dim=80), dict(head_dim=0)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_entries_refuse_a_bad_cache(bad):
    for f in (append, gather, attend):
        assert f(desc(**bad)) in (-1, -3)
        assert b"wt_kv_" in _lib.load().wt_last_error()


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 2), dict(k=A + 8), dict(dtype=0), dict(dtype=3), dict(k_row=130), dict(v_head=4), dict(n_rows=-1),
                                 dict(n_rows=3), dict(pos=None), dict(table=None), dict(stride=3), dict(width=0), dict(width=1 << 28), dict(n_seqs=-1)],
                         ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_append_refuses(bad):
    assert append(**bad) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 2), dict(dtype=0), dict(dtype=3), dict(n_rows=-1), dict(n_rows=3), dict(pos=None),
                                 dict(table=None), dict(stride=3), dict(width=0)], ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_gather_refuses(bad):
    assert gather(**bad) == -1


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(lengths=None), dict(dtype=0), dict(dtype=3), dict(n_q_heads=0), dict(n_q_heads=3),
                                 dict(n_seqs=-1), dict(table=None), dict(stride=3), dict(width=0), dict(n_seqs=1 << 30, n_q_heads=4)],
                         ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_attend_refuses(bad):
    assert attend(**bad) == -1


def test_nothing_to_do():
    assert append(n_rows=0) == 0 and gather(n_rows=0) == 0 and attend(n_seqs=0) == 0


def test_cache_descriptor_matches_the_header():
    assert ctypes.sizeof(_lib.KvCache) == 112
    assert [getattr(_lib.KvCache, n).offset for n in ("k", "v_exp", "k_page_stride", "v_slot_stride", "n_pages", "head_dim", "dtype", "error")] == \
        [0, 24, 32, 72, 80, 92, 96, 104]
