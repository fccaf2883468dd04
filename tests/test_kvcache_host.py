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
    (pages(4, 2, 16, 64).transpose(0, 2), pages(4, 2, 16, 64).transpose(0, 2), None, None, "GPU"),
    (pages(4, 2, 16, 128)[..., :64], pages(4, 2, 16, 128)[..., 64:], None, None, "GPU"),
    (torch.zeros(9000, dtype=torch.float16).as_strided((4, 2, 16, 64), (128, 64, 512, 1)), pages(4, 2, 16, 64), None, None, "GPU"),
    (torch.zeros(9000, dtype=torch.float16).as_strided((4, 2, 16, 64), (1024, 1024, 64, 1)), pages(4, 2, 16, 64), None, None, "overlap"),
    ([1], pages(4, 2, 16, 64), None, None, "k: not a tensor"),
    (pages(1, 70000, 1, 32), pages(1, 70000, 1, 32), None, None, "65535 heads"),
    (pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, dtype=torch.uint8), pages(4, 2, 17, dtype=torch.uint8).reshape(-1)[1:129].view(4, 2, 16), "16-byte aligned"),
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


def test_the_same_exponents_twice():
    k, v, e = pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, dtype=torch.uint8)
    with pytest.raises(WtError, match="k_exp and v_exp are the same memory"):
        PagedKVCache(k, v, e, e)


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


BAD_CACHES = [dict(k=None), dict(v=None), dict(n_pages=0), dict(n_heads=0), dict(n_heads=65536), dict(page_size=0), dict(reserved=1), dict(dtype=4), dict(dtype=0), dict(k=A + 8),
              dict(k_exp=A), dict(dtype=3), dict(k_slot_stride=65), dict(v_head_stride=-64), dict(head_dim=80), dict(head_dim=0)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_entries_refuse_a_bad_cache(bad):
    for f in (append, gather, attend):
        assert f(desc(**bad)) in (-1, -3)
        assert b"wt_kv_" in _lib.load().wt_last_error()


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=A + 2), dict(k=A + 8), dict(dtype=0), dict(dtype=3), dict(k_row=130), dict(v_head=4), dict(n_rows=-1), dict(n_rows=(1 << 30) + 1, seq=A),
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


# The calls' own checks, on a cache whose tensors are the host's: what is right but for that is refused at the end.
def host_cache(dtype=torch.float16, heads=2, page=16, width=64):
    from whisper_timestamped import kvcache
    cache = object.__new__(PagedKVCache)
    k, v = pages(4, heads, page, width, dtype=dtype), pages(4, heads, page, width, dtype=dtype)
    e = [pages(4, heads, page, dtype=torch.uint8) if dtype == E4M3 else None for _ in range(2)]
    cache._calls = kvcache._calls()
    cache._handle, cache.error = cache._calls.make(k, v, *e, True)
    cache._keep = k, v, e
    return cache


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


TABLE = torch.zeros((3, 4), dtype=torch.int32)
ROWS = pages(3, 2, 64)


@pytest.mark.parametrize("change,said", [
    ({}, "only run on the GPU"),
    (dict(k=None), "k: not a tensor"),
    (dict(k=pages(3, 2, 64, dtype=torch.float32)), "k and v differ"),
    (dict(k=pages(3, 2, 64, dtype=torch.float32), v=pages(3, 2, 64, dtype=torch.float32)), "Float with a cache of Half"),
    (dict(v=pages(3, 1, 64)), r"v: \(3, 1, 64\), not \(3, 2, 64\)"),
    (dict(k=pages(3, 128)), "k: 2 dimensions"),
    (dict(k=pages(3, 2, 128)[..., ::2]), "k: a head's values stand side by side"),
    (dict(k=pages(3, 2, 65)[..., :64]), "16-byte"),
    (dict(k=pages(3, 2, 72)[..., 4:68]), "16-byte"),
    (dict(positions=i32(0, 1)), r"k: \(3, 2, 64\), not \(2, 2, 64\)"),
    (dict(positions=torch.zeros(3)), "positions: 3 int32"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions: 3 int32"),
    (dict(positions=torch.zeros((3, 1), dtype=torch.int32)), "positions: 2 dimensions"),
    (dict(positions=torch.zeros(6, dtype=torch.int32)[::2]), "side by side"),
    (dict(sequences=i32(0, 1)), "sequences: 3 int32"),
    (dict(k=pages(4, 2, 64), v=pages(4, 2, 64), positions=i32(0, 1, 2, 3)), "4 rows for 3 sequences"),
    (dict(table=TABLE.long()), "page table: not int32"),
    (dict(table=TABLE[0]), "page table: 1 dimensions"),
    (dict(table=TABLE.t().contiguous().t()), "side by side"),
    (dict(table=TABLE[:1].expand(3, 4)), "its rows apart"),
    (dict(table=torch.zeros((3, 0), dtype=torch.int32)), "page table"),
])
def test_append_arguments(change, said):
    a = dict(k=ROWS, v=ROWS, table=TABLE, positions=i32(0, 1, 2), sequences=None)
    with pytest.raises(WtError, match=said):
        host_cache().append(**dict(a, **change))


@pytest.mark.parametrize("dtype,change,said", [
    (torch.float16, {}, "only run on the GPU"),
    (torch.float16, dict(dtype=torch.float32), "Float with a cache of Half"),
    (E4M3, dict(dtype=torch.float64), "Double"),
    (E4M3, dict(dtype=E4M3), "Float8"),
    (E4M3, dict(dtype=torch.bfloat16), "only run on the GPU"),
    (torch.float16, dict(dtype="float16"), "torch.dtype"),
    (torch.float16, dict(out=ROWS), "out: two tensors"),
    (torch.float16, dict(out=(ROWS, ROWS)), "the same memory"),
    (torch.float16, dict(out=(ROWS, pages(2, 2, 64))), r"out\[1\]"),
    (torch.float16, dict(out=(ROWS, pages(3, 2, 64, dtype=torch.float32))), "out: Half and Float"),
    (torch.float16, dict(out=(pages(3, 4, 64)[:, :2], ROWS)), "not contiguous"),
    (torch.float16, dict(out=(ROWS, pages(3, 2, 64)), dtype=torch.bfloat16), "out: Half"),
    (torch.float16, dict(positions=torch.zeros(3)), "positions"),
])
def test_gather_arguments(dtype, change, said):
    a = dict(table=TABLE, positions=i32(0, 1, 2), sequences=None, dtype=None, out=None)
    with pytest.raises(WtError, match=said):
        host_cache(dtype).gather(**dict(a, **change))


Q = pages(3, 4, 64)


@pytest.mark.parametrize("change,said", [
    ({}, "only run on the GPU"),
    (dict(q=pages(3, 3, 64)), "3 query heads over 2"),
    (dict(q=pages(3, 0, 64)), "0 query heads"),
    (dict(q=pages(2, 4, 64)), r"q: \(2, 4, 64\), not \(3, 4, 64\)"),
    (dict(q=pages(3, 4, 32)), "q:"),
    (dict(q=pages(3, 4, 64, dtype=torch.bfloat16)), "BFloat16 with a cache of Half"),
    (dict(q=pages(3, 4, 128)[..., ::2]), "side by side"),
    (dict(lengths=torch.zeros(3)), "lengths"),
    (dict(lengths=i32(1, 2)), "lengths: 3 int32"),
    (dict(out=pages(3, 4, 64, dtype=torch.float32)), "out: Float"),
    (dict(out=3), "out: not a tensor"),
    (dict(out=pages(1, 4, 64).expand(3, 4, 64)), "one place"),
    (dict(out=pages(3, 1, 64).expand(3, 4, 64)), "one place"),
    (dict(out=torch.zeros(3 * 64 + 512, dtype=torch.float16).as_strided((3, 4, 64), (64, 64, 1))), "one place"),
    (dict(out=torch.zeros(12 * 64, dtype=torch.float16).as_strided((3, 4, 64), (64, 192, 1))), "only run on the GPU"),
    (dict(workspace=pages(100)), "workspace"),
    (dict(table=TABLE[:2]), "q:"),
])
def test_attend_arguments(change, said):
    a = dict(q=Q, table=TABLE, lengths=i32(1, 2, 3))
    with pytest.raises(WtError, match=said):
        host_cache().attend(**dict(a, **change))


def test_gradients_are_refused():
    """Recorded calls would silently lack their gradient; under no_grad the same tensors are taken."""
    w = [pages(3, 2, 64).requires_grad_() for _ in range(2)]
    q = Q.clone().requires_grad_()
    c = host_cache()
    for f in (lambda: c.append(w[0], ROWS, TABLE, i32(0, 1, 2)), lambda: c.append(ROWS, w[1], TABLE, i32(0, 1, 2)), lambda: c.attend(q, TABLE, i32(1, 2, 3)),
              lambda: c.attend(Q, TABLE, i32(1, 2, 3), out=q), lambda: c.gather(TABLE, i32(0, 1, 2), out=tuple(w))):
        with pytest.raises(WtError, match="gradient"):
            f()
        with torch.no_grad(), pytest.raises(WtError, match="only run on the GPU"):
            f()
    with pytest.raises(WtError, match="no gradient"):
        PagedKVCache(pages(4, 2, 16, 64).requires_grad_(), pages(4, 2, 16, 64))


def test_attend_wrong_python_types():
    with pytest.raises(TypeError):
        host_cache().attend(Q, TABLE, i32(1, 2, 3), scale="x")
    with pytest.raises(TypeError):
        host_cache().attend_workspace("x", TABLE)
    with pytest.raises(WtError, match="0 query heads"):
        host_cache().attend_workspace(0, TABLE)


def test_the_cache_keeps_its_memory():
    """What a call's addresses point into is held by the cache itself, whatever becomes of the tensors that named it."""
    from whisper_timestamped import kvcache
    k, v = pages(4, 2, 16, 64, dtype=E4M3), pages(4, 2, 16, 64, dtype=E4M3)
    e = [pages(4, 2, 16, dtype=torch.uint8) for _ in range(2)]
    uses = lambda: [torch._C._storage_Use_Count(t.untyped_storage()._cdata) for t in (k, v, *e)]
    before = uses()
    handle, error = kvcache._calls().make(k, v, *e, True)
    assert uses() == [n + 1 for n in before]
    del handle
    assert uses() == before


def test_paged_decoder_leaves_shadowed_modules_alone():
    """A backend whose attention, or whose cache hooks, somebody else has replaced on the instance keeps its own cache."""
    import types
    from whisper_timestamped.paged_decoder import supported

    class Attn:
        query = key = value = out = qkv_attention = forward = None

    class Model:
        dims = types.SimpleNamespace(n_text_state=128, n_text_head=2)
        install_kv_cache_hooks = None

        def __init__(self):
            self.decoder = types.SimpleNamespace(blocks=[types.SimpleNamespace(attn=Attn()) for _ in range(2)])

    assert supported(Model(), torch.float16)
    m = Model()
    m.decoder.blocks[1].attn.forward = lambda x: x
    assert not supported(m, torch.float16)
    m = Model()
    m.install_kv_cache_hooks = lambda cache=None: None
    assert not supported(m, torch.float16)
