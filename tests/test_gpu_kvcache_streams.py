"""The paged cache's calls beside other calls: threads, streams, graphs."""
import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"


def long_cache(n=12000, heads=2, width=64, dtype=F16, seed=0):
    from whisper_timestamped import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    pages = -(-n // 64)
    k, v = (torch.randn((pages, heads, 64, width), generator=g).to(dtype).to(DEV) for _ in range(2))
    return PagedKVCache(k, v), torch.randperm(pages, generator=g).int().to(DEV)[None], torch.tensor([n], dtype=torch.int32, device=DEV)


def test_two_threads_on_their_own_streams():
    """The library's own workspace of hipStreamPerThread is the calling thread's: two threads whose calls split long sequences run
    at the same time, each result as when it runs alone."""
    from whisper_timestamped import _lib
    L = _lib.load()
    cache, table, lens = long_cache()
    stride = lambda x: x.stride()[:3]  # noqa: E731
    desc = _lib.KvCache(k=cache.k.data_ptr(), v=cache.v.data_ptr(), k_exp=None, v_exp=None, k_page_stride=stride(cache.k)[0],
                        k_head_stride=stride(cache.k)[1], k_slot_stride=stride(cache.k)[2], v_page_stride=stride(cache.v)[0],
                        v_head_stride=stride(cache.v)[1], v_slot_stride=stride(cache.v)[2], n_pages=cache.n_pages, n_heads=2, page_size=64,
                        head_dim=64, dtype=_lib.WT_DTYPE_F16, reserved=0, error=None)
    heads = (4, 34)
    qs = [torch.randn((1, h, 64), generator=torch.Generator().manual_seed(h)).half().to(DEV) for h in heads]
    want = [cache.attend(q, table, lens) for q in qs]
    outs = [[torch.zeros_like(q) for _ in range(30)] for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        torch.cuda.set_device(0)
        for out in outs[i]:
            rc = L.wt_kv_attend(ctypes.byref(desc), qs[i].data_ptr(), _lib.WT_DTYPE_F16, heads[i] * 64, 64, 1, heads[i], 0.125, table.data_ptr(),
                                table.shape[1], table.shape[1], lens.data_ptr(), out.data_ptr(), heads[i] * 64, 64, None, None, 0, 2)
            if rc:
                bad.append((rc, L.wt_last_error()))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad
    for w, results in zip(want, outs):
        assert all(torch.equal(r, w) for r in results)


def test_check_waits_for_every_stream():
    """A call on another stream, still waiting behind other work, counts for check()."""
    from whisper_timestamped._lib import WtError
    cache, table, lens = long_cache(n=500)
    q = torch.zeros((1, 2, 64), dtype=F16, device=DEV)
    busy = torch.randn((4096, 4096), device=DEV)
    bad = torch.tensor([table.shape[1] * 64 + 1], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(30):
            busy = busy @ busy * 1e-2
        cache.attend(q, table, bad)
    with pytest.raises(WtError, match="length"):
        cache.check()
    cache.check()


@pytest.mark.parametrize("width,group,columns", [(256, 16, None), (128, 32, 2100), (32, 24, None)])
@pytest.mark.parametrize("given", [False, True])
def test_captured_calls_with_much_shared_memory(width, group, columns, given):
    """16 queries of 256 values and 32 of 128 need more LDS than a launch gets unasked, and split tables a workspace: captured, replayed
    several times with other queries and lengths and with eager calls between, each replay as the eager call."""
    cache, table, _ = long_cache(n=9000, heads=1, width=width, dtype=BF16)
    if columns:
        table = torch.cat([table, torch.full((1, columns - table.shape[1]), -7, dtype=torch.int32, device=DEV)], 1)
    q, out = torch.zeros((1, group, width), dtype=BF16, device=DEV), torch.zeros((1, group, width), dtype=BF16, device=DEV)
    lens = torch.tensor([9000], dtype=torch.int32, device=DEV)
    ws = cache.attend_workspace(group, table)
    assert ws is not None
    cache.attend(q, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, table, lens, out=out, workspace=ws if given else None)
    for turn, n in enumerate((9000, 1, 0, 4321, 9000)):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
        lens.fill_(n)
        want = cache.attend(q, table, lens)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        graph.replay()
        again = cache.attend(q, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want), n
    cache.check()
