"""Which memory the paged cache's calls take: pieces that share a byte where both are written, or one read and one written, are refused."""
import os
import random
import shutil
import subprocess

import pytest
import torch

from test_kvcache_host import E4M3, TABLE, host_cache, i32, pages
from whisper_timestamped import PagedKVCache
from whisper_timestamped._lib import WtError

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "whisper-timestamped_amd", "csrc")


def test_overlap_of_strided_pieces(tmp_path):
    """csrc/wt_overlap.h against the bytes listed one by one, for pieces of up to three dimensions in any order, a few of them nested,
    interleaved or with strides of zero."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    rng = random.Random(0)
    lines, want = [], []
    for _ in range(4000):
        both, same = [], rng.random() < 0.4
        for _ in range(2):
            dims = [(rng.choice([1, 2, 2, 3, 5]), rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48, 64, 100])) for _ in range(3)]
            if same and both:
                dims = list(both[0][2])
                rng.shuffle(dims)
            both.append((rng.randrange(200), rng.choice([1, 2, 4, 5, 16]), dims))
        seen = [{at + sum(i * s for i, (_, s) in zip((x, y, z), dims)) + b for x in range(dims[0][0]) for y in range(dims[1][0])
                 for z in range(dims[2][0]) for b in range(row)} for at, row, dims in both]
        want.append(int(bool(seen[0] & seen[1])))
        lines.append(" ".join(str(v) for at, row, dims in both for v in (at, row, *[n for n, _ in dims], *[s for _, s in dims])))
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text("""#include <cstdio>
#include "wt_overlap.h"
int main() {
    long long a[16];
    static char memory[4096];
    for (;;) {
        wt::Strided3 s[2];
        for (int i = 0; i < 16; ++i) if (std::scanf("%lld", a + i) != 1) return 0;
        for (int i = 0; i < 2; ++i) {
            const int64_t n[3] = {a[8 * i + 2], a[8 * i + 3], a[8 * i + 4]}, st[3] = {a[8 * i + 5], a[8 * i + 6], a[8 * i + 7]};
            s[i] = wt::Strided3(memory + a[8 * i], a[8 * i + 1], 3, n, st);
        }
        std::printf("%d\\n", (int)wt::overlap(s[0], s[1]));
    }
}
""")
    subprocess.check_call([cxx, "-O1", "-std=c++17", "-Wall", "-Werror", "-I" + CSRC, str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)], input="\n".join(lines), text=True).split()]
    assert got == want and 500 < sum(want) < 3500


def cut(base, at, shape, strides):
    return base.as_strided(shape, strides, at)


BASE = torch.zeros(40000, dtype=torch.float16)
SHAPE = (4, 2, 16, 64)


@pytest.mark.parametrize("k,v,shared", [
    ((0, (2048, 1024, 64, 1)), (8192, (2048, 1024, 64, 1)), False),                # one behind the other
    ((0, (2048, 1024, 64, 1)), (2048, (2048, 1024, 64, 1)), True),                 # a page further on
    ((0, (2048, 1024, 64, 1)), (8192 - 64, (2048, 1024, 64, 1)), True),            # the last row
    ((0, (4096, 1024, 64, 1)), (2048, (4096, 1024, 64, 1)), False),                # pages in turn
    ((0, (4096, 1024, 64, 1)), (2048 - 8, (4096, 1024, 64, 1)), True),
    ((0, (4096, 2048, 128, 1)), (64, (4096, 2048, 128, 1)), False),                # side by side in a slot
    ((0, (4096, 2048, 128, 1)), (56, (4096, 2048, 128, 1)), True),
    ((0, (4096, 2048, 64, 1)), (1024, (4096, 2048, 64, 1)), False),                # heads in turn
    ((0, (4096, 1024, 64, 1)), (2048, (4096, 64, 128, 1)), False),                 # pages in turn, another order inside
    ((0, (4096, 1024, 64, 1)), (1984, (4096, 64, 128, 1)), True),
    ((0, (64, 4096, 256, 1)), (20000, (2048, 1024, 64, 1)), False),
    ((0, (64, 4096, 256, 1)), (64, (2048, 1024, 64, 1)), True),
])
def test_keys_and_values_share_nothing(k, v, shared):
    with pytest.raises(WtError, match="share memory" if shared else "GPU"):
        PagedKVCache(cut(BASE, k[0], SHAPE, k[1]), cut(BASE, v[0], SHAPE, v[1]))


def test_exponents_share_nothing():
    k, v = pages(*SHAPE, dtype=E4M3), pages(*SHAPE, dtype=E4M3)
    e = torch.zeros(400, dtype=torch.uint8)
    one, two = e[:128].view(4, 2, 16), e[112:240].view(4, 2, 16)
    with pytest.raises(WtError, match="k_exp and v_exp share memory"):
        PagedKVCache(k, v, one, two)
    inside = v.view(torch.uint8).reshape(-1)[1024:1152].view(4, 2, 16)
    with pytest.raises(WtError, match="v and k_exp share memory"):
        PagedKVCache(k, v, inside, two)
    with pytest.raises(WtError, match="GPU"):
        PagedKVCache(k, v, one, e[128:256].view(4, 2, 16))


def cache_over(k, v, *e):
    from whisper_timestamped import kvcache
    cache = object.__new__(PagedKVCache)
    cache._calls = kvcache._calls()
    cache._handle, cache.error = cache._calls.make(k, v, *(e or (None, None)), True)
    return cache


def test_rows_are_not_the_caches_own_memory():
    """append reads rows while it writes the cache, gather and attend write results while they read it."""
    mem = torch.zeros(3, *SHAPE, dtype=torch.float16)
    cache = cache_over(mem[0], mem[1])
    free = mem[2].reshape(-1)[:3 * 2 * 64].view(3, 2, 64)
    own = [m.reshape(-1)[256:256 + 3 * 2 * 64].view(3, 2, 64) for m in mem[:2]]
    pos = i32(0, 1, 2)
    for mine in own:
        for k, v, name in ((mine, free, "k"), (free, mine, "v")):
            with pytest.raises(WtError, match=f"{name}: the cache's own memory"):
                cache.append(k, v, TABLE, pos)
            with pytest.raises(WtError, match=r"out\[%d\]: the cache's own memory" % (name == "v")):
                cache.gather(TABLE, pos, out=(k, v.clone()) if name == "k" else (k.clone(), v))
        with pytest.raises(WtError, match="out: the cache's own memory"):
            cache.attend(free, TABLE, pos, out=mine)
    with pytest.raises(WtError, match="only run on the GPU"):
        cache.append(free, free, TABLE, pos)                      # (beside the cache in one piece of memory: fine)
    e = [torch.zeros(4, 2, 16, dtype=torch.uint8) for _ in range(2)]
    cache = cache_over(pages(*SHAPE, dtype=E4M3), pages(*SHAPE, dtype=E4M3), *e)
    wide = pages(3, 2, 64)
    rows = e[1].reshape(-1).view(torch.float16).as_strided((3, 2, 64), (0, 0, 1))
    with pytest.raises(WtError, match="k: the cache's own memory"):
        cache.append(rows, wide, TABLE, pos)


def test_results_and_queries():
    """out is q itself, or shares nothing with it: side by side in one tensor is fine, a few values or rows apart is not."""
    base = torch.zeros(4000, dtype=torch.float16)
    q = base.as_strided((3, 4, 64), (512, 64, 1), 0)
    for out, said in ((q, "GPU"), (base.as_strided((3, 4, 64), (512, 64, 1), 256), "GPU"), (base.as_strided((3, 4, 64), (512, 64, 1), 255), "out: shares memory"),
                      (base.as_strided((3, 4, 64), (512, 64, 1), 64), "out: shares memory"), (base.as_strided((3, 4, 64), (512, 64, 1), 512), "out: shares memory"),
                      (base.as_strided((3, 4, 64), (256, 64, 1), 0), "out: shares memory"), (base.as_strided((3, 4, 64), (256, 64, 1), 1536), "GPU")):
        with pytest.raises(WtError, match=said):
            host_cache().attend(q, TABLE, i32(1, 2, 3), out=out)
    # one query for two sequences and the results of both: the first one's result is where the second still reads
    both = torch.zeros(512, dtype=torch.float16)
    with pytest.raises(WtError, match="out: shares memory"):
        host_cache().attend(both.as_strided((2, 4, 64), (0, 64, 1)), TABLE[:2], i32(1, 2), out=both.view(2, 4, 64))


def test_lazy_clones_are_pieces_of_their_own():
    """Two lazy clones of one tensor share its memory until one is written: they are two tensors, and what they came from is a third."""
    base = pages(*SHAPE)
    k, v = base._lazy_clone(), base._lazy_clone()
    cache = cache_over(k, v)
    rows = base.reshape(-1)[:3 * 2 * 64].view(3, 2, 64)
    with pytest.raises(WtError, match="only run on the GPU"):
        cache.append(rows, rows, TABLE, i32(0, 1, 2))
    mine = k.reshape(-1)[:3 * 2 * 64].view(3, 2, 64)
    with pytest.raises(WtError, match="k: the cache's own memory"):
        cache.append(mine, rows, TABLE, i32(0, 1, 2))
