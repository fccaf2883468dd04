#!/usr/bin/env python3
"""The paged cache's kernels on buffers whose neighbours are unmapped pages, as run_guarded.py does for the others: every
pages tensor, exponents, table, positions, lengths, queries, results and workspace ends at the last mapped byte of its mapping
(or starts at the first), and results are compared bit for bit with the same calls on ordinary tensors.

    python tests/guard/run_guarded_kv.py CASE MODE        CASE in CASES, MODE in {end, start}
"""
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
for p in (HERE, os.path.dirname(HERE), os.path.join(os.path.dirname(os.path.dirname(HERE)), "whisper-timestamped_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)

from run_guarded import guarded as fence  # noqa: E402

E4M3 = torch.float8_e4m3fn
# name: (cache type, q / rows type, head_dim, page size, key heads, query heads, lengths): the last page's last slot is in
# use (the longest access there is) and the last page is cut, tables as wide as their longest row
CASES = {
    "f16_pages_of_16": (torch.float16, torch.float16, 64, 16, 2, 4, [33, 0, 128, 1]),
    "bf16_pages_of_64": (torch.bfloat16, torch.bfloat16, 128, 64, 2, 6, [64, 190, 1]),
    "f32_pages_of_24": (torch.float32, torch.float32, 96, 24, 1, 2, [24, 71, 5]),
    "f32_pages_of_7": (torch.float32, torch.float32, 32, 7, 3, 3, [49, 6]),
    "e4m3_pages_of_32": (E4M3, torch.float16, 64, 32, 2, 34, [32, 95, 0]),
    "e4m3_pages_of_5": (E4M3, torch.float32, 96, 5, 2, 4, [25, 11]),
    "e4m3_pages_of_8": (E4M3, torch.bfloat16, 256, 8, 1, 8, [40, 7]),
    "f16_256_pages_of_100": (torch.float16, torch.float16, 256, 100, 1, 1, [100, 99]),
    "split_f16": (torch.float16, torch.float16, 128, 64, 1, 3, [5000, 1, 2999]),
    "split_e4m3": (E4M3, torch.bfloat16, 128, 16, 1, 20, [4096, 4095]),
    "split_f32": (torch.float32, torch.float32, 64, 50, 1, 16, [3000, 1500]),
    "split_bf16_48_queries": (torch.bfloat16, torch.bfloat16, 128, 24, 1, 48, [2500, 0, 3001]),
}
_BITS = {torch.bfloat16: torch.int16, E4M3: torch.uint8}


def guarded(t, mode):
    if t.dtype in _BITS:                     # (types the array interface does not name travel as others of their width)
        b = t.contiguous().view(_BITS[t.dtype])
        return (guarded(b.view(torch.float16), mode) if b.dtype == torch.int16 else fence(b, mode)).view(t.dtype)
    return fence(t, mode)


def calls(name, wrap):
    from whisper_timestamped import PagedKVCache
    dtype, q_dtype, d, page, heads, q_heads, lengths = CASES[name]
    g = torch.Generator().manual_seed(len(name))

    def rand(*shape, dtype):
        return torch.randn(shape, generator=g).to(dtype)

    pages_of = [-(-n // page) for n in lengths]
    n_pages = sum(pages_of)
    table = torch.full((len(lengths), max(pages_of)), -1, dtype=torch.int32)
    ids = torch.randperm(n_pages, generator=g).int()
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = ids[at:at + n]
        at += n
    shape = (n_pages, heads, page, d)
    cuda = lambda t: wrap(t.cuda())  # noqa: E731
    if dtype == E4M3:
        pages = [cuda(rand(*shape, dtype=torch.float32).to(E4M3)) for _ in range(2)] + \
            [cuda(torch.randint(120, 130, shape[:3], generator=g, dtype=torch.uint8)) for _ in range(2)]
    else:
        pages = [cuda(rand(*shape, dtype=dtype)) for _ in range(2)]
    cache = PagedKVCache(*pages)
    rows = [(b, p) for b, n in enumerate(lengths) for p in range(max(0, n - 9), n)]
    seq, pos = (cuda(torch.tensor([r[i] for r in rows], dtype=torch.int32)) for i in range(2))
    table = cuda(table)
    cache.append(cuda(rand(len(rows), heads, d, dtype=q_dtype)), cuda(rand(len(rows), heads, d, dtype=q_dtype)), table, pos, sequences=seq)
    out = tuple(cuda(torch.zeros((len(rows), heads, d), dtype=q_dtype)) for _ in range(2))
    cache.gather(table, pos, sequences=seq, out=out)
    q = cuda(rand(len(lengths), q_heads, d, dtype=q_dtype))
    lens = cuda(torch.tensor(lengths, dtype=torch.int32))
    ws = cache.attend_workspace(q_heads, table)
    assert (ws is not None) == name.startswith("split")
    res = cuda(torch.zeros_like(q))
    for _ in range(2):                       # (the second call finds the workspace as the first left it)
        cache.attend(q, table, lens, out=res, workspace=None if ws is None else (ws if wrap is plain else wrap(ws)))
    torch.cuda.synchronize()
    cache.check()
    return [*pages, *out, res]


def plain(t):
    return t


def main():
    name, mode = sys.argv[1:3]
    want = calls(name, plain)
    print(f"guarded {name}/{mode}: running", flush=True)
    got = calls(name, lambda t: guarded(t, mode))
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), f"{name}/{mode}: tensor {i} differs"
    print(f"guarded {name}/{mode}: ok", flush=True)


if __name__ == "__main__":
    main()
