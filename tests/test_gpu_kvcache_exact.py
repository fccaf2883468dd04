"""The attention over paged caches on inputs whose results are known to the last bit or nearly so: a weight that lost bits, a key
that was lost or counted twice is in plain sight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, E4M3), (F16, E4M3), (BF16, E4M3)]
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def cache_of(k, v, page, dtype, exponents=(127, 127)):
    """A cache that holds k, v (positions, heads, width; exact in `dtype`) as one sequence, pages in a scrambled order, NaN behind the
    end; (cache, table row)."""
    from whisper_timestamped import PagedKVCache
    n, heads, width = k.shape
    n_pages = -(-n // page)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(n))
    both = []
    for x in (k, v):
        pages = torch.full((n_pages * page, heads, width), math.nan)
        pages[:n] = x.float()
        held = torch.empty((n_pages, heads, page, width))
        held[order] = pages.reshape(n_pages, page, heads, width).transpose(1, 2)
        both.append(held.to(dtype).to(DEV))
    e = [torch.full(both[0].shape[:3], x, dtype=torch.uint8, device=DEV) if dtype == E4M3 else None for x in exponents]
    return PagedKVCache(*both, *e), order.int().to(DEV)[None]


@pytest.mark.parametrize("n,spread", [(1, 0.0), (2, 1.0), (31, 3.5), (64, 3.5), (64, 20.0)])
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_each_weight_by_itself(q_dtype, dtype, n, spread):
    """Key t has a value in column t alone, so element t of the result is its weight: each has as many bits as the result's type,
    also one that is e^-20 of the largest.  Scores are single products, exact."""
    width = 64
    g = torch.Generator().manual_seed(n)
    away = torch.linspace(0, spread, n)[torch.randperm(n, generator=g)]
    k, v = torch.zeros((n, 1, width)), torch.zeros((n, 1, width))
    k[:, 0, 0] = -away
    k = k.to(dtype).float()                                       # (what the type holds of them: the spacing is of no matter)
    top = 2.0 ** 14 if q_dtype == F16 else 1.0                    # keeps e^-20 away from f16's subnormal numbers
    v[torch.arange(n), 0, torch.arange(n)] = 1.0 if dtype == E4M3 else top
    cache, table = cache_of(k, v, 8, dtype, (127, 127 + (14 if top > 1 else 0)))
    q = torch.zeros((1, 1, width), dtype=q_dtype, device=DEV)
    q[..., 0] = 1.0
    out, lse = cache.attend(q, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0, return_lse=True)
    w = k[:, 0, 0].double()
    want = torch.zeros(width, dtype=torch.float64)
    want[:n] = torch.softmax(w, 0) * top
    far = w.max() - w
    # steps of 2^-24 of a weight: its exponent's product with log2 e 1.5 per unit of distance (up to 11 more to the running reference),
    # the exponential 2, once more for each of two moves of the reference and one join of waves; of the sums 8 + 2 + 4 below and 4
    # above the line, the quotient 1; 16-bit results: a weight of two 16-bit parts 2^-17 at most; below 2^-14 f16 has steps of 2^-24,
    # half a step off: 2^-25 (the least weight of 20.0 is 16384 e^-20 / 3.5 = 2^-17)
    steps = torch.zeros(width, dtype=torch.float64)
    steps[:n] = 1.5 * (far + (11 if q_dtype != F32 else 0)) + (2 if spread < 4 else 8) + 14 + 4 + 1
    allowed = want * (steps * 2.0 ** -24 + (2.0 ** -17 if q_dtype != F32 else 0.0))
    allowed += HALF_STEP[q_dtype] * (want + allowed) + (2.0 ** -25 if q_dtype == F16 else 0.0)
    got = out[0, 0].double().cpu()
    assert bool((got[n:] == 0).all())
    assert float(((got - want).abs()[:n] / allowed[:n]).max()) <= 1.0
    assert abs(float(lse) - float(torch.logsumexp(w, 0))) <= 2.0 ** -20 * (1 + abs(float(torch.logsumexp(w, 0))))
    cache.check()
