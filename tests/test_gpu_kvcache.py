"""The paged key-value cache on the GPU: append, gather, attention of one new token, against 64 bits on the CPU."""
import math

import numpy as np
import pytest
import torch

import kv_oracle as O

pytestmark = pytest.mark.gpu
F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
DEV = "cuda"


def make(seqs_lengths, heads, width, page, dtype, seed=0, layout="page_head_slot", spare=3, junk=True, gain=1.0):
    """A cache that holds seqs_lengths[b] positions of sequence b, its table, and CPU copies.  Slots behind the last position
    hold NaN and infinities (8 bits: NaN codes and the largest power), table entries behind the last page point nowhere."""
    from whisper_timestamped import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    rng = np.random.RandomState(seed)
    pages_of = [-(-n // page) for n in seqs_lengths]
    n_pages = sum(pages_of) + spare
    ids = rng.permutation(n_pages)
    table = np.full((len(seqs_lengths), max([1] + pages_of) + 2), -7, dtype=np.int32)
    table[:, -1] = 2 ** 31 - 1
    shape = (n_pages, heads, page, width)
    kv, exps = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g) * gain
        if dtype == E4M3:
            code, e = O.quantise(x.half().float())
            kv.append(code.float().to(E4M3)), exps.append(e.to(torch.uint8))
        else:
            kv.append(x.to(dtype)), exps.append(None)
    held = torch.zeros(n_pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(seqs_lengths):
        table[b, :pages_of[b]] = ids[at:at + pages_of[b]]
        for p in range(n):
            held[int(table[b, p // page]), p % page] = True
        at += pages_of[b]
    if junk:
        free = ~held[:, None, :].expand(n_pages, heads, page)
        for i, x in enumerate(kv):
            if dtype == E4M3:
                x.view(torch.uint8)[free] = 0x7f
                exps[i][free] = 254
            else:
                x[free] = torch.tensor([math.nan, math.inf, -math.inf][seed % 3], dtype=dtype)
    dev = []
    for x in kv:
        x = x.to(DEV)
        if layout == "page_slot_head":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "side_by_side":       # keys and values of a slot next to each other
            wide = torch.zeros((n_pages, heads, page, 2 * width), dtype=torch.uint8 if dtype == E4M3 else dtype, device=DEV)
            half = wide[..., :width] if not dev else wide[..., width:]
            half.copy_(x.view(torch.uint8) if dtype == E4M3 else x)
            x = half.view(dtype) if dtype == E4M3 else half
        dev.append(x)
    e = [None if t is None else t.to(DEV) for t in exps]
    cache = PagedKVCache(dev[0], dev[1], e[0], e[1])
    return cache, torch.from_numpy(table).to(DEV), kv, exps, table


def queries(B, heads, width, dtype, seed, gain=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn((B, heads, width), generator=g) * gain).to(dtype)


def check_attend(lengths, group, heads, width, page, q_dtype, dtype, seed=0, layout="page_head_slot", gain=1.0, scale=None, q_gain=1.0):
    cache, table, (k, v), (ke, ve), t = make(lengths, heads, width, page, dtype, seed, layout, gain=gain)
    q = queries(len(lengths), heads * group, width, q_dtype, seed, q_gain)
    wide = torch.full((len(lengths) + 1, heads * group + 2, width), 7.0, dtype=q_dtype, device=DEV)
    wide[:-1, 1:-1] = q.to(DEV)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(wide[:-1, 1:-1], table, lens, scale=scale, return_lse=True)
    again = cache.attend(wide[:-1, 1:-1], table, lens, scale=scale)
    assert torch.equal(out, again), "two calls differ"
    worst = 0.0
    sc = width ** -0.5 if scale is None else scale
    for b, n in enumerate(lengths):
        kk = O.rows(k, ke, t, [b] * n, range(n)) if n else torch.zeros((0, heads, width), dtype=torch.float64)
        vv = O.rows(v, ve, t, [b] * n, range(n)) if n else kk
        want, wlse, bound, lbound = O.attend(q[b].double(), kk, vv, sc)
        worst = max(worst, O.far(out[b], want, bound, q_dtype))
        if n == 0:
            assert torch.equal(out[b].cpu(), torch.zeros_like(q[b])) and bool((lse[b] == -math.inf).all())
        else:
            assert float(((lse[b].double().cpu() - wlse).abs() / lbound).max()) <= 1.0, (b, n)
    assert worst <= 1.0, worst
    cache.check()
    return worst


PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, E4M3), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize("width", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_types_and_widths(q_dtype, dtype, width):
    check_attend([0, 1, 2, 31, 32, 33, 65, 200], 2, 3, width, 16, q_dtype, dtype, seed=width)


@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 31, 32, 33, 64, 96, 100, 128, 512])
@pytest.mark.parametrize("q_dtype,dtype", [(F16, F16), (F32, F32), (BF16, E4M3)])
def test_attend_page_sizes(page, q_dtype, dtype):
    check_attend([129, 0, 63, 97, 1, 300], 1, 2, 64, page, q_dtype, dtype, seed=page)


@pytest.mark.parametrize("group,heads", [(1, 1), (1, 20), (2, 4), (3, 2), (5, 1), (8, 2), (15, 1), (16, 2), (17, 1), (24, 2), (40, 1)])
@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, F32), (F16, E4M3)])
def test_attend_groups(group, heads, q_dtype, dtype):
    check_attend([77, 5, 0, 1, 260], group, heads, 128, 32, q_dtype, dtype, seed=group)


@pytest.mark.parametrize("group,page,width,lengths", [(18, 16, 32, [70, 0, 1, 33]), (32, 64, 64, [257, 31]), (33, 32, 96, [64, 5, 0]), (49, 24, 128, [1, 129]),
                                                      (31, 10, 128, [90, 300]), (64, 3, 64, [40]), (24, 64, 128, [40001]), (32, 100, 128, [9000, 0, 1, 3001]),
                                                      (17, 16, 96, [12000, 700]), (48, 32, 32, [30001]), (24, 16, 256, [5000, 17])])
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_wide_groups(group, page, width, lengths, q_dtype, dtype):
    """More than 16 query heads a key head: two tiles of them at a time, whole and split, with joins in groups."""
    check_attend(lengths, group, 1, width, page, q_dtype, dtype, seed=group)


@pytest.mark.parametrize("layout", ["page_slot_head", "side_by_side"])
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_layouts(layout, q_dtype, dtype):
    check_attend([1, 40, 131], 2, 4, 64, 16, q_dtype, dtype, seed=5, layout=layout)


@pytest.mark.parametrize("lengths", [[4097], [3000, 1, 0, 2999], [8191, 8192, 8193], [20000]])
@pytest.mark.parametrize("q_dtype,dtype", [(F16, F16), (F32, F32), (BF16, E4M3), (BF16, BF16)])
def test_attend_long(lengths, q_dtype, dtype):
    check_attend(lengths, 4, 1, 64, 64, q_dtype, dtype, seed=len(lengths))


@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_many_short_sequences(q_dtype, dtype):
    check_attend([(7 * i) % 40 for i in range(150)], 1, 6, 32, 8, q_dtype, dtype, seed=9)


@pytest.mark.parametrize("group,heads,width,q_dtype,dtype", [(1, 2, 128, BF16, BF16), (17, 1, 64, F32, F32), (20, 1, 96, F16, E4M3), (2, 1, 256, F16, F16), (3, 2, 32, BF16, E4M3)])
def test_attend_shares_of_many_sequences(group, heads, width, q_dtype, dtype):
    """Long tables over more sequences than a wave has lanes: empty ones at every place where the prefix sums change hands,
    ones of a single key, some that many workgroups share."""
    lengths = [(i * 37) % 90 for i in range(150)]
    for i in (0, 62, 63, 64, 127, 128, 149):
        lengths[i] = 0
    item = {F32: 4, E4M3: 1}.get(dtype, 2)
    long = 600000 // (2 * width * item)                  # beyond what one workgroup takes by itself
    lengths[1], lengths[65], lengths[66], lengths[148] = long, 3 * long + 1, 1, 2 * long - 3
    check_attend(lengths, group, heads, width, 16, q_dtype, dtype, seed=group)


def test_attend_shares_of_empty_sequences():
    cache, table, _, _, _ = make([0] * 70, 2, 64, 16, F16)
    wide = torch.zeros((70, 5000), dtype=torch.int32, device=DEV)
    out, lse = cache.attend(queries(70, 2, 64, F16, 0).to(DEV), wide, torch.zeros(70, dtype=torch.int32, device=DEV), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    cache.check()


def test_attend_workspace():
    """One workspace for calls of different shapes, one after the other; another's size, type or device is refused."""
    from whisper_timestamped._lib import WtError
    cache, table, _, _, _ = make([4000, 3, 2500], 2, 64, 16, F16, seed=5)
    lens = torch.tensor([4000, 3, 2500], dtype=torch.int32, device=DEV)
    ws = cache.attend_workspace(8, table)
    assert ws is not None and cache.attend_workspace(8, table[:, :16]) is None
    for heads in (8, 2, 8, 4):
        q = queries(3, heads, 64, F16, heads).to(DEV)
        want = cache.attend(q, table, lens)
        assert torch.equal(cache.attend(q, table, lens, workspace=ws), want)
        assert torch.equal(cache.attend(q[:2], table[:2], lens[:2], workspace=ws), want[:2])
    assert bool((ws[:16384] == 0).all()), "a call leaves the counters at zero"
    for bad in (ws[:20000], ws.view(torch.int32), ws.cpu(), ws[1:]):
        with pytest.raises(WtError, match="workspace"):
            cache.attend(q, table, lens, workspace=bad)


def test_attend_workspace_for_fewer_sequences():
    """A workspace for a table's shape does for its first sequences too, also where only those are split."""
    cache, table, _, _, _ = make([1792] * 16, 8, 64, 16, F16, seed=6)
    lens = torch.full((16,), 1792, dtype=torch.int32, device=DEV)
    ws = cache.attend_workspace(8, table)
    assert ws is not None
    q = queries(16, 8, 64, F16, 1).to(DEV)
    for n in (16, 3, 1):
        assert torch.equal(cache.attend(q[:n], table[:n], lens[:n], workspace=ws), cache.attend(q[:n], table[:n], lens[:n]))
    assert bool((ws[:16384] == 0).all())


@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
@pytest.mark.parametrize("scale,q_gain", [(1.0, 4.0), (-0.5, 1.0), (0.0, 1.0), (1e-3, 1.0)])
def test_attend_scales(q_dtype, dtype, scale, q_gain):
    """Peaked rows, a negative scale (the least product wins), no scale at all (the mean of the values)."""
    check_attend([1, 50, 333], 2, 2, 64, 16, q_dtype, dtype, seed=3, scale=scale, q_gain=q_gain)


@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_one_weight_against_many_small_ones(q_dtype, dtype):
    """One key ahead of 2000 equal ones by 9: their weights, 2^-13 each, carry a fifth of the result between them."""
    cache, table, (k, v), (ke, ve), t = make([2001], 1, 64, 64, dtype, seed=4)
    for x in (cache.k, k):
        x.view(torch.uint8).zero_() if dtype == E4M3 else x.zero_()
    if dtype == E4M3:
        cache.k_exp.fill_(127), ke.fill_(127)
    page, slot = int(t[0, 1000 // 64]), 1000 % 64
    for x in (cache.k, k):
        x[page, 0, slot] = torch.full((64,), 1.125, dtype=F32).to(dtype).to(x.device)
    q = torch.ones((1, 1, 64), dtype=q_dtype)
    out, lse = cache.attend(q.to(DEV), table, torch.tensor([2001], dtype=torch.int32, device=DEV), scale=0.125, return_lse=True)
    want, wlse, bound, lb = O.attend(q[0].double(), O.rows(k, ke, t, [0] * 2001, range(2001)), O.rows(v, ve, t, [0] * 2001, range(2001)), 0.125)
    assert O.far(out[0], want, bound, q_dtype) <= 1.0
    assert float((lse[0].double().cpu() - wlse).abs() / lb) <= 1.0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attend_infinite_scores(dtype):
    """A key of -inf weighs nothing (wherever it stands), all of them at -inf leave no result, NaN and +inf likewise: as the
    formula has it.  Head 1 is untouched by what head 0 holds."""
    cache, table, (k, v), _, t = make([200] * 5, 2, 64, 16, dtype, seed=1)
    q = queries(5, 2, 64, dtype, 1).abs() + 0.5

    def put(b, positions, value):
        for p in positions:
            cache.k[int(t[b, p // 16]), 0, p % 16] = value
            k[int(t[b, p // 16]), 0, p % 16] = value

    put(0, range(0, 130), -math.inf)
    put(1, range(200), -math.inf)
    put(2, [199], math.nan)
    put(3, [0], math.inf)
    out, lse = cache.attend(q.to(DEV), table, torch.full((5,), 200, dtype=torch.int32, device=DEV), return_lse=True)
    for b in range(5):
        kk, vv = (O.rows(x, None, t, [b] * 200, range(200)) for x in (k, v))
        if b == 0:
            low = torch.isinf(kk[:, 0, 0])
            want0 = O.attend(q[b, :1].double(), kk[~low][:, :1], vv[~low][:, :1], 0.125)
            assert O.far(out[b, :1], want0[0], want0[2], dtype) <= 1.0
        elif b < 4:
            assert bool(torch.isnan(out[b, 0]).all()), b
        want = O.attend(q[b, 1:].double(), kk[:, 1:], vv[:, 1:], 0.125)
        assert O.far(out[b, 1:], want[0], want[2], dtype) <= 1.0
    cache.check()


@pytest.mark.parametrize("dtype", [F16, F32, E4M3])
def test_attend_equal_scores_and_infinite_values(dtype):
    """An infinity or NaN among the values that do take part is in the result, one behind the end is not."""
    n = 37
    cache, table, (k, v), (ke, ve), t = make([n, n], 1, 64, 16, dtype, seed=2)
    if dtype != E4M3:
        cache.v[int(t[1, 1]), 0, 3, 5] = math.inf
        cache.v[int(t[1, 1]), 0, 3, 6] = math.nan
        cache.v[int(t[1, 1]), 0, 3, 7] = -math.inf
    else:
        cache.v.view(torch.uint8)[int(t[1, 1]), 0, 3, 5:8] = 0x7f
    qd = F16 if dtype == E4M3 else dtype
    out = cache.attend(queries(2, 1, 64, qd, 2).to(DEV), table, torch.full((2,), n, dtype=torch.int32, device=DEV))
    assert bool(torch.isfinite(out[0]).all())
    row = out[1, 0]
    assert bool(torch.isfinite(row[:5]).all()) and bool(torch.isfinite(row[8:]).all()) and not bool(torch.isfinite(row[5:8]).any())


def test_attend_in_place_strided_out_and_rows_behind():
    cache, table, _, _, _ = make([30, 0, 77], 2, 64, 16, F16, seed=6)
    lens = torch.tensor([30, 0, 77], dtype=torch.int32, device=DEV)
    q = queries(3, 4, 64, F16, 6).to(DEV)
    want = cache.attend(q, table, lens)
    big = torch.full((5, 6, 80), 3.0, dtype=F16, device=DEV)
    view = big[1:4, 1:5, 8:72]
    got = cache.attend(q, table, lens, out=view)
    assert got is view and torch.equal(view, want)
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[1:4, 1:5, 8:72] = False
    assert bool((big[mask] == 3.0).all())
    inplace = q.clone()
    cache.attend(inplace, table, lens, out=inplace)
    assert torch.equal(inplace, want)
    # an odd number of values between the heads' rows: neither side is 16-byte aligned
    odd = torch.zeros((3, 4, 65), dtype=F16, device=DEV)
    odd[..., 1:] = q
    res = torch.zeros((3, 4, 65), dtype=F16, device=DEV)
    cache.attend(odd[..., 1:], table, lens, out=res[..., 1:])
    assert torch.equal(res[..., 1:], want) and bool((res[..., 0] == 0).all())


def test_empty_calls():
    cache, table, _, _, _ = make([5], 2, 64, 16, F16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert cache.attend(torch.zeros((0, 2, 64), dtype=F16, device=DEV), table[:0], none).shape == (0, 2, 64)
    rows = torch.zeros((0, 2, 64), dtype=F16, device=DEV)
    before = cache.k.clone()
    cache.append(rows, rows, table, none)
    k, v = cache.gather(table, none)
    assert k.shape == v.shape == (0, 2, 64)
    assert torch.equal(cache.k.view(torch.int16), before.view(torch.int16))


# ----------------------------------------------------------------------------------------------------------------------
# writing and reading
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("width", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_append_and_gather(q_dtype, dtype, width):
    page, heads, lengths, new = 7, 3, [0, 1, 13, 20], [5, 1, 0, 16]
    cache, table, (k, v), (ke, ve), t = make([a + b for a, b in zip(lengths, new)], heads, width, page, dtype, seed=width, junk=False)
    before = [x.clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8))]
    seq = [b for b, n in enumerate(new) for _ in range(n)]
    pos = [lengths[b] + i for b, n in enumerate(new) for i in range(n)]
    perm = np.random.RandomState(width).permutation(len(seq))
    seq, pos = [seq[i] for i in perm], [pos[i] for i in perm]
    g = torch.Generator().manual_seed(width)
    wide = (torch.randn((len(seq) + 2, 2 * heads + 1, width), generator=g) * torch.exp(torch.randn((len(seq) + 2, 1, 1), generator=g) * 3)).to(q_dtype).to(DEV)
    nk, nv = wide[:-2, :heads], wide[:-2, heads:2 * heads]
    st, pt = torch.tensor(seq + [0, 1], dtype=torch.int32, device=DEV)[:-2], torch.tensor(pos + [0, 0], dtype=torch.int32, device=DEV)[:-2]
    cache.append(nk, nv, table, pt, sequences=st)
    k2, v2 = cache.gather(table, pt, sequences=st, dtype=q_dtype)
    for new_rows, got in ((nk, k2), (nv, v2)):
        if dtype == E4M3:
            code, e = O.quantise(new_rows.float().cpu())
            want = (code * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 127).double())[..., None]).to(q_dtype)
            assert torch.equal(got.cpu().double(), want.double())
        else:
            assert torch.equal(got, new_rows)
    touched = torch.zeros((cache.n_pages, page), dtype=torch.bool, device=DEV)
    for s, p in zip(seq, pos):
        touched[int(t[s, p // page]), p % page] = True
    for x, old in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8)), before):
        same = (x == old).reshape(cache.n_pages, heads, page, -1).all(-1).all(1)
        assert bool((same | touched).all()), "a slot that no row names was written"
    cache.check()


def test_quantising_at_its_borders():
    """Rows whose largest value sits on and beside 448 2^E, codes halfway between two, values below the least code, zeros,
    subnormal numbers of float32, infinities and NaN."""
    rng = np.random.RandomState(0)
    rows = []
    for E in (-140, -126, -20, -1, 0, 3, 100, 118, 119):
        for f in (448.0, np.nextafter(np.float32(448), np.float32(0)), np.nextafter(np.float32(448), np.float32(999)), 1.0, 447.0, 225.0):
            r = rng.uniform(-1, 1, 64) * float(f)
            r[0] = float(f)
            r[1:9] = [2.0 ** -10, 1.5 * 2.0 ** -9, 2.5 * 2.0 ** -9, 17.0, 19.0, 2.0 ** -9, -(2.0 ** -10), -26.0]
            rows.append(r * 2.0 ** E)
    rows.append(np.zeros(64))
    rows = np.clip(np.array(rows), -3.4e38, 3.4e38).astype(np.float32)
    special = np.tile(rows[10], (4, 1))
    special[0, 5], special[1, 5], special[2, 5] = np.inf, -np.inf, np.nan
    special[3] = np.nan
    x = torch.from_numpy(np.concatenate([rows, special])).reshape(-1, 1, 64)
    from whisper_timestamped import PagedKVCache
    cache = PagedKVCache.allocate(9, 1, 64, 8, dtype=E4M3, device=DEV)
    n = x.shape[0]
    table = torch.arange(9, dtype=torch.int32, device=DEV)[None]
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    seq = torch.zeros(n, dtype=torch.int32, device=DEV)
    cache.append(x.to(DEV), (-x).to(DEV), table, pos, sequences=seq)
    code, e = O.quantise(x)
    got = cache.k.reshape(72, 64)[:n].float().cpu().double()
    assert torch.equal(cache.k_exp.reshape(72)[:n].cpu().long(), e[:, 0])
    assert torch.equal(torch.isnan(got), torch.isnan(code[:, 0]))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(code[:, 0]))
    k, v = cache.gather(table, pos, sequences=seq)
    assert k.dtype == F32 and torch.equal(torch.nan_to_num(k), torch.nan_to_num(-v))


def test_padded_rows_and_out_of_range():
    from whisper_timestamped import PagedKVCache
    from whisper_timestamped._lib import WtError
    cache, table, (k, v), _, t = make([20, 20, 20], 2, 64, 8, F16, seed=8, junk=False)
    before = cache.k.clone(), cache.v.clone()
    rows = torch.ones((6, 2, 64), dtype=F16, device=DEV)
    width = table.shape[1]
    bad_pos = torch.tensor([-1, width * 8, 2 ** 31 - 1, -5, 24, 3], dtype=torch.int32, device=DEV)   # 24: in an entry that names no page
    seq = torch.tensor([0, 1, 2, 0, 1, 3], dtype=torch.int32, device=DEV)                                # 3: no such sequence
    cache.append(rows, rows, table, bad_pos, sequences=seq)
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    with pytest.raises(WtError, match="position.*page.*sequence"):
        cache.check()
    cache.check()
    gk, gv = cache.gather(table, bad_pos, sequences=seq)
    for x in (gk, gv):
        assert bool((x[[0, 3]] == 0).all()) and bool(torch.isnan(x[[1, 2, 4, 5]]).all())
    with pytest.raises(WtError):
        cache.check()
    assert isinstance(PagedKVCache, type)


@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_attend_bad_pages_and_lengths(q_dtype, dtype):
    """A sequence with a bad length or page gives NaN and raises in check(); its neighbours are right."""
    from whisper_timestamped._lib import WtError
    lengths = [40, 700, 40, 40, 40, 700]
    cache, table, _, _, t = make(lengths, 2, 64, 16, dtype, seed=11)
    q = queries(6, 4, 64, q_dtype, 11).to(DEV)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = cache.attend(q, table, lens)
    cache.check()
    bad_table, bad_lens = table.clone(), lens.clone()
    bad_table[1, 30] = cache.n_pages
    bad_table[2, 0] = -1
    bad_lens[3] = table.shape[1] * 16 + 1
    bad_lens[4] = -2
    got, lse = cache.attend(q, bad_table, bad_lens, return_lse=True)
    assert bool(torch.isnan(got[1:5]).all()) and bool(torch.isnan(lse[1:5]).all())
    assert torch.equal(got[0], want[0]) and torch.equal(got[5], want[5])
    with pytest.raises(WtError, match="position.*page"):
        cache.check()
    assert torch.equal(cache.attend(q, table, lens), want)
    cache.check()


# ----------------------------------------------------------------------------------------------------------------------
# together, as a decoder uses them
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_dtype,dtype", PAIRS)
def test_decoder_steps(q_dtype, dtype):
    """Prompts of different lengths, then token after token, sequences ending at different steps: every step against
    attention in 64 bits over what the cache gives back."""
    from whisper_timestamped import PagedKVCache
    B, H, G, W, page, steps = 5, 2, 2, 64, 8, 12
    cache = PagedKVCache.allocate(40, H, W, page, dtype=dtype, device=DEV)
    ids = np.random.RandomState(3).permutation(40).reshape(B, 8).astype(np.int32)
    table = torch.from_numpy(ids).to(DEV)
    prompts = [3, 8, 0, 17, 1]
    g = torch.Generator().manual_seed(2)

    def new(n, heads):
        return torch.randn((n, heads, W), generator=g).to(q_dtype)

    seq = [b for b, n in enumerate(prompts) for _ in range(n)]
    pos = [i for n in prompts for i in range(n)]
    k, v = new(len(seq), H), new(len(seq), H)
    cache.append(k.to(DEV), v.to(DEV), table, torch.tensor(pos, dtype=torch.int32, device=DEV), sequences=torch.tensor(seq, dtype=torch.int32, device=DEV))
    lengths = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    for step in range(steps):
        alive = torch.tensor([step < 4 * (b + 1) for b in range(B)], device=DEV)
        q, k, v = new(B, H * G), new(B, H), new(B, H)
        cache.append(k.to(DEV), v.to(DEV), table, torch.where(alive, lengths, -1).int())
        lengths += alive.int()
        out = cache.attend(q.to(DEV), table, lengths)
        cache.check()
        for b, n in enumerate(lengths.tolist()):
            kk, vv = cache.gather(table, torch.arange(n, dtype=torch.int32, device=DEV), sequences=torch.full((n,), b, dtype=torch.int32, device=DEV), dtype=q_dtype)
            if alive[b]:
                want = k[b].double()
                if dtype == E4M3:
                    code, e = O.quantise(k[b].float())
                    want = (code * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 127).double())[..., None]).to(q_dtype).double()
                assert torch.equal(kk[-1].double().cpu(), want)
            want, _, bound, _ = O.attend(q[b].double(), kk.double().cpu(), vv.double().cpu(), W ** -0.5)
            assert O.far(out[b], want, bound, q_dtype) <= 1.0, (step, b)


@pytest.mark.parametrize("long", [False, True])
def test_captured_step_follows_its_tensors(long):
    """append + attend captured once and replayed with other tokens and lengths, eager work between the replays; two graphs
    over two caches replayed at the same time on two streams."""
    from whisper_timestamped import PagedKVCache
    n0 = 6000 if long else 50
    made = [make([n0, n0 // 2, 1], 2, 64, 16, F16, seed=20 + i, spare=8) for i in range(2)]
    graphs = []
    for cache, table, _, _, _ in made:
        q, k, v = (torch.zeros((3, h, 64), dtype=F16, device=DEV) for h in (4, 2, 2))
        lens = torch.tensor([n0 - 9, n0 // 2 - 9, 0], dtype=torch.int32, device=DEV)
        out = torch.zeros_like(q)
        static = dict(q=q, k=k, v=v, lens=lens, out=out)

        def step(cache=cache, table=table, s=static):
            cache.append(s["k"], s["v"], table, s["lens"])
            cache.attend(s["q"], table, s["lens"] + 1, out=s["out"])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, static, step))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        want = []
        for i, (graph, s, step) in enumerate(graphs):
            for x in ("q", "k", "v"):
                h = s[x].shape[1]
                s[x].copy_(queries(3, h, 64, F16, 100 * turn + 10 * i + h).to(DEV))
            s["lens"].add_(1)
            step()
            torch.cuda.synchronize()
            want.append(s["out"].clone())
            s["out"].zero_()
        torch.cuda.synchronize()
        for (graph, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, s, _), w in zip(graphs, want):
            assert torch.equal(s["out"], w)
    for m in made:
        m[0].check()
    assert isinstance(PagedKVCache, type)


def test_two_streams_at_once():
    """The same cache read on two streams at the same time, many times over."""
    lengths = [5000, 17, 900, 2500]
    cache, table, _, _, _ = make(lengths, 2, 128, 32, BF16, seed=30)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    qs = [queries(4, 8, 128, BF16, 40 + i).to(DEV) for i in range(2)]
    want = [cache.attend(q, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(cache.attend(qs[i], table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_offsets_beyond_32_bits():
    """Pages behind the 2^32nd byte and element of a cache."""
    from whisper_timestamped import PagedKVCache
    n_pages = (2 ** 32) // (8 * 64 * 128) + 16
    cache = PagedKVCache.allocate(n_pages, 8, 128, 64, dtype=E4M3, device=DEV)
    table = torch.tensor([[n_pages - 1, n_pages // 2 + 3, 0, n_pages - 2]], dtype=torch.int32, device=DEV)
    n = 250
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn((m, 8, 128), generator=g).to(BF16) for m in (n, n, 1))
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    seq = torch.zeros(n, dtype=torch.int32, device=DEV)
    cache.append(k.to(DEV), v.to(DEV), table, pos, sequences=seq)
    kk, vv = cache.gather(table, pos, sequences=seq)
    code, e = O.quantise(k.float())
    assert torch.equal(kk.cpu().double(), code * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 127).double())[..., None])
    out = cache.attend(q.to(DEV), table, torch.tensor([n], dtype=torch.int32, device=DEV))
    want, _, bound, _ = O.attend(q[0].double(), kk.double().cpu(), vv.double().cpu(), 128 ** -0.5)
    assert O.far(out[0], want, bound, BF16) <= 1.0
    cache.check()


# ----------------------------------------------------------------------------------------------------------------------
# the path that calls it: B decoder streams with their text in paged caches
# ----------------------------------------------------------------------------------------------------------------------
def test_streams_over_paged_caches_match_the_reference(monkeypatch):
    """transcribe_batch with streams.PAGED_SELF_ATTENTION: ragged prompts, several windows, every recording against the
    reference's own output at the bars of the concatenated cache; every layer of every call goes through the caches, and
    the backend is as it was afterwards."""
    from test_gpu_streams_batch import _check_against_reference
    from test_streams_host import run_batch, same_model_cases
    from whisper_timestamped import PagedKVCache, streams
    calls = {"append": 0, "attend": 0}
    for name in calls:
        def counted(self, *a, _f=getattr(PagedKVCache, name), _n=name, **kw):
            calls[_n] += 1
            return _f(self, *a, **kw)
        monkeypatch.setattr(PagedKVCache, name, counted)
    monkeypatch.setattr(streams, "PAGED_SELF_ATTENTION", True)
    cases = same_model_cases() + same_model_cases()[::-1]
    for raw, case in zip(run_batch(cases, device="cuda:0"), cases):
        _check_against_reference(raw, case)
    assert calls["attend"] > 50 and calls["append"] > calls["attend"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_paged_decoder_against_the_backends_own(dtype):
    """The decoder's logits call by call, over paged caches and over the backend's concatenated ones."""
    import whisper_double as W
    from whisper_double.model import build_model
    from whisper_timestamped.paged_decoder import PagedText, supported
    W.install()
    model = build_model("tiny", device="cuda:0")             # (its modules cast their weights to the activations)
    assert supported(model, dtype)
    g = torch.Generator().manual_seed(0)
    feats = torch.randn((3, 1500, 384), generator=g).to(dtype).cuda()
    prompt = torch.randint(0, 50000, (3, 11), generator=g).cuda()
    steps = torch.randint(0, 50000, (3, 40), generator=g).cuda()

    def logits():
        cache, hooks = model.install_kv_cache_hooks()
        try:
            with torch.no_grad():
                out = [model.decoder(prompt, feats, kv_cache=cache)[:, -1:]]
                for i in range(steps.shape[1]):
                    out.append(model.decoder(steps[:, i:i + 1], feats, kv_cache=cache))
        finally:
            for h in hooks:
                h.remove()
        return torch.cat(out, 1)

    want = logits()
    text = PagedText(model, 4, dtype)
    for _ in range(2):                                   # (a second loop starts from empty caches)
        with text.attached():
            got = logits()
        # attention in 32 bits against the backend's in the model's type: layer by layer a few roundings of the residual
        # stream apart, 4 layers, logits of standard deviation ~ 10; f32 2^-24, f16 2^-11 a rounding
        tol = (1e-3 if dtype == torch.float32 else 0.5)
        assert float((got - want).abs().max()) <= tol
    assert "forward" not in vars(model.decoder.blocks[0].attn) and "install_kv_cache_hooks" not in vars(model)
    assert torch.equal(logits(), want)
    for c in text.caches:
        c.check()
    from whisper_timestamped._lib import WtError
    with text.attached(), pytest.raises(WtError, match="room for 4"):
        model.decoder(prompt[:1].repeat(5, 1), feats[:1].repeat(5, 1, 1), kv_cache=model.install_kv_cache_hooks()[0])
