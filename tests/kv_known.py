"""TEST INFRASTRUCTURE: attention over a paged cache with results that are known without a kernel's order of sums, and the shapes that
take every schedule the library has.  Shares no code with the package."""
import torch

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, E4M3), (F16, E4M3), (BF16, E4M3)]
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
RUN = 16          # keys in a row that count for one column: no wave takes fewer at a time
BLOCK = 32        # keys in a row that hold one peak
PEAK = 20.0


# ----------------------------------------------------------------------------------------------------------------------
# counting: all scores zero, so every weight is exactly 1; the values of RUN keys in a row are 1 in one column of the head and
# 0 elsewhere, so a result is a count over the length: whole numbers below 2^24 and one quotient, known to the last bit
# ----------------------------------------------------------------------------------------------------------------------
def counting_values(n, heads, width):
    v = torch.zeros((n, heads, width))
    t, h = torch.arange(n)[:, None], torch.arange(heads)[None]
    v[t, h, (t // RUN + 5 * h) % width] = 1.0
    return v


def counted(v, length, dtype, without=None, twice=None):
    """(heads, width) in `dtype`: without / twice: the mistake of leaving out, or taking twice, RUN keys from there on."""
    weight = torch.ones(v.shape[0])
    weight[length:] = 0
    if without is not None:
        weight[without:without + RUN] = 0
    if twice is not None:
        weight[twice:min(twice + RUN, length)] = 2
    total = weight.sum()
    return ((weight[:, None, None] * v).sum(0) / total).to(dtype), total


# ----------------------------------------------------------------------------------------------------------------------
# peaks: one key of every BLOCK scores PEAK with the queries of one column, all others score 0
# ----------------------------------------------------------------------------------------------------------------------
def peaked(n, heads, width, dtype, seed=0):
    """keys, values (n, heads, width), exact in `dtype`, and the column that each key peaks for (-1: none)."""
    g = torch.Generator().manual_seed(seed)
    k, at = torch.zeros((n, heads, width)), torch.full((n,), -1)
    for b in range(0, n, BLOCK):
        p = b + int(torch.randint(0, min(BLOCK, n - b), (1,), generator=g))
        at[p] = b // BLOCK % width
        k[p, :, at[p]] = 1.0
    v = torch.rand((n, heads, width), generator=g) * 2 - 1
    return k, (v * 8).round() / 8 if dtype == E4M3 else v.to(dtype).float(), at


def peak_queries(seqs, heads, group, width, dtype):
    """(seqs, heads * group, width): query j of sequence s peaks in column (s * group + j) % width; and the columns."""
    c = (torch.arange(seqs)[:, None] * group + torch.arange(group)[None]) % width
    q = torch.zeros((seqs, heads, group, width))
    for j in range(group):
        q[torch.arange(seqs), :, j, c[:, j]] = PEAK
    return q.reshape(seqs, heads * group, width).to(dtype), c


def peak_results(v, at, length, columns, dtype, depth, without=None):
    """(heads, columns, width) float64 and what each may be off by, given the longest chain of sums: a weight 2^-24 times 1.5 for
    every unit of its exponent's distance (PEAK, and the 8 that the reference may lag) and 16 for exponentials and moves of the
    reference, twice (also in the sum below the line), 2^-17 for its 16-bit parts where results have 16 bits; `depth` roundings above
    and below the line; half a step for the result."""
    w = torch.where(at[:length, None] == columns[None], float(torch.exp(torch.tensor(PEAK, dtype=torch.float64))), 1.0).double()      # (length, columns)
    if without is not None:
        w[without:without + RUN] = 0
    x = v[:length].double()
    total = w.sum(0)[None, :, None]
    out = torch.einsum("tc,thd->hcd", w, x) / total
    size = torch.einsum("tc,thd->hcd", w, x.abs()) / total
    off = size * (2.0 ** -24 * (2 * (1.5 * (PEAK + 8) + 16) + 2 * depth) + (2.0 ** -17 if dtype != F32 else 0.0))
    return out, off + HALF_STEP[dtype] * (out.abs() + off) + (2.0 ** -25 if dtype == F16 else 0.0)


# ----------------------------------------------------------------------------------------------------------------------
# shapes and the schedule that each is there for: (whole, waves, tiles of 16 queries), on 256 compute units
# ----------------------------------------------------------------------------------------------------------------------
class Shape:
    def __init__(self, name, q_dtype, dtype, width, page, heads, group, lengths, columns, whole, waves, tiles, parts=0):
        self.name, self.q_dtype, self.dtype, self.width, self.page, self.heads, self.group = name, q_dtype, dtype, width, page, heads, group
        self.lengths, self.columns = list(lengths), columns      # columns: of the table, which may be wider than its longest row
        self.whole, self.waves, self.tiles, self.parts = whole, waves, tiles, parts       # parts: that the longest pair falls into, at least

    def __repr__(self):
        return self.name

    def key_bytes(self):
        return 2 * self.width * {F32: 4, E4M3: 1}.get(self.dtype, 2)

    def unit(self):
        return 4 * (16 if self.dtype == F32 else 32)

    def share(self, cus=256):
        """Units of a workgroup where tables are split: an equal part of all, each pair with two for itself."""
        pairs = self.heads * -(-self.group // (16 * self.tiles))
        total = pairs * sum(-(-n // self.unit()) + 2 for n in self.lengths)
        return max(2 if self.unit() * self.key_bytes() < 32 * 1024 else 1, -(-total // cus))

    def depth(self):
        """Roundings in the longest chain of sums: up to 3 products of 32 keys each for every block of a wave, of the weights 8, and the
        joins of waves and parts."""
        blocks = max(-(-n // (self.unit() // 4 * self.waves)) for n in self.lengths) if self.whole else self.share()
        return 3 * blocks + 96 + 8 * blocks + 4 + (0 if self.whole else 3 * 16 + 64)


def shapes():
    out = []
    name = {F32: "f32", F16: "f16", BF16: "bf16", E4M3: "e4m3"}
    for q, d in PAIRS:
        tag = name[q] if q == d else f"{name[d]}_{name[q]}"
        key = lambda width: 2 * width * {F32: 4, E4M3: 1}.get(d, 2)  # noqa: E731
        block = 16 if d == F32 else 32
        for width in (32, 64, 96, 128):
            # more than 16 queries a key head, whole tables, enough of them to fill the card; 96 and 128 values of fewer than 32 bits: tables of 128 KB
            page = {32: 8, 64: 32, 96: 7, 128: 16}[width]
            most = 128 * 1024 // (key(width) * page) + 2 if width > 64 and d != F32 else 0
            out.append(Shape(f"whole_wide_{tag}_{width}", q, d, width, page, 2, {32: 17, 64: 24, 96: 32, 128: 40}[width],
                             [(i * 37) % 250 if i % 5 else 0 for i in range(150)], max(most, -(-250 // page) + 1), True, 4, 2))
            # the same over a split table: all of one sequence's 157 and more parts meet in three levels of joins
            unit = block * 4
            least = 2 if unit * key(width) < 32 * 1024 else 1
            n = 157 * unit * least - 5
            page = {32: 16, 64: 64, 96: 24, 128: 100}[width]
            out.append(Shape(f"split_wide_{tag}_{width}", q, d, width, page, 1, {32: 32, 64: 17, 96: 24, 128: 20}[width], [n, 0, 1][:1 + 2 * (width == 64)],
                             64 * 1024 * 1024 // (key(width) * page) + 1, False, 4, 2, 157))
        for width in (32, 64, 96, 128, 256):
            # enough heads to fill the card: workgroups of two waves
            seqs = {F32: 100, E4M3: 200}.get(d, 40)
            page = {32: 32, 64: 8, 96: 64, 128: 5, 256: 16}[width]
            out.append(Shape(f"two_waves_{tag}_{width}", q, d, width, page, 16, 1, [(i * 29) % 200 for i in range(seqs)], -(-200 // page) + 1, True, 2, 1))
            # few heads over a long table: 40 and more parts, two levels of joins (16 queries and fewer a key head)
            unit, least = block * 4, 2 if block * 4 * key(width) < 32 * 1024 else 1
            n = 45 * unit * least + 3
            page = {32: 10, 64: 32, 96: 8, 128: 64, 256: 24}[width]
            out.append(Shape(f"split_{tag}_{width}", q, d, width, page, 1, {32: 16, 64: 1, 96: 9, 128: 5, 256: 12}[width], [n], max(-(-n // page), 512 * 1024 // (key(width) * page) + 1), False, 4, 1, 45))
    return out
