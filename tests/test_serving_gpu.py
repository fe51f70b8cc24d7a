"""Serving operators on device buffers against their definitions in 64 bits.

Tolerances, with u = half a step of a type relative to a value (FP32 2^-24, BF16 2^-8, e4m3 2^-4):
 * attention, |v| <= V, scores within +-16 in the tests: an FP32 score is off by a few u of its size, 16 * 2^-20 in all with the pairs' rests
   (2^-22) and the sum over the entries, which is the relative error of a weight; the weighted mean is off by twice that times V: 2^-15 V.
   BF16 queries: weights rounded to FP16 (2^-11 of the largest weight each, in numerator only): 2^-10 V, and the result's own rounding.
 * 4-bit products: operands are exact (FP32: within 2^-21 of the tile's largest input), sums FP32: 2^-18 sum |x w|, and the result's rounding.
 * log probabilities: FP32 sums and logarithms, values up to 40 or so: 2^-18 * (1 + |value|).
"""
import math

import pytest
import torch

import puppygrad_b200 as pg
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return i32(out)


class Cache:
    """A pool with codes of earlier tokens; bytes and scales that no live token owns are 0xFF, NaN."""

    def __init__(self, lens, kvh, dim, page, seed, spread=2, spare=3, per_seq=None):
        g = gen(seed)
        used = [-(-n // page) for n in lens]
        self.page, self.dim, self.kvh, self.lens = page, dim, kvh, lens
        n_pages, per_seq = sum(used) + spare, per_seq or max(1, max(used)) + 1
        self.pool = torch.full(pg.Kv8Cache.pool_shape(n_pages, kvh, page, dim), 255, dtype=torch.uint8, device=DEV)
        self.scales = torch.full((n_pages, kvh, 2), math.nan, device=DEV)
        self.table = torch.full((len(lens), per_seq), -1, dtype=torch.int32, device=DEV)
        order, at = torch.randperm(n_pages, generator=g, device=DEV).tolist(), 0
        k, v = ref.blocks(self.pool, page, dim)
        for b, n in enumerate(lens):
            for i in range(used[b]):
                p, live = order[at], min(page, n - i * page)
                at += 1
                self.table[b, i] = p
                values = (torch.randn(2, kvh, live, dim, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                k[p, :, :live] = 0
                k[p, :, :live, :dim] = values[0]
                v[p, :, :dim, :live] = values[1].transpose(-1, -2)
                self.scales[p] = torch.exp2(torch.randint(-8, -8 + spread, (kvh, 2), generator=g, device=DEV).float())
        self.handle = pg.Kv8Cache(self.pool, self.scales, self.table, page_tokens=page, head_dim=dim)

    def kv(self, b, length=None):
        return ref.sequence_kv(self.pool, self.scales, self.table[b], self.lens[b] if length is None else length, self.page, self.dim)


def workspace(cache, rows, heads, dtype):
    return torch.zeros(cache.handle.workspace_bytes(rows, heads, dtype), dtype=torch.uint8, device=DEV)


def check_attention(cache, q, out, rows, scale, window=0, keep=0):
    at = 0
    for b, n in enumerate(rows):
        length = cache.lens[b]
        keys, values = cache.kv(b)
        want = ref.attention(q[at:at + n].double(), keys, values, torch.arange(length - n, length, device=DEV), scale, window, keep)
        got, u = out[at:at + n].double(), U[q.dtype]
        top = float(values.abs().max()) if length else 0.0
        tol = top * (2.0 ** -15 if q.dtype == F32 else 2.0 ** -10) + u * want.abs()
        assert torch.isfinite(got).all(), (b, n, length)
        assert ((got - want).abs() <= tol).all(), (b, n, length, float(((got - want).abs() - tol).max()), top)
        at += n


ATTENTION = [
    # lens, rows, heads, kv heads, dim, page, window, keep
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([777], [1], 12, 12, 64, 32, 0, 0),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500], [1] * 16, 8, 2, 64, 16, 0, 0),
    ([0, 1, 16, 63, 64, 65, 129, 1000], [1] * 8, 10, 2, 96, 32, 0, 0),
    ([300, 1, 64, 2000], [1] * 4, 32, 2, 128, 64, 0, 0),
    ([130, 70], [1, 1], 48, 2, 80, 64, 0, 0),  # 24 rows for a head: more than a tile
    ([5000], [1], 4, 1, 256, 64, 0, 0),
    ([333, 90], [1, 1], 6, 3, 192, 16, 0, 0),
    ([40, 70], [1, 1], 3, 3, 2, 16, 0, 0),
    ([700, 64, 0, 130], [5, 64, 0, 3], 8, 2, 128, 64, 0, 0),
    ([200, 3, 90], [7, 5, 1], 4, 4, 32, 32, 0, 0),  # more rows than tokens: the first see nothing
    ([1000, 100, 64, 10], [1] * 4, 8, 4, 64, 64, 50, 0),
    ([1000, 300, 64, 10], [3, 200, 64, 2], 8, 4, 64, 16, 100, 70),
    ([1000, 131], [1, 60], 4, 1, 128, 32, 1, 0),  # each row sees itself alone
    ([900], [1], 4, 4, 64, 64, 1000, 5),
    # many rows of a sequence
    ([500, 260, 3], [300, 260, 1], 6, 2, 96, 32, 0, 0),
    ([300], [129], 2, 2, 256, 64, 0, 0),
    ([200], [200], 5, 1, 192, 16, 0, 0),
    ([70, 1000], [70, 65], 16, 1, 64, 64, 0, 0),
    ([50, 0, 64], [200, 100, 128], 2, 2, 128, 16, 0, 0),  # more rows than tokens, and rows of an empty sequence
    ([1500, 90], [700, 1], 4, 2, 80, 64, 333, 70),
    ([600], [600], 3, 1, 2, 32, 5, 0),
    ([777, 512], [500, 512], 8, 8, 64, 64, 0, 0),
    # ... few of them, far into a sequence: cut along the positions
    ([9000], [130], 2, 1, 128, 64, 0, 0),
    ([5000], [70], 4, 2, 64, 32, 0, 0),
    ([4100], [200], 1, 1, 256, 64, 0, 0),
    ([6000, 300], [40, 35], 4, 1, 96, 16, 3000, 100),
    ([2100], [90], 3, 1, 192, 64, 0, 0),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,rows,heads,kvh,dim,page,window,keep", ATTENTION)
def test_attention(lens, rows, heads, kvh, dim, page, window, keep, dtype):
    cache = Cache(lens, kvh, dim, page, 11 + sum(lens))
    n, scale = sum(rows), dim ** -0.5
    q = torch.randn(n, heads, dim, generator=gen(3), device=DEV).to(dtype)
    out = torch.full((n + 2, heads, dim), 7.0, device=DEV, dtype=dtype)  # two rows behind the last sequence
    ws = workspace(cache, n, heads, dtype)
    one = all(r == 1 for r in rows)
    for call in range(2):  # the workspace is left as it was
        cache.handle.attention(q, out[:n], i32(lens), ws, row_start=None if one else starts(rows), max_rows=max(rows), window=window, keep_first=keep)
        check_attention(cache, q, out[:n], rows, scale, window, keep)
    assert (out[n:] == 7).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long_sequences_are_shared_out_over_all_blocks(dtype):
    lens = [70001, 3, 20000]
    cache = Cache(lens, 2, 64, 64, 5)
    q = torch.randn(3, 8, 64, generator=gen(4), device=DEV).to(dtype)
    out, ws = torch.empty_like(q), workspace(cache, 3, 8, dtype)
    cache.handle.attention(q, out, i32(lens), ws)
    check_attention(cache, q, out, [1, 1, 1], 64 ** -0.5)
    again = torch.empty_like(q)
    cache.handle.attention(q, again, i32(lens), ws)
    assert torch.equal(out, again)  # the order of the parts is fixed


def test_attention_many_sequences():
    lens = [(i * 37) % 90 for i in range(700)]
    cache = Cache(lens, 1, 64, 16, 6)
    q = torch.randn(700, 2, 64, generator=gen(4), device=DEV)
    out = torch.empty_like(q)
    cache.handle.attention(q, out, i32(lens), workspace(cache, 700, 2, F32))
    check_attention(cache, q, out, [1] * 700, 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_blocks_of_very_different_scales(dtype):
    """The largest weight may belong to a block whose values are 2^40 times smaller than another block's."""
    cache = Cache([256], 1, 64, 64, 8)
    cache.scales[cache.table[0, 0].long()] = torch.tensor([2.0 ** -7, 2.0 ** -45], device=DEV)
    cache.scales[cache.table[0, 2].long()] = torch.tensor([0.0, 2.0 ** -100], device=DEV)
    q = torch.randn(1, 4, 64, generator=gen(9), device=DEV).to(dtype)
    keys, values = cache.kv(0)
    q[0, 0] = (keys[5, 0] * 8).to(dtype)  # head 0 looks at a token of the first block alone
    out = torch.empty_like(q)
    cache.handle.attention(q, out, i32([256]), workspace(cache, 1, 4, dtype))
    check_attention(cache, q, out, [1], 0.125)
    q2 = q[:, :1].contiguous()
    out2 = torch.empty_like(q2)
    cache.handle.attention(q2, out2, i32([40]), workspace(cache, 1, 1, dtype))  # the first block alone: tiny values, whole precision
    want = ref.attention(q2.double(), keys[:40], values[:40], torch.tensor([39], device=DEV), 0.125)
    assert ((out2.double() - want).abs() <= (2.0 ** -15 if dtype == F32 else 2.0 ** -10) * values[:40].abs().max() + U[dtype] * want.abs()).all()


def test_attention_pages_that_are_none_and_lengths_beyond_the_table():
    cache = Cache([300, 200], 2, 64, 32, 12)
    cache.table[0, 3] = -1
    cache.table[0, 4] = 10 ** 6
    q = torch.randn(2, 4, 64, generator=gen(1), device=DEV)
    out, ws = torch.empty_like(q), workspace(cache, 2, 4, F32)
    lens = i32([300, 10 ** 6])
    cache.handle.attention(q, out, lens, ws)
    table = cache.table.clone()
    cache.table.clamp_(0, cache.pool.shape[0] - 1)
    keys, values = cache.kv(0)
    gone = (torch.arange(300, device=DEV) >= 96) & (torch.arange(300, device=DEV) < 160)
    want = ref.attention(q[:1].double(), keys, values, torch.tensor([299], device=DEV), 0.125, missing=gone)
    assert ((out[:1].double() - want).abs() <= 2.0 ** -15 * values.abs().max() + 2.0 ** -24 * want.abs()).all()
    # of the second sequence the table's pages are seen, all but those that are none
    known = int((table[1] >= 0).sum()) * 32
    assert known == 224
    keys, values = cache.kv(1, known)  # tokens 200..223 of the last page hold NaN bytes: they count as stored
    assert torch.isnan(values).any() and torch.isnan(out[1]).any()


def test_attention_rows_outside_every_sequence_are_left():
    cache = Cache([50, 60], 1, 64, 16, 2)
    q = torch.randn(9, 2, 64, generator=gen(1), device=DEV)
    out, ws = torch.full_like(q, 5.0), workspace(cache, 9, 2, F32)
    cache.handle.attention(q, out, i32([50, 60]), ws, row_start=i32([2, 4, 7]), max_rows=3)
    assert (out[:2] == 5).all() and (out[7:] == 5).all()
    check_attention(cache, q[2:7], out[2:7], [2, 3], 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_rows_with_gaps_and_odd_addresses(dtype):
    cache = Cache([500, 77], 2, 80, 16, 21)
    wide = torch.randn(2, 4 * 80 + 13, generator=gen(2), device=DEV).to(dtype)
    q = wide[:, 3:3 + 320].view(2, 4, 80)
    big = torch.full((2, 4 * 80 + 7), 9.0, device=DEV, dtype=dtype)
    out = big[:, 1:321].view(2, 4, 80)
    cache.handle.attention(q, out, i32([500, 77]), workspace(cache, 2, 4, dtype))
    check_attention(cache, q, out, [1, 1], 80 ** -0.5)
    assert (big[:, 0] == 9).all() and (big[:, 321:] == 9).all()


@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_attention_queries_far_from_one(size):
    cache = Cache([300], 1, 64, 16, 3)
    q = torch.randn(1, 2, 64, generator=gen(1), device=DEV)
    out, ws = torch.empty_like(q), workspace(cache, 1, 2, F32)
    want = torch.empty_like(q)
    cache.handle.attention(q, want, i32([300]), ws)
    cache.handle.attention(q * size, out, i32([300]), ws, scale=0.125 / size)
    check_attention(cache, q, out, [1], 0.125)


@pytest.mark.parametrize("window,keep", [(2 ** 31 - 1, 0), (2 ** 30, 2 ** 31 - 1), (50, 40), (50, 2 ** 31 - 1), (2 ** 30 - 1, 7)])
@pytest.mark.parametrize("rows", [[1, 3, 2], [90, 3, 70]])
def test_attention_lengths_and_windows_at_the_end_of_32_bits(rows, window, keep):
    """A length beyond the table stands for tokens that are not stored: its rows see those of the table that are in reach."""
    known = [192, 64, 128]
    cache = Cache(known, 2, 64, 64, 31, per_seq=3)
    lens = [2 ** 31 - 1, 64, 2 ** 31 - 1]
    n = sum(rows)
    q = torch.randn(n, 4, 64, generator=gen(4), device=DEV)
    out = torch.full_like(q, 7.0)
    cache.handle.attention(q, out, i32(lens), workspace(cache, n, 4, F32), row_start=starts(rows), max_rows=max(rows), window=window, keep_first=keep)
    at = 0
    for b, r in enumerate(rows):
        keys, values = cache.kv(b)
        # (a window of 2^30 or more, wider than any table, is none)
        want = ref.attention(q[at:at + r].double(), keys, values, torch.arange(lens[b] - r, lens[b], device=DEV), 0.125, window if window < 2 ** 30 else 0, keep)
        assert ((out[at:at + r].double() - want).abs() <= 2.0 ** -15 * values.abs().max() + 2.0 ** -24 * want.abs()).all(), b
        at += r


def test_attention_row_starts_that_decrease_are_without_effect_on_later_calls():
    cache = Cache([50, 60, 40], 1, 64, 16, 2)
    q = torch.randn(9, 2, 64, generator=gen(1), device=DEV)
    out, ws = torch.full_like(q, 5.0), workspace(cache, 9, 2, F32)
    cache.handle.attention(q, out, i32([50, 60, 40]), ws, row_start=i32([0, 9, 2, 9]), max_rows=9)
    assert (out == 5).all() and not ws[:256].any()
    cache.handle.attention(q, out, i32([50, 60, 40]), ws, row_start=i32([0, 3, 5, 9]), max_rows=4)
    check_attention(cache, q, out, [3, 2, 4], 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_more_sequences_than_threads_with_rows_of_all_numbers(dtype):
    rows = [(0, 1, 1, 2, 5, 1, 33, 0, 70)[i % 9] for i in range(1100)]
    lens = [(i * 29) % 120 for i in range(1100)]
    cache = Cache(lens, 1, 64, 32, 13)
    n = sum(rows)
    q = torch.randn(n, 2, 64, generator=gen(6), device=DEV).to(dtype)
    out = torch.full_like(q, 5.0)
    cache.handle.attention(q, out, i32(lens), workspace(cache, n, 2, dtype), row_start=starts(rows), max_rows=70)
    check_attention(cache, q, out, rows, 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_cache_of_more_than_4_gb(dtype):
    """The last pages of a pool whose offsets need 33 bits: append, then both attention kernels."""
    page, kvh, dim = 64, 8, 128
    n_pages = (1 << 32) // (kvh * 2 * page * dim) + 40
    pool = torch.empty(pg.Kv8Cache.pool_shape(n_pages, kvh, page, dim), dtype=torch.uint8, device=DEV)
    assert pool.numel() > 1 << 32
    cache = Cache([0, 0], kvh, dim, page, 3)
    cache.pool, cache.scales = pool, torch.empty(n_pages, kvh, 2, device=DEV)
    cache.table = torch.arange(n_pages - 8, n_pages, dtype=torch.int32, device=DEV).view(2, 4)
    cache.handle, cache.lens = pg.Kv8Cache(pool, cache.scales, cache.table, page_tokens=page, head_dim=dim), [200, 150]
    x = torch.randn(350, kvh, dim, generator=gen(2), device=DEV).to(dtype)
    cache.handle.append(x, x, i32([200, 150]), row_start=starts([200, 150]))
    keys, values = cache.kv(1)
    assert ((values - x[200:].double()).abs() <= 0.07 * x[200:].abs().double() + 1e-2).all() and torch.equal(keys, values)
    for rows in ([1, 1], [200, 90]):
        q = torch.randn(sum(rows), kvh, dim, generator=gen(5), device=DEV).to(dtype)
        out, ws = torch.empty_like(q), workspace(cache, sum(rows), kvh, dtype)
        cache.handle.attention(q, out, i32([200, 150]), ws, row_start=starts(rows), max_rows=max(rows))
        check_attention(cache, q, out, rows, dim ** -0.5)


# ------------------------------------------------------------------ append
def quantised(x, scale):
    """Half a step around each value: how far a code times its scale may be from x (both float64)."""
    return scale * torch.maximum((x / scale).abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64, device=x.device))


APPEND = [
    # lens (with the new), rows, heads, kv heads, dim, page, rotated
    ([1], [1], 4, 4, 64, 16, 64),
    ([300], [1], 12, 12, 64, 32, 0),
    ([1, 16, 17, 64, 65, 1000, 33], [1] * 7, 8, 2, 128, 16, 128),
    ([700, 64, 5, 130, 40], [500, 64, 0, 3, 40], 8, 2, 128, 64, 64),
    ([65, 100], [2, 37], 6, 2, 96, 64, 48),
    ([40, 100], [15, 33], 5, 1, 80, 32, 2),
    ([300], [290], 2, 2, 256, 64, 256),
    ([70], [70], 3, 3, 2, 16, 2),
    ([100, 3], [60, 3], 4, 2, 192, 32, 96),
    ([65, 64], [2, 64], 4, 1, 64, 16, 32),
]


@pytest.mark.parametrize("odd", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,rows,heads,kvh,dim,page,rot", APPEND)
def test_append(lens, rows, heads, kvh, dim, page, rot, dtype, odd):
    before = [n - r for n, r in zip(lens, rows)]
    cache = Cache(before, kvh, dim, page, 40 + sum(lens), spare=3 + sum(-(-n // page) for n in lens))
    free = [p for p in range(cache.pool.shape[0]) if p not in set(cache.table.flatten().tolist())]
    table = torch.full((len(lens), max(-(-n // page) for n in lens)), -1, dtype=torch.int32, device=DEV)
    table[:, :cache.table.shape[1]] = cache.table[:, :table.shape[1]]
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            if table[b, i] < 0:
                table[b, i] = free.pop()
    cache.table = table
    handle = pg.Kv8Cache(cache.pool, cache.scales, table, page_tokens=page, head_dim=dim)
    total = sum(rows)
    # rows of a product with more outputs than these: gaps between rows, odd addresses
    gap = 5 if odd else 8
    wide = (torch.randn(total, (heads + 2 * kvh) * dim + gap, generator=gen(1), device=DEV) * 1.7).to(dtype)
    qkv = wide[:, gap // 5 * odd:][:, :(heads + 2 * kvh) * dim].view(total, heads + 2 * kvh, dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
    old_pool, old_scales, before_q = cache.pool.clone(), cache.scales.clone(), q.double()
    old = [ref.sequence_kv(old_pool, old_scales, table[b], n, page, dim) for b, n in enumerate(before)]
    one = all(r == 1 for r in rows)
    handle.append(k, v, i32(lens), row_start=None if one else starts(rows), q=q, q_out=q, rot_dims=rot)
    at, mine = 0, set()
    for b, (n, length) in enumerate(zip(rows, lens)):
        pos = torch.arange(length - n, length, device=DEV)
        turned = ref.rotate(before_q[at:at + n], pos, rot, 10000.0)
        got = qkv[at:at + n, :heads].double()
        # turned in FP32: two products and a sum, then the type's rounding
        assert ((got - turned).abs() <= U[dtype] * turned.abs() + 2.0 ** -22 * before_q[at:at + n].abs().amax(-1, keepdim=True)).all()
        new = [ref.rotate(k[at:at + n].double(), pos, rot, 10000.0), v[at:at + n].double()]
        held = ref.sequence_kv(cache.pool, cache.scales, table[b], length, page, dim)
        for first in range((length - n) // page * page if n else length, length, page):
            p, o, end = int(table[b, first // page]), max(length - n - first, 0), min(length - first, page)
            mine.add(p)
            for side in range(2):
                part = new[side][first + o - (length - n):first + end - (length - n)]
                for h in range(kvh):
                    scale, amax = float(cache.scales[p, h, side]), float(part[:, h].abs().max())
                    wants = {max(ref.block_scale(amax * f), float(old_scales[p, h, side]) if o else 0.0) for f in (1 - 1e-6, 1, 1 + 1e-6)}
                    assert scale in wants, (b, first, side, h, scale, wants)
                    x = held[side][first + o:first + end, h]
                    assert ((x - part[:, h]).abs() <= quantised(part[:, h], scale) * (1 + 1e-6) + 1e-6 * amax).all()
                    if o:  # earlier tokens: exact, or rounded once more where they became subnormal
                        was, now = old[b][side][first:first + o, h], held[side][first:first + o, h]
                        assert ((was - now).abs() <= (0.0 if scale == float(old_scales[p, h, side]) else scale * 2.0 ** -10)).all()
        at += n
    others = [p for p in range(cache.pool.shape[0]) if p not in mine]
    assert torch.equal(cache.pool[others], old_pool[others])
    assert torch.equal(cache.scales[others].view(torch.int32), old_scales[others].view(torch.int32))
    # what lies behind the last token of a page is not touched
    for b, length in enumerate(lens):
        if rows[b] and length % page:
            kb, vb = ref.blocks(cache.pool[table[b, length // page].long()], page, dim)
            ko, vo = ref.blocks(old_pool[table[b, length // page].long()], page, dim)
            assert torch.equal(kb[:, length % page:], ko[:, length % page:]) and torch.equal(vb[..., length % page:], vo[..., length % page:])


def empty_cache(seqs, pages_per_seq, kvh, dim, page):
    n = seqs * pages_per_seq
    pool = torch.full(pg.Kv8Cache.pool_shape(n, kvh, page, dim), 255, dtype=torch.uint8, device=DEV)
    scales = torch.full((n, kvh, 2), math.nan, device=DEV)
    table = torch.randperm(n, device=DEV).to(torch.int32).view(seqs, pages_per_seq)
    return pg.Kv8Cache(pool, scales, table, page_tokens=page, head_dim=dim)


def test_append_token_by_token_is_append_at_once_up_to_subnormal_codes():
    n, kvh, dim, page = 100, 2, 64, 32
    g = gen(7)
    k, v = (torch.randn(n, kvh, dim, generator=g, device=DEV) * torch.exp2(torch.rand(n, 1, 1, generator=g, device=DEV) * 6) for _ in range(2))
    whole, single = empty_cache(1, 4, kvh, dim, page), empty_cache(1, 4, kvh, dim, page)
    whole.append(k, v, i32([n]), row_start=i32([0, n]), rot_dims=dim)
    for t in range(n):
        single.append(k[t:t + 1], v[t:t + 1], i32([t + 1]), rot_dims=dim)
    for i in range(4):
        a, b = whole.scales[whole.page_table[0, i].long()], single.scales[single.page_table[0, i].long()]
        assert torch.equal(a, b)
    for x, y in zip(*(ref.sequence_kv(c.pool, c.scales, c.page_table[0], n, page, dim) for c in (whole, single))):
        s = torch.stack([whole.scales[whole.page_table[0, t // page].long()] for t in range(n)]).amax(-1)[..., None]
        # each growth of the scale rounds a subnormal code by at most half its step of 2^-9; the errors halve from growth to growth
        assert ((x - y).abs() <= 2.0 ** -8 * s).all()
        assert (x != y).float().mean() < 0.2


def test_append_blocks_with_nan_or_infinity_and_zeros():
    c = empty_cache(1, 3, 1, 64, 16)
    k, v = torch.randn(40, 1, 64, device=DEV), torch.randn(40, 1, 64, device=DEV)
    k[3, 0, 5], v[20, 0, 0] = math.nan, -math.inf
    k[32:] = 0
    v[33:] = 0
    v[32] = 1e-38
    c.append(k, v, i32([40]), row_start=i32([0, 40]))
    s = c.scales[c.page_table[0].long()][:, 0]
    assert torch.isnan(s[0, 0]) and torch.isfinite(s[0, 1]) and torch.isfinite(s[1, 0]) and torch.isnan(s[1, 1])
    assert s[2, 0] == 2.0 ** -100 and s[2, 1] == 2.0 ** -100
    q, out = torch.randn(1, 1, 64, device=DEV), torch.empty(1, 1, 64, device=DEV)
    ws = torch.zeros(c.workspace_bytes(1, 1, F32), dtype=torch.uint8, device=DEV)
    c.attention(q, out, i32([40]), ws)
    assert torch.isnan(out).all()
    c.attention(q, out, i32([40]), ws, window=8)  # the bad blocks are out of sight
    assert torch.isfinite(out).all()
    c.append(k[:1], v[:1], i32([21]))  # a page position in the middle: the block stays NaN
    assert torch.isnan(c.scales[c.page_table[0, 1].long()][0, 1])
    c.append(k[4:16], v[4:16], i32([12]), row_start=i32([0, 12]))  # the page anew
    assert torch.isfinite(c.scales[c.page_table[0, 0].long()]).all()


def test_append_rows_that_have_no_place():
    c = empty_cache(3, 2, 1, 64, 16)
    c.page_table[1, 0] = -1
    c.page_table[1, 1] = 99
    pool = c.pool.clone()
    x = torch.randn(60, 1, 64, device=DEV)
    # sequence 0: more rows than tokens, so its first rows lie before position 0; 1: no pages; 2: beyond its table
    c.append(x, x, i32([3, 20, 40]), row_start=i32([0, 10, 30, 60]))
    k, v = ref.sequence_kv(c.pool, c.scales, c.page_table[0], 3, 16, 64)
    assert ((k - x[7:10].double()).abs() <= 0.07 * x[7:10].abs().double() + 1e-2).all()
    assert ((v - x[7:10].double()).abs() <= 0.07 * x[7:10].abs().double() + 1e-2).all()
    k, _ = ref.sequence_kv(c.pool, c.scales, c.page_table[2], 32, 16, 64)  # its rows 30..51 are positions 10..31
    assert torch.isnan(k[10:16]).all()  # in a block that no append began, whose scale was NaN
    assert ((k[16:] - x[36:52].double()).abs() <= 0.07 * x[36:52].abs().double() + 1e-2).all()
    mine = set(c.page_table[[0, 2]].flatten().tolist()) - {int(c.page_table[0, 1])}
    others = [p for p in range(6) if p not in mine]
    assert torch.equal(c.pool[others], pool[others])


# ------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,k,group", [(1, 1, 64), (16, 64, 64), (17, 65, 64), (33, 200, 128), (100, 129, 128), (48, 1024, 128), (5, 4096, 64)])
def test_quantize_q4(n, k, group, dtype):
    w = (torch.randn(n, k + 3, generator=gen(n + k), device=DEV) * torch.rand(n, 1, device=DEV)).to(dtype)[:, 1:k + 1]
    w[0, :min(k, group)] = 0
    ps, ss = pg.q4_shapes(n, k, group)
    packed, scales = torch.full(ps, 77, dtype=torch.uint8, device=DEV), torch.full(ss, 3.0, dtype=BF16, device=DEV)
    pg.quantize_q4(w, packed, scales, group)
    x = torch.nn.functional.pad(w.float(), (0, ss[0] * group - k)).view(n, ss[0], group)
    want = (x.abs().amax(-1) / 7).to(BF16)
    assert torch.equal(scales[:, :n].t(), want) and (scales[:, n:] == 0).all()
    s = want.float()[..., None]
    code = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)), 0.0).clamp(-8, 7).view(n, -1)
    full = ref.q4_codes(packed, ps[0] * 16, ps[1] * 64)
    assert torch.equal(full[:n, :k].float() - 8, code[:, :k])
    assert (full[n:] == 8).all() and (full[:, k:] == 8).all()


LINEAR = [(1, 1, 1, 64), (1, 2304, 768, 64), (2, 17, 65, 64), (8, 100, 1600, 128), (9, 31, 200, 64), (16, 640, 4096, 128), (5, 4000, 300, 128), (3, 48, 16384, 64),
          (16, 9000, 513, 64), (7, 33000, 70, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k,group", LINEAR)
def test_linear_q4(m, n, k, group, dtype):
    g = gen(m + n + k)
    ps, ss = pg.q4_shapes(n, k, group)
    packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
    pg.quantize_q4(torch.randn(n, k, generator=g, device=DEV) * 0.05, packed, scales, group)
    w = ref.q4_weights(packed, scales, n, k, group)
    for gap, bias in ((0, True), (3, False)):  # rows with gaps are read value by value
        x = torch.randn(m, k + gap, generator=g, device=DEV).to(dtype)[:, gap:]
        b = torch.randn(n, generator=g, device=DEV).to(dtype) if bias else None
        big = torch.full((m, n + 5), 9.0, device=DEV, dtype=dtype)
        pg.linear_q4(x, packed, scales, big[:, 2:n + 2], group, bias=b)
        want = x.double() @ w.t() + (b.double() if bias else 0.0)
        size = x.double().abs() @ w.abs().t() + (b.double().abs() if bias else 0.0)
        tile = x.double().abs().amax(-1, keepdim=True) * w.abs().sum(-1)  # a pair's rest is lost relative to the largest input of its tile
        tol = 2.0 ** -18 * size + U[dtype] * want.abs() + (2.0 ** -21 * tile if dtype == F32 else 0.0)
        assert ((big[:, 2:n + 2].double() - want).abs() <= tol).all()
        assert (big[:, :2] == 9).all() and (big[:, n + 2:] == 9).all()


def test_linear_q4_inputs_of_all_sizes():
    n, k = 64, 256
    ps, ss = pg.q4_shapes(n, k, 64)
    packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
    pg.quantize_q4(torch.randn(n, k, generator=gen(1), device=DEV), packed, scales, 64)
    w = ref.q4_weights(packed, scales, n, k, 64)
    x = torch.randn(4, k, generator=gen(2), device=DEV)
    x[0] *= 1e-30
    x[1] *= 1e30
    x[2, :64] *= 1e8  # tiles of one row that differ
    x[3] = 0
    out = torch.empty(4, n, device=DEV)
    pg.linear_q4(x, packed, scales, out, 64)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert ((out.double() - want).abs() <= 2.0 ** -18 * size).all()


# ------------------------------------------------------------------ log probabilities
def scores(x, targets, top):
    """log p of targets, entropy, ids and log p of the top entries in float64, by the definition."""
    x = x.double()
    d = x - x.amax(-1, keepdim=True)  # values may be so large that the logarithm of their sum loses all but the maximum
    p = d - torch.logsumexp(d, -1, keepdim=True)
    lp = p.gather(1, targets.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    ent = -(p.exp() * p.clamp(min=-1e30)).sum(-1)
    ids = torch.argsort(-x, dim=-1, stable=True)[:, :top]
    return lp, ent, ids, p.gather(1, ids)


def run_scores(x, targets, top):
    rows = x.shape[0]
    lp, ent = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    ids = torch.full((rows, top), -7, dtype=torch.int32, device=DEV) if top else None
    values = torch.empty(rows, top, device=DEV) if top else None
    pg.token_logprobs(x, targets, lp, ent, ids, values)
    return lp, ent, ids, values


def check_scores(x, targets, top):
    got, want = run_scores(x, targets, top), scores(x, targets, top)
    for a, b in ((got[0], want[0]), (got[1], want[1])) + (((got[3], want[3]),) if top else ()):
        a = a.double()
        same = (a == b) | ((a - b).abs() <= 2.0 ** -18 * (1 + b.abs()))
        assert same.all(), (a[~same][:4], b[~same][:4])
    if top:
        assert torch.equal(got[2].long(), want[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 7, 7), (3, 33, 32), (1, 50257, 5), (8, 50257, 20), (200, 1000, 1), (149, 5003, 32), (5, 128256, 8), (600, 2049, 0),
                                            (1, 1000003, 32), (40, 40, 32), (2000, 777, 3), (1800, 4000, 32), (1000, 3001, 20), (1900, 9000, 20)])
def test_token_logprobs(rows, vocab, top, dtype):
    g = gen(rows + vocab)
    x = (torch.randn(rows, vocab + 3, generator=g, device=DEV) * 3).to(dtype)[:, 1:vocab + 1]  # rows at odd addresses
    x[:, torch.randint(0, vocab, (vocab // 10,), generator=g, device=DEV)] = -math.inf
    x[torch.isinf(x).all(-1)] = 0.5
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
    check_scores(x, targets, top)
    check_scores(x.contiguous(), targets, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("repeat", [1, 90, 200])
@pytest.mark.parametrize("vocab", [5, 600, 50257])
def test_token_logprobs_masks_and_ties(dtype, vocab, repeat):
    """Ties go to the lower id, masked entries have no weight, rows of one kind of value work."""
    low = torch.finfo(dtype).min
    x = torch.zeros(10, vocab, device=DEV, dtype=dtype)  # row 0: all equal
    x[1] = -math.inf
    x[1, vocab - 2] = 3.0  # one entry
    x[2] = low
    x[2, 1] = -1.0
    x[3] = low  # all at the lowest value: as good as equal
    x[4] = torch.arange(vocab, device=DEV).to(dtype)  # rising: the last are the largest
    x[5] = -torch.arange(vocab, device=DEV).to(dtype)
    x[6, ::2] = -0.0  # equal to 0
    x[7] = torch.where(torch.arange(vocab, device=DEV) % 3 == 0, 2.0, -math.inf)
    x[8] = torch.finfo(dtype).max
    x[9, -1] = 3e38
    top = min(5, vocab)
    x = x.repeat(repeat, 1) if vocab < 50257 else x
    t = torch.tensor([0, vocab - 2, 1, 2, vocab - 1, 0, 1, 0, 3, vocab - 1], dtype=torch.int32, device=DEV)
    check_scores(x, t.repeat(x.shape[0] // 10), top)


@pytest.mark.parametrize("offset", [1000.0, -30000.0])
def test_token_logprobs_of_logits_far_from_zero(offset):
    x = torch.randn(20, 5000, generator=gen(1), device=DEV) + offset
    check_scores(x, torch.arange(20, dtype=torch.int32, device=DEV), 5)


@pytest.mark.parametrize("repeat", [1, 160, 400])  # a block, four warps, (of the short rows) a warp for each row
def test_token_logprobs_rows_without_a_distribution_and_odd_targets(repeat):
    for vocab in (9, 3000, 50257):
        x = torch.randn(6, vocab, device=DEV)
        x[1, vocab - 1] = math.nan
        x[2, 0] = math.inf
        x[3] = -math.inf
        t = torch.tensor([-1, 0, 0, 0, vocab, -2], dtype=torch.int32, device=DEV)
        lp, ent, ids, values = (o[-6:] for o in run_scores(x.repeat(repeat, 1), t.repeat(repeat), 3))
        assert lp[0] == 0 and torch.isnan(lp[1:]).all()
        assert torch.isnan(ent[1:4]).all() and torch.isfinite(ent[[0, 4, 5]]).all()
        assert (ids[1:4] == -1).all() and torch.isnan(values[1:4]).all() and (ids[[0, 4, 5]] >= 0).all()


def test_token_logprobs_each_output_alone():
    x = torch.randn(3, 777, device=DEV)
    t = i32([5, 6, 776])
    want = scores(x, t, 4)
    lp, ent = torch.empty(3, device=DEV), torch.empty(3, device=DEV)
    pg.token_logprobs(x, targets=t, logprobs=lp)
    pg.token_logprobs(x, entropy=ent)
    ids, values = torch.empty(3, 4, dtype=torch.int32, device=DEV), torch.empty(3, 4, device=DEV)
    pg.token_logprobs(x, top_ids=ids, top_logprobs=values)
    assert ((lp - want[0]).abs() < 1e-4).all() and ((ent - want[1]).abs() < 1e-4).all()
    assert torch.equal(ids.long(), want[2])


def test_token_logprobs_rows_further_apart_than_31_bits():
    far = (1 << 31) + 24
    store = torch.empty(far + 5000, dtype=BF16, device=DEV)
    x = torch.as_strided(store, (2, 5000), (far, 1))
    x.copy_(torch.randn(2, 5000, generator=gen(3), device=DEV))
    t, want = i32([4999, 17]), None
    lp, ent, ids, values = torch.empty(2, device=DEV), torch.empty(2, device=DEV), torch.empty(2, 6, dtype=torch.int32, device=DEV), torch.empty(2, 6, device=DEV)
    pg.token_logprobs(x, targets=t, logprobs=lp, entropy=ent, top_ids=ids, top_logprobs=values)
    want = scores(x, t, 6)
    assert ((lp - want[0]).abs() <= 2.0 ** -18 * (1 + want[0].abs())).all() and ((ent - want[1]).abs() <= 2.0 ** -18 * (1 + want[1].abs())).all()
    assert torch.equal(ids.long(), want[2])


def test_linear_q4_codes_beyond_32_bits():
    n, k = 1 << 17, (1 << 16) + 64
    ps, ss = pg.q4_shapes(n, k, 128)
    packed, scales = torch.zeros(ps, dtype=torch.uint8, device=DEV), torch.zeros(ss, dtype=BF16, device=DEV)
    assert packed.numel() > 1 << 32
    packed[-1] = torch.randint(0, 256, packed[-1].shape, generator=gen(2), device=DEV).to(torch.uint8)
    scales[:, -16:] = 0.25
    x, out = torch.randn(3, k, generator=gen(3), device=DEV), torch.full((3, n), 5.0, device=DEV)
    pg.linear_q4(x, packed, scales, out, 128)
    w = ref.q4_weights(packed[-1:].clone(), scales[:, -16:].clone(), 16, k, 128)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    tile = x.double().abs().amax(-1, keepdim=True) * w.abs().sum(-1)
    # (a warp adds 129 sums up, half a step of 2^-24 each: within 2^-16)
    assert ((out[:, -16:].double() - want).abs() <= 2.0 ** -16 * size + 2.0 ** -24 * want.abs() + 2.0 ** -21 * tile).all()
    assert (out[:, :-16] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_q4_rows_that_are_not_finite_stay_alone(dtype):
    n, k = 40, 200
    ps, ss = pg.q4_shapes(n, k, 64)
    packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
    pg.quantize_q4(torch.randn(n, k, generator=gen(1), device=DEV), packed, scales, 64)
    x = torch.randn(12, k, generator=gen(2), device=DEV).to(dtype)
    want, got = torch.empty(12, n, dtype=dtype, device=DEV), torch.empty(12, n, dtype=dtype, device=DEV)
    pg.linear_q4(x, packed, scales, want, 64)
    x[3, 7], x[9, 150], x[10, 199] = math.nan, math.inf, -math.inf
    pg.linear_q4(x, packed, scales, got, 64)
    odd = torch.tensor([3, 9, 10], device=DEV)
    keep = torch.tensor([i for i in range(12) if i not in (3, 9, 10)], device=DEV)
    assert torch.isnan(got[odd]).all() and torch.equal(got[keep], want[keep])


# ------------------------------------------------------------------ together
class Layer:
    """One layer's step as a serving program builds it from the operators: products in 4 bits around the 8-bit cache, then a head."""

    def __init__(self, dtype, seqs, heads=8, kvh=2, dim=64, vocab=1000, page=16, pages=8):
        g = gen(5)
        self.dtype, self.heads, self.kvh, self.dim, self.width = dtype, heads, kvh, dim, heads * dim
        self.cache = empty_cache(seqs, pages, kvh, dim, page)
        self.weights = {}
        for name, n, k in (("qkv", (heads + 2 * kvh) * dim, self.width), ("o", self.width, self.width), ("head", vocab, self.width)):
            ps, ss = pg.q4_shapes(n, k, 64)
            packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
            pg.quantize_q4(torch.randn(n, k, generator=g, device=DEV) * k ** -0.5, packed, scales, 64)
            self.weights[name] = packed, scales
        e = lambda *s, t=dtype: torch.empty(*s, dtype=t, device=DEV)
        self.x, self.lens = e(seqs, self.width), torch.zeros(seqs, dtype=torch.int32, device=DEV)
        self.qkv, self.attn, self.y, self.logits = e(seqs, (heads + 2 * kvh) * dim), e(seqs, heads, dim), e(seqs, self.width), e(seqs, vocab)
        self.ids, self.values, self.ent = e(seqs, 4, t=torch.int32), e(seqs, 4, t=F32), e(seqs, t=F32)
        self.ws = torch.zeros(self.cache.workspace_bytes(seqs, heads, dtype), dtype=torch.uint8, device=DEV)

    def step(self):
        s = torch.cuda.current_stream().cuda_stream
        h, kvh = self.heads, self.kvh
        pg.linear_q4(self.x, *self.weights["qkv"], self.qkv, 64, stream=s)
        rows = self.qkv.view(-1, h + 2 * kvh, self.dim)
        q, k, v = rows[:, :h], rows[:, h:h + kvh], rows[:, h + kvh:]
        self.cache.append(k, v, self.lens, q=q, q_out=q, rot_dims=self.dim, stream=s)
        self.cache.attention(q, self.attn, self.lens, self.ws, stream=s)
        pg.linear_q4(self.attn.view(-1, self.width), *self.weights["o"], self.y, 64, stream=s)
        pg.linear_q4(self.y, *self.weights["head"], self.logits, 64, stream=s)
        pg.token_logprobs(self.logits, entropy=self.ent, top_ids=self.ids, top_logprobs=self.values, stream=s)

    def weight(self, name, n):
        return ref.q4_weights(*self.weights[name], n, self.width, 64)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_step_of_all_operators_eager_and_captured(dtype):
    seqs = 5
    eager, captured = Layer(dtype, seqs), Layer(dtype, seqs)
    captured.cache.page_table.copy_(eager.cache.page_table)
    for l in (eager, captured):  # different lengths to begin with
        l.lens.copy_(torch.arange(seqs))
    stream = torch.cuda.Stream()
    captured.x.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured.step()
    inputs = torch.randn(60, seqs, eager.width, generator=gen(8), device=DEV).to(dtype)
    # both caches start with the same tokens at the positions before the first step
    for l in (eager, captured):
        kv = torch.randn(int(sum(range(seqs))), 2, 64, generator=gen(9), device=DEV).to(dtype)
        l.cache.append(kv, kv, l.lens, row_start=starts(list(range(seqs))))
    history = [[] for _ in range(seqs)]
    for t in range(60):
        for l in (eager, captured):
            l.x.copy_(inputs[t])
            l.lens.add_(1)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("qkv", "attn", "y", "logits", "ids", "values", "ent"):
            assert torch.equal(getattr(eager, name), getattr(captured, name)), (t, name)
        if t not in (0, 20, 59):
            continue
        # each operator against its definition, from what the one before it gave
        n = eager.qkv.shape[1]
        raw = eager.x.double() @ eager.weight("qkv", n).t()
        size = eager.x.double().abs() @ eager.weight("qkv", n).abs().t()
        v = eager.qkv.view(seqs, -1, 64)[:, 10:].double()
        assert ((v.flatten(1) - raw[:, 640:]).abs() <= 2.0 ** -17 * size[:, 640:] + U[dtype] * raw[:, 640:].abs()).all()
        for b in range(seqs):
            length = int(eager.lens[b])
            keys, values = ref.sequence_kv(eager.cache.pool, eager.cache.scales, eager.cache.page_table[b], length, 16, 64)
            want = ref.attention(eager.qkv.view(seqs, -1, 64)[b:b + 1, :8].double(), keys, values, torch.tensor([length - 1], device=DEV), 0.125)
            tol = values.abs().max() * (2.0 ** -15 if dtype == F32 else 2.0 ** -10) + U[dtype] * want.abs()
            assert ((eager.attn[b:b + 1].double() - want).abs() <= tol).all()
        want = scores(eager.logits, torch.zeros(seqs, device=DEV), 4)
        assert torch.equal(eager.ids.long(), want[2]) and ((eager.ent - want[1]).abs() <= 2.0 ** -16 * (1 + want[1])).all()


def test_two_streams_at_once():
    """Calls that overlap, each with a workspace of its own, give what they give alone."""
    a, b = Cache([9000, 40], 2, 64, 64, 1), Cache([8000, 50], 2, 64, 64, 2)
    qs = [torch.randn(2, 8, 64, generator=gen(i), device=DEV) for i in range(2)]
    alone, both = [], [torch.empty_like(q) for q in qs]
    spaces = [workspace(c, 2, 8, F32) for c in (a, b)]
    lens = [i32(c.lens) for c in (a, b)]
    for c, q, l, w in zip((a, b), qs, lens, spaces):
        out = torch.empty_like(q)
        c.handle.attention(q, out, l, w)
        alone.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, q, l, w, o, s in zip((a, b), qs, lens, spaces, both, streams):
            c.handle.attention(q, o, l, w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(alone, both))


class Prompts:
    """Portions of prompts as a serving program has them: append, then attention, over one cache."""

    def __init__(self, dtype, seed, seqs=3, heads=4, kvh=2, dim=64, room=200):
        self.cache = empty_cache(seqs, 20, kvh, dim, 16)
        e = lambda *s, t=dtype: torch.zeros(*s, dtype=t, device=DEV)
        self.q, self.k, self.v, self.turned, self.out = e(room, heads, dim), e(room, kvh, dim), e(room, kvh, dim), e(room, heads, dim), e(room, heads, dim)
        self.lens, self.start, self.g = e(seqs, t=torch.int32), e(seqs + 1, t=torch.int32), gen(seed)
        self.ws = torch.zeros(self.cache.workspace_bytes(room, heads, dtype), dtype=torch.uint8, device=DEV)
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=self.g, device=DEV))

    def call(self):
        s = torch.cuda.current_stream().cuda_stream
        self.cache.append(self.k, self.v, self.lens, row_start=self.start, q=self.q, q_out=self.turned, rot_dims=64, stream=s)
        self.cache.attention(self.turned, self.out, self.lens, self.ws, row_start=self.start, max_rows=200, stream=s)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_portions_of_prompts_eager_and_captured(dtype):
    eager, captured = Prompts(dtype, 1), Prompts(dtype, 1)
    captured.cache.page_table.copy_(eager.cache.page_table)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        captured.call()
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    for rows in ([100, 40, 60], [1, 1, 1], [0, 120, 2], [50, 0, 0], [0, 0, 0], [100, 60, 40]):
        lens += i32(rows)
        for p in (eager, captured):
            p.lens.copy_(lens)
            p.start.copy_(starts(rows))
            p.out.fill_(3.0)
        eager.call()
        graph.replay()
        torch.cuda.synchronize()
        n = sum(rows)
        assert torch.equal(eager.out, captured.out) and (eager.out[n:] == 3).all()
        at = 0
        for b, r in enumerate(rows):
            length = int(lens[b])
            keys, values = ref.sequence_kv(eager.cache.pool, eager.cache.scales, eager.cache.page_table[b], length, 16, 64)
            want = ref.attention(eager.turned[at:at + r].double(), keys, values, torch.arange(length - r, length, device=DEV), 0.125)
            tol = (values.abs().max() if length else 0.0) * (2.0 ** -15 if dtype == F32 else 2.0 ** -10) + U[dtype] * want.abs()
            assert ((eager.out[at:at + r].double() - want).abs() <= tol).all(), (rows, b)
            at += r


@pytest.mark.parametrize("lens", [[130, 69, 1], [200, 70, 1]])  # (the second: tokens that were never appended lie before the rows, NaN)
def test_two_streams_of_portions_at_once(lens):
    both, alone = [Prompts(BF16, i) for i in (1, 2)], [Prompts(BF16, i) for i in (1, 2)]
    for p, o in zip(both, alone):
        o.cache.page_table.copy_(p.cache.page_table)
        for x in (p, o):
            x.lens.copy_(i32(lens))
            x.start.copy_(starts([130, 69, 1]))
    for p in alone:
        p.call()
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip(both, streams):
            with torch.cuda.stream(s):
                p.call()
    torch.cuda.synchronize()
    for p, o in zip(both, alone):
        assert torch.isnan(p.out).any() == (lens[0] > 130) and torch.equal(p.out.view(torch.int16), o.out.view(torch.int16))


# ------------------------------------------------------------------ one workspace, queries and inputs of every finite size, long tails
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_calls_of_all_sizes_share_a_workspace(dtype):
    """Steps, mixed calls with more rows and calls over another cache, one after the other: whatever one leaves, the next gives all its rows."""
    lens = [1600] + [100 + i * 53 % 900 for i in range(63)]
    wide, small = Cache(lens, 8, 128, 64, 41), Cache([5000, 70, 3000], 1, 64, 16, 42)
    size = max(wide.handle.workspace_bytes(2000, 32, dtype), small.handle.workspace_bytes(3, 8, dtype))
    ws = torch.zeros(size, dtype=torch.uint8, device=DEV)
    calls = [(wide, 32, [1] * 64), (wide, 32, [1500] + [1] * 63), (small, 8, [1] * 3), (wide, 32, [700] + [3] * 63), (wide, 32, [1] * 64), (small, 8, [1, 60, 2])]
    for i, (cache, heads, rows) in enumerate(calls):
        q = torch.randn(sum(rows), heads, cache.dim, generator=gen(i), device=DEV).to(dtype)
        out = torch.full_like(q, 1e4)
        cache.handle.attention(q, out, i32(cache.lens), ws, row_start=starts(rows), max_rows=max(rows))
        check_attention(cache, q, out, rows, cache.dim ** -0.5)


def test_linear_q4_inputs_at_the_ends_of_the_range():
    n, k = 64, 256
    ps, ss = pg.q4_shapes(n, k, 64)
    packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
    pg.quantize_q4(torch.randn(n, k, generator=gen(1), device=DEV), packed, scales, 64)
    w = ref.q4_weights(packed, scales, n, k, 64)
    x = torch.randn(12, k, generator=gen(2), device=DEV)
    x[0:4] *= 2.0 ** 116  # 64 magnitudes add up to 2^122
    x[4:8] *= 2.0 ** -120
    out = torch.empty(12, n, device=DEV)
    pg.linear_q4(x, packed, scales, out, 64)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert ((out.double() - want).abs() <= 2.0 ** -18 * size).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** 120])
def test_attention_queries_at_the_ends_of_the_range(size, rows, dtype):
    cache = Cache([300], 1, 64, 16, 3)
    q = (torch.randn(rows, 2, 64, generator=gen(1), device=DEV) * size).to(dtype)
    out = torch.full_like(q, 1e4)
    cache.handle.attention(q, out, i32([300]), workspace(cache, rows, 2, dtype), row_start=starts([rows]), max_rows=rows, scale=0.125 / size)
    check_attention(cache, q, out, [rows], 0.125 / size)


def test_linear_q4_outlier_with_weights_of_zero():
    """An input that is far larger than the others of its row and meets weights of zero: the sums do not know it. Sums as in test_linear_q4."""
    n, k = 48, 256
    w = torch.randn(n, k, generator=gen(1), device=DEV)
    w[:, 70] = 0
    ps, ss = pg.q4_shapes(n, k, 64)
    packed, scales = torch.empty(ps, dtype=torch.uint8, device=DEV), torch.empty(ss, dtype=BF16, device=DEV)
    pg.quantize_q4(w, packed, scales, 64)
    w = ref.q4_weights(packed, scales, n, k, 64)
    assert (w[:, 70] == 0).all()
    for m in (3, 16):
        x = torch.randn(m, k, generator=gen(2), device=DEV).to(BF16)
        x[:, 70] = torch.logspace(3, 8, m, device=DEV).to(BF16)
        out = torch.empty(m, n, device=DEV, dtype=BF16)
        pg.linear_q4(x, packed, scales, out, 64)
        want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
        assert ((out.double() - want).abs() <= 2.0 ** -18 * size + U[BF16] * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("seqs,rows,heads,dim", [(2400, 1, 1, 64), (100, 2, 128, 64), (80, 2, 128, 128)])  # few rows of a sequence, portions; tiles that are not cut
def test_attention_long_tail_behind_one_large_weight(seqs, rows, heads, dim, dtype):
    """One token outweighs each of the 131071 others by 2^25.6, and they together are 2.6 thousandths: the mean of their equal values must keep them."""
    n, page = 131072, 64
    pages = n // page
    pool = torch.zeros(pg.Kv8Cache.pool_shape(pages, 1, page, dim), dtype=torch.uint8, device=DEV)
    keys, values = ref.blocks(pool, page, dim)
    keys[0, 0, 0, 0] = 0x38  # 1: the first token's score is 17.75, the others' 0
    values[..., :dim, :] = 0x38
    values[0, 0, :, 0] = 0
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(seqs, 1)  # sequences may share pages
    cache = pg.Kv8Cache(pool, torch.ones(pages, 1, 2, device=DEV), table, page_tokens=page, head_dim=dim)
    q = torch.zeros(seqs * rows, heads, dim, device=DEV, dtype=dtype)
    q[..., 0] = 17.75
    out = torch.full_like(q, 7.0)
    ws = torch.zeros(cache.workspace_bytes(seqs * rows, heads, dtype), dtype=torch.uint8, device=DEV)
    cache.attention(q, out, i32([n] * seqs), ws, row_start=starts([rows] * seqs), max_rows=rows, scale=1.0)
    for r in range(rows):
        tail = (n - rows + r) * math.exp(-17.75)
        want = tail / (1 + tail)
        # weights to half a step each (FP32 rows: pairs and their sums, 2^-15 of the result; BF16: FP16 numbers), tokens not lost but rounded to 2^-37 of the largest
        tol = want * (2.0 ** -15 if dtype == F32 else 2.0 ** -10 + 2.0 ** -8) + n * 2.0 ** -37
        assert ((out[r::rows].double() - want).abs() <= tol).all(), (float(out[r::rows].double().min()), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("seqs,rows,heads", [(2400, 1, 1), (40, 3, 128), (1, 130, 2)])  # few rows of a sequence; portions in one part, in several
def test_attention_long_sums_of_values_of_one_sign(seqs, rows, heads, dim, dtype):
    """Values around 1: the sums over 40000 tokens only grow, and whatever cuts them off adds up."""
    n, page = 40000, 64
    pages, g = -(-n // page), gen(dim)
    pool = torch.zeros(pg.Kv8Cache.pool_shape(pages, 1, page, dim), dtype=torch.uint8, device=DEV)
    keys, values = ref.blocks(pool, page, dim)
    keys[..., :dim] = torch.randn(pages, 1, page, dim, generator=g, device=DEV).to(torch.float8_e4m3fn).view(torch.uint8)
    values[..., :dim, :] = (1 + 0.25 * torch.randn(pages, 1, dim, page, generator=g, device=DEV)).to(torch.float8_e4m3fn).view(torch.uint8)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(seqs, 1)  # sequences may share pages
    cache = pg.Kv8Cache(pool, torch.ones(pages, 1, 2, device=DEV), table, page_tokens=page, head_dim=dim)
    q = torch.randn(seqs * rows, heads, dim, generator=g, device=DEV).to(dtype)
    out = torch.full_like(q, 7.0)
    ws = torch.zeros(cache.workspace_bytes(seqs * rows, heads, dtype), dtype=torch.uint8, device=DEV)
    for call in range(2):
        cache.attention(q, out, i32([n] * seqs), ws, row_start=starts([rows] * seqs), max_rows=rows)
    k, v = ref.sequence_kv(pool, cache.scales, table[0], n, page, dim)
    top, h = float(v.abs().max()), min(heads, 2)
    for b in {0, seqs // 2, seqs - 1}:
        some = slice(b * rows, b * rows + min(rows, 3))
        want = ref.attention(q[some, :h].double(), k, v, torch.arange(n - rows, n, device=DEV)[:3], dim ** -0.5)
        tol = top * (2.0 ** -15 if dtype == F32 else 2.0 ** -10) + U[dtype] * want.abs()
        assert ((out[some, :h].double() - want).abs() <= tol).all(), (b, float(((out[some, :h].double() - want) / want).mean()))


def test_attention_status_of_the_workspace():
    """The first 32 bits: left alone by calls whose waits end, so that what an earlier call said stays until the caller zeroes it."""
    cache = Cache([9000, 300], 2, 128, 64, 3)
    for before in (0, 1):
        for rows in ([1, 1], [130, 5]):
            ws = workspace(cache, sum(rows), 4, F32)
            ws[:4].view(torch.int32).fill_(before)
            q = torch.randn(sum(rows), 4, 128, generator=gen(1), device=DEV)
            out = torch.empty_like(q)
            cache.handle.attention(q, out, i32(cache.lens), ws, row_start=starts(rows), max_rows=max(rows))
            check_attention(cache, q, out, rows, 128 ** -0.5)
            assert int(ws[:4].view(torch.int32)) == before


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_sums_in_memory_of_more_blocks_than_run_at_once(dim):
    """FP32 portions long enough for sums in memory, more of them than there are places for those: all sequences alike, so all results alike."""
    n, seqs, rows, heads, page = 3000, 450, 2, 64, 64
    one = Cache([n], 1, dim, page, 5)
    one.table = one.table.repeat(seqs, 1)
    one.handle = pg.Kv8Cache(one.pool, one.scales, one.table, page_tokens=page, head_dim=dim)
    q = torch.randn(rows, heads, dim, generator=gen(2), device=DEV).repeat(seqs, 1, 1)
    out = torch.full_like(q, 1e4)
    one.handle.attention(q, out, i32([n] * seqs), workspace(one, seqs * rows, heads, F32), row_start=starts([rows] * seqs), max_rows=rows)
    check_attention(one, q[:rows], out[:rows], [rows], dim ** -0.5)
    assert (out.view(seqs, -1) == out[:rows].reshape(1, -1)).all()


@pytest.mark.parametrize("window,keep,gone", [(0, 0, 2600), (2600, 2400, 0), (4500, 100, 7000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_portions_whose_first_pieces_are_not_seen(window, keep, gone, dtype):
    """Pieces of which a row sees nothing come first: on no page, or kept for other rows."""
    n, rows, heads = 9000, 150, 4
    cache = Cache([n], 2, 64, 64, 9)
    cache.table[0, :gone // 64] = -1
    q = torch.randn(rows, heads, 64, generator=gen(4), device=DEV).to(dtype)
    out = torch.full_like(q, 1e4)
    cache.handle.attention(q, out, i32([n]), workspace(cache, rows, heads, dtype), row_start=starts([rows]), max_rows=rows, window=window, keep_first=keep)
    cache.table.clamp_(min=0)
    keys, values = cache.kv(0)
    want = ref.attention(q.double(), keys, values, torch.arange(n - rows, n, device=DEV), 0.125, window, keep, missing=torch.arange(n, device=DEV) < gone // 64 * 64)
    tol = float(values.abs().max()) * (2.0 ** -15 if dtype == F32 else 2.0 ** -10) + U[dtype] * want.abs()
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 40])
def test_append_at_far_positions(rows, dtype):
    """Angles of positions around a million, of the tokens and of the queries."""
    page, dim, heads, length = 64, 64, 2, 1000000
    pages = 3
    pool = torch.zeros(pg.Kv8Cache.pool_shape(pages, 1, page, dim), dtype=torch.uint8, device=DEV)
    table = torch.full((1, -(-length // page)), -1, dtype=torch.int32, device=DEV)
    table[0, -pages:] = torch.arange(pages, dtype=torch.int32, device=DEV)
    cache = pg.Kv8Cache(pool, torch.zeros(pages, 1, 2, device=DEV), table, page_tokens=page, head_dim=dim)
    q, k = (torch.randn(rows, h, dim, generator=gen(h), device=DEV).to(dtype) for h in (heads, 1))
    out = torch.empty_like(q)
    cache.append(k, k, i32([length]), row_start=None if rows == 1 else starts([rows]), q=q, q_out=out, rot_dims=dim)
    pos = torch.arange(length - rows, length, device=DEV)
    want = ref.rotate(q.double(), pos, dim, 10000.0)
    assert ((out.double() - want).abs() <= U[dtype] * want.abs() + 2.0 ** -22 * q.double().abs().amax(-1, keepdim=True)).all()
    keys, _ = ref.sequence_kv(pool, cache.scales, table[0, -pages:], pages * page, page, dim)
    held, want = keys[-rows:], ref.rotate(k.double(), pos, dim, 10000.0)  # the last page is full
    assert ((held - want).abs() <= 0.07 * want.abs() + 1e-2).all()
