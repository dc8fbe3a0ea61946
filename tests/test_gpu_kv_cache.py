"""GPU: the quantised, paged cache and attention over it against their definitions in 64 bits (oracle/mx.py).

Written and read-back values are exact.  Attention's result may be off by its own rounding (u |o|), by the rounding
of the probabilities to 16 bits (u sum p |v|; in f16 also 2^-25 sum |v|, below its normal range), and by the
scores' fp32 sums: delta = 2^-24 (D + 8) sum |q k| scale moves every p by at most 2 delta; exp2 and the fp32 sums add
2^-20."""
import math

import pytest
import torch

from mpq_amd.kv_cache import QuantizedKVCache
from oracle import mx as om

pytestmark = pytest.mark.gpu

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}


class _Batch:
    """Sequences of given lengths in a cache whose pages lie at random places, all other memory garbage."""

    def __init__(self, gpu, lens, heads, dim, page, fmt, dtype, seed=0, spare=2, garbage=True):
        g = torch.Generator().manual_seed(seed)
        self.gpu, self.lens, self.page, self.dtype, self.fmt, self.g = gpu, lens, page, dtype, fmt, g
        need = [-(-n // page) for n in lens]
        pool = sum(need) + spare
        self.cache = QuantizedKVCache(pool, page, heads, dim, fmt=fmt, dtype=dtype, device=gpu)
        if garbage:
            for t in (self.cache.k_codes, self.cache.k_scales, self.cache.v_codes, self.cache.v_scales):
                t.fill_(255)
        place = torch.randperm(pool, generator=g)
        self.table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = place[at: at + n].int()
            at += n
        total = sum(lens)
        c = torch.exp(0.5 * torch.randn(heads, dim, generator=g))
        self.k = (torch.randn(total, heads, dim, generator=g) * c).to(dtype)
        self.v = torch.randn(total, heads, dim, generator=g).to(dtype)
        self.starts = [0]
        for n in lens:
            self.starts.append(self.starts[-1] + n)
        self.slots = torch.cat([self.table[i, torch.arange(n) // page].long() * page + torch.arange(n) % page
                                for i, n in enumerate(lens)]) if total else torch.zeros(0, dtype=torch.int64)

    def fill(self):
        self.cache.write(self.k.to(self.gpu), self.v.to(self.gpu), self.slots.to(self.gpu))
        return self

    def read(self):
        return self.cache.read(self.table.to(self.gpu), torch.tensor(self.starts, dtype=torch.int32, device=self.gpu),
                               sum(self.lens))

    def attend(self, new, group, causal=True, q=None, **more):
        heads, dim = self.cache.heads, self.cache.head_dim
        if q is None:
            q = torch.randn(sum(new), heads * group, dim, generator=self.g).to(self.dtype)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.gpu)  # noqa: E731
        got = self.cache.attend(q.to(self.gpu), self.table.to(self.gpu), i32(self.lens), i32(starts),
                                max(new + [0]), causal=causal, **more)
        return q, starts, got

    def check(self, new, group, causal=True, scale=None, **more):
        q, starts, (o, lse) = self.attend(new, group, causal, return_lse=True, scale=scale, **more)
        o, lse = o.cpu().double(), lse.cpu().double()
        dim = self.cache.head_dim
        u = UNIT[self.dtype]
        for i, n in enumerate(self.lens):
            a, b = starts[i], starts[i + 1]
            k, v = (om.values(t[self.starts[i]: self.starts[i + 1]], self.fmt) for t in (self.k, self.v))
            want, wl, pv, mass, big = om.attend(q[a:b], k, v, new[i], dim ** -0.5 if scale is None else scale, causal)
            delta = (2.0 ** -24 * (dim + 8) * big).unsqueeze(-1)
            tol = u * want.abs() * 1.01 + (1.01 * u + 2 * delta + 2.0 ** -20) * pv + 1e-30
            if self.dtype == torch.float16:
                tol = tol + 2.0 ** -25 * (1 + mass)
            err = (o[a:b] - want).abs()
            assert bool((err <= tol).all()), (i, float((err / tol).max()))
            seen = torch.isfinite(wl)
            assert torch.equal(seen, torch.isfinite(lse[a:b])) and bool((lse[a:b][~seen] == -math.inf).all())
            le = (lse[a:b] - wl)[seen].abs()
            assert bool((le <= (2.0 ** -20 * (1 + wl.abs()) + 2 * delta.squeeze(-1))[seen]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("lens,heads,dim,page", [([1], 1, 64, 16), ([17, 0, 64], 2, 128, 16), ([300, 5], 3, 64, 64),
                                                 ([40, 129, 16, 1], 8, 128, 32), ([0], 1, 128, 16)])
def test_write_read(gpu, dtype, fmt, lens, heads, dim, page):
    b = _Batch(gpu, lens, heads, dim, page, fmt, dtype).fill()
    for got, x in zip(b.read(), (b.k, b.v)):
        assert got.dtype == dtype and torch.equal(got.cpu(), om.values(x, fmt).to(dtype))


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_write_layout(gpu, fmt):
    """The stored bytes are where the documented layout says."""
    b = _Batch(gpu, [70], 2, 64, 32, fmt, torch.bfloat16, garbage=False).fill()
    for t in (0, 1, 2, 3, 4, 37, 69):
        at, row = int(b.slots[t]) // 32, int(b.slots[t]) % 32
        for codes, scales, x in ((b.cache.k_codes[at, :, row], b.cache.k_scales[at, :, row], b.k[t]),
                                 (b.cache.v_codes[at, :, row // 4, :, row % 4].flatten(-2),
                                  b.cache.v_scales[at, :, row // 4, :, row % 4], b.v[t])):
            c, s, _ = om.encode(x, fmt)
            assert torch.equal(codes.cpu(), om.pack(c, fmt)) and torch.equal(scales.cpu(), s)


def test_write_leaves_other_tokens_and_skips_padding(gpu):
    b = _Batch(gpu, [33, 20], 2, 128, 16, "mxfp4", torch.bfloat16).fill()
    before = [t.clone() for t in (b.cache.k_codes, b.cache.k_scales, b.cache.v_codes, b.cache.v_scales)]
    slots = torch.tensor([-1, 16 * b.cache.num_pages, 2 ** 40, -(2 ** 40)], device=gpu)
    b.cache.write(b.v[:4].to(gpu), b.k[:4].to(gpu), slots)
    for t, want in zip((b.cache.k_codes, b.cache.k_scales, b.cache.v_codes, b.cache.v_scales), before):
        assert torch.equal(t, want)
    b.cache.write(b.k[5:6].to(gpu), b.v[5:6].to(gpu), b.slots[7:8].to(gpu))  # token 7 of sequence 0 changes, no other
    b.k[7], b.v[7] = b.k[5], b.v[5]
    for got, x in zip(b.read(), (b.k, b.v)):
        assert torch.equal(got.cpu(), om.values(x, "mxfp4").to(torch.bfloat16))


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_write_strided(gpu, fmt):
    """Keys and values as slices of one fused projection, and with heads outermost."""
    b = _Batch(gpu, [50], 2, 64, 16, fmt, torch.float16)
    fused = torch.cat([torch.zeros(50, 3, 64, dtype=torch.float16), b.k, b.v], 1).to(gpu)
    b.cache.write(fused[:, 3:5], fused[:, 5:7], b.slots.to(gpu))
    for got, x in zip(b.read(), (b.k, b.v)):
        assert torch.equal(got.cpu(), om.values(x, fmt).to(torch.float16))
    turned = b.v.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    b.cache.write(turned, b.k.to(gpu), b.slots.to(gpu))
    for got, x in zip(b.read(), (b.v, b.k)):
        assert torch.equal(got.cpu(), om.values(x, fmt).to(torch.float16))


def test_read_of_missing_pages_is_zero(gpu):
    b = _Batch(gpu, [40], 1, 64, 16, "mxfp8", torch.bfloat16).fill()
    for bad in (-1, b.cache.num_pages, 2 ** 31 - 1, -(2 ** 31)):
        b.table[0, 1] = bad
        for got, x in zip(b.read(), (b.k, b.v)):
            want = om.values(x, "mxfp8")
            want[16:32] = 0
            assert torch.equal(got.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,heads,group,page", [
    ([1], [1], 1, 1, 16),                                  # the first token
    ([5, 33, 16], [1, 1, 1], 2, 4, 16),                    # a decoding batch
    ([700, 31, 1300, 32], [1, 1, 1, 1], 1, 7, 64),         # shared by an odd number of heads
    ([40, 100, 7], [40, 100, 7], 2, 1, 16),                # whole prompts
    ([150, 90, 64, 200], [33, 0, 64, 1], 2, 4, 32),        # chunks, a sequence without new tokens
    ([513], [300], 1, 16, 128),
    ([600, 129], [300, 129], 2, 4, 16),
    ([0, 20], [3, 2], 1, 4, 16),                           # rows that see nothing
])
def test_attend(gpu, dtype, fmt, dim, lens, new, heads, group, page):
    _Batch(gpu, lens, heads, dim, page, fmt, dtype, seed=dim + len(lens)).fill().check(new, group)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("lens,new,group", [([3, 40], [5, 2], 2), ([100, 260], [9, 130], 4), ([2, 0], [40, 1], 8)])
def test_attend_more_new_tokens_than_positions_and_not_causal(gpu, fmt, lens, new, group):
    for causal in (True, False):
        _Batch(gpu, lens, 2, 128, 16, fmt, torch.bfloat16).fill().check(new, group, causal)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 150])
def test_attend_long(gpu, dim, new):
    """Runs of keys joined, few rows over a long sequence; an estimate of the length that is too small or large."""
    b = _Batch(gpu, [5003, 77], 1, dim, 16, "mxfp4", torch.bfloat16).fill()
    for max_kv in (None, 77, 0, 2000):
        b.check([new, min(new, 77)], 4, max_kv=max_kv)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_attend_chunk_over_a_long_context(gpu, fmt):
    """Enough rows and positions for the largest tiles; ragged on both sides."""
    lens, new = [1300, 1111] * 8, [300, 290] * 8
    _Batch(gpu, lens, 8, 128, 32, fmt, torch.bfloat16).fill().check(new, 4)


@pytest.mark.parametrize("heads,dim,fmt", [(8, 128, "mxfp8"), (16, 64, "mxfp4")])
def test_offsets_beyond_32_bits(gpu, heads, dim, fmt):
    """A pool whose codes need more than 32 bits of offset, used at its end."""
    page, spare = 64, 3
    wide = 1 if fmt == "mxfp8" else 2
    pages = (1 << 32) // (heads * page * dim // wide) + spare
    cache = QuantizedKVCache(pages, page, heads, dim, fmt=fmt, dtype=torch.bfloat16, device=gpu)
    b = _Batch(gpu, [150], heads, dim, page, fmt, torch.bfloat16, spare=0)
    b.cache, b.table, b.slots = cache, b.table + (pages - 3), b.slots + (pages - 3) * page
    b.fill()
    for got, x in zip(b.read(), (b.k, b.v)):
        assert torch.equal(got.cpu(), om.values(x, fmt).to(torch.bfloat16))
    b.check([1], 2)
    b.check([140], 2)


@pytest.mark.parametrize("new", [1, 100])
def test_attend_wide_table(gpu, new):
    """A table for far longer sequences than there are."""
    b = _Batch(gpu, [200, 130], 2, 128, 16, "mxfp8", torch.bfloat16).fill()
    b.table = torch.cat([b.table, torch.full((2, 4000), -1, dtype=torch.int32)], 1)
    b.check([new, new], 4)


@pytest.mark.parametrize("scale", [0.0, 3.0, -0.5])
def test_attend_scale(gpu, scale):
    """Peaked, flat and inverted softmax."""
    _Batch(gpu, [130, 300], 1, 64, 16, "mxfp8", torch.bfloat16).fill().check([100, 1], 2, scale=scale)


@pytest.mark.parametrize("new", [1, 40, 200])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_nan_and_infinity_reach_only_rows_that_see_them(gpu, new, dim):
    """A NaN key poisons the rows that see it, a NaN value their block of the head; behind a row's last position
    neither does anything."""
    n = 260
    b = _Batch(gpu, [n], 1, dim, 16, "mxfp4", torch.bfloat16)
    p_k, p_v = n - 3, n - 20
    b.k[p_k, 0, 3] = math.inf
    b.v[p_v, 0, 40] = math.nan
    b.fill()
    _, _, o = b.attend([new], 2)
    o = o.cpu()
    last = n - new + torch.arange(new)
    want = torch.zeros(new, 2, dim, dtype=torch.bool)
    want[last >= p_v, :, 32:64] = True
    want[last >= p_k] = True
    assert torch.equal(o.isnan(), want)
    clean = _Batch(gpu, [n], 1, dim, 16, "mxfp4", torch.bfloat16).fill()
    q, _, _ = b.attend([new], 2)
    _, _, o = b.attend([new], 2, q=q)
    _, _, c = clean.attend([new], 2, q=q)
    assert torch.equal(o[last.to(gpu) < p_v], c[last.to(gpu) < p_v])


def test_attend_missing_page_is_not_seen(gpu):
    b = _Batch(gpu, [64], 1, 128, 16, "mxfp8", torch.bfloat16).fill()
    q, _, want = b.attend([1], 4)
    b.table[0, 3] = -1
    b.lens = [64]
    _, _, got = b.attend([1], 4, q=q)
    short = _Batch(gpu, [48], 1, 128, 16, "mxfp8", torch.bfloat16)
    short.k, short.v = b.k[:48], b.v[:48]
    short.fill()
    _, _, o = short.attend([1], 4, q=q)
    assert torch.allclose(got.float(), o.float(), rtol=2 ** -7, atol=2 ** -8) and not torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 90])
def test_attend_strided_queries_out_streams_and_repeats(gpu, new):
    b = _Batch(gpu, [700, 90], 2, 128, 32, "mxfp4", torch.float16).fill()
    q, _, want = b.attend([new, new], 4)
    wide = torch.zeros(2 * new, 13, 128, dtype=torch.float16)
    wide[:, 2:10] = q
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    args = (b.table.to(gpu), i32([700, 90]), i32([0, new, 2 * new]), new)
    out = torch.empty_like(want)
    assert b.cache.attend(wide.to(gpu)[:, 2:10], *args, out=out) is out and torch.equal(out, want)
    turned = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    assert torch.equal(b.cache.attend(turned, *args), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = b.cache.attend(turned, *args)
    stream.synchronize()
    assert torch.equal(got, want)


def test_step_in_a_graph(gpu):
    """Write and attend captured once, replayed as the sequence grows."""
    b = _Batch(gpu, [600], 2, 64, 16, "mxfp8", torch.bfloat16).fill()
    table = b.table.to(gpu)
    lens = torch.tensor([500], dtype=torch.int32, device=gpu)
    slot, k, v = b.slots[499:500].to(gpu), b.k[499:500].to(gpu), b.v[499:500].to(gpu)
    q = torch.randn(1, 8, 64, generator=b.g).to(torch.bfloat16).to(gpu)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    out = torch.empty_like(q)

    def step():
        b.cache.write(k, v, slot)
        b.cache.attend(q, table, lens, starts, 1, out=out)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in (520, 555, 600):
        lens.fill_(n)
        slot.copy_(b.slots[n - 1: n])
        k.copy_(b.k[n - 1: n])
        v.copy_(b.v[n - 1: n])
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        assert torch.equal(got, out)


def test_refusals(gpu):
    new = lambda **k: QuantizedKVCache(**{**dict(num_pages=4, page_size=16, heads=2, head_dim=64, device=gpu), **k})  # noqa: E731
    for bad, match in ((dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"),
                       (dict(head_dim=80), "head_dim"), (dict(heads=0), "one head"),
                       (dict(fmt="int4"), "unknown microscaled"), (dict(dtype=torch.float32), "bfloat16 or float16"),
                       (dict(device="cpu"), "ROCm device")):
        with pytest.raises(ValueError, match=match):
            new(**bad)
    c = new()
    with pytest.raises(ValueError, match="v_scales must be"):
        QuantizedKVCache.from_tensors(c.k_codes, c.k_scales, c.v_codes, c.v_scales[:, :, :2])
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    slots = torch.zeros(3, dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError, match="k must be torch.bfloat16"):
        c.write(k.half(), k, slots)
    with pytest.raises(ValueError, match="one shape"):
        c.write(k, k[:2], slots)
    with pytest.raises(ValueError, match="slots must be"):
        c.write(k, k, slots.int())
    table = torch.zeros(1, 2, dtype=torch.int32, device=gpu)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    with pytest.raises(ValueError, match="starts must be"):
        c.read(table, i32([0]), 1)
    with pytest.raises(ValueError, match="total"):
        c.read(table, i32([0, 1]), -1)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=gpu)
    good = (table, i32([5]), i32([0, 1]), 1)
    with pytest.raises(ValueError, match="query heads"):
        c.attend(q[:, :3], *good)
    with pytest.raises(ValueError, match="q must be"):
        c.attend(q[..., :32], *good)
    with pytest.raises(ValueError, match="kv_lens must be"):
        c.attend(q, table, i32([5, 5]), i32([0, 1]), 1)
    with pytest.raises(ValueError, match="do not fit"):
        c.attend(q, table, i32([5]), i32([0, 1]), 0)
    with pytest.raises(ValueError, match="max_kv"):
        c.attend(q, *good, max_kv=33)
    with pytest.raises(ValueError, match="out must be"):
        c.attend(q, *good, out=q.float())
    with pytest.raises(ValueError, match="block_table"):
        c.attend(q, table.long(), *good[1:])
    c.write(k[:0], k[:0], slots[:0])
    assert c.attend(q[:0], table[:0], i32([]), i32([0]), 0).shape == (0, 4, 64)


def _poisoned_and_clean(b, clean, spots, new, group):
    """Outputs over a cache with NaN blocks and over the same one without, and where the first must be NaN.  ``spots``:
    (sequence, position, block of the head or None for the key)."""
    heads, dim = b.cache.heads, b.cache.head_dim
    q, _, o = b.attend(new, group)
    _, _, c = clean.attend(new, group, q=q)
    want = torch.zeros(sum(new), heads, group, dim, dtype=torch.bool)
    for i, pos, head, block in spots:
        a = sum(new[:i])
        sees = a + torch.nonzero(b.lens[i] - new[i] + torch.arange(new[i]) >= pos).flatten()
        if block is None:
            want[sees, head] = True
        else:
            want[sees, head, :, 32 * block: 32 * block + 32] = True
    return o.cpu(), c.cpu(), want.flatten(1, 2)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 30, 40, 200])
def test_attend_nan_blocks_in_each_format(gpu, bad, fmt, dtype, dim, new):
    """16-row tiles (1 and 30 new tokens) and 128-row ones: NaN exactly where a row sees the key or the value block; all
    else is bit for bit what it is without them, in the tile that holds them too."""
    n = 260
    p_k, p_v = n - 3, n - 20
    b, clean = (_Batch(gpu, [n], 2, dim, 16, fmt, dtype) for _ in range(2))
    b.k[p_k, 0, 3], b.v[p_v, 1, 40], b.v[p_v + 9, 1, 7] = bad, bad, bad
    o, c, want = _poisoned_and_clean(b.fill(), clean.fill(), [(0, p_k, 0, None), (0, p_v, 1, 1), (0, p_v + 9, 1, 0)],
                                     [new], 2)
    assert torch.equal(o.isnan(), want) and torch.equal(o[~want], c[~want])


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_attend_nan_blocks_in_the_largest_tiles(gpu, fmt):
    """256 rows a work-group, as above."""
    lens, new = [300] * 16, [70] * 16
    b, clean = (_Batch(gpu, lens, 8, 128, 32, fmt, torch.bfloat16) for _ in range(2))
    b.v[5 * 300 + 270, 3, 100], b.k[7 * 300 + 290, 6, 1] = math.nan, math.inf
    o, c, want = _poisoned_and_clean(b.fill(), clean.fill(), [(5, 270, 3, 3), (7, 290, 6, None)], new, 4)
    assert torch.equal(o.isnan(), want) and torch.equal(o[~want], c[~want])


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_read_nan_blocks(gpu, fmt, dtype):
    """A block with a NaN or an infinity reads back as NaN in 16 bits, the other blocks as they are."""
    b = _Batch(gpu, [40], 2, 64, 16, fmt, dtype)
    b.k[3, 1, 40], b.k[9, 0, 0], b.v[5, 0, 2], b.v[6, 1, 63] = math.nan, math.inf, -math.inf, math.nan
    b.fill()
    for got, x in zip(b.read(), (b.k, b.v)):
        got, want = got.cpu(), om.values(x, fmt).to(dtype)
        assert int(want.isnan().sum()) == 64 and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,dim,group", [
    ([40, 17], [1, 1], 64, 4),          # 16 rows, one run of keys
    ([3000, 1500], [1, 2], 128, 7),     # 16 rows, runs joined
    ([300, 200], [90, 40], 128, 2),     # 128 rows, one run
    ([6000, 900], [60, 33], 64, 4),     # 128 rows, runs joined
])
def test_attend_tokens_outside_every_sequence_are_zero(gpu, dtype, lens, new, dim, group):
    """Padding before and behind the sequences, and a sequence longer than max_q: 0 with lse -inf; every other token is bit
    for bit what it is without them."""
    b = _Batch(gpu, lens, 2, dim, 16, "mxfp8", dtype).fill()
    n = sum(new)
    table, kv = b.table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    q = torch.randn(n + 9, 2 * group, dim, generator=b.g).to(dtype).to(gpu)
    starts, most = [4, 4 + new[0], 4 + n], max(new)
    front = torch.cat([q[4: 4 + n], q[:9]])  # as many tokens: the same split of the work
    want, lse = (t[:n] for t in b.cache.attend(front, table, kv, i32([0, new[0], n]), max(most, n + 9), return_lse=True))
    out = torch.full_like(q, math.nan)
    torch.full((n + 9, 2 * group), math.nan, device=gpu)  # what the memory of lse may hold
    got, gl = b.cache.attend(q, table, kv, i32(starts), max(most, n + 9), out=out, return_lse=True)
    none = torch.ones(n + 9, dtype=torch.bool)
    none[4: 4 + n] = False
    assert not bool(got[none].any()) and bool((gl[none] == -math.inf).all())
    assert torch.equal(got[4: 4 + n], want) and torch.equal(gl[4: 4 + n], lse)


@pytest.mark.parametrize("lens,new,max_q,group", [([50, 60], [5, 1], 3, 4), ([4000, 60], [5, 1], 3, 4),
                                                  ([500, 300], [200, 5], 103, 2), ([6000, 300], [100, 5], 53, 2)])
def test_attend_tokens_behind_max_q_are_zero(gpu, lens, new, max_q, group):
    """A caller's max_q below a sequence's new tokens: those behind it are 0, the others are right."""
    dim = 64
    b = _Batch(gpu, lens, 1, dim, 16, "mxfp4", torch.bfloat16).fill()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    n = sum(new)
    q = torch.randn(n, group, dim, generator=b.g).to(torch.bfloat16).to(gpu)
    args = (b.table.to(gpu), i32(lens), i32([0, new[0], n]))
    got, lse = b.cache.attend(q, *args, max_q, out=torch.full_like(q, math.nan), return_lse=True)
    want, wl = b.cache.attend(q, *args, max(new), return_lse=True)
    held = torch.cat([torch.arange(m) < max_q for m in new])
    assert not bool(got[~held].any()) and bool((lse[~held] == -math.inf).all())
    assert torch.allclose(got[held].float(), want[held].float(), rtol=2 ** -6, atol=2 ** -8)
    assert torch.allclose(lse[held], wl[held], rtol=1e-5, atol=1e-5)


def test_attend_refuses_tokens_without_sequences(gpu):
    """The C entry: tokens, but no sequence or none with a token."""
    from mpq_amd import _lib

    c = QuantizedKVCache(2, 16, 1, 64, device=gpu)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    out, lens = torch.empty_like(q), torch.zeros(2, dtype=torch.int32, device=gpu)
    for batch, max_q in ((0, 3), (1, 0)):
        rc = _lib.load().mpq_kv_attend(q.data_ptr(), 1, 3, 128, 64, 2, batch, lens.data_ptr(), 1, lens.data_ptr(),
                                       lens.data_ptr(), max_q, 16, *c._call, 0.125, 1, out.data_ptr(), None, None, 0,
                                       _lib.stream_handle(gpu))
        with pytest.raises(Exception, match="do not fit"):
            _lib.check(rc, "mpq_kv_attend")


def test_attend_backward_raises(gpu):
    b = _Batch(gpu, [40], 1, 64, 16, "mxfp8", torch.bfloat16).fill()
    q, _, want = b.attend([3], 2)
    for which in (0, 1):
        _, _, got = b.attend([3], 2, q=q.clone().requires_grad_(), return_lse=True)
        assert torch.equal(got[0], want)
        with pytest.raises(RuntimeError, match="attend has no gradient"):
            got[which].float().sum().backward()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_write_more_tokens_than_a_launch_has_threads(gpu, fmt):
    """A lane an octet: 2^19 tokens of 1024 heads of 64 are 2^32 threads, more than one launch takes."""
    H, n = 1024, (1 << 19) + 9
    cache = QuantizedKVCache(2, 16, H, 64, fmt=fmt, device=gpu)
    at = [0, (1 << 18) - 1, 1 << 18, (1 << 19) - 1, 1 << 19, n - 1]
    slots = torch.full((n,), -1, dtype=torch.int64, device=gpu)
    slots[torch.tensor(at, device=gpu)] = torch.arange(6, device=gpu)
    g = torch.Generator().manual_seed(3)
    base = torch.randn(n + 64 * 8, generator=g).to(torch.bfloat16)  # a token's rows start one value after its predecessor's
    k = base.to(gpu).as_strided((n, H, 64), (1, 0, 1))
    cache.write(k, k, slots)
    table = torch.tensor([[0]], dtype=torch.int32, device=gpu)
    got = cache.read(table, torch.tensor([0, 6], dtype=torch.int32, device=gpu), 6)
    want = torch.stack([om.values(base[i: i + 64], fmt) for i in at]).to(torch.bfloat16).unsqueeze(1).expand(6, H, 64)
    for t in got:
        assert torch.equal(t.cpu(), want)


def test_read_more_tokens_than_a_launch_has_threads(gpu):
    """As above, 64 GiB of keys and as many of values."""
    H, n = 1024, (1 << 19) + 9
    torch.cuda.empty_cache()
    cache = QuantizedKVCache(3, 16, H, 64, device=gpu)
    g = torch.Generator().manual_seed(3)
    k = torch.randn(48, H, 64, generator=g).to(torch.bfloat16)
    cache.write(k.to(gpu), -k.to(gpu), torch.arange(48, device=gpu))
    table = torch.full((1, n // 16 + 1), -1, dtype=torch.int32, device=gpu)
    pages = {0: 2, (1 << 18) // 16 - 1: 0, (1 << 18) // 16: 1, (1 << 19) // 16 - 1: 2, (1 << 19) // 16: 0}
    for at, page in pages.items():
        table[0, at] = page
    got = cache.read(table, torch.tensor([0, n], dtype=torch.int32, device=gpu), n)
    values = om.values(k, "mxfp8").to(torch.bfloat16)
    for t, sign in zip(got, (1, -1)):
        for at, page in pages.items():
            some = t[16 * at: 16 * at + 16].cpu()
            assert torch.equal(some, sign * values[16 * page: 16 * page + len(some)])
            for empty in (16 * at - 1, 16 * at + 16):
                if 0 <= empty < n and empty // 16 not in pages:
                    assert not bool(t[empty].any())
    del got, t
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt,dtype", [("mxfp8", torch.bfloat16), ("mxfp4", torch.float16)])
@pytest.mark.parametrize("lens,new,heads,group,page", [
    ([200, 90], [1, 5], 2, 4, 16),       # 16 rows, one run of keys
    ([3000, 170], [2, 1], 2, 4, 64),     # 16 rows, runs joined
    ([300, 130], [100, 70], 2, 2, 16),   # 128 rows
    ([5000, 300], [60, 3], 1, 4, 32),    # 128 rows, runs joined
    ([300] * 16, [70] * 16, 8, 4, 32),   # 256 rows
])
def test_attend_missing_pages_inside_the_context(gpu, fmt, dtype, lens, new, heads, group, page):
    """The first page, one in the middle and the last one of a sequence are named wrongly: their positions are seen by no
    row, against 64 bits."""
    dim = 128 if heads != 2 else 64
    b = _Batch(gpu, lens, heads, dim, page, fmt, dtype, seed=3).fill()
    held, whole = (lens, b.table.clone()), -(-lens[0] // page)
    for bad, at in ((-1, [whole // 2]), (b.cache.num_pages, [0, whole // 2]), (2 ** 31 - 1, [whole - 1]),
                    (-(2 ** 31), [0, 1, whole - 1])):
        b.table = held[1].clone()
        b.table[0, at] = bad
        q, starts, (o, lse) = b.attend(new, group, return_lse=True)
        for i, n in enumerate(lens):
            hidden = torch.zeros(n, dtype=torch.bool)
            if i == 0:
                hidden = torch.isin(torch.arange(n) // page, torch.tensor(at))
            _compare(b, i, q[starts[i]: starts[i + 1]], o[starts[i]: starts[i + 1]], lse[starts[i]: starts[i + 1]], new[i],
                     hidden)


def _compare(b, i, q, o, lse, new, hidden):
    """Sequence i against 64 bits, within the bounds of _Batch.check."""
    dim, u = b.cache.head_dim, UNIT[b.dtype]
    o, lse = o.cpu().double(), lse.cpu().double()
    k, v = (om.values(t[b.starts[i]: b.starts[i + 1]], b.fmt) for t in (b.k, b.v))
    want, wl, pv, mass, big = om.attend(q, k, v, new, dim ** -0.5, True, hidden)
    delta = (2.0 ** -24 * (dim + 8) * big).unsqueeze(-1)
    tol = u * want.abs() * 1.01 + (1.01 * u + 2 * delta + 2.0 ** -20) * pv + 1e-30
    if b.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (1 + mass)
    assert bool(((o - want).abs() <= tol).all()), (i, float(((o - want).abs() / tol).max()))
    seen = torch.isfinite(wl)
    assert torch.equal(seen, torch.isfinite(lse)) and bool((lse[~seen] == -math.inf).all())
    assert bool(((lse - wl)[seen].abs() <= (2.0 ** -20 * (1 + wl.abs()) + 2 * delta.squeeze(-1))[seen]).all())


@pytest.mark.parametrize("fmt,dtype,dim", [("mxfp8", torch.bfloat16, 128), ("mxfp4", torch.float16, 64)])
def test_attend_chunk_beside_single_tokens(gpu, fmt, dtype, dim):
    """One batch of a chunk, single tokens over long and short contexts and an idle sequence: tiles of 128 rows of which the
    single tokens fill few, runs that some rows do not reach."""
    _Batch(gpu, [2100, 700, 1, 1500, 33, 900], 2, dim, 16, fmt, dtype).fill().check([300, 1, 1, 1, 0, 2], 4)
    _Batch(gpu, [5000, 700, 4000], 1, dim, 16, fmt, dtype).fill().check([40, 1, 1], 4)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -20, 2.0 ** -15])
@pytest.mark.parametrize("new", [1, 90])
def test_small_float16_values_are_kept(gpu, fmt, size, new):
    """A float16 input is a multiple of 2^-24 and so is its quantised value, in at most four significant bits: float16
    operands hold what a float16 cache was given."""
    b = _Batch(gpu, [150], 1, 64, 16, fmt, torch.float16)
    b.k, b.v = (b.k.float() * size).half(), (b.v.float() * size).half()
    b.fill()
    for got, x in zip(b.read(), (b.k, b.v)):
        assert torch.equal(got.cpu(), om.values(x, fmt).half())
    b.check([new], 2, scale=1.0 / size / 8)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("lens,new", [([260], [20]), ([3000], [3]), ([260], [150]), ([6000], [60])])
def test_attend_nan_queries_stay_in_their_rows(gpu, fmt, lens, new):
    """A NaN or infinite query makes its own row NaN; its neighbours in the tile keep their bits."""
    b = _Batch(gpu, lens, 2, 64, 16, fmt, torch.bfloat16).fill()
    q, _, want = b.attend(new, 2)
    q[1, 3, 5], q[-1, 0, 0] = math.nan, math.inf
    _, _, got = b.attend(new, 2, q=q)
    bad = torch.zeros(sum(new), 4, dtype=torch.bool)
    bad[1, 3], bad[-1, 0] = True, True
    got, want = got.cpu(), want.cpu()
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], want[~bad])
