"""Paged 4-bit cache on the GPU: every operator against its definition in 64 bits (tests/_kv4.py), and what must not happen."""
import ctypes as C
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _kv4  # noqa: E402

pytestmark = pytest.mark.gpu


def queries(rows, heads, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, heads * 128, generator=g) * scale).bfloat16().cuda()


def check_attention(cache, b, entries, q, out, layer=0):
    """entries: (sequence, first position, first row, rows) of what is to be compared."""
    torch.cuda.synchronize()
    for seq, first, r0, n in entries:
        want, bound = _kv4.attention(cache, seq, first, q[r0:r0 + n], layer)
        off = (out[r0:r0 + n].double().cpu() - want).abs()
        assert bool((off <= bound).all()), (seq, first, n, float((off / bound).max()))


LAYOUTS = [(32, 8), (8, 8), (16, 1), (6, 2), (10, 2), (1, 1)]


@pytest.mark.parametrize("q_heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 200, 1000])
def test_single_tokens(mine, capi, q_heads, kv_heads, length):
    cache = _kv4.Cache(mine, capi, 40, kv_heads=kv_heads, q_heads=q_heads, stride=16)
    _kv4.fill(cache, 2, length, seed=length)
    b = cache.batch([2], [1], [length - 1])
    q = queries(1, q_heads)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(2, length - 1, 0, 1)], q, out)


@pytest.mark.parametrize("q_heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("first,rows", [(0, 2), (0, 17), (62, 3), (63, 2), (100, 7), (120, 40), (5, 64), (0, 130), (300, 129), (1, 255), (64, 64)])
def test_slices(mine, capi, q_heads, kv_heads, first, rows):
    cache = _kv4.Cache(mine, capi, 40, kv_heads=kv_heads, q_heads=q_heads, stride=16, rows=rows)
    _kv4.fill(cache, 1, first + rows, seed=rows)
    b = cache.batch([1], [rows], [first])
    q = queries(rows, q_heads)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(1, first, 0, rows)], q, out)


@pytest.mark.parametrize("hint", [None, 0, 1, 2, 5, 1000])
def test_ragged_batch_of_tokens_and_slices(mine, capi, hint):
    """Single tokens, slices, an entry without rows, refused entries and padding in one batch; the hint does not change what is right."""
    lens, counts = [500, 3, 77, 1, 640, 130], [1, 3, 0, 1, 33, 70]
    cache = _kv4.Cache(mine, capi, 60, kv_heads=2, q_heads=8, max_seqs=9, stride=12, rows=200)
    seqs = [7, 0, 3, 5, 1, 2]
    for i, (s, t) in enumerate(zip(seqs, lens)):
        _kv4.fill(cache, s, t, seed=i)
    pos0 = [t - n for t, n in zip(lens, counts)]
    total = sum(counts)
    # two more entries that see nothing: refused by reserve, and of a sequence that is not there
    b = cache.batch(seqs + [8, 99, -1], counts + [2, 3, 1], pos0 + [-1, 4, 4], rows=total + 6 + 5, max_rows=hint)
    q = queries(b.rows, 8)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    at, entries = 0, []
    for s, p, n in zip(seqs, pos0, counts):
        entries.append((s, p, at, n))
        at += n
    check_attention(cache, b, [e for e in entries if e[3]], q, out)
    assert bool((out[total:total + 6] == 0).all()) and bool((out[total + 6:] == 7).all())


def test_positions_without_a_page_are_left_out(mine, capi):
    cache = _kv4.Cache(mine, capi, 20, kv_heads=2, q_heads=8, stride=8, rows=80)
    _kv4.fill(cache, 0, 400, seed=1)
    cache.table[0, 2], cache.table[0, 4], cache.table[0, 5] = -1, 20, 2 ** 31 - 1  # freed, and outside the pool
    for first, n in ((399, 1), (330, 70), (150, 1), (128, 40)):
        b = cache.batch([0], [n], [first])
        q = queries(n, 8)
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        check_attention(cache, b, [(0, first, 0, n)], q, out)
    cache.table[0, :] = -1
    for n in (1, 70):
        b = cache.batch([0], [n], [100])
        q = queries(n, 8)
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        torch.cuda.synchronize()
        assert bool((out == 0).all())


def test_positions_behind_the_table_are_left_out(mine, capi):
    """A position may be larger than the table has room for: what the table has is seen."""
    cache = _kv4.Cache(mine, capi, 20, kv_heads=1, q_heads=4, stride=2, rows=40)
    _kv4.fill(cache, 0, 128, seed=1)
    q = queries(33, 4)
    for n in (1, 33):
        for first in (127, 128, 1000, 2 ** 30):
            b = cache.batch([0], [n], [first])
            out = torch.full_like(q[:n], 7.0)
            cache.attention(b, q[:n].contiguous(), out)
            torch.cuda.synchronize()
            k, v, mass, _ = cache.values(0, 128)
            for r in range(n):
                want, bound = _kv4.attention(cache, 0, 127, q[r:r + 1])
                if first + r >= 127:
                    assert bool(((out[r:r + 1].double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("rows", [1, 2, 40, 200])
def test_garbage_behind_the_last_position_is_not_seen(mine, capi, rows):
    """Pools start as NaN bytes in these tests, so every block's tail holds NaN scales; here the masked scores would be the largest too."""
    cache = _kv4.Cache(mine, capi, 20, kv_heads=2, q_heads=8, stride=8, rows=rows, fill=0x7B)  # f16 0x7B7B = 61280
    _kv4.fill(cache, 0, 200 + rows, seed=3)
    b = cache.batch([0], [rows], [200])
    q = queries(rows, 8)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(0, 200, 0, rows)], q, out)


@pytest.mark.parametrize("scale", [1e-3, 1e-2, 30.0, 300.0])
@pytest.mark.parametrize("rows", [1, 150])
def test_value_ranges(mine, capi, scale, rows):
    """Keys and values far from 1, queries the other way round so that the scores stay moderate."""
    cache = _kv4.Cache(mine, capi, 20, kv_heads=2, q_heads=8, stride=8, rows=rows)
    _kv4.fill(cache, 0, 330, seed=5, scale=scale)
    b = cache.batch([0], [rows], [330 - rows])
    q = queries(rows, 8, scale=1.5 / scale)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(0, 330 - rows, 0, rows)], q, out)


@pytest.mark.parametrize("rows", [1, 20, 150])
def test_values_at_the_ends_of_f16(mine, capi, rows):
    """Groups that stand for -65504 .. 65536: nothing on the way may leave f16.  (The bound of _kv4.attention holds relative to what is summed.)"""
    cache = _kv4.Cache(mine, capi, 20, kv_heads=2, q_heads=8, stride=8, rows=rows)
    _kv4.fill(cache, 0, 330, seed=5, scale=1e6)
    assert float(cache.values(0, 330)[1].abs().max()) > 65504
    b = cache.batch([0], [rows], [330 - rows])
    q = queries(rows, 8, scale=1e-6)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(0, 330 - rows, 0, rows)], q, out)


@pytest.mark.parametrize("rows", [1, 3, 33, 150])
def test_out_may_be_the_queries(mine, capi, rows):
    cache = _kv4.Cache(mine, capi, 40, kv_heads=2, q_heads=8, stride=32, rows=rows)
    _kv4.fill(cache, 0, 1500, seed=5)
    b = cache.batch([0], [rows], [1500 - rows])
    q = queries(rows, 8)
    out, both = torch.full_like(q, 7.0), q.clone()
    cache.attention(b, q, out)
    cache.attention(b, both, both)
    torch.cuda.synchronize()
    assert torch.equal(both, out)


@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (6, 2), (16, 1)])
def test_many_slices(mine, capi, q_heads, kv_heads):
    """More units than there are SMs, of all lengths: CTAs that end one unit, have others whole and begin a third; next to single tokens."""
    import random
    rng = random.Random(q_heads)
    counts = [rng.choice((1, 2, 17, 40, 64, 65, 100, 128, 129, 200, 300)) for _ in range(14)]
    firsts = [rng.choice((0, 1, 63, 64, 100, 500)) for _ in counts]
    total = sum(counts)
    cache = _kv4.Cache(mine, capi, 200, kv_heads=kv_heads, q_heads=q_heads, max_seqs=14, stride=16, rows=total)
    for i, (p, n) in enumerate(zip(firsts, counts)):
        _kv4.fill(cache, i, p + n, seed=i)
    b = cache.batch(range(14), counts, firsts)
    q = queries(total, q_heads)
    outs = []
    for _ in range(3):
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        outs.append(out)
    at, entries = 0, []
    for i, (p, n) in enumerate(zip(firsts, counts)):
        entries.append((i, p, at, n))
        at += n
    check_attention(cache, b, entries, q, outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)
    cache.call("status", None)


def test_a_long_slice(mine, capi):
    """CTAs that walk many pages of a unit, and units cut over many CTAs."""
    cache = _kv4.Cache(mine, capi, 120, kv_heads=1, q_heads=4, max_seqs=1, stride=128, rows=700)
    _kv4.fill(cache, 0, 7000, seed=3)
    q = queries(700, 4)
    for n in (700, 65):
        b = cache.batch([0], [n], [7000 - n])
        out = torch.full_like(q[:n], 7.0)
        cache.attention(b, q[:n].contiguous(), out)
        check_attention(cache, b, [(0, 7000 - n, 0, n)], q[:n], out)


LINES = {
    "no more than a warp's worth each": [1, 3, 16, 2, 40],
    "parts of CTAs": [700, 640, 650, 700, 690, 610, 500, 700, 100],
    "one far longer than the others": [6000] + [90, 100, 1, 64] * 4,
    "parts of warps": [500, 513, 480, 511, 512, 497] * 4 + [513, 1],
    "stretches of warps": [2100, 300, 64, 1, 1700, 900, 17, 3000] * 3,
    "more units than warps": [33, 70, 1, 16, 128, 64, 99, 130, 5, 48] * 16,
}


@pytest.mark.parametrize("name", LINES)
@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (16, 1)])
def test_lines_of_single_tokens(mine, capi, name, q_heads, kv_heads):
    """Batches of single tokens that are cut in each of the ways there are, three times with the same bits."""
    lens = LINES[name]
    n = len(lens)
    cache = _kv4.Cache(mine, capi, sum((x + 63) // 64 for x in lens) + 1, kv_heads=kv_heads, q_heads=q_heads, max_seqs=n, stride=96, rows=n)
    for i, x in enumerate(lens):
        _kv4.fill(cache, i, x, seed=i)
    b = cache.batch(range(n), [1] * n, [x - 1 for x in lens])
    q = queries(n, q_heads)
    outs = []
    for _ in range(3):
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        outs.append(out)
    check_attention(cache, b, [(i, x - 1, i, 1) for i, x in enumerate(lens)], q, outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("lens,counts", [([7000] + [50] * 12, [32] + [40] * 12), ([300, 250, 333], [70, 64, 65]), ([64] * 3, [33] * 3), ([4000, 3900], [300, 290])])
def test_few_slices_of_unequal_lengths(mine, capi, lens, counts):
    """No more units than SMs, cut into parts of their own or, where one is far longer, along one line."""
    n, total = len(lens), sum(counts)
    cache = _kv4.Cache(mine, capi, sum((x + 63) // 64 for x in lens) + 1, kv_heads=8, q_heads=32, max_seqs=n, stride=110, rows=total)
    for i, x in enumerate(lens):
        _kv4.fill(cache, i, x, seed=i)
    firsts = [x - c for x, c in zip(lens, counts)]
    b = cache.batch(range(n), counts, firsts)
    q = queries(total, 32)
    outs = []
    for _ in range(2):
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        outs.append(out)
    check_attention(cache, b, [(i, p, sum(counts[:i]), c) for i, (p, c) in enumerate(zip(firsts, counts))], q, outs[0])
    assert torch.equal(outs[0], outs[1])
    cache.call("status", None)


@pytest.mark.parametrize("q_heads,kv_heads", [(48, 3), (32, 8)])
def test_many_slices_of_few_rows(mine, capi, q_heads, kv_heads):
    """Units with rows in one of their two tiles, several to a CTA: a result is not read before its last product, whatever the other tile does meanwhile."""
    n, group = 200, q_heads // kv_heads
    counts = [9 * 4 // group + i % 7 for i in range(n)]
    lens = [c + 60 + 7 * (i % 13) for i, c in enumerate(counts)]
    total = sum(counts)
    cache = _kv4.Cache(mine, capi, sum((x + 63) // 64 for x in lens) + 1, kv_heads=kv_heads, q_heads=q_heads, max_seqs=n, stride=4, rows=total)
    for i, x in enumerate(lens):
        _kv4.fill(cache, i, x, seed=i)
    firsts = [x - c for x, c in zip(lens, counts)]
    b = cache.batch(range(n), counts, firsts, max_rows=1000)
    q = queries(total, q_heads)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(i, firsts[i], sum(counts[:i]), counts[i]) for i in range(0, n, 9)], q, out)
    for _ in range(200):
        again = torch.full_like(q, 7.0)
        cache.attention(b, q, again)
        assert torch.equal(again, out)
    cache.call("status", None)


def test_as_many_sequences_as_a_batch_takes(mine, capi):
    n = 1024
    cache = _kv4.Cache(mine, capi, 1100, kv_heads=1, q_heads=2, max_seqs=n, stride=2, rows=n + 40)
    cache.refs[:] = 0
    book = [(i * 7) % 61 + 1 for i in range(n)]
    b = cache.batch(range(n), book, max_rows=100)
    cache.reserve(b)
    torch.cuda.synchronize()
    assert cache.info.cpu().tolist() == [1100 - n, 0] and cache.table[:, 0].cpu().tolist() == list(range(n))
    for i in (0, 1, 511, 512, 1022, 1023):
        _kv4.fill(cache, i, book[i], seed=i, order=torch.tensor([i]))
    b = cache.batch(range(n), [1] * n, [t - 1 for t in book])
    q = queries(n, 2)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(i, book[i] - 1, i, 1) for i in (0, 1, 511, 512, 1022, 1023)], q, out)
    b = cache.batch(range(n), [1] * 511 + [40] + [1] * 512, [max(0, t - 1) for t in book])  # one of them a slice
    cache.pages[511:513] = 0
    q = queries(n + 39, 2)
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    check_attention(cache, b, [(0, book[0] - 1, 0, 1), (1023, book[1023] - 1, n + 38, 1)], q, out)


@pytest.mark.parametrize("rows", [1, 33])
def test_queries_of_zero_and_of_extreme_size(mine, capi, rows):
    cache = _kv4.Cache(mine, capi, 20, kv_heads=1, q_heads=4, stride=8, rows=rows)
    _kv4.fill(cache, 0, 100, seed=5)
    b = cache.batch([0], [rows], [100 - rows])
    for scale in (0.0, 1e-38, 1e-20):
        q = queries(rows, 4, scale=scale)
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        check_attention(cache, b, [(0, 100 - rows, 0, rows)], q, out)
    q = queries(rows, 4)
    q[0, 5], q[0, 3 * 128 + 7] = float("nan"), float("inf")
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    torch.cuda.synchronize()
    assert bool(out[0, :128].isnan().all()) and not bool(out[0, 128:256].isnan().any())
    if rows > 1:  # another row's queries are another row's
        want, bound = _kv4.attention(cache, 0, 100 - rows + 1, q[1:])
        assert bool(((out[1:].double().cpu() - want).abs() <= bound).all())


def test_long_sequence_is_put_together_the_same_every_time(mine, capi):
    """Many CTAs share each unit; the result does not depend on which of them ends last.  The counters are back at zero each time."""
    cache = _kv4.Cache(mine, capi, 700, kv_heads=2, q_heads=8, max_seqs=3, stride=512)
    _kv4.fill(cache, 0, 32000, seed=1)
    _kv4.fill(cache, 2, 9000, seed=2)
    b = cache.batch([0, 2], [1, 2], [31999, 8998])
    q = queries(3, 8)
    outs = []
    for _ in range(20):
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        outs.append(out)
    check_attention(cache, b, [(0, 31999, 0, 1), (2, 8998, 1, 2)], q, outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)
    assert not bool(cache.work[:256].any()) and not bool(cache.work[-64 * 2 * 4:].any())


def test_one_workspace_for_calls_of_all_sizes(mine, capi):
    """Calls with different numbers of rows, page operators between them: each finds the counters at zero."""
    cache = _kv4.Cache(mine, capi, 60, kv_heads=2, q_heads=8, max_seqs=3, stride=32, rows=300)
    _kv4.fill(cache, 0, 1300, seed=1)
    q = queries(300, 8)
    for i, rows in enumerate((1, 70, 2, 300, 1, 33, 5, 256, 3, 8)):
        b = cache.batch([0], [rows], [1300 - rows])
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        check_attention(cache, b, [(0, 1300 - rows, 0, rows)], q, out)
        if i % 3 == 2:
            cache.fork([0], [1], [1000])
            cache.release([1])
            cache.compact()


def test_offsets_beyond_32_bits(mine, capi):
    """A pool of 6.5 GB; the sequence's pages lie at both ends of it."""
    layers, heads = 36, 8
    cache = _kv4.Cache(mine, capi, 2200, layers=layers, kv_heads=heads, q_heads=32, max_seqs=2, stride=8, rows=70, fill=0)
    order = torch.tensor([2199, 0, 1500, 2198])
    _kv4.fill(cache, 1, 250, seed=1, order=order, layer=35)
    for n in (1, 70):
        b = cache.batch([1], [n], [250 - n])
        q = queries(n, 32)
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out, layer=35)
        check_attention(cache, b, [(1, 250 - n, 0, n)], q, out, layer=35)
    qkv = queries(3, 48)
    q = torch.zeros(3, 32 * 128, dtype=torch.bfloat16, device="cuda")
    b = cache.batch([1], [3], [191])  # the end of page 1500, the start of page 2198
    cache.append(b, qkv, q, layer=35)
    torch.cuda.synchronize()
    _, v, _, _ = cache.values(1, 194, layer=35)
    want = _kv4.quantise(qkv[:, 40 * 128:].float().cpu().view(3, 8, 128).transpose(0, 1))
    assert torch.equal(v[:, 191:194], want[0].double() * want[1].double() + want[2].double())


# ---- append and read ------------------------------------------------------------------------------------------------------

def rotated(x, w, pos, eps, base):
    """Norm and rotation of heads x [rows, heads, 128] in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a = pos.double()[:, None, None] * base ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    z = torch.empty_like(y)
    z[..., 0::2] = y[..., 0::2] * a.cos() - y[..., 1::2] * a.sin()
    z[..., 1::2] = y[..., 0::2] * a.sin() + y[..., 1::2] * a.cos()
    return z


def check_append(cache, b, entries, qkv, q, q_norm, k_norm, eps, base, layer=0):
    torch.cuda.synchronize()
    hq, hk = cache.q_heads, cache.kv_heads
    x = qkv.cpu().view(qkv.shape[0], hq + 2 * hk, 128)
    cpu = lambda t: None if t is None else t.cpu()  # noqa: E731
    for seq, first, r0, n in entries:
        pos, rows = torch.arange(first, first + n), slice(r0, r0 + n)
        want = rotated(x[rows, :hq], cpu(q_norm), pos, eps, base)
        # 32 bits: a norm within 2^-20 (128 squares, a root, a quotient, two products), an angle's cosine and sine within 2^-22, the turn
        # within 2^-22 of the pair's length, which is at most sqrt(2) times its larger part; then bf16
        pair = want.unflatten(-1, (64, 2)).norm(dim=-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
        off = (q[rows].double().cpu().view_as(want) - want).abs()
        assert bool((off <= want.abs() * 2 ** -8 + pair * 2 ** -19).all())
        k, v, _, there = cache.values(seq, first + n, layer)
        assert bool(there[first:].all())
        # values are quantised from what came in: the documented rule to the bit
        c, s, m = _kv4.quantise(x[rows, hq + hk:].float().transpose(0, 1))
        assert torch.equal(v[:, first:], c.double() * s.double() + m.double())
        # keys from the 32-bit result: half a step, the f16 roundings of m (2^-11) and of s (2^-11, fifteen times), and that result's own error
        want = rotated(x[rows, hq:hq + hk], cpu(k_norm), pos, eps, base).transpose(0, 1)
        g = want.unflatten(-1, (4, 32))
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = (hi - lo) / 15
        # both roundings may leave the ends outside: a value there is off by what they are off by
        bound = step * 0.5 + 2 ** -11 * (lo.abs() + 15 * step) + g.abs().amax(-1, keepdim=True) * 2 ** -17 + 2 ** -24 * 16
        assert bool(((k[:, first:].unflatten(-1, (4, 32)) - g).abs() <= bound).all())


@pytest.mark.parametrize("q_heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("first,rows", [(0, 1), (15, 1), (513, 1), (0, 16), (7, 30), (60, 9), (0, 200), (129, 300)])
def test_append(mine, capi, q_heads, kv_heads, first, rows):
    cache = _kv4.Cache(mine, capi, 20, layers=2, kv_heads=kv_heads, q_heads=q_heads, stride=12, rows=rows)
    pages = torch.randperm(20)[:-(-(first + rows) // 64)].int().cuda()
    cache.table[3, :len(pages)] = pages
    b = cache.batch([3], [rows], [first])
    qkv = queries(rows, q_heads + 2 * kv_heads, seed=first)
    g = torch.Generator().manual_seed(9)
    q_norm, k_norm = ((1 + 0.3 * torch.randn(128, generator=g)).bfloat16().cuda() for _ in range(2))
    for layer, (qn, kn), eps, base in ((1, (q_norm, k_norm), 1e-6, 1e6), (0, (None, None), 1e-6, 1e4), (1, (None, k_norm), 1e-2, 1e6)):
        q = torch.full((rows, q_heads * 128), 7.0, dtype=torch.bfloat16, device="cuda")
        before = cache.pages.clone()
        cache.append(b, qkv, q, layer=layer, q_norm=qn, k_norm=kn, eps=eps, base=base)
        check_append(cache, b, [(3, first, 0, rows)], qkv, q, qn, kn, eps, base, layer)
        assert torch.equal(cache.pages[:, 1 - layer], before[:, 1 - layer])  # the other layer
        k, v, mass, there = cache.values(3, first + rows, layer)
        unwritten = [p for p in range(20) if p not in pages.tolist()]
        assert torch.equal(cache.pages[unwritten], before[unwritten])


@pytest.mark.parametrize("rows", [296, 592, 593, 1185, 1777, 2371])
def test_append_and_read_many_rows(mine, capi, rows):
    """From one row to four of a CTA, the last of them partly padding."""
    cache = _kv4.Cache(mine, capi, 40, kv_heads=1, q_heads=3, stride=40, rows=rows + 3)
    counts = [rows - 100, 100]
    b = cache.batch([1, 3], counts, rows=rows + 3)
    cache.reserve(b)
    qkv = queries(rows + 3, 5)
    q = torch.full((rows + 3, 3 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    cache.append(b, qkv, q)
    check_append(cache, b, [(1, 0, 0, counts[0]), (3, 0, counts[0], 100)], qkv, q, None, None, 1e-6, 1e6)
    assert bool((q[rows:] == 7).all())
    got = [torch.full((rows + 3, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.call("read", C.byref(b.c), 0, got[0].data_ptr(), got[1].data_ptr(), None)
    torch.cuda.synchronize()
    for seq, r0, n in ((1, 0, counts[0]), (3, counts[0], 100)):
        for out, held in zip(got, cache.values(seq, n)[:2]):
            assert torch.equal(out[r0:r0 + n].cpu(), held[0].bfloat16())
    assert all(bool((out[rows:] == 7).all()) for out in got)


def test_append_far_positions(mine, capi):
    """Positions near the end of the longest sequence of this repository: the angle of the fastest pair is 32767 radians."""
    cache = _kv4.Cache(mine, capi, 20, kv_heads=2, q_heads=8, stride=512)
    cache.table[0, 500:512] = torch.arange(12).int().cuda()
    b = cache.batch([0], [64], [32704])
    qkv = queries(64, 12)
    q = torch.zeros(64, 8 * 128, dtype=torch.bfloat16, device="cuda")
    cache.append(b, qkv, q)
    torch.cuda.synchronize()
    want = rotated(qkv.cpu().view(64, 12, 128)[:, :8], None, torch.arange(32704, 32768), 0, 1e6)
    pair = want.unflatten(-1, (64, 2)).norm(dim=-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
    assert bool(((q.double().cpu().view_as(want) - want).abs() <= want.abs() * 2 ** -8 + pair * 2 ** -19).all())


def test_append_ragged_batch(mine, capi):
    """Entries without rows, without pages, refused ones and padding: their neighbours' bytes stay."""
    cache = _kv4.Cache(mine, capi, 30, kv_heads=2, q_heads=8, max_seqs=6, stride=4, rows=300, fill=0x11)
    held = {0: 130, 1: 64, 2: 5, 3: 40, 4: 256}
    for s, t in held.items():
        _kv4.fill(cache, s, t, seed=s)
    cache.table[3, 0] = -1
    before = cache.pages.clone()
    seqs, counts, pos0 = [1, 0, 2, 3, 4, 5, 77], [64, 7, 0, 10, 3, 2, 2], [0, 110, 5, 30, 255, -1, 0]
    b = cache.batch(seqs, counts, pos0, rows=95)  # sequence 4: two of its rows lie behind the table
    qkv = queries(95, 12)
    q = torch.full((95, 8 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    cache.append(b, qkv, q, base=1e6)
    check_append(cache, b, [(1, 0, 0, 64), (0, 110, 64, 7), (4, 255, 81, 1)], qkv, q, None, None, 0, 1e6)
    want = rotated(qkv.cpu().view(95, 12, 128)[71:84, :8], None, torch.cat([torch.arange(30, 40), torch.arange(255, 258)]), 0, 1e6).reshape(13, -1)
    assert bool(((q[71:84].double().cpu() - want).abs() <= want.abs() * 2 ** -8 + 1e-4).all())  # (|pair| < 12: 12 * 2^-19 = 2.3e-5)
    assert bool((q[84:88] == 0).all()) and bool((q[88:] == 7).all())
    now, then = cache.pages.clone(), before.clone()
    for s, a, e in ((1, 0, 64), (0, 110, 117), (4, 255, 256)):  # blank what was to be written; the rest is as it was
        for p in range(a, e):
            page, blk, i = int(cache.table[s, p // 64]), p % 64 // 16, p % 16
            for which in (0, 1):
                byte, _, at_s, at_m = (t[i] for t in _kv4.places(which))
                for at in (byte, at_s, at_s + 1, at_m, at_m + 1):
                    now[page, :, :, blk, at.cuda()] = 0
                    then[page, :, :, blk, at.cuda()] = 0
    assert torch.equal(now, then)


def test_append_of_extreme_values(mine, capi):
    """Zeros, equal channels, values beyond f16, infinities and NaN in one head each."""
    cache = _kv4.Cache(mine, capi, 4, kv_heads=6, q_heads=6, stride=2)
    cache.table[0, 0] = 1
    x = torch.zeros(1, 18, 128)
    x[0, 13] = 2.5
    x[0, 14] = torch.linspace(-1e6, 1e6, 128)
    x[0, 15] = torch.linspace(-1, 1, 128)
    x[0, 15, 3], x[0, 15, 40], x[0, 15, 41] = float("nan"), float("inf"), -float("inf")
    x[0, 16] = float("nan")
    x[0, 17] = torch.linspace(-1, 1, 128) * 1e-6
    qkv = x.bfloat16().view(1, -1).cuda()
    b = cache.batch([0], [1], [9])
    q = torch.zeros(1, 6 * 128, dtype=torch.bfloat16, device="cuda")
    cache.append(b, qkv, q)
    torch.cuda.synchronize()
    _, v, _, _ = cache.values(0, 10)
    v, x = v[:, 9], qkv.cpu().float().view(18, 128)[12:]
    assert bool((v[0] == 0).all()) and bool((v[1] == 2.5).all())
    fine = [0, 1, 2, 5]
    c, s, m = _kv4.quantise(x[fine])
    assert torch.equal(v[fine], c.double() * s.double() + m.double())
    want = x[3].double().clamp(-65504, 65504)
    assert bool(v.isfinite().all())
    keep = torch.ones(128, dtype=torch.bool)
    keep[3] = False
    assert bool((v[3, :32][keep[:32]] - want[:32][keep[:32]]).abs().max() < 0.02)     # the group with the NaN: its others are as ever
    assert float(v[3, 3]) == float(v[3, 0])                                           # ... and it stands for the smallest
    assert abs(float(v[3, 40]) - 65504) < 70 and abs(float(v[3, 41]) + 65504) < 70
    assert bool((v[4] == 0).all())


@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (3, 3), (16, 1)])
def test_read(mine, capi, q_heads, kv_heads):
    cache = _kv4.Cache(mine, capi, 20, layers=2, kv_heads=kv_heads, q_heads=q_heads, max_seqs=5, stride=4, rows=400)
    _kv4.fill(cache, 0, 250, seed=1, layer=1)
    _kv4.fill(cache, 3, 70, seed=2, layer=1)
    cache.table[0, 1] = -1
    b = cache.batch([3, 0, 0, 4, 9], [70, 250, 0, 3, 2], [0, 0, 5, -1, 0], rows=330)
    k = torch.full((330, kv_heads * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    cache.read(b, k, v, layer=1)
    torch.cuda.synchronize()
    for seq, r0, n in ((3, 0, 70), (0, 70, 250)):
        want_k, want_v, _, there = cache.values(seq, n, layer=1)
        for got, want in ((k, want_k), (v, want_v)):
            want = torch.where(there[None, :, None], want, 0.0)
            assert torch.equal(got[r0:r0 + n].cpu(), want.float().transpose(0, 1).reshape(n, -1).bfloat16())
    for got in (k, v):
        assert bool((got[320:325] == 0).all()) and bool((got[325:] == 7).all())


# ---- page operators -------------------------------------------------------------------------------------------------------

class Book:
    """What the page operators do, step by step."""

    def __init__(self, cache):
        self.n, self.stride = cache.n_pages, cache.stride
        self.table, self.lens, self.refs = (t.cpu().tolist() for t in (cache.table, cache.lens, cache.refs))
        self.mark = cache.pages[:, 0, 0, 0, 0].cpu().tolist()

    def free(self):
        return [p for p in range(self.n) if self.refs[p] == 0]

    def release(self, seqs):
        for s in seqs:
            for page in self.table[s]:
                if 0 <= page < self.n:
                    self.refs[page] -= 1
            self.table[s], self.lens[s] = [-1] * self.stride, 0

    def reserve(self, seqs, counts):
        free, upto, pos0, refused, taken = self.free(), 0, [], 0, 0
        for s, n in zip(seqs, counts):
            held = self.lens[s]
            first, last = -(-held // 64), -(-(held + n) // 64)
            need = last - first
            upto += need
            if last > self.stride or (need and upto > len(free)):
                pos0.append(-1)
                refused += 1
                continue
            for i in range(need):
                page = free[upto - need + i]
                self.table[s][first + i], self.refs[page] = page, 1
            taken += need
            pos0.append(held)
            self.lens[s] += n
        return pos0, [len(free) - taken, refused]

    def fork(self, parents, children, tokens):
        self.release(children)
        free, refused = self.free(), 0
        for p, c, t in zip(parents, children, tokens):
            t = self.lens[p] if t < 0 else min(t, self.lens[p])
            full, rest = divmod(t, 64)
            tail = self.table[p][full] if rest else -1
            if 0 <= tail < self.n:
                if not free:
                    refused += 1
                    continue
                page = free.pop(0)
                self.refs[page], self.table[c][full], self.mark[page] = 1, page, self.mark[tail]
            self.lens[c] = t
            for j in range(full):
                page = self.table[p][j]
                if 0 <= page < self.n:
                    self.table[c][j] = page
                    self.refs[page] += 1
        return [len(free), refused]

    def compact(self):
        used = sum(r != 0 for r in self.refs)
        source = [p for p in range(used, self.n) if self.refs[p]]
        to = [p for p in range(used) if not self.refs[p]]
        new = dict(zip(source, to))
        for a, b in new.items():
            self.mark[b], self.refs[b], self.refs[a] = self.mark[a], self.refs[a], 0
        self.table = [[new.get(p, p) for p in row] for row in self.table]
        return [self.n - used, len(new)]

    def check(self, cache, info=None):
        torch.cuda.synchronize()
        assert cache.table.cpu().tolist() == self.table
        assert cache.lens.cpu().tolist() == self.lens
        assert cache.refs.cpu().tolist() == self.refs
        flat = cache.pages.flatten(1)
        assert flat[:, 0].cpu().tolist() == self.mark
        assert bool((flat == flat[:, :1]).all())  # every byte of a page moved with it
        if info is not None:
            assert cache.info.cpu().tolist() == info


def marked(mine, capi, n_pages, **kw):
    cache = _kv4.Cache(mine, capi, n_pages, **kw)
    cache.pages.copy_((torch.arange(n_pages) % 251).to(torch.uint8).cuda()[:, None, None, None, None].expand_as(cache.pages))
    return cache


@pytest.mark.parametrize("n_pages,seqs,seed", [(7, 3, 0), (40, 6, 1), (300, 40, 2), (300, 256, 3), (5000, 60, 4), (9001, 30, 5)])
def test_pages_random_walk(mine, capi, n_pages, seqs, seed):
    """Reserve, fork, release and compact in a random order, with pools that run out, against the step-by-step book."""
    import random
    rng = random.Random(seed)
    cache = marked(mine, capi, n_pages, layers=2, kv_heads=1, q_heads=1, max_seqs=seqs, stride=24)
    book = Book(cache)
    for _ in range(25):
        what = rng.choice(("reserve", "reserve", "fork", "release", "compact"))
        some = rng.sample(range(seqs), rng.randint(1, min(seqs, 200)))
        if what == "reserve":
            counts = [rng.choice((0, 1, 1, 63, 64, 65, rng.randint(0, 700))) for _ in some]
            b = cache.batch(some, counts)
            cache.reserve(b)
            pos0, info = book.reserve(some, counts)
            assert b.pos0.cpu().tolist() == pos0
        elif what == "fork":
            cut = max(1, len(some) // 2)
            children = some[:cut]
            parents = [rng.choice(some[cut:]) for _ in children] if some[cut:] else None
            if parents is None:
                continue
            tokens = [rng.choice((-1, 0, 1, 64, 128, rng.randint(0, 1500))) for _ in children]
            cache.fork(parents, children, tokens)
            info = book.fork(parents, children, tokens)
        elif what == "release":
            some = some[: max(1, len(some) // 3)]
            cache.release(some)
            book.release(some)
            info = None
        else:
            cache.compact()
            info = book.compact()
        book.check(cache, info)


def test_pool_runs_out_in_order(mine, capi):
    cache = marked(mine, capi, 6, layers=1, kv_heads=1, q_heads=1, max_seqs=6, stride=4)
    book = Book(cache)
    for seqs, counts in (([0, 1, 2, 3], [100, 64, 200, 10]), ([4, 5, 1], [0, 1, 1]), ([0, 3, 5], [300, 1, 64]), ([2], [1])):
        b = cache.batch(seqs, counts)
        cache.reserve(b)
        pos0, info = book.reserve(seqs, counts)
        book.check(cache, info)
        assert b.pos0.cpu().tolist() == pos0
    cache.fork([0, 1], [4, 5], [90, -1])  # 1 holds a full page: shared; 0's second page has to be copied
    book.check(cache, book.fork([0, 1], [4, 5], [90, -1]))


def test_a_sequence_that_stands_in_a_batch_twice(mine, capi):
    """Reserve serves the first entry and refuses the others; no page is lost."""
    n = 1024
    cache = _kv4.Cache(mine, capi, 900, kv_heads=1, q_heads=1, max_seqs=5000, stride=4, rows=3 * n)
    seqs = [i * 37 % 400 * 7 for i in range(n)]
    b = cache.batch(seqs, [1 + i % 3 for i in range(n)])
    cache.reserve(b)
    torch.cuda.synchronize()
    seen, want = set(), []
    for s in seqs:
        want.append(-1 if s in seen else 0)
        seen.add(s)
    assert b.pos0.cpu().tolist() == want
    assert cache.info.cpu().tolist() == [900 - len(seen), n - len(seen)]
    assert sorted(cache.table[cache.table >= 0].cpu().tolist()) == list(range(len(seen)))
    cache.reserve(cache.batch([3, 4, 3, -1, 5000, 4], [1, 0, 70, 1, 1, 0]))
    torch.cuda.synchronize()
    assert cache.info.cpu().tolist()[1] == 4


def test_empty_and_unusual_calls(mine, capi):
    cache = marked(mine, capi, 5, layers=1, kv_heads=1, q_heads=1, max_seqs=3, stride=2)
    book = Book(cache)
    cache.call("reserve", C.byref(cache.batch([], []).c), cache.info.data_ptr(), None)
    book.check(cache, [5, 0])
    cache.info.fill_(-7)
    cache.call("fork", None, None, None, 0, cache.info.data_ptr(), None)
    book.check(cache, [5, 0])
    cache.compact()
    book.check(cache, [5, 0])
    cache.release([0, 1, 2])
    book.check(cache)
    cache.fork([0], [1], [-1])  # nothing to share
    book.check(cache, book.fork([0], [1], [-1]))
    # sequences that are not there are refused, and the others are served
    b = cache.batch([7, 1, -2], [10, 20, 30])
    cache.reserve(b)
    torch.cuda.synchronize()
    assert b.pos0.cpu().tolist() == [-1, 0, -1] and cache.info.cpu().tolist() == [4, 2] and cache.lens.cpu().tolist() == [0, 20, 0]
    # a pool in which all is used, and one in which the table alone is short
    b = cache.batch([0, 2, 1], [128, 128, 200])
    cache.reserve(b)
    torch.cuda.synchronize()
    assert b.pos0.cpu().tolist() == [0, 0, -1] and cache.info.cpu().tolist() == [0, 1]
    cache.compact()
    assert cache.info.cpu().tolist() == [0, 0]


def test_unaligned_reference_counts(mine, capi):
    cache = marked(mine, capi, 4099, layers=1, kv_heads=1, q_heads=1, max_seqs=3, stride=64)
    shifted = torch.zeros(4103, dtype=torch.int32, device="cuda")
    cache.refs = shifted[3:4102]
    cache.c.refs = cache.refs.data_ptr()
    cache.refs[:4097] = 1
    book = Book(cache)
    b = cache.batch([0, 1], [64, 65])
    cache.reserve(b)
    pos0, info = book.reserve([0, 1], [64, 65])
    book.check(cache, info)
    cache.compact()
    book.check(cache, book.compact())
    assert int(shifted[:3].abs().sum()) == 0 and int(shifted[4102:].abs().sum()) == 0


# ---- together ---------------------------------------------------------------------------------------------------------------

def test_a_server_run(mine, capi):
    """Prompts, forks of a voice, lockstep ticks, ends and compaction, on a stream of their own.  Attention is compared with the pages'
    own contents; the pages of forked and compacted sequences with those of a run that shares and moves nothing."""
    hq, hk, layers = 32, 8, 2
    side = torch.cuda.Stream()
    st = C.c_void_p(side.cuda_stream)
    shared = _kv4.Cache(mine, capi, 40, layers=layers, kv_heads=hk, q_heads=hq, max_seqs=6, stride=8, rows=400)
    apart = _kv4.Cache(mine, capi, 60, layers=layers, kv_heads=hk, q_heads=hq, max_seqs=6, stride=8, rows=400)
    g = torch.Generator().manual_seed(4)
    norm = (1 + 0.2 * torch.randn(128, generator=g)).bfloat16().cuda()
    torch.cuda.synchronize()
    rows_of = {}

    def step(seqs, counts, seed, caches):
        x = {layer: queries(sum(counts), hq + 2 * hk, seed=seed + layer) for layer in range(layers)}
        torch.cuda.synchronize()
        outs = []
        for cache in caches:
            b = cache.batch(seqs, counts)
            torch.cuda.synchronize()
            cache.reserve(b, st)
            for layer in range(layers):
                q = torch.zeros(sum(counts), hq * 128, dtype=torch.bfloat16, device="cuda")
                out = torch.zeros_like(q)
                torch.cuda.synchronize()
                cache.append(b, x[layer], q, layer=layer, q_norm=norm, k_norm=norm, stream=st)
                cache.attention(b, q, out, layer=layer, stream=st)
                side.synchronize()
                entries, at = [], 0
                for s, n, p in zip(seqs, counts, b.pos0.cpu().tolist()):
                    assert p >= 0
                    if n:
                        entries.append((s, p, at, n))
                    at += n
                check_attention(cache, b, entries, q, out, layer)
                outs.append(out)
        if len(caches) == 2:
            half = len(outs) // 2
            assert all(torch.equal(a, b) for a, b in zip(outs[:half], outs[half:]))

    step([0], [203], 1, (shared, apart))                     # a voice
    shared.fork([0, 0, 0], [1, 2, 3], [-1, 200, 192], st)
    side.synchronize()
    for child, t in ((1, 203), (2, 200), (3, 192)):          # the same sequences without sharing: the bytes copied
        for c in range(-(-t // 64)):
            page = 20 + child * 8 + c
            apart.pages[page] = apart.pages[int(apart.table[0, c])]
            apart.table[child, c], apart.refs[page] = page, 1
        apart.lens[child] = t
    torch.cuda.synchronize()
    assert int(shared.refs[int(shared.table[0, 0])]) == 4 and int(shared.info[1]) == 0
    step([1, 2, 3], [40, 1, 13], 10, (shared, apart))
    for tick in range(4):
        step([3, 1, 2], [1, 1, 1], 20 + 5 * tick, (shared, apart))
    shared.release([0, 2], st)                               # the voice goes; its pages stay with its children
    shared.compact(st)
    side.synchronize()
    assert int((shared.refs > 0).sum()) == int(shared.table.max()) + 1
    step([1, 3], [30, 70], 50, (shared, apart))
    step([4, 1, 3], [5, 1, 1], 60, (shared,))
    rows_of.clear()
    shared.call("status", None)


def test_a_captured_tick_replays_as_the_sequences_grow(mine, capi):
    hq, hk = 8, 2
    cache = _kv4.Cache(mine, capi, 40, layers=1, kv_heads=hk, q_heads=hq, max_seqs=4, stride=8)
    again = _kv4.Cache(mine, capi, 40, layers=1, kv_heads=hk, q_heads=hq, max_seqs=4, stride=8)
    qkv = [queries(3, hq + 2 * hk, seed=i) for i in range(100)]
    static = torch.zeros_like(qkv[0])
    q, out = (torch.zeros(3, hq * 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for c in (cache, again):
        for s, t in ((0, 62), (1, 1), (3, 130)):
            _kv4.fill(c, s, t, seed=s, order=torch.arange(8 * s, 8 * s + -(-t // 64)))
            c.refs[8 * s: 8 * s + -(-t // 64)] = 1
    b = cache.batch([3, 0, 1], [1, 1, 1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        cache.reserve(b, st)
        cache.append(b, static, q, stream=st)
        cache.attention(b, q, out, stream=st)
    q2, out2 = torch.zeros_like(q), torch.zeros_like(out)
    for i in range(100):
        static.copy_(qkv[i])
        graph.replay()
        b2 = again.batch([3, 0, 1], [1, 1, 1])
        again.reserve(b2)
        again.append(b2, qkv[i], q2)
        again.attention(b2, q2, out2)
        torch.cuda.synchronize()
        assert torch.equal(b.pos0, b2.pos0) and torch.equal(q, q2) and torch.equal(out, out2)
    assert torch.equal(cache.table, again.table) and cache.lens.cpu().tolist() == [162, 101, 0, 230]


def test_captured_mixed_batches_with_one_workspace(mine, capi):
    """Two graphs on one workspace, of slices and of tokens; what the batches hold changes between replays."""
    hq, hk, n, rows = 8, 2, 6, 260
    cache = _kv4.Cache(mine, capi, 80, kv_heads=hk, q_heads=hq, max_seqs=n, stride=16, rows=rows)
    other = _kv4.Cache(mine, capi, 80, kv_heads=hk, q_heads=hq, max_seqs=n, stride=16, rows=rows)
    lens = [700, 64, 300, 129, 500, 260]
    for i, x in enumerate(lens):
        _kv4.fill(cache, i, x, seed=i)
    other.pages.copy_(cache.pages)
    other.table.copy_(cache.table)
    q = queries(rows, hq)
    slices, tokens = cache.batch(range(n), [0] * n, [0] * n, rows=rows, max_rows=rows), cache.batch(range(n), [1] * n, [0] * n)
    out, out1 = torch.zeros_like(q), torch.zeros_like(q[:n])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for b, to in ((slices, out), (tokens, out1)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            cache.attention(b, q, to, stream=C.c_void_p(torch.cuda.current_stream().cuda_stream))
        graphs.append(g)
    for counts in ([1, 64, 1, 1, 100, 1], [200, 1, 33, 2, 1, 0], [1] * 6, [0, 0, 0, 0, 0, 260], [5, 40, 60, 7, 50, 40]):
        row0 = [0]
        for c in counts:
            row0.append(row0[-1] + c)
        slices.row0.copy_(torch.tensor(row0, dtype=torch.int32))
        slices.pos0.copy_(torch.tensor([x - c for x, c in zip(lens, counts)], dtype=torch.int32))
        tokens.pos0.copy_(torch.tensor([x - 1 - counts[0] % 7 for x in lens], dtype=torch.int32))
        for g, b, to in ((graphs[0], slices, out), (graphs[1], tokens, out1)) * 2:
            to.fill_(7.0)
            g.replay()
            want = torch.full_like(to, 7.0)
            other.attention(b, q, want)
            torch.cuda.synchronize()
            assert torch.equal(to, want)
        check_attention(cache, slices, [(i, lens[i] - c, row0[i], c) for i, c in enumerate(counts) if c], q, out)
    cache.call("status", None)


def test_a_wait_that_gives_up_is_told_and_leaves_nothing_behind(testlib, capi):
    """The deadline of the slices' bounded waits lowered until one runs out: the call ends, the status says so once, and with the deadline
    restored the next call is right."""
    capi.bind(testlib, capi.EXT_PROTOTYPES)
    testlib.kv4_slices_set_wait_ns.argtypes = [C.c_ulonglong]
    cache = _kv4.Cache(testlib, capi, 60, kv_heads=2, q_heads=8, max_seqs=2, stride=40, rows=400)
    _kv4.fill(cache, 0, 2400, seed=1)
    b = cache.batch([0], [400], [2000])
    q = queries(400, 8)
    out = torch.full_like(q, 7.0)
    try:
        assert testlib.kv4_slices_set_wait_ns(100) == 0
        for _ in range(50):
            cache.attention(b, q, out)
            said = cache.status("status", None)
            assert said in (0, -8)
            if said:
                break
        assert said == -8
    finally:
        assert testlib.kv4_slices_set_wait_ns(2_000_000_000) == 0
    cache.call("status", None)
    cache.attention(b, q, out)
    check_attention(cache, b, [(0, 2000, 0, 400)], q, out)
    cache.call("status", None)


def test_caches_share_a_workspace(mine, capi):
    """Of other sizes, in turn."""
    caches = [_kv4.Cache(mine, capi, n, kv_heads=h, q_heads=4 * h, stride=24, rows=300) for n, h in ((30, 2), (500, 8), (25, 1))]
    for c in caches:
        _kv4.fill(c, 0, 1400, seed=c.n_pages)
        c.work = caches[1].work
        c.c.work, c.c.work_bytes = c.work.data_ptr(), c.work.numel()
    for turn in range(3):
        for rows in (1, 20, 300):
            for c in caches:
                b = c.batch([0], [rows], [1400 - rows])
                q = queries(rows, c.q_heads, seed=turn)
                out = torch.full_like(q, 7.0)
                c.attention(b, q, out)
                check_attention(c, b, [(0, 1400 - rows, 0, rows)], q, out)
                if turn == 1:
                    c.compact()


def test_two_streams_with_a_workspace_each(mine, capi):
    """Two caches worked on at once."""
    pairs = []
    for i in range(2):
        cache = _kv4.Cache(mine, capi, 60, kv_heads=2, q_heads=8, max_seqs=2, stride=40, rows=200)
        _kv4.fill(cache, 0, 2000, seed=i)
        pairs.append((cache, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for turn in range(10):
        for i, (cache, stream) in enumerate(pairs):
            rows = (1, 200, 9)[(turn + i) % 3]
            with torch.cuda.stream(stream):
                b = cache.batch([0], [rows], [2000 - rows])
                q = queries(rows, 8, seed=turn)
                out = torch.full_like(q, 7.0)
                cache.attention(b, q, out, stream=C.c_void_p(stream.cuda_stream))
                outs.append((cache, b, rows, q, out))
    torch.cuda.synchronize()
    for cache, b, rows, q, out in outs:
        check_attention(cache, b, [(0, 2000 - rows, 0, rows)], q, out)
