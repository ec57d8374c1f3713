"""Paged 4-bit cache on the GPU, close: attention against what independent roundings leave (tests/_kv4.py: attention_close), and the corners of its rules."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _kv4  # noqa: E402

pytestmark = pytest.mark.gpu


def gauss(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def close(cache, entries, q, out):
    """entries: (sequence, first position, first row, rows)."""
    torch.cuda.synchronize()
    for seq, first, r0, n in entries:
        want, bound = _kv4.attention_close(cache, seq, first, q[r0:r0 + n])
        off = (out[r0:r0 + n].double() - want).abs()
        assert bool((off <= bound).all()), (seq, first, n, float((off / bound).max()), float((off.norm() / want.norm())))


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (3, 3), (16, 1)])
@pytest.mark.parametrize("first,rows", [(0, 1), (0, 130), (5, 1), (70, 3), (70, 100)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_query_that_is_not_finite_makes_its_head_nan(mine, capi, q_heads, kv_heads, first, rows, bad):
    """Whatever the signs of the keys that it meets: of one sign, of the other, of zero; other heads and rows are as ever."""
    length = first + rows
    for sign in (1.0, -1.0, 0.0):
        cache = _kv4.Cache(mine, capi, 8, kv_heads=kv_heads, q_heads=q_heads, stride=4, rows=rows)
        k = gauss(kv_heads, length, 128, seed=1)
        k[..., 9] = sign * k[..., 9].abs()
        if sign == 0.0:
            k[..., :32] = 0.0
        _kv4.store(cache, 1, k, gauss(kv_heads, length, 128, seed=2))
        b = cache.batch([1], [rows], [first])
        q = (gauss(rows, q_heads * 128, seed=3) * 1.5).bfloat16()
        clean = q.clone()
        spoilt = sorted({(0, 0), (0, q_heads - 1), (rows - 1, 1), (rows // 2, q_heads // 2)})
        for r, h in spoilt:
            q[r, h * 128 + 9] = bad
        out = torch.full_like(q, 7.0)
        cache.attention(b, q, out)
        want, bound = _kv4.attention_close(cache, 1, first, clean)
        off = (out.double() - want).abs().view(rows, q_heads, 128)
        fine = torch.ones(rows, q_heads, dtype=torch.bool, device="cuda")
        for r, h in spoilt:
            fine[r, h] = False
            assert bool(out[r, h * 128:(h + 1) * 128].isnan().all()), (sign, r, h, out[r, h * 128:h * 128 + 4])
        assert bool((off <= bound.view_as(off))[fine].all())
        # ... of a row that sees nothing it leaves zeros
        cache.table[1, :] = -1
        cache.attention(b, q, out)
        torch.cuda.synchronize()
        assert bool((out == 0).all())


@pytest.mark.parametrize("scale", [1e-5, 1e-4, 1e-3, 1e-2, 0.1, 10.0, 1000.0])
@pytest.mark.parametrize("length,rows", [(40, 1), (3000, 1), (3000, 3), (16000, 1)])
def test_values_of_any_size_for_tokens(mine, capi, scale, length, rows):
    """The weights' products with s stay where f16 has all its bits."""
    cache = _kv4.Cache(mine, capi, 260, kv_heads=2, q_heads=8, stride=256)
    _kv4.store(cache, 0, gauss(2, length, 128, seed=1), gauss(2, length, 128, seed=2) * scale)
    b = cache.batch([0], [rows], [length - rows])
    q = (gauss(rows, 8 * 128, seed=3) * 1.5).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    close(cache, [(0, length - rows, 0, rows)], q, out)


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (16, 1)])
@pytest.mark.parametrize("sizes", [(1e-3, 1.0, 20.0, 1.0), (1e-3, 100.0), (1.0, 300.0, 1e4), (1e4, 1e-3), (1e-4, 1e-3, 1e-2, 0.1, 1.0, 10.0, 100.0, 1000.0)])
def test_values_whose_size_changes_along_a_sequence(mine, capi, sizes, rows, q_heads, kv_heads):
    """What has been summed is carried over when s outgrows what the weights were scaled for; the groups of a head differ by a factor of 16 besides."""
    length = 2300
    cache = _kv4.Cache(mine, capi, 40, kv_heads=kv_heads, q_heads=q_heads, stride=40)
    grow = torch.tensor(sizes, device="cuda").repeat_interleave(-(-length // len(sizes)))[:length, None]
    v = gauss(kv_heads, length, 128, seed=2) * grow * torch.tensor([1.0, 4.0, 0.25, 2.0], device="cuda").repeat_interleave(32)
    _kv4.store(cache, 0, gauss(kv_heads, length, 128, seed=1), v)
    b = cache.batch([0], [rows], [length - rows])
    q = (gauss(rows, q_heads * 128, seed=3) * 1.5).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    close(cache, [(0, length - rows, 0, rows)], q, out)


@pytest.mark.parametrize("scale", [3e-7, 1e-6, 1e-5, 1e-4, 1e-3, 1.0, 1000.0])
@pytest.mark.parametrize("what", ["keys", "values", "both"])
@pytest.mark.parametrize("length,rows", [(130, 130), (2000, 70)])
def test_keys_and_values_of_any_size_for_slices(mine, capi, scale, what, length, rows):
    """s c + m has all the bits that the cache holds, down to f16's smallest numbers."""
    cache = _kv4.Cache(mine, capi, 40, kv_heads=2, q_heads=8, stride=40, rows=rows)
    ks, vs = (scale if what in (name, "both") else 1.0 for name in ("keys", "values"))
    _kv4.store(cache, 0, gauss(2, length, 128, seed=1) * ks, gauss(2, length, 128, seed=2) * vs)
    b = cache.batch([0], [rows], [length - rows])
    q = (gauss(rows, 8 * 128, seed=3) * 1.5 / ks).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    close(cache, [(0, length - rows, 0, rows)], q, out)


@pytest.mark.parametrize("rows", [1, 130])
def test_groups_that_reach_beyond_f16(mine, capi, rows):
    """The largest value of a group of the widest range is 65536, which f16 has not: it counts as 65504 at the least, the values beside it as they are."""
    length = 200
    cache = _kv4.Cache(mine, capi, 8, kv_heads=2, q_heads=8, stride=4, rows=rows)
    v = gauss(2, length, 128, seed=2)
    v[:, ::3] *= 1e6
    v[:, 1::3, 32:64] *= 65504 / v[:, 1::3, 32:64].abs().amax(-1, keepdim=True)
    top = 65504 - torch.rand(2, 66, 1, generator=torch.Generator("cuda").manual_seed(4), device="cuda").mul(11).exp()  # ranges of 1 to 60000 below the largest
    v[:, 2:200:3, 96:] = top + (65504 - top) * torch.rand(2, 66, 32, generator=torch.Generator("cuda").manual_seed(5), device="cuda")
    v[:, 2:200:3, 100] = 65504
    v[:, 2:200:3, 101] = (top[..., 0] / 16).round() * 16
    k = gauss(2, length, 128, seed=1)
    k[:, ::5, 64:96] *= 1e6
    _kv4.store(cache, 0, k, v)
    b = cache.batch([0], [rows], [length - rows])
    q = gauss(rows, 8 * 128, seed=3).view(rows, 8, 4, 32)
    q[:, :, 2] *= 1e-5
    q = q.reshape(rows, -1).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    close(cache, [(0, length - rows, 0, rows)], q, out)


# ---- parts --------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens", [[32000], [32000, 9000], [700, 640, 650, 700, 690, 610, 500, 700, 100], [6000] + [90, 100, 1, 64] * 4, [500, 513, 480, 511] * 7,
                                  [2100, 300, 64, 1, 1700, 900, 17, 3000] * 3, [33, 70, 1, 16, 128, 64, 99, 130] * 20])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (16, 1), (32, 8)])
def test_no_part_of_a_sequence_is_lost_for_tokens(mine, capi, lens, q_heads, kv_heads):
    """Weights that hardly differ, so that every part, piece and page counts alike: one of 500 that is left out is off by several bounds."""
    n = len(lens)
    cache = _kv4.Cache(mine, capi, sum((x + 63) // 64 for x in lens) + 1, kv_heads=kv_heads, q_heads=q_heads, max_seqs=n, stride=512, rows=n)
    for i, x in enumerate(lens):
        _kv4.store(cache, i, gauss(kv_heads, x, 128, seed=2 * i), gauss(kv_heads, x, 128, seed=2 * i + 1))
    b = cache.batch(range(n), [1] * n, [x - 1 for x in lens])
    q = (gauss(n, q_heads * 128, seed=9) * 0.3).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    close(cache, [(i, x - 1, i, 1) for i, x in enumerate(lens)], q, out)


@pytest.mark.parametrize("lens,counts", [([7000], [700]), ([7000], [65]), ([1000], [1000]), ([7000] + [50] * 12, [32] + [40] * 12), ([300, 250, 333], [70, 64, 65]),
                                         ([4000, 3900], [300, 290]), ([1500] * 16, [1] * 15 + [512]), ([64, 500, 129, 700] * 4, [64, 100, 128, 33] * 4)])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (16, 1), (32, 8)])
def test_no_part_of_a_sequence_is_lost_for_slices(mine, capi, lens, counts, q_heads, kv_heads):
    n, total = len(lens), sum(counts)
    cache = _kv4.Cache(mine, capi, sum((x + 63) // 64 for x in lens) + 1, kv_heads=kv_heads, q_heads=q_heads, max_seqs=n, stride=128, rows=total)
    for i, x in enumerate(lens):
        _kv4.store(cache, i, gauss(kv_heads, x, 128, seed=2 * i), gauss(kv_heads, x, 128, seed=2 * i + 1))
    b = cache.batch(range(n), counts, [x - c for x, c in zip(lens, counts)])
    q = (gauss(total, q_heads * 128, seed=9) * 0.3).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    entries = []
    for i, (x, c) in enumerate(zip(lens, counts)):
        for r in range(0, c, 128):  # (a few rows at a time: the weights are in 64 bits)
            m = min(128, c - r)
            entries.append((i, x - c + r, sum(counts[:i]) + r, m))
    close(cache, entries, q, out)


# ---- pages --------------------------------------------------------------------------------------------------------------------

def test_reserve_of_more_pages_than_two_to_the_twentieth(mine, capi):
    """All of them are given, or none."""
    n_pages, need = 2 ** 20 + 100, 2 ** 20 + 5
    cache = _kv4.Cache(mine, capi, 1, kv_heads=1, q_heads=1, max_seqs=3, stride=2 ** 20 + 200, rows=1)
    pool = torch.empty(n_pages * _kv4.BLOCK * 4, dtype=torch.uint8, device="cuda")
    cache.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    cache.c.pages, cache.c.refs, cache.c.n_pages = pool.data_ptr(), cache.refs.data_ptr(), n_pages
    for seqs, counts, pos0, info in (([0, 1, 2], [64 * need, 64 * 95, 1], [0, 0, -1], [0, 1]),       # all pages there are, and one more
                                     ([0], [64 * (n_pages + 1)], [-1], [n_pages, 1]),                 # more than the pool has
                                     ([0, 1], [64 * (n_pages - 1), 65], [0, -1], [1, 1]),
                                     ([0, 1], [64 * n_pages - 63, 0], [0, 0], [0, 0])):
        cache.refs.zero_()
        cache.table.fill_(-1)
        cache.lens.zero_()
        b = cache.batch(seqs, counts)
        cache.reserve(b)
        torch.cuda.synchronize()
        assert b.pos0.cpu().tolist() == pos0 and cache.info.cpu().tolist() == info
        at = 0
        for s, c, p in zip(seqs, counts, pos0):
            given = -(-c // 64) if p >= 0 else 0
            assert int(cache.lens[s]) == (c if p >= 0 else 0)
            assert torch.equal(cache.table[s, :given], torch.arange(at, at + given, dtype=torch.int32, device="cuda"))
            assert bool((cache.table[s, given:] == -1).all())
            at += given
        assert int(cache.refs.sum()) == at and bool((cache.refs[:at] == 1).all())


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e7, 1e10, 1e20, 1e29])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 3000.0])
def test_queries_that_see_one_key(mine, capi, size, scale, rows):
    """Logits from 10^4 to 10^30, each row's along one key: that position's value comes out, and nothing leaves f16 on the way."""
    length = 700
    cache = _kv4.Cache(mine, capi, 12, kv_heads=1, q_heads=4, stride=12, rows=rows)
    _kv4.store(cache, 0, gauss(1, length, 128, seed=1), gauss(1, length, 128, seed=2) * scale)
    held = [torch.zeros(length, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(cache.batch([0], [length], [0]), *held)
    at = torch.randint(0, length - rows, (rows, 4), generator=torch.Generator().manual_seed(7)).cuda()
    q = (held[0][at].float() * size).bfloat16().view(rows, -1)  # |k|^2 is about 128, other products at most 6 times 11
    b = cache.batch([0], [rows], [length - rows])
    out = torch.full_like(q, 7.0)
    cache.attention(b, q, out)
    torch.cuda.synchronize()
    # the weight of any other is below e^(-size 60 / sqrt(128)); f16 twice and bf16 twice, the second for what is compared with
    want = held[1][at].double().view(rows, -1)
    off = (out.double() - want).abs()
    top = want.abs().view(rows, 4, 128).amax(-1, keepdim=True).expand(-1, -1, 128).reshape(rows, -1)
    assert bool((off <= want.abs() * 2 ** -7 * 1.01 + top * 2 ** -9).all()), float((off / top).max())
