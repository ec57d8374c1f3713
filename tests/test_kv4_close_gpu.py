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
