"""Values at the ends of their range in the rotary positions and the attention over the paged cache. The
restatement in float64 and the tolerances are those of test_gpu_paged."""
import math

import pytest
import torch

from helpers import dev
from test_gpu_paged import LONG, Batch, attend64, check_attention, few, gen

pytestmark = pytest.mark.gpu

FORMS = [([1, 1], [300, 200], 0), ([3], [700], 0), ([40, 50], [300, 90], LONG)]  # 16-row tiles, 128-row tiles


# ------------------------------------------------------------------ infinities in attended values
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,total,room", FORMS)
def test_attended_infinities(pkg, new, total, room, dim):
    """Of tokens that every row attends, in steps without a masked place: a channel with one infinity is
    that infinity, one with both or with NaN is NaN, the others are as they were."""
    b = Batch(new, total, 16, 2, dim, seed=dim, extra=2 + room // 16)
    assert few(b, 2, 2) == (room == 0)
    q = torch.randn(b.n, 2, dim, generator=gen(1)).to(torch.bfloat16)
    o, big = attend64(b, q)
    inf = float("inf")
    want = o.clone()
    for p, h, d, x in ((7, 0, 5, inf), (40, 0, 20, -inf), (9, 1, 33, inf), (41, 1, 33, -inf), (12, 1, 50, float("nan"))):
        id, off = b.place(0, p)
        b.v[id, h, d, off] = x
        want[:new[0], h, d] += x
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    odd = ~torch.isfinite(want)
    assert int(odd.sum()) == 4 * new[0]
    assert torch.allclose(got[odd].double(), want[odd], equal_nan=True)
    check_attention(torch.where(odd, o.to(got.dtype), got), o, big, few(b, 2, 2))


# ------------------------------------------------------------------ scores of any size
@pytest.mark.parametrize("power", [8, 14, 20, 40, 54])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("new,total,room", FORMS)
def test_scores_beyond_the_exponential(pkg, new, total, room, sign, power):
    """Scores of 2^(2 power) and more, exact in float32 and apart by 2^-7 of themselves: each row takes the
    largest alone (equal ones in equal parts)."""
    b = Batch(new, total, 16, 1, 64, seed=power, extra=2 + room // 16)
    assert few(b, 1, 1) == (room == 0)
    q = torch.full((b.n, 1, 64), sign * 2.0 ** power, dtype=torch.bfloat16)
    j = torch.randint(0, 128, (b.pages, 1, 16, 1), generator=gen(power))
    b.k = ((1 + j / 128) * 2.0 ** power).expand(b.pages, 1, 16, 64).to(torch.bfloat16).contiguous()
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu(), scale=0.1)
    check_attention(got, *attend64(b, q, 0.1), few(b, 1, 1))


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -126, 2.0 ** -130])
@pytest.mark.parametrize("new,total,room", FORMS)
def test_scales_next_to_zero(pkg, new, total, room, scale):
    """Scores up to 2^126 under scales that leave next to nothing of them: 0 takes the mean."""
    b = Batch(new, total, 16, 1, 64, seed=3, extra=2 + room // 16)
    q = torch.full((b.n, 1, 64), 2.0 ** 60, dtype=torch.bfloat16)
    j = torch.randint(0, 64, (b.pages, 1, 16, 1), generator=gen(4))
    b.k = ((j - 32) / 32 * 2.0 ** 60).expand(b.pages, 1, 16, 64).to(torch.bfloat16).contiguous()
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu(), scale=scale)
    check_attention(got, *attend64(b, q, scale), few(b, 1, 1))


@pytest.mark.parametrize("scale", [0.25, 0.5, 0.68])
@pytest.mark.parametrize("new,total,room", FORMS)
def test_scores_next_to_the_lowest_float(pkg, new, total, room, scale):
    """Every score is 64 * -2^60 * 1.875 * 2^61 = -3.19e38, finite: the mean, not a row of nothing."""
    b = Batch(new, total, 16, 1, 64, seed=5, extra=2 + room // 16)
    q = torch.full((b.n, 1, 64), -(2.0 ** 60), dtype=torch.bfloat16)
    b.k.fill_(1.875 * 2.0 ** 61)
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu(), scale=scale)
    check_attention(got, *attend64(b, q, scale), few(b, 1, 1))


# ------------------------------------------------------------------ angles next to the zeros of cos and sin
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles_next_to_a_quarter_turn(pkg, layout):
    """(1, 0) turned by angles within 2^-24 of multiples of a quarter turn is (cos, sin), good to 2^-21 of
    itself however small: the angle beyond a float32 must not be lost. (sincospif is good to 4 units of
    2^-23; what a float32 half turn leaves of the angle is added to first order, 2^-50 off; the float64 product
    is good to 2^-51 of angles up to 7, and the rest is room for the float64 restatement's own 2 pi.)"""
    k = torch.arange(1, 5, dtype=torch.float64)[:, None]
    part = torch.tensor([-0.45, -0.2, -0.01, 0.03, 0.3, 0.48], dtype=torch.float64)[None]
    f = (math.pi * (0.5 * k + part * 2.0 ** -24)).flatten()
    x = torch.zeros(1, 1, 2 * f.numel(), dtype=torch.float32)
    i = torch.arange(f.numel())
    first, second = (i, i + f.numel()) if layout == "half" else (2 * i, 2 * i + 1)
    x[..., first] = 1.0
    y = pkg.ops.rotary(x.to(dev()), torch.ones(1, dtype=torch.int64, device=dev()), f.to(dev()), layout).cpu().double()
    for got, want in ((y[0, 0, first], f.cos()), (y[0, 0, second], f.sin())):
        assert bool(((got - want).abs() <= 2.0 ** -21 * want.abs() + 2.0 ** -48).all()), (got - want).abs().max()


# ------------------------------------------------------------------ masked places and rows of nothing, both tiles
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,total,room", [([5, 3], [70, 3], 0), ([70, 60], [90, 400], LONG), ([130, 33], [900, 40], LONG)])
def test_what_is_masked_does_not_reach_a_row(pkg, new, total, room, dim):
    """NaN and infinities behind the sequences' ends and in pages that no table names; then in the last new token's
    value (three channels) and key: that row alone has them."""
    b = Batch(new, total, 16, 2, dim, seed=dim, extra=2 + room // 16)
    assert few(b, 2, 2) == (room == 0)
    q = torch.randn(b.n, 2, dim, generator=gen(2)).to(torch.bfloat16)
    clean, big = attend64(b, q)
    for s, t in enumerate(total):
        id, off = b.place(s, t - 1)
        b.k[id, :, off + 1:] = float("nan")
        b.v[id, 0, :, off + 1:], b.v[id, 1, :, off + 1:] = float("inf"), float("nan")
    unused = sorted(set(range(b.pages)) - set(b.table.flatten().tolist()))
    b.k[unused], b.v[unused] = float("nan"), -float("inf")
    check_attention(pkg.ops.paged_attention(q.to(dev()), *b.gpu()), clean, big, few(b, 2, 2))
    last = new[0] - 1
    id, off = b.place(0, total[0] - 1)
    for h, d, x in ((0, 5, float("nan")), (0, dim - 1, float("inf")), (1, 33, -float("inf"))):
        b.v[id, h, d, off] = x
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    assert math.isnan(got[last, 0, 5]) and got[last, 0, dim - 1] == float("inf") and got[last, 1, 33] == -float("inf")
    keep = torch.ones(got.shape, dtype=torch.bool)
    keep[last, 0, 5] = keep[last, 0, dim - 1] = keep[last, 1, 33] = False
    check_attention(torch.where(keep, got, clean.to(got.dtype)), clean, big, few(b, 2, 2))
    b.v[id, 0, 5, off] = b.v[id, 0, dim - 1, off] = b.v[id, 1, 33, off] = 0.0
    b.k[id, 0, off, 3] = float("nan")
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    assert bool(torch.isnan(got[last, 0]).all())
    got[last], clean[last] = 0, 0
    check_attention(got, clean, big, few(b, 2, 2))


@pytest.mark.parametrize("scale", [0.125, 1.0, 4.0, -0.5])
@pytest.mark.parametrize("new,total,room", [([2], [60], 0), ([40], [60], LONG), ([40], [1500], LONG), ([1], [2000], 0)])
def test_rows_of_minus_infinity_in_both_tiles(pkg, new, total, room, scale):
    """Scores of -inf for every attended token give zeros; one finite score among them, in whichever range, that
    token's value; a NaN among them NaN."""
    b = Batch(new, total, 16, 1, 64, seed=9, extra=2 + room // 16)
    assert few(b, 1, 1) == (room == 0)
    kp, vp, table, lens, cu = b.gpu()
    q = torch.full((b.n, 1, 64), 1.0 if scale > 0 else -1.0, dtype=torch.bfloat16, device=dev())
    kp.fill_(float("-inf"))
    assert not pkg.ops.paged_attention(q, kp, vp, table, lens, cu, scale=scale).any()
    for p in (5, total[0] - new[0]):  # the first row's own place among them
        id, off = b.place(0, p)
        kp[id, 0, off] = -3.0
        got = pkg.ops.paged_attention(q, kp, vp, table, lens, cu, scale=scale)[:, 0]
        assert torch.equal(got, vp[id, 0, :, off].expand(b.n, 64))
        kp[id, 0, off] = float("nan")
        assert bool(pkg.ops.paged_attention(q, kp, vp, table, lens, cu, scale=scale).isnan().all())
        kp[id, 0, off] = float("-inf")
