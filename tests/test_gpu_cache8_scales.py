"""Appends onto blocks of the 8-bit cache whose older tokens have a scale that no append writes, as in a cache that was quantised
elsewhere: bytes below 10 (an all-small block), above 246, and 255, which is no number. The older tokens are brought to the scale
that the block then has, whichever way the new tokens' values go out. Exact: a byte is one rounding to e4m3."""
import pytest
import torch

from helpers import dev
from test_gpu_cache8 import E4, E8, least, round8
from test_gpu_paged import gen

pytestmark = pytest.mark.gpu

STORED = [0, 1, 3, 5, 8, 9, 10, 11, 127, 200, 245, 246, 247, 248, 251, 254, 255]


def bring(x8, stored, byte):
    """Values of the scale 2^(stored - 127) at 2^(byte - 127): what bfloat16 has room for is at most 448, the rest no number."""
    y = x8 * 2.0 ** (stored - byte) if stored < 255 else torch.full_like(x8, float("nan"))
    return torch.where(y.abs() < 512, round8(y), float("nan"))


@pytest.mark.parametrize("size", [0.0, 2.0 ** -126, 1.0, 2.0 ** 127], ids=["zeros", "small", "ones", "large"])
@pytest.mark.parametrize("lo,nt", [(1, 1), (15, 1), (3, 4), (3, 5), (9, 7), (12, 20)])
@pytest.mark.parametrize("dim,heads", [(128, 1), (64, 3)])
def test_append_onto_scales_of_elsewhere(pkg, dim, heads, lo, nt, size):
    """A sequence for each stored byte; its first block holds lo tokens, the new ones fill it and may go on in the next."""
    n = len(STORED)
    g = gen(lo + 16 * nt + dim)
    held = round8(448 * (2 * torch.rand(2, n, heads, 16, dim, generator=g).double() - 1) * torch.exp2(-torch.randint(0, 14, (2, n, heads, 16, 1), generator=g).double()))
    held[..., 0, 0], held[..., 0, 1], held[..., 0, 2] = 448, -2.0 ** -9, float("nan")
    held[0, 0, 0, 0, 3] = 0
    new = (size * (2 * torch.rand(2, n * nt, heads, dim, generator=g) - 1)).float()
    pages = 2 * n
    k, v = torch.zeros(pages, heads, 16, dim, dtype=E4), torch.zeros(pages, heads, 1, dim, 16, dtype=E4)
    k[:n], v[:n, :, 0] = held[0].float().to(E4), held[1].transpose(2, 3).float().to(E4)
    scales = [torch.tensor(STORED + [127] * n, dtype=torch.uint8)[:, None, None].expand(pages, heads, 1).contiguous() for _ in range(2)]
    table = torch.stack((torch.arange(n), n + torch.arange(n)), 1).int()
    lens = torch.full((n,), lo + nt, dtype=torch.int32)
    cache = [t.to(dev()) for t in (k, v, table, lens, torch.arange(0, (n + 1) * nt, nt, dtype=torch.int32))]
    s = tuple(x.view(E8).to(dev()) for x in scales)
    pkg.ops.kv_append(new[0].to(dev()), new[1].to(dev()), *cache, scales=s)
    got = cache[0].cpu().double()[:n], cache[1].cpu().double()[:n, :, 0].transpose(2, 3)
    first = min(nt, 16 - lo)
    rows = pkg.ops.kv_read(*cache[:3], lens.to(dev()), torch.arange(0, (n + 1) * (lo + nt), lo + nt, dtype=torch.int32).to(dev()),
                           n * (lo + nt), scales=s)
    for side, name in enumerate(("k", "v")):
        bytes_ = s[side].cpu().view(torch.uint8)[:n, :, 0]
        read = rows[side].cpu().double().view(n, lo + nt, heads, dim)
        for i, stored in enumerate(STORED):
            for h in range(heads):
                x = new[side, i * nt:i * nt + first, h].double()
                byte = max(least(float(x.abs().max())) + 127, min(max(stored, 10), 246))
                assert int(bytes_[i, h]) == byte, (name, stored, int(bytes_[i, h]), byte)
                old = held[side, i, h, :lo] if byte == stored else bring(held[side, i, h, :lo], stored, byte)
                want = torch.cat((old, round8(x * 2.0 ** (127 - byte))))
                have = got[side][i, h, :lo + first]
                assert bool(((have == want) | (torch.isnan(have) & torch.isnan(want))).all()), (name, stored, byte)
                back = read[i, :lo + first, h]
                want = want * 2.0 ** (byte - 127)
                assert bool(((back == want) | (torch.isnan(back) & torch.isnan(want))).all()), (name, stored, byte)


def test_read_of_scales_of_elsewhere(pkg):
    """Each byte at each of the 256 scales: the product, rounded once to bfloat16 (subnormal numbers among them); 255 is no number."""
    pages, dim = 256, 64
    b = torch.arange(16 * dim).remainder(256).to(torch.uint8)
    k = b.view(1, 1, 16, dim).expand(pages, 1, 16, dim).contiguous().view(E4)
    v = b.view(1, 1, 1, dim, 16).expand(pages, 1, 1, dim, 16).contiguous().view(E4)
    s = torch.arange(pages).to(torch.uint8).view(pages, 1, 1)
    table, lens = torch.arange(pages).int()[:, None], torch.full((pages,), 16, dtype=torch.int32)
    got = pkg.ops.kv_read(*(t.to(dev()) for t in (k, v, table, lens, torch.arange(0, 16 * pages + 1, 16).int())), 16 * pages,
                          scales=(s.to(dev()).view(E8), s.to(dev()).view(E8).clone()))
    power = torch.exp2(torch.arange(pages).double() - 127)
    power[255] = float("nan")
    for x, held in zip(got, (k.view(pages, 16, dim), v.view(pages, dim, 16).transpose(1, 2))):
        want = (held.double() * power[:, None, None]).to(torch.bfloat16).double()  # (float64 to bfloat16: one rounding)
        x = x.cpu().double().view(pages, 16, dim)
        assert bool(((x == want) | (torch.isnan(x) & torch.isnan(want))).all())
