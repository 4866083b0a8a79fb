"""GPU parity of the paged cache of 8 bits: the append that quantises, the read, and the attention over it; and of the
attention's window and first tokens over both caches. Against plain restatements in float64.

Tolerances:

* The append without norms and rotation is exact: the scale is a comparison, the value one rounding of a float32 number that
  is at hand, old values a shift and one rounding. So is the read: a value of 8 bits times its scale is a bfloat16 number.
* With them, what is rounded is off by d = 2^-19 (|y1| + |y2|) (the norm and the turn in float32, as derived for them
  elsewhere), and the rounding to e4m3 is half a step: 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it. The
  scale is the least that holds the largest value, which is itself off by d.
* Attention: as over the bfloat16 numbers that the cache stands for: the result's rounding 2^-8 |o|, and
  (2^-8 + 2^-10) sum_t p_t |v_t| for P as one bf16 value and the float32 scores, exponentials and sums.
"""
import pytest
import torch

from helpers import dev
from test_gpu_paged import Batch, check_attention, gen
from test_gpu_qk_norm import norm64, turn64

pytestmark = pytest.mark.gpu

E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------ the restatement
def round8(x):
    """x rounded to e4m3: four significant bits, steps of 2^-9 below 2^-6, ties to even, 448 the largest."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6, max=448.0))) - 3.0)
    return (torch.round(x / step) * step).clamp(-448, 448)


def least(top):
    """Exponent of the least power of two whose 448-fold is no less than top, within -117 and 119."""
    if top == 0:
        return -117
    n = int(torch.tensor(top / 448.0, dtype=torch.float64).log2().ceil())
    while 448.0 * 2.0 ** (n - 1) >= top:
        n -= 1
    while 448.0 * 2.0 ** n < top:
        n += 1
    return max(-117, min(119, n))


class Batch8(Batch):
    """The batch over a cache of 8 bits: k8 and v8 [pages, heads, page / 16, 16, D] float64, what is held before the scale;
    ek and ev its exponents. Every place and scale holds something from the start, NaN in what no sequence has."""

    def __init__(self, new, total, page, kv_heads, dim, seed=0, spare=3, extra=2, size=1.0):
        super().__init__(new, total, page, kv_heads, dim, seed, spare, extra)
        shape = (self.pages, kv_heads, page // 16, 16, dim)
        g = gen(seed + 1)
        self.k8, self.v8 = (round8(448 * (2 * torch.rand(shape, generator=g).double() - 1)) for _ in range(2))
        self.ek, self.ev = (torch.randint(-9, -5, shape[:3], generator=g) for _ in range(2))
        self.held = torch.zeros(self.pages, page, dtype=torch.bool)
        for s, t in enumerate(total):
            for p in range(max(0, t)):
                at = self.place(s, p)
                if at:
                    self.held[at] = True
        nowhere = ~self.held.view(self.pages, 1, page // 16, 16, 1).expand(shape)
        self.k8[nowhere], self.v8[nowhere] = float("nan"), float("nan")

    def cache(self):
        """(k_pages, v_pages, table, lens, cu), scales, on the GPU."""
        p, h, b, _, d = self.k8.shape
        k = self.k8.float().to(E4).reshape(p, h, self.page, d)
        v = self.v8.transpose(3, 4).float().to(E4).contiguous()
        s = [(e + 127).to(torch.uint8).view(E8).to(dev()) for e in (self.ek, self.ev)]
        return [t.to(dev()) for t in (k, v, self.table, self.lens, self.cu)], s

    def wide(self):
        """The numbers that the cache stands for, as Batch has them."""
        p, h, b, _, d = self.k8.shape
        self.k = (self.k8 * torch.exp2(self.ek.double())[..., None, None]).reshape(p, h, self.page, d)
        self.v = (self.v8 * torch.exp2(self.ev.double())[..., None, None]).reshape(p, h, self.page, d).transpose(2, 3)
        return self

    def append(self, k, v):
        """k and v [n, heads, D] float64 into the cache, block by block."""
        for s, (n, t) in enumerate(zip(self.new, self.total)):
            for block in range((t - n) // 16, (t - 1) // 16 + 1 if n else (t - n) // 16):
                ps = [p for p in range(16 * block, 16 * block + 16) if t - n <= p < t]
                at = self.place(s, ps[0])
                if not at:
                    continue
                rows = [int(self.cu[s]) + p - (t - n) for p in ps]
                page, b, lo = at[0], at[1] // 16, ps[0] % 16
                for x, x8, e in ((k, self.k8, self.ek), (v, self.v8, self.ev)):
                    for h in range(x.shape[1]):
                        y = x[rows, h]
                        fine = torch.isfinite(y)
                        need = least(float(y[fine].abs().max()) if bool(fine.any()) else 0.0)
                        old = int(e[page, h, b])
                        if lo > 0:
                            need = max(need, old)
                            x8[page, h, b, :lo] = round8(x8[page, h, b, :lo] * 2.0 ** (old - need))
                        e[page, h, b] = need
                        x8[page, h, b, lo:lo + len(ps)] = torch.where(fine, round8(y * 2.0 ** -need), float("nan"))

    def check(self, cache, scales, what=""):
        """Every byte of the cache, NaN as NaN, and every scale."""
        p, h, b, _, d = self.k8.shape
        got = cache[0].cpu().double().view(p, h, b, 16, d), cache[1].cpu().double().transpose(3, 4)
        for name, x, x8, s, e in (("k", got[0], self.k8, scales[0], self.ek), ("v", got[1], self.v8, scales[1], self.ev)):
            assert torch.equal(s.cpu().view(torch.uint8).long() - 127, e.long()), f"{what} scales of {name}"
            bad = ~((x == x8) | (torch.isnan(x) & torch.isnan(x8)))
            assert not bool(bad.any()), f"{what} {name}: {int(bad.sum())} off, first at {bad.nonzero()[0].tolist()}: {float(x[bad][0])} for {float(x8[bad][0])}"


# ------------------------------------------------------------------ append
APP = [  # new, total, page, heads, kv_heads, dim
    ([1], [1], 16, 1, 1, 128), ([1, 1, 1], [17, 100, 16], 16, 12, 12, 128), ([40, 1, 7], [40, 33, 100], 32, 10, 2, 64),
    ([130, 0, 5], [200, 9, 3], 64, 3, 3, 128), ([16, 48], [32, 48], 16, 1, 1, 64), ([15, 16, 17, 2], [31, 40, 49, 18], 128, 9, 9, 64),
    ([3] * 9, [5 + 7 * i for i in range(9)], 16, 5, 5, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("new,total,page,heads,kv_heads,dim", APP)
def test_append_is_exact(pkg, new, total, page, heads, kv_heads, dim, dtype):
    """Without rotation: every byte, of old tokens and of untouched places too; values of all sizes."""
    b = Batch8(new, total, page, kv_heads, dim, seed=page + dim)
    g = gen(dim)
    kv = torch.randn(2, b.n + 2, kv_heads, dim, generator=g) * torch.exp2(torch.randint(-6, 7, (2, b.n + 2, kv_heads, 1), generator=g).float())
    kv = kv.to(dtype)
    cache, scales = b.cache()
    d = kv.to(dev())
    assert pkg.ops.kv_append(d[0], d[1], *cache, scales=scales) is None
    b.append(kv[0].double(), kv[1].double())
    b.check(cache, scales)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_token_by_token(pkg, dim):
    """Growing values: the scale of a block grows under its old tokens, by small and by large steps."""
    b = Batch8([1], [1], 16, 2, dim, seed=4, extra=4)
    b.table[0] = torch.tensor([1, 0, 3, 2, -1][:b.table.shape[1]])
    cache, scales = b.cache()
    g = gen(5)
    for i in range(40):
        x = torch.randn(2, 1, 2, dim, generator=g) * 2.0 ** [i, 3 * i - 60, -i, 20 * (i % 5) - 40][i // 10]
        b.total, b.lens = [i + 1], torch.tensor([i + 1], dtype=torch.int32)
        cache[3].fill_(i + 1)
        pkg.ops.kv_append(x[0].to(dev()), x[1].to(dev()), *cache, scales=scales)
        b.append(x[0].double(), x[1].double())
        b.check(cache, scales, f"token {i}")


def test_append_of_special_values(pkg):
    """Zeros, the ends of the range, what is not finite, the borders of a scale and of a rounding."""
    b = Batch8([80], [83], 32, 2, 64, seed=6)
    x = torch.zeros(2, 80, 2, 64)
    flat = x.view(2, 80, -1)
    flat[:, 0:13] = 0.0                                                     # with the three tokens before
    flat[:, 13:29] = torch.finfo(torch.float32).tiny * torch.randn(16, 128, generator=gen(1))
    flat[:, 29:45] = 3.0e38 * (2 * torch.rand(16, 128, generator=gen(2)) - 1)
    flat[:, 29, 0], flat[:, 30, 1] = torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max
    flat[:, 45:61] = torch.randn(16, 128, generator=gen(3))
    flat[:, 45, 5], flat[:, 46, 70], flat[:, 47, 9] = float("inf"), -float("inf"), float("nan")
    flat[:, 61:77, :64] = 448.0                                             # exactly a border
    flat[:, 61:77, 64:] = 448.0 * (1 + 2.0 ** -23)                          # and beyond it
    every = torch.arange(256, dtype=torch.uint8).view(E4).float()
    every = every[torch.isfinite(every)]
    mid = (every[:-1] + every[1:]) / 2                                      # ties
    flat[:, 77, :64], flat[:, 78, :64], flat[:, 79, :64] = mid[:64], mid[60:124], mid[125:189]
    flat[:, 77:80, 64:] = torch.tensor([448.0, 2.0 ** -9, 3 * 2.0 ** -11]).view(3, 1)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        c = Batch8([80], [83], 32, 2, 64, seed=6)
        cache, scales = c.cache()
        pkg.ops.kv_append(y[0].to(dev()), y[1].to(dev()), *cache, scales=scales)
        c.append(y[0].double(), y[1].double())
        c.check(cache, scales, str(dtype))


def test_append_of_every_bf16_value(pkg):
    """Each finite bfloat16 value beside the largest that its block's scale holds, and alone."""
    every = torch.arange(1 << 16).to(torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[torch.isfinite(every)]
    n = every.numel() // 128
    k = every[:n * 128].view(n, 1, 128)
    v = k.flip(0).clone()
    v[:, :, 0] = v[:, :, 0].clamp(-1, 1) * 300
    b = Batch8([n], [n + 5], 64, 1, 128, seed=7)
    cache, scales = b.cache()
    pkg.ops.kv_append(k.to(dev()), v.to(dev()), *cache, scales=scales)
    b.append(k.double(), v.double())
    b.check(cache, scales)


def test_append_where_no_page_is(pkg):
    """Entries outside the cache, lengths beyond the table and below the new tokens, rows behind the last sequence."""
    b = Batch8([5, 20, 3], [40, 20, 1], 16, 2, 64, seed=8, extra=0)
    b.table[0, 2] = b.pages
    b.table[1, 0] = -1
    b.lens[2], b.total[2] = 60, 60  # beyond the table's 3 pages: positions 57 .. 59
    kv = torch.randn(2, b.n + 3, 2, 64, generator=gen(9)).to(torch.bfloat16).to(dev())
    cache, scales = b.cache()
    out = torch.full((b.n + 3, 2, 64), 5.0, dtype=torch.bfloat16, device=dev())
    q = torch.randn(b.n + 3, 2, 64, device=dev()).bfloat16()
    pkg.ops.kv_append(kv[0], kv[1], *cache, q=q, q_out=out, scales=scales)
    b.append(kv[0].cpu().double(), kv[1].cpu().double())
    b.check(cache, scales)
    assert torch.equal(out[:b.n], q[:b.n]) and bool((out[b.n:] == 5).all())
    b = Batch8([4], [2], 16, 2, 64, seed=8)  # two of the rows at negative positions
    cache, scales = b.cache()
    got = pkg.ops.kv_append(kv[0, :6], kv[1, :6], *cache, q=q[:6], scales=scales)
    assert torch.equal(got[:4], q[:4]) and not bool(got[4:].any())
    b.new, b.total, b.cu = [2], [2], torch.tensor([2, 4], dtype=torch.int32)  # as though only the others were there
    b.append(kv[0].cpu().double(), kv[1].cpu().double())
    b.check(cache, scales)


@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)],
                         ids=["bf16", "bf16-w32", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("new,total,page,heads,kv_heads,dim,rd,norm", [
    ([1], [1], 16, 4, 4, 128, 128, True), ([1, 1, 1], [17, 100, 16], 16, 12, 12, 128, 128, True), ([40, 1, 7], [40, 33, 100], 32, 10, 2, 64, 32, True),
    ([130, 0, 5], [200, 9, 3], 64, 3, 3, 128, 64, True), ([40, 1, 7], [40, 33, 100], 32, 6, 6, 64, 64, False),
    ([3, 30], [25, 33], 16, 5, 5, 128, 0, True), ([33, 2], [50, 40], 16, 2, 1, 128, 48, False), ([33, 2], [50, 40], 16, 2, 1, 64, 0, True)])
def test_append_with_norms_and_rotation(pkg, new, total, page, heads, kv_heads, dim, rd, norm, layout, dtype, wdtype, eight):
    if not norm and wdtype != dtype:
        pytest.skip("no weights")
    ops = pkg.ops
    b = Batch8(new, total, page, kv_heads, dim, seed=page)
    f, mscale = (ops.rotary_frequencies(rd, scaling="yarn", factor=4.0)) if rd else (None, 1.0)
    m32 = float(torch.tensor(mscale, dtype=torch.float32))
    qkv = torch.randn(b.n + 2, heads + 2 * kv_heads, dim, generator=gen(dim)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen(i))).to(wdtype) for i in (1, 2))
    eps = float(torch.tensor(1e-4, dtype=torch.float32))
    d = qkv.to(dev())
    cache, scales = b.cache() if eight else (b.gpu(), None)
    more = dict(inv_freq=f.to(dev()) if rd else None, layout=layout, mscale=mscale, scales=scales)
    if norm:
        more |= dict(q_weight=wq.to(dev()), k_weight=wk.to(dev()), eps=eps)
    q = ops.kv_append(d[:, heads:heads + kv_heads], d[:, heads + kv_heads:], *cache, q=d[:, :heads], **more)
    pos = torch.zeros(b.n, dtype=torch.int64)
    for row, _, p in b.rows():
        pos[row] = p

    def turned(x, w):  # (values, how far off before the rounding)
        if norm:
            x = x.double()
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
        y, big = turn64(x.double(), pos, f, layout, m32) if rd else (x.double(), x.double().abs())
        return y, 2.0 ** -19 * big if norm or rd else 0 * big

    want, off = turned(qkv[:b.n, :heads], wq)
    assert bool(((q[:b.n].cpu().double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -8) * want.abs() + off).all())
    assert not bool(q[b.n:].any())
    k, off = turned(qkv[:b.n, heads:heads + kv_heads], wk)
    v = qkv[:b.n, heads + kv_heads:].double()
    if not eight:
        for row, s, p in b.rows():
            at = b.place(s, p)
            if at:
                got = cache[0][at[0], :, at[1]].cpu().double()
                assert bool(((got - k[row]).abs() <= 2.0 ** -8 * (1 + 2.0 ** -8) * k[row].abs() + off[row]).all())
        return
    got8 = cache[0].cpu().double().view(b.k8.shape)
    sk = scales[0].cpu().view(torch.uint8).long() - 127
    before = b.ek.clone()
    old8 = b.k8.clone()
    b.append(k, v)
    near = torch.exp2(sk.double())
    for row, s, p in b.rows():
        at = b.place(s, p)
        if not at:
            continue
        page_, blk, i = at[0], at[1] // 16, at[1] % 16
        for h in range(kv_heads):
            e, want_e = int(sk[page_, h, blk]), int(b.ek[page_, h, blk])
            if e != want_e:  # only where the largest value is that near to a border
                rows = [r for r, s2, p2 in b.rows() if s2 == s and p2 // 16 == p // 16]
                top, slack = float(k[rows, h].abs().max()), float(off[rows, h].max())
                assert abs(e - want_e) == 1 and abs(448.0 * 2.0 ** min(e, want_e) - top) <= slack
            x = got8[page_, h, blk, i] * near[page_, h, blk]
            tol = torch.maximum(2.0 ** -4 * k[row, h].abs(), torch.tensor(2.0 ** -10 * 2.0 ** e, dtype=torch.float64)) * (1 + 2.0 ** -4) + off[row, h]
            assert bool(((x - k[row, h]).abs() <= tol).all())
    same = (sk == b.ek.long())[..., None, None].expand(got8.shape)
    fresh = torch.zeros(b.pages, page, dtype=torch.bool)
    for row, s, p in b.rows():
        if b.place(s, p):
            fresh[b.place(s, p)] = True
    rest = same & ~fresh.view(b.pages, 1, page // 16, 16, 1)
    a, w = got8[rest], b.k8[rest]
    assert bool(((a == w) | (torch.isnan(a) & torch.isnan(w))).all())  # old tokens and untouched places
    b.k8, b.ek = got8, sk  # the values are exact
    b.check(cache, scales)


@pytest.mark.parametrize("seqs", [255, 257, 520])
def test_many_sequences(pkg, seqs):
    new = [1] * seqs
    for s in (0, 63, 64, 200, 255, 256, 257, 511):
        if s < seqs:
            new[s] = 0 if s % 2 == 0 else 3
    total = [n + s % 23 for s, n in enumerate(new)]
    b = Batch8(new, total, 16, 1, 64, seed=seqs)
    kv = torch.randn(2, b.n + 2, 1, 64, generator=gen(seqs)).to(torch.bfloat16)
    q = torch.randn(b.n + 2, 2, 64, generator=gen(seqs + 1)).to(torch.bfloat16)
    cache, scales = b.cache()
    pkg.ops.kv_append(kv[0].to(dev()), kv[1].to(dev()), *cache, scales=scales)
    b.append(kv[0].double(), kv[1].double())
    b.check(cache, scales)
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=9, sinks=2)
    check_attention(got[:b.n], *attend(b.wide(), q[:b.n], 9, 2), False)
    assert not bool(got[b.n:].any())
    k, v = pkg.ops.kv_read(*cache, b.n + 2, scales=scales)
    check_read(b, k, v)


# ------------------------------------------------------------------ read
def check_read(b, k, v):
    want = torch.zeros(2, *k.shape, dtype=torch.float64)
    for row, s, p in b.rows():
        at = b.place(s, p)
        if at:
            want[0, row], want[1, row] = b.k[at[0], :, at[1]].double(), b.v[at[0], :, :, at[1]].double()
    for got, w in ((k, want[0]), (v, want[1])):
        got = got.cpu().double()
        assert bool(((got == w) | (torch.isnan(got) & torch.isnan(w))).all())


@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("new,total,page,kv_heads,dim", [
    ([1], [1], 16, 1, 128), ([17, 0, 100], [17, 0, 100], 16, 12, 128), ([77, 33], [77, 40], 64, 2, 64), ([5, 16, 130], [40, 33, 200], 128, 9, 64),
    ([4, 3], [2, 60], 16, 5, 128)])
def test_read(pkg, new, total, page, kv_heads, dim, eight):
    """Whole sequences and their last rows; entries and positions that hold no token are zeros; rows of no sequence."""
    b = Batch8(new, total, page, kv_heads, dim, seed=dim)
    if len(new) > 1 and b.table.shape[1] > 2:
        b.table[-1, 1] = -1
        b.table[0, 0] = b.pages + 3
    cache, scales = b.cache() if eight else (b.gpu(), None)
    if eight:
        b.wide()
    k, v = pkg.ops.kv_read(*cache, b.n + 3, scales=scales)
    assert k.dtype == v.dtype == torch.bfloat16 and k.shape == v.shape == (b.n + 3, kv_heads, dim)
    check_read(b, k, v)
    out = tuple(torch.full_like(k, 9.0) for _ in range(2))
    assert pkg.ops.kv_read(*cache, scales=scales, out=out) is out
    for x, y in zip(out, (k, v)):
        assert torch.equal(x[:b.n].view(torch.int16), y[:b.n].view(torch.int16)) and bool((x[b.n:] == 9).all())
    assert pkg.ops.kv_read(*cache, 0, scales=scales)[0].shape == (0, kv_heads, dim)


def test_read_of_every_value_at_every_scale(pkg):
    """256 bytes times the 237 scales: bfloat16 numbers, from 2^-126 to 448 * 2^119, exactly."""
    page, heads, dim = 16, 1, 128
    pages = 237
    byte = (torch.arange(16 * dim) % 256).to(torch.uint8).view(16, dim)
    k = byte.expand(pages, heads, 16, dim).contiguous().view(E4)
    v = byte.t().expand(pages, heads, 1, dim, 16).contiguous().view(E4)
    s = torch.arange(10, 247, dtype=torch.uint8).view(pages, 1, 1)
    table = torch.arange(pages, dtype=torch.int32).view(1, pages)
    lens, cu = torch.tensor([pages * 16], dtype=torch.int32), torch.tensor([0, pages * 16], dtype=torch.int32)
    got = pkg.ops.kv_read(*(t.to(dev()) for t in (k, v, table, lens, cu)), pages * 16, scales=(s.view(E8).to(dev()), s.clone().view(E8).to(dev())))
    want = byte.view(E4).double()[None] * torch.exp2(s.double() - 127)
    for x in got:
        x = x.cpu().double().view(pages, 16, dim)
        assert bool(((x == want) | (torch.isnan(x) & torch.isnan(want))).all())
        assert int(torch.isnan(x).sum()) == int(torch.isnan(want).sum()) > 0


@pytest.mark.parametrize("new,total", [([1, 1], [17, 40]), ([70, 3], [90, 3])])
def test_append_onto_the_queries_with_norms(pkg, new, total):
    """q_out = q, both caches: the bits of a result of its own; weights that start anywhere in another tensor."""
    ops = pkg.ops
    b = Batch8(new, total, 16, 2, 128, seed=2)
    f = ops.rotary_frequencies(128)[0].to(dev())
    w = (1 + 0.3 * torch.randn(3 * 128 + 1, generator=gen(1))).to(torch.bfloat16).to(dev())
    q, k, v = (torch.randn(b.n + 1, h, 128, generator=gen(h)).to(torch.bfloat16).to(dev()) for h in (6, 2, 2))
    for eight in (True, False):
        cache, scales = b.cache() if eight else (b.gpu(), None)
        more = dict(inv_freq=f, scales=scales, q_weight=w[1:129], k_weight=w[200:328])
        want = ops.kv_append(k, v, *cache, q=q, **more)
        again = dict(more, q_weight=w[1:129].clone(), k_weight=w[200:328].clone())
        own = q.clone()
        assert ops.kv_append(k, v, *cache, q=own, q_out=own, **again) is own
        assert torch.equal(own[:b.n], want[:b.n]) and torch.equal(own[b.n:], q[b.n:])


def test_append_then_read_over_long_tables(pkg):
    """A cache whose places lie beyond 2^31 bytes: the last pages of one."""
    pages, page, heads, dim = 1100, 4096, 4, 128  # 2.3e9 bytes of keys, as many of values
    k, v = (torch.empty(s, dtype=E4, device=dev()) for s in ((pages, heads, page, dim), (pages, heads, page // 16, dim, 16)))
    s = [torch.empty(pages, heads, page // 16, dtype=E8, device=dev()) for _ in range(2)]
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev())
    lens, cu = torch.tensor([page + 40], dtype=torch.int32, device=dev()), torch.tensor([0, 90], dtype=torch.int32, device=dev())
    x = torch.randn(2, 90, heads, dim, generator=gen(3)).to(torch.bfloat16).to(dev())
    # (the block of the first new token, 4046, holds tokens from before: values of 1)
    k.view(torch.uint8)[-1, :, -64:] = v.view(torch.uint8)[-1, :, -4:] = 0x38
    s[0].view(torch.uint8)[-1, :, -4:] = s[1].view(torch.uint8)[-1, :, -4:] = 127
    pkg.ops.kv_append(x[0], x[1], k, v, table, lens, cu, scales=s)
    got = pkg.ops.kv_read(k, v, table, lens, cu, 90, scales=s)
    for a, b in zip(got, x):
        assert bool(((a - b).abs().float() <= 2.0 ** -4 * b.abs().float() + 2.0 ** -8).all())  # (scales of 2^-6 and 1: 2^-10 of 1 is 2^-10)
    q = torch.randn(90, 4, dim, generator=gen(4)).to(torch.bfloat16).to(dev())
    o = pkg.ops.paged_attention(q, k, v, table, lens, cu, scales=s, window=50)
    kk, vv = (t.double().transpose(0, 1) for t in got)
    p = torch.matmul(q.double().transpose(0, 1), kk.transpose(1, 2)) * dim ** -0.5
    i = torch.arange(90, device=dev())
    hidden = (i[None] > i[:, None]) | (i[None] <= i[:, None] - 50)
    w = torch.softmax(p.masked_fill(hidden, -float("inf")), -1)
    check_attention(o[49:], torch.matmul(w, vv).transpose(0, 1)[49:].cpu(), torch.matmul(w, vv.abs()).transpose(0, 1)[49:].cpu(), False)


# ------------------------------------------------------------------ attention
def attend(b, q, window=0, sinks=0, scale=None):
    """(o, sum_t p_t |v_t|) float64 of b.k and b.v, rows that attend nothing zero; on the GPU, sequence by sequence."""
    scale = b.dim ** -0.5 if scale is None else scale
    hq, hkv, cap = q.shape[1], b.k.shape[1], b.table.shape[1] * b.page
    o, big = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    for s, (n, t) in enumerate(zip(b.new, b.total)):
        ps = torch.arange(max(0, min(t, cap)))
        entry = b.table[s, ps // b.page].long() if len(ps) else ps
        ok = (entry >= 0) & (entry < b.pages)
        ps, entry = ps[ok], entry[ok]
        if not n or not len(ps):
            continue
        k = b.k.transpose(1, 2)[entry, ps % b.page].double().to(dev()).transpose(0, 1).repeat_interleave(hq // hkv, 0)
        v = b.v.permute(0, 3, 1, 2)[entry, ps % b.page].double().to(dev()).transpose(0, 1).repeat_interleave(hq // hkv, 0)
        rows = slice(int(b.cu[s]), int(b.cu[s]) + n)
        x = torch.matmul(q[rows].double().to(dev()).transpose(0, 1), k.transpose(1, 2).contiguous()) * scale
        far = torch.arange(t - n, t)[:, None] - ps[None]
        seen = far >= 0
        if window:
            seen &= (far < window) | (ps < sinks)
        seen = seen.to(dev())
        x = x.masked_fill(~seen, -float("inf"))
        p = torch.softmax(x, -1)
        p = torch.where(seen.any(-1)[None, :, None], p, 0.0)
        v = torch.where(seen.any(0)[None, :, None], v, 0.0)  # (a value that no row attends: 0 times NaN)
        o[rows], big[rows] = torch.matmul(p, v).transpose(0, 1).cpu(), torch.matmul(p, v.abs()).transpose(0, 1).cpu()
    return o, big


ATT = [  # new, total, page, heads, kv_heads, dim
    ([1], [1], 16, 1, 1, 128), ([1], [700], 16, 12, 12, 128), ([1, 1, 1], [130, 1, 257], 32, 8, 2, 128), ([1] * 5, [31, 32, 33, 64, 500], 16, 16, 1, 64),
    ([2, 5, 1], [40, 5, 129], 64, 6, 2, 64), ([20, 3], [20, 900], 16, 1, 1, 128), ([33, 0, 40], [33, 50, 41], 16, 5, 1, 128),
    ([1, 1], [5000, 1025], 16, 2, 2, 128), ([700, 1, 64], [700, 90, 400], 32, 64, 8, 64), ([500, 3, 129], [900, 70, 129], 16, 24, 4, 128),
    ([600], [4000], 256, 8, 8, 128)]
WINDOWS = [(0, 0), (1, 0), (1, 1), (16, 3), (100, 0), (129, 70), (3000, 4), (64, 1000), (1 << 40, 0), (40, 1 << 40)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("new,total,page,heads,kv_heads,dim", ATT)
def test_attention(pkg, new, total, page, heads, kv_heads, dim, eight, window, sinks):
    if not eight and not window:
        pytest.skip("tested elsewhere")
    b = Batch8(new, total, page, kv_heads, dim, seed=page + dim)
    cache, scales = b.cache() if eight else (b.gpu(), None)
    if eight:
        b.wide()
    q = torch.randn(b.n + 2, heads, dim, generator=gen(1)).to(torch.bfloat16)
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window or None, sinks=sinks)
    check_attention(got[:b.n], *attend(b, q[:b.n], window, sinks), False)
    assert not bool(got[b.n:].any())
    own = q.to(dev())
    assert pkg.ops.paged_attention(own, *cache, out=own, scales=scales, window=window or None, sinks=sinks) is own
    assert torch.equal(own[:b.n], got[:b.n]) and torch.equal(own[b.n:].cpu(), q[b.n:])


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("seqs,spread,dim", [(2, 900, 128), (3, 900, 64), (63, 400, 64), (64, 400, 64), (64, 10, 64), (65, 400, 64)])
def test_tiles_in_the_order_of_their_work(pkg, seqs, spread, dim, eight, window, sinks):
    """Up to 64 sequences, and one more, in tiles of 128 rows: lengths of all kinds and nearly equal ones, sequences without rows, at
    the ends too, rows of no sequence behind."""
    rnd = torch.randint(0, 1 << 30, (2, seqs), generator=gen(seqs + spread)).tolist()
    new = [(300 if seqs < 4 else [0, 1, 5, 40, 130][x % 5]) for x in rnd[0]]
    new[0], new[-1] = (0, new[-1]) if seqs % 2 else (new[0], 0)
    total = [n + (0 if n == 0 and x % 3 == 0 else 150 - min(n, 150) + x % spread) for n, x in zip(new, rnd[1])]
    b = Batch8(new, total, 16, 8, dim, seed=seqs)
    cache, scales = b.cache() if eight else (b.gpu(), None)
    if eight:
        b.wide()
    q = torch.randn(b.n + 5, 64, dim, generator=gen(1)).to(torch.bfloat16)
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window or None, sinks=sinks)
    check_attention(got[:b.n], *attend(b, q[:b.n], window, sinks), False)
    assert not bool(got[b.n:].any())
    again = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window or None, sinks=sinks)
    assert torch.equal(again, got)


@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("new,total,heads,kv_heads,dim", [([2, 1, 3], [300, 90, 41], 4, 2, 128), ([400, 70, 1], [700, 300, 90], 64, 8, 64),
                                                           ([400, 70], [700, 300], 48, 8, 128)])
def test_what_is_out_of_the_window_does_not_reach_a_row(pkg, new, total, heads, kv_heads, dim, eight):
    """NaN behind the ends, in the gap between first tokens and window, in pages of others, -1 for pages that no window reaches,
    scales of pages that nothing was appended to; then NaN in an attended place."""
    window, sinks, page = 50, 5, 16
    b = Batch8(new, total, page, kv_heads, dim, seed=9)
    if not eight:
        b.k, b.v = b.k.double(), b.v.double()
    else:
        b.wide()
    q = torch.randn(b.n, heads, dim, generator=gen(2)).to(torch.bfloat16)
    want, big = attend(b, q, window, sinks)
    for s, (n, t) in enumerate(zip(new, total)):
        first = max(0, t - n - window + 1)  # of the first row's window
        for p in range(sinks, first):
            at = b.place(s, p)
            b.k8[at[0], :, at[1] // 16, at[1] % 16], b.v8[at[0], :, at[1] // 16, at[1] % 16] = float("nan"), float("nan")
            b.k[at[0], :, at[1]], b.v[at[0], :, :, at[1]] = float("nan"), float("inf")
        for j in range(1, first // page):
            b.table[s, j] = -1
    b.k[~b.held.any(1)], b.v[~b.held.any(1)] = float("nan"), float("nan")
    cache, scales = b.cache() if eight else ([t.to(dev()) for t in (b.k.bfloat16(), b.v.bfloat16(), b.table, b.lens, b.cu)], None)
    if eight:
        for x in scales:
            x.view(torch.uint8)[(~b.held.any(1)).to(dev())] = 255
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window, sinks=sinks)
    check_attention(got, want, big, False)
    # the second token of sequence 0, one that stays visible: rows of it whose window does not reach it attend it
    at = b.place(0, 1)
    if eight:
        cache[1].view(torch.uint8)[at[0], 0, 0, 5, 1] = 0x7f
    else:
        cache[1][at[0], 0, 5, 1] = float("nan")
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window, sinks=sinks).cpu()
    group = heads // kv_heads
    assert bool(torch.isnan(got[:new[0], :group, 5]).all())
    got[:new[0], :group, 5] = 0
    want[:new[0], :group, 5] = 0
    check_attention(got, want, big, False)
    # and one in the middle of a window: the rows within its reach alone
    if eight:
        cache[1].view(torch.uint8)[at[0], 0, 0, 5, 1] = 0
    else:
        cache[1][at[0], 0, 5, 1] = 0.0
    p = total[0] - 1 - window // 2
    at = b.place(0, p)
    if eight:
        cache[1].view(torch.uint8)[at[0], 0, at[1] // 16, 7, at[1] % 16] = 0xff
    else:
        cache[1][at[0], 0, 7, at[1]] = float("nan")
    got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window, sinks=sinks).cpu()
    mine = torch.tensor([0 <= total[0] - new[0] + i - p < window for i in range(new[0])])
    bad = torch.isnan(got[:new[0], :group, 7])
    assert torch.equal(bad, mine[:, None].expand_as(bad))
    assert int(torch.isnan(got).sum()) == int(bad.sum())


def test_lengths_beyond_the_table_with_a_window(pkg):
    """Positions that the table has no room for attend what their window and the first tokens hold of it, or nothing."""
    for new, heads, kv_heads in (([4, 3], 2, 1), ([300, 280], 64, 8)):
        for eight in (True, False):
            b = Batch8(new, [310, 290], 16, kv_heads, 64, seed=3, extra=0)
            room = b.table.shape[1] * 16
            b.total = [room + 30, room + 400]
            b.lens = torch.tensor(b.total, dtype=torch.int32)
            b.held[:] = True
            b.k8.nan_to_num_(1.0), b.v8.nan_to_num_(1.0)
            cache, scales = b.cache() if eight else (b.gpu(), None)
            if eight:
                b.wide()
            q = torch.randn(b.n, heads, 64, generator=gen(1)).to(torch.bfloat16)
            for window, sinks in ((40, 0), (40, 7)):
                got = pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales, window=window, sinks=sinks)
                o, big = attend(b, q, window, sinks)
                check_attention(got, o, big, False)
                assert sinks or not bool(got[-1].any())


def test_scales_of_the_score_with_8_bits(pkg):
    for new, total, heads, kv_heads in (([2, 3], [70, 300], 4, 2), ([300, 200], [500, 200], 64, 8)):
        b = Batch8(new, total, 16, kv_heads, 64, seed=5).wide()
        cache, scales = b.cache()
        qkv = torch.randn(b.n, heads + 2, 64, generator=gen(6)).to(torch.bfloat16)
        for scale in (0.25, -0.05, 0.0):
            got = pkg.ops.paged_attention(qkv.to(dev())[:, 1:1 + heads], *cache, scale=scale, scales=scales, window=90)
            check_attention(got, *attend(b, qkv[:, 1:1 + heads], 90, 0, scale), False)


def test_blocks_of_very_different_scales(pkg):
    """Values of one block 2^30 times those of the next: each row's error is bounded by what it adds up."""
    for new, total, heads, kv_heads in (([3], [200], 4, 2), ([300], [500], 64, 8)):
        b = Batch8(new, total, 16, kv_heads, 64, seed=5)
        b.ev = torch.where(torch.rand(b.ev.shape, generator=gen(3)) < 0.5, b.ev, b.ev - 30)
        b.ek = b.ek - torch.randint(0, 3, b.ek.shape, generator=gen(4))
        b.wide()
        cache, scales = b.cache()
        q = torch.randn(b.n, heads, 64, generator=gen(1)).to(torch.bfloat16)
        check_attention(pkg.ops.paged_attention(q.to(dev()), *cache, scales=scales), *attend(b, q), False)


def test_tokens_appended_one_by_one_as_a_server_does(pkg):
    """Prompts in chunks, then a captured step of norm, rotation, append and windowed attention, replayed with eager work
    between; on another stream; everything the same as eager, and as the read of the cache says."""
    ops = pkg.ops
    heads, kv_heads, dim, page, S = 6, 2, 64, 16, 3
    f = ops.rotary_frequencies(dim)[0].to(dev())
    w = (1 + 0.2 * torch.randn(2, dim, generator=gen(1))).to(torch.bfloat16).to(dev())
    table = torch.randperm(S * 12, generator=gen(2)).view(S, 12).to(torch.int32).to(dev())

    def fresh():
        (k, v), s = ops.paged_cache8(S * 12, page, kv_heads, dim, dev())
        for x in (k, v, *s):
            x.view(torch.uint8).fill_(255)
        return k, v, s, torch.zeros(S, dtype=torch.int32, device=dev())

    def call(c, qkv, cu):
        k, v, s, lens = c
        q = ops.kv_append(qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], k, v, table, lens, cu, f, q=qkv[:, :heads],
                          q_weight=w[0], k_weight=w[1], scales=s)
        return ops.paged_attention(q, k, v, table, lens, cu, scales=s, window=40, sinks=4), q

    def prompt(c):
        for n in ([70, 5, 41], [0, 30, 2]):
            cu = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32, device=dev())
            c[3].add_(torch.tensor(n, dtype=torch.int32, device=dev()))
            o, q = call(c, torch.randn(sum(n), heads + 2 * kv_heads, dim, generator=gen(sum(n))).to(torch.bfloat16).to(dev()), cu)
        return o, q, cu

    one = torch.arange(S + 1, dtype=torch.int32, device=dev())
    xs = [torch.randn(S, heads + 2 * kv_heads, dim, generator=gen(50 + i)).to(torch.bfloat16).to(dev()) for i in range(12)]
    a, c = fresh(), fresh()
    o, q, cu = prompt(a)
    prompt(c)
    for x, y in zip((*a[:2], *a[2], a[3]), (*c[:2], *c[2], c[3])):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # the same bits
    # the last chunk against the cache read back
    lens = a[3].cpu()
    b = Batch([0, 30, 2], lens.tolist(), page, kv_heads, dim)
    b.table, b.pages = table.cpu(), S * 12
    b.k, b.v = torch.zeros(S * 12, kv_heads, page, dim, dtype=torch.float64), torch.zeros(S * 12, kv_heads, dim, page, dtype=torch.float64)
    full = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).to(torch.int32)]).to(dev())
    k, v = ops.kv_read(a[0], a[1], table, a[3], full, int(lens.sum()), scales=a[2])
    row = 0
    for s in range(S):
        for p in range(int(lens[s])):
            at = b.place(s, p)
            b.k[at[0], :, at[1]], b.v[at[0], :, :, at[1]] = k[row].cpu().double(), v[row].cpu().double()
            row += 1
    check_attention(o, *attend(b, q.cpu(), 40, 4), False)
    # eager steps on `a`; a captured one on `c`
    side, x_t = torch.cuda.Stream(), xs[0].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up, taken back
        keep = [t.clone() for t in (c[0].view(torch.uint8), c[1].view(torch.uint8), *(t.view(torch.uint8) for t in c[2]), c[3])]
        c[3].add_(1)
        call(c, x_t, one)
        for t, old in zip((c[0].view(torch.uint8), c[1].view(torch.uint8), *(t.view(torch.uint8) for t in c[2]), c[3]), keep):
            t.copy_(old)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c[3].add_(1)
        got, _ = call(c, x_t, one)
    for i, x in enumerate(xs):
        a[3].add_(1)
        want, _ = call(a, x, one)
        x_t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
    for x, y in zip((*a[:2], *a[2], a[3]), (*c[:2], *c[2], c[3])):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_opcheck(pkg):
    from torch.library import opcheck
    t = pkg._lib.torch_ops()
    b = Batch8([3, 2], [20, 5], 16, 2, 64)
    cache, s = b.cache()
    f = pkg.ops.rotary_frequencies(64)[0].to(dev())
    q, k, v = (torch.randn(5, h, 64, device=dev(), dtype=torch.bfloat16) for h in (4, 2, 2))
    w = torch.ones(64, device=dev())
    out = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=dev())
    # (test_schema multiplies its arguments, which torch does not for 8-bit types)
    tests = ("test_autograd_registration", "test_faketensor")
    for op, args in ((t.paged_attention, (q, *cache, 0.1, *s, 3, 1)), (t.kv_read, (*cache, 5, *s)),
                     (t.paged_attention, (q, *b.gpu(), 0.1, None, None, 3, 1)), (t.kv_read, (*b.gpu(), 5)),
                     (t.kv_read_into, (*b.gpu(), out, out.clone())),
                     (t.kv_append_q, (q, k, v, *cache, f, "half", 1.0, w, w, 1e-5, *s)),
                     (t.kv_append_q, (q, k, v, *b.gpu(), f, "half", 1.0, w, w, 1e-5))):
        print(f"opcheck {op}", flush=True)
        eight = any(torch.is_tensor(a) and a.dtype == E4 for a in args)
        opcheck(op, args, test_utils=tests if eight else ("test_schema", *tests))


def test_refusals(pkg):
    ops = pkg.ops
    b = Batch8([2], [20], 16, 2, 64)
    (kp, vp, table, lens, cu), (ks, vs) = b.cache()
    c, s = (kp, vp, table, lens, cu), (ks, vs)
    kb, vb = b.gpu()[:2]
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev())
    w = torch.ones(64, device=dev())
    out = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev())
    for bad in (lambda: ops.paged_attention(x, *c), lambda: ops.paged_attention(x, kb, vb, *c[2:], scales=s),
                lambda: ops.paged_attention(x, kp, vb, *c[2:], scales=s), lambda: ops.paged_attention(x, *c, scales=(ks, None)),
                lambda: ops.paged_attention(x, *c, scales=(ks, vs.view(torch.uint8))), lambda: ops.paged_attention(x, *c, scales=(ks, vs[:-1])),
                lambda: ops.paged_attention(x, *c, scales=(ks[..., None], vs)), lambda: ops.paged_attention(x, kp, vp.transpose(3, 4), *c[2:], scales=s),
                lambda: ops.paged_attention(x, *c, scales=s, window=0), lambda: ops.paged_attention(x, *c, scales=s, window=-5),
                lambda: ops.paged_attention(x, *c, scales=s, sinks=3), lambda: ops.paged_attention(x, *c, scales=s, window=3, sinks=-1),
                lambda: ops.paged_attention(x, *c, scales=(ks.cpu(), vs)),
                lambda: ops.kv_append(x, x, *c), lambda: ops.kv_append(x, x, kb, vb, *c[2:], scales=s), lambda: ops.kv_append(x, x, *c, scales=(ks, ks)),
                lambda: ops.kv_append(x, x, *c, scales=(ks, None)), lambda: ops.kv_append(x, x, *c, scales=s, q_weight=w),
                lambda: ops.kv_append(x, x, *c, scales=s, q=x.clone(), q_weight=w), lambda: ops.kv_append(x, x, *c, scales=s, q=x.clone(), k_weight=w),
                lambda: ops.kv_append(x, x, *c, scales=s, k_weight=w[:32]), lambda: ops.kv_append(x, x, *c, scales=s, k_weight=w.half()),
                lambda: ops.kv_append(x, x, *c, scales=s, k_weight=w, eps=-1e-6), lambda: ops.kv_append(x, x, *c, scales=s, k_weight=w[None]),
                lambda: ops.kv_append(x, x, *c, scales=s, k_weight=w.clone().requires_grad_()),
                lambda: ops.kv_append(kp.view(torch.bfloat16)[0, 0, :4].reshape(2, 2, 32).repeat(1, 1, 2), x, *c, scales=(ks, ks.clone()[:, :1])),
                lambda: ops.kv_read(*c, 2), lambda: ops.kv_read(*c, -1, scales=s), lambda: ops.kv_read(*c, scales=s),
                lambda: ops.kv_read(*c, 3, scales=s, out=(out, out.clone())), lambda: ops.kv_read(*c, scales=s, out=(out, out)),
                lambda: ops.kv_read(*c, scales=s, out=(out, out[:1])), lambda: ops.kv_read(*c, scales=s, out=(out.float(), out.float())),
                lambda: ops.kv_read(kb, vb, *c[2:], out=(kb[0, :, :4].reshape(2, 2, 128)[..., :64], out)),
                lambda: ops.kv_read(kb, vb, *c[2:], out=(kb.view(-1)[:256].view(2, 2, 64), out))):
        with pytest.raises(RuntimeError, match="prunepath"):
            bad()


# ------------------------------------------------------------------ uneven batches
@pytest.mark.parametrize("eight", [True, False], ids=["8-bit", "16-bit"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 4), (60, 0)])
@pytest.mark.parametrize("seqs,kv_heads,group,dim", [(2, 8, 4, 128), (20, 8, 1, 64), (64, 8, 2, 64), (63, 8, 1, 128)])
def test_uneven_batches_of_more_tiles_than_one(pkg, seqs, kv_heads, group, dim, window, sinks, eight):
    """128-row tiles, up to five a sequence, of caches between one and a few thousand tokens: with gaps in the tiles' numbers, sequences
    without rows, and rows of no sequence behind. In any order of the batch the same bits."""
    rnd = torch.randint(0, 1 << 30, (2, seqs), generator=gen(seqs + dim)).tolist()
    new = [(150 if seqs > 2 else 500) + x % 60 if x % 5 else 0 for x in rnd[0]]
    new[0] = new[0] or 131
    total = [n + (x % 2600 if x % 3 else x % 40) for n, x in zip(new, rnd[1])]
    order = torch.randperm(seqs, generator=gen(4)).tolist()
    b = Batch8(new, total, 16, kv_heads, dim, seed=seqs)
    cache, scales = b.cache() if eight else (b.gpu(), None)
    if eight:
        b.wide()
    q = torch.randn(b.n + 3, kv_heads * group, dim, generator=gen(1)).to(torch.bfloat16)
    kw = dict(scales=scales, window=window or None, sinks=sinks)
    got = pkg.ops.paged_attention(q.to(dev()), *cache, **kw)
    check_attention(got[:b.n], *attend(b, q[:b.n], window, sinks), False)
    assert not bool(got[b.n:].any())
    rows = torch.cat([torch.arange(int(b.cu[s]), int(b.cu[s + 1])) for s in order])
    cu = torch.tensor([0] + [new[s] for s in order]).cumsum(0).int().to(dev())
    at = torch.tensor(order, device=dev())
    other = pkg.ops.paged_attention(q[rows].to(dev()), *cache[:2], cache[2][at].contiguous(), cache[3][at].contiguous(), cu, **kw)
    assert torch.equal(other, got[rows.to(dev())])
