"""GPU parity of the rotary positions, the append to the paged cache and the attention over it,
against plain restatements in float64 on the CPU.

Tolerances, from the roundings alone (half a step: bf16 2^-8, fp32 2^-24 of the value):

* rotary: the result's own rounding, and 2^-21 (|x1| + |x2|) mscale for cos and sin (the angle in
  turns is rounded to float32 once, 2^-25 of at most one half turn, and sin / cos are good to 2^-22)
  and the two products' float32 roundings; and 2^-51 of the angle itself, which at a position of 2^40
  is 5e-4: a float64 product is rounded by up to 2^-53 of its value, once in the restatement here
  (position * inv_freq) and three times in the kernel (1 / 2 pi, times inv_freq, times position).
* attention: the result's rounding 2^-8 |o|, plus (e_P + 2^-10) sum_t p_t |v_t|: e_P = 2^-8 where P
  enters the second product as one bf16 value (tiles of 128 rows), 2^-16 where it enters as two;
  2^-10 covers the float32 scores (sizes here: scale |q| |k| <= 64, 2^-24 x 128 sums), the
  exponentials and the sums.
"""
import math

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: BF}


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ rotary
def turn64(x, pos, f, layout, mscale=1.0, inverse=False):
    """(y, per channel (|x1| + |x2|) times the error of cos and sin) in float64: x [..., heads, D],
    pos [...]."""
    x, rd = x.double(), 2 * f.numel()
    a = pos.double().unsqueeze(-1) * f
    c, s = (a.cos() * mscale).unsqueeze(-2), (a.sin() * (-mscale if inverse else mscale)).unsqueeze(-2)
    i = torch.arange(rd // 2)
    first, second = (i, i + rd // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y, big = x.clone(), torch.zeros_like(x)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    off = 2.0 ** -21 + 2.0 ** -51 * a.abs().unsqueeze(-2)
    big[..., first] = big[..., second] = (x[..., first].abs() + x[..., second].abs()) * mscale * off
    return y, big


def check_turn(got, x, pos, f, layout, mscale=1.0, inverse=False, what=""):
    y, big = turn64(x.cpu(), pos.cpu(), f.cpu(), layout, mscale, inverse)
    tol = HALF[got.dtype] * (1 + 2.0 ** -8) * y.abs() + big
    err = (got.cpu().double() - y).abs()
    bad = int((~(err <= tol)).sum())
    assert bad == 0, f"{what}: {bad} off, the worst by {float((err - tol).max())} at {int((err - tol).argmax())}"


ROT = [  # shape of x, rotary_dim, position of the first token
    ((1, 24, 128), 128, 1024), ((5, 3, 64), 64, 0), ((3, 7, 5, 80), 32, 1000000), ((2, 33, 2, 128), 64, 77),
    ((4, 1, 2), 2, 3), ((2, 3, 3, 50), 50, 9), ((3, 2, 36), 16, 1 << 40), ((1, 1, 1024), 1024, 5), ((300, 12, 128), 128, 0),
    ((9, 2, 24), 8, -5)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape,rd,first", ROT)
def test_rotary(pkg, shape, rd, first, layout, dtype):
    ops = pkg.ops
    f, mscale = ops.rotary_frequencies(rd, scaling="yarn", factor=4.0)
    x = torch.randn(shape, generator=gen(rd)).to(dtype)
    pos = (first + torch.arange(math.prod(shape[:-2]))).view(shape[:-2])
    y = ops.rotary(x.to(dev()), pos.to(dev()), f.to(dev()), layout, mscale)
    assert y.dtype == dtype and y.shape == x.shape
    check_turn(y, x, pos, f, layout, float(torch.tensor(mscale, dtype=torch.float32)), what=f"{shape} {rd}")
    assert torch.equal(y[..., rd:].cpu(), x[..., rd:])  # the rest is copied


def test_rotary_strides_positions_and_views(pkg):
    ops = pkg.ops
    f, _ = ops.rotary_frequencies(64)
    fd = f.to(dev())
    qkv = torch.randn(3, 11, 9, 64, generator=gen(1)).to(torch.bfloat16).to(dev())
    pos = torch.randint(0, 5000, (3, 11), generator=gen(2))
    for name, x in {"front heads": qkv[:, :, :4], "back heads": qkv[:, :, 5:], "every other token": qkv[:, ::2],
                    "heads first": torch.randn(3, 4, 11, 64, device=dev()).transpose(1, 2),
                    "channels strided": torch.randn(3, 11, 64, 4, device=dev()).transpose(2, 3),
                    "unaligned": torch.randn(3 * 11 * 4 * 64 + 1, device=dev())[1:].view(3, 11, 4, 64),
                    "odd rows": torch.randn(3, 11, 4, 67, device=dev())[..., :64],
                    "broadcast heads": torch.randn(3, 11, 1, 64, device=dev()).expand(3, 11, 4, 64)}.items():
        p = pos[:, :x.shape[1]]
        for q in (p.to(dev()), p.to(torch.int32).to(dev()), p.to(dev()).t().contiguous().t()):
            check_turn(ops.rotary(x, q, fd), x, p, f, "half", what=name)
    one = torch.arange(11, device=dev())
    check_turn(ops.rotary(qkv[:, :, :4], one.expand(3, 11), fd), qkv[:, :, :4], one.expand(3, 11), f, "half")
    assert ops.rotary(qkv[:0, :, :4], pos[:0].to(dev()), fd).shape == (0, 11, 4, 64)
    assert ops.rotary(qkv[:, :, :0], pos.to(dev()), fd).shape == (3, 11, 0, 64)


def test_rotary_non_finite_values_stay_in_their_pair(pkg):
    f, _ = pkg.ops.rotary_frequencies(32)
    x = torch.randn(4, 2, 64, generator=gen(4))
    x[1, 0, 3], x[2, 1, 40] = float("nan"), float("inf")
    y = pkg.ops.rotary(x.to(dev()), torch.arange(1, 5, device=dev()), f.to(dev())).cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 19] = want[2, 1, 40] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradients(pkg, layout, dtype):
    """Against the formula (the turn by the opposite angles) and, in float32, against differences of
    the float64 forward; a broadcast input's gradient is the sum over its copies."""
    ops = pkg.ops
    f, mscale = ops.rotary_frequencies(16, scaling="yarn", factor=2.0)
    m32 = float(torch.tensor(mscale, dtype=torch.float32))
    x = torch.randn(3, 5, 4, 24, generator=gen(5)).to(dtype)
    g = torch.randn(3, 5, 4, 24, generator=gen(6)).to(dtype)
    pos = torch.randint(0, 900, (3, 5), generator=gen(7))
    xd = x.to(dev()).requires_grad_()
    y = ops.rotary(xd, pos.to(dev()), f.to(dev()), layout, mscale)
    grad, = torch.autograd.grad(y, xd, g.to(dev()))
    assert grad.dtype == dtype
    check_turn(grad, g, pos, f, layout, m32, inverse=True, what="gradient")
    d = torch.randn(x.shape, generator=gen(8), dtype=torch.float64)
    h = 1e-3
    up, down = (turn64(x.double() + e * d, pos, f, layout, m32)[0] for e in (h, -h))
    slope = float(((up - down) / (2 * h) * g.double()).sum())
    # the gradient's entries are off by at most the rounding and 2^-21 of their pair (see above)
    lim = float(((HALF[dtype] + 2.0 ** -20) * 2 * mscale * g.double().abs().max() * d.abs()).sum()) + 1e-6
    assert abs(float((grad.cpu().double() * d).sum()) - slope) <= lim
    one = torch.randn(3, 5, 1, 24, generator=gen(9)).to(dev()).requires_grad_()
    g32 = g.float().to(dev())
    ops.rotary(one.expand(3, 5, 4, 24), pos.to(dev()), f.to(dev()), layout, mscale).backward(g32)
    each = turn64(g.float(), pos, f, layout, m32, inverse=True)[0].sum(2, keepdim=True)
    assert float((one.grad.cpu().double() - each).abs().max()) <= 4 * (2.0 ** -20) * 4 * float(g.abs().max()) * mscale


def test_rotary_second_gradient(pkg):
    """The map is linear and its gradient's map is one too: the gradient of the gradient's product
    with v is the turn of v."""
    f = pkg.ops.rotary_frequencies(32)[0]
    x = torch.randn(6, 2, 32, generator=gen(1), dtype=torch.float32).to(dev()).requires_grad_()
    g = torch.randn(6, 2, 32, generator=gen(2)).to(dev()).requires_grad_()
    v = torch.randn(6, 2, 32, generator=gen(3))
    pos = torch.arange(6)
    grad, = torch.autograd.grad(pkg.ops.rotary(x, pos.to(dev()), f.to(dev())), x, g, create_graph=True)
    (grad * v.to(dev())).sum().backward()
    check_turn(g.grad, v, pos, f, "half", what="second gradient")


def test_rotary_backward_twice_and_forward_mode(pkg):
    """The graph of a call serves one backward, or more where it is kept; forward mode is refused."""
    ops = pkg.ops
    f, pos = ops.rotary_frequencies(32)[0].to(dev()), torch.arange(3, device=dev())
    x = torch.randn(3, 2, 32, device=dev()).requires_grad_()
    y = ops.rotary(x, pos, f).sum()
    a, = torch.autograd.grad(y, x, retain_graph=True)
    b, = torch.autograd.grad(y, x)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x)
    y = ops.rotary(x, pos, f)
    pos.add_(1)  # what the backward needs is no longer there
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ops.rotary(fw.make_dual(x.detach(), torch.ones_like(x)), pos, f)


def test_rotary_refusals(pkg):
    ops = pkg.ops
    f = ops.rotary_frequencies(32)[0].to(dev())
    x, p = torch.zeros(2, 3, 32, device=dev()), torch.zeros(2, dtype=torch.int64, device=dev())
    for bad in (lambda: ops.rotary(x.half(), p, f), lambda: ops.rotary(x, p.float(), f), lambda: ops.rotary(x, p[:1], f),
                lambda: ops.rotary(x, p, f.float()), lambda: ops.rotary(x, p, f, "other"),
                lambda: ops.rotary(x[..., :16], p, f), lambda: ops.rotary(x[0], p, f), lambda: ops.rotary(x, p.cpu(), f)):
        with pytest.raises(RuntimeError, match="prunepath"):
            bad()


# ------------------------------------------------------------------ the paged cache
class Batch:
    """A ragged batch: new[s] new tokens, total[s] with the cached ones; every page distinct, in
    random order, entries behind a sequence's last page -1."""

    def __init__(self, new, total, page, kv_heads, dim, seed=0, spare=3, extra=2):
        g = gen(seed)
        self.new, self.total, self.page, self.dim = new, total, page, dim
        used = [max(0, -(-t // page)) for t in total]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((len(new), max(used + [0]) + extra), -1, dtype=torch.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u].to(torch.int32)
            at += u
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(total, dtype=torch.int32)
        self.k = torch.randn(self.pages, kv_heads, page, dim, generator=g).to(torch.bfloat16)
        self.v = torch.randn(self.pages, kv_heads, dim, page, generator=g).to(torch.bfloat16)
        self.n = sum(new)

    def gpu(self):
        return [t.to(dev()) for t in (self.k, self.v, self.table, self.lens, self.cu)]

    def rows(self):
        """(row, sequence, position) of every new token."""
        for s, (n, t) in enumerate(zip(self.new, self.total)):
            for i in range(n):
                yield int(self.cu[s]) + i, s, t - n + i

    def place(self, s, p):
        """(page, place) of position p, or None."""
        if p < 0 or p // self.page >= self.table.shape[1]:
            return None
        id = int(self.table[s, p // self.page])
        return (id, p % self.page) if 0 <= id < self.pages else None


def attend64(b, q, scale=None):
    """(o, sum_t p_t |v_t|) float64 [N, heads, D]; rows that attend nothing are zero."""
    scale = b.dim ** -0.5 if scale is None else scale
    hq, hkv = q.shape[1], b.k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64)
    big = torch.zeros(q.shape, dtype=torch.float64)
    for s in range(len(b.new)):
        at = [(p, b.place(s, p)) for p in range(max(0, b.total[s]))]
        at = [(p, x) for p, x in at if x is not None]
        if not at:
            continue
        pos = torch.tensor([p for p, _ in at])
        pg, off = torch.tensor([x[0] for _, x in at]), torch.tensor([x[1] for _, x in at])
        k, v = b.k[pg, :, off].double(), b.v[pg, :, :, off].double()  # [T, hkv, D]
        for row, s2, p in b.rows():
            if s2 != s:
                continue
            live = pos <= p
            if not bool(live.any()):
                continue
            kk, vv = (x[live].repeat_interleave(hq // hkv, 1) for x in (k, v))
            w = torch.softmax((q[row].double()[None] * kk).sum(-1) * scale, 0).unsqueeze(-1)
            o[row], big[row] = (w * vv).sum(0), (w * vv.abs()).sum(0)
    return o, big


def few(b, hq, hkv):
    """Whether the call takes the small tiles, where P enters as two bf16 values: at most 16 rows a
    sequence, or little work by what the table could hold."""
    rows = b.n * (hq // hkv)
    work = max(1, rows // 16 + len(b.new)) * hkv * -(-b.table.shape[1] * b.page // 128)
    return rows <= 16 * len(b.new) or work <= 4096


def check_attention(got, o, big, small):
    tol = BF * (1 + BF) * o.abs() + ((2.0 ** -16 if small else BF) + 2.0 ** -10) * big
    err = (got.cpu().double() - o).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
                                f"{float(got.cpu().flatten()[bad.flatten().nonzero()[0, 0]])} for " \
                                f"{float(o.flatten()[bad.flatten().nonzero()[0, 0]])}"


ATT = [  # new, total, page, heads, kv_heads, dim
    ([1], [1], 16, 1, 1, 128), ([1], [17], 16, 2, 2, 64), ([1], [700], 16, 12, 12, 128), ([1, 1, 1], [130, 1, 257], 32, 8, 2, 128),
    ([1] * 5, [31, 32, 33, 64, 500], 16, 16, 1, 128), ([3], [3], 16, 4, 4, 128), ([2, 5, 1], [40, 5, 129], 64, 6, 2, 64),
    ([20], [20], 16, 1, 1, 128), ([25, 30], [25, 300], 128, 2, 2, 64), ([40], [40], 16, 3, 3, 128),
    ([129], [129], 16, 2, 2, 128), ([64, 1, 70], [300, 200, 70], 32, 8, 4, 64), ([200], [1500], 64, 4, 1, 128),
    ([33, 0, 40], [33, 50, 41], 16, 5, 1, 128), ([150], [2000], 256, 1, 1, 64), ([0, 0, 1], [5, 0, 5], 16, 2, 1, 128)]


LONG = 1 << 20  # tokens that a table has room for beyond what is used: the large tiles where there are more than 16 rows


@pytest.mark.parametrize("room", [0, LONG], ids=["", "long-table"])
@pytest.mark.parametrize("new,total,page,heads,kv_heads,dim", ATT)
def test_paged_attention(pkg, new, total, page, heads, kv_heads, dim, room):
    b = Batch(new, total, page, kv_heads, dim, seed=len(new) + page, extra=2 + room // page)
    assert few(b, heads, kv_heads) == (room == 0 or b.n * (heads // kv_heads) <= 16 * len(new))
    q = (2 * torch.randn(b.n, heads, dim, generator=gen(dim))).to(torch.bfloat16)
    print(new, total, page, heads, kv_heads, dim, flush=True)
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
    o, big = attend64(b, q)
    check_attention(got, o, big, few(b, heads, kv_heads))
    again = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
    assert torch.equal(got, again)


def test_attention_lengths_and_tables_that_hold_no_token(pkg):
    """Lengths below the new tokens (rows at negative positions), of zero, beyond the table; entries
    of -1 and beyond the cache in the middle: those tokens are not attended, empty rows are zero."""
    for new, total in (([3, 2, 4, 1], [1, 0, 300, 90]), ([60, 80, 50, 70], [40, 0, 400, 100])):
        b = Batch(new, total, 16, 2, 128, seed=3, extra=0)
        if new[0] > 3:
            b.table = torch.cat([b.table, torch.full((4, LONG // 16), -1, dtype=torch.int32)], 1)
        b.table[2, 2], b.table[2, 5], b.table[3, 0] = -1, b.pages, -7
        if new[0] == 3:
            b.table[3, :] = -1  # a row with no page at all
        b.total[2] = int(b.lens[2]) + 500  # longer than the table
        b.lens[2] += 500
        q = torch.randn(b.n, 4, 128, generator=gen(1)).to(torch.bfloat16)
        got = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
        o, big = attend64(b, q)
        check_attention(got, o, big, few(b, 4, 2))
        assert bool((got[:new[0] - total[0]] == 0).all()) and not bool(torch.isnan(got).any())


@pytest.mark.parametrize("new,total,room", [([5, 3], [70, 3], 0), ([70, 60], [90, 400], 0), ([70, 60], [90, 400], LONG)])
def test_attention_masked_places_do_not_reach_a_row(pkg, new, total, room):
    """NaN and infinities in the places behind a sequence's end, in pages of other sequences and in
    later tokens' keys and values: earlier rows are as if they were not there; rows that attend them
    are not finite in the channels of V that are not."""
    b = Batch(new, total, 32, 2, 64, seed=9, extra=2 + room // 32)
    assert few(b, 2, 2) == (room == 0)
    q = torch.randn(b.n, 2, 64, generator=gen(2)).to(torch.bfloat16)
    clean, big = attend64(b, q)
    for s, t in enumerate(total):  # behind the end
        id, off = b.place(s, t - 1)
        b.k[id, :, off + 1:] = float("nan")
        b.v[id, :, :, off + 1:] = float("inf")
    unused = sorted(set(range(b.pages)) - set(b.table.flatten().tolist()))
    b.k[unused], b.v[unused] = float("nan"), float("nan")
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
    check_attention(got, clean, big, few(b, 2, 2))
    # the last new token of sequence 0 has NaN, +inf and -inf in three channels of its value
    id, off = b.place(0, total[0] - 1)
    b.v[id, 0, 5, off], b.v[id, 0, 6, off], b.v[id, 1, 7, off] = float("nan"), float("inf"), -float("inf")
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    last = new[0] - 1
    assert math.isnan(got[last, 0, 5]) and got[last, 0, 6] == float("inf") and got[last, 1, 7] == -float("inf")
    keep = torch.ones(got.shape, dtype=torch.bool)
    keep[last, 0, 5] = keep[last, 0, 6] = keep[last, 1, 7] = False
    assert bool(torch.isfinite(got[keep]).all())
    check_attention(torch.where(keep, got, clean.to(got.dtype)), clean, big, few(b, 2, 2))
    # and NaN in its key: the last row alone
    b.v[id, 0, 5, off] = b.v[id, 0, 6, off] = b.v[id, 1, 7, off] = 0.0
    b.k[id, 0, off, 3] = float("nan")
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    assert bool(torch.isnan(got[last, 0]).all())
    got[last], o = 0, clean.clone()
    o[last] = 0
    check_attention(got, o, big, few(b, 2, 2))


def test_attention_rows_behind_the_last_sequence(pkg):
    for new, total, room in (([2, 1], [40, 33], 0), ([70, 66], [70, 200], 0), ([70, 66], [70, 200], LONG)):
        b = Batch(new, total, 16, 1, 128, seed=4, extra=2 + room // 16)
        q = torch.randn(b.n + 9, 2, 128, generator=gen(3)).to(torch.bfloat16).to(dev())
        got = pkg.ops.paged_attention(q, *b.gpu())
        o, big = attend64(b, q[:b.n].cpu())
        check_attention(got[:b.n], o, big, False)
        assert bool((got[b.n:] == 0).all())
        out = torch.full_like(q, 7.0)
        assert pkg.ops.paged_attention(q, *b.gpu(), out=out) is out
        assert torch.equal(out[:b.n], got[:b.n]) and bool((out[b.n:] == 7).all())
    empty = Batch([], [], 16, 1, 128)
    got = pkg.ops.paged_attention(q[:3], *empty.gpu())
    assert got.shape == (3, 2, 128) and bool((got == 0).all())
    assert pkg.ops.paged_attention(q[:0], *b.gpu()).shape == (0, 2, 128)


def test_attention_strided_queries_scale_and_shared_pages(pkg):
    """q as part of a joint projection's rows; another scale; two sequences that share a prefix."""
    b = Batch([2, 2], [50, 66], 16, 2, 128, seed=5)
    b.table[1, :3] = b.table[0, :3]
    qkv = torch.randn(4, 8, 128, generator=gen(6)).to(torch.bfloat16)
    q = qkv.to(dev())[:, 2:6]
    got = pkg.ops.paged_attention(q, *b.gpu(), scale=0.25)
    check_attention(got, *attend64(b, qkv[:, 2:6], 0.25), True)
    got = pkg.ops.paged_attention(q, *b.gpu(), scale=-0.05)
    check_attention(got, *attend64(b, qkv[:, 2:6], -0.05), True)
    got = pkg.ops.paged_attention(q, *b.gpu(), scale=0.0)
    check_attention(got, *attend64(b, qkv[:, 2:6], 0.0), True)
    with pytest.raises(RuntimeError, match="scale"):
        pkg.ops.paged_attention(q, *b.gpu(), scale=float("inf"))
    b = Batch([70], [150], 16, 2, 128, seed=5, extra=LONG // 16)
    qkv = torch.randn(70, 8, 128, generator=gen(6)).to(torch.bfloat16)
    for scale in (0.25, -0.05, 0.0):
        got = pkg.ops.paged_attention(qkv.to(dev())[:, 2:6], *b.gpu(), scale=scale)
        check_attention(got, *attend64(b, qkv[:, 2:6], scale), False)


def test_attention_large_scores(pkg):
    """Scores far beyond the exponential's range: one token takes all, whichever step it is in."""
    for new, total, room in (([1, 1], [300, 45], 0), ([40, 50], [300, 50], LONG)):
        b = Batch(new, total, 16, 1, 64, seed=6, extra=2 + room // 16)
        q = torch.randn(b.n, 1, 64, generator=gen(7)).to(torch.bfloat16) * 100
        b.k *= 100
        o, big = attend64(b, q)
        got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu().double()
        # scores up to 1e6 have float32 steps of 2^-4: a row whose two best are that near is left out
        near = torch.zeros(b.n, dtype=torch.bool)
        for row, s, p in b.rows():
            at = [b.place(s, i) for i in range(p + 1)]
            sc = torch.stack([(q[row, 0].double() * b.k[i, 0, j].double()).sum() for i, j in at]).sort(descending=True)[0] / 8
            near[row] = len(at) > 1 and bool(sc[0] - sc[1] < 20)
        assert int(near.sum()) < b.n / 4
        assert bool(((got - o).abs() <= BF * (1 + BF) * o.abs() + 2.0 ** -10 * big)[~near].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("new,total,page,heads,kv_heads,dim,rd",
                         [([1], [1], 16, 4, 4, 128, 128), ([1, 1, 1], [17, 100, 16], 16, 12, 12, 128, 128),
                          ([40, 1, 7], [40, 33, 100], 32, 10, 2, 64, 32), ([130, 0, 5], [200, 9, 3], 64, 3, 3, 128, 64),
                          ([16, 48], [32, 48], 16, 1, 1, 64, 64)])
def test_kv_append(pkg, new, total, page, heads, kv_heads, dim, rd, layout, dtype):
    b = Batch(new, total, page, kv_heads, dim, seed=page)
    f, mscale = pkg.ops.rotary_frequencies(rd, scaling="yarn", factor=4.0)
    m32 = float(torch.tensor(mscale, dtype=torch.float32))
    qkv = torch.randn(b.n + 2, heads + 2 * kv_heads, dim, generator=gen(dim)).to(dtype)  # two rows of padding
    d = qkv.to(dev())
    kp, vp, table, lens, cu = b.gpu()
    args = (d[:, heads:heads + kv_heads], d[:, heads + kv_heads:], kp, vp, table, lens, cu, f.to(dev()), layout, mscale)
    q = pkg.ops.kv_append(*args, q=d[:, :heads])
    want_v, written = b.v.clone(), torch.zeros(b.pages, page, dtype=torch.bool)
    pos = torch.zeros(b.n, dtype=torch.int64)
    for row, s, p in b.rows():
        pos[row] = p
        at = b.place(s, p)
        if at:
            written[at] = True
            want_v[at[0], :, :, at[1]] = qkv[row, heads + kv_heads:].to(torch.bfloat16)
            check_turn(kp[at[0], :, at[1]][None], qkv[row, heads:heads + kv_heads][None], torch.tensor([p]), f, layout, m32, what="k")
    assert torch.equal(vp.cpu(), want_v)
    assert torch.equal(kp.cpu().transpose(1, 2)[~written], b.k.transpose(1, 2)[~written])  # nothing else was written
    assert q.dtype == torch.bfloat16
    check_turn(q[:b.n], qkv[:b.n, :heads], pos, f, layout, m32, what="q")
    assert bool((q[b.n:] == 0).all())
    # q_out: the rows behind the last sequence stay; without q the cache is the same
    out = torch.full_like(q, 3.0)
    assert pkg.ops.kv_append(*args, q=d[:, :heads], q_out=out) is out
    assert torch.equal(out[:b.n], q[:b.n]) and bool((out[b.n:] == 3).all())
    kp2, vp2 = b.k.to(dev()), b.v.to(dev())
    assert pkg.ops.kv_append(args[0], args[1], kp2, vp2, *args[4:]) is None
    assert torch.equal(kp2, kp) and torch.equal(vp2, vp)
    if dtype == torch.bfloat16:  # in place
        own = d[:, :heads].contiguous()
        pkg.ops.kv_append(*args, q=own, q_out=own)
        assert torch.equal(own[:b.n], q[:b.n]) and torch.equal(own[b.n:].cpu(), qkv[b.n:, :heads])


def test_kv_append_without_rotation_and_without_a_place(pkg):
    """inv_freq None: k as it is. Entries outside the cache, lengths beyond the table and below the
    new tokens: those tokens are dropped, nothing else is touched."""
    b = Batch([5, 20, 3], [40, 20, 1], 16, 2, 64, seed=8, extra=0)
    b.table[0, 2] = b.pages
    b.table[1, 0] = -1
    b.lens[2], b.total[2] = 60, 60  # beyond the table's 3 pages: positions 57 .. 59
    kv = torch.randn(2, b.n, 2, 64, generator=gen(9)).to(torch.bfloat16)
    kp, vp, table, lens, cu = b.gpu()
    pkg.ops.kv_append(kv[0].to(dev()), kv[1].to(dev()), kp, vp, table, lens, cu)
    want_k, want_v = b.k.clone(), b.v.clone()
    n = 0
    for row, s, p in b.rows():
        at = b.place(s, p)
        if at:
            n += 1
            want_k[at[0], :, at[1]], want_v[at[0], :, :, at[1]] = kv[0, row], kv[1, row]
    assert 0 < n < b.n
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)


@pytest.mark.parametrize("seqs", [255, 256, 257, 300, 520])
def test_many_sequences(pkg, seqs):
    """Offsets are looked through 256 sequences at a time: single tokens, empty sequences and chunks
    around the borders of such blocks, appended and attended."""
    new = [1] * seqs
    for s in (0, 63, 64, 200, 255, 256, 257, 511):
        if s < seqs:
            new[s] = 0 if s % 2 == 0 else 3
    total = [n + s % 23 for s, n in enumerate(new)]
    b = Batch(new, total, 16, 1, 64, seed=seqs)
    kv = torch.randn(2, b.n + 2, 1, 64, generator=gen(seqs)).to(torch.bfloat16)
    q = torch.randn(b.n + 2, 2, 64, generator=gen(seqs + 1)).to(torch.bfloat16)
    kp, vp, table, lens, cu = b.gpu()
    pkg.ops.kv_append(kv[0].to(dev()), kv[1].to(dev()), kp, vp, table, lens, cu)
    for row, s, p in b.rows():
        at = b.place(s, p)
        b.k[at[0], :, at[1]], b.v[at[0], :, :, at[1]] = kv[0, row], kv[1, row]
    assert torch.equal(kp.cpu(), b.k) and torch.equal(vp.cpu(), b.v)
    got = pkg.ops.paged_attention(q.to(dev()), kp, vp, table, lens, cu)
    o, big = attend64(b, q[:b.n])
    check_attention(got[:b.n], o, big, few(b, 2, 1))
    assert bool((got[b.n:] == 0).all())


def test_rotary_entry_point_in_place(pkg):
    """The C entry point writes a tensor onto itself, with strides of its own."""
    import ctypes
    lib = pkg._lib.lib()
    f = pkg.ops.rotary_frequencies(32)[0].to(dev())
    for D, first in ((64, 0), (36, 1)):  # whole vectors, and elements one by one
        rows = torch.randn(2, 7, 9, D, generator=gen(D)).to(dev())
        x = rows[:, :, first:first + 4]
        want = pkg.ops.rotary(x, torch.arange(7, device=dev()).expand(2, 7), f)
        pos = torch.arange(7, device=dev())
        st = (ctypes.c_int64 * 3)(*x.stride()[:3])
        ps = (ctypes.c_int64 * 2)(0, 1)
        p = ctypes.c_void_p
        keep = rows.clone()
        rc = lib.pp_rotary(p(x.data_ptr()), 0, st, p(pos.data_ptr()), 1, ps, 2, 7, 4, D, p(f.data_ptr()), 32, 0, 1.0, 0,
                           p(x.data_ptr()), st, p(torch.cuda.current_stream().cuda_stream))
        pkg._lib.check(rc, "pp_rotary")
        assert torch.equal(x, want)
        keep[:, :, first:first + 4] = want
        assert torch.equal(rows, keep)  # nothing beside it


def test_paged_refusals(pkg):
    ops = pkg.ops
    b = Batch([2], [20], 16, 2, 64)
    kp, vp, table, lens, cu = b.gpu()
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev())
    f = ops.rotary_frequencies(64)[0].to(dev())
    for bad in (lambda: ops.paged_attention(x.float(), kp, vp, table, lens, cu),
                lambda: ops.paged_attention(x[:, :1], kp, vp, table, lens, cu),
                lambda: ops.paged_attention(x, kp, kp, table, lens, cu),
                lambda: ops.paged_attention(x, kp, vp, table.long(), lens, cu),
                lambda: ops.paged_attention(x, kp, vp, table, lens, cu[:1]),
                lambda: ops.paged_attention(x, kp[:, :, :8], vp[..., :8], table, lens, cu),
                lambda: ops.paged_attention(x.transpose(1, 2), kp, vp, table, lens, cu),
                lambda: ops.paged_attention(x, kp, vp, table, lens, cu, out=x.float()),
                lambda: ops.kv_append(x[:1], x, kp, vp, table, lens, cu),
                lambda: ops.kv_append(x[:, :1], x[:, :1], kp, vp, table, lens, cu),
                lambda: ops.kv_append(x, x.float(), kp, vp, table, lens, cu),
                lambda: ops.kv_append(x, x, kp, vp, table, lens, cu, f.float()),
                lambda: ops.kv_append(x, x, kp, vp, table, lens, cu, f[:4]),
                lambda: ops.kv_append(x, x, kp, vp, table, lens, cu, f, "other"),
                lambda: ops.kv_append(x, x, kp, vp, table, lens, cu, f, q=x[:1]),
                lambda: ops.kv_append(x, x, kp, vp, table, lens, cu, f, q_out=x)):
        with pytest.raises(RuntimeError, match="prunepath"):
            bad()


def test_gradients_and_overlaps_are_refused(pkg):
    ops = pkg.ops
    kp, vp, table, lens, cu = Batch([2], [20], 16, 2, 64).gpu()
    cache = (kp, vp, table, lens, cu)
    x = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=dev())
    f = ops.rotary_frequencies(64)[0].to(dev())
    want = x.clone().requires_grad_()
    pos = torch.arange(2, device=dev())
    rows = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=dev())
    for bad in (lambda: ops.paged_attention(want, *cache), lambda: ops.paged_attention(x, *cache, out=want),
                lambda: ops.kv_append(want, x, *cache), lambda: ops.kv_append(x, want, *cache),
                lambda: ops.kv_append(x, x, *cache, q=want), lambda: ops.rotary(x, pos, f.clone().requires_grad_()),
                lambda: ops.paged_attention(rows[:2], *cache, out=rows[1:3]),
                lambda: ops.paged_attention(x, *cache, out=kp[0, 0, :4].view(2, 2, 64)),
                lambda: ops.kv_append(x, x, *cache, q=rows[:2], q_out=rows[1:3]),
                lambda: ops.kv_append(x, x, *cache, q=x, q_out=x),  # q itself, but k and v too
                lambda: ops.kv_append(x, x, kp, kp.view(vp.shape), table, lens, cu),
                lambda: ops.kv_append(kp[0, 0, :4].view(2, 2, 64), x, *cache)):
        with pytest.raises(RuntimeError, match="prunepath.*(gradient|overlaps)"):
            bad()
    with torch.no_grad():
        a = ops.paged_attention(want, *cache)
    b = x.clone()
    assert ops.paged_attention(b, *cache, out=b) is b and torch.equal(a, b)  # q itself


@pytest.mark.parametrize("new,total,page,heads,kv_heads,room", [
    ([1, 3], [700, 40], 16, 8, 2, 0), ([200, 1], [1500, 9], 64, 4, 1, 0), ([200, 1], [1500, 9], 64, 4, 1, LONG),
    ([70, 60], [90, 400], 16, 4, 4, LONG)])
def test_attention_into_the_queries(pkg, new, total, page, heads, kv_heads, room):
    """out = q, in one range and in several, by both tiles: the bits of a result of its own."""
    b = Batch(new, total, page, kv_heads, 128, extra=2 + room // page)
    cache = b.gpu()
    q = torch.randn(b.n, heads, 128, generator=gen(5)).to(torch.bfloat16).to(dev())
    want = pkg.ops.paged_attention(q, *cache)
    assert pkg.ops.paged_attention(q, *cache, out=q) is q and torch.equal(q, want)


def test_strides_of_single_rows_and_heads_say_nothing(pkg):
    """One token or one head at a stride that is no multiple of 8 elements."""
    ops = pkg.ops
    f = ops.rotary_frequencies(64)[0]
    kp, vp, table, lens, cu = Batch([1], [20], 16, 1, 64).gpu()
    x = torch.randn(64, generator=gen(3)).to(torch.bfloat16).to(dev())
    odd, even = x.as_strided((1, 1, 64), (77, 33, 1)), x.clone().view(1, 1, 64)
    assert torch.equal(ops.kv_append(odd, odd, kp, vp, table, lens, cu, f.to(dev()), q=odd),
                       ops.kv_append(even, even, kp, vp, table, lens, cu, f.to(dev()), q=even))
    assert torch.equal(ops.paged_attention(odd, kp, vp, table, lens, cu),
                       ops.paged_attention(even, kp, vp, table, lens, cu))
    check_turn(ops.rotary(odd, torch.full((1,), 7, device=dev()), f.to(dev())), odd, torch.full((1,), 7), f, "half")


def test_rows_of_nothing_but_minus_infinity(pkg):
    """Scores of -inf for every attended token give zeros, a single finite one that token's value."""
    for new in (2, 40):
        b = Batch([new], [60], 16, 1, 64, seed=9)
        kp, vp, table, lens, cu = b.gpu()
        q = torch.ones(new, 1, 64, dtype=torch.bfloat16, device=dev())
        kp.fill_(float("-inf"))
        assert not pkg.ops.paged_attention(q, kp, vp, table, lens, cu).any()
        page, place = int(b.table[0, 5 // 16]), 5
        kp[page, 0, place] = 0
        assert torch.equal(pkg.ops.paged_attention(q, kp, vp, table, lens, cu)[:, 0], vp[page, 0, :, place].expand(new, 64))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(12, 12, 128, 16), (6, 2, 64, 32)])
def test_chunks_then_tokens_as_a_server_runs_them(pkg, heads, kv_heads, dim, page):
    """Three sequences' prompts in chunks, then single tokens, appended and attended call by call;
    every output against the float64 attention over what has been appended so far, and the decode
    step captured once and replayed with eager work between the replays."""
    ops = pkg.ops
    f = ops.rotary_frequencies(dim)[0]
    fd = f.to(dev())
    total = [70, 5, 41]
    S = len(total)
    per = -(-(max(total) + 6) // page)
    kp, vp = ops.paged_cache(S * per, page, kv_heads, dim, dev())
    kp.fill_(float("nan"))
    vp.fill_(float("nan"))  # nothing that was not appended is attended
    table = torch.randperm(S * per, generator=gen(1)).view(S, per).to(torch.int32)
    td = table.to(dev())
    lens = [0] * S
    hist = [[] for _ in range(S)]

    def data(n, seed):
        return torch.randn(n, heads + 2 * kv_heads, dim, generator=gen(seed)).to(torch.bfloat16)

    def expected(new, qkv):
        o, big = (torch.zeros(qkv.shape[0], heads, dim, dtype=torch.float64) for _ in range(2))
        row = 0
        for s in range(S):
            for i in range(new[s]):
                p = lens[s] - new[s] + i
                k = turn64(qkv[row:row + 1, heads:heads + kv_heads], torch.tensor([p]), f, "half")[0]
                hist[s].append((k[0].to(torch.bfloat16).double(), qkv[row, heads + kv_heads:].double()))
                q = turn64(qkv[row:row + 1, :heads], torch.tensor([p]), f, "half")[0][0].to(torch.bfloat16).double()
                kk, vv = (torch.stack([h[j] for h in hist[s]]).repeat_interleave(heads // kv_heads, 1) for j in (0, 1))
                w = torch.softmax((q * kk).sum(-1) * dim ** -0.5, 0).unsqueeze(-1)
                o[row], big[row] = (w * vv).sum(0), (w * vv.abs()).sum(0)
                row += 1
        return o, big

    def call(qkv, ld, cd):
        q = ops.kv_append(qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], kp, vp, td, ld, cd, fd,
                          q=qkv[:, :heads])
        return ops.paged_attention(q, kp, vp, td, ld, cd)

    def near(got, o, big):  # as above, and two roundings of q and k to bf16 that may fall the other way (2^-8 of a score of at most 4)
        assert bool(((got.cpu().double() - o).abs() <= BF * (1 + BF) * o.abs() + (BF + 2.0 ** -6) * big).all())

    seed = 10
    while any(l < t for l, t in zip(lens, total)):
        new = [min(33, t - l) for l, t in zip(lens, total)]
        lens = [l + n for l, n in zip(lens, new)]
        cu = torch.tensor([sum(new[:i]) for i in range(S + 1)], dtype=torch.int32)
        qkv = data(sum(new), seed)
        got = call(qkv.to(dev()), torch.tensor(lens, dtype=torch.int32, device=dev()), cu.to(dev()))
        near(got, *expected(new, qkv))
        seed += 1
    ld = torch.tensor(lens, dtype=torch.int32, device=dev())
    cd = torch.arange(S + 1, dtype=torch.int32, device=dev())
    x = torch.zeros(S, heads + 2 * kv_heads, dim, dtype=torch.bfloat16, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ld.add_(1)  # the warm-up appends zeros where the first step goes
    with torch.cuda.stream(side):
        call(x, ld, cd)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(x, ld, cd)
    for i in range(4):
        qkv = data(S, seed + i)
        x.copy_(qkv)
        if i:
            ld.add_(1)
        lens = [l + 1 for l in lens]
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        near(got, *expected([1] * S, qkv))
        assert torch.equal(call(x, ld, cd), got)  # eager, the same bits
        out.zero_()


def test_two_graphs_and_two_streams(pkg):
    """Two captured calls replayed one after the other many times, and eager calls on two streams at
    once: each has its own workspace, so the results are the single calls'."""
    ops = pkg.ops
    cases = []
    for seed, (new, total, hq) in enumerate([([1], [3000], 2), ([1, 1], [2000, 900], 4), ([140], [2500], 2)]):
        b = Batch(new, total, 16, 2, 128, seed=seed, extra=LONG // 16)
        q = torch.randn(b.n, hq, 128, generator=gen(seed)).to(torch.bfloat16).to(dev())
        args = b.gpu()
        cases.append((q, args, ops.paged_attention(q, *args).clone()))
    graphs = []
    for q, args, want in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.paged_attention(q, *args)
        graphs.append((g, out))
    for _ in range(5):
        for (g, out), (q, args, want) in zip(graphs, cases):
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        for (g, out), (q, args, want) in zip(graphs, cases):
            assert torch.equal(out, want)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st, (q, args, want) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append((ops.paged_attention(q, *args), want))
    torch.cuda.synchronize()
    for a, w in got:
        assert torch.equal(a, w)


def test_rotary_captured_forward_and_backward(pkg):
    """A training step captured after a warm-up on a side stream and replayed; no eager graph of the
    same leaf is alive during the capture."""
    ops = pkg.ops
    f = ops.rotary_frequencies(64)[0].to(dev())
    x = torch.randn(4, 9, 2, 64, device=dev()).requires_grad_()
    g = torch.randn(4, 9, 2, 64, device=dev())
    pos = torch.arange(9, device=dev()).expand(4, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.rotary(x, pos, f), x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, pos, f)
        gx, = torch.autograd.grad(y, x, g)
        y = y.detach()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(4, 9, 2, 64, generator=gen(i)))
            g.copy_(torch.randn(4, 9, 2, 64, generator=gen(10 + i)))
        graph.replay()
        torch.cuda.synchronize()
        check_turn(y, x.detach(), pos, f, "half")
        check_turn(gx, g, pos, f, "half", inverse=True)
