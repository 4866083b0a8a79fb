"""GPU parity of the norms of queries and keys with the rotation in the same pass, and of their gradients, against plain
restatements in float64 on the CPU.

Tolerances, from the roundings alone (half a step: bf16 2^-8, fp32 2^-24 of the value; e = 2^-24):

* y = R (w x r): r = 1 / sqrt(mean + eps) of a sum of at most 256 squares, of which a lane adds at most 16 and a tree of at most
  6 levels the rest: (16 + 6 + 2) e / 2 and 2 e for the root; three products, 3 e; cos and sin good to 2^-21, two products and a
  sum, 3 e. Together below 20 e + 2^-21 < 2^-19 of |y1| + |y2| of the pair, besides the result's own rounding.
* g = R^T dy is off by (2^-21 + 3 e) (|dy1| + |dy2|) =: below 2^-20 G. dx = r (w g - x^ mean(w g x^)): each of its two terms is
  off by that, r's 14 e (twice in x^ mean) and the mean's 24 e + 4 e: below 2^-18 r (|w| G + |x^| mean(|w| G |x^|)).
* dw = sum of g x^: each term below 2^-19.5 G |x^|, and the order of the sum: a thread adds up what its workgroup takes, here
  fewer than 128 terms, then trees and 64 partial sums in turn at most: 200 e < 2^-16.3. Together 2^-16 sum(G |x^|).
"""
import math

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pairs(x, f, layout):
    """Channels of the first and of the second of every pair."""
    i = torch.arange(f.numel())
    return (i, i + f.numel()) if layout == "half" else (2 * i, 2 * i + 1)


def turn64(x, pos, f, layout, mscale, back=False):
    """(x turned, |x1| + |x2| of each channel's pair; |x| where it is not turned)"""
    a = pos.double().unsqueeze(-1) * f
    c, s = (a.cos() * mscale).unsqueeze(-2), (a.sin() * (-mscale if back else mscale)).unsqueeze(-2)
    first, second = pairs(x, f, layout)
    y, big = x.clone(), x.abs()
    y[..., first], y[..., second] = x[..., first] * c - x[..., second] * s, x[..., first] * s + x[..., second] * c
    big[..., first] = big[..., second] = (x[..., first].abs() + x[..., second].abs()) * mscale
    return y, big


def norm64(x, w, pos, f, layout="half", mscale=1.0, eps=1e-6):
    x, w = x.double(), w.double()
    return turn64(x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w, pos, f, layout, mscale)


def grads64(dy, x, w, pos, f, layout, mscale, eps):
    """((dx, its bound), (dw, its bound)), the bounds without their factors 2^-18 and 2^-16."""
    x, w = x.double(), w.double()
    g, G = turn64(dy.double(), pos, f, layout, mscale, back=True)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    u, h, H = x * r, w * g, w.abs() * G
    dx = r * (h - u * (h * u).mean(-1, keepdim=True))
    big = r * (H + u.abs() * (H * u.abs()).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return (dx, big), ((g * u).sum(lead), (G * u.abs()).sum(lead))


def close(got, want, big, factor, what):
    tol = HALF[got.dtype] * (1 + 2.0 ** -8) * want.abs() + factor * big
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by {float((err - tol).max())}"


CASES = [  # leading shape, query heads, key heads, D, rotary_dim, first position
    ((1,), 12, 12, 128, 128, 1024), ((2, 33), 4, 2, 64, 64, 0), ((3, 7), 20, 4, 80, 32, 1000000), ((5,), 3, 1, 256, 256, 7),
    ((4,), 2, 1, 256, 2, 3), ((9,), 1, 3, 2, 2, 5), ((2, 3), 3, 3, 50, 50, 9), ((70,), 5, 5, 36, 16, 1 << 33), ((600,), 12, 4, 128, 64, -3),
    ((11,), 3, 2, 7, 2, 4), ((5000,), 12, 2, 128, 128, 0), ((13,), 0, 2, 64, 64, 1), ((13,), 2, 0, 64, 32, 1), ((700,), 2, 2, 18, 18, 0)]


def make(lead, hq, hk, D, rd, first, dtype, wdtype, seed=0):
    g = gen(seed + D + rd)
    q, k = (torch.randn(*lead, h, D, generator=g).mul(torch.rand(*lead, h, 1, generator=g) * 3).to(dtype) for h in (hq, hk))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdtype) for _ in range(2))
    pos = (first + torch.arange(math.prod(lead))).view(lead)
    return q, k, wq, wk, pos


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)],
                         ids=["bf16", "bf16-w32", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("lead,hq,hk,D,rd,first", CASES)
def test_values_and_gradients(pkg, lead, hq, hk, D, rd, first, layout, dtype, wdtype):
    ops = pkg.ops
    q, k, wq, wk, pos = make(lead, hq, hk, D, rd, first, dtype, wdtype)
    f, mscale = ops.rotary_frequencies(rd, scaling="yarn", factor=4.0)
    m32, eps = float(torch.tensor(mscale, dtype=torch.float32)), float(torch.tensor(1e-5, dtype=torch.float32))
    leaves = [t.to(dev()).requires_grad_() for t in (q, k, wq, wk)]
    y = ops.qk_norm_rotary(*leaves, pos.to(dev()), f.to(dev()), layout, mscale, eps)
    dy = [torch.randn(*lead, h, D, generator=gen(h)).to(dtype) for h in (hq, hk)]
    grads = torch.autograd.grad(y, leaves, [d.to(dev()) for d in dy])
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        assert y[i].dtype == dtype and y[i].shape == x.shape and y[i].is_contiguous()
        if x.numel() == 0:
            assert not bool(grads[2 + i].any())
            continue
        close(y[i], *norm64(x, w, pos, f, layout, m32, eps), 2.0 ** -19, f"y{i}")
        (dx, bx), (dw, bw) = grads64(dy[i], x, w, pos, f, layout, m32, eps)
        assert grads[i].dtype == dtype and grads[2 + i].dtype == wdtype
        close(grads[i], dx, bx, 2.0 ** -18, f"dx{i}")
        close(grads[2 + i], dw, bw, 2.0 ** -16, f"dw{i}")
    again = torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos.to(dev()), f.to(dev()), layout, mscale, eps), leaves, [d.to(dev()) for d in dy])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))  # the same bits


def test_gradients_against_differences(pkg):
    """Along random directions: the float32 gradients against central differences of the float64 forward."""
    ops = pkg.ops
    q, k, wq, wk, pos = make((3, 5), 4, 2, 48, 16, 11, torch.float32, torch.float32)
    f, _ = ops.rotary_frequencies(16)
    dy = [torch.randn(3, 5, h, 48, generator=gen(h)) for h in (4, 2)]

    def loss(a, b, c, d):
        return sum((norm64(x, w, pos, f)[0] * g.double()).sum() for x, w, g in ((a, c, dy[0]), (b, d, dy[1])))

    leaves = [t.to(dev()).requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos.to(dev()), f.to(dev())), leaves, [d.to(dev()) for d in dy])
    at = [t.double() for t in (q, k, wq, wk)]
    for i in range(4):
        v = torch.randn(at[i].shape, generator=gen(40 + i)).double()
        h = 1e-4  # the third derivative's share, h^2, and the forward's 2^-53 / h both stay below 1e-7 of the sums here
        up, down = ([x + (s * h * v if j == i else 0) for j, x in enumerate(at)] for s in (1, -1))
        want = float(loss(*up) - loss(*down)) / (2 * h)
        got = float((grads[i].cpu().double() * v).sum())
        # the gradient's own bound, 2^-18 of sums that are below 8 |grad| |v| here, and 1e-6 for the differences
        assert abs(got - want) <= (2.0 ** -15 + 1e-6) * float(grads[i].cpu().double().norm() * v.norm()), i


def test_strides_views_and_broadcasts(pkg):
    ops = pkg.ops
    f, _ = ops.rotary_frequencies(64)
    fd = f.to(dev())
    w = (1 + 0.3 * torch.randn(2, 64, generator=gen(1))).to(torch.bfloat16)
    wd = w.to(dev())
    qkv = torch.randn(3, 11, 9, 64, generator=gen(2)).to(torch.bfloat16).to(dev())
    pos = torch.randint(0, 5000, (3, 11), generator=gen(3))
    flat = torch.randn(3 * 11 * 4 * 64 + 1, device=dev()).bfloat16()
    for name, q in {"front heads": qkv[:, :, :4], "every other token": qkv[:, ::2, :4], "heads first": torch.randn(3, 4, 11, 64, device=dev()).bfloat16().transpose(1, 2),
                    "channels strided": torch.randn(3, 11, 64, 4, device=dev()).bfloat16().transpose(2, 3), "unaligned": flat[1:].view(3, 11, 4, 64),
                    "odd rows": torch.randn(3, 11, 4, 67, device=dev()).bfloat16()[..., :64],
                    "broadcast heads": qkv[:, :, :1].expand(3, 11, 4, 64), "one token everywhere": qkv[:1, :1, :4].expand(3, 11, 4, 64)}.items():
        p = pos[:, :q.shape[1]]
        k = qkv[:, :q.shape[1], 4:6]
        for at in (p.to(dev()), p.to(torch.int32).to(dev()), p.to(dev()).t().contiguous().t()):
            yq, yk = ops.qk_norm_rotary(q, k, wd[0], wd[1], at, fd)
            close(yq, *norm64(q.cpu(), w[0], p, f), 2.0 ** -19, name)
            close(yk, *norm64(k.cpu(), w[1], p, f), 2.0 ** -19, name)
    # a broadcast leaf's gradient is the sum over its copies; a gradient of one value everywhere has strides of 0
    one = torch.randn(3, 11, 1, 64, generator=gen(4)).to(dev()).requires_grad_()
    w32 = w[0].float().to(dev())
    y, _ = ops.qk_norm_rotary(one.expand(3, 11, 4, 64), qkv[:, :, :1].float(), w32, w32, pos.to(dev()), fd)
    g, = torch.autograd.grad(y.sum(), one)
    ones = torch.ones(3, 11, 4, 64)
    (dx, bx), _ = grads64(ones, one.detach().cpu().expand(3, 11, 4, 64), w[0].float(), pos, f, "half", 1.0, 1e-6)
    close(g, dx.sum(2, keepdim=True), bx.sum(2, keepdim=True), 2.0 ** -18 + 4 * 2.0 ** -24, "broadcast")
    for shape in ((0, 11), (3, 0)):
        a, b = ops.qk_norm_rotary(qkv[:shape[0], :shape[1], :4], qkv[:shape[0], :shape[1], 4:6], wd[0], wd[1], pos[:shape[0], :shape[1]].to(dev()), fd)
        assert a.shape == (*shape, 4, 64) and b.shape == (*shape, 2, 64)


def test_which_gradients_are_asked(pkg):
    """Any of the four leaves, either of the outputs: what is asked for is the same as with all of them."""
    ops = pkg.ops
    q, k, wq, wk, pos = make((40,), 3, 2, 64, 64, 5, torch.bfloat16, torch.float32)
    f = ops.rotary_frequencies(64)[0].to(dev())
    dy = [torch.randn(40, h, 64, generator=gen(h)).to(torch.bfloat16).to(dev()) for h in (3, 2)]
    base = [t.to(dev()) for t in (q, k, wq, wk)]
    leaves = [t.clone().requires_grad_() for t in base]
    want = torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos.to(dev()), f), leaves, dy)
    for i in range(4):
        args = [t.clone().requires_grad_(j == i) for j, t in enumerate(base)]
        y = ops.qk_norm_rotary(*args, pos.to(dev()), f)
        assert y[0].requires_grad and y[1].requires_grad
        g, = torch.autograd.grad([y[i % 2]], [args[i]], [dy[i % 2]])  # the other output takes no part
        if i < 2:
            assert torch.equal(g, want[i])
        else:  # (a sum whose order goes by the heads that take part)
            x, w = ((q, wq), (k, wk))[i - 2]
            close(g, *grads64(dy[i - 2].cpu(), x, w, pos, f.cpu(), "half", 1.0, 1e-6)[1], 2.0 ** -16, f"dw{i - 2}")
    y = ops.qk_norm_rotary(*leaves, pos.to(dev()), f)
    g = torch.autograd.grad([y[1]], leaves, [dy[1]], allow_unused=True)
    assert g[0] is None and g[2] is None and torch.equal(g[1], want[1])
    with torch.no_grad():
        assert not ops.qk_norm_rotary(*leaves, pos.to(dev()), f)[0].requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_ends_of_the_range(pkg, dtype, eps):
    """Heads whose squares leave float32's range at either end, zeros, and what is not finite stays in its head."""
    ops = pkg.ops
    f = ops.rotary_frequencies(32)[0]
    x = torch.randn(8, 1, 64, generator=gen(7))
    for i, e in enumerate((-120, -100, -70, -64, 0, 62, 100, 124)):
        x[i] *= 2.0 ** e
    x = x.to(dtype)
    w = torch.ones(64)
    pos = torch.arange(8)
    xd = x.to(dev()).requires_grad_()
    e32 = float(torch.tensor(eps, dtype=torch.float32))
    y, _ = ops.qk_norm_rotary(xd, xd.detach()[:, :0], w.to(dev()), w.to(dev()), pos.to(dev()), f.to(dev()), eps=eps)
    want, big = norm64(x, w, pos, f, eps=e32)
    # (below 2^-126 float32 rounds by up to 2^-150; a head's largest values are above that but for the smallest heads with an eps)
    close(y, want, big + 2.0 ** -120, 2.0 ** -19, "y")
    dy = torch.randn(8, 1, 64, generator=gen(8)).to(dtype)
    g, = torch.autograd.grad(y, xd, dy.to(dev()))
    (dx, bx), _ = grads64(dy, x, w, pos, f, "half", 1.0, e32)
    keep = dx.abs().amax((1, 2)) < 2.0 ** 126  # 1 / size itself must be a float32
    keep &= dx.abs().amax((1, 2)) > 2.0 ** -110  # and so must the gradient
    assert int(keep.sum()) >= 5
    close(g[keep.to(dev())], dx[keep], bx[keep], 2.0 ** -18, "dx")
    bad = torch.randn(4, 2, 64, generator=gen(9)).to(dtype)
    bad[1, 0, 3], bad[2, 1, 40] = float("nan"), float("inf")
    y, _ = ops.qk_norm_rotary(bad.to(dev()), bad.to(dev())[:, :0], w.to(dev()), w.to(dev()), pos[:4].to(dev()), f.to(dev()))
    fine = torch.isfinite(y).all(-1).cpu()
    assert torch.equal(fine, torch.tensor([[True, True], [False, True], [True, False], [True, True]]))
    z = torch.zeros(3, 2, 64, dtype=dtype, device=dev())
    assert not ops.qk_norm_rotary(z, z, w.to(dev()), w.to(dev()), pos[:3].to(dev()), f.to(dev()))[0].any()


def test_refusals(pkg):
    ops = pkg.ops
    q, k = (torch.zeros(5, h, 64, dtype=torch.bfloat16, device=dev()) for h in (4, 2))
    w, pos, f = torch.ones(64, device=dev()), torch.arange(5, device=dev()), ops.rotary_frequencies(64)[0].to(dev())
    one = torch.zeros(5, 2, 300, device=dev())
    for bad in (lambda: ops.qk_norm_rotary(q, k.float(), w, w, pos, f), lambda: ops.qk_norm_rotary(q, k[:4], w, w, pos, f),
                lambda: ops.qk_norm_rotary(q, k[..., :32], w, w, pos, f), lambda: ops.qk_norm_rotary(q, k, w[:32], w, pos, f),
                lambda: ops.qk_norm_rotary(q, k, w, w.bfloat16(), pos, f), lambda: ops.qk_norm_rotary(q, k, w.half(), w.half(), pos, f),
                lambda: ops.qk_norm_rotary(q.float(), k.float(), w.bfloat16(), w.bfloat16(), pos, f),
                lambda: ops.qk_norm_rotary(q, k, w, w, pos[:4], f), lambda: ops.qk_norm_rotary(q, k, w, w, pos.float(), f),
                lambda: ops.qk_norm_rotary(q, k, w, w, pos, f.float()), lambda: ops.qk_norm_rotary(q, k, w, w, pos, f[:0]),
                lambda: ops.qk_norm_rotary(q, k, w, w, pos, f, "other"), lambda: ops.qk_norm_rotary(q, k, w, w, pos, f, eps=-1.0),
                lambda: ops.qk_norm_rotary(q, k, w, w, pos, f, eps=float("nan")), lambda: ops.qk_norm_rotary(q.half(), k.half(), w, w, pos, f),
                lambda: ops.qk_norm_rotary(one, one, one[0, 0], one[0, 0], pos, f), lambda: ops.qk_norm_rotary(q.cpu(), k, w, w, pos, f),
                lambda: ops.qk_norm_rotary(q, k, w[::2].repeat_interleave(2)[None], w, pos, f),
                lambda: ops.qk_norm_rotary(q, k, w, w, pos, f.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="prunepath"):
            bad()
    x = q.clone().requires_grad_()
    y, _ = ops.qk_norm_rotary(x, k, w, w, pos, f)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    y, _ = ops.qk_norm_rotary(x, k, w, w, pos, f)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        y.sum().backward()
    y, _ = ops.qk_norm_rotary(x, k, w, w, pos, f)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def test_opcheck(pkg):
    from torch.library import opcheck
    t = pkg._lib.torch_ops()
    q, k, wq, wk, pos = (x.to(dev()) for x in make((5,), 4, 2, 64, 32, 3, torch.bfloat16, torch.float32))
    f = pkg.ops.rotary_frequencies(32)[0].to(dev())
    for op, args in ((t.qk_norm_rotary, (q, k, wq, wk, pos, f)),
                     (t.qk_norm_rotary, (q.clone().requires_grad_(), k, wq.clone().requires_grad_(), wk, pos, f, "interleaved", 1.5, 1e-5)),
                     (t.qk_norm_rotary_bwd, (q, k, q, k, wq, wk, pos, f)),
                     (t.qk_norm_rotary_bwd, (q, k, q, k, wq, wk, pos, f, "half", 1.0, 1e-6, False))):
        print(f"opcheck {op}", flush=True)
        opcheck(op, args)


def test_compiled_training_step(pkg):
    """Traced with its gradient: the same numbers as eager."""
    q, k, wq, wk, pos = (x.to(dev()) for x in make((40,), 4, 2, 64, 32, 3, torch.bfloat16, torch.float32))
    f = pkg.ops.rotary_frequencies(32)[0].to(dev())
    t = pkg._lib.torch_ops()
    dy = [torch.randn_like(q), torch.randn_like(k)]

    def run(fn):
        leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
        y = fn(*leaves)
        return (*y, *torch.autograd.grad(y, leaves, dy))

    plain = lambda a, b, c, d: t.qk_norm_rotary(a, b, c, d, pos, f, "interleaved", 1.0, 1e-5)  # noqa: E731
    torch._dynamo.reset()
    for a, b in zip(run(torch.compile(plain, backend="aot_eager")), run(plain)):
        assert torch.equal(a, b)


def test_captured_with_its_backward(pkg):
    """A training step of the norm captured and replayed, eager work of its own between the replays; another stream."""
    ops = pkg.ops
    q, k, wq, wk, pos = (x.to(dev()) for x in make((300,), 4, 2, 128, 128, 3, torch.bfloat16, torch.bfloat16))
    f = ops.rotary_frequencies(128)[0].to(dev())
    dy = [torch.randn_like(q), torch.randn_like(k)]

    def step(leaves):
        y = ops.qk_norm_rotary(*leaves, pos, f)
        return (*[t.detach() for t in y], *torch.autograd.grad(y, leaves, dy))

    def leaves():
        return [t.clone().requires_grad_() for t in (q, k, wq, wk)]

    want = step(leaves())
    mine = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(mine)
    for i in range(4):
        with torch.no_grad():
            mine[0].copy_(q * (i + 1))
            mine[2].copy_(wq + i)
        graph.replay()
        torch.cuda.synchronize()
        eager = [q * (i + 1), k, wq + i, wk]
        for a, b in zip(out, step([t.clone().requires_grad_() for t in eager])):
            assert torch.equal(a, b), i
