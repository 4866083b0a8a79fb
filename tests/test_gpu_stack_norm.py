"""A decoder layer whose heads are normed, trained after a call under inference_mode, and a static step that is captured before
any other call.

Tolerance of the gradients: float32 throughout. A weight's gradient goes through six sums of at most 256 terms (projection, norm,
scores, values, output and their mirror images), each off by at most 256 2^-24 of the sum of its terms' magnitudes, together 2^-13.4;
magnitudes may be a few times what is left of a sum: 2^-11 of the largest entry of that gradient."""
import math

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

D, HEADS, LENGTH = 256, 2, 7


def plain(x, w, eps, window, sinks):
    """The layer in float64: the sum over its output, weighted, with norms and turns written out."""
    hd = D // HEADS
    q, k, v = (x @ w["qkv.weight"].t()).view(LENGTH, 3, HEADS, hd).permute(1, 2, 0, 3)
    inv = 10000.0 ** (-2.0 * torch.arange(hd // 2).double() / hd)
    ang = torch.arange(LENGTH).double()[:, None] * inv

    def turned(y, weight):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        return torch.cat((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()), -1)

    q, k = turned(q, w["q_norm.weight"]), turned(k, w["k_norm.weight"])
    s = q @ k.transpose(1, 2) / math.sqrt(hd)
    i, j = torch.arange(LENGTH)[:, None], torch.arange(LENGTH)[None]
    seen = (j <= i) & ((j > i - window) | (j < sinks)) if window else j <= i
    o = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v
    return o.transpose(0, 1).reshape(LENGTH, D) @ w["o.weight"].t()


@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 1)])
def test_trained_after_a_call_under_inference_mode(pkg, window, sinks):
    torch.manual_seed(5)
    attn = pkg.decoder_stack.Attention(D, HEADS, 16, qk_norm=True, window=window, sinks=sinks)
    with torch.no_grad():
        for n in (attn.q_norm, attn.k_norm):
            n.weight.add_(0.5 * torch.randn(n.weight.shape))
    attn = attn.to(dev())
    x, g = torch.randn(2, LENGTH, D).unbind(0)
    with torch.inference_mode():
        attn.reset(1, dev(), torch.float32)
        first = attn(x[None].to(dev()))
    attn.reset(1, dev(), torch.float32)
    y = attn(x[None].to(dev()))
    assert torch.equal(y.detach(), first)
    y.backward(g[None].to(dev()))
    w = {k: v.detach().cpu().double().requires_grad_() for k, v in attn.named_parameters()}
    want = plain(x.double(), w, attn.q_norm.eps, window, sinks)
    want.backward(g.double())
    for name, p in attn.named_parameters():
        exact = w[name].grad
        assert float((p.grad.cpu().double() - exact).abs().max()) <= 2.0 ** -11 * float(exact.abs().max()), name


def test_a_step_that_is_captured_first(pkg):
    """No call before the capture; replays with eager work between them, each against the eager step."""
    torch.manual_seed(6)
    pair = [pkg.decoder_stack.Attention(D, HEADS, 16, qk_norm=True).to(dev()) for _ in range(2)]
    pair[1].load_state_dict(pair[0].state_dict())
    x, pos, mask = torch.zeros(1, 1, D, device=dev()), torch.zeros(1, dtype=torch.int64, device=dev()), torch.zeros(16, device=dev())
    (x @ pair[0].qkv.weight.t())  # the library's own set-up
    with torch.no_grad():
        for a in pair:
            a.reset(1, dev(), torch.float32)
        warm = torch.cuda.Stream()
        with torch.cuda.stream(warm):
            torch.matmul(torch.zeros(1, HEADS, 1, D // HEADS, device=dev()), pair[0].kt_cache)
            torch.matmul(torch.zeros(1, HEADS, 1, 16, device=dev()), pair[0].v_cache)
            torch.nn.functional.linear(x, pair[0].qkv.weight)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pair[0].forward_static(x, pos, mask)
        for t in range(5):
            x.copy_(torch.randn(1, 1, D))
            pos.fill_(t)
            mask.copy_(torch.where(torch.arange(16) <= t, 0.0, float("-inf")))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, pair[1].forward_static(x, pos, mask)), t
