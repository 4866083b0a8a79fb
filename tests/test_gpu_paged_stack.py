"""The decoder stack served through the paged cache: the attention layer against its float64
restatement over ragged chunks, and whole generations, captured steps against eager ones."""
import math

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stack(pkg):
    ds = pkg.decoder_stack
    torch.manual_seed(0)
    model = ds.DecoderStack(layers=2, hidden=512, heads=4, experts=16, group=64, tau=0.9, vocab=977, max_len=160).to(dev())
    model.init_random(3, std=0.05)
    model = model.to(torch.bfloat16).eval()
    for blk in model.layers:
        blk.mlp.moelayer.float()
    model.prepare_inference(0.9)
    return model


def _ids(n, seed):
    return torch.randint(0, 977, (n,), generator=torch.Generator().manual_seed(seed))


@torch.no_grad()
def test_attention_layer_against_float64(pkg, stack):
    """Two calls (chunks of 40 and 5, then 1 and 30 tokens) of one layer. The rest of the layer in
    float64 on the rounded values that the kernels meet: q, k, v and the attention's result are bf16."""
    attn = stack.layers[0].self_attn
    H, hd = attn.h, attn.hd
    kv = pkg.decoder_stack.PagedKV(1, 2, 80, H, hd, 16, dev())
    f = kv.inv_freq.cpu()
    g = torch.Generator().manual_seed(1)
    hist = [[], []]
    for new in ([40, 5], [1, 30]):
        x = torch.randn(sum(new), H * hd, generator=g).to(torch.bfloat16)
        kv.lens.add_(torch.tensor(new, dtype=torch.int32, device=dev()))
        cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=dev())
        got = attn.forward_paged(x.to(dev()), kv, 0, cu).cpu().double()
        qkv = attn.qkv(x.to(dev())).cpu().double().view(-1, 3, H, hd)
        want = torch.zeros(sum(new), H, hd, dtype=torch.float64)
        row = 0
        for s in range(2):
            for _ in range(new[s]):
                p = len(hist[s])
                c, sn = (p * f).cos(), (p * f).sin()

                def turn(t):
                    a, b = t[:, :hd // 2], t[:, hd // 2:]
                    return torch.cat([a * c - b * sn, a * sn + b * c], -1).to(torch.bfloat16).double()

                hist[s].append((turn(qkv[row, 1]), qkv[row, 2]))
                k, v = (torch.stack([h[i] for h in hist[s]]) for i in (0, 1))  # [T, H, hd]
                w = torch.softmax((turn(qkv[row, 0]) * k).sum(-1) / math.sqrt(hd), 0)
                want[row] = (w.unsqueeze(-1) * v).sum(0)
                row += 1
        want = want.to(torch.bfloat16).double().view(sum(new), -1) @ attn.o.weight.cpu().double().t()
        # roundings to bf16 of the attention's result, of P in the large tiles and of the output, each
        # 2^-8 of a value at most, in the 2-norm: three of them
        assert float((got - want).norm() / want.norm()) < 3 * 2.0 ** -8


@torch.no_grad()
def test_generate_captured_equals_eager(pkg, stack):
    ds = pkg.decoder_stack
    prompts = [_ids(n, 50 + n) for n in (3, 90, 17, 64)]
    a = ds.generate(stack, prompts, 9, chunk=32)
    b = ds.generate(stack, prompts, 9, chunk=32, capture=False)
    assert a.shape == (4, 9) and torch.equal(a, b)
    assert int(a.min()) >= 0 and int(a.max()) < 977
    assert ds.generate(stack, prompts[:1], 1).shape == (1, 1)
    with pytest.raises(ValueError):
        ds.generate(stack, [], 3)
    with pytest.raises(ValueError):
        ds.generate(stack, [_ids(0, 0)], 3)
