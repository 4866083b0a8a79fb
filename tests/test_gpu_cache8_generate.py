"""Generation by a stack that norms its query and key heads and attends a window and the first tokens, through the paged
caches of 16 and of 8 bits, against the plain stack: each prompt alone through the contiguous cache, teacher-forced with
the tokens that were generated."""
import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

VOCAB = 977


@pytest.fixture(scope="module", params=[(None, 0), (24, 3)], ids=["all", "window"])
def stack(request, pkg):
    """tau next to 1: what an expert more or less changes is at most 1e-4 of a layer's output."""
    ds = pkg.decoder_stack
    torch.manual_seed(0)
    window, sinks = request.param
    model = ds.DecoderStack(layers=2, hidden=512, heads=4, experts=16, group=64, tau=0.9999, vocab=VOCAB, max_len=160, qk_norm=True,
                            window=window, sinks=sinks).to(dev())
    model.init_random(7, std=0.05)
    with torch.no_grad():
        for blk in model.layers:  # weights that tell the heads' channels, and q from k
            for norm in (blk.self_attn.q_norm, blk.self_attn.k_norm):
                norm.weight.copy_(1 + 0.5 * torch.randn(norm.weight.shape, generator=torch.Generator().manual_seed(3)).to(dev()))
            blk.self_attn.k_norm.weight.mul_(1.3)
    model = model.to(torch.bfloat16).eval()
    for blk in model.layers:
        blk.mlp.moelayer.float()
    model.prepare_inference(0.9999)
    return model


@torch.no_grad()
def plain_logits(model, ids):
    return model(ids.to(dev())[None]).float().cpu().view(VOCAB)


@torch.no_grad()
@pytest.mark.parametrize("bits,chunk,page", [(16, 32, 16), (8, 32, 16), (8, 512, 64), (8, 7, 16)])
def test_generated_tokens_are_the_plain_stacks(pkg, stack, bits, chunk, page):
    """A generated token's plain logit is the highest, up to 0.25 of the logits' rms: some 30 roundings to bf16 on either way, each
    2^-8 of a value (in the 2-norm sqrt(60) 2^-8 = 0.03), a factor of 8 for single logits. With 8 bits the keys and values
    are off by up to 2^-4 each, 2^-5.8 (0.018) as the 2-norm of a rounding that is spread evenly, in two layers: four
    of them, 0.036, beside the 0.03; the same factor of 8 gives 0.375 for 0.047 together."""
    lengths, steps = (3, 32, 33, 96, 1), 6
    limit = 0.25 if bits == 16 else 0.375
    prompts = [torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(n)) for n in lengths]
    got = pkg.decoder_stack.generate(stack, prompts, steps, chunk=chunk, page_size=page, bits=bits).cpu()
    assert got.shape == (len(lengths), steps)
    wrong = 0
    for s, p in enumerate(prompts):
        for blk in stack.layers:
            blk.self_attn.reset(1, dev(), torch.bfloat16)
        logits = plain_logits(stack, p)
        for i in range(steps):
            short = float((logits.max() - logits[got[s, i]]) / logits.pow(2).mean().sqrt())
            assert short <= limit, (lengths[s], i, short)
            other = got[(s + 1) % len(lengths), i]
            wrong += float((logits.max() - logits[other]) / logits.pow(2).mean().sqrt()) > limit
            logits = plain_logits(stack, got[s, i:i + 1])
    assert wrong > 0.8 * len(lengths) * steps  # the bound tells the sequences apart


@torch.no_grad()
def test_captured_equals_eager_and_static_step(pkg, stack):
    ds = pkg.decoder_stack
    prompts = [torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(n)) for n in (3, 90, 17, 64)]
    for bits in (8, 16):
        a = ds.generate(stack, prompts, 9, chunk=32, bits=bits)
        assert torch.equal(a, ds.generate(stack, prompts, 9, chunk=32, capture=False, bits=bits))
    with pytest.raises(ValueError, match="8 or 16"):
        ds.generate(stack, prompts, 2, bits=4)
    # one token at a device position over the whole contiguous cache: as the eager step
    p, nxt = prompts[1].to(dev()), prompts[0][:1].to(dev())
    for blk in stack.layers:
        blk.self_attn.reset(1, dev(), torch.bfloat16)
    stack(p[None])
    kept = [(blk.self_attn.kt_cache.clone(), blk.self_attn.v_cache.clone()) for blk in stack.layers]
    eager = stack(nxt[None]).float().view(VOCAB)
    for blk, (k, v) in zip(stack.layers, kept):
        blk.self_attn.kt_cache, blk.self_attn.v_cache = k, v
    tok = nxt.view(1, 1).clone()
    pos = torch.tensor([90], device=dev())
    stack.step_static(tok, pos)
    assert int(pos) == 91 and float((eager.max() - eager[int(tok)]) / eager.pow(2).mean().sqrt()) <= 0.25
    first = int(tok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.step_static(tok, pos)
    for _ in range(3):
        pos.fill_(90)
        tok.copy_(nxt.view(1, 1))
        graph.replay()
        assert int(tok) == first


@torch.no_grad()
def test_read_of_a_layer(pkg):
    """The cache of 8 bits beside the one of 16 after the same calls: its values within their rounding."""
    ds, ops = pkg.decoder_stack, pkg.ops
    kvs = [ds.PagedKV(1, 3, 80, 2, 64, 16, dev(), bits=b) for b in (16, 8)]
    g = torch.Generator().manual_seed(1)
    for new in ([40, 5, 0], [1, 30, 17], [1, 1, 1]):
        cu = torch.tensor([sum(new[:i]) for i in range(4)], dtype=torch.int32, device=dev())
        x = torch.randn(2, sum(new), 2, 64, generator=g).to(torch.bfloat16).to(dev())
        for kv in kvs:
            kv.lens.add_(torch.tensor(new, dtype=torch.int32, device=dev()))
            ops.kv_append(x[0], x[1], *kv.pages[0], kv.table, kv.lens, cu, inv_freq=kv.inv_freq, scales=kv.scales[0])
    (k, v, at), (k8, v8, at8) = (kv.read(0) for kv in kvs)
    assert at.tolist() == at8.tolist() == [0, 42, 78, 96] and k.shape == k8.shape == (96, 2, 64)
    for a, b in ((k, k8), (v, v8)):
        # half a step of e4m3, twice where a block's scale grew, and half a step of bf16 of the other side's; steps of 2^-9 of scales
        # that are at most 2^-6 (values below 7)
        a, b = a.float(), b.float()
        assert bool(((a - b).abs() <= (2 * 2.0 ** -4 + 2.0 ** -8) * (1 + 2.0 ** -4) * a.abs() + 2 * 2.0 ** -16).all())
