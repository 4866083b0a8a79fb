"""Generation through the paged cache against the plain decoder stack: each prompt alone through the contiguous
cache, teacher-forced with the tokens that were generated."""
import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

VOCAB = 977


@pytest.fixture(scope="module")
def stack(pkg):
    """tau next to 1: what an expert more or less changes is at most 1e-4 of a layer's output, so that the two
    ways differ by their roundings alone."""
    ds = pkg.decoder_stack
    torch.manual_seed(0)
    model = ds.DecoderStack(layers=2, hidden=512, heads=4, experts=16, group=64, tau=0.9999, vocab=VOCAB, max_len=160).to(dev())
    model.init_random(7, std=0.05)
    model = model.to(torch.bfloat16).eval()
    for blk in model.layers:
        blk.mlp.moelayer.float()
    model.prepare_inference(0.9999)
    return model


@torch.no_grad()
def plain_logits(model, ids):
    """Logits of the next token [VOCAB] through the contiguous cache, which goes on."""
    return model(ids.to(dev())[None]).float().cpu().view(VOCAB)


@torch.no_grad()
@pytest.mark.parametrize("chunk,page", [(32, 16), (512, 64), (7, 16)])
def test_generated_tokens_are_the_plain_stacks(pkg, stack, chunk, page):
    """Prompts shorter than a chunk, as long, longer by one and several chunks long. A generated token's plain
    logit is the highest, up to 0.25 of the logits' rms: 30 roundings to bf16 on either way through two layers, each
    2^-8 of a value and independent (in the 2-norm sqrt(60) 2^-8 = 0.03), a factor of 8 for single logits. The
    token of another row or position falls short by several times that."""
    lengths, steps = (3, 32, 33, 96, 1), 6
    prompts = [torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(n)) for n in lengths]
    got = pkg.decoder_stack.generate(stack, prompts, steps, chunk=chunk, page_size=page).cpu()
    assert got.shape == (len(lengths), steps)
    wrong = 0
    for s, p in enumerate(prompts):
        for blk in stack.layers:
            blk.self_attn.reset(1, dev(), torch.bfloat16)
        logits = plain_logits(stack, p)
        for i in range(steps):
            short = float((logits.max() - logits[got[s, i]]) / logits.pow(2).mean().sqrt())
            assert short <= 0.25, (lengths[s], i, short)
            other = got[(s + 1) % len(lengths), i]
            wrong += float((logits.max() - logits[other]) / logits.pow(2).mean().sqrt()) > 0.25
            logits = plain_logits(stack, got[s, i:i + 1])
    assert wrong > 0.8 * len(lengths) * steps  # the bound tells the sequences apart
