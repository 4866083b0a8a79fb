"""The frequencies of a decoder layer whose heads are normed: there from the start, float64 whatever the layer is converted to,
on its device, and fit for training after calls under inference_mode. Without a GPU: the operator itself is stood in for."""
import copy

import pytest
import torch

from conftest import import_pkg


@pytest.fixture()
def stack(monkeypatch):
    ds = import_pkg().decoder_stack
    seen = []

    def turned(q, k, wq, wk, pos, inv_freq, eps):
        seen.append(inv_freq)
        return q * wq, k * wk

    monkeypatch.setattr(ds.ops, "qk_norm_rotary", turned)
    return ds, seen


def layer(ds):
    return ds.Attention(256, 2, 16, qk_norm=True)


def test_trained_after_a_call_under_inference_mode(stack):
    ds, seen = stack
    attn = layer(ds)
    for mode in (torch.inference_mode, torch.enable_grad):
        with mode():
            attn.reset(1, "cpu", torch.float32)
            y = attn(torch.ones(1, 3, 256))
    y.sum().backward()
    assert attn.q_norm.weight.grad is not None
    for f in seen:  # what a backward may save
        assert not f.is_inference() and f.dtype == torch.float64 and f.shape == (64,)
        (torch.ones((), dtype=torch.float64, requires_grad=True) * f).sum().backward()


def test_there_before_the_first_call(stack):
    """A first call under a graph's capture copies nothing from the host: it takes the tensor that there was."""
    ds, seen = stack
    attn = layer(ds)
    want = ds.ops.rotary_frequencies(128)[0]
    f = attn.inv_freq
    assert torch.equal(f, want)
    attn.reset(1, "cpu", torch.float32)
    attn.forward_static(torch.ones(1, 1, 256), torch.zeros(1, dtype=torch.int64), torch.zeros(16))
    assert seen[0] is f


def test_conversions_moves_and_copies(stack):
    ds, seen = stack
    want = ds.ops.rotary_frequencies(128)[0]
    for change in (lambda a: a.to(torch.bfloat16), lambda a: a.half(), lambda a: a.float(), copy.deepcopy, lambda a: a.to("meta").to_empty(device="cpu")):
        attn = change(layer(ds))
        assert attn.inv_freq.dtype == torch.float64 and torch.equal(attn.inv_freq, want)
    assert layer(ds).to("meta").inv_freq.device.type == "meta"
    with torch.inference_mode():
        assert not layer(ds).inv_freq.is_inference() and not layer(ds).float().inv_freq.is_inference()
    with torch.device("meta"):
        attn = layer(ds)
    attn.load_state_dict({k: torch.zeros(v.shape) for k, v in attn.state_dict().items()}, assign=True)  # moved without a word
    attn.reset(1, "cpu", torch.float32)
    attn(torch.ones(1, 3, 256))
    assert torch.equal(seen[-1], want)
    assert set(attn.state_dict()) == {"qkv.weight", "o.weight", "q_norm.weight", "k_norm.weight"}
    assert ds.Attention(256, 2, 16).inv_freq is None


def test_windows_that_say_nothing(stack):
    """A window of no token would leave rows that attend nothing, NaN in the plain path; first tokens without a window were ignored there
    and refused by the paged one."""
    ds, _ = stack
    for window, sinks in ((0, 0), (-1, 0), (None, 2), (5, -1)):
        with pytest.raises(ValueError, match="window"):
            ds.Attention(256, 2, 16, window=window, sinks=sinks)
        with pytest.raises(ValueError, match="window"):
            ds.DecoderStack(layers=1, hidden=64, heads=1, experts=2, group=32, vocab=16, max_len=8, window=window, sinks=sinks)
    assert ds.Attention(256, 2, 16, window=1, sinks=0).window == 1
