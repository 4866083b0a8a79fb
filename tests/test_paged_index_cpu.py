"""CPU checks of the paged-cache kernels' work items: the item -> (sequence, rows) maps of
csrc/paged.h, csrc/rotary.hip and csrc/attention.hip restated in Python, over ragged batches with
empty sequences, padding rows and lengths shorter than the new tokens. Every row has exactly one
item, every position group one page, the ranges of a tile cover its tokens once, and offsets out of
order stay inside the arrays. Also the refusals of the three entry points, before any launch."""
import ctypes
import random

import pytest

from conftest import import_pkg


def start(cu, s, n_rows):
    if s <= 0:
        return 0
    if s > len(cu) - 1:
        return n_rows
    return min(max(cu[s], 0), n_rows)


def seq_of(cu, n_rows, t, first):
    """paged_find: blocks of 256 sequences, stopping at the first block that is not all below t."""
    B, n = len(cu) - 1, 0
    for s0 in range(0, B + 1, 256):
        hits = [s <= B and first(start(cu, s, n_rows), s) <= t for s in range(s0, s0 + 256)]
        n += sum(hits)
        if not all(hits):
            break
    return max(n - 1, 0)


def batches():
    rng = random.Random(7)
    for B in (0, 1, 2, 3, 64, 130, 255, 256, 300):
        for kind in ("one", "ragged", "empty"):
            new = [1 if kind == "one" else rng.choice([0, 1, 2, 17, 40]) if kind == "ragged" else 0 for _ in range(B)]
            for pad in (0, 1, 37):
                cu = [sum(new[:i]) for i in range(B + 1)]
                if cu[-1] + pad:
                    yield cu, cu[-1] + pad, [max(0, n + rng.choice([-3, 0, 1, 15, 100])) for n in new]


@pytest.mark.parametrize("R,group", [(16, 1), (16, 5), (32, 3), (128, 1), (128, 8)])
def test_attention_tiles_cover_every_row_once(R, group):
    for cu, N, kv in batches():
        B = len(cu) - 1
        first = lambda c, s: c * group // R + s  # noqa: E731
        seen = set()
        for t in range(N * group // R + B + 1):
            s = seq_of(cu, N, t, first)
            c0 = start(cu, s, N)
            length = max(start(cu, s + 1, N) - c0, 0)
            r0 = (t - first(c0, s)) * R
            nr = max(0, min(R, length * group - r0))
            for r in range(nr):
                i, h = divmod(min(r0, length * group) + r, group)
                assert 0 <= c0 + i < N and (c0 + i, h) not in seen
                seen.add((c0 + i, h))
        assert len(seen) == N * group


def test_append_groups_cover_every_token_once():
    for cu, N, kv in batches():
        B = len(cu) - 1
        seen = set()
        for t in range((N >> 4) + 2 * (B + 1)):
            first = lambda c, s: (c >> 4) + 2 * s  # noqa: E731
            s = seq_of(cu, N, t, first)
            c0 = start(cu, s, N)
            length = max(start(cu, s + 1, N) - c0, 0)
            p = 0 if s == B else kv[s] - length
            p0 = (p & ~15) + 16 * (t - first(c0, s))
            lo, hi = max(0, p - p0), min(16, p + length - p0)
            for i in range(lo, hi):
                row = c0 + (p0 - p) + i
                assert c0 <= row < c0 + length and row not in seen
                assert row - c0 + p == p0 + i  # the row's position
                seen.add(row)
        assert len(seen) == N


def test_append_value_items_cover_every_token_once():
    """Items of 64 positions: their four groups to the four waves, or the one group that has tokens to all."""
    for cu, N, kv in batches():
        B = len(cu) - 1
        seen = {}
        for t in range((N >> 6) + 2 * (B + 1)):
            first = lambda c, s: (c >> 6) + 2 * s  # noqa: E731
            s = seq_of(cu, N, t, first)
            c0 = start(cu, s, N)
            length = max(start(cu, s + 1, N) - c0, 0)
            p = 0 if s == B else kv[s] - length
            at = ((p >> 6) + t - first(c0, s)) << 6
            begin = max(at, p & ~15)
            alone = min(at + 64, p + length) - begin <= 16
            for p0 in [begin] if alone else range(at, at + 64, 16):
                for i in range(max(0, p - p0), min(16, p + length - p0)):
                    row = c0 + (p0 - p) + i
                    assert c0 <= row < c0 + length and row not in seen
                    seen[row] = p0 & 15
        assert len(seen) == N and not any(seen.values())  # groups start at multiples of 16: in one page


def test_offsets_out_of_order_stay_inside():
    rng = random.Random(3)
    for _ in range(200):
        B, N, group, R = rng.randint(1, 70), rng.randint(1, 90), rng.choice([1, 4]), 16
        cu = [rng.randint(-50, 150) for _ in range(B + 1)]
        first = lambda c, s: c * group // R + s  # noqa: E731
        for t in range(N * group // R + B + 1):
            s = seq_of(cu, N, t, first)
            c0 = start(cu, s, N)
            length = max(start(cu, s + 1, N) - c0, 0)
            r0 = (t - first(c0, s)) * R
            nr = 0 if r0 < 0 else max(0, min(R, length * group - r0))
            assert 0 <= s <= B
            if nr > 0:
                assert 0 <= c0 + r0 // group and c0 + (r0 + nr - 1) // group < N


@pytest.mark.parametrize("splits,least", [(1, 128), (7, 128), (64, 128), (5, 512)])
def test_ranges_cover_the_tokens(splits, least):
    for nt in [1, 2, 31, 127, 128, 129, 1152, 4095, 4097, 30011, 1 << 20]:
        cut = max(1, min(splits, -(-nt // least)))
        per = (-(-nt // cut) + 127) // 128 * 128
        ns = -(-nt // per)
        at = 0
        for i in range(ns):
            lo = min(i * per, nt)
            hi = min(nt, lo + per)
            assert lo == at and hi > lo and lo % 128 == 0
            at = hi
        assert at == nt and 1 <= ns <= splits


# ------------------------------------------------------------------ refusals
def _lib():
    return import_pkg()._lib.lib()


P = ctypes.c_void_p(1 << 20)  # an aligned address that nothing reads: every call here is refused
S3 = (ctypes.c_int64 * 3)(1 << 20, 1 << 14, 128)
S2 = (ctypes.c_int64 * 2)(1 << 14, 128)


def _rotary(**kw):
    a = dict(x=P, dtype=0, xs=S3, pos=P, pos64=1, ps=S2, B=1, L=4, heads=2, D=128, f=P, rd=128, layout=0, y=P)
    a.update(kw)
    return _lib().pp_rotary(a["x"], a["dtype"], a["xs"], a["pos"], a["pos64"], a["ps"], a["B"], a["L"], a["heads"],
                            a["D"], a["f"], a["rd"], a["layout"], 1.0, 0, a["y"], a["xs"], None)


@pytest.mark.parametrize("kw,code", [(dict(dtype=2), 1), (dict(layout=2), 1), (dict(D=0), 3), (dict(D=1026), 3),
                                     (dict(rd=0), 1), (dict(rd=3), 1), (dict(rd=130), 1), (dict(L=-1), 3),
                                     (dict(B=1 << 20, L=1 << 20), 3), (dict(x=None), 1), (dict(f=None), 1),
                                     (dict(pos=None), 1), (dict(L=0, x=None), 0), (dict(heads=0, x=None), 0)])
def test_rotary_refusals(kw, code):
    assert _rotary(**kw) == code
    assert code == 0 or "pp_rotary" in _lib().pp_last_error().decode()


def _append(**kw):
    a = dict(q=P, qs=S2, k=P, ks=S2, v=P, vs=S2, dtype=1, n=4, seqs=2, cu=P, kv=P, table=P, maxp=8, pages=9, page=16,
             Hq=4, Hkv=2, D=128, f=P, rd=128, layout=0, kp=P, vp=P, out=P)
    a.update(kw)
    return _lib().pp_kv_append(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["dtype"], a["n"], a["seqs"], a["cu"],
                               a["kv"], a["table"], a["maxp"], a["pages"], a["page"], a["Hq"], a["Hkv"], a["D"], a["f"],
                               a["rd"], a["layout"], 1.0, a["kp"], a["vp"], a["out"], 0, None)


def _attend(**kw):
    a = dict(q=P, qs=S2, n=4, seqs=2, cu=P, kv=P, table=P, maxp=64, kp=P, vp=P, pages=9, page=16, Hq=4, Hkv=2, D=128,
             out=P, ws=P, bytes=1 << 30)
    a.update(kw)
    return _lib().pp_paged_attention(a["q"], a["qs"], a["n"], a["seqs"], a["cu"], a["kv"], a["table"], a["maxp"], a["kp"],
                                     a["vp"], a["pages"], a["page"], a["Hq"], a["Hkv"], a["D"], 0.1, a["out"], 0, a["ws"],
                                     a["bytes"], None)


BOTH = [(dict(D=96), 3), (dict(D=256), 3), (dict(page=8), 3), (dict(page=24), 3), (dict(page=8192), 3),
        (dict(Hq=3), 1), (dict(Hkv=0), 1), (dict(maxp=0), 1), (dict(pages=0), 1), (dict(n=-1), 3),
        (dict(n=1 << 30), 3), (dict(maxp=1 << 27), 3), (dict(seqs=-1), 1), (dict(cu=None), 1), (dict(kv=None), 1),
        (dict(table=None), 1), (dict(kp=None), 1), (dict(vp=ctypes.c_void_p((1 << 20) + 8)), 1)]


@pytest.mark.parametrize("kw,code", BOTH + [(dict(dtype=3), 1), (dict(layout=5), 1), (dict(rd=24), 3), (dict(rd=144), 3),
                                            (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1),
                                            (dict(ks=(ctypes.c_int64 * 2)(1 << 14, 130)), 1),
                                            (dict(q=ctypes.c_void_p((1 << 20) + 2)), 1), (dict(n=0, cu=None), 0)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code
    assert code == 0 or "pp_kv_append" in _lib().pp_last_error().decode()


@pytest.mark.parametrize("kw,code", BOTH + [(dict(Hq=0), 1), (dict(q=None), 1), (dict(out=None), 1),
                                            (dict(out=ctypes.c_void_p((1 << 20) + 8)), 1),
                                            (dict(qs=(ctypes.c_int64 * 2)(1 << 14, 132)), 1), (dict(bytes=16), 1),
                                            (dict(ws=None), 1), (dict(n=0, cu=None), 0)])
def test_attention_refusals(kw, code):
    assert _attend(**kw) == code
    assert code == 0 or "pp_paged_attention" in _lib().pp_last_error().decode()


def test_frequencies():
    import torch
    ops = import_pkg().ops
    f, m = ops.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0 and f[0] == 1.0
    assert abs(float(f[-1]) - 10000.0 ** (-62 / 64)) < 1e-18
    g, _ = ops.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(g, f / 4)
    g, _ = ops.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert g[0] == 1.0 and abs(float(g[-1] / f[-1]) - 1 / 8) < 1e-12
    g, m = ops.rotary_frequencies(64, scaling="yarn", factor=8.0)
    assert g[0] == f[0] and abs(float(g[-1] / f[-1]) - 1 / 8) < 1e-12 and abs(m - 1.2079441541679836) < 1e-12
    assert bool((g[1:] < g[:-1]).all())
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, factor=0.0),
                dict(dim=8, scaling="yarn", turns=(32.0, 1.0))):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


def test_wrappers_refuse_cpu_tensors():
    import torch
    ops = import_pkg().ops
    f, _ = ops.rotary_frequencies(64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.rotary(torch.zeros(2, 3, 64), torch.zeros(2, dtype=torch.int64), f)
    kp, vp = ops.paged_cache(2, 16, 1, 64)
    i = torch.zeros(1, dtype=torch.int32)
    args = (kp, vp, torch.zeros(1, 1, dtype=torch.int32), i, torch.tensor([0, 1], dtype=torch.int32))
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.kv_append(x, x, *args)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_attention(x, *args)


def test_shapes_without_a_gpu():
    """Fake tensors: the ops' results have their shapes and types, the in-place ones return nothing."""
    import torch
    t = import_pkg()._lib.torch_ops()
    m = dict(device="meta")
    f = torch.empty(32, dtype=torch.float64, **m)
    x = torch.empty(3, 5, 4, 64, dtype=torch.bfloat16, **m).transpose(1, 2)
    y = t.rotary(x.transpose(1, 2), torch.empty(3, 5, dtype=torch.int64, **m), f)
    assert y.shape == (3, 5, 4, 64) and y.dtype == torch.bfloat16
    cache = (torch.empty(9, 2, 16, 64, dtype=torch.bfloat16, **m), torch.empty(9, 2, 64, 16, dtype=torch.bfloat16, **m),
             torch.empty(2, 3, dtype=torch.int32, **m), torch.empty(2, dtype=torch.int32, **m),
             torch.empty(3, dtype=torch.int32, **m))
    kv, q = torch.empty(5, 2, 64, **m), torch.empty(5, 4, 64, **m)
    assert t.kv_append(kv, kv, *cache, f) is None
    r = t.kv_append_q(q, kv, kv, *cache, f)
    assert r.shape == q.shape and r.dtype == torch.bfloat16
    assert t.kv_append_q_into(q, r, kv, kv, *cache, f) is None
    assert t.paged_attention(r, *cache, 0.1).shape == r.shape
    assert t.paged_attention_into(r, *cache, 0.1, r) is None


def test_rotary_strides_without_a_gpu():
    """A fake result has the strides of the real one: the input's where its channels are next to each other,
    contiguous otherwise."""
    import torch
    t = import_pkg()._lib.torch_ops()
    f, pos = torch.empty(32, dtype=torch.float64, device="meta"), torch.empty(3, 5, dtype=torch.int64, device="meta")
    for make, want in ((lambda z: z(3, 4, 5, 64).transpose(1, 2), (1280, 64, 320, 1)),
                       (lambda z: z(3, 5, 64, 4).transpose(2, 3), (1280, 256, 64, 1)),
                       (lambda z: z(3, 5, 9, 64)[:, :, :4], (1280, 256, 64, 1))):
        assert t.rotary(make(lambda *n: torch.empty(*n, device="meta")), pos, f).stride() == want


def test_generate_refusals():
    import torch
    ds = import_pkg().decoder_stack
    one = torch.ones(3, dtype=torch.int64)
    for kw in (dict(prompts=[one], steps=0), dict(prompts=[], steps=2), dict(prompts=[one[:0]], steps=2),
               dict(prompts=[one], steps=2, chunk=0), dict(prompts=[one], steps=2, chunk=-4),
               dict(prompts=[one.view(1, 3)], steps=2)):
        with pytest.raises(ValueError, match="generate"):
            ds.generate(None, **kw)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 3.0e38])
def test_scales_beyond_float32_are_refused(scale):
    assert _lib().pp_paged_attention(P, S2, 4, 2, P, P, P, 64, P, P, 9, 16, 4, 2, 128, scale, P, 0, P, 1 << 30, None) == 1


def test_launches_beyond_the_grid_are_refused():
    rc = _lib().pp_paged_attention(P, S2, 1 << 20, 1 << 20, P, P, P, 600, P, P, 9, 16, 32, 2, 64, 0.1, P, 0, P, 1 << 62, None)
    assert rc == 3 and "workgroups" in _lib().pp_last_error().decode()


@pytest.mark.parametrize("seqs", [0, 1, 5])
@pytest.mark.parametrize("n,maxp", [(1, 1), (4096, 8), (1 << 20, 1 << 16)])
def test_workspace_of_any_batch(n, seqs, maxp):
    """No sequence at all among them; room for at most 64 ranges of a row."""
    b = _lib().pp_paged_attention_workspace_bytes(n, seqs, maxp, 16, 12, 4, 128)
    assert 0 <= b <= n * 12 * (64 * 130 * 4 + 4)
