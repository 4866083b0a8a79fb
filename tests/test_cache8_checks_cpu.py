"""Without a GPU: refusals of the entry points of the normed rotation, the 8-bit cache and the windowed attention, before any
launch; the shapes and types that fake calls check; gradients, tangents and versions; and, restated in Python, the windowed
attention's walk over a sequence and the bytes of scales."""
import ctypes
import random

import pytest

from conftest import import_pkg
from test_paged_checks_cpu import _fake
from test_paged_index_cpu import BOTH, P, S2, S3, _lib

ODD = ctypes.c_void_p((1 << 20) + 8)


# ------------------------------------------------------------------ entry points
def _norm(**kw):
    a = dict(q=P, qs=S3, k=P, ks=S3, dtype=1, qw=P, kw=P, wd=0, pos=P, ps=S2, B=1, L=4, Hq=4, Hk=2, D=128, f=P, rd=128, layout=0, eps=1e-6, qo=P, ko=P)
    a.update(kw)
    return _lib().pp_qk_norm_rotary(a["q"], a["qs"], a["k"], a["ks"], a["dtype"], a["qw"], a["kw"], a["wd"], a["pos"], 1, a["ps"], a["B"], a["L"],
                                    a["Hq"], a["Hk"], a["D"], a["f"], a["rd"], a["layout"], 1.0, a["eps"], a["qo"], a["ko"], None)


def _norm_bwd(**kw):
    a = dict(q=P, qs=S3, k=P, ks=S3, dtype=1, qw=P, kw=P, wd=0, pos=P, ps=S2, B=1, L=4, Hq=4, Hk=2, D=128, f=P, rd=128, layout=0, eps=1e-6, qo=P, ko=P,
             dq=P, dk=P, wq=P, wk=P, ws=P, bytes=1 << 30)
    a.update(kw)
    return _lib().pp_qk_norm_rotary_bwd(a["dq"], a["qs"], a["dk"], a["ks"], a["q"], a["qs"], a["k"], a["ks"], a["dtype"], a["qw"], a["kw"], a["wd"],
                                        a["pos"], 1, a["ps"], a["B"], a["L"], a["Hq"], a["Hk"], a["D"], a["f"], a["rd"], a["layout"], 1.0, a["eps"],
                                        a["qo"], a["ko"], a["wq"], a["wk"], a["ws"], a["bytes"], None)


NORM = [(dict(dtype=2), 1), (dict(layout=2), 1), (dict(D=1), 3), (dict(D=258), 3), (dict(rd=0), 1), (dict(rd=3), 1), (dict(rd=130), 1),
        (dict(L=-1), 3), (dict(B=1 << 20, L=1 << 20), 3), (dict(Hq=1 << 17), 3), (dict(Hk=-1), 3), (dict(wd=1, dtype=0), 1), (dict(wd=3), 1),
        (dict(eps=-1.0), 1), (dict(eps=float("inf")), 1), (dict(eps=float("nan")), 1), (dict(q=None), 1), (dict(k=None), 1), (dict(qw=None), 1),
        (dict(kw=None), 1), (dict(f=None), 1), (dict(pos=None), 1), (dict(qo=None), 1), (dict(ko=None), 1)]


@pytest.mark.parametrize("kw,code", NORM + [(dict(L=0, q=None), 0), (dict(Hq=0, Hk=0, q=None), 0)])
def test_norm_refusals(kw, code):
    assert _norm(**kw) == code
    assert code == 0 or "pp_qk_norm_rotary" in _lib().pp_last_error().decode()


@pytest.mark.parametrize("kw,code", NORM + [(dict(dq=None), 1), (dict(dk=None), 1), (dict(ws=None), 1), (dict(bytes=64), 1), (dict(ws=ODD), 1),
                                            (dict(L=0, q=None, wq=None, wk=None), 0)])
def test_norm_gradient_refusals(kw, code):
    assert _norm_bwd(**kw) == code
    assert code == 0 or "pp_qk_norm_rotary_bwd" in _lib().pp_last_error().decode()


def test_norm_workspace():
    b = _lib().pp_qk_norm_rotary_workspace_bytes
    assert b(1, 1, 1, 4, 2, 128, 128) >= 2 * 128 * 4 and b(1, 1, 1, 4, 2, 512, 128) == 0 and b(1, 1, 0, 4, 2, 128, 128) == 0
    assert b(1, 8, 1 << 20, 12, 12, 128, 128) <= 16 << 20  # bounded, however many tokens


def _append(**kw):
    a = dict(q=P, qs=S2, k=P, ks=S2, v=P, vs=S2, dtype=1, n=4, seqs=2, cu=P, kv=P, table=P, maxp=8, pages=9, page=16, Hq=4, Hkv=2, D=128, f=P, rd=128,
             layout=0, qw=P, kw=P, wd=0, eps=1e-6, kp=P, vp=P, ksc=P, vsc=P, out=P)
    a.update(kw)
    return _lib().pp_kv_append_with(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["dtype"], a["n"], a["seqs"], a["cu"], a["kv"], a["table"],
                                    a["maxp"], a["pages"], a["page"], a["Hq"], a["Hkv"], a["D"], a["f"], a["rd"], a["layout"], 1.0, a["qw"], a["kw"],
                                    a["wd"], a["eps"], a["kp"], a["vp"], a["ksc"], a["vsc"], a["out"], 0, None)


@pytest.mark.parametrize("kw,code", BOTH + [(dict(dtype=3), 1), (dict(layout=5), 1), (dict(rd=24), 3), (dict(rd=144), 3), (dict(k=None), 1), (dict(v=None), 1),
                                            (dict(out=None), 1), (dict(ksc=None), 1), (dict(vsc=None), 1), (dict(qw=None), 1), (dict(kw=None), 1),
                                            (dict(q=None, qw=None, n=0), 0), (dict(wd=2), 1), (dict(qw=ODD), 1), (dict(kw=ODD), 1), (dict(wd=1, dtype=0), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
                                            (dict(vs=(ctypes.c_int64 * 2)(1 << 14, 130)), 1), (dict(n=0, cu=None), 0), (dict(seqs=1 << 20, Hkv=32, Hq=32), 3)])
def test_append_refusals(kw, code):
    assert _append(**kw) == code
    assert code == 0 or "pp_kv_append_with" in _lib().pp_last_error().decode()


def _read(**kw):
    a = dict(kp=P, vp=P, ksc=P, vsc=P, n=4, seqs=2, cu=P, kv=P, table=P, maxp=8, pages=9, page=16, Hkv=2, D=128, ko=P, vo=P)
    a.update(kw)
    return _lib().pp_kv_read(a["kp"], a["vp"], a["ksc"], a["vsc"], a["n"], a["seqs"], a["cu"], a["kv"], a["table"], a["maxp"], a["pages"], a["page"],
                             a["Hkv"], a["D"], a["ko"], a["vo"], 0, None)


@pytest.mark.parametrize("kw,code", [(k, c) for k, c in BOTH if "Hq" not in k] + [
    (dict(ksc=None), 1), (dict(vsc=None), 1), (dict(ko=None), 1), (dict(vo=ODD), 1), (dict(n=0, cu=None), 0), (dict(n=(1 << 31) - 1, Hkv=1, D=64), 3)])
def test_read_refusals(kw, code):
    assert _read(**kw) == code
    assert code == 0 or "pp_kv_read" in _lib().pp_last_error().decode()


def _attend(**kw):
    a = dict(q=P, qs=S2, n=4, seqs=2, cu=P, kv=P, table=P, maxp=64, kp=P, vp=P, ksc=P, vsc=P, pages=9, page=16, Hq=4, Hkv=2, D=128, scale=0.1, window=5,
             sinks=2, out=P, ws=P, bytes=1 << 30)
    a.update(kw)
    return _lib().pp_paged_attention_with(a["q"], a["qs"], a["n"], a["seqs"], a["cu"], a["kv"], a["table"], a["maxp"], a["kp"], a["vp"], a["ksc"], a["vsc"],
                                          a["pages"], a["page"], a["Hq"], a["Hkv"], a["D"], a["scale"], a["window"], a["sinks"], a["out"], 0, a["ws"],
                                          a["bytes"], None)


@pytest.mark.parametrize("kw,code", BOTH + [(dict(Hq=0), 1), (dict(q=None), 1), (dict(out=None), 1), (dict(window=-1), 1), (dict(sinks=-1), 1),
                                            (dict(ksc=None), 1), (dict(vsc=None), 1), (dict(scale=float("inf")), 1), (dict(window=0, bytes=16), 1),
                                            (dict(qs=(ctypes.c_int64 * 2)(1 << 14, 132)), 1), (dict(n=0, cu=None), 0)])
def test_attention_refusals(kw, code):
    assert _attend(**kw) == code
    assert code == 0 or "pp_paged_attention_with" in _lib().pp_last_error().decode()


def test_workspace_of_windows():
    """No more than without one, and none that goes by the table's width."""
    b = _lib().pp_paged_attention_with_workspace_bytes
    for n, seqs, hq, hkv in ((1, 1, 12, 12), (64, 64, 12, 12), (4096, 1, 12, 12), (300, 9, 24, 4)):
        for eight in (0, 1):
            sizes = [b(n, seqs, maxp, 16, hq, hkv, 128, eight, 1000, 4) for maxp in (100, 1 << 10, 1 << 16)]
            assert sizes[1] == sizes[2] and all(x <= n * hq * (64 * 130 * 4 + 4) for x in sizes)
            assert b(n, seqs, 1 << 10, 16, hq, hkv, 128, eight, -1, 4) == 0
            for most in (1 << 62, (1 << 63) - 1):  # as without a window, or less
                assert b(n, seqs, 1 << 10, 16, hq, hkv, 128, eight, most, most) <= n * hq * (64 * 130 * 4 + 4)


# ------------------------------------------------------------------ the windowed walk, restated
@pytest.mark.parametrize("step", [32, 64])
@pytest.mark.parametrize("rows,group", [(16, 1), (16, 5), (128, 1), (128, 8)])
def test_walk_over_a_window(step, rows, group):
    """Every token that a row of the tile attends is met once, in a step on one side of the gap, from a group of 16 that starts at a
    multiple of 16; what is met and not attended is masked by the row's own limits."""
    rng = random.Random(step + rows + group)
    for _ in range(300):
        window, sinks = rng.choice([1, 5, 16, 17, 63, 64, 100, 500]), rng.choice([0, 0, 1, 4, 16, 33, 64, 200])
        n = rng.randint(1, 40)
        length, capacity = rng.randint(0, 1200), rng.choice([64, 320, 2048])
        r0 = rows * rng.randint(0, (n * group - 1) // rows)
        nr = min(rows, n * group - r0)
        p0 = length - n
        nt = max(0, min(p0 + (r0 + max(nr, 1) - 1) // group + 1, capacity))
        start = max(0, min(p0 + r0 // group - window + 1, nt))
        keep = (min(sinks, start) + step - 1) // step * step
        gap = max(0, (start & ~15) - keep)
        at = lambda t: t if t < keep else t + gap  # noqa: E731
        assert gap % 16 == 0 and keep % step == 0 and nt - gap >= 0
        met = []
        for t in range(0, nt - gap, step):
            assert at(t) % 16 == 0 and at(t + step - 1) == at(t) + step - 1
            met += [at(t) + i for i in range(step) if t + i < nt - gap]
        assert len(met) == len(set(met)) and all(0 <= t < nt for t in met)
        for r in range(nr):
            p = p0 + (r0 + r) // group
            attended = {t for t in range(0, min(p + 1, capacity)) if t > p - window or t < sinks}
            limit, first = min(p, capacity - 1), max(p - window + 1, 0)
            assert attended == {t for t in met if t <= limit and (t >= first or t < sinks)}


@pytest.mark.parametrize("group", [1, 3, 8])
def test_tiles_in_the_order_of_their_work(group):
    """Every tile number once, whatever the lengths; where they differ, the sequences with rows by their lengths, each one's last
    tiles first, the rows of none last; offsets out of order give numbers within the tiles or none."""
    rng = random.Random(group)
    for case in range(300):
        n = rng.choice([2, 3, 9, 40, 63, 64])
        new = [rng.choice([0, 1, 1, 5, 128, 300]) for _ in range(n)]
        lens = [rng.choice([0, 7, 500, 500, 4000, 1 << 26]) if case % 3 else 900 + rng.randint(0, 100) for _ in range(n)]
        cu = [sum(new[:i]) for i in range(n + 1)]
        rows = cu[-1] + rng.choice([0, 3, 500])
        if case % 4 == 3:
            cu = [rng.randint(-5, rows + 5) for _ in cu]
        tiles = rows * group // 128 + n + 1
        row = lambda s: 0 if s == 0 else min(max(cu[s], 0), rows)  # noqa: E731
        first = lambda s: row(s) * group // 128 + s  # noqa: E731
        lo, tail = [first(s) for s in range(n)], first(n)
        count = [max(first(s + 1) - lo[s], 0) for s in range(n)]
        key = [min(max(lens[s], 1), (1 << 25) - 1) << 6 | (63 - s) if row(s + 1) > row(s) else 0 for s in range(n)]
        before = [sum(count[j] for j in range(n) if key[j] > key[s] or (key[j] == key[s] and j < s)) for s in range(n)]
        some = [k >> 6 for k in key if k]
        by_length = bool(some) and max(some) - min(some) > max(some) // 4
        got = []
        for u in range(tiles):
            t = tiles - 1 - u
            if by_length:
                mine = [s for s in range(n) if before[s] <= u < before[s] + count[s]]
                t = lo[mine[0]] + count[mine[0]] - 1 - (u - before[mine[0]]) if mine else tiles - 1 - (u - tail)
            else:
                mine = [s for s in range(n) if lo[s] <= t < lo[s] + count[s]]
            if not 0 <= t < tiles:
                assert case % 4 == 3
                continue
            if case % 4 != 3:
                assert len(mine) <= 1 and bool(mine) == (t < tail)
                assert not mine or mine[0] == max(s for s in range(n) if lo[s] <= t)
            got.append((t, mine[0] if mine else n))
        if case % 4 == 3:
            continue
        assert sorted(t for t, _ in got) == list(range(tiles))
        if by_length:
            lengths = [key[s] >> 6 if s < n else 0 for _, s in got]
            assert lengths == sorted(lengths, reverse=True)


@pytest.mark.parametrize("group", [1, 3, 8, 16, 40])
def test_tiles_with_rows_come_first(group):
    """16-row tiles of up to 64 sequences: every row of a sequence, and of none, once; no tile without rows before one of a
    sequence with some; offsets out of order stay inside."""
    rng = random.Random(group)
    for case in range(300):
        n = rng.choice([1, 2, 9, 33, 63, 64])
        new = [rng.choice([0, 1, 1, 1, 2, 17]) for _ in range(n)]
        cu = [sum(new[:i]) for i in range(n + 1)]
        N = cu[-1] + rng.choice([0, 1, 40])
        if N == 0:
            continue
        if case % 4 == 3:
            cu = [rng.randint(-5, N + 5) for _ in cu]
        row = lambda s: 0 if s == 0 else min(max(cu[s], 0), N)  # noqa: E731
        first = lambda c, s: c * group // 16 + s  # noqa: E731
        rows = [max(row(s + 1) - row(s), 0) for s in range(n)]
        tiles = [(r * group + 15) // 16 for r in rows]
        upto = [sum(tiles[:s + 1]) for s in range(n)]
        seen, empty = [], False
        for u in range(N * group // 16 + n + 1):
            mine = [s for s in range(n) if upto[s] - tiles[s] <= u < upto[s]]
            s = mine[0] if mine else n
            c0, length = (row(s), rows[s]) if mine else (row(n), N - row(n))
            t = first(c0, s) + u - (upto[s] - tiles[s] if mine else upto[-1])
            r0 = (t - first(c0, s)) * 16
            nr = max(0, min(16, length * group - r0)) if r0 >= 0 else 0
            for r in range(nr):
                i, h = divmod(r0 + r, group)
                assert 0 <= c0 + i < N
                seen.append((c0 + i, h))
            if case % 4 != 3:
                assert not (empty and mine)
                empty = empty or nr == 0 or not mine
        if case % 4 != 3:
            assert sorted(seen) == [(i, h) for i in range(N) for h in range(group)]


def test_bytes_of_scales():
    """The least scale whose 448-fold holds a magnitude, from its bits; and the ends of bfloat16."""
    import struct
    bits = lambda x: struct.unpack("<I", struct.pack("<f", x))[0]  # noqa: E731
    byte = lambda x: min(max(((bits(x) + 0x1fffff) >> 23) - 8, 10), 246)  # noqa: E731
    rng = random.Random(3)
    values = [448.0 * 2.0 ** n * f for n in range(-100, 100) for f in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24, 1.1, 0.6)]
    for x in values + [2.0 ** rng.uniform(-100, 120) for _ in range(1000)]:
        x = struct.unpack("<f", struct.pack("<f", x))[0]
        s = 2.0 ** (byte(x) - 127)
        assert 448 * s >= x and 224 * s < x
    assert byte(0.0) == 10 and byte(1e-45) == 10 and byte(3.4e38) == 246
    assert 2.0 ** -9 * 2.0 ** (10 - 127) == 2.0 ** -126 and 448 * 2.0 ** (246 - 127) == bits(0) + 1.75 * 2.0 ** 127


# ------------------------------------------------------------------ torch
def _fake8(**kw):
    """(ops, q, k, v, cache, scales, inv_freq, weights) over a cache of 8 bits, without values."""
    import torch
    t, q, k, v, cache, f = _fake(**kw)
    m, (p, h, page, d) = dict(device=cache[0].device), cache[0].shape
    kp, vp = (torch.empty(s, dtype=torch.float8_e4m3fn, **m) for s in ((p, h, page, d), (p, h, page // 16, d, 16)))
    scales = tuple(torch.empty(p, h, page // 16, dtype=torch.float8_e8m0fnu, **m) for _ in range(2))
    return t, q, k, v, (kp, vp, *cache[2:]), scales, f, (torch.empty(d, **m), torch.empty(d, **m))


def _calls8():
    import torch
    e = torch.empty_like
    return {"kv_append": lambda t, q, k, v, c, s, f, w: t.kv_append(k, v, *c, f, "half", 1.0, w[1], 1e-6, *s),
            "kv_append_q": lambda t, q, k, v, c, s, f, w: t.kv_append_q(q, k, v, *c, f, "half", 1.0, *w, 1e-6, *s),
            "kv_append_q_into": lambda t, q, k, v, c, s, f, w: t.kv_append_q_into(q, e(q), k, v, *c, f, "half", 1.0, *w, 1e-6, *s),
            "kv_read": lambda t, q, k, v, c, s, f, w: t.kv_read(*c, 5, *s),
            "kv_read_into": lambda t, q, k, v, c, s, f, w: t.kv_read_into(*c, e(k), e(v), *s),
            "paged_attention": lambda t, q, k, v, c, s, f, w: t.paged_attention(q, *c, 0.1, *s, 7, 1),
            "paged_attention_into": lambda t, q, k, v, c, s, f, w: t.paged_attention_into(q, *c, 0.1, e(q), *s, 7, 1)}


@pytest.mark.parametrize("name", list(_calls8()))
def test_fake_results_and_refused_gradients(name):
    import torch
    args = _fake8()
    call = _calls8()[name]
    out = call(*args)
    if name.startswith("kv_read") and out is not None:
        assert [x.shape for x in out] == [(5, 2, 64)] * 2 and out[0].dtype == torch.bfloat16
    elif out is not None:
        assert out.shape == (5, 4, 64) and out.dtype == torch.bfloat16
    if "append" in name:  # a weight that requires a gradient
        w = tuple(x.clone().requires_grad_() for x in args[-1])
        with pytest.raises(RuntimeError, match=f"prunepath.{name}: inference only"):
            call(*args[:-1], w)
        with torch.no_grad():
            call(*args[:-1], w)
    elif name.startswith("paged"):
        with pytest.raises(RuntimeError, match=f"prunepath.{name}: inference only"):
            call(args[0], args[1].clone().requires_grad_(), *args[2:])


def test_fake_calls_check_what_real_ones_do():
    import torch
    t, q, k, v, c, s, f, w = _fake8()
    kp, vp, table, lens, cu = c
    kb, vb = _fake()[4][:2]
    n, pos = t.qk_norm_rotary, torch.empty(5, dtype=torch.int64, device="meta")
    e = torch.empty_like
    bad = {"one scale": lambda: t.paged_attention(q, *c, 0.1, s[0], None), "no scales": lambda: t.paged_attention(q, *c, 0.1),
           "scales of the 16-bit cache": lambda: t.paged_attention(q, kb, vb, *c[2:], 0.1, *s), "values as keys": lambda: t.paged_attention(q, kp, kp, *c[2:], 0.1, *s),
           "values as of 16 bits": lambda: t.paged_attention(q, kp, vp.view(9, 2, 64, 16), *c[2:], 0.1, *s),
           "types of scales": lambda: t.paged_attention(q, *c, 0.1, *(x.view(torch.uint8) for x in s)), "fewer scales": lambda: t.paged_attention(q, *c, 0.1, s[0], s[1][:3]),
           "a window": lambda: t.paged_attention(q, *c, 0.1, *s, -1, 0), "first tokens": lambda: t.paged_attention(q, *c, 0.1, *s, 5, -1),
           "first tokens alone": lambda: t.paged_attention(q, *c, 0.1, *s, 0, 2), "read without scales": lambda: t.kv_read(*c, 5), "rows": lambda: t.kv_read(*c, -1, *s),
           "results": lambda: t.kv_read_into(*c, e(k), e(v)[:4], *s), "float results": lambda: t.kv_read_into(*c, e(k).float(), e(v).float(), *s),
           "one weight": lambda: t.kv_append_q(q, k, v, *c, f, "half", 1.0, w[0], None, 1e-6, *s), "weights": lambda: t.kv_append(k, v, *c, f, "half", 1.0, w[1][:32], 1e-6, *s),
           "half weights": lambda: t.kv_append(k, v, *c, f, "half", 1.0, w[1].half(), 1e-6, *s), "an append's scale": lambda: t.kv_append(k, v, *c, f, "half", 1.0, None, 1e-6, s[0], None),
           "tokens": lambda: n(q, k[:4], *w, pos, f), "types": lambda: n(q, k.float(), *w, pos, f), "a norm's weights": lambda: n(q, k, w[0][:5], w[1], pos, f),
           "weights of two types": lambda: n(q, k, w[0], w[1].bfloat16(), pos, f), "positions": lambda: n(q, k, *w, pos[:4], f), "a layout": lambda: n(q, k, *w, pos, f, "other"),
           "pairs": lambda: n(q[..., :32], k[..., :32], w[0][:32], w[1][:32], pos, f), "frequencies": lambda: n(q, k, *w, pos, f.float()),
           "gradients": lambda: t.qk_norm_rotary_bwd(q[:4], k, q, k, *w, pos, f), "types of gradients": lambda: t.qk_norm_rotary_bwd(q.float(), k, q, k, *w, pos, f)}
    for what, call in bad.items():
        with pytest.raises(RuntimeError, match="prunepath"):
            call()
            print("not refused:", what)


def test_written_arguments_count_as_changed():
    import torch
    t, q, k, v, c, s, f, w = _fake8()
    out, ko, vo = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    every = [q, k, v, *c, *s, f, *w, out, ko, vo]
    for op, args in ((t.kv_append, (k, v, *c, f, "half", 1.0, w[1], 1e-6, *s)), (t.kv_append_q, (q, k, v, *c, f, "half", 1.0, *w, 1e-6, *s)),
                     (t.kv_append_q_into, (q, out, k, v, *c, f, "half", 1.0, *w, 1e-6, *s)), (t.kv_read, (*c, 5, *s)), (t.kv_read_into, (*c, ko, vo, *s)),
                     (t.paged_attention, (q, *c, 0.1, *s, 3, 1)), (t.paged_attention_into, (q, *c, 0.1, out, *s, 3, 1))):
        schema = op.default._schema.arguments
        writes = [a for a, x in zip(args, schema) if x.alias_info is not None and x.alias_info.is_write]
        assert len(writes) == {"kv_append": 4, "kv_append_q": 4, "kv_append_q_into": 5, "kv_read": 0, "kv_read_into": 2, "paged_attention": 0,
                               "paged_attention_into": 1}[op.default._schema.name.split("::")[1]]
        before = [x._version for x in every]
        op(*args)
        for x, old in zip(every, before):
            assert x._version == old + any(x is y for y in writes), op


def test_gradients_of_the_norm_without_a_gpu():
    """Which leaves get one, what double and forward mode say, and that a saved tensor that changed raises."""
    import torch
    import torch.autograd.forward_ad as fw
    t, q, k, v, c, s, f, w = _fake8()
    pos = torch.empty(5, dtype=torch.int64, device="meta")
    leaves = [x.clone().requires_grad_() for x in (q, k, *w)]
    y = t.qk_norm_rotary(*leaves, pos, f)
    g = torch.autograd.grad(y, leaves, [torch.empty_like(x) for x in y])
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(g, leaves))
    y = t.qk_norm_rotary(*leaves, pos, f)
    g = torch.autograd.grad([y[0]], leaves, [torch.empty_like(y[0])], allow_unused=True)
    assert g[1] is None and g[3] is None and g[0].shape == q.shape and g[2].shape == (64,)
    y = t.qk_norm_rotary(*leaves, pos, f)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y[0].sum(), leaves[0], create_graph=True)
    y = t.qk_norm_rotary(*leaves, pos, f)
    with torch.no_grad():
        leaves[2].add_(1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(y[0].sum(), leaves[0])
    with pytest.raises(RuntimeError, match="no gradient in inv_freq"):
        t.qk_norm_rotary(q, k, *w, pos, f.clone().requires_grad_())
    with fw.dual_level():
        for i in range(4):
            args = [fw.make_dual(x, torch.empty_like(x)) if j == i else x for j, x in enumerate((q, k, *w))]
            with pytest.raises(RuntimeError, match="no forward-mode"):
                t.qk_norm_rotary(*args, pos, f)


def test_symbolic_sizes():
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    t, q, k, v, c, s, f, w = _fake8()

    def step(q, k, v, kp, vp, table, lens, cu, ks, vs, f, wq, wk):
        q = t.kv_append_q(q, k, v, kp, vp, table, lens, cu, f, "half", 1.0, wq, wk, 1e-6, ks, vs)
        return t.paged_attention(q, kp, vp, table, lens, cu, 0.1, ks, vs, 100, 4), t.kv_read(kp, vp, table, lens, cu, q.shape[0], ks, vs)

    with torch.no_grad():
        gm = make_fx(step, tracing_mode="symbolic")(q, k, v, *c, *s, f, *w)
    out = [n.meta["val"] for n in gm.graph.nodes if n.op == "call_function" and ("paged_attention" in str(n.target) or "kv_read" in str(n.target))]
    assert len(out) == 2 and not isinstance(out[0].shape[0], int) and out[1][0].shape[0] == out[0].shape[0]


def test_wrappers_refuse():
    import torch
    ops = import_pkg().ops
    (k, v), s = ops.paged_cache8(3, 32, 2, 64)
    assert k.shape == (3, 2, 32, 64) and v.shape == (3, 2, 2, 64, 16) and s[0].shape == s[1].shape == (3, 2, 2)
    x, i = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    cache = (k, v, torch.zeros(1, 3, dtype=torch.int32), i, torch.zeros(2, dtype=torch.int32))
    w = torch.ones(64)
    for bad in (lambda: ops.paged_attention(x, *cache, scales=s), lambda: ops.kv_append(x, x, *cache, scales=s), lambda: ops.kv_read(*cache, 1, scales=s),
                lambda: ops.qk_norm_rotary(x, x, w, w, i, ops.rotary_frequencies(64)[0])):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            bad()
    for bad in (lambda: ops.paged_attention(x, *cache, scales=s, window=0), lambda: ops.kv_read(*cache, scales=s), lambda: ops.kv_append(x, x, *cache, q_weight=w),
                lambda: ops.kv_read(*cache, 3, scales=s, out=(x, x))):
        with pytest.raises(RuntimeError, match="prunepath"):
            bad()


def test_fake_calls_refuse_strided_arguments():
    """What a real call takes contiguous only, a traced one does too: the weights of an append's norms, the frequencies, the cache, its
    scales and the batch's integers."""
    import torch
    t, q, k, v, c, s, f, w = _fake8()

    def strided(x):  # its shape, every other element of a row
        return torch.empty(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype, device=x.device)[..., ::2]

    def put(args, i, x):
        return (*args[:i], x, *args[i + 1:])

    calls = [lambda c=c, s=s, f=f, w=w: t.kv_append_q(q, k, v, *c, f, "half", 1.0, *w, 1e-6, *s),
             lambda c=c, s=s, f=f, w=w: t.kv_append_q_into(q, torch.empty_like(q), k, v, *c, f, "half", 1.0, *w, 1e-6, *s),
             lambda c=c, s=s, f=f, w=w: t.kv_append(k, v, *c, f, "half", 1.0, w[1], 1e-6, *s)]
    reads = [lambda c=c, s=s: t.kv_read(*c, 5, *s), lambda c=c, s=s: t.kv_read_into(*c, torch.empty_like(k), torch.empty_like(v), *s),
             lambda c=c, s=s: t.paged_attention(q, *c, 0.1, *s, 7, 1), lambda c=c, s=s: t.paged_attention_into(q, *c, 0.1, torch.empty_like(q), *s)]
    bad = []
    for call in calls:
        call()
        bad += [(call, dict(f=strided(f))), (call, dict(w=put(w, 1, strided(w[1]))))]
    bad += [(call, dict(w=put(w, 0, strided(w[0])))) for call in calls[:2]]
    for call in calls + reads:
        call()
        bad += [(call, dict(c=put(c, i, strided(c[i])))) for i in range(5)] + [(call, dict(s=put(s, i, strided(s[i])))) for i in range(2)]
    for call, kw in bad:
        with pytest.raises(RuntimeError, match="prunepath.*contiguous"):
            call(**kw)
            print("not refused:", list(kw))


@pytest.mark.parametrize("group", [1, 3, 8])
def test_gaps_come_behind_the_tiles_of_uneven_batches(group):
    """128-row tiles of sequences whose lengths differ by more than a quarter, restated: every row of a sequence, and of none, once, the
    longest sequences first, each one's last tiles first, no tile without rows before one of a sequence with some; the four waves' counts
    together are those of one; offsets out of order stay inside."""
    rng = random.Random(group)
    for case in range(60):
        n = rng.choice([2, 3, 9, 40, 63, 64])
        new = [rng.choice([0, 1, 1, 5, 128, 200, 300]) for _ in range(n)]
        lens = [rng.choice([0, 7, 500, 500, 4000, 1 << 26]) for _ in range(n)]
        cu = [sum(new[:i]) for i in range(n + 1)]
        N = cu[-1] + rng.choice([0, 3, 500])
        if case % 4 == 3:
            cu = [rng.randint(-5, N + 5) for _ in cu]
        row = lambda s: 0 if s == 0 else min(max(cu[s], 0), N)  # noqa: E731
        first = lambda c, s: c * group // 128 + s  # noqa: E731
        rows = [max(row(s + 1) - row(s), 0) for s in range(n)] + [0] * (64 - n)
        tiles = [-(-r * group // 128) for r in rows]
        key = [((min(max(lens[s], 1), (1 << 25) - 1) << 6) if tiles[s] else 0) | (63 - s) for s in range(n)] + [63 - s for s in range(n, 64)]
        assert len(set(key)) == 64
        parts = [[sum(tiles[j] for j in range(16 * w, 16 * w + 16) if key[j] > key[s]) for s in range(64)] for w in range(4)]
        before, total = [sum(p[s] for p in parts) for s in range(64)], sum(tiles)
        seen, order, empty = [], [], False
        for u in range(N * group // 128 + n + 1):
            mine = [s for s in range(64) if before[s] <= u < before[s] + tiles[s]]
            assert len(mine) <= 1
            s = mine[0] if mine else n
            c0, length = (row(s), rows[s]) if mine else (row(n), N - row(n))
            t = first(c0, s) + (before[s] + tiles[s] - 1 - u if mine else u - total)
            r0 = (t - first(c0, s)) * 128
            assert r0 >= 0
            nr = max(0, min(128, length * group - r0))
            for r in range(nr):
                i, h = divmod(r0 + r, group)
                assert 0 <= c0 + i < N
                seen.append((c0 + i, h))
            if case % 4 != 3:
                assert not (empty and mine) and (not mine or nr)
                empty = empty or not mine
                if mine:
                    order.append((key[s], r0))
        if case % 4 != 3:
            assert sorted(seen) == [(i, h) for i in range(N) for h in range(group)]
            assert order == sorted(order, reverse=True)


@pytest.mark.parametrize("group", [1, 3, 8])
def test_windowed_tiles_by_their_walks(group):
    """With a window, restated: the key of the order is no less than what the sequence's longest tile walks beyond the window's start and
    the first tokens, and not the cache's length; walks that are alike go from the batch's last sequence to its first, tiles with rows
    before all gaps."""
    rng = random.Random(group)
    for case in range(80):
        n = rng.choice([2, 9, 40, 64])
        window, sinks = rng.choice([1, 60, 700, 1 << 30]), rng.choice([0, 4, 300])
        new = [rng.choice([0, 1, 128, 200, 300]) for _ in range(n)]
        lens = [r + rng.choice([0, 500, 4000, 20000]) for r in new]
        cu = [sum(new[:i]) for i in range(n + 1)]
        N = cu[-1] + rng.choice([0, 3])
        walk = min(window + sinks + 128, (1 << 25) - 1)
        tiles = [-(-r * group // 128) for r in new]
        keys = [min(max(x, 1), walk) for x, k in zip(lens, tiles) if k]
        for x, r in zip(lens, new):
            for r0 in range(0, r * group, 128):  # what the tile's rows attend
                last, start = x - r + (r0 + min(128, r * group - r0) - 1) // group, max(0, x - r + r0 // group - window + 1)
                assert min(max(x, 1), walk) >= min(sinks, start) + last + 1 - start
        if keys and max(keys) - min(keys) > max(keys) // 4:
            continue  # sorted, as without a window
        total, seen = sum(tiles), []
        before = [total - sum(tiles[:s + 1]) for s in range(n)]
        for u in range(N * group // 128 + n + 1):
            mine = [s for s in range(n) if before[s] <= u < before[s] + tiles[s]]
            assert len(mine) == (u < total)
            if mine:
                seen.append((mine[0], before[mine[0]] + tiles[mine[0]] - 1 - u))
        assert seen == [(s, i) for s in range(n - 1, -1, -1) for i in range(tiles[s] - 1, -1, -1)]
