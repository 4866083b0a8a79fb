"""Timed cases of the normed rotation of queries and keys, of the cache in 8 bits, and of attention that sees a window and
a few first tokens.

A case is a dict:

* ``kind`` "norm": ``batch`` x ``length`` tokens of ``heads`` query and ``kv_heads`` key heads of ``dim`` channels, every head
  normed and its first ``rotary`` channels rotated (``layout`` "half" or "interleaved"), positions from ``start`` on.
  ``packed``: q and k are parts of one projection's rows. ``backward``: the gradients of q, k and the weights too.
* ``kind`` "append": ``seqs`` sequences, each with up to ``new`` new tokens after up to ``ctx`` cached ones (``mix`` draws the
  lengths, 0: all at the largest), into an 8-bit cache in pages of ``page`` tokens, rotated, and normed before if ``norm``;
  q, k and v are parts of one projection's rows.
* ``kind`` "read": all tokens of such sequences read back from the cache.
* ``kind`` "attend": the attention of the new tokens over the cache that holds them (``bits`` 8 or 16); ``window`` and ``sinks``:
  a token sees the last ``window`` tokens, itself among them, and the sequence's first ``sinks`` (window 0: all).
* ``kind`` "step": append and attention, as one layer of a serving step has them.

The 8-bit cache: k_pages [pages, kv_heads, page, dim] and v_pages [pages, kv_heads, page / 16, dim, 16], float8_e4m3fn;
k_scales and v_scales [pages, kv_heads, page / 16], float8_e8m0fnu: a power of two for each block of 16 tokens and head. The
least 2^n whose 448-fold holds the block's values; a block that held tokens before keeps its scale if that is more, and
is brought to the new one if that is less. The cache in 16 bits: [pages, kv_heads, page, dim] and [pages, kv_heads, dim, page].
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
BASE = 10000.0
EPS = 1e-6
STEP_COST = 2.2e9  # no drawn case has more work than the largest listed one


def _ops():
    return importlib.import_module("prune_path_openpangu-embedded-1b_amd").ops


def _norm(name, batch, length, heads, kv_heads, dim, rotary, layout, dtype, start=0, packed=False, backward=False):
    return {"name": name, "kind": "norm", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "layout": layout, "dtype": dtype, "start": start, "packed": packed, "backward": backward}


def _cached(name, kind, seqs, new, ctx, heads, kv_heads, dim, page, mix=0, bits=8, window=0, sinks=0, rotary=0, layout="half",
            dtype="bf16", norm=False):
    return {"name": name, "kind": kind, "seqs": seqs, "new": new, "ctx": ctx, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "mix": mix, "bits": bits, "window": window, "sinks": sinks, "rotary": rotary or dim,
            "layout": layout, "dtype": dtype, "norm": norm}


def listed():
    return [
        # one generated token's query and key heads
        _norm("norm_1_token", 1, 1, 12, 12, 128, 128, "half", "bf16", start=1024),
        # a training batch with its gradients; q and k are parts of a joint projection's rows
        _norm("norm_train_4x2048", 4, 2048, 12, 12, 128, 128, "half", "bf16", packed=True, backward=True),
        # shared key heads of an odd size, part of them rotated, far positions, float32
        _norm("norm_part_f32", 3, 1111, 20, 4, 80, 32, "interleaved", "f32", start=1000000, backward=True),
        # a decode step of a served batch
        _cached("append8_decode_32", "append", 32, 1, 4096, 12, 12, 128, 16, mix=3),
        # a long prompt's first chunk, with the norms
        _cached("append8_chunk_8192", "append", 1, 8192, 0, 12, 12, 128, 64, norm=True),
        # a few sequences of odd lengths moved out of the cache
        _cached("read8_ragged_5", "read", 5, 1, 777, 32, 8, 64, 32, mix=5),
        # a whole batch of long sequences read back
        _cached("read8_64", "read", 64, 1, 8191, 12, 12, 128, 16, mix=7),
        # one user's token at the decoder stack's full length
        _cached("attend8_decode_1", "attend", 1, 1, 1151, 12, 12, 128, 16),
        # a served batch of sequences of any length
        _cached("attend8_decode_64", "attend", 64, 1, 8191, 12, 12, 128, 16, mix=7),
        # chunks and single tokens together, odd lengths, many query heads on few key heads
        _cached("attend8_mixed_9", "attend", 9, 700, 4000, 24, 4, 128, 32, mix=11),
        # a long prompt in a model whose layers see a window and the first tokens, cache in 16 bits
        _cached("window_prompt_8192", "attend", 1, 8192, 0, 12, 12, 128, 16, bits=16, window=1024, sinks=4),
        # one such layer of a serving step far into long sequences, cache in 8 bits
        _cached("window_step_32", "step", 32, 1, 16384, 24, 8, 128, 16, mix=2, window=1000, sinks=4, norm=True),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "append", "read", "attend", "attend", "step"])
        kv = rng.choice([1, 2, 4, 8, 12, 12])
        heads = kv * rng.choice([1, 1, 2, 3, 5, 8])
        if kind == "norm":
            dim = 2 * _spread(rng, 8, 128)
            c = {"kind": kind, "batch": _spread(rng, 1, 8), "length": _spread(rng, 1, 4096), "heads": heads, "kv_heads": kv,
                 "dim": dim, "rotary": rng.choice([dim, 2 * rng.randint(1, dim // 2)]),
                 "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["bf16", "f32"]),
                 "start": rng.choice([0, _spread(rng, 1, 2000000)]), "packed": rng.random() < 0.5,
                 "backward": rng.random() < 0.5}
        else:
            dim = rng.choice([64, 128, 128])
            windowed = kind in ("attend", "step") and rng.random() < 0.5
            c = {"kind": kind, "seqs": _spread(rng, 1, 64), "new": rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 2, 2048)]),
                 "ctx": _spread(rng, 1, 16384), "heads": heads, "kv_heads": kv, "dim": dim,
                 "page": rng.choice([16, 16, 32, 64, 128]), "mix": rng.randint(0, 1 << 20),
                 "bits": rng.choice([8, 16]) if windowed and kind == "attend" else 8,
                 "window": _spread(rng, 16, 4096) if windowed else 0, "sinks": rng.choice([0, 1, 4, 130]) if windowed else 0,
                 "rotary": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                 "dtype": rng.choice(["bf16", "f32"]), "norm": rng.random() < 0.5}
            if kind in ("attend", "read"):
                c |= {"rotary": dim, "layout": "half", "dtype": "bf16", "norm": False}
        if _cost(c) <= STEP_COST and _held(c) <= 6.0e9:
            return c


def _lengths(case):
    """(new tokens, tokens in the cache after them) of each sequence."""
    rng, B = random.Random(case["mix"]), case["seqs"]
    if not case["mix"]:
        return [case["new"]] * B, [case["ctx"] + case["new"]] * B
    new = [1 if case["new"] == 1 or rng.random() < 0.5 else rng.randint(1, case["new"]) for _ in range(B)]
    new[rng.randrange(B)] = case["new"]
    ctx = [rng.randint(0, case["ctx"]) for _ in range(B)]
    ctx[rng.randrange(B)] = case["ctx"]
    return new, [n + c for n, c in zip(new, ctx)]


def _first_seen(case, p):
    """The first position of the window of the token at p."""
    return max(0, p - case["window"] + 1) if case["window"] else 0


def _pairs(case):
    """Attended (token, cached token) pairs."""
    return sum((p + 1 - _first_seen(case, p)) + min(case["sinks"], _first_seen(case, p))
               for n, t in zip(*_lengths(case)) for p in range(t - n, t))


def _seen(case):
    """Cached tokens that any new token attends."""
    return sum(t - _first_seen(case, t - n) + min(case["sinks"], _first_seen(case, t - n)) for n, t in zip(*_lengths(case)))


def work(case):
    D, Hq, Hkv = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "norm":
        tokens = case["batch"] * case["length"]
        n = tokens * (Hq + Hkv) * D
        passes = 5 if case["backward"] else 2  # x, y; x, dy, dx
        return {"bytes": passes * n * SIZE[case["dtype"]] + 8 * tokens + 4 * D * SIZE[case["dtype"]],
                "flops": (20 if case["backward"] else 7) * n}
    new, total = _lengths(case)
    N, blocks = sum(new), sum(-(-t // 16) for t in total)
    if case["kind"] == "read":
        n = 2 * sum(total) * Hkv * D
        return {"bytes": 3 * n + 2 * blocks * Hkv, "flops": n}
    table = 4 * sum(-(-t // case["page"]) for t in total) + 8 * case["seqs"]
    touched = sum((t - 1) // 16 - (t - n) // 16 + 1 for n, t in zip(new, total))
    append = N * D * ((Hq + 2 * Hkv) * SIZE[case["dtype"]] + Hq * 2 + 2 * Hkv) + 2 * 2 * touched * Hkv
    held = case["bits"] // 8
    attend = 2 * D * 2 * N * Hq + 2 * _seen(case) * Hkv * D * held + (2 * _seen(case) // 16 * Hkv if held == 1 else 0) + table
    flops = 4 * D * Hq * _pairs(case)
    if case["kind"] == "append":
        return {"bytes": append + 8 * case["seqs"], "flops": (10 if case["norm"] else 6) * N * D * (Hq + Hkv)}
    return {"bytes": attend + (append if case["kind"] == "step" else 0), "flops": flops}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _held(case):
    """Bytes of the plain form's largest matrix."""
    if case["kind"] == "norm":
        return 0
    new, total = _lengths(case)
    B, T = case["seqs"], max(total)
    scores = case["heads"] * max(new) if case["kind"] in ("attend", "step") else 0
    return 4 * B * T * max(scores, case["kv_heads"] * case["dim"])


def _frequencies(rotary):
    return BASE ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64) / rotary)


# ---- 8 bits: a block's exponent n (the scale is 2^n) and its values x 2^-n, rounded to e4m3
def _exponent(top):
    """Least n with top <= 448 * 2^n."""
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    n = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top > 0, n, -117).clamp(-117, 119)


def _to8(x, n):
    return torch.ldexp(x, -n).to(torch.float8_e4m3fn)


def _from8(x, n):
    return torch.ldexp(x.float(), n)


def _to_scales(n):
    return (n + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_scales(s):
    return s.view(torch.uint8).int() - 127


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    dt = DTYPES[case["dtype"]]
    D, Hq, Hkv = case["dim"], case["heads"], case["kv_heads"]
    s = {"case": case, "inv_freq": _frequencies(case["rotary"]).to(dev),
         "q_weight": (1.0 + 0.2 * normal(D)).to(dt), "k_weight": (1.0 + 0.2 * normal(D)).to(dt)}
    if case["kind"] == "norm":
        B, L = case["batch"], case["length"]
        # heads differ in size, as a projection's do
        every = Hq + Hkv * (2 if case["packed"] else 1)
        wide = (normal(B, L, every, D) * torch.exp(0.5 * normal(1, 1, every, 1))).to(dt)
        s["q"], s["k"] = wide[:, :, :Hq], wide[:, :, Hq:Hq + Hkv]
        if not case["packed"]:
            s["q"], s["k"] = s["q"].contiguous(), s["k"].contiguous()
        s["positions"] = torch.arange(case["start"], case["start"] + L, device=dev).expand(B, L)
        if case["backward"]:
            s["wrt"] = [s[n].requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
            s["dq"], s["dk"] = normal(B, L, Hq, D).to(dt), normal(B, L, Hkv, D).to(dt)
        return s
    B, ps = case["seqs"], case["page"]
    new, total = _lengths(case)
    N, per, blocks = sum(new), -(-max(total) // ps), ps // 16
    s["new"], s["total"] = new, total
    s["kv_lens"] = torch.tensor(total, dtype=torch.int32, device=dev)
    rows = total if case["kind"] == "read" else new
    s["cu_q"] = torch.tensor([sum(rows[:i]) for i in range(B + 1)], dtype=torch.int32, device=dev)
    used = [-(-t // ps) for t in total]
    order = torch.randperm(sum(used) + 1, generator=g, device=dev).to(torch.int32)[:sum(used)]
    first = torch.tensor([sum(used[:i]) for i in range(B)], device=dev)[:, None]
    j = torch.arange(per, device=dev)[None]
    there = j < torch.tensor(used, device=dev)[:, None]
    s["table"] = torch.where(there, order[(first + j).clamp(max=sum(used) - 1)], -1).to(torch.int32).contiguous()
    pages = sum(used) + 1
    # values differ in size from page to page and from head to head
    k = normal(pages, Hkv, ps, D) * torch.exp(0.3 * normal(pages, Hkv, 1, 1))
    v = (0.5 * normal(pages, Hkv, ps, D) + 0.5 * normal(1, Hkv, 1, D)) * torch.exp(0.5 * normal(pages, Hkv, 1, 1))
    if case["bits"] == 16:
        s["k_pages"], s["v_pages"] = k.to(torch.bfloat16), v.transpose(2, 3).to(torch.bfloat16).contiguous()
    else:
        for name, x in (("k", k), ("v", v)):
            x = x.view(pages, Hkv, blocks, 16, D)
            n = _exponent(x.abs().amax((3, 4)))
            x8 = _to8(x, n[..., None, None]).view(torch.uint8)
            x8 = x8.transpose(3, 4).contiguous() if name == "v" else x8.reshape(pages, Hkv, ps, D)
            s[name + "_pages"], s[name + "_scales"] = x8.view(torch.float8_e4m3fn), _to_scales(n)
    if case["kind"] == "read":
        return s
    if case["kind"] == "attend":
        s["q"] = (2.0 * normal(N, Hq, D)).to(torch.bfloat16)
        return s
    qkv = normal(N, Hq + 2 * Hkv, D)
    qkv[:, :Hq] *= 2.0
    qkv = qkv.to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    return s


# ---- the plain forms: elementary torch operations, float32 (angles float64), rounded once at the end
def _turn(y, positions, inv_freq, layout, rotary, back=False):
    """y [..., heads, dim] rotated by positions [...]; `back`: by the opposite angles."""
    angle = positions.to(torch.float64)[..., None] * inv_freq
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    if back:
        sin = -sin
    r, rest = y[..., :rotary], y[..., rotary:]
    a, b = (r[..., :rotary // 2], r[..., rotary // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([r, rest], -1)


def _normed(x, weight):
    y = x.float()
    return y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_norm(s):
    c = s["case"]
    args = (s["positions"], s["inv_freq"], c["layout"], c["rotary"])
    out = tuple(_turn(_normed(s[n].detach(), s[n + "_weight"].detach()), *args).to(s[n].dtype) for n in "qk")
    if not c["backward"]:
        return out
    dx, dw = [], []
    for n in "qk":
        x, w, g = s[n].detach().float(), s[n + "_weight"].detach().float(), _turn(s["d" + n].float(), *args, back=True)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        dw.append((g * x * r).sum((0, 1, 2)).to(s[n + "_weight"].dtype))
        dx.append((r * (w * g - x * r * r * (w * g * x).mean(-1, keepdim=True))).to(s[n].dtype))
    return out + tuple(dx) + tuple(dw)


def _places(s):
    """Sequence and place in it of every row."""
    n = torch.arange(s["rows"] if "rows" in s else s["q"].shape[0], device=s["kv_lens"].device)
    seq = torch.searchsorted(s["cu_q"][1:].long(), n, right=True)
    return seq, (s["kv_lens"].long()[seq] - s["cu_q"].long()[seq + 1]) + n


def _plain_append(s):
    c = s["case"]
    ps, D, Hkv = c["page"], c["dim"], c["kv_heads"]
    seq, pos = _places(s)
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q, k = _normed(s["q"], s["q_weight"]), _normed(s["k"], s["k_weight"])
    q, k = (_turn(x, pos, s["inv_freq"], c["layout"], c["rotary"]) for x in (q, k))
    block = s["table"][seq, pos // ps].long() * (ps // 16) + pos % ps // 16        # of each token, in the whole cache
    first = s["kv_lens"].long() - (s["cu_q"][1:] - s["cu_q"][:-1]).long()         # each sequence's first new place
    front = s["table"][torch.arange(c["seqs"], device=seq.device), first // ps].long() * (ps // 16) + first % ps // 16
    begun = first % 16 > 0                                                          # the block there holds tokens
    place = torch.arange(16, device=seq.device)
    for name, x in (("k", k), ("v", v)):
        p8 = s[name + "_pages"].view(torch.uint8)
        p8 = p8.view(-1, Hkv, ps // 16, 16, D) if name == "k" else p8.transpose(3, 4)  # [pages, heads, block, 16, D]
        n = _from_scales(s[name + "_scales"]).transpose(1, 2).reshape(-1, Hkv)      # of every block and head
        top = torch.zeros(n.shape, device=n.device).index_reduce_(0, block, x.abs().amax(-1), "amax")
        need = _exponent(top)
        need[front] = torch.where(begun[:, None], torch.maximum(need[front], n[front]), need[front])
        at = front // (ps // 16), slice(None), front % (ps // 16)
        old = _to8(_from8(p8[at].view(torch.float8_e4m3fn), n[front][..., None, None]), need[front][..., None, None]).view(torch.uint8)
        p8[at] = torch.where((place < first[:, None] % 16)[:, None, :, None], old, p8[at])
        n[block] = need[block]
        p8[block // (ps // 16), :, block % (ps // 16), pos % 16] = _to8(x, n[block][..., None]).view(torch.uint8)
        s[name + "_scales"].copy_(_to_scales(n.view(-1, ps // 16, Hkv).transpose(1, 2)))
    return q.to(torch.bfloat16)


def _wide(s, table):
    """(keys, values) [*table.shape, heads, page, dim] of the pages that the table names, float32."""
    c = s["case"]
    ps, D, Hkv = c["page"], c["dim"], c["kv_heads"]
    if c["bits"] == 16:
        return s["k_pages"][table].float(), s["v_pages"][table].transpose(-1, -2).float()
    nk, nv = (_from_scales(s[n])[table] for n in ("k_scales", "v_scales"))
    k = s["k_pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float().view(*table.shape, Hkv, ps // 16, 16, D)
    v = s["v_pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float().transpose(-1, -2)
    shape = (*table.shape, Hkv, ps, D)
    return torch.ldexp(k, nk[..., None, None]).view(shape), torch.ldexp(v, nv[..., None, None]).reshape(shape)


def _plain_read(s):
    c = s["case"]
    seq, pos = _places(s | {"rows": sum(s["total"])})
    table = s["table"].long().clamp(min=0)
    k, v = _wide(s, table)                                              # [seqs, pages, heads, page, dim]
    at = seq, pos // c["page"], slice(None), pos % c["page"]
    return k[at].to(torch.bfloat16), v[at].to(torch.bfloat16)


def _plain_attend(s, q):
    c = s["case"]
    B, D, Hkv, T, L = c["seqs"], c["dim"], c["kv_heads"], s["table"].shape[1] * c["page"], max(s["new"])
    group = c["heads"] // Hkv
    k, v = (x.transpose(1, 2).reshape(B, Hkv, T, D) for x in _wide(s, s["table"].long().clamp(min=0)))
    k = k.transpose(2, 3).contiguous()
    seq, pos = _places(s)
    row = torch.arange(q.shape[0], device=q.device) - s["cu_q"].long()[seq]
    x = torch.zeros(B, L, Hkv, group, D, device=q.device)
    x[seq, row] = q.float().view(-1, Hkv, group, D)
    last = torch.zeros(B, L, dtype=torch.long, device=q.device)
    last[seq, row] = pos
    t = torch.arange(T, device=q.device)
    hidden = t > last[:, :, None]                                              # [B, L, T]
    if c["window"]:
        hidden |= (t <= last[:, :, None] - c["window"]) & (t >= c["sinks"])
    p = torch.matmul(x.permute(0, 2, 3, 1, 4).reshape(B, Hkv, group * L, D), k).view(B, Hkv, group, L, T)
    p = p.mul_(D ** -0.5).masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, group * L, T), v).view(B, Hkv, group, L, D) / total
    return o.permute(0, 3, 1, 2, 4)[seq, row].reshape(-1, c["heads"], D).to(torch.bfloat16)


def _own(s):
    ops, c = _ops(), s["case"]
    if c["kind"] == "norm":
        y = ops.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"], layout=c["layout"], eps=EPS)
        if not c["backward"]:
            return y
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, s["wrt"], (s["dq"], s["dk"]))
    scales = (s["k_scales"], s["v_scales"]) if c["bits"] == 8 else None
    cache = (s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["cu_q"])
    if c["kind"] == "read":
        return ops.kv_read(*cache, sum(s["total"]), scales=scales)
    q = s["q"]
    if c["kind"] != "attend":
        weights = {"q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": EPS} if c["norm"] else {}
        q = ops.kv_append(s["k"], s["v"], *cache, inv_freq=s["inv_freq"], layout=c["layout"], q=q, scales=scales, **weights)
    if c["kind"] == "append":
        return q, s["k_pages"], s["v_pages"], *scales
    o = ops.paged_attention(q, *cache, scales=scales, window=c["window"] or None, sinks=c["sinks"])
    return (o,) if c["kind"] == "attend" else (o, q, s["k_pages"], s["v_pages"], *scales)


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "read":
        return _plain_read(state)
    if kind == "attend":
        return (_plain_attend(state, state["q"]),)
    q = _plain_append(state)
    out = (_plain_attend(state, q),) if kind == "step" else ()
    return out + (q, state["k_pages"], state["v_pages"], state["k_scales"], state["v_scales"])


# ---- the definition in 64 bits, one sequence and one key head at a time
def _exact_turn(z, pos, f, layout, rotary, sign=1.0):
    first = torch.arange(rotary // 2, device=z.device) * (1 if layout == "half" else 2)
    second = first + (rotary // 2 if layout == "half" else 1)
    unit = torch.polar(torch.ones_like(f).expand(*pos.shape, -1), sign * pos.double().unsqueeze(-1) * f)
    w = torch.complex(z[..., first].contiguous(), z[..., second].contiguous()) * unit.unsqueeze(-2)
    out = z.clone()
    out[..., first], out[..., second] = w.real, w.imag
    return out


def _exact_normed(x, weight):
    z = x.detach().double()
    return z / torch.sqrt(z.square().sum(-1, keepdim=True) / z.shape[-1] + EPS) * weight.detach().double()


def _exact_8(x):
    """x / scale rounded to four significant bits (steps of 2^-9 below 2^-6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step


def _exact_norm(s):
    c = s["case"]
    args = (s["positions"], s["inv_freq"], c["layout"], c["rotary"])
    out = tuple(_exact_turn(_exact_normed(s[n], s[n + "_weight"]), *args) for n in "qk")
    if not c["backward"]:
        return out
    dx, dw = [], []
    for n in "qk":
        x = s[n].detach().double()
        g = _exact_turn(s["d" + n].double(), *args, sign=-1.0)
        size = torch.sqrt(x.square().sum(-1, keepdim=True) / c["dim"] + EPS)
        unit, h = x / size, g * s[n + "_weight"].detach().double()
        dw.append((g * unit).sum((0, 1, 2)))
        dx.append((h - unit * (h * unit).sum(-1, keepdim=True) / c["dim"]) / size)
    return out + tuple(dx) + tuple(dw)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    ps, Hkv, D = case["page"], case["kv_heads"], case["dim"]
    group, n0, outs, ks, vs = case["heads"] // Hkv, 0, [], [], []
    kc, vc = s["k_pages"].double(), s["v_pages"].double()  # as they are held
    if case["bits"] == 8:
        kc, vc = kc.view(-1, Hkv, ps // 16, 16, D), vc.transpose(3, 4).contiguous()
        sk, sv = (torch.exp2(s[n].view(torch.uint8).double() - 127.0) for n in ("k_scales", "v_scales"))
    else:
        kc, vc = kc.view(-1, Hkv, ps // 16, 16, D), vc.transpose(2, 3).reshape(-1, Hkv, ps // 16, 16, D)
        sk = sv = torch.ones(kc.shape[:3], dtype=torch.float64, device=kc.device)
    q = s["q"].double() if "q" in s else None
    appends = case["kind"] in ("append", "step")
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        rows = slice(n0, n0 + n)
        n0 += n
        pages = s["table"][b].long()
        pos = torch.arange(t - n, t, device=pages.device)
        if appends:
            new = []
            for name in "qk":
                x = _exact_normed(s[name][rows], s[name + "_weight"]) if case["norm"] else s[name][rows].double()
                new.append(_exact_turn(x, pos, s["inv_freq"], case["layout"], case["rotary"]))
            q[rows] = new[0]
            # whole blocks from the first one that gets a token: what they hold, with the new tokens in it
            lo, hi = (t - n) // 16, (t - 1) // 16 + 1
            blocks = torch.arange(lo, hi, device=pages.device)
            at = pages[blocks * 16 // ps], slice(None), blocks % (ps // 16)
            for c8, sc, x in ((kc, sk, new[1]), (vc, sv, s["v"][rows].double())):
                before, scale = c8[at], sc[at]                                  # [blocks, heads, 16, D], [blocks, heads]
                held = (before * scale[..., None, None]).transpose(1, 2).reshape(-1, Hkv, D)
                held[t - n - 16 * lo:t - 16 * lo] = x
                mine = torch.zeros(held.shape[0], dtype=torch.bool, device=x.device)
                mine[t - n - 16 * lo:t - 16 * lo] = True
                top = (held.abs() * mine[:, None, None]).view(-1, 16, Hkv, D).amax((1, 3))
                need = torch.exp2(torch.ceil(torch.log2((top / 448.0).clamp(min=2.0 ** -117))))
                if (t - n) % 16:
                    need[0] = torch.maximum(need[0], scale[0])
                as8 = _exact_8(held.view(-1, 16, Hkv, D) / need[:, None, :, None]).transpose(1, 2)
                valid = (torch.arange(held.shape[0], device=x.device) < t - 16 * lo).view(-1, 1, 16, 1)
                c8[at], sc[at] = torch.where(valid, as8, before), need
        if case["kind"] == "append":
            continue
        page = pages[torch.arange(t, device=pages.device) // ps]
        block, place = torch.arange(t, device=pages.device) % ps // 16, torch.arange(t, device=pages.device) % 16
        if case["kind"] == "read":
            ks.append(kc[page, :, block, place] * sk[page, :, block][..., None])
            vs.append(vc[page, :, block, place] * sv[page, :, block][..., None])
            continue
        # what the attention reads of the queries is what 16 bits hold
        held = q[rows].to(torch.bfloat16).double()
        far = pos[:, None] - torch.arange(t, device=q.device)
        seen = far >= 0
        if case["window"]:
            seen &= (far < case["window"]) | (torch.arange(t, device=q.device) < case["sinks"])
        o = torch.empty(n, case["heads"], D, dtype=torch.float64, device=q.device)
        for h in range(Hkv):
            k = kc[page, h, block, place] * sk[page, h, block][:, None]
            v = vc[page, h, block, place] * sv[page, h, block][:, None]
            for i in range(group):
                e = held[:, h * group + i] @ k.t() / math.sqrt(D)
                o[:, h * group + i] = torch.softmax(e.masked_fill(~seen, -math.inf), -1) @ v
        outs.append(o)
    if case["kind"] == "read":
        return torch.cat(ks), torch.cat(vs)
    out = () if case["kind"] == "append" else (torch.cat(outs),)
    if case["kind"] == "attend":
        return out
    return out + (q, kc.reshape(s["k_pages"].shape), vc.transpose(3, 4), sk, sv)
