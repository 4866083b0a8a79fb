"""Refusals and registrations of the rotary positions and the paged cache, without a GPU: sizes that
wrap, outputs that overlap what a call reads, gradients and tangents that a traced call would lose, versions of
what a call writes, shapes of fake tensors."""
import pytest

from conftest import import_pkg
from test_paged_index_cpu import _append, _attend, _lib


@pytest.mark.parametrize("kw", [dict(n=1 << 62), dict(n=1 << 60, Hq=16, Hkv=16), dict(n=(1 << 63) - 1), dict(n=(1 << 62) + 1)])
def test_sizes_that_wrap_are_refused(kw):
    assert _append(**kw) == 3 and "pp_kv_append" in _lib().pp_last_error().decode()
    assert _attend(**kw) == 3 and "pp_paged_attention" in _lib().pp_last_error().decode()


@pytest.mark.parametrize("n,seqs,maxp,page,hq,hkv,d", [(1 << 62, 2, 8, 16, 4, 2, 128), (1 << 60, 1, 64, 16, 16, 16, 128),
                                                       (4, 2, 1 << 30, 1 << 30, 4, 2, 128), (4, 2, 8, 16, 4, 3, 128),
                                                       (4, 1 << 30, 8, 16, 4, 2, 64), (4, 2, 8, 16, 1 << 30, 1 << 30, 64)])
def test_workspace_of_sizes_that_are_refused(n, seqs, maxp, page, hq, hkv, d):
    """None: the call itself says what is wrong with them."""
    assert _lib().pp_paged_attention_workspace_bytes(n, seqs, maxp, page, hq, hkv, d) == 0


# ------------------------------------------------------------------ gradients and tangents
def _fake(device="meta", seqs=2, n=5, heads=4, kv=2, dim=64, page=16):
    """(ops, q, k, v, cache, inv_freq) of a call, on a device without values."""
    import torch
    m = dict(device=device)
    bf = dict(dtype=torch.bfloat16, **m)
    cache = (torch.empty(9, kv, page, dim, **bf), torch.empty(9, kv, dim, page, **bf),
             torch.empty(seqs, 3, dtype=torch.int32, **m), torch.empty(seqs, dtype=torch.int32, **m),
             torch.empty(seqs + 1, dtype=torch.int32, **m))
    return (import_pkg()._lib.torch_ops(), torch.empty(n, heads, dim, **bf), torch.empty(n, kv, dim, **bf),
            torch.empty(n, kv, dim, **bf), cache, torch.empty(dim // 2, dtype=torch.float64, **m))


def _calls():
    """(name, call(ops, q, k, v, cache, inv_freq)) of every op for inference."""
    import torch
    return {"kv_append": lambda t, q, k, v, c, f: t.kv_append(k, v, *c, f),
            "kv_append_q": lambda t, q, k, v, c, f: t.kv_append_q(q, k, v, *c, f),
            "kv_append_q_into": lambda t, q, k, v, c, f: t.kv_append_q_into(q, torch.empty_like(q), k, v, *c, f),
            "paged_attention": lambda t, q, k, v, c, f: t.paged_attention(q, *c, 0.1),
            "paged_attention_into": lambda t, q, k, v, c, f: t.paged_attention_into(q, *c, 0.1, torch.empty_like(q))}


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("name", list(_calls()))
def test_gradients_are_refused_without_a_gpu(name, which):
    """Whichever argument (q, k, v, k_pages, inv_freq) requires one, if the call takes it; not under no_grad."""
    import torch
    t, q, k, v, cache, f = _fake()
    (q, k, v, cache[0], f)[which].requires_grad_()
    takes = {"kv_append": (1, 2, 3, 4), "paged_attention": (0, 3), "paged_attention_into": (0, 3)}.get(name, range(5))
    if which in takes:
        with pytest.raises(RuntimeError, match=f"prunepath.{name}: inference only"):
            _calls()[name](t, q, k, v, cache, f)
    with torch.no_grad():
        _calls()[name](t, q, k, v, cache, f)


@pytest.mark.parametrize("name", list(_calls()))
def test_tangents_are_refused(name):
    import torch
    import torch.autograd.forward_ad as fw
    t, q, k, v, cache, f = _fake()
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.empty_like(x))  # noqa: E731
        for args in ((dual(q), k, v, cache, f), (q, dual(k), v, cache, f), (q, k, v, (cache[0], dual(cache[1]), *cache[2:]), f)):
            if name.startswith("paged") and args[1] is not k or name == "kv_append" and args[0] is not q:
                continue
            with torch.no_grad(), pytest.raises(RuntimeError, match=f"prunepath.{name}: .*forward-mode"):
                _calls()[name](t, *args)


def test_tangents_of_the_rotation_are_refused():
    """Of x and of the frequencies alike."""
    import torch
    import torch.autograd.forward_ad as fw
    t, q, _, _, _, f = _fake()
    pos = torch.empty(5, dtype=torch.int64, device="meta")
    with fw.dual_level():
        for x, g in ((fw.make_dual(q, torch.empty_like(q)), f), (q, fw.make_dual(f, torch.empty_like(f)))):
            with pytest.raises(RuntimeError, match="prunepath.rotary: no forward-mode"):
                t.rotary(x, pos, g)
    assert t.rotary(q, pos, f).shape == q.shape


def test_gradients_are_refused_in_compiled_code():
    """A traced call meets the refusal as an eager one does: no result without its gradient."""
    import torch
    t, q, k, v, cache, f = _fake()
    p = torch.empty(64, 64, dtype=torch.bfloat16, device="meta", requires_grad=True)
    w = torch.empty(64, 3, dtype=torch.bfloat16, device="meta", requires_grad=True)
    attend = lambda q, p, w: (t.paged_attention(q @ p, *cache, 0.1) @ w).sum()  # noqa: E731
    append = lambda q, p, w: (t.kv_append_q(q @ p, k, v, *cache, f) @ w).sum()  # noqa: E731
    for fn in (attend, append):
        torch._dynamo.reset()
        with pytest.raises(Exception, match="inference only"):
            torch.compile(fn, backend="aot_eager")(q, p, w)
    with torch.no_grad():
        torch._dynamo.reset()
        assert torch.compile(attend, backend="aot_eager")(q, p, w).shape == ()


# ------------------------------------------------------------------ versions
def test_written_arguments_count_as_changed():
    """Each op bumps the version of what its schema says it writes, and of nothing else."""
    import torch
    t, q, k, v, cache, f = _fake()
    out = torch.empty_like(q)
    every = [q, k, v, *cache, f, out]
    for op, args in ((t.kv_append, (k, v, *cache, f)), (t.kv_append_q, (q, k, v, *cache, f)),
                     (t.kv_append_q_into, (q, out, k, v, *cache, f)), (t.paged_attention, (q, *cache, 0.1)),
                     (t.paged_attention_into, (q, *cache, 0.1, out))):
        schema = op.default._schema.arguments
        writes = [a for a, s in zip(args, schema) if s.alias_info is not None and s.alias_info.is_write]
        before = [x._version for x in every]
        op(*args)
        for x, old in zip(every, before):
            assert x._version == old + any(x is w for w in writes), op


def test_a_backward_that_saved_what_a_call_overwrote_raises():
    import torch
    t, q, k, v, cache, f = _fake()
    w = torch.empty_like(q, requires_grad=True)
    for call in (lambda b: t.paged_attention_into(q, *cache, 0.1, b), lambda b: t.kv_append_q_into(q, b, k, v, *cache, f)):
        buf = torch.empty_like(q)
        y = (buf * w).sum()
        call(buf)
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    y = (cache[0] * torch.empty_like(cache[0], requires_grad=True)).sum()
    t.kv_append(k, v, *cache, f)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()


def test_inference_tensors_are_written_as_before():
    """Tensors made in inference mode have no version: a call outside of it writes them all the same."""
    import torch
    with torch.inference_mode():
        t, q, k, v, cache, f = _fake()
        t.kv_append(k, v, *cache, f)
    with torch.no_grad():
        t.kv_append(k, v, *cache, f)
        t.paged_attention_into(q, *cache, 0.1, torch.empty_like(q))


def test_what_the_expert_ops_write_counts_as_changed():
    """The in-place ops of the experts: workspaces, outputs and routing outputs, as their schemas say."""
    import torch
    t = import_pkg()._lib.torch_ops()
    m = dict(device="meta")
    E, G, H, N = 16, 32, 256, 5
    u8 = lambda: torch.empty(4096, dtype=torch.uint8, **m)  # noqa: E731
    x, rp, packed = torch.empty(N, H, **m), torch.empty(E, H, **m), u8()
    out, logits, mask = torch.empty(N, H, dtype=torch.bfloat16, **m), torch.empty(N, E, **m), torch.empty(N, E, dtype=torch.uint8, **m)
    common = (rp, None, E, G, 0.7, packed)
    for op, args in ((t.decode_workspace_init, (u8(), H, E)), (t.moe_decode, (x[0], *common, u8())),
                     (t.moe_decode_into, (x[0], *common, u8(), out[:1])), (t.moe_decode_batch, (x, *common, u8(), u8())),
                     (t.moe_decode_batch_into, (x, *common, u8(), u8(), out, logits, mask)),
                     (t.moe_decode_batch_into, (x, *common, u8(), u8(), out)),
                     (t.moe_prefill_into, (x, *common, u8(), out, logits, mask)), (t.moe_prefill_into, (x, *common, u8(), out))):
        schema = op.default._schema.arguments
        tensors = [(a, s.alias_info is not None and s.alias_info.is_write) for a, s in zip(args, schema) if torch.is_tensor(a)]
        before = [a._version for a, _ in tensors]
        op(*args)
        assert [a._version - b for (a, _), b in zip(tensors, before)] == [int(w) for _, w in tensors], op


# ------------------------------------------------------------------ threads
def test_backwards_of_one_graph_in_several_threads():
    """Threads that run the backward of one graph, which its first one releases: each has its gradient or is told
    that the graph is used up, and none meets what another is releasing."""
    import threading
    import torch
    t, q, _, _, _, f = _fake()
    pos = torch.empty(5, dtype=torch.int64, device="meta")
    x = q.detach().requires_grad_()
    g = torch.empty_like(q)
    for keep in (True, False):
        for _ in range(30):
            y, odd, got = t.rotary(x, pos, f), [], []
            ready = threading.Barrier(4)

            def run():
                ready.wait()
                try:
                    for _ in range(3):
                        got.append(torch.autograd.grad(y, x, g, retain_graph=keep)[0].shape)
                except RuntimeError as e:
                    if "second time" not in str(e):
                        odd.append(e)

            threads = [threading.Thread(target=run) for _ in range(4)]
            for th in threads:
                th.start()
            for th in threads:
                th.join()
            assert not odd and got and all(s == x.shape for s in got)
            assert not keep or len(got) == 12


# ------------------------------------------------------------------ shapes of fake tensors
def test_fake_calls_check_what_real_ones_do():
    import torch
    t, q, k, v, cache, f = _fake()
    kp, vp, table, lens, cu = cache
    pos, i32 = torch.empty(5, dtype=torch.int64, device="meta"), dict(dtype=torch.int32, device="meta")
    e = torch.empty_like
    bad = {"positions of another length": lambda: t.rotary(q, pos[:4], f), "float positions": lambda: t.rotary(q, pos.float(), f),
           "more pairs than channels": lambda: t.rotary(q[..., :32], pos, f), "float frequencies": lambda: t.rotary(q, pos, f.float()),
           "no pairs": lambda: t.rotary(q, pos, f[:0]), "a layout": lambda: t.rotary(q, pos, f, "other"),
           "half precision": lambda: t.rotary(q.half(), pos, f), "two dimensions": lambda: t.rotary(q[0], pos, f),
           "heads on no multiple": lambda: t.paged_attention(q[:, :3].contiguous(), *cache, 0.1),
           "channels": lambda: t.paged_attention(torch.empty(5, 3, 96, dtype=q.dtype, device="meta"), *cache, 0.1),
           "head size": lambda: t.paged_attention(torch.empty(5, 2, 96, dtype=q.dtype, device="meta"), kp.new_empty(9, 2, 16, 96),
                                                  vp.new_empty(9, 2, 96, 16), table, lens, cu, 0.1),
           "float queries": lambda: t.paged_attention(q.float(), *cache, 0.1),
           "pages as they are": lambda: t.paged_attention(q, kp, kp, table, lens, cu, 0.1),
           "offsets": lambda: t.paged_attention(q, kp, vp, table, lens, cu[:2], 0.1),
           "a long table": lambda: t.paged_attention(q, kp, vp, table.long(), lens, cu, 0.1),
           "an output": lambda: t.paged_attention_into(q, *cache, 0.1, e(q)[:, :2]),
           "a float output": lambda: t.paged_attention_into(q, *cache, 0.1, q.float()),
           "sequences": lambda: t.kv_append(k, v, kp, vp, table, torch.empty(3, **i32), torch.empty(4, **i32), f),
           "values": lambda: t.kv_append(k, v[:4], *cache, f), "types": lambda: t.kv_append(k, v.float(), *cache, f),
           "heads of the cache": lambda: t.kv_append(k[:, :1], v[:, :1], *cache, f),
           "pairs": lambda: t.kv_append(k, v, *cache, f[:4]), "a layout of the append": lambda: t.kv_append(k, v, *cache, f, "other"),
           "query rows": lambda: t.kv_append_q(q[:4], k, v, *cache, f), "query type": lambda: t.kv_append_q(q.float(), k, v, *cache, f),
           "query output": lambda: t.kv_append_q_into(q, e(q).transpose(0, 1), k, v, *cache, f)}
    for what, call in bad.items():
        with pytest.raises(RuntimeError, match="prunepath"):
            call()
            print("not refused:", what)


def test_fake_calls_with_symbolic_sizes():
    """Tokens, sequences and the table's width may be symbols; the result follows them."""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    t, q, k, v, cache, f = _fake()

    def step(q, k, v, kp, vp, table, lens, cu, f):
        return t.paged_attention(t.kv_append_q(q, k, v, kp, vp, table, lens, cu, f), kp, vp, table, lens, cu, 0.1)

    with torch.no_grad():
        gm = make_fx(step, tracing_mode="symbolic")(q, k, v, *cache, f)
    out = [n.meta["val"] for n in gm.graph.nodes if n.op == "call_function" and "paged_attention" in str(n.target)]
    assert len(out) == 1 and not isinstance(out[0].shape[0], int) and out[0].dtype == torch.bfloat16


# ------------------------------------------------------------------ ranges of the attention's tiles
@pytest.mark.parametrize("n,seqs,hq,hkv,d", [(1, 1, 12, 12, 128), (64, 64, 12, 12, 128), (256, 256, 32, 8, 128),
                                             (4096, 256, 12, 12, 128), (4096, 256, 32, 32, 128), (2048, 1, 12, 12, 64),
                                             (1736, 9, 24, 4, 128), (65536, 4096, 64, 8, 128)])
def test_workspace_does_not_follow_the_tables_width(n, seqs, hq, hkv, d):
    """A range of every row, and of all together at most 16 tiles of 16 rows (or two of 128) for each of 256 CUs: no
    table of any width asks for more."""
    rows = n * hq
    most = rows * (4 * (d + 2) * 2 + 4) + 256 * 16 * 16 * 4 * (d + 2)
    for pages in (8, 64, 512, 4096, 65536):
        assert 0 <= _lib().pp_paged_attention_workspace_bytes(n, seqs, pages, 16, hq, hkv, d) <= most


def test_ranges_by_length_cover_the_tokens():
    """The cut of csrc/attention.hip restated: any bounds, any lengths; never more ranges than the workspace has."""
    up = lambda x, y: -(-x // y)  # noqa: E731
    for splits in (1, 2, 7, 21, 64):
        for base, behind in ((1, 1), (2, 2), (5, 4), (21, 21), (64, 64), (256, 0)):
            for nt in (1, 31, 128, 384, 385, 511, 513, 1024, 2049, 8191, 30011, 65537, 1 << 20):
                for few, far in ((True, False), (False, False), (False, True)):
                    cut = (1 if nt <= 384 else max(min(base, up(nt, 128)), nt >> 10)) if few else min(behind if far else base, up(nt, 512))
                    cut = max(1, min(cut, splits))
                    per = up(up(nt, cut), 128) * 128
                    ns = up(nt, per)
                    assert 1 <= ns <= splits and (ns - 1) * per < nt <= ns * per


def test_items_of_16_row_tiles_are_each_taken_once():
    """Workgroups -> (split, tile, head) of csrc/attention.hip restated."""
    for tiles, heads, splits in ((1, 1, 1), (1, 3, 4), (2, 12, 21), (18, 12, 8), (65, 4, 8), (70, 1, 11), (9, 5, 64)):
        items, seen = (tiles - 1) * heads, set()
        for b in range(tiles * heads * splits):
            if b < items * splits:
                split = b // items
                item = (b - split * items + (split * (items - 4) & 7)) % items
            else:
                split, item = (b - items * splits) // heads, items + (b - items * splits) % heads
            seen.add((split, item // heads, item % heads))
        assert len(seen) == tiles * heads * splits and max(s for s, _, _ in seen) == splits - 1
        assert max(t for _, t, _ in seen) == tiles - 1
