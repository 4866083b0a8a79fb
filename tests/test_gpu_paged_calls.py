"""Calls of the rotary positions and the paged cache that the other files do not make: outputs on top of the
tables that a call reads, gradients and versions around calls in place, schemas and fake results of the ops."""
import pytest
import torch

from helpers import dev
from test_gpu_paged import LONG, Batch, attend64, check_attention, few, gen

pytestmark = pytest.mark.gpu


def test_outputs_on_top_of_the_tables_are_refused(pkg):
    """block_table, kv_lens, cu_q and inv_freq are read while pages and outputs are written."""
    ops = pkg.ops
    kp, vp, table, lens, cu = Batch([2], [20], 16, 2, 64).gpu()
    cache = (kp, vp, table, lens, cu)
    x = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=dev())
    f = ops.rotary_frequencies(64)[0].to(dev())

    def inside(t, like):  # like's size and type, in t's memory
        return t.view(-1).view(like.dtype)[:like.numel()].view(like.shape).copy_(like)

    for given in (kp, vp):
        for i in (2, 3, 4):
            with pytest.raises(RuntimeError, match="prunepath.*overlaps"):
                ops.kv_append(x, x.clone(), *cache[:i], inside(given, cache[i]), *cache[i + 1:])
        with pytest.raises(RuntimeError, match="prunepath.*overlaps"):
            ops.kv_append(x, x.clone(), *cache, inside(given, f))
    out = torch.zeros_like(x)
    for i in (2, 3, 4):
        on = (*cache[:i], inside(out, cache[i]), *cache[i + 1:])
        with pytest.raises(RuntimeError, match="prunepath.*overlaps"):
            ops.paged_attention(x, *on, out=out)
        with pytest.raises(RuntimeError, match="prunepath.*overlaps"):
            ops.kv_append(x, x.clone(), *on, q=x.clone(), q_out=out)
    with pytest.raises(RuntimeError, match="prunepath.*overlaps"):
        ops.kv_append(x, x.clone(), *cache, inside(out, f), q=x.clone(), q_out=out)


def test_opcheck(pkg):
    """Schemas, registrations and fake results of the six ops, with and without gradients where there are any."""
    from torch.library import opcheck
    t = pkg._lib.torch_ops()
    kp, vp, table, lens, cu = Batch([3, 2], [20, 5], 16, 2, 64).gpu()
    cache = (kp, vp, table, lens, cu)
    f = pkg.ops.rotary_frequencies(64)[0].to(dev())
    q, k, v = (torch.randn(5, h, 64, device=dev(), dtype=torch.bfloat16) for h in (4, 2, 2))
    pos = torch.arange(5, device=dev())
    x = torch.randn(5, 3, 64, device=dev())
    for op, args in ((t.rotary, (x, pos, f)), (t.rotary, (x.clone().requires_grad_(), pos, f, "interleaved", 1.5, True)),
                     (t.rotary, (x.bfloat16().transpose(1, 2).contiguous().transpose(1, 2), pos.int(), f)),
                     (t.kv_append, (k, v, *cache, f)), (t.kv_append, (k.float(), v.float(), *cache)),
                     (t.kv_append_q, (q, k, v, *cache, f, "interleaved", 1.5)),
                     (t.kv_append_q_into, (q, torch.zeros_like(q), k, v, *cache, f)),
                     (t.paged_attention, (q, *cache, 0.1)), (t.paged_attention_into, (q, *cache, 0.1, torch.zeros_like(q)))):
        print(f"opcheck {op}", flush=True)
        opcheck(op, args)


@pytest.mark.parametrize("new,total,heads,kv_heads,dim", [
    ([1] * 20, [3000, 1, 17, 384, 385, 1023, 1025, 2047, 2600, 40, 700, 129, 2049, 5, 64, 1500, 1, 900, 3001, 333], 4, 2, 128),
    ([2] * 7, [2, 5000, 100, 2048, 4097, 33, 1024], 8, 1, 64), ([1], [5000], 12, 12, 128), ([150], [3000], 2, 2, 128),
    ([1500], [1500], 2, 1, 128), ([40, 30, 90], [2500, 30, 700], 6, 3, 64)])
def test_tables_wider_than_their_sequences(pkg, new, total, heads, kv_heads, dim):
    """A table of 65536 tokens and one as long as the longest sequence: several ranges and the join in both."""
    for extra in (0, 65536 // 32 - -(-max(total) // 32)):
        b = Batch(new, total, 32, kv_heads, dim, seed=dim, extra=extra)
        q = (1.5 * torch.randn(b.n, heads, dim, generator=gen(3))).to(torch.bfloat16)
        rows = slice(0, b.n) if b.n < 200 else slice(b.n - 40, b.n)
        got = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
        if b.n >= 200:  # (the last rows of a long prompt stand for all)
            b.rows = lambda b=b: ((r, s, p) for r, s, p in Batch.rows(b) if r >= rows.start)
        o, big = attend64(b, q)
        check_attention(got[rows], o[rows], big[rows], few(b, heads, kv_heads))


@pytest.mark.parametrize("singles,chunk,heads,kv_heads,dim", [(40, 200, 2, 2, 128), (64, 130, 8, 2, 64), (100, 33, 12, 12, 128)])
def test_a_chunk_among_single_tokens(pkg, singles, chunk, heads, kv_heads, dim):
    """The step of a server: single tokens of many sequences and one sequence's chunk."""
    new = [1] * (singles // 2) + [chunk] + [1] * (singles - singles // 2)
    total = [n + (37 * i) % 301 for i, n in enumerate(new)]
    b = Batch(new, total, 16, kv_heads, dim, seed=chunk, extra=4096)
    q = (1.5 * torch.randn(b.n, heads, dim, generator=gen(chunk))).to(torch.bfloat16)
    check_attention(pkg.ops.paged_attention(q.to(dev()), *b.gpu()), *attend64(b, q), False)


@pytest.mark.parametrize("new", [[1] * 30 + [100] + [1] * 40, [4] * 66, [2] * 70, [1] * 64 + [1100]], ids=len)
def test_append_of_uneven_batches(pkg, new):
    """Many sequences with few tokens each, and a chunk among single tokens: keys and values as they are, without a
    rotation, in their places and nowhere else."""
    total = [n + (29 * i) % 90 for i, n in enumerate(new)]
    b = Batch(new, total, 16, 5, 64, seed=len(new))
    kv = torch.randn(2, b.n + 3, 5, 64, generator=gen(7)).to(torch.bfloat16)
    kp, vp, table, lens, cu = b.gpu()
    pkg.ops.kv_append(kv[0].to(dev()), kv[1].to(dev()), kp, vp, table, lens, cu)
    for row, s, p in b.rows():
        at = b.place(s, p)
        b.k[at[0], :, at[1]], b.v[at[0], :, :, at[1]] = kv[0, row], kv[1, row]
    assert torch.equal(kp.cpu(), b.k) and torch.equal(vp.cpu(), b.v)


@pytest.mark.parametrize("seqs", [255, 256, 257, 300])
def test_many_sequences_in_large_tiles(pkg, seqs):
    """Around the borders of 256 sequences with tiles of 128 rows: chunks, single tokens, empty sequences and rows
    of no sequence."""
    new = [(i * 7) % 4 for i in range(seqs)]
    for s in (0, 63, 64, 254, 255, 256, 257, 299):
        if s < seqs:
            new[s] = 9 + s % 30
    total = [n + i % 40 for i, n in enumerate(new)]
    b = Batch(new, total, 16, 1, 64, seed=seqs, extra=LONG // 16 // 64)
    assert not few(b, 16, 1)
    q = torch.randn(b.n + 5, 16, 64, generator=gen(seqs)).to(torch.bfloat16)
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu())
    check_attention(got[:b.n], *attend64(b, q[:b.n]), False)
    assert bool((got[b.n:] == 0).all())


@pytest.mark.parametrize("new,total,heads,kv_heads,dim,ranges", [
    ([300] * 4, [1900, 300, 1100, 650], 24, 12, 128, 2), ([700, 1, 600], [1300, 900, 2100], 12, 12, 128, 4),
    ([900] * 3, [1000, 2500, 900], 8, 8, 64, 4), ([1000], [2600], 12, 12, 128, 5)])
def test_large_tiles_in_a_few_ranges(pkg, new, total, heads, kv_heads, dim, ranges):
    """2 to 8 ranges of a tile, joined by the rows' own threads. The last rows of every sequence, which attend most,
    stand for all."""
    page = 64
    b = Batch(new, total, page, kv_heads, dim, seed=ranges, extra=2 + LONG // page)
    each = (b.n * (heads // kv_heads) // 128 + len(new)) * kv_heads
    slots = (3 if dim == 64 else 2) * 256
    assert not few(b, heads, kv_heads) and ranges == (slots // each if slots // each >= 4 else -(-slots // each))
    q = (1.5 * torch.randn(b.n, heads, dim, generator=gen(5))).to(torch.bfloat16)
    got = pkg.ops.paged_attention(q.to(dev()), *b.gpu()).cpu()
    rows = [(r, s, p) for r, s, p in b.rows() if p >= b.total[s] - 6 or p == b.total[s] - b.new[s]]
    b.rows = lambda: rows
    o, big = attend64(b, q)
    at = [r for r, _, _ in rows]
    check_attention(got[at], o[at], big[at], False)
