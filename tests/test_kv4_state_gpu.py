"""What the 4-bit cache and its operators keep between calls, on the GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_kv4_gpu import _bf, _cache, _i32

from oracle import kv4 as ok

pytestmark = pytest.mark.gpu


def _attention(which, cuda, seed, lengths, head_dim=128, hq=32, hkv=4):
    """A call of one of the attentions over a cache of its own."""
    from mrun_b200.paged_kv4 import kv4_paged_attention, kv4_prefill_attention

    rng = np.random.default_rng(seed)
    pool, table, _ = _cache(rng, lengths, hkv, head_dim, head_dim, 64, cuda)
    q = _bf(ok.bf16(rng.standard_normal((len(lengths), hq, head_dim))), cuda)
    common = dict(group=head_dim, block_table=table, row_len=_i32(lengths, cuda))
    if which == "decode":
        return lambda: kv4_paged_attention(q, pool, max_total_tokens=max(lengths), **common)
    starts = _i32(list(range(len(lengths) + 1)), cuda)
    return lambda: kv4_prefill_attention(q, pool, q_starts=starts, **common)


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_captured_calls_outlive_the_streams_workspace(which, cuda):
    """Warm-up and two captures on one stream with default workspaces, a larger call on it, its old
    memory taken by others: the graphs, replayed on two other streams at once, still give the same."""
    small = _attention(which, cuda, 1, [4000], head_dim=64)
    large = _attention(which, cuda, 2, [3000] * 32, head_dim=128)
    want = small()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        small()
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(small())
        graphs.append(graph)
    with torch.cuda.stream(side):
        large()
    torch.cuda.synchronize()
    taken = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda) for _ in range(64)]
    streams = [torch.cuda.Stream(cuda) for _ in graphs]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(side):
            eager = small()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in (*outs, eager))
    assert all((t == 255).all() for t in taken)


def test_the_cache_passes_a_prefill_workspace_on(cuda):
    from mrun_b200.paged_kv4 import PagedKV4Cache

    c = PagedKV4Cache(num_layers=1, num_pages=40, kv_heads=2, head_dim=64, max_seqs=1, max_pages_per_seq=40, device=cuda)
    plan = c.plan_step(_i32([600], cuda), max_tokens=600)
    rng = np.random.default_rng(3)
    rows = _bf(rng.standard_normal((600, 12 * 64)), cuda)
    q = c.append(0, rows[:, 512:640], rows[:, 640:], plan, q_rows=rows[:, :512], num_heads=8)
    ws = torch.zeros(c.prefill_workspace_bytes(), dtype=torch.uint8, device=cuda)
    assert torch.equal(c.attend_prefill(0, q, plan, workspace=ws), c.attend_prefill(0, q, plan))
    with pytest.raises(ValueError, match="workspace too small"):
        c.attend_prefill(0, q, plan, workspace=ws[:100])
    c.check_errors()


def _dense(cuda, **kw):
    from mrun_b200.dense_engine import DenseConfig, DenseDecoder, DenseWeights

    cfg = DenseConfig(num_layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000)
    args = dict(max_batch=2, max_seq_len=192, device=cuda, max_prefill_tokens=192, kv_bits=4) | kw
    return cfg, DenseDecoder(DenseWeights.synthetic(cfg, cuda, seed=5), **args)


def test_capture_while_the_stream_is_busy(cuda):
    """The state that a capture's warm-up changes is copied before the warm-up runs, whatever is queued
    on the stream (here work of tens of milliseconds, with no word to the host in between)."""
    cfg, dec = _dense(cuda)
    ids = torch.arange(128) % cfg.vocab
    firsts = dec.prefill_batch([0, 1], [ids[:64], ids[:63]])  # the next token of row 0 takes a page
    dec.begin_decode(2, firsts, [64, 63])
    table, free = dec.kv.block_table.clone(), dec.kv.free_count.item()
    a = torch.randn(8192, 8192, device=cuda, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(40):
        a = torch.mm(a, a)
    dec.capture(2)
    assert dec.kv.lengths.tolist() == [64, 63] and dec.kv.free_count.item() == free
    assert torch.equal(dec.kv.block_table, table)
    assert dec.positions[:2].tolist() == [64, 63] and dec.row_len[:2].tolist() == [65, 64]
    assert torch.equal(dec.in_ids[:2], firsts)
    dec.check_errors()


def test_rows_that_are_cut_are_reported(cuda):
    """A row longer than max_total_tokens, or than its block-table row, is cut there, and says so."""
    from mrun_b200.paged_kv4 import KV_TOO_LONG, kv4_paged_attention, kv4_prefill_attention

    from test_paged_kv4_gpu import _check

    rng = np.random.default_rng(5)
    lengths = [40, 64, 100]
    pool, table, cache = _cache(rng, lengths, 2, 64, 32, 16, cuda)
    q = ok.bf16(rng.standard_normal((3, 4, 64)))
    ln, starts = _i32(lengths, cuda), _i32([0, 1, 2, 3], cuda)
    narrow = table[:, :4].contiguous()
    for table_, most, cut in ((table, 100, 100), (table, 64, 64), (table, 0, 0), (narrow, 100, 64)):
        for prefill in (False, True):
            if prefill and table_ is table:
                continue
            flag = torch.zeros(1, dtype=torch.int32, device=cuda)
            common = dict(group=32, block_table=table_, row_len=ln, error_flag=flag)
            got = (kv4_prefill_attention(_bf(q, cuda), pool, q_starts=starts, **common) if prefill else
                   kv4_paged_attention(_bf(q, cuda), pool, max_total_tokens=most, **common))
            assert flag.item() == (KV_TOO_LONG if cut < 100 else 0)
            for r in range(3):
                _check(got[r], *ok.attend(q[r], cache[r], min(lengths[r], cut), 64 ** -0.5))


def test_negative_lengths_are_none(cuda):
    from mrun_b200.paged_kv4 import kv4_paged_attention, kv4_prefill_attention

    rng = np.random.default_rng(6)
    pool, table, _ = _cache(rng, [40] * 4, 2, 64, 32, 16, cuda)
    q = _bf(ok.bf16(rng.standard_normal((4, 4, 64))), cuda)
    common = dict(group=32, block_table=table, row_len=_i32([-2 ** 31, -1, 0, 40], cuda))
    a = kv4_paged_attention(q, pool, max_total_tokens=40, **common)
    b = kv4_prefill_attention(q, pool, q_starts=_i32([0, 1, 2, 3, 4], cuda), **common)
    for out in (a, b):
        assert not out[:3].any() and out[3].any()


def test_queries_of_no_block_give_zeros(cuda):
    """Padding past the last block, every query after a plan that did not fit, and a call without rows."""
    from mrun_b200.paged_kv4 import KVStepPlan, PagedKV4Cache, kv4_prefill_attention

    rng = np.random.default_rng(7)
    for head_dim, tokens in ((64, 40), (128, 3000)):
        c = PagedKV4Cache(num_layers=1, num_pages=4, kv_heads=2, head_dim=head_dim, max_seqs=2, max_pages_per_seq=2,
                          device=cuda)
        q = _bf(rng.standard_normal((tokens, 6, head_dim)), cuda)
        rows = _bf(rng.standard_normal((tokens, 4 * head_dim)), cuda)
        plan = KVStepPlan.empty(2, tokens, cuda)
        for new, fits in (([9, 21], True), ([0, 0], True), ([9, 40], False)):
            c.plan_step(_i32(new, cuda), max_tokens=tokens, out=plan)
            c.append(0, rows[:, :2 * head_dim], rows[:, 2 * head_dim:], plan)
            used = sum(new) if fits else 0
            poison = torch.full_like(q, float("nan"))  # what the outputs' memory held before
            del poison
            got = c.attend_prefill(0, q, plan)
            assert got[:used].any(-1).all() and not got[used:].any()
            kept = c.attend_prefill(0, q, plan, out=torch.full_like(q, 7))
            assert torch.equal(kept[:used], got[:used]) and (kept[used:] == 7).all()
            if fits:
                c.check_errors()
            c.release(_i32([0, 1], cuda))
        none = _i32([], cuda)
        poison = torch.full_like(q, float("nan"))
        del poison
        got = kv4_prefill_attention(q, c.pool[0], group=head_dim, block_table=c.block_table, q_starts=_i32([0], cuda),
                                    row_len=none)
        assert not got.any()


@pytest.mark.parametrize("tokens", [1, 37])
@pytest.mark.parametrize("head_dim,group,interleaved", [(64, 32, True), (128, 128, False)])
def test_append_of_separate_projections(head_dim, group, interleaved, tokens, cuda):
    """Queries, keys and values of one fused row, of three tensors, and of slices of wider ones."""
    from mrun_b200.paged_kv4 import rope_kv4_append

    rng = np.random.default_rng(head_dim)
    hq, hkv = 7, 2
    fused = _bf(rng.standard_normal((tokens, (hq + 2 * hkv) * head_dim)), cuda)
    parts = fused.split([hq * head_dim, hkv * head_dim, hkv * head_dim], 1)
    apart = [x.contiguous() for x in parts]
    wide = [torch.cat([x, torch.zeros(tokens, 4 * (i + 1), dtype=x.dtype, device=cuda)], 1)[:, :x.shape[1]]
            for i, x in enumerate(parts)]
    cos, sin = (torch.randn(tokens, head_dim // 2, device=cuda) for _ in range(2))
    at = _i32(list(range(tokens)), cuda)
    results = []
    for q, k, v in (parts, apart, wide, (apart[0], parts[1], wide[2])):
        pool = torch.zeros(3, hkv, 1, ok.block_bytes(head_dim, group), dtype=torch.uint8, device=cuda)
        out = rope_kv4_append(k, v, pool, group=group, head_dim=head_dim, slots=at, positions=at, q_in=q, num_heads=hq,
                              rope=(cos, sin), interleaved=interleaved)
        results.append((out, pool))
    assert results[0][0].any() and results[0][1].any()
    for out, pool in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(pool, results[0][1])


def test_prefill_leaves_the_values_of_its_tokens(cuda):
    """next_val holds the logit of each prefilled sequence's next token, as with a bf16 cache."""
    from mrun_b200.dense_qstore_cuda import qrow_argmax

    cfg, dec = _dense(cuda)
    ids = torch.arange(100) * 3 % cfg.vocab
    dec.next_val.fill_(float("nan"))
    tokens = dec.prefill_batch([1, 0], [ids[:30], ids[30:]])
    last = dec.buf["normed"][[29, 99]]
    _, value, logits = qrow_argmax(dec.w.head.codes, dec.w.head.scales, last)
    assert torch.equal(dec.next_val[[1, 0]], value) and dec.next_val.isfinite().all()
    assert torch.equal(dec.next_ids[[1, 0]], tokens)
    dec.next_val.fill_(float("nan"))
    dec.prefill(0, ids[:5])
    assert dec.next_val[0].isfinite() and dec.next_val[1].isnan()


def test_two_generations_share_a_small_pool(cuda):
    """A reservation outlives its generation until the sequence is released."""
    cfg, dec = _dense(cuda, num_pages=3)
    ids = torch.arange(20) % cfg.vocab
    dec.generate(ids, 60)  # 80 tokens reserved: 2 pages
    dec.prefill(1, ids)
    with pytest.raises(MemoryError):
        dec.reserve(1, 65)
    dec.release(0)
    dec.reserve(1, 65)
    dec.check_errors()


def test_the_largest_plan(cuda):
    """As many requests and sequences as a step takes: the most shared memory that the clusters need."""
    from mrun_b200.paged_kv4 import kv_plan_step

    rows, seqs, page = 8192, 1 << 18, 16
    rng = np.random.default_rng(8)
    new = rng.integers(0, 12, rows)
    order = rng.permutation(seqs)[:rows]
    lengths = rng.integers(0, 2 * page, seqs)
    have, need = -(-lengths[order] // page), -(-(lengths[order] + new) // page)
    table = np.full((seqs, 4), -1, np.int32)
    ids = rng.permutation(2 * seqs + int((need - have).sum())).astype(np.int32)
    table[:, :2] = ids[:2 * seqs].reshape(seqs, 2)
    table[np.arange(4) >= -(-lengths // page)[:, None]] = -1
    free = ids[2 * seqs:]
    tb = torch.from_numpy(table).to(cuda)
    ln, fc = _i32(lengths.tolist(), cuda), _i32([len(free)], cuda)
    flag = _i32([0], cuda)
    p = kv_plan_step(_i32(new.tolist(), cuda), ln, tb, torch.from_numpy(free).to(cuda), fc, row_seq=_i32(order.tolist(), cuda),
                     page_size=page, max_tokens=int(new.sum()), error_flag=flag)
    assert flag.item() == 0 and fc.item() == 0
    taken = 0
    for r in range(rows):
        for j in range(have[r], need[r]):
            table[order[r], j] = free[len(free) - 1 - taken]
            taken += 1
    row = np.repeat(np.arange(rows), new)
    pos = lengths[order][row] + np.arange(new.sum()) - (np.cumsum(new) - new)[row]
    assert np.array_equal(tb.cpu().numpy(), table)
    assert np.array_equal(p.positions.cpu().numpy(), pos)
    assert np.array_equal(p.token_rows.cpu().numpy(), order[row])
    assert np.array_equal(p.slots.cpu().numpy(), table[order[row], pos // page] * page + pos % page)
    lengths[order] += new
    assert np.array_equal(ln.cpu().numpy(), lengths)


def test_captured_projections_outlive_the_streams_workspace(cuda):
    """The same of the default workspace that row-quantised projections split their tiles through."""
    from mrun_b200.dense_qstore_cuda import qrow_linear

    gen = torch.Generator(device=cuda).manual_seed(3)

    def page(rows, k):
        return (torch.randint(-127, 128, (rows, k), generator=gen, device=cuda, dtype=torch.int8),
                torch.rand(rows, generator=gen, device=cuda) / 127)

    x = torch.randn(1, 4096, generator=gen, device=cuda).to(torch.bfloat16)
    small, large = page(3584, 4096), page(40000, 4096)
    want = qrow_linear(*small, x)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qrow_linear(*small, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = qrow_linear(*small, x)
    with torch.cuda.stream(side):
        qrow_linear(*large, x)
    torch.cuda.synchronize()
    taken = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda) for _ in range(16)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all((t == 255).all() for t in taken)
