"""The 4-bit cache's ops as an engine runs them: block tables from lengths, the new keys and values into the cache,
attention over it, step after step; eager, through torch.ops and in a captured graph.

The cache is held to the definition of the codes (equal bytes), the attention to the formula in 64 bits within the bounds
of test_mxfp4_attention.py.
"""
import pytest
import torch

import flaggems_vllm as fv

from .test_mxfp4_attention import BF, DEV, FP, compare, reference
from .test_mxfp4_kv_cache import empty_cache, parts, quantise


class Engine:
    """Requests that grow, their keys and values kept aside on the way into the cache."""

    def __init__(self, seed, reqs, blocks, width, heads, kv_heads, dim, page, dtype):
        g = self.g = torch.Generator().manual_seed(seed)
        self.reqs, self.heads, self.kv_heads, self.dim, self.page, self.dtype = reqs, heads, kv_heads, dim, page, dtype
        self.cache = empty_cache(blocks, kv_heads, page, dim, 0xFF)
        self.table = torch.full((reqs, width), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(blocks, generator=g).to(torch.int32).to(DEV)
        self.num_free = torch.tensor([blocks], dtype=torch.int32, device=DEV)
        self.context = torch.zeros(reqs, dtype=torch.int32, device=DEV)
        self.kept = [(torch.zeros(0, kv_heads, dim, dtype=dtype, device=DEV),) * 2 for _ in range(reqs)]

    def rows(self, n, heads):
        return torch.randn(n, heads, self.dim, generator=self.g).to(self.dtype).to(DEV)

    def step(self, q, k, v, query, rows, ops=fv, **kw):
        """One step in `rows` rows; what it returns is of the device."""
        start, lens, positions, slots, self.num_free = ops.build_block_tables(
            self.context, query, self.table, self.free, self.num_free, self.page, rows, -1)
        ops.mxfp4_kv_quant_and_cache(k, v, self.cache, slots)
        out, lse = ops.mxfp4_paged_attention(q, self.cache, self.table, lens, self.dim ** -0.5, query_start_loc=start, **kw)
        return start, lens, positions, out, lse

    def check(self, query, k, v, start, lens, positions, out, lse, q, window=None):
        at = 0
        for b, n in enumerate(query):
            old_k, old_v = self.kept[b]
            assert positions[at:at + n].tolist() == list(range(len(old_k), len(old_k) + n))
            self.kept[b] = torch.cat([old_k, k[at:at + n]]), torch.cat([old_v, v[at:at + n]])
            at += n
        assert start.tolist() == [sum(query[:i]) for i in range(len(query) + 1)]
        assert lens.tolist() == [len(kk) for kk, _ in self.kept]
        seen = set()
        for b, (kk, vv) in enumerate(self.kept):
            if len(kk) == 0:
                continue
            pos = torch.arange(len(kk), device=DEV)
            block = self.table[b, pos // self.page].long()
            assert bool((block >= 0).all()) and not seen & set(block.tolist())
            seen |= set(block.tolist())
            for x, codes, scales in zip((kk, vv), parts(self.cache)[:2], parts(self.cache)[2:]):
                c, s = quantise(x)
                assert torch.equal(codes[block, :, pos % self.page], c) and torch.equal(scales[block, :, pos % self.page], s)
        compare(out, lse, *reference(q, self.cache, self.table, lens, start, self.dim ** -0.5, window))


STEPS = [[37, 5, 200, 1], [1, 90, 1, 1], [1, 1, 1, 0], [130, 1, 0, 1], [1, 1, 1, 1], [1, 1, 1, 33]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,window",
                         [(BF, 8, 2, 128, 16, None), (FP, 6, 6, 64, 32, 50), (BF, 16, 1, 256, 48, None)])
def test_gpu_steps(dtype, heads, kv_heads, dim, page, window):
    """Prompts, then batches that mix chunks, single tokens and requests that sit a step out, in padded buffers."""
    e = Engine(1, 4, 60, 40, heads, kv_heads, dim, page, dtype)
    for turn, query in enumerate(STEPS):
        print(f"\n[case] step {turn} {query} {dtype} {dim}", flush=True)
        rows = sum(query) + 7  # a padded buffer
        q, k, v = e.rows(rows, heads), e.rows(rows, kv_heads), e.rows(rows, kv_heads)
        into = torch.full_like(q, 3.0)
        got = e.step(q, k, v, torch.tensor(query, dtype=torch.int32, device=DEV), rows, window_size=window,
                     max_query_len=max(query), out=into)
        torch.cuda.synchronize()
        e.check(query, k, v, *got, q, window)
        assert bool((into[sum(query):] == 3).all())
        e.context = got[1]


@pytest.mark.gpu
def test_gpu_steps_through_torch_ops():
    class Ops:
        build_block_tables = torch.ops.flaggems_vllm.build_block_tables
        mxfp4_kv_quant_and_cache = torch.ops.flaggems_vllm.mxfp4_kv_quant_and_cache
        mxfp4_paged_attention = torch.ops.flaggems_vllm.mxfp4_paged_attention

    e, f = Engine(2, 4, 60, 40, 8, 2, 128, 16, BF), Engine(2, 4, 60, 40, 8, 2, 128, 16, BF)
    for query in STEPS[:3]:
        rows = sum(query)
        q, k, v = e.rows(rows, 8), e.rows(rows, 2), e.rows(rows, 2)
        lens = torch.tensor(query, dtype=torch.int32, device=DEV)
        got, want = f.step(q, k, v, lens, rows, Ops), e.step(q, k, v, lens, rows)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        e.context, f.context = want[1], got[1]


@pytest.mark.gpu
@pytest.mark.parametrize("query_rows", [1, 5])
def test_gpu_steps_in_a_graph(query_rows):
    """Single tokens, and a few at a time, as one graph that moves its own lengths on; every replay against an eager twin
    and the formula."""
    reqs, heads, kv_heads, dim, page = 6, 8, 2, 128, 16
    e, f = (Engine(3, reqs, 60, 20, heads, kv_heads, dim, page, BF) for _ in range(2))
    first = [30, 1, 17, 64, 3, 100]
    q, k, v = e.rows(sum(first), heads), e.rows(sum(first), kv_heads), e.rows(sum(first), kv_heads)
    for x in (e, f):
        got = x.step(q, k, v, torch.tensor(first, dtype=torch.int32, device=DEV), sum(first))
        x.context = got[1]
    e.check(first, k, v, *got, q)
    rows = reqs * query_rows
    fixed = [torch.zeros(rows, h, dim, dtype=BF, device=DEV) for h in (heads, kv_heads, kv_heads)]
    query = torch.zeros(reqs, dtype=torch.int32, device=DEV)
    free = e.num_free.clone()

    def step():
        e.num_free = free
        got = e.step(*fixed, query, rows, max_query_len=query_rows, max_seq_len=20 * page)
        free.copy_(e.num_free)
        e.context.copy_(got[1])
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # queries of no length: nothing changes
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(8):
        print(f"\n[case] replay {turn} of {query_rows}", flush=True)
        lens = [query_rows - (b + turn) % 3 if (b + turn) % 3 < query_rows else 0 for b in range(reqs)]
        for x, h in zip(fixed, (heads, kv_heads, kv_heads)):
            x.copy_(e.rows(rows, h))
        query.copy_(torch.tensor(lens))
        graph.replay()
        n = sum(lens)
        have = [t.clone() for t in got]
        want = f.step(*fixed, query, rows, max_query_len=query_rows, max_seq_len=20 * page)
        f.context = want[1]
        torch.cuda.synchronize()
        for x, y in zip(have[:3], want[:3]):
            assert torch.equal(x, y)
        assert torch.equal(have[3][:n], want[3][:n]) and torch.equal(have[4][:n], want[4][:n])
        assert torch.equal(e.table, f.table) and torch.equal(e.cache, f.cache) and torch.equal(free, f.num_free)
        e.check(lens, *(x[:n] for x in fixed[1:]), have[0], have[1], have[2], have[3][:n], have[4][:n], fixed[0][:n])


@pytest.mark.gpu
def test_gpu_blocks_run_out():
    """Without a free block a token has no slot: it is not cached, and its key is seen by nobody."""
    e = Engine(4, 3, 4, 8, 4, 2, 64, 16, BF)
    query = [16, 40, 20]
    q, k, v = e.rows(76, 4), e.rows(76, 2), e.rows(76, 2)
    start, lens, positions, out, lse = e.step(q, k, v, torch.tensor(query, dtype=torch.int32, device=DEV), 76)
    assert e.num_free.item() == 4 - (1 + 3 + 2) and e.table[2, :2].tolist() == [-1, -1]
    compare(out, lse, *reference(q, e.cache, e.table, lens, start, 64 ** -0.5))
    assert not bool(out[56:].any()) and bool(torch.isposinf(lse[56:]).all())
