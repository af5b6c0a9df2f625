"""The workspace of fgv_mxfp4_paged_attention through the C ABI: nothing is written behind the bytes that the size query
names, fewer mean whole tiles, and a window never needs more than the query, which does not know it, says."""
import random

import pytest
import torch

from flaggems_vllm import _native

from .test_mxfp4_attention import BF, FP, Case


def need(c, most_q, most_s):
    tokens, heads, dim = c.q.shape
    return _native.lib().fgv_mxfp4_paged_attention_workspace_bytes(tokens, heads, c.kv_heads, dim, len(c.lens), most_q, most_s)


def call(c, ws, ws_bytes, most_q, most_s, window=0):
    """(status, out, lse) with the workspace at address ws."""
    tokens, heads, dim = c.q.shape
    out, lse = torch.full_like(c.q, 7.0), torch.full((tokens, heads), 7.0, device=c.q.device)
    rc = _native.lib().fgv_mxfp4_paged_attention(
        c.q.data_ptr(), c.q.stride(0), c.q.stride(1), int(c.dtype == FP), tokens, heads, c.kv_heads, dim, c.cache.data_ptr(),
        c.cache.stride(0), len(c.cache), c.page, c.table.data_ptr(), c.table.stride(0), c.table.shape[1], c.lens.data_ptr(),
        None if c.one else c.start.data_ptr(), len(c.lens), most_q, most_s, c.scale, window, None, out.data_ptr(), out.stride(0),
        out.stride(1), lse.data_ptr(), lse.stride(0), ws, ws_bytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc, out, lse


CASES = [  # lengths, query tokens, heads, key heads, dim
    ([6000, 2500, 9000, 40], [70, 5, 300, 1], 8, 2, 128),  # cuts in both launches
    ([20000], None, 8, 8, 128), ([9001, 3, 4097], None, 16, 1, 256), ([9000], [200], 4, 4, 64), ([5000] * 9, [3] * 9, 12, 3, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,query,heads,kv_heads,dim", CASES)
def test_gpu_workspace_of_exactly_the_size_named(dtype, lens, query, heads, kv_heads, dim):
    print(f"\n[case] workspace {dtype} {lens} {query} {dim}", flush=True)
    c = Case(60, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    most = max(query or [1]), max(lens)
    n, guard = need(c, *most), 1 << 16
    assert n > 0
    ws = torch.full((n + guard,), 0xA5, dtype=torch.uint8, device=c.q.device)
    rc, out, lse = call(c, ws.data_ptr(), n, *most)
    assert rc == 0 and bool((ws[n:] == 0xA5).all()) and not bool((ws[:n] == 0xA5).all())
    c.check(got=(out, lse))
    for x, y in zip((out, lse), c.run(max_query_len=most[0], max_seq_len=most[1])):
        assert torch.equal(x, y)
    # a byte too few, or none: whole tiles, the workspace left alone
    ws.fill_(0xA5)
    whole = []
    for args in ((ws.data_ptr(), n - 1), (ws.data_ptr(), 0), (None, 0), (None, n)):
        rc, *got = call(c, *args, *most)
        assert rc == 0
        c.check(got=tuple(got))
        whole.append(got)
    assert bool((ws == 0xA5).all())
    for got in whole[1:]:
        assert torch.equal(got[0], whole[0][0]) and torch.equal(got[1], whole[0][1])
    rc, out, lse = call(c, ws.data_ptr() + 8, n, *most)
    assert rc == -3 and bool((out == 7).all()) and bool((lse == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_gpu_windows_need_no_more(seed):
    """With a window, the bytes named without it are enough: more of them change no bit."""
    r = random.Random(seed)
    reqs, kv_heads, dim = r.choice((1, 2, 5, 40)), r.choice((1, 2, 4)), r.choice((64, 128, 256))
    heads = kv_heads * r.choice((1, 4, 7))
    lens = [r.randrange(1, 12000) for _ in range(reqs)]
    query = [min(n, r.choice((1, 4, 90, 300))) for n in lens]
    c = Case(seed, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=r.choice((BF, FP)), page=64)
    most = max(query), max(lens)
    n = need(c, *most)
    ws = torch.full((n + (64 << 20),), 0xA5, dtype=torch.uint8, device=c.q.device)
    for window in (1, 600, 700, 1280, 1281, 2500, 6000, 20000):
        print(f"\n[case] window's workspace {seed} {reqs} {heads} {kv_heads} {dim} {window} {n}", flush=True)
        rc, out, lse = call(c, ws.data_ptr(), n, *most, window)
        assert rc == 0 and bool((ws[n:] == 0xA5).all())
        rc, *more = call(c, ws.data_ptr(), len(ws), *most, window)
        assert rc == 0 and torch.equal(out, more[0]) and torch.equal(lse, more[1])


def test_size_named_for_nothing():
    size = _native.lib().fgv_mxfp4_paged_attention_workspace_bytes
    assert size(0, 8, 2, 128, 0, 1, 100000) == 0 and size(4, 1, 2, 128, 4, 1, 100000) == 0
    assert size(4, 8, 2, 128, 4, 1, 1000) == 0 < size(4, 8, 2, 128, 4, 1, 100000)
