"""The 4-bit cache's ops at the ends of what they take: softmax scales and queries of any size, value blocks whose sums
pass 32 bits' range, against the formula in 64 bits within the bounds of test_mxfp4_attention.py.
"""
import pytest
import torch

import flaggems_vllm as fv
from flaggems_vllm import _native

from .test_mxfp4_attention import BF, FP, Case
from .test_mxfp4_kv_cache import empty_cache, expected, parts, rows, values

QUERIES = [None, [70, 3, 1]]  # single tokens (16-row tiles), and a request whose rows take 128-row tiles up to D = 128


def small(seed, query, dtype, dim, exponent):
    """Rows whose largest value is in [2^exponent, 2^(exponent + 1))."""
    c = Case(seed, [150, 40, 9], query, dtype=dtype, dim=dim)
    x = c.q.double()
    x = x / x.abs().amax(2, keepdim=True) * 1.5 * 2.0 ** exponent
    c.q = x.to(dtype)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("query", QUERIES)
def test_gpu_tiny_softmax_scales(dtype, dim, query):
    """Scores of nothing, row maximum times scale from 2^-96 to 2^-140: the mean of the values, lse the keys' logarithm."""
    for exponent in (0, -9, -14):
        c = small(40, query, dtype, dim, exponent)
        for s in range(96, 140):
            c.scale = 2.0 ** (-s - exponent)
            c.check(max_query_len=70)
    for scale, exponent in ((1e-31, -9), (1e-28, -16), (1e-30, 0), (-1e-31, -9), (1e-45, 3)):
        c = small(41, query, dtype, dim, max(exponent, -14) if dtype == FP else exponent)
        c.scale = scale
        c.check(max_query_len=70)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("query", [None, [50, 1, 20]])
def test_gpu_queries_that_are_not_finite(dtype, dim, query):
    """Their rows are NaN and no others, at the head sizes beside 128 too."""
    c = Case(42, [77, 0, 200], query, dtype=dtype, dim=dim)
    c.q[0, 0, 3], c.q[0, 5, 60], c.q[-1, 2, dim - 1], c.q[1, 1, 0] = torch.nan, torch.inf, -torch.inf, torch.nan
    for scale in (c.scale, 1e-31):
        c.scale = scale
        out, lse = c.check(max_query_len=50)
        assert bool(torch.isnan(out[0, 0]).all()) and bool(torch.isnan(lse[0, 5])) and not bool(torch.isnan(out[0, 1]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,query", [([300, 80, 190], [1, 1, 1]), ([300, 80, 190], [100, 9, 190]), ([300, 64], [5, 3])])
def test_gpu_value_bytes_past_the_range(dtype, dim, lens, query):
    """Value blocks under bytes 253 and 254, which no op here writes, are NaN as under 255: for the rows that see them,
    and for no other row of their tile."""
    for byte in (253, 254):
        for at in (0, 70, 189, 295):
            print(f"\n[case] byte {byte} {dtype} {dim} {query} {at}", flush=True)
            c = Case(50, lens, query, dim=dim, dtype=dtype)
            codes, scales = parts(c.cache)[1], parts(c.cache)[3]
            where = [(int(c.table[b, at // 16]), b) for b, n in enumerate(lens) if at < n]
            for block, _ in where:
                codes[block, :, at % 16] = 0x7F  # 6 and -6
            got = []
            for x in (byte, 255):
                for block, _ in where:
                    scales[block, 1, at % 16, dim // 64] = x
                got.append((c.run(max_query_len=max(query)), c.run(max_query_len=max(query), window_size=40)))
            c.check(got=got[0][0])
            c.check(40, got=got[0][1])
            c.check(got=got[1][0])


SIZES = [  # lengths, query tokens, heads, key heads, dim
    ([700, 64, 23], None, 8, 2, 128), ([700, 64, 23], None, 16, 1, 256), ([700, 64, 23], None, 8, 8, 64),
    ([700, 300], [700, 70], 8, 2, 128), ([700, 300], [650, 1], 2, 1, 64), ([700, 300], [90, 70], 8, 2, 256),
    ([9000], None, 8, 1, 128), ([9000], [130], 4, 4, 64), ([9000, 5000], [3, 200], 8, 2, 128), ([9000], None, 4, 1, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,query,heads,kv_heads,dim", SIZES)
def test_gpu_large_values_of_one_sign(dtype, lens, query, heads, kv_heads, dim):
    """Scores all alike over values all alike, the largest that a cache is written with among them: their mean is that
    value, though their sum is past 32 bits' range; tiles whole and cut."""
    for byte in (252, 245, 230, 217, 216, 215, 127) if dtype == BF else (252, 217, 140, 127):
        print(f"\n[case] one sign {dtype} {lens} {query} {dim} {byte}", flush=True)
        c = Case(44, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        codes, scales = parts(c.cache)[1], parts(c.cache)[3]
        codes.fill_(0x77)
        codes[:, :, :, 1] = 0xFF
        scales[scales != 255] = byte
        for shrink in (0.0, 1.0):  # scores all alike, and the usual ones
            c.q = c.q * shrink if shrink else Case(45, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype).q
            out, _ = c.check(max_query_len=max(query or [1]))
            if dtype == BF:
                want = torch.full_like(out, 6 * 2.0 ** (byte - 127))
                want[..., 2:4] *= -1
                assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,query,heads,kv_heads,dim", SIZES)
def test_gpu_large_values_here_and_there(dtype, lens, query, heads, kv_heads, dim):
    """The largest values at some tokens only, early, late and throughout, of both signs, beside ordinary ones."""
    for seed, where in enumerate([slice(0, 1), slice(600, 640), slice(20, 5000, 37), slice(0, 9000)]):
        print(f"\n[case] here and there {dtype} {lens} {query} {dim} {where}", flush=True)
        c = Case(46 + seed, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        at = torch.arange(lens[0], device=c.cache.device)[where]
        block = c.table[0, at // 16].long()
        for h in range(kv_heads):
            byte = torch.randint(205, 253, (len(at), dim // 32), generator=c.g).to(torch.uint8).to(at.device)
            parts(c.cache)[3][block, h, at % 16] = byte
        c.check(max_query_len=max(query or [1]))
        c.check(window=333, sink=torch.randn(heads, device=at.device), max_query_len=max(query or [1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("query", QUERIES)
def test_gpu_scaled_queries_past_the_range(dim, query):
    """A row whose largest value times the scale (and log2 e) is 2^135 or more counts as one that holds an infinity, whatever its
    keys are; below that scores are what they are."""
    c = Case(43, [90, 40, 9], query, dim=dim, dtype=BF)
    parts(c.cache)[2].masked_fill_(parts(c.cache)[2] != 255, 1)  # keys of at most 6 * 2^-126
    c.q = (c.q.double() / c.q.double().abs().amax(2, keepdim=True) * 1.5).to(BF)
    c.q[:, 1::2] *= 2.0 ** 116
    c.q[:, 0::2] *= 2.0 ** 110
    c.scale = 2.0 ** 18  # 2^134 is inside, 2^128 well so
    c.check(max_query_len=70)
    c.scale = 2.0 ** 19
    out, lse = c.run(max_query_len=70)
    torch.cuda.synchronize()
    assert bool(torch.isnan(out[:, 1::2]).all()) and bool(torch.isnan(lse[:, 1::2]).all())
    assert not bool(torch.isnan(out[:, 0::2]).any()) and not bool(torch.isnan(lse[:, 0::2]).any())
    c.scale = -2.0 ** 22
    assert bool(torch.isnan(c.run(max_query_len=70)[0][:, 1::2]).all())


def call_c(tokens, heads, reqs, start=16):
    return _native.lib().fgv_mxfp4_paged_attention(
        16, 64 * heads, 64, 0, tokens, heads, heads, 64, 16, heads * 16 * 68, 5, 16, 16, 4, 4, 16, start, reqs, 1, 64, 0.1,
        0, None, 16, 64 * heads, 64, 16, heads, None, 0, None)


@pytest.mark.parametrize("tokens,heads", [(1 << 48, 65536), (1 << 62, 4), ((1 << 58) + 1, 64), (1 << 30, 1), (1 << 29, 3)])
def test_c_abi_refuses_rows_whose_number_wraps(tokens, heads):
    """tokens * heads past 64 bits is too large, not small."""
    assert call_c(tokens, heads, 3) == -5
    assert b"2^30 - 1 query rows" in _native.lib().fgv_last_error()
    assert call_c(tokens, heads, 1 << 62) == -5
    assert _native.lib().fgv_mxfp4_paged_attention_workspace_bytes(tokens, heads, heads, 64, 3, 100, 100000) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("query_heads", [64, 128])
def test_gpu_attention_in_more_workgroups_than_a_launch_has(query_heads):
    """2^18 + 1 requests of one token and 64 key heads: 2^24 + 64 workgroups of 256 threads, of which a launch of 2^32
    and more has only what is left of 32 bits."""
    reqs, heads, dim = 2 ** 18 + 1, 64, 64
    c = Case(51, [16] * 40, heads=query_heads, kv_heads=heads, dim=dim, dtype=BF)
    g = torch.Generator().manual_seed(52)
    live = c.table[:, 0]
    table = live[torch.randint(0, 40, (reqs,), generator=g).to(live.device)][:, None]
    lens = torch.ones(reqs, dtype=torch.int32, device=live.device)
    lens[77::1000] = 0
    out, lse = fv.mxfp4_paged_attention(c.q[:1].expand(reqs, -1, -1), c.cache, table, lens, c.scale)
    first = values(parts(c.cache)[1][live.long(), :, 0], parts(c.cache)[3][live.long(), :, 0])  # [40, heads, dim]
    want = first.to(BF).repeat_interleave(query_heads // heads, 1)
    at = torch.empty(len(c.cache), dtype=torch.long, device=live.device)
    at[live.long()] = torch.arange(40, device=live.device)
    for b in range(0, reqs, 1 << 14):
        mine = want[at[table[b:b + (1 << 14), 0].long()]] * (lens[b:b + (1 << 14)] > 0)[:, None, None]
        assert torch.equal(out[b:b + (1 << 14)], mine), b
    assert bool((torch.isposinf(lse) == (lens == 0)[:, None]).all())


@pytest.mark.gpu
def test_gpu_insert_in_more_workgroups_than_a_launch_has():
    """2^24 + 3 tokens of 8 heads of 256, a workgroup each."""
    tokens, heads, dim, page = 2 ** 24 + 3, 8, 256, 16
    k, v = rows(53, 1, heads, dim, dtype=BF), rows(54, 1, heads, dim, dtype=BF)
    cache = empty_cache(4, heads, page, dim)
    slots = torch.full((tokens,), -1, dtype=torch.int64)
    at = torch.tensor([0, 5, 2 ** 21 - 1, 2 ** 21, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 24, tokens - 1])
    slots[at] = torch.arange(len(at)) * 5 + 3
    want = expected(cache, k.expand(len(at), -1, -1), v.expand(len(at), -1, -1), slots[at])
    fv.mxfp4_kv_quant_and_cache(k.expand(tokens, -1, -1), v.expand(tokens, -1, -1), cache, slots.to(k.device))
    torch.cuda.synchronize()
    assert torch.equal(cache.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("starts", [[20, 120, 70, 170], [20, 170, 20, 170, 20, 170], [170, 20, 170, 20, 100, 60, 170]])
def test_gpu_requests_that_share_rows(dim, starts):
    """More tiles than the launch has workgroups for, whole and dealt out: rows of no request stay, and the next call is as
    ever."""
    reqs = len(starts) - 1
    for lens in ([60] * reqs, [5000] * reqs):
        c = Case(55, lens, [50] * reqs, heads=8, kv_heads=2, dim=dim)
        want = c.check(max_query_len=50)
        q = torch.cat([c.q, c.q])[:190].contiguous()
        out = torch.full_like(q, 7.0)
        for most in (1, 50, 190):
            print(f"\n[case] shared rows {dim} {starts} {lens[0]} {most}", flush=True)
            fv.mxfp4_paged_attention(q, c.cache, c.table, c.lens, c.scale, max_query_len=most, out=out,
                                     query_start_loc=torch.tensor(starts, dtype=torch.int32, device=q.device))
            torch.cuda.synchronize()
            assert bool((out[:20] == 7).all()) and bool((out[170:] == 7).all())
        for x, y in zip(c.run(max_query_len=50), want):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_starts_that_fall_to_nothing():
    """A batch padded with starts of 0, or of any row: those requests have no tokens, and the others what is theirs."""
    c = Case(56, [300, 64, 500], [30, 2, 70])
    want = c.check(max_query_len=70)
    for pad in ([0, 0, 0], [101, 3, 3], [102, 0, 0]):
        table = torch.cat([c.table, c.table])
        out, lse = fv.mxfp4_paged_attention(
            c.q, c.cache, table, torch.cat([c.lens, c.lens]), c.scale, max_query_len=70,
            query_start_loc=torch.cat([c.start, torch.tensor(pad, dtype=torch.int32, device=table.device)]))
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("query", [None, [70]])
def test_gpu_small_weights_of_large_values(dtype, dim, query):
    """One key's score 118 binades above all others, and its values 0: what the others' weights leave of values of 6 * 2^103 is
    the output, also where their sum could never pass the range."""
    c = Case(57, [700], query, heads=2, kv_heads=2, dim=dim, dtype=dtype)
    kc, vc, ks, vs = parts(c.cache)
    live = c.table[0, :-(-700 // 16)].long()
    kc[live], vc[live], ks[live], vs[live] = 0, 0x77, 127, 230
    one = int(c.table[0, 0])
    kc[one, :, 5, 0], vc[one, :, 5] = 0x07, 0  # 6 in dim 0
    c.q.zero_()
    c.q[:, :, 0] = 13.625  # 6 * 13.625 = 117.9 ln 2
    c.scale = 1.0
    out, _ = c.check(max_query_len=max(query or [1]))
    assert bool((out > 0.1).all())


@pytest.mark.gpu
def test_gpu_columns_without_a_block_stay_and_blocks_come_back_by_the_caller():
    """What a step that ran out leaves behind, as the next steps see it; a finished request's blocks put back on the stack."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table, free = torch.full((2, 6), -1, dtype=torch.int32, device="cuda"), i32(10, 11, 12, 13)
    _, lens, _, slots, left = fv.build_block_tables(i32(0, 0), i32(40, 40), table, free, i32(4), 16, 80)
    assert table[:, :3].tolist() == [[13, 12, 11], [10, -1, -1]] and left.tolist() == [-2]
    assert (slots >= 0).sum().item() == 56
    # the first request ends: its blocks go back behind what is left (a negative count as 0)
    free[:3], left = table[0, :3].clone(), i32(3)
    _, lens, _, slots, left = fv.build_block_tables(i32(0, 40), i32(0, 9), table, free, left, 16, 9)
    assert table[1].tolist() == [10, -1, -1, 11, -1, -1] and left.tolist() == [2] and lens.tolist() == [0, 49]
    assert slots.tolist() == [-1] * 8 + [11 * 16]
    # taken back to the length that its blocks hold, it goes on
    _, lens, _, slots, left = fv.build_block_tables(i32(0, 16), i32(0, 20), table, free, left, 16, 20)
    assert table[1, :3].tolist() == [10, 12, 13] and left.tolist() == [0]
    assert slots.tolist() == [12 * 16 + i for i in range(16)] + [13 * 16 + i for i in range(4)]
