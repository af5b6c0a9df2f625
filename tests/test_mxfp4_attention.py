"""mxfp4_paged_attention against the formula in 64 bits, and its refusals.

What the kernels may be off, row by row (``bounds``), counted before their first run:

* the query enters as e4m3 pieces under one power of two per row that puts its maximum into
  [128, 256).  The first piece leaves of small values up to 1/16 (it takes multiples of 1/8) and of
  others what 4 bits do not hold; of what it leaves of a small value, at most 1 after the factor 16,
  the second leaves half a step of 4 bits below 1, 2^-5: 2^-9 in all, 2^-16 of the row's maximum
  (large bf16 values are held whole).  A third piece (fp16) leaves 2^-5 of 2^-4 of that;
* the matrix instruction adds at most 32 products at a time, each cut below
  2^(E - 13), E the largest exponent among them.  A product has 6 bits, and the codes'
  exponents span 3 binades, so only products of query values more than 6 binades
  below their block's largest are cut, each by less than 2^-13 of 2^E; of the pieces
  behind the first, 2^-4 as large at least, any may be;
* scores are scaled and exp2 taken in 32 bits: 2^-20 (1 + |s|) together covers the
  scaling, the subtraction and two ulp of the exponential;
* P enters as two bf16 pieces (2^-16).  Where D is at most 128 and a request has more than 64 rows for a
  key head (or is alone, or among so few that all their key heads together are at most a quarter of the
  CUs: such may share the others' tiles), bf16 calls have one fp16 piece of it, half a step of its 11
  bits or 2^-11, an eighth of what the output's rounding takes, and both types lose of P times 2^7 what
  lies below fp16's least step, half of 2^-24: under a reference of at most 2^4 times the row's largest
  that is 2^(-25 - 7 + 4) = 2^-28 of the row's largest a key;
* P below 2^-126 is nothing in 32 bits (the first run showed that this had been left out: a dim
  where all keys but such ones hold zeros came out as 0 instead of 4e-39).  P is taken under a
  reference of at most 2^4 times the row's largest, so that is 2^-122 |v| a key, as a score
  and again as a sum that is joined;
* sums in 32 bits: a step of 2^-23 per 32 keys and per joined part;
* the output is rounded once (eps / 2 of the type, or half its least subnormal).
"""
import math

import pytest
import torch

import flaggems_vllm as fv
from flaggems_vllm import _native, library

from .test_mxfp4_kv_cache import empty_cache, parts, quantise, values

DEV = torch.device("cuda:0")
BF, FP = torch.bfloat16, torch.float16


class Case:
    """A cache filled through block tables in random order, queries and lengths, on the GPU."""

    def __init__(self, seed, lens, query=None, heads=8, kv_heads=2, dim=128, page=16, dtype=BF, spare=3, fill=0xFF,
                 size=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dim, self.page, self.dtype, self.kv_heads = g, dim, page, dtype, kv_heads
        query = [1] * len(lens) if query is None else query
        used = [-(-n // page) for n in lens]
        width = max(used + [1]) + 1
        ids = torch.randperm(sum(used) + spare, generator=g).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        self.cache = empty_cache(sum(used) + spare, kv_heads, page, dim, fill)
        rows = []
        for b, n in enumerate(used):
            mine = [ids.pop() for _ in range(n)]
            table[b, :n] = torch.tensor(mine, dtype=torch.int32)
            rows += [mine[j // page] * page + j % page for j in range(lens[b])]
        shape = (len(rows), kv_heads, dim)
        k = torch.randn(shape, generator=g) * size * torch.exp2(torch.randn(kv_heads, 1, generator=g))
        k[:, :, torch.randint(0, dim, (3,), generator=g)] *= 6
        v = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-3, 4, (kv_heads, dim), generator=g).float())
        if rows:
            at = torch.tensor(rows, device=DEV)
            for x, codes, scales in zip((k, v), parts(self.cache)[:2], parts(self.cache)[2:]):
                c, s = quantise(x.to(dtype).to(DEV))
                codes[at // page, :, at % page] = c
                scales[at // page, :, at % page] = s
        self.q = (torch.randn(sum(query), heads, dim, generator=g) * size).to(dtype).to(DEV)
        self.table, self.lens = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.start = torch.tensor([sum(query[:i]) for i in range(len(query) + 1)], dtype=torch.int32, device=DEV)
        self.one = all(n == 1 for n in query)
        self.scale = dim ** -0.5

    def run(self, **kw):
        if not self.one or "query_start_loc" in kw:
            kw = {"query_start_loc": self.start, **kw}
        return fv.mxfp4_paged_attention(self.q, self.cache, self.table, self.lens, self.scale, **kw)

    def check(self, window=None, sink=None, got=None, ways=({},), **kw):
        """The call (each of several ways to make it) against the reference; what the last one gave."""
        want = reference(self.q, self.cache, self.table, self.lens, self.start, self.scale, window, sink)
        for way in ways:
            out, lse = got or self.run(window_size=window, attn_sink=sink, **kw, **way)
            torch.cuda.synchronize()
            compare(out, lse, *want)
        return out, lse


def keys_of(cache, row, n):
    """The first n keys and values of a block-table row in 64 bits and their scale bytes; which of them exist."""
    page = cache.shape[2]
    at = torch.arange(n, device=cache.device)
    block = row.long()[(at // page).clamp(max=len(row) - 1)]
    real = (at // page < len(row)) & (block >= 0) & (block < len(cache))
    block = block.clamp(0, max(len(cache) - 1, 0))
    kc, vc, ks, vs = (p[block, :, at % page].transpose(0, 1) for p in parts(cache))
    return values(kc, ks), values(vc, vs), ks, real


def reference(q, cache, table, lens, start, scale, window=None, sink=None):
    """(out, lse, bound of out, bound of lse, rows) in 64 bits."""
    tokens, heads, dim = q.shape
    kv_heads, three = cache.shape[1], q.dtype == FP
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((tokens, heads), torch.inf, dtype=torch.float64, device=q.device)
    obound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    mine = torch.zeros(tokens, dtype=torch.bool, device=q.device)
    for b, n in enumerate(lens.tolist()):
        t0, t1 = start[b].item(), start[b + 1].item()
        if t1 <= t0:
            continue
        mine[t0:t1] = True
        if n <= 0:
            continue
        k, v, kbytes, real = keys_of(cache, table[b], n)
        pos = torch.arange(n - (t1 - t0), n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        seen = (j <= pos) & real
        if window:
            seen &= j > pos - window
        group = heads // kv_heads
        for h in range(heads):
            x, kh, vh = q[t0:t1, h].double(), k[h // group], v[h // group]
            s = torch.where(seen, x @ torch.where(seen.any(0)[:, None], kh, 0.0).t().contiguous() * scale, -torch.inf)
            s = torch.where(torch.isnan(x).any(1, keepdim=True) | torch.isinf(x).any(1, keepdim=True),
                            torch.where(seen, torch.nan, -torch.inf), s)
            some = seen.any(1)
            l = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(some, l, 0.0)[:, None])
            # 0 times a NaN that a row does not see is nothing
            nan = torch.isnan(vh)
            o = p @ torch.where(nan, 0.0, vh)
            o = torch.where((seen.double() @ nan.double()) > 0, torch.nan, o)
            share = torch.ones_like(l) if sink is None else 1 / (1 + torch.exp(sink[h].double() - l))
            # the bounds
            top = x.abs().amax(1, keepdim=True)
            blocks = x.abs().unflatten(1, (-1, 32))
            e = torch.floor(torch.log2(blocks.clamp(min=1e-300)))
            far = ((blocks > 0) & (e < e.amax(2, keepdim=True) - 6)).sum(2) + 2.125
            cut = far * 2.0 ** -13 * torch.exp2(e.amax(2)) * (blocks.amax(2) > 0)
            kscale = torch.exp2(kbytes[h // group].double() - 127) * 4
            kabs = torch.where(torch.isnan(kh), 0.0, kh).abs().sum(1)
            d = abs(scale) * (cut @ torch.where(kscale > 1e30, 0.0, kscale).t().contiguous()
                             + 2.0 ** (-20 if three else -16) * top * kabs)
            d = torch.where(seen, d + 2.0 ** -20 * (1 + s.abs()), 0.0).nan_to_num(0.0).amax(1)
            steps = (n / 32 + 40) * 2.0 ** -23
            weight = p @ torch.where(nan, 0.0, vh).abs() * share[:, None]
            o = o * share[:, None]
            half = torch.finfo(q.dtype).eps / 2
            cus = torch.cuda.get_device_properties(q.device).multi_processor_count
            many = dim <= 128 and ((t1 - t0) * group > 64 or len(lens) == 1
                                 or (len(q) * group > 64 and len(lens) * kv_heads <= cus // 4))
            ob = weight * ((2.0 ** -11 if many and not three else 2.0 ** -16) + 2.5 * d + steps)[:, None] * (1 + half)
            if many:
                ob = ob + 2.0 ** -28 * (p.amax(1) * share)[:, None] * torch.where(nan, 0.0, vh).abs().sum(0)
            ob = ob + half * o.abs() + torch.finfo(q.dtype).smallest_normal * half
            ob = ob + 2.0 ** -121 * torch.where(nan, 0.0, vh).abs().sum(0)
            out[t0:t1, h] = torch.where(some[:, None], o, 0.0)
            lse[t0:t1, h] = torch.where(some, l, torch.inf)
            obound[t0:t1, h] = ob
            lbound[t0:t1, h] = d + steps + 2.0 ** -22 * (1 + l.abs())
    return out, lse, obound, lbound, mine


def compare(out, lse, want, want_lse, obound, lbound, mine):
    top = torch.finfo(out.dtype).max
    out, lse = out.double()[mine], lse.double()[mine]
    want, want_lse, obound, lbound = want[mine], want_lse[mine], obound[mine], lbound[mine]
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    # what may lie past the type's largest value may be an infinity
    past = torch.isinf(out) & (out.sign() == want.sign()) & (want.abs() + obound >= top)
    fine = ~torch.isnan(want) & ~past
    over = ((out - want).abs() / obound.clamp(min=1e-300))[fine & (obound > 0)]
    assert bool((out == want)[fine & (obound == 0)].all())
    assert over.numel() == 0 or over.max() <= 1, over.max().item()
    fine = torch.isfinite(want_lse)
    over = ((lse - want_lse).abs() / lbound)[fine]
    assert over.numel() == 0 or over.max() <= 1, over.max().item()


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 255, 256, 257, 700, 1025, 2, 33]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,page", [(8, 2, 16), (1, 1, 48), (7, 7, 32), (16, 1, 64), (15, 3, 16), (36, 2, 128)])
def test_gpu_decode(dtype, dim, heads, kv_heads, page):
    """One token per request: lengths each side of every tile and page, none among them, and every group size class."""
    print(f"\n[case] decode {dtype} {dim} {heads} {kv_heads} {page}", flush=True)
    c = Case(dim + heads, LENS, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    c.check(ways=({}, dict(max_seq_len=1025, max_query_len=1)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (FP, 256), (BF, 256), (BF, 64), (FP, 128)])
@pytest.mark.parametrize("query", [[2, 5, 1, 0, 3, 8], [33, 1, 130, 17, 0, 64], [300, 1, 1, 2, 129, 128]])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (10, 2), (16, 1)])
def test_gpu_many_tokens(dtype, dim, query, heads, kv_heads):
    """Several tokens per request, causal among themselves, prompts from their first token and chunks behind a context."""
    print(f"\n[case] tokens {dtype} {dim} {query} {heads} {kv_heads}", flush=True)
    lens = [q + c for q, c in zip(query, (0, 100, 63, 40, 7, 513))]
    c = Case(sum(query), lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    # the last bounds do not hold: that costs time only
    c.check(ways=({}, dict(max_seq_len=max(lens), max_query_len=max(query)), dict(max_seq_len=1, max_query_len=1)))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 16, 65, 100, 1000, 10 ** 6])
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (BF, 256)])
def test_gpu_window_and_sink(window, dtype, dim):
    print(f"\n[case] window {window} {dtype} {dim}", flush=True)
    sink = torch.tensor([0.0, -3.0, 50.0, -torch.inf, 2.5, -1e30, 9.0, 300.0], device=DEV)
    Case(window % 97, LENS, dim=dim, dtype=dtype).check(window, sink)
    query = [40, 1, 7, 200, 3]
    Case(window % 89, [40, 333, 300, 290, 700], query, dim=dim, dtype=dtype).check(window, sink, max_query_len=200)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([20000], 8, 8, 128), ([9001, 3, 4097], 16, 1, 256),
                                                     ([30001], 8, 1, 64), ([5000] * 5 + [1], 12, 3, 128)])
def test_gpu_long(dtype, lens, heads, kv_heads, dim):
    """Few rows over a long axis."""
    print(f"\n[case] long {dtype} {lens} {heads} {kv_heads} {dim}", flush=True)
    c = Case(7, lens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=64)
    first = c.check()
    for _ in range(3):  # the same bits every time
        for x, y in zip(first, c.run()):
            assert torch.equal(x, y)
    c.check(4444, torch.randn(heads, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_gpu_long_context_with_many_tokens(dtype):
    print(f"\n[case] long with many tokens {dtype}", flush=True)
    c = Case(8, [6000, 2500, 100], [70, 300, 100], heads=8, kv_heads=2, dtype=dtype)
    c.check(max_query_len=300, max_seq_len=6000)
    c.check(2000, torch.randn(8, device=DEV), max_query_len=300, max_seq_len=6000)
    c = Case(9, [9000, 7], [5, 2], heads=16, kv_heads=2, dtype=dtype)
    c.check(max_query_len=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_gpu_queries_before_the_first_position(dtype):
    """More query tokens than keys: the first of them see nothing."""
    c = Case(3, [5, 0, 64, 20], [9, 4, 100, 20], dtype=dtype)
    out, lse = c.check(sink=torch.randn(8, device=DEV))
    assert not bool(out[:4].any()) and bool(torch.isposinf(lse[:4]).all())
    assert not bool(out[9:13].any()) and bool(torch.isposinf(lse[9:13]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("query", [[1, 1, 1], [4, 1, 70]])
def test_gpu_rows_of_no_request(query):
    """Rows in front of the first request, behind the last one and between two stay as they were."""
    c = Case(4, [100, 50, 90], query)
    n = sum(query)
    q = torch.randn(n + 13, 8, 128, device=DEV).to(BF)
    q[5:5 + n] = c.q
    c.q, c.start = q, c.start + 5
    out = torch.full_like(q, 7.0)
    got, lse = c.run(out=out, query_start_loc=c.start)
    assert got is out or got.data_ptr() == out.data_ptr()
    c.check(got=(out, lse))
    assert bool((out[:5] == 7).all()) and bool((out[5 + n:] == 7).all())
    # a request without tokens in the middle, starts that do not rise, and starts past the rows
    c.start[1] = c.start[2]
    c.check(query_start_loc=c.start)
    c.start[-1] = n + 100
    out.fill_(7.0)
    c.run(out=out, query_start_loc=c.start)
    torch.cuda.synchronize()
    assert bool((out[:5] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("query", [None, [6, 1, 40, 3]])
def test_gpu_bad_pages(dtype, query):
    """Entries that are no block of the cache, and lengths past the table: those keys are seen by nobody."""
    c = Case(5, [200, 64, 333, 90], query, dtype=dtype)
    c.table[0, 3], c.table[0, 7], c.table[1, 0], c.table[2, 20] = -1, len(c.cache), 2 ** 31 - 1, -2 ** 31
    c.table[3] = -1
    out, lse = c.check(max_query_len=40)
    assert not bool(out[c.start[3]:].any()) and bool(torch.isposinf(lse[c.start[3]:]).all())
    c.lens[1] += 500
    c.check()
    c.check(window=30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (BF, 256), (FP, 128)])
def test_gpu_nan_blocks(dtype, dim):
    """A NaN key makes the rows NaN that see it, a NaN value block their dims; rows before it or past its window do not."""
    for seed, (lens, query) in enumerate([([300, 80, 190], [1, 1, 1]), ([300, 80, 190], [100, 9, 190]), ([300, 64], [5, 3])]):
        print(f"\n[case] nan {dtype} {dim} {query}", flush=True)
        for which in (2, 3):
            for at in (0, 70, 189, 295):
                c = Case(seed, lens, query, dim=dim, dtype=dtype)
                kind = parts(c.cache)[which]
                for b, n in enumerate(lens):
                    if at < n:
                        kind[int(c.table[b, at // 16]), 1, at % 16, dim // 64] = 255
                c.check(max_query_len=max(query))
                c.check(40, max_query_len=max(query))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("query", [None, [50, 1, 20]])
def test_gpu_queries_that_are_not_finite(dtype, query):
    c = Case(6, [77, 0, 200], query, dtype=dtype)
    c.q[0, 0, 3], c.q[0, 5, 90], c.q[-1, 2, 127], c.q[1, 1, 0] = torch.nan, torch.inf, -torch.inf, torch.nan
    out, lse = c.check(max_query_len=50)
    assert bool(torch.isnan(out[0, 0]).all()) and bool(torch.isnan(lse[0, 5])) and not bool(torch.isnan(out[0, 1]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_gpu_query_sizes(dtype, dim):
    """Queries of every size of the type: rows of zeros, of subnormals, of the largest values, and values of all
    sizes in one row (only those count that come near the row's largest)."""
    c = Case(11, [150] * 24, dtype=dtype, dim=dim)
    top, low = (120, -133) if dtype == BF else (15, -24)
    g = torch.Generator().manual_seed(1)
    for i in range(24):
        e = torch.randint(low, top, (8, dim), generator=g) if i % 2 else torch.full((8, dim), low + (top - low) * i // 24)
        x = torch.ldexp(1 + torch.rand(8, dim, generator=g, dtype=torch.float64), e)
        c.q[i] = (x * (2 * torch.randint(0, 2, (8, dim), generator=g) - 1)).to(dtype)
    c.q[22] = 0
    # scores of a size that the softmax resolves, row by row
    for i in range(0, 24, 2):
        one = Case.__new__(Case)
        one.__dict__.update(c.__dict__)
        one.q, one.table, one.lens, one.start = c.q[i:i + 1], c.table[i:i + 1], c.lens[i:i + 1], c.start[:2]
        one.scale = 0.5 / max(float(one.q.double().abs().amax()) * dim ** 0.5, 1e-29)
        one.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_gpu_every_scale_byte(dtype):
    """Key and value blocks under every byte that bf16 values need (1..252), and 0."""
    c = Case(12, [256 * 16], dtype=dtype, fill=0, heads=2, kv_heads=2)
    kc, vc, ks, vs = parts(c.cache)
    order = c.table[0, :256].long()
    byte = torch.arange(256, device=DEV).clamp(max=252)
    vs[order, 1] = byte[:, None, None].to(torch.uint8)
    c.check()
    # one key at a time: its value comes back whole, at any size that the type holds
    for b in (0, 1, 100, 120, 127, 135, 200, 252) if dtype == BF else (104, 127, 139):
        one = Case(b, [1], dtype=dtype, heads=2, kv_heads=2)
        parts(one.cache)[3][int(one.table[0, 0]), :, 0] = b
        out, _ = one.run()
        want = values(*(p[int(one.table[0, 0]), :, 0] for p in parts(one.cache)[1::2]))
        assert torch.equal(out[0].double(), want.to(dtype).double()), b
    # keys of every size against a query that brings their scores into range
    for b in (1, 60, 127, 190, 250):
        one = Case(b, [90], dtype=dtype, heads=2, kv_heads=2)
        live = one.table[0, :6].long()
        ks = parts(one.cache)[2]
        ks[live] = torch.where(ks[live] == 255, 255, b).to(torch.uint8)
        one.scale = one.scale * 2.0 ** min(max(127 - b, -90), 90)
        one.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(BF, 64), (FP, 128), (BF, 128), (BF, 256), (FP, 256)])
def test_gpu_value_sizes_with_many_tokens(dtype, dim):
    """Value blocks each side of what fp16 holds, from the first key on, from a later one, and only here and there."""
    for seed, where in enumerate([slice(0, 700), slice(640, 700), slice(300, 301), slice(100, 700, 37)]):
        for low, high in ((109, 114), (145, 150), (0, 3), (111, 148), (1, 253)):
            print(f"\n[case] value sizes {dtype} {dim} {where} {low} {high}", flush=True)
            c = Case(30 + seed, [700, 90], [130, 1], dtype=dtype, dim=dim)
            at = torch.arange(700)[where]
            block = c.table[0, at.to(DEV) // 16].long()
            vs = parts(c.cache)[3]
            for h in range(2):
                byte = torch.randint(low, high, (len(at), dim // 32), generator=c.g).to(torch.uint8)
                vs[block, h, at.to(DEV) % 16] = byte.to(DEV)
            c.check()
            c.check(window=77)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,query,heads,kv_heads,dim", [
    ([5000], [5000], 2, 1, 64), ([3000, 9, 2000], [2500, 9, 2000], 8, 2, 128), ([20000], [129], 4, 1, 128),
    ([9000, 100], [33, 1], 12, 2, 256), ([300] * 40, [65] * 40, 3, 3, 64), ([40000], [7], 16, 1, 256),
    ([20001] + [5] * 300, [200] + [1] * 300, 4, 2, 64)])
def test_gpu_prompts(dtype, lens, query, heads, kv_heads, dim):
    """Prompts, chunks and mixed batches, their tiles whole and cut, and the same bits every time."""
    print(f"\n[case] prompts {dtype} {lens[:3]} {query[:3]} {heads} {kv_heads} {dim}", flush=True)
    c = Case(21, lens, query, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=32)
    first = c.check(max_query_len=max(query), max_seq_len=max(lens))
    for x, y in zip(first, c.run(max_query_len=max(query), max_seq_len=max(lens))):
        assert torch.equal(x, y)
    c.check(500, torch.randn(heads, device=DEV), max_query_len=1000)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_gpu_peaked_and_far_apart_scores(dtype):
    """Scores hundreds apart, rising and falling along the keys, so that the running maximum moves late or never."""
    for size in (4.0, 12.0):
        c = Case(13, [700, 64, 1000], dtype=dtype, size=size)
        c.check()
        c.scale = -c.scale
        c.check()
        c.scale = 0.0
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("query", [None, [3, 90, 20]])
def test_gpu_strides(dtype, query):
    """q out of a fused projection's rows at any element, out into a wider buffer, a cache and a table out of larger ones."""
    for off in (0, 1, 8):
        print(f"\n[case] strides {dtype} {query} {off}", flush=True)
        c = Case(14, [100, 90, 333], query, dtype=dtype)
        n = len(c.q)
        wide = torch.randn(n, 8 * 128 + 50, device=DEV).to(dtype)
        wide[:, off:off + 1024] = c.q.flatten(1)
        c.q = wide[:, off:off + 1024].unflatten(1, (8, 128))
        buf = torch.full((n, 8, 128 + 40), 3.0, dtype=dtype, device=DEV)
        cache = torch.zeros(len(c.cache), 2 * 16 * 136 + 64, dtype=torch.uint8, device=DEV)
        cache[:, 48:-16] = c.cache.flatten(1)
        c.cache = cache[:, 48:-16].unflatten(1, (2, 16, 136))
        table = torch.full((3, 70), 1 << 30, dtype=torch.int32, device=DEV)
        table[:, 3:3 + c.table.shape[1]] = c.table
        c.table = table[:, 3:3 + c.table.shape[1]]
        out = buf[:, :, off:off + 128]
        c.check(got=c.run(out=out))
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[:, :, off:off + 128] = False
        assert bool((buf[rest] == 3).all())
        by_head = c.q.transpose(0, 1).contiguous().transpose(0, 1)
        want = out.clone()
        c.q = by_head
        assert torch.equal(c.run()[0], want)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    page, heads, dim = 64, 8, 128
    blocks = (9 << 30) // (page * heads * 136)
    c = Case(15, [300, 100], [4, 1], heads=16, kv_heads=heads, page=page)
    big = torch.full((blocks, heads, page, 136), 255, dtype=torch.uint8, device=DEV)
    ids = torch.tensor([blocks - 1, 0, blocks // 2 + 1, blocks - 2, 7, blocks // 2, blocks - 3], dtype=torch.int32, device=DEV)
    table = torch.full_like(c.table, -1)
    live = c.table >= 0
    table[live] = ids[:int(live.sum())]
    big[table[live].long()] = c.cache[c.table[live].long()]
    c.cache, c.table = big, table
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("query", [None, [1, 30, 200, 2]])
def test_gpu_two_graphs_and_eager_calls(query):
    """Two captured calls with workspaces in one pool, replayed with the program's own calls in between, on lengths
    that change: every replay is the eager result."""
    c, d = Case(16, [4000, 70, 900, 333], query, dim=128), Case(17, [9000], None, heads=16, kv_heads=1, dim=64, dtype=FP)
    kw = dict(max_query_len=200, max_seq_len=4000, attn_sink=torch.randn(8, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(**kw), d.run()
    torch.cuda.current_stream().wait_stream(side)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, run in zip(graphs, (lambda: c.run(**kw), d.run)):
        with torch.cuda.graph(graph, pool=pool):
            outs.append([t for t in run()])
    for turn in range(4):
        c.lens.copy_(torch.tensor([4000 - 777 * turn, 70 - turn, 900 - 99 * turn, 333 + 0 * turn]))
        d.lens.fill_(9000 - 2500 * turn)
        graphs[0].replay()
        got = [t.clone() for t in outs[0]]
        want = c.run(**kw)
        graphs[1].replay()
        other, want_other = [t.clone() for t in outs[1]], d.run()
        torch.cuda.synchronize()
        for x, y in zip(got + other, [*want, *want_other]):
            assert torch.equal(x, y), turn
        c.check(sink=kw["attn_sink"], got=got)


@pytest.mark.gpu
def test_gpu_streams_at_the_same_time():
    """Calls in flight on two streams, each with a workspace of its own."""
    c, d = Case(18, [8000, 100]), Case(19, [300, 5000], [200, 3])
    want = [*c.check(), *d.check()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, x in zip(streams, (c, d)):
            with torch.cuda.stream(s):
                got.append(x.run())
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(got):
        assert torch.equal(x, want[2 * (i % 2)]) and torch.equal(y, want[2 * (i % 2) + 1])


@pytest.mark.gpu
def test_gpu_nothing_and_many_requests():
    c = Case(20, [3, 1])
    none = fv.mxfp4_paged_attention(c.q[:0], c.cache, c.table[:0], c.lens[:0], 1.0)
    assert none[0].shape == (0, 8, 128) and none[1].shape == (0, 8)
    out, lse = fv.mxfp4_paged_attention(c.q, c.cache[:0], c.table, c.lens, 1.0)  # a cache without a block
    assert not bool(out.any()) and bool(torch.isposinf(lse).all())
    out, lse = fv.mxfp4_paged_attention(c.q, c.cache, c.table[:, :0], c.lens, 1.0)  # a table without a column
    assert not bool(out.any()) and bool(torch.isposinf(lse).all())
    many = Case(21, [(7 * i) % 50 for i in range(700)], heads=4, kv_heads=2, dim=64)
    many.check(ways=({}, dict(query_start_loc=many.start)))
    c = Case(22, [5 + i % 40 for i in range(300)], [1 + (i * i) % 5 for i in range(300)], heads=4, kv_heads=2, dim=64)
    c.check(max_query_len=5)
    # a batch padded with requests of no key: out 0, lse +inf
    c = Case(23, [50, 20, 0, 0, 0])
    out, lse = c.check()
    assert not bool(out[2:].any())


def test_fake_ops_and_names():
    from torch._subclasses.fake_tensor import FakeTensorMode

    for name in library.REGISTERED_PAGED:
        assert hasattr(torch.ops.flaggems_vllm, name)
    with FakeTensorMode():
        q = torch.empty(5, 8, 128, dtype=BF, device="cuda")
        cache = torch.empty(9, 2, 16, 136, dtype=torch.uint8, device="cuda")
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")
        out, lse = torch.ops.flaggems_vllm.mxfp4_paged_attention(q, cache, i32(5, 4), i32(5), 0.1)
        assert out.shape == q.shape and out.dtype == BF and lse.shape == (5, 8) and lse.dtype == torch.float32
        got = torch.ops.flaggems_vllm.build_block_tables(i32(5), i32(5), i32(5, 4), i32(9), i32(1), 16, 30)
        assert [t.shape[0] for t in got] == [6, 5, 30, 30, 1]
        assert [t.dtype for t in got] == [torch.int32, torch.int32, torch.int64, torch.int64, torch.int32]


@pytest.mark.gpu
def test_gpu_torch_ops():
    c = Case(24, [50, 700])
    want = c.run()
    got = torch.ops.flaggems_vllm.mxfp4_paged_attention(c.q, c.cache, c.table, c.lens, c.scale)
    out = torch.empty_like(c.q)
    lse = torch.ops.flaggems_vllm.mxfp4_paged_attention_out(c.q, c.cache, c.table, c.lens, c.scale, out)
    for x, y in zip((*got, out, lse), (*want, *want)):
        assert torch.equal(x, y)


def cpu_args(**kw):
    a = dict(q=torch.zeros(3, 8, 128, dtype=BF), kv_cache=torch.zeros(5, 2, 16, 136, dtype=torch.uint8),
             block_table=torch.zeros(3, 4, dtype=torch.int32), seq_lens=torch.zeros(3, dtype=torch.int32), softmax_scale=0.1)
    return {**a, **kw}


I32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(),  # CPU tensors
    dict(q=torch.zeros(3, 8, 64, dtype=BF)), dict(q=torch.zeros(3, 7, 128, dtype=BF)), dict(q=torch.zeros(3, 8, 128)),
    dict(q=torch.zeros(3, 1024, dtype=BF)), dict(q=torch.zeros(3, 8, 256, dtype=BF)[..., ::2]), dict(q=torch.zeros(4, 8, 128, dtype=BF)),
    dict(q=torch.zeros(3, 8, 128, dtype=BF, requires_grad=True)),
    dict(kv_cache=torch.zeros(5, 2, 16, 128, dtype=torch.uint8)), dict(kv_cache=torch.zeros(5, 2, 8, 136, dtype=torch.uint8)),
    dict(kv_cache=torch.zeros(5, 16, 2, 136, dtype=torch.uint8).transpose(1, 2)), dict(kv_cache=torch.zeros(5, 0, 16, 136, dtype=torch.uint8)),
    dict(kv_cache=torch.zeros(5, 2, 16, 136, dtype=torch.int8)),
    dict(block_table=torch.zeros(2, 4, **I32)), dict(block_table=torch.zeros(3, 4, dtype=torch.int64)),
    dict(block_table=torch.zeros(4, 3, **I32).t()), dict(seq_lens=torch.zeros(3, dtype=torch.int64)),
    dict(seq_lens=torch.zeros(6, **I32)[::2]), dict(seq_lens=torch.zeros(3, 1, **I32)),
    dict(query_start_loc=torch.zeros(3, **I32)), dict(query_start_loc=torch.zeros(4, dtype=torch.int64)),
    dict(softmax_scale=math.inf), dict(softmax_scale=math.nan), dict(window_size=0), dict(window_size=-1),
    dict(max_query_len=-1), dict(max_seq_len=-1), dict(attn_sink=torch.zeros(7)), dict(attn_sink=torch.zeros(8, dtype=BF)),
    dict(attn_sink=torch.zeros(16)[::2]), dict(attn_sink=torch.zeros(8, requires_grad=True)),
    dict(out=torch.zeros(3, 8, 128)), dict(out=torch.zeros(3, 8, 64, dtype=BF)), dict(out=torch.zeros(3, 8, 256, dtype=BF)[..., ::2]),
    dict(out=torch.zeros(8, 3, 128, dtype=BF).transpose(0, 1)), dict(out=torch.zeros(1, 8, 128, dtype=BF).expand(3, 8, 128)),
    dict(out=torch.zeros(3, 1, 128, dtype=BF).expand(3, 8, 128)),
])
def test_refusals(kw):
    with pytest.raises(AssertionError):
        fv.mxfp4_paged_attention(**cpu_args(**kw))


def test_refuses_an_output_over_an_input():
    q = torch.zeros(3, 8, 128, dtype=BF)
    with pytest.raises(AssertionError, match="overlap"):
        fv.mxfp4_paged_attention(**cpu_args(q=q, out=q))


def call_c(**kw):
    a = dict(q=16, dtype=0, tokens=3, heads=8, kv=2, dim=128, cache=16, stride=2 * 16 * 136, blocks=5, page=16, table=16,
             width=4, lens=16, start=None, reqs=3, mq=1, ms=64, scale=0.1, window=0, out=16, lse=16)
    a.update(kw)
    return _native.lib().fgv_mxfp4_paged_attention(
        a["q"], 1024, 128, a["dtype"], a["tokens"], a["heads"], a["kv"], a["dim"], a["cache"], a["stride"], a["blocks"],
        a["page"], a["table"], a["width"], a["width"], a["lens"], a["start"], a["reqs"], a["mq"], a["ms"], a["scale"],
        a["window"], None, a["out"], 1024, 128, a["lse"], 8, None, 0, None)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), -2), (dict(heads=-1), -2), (dict(blocks=-1), -2), (dict(reqs=-1), -2), (dict(width=-1), -2),
    (dict(window=-1), -2), (dict(mq=-1), -2), (dict(ms=-1), -2), (dict(dim=96), -2), (dict(dtype=2), -2), (dict(page=20), -2),
    (dict(kv=3), -2), (dict(kv=0), -2), (dict(reqs=2), -2), (dict(scale=math.inf), -2), (dict(scale=math.nan), -2),
    (dict(page=8192, stride=1 << 30), -5), (dict(width=1 << 27), -5), (dict(tokens=1 << 28, reqs=1 << 28), -5),
    (dict(heads=131072, kv=1), -5), (dict(q=None), -1), (dict(out=None), -1), (dict(lse=None), -1), (dict(lens=None), -1),
    (dict(table=None), -1), (dict(cache=None), -1), (dict(stride=2 * 16 * 136 - 16), -4), (dict(stride=2 * 16 * 136 + 8), -4),
    (dict(cache=24), -3), (dict(q=17), -3), (dict(out=17), -3), (dict(lse=18), -3),
])
def test_c_abi_refusals(kw, code):
    assert call_c(**kw) == code
    assert _native.lib().fgv_last_error()


def test_c_abi_nothing_to_do():
    assert call_c(tokens=0, reqs=0, q=None, out=None, lse=None) == 0
    assert call_c(heads=0, kv=0, q=None, out=None, lse=None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 9, 2, 9], [9, 0, 9, 0], [-5, 4, 2 ** 31 - 1, 3]])
def test_gpu_starts_that_fall(starts):
    """No request should have such starts: rows outside of them stay, and the next call is as ever."""
    c = Case(25, [3000, 64, 500], [3, 3, 3])
    want = c.check(max_query_len=3)
    out = torch.full_like(torch.cat([c.q, c.q]), 7.0)
    for most in (3, 100):
        fv.mxfp4_paged_attention(torch.cat([c.q, c.q]), c.cache, c.table, c.lens, c.scale, max_query_len=most, out=out,
                                 query_start_loc=torch.tensor(starts, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        if max(starts[1:]) <= 9:
            assert bool((out[9:] == 7).all())
    for x, y in zip(c.run(max_query_len=3), want):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("query", [None, [1, 90]])
def test_gpu_lengths_and_windows_at_their_ends(query):
    """Lengths up to int32's end are the table's keys, pages without a block among them; a window near 2^30 is none."""
    c = Case(26, [320, 320], query)
    c.table = c.table[:, :20].contiguous()
    c.table[0, 3], c.table[1, 7] = -1, len(c.cache)
    want = c.check()
    for window in (2 ** 30 - 2, 2 ** 30 - 1, 2 ** 62):
        for x, y in zip(c.run(window_size=window), want):
            assert torch.equal(x, y)
    if query is None:
        for n in (2 ** 31 - 1, 2 ** 31 - 2 ** 13, 2 ** 30):
            c.lens.fill_(n)
            for x, y in zip(c.run(), want):
                assert torch.equal(x, y)
        out, lse = c.run(window_size=1000)  # a window behind the table
        assert not bool(out.any()) and bool(torch.isposinf(lse).all())
    for most in (2 ** 62, 2 ** 31):
        c.run(max_query_len=most, max_seq_len=most)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads", [257, 600])
def test_gpu_many_key_heads(kv_heads):
    """More key heads than there are workgroups to deal work out to."""
    c = Case(27, [1500, 3], [2, 1], heads=kv_heads, kv_heads=kv_heads, dim=64)
    c.check()
    Case(28, [1100], [70], heads=kv_heads, kv_heads=kv_heads, dim=64).check()
