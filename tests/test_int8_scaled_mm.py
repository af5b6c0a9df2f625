"""int8_scaled_mm against its definition: the exact integer sum, then
(sum * scale_a) * scale_b + bias.

Two references.  In 64 bits: the kernel rounds the sum to binary32, the two
products and the addition, each by at most 2^-24 of its value, and the output by
half a step of its type; a product's rounding carries through, so
  |out - ref| <= eps/2 |ref| + 2^-22 (|sum scale_a scale_b| + |bias|)
(four roundings of 2^-24 of terms no larger than that; fp16's subnormal step
2^-25 is added).  And bit for bit: the same chain of separately rounded binary32
operations on the exact sum, which leaves no freedom (zeros compare equal).
"""
import pytest
import torch

import flaggems_vllm as fv

DEV = torch.device("cuda:0")
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _say(msg):
    print(f"\n[case] {msg}", flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _codes(rows, cols, seed):
    return torch.randint(-128, 128, (rows, cols), generator=_gen(seed), dtype=torch.int32).to(torch.int8)


def _scales(n, seed):
    return torch.rand(n, generator=_gen(seed)) * 0.01 + 1e-4


def exact_sum(a, b):
    """a b^T in binary64 on the GPU: every partial sum is a whole number below 2^31."""
    return (a.to(DEV).double() @ b.to(DEV).double().t()).cpu()


def check(out, a, b, sa, sb, bias, out_dtype):
    assert out.dtype == out_dtype and out.shape == (a.shape[0], b.shape[0])
    total = exact_sum(a, b) if a.shape[1] else torch.zeros(a.shape[0], b.shape[0], dtype=F64)
    sa, sb = sa.reshape(-1, 1), sb.reshape(1, -1)
    ref = total * sa.to(F64) * sb.to(F64)
    size = ref.abs()
    if bias is not None:
        ref = ref + bias.to(F64)
        size = size + bias.to(F64).abs()
    got = out.cpu()
    limit = torch.finfo(out_dtype).eps / 2 * ref.abs() + 2.0 ** -22 * size + (2.0 ** -25 if out_dtype == F16 else 0)
    err = (got.to(F64) - ref).abs()
    assert bool((err <= limit).all()), float((err / limit.clamp(min=1e-300)).max())
    chain = total.to(F32) * sa * sb
    if bias is not None:
        chain = chain + bias.to(F32)
    assert bool((got == chain.to(out_dtype)).all())


def run(m, n, k, out_dtype=BF16, bias_dtype=None, seed=0, **kw):
    a, b = _codes(m, k, seed + 1), _codes(n, k, seed + 2)
    sa, sb = _scales(m, seed + 3), _scales(n, seed + 4)
    bias = None if bias_dtype is None else torch.randn(n, generator=_gen(seed + 5)).to(bias_dtype)
    out = fv.int8_scaled_mm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), None if bias is None else bias.to(DEV),
                            out_dtype, **kw)
    torch.cuda.synchronize()
    check(out, a, b, sa, sb, bias, out_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 127, 128, 129, 192, 255, 256, 257, 513])
def test_gpu_rows(m):
    _say(f"int8 mm rows {m}")
    run(m, 272, 384, seed=m)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 127, 129, 255, 256, 257, 511, 769])
@pytest.mark.parametrize("m", [3, 300])
def test_gpu_channels(m, n):
    _say(f"int8 mm channels {n} rows {m}")
    run(m, n, 256, F16, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [0, 1, 2, 15, 16, 17, 63, 64, 65, 112, 127, 128, 129, 144, 240, 255, 256, 257, 384, 400,
                               511, 512, 640, 1024, 1040, 2047, 2048, 4111])
@pytest.mark.parametrize("m", [5, 40, 290])
def test_gpu_sums(m, k):
    _say(f"int8 mm sum {k} rows {m}")
    run(m, 130, k, F32, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [7, 150, 520])
@pytest.mark.parametrize("out_dtype,bias_dtype", [(BF16, None), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32),
                                                  (F32, None), (F32, F32)])
def test_gpu_types(m, out_dtype, bias_dtype):
    _say(f"int8 mm rows {m} {out_dtype} bias {bias_dtype}")
    run(m, 320, 1152, out_dtype, bias_dtype, seed=m)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 7168, 2048), (24, 2048, 7168), (64, 1024, 4096), (200, 1536, 2048),
                                   (300, 2304, 1024), (700, 1024, 3584), (1021, 1031, 1111), (1024, 1024, 1024),
                                   (2048, 2048, 512), (2500, 4096, 640), (4096, 4096, 256)])
def test_gpu_sizes(m, n, k):
    """Sizes that take every schedule: rows from memory, split sums, small and large tiles, ragged edges."""
    _say(f"int8 mm {m} x {n} x {k}")
    run(m, n, k, seed=m + n)


# sizes with ragged edges that take, on 256 CUs, workgroups straight from memory (split 64 x 64 tiles at the longest
# sum), 64 x 64, 128 x 64, 128 x 128, 128 x 192, 192 x 128, 256 x 128, 192 x 256, 256 x 192 and 256 x 256 tiles
TILE_SIZES = [(300, 300), (500, 1030), (1000, 1030), (1000, 2050), (1021, 4099), (1500, 4090), (2000, 3900),
              (3000, 4090), (4090, 3000), (4000, 4090)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", TILE_SIZES)
@pytest.mark.parametrize("k", [128, 256, 384, 640, 1111, 2064, 5120])
def test_gpu_every_tile(m, n, k):
    """From fewer K blocks than a ring has stages to many; a K that is no multiple of 128, and rows that start at
    any byte."""
    _say(f"int8 mm tiles {m} x {n} x {k}")
    run(m, n, k, F16 if k == 384 else BF16, F32 if k in (384, 1111) else None, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", TILE_SIZES)
def test_gpu_every_tile_float32(m, n):
    _say(f"int8 mm tiles {m} x {n} float32")
    run(m, n, 1024, F32, F32 if m in (500, 4000) else None, seed=m)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", TILE_SIZES)
def test_gpu_every_tile_writes_its_rows_only(m, n):
    """out as a view into a wider buffer: what lies around it stays."""
    _say(f"int8 mm tiles {m} x {n} into a wider buffer")
    a, b, sa, sb = _codes(m, 256, 1), _codes(n, 256, 2), _scales(m, 3), _scales(n, 4)
    buf = torch.full((m + 2, n + 21), 3.0, dtype=BF16, device=DEV)
    got = fv.int8_scaled_mm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), out=buf[1:m + 1, 13:13 + n])
    torch.cuda.synchronize()
    check(got, a, b, sa, sb, None, BF16)
    buf[1:m + 1, 13:13 + n] = 3.0
    assert bool((buf == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(40000, 60000, 128),      # the output: 2^31 elements and more
                                   (2 ** 20, 72, 4224),      # a: past 2^32 bytes, straight and (next) packed
                                   (2 ** 20, 72, 4223),
                                   (5, 2 ** 21, 2176),       # b: the same, rows from memory
                                   (300, 2 ** 21, 2176),     # b: in tiles, straight and packed
                                   (300, 2 ** 21, 2175)])
def test_gpu_offsets_past_32_bits(m, n, k):
    """The first and last rows and channels, and those each side of the middle."""
    _say(f"int8 mm {m} x {n} x {k}")
    if torch.cuda.mem_get_info()[0] < 24 * 2 ** 30:
        pytest.skip("needs 24 GiB of device memory")
    g = torch.Generator(DEV).manual_seed(m + n)
    a = torch.empty(m, k, dtype=torch.int8, device=DEV).random_(-128, 128, generator=g)
    b = torch.empty(n, k, dtype=torch.int8, device=DEV).random_(-128, 128, generator=g)
    sa, sb = _scales(m, 3), _scales(n, 4)
    out = fv.int8_scaled_mm(a, b, sa.to(DEV), sb.to(DEV))
    pick = [torch.unique(torch.cat([torch.arange(min(40, x)), torch.arange(max(0, x // 2 - 20), min(x, x // 2 + 20)),
                                    torch.arange(max(0, x - 40), x)])) for x in (m, n)]
    rows, cols = pick[0].to(DEV), pick[1].to(DEV)
    check(out[rows][:, cols], a[rows], b[cols], sa[pick[0]], sb[pick[1]], None, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 70), (3, 4100), (9, 4096), (20, 4111), (31, 130), (40, 4000), (64, 4096), (100, 2000)])
@pytest.mark.parametrize("k", [127, 129, 383, 1023, 2049, 4111])
@pytest.mark.parametrize("a_at,b_at", [(0, 0), (1, 2), (3, 1), (2, 3)])
def test_gpu_few_rows_at_any_byte(m, n, k, a_at, b_at):
    """Rows that start at any byte of a word, a's and b's apart: what lies before and behind each row in its words
    must not count.  The neighbours' bytes are the largest there are."""
    _say(f"int8 mm few rows {m} x {n} x {k} at {a_at}, {b_at}")
    def placed(codes, at, pad):
        buf = torch.full((codes.shape[0] * (k + pad) + 16,), 127, dtype=torch.int8, device=DEV)
        view = buf.as_strided((codes.shape[0], k), (k + pad, 1), at)
        view.copy_(codes)
        return view
    a, b, sa, sb = _codes(m, k, 1), _codes(n, k, 2), _scales(m, 3), _scales(n, 4)
    out = fv.int8_scaled_mm(placed(a, a_at, 2 - k % 2), placed(b, b_at, 1), sa.to(DEV), sb.to(DEV))
    check(out, a, b, sa, sb, None, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [20, 300, 1500])
def test_gpu_broadcast_rows(m):
    """One row of a for every token and one of b for every channel, as expanded views, under one scale each."""
    _say(f"int8 mm broadcast rows {m}")
    a, b = _codes(1, 640, 1), _codes(1, 640, 2)
    sa, sb = torch.tensor([0.01]), torch.tensor([0.02])
    out = fv.int8_scaled_mm(a.to(DEV).expand(m, 640), b.to(DEV).expand(600, 640), sa.to(DEV), sb.to(DEV))
    check(out, a.expand(m, 640), b.expand(600, 640), sa, sb, None, BF16)


# sizes that split 64 x 64 tiles along K on 256 CUs, 3 to 7 times at the longest
SPLIT_SIZES = [(330, 600), (450, 333), (257, 1000), (48, 2048), (100, 601)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", SPLIT_SIZES)
@pytest.mark.parametrize("k,out_dtype,bias_dtype", [(2048, BF16, None), (2064, F16, F32), (3001, F32, F32), (5120, BF16, BF16),
                                                    (7168, F16, F16), (7168, F32, None)])
def test_gpu_split_sums(m, n, k, out_dtype, bias_dtype):
    """Whole and cut K blocks, packed rows, every output; twice, into a view of a wider buffer the second time."""
    _say(f"int8 mm split {m} x {n} x {k} {out_dtype} bias {bias_dtype}")
    run(m, n, k, out_dtype, bias_dtype, seed=k)
    a, b, sa, sb = _codes(m, k, 1), _codes(n, k, 2), _scales(m, 3), _scales(n, 4)
    buf = torch.full((m + 2, n + 5), 3.0, dtype=out_dtype, device=DEV)
    got = fv.int8_scaled_mm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), None, out_dtype, out=buf[1:m + 1, 3:3 + n])
    torch.cuda.synchronize()
    check(got, a, b, sa, sb, None, out_dtype)
    buf[1:m + 1, 3:3 + n] = 3.0
    assert bool((buf == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(400, 600, 4096), (500, 700, 4111)])
def test_gpu_workspaces_apart(m, n, k):
    """Calls with workspaces: in flight at once on two streams, and in two graphs of one pool, replayed in turn
    with eager calls between."""
    from flaggems_vllm import _native

    _say(f"int8 mm workspaces {m} x {n} x {k}")
    data = [(_codes(m, k, s).to(DEV), _codes(n, k, s + 1).to(DEV)) for s in (61, 71)]
    sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
    assert _native.lib().fgv_int8_scaled_mm_workspace_bytes(data[0][0].data_ptr(), k, data[0][1].data_ptr(), k, m, n,
                                                            k) > 0
    expect = [fv.int8_scaled_mm(a, b, sa, sb) for a, b in data]
    torch.cuda.synchronize()
    for out, (a, b) in zip(expect, data):
        check(out, a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None, BF16)
    streams, outs = [torch.cuda.Stream() for _ in data], [[], []]
    for _ in range(4):
        for i, (a, b) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                outs[i].append(fv.int8_scaled_mm(a, b, sa, sb))
    torch.cuda.synchronize()
    assert all(torch.equal(out, e) for got, e in zip(outs, expect) for out in got)
    graphs, outs, pool = [], [], None
    for a, b in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(fv.int8_scaled_mm(a, b, sa, sb))
        pool = g.pool()
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for i in order:
            outs[i].zero_()
            fv.int8_scaled_mm(*data[1 - i], sa, sb)
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], expect[i]), (order, i)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(300, 300, 5120), (1000, 1030, 1111), (300, 700, 384), (2000, 3000, 256)])
def test_gpu_without_workspace(m, n, k):
    """The C ABI without a workspace, or with one too small: the same bits straight from memory."""
    from flaggems_vllm import _native

    _say(f"int8 mm without workspace {m} x {n} x {k}")
    L = _native.lib()
    a, b = _codes(m, k, 1).to(DEV), _codes(n, k, 2).to(DEV)
    sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
    ref = fv.int8_scaled_mm(a, b, sa, sb)
    need = L.fgv_int8_scaled_mm_workspace_bytes(a.data_ptr(), k, b.data_ptr(), k, m, n, k)
    assert (need > 0) == ((m, n, k) in ((300, 300, 5120), (1000, 1030, 1111)))
    small = torch.full((256,), 7, dtype=torch.uint8, device=DEV)
    for ws, size in ((None, 0), (small.data_ptr(), min(256, need - 1) if need else 256)):
        out = torch.empty(m, n, dtype=BF16, device=DEV)
        rc = L.fgv_int8_scaled_mm(a.data_ptr(), k, b.data_ptr(), k, sa.data_ptr(), 1, sb.data_ptr(), 1, None, 0,
                                  out.data_ptr(), n, m, n, k, 0, ws, size, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and bool((small == 7).all())


@pytest.mark.gpu
def test_gpu_workspace_is_enough():
    """Guard bytes behind a workspace of exactly the size asked for stay as they were."""
    from flaggems_vllm import _native

    _say("int8 mm workspace guard")
    L = _native.lib()
    for m, n, k in ((300, 300, 5120), (401, 733, 3001), (1000, 1030, 1111)):
        a, b = _codes(m, k, 1).to(DEV), _codes(n, k, 2).to(DEV)
        sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
        need = L.fgv_int8_scaled_mm_workspace_bytes(a.data_ptr(), k, b.data_ptr(), k, m, n, k)
        ws = torch.full((need + 4096,), 7, dtype=torch.uint8, device=DEV)
        out = torch.empty(m, n, dtype=BF16, device=DEV)
        rc = L.fgv_int8_scaled_mm(a.data_ptr(), k, b.data_ptr(), k, sa.data_ptr(), 1, sb.data_ptr(), 1, None, 0,
                                  out.data_ptr(), n, m, n, k, 0, ws.data_ptr(), need,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and need > 0
        check(out, a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None, BF16)
        assert bool((ws[need:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 33, 300])
def test_gpu_largest_sum(m):
    """The largest sum there is, 131071 products of (-128)^2, and its negative: int32 holds both."""
    _say(f"int8 mm largest sum, rows {m}")
    k, n = 131071, 20
    a = torch.full((m, k), -128, dtype=torch.int8)
    b = torch.full((n, k), -128, dtype=torch.int8)
    b[1::2] = 127
    sa, sb = _scales(m, 1), _scales(n, 2)
    out = fv.int8_scaled_mm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV), None, F32)
    check(out, a, b, sa, sb, None, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 40, 300])
@pytest.mark.parametrize("pad,offset", [(16, 0), (16, 16), (48, 16), (1, 0), (7, 3), (16, 1)])
def test_gpu_strided_rows(m, pad, offset):
    """Rows out of wider buffers: 16-byte aligned ones and others; out into the middle of a wider buffer whose
    other columns and rows stay as they were."""
    _say(f"int8 mm strided rows {m} pad {pad} offset {offset}")
    n, k = 140, 400
    A, B = _codes(m, k + pad + offset, 1), _codes(n, k + pad + offset, 2)
    a, b = A.to(DEV)[:, offset:offset + k], B.to(DEV)[:, offset:offset + k]
    sa, sb = _scales(m, 3), _scales(n, 4)
    buf = torch.full((m + 1, n + 9), 3.0, dtype=BF16, device=DEV)
    got = fv.int8_scaled_mm(a, b, sa.to(DEV), sb.to(DEV), out=buf[:m, 5:5 + n])
    torch.cuda.synchronize()
    assert got.data_ptr() == buf[:, 5:].data_ptr()
    check(got, a.cpu(), b.cpu(), sa, sb, None, BF16)
    rest = buf.clone()
    rest[:m, 5:5 + n] = 3.0
    assert bool((rest == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 300])
def test_gpu_scale_layouts(m):
    """One scale, [M, 1], [N, 1], [1, N], strided and expanded scales; rows expanded from one."""
    _say(f"int8 mm scale layouts rows {m}")
    n, k = 96, 256
    a, b = _codes(m, k, 1), _codes(n, k, 2)
    sa, sb = _scales(m, 3), _scales(n, 4)
    wide_a, wide_b = torch.zeros(m, 3), torch.zeros(n, 5)
    wide_a[:, 1], wide_b[:, 2] = sa, sb
    ad, bd = a.to(DEV), b.to(DEV)
    for x, y in ((sa[:, None], sb[None]), (sa, sb[:, None]), (wide_a.to(DEV)[:, 1], wide_b.to(DEV)[:, 2:3]),
                 (torch.tensor([0.5]), sb), (sa, torch.tensor(0.25)), (torch.tensor([[0.5]]), torch.tensor([[0.25]])),
                 (torch.tensor([0.5]).expand(m), sb)):
        out = fv.int8_scaled_mm(ad, bd, x.to(DEV), y.to(DEV), None, F32)
        check(out, a, b, x.cpu().reshape(-1).expand(m), y.cpu().reshape(-1).expand(n), None, F32)
    out = fv.int8_scaled_mm(ad[:1].expand(m, k), bd, sa.to(DEV), sb.to(DEV), None, F32)
    check(out, a[:1].expand(m, k), b, sa, sb, None, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 300])
def test_gpu_scales_that_are_not_finite(m):
    """The scale of a row with a NaN (as the quantising ops write it) makes that row NaN and no other; an
    infinite channel scale reaches its channel alone."""
    _say(f"int8 mm NaN scales rows {m}")
    a, b = _codes(m, 256, 1).abs().clamp(min=1), _codes(40, 256, 2).abs().clamp(min=1)
    sa, sb = _scales(m, 3), _scales(40, 4)
    sa[1], sb[7] = torch.nan, torch.inf
    out = fv.int8_scaled_mm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV)).cpu()
    nan, inf = torch.isnan(out), torch.isinf(out)
    assert bool(nan[1].all()) and int(nan.sum()) == 40
    assert bool(inf[torch.arange(m) != 1, 7].all()) and int(inf.sum()) == m - 1


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(3, 70, 256), (40, 130, 384), (300, 300, 5120), (500, 1030, 384), (1000, 1030, 1111)])
def test_gpu_sign_of_zero(m, n, k, out_dtype):
    """Sums of zero under scales of either sign, without a bias: (0 * scale_a) * scale_b has the scales' sign, in
    every schedule and with or without a workspace; a bias of zero makes it +0."""
    from flaggems_vllm import _native

    _say(f"int8 mm sign of zero {m} x {n} x {k} {out_dtype}")
    L = _native.lib()
    a, b = torch.zeros(m, k, dtype=torch.int8, device=DEV), _codes(n, k, 2).to(DEV)
    sa, sb = _scales(m, 3), _scales(n, 4)
    sa[::3] *= -1
    sb[::2] *= -1
    negative = torch.signbit(sa)[:, None] ^ torch.signbit(sb)[None]
    sa, sb = sa.to(DEV), sb.to(DEV)
    out = fv.int8_scaled_mm(a, b, sa, sb, None, out_dtype)
    bare = torch.empty_like(out)
    rc = L.fgv_int8_scaled_mm(a.data_ptr(), k, b.data_ptr(), k, sa.data_ptr(), 1, sb.data_ptr(), 1, None, 0,
                              bare.data_ptr(), n, m, n, k, (BF16, F16, F32).index(out_dtype), None, 0,
                              torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    biased = fv.int8_scaled_mm(a, b, sa, sb, torch.zeros(n, device=DEV), out_dtype)
    for got in (out, bare, biased):
        assert not bool(got.any())
    assert torch.equal(torch.signbit(out).cpu(), negative) and torch.equal(torch.signbit(bare).cpu(), negative)
    assert not bool(torch.signbit(biased).any())


# (tokens, channels, sum, bytes behind each row) that tiles could only take packed
FEW_ROWS_OF_WIDE_WEIGHTS = [(17, 16384, 2880, 0), (24, 16384, 2880, 0), (32, 10240, 2368, 0), (24, 8704, 7008, 16),
                            (32, 9000, 5136, 48), (24, 16384, 2879, 0), (32, 8224, 1375, 2)]


@pytest.mark.parametrize("m,n,k,pad", FEW_ROWS_OF_WIDE_WEIGHTS)
def test_few_rows_do_not_copy_the_weights(m, n, k, pad):
    """Up to 32 tokens read b once; a call that packs it first reads it twice and writes it."""
    from flaggems_vllm import _native

    assert _native.lib().fgv_int8_scaled_mm_workspace_bytes(16, k + pad, 16, k + pad, m, n, k) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,pad", FEW_ROWS_OF_WIDE_WEIGHTS)
def test_gpu_few_rows_of_wide_weights(m, n, k, pad):
    _say(f"int8 mm few rows {m} x {n} x {k} pad {pad}")
    a, b, sa, sb = _codes(m, k, 1), _codes(n, k, 2), _scales(m, 3), _scales(n, 4)
    wide = [torch.full((x.shape[0], k + pad), 127, dtype=torch.int8, device=DEV) for x in (a, b)]
    for w, x in zip(wide, (a, b)):
        w[:, :k] = x.to(DEV)
    out = fv.int8_scaled_mm(wide[0][:, :k], wide[1][:, :k], sa.to(DEV), sb.to(DEV))
    torch.cuda.synchronize()
    check(out, a, b, sa, sb, None, BF16)


@pytest.mark.gpu
def test_gpu_empty():
    _say("int8 mm empty")
    e = torch.empty(0, 64, dtype=torch.int8, device=DEV)
    f = torch.zeros(3, 64, dtype=torch.int8, device=DEV)
    one = torch.ones(1, device=DEV)
    assert fv.int8_scaled_mm(e, f, torch.empty(0, device=DEV), one).shape == (0, 3)
    assert fv.int8_scaled_mm(f, e, one, torch.empty(0, device=DEV)).shape == (3, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [24, 200, 1030])
def test_gpu_same_bits_every_time(m):
    """Two calls in a row on other data, and the first again: no call sees another's workspace."""
    _say(f"int8 mm repeated rows {m}")
    n, k = 1536, 2048
    pairs = [(_codes(m, k, s).to(DEV), _codes(n, k, s + 1).to(DEV)) for s in (1, 11)]
    sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
    first = [fv.int8_scaled_mm(a, b, sa, sb) for a, b in pairs]
    again = [fv.int8_scaled_mm(a, b, sa, sb) for a, b in pairs]
    torch.cuda.synchronize()
    for x, y, (a, b) in zip(first, again, pairs):
        assert torch.equal(x, y)
        check(x, a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None, BF16)


@pytest.mark.gpu
def test_gpu_two_streams():
    """Two calls in flight at once on two streams, each with its own data."""
    _say("int8 mm two streams")
    m, n, k = 200, 1536, 2048
    data = [(_codes(m, k, s).to(DEV), _codes(n, k, s + 1).to(DEV)) for s in (21, 31)]
    sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in data], [[], []]
    for _ in range(4):
        for i, (a, b) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                outs[i].append(fv.int8_scaled_mm(a, b, sa, sb))
    torch.cuda.synchronize()
    for (a, b), got in zip(data, outs):
        check(got[0], a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None, BF16)
        assert all(torch.equal(got[0], g) for g in got[1:])


# sums cut along K, packed rows, packed rows of few tokens, and both at once
WORKSPACE_SIZES = [(400, 600, 4096), (500, 700, 1111), (40, 8224, 2880), (257, 1000, 3001)]


@pytest.mark.parametrize("m,n,k", WORKSPACE_SIZES + [(200, 1536, 2048), (500, 700, 4111)])
def test_sizes_that_need_a_workspace(m, n, k):
    """Those of the next test, and of the calls in flight together above."""
    from flaggems_vllm import _native

    assert _native.lib().fgv_int8_scaled_mm_workspace_bytes(256, k, 256, k, m, n, k) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", WORKSPACE_SIZES)
def test_gpu_calls_in_a_row_with_workspaces(m, n, k):
    """Calls on other data, one after the other without a pause, whose workspaces take each other's memory."""
    _say(f"int8 mm workspaces in a row {m} x {n} x {k}")
    pairs = [(_codes(m, k, s).to(DEV), _codes(n, k, s + 1).to(DEV)) for s in (1, 11, 21)]
    sa, sb = _scales(m, 3).to(DEV), _scales(n, 4).to(DEV)
    runs = [[fv.int8_scaled_mm(a, b, sa, sb) for a, b in pairs] for _ in range(3)]
    torch.cuda.synchronize()
    for out, (a, b) in zip(runs[0], pairs):
        check(out, a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None, BF16)
    assert all(torch.equal(x, y) for again in runs[1:] for x, y in zip(again, runs[0]))


# ----------------------------------------------------------------- refusals ----

def _args(**over):
    a = dict(a=torch.zeros(4, 64, dtype=torch.int8), b=torch.zeros(8, 64, dtype=torch.int8), scale_a=torch.ones(4, 1),
             scale_b=torch.ones(8))
    a.update(over)
    return a


_BUF = torch.zeros(4, 64, dtype=torch.int8)


@pytest.mark.parametrize("bad,match", [
    (dict(a=torch.zeros(4, 1, 64, dtype=torch.int8)), "must be \\[M, K\\]"),
    (dict(b=torch.zeros(8, 63, dtype=torch.int8)), "must be \\[M, K\\]"),
    (dict(a=torch.zeros(4, 64, dtype=torch.uint8)), "must be int8"),
    (dict(b=torch.zeros(8, 64)), "must be int8"),
    (dict(a=torch.zeros(64, 4, dtype=torch.int8).t()), "rows must be contiguous"),
    (dict(b=torch.zeros(64, 8, dtype=torch.int8).t()), "rows must be contiguous"),
    (dict(scale_a=torch.ones(5)), "scale_a"),
    (dict(scale_a=torch.ones(1, 4)), "scale_a"),
    (dict(scale_a=torch.ones(4, dtype=F64)), "scale_a"),
    (dict(scale_a=torch.ones(4, 1, 1)), "scale_a"),
    (dict(scale_b=torch.ones(7)), "scale_b"),
    (dict(scale_b=torch.ones(2, 4)), "scale_b"),
    (dict(scale_b=torch.ones(8, dtype=BF16)), "scale_b"),
    (dict(bias=torch.ones(7)), "bias must be"),
    (dict(bias=torch.ones(8, 1)), "bias must be"),
    (dict(bias=torch.ones(16)[::2]), "bias must be"),
    (dict(bias=torch.ones(8, dtype=F16)), "bias must be float32 or"),
    (dict(out_dtype=torch.int32), "out_dtype"),
    (dict(out=torch.zeros(4, 7, dtype=BF16)), "out must be"),
    (dict(out=torch.zeros(4, 8, dtype=F16)), "out must be"),
    (dict(out=torch.zeros(8, 4, dtype=BF16).t()), "contiguous and apart"),
    (dict(out=torch.zeros(1, 8, dtype=BF16).expand(4, 8)), "contiguous and apart"),
    (dict(a=_BUF, out=_BUF.view(BF16)[:, :8]), "must not overlap"),
    (dict(scale_a=torch.ones(4, requires_grad=True)), "inference only"),
    ({}, "GPU"),
])
def test_refuses(bad, match):
    with pytest.raises(AssertionError, match=match):
        fv.int8_scaled_mm(**_args(**bad))


@pytest.mark.parametrize("kw,code", [
    (dict(m=-1), -2), (dict(n=-1), -2), (dict(k=-1), -2), (dict(od=3), -2), (dict(bd=-1), -2),
    (dict(k=131072), -5), (dict(m=(1 << 20) + 1), -5), (dict(n=(1 << 24) + 1), -5),
    (dict(a=None), -1), (dict(b=None), -1), (dict(sa=None), -1), (dict(sb=None), -1), (dict(out=None), -1),
    (dict(sa=18), -3), (dict(out=17), -3), (dict(od=2, out=18), -3), (dict(bias=17), -3),
    (dict(m=0, a=None), 0), (dict(n=0, out=None), 0),
])
def test_c_abi_rejects(kw, code):
    from flaggems_vllm import _native

    p = dict(a=16, b=16, sa=16, sb=16, bias=16, bd=0, out=16, m=4, n=8, k=64, od=0)
    p.update(kw)
    rc = _native.lib().fgv_int8_scaled_mm(p["a"], 64, p["b"], 64, p["sa"], 1, p["sb"], 1, p["bias"], p["bd"],
                                          p["out"], 8, p["m"], p["n"], p["k"], p["od"], None, 0, None)
    assert rc == code
