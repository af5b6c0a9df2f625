"""mxfp4_kv_quant_and_cache: codes and scale bytes equal to the definition in 64
bits, the cache's layout, strides and skipped slots; its refusals."""
import pytest
import torch

import flaggems_vllm as fv
from flaggems_vllm import _native

DEV = torch.device("cuda:0")
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# 2^(i - 127), looked up: ldexp and exp2 on the GPU may be off by an ulp
POW2 = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64)


def empty_cache(blocks, heads, page, dim, fill=0xFF, device=DEV):
    return torch.full((blocks, heads, page, dim + dim // 16), fill, dtype=torch.uint8, device=device)


def parts(cache):
    """Views of a cache: key codes, value codes [blocks, heads, page, D / 2], key scales, value scales [..., D / 32]."""
    n, h, page, width = cache.shape
    dim = width * 16 // 17
    flat, a, b = cache.reshape(n, h, page * width), page * dim // 2, page * dim // 32
    cut = (0, a, 2 * a, 2 * a + b, 2 * a + 2 * b)
    return [flat[:, :, cut[i]:cut[i + 1]].unflatten(2, (page, -1)) for i in range(4)]


def quantise(x):
    """Packed codes [..., D / 2] and scale bytes [..., D / 32] of x [..., D], by the definition in 64 bits."""
    y = x.double().unflatten(-1, (-1, 32))
    most = y.abs().amax(-1)
    bad = ~torch.isfinite(y).all(-1)
    m, e = torch.frexp(torch.where(bad, 1.0, most))  # most = m 2^e: ceil(log2(most / 6)) = e - 3, one more above 3/4
    k = torch.where(most > 0, e - 3 + (m > 0.75).int(), -126).clamp(-126, 125)
    z = torch.where(bad[..., None], 0.0, y * POW2.to(y.device)[127 - k.long()][..., None])
    off = (z.abs()[..., None] - E2M1.to(z.device)).abs()
    near = off.amin(-1, keepdim=True)
    tied = off == near  # at most two, next to one another: the even code of them
    order = torch.arange(8, device=z.device)
    code = torch.where(tied, order + 100 * (order % 2), 1000).amin(-1) % 100
    code = torch.where(bad[..., None], 0, code + 8 * torch.signbit(z).long()).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), torch.where(bad, 255, k + 127).to(torch.uint8)


def values(codes, scales):
    """The 64-bit values of packed codes under their scale bytes (255: NaN)."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    x = E2M1.to(codes.device)[c & 7] * (1.0 - 2.0 * (c >> 3).double())
    s = POW2.to(scales.device)[scales.long()]
    s = torch.where(scales == 255, torch.nan, s)
    return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def expected(cache, k, v, slots):
    """The cache (on the CPU) with the tokens written, one after the other."""
    cache = cache.cpu().clone()
    n, h, page, _ = cache.shape
    kc, vc, ks, vs = parts(cache)
    for rows, codes, scales in ((k, kc, ks), (v, vc, vs)):
        c, s = (x.cpu() for x in quantise(rows))
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < n * page:
                codes[slot // page, :, slot % page] = c[t]
                scales[slot // page, :, slot % page] = s[t]
    return cache


def check(k, v, cache, slots):
    want = expected(cache, k, v, slots)
    fv.mxfp4_kv_quant_and_cache(k, v, cache, slots)
    torch.cuda.synchronize()
    assert torch.equal(cache.cpu(), want)


def rows(seed, *shape, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-8, 9, shape[:-1], generator=g).float())[..., None]
    return x.to(dtype).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (3, 5, 16), (33, 8, 48), (257, 2, 128), (1000, 3, 16)])
def test_gpu_insert(dtype, dim, tokens, heads, page):
    print(f"\n[case] insert {dtype} {dim} {tokens} {heads} {page}", flush=True)
    blocks = tokens // page + 3
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(blocks * page, generator=g)[:tokens].to(DEV)
    slots[tokens // 2] = -1
    slots[tokens // 3] = blocks * page + 5
    check(rows(1, tokens, heads, dim, dtype=dtype), rows(2, tokens, heads, dim, dtype=dtype),
          empty_cache(blocks, heads, page, dim), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_every_value(dtype):
    """All 65536 patterns of the type, under block maxima of their own size and up to 12 binades above it,
    infinities, NaN and subnormals among them; every tie between two codes is met."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    for up in range(13):
        # 31 values and, above them, one that sets the scale
        x = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(up)) if up > 8 else torch.arange(65536)]
        x = x[:65536 // 31 * 31].view(-1, 31)
        top = (x.float().abs().amax(1, keepdim=True) * 2.0 ** up).to(dtype)
        x = torch.cat((x, top), 1)
        x = torch.cat((x, x[:(-len(x)) % 4]))  # heads of 128
        k = x.view(-1, 1, 128).to(DEV)
        n = len(k)
        print(f"\n[case] every value {dtype} up {up} rows {n}", flush=True)
        check(k, k.flip(2), empty_cache((n + 15) // 16, 1, 16, 128), torch.arange(n, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_ties_and_scales(dtype):
    """Every border between codes at every scale of the type, on both sides of zero; blocks of zeros."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 0.0, 0.125])
    lo, hi = (-133, 128) if dtype == torch.bfloat16 else (-24, 16)
    x = torch.cat([torch.cat((borders, -borders))[None] * 2.0 ** e for e in range(lo, hi)]).double()
    top = torch.finfo(dtype).max
    x = x.clamp(-top, top).to(dtype)
    x = torch.cat((x, torch.zeros((-len(x)) % 2 + 2, 32, dtype=dtype), -torch.zeros(2, 32, dtype=dtype)))
    k = x.view(-1, 1, 64).to(DEV)
    check(k, -k, empty_cache((len(k) + 31) // 32, 1, 32, 64), torch.arange(len(k), device=DEV))


@pytest.mark.gpu
def test_gpu_strides_and_offsets():
    """k and v out of a fused projection's rows at any element, a cache out of a wider buffer, fewer slots than rows."""
    for off in (0, 1, 3, 8):
        for dim, heads in ((128, 4), (64, 3)):
            print(f"\n[case] strides off {off} dim {dim}", flush=True)
            wide = rows(off, 50, 3 * heads * dim + 19, dtype=torch.bfloat16)
            k = wide[:, off:off + heads * dim].unflatten(1, (heads, dim))
            v = wide[:, off + heads * dim + 1:off + 2 * heads * dim + 1].unflatten(1, (heads, dim))
            v = v if off else v.transpose(0, 1).contiguous().transpose(0, 1)
            buf = torch.full((7, heads * 16 * (dim + dim // 16) + 48), 0xAB, dtype=torch.uint8, device=DEV)
            cache = buf[:, 32:-16].unflatten(1, (heads, 16, -1))
            before = buf.clone()
            slots = torch.randperm(7 * 16, generator=torch.Generator().manual_seed(off))[:41].to(DEV)
            check(k, v, cache, slots)
            buf[:, 32:-16] = before[:, 32:-16]
            assert torch.equal(buf, before)  # nothing beside the blocks


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    page, heads, dim = 64, 8, 128
    blocks = (5 << 30) // (page * heads * 136)
    cache = torch.zeros(blocks, heads, page, 136, dtype=torch.uint8, device=DEV)
    k, v = rows(1, 70, heads, dim, dtype=torch.bfloat16), rows(2, 70, heads, dim, dtype=torch.bfloat16)
    slots = torch.arange(blocks * page - 70, blocks * page, device=DEV)
    fv.mxfp4_kv_quant_and_cache(k, v, cache, slots)
    want = expected(cache[-3:] * 0, k, v, slots.cpu() - (blocks - 3) * page)
    assert torch.equal(cache[-3:].cpu(), want)
    assert not bool(cache[:4].any())


@pytest.mark.gpu
def test_gpu_other_stream_graph_and_nothing():
    k, v = rows(3, 20, 2, 128, dtype=torch.float16), rows(4, 20, 2, 128, dtype=torch.float16)
    slots = torch.arange(20, device=DEV)
    want = expected(empty_cache(2, 2, 16, 128), k, v, slots)
    side = torch.cuda.Stream()
    cache = empty_cache(2, 2, 16, 128)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fv.mxfp4_kv_quant_and_cache(k, v, cache, slots)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(cache.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fv.mxfp4_kv_quant_and_cache(k, v, cache, slots)
    for _ in range(3):
        cache.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.cpu(), want)
    fv.mxfp4_kv_quant_and_cache(k[:0], v[:0], cache, slots[:0])
    fv.mxfp4_kv_quant_and_cache(k, v, cache[:0], slots)
    assert torch.equal(cache.cpu(), want)


def cpu_args(**kw):
    a = dict(k=torch.zeros(5, 2, 128, dtype=torch.bfloat16), v=torch.zeros(5, 2, 128, dtype=torch.bfloat16),
             kv_cache=torch.zeros(3, 2, 16, 136, dtype=torch.uint8), slot_mapping=torch.zeros(5, dtype=torch.int64))
    return {**a, **kw}


BF = torch.bfloat16


@pytest.mark.parametrize("kw", [
    dict(),  # CPU tensors
    dict(kv_cache=torch.zeros(3, 2, 16, 128, dtype=torch.uint8)), dict(kv_cache=torch.zeros(3, 2, 16, 136)),
    dict(kv_cache=torch.zeros(3, 2, 24, 136, dtype=torch.uint8)), dict(kv_cache=torch.zeros(3, 2, 0, 136, dtype=torch.uint8)),
    dict(kv_cache=torch.zeros(3, 2, 136, 16, dtype=torch.uint8).transpose(2, 3)),
    dict(kv_cache=torch.zeros(3, 3, 16, 136, dtype=torch.uint8)), dict(kv_cache=torch.zeros(3, 2, 4112, 136, dtype=torch.uint8)),
    dict(k=torch.zeros(5, 2, 64, dtype=BF)), dict(k=torch.zeros(5, 256, dtype=BF)), dict(v=torch.zeros(4, 2, 128, dtype=BF)),
    dict(v=torch.zeros(5, 2, 128, dtype=torch.float16)), dict(k=torch.zeros(5, 2, 128), v=torch.zeros(5, 2, 128)),
    dict(k=torch.zeros(5, 2, 256, dtype=BF)[..., ::2]), dict(slot_mapping=torch.zeros(6, dtype=torch.int64)),
    dict(slot_mapping=torch.zeros(5, dtype=torch.int32)), dict(slot_mapping=torch.zeros(10, dtype=torch.int64)[::2]),
    dict(k=torch.zeros(5, 2, 128, dtype=BF, requires_grad=True)),
])
def test_refusals(kw):
    with pytest.raises(AssertionError):
        fv.mxfp4_kv_quant_and_cache(**cpu_args(**kw))


def test_refuses_a_cache_over_its_inputs():
    cache = torch.zeros(3, 2, 16, 136, dtype=torch.uint8)
    k = cache.view(-1)[:5 * 2 * 128 * 2].view(BF).view(5, 2, 128)
    with pytest.raises(AssertionError, match="overlap"):
        fv.mxfp4_kv_quant_and_cache(**cpu_args(kv_cache=cache, k=k))


@pytest.mark.parametrize("kw,code", [
    (dict(dim=96), -2), (dict(dtype=2), -2), (dict(page=8), -2), (dict(page=0), -2), (dict(tokens=-1), -2), (dict(heads=-1), -2),
    (dict(blocks=-1), -2), (dict(page=4112, stride=1 << 30), -5), (dict(heads=65537), -5), (dict(tokens=1 << 40), -5),
    (dict(k=None), -1), (dict(cache=None), -1), (dict(slots=None), -1), (dict(stride=16 * 2 * 136 - 16), -4),
    (dict(stride=16 * 2 * 136 + 8), -4), (dict(cache=24), -3), (dict(slots=20), -3), (dict(k=17), -3),
])
def test_c_abi_refusals(kw, code):
    a = dict(k=16, v=16, dtype=0, tokens=4, heads=2, dim=128, cache=16, stride=16 * 2 * 136, blocks=3, page=16, slots=16)
    a.update(kw)
    rc = _native.lib().fgv_mxfp4_kv_quant_and_cache(a["k"], 256, 128, a["v"], 256, 128, a["dtype"], a["tokens"], a["heads"],
                                                    a["dim"], a["cache"], a["stride"], a["blocks"], a["page"], a["slots"], None)
    assert rc == code and _native.lib().fgv_last_error()
