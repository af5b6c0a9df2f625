"""fused_add_rms_norm_quant and fused_silu_mul_quant against their definition in
64 bits: every code, the scales and the residual sum.

Codes: equal, all of them.  In the norm the rounded quotient 127 h w / max|h w|
(448 for e4m3fn) is a ratio of integers of at most 42 bits, so binary64 tells
on which side of a border it lies; in the activation a quotient within 1e-9 of a
border is left out (binary64's exp is good to 2^-52, so nothing else can move).
Scales: formed in binary64 and rounded once, a relative 2^-24 from the 64-bit
value, plus 2^-50 for the sums.  The residual sum: one rounding of an exact
binary32 sum of two 16-bit values is the nearest 16-bit value, so it is equal.
"""
import pytest
import torch

import flaggems_vllm as fv

DEV = torch.device("cuda:0")
I8, F8 = torch.int8, torch.float8_e4m3fn
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
EPS = 1e-6
GROUP = 128


def _say(msg):
    print(f"\n[case] {msg}", flush=True)


# ------------------------------------------------------------ 64-bit oracle ----

def e4m3_nearest(v):
    """The e4m3fn value nearest to each |v| <= 448 (ties to even), in 64 bits."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=-6).to(F64) - 3)
    return torch.round(v / step) * step


def quantise64(y, dtype):
    """(codes as 64-bit values, largest magnitudes, steps from the nearest border) of the 64-bit rows y."""
    rows, cols = y.shape
    q = 127.0 if dtype == I8 else 448.0
    z = y.view(rows, -1, cols if dtype == I8 else GROUP)
    most = z.abs().amax(2, keepdim=True)  # (NaN goes through)
    ok = torch.isfinite(most) & (most > 0)
    t = torch.where(ok, z * q / torch.where(ok, most, 1.0), 0.0)
    codes = torch.round(t) if dtype == I8 else e4m3_nearest(t)
    step = 1.0 if dtype == I8 else torch.exp2((torch.frexp(t)[1] - 1).clamp(min=-6).to(F64) - 3)
    border = ((t / step).abs().frac() - 0.5).abs()
    return codes.view(rows, cols), most.squeeze(2), border.view(rows, cols)


def norm64(x, residual, weight, dtype, eps=EPS):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hd = h.to(F64)
    ss = (hd * hd).sum(1, keepdim=True)
    r = 1.0 / torch.sqrt(ss / x.shape[1] + eps)
    r = torch.where(torch.isfinite(ss), r, torch.nan)
    codes, most, _ = quantise64(hd * weight.to(F64), dtype)
    scales = torch.where(torch.isfinite(most), most * r / (127.0 if dtype == I8 else 448.0), torch.nan)
    return codes, scales, h


def silu64(x, dtype):
    g, u = x.to(F64).chunk(2, 1)
    codes, most, border = quantise64(g / (1 + torch.exp(-g)) * u, dtype)
    scales = torch.where(torch.isfinite(most), most / (127.0 if dtype == I8 else 448.0), torch.nan)
    return codes, scales, border


def check_scales(got, ref):
    got, ref = got.cpu().to(F64), ref
    assert got.shape == ref.shape
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    # a value past binary32's range (200 * 3e38 / 127) rounds to infinity
    over = torch.isinf(ref.to(F32))
    assert torch.equal(torch.isinf(got), over)
    err = (got - ref).abs()
    # below 2^-126 a binary32 has an absolute step of 2^-149
    limit = ref * (2.0 ** -24 + 2.0 ** -50) + 2.0 ** -150
    assert bool((err <= limit)[~nan & ~over].all()), (err / ref)[~nan & ~over].max()


def check_codes(got, ref, border=None):
    got = got.cpu().to(F64)
    assert got.shape == ref.shape
    off = got != ref
    if border is not None:
        off &= border > 1e-9
    assert not bool(off.any()), (int(off.sum()), got[off][:4], ref[off][:4])


def check_norm(x, residual, weight, dtype, eps=EPS, **kw):
    got = fv.fused_add_rms_norm_quant(x.to(DEV), None if residual is None else residual.to(DEV), weight.to(DEV), eps,
                                      dtype, **kw)
    torch.cuda.synchronize()
    codes, scales, h = norm64(x, residual, weight, dtype, eps)
    assert got[0].dtype == dtype and got[1].dtype == F32 and got[2].dtype == x.dtype
    same = (got[2].cpu() == h) | (torch.isnan(got[2].cpu()) & torch.isnan(h))
    assert bool(same.all())
    check_scales(got[1], scales)
    check_codes(got[0], codes)


# ------------------------------------------------------------------- inputs ----

def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _x(rows, cols, dtype, seed, scale=1.0):
    return (torch.randn(rows, cols, generator=_gen(seed)) * scale).to(dtype)


def _weight(cols, dtype, seed):
    return (1 + 0.3 * torch.randn(cols, generator=_gen(seed))).to(dtype)


# --------------------------------------------------------------------- norm ----

# widths each side of every thread layout's limit, odd ones, one column
WIDTHS = [1, 7, 8, 63, 511, 512, 513, 1023, 1025, 2048, 2049, 4095, 4097, 8192, 8193, 16385, 32769, 65536]


@pytest.mark.gpu
@pytest.mark.parametrize("cols", WIDTHS)
def test_gpu_norm_int8_widths(cols):
    _say(f"norm int8 cols {cols}")
    rows = 5 if cols <= 8192 else 2
    check_norm(_x(rows, cols, BF16, 1), _x(rows, cols, BF16, 2), _weight(cols, BF16, 3), I8)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [128, 384, 512, 640, 1024, 1920, 2176, 4096, 7168, 8320, 16512, 33024, 65536])
def test_gpu_norm_fp8_widths(cols):
    _say(f"norm fp8 cols {cols}")
    rows = 5 if cols <= 8192 else 2
    check_norm(_x(rows, cols, BF16, 1), _x(rows, cols, BF16, 2), _weight(cols, BF16, 3), F8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("f32_weight", [False, True])
@pytest.mark.parametrize("with_residual", [False, True])
def test_gpu_norm_types(dtype, kind, f32_weight, with_residual):
    """Enough rows that elements beside a border, one in some thousand, occur in every combination."""
    _say(f"norm {dtype} {kind} f32 weight {f32_weight} residual {with_residual}")
    rows, cols = 70, 1536
    check_norm(_x(rows, cols, kind, 4), _x(rows, cols, kind, 5, 3.0) if with_residual else None,
               _weight(cols, F32 if f32_weight else kind, 6), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 255, 257, 1030])
def test_gpu_norm_rows(rows):
    _say(f"norm rows {rows}")
    check_norm(_x(rows, 256, BF16, 7), _x(rows, 256, BF16, 8), _weight(256, BF16, 9), I8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
def test_gpu_norm_ties(dtype):
    """Values on a coarse grid under a maximum that puts many quotients exactly on a border."""
    _say(f"norm ties {dtype}")
    g = _gen(10)
    x = torch.randint(-254, 255, (40, 512), generator=g).float() / 2
    x[:, 0::128] = 127.0          # int8: quotient = the value, ties at every half
    if dtype == F8:
        x[:, 0::128] = 448.0 / 4  # e4m3fn: quotient = 4 x the value
    check_norm(x.to(F16), None, torch.ones(512, dtype=F16), dtype)
    check_norm(x.to(BF16), None, torch.full((512,), 2.0, dtype=F32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("f32_weight", [False, True])
def test_gpu_norm_extremes(dtype, f32_weight):
    """Zero rows, products past binary32's range both ways, huge spreads, infinities and NaN, one per row."""
    _say(f"norm extremes {dtype} f32 weight {f32_weight}")
    cols = 512
    x = _x(12, cols, BF16, 11)
    w = _weight(cols, F32 if f32_weight else BF16, 12)
    w[5], w[200], w[300] = 1e30, 1e-30, 0.0
    x[0] = 0
    x[1] *= 1e38            # the product overflows binary32
    x[2] *= 1e-38           # ... and leaves its normal range
    x[3, 7] = torch.inf
    x[4, 130] = -torch.inf
    x[5, 300] = torch.nan   # under a weight of 0
    x[6, :256] = 0
    x[7] = 1e-20
    x[8, 5] = 3e38
    x[9] = 3e38
    x[10] = -0.0
    check_norm(x, None, w, dtype)
    check_norm(x, _x(12, cols, BF16, 13), w, dtype)


@pytest.mark.gpu
def test_gpu_norm_residual_cancels_and_overflows():
    """x + residual = 0 in whole rows; sums past fp16's range become infinite, as in torch."""
    _say("norm residual cancels")
    x = _x(4, 1000, F16, 14)
    res = -x.clone()
    res[1] = 7
    x[2, 3], res[2, 3] = 60000.0, 60000.0
    check_norm(x, res, _weight(1000, F16, 15), I8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("where", ["x", "residual", "beside"])
def test_gpu_norm_in_place_and_strided(dtype, where):
    """Rows out of wider buffers at an odd element offset; hidden written over x, over residual, or into
    columns beside x of the same buffer.  What lies around the rows stays as it was."""
    _say(f"norm in place {where} {dtype}")
    rows, cols, wide = 9, 1280, 2 * 1280 + 43
    bx = _x(rows, wide, BF16, 16).to(DEV)
    br = _x(rows, wide, BF16, 17).to(DEV)
    w = _weight(cols, BF16, 18)
    x, res = bx[:, 3:3 + cols], br[:, 5:5 + cols]
    x0, r0, bx0, br0 = x.clone(), res.clone(), bx.clone(), br.clone()
    out = {"x": x, "residual": res, "beside": bx[:, 1290:1290 + cols]}[where]
    codes, scales, hidden = fv.fused_add_rms_norm_quant(x, res, w.to(DEV), EPS, dtype, hidden_out=out)
    torch.cuda.synchronize()
    assert hidden.data_ptr() == out.data_ptr()
    rc, rs, rh = norm64(x0.cpu(), r0.cpu(), w, dtype)
    check_codes(codes, rc)
    check_scales(scales, rs)
    assert torch.equal(hidden.cpu(), rh)
    # restore what was to be written: nothing else may have changed
    {"x": bx, "residual": br, "beside": bx}[where][:, {"x": 3, "residual": 5, "beside": 1290}[where]:][:, :cols] = \
        {"x": bx0, "residual": br0, "beside": bx0}[where][:, {"x": 3, "residual": 5, "beside": 1290}[where]:][:, :cols]
    assert torch.equal(bx, bx0) and torch.equal(br, br0)


@pytest.mark.gpu
def test_gpu_norm_broadcast_inputs():
    """One row expanded to many (row stride 0), as x and as residual."""
    _say("norm broadcast")
    x = _x(1, 640, BF16, 19)
    res = _x(6, 640, BF16, 20)
    w = _weight(640, BF16, 21)
    for a, b in ((x.expand(6, 640), res), (res, x.expand(6, 640))):
        got = fv.fused_add_rms_norm_quant(a.to(DEV) if a.stride(0) else x.to(DEV).expand(6, 640),
                                          b.to(DEV) if b.stride(0) else x.to(DEV).expand(6, 640), w.to(DEV), EPS, F8)
        codes, scales, h = norm64(a, b, w, F8)
        check_codes(got[0], codes)
        check_scales(got[1], scales)
        assert torch.equal(got[2].cpu(), h)


@pytest.mark.gpu
def test_gpu_norm_eps_decides_tiny_rows():
    _say("norm eps")
    x = _x(3, 300, F16, 22, 1e-4)
    for eps in (1e-12, 1e-5, 1.0):
        check_norm(x, None, _weight(300, F16, 23), I8, eps)


@pytest.mark.gpu
def test_gpu_norm_codes_end_at_the_row():
    """The code and hidden buffers past the last row, through the C ABI with padded rows, keep their bytes."""
    from flaggems_vllm import _native

    _say("norm guard bytes")
    rows, cols = 3, 37
    x, res, w = _x(rows, cols, BF16, 24).to(DEV), _x(rows, cols, BF16, 25).to(DEV), _weight(cols, BF16, 26).to(DEV)
    codes = torch.full((rows + 1, 51), 99, dtype=I8, device=DEV)
    hidden = torch.full((rows + 1, 44), 5.0, dtype=BF16, device=DEV)
    scales = torch.full((rows + 1, 2), -1.0, device=DEV)
    rc = _native.lib().fgv_add_rms_norm_quant(x.data_ptr(), cols, res.data_ptr(), cols, w.data_ptr(), 0,
                                              hidden.data_ptr(), 44, codes.data_ptr(), 51, scales.data_ptr(), 2, rows,
                                              cols, EPS, 0, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    ref = norm64(x.cpu(), res.cpu(), w.cpu(), I8)
    check_codes(codes[:rows, :cols], ref[0])
    check_scales(scales[:rows, :1], ref[1])
    assert bool((codes[:, cols:] == 99).all()) and bool((codes[rows] == 99).all())
    assert bool((hidden[:, cols:] == 5.0).all()) and bool((hidden[rows] == 5.0).all())
    assert bool((scales[:, 1] == -1.0).all()) and bool((scales[rows] == -1.0).all())


# --------------------------------------------------------------------- silu ----

def check_silu(x, dtype):
    codes, scales = fv.fused_silu_mul_quant(x.to(DEV) if not x.is_cuda else x, dtype)
    torch.cuda.synchronize()
    rc, rs, border = silu64(x.cpu(), dtype)
    assert codes.dtype == dtype and scales.dtype == F32
    check_scales(scales, rs)
    check_codes(codes, rc, border)


def _gate_up(rows, cols, kind, seed):
    g = _gen(seed)
    return torch.cat([torch.randn(rows, cols, generator=g) * 3 - 1, torch.randn(rows, cols, generator=g)], 1).to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", WIDTHS)
def test_gpu_silu_int8_widths(cols):
    _say(f"silu int8 cols {cols}")
    check_silu(_gate_up(5 if cols <= 8192 else 2, cols, BF16, 31), I8)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [128, 384, 512, 1024, 1920, 4096, 8320, 16512, 65536])
def test_gpu_silu_fp8_widths(cols):
    _say(f"silu fp8 cols {cols}")
    check_silu(_gate_up(5 if cols <= 8192 else 2, cols, BF16, 32), F8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind", [BF16, F16])
def test_gpu_silu_types(dtype, kind):
    _say(f"silu {dtype} {kind}")
    check_silu(_gate_up(130, 1408, kind, 33), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
def test_gpu_silu_extremes(dtype):
    """Zero rows; gates at which exp under- and overflows, beside up values that bring the product back into
    range; products past binary32; infinities and NaN."""
    _say(f"silu extremes {dtype}")
    cols = 384
    x = _gate_up(14, cols, BF16, 34)
    g, u = x[:, :cols], x[:, cols:]
    x[0] = 0
    u[1] = 0
    g[2] = -95.0                      # sigmoid below binary32's normal range
    g[3], u[3] = -95.0, u[3] * 1e37   # ... and the product back in it
    g[4, 5], u[4, 5] = -80.0, 3e38
    g[5], u[5] = 200.0, 3e38          # the product past binary32
    g[6], u[6] = g[6] * 1e-30, u[6] * 1e-30
    g[7, 9] = torch.inf
    g[8, 9] = -torch.inf
    u[9, 130] = torch.nan
    u[10, 383] = -torch.inf
    g[11] = torch.linspace(-130, 130, cols).to(BF16)
    g[12] = torch.linspace(-130, 0, cols).to(BF16)
    u[12] = 1.0
    u[13] = 1e38
    check_silu(x, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("gate", [-60.0, -85.0, -87.0, -104.0, -2.0 ** 20, -2.0 ** 30, -1e20, -1e38, -3e38])
def test_gpu_silu_far_negative_gates(dtype, gate):
    """Gates of which nothing is left, one or many to a row, beside ordinary values, under small and large up
    values: their products are 0, however far out they lie, and the largest magnitude is the others'."""
    _say(f"silu far negative gates {gate} {dtype}")
    cols = 256
    x = _gate_up(6, cols, BF16, 38)
    g, u = x[:, :cols], x[:, cols:]
    g[0, 17] = gate
    g[1, ::2] = gate
    g[2] = gate                       # nothing else in the row
    g[3, 5], u[3, 5] = gate, 1e6
    g[4, 5], u[4, 5] = gate, 3e38
    g[5, 1::2], u[5, 0::2] = gate, 1e-12
    check_silu(x, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
def test_gpu_silu_strided(dtype):
    """Rows out of a wider buffer, at an odd offset."""
    _say(f"silu strided {dtype}")
    buf = torch.randn(7, 2 * 896 + 29, generator=_gen(35)).to(F16).to(DEV)
    check_silu(buf[:, 11:11 + 2 * 896], dtype)


@pytest.mark.gpu
def test_gpu_silu_every_bf16_gate():
    """All finite bf16 gates under an up value of 1: the largest value of each row is in the same row, so the
    codes and scales go through every magnitude of the activation."""
    _say("silu every gate")
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF16)
    gates = bits[torch.isfinite(bits)]
    gates = gates[gates.float().abs().argsort()]
    n = gates.numel() // 256 * 256
    gates = gates[:n].view(-1, 256)
    check_silu(torch.cat([gates, torch.ones_like(gates)], 1), I8)
    check_silu(torch.cat([gates, torch.ones_like(gates)], 1), F8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("dtype,cols", [(I8, 9), (I8, 300), (I8, 1000), (I8, 3001), (I8, 9000), (I8, 20000),
                                        (F8, 128), (F8, 640), (F8, 4224), (F8, 20480)])
def test_gpu_silu_extremes_at_widths(dtype, cols, kind):
    """What leaves the binary32 path, in the first, a middle and the last element of rows of every thread layout."""
    _say(f"silu extremes {dtype} {cols} {kind}")
    big = torch.finfo(kind).max
    specials = [(0.0, big), (-big, 1.0), (-big, big), (big, big), (torch.inf, 1.0), (-torch.inf, 1.0), (torch.nan, 0.0),
                (1.0, torch.inf), (0.0, torch.inf), (-100.0, torch.inf), (1.0, torch.nan), (-20.0, big), (30.0, 1e-5)]
    places = [0, cols // 2, cols - 1]
    x = _gate_up(3 * len(specials) + 1, cols, kind, 45)
    for i, (g, u) in enumerate(specials):
        for j, at in enumerate(places):
            x[3 * i + j, at], x[3 * i + j, cols + at] = g, u
    x[-1] *= 1e-7
    check_silu(x, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cols", [(I8, 9), (I8, 300), (I8, 1000), (I8, 3001), (I8, 9000), (I8, 20000), (I8, 40000),
                                        (F8, 128), (F8, 640), (F8, 4224), (F8, 20480)])
def test_gpu_norm_extremes_at_widths(dtype, cols):
    """The same of the norm, by the row (infinities, NaN, products past binary32) and by the weight."""
    _say(f"norm extremes {dtype} {cols}")
    x, res = _x(14, cols, BF16, 46), _x(14, cols, BF16, 47)
    for i, at in enumerate((0, cols // 2, cols - 1)):
        x[i, at] = torch.inf
        x[3 + i, at] = torch.nan
        x[6 + i, at] = 3e38
        x[9 + i] = 0
        x[9 + i, at] = 1e-38
    x[12], res[12] = 0, 0
    w = _weight(cols, F32, 48)
    check_norm(x, None, w, dtype)
    check_norm(x, res, w, dtype)
    for value in (torch.inf, torch.nan, 3e38, 1e-40, -2.0):
        w = _weight(cols, F32, 48)
        w[cols // 2] = value
        check_norm(x, res, w, dtype)
    check_norm(x, res, torch.zeros(cols, dtype=BF16), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
def test_gpu_inference_mode(dtype):
    """The outputs of calls under inference mode are those of calls outside it."""
    _say(f"inference mode {dtype}")
    x = _x(5, 512, BF16, 49).to(DEV)
    w = _weight(256, BF16, 50).to(DEV)
    ref = fv.fused_silu_mul_quant(x, dtype), fv.fused_add_rms_norm_quant(x[:, :256], x[:, 256:], w, EPS, dtype)
    with torch.inference_mode():
        got = fv.fused_silu_mul_quant(x, dtype), fv.fused_add_rms_norm_quant(x[:, :256], x[:, 256:], w, EPS, dtype)
        if dtype == I8:
            mm = fv.int8_scaled_mm(got[0][0], got[1][0], got[0][1], got[1][1])
            assert torch.equal(mm, fv.int8_scaled_mm(ref[0][0], ref[1][0], ref[0][1], ref[1][1]))
    for a, b in zip(ref[0] + ref[1], got[0] + got[1]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ----------------------------------------------------------- both, elsewhere ----

def _free_gib():
    return torch.cuda.mem_get_info()[0] / 2 ** 30


@pytest.mark.gpu
def test_gpu_norm_more_rows_than_a_launch():
    """2^25 + 9 rows of 8 columns, 64 threads to a row: 2^31 threads and more, so the call takes two launches."""
    _say("norm 2^25 + 9 rows")
    rows = 2 ** 25 + 9
    g = torch.Generator(DEV).manual_seed(40)
    x = torch.randn(rows, 8, generator=g, device=DEV, dtype=BF16)
    res = torch.randn(rows, 8, generator=g, device=DEV, dtype=BF16)
    w = _weight(8, BF16, 41).to(DEV)
    codes, scales, h = fv.fused_add_rms_norm_quant(x, res, w, EPS)
    for lo in (0, 2 ** 25 - 40, rows - 50):
        ref = norm64(x[lo:lo + 50].cpu(), res[lo:lo + 50].cpu(), w.cpu(), I8)
        check_codes(codes[lo:lo + 50], ref[0])
        check_scales(scales[lo:lo + 50], ref[1])
        assert torch.equal(h[lo:lo + 50].cpu(), ref[2])
    for lo in range(0, rows, 2 ** 23):
        hi = min(rows, lo + 2 ** 23)
        c, s, hh = fv.fused_add_rms_norm_quant(x[lo:hi], res[lo:hi], w, EPS)
        assert torch.equal(c, codes[lo:hi]) and torch.equal(s, scales[lo:hi]) and torch.equal(hh, h[lo:hi])


@pytest.mark.gpu
def test_gpu_silu_more_rows_than_a_launch():
    """2^23 + 9 rows of one 128-column group, 256 threads to a row: two launches, and offsets past 2^32 bytes."""
    _say("silu 2^23 + 9 rows")
    if _free_gib() < 16:
        pytest.skip("needs 16 GiB of device memory")
    rows = 2 ** 23 + 9
    x = torch.randn(rows, 256, generator=torch.Generator(DEV).manual_seed(42), device=DEV, dtype=BF16)
    codes, scales = fv.fused_silu_mul_quant(x, F8)
    for lo in (0, 2 ** 23 - 40, rows - 50):
        ref = silu64(x[lo:lo + 50].cpu(), F8)
        check_codes(codes[lo:lo + 50], ref[0], ref[2])
        check_scales(scales[lo:lo + 50], ref[1])
    for lo in range(0, rows, 2 ** 21):
        hi = min(rows, lo + 2 ** 21)
        c, s = fv.fused_silu_mul_quant(x[lo:hi], F8)
        assert torch.equal(c.view(torch.uint8), codes[lo:hi].view(torch.uint8)) and torch.equal(s, scales[lo:hi])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,first,cols", [
    (F8, 65535 * 4, 128),   # a wave to a row, four rows to a workgroup, 65535 workgroups along the rows
    (I8, 2 ** 25, 8),       # 64 threads to a row, 2^31 threads
])
def test_gpu_silu_rows_of_a_second_launch(dtype, first, cols):
    """A few rows more than the first launch takes: those each side of its end, and all of them against calls that
    take one launch."""
    _say(f"silu rows past a launch {dtype}")
    rows = first + 9
    x = torch.randn(rows, 2 * cols, generator=torch.Generator(DEV).manual_seed(52), device=DEV, dtype=BF16)
    codes, scales = fv.fused_silu_mul_quant(x, dtype)
    for lo in (0, first - 40, rows - 50):
        ref = silu64(x[lo:lo + 50].cpu(), dtype)
        check_codes(codes[lo:lo + 50], ref[0], ref[2])
        check_scales(scales[lo:lo + 50], ref[1])
    step = first // 4 + 1
    for lo in range(0, rows, step):
        c, s = fv.fused_silu_mul_quant(x[lo:lo + step], dtype)
        assert torch.equal(c.view(torch.uint8), codes[lo:lo + step].view(torch.uint8))
        assert torch.equal(s, scales[lo:lo + step])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, F8])
def test_gpu_offsets_past_32_bits(dtype):
    """33000 rows of 65536 columns: more than 2^31 elements, 2^32 bytes, in each tensor."""
    _say(f"norm and silu offsets past 32 bits {dtype}")
    if _free_gib() < 40:
        pytest.skip("needs 40 GiB of device memory")
    rows, cols = 33000, 65536
    x = torch.randn(rows, cols, generator=torch.Generator(DEV).manual_seed(43), device=DEV, dtype=BF16)
    res = x.flip(0)
    w = _weight(cols, BF16, 44).to(DEV)
    codes, scales, h = fv.fused_add_rms_norm_quant(x, res, w, EPS, dtype)
    for lo in (0, 32766, rows - 2):
        ref = norm64(x[lo:lo + 2].cpu(), res[lo:lo + 2].cpu(), w.cpu(), dtype)
        check_codes(codes[lo:lo + 2], ref[0])
        check_scales(scales[lo:lo + 2], ref[1])
        assert torch.equal(h[lo:lo + 2].cpu(), ref[2])
    del res, h, codes, scales
    both = torch.cat([x, x.flip(0)], 1)
    codes, scales = fv.fused_silu_mul_quant(both, dtype)
    for lo in (0, 32766, rows - 2):
        ref = silu64(both[lo:lo + 2].cpu(), dtype)
        check_codes(codes[lo:lo + 2], ref[0], ref[2])
        check_scales(scales[lo:lo + 2], ref[1])


@pytest.mark.gpu
def test_gpu_no_rows():
    _say("no rows")
    x = torch.empty(0, 256, dtype=BF16, device=DEV)
    c, s, h = fv.fused_add_rms_norm_quant(x, x, torch.ones(256, dtype=BF16, device=DEV), EPS)
    assert c.shape == (0, 256) and s.shape == (0, 1) and h.shape == (0, 256)
    c, s = fv.fused_silu_mul_quant(x, F8)
    assert c.shape == (0, 128) and s.shape == (0, 1)


@pytest.mark.gpu
def test_gpu_other_stream():
    """Inputs made on a side stream, the calls on that stream: ordered there."""
    _say("side stream")
    side = torch.cuda.Stream()
    xs = _x(300, 2048, BF16, 36)
    w = _weight(2048, BF16, 37)
    with torch.cuda.stream(side):
        x = xs.to(DEV, non_blocking=True)
        for _ in range(3):
            x = x.clone()
        codes, scales, hidden = fv.fused_add_rms_norm_quant(x, x, w.to(DEV), EPS)
        c2, s2 = fv.fused_silu_mul_quant(hidden)
    side.synchronize()
    rc, rs, rh = norm64(xs, xs, w, I8)
    check_codes(codes, rc)
    check_scales(scales, rs)
    rc, rs, border = silu64(rh, I8)
    check_codes(c2, rc, border)
    check_scales(s2, rs)


# ----------------------------------------------------------------- refusals ----

def _norm_args(**over):
    a = dict(x=torch.zeros(4, 256, dtype=BF16), residual=torch.zeros(4, 256, dtype=BF16),
             weight=torch.zeros(256, dtype=BF16), eps=1e-6)
    a.update(over)
    return a


_SHARED = torch.zeros(4, 600, dtype=BF16)


@pytest.mark.parametrize("bad,match", [
    (dict(x=torch.zeros(4, 2, 128, dtype=BF16)), "must be 2D"),
    (dict(x=torch.zeros(4, 256)), "x's type or float32"),
    (dict(x=torch.zeros(4, 256), residual=None, weight=torch.zeros(256)), "bfloat16 or float16"),
    (dict(x=torch.zeros(256, 4, dtype=BF16).t()), "rows must be contiguous"),
    (dict(x=torch.zeros(4, 0, dtype=BF16), residual=None, weight=torch.zeros(0, dtype=BF16)), "1 to 65536"),
    (dict(x=torch.zeros(1, 65537, dtype=BF16), residual=None, weight=torch.zeros(65537, dtype=BF16)), "1 to 65536"),
    (dict(residual=torch.zeros(4, 255, dtype=BF16)), "residual must have"),
    (dict(residual=torch.zeros(4, 256, dtype=F16)), "residual must have"),
    (dict(residual=torch.zeros(256, 4, dtype=BF16).t()), "residual's rows"),
    (dict(weight=torch.zeros(255, dtype=BF16)), "weight must be"),
    (dict(weight=torch.zeros(512, dtype=BF16)[::2]), "weight must be"),
    (dict(weight=torch.zeros(256, dtype=F16)), "x's type or float32"),
    (dict(eps=0.0), "eps must be positive"),
    (dict(eps=float("nan")), "eps must be positive"),
    (dict(eps=float("inf")), "eps must be positive"),
    (dict(dtype=torch.uint8), "dtype must be"),
    (dict(dtype=torch.float8_e5m2), "dtype must be"),
    (dict(x=torch.zeros(4, 200, dtype=BF16), residual=None, weight=torch.zeros(200, dtype=BF16), dtype=F8),
     "multiple of 128"),
    (dict(x=torch.zeros(4, 256, dtype=BF16, requires_grad=True)), "inference only"),
    (dict(weight=torch.zeros(256, dtype=BF16, requires_grad=True)), "inference only"),
    (dict(residual=None, hidden_out=torch.zeros(4, 256, dtype=BF16)), "needs a residual"),
    (dict(hidden_out=torch.zeros(4, 255, dtype=BF16)), "hidden_out must have"),
    (dict(hidden_out=torch.zeros(4, 256, dtype=F16)), "hidden_out must have"),
    (dict(hidden_out=torch.zeros(1, 256, dtype=BF16).expand(4, 256)), "contiguous and apart"),
    (dict(x=_SHARED[:, :256], hidden_out=_SHARED[:, 8:264]), "apart from every input"),     # shifted rows
    (dict(residual=_SHARED[:, :256], hidden_out=_SHARED[:, 255:511]), "apart from every input"),
    (dict(weight=_SHARED[0, :256], hidden_out=_SHARED[:, 100:356]), "apart from every input"),
    ({}, "GPU"),
])
def test_norm_refuses(bad, match):
    with pytest.raises(AssertionError, match=match):
        fv.fused_add_rms_norm_quant(**_norm_args(**bad))


def test_norm_hidden_beside_x_passes_the_checks():
    """Rows side by side in one buffer are apart: the call gets as far as asking for a GPU."""
    for out in (_SHARED[:, 256:512], _SHARED[:, 300:556], _SHARED[:, :256]):
        with pytest.raises(AssertionError, match="GPU"):
            fv.fused_add_rms_norm_quant(**_norm_args(x=_SHARED[:, :256], hidden_out=out))


@pytest.mark.parametrize("x,kw,match", [
    (torch.zeros(4, 3, 256, dtype=BF16), {}, "must be 2D"),
    (torch.zeros(4, 255, dtype=BF16), {}, "gate beside up"),
    (torch.zeros(4, 256), {}, "bfloat16 or float16"),
    (torch.zeros(256, 4, dtype=BF16).t(), {}, "rows must be contiguous"),
    (torch.zeros(4, 200, dtype=BF16), dict(dtype=F8), "multiple of 128"),
    (torch.zeros(4, 0, dtype=BF16), {}, "1 to 65536"),
    (torch.zeros(1, 2 * 65537, dtype=BF16), {}, "1 to 65536"),
    (torch.zeros(4, 256, dtype=BF16, requires_grad=True), {}, "inference only"),
    (torch.zeros(4, 256, dtype=BF16), dict(dtype=torch.int16), "dtype must be"),
    (torch.zeros(4, 256, dtype=BF16), {}, "GPU"),
])
def test_silu_refuses(x, kw, match):
    with pytest.raises(AssertionError, match=match):
        fv.fused_silu_mul_quant(x, **kw)


def test_weights_that_train_elsewhere_pass_without_grad_mode():
    """A parameter is taken as it is where no gradient is recorded."""
    with torch.no_grad(), pytest.raises(AssertionError, match="GPU"):
        fv.fused_add_rms_norm_quant(**_norm_args(weight=torch.zeros(256, dtype=BF16, requires_grad=True)))


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), -2), (dict(cols=0), -2), (dict(cols=65537), -5), (dict(rows=1 << 31), -5),
    (dict(cols=200, code=1), -2), (dict(eps=0.0), -2), (dict(eps=float("inf")), -2), (dict(kind=2), -2), (dict(code=2), -2),
    (dict(x=None), -1), (dict(codes=None), -1), (dict(scales=None), -1), (dict(w=None), -1),
    (dict(hidden=None), -1), (dict(x=17), -3), (dict(scales=18), -3), (dict(w=18, w32=1), -3), (dict(rows=0, x=None), 0),
])
def test_norm_c_abi_rejects(kw, code):
    from flaggems_vllm import _native

    a = dict(x=16, res=16, w=16, w32=0, hidden=16, codes=16, scales=16, rows=4, cols=256, eps=1e-6, kind=0, code=0)
    a.update(kw)
    rc = _native.lib().fgv_add_rms_norm_quant(a["x"], 256, a["res"], 256, a["w"], a["w32"], a["hidden"], 256,
                                              a["codes"], 256, a["scales"], 1, a["rows"], a["cols"], a["eps"],
                                              a["kind"], a["code"], None)
    assert rc == code


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), -2), (dict(cols=0), -2), (dict(cols=1 << 40), -5), (dict(cols=100, code=1), -2),
    (dict(x=None), -1), (dict(codes=None), -1), (dict(scales=None), -1), (dict(x=17), -3), (dict(rows=0), 0),
])
def test_silu_c_abi_rejects(kw, code):
    from flaggems_vllm import _native

    a = dict(x=16, codes=16, scales=16, rows=4, cols=256, kind=0, code=0)
    a.update(kw)
    rc = _native.lib().fgv_silu_mul_quant(a["x"], 512, a["codes"], 256, a["scales"], 1, a["rows"], a["cols"],
                                          a["kind"], a["code"], None)
    assert rc == code


@pytest.mark.parametrize("cols", [-1, 5 - (1 << 32), 256 - (1 << 40), -(1 << 63)])
def test_c_abi_rejects_negative_widths_of_any_size(cols):
    """Also those whose low 32 bits are a width that exists (no rows, so that nothing could be launched)."""
    from flaggems_vllm import _native

    L = _native.lib()
    assert L.fgv_add_rms_norm_quant(16, 256, 16, 256, 16, 0, 16, 256, 16, 256, 16, 1, 0, cols, 1e-6, 0, 0, None) == -2
    assert L.fgv_silu_mul_quant(16, 512, 16, 256, 16, 1, 0, cols, 0, 0, None) == -2
