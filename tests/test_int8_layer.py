"""The 8-bit linear ops as a layer runs them, one after the other: every step is
held to its own 64-bit reference on the step's actual inputs, so an error has
nowhere to hide behind a later one.  Also inside captured graphs, through
torch.ops and against the ops that read their outputs."""
import pytest
import torch

import flaggems_vllm as fv
import oracle
from flaggems_vllm import library

from .test_act_quant import check_codes, check_scales, norm64, silu64
from .test_fp8_einsum import _check as check_einsum
from .test_fp8_einsum import make_inputs as einsum_inputs
from .test_int8_scaled_mm import check as check_mm

DEV = torch.device("cuda:0")
I8, F8 = torch.int8, torch.float8_e4m3fn
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def _say(msg):
    print(f"\n[case] {msg}", flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(*shape, seed, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=_gen(seed)) * scale).to(dtype)


def _weights(n, k, seed):
    """int8 weights of a projection with a scale per channel, as a checkpoint holds them."""
    w = torch.randn(n, k, generator=_gen(seed)) / k ** 0.5
    s = w.abs().amax(1, keepdim=True) / 127
    return torch.round(w / s).to(I8), s


class Block:
    """A gated feed-forward block with int8 weights, and the norm in front of it."""

    def __init__(self, size, inner, seed):
        self.norm = _randn(size, seed=seed, scale=0.2) + 1
        self.w1, self.s1 = _weights(2 * inner, size, seed + 1)
        self.w2, self.s2 = _weights(size, inner, seed + 2)

    def to(self, dev):
        for k, v in vars(self).items():
            setattr(self, k, v.to(dev))
        return self

    def run(self, x, hidden, hidden_out=None):
        a8, sa, hidden = fv.fused_add_rms_norm_quant(x, hidden, self.norm, EPS, hidden_out=hidden_out)
        gate_up = fv.int8_scaled_mm(a8, self.w1, sa, self.s1)
        b8, sb = fv.fused_silu_mul_quant(gate_up)
        return (a8, sa, hidden), gate_up, (b8, sb), fv.int8_scaled_mm(b8, self.w2, sb, self.s2)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 33, 300])
@pytest.mark.parametrize("size,inner", [(1024, 1408), (515, 333)])
def test_gpu_feed_forward_block(tokens, size, inner):
    """Norm, gate and up projection, activation, down projection, twice: the second block's norm adds the first
    one's output to the residual stream, in place."""
    _say(f"int8 block tokens {tokens} size {size} inner {inner}")
    x, hidden = _randn(tokens, size, seed=1).to(DEV), _randn(tokens, size, seed=2, scale=3.0).to(DEV)
    for layer in range(2):
        block = Block(size, inner, 10 * layer + 3).to(DEV)
        x0, h0 = x.cpu(), hidden.cpu()
        (a8, sa, hidden), gate_up, (b8, sb), x = block.run(x, hidden, hidden if layer else None)
        torch.cuda.synchronize()
        codes, scales, h = norm64(x0, h0, block.norm.cpu(), I8)
        check_codes(a8, codes)
        check_scales(sa, scales)
        assert torch.equal(hidden.cpu(), h)
        check_mm(gate_up, a8.cpu(), block.w1.cpu(), sa.cpu(), block.s1.cpu(), None, BF16)
        codes, scales, border = silu64(gate_up.cpu(), I8)
        check_codes(b8, codes, border)
        check_scales(sb, scales)
        check_mm(x, b8.cpu(), block.w2.cpu(), sb.cpu(), block.s2.cpu(), None, BF16)


@pytest.mark.gpu
def test_gpu_padded_batch():
    """Rows of zeros behind the last sequence come through as zeros, whatever stands beside them, and the rows
    in front of them are those of the call without them."""
    _say("int8 block padded batch")
    block = Block(768, 512, 5).to(DEV)
    x, hidden = _randn(20, 768, seed=6).to(DEV), _randn(20, 768, seed=7).to(DEV)
    alone = block.run(x[:13], hidden[:13])[3]
    x[13:], hidden[13:] = 0, 0
    (a8, sa, h), gate_up, (b8, sb), out = block.run(x, hidden)
    assert torch.equal(out[:13], alone)
    assert not bool(a8[13:].any()) and not bool(sa[13:].any()) and not bool(h[13:].any())
    assert not bool(gate_up[13:].any()) and not bool(b8[13:].any()) and not bool(sb[13:].any())
    assert not bool(out[13:].any())


@pytest.mark.gpu
def test_gpu_one_bad_token():
    """A token with a NaN ends as NaN; the others do not see it."""
    _say("int8 block with a NaN")
    block = Block(640, 384, 8).to(DEV)
    x, hidden = _randn(9, 640, seed=9).to(DEV), _randn(9, 640, seed=10).to(DEV)
    clean = block.run(x, hidden)[3]
    x[4, 77] = torch.nan
    out = block.run(x, hidden)[3]
    assert bool(torch.isnan(out[4]).all())
    keep = torch.arange(9, device=DEV) != 4
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 24, 130])
def test_gpu_qkv_projection_feeds_the_norms(tokens):
    """Norm to int8, the fused low-rank q / kv projection, and fused_q_kv_rmsnorm on its two column ranges."""
    _say(f"int8 q/kv projection tokens {tokens}")
    size = 1280
    x, norm = _randn(tokens, size, seed=11), _randn(size, seed=12, scale=0.2) + 1
    w, s = _weights(1536 + 512, size, 13)
    qw, kw = _randn(1536, seed=14), _randn(512, seed=15)
    a8, sa, h = fv.fused_add_rms_norm_quant(x.to(DEV), None, norm.to(DEV), EPS)
    assert torch.equal(h.cpu(), x)
    qkv = fv.int8_scaled_mm(a8, w.to(DEV), sa, s.to(DEV))
    check_mm(qkv, a8.cpu(), w, sa.cpu(), s, None, BF16)
    q, kv = fv.fused_q_kv_rmsnorm(qkv[:, :1536], qkv[:, 1536:], qw.to(DEV), kw.to(DEV), EPS)
    rq, rk = oracle.fused_q_kv_rmsnorm(qkv[:, :1536].contiguous().cpu(), qkv[:, 1536:].contiguous().cpu(), qw, kw, EPS)
    assert torch.equal(q.cpu(), rq) and torch.equal(kv.cpu(), rk)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("op", ["norm", "silu"])
def test_gpu_fp8_codes_feed_the_block_product(tokens, op):
    """e4m3fn codes and scales per 128 columns go into fp8_einsum as they are, as one head."""
    _say(f"fp8 codes into the block product, tokens {tokens} {op}")
    size = 512
    if op == "norm":
        x, res = _randn(tokens, size, seed=16).to(DEV), _randn(tokens, size, seed=17).to(DEV)
        codes, scales, _ = fv.fused_add_rms_norm_quant(x, res, (_randn(size, seed=18, scale=0.2) + 1).to(DEV), EPS, F8)
    else:
        codes, scales = fv.fused_silu_mul_quant(_randn(tokens, 2 * size, seed=19).to(DEV), F8)
    y, ys = einsum_inputs(2, 1, size, 256, seed=20)[2:]
    out = fv.fp8_einsum("bhr,hdr->bhd", codes[:, None], scales[:, None], y.to(DEV), ys.to(DEV))
    torch.cuda.synchronize()
    check_einsum(out, codes[:, None].cpu(), scales[:, None].cpu(), y, ys, BF16)


# ------------------------------------------------------------------- graphs ----

@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_gpu_graph_of_a_block(tokens):
    """A captured block, split sums and packed rows among its schedules, replayed on changing inputs with eager
    calls of the same ops in between: every replay equals the eager call."""
    _say(f"int8 block graph tokens {tokens}")
    block = Block(1031, 2048, 21).to(DEV)
    x, hidden = torch.zeros(tokens, 1031, dtype=BF16, device=DEV), torch.zeros(tokens, 1031, dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.run(x, hidden)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (_, _, h), _, _, out = block.run(x, hidden)
    for i in range(4):
        x.copy_(_randn(tokens, 1031, seed=30 + i))
        hidden.copy_(_randn(tokens, 1031, seed=40 + i))
        (_, _, eh), _, _, eager = block.run(x, hidden)
        block.run(hidden, x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, eh) and torch.equal(out, eager), f"replay {i}"


@pytest.mark.gpu
def test_gpu_two_graphs_of_one_pool():
    """Two graphs captured into the same memory pool, each with a workspace, replayed in turn and in either order."""
    _say("int8 two graphs, one pool")
    m, n, k = 300, 300, 4096
    a = [torch.randint(-127, 128, (m, k), generator=_gen(s), dtype=torch.int32).to(I8).to(DEV) for s in (1, 2)]
    b = torch.randint(-127, 128, (n, k), generator=_gen(3), dtype=torch.int32).to(I8).to(DEV)
    one = torch.full((1,), 1e-4, device=DEV)
    expect = [fv.int8_scaled_mm(x, b, one, one) for x in a]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for x in a:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(fv.int8_scaled_mm(x, b, one, one))
        pool = g.pool()
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for i in order:
            outs[i].zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], expect[i]), (order, i)


def _workspace_bytes(m, n, k):
    from flaggems_vllm import _native

    return _native.lib().fgv_int8_scaled_mm_workspace_bytes(256, k, 256, k, m, n, k)


# block sizes whose two products take a workspace at the token counts of the next test: packed rows (a sum of 1031) and
# sums cut along K (of 2048 and 4096)
WORKSPACE_BLOCKS = [(1031, 2048, 300), (600, 4096, 400)]


@pytest.mark.parametrize("size,inner,tokens", WORKSPACE_BLOCKS)
def test_blocks_that_need_workspaces(size, inner, tokens):
    """What the next test, and the blocks of 1031 channels and 300 tokens above, rest on."""
    assert _workspace_bytes(tokens, 2 * inner, size) > 0 and _workspace_bytes(tokens, size, inner) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("size,inner,tokens", WORKSPACE_BLOCKS)
def test_gpu_two_graphs_share_their_workspaces_memory(size, inner, tokens):
    """Two captured blocks in one memory pool, so that what one graph freed is the other's too, and eager blocks in
    between: each replay gives what the block gave alone."""
    _say(f"int8 blocks in two graphs of one pool, {size} {inner} {tokens}")
    blocks = [Block(size, inner, 70 + i).to(DEV) for i in range(2)]
    ins = [(_randn(tokens, size, seed=80 + i).to(DEV), _randn(tokens, size, seed=90 + i).to(DEV)) for i in range(2)]
    expect = [block.run(*data)[3] for block, data in zip(blocks, ins)]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for block, data in zip(blocks, ins):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(block.run(*data)[3])
        pool = g.pool()
        graphs.append(g)
    for order in ((0, 1), (1, 0), (1, 1, 0), (0, 0, 1)):
        for i in order:
            outs[i].zero_()
            assert torch.equal(blocks[1 - i].run(*ins[1 - i])[3], expect[1 - i])
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], expect[i]), (order, i)


# ---------------------------------------------------------------- torch.ops ----

def _op(name):
    return getattr(torch.ops.flaggems_vllm, name).default


@pytest.mark.parametrize("name", library.REGISTERED_LINEAR)
def test_schema_declares_exactly_the_written_tensors(name):
    written = {a.name for a in _op(name)._schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert written == ({"out"} if name == "int8_scaled_mm_out" else set())


def test_fake_layouts():
    x = torch.empty(5, 512, dtype=BF16, device="meta")
    w = torch.empty(512, dtype=BF16, device="meta")
    for dtype, blocks in ((I8, 1), (F8, 4)):
        c, s, h = _op("fused_add_rms_norm_quant")(x, x, w, EPS, dtype)
        assert c.shape == (5, 512) and c.dtype == dtype and s.shape == (5, blocks) and s.dtype == F32
        assert h.shape == (5, 512) and h.dtype == BF16
        assert _op("fused_add_rms_norm_quant")(x, None, w, EPS, dtype)[2].shape == (0,)
        c, s = _op("fused_silu_mul_quant")(x, dtype)
        assert c.shape == (5, 256) and c.dtype == dtype and s.shape == (5, blocks // 2 or 1)
    a, b = torch.empty(5, 64, dtype=I8, device="meta"), torch.empty(7, 64, dtype=I8, device="meta")
    s = torch.empty(1, device="meta")
    out = _op("int8_scaled_mm")(a, b, s, s, None, torch.float16)
    assert out.shape == (5, 7) and out.dtype == torch.float16


@pytest.mark.gpu
def test_gpu_torch_ops_match_the_functions():
    _say("torch.ops of the 8-bit linear ops")
    check = dict(test_utils=("test_schema", "test_faketensor"))
    x, res = _randn(6, 512, seed=50).to(DEV), _randn(6, 512, seed=51).to(DEV)
    w = (_randn(512, seed=52, scale=0.1) + 1).to(DEV)
    bits = lambda t: t.view(torch.uint8)  # noqa: E731
    for dtype in (I8, F8):
        for r in (res, None):
            f = fv.fused_add_rms_norm_quant(x, r, w, EPS, dtype)
            o = _op("fused_add_rms_norm_quant")(x, r, w, EPS, dtype)
            assert all(torch.equal(bits(p), bits(q)) for p, q in zip(f[:2] if r is None else f, o))
            torch.library.opcheck(_op("fused_add_rms_norm_quant"), (x, r, w, EPS, dtype), **check)
        f, o = fv.fused_silu_mul_quant(x, dtype), _op("fused_silu_mul_quant")(x, dtype)
        assert all(torch.equal(bits(p), bits(q)) for p, q in zip(f, o))
        torch.library.opcheck(_op("fused_silu_mul_quant"), (x, dtype), **check)
    a8, sa = fv.fused_silu_mul_quant(x)
    b8, sb = _weights(40, 256, 53)
    b8, sb = b8.to(DEV), sb.to(DEV)
    bias = torch.randn(40, generator=_gen(54)).to(DEV)
    f = fv.int8_scaled_mm(a8, b8, sa, sb, bias)
    assert torch.equal(f, _op("int8_scaled_mm")(a8, b8, sa, sb, bias))
    out = torch.empty_like(f)
    _op("int8_scaled_mm_out")(a8, b8, sa, sb, bias, out)
    assert torch.equal(f, out)
    torch.library.opcheck(_op("int8_scaled_mm"), (a8, b8, sa, sb, bias, BF16), **check)
    torch.library.opcheck(_op("int8_scaled_mm_out"), (a8, b8, sa, sb, bias, out), **check)


# ----------------------------------------------------------- forward-mode duals ----

def _dual_calls(dev):
    """Calls in which one tensor carries a tangent, made within a dual level: {what: call}."""
    from torch.autograd.forward_ad import make_dual

    x, w = _randn(4, 256, seed=60).to(dev), (_randn(256, seed=61, scale=0.1) + 1).to(dev)
    a, b = torch.ones(4, 64, dtype=I8, device=dev), torch.ones(8, 64, dtype=I8, device=dev)
    sa, sb, bias = torch.ones(4, device=dev), torch.ones(8, device=dev), torch.zeros(8, device=dev)
    out = torch.zeros(4, 8, dtype=BF16, device=dev)
    dual = lambda t: make_dual(t, torch.ones_like(t))  # noqa: E731
    norm, mm = fv.fused_add_rms_norm_quant, fv.int8_scaled_mm
    return {"x": lambda: norm(dual(x), None, w, EPS), "residual": lambda: norm(x, dual(x), w, EPS),
            "weight": lambda: norm(x, x, dual(w), EPS, F8), "hidden_out": lambda: norm(x, x, w, EPS, hidden_out=dual(x)),
            "gate_up": lambda: fv.fused_silu_mul_quant(dual(x)), "scale_a": lambda: mm(a, b, dual(sa), sb),
            "scale_b": lambda: mm(a, b, sa, dual(sb)), "bias": lambda: mm(a, b, sa, sb, dual(bias)),
            "out": lambda: mm(a, b, sa, sb, out=dual(out))}


DUALS = ["x", "residual", "weight", "hidden_out", "gate_up", "scale_a", "scale_b", "bias", "out"]


@pytest.mark.parametrize("what", DUALS)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_refuses_tangents(what, grad_mode):
    """A tangent would be dropped without a word; no_grad does not switch tangents off."""
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        with pytest.raises(AssertionError, match="inference only.*tangent"):
            _dual_calls("cpu")[what]()


def test_duals_pass_under_inference_mode():
    """Where no derivative is recorded at all the value is taken: the call gets as far as asking for a GPU."""
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.zeros(4, 256), torch.ones(4, 256)).to(BF16)
        with torch.inference_mode(), pytest.raises(AssertionError, match="GPU"):
            fv.fused_silu_mul_quant(dual)


@pytest.mark.gpu
def test_gpu_refuses_tangents():
    """On the GPU too, and through torch.ops."""
    _say("tangents refused")
    with torch.autograd.forward_ad.dual_level():
        for what, call in _dual_calls(DEV).items():
            with pytest.raises(AssertionError, match="tangent"):
                call()
        x = torch.autograd.forward_ad.make_dual(_randn(4, 256, seed=62).to(DEV), _randn(4, 256, seed=63).to(DEV))
        with pytest.raises((AssertionError, RuntimeError, NotImplementedError)):
            _op("fused_silu_mul_quant")(x)


# ------------------------------------------------------- lazily negated views ----

def _negated_calls(dev):
    """Calls in which one tensor is a view whose values in memory have the other sign: {what: call}."""
    x, w = _randn(4, 256, seed=64).to(dev), (_randn(256, seed=65, scale=0.1) + 1).to(dev)
    a, b = torch.ones(4, 64, dtype=I8, device=dev), torch.ones(8, 64, dtype=I8, device=dev)
    sa, sb, bias = torch.ones(4, device=dev), torch.ones(8, device=dev), torch.zeros(8, device=dev)
    out = torch.zeros(4, 8, dtype=BF16, device=dev)
    neg, norm, mm = torch._neg_view, fv.fused_add_rms_norm_quant, fv.int8_scaled_mm
    imag = torch.complex(torch.zeros(8, device=dev), torch.ones(8, device=dev)).conj().imag
    assert imag.is_neg() and imag[:4].is_neg()
    return {"x": lambda: norm(neg(x), None, w, EPS), "residual": lambda: norm(x, neg(x), w, EPS),
            "weight": lambda: norm(x, x, neg(w), EPS, F8), "hidden_out": lambda: norm(x, x, w, EPS, hidden_out=neg(x)),
            "gate_up": lambda: fv.fused_silu_mul_quant(neg(x)), "a": lambda: mm(neg(a), b, sa, sb),
            "b": lambda: mm(a, neg(b), sa, sb), "scale_a": lambda: mm(a, b, imag[:4], sb),
            "scale_b": lambda: mm(a, b, sa, imag), "bias": lambda: mm(a, b, sa, sb, neg(bias)),
            "out": lambda: mm(a, b, sa, sb, out=neg(out))}


@pytest.mark.parametrize("what", ["x", "residual", "weight", "hidden_out", "gate_up", "a", "b", "scale_a", "scale_b",
                                  "bias", "out"])
def test_refuses_lazily_negated_views(what):
    with pytest.raises(AssertionError, match="lazily negated"):
        _negated_calls("cpu")[what]()


@pytest.mark.gpu
def test_gpu_negated_views():
    """Refused by the functions; torch.ops gives the kernel the negated values."""
    _say("lazily negated views")
    for call in _negated_calls(DEV).values():
        with pytest.raises(AssertionError, match="lazily negated"):
            call()
    a, b = torch.ones(4, 64, dtype=I8, device=DEV), torch.ones(8, 64, dtype=I8, device=DEV)
    imag = torch.complex(torch.zeros(8, device=DEV), torch.ones(8, device=DEV)).conj().imag
    out = _op("int8_scaled_mm")(a, b, torch.ones(4, device=DEV), imag)
    assert bool((out == -64).all())
    assert torch.equal(out, fv.int8_scaled_mm(a, b, torch.ones(4, device=DEV), imag.resolve_neg()))


# ------------------------------------------------------- tensors without memory ----

def _calls_without_memory():
    """Calls in which one tensor has no memory and its view an offset into it (an address of some hundred bytes, which
    is not null): {what: call}.  The others lie on the CPU, so that nothing could be launched."""
    def bare(t):
        base = torch.empty(t.numel() + 256, dtype=t.dtype)
        view = base[256:].view(t.shape)
        base.untyped_storage().resize_(0)
        return view

    x, w = _randn(4, 256, seed=66), _randn(256, seed=67)
    a, b = torch.ones(4, 64, dtype=I8), torch.ones(8, 64, dtype=I8)
    sa, sb, bias, out = torch.ones(4), torch.ones(8), torch.zeros(8), torch.zeros(4, 8, dtype=BF16)
    norm, mm = fv.fused_add_rms_norm_quant, fv.int8_scaled_mm
    return {"x": lambda: norm(bare(x), None, w, EPS), "residual": lambda: norm(x, bare(x), w, EPS),
            "weight": lambda: norm(x, x, bare(w), EPS, F8), "hidden_out": lambda: norm(x, x, w, EPS, hidden_out=bare(x)),
            "gate_up": lambda: fv.fused_silu_mul_quant(bare(x)), "a": lambda: mm(bare(a), b, sa, sb),
            "b": lambda: mm(a, bare(b), sa, sb), "scale_a": lambda: mm(a, b, bare(sa), sb),
            "scale_b": lambda: mm(a, b, sa, bare(sb)), "bias": lambda: mm(a, b, sa, sb, bare(bias)),
            "out": lambda: mm(a, b, sa, sb, out=bare(out))}


@pytest.mark.parametrize("what", ["x", "residual", "weight", "hidden_out", "gate_up", "a", "b", "scale_a", "scale_b",
                                  "bias", "out"])
def test_refuses_tensors_whose_memory_is_gone(what):
    """Such as a parameter whose storage a sharding wrapper has freed."""
    with pytest.raises(AssertionError, match="memory"):
        _calls_without_memory()[what]()


def test_refuses_fake_tensors():
    """The functions (unlike torch.ops) run kernels whatever mode is on: fake tensors, which say that they are on
    the GPU, are refused before anything is allocated or launched."""
    from torch._subclasses import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(5, 512, dtype=BF16, device="cuda")[1:]
        a = torch.empty(5, 64, dtype=I8, device="cuda")[1:]
        s = torch.empty(5, device="cuda")[1:]
        for call in (lambda: fv.fused_silu_mul_quant(x), lambda: fv.fused_add_rms_norm_quant(x, x, x[0], EPS),
                     lambda: fv.int8_scaled_mm(a, a, s, s)):
            with pytest.raises((AssertionError, RuntimeError), match="memory"):
                call()
