"""build_block_tables: block tables, positions and slots from request lengths,
against a loop over requests and tokens; its refusals."""
import pytest
import torch

import flaggems_vllm as fv
from flaggems_vllm import _native

DEV = torch.device("cuda:0")
NAMES = ("query_start_loc", "seq_lens", "positions", "slot_mapping", "num_free")


def reference(ctx, query, table, free, num_free, page, most, pad=-1):
    """The definition, request by request and token by token (lists and a numpy-like table of lists)."""
    table = [row[:] for row in table]
    width = len(table[0]) if table else 0
    left = stack = min(max(num_free, 0), len(free))
    start, lens, positions, slots = [0], [], [0] * most, [pad] * most
    for b, (c, q) in enumerate(zip(ctx, query)):
        c, q = max(c, 0), min(max(q, 0), most - start[-1])
        for column in range(min(-(-c // page), width), min(-(-(c + q) // page), width)):
            left -= 1
            table[b][column] = free[left] if left >= 0 else -1
        for i in range(q):
            p = c + i
            positions[start[-1] + i] = p
            if p // page < width and table[b][p // page] >= 0:
                slots[start[-1] + i] = table[b][p // page] * page + p % page
        start.append(start[-1] + q)
        lens.append(c + q)
    assert stack >= left
    return start, lens, positions, slots, [left], table


def call(ctx, query, table, free, num_free, page, most, pad=-1, run=fv.build_block_tables):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    bt = table.to(DEV) if isinstance(table, torch.Tensor) else i32(table)
    out = run(i32(ctx), i32(query), bt, i32(free), i32([num_free]), page, most, pad)
    torch.cuda.synchronize()
    return [t.tolist() for t in out] + [bt.tolist()]


def random_case(seed, reqs, width, page, context, query, shortage=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda hi, n: torch.randint(0, hi + 1, (n,), generator=g).tolist()
    ctx, q = r(context, reqs), r(query, reqs)
    for i in range(0, reqs, 7):
        q[i] = 0
    for i in range(3, reqs, 11):
        ctx[i] = ctx[i] // page * page  # a context that fills its last block
    held = [min(-(-c // page), width) for c in ctx]
    ids = torch.randperm(sum(held) + reqs * (query // page + 2) + 3, generator=g).tolist()
    table = [[-9] * width for _ in range(reqs)]
    for b, n in enumerate(held):
        table[b][:n] = [ids.pop() for _ in range(n)]
    wanted = sum(min(-(-(c + n) // page), width) - h for c, n, h in zip(ctx, q, held))
    return ctx, q, table, ids, max(wanted - shortage, 0) if shortage else len(ids), page, sum(q)


CASES = [(1, 4, 16, 40, 3), (1, 1, 16, 0, 1), (2, 9, 16, 100, 30), (200, 40, 16, 500, 1), (255, 12, 16, 150, 2),
         (257, 12, 48, 400, 9), (37, 40, 7, 200, 70), (1023, 5, 16, 60, 1), (1025, 5, 16, 60, 3), (2100, 4, 1, 3, 1),
         (5, 300, 16, 3000, 1500), (64, 3, 1024, 2000, 900)]


@pytest.mark.gpu
@pytest.mark.parametrize("reqs,width,page,context,query", CASES)
@pytest.mark.parametrize("more,shortage", [(0, 0), (77, 0), (300, 2), (5, 10 ** 6)])
def test_gpu_tables(reqs, width, page, context, query, more, shortage):
    print(f"\n[case] tables {reqs} {width} {page} {context} {query} {more} {shortage}", flush=True)
    case = random_case(reqs + page, reqs, width, page, context, query, shortage)
    case = (*case[:6], case[6] + more)
    got, want = call(*case), reference(*case)
    for name, x, y in zip((*NAMES, "block_table"), got, want):
        assert x == list(y), name


@pytest.mark.gpu
def test_gpu_tokens_past_the_buffers_are_dropped():
    """Query lengths are cut where the step's rows end, and no block is taken for what is dropped."""
    case = random_case(5, 40, 20, 16, 100, 60)
    total = case[6]
    for most in (0, 1, total // 3, total - 1):
        args = (*case[:6], most, -7)
        for name, x, y in zip((*NAMES, "block_table"), call(*args), reference(*args)):
            assert x == list(y), (most, name)


@pytest.mark.gpu
def test_gpu_negative_lengths_and_a_count_past_the_stack():
    args = ([-5, 3, -1], [4, -2, 2], [[-1, -1], [8, -1], [-1, -1]], [1, 2, 3, 4], 100, 16, 9)
    for name, x, y in zip((*NAMES, "block_table"), call(*args), reference(*args)):
        assert x == list(y), name
    args = ([0, 3], [4, 20], [[-1, -1], [8, -1]], [1, 2, 3, 4], -3, 16, 30)
    assert call(*args)[4] == [-2]
    for name, x, y in zip((*NAMES, "block_table"), call(*args), reference(*args)):
        assert x == list(y), name


@pytest.mark.gpu
def test_gpu_nothing_to_do():
    """No request, no token, no table, no free block."""
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    start, lens, pos, slots, left = fv.build_block_tables(i32(0), i32(0), i32(0, 4), i32(3), 3 * one, 16, 5)
    assert start.tolist() == [0] and lens.tolist() == [] and left.tolist() == [3]
    assert pos.tolist() == [0] * 5 and slots.tolist() == [-1] * 5
    start, lens, pos, slots, left = fv.build_block_tables(i32(2), one.repeat(2), i32(2, 0), i32(0), one, 16, 0)
    assert start.tolist() == [0, 0, 0] and pos.numel() == 0 and left.tolist() == [0]
    start, lens, pos, slots, left = fv.build_block_tables(i32(2), one.repeat(2), i32(2, 0), i32(0), one, 16, 2)
    assert start.tolist() == [0, 1, 2] and slots.tolist() == [-1, -1] and lens.tolist() == [1, 1]


@pytest.mark.gpu
def test_gpu_wide_rows_and_far_slots():
    """A table out of a wider buffer, whose other columns stay, and slots past 32 bits."""
    case = random_case(9, 50, 12, 128, 900, 200)
    buf = torch.full((50, 31), -5, dtype=torch.int32)
    far = [2 ** 31 - 1 - i for i in range(len(case[3]))]
    buf[:, 4:16] = torch.tensor(case[2], dtype=torch.int32)
    dev = buf.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    out = fv.build_block_tables(i32(case[0]), i32(case[1]), dev[:, 4:16], i32(far), i32([case[4]]), 128, case[6])
    want = reference(*case[:3], far, *case[4:])
    for x, y in zip(out, want):
        assert x.tolist() == list(y)
    assert max(out[3].tolist()) > 2 ** 32
    buf[:, 4:16] = torch.tensor(want[5], dtype=torch.int32)
    assert torch.equal(dev.cpu(), buf)


@pytest.mark.gpu
def test_gpu_steps_in_a_graph():
    """A captured step, replayed while lengths and stack move on, is the eager one each time."""
    page, reqs, width, most = 16, 70, 30, 200
    g = torch.Generator().manual_seed(3)
    ctx = torch.randint(0, 200, (reqs,), generator=g, dtype=torch.int32).to(DEV)
    query = torch.ones(reqs, dtype=torch.int32, device=DEV)
    ids = torch.randperm(4100, generator=g, dtype=torch.int32).to(DEV)
    free = torch.tensor([2000], dtype=torch.int32, device=DEV)
    table = ids[2000:2000 + reqs * width].reshape(reqs, width).clone()
    run = lambda t: fv.build_block_tables(ctx, query, t, ids, free, page, most)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(table.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    captured = table.clone()
    with torch.cuda.graph(graph):
        out = run(captured)
    for step in range(40):
        query.copy_(torch.randint(0, 4, (reqs,), generator=g, dtype=torch.int32))
        graph.replay()
        want = run(table)
        torch.cuda.synchronize()
        assert torch.equal(captured, table), step
        for x, y in zip(out, want):
            assert torch.equal(x, y), step
        ctx.copy_(want[1])
        free.copy_(want[4])
    assert int(free) < 2000


@pytest.mark.gpu
def test_gpu_feeds_slot_mapping():
    """The slots are those that compute_slot_mapping_parallel makes of the same table and positions."""
    case = random_case(21, 60, 20, 16, 200, 50)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = i32(case[2])
    start, _, pos, slots, _ = fv.build_block_tables(i32(case[0]), i32(case[1]), table, i32(case[3]), i32([case[4]]),
                                                    16, case[6] + 9)
    again = torch.empty_like(slots)
    fv.compute_slot_mapping_parallel(case[6], case[6] + 9, start, 60, pos, table, again, 16)
    assert torch.equal(slots, again)


def cpu_args(**kw):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    a = dict(context_lens=i32(3), query_lens=i32(3), block_table=i32(3, 4), free_blocks=i32(5), num_free=i32(1),
             block_size=16, max_num_tokens=8)
    return {**a, **kw}


@pytest.mark.parametrize("kw", [
    dict(),  # CPU tensors
    dict(context_lens=torch.zeros(3)), dict(context_lens=torch.zeros(3, 1, dtype=torch.int32)),
    dict(query_lens=torch.zeros(2, dtype=torch.int32)), dict(query_lens=torch.zeros(3, dtype=torch.int64)),
    dict(query_lens=torch.zeros(6, dtype=torch.int32)[::2]),
    dict(block_table=torch.zeros(2, 4, dtype=torch.int32)), dict(block_table=torch.zeros(3, 4)),
    dict(block_table=torch.zeros(4, 3, dtype=torch.int32).t()),
    dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)),
    dict(free_blocks=torch.zeros(10, dtype=torch.int32)[::2]), dict(free_blocks=torch.zeros(5, dtype=torch.int64)),
    dict(num_free=torch.zeros(2, dtype=torch.int32)), dict(num_free=torch.zeros(1)),
    dict(block_size=0), dict(max_num_tokens=-1),
])
def test_refusals(kw):
    with pytest.raises(AssertionError):
        fv.build_block_tables(**cpu_args(**kw))


def test_refuses_a_table_over_its_inputs():
    buf = torch.zeros(20, dtype=torch.int32)
    for name in ("context_lens", "query_lens", "free_blocks"):
        with pytest.raises(AssertionError, match="overlap"):
            fv.build_block_tables(**cpu_args(block_table=buf[:12].view(3, 4), **{name: buf[10:13]}))


@pytest.mark.parametrize("kw,code", [
    (dict(reqs=-1), -2), (dict(most=-1), -2), (dict(width=-1), -2), (dict(size=-1), -2), (dict(page=0), -2),
    (dict(reqs=1 << 30), -5), (dict(most=1 << 30), -5), (dict(width=1 << 31), -5), (dict(page=1 << 31), -2),
    (dict(ctx=None), -1), (dict(table=None), -1), (dict(free=None), -1), (dict(slots=None), -1), (dict(nfree=None), -1),
    (dict(stride=3), -4), (dict(slots=20), -3),
])
def test_c_abi_refusals(kw, code):
    a = dict(ctx=16, q=16, reqs=4, table=16, stride=4, width=4, free=16, size=5, nfree=16, page=16, most=8, qsl=16,
             lens=16, pos=16, slots=16, out=16)
    a.update(kw)
    rc = _native.lib().fgv_build_block_tables(a["ctx"], a["q"], a["reqs"], a["table"], a["stride"], a["width"], a["free"],
                                              a["size"], a["nfree"], a["page"], a["most"], -1, a["qsl"], a["lens"],
                                              a["pos"], a["slots"], a["out"], None)
    assert rc == code and _native.lib().fgv_last_error()
