"""What shows only in the gfx950 assembly that hipcc makes of int8_scaled_mm.hip
(compiled here; no GPU needed).  The tile kernels' MFMAs, LDS DMAs and
v_readfirstlanes are inline assembly, inside which the compiler keeps no wait
states and of whose LDS DMAs it knows nothing: that the code around them leaves
the distances and waits they need is checked in the result."""
import os
import re
import subprocess

import pytest

from flaggems_vllm import _native


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: instructions and labels} of the tile kernels, and the whole text."""
    out = tmp_path_factory.mktemp("asm") / "int8.s"
    flags = [f for f in _native.HIPCC_FLAGS if f not in ("-fPIC", "-shared")]
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *flags, "-S", "--cuda-device-only",
                    f"-I{_native._INCLUDE}", f"-I{_native._CSRC}", os.path.join(_native._CSRC, "int8_scaled_mm.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    text, found = open(out).read(), {}
    for m in re.finditer(r"^(_ZN\w*int8_mm_tile_kernel\w*):[^\n]*\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        lines = (line.split(";")[0].strip() for line in m.group(2).split("\n"))
        found[m.group(1)] = [x for x in lines if x and not x.startswith((".p2align", ".loc"))]
    assert len(found) >= 10
    return found


def registers(operand):
    """The registers of v[3:6], v7, a[0:3], s4 and the like."""
    m = re.match(r"([vas])\[(\d+):(\d+)\]$", operand)
    if m:
        return {f"{m.group(1)}{i}" for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    return {operand} if re.match(r"[vas]\d+$", operand) else set()


def operands(line):
    return [x.strip() for x in line.split(None, 1)[1].split(",")] if " " in line or "\t" in line else []


def written(line):
    ops = operands(line)
    return registers(ops[0]) if ops and not line.startswith(("s_wait", "s_barrier", "global_store", "ds_write")) else set()


def settled(code):
    """Where the wait behind the K loop stands."""
    return next(i for i in range(len(code)) if code[i] == "s_nop 15" and code[i + 1] == "s_nop 7")


def loop(code):
    """The K loop: from the label before the first MFMA to the last."""
    mfmas = [i for i, x in enumerate(code) if x.startswith("v_mfma")]
    return code[max(i for i in range(mfmas[0]) if code[i].endswith(":")):mfmas[-1] + 1]


def test_k_loop_moves_and_spills_nothing(kernels):
    for name, code in kernels.items():
        part = loop(code)
        assert sum(x.startswith("v_mfma") for x in part) >= 8, name  # two slices of 2 x 2 at least
        assert not [x for x in part if x.startswith(("scratch_", "v_accvgpr", "v_readlane", "v_writelane"))], name


def test_no_operand_comes_straight_from_the_valu(kernels):
    """An MFMA's sources are written by LDS reads alone, or by VALU instructions at least four before it; an
    accumulator written by the VALU (its zero) likewise."""
    for name, code in kernels.items():
        for i, line in enumerate(code):
            if not line.startswith("v_mfma"):
                continue
            used = set().union(*(registers(x) for x in operands(line)[1:4]))
            for back in code[max(0, i - 4):i]:
                if back.startswith("v_") and not back.startswith("v_mfma"):
                    assert not (written(back) & used), (name, back, line)


def test_accumulators_settle_before_they_are_read(kernels):
    """Behind the last MFMA, s_nop 15 and s_nop 7 stand before anything reads an accumulator."""
    for name, code in kernels.items():
        mfmas = [i for i, x in enumerate(code) if x.startswith("v_mfma")]
        sums = set().union(*(registers(operands(code[i])[0]) for i in mfmas))
        reads = [i for i, x in enumerate(code) if i > mfmas[0] and not x.startswith("v_mfma") and
                 any(registers(op) & sums for op in operands(x)[0 if x.startswith("global_store") else 1:])]
        assert mfmas[-1] < settled(code), name
        assert reads and min(reads) > settled(code) + 1, (name, code[min(reads)])


def test_scalars_from_the_valu_keep_their_distance(kernels):
    """A v_readfirstlane does not follow the VALU write of its source, and five wait states lie between a VALU
    write of a scalar register and the LDS DMA that takes its address from it."""
    for name, code in kernels.items():
        for i, line in enumerate(code):
            if line.startswith("v_readfirstlane"):
                source = registers(operands(line)[1])
                back = code[i - 1]
                assert not (back.startswith("v_") and written(back) & source), (name, back, line)
            if line.startswith("global_load_lds_dwordx4"):
                base, waits = registers(operands(line)[1]), 0
                for back in reversed(code[max(0, i - 8):i]):
                    if back.startswith("v_") and written(back) & base:
                        assert waits >= 5, (name, code[i - 8:i + 1])
                    m = re.match(r"s_nop (\d+)", back)
                    waits += int(m.group(1)) + 1 if m else 1


def test_every_block_is_waited_for(kernels):
    """Every barrier stands behind a wait for LDS (the operands read of the stage that is given back), and the K
    loop waits for vector memory (the block's DMAs)."""
    for name, code in kernels.items():
        plain = [x for x in code if not x.endswith(":")]
        for i, x in enumerate(plain):
            if x.startswith("s_barrier"):
                assert re.match(r"s_waitcnt\b.*lgkmcnt\(0\)", plain[i - 1]), (name, plain[i - 3:i + 1])
        first = next(i for i, x in enumerate(code) if x.startswith("v_mfma"))
        assert any(re.match(r"s_waitcnt\b.*vmcnt", x) for x in code[first:settled(code)]), name


# ------------------------------------------------------- the ring's hand-over ----

def shape(name):
    """WM, WN, TM, TN, NS of a tile kernel, and the DMAs that a wave sends for a K block."""
    wm, wn, tm, tn, ns = (int(x) for x in re.search(r"tile_kernelI" + r"Li(\d+)E" * 5, name).groups())
    return ns, (2 * tm * wm + 2 * tn * wn) // (wm * wn)


def waits_at_barriers(code):
    """{barrier: the counts of the last vector memory wait on every way to it}; None for a way with an LDS DMA behind
    its last wait, or without one.  Ways are followed forwards, with the flags that the compiler sets to 0 or -1 in
    scalar registers and tests through vcc (which choose between two waits), so that no way is taken that is none."""
    labels = {x[:-1]: i for i, x in enumerate(code) if x.endswith(":")}
    found, seen, todo = {}, set(), [(0, None, frozenset(), None)]
    while todo:
        i, wait, flags, vcc = todo.pop()
        while i < len(code) and (i, wait, flags, vcc) not in seen:
            seen.add((i, wait, flags, vcc))
            x = code[i]
            ops = operands(x)
            i += 1
            if x.endswith(":"):
                continue
            m = re.match(r"s_waitcnt\b.*vmcnt\((\d+)\)", x)
            if m:
                wait = int(m.group(1))
            elif x.startswith("global_load_lds"):
                wait = None
            elif x.startswith("s_barrier"):
                found.setdefault(i - 1, set()).add(wait)
            elif x.startswith("s_endpgm"):
                break
            elif x.startswith("s_branch"):
                i = labels[ops[0]]
            elif x.startswith("s_cbranch"):
                taken = None
                if x.startswith(("s_cbranch_vccnz", "s_cbranch_vccz")) and vcc is not None:
                    taken = vcc == x.startswith("s_cbranch_vccnz")
                if taken is None:
                    todo.append((labels[ops[0]], wait, flags, vcc))
                elif taken:
                    i = labels[ops[0]]
            elif ops:
                if ops[0] == "vcc" or x.startswith("v_cmp"):
                    vcc = None
                    if x.startswith("s_andn2_b64 vcc, exec, "):  # all lanes run: exec is not 0
                        vcc = {"0": True, "-1": False}.get(dict(flags).get(ops[2]))
                flags = frozenset(f for f in flags if not registers(f[0]) & registers(ops[0]))
                if x.startswith("s_mov_b64 s[") and ops[1] in ("0", "-1"):
                    flags |= {(ops[0], ops[1])}
    return found


def check_hand_over(name, code):
    """The first barrier lets blocks 1 to NS - 1 be under way, the loop's blocks kb + 2 to kb + NS - 1; where no more
    are sent both wait for all.  Counts above these would hand over a stage that has not landed."""
    ns, per = shape(name)
    sends = sum(x.startswith("global_load_lds_dwordx4") for x in code)
    assert sends == (ns + 1) * per, (name, sends)
    barriers = [i for i, x in enumerate(code) if x.startswith("s_barrier")]
    assert len(barriers) == 2, name
    first = next(i for i, x in enumerate(code) if x.startswith("global_load_lds_dwordx4"))
    behind = [sum(x.startswith("global_load_lds_dwordx4") for x in code[first:b]) for b in barriers]
    assert behind == [ns * per, ns * per], (name, behind)  # no DMA of the loop stands between the two
    waits = waits_at_barriers(code)
    for b, most in zip(barriers, ((ns - 1) * per, (ns - 2) * per)):
        counts = waits[b]
        assert None not in counts and 0 in counts and max(counts) <= most, (name, counts, most)


def test_every_stage_has_landed_at_its_barrier(kernels):
    for name, code in kernels.items():
        check_hand_over(name, code)


def test_a_late_or_short_wait_is_seen(kernels):
    """The check above, on code with one mistake in it: a wait gone, a count one block too large, a DMA between the
    wait and its barrier."""
    for name, code in kernels.items():
        per = shape(name)[1]
        sends = [i for i, x in enumerate(code) if x.startswith("global_load_lds_dwordx4")]
        bad = []
        for i in range(sends[0], settled(code)):
            m = re.match(r"s_waitcnt\b.*vmcnt\((\d+)\)", code[i])
            if m:
                bad.append(code[:i] + code[i + 1:])
                bad.append(code[:i] + [f"s_waitcnt vmcnt({int(m.group(1)) + per})"] + code[i + 1:])
            elif code[i].startswith("s_barrier"):
                bad.append(code[:i] + [code[sends[-1]]] + code[i:])
        assert len(bad) >= 8, name
        for wrong in bad:
            with pytest.raises(AssertionError):
                check_hand_over(name, wrong)
