"""Build-time checks on the compiled gfx950 ISA of the chunk kernels of linear attention (hipcc cross-compiles here, no GPU needed).

A chunk's rows are loaded into LDS by inline assembly that the compiler keeps no count of.  The wait at the front of the next chunk leaves the
stores of the last one outstanding, which is right only where those go out behind the loads: that is shown here for every path.

The result of a matrix instruction is there a number of instructions behind it, which the compiler has to see to; where a branch leads around a
block it has been found to count the block's instructions in.  That is looked for on every path as well."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from rnn_train_ring_attractor_amd.build import CSRC, HIPCC_FLAGS, INCLUDE

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
KINDS = ("f32", "bf16", "f16")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    folder = tmp_path_factory.mktemp("isa")

    def compiled(kind):
        out = folder / f"{kind}.s"
        cmd = [HIPCC, *(f for f in HIPCC_FLAGS if f not in ("-shared", "-fPIC")), "-S", "--cuda-device-only", f"-I{INCLUDE}", f"-I{CSRC}",
               os.path.join(CSRC, f"ring_linattn_{kind}.hip"), "-o", str(out)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        assert proc.returncode == 0, proc.stderr[-2000:]
        return kernels(out.read_text())

    with ThreadPoolExecutor(len(KINDS)) as pool:
        return dict(zip(KINDS, pool.map(compiled, KINDS)))


def kernels(text):
    """{name: (instructions as (opcode, operands), {label: where it stands})}"""
    out = {}
    for m in re.finditer(r"^(_Z\w*ring_linattn_kernel\w*):.*$", text, re.M):
        code, labels = [], {}
        for line in text[m.end():text.index(".Lfunc_end", m.end())].split("\n"):
            line = line.split(";")[0].strip()
            if line.startswith(".LBB") and line.endswith(":"):
                labels[line[:-1]] = len(code)
            elif line and line[0] != ".":
                opcode, _, rest = line.partition(" ")
                code.append((opcode, [x.strip() for x in re.split(r",\s*(?![^\[]*\])", rest)] if rest else []))
        out[m.group(1)] = code, labels
    return out


def behind(code, labels, i):
    """Where control can be behind instruction i."""
    opcode, operands = code[i]
    if opcode == "s_branch":
        return [labels[operands[0]]]
    if opcode.startswith("s_cbranch"):
        return [labels[operands[0]], i + 1]
    return [] if opcode in ("s_endpgm", "s_setpc_b64") else [i + 1]


def registers(operand):
    m = re.match(r"-?\|?([va])\[(\d+):(\d+)\]", operand) or re.match(r"-?\|?([va])(\d+)\b", operand)
    if not m:
        return frozenset()
    return frozenset((m.group(1), r) for r in range(int(m.group(2)), int(m.group(m.lastindex)) + 1))


def loads_behind_stores(code, labels):
    """Loads into LDS that a store separates from another of the same chunk, no barrier between."""
    bad = []
    for start, (opcode, _) in enumerate(code):
        if not opcode.startswith("global_load_lds"):
            continue
        todo, seen = [(j, False) for j in behind(code, labels, start)], set()
        while todo:
            at = todo.pop()
            if at in seen:
                continue
            seen.add(at)
            i, stored = at
            opcode = code[i][0]
            if opcode == "s_barrier":
                continue
            if opcode.startswith("global_load_lds") and stored:
                bad.append((start, i))
            todo += [(j, stored or opcode.startswith("global_store")) for j in behind(code, labels, i)]
    return bad


# Instructions between a matrix instruction and one that reads what it writes: passes of four clocks, and 2 (fp32 operands) or 4 more
WAITS = {"v_mfma_f32_16x16x4_f32": 8 + 2, "v_mfma_f32_16x16x32_bf16": 4 + 4}


def results_read_early(code, labels):
    bad = []
    for start, (opcode, operands) in enumerate(code):
        if not opcode.startswith("v_mfma"):
            continue
        wait = WAITS[opcode]
        todo, seen = [(start + 1, 0, registers(operands[0]))], {}
        while todo:
            i, states, live = todo.pop()
            if states >= wait or not live or seen.get((i, live), wait) <= states:
                continue
            seen[i, live] = states
            opcode, operands = code[i]
            if opcode == "s_nop":
                states += int(operands[0], 0)
            elif opcode.startswith("v_mfma"):
                # (the same registers taken on as the sum need no wait)
                if (registers(operands[1]) | registers(operands[2])) & live:
                    bad.append((start, i, states))
                live -= registers(operands[0])
            elif opcode.startswith(("v_", "ds_", "global_", "scratch_")):
                first = opcode.startswith(("v_", "ds_read", "global_load_dword", "scratch_load")) and not opcode.startswith("v_cmp")
                read = frozenset().union(*map(registers, operands[first:]))
                written = registers(operands[0]) if opcode.startswith("v_") and first else frozenset()
                if (read | written) & live:
                    bad.append((start, i, states))
                    live -= read | written
            todo += [(j, states + 1, live) for j in behind(code, labels, i)]
    return bad


@pytest.mark.parametrize("kind", KINDS)
def test_stores_that_a_wait_leaves_out_go_out_behind_the_loads(kind, assembly):
    waiting = 0
    for name, (code, labels) in assembly[kind].items():
        assert not loads_behind_stores(code, labels), name
        waiting += any(op == "s_waitcnt" and re.match(r"vmcnt\([12]\) lgkmcnt\(0\)", " ".join(args)) for op, args in code)
    assert waiting                                                       # (the wait that this is about)


@pytest.mark.parametrize("kind", KINDS)
def test_results_of_matrix_instructions_are_there_when_they_are_read(kind, assembly):
    for name, (code, labels) in assembly[kind].items():
        assert any(op.startswith("v_mfma") for op, _ in code)
        assert not results_read_early(code, labels), name


def test_the_checks_find_what_they_look_for():
    text = """_Z3ring_linattn_kernelv: ; planted
    global_load_lds_dwordx4 v0, s[0:1]
    {store}
    global_load_lds_dwordx4 v1, s[0:1]
    s_cbranch_scc1 .LBB0_2
    v_mfma_f32_16x16x4_f32 v[8:11], v2, v3, v[8:11]
    s_cbranch_vccnz .LBB0_1
    {nops}
.LBB0_1:
    {gap}
    v_mul_f32_e32 v11, v4, v11
.LBB0_2:
    s_endpgm
.Lfunc_end0:
"""
    found = lambda **k: [f(*kernels(text.format(**{**dict(store="", nops="s_nop 15", gap="s_nop 8"), **k}))["_Z3ring_linattn_kernelv"])
                         for f in (loads_behind_stores, results_read_early)]
    assert found() == [[], []]
    assert found(store="global_store_dword v9, v9, s[0:1]") == [[(0, 2)], []]
    assert found(gap="s_nop 7") == [[], [(3, 7, 9)]]                     # around the block: the branch and eight
    assert found(gap="s_nop 7", nops="s_nop 0") == [[], [(3, 7, 9)]]
    assert found(gap="s_nop 0")[1] == [(3, 7, 2)]
