"""Wait states before the copies into LDS, read off the built library's own
listing.  The kernels issue these copies as inline assembly, in which the
compiler inserts none of the wait states that it keeps around its own loads:

* a load into LDS must not directly follow the write of m0, where its
  destination stands (1 wait state);
* a memory instruction must not read a scalar register within 5 wait states of
  a vector instruction's write to it (the buffer descriptor, where the compiler
  holds a value of it in vector registers).

Every instruction is a wait state, s_nop n is n + 1.  Blocks that several
others lead to take the least of their counts.  No GPU."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pyramid-forcing_amd", "pyramidkv", "_lib",
                   "libpyramidkv_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MEMORY = ("buffer_", "global_", "flat_", "scratch_")
SALU_LAST = ("s_branch", "s_endpgm", "s_setpc")
M0, FAR = "m0", 5
# vector instructions with a scalar result in their second operand
SECOND = re.compile(r"v_(\w+_co_|mad_[iu]64_[iu]32|div_scale)")


def scalars(operand):
    """The scalar registers that an operand names."""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return [f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)]
    if operand == "vcc":
        return ["vcc_lo", "vcc_hi"]
    return [operand] if re.fullmatch(r"s\d+|vcc_lo|vcc_hi|m0", operand) else []


def kernels(listing):
    """name -> [(address, mnemonic, operands, address it may jump to)]"""
    out, name, start = {}, None, {}
    for line in listing.splitlines():
        m = re.match(r"([0-9a-f]+) <(.+)>:$", line)
        if m:
            name = m[2]
            start[name] = int(m[1], 16)
            out[name] = []
            continue
        m = re.match(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not m or name is None:
            continue
        to = re.search(r"<(.+?)(?:\+0x([0-9a-f]+))?>$", line) if m[1].startswith(("s_branch", "s_cbranch")) else None
        out[name].append((int(m[3], 16), m[1], [o.strip() for o in re.split(r",|\s+(?=offen|lds|nt|sc|off)", m[2])],
                          start[to[1]] + int(to[2] or "0", 16) if to else None))
    return out


def step(ins, state):
    """state (register -> wait states since its write, where below FAR) after an instruction."""
    _, op, args, _ = ins
    n = int(args[0]) + 1 if op == "s_nop" else 1
    state = {r: c + n for r, c in state.items() if c + n < FAR}
    if op.startswith("v_"):
        for r in [*scalars(args[0]), *(scalars(args[1]) if SECOND.match(op) and len(args) > 1 else [])]:
            state[r] = 0
    elif op.startswith("s_"):  # a scalar instruction's write is waited for, m0's before a copy into LDS is not
        for r in scalars(args[0]) if args else []:
            state.pop(r, None)
            if r == M0:
                state[M0] = 0
    return state


def faults(code):
    """Instructions that come too early."""
    at = {ins[0]: i for i, ins in enumerate(code)}
    entry, todo, bad = {0: {}}, [0], set()
    while todo:
        i = todo.pop()
        state = entry[i]
        while True:
            ins = code[i]
            _, op, args, to = ins
            if op.startswith(MEMORY):
                if "lds" in args and M0 in state and state[M0] < 1:
                    bad.add((i, "m0"))
                bad.update((i, r) for a in args for r in scalars(a) if r != M0 and r in state)
            state = step(ins, state)
            for j in ([at[to]] if to in at else []) + ([i + 1] if i + 1 < len(code) and not op.startswith(SALU_LAST) else []):
                if j == i + 1 and to is None and j not in entry:
                    continue
                old = entry.get(j)
                new = state if old is None else {r: min(old.get(r, FAR), state.get(r, FAR)) for r in {*old, *state}}
                if new != old:
                    entry[j] = new
                    todo.append(j)
            if to is not None or op.startswith(SALU_LAST) or i + 1 >= len(code) or i + 1 in entry:
                break
            i += 1
    return sorted(bad)


def listing(tmp_path):
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    for f in sorted(tmp_path.iterdir()):
        if "gfx950" in f.name:
            yield subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", f.name], cwd=tmp_path, check=True, stdout=subprocess.PIPE,
                                 text=True).stdout


def _code(*lines):
    return [(8 * i, l.split()[0], [o.strip(",") for o in l.split()[1:]], None) for i, l in enumerate(lines)]


def test_what_counts():
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    assert faults(_code("s_mov_b32 m0, s1", load)) == [(1, "m0")]
    assert not faults(_code("s_mov_b32 m0, s1", "s_nop 0", load))
    assert faults(_code("v_readfirstlane_b32 s6, v1", "s_mov_b32 m0, s1", "s_nop 2", load)) == [(3, "s6")]
    assert not faults(_code("v_readfirstlane_b32 s6, v1", "s_mov_b32 m0, s1", "s_nop 3", load))
    assert not faults(_code("v_readfirstlane_b32 s6, v1", "s_mov_b32 s6, s6", "s_nop 0", load))
    assert faults(_code("v_cmp_lt_i32 s[4:5], v1, v2", load)) == [(1, "s4"), (1, "s5")]
    loop = _code("s_nop 9", load, "v_readfirstlane_b32 s4, v0", "s_cbranch_scc0 x", "s_endpgm")
    loop[3] = (24, "s_cbranch_scc0", [], 8)
    assert faults(loop) == [(1, "s4")]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
@pytest.mark.parametrize("what", [M0, "descriptor"])
def test_copies_into_lds_wait(what, tmp_path):
    copies, bad = 0, []
    for text in listing(tmp_path):
        for name, code in kernels(text).items():
            copies += sum("lds" in args and op.startswith(MEMORY) for _, op, args, _ in code)
            bad += [f"{name} +{code[i][0] - code[0][0]:#x} {code[i][1]} {','.join(code[i][2])}: {r}" for i, r in faults(code)
                    if (r == M0) == (what == M0)]
    assert copies > 100 and not bad, f"{len(bad)} of {copies} copies:\n" + "\n".join(bad[:40])
