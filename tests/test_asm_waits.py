"""Loads into LDS that inline assembly makes keep the wait states that the hardware asks for.

The compiler puts them before loads that it makes itself; it sees none inside inline assembly.  Such a load needs one wait state
(an instruction, or s_nop) between a scalar write of M0, which holds its place in LDS, and itself, and five between a vector
instruction that writes its scalar base address (v_readfirstlane and its like) and itself.  Checked in the library as it was
built, over every way that leads to a load.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import PKG_DIR

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
LINE = re.compile(r"^\t(\S+)(?: (.*?))?\s*// ([0-9A-F]+): [0-9A-F ]+(?:<(\S+?)(?:\+0x([0-9a-f]+))?>)?\s*$")
HEAD = re.compile(r"^([0-9a-f]+) <(\S+)>:$")
BASE_WAITS, M0_WAITS = 5, 1


def instructions(listing):
    """[(mnemonic, operands, index of its branch target or None)] of a listing."""
    out, at, symbol, jumps = [], {}, {}, []
    for l in listing.splitlines():
        m = LINE.match(l)
        if m:
            at[int(m[3], 16)] = len(out)
            if m[1].startswith(("s_cbranch", "s_branch")):
                jumps.append((len(out), m[4], int(m[5] or "0", 16)))
            out.append([m[1], m[2] or "", None])
        else:
            h = HEAD.match(l)
            if h:
                symbol[h[2]] = int(h[1], 16)
    for i, name, off in jumps:
        out[i][2] = at[symbol[name] + off]
    return out


def states(op, args):
    return int(args.split()[0], 0) + 1 if op == "s_nop" else 1


def scalars(text):
    """Scalar registers that a text names."""
    regs = set()
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\bvcc(_lo|_hi)?\b", text):
        if m[0].startswith("vcc"):
            regs |= {"": {106, 107}, "_lo": {106}, "_hi": {107}}[m[4] or ""]
        else:
            regs |= set(range(int(m[1] or m[3]), int(m[2] or m[3]) + 1))
    return regs


def written_by_vector(op, args):
    """Scalar registers that a vector instruction writes."""
    if not op.startswith("v_"):
        return set()
    regs = set()
    for a in args.split(", ")[:2 if "_co_" in op or "div_scale" in op or "mad_u64" in op or "mad_i64" in op else 1]:
        regs |= scalars(a.strip())
    return regs


def faults(code):
    """Loads into LDS that come too soon: [(index, what)]."""
    sources = {}
    for i, (_, _, to) in enumerate(code):
        if to is not None:
            sources.setdefault(to, []).append(i)

    def before(i):                               # instructions after which instruction i may run
        if i and code[i - 1][0] not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            yield i - 1
        yield from sources.get(i, ())

    bad = []
    for i, (op, args, _) in enumerate(code):
        if not (op.startswith("global_load_lds") or (op.startswith("buffer_load") and re.search(r"\blds\b", args))):
            continue
        base = scalars(args)
        ways = [(p, 0) for p in before(i)]       # (instruction, wait states between it and the load)
        while ways:
            p, n = ways.pop()
            o, a, _ = code[p]
            if n < M0_WAITS and a.split(",")[0] == "m0" and o.startswith("s_"):
                bad.append((i, f"M0 by {o} {a}, {n} wait states before {op}"))
            if base & written_by_vector(o, a):
                bad.append((i, f"base by {o} {a}, {n} wait states before {op} {args}"))
            n += states(o, a)
            if n < BASE_WAITS:
                ways += [(q, n) for q in before(p)]
    return bad


def test_the_checker_sees_faults():
    head = "0000000000000000 <k>:\n"
    load = "global_load_lds_dwordx4 v1, s[4:5]"

    def line(at, text, to=None):
        return f"\t{text}    // {at:08X}: 00000000{'' if to is None else f' <k+{to:#x}>'}\n"

    def code(*texts):
        return instructions(head + "".join(line(4 * i, *t) if isinstance(t, tuple) else line(4 * i, t) for i, t in enumerate(texts)))

    assert len(faults(code("s_mov_b32 m0, s3", load))) == 1
    assert not faults(code("s_mov_b32 m0, s3", "s_nop 0", load))
    assert len(faults(code("v_readfirstlane_b32 s5, v2", "s_mov_b32 m0, s3", "s_nop 2", load))) == 1
    assert not faults(code("v_readfirstlane_b32 s5, v2", "s_mov_b32 m0, s3", "s_nop 3", load))
    assert not faults(code("v_readfirstlane_b32 s6, v2", "s_nop 0", load))
    assert len(faults(code("v_cmp_gt_f32_e64 s[4:5], v2, v3", "s_nop 1", load))) == 1
    assert len(faults(code("v_cmp_gt_f32_e32 vcc, v2, v3", "global_load_lds_dword v1, vcc offset:16"))) == 1
    # by way of a branch
    assert len(faults(code("v_readfirstlane_b32 s4, v2", ("s_cbranch_scc0 3", 16), "s_nop 7", "s_nop 7", load))) == 1
    assert not faults(code("v_readfirstlane_b32 s4, v2", ("s_branch 1", 12), load, "s_endpgm"))


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no disassembler for the library's own kernels")
def test_loads_into_lds_wait(rt4, tmp_path):
    for name in ("librt4k.so", "librt4probe.so"):
        shutil.copy(PKG_DIR / "rt4_amd" / "lib" / name, tmp_path / name)
        subprocess.run([str(OBJDUMP), "--offloading", str(tmp_path / name)], check=True, capture_output=True, cwd=tmp_path)
    seen = 0
    for obj in sorted(tmp_path.glob("*gfx950")):
        text = subprocess.run([str(OBJDUMP), "-d", "--mcpu=gfx950", str(obj)], check=True, capture_output=True, text=True).stdout
        if not re.search(r"\tglobal_load_lds|\tbuffer_load.*\blds\b", text):
            continue
        code = instructions(text)
        seen += sum(op.startswith("global_load_lds") for op, _, _ in code)
        bad = faults(code)
        assert not bad, (obj.name, len(bad), bad[:5])
    assert seen > 500
