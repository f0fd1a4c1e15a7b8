"""Build check for the inline-assembly direct global -> LDS loads
(lds_load16 / lds_load4 in csrc/common.hpp).

Each of those loads is one asm statement holding

    s_mov_b32 m0, <sgpr>
    s_nop 0
    buffer_load_dword[x4] <vgpr>, <rsrc>, <soffset sgpr> offen lds

which overwrites m0 (the LDS destination address) behind the compiler's
back. That is safe only while the compiler keeps nothing of its own in m0
in the same kernel, and while the wait states stand there that the hardware
does not provide by itself: the compiler's hazard pass does not look into
inline assembly. This script reads the device assembly of a translation
unit (hipcc --cuda-device-only -S) and fails the build when any function in
it breaks that. check(), who has m0:

  - an instruction outside an inline-asm block names m0 (the compiler set or
    read it for its own use);
  - an inline-asm block that names m0 is anything but a load with its m0 (it
    does not ask for the s_nop: check_waits does);
  - an instruction that uses m0 implicitly appears outside the asm blocks
    (s_sendmsg*, s_ttracedata, s_movrel* / v_movrel*, v_interp*, ds_gws*,
    ds_append / ds_consume / ds_ordered_count, the *_addtid LDS forms, and
    buffer / global loads to LDS).

check_waits(), the wait states of the direct loads:

  - fewer than one between the s_mov_b32 m0 and the load: on gfx9 a load to
    LDS may still see the m0 from before (the compiler puts an s_nop 0 or
    another instruction between the two of its own);
  - fewer than five between a vector instruction that writes an SGPR
    (v_readfirstlane, v_readlane, v_cmp, a carry) and a load that reads it,
    over every path that leads there.

Usage: python3 check_m0.py FILE.s [FILE.s ...]; exit status 1 with a report
on the first violations, 0 (and one summary line) otherwise.
"""
from __future__ import annotations

import re
import sys

M0 = re.compile(r"\bm0\b")
PAIR_MOV = re.compile(r"^s_mov_b32\s+m0,\s*s\d+$")
PAIR_LOAD = re.compile(r"^buffer_load_dword(x4)?\s+v\d+,\s*s\[\d+:\d+\],\s*(s\d+|\d+)\s+offen\s+lds$")
NOP = re.compile(r"^s_nop\s+(\d+)$")
SGPR_LOAD = re.compile(r"^buffer_load_dword(x4)?\s+v\d+,\s*s\[\d+:\d+\],\s*s\d+\s+offen\s+lds$")
IMPLICIT = re.compile(r"^(s_sendmsg|s_ttracedata|s_movrel|v_movrel|v_interp|ds_gws|ds_append|ds_consume|"
                      r"ds_ordered_count|ds_read_addtid|ds_write_addtid|ds_load_addtid|ds_store_addtid)"
                      r"|^(buffer|global)_load\S*\s.*\blds\b")
FUNC = re.compile(r"^([A-Za-z_.$][\w.$]*):")


def _instr(line: str) -> str:
    """The instruction text of an assembly line ('' for labels, directives,
    comments and blank lines)."""
    s = line.split(";", 1)[0].strip()
    if not s or s.startswith(".") or s.endswith(":"):
        return ""
    return s


def check(path: str) -> tuple[list[str], int, int]:
    """(violations, functions seen, m0 pairs seen) for one assembly file."""
    bad: list[str] = []
    func = "?"
    nfunc = pairs = 0
    in_asm = False
    block: list[tuple[int, str]] = []
    with open(path) as f:
        for no, raw in enumerate(f, 1):
            line = raw.rstrip("\n")
            m = FUNC.match(line)
            if m and not line.startswith(("\t", " ")) and not m.group(1).startswith(".L"):
                func = m.group(1)
                nfunc += 1
            if ";;#ASMSTART" in line:
                in_asm, block = True, []
                continue
            if ";;#ASMEND" in line:
                in_asm = False
                ins = [(n, s) for n, s in block if s]
                if any(M0.search(s) for _, s in ins):
                    ok = PAIR_MOV.match(ins[0][1]) and (
                        len(ins) == 2 and PAIR_LOAD.match(ins[1][1])
                        or len(ins) == 3 and NOP.match(ins[1][1]) and SGPR_LOAD.match(ins[2][1]))
                    if ok:
                        pairs += 1
                    else:
                        bad.append(f"{path}:{block[0][0] if block else no}: {func}: inline asm naming m0 is not "
                                   f"the s_mov_b32 m0 (+ s_nop) + buffer_load ... lds: {[s for _, s in ins]}")
                continue
            s = _instr(line)
            if in_asm:
                block.append((no, s))
                continue
            if not s:
                continue
            if M0.search(s):
                bad.append(f"{path}:{no}: {func}: compiler-generated use of m0: {s}")
            elif IMPLICIT.search(s):
                bad.append(f"{path}:{no}: {func}: instruction that uses m0 implicitly: {s}")
    return bad, nfunc, pairs


M0_WAITS, SGPR_WAITS = 1, 5  # wait states before a load to LDS / any vector-memory instruction on gfx9
CARRY = re.compile(r"^v_(add_co|addc_co|sub_co|subb_co|subrev_co|subbrev_co|div_scale|mad_u64_u32|mad_i64_i32)")


def _sgprs(operand: str) -> set[int]:
    m = re.match(r"^s\[(\d+):(\d+)\]$", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.match(r"^s(\d+)$", operand)
    return {int(m.group(1))} if m else set()


def _operands(s: str) -> list[str]:
    return [a for a in re.split(r"[ ,\t]+", s)[1:] if a]


def _functions(path: str):
    """(name, [(line number, instruction or 'label:')]) of each function."""
    name, ins = "?", []
    with open(path) as f:
        for no, line in enumerate(f, 1):
            m = FUNC.match(line)
            if m and not m.group(1).startswith(".L"):
                if ins:
                    yield name, ins
                name, ins = m.group(1), []
            elif m:
                ins.append((no, m.group(1) + ":"))
            elif s := _instr(line):
                ins.append((no, s))
    if ins:
        yield name, ins


def check_waits(path: str) -> list[str]:
    """Direct loads that follow a write of their m0 or SGPRs too closely."""
    bad: list[str] = []
    for func, ins in _functions(path):
        loads = [i for i, (_, s) in enumerate(ins) if IMPLICIT.search(s) and re.search(r"\blds\b", s)]
        if not loads:
            continue
        labels = {s[:-1]: i for i, (_, s) in enumerate(ins) if s.endswith(":")}
        before: list[list[int]] = [[] for _ in ins]
        for i, (_, s) in enumerate(ins):
            op = s.split()[0]
            if op in ("s_endpgm", "s_setpc_b64"):
                continue
            if op != "s_branch" and i + 1 < len(ins):
                before[i + 1].append(i)
            if op == "s_branch" or op.startswith("s_cbranch"):
                before[labels[_operands(s)[0]]].append(i)
        for at in loads:
            need = set().union(*(_sgprs(a) for a in _operands(ins[at][1])))
            # backwards over every path: (instruction, wait states behind it, what of m0 and the SGPRs is still the load's)
            todo = [(i, 0, frozenset(need), True) for i in before[at]]
            seen = set(todo)
            while todo:
                i, states, regs, m0 = todo.pop()
                no, s = ins[i]
                args = [] if s.endswith(":") else _operands(s)
                wrote = _sgprs(args[0]) if args else set()
                if s.startswith("v_") and len(args) > 1 and CARRY.match(s):
                    wrote |= _sgprs(args[1])
                if m0 and args and args[0] == "m0":
                    if states < M0_WAITS:
                        bad.append(f"{path}:{ins[at][0]}: {func}: {states} wait states between m0 and the load: "
                                   f"{s}; {ins[at][1]}")
                    m0 = False
                if wrote & regs:
                    if s.startswith("v_") and states < SGPR_WAITS:
                        bad.append(f"{path}:{ins[at][0]}: {func}: {states} wait states between a vector instruction's "
                                   f"SGPR and the load: {s}; {ins[at][1]}")
                    if s.startswith(("v_", "s_")) and not s.startswith(("s_cmp", "s_bitcmp")):
                        regs = regs - wrote
                nop = NOP.match(s)
                states += 0 if s.endswith(":") else int(nop.group(1)) + 1 if nop else 1
                if states >= SGPR_WAITS or not (regs or m0):
                    continue
                for j in before[i]:
                    nxt = (j, states, regs, m0)
                    if nxt not in seen:
                        seen.add(nxt)
                        todo.append(nxt)
    return bad


def main(argv: list[str]) -> int:
    if len(argv) < 2:
        print(__doc__.strip().splitlines()[-2], file=sys.stderr)
        return 2
    failed = False
    for path in argv[1:]:
        bad, nfunc, pairs = check(path)
        bad += check_waits(path)
        if bad:
            failed = True
            print(f"check_m0: {path}: {len(bad)} violation(s)", file=sys.stderr)
            for b in bad[:20]:
                print("  " + b, file=sys.stderr)
        else:
            print(f"check_m0: {path}: ok ({nfunc} functions, {pairs} LDS loads with their m0 and waits, no other m0 use)")
    return 1 if failed else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv))
