"""Static check of loads into LDS in the gfx950 assembly.

A load straight into LDS (``buffer_load_* ... lds``, ``global_load_lds_*``)
takes its place in LDS from m0, and the hardware does not wait for two of the
registers it reads:

  * between a scalar write of m0 and the load there has to be one wait state;
  * between a vector instruction that writes a scalar register (a
    ``v_readfirstlane_b32``, a compare) and a memory instruction that reads it,
    five.

The compiler inserts them for instructions of its own and not for inline
assembly.  A load that comes too early reads the register's value from before, so that
its bytes may land in another place of LDS or come from another buffer.

An instruction is one wait state and ``s_nop N`` is N + 1.  The check follows
every path through a function's blocks and takes the shortest.  build.py runs
it on the source whose loads are inline assembly; run it directly (optionally
with a source path) to print the report.
"""
from __future__ import annotations

import os
import re
import sys
from typing import Dict, List, Tuple

try:
    from . import check_lgkm
except ImportError:  # loaded by path, as build.py does
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    import check_lgkm

M0_STATES, SGPR_STATES = 1, 5
_SREG = re.compile(r"\bs(\d+)\b|\bs\[(\d+):(\d+)\]")
# vector instructions whose second operand is a scalar destination
_CARRY = re.compile(r"^v_(add|sub|subrev|addc|subb|subbrev)_co_|^v_div_scale_|^v_mad_[ui]64_")

State = Dict[str, int]  # register -> wait states since the write that counts, where fewer than needed


def _sregs(text: str) -> List[str]:
    out: List[str] = []
    for m in _SREG.finditer(text):
        lo = int(m.group(1) or m.group(2))
        out += [f"s{r}" for r in range(lo, int(m.group(1) or m.group(3)) + 1)]
    return out


def _is_lds_load(op: str, rest: str) -> bool:
    return op.startswith("global_load_lds") or op.startswith("buffer_load") and rest.split()[-1:] == ["lds"]


def _step(state: State, op: str, rest: str, where: str, problems: List[str]) -> State:
    if _is_lds_load(op, rest):
        if "m0" in state:
            problems.append(f"{where}: {op} follows the write of m0 without a wait state")
        for r in _sregs(rest):
            if r in state:
                problems.append(f"{where}: {op} reads {r} {state[r]} wait states after a vector instruction wrote it")
    passed = int(rest, 0) + 1 if op == "s_nop" else 1
    out = {r: n + passed for r, n in state.items()
           if n + passed < (M0_STATES if r == "m0" else SGPR_STATES)}
    operands = [p.strip() for p in rest.split(",")]
    if op.startswith("s_"):
        if operands[0] == "m0":
            out["m0"] = 0
        elif not op.startswith(("s_cmp", "s_bitcmp", "s_nop", "s_waitcnt", "s_cbranch", "s_branch")):
            for r in _sregs(operands[0]):  # a scalar write needs no wait
                out.pop(r, None)
    elif op.startswith("v_"):
        for o in operands[:2] if _CARRY.match(op) else operands[:1]:
            for r in _sregs(o):
                out[r] = 0
    return out


def check_function(name: str, lines: List[Tuple[int, str]]) -> Tuple[int, List[str]]:
    """(loads into LDS, problems)."""
    blocks: List[Tuple[str, List[Tuple[int, str, str]]]] = [("<entry>", [])]
    for i, ln in lines:
        # labels of inline assembly are numbers: a branch to one stays within its block's instructions
        label = re.match(r"^(\.LBB[\w.]+):", ln)
        if label:
            blocks.append((label.group(1), []))
            continue
        s = ln.split(";", 1)[0].strip()
        if not s or s.startswith(".") or re.match(r"^\d+:\s*$", s):
            continue
        s = re.sub(r"^\d+:\s*", "", s)
        op, rest = (s.split(None, 1) + [""])[:2]
        blocks[-1][1].append((i, op, rest))
        if op in ("s_branch", "s_endpgm", "s_setpc_b64") and not re.match(r"^\d+[fb]$", rest) \
                or op.startswith("s_cbranch") and rest.startswith(".LBB"):
            blocks.append((f"<after line {i}>", []))
    index = {label: k for k, (label, _) in enumerate(blocks)}
    loads = sum(_is_lds_load(op, rest) for _, ins in blocks for _, op, rest in ins)
    states: Dict[int, State] = {0: {}}
    work, problems = [0], []
    while work:
        k = work.pop()
        st = states[k]
        targets = [k + 1] if k + 1 < len(blocks) else []
        for line, op, rest in blocks[k][1]:
            st = _step(st, op, rest, f"{name}: line {line}", problems)
            if op == "s_branch" and rest in index or op in ("s_endpgm", "s_setpc_b64"):
                targets = []
            if (op == "s_branch" or op.startswith("s_cbranch")) and rest in index:
                targets.append(index[rest])
        for t in targets:
            old = states.get(t)
            new = dict(st) if old is None else {r: min(old.get(r, 99), st.get(r, 99)) for r in {*old, *st}}
            if new != old:
                states[t] = new
                work.append(t)
    return loads, sorted(set(problems))


def check_asm(asm: str) -> Tuple[int, List[str]]:
    """(loads into LDS, problems) of all functions of `asm`."""
    loads, problems = 0, []
    for name, lines in check_lgkm._functions(asm):
        n, p = check_function(name, lines)
        loads += n
        problems += p
    return loads, problems


def check_source(src: str, hipcc: str, flags: List[str]) -> Tuple[int, List[str]]:
    return check_asm(check_lgkm.compile_asm(src, hipcc, flags))


def main() -> int:
    here = os.path.dirname(os.path.abspath(__file__))
    sys.path.insert(0, os.path.dirname(os.path.dirname(here)))
    from qtpytorch_amd.csrc import build as b

    src = sys.argv[1] if len(sys.argv) > 1 else os.path.join(here, "mxk_mxfp4_gemm.hip")
    n, problems = check_source(src, b.hipcc(), b.HIPCC_FLAGS)
    for p in problems:
        print(p)
    print(f"{os.path.basename(src)}: {n} loads into LDS checked, {len(problems)} problems")
    return 1 if problems else 0


if __name__ == "__main__":
    sys.exit(main())
