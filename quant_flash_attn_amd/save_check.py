"""Checks the assembly of kernels that have no vector register to spare, as the compiler wrote it: no register is saved while lanes may be off.

Where a branch that some lanes take joins again, the compiler has saved registers that all lanes need (a thread's own index among
them) before it turned the other lanes back on; these then read back what the place of the save held before, and stored out of bounds.
So the build looks at every save -- of a vector register to an accumulation register, of either to scratch -- and wants it where all lanes are
on, on every path, or of a value made under the same mask (the other lanes have none that could be lost).

All lanes are on at a kernel's start (workgroups are whole waves) and wherever exec is set from a scalar register that was written from
exec while they all were; such registers are followed through copies and through the lanes of vector registers that hold spilled
scalars.  Whatever else happens to exec counts as turning lanes off.

Kernels that wait for loads by their number (COUNTING) load keys into LDS and count the loads behind those.  They may have no scratch at all, since what the
compiler spills counts too; on every path from the last load into LDS to such a wait there are at least as many vector memory requests as the wait leaves on
their way; and behind such a wait, where the keys are read, LDS is loaded again only after a wait for all of its reads.  (These waits are statements that no
access of memory is moved across.)

    python -m quant_flash_attn_amd.save_check FILE.s
"""
from __future__ import annotations

import re
import sys
from typing import Dict, FrozenSet, List, Optional, Tuple

from .acc_check import _kernels

_SGPR = re.compile(r"^s(?:(\d+)|\[(\d+):(\d+)\])$")
_SAVE = re.compile(r"v_accvgpr_write_b32 a\S+ v\d+$|scratch_store_\w+ \S+ [av]")

COUNTING = ("paged_list_few_kernel",)

# what is known at an instruction: whether all lanes are on, and the scalar halves ("s", n) or spilled ones ("v", n, lane) that hold the
# low (0) or high (1) half of a mask of all lanes
State = Tuple[bool, FrozenSet[Tuple]]


def _scalars(op: str) -> List[Tuple[str, int]]:
    if op == "vcc":
        return [("vcc", 0), ("vcc", 1)]
    if op in ("vcc_lo", "vcc_hi"):
        return [("vcc", int(op == "vcc_hi"))]
    m = _SGPR.match(op)
    if not m:
        return []
    if m.group(1) is not None:
        return [("s", int(m.group(1)))]
    return [("s", n) for n in range(int(m.group(2)), int(m.group(3)) + 1)]


def _step(i, state: State) -> State:
    on, held = state
    ops = [x.strip() for x in re.split(r",\s*(?![^\[]*\])", i.text.partition(" ")[2]) if x.strip()]
    if not ops:
        return state
    whole = lambda op: len(_scalars(op)) == 2 and all((r, h) in held for h, r in enumerate(_scalars(op)))   # noqa: E731
    without = lambda regs: frozenset(x for x in held if x[0] not in regs)                               # noqa: E731
    with_pair = lambda op: without(_scalars(op)) | {(r, h) for h, r in enumerate(_scalars(op))}            # noqa: E731

    if i.op.endswith("_saveexec_b64"):
        after = i.op == "s_or_saveexec_b64" and (ops[1] == "-1" or whole(ops[1]) or on)
        return after, (with_pair(ops[0]) if on else without(_scalars(ops[0])))
    if ops[0] in ("exec", "exec_lo", "exec_hi"):
        if i.op == "s_mov_b64":
            return ops[1] == "-1" or whole(ops[1]), held
        if i.op == "s_or_b64":
            return on or any(whole(x) or x == "-1" for x in ops[1:]), held
        return False, held
    if i.op.startswith("v_cmpx"):
        return False, held
    if i.op == "v_writelane_b32":
        to = ("v", ops[0], ops[2])
        rest = without([to])
        src = _scalars(ops[1])
        return on, rest | {(to, h) for h in (0, 1) if src and (src[0], h) in held}
    if i.op == "v_readlane_b32":
        to, src = _scalars(ops[0]), ("v", ops[1], ops[2])
        return on, without(to) | {(to[0], h) for h in (0, 1) if (src, h) in held}
    if i.op == "s_mov_b64" and ops[1] == "exec":
        return on, (with_pair(ops[0]) if on else without(_scalars(ops[0])))
    if i.op in ("s_mov_b64", "s_mov_b32"):
        to, src = _scalars(ops[0]), _scalars(ops[1])
        new = {(t, h) for t, s in zip(to, src) for h in (0, 1) if (s, h) in held}
        return on, without(to) | new
    if i.op.startswith("s_") and not i.op.startswith(("s_cbranch", "s_branch", "s_cmp", "s_waitcnt", "s_nop", "s_bitcmp")):
        return on, without(_scalars(ops[0]))
    if i.op.startswith("v_"):   # results of comparisons and carries, and of lanes; a vector register written whole holds no spilled scalars
        gone = [r for op in ops[:2] for r in _scalars(op)] + ([("vcc", 0), ("vcc", 1)] if i.op.startswith("v_cmp") and i.op.endswith("_e32") else [])
        written = {f"v{n}" for kind, n in i.writes if kind == "v"}
        return on, frozenset(x for x in without(gone) if not (x[0][0] == "v" and x[0][1] in written))
    return state


def _saved(i) -> Optional[FrozenSet[Tuple[str, int]]]:
    m = _SAVE.match(i.text)
    if i.inline or not m:
        return None
    return i.reads or None


def _into_lds(i) -> bool:
    return i.op.startswith("buffer_load") and "lds" in i.text.split()


def _left(i, counter: str) -> int:
    """How many requests a wait in inline assembly leaves on their way; -1: it is none of that counter's."""
    m = re.search(counter + r"\((\d+)\)", i.text) if i.inline and i.op == "s_waitcnt" else None
    return int(m.group(1)) if m else -1


def _counts(ins, labels) -> List[Tuple[int, str]]:
    """What breaks a COUNTING kernel's rules: the index of an instruction, and what is wrong with it."""
    before: Dict[int, List[int]] = {}
    for k, i in enumerate(ins):
        if k + 1 < len(ins) and i.op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before.setdefault(k + 1, []).append(k)
        if i.target in labels:
            before.setdefault(labels[i.target], []).append(k)
    bad: List[Tuple[int, str]] = []
    for k, i in enumerate(ins):
        want = _left(i, "vmcnt")
        if want > 0:   # back to the loads into LDS
            todo, seen = [(k, 0)], set()
            while todo:
                p, n = todo.pop()
                if (p, n) in seen:
                    continue
                seen.add((p, n))
                n += not _into_lds(ins[p]) and bool(re.match(r"(global|buffer|flat|scratch)_(load|store|atomic)", ins[p].op))
                if n >= want:
                    continue
                if _into_lds(ins[p]) or p == 0:
                    bad.append((k, f"{n} requests behind the loads into LDS"))
                    break
                todo += [(q, n) for q in before.get(p, [])]
        if _into_lds(i):   # back to the wait for what has been read there (or the start), not to the one in front of those reads
            todo, seen = list(before.get(k, [])), set()
            while todo:
                p = todo.pop()
                if p in seen or _left(ins[p], "lgkmcnt") == 0:
                    continue
                seen.add(p)
                if _left(ins[p], "vmcnt") > 0:
                    bad.append((k, "a load into LDS that may still be read"))
                    break
                todo += before.get(p, [])
    return bad


def check(path: str) -> List[str]:
    """What is wrong, one line each; empty: nothing."""
    bad: List[str] = []
    for name, ins, labels, scratch in _kernels(path):
        if scratch and any(k in name for k in COUNTING):
            bad.append(f"{path}: {name}: counts its loads, and has {scratch} bytes of scratch")
        if any(k in name for k in COUNTING):
            bad += [f"{path}:{ins[k].line}: {name}: {what}: {ins[k].text}" for k, what in _counts(ins, labels)]
        if not any(_saved(i) for i in ins):
            continue
        after: Dict[int, List[int]] = {}
        for k, i in enumerate(ins):
            if k + 1 < len(ins) and i.op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                after.setdefault(k, []).append(k + 1)
            if i.target in labels:
                after.setdefault(k, []).append(labels[i.target])
        # vector registers written since lanes were last all on, on every path, beside the state of exec
        at: Dict[int, Tuple[State, FrozenSet]] = {0: ((True, frozenset()), frozenset())}
        todo = [0]
        while todo:
            k = todo.pop()
            state, made = at[k]
            new = _step(ins[k], state)
            made = frozenset() if new[0] else made | ins[k].writes if not state[0] else frozenset()
            for n in after.get(k, []):
                if n not in at:
                    at[n] = (new, made)
                else:
                    (on, held), was = at[n]
                    both = ((on and new[0], held & new[1]), was & made)
                    if both == at[n]:
                        continue
                    at[n] = both
                todo.append(n)
        for k, i in enumerate(ins):
            what = _saved(i)
            if what and k in at and not at[k][0][0] and not what <= at[k][1]:
                bad.append(f"{path}:{i.line}: {name}: a register is saved while lanes may be off: {i.text}")
    return bad


if __name__ == "__main__":
    found = [b for path in sys.argv[1:] for b in check(path)]
    print("\n".join(found) or "nothing found")
    sys.exit(1 if found else 0)
