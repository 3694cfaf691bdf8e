"""A check of hand-written counted waits in a kernel's assembly listing (used by the build).

Copies from global memory into LDS are not known to the compiler as writes of what is
read from LDS behind them; the kernel waits for them itself, by `s_waitcnt vmcnt(n)` in
an asm statement.  Such a wait leaves the n youngest loads in flight, and so is one for
the copies only if n loads at least follow them.  How many loads there are is the
compiler's choice: it may join two, or drop one.  This counts them, on every path.
"""
from __future__ import annotations

import re
from collections import defaultdict

_LABEL = re.compile(r"^([.\w$]+):")
_VMCNT = re.compile(r"\bvmcnt\((\d+)\)")
_LOAD = re.compile(r"^(global|buffer|scratch)_load_")
# what ends a kernel's straight line or leaves it in a way that is not followed here
_JUMP = re.compile(r"^(s_branch|s_cbranch_\w+)\s+(\S+)$")
_END = "s_endpgm"
_UNKNOWN = re.compile(r"^(s_setpc|s_swappc|s_call|s_rfe|s_cbranch_g_fork|s_cbranch_i_fork|s_cbranch_join)")


def _blocks(lines):
    """The blocks of a kernel in order: [(label, [(instruction, written by hand)])].  A
    block ends behind each jump, so that only its last instruction is one."""
    blocks, asm = [("", [])], False
    for raw in lines:
        text = raw.strip()
        if text.startswith(";;#ASMSTART") or text.startswith(";;#ASMEND"):
            asm = text.startswith(";;#ASMSTART")
            continue
        text = text.split(";", 1)[0].strip()
        label = _LABEL.match(text)
        if label:
            blocks.append((label.group(1), []))
        elif text and not text.startswith("."):
            blocks[-1][1].append((text, asm))
            if _JUMP.match(text) or text == _END:
                blocks.append(("", []))
    return blocks


def _walk(block, loads, found=None):
    """The fewest loads behind the last copy that may be in flight (None: none is) at a
    block's end, from that at its start; found gets (n, loads) of each hand-written
    wait."""
    for text, asm in block:
        if _LOAD.match(text):
            if re.search(r"\blds\b", text) or "_load_lds_" in text:
                loads = 0
            elif loads is not None:
                loads += 1
        elif text.startswith("s_waitcnt"):
            n = _VMCNT.search(text)
            if n is None:
                continue
            n = int(n.group(1))
            if asm and found is not None:
                found.append((n, loads))
            if loads is not None and n <= loads:
                loads = None
    return loads


def _kernel_waits(name, lines):
    blocks = _blocks(lines)
    at = {label: i for i, (label, _) in enumerate(blocks) if label}
    after = defaultdict(list)
    for i, (_, block) in enumerate(blocks):
        for text, _ in block:
            if _UNKNOWN.match(text):
                raise RuntimeError(f"{name}: {text}: a jump that cannot be followed")
        last = block[-1][0] if block else ""
        jump = _JUMP.match(last)
        if jump:
            if jump.group(2) not in at:
                raise RuntimeError(f"{name}: {last}: a jump that cannot be followed")
            after[i].append(at[jump.group(2)])
        if last != _END and not last.startswith("s_branch") and i + 1 < len(blocks):
            after[i].append(i + 1)
    # the fewest loads at each block's start, over all paths to it (many: no copy in flight)
    many = 1 << 30
    start, todo = {0: many}, [0]
    while todo:
        i = todo.pop()
        end = _walk(blocks[i][1], None if start[i] == many else start[i])
        end = many if end is None else min(end, 64)
        for j in after[i]:
            if end < start.get(j, many + 1):
                start[j] = end
                todo.append(j)
    found = []
    for i, s in start.items():
        _walk(blocks[i][1], None if s == many else s, found)
    return found


def check_waits(listing: str) -> int:
    """The number of counted waits (vmcnt(n), n > 0, in asm statements) in the kernels of
    an assembly listing; raises where fewer than n loads may follow a copy into LDS that
    the wait is for."""
    kernels, name, lines = [], None, []
    for line in listing.splitlines():
        if name is None:
            label = _LABEL.match(line)
            if label and not line.startswith("."):
                name, lines = label.group(1), []
        elif line.startswith(".Lfunc_end"):
            kernels.append((name, lines))
            name = None
        else:
            lines.append(line)
    count = 0
    for name, lines in kernels:
        for n, loads in _kernel_waits(name, lines):
            if n == 0:
                continue
            count += 1
            if loads is not None and loads < n:
                raise RuntimeError(f"{name}: s_waitcnt vmcnt({n}) may leave a copy into LDS in flight: "
                                   f"only {loads} loads follow it")
    return count
