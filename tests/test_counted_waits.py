"""The build's check of hand-written counted waits: a copy into LDS has to be followed by
as many loads as the wait leaves in flight, on every path."""
import re

import pytest

from nanokv_amd import build
from nanokv_amd._waits import check_waits

COPY = ["buffer_load_dwordx4 v1, s[8:11], 0 offen lds"]
LOAD = ["global_load_dwordx4 v[2:5], v[6:7], off"]
PAIR = ["global_load_dwordx2 v[2:3], v[6:7], off offset:64"]
READ = ["ds_read_b128 v[2:5], v6"]
END = ["s_endpgm"]


def wait(n):
    return [";;#ASMSTART", f"s_waitcnt vmcnt({n})", ";;#ASMEND"]


def kernel(*parts, name="_Z1kv"):
    lines = [x for part in parts for x in part]
    body = "\n".join(x if x.endswith(":") or x.startswith(";;") else "\t" + x for x in lines)
    return f"\t.text\n{name}:                 ; @{name}\n; %bb.0:\n{body}\n.Lfunc_end0:\n\t.size x, 1\n"


def test_as_many_loads_as_the_wait_leaves():
    assert check_waits(kernel(COPY * 4, LOAD * 4, PAIR * 4, wait(8), READ, END)) == 1
    assert check_waits(kernel(COPY, LOAD * 9, wait(8), READ, END)) == 1
    assert check_waits(kernel(COPY, wait(0), READ, END)) == 0
    assert check_waits("\t.text\n") == 0


@pytest.mark.parametrize("loads", range(8))
def test_a_load_that_is_missing(loads):
    with pytest.raises(RuntimeError, match="vmcnt\\(8\\) may leave a copy"):
        check_waits(kernel(COPY * 4, LOAD * loads, wait(8), READ, END))


def test_loads_before_the_last_copy_and_other_instructions_do_not_count():
    with pytest.raises(RuntimeError, match="only 7"):
        check_waits(kernel(COPY, LOAD, COPY, LOAD * 7, wait(8), READ, END))
    with pytest.raises(RuntimeError, match="only 7"):
        check_waits(kernel(COPY, LOAD * 7, ["global_store_dword v1, v2, s[0:1]", "s_load_dword s0, s[2:3]",
                                            "ds_write_b32 v0, v1"], READ, wait(8), END))


def test_a_path_that_skips_a_load():
    with pytest.raises(RuntimeError, match="only 7"):
        check_waits(kernel(COPY, LOAD * 7, ["s_cbranch_scc1 .LBB0_2"], LOAD, [".LBB0_2:"], wait(8), READ, END))


def test_a_loop_is_followed_around():
    def loop(before, inside):
        return kernel(COPY, LOAD * before, [".LBB0_1:"], wait(8), READ, COPY, LOAD * inside,
                      ["s_cbranch_scc1 .LBB0_1"], wait(8), READ, END)
    assert check_waits(loop(8, 8)) == 2
    for before, inside in ((7, 8), (8, 7)):
        with pytest.raises(RuntimeError, match="only 7"):
            check_waits(loop(before, inside))


def test_copies_that_have_arrived_need_no_loads():
    for arrived in (["s_waitcnt vmcnt(0) lgkmcnt(0)"], LOAD + ["s_waitcnt vmcnt(1)"], wait(0)):
        assert check_waits(kernel(COPY, arrived, LOAD, wait(8), READ, END)) == 1
    with pytest.raises(RuntimeError):
        check_waits(kernel(COPY, ["s_waitcnt vmcnt(1)", "s_waitcnt lgkmcnt(0)"], LOAD, wait(8), READ, END))


def test_the_kernel_is_named_and_others_pass():
    good, bad = kernel(COPY, LOAD * 8, wait(8), END, name="good"), kernel(COPY, wait(8), END, name="bad")
    with pytest.raises(RuntimeError, match="^bad:"):
        check_waits(good + bad + good)
    assert check_waits(good + good) == 2


def test_a_jump_that_cannot_be_followed():
    for jump in ("s_setpc_b64 s[0:1]", "s_branch .LBB9_9"):
        with pytest.raises(RuntimeError, match="cannot be followed"):
            check_waits(kernel(COPY, LOAD * 8, [jump], wait(8), END))


@pytest.mark.parametrize("src", build.COUNTED_WAITS)
def test_the_built_kernels(src):
    """Each kernel's waits are found, and they no longer pass once a load is gone."""
    path = build.listing(src)
    if not path.exists():
        pytest.skip("the library was built elsewhere")
    text = path.read_text()
    assert check_waits(text) == text.count("s_waitcnt vmcnt(8)\n\t;;#ASMEND") > 0
    # one kernel's loads, each of which is taken out in turn (those of the first tile may
    # be waited for before the loop, those of the tiles to come are not)
    start = text.rindex("\n_Z", 0, text.index("s_waitcnt vmcnt(8)\n\t;;#ASMEND"))
    lines = text[start + 1:text.index("\n.Lfunc_end", start) + 13].split("\n")
    assert check_waits("\n".join(lines)) == 2
    refused = 0
    for i, line in enumerate(lines):
        if re.match(r"\s+global_load_dwordx[24] ", line):
            try:
                check_waits("\n".join(lines[:i] + lines[i + 1:]))
            except RuntimeError as e:
                refused += "only 7" in str(e)
    assert refused >= 8
