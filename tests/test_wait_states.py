"""Wait states that the hardware leaves to the program, in the code that was
built. A vector memory instruction that reads a scalar register which a vector
instruction wrote has to come 5 wait states after it. The compiler sees to that
for its own instructions, but not for those inside an asm statement, which have
to keep the distance themselves whatever comes before them."""
import re

import pytest

from tests import code_object

pytestmark = pytest.mark.skipif(not code_object.available(), reason="library not built, or no ROCm tools")
NEEDED = 5


def scalars(text):
    """The scalar registers among operands."""
    out = set()
    for a, b in re.findall(r"(?<![\w:])s\[(\d+):(\d+)\]", text):
        out.update(range(int(a), int(b) + 1))
    out.update(int(x) for x in re.findall(r"(?<![\w:])s(\d+)\b", text))
    return out | ({"vcc"} if re.search(r"\bvcc", text) else set())


def written(i):
    """The scalar registers that a vector instruction writes: its first operand,
    or the carry behind it."""
    if not i.op.startswith("v_"):
        return set()
    args = i.args.split(", ")
    out = scalars(args[0])
    if len(args) > 1 and re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co_|v_div_scale|v_mad_[iu]64", i.op):
        out |= scalars(args[1])
    return out


def states(i):
    return int(i.args, 0) + 1 if i.op == "s_nop" else 1


def too_close(body):
    """(distance, writer, reader) of every vector memory instruction that comes
    too early, by any way through the function."""
    at = {x.at: k for k, x in enumerate(body)}
    before = [[] for _ in body]
    for k, x in enumerate(body):
        if k + 1 < len(body) and x.op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[k + 1].append(k)
        if x.op.startswith(("s_branch", "s_cbranch")) and x.to in at:
            before[at[x.to]].append(k)
    out = []
    for k, x in enumerate(body):
        if not x.op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            continue
        reads = scalars(x.args)
        ways = [(j, 0) for j in before[k]]
        while reads and ways:
            j, passed = ways.pop()
            if passed >= NEEDED:
                continue
            if written(body[j]) & reads:
                out.append((passed, body[j], x))
                continue
            ways += [(i, passed + states(body[j])) for i in before[j]]
    return out


def faults(*names):
    found = {name: too_close(body) for name, body in code_object.functions().items() if any(n in name for n in names)}
    assert found
    return {name: x for name, x in found.items() if x}


def test_the_check_finds_what_it_looks_for():
    I = code_object.Instruction
    read = I("v_readlane_b32", "s5, v1, 3", 0, None)
    load = I("buffer_load_dwordx4", "v2, s[8:11], s5 offen lds", 40, None)
    move = I("s_mov_b32", "m0, s6", 8, None)
    for nops, n in ((0, 1), (2, 1), (3, 0)):
        assert len(too_close([read, move, I("s_nop", str(nops), 12, None), load])) == n
    # round a loop: the branch to the load counts
    body = [load, I("s_nop", "4", 48, None), read._replace(at=52), I("s_cbranch_scc1", "65000", 56, 40), I("s_endpgm", "", 60, None)]
    assert [x[0] for x in too_close(body)] == [1]
    assert not too_close([I("s_add_u32", "s5, s5, s6", 0, None), load])
    assert too_close([I("v_add_co_u32", "v1, s[8:9], v1, v2", 0, None), load])


def test_rows_of_the_paged_cache():
    assert not faults("paged_rows_kernel")


def test_every_kernel():
    assert not faults("")


def test_loads_into_lds_keep_the_distance_themselves():
    """Whatever the compiler puts before them: a move to M0 and the waits, then
    loads that go on by the same registers."""
    n = 0
    for name, body in code_object.functions().items():
        for k, x in enumerate(body):
            if not x.op.startswith("buffer_load") or not re.search(r"\blds$", x.args):
                continue
            passed, j = 0, k
            while body[j].op.startswith(("buffer_load", "s_nop")) or body[j].args.startswith("m0, m0,"):
                passed += states(body[j]) if j < k else 0
                assert j == k or scalars(body[j].args) <= scalars(x.args), name
                j -= 1
            assert body[j].op == "s_mov_b32" and body[j].args.startswith("m0,") and passed + 1 >= NEEDED, name
            n += 1
    assert n > 1000
