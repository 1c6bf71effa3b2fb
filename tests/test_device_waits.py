"""Wait states that the architecture asks of the program, on the gfx950 machine code of this build's own lib/libom_hip.so
(CPU only). The compiler keeps them for the instructions that it emits itself and cannot see into an inline assembly string:

- a scalar write of m0 and a load with an LDS destination, which reads m0, need one wait state between them;
- a vector instruction's write of a scalar register and a vector memory instruction that reads that register as its address
  need five.

The loads' assembly is safe besides because nothing else in the library names m0: every instruction that does is the load's own
move, followed by its wait state and the load. (test_device_code.py asks for the load directly behind the move, without the wait
state: that one assertion does not hold for sound code.)
"""
import os
import re
import subprocess

from test_device_code import LLVM, _code_objects


def _functions(path):
    """Name and instructions of each function of a code object."""
    dis = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", path], check=True,
                         capture_output=True, text=True).stdout
    name, ins = "", []
    for line in dis.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if m:
            yield name, ins
            name, ins = m.group(1), []
            continue
        i = line.split("//")[0].strip()
        if i and not i.endswith(":"):
            ins.append(i)
    yield name, ins


def _wait_states(ins):
    """Wait states that an instruction is worth: one, s_nop N one more for each of N."""
    return 1 + (int(ins.split()[1], 0) if ins.startswith("s_nop") else 0)


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m.group(1))} if m else set()


def _operands(ins):
    parts = ins.split(None, 1)
    return [o.split()[0] for o in parts[1].split(",")] if len(parts) > 1 else []


def _faults(functions):
    loads, faults = 0, []
    for name, ins in functions:
        for at, load in enumerate(ins):
            if not load.startswith("global_load_lds"):
                continue
            loads += 1
            address = set().union(*(_scalars(o) for o in _operands(load)))
            waited = 0
            for before in reversed(ins[max(0, at - 5):at]):
                ops = _operands(before)
                if waited < 1 and before.startswith("s_") and ops[:1] == ["m0"]:
                    faults.append((name, before, load))
                if waited < 5 and before.startswith("v_") and ops and _scalars(ops[0]) & address:
                    faults.append((name, before, load))
                waited += _wait_states(before)
    return loads, faults


def test_loads_into_lds_keep_their_wait_states(tmp_path):
    loads, faults = 0, []
    for co in _code_objects(str(tmp_path)):
        n, f = _faults(_functions(co))
        loads, faults = loads + n, faults + f
    assert loads > 0 and not faults, (len(faults), loads, faults[:3])


def test_only_the_loads_own_moves_name_m0(tmp_path):
    moves = loads = 0
    for co in _code_objects(str(tmp_path)):
        for name, ins in _functions(co):
            for at, i in enumerate(ins):
                loads += i.startswith("global_load_lds")
                if re.search(r"\bm0\b", i):
                    moves += 1
                    assert i.startswith("s_mov_b32 m0, "), (name, i)
                    assert ins[at + 1:at + 2] == ["s_nop 0"], (name, ins[at:at + 3])
                    assert at + 2 < len(ins) and ins[at + 2].startswith("global_load_lds"), (name, ins[at:at + 3])
    assert moves == loads > 0, (moves, loads)


def test_the_look_itself():
    """What it finds and what it lets pass."""
    load = "global_load_lds_dwordx4 v1, s[4:5]"
    for ins, want in ((["s_mov_b32 m0, s3", load], 1), (["s_mov_b32 m0, s3", "s_nop 0", load], 0),
                      (["s_add_i32 m0, s3, s2", load], 1), (["s_mov_b32 m0, s3", "v_add_u32_e32 v3, v4, v5", load], 0),
                      (["v_readfirstlane_b32 s5, v9", "s_nop 3", load], 1), (["v_readfirstlane_b32 s5, v9", "s_nop 4", load], 0),
                      (["v_readfirstlane_b32 s6, v9", load], 0)):
        assert _faults([("f", ins)]) == (1, [("f", ins[0], load)] * want), ins
