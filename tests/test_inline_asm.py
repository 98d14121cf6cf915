"""What the compiler is told about inline assembly: nothing keeps m0 as one statement left it until the next, so a load into LDS, which addresses through m0, sets it in
its own statement."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "camelid_amd", "csrc")


def statements(text):
    """The text of every asm statement's instructions."""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", text):
        yield "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))


def strays(text):
    """Statements that load into LDS and do not set m0 first, or that set it for a later one."""
    found = []
    for s in statements(text):
        ops = [i.strip().split()[0:2] for i in re.split(r"\\n(?:\\t)?|;", s) if i.strip()]
        sets = [k for k, op in enumerate(ops) if op[0].startswith("s_mov") and len(op) > 1 and op[1].startswith("m0")]
        loads = [k for k, op in enumerate(ops) if op[0].startswith(("global_load_lds", "buffer_load")) and "lds" in s]
        if any(not [k for k in sets if k < at] for at in loads) or (sets and not [at for at in loads if at > sets[-1]]):
            found.append(s)
    return found


def test_the_check_finds_a_stray():
    assert len(strays('asm volatile("s_mov_b32 m0, %0" ::"s"(a) : "memory", "m0"); asm volatile("s_nop 0\\n\\tglobal_load_lds_dword %0, off" ::"v"(p) : "memory");')) == 2
    assert not strays('asm volatile("s_mov_b32 m0, %1\\n\\ts_nop 0\\n\\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(a) : "memory", "m0");')


def test_every_load_into_lds_sets_m0_itself():
    n = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        text = open(path).read()
        n += len(list(statements(text)))
        assert strays(text) == [], path
    assert n > 5  # (statements were found)
