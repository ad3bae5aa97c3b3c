"""What the compiler makes of the F8 products and the router: wait states
(tests/wait_states.py), and the copies to LDS of the tiled product."""
import re
import subprocess

import pytest
import wait_states
from turboqwenfare_amd import build

SOURCES = ["tqf_f8.hip", "tqf_router.hip"]


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm")
    procs = {}
    for src in SOURCES:
        cmd = [build.hipcc_path(), *build.HIPCC_FLAGS, *build.EXTRA_FLAGS.get(src, []), "-w", "-S", "--cuda-device-only",
               str(build.CSRC / src), "-o", str(out / (src + ".s"))]
        procs[src] = subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    for src, p in procs.items():
        text, _ = p.communicate()
        assert p.returncode == 0, text.decode()
    return {src: (out / (src + ".s")).read_text() for src in SOURCES}


def kernels(text: str) -> dict:
    """The body of each kernel, by name."""
    out = {}
    for name in re.findall(r"^\s*\.amdhsa_kernel (\S+)", text, re.M):
        start = text.index(f"\n{name}:")
        out[name] = text[start:text.index("s_endpgm", text.rindex("s_endpgm", start, text.index(f".amdhsa_kernel {name}")) - 1)]
    return out


def copy_loops(body: str) -> list:
    """The copies to LDS that stand in a loop over the values of a vector register: the lanes whose value is the first
    one's copy, the others go round again, with EXEC narrowed by each pass."""
    lines = [line.split(";")[0].strip() for line in body.split("\n")]
    found = []
    for i, line in enumerate(lines):
        if line.startswith("buffer_load") and line.endswith("lds"):
            # such a loop narrows EXEC just before the copy, and takes the copied lanes out just after it
            near = [b for b in lines[max(0, i - 6):i] if b]
            after = [b for b in lines[i + 1:i + 4] if b]
            if any("saveexec" in b for b in near) and any("s_xor" in b or "s_andn2" in b for b in after):
                found.append(line)
    return found


@pytest.mark.parametrize("src", SOURCES)
def test_no_use_comes_too_soon(assembly, src):
    assert wait_states.violations(assembly[src]) == []


def test_copies_to_lds_are_not_looped(assembly):
    """A copy whose offset or descriptor the compiler keeps in vector registers becomes a loop that ends with EXEC empty;
    moves to other registers that are placed before EXEC is restored are then lost, and with them the rows' addresses."""
    seen = 0
    for name, body in kernels(assembly["tqf_f8.hip"]).items():
        copies = len(re.findall(r"buffer_load_dword\S* .*\blds\b", body))
        seen += copies
        assert copies or "tiled" not in name, name
        assert copy_loops(body) == [], name
    assert seen


def test_barriers_wait_for_the_block_they_publish(assembly):
    """The tiled product's barrier lets the newest N loads be under way, those of the block after the one that is
    needed: at least so many must have been issued since the barrier before."""
    seen = 0
    for name, body in kernels(assembly["tqf_f8.hip"]).items():
        lines = [line.split(";")[0].strip() for line in body.split("\n")]
        loads = None
        for line, after in zip(lines, lines[1:]):
            wait = re.match(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)$", line)
            if wait and after == "s_barrier":
                if loads is not None and int(wait[1]):
                    assert loads >= int(wait[1]), name
                    seen += 1
                loads = 0
            elif re.match(r"(buffer|global)_load", line):
                loads = None if loads is None else loads + 1
            elif re.match(r"\.LBB|s_c?branch", line):
                loads = None  # another path may lead here, or this one elsewhere
    assert seen


def test_no_register_spills(assembly):
    for src in SOURCES:
        assert set(re.findall(r"; ScratchSize: (\d+)", assembly[src])) == {"0"}


def test_the_check_sees_a_loop():
    loop = """
    s_mov_b64 s[2:3], exec
.LBB0_1:
    v_readfirstlane_b32 s6, v9
    v_cmp_eq_u32_e32 vcc, s6, v9
    s_and_saveexec_b64 vcc, vcc
    buffer_load_dwordx4 v1, s[8:11], s6 offen lds
    s_xor_b64 exec, exec, vcc
    s_cbranch_execnz .LBB0_1
"""
    assert len(copy_loops(loop)) == 1
    assert copy_loops(loop.replace("s_and_saveexec_b64 vcc, vcc", "s_nop 0")) == []
