"""What the compiler makes of the attention's kernels: wait states, copies to LDS outside of loops over lanes, and no
registers in memory."""
import re
import subprocess

import pytest
import wait_states
from test_f8_assembly import copy_loops, kernels
from turboqwenfare_amd import build

SOURCES = ["tqf_rope.hip", "tqf_prompt.hip", "tqf_paged.hip"]


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


@pytest.mark.parametrize("src", SOURCES)
def test_no_use_comes_too_soon(assembly, src):
    assert wait_states.violations(assembly[src]) == []


@pytest.mark.parametrize("src, kernel", [("tqf_prompt.hip", "prompt_kernel"), ("tqf_paged.hip", "paged_kernel")])
def test_copies_to_lds_are_not_looped(assembly, src, kernel):
    """Descriptors and scalar offsets are the same in every lane, and the compiler knows it."""
    seen = 0
    for name, body in kernels(assembly[src]).items():
        copies = len(re.findall(r"buffer_load_dword\S* .*\blds\b", body))
        assert copies or kernel not in name, name
        assert copy_loops(body) == [], name
        seen += copies
    assert seen


@pytest.mark.parametrize("src", SOURCES)
def test_no_registers_in_memory(assembly, src):
    sizes = re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", assembly[src])
    assert sizes and set(sizes) == {"0"}
