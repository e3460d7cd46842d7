"""Properties of the compiled kernels of the experts' products that no result shows, or only now and then (no GPU needed).

1. No kernel spills a register.
2. expert_mm.hip writes its matrix instructions, its copies into LDS and their waits in assembly, which the compiler does not look into: a copy's
   descriptor has to be there when it is read, nothing but matrix instructions may write an accumulator among them, and no wait of the
   compiler's own may stand between them.
   So does expert_mm_few.hip with its copies and their waits."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_kernel_waits import _build_module

SOURCES = ["expert_mm.hip", "expert_mm_few.hip", "swiglu_grad.hip", "int8_quant.hip", "grad_norm.hip"]


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    build = _build_module()
    if not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm")
    started = [subprocess.Popen([build.HIPCC] + build.HIP_FLAGS + ["--cuda-device-only", "-S", os.path.join(build.CSRC, s), "-o", str(out / s)],
                                stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL) for s in SOURCES]
    assert [p.wait() for p in started] == [0] * len(started)
    return {s: (out / s).read_text() for s in SOURCES}


def kernels(text, name):
    """{kernel: its instructions and labels}"""
    found = {}
    for m in re.finditer(rf"^(_ZN5esmoe\d+{name}I\w+):", text, re.M):
        body = text[m.end():text.index(".end_amdhsa_kernel", m.end())]
        lines = [re.sub(r"\s+", " ", line).strip() for line in body.split("\n")]
        found[m.group(1)] = [line for line in lines if line and not line.startswith((";", ".p2", ".loc", ".set", ".section"))]
    return found


@pytest.mark.parametrize("source", SOURCES)
def test_no_kernel_spills(asm, source):
    text = asm[source]
    numbers = {key: re.findall(rf"\.{key}:\s+(\d+)", text) for key in ("private_segment_fixed_size", "sgpr_spill_count", "vgpr_spill_count")}
    count = len(re.findall(r"^\.end_amdhsa_kernel|^\s+\.end_amdhsa_kernel", text, re.M))
    assert count and numbers == {key: ["0"] * count for key in numbers}


def registers(operand):
    m = re.fullmatch(r"v\[(\d+):(\d+)\]", operand) or re.fullmatch(r"v(\d+)()", operand)
    return set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1)) if m else set()


@pytest.mark.parametrize("source", ["expert_mm", "expert_mm_few"])
def test_a_copys_descriptor_is_there_when_it_is_read(asm, source):
    """A vector instruction's write of a scalar register takes five slots until a memory instruction may read it."""
    copies = 0
    for name, lines in kernels(asm[source + ".hip"], source + "_kernel").items():
        for at, line in enumerate(lines):
            m = re.match(r"buffer_load_dwordx4 v\d+, s\[(\d+):(\d+)\].* lds", line)
            if not m:
                continue
            copies += 1
            slots = 0
            for before in reversed(lines[max(at - 14, 0):at]):
                w = re.match(r"v_read(?:first)?lane_b32 s(\d+)", before)
                if w and int(m.group(1)) <= int(w.group(1)) <= int(m.group(2)):
                    assert slots >= 5, (name, before, line)
                nop = re.match(r"s_nop (\d+)", before)
                slots += 0 if before.endswith(":") else int(nop.group(1)) + 1 if nop else 1
    assert copies > 100


def test_nothing_stands_between_the_matrix_instructions(asm):
    found = kernels(asm["expert_mm.hip"], "expert_mm_kernel")
    # two 16-bit types x (three forward forms and the rows' gradient, two ways to read the weights; the weights' gradient), int8: two forms, two ways
    assert len(found) == 2 * (4 * 2 + 1) + 2 * 2
    for name, lines in found.items():
        matrix = [i for i, line in enumerate(lines) if line.startswith("v_mfma")]
        between = lines[matrix[0]:matrix[-1] + 1]
        assert len(matrix) == 64, (name, len(matrix))   # one step's, once
        assert not [line for line in between if "vmcnt" in line and "explicit" not in line], name
        sums = set().union(*(registers(lines[i].split()[1].rstrip(",")) for i in matrix))
        assert len(sums) == 128, name
        for line in between:
            m = re.match(r"(v_|ds_read|buffer_load|global_load)(?!mfma|cmp)\S* (\S+?),", line)
            if m and " lds" not in line:
                assert not registers(m.group(2)) & sums, (name, line)


def loop_waits(lines):
    """Waits for memory in the innermost loop around all of a kernel's matrix instructions."""
    matrix = [i for i, line in enumerate(lines) if line.startswith("v_mfma")]
    labels = {line.split(":")[0]: i for i, line in enumerate(lines) if re.match(r"\.LBB\w+:", line)}
    back = [(labels[m.group(1)], i) for i, line in enumerate(lines) for m in [re.match(r"s_c?branch\w* (\.LBB\w+)", line)]
            if m and labels.get(m.group(1), i) < matrix[0] and i > matrix[-1]]
    begin, end = max(back)
    waits = [re.search(r"vmcnt\((\d+)\)( ; explicit)?", line) for line in lines[begin:end] if "vmcnt" in line]
    assert all(w.group(2) for w in waits)
    return len(matrix), [int(w.group(1)) for w in waits]


def test_few_rows_keep_their_copies_under_way(asm):
    """In the loop over steps: a wait for copies that leaves all but the oldest step's under way (and stores that are younger), and none of the compiler's."""
    found = kernels(asm["expert_mm_few.hip"], "expert_mm_few_kernel")
    # 16-bit: three shapes of three forward forms, two of the gradient; int8; two ways to read the weights
    assert len(found) == 2 * (2 * (3 * 3 + 2) + 2 * 3)
    for name, lines in found.items():
        row_tiles, col_tiles, depth = map(int, re.search(r"Li(\d+)ELi(\d+)ELi(\d+)ELb[01]EEEvNS_12", name).groups())
        assert loop_waits(lines) == (2 * row_tiles * col_tiles, [(depth - 1) * 2 * (row_tiles + col_tiles)]), name
    found = kernels(asm["expert_mm_few.hip"], "expert_mm_few_outer_kernel")
    assert len(found) == 2 and all(loop_waits(lines) == (16, [8, 16]) for lines in found.values())
