"""What a kernel that starts before its predecessor on the stream has ended (a programmatic dependent
launch) may and may not do, read off the sources: the memory it reads is still being written while it
is resident, and only ``griddepcontrol.wait`` ends that."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "qwen-ascend_b200" / "csrc"


def functions():
    """``{name: (declaration, body)}`` of the kernels and device functions, comments left out."""
    out = {}
    for path in sorted(CSRC.glob("*.cuh")):
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)
        for m in re.finditer(r"^(?:__global__|FNX_DEV)\b[^;{}]*?\b(?!__launch)(\w+)\(([^;{}]*)\)\s*\{", text, flags=re.M):
            depth, i = 1, m.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[i], 0)
                i += 1
            out[m.group(1)] = (m.group(0), text[m.end():i])
    return out


FUNCTIONS = functions()
DEPENDENT = {n for n, (d, b) in FUNCTIONS.items() if d.startswith("__global__") and "pdl_wait()" in b}


def test_the_dependent_kernels_are_found():
    assert {"column_sum_kernel", "decode_stream_kernel", "ffn_gemm_kernel", "ffn_small_kernel", "inject_norm_kernel",
            "inject_norm_bwd_kernel", "inject_norm_bwd_wide_kernel", "w4_dense_kernel",
            "w4_dense_tma_kernel"} <= DEPENDENT


def test_no_dependent_kernel_declares_its_memory_unaliased():
    """``__restrict__`` says that nobody else writes the memory while the kernel runs, which lets the
    compiler load it early or through the read-only path: before the wait that makes it valid."""
    assert [n for n in sorted(DEPENDENT) if "__restrict__" in FUNCTIONS[n][0]] == []


def test_nothing_a_dependent_kernel_calls_reads_through_the_read_only_path():
    """``__ldg`` carries the same promise to the compiler and the cache as ``__restrict__``."""
    reached, todo = set(), sorted(DEPENDENT)
    while todo:
        name = todo.pop()
        reached.add(name)
        todo += [c for c in re.findall(r"\b(\w+)\s*(?:<[^;(){}]*>)?\(", FUNCTIONS[name][1])
                 if c in FUNCTIONS and c not in reached]
    assert "d2_stage_rows" in reached
    assert [n for n in sorted(reached) if re.search(r"__ldg\b|\bld_nc_v4\b|ld\.global\.nc", FUNCTIONS[n][1])] == []


def test_bounded_waits_begin_after_the_predecessor_has_ended():
    """A bounded wait counts the time that a copy or a product may take.  Begun before the kernel's own
    ``pdl_wait`` it would count what is left of the kernel before, and give up on a launch that lacks
    nothing.  Every warp's path through a kernel therefore waits for the predecessor first."""
    for name, roles in (("ffn_small_kernel", 3), ("ffn_gemm_kernel", 1), ("inject_norm_bwd_kernel", 1),
                        ("w4_dense_tma_kernel", 1)):
        # one pdl_wait at the head of the kernel, or (ffn_small) one in each warp's branch
        branches = re.split(r"\} else if \(warp [=<]+ \d+\) \{", FUNCTIONS[name][1]) if roles > 1 else [FUNCTIONS[name][1]]
        assert len(branches) == roles, name
        for branch in branches:
            first = re.search(r"\b(?:mbar_\w*wait\w*|mbar_spin|ffn_copy_tile\S*|ffn_multiply_tile\S*)\(", branch)
            assert first and 0 <= branch.find("pdl_wait()") < first.start(), (name, branch[:60])


def test_a_block_gives_up_as_one():
    """Each thread's own clock ends its bounded wait.  Where the threads meet at block barriers inside the
    loop behind it, one that gave up alone would leave the others with sums that lack its part."""
    body = FUNCTIONS["inject_norm_bwd_kernel"][1]
    said = re.search(r"const bool (\w+) = mbar_wait\(&full", body)
    assert said and f"if (!__syncthreads_and({said.group(1)}))" in body
