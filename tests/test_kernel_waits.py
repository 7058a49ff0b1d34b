"""What the kernels for scoring and for drafted tokens do about waits, read from their sources: no input makes a wait run out."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "glm_tpu_b200" / "csrc"
KERNELS = ("tree_attention.cu", "head_logprobs_tcgen05.cu")


def code_of(name: str) -> str:
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", KERNELS)
def test_waits_are_a_whole_warps(name):
    """Instructions of the whole warp follow every wait, and a lane whose wait ran out alone would leave the others waiting for it."""
    code = code_of(name)
    assert "mbar_wait_warp(" in code and not re.search(r"\bmbar_wait\(", code)
    assert not re.search(r"(\|\||&& !)\s*fail\b", code)  # nor does a lane decide by itself to leave


@pytest.mark.parametrize("name, load", [("tree_attention.cu", "ta_tmem_ld32_nowait"), ("head_logprobs_tcgen05.cu", "hl_tmem_ld32_nowait"), ("tcgen05.cuh", "tmem_ld32"), ("tcgen05.cuh", "tmem_ld16")])
def test_a_warp_meets_before_it_loads_from_tensor_memory(name, load):
    body = code_of(name).split(f"void {load}(")[1].split("asm volatile")[0]
    assert "__syncwarp();" in body


@pytest.mark.parametrize("name", KERNELS)
def test_who_reads_the_failure_word_decides_for_a_whole_warp(name):
    """Other warps set it whenever their waits run out: what one warp reads, the next one need not."""
    code = code_of(name)
    reads = [code[: m.end()] for m in re.finditer(r"\bfail\b(?! = )", code) if not code[: m.start()].endswith("uint32_t ")]
    assert reads and all(read.endswith("__any_sync(0xffffffffu, fail") for read in reads), [read[-60:] for read in reads]


def test_warps_that_join_copies_leave_together():
    """Their barrier has no limit, so a segment's first one also decides, for all four, whether there will be a next one."""
    output = code_of("tree_attention.cu").split("if (!ok && !JOINS) break;")[1].split("mbar_arrive(o_free + t);")[0]
    first, rest = output.split("ok = !ta_any_of_group(!ok);")
    assert "bar.sync" not in first and not re.search(r"\bok\b", first) and rest.lstrip().startswith("if (!ok) break;")
    assert rest.count("bar.sync 1, 128") == 2 and not re.search(r"\bok\b|\bfail\b", rest.split("if (!ok) break;", 1)[1])


def test_sums_that_a_lost_wait_leaves_out_are_no_numbers():
    """The status word may be nobody's: what was not summed up must not be read as if it had been."""
    code = code_of("head_logprobs_tcgen05.cu")
    assert code.count("C::commit(acc_full + acc)") == 1 and "if (ok && elect_one()) C::commit(acc_full + acc);" in code  # abandoned sums are not announced
    lost = code.split("GLMB_STATUS_WAIT_TIMEOUT);")[1].split("} else if (plan.keeps")[0]
    assert "p.part[" in lost and "__int_as_float(0x7fffffff)" in lost and "while (!plan.keeps && hl_tile(" in lost
    code = code_of("tree_attention.cu")
    after = code.split("raise_status(a.status, GLMB_STATUS_WAIT_TIMEOUT);")[1].split("if (sh.whole && a.clear_rest)")[0]
    assert "if (MODE != TA_SINGLE || t == 0) tree_lost<MODE, COPIES, JOINS>(a, sh, walk, s, t, quarter * 32 + lane);" in after  # the group that stores the output
    lost = code.split("void tree_lost(")[1].split("while (walk.next(a, sh, s));")[0]
    assert "make_float2(none, none)" in lost and "make_uint4(~0u, ~0u, ~0u, ~0u)" in lost
