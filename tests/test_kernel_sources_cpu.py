"""Rules of the kernels' sources that no run shows (CPU only)."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "retree_b200" / "csrc"


def _code(name: str) -> str:
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", [p.name for p in sorted(CSRC.glob("*.cu")) if "setmaxnreg" in p.read_text()])
def test_a_warpgroup_changes_its_registers_in_one_instruction(name):
    """Every thread of a warpgroup has to run the same setmaxnreg: it opens a branch of whole warpgroups."""
    code = _code(name)
    sites = [m.start() for m in re.finditer(r"setmaxnreg", code)]
    assert sites
    for at in sites:
        before = code[:at].rstrip()
        assert before.endswith('asm volatile("'), before[-80:]
        opening = before[: -len('asm volatile("')].rstrip().splitlines()[-1].strip()
        split = re.fullmatch(r"(?:\} else )?if \(warp (?:<|>=) (\d+)\) \{", opening)
        assert opening == "} else {" or (split and int(split.group(1)) % 4 == 0), opening
    # one for each direction of a kernel
    kernels = code.count("__global__")
    assert code.count("setmaxnreg.dec") <= kernels and code.count("setmaxnreg.inc") <= kernels


def test_a_launch_control_answer_is_read_before_its_slot_is_freed():
    """The next answer is written by the async proxy: a proxy fence orders this one's reads before it."""
    body = _code("prompt_attn.cu").split("bool prompt_next(", 1)[1].split("return true;", 1)[0]
    read, fence = body.index("clc_taken("), body.index("fence_proxy_async_smem()")
    frees = [m.start() for m in re.finditer(r"mbar_arrive(_warp)?\(&bar\.clc_empty", body)]
    assert len(frees) == 2 and read < fence < min(frees)


def test_a_ring_stage_is_refilled_after_every_lane_has_read_it():
    """Votes order no memory; a __syncwarp does."""
    code = _code("tree_attn_q4.cu")
    refill = code.index("if (lane == 0 && i + kQsStages < tiles) issue(i + kQsStages);")
    assert code[:refill].rstrip().endswith("__syncwarp();")


def test_warps_are_whole_where_they_change_their_registers():
    """A lane's own branch right before an aligned instruction ends in a __syncwarp (or a block barrier)."""
    for name in ("prompt_attn.cu", "tree_attn_q4.cu"):
        code = _code(name)
        for m in re.finditer(r"setmaxnreg\.dec", code):
            before = code[: m.start()]
            barrier = max(before.rfind("__syncthreads();"), before.rfind("__syncwarp();"))
            assert not re.search(r"(tid|lane) == 0", before[barrier:]), name


def test_a_failed_cluster_query_is_asked_again_and_answers_are_per_device():
    body = _code("tree_attn_q4.cu").split("static int q4_clusters_fit(", 1)[1].split("\n}\n", 1)[0]
    assert "cudaGetDevice(&dev)" in body and "cache[dev]" in body
    assert body.index("if (n < 0) return 0;") < body.rindex("cache[dev]")
