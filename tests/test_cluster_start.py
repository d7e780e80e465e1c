"""A cluster's CTAs may be written to only once all of them run.  Their kernels arrive at the cluster's barrier when they
begin and wait there before the first store to another CTA's shared memory; loads from it all follow a full barrier.  Which
CTA starts first is not a test's to choose, so the order is read in the source."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llm-inference-optimizer_b200" / "csrc"


def body(file: str, kernel: str) -> str:
    """The kernel's text from its name on, without comments."""
    text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
    begin = re.search(rf"\b{kernel}\(", text).end()
    depth = 0
    for i in range(text.index("{", begin), len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[begin:i]
    raise AssertionError(f"{kernel} does not end")


@pytest.mark.parametrize("file,kernel,store", [("qsample.cuh", "sample_kernel", r"all_u32<"),
                                               ("qdec.cuh", "qdec_kernel", r"st_dsmem_f32\("),
                                               ("qgemm.cuh", "qgemm_kernel", r"st_dsmem_f32\(")])
def test_all_run_before_the_first_store(file, kernel, store):
    text = body(file, kernel)
    at = [re.search(pattern, text) for pattern in (r"cluster_arrive_relaxed\(\)", r"cluster_wait\(\)", store)]
    assert all(at), f"{kernel}: the cluster's CTAs are not waited for"
    assert at[0].start() < at[1].start() < at[2].start()
