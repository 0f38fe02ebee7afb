"""Blocks of a cluster may touch one another's shared memory only after all of them run: a kernel that
does so has a cluster barrier in front of its first such access.  Read from the sources: on the GPU the
missing barrier is a race that mostly goes well."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flash_muon_b200" / "csrc"
REMOTE = re.compile(r"map_shared_rank\(|ptx::mapa\(")
BARRIER = re.compile(r"barrier_wait\(|cluster\.sync\(|cluster_sync\(")


def first_remote_accesses(source):
    """For each kernel that touches another block's shared memory, its text up to there."""
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    for kernel in text.split("__global__")[1:]:
        remote = REMOTE.search(kernel)
        if remote:
            yield kernel[:remote.start()]


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.cu")))
def test_remote_shared_memory_is_touched_behind_a_cluster_barrier(source):
    for before in first_remote_accesses(source):
        assert BARRIER.search(before), before[:120]


def test_the_rule_sees_the_kernels_with_clusters():
    assert [len(list(first_remote_accesses(s))) for s in ("grad_norm.cu", "gemm_tc2.cu", "adamw.cu")] == [1, 1, 0]
