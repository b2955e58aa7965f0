"""What the kernels with tensor memory owe one another and cannot show by running: an allocation waits without a limit, and tensor memory that another
CTA's MMAs write is handed over by barriers.  Read from the sources."""
import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "miori_b200", "csrc")


def code(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


def kernels():
    """(name, body) of every kernel that allocates tensor memory."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        for part in code(path).split("__global__")[1:]:
            if "tcgen05.alloc" in part:
                found.append((re.search(r"(\w+_kernel)\(", part).group(1), part))
    return found


def test_they_are_found():
    assert {name for name, _ in kernels()} >= {"gemm_fp8_pair_kernel", "gemm_fp8_swap_kernel", "gemm_skinny_kernel", "attention_prompt_kernel"}
    assert len(kernels()) >= 6


@pytest.mark.parametrize("name,body", kernels(), ids=[name for name, _ in kernels()])
def test_dependents_start_behind_the_allocation(name, body):
    """A dependent grid may take an SM's free columns as soon as it is let go, and keeps them until this grid is done: a CTA that has yet to allocate would wait for it, and
    it for the CTA.  One warp allocates and then lets go, and nobody else does."""
    assert body.count("pdl_launch_dependents") == 1 and body.count("tcgen05.alloc") == 1
    assert body.index("tcgen05.alloc") < body.index("pdl_launch_dependents")
    between = body[body.index("tcgen05.alloc"):body.index("pdl_launch_dependents")]
    assert "}" not in re.sub(r'"[^"]*"', "", between), "in the allocating warp's own block"


def test_hand_overs_between_ctas():
    """The second CTA of a pair tells the leader that its sums are read, and the leader's MMAs write over them.  Of tensor memory: fences on either side of a barrier whose
    arrival and wait reach over the cluster, in the thread that passes the word on too.  Sums in shared memory: released, and acquired, by the cluster."""
    fp8 = code(os.path.join(CSRC, "gemm_fp8.cuh"))
    remote = re.findall(r"mapa\.shared::cluster\.u32 ra.*?\[ra\]", fp8)
    assert remote and all("mbarrier.arrive.relaxed.cluster" in a for a in remote)
    relay = fp8[:fp8.index("arrive_leader(taken(b))")].rsplit("mbar_wait(taken(b)", 1)[1]
    assert relay.index("fence_after();") < relay.index("fence_before();")
    leader = fp8[fp8.index("warp_wait<Order::TENSOR>(taken(b)"):]
    assert leader.index("fence_after();") < leader.index("umma_e4m3<2>")
    wait = code(os.path.join(CSRC, "common.cuh"))
    assert wait.count("mbarrier.try_wait.parity.relaxed.cluster") == 1 and wait.count("mbarrier.try_wait.parity.acquire.cluster") == 1
    assert "mbar_wait<true, Order::CLUSTER>(smem_addr(&arrived)" in code(os.path.join(CSRC, "moe.cuh"))


def test_whole_warps_come_to_barriers_of_whole_warps():
    """barrier.cluster and bar.sync in their aligned forms take warps whose lanes are together.  Behind code whose lanes part, a loop over columns or one that leaves at an abort,
    they are brought together first."""
    fp8 = code(os.path.join(CSRC, "gemm_fp8.cuh"))
    swap = fp8[fp8.index("gemm_fp8_swap_kernel("):fp8.index("struct GemmOperands")]
    barriers = [m.start() for m in re.finditer(r"if \(geo\.cs > 1u\) cluster_barrier\(\);|asm volatile\(\"bar\.sync 1, 128;", swap)]
    assert len(barriers) == 4
    for at in barriers:
        before = [line.strip() for line in swap[:at].splitlines() if line.strip()]
        # ... or nothing lies between it and such a place but stores that every lane makes
        tail = "\n".join(before[-26:])
        assert "__syncwarp();" in tail and "continue" not in tail.rsplit("__syncwarp();", 1)[1] and "break" not in tail.rsplit("__syncwarp();", 1)[1], tail
    for part in (fp8[:fp8.index("gemm_fp8_swap_kernel(")], swap):
        leaving = part[part.index("__nanosleep"):]
        assert leaving.index("__syncwarp();") < leaving.index("__syncthreads();")


def test_a_cluster_is_waited_for_without_tensor_memory():
    """A CTA of gemm_fp8's few-row kernel frees its columns in front of its first wait for others of its cluster: theirs may be waiting for columns, without a limit, that a CTA
    holds which waits for this one.  (Pairs allocate together, and their registers leave an SM to them alone.)"""
    swap = code(os.path.join(CSRC, "gemm_fp8.cuh"))
    swap = swap[swap.index("gemm_fp8_swap_kernel("):swap.index("struct GemmOperands")]
    freed, meeting = swap.index("tcgen05.dealloc"), swap.index("cluster_barrier()")
    assert freed < meeting
    before = swap[:freed]
    assert before.rindex('"bar.sync 2, 160;"') < before.rindex("fence_after();")  # behind the warps that read it
    readers = swap[:swap.index('"bar.arrive 2, 160;"')]
    assert readers.rindex("tmem_wait16") < readers.rindex("fence_before();")
