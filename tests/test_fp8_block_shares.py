"""Tiles that several clusters of the block-scaled GEMM share: how they are counted off, on the CPU, and that the counters are zero
again behind a call, on the GPU."""
import os
import random
import re

import pytest
import torch

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llmqrt_b200", "csrc", "gemm_fp8_block.cu")


def _sharer_of(u, total, sharers):
    return ((u + 1) * sharers - 1) // total


def _walk(cluster, rest, kb, sharers):
    """The shared tiles of a cluster and its K blocks of each (PairWork)."""
    u, end = cluster * rest * kb // sharers, (cluster + 1) * rest * kb // sharers
    while u < end:
        tile, k0 = divmod(u, kb)
        k1 = min(kb, k0 + end - u)
        u += k1 - k0
        yield tile, k0, k1


def test_every_share_is_counted_once():
    """A counter has an arrival of each cluster between the tile's first and its last, and of no other, whatever the order; clusters that gave
    up arrive like the others, so every counter ends at zero."""
    rng = random.Random(0)
    for _ in range(300):
        kb, rest = rng.randint(1, 200), rng.randint(1, 73)
        sharers = rng.choice([s for s in (3 * rest, 2 * rest, 74) if s >= rest and rest * kb >= 4 * s] or [rest])
        arrivals = [(tile, c) for c in range(sharers) for tile, k0, k1 in _walk(c, rest, kb, sharers) if k1 - k0 < kb]
        rng.shuffle(arrivals)
        counters, finished = [0] * rest, []
        for tile, _ in arrivals:
            first, last = (_sharer_of(u, rest * kb, sharers) for u in (tile * kb, tile * kb + kb - 1))
            before, counters[tile] = counters[tile], counters[tile] + 1
            if before == last - first:
                counters[tile] = 0
                finished.append(tile)
        assert not any(counters) and sorted(finished) == sorted({t for t, _ in arrivals})


def test_a_warp_that_gives_up_counts_itself_off():
    """The epilogue leaves its walk over the tiles only behind the loop that counts off what is left of its share."""
    src = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    kernel = src[src.index("block_pair_kernel(const"):]
    epilogue = kernel[kernel.index("setmaxnreg.inc"):kernel.index("tma_stores_done")]
    leaves = [m.start() for m in re.finditer(r"\bbreak;|\breturn;", epilogue)]
    assert len(leaves) == 1
    given_up = epilogue[epilogue.index("warp_aborted(abort)"):leaves[0]]
    assert re.search(r"do \{.*counted_off\(.*\} while \(work\.next\(", given_up, re.S)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(256, 300, 18944), (300, 300, 3584), (512, 896, 4864), (2048, 3584, 18944), (1000, 4608, 3584), (333, 3584, 8960)])
def test_counters_are_zero_behind_a_call(M, N, K):
    from llmqrt_b200 import _lib, ops
    f8 = lambda *s: torch.ones(s, device="cuda").to(torch.float8_e4m3fn)  # noqa: E731
    kb, dev = -(-K // 128), torch.device("cuda", torch.cuda.current_device())
    a_s, w_s = torch.ones(M, kb, device="cuda"), torch.ones(-(-N // 128), kb, device="cuda")
    for _ in range(2):
        out = ops.fp8_linear_block(f8(M, K), f8(N, K), None, a_s, w_s, torch.bfloat16)
        assert (out == torch.tensor(float(K), device="cuda").bfloat16()).all()
        assert not _lib.workspace(dev)[: _lib.STATUS_OFFSET - 4].any() and _lib.kernel_status(dev) == 0
