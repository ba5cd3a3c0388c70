"""Host time of grouped mxfp4 calls."""

import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_call_costs_the_host_the_same_for_many_experts():
    """What the host works out before a launch does not grow with the experts (or the rows).

    A call takes the host some 25 us for its launches; a dependent product for each of up to 6.9 E rows
    made that 111 us for 16384 experts.  The smallest of 40 calls, so that a busy host does not count.
    """
    from mlxturbo_b200 import ops

    def least(E):
        rows, N, K = 4 * E, 16, 32
        w = torch.zeros(E, N, K // 8, dtype=torch.int32, device="cuda")
        s = torch.full((E, N, 1), 120, dtype=torch.uint8, device="cuda")
        ids = torch.arange(E, dtype=torch.int32, device="cuda").repeat_interleave(4)
        x = torch.zeros(rows, 1, K, dtype=torch.bfloat16, device="cuda")
        best = float("inf")
        for _ in range(40):
            torch.cuda.synchronize()
            t = time.perf_counter()
            ops.gather_qmm(x, w, s, None, rhs_indices=ids, group_size=32, bits=4, mode="mxfp4", sorted_indices=True)
            best = min(best, time.perf_counter() - t)
        torch.cuda.synchronize()
        return best * 1e6

    few, many = least(64), least(16384)
    print(f"host us: 64 experts {few:.1f}, 16384 experts {many:.1f}")
    assert many < 2 * few + 20
