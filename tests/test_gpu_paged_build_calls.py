"""Plans built on the GPU: calls that test_gpu_paged_build.py does not make."""
import numpy as np
import pytest

from test_gpu_paged import Q8
from test_gpu_paged_build import I32, Lists

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [0, 1], ids=["one", "many"])
def test_pages_of_sequences_without_new_tokens_under_a_window(gctx, spread):
    """No new token sees them: they may be absent, as they may in plans set from the host.  By the
    kernel of one workgroup, and (among many sequences of nothing) by those of several."""
    n = 3 + 3000 * spread
    pool = gctx.pool(1, 1, 64, 16, Q8)
    pool.take(16)
    tables = np.full((n, 6), -1, I32)
    tables[1, 3:5] = 3, 4
    for window, sinks, M, code in ((70, 0, 2, 0), (70, 65, 0, 0), (1 << 20, 0, 0, 0), (0, 0, 0, -1)):
        plan = pool.device_plan(n, 4, 4, 6, 2, window=window, sinks=sinks)
        ls = Lists(gctx, [300] * 3 + [0] * (n - 3), [0, M, 0] + [0] * (n - 3), tables, [9], 0, 4)
        ls.build(plan)
        if code:
            ls.refused(code)
        else:
            ls.check()
        ls.free(), plan.free()
    host = pool.plan([([-1] * 5, 300, 0), ([-1, -1, -1, 3, 4], 300, 2)], 2, 70)
    host.free()
    pool.free()
