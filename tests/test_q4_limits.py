"""Host limits of the rotating appends, and workspaces of the 4-bit cache (CPU: every call
here is refused before it reaches a GPU)."""
import pytest

import kvhp
from test_q4_args import UNSUPPORTED, _append, _q4_append, _refused


@pytest.mark.parametrize("call", [_append, _q4_append])
@pytest.mark.parametrize("batch,rows", [(1 << 14, 1 << 14), ((1 << 27) + 1, 1), (1, (1 << 31) - 1), (1 << 15, 1 << 15)])
def test_more_tokens_than_a_grid_holds(call, batch, rows):
    """Past 2^27 tokens a launch would fail where it is enqueued, with no word of the sizes."""
    for d in (64, 128):
        _refused(call(batch=batch, rows=rows, d=d, sq=8 * d, sk=2 * d, sv=2 * d), UNSUPPORTED, "rows")


def test_less_work_may_need_more_workspace():
    """What kvhp_c.h says of the sizes: each call's own is to be asked for."""
    rows, step = kvhp.q4_prefill_workspace_bytes, kvhp.q4_decode_workspace_bytes
    assert rows(1, 8192, 32, 8, 128, 8192) == 0 < rows(1, 128, 32, 8, 128, 8192) < 34.1e6
    assert rows(1, 1, 32, 8, 128, 8192) < rows(1, 20, 32, 8, 128, 8192)
    assert step(5, 32, 8, 128, 3904) < step(5, 32, 8, 128, 3840)
