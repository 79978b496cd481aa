"""Host limits of the rotating appends (CPU: every call here is refused before it reaches
a GPU)."""
import pytest

from test_q4_args import UNSUPPORTED, _append, _q4_append, _refused


@pytest.mark.parametrize("call", [_append, _q4_append])
@pytest.mark.parametrize("batch,rows", [(1 << 14, 1 << 14), ((1 << 27) + 1, 1), (1, (1 << 31) - 1), (1 << 15, 1 << 15)])
def test_more_tokens_than_a_grid_holds(call, batch, rows):
    """Past 2^27 tokens a launch would fail where it is enqueued, with no word of the sizes."""
    for d in (64, 128):
        _refused(call(batch=batch, rows=rows, d=d, sq=8 * d, sk=2 * d, sv=2 * d), UNSUPPORTED, "rows")
