"""The paged operators in calls that other tests do not make."""
import pytest

import paged_oracle
from test_paged_select_gpu import made, queries as tokens, selection

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu", [False, True])
@pytest.mark.parametrize("each,B", [(1, 3), (150, 4)])
def test_selection_in_a_wide_table(each, B, cu):
    """Tables much wider than any sequence, and more tokens than one round of the selection takes."""
    lens = [each, 700, 333 + each, 1100][:B]
    cache = paged_oracle.Cache(lens, 2, 64, cols=30001)
    boxes = made(cache)
    q = tokens(B * each + 2, 4, 64) if cu else tokens(B, each, 4, 64)
    selection(cache, boxes, q, [each] * B, 9, 1, 2, cu=cu)
