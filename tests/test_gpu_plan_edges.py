"""The plan of a step where a length is out of range and positions go by the lengths."""
import pytest

from tests.test_gpu_paged_plan import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [-1, -9, -2 ** 31])
@pytest.mark.parametrize("batch", [2, 300])
@pytest.mark.parametrize("rows", [12, 17000])
def test_positions_of_a_clamped_length(session, length, batch, rows):
    """A length below 0 counts as 0, for the slots and, without `seen`, for the positions as well."""
    lengths, counts = [length, 5] + [0] * (batch - 2), [6, 3] + [0] * (batch - 2)
    held, table = [0, 1] + [0] * (batch - 2), [[-9, -9], [3, -9]] + [[-9, -9]] * (batch - 2)
    ring = [0, 1, 2] + [-8] * 5
    for seen in (None, [40, 50] + [0] * (batch - 2)):
        check(session, table, lengths, counts, held, seen, ring, [0, 3], 8, rows)
