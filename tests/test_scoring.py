"""How continuations are divided over passes (CPU)."""

import pytest

from aiproj_amd.inference.scoring import _passes


@pytest.mark.parametrize("lengths,most,runs", [
    ([1], 4, [(0, 1)]),
    ([2, 2, 1, 4, 3], 4, [(0, 2), (2, 3), (3, 4), (4, 5)]),
    ([9, 1, 9], 4, [(0, 1), (1, 2), (2, 3)]),              # longer than a pass: one of its own
    ([1, 1, 1, 1], 100, [(0, 4)]),
    ([3, 3], 3, [(0, 1), (1, 2)]),
])
def test_passes(lengths, most, runs):
    assert _passes(lengths, most) == [range(a, b) for a, b in runs]
