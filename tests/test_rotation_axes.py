"""The axes of a rotation's pairs as the Python call takes them (CPU only)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from antfly_amd import _lib, paged  # noqa: E402


def rotation(pair_axes):
    key = torch.zeros(3, 2, 64)
    return paged.headRotation(None, key, None, key, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(8), pair_axes=pair_axes)


def test_axes_of_pairs():
    want = [0, 1, 1, 0, 1, 0, 0, 1]
    for given in (want, tuple(want), bytes(want), np.array(want), np.array(want, np.uint8), torch.tensor(want)):
        assert list(rotation(given).pair_axes) == want + [0] * 120
    assert list(rotation(None).pair_axes) == [0] * 128


def test_a_number_is_no_list_of_axes():
    for given in (8, np.int64(8), torch.tensor(8), 0, 1.0, [0.5] * 8, [256] * 8, ["0"] * 8):
        with pytest.raises(_lib.InvalidHipState):
            rotation(given)
    for given in ([], [0] * 7, np.zeros(16, np.uint8)):
        with pytest.raises(_lib.InvalidShape):
            rotation(given)
