"""CPU: calls that the attention's entry points have to refuse because no kernel can answer them as the documentation says."""
import pytest

from dagnet_amd._capi import DagnetHipError
from dagnet_amd.attention import RotaryAxes, SceneLayout


@pytest.mark.parametrize("q,k", [([0, 1], [0, 2 ** 24 + 1]), ([0, 3, 2 ** 24 + 4], [0, 5, 6])])
def test_places_that_are_no_fp32_numbers(q, k):
    """Place 2^24 + 1 rounds to its neighbour: the distance of two rows side by side would be 0 or 2."""
    with pytest.raises(DagnetHipError, match="2\\^24"):
        SceneLayout(q, k).places(0)


def test_the_last_place_that_is():
    lay = SceneLayout([0, 1], [0, 2 ** 24])
    assert not lay.far and lay._at.max() == 2 ** 24 - 1 == lay._k_at.max()


@pytest.mark.parametrize("theta", [(100.0, 10.0, 5.0), (100.0,), [[100.0, 10.0]], ()])
def test_theta_of_another_number_of_axes(theta):
    with pytest.raises(DagnetHipError, match="one per axis"):
        RotaryAxes(16, (4, 4), theta=theta)
    assert RotaryAxes(16, (8,), theta=100.0).freq[0] == RotaryAxes(16, (8,), theta=[100.0]).freq[0] == 1.0
