"""What the tests' own comparison has to catch."""
import pytest
import torch

from tests.helpers import assert_within


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 1.26])
def test_one_wrong_element_fails(bad):
    ref = torch.ones(3, 4, dtype=torch.float64)
    tol = torch.full_like(ref, 0.25)
    got = ref.float()
    got[1, 2] = 1.25
    assert_within(got, ref, tol)
    got[1, 2] = bad
    with pytest.raises(AssertionError):
        assert_within(got, ref, tol)
