"""Host arrays of slots, positions, lengths and parents: no value is changed on
its way to the library."""
import numpy as np
import pytest

from leap_b200.attention import _ints


@pytest.mark.parametrize("bad", [np.array([2**32]), np.array([0, -2**31 - 1]), [2**31], np.array([2**63], np.uint64),
                                 np.array([1.0]), [0.7], np.array([True]), np.array(["1"]), np.array([1 + 0j])])
def test_what_is_not_a_32_bit_whole_number_is_refused(bad):
    with pytest.raises(ValueError, match="slots"):
        _ints(bad, "slots")


@pytest.mark.parametrize("good", [[0, 5, -1], (3,), np.array([2**31 - 1, -2**31]), np.array([7, 8], np.uint8), [],
                                  np.array([], np.float64), np.arange(10)[::2], np.arange(10, dtype=np.int32)[::3]])
def test_whole_numbers_arrive(good):
    a = _ints(good, "slots")
    assert a.dtype == np.int32 and a.flags.c_contiguous
    assert a.tolist() == [int(x) for x in good]


def test_torch_tensors_arrive():
    torch = pytest.importorskip("torch")
    assert _ints(torch.tensor([4, 2]), "slots").tolist() == [4, 2]
    with pytest.raises(ValueError):
        _ints(torch.tensor([2**33]), "slots")
