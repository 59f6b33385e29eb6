"""pack_q4: codes of the 4-bit product's packed format, and what is none."""
import numpy as np
import pytest


@pytest.mark.parametrize("dtype", [np.uint8, np.int8, np.int32, np.uint32, np.int64, np.uint64])
def test_codes_of_any_whole_type(abi, dtype):
    codes = np.arange(35, dtype=dtype).reshape(5, 7) % 16
    words = abi.pack_q4(codes)
    assert words.dtype == np.uint32 and len(words) == 5
    flat = codes.reshape(-1)
    assert [(int(words[i // 8]) >> 4 * (i % 8)) & 15 for i in range(35)] == list(flat)


@pytest.mark.parametrize("codes", [[[0, 16]], [[-1, 3]], [[255, 0]], [[1 << 40, 0]], np.array([[200, -1]], np.int16),
                                   np.array([[1.0, 2.5]]), np.array([[np.nan, 1.0]])])
def test_other_values_are_refused(abi, codes):
    """They would change the codes beside them."""
    with pytest.raises(ValueError, match="codes must be whole numbers from 0 to 15"):
        abi.pack_q4(codes)


def test_no_codes(abi):
    assert len(abi.pack_q4(np.zeros((0, 8), np.uint8))) == 0
