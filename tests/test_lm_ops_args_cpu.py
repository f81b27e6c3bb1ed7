"""Arguments of the language-model operators' host side that need no GPU."""
import numpy as np
import pytest

from vectorcore_b200 import backend as B


@pytest.mark.parametrize("dtype,size", [(np.int8, 1), ("int8", 1), (np.float32, 4), (np.dtype(np.int64), 8), (np.int64, 8)])
def test_borrowed_storages_take_any_spelling_of_a_type(dtype, size):
    s = B.CudaStorage.borrow(1 << 20, 12, dtype)
    assert s.dtype == np.dtype(dtype) and s.nbytes == 12 * size
    assert B._at(s, 12, np.dtype(dtype), "s") == 1 << 20
    with pytest.raises(ValueError, match="s is"):
        B._at(s, 12, np.dtype(np.float64), "s")
