"""GPU: tensors that start inside an element are refused by the language-model
operators before anything is launched."""
import numpy as np
import pytest

from vectorcore_b200 import _abi

pytestmark = pytest.mark.gpu

# the C entry point, its arguments for 4 rows of 16 (f, k, q: device addresses of
# float, int64 and int8 tensors), and which of them are tensors of floats or int64s
CALLS = [
    ("vc_cuda_rms_norm", lambda f, k, q: [f, 16, f, 16, f, 4, 16, 1e-6, f, f, f], (0, 2, 4, 8, 9, 10)),
    ("vc_cuda_rms_norm_backward", lambda f, k, q: [f, f, f, f, f, 4, 16, f, f], (0, 1, 2, 3, 4, 7, 8)),
    ("vc_cuda_rms_norm_backward", lambda f, k, q: [f, f, f, f, f, 0, 16, f, f], (8,)),
    ("vc_cuda_rms_norm_q8", lambda f, k, q: [f, 16, f, 16, f, 4, 16, 1e-6, f, q, 16, f], (0, 2, 4, 8, 11)),
    ("vc_cuda_quantize_q8", lambda f, k, q: [f, 16, 4, 16, q, 16, f], (0, 6)),
    ("vc_cuda_matmul_q8", lambda f, k, q: [q, 16, f, q, 16, f, f, 4, 4, 16, f], (2, 5, 6, 10)),
    ("vc_cuda_matmul_q8", lambda f, k, q: [q, 16, f, q, 16, f, f, 4, 4, 0, f], (2, 5, 6, 10)),
    ("vc_cuda_sample", lambda f, k, q: [f, 16, f, 16, f, k, f, f, 4, 16, k, f], (0, 2, 4, 5, 6, 7, 10, 11)),
]


@pytest.mark.parametrize("name,arguments,tensors", CALLS)
def test_tensors_inside_an_element(backend, name, arguments, tensors):
    f, k, q = backend.allocate(1024), backend.allocate(128, np.int64), backend.allocate(1024, np.int8)
    for which in tensors:
        args = arguments(f.ptr, k.ptr, q.ptr)
        for off in (1, 2, 3, *((4,) if args[which] == k.ptr else ())):
            bad = list(args)
            bad[which] += off
            with pytest.raises(ValueError, match="inside an element"):
                _abi.call(name, *bad)
    backend.synchronize()
