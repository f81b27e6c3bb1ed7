"""The C++ forms of the language-model operators refuse storages that are too
short or of another type, before the device sees them. Without a GPU: the C
ABI under them only counts."""
import ctypes

import _host_forms as H


def test_short_storages_and_other_types_are_refused(tmp_path):
    lib = H.build(tmp_path, H.FORMS / "fake_abi.c")
    assert H.refusals(lib) == H.REFUSALS
    assert ctypes.c_int.in_dll(lib, "operators_reached").value == 0
