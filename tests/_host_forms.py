"""The C++ forms of the language-model operators (vectorcore::CudaBackend)
built against a stand-in for the host's headers, as a library for ctypes."""
import ctypes
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
FORMS = Path(__file__).resolve().parent / "host_forms"
HOST = ROOT / "vectorcore_b200" / "csrc" / "host"


def build(folder, abi):
    """The forms over `abi`: the CUDA library, or a C source in its place."""
    flags = ["-std=c++20", "-O1", "-Wall", "-Werror", "-fPIC", f"-I{FORMS}", f"-I{ROOT / 'include'}", f"-I{HOST}"]
    objects = []
    for source in (HOST / "cuda_backend.cpp", FORMS / "forms.cpp"):
        objects.append(str(folder / f"{source.stem}.o"))
        subprocess.run(["g++", *flags, "-c", str(source), "-o", objects[-1]], check=True)
    if abi.suffix == ".c":
        objects.append(str(folder / f"{abi.stem}.o"))
        subprocess.run(["gcc", "-O1", "-fPIC", "-c", str(abi), "-o", objects[-1]], check=True)
        abi = None
    out = folder / "libforms.so"
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", *objects, *([] if abi is None else [str(abi)]), "-o", str(out)],
                   check=True)
    return ctypes.CDLL(str(out))


# statuses of the C ABI, as its exceptions come back (vc_cuda.h)
INVALID, OUT_OF_RANGE, OVERFLOW = 1, 2, 3
# of form_refusals, in its order: short storages, products that overflow, other types
REFUSALS = [OUT_OF_RANGE] * 23 + [OVERFLOW] * 2 + [INVALID] * 8


def refusals(lib):
    status = (ctypes.c_int * 100)()
    n = lib.form_refusals(status, 100)
    return list(status)[:n]
