"""The C ABI surface of libgen9blas_llm.so, checked without a GPU: what include/gen9blas_llm.h declares is exported and
nothing else is; the module's signatures name exactly these functions; without a device every entry point reports
GEN9BLAS_ERR_NO_DEVICE and a text."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.realpath(__file__)))
LIB = os.path.join(ROOT, "gen9-gpu-blas_amd", "libgen9blas_llm.so")


def declared():
    text = open(os.path.join(ROOT, "include", "gen9blas_llm.h")).read()
    return set(re.findall(r"GEN9BLAS_API\s+[\w\s\*]+?\b(gen9blas_\w+)\s*\(", text))


def test_exports_exactly_the_header():
    out = subprocess.run(["nm", "-D", "--defined-only", LIB], capture_output=True, text=True, check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if line.strip()} == declared()


def test_module_signatures():
    import gen9blas
    assert {"gen9blas_" + item.split("=")[0] for item in gen9blas._LLM_SIGNATURES.split()} == declared()
    for f in ("MX4", "mx4_quantize", "mx4_load", "mx4_dequantize", "mx4_gemm", "moe_route", "moe_gemm"):
        assert callable(getattr(gen9blas, f)), f


def test_header_is_c():
    """The header is C: a C compiler takes it alone."""
    r = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-x", "c", "-I" + os.path.join(ROOT, "include"), "-"],
                       input="#include \"gen9blas_llm.h\"\n", text=True, capture_output=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present: the no-device path is not reachable")
def test_no_device_status():
    L = ctypes.CDLL(LIB)
    L.gen9blas_llm_error.restype = ctypes.c_char_p
    L.gen9blas_mx4_create.restype = ctypes.c_void_p
    NO_DEV = -5
    assert L.gen9blas_mx4_create(1, 4, 4) is None
    assert L.gen9blas_llm_last_status() == NO_DEV and L.gen9blas_llm_error()
    f = ctypes.c_float(1)
    p = ctypes.c_void_p(None)
    assert L.gen9blas_mx4_gemm(1, 1, p, 4, p, p, 4) == NO_DEV
    assert L.gen9blas_moe_route(1, 1, 8, p, 8, p, 0, 1, 1, 2, 1, f, p, p) == NO_DEV
    L.gen9blas_mx4_free(p)
