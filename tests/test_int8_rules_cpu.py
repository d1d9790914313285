"""Where the 8-bit operators send a call, compiled for the host and checked at the sizes where each form was measured. 148 SMs."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    work = tmp_path_factory.mktemp("rules")
    src, lib = work / "rules.cpp", work / "rules.so"
    src.write_text('#include "rules.h"\nextern "C" bool gemm_i8_rowdot(long long m, long long n, long long k, int x16) {'
                   " return b200ait::gemm_i8_rowdot(m, n, k, x16 != 0); }\n")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(ROOT, "aitemplate_b200", "csrc"),
                    str(src), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))
    lib.gemm_i8_rowdot.restype = ctypes.c_bool
    return lambda m, n, k, x16: lib.gemm_i8_rowdot(*map(ctypes.c_longlong, (m, n, k)), int(x16))


@pytest.mark.parametrize("m,n,k,of_8,of_16", [
    (0, 64, 64, False, False), (1, 1, 1, True, True), (1, 8192, 8192, True, True), (1, 8, 131071, True, True), (2, 2048, 2048, True, True),
    (2, 8192, 8192, False, True), (2, 4096, 512, False, True), (2, 100, 64, True, True), (2, 8, 131071, False, False), (3, 1024, 1024, False, True),
    (4, 2048, 2048, False, True), (4, 4096, 4096, False, False), (5, 64, 64, False, False),
])
def test_few_rows(rules, m, n, k, of_8, of_16):
    assert rules(m, n, k, False) == of_8 and rules(m, n, k, True) == of_16
