"""Which kernels the GPU tests of the experts in 8-bit blocks are on, by the rules of csrc/launch_rules.h."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

import test_gpu_fp8_many_rows as M
from piper_amd import _lib

CUS = 256
SOURCE = """
#include "launch_rules.h"
using namespace pk_rules;
extern "C" {
int exact(int short_sums, int64_t A, int64_t E) { return fp8_exact(short_sums != 0, A, E); }
int narrow(int64_t A, int64_t E, int64_t N) { return fp8_narrow(A, E, N); }
int few(int64_t A, int64_t E) { return fp8_few_rows(A, E); }
int stream_up(int64_t A, int64_t E, int64_t I) { return fp8_stream_up(A, E, I); }
int down_tiles(int64_t A, int64_t E, int64_t H) { return fp8_down_tiles(A, E, H); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    csrc = Path(_lib.__file__).resolve().parent / "csrc"
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{csrc}", str(d / "rules.cpp"), "-o", str(d / "rules.so")], check=True,
                   timeout=120)
    lib, i64 = ctypes.CDLL(str(d / "rules.so")), ctypes.c_int64
    lib.exact.argtypes = [ctypes.c_int, i64, i64]
    lib.few.argtypes = [i64, i64]
    for f in (lib.narrow, lib.stream_up, lib.down_tiles):
        f.argtypes = [i64, i64, i64]
    return lib


def _units(counts, N):
    return sum(-(-c // 128) for c in counts) * -(-N // 256)


def test_sums_are_short_only_where_they_are_asked_for(rules):
    for A, E in ((1, 1), (128, 1), (129, 1), (5120, 128), (5121, 128), (65536, 128), (2 ** 31 - 1, 4)):
        assert rules.exact(0, A, E) == 1
        assert rules.exact(1, A, E) == (A <= max(128, 40 * E))


def test_the_kernels_of_real_sizes_are_tested(rules):
    second = {"down": 0, "d_h": 0}
    for E, H, I, counts, spare in M.KERNELS.values():
        A = sum(counts) + spare
        assert not rules.few(A, E) and not rules.exact(1, A, E)
        for what, N in (("down", H), ("d_h", I)):
            if not rules.narrow(A, E, N):
                second[what] += _units(counts, N) > CUS      # a workgroup has more than one unit
    assert second == {"down": 4, "d_h": 4}
    # and the narrow ones
    assert rules.narrow(sum(M.KERNELS["4096 x 384"][3]), 8, 384) and rules.narrow(sum(M.KERNELS["384 x 4096"][3]), 8, 384)
    # the benchmark's widths run wide units and decoded values
    for tokens in (1777, 4096, 8192):
        assert not rules.narrow(tokens * 8, 128, 2048) and not rules.narrow(tokens * 8, 128, 768) and rules.exact(0, tokens * 8, 128)


def test_the_variants_for_few_rows_are_tested(rules):
    for E, H, I, A in M.STREAMED:
        assert rules.few(A, E) and rules.stream_up(A, E, I) and rules.down_tiles(A, E, H) == 4
        assert -(-H // 128) > 4 and 4 * -(-I // 128) > 6
    assert not rules.stream_up(8, 128, 768) and rules.down_tiles(8, 128, 2048) == 1
