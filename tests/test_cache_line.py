"""How a launch of the attention over a serving cache cuts its work (csrc/cache_line.h, built for the host): every
round of every unit taken once, at sizes whose rounds do not fit 32 bits too. No GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("line") / "cache_line_host.so")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", so,
                           os.path.join(HERE, "cpp", "cache_line_host.cc")])
    return C.CDLL(so)


@pytest.mark.parametrize("unit, units, rounds", [
    (0, 1, 1), (3, 8, 17), (7, 8, 1),
    # the last unit of the most row groups that the sizes allow (2^26 query rows, 128 a group) over 2^20
    # positions, 128 a round: units x rounds = 2^32
    (2 ** 19 - 1, 2 ** 19, 2 ** 13), (2 ** 19 - 2 ** 3, 2 ** 19, 2 ** 13), (2 ** 18, 2 ** 19, 2 ** 20),
    (12345, 2 ** 20, 2 ** 22 - 1)])
def test_a_workgroup_alone_with_its_unit(host, unit, units, rounds):
    out = (C.c_uint32 * 9)()
    assert host.line_whole(C.c_uint32(unit), C.c_uint32(units), C.c_uint32(rounds), out, 3) == 1
    assert list(out[:3]) == [unit, 0, rounds]


@pytest.mark.parametrize("seed", range(20))
def test_every_round_of_a_line_once(host, seed):
    rng = np.random.default_rng(seed)
    entries, units = int(rng.integers(1, 70)), int(rng.integers(1, 30))
    rounds = rng.integers(1, [2, 30, 400][seed % 3], entries).astype(np.uint32)
    total = int(rounds.sum()) * units
    for groups in {1, min(total, 7), min(total, 256), min(total, 512), total}:
        assert host.line_check(entries, C.c_uint32(units), rounds.ctypes.data_as(C.c_void_p), C.c_uint32(groups)) == 0


def test_lines_fit_31_bits(host):
    assert not host.line_too_long(C.c_int64(2047), C.c_int64(2 ** 20))
    assert host.line_too_long(C.c_int64(1024), C.c_int64(2 ** 22))
