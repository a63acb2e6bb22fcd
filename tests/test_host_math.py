"""The host's sin / cos of the position and RoPE tables (ct2x_host_sin_cos): the installed MKL's own, or the C
library's. No GPU."""
import ctypes as C

import numpy as np
import pytest

import _oracle as O
from ctranslate2_amd import _lib


def host_sin_cos(x):
    s, c = np.empty_like(x), np.empty_like(x)
    _lib.check(_lib.lib().ct2x_host_sin_cos(C.c_int64(len(x)), x.ctypes.data_as(C.c_void_p),
                                            s.ctypes.data_as(C.c_void_p), c.ctypes.data_as(C.c_void_p)))
    return s, c


def backend():
    L = _lib.lib()
    L.ct2x_host_math_backend.restype = C.c_char_p
    return L.ct2x_host_math_backend().decode()


ARGUMENTS = {
    "table": (np.arange(1, 2001, dtype=np.float32)[:, None] *
              np.exp(-np.float32(0.036) * np.arange(256, dtype=np.float32))[None, :]).astype(np.float32).ravel(),
    "random": np.random.default_rng(3).uniform(-10000, 10000, 200_000).astype(np.float32),
    "far": np.random.default_rng(4).uniform(1e4, 1e6, 100_000).astype(np.float32),
    "special": np.array([0.0, -0.0, 1e-30, np.pi, -np.pi, np.pi / 2], np.float32),
}


@pytest.mark.parametrize("kind", ARGUMENTS)
def test_host_sin_cos_is_the_library_s(kind):
    x = ARGUMENTS[kind]
    s, c = host_sin_cos(x)
    if backend() == "mkl-vml":
        assert np.array_equal(s.view(np.uint32), O.vml_sin(x).view(np.uint32))
        assert np.array_equal(c.view(np.uint32), O.vml_cos(x).view(np.uint32))
    else:
        m = C.CDLL("libm.so.6")
        for f, got in ((m.sinf, s), (m.cosf, c)):
            f.restype, f.argtypes = C.c_float, [C.c_float]
            want = np.array([f(float(v)) for v in x[:5000]], np.float32)
            assert np.array_equal(got[:5000].view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("kind", ARGUMENTS)
def test_host_sin_cos_within_an_ulp(kind):
    """Either library is documented to be within one step of the value, which is at most 2^-23 of it."""
    x = ARGUMENTS[kind]
    s, c = host_sin_cos(x)
    for got, want in ((s, np.sin(x.astype(np.float64))), (c, np.cos(x.astype(np.float64)))):
        assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 1e-40)


def test_a_partial_mkl_is_passed_over(tmp_path):
    """libmkl_rt alone, without the libraries that it loads when it is called, ends a process: it is not used."""
    import glob
    import os
    import shutil
    import subprocess
    import sys
    rt = sorted(glob.glob("/opt/conda/lib/libmkl_rt.so*"))
    if not rt:
        pytest.skip("no MKL runtime")
    shutil.copy(rt[0], tmp_path / "libmkl_rt.so.1")
    code = ("import sys; sys.path[:0] = %r; import numpy as np, test_host_math as T; "
            "x = np.array([0.5, 2.0], np.float32); s, c = T.host_sin_cos(x); "
            "assert abs(s - np.sin(x)).max() < 1e-6; print('BACKEND', T.backend())" %
            [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))])
    env = dict(os.environ, CT2X_MKL_PATH=str(tmp_path))
    p = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "BACKEND" in p.stdout, p.stderr[-2000:]
