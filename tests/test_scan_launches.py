"""The host side of the leaky scan against a runtime that refuses a launch (fake_cudart.cpp): every launch of a call
is checked, so that a call whose kernels did not all start does not return SNN_OK."""
import ctypes as C
import glob
import os
import shutil
import subprocess

import pytest

import snn_b200 as snn

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "pure-snn-language_b200")


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    objects = sorted(glob.glob(os.path.join(PKG, "_build", "scan*.o")))
    if not objects or shutil.which("g++") is None:
        pytest.skip("wants g++ and the objects of the build (pure-snn-language_b200/_build)")
    out = str(tmp_path_factory.mktemp("fake") / "libfake.so")
    cmd = ["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I/usr/local/cuda/include",
           "-I", os.path.join(os.path.dirname(HERE), "include"), "-I", os.path.join(PKG, "csrc"),
           os.path.join(HERE, "fake_cudart.cpp"), *objects, "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    L = C.CDLL(out)
    L.fake_scan.argtypes = [C.c_int, C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_int]
    return L


CHANNEL = snn.SCAN_CHANNEL | snn.SCAN_LOGIT


@pytest.mark.parametrize("flags,b,t,d,grad,launches", [
    (0, 2, 4, 100, 0, 1),             # steps
    (0, 2, 100, 100, 0, 1),           # tiles
    (0, 1, 13000, 40, 0, 3),          # chunks: maps, join, steps
    (CHANNEL, 1, 13000, 40, 0, 3),
    (0, 2, 100, 100, 1, 1),
    (CHANNEL, 2, 100, 100, 1, 2),     # and the channel gate's sum
    (0, 1, 13000, 40, 1, 3),
    (CHANNEL, 1, 13000, 40, 1, 4),
    (CHANNEL | snn.SCAN_RASTER, 1, 13000, 40, 1, 4)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_every_launch_is_checked(fake, kind, flags, b, t, d, grad, launches):
    fake.fake_fail(-1)
    assert fake.fake_scan(kind, flags, b, t, d, grad) == 0 and fake.fake_launches() == launches
    for n in range(launches):
        fake.fake_fail(n)
        assert fake.fake_scan(kind, flags, b, t, d, grad) == 2, n  # SNN_ERR_CUDA
