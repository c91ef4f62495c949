"""The correctly rounded functions that the oracle links where the reference
tree is not present: built on their own, and equal to exact arithmetic rounded
once (integers and fractions for powers, decimal for exp and log, the integer
square root for pow(x, 0.5))."""
import ctypes
import math
import os
import random
import shutil
import struct
import subprocess
from decimal import Decimal, localcontext
from fractions import Fraction

import pytest

ORACLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle")


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """The oracle built in a directory of its own, without a reference tree."""
    at = tmp_path_factory.mktemp("oracle")
    for name in os.listdir(ORACLE):
        if name == "Makefile" or name.endswith((".c", ".h")):
            shutil.copy(os.path.join(ORACLE, name), at)
    subprocess.run(["make", "-s", "-C", str(at), "REFERENCE="], check=True)
    return at


@pytest.fixture(scope="module")
def fn(built):
    L = ctypes.CDLL(str(built / "librounded_math.so"))

    def get(name, n=1, real=ctypes.c_double):
        f = getattr(L, "chelis_crmath_ffi_" + name)
        f.restype, f.argtypes = real, [real] * n
        return f
    return get


def _f32(fraction):
    """A positive fraction in the normal range to the nearest binary32."""
    e = math.frexp(float(fraction))[1]
    step = Fraction(2) ** (e - 24)
    return float(round(fraction / step) * step)


def test_the_oracle_builds_and_loads_without_the_reference_tree(built):
    L = ctypes.CDLL(str(built / "liborc.so"))
    L.orc_expf.restype, L.orc_expf.argtypes = ctypes.c_float, [ctypes.c_float]
    assert L.orc_expf(0.0) == 1.0


def test_powers_of_few_bits(fn):
    """Squares to fifth powers, many of them in the middle of two numbers."""
    rng = random.Random(1)
    pow64, pow32 = fn("pow", 2), fn("powf", 2, ctypes.c_float)
    for _ in range(20000):
        x, n = float(rng.getrandbits(rng.choice([11, 14, 18, 27, 28, 53])) | 1), rng.choice([2, 3, 4, 5])
        assert pow64(x, n) == float(Fraction(x) ** n)
    for _ in range(20000):
        x, n = float(rng.getrandbits(rng.choice([9, 13, 24])) | 1), rng.choice([2, 3])
        assert pow32(x, n) == _f32(Fraction(x) ** n)


def test_square_roots_by_pow(fn):
    rng = random.Random(2)
    pow64 = fn("pow", 2)
    for x in [1 - 2.0 ** -53, 1 + 2.0 ** -52, 1.7976931348623157e308, 5e-324] + \
             [rng.random() * 2.0 ** rng.randint(-500, 500) for _ in range(20000)]:
        assert pow64(x, 0.5) == math.sqrt(x)


def test_exp_and_log(fn):
    rng = random.Random(3)
    exp64, log64 = fn("exp"), fn("log")
    exp32, log32 = fn("expf", real=ctypes.c_float), fn("logf", real=ctypes.c_float)
    with localcontext() as ctx:
        ctx.prec = 60
        for _ in range(2000):
            x = struct.unpack("f", struct.pack("f", rng.uniform(-80, 80)))[0]
            want = Decimal(x).exp()
            assert exp64(x) == float(want) and exp32(x) == _f32(Fraction(want))
            x = struct.unpack("f", struct.pack("f", (1.0 + rng.random()) * 2.0 ** rng.randint(1, 100)))[0]
            want = Decimal(x).ln()
            assert log64(x) == float(want) and log32(x) == _f32(Fraction(want))


def test_special_values(fn):
    inf, nan = math.inf, math.nan

    def bits(v):
        return struct.pack("d", v)
    quiet = struct.pack("Q", 0x7ff8000000000000)
    for name in ("exp", "log", "sin", "cos", "tan", "atan", "tanh", "erf", "erfc"):
        assert bits(fn(name)(-nan)) == quiet
    assert bits(fn("log")(-1.0)) == quiet and bits(fn("sin")(inf)) == quiet
    assert fn("exp")(-inf) == 0.0 and fn("exp")(inf) == inf and fn("log")(0.0) == -inf
    for name in ("sin", "tan", "atan", "tanh", "erf"):
        assert bits(fn(name)(-0.0)) == bits(-0.0)
        assert fn(name)(5e-324) == 5e-324
    assert fn("pow", 2)(nan, 0.0) == 1.0 and fn("pow", 2)(-2.0, 3.0) == -8.0
    assert bits(fn("pow", 2)(-2.0, 0.5)) == quiet
