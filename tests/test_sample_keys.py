"""The keys by which the draw orders logits: every number's key is the one next to its neighbour's, both zeros' is the same.
The two functions are taken from the kernel's source and run on the CPU."""
import os
import re
import subprocess

import numpy as np
import pytest

from .conftest import ROOT

SHIM = """
#include <stdint.h>
#include <string.h>
static unsigned __float_as_uint(float x) { unsigned u; memcpy(&u, &x, 4); return u; }
static float __uint_as_float(unsigned u) { float x; memcpy(&x, &u, 4); return x; }
struct type {
%s
%s
};
extern "C" void keys(const float *x, unsigned *k, long n) { for (long i = 0; i < n; i++) k[i] = type::key(x[i]); }
extern "C" void values(const unsigned *k, float *x, long n) { for (long i = 0; i < n; i++) x[i] = type::value(k[i]); }
"""


@pytest.fixture(scope="module", params=["float", "__nv_bfloat16"])
def order(request, tmp_path_factory):
    """(bf16, keys of floats, numbers of keys)"""
    import ctypes
    text = open(os.path.join(ROOT, "irptx_b200", "csrc", "kernels", "sample.cu")).read()
    at = text.index(f"template <> struct smp_type<{request.param}> {{")
    struct = text[at:text.index("\n};\n", at)]
    key = re.search(r"__device__ static __forceinline__ unsigned key\(float x\)\n    \{.*?\n    \}", struct, re.S).group(0)
    value = re.search(r"__device__ static __forceinline__ float value\(unsigned k\)[^\n]*", struct).group(0)
    where = tmp_path_factory.mktemp("keys")
    src = SHIM % tuple(s.replace("__device__ static __forceinline__", "static") for s in (key, value))
    (where / "keys.cpp").write_text(src)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(where / "keys.so"), str(where / "keys.cpp")], check=True)
    lib = ctypes.CDLL(str(where / "keys.so"))

    def call(f, a, to):
        out = np.empty(len(a), to)
        f(a.ctypes.data_as(ctypes.c_void_p), out.ctypes.data_as(ctypes.c_void_p), ctypes.c_long(len(a)))
        return out
    return (request.param != "float", lambda x: call(lib.keys, np.ascontiguousarray(x, np.float32), np.uint32),
            lambda k: call(lib.values, np.ascontiguousarray(k, np.uint32), np.float32))


def numbers(bf16, at, count):
    """`count` numbers next to each other, ascending, from `at` on; one zero."""
    step = 16 if bf16 else 0
    bits = int(np.float32(at).view(np.uint32)) >> step
    top = 1 << (31 - step)
    place = top - (bits - top) if bits >= top else top + bits            # 0 at the middle
    out = []
    for p in range(place, place + count):
        out.append((top + (top - p) if p < top else p - top) << step)
    return np.array(out, np.uint32).view(np.float32)


STARTS = [-np.inf, -3e38, -1e30, -2.0, -1.0, -1.1754944e-38, -2e-41, -1.4e-45, 0.0, 1.1e-38, 1.0, 1.5]


@pytest.mark.parametrize("start", STARTS)
def test_neighbours_have_neighbouring_keys(order, start):
    bf16, key, value = order
    x = numbers(bf16, start, 100 if bf16 and start in (1.1e-38,) else 400 if not np.isinf(start) else 300)
    assert (np.diff(x.astype(np.float64)[1 if np.isinf(start) else 0:]) > 0).all()
    k = key(x)
    assert (np.diff(k.astype(np.int64)) == 1).all()
    assert (value(k) == x).all()


def test_both_zeros_are_one_number(order):
    _, key, value = order
    k = key(np.array([0.0, -0.0], np.float32))
    assert k[0] == k[1] and value(k[:1])[0] == 0.0


def test_above_the_key_below_is_all_of_a_number(order):
    """What stands for "all that are equal to x" is "above the number of the key below"."""
    bf16, key, value = order
    x = np.concatenate([numbers(bf16, s, 200) for s in STARTS if np.isfinite(s)] + [np.array([-0.0], np.float32)])
    assert (x > value(key(x) - 1)).all()


def test_every_bf16_key(order):
    bf16, key, value = order
    if not bf16:
        pytest.skip("2^32 of them")
    lowest, highest = key(np.array([-np.inf, np.inf], np.float32))
    k = np.arange(lowest, highest + 1, dtype=np.uint32)
    x = value(k)
    assert (key(x) == k).all() and (x[1:] > x[:-1]).all()
