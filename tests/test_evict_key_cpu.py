"""The keys' range that the eviction's selection starts from (csrc/evict_key.cuh, compiled here for the host)."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "fused_kernels_cutedsl_lib_b200" / "csrc"

# The range of n keys that are dealt to lanes in rounds, with kNoKey behind the last one: joined over lanes,
# warps and CTAs as the kernel does. lanes * rounds >= n.
HOST = r"""
#include <cstring>
#include "evict_key.cuh"
using namespace fk::evict;
extern "C" void key_range(const float* f, int n, int lanes, int rounds, unsigned* out) {
  KeyRange all;
  for (int lane = 0; lane < lanes; ++lane) {
    KeyRange r;
    for (int u = 0; u < rounds; ++u) {
      const int i = u * lanes + lane;
      unsigned bits = 0;
      if (i < n) { const float v = f[i] + 0.f; std::memcpy(&bits, &v, 4); }
      r.add(i < n ? key_of_bits(bits) : kNoKey);
    }
    all.join(r.below, r.greatest);
  }
  out[0] = all.least();
  out[1] = all.greatest;
}
extern "C" unsigned key(float f) { unsigned b; f += 0.f; std::memcpy(&b, &f, 4); return key_of_bits(b); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("evict_key")
    (d / "host.cc").write_text(HOST)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", "host.cc", "-o", "host.so"], cwd=d,
                   check=True)
    lib = ctypes.CDLL(str(d / "host.so"))
    lib.key.argtypes, lib.key.restype = [ctypes.c_float], ctypes.c_uint
    lib.key_range.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 3 + [ctypes.c_void_p]
    return lib


def test_keys_are_in_the_order_of_masses(host):
    values = [-math.inf, -3e38, -1.0, -1e-45, 0.0, 1e-45, 1e-38, 0.5, 1.0, 3e38, math.inf, math.nan]
    keys = [host.key(v) for v in values]
    assert keys == sorted(keys) and len(set(keys)) == len(keys) and keys[0] > 0
    assert host.key(-0.0) == host.key(0.0)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 2277, 4096])
@pytest.mark.parametrize("lanes", [1, 32, 1024, 4096])
def test_places_without_a_candidate_do_not_widen_the_range(host, n, lanes):
    rng = np.random.RandomState(n + lanes)
    for masses in (np.exp(rng.randn(n)), rng.randn(n), np.zeros(n), np.full(n, -np.inf), np.full(n, np.nan)):
        f = masses.astype(np.float32)
        keys = [host.key(float(v)) for v in f]
        for rounds in (-(-n // lanes), -(-n // lanes) + 1):  # lanes with a place to spare, and without any candidate
            out = (ctypes.c_uint * 2)()
            host.key_range(f.ctypes.data, n, lanes, rounds, out)
            assert list(out) == [min(keys), max(keys)]
