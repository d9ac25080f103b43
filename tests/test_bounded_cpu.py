"""The bounded-cache calls without a device: argument checks that need no handle, and the plain eviction list against its
definition."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from bruce_engine_b200 import capi
from tests import bounded_ref as R


def test_null_handles_are_refused():
    lib = capi.load()
    n, sk, pg = C.c_size_t(), capi.CSinks(None, None, 4, 0), capi.CPages(None, None, None, 1, 1, 1, 128)
    buf = (C.c_uint8 * 64)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 16
    assert lib.battn_sinks_bytes(None, 128, C.byref(n)) == capi.ERR_ARG
    assert lib.battn_track_workspace_bytes(None, 1, 1, 1, C.byref(n)) == capi.ERR_ARG
    assert lib.battn_evict_workspace_bytes(None, 1, C.byref(n)) == capi.ERR_ARG
    assert lib.battn_sinks_store(None, p, p, C.byref(sk), p, None, None, 1, 1, None) == capi.ERR_ARG
    assert lib.battn_attend_sinks(None, p, p, p, p, C.byref(sk), p, None, None, p, 1, 1, 0, None) == capi.ERR_ARG
    assert lib.battn_attend_track(None, p, p, p, p, p, p, p, None, None, p, 64, 1, 1, None) == capi.ERR_ARG
    assert lib.battn_evict(None, p, p, p, p, p, p, None, None, None, p, 4, 0, 0, 1, None) == capi.ERR_ARG
    # a page descriptor is checked before the handle
    assert lib.battn_attend_sinks_paged(None, p, p, C.byref(pg), C.byref(sk), p, None, None, p, 1, 1, None) == capi.ERR_ARG
    assert lib.battn_attend_track_paged(None, p, p, p, p, C.byref(pg), p, None, None, p, 64, 1, 1, None) == capi.ERR_ARG
    assert lib.battn_evict_paged(None, C.byref(pg), p, p, p, p, None, None, None, p, 4, 0, 0, 1, None) == capi.ERR_ARG


@pytest.mark.parametrize("n,budget,n_sink,n_recent", [(1, 1, 0, 0), (9, 5, 2, 2), (40, 17, 0, 0), (40, 17, 17, 0), (40, 17, 0, 17),
                                                      (40, 39, 3, 5), (8, 20, 3, 3)])
def test_the_plain_list_is_the_definition(n, budget, n_sink, n_recent):
    rng = np.random.default_rng(n + budget)
    for _ in range(20):
        s = rng.choice([0.0, -0.0, 1.0, 2.0, np.nan, np.inf, -np.inf], size=n).astype(np.float32)
        got = R.evict_list(s, budget, n_sink, n_recent)
        assert len(got) == min(n, budget) and (np.diff(got) > 0).all()
        if n <= budget:
            continue
        held = set(got.tolist())
        assert set(range(n_sink)) <= held and set(range(n - n_recent, n)) <= held
        worth = lambda i: (not np.isnan(s[i]), 0.0 if np.isnan(s[i]) else float(s[i]) + 0.0, -i)      # NaN lowest, ties to the lower
        mid = range(n_sink, n - n_recent)
        left = [worth(i) for i in mid if i not in held]
        kept = [worth(i) for i in mid if i in held]
        assert not kept or not left or min(kept) > max(left)


def test_pages_of_bounded_rows_return_to_the_pool(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "bounded_pages_test")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-pthread", "-Wall", "-Wextra", "-I", os.path.join(root, "include"),
                        os.path.join(root, "tests", "host", "bounded_pages_test.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
