"""The caching allocator (csrc/np_devalloc.h) over a host stand-in of the runtime calls it makes (tests/model/devalloc_host.cpp).  (CPU)"""
import os
import subprocess

import pytest

MODEL = os.path.join(os.path.dirname(os.path.abspath(__file__)), "model")


@pytest.fixture(scope="module", autouse=True)
def _program():
    p = subprocess.run(["make", "-C", MODEL, "devalloc_host"], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr[-1500:]


def run(what, **env):
    p = subprocess.run([os.path.join(MODEL, "devalloc_host"), what], capture_output=True, text=True, timeout=60, env=dict(os.environ, **env))
    assert p.returncode == 0, p.stderr[-1500:]
    w = p.stdout.split()
    return {k: int(v) for k, v in zip(w[::2], w[1::2])}


@pytest.mark.parametrize("mb", [None, "0", "1", "no number", "-1", "256", "16384", "17592186044416"])
def test_buffers_taken_and_given_back_again_and_again_make_no_release(mb):
    # 40 sizes: the first pass allocates them, the other 24 find them; whatever the bound is set to, no release reaches the runtime
    got = run("reuse", **({} if mb is None else {"NP_DEVCACHE_MB": mb, "NP_PINCACHE_MB": mb}))
    assert got["frees"] == 0 and got["host_frees"] == 0, got
    assert 0 < got["mallocs"] <= 40 and 0 < got["host_mallocs"] <= 40, got


@pytest.mark.parametrize("what", ["free_beside_destroy", "flush_beside_destroy"])
def test_no_stream_is_used_by_a_release_after_another_thread_destroyed_it(what):
    got = run(what)
    assert got == {"used_destroyed": 0, "left": 4, "gone": 1}, got
