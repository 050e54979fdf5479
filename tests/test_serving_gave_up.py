"""A call of the token-by-token operators that gave up is heard of by whoever reads a result, once, and its counters are zero in front of the next call.  On the CPU:
the kernels do nothing there (tests/cabi/fake_cudart.c), and the test sets the word that one of them would have set."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA_INCLUDE = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")

DRIVER = r"""
import ctypes as C
import os
import sys
import numpy as np
import zklm_compile_b200 as zk
from zklm_compile_b200 import _lib, serving as zs

fake = C.CDLL(None)
fake.fake_unordered.restype, fake.fake_unordered.argtypes = C.c_long, [C.c_void_p]
ctx = zk.Context(0)
word = C.POINTER(C.c_int).in_dll(fake, "gave_up_word")
z = lambda n: ctx.upload(np.zeros(n, np.uint32))
C.c_size_t.in_dll(fake, "serving_counters").value = 768
cache, q, out = zs.KvCache(ctx, 4, 2, 16, 4), z(64), z(64)
attend = lambda: zs.paged_attention(cache, q, z(2), 1, 2, z(1), 4, z(65536), out, z(1))
attend()
counters = C.POINTER(C.c_uint32).in_dll(fake, "counter_words")
read = {"sync": ctx.sync, "download": out.download}
first, second = read[sys.argv[1]], read[sys.argv[2]]
for _ in range(2):
    first()
    word[0] = 1
    counters[3], counters[148] = 2, 2 << 16
    try:
        first()
        raise SystemExit("a call that gave up was not reported")
    except zk.ZkbError as e:
        assert e.code == 8 and "not valid" in str(e), e
    assert not any(counters[i] for i in range(192))
    assert fake.fake_unordered(ctx.stream) == 0, "the counters are cleared behind the next call's back"
    second()
    first()
    attend()
sys.stdout.flush()
os._exit(0)
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    libs = []
    for name in ("fake_serving", "fake_cudart"):
        libs.append(str(d / f"lib{name}.so"))
        subprocess.run(["gcc", "-std=gnu11", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CUDA_INCLUDE, os.path.join(ROOT, "tests", "cabi", name + ".c"), "-o", libs[-1], "-ldl"],
                       check=True)
    return ":".join(libs)


@pytest.mark.parametrize("first,second", [("sync", "download"), ("download", "sync")])
def test_reported_once_and_cleared(runtime, first, second):
    r = subprocess.run([sys.executable, "-c", DRIVER, first, second], cwd=ROOT, env=dict(os.environ, LD_PRELOAD=runtime, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
