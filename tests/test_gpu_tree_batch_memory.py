"""Tree passes where the device has no memory for the attention's scratch: the results are the same. The passes run
in a child process whose hipMalloc fails from a size on (native/failing_malloc.cpp)."""

import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def child(shim):
    sys.path.insert(0, ROOT)
    lib = C.CDLL(shim, mode=C.RTLD_GLOBAL)  # before the library, which then finds this hipMalloc first
    lib.malloc_fails_from.argtypes = [C.c_void_p, C.c_size_t]
    lib.malloc_failures.restype = C.c_long
    from taco_amd import hip, synth
    hip.lib()
    from tests.attention_ref import random_parents
    from tests.test_gpu_tree_cache_streams import runtime
    real = C.cast(runtime().hipMalloc, C.c_void_p).value
    lib.malloc_fails_from(real, 0)
    n_ctx, vocab = 2400, 200
    dims = synth.Dims(n_layer=1, n_head=2, d_model=128, d_ff=128, vocab=vocab, n_ctx=n_ctx)
    model = hip.HipModel.load(hip.HipDevice.open(0), synth.build_model(dims, seed=0x7EE4))
    r = np.random.default_rng(4)
    prompt = [(0, int(x)) for x in r.integers(0, vocab - 1, 2200)]
    tree, parents = [(0, int(x)) for x in r.integers(0, vocab - 1, 40)], random_parents(r, 40)
    rows = []
    for fails in (False, True):
        batch = hip.HipBatch(model, 1, 64)
        batch.run_without_readback(prompt)
        print("prompt run", flush=True)
        before = lib.malloc_failures()
        # the tree's own arrays take 2 KiB at most, the scratch 253,440 bytes
        lib.malloc_fails_from(real, 65_536 if fails else 0)
        got = [batch.run_tree_weights(tree, parents)]
        assert (lib.malloc_failures() > before) == fails
        batch.commit_paths({0: [0]})
        got.append(batch.run_weights([(0, 7)]))  # the scratch given up for the tree's is not needed
        lib.malloc_fails_from(real, 0)
        got.append(batch.run_tree_weights(tree, parents))
        got.append(batch.run_weights([(0, 7)]))
        rows.append(got)
        print("passes run", flush=True)
    for a, b in zip(*rows):
        assert a.any() and np.array_equal(a, b)
    print("ok", flush=True)


def test_a_tree_without_memory_for_its_scratch(tmp_path):
    shim = str(tmp_path / "failing_malloc.so")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", shim, os.path.join(HERE, "native", "failing_malloc.cpp")], check=True)
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__), shim], capture_output=True, text=True, timeout=110,
                       cwd=ROOT)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), (r.returncode, r.stdout + r.stderr)


if __name__ == "__main__":
    child(sys.argv[1])
