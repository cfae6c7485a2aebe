"""HIP calls that fail, or are counted: a small library in front of the HIP
runtime's own functions, in a process of its own. The failures are returned by it
on the host; nothing reaches the GPU in their place."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SHIM = r"""
#include <dlfcn.h>
#include <stddef.h>

static void *hip;
int shim_fail_memset, shim_memsets, shim_host_allocs;

int shim_open(const char *path) { return (hip = dlopen(path, RTLD_NOW)) != NULL; }

int hipMemsetAsync(void *p, int v, size_t n, void *s) {
    ++shim_memsets;
    if (shim_fail_memset) return 1;  /* hipErrorInvalidValue */
    return ((int (*)(void *, int, size_t, void *))dlsym(hip, "hipMemsetAsync"))(p, v, n, s);
}

int hipHostMalloc(void **p, size_t n, unsigned flags) {
    ++shim_host_allocs;
    return ((int (*)(void **, size_t, unsigned))dlsym(hip, "hipHostMalloc"))(p, n, flags);
}
"""

START = r"""
import ctypes, sys
import numpy as np
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from cheetah_amd import configs, hip, synth
hip.lib()
runtime = next(l.split()[-1] for l in open("/proc/self/maps") if "libamdhip64" in l)
assert shim.shim_open(runtime.encode())
fail, memsets, host_allocs = (ctypes.c_int.in_dll(shim, "shim_" + n) for n in ("fail_memset", "memsets", "host_allocs"))
hip.init(0)
shape = configs.TINY_LLAMA.replace(vocab_size=9001)  # rows of several segments
model = hip.HipForward(shape, synth.make_weights(shape), kv_capacity=256, max_chunk_rows=64)
text = synth.make_tokens(shape.vocab_size, 30, seed=7)
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    where = tmp_path_factory.mktemp("shim")
    (where / "shim.c").write_text(SHIM)
    out = where / "libshim.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(out), str(where / "shim.c"), "-ldl"], check=True)
    return str(out)


def run(shim, body):
    # The persistent decode kernel is launched cooperatively, which one process may
    # at a time: the tests' own, once it has.
    done = subprocess.run([sys.executable, "-c", START + body, shim], cwd=ROOT, capture_output=True, text=True, timeout=100,
                          env={**os.environ, "CHEETAH_HIP_FUSED": "0"})
    assert done.returncode == 0, done.stdout + done.stderr
    assert done.stdout.endswith("done\n")


def test_a_workspace_that_was_not_cleared_is_not_used(shim):
    """The counts of a scored chunk's segments: a call whose clearing fails says
    so, and the next one clears them before it uses them."""
    run(shim, r"""
want = model.clone().forward_logprobs(text, 0, targets=text, top=3)
fail.value = 1
for _ in range(2):
    before = memsets.value
    try:
        model.forward_logprobs(text, 0, targets=text, top=3)
        raise SystemExit("no error")
    except hip.HipError:
        pass
    assert memsets.value > before and model.kv_len() == 0
fail.value = 0
before = memsets.value
got = model.forward_logprobs(text, 0, targets=text, top=3)
assert memsets.value == before + 1
assert all(a.tobytes() == b.tobytes() for a, b in zip(got, want))
before = memsets.value
model.clear_cache()
assert all(a.tobytes() == b.tobytes() for a, b in zip(model.forward_logprobs(text, 0, targets=text, top=3), want))
assert memsets.value == before
print("done")
""")


def test_an_op_level_workspace_that_was_not_cleared_is_not_used(shim):
    run(shim, r"""
x = np.random.default_rng(1).standard_normal((3, 30000)).astype(np.float32)
fail.value = 1
try:
    hip.logprobs(x, [1, 2, 3], 5)
    raise SystemExit("no error")
except hip.HipError:
    pass
fail.value = 0
before = memsets.value
a = hip.logprobs(x, [1, 2, 3], 5)
assert memsets.value == before + 1
b = hip.logprobs(x, [1, 2, 3], 5)
assert memsets.value == before + 1
assert all(p.tobytes() == q.tobytes() for p, q in zip(a, b))
print("done")
""")


def test_a_clone_takes_no_buffers_of_trees(shim):
    """They come with its first tree; a clone costs what it did without them:
    pinned memory for its words, its tokens and its logits."""
    run(shim, r"""
before = host_allocs.value
g = model.clone()
assert host_allocs.value == before + 3
first = g.forward_greedy(text, 0)
g.decode_greedy(first, 30, 4)
g.forward_logprobs(text[:2], 34)
assert host_allocs.value == before + 3
a = g.forward_tree([5, 6, 7], [-1, 0, 0], 36)
assert host_allocs.value == before + 4
assert g.forward_tree([5, 6, 7], [-1, 0, 0], 36).tolist() == a.tolist()
g.commit_tree([0, 2])
g.verify_tree([3, 4], [-1, 0], 38)
assert host_allocs.value == before + 4
print("done")
""")
