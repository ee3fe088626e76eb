"""CPU tests of the sizes that attention over the 4-bit cache asks for.  A handle is faked as zeroed memory: a machine of no SMs."""
import ctypes as C
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS = [1, 64, 65, 127, 128, 255, 256, 300, 70000]

# in a process of its own: a division by zero on the host would end this one
CHILD = """
import ctypes as C
from oxicuda_b200 import _ffi
lib, fake, n = _ffi.load(), C.create_string_buffer(4096), C.c_size_t(0)
cache = _ffi.kv4_cache(0x1000, 0x2000, 0x3000, 0x4000, 8, 16, 2, 128, 64)
for tokens in %r:
    for most in (0, 1, 20, tokens):
        for width in (0, 4, 4096):
            n.value = 7
            batch = _ffi.kv4_batch(0x5000, width, 0x6000, 0x7000, %d, tokens)
            assert lib.oxq_kv4_attention_workspace_bytes(fake, cache, batch, 2, most, C.byref(n)) == 0
            if %d == 0 or tokens == 0:
                assert n.value == 0
print("done")
"""


@pytest.mark.parametrize("seqs", [0, 1, 3])
def test_workspace_of_any_number_of_sequences(seqs):
    """A call without sequences (or without tokens) needs no workspace, however many query rows it has."""
    from oxicuda_b200 import _build
    _build.build()
    r = subprocess.run([sys.executable, "-c", CHILD % ([0] + ROWS, seqs, seqs)], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stderr[-2000:])


READ_ONLY = re.compile(r"__ldg\s*\(|\bld16\s*\(|\bld16_stream\s*\(|\.nc\b|__restrict__")


@pytest.mark.parametrize("name", ["oxq_kv4.cu", "oxq_kv4.cuh", "oxq_kv4_attn.cu", "oxq_kv4_attn.cuh", "oxq_kv4_tiles.cu", "oxq_resnorm.cu"])
def test_nothing_that_kernels_write_is_read_through_the_read_only_path(name):
    """A kernel that starts early is resident while the one before it writes the pool, the queries or the residual; the read-only path is for data
    that nobody writes then.  The norm's weights are."""
    with open(os.path.join(ROOT, "oxicuda_b200", "csrc", name)) as f:
        lines = [line.split("//")[0] for line in f]
    found = [line.strip() for line in lines if READ_ONLY.search(line)]
    assert all("reinterpret_cast<const float4*>(p)" in line and name == "oxq_resnorm.cu" for line in found), found


@pytest.mark.parametrize("apart,dtype,status", [(0, 1, 15), (16, 1, 15), (3 * 2 * 128 * 2 - 16, 1, 15), (3 * 2 * 128 * 2, 1, 13), (3 * 2 * 128 * 2, 0, 15),
                                                (3 * 2 * 128 * 4, 0, 13), (3 * 2 * 128 * 2, 2, 13)])
def test_read_into_outputs_that_overlap(apart, dtype, status):
    """13: all is right but for the machine, which has compute capability 0.0."""
    from oxicuda_b200 import _build, _ffi
    _build.build()
    lib, fake = _ffi.load(), C.create_string_buffer(4096)
    cache = _ffi.kv4_cache(0x1000, 0x2000, 0x3000, 0x4000, 8, 16, 2, 128, 64)
    batch = _ffi.kv4_batch(0x5000, 4, 0x6000, 0x7000, 2, 3)
    for k, v in ((0x100000, 0x100000 + apart), (0x100000 + apart, 0x100000)):
        assert lib.oxq_kv4_read(fake, cache, batch, k, v, dtype) == status


def test_attention_in_place():
    """An item's rows are read by every CTA that has a part of its keys, so its output cannot take their place."""
    from oxicuda_b200 import _build, _ffi
    _build.build()
    lib, fake = _ffi.load(), C.create_string_buffer(4096)
    cache = _ffi.kv4_cache(0x1000, 0x2000, 0x3000, 0x4000, 8, 16, 2, 128, 64)
    batch = _ffi.kv4_batch(0x5000, 4, 0x6000, 0x7000, 2, 3)
    for out, status in ((0x8000, 15), (0x18000, 13)):
        args = _ffi.kv4_attention_args(0x8000, 1024, 128, out, 1024, 128, 0, 8, 0, 0, 0.1, 1, 1)
        assert lib.oxq_kv4_attention(fake, cache, batch, args, 0x10000, 1 << 30) == status
