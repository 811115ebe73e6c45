"""LDS of attention kernels goes by the bias's reach and the query heads of a key head, from call to call: no
launch may want more of it than was asked for before. Without a GPU: the entries run in a process of their own
whose HIP calls are answered by a few lines of C that compare what is asked for and what is launched."""

from __future__ import annotations

import ctypes
import json
import shutil
import subprocess
import sys

import pytest

HIP = r"""
#include <stddef.h>
typedef struct { unsigned x, y, z; } dim3;
static struct { const void* f; size_t asked; } known[4096];
static int count;
static dim3 grid_, block_;
static size_t lds_;
static void* stream_;
int launches, large, over;
size_t most;

int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int what, int d) { *v = 256; return 0; }
int hipGetLastError(void) { return 0; }
int hipFuncSetAttribute(const void* f, int what, int value) {
  int i = 0;
  while (i < count && known[i].f != f) ++i;
  if (i == count) known[count++].f = f;
  known[i].asked = value;
  return value > 160 * 1024;
}
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, void* s) { grid_ = g, block_ = b, lds_ = lds, stream_ = s; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, void** s) { *g = grid_, *b = block_, *lds = lds_, *s = stream_; return 0; }
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t lds, void* s) {
  size_t asked = 65536;
  for (int i = 0; i < count; ++i)
    if (known[i].f == f && known[i].asked > asked) asked = known[i].asked;
  ++launches, large += lds > 65536, over += lds > asked;
  if (lds > most) most = lds;
  return 0;
}
"""

CHILD = r"""
import ctypes, json, sys
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
for name, args in json.load(sys.stdin):
    held = [ctypes.create_string_buffer(bytes.fromhex(a), len(a) // 2) if isinstance(a, str) else None for a in args]
    rc = getattr(lib, name)(*[ctypes.c_void_p(a) if h is None else h for a, h in zip(args, held)])
    lib.hi3d_last_error.restype = ctypes.c_char_p
    assert rc == 0, (name, rc, lib.hi3d_last_error())
print(json.dumps({n: ctypes.c_int.in_dll(hip, n).value for n in ("launches", "large", "over")} |
                 {"most": ctypes.c_size_t.in_dll(hip, "most").value}))
"""


def _desc(attention, dim, heads, key_heads, dtype, length):
    d = attention._Desc()
    d.q, d.k, d.v = 4096, 8192, 12288
    q, k = heads * dim, key_heads * dim
    d.strides[:] = [length * q, q, dim, length * k, k, dim, length * k, k, dim]
    d.total_q = d.total_k = 2 * length
    d.batch, d.len_q, d.len_k = 2, length, length
    d.heads_q, d.heads_k, d.dim, d.dtype, d.causal, d.scale = heads, key_heads, dim, dtype, 1, 0.125
    return d


@pytest.mark.parametrize("order", [(0, 30, 300, 1024), (1024, 300, 30, 0)])
def test_no_launch_wants_more_lds_than_was_asked_for(tmp_path, order):
    from hi3d_amd import _lib, attention

    compiler = shutil.which("gcc") or shutil.which("g++")
    if compiler is None:
        pytest.skip("no C compiler")
    source, shim = tmp_path / "hip.c", tmp_path / "hip.so"
    source.write_text(HIP)
    subprocess.run([compiler, "-x", "c", "-shared", "-fPIC", "-w", "-o", str(shim), str(source)], check=True)
    room, at = 1 << 40, 4096  # addresses that nothing reads
    calls = []
    for far in order:
        for dim in (32, 64, 96, 128):
            for dtype in (1, 2):
                for heads, key_heads in ((32, 8), (16, 16)):
                    for length in (1, 40, 100, 440, 9000):
                        d = bytes(_desc(attention, dim, heads, key_heads, dtype, length)).hex()
                        for cap in (0.0, 30.0):
                            t = bytes(attention._TermsDesc(None, at, at, None, 1, 4, far, cap)).hex()
                            s = bytes(attention._SharedDesc(at, at, None, (key_heads * dim, dim, key_heads * dim, dim), 500)).hex()
                            calls.append(("hi3d_attention_terms_forward", (d, t, at, None, at, at, room, None)))
                            calls.append(("hi3d_attention_terms_backward", (d, t, at, None, at, at, None, at, at, at, at, at, room, None)))
                            calls.append(("hi3d_attention_shared_forward", (d, t, s, at, at, at, room, None)))
    out = subprocess.run([sys.executable, "-c", CHILD, str(shim), str(_lib.LIB_PATH)], input=json.dumps(calls), capture_output=True,
                         text=True)
    assert out.returncode == 0, out.stderr
    seen = json.loads(out.stdout)
    assert seen["large"] > 100 and 65536 < seen["most"] <= 160 * 1024, seen
    assert seen["over"] == 0, seen


def test_sizes_of_the_descriptors():
    """What the calls above hand over as bytes."""
    from hi3d_amd import attention

    assert ctypes.sizeof(attention._TermsDesc) == 48 and ctypes.sizeof(attention._SharedDesc) == 64
