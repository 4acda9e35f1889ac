"""CPU checks of the gated delta rule's C entries: bad calls return an error code before any launch (the pointers are
fake, nothing is dereferenced), the launches of large calls, and what the Python functions refuse."""
import ctypes
import json
import os
import shutil
import subprocess
import sys

import pytest
import torch

OK, INVALID, UNSUPPORTED, ALIGNMENT = 0, 1, 2, 4
F32, BF16 = 0, 1
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "rwkv-megatron_amd", "librwkv6_amd.so")


def _p(addr):
    return ctypes.c_void_p(addr)


A = [_p(0x10000000 * i) for i in range(1, 20)]        # 256 MB apart
DENSE = dict(q=(2 * 100 * 64, 100 * 64, 64), v=(4 * 100 * 64, 100 * 64, 64))


def _strides(*ts):
    flat = [x for t in ts for x in t]
    return (ctypes.c_int64 * len(flat))(*flat)


QK, V = DENSE["q"], DENSE["v"]


def _fwd(L, **kw):
    a = dict(q=A[0], k=A[1], v=A[2], strides=_strides(QK, QK, V), g=A[3], beta=A[4], bdt=BF16, h0=A[5], o=A[6], hT=A[7], saved=A[8],
             ws=None, B=2, H=2, HV=4, T=100, K=64, V=64, scale=1.0, stream=None)
    a.update(kw)
    return L.rwkv6_gated_delta_fwd(*a.values())


def _bwd(L, **kw):
    a = dict(q=A[0], k=A[1], v=A[2], do=A[3], strides=_strides(QK, QK, V, V), beta=A[4], bdt=F32, dhT=A[5], saved=A[6], dq=A[7], dk=A[8],
             dv=A[9], dg=A[10], db=A[11], dh0=A[12], ws=A[13], B=2, H=2, HV=4, T=100, K=64, V=64, scale=1.0, stream=None)
    a.update(kw)
    return L.rwkv6_gated_delta_bwd(*a.values())


def _step(L, **kw):
    a = dict(q=A[0], k=A[1], v=A[2], strides=_strides(QK, QK, V), g=A[3], beta=A[4], bdt=F32, state=A[5],
             ss=(ctypes.c_int64 * 2)(4 * 4096, 4096), o=A[6], B=2, H=2, HV=4, T=1, K=64, V=64, scale=1.0, stream=None)
    a.update(kw)
    return L.rwkv6_gated_delta_step(*a.values())


def test_refused_before_launch(pkg):
    L = pkg._lib.load()
    for call in (_fwd, _bwd, _step):
        assert call(L, B=0) == OK
        for kw in (dict(q=None), dict(k=None), dict(v=None), dict(beta=None), dict(strides=None), dict(bdt=2), dict(B=-1), dict(T=-1), dict(H=0),
                   dict(HV=3), dict(HV=0), dict(V=0)):
            assert call(L, **kw) == INVALID, (call, kw)
        for kw in (dict(K=32), dict(K=192), dict(V=96), dict(V=576), dict(T=1 << 31), dict(B=1 << 24), dict(B=1 << 20, T=64 * 64)):
            assert call(L, **kw) == UNSUPPORTED, (call, kw)
        for n in ("q", "k", "v"):
            assert call(L, **{n: _p(0x150000008)}) == ALIGNMENT, (call, n)
        odd = _strides((12804, 6400, 64), QK, V, V)
        negative = _strides((-12800, 6400, 64), QK, V, V)
        far = _strides((1 << 41, 6400, 64), QK, V, V)
        assert (call(L, strides=odd), call(L, strides=negative), call(L, strides=far)) == (ALIGNMENT, INVALID, UNSUPPORTED), call
    for kw in (dict(g=None), dict(o=None), dict(saved=None), dict(o=A[2]), dict(hT=A[6]), dict(saved=A[0]), dict(hT=A[5]),
               dict(saved=None, ws=A[3]), dict(o=_p(A[0].value + 2 * 2 * 100 * 64 * 2 - 16))):
        assert _fwd(L, **kw) == INVALID, kw
    for n in ("h0", "o", "hT", "saved"):
        assert _fwd(L, **{n: _p(0x150000004)}) == ALIGNMENT, n
    for kw in (dict(do=None), dict(saved=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dg=None), dict(db=None), dict(ws=None),
               dict(dq=A[0]), dict(dv=A[3]), dict(dh0=A[5]), dict(ws=A[6]), dict(dk=A[7]), dict(dg=A[11])):
        assert _bwd(L, **kw) == INVALID, kw
    strides = lambda sb, sh: (ctypes.c_int64 * 2)(sb, sh)
    for kw in (dict(g=None), dict(o=None), dict(state=None), dict(ss=None), dict(o=A[5]), dict(state=A[0]), dict(ss=strides(0, 4096)),
               dict(ss=strides(4096, 4096)), dict(ss=strides(4 * 4096 - 4, 4096)), dict(ss=strides(16384, 4092)), dict(ss=strides(-16384, 4096))):
        assert _step(L, **kw) == INVALID, kw
    for kw in (dict(ss=strides(16386, 4096)), dict(state=_p(0x150000004)), dict(ss=strides(40000, 4098))):
        assert _step(L, **kw) == ALIGNMENT, kw
    assert _step(L, T=0) == OK


def test_sizes(pkg):
    L = pkg._lib.load()
    B, HV, T = 8, 32, 4096
    chunks = B * HV * T // 64
    # 64 tokens of a head: T 10 KB, G and beta, states and written values of 16 KB
    assert L.rwkv6_gated_delta_saved_bytes(B, HV, T, 64, 64) == chunks * (10240 + 512 + 256 + 16384 + 16384)
    assert L.rwkv6_gated_delta_workspace_bytes(B, HV, T, 64, 64, 0) == chunks * (10240 + 512 + 256)
    assert L.rwkv6_gated_delta_workspace_bytes(B, HV, T, 64, 64, 1) == chunks * (16384 + 16384)
    # few heads, many chunks: a map [K,K] and a state [K,V] for each of up to 16 segments but the last
    maps = L.rwkv6_gated_delta_workspace_bytes(1, 4, 65536, 64, 64, 0) - 4096 * (10240 + 512 + 256)
    assert maps == 4 * 15 * 64 * 128 * 4
    assert L.rwkv6_gated_delta_saved_bytes(1, 4, 65536, 64, 64) == 4096 * (10240 + 512 + 256 + 16384 + 16384) + maps
    assert L.rwkv6_gated_delta_workspace_bytes(1, 4, 65536, 64, 64, 1) == 4096 * (16384 + 16384) + maps
    assert L.rwkv6_gated_delta_saved_bytes(1, 1, 1, 128, 64) == 10240 + 512 + 256 + 32768 + 16384
    assert L.rwkv6_gated_delta_saved_bytes(B, HV, 0, 64, 64) == 0 == L.rwkv6_gated_delta_saved_bytes(B, HV, T, 32, 64)


RUNTIME = r"""
#include <stddef.h>
#include <stdint.h>
typedef struct { uint32_t x, y, z; } dim;
static dim grid, block; static size_t lds; static void* stream;
uint64_t seen[64][3]; int count;
int __hipPushCallConfiguration(dim g, dim b, size_t s, void* st) { grid = g; block = b; lds = s; stream = st; return 0; }
int __hipPopCallConfiguration(dim* g, dim* b, size_t* s, void** st) { *g = grid; *b = block; *s = lds; *st = stream; return 0; }
int hipLaunchKernel(const void* f, dim g, dim b, void** a, size_t s, void* st) {
    if (count < 64) { seen[count][0] = (uint64_t)g.x * g.y * g.z; seen[count][1] = (uint64_t)b.x * b.y * b.z; seen[count][2] = s; ++count; }
    return 0;
}
int hipGetLastError(void) { return 0; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return v > 163840; }
"""

CHILD = r"""
import ctypes, json, sys
run = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(sys.argv[2])
vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
seen, count = (ctypes.c_uint64 * 3 * 64).in_dll(run, "seen"), ctypes.c_int.in_dll(run, "count")
at = lambda k: vp(k << 50)

def call(what, B, H, HV, T, K, V):
    count.value = 0
    dense = lambda heads, C: [heads * T * C, T * C, C]
    st = (i64 * 12)(*dense(H, K), *dense(H, K), *dense(HV, V), *dense(HV, V))
    size = [i64(x) for x in (B, H, HV, T, K, V)]
    if what == "fwd":
        r = L.rwkv6_gated_delta_fwd(at(1), at(2), at(3), st, at(4), at(5), i32(0), None, at(6), at(7), None, at(8), *size, f32(1), None)
    elif what == "bwd":
        r = L.rwkv6_gated_delta_bwd(at(1), at(2), at(3), at(4), st, at(5), i32(1), None, at(6), at(7), at(8), at(9), at(10), at(11), at(12), at(13),
                                    *size, f32(1), None)
    else:
        r = L.rwkv6_gated_delta_step(at(1), at(2), at(3), st, at(4), at(5), i32(0), at(6), (i64 * 2)(HV * K * V, K * V), at(7), *size, f32(1), None)
    return [r] + [list(seen[i]) for i in range(count.value)]

print(json.dumps([call(*c) for c in json.loads(sys.argv[3])]))
"""


def test_launches_of_large_calls(tmp_path):
    """A launch holds fewer than 2^32 threads and at most 160 KB of LDS a block; the entry points run with a runtime
    that only writes down what it is given."""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None or not os.path.exists(LIB):
        pytest.skip("needs a C compiler and the built library")
    (tmp_path / "runtime.c").write_text(RUNTIME)
    (tmp_path / "child.py").write_text(CHILD)
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(tmp_path / "runtime.so"), str(tmp_path / "runtime.c")], check=True)
    sizes = [(1, 1, 1, 1, 64, 64), (1, 1, 1, 1, 128, 512), (8, 32, 32, 4096, 64, 64), (4, 16, 32, 2048, 128, 128), (1, 16, 16, 1 << 24, 64, 64),
             ((1 << 17) - 1, 64, 64, 1, 64, 64), (1, 1, 1, 1 << 28, 128, 64), (6, 7, 21, 777, 128, 320)]
    calls = [(w, *s) for w in ("fwd", "bwd", "step") for s in sizes]
    out = subprocess.run([sys.executable, str(tmp_path / "child.py"), str(tmp_path / "runtime.so"), LIB, json.dumps(calls)], check=True,
                         capture_output=True, text=True)
    for c, (status, *launches) in zip(calls, json.loads(out.stdout.splitlines()[-1])):
        long = c[4] >= 1 << 24                                   # the walks' segments, and what joins them
        assert status == OK and len(launches) == {"fwd": 4 if long else 2, "bwd": 4 if long else 2, "step": 1}[c[0]], (c, status, launches)
        for blocks, threads, lds in launches:
            assert 0 < blocks * threads < 1 << 32 and threads <= 1024 and lds <= 163840, (c, launches)


def test_python_refuses(pkg):
    gd = pkg.gated_delta
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    args = [t(1, 2, 5, 64), t(1, 2, 5, 64), t(1, 4, 5, 64), t(1, 4, 5), t(1, 4, 5)]
    with pytest.raises(ValueError, match="GPU"):
        gd.gated_delta_rule(*args)
    with pytest.raises(ValueError, match="GPU"):
        gd.gated_delta_step(*args, t(1, 4, 64, 64, dt=torch.float32))
    with pytest.raises(TypeError, match="q must be"):
        gd.gated_delta_rule(None, *args[1:])
