"""The launches of the largest calls, on the CPU: the entry points run in a process where the HIP runtime's launch
functions only write down what they are given, so that calls of any size can be looked at.  A launch holds fewer
than 2^32 threads (the hardware counts them in 32 bits); a larger one is refused by the runtime, for the optimizer's
step after its count has gone up."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "rwkv-megatron_amd", "librwkv6_amd.so")

RUNTIME = r"""
#include <stddef.h>
#include <stdint.h>
typedef struct { uint32_t x, y, z; } dim;
static dim grid, block; static size_t lds; static void* stream;
uint64_t seen[1024][2]; int count;
int __hipPushCallConfiguration(dim g, dim b, size_t s, void* st) { grid = g; block = b; lds = s; stream = st; return 0; }
int __hipPopCallConfiguration(dim* g, dim* b, size_t* s, void** st) { *g = grid; *b = block; *s = lds; *st = stream; return 0; }
int hipLaunchKernel(const void* f, dim g, dim b, void** a, size_t s, void* st) {
    if (count < 1024) { seen[count][0] = (uint64_t)g.x * g.y * g.z; seen[count][1] = (uint64_t)b.x * b.y * b.z; ++count; }
    return 0;
}
int hipGetLastError(void) { return 0; }
"""

CHILD = r"""
import ctypes, json, sys
run = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(sys.argv[2])
vp, i64, i32, f32, f64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_double
seen, count = (ctypes.c_uint64 * 2 * 1024).in_dll(run, "seen"), ctypes.c_int.in_dll(run, "count")
at = lambda k: vp(k << 50)

def launches(fn, *args):
    count.value = 0
    status = fn(*args)
    return [status] + [list(seen[i]) for i in range(count.value)]

def adamw(sizes, eight, fn=L.rwkv6_adamw_step):
    n = len(sizes)
    lists = lambda base: (vp * n)(*[(base << 50) + (i << 42) for i in range(n)])
    ints = lambda v: (i32 * n)(*[v] * n)
    return launches(fn, lists(1), ints(1), lists(2), ints(1), lists(3), lists(4), lists(5) if eight else None, lists(6) if eight else None,
                    (i64 * n)(*sizes), i64(n), at(7), f64(1e-3), None, f64(.9), f64(.99), f64(1e-8), f64(.1), None, i64(0), f32(1), None, at(8), None)

def norm(sizes):
    n = len(sizes)
    return launches(L.rwkv6_grad_norm_sums, (vp * n)(*[(2 << 50) + (i << 42) for i in range(n)]), (i32 * n)(*[1] * n), (i64 * n)(*sizes), i64(n), at(7), None)

def loss(N, V, dt, back):
    if back:
        return launches(L.rwkv6_cross_entropy_bwd, at(1), i32(dt), i64(V), at(2), i64(-100), at(3), at(4), at(5), i64(N), i64(V), None)
    return launches(L.rwkv6_cross_entropy_fwd, at(1), i32(dt), i64(V), at(2), i64(-100), at(3), at(4), i64(N), i64(V), None)

def residual(N, C, back, gate):
    g, dg = (at(8), at(9)) if gate else (None, None)
    if back:
        return launches(L.rwkv6_residual_norm_bwd, at(1), i32(1), at(2), None, i32(0), g, f32(1), i32(0), at(3), i32(0), at(4), at(5), None, at(6), at(7),
                        at(10), dg, at(11), at(12), i32(0), None, at(13), i64(N), i64(C), None)
    return launches(L.rwkv6_residual_norm_fwd, at(1), i32(1), at(2), None, i32(0), g, f32(1), i32(0), at(3), at(4), i32(0), f32(1e-5), at(5), at(6), at(7), at(10),
                    i64(N), i64(C), None)

print(json.dumps(eval(sys.argv[3])))
"""


@pytest.fixture(scope="module")
def look(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None or not os.path.exists(LIB):
        pytest.skip("needs a C compiler and the built library")
    d = tmp_path_factory.mktemp("runtime")
    (d / "runtime.c").write_text(RUNTIME)
    (d / "child.py").write_text(CHILD)
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(d / "runtime.so"), str(d / "runtime.c")], check=True)

    def run(call):
        out = subprocess.run([sys.executable, str(d / "child.py"), str(d / "runtime.so"), LIB, call], check=True, capture_output=True, text=True)
        status, *launches = json.loads(out.stdout.splitlines()[-1])
        return status, launches

    return run


# One buffer of all parameters in bf16 with 8-bit states takes 6 bytes an element: 2^35 of them, 206 GB, fit the card.
@pytest.mark.parametrize("sizes", ["[1 << 34]", "[(1 << 35) - 2047]", "[1 << 35]", "[1 << 35, 5, 1 << 34]", "[1 << 37]", "[1 << 30] * 128",
                                   "[(1 << 31) + 1] * 60"])
@pytest.mark.parametrize("eight", [False, True])
def test_adamw(look, sizes, eight):
    for fn in ("rwkv6_adamw_step", "rwkv6_adamw_step_stochastic"):
        status, launches = look(f"adamw({sizes}, {eight}, L.{fn})")
        assert status == 0 and len(launches) == 1 + -(-len(eval(sizes)) // 60)
        assert all(0 < g * b < 1 << 32 for g, b in launches), launches
    status, launches = look(f"norm({sizes})")
    assert status == 0 and launches and all(0 < g * b < 1 << 32 for g, b in launches), launches


def test_a_call_past_the_limit_launches_nothing(look):
    for sizes in ("[(1 << 37) + 1]", "[1 << 36] * 3"):
        assert look(f"adamw({sizes}, True)") == (2, []) == look(f"norm({sizes})")


# 256 GiB of bf16 logits, and more rows than a grid's blocks at every number of threads a row.
@pytest.mark.parametrize("N,V", [(1 << 21, 65536), (1 << 22, 32768), (1 << 23, 8192), (1 << 26, 512), (1 << 35, 8), (1 << 40, 1)])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("dt", [0, 1])
def test_cross_entropy(look, N, V, back, dt):
    status, launches = look(f"loss({N}, {V}, {dt}, {back})")
    assert status == 0 and len(launches) == 1 and 0 < launches[0][0] * launches[0][1] < 1 << 32, launches


@pytest.mark.parametrize("N,C", [(1 << 37, 8), (1 << 32, 256), (1 << 30, 1024), (1 << 28, 4096), (1 << 27, 8192)])
@pytest.mark.parametrize("gate", [False, True])
def test_residual_norm(look, N, C, gate):
    for back in (False, True):
        status, launches = look(f"residual({N}, {C}, {back}, {gate})")
        assert status == 0 and len(launches) == 1 + back and all(0 < g * b < 1 << 32 for g, b in launches), launches
