"""What memory gd_kv_attn takes for the partials of split keys, on the CPU: in a process whose
HIP runtime is a stand-in (below) that counts allocations, refuses those past a limit and
notes what is launched.  A call that can do with less memory does, and batches that grow do
not make the workspace anew each time."""
import subprocess
import sys
from pathlib import Path

import pytest

HIP = r"""
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>
#define F __attribute__((visibility("default")))
typedef struct { uint32_t x, y, z; } dim3;
size_t limit = ~(size_t)0;
int mallocs, syncs, launches, n_live;
struct { uintptr_t at; size_t size; } live[64];
/* of the last kernel of `most`: */
int splits;
uintptr_t part;
static dim3 grid, block;
F int hipGetDeviceCount(int *n) { *n = 1; return 0; }
F int hipSetDevice(int d) { return 0; }
F int hipStreamCreateWithFlags(void **s, unsigned f) { *s = (void *)8; return 0; }
F int hipStreamDestroy(void *s) { return 0; }
F int hipStreamSynchronize(void *s) { syncs++; return 0; }
F int hipEventCreate(void **e) { *e = (void *)8; return 0; }
F int hipEventDestroy(void *e) { return 0; }
F int hipGetDevicePropertiesR0600(void *p, int d) { return 1; }
F int hipGetSymbolAddress(void **p, const void *s) { *p = 0; return 1; }
F int hipThreadExchangeStreamCaptureMode(int *m) { return 0; }
F int hipGetLastError(void) { return 0; }
F const char *hipGetErrorString(int e) { return "out of memory"; }
F int hipMalloc(void **p, size_t n) {
    static uintptr_t next = 1ull << 40;
    mallocs++;
    *p = 0;
    if (n > limit || n_live == 64) return 2;
    *p = (void *)next;
    live[n_live].at = next;
    live[n_live++].size = n;
    next += (n + 4095) / 4096 * 4096 + 4096;
    return 0;
}
F int hipFree(void *p) {
    for (int i = 0; i < n_live; i++)
        if (live[i].at == (uintptr_t)p) live[i] = live[--n_live];
    return 0;
}
F int __hipPushCallConfiguration(dim3 g, dim3 b, size_t l, void *s) { grid = g; block = b; return 0; }
F int __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *l, void **s) { *g = grid; *b = block; *l = 0; *s = (void *)8; return 0; }
F int hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t l, void *s) {
    if (launches++ % 2 == 0) {      /* cache, rows, q, stride, gate, stride, out, partials, splits */
        part = *(uintptr_t *)args[7];
        splits = *(int *)args[8];
    }
    return 0;
}
F int hipStreamBeginCapture(void *s, int m) { return 0; }
F int hipStreamEndCapture(void *s, void **g) { *g = (void *)8; return 0; }
F int hipGraphInstantiate(void **e, void *g, void *n, void *l, size_t z) { *e = (void *)8; return 0; }
F int hipGraphExecDestroy(void *e) { return 0; }
F int hipGraphDestroy(void *g) { return 0; }
"""

PROGRAM = r"""
import ctypes as C, sys
hip = C.CDLL(sys.argv[1], C.RTLD_GLOBAL)
import gadeon_amd as ga
MB = 1 << 20
i = lambda name: C.c_int.in_dll(hip, name)
limit = C.c_size_t.in_dll(hip, "limit")
class Live(C.Structure):
    _fields_ = [("at", C.c_size_t), ("size", C.c_size_t)]
live = (Live * 64).in_dll(hip, "live")
P, hd, H = 1 << 20, 128, 16
def attend(ctx, rows, positions):
    # a chunk of `rows` behind `positions`; -> splits, whose partials lie inside one allocation
    kv = ga.KV(k=P, v=P, k_exp=P, v_exp=P, n_pages=10, dtype=ga.I8, n_head_kv=2, head_dim=hd, page_size=16)
    s = ga.Seqs(n_rows=rows, row_start=P, pos=P, rope_shift=None, page_table=P, n_seq=1, max_pages=positions // 16, max_len=0)
    i("launches").value = 0
    ctx.gd_kv_attn(kv, s, P, H * hd, None, 0, P + (1 << 32), ga.F32, H, 0.1, 0, 0)
    n, at = i("splits").value, C.c_size_t.in_dll(hip, "part").value
    assert i("launches").value == (2 if n > 1 else 1)
    need = rows * H * (hd + 3) * 4 * n
    assert n == 1 or any(l.at <= at and at + need <= l.at + l.size for l in live[:i("n_live").value]), (rows, n)
    return n
"""


def run(tmp_path, body):
    src, lib = tmp_path / "hip.c", tmp_path / "libstandin.so"
    src.write_text(HIP)
    cc = subprocess.run(["g++", "-x", "c", "-w", "-shared", "-fPIC", "-O1", str(src), "-o", str(lib)], capture_output=True, text=True)
    assert cc.returncode == 0, cc.stderr
    r = subprocess.run([sys.executable, "-c", PROGRAM + body, str(lib)], cwd=Path(__file__).resolve().parents[1],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_without_memory_for_the_workspace(tmp_path):
    """No workspace, an old one, no scratch either: fewer splits, and never a failure."""
    run(tmp_path, r"""
ctx = ga.Context(0)
most = attend(ctx, 300, 16000)
assert most == 63                                          # 159 MB of partials
small = ga.Context(0)
limit.value = 10 * MB                                      # (the attention scratch, 8 MB, is there)
few = attend(small, 300, 16000)
assert few == 8 * MB // (300 * H * (hd + 3) * 4) == 3
assert attend(small, 600, 16000) == 1 and attend(small, 100, 16000) == 10
limit.value = 70 * MB
assert attend(small, 60, 16000) == 63                      # 32 MB
assert attend(small, 1000, 16000) == 4                     # no 256 MB: what the 32 hold
assert attend(small, 60, 16000) == 63 and attend(ctx, 300, 16000) == most
limit.value = 1 * MB
bare = ga.Context(0)
assert attend(bare, 300, 16000) == 1 and attend(bare, 2, 16000) == 1
""")


def test_a_recording_takes_the_workspace_as_it_is(tmp_path):
    run(tmp_path, r"""
ctx = ga.Context(0)
n = i("mallocs").value
ctx.gd_graph_begin()
assert attend(ctx, 60, 16000) == 16 and i("mallocs").value == n + 1      # the recording's own scratch
g = C.c_void_p()
ctx.gd_graph_end(C.byref(g))
assert attend(ctx, 60, 16000) == 63                        # 32 MB
ctx.gd_graph_begin()
assert attend(ctx, 60, 16000) == 63
h = C.c_void_p()
ctx.gd_graph_end(C.byref(h))
held = i("n_live").value
attend(ctx, 1500, 16000)                                   # a larger workspace beside the one that h holds
assert i("n_live").value == held + 1
ctx.lib.gd_graph_destroy(h)
assert i("n_live").value == held
ctx.lib.gd_graph_destroy(g)
""")


def test_growing_batches_seldom_grow_the_workspace(tmp_path):
    run(tmp_path, r"""
ctx = ga.Context(0)
n, s = i("mallocs").value, i("syncs").value
for rows in range(50, 2000, 10):
    attend(ctx, rows, 16000)
assert i("mallocs").value - n <= 5 and i("syncs").value - s <= 4         # 16, 32, .. 256 MB
assert max(l.size for l in live[:i("n_live").value]) == 256 * MB
""")
