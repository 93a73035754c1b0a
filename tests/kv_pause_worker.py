"""Run by tests/test_kv_pause_host.py in a process of its own, on the host stand-in (argv[1]): which calls are refused while paused.
Nothing reads the addresses."""
import ctypes as C
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from asystem_amem_amd import binding as B  # noqa: E402
from asystem_amem_amd import kv  # noqa: E402

lib = B.load(sys.argv[1])
for name, (res, args) in kv._SIGNATURES.items():
    fn = getattr(lib, name)
    fn.restype, fn.argtypes = res, args
MiB = 1 << 20


def region():
    va, handle, size = C.c_uint64(), C.c_uint64(), C.c_uint64()
    assert lib.amem_vmm_alloc(4 * MiB, 0, C.byref(va), C.byref(handle), C.byref(size)) == 0
    return va.value, handle.value, size.value


mine, _, _ = region()                                  # not tracked
their, handle, size = region()
assert lib.amem_add_alloc_info(their, size, B.TYPE_LOCAL, 0, handle, -1, 0, None, B.CALLER_P2P) == 0

PAGES, HEADS, PAGE, DIM, TOKENS, Q = 10, 4, 64, 128, 20, 8


def arguments():
    a = mine
    cache = kv.CacheInfo(a, a, a, a, HEADS * PAGE * DIM, PAGE * DIM, DIM, 8, 2, kv.E4M3, 0, PAGES, HEADS, PAGE, 32, DIM, 0)
    batch = kv.BatchInfo(a, a, a, 5, 3, 5, TOKENS, 8, 320, 0)
    app = kv.AppendArgs(a, a, a, a, a, a, a, 512, 128, 512, 128, 1024, 128, 1024, 128, TOKENS, kv.BF16, Q, 128, 0, 1000, 1)
    att = kv.AttentionArgs(a, a, a, a, 4096, 1024, 128, 1024, 128, 0.1, kv.BF16, Q, 1, 0, 0)
    return cache, batch, app, att


def call(cache, batch, app, att):
    return (lib.amem_kv_append(C.byref(cache), C.byref(batch), C.byref(app), None),
            lib.amem_kv_attention(C.byref(cache), C.byref(batch), C.byref(att), None))


# bytes of every tensor: record, field, how many, which of the two calls names it
ROWS, LONG = (TOKENS - 1) * 1024 + HEADS * 256, (TOKENS - 1) * 2048 + Q * 256
TENSORS = [(0, "k", PAGES * HEADS * PAGE * DIM, (1, 1)), (0, "v", PAGES * HEADS * PAGE * DIM, (1, 1)), (0, "k_scale", PAGES * 8 * 4, (1, 1)),
           (0, "v_scale", PAGES * 8 * 4, (1, 1)), (1, "page_table", 15 * 4, (1, 1)), (1, "context", 12, (1, 1)), (1, "cu_tokens", 16, (1, 1)),
           (2, "k", ROWS, (1, 0)), (2, "v", ROWS, (1, 0)), (2, "q", LONG, (1, 0)), (2, "q_out", LONG, (1, 0)), (2, "cos", 1000 * 256, (1, 0)),
           (2, "sin", 1000 * 256, (1, 0)), (2, "positions", TOKENS * 4, (1, 0)), (3, "q", LONG, (0, 1)), (3, "out", LONG, (0, 1)),
           (3, "lse", TOKENS * Q * 4, (0, 1)), (3, "workspace", 4096, (0, 1))]


def down(x):
    return x // 16 * 16


assert call(*arguments()) == (0, 0) and lib.kv_host_launches() == 2
for paused in (False, True):
    if paused:
        assert lib.ncclPause(None) == 0
    before = lib.kv_host_launches()
    assert call(*arguments()) == (0, 0), "memory that is not tracked"
    assert lib.kv_host_launches() == before + 2
    for record, field, nbytes, named in TENSORS:
        # the first byte, the last one, one that begins before the region and reaches into it; and just outside of it
        for at, inside in ((their, True), (their + size - 16, True), (their - down(nbytes - 1), True), (their - down(nbytes + 15), False),
                           (their + size, False)):
            a = arguments()
            setattr(a[record], field, at)
            want = tuple(int(paused and inside and bool(n)) for n in named)
            assert call(*a) == want, (paused, field, record, at - their, inside)
assert lib.ncclResume(None) == 0
a = arguments()
a[0].k = their
assert call(*a) == (0, 0)
print("kv pause worker: all done")
