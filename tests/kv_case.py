"""A paged key/value cache in device memory for the tests: built from numpy arrays, through the C ABI alone (no torch)."""
import ctypes as C

import numpy as np

from asystem_amem_amd import kv
from tests import kv_oracle as O

MiB = 1 << 20
KINDS = {"bf16": kv.BF16, "f16": kv.F16}


class Arena:
    """Device memory cut into 256-byte aligned pieces; fresh ones hold 0xA5 bytes."""

    def __init__(self, lib, size=64 * MiB):
        self.lib, self.size, self.at = lib, size, 0
        va, h, n = C.c_uint64(), C.c_uint64(), C.c_uint64()
        assert lib.amem_vmm_alloc(size, 0, C.byref(va), C.byref(h), C.byref(n)) == 0
        self.va, self.handle, self.alloc = va.value, h.value, n.value
        self.reset()

    def reset(self):
        self.at = 0

    def take(self, nbytes):
        at = self.at
        self.at += (int(nbytes) + 511) // 256 * 256
        assert self.at <= self.size, "arena is full"
        return self.va + at

    def put(self, a):
        a = np.ascontiguousarray(a)
        at = self.take(max(a.nbytes, 16))
        self.write(at, a)
        return at

    def blank(self, nbytes):
        return self.put(np.full(max(int(nbytes), 16), 0xA5, np.uint8))

    def write(self, at, a):
        a = np.ascontiguousarray(a)
        if a.nbytes:
            assert self.lib.amem_copy_to_device(at, a.ctypes.data, a.nbytes) == 0

    def read(self, at, shape, dtype):
        a = np.empty(shape, dtype)
        if a.nbytes:
            assert self.lib.amem_copy_from_device(a.ctypes.data, at, a.nbytes) == 0
        return a

    def free(self):
        self.lib.amem_vmm_free(self.va, self.alloc, 0)


class Case:
    """`lengths`: (new tokens, context) of every sequence. `slot_major`: the cache is [page][slot][head][dim]."""

    def __init__(self, arena, lengths, dim=128, q_heads=4, kv_heads=2, kind="bf16", eight=False, page=16, block=16,
                 seed=0, slot_major=False, behind=0, uniform=False, spare_pages=2, spread=1.0):
        self.arena, self.lib = arena, kv.load()
        self.r = r = np.random.RandomState(seed)
        self.lengths, self.dim, self.q_heads, self.kv_heads = lengths, dim, q_heads, kv_heads
        self.kind, self.eight, self.page, self.block, self.slot_major = kind, eight, page, block if eight else 0, slot_major
        self.tokens = sum(n for n, _ in lengths) + behind
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in lengths])]).astype(np.int32)
        self.context = np.array([c for _, c in lengths], np.int32)
        used = [-(-max(c, 0) // page) for c in self.context]
        self.table_pages = max(used + [1]) + 1
        self.pages = sum(used) + spare_pages
        self.table = np.full((len(lengths), self.table_pages), -7, np.int32)   # entries that nothing may use
        order = r.permutation(self.pages)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, dim)
        if eight:
            self.k, self.v = (O.e4m3_code(np.clip(r.standard_normal(shape) * 60 * spread, -448, 448)) for _ in "kv")
            scales = (self.pages, kv_heads, page // block)
            self.k_scale, self.v_scale = (np.exp2(r.randint(-8, -4, scales)).astype(np.float32) for _ in "kv")
        else:
            self.k, self.v = (O.encode(r.standard_normal(shape) * spread, kind) for _ in "kv")
            self.k_scale = self.v_scale = None
        self.uniform = uniform
        self.max_tokens = max([n for n, _ in lengths] + [0]) if not behind or not uniform else 0
        self.max_context = int(max(self.context.max(initial=0), 0))

    # ---- device side ----

    def upload(self):
        a = self.arena
        lay = (lambda x: x.transpose(0, 2, 1, 3)) if self.slot_major else (lambda x: x)
        self.d_k, self.d_v = a.put(lay(self.k)), a.put(lay(self.v))
        self.d_ks, self.d_vs = (a.put(self.k_scale), a.put(self.v_scale)) if self.eight else (0, 0)
        self.d_table, self.d_context, self.d_cu = a.put(self.table), a.put(self.context), a.put(self.cu)
        h, p, d = self.kv_heads, self.page, self.dim
        head, slot = (d, h * d) if self.slot_major else (p * d, d)
        blocks = self.page // self.block if self.eight else 0
        self.cache = kv.CacheInfo(self.d_k, self.d_v, self.d_ks, self.d_vs, h * p * d, head, slot, h * blocks, blocks,
                                  kv.E4M3 if self.eight else KINDS[self.kind], 0, self.pages, h, p, self.block, d, 0)
        self.batch = kv.BatchInfo(self.d_table, self.d_context, 0 if self.uniform else self.d_cu, self.table_pages,
                                  len(self.lengths), self.table_pages, self.tokens, self.max_tokens, self.max_context, 0)
        return self

    def download(self):
        """(k, v, k_scale, v_scale) as the device has them."""
        dt = np.uint8 if self.eight else np.uint16
        shape = (self.pages, self.page, self.kv_heads, self.dim) if self.slot_major else self.k.shape
        k, v = (self.arena.read(x, shape, dt) for x in (self.d_k, self.d_v))
        if self.slot_major:
            k, v = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
        if not self.eight:
            return k, v, None, None
        return (k, v) + tuple(self.arena.read(x, self.k_scale.shape, np.float32) for x in (self.d_ks, self.d_vs))

    def rows(self, heads, spread=1.0):
        return O.encode(self.r.standard_normal((self.tokens, heads, self.dim)) * spread, self.kind)

    # ---- oracle ----

    def gathered(self, s, h):
        """Keys and values [context][dim] of a sequence and head, in 64 bits."""
        p = np.arange(max(self.context[s], 0))
        page, slot = self.table[s, p // self.page], p % self.page
        k, v = self.k[page, h, slot], self.v[page, h, slot]
        if not self.eight:
            return O.decode(k, self.kind), O.decode(v, self.kind)
        b = slot // self.block
        return O.E4M3[k] * self.k_scale[page, h, b][:, None], O.E4M3[v] * self.v_scale[page, h, b][:, None]

    def visible(self, s, causal, window):
        n, c = self.lengths[s]
        at = (c - n + np.arange(n))[:, None]
        p = np.arange(max(c, 0))
        m = np.ones((n, len(p)), bool)
        if causal:
            m &= p <= at
        if window:
            m &= p > at - window
        return m
