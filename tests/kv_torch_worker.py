"""Run by tests/test_gpu_kv.py in a process of its own: the Python entry points on torch tensors."""
import os
import sys

os.environ.setdefault("AMEM_ENABLE", "1")
os.environ.setdefault("GMM_LOG", "1")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import torch  # noqa: E402  (before the library: one HIP runtime for both)

from asystem_amem_amd import kv  # noqa: E402

DEV = "cuda"


def step(name):
    print(name, flush=True)


def tables(rows, pairs):
    a = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * torch.rand(pairs, device=DEV, dtype=torch.float64)
    return a.cos().float(), a.sin().float()


class World:
    """A decoding batch of `batch` sequences over a cache of 16 or 8 bits."""

    def __init__(self, batch, context, eight, dtype=torch.bfloat16, heads=8, kv_heads=2, dim=128, page=32, block=16, tokens=1):
        g = torch.Generator(device=DEV)
        g.manual_seed(1)
        pages = batch * (-(-context // page)) + 1
        shape = (pages, kv_heads, page, dim)
        x = torch.randn(2, *shape, device=DEV, generator=g)
        if eight:
            self.k, self.v = (x * 50).to(torch.float8_e4m3fn)
            self.ks, self.vs = torch.full((2, pages, kv_heads, page // block), 2.0 ** -6, device=DEV)
        else:
            self.k, self.v = x.to(dtype)
            self.ks = self.vs = None
        self.table = torch.randperm(pages, device=DEV, generator=g)[:batch * (-(-context // page))].view(batch, -1).int()
        self.context = torch.randint(tokens, context + 1, (batch,), device=DEV, generator=g).int()
        n = batch * tokens
        self.new_k, self.new_v = torch.randn(2, n, kv_heads, dim, device=DEV, generator=g).to(dtype)
        self.q = torch.randn(n, heads, dim, device=DEV, generator=g).to(dtype)
        self.turned, self.out = torch.empty_like(self.q), torch.empty_like(self.q)
        self.lse = torch.empty(n, heads, device=DEV)
        self.cache = kv.Cache(self.k, self.v, self.ks, self.vs)
        self.batch = kv.Batch(self.table, self.context, tokens=n, max_context=context)
        self.rotation = kv.Rotation(*tables(context, dim // 2))
        self.workspace = torch.empty(max(16, kv.attention_workspace(self.cache, self.batch, heads)), dtype=torch.uint8, device=DEV)

    def run(self, workspace=None):
        s = torch.cuda.current_stream().cuda_stream
        kv.append(self.cache, self.batch, self.new_k, self.new_v, self.q, self.turned, rotation=self.rotation, stream=s)
        kv.attention(self.cache, self.batch, self.turned, self.out, lse=self.lse, workspace=self.workspace if workspace is None else workspace,
                     stream=s)

    def state(self):
        torch.cuda.synchronize()
        return [t.clone().view(torch.uint8) for t in (self.k, self.v, self.out, self.lse, self.turned)] + (
            [self.ks.clone(), self.vs.clone()] if self.ks is not None else [])


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def refused(fn, *args, **kw):
    try:
        fn(*args, **kw)
    except ValueError:
        return True
    return False


step("strided views are read as they are")
for eight in (False, True):
    w = World(5, 200, eight, tokens=3)
    w.run()
    plain = w.state()
    wide = torch.zeros(w.q.shape[0], 12, 128, device=DEV, dtype=w.q.dtype)      # queries, keys, values of one product
    wide[:, :8], wide[:, 8:10], wide[:, 10:] = w.q, w.new_k, w.new_v
    out = torch.full((8, w.q.shape[0], 128), 7.0, device=DEV, dtype=w.q.dtype)
    s = torch.cuda.current_stream().cuda_stream
    kv.append(w.cache, w.batch, wide[:, 8:10], wide[:, 10:], wide[:, :8], wide[:, :8], rotation=w.rotation, stream=s)
    kv.attention(w.cache, w.batch, wide[:, :8], out.transpose(0, 1), workspace=w.workspace, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :8], w.turned) and torch.equal(out.transpose(0, 1), w.out)
    assert same(plain, w.state())

step("another stream than the tensors' own")
w = World(4, 300, True)
w.run()
want = w.state()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
w.out.zero_()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    w.run()
side.synchronize()
assert same(want, w.state())

step("two calls at once, on two streams with a workspace each")
a, b = World(2, 20000, True), World(3, 700, False, tokens=30)
wants = []
for w in (a, b):
    w.run()
    wants.append(w.state())
streams = [torch.cuda.Stream(), torch.cuda.Stream()]
for w in (a, b):
    w.out.zero_()
    w.lse.zero_()
torch.cuda.synchronize()
for _ in range(20):
    for w, side in zip((a, b), streams):
        with torch.cuda.stream(side):
            w.run()
assert same(wants[0], a.state()) and same(wants[1], b.state())

step("the result in the queries' place, no tokens at all, an error of the caller's that is not this call's")
for tokens, context in ((1, 3000), (3, 100), (40, 90)):
    w = World(3, context, True, tokens=tokens)
    w.run()
    torch.cuda.synchronize()
    s = torch.cuda.current_stream().cuda_stream
    kv.attention(w.cache, w.batch, w.turned, w.turned, workspace=w.workspace, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(w.turned, w.out)
none = kv.Batch(w.table, w.context, tokens=0, cu_tokens=torch.zeros(4, dtype=torch.int32, device=DEV), max_context=90)
before = w.state()
kv.append(w.cache, none, w.new_k[:0], w.new_v[:0], w.q[:0], w.q[:0], rotation=w.rotation, stream=s)
kv.attention(w.cache, none, w.q[:0], w.out[:0], workspace=w.workspace, stream=s)
big = torch.randn(8192, 8192, device=DEV)
big @ big
e = torch.cuda.Event()
e.record()
e.query()                         # most likely not ready
kv.attention(w.cache, w.batch, w.q, w.out, workspace=w.workspace, stream=s)
torch.cuda.synchronize()

step("captured and replayed, with eager work in between, two graphs on one workspace")
for eight in (False, True):
    a, b = World(6, 1500, eight), World(3, 4000, eight, tokens=2)
    shared = torch.empty(max(a.workspace.numel(), b.workspace.numel()), dtype=torch.uint8, device=DEV)
    graphs = []
    for w in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.run(shared)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            w.run(shared)
        graphs.append(g)
    for turn in range(4):
        wants = []
        for w in (a, b):          # new tokens, other contexts, eagerly
            w.q.normal_()
            w.new_k.normal_()
            w.new_v.normal_()
            w.context.sub_(1).clamp_(min=2)
            keep = w.state()[:2] + ([w.ks.clone(), w.vs.clone()] if eight else [])
            w.run()
            wants.append(w.state())
            for t, x in zip((w.k, w.v) + ((w.ks, w.vs) if eight else ()), keep):
                t.view(torch.uint8).copy_(x.view(torch.uint8))
            w.out.zero_()
            w.lse.zero_()
            w.turned.zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        assert same(wants[0], a.state()) and same(wants[1], b.state()), turn

step("refusals")
w = World(2, 64, True)
s = 0
half = w.q.half()
assert refused(kv.append, w.cache, w.batch, w.new_k, w.new_v[:1])
assert refused(kv.append, w.cache, w.batch, w.new_k, w.new_v.half())
assert refused(kv.append, w.cache, w.batch, w.new_k.float(), w.new_v.float())
assert refused(kv.append, w.cache, w.batch, w.new_k, w.new_v, w.q)
assert refused(kv.append, w.cache, w.batch, w.new_k.cpu(), w.new_v)
assert refused(kv.append, w.cache, w.batch, w.new_k, w.new_v, positions=w.context)
assert refused(kv.attention, w.cache, w.batch, w.q, half)
assert refused(kv.attention, w.cache, w.batch, w.q, w.out[:, :4])
assert refused(kv.attention, w.cache, w.batch, w.q, w.out, lse=w.lse.double())
assert refused(kv.attention, w.cache, w.batch, w.q.transpose(1, 2), w.out)
assert refused(kv.attention, w.cache, w.batch, w.q, w.out, window=1 << 40)
assert refused(kv.attention, w.cache, w.batch, w.q, w.out, window=1.5)
assert refused(kv.attention, w.cache, w.batch, w.q, w.out, scale=1e300)
assert refused(kv.Cache, w.k, w.v)
assert refused(kv.Cache, w.k, w.v, w.ks[:1], w.vs[:1])
assert refused(kv.Cache, w.k.transpose(2, 3), w.v.transpose(2, 3), w.ks, w.vs)
assert refused(kv.Batch, w.table.long(), w.context, tokens=2, max_context=64)
assert refused(kv.Batch, w.table, w.context, tokens=2)
assert refused(kv.Rotation, w.lse, w.lse[:1])
assert refused(kv.Rotation, *tables(10, 64), sections=(10, 10))
for kw in (dict(window=-1), dict(scale=float("inf"))):
    try:
        kv.attention(w.cache, w.batch, w.q, w.out, workspace=w.workspace, **kw)
        assert False
    except kv.KvError as e:
        assert e.code == 1
big = World(1, 20000, True)
if kv.attention_workspace(big.cache, big.batch, 8):
    try:
        kv.attention(big.cache, big.batch, big.q, big.out)
        assert False
    except kv.KvError as e:
        assert e.code == 1
w.run()
torch.cuda.synchronize()
print("kv torch worker: all done", flush=True)
