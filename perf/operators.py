"""What is measured of the operators on a paged key/value cache: appending to it and attention over it.

Each case has a plain form in elementary torch operations, a definition in 64 bits written apart from it, and the call
of the library's own kernels (asystem_amem_amd.kv), taken where `own` is true.

The cache is [page][key/value head][slot][dim]; position p of a sequence is in slot p % page of the page that its row
of the page table names for p // page. With 8 bits a cache holds e4m3 codes and one power of two for each
(page, head, block of slots).
"""
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases

def _case(name, op, batch, tokens, context, heads, kv_heads, dim, dtype, bits, page, block=0, ragged=True, axes=1,
          interleaved=False, rotary=0, window=0):
    c = dict(op=op, batch=batch, tokens=tokens, context=context, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
             bits=bits, page=page, block=block, ragged=ragged, axes=axes, interleaved=interleaved, rotary=rotary,
             window=window)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user, one token: only latency counts
        _case("append-one", "append", 1, 1, 777, 32, 8, 128, "bf16", 16, 16, rotary=128, ragged=False),
        # a decoding batch with an 8-bit cache: every token joins a block that holds earlier ones
        _case("append-batch-8bit", "append", 128, 1, 4000, 32, 8, 128, "bf16", 8, 64, 32, rotary=128, ragged=False),
        # a few prompts of different lengths behind what is cached already; half of a head is rotated
        _case("append-prompts", "append", 6, 2500, 4001, 32, 4, 64, "f16", 16, 32, rotary=32, interleaved=True),
        # two long prompts with pictures: positions of three axes, 8 bits
        _case("append-long-8bit-axes", "append", 2, 8192, 8192, 64, 8, 128, "bf16", 8, 64, 32, rotary=128, axes=3),
        # one user, one token, a short conversation: latency
        _case("decode-one-8bit", "attend", 1, 1, 1000, 32, 8, 128, "bf16", 8, 64, 32, ragged=False),
        # the ordinary serving batch: contexts of many lengths
        _case("decode-batch-8bit", "attend", 64, 1, 8192, 32, 8, 128, "bf16", 8, 64, 32, ragged=False),
        # few users with very long contexts: the work has to be split along them
        _case("decode-long-8bit", "attend", 4, 1, 131072, 32, 8, 128, "bf16", 8, 128, 64, ragged=False),
        # every query head with keys of its own, 16 bits, small pages
        _case("decode-batch-mha", "attend", 32, 1, 4096, 16, 16, 128, "bf16", 16, 16, ragged=False),
        # drafted tokens to be checked: a few rows for each sequence
        _case("draft-rows", "attend", 24, 5, 6001, 64, 8, 64, "f16", 16, 32, ragged=False),
        # prompts of different lengths, some behind a cached prefix
        _case("prompts", "attend", 4, 3500, 4097, 32, 8, 128, "bf16", 16, 16),
        # a chunk of a long prompt over what is cached of it, 8 bits
        _case("chunk-8bit", "attend", 1, 4096, 16384, 32, 8, 128, "bf16", 8, 64, 32, ragged=False),
        # wide heads, one set of keys for all, a sliding window
        _case("window-wide", "attend", 2, 3001, 5000, 8, 1, 256, "f16", 16, 64, window=1024),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8])
    dtype, bits = rng.choice(["bf16", "bf16", "f16"]), rng.choice([8, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64) if b <= page]) if bits == 8 else 0
    form = rng.choice(["token", "draft", "prompt"])
    axes, inter, rotary, window = 1, False, 0, 0
    if op == "append":
        rotary = rng.choice([dim, dim, dim // 2, 0])
        inter = rng.random() < 0.4
        axes = rng.choice([1, 1, 2, 3]) if rotary else 1
    elif rng.random() < 0.25:
        window = _spread(rng, 16, 4096)
    if form == "prompt":
        total = _spread(rng, 200, 16384 if op == "append" else 6000)
        batch = _spread(rng, 1, 8)
        tokens = max(2, total // batch)
        context = tokens + rng.choice([0, _spread(rng, 1, 4000)])
        if op == "attend" and dim == 256:
            kv_heads = min(kv_heads, 2)
    else:
        tokens = 1 if form == "token" else rng.randint(2, 8)
        batch = _spread(rng, 1, 200)
        room = 4 * 131072 * 8 * 128 // 2  # at most half of the largest listed cache
        context = _spread(rng, 20, max(64, min(60000, room // (batch * kv_heads * dim))))
    context = max(context, tokens)
    return _case(None, op, batch, tokens, context, group * kv_heads, kv_heads, dim, dtype, bits, page, block,
                 rng.random() < 0.6, axes, inter, rotary, window)


def _lengths(case):
    """(new tokens, context with them) of every sequence: the case's own, whatever the seed."""
    r = random.Random(case["batch"] * 1000003 + case["context"] * 101 + case["tokens"])
    new, ctx = [], []
    for i in range(case["batch"]):
        n = case["tokens"] if i == 0 or not case["ragged"] else r.randint(0 if case["batch"] > 3 else 1, case["tokens"])
        longest = case["context"]
        new.append(n)
        ctx.append(longest if i == 0 else r.randint(max(n, longest // 4), longest))
    return new, ctx


def _sections(case):
    """How many pairs each axis has: the first the most."""
    half, axes = case["rotary"] // 2, case["axes"]
    rest = [half // (axes + 1) // 4 * 4 or 4] * (axes - 1)
    return [half - sum(rest)] + rest


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    new, ctx = _lengths(case)
    dt, page, d, hq, hk = TYPES[case["dtype"]], case["page"], case["dim"], case["heads"], case["kv_heads"]
    pages_of = [-(-c // page) for c in ctx]
    pages = sum(pages_of) + 3
    order = r.permutation(pages)
    table = np.zeros((case["batch"], max(max(pages_of), 1)), np.int32)
    at = 0
    for i, n in enumerate(pages_of):
        table[i, :n] = order[at:at + n]
        at += n
    total = sum(new)

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    s = {"case": case, "total": total, "most": max(new), "longest": max(ctx),
         "table": torch.from_numpy(table).to(DEV),
         "ctx": torch.tensor(ctx, dtype=torch.int32, device=DEV),
         "cu": torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)}
    # channels of different size, as keys and values have them
    wide = torch.exp(0.5 * normal(2, 1, hk, 1, d))
    if case["bits"] == 8:
        blocks = page // case["block"]
        s["k_scale"], s["v_scale"] = (
            ((torch.randint(-9, -5, (pages, hk, blocks), device=DEV, generator=g, dtype=torch.int32) + 127) << 23).view(torch.float32)
            for _ in "kv")
        # codes of both signs up to the largest
        s["k"], s["v"] = ((normal(pages, hk, page, d) * 100 * wide[i]).clamp(-448, 448).to(E4M3) for i in (0, 1))
    else:
        s["k"], s["v"] = ((normal(pages, hk, page, d) * wide[i]).to(dt) for i in (0, 1))
    s["q"] = (normal(total, hq, d) * (1 if case["op"] == "append" else 0.7)).to(dt)
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "append":
        s["new_k"], s["new_v"] = ((normal(total, hk, d) * wide[i, 0].transpose(0, 1)).to(dt) for i in (0, 1))
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = torch.arange(case["context"], device=DEV, dtype=torch.float64)[:, None] * torch.pow(
                10000.0, -torch.arange(half, device=DEV, dtype=torch.float64) / half)
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
            if case["axes"] > 1:
                s["positions"] = torch.from_numpy(r.randint(0, case["context"], (case["axes"], total)).astype(np.int32)).to(DEV)
    else:
        s["lse"] = torch.empty(total, hq, device=DEV)
    if own:  # descriptors of the tensors above (addresses, sizes, strides) that a program keeps beside its cache
        from asystem_amem_amd import kv
        s["cache"] = kv.Cache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
        s["batch"] = kv.Batch(s["table"], s["ctx"], tokens=total, cu_tokens=s["cu"] if case["ragged"] else None,
                              max_tokens=s["most"], max_context=s["longest"])
        if case["op"] == "attend":
            s["workspace"] = torch.empty(max(16, kv.attention_workspace(s["cache"], s["batch"], hq)), dtype=torch.uint8, device=DEV)
        elif case["rotary"]:
            s["rotation"] = kv.Rotation(s["cos"], s["sin"], sections=_sections(case), interleaved=case["interleaved"])
    return s


def work(case):
    new, ctx = _lengths(case)
    hq, hk, d, t = case["heads"], case["kv_heads"], case["dim"], sum(new)
    element = case["bits"] // 8
    if case["op"] == "append":
        moved = t * (2 * hk * d * (2 + element) + 2 * hq * d * 2)
        table = min(case["context"], t * case["axes"]) * case["rotary"] * 4
        return {"bytes": moved + table, "flops": t * (hk + hq) * case["rotary"] * 3}
    read, pairs = 0, 0
    for n, c in zip(new, ctx):
        if not n:
            continue
        w = case["window"] or c + 1
        first = max(0, c - n - w + 1)  # the first position that any of the rows sees
        read += (c - first) * hk * 2 * d * element
        if element == 1:
            read += (c - first) // case["block"] * hk * 8
        rows = np.arange(c - n, c, dtype=np.int64)
        pairs += int((np.minimum(rows + 1, w)).sum())
    return {"bytes": read + 2 * t * hq * d * 2 + t * hq * 4, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ plain forms

def _places(s):
    """Of every new token: its sequence and its position in the cache."""
    new = s["cu"][1:] - s["cu"][:-1]
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), new, output_size=s["total"])
    pos = s["ctx"][seq] - new[seq] + torch.arange(s["total"], device=DEV) - s["cu"][seq]
    return seq, pos


def _angles(s, pos, kind):
    """cos and sin of every (token, pair)."""
    case = s["case"]
    half = case["rotary"] // 2
    if case["axes"] == 1:
        return s["cos"][pos].to(kind), s["sin"][pos].to(kind)
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEV), torch.tensor(_sections(case), device=DEV), output_size=half)
    row = s["positions"][axis].t().long()  # token, pair
    pair = torch.arange(half, device=DEV)
    return s["cos"][row, pair].to(kind), s["sin"][row, pair].to(kind)


def _rotated(case, x, cos, sin):
    if not case["rotary"]:
        return x
    r = case["rotary"]
    turn, keep = x[..., :r], x[..., r:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if case["interleaved"] else (turn[..., :r // 2], turn[..., r // 2:])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, b * c + a * s
    turn = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turn, keep), -1)


def _power(e):
    """2 ** e in 64 bits, exactly, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _to_grid(x):
    """The nearest e4m3 value, ties to even, of what is at most 448 in size; anything that is not finite becomes NaN."""
    _, e = torch.frexp(x)
    step = _power((e - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, torch.nan)


def _plain_append(s):
    case = s["case"]
    seq, pos = _places(s)
    page = case["page"]
    where, slot = s["table"][seq, pos // page].long(), pos % page
    eight = case["bits"] == 8
    kind = torch.float64 if eight else torch.float32  # a code may hang on the last bit of a rotated key
    cos, sin = _angles(s, pos, torch.float32) if case["rotary"] else (None, None)
    q = _rotated(case, s["q"].float(), cos, sin).to(s["q"].dtype)
    if eight and case["rotary"]:
        cos, sin = cos.double(), sin.double()
    k, v = _rotated(case, s["new_k"].to(kind), cos, sin), s["new_v"].to(kind)
    if not eight:
        s["k"][where, :, slot], s["v"][where, :, slot] = k.to(s["k"].dtype), v.to(s["v"].dtype)
        return {"k": s["k"], "v": s["v"], "q": q}
    # 8 bits: all blocks that a new token falls into, [block][head][slot][dim]
    size = case["block"]
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    first = s["ctx"].long() - new
    n = (s["most"] - 1) // size + 2
    start = (first // size * size)[:, None] + torch.arange(n, device=DEV) * size
    touched = (start < s["ctx"][:, None]) & (new[:, None] > 0)
    at, which = torch.nonzero(touched, as_tuple=True)
    start = start[at, which]
    where, slot = s["table"][at, start // page].long(), start % page
    p = start[:, None] + torch.arange(size, device=DEV)
    fresh = (p >= first[at, None]) & (p < s["ctx"][at, None])
    token = (s["cu"][at, None] + p - first[at, None]).clamp(0, s["total"] - 1)
    begun = fresh[:, 0]
    slots = slot[:, None] + torch.arange(size, device=DEV)
    for values, codes, scales in ((k, s["k"], s["k_scale"]), (v, s["v"], s["v_scale"])):
        x = values[token].transpose(1, 2)  # block, head, slot, dim
        size_of = torch.where(fresh[:, None, :, None] & torch.isfinite(x), x.abs(), 0.0).amax((2, 3))
        m, e = torch.frexp(size_of)
        e = torch.where(size_of > 0, e - 9 + (m > 0.875), -64).clamp(-64, 119)
        need = _power(e)
        old = scales[where, :, slot // size].double()
        scale = torch.where(begun[:, None], need, torch.maximum(old, need))
        held = codes[where[:, None], :, slots].transpose(1, 2).double()
        held = _to_grid(held * (old / scale)[..., None, None])
        x = torch.where(fresh[:, None, :, None], _to_grid(x / scale[..., None, None]), held)
        keep = codes[where[:, None], :, slots]  # slots behind the new ones stay as they were
        x = torch.where((p < s["ctx"][at, None])[:, :, None, None], x.transpose(1, 2).float().to(E4M3).view(torch.uint8), keep.view(torch.uint8))
        codes.view(torch.uint8)[where[:, None], :, slots] = x
        scales[where, :, slot // size] = scale.float()
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"], "q": q}


def _plain_attend(s):
    case = s["case"]
    d, hk, page = case["dim"], case["kv_heads"], case["page"]
    group, batch, most = case["heads"] // hk, case["batch"], s["most"]
    table = s["table"].long()

    def gathered(codes, scales):
        x = codes[table].float()  # sequence, page, head, slot, dim
        if scales is not None:
            x = x * torch.repeat_interleave(scales[table], case["block"], -1)[..., None]
        return x.transpose(1, 2).reshape(batch, hk, -1, d)

    new = (s["cu"][1:] - s["cu"][:-1]).long()
    token = (s["cu"][:-1, None] + torch.arange(most, device=DEV)).clamp(max=s["total"] - 1)
    q = s["q"].float()[token]  # sequence, row, head, dim
    q = q.view(batch, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, d)
    keys = gathered(s["k"], s.get("k_scale"))
    scores = (q @ keys.transpose(-1, -2)) * d ** -0.5
    del keys
    length = scores.shape[-1]
    p = torch.arange(length, device=DEV)
    row = (s["ctx"].long() - new)[:, None] + torch.arange(most, device=DEV)
    seen = (p <= row[..., None]) & (p < s["ctx"][:, None, None])
    if case["window"]:
        seen &= p > row[..., None] - case["window"]
    scores = scores.view(batch, hk, group, most, length).masked_fill_(~seen[:, None, None], -torch.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    scores = scores.sub_(m).exp_()
    total = scores.sum(-1, keepdim=True)
    lse = torch.log(total) + m
    values = gathered(s["v"], s.get("v_scale"))
    out = scores.view(batch, hk, group * most, length) @ values
    out = out.view(batch, hk, group, most, d) / torch.where(total > 0, total, 1.0)
    seq, pos = _places(s)
    at = pos - (s["ctx"].long() - new)[seq]
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, hk * group, d)[seq, at].to(s["q"].dtype)
    lse = lse.squeeze(-1).permute(0, 3, 1, 2).reshape(batch, most, hk * group)[seq, at]
    return {"out": out, "lse": lse}


def run(s):
    case = s["case"]
    if not own:
        return _plain_append(s) if case["op"] == "append" else _plain_attend(s)
    from asystem_amem_amd import kv
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "append":
        kv.append(s["cache"], s["batch"], s["new_k"], s["new_v"], s["q"], s["out"], rotation=s.get("rotation"),
                  positions=s.get("positions"), stream=stream)
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]} if case["bits"] == 8 else {}
        return {"k": s["k"], "v": s["v"], **scales, "q": s["out"]}
    kv.attention(s["cache"], s["batch"], s["q"], s["out"], lse=s["lse"], scale=case["dim"] ** -0.5, causal=True,
                 window=case["window"], workspace=s["workspace"], stream=stream)
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits

def _near(x):
    """Nearest e4m3 value by its definition: three bits behind the leading one, none smaller than 2^-9."""
    size = np.abs(x)
    _, e = np.frexp(size)  # size = m * 2 ** e with m in [1/2, 1)
    unit = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(x / unit) * unit


def _exact_append(case, s):
    new, ctx = _lengths(case)
    r, d, page, size = case["rotary"], case["dim"], case["page"], case["block"]
    table = s["table"].cpu().numpy()

    def turned(x, rows):
        """x [token][head][dim] turned by the angles of rows [token][pair]."""
        y = x.double().cpu().numpy()
        if not r:
            return y
        i = np.arange(r // 2)
        one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        c, t = (s[n].double().cpu().numpy()[rows, i][:, None] for n in ("cos", "sin"))
        a, b = y[..., one].copy(), y[..., two].copy()
        y[..., one] = a * c - b * t
        y[..., two] = b * c + a * t
        return y

    rows = None
    if r:
        if case["axes"] == 1:
            rows = np.concatenate([np.arange(c - n, c) for n, c in zip(new, ctx)])[:, None] + np.zeros(r // 2, np.int64)
        else:
            given = s["positions"].cpu().numpy()
            rows = np.concatenate([np.repeat(given[a][:, None], n, 1) for a, n in enumerate(_sections(case))], 1)
    k, v, q = turned(s["new_k"], rows), s["new_v"].double().cpu().numpy(), turned(s["q"], rows)
    out = {"q": torch.from_numpy(q)}
    for name, x in (("k", k), ("v", v)):
        held = s[name].double().cpu().numpy()
        scales = s[name + "_scale"].double().cpu().numpy() if size else None
        base = 0
        for i, (n, c) in enumerate(zip(new, ctx)):
            p = c - n
            while p < c:  # page by page, or block by block
                unit = size or page
                stop = min(c, (p // unit + 1) * unit)
                where, slot = table[i, p // page], p % page
                part = x[base + p - (c - n):base + stop - (c - n)].transpose(1, 0, 2)  # head, slot, dim
                if size:
                    b = slot // size
                    most = np.abs(part).max((1, 2))
                    need = np.full(most.shape, 2.0 ** -64)
                    for e in range(-64, 119):
                        need = np.where(most > 448 * 2.0 ** e, 2.0 ** (e + 1), need)
                    old = scales[where, :, b].copy()
                    scale = need if slot % size == 0 else np.maximum(old, need)
                    earlier = held[where, :, b * size:slot]
                    held[where, :, b * size:slot] = _near(earlier * (old / scale)[:, None, None])
                    part = _near(part / scale[:, None, None])
                    scales[where, :, b] = scale
                held[where, :, slot:slot + stop - p] = part
                p = stop
            base += n
        out[name] = torch.from_numpy(held)
        if size:
            out[name + "_scale"] = torch.from_numpy(scales)
    return out


def _exact_attend(case, s):
    new, ctx = _lengths(case)
    d, hk, page = case["dim"], case["kv_heads"], case["page"]
    group = case["heads"] // hk
    out = torch.zeros(s["total"], case["heads"], d, dtype=torch.float64, device=DEV)
    lse = torch.full((s["total"], case["heads"]), -torch.inf, dtype=torch.float64, device=DEV)
    base = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        p = torch.arange(c, device=DEV)
        where, slot = s["table"][i, p // page].long(), p % page
        for h in range(hk if n else 0):
            k, v = s["k"][where, h, slot].double(), s["v"][where, h, slot].double()
            if case["block"]:
                k *= s["k_scale"][where, h, slot // case["block"]].double()[:, None]
                v *= s["v_scale"][where, h, slot // case["block"]].double()[:, None]
            at = torch.arange(c - n, c, device=DEV)[:, None]
            hidden = p > at
            if case["window"]:
                hidden |= p <= at - case["window"]
            for j in range(h * group, (h + 1) * group):
                x = s["q"][base:base + n, j].double() @ k.t() / d ** 0.5
                x[hidden] = -torch.inf
                lse[base:base + n, j] = torch.logsumexp(x, -1)
                out[base:base + n, j] = torch.softmax(x, -1) @ v
        base += n
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attend(case, s)
