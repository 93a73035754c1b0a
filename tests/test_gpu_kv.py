"""The operators on a paged key/value cache on the GPU, through the C ABI, against a plain restatement in 64 bits.

Tolerances, from the number formats alone:
  append, 16 bits: a rotated element is a c - b s with products and sum in 32 bits (2^-24 each, relative to |a c| + |b s|),
  then rounded once, off by at most half a step (2^-8 bf16, 2^-11 fp16, relative) or half the smallest fp16 step.
  append, 8 bits: codes and scales are the definition's, bit for bit.
  attention: the weights are rounded to 16 bits before they meet the values (half a step: 2^-8 where values are bf16, 2^-11 where
  they are fp16 or e4m3), relative to sum w |v|; scores are sums of dim products in 32 bits, off by at most dim * 2^-23 of the
  largest sum |q k| scale, which weights see as a factor; exp, sums and quotient add 2^-18; the result is rounded once.
"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from asystem_amem_amd import binding as B
from asystem_amem_amd import kv
from tests import kv_oracle as O
from tests.kv_case import KINDS, Arena, Case

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def arena(gpu):
    a = Arena(gpu)
    yield a
    a.free()


@pytest.fixture(autouse=True)
def _fresh_arena(request):
    if "arena" in request.fixturenames:
        request.getfixturevalue("arena").reset()




# ------------------------------------------------------------------------------------------------ append

def run_append(case, k, v, q=None, rotary=0, interleaved=False, sections=None, positions=None, rows=None, expect=0, in_place=False):
    """Calls the operator; returns q_out. cos and sin are kept on the case for the oracle."""
    a = case.arena
    rows = rows or max(1, case.max_context)
    r = np.random.RandomState(99)
    angle = r.uniform(-50, 50, (rows, max(rotary // 2, 1)))
    case.cos, case.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    h, d, kind = case.kv_heads, case.dim, KINDS[case.kind]
    qh = q.shape[1] if q is not None else 0
    dq = a.put(q) if q is not None else 0
    dqo = dq if in_place else a.blank(q.nbytes) if q is not None else 0
    args = kv.AppendArgs(a.put(k), a.put(v), dq, dqo, a.put(case.cos) if rotary else 0, a.put(case.sin) if rotary else 0,
                         a.put(positions) if positions is not None else 0, h * d, d, h * d, d, qh * d, d, qh * d, d, case.tokens, kind, qh,
                         rotary, int(interleaved), rows, len(sections) if sections else 1)
    if sections:
        args.sections = (C.c_int32 * 4)(*(list(sections) + [0] * (4 - len(sections))))
    assert case.lib.amem_kv_append(C.byref(case.cache), C.byref(case.batch), C.byref(args), None) == expect
    case.args = args
    return a.read(dqo, q.shape, np.uint16) if q is not None else None


def expected_append(case, k, v, q, rotary, interleaved, sections=None, positions=None):
    """What run_append should have made of the case's cache, in place (codes and scales, or 64-bit values before their
    rounding in a dict), and q."""
    ek, ev = {}, {}
    cos, sin = case.cos.astype(np.float64), case.sin.astype(np.float64)
    eq = O.decode(q, case.kind) if q is not None else None
    dk, dv = O.decode(k, case.kind), O.decode(v, case.kind)
    for s, (n, c) in enumerate(case.lengths):
        for j in range(n):
            row, p = case.cu[s] + j, c - n + j
            at = positions[:, row] if positions is not None else None
            dk[row] = O.turn(dk[row], p, cos, sin, rotary, interleaved, sections, at)
            if q is not None:
                eq[row] = O.turn(eq[row], p, cos, sin, rotary, interleaved, sections, at)
        first = c - n
        if not case.eight:
            for j in range(n):
                p = c - n + j
                if p < 0:
                    continue
                page, slot = case.table[s, p // case.page], p % case.page
                ek[page, slot], ev[page, slot] = dk[case.cu[s] + j], dv[case.cu[s] + j]
            continue
        p = max(first, 0)
        while p < c:
            stop = min(c, (p // case.block + 1) * case.block)
            page, slot = case.table[s, p // case.page], p % case.page
            b = slot // case.block
            for new, codes, scales in ((dk, case.k, case.k_scale), (dv, case.v, case.v_scale)):
                for h in range(case.kv_heads):
                    x = new[case.cu[s] + p - first:case.cu[s] + stop - first, h]
                    need = O.need_of(np.abs(x[np.isfinite(x)]).max(initial=0))
                    old = float(scales[page, h, b])
                    if not (old > 0 and np.isfinite(old)):
                        old = need
                    scale = need if slot % case.block == 0 else max(old, need)
                    held = codes[page, h, b * case.block:slot]
                    if scale > old:
                        codes[page, h, b * case.block:slot] = O.e4m3_code(O.E4M3[held] * (old / scale))
                    codes[page, h, slot:slot + stop - p] = O.e4m3_code(x / scale)
                    scales[page, h, b] = scale
            p = stop
    return ek, ev, eq


def near(got, want, kind, slack=0.0):
    """got: 16-bit patterns; want: 64 bits; slack: error before the rounding."""
    x = O.decode(got, kind)
    same = (np.isnan(x) & np.isnan(want)) | (x == want)
    with np.errstate(invalid="ignore"):
        ok = np.abs(x - want) <= (HALF[kind] * np.abs(want) + TINY[kind]) * (1 + 2.0 ** -9) + slack
    assert (same | ok).all(), np.abs(x - want)[~(same | ok)].max()


def check_append(case, k, v, q=None, rotary=0, interleaved=False, sections=None, positions=None, in_place=False):
    before_k, before_v = case.k.copy(), case.v.copy()
    got_q = run_append(case, k, v, q, rotary, interleaved, sections, positions, in_place=in_place)
    ek, ev, eq = expected_append(case, k, v, q, rotary, interleaved, sections, positions)
    gk, gv, gks, gvs = case.download()
    slack = 3 * 2.0 ** -24 * 2 * 8       # |a c| + |b s| is at most 8 for what rows() makes
    if case.eight:
        assert np.array_equal(gks, case.k_scale) and np.array_equal(gvs, case.v_scale)
        assert np.array_equal(gk, case.k) and np.array_equal(gv, case.v)
    else:
        touched = np.zeros((case.pages, case.page), bool)
        for (page, slot), want in ek.items():
            near(gk[page, :, slot], want, case.kind, slack)
            assert np.array_equal(O.decode(gv[page, :, slot], case.kind), ev[page, slot])
            touched[page, slot] = True
        keep = ~touched[:, None, :, None] & np.ones(gk.shape, bool)
        assert np.array_equal(gk[keep], before_k[keep]) and np.array_equal(gv[keep], before_v[keep])
    if q is not None:
        n = case.cu[-1]
        near(got_q[:n], eq[:n], case.kind, slack)
        if not in_place:
            assert (got_q[n:] == 0xA5A5).all()


LENGTHS = {
    "one": [(1, 1)],
    "one far": [(1, 300)],
    "starts a block": [(1, 33), (1, 17), (1, 129)],
    "batch": [(1, c) for c in (1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 200, 333)],
    "drafts": [(5, 5), (3, 20), (8, 71), (1, 64), (4, 18)],
    "prompts": [(100, 100), (33, 50), (64, 64), (0, 40), (1, 7), (129, 400)],
    "empty ones": [(0, 0), (0, 9), (3, 3), (0, 0), (2, 40), (0, 0)],
}


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("name", LENGTHS)
def test_append_lengths(arena, name, eight):
    case = Case(arena, LENGTHS[name], dim=128, kv_heads=2, eight=eight, page=32, block=16, seed=3).upload()
    check_append(case, case.rows(2), case.rows(2), case.rows(4), rotary=128)


@pytest.mark.parametrize("dim,rotary,interleaved,sections,kind,eight,page,block", [
    (64, 64, True, None, "f16", False, 1, 0),
    (64, 32, False, None, "bf16", True, 16, 16),
    (128, 0, False, None, "f16", True, 64, 64),
    (128, 48, True, None, "bf16", False, 2, 0),
    (128, 128, False, (16, 24, 24), "bf16", True, 128, 128),
    (128, 128, True, (64, 0), "f16", False, 64, 0),
    (256, 256, False, (50, 41, 30, 7), "f16", True, 64, 32),
    (256, 16, False, None, "bf16", False, 1024, 0),
    (256, 256, True, (0, 128), "bf16", True, 32, 32),
])
def test_append_rotations(arena, dim, rotary, interleaved, sections, kind, eight, page, block):
    lengths = [(7, 7), (1, 50), (40, 77), (0, 3)]
    case = Case(arena, lengths, dim=dim, kv_heads=3, kind=kind, eight=eight, page=page, block=block, seed=5).upload()
    positions = case.r.randint(0, 77, (len(sections), case.tokens)).astype(np.int32) if sections else None
    check_append(case, case.rows(3), case.rows(3), case.rows(6), rotary, interleaved, sections, positions)


def test_append_without_queries_and_in_place(arena):
    case = Case(arena, [(3, 9), (2, 2)], eight=True, seed=1).upload()
    check_append(case, case.rows(2), case.rows(2))
    case = Case(arena, [(3, 9), (2, 2)], seed=2).upload()
    check_append(case, case.rows(2), case.rows(2), case.rows(5), rotary=128, in_place=True)


@pytest.mark.parametrize("eight", [False, True])
def test_append_slot_major_strides_uniform_and_rows_behind(arena, eight):
    case = Case(arena, [(2, 19), (2, 2), (2, 64)], kv_heads=3, eight=eight, page=32, block=32, slot_major=True, seed=4, uniform=True).upload()
    check_append(case, case.rows(3), case.rows(3), case.rows(3), rotary=64)
    case = Case(arena, [(2, 19), (4, 6)], eight=eight, page=32, block=32, seed=4, behind=5).upload()
    check_append(case, case.rows(2), case.rows(2), case.rows(4), rotary=64)


def test_append_one_by_one_then_again(arena):
    """A block filled token by token, each larger than the last: earlier codes follow the growing scale. Then the same
    positions once more, as after drafted tokens were turned down."""
    case = Case(arena, [(1, 1)], eight=True, page=16, block=16, seed=6).upload()
    order = list(range(1, 20)) + [18, 19, 20, 17]
    for step, c in enumerate(order):
        case.lengths, case.context = [(1, c)], np.array([c], np.int32)
        if c > case.page * 1 and case.table[0, 1] < 0:
            case.table[0, 1] = [x for x in range(case.pages) if x != case.table[0, 0]][0]
            arena.write(case.d_table, case.table)
        arena.write(case.d_context, case.context)
        case.batch.max_context = c
        size = 2.0 ** (step % 11 - 5)
        check_append(case, case.rows(2, size), case.rows(2, size), rotary=128)


def test_append_all_codes_and_borders(arena):
    """Values on and next to every rounding border of e4m3, sizes at the border of a scale, tiny and huge, zeros."""
    grid = np.unique(O._SIZES)
    mid = (grid[1:] + grid[:-1]) / 2
    values = np.concatenate([grid, mid, [448]])
    for seed, top in enumerate((448.0, 449.0, 447.0, 2.0 ** -60, 2.0 ** -66, 0.0, 2.0 ** 126)):
        case = Case(arena, [(16, 16)], dim=128, kv_heads=1, eight=True, seed=seed).upload()
        x = case.r.choice(values, (16, 1, 128)) * case.r.choice([-1, 1], (16, 1, 128)) / 448 * top
        x[0, 0, 0] = top
        rows = O.encode(x, "bf16")
        check_append(case, rows, rows)
        arena.reset()


def test_append_not_finite(arena):
    for eight in (False, True):
        case = Case(arena, [(4, 20)], eight=eight, seed=8).upload()
        k, v = case.rows(2), case.rows(2)
        for x in (k, v):
            x[0, 0, 3], x[1, 1, 100], x[2, 0, 5] = 0x7F80, 0xFF80, 0x7FC1       # inf, -inf, NaN
            x[3, 1] = 0x7FC0
        run_append(case, k, v)
        expected = expected_append(case, k, v, None, 0, False)
        gk, gv, gks, gvs = case.download()
        if eight:
            assert np.array_equal(gks, case.k_scale) and np.array_equal(gvs, case.v_scale)
            for got, want in ((gk, case.k), (gv, case.v)):
                nan = np.isnan(O.E4M3[want])
                assert nan.sum() >= 131 and np.array_equal(nan, np.isnan(O.E4M3[got])) and np.array_equal(got[~nan], want[~nan])
        else:
            for (page, slot), want in expected[1].items():
                assert np.array_equal(O.decode(gv[page, :, slot], "bf16"), want, equal_nan=True)


def test_append_bad_scales_count_as_none(arena):
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        case = Case(arena, [(3, 9)], eight=True, seed=9)
        case.k_scale[:] = bad
        case.v_scale[:] = bad
        case.upload()
        touched = case.table[0, 0]
        k, v = case.rows(2), case.rows(2)
        run_append(case, k, v)
        expected_append(case, k, v, None, 0, False)
        gk, gv, gks, gvs = case.download()
        assert np.array_equal(gk, case.k) and np.array_equal(gv, case.v)
        assert np.array_equal(gks[touched], case.k_scale[touched]) and np.array_equal(gvs[touched], case.v_scale[touched])


@pytest.mark.parametrize("eight", [False, True])
def test_append_out_of_range_writes_nothing(arena, eight):
    """Contexts above the limit or negative, pages that are none, rows of the table that are none: those sequences and tokens
    alone are left out; so are tokens at negative positions."""
    case = Case(arena, [(2, 20), (2, 20), (2, 20), (3, 20), (5, 3)], eight=eight, page=16, seed=10)
    case.context[0], case.context[1] = 10 ** 6, -4
    case.table[2, 1], case.table[3, 1] = case.pages, -1
    case.max_context = 32
    case.upload()
    k, v, q = case.rows(2), case.rows(2), case.rows(4)
    got = run_append(case, k, v, q, rotary=64, rows=18)      # the table ends inside the positions of some
    case.lengths = [(0, 0), (0, 0), (0, 0), (0, 0), (5, 3)]
    case.cu = np.array([0, 0, 0, 0, 9, 14], np.int32)
    ek, ev, eq = expected_append(case, k, v, None, 64, False)
    gk, gv, gks, gvs = case.download()
    if eight:
        assert np.array_equal(gk, case.k) and np.array_equal(gv, case.v) and np.array_equal(gks, case.k_scale)
    else:
        for (page, slot), want in ev.items():
            assert np.array_equal(O.decode(gv[page, :, slot], case.kind), want)
            gv[page, :, slot] = case.v[page, :, slot]
        assert np.array_equal(gv, case.v)
    # sequences 0 and 1 have no positions, 2 has 18 and 19, 3 has 17 to 19: of all these only 17 is in the table
    turned = O.decode(got, case.kind)[:9, :, :64]
    assert np.isnan(np.delete(turned, 6, 0)).all() and np.isfinite(turned[6]).all()
    assert np.array_equal(got[:9, :, 64:], q[:9, :, 64:])


# ------------------------------------------------------------------------------------------------ attention

def run_attend(case, q, causal=True, window=0, scale=None, lse=True, expect=0, workspace=None, q_layout=None):
    a, d, h = case.arena, case.dim, q.shape[1]
    n = C.c_uint64()
    assert case.lib.amem_kv_attention_workspace(C.byref(case.cache), C.byref(case.batch), h, C.byref(n)) == 0
    ws = a.blank(n.value) if workspace is None else workspace
    out, dl = a.blank(q.nbytes), a.blank(case.tokens * h * 4) if lse else 0
    token, head = (h * d, d) if q_layout is None else (d, case.tokens * d)       # head-major rows
    dq = a.put(q if q_layout is None else q.transpose(1, 0, 2))
    args = kv.AttentionArgs(dq, out, dl, ws, n.value, token, head, token, head, d ** -0.5 if scale is None else scale, KINDS[case.kind], h,
                            int(causal), window, 0)
    assert case.lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(args), None) == expect
    case.args = args
    shape = (case.tokens, h, d) if q_layout is None else (h, case.tokens, d)
    got = a.read(out, shape, np.uint16)
    if q_layout is not None:
        got = got.transpose(1, 0, 2)
    return got, a.read(dl, (case.tokens, h), np.float32) if lse else None


def check_attend(case, q, causal=True, window=0, scale=None, sequences=None, q_layout=None):
    scale_ = case.dim ** -0.5 if scale is None else scale
    got, lse = run_attend(case, q, causal, window, scale, q_layout=q_layout)
    group = case.q_heads // case.kv_heads
    weight = HALF["f16"] if case.eight else HALF[case.kind]
    for s in range(len(case.lengths)) if sequences is None else sequences:
        n, c = case.lengths[s]
        if not n:
            continue
        rows = slice(case.cu[s], case.cu[s] + n)
        seen = case.visible(s, causal, window)
        for h in range(case.q_heads):
            k, v = case.gathered(s, h // group)
            out, l, size, top = O.attend(O.decode(q[rows, h], case.kind), k, v, scale_, seen)
            score = case.dim * 2.0 ** -23 * top + 2.0 ** -18
            with np.errstate(invalid="ignore"):
                slack = (weight + score)[:, None] * size + 2.0 ** -30 * np.abs(np.nan_to_num(v, posinf=0, neginf=0)).max(initial=0)
            near(got[rows, h], out, case.kind, slack)
            same = (lse[rows, h] == l) | (np.isnan(lse[rows, h]) & np.isnan(l))
            with np.errstate(invalid="ignore"):
                ok = np.abs(lse[rows, h] - l) <= score + 2.0 ** -22 * np.abs(l)
            assert (same | ok).all(), (s, h)
    n = case.cu[-1]
    assert (got[n:] == 0xA5A5).all() and (lse.view(np.uint32)[n:] == 0xA5A5A5A5).all()
    return got, lse


CONTEXTS = {
    "one": [(1, 1)],
    "short": [(1, c) for c in (1, 2, 3, 15, 16, 17, 31, 32, 33)],
    "tiles": [(1, c) for c in (63, 64, 65, 127, 128, 129, 255, 257, 511, 513)],
    "long": [(1, 5000), (1, 17), (1, 2049), (1, 1024)],
    "drafts": [(5, 5), (3, 130), (8, 71), (1, 300), (2, 2)],
    "rows": [(17, 17), (33, 100), (16, 16), (31, 64)],
    "prompts": [(100, 100), (130, 333), (64, 64), (0, 40), (1, 7), (257, 257)],
    "long prompt": [(300, 1300)],
    "empty": [(0, 0), (3, 3), (0, 12), (2, 0), (4, 2), (1, 0)],
}
TYPES = [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)]


@pytest.mark.parametrize("kind,eight", TYPES)
@pytest.mark.parametrize("name", CONTEXTS)
def test_attention_lengths(arena, name, kind, eight):
    case = Case(arena, CONTEXTS[name], dim=128, q_heads=8, kv_heads=2, kind=kind, eight=eight, page=32, block=16, seed=11).upload()
    check_attend(case, case.rows(8))


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kind,eight", TYPES)
@pytest.mark.parametrize("lengths", [[(1, 700), (1, 31)], [(4, 90), (6, 6)], [(90, 200), (150, 150)]], ids=["token", "draft", "prompt"])
def test_attention_dims(arena, lengths, kind, eight, dim):
    case = Case(arena, lengths, dim=dim, q_heads=4, kv_heads=2, kind=kind, eight=eight, page=16, block=16, seed=12).upload()
    check_attend(case, case.rows(4))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (3, 3), (7, 1), (12, 1), (32, 2), (40, 1), (14, 2)])
def test_attention_heads(arena, q_heads, kv_heads, eight):
    for lengths in ([(1, 150), (1, 90)], [(3, 70), (6, 200)], [(70, 100)]):
        case = Case(arena, lengths, dim=64, q_heads=q_heads, kv_heads=kv_heads, eight=eight, page=16, block=16, seed=13).upload()
        check_attend(case, case.rows(q_heads))
        arena.reset()


@pytest.mark.parametrize("page,block,eight", [(1, 0, False), (2, 0, False), (8, 0, False), (256, 0, False), (1024, 0, False),
                                              (16, 16, True), (128, 16, True), (128, 128, True), (1024, 64, True)])
def test_attention_pages(arena, page, block, eight):
    lengths = [(1, 130), (5, 261), (80, 90)]
    case = Case(arena, lengths, dim=128, q_heads=4, kv_heads=1, eight=eight, page=page, block=block, seed=14).upload()
    check_attend(case, case.rows(4))


@pytest.mark.parametrize("kind,eight", TYPES)
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 37), (False, 20), (True, 64), (True, 100000)])
def test_attention_masks(arena, causal, window, kind, eight):
    lengths = [(1, 300), (6, 90), (100, 260), (4, 2), (70, 33)]
    case = Case(arena, lengths, dim=64, q_heads=6, kv_heads=2, kind=kind, eight=eight, page=16, block=16, seed=15).upload()
    check_attend(case, case.rows(6), causal, window)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("causal,window", [(False, 0), (False, 20), (True, 20), (True, 700)])
def test_attention_masks_of_long_contexts(arena, causal, window, eight):
    """Contexts that are cut into stretches: a window bounds what a row sees only where the mask is causal."""
    for lengths in ([(1, 1500), (4, 900)], [(80, 1500)]):
        case = Case(arena, lengths, dim=64, q_heads=4, kv_heads=2, eight=eight, page=32, block=32, seed=26).upload()
        check_attend(case, case.rows(4), causal, window)
        arena.reset()


@pytest.mark.parametrize("eight", [False, True])
def test_attention_strides(arena, eight):
    for lengths in ([(1, 100), (1, 20)], [(50, 90), (2, 40)]):
        case = Case(arena, lengths, dim=128, q_heads=6, kv_heads=3, eight=eight, page=32, block=32, slot_major=True, seed=16, behind=3).upload()
        check_attend(case, case.rows(6), q_layout="head-major")
        arena.reset()
    case = Case(arena, [(2, 100), (2, 20), (2, 2)], dim=128, q_heads=6, kv_heads=3, eight=eight, page=32, block=32, seed=16, uniform=True).upload()
    check_attend(case, case.rows(6))


@pytest.mark.parametrize("kind,eight,dim", [("bf16", False, 128), ("f16", False, 64), ("bf16", True, 128), ("f16", True, 128), ("f16", True, 64)])
def test_attention_many_sequences(arena, kind, eight, dim):
    """Enough prompts to fill the chip with the largest workgroups; a long one among them, and ones with bad values and hidden NaN."""
    lengths = [(40, 40 + i % 50) for i in range(70)]
    lengths[3], lengths[9], lengths[50] = (300, 700), (0, 0), (65, 64)
    case = Case(arena, lengths, dim=dim, q_heads=8, kv_heads=8, kind=kind, eight=eight, page=16, block=16, seed=25)
    nan = 0x7F if eight else 0x7FC0 if kind == "bf16" else 0x7E00
    poison(case, 3, 500, k=nan)
    poison(case, 3, 650, v=nan)
    poison(case, 3, 699, v=nan)
    case.table[20, 1] = -1
    case.upload()
    got, lse = check_attend(case, case.rows(8), sequences=[0, 3, 9, 19, 50, 69])
    rows = O.decode(got, kind)[case.cu[20]:case.cu[21]]
    n, c = lengths[20]
    first = max(0, 16 - (c - n))
    assert np.isnan(rows[first:]).all() and np.isfinite(rows[:first]).all()


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1000), (False, 0)])
@pytest.mark.parametrize("dim,sequences,tokens,eight,uniform", [(256, 33, 40, False, True), (256, 33, 40, True, False), (128, 65, 40, True, True),
                                                                (128, 40, 130, False, True), (64, 100, 40, True, True)])
def test_attention_last_round_is_cut(gpu, dim, sequences, tokens, eight, uniform, causal, window):
    """More workgroups than fit at once, and a few more: those (the first sequences') are cut into stretches, the others are not."""
    big = Arena(gpu, 512 << 20)
    try:
        lengths = [(tokens, tokens + i % 50) for i in range(sequences)]
        lengths[0], lengths[1], lengths[sequences - 1] = (tokens, 1600), (tokens, 700), (tokens, 1100)
        if not uniform:
            lengths[2], lengths[5] = (3, 1500), (0, 9)
        case = Case(big, lengths, dim=dim, q_heads=8, kv_heads=8, eight=eight, page=32, block=32, uniform=uniform, seed=27).upload()
        got, lse = check_attend(case, case.rows(8), causal, window, sequences=[0, 1, 2, 3, 5, 6, sequences // 2, sequences - 1])
        assert np.isfinite(O.decode(got, case.kind)).all() and np.isfinite(lse).all()
    finally:
        big.free()


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1000), (False, 0)])
@pytest.mark.parametrize("dim,sequences,tokens,kind,eight,uniform", [(256, 33, 1, "bf16", False, True), (256, 65, 2, "f16", True, False), (128, 65, 1, "bf16", True, True),
                                                                     (128, 70, 3, "bf16", False, False), (64, 97, 1, "f16", False, True), (128, 33, 1, "bf16", True, True)])
def test_attention_last_round_of_few_rows_is_cut(gpu, dim, sequences, tokens, kind, eight, uniform, causal, window):
    big = Arena(gpu, 512 << 20)
    try:
        lengths = [(tokens, tokens + 7 * i % 200) for i in range(sequences)]
        lengths[0], lengths[1], lengths[sequences - 1] = (tokens, 2600), (tokens, 700), (tokens, 2100)
        if not uniform:
            lengths[2], lengths[5] = (1, 1500), (0, 9)
        case = Case(big, lengths, dim=dim, q_heads=16, kv_heads=8, kind=kind, eight=eight, page=32, block=32, uniform=uniform, seed=28).upload()
        got, lse = check_attend(case, case.rows(16), causal, window, sequences=[0, 1, 2, 3, 5, 6, sequences // 2, sequences - 1])
        assert np.isfinite(O.decode(got, case.kind)).all() and np.isfinite(lse).all()
    finally:
        big.free()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 8.0])
def test_attention_scales(arena, scale):
    """From weights that are all equal to a single one."""
    for eight in (False, True):
        case = Case(arena, [(1, 200), (40, 60), (3, 90)], dim=64, q_heads=4, kv_heads=2, eight=eight, page=16, seed=17).upload()
        check_attend(case, case.rows(4), scale=scale)
        arena.reset()


def poison(case, s, p, k=None, v=None):
    """Puts a bit pattern into the keys or values of a position."""
    page, slot = case.table[s, p // case.page], p % case.page
    if k is not None:
        case.k[page, :, slot] = k
    if v is not None:
        case.v[page, :, slot] = v


@pytest.mark.parametrize("kind,eight", TYPES)
@pytest.mark.parametrize("lengths", [[(1, 70)], [(6, 70)], [(80, 150)]], ids=["token", "draft", "prompt"])
def test_attention_hidden_infinities_and_nan(arena, lengths, kind, eight):
    """NaN and infinities behind the context, and at positions that some rows see and others do not."""
    nan, inf = (0x7F, 0x7F) if eight else ((0x7FC0, 0x7F80) if kind == "bf16" else (0x7E00, 0x7C00))
    n, c = lengths[0]
    case = Case(arena, lengths, dim=128, q_heads=4, kv_heads=2, kind=kind, eight=eight, page=32, seed=18)
    page, slot = case.table[0, c // case.page], c % case.page
    if page >= 0:
        case.k[page, :, slot:], case.v[page, :, slot:] = nan, inf
    if n > 3:
        poison(case, 0, c - 2, v=nan)                    # the last two rows see it
        poison(case, 0, c - 1, v=inf)
        poison(case, 0, c - 3, k=nan)
    if n > 60:
        case.v[case.table[0, (c - 40) // case.page], 1, (c - 40) % case.page, 5] = inf     # one value alone
    case.upload()
    got, lse = check_attend(case, case.rows(4))
    if n > 3:
        assert np.isfinite(O.decode(got, kind)[:n - 41]).all() and np.isnan(O.decode(got, kind)[n - 1]).any()
    # and in front of a window
    case = Case(arena, lengths, dim=128, q_heads=4, kv_heads=2, kind=kind, eight=eight, page=32, seed=19)
    poison(case, 0, 3, k=nan, v=nan)
    poison(case, 0, c - n - 5, v=inf)
    case.upload()
    check_attend(case, case.rows(4), window=9)
    check_attend(case, case.rows(4), window=c - 3)


def test_attention_infinite_scores(arena):
    """Keys of infinite size: NaN where the definition gives it, and no weight where the score is -infinity."""
    for lengths in ([(1, 80)], [(70, 80)]):
        case = Case(arena, lengths, dim=64, q_heads=2, kv_heads=1, page=16, seed=20)
        poison(case, 0, 5, k=0)
        case.k[case.table[0, 0], 0, 5, 0] = 0x7F80
        case.upload()
        q = case.rows(2)
        q[..., 0] = 0xBF80                                   # -1: that score is -infinity
        got, _ = check_attend(case, q)
        assert np.isfinite(O.decode(got, "bf16")).all()
        arena.reset()
        case = Case(arena, lengths, dim=64, q_heads=2, kv_heads=1, page=16, seed=20)
        case.k[:, :, :, 0] = 0x7F80
        case.upload()
        got, lse = check_attend(case, q)                     # nothing but -infinity
        assert (O.decode(got, "bf16") == 0).all() and (lse == -np.inf).all()
        arena.reset()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths", [[(1, 40), (1, 90), (1, 90), (1, 90)], [(2, 40), (70, 90), (5, 90), (40, 90)]], ids=["token", "prompt"])
def test_attention_out_of_range_gives_nan(arena, lengths, eight):
    case = Case(arena, lengths, dim=128, q_heads=4, kv_heads=2, eight=eight, page=16, seed=21)
    case.context[1] = 10 ** 7
    case.context[3] = -1
    case.table[2, 5] = case.pages + 3                        # positions 80 to 95
    case.max_context = 96
    case.upload()
    got, lse = check_attend(case, case.rows(4), sequences=[0])
    x = O.decode(got, case.kind)
    for s in (1, 3):
        assert np.isnan(x[case.cu[s]:case.cu[s + 1]]).all() and np.isnan(lse[case.cu[s]:case.cu[s + 1]]).all()
    n, c = case.lengths[2]
    first = max(0, 80 - (c - n))                             # rows at position 80 and behind
    rows = x[case.cu[2]:case.cu[3]]
    assert np.isnan(rows[first:]).all() and np.isfinite(rows[:first]).all()


def test_attention_same_bits_again_and_any_workspace(arena):
    case = Case(arena, [(1, 5000), (1, 300), (1, 2000)], dim=128, q_heads=8, kv_heads=2, eight=True, page=64, block=32, seed=22).upload()
    q = case.rows(8)
    one, l1 = run_attend(case, q)
    ws = arena.put(np.full(4 * Case_MiB, 0xFF, np.uint8))    # NaN patterns
    for _ in range(3):
        two, l2 = run_attend(case, q, workspace=ws)
        assert np.array_equal(one, two) and np.array_equal(l1, l2)


Case_MiB = 1 << 20


@pytest.mark.parametrize("eight", [False, True])
def test_max_tokens_is_a_guide(arena, eight):
    """Ragged rows with max_tokens too small, and too large: another kernel takes them, with the same definition."""
    for most, lengths in ((1, [(50, 90), (1, 30), (7, 7)]), (20, [(1, 30), (2, 90), (17, 40)]), (0, [(3, 9)])):
        case = Case(arena, lengths, dim=128, q_heads=8, kv_heads=2, eight=eight, page=16, seed=27)
        case.max_tokens = most
        case.upload()
        check_attend(case, case.rows(8))
        arena.reset()


@pytest.mark.parametrize("eight", [False, True])
def test_offsets_beyond_32_bits(gpu, arena, eight):
    """A cache whose pages are 2.25 GiB apart."""
    far = Arena(gpu, 10 << 30)
    try:
        for lengths in ([(1, 70), (2, 100)], [(90, 120), (1, 40)]):
            case = Case(arena, lengths, dim=128, q_heads=4, kv_heads=2, eight=eight, page=64, block=32, seed=28, spare_pages=0).upload()
            gap = 9 << 28
            assert 4 << 30 < (int(case.pages) - 1) * gap < 9 << 30
            element = 1 if eight else 2
            case.cache.k, case.cache.v, case.cache.page_stride = far.va, far.va + (1 << 28), gap // element

            def each(what):
                for i in range(case.pages):
                    what(i, far.va + i * gap, far.va + i * gap + (1 << 28))
            each(lambda i, k, v: (far.write(k, case.k[i]), far.write(v, case.v[i])))

            def download():
                k, v = np.empty_like(case.k), np.empty_like(case.v)

                def one(i, kp, vp):
                    k[i], v[i] = far.read(kp, k[i].shape, k.dtype), far.read(vp, v[i].shape, v.dtype)
                each(one)
                scales = tuple(arena.read(x, case.k_scale.shape, np.float32) for x in (case.d_ks, case.d_vs)) if eight else (None, None)
                return (k, v) + scales
            case.download = download
            check_append(case, case.rows(2), case.rows(2), case.rows(4), rotary=128)
            case.k, case.v = download()[:2]
            check_attend(case, case.rows(4))
            arena.reset()
    finally:
        far.free()


def test_append_then_attend_as_used(arena):
    """A conversation of two sequences: prompts, tokens one by one, drafted tokens of which some are taken back; the cache in 8
    bits. The attention is held to the cache as the definition of append leaves it."""
    case = Case(arena, [(70, 70), (20, 20)], dim=64, q_heads=4, kv_heads=2, eight=True, page=32, block=16, seed=23, spare_pages=8)
    free = [p for p in range(case.pages) if p not in case.table]
    table = np.full((2, 8), -1, np.int32)
    table[:, :case.table_pages] = case.table
    for s in range(2):
        for i in range(8):
            if table[s, i] < 0 and i < 5 and free:
                table[s, i] = free.pop()
    case.table, case.table_pages = table, 8
    case.upload()
    for step in ([(70, 70), (20, 20)], [(1, 71), (1, 21)], [(4, 75), (4, 25)], [(3, 75), (1, 23)], [(0, 75), (10, 33)], [(1, 76), (1, 34)]):
        case.lengths = step
        case.tokens = sum(n for n, _ in step)
        case.cu, case.context = np.concatenate([[0], np.cumsum([n for n, _ in step])]).astype(np.int32), np.array([c for _, c in step], np.int32)
        arena.write(case.d_cu, case.cu)
        arena.write(case.d_context, case.context)
        case.batch.tokens, case.batch.max_tokens, case.batch.max_context = case.tokens, max(n for n, _ in step), 160
        check_append(case, case.rows(2), case.rows(2), case.rows(4), rotary=64)
        check_attend(case, case.rows(4))


def test_refused_while_paused_and_whole_after_resume(gpu, fresh):
    """The cache in tracked memory: operators that were enqueued have run when the pause begins, calls are refused while its memory
    is gone, and after the resume the same attention has the same bits."""
    lib = fresh
    arena = Arena(lib, 16 * (1 << 20))
    try:
        assert lib.amem_add_alloc_info(arena.va, arena.alloc, B.TYPE_LOCAL, 0, arena.handle, -1, 0, None, B.CALLER_P2P) == 0
        case = Case(arena, [(1, 500), (40, 70)], dim=128, q_heads=4, kv_heads=2, eight=True, page=32, block=32, seed=24).upload()
        k, v, q = case.rows(2), case.rows(2), case.rows(4)
        run_append(case, k, v, q, rotary=128)
        app = case.args
        one, l1 = check_attend_after(case, q)
        att = case.args
        assert lib.amem_kv_append(C.byref(case.cache), C.byref(case.batch), C.byref(app), None) == 0     # the same rows again, unwaited
        assert lib.ncclPause(None) == 0
        assert lib.amem_kv_append(C.byref(case.cache), C.byref(case.batch), C.byref(app), None) == 1
        assert lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(att), None) == 1
        assert lib.ncclResume(None) == 0
        assert lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(att), None) == 0
        two = arena.read(att.out, one.shape, np.uint16)
        assert np.array_equal(one, two)
        assert lib.amem_del_alloc_info(arena.va, 0, 0) == 0
    finally:
        arena.free()


def check_attend_after(case, q):
    return run_attend(case, q)


def test_through_torch_streams_and_graphs():
    """The Python entry points on torch tensors, in a process of their own (torch brings a HIP runtime along, which has to be the
    only one): strided views, another stream than the tensors' own, refusals, captured graphs replayed between eager work."""
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "tests", "kv_torch_worker.py")], cwd=ROOT, capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert "kv torch worker: all done" in r.stdout
