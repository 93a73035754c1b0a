"""Attention over a paged key/value cache on the GPU where tiles, masks, scales and lengths meet badly; against the restatement in 64
bits and at the tolerances of test_gpu_kv.py."""
import ctypes as C

import numpy as np
import pytest

from asystem_amem_amd import kv
from tests import kv_oracle as O
from tests.kv_case import KINDS, Arena, Case
from tests.test_gpu_kv import TYPES, check_attend, poison

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena(gpu):
    a = Arena(gpu)
    yield a
    a.free()


@pytest.fixture(autouse=True)
def _fresh_arena(request):
    if "arena" in request.fixturenames:
        request.getfixturevalue("arena").reset()


def bad_patterns(kind, eight):
    """NaN and infinity (e4m3 has none: NaN)."""
    return (0x7F, 0x7F) if eight else (0x7FC0, 0x7F80) if kind == "bf16" else (0x7E00, 0x7C00)


@pytest.mark.parametrize("kind,eight", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,at", [(0, 500), (0, 430), (200, 300), (200, 650)])
def test_visible_infinities_and_nan_reach_every_row(arena, dim, kind, eight, window, at):
    """Values that are not finite in tiles that some waves of a workgroup see whole and others in part, or not at all."""
    nan, inf = bad_patterns(kind, eight)
    for bad in (nan, inf):
        case = Case(arena, [(300, 700)], dim=dim, q_heads=2, kv_heads=2, kind=kind, eight=eight, page=16, block=16, seed=31)
        poison(case, 0, at, v=bad)
        case.v[case.table[0, (at + 3) // 16], 1, (at + 3) % 16, 5] = nan     # one value of one head
        case.upload()
        got, _ = check_attend(case, case.rows(2), window=window)
        rows = O.decode(got, kind)
        seen = case.visible(0, True, window)[:, at]
        assert 0 < seen.sum() < 300
        assert not np.isfinite(rows[seen]).any() and np.isfinite(rows[~seen, 0]).all()
        arena.reset()


@pytest.mark.parametrize("kind,eight", TYPES)
def test_visible_nan_in_the_largest_workgroups(arena, kind, eight):
    """Enough prompts to fill the chip with eight waves of 32 rows each, a long one among them."""
    lengths = [(40, 40 + i % 50) for i in range(70)]
    lengths[3] = (300, 700)
    case = Case(arena, lengths, dim=128, q_heads=8, kv_heads=8, kind=kind, eight=eight, page=16, block=16, seed=32)
    nan, inf = bad_patterns(kind, eight)
    poison(case, 3, 500, v=nan)
    poison(case, 3, 420, v=inf)
    case.upload()
    check_attend(case, case.rows(8), sequences=[0, 3, 69])


@pytest.mark.parametrize("most", [1, 200], ids=["few rows", "many rows"])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("cu", [(0, 8, 15, 16, 16, 11, 14), (0, 16, 2, 16, 3, 9, 5), (7, 5, 3, 16, -4, 1 << 30, 2)])
def test_offsets_that_do_not_ascend_stay_inside_the_tensors(arena, cu, eight, most):
    """What lies around the result and lse keeps its bytes; which rows get what is not defined."""
    case = Case(arena, [(8, 30), (7, 20), (1, 20), (0, 20), (0, 9), (0, 20)], dim=128, q_heads=8, kv_heads=2, eight=eight, page=16, seed=33)
    assert case.tokens == 16
    case.cu, case.max_tokens = np.array(cu, np.int32), min(most, 16)
    case.upload()
    q, guard = case.rows(8), 1 << 16
    n = C.c_uint64()
    assert case.lib.amem_kv_attention_workspace(C.byref(case.cache), C.byref(case.batch), 8, C.byref(n)) == 0
    out, lse = arena.blank(q.nbytes + 2 * guard), arena.blank(16 * 8 * 4 + 2 * guard)
    args = kv.AttentionArgs(arena.put(q), out + guard, lse + guard, arena.blank(n.value), n.value, 1024, 128, 1024, 128, 0.1, KINDS["bf16"], 8, 1, 0, 0)
    assert case.lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(args), None) == 0
    for at, size in ((out, q.nbytes), (lse, 16 * 8 * 4)):
        x = arena.read(at, (size + 2 * guard,), np.uint8)
        assert (x[:guard] == 0xA5).all() and (x[guard + size:] == 0xA5).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30])
def test_the_widest_windows(arena, window, causal):
    """They hide nothing, from rows at negative positions neither."""
    for lengths in ([(4, 2), (1, 1300), (3, 1)], [(70, 33), (40, 1300), (300, 280)]):
        case = Case(arena, lengths, dim=64, q_heads=4, kv_heads=2, page=16, seed=34).upload()
        check_attend(case, case.rows(4), causal, window)
        arena.reset()
