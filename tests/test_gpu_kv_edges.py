"""Attention over a paged key/value cache on the GPU where tiles, masks, scales and lengths meet badly; against the restatement in 64
bits and at the tolerances of test_gpu_kv.py."""
import ctypes as C

import numpy as np
import pytest

from asystem_amem_amd import binding as B
from asystem_amem_amd import kv
from tests import kv_oracle as O
from tests.kv_case import KINDS, Arena, Case
from tests.test_gpu_kv import HALF, TYPES, check_append, check_attend, near, poison, run_attend

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


FAR, NEAR, LATE = 2.0 ** -33, 2.0 ** -25, 2.0 ** -25


def check_scaled(case, q, step):
    """Values in e4m3 of scales that may be far apart. Beside the roundings of weights, scores and result: a product of weight and scale far below
    the largest loses bits, to steps of 2^-33 of the largest at most, as fp16 has them for numbers whose largest is at least 2^8; or, while all scales
    are within 2^8 of each other (NEAR), a weight does, whose scale may be 2^8 of the largest product's; times codes of up to 448, for each
    position. Where near scales go before far ones the largest product is known within 2^15 at first: 2^8 of scales, and 2^7 of weights (LATE)."""
    got, lse = run_attend(case, q)
    group, d = case.q_heads // case.kv_heads, case.dim
    for s, (n, c) in enumerate(case.lengths):
        rows, seen = slice(case.cu[s], case.cu[s] + n), case.visible(s, True, 0)
        p = np.arange(c)
        page, block = case.table[s, p // case.page], p % case.page // case.block
        for h in range(case.q_heads):
            k, v = case.gathered(s, h // group)
            x = O.decode(q[rows, h], case.kind)
            out, l, size, top = O.attend(x, k, v, d ** -0.5, seen)
            with np.errstate(all="ignore"):
                weight = np.where(seen, np.exp(x @ k.T * d ** -0.5 - l[:, None]), 0)
            most = (weight * case.v_scale[page, h // group, block].astype(np.float64)).max(1)
            lost = c * 448 * step * most
            score = d * 2.0 ** -23 * top + 2.0 ** -18
            near(got[rows, h], out, case.kind, (HALF["f16"] + score)[:, None] * size + lost[:, None])
            assert (np.abs(lse[rows, h] - l) <= score + 2.0 ** -22 * np.abs(l)).all()
    return got


def scaled_case(arena, lengths, dim, kind, exponents, bias, seed=35, **more):
    """Blocks take the scales 2^e in turn, and keys make the first of them lose `bias` (of the natural logarithm of a weight) to the others."""
    case = Case(arena, lengths, dim=dim, q_heads=4, kv_heads=2, kind=kind, eight=True, page=32, block=16, seed=seed, **more)
    case.v &= 0xDF                                    # codes of at most 28, so that weighted means stay inside the types
    case.k_scale[:] = 2.0 ** -6
    case.k[..., 0] = O.e4m3_code(np.float64(448))
    for s, (n, c) in enumerate(case.lengths):
        for i, p in enumerate(range(0, c, 16)):
            page, at = case.table[s, p // 32], p % 32
            case.v_scale[page, :, at // 16] = 2.0 ** exponents[i % len(exponents)]
            if i % len(exponents) == 0:
                case.k[page, :, at:at + 16, 0] = O.e4m3_code(np.float64(-448))
    case.upload()
    q = case.r.standard_normal((case.tokens, 4, dim)) * 0.5
    q[..., 0] = bias * dim ** 0.5 / 14                # the first dim's part of a score is bias / 2, or - bias / 2
    return case, O.encode(q, kind)


FORMS = {"token": [(1, 700)], "draft": [(5, 330)], "prompt": [(100, 700)], "long": [(1, 2500), (2, 900)], "long prompt": [(300, 1300)]}


@pytest.mark.parametrize("dim,kind", [(64, "f16"), (128, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("exponents,bias", [((0, -14), 0), ((0, -14), 9.7), ((0, -14), 30), ((-14, 0), 5), ((9, -3, -9, 2), 12), ((-3, -7), 4), ((-3, -11), 4), ((-3, -12), 4), ((-7, -7, -7, -7, -3), 2),
                                            ((-7, -7, -7, -7, -2), 2)])
def test_scales_of_values_far_apart(arena, form, dim, kind, exponents, bias):
    """A large scale takes no bits of small ones that have the weight, on either side of the border between scales that are near and far."""
    case, q = scaled_case(arena, FORMS[form], dim, kind, exponents, bias)
    check_scaled(case, q, NEAR if max(exponents) - min(exponents) <= 8 else FAR)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("exponents,bias", [((0, -30), 0), ((0, -30), 21), ((0, -30), 60), ((50, -50), 80), ((-50, 50), 3), ((119, 119), 1), ((119, 30), 40),
                                            ((-64, -64), 1), ((-64, 0), 30), ((30, -30, 0, 5, -64, 10), 30)])
def test_scales_of_the_whole_range(arena, form, dim, exponents, bias):
    case, q = scaled_case(arena, FORMS[form], dim, "bf16", exponents, bias)
    check_scaled(case, q, NEAR if max(exponents) - min(exponents) <= 8 else FAR)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("form", ["draft", "prompt", "long prompt"])
def test_hidden_scales_and_bad_values_among_scales_far_apart(arena, form, kind):
    """A scale of rows that come later is of no account to those before; NaN that some rows see, in a cache whose scales are far apart."""
    case, q = scaled_case(arena, FORMS[form], 128, kind, (0, -14), 12, seed=36)
    n, c = case.lengths[0]
    last = c - 1
    page, block = case.table[0, last // 32], last % 32 // 16
    case.v_scale[page, :, block] = 2.0 ** 100
    case.v[page, :, last % 32] = 0                     # the last position's block is huge; but for that position it holds zeros
    for p in range(last // 16 * 16, last):
        case.v[page, :, p % 32] = 0
    case.v[page, 1, last % 32, 7] = 0x7F
    poison(case, 0, c - n + 1, v=0x7F)
    case.upload()
    got = O.decode(check_scaled(case, q, FAR), kind)
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("far", [-40, 40])
def test_scales_that_part_late(arena, form, dim, far):
    """Near ones for half of the context, then one block far from them: with little weight, and with all of it for the last rows."""
    for value in (-448, 448):
        lengths = FORMS[form]
        case, q = scaled_case(arena, lengths, dim, "bf16", (0, -3), 6, seed=37)
        for s, (n, c) in enumerate(lengths):
            p = c // 2 // 16 * 16
            page, at = case.table[s, p // 32], p % 32
            case.v_scale[page, :, at // 16] = 2.0 ** far
            case.k[page, :, at:at + 16, 1] = O.e4m3_code(np.float64(value))
        case.upload()
        x = O.decode(q, "bf16")
        x[..., 1] = 4 * dim ** 0.5
        check_scaled(case, O.encode(x, "bf16"), LATE)
        arena.reset()


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -140, -2.0 ** -110])
def test_a_scale_of_zero_or_hardly_more(arena, scale):
    """All weights are equal, whatever the size of the scores; an infinite one times zero is NaN."""
    for lengths in ([(1, 90)], [(5, 200)], [(70, 200)], [(300, 700)]):
        n, c = lengths[0]
        for infinite in (False, True):
            case = Case(arena, lengths, dim=64, q_heads=2, kv_heads=1, page=16, seed=38)
            case.k = O.encode(O.decode(case.k, "bf16") * 2.0 ** 100, "bf16")
            if infinite:
                page, slot = case.table[0, (c - 1) // 16], (c - 1) % 16
                case.k[page, 0, slot, 0] = 0x7F80                      # the last row sees it
            case.upload()
            got, _ = check_attend(case, case.rows(2), scale=scale)
            assert np.isfinite(O.decode(got, "bf16")[:n - 1]).all()
            if infinite and scale == 0:
                assert np.isnan(O.decode(got, "bf16")[n - 1]).all()
            arena.reset()


def test_memory_that_is_not_tracked_is_used_while_paused(gpu, fresh):
    """A pause takes the communication buffers; a cache elsewhere is written and read meanwhile, with the same results."""
    lib = fresh
    arena, buffers = Arena(lib, 16 << 20), Arena(lib, 8 << 20)
    try:
        assert lib.amem_add_alloc_info(buffers.va, buffers.alloc, B.TYPE_LOCAL, 0, buffers.handle, -1, 0, None, B.CALLER_P2P) == 0
        case = Case(arena, [(1, 2000), (40, 70)], dim=128, q_heads=4, kv_heads=2, eight=True, page=32, block=32, seed=39).upload()
        q = case.rows(4)
        one, l1 = run_attend(case, q)
        assert lib.ncclPause(None) == 0
        check_append(case, case.rows(2), case.rows(2), q, rotary=128)
        check_attend(case, q)
        case.args.workspace = buffers.va
        case.args.workspace_bytes = 8 << 20
        n = C.c_uint64()
        assert lib.amem_kv_attention_workspace(C.byref(case.cache), C.byref(case.batch), 4, C.byref(n)) == 0 and n.value
        assert lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(case.args), None) == 1
        assert lib.ncclResume(None) == 0
        assert lib.amem_kv_attention(C.byref(case.cache), C.byref(case.batch), C.byref(case.args), None) == 0
        assert lib.amem_del_alloc_info(buffers.va, 0, 0) == 0
    finally:
        arena.free()
        buffers.free()


@pytest.mark.parametrize("bad", [0.0, -1.0, 2.0 ** 120, float("nan"), float("inf"), 1e-45])
@pytest.mark.parametrize("lengths,window", [([(1, 300)], 40), ([(1, 1500)], 1000), ([(6, 330)], 100), ([(100, 400)], 30), ([(300, 1300)], 200)])
def test_scales_of_hidden_blocks_may_be_anything(arena, lengths, window, bad):
    """In front of what a window lets the first row see, in tiles of their own and beside seen blocks, and behind the context."""
    for dim in (64, 128):
        case = Case(arena, lengths, dim=dim, q_heads=4, kv_heads=2, eight=True, page=32, block=16, seed=40)
        (n, c), = lengths
        for p in range(0, case.table_pages * 32, 16):
            page = case.table[0, p // 32]
            if page >= 0 and (p + 15 <= c - n - window or p >= c):
                case.k_scale[page, :, p % 32 // 16] = case.v_scale[page, :, p % 32 // 16] = bad
        case.upload()
        got, lse = check_attend(case, case.rows(4), window=window)
        assert np.isfinite(O.decode(got, "bf16")).all() and np.isfinite(lse).all()
        arena.reset()
