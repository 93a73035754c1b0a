"""The operators on a paged key/value cache, the part that needs no GPU: the header and its binding agree, arguments are
refused with a reason, and the index arithmetic stays inside its tensors whatever device memory holds."""
import ctypes as C
import os
import re
import subprocess

import pytest

from asystem_amem_amd import binding as B
from asystem_amem_amd import kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, NO_DEVICE = 1, 100


def test_header_library_and_binding_agree(lib, tmp_path):
    text = open(os.path.join(ROOT, "include", "amem_kv.h")).read()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(amem_kv_[a-z_]*)\s*\(", code))
    assert declared == set(kv.kv_abi_names())
    out = subprocess.run(["nm", "-D", "--defined-only", B.LIB_PATH], check=True, capture_output=True, text=True).stdout
    assert declared <= {line.split()[-1] for line in out.splitlines()}
    # every field at the place where C has it
    structs = {"amem_kv_cache": kv.CacheInfo, "amem_kv_batch": kv.BatchInfo, "amem_kv_append_args": kv.AppendArgs,
               "amem_kv_attention_args": kv.AttentionArgs}
    src = ['#include <stdio.h>', '#include "amem_kv.h"', 'int main(void) {']
    for name, s in structs.items():
        src.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        src += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f[0], name, f[0]) for f in s._fields_]
    (tmp_path / "t.c").write_text("\n".join(src + ["return 0; }"]))
    exe = str(tmp_path / "t")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I" + os.path.join(ROOT, "include"),
                    str(tmp_path / "t.c"), "-o", exe], check=True)
    got = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, s in structs.items():
        assert int(got[name]) == C.sizeof(s)
        for f in s._fields_:
            assert int(got["%s.%s" % (name, f[0])]) == getattr(s, f[0]).offset, (name, f[0])


def valid(eight=False):
    """Arguments that nothing is wrong with, at addresses that nothing is at."""
    A = 0x10000
    cache = kv.CacheInfo(A, A, A if eight else 0, A if eight else 0, 4 * 64 * 128, 64 * 128, 128, 8, 2,
                         kv.E4M3 if eight else kv.BF16, 0, 10, 4, 64, 32 if eight else 0, 128, 0)
    batch = kv.BatchInfo(A, A, A, 5, 3, 5, 20, 8, 320, 0)
    app = kv.AppendArgs(A, A, A, A, A, A, A, 512, 128, 512, 128, 1024, 128, 1024, 128, 20, kv.BF16, 8, 128, 0, 1000, 1)
    att = kv.AttentionArgs(A, A, A, A, 1 << 40, 1024, 128, 1024, 128, 0.1, kv.BF16, 8, 1, 0, 0)
    return cache, batch, app, att


def calls(lib, cache, batch, app, att):
    kv.load()
    return (lib.amem_kv_append(C.byref(cache), C.byref(batch), C.byref(app), None),
            lib.amem_kv_attention(C.byref(cache), C.byref(batch), C.byref(att), None))


@pytest.mark.parametrize("eight", [False, True])
def test_valid_arguments_need_a_gpu(lib, eight):
    if lib.amem_device_count():
        pytest.skip("the addresses are made up: only where nothing can run")
    assert calls(lib, *valid(eight)) == (NO_DEVICE, NO_DEVICE)


@pytest.mark.parametrize("eight", [False, True])
def test_empty_calls_do_nothing(lib, eight):
    cache, batch, app, att = valid(eight)
    batch.tokens = batch.max_tokens = 0
    app.k = app.v = app.q = app.q_out = att.q = att.out = 0      # an empty tensor has no address
    assert calls(lib, cache, batch, app, att) == (0, 0)


CACHE = [("type", 3), ("type", -1), ("k", 0), ("v", 0), ("k", 0x10008), ("head_dim", 96), ("head_dim", 0), ("pages", 0), ("kv_heads", 0),
         ("kv_heads", 1 << 20), ("page_slots", 0), ("page_slots", 48), ("page_slots", 2048), ("page_stride", 4), ("page_stride", -128),
         ("slot_stride", 130), ("head_stride", 1 << 41), ("reserved", 1), ("page_slots", -16)]
BATCH = [("context", 0), ("context", 0x10002), ("page_table", 0), ("page_table", 0x10001), ("cu_tokens", 0x10001), ("cu_tokens", 0),
         ("table_stride", 4), ("table_pages", -1), ("tokens", -1), ("tokens", 1 << 25), ("max_tokens", 21), ("max_tokens", -1),
         ("max_context", 321), ("max_context", -1), ("sequences", -1), ("reserved", 2)]
APPEND = [("type", kv.E4M3), ("type", 7), ("k", 0), ("v", 0), ("k", 0x10008), ("k_token_stride", 516), ("v_head_stride", -8), ("q", 0), ("q_out", 0),
          ("q_heads", 0), ("q_out_token_stride", 1 << 40), ("rotary_dim", 8), ("rotary_dim", 144), ("rotary_dim", -16), ("cos", 0), ("sin", 0x10004),
          ("table_rows", 0), ("axes", 0), ("axes", 5), ("axes", 2), ("positions", 0x10002)]
ATTEND = [("type", kv.E4M3), ("q", 0), ("out", 0), ("out", 0x10008), ("q_token_stride", 4), ("out_head_stride", 12), ("q_heads", 6), ("q_heads", 0),
          ("lse", 0x10002), ("window", -1), ("scale", float("nan")), ("scale", float("inf")), ("reserved", 1)]


def _refused(lib, which, field, value, eight=False):
    args = valid(eight)
    setattr(args[which], field, value)
    return calls(lib, *args)


@pytest.mark.parametrize("field,value", CACHE + BATCH)
def test_cache_and_batch_are_checked(lib, field, value):
    which = 0 if (field, value) in CACHE and hasattr(kv.CacheInfo, field) else 1
    assert _refused(lib, which, field, value) == (INVALID, INVALID)


@pytest.mark.parametrize("field,value", [("k_scale", 0), ("v_scale", 0x10002), ("block_slots", 0), ("block_slots", 8), ("block_slots", 128),
                                         ("block_slots", 24), ("scale_page_stride", -1), ("slot_stride", 136)])
def test_8_bit_cache_is_checked(lib, field, value):
    assert _refused(lib, 0, field, value, eight=True) == (INVALID, INVALID)


@pytest.mark.parametrize("field,value", [("k_scale", 0x10000), ("block_slots", 16), ("type", kv.F16)])
def test_16_bit_cache_has_no_scales_and_the_rows_type(lib, field, value):
    assert _refused(lib, 0, field, value) == (INVALID, INVALID)


@pytest.mark.parametrize("field,value", APPEND)
def test_append_is_checked(lib, field, value):
    assert _refused(lib, 2, field, value)[0] == INVALID


@pytest.mark.parametrize("sections", [(32, 16, 15, 0), (-8, 72, 0, 0), (2 ** 31 - 1, 2 ** 31 - 1, 66, 0)])
def test_sections_are_checked(lib, sections):
    cache, batch, app, att = valid()
    app.axes, app.sections = 3, (C.c_int32 * 4)(*sections)
    assert calls(lib, cache, batch, app, att)[0] == INVALID


@pytest.mark.parametrize("field,value", ATTEND)
def test_attention_is_checked(lib, field, value):
    assert _refused(lib, 3, field, value)[1] == INVALID


def test_uniform_rows_have_to_add_up(lib):
    cache, batch, app, att = valid()
    batch.cu_tokens, batch.max_tokens = 0, 7                       # 3 * 7 is not 20
    assert calls(lib, cache, batch, app, att) == (INVALID, INVALID)


@pytest.mark.parametrize("tokens,sequences,kv_heads,q_heads", [(1 << 22, 5, 4, 64), (1 << 21, 5, 64, 64), (100, 1 << 20, 4, 4), (1 << 20, 5, 128, 128)])
def test_sizes_beyond_a_launch_are_refused(lib, tokens, sequences, kv_heads, q_heads):
    cache, batch, app, att = valid(True)
    batch.tokens, batch.max_tokens, batch.sequences = tokens, tokens, sequences
    cache.kv_heads, att.q_heads = kv_heads, q_heads
    kv.load()
    assert lib.amem_kv_attention(C.byref(cache), C.byref(batch), C.byref(att), None) == INVALID
    n = C.c_uint64()
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), q_heads, C.byref(n)) == INVALID


def test_null_structs(lib):
    cache, batch, app, att = valid()
    kv.load()
    for i in range(3):
        a = [C.byref(x) for x in (cache, batch, app)]
        a[i] = None
        assert lib.amem_kv_append(*a, None) == INVALID
        a = [C.byref(x) for x in (cache, batch, att)]
        a[i] = None
        assert lib.amem_kv_attention(*a, None) == INVALID


def test_workspace_is_checked(lib):
    cache, batch, app, att = valid()
    batch.sequences, batch.tokens, batch.max_tokens, batch.cu_tokens = 1, 1, 1, 0
    batch.table_pages = batch.table_stride = 4096
    batch.max_context = 4096 * 64
    kv.load()
    n = C.c_uint64(7)
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), 8, C.byref(n)) == 0
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), 7, C.byref(n)) == INVALID
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), 8, None) == INVALID
    if n.value:
        for field, value in (("workspace", 0), ("workspace", 0x10008), ("workspace_bytes", n.value - 1)):
            a = kv.AttentionArgs.from_buffer_copy(att)
            setattr(a, field, value)
            assert lib.amem_kv_attention(C.byref(cache), C.byref(batch), C.byref(a), None) == INVALID


def test_indexes_stay_inside(tmp_path):
    """kv_index.h in a host build with sanitizers: lengths, offsets and page numbers of every kind, right and wrong."""
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "asystem-amem_amd", "csrc"), os.path.join(ROOT, "tests", "kv_index", "index_driver.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ok" in r.stdout


def test_packed_arguments_are_the_structures():
    """kv.py hands records over as bytes: the same ones as the structures."""
    numbers = list(range(1, 27))
    a = kv.AppendArgs.from_buffer_copy(kv._append_args(*numbers))
    got = [getattr(a, f[0]) for f in a._fields_[:-1]] + list(a.sections)
    assert got == numbers and C.sizeof(a) == len(kv._append_args(*numbers))
    numbers = list(range(1, 16))
    a = kv.AttentionArgs.from_buffer_copy(kv._attention_args(*numbers))
    assert [getattr(a, f[0]) for f in a._fields_] == numbers and C.sizeof(a) == len(kv._attention_args(*numbers))


@pytest.mark.parametrize("sequences,tokens,max_tokens", [(3, 20, 7), (1 << 15, 1 << 15, 1 << 15), (1 << 16, 1 << 19, 1 << 19)])
def test_the_workspace_of_rows_that_do_not_add_up_is_refused(lib, sequences, tokens, max_tokens):
    """As by the call itself; their number of units can pass 32 bits."""
    cache, batch, app, att = valid()
    batch.sequences, batch.tokens, batch.max_tokens = sequences, tokens, max_tokens
    kv.load()
    n = C.c_uint64()
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), 16, C.byref(n)) == 0       # with offsets: a guide
    batch.cu_tokens = 0
    assert lib.amem_kv_attention_workspace(C.byref(cache), C.byref(batch), 16, C.byref(n)) == INVALID


@pytest.mark.parametrize("record,field,value,refused", [
    (2, "q_out_token_stride", 0, (1, 0)), (2, "q_out_head_stride", 0, (1, 0)), (2, "q_out_token_stride", 512, (1, 0)), (2, "q_out_head_stride", 64, (1, 0)),
    (3, "out_token_stride", 0, (0, 1)), (3, "out_head_stride", 0, (0, 1)), (3, "out_token_stride", 1016, (0, 1)), (3, "out_head_stride", 64, (0, 1)),
    (0, "page_stride", 0, (1, 0)), (0, "head_stride", 0, (1, 0)), (0, "slot_stride", 0, (1, 0)), (0, "head_stride", 128, (1, 0)), (0, "page_stride", 3 * 64 * 128, (1, 0)),
    (0, "scale_page_stride", 0, (1, 0)), (0, "scale_head_stride", 1, (1, 0)), (0, "scale_page_stride", 7, (1, 0)),
    (2, "k_token_stride", 0, (0, 0)), (2, "v_head_stride", 0, (0, 0)), (2, "q_token_stride", 0, (0, 0)), (3, "q_head_stride", 0, (0, 0))])
def test_what_is_written_must_not_overlap_itself(lib, record, field, value, refused):
    """What is only read may: the same row for all, the same keys for all heads."""
    if lib.amem_device_count():
        pytest.skip("the addresses are made up: only where nothing can run")
    args = valid(True)
    setattr(args[record], field, value)
    assert calls(lib, *args) == tuple(INVALID if r else NO_DEVICE for r in refused)


def test_layouts_that_keep_rows_apart_are_taken(lib):
    """Heads before tokens, slots before heads, a part of a wider tensor, one of each dimension with any stride."""
    if lib.amem_device_count():
        pytest.skip("the addresses are made up: only where nothing can run")
    for change in ({"out_token_stride": 128, "out_head_stride": 20 * 128}, {"out_token_stride": 4096}, {"out_head_stride": 256, "out_token_stride": 2048}):
        cache, batch, app, att = valid(True)
        for k, v in change.items():
            setattr(att, k, v)
            setattr(app, "q_" + k, v)
        assert calls(lib, cache, batch, app, att) == (NO_DEVICE, NO_DEVICE), change
    cache, batch, app, att = valid(True)
    cache.head_stride, cache.slot_stride = 128, 4 * 128                            # [page][slot][head][dim]
    assert calls(lib, cache, batch, app, att) == (NO_DEVICE, NO_DEVICE)
    cache.page_stride, cache.slot_stride = 128 * 4, 10 * 4 * 128                   # [slot][page][head][dim]
    assert calls(lib, cache, batch, app, att) == (NO_DEVICE, NO_DEVICE)
    cache, batch, app, att = valid(True)
    cache.pages = cache.kv_heads = 1
    cache.page_stride = cache.head_stride = cache.scale_page_stride = cache.scale_head_stride = 0
    att.q_heads = app.q_heads = 1
    att.out_head_stride = app.q_out_head_stride = 0
    assert calls(lib, cache, batch, app, att) == (NO_DEVICE, NO_DEVICE)
