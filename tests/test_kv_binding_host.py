"""kv.py's own checks, with stand-ins for tensors (nothing reaches a GPU), and the rule by which attention is cut."""
import os
import subprocess

import pytest

from asystem_amem_amd import kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Device:
    def __init__(self, kind="cuda", index=0):
        self.type, self.index = kind, index

    def __eq__(self, other):
        return (self.type, self.index) == (other.type, other.index)

    def __ne__(self, other):
        return not self == other


class Kind:
    def __init__(self, name):
        self.name = name

    def __str__(self):
        return "torch." + self.name


KINDS = {n: Kind(n) for n in ("bfloat16", "float16", "float8_e4m3fn", "float32", "int32", "int64")}


class Tensor:
    def __init__(self, shape, dtype="bfloat16", strides=None, device=None):
        self.shape, self.dtype, self.device = tuple(shape), KINDS[dtype], device or Device()
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.insert(0, n)
                n *= s
        self._strides = tuple(strides)

    def stride(self):
        return self._strides

    def data_ptr(self):
        return 0x10000

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def element_size(self):
        return 1

    def is_contiguous(self):
        return self._strides == Tensor(self.shape)._strides


def cache(**k):
    return kv.Cache(Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 64)))


def batch(**k):
    a = dict(page_table=Tensor((3, 4), "int32"), context=Tensor((3,), "int32"), tokens=5, cu_tokens=Tensor((4,), "int32"), max_tokens=2, max_context=64)
    a.update(k)
    return kv.Batch(**a)


OTHER = Device(index=1)


@pytest.mark.parametrize("k,v,scales", [
    (Tensor((9, 2, 16)), Tensor((9, 2, 16)), ()),
    (Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 128)), ()),
    (Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 64), "float16"), ()),
    (Tensor((9, 2, 16, 64), "float32"), Tensor((9, 2, 16, 64), "float32"), ()),
    (Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 64), strides=(2048, 64, 128, 1)), ()),
    (Tensor((9, 2, 16, 64), strides=(2048, 1024, 1, 16)), Tensor((9, 2, 16, 64), strides=(2048, 1024, 1, 16)), ()),
    (Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 64), device=OTHER), ()),
    (Tensor((9, 2, 16, 64), device=Device("cpu")), Tensor((9, 2, 16, 64), device=Device("cpu")), ()),
    (Tensor((9, 2, 16, 64)), Tensor((9, 2, 16, 64)), (Tensor((9, 2, 1), "float32"),) * 2),
    (Tensor((9, 2, 16, 64), "float8_e4m3fn"), Tensor((9, 2, 16, 64), "float8_e4m3fn"), ()),
    (Tensor((9, 2, 16, 64), "float8_e4m3fn"), Tensor((9, 2, 16, 64), "float8_e4m3fn"), (Tensor((9, 2, 1), "float32"), None)),
    (Tensor((9, 2, 16, 64), "float8_e4m3fn"), Tensor((9, 2, 16, 64), "float8_e4m3fn"), (Tensor((9, 2, 3), "float32"),) * 2),
    (Tensor((9, 2, 16, 64), "float8_e4m3fn"), Tensor((9, 2, 16, 64), "float8_e4m3fn"), (Tensor((9, 2, 1), "float16"),) * 2),
])
def test_caches_that_are_refused(k, v, scales):
    with pytest.raises(ValueError):
        kv.Cache(k, v, *scales)


@pytest.mark.parametrize("changed", [
    dict(context=Tensor((), "int32")), dict(context=Tensor((3, 1), "int32")), dict(context=Tensor((3,), "int64")), dict(context=Tensor((4,), "int32")),
    dict(context=Tensor((3,), "int32", (2,))), dict(page_table=Tensor((12,), "int32")), dict(page_table=Tensor((3, 4), "int32", (1, 3))),
    dict(page_table=Tensor((3, 4), "int32", (3, 1))), dict(page_table=Tensor((3, 4), "int32", device=OTHER)),
    dict(cu_tokens=Tensor((3,), "int32")), dict(cu_tokens=Tensor((4,), "int64")), dict(cu_tokens=Tensor((4, 1), "int32")), dict(max_context=None)])
def test_batches_that_are_refused(changed):
    batch()
    with pytest.raises(ValueError):
        batch(**changed)


@pytest.mark.parametrize("changed", [
    dict(q=Tensor((5, 4, 32))), dict(q=Tensor((4, 4, 64))), dict(q=Tensor((5, 256))), dict(q=Tensor((5, 4, 64), "float32")), dict(out=Tensor((5, 2, 64))),
    dict(out=Tensor((5, 4, 64), "float16")), dict(out=Tensor((5, 4, 64), device=OTHER)), dict(q=Tensor((5, 4, 64), strides=(256, 1, 4))),
    dict(lse=Tensor((4, 5), "float32")), dict(lse=Tensor((5, 4))), dict(lse=Tensor((5, 4), "float32", (1, 5))), dict(window="wide"), dict(scale="small"),
    dict(window=1 << 40), dict(workspace=Tensor((64,), device=OTHER)), dict(workspace=Tensor((64,), strides=(2,))),
    dict(batch=batch(context=Tensor((3,), "int32", device=OTHER), page_table=Tensor((3, 4), "int32", device=OTHER), cu_tokens=Tensor((4,), "int32", device=OTHER)))])
def test_attention_arguments_that_are_refused(changed):
    a = dict(cache=cache(), batch=batch(), q=Tensor((5, 4, 64)), out=Tensor((5, 4, 64)))
    a.update(changed)
    with pytest.raises(ValueError):
        kv.attention(**a)


TABLES = kv.Rotation(Tensor((99, 32), "float32"), Tensor((99, 32), "float32"))
AXES = kv.Rotation(Tensor((99, 32), "float32"), Tensor((99, 32), "float32"), sections=(16, 16))


@pytest.mark.parametrize("changed", [
    dict(k=Tensor((5, 4, 64))), dict(v=Tensor((5, 2, 64), "float16")), dict(k=Tensor((5, 2, 64), "float32"), v=Tensor((5, 2, 64), "float32")), dict(k=Tensor((5, 128))),
    dict(q=Tensor((5, 4, 64))), dict(q=Tensor((5, 4, 64)), q_out=Tensor((5, 2, 64))), dict(q=Tensor((5, 4, 64)), q_out=Tensor((5, 4, 64), device=OTHER)),
    dict(positions=Tensor((5,), "int32")), dict(rotation=AXES), dict(rotation=AXES, positions=Tensor((5,), "int32")),
    dict(rotation=AXES, positions=Tensor((2, 5), "int32", (1, 2))), dict(rotation=TABLES, positions=Tensor((5,), "int64")), dict(rotation=TABLES, positions=Tensor((4,), "int32")),
    dict(rotation=kv.Rotation(Tensor((99, 32), "float32", device=OTHER), Tensor((99, 32), "float32", device=OTHER)))])
def test_append_arguments_that_are_refused(changed):
    a = dict(cache=cache(), batch=batch(), k=Tensor((5, 2, 64)), v=Tensor((5, 2, 64)))
    a.update(changed)
    with pytest.raises(ValueError):
        kv.append(**a)


@pytest.mark.parametrize("cos,sin,sections", [
    (Tensor((99, 32)), Tensor((99, 32)), None), (Tensor((99, 32), "float32"), Tensor((98, 32), "float32"), None), (Tensor((99,), "float32"), Tensor((99,), "float32"), None),
    (Tensor((99, 32), "float32"), Tensor((99, 32), "float32"), (16, 8)), (Tensor((99, 32), "float32"), Tensor((99, 32), "float32"), (8, 8, 8, 4, 4)),
    (Tensor((99, 32), "float32"), Tensor((99, 32), "float32"), (40, -8)), (Tensor((99, 32), "float32", (64, 1)), Tensor((99, 32), "float32", (64, 1)), None)])
def test_rotations_that_are_refused(cos, sin, sections):
    with pytest.raises(ValueError):
        kv.Rotation(cos, sin, sections)


def test_cuts_fit_the_workspace(tmp_path):
    """kv_cut.h in a host build with sanitizers."""
    exe = str(tmp_path / "cut")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "asystem-amem_amd", "csrc"), os.path.join(ROOT, "tests", "kv_index", "cut_driver.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ok" in r.stdout


@pytest.mark.parametrize("changed", [
    dict(max_context=(1 << 32) + 64), dict(max_context=1 << 31), dict(max_tokens=(1 << 32) + 2), dict(tokens=(1 << 32) + 5), dict(tokens=-(1 << 32)), dict(max_context=64.0),
    dict(max_tokens="2"), dict(max_context=None, page_slots=1 << 30)])
def test_numbers_of_a_batch_are_not_cut_to_32_bits(changed):
    with pytest.raises(ValueError):
        batch(**changed)


def test_numbers_of_a_batch_arrive():
    b = batch(tokens=5, max_tokens=2, max_context=(1 << 31) - 1)
    assert (b.info.tokens, b.info.max_tokens, b.info.max_context, b.info.sequences, b.info.table_pages) == (5, 2, (1 << 31) - 1, 3, 4)


def test_a_cache_of_too_many_pages_is_refused():
    k = Tensor(((1 << 32) + 9, 2, 16, 64))
    with pytest.raises(ValueError):
        kv.Cache(k, k)


@pytest.mark.parametrize("q_heads", [(1 << 32) + 4, 4.0, None])
def test_the_workspace_of_heads_that_are_no_number_is_refused(lib, q_heads):
    assert kv.attention_workspace(cache(), batch(), 4) >= 0
    with pytest.raises(ValueError):
        kv.attention_workspace(cache(), batch(), q_heads)


def test_a_place_for_queries_without_queries_is_refused():
    with pytest.raises(ValueError):
        kv.append(cache(), batch(), Tensor((5, 2, 64)), Tensor((5, 2, 64)), q_out=Tensor((5, 4, 64)))


def test_entry_points_are_there_all_at_once(monkeypatch):
    """Another thread that makes its first call meanwhile finds none of them, or all."""
    class Library:
        def __getattr__(self, name):
            assert not kv._entry, "some of the entry points are already there"
            return lambda *a: 0

    monkeypatch.setattr(kv, "_entry", {})
    monkeypatch.setattr(kv.binding, "load", Library)
    kv.load()
    assert sorted(kv._entry) == kv.kv_abi_names()
