"""The operators on block tables and on the cache in 4 bits refuse the same arguments natively as their Python assertions do, argument by argument, and their
C entry points refuse sizes, alignments and overlaps before anything is launched.  No GPU."""
from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from test_attention_operator_checks import PAGED, SPARSE, TEXT, moved
from test_host_checks_agree import BF16, DLPACK, F32, I32, I64, U8, Spec, changed_number

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="accepted calls would launch on addresses that are not memory")

BOOL = torch.bool
CACHE = Spec(U8, 3, 64 * 368)
INSERT = (Spec(BF16, 5, 4, 512), Spec(BF16, 5, 512), CACHE, Spec(I64, 5), Spec(I64, 5), Spec(F32, 99, 64), 1e-6, 64)
POOL = (Spec(I32, 6, 9), Spec(I32, 40), Spec(I32, 1))
RESULTS = (Spec(I32, 7), Spec(I32, 6), Spec(I64, 20), Spec(I64, 20), Spec(I32, 20), Spec(I32, 1), Spec(I32, 1))


def extend(*args):
    return fg.extend_block_tables(*args[:7], args[7:] if len(args) > 7 else None)


OPS = {
    "insert": (fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert, "_call", "prologue_mxfp4", INSERT),
    "paged": (fg.paged_latent_attention_mxfp4, "_paged_mxfp4", "paged_latent_attention_mxfp4", PAGED[:1] + (CACHE,) + PAGED[2:]),
    "sparse": (fg.sparse_latent_attention_mxfp4, "_sparse_mxfp4", "sparse_latent_attention_mxfp4", SPARSE[:1] + (CACHE,) + SPARSE[2:]),
    "extend": (extend, "_extend", "extend_block_tables", (Spec(I32, 6), Spec(I32, 6), *POOL, 16, 20)),
    "extend, given results": (extend, "_extend", "extend_block_tables", (Spec(I32, 6), Spec(I32, 6), *POOL, 16, 20, *RESULTS)),
    "release": (fg.release_block_tables, "_release", "release_block_tables", (Spec(I32, 6), Spec(BOOL, 6), *POOL, 16, Spec(I32, 1))),
}


def accepts(name, args, native, monkeypatch):
    op, attribute, entry, _ = OPS[name]
    module = importlib.import_module((fg.extend_block_tables if op is extend else op).__module__)
    call = getattr(_native.host_calls(), entry)
    monkeypatch.setattr(module, attribute, call if native else (lambda *a: None))
    monkeypatch.setitem(DLPACK, BOOL, (6, 8))
    keep, tensors = [], []
    for i, a in enumerate(args):
        if isinstance(a, Spec):
            a = a.make(keep) if a.device is None else moved(a.make, keep, (i + 1) << 40)  # no two overlap
        tensors.append(a)
    try:
        op(*tensors)
        return True, ""
    except _native.Dsv4Error as e:
        return (not native or "refused" not in str(e)), str(e)
    except (AssertionError, TypeError, ValueError, IndexError, AttributeError, ArithmeticError) as e:
        return False, f"{type(e).__name__} {e}"
    except RuntimeError as e:
        return native and "driver" in str(e), str(e)


@pytest.mark.parametrize("name", OPS)
def test_both_accept_the_same(name, monkeypatch):
    monkeypatch.setattr(torch.cuda, "_lazy_init", lambda: None)
    args = OPS[name][3]
    assert accepts(name, args, True, monkeypatch)[0] and accepts(name, args, False, monkeypatch)[0]
    refused = 0
    for i, a in enumerate(args):
        for c in a.changed() if isinstance(a, Spec) else changed_number(a):
            changed = args[:i] + (c,) + args[i + 1 :]
            (native, why), (python, _) = accepts(name, changed, True, monkeypatch), accepts(name, changed, False, monkeypatch)
            if python and c in TEXT:
                assert native or "the call was refused (" in why, (i, c, why)
            else:
                assert native == python, (i, c, why)
            refused += not native
    assert refused > 20


def library():
    return ctypes.CDLL(str(_native.LIB_PATH))


i64, f32, ptr = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
STEP = 1 << 40


def places(names):
    return {n: STEP * (i + 1) for i, n in enumerate(names)}


EXTEND = ("context", "new", "table", "free", "num_free", "starts", "lens", "positions", "slots", "requests", "left", "missing")
EXTEND_BYTES = dict(zip(EXTEND, (24, 24, 5 * 48 + 36, 160, 4, 28, 24, 160, 160, 80, 4, 4)))


def c_extend(at=None, reqs=6, stride=12, width=9, capacity=40, bs=16, tokens=20):
    a = at or places(EXTEND)
    return library().dsv4_extend_block_tables(ptr(a["context"]), ptr(a["new"]), i64(reqs), ptr(a["table"]), i64(stride), i64(width), ptr(a["free"]), i64(capacity), ptr(a["num_free"]), i64(bs),
                                              i64(tokens), *(ptr(a[n]) for n in EXTEND[5:]), ptr(0))


RELEASE = ("lens", "finished", "table", "free", "num_free", "left")
RELEASE_BYTES = dict(zip(RELEASE, (24, 6, 5 * 48 + 36, 160, 4, 4)))


def c_release(at=None, reqs=6, stride=12, width=9, capacity=40, bs=16):
    a = at or places(RELEASE)
    return library().dsv4_release_block_tables(ptr(a["lens"]), ptr(a["finished"]), i64(reqs), ptr(a["table"]), i64(stride), i64(width), ptr(a["free"]), i64(capacity), ptr(a["num_free"]), i64(bs),
                                               ptr(a["left"]), ptr(0))


def test_library_refuses_sizes_and_pointers_of_block_tables():
    before = _native.launch_count()
    big = 1 << 31
    for call, names in ((c_extend, EXTEND), (c_release, RELEASE)):
        assert call() > 0  # CUDA's own error: there is no device
        for bad, code in (({"reqs": -1}, -2), ({"width": -1}, -2), ({"capacity": -1}, -2), ({"bs": 0}, -2), ({"stride": 8}, -2), ({"reqs": 8193, "stride": 9}, -5), ({"width": big // 6 + 1, "stride": big}, -5), ({"width": big, "stride": big}, -5),
                          ({"capacity": big}, -5), ({"bs": big}, -5)):
            assert call(**bad) == code, bad
        assert call(stride=9) > 0
        for n in names:
            at = places(names)
            at[n] = 0
            assert call(at) == -1, n
            if n != "finished":
                at[n] = STEP * 50 + 2
                assert call(at) == -3, n
    assert c_extend(tokens=-1) == -2 and c_extend(tokens=big) == -5
    for n in ("positions", "slots"):
        assert c_extend(places(EXTEND) | {n: STEP * 50 + 4}) == -3
    assert _native.launch_count() == before


@pytest.mark.parametrize("call,sizes,results,own", [(c_extend, EXTEND_BYTES, ("table",) + EXTEND[5:], {("lens", "context"), ("left", "num_free")}), (c_release, RELEASE_BYTES, ("free", "left"), {("left", "num_free")})])
def test_library_refuses_results_that_overlap(call, sizes, results, own):
    up = lambda n: -(-n // 8) * 8  # noqa: E731
    for result in results:
        for other in set(sizes) - {result}:
            # in its place, on its last bytes, with its own last bytes on the other's first; then behind it, and in front of it
            for offset in (0, (sizes[other] - 1) // 8 * 8, -((sizes[result] - 1) // 8 * 8)):
                allowed = offset == 0 and ((result, other) in own or (other, result) in own)
                code = call(places(sizes) | {result: STEP * 40 + offset, other: STEP * 40})
                assert code > 0 if allowed else code == -6, (result, other, offset, code)
            for offset in (up(sizes[other]), -up(sizes[result])):
                assert call(places(sizes) | {result: STEP * 40 + offset, other: STEP * 40}) > 0, (result, other, offset)


def test_library_refuses_sizes_of_the_cache_in_4_bits():
    lib, a, before = library(), 1 << 32, _native.launch_count()

    def write(bs=64, pitch=64 * 368, tokens=4, inserted=4, q=a):
        return lib.dsv4_qnorm_rope_kv_insert_mxfp4(ptr(q), ptr(a), ptr(a), ptr(a), ptr(a), ptr(a), f32(1e-6), i64(tokens), i64(8), i64(inserted), i64(bs), i64(pitch), ptr(0))

    assert write() > 0 and write(tokens=0, inserted=0) == 0
    for bad, code in (({"pitch": 64 * 368 - 1}, -2), ({"bs": 65}, -2), ({"bs": 0}, -2), ({"bs": 1 << 61}, -2), ({"inserted": 5}, -2), ({"tokens": -1}, -2), ({"q": 0}, -1), ({"q": a + 1}, -3)):
        assert write(**bad) == code, bad

    def paged(pitch=64 * 368, bs=64):
        return lib.dsv4_paged_latent_attention_mxfp4(ptr(a), i64(2048), i64(512), ptr(2 * a), i64(3), i64(pitch), i64(bs), ptr(3 * a), i64(5), i64(5), ptr(4 * a), ptr(5 * a), i64(2), i64(0), i64(0), ptr(0),
                                                     f32(0.05), ptr(6 * a), i64(2048), i64(512), ptr(0), i64(0), i64(0), i64(6), i64(4), ptr(7 * a), ptr(0))

    def sparse(pitch=64 * 368, bs=64):
        return lib.dsv4_sparse_latent_attention_mxfp4(ptr(a), i64(2048), i64(512), ptr(2 * a), i64(3), i64(pitch), i64(bs), ptr(3 * a), i64(32), i64(32), ptr(4 * a), ptr(0), f32(0.05), ptr(6 * a), i64(2048),
                                                      i64(512), ptr(0), i64(0), i64(0), i64(6), i64(4), ptr(7 * a), ptr(0))

    for call in (paged, sparse):
        assert call() > 0 and call(pitch=64 * 368 - 16) == -2 and call(bs=65) == -2 and call(pitch=64 * 368 + 8) == -3
    assert _native.launch_count() == before
