"""The native front ends of the norm and attention operators refuse what the Python assertions behind them refuse, argument by argument;
no GPU (see test_host_checks_agree.py, whose tensors without memory are used)."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from test_host_checks_agree import BF16, F16, F32, I32, U8, Spec, changed_number

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="accepted calls would launch on addresses that are not memory")


def far(spec, at):
    """The same tensor in name, with an address of its own: the operators refuse outputs that overlap their inputs."""
    make = spec.make
    spec.make = lambda keep: make(keep) if spec.device is None else moved(make, keep, at)
    return spec


def moved(make, keep, at):
    t = make(keep)
    keep[-1].data = at
    return torch.utils.dlpack.from_dlpack(_capsule(keep[-1]))


def _capsule(t):
    import ctypes

    new = ctypes.pythonapi.PyCapsule_New
    new.restype, new.argtypes = ctypes.py_object, [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
    return new(ctypes.addressof(t), b"dltensor", None)


PAGED = (Spec(BF16, 6, 4, 512), Spec(U8, 3, 64 * 584), Spec(I32, 2, 5), Spec(I32, 2), Spec(I32, 3), 64, 0.05, 128, 4, Spec(F32, 4), Spec(BF16, 6, 4, 512), Spec(F32, 6, 4))
SPARSE = (Spec(BF16, 6, 4, 512), Spec(U8, 3, 64 * 584), Spec(I32, 6, 32), Spec(I32, 6), 64, 0.05, Spec(F32, 4), Spec(BF16, 6, 4, 512), Spec(F32, 6, 4))
NORM = (Spec(BF16, 6, 512), Spec(BF16, 6, 512), Spec(BF16, 512), 1e-6, 128, True, False)
OPS = {"paged": (fg.paged_latent_attention, PAGED, 10), "sparse": (fg.sparse_latent_attention, SPARSE, 7), "norm": (fg.fused_add_rmsnorm_quant_fp8, NORM, 1),
       "norm, fp16, weights in 32 bits": (fg.fused_add_rmsnorm_quant_fp8, (Spec(F16, 6, 512), Spec(F16, 6, 512), Spec(F32, 512), 1e-6, 512, False, True), 1)}
NATIVE = {fg.paged_latent_attention: ("_paged", "paged_latent_attention"), fg.sparse_latent_attention: ("_sparse", "sparse_latent_attention"),
          fg.fused_add_rmsnorm_quant_fp8: ("_call", "add_rmsnorm_quant")}
# Accepted by the assertions, refused by the library, which says why: numbers that are none, sizes of more than 64 bits.
TEXT = ("x", None)


def accepts(op, args, apart, native, monkeypatch):
    import importlib

    module, keep = importlib.import_module(op.__module__), []
    attribute, entry = NATIVE[op]
    call = getattr(_native.host_calls(), entry)
    monkeypatch.setattr(module, attribute, call if native else (lambda *a: None))
    tensors = []
    for i, a in enumerate(args):
        if isinstance(a, Spec):
            a = a.make(keep) if i != apart or a.device is None else moved(a.make, keep, 1 << 40)
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
    op, args, apart = OPS[name]
    assert accepts(op, args, apart, True, monkeypatch)[0] and accepts(op, args, apart, False, monkeypatch)[0]
    refused = 0
    for i, a in enumerate(args):
        if isinstance(a, bool):
            continue
        for c in a.changed() if isinstance(a, Spec) else changed_number(a) + ([0.0, -1.0, float("nan"), float("inf"), 1e300] if isinstance(a, float) else []):
            changed = args[:i] + (c,) + args[i + 1 :]
            (native, why), (python, _) = accepts(op, changed, apart, True, monkeypatch), accepts(op, changed, apart, False, monkeypatch)
            if python and c in TEXT:
                assert native or "the call was refused (" in why, (i, c, why)
            else:
                assert native == python, (i, c, why)
            refused += not native
    assert refused > 20


@pytest.mark.parametrize("name", OPS)
def test_optional_tensors_may_be_absent(name, monkeypatch):
    monkeypatch.setattr(torch.cuda, "_lazy_init", lambda: None)
    op, args, apart = OPS[name]
    optional = {"paged": (7, 9, 10, 11), "sparse": (6, 7, 8)}.get(name, (1,))
    for i in optional:
        changed = args[:i] + (None,) + args[i + 1 :]
        assert accepts(op, changed, apart, True, monkeypatch)[0] and accepts(op, changed, apart, False, monkeypatch)[0]


def test_library_refuses_sizes_before_any_launch():
    """The C entry points themselves, called with addresses that nothing may read."""
    import ctypes

    lib = ctypes.CDLL(str(_native.LIB_PATH))
    i64, f32, ptr = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
    before = _native.launch_count()
    a = 1 << 32

    def paged(q=a, qs=(2048, 512), cache=a, blocks=3, pitch=64 * 584, bs=64, table=a, max_blocks=5, seq=a, start=a, reqs=2, window=0, first=0, scale=0.05, out=2 * a,
              tokens=6, heads=4, workspace=a):
        return lib.dsv4_paged_latent_attention(ptr(q), i64(qs[0]), i64(qs[1]), ptr(cache), i64(blocks), i64(pitch), i64(bs), ptr(table), i64(5), i64(max_blocks), ptr(seq), ptr(start),
                                               i64(reqs), i64(window), i64(first), ptr(0), f32(scale), ptr(out), i64(2048), i64(512), ptr(0), i64(0), i64(0), i64(tokens),
                                               i64(heads), ptr(workspace), ptr(0))

    for bad, code in (({"tokens": -1}, -2), ({"heads": -1}, -2), ({"bs": 0}, -2), ({"bs": 65}, -2), ({"pitch": 64 * 584 - 16}, -2), ({"bs": 1 << 62}, -2), ({"scale": 0.0}, -2),
                      ({"scale": float("nan")}, -2), ({"scale": float("inf")}, -2), ({"reqs": -1}, -2), ({"window": -1}, -2), ({"first": -1}, -2), ({"max_blocks": -1}, -2),
                      ({"tokens": 1 << 31}, -5), ({"tokens": 1 << 30, "heads": 2}, -5), ({"blocks": 1 << 31}, -5), ({"reqs": 1 << 31}, -5), ({"q": 0}, -1), ({"out": 0}, -1),
                      ({"cache": 0}, -1), ({"table": 0}, -1), ({"seq": 0}, -1), ({"start": 0}, -1), ({"q": a + 2}, -3), ({"out": a + 8}, -3), ({"cache": a + 8}, -3),
                      ({"qs": (2048, 516)}, -3), ({"pitch": 64 * 584 + 8}, -3)):
        assert paged(**bad) == code, bad
    assert paged(tokens=0) == 0 and paged(heads=0) == 0 and paged(reqs=0) == 0

    def norm(x=a, residual=2 * a, w=a, out=3 * a, scales=a, rows=4, cols=512, group=128, strides=(512, 512)):
        return lib.dsv4_fused_add_rmsnorm_quant_fp8(ptr(x), i64(strides[0]), ptr(residual), i64(strides[1]), ptr(w), ptr(out), ptr(scales), i64(4), i64(1), i64(rows), i64(cols),
                                                    i64(group), f32(1e-6), 0, 0, 0, ptr(0))

    for bad, code in (({"rows": -1}, -2), ({"cols": -8}, -2), ({"cols": 508, "group": 508}, -2), ({"group": 96}, -2), ({"group": 0}, -2), ({"group": 512 * 2}, -2),
                      ({"strides": (504, 512)}, -2), ({"strides": (512, 504)}, -2), ({"x": 0}, -1), ({"w": 0}, -1), ({"out": 0}, -1), ({"scales": 0}, -1), ({"x": a + 8}, -3),
                      ({"residual": a + 8}, -3), ({"w": a + 8}, -3), ({"strides": (516, 512)}, -3), ({"cols": 32768 + 128, "strides": (1 << 20, 1 << 20)}, -5),
                      ({"rows": 1 << 31}, -5)):
        assert norm(**bad) == code, bad
    assert norm(rows=0) == 0 and norm(cols=0, group=128) == 0
    assert _native.launch_count() == before
