"""Results of the attention operators and the residual norm that share memory with another argument are refused before anything is launched; results
that only lie between another argument's rows are not."""
from __future__ import annotations

import ctypes
import itertools
import subprocess

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native, build
from test_latent_attention import make_cache

i64, f32, ptr = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
OVERLAP, STEP = -6, 1 << 32
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="accepted calls would launch on addresses that are not memory")
NAMES = ("q", "cache", "table", "seq", "start", "sink", "out", "lse", "workspace")


def paged(at, out_strides=(2048, 512), lse_strides=(4, 1), q_strides=(2048, 512), tokens=6, heads=4):
    return ctypes.CDLL(str(_native.LIB_PATH)).dsv4_paged_latent_attention(
        ptr(at["q"]), i64(q_strides[0]), i64(q_strides[1]), ptr(at["cache"]), i64(3), i64(64 * 584), i64(64), ptr(at["table"]), i64(5), i64(5), ptr(at["seq"]), ptr(at["start"]), i64(2),
        i64(0), i64(0), ptr(at["sink"]), f32(0.05), ptr(at["out"]), i64(out_strides[0]), i64(out_strides[1]), ptr(at["lse"]), i64(lse_strides[0]), i64(lse_strides[1]), i64(tokens),
        i64(heads), ptr(at["workspace"]), ptr(0))


def places():
    return {name: STEP * (i + 1) for i, name in enumerate(NAMES)}


def accepted(code):
    return code > 0  # an error of CUDA: there is no device here


@no_gpu
def test_paged_results_that_overlap_an_argument():
    sizes = {"q": 6 * 4 * 1024, "cache": 3 * 64 * 584, "table": 40, "seq": 8, "start": 12, "sink": 16, "out": 6 * 4 * 1024, "lse": 6 * 4 * 4}
    assert accepted(paged(places()))
    for result in ("out", "lse"):
        for other in set(sizes) - {result}:
            if other == "out" and result == "lse":
                continue  # (the pair the other way round)
            step = 16 if result == "out" else 4
            for offset, wrong in ((0, True), (step - sizes[result], True), (-sizes[result], False), ((sizes[other] - 1) // step * step, True), (-(-sizes[other] // step) * step, False)):
                at = places()
                at[result] = at[other] + offset
                code = paged(at)
                assert code == OVERLAP if wrong else accepted(code), (result, other, offset, code)


@no_gpu
def test_results_between_the_rows_of_another_argument():
    """q, out and lse as parts of one wide buffer: every head 512 of 1088 values for q, 512 for out and 2 (one fp32) of the rest."""
    at = places()
    wide = (4 * 1088, 1088)
    for out, lse, wrong in ((1024, 2048, False), (1008, 2048, True), (1024, 2040, True), (1024, 2172, False), (1168, 2048, True), (1152, 2048, True)):
        at["out"], at["lse"] = at["q"] + out, at["q"] + lse
        code = paged(at, wide, (4 * 544, 544), wide)
        assert code == OVERLAP if wrong else accepted(code), (out, lse, code)


@no_gpu
def test_sparse_results_that_overlap_an_argument():
    def sparse(at):
        return ctypes.CDLL(str(_native.LIB_PATH)).dsv4_sparse_latent_attention(
            ptr(at["q"]), i64(2048), i64(512), ptr(at["cache"]), i64(3), i64(64 * 584), i64(64), ptr(at["table"]), i64(32), i64(32), ptr(at["seq"]), ptr(at["sink"]), f32(0.05),
            ptr(at["out"]), i64(2048), i64(512), ptr(at["lse"]), i64(4), i64(1), i64(6), i64(4), ptr(at["workspace"]), ptr(0))

    assert accepted(sparse(places()))
    for result, other in itertools.product(("out", "lse"), ("q", "cache", "table", "seq", "sink", "lse")):
        at = places()
        if result != other:
            at[result] = at[other]
            assert sparse(at) == OVERLAP, (result, other)


@no_gpu
def test_norm_results_that_overlap_an_argument():
    def norm(at, strides=(512, 512), scale_strides=(4, 1)):
        return ctypes.CDLL(str(_native.LIB_PATH)).dsv4_fused_add_rmsnorm_quant_fp8(
            ptr(at["x"]), i64(strides[0]), ptr(at["residual"]), i64(strides[1]), ptr(at["w"]), ptr(at["out"]), ptr(at["scales"]), i64(scale_strides[0]), i64(scale_strides[1]), i64(4),
            i64(512), i64(128), f32(1e-6), 0, 0, 0, ptr(0))

    names = ("x", "residual", "w", "out", "scales")
    fresh = lambda: {name: STEP * (i + 1) for i, name in enumerate(names)}  # noqa: E731
    assert accepted(norm(fresh()))
    for a, b in itertools.combinations(names, 2):
        at = fresh()
        at[a] = at[b]
        code = norm(at)
        assert code == OVERLAP if (a, b) != ("x", "w") else accepted(code), (a, b, code)
    at = fresh()
    at["residual"] = at["x"] + 1024  # the right halves of rows of 1024
    assert accepted(norm(at, (1024, 1024))) and norm(at, (1016, 1016)) == OVERLAP


@pytest.fixture(scope="module")
def regions(tmp_path_factory):
    """memory_regions.h behind a C function."""
    at = tmp_path_factory.mktemp("regions")
    (at / "r.cpp").write_text(f'''#include "{build.CSRC / 'memory_regions.h'}"
extern "C" int apart(const int64_t* a, const int64_t* b) {{
    const auto region = [](const int64_t* v) {{ return dsv4::Region(reinterpret_cast<const void*>(v[0]), v[1], {{{{v[2], v[3]}}, {{v[4], v[5]}}, {{v[6], v[7]}}}}); }};
    return dsv4::regions_apart(region(a), region(b));
}}''')
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-o", str(at / "r.so"), str(at / "r.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "r.so"))
    return lambda a, b: bool(lib.apart((i64 * 8)(*a), (i64 * 8)(*b)))


def test_regions_against_their_bytes(regions):
    """Never apart where a byte is shared; apart where ranges, or the columns of one pitch, are."""
    import random

    rng = random.Random(1)

    def some():
        return [rng.randrange(1000, 1060), rng.randrange(0, 6), *(v for _ in range(3) for v in (rng.randrange(0, 4), rng.choice([0, 1, 2, 3, 5, 6, 8, 12, 24, -6, -8])))]

    def bytes_of(v):
        return {v[0] + i * v[3] + j * v[5] + k * v[7] + n for i in range(v[2]) for j in range(v[4]) for k in range(v[6]) for n in range(v[1])}

    both = [0, 0]
    for _ in range(20000):
        a, b = some(), some()
        share = bool(bytes_of(a) & bytes_of(b))
        answer = regions(a, b)
        assert not (share and answer), (a, b)
        both[answer] += not share
    assert both[1] > 2 * both[0]
    far = 1 << 62
    assert regions([1000, 1 << 40, far, far, 1, 0, 1, 0], [1000, 0, 1, 0, 1, 0, 1, 0]) and not regions([1000, 1 << 40, far, far, 1, 0, 1, 0], [1000 + far, 4, 1, 0, 1, 0, 1, 0])


def test_tensors_against_their_elements():
    """The assertions' form of the same decision: never apart where an element is shared, apart for disjoint columns of one buffer."""
    import random

    from flaggems_vllm.utils.memory import apart

    rng, buffer = random.Random(2), torch.arange(4000, dtype=torch.int16)

    def some():
        return buffer.as_strided((rng.randrange(1, 4), rng.randrange(1, 4), rng.randrange(1, 6)), (rng.choice([1, 5, 6, 8, 12, 24, 48]), rng.choice([1, 5, 6, 8, 12, 24]), 1), rng.randrange(60))

    for _ in range(5000):
        a, b = some(), some()
        assert not (apart(a, b) and set(a.flatten().tolist()) & set(b.flatten().tolist())), (a.stride(), a.shape, b.stride(), b.shape)
    wide = buffer.view(10, 20, 20)
    assert apart(wide[:, :8], wide[:, 8:]) and apart(wide[..., :12], wide[..., 12:]) and apart(wide[:, 3:7, 5:9], wide[:, 2:9, 9:14])
    assert not apart(wide[:, :9], wide[:, 8:]) and not apart(wide[..., :13], wide[..., 12:])


@pytest.mark.gpu
def test_disjoint_parts_of_one_buffer_are_taken():
    """q and out, x and residual as columns of one buffer: what a call with tensors of their own gives."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(5, 6, 512, generator=g).to(torch.bfloat16).to("cuda:0")
    cache = torch.randint(0, 120, (3, 64 * 584), generator=g, dtype=torch.uint8).to("cuda:0")
    indices = torch.randint(0, 3 * 64, (5, 40), generator=g, dtype=torch.int32).to("cuda:0")
    lens = torch.full((5,), 40, dtype=torch.int32, device="cuda:0")
    bits = lambda t: t.view(torch.int16)  # noqa: E731  (any bytes are a cache: rows may be NaN)
    for cache in (cache, make_cache(3, 64, g).to("cuda:0")):
        want = fg.sparse_latent_attention(q, cache, indices, lens, 64, 0.05)
        for wide, (a, b) in ((torch.zeros(5, 6, 1024, dtype=torch.bfloat16, device="cuda:0"), (lambda t: t[..., :512], lambda t: t[..., 512:])),
                             (torch.zeros(5, 12, 512, dtype=torch.bfloat16, device="cuda:0"), (lambda t: t[:, 6:], lambda t: t[:, :6]))):
            a(wide).copy_(q)
            assert torch.equal(bits(fg.sparse_latent_attention(a(wide), cache, indices, lens, 64, 0.05, None, b(wide))), bits(want)) and torch.equal(a(wide), q)
    assert torch.isfinite(want).all()
    x, residual = (torch.randn(9, 640, generator=g).to(torch.bfloat16).to("cuda:0") for _ in range(2))
    wide = torch.cat([x, residual], 1)
    weight = torch.ones(640, dtype=torch.bfloat16, device="cuda:0")
    want = fg.fused_add_rmsnorm_quant_fp8(x, residual, weight, 1e-6)
    got = fg.fused_add_rmsnorm_quant_fp8(wide[:, :640], wide[:, 640:], weight, 1e-6)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want)) and torch.equal(wide, torch.cat([x, residual], 1))


@pytest.mark.gpu
def test_overlapping_lse_and_cache_are_refused():
    q = torch.zeros(2, 4, 512, dtype=torch.bfloat16, device="cuda:0")
    cache = torch.zeros(2, 64 * 584, dtype=torch.uint8, device="cuda:0")
    ints = [torch.zeros(s, dtype=torch.int32, device="cuda:0") for s in ((1, 2), (1,), (2,))]
    out = torch.zeros_like(q)
    for o, lse in ((out, q.view(torch.float32)[:, :, 0]), (out, out.view(torch.float32)[:, :, 3]), (cache[0, : q.numel() * 2].view(torch.bfloat16).view(q.shape), None)):
        with pytest.raises(_native.Dsv4Error, match="overlap"):
            fg.paged_latent_attention(q, cache, *ints, 64, 0.05, None, 0, None, o, lse)
        with pytest.raises(_native.Dsv4Error, match="overlap"):
            fg.sparse_latent_attention(q, cache, torch.zeros(2, 3, dtype=torch.int32, device="cuda:0"), torch.zeros(2, dtype=torch.int32, device="cuda:0"), 64, 0.05, None, o, lse)
    weights = torch.ones(512, dtype=torch.bfloat16, device="cuda:0")
    with pytest.raises(_native.Dsv4Error, match="overlap"):
        fg.fused_add_rmsnorm_quant_fp8(torch.zeros(1, 512, dtype=torch.bfloat16, device="cuda:0"), weights.view(1, 512), weights, 1e-6)


@no_gpu
def test_front_ends_and_assertions_agree_on_parts_of_one_buffer(monkeypatch):
    """Native front end and Python assertions on out beside q, and residual beside x, in one buffer that is no memory."""
    from test_attention_operator_checks import OPS, accepts
    from test_host_checks_agree import BF16, Spec

    monkeypatch.setattr(torch.cuda, "_lazy_init", lambda: None)

    class At(Spec):
        def __init__(self, offset, *args, **kwargs):
            super().__init__(*args, **kwargs)
            self.offset = offset

        def make(self, keep):
            from test_attention_operator_checks import _capsule

            super().make(keep)
            keep[-1].data = (1 << 32) + self.offset
            return torch.utils.dlpack.from_dlpack(_capsule(keep[-1]))

    for name, index in (("paged", 10), ("sparse", 7)):
        op, args, _ = OPS[name]
        taken = 0
        for token, head, offset in ((4096, 1024, 1024), (4096, 1024, 1008), (4096, 512, 4096), (2048, 512, 4096), (4096, 1024, 1040), (4608, 1024, 1024), (4096, 512, 2048), (2064, 512, 4096)):
            changed = list(args)
            changed[0], changed[index] = At(0, BF16, 6, 4, 512, strides=(token, head, 1)), At(offset, BF16, 6, 4, 512, strides=(token, head, 1))
            native, python = accepts(op, tuple(changed), None, True, monkeypatch), accepts(op, tuple(changed), None, False, monkeypatch)
            assert native[0] == python[0], (name, token, head, offset, native, python)
            taken += native[0]
        assert taken == 2
    op, args, _ = OPS["norm"]
    for pitch, offset, fine in ((1024, 1024, True), (1016, 1024, False), (1024, 1008, False), (1024, 1040, False), (1040, 1040, True), (4096, 4096, True)):
        changed = (At(0, BF16, 6, 512, strides=(pitch, 1)), At(offset, BF16, 6, 512, strides=(pitch, 1))) + args[2:]
        assert accepts(op, changed, None, True, monkeypatch)[0] == accepts(op, changed, None, False, monkeypatch)[0] == fine, (pitch, offset)
