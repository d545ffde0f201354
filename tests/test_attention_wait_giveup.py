"""Waits of the latent attention that run out (csrc/latent_attention.cu), without faulting or hanging anything.

Every wait of that kernel has a limit, and the limit is a setting: how often a try, of up to two microseconds, is made again.  With 0 to 12 the calls below, which
take 20 us and more, do not get through: some CTAs get further than others, so pieces of tiles are missing when the kernel behind joins them.
What must then happen: both kernels return by themselves, bit 1 of the device error word is set and cleared by the read, memory beside the
results stays, and the next ordinary call gives what it gave before, bit for bit."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from test_latent_attention import DEV, SCALE, Batch, sparse_case

DEFAULT = 1 << 22


def test_limit_round_trip():
    lib = _native.lib()
    assert lib.dsv4_set_attention_wait_retries(-1) == DEFAULT  # only reads
    try:
        assert lib.dsv4_set_attention_wait_retries(0) == DEFAULT
        assert lib.dsv4_set_attention_wait_retries(1 << 40) == 0
        assert lib.dsv4_set_attention_wait_retries(7) == DEFAULT  # clamped
    finally:
        assert lib.dsv4_set_attention_wait_retries(DEFAULT) == 7
    assert lib.dsv4_set_attention_wait_retries(-1) == DEFAULT


def _calls():
    """Name -> a call that writes into the tensor it is given: tiles that are cut (one token each, several), whole ones, lists of slots."""
    calls = {}
    for name, lens, new, heads, window in (("cut, one token", [9000, 77, 3001], [1, 1, 1], 128, None), ("cut, several tokens", [4000, 900], [37, 5], 16, None),
                                           ("whole", [330, 130], [3, 1], 64, 128)):
        b = Batch(lens, new, heads, 64, seed=len(name))
        args = (b.q.to(DEV), b.cache.to(DEV), b.table.to(DEV), torch.tensor(b.seq_lens, dtype=torch.int32, device=DEV), b.starts.to(DEV), 64, SCALE, window, 2, b.sink.to(DEV))
        calls[name] = (args[0].shape, lambda out, args=args: fg.paged_latent_attention(*args, out))
    cache, indices, lens, q, sink = (t.to(DEV) for t in sparse_case(30, 128, 1500, seed=3))
    calls["list"] = (q.shape, lambda out: fg.sparse_latent_attention(q, cache, indices, lens, 64, SCALE, sink, out))
    return calls


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["cut, one token", "cut, several tokens", "whole", "list"])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(name):
    shape, call = _calls()[name]
    lib = _native.lib()
    holder = torch.full((shape[0] + 2, *shape[1:]), 7.0, dtype=torch.bfloat16, device=DEV)
    out = holder[1:-1]
    call(out)
    torch.cuda.synchronize()
    want = out.clone()
    assert _native.device_error() == 0
    reported = 0
    for tries in (0, 1, 2, 3, 4, 6, 8, 12, 0):
        assert lib.dsv4_set_attention_wait_retries(tries) == DEFAULT
        try:
            call(out)
            torch.cuda.synchronize()  # returns: the kernels ended by themselves
        finally:
            assert lib.dsv4_set_attention_wait_retries(DEFAULT) == tries
        error = _native.device_error()
        assert error == 2 or (error == 0 and torch.equal(out, want))
        reported += error == 2
        assert _native.device_error() == 0, "reading the error word clears it"
        assert (holder[0] == 7).all() and (holder[-1] == 7).all()
        out.fill_(3.0)
        call(out)
        torch.cuda.synchronize()
        assert _native.device_error() == 0 and torch.equal(out, want)
    assert reported > 0, "none of the waits ran out"
