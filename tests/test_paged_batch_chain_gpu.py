"""Steps whose lengths, table and pool go on in place, one launch behind another without a synchronisation: what one SM wrote is read by the next launch on others.
Every step of more than 1024 tokens is made by several CTAs.  Eager and replayed chains have to give the numbers of the definition."""
from __future__ import annotations

import random

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from test_paged_batch import DEV, Pool, extended, i32, released

pytestmark = pytest.mark.gpu
BS = 16


def kept(finished, lens):
    return [0 if f else n for f, n in zip(finished, lens)]


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("requests,chunk,steps", [(2000, 1, 25), (8192, 1, 10), (61, 130, 12), (1500, 9, 8)])
def test_chain_in_place(requests, chunk, steps, captured, mode):
    r = random.Random(requests)
    new = [r.randint(0, chunk) if chunk > 1 else 1 for _ in range(requests)]
    done = [[r.random() < 0.3 for _ in range(requests)] for _ in range(2)]  # who ends in even steps, and in odd ones
    p = Pool([r.randrange(200) for _ in range(requests)], [(steps + 1) * n for n in new], BS, seed=requests, spare=9)
    tokens = sum(new)
    context, table, free, count, seen = p.context, p.table, p.free, p.num_free, []
    for step in range(steps):
        want, table = extended(context, new, table, free, count, BS, tokens)
        free, count = released(want[1], done[step & 1], table, free, want[5][0], BS)
        context = kept(done[step & 1], want[1])
        seen.append((want[0], *want[2:5]))

    before = _native.set_pdl(mode)
    try:
        (lens, _, tab, stack, num_free), _ = p.tensors()
        new_lens, finished = i32(new).to(DEV), [torch.tensor(d, device=DEV) for d in done]
        out = [torch.zeros(requests + 1, dtype=torch.int32, device=DEV), lens, *(torch.zeros(tokens, dtype=torch.int64, device=DEV) for _ in range(2)),
               torch.zeros(tokens, dtype=torch.int32, device=DEV), num_free, torch.zeros(1, dtype=torch.int32, device=DEV)]
        results = [[torch.zeros_like(out[i]) for i in (0, 2, 3, 4)] for _ in range(steps)]

        def chain():
            for step in range(steps):
                fg.extend_block_tables(lens, new_lens, tab, stack, num_free, BS, tokens, out)
                fg.release_block_tables(lens, finished[step & 1], tab, stack, num_free, BS, num_free)
                lens.masked_fill_(finished[step & 1], 0)
                for to, i in zip(results[step], (0, 2, 3, 4)):
                    to.copy_(out[i])

        state = [(t, t.clone()) for t in (lens, tab, stack, num_free)]
        if captured:
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                chain()
                for t, k in state:
                    t.copy_(k)
                with torch.cuda.graph(graph, stream=stream):
                    chain()
            stream.synchronize()
        for _ in range(2):
            for t, k in state:
                t.copy_(k)
            graph.replay() if captured else chain()
            torch.cuda.synchronize()
            for step, (got, want) in enumerate(zip(results, seen)):
                assert [t.tolist() for t in got] == [list(w) for w in want], step
            assert lens.tolist() == context and num_free.tolist() == [count] and tab.tolist() == table and stack.tolist()[:count] == free[:count]
    finally:
        _native.set_pdl(before)


@pytest.mark.parametrize("requests,steps", [(2000, 40), (8192, 25)])
def test_extends_directly_behind_one_another(requests, steps):
    """Nothing but launches that start while the one in front ends: lengths written by one CTA are read by all of the next launch."""
    p = Pool([(11 * i) % 100 for i in range(requests)], [steps] * requests, BS, seed=steps, spare=3)
    (lens, _, table, free, num_free), _ = p.tensors()
    ones = torch.ones(requests, dtype=torch.int32, device=DEV)
    results = []
    for _ in range(steps):
        out = [torch.zeros(requests + 1, dtype=torch.int32, device=DEV), lens, *(torch.zeros(requests, dtype=torch.int64, device=DEV) for _ in range(2)),
               torch.zeros(requests, dtype=torch.int32, device=DEV), num_free, torch.zeros(1, dtype=torch.int32, device=DEV)]
        results.append(out)
    torch.cuda.synchronize()
    for out in results:
        fg.extend_block_tables(lens, ones, table, free, num_free, BS, requests, out)
    left = fg.release_block_tables(lens, ones.bool(), table, free, num_free, BS)
    torch.cuda.synchronize()
    context, rows, count = p.context, p.table, p.num_free
    for out in results:
        want, rows = extended(context, [1] * requests, rows, p.free, count, BS, requests)
        context, count = want[1], want[5][0]
        assert [out[i].tolist() for i in (0, 2, 3, 4)] == [want[i] for i in (0, 2, 3, 4)]
    stack, total = released(context, [True] * requests, rows, p.free, count, BS)
    assert lens.tolist() == context and table.tolist() == rows and left.tolist() == [total] and free.tolist() == stack
