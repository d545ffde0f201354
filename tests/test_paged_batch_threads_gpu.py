"""Block tables extended by two host threads at once, each on a stream and a pool of its own, with numbers of requests that need different amounts of shared memory:
what one call asks of the kernel must not be taken back by another."""
from __future__ import annotations

import threading

import pytest
import torch

import flaggems_vllm as fg
from test_paged_batch import DEV, Pool, extended

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,second", [(3500, 8192), (8192, 4097), (100, 8192)])
def test_two_threads_with_different_numbers_of_requests(first, second):
    calls = 4000
    pools = [Pool([(7 * i) % 90 for i in range(n)], [1] * n, 16, seed=n) for n in (first, second)]
    held, start, failures, last = [p.tensors()[0] for p in pools], threading.Barrier(2), [], [None, None]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()

    def work(which, requests):
        with torch.cuda.stream(streams[which]):
            out = fg.extend_block_tables(*held[which], 16, requests)
            start.wait()
            for call in range(calls):
                try:
                    last[which] = fg.extend_block_tables(*held[which], 16, requests, out)
                except Exception as error:  # noqa: BLE001
                    failures.append((requests, call, str(error)))
                    return

    threads = [threading.Thread(target=work, args=(i, n)) for i, n in enumerate((first, second))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert failures == []
    for p, got, requests in zip(pools, last, (first, second)):
        want, _ = extended(p.context, p.new, p.table, p.free, p.num_free, 16, requests)
        assert [t.tolist() for t in got] == list(want)
