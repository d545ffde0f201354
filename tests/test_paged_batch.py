"""Block tables and slots of a step against their definition, a loop over requests on the host: every number is whole and has to be equal."""
from __future__ import annotations

import random

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native

gpu = pytest.mark.gpu
DEV = "cuda:0"
INT_MAX = 2**31 - 1


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


def extended(context, new, table, free, num_free, bs, num_tokens):
    """The definition.  Returns the PagedBatch as lists, and the table."""
    table, stack = [list(row) for row in table], list(free[: min(max(num_free, 0), len(free))])
    width = len(table[0]) if table else 0
    missing, starts, lens, tokens = 0, [0], [], []
    for r, (c, n) in enumerate(zip(context, new)):
        c, n = max(c, 0), max(n, 0)
        end = min(c + n, INT_MAX)
        for page in range(min(-(-c // bs), width), min(-(-end // bs), width)):
            empty = not stack
            table[r][page] = -1 if empty else stack.pop()
            missing += empty
        for p in range(c, c + min(n, max(0, num_tokens - len(tokens)))):
            block = table[r][p // bs] if p <= INT_MAX and p // bs < width else -1
            tokens.append((p, block * bs + p % bs if block >= 0 else -1, r))
        starts.append(min(starts[-1] + n, INT_MAX))
        lens.append(end)
    tokens += [(0, -1, 0)] * (num_tokens - len(tokens))
    return (starts, lens, *([t[i] for t in tokens] for i in range(3)), [len(stack)], [missing]), table


def released(lens, finished, table, free, num_free, bs):
    free, num_free = list(free), min(max(num_free, 0), len(free))
    back = [e for n, done, row in zip(lens, finished, table) if done for e in row[: -(-max(n, 0) // bs)] if e >= 0]
    for i, e in enumerate(reversed(back)):
        if num_free + i < len(free):
            free[num_free + i] = e
    return free, min(num_free + len(back), len(free))


class Pool:
    """Requests with blocks of their own out of a shuffled pool, and the rest of it as the stack."""

    def __init__(self, context, new, bs, seed=0, width=None, spare=3, short=0, row=0, holes=False):
        r = random.Random(seed)
        self.context, self.new, self.bs = list(context), list(new), bs
        held = [-(-max(c, 0) // bs) for c in context]
        need = [-(-(max(c, 0) + max(n, 0)) // bs) for c, n in zip(context, new)]
        self.width = max(need + [1]) if width is None else width
        blocks = list(range(sum(held) + sum(need) - sum(held) + spare))
        r.shuffle(blocks)
        self.table = [[blocks.pop() if i < h else -7 for i in range(self.width)] for h in held]
        if holes:
            for row_of in self.table:
                for i in range(self.width):
                    if row_of[i] >= 0 and r.random() < 0.2:
                        row_of[i] = -1
        self.num_free = max(0, len(blocks) - spare - short)
        self.free = blocks
        self.row = row  # entries between the rows

    def tensors(self):
        wide = torch.full((len(self.context), self.width + self.row), -9, dtype=torch.int32)
        wide[:, : self.width] = i32(self.table).view(len(self.context), self.width)
        wide = wide.to(DEV)
        return (i32(self.context).to(DEV), i32(self.new).to(DEV), wide[:, : self.width], i32(self.free).to(DEV), i32([self.num_free]).to(DEV)), wide

    def check(self, num_tokens=None, **options):
        num_tokens = sum(max(n, 0) for n in self.new) if num_tokens is None else num_tokens
        args, wide = self.tensors()
        got = fg.extend_block_tables(*args, self.bs, num_tokens, **options)
        want, table = extended(self.context, self.new, self.table, self.free, self.num_free, self.bs, num_tokens)
        for name, t, w in zip(got._fields, got, want):
            assert t.tolist() == w, name
        assert args[2].tolist() == table and (wide[:, self.width :] == -9).all()
        assert args[0].tolist() == self.context and args[3].tolist() == self.free and args[4].tolist() == [self.num_free]
        return got, args


@gpu
@pytest.mark.parametrize("bs", [1, 7, 16, 64, 256])
@pytest.mark.parametrize("context,new", [([0], [0]), ([0], [1]), ([1000], [1]), ([63, 64, 65], [1, 1, 1]), ([0, 5, 0, 300], [130, 0, 1, 70]), ([-3, 4], [2, -5])])
def test_extend_small(context, new, bs):
    Pool(context, new, bs).check()


@gpu
@pytest.mark.parametrize("requests,chunk,context,bs", [(61, 1, 16384, 64), (128, 1, 500, 16), (129, 3, 500, 16), (513, 2, 90, 16), (1024, 1, 200, 32), (1025, 9, 77, 16), (300, 170, 999, 64),
                                                       (4096, 7, 100, 16), (8192, 2, 40, 16), (1, 20000, 3, 64), (2, 40000, 100, 16), (3, 400000, 70, 64)])
def test_extend_large(requests, chunk, context, bs):
    r = random.Random(requests)
    Pool([r.randrange(context) for _ in range(requests)], [r.randint(0, chunk) for _ in range(requests)], bs, seed=requests, row=5).check()


@gpu
@pytest.mark.parametrize("missing", [1, 5, 1000])
def test_extend_with_too_few_free_blocks(missing):
    got, _ = Pool([10, 20, 30, 0], [100, 50, 3, 90], 16, short=missing).check()
    assert 0 < got.num_missing.item() <= missing and (got.slot_mapping == -1).any()


@gpu
def test_extend_counts_of_free_blocks_outside_the_stack():
    for count in (-1, -(2**31), 10**6, INT_MAX):
        p = Pool([10, 0], [50, 40], 16)
        p.num_free = count
        p.check()


@gpu
@pytest.mark.parametrize("width", [0, 1, 3, 5])
def test_extend_tables_that_are_too_narrow(width):
    Pool([20, 70, 0], [60, 40, 33], 16, width=width).check()


@gpu
@pytest.mark.parametrize("num_tokens", [0, 1, 10, 99, 100, 101, 131, 5000])
def test_extend_padded_and_cut_batches(num_tokens):
    Pool([3, 0, 40], [30, 0, 70], 16, spare=8).check(num_tokens)


@gpu
def test_extend_without_requests():
    args = (i32([]).to(DEV), i32([]).to(DEV), torch.empty(0, 4, dtype=torch.int32, device=DEV), i32([5, 6]).to(DEV), i32([2]).to(DEV))
    got = fg.extend_block_tables(*args, 16, 3)
    assert [t.tolist() for t in got] == [[0], [], [0, 0, 0], [-1, -1, -1], [0, 0, 0], [2], [0]]
    args = args[:3] + (i32([]).to(DEV), i32([0]).to(DEV))
    assert fg.extend_block_tables(*args, 16, 0).num_free.tolist() == [0]


@gpu
def test_extend_lengths_at_the_end_of_32_bits():
    """Sums stop at 2^31 - 1, positions go on in 64 bits; a block number times a block's tokens passes 32 bits."""
    p = Pool([0, 0, 0], [3, 3, 3], 1 << 20, width=2)
    p.table = [[INT_MAX, 1], [5, INT_MAX - 1], [-1, 2]]
    p.context, p.new = [17, INT_MAX - 2, (1 << 20) + 4], [INT_MAX, 9, 2]
    p.check(40)
    p.new = [2, 9, 2]
    got, _ = p.check(13)
    assert got.slot_mapping[0].item() == INT_MAX * (1 << 20) + 17 and got.position_ids[10].item() == INT_MAX + 6


@gpu
def test_extend_block_numbers_of_the_stack_are_copied():
    p = Pool([0], [3], 1, spare=0)
    p.free = [INT_MAX, -5, 0]
    p.num_free = 3
    got, args = p.check()
    assert args[2].tolist() == [[0, -5, INT_MAX]] and got.slot_mapping.tolist() == [0, -1, INT_MAX]


@gpu
def test_extend_writes_into_given_tensors_and_leaves_what_lies_around():
    p = Pool([5, 17, 0], [20, 1, 9], 16)
    args, _ = p.tensors()
    n, t = 3, 33
    room = {torch.int32: torch.full((200,), 77, dtype=torch.int32, device=DEV), torch.int64: torch.full((200,), 77, dtype=torch.int64, device=DEV)}
    at, out, live = {torch.int32: 1, torch.int64: 1}, [], {k: torch.zeros(200, dtype=torch.bool) for k in room}
    for of, size in zip((torch.int32, torch.int32, torch.int64, torch.int64, torch.int32, torch.int32, torch.int32), (n + 1, n, t, t, t, 1, 1)):
        out.append(room[of][at[of] : at[of] + size])
        live[of][at[of] : at[of] + size] = True
        at[of] += size + 1
    got = fg.extend_block_tables(*args, 16, t, out)
    want, _ = extended(p.context, p.new, p.table, p.free, p.num_free, 16, t)
    assert all(a.data_ptr() == b.data_ptr() and a.tolist() == w for a, b, w in zip(got, out, want))
    for of in room:
        assert (room[of].cpu()[~live[of]] == 77).all()
    assert fg.extend_block_tables(*args, 16, t, got) is got


def decode_steps(steps, requests, bs, seed):
    """What `steps` steps of one token a request make of lengths, table and stack, by the definition."""
    r = random.Random(seed)
    p = Pool([r.randrange(200) for _ in range(requests)], [steps + 1] * requests, bs, seed=seed, spare=4)
    context, table, count, slots = list(p.context), p.table, p.num_free, []
    for _ in range(steps):
        want, table = extended(context, [1] * requests, table, p.free, count, bs, requests)
        context, count = want[1], want[5][0]
        slots.append(want[3])
    return p, context, table, count, slots


@gpu
def test_extend_captured_with_its_state_in_place():
    """A decode step in a graph whose lengths and stack go on by themselves: 40 replays."""
    steps, requests, bs = 40, 37, 16
    p, context, table, count, slots = decode_steps(steps, requests, bs, 5)
    (lens, _, tab, free, num_free), _ = p.tensors()
    ones = torch.ones(requests, dtype=torch.int32, device=DEV)
    out = [torch.zeros(requests + 1, dtype=torch.int32, device=DEV), lens, *(torch.zeros(requests, dtype=torch.int64, device=DEV) for _ in range(2)),
           torch.zeros(requests, dtype=torch.int32, device=DEV), num_free, torch.zeros(1, dtype=torch.int32, device=DEV)]
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    kept = [t.clone() for t in (lens, tab, num_free)]
    with torch.cuda.stream(stream):
        fg.extend_block_tables(lens, ones, tab, free, num_free, bs, requests, out)
    torch.cuda.synchronize()
    for t, k in zip((lens, tab, num_free), kept):
        t.copy_(k)
    with torch.cuda.graph(graph):
        fg.extend_block_tables(lens, ones, tab, free, num_free, bs, requests, out)
    for step in range(steps):
        graph.replay()
        assert out[3].tolist() == slots[step]
    assert lens.tolist() == context and tab.tolist() == table and num_free.tolist() == [count]


@gpu
@pytest.mark.parametrize("tokens", [900, 1025, 5000, 30000])
def test_extend_in_place_with_many_tokens(tokens):
    r = random.Random(tokens)
    new = [r.randint(0, 2 * tokens // 40) for _ in range(40)]
    p = Pool([r.randrange(300) for _ in range(40)], new, 16, seed=tokens, spare=9)
    (lens, new_lens, table, free, num_free), _ = p.tensors()
    n = sum(new)
    out = [torch.zeros(41, dtype=torch.int32, device=DEV), lens, *(torch.zeros(n, dtype=torch.int64, device=DEV) for _ in range(2)), torch.zeros(n, dtype=torch.int32, device=DEV), num_free,
           torch.zeros(1, dtype=torch.int32, device=DEV)]
    fg.extend_block_tables(lens, new_lens, table, free, num_free, 16, n, out)
    want, wanted_table = extended(p.context, p.new, p.table, p.free, p.num_free, 16, n)
    assert [t.tolist() for t in out] == list(want) and table.tolist() == wanted_table


@gpu
@pytest.mark.parametrize("requests,context,bs,share", [(1, 100, 16, 1.0), (1, 100, 16, 0.0), (61, 16384, 64, 0.1), (61, 3000, 1, 0.5), (1021, 4000, 16, 0.5), (8192, 60, 16, 1.0), (33, 0, 16, 1.0), (3, 90000, 7, 1.0), (17, 20000, 1, 0.9)])
@pytest.mark.parametrize("holes", [False, True])
def test_release(requests, context, bs, share, holes):
    r = random.Random(requests)
    p = Pool([r.randint(0, context) for _ in range(requests)], [0] * requests, bs, seed=3, spare=17, holes=holes, row=2)
    p.num_free = 13
    finished = [r.random() < share for _ in range(requests)]
    p.free += [0] * sum(-(-c // bs) for c in p.context)
    (lens, _, table, free, num_free), _ = p.tensors()
    before = table.clone()
    got = fg.release_block_tables(lens, torch.tensor(finished, device=DEV), table, free, num_free, bs)
    want, count = released(p.context, finished, p.table, p.free, 13, bs)
    assert free.tolist() == want and got.tolist() == [count] and num_free.tolist() == [13] and torch.equal(table, before)


@gpu
def test_release_as_many_entries_as_a_table_can_have():
    """2^31 - 1 entries of one row: the last warp's part ends where a 32-bit position does."""
    n = INT_MAX
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GiB")
    table, free = torch.arange(n, dtype=torch.int32, device=DEV)[None], torch.full((n,), -7, dtype=torch.int32, device=DEV)
    got = fg.release_block_tables(i32([n]).to(DEV), torch.tensor([True], device=DEV), table, free, i32([0]).to(DEV), 1)
    assert got.tolist() == [n]
    for a in range(0, n, 1 << 28):
        b = min(a + (1 << 28), n)
        assert torch.equal(free[a:b], torch.arange(n - 1 - a, n - 1 - b, -1, dtype=torch.int32, device=DEV))
    table[0, -1] = -1  # a part with a hole: entry by entry
    got = fg.release_block_tables(i32([n]).to(DEV), torch.tensor([True], device=DEV), table, free, i32([0]).to(DEV), 1)
    assert got.tolist() == [n - 1] and free[:2].tolist() == [n - 2, n - 3] and free[n - 3 :].tolist() == [1, 0, 0]


@gpu
def test_release_stack_without_room_and_lengths_behind_the_table():
    p = Pool([100, 30, 500], [0] * 3, 16, spare=9, width=8)
    for count, lens in ((9, [100, 30, 500]), (3, [INT_MAX, -4, 128]), (-5, [0, 1, 16]), (10**9, [100, 30, 500])):
        (_, _, table, free, _), _ = p.tensors()
        got = fg.release_block_tables(i32(lens).to(DEV), torch.tensor([True, True, True], device=DEV), table, free, i32([count]).to(DEV), 16)
        want, left = released(lens, [True] * 3, p.table, p.free, count, 16)
        assert free.tolist() == want and got.tolist() == [left]


@gpu
def test_release_undoes_extend():
    """New requests take blocks and give them back: the stack is what it was, in its order."""
    p = Pool([0] * 50, [random.Random(i).randint(1, 900) for i in range(50)], 32, seed=9, spare=6)
    (context, new, table, free, num_free), _ = p.tensors()
    before = free.clone()
    batch = fg.extend_block_tables(context, new, table, free, num_free, 32, 0)
    assert batch.num_missing.item() == 0 and batch.num_free.item() < num_free.item()
    free[batch.num_free.item() :] = -3
    back = fg.release_block_tables(batch.seq_lens, torch.ones(50, dtype=torch.bool, device=DEV), table, free, batch.num_free, 32, batch.num_free)
    assert back.data_ptr() == batch.num_free.data_ptr() and back.item() == num_free.item()
    n = num_free.item()
    assert torch.equal(free[:n], before[:n])


@gpu
def test_release_without_requests():
    free = i32([4, 5, 6]).to(DEV)
    got = fg.release_block_tables(i32([]).to(DEV), torch.empty(0, dtype=torch.bool, device=DEV), torch.empty(0, 3, dtype=torch.int32, device=DEV), free, i32([2]).to(DEV), 16)
    assert got.tolist() == [2] and free.tolist() == [4, 5, 6]


@gpu
def test_calls_on_two_streams():
    """Two pools at once, each on a stream of its own."""
    pools = [Pool([random.Random(i + j).randrange(500) for i in range(400)], [5] * 400, 16, seed=j) for j in range(2)]
    held = [p.tensors()[0] for p in pools]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j] = fg.extend_block_tables(*held[j], 16, 2000)
    torch.cuda.synchronize()
    for p, g in zip(pools, got):
        want, _ = extended(p.context, p.new, p.table, p.free, p.num_free, 16, 2000)
        assert [t.tolist() for t in g] == list(want)


@gpu
def test_refusals_on_the_gpu():
    (context, new, table, free, num_free), _ = Pool([5, 17], [20, 1], 16).tensors()
    call = lambda *a, **k: fg.extend_block_tables(*a, **k)  # noqa: E731
    good = call(context, new, table, free, num_free, 16, 21)
    for bad in ({0: context.long()}, {1: new[:1]}, {2: table.t()}, {3: free.view(1, -1)}, {4: num_free.long()}, {5: 0}, {6: -1}, {2: table[:1]}, {0: context.cpu()}):
        args = [context, new, table, free, num_free, 16, 21]
        for i, v in bad.items():
            args[i] = v
        with pytest.raises(AssertionError):
            call(*args)
    with pytest.raises(_native.Dsv4Error, match="overlap"):
        call(context, new, table, table[0], num_free, 16, 21)
    for i, v in ((0, good.query_start_loc[:2]), (2, good.position_ids.int()), (4, good.seq_lens)):
        out = list(good)
        out[i] = v
        with pytest.raises(AssertionError):
            call(context, new, table, free, num_free, 16, 21, out)
    for i, v in ((1, new), (5, good.num_missing), (6, num_free)):
        out = list(good)
        out[i] = v
        with pytest.raises(_native.Dsv4Error, match="overlap"):
            call(context, new, table, free, num_free, 16, 21, out)
    with pytest.raises(AssertionError):
        call(context, new, table, free, num_free, 16, 21, list(good)[:6])
    done = torch.tensor([True, False], device=DEV)
    for bad in ({1: done.int()}, {1: done[:1]}, {6: num_free.long()}):
        args = [context, done, table, free, num_free, 16, None]
        for i, v in bad.items():
            args[i] = v
        with pytest.raises(AssertionError):
            fg.release_block_tables(*args)
    for bad in ({3: table[0]}, {6: free[:1]}):
        args = [context, done, table, free, num_free, 16, None]
        for i, v in bad.items():
            args[i] = v
        with pytest.raises(_native.Dsv4Error, match="overlap"):
            fg.release_block_tables(*args)
