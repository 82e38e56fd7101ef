"""Pages and places of a step's tokens (ops.plan_paged_step) against a plain walk over the sequences."""
import random

import pytest
import torch

from sharq_b200 import ops

pytestmark = pytest.mark.gpu


def walk(table, lengths, counts, stack, free, page, rows, released, max_tokens=None):
    """The step on lists, sequence by sequence -> (offsets, positions, sequences, bad); the lists change as the operator's tensors do."""
    most = len(table[0])
    bad = not 0 <= free[0] <= len(stack)
    no_stack = bad
    top = 0 if bad else free[0]
    for i, ended in enumerate(released):
        if ended:
            if 0 <= lengths[i] <= most * page:
                for at in reversed(range(-(-lengths[i] // page))):
                    if no_stack or top >= len(stack):
                        bad = True
                    else:
                        stack[top] = table[i][at]
                        top += 1
            else:
                bad = True
            lengths[i] = 0
    offsets, positions, sequences, short, total = [0], [], [], False, 0
    for i, count in enumerate(counts):
        fits = lengths[i] >= 0 and count >= 0 and lengths[i] + count <= min(most * page, max_tokens or most * page)
        n = max(count, 0)
        total += n
        need = -(-(lengths[i] + count) // page) - -(-lengths[i] // page) if fits else 0
        bad = bad or not fits or total > rows
        short = short or need > top
        given = fits and not no_stack and total <= rows and not (short and need > 0)
        if given:
            held = -(-lengths[i] // page)
            for at in range(held, held + need):
                top -= 1
                table[i][at] = stack[top]
        here = min(n, rows - len(positions))
        positions += [lengths[i] + j if given else -1 for j in range(here)]
        sequences += [i] * here
        lengths[i] += n if given else 0
        offsets.append(min(total, rows))
    positions += [-1] * (rows - len(positions))
    sequences += [0] * (rows - len(sequences))
    if not no_stack:
        free[0] = top
    return offsets, positions, sequences, bad


class Server:
    def __init__(self, lengths, page, most, spare, seed, room=0):
        """Sequences in mid-flight, pages in random order; `spare` free ones, and places on the stack beyond all pages for `room` more."""
        rng = random.Random(seed)
        held = [-(-n // page) for n in lengths]
        order = list(range(sum(held) + spare))
        rng.shuffle(order)
        self.page, self.lengths, self.table, at = page, list(lengths), [], 0
        for n in held:
            self.table.append(order[at:at + n] + [-7] * (most - n))
            at += n
        self.stack = order[at:] + [-9] * (at + room)
        self.free = [spare]

    def step(self, counts, rows, released=None, stride=0, max_tokens=None):
        """One step by the operator and by the walk: both have to agree in everything -> (offsets, positions, sequences)."""
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        wide = torch.full((len(self.table), len(self.table[0]) + stride), -3, dtype=torch.int32, device="cuda")
        table = wide[:, :len(self.table[0])]
        table.copy_(dev(self.table))
        lengths, stack, free = dev(self.lengths), dev(self.stack), dev(self.free)
        flags = None if released is None else torch.tensor(released, dtype=torch.bool, device="cuda")
        got = ops.plan_paged_step(table, lengths, dev(counts), stack, free, self.page, rows, released=flags, max_tokens=max_tokens)
        *want, bad = walk(self.table, self.lengths, list(counts), self.stack, self.free, self.page, rows, released or [False] * len(counts),
                          max_tokens)
        for g, w in zip(got, want):
            assert g.tolist() == w
        assert table.tolist() == self.table and lengths.tolist() == self.lengths
        assert stack.tolist() == self.stack and free.tolist() == self.free
        assert (wide[:, len(self.table[0]):] == -3).all()
        if bad:
            with pytest.raises(RuntimeError, match="plan_paged_step"):
                ops.check_device_errors()
        ops.check_device_errors()
        return want


@pytest.mark.parametrize("seqs", [1, 5, 128, 129, 256, 257, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_decode_steps(seqs, page):
    rng = random.Random(seqs * 100 + page)
    server = Server([rng.randint(0, 60) for _ in range(seqs)], page, 80, 70 * seqs, seqs)
    for _ in range(3):
        server.step([1] * seqs, seqs)
    server.step([rng.randint(0, 1) for _ in range(seqs)], seqs, stride=3)


@pytest.mark.parametrize("seqs,longest,page", [(1, 5000, 16), (3, 4000, 24), (40, 700, 64), (300, 90, 8), (1500, 40, 16), (2049, 9, 1)])
def test_sequences_end_and_begin(seqs, longest, page):
    rng = random.Random(seqs + page)
    most = -(-2 * longest // page) + 3
    server = Server([rng.randint(0, longest) for _ in range(seqs)], page, most, seqs * (most // 2 + 1), 2)
    for _ in range(4):
        released = [rng.random() < 0.4 for _ in range(seqs)]
        counts = [rng.randint(0, longest) if r and rng.random() < 0.8 else int(rng.random() < 0.9) for r in released]
        counts = [min(c, most * page - (0 if r else n)) for c, r, n in zip(counts, released, server.lengths)]
        server.step(counts, sum(counts) + rng.choice((0, 1, 700)), released)


def test_pages_that_do_not_suffice():
    """All or nothing for a sequence; later ones that need a page get none either, those that need none go on."""
    server = Server([16, 5, 32, 7, 0, 16], 16, 9, 3, 5)
    offsets, positions, _ = server.step([1, 40, 1, 2, 0, 1], 60)
    assert positions[0] == 16 and positions[1:41] == list(range(5, 45)) and positions[41] == -1 and positions[42:44] == [7, 8] and positions[44] == -1
    assert offsets == [0, 1, 41, 42, 44, 44, 45]
    # the pages of a sequence that ends serve the step itself
    server = Server([64, 16, 16], 16, 9, 0, 6)
    server.step([0, 1, 1], 2, [True, False, False])
    assert server.free == [2] and server.lengths == [0, 17, 17]


@pytest.mark.parametrize("seqs", [6, 1100])
def test_what_cannot_be_is_reported(seqs):
    good = [20] * seqs
    for at, (length, count) in enumerate([(-1, 1), (20, -1), (20, 2 ** 31 - 1), (2 ** 31 - 1, 1), (9 * 16, 1), (9 * 16 + 1, 0)]):
        server = Server(good, 16, 9, 3 * seqs, 7)
        server.lengths[at % seqs] = length
        counts = [1] * seqs
        counts[at % seqs] = count
        server.step(counts, seqs + 5)
        if count >= 0:
            server = Server(good, 16, 9, 3 * seqs, 8)
            server.lengths[at % seqs] = length
            server.step(counts, seqs + 5, [i == at % seqs for i in range(seqs)])
    for free in (-1, 10 ** 6):
        server = Server(good, 16, 9, 3 * seqs, 9)
        server.free = [free]
        server.step([13] * seqs, 13 * seqs, [i % 2 == 0 for i in range(seqs)])
    server = Server(good, 16, 9, 3 * seqs, 9)
    server.step([1] * (seqs - 1) + [2], seqs + 1, max_tokens=21)
    server.step([1] * seqs, seqs, [True] * (seqs // 2) + [False] * (seqs - seqs // 2), max_tokens=1)
    # fewer rows than tokens
    server = Server(good, 16, 9, 3 * seqs, 10)
    server.step([2] * seqs, 2 * seqs - 3)
    server.step([2] * seqs, 0)
    # more pages come back than the stack has room for
    server = Server(good, 16, 9, 2, 11)
    server.stack = server.stack[:3]
    server.step([0] * seqs, 4, [True] * seqs)


def test_no_sequence_asks_for_anything_and_no_pages_at_all():
    server = Server([3, 0, 16], 16, 4, 0, 12)
    server.step([0, 0, 0], 0)
    server.step([1, 1, 1], 3)


def test_steps_of_a_captured_graph():
    """A replayed step reads what the step before it left."""
    n, page = 37, 16
    server = Server([i % 50 for i in range(n)], page, 40, 900, 13)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lengths, stack, free, counts = dev(server.table), dev(server.lengths), dev(server.stack), dev(server.free), dev([1] * n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.plan_paged_step(table, lengths, counts, stack, free, page, n)
        walk(server.table, server.lengths, [1] * n, server.stack, server.free, page, n, [False] * n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.plan_paged_step(table, lengths, counts, stack, free, page, n)
    for _ in range(20):
        graph.replay()
        offsets, positions, sequences, _ = walk(server.table, server.lengths, [1] * n, server.stack, server.free, page, n, [False] * n)
        assert [t.tolist() for t in got] == [offsets, positions, sequences]
    assert table.tolist() == server.table and lengths.tolist() == server.lengths and free.tolist() == server.free
    ops.check_device_errors()


def test_refusals():
    dev = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(page_table=dev(3, 4), lengths=dev(3), counts=dev(3), free_pages=dev(9), free_count=dev(1), page_size=16, rows=5)
    ops.plan_paged_step(**good)
    for name, value in [("page_table", dev(3, 4).long()), ("page_table", dev(4, 3).T), ("page_table", dev(3)), ("page_table", dev(3, 0)), ("lengths", dev(2)),
                        ("page_table", dev(1, 4).expand(3, 4)), ("lengths", dev(3).long()), ("lengths", dev(6)[::2]), ("counts", dev(3).cpu()),
                        ("free_pages", dev(9).long()), ("free_pages", dev(3, 3)), ("free_count", dev(2)), ("page_size", 0), ("page_size", -4),
                        ("rows", -1), ("max_tokens", 0), ("max_tokens", -1), ("rows", 2 ** 31), ("released", dev(3)), ("released", torch.zeros(2, dtype=torch.bool, device="cuda"))]:
        with pytest.raises(RuntimeError):
            ops.plan_paged_step(**{**good, name: value})
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.plan_paged_step(**{**good, "page_table": dev(3, 4).cpu()})
    ops.check_device_errors()
