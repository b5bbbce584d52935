"""Page operations against lists on the host: tables, counts, lengths and contents have to be equal."""

import random

import numpy as np
import pytest
import torch

from diffspec_mi355x.core.kv_cache import compact_pages, extend_pages, fork_pages, free_pages
from oracle import pages as oracle

pytestmark = pytest.mark.gpu


class Pool:
    """A pool on the device and its restatement on the host."""

    def __init__(self, gpu, B, P, n_log, ps=4, L=2, Hk=2, D=8, dtype=torch.float32, lens=torch.int32, seed=0):
        self.gpu, self.ps = gpu, ps
        g = torch.Generator().manual_seed(seed)
        kv = torch.randn((L, 2, P, Hk, ps, D), generator=g).to(dtype)
        self.kv, self.dkv = kv.float().numpy().copy(), kv.to(gpu)
        self.table, self.ref, self.lens = [[-1] * n_log for _ in range(B)], [0] * P, [0] * B
        self.dtable = torch.full((B, n_log), -1, dtype=torch.int32, device=gpu)
        self.dref = torch.zeros(P, dtype=torch.int32, device=gpu)
        self.dlens = torch.zeros(B, dtype=lens, device=gpu)

    def idx(self, x, dtype=torch.int32):
        return torch.tensor(x, dtype=dtype, device=self.gpu)

    def fork(self, parents, children, dtype=torch.int32):
        want = oracle.fork(self.kv, self.table, self.ref, self.lens, parents, children, self.ps)
        got = fork_pages(self.dkv, self.dtable, self.dref, self.dlens, self.idx(parents, dtype), self.idx(children, dtype))
        self.same(want, got)
        return want

    def extend(self, new, dtype=torch.int32):
        want = oracle.extend(self.table, self.ref, self.lens, new, self.ps)
        got = extend_pages(self.dtable, self.dref, self.dlens, self.idx(new, dtype), self.ps)
        self.same(want, got)
        return want

    def free(self, seqs, window=None, sinks=0):
        oracle.free(self.table, self.ref, self.lens, seqs, self.ps, window, sinks)
        free_pages(self.dtable, self.dref, self.dlens, self.idx(seqs), self.ps, window, sinks)
        self.same()

    def compact(self):
        want = oracle.compact(self.kv, self.table, self.ref)
        self.same(want, compact_pages(self.dkv, self.dtable, self.dref))
        return want

    def same(self, want=None, got=None):
        if want is not None:
            assert tuple(got.tolist()) == want
        assert self.dtable.tolist() == self.table
        assert self.dref.tolist() == self.ref
        assert self.dlens.tolist() == self.lens
        assert np.array_equal(self.dkv.float().cpu().numpy(), self.kv)


def test_fork_extend_free(gpu):
    p = Pool(gpu, B=7, P=40, n_log=6)
    assert p.extend([9, 0, 8, 0, 0, 0, 1]) == (6, 0, 0)
    assert p.fork([0, 2, 0, 6], [1, 3, 4, 5]) == (3, 0, 0)   # sequence 2 ends with its page
    p.extend([12, 13, 9, 0, 24, 1, 1])
    p.free([0, 0, 4])                                        # named twice: once
    p.free([3, -1, 99])                                      # out of range: skipped
    p.extend([4, 13, 9, 0, 24, 1, 1])
    p.free([1, 2, 5, 6, 0])
    p.free([4])
    assert sum(p.ref) == 0


@pytest.mark.parametrize("B", [5, 1100])
def test_extend_keeps_pages_behind_the_length(gpu, B):
    """Lengths set back after rejected tokens: their pages are used again, none is lost."""
    p = Pool(gpu, B=B, P=30 * B, n_log=80, L=1, Hk=1, lens=torch.int64)
    rng = random.Random(B)
    for _ in range(4):
        p.extend([min(320, n + rng.choice([0, 1, 3, 30, 33, 100])) for n in p.lens])
        p.free([rng.randrange(B) for _ in range(B // 3)], window=9, sinks=2)
        for b in range(B):
            p.lens[b] = rng.randint(0, p.lens[b]) if p.lens[b] and rng.random() < 0.5 else p.lens[b]
        p.dlens.copy_(torch.tensor(p.lens))
        assert sum(x >= 0 for row in p.table for x in row) == sum(p.ref)
        p.same()
    p.free(list(range(B)))
    assert sum(p.ref) == 0


def test_empty_lists_and_strided_indices(gpu):
    p = Pool(gpu, B=4, P=12, n_log=4)
    p.extend([5, 0, 9, 0])
    p.fork([], [])
    p.free([])
    p.extend([0, 0, 0, 0])
    wide = torch.tensor([0, 7, 2, 7], device=gpu)
    kids = torch.tensor([1, 7, 3, 7], device=gpu)
    oracle.fork(p.kv, p.table, p.ref, p.lens, [0, 2], [1, 3], p.ps)
    fork_pages(p.dkv, p.dtable, p.dref, p.dlens, wide[::2], kids[::2])
    p.same()
    oracle.free(p.table, p.ref, p.lens, [0, 2], p.ps)
    free_pages(p.dtable, p.dref, p.dlens, wide[::2], p.ps)
    p.same()


def test_nothing_happens_without_enough_pages(gpu):
    p = Pool(gpu, B=5, P=6, n_log=8)
    p.extend([9, 9, 0, 0, 0])
    assert p.extend([13, 0, 4, 0, 0]) == (0, 2, 0)           # none left
    assert p.fork([0, 1], [2, 3]) == (0, 2, 0)
    p.free([1])
    assert p.fork([0, 0, 0], [2, 3, 4]) == (3, 0, 0)
    assert p.extend([33, 0, 9, 9, 9]) == (0, 0, 1)           # beyond the table's row
    assert p.extend([2, 0, 1, 9, 9]) == (0, 0, 0)            # shorter: as they are


def test_refused_pairs(gpu):
    p = Pool(gpu, B=6, P=30, n_log=4)
    p.extend([5, 6, 0, 0, 0, 0])
    for parents, children in [([0], [0]), ([0], [1]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([6], [2]), ([-1], [2]), ([0], [6]),
                              ([0, 0], [2, -3])]:
        n = p.fork(parents, children)
        assert n[0] == 0 and n[2] > 0
    assert p.fork([], []) == (0, 0, 0)
    assert p.fork([2, 3], [4, 5]) == (0, 0, 0)               # empty parents: empty children


@pytest.mark.parametrize("sinks,window", [(0, 1), (1, 5), (4, 8), (9, 3), (0, 1000)])
def test_free_behind_the_window(gpu, sinks, window):
    p = Pool(gpu, B=4, P=80, n_log=20, lens=torch.int64)
    p.extend([79, 8, 33, 0], dtype=torch.int64)
    p.fork([0], [3])
    p.free([0, 2, 1], window, sinks)
    p.extend([80, 9, 40, 79])
    p.free([0, 1, 2, 3], window, sinks)
    p.compact()
    p.free([0, 1, 2, 3])
    assert sum(p.ref) == 0


@pytest.mark.parametrize("huge", [1 << 62, 1 << 63, (1 << 64) + 1])
def test_free_behind_a_window_beyond_64_bits(gpu, huge):
    """Nothing lies behind a window (or outside sinks) beyond every token."""
    p = Pool(gpu, B=2, P=40, n_log=20)
    p.extend([79, 33])
    p.free([0, 1], window=huge)
    p.free([0, 1], window=1, sinks=huge)
    assert sum(p.ref) == 20 + 9


@pytest.mark.parametrize("dtype,ps,Hk,D,L", [(torch.bfloat16, 16, 8, 128, 2), (torch.float16, 1, 1, 8, 1),
                                             (torch.float32, 8, 3, 20, 3), (torch.bfloat16, 64, 5, 72, 1)])
def test_random_calls(gpu, dtype, ps, Hk, D, L):
    """Many rounds of all four, with shared pages freed in any order."""
    rng = random.Random(ps * 7 + D)
    B, n_log, P = 9, 5, 30
    p = Pool(gpu, B, P, n_log, ps, L, Hk, D, dtype)
    for _ in range(25):
        live = [b for b in range(B) if p.lens[b]]
        empty = [b for b in range(B) if not p.lens[b]]
        k = rng.randrange(5)
        if k == 0:
            p.extend([rng.randrange(0, n_log * ps + 1) for _ in range(B)])
        elif k == 1 and live and empty:
            kids = rng.sample(empty, rng.randint(1, len(empty)))
            p.fork([rng.choice(live) for _ in kids], kids, torch.int64)
        elif k == 2:
            p.free(rng.sample(range(B), 3))
        elif k == 3:
            p.free(rng.sample(range(B), 4), window=rng.randint(1, 2 * ps), sinks=rng.choice([0, 1, ps]))
        else:
            p.compact()
    p.free(list(range(B)))
    assert sum(p.ref) == 0
    assert p.compact() == (0, 0, 0)


def test_many_pages_and_sequences(gpu):
    """More pages than a scan step and more sequences than threads."""
    p = Pool(gpu, B=1500, P=40000, n_log=30, ps=2, L=1, Hk=1, D=8, dtype=torch.bfloat16)
    rng = random.Random(3)
    p.extend([rng.randrange(0, 40) if b < 1400 else 0 for b in range(1500)])
    p.free(rng.sample(range(1400), 700))
    p.fork([b for b in range(1400) if p.lens[b]][:100], list(range(1400, 1500)))
    n = p.compact()
    assert n[1] > 0
    p.extend([60] * 1500)      # 1500 x 30 pages: too many
    p.extend([50] * 1500)
    p.compact()


def test_strided_pool(gpu):
    """Layers, halves, heads and tokens at strides of their own."""
    P, L, Hk, ps, D = 12, 2, 3, 4, 16
    p = Pool(gpu, 4, P, 6, ps, L, Hk, D, torch.bfloat16)
    big = torch.zeros(P, 2, L + 1, ps, Hk, D + 8, dtype=torch.bfloat16, device=gpu)
    view = big.permute(2, 1, 0, 4, 3, 5)[:L, ..., :D]
    view.copy_(p.dkv)
    p.dkv = view
    rows = torch.full((4, 9), -7, dtype=torch.int32, device=gpu)
    rows[:, :6] = p.dtable
    p.dtable = rows[:, :6]
    p.dref = torch.zeros(P + 1, dtype=torch.int32, device=gpu)[1:]  # 4-byte aligned
    p.extend([10, 3, 0, 0])
    p.fork([0, 1], [2, 3])
    p.free([0])
    p.compact()
    assert bool((rows[:, 6:] == -7).all())                    # behind the rows: as they were
    assert bool((big[:, :, L:] == 0).all()) and bool((big[..., D:] == 0).all())


def test_graph_replays(gpu):
    """fork + extend + free captured once and replayed from restored tables."""
    p = Pool(gpu, B=6, P=30, n_log=5)
    p.extend([9, 7, 0, 0, 0, 0])
    state = [p.dtable, p.dref, p.dlens, p.dkv]
    saved = [x.clone() for x in state]
    args = [p.idx([0, 1, 0]), p.idx([2, 3, 4]), p.idx([12, 8, 9, 9, 20, 0]), p.idx([0, 3])]

    def calls():
        a = fork_pages(p.dkv, p.dtable, p.dref, p.dlens, args[0], args[1])
        b = extend_pages(p.dtable, p.dref, p.dlens, args[2], p.ps)
        free_pages(p.dtable, p.dref, p.dlens, args[3], p.ps)
        return a, b, compact_pages(p.dkv, p.dtable, p.dref)

    info = [x.tolist() for x in calls()]
    want = [x.clone() for x in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for _ in range(3):
        for x, y in zip(state, saved):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(state, want):
            assert torch.equal(x, y)
        assert [x.tolist() for x in out] == info
