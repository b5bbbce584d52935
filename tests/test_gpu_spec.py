"""speculative_accept against the rule in float64 (exact: paths and tokens are whole numbers)."""

import numpy as np
import pytest
import torch

from diffspec_mi355x import workloads as wl
from diffspec_mi355x.draft.tree_verification import kv_commit, speculative_accept
from oracle import spec as oracle

pytestmark = pytest.mark.gpu


def make(T, M, V, dtype, sampled, seed, chain=False, peak=2.5, gap=0.8):
    """Target and draft rows, trees, tokens drawn from the draft, numbers."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((T, M, V), generator=g) * peak
    p = torch.softmax(z, -1).to(dtype)
    q = torch.softmax(z + gap * torch.randn((T, M, V), generator=g), -1).to(dtype)
    parents, draft = [], np.zeros((T, M), dtype=np.int64)
    for t in range(T):
        par = list(range(-1, M - 1)) if chain else wl.make_tree(M, max_depth=M, max_outdeg=4, seed=seed + t)[0]
        parents.append(wl.parent_to_reference(par))
        for i in range(1, M):
            row = q[t, par[i]].double().numpy()
            draft[t, i] = rng.choice(V, p=row / row.sum()) if sampled else int(rng.choice(np.argsort(-row)[:6]))
    u = torch.rand((T, M), generator=g)
    return p, q if sampled else None, torch.from_numpy(draft), torch.tensor(parents, dtype=torch.int64).view(T, M - 1), u


def check(gpu, p, q, draft, parent, u):
    r = speculative_accept(p.to(gpu), draft.to(gpu), parent.to(gpu), u.to(gpu), None if q is None else q.to(gpu))
    T, M, _ = p.shape
    pn, qn = p.double().numpy(), None if q is None else q.double().numpy()
    for t in range(T):
        path, nxt = oracle.speculative_walk(pn[t], draft[t].tolist(), parent[t].tolist(), u[t].tolist(),
                                            None if qn is None else qn[t])
        assert r["info"][t].tolist() == [path[-1], len(path) - 1, nxt, len(path)], t
        assert r["path"][t].tolist() == path + [-1] * (M - len(path))
        assert r["tokens"][t].tolist() == [int(draft[t, i]) for i in path] + [-1] * (M - len(path))
    return r


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,M,V,chain", [(1, 1, 1, False), (1, 2, 2, True), (3, 6, 4096, True), (2, 6, 4097, True),
                                         (4, 17, 129, False), (2, 64, 5003, False), (1, 70, 8191, False),
                                         (2, 17, 32768, False), (3, 17, 32769, False), (200, 3, 33333, True)])
def test_rule(gpu, T, M, V, chain, dtype, sampled):
    check(gpu, *make(T, M, V, dtype, sampled, seed=T * 100 + M, chain=chain))


@pytest.mark.parametrize("gap", [0.0, 0.3, 3.0])
def test_many_trees_of_siblings(gpu, gap):
    """Many walks, so that second and third siblings are tested after sweeps (gap 0: draft and target agree)."""
    check(gpu, *make(64, 24, 700, torch.float32, True, seed=5, gap=gap, peak=1.0))
    check(gpu, *make(64, 24, 700, torch.float32, False, seed=6, gap=gap, peak=1.0))


def test_large_vocabulary(gpu):
    check(gpu, *make(2, 5, 128256, torch.float32, True, seed=9, chain=True))
    check(gpu, *make(2, 5, 128256, torch.bfloat16, False, seed=10))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,gap", [(1, 0.8), (4, 3.0)])
def test_sampled_trees_over_a_large_vocabulary(gpu, T, gap, dtype):
    """Siblings' masses where a row is shared out over workgroups, each of which sums the whole row for them."""
    p, q, draft, parent, u = make(T, 13, 128256, dtype, True, seed=T, gap=gap, peak=1.0)
    check(gpu, p, q, draft, parent, u)
    # Every number the largest: all siblings of every node on the way are tested that the rule can reject.
    check(gpu, p, q, draft, parent, torch.full_like(u, 0.99999994))


def test_1024_nodes_and_unordered_trees(gpu):
    """A child may have a lower index than its parent; malformed parents belong to nobody."""
    p, q, draft, parent, u = make(2, 1024, 40, torch.float32, True, seed=3, peak=1.0)
    check(gpu, p, q, draft, parent, u)
    p, q, draft, parent, u = make(4, 12, 30, torch.float32, True, seed=4)
    perm = torch.tensor([0, 7, 3, 11, 1, 9, 5, 2, 10, 4, 8, 6])  # new index of node i
    for t in range(4):
        full = [-1] + [int(x) + 1 for x in parent[t]]
        new_par, nd = [0] * 12, torch.zeros(12, dtype=torch.int64)
        for i in range(12):
            nd[perm[i]] = draft[t, i]
            if i:
                new_par[perm[i]] = int(perm[full[i]])
        draft[t] = nd
        parent[t] = torch.tensor([x - 1 for x in new_par[1:]])
    check(gpu, p, q, draft, parent, u)
    parent[:, 3] = 55   # no such node
    parent[:, 5] = -7
    parent[:, 8] = 8    # its own place: the root
    check(gpu, p, q, draft, parent, u)


@pytest.mark.parametrize("V", [4500, 50001])
def test_strides_and_unaligned_rows(gpu, V):
    """Rows of an odd stride at an odd offset, reversed-order views of the small inputs."""
    p, q, draft, parent, u = make(3, 9, V, torch.bfloat16, True, seed=21)
    big = torch.zeros(3, 10, V + 7, dtype=torch.bfloat16, device=gpu)
    pv = big[:, 1:, 3:V + 3]
    pv.copy_(p)
    qv = torch.zeros(9, 3, V + 1, dtype=torch.bfloat16, device=gpu)[:, :, 1:].transpose(0, 1)
    qv.copy_(q)
    want = check(gpu, p, q, draft, parent, u)
    got = speculative_accept(pv, draft.to(gpu).t().contiguous().t(), parent.to(gpu), u.to(gpu).t().contiguous().t(), qv)
    for k in want:
        assert torch.equal(want[k], got[k])


@pytest.mark.parametrize("V", [50, 40007])
def test_edges(gpu, V):
    M = 4
    p = torch.full((6, M, V), 1.0 / V)
    q = p.clone()
    draft = torch.tensor([[0, 3, 4, 5]] * 6)
    parent = torch.tensor([[-1, -1, -1]] * 6)  # three children of the root
    u = torch.full((6, M), 0.5)
    # 0: the draft's row is the target's: every test passes.  1: the target has nothing where the draft has.
    p[1, 0, :10] = 0.0
    # 2: NaN, infinities and negative entries count as nothing.
    p[2, 0, 0], p[2, 0, 1], p[2, 0, 2], p[2, 0, 3] = float("nan"), float("inf"), -1.0, float("-inf")
    # 3: an all-zero target row draws token 0.  4: tokens outside the vocabulary.
    p[3, 0] = 0.0
    draft[4, 1:] = torch.tensor([-1, V, 1 << 40])
    # 5: numbers outside [0, 1).
    u[5] = torch.tensor([1.0, float("nan"), -3.0, 7.0])
    check(gpu, p, q, draft, parent, u)
    check(gpu, p, None, draft, parent, u)
    # Repeated given tokens are rejected once rejected.
    draft[:, 1:] = 7
    u[:, 1:] = 0.9
    check(gpu, p, None, draft, parent, u)
    # All mass rejected: the row itself is drawn from.
    p[:] = 0.0
    p[:, 0, 7] = 1.0
    q[:] = 0.0
    q[:, 0, 7] = 4.0
    check(gpu, p, q, draft, parent, torch.full((6, M), 0.99))


@pytest.mark.parametrize("V", [3 * 4096 + 5, 128 * 512 + 77])
def test_draw_at_both_ends(gpu, V):
    """The next token for the smallest and largest numbers, weights in the first and last sub-block only."""
    p = torch.zeros(4, 1, V)
    p[:2, 0, 2], p[:2, 0, V - 1] = 0.25, 0.75
    p[2:, 0, 4095], p[2:, 0, 4096] = 0.5, 0.5
    u = torch.tensor([[0.0], [0.99999994], [0.49999997], [0.5]])
    r = check(gpu, p, None, torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 0, dtype=torch.int64), u)
    assert r["info"][:, 2].tolist() == [2, V - 1, 4095, 4096]


def test_distribution_of_the_first_token(gpu):
    """The first token after the root follows the target (chi-square over 16 tokens, 40000 given numbers)."""
    n, V = 40000, 16
    g = torch.Generator().manual_seed(77)
    p = torch.softmax(torch.randn(V, generator=g), 0)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    kids = torch.multinomial(q, 2 * n, replacement=True, generator=g).view(n, 2)
    draft = torch.cat([torch.zeros(n, 1, dtype=torch.int64), kids], 1)
    parent = torch.full((n, 2), -1)
    rows = lambda x: x.to(gpu).view(1, 1, V).expand(n, 3, V)  # noqa: E731
    r = speculative_accept(rows(p), draft.to(gpu), parent.to(gpu), torch.rand((n, 3), generator=g).to(gpu), rows(q))
    info = r["info"].cpu()
    first = torch.where(info[:, 1] > 0, r["tokens"][:, 1].cpu(), info[:, 2])
    count = torch.bincount(first, minlength=V).double()
    exp = p.double() * n
    # 15 degrees of freedom: mean 15, deviation 5.5; 60 lies beyond 1e-6.
    assert float(((count - exp) ** 2 / exp).sum()) < 60.0


def test_streams_graph_and_commit(gpu):
    """On a side stream and captured (replayed with other inputs), and the commit of its path."""
    a = make(3, 16, 3000, torch.float32, True, seed=31)
    b = make(3, 16, 3000, torch.float32, True, seed=32)
    bufs = [x.to(gpu) for x in a]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = speculative_accept(bufs[0], bufs[2], bufs[3], bufs[4], bufs[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = speculative_accept(bufs[0], bufs[2], bufs[3], bufs[4], bufs[1])
    for x in (a, b, a):
        for dst, src in zip(bufs, x):
            dst.copy_(src)
        graph.replay()
        ref = check(gpu, x[0], x[1], x[2], x[3], x[4])
        for k in out:
            assert torch.equal(out[k], ref[k]), k
    assert torch.equal(want["info"], out["info"])
    cache = torch.randn(2, 4, 100, 16, device=gpu)
    before = cache.clone()
    kv_commit(cache, 50, out["path"], out["info"], tree=1)
    path = [i for i in out["path"][1].tolist() if i >= 0]
    assert torch.equal(cache[:, :, 50:50 + len(path)], before[:, :, [50 + i for i in path]])
