"""A speculative decoding loop over a paged cache: extend, append, windowed tree attention, verification,
commit, free behind the window, fork and compact, every step against its restatement on the host."""

import numpy as np
import pytest
import torch

from diffspec_mi355x import workloads as wl
from diffspec_mi355x.core.kv_cache import compact_pages, extend_pages, fork_pages, free_pages
from diffspec_mi355x.draft.tree_verification import kv_commit, speculative_accept
from diffspec_mi355x.runtime.cache_state import append_tree_kv
from diffspec_mi355x.runtime.window_attention import window_attn_with_kvcache
from oracle import pages as opages
from oracle import window as owindow
from test_gpu_spec import check as check_accept
from test_gpu_window import bounds

pytestmark = pytest.mark.gpu

B, M, H, HK, D, PS, V = 4, 12, 8, 2, 64, 16, 96
P, N_LOG = 40, 20
WINDOW, SINKS = 40, 20


class Loop:
    """The device's tensors and lists that restate them (rows[b]: K and V of every token)."""

    def __init__(self, gpu, dtype):
        self.gpu, self.dtype = gpu, dtype
        self.g = torch.Generator().manual_seed(11)
        # (Pages that nobody wrote hold NaN, as freed memory may.)
        self.kv = torch.full((1, 2, P, HK, PS, D), float("nan"), dtype=dtype, device=gpu)
        self.dtable = torch.full((B, N_LOG), -1, dtype=torch.int32, device=gpu)
        self.dref = torch.zeros(P, dtype=torch.int32, device=gpu)
        self.dlens = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.table, self.ref, self.lens = [[-1] * N_LOG for _ in range(B)], [0] * P, [0] * B
        self.rows = [np.zeros((2, 0, HK, D)) for _ in range(B)]
        pars = [wl.make_tree(M, max_depth=M, max_outdeg=3, seed=40 + b)[0] for b in range(B)]
        self.par = torch.tensor(pars, dtype=torch.int32, device=gpu)
        self.pars = pars
        self.ref_par = torch.tensor([wl.parent_to_reference(p) for p in pars], dtype=torch.int64, device=gpu)

    def rand(self, *s):
        return torch.randn(s, generator=self.g).to(self.dtype).to(self.gpu)

    def inputs(self):
        return dict(k=self.rand(B, M, HK, D), v=self.rand(B, M, HK, D), q=self.rand(B, M, H, D),
                    draft_probs=torch.softmax(torch.randn((B, M, V), generator=self.g), -1).to(self.gpu),
                    draft=torch.randint(0, V, (B, M), generator=self.g).to(self.gpu),
                    uniform=torch.rand((B, M), generator=self.g).to(self.gpu))

    def device_step(self, x, start, new):
        """One step of the sequences with start[b] >= 0 tokens (host numbers; others stand still)."""
        info = extend_pages(self.dtable, self.dref, self.dlens, new, PS)
        for b in range(B):
            if start[b] >= 0:
                append_tree_kv(x["k"][b], x["v"][b], self.kv[0, 0], self.kv[0, 1], start[b], page_table=self.dtable[b])
        out, lse = window_attn_with_kvcache(x["q"], self.kv[0, 0], self.kv[0, 1], WINDOW, SINKS, self.dlens, self.dtable,
                                            self.par, return_softmax_lse=True)
        probs = torch.softmax(out.reshape(B, M, H * D)[..., :V].float() * 4.0, -1)
        r = speculative_accept(probs, x["draft"], self.ref_par, x["uniform"], x["draft_probs"])
        for b in range(B):
            if start[b] >= 0:
                kv_commit(self.kv, start[b], r["path"], r["info"], self.dtable[b], tree=b)
        self.dlens.copy_(torch.where(new > 0, self.dlens - M + r["info"][:, 3].int(), self.dlens))
        return dict(info=info, out=out, lse=lse, probs=probs, **{k: r[k] for k in ("path", "tokens")}, accepted=r["info"])

    def prompt(self, b, n):
        """n first tokens of sequence b: their keys and values, and causal attention."""
        new = [n if i == b else 0 for i in range(B)]
        got = extend_pages(self.dtable, self.dref, self.dlens, torch.tensor(new, dtype=torch.int32, device=self.gpu), PS)
        assert tuple(got.tolist()) == opages.extend(self.table, self.ref, self.lens, new, PS)
        k, v, q = self.rand(n, HK, D), self.rand(n, HK, D), self.rand(1, n, H, D)
        append_tree_kv(k, v, self.kv[0, 0], self.kv[0, 1], 0, page_table=self.dtable[b])
        out, lse = window_attn_with_kvcache(q, self.kv[0, 0], self.kv[0, 1], WINDOW, SINKS, self.dlens[b:b + 1],
                                            self.dtable[b:b + 1], return_softmax_lse=True)
        self.rows[b] = rows = torch.stack([k, v]).double().cpu().numpy()
        w, wl_, absum, reach = owindow.attend(q[0].double().cpu().numpy(), rows[0], rows[1], owindow.visible(n, n, WINDOW, SINKS))
        tol, ltol = bounds(self.dtype, self.dtype, w, wl_, absum, reach, min(n, WINDOW + SINKS), D, np.abs(rows[1]).max())
        assert (np.abs(out[0].double().cpu().numpy() - w) <= tol).all()
        assert (np.abs(lse[0].double().cpu().numpy() - wl_) <= ltol).all()
        self.same()

    def step(self, live):
        x = self.inputs()
        start = [self.lens[b] if b in live else -1 for b in range(B)]
        new = [self.lens[b] + M if b in live else 0 for b in range(B)]
        got = self.device_step(x, start, torch.tensor(new, dtype=torch.int64, device=self.gpu))
        want = opages.extend(self.table, self.ref, self.lens, new, PS)
        assert tuple(got["info"].tolist()) == want and want[1:] == (0, 0)
        check_accept(self.gpu, got["probs"].cpu(), x["draft_probs"].cpu(), x["draft"].cpu(), self.ref_par.cpu(), x["uniform"].cpu())
        for b in range(B):
            kv = torch.stack([x["k"][b], x["v"][b]]).double().cpu().numpy()
            out, lse = got["out"][b].double().cpu().numpy(), got["lse"][b].double().cpu().numpy()
            if b in live:
                rows = np.concatenate([self.rows[b], kv], axis=1)
                keys = owindow.visible(M, rows.shape[1], WINDOW, SINKS, self.pars[b])
                w, wl_, absum, reach = owindow.attend(x["q"][b].double().cpu().numpy(), rows[0], rows[1], keys)
                seen = np.unique(np.concatenate(keys))
                tol, ltol = bounds(self.dtype, self.dtype, w, wl_, absum, reach, max(k.size for k in keys), D,
                                   np.abs(rows[1][seen]).max())
                assert (np.abs(out - w) <= tol).all() and (np.abs(lse - wl_) <= ltol).all(), b
                path = [i for i in got["path"][b].tolist() if i >= 0]
                self.rows[b] = np.concatenate([self.rows[b], kv[:, path]], axis=1)
                self.lens[b] = self.rows[b].shape[1]
            elif self.lens[b] == 0:
                assert (out == 0).all() and (lse == -np.inf).all()
        self.same()

    def same(self):
        assert self.dlens.tolist() == self.lens and self.dtable.tolist() == self.table and self.dref.tolist() == self.ref
        pool = self.kv[0].double().cpu().numpy()
        for b in range(B):
            for n in range(self.lens[b]):
                page = self.table[b][n // PS]
                if page >= 0:
                    assert np.array_equal(pool[:, page, :, n % PS], self.rows[b][:, n]), (b, n)

    def free(self, seqs, window=None, sinks=0):
        free_pages(self.dtable, self.dref, self.dlens, torch.tensor(seqs, device=self.gpu), PS, window, sinks)
        opages.free(self.table, self.ref, self.lens, seqs, PS, window, sinks)
        if window is None:
            for b in seqs:
                self.rows[b] = self.rows[b][:, :0]
        self.same()

    def fork(self, parents, children):
        got = fork_pages(self.kv, self.dtable, self.dref, self.dlens, torch.tensor(parents, device=self.gpu),
                         torch.tensor(children, device=self.gpu))
        assert tuple(got.tolist()) == opages.fork(np.zeros((1, 2, P, 1, 1, 1)), self.table, self.ref, self.lens, parents, children, PS)
        for a, c in zip(parents, children):
            self.rows[c] = self.rows[a].copy()
        self.same()

    def compact(self):
        got = compact_pages(self.kv, self.dtable, self.dref)
        assert tuple(got.tolist()) == opages.compact(np.zeros((1, 2, P, 1, 1, 1)), self.table, self.ref)
        self.same()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_loop(gpu, dtype):
    p = Loop(gpu, dtype)
    p.prompt(0, 70)
    p.prompt(1, 33)
    for _ in range(20):
        p.step([0, 1])
        p.free([0, 1], WINDOW, SINKS)
    assert -1 in p.table[0][:p.lens[0] // PS] or -1 in p.table[1][:p.lens[1] // PS]   # something left the window
    p.fork([0, 0], [2, 3])
    for _ in range(4):
        p.step([0, 1, 2, 3])
        p.free([0, 1, 2, 3], WINDOW, SINKS)
    p.free([1])
    p.compact()
    for _ in range(3):
        p.step([0, 2, 3])
    p.free([0, 2, 3])
    assert sum(p.ref) == 0


def test_loop_captured(gpu):
    """One step as a graph: every replay, from the same state with other inputs, as the eager step."""
    p = Loop(gpu, torch.bfloat16)
    for _ in range(4):
        p.step([0, 1, 3])
    start = [p.lens[b] if b != 2 else -1 for b in range(B)]
    new = torch.tensor([n + M if n >= 0 else 0 for n in start], dtype=torch.int64, device=gpu)
    state = [t.clone() for t in (p.kv, p.dtable, p.dref, p.dlens)]

    def restore():
        for dst, src in zip((p.kv, p.dtable, p.dref, p.dlens), state):
            dst.copy_(src)

    xs = [p.inputs() for _ in range(3)]
    want = []
    for x in xs:
        restore()
        got = p.device_step(x, start, new)
        want.append({k: v.clone() for k, v in {**got, "kv": p.kv, "table": p.dtable, "ref": p.dref, "lens": p.dlens}.items()})
    buf = {k: v.clone() for k, v in xs[0].items()}
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.device_step(buf, start, new)
    for i in (1, 2, 0, 1):
        restore()
        for k in buf:
            buf[k].copy_(xs[i][k])
        graph.replay()
        torch.cuda.synchronize()
        for k, v in {**got, "kv": p.kv, "table": p.dtable, "ref": p.dref, "lens": p.dlens}.items():
            # (Bytes: pages that nobody wrote hold NaN.)
            assert torch.equal(v.contiguous().view(torch.uint8), want[i][k].contiguous().view(torch.uint8)), (i, k)


def test_two_streams_at_once(gpu):
    """Calls that share keys and rows out over workgroups, on two streams at once, as one after the other."""
    g = torch.Generator().manual_seed(2)
    q = [torch.randn((2, m, 8, 64), generator=g).to(torch.bfloat16).to(gpu) for m in (1, 40)]
    k, v = (torch.randn((2, 4000, 2, 64), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    probs = [torch.softmax(torch.randn((3, 6, 60000), generator=g), -1).to(gpu) for _ in range(2)]
    draft = torch.randint(0, 60000, (3, 6), generator=g).to(gpu)
    parent = torch.arange(-1, 4, device=gpu).expand(3, -1)
    uniform = torch.rand((3, 6), generator=g).to(gpu)

    def run(i):
        out, lse = window_attn_with_kvcache(q[i], k, v, 3000, 4, return_softmax_lse=True)
        return out, lse, speculative_accept(probs[i], draft, parent, uniform, probs[1 - i])["info"]

    want = [run(0), run(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("M", [5, 60])
def test_forms_of_the_tree(gpu, M):
    """One tree for all sequences or one each, int32 or int64, at any stride: the same result."""
    g = torch.Generator().manual_seed(3)
    q = torch.randn((3, M, 8, 64), generator=g).to(torch.bfloat16).to(gpu)
    k, v = (torch.randn((3, 300, 2, 64), generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    lens = torch.tensor([300, M, M + 31], device=gpu)
    par = torch.tensor(wl.make_tree(M, max_depth=M, max_outdeg=3, seed=5)[0], device=gpu)
    f = lambda p: window_attn_with_kvcache(q, k, v, 100, 7, lens, parent=p, return_softmax_lse=True)  # noqa: E731
    want = f(par)
    wide = torch.full((3, 2 * M + 1), 99, dtype=torch.int64, device=gpu)
    wide[:, 1::2] = par
    for p in (par.int(), par[None], par.int().expand(3, -1), par.repeat(3, 1), wide[:, 1::2]):
        got = f(p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = window_attn_with_kvcache(q[:1], k[:1], v[:1], 100, 7, 300, parent=par)
    assert torch.equal(one[0], want[0][0])
