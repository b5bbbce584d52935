"""Cases of the operators of a serving loop whose cache holds one latent vector per token.

Such a cache keeps, of every token, a compressed vector that all heads share
(keys and values alike) and a small rotated key part.  A step maps the new
tokens of its requests to places in the page pool, writes their latent rows,
and attends: single tokens, drafted trees and short chunks over the cache
itself (absorbed form: the queries are already in the latent space), long
prompts over keys and values expanded per head.  Each kind of call is one
``kind`` below.

    kind      entry points
    slots     token_slots (block tables and slot maps from request lengths)
    append    append_latent_kv (norm, rotation and scatter of new rows, rotation of the queries)
    absorbed  latent_attn_with_kvcache (single tokens, chunks, trees; paged and dense caches)
    expanded  latent_attn_expanded (prompts and chunks of them, whole and causal)

Where ``own`` is false, ``run`` computes the operators with elementary torch
operations; where it is true, it calls the package.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda"
_EPS = 1e-6
# Bounds of a drawn case: what the largest listed cases do (operations of fp32
# cases count 16 times, the ratio of the 16-bit to the fp32 matrix rate).
_MAX_BYTES = 6.2e8
_MAX_FLOPS = 3.4e11


# ----------------------------------------------------------------------------
# The cases
# ----------------------------------------------------------------------------

def listed():
    return [
        # A decoding step: one new token of each active request, some sequences idle.
        dict(name="slots_decode", kind="slots", B=64, n=48, cap=64, lo=1, hi=30000, new=1, page=16),
        # Admission of many prompts at once, room left behind the last token.
        dict(name="slots_prompts", kind="slots", B=700, n=512, cap=300000, lo=1, hi=8000, new=1000, page=64),
        # The new rows of a decoding step of 48 requests, padded to 64: latency.
        dict(name="append_step", kind="append", T=64, valid=48, dc=512, dr=64, H=16, page=16, P=4096, inter=True, norm=True,
             dtype="bf16"),
        # The rows of a batch of prompts.
        dict(name="append_prompts", kind="append", T=65536, valid=65001, dc=512, dr=64, H=16, page=64, P=1100, inter=False,
             norm=True, dtype="bf16"),
        # One request decoding token by token, all heads on one GPU: latency.
        dict(name="lat_decode_one", kind="absorbed", B=1, M=1, lo=2900, hi=2900, H=128, dc=512, dr=64, page=64, tree=False,
             dtype="bf16"),
        # A full batch of long requests, heads shared out over GPUs: cache traffic.
        dict(name="lat_decode_batch", kind="absorbed", B=64, M=1, lo=1, hi=16384, H=16, dc=512, dr=64, page=64, tree=False,
             dtype="bf16"),
        # All heads on one GPU: traffic and matrix work are near each other.
        dict(name="lat_decode_heads", kind="absorbed", B=32, M=1, lo=1000, hi=8192, H=128, dc=512, dr=64, page=16, tree=False,
             dtype="f16"),
        # Eight requests verify a 64-node tree each: matrix work.
        dict(name="lat_tree", kind="absorbed", B=8, M=64, lo=2000, hi=6000, H=32, dc=512, dr=64, page=32, tree=True,
             dtype="bf16"),
        # Short odd chunks in fp32, a narrower latent, dense cache.
        dict(name="lat_chunk_f32", kind="absorbed", B=3, M=5, lo=4, hi=3001, H=20, dc=256, dr=32, page=0, tree=False,
             dtype="f32"),
        # A whole prompt: the largest matrix work.
        dict(name="exp_prompt", kind="expanded", B=1, M=8192, lo=8192, hi=8192, H=16, dn=128, dr=64, causal=True, dtype="bf16"),
        # Odd chunks of two longer prompts.
        dict(name="exp_chunk", kind="expanded", B=2, M=1001, lo=5000, hi=12007, H=8, dn=128, dr=64, causal=True, dtype="f16"),
        # A short batch in fp32, some prompts shorter than the chunk.
        dict(name="exp_short_f32", kind="expanded", B=4, M=77, lo=30, hi=500, H=5, dn=64, dr=32, causal=True, dtype="f32"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["slots", "append", "absorbed", "absorbed", "absorbed", "expanded", "expanded"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "slots":
        B = _logint(rng, 1, 4000)
        n, page = rng.randint(max(1, B // 2), B), rng.choice([8, 16, 32, 64, 128])
        hi, new = _logint(rng, 64, 40000), rng.choice([1, 1, _logint(rng, 2, 4000)])
        return dict(kind=kind, B=B, n=n, cap=_logint(rng, 16, 400000), lo=rng.choice([1, hi // 2, hi]), hi=hi, new=new, page=page)
    if kind == "append":
        T, page = _logint(rng, 1, 65536), rng.choice([8, 16, 32, 64, 128])
        valid = rng.randint((T + 1) // 2, T)
        return dict(kind=kind, T=T, valid=valid, dc=rng.choice([256, 512]), dr=rng.choice([32, 64]),
                    H=rng.choice([0, 1, 5, 16, 32, 128]), page=page, P=-(-valid // page) + rng.randint(0, 64),
                    inter=rng.random() < 0.5, norm=rng.random() < 0.7, dtype=dt)
    if kind == "absorbed":
        form = rng.choice(["decode", "decode", "chunk", "tree"])
        M = {"decode": 1, "chunk": _logint(rng, 2, 1024), "tree": _logint(rng, 2, 256)}[form]
        hi = max(_logint(rng, 16, 40000), M + 1)
        lo = rng.choice([hi, max(1, hi // 2), 1])
        return dict(kind=kind, B=_logint(rng, 1, 96), M=M, lo=max(lo, M) if form == "tree" else lo, hi=hi,
                    H=rng.choice([1, 3, 8, 16, 16, 20, 32, 64, 128]), dc=rng.choice([256, 512, 512]), dr=rng.choice([32, 64, 64]),
                    page=rng.choice([0, 16, 32, 64, 128]), tree=form == "tree", dtype=dt)
    M = _logint(rng, 1, 8192)
    hi = max(_logint(rng, 16, 20000), M)
    return dict(kind=kind, B=_logint(rng, 1, 8), M=M, lo=rng.choice([hi, max(1, hi // 2), 1]), hi=hi,
                H=rng.choice([1, 3, 8, 16, 32, 128]), dn=rng.choice([64, 128, 128]), dr=rng.choice([32, 64, 64]),
                causal=rng.random() < 0.8, dtype=dt)


def _state_bytes(c):
    """Of the caches and tables that a state holds."""
    if c["kind"] == "slots":
        return 4 * c["B"] * _width(c)
    es = _BYTES[c["dtype"]]
    if c["kind"] == "append":
        return (c["P"] * c["page"] + c["T"]) * (c["dc"] + c["dr"]) * es
    if c["kind"] == "absorbed":
        rows = c["B"] * c["hi"] if c["page"] == 0 else sum(_lens(c))
        return rows * (c["dc"] + c["dr"]) * es
    return c["B"] * c["hi"] * (2 * c["H"] * c["dn"] + c["dr"]) * es


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if (w["bytes"] <= _MAX_BYTES and w["flops"] * (16 if c.get("dtype") == "f32" else 1) <= _MAX_FLOPS
                and _state_bytes(c) <= 1.2e9):
            return c


# ----------------------------------------------------------------------------
# Shapes that follow from the case alone
# ----------------------------------------------------------------------------

def _lens(c, n=None):
    """Lengths of the sequences, the new tokens included."""
    r = random.Random(c["lo"] * 1000003 + c["hi"] * 31 + c["B"])
    return [c["hi"]] + [r.randint(min(c["lo"], c["hi"]), c["hi"]) for _ in range((n or c["B"]) - 1)]


def _news(c):
    """New tokens of the requests (never more than the shortest sequence may hold)."""
    r = random.Random(c["new"] * 7919 + c["n"])
    return [r.randint(1, c["new"]) for _ in range(c["n"])]


def _width(c):
    return -(-c["hi"] // c["page"]) + 2


def _pairs(c):
    """Query rows times the keys that they see."""
    total = 0
    for n in _lens(c):
        n0 = n - c["M"]
        if c["kind"] == "expanded" and not c["causal"]:
            total += c["M"] * n
        elif c.get("tree"):
            total += c["M"] * (n0 + 1)                # of the tree at least itself
        else:
            p = np.arange(max(n0, 0), n, dtype=np.int64)
            total += int((p + 1).sum())
    return total * c["H"]


def work(case):
    c = case
    if c["kind"] == "slots":
        pages = sum(-(-n // c["page"]) for n in _lens(c)[:c["n"]])
        tok = min(c["cap"], sum(_news(c)))
        return {"bytes": 4 * (pages + c["n"] * _width(c)) + 16 * c["cap"] + 8 * 4 * c["n"], "flops": tok}
    es = _BYTES[c["dtype"]]
    if c["kind"] == "append":
        row = (c["dc"] + c["dr"]) * es
        return {"bytes": c["valid"] * (2 * row + 2 * c["dr"] * 4) + c["T"] * (2 * c["H"] * c["dr"] * es + 12),
                "flops": c["valid"] * (4 * c["dc"] + 3 * c["dr"]) + 3 * c["T"] * c["H"] * c["dr"]}
    q = c["B"] * c["M"] * c["H"]
    if c["kind"] == "absorbed":
        d = c["dc"] + c["dr"]
        return {"bytes": sum(_lens(c)) * d * es + q * ((d + c["dc"]) * es + 4), "flops": 2 * (d + c["dc"]) * _pairs(c)}
    d = c["dn"] + c["dr"]
    return {"bytes": sum(_lens(c)) * (2 * c["H"] * c["dn"] + c["dr"]) * es + q * ((d + c["dn"]) * es + 4),
            "flops": 2 * (d + c["dn"]) * _pairs(c)}


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(g, shape, dtype, scale=1.0):
    """N(0, scale) in pieces, so that no fp32 copy of a large pool is made."""
    out = torch.empty(shape, dtype=dtype, device=_DEV)
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=_DEV) * scale
    return out


def _tree(rng, M):
    """Per-node parents (-1: root): depths of about eight, up to four children."""
    parent, depth, kids = [-1], [0], [0]
    for i in range(1, M):
        cand = [j for j in range(max(0, i - 12), i) if kids[j] < 4 and depth[j] < 8] or [i - 1]
        p = rng.choice(cand)
        parent.append(p)
        depth.append(depth[p] + 1)
        kids[p] += 1
        kids.append(0)
    return parent


def _page_table(rng, lens, page, width):
    """Pages for every token, shuffled over a pool with a few to spare."""
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    pages, at = rng.permutation(P), 0
    table = np.full((len(lens), width), -1, dtype=np.int32)
    for b, k in enumerate(need):
        table[b, :k] = pages[at:at + k]
        at += k
    return table, P


def _prepare_slots(c, seed):
    rng = np.random.default_rng(seed)
    news, seqs = _news(c), rng.permutation(c["B"])[:c["n"]]
    lens = np.array(_lens(c))
    lens[seqs] = np.maximum(lens[:c["n"]], news)           # the requests' lengths stand first in _lens
    lens = np.minimum(lens, c["hi"])
    news = np.minimum(news, lens[seqs])
    table, _ = _page_table(rng, lens, c["page"], _width(c))
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(_DEV)  # noqa: E731
    return {"case": c, "table": i32(table), "lens": i32(lens), "seqs": i32(seqs), "news": i32(news)}


def _prepare_append(c, seed):
    g, rng, dt = _gen(seed), np.random.default_rng(seed), _DTYPE[c["dtype"]]
    T, dc, dr = c["T"], c["dc"], c["dr"]
    # The projection's output: latent and key part of a token side by side.
    kv = _randn(g, (T, dc + dr), dt, 1.3)
    slots = np.full(T, -1, dtype=np.int64)
    slots[:c["valid"]] = rng.permutation(c["P"] * c["page"])[:c["valid"]]
    n_pos = 8192
    ang = torch.arange(n_pos, device=_DEV, dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(0, dr, 2, device=_DEV, dtype=torch.float64) / dr))
    ang = ang.repeat_interleave(2, -1) if c["inter"] else torch.cat([ang, ang], -1)
    q = _randn(g, (T, c["H"], 128 + dr), dt) if c["H"] else None
    return {"case": c, "kv": kv, "cache": torch.zeros((c["P"], c["page"], dc + dr), dtype=dt, device=_DEV),
            "slots": torch.from_numpy(slots).to(_DEV), "cos": ang.cos().float(), "sin": ang.sin().float(),
            "positions": torch.from_numpy(rng.integers(0, n_pos, T).astype(np.int32)).to(_DEV),
            "weight": (1 + 0.2 * torch.randn(dc, generator=g, device=_DEV)).to(dt) if c["norm"] else None, "q": q}


def _prepare_absorbed(c, seed):
    g, rng, dt = _gen(seed), np.random.default_rng(seed), _DTYPE[c["dtype"]]
    B, M, d = c["B"], c["M"], c["dc"] + c["dr"]
    lens = _lens(c)
    st = {"case": c, "lens": lens, "q": _randn(g, (B, M, c["H"], d), dt), "table": None, "parent": None,
          "scale": 1.5 / math.sqrt(d), "seqlens": torch.tensor(lens, dtype=torch.int32, device=_DEV)}
    if c["page"]:
        table, P = _page_table(rng, lens, c["page"], -(-c["hi"] // c["page"]))
        st["table"] = torch.from_numpy(table).to(_DEV)
        st["kv"] = _randn(g, (P, c["page"], d), dt)
    else:
        st["kv"] = _randn(g, (B, c["hi"], d), dt)
    if c["tree"]:
        r = random.Random(int(rng.integers(1 << 40)))
        st["parent"] = torch.tensor([_tree(r, M) for _ in range(B)], dtype=torch.int32, device=_DEV)
    return st


def _prepare_expanded(c, seed):
    g, dt = _gen(seed), _DTYPE[c["dtype"]]
    B, H, dn, dr = c["B"], c["H"], c["dn"], c["dr"]
    lens = _lens(c)
    # The expansion's output: a head's key and value part side by side.
    kv = _randn(g, (B, c["hi"], H, 2 * dn), dt)
    return {"case": c, "lens": lens, "q": _randn(g, (B, c["M"], H, dn + dr), dt, 1.5), "k": kv[..., :dn], "v": kv[..., dn:],
            "k_pe": _randn(g, (B, c["hi"], dr), dt), "seqlens": torch.tensor(lens, dtype=torch.int32, device=_DEV)}


_PREPARE = dict(slots=_prepare_slots, append=_prepare_append, absorbed=_prepare_absorbed, expanded=_prepare_expanded)


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, seed)


# ----------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------

def _plain_slots(st):
    c, table = st["case"], st["table"].long()
    ps, cap = c["page"], c["cap"]
    seqs = st["seqs"].long()
    lens = st["lens"].long()[seqs]
    ends = st["news"].long().cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    tok = torch.arange(cap, device=_DEV)
    req = (tok.view(-1, 1) >= ends.view(1, -1)).sum(1) if cap * c["n"] <= 1 << 24 else torch.bucketize(tok, ends, right=True)
    real = tok < ends[-1]
    r = req.clamp(max=c["n"] - 1)
    pos = lens[r] - (ends[r] - tok)
    pos = torch.where(real, pos, torch.zeros_like(pos))
    page = table[seqs[r], pos // ps]
    none = torch.full_like(pos, -1)
    j = torch.arange(table.shape[1], device=_DEV)
    block = torch.where(j * ps < lens.view(-1, 1), table[seqs], torch.full_like(table[seqs], -1))
    return {"slots": torch.where(real & (page >= 0), page * ps + pos % ps, none), "positions": torch.where(real, pos, none).int(),
            "requests": torch.where(real, r, none).int(), "cu_seqlens": cu.int(), "block_table": block.int(), "lens": lens.int()}


def _turned(x, inter):
    """Each element's partner in its rotation, signed."""
    if inter:
        return torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)
    h = x.shape[-1] // 2
    return torch.cat([-x[..., h:], x[..., :h]], -1)


def _plain_append(st):
    c, dt = st["case"], st["kv"].dtype
    dc = c["dc"]
    x = st["kv"][:, :dc].float()
    if c["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * st["weight"].float()
    pos = st["positions"].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    pe = st["kv"][:, dc:].float()
    pe = pe * cos + _turned(pe, c["inter"]) * sin
    row = torch.cat([x, pe], -1).to(dt)
    cache = st["cache"].view(-1, dc + c["dr"])
    keep = st["slots"] >= 0
    cache[st["slots"][keep]] = row[keep]
    out = {"cache": st["cache"]}
    if st["q"] is not None:
        qp = st["q"][..., 128:].float()
        out["q_pe"] = (qp * cos.unsqueeze(1) + _turned(qp, c["inter"]) * sin.unsqueeze(1)).to(dt)
    return out


def _softmax_rows(s, keep):
    """exp(s - max) of the kept entries, their sum and the maximum; rows without any: zeros, 0 and -inf."""
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    mx = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(mx > -math.inf, mx, torch.zeros_like(mx)))
    return e, e.sum(-1, keepdim=True), mx


def _plain_absorbed(st):
    c, q = st["case"], st["q"]
    B, M, H, dc, d = c["B"], c["M"], c["H"], c["dc"], c["dc"] + c["dr"]
    out = torch.zeros((B, M, H, dc), dtype=q.dtype, device=_DEV)
    lse = torch.full((B, H, M), -math.inf, device=_DEV)
    for b, n in enumerate(st["lens"]):
        n0 = n - M
        idx = torch.arange(n, device=_DEV)
        if st["table"] is None:
            kv = st["kv"][b, :n].float()
        else:
            kv = st["kv"][st["table"][b].long()[idx // c["page"]], idx % c["page"]].float()
        if c["tree"]:
            par = st["parent"][b].long()
            up = torch.eye(M, dtype=torch.bool, device=_DEV)      # ancestor or self
            for m in range(1, M):                                  # parents precede their children
                up[m] |= up.index_select(0, par[m:m + 1])[0]
        step = max(1, 4096 // H)                                   # positions at a time
        for m0 in range(0, M, step):
            m1 = min(M, m0 + step)
            if c["tree"]:
                keep = torch.cat([torch.ones((m1 - m0, n0), dtype=torch.bool, device=_DEV), up[m0:m1]], 1)
            else:
                keep = idx <= n0 + torch.arange(m0, m1, device=_DEV).view(-1, 1)
            rows = q[b, m0:m1].float().view((m1 - m0) * H, d)
            s = torch.matmul(rows, kv.T).view(m1 - m0, H, n) * st["scale"]
            e, z, mx = _softmax_rows(s, keep.unsqueeze(1))
            o = torch.matmul(e.view(-1, n), kv[:, :dc]).view(m1 - m0, H, dc) / torch.where(z > 0, z, torch.ones_like(z))
            out[b, m0:m1] = o.to(q.dtype)
            lse[b, :, m0:m1] = (mx + torch.log(z))[..., 0].T
    return {"out": out, "lse": lse}


def _plain_expanded(st):
    c, q = st["case"], st["q"]
    B, M, H, dn = c["B"], c["M"], c["H"], c["dn"]
    out = torch.zeros((B, M, H, dn), dtype=q.dtype, device=_DEV)
    lse = torch.full((B, H, M), -math.inf, device=_DEV)
    scale = 1.0 / math.sqrt(dn + c["dr"])
    for b, n in enumerate(st["lens"]):
        pe = st["k_pe"][b, :n].float().unsqueeze(0).expand(H, n, c["dr"])
        k = torch.cat([st["k"][b, :n].float().transpose(0, 1), pe], -1)
        kt = k.transpose(1, 2).contiguous()
        v = st["v"][b, :n].float().transpose(0, 1).contiguous()
        step = 512
        for m0 in range(0, M, step):
            m1 = min(M, m0 + step)
            hi = min(n, max(0, n - M + m1)) if c["causal"] else n
            if hi == 0:
                continue
            idx = torch.arange(hi, device=_DEV)
            keep = idx <= n - M + torch.arange(m0, m1, device=_DEV).view(-1, 1) if c["causal"] else (idx >= 0).view(1, -1)
            rows = q[b, m0:m1].float().transpose(0, 1).contiguous()
            e, z, mx = _softmax_rows(torch.matmul(rows, kt[..., :hi].contiguous()) * scale, keep)
            o = torch.matmul(e, v[:, :hi].contiguous()) / torch.where(z > 0, z, torch.ones_like(z))
            out[b, m0:m1] = o.transpose(0, 1).to(q.dtype)
            lse[b, :, m0:m1] = (mx + torch.log(z))[..., 0]
    return {"out": out, "lse": lse}


# ----------------------------------------------------------------------------
# The package's operators
# ----------------------------------------------------------------------------

def _pkg():
    # The package lives in a subfolder of the working folder (the repository root).
    pkg = os.path.join(os.getcwd(), "specdiff-ae_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _own_slots(st):
    _pkg()
    from diffspec_mi355x.core.kv_cache.paged_kv import token_slots
    c = st["case"]
    return token_slots(st["table"], st["lens"], st["news"], c["page"], c["cap"], seqs=st["seqs"])


def _own_append(st):
    _pkg()
    from diffspec_mi355x.runtime.cache_state import append_latent_kv
    c = st["case"]
    q = append_latent_kv(st["kv"][:, :c["dc"]], st["kv"][:, c["dc"]:], st["cache"], st["slots"], norm_weight=st["weight"],
                         eps=_EPS, cos=st["cos"], sin=st["sin"], positions=st["positions"], interleaved=c["inter"],
                         q_pe=None if st["q"] is None else st["q"][..., 128:])
    return {"cache": st["cache"]} if q is None else {"cache": st["cache"], "q_pe": q}


def _own_absorbed(st):
    _pkg()
    from diffspec_mi355x.runtime.latent_attention import latent_attn_with_kvcache
    out, lse = latent_attn_with_kvcache(st["q"], st["kv"], st["case"]["dc"], st["scale"], cache_seqlens=st["seqlens"],
                                        page_table=st["table"], parent=st["parent"], return_softmax_lse=True)
    return {"out": out, "lse": lse}


def _own_expanded(st):
    _pkg()
    from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded
    out, lse = latent_attn_expanded(st["q"], st["k"], st["k_pe"], st["v"], cache_seqlens=st["seqlens"],
                                    causal=st["case"]["causal"], return_softmax_lse=True)
    return {"out": out, "lse": lse}


_PLAIN = dict(slots=_plain_slots, append=_plain_append, absorbed=_plain_absorbed, expanded=_plain_expanded)
_OWN = dict(slots=_own_slots, append=_own_append, absorbed=_own_absorbed, expanded=_own_expanded)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ----------------------------------------------------------------------------
# The definitions in 64 bits
# ----------------------------------------------------------------------------

def _exact_slots(c, st):
    table, lens = st["table"].cpu().numpy(), st["lens"].cpu().numpy()
    ps, cap = c["page"], c["cap"]
    slots, posn, reqs = np.full(cap, -1, dtype=np.int64), np.full(cap, -1, dtype=np.int32), np.full(cap, -1, dtype=np.int32)
    block = np.full((c["n"], table.shape[1]), -1, dtype=np.int32)
    cu, length = [0], []
    for i, (s, k) in enumerate(zip(st["seqs"].tolist(), st["news"].tolist())):
        n, at = int(lens[s]), cu[-1]
        p = np.arange(n - k, n)[:max(0, cap - at)]
        pg = table[s, p // ps].astype(np.int64)
        slots[at:at + len(p)] = np.where(pg >= 0, pg * ps + p % ps, -1)
        posn[at:at + len(p)], reqs[at:at + len(p)] = p, i
        used = -(-n // ps)
        block[i, :used] = table[s, :used]
        cu.append(at + k)
        length.append(n)
    dev = lambda a, t: torch.from_numpy(np.asarray(a, dtype=t)).to(_DEV)  # noqa: E731
    return {"slots": dev(slots, np.int64), "positions": dev(posn, np.int32), "requests": dev(reqs, np.int32),
            "cu_seqlens": dev(cu, np.int32), "block_table": dev(block, np.int32), "lens": dev(length, np.int32)}


def _exact_append(c, st):
    dc, dr, T = c["dc"], c["dr"], c["T"]
    x = st["kv"].double()
    lat = x[:, :dc]
    if c["norm"]:
        lat = lat * torch.rsqrt(lat.square().sum(1, keepdim=True) / dc + _EPS) * st["weight"].double()
    cos, sin = (st[k].double().index_select(0, st["positions"].long()) for k in ("cos", "sin"))
    # A rotation of the pairs (a, b) as a product of complex numbers.
    a, b = (slice(0, dr, 2), slice(1, dr, 2)) if c["inter"] else (slice(0, dr // 2), slice(dr // 2, dr))

    def rotate(y, cs, sn):
        z = torch.empty_like(y)
        z[..., a] = y[..., a] * cs[..., a] - y[..., b] * sn[..., a]
        z[..., b] = y[..., b] * cs[..., b] + y[..., a] * sn[..., b]
        return z

    cache = torch.zeros((c["P"] * c["page"], dc + dr), dtype=torch.float64, device=_DEV)
    v = c["valid"]
    cache[st["slots"][:v]] = torch.cat([lat[:v], rotate(x[:v, dc:], cos[:v], sin[:v])], 1)
    out = {"cache": cache.view(c["P"], c["page"], dc + dr)}
    if st["q"] is not None:
        out["q_pe"] = rotate(st["q"][..., 128:].double(), cos.view(T, 1, dr), sin.view(T, 1, dr))
    return out


def _ancestors(par):
    M = len(par)
    see = np.zeros((M, M), dtype=bool)
    for m in range(M):
        a = m
        while a >= 0:
            see[m, a] = True
            a = par[a]
    return see


def _exact_absorbed(c, st):
    B, M, H, dc = c["B"], c["M"], c["H"], c["dc"]
    out = torch.zeros((B, M, H, dc), dtype=torch.float64, device=_DEV)
    lse = torch.full((B, H, M), -math.inf, dtype=torch.float64, device=_DEV)
    for b, n in enumerate(st["lens"]):
        if st["table"] is None:
            x = st["kv"][b, :n].double()
        else:
            used = st["table"][b, :-(-n // c["page"])].long()
            x = st["kv"][used].flatten(0, 1)[:n].double()
        see = np.tril(np.ones((M, n), dtype=bool), n - M)
        if c["tree"]:
            see[:, :n - M] = True
            see[:, n - M:] = _ancestors(st["parent"][b].tolist())
        for m0 in range(0, M, 64):
            vis = torch.from_numpy(see[m0:m0 + 64]).to(_DEV)
            for h in range(H) if M > 1 else [slice(None)]:
                s = st["q"][b, m0:m0 + 64, h].double().reshape(-1, x.shape[1]) @ x.T * st["scale"]
                s = s.masked_fill(~(vis if M > 1 else vis.expand(s.shape[0], n)), -math.inf)
                l = torch.logsumexp(s, -1)
                w = torch.exp(s - torch.nan_to_num(l, neginf=0.0)[:, None])
                if M > 1:
                    lse[b, h, m0:m0 + 64], out[b, m0:m0 + 64, h] = l, w @ x[:, :dc]
                else:
                    lse[b, :, 0], out[b, 0] = l, w @ x[:, :dc]
    return {"out": out, "lse": lse}


def _exact_expanded(c, st):
    B, M, H, dn = c["B"], c["M"], c["H"], c["dn"]
    out = torch.zeros((B, M, H, dn), dtype=torch.float64, device=_DEV)
    lse = torch.full((B, H, M), -math.inf, dtype=torch.float64, device=_DEV)
    for b, n in enumerate(st["lens"]):
        for h in range(H):
            k, v, pe = st["k"][b, :n, h].double(), st["v"][b, :n, h].double(), st["k_pe"][b, :n].double()
            q = st["q"][b, :, h].double()
            for m0 in range(0, M, 2048):
                s = (q[m0:m0 + 2048, :dn] @ k.T + q[m0:m0 + 2048, dn:] @ pe.T) / math.sqrt(dn + c["dr"])
                if c["causal"]:
                    hidden = torch.ones_like(s, dtype=torch.bool).triu(n - M + m0 + 1)
                    s = s.masked_fill(hidden, -math.inf)
                l = torch.logsumexp(s, -1)
                lse[b, h, m0:m0 + 2048] = l
                out[b, m0:m0 + 2048, h] = torch.exp(s - torch.nan_to_num(l, neginf=0.0)[:, None]) @ v
    return {"out": out, "lse": lse}


_EXACT = dict(slots=_exact_slots, append=_exact_append, absorbed=_exact_absorbed, expanded=_exact_expanded)


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["kind"]](case, prepare(case, seed))
