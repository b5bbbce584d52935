"""Refusals of the latent cache's operators (CPU only: nothing is launched)."""

import pytest
import torch

from diffspec_mi355x import _ext
from diffspec_mi355x.core.kv_cache import token_slots
from diffspec_mi355x.runtime.cache_state import append_latent_kv
from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
WS = torch.empty((1 << 27) + 256, dtype=torch.uint8)
PTR = (WS.data_ptr() + 255) // 256 * 256


@pytest.fixture()
def dry(dsv_lib):
    dsv_lib.dsv_set_dry_run(1)
    yield dsv_lib
    dsv_lib.dsv_set_dry_run(0)


def f(*s, dtype=torch.bfloat16):
    return torch.zeros(s, dtype=dtype)


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def absorbed(lib, B=2, M=3, H=4, dc=512, dr=64, N=40, n_keys=-1, scale=0.1, v_dim=None, nbytes=1 << 27, ws=PTR, **kw):
    t = dict(q=f(B, M, H, dc + dr), kv=f(B, N, dc + dr), table=None, lens=None, parent=None, out=f(B, M, H, dc),
             lse=f(B, H, M, dtype=torch.float32))
    t.update(kw)
    d = {k: _ext.desc(x) for k, x in t.items()}
    return lib.dsv_latent_attention(d["q"], d["kv"], dc if v_dim is None else v_dim, d["table"], d["lens"], n_keys, scale, d["parent"],
                                    d["out"], d["lse"], ws, nbytes, None)


def test_absorbed(dry):
    paged = dict(kv=f(7, 8, 576), table=i32(2, 5))
    assert absorbed(dry) == 0
    assert absorbed(dry, lse=None) == 0
    assert absorbed(dry, n_keys=10 ** 12) == 0
    assert absorbed(dry, **paged) == 0
    assert absorbed(dry, **{**paged, "table": torch.zeros(5, dtype=torch.int64)}) == 0
    assert absorbed(dry, dc=256, dr=32) == 0
    assert absorbed(dry, parent=i32(3), lens=i32(2)) == 0
    assert absorbed(dry, parent=i32(2, 3).long(), lens=i32(2).long()) == 0
    assert absorbed(dry, out=f(2, 3, 4, 512, dtype=torch.float32)) == 0
    assert absorbed(dry, kv=f(2, 40, 584)[..., :576]) == 0
    for bad in [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-60),
                dict(v_dim=0), dict(v_dim=600), dict(q=f(2, 3, 576)), dict(q=f(2, 0, 4, 576), out=f(2, 0, 4, 512)),
                dict(kv=f(2, 40, 512)), dict(kv=f(3, 40, 576)), dict(kv=f(2, 40, 576, dtype=torch.float16)), dict(kv=f(2, 40, 577)[..., 1:]),
                dict(kv=f(2, 40, 580)[..., :576]), dict(q=f(2 * 3 * 4 * 576 + 1)[1:].view(2, 3, 4, 576)), dict(out=f(2, 3, 4, 576)),
                dict(out=f(2, 3, 4, 512, dtype=torch.int32)), dict(out=f(2, 3, 512, 4).transpose(2, 3)), dict(lse=f(2, 3, 4, dtype=torch.float32)),
                dict(lse=f(2, 4, 3)), dict(lens=i32(3)), dict(lens=f(2)), dict(lens=i32(4)[::2]), dict(parent=i32(4)), dict(parent=i32(3, 3)),
                dict(parent=f(3)), {**paged, "table": i32(3, 5)}, {**paged, "table": f(2, 5)}, {**paged, "table": i32(5, 2).t()},
                {**paged, "table": i32(1, 2, 5)}]:
        assert absorbed(dry, **bad) == INVALID, (bad.keys(), _ext.last_error())
    assert absorbed(dry, v_dim=500) == UNSUPPORTED
    assert absorbed(dry, dc=128) == UNSUPPORTED
    assert absorbed(dry, dr=16) == UNSUPPORTED
    assert absorbed(dry, **{**paged, "kv": f(7, 6, 576)}) == UNSUPPORTED
    assert absorbed(dry, B=1, M=1025, parent=i32(1025)) == UNSUPPORTED
    one = f(1, 1, 1, 576)
    for B, M, H in ((1, (1 << 24) + 1, 1), (1, 1 << 20, 32), ((1 << 20) + 1, 1, 1), (1, 1, 65537), (1 << 20, 64, 64)):
        assert absorbed(dry, B=1, q=one.expand(B, M, H, 576), kv=f(1, 40, 576).expand(B, 40, 576),
                        out=f(1, 1, 1, 512).expand(B, M, H, 512), lse=None) == UNSUPPORTED, (B, M, H)
        assert dry.dsv_latent_workspace_bytes(B, M, H, 512, 0, 40, 0, 0) == 0
    many = dict(B=1, N=8192)  # (keys shared out over workgroups)
    need = dry.dsv_latent_workspace_bytes(1, 3, 4, 512, 0, 8192, 0, 0)
    assert 0 < need <= 1 << 27
    assert absorbed(dry, nbytes=need, **many) == 0
    assert absorbed(dry, nbytes=need - 1, **many) == WORKSPACE
    assert absorbed(dry, ws=None, **many) == WORKSPACE
    assert absorbed(dry, ws=PTR + 64, nbytes=need, **many) == WORKSPACE
    q = f(2, 3, 4, 576)
    assert absorbed(dry, q=q, out=q[..., :512]) == INVALID
    assert absorbed(dry, q=q.float(), kv=f(2, 40, 576).float(), out=f(2, 3, 4, 512), lse=q.float().view(-1)[:24].view(2, 4, 3)) == 0


def expanded(lib, B=2, M=3, H=4, dn=128, dr=64, N=40, n_keys=-1, scale=0.1, causal=1, nbytes=1 << 27, ws=PTR, **kw):
    t = dict(q=f(B, M, H, dn + dr), k=f(B, N, H, dn), pe=f(B, N, dr), v=f(B, N, H, dn), lens=None, out=f(B, M, H, dn),
             lse=f(B, H, M, dtype=torch.float32))
    t.update(kw)
    d = {k: _ext.desc(x) for k, x in t.items()}
    return lib.dsv_latent_expanded(d["q"], d["k"], d["pe"], d["v"], d["lens"], n_keys, causal, scale, d["out"], d["lse"], ws, nbytes, None)


def test_expanded(dry):
    kv = f(2, 40, 4, 256)
    assert expanded(dry) == 0 and expanded(dry, causal=0, lens=i32(2), lse=None) == 0
    assert expanded(dry, dn=64, dr=32) == 0
    assert expanded(dry, k=kv[..., :128], v=kv[..., 128:], pe=f(2, 40, 576)[..., 512:]) == 0
    for bad in [dict(scale=0.0), dict(q=f(2, 3, 4, 128)), dict(k=f(2, 41, 4, 128)), dict(v=f(2, 41, 4, 128)), dict(pe=f(2, 41, 64)),
                dict(k=f(2, 40, 2, 128)), dict(v=f(1, 40, 4, 128)), dict(pe=f(2, 40, 64).half()), dict(pe=f(2, 40, 4, 64)),
                dict(lens=i32(3)), dict(out=f(2, 3, 4, 64)), dict(lse=f(2, 3, 4, dtype=torch.float32)), dict(v=f(2, 40, 4, 129)[..., 1:])]:
        assert expanded(dry, **bad) == INVALID, (bad.keys(), _ext.last_error())
    assert expanded(dry, dn=96) == UNSUPPORTED
    assert expanded(dry, dr=128) == UNSUPPORTED
    assert expanded(dry, v=f(2, 40, 4, 64)) == UNSUPPORTED
    need = dry.dsv_latent_workspace_bytes(1, 3, 4, 128, 0, 8192, 0, 1)
    assert need > 0 and expanded(dry, B=1, N=8192, nbytes=need) == 0 and expanded(dry, B=1, N=8192, nbytes=need - 1) == WORKSPACE
    assert dry.dsv_latent_workspace_bytes(1, 3, 4, 96, 0, 8192, 0, 1) == 0
    assert dry.dsv_latent_workspace_bytes(1, 3, 4, 128, 3, 8192, 0, 1) == 0
    out = kv[:, :3, :, :128]
    assert expanded(dry, k=kv[..., :128], v=kv[..., 128:], out=out) == INVALID


def slots(lib, B=3, n=2, n_log=5, page=8, cap=9, with_seqs=True, **kw):
    t = dict(table=i32(B, n_log), lens=i32(B), news=i32(n), seqs=i32(n) if with_seqs else None, slots=torch.zeros(cap, dtype=torch.int64),
             pos=i32(cap), req=i32(cap), cu=i32(n + 1), block=i32(n, n_log), out=i32(n))
    t.update(kw)
    d = {k: _ext.desc(x) for k, x in t.items()}
    return lib.dsv_token_slots(d["table"], d["lens"], d["news"], d["seqs"], page, d["slots"], d["pos"], d["req"], d["cu"], d["block"],
                               d["out"], None)


def test_slots(dry):
    assert slots(dry) == 0 and slots(dry, n=3, with_seqs=False) == 0 and slots(dry, cap=0) == 0 and slots(dry, n=0) == 0
    assert slots(dry, lens=i32(3).long(), news=i32(2).long(), seqs=i32(4).long()[::2]) == 0
    for bad in [dict(n=2, with_seqs=False), dict(table=i32(15)), dict(table=i32(3, 5).long()), dict(table=i32(5, 3).t()), dict(lens=i32(4)),
                dict(lens=f(3)), dict(lens=i32(6)[::2]), dict(news=f(2)), dict(seqs=i32(3)), dict(slots=i32(9)), dict(pos=i32(8)),
                dict(req=i32(9).long()), dict(cu=i32(2)), dict(block=i32(2, 4)), dict(block=i32(1, 5).expand(2, 5)), dict(out=i32(3)),
                dict(pos=i32(18)[::2])]:
        assert slots(dry, **bad) == INVALID, (bad.keys(), _ext.last_error())
    assert slots(dry, page=6) == UNSUPPORTED and slots(dry, page=0) == UNSUPPORTED
    assert slots(dry, page=1 << 30) == UNSUPPORTED
    lens = i32(3)
    assert slots(dry, lens=lens, out=lens[:2]) == INVALID
    x = i32(20)
    assert slots(dry, pos=x[:9], req=x[8:17]) == INVALID


def append(lib, T=6, dc=64, dr=32, H=2, P=3, page=8, n_pos=20, inter=0, eps=1e-6, with_q=True, rope=True, positions=True, **kw):
    t = dict(c=f(T, dc), pe=f(T, dr), w=None, cos=f(n_pos, dr) if rope else None, sin=f(n_pos, dr) if rope else None,
             pos=i32(T) if rope and positions else None, slots=i32(T), cache=f(P, page, dc + dr), q=f(T, H, dr) if with_q else None,
             qo=f(T, H, dr) if with_q else None)
    t.update(kw)
    d = {k: _ext.desc(x) for k, x in t.items()}
    return lib.dsv_latent_append(d["c"], d["pe"], d["w"], eps, d["cos"], d["sin"], d["pos"], inter, d["slots"], d["cache"], d["q"],
                                 d["qo"], None)


def test_append(dry):
    assert append(dry) == 0 and append(dry, with_q=False) == 0 and append(dry, rope=False) == 0
    assert append(dry, positions=False, n_pos=6) == 0
    assert append(dry, cache=f(24, 96), w=f(64), slots=i32(6).long()) == 0
    assert append(dry, cos=f(20, 32).float(), sin=f(20, 32).float()) == 0
    kv = f(6, 96)
    assert append(dry, c=kv[:, :64], pe=kv[:, 64:]) == 0
    q = f(6, 2, 32)
    assert append(dry, q=q, qo=q) == 0
    for bad in [dict(c=f(7, 64)), dict(pe=f(7, 32)), dict(c=f(6, 64).half()), dict(cache=f(3, 8, 104)), dict(cache=f(3, 8, 96).half()),
                dict(cos=None), dict(sin=f(20, 40)), dict(sin=f(19, 32)), dict(cos=f(20, 32).half(), sin=f(20, 32).half()),
                dict(positions=False), dict(pos=i32(7)), dict(pos=f(6)), dict(pos=i32(12)[::2]), dict(slots=i32(5)), dict(slots=f(6)),
                dict(slots=i32(12)[::2]), dict(w=f(63)), dict(w=f(64), eps=-1.0), dict(w=f(64), eps=float("nan")), dict(q=None),
                dict(qo=f(6, 3, 32)), dict(q=f(5, 2, 32), qo=f(5, 2, 32)), dict(qo=f(6, 1, 32).expand(6, 2, 32)),
                dict(cache=f(1, 8, 96).expand(3, 8, 96)), dict(cache=f(3, 1, 96).expand(3, 8, 96)), dict(rope=False, pos=i32(6)),
                dict(c=f(6, 65)[:, 1:]), dict(pe=f(0, 32), c=f(0, 64))]:
        assert append(dry, **bad) == INVALID, (bad.keys(), _ext.last_error())
    assert append(dry, dc=60) == INVALID
    assert append(dry, c=f(6, 64)[:, :60], cache=f(3, 8, 96)[..., :92]) == UNSUPPORTED
    assert append(dry, dr=24) == UNSUPPORTED
    assert append(dry, page=6) == UNSUPPORTED
    assert append(dry, dc=2056) == UNSUPPORTED
    for T, want in ((1 << 24, 0), ((1 << 24) + 1, UNSUPPORTED)):
        assert append(dry, T=1, rope=False, with_q=False, c=f(1, 64).expand(T, 64), pe=f(1, 32).expand(T, 32),
                      slots=torch.empty(T, dtype=torch.int32)) == want
    none = dict(T=0, slots=i32(0))
    assert append(dry, **none) == 0 and append(dry, with_q=False, rope=False, **none) == 0
    assert append(dry, T=0, slots=i32(1)) == INVALID and append(dry, pe=f(0, 24), **none) == INVALID
    cache = f(3, 8, 96)
    assert append(dry, cache=cache, c=cache.view(24, 96)[:6, :64]) == INVALID
    assert append(dry, q=q, qo=q.view(2, 6, 32).transpose(0, 1)) == INVALID
    assert append(dry, cache=cache, qo=cache.view(-1)[:384].view(6, 2, 32)) == INVALID


def test_workspace_of_every_plan(dry):
    """Few enough partials for the largest batches, and none where every workgroup has a unit of its own."""
    ws = dry.dsv_latent_workspace_bytes
    assert ws(1 << 20, 1, 512, 128, 0, 64, 0, 1) == 0        # (512 units fill 256 CUs twice)
    assert ws(1 << 20, 1, 200, 128, 0, 64, 0, 1) > 0         # (rows to be joined of 2^27.6 blocks of 256)
    assert ws(1, 8192, 128, 128, 0, 8192, 0, 1) == 0
    assert ws(1 << 20, 1, 1024, 512, 0, 1 << 20, 0, 0) == 0  # (beyond the range: too many tiles)
    for B, M, H, n in ((1, 1, 16, 1), (1, 1, 128, 1 << 20), (64, 1, 128, 4096), (7, 48, 16, 5000), (3, 1, 1, 200)):
        for dtype in (0, 1, 2):
            assert ws(B, M, H, 512, dtype, n, 0, 0) <= 512 * 2 * 2 * 4 * 64 * (512 + 2) * 4


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="GPU only"):
        token_slots(i32(2, 3), i32(2), i32(2), 8, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        append_latent_kv(f(2, 64), f(2, 32), f(2, 8, 96), i32(2))
    with pytest.raises(RuntimeError, match="GPU only"):
        latent_attn_with_kvcache(f(1, 1, 1, 576), f(1, 4, 576), 512, 0.1)
    with pytest.raises(RuntimeError, match="GPU only"):
        latent_attn_expanded(f(1, 1, 1, 192), f(1, 4, 1, 128), f(1, 4, 64), f(1, 4, 1, 128))
