"""Operators on packed sequences (ait_amd/packed.py) against their definitions in 64 bits, and their refusals.

Tolerances are bounds, element by element, from the roundings the kernels make: u = eps / 2 of the tensors' type for every
value that is rounded to it (the probabilities and dS where they enter a product, the results), 2^-24 for an f32 operation, and
the error of a score, es, passed on by exp.  They are computed beside the reference, before anything is compared."""
import ctypes
import math

import pytest
import torch

from ait_amd import _lib, ops, packed

F8 = torch.float64


def starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


# ------------------------------------------------------------------------------------------
# attention: reference and bounds
# ------------------------------------------------------------------------------------------
def attn_ref(q, k, v, ql, qs, kl, ks, causal, scale, table=None, bucket_of=None, do=None):
    """results and bounds {name: (value, bound)} in 64 bits on the CPU"""
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = (t.detach().cpu().to(F8) for t in (q, k, v))
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    z = lambda t: torch.zeros_like(t)
    o, eo, dq, edq, dk, edk, dv, edv = z(q), z(q), z(q), z(q), z(k), z(k), z(v), z(v)
    if table is not None:
        table, bucket_of = table.detach().cpu().to(F8), bucket_of.cpu().long()
        m = bucket_of.numel() // 2
        dt, edt = z(table), z(table)
    do = None if do is None else do.detach().cpu().to(F8)
    f = 2.0 ** -24
    for a, qa, b, kb in zip(ql, qs, kl, ks):
        if a <= 0 or b <= 0:
            continue
        rel = torch.arange(b)[None, :] - torch.arange(a)[:, None] - (b - a)
        for h in range(H):
            c = h * Hk // H
            Q, K, V = q[qa:qa + a, h], k[kb:kb + b, c], v[kb:kb + b, c]
            s = scale * Q @ K.t()
            es = (d + 8) * f * (abs(scale) * Q.abs() @ K.abs().t())
            if table is not None:
                t = table[:, h][bucket_of[rel.clamp(-m, m) + m]]
                s, es = s + t, es + 4 * f * t.abs()
            es = es + 8 * f * s.abs()
            hide = rel > 0 if causal else torch.zeros_like(rel, dtype=torch.bool)
            s = s.masked_fill(hide, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(hide | (top == -math.inf), torch.zeros_like(s), torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)))
            tot = p.sum(1, keepdim=True)
            p = p / torch.where(tot > 0, tot, torch.ones_like(tot))
            es = torch.where(hide | ~torch.isfinite(s), torch.zeros_like(es), es)
            rp = es + es.amax(1, keepdim=True) + (2 * b + 16) * f                    # relative error of a probability
            po = p * (rp + u)
            O = p @ V
            o[qa:qa + a, h] = O
            EO = po @ V.abs() + (b + 8) * f * (p @ V.abs())
            EO = EO + u * (O.abs() + EO)
            eo[qa:qa + a, h] = EO
            if do is None:
                continue
            G = do[qa:qa + a, h]
            dp = G @ V.t()
            delta = (G * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = (d + 4) * f * (G.abs() @ V.abs().t())
            edelta = (G.abs() * EO).sum(1, keepdim=True) + (d + 4) * f * (G.abs() * O.abs()).sum(1, keepdim=True)
            eds = p * (edp + edelta) + ds.abs() * (rp + 4 * f) + p * rp * edelta
            edsr = eds + u * (ds.abs() + eds)                                        # ... rounded where it enters a product
            n = (a * H // Hk + b + 16) * f
            dv[kb:kb + b, c] += p.t() @ G
            edv[kb:kb + b, c] += (po + n * p).t() @ G.abs()
            dq[qa:qa + a, h] = scale * ds @ K
            edq[qa:qa + a, h] = abs(scale) * (edsr + n * ds.abs()) @ K.abs()
            dk[kb:kb + b, c] += scale * ds.t() @ Q
            edk[kb:kb + b, c] += abs(scale) * (edsr + n * ds.abs()).t() @ Q.abs()
            if table is not None:
                at = bucket_of[rel.clamp(-m, m) + m].reshape(-1)
                dt[:, h].index_add_(0, at, ds.reshape(-1))
                edt[:, h].index_add_(0, at, (eds + (a * b) ** 0.5 * 8 * f * ds.abs()).reshape(-1))
    out = {"o": (o, eo)}
    if do is not None:
        r = lambda x, e: (x, e + u * (x.abs() + e))
        out.update(dq=r(dq, edq), dk=r(dk, edk), dv=r(dv, edv))
        if table is not None:
            out["dt"] = (dt, edt + 64 * f * dt.abs())
    return out


def within(got, want, what):
    x, e = want
    off = (got.detach().cpu().to(F8) - x).abs()
    bad = ~(off <= e * 1.001 + 1e-30)
    assert not bool(bad.any()), "%s: %d of %d outside, worst %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max() if bool(bad.any()) else 0), float(e[bad][off[bad].argmax()] if bool(bad.any()) else 0))


def make(lens_q, lens_k, H, Hk, d, dtype, seed, fused=False, cache=0):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(lens_q) + 3, (cache * len(lens_k) if cache else sum(lens_k)) + 2        # (a few rows of no sequence)
    if fused and tq + 2 >= tk:
        w = torch.randn(max(tq, tk), (H + 2 * Hk) * d, generator=g).to(dtype).cuda()
        q = w[:tq, :H * d].view(tq, H, d)
        k, v = (w[:tk, (H + i * Hk) * d:(H + (i + 1) * Hk) * d].view(tk, Hk, d) for i in (0, 1))
    else:
        q, k, v = (torch.randn(t, n, d, generator=g).to(dtype).cuda() for t, n in ((tq, H), (tk, Hk), (tk, Hk)))
    do = torch.randn(tq, H, d, generator=g).to(dtype).cuda()
    return q, k, v, do


RAGGED = [5, 0, 1, 64, 63, 130, 17, 65]
LONG = [300, 1, 257]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,H,Hk,d,causal", [
    ([1], 1, 1, 8, True), (RAGGED, 2, 1, 64, True), (RAGGED, 3, 3, 40, False), (LONG, 4, 2, 128, True), ([200, 70], 8, 1, 96, False),
    (LONG, 6, 2, 72, True), ([33] * 9, 8, 8, 64, False), ([1, 2, 3, 4], 16, 2, 128, True)])
def test_self_attention(dtype, lens, H, Hk, d, causal):
    q, k, v, do = make(lens, lens, H, Hk, d, dtype, 1 + H + d, fused=True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    cu = starts(lens)
    o = packed.packed_attention(*leaves, cu.cuda(), causal=causal)
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), causal, d ** -0.5, do=do)
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t, want[n], n)
        assert bool((t[sum(lens):] == 0).all()), n + ": rows behind the last sequence"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ql,kl,H,Hk,d,causal", [
    ([64, 64], [149, 150], 8, 8, 64, False), ([10, 3, 0, 70], [0, 200, 40, 65], 4, 2, 64, True), ([90, 5], [20, 300], 2, 2, 128, True),
    ([7, 1, 2], [513, 64, 1], 8, 2, 24, True), ([150], [31], 2, 1, 64, True)])
def test_queries_and_keys_of_different_lengths(dtype, ql, kl, H, Hk, d, causal):
    """with a causal mask and more queries than keys the first queries see nothing"""
    q, k, v, do = make(ql, kl, H, Hk, d, dtype, 7)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cq, ck = starts(ql), starts(kl)
    o = packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=causal, scale=0.2, max_q=max(ql), max_k=max(kl))
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(q, k, v, ql, cq.tolist(), kl, ck.tolist(), causal, 0.2, do=do)
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t, want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,H,Hk,d,causal,n,m,two", [
    (RAGGED, 2, 2, 64, False, 8, 20, True), (LONG, 4, 1, 64, True, 32, 128, False), (LONG, 2, 1, 128, False, 32, 100, True),
    ([500], 1, 1, 32, True, 16, 9, False), ([40, 64, 3], 8, 8, 64, False, 16, 2000, True)])
def test_relative_position_bias(dtype, lens, H, Hk, d, causal, n, m, two):
    q, k, v, do = make(lens, lens, H, Hk, d, dtype, 11 + m)
    bias = packed.RelativePositionBias(H, n, m, two).cuda()
    with torch.no_grad():
        bias.weight.copy_(torch.randn(n, H, generator=torch.Generator().manual_seed(5)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)] + [bias.weight]
    cu = starts(lens)
    o = packed.packed_attention(q, k, v, cu.cuda(), causal=causal, bias=bias)
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), causal, d ** -0.5, bias.weight, bias.bucket_of, do)
    for name, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new,kl,cap,H,Hk,d,bias", [
    ([1] * 4, [30, 1, 0, 77], 80, 8, 8, 64, False), ([1] * 2, [5000, 4097], 5001, 8, 2, 128, False), ([1, 1, 3], [700, 64, 65], 900, 32, 4, 64, True),
    ([7], [3000], 3000, 4, 4, 40, True), ([1], [1], 1, 1, 1, 8, True), ([40, 2], [1500, 2], 1600, 8, 2, 64, True)])
def test_new_tokens_over_caches(dtype, new, kl, cap, H, Hk, d, bias):
    """what lies behind a cache's length, and rows of no sequence, may hold anything"""
    q, k, v, _ = make(new, kl, H, Hk, d, dtype, 23, cache=cap)
    ks = [i * cap for i in range(len(kl) + 1)]
    for i, n in enumerate(kl):
        for t in (k, v):
            t[ks[i] + n:ks[i + 1]] = float("nan") if i % 2 else float("inf")
    k[ks[-1]:] = float("nan")
    q[sum(new):] = float("nan")
    b = None
    if bias:
        b = (torch.randn(32, H, generator=torch.Generator().manual_seed(3)).cuda(), packed.relative_buckets(32, 128, False, "cuda"))
    with torch.no_grad():
        o = packed.packed_attention(q, k, v, starts(new).cuda(), torch.tensor(ks, dtype=torch.int32).cuda(),
                                    k_len=torch.tensor(kl, dtype=torch.int32).cuda(), causal=True, bias=b, max_q=max(new), max_k=max(kl))
    k, v = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (k, v))
    want = attn_ref(q, k, v, new, starts(new).tolist(), kl, ks, True, d ** -0.5, *(b or (None, None)))
    within(o[:sum(new)], tuple(t[:sum(new)] for t in want["o"]), "o")
    assert bool((o[sum(new):] == 0).all())


def test_relative_buckets_are_the_definition():
    for n, two in ((2, False), (8, False), (50, False), (4, True), (32, True), (50, True)):
        side = n // 2 if two else n
        e = side // 2
        for m in (side + 1, 128, 517):
            if m <= e:
                continue
            got = packed.relative_buckets(n, m, two)
            assert got.dtype == torch.int32 and got.numel() == 2 * m + 1
            for rel in range(-m, m + 1):
                a = abs(rel) if two else max(0, -rel)
                if a < e:
                    want = a
                else:      # the logarithms, away from their borders
                    x = math.log(a / e) / math.log(m / e) * (side - e)
                    if abs(x - round(x)) < 1e-9 and a < m:
                        want = min(side - 1, e + round(x))
                    else:
                        want = min(side - 1, e + int(x))
                assert int(got[rel + m]) == want + (side if two and rel > 0 else 0), (n, two, m, rel)
    for bad in ((0, 10, False), (1, 10, False), (3, 10, True), (2, 10, True), (16, 8, False), (600, 1000, False), (32, 5000, True)):
        with pytest.raises(ValueError):
            packed.relative_buckets(*bad)


def test_attention_refuses_what_it_does_not_take():
    t = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)
    cu = starts([2, 3])
    good = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cu_q=cu)
    table, of = t(8, 4), packed.relative_buckets(8, 20, True)
    with pytest.raises(_lib.AitHipError, match="no CPU fallback"):
        packed.packed_attention(**good)
    for change in (dict(q=t(5, 256)), dict(q=t(5, 4, 64, dt=torch.float16)), dict(q=t(5, 4, 64, dt=torch.bfloat16)), dict(q=t(5, 3, 64)),
                   dict(q=t(5, 4, 32)), dict(v=t(4, 2, 64)), dict(v=t(5, 2, 32)), dict(q=t(5, 4, 136), k=t(5, 2, 136), v=t(5, 2, 136)),
                   dict(q=t(5, 4, 12), k=t(5, 2, 12), v=t(5, 2, 12)), dict(cu_q=cu.long()), dict(cu_q=cu[None]), dict(cu_k=starts([5])),
                   dict(k_len=cu), dict(k_len=starts([2]).float()), dict(bias=(t(8, 3), of)), dict(bias=(table, of[1:])),
                   dict(bias=(table, of.long())), dict(bias=(table.half(), of)), dict(bias=(t(600, 4), of)),
                   dict(bias=(table, torch.zeros(2 * 2049 + 1, dtype=torch.int32)))):
        with pytest.raises(_lib.AitHipError):
            packed.packed_attention(**{**good, **change})
            pytest.fail("taken: %s" % list(change))


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    base = dict(n_seq=2, total_q=5, total_k=5, heads=4, kv_heads=2, d=64, dtype=0, scale=1.0, cu_q=4096, cu_k=4096)

    def fwd(qptr=4096, qrow=256, qhead=64, **kw):
        p = _lib.PackedAttn(**{**base, **kw})
        return L.ait_packed_attn_fwd(ctypes.byref(p), qptr, qrow, qhead, *(4096, 128, 64) * 2, 4096, 256, 64, None, None, 0, None)

    def bwd(ws=4096, n=1 << 30, lse=4096, **kw):
        p = _lib.PackedAttn(**{**base, **kw})
        return L.ait_packed_attn_bwd(ctypes.byref(p), *(4096, 256, 64), *(4096, 128, 64) * 2, *(4096, 256, 64) * 2, lse, *(4096, 256, 64),
                                     *(4096, 128, 64) * 2, None, ws, n, None)
    EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -4
    for f in (fwd, bwd):
        for kw in (dict(heads=0), dict(kv_heads=3), dict(n_seq=-1), dict(total_q=-1), dict(d=0), dict(dtype=2), dict(cu_q=None), dict(cu_k=None),
                   dict(max_q=-1), dict(scale=float("nan")), dict(bias_table=4096), dict(bias_table=4096, bucket_of=4096, n_buckets=0)):
            assert f(**kw) == EINVAL, kw
        for kw in (dict(d=136), dict(d=12), dict(bias_table=4096, bucket_of=4096, n_buckets=513), dict(total_q=2 ** 30),
                   dict(bias_table=4096, bucket_of=4096, n_buckets=4, max_distance=2049)):
            assert f(**kw) == EUNSUPPORTED, kw
        assert f(n_seq=0) == 0
    assert fwd(qptr=None) == EINVAL and fwd(qptr=4100) == EUNSUPPORTED and fwd(qrow=255) == EUNSUPPORTED and fwd(qhead=65) == EUNSUPPORTED
    assert fwd(qrow=1 << 24) == EUNSUPPORTED
    assert bwd(lse=None) == EINVAL and bwd(ws=None) == EWORKSPACE and bwd(n=2 * 4 * 5 * 4 - 1) == EWORKSPACE
    assert L.ait_packed_attn_fwd(None, *(None, 0, 0) * 4, None, None, 0, None) == EINVAL
    # a few tokens over a long key axis are cut along it: a workspace is asked for, and a small one refused
    p = dict(n_seq=2, total_q=2, total_k=20000, max_q=1, max_k=10000)
    need = L.ait_packed_attn_fwd_workspace_bytes(ctypes.byref(_lib.PackedAttn(**{**base, **p})))
    assert need > 0 and fwd(**p) == EWORKSPACE
