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
        table_type, table, bucket_of = table.dtype, table.detach().cpu().to(F8), bucket_of.cpu().long()
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
            eo[qa:qa + a, h] = EO + u * (O.abs() + EO)
            EO = EO + max(u * u, f) * (O.abs() + EO) * 1.01          # ... and the backward has what its rounding took
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
            edt = edt + 64 * f * dt.abs()
            out["dt"] = (dt, edt + torch.finfo(table_type).eps / 2 * (dt.abs() + edt))
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
    ([500], 1, 1, 32, True, 16, 9, False), ([40, 64, 3], 8, 8, 64, False, 16, 2000, True), ([300, 33], 2, 1, 128, False, 512, 2048, True)])
def test_relative_position_bias(dtype, lens, H, Hk, d, causal, n, m, two):
    q, k, v, do = make(lens, lens, H, Hk, d, dtype, 11 + m)
    bias = packed.RelativePositionBias(H, n, m, two).to("cuda", dtype if H > 1 else torch.float32)
    with torch.no_grad():
        bias.weight.copy_(torch.randn(n, H, generator=torch.Generator().manual_seed(5)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)] + [bias.weight]
    cu = starts(lens)
    o = packed.packed_attention(q, k, v, cu.cuda(), causal=causal, bias=bias)
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), causal, d ** -0.5, bias.weight, bias.bucket_of, do)
    for name, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[name], name)
    assert grads[3].dtype == bias.weight.dtype


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ql,kl,H,Hk,d,causal,bias,max_q,max_k", [
    ([40, 64, 3, 0, 33], None, 4, 2, 64, True, True, 64, 64), ([40, 64, 3, 0, 33], None, 2, 2, 128, False, True, 64, 64),
    ([64], [1500], 2, 1, 64, False, True, 64, 1500), ([50, 9], [700, 1200], 2, 2, 128, True, True, 50, 1200),
    ([100], [2500], 1, 1, 32, False, False, 100, 2500), ([130, 70, 300], None, 2, 1, 64, True, True, 1, 1), ([130, 300], None, 2, 1, 128, True, False, 64, 64)])
def test_how_the_work_is_cut_up_does_not_show(dtype, ql, kl, H, Hk, d, causal, bias, max_q, max_k):
    """small workgroups, one tile at a time, the key axis in parts -- and hints that are too small"""
    kl = ql if kl is None else kl
    q, k, v, do = make(ql, kl, H, Hk, d, dtype, 31)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    b = None
    if bias:
        b = (torch.randn(12, H, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True), packed.relative_buckets(12, 50, True, "cuda"))
        leaves.append(b[0])
    cq, ck = starts(ql), starts(kl)
    run = lambda: packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=causal, bias=b, max_q=max_q, max_k=max_k)
    o = run()
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(q, k, v, ql, cq.tolist(), kl, ck.tolist(), causal, d ** -0.5, *(b or (None, None)), do=do)
    for n, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[n], n)
    o2 = run()
    again = torch.autograd.grad(o2, leaves, do)
    assert torch.equal(o, o2) and all(torch.equal(x, y) for x, y in zip(grads, again)), "not the same twice"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ql,kl,cap,H,Hk,d,causal,bias", [
    ([1100], [70], 90, 4, 2, 64, False, True), ([2100], [64], 64, 1, 1, 128, True, False), ([700, 40, 0, 300], [600, 700, 5, 0], 701, 8, 2, 128, True, False),
    ([1300], [520], 530, 2, 1, 72, False, False), ([640, 90], [3, 200], 257, 16, 2, 128, False, True), ([900], [900], 900, 2, 2, 64, True, True)])
def test_gradients_of_few_keys_in_parts(dtype, ql, kl, cap, H, Hk, d, causal, bias):
    """many queries on few keys: the query axis of the keys' gradients in parts that begin inside a head's tiles; wide blocks of
    keys; cache rows behind a sequence's length and rows of no sequence get zeros and may hold anything"""
    q, k, v, do = make(ql, kl, H, Hk, d, dtype, 41, cache=cap)
    ks = [i * cap for i in range(len(kl) + 1)]
    for t in (k, v):
        for i, n in enumerate(kl):
            t[ks[i] + n:ks[i + 1]] = float("nan")
        t[ks[-1]:] = float("inf")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    b = None
    if bias:
        b = (torch.randn(12, H, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True), packed.relative_buckets(12, 50, True, "cuda"))
        leaves.append(b[0])
    args = starts(ql).cuda(), torch.tensor(ks, dtype=torch.int32).cuda()
    run = lambda: packed.packed_attention(q, k, v, *args, k_len=torch.tensor(kl, dtype=torch.int32).cuda(), causal=causal, bias=b,
                                          max_q=max(ql), max_k=max(kl))
    o = run()
    grads = torch.autograd.grad(o, leaves, do)
    k, v = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)).detach() for t in (k, v))
    want = attn_ref(q, k, v, ql, starts(ql).tolist(), kl, ks, causal, d ** -0.5, *(b or (None, None)), do=do)
    for n, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[n], n)
    k, v = leaves[1:3]
    o2 = run()
    assert all(torch.equal(x, y) for x, y in zip((o, *grads), (o2, *torch.autograd.grad(o2, leaves, do)))), "not the same twice"


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
        return L.ait_packed_attn_fwd(ctypes.byref(p), qptr, qrow, qhead, *(4096, 128, 64) * 2, 4096, 256, 64, None, None, None, 0, None)

    def bwd(ws=4096, n=1 << 30, lse=4096, **kw):
        p = _lib.PackedAttn(**{**base, **kw})
        return L.ait_packed_attn_bwd(ctypes.byref(p), *(4096, 256, 64), *(4096, 128, 64) * 2, *(4096, 256, 64), None, *(4096, 256, 64), lse, *(4096, 256, 64),
                                     *(4096, 128, 64) * 2, None, ws, n, None)
    EINVAL, EWORKSPACE, EUNSUPPORTED = -1, -2, -4
    for f in (fwd, bwd):
        for kw in (dict(heads=0), dict(kv_heads=3), dict(n_seq=-1), dict(total_q=-1), dict(d=0), dict(dtype=2), dict(cu_q=None), dict(cu_k=None),
                   dict(max_q=-1), dict(scale=float("nan")), dict(bias_table=4096), dict(bias_table=4096, bucket_of=4096, n_buckets=0)):
            assert f(**kw) == EINVAL, kw
        for kw in (dict(d=136), dict(d=12), dict(n_seq=1 << 27), dict(bias_table=4096, bucket_of=4096, n_buckets=513), dict(total_q=2 ** 30),
                   dict(bias_table=4096, bucket_of=4096, n_buckets=4, max_distance=2049)):
            assert f(**kw) == EUNSUPPORTED, kw
        assert f(n_seq=0) == 0
    assert fwd(qptr=None) == EINVAL and fwd(qptr=4100) == EUNSUPPORTED and fwd(qrow=255) == EUNSUPPORTED and fwd(qhead=65) == EUNSUPPORTED
    assert fwd(qrow=1 << 24) == EUNSUPPORTED
    assert bwd(lse=None) == EINVAL and bwd(ws=None) == EWORKSPACE and bwd(n=4 * 5 * 4 - 1) == EWORKSPACE
    assert L.ait_packed_attn_fwd(None, *(None, 0, 0) * 4, None, None, None, 0, None) == EINVAL
    # a few tokens over a long key axis are cut along it: a workspace is asked for, and a small one refused
    p = dict(n_seq=2, total_q=2, total_k=20000, max_q=1, max_k=10000)
    need = L.ait_packed_attn_fwd_workspace_bytes(ctypes.byref(_lib.PackedAttn(**{**base, **p})))
    assert need > 0 and fwd(**p) == EWORKSPACE
    # sizes of nothing are sizes too
    for kw in (dict(n_seq=0), dict(n_seq=0, total_q=0, total_k=0), dict(total_q=0), dict(total_k=0), dict(total_q=1, max_q=1, total_k=0)):
        for f in (L.ait_packed_attn_fwd_workspace_bytes, L.ait_packed_attn_bwd_workspace_bytes):
            assert f(ctypes.byref(_lib.PackedAttn(**{**base, **kw}))) < 1 << 20
    assert L.ait_packed_attn_fwd_workspace_bytes(None) == 0 and L.ait_packed_attn_bwd_workspace_bytes(None) == 0
    assert L.ait_gated_norm_bwd_workspace_bytes(None) == 0
    assert L.ait_gated_norm_bwd_workspace_bytes(ctypes.byref(_lib.GatedNorm(w_post=4096, w_pre=4096, rows=0, width=8))) == 0


# ------------------------------------------------------------------------------------------
# gated norm: reference and bounds
# ------------------------------------------------------------------------------------------
def norm_ref(x, f, post, pre, post_b, pre_b, gate, scale, layer, eps, cu, dy, dh):
    """[(value, bound)] of y, h, dx, df, post, post_b, pre, pre_b, gate, scale gradients in 64 bits (None where there is none);
    rows of no sequence are not part of it.  Sums of a row are trees of at most 40 terms' depth (32 values a lane, 6 steps in a
    wave, 8 waves), columns' are as deep as there are rows."""
    ux, uf, e1 = torch.finfo(x.dtype).eps / 2, torch.finfo(f.dtype).eps / 2, 2.0 ** -24
    c = lambda t: None if t is None else t.detach().cpu().to(F8)
    x, f, post, pre, post_b, pre_b, gate, scale, dy, dh = (c(t) for t in (x, f, post, pre, post_b, pre_b, gate, scale, dy, dh))
    n = x.shape[0] if cu is None else int(cu[-1])
    x, f, dy, dh = x[:n], f[:n], dy[:n], dh[:n]
    mean = lambda t: t.mean(1, keepdim=True)
    seq = None if cu is None else torch.repeat_interleave(torch.arange(len(cu) - 1), torch.tensor([int(b - a) for a, b in zip(cu[:-1], cu[1:])]))
    G = torch.ones_like(x) if gate is None else gate if cu is None else gate[seq]
    S = torch.ones(x.shape[1], dtype=F8) if scale is None else scale
    D = 48 * e1

    def hat(t, et):
        tc = t - mean(t) if layer else t
        r = (mean(tc * tc) + eps) ** -0.5
        ec = et + (mean(et) + D * mean(t.abs()) if layer else 0) + e1 * t.abs()
        th = tc * r
        rr = mean(th.abs() * r * ec) * 1.01 + D                      # relative error of r
        return th, r, r * ec + th.abs() * rr * 1.01 + e1 * th.abs(), rr

    def back(d, th, eth, r, rr, ed):
        s1, s2 = mean(d * th), (mean(d) if layer else torch.zeros_like(mean(d)))
        es1 = mean(d.abs() * eth + ed * th.abs()) * 1.01 + D * mean((d * th).abs())
        es2 = (mean(ed) + D * mean(d.abs())) if layer else 0
        out = r * (d - s2 - th * s1)
        return out, r * (ed + 4 * e1 * (d.abs() + s2.abs() + (th * s1).abs()) + es2 + th.abs() * es1 + eth * s1.abs()) * 1.01 + out.abs() * rr * 1.01

    zero = torch.zeros_like(x)
    fh, fr, efh, frr = hat(f, zero)
    b = 0 if post_b is None else post_b
    m = fh * post + b
    em = efh * post.abs() + 4 * e1 * ((fh * post).abs() + (0 if post_b is None else post_b.abs()))
    sg = S * G
    y = x + sg * m
    ey = sg.abs() * em + 6 * e1 * (x.abs() + (sg * m).abs())
    yh, yr, eyh, yrr = hat(y, ey)
    h = yh * pre + (0 if pre_b is None else pre_b)
    eh = eyh * pre.abs() + 4 * e1 * ((yh * pre).abs() + (0 if pre_b is None else pre_b.abs()))
    rnd = lambda t, e, u: (t, e + u * (t.abs() + e))
    d = dh * pre
    bk, ebk = back(d, yh, eyh, yr, yrr, e1 * d.abs())
    t = dy + bk
    et = ebk + 2 * e1 * (dy.abs() + bk.abs())
    dm, edm = t * sg, sg.abs() * et + 4 * e1 * (t * sg).abs()
    df, edf = back(dm * post, fh, efh, fr, frr, edm * post.abs() + e1 * (dm * post).abs())
    N = (n + 80) * e1
    col = lambda v, e: (v.sum(0), (e + N * v.abs()).sum(0))
    out = dict(y=rnd(y, ey, ux), h=rnd(h, eh, uf), x=rnd(t, et, ux), f=rnd(df, edf, uf),
               post=col(dm * fh, edm * fh.abs() + dm.abs() * efh), pre=col(dh * yh, dh.abs() * eyh))
    if post_b is not None:
        out["post_b"] = col(dm, edm)
    if pre_b is not None:
        out["pre_b"] = col(dh, 0 * dh)
    k = t * G * m
    if scale is not None:
        out["scale"] = col(k, (et * m.abs() + t.abs() * em) * G.abs() + 4 * e1 * k.abs())
    if gate is not None:
        k = t * S * m
        ek = (et * m.abs() + t.abs() * em) * S.abs() + 4 * e1 * k.abs()
        if cu is not None:
            z = torch.zeros(gate.shape, dtype=F8)
            k, ek = z.index_add(0, seq, k), z.index_add(0, seq, ek + N * k.abs())
        out["gate"] = rnd(k, ek, uf)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("rows,width,kind,gate,scale,odd", [
    (1, 8, "rms", "row", True, False), (37, 512, "layer", "none", True, False), (300, 512, "rms", "sequence", True, False), (5, 17, "layer", "row", False, False),
    (64, 513, "layer", "sequence", True, False), (130, 1024, "rms", "row", True, True), (9, 2048, "layer", "sequence", False, False),
    (21, 4096, "rms", "sequence", True, True), (17, 8192, "layer", "row", True, False), (600, 100, "layer", "sequence", True, False), (3, 5120, "rms", "none", False, False),
    (2100, 40, "layer", "sequence", True, True), (5, 1, "rms", "row", True, False), (0, 64, "layer", "sequence", True, False), (30, 1536, "rms", "row", True, False),
    (11, 2600, "layer", "none", True, True), (9, 6144, "layer", "row", True, False), (40, 5120, "layer", "sequence", True, False)])
def test_gated_norm(types, rows, width, kind, gate, scale, odd):
    xt, ft = (getattr(torch, t) for t in types)
    g = torch.Generator().manual_seed(rows + width)
    r = lambda *s: torch.randn(*s, generator=g)
    def rowed(t, dt):          # odd: rows of a wider matrix
        if not odd:
            return t.to(dt).cuda()
        w = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=dt, device="cuda")
        w[:, 8:8 + t.shape[1]] = t.to(dt)
        return w[:, 8:8 + t.shape[1]]
    x, f = rowed(r(rows, width) * 2, xt), rowed(r(rows, width) + 0.5, ft)
    cu, n = None, rows
    if gate == "sequence":
        cut = [0, rows // 3, rows // 3, rows // 3 + 1 if rows > 3 else rows // 3, rows // 2, rows - rows // 10]
        cu, n = torch.tensor(cut, dtype=torch.int32).cuda(), cut[-1]
        x[n:], f[n:] = float("nan"), float("inf")
    gt = None if gate == "none" else rowed(torch.sigmoid(r(rows if gate == "row" else 5, width)), ft)
    par = {k: (1 if k in ("post", "pre") else 0.2) + 0.3 * r(width).cuda() for k in ("post", "pre", "scale", "post_b", "pre_b")}
    if not scale:
        par["scale"] = None
    if kind == "rms":
        par["post_b"] = par["pre_b"] = None
    leaves = {k: t.detach().requires_grad_(True) for k, t in dict(x=x, f=f, gate=gt, **par).items() if t is not None}
    L = leaves.get
    dy, dh = rowed(r(rows, width), xt), rowed(r(rows, width), ft)
    y, h = packed.gated_norm(L("x"), L("f"), post_weight=L("post"), pre_weight=L("pre"), post_bias=L("post_b"), pre_bias=L("pre_b"), gate=L("gate"),
                             scale=L("scale"), kind=kind, eps=1e-5, cu_seqlens=cu)
    names = list(leaves)
    got = dict(zip(names, torch.autograd.grad([y, h], [leaves[k] for k in names], [dy, dh])), y=y, h=h)
    want = norm_ref(x, f, par["post"], par["pre"], par["post_b"], par["pre_b"], gt, par["scale"], kind == "layer", 1e-5,
                    None if cu is None else cu.tolist(), dy, dh)
    assert set(want) == set(got)
    for k, w in want.items():
        t = got[k]
        if k in ("x", "f", "y", "h"):
            assert bool((t[n:] == 0).all()), k + ": rows behind the last sequence"
            t = t[:n]
        within(t, w, k)


def test_gated_norm_refuses_what_it_does_not_take():
    t = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)
    good = dict(x=t(6, 32), f=t(6, 32), post_weight=t(32), pre_weight=t(32))

    def call(**kw):
        a = {**good, **kw}
        return packed.gated_norm(a.pop("x"), a.pop("f"), **a)
    with pytest.raises(_lib.AitHipError, match="no CPU fallback"):
        call()
    cu = starts([2, 4])
    for change in (dict(x=t(6, 31)), dict(x=t(6, 32, dt=torch.float16), f=t(6, 32, dt=torch.float16)), dict(x=t(6, 32, dt=torch.bfloat16)),
                   dict(post_weight=t(31)), dict(pre_weight=None), dict(scale=t(6, 32)), dict(gate=t(5, 32)), dict(gate=t(6, 32, dt=torch.bfloat16)),
                   dict(cu_seqlens=cu), dict(gate=t(6, 32), cu_seqlens=cu), dict(gate=t(2, 32), cu_seqlens=cu.long()), dict(post_bias=t(32).half()),
                   dict(x=t(6, 8200), f=t(6, 8200), post_weight=t(8200), pre_weight=t(8200)), dict(x=t(2, 3, 32), f=t(2, 3, 32), gate=t(2, 32), cu_seqlens=cu),
                   dict(x=t(2, 3, 32), f=t(2, 3, 32), gate=t(6, 32))):
        with pytest.raises(_lib.AitHipError):
            call(**change)
            pytest.fail("taken: %s" % list(change))
    with pytest.raises(ValueError):
        call(kind="batch")
    L = _lib.lib()
    base = dict(x=4096, f=4096, w_post=4096, w_pre=4096, x_row=32, f_row=32, rows=6, width=32, dtype_x=0, dtype_f=0, eps=1e-6)
    fwd = lambda y=4096, yr=32, **kw: L.ait_gated_norm_fwd(ctypes.byref(_lib.GatedNorm(**{**base, **kw})), y, yr, 4096, 32, None, None)
    bwd = lambda ws=4096, n=1 << 30, dg=None, **kw: L.ait_gated_norm_bwd(
        ctypes.byref(_lib.GatedNorm(**{**base, **kw})), 4096, *(4096, 32) * 4, dg, 32, 4096, 4096, None, None, None, ws, n, None)
    for f in (fwd, bwd):
        for kw in (dict(rows=-1), dict(width=0), dict(dtype_x=2), dict(dtype_f=-1), dict(w_post=None), dict(w_pre=None), dict(x=None), dict(f=None),
                   dict(eps=-1.0), dict(cu_seqlens=4096), dict(x_row=-1), dict(n_seq=-1)):
            assert f(**kw) == -1, kw
        for kw in (dict(width=8193), dict(dtype_x=1, dtype_f=0), dict(rows=2 ** 31 - 4096)):
            assert f(**kw) == -4, kw
    assert fwd(y=None) == -1 and fwd(yr=31) == -1 and fwd(rows=1 << 27) == -4
    assert bwd(ws=None) == -2 and bwd(n=64) == -2 and bwd(scale=4096) == -1 and bwd(gate=4096, gate_row=32) == -1


# ------------------------------------------------------------------------------------------
# what calls may do
# ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_key_has_no_gradient_of_its_score(dtype):
    ql, kl = [3, 0, 70, 1], [1, 1, 1, 0]
    q, k, v, do = make(ql, kl, 4, 2, 96, dtype, 3)
    table, of = torch.randn(8, 4).cuda().requires_grad_(True), packed.relative_buckets(8, 20, True, "cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)] + [table]
    o = packed.packed_attention(q, k, v, starts(ql).cuda(), starts(kl).cuda(), bias=(table, of))
    dq, dk, dv, dt = torch.autograd.grad(o, leaves, do)
    assert all(bool((t == 0).all()) for t in (dq, dk, dt))
    want = attn_ref(q, k, v, ql, starts(ql).tolist(), kl, starts(kl).tolist(), False, 96 ** -0.5, table, of, do)
    within(o, want["o"], "o")
    within(dv, want["dv"], "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_any_scale(scale):
    lens = [70, 130]
    q, k, v, do = make(lens, lens, 2, 1, 64, torch.float32, 5)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cu = starts(lens)
    o = packed.packed_attention(q, k, v, cu.cuda(), causal=True, scale=scale)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), True, scale, do=do)
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))):
        within(t, want[n], n)


@pytest.mark.gpu
def test_many_short_sequences():
    """more sequences than one look at 64 starts, and than two"""
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 4, (4300,), generator=g).tolist()
    q, k, v, do = make(lens, lens, 1, 1, 16, torch.float32, 9)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cu = starts(lens)
    o = packed.packed_attention(q, k, v, cu.cuda(), causal=True, max_q=3, max_k=3)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), True, 0.25, do=do)
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))):
        within(t, want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["heads first", "one key head for all", "odd rows", "unaligned", "backwards gradient"])
def test_layouts(layout):
    lens, dt = [37, 90], torch.bfloat16
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    n, H, d = sum(lens), 4, 64
    q, k, v, do = r(n, H, d), r(n, H, d), r(n, H, d), r(n, H, d)
    if layout == "heads first":
        q, k, v, do = (t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v, do))
    if layout == "one key head for all":
        k, v = k[:, :1].expand(n, H, d), v[:, :1].expand(n, H, d)
    if layout == "odd rows":
        q, k, v = (torch.cat([t.reshape(n, -1), t.reshape(n, -1)[:, :3]], 1)[:, :H * d].view(n, H, d) for t in (q, k, v))
    if layout == "unaligned":
        q, k, v = (torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(n, H, d) for t in (q, k, v))
    if layout == "backwards gradient":
        do = do.flip(2)[:, :, ::2].repeat_interleave(2, 2)[..., :d].transpose(0, 2).contiguous().transpose(0, 2)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    cu = starts(lens)
    o = packed.packed_attention(*leaves, cu.cuda(), causal=True)
    want = attn_ref(q, k, v, lens, cu.tolist(), lens, cu.tolist(), True, d ** -0.5, do=do)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do))):
        within(t, want[name], name)


@pytest.mark.gpu
def test_offsets_past_four_gibibytes():
    """a cache of 2.2 million rows: a sequence far behind the start, and one that is itself longer than 32-bit offsets"""
    rows, Hk, d, dt = 2200000, 8, 128, torch.bfloat16
    k, v = torch.zeros(rows, Hk, d, dtype=dt, device="cuda"), torch.zeros(rows, Hk, d, dtype=dt, device="cuda")
    g = torch.Generator().manual_seed(4)
    k[-200:], v[-200:] = torch.randn(200, Hk, d, generator=g).to(dt).cuda(), torch.randn(200, Hk, d, generator=g).to(dt).cuda()
    q = torch.randn(2, Hk, d, generator=g).to(dt).cuda()
    cu = torch.tensor([0, rows - 200, rows], dtype=torch.int32).cuda()
    o = packed.packed_attention(q, k, v, starts([1, 1]).cuda(), cu, k_len=torch.tensor([3, 200], dtype=torch.int32).cuda(), causal=True, max_q=1, max_k=200)
    want = attn_ref(q, k[-200:], v[-200:], [0, 1], [0, 1], [0, 200], [0, 0], True, d ** -0.5)["o"]
    within(o[1], tuple(t[1] for t in want), "o")
    assert bool((o[0] == 0).all())
    # all keys before the last 200 are zero, and so are their values: they only add exp(-top) each to the sums
    q = q[:1] * 4
    o = packed.packed_attention(q, k, v, starts([1]).cuda(), torch.tensor([0, rows], dtype=torch.int32).cuda(), causal=True, max_q=1, max_k=rows)
    s = torch.einsum("hd,khd->hk", q[0].cpu().to(F8), k[-200:].cpu().to(F8)) * d ** -0.5
    p = torch.exp(s - s.amax(1, keepdim=True))
    p = p / (p.sum(1, keepdim=True) + (rows - 200) * torch.exp(-s.amax(1, keepdim=True)))
    vv = v[-200:].cpu().to(F8).permute(1, 0, 2)
    ref, size = torch.matmul(p[:, None], vv)[:, 0], torch.matmul(p[:, None], vv.abs())[:, 0]
    # u for a probability, u for the result; 2^-11 for a sum of 2.2 million equal terms, 34000 a lane at worst
    within(o[0], (ref, size * (2 ** -8 + 2 ** -11) + 2 ** -8 * ref.abs()), "o")


@pytest.mark.gpu
def test_a_given_output_keeps_its_other_rows():
    lens = [20, 45]
    q, k, v, _ = make(lens, lens, 2, 2, 64, torch.bfloat16, 6)
    cu = starts(lens).cuda()
    out = torch.full((q.shape[0], 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    p, keep = ops.packed_attn_desc(q, k, v, cu, cu, causal=True)
    got, _, _ = ops.packed_attn_fwd(p, q, k, v, out=out[:, 1:3])
    assert got.data_ptr() == out[:, 1:3].data_ptr()
    assert torch.equal(got[:65], packed.packed_attention(q, k, v, cu, causal=True)[:65])
    assert bool((out[65:] == 7).all()) and bool((out[:, 0] == 7).all()) and bool((out[:, 3] == 7).all())
    for bad in (out[:, :2].float(), out[:-1, :2], out[:, :1].expand(-1, 2, -1), out[:, 1:3, :].transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(_lib.AitHipError):
            ops.packed_attn_fwd(p, q, k, v, out=bad)
    empty = packed.packed_attention(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert empty.shape == (0, 2, 64)
    none = packed.packed_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert bool((none == 0).all())


def _step(x, w, cu, table, of):
    """a training step's operators on packed rows, everything a gradient flows to returned"""
    q, k, v = (x @ w[i] for i in range(3))
    n, H = x.shape[0], 2
    o = packed.packed_attention(q.view(n, H, -1), k.view(n, H, -1), v.view(n, H, -1), cu, causal=True, bias=(table, of))
    y, h = packed.gated_norm(x, o.reshape(n, -1), post_weight=w[3, 0], pre_weight=w[3, 1], scale=w[3, 2], kind="rms")
    return [y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, w, table], [y.detach() * 0.5, h.detach()])]


@pytest.mark.gpu
def test_streams_threads_and_graphs():
    import threading
    lens = [70, 1, 200]
    cu = starts(lens).cuda()
    g = torch.Generator().manual_seed(1)
    of = packed.relative_buckets(16, 60, False, "cuda")
    x, w, t = (torch.randn(*s, generator=g).cuda().mul_(f).requires_grad_(True) for s, f in (((sum(lens), 64), 1.0), ((4, 64, 64), 0.2), ((16, 2), 1.0)))
    want = _step(x, w, cu, t, of)
    # two streams at once, and a thread each
    got = {}

    def work(i):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(st):
            got[i] = [_step(x, w, cu, t, of) for _ in range(3)][-1]
        st.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [th.start() for th in threads]
    [th.join() for th in threads]
    assert len(got) == 3
    for r in got.values():
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    # forward and backward in a graph, replayed on other values between eager work
    static = [a.detach().clone().requires_grad_(True) for a in (x, w, t)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(static[0], static[1], cu, static[2], of)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _step(static[0], static[1], cu, static[2], of)))
    for i in range(4):
        new = [a.detach() * (1 + 0.1 * i) for a in (x, w, t)]
        with torch.no_grad():
            for s, a in zip(static, new):
                s.copy_(a)
        eager = _step(*[a.clone().requires_grad_(True) for a in new[:2]], cu, new[2].clone().requires_grad_(True), of)
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), "replay %d" % i


@pytest.mark.gpu
def test_new_tokens_in_a_graph_as_the_caches_grow():
    """lengths are read on the device: one captured call serves every step"""
    cap, B, H, Hk, d = 700, 3, 8, 2, 64
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(B * cap, Hk, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(B, H, d, generator=g).to(torch.bfloat16).cuda()
    cq, ck = starts([1] * B).cuda(), starts([cap] * B).cuda()
    kl = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    call = lambda: packed.packed_attention(q, k, v, cq, ck, k_len=kl, causal=True, max_q=1, max_k=cap)
    with torch.no_grad():
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for lens in ([1, 5, 0], [64, 65, 63], [700, 1, 300], [699, 128, 129]):
            kl.copy_(torch.tensor(lens, dtype=torch.int32))
            graph.replay()
            want = attn_ref(q, k, v, [1] * B, [0, 1, 2], lens, ck.tolist(), True, d ** -0.5)
            within(out, want["o"], str(lens))


def _norm64(t, w, layer):
    t = t - t.mean(1, keepdim=True) if layer else t
    return t * (t.pow(2).mean(1, keepdim=True) + 1e-6) ** -0.5 * w


@pytest.mark.gpu
def test_a_block_of_them_together():
    """norm - projections - attention with a bias - projection - gated norm, twice over, against the same in 64 bits"""
    lens, W, H, Hk, d = [50, 3, 81], 96, 6, 2, 16
    n = sum(lens)
    g = torch.Generator().manual_seed(12)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F8)
    par = dict(x=r(n, W), f=r(n, W), wq=r(2, W, H * d) * W ** -0.5, wk=r(2, W, Hk * d) * W ** -0.5, wv=r(2, W, Hk * d) * W ** -0.5,
               wo=r(2, H * d, W) * (H * d) ** -0.5, table=r(8, H), post=1 + 0.1 * r(3, W), pre=1 + 0.1 * r(3, W), gate=torch.sigmoid(r(len(lens), W)),
               scale=0.5 + 0.1 * r(W))
    cu, of = starts(lens), packed.relative_buckets(8, 24, False)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))

    def model(p, norm, attend, of, cu):
        y, h = norm(p["x"], p["f"], p, 0)
        for i in range(2):
            q, k, v = (h @ p[m][i] for m in ("wq", "wk", "wv"))
            o = attend(q.view(n, H, d), k.view(n, Hk, d), v.view(n, Hk, d), p["table"], of, cu)
            y, h = norm(y, o.reshape(n, H * d) @ p["wo"][i], p, i + 1)
        return (y * h).sum() / n + h.pow(2).sum() / n

    def norm64(x, f, p, i):
        y = x + p["scale"] * p["gate"][seq] * _norm64(f, p["post"][i], True)
        return y, _norm64(y, p["pre"][i], True)

    def attend64(q, k, v, table, of, cu):
        out = []
        m = of.numel() // 2
        for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
            rel = torch.arange(b - a)[None] - torch.arange(b - a)[:, None]
            s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(H // Hk, 1)) * d ** -0.5 + table[of.long()[rel.clamp(-m, m) + m]].permute(2, 0, 1)
            out.append(torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(rel > 0, -math.inf), 2), v[a:b].repeat_interleave(H // Hk, 1)))
        return torch.cat(out)

    def norm_hip(x, f, p, i):
        return packed.gated_norm(x, f, post_weight=p["post"][i], pre_weight=p["pre"][i], gate=p["gate"], scale=p["scale"], kind="layer", cu_seqlens=cu_d)
    ref = {m: t.clone().requires_grad_(True) for m, t in par.items()}
    loss = model(ref, norm64, attend64, of, cu)
    want = torch.autograd.grad(loss, list(ref.values()))
    cu_d = cu.cuda()
    hip = {m: t.float().cuda().requires_grad_(True) for m, t in par.items()}
    got_loss = model(hip, norm_hip, lambda q, k, v, table, of, cu: packed.packed_attention(q, k, v, cu, causal=True, bias=(table, of)), of.cuda(), cu_d)
    got = torch.autograd.grad(got_loss, list(hip.values()))
    # f32 throughout: every stage (five norms' worth of rows, six products of 96 terms, two softmaxes, and their backwards) adds at
    # most about 16 units of 2^-24, in random directions over some 30 stages, and a norm's 1 / deviation amplifies by up to 4
    tol = 4 * 16 * 30 ** 0.5 * 2.0 ** -24
    assert abs(float(got_loss) - float(loss)) < tol * abs(float(loss))
    for m, a, b in zip(par, got, want):
        assert float((a.cpu().to(F8) - b).norm()) < tol * float(b.norm()), m


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["attention", "norm"])
def test_gradients_against_differences(what):
    lens = [40, 75]
    cu = starts(lens).cuda()
    g = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    n = sum(lens)
    if what == "attention":
        of = packed.relative_buckets(8, 30, True, "cuda")
        leaves = [r(n, 4, 32), r(n, 2, 32), r(n, 2, 32), r(8, 4)]
        f = lambda a: [packed.packed_attention(a[0], a[1], a[2], cu, causal=True, bias=(a[3], of))]
        weight = [r(n, 4, 32)]
    else:
        leaves = [r(n, 72), r(n, 72), 1 + 0.2 * r(72), 1 + 0.2 * r(72), torch.sigmoid(r(2, 72)), r(72), 0.3 * r(72)]
        f = lambda a: list(packed.gated_norm(a[0], a[1], post_weight=a[2], pre_weight=a[3], gate=a[4], scale=a[5], post_bias=a[6], kind="layer", cu_seqlens=cu))
        weight = [r(n, 72), r(n, 72)]
    loss = lambda a: float(sum((o.double() * w.double()).sum() for o, w in zip(f(a), weight)))
    at = [t.clone().requires_grad_(True) for t in leaves]
    outs = f(at)
    grads = torch.autograd.grad(outs, at, weight)
    noise = 2.0 ** -20 * float(sum((o.double() * w.double()).pow(2).sum() for o, w in zip(outs, weight))) ** 0.5      # of a sum of values off by 2^-20
    for i, t in enumerate(leaves):
        d = r(*t.shape)
        slope = lambda e: (loss(leaves[:i] + [t + e * d] + leaves[i + 1:]) - loss(leaves[:i] + [t - e * d] + leaves[i + 1:])) / (2 * e)
        e = 2.0 ** -7
        near, far = slope(e), slope(2 * e)
        # the steps' error falls by four from 2 e to e: what is left at e is a third of what they differ by
        assert abs(float((grads[i].double() * d.double()).sum()) - near) <= abs(near - far) / 3 * 1.5 + 4 * noise / e, (what, i)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["attention", "norm"])
def test_a_graph_is_walked_twice_and_has_no_second_derivative(what):
    g = torch.Generator().manual_seed(77)
    t = lambda *s: torch.randn(*s, generator=g).cuda().requires_grad_(True)
    if what == "attention":
        leaves, cu = [t(20, 2, 16) for _ in range(3)], starts([9, 11]).cuda()
        out = (packed.packed_attention(*leaves, cu, causal=True),)
    else:
        leaves = [t(20, 24), t(20, 24), t(24), t(24)]
        out = packed.gated_norm(leaves[0], leaves[1], post_weight=leaves[2], pre_weight=leaves[3])
    up = [torch.randn(o.shape, generator=g).cuda() for o in out]
    first = torch.autograd.grad(out, leaves, up, retain_graph=True)
    second = torch.autograd.grad(out, leaves, up, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    up = [u.requires_grad_(True) for u in up]
    third = torch.autograd.grad(out, leaves, up, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, third))
    with pytest.raises(RuntimeError):
        third[0].sum().backward()


def test_arguments_that_are_no_tensors_are_refused():
    t = lambda *s: torch.zeros(*s, requires_grad=True)
    cu = starts([2, 3])
    table, of = t(8, 4), packed.relative_buckets(8, 20, True)
    for change in (dict(bias=([1.0], of)), dict(bias=(table, [0, 1, 2])), dict(bias=(table,)), dict(bias=table), dict(cu_q=[0, 2, 5]), dict(cu_k=(0, 5)),
                   dict(k_len=[2, 3]), dict(q=[1.0]), dict(v=None)):
        with pytest.raises(_lib.AitHipError):
            packed.packed_attention(**{**dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cu_q=cu), **change})
            pytest.fail("taken: %s" % list(change))
    for change in (dict(gate=[1.0]), dict(gate=1.0), dict(x=t(2, 5, 8), f=t(2, 5, 8), gate=2.0), dict(scale=1.0), dict(cu_seqlens=[0, 5], gate=t(1, 8)),
                   dict(x=t(2, 3, 0), f=t(2, 3, 0)), dict(x=None), dict(f=3.0), dict(post_weight=None), dict(pre_weight=1.0)):
        with pytest.raises(_lib.AitHipError):
            packed.gated_norm(**{**dict(x=t(5, 8), f=t(5, 8), post_weight=t(8), pre_weight=t(8)), **change})
            pytest.fail("taken: %s" % list(change))


def test_loads_in_asm_read_settled_scalars(tmp_path):
    """The tiles' loads are inline asm, which the compiler does not look into: a scalar that a vector instruction wrote must be five
    wait states old where they read it.  Read from the built objects, straight back from every such load."""
    import os
    import re
    import subprocess
    from ait_amd import build
    llvm, seen = "/opt/rocm/lib/llvm/bin/", 0
    build.build()
    for name in ("packed_attn", "packed_attn_bwd"):
        fat, co = str(tmp_path / "fat.bin"), str(tmp_path / "dev.co")
        subprocess.check_call([llvm + "llvm-objcopy", "--dump-section", ".hip_fatbin=" + fat, os.path.join(build.OBJ, name + ".o"), str(tmp_path / "copy.o")])
        subprocess.check_call([llvm + "clang-offload-bundler", "--type=o", "--unbundle", "--input=" + fat,
                               "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + co])
        text = subprocess.run([llvm + "llvm-objdump", "-d", "--no-show-raw-insn", co], stdout=subprocess.PIPE, text=True, check=True).stdout
        lines = [l.split("//")[0].strip() for l in text.splitlines() if l.startswith("\t")]
        for i, line in enumerate(lines):
            m = re.match(r"buffer_load_dword(?:x4)? \S+ s\[(\d+):(\d+)\],.* lds", line)
            if not m:
                continue
            seen += 1
            read, waited, j = set(range(int(m[1]), int(m[2]) + 1)), 0, i - 1
            while j >= 0 and waited < 5:
                w = re.match(r"v_\S+ (?:s\[(\d+):(\d+)\]|s(\d+))", lines[j])
                if w:
                    wrote = {int(w[3])} if w[3] else set(range(int(w[1]), int(w[2]) + 1))
                    assert not wrote & read, "%s: `%s` %d wait states before `%s`" % (name, lines[j], waited, line)
                n = re.match(r"s_nop (\d+)", lines[j])
                waited += int(n[1]) + 1 if n else 1
                j -= 1
    assert seen > 500


# ------------------------------------------------------------------------------------------
# scores so large that a row's logarithm of its sum no longer holds the sum
# ------------------------------------------------------------------------------------------
def absorbed_ref(q, k, v, ql, qs, kl, ks, causal, scale, table, bucket_of, do):
    """attn_ref for tables whose values are below 16 in size, -inf or below -1e8: a score is an f32 value, and next to a bias of -1e9
    its step is 64 or more, so that with products under 16 (asserted) the score IS the bias, whatever the product: such keys share
    a row's probability evenly where it sees no others, and have none where it does.  Bounds as in attn_ref, with no error of
    such a score."""
    u, f = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    table_type = table.dtype
    q, k, v, do, table = (t.detach().cpu().to(F8) for t in (q, k, v, do, table))
    bucket_of = bucket_of.cpu().long()
    H, Hk, d, m = q.shape[1], k.shape[1], q.shape[2], bucket_of.numel() // 2
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("dt", table))}
    for a, qa, b, kb in zip(ql, qs, kl, ks):
        if a <= 0 or b <= 0:
            continue
        rel = torch.arange(b)[None, :] - torch.arange(a)[:, None] - (b - a)
        at = bucket_of[rel.clamp(-m, m) + m]
        for h in range(H):
            c = h * Hk // H
            Q, K, V, G = q[qa:qa + a, h], k[kb:kb + b, c], v[kb:kb + b, c], do[qa:qa + a, h]
            t = table[:, h][at]
            assert bool(((t.abs() < 16) | (t < -1e8)).all()) and float((scale * Q.abs() @ K.abs().t()).max()) < 16
            down = t < -1e8
            s = torch.where(down, t, scale * Q @ K.t() + t)
            es = torch.where(down, 0.0, (d + 8) * f * (abs(scale) * Q.abs() @ K.abs().t()) + 12 * f * (s.abs() + t.abs()))
            s = s.masked_fill(rel > 0, -math.inf) if causal else s
            none = s.amax(1, keepdim=True) == -math.inf
            es = torch.where(torch.isfinite(s), es, 0.0)
            p = torch.softmax(torch.where(none, 0.0, s), 1) * ~none
            rp = es + es.amax(1, keepdim=True) + (2 * b + 16) * f
            O, dp = p @ V, G @ V.t()
            EO = (p * (rp + u)) @ V.abs() + (b + 8) * f * (p @ V.abs())
            delta = (G * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = p * ((d + 4) * f * (G.abs() @ V.abs().t()) + (G.abs() * EO).sum(1, keepdim=True) + (d + 4) * f * (G.abs() * O.abs()).sum(1, keepdim=True))
            eds = eds + ds.abs() * (rp + 4 * f) + p * rp * (G.abs() * EO).sum(1, keepdim=True)
            edr = eds + u * (ds.abs() + eds) + (a * H // Hk + b + 16) * f * ds.abs()
            for name, i, x, e in (("o", (slice(qa, qa + a), h), O, EO), ("dq", (slice(qa, qa + a), h), scale * ds @ K, abs(scale) * edr @ K.abs()),
                                  ("dk", (slice(kb, kb + b), c), scale * ds.t() @ Q, abs(scale) * edr.t() @ Q.abs()),
                                  ("dv", (slice(kb, kb + b), c), p.t() @ G, (p * (rp + u + (a * H // Hk + b + 16) * f)).t() @ G.abs())):
                out[name][0][i] += x
                out[name][1][i] += e
            out["dt"][0][:, h].index_add_(0, at.reshape(-1), ds.reshape(-1))
            out["dt"][1][:, h].index_add_(0, at.reshape(-1), (eds + (a * b) ** 0.5 * 8 * f * ds.abs()).reshape(-1))
    out["dt"][1] += 64 * f * out["dt"][0].abs()
    r = lambda n, x, e: (x, e + (torch.finfo(table_type).eps / 2 if n == "dt" else u) * (x.abs() + e))
    return {n: r(n, *xe) for n, xe in out.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-1e9, "lowest"])
@pytest.mark.parametrize("ql,kl,Hk,d,causal,max_q,max_k", [
    ([200, 1, 70], None, 2, 64, True, 200, 200), ([150, 30], None, 4, 128, True, 150, 150), ([33, 64, 2], None, 1, 40, False, 64, 64),
    ([5, 3], [900, 40], 4, 64, True, 5, 900), ([60], [700], 2, 128, False, 60, 700)])
def test_rows_that_see_only_buckets_far_down(dtype, low, ql, kl, Hk, d, causal, max_q, max_k):
    """heads whose tables hold a mask's value (and -inf) for all distances, the near ones, the far ones: rows that see nothing else
    still have their softmax, and the backward the same one as the forward -- in blocks near the diagonal and far from it, and
    with the key axis in parts"""
    kl, H = ql if kl is None else kl, 4
    q, k, v, do = make(ql, kl, H, Hk, d, dtype, 17)
    q, k = (q * 0.5).requires_grad_(True), (k * 0.5).requires_grad_(True)
    v.requires_grad_(True)
    value = torch.finfo(dtype).min if low == "lowest" else low
    table = torch.randn(10, H, generator=torch.Generator().manual_seed(2)).to(dtype)
    of = packed.relative_buckets(10, 20, not causal)
    far, ahead = int(of[0]), int(of[-1])
    table[:, 0] = value
    table[:, 1] = value
    table[far, 1] = 0.5                       # ... but the far ones behind
    table[[far, ahead], 2] = value            # only the far ones
    table[:3, 3], table[3:, 3] = -math.inf, value
    table = table.cuda().requires_grad_(True)
    cq, ck = starts(ql), starts(kl)
    o = packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=causal, bias=(table, of.cuda()), scale=0.1, max_q=max_q, max_k=max_k)
    grads = torch.autograd.grad(o, [q, k, v, table], do)
    want = absorbed_ref(q, k, v, ql, cq.tolist(), kl, ck.tolist(), causal, 0.1, table, of, do)
    for n, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [-1e3, -1e4, -1e6, 1e6, "highest"])
def test_probabilities_of_a_row_add_up_to_one(dtype, value):
    """whatever the bias that all of a head's keys have: with dO = 1 a sequence's dV adds up to the number of its rows.  A row's
    probabilities are off from their sum by the f32 roundings of 260 terms (2^-15 covers them), and each dV by its rounding"""
    lens, H, d = [260, 3], 2, 64
    q, k, v, do = make(lens, lens, H, H, d, dtype, 19)
    v.requires_grad_(True)
    do = torch.ones_like(do)
    if value == "highest":
        value = torch.finfo(dtype).max
    table, of = torch.full((8, H), value, dtype=dtype, device="cuda"), packed.relative_buckets(8, 20, False, "cuda")
    o = packed.packed_attention(q, k, v, starts(lens).cuda(), causal=True, bias=(table, of))
    dv, = torch.autograd.grad(o, [v], do)
    u = torch.finfo(dtype).eps / 2
    for s, n in zip(starts(lens).tolist(), lens):
        t = dv[s:s + n].double()
        # (bf16: a probability is rounded where it enters the product, and so is dV)
        assert bool(((t.sum(0) - n).abs() <= n * 2.0 ** -15 + (2 * u * n if dtype == torch.bfloat16 else u * n)).all()), float((t.sum(0) / n - 1).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [24, 36])
@pytest.mark.parametrize("ql,kl,d", [([70, 5], [130, 64], 64), ([3], [700], 128), ([600], [600], 128)])
def test_scores_of_any_size(dtype, power, ql, kl, d):
    """products of 2^power times 0, 1 or 2 (exact: one value of a head is not zero): the keys with the largest share a row evenly"""
    H, half = 2, 2.0 ** (power // 2)
    q, k, v, do = make(ql, kl, H, H, d, dtype, 29)
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        q.zero_(), k.zero_()
        q[:, :, 5] = half
        k[:, :, 5] = half * torch.randint(0, 3, k.shape[:2], generator=g).to(dtype).cuda()
    cq, ck = starts(ql), starts(kl)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), scale=1.0, max_q=max(ql), max_k=max(kl))
    dv, = torch.autograd.grad(o, [v], do)
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    vv, gg, kk = v.detach().cpu().to(F8), do.cpu().to(F8), k.detach().cpu().to(F8)[:, :, 5]
    for a, qa, b, kb in zip(ql, cq.tolist(), kl, ck.tolist()):
        for h in range(H):
            top = kk[kb:kb + b, h] == kk[kb:kb + b, h].max()
            p = (top / top.sum())[None].expand(a, b).to(F8)
            V, G = vv[kb:kb + b, h], gg[qa:qa + a, h]
            e = u + (2 * b + 16) * f
            within(o[qa:qa + a, h], (p @ V, 1.01 * e * (p @ V.abs()) + u * (p @ V).abs()), "o")
            within(dv[kb:kb + b, h], (p.t() @ G, 1.01 * (e + a * f) * (p.t() @ G.abs()) + u * (p.t() @ G).abs()), "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ql,kl,H,Hk,d,bias,max_k", [([70, 5], [2, 0], 4, 2, 64, True, 64), ([300, 90], [150, 70], 2, 1, 128, False, 150), ([1300], [600], 2, 1, 128, False, 600),
                                                     ([200], [33], 2, 2, 40, True, 33)])
def test_rows_that_see_no_key_may_hold_anything(dtype, ql, kl, H, Hk, d, bias, max_k):
    """the padding in front of a sequence with a causal mask: neither its queries nor its gradients enter those of the keys"""
    q, k, v, do = make(ql, kl, H, Hk, d, dtype, 43)
    cq, ck = starts(ql), starts(kl)
    want_q, want_do = q.clone(), do.clone()
    for a, n, m in zip(cq.tolist(), ql, kl):
        q[a:a + n - m], do[a:a + n - m] = float("nan"), float("inf")
        want_q[a:a + n - m], want_do[a:a + n - m] = 0, 0
    b = None
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    if bias:
        b = (torch.randn(12, H, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True), packed.relative_buckets(12, 50, False, "cuda"))
        leaves.append(b[0])
    o = packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=True, bias=b, max_q=max(ql), max_k=max_k)
    grads = torch.autograd.grad(o, leaves, do)
    want = attn_ref(want_q, k, v, ql, cq.tolist(), kl, ck.tolist(), True, d ** -0.5, *(b or (None, None)), do=want_do)
    for n, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *grads)):
        within(t, want[n], n)
    # ... and they are zeros next to a value that is none
    with torch.no_grad():
        v[max(0, kl[0] - 1)] = float("nan")
        o = packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=True, bias=b, max_q=max(ql), max_k=max_k)
    assert all(bool((o[a:a + n - m] == 0).all()) for a, n, m in zip(cq.tolist(), ql, kl))


def test_forward_mode_derivatives_are_refused():
    """a dual tensor requires no gradient: taken, its tangent would be lost without a word"""
    import torch.autograd.forward_ad as fwd_ad
    t = lambda *s: torch.zeros(*s)
    cu, table, of = starts([2, 3]), t(8, 4), packed.relative_buckets(8, 20, True)
    good = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cu_q=cu, bias=(table, of))
    norm = dict(x=t(5, 8), f=t(5, 8), post_weight=t(8), pre_weight=t(8), post_bias=t(8), pre_bias=t(8), gate=t(5, 8), scale=t(8))
    with fwd_ad.dual_level():
        dual = lambda x: fwd_ad.make_dual(x, torch.ones_like(x))
        for change in (dict(q=dual(good["q"])), dict(k=dual(good["k"])), dict(v=dual(good["v"])), dict(bias=(dual(table), of))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(_lib.AitHipError, match="forward-mode"):
                    packed.packed_attention(**{**good, **change})
        for n in norm:
            with pytest.raises(_lib.AitHipError, match="forward-mode"):
                packed.gated_norm(**{**norm, n: dual(norm[n])})
        with pytest.raises(_lib.AitHipError, match="no CPU fallback"):
            packed.packed_attention(**good)


def test_a_scale_with_a_gradient_is_refused():
    """the scale is a number: as a tensor that wants a gradient it would get none"""
    t = lambda *s: torch.zeros(*s)
    good = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cu_q=starts([2, 3]))
    for bad in (torch.tensor(0.5, requires_grad=True), torch.ones(3), "large"):
        with pytest.raises(_lib.AitHipError, match="scale"):
            packed.packed_attention(**good, scale=bad)
    for number in (0.5, 1, torch.tensor(0.5)):
        with pytest.raises(_lib.AitHipError, match="no CPU fallback"):
            packed.packed_attention(**good, scale=number)


# ------------------------------------------------------------------------------------------
# how exact bf16 attention is, by norms
# ------------------------------------------------------------------------------------------
def _norms64(q, k, v, do, ql, kl, causal, scale, table, of):
    """in 64 bits: o, dq, dk, dv, d table, and the d table of a backward whose delta comes from a rounded o (`once`), or from one
    that was formed of rounded probabilities too (`twice`)"""
    b16 = lambda t: t.to(torch.bfloat16).to(F8)
    q, k, v, do, table = (t.detach().cpu().to(F8) for t in (q, k, v, do, table))
    H, Hk, m = q.shape[1], k.shape[1], of.numel() // 2
    r = dict(o=torch.zeros_like(q), dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    r.update({n: torch.zeros_like(table) for n in ("dt", "once", "twice")})
    for a, qa, b, kb in zip(ql, starts(ql).tolist(), kl, starts(kl).tolist()):
        rel = torch.arange(b)[None, :] - torch.arange(a)[:, None] - (b - a)
        at = of.long()[rel.clamp(-m, m) + m]
        for h in range(H):
            c = h * Hk // H
            Q, K, V, G = q[qa:qa + a, h], k[kb:kb + b, c], v[kb:kb + b, c], do[qa:qa + a, h]
            s = scale * Q @ K.t() + table[:, h][at]
            s = s.masked_fill(rel > 0, -math.inf) if causal else s
            e = torch.exp(s - s.amax(1, keepdim=True))
            p = e / e.sum(1, keepdim=True)
            O, dp = p @ V, G @ V.t()
            r["o"][qa:qa + a, h] = O
            for name, o in (("dt", O), ("once", b16(O)), ("twice", b16(b16(e) @ V / e.sum(1, keepdim=True)))):
                ds = p * (dp - (G * o).sum(1, keepdim=True))
                r[name][:, h].index_add_(0, at.reshape(-1), ds.reshape(-1))
            ds = p * (dp - (G * O).sum(1, keepdim=True))
            r["dq"][qa:qa + a, h] = scale * ds @ K
            r["dk"][kb:kb + b, c] += scale * ds.t() @ Q
            r["dv"][kb:kb + b, c] += p.t() @ G
    return r


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,H,Hk,d,causal,few", [(LONG, None, 4, 1, 64, True, False), ([400], None, 2, 2, 128, False, False), (LONG, None, 4, 2, 40, True, False),
                                                      ([60], [1500], 2, 2, 128, False, True), ([5, 9], [700, 400], 8, 2, 72, True, True),
                                                      ([33, 40], None, 2, 1, 64, True, True)])
def test_how_exact_bf16_attention_is(ql, kl, H, Hk, d, causal, few):
    """A bf16 value's rounding is off by up to 2^-8 / m of it, m in 1 .. 2 its significand; over spread values that is
    2^-8 / sqrt(3 E[m^2]) = 0.0015 to 0.0017 of a tensor's norm, and a sum of products with one rounded factor is off by as much.  So
    what is rounded once is within 0.0019, what is the rounded sum of products with a rounded factor within 1.15 sqrt(2) 0.0017 =
    0.0027 of its norm.  What rounding took from o is kept for the backward: o and it together leave 2^-8 2^-8 of o and the f32 sums'
    errors, 2^-14 with room.  The table's gradient (here of an f32 table: no rounding of its own) must be nearer than a quarter
    of what losing that rest, in o or in the probabilities, would take it away."""
    kl = ql if kl is None else kl
    q, k, v, do = (t[:sum(n)] for t, n in zip(make(ql, kl, H, Hk, d, torch.bfloat16, 53), (ql, kl, kl, ql)))
    table = torch.randn(12, H, generator=torch.Generator().manual_seed(3)).cuda()
    of = packed.relative_buckets(12, 50, not causal)
    cq, ck = starts(ql).cuda(), starts(kl).cuda()
    scale = d ** -0.5
    want = _norms64(q, k, v, do, ql, kl, causal, scale, table, of)
    off = lambda t, n, ref=None: float((t.detach().cpu().to(F8) - want[n]).norm() / (want[n] if ref is None else ref).norm())
    hints = dict(max_q=max(ql), max_k=max(kl))
    with torch.no_grad():
        o = packed.packed_attention(q, k, v, cq, ck, causal=causal, bias=(table, of.cuda()), **hints)
    assert off(o, "o") < (0.0019 if few else 0.0027)
    p, keep = ops.packed_attn_desc(q, k, v, cq, ck, causal=causal, table=table, bucket_of=of.cuda(), **hints)
    o, lse, rest = ops.packed_attn_fwd(p, q, k, v, for_backward=True)
    assert off(o, "o") < 0.0019
    assert off(o.double() + rest.double(), "o") < 2.0 ** -14
    dq, dk, dv, dt = ops.packed_attn_bwd(p, q, k, v, o, rest, do, lse, want_table=True)
    for n, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert off(t, n) < 0.0027, n
    err = (dt.cpu().to(F8) - want["dt"]).norm()
    for n in ("once", "twice"):
        assert float(err) < 0.25 * float((want[n] - want["dt"]).norm()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("ql,kl,d,bias", [([70, 130], None, 40, False), ([70, 130], None, 64, True), ([70, 130], None, 128, False), ([5, 2], [900, 70], 64, True),
                                          ([3], [700], 128, False)])
def test_a_scale_of_any_sign_in_both_types(dtype, scale, ql, kl, d, bias):
    """with a bias, over the key axis in parts, at widths below the tiles'"""
    kl = ql if kl is None else kl
    q, k, v, do = make(ql, kl, 4, 2, d, dtype, 5)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    b = None
    if bias:
        b = (torch.randn(8, 4, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True), packed.relative_buckets(8, 30, False, "cuda"))
        leaves.append(b[0])
    cq, ck = starts(ql), starts(kl)
    call = lambda: packed.packed_attention(q, k, v, cq.cuda(), ck.cuda(), causal=True, scale=scale, bias=b, max_q=max(ql), max_k=max(kl))
    o = call()
    want = attn_ref(q, k, v, ql, cq.tolist(), kl, ck.tolist(), True, scale, *(b or (None, None)), do=do)
    for n, t in zip(("o", "dq", "dk", "dv", "dt"), (o, *torch.autograd.grad(o, leaves, do))):
        within(t, want[n], n)
    with torch.no_grad():
        within(call(), want["o"], "o without a gradient")


def test_scratch_of_the_kernels():
    """Bytes a lane that spill, read from the built objects.  Attention: none, but for queries with a bias in two waves of 128-wide
    bf16 heads.  The norm's backward: rows of ten and twelve waves with biases, rows of two blocks a lane (over 6144 values, or over
    4096 that take single loads)."""
    import os
    import re
    from ait_amd import build
    from test_abi import _kernel_scratch
    build.build()
    for name in ("packed_attn", "packed_attn_bwd"):
        kernels = _kernel_scratch(os.path.join(build.OBJ, name + ".o"))
        assert len(kernels) > 20
        for k, n in kernels.items():
            assert n <= (32 if "packed_bwd_q_kernelIDF16bLi128ELb1ELi2E" in k else 0), "%s: %d bytes of scratch a lane" % (k, n)
    kernels = _kernel_scratch(os.path.join(build.OBJ, "gated_norm.o"))
    seen = 0
    for k, n in kernels.items():
        m = re.search(r"gated_norm_(fwd|bwd)_kernelI(.*?)Li(\d+)ELi(\d)ELb(\d)E(?:Lb(\d)E)?", k)
        if not m:
            assert n == 0, k
            continue
        seen += 1
        waves, blocks, wide, biases = int(m[3]), int(m[4]), m[5] == "1", m[6] == "1"
        limit = 0 if m[1] == "fwd" else (204 if wide else 476) if blocks == 2 and biases else (36 if wide else 208) if blocks == 2 else 48 if waves >= 10 and biases else 0
        assert n <= limit, "%s: %d bytes of scratch a lane (limit %d)" % (k, n, limit)
    assert seen >= 60
