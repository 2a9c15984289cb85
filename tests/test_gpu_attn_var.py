"""Attention over packed rows (ops.attn_var) against its definition in 64 bits, forward and gradients, at the sizes and masks where it can
go wrong; bounds derived in attn_ref."""
import numpy as np
import pytest
import torch

from cikm2020_dmt_amd import _lib as L
from cikm2020_dmt_amd import ops
from tests import attn_ref as A

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _make(ql, kl, H, Hkv, dh, dtype, seed, std=1.0, gap=0):
    g = torch.Generator().manual_seed(seed)
    qo = np.concatenate([[0], np.cumsum(np.array(ql) + gap)])[:-1].tolist()
    ko = np.concatenate([[0], np.cumsum(np.array(kl) + gap)])[:-1].tolist()
    rq, rk = int(sum(ql) + gap * len(ql)), int(sum(kl) + gap * len(kl))
    n = lambda r, w, s=1.0: (torch.randn((r, w), generator=g) * s).to(dtype)  # noqa: E731
    return n(rq, H * dh, std), n(rk, Hkv * dh, std), n(rk, Hkv * dh), n(rq, H * dh), qo, ko


def _check(cuda, ql, kl, H, Hkv, dh, dtype=BF, seed=0, std=1.0, gap=0, slopes=None, docs=None, prefix=None, train=True, **kw):
    q, k, v, do, qo, ko = _make(ql, kl, H, Hkv, dh, dtype, seed, std, gap)
    sl = None if slopes is None else torch.tensor(slopes, dtype=F32)
    ref = A.attn_var(q, k, v, H, Hkv, ql, kl, qo, ko, slopes=sl, docs=docs, prefix=prefix, dout=do if train else None, **kw)
    seqs = ops.AttnSeqs(ql, kl, qo, ko, device=cuda)
    lv = [t.to(cuda).requires_grad_(train) for t in (q, k, v)] + ([sl.to(cuda).requires_grad_(train)] if sl is not None else [])
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).to(cuda)  # noqa: E731
    out, lse = ops.attn_var(*lv[:3], seqs, H, Hkv, slopes=lv[3] if sl is not None else None, want_lse=True,
                            docs=None if docs is None else tuple(map(i32, docs)), prefix=None if prefix is None else i32(prefix), **kw)
    A.close(out, ref["out"], ref["out_tol"], "out")
    A.close(lse, ref["lse"], ref["lse_tol"], "lse")
    if not train:
        return
    grads = torch.autograd.grad(out, lv, do.to(cuda))
    for t, n in zip(grads, ("dq", "dk", "dv", "dslope")):
        A.close(t, ref[n], ref[n + "_tol"], n)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dh", [16, 24, 40, 64, 80, 96, 128])
def test_head_sizes(cuda, dh, dtype):
    _check(cuda, [70, 1, 33], [70, 1, 33], 4, 2, dh, dtype, causal=True)
    _check(cuda, [5, 130], [67, 129], 2, 1, dh, dtype, slopes=[0.3, 0.02])


@pytest.mark.parametrize("dh", [4, 20, 100])
def test_head_sizes_of_fp32(cuda, dh):
    _check(cuda, [70, 1, 33], [70, 1, 33], 4, 4, dh, F32, causal=True, cap=3.0)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", [([1], [1]), ([1], [2]), ([2], [1]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [63, 64, 65]),
                                   ([127, 128, 129], [127, 128, 129]), ([1, 1, 3], [200, 64, 65]), ([200, 65], [7, 64]), ([0, 5, 0], [9, 0, 0]),
                                   ([0, 5, 4], [0, 5, 4]), ([257, 300], [257, 511])])
def test_lengths(cuda, ql, kl, causal):
    _check(cuda, ql, kl, 2, 2, 32, causal=causal)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (8, 1), (8, 2), (6, 3), (16, 16)])
def test_shared_heads(cuda, H, Hkv):
    _check(cuda, [40, 77], [90, 77], H, Hkv, 32, causal=True, slopes=[0.5 / (h + 1) for h in range(H)])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kw", [dict(cap=5.0), dict(cap=5.0, causal=True, slopes=[0.1, 0.0, 1.0, 0.01]), dict(slopes=[0.0, 2.0, -0.01, 0.3]),
                                dict(cap=0.01), dict(scale=0.5), dict(cap=30.0, scale=2.0, causal=True)])
def test_shaped_scores(cuda, kw, dtype):
    _check(cuda, [100, 37], [100, 90], 4, 2, 64, dtype, std=1.5, **kw)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("prefix", [[0, 0, 0], [1, 64, 10], [1000, 65, 130], [-5, 3, 63]])
def test_prefix(cuda, prefix, causal):
    pre = [min(max(x, 0), k) for x, k in zip(prefix, [150, 65, 200])]
    ql, kl = [150, 65, 70], [150, 65, 200]
    q, k, v, do, qo, ko = _make(ql, kl, 2, 1, 32, BF, 3)
    ref = A.attn_var(q, k, v, 2, 1, ql, kl, qo, ko, causal=causal, prefix=pre)
    out = ops.attn_var(q.to(cuda), k.to(cuda), v.to(cuda), ops.AttnSeqs(ql, kl, device=cuda), 2, 1, causal=causal,
                       prefix=torch.tensor(prefix, dtype=torch.int32, device=cuda))
    A.close(out, ref["out"], ref["out_tol"], "out")
    _check(cuda, ql, kl, 2, 1, 32, causal=causal, prefix=pre, seed=3)


def _docs(kind, ql, kl, seed):
    r = np.random.RandomState(seed)
    kd = [{"rising": lambda n: np.arange(n) // 37, "any": lambda n: r.randint(-3, 4, n), "own": lambda n: np.arange(n)}[kind](n) for n in kl]
    qd = [d[len(d) - n:] if n <= len(d) else np.concatenate([np.full(n - len(d), 99), d]) for n, d in zip(ql, kd)]
    return tuple(torch.as_tensor(np.concatenate(x), dtype=torch.int32) for x in (qd, kd))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (False, [70, 0, 5]), (True, [70, 0, 5])])
@pytest.mark.parametrize("kind", ["rising", "any", "own"])
def test_documents(cuda, kind, causal, prefix, dtype):
    """query ids 99 (rows before the first key) match no key: rows that see nothing"""
    ql, kl = [200, 90, 150], [200, 64, 150]
    _check(cuda, ql, kl, 2, 1, 32, dtype, causal=causal, prefix=prefix, docs=_docs(kind, ql, kl, 1))


def test_long_histories(cuda):
    _check(cuda, [1100], [1100], 2, 1, 80, causal=True, slopes=[0.01, 0.2])
    _check(cuda, [3, 600], [2500, 1300], 2, 2, 128, cap=8.0)


def test_rows_of_no_example_stay(cuda):
    """gaps between the examples: zeros in what autograd returns, untouched in buffers handed to the C entry"""
    _check(cuda, [40, 0, 65], [40, 0, 65], 2, 1, 32, gap=3, causal=True)
    q, k, v, do, qo, ko = (t.to(cuda) if isinstance(t, torch.Tensor) else t for t in _make([40, 65], [40, 65], 2, 1, 32, BF, 5, gap=3))
    seqs = ops.AttnSeqs([40, 65], None, qo, device=cuda)
    cfg = (2, 1, 0.2, 0.0, True, 65, 65)
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[0], 2), 7.0, device=cuda)
    lens = (seqs.q_lens, seqs.q_off, seqs.k_lens, seqs.k_off)
    d = ops._attn_var_desc(q, k, v, None, None, None, None, None, lens, out, lse, None, cfg)
    L.check(L.load().dmt_attn_var_fwd(d, ops.stream_ptr()))
    dq, dk, dv = torch.full_like(q, 7.0), torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    d.dout, d.do_rs, d.dQ, d.dq_rs, d.dK, d.dk_rs, d.dV, d.dv_rs = (do.data_ptr(), 64, dq.data_ptr(), 64, dk.data_ptr(), 32, dv.data_ptr(), 32)
    ws = torch.empty(int(L.load().dmt_attn_var_ws_bytes(d)), dtype=torch.uint8, device=cuda)
    d.ws, d.ws_bytes = ws.data_ptr(), ws.numel()
    L.check(L.load().dmt_attn_var_bwd(d, ops.stream_ptr()))
    torch.cuda.synchronize()
    gap = torch.ones(q.shape[0], dtype=torch.bool, device=cuda)
    for o, n in zip(qo, (40, 65)):
        gap[o:o + n] = False
    for t in (out, lse, dq, dk, dv):
        assert (t[gap] == 7.0).all() and not (t[~gap] == 7.0).all(1).any()
    del ws


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v", "kv"])
def test_masked_places_may_hold_anything(cuda, where, bad, dtype):
    """NaN / infinity in the last key of a causal history reaches the last row alone; in a document of its own it reaches nobody; rows of no
    example hold it too"""
    ql = [100, 150]
    q, k, v, do, qo, ko = _make(ql, ql, 2, 1, 32, dtype, 9, gap=2)
    last = [qo[0] + 99, qo[1] + 149]
    for r in last + [qo[0] + 100, qo[1] + 151]:
        if "k" in where:
            k[r] = bad
        if "v" in where:
            v[r] = bad
    q[qo[0] + 101], do[qo[1] + 150] = bad, bad
    do[last] = 0
    own = torch.zeros(q.shape[0], dtype=torch.int32)
    own[last] = 1
    for kw, docs, clean in ((dict(causal=True), None, last), (dict(), (torch.zeros_like(own), own), [])):
        seqs = ops.AttnSeqs(ql, None, qo, device=cuda)
        lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
        out = ops.attn_var(*lv, seqs, 2, 1, docs=None if docs is None else tuple(t.to(cuda) for t in docs), **kw)
        k0, v0 = k.clone(), v.clone()
        k0[~torch.isfinite(k0)], v0[~torch.isfinite(v0)] = 0, 0
        ref = A.attn_var(q, k0, v0, 2, 1, ql, ql, qo, ko, docs=docs, dout=do, **kw)
        keep = torch.ones(q.shape[0], dtype=torch.bool)
        keep[clean] = False
        A.close(out[keep.to(cuda)], ref["out"][keep], ref["out_tol"][keep], "out")
        if clean:
            continue                                   # (rows that see the value have gradients of their own)
        for t, n in zip(torch.autograd.grad(out, lv, do.to(cuda)), ("dq", "dk", "dv")):
            A.close(t[keep.to(cuda)], ref[n][keep], ref[n + "_tol"][keep], n)


def test_lowest_and_large_scores(cuda):
    """scores of 1e4 and more (one key takes all), and columns of the type's lowest value in V"""
    _check(cuda, [70], [70], 2, 1, 32, std=60.0, causal=True)
    q, k, v, do, qo, ko = _make([64], [64], 1, 1, 32, BF, 2)
    v[:, 0] = torch.finfo(BF).min
    ref = A.attn_var(q, k, v, 1, 1, [64], [64], qo, ko, causal=True)
    out = ops.attn_var(q.to(cuda), k.to(cuda), v.to(cuda), ops.AttnSeqs([64], device=cuda), 1, causal=True)
    A.close(out[:, 1:], ref["out"][:, 1:], ref["out_tol"][:, 1:], "out")
    assert (out[:, 0].float() < -3.3e38).all()


def test_strides_alignment_and_order(cuda):
    """column slices of a packed projection, examples in any order, an operand whose rows are not aligned"""
    H, Hkv, dh = 4, 2, 16
    ql, qo = [50, 70, 9], [79, 9, 0]
    g = torch.Generator().manual_seed(1)
    pk = torch.randn((129, (H + 2 * Hkv) * dh), generator=g).to(BF)
    do = torch.randn((129, H * dh), generator=g).to(BF)
    cut = lambda t: (t[:, :64], t[:, 64:96], t[:, 96:])  # noqa: E731
    ref = A.attn_var(*cut(pk), H, Hkv, ql, ql, qo, qo, causal=True, dout=do)
    x = pk.to(cuda).requires_grad_(True)
    seqs = ops.AttnSeqs(ql, None, qo, device=cuda)
    out = ops.attn_var(*cut(x), seqs, H, Hkv, causal=True)
    A.close(out, ref["out"], ref["out_tol"], "out")
    (dx,) = torch.autograd.grad(out, x, do.to(cuda))
    for t, n in zip(cut(dx), ("dq", "dk", "dv")):
        A.close(t, ref[n], ref[n + "_tol"], n)
    odd = torch.zeros((129, 65), dtype=BF, device=cuda)[:, 1:]
    odd.copy_(x[:, :64].detach())
    out = ops.attn_var(odd, x.detach()[:, 64:96], x.detach()[:, 96:], seqs, H, Hkv, causal=True)
    A.close(out, ref["out"], ref["out_tol"], "out of unaligned rows")
    wide = torch.zeros((129, 130), dtype=BF, device=cuda)
    out = ops.attn_var(*cut(x), seqs, H, Hkv, causal=True)
    (dx2,) = torch.autograd.grad(out, x, wide[:, 1:65].copy_(do.to(cuda)))
    assert torch.equal(dx2, dx)


def test_shared_key_rows_forward_only(cuda):
    """several examples over the same keys (candidates of one user): forward; the backward refuses"""
    q, k, v, do, qo, ko = _make([5, 7, 3], [90], 2, 1, 32, BF, 4)
    kl, ko = [90, 90, 50], [0, 0, 20]
    ref = A.attn_var(q, k, v, 2, 1, [5, 7, 3], kl, qo, ko)
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    out = ops.attn_var(*lv, ops.AttnSeqs([5, 7, 3], kl, None, ko, device=cuda), 2, 1)
    A.close(out, ref["out"], ref["out_tol"], "out")
    with pytest.raises(RuntimeError, match="share key rows"):
        out.sum().backward()


def test_gradients_against_differences(cuda):
    """fp32, every feature at once: the directional derivative of a weighted sum against central differences in 64 bits of the definition"""
    ql, kl, H, Hkv, dh = [20, 9], [25, 9], 2, 1, 20
    q, k, v, do, qo, ko = _make(ql, kl, H, Hkv, dh, F32, 11)
    sl, pre, docs = torch.tensor([0.1, 0.4]), [4, 0], _docs("any", ql, kl, 2)
    kw = dict(causal=True, cap=2.0)

    def f(q, k, v, sl):
        return float((A.attn_var(q, k, v, H, Hkv, ql, kl, qo, ko, slopes=sl, prefix=pre, docs=docs, **kw)["out"] * do.double()).sum())

    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v, sl)]
    out = ops.attn_var(*lv[:3], ops.AttnSeqs(ql, kl, device=cuda), H, Hkv, slopes=lv[3], prefix=torch.tensor(pre, dtype=torch.int32, device=cuda),
                       docs=tuple(t.to(cuda) for t in docs), **kw)
    grads = torch.autograd.grad(out, lv, do.to(cuda))
    g = torch.Generator().manual_seed(5)
    for i, x in enumerate((q, k, v, sl)):
        d = torch.randn(x.shape, generator=g).double()
        a = [t.double() for t in (q, k, v, sl)]
        a[i] = x.double() + 1e-5 * d
        hi = f(*a)
        a[i] = x.double() - 1e-5 * d
        lo = f(*a)
        want, got = (hi - lo) / 2e-5, float((grads[i].cpu().double() * d).sum())
        assert abs(got - want) <= 2e-5 * float((grads[i].cpu().double() * d).abs().sum()) + 1e-6, (i, got, want)


def test_replays_and_runs_are_identical(cuda):
    """a forward + backward captured in a graph, replayed with eager work of the same leaves between: every replay equals the eager result"""
    ql = [130, 64, 201]
    q, k, v, do, qo, ko = (t.to(cuda) if isinstance(t, torch.Tensor) else t for t in _make(ql, ql, 4, 2, 64, BF, 7))
    seqs = ops.AttnSeqs(ql, device=cuda)
    sl = torch.tensor([0.1, 0.2, 0.3, 0.4], device=cuda)
    docs = tuple(t.to(cuda) for t in _docs("rising", ql, ql, 1))
    lv = [t.requires_grad_(True) for t in (q, k, v, sl)]

    def step():
        out, lse = ops.attn_var(*lv[:3], seqs, 4, 2, slopes=lv[3], causal=True, cap=9.0, docs=docs, want_lse=True)
        return (out.detach(), lse) + torch.autograd.grad(out, lv, do)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, again):
        assert torch.equal(a, b)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = step()
    with torch.cuda.graph(g2):
        r2 = step()
    for _ in range(3):
        for t in r1 + r2:
            t.fill_(float("nan"))
        g1.replay()
        step()
        g2.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, r1, r2):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dh,kw", [(80, dict(slopes=True)), (80, dict()), (64, dict(slopes=True, cap=20.0, causal=True)), (128, dict(causal=True)),
                                   (32, dict(slopes=True, causal=True))])
def test_many_histories_give_the_same_results_again(cuda, dh, kw):
    """a device full of histories whose last tile lacks a few rows, forward and backward several times: identical every time, and right against
    plain fp32 (a wait that is missing behind a matrix product shows up here as a few rows that change from run to run)"""
    H, B = 4, 200
    ql = [60 + (i % 5) + 64 * (i % 3) for i in range(B)]
    q, k, v, do, qo, _ = _make(ql, ql, H, H, dh, BF, 21)
    kw = dict(kw)
    sl = (0.5 * torch.exp2(-2.0 * torch.arange(1, H + 1)) if kw.pop("slopes", False) else None)
    seqs = ops.AttnSeqs(ql, device=cuda)
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)] + ([sl.to(cuda).requires_grad_(True)] if sl is not None else [])

    def step():
        out, lse = ops.attn_var(*lv[:3], seqs, H, slopes=lv[3] if sl is not None else None, want_lse=True, **kw)
        return [out.detach(), lse] + list(torch.autograd.grad(out, lv, do.to(cuda)))

    first = step()
    for _ in range(5):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)
    most = max(ql)
    at = torch.as_tensor(qo, device=cuda)[:, None] + torch.arange(most, device=cuda)[None]
    ok = torch.arange(most, device=cuda)[None] < torch.as_tensor(ql, device=cuda)[:, None]
    x = [t.to(cuda).float()[at.clamp(max=q.shape[0] - 1)].reshape(B, most, H, dh).transpose(1, 2) for t in (q, k, v)]
    z = x[0] @ x[1].transpose(-1, -2) * dh ** -0.5
    if kw.get("cap"):
        z = kw["cap"] * torch.tanh(z / kw["cap"])
    i = torch.arange(most, device=cuda)
    if sl is not None:
        z = z - sl.to(cuda)[None, :, None, None] * (i[:, None] - i[None]).abs()
    see = ok[:, None, None, :] & ((i[:, None] >= i[None]) if kw.get("causal") else torch.ones_like(i[:, None] >= i[None]))
    z = z.masked_fill(~see, -np.inf)
    want = (torch.softmax(z, -1) @ x[2].masked_fill(~ok[:, None, :, None], 0)).transpose(1, 2).reshape(B, most, H * dh)[ok]
    lse = torch.logsumexp(z, -1).transpose(1, 2)[ok]
    assert (first[0].float() - want).abs().max() <= 2.0 ** -8 * 2 * float(v.abs().max())      # two roundings of values of at most max |v|
    assert (first[1] - lse).abs().max() <= 1e-4


def test_slopes_without_queries_or_keys(cuda):
    """gradients where there is nothing to see: zeros, and nothing left unwritten"""
    sl = torch.tensor([0.3, 0.1], device=cuda)
    for ql, kl in (([0, 0], [5, 3]), ([4, 2], [0, 0]), ([0], [0])):
        lv = [torch.randn((n, 2 * 32), device=cuda).to(BF).requires_grad_(True) for n in (sum(ql), sum(kl), sum(kl))] + [sl.clone().requires_grad_(True)]
        out = ops.attn_var(*lv[:3], ops.AttnSeqs(ql, kl, device=cuda), 2, slopes=lv[3])
        assert (out == 0).all()
        for g, x in zip(torch.autograd.grad(out, lv, torch.ones_like(out)), lv):
            assert g.shape == x.shape and (g == 0).all()


def test_gradients_of_gradients_and_changed_masks_are_refused(cuda):
    q, k, v, do, _, _ = _make([9, 4], [9, 4], 2, 2, 32, F32, 3)
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    seqs = ops.AttnSeqs([9, 4], device=cuda)
    prefix = torch.tensor([2, 0], dtype=torch.int32, device=cuda)
    out = ops.attn_var(*lv, seqs, 2, causal=True, prefix=prefix)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out, lv, do.to(cuda), create_graph=True)
    out = ops.attn_var(*lv, seqs, 2, causal=True, prefix=prefix)
    prefix[0] = 4
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, lv, do.to(cuda))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_padded_batch_is_a_packed_one(cuda, dtype):
    """rows [B, T, d] with lengths: offsets b T, nothing copied; the padding of the results is zero and what stands in the operands' padding
    (NaN here) reaches nothing.  Same kernels, same rows: bit-equal to the packed call"""
    B, T, H, dh = 3, 70, 2, 32
    ql = [70, 1, 33]
    q, k, v, do, _, _ = (t.to(cuda) if isinstance(t, torch.Tensor) else t for t in _make(ql, ql, H, H, dh, dtype, 4))
    at = torch.cat([b * T + torch.arange(n) for b, n in enumerate(ql)]).to(cuda)

    def spread(t):
        x = torch.full((B * T, H * dh), float("nan"), dtype=dtype, device=cuda)
        x[at] = t
        return x

    packed = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = ops.attn_var(*packed, ops.AttnSeqs(ql, device=cuda), H, causal=True)
    gw = torch.autograd.grad(want, packed, do)
    dense = [spread(t).requires_grad_(True) for t in (q, k, v)]
    got = ops.attn_var(*dense, ops.AttnSeqs(ql, q_off=[b * T for b in range(B)], device=cuda), H, causal=True)
    gg = torch.autograd.grad(got, dense, spread(do))
    pad = torch.ones(B * T, dtype=torch.bool, device=cuda)
    pad[at] = False
    for a, b in zip((want,) + gw, (got,) + gg):
        assert torch.equal(a, b[at]) and (b[pad] == 0).all()


def test_a_broadcast_gradient_and_parts_of_one_tensor(cuda):
    """the gradient of a sum (a tensor without strides), and q, k, v as column slices of one projection"""
    H, dh, ql = 2, 32, [40, 7]
    g = torch.Generator().manual_seed(6)
    x = torch.randn((47, 3 * H * dh), generator=g).to(BF)
    leaf = x.to(cuda).requires_grad_(True)
    d = H * dh
    out = ops.attn_var(leaf[:, :d], leaf[:, d:2 * d], leaf[:, 2 * d:], ops.AttnSeqs(ql, device=cuda), H, causal=True)
    out.sum().backward()
    ref = A.attn_var(x[:, :d], x[:, d:2 * d], x[:, 2 * d:], H, H, ql, ql, [0, 40], [0, 40], causal=True, dout=torch.ones((47, d), dtype=BF))
    for n, c in (("dq", 0), ("dk", 1), ("dv", 2)):
        A.close(leaf.grad[:, c * d:(c + 1) * d], ref[n], ref[n + "_tol"], n)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_one_example_past_4_gib(cuda, dtype):
    """300 rows of q, k, v and dout as columns of one matrix whose rows take nearly 16 MB: the example reaches past 2 and 4 GiB.  The head size is no
    tile size, and what stands beside the columns (ones) belongs to no operand."""
    L_, dh, es = 300, 96, torch.finfo(dtype).bits // 8
    buf = torch.ones((L_, ((1 << 24) - 16) // es), dtype=dtype, device=cuda)
    q, k, v, do, _, _ = _make([L_], [L_], 1, 1, dh, dtype, 11)
    cols = []
    for n, t in enumerate((q, k, v, do)):
        buf[:, n * dh:n * dh + dh] = t.to(cuda)
        cols.append(buf[:, n * dh:n * dh + dh])
    ref = A.attn_var(q, k, v, 1, 1, [L_], [L_], [0], [0], causal=True, dout=do)
    lv = [c.detach().requires_grad_(True) for c in cols[:3]]
    out, lse = ops.attn_var(*lv, ops.AttnSeqs([L_], device=cuda), 1, causal=True, want_lse=True)
    grads = torch.autograd.grad(out, lv, cols[3])
    for t, n in zip((out, lse) + grads, ("out", "lse", "dq", "dk", "dv")):
        A.close(t, ref[n], ref[n + "_tol"], n)


def test_contiguous_rows_of_one_example_past_4_gib(cuda):
    """360000 query rows of 64 heads of 96 (12 KB each) over 64 keys: q, out, dout and dq pass 4 GiB"""
    g = torch.Generator(device=cuda).manual_seed(5)
    n, kl, H, Hkv, dh = 360000, 64, 64, 2, 96
    q, do = (torch.empty((n, H * dh), dtype=BF, device=cuda).normal_(generator=g) for _ in range(2))
    k, v = (torch.empty((kl, Hkv * dh), dtype=BF, device=cuda).normal_(generator=g) for _ in range(2))
    lv = [t.requires_grad_(True) for t in (q, k, v)]
    out = ops.attn_var(*lv, ops.AttnSeqs([n], [kl], device=cuda), H, Hkv)
    dq, dk, dv = torch.autograd.grad(out, lv, do)
    two, four = 2 ** 31 // (H * dh * 2), 2 ** 32 // (H * dh * 2)
    rows = torch.cat([torch.arange(a, b) for a, b in ((0, 130), (two - 70, two + 70), (four - 70, four + 70), (n - 130, n))]).to(cuda)
    ok = torch.ones((n, kl), dtype=torch.bool, device=cuda)
    dist = torch.zeros((1, 1), dtype=torch.int64, device=cuda)
    u = torch.finfo(BF).eps / 2
    sums = {x: torch.zeros((kl, Hkv * dh), dtype=torch.float64, device=cuda) for x in ("dk", "dv", "dk_tol", "dv_tol")}
    with torch.no_grad():
        for h in range(H):
            c, ck = slice(h * dh, h * dh + dh), slice(h // 32 * dh, h // 32 * dh + dh)
            r = A.head(q[:, c], k[:, ck], v[:, ck], ok, dist, dh ** -0.5, 0.0, None, BF, do[:, c])
            for t, x in ((out, "out"), (dq, "dq")):
                A.close(t[rows, c], r[x][rows].cpu(), r[x + "_tol"][rows].cpu(), "%s of head %d" % (x, h))
            for x in sums:
                sums[x][:, ck] += r[x]
        for t, x in ((dk, "dk"), (dv, "dv")):
            A.close(t, sums[x].cpu(), (sums[x + "_tol"] + u * sums[x].abs() + 1e-30).cpu(), x)


@pytest.mark.parametrize("cap", [0.01, 1.0, 30.0, 50.0, 1e3, 1e6, 1e30, 9e37])
def test_capped_scores_keep_their_bits(cuda, cap):
    """One visible key: lse is the score.  x is exact in fp32 (one product, a scale of 1), so what is off is the cap alone: the tanh form (under
    2^-20 of the value: a polynomial below x = 0.35 cap, 1 - 2 / (1 + e^2x) above, with v_rcp_f32 and v_exp_f32 of 1 ulp) and three
    products that turn it to log2 units and back (2^-24 each).  Nothing may grow with the cap."""
    mags = torch.logspace(-6, 4, 401, dtype=torch.float64).to(F32)
    if cap < 1e4:
        mags = torch.cat([mags, torch.linspace(0.01, 4, 400, dtype=torch.float64).to(F32) * cap])
    x = torch.cat([mags, -mags, torch.zeros(1)])
    q = torch.zeros((len(x), 16), dtype=F32)
    q[:, 3] = x
    k = torch.zeros((1, 16), dtype=F32)
    k[0, 3] = 1.0
    out, lse = ops.attn_var(q.to(cuda), k.to(cuda), k.to(cuda), ops.AttnSeqs([len(x)], [1], device=cuda), 1, scale=1.0, cap=cap, want_lse=True)
    want = cap * torch.tanh(x.double() / cap)
    assert ((lse[:, 0].cpu().double() - want).abs() <= 2.0 ** -19 * want.abs()).all()
    assert torch.equal(out.cpu(), k.expand(len(x), 16))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30])
def test_caps_far_over_the_scores_change_nothing(cuda, cap, dtype):
    """Scores of about 8 under a cap of 1e4 and more: y = x (1 - (x / cap)^2 / 3 ...) is x to 1e-6 of it.  The bounds are those of scores without a
    cap (which do not grow with it), plus that difference in the scores' own bound (FP32 = 2^-17 holds it)."""
    ql, kl, H, Hkv, dh = [100, 37], [100, 90], 4, 2, 64
    q, k, v, do, qo, ko = _make(ql, kl, H, Hkv, dh, dtype, 12, 1.5)
    sl = torch.tensor([0.1, 0.0, 1.0, 0.01])
    ref = A.attn_var(q, k, v, H, Hkv, ql, kl, qo, ko, causal=True, slopes=sl, dout=do)
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v, sl)]
    out, lse = ops.attn_var(*lv[:3], ops.AttnSeqs(ql, kl, device=cuda), H, Hkv, slopes=lv[3], causal=True, cap=cap, want_lse=True)
    for t, n in zip((out, lse) + torch.autograd.grad(out, lv, do.to(cuda)), ("out", "lse", "dq", "dk", "dv", "dslope")):
        A.close(t, ref[n], ref[n + "_tol"], n)


@pytest.mark.parametrize("causal", [True, False])
def test_lengths_past_the_bounds_are_cut_where_they_stand(cuda, causal):
    """A replayed graph's lengths may outgrow max_q / max_k: the rows past them are cut, and those before keep their positions (i + Lk - Lq of the
    stated lengths): nothing sees a key that it would not see in the whole history"""
    for mq, mk, ql, kl in ((40, 90, 70, 90), (70, 50, 70, 90), (33, 65, 150, 170), (40, 200, 100, 30)):
        q, k, v, do, _, _ = _make([ql], [kl], 2, 1, 32, F32, 13)
        seqs = ops.AttnSeqs([min(ql, mq)], [min(kl, mk)], device=cuda, max_q=mq, max_k=mk, zero_fill=True)
        seqs.q_lens.fill_(ql)
        seqs.k_lens.fill_(kl)
        nq, nk = min(ql, mq), min(kl, mk)
        sl = torch.tensor([0.2, 0.05])
        lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v, sl)]
        out, lse = ops.attn_var(*lv[:3], seqs, 2, 1, slopes=lv[3], causal=causal, want_lse=True)
        grads = torch.autograd.grad(out, lv, do.to(cuda))
        dist = torch.arange(nq)[:, None] + kl - ql - torch.arange(nk)[None]
        ok = dist >= 0 if causal else torch.ones((nq, nk), dtype=torch.bool)
        dk, dv, tk, tv = (torch.zeros((nk, 32), dtype=torch.float64) for _ in range(4))
        for h in range(2):
            c = slice(32 * h, 32 * h + 32)
            r = A.head(q[:nq, c], k[:nk], v[:nk], ok, dist, 32 ** -0.5, 0.0, sl[h].double(), F32, do[:nq, c])
            A.close(out[:nq, c], r["out"], r["out_tol"], "out")
            A.close(lse[:nq, h], r["lse"], r["lse_tol"], "lse")
            A.close(grads[0][:nq, c], r["dq"], r["dq_tol"], "dq")
            A.close(grads[3][h:h + 1], r["dslope"][None], r["dslope_tol"][None], "dslope")
            dk, dv, tk, tv = dk + r["dk"], dv + r["dv"], tk + r["dk_tol"], tv + r["dv_tol"]
        A.close(grads[1][:nk], dk, tk + 2.0 ** -24 * dk.abs() + 1e-30, "dk")
        A.close(grads[2][:nk], dv, tv + 2.0 ** -24 * dv.abs() + 1e-30, "dv")
        assert (out[nq:] == 0).all() and (grads[0][nq:] == 0).all() and (grads[1][nk:] == 0).all() and (grads[2][nk:] == 0).all()


@pytest.mark.parametrize("rows", [0, 3])
@pytest.mark.parametrize("most", [None, 4])
def test_an_empty_batch_has_gradients(cuda, rows, most):
    """no example at all, with and without rows of no example: everything is zero, the slopes' gradient too"""
    lv = [torch.randn((rows, 64), device=cuda).to(BF).requires_grad_(True) for _ in range(3)] + [torch.tensor([0.3, 0.1], device=cuda, requires_grad=True)]
    keep = torch.full((2,), 7.0, device=cuda)
    del keep                                                                     # (the allocator hands this memory out again: nothing may be left unwritten)
    out = ops.attn_var(*lv[:3], ops.AttnSeqs([], device=cuda, max_q=most, max_k=most), 2, slopes=lv[3])
    assert out.shape == (rows, 64) and (out == 0).all()
    for g, x in zip(torch.autograd.grad(out, lv, torch.ones_like(out)), lv):
        assert g.shape == x.shape and (g == 0).all()


def test_nothing_is_kept_for_a_backward_that_will_not_run(cuda, monkeypatch):
    """under no_grad the part of the output that rounding took away is neither allocated nor written, whatever the operands require"""
    seen, orig = [], ops._attn_var_desc
    monkeypatch.setattr(ops, "_attn_var_desc", lambda *a, **kw: seen.append(a[11]) or orig(*a, **kw))
    lv = [torch.randn((9, 64), device=cuda).to(BF).requires_grad_(True) for _ in range(3)]
    seqs = ops.AttnSeqs([9], device=cuda)
    with torch.no_grad():
        a = ops.attn_var(*lv, seqs, 2)
    b = ops.attn_var(*lv, seqs, 2)
    ops.attn_var(*(t.detach() for t in lv), seqs, 2)
    assert seen[0] is None and seen[1] is not None and seen[2] is None
    assert torch.equal(a, b)


@pytest.mark.parametrize("dh,dtype", [(20, F32), (64, F32), (80, F32), (128, F32), (64, BF), (80, BF), (128, BF)])
def test_fp32_results_have_fp32_bits(cuda, dh, dtype):
    """Held to the bound of fp32 arithmetic (out in fp32, lse in both types), under what rounding the operands or the weights to a shorter type would
    leave in rows of few keys (2^-12 for fp16, 2^-9 for bf16).  q and k are multiples of 1/8 up to 1: every partial sum of q . k is a multiple of
    1/64 under 2^7, exact in any order.  z = x / 16, |z| <= 8; in log2 units its two products and the subtraction of the maximum round by 2^-24 of up
    to 23 each: 2^-18 in the exponent, as much in the weight; v_exp_f32: 1 ulp, 2^-23.  The sums of weights and of weights times v over at most 300
    keys: 300 2^-24 = 2^-15.8 of the absolute sum in the worst order, each.  Together under 2^-14.5 of sum p |v|, and of the sum for lse."""
    g = torch.Generator().manual_seed(dh)
    ql, kl = [300, 70], [300, 200]
    n = lambda r: (torch.randint(-8, 9, (r, 2 * dh), generator=g) / 8.0)  # noqa: E731
    q, k, v = n(370), n(500), n(500)
    scale = 1.0 / 16
    out, lse = ops.attn_var(*(t.to(dtype).to(cuda) for t in (q, k, v)), ops.AttnSeqs(ql, kl, device=cuda), 2, scale=scale, causal=True, want_lse=True)
    qo, ko = [0, 300], [0, 300]
    for b in range(2):
        for h in range(2):
            c = slice(h * dh, h * dh + dh)
            qq, kk, vv = q[qo[b]:qo[b] + ql[b], c].double(), k[ko[b]:ko[b] + kl[b], c].double(), v[ko[b]:ko[b] + kl[b], c].double()
            z = qq @ kk.T * scale
            see = torch.arange(kl[b])[None] <= torch.arange(ql[b])[:, None] + kl[b] - ql[b]
            z = z.masked_fill(~see, -np.inf)
            assert float(z[see].abs().max()) <= 8
            p = torch.softmax(z, -1)
            # lse: the sum's relative error and 2^-22 of the value (two products, v_log_f32)
            want = torch.logsumexp(z, -1)
            assert ((lse[qo[b]:qo[b] + ql[b], h].cpu().double() - want).abs() <= 2.0 ** -14.5 + 2.0 ** -22 * want.abs()).all()
            if dtype is F32:
                assert ((out[qo[b]:qo[b] + ql[b], c].cpu().double() - p @ vv).abs() <= 2.0 ** -14.5 * (p @ vv.abs()) + 1e-30).all()


def _masked_reference(q, k, v, do, ok, dist, scale, slope):
    """one head in 64 bits, with sums over the visible places alone: what stands in a masked one does not enter even as 0 * NaN"""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    z = torch.where(ok, (q[:, None] * k[None]).sum(-1) * scale - slope * dist.abs(), torch.full(ok.shape, -np.inf, dtype=torch.float64))
    p = torch.where(ok, torch.softmax(z, -1), torch.zeros_like(z))
    over = lambda w, x, dim: torch.where(ok[..., None], w[..., None] * x, torch.zeros((), dtype=torch.float64)).sum(dim)  # noqa: E731
    out = over(p, v[None], 1)
    D = (do * out).sum(-1, keepdim=True)
    dx = torch.where(ok, p * ((do[:, None] * v[None]).sum(-1) - D), torch.zeros_like(z))
    return dict(out=out, dq=over(dx, k[None], 1) * scale, dk=over(dx, q[:, None], 0) * scale, dv=over(p, do[:, None], 0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("where", ["q", "k", "v", "v dims", "do", "all v"])
@pytest.mark.parametrize("dh", [32, 80, 128])
def test_nan_reaches_what_sees_it_and_nothing_else(cuda, dh, where, dtype):
    """NaN in some places of a causal history with slopes: the same places of every result are NaN as by the definition, with sums over the visible
    places alone, and the others hold the bounds of the history without it"""
    n, H = 150, 2
    q, k, v, do, _, _ = _make([n], [n], H, 1, dh, dtype, 31)
    clean = [t.clone() for t in (q, k, v, do)]
    if where == "q":
        q[70, 5] = np.nan
    elif where == "k":
        k[[100, 149], 3] = np.nan
    elif where == "v":
        v[[64, 140]] = np.nan
    elif where == "v dims":
        v[130, [0, dh - 1]], v[20, 17] = np.nan, np.nan
    elif where == "do":
        do[90, dh + 1] = np.nan
    else:
        v[:, 9] = np.nan
    sl = torch.tensor([0.1, 0.02])
    ref = A.attn_var(*clean[:3], H, 1, [n], [n], [0], [0], causal=True, slopes=sl, dout=clean[3])
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    out = ops.attn_var(*lv, ops.AttnSeqs([n], device=cuda), H, 1, slopes=sl.to(cuda), causal=True)
    grads = torch.autograd.grad(out, lv, do.to(cuda))
    dist = (torch.arange(n)[:, None] - torch.arange(n)[None]).double()
    want = dict(out=torch.zeros(q.shape, dtype=torch.float64), dq=torch.zeros(q.shape, dtype=torch.float64), dk=0, dv=0)
    for h in range(H):
        c = slice(h * dh, h * dh + dh)
        r = _masked_reference(q[:, c], k, v, do[:, c], dist >= 0, dist, dh ** -0.5, float(sl[h]))
        want["out"][:, c], want["dq"][:, c] = r["out"], r["dq"]
        want["dk"], want["dv"] = want["dk"] + r["dk"], want["dv"] + r["dv"]
    for t, x in zip((out,) + grads, ("out", "dq", "dk", "dv")):
        assert want[x].isnan().any() or (where == "do" and x == "out") or (where in ("v", "v dims", "all v") and x == "dv")
        A.close(t, torch.where(want[x].isnan(), want[x], ref[x]), ref[x + "_tol"], x)


@pytest.mark.parametrize("where", ["q", "v"])
def test_nan_in_every_row_is_not_a_matter_of_minutes(cuda, where):
    """a step whose operands hold NaN everywhere (one NaN weight is enough): the rows that are looked at again stop where NaN has settled them.  Walking
    them to the end took several hundred times the step; a clean one here takes some 0.2 ms"""
    n, H, dh = 2048, 8, 64
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k, v, do = (torch.empty((2 * n, H * dh), dtype=BF, device=cuda).normal_(generator=g) for _ in range(4))
    seqs = ops.AttnSeqs([n, n], device=cuda)

    def step(*ops_):
        lv = [t.detach().requires_grad_(True) for t in ops_]
        torch.cuda.synchronize()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        out = ops.attn_var(*lv, seqs, H, causal=True)
        grads = torch.autograd.grad(out, lv, do)
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b), out, grads

    fine = min(step(q, k, v)[0] for _ in range(4))
    bad = [t.clone() for t in (q, k, v)]
    if where == "q":
        bad[0][:, ::dh] = np.nan
    else:
        bad[2][:, ::dh] = np.nan
    took, out, grads = min((step(*bad) for _ in range(3)), key=lambda r: r[0])
    cols = torch.arange(H * dh, device=cuda) % dh == 0
    assert out.isnan().all() if where == "q" else (out[:, cols].isnan().all() and not out[:, ~cols].isnan().any())
    assert grads[0].isnan().all() and grads[1].isnan().all()
    assert took < 60 * max(fine, 0.1), "%.2f ms, %.2f ms without NaN" % (took, fine)


@pytest.mark.parametrize("cap,Hkv", [(0.0, 4), (20.0, 1)])
def test_gradients_with_documents_are_as_exact_as_their_rounding(cuda, cap, Hkv):
    """bf16, sessions of a causal history behind a common prefix: few keys share a row's weight, and what dX loses as an operand and rowsum(dout out)
    through the rounded weights adds up to half of what the rounding of dq and dk themselves takes (0.0025 of the norm against 0.0017).  With the
    rest of dX multiplied too, all that is left beside that rounding may be 0.66 of it: 1.2 times in norm."""
    T, H, dh, prefix = 1024, 4, 64, 40
    g = torch.Generator().manual_seed(41)
    n = lambda w: torch.randn((T, w), generator=g).to(BF)  # noqa: E731
    q, k, v, do = n(H * dh), n(Hkv * dh), n(Hkv * dh), n(H * dh)
    doc = (torch.arange(T) * 9 // T).to(torch.int32)
    ref = A.attn_var(q, k, v, H, Hkv, [T], [T], [0], [0], causal=True, cap=cap, prefix=[prefix], docs=(doc, doc), dout=do)
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    d = doc.to(cuda)
    out = ops.attn_var(*lv, ops.AttnSeqs([T], device=cuda), H, Hkv, causal=True, cap=cap, docs=(d, d), prefix=torch.tensor([prefix], dtype=torch.int32, device=cuda))
    for t, x in zip(torch.autograd.grad(out, lv, do.to(cuda))[:2], ("dq", "dk")):
        alone = (ref[x].to(BF).double() - ref[x]).norm()
        assert (t.cpu().double() - ref[x]).norm() <= 1.2 * alone, x


@pytest.mark.parametrize("dh", [32, 64, 80, 128])
@pytest.mark.parametrize("cap", [64.0, 65.0, 400.0])
def test_caps_on_both_sides_of_the_short_form(cuda, cap, dh):
    """bf16 takes the short form of a cap up to 64, kernels of their own beyond; few and many rows a workgroup, with and without documents, scores that
    reach the cap"""
    docs = (np.arange(200) * 5 // 200, np.arange(200) * 5 // 200)
    _check(cuda, [130, 70], [130, 70], 4, 2, dh, std=8.0, cap=cap, causal=True, slopes=[0.1, 0.0, 1.0, 0.01], scale=0.5)
    _check(cuda, [130, 70], [130, 70], 2, 2, dh, std=2.0, cap=cap, docs=tuple(torch.as_tensor(d) for d in docs), prefix=[3, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("where", ["q", "v", "v dims", "do"])
def test_nan_stays_in_its_document(cuda, where, dtype):
    """NaN in one session of a causal history behind a prefix: what sees that session, and nothing else"""
    n, H, dh, prefix = 160, 2, 64, 5
    q, k, v, do, _, _ = _make([n], [n], H, 1, dh, dtype, 51)
    clean = [t.clone() for t in (q, k, v, do)]
    t, at = {"q": (q, (90,)), "v": (v, (100,)), "v dims": (v, (85, [0, 63])), "do": (do, (95, slice(0, dh)))}[where]
    t[at] = np.nan
    doc = torch.as_tensor(np.arange(n) // 40, dtype=torch.int32)
    ref = A.attn_var(*clean[:3], H, 1, [n], [n], [0], [0], causal=True, prefix=[prefix], docs=(doc, doc), dout=clean[3])
    lv = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    d = doc.to(cuda)
    out = ops.attn_var(*lv, ops.AttnSeqs([n], device=cuda), H, 1, causal=True, docs=(d, d), prefix=torch.tensor([prefix], dtype=torch.int32, device=cuda))
    grads = torch.autograd.grad(out, lv, do.to(cuda))
    ok, dist = A.visible(n, n, True, prefix, doc, doc), (torch.arange(n)[:, None] - torch.arange(n)[None]).double()
    want = dict(out=torch.zeros(q.shape, dtype=torch.float64), dq=torch.zeros(q.shape, dtype=torch.float64), dk=0, dv=0)
    for h in range(H):
        c = slice(h * dh, h * dh + dh)
        r = _masked_reference(q[:, c], k, v, do[:, c], ok, dist, dh ** -0.5, 0.0)
        want["out"][:, c], want["dq"][:, c] = r["out"], r["dq"]
        want["dk"], want["dv"] = want["dk"] + r["dk"], want["dv"] + r["dv"]
    for t, x in zip((out,) + grads, ("out", "dq", "dk", "dv")):
        nan = want[x].isnan()
        assert not nan[:80].all() and not nan[120:].any()
        A.close(t, torch.where(nan, want[x], ref[x]), ref[x + "_tol"], x)
