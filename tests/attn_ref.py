"""The definition of attn_var and of the cached attention in 64 bits, one head of one example at a time, with the bounds that the roundings of
the kernels allow: every operand and result is rounded to its type once, the weights P (and dX) are rounded to the operands' type before
they enter a matrix product.  One rounding is off by at most u = eps / 2 of the value; FP32 covers fp32 accumulation (sums of n terms of
mixed signs: 2^-24 times a few of them, taken at 2^-18 of the absolute sum), v_exp_f32 / v_rcp_f32 and the tanh form (2^-21)."""
import numpy as np
import torch

F = torch.float64
FP32 = 2.0 ** -17


def visible(ql, kl, causal, prefix, qd, kd):
    i, j = torch.arange(ql)[:, None], torch.arange(kl)[None]
    ok = torch.ones((ql, kl), dtype=torch.bool)
    if causal:
        ok &= j <= i + kl - ql
    if qd is not None:
        ok &= qd[:, None] == kd[None]
    if prefix is not None:
        ok |= j < prefix
    return ok


def head(q, k, v, ok, dist, scale, cap, slope, dtype, dout=None):
    """One head: dict of results and of elementwise bounds of what a kernel in `dtype` may be off by."""
    u = torch.finfo(dtype).eps / 2
    q, k, v = q.to(F), k.to(F), v.to(F)
    x = q @ k.T * scale
    t = torch.tanh(x / cap) if cap else None
    y = cap * t if cap else x
    z = y - slope * dist.abs().to(F) if slope is not None else y
    z = z.masked_fill(~ok, -np.inf)
    lse = torch.logsumexp(z, -1)
    p = torch.where(ok, torch.exp(z - lse[:, None]), torch.zeros_like(z))
    v0 = torch.where(ok.any(0)[:, None], v, torch.zeros_like(v))           # (what nobody sees may hold anything)
    k0 = torch.where(ok.any(0)[:, None], k, torch.zeros_like(k))
    out = p @ v0
    # scores: relative error of a weight from the fp32 scores (their absolute error is FP32 times the terms that make them)
    mag = (q.abs() @ k0.abs().T * scale) if not cap else torch.full_like(x, float(cap)).minimum(q.abs() @ k0.abs().T * scale) + cap * 2.0 ** -4
    if slope is not None:
        mag = mag + abs(float(slope)) * dist.abs().to(F)
    ez = FP32 * (torch.where(ok, mag, torch.zeros_like(mag)).amax(-1, keepdim=True) + 1)
    A = p @ v0.abs()
    r = dict(out=out, lse=lse, out_tol=(u + 2 * ez) * A + u * out.abs() + 1e-30, lse_tol=ez[:, 0] + 2.0 ** -20 * lse.abs().nan_to_num(posinf=0, neginf=0))
    if dout is None:
        return r
    g = dout.to(F)
    seen = ok.any(-1)
    dp = g @ v0.T
    D = (g * out).sum(-1, keepdim=True)
    dz = p * (dp - D)
    f = (1 - t * t) if cap else torch.ones_like(x)
    dx = dz * f
    eD = (g.abs() * r["out_tol"]).sum(-1, keepdim=True) + FP32 * (g.abs() * out.abs()).sum(-1, keepdim=True)
    edx = u * dx.abs() + p * (eD + 2 * ez * (dp.abs() + D.abs()) + FP32 * (g.abs() @ v0.abs().T))
    g0 = torch.where(seen[:, None], g, torch.zeros_like(g))
    r.update(dq=dx @ k0 * scale, dk=dx.T @ q * scale, dv=p.T @ g0)
    r["dq_tol"] = (edx + FP32 * dx.abs()) @ k0.abs() * scale + u * r["dq"].abs() + 1e-30
    r["dk_tol"] = (edx + FP32 * dx.abs()).T @ q.abs() * scale
    r["dv_tol"] = (p * (u + 2 * ez)).T @ g0.abs() + 1e-30
    if slope is not None:
        a = dist.abs().to(F)
        r["dslope"] = -(dz * a).sum()
        r["dslope_tol"] = 8 * (ez * p * (dp.abs() + D.abs()) * (a + (p * a).sum(-1, keepdim=True))).sum() + 1e-30
    return r


def attn_var(q, k, v, H, Hkv, ql, kl, qo, ko, causal=False, cap=0.0, slopes=None, prefix=None, docs=None, scale=None, dout=None):
    """All heads and examples, operands on the CPU in their own type; rows of no example: zero (lse -inf)."""
    dh, G, u = q.shape[1] // H, H // Hkv, torch.finfo(q.dtype).eps / 2
    scale = dh ** -0.5 if scale is None else scale
    z = lambda t: torch.zeros(t.shape, dtype=F)  # noqa: E731
    R = dict(out=z(q), out_tol=z(q), lse=torch.full((q.shape[0], H), -np.inf, dtype=F), lse_tol=torch.zeros((q.shape[0], H), dtype=F))
    if dout is not None:
        R.update(dq=z(q), dq_tol=z(q), dk=z(k), dk_tol=z(k), dv=z(v), dv_tol=z(v), dslope=torch.zeros(H, dtype=F), dslope_tol=torch.zeros(H, dtype=F))
    for b in range(len(ql)):
        if not ql[b] or not kl[b]:
            continue
        qs, ks = slice(qo[b], qo[b] + ql[b]), slice(ko[b], ko[b] + kl[b])
        ok = visible(ql[b], kl[b], causal, None if prefix is None else int(prefix[b]), *((None, None) if docs is None else (docs[0][qs], docs[1][ks])))
        dist = torch.arange(ql[b])[:, None] + kl[b] - ql[b] - torch.arange(kl[b])[None]
        for h in range(H):
            c, ck = slice(h * dh, h * dh + dh), slice(h // G * dh, h // G * dh + dh)
            r = head(q[qs, c], k[ks, ck], v[ks, ck], ok, dist, scale, cap, None if slopes is None else slopes[h].to(F), q.dtype,
                     None if dout is None else dout[qs, c])
            for n in ("out", "out_tol"):
                R[n][qs, c] = r[n]
            for n in ("lse", "lse_tol"):
                R[n][qs, h] = r[n]
            if dout is not None:
                for n in ("dq", "dq_tol"):
                    R[n][qs, c] = r[n]
                for n in ("dk", "dk_tol", "dv", "dv_tol"):
                    R[n][ks, ck] += r[n]
                if slopes is not None:
                    R["dslope"][h] += r["dslope"]
                    R["dslope_tol"][h] += r["dslope_tol"]
    if dout is not None:                                       # the one rounding of the summed gradients
        R["dk_tol"] += u * R["dk"].abs() + 1e-30
        R["dv_tol"] += u * R["dv"].abs()
    return R


def close(got, want, tol, what):
    got = got.detach().cpu().to(F)
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of the bound (got %.6g, want %.6g)" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).nan_to_num(nan=np.inf).max()), float(got[bad][0]), float(want[bad][0]))
