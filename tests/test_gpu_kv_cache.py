"""The 8-bit K / V cache: plan (block tables, slots), append, read, attention, release -- each against a plain statement on the host, and a
run of them together as a serving loop uses them."""
import numpy as np
import pytest
import torch

from cikm2020_dmt_amd import kv_cache as KV
from tests import attn_ref as A

pytestmark = pytest.mark.gpu
BF, BS = torch.bfloat16, KV.BLOCK
F64 = torch.float64


def _i(x, cuda):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(cuda)


# ------------------------------------------------------------------------------------------------ plan
def _plan_ref(lens, new, table, free, n_free, rows):
    n, width = table.shape
    table, free_left, cum = table.copy(), n_free, 0
    off, after, slots, runs, refused = [0], [], np.full(rows, -1), [], 0
    for r in range(n):
        m = max(int(new[r]), 0)
        first, end = off[-1], off[-1] + m
        off.append(end)                        # (unclipped here: row_off itself is cut at 2^31 - 1)
        fits = new[r] >= 0 and lens[r] >= 0 and lens[r] + m <= width * BS and end <= rows
        have = -(-int(lens[r]) // BS)
        need = -(-(int(lens[r]) + m) // BS) - have if fits else 0
        cum += need
        ok = fits and (need == 0 or cum <= n_free)
        after.append(int(lens[r]) + m if ok else int(lens[r]))
        if not ok:
            refused += 1
            continue
        for j in range(need):
            table[r, have + j] = free[n_free - 1 - (cum - need + j)]
        free_left -= need
        for t in range(first, end):
            pos = int(lens[r]) + t - first
            slots[t] = table[r, pos // BS] * BS + pos % BS
            if t == first or pos % BS == 0:
                runs.append([t, 0])
            runs[-1][1] += 1
    cap = min(rows, rows // BS + 2 * n)
    runs = np.array(runs + [[-1, 0]] * (cap - len(runs))).reshape(cap, 2)
    return np.minimum(off, 2 ** 31 - 1), after, slots, runs, free_left, refused, table


def _check_plan(cuda, lens, new, width, n_free=None, rows=None, seed=0):
    r = np.random.RandomState(seed)
    lens, new = np.asarray(lens, dtype=np.int64), np.asarray(new, dtype=np.int64)
    have = -(-np.maximum(lens, 0) // BS)
    rows = int(np.maximum(new, 0).sum()) if rows is None else rows
    total = min(int(have.sum() + (np.maximum(new, 0) // BS + 1).sum()), 100000)
    ids = r.permutation(total + 5)
    table, at = np.full((len(lens), width), -1), 0
    for i, h in enumerate(np.minimum(have, width)):
        table[i, :h] = ids[at:at + h]
        at += h
    free = ids[at:]
    n_free = len(free) if n_free is None else n_free
    want = _plan_ref(lens, new, table, free, n_free, rows)
    tb, fr = _i(table, cuda), _i(free, cuda)
    for _ in range(2):                         # again: the same plan
        p = KV.kv_plan(_i(lens, cuda), _i(new, cuda), tb, fr, _i([n_free], cuda), rows)
        for got, w in zip((p.row_off, p.lens, p.slots, torch.stack([p.run_row, p.run_len], 1), p.n_free, p.refused, tb),
                          want[:4] + ([want[4]], [want[5]], want[6])):
            np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(w).reshape(got.shape))
        assert torch.equal(fr.cpu(), torch.as_tensor(free, dtype=torch.int32))


@pytest.mark.parametrize("lens,new", [([0], [1]), ([63], [1]), ([64], [1]), ([0], [64]), ([1], [64]), ([5], [0]), ([0, 0, 0], [0, 0, 0]),
                                      ([10, 64, 127, 0], [1, 1, 1, 200]), ([130], [1000]), ([7, 8, 9], [0, 300, 0])])
def test_plan_lengths(cuda, lens, new):
    _check_plan(cuda, lens, new, 40)


def test_plan_many(cuda):
    r = np.random.RandomState(1)
    _check_plan(cuda, r.randint(0, 900, 2500), r.randint(0, 3, 2500), 20)
    _check_plan(cuda, r.randint(0, 900, 1025), r.randint(0, 300, 1025), 30)
    _check_plan(cuda, np.zeros(1, int), [70000], 1200)


def test_plan_refuses_requests_and_serves_the_others(cuda):
    _check_plan(cuda, [0, 0, 60, 0], [65, 65, 3, 1], 10, n_free=3)             # the second does not fit the pool; the third needs no block
    _check_plan(cuda, [0, 100, 0], [65, 100, 64], 2)                           # the second passes the table's width
    _check_plan(cuda, [3, -1, 5, 7], [2, 2, -4, 1], 4)                         # bad lengths
    _check_plan(cuda, [0, 0, 0], [10, 10, 10], 4, rows=25)                     # rows that the matrices do not have
    _check_plan(cuda, [0, 0], [10, 10], 4, rows=40)                            # rows of nobody
    _check_plan(cuda, [0, 0], [1, 1], 4, n_free=0)
    _check_plan(cuda, [0, 0], [2 ** 30, 2 ** 30 + 5], 4, rows=10)              # row sums that pass 31 bits


def test_plan_of_no_request_and_no_row(cuda):
    e = _i(np.zeros(0), cuda)
    p = KV.kv_plan(e, e, torch.empty((0, 4), dtype=torch.int32, device=cuda), _i([3], cuda), _i([1], cuda), 0)
    assert p.row_off.tolist() == [0] and p.n_free.tolist() == [1] and p.refused.tolist() == [0]
    p = KV.kv_plan(e, e, torch.empty((0, 4), dtype=torch.int32, device=cuda), _i([3], cuda), _i([1], cuda), 7)
    assert p.slots.tolist() == [-1] * 7
    _check_plan(cuda, [5, 6], [0, 0], 4, rows=0)


def test_release(cuda):
    lens, table = _i([130, 0, 64, 1], cuda), _i([[5, 6, 7], [-1] * 3, [9, -1, -1], [2, -1, -1]], cuda)
    free, n_free = _i([100, 101, 0, 0, 0, 0, 0, 0], cuda), _i([2], cuda)
    KV.kv_release(_i([1, 1, 0, 1], cuda), lens, table, free, n_free)
    assert lens.tolist() == [0, 0, 64, 0] and n_free.tolist() == [6] and free.tolist()[:6] == [100, 101, 5, 6, 7, 2]
    KV.kv_release(_i([1, 1, 0, 1], cuda), lens, table, free, n_free)           # again: nothing left to give
    assert n_free.tolist() == [6]
    lens2, free2, nf2 = _i([64 * 3] * 3000, cuda), _i(np.zeros(8000), cuda), _i([10], cuda)
    KV.kv_release(_i(np.ones(3000), cuda), lens2, _i(np.arange(9000).reshape(3000, 3), cuda), free2, nf2)      # more than the stack holds
    assert nf2.tolist() == [8000] and free2.tolist()[10:] == list(range(7990))


# ------------------------------------------------------------------------------------------------ append / read
def _place(t):
    return 16 * ((t // 4) % 4) + 4 * (t // 16) + t % 4


def _e4m3(x):
    """nearest of the 8-bit values; past the largest (infinities too): +-448; NaN stays"""
    a = np.minimum(np.abs(x), 448.0)
    with np.errstate(divide="ignore"):
        e = np.maximum(np.floor(np.log2(np.maximum(a, 1e-300))), -6)
    step = 2.0 ** (e - 3)
    return np.where(np.isnan(x), np.nan, np.sign(x) * np.minimum(np.rint(a / step) * step, 448.0))


class Host:
    """The cache as numbers: values [blocks, Hkv, 64, dh] in units of the scale, and the scales."""

    def __init__(self, n, Hkv, dh):
        self.val = [np.zeros((n, Hkv, BS, dh)) for _ in range(2)]
        self.scale = [np.ones((n, Hkv)) for _ in range(2)]

    def append(self, rows, slots, runs):
        for w in range(2):
            val, sc = self.val[w], self.scale[w]
            x = rows[w].double().numpy().reshape(len(slots), *val.shape[1:2], -1)
            for row, n in runs:
                if row < 0:
                    continue
                blk, first = divmod(int(slots[row]), BS)
                for h in range(val.shape[1]):
                    y = x[row:row + n, h]
                    top = np.abs(y[np.isfinite(y)]).max(initial=0.0)
                    s = 2.0 ** -100
                    while top > 448 * s:
                        s *= 2
                    if first:
                        s = max(s, sc[blk, h])
                        val[blk, h, :first] = _e4m3(val[blk, h, :first] * (sc[blk, h] / s))
                    val[blk, h, first:first + n] = _e4m3(y / s)
                    sc[blk, h] = s


def _same(got, want):
    got = got.cpu().to(F64).numpy()
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("Hkv,dh", [(1, 16), (3, 48), (4, 80), (2, 128), (8, 64)])
def test_append_and_read(cuda, Hkv, dh):
    """steps of one token, of a few and of several blocks, amplitudes that make the scales grow and subnormals appear"""
    r = np.random.RandomState(dh)
    g = torch.Generator().manual_seed(dh)
    n, width = 5, 8
    cache, host = KV.KVCache.empty(n * width, Hkv, dh, cuda), Host(n * width, Hkv, dh)
    lens, free, n_free = _i(np.zeros(n), cuda), _i(r.permutation(n * width), cuda), _i([n * width], cuda)
    table = torch.full((n, width), -1, dtype=torch.int32, device=cuda)
    for step, (new, amp) in enumerate([([70, 1, 0, 64, 33], 1.0), ([1, 1, 1, 1, 1], 8.0), ([1, 2, 0, 63, 100], 0.001), ([1, 1, 1, 1, 1], 5000.0),
                                       ([5, 130, 1, 1, 0], 1e-30), ([1, 1, 1, 1, 1], 1e30)]):
        rows = sum(new)
        plan = KV.kv_plan(lens, _i(new, cuda), table, free, n_free, rows)
        wide = torch.randn((rows, Hkv * dh + 16), generator=g) * amp * torch.exp2(torch.randint(-9, 3, (rows, 1), generator=g).float())
        kr, vr = wide[:, :Hkv * dh].to(BF), wide.flip(0)[:, 16:].to(BF).contiguous()
        dev = wide.to(BF).to(cuda)
        KV.kv_append(cache, dev[:, :Hkv * dh], vr.to(cuda), plan)
        host.append((kr, vr), plan.slots.cpu().numpy(), torch.stack([plan.run_row, plan.run_len], 1).cpu().numpy())
        lens, n_free = plan.lens, plan.n_free
        held = [(t.tolist(), int(L)) for t, L in zip(table.cpu(), lens.cpu())]
        slots = np.array([t[p // BS] * BS + p % BS for t, L in held for p in range(L)] + [-1, n * width * BS, 2 ** 31 - 1])
        k, v = KV.kv_read(cache, _i(slots, cuda))
        for got, w in ((k, 0), (v, 1)):
            want = np.stack([host.val[w][s // BS, :, s % BS] * host.scale[w][s // BS][:, None] for s in slots[:-3]]).reshape(len(slots) - 3, -1)
            _same(got[:-3], want)
            assert (got[-3:] == 0).all()
        _same(cache.k_scale, host.scale[0])
        # (a second append of the same rows changes nothing)
        before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
        KV.kv_append(cache, dev[:, :Hkv * dh], vr.to(cuda), plan)
        for a, b in zip(before, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
            assert torch.equal(a, b)


def test_append_of_non_finite_values_and_zeros(cuda):
    cache, host = KV.KVCache.empty(2, 1, 16, cuda), Host(2, 1, 16)
    x = torch.linspace(-3, 3, 66 * 16).reshape(66, 16).to(BF)
    x[0, 0], x[1, 1], x[2, 2], x[65] = float("inf"), -float("inf"), float("nan"), 0
    plan = KV.kv_plan(_i([0], cuda), _i([66], cuda), _i([[-1, -1]], cuda), _i([1, 0], cuda), _i([2], cuda), 66)
    KV.kv_append(cache, x.to(cuda), -x.to(cuda), plan)
    host.append((x, -x), plan.slots.cpu().numpy(), torch.stack([plan.run_row, plan.run_len], 1).cpu().numpy())
    k, v = KV.kv_read(cache, plan.slots)
    for got, w in ((k, 0), (v, 1)):
        _same(got, np.stack([host.val[w][s // BS, :, s % BS] * host.scale[w][s // BS][:, None] for s in plan.slots.tolist()]).reshape(66, 16))


def test_append_leaves_other_blocks(cuda):
    """refused requests, rows of nobody and runs outside the pool write nothing"""
    cache = KV.KVCache.empty(4, 2, 32, cuda)
    cache.k.view(torch.uint8).fill_(77), cache.v.view(torch.uint8).fill_(77)
    rows = torch.ones((9, 64), dtype=BF, device=cuda)
    plan = KV.kv_plan(_i([0, 0], cuda), _i([3, 3], cuda), _i([[-1], [-1]], cuda), _i([2], cuda), _i([1], cuda), 9)
    assert plan.slots.tolist() == [128, 129, 130] + [-1] * 6 and plan.refused.tolist() == [1]
    KV.kv_append(cache, rows, rows, plan)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    place = torch.tensor([_place(t) for t in range(3)], device=cuda)
    assert (k[[0, 1, 3]] == 77).all() and (v[[0, 1, 3]] == 77).all() and (k[2, :, 3:] == 77).all()
    rest = torch.ones(BS, dtype=torch.bool, device=cuda)
    rest[place] = False
    assert (v[2][..., rest] == 77).all() and (k[2, :, :3] != 77).all() and (v[2][..., place] != 77).all()
    bad = plan._replace(slots=_i([4 * BS] * 9, cuda))
    KV.kv_append(cache, rows, rows, bad)
    assert (k[[0, 1, 3]] == 77).all()


# ------------------------------------------------------------------------------------------------ attention
def _cache_of(cuda, lens, Hkv, dh, seed, width=None, spare=2, amp=1.0):
    """a cache holding random values for requests of these lengths, blocks in random order, never written places NaN"""
    g = torch.Generator().manual_seed(seed)
    have = [-(-L // BS) for L in lens]
    n_blocks = sum(have) + spare
    width = max(have + [1]) if width is None else width
    ids = torch.randperm(n_blocks, generator=g).tolist()
    table, at = np.full((len(lens), width), n_blocks + 3), 0
    k = torch.full((n_blocks, Hkv, BS, dh), float("nan"))
    v = torch.full((n_blocks, Hkv, BS, dh), float("nan"))
    ks, vs = (torch.exp2(torch.randint(-9, -6, (n_blocks, Hkv), generator=g).float()) for _ in range(2))
    for r, L in enumerate(lens):
        for j in range(have[r]):
            b = ids[at]
            at += 1
            table[r, j] = b
            n = min(BS, L - j * BS)
            k[b, :, :n] = (torch.randn((Hkv, n, dh), generator=g) * 100 * amp).clamp(-448, 448)
            v[b, :, :n] = (torch.randn((Hkv, n, dh), generator=g) * 100).clamp(-448, 448)
    k, v = k.to(KV.F8), v.to(KV.F8)
    order = torch.tensor([_place(t) for t in range(BS)])
    vt = torch.empty((n_blocks, Hkv, dh, BS), dtype=torch.uint8)
    vt[..., order] = v.view(torch.uint8).transpose(-1, -2)
    cache = KV.KVCache(k.to(cuda), vt.view(KV.F8).to(cuda), ks.to(cuda), vs.to(cuda))
    dense = []
    for r, L in enumerate(lens):
        b = torch.as_tensor(table[r, :have[r]], dtype=torch.long)
        dense.append(tuple((x[b].double() * s[b].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, dh)[:, :L] for x, s in ((k, ks), (v, vs))))
    return cache, _i(table, cuda), dense


def _attn_check(cuda, lens, m, H, Hkv, dh, causal=True, cap=0.0, slopes=None, seed=0, width=None, max_len=None, extra=0, max_q=None, amp=1.0, scale=None):
    g = torch.Generator().manual_seed(seed + 1)
    cache, table, dense = _cache_of(cuda, lens, Hkv, dh, seed, width, amp=amp)
    off = np.concatenate([[0], np.cumsum(m)])
    q = torch.randn((int(off[-1]) + extra, H * dh), generator=g).to(BF)
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32)
    out = torch.full_like(q, 7.0).to(cuda)
    got, lse = KV.kv_attn(cache, q.to(cuda), table, _i(lens, cuda), _i(off, cuda), H, max(m) if max_q is None else max_q, max_len, causal=causal, cap=cap,
                          slopes=None if sl is None else sl.to(cuda), scale=scale, out=out, want_lse=True)
    assert got is out and (out[off[-1]:] == 7.0).all()
    sc = dh ** -0.5 if scale is None else scale
    for r, L in enumerate(lens):
        if not m[r]:
            continue
        rs = slice(int(off[r]), int(off[r + 1]))
        pos = (L - m[r] + torch.arange(m[r])) if causal else torch.full((m[r],), L)
        dist = pos[:, None] - torch.arange(L)[None]
        ok = dist >= 0 if causal else torch.ones((m[r], L), dtype=torch.bool)
        for h in range(H):
            c, hk = slice(h * dh, h * dh + dh), h // (H // Hkv)
            if L == 0:
                assert (got[rs, c] == 0).all() and (lse[rs, h] == -np.inf).all()
                continue
            ref = A.head(q[rs, c], dense[r][0][hk], dense[r][1][hk], ok, dist, sc, cap, None if sl is None else sl[h].double(), BF)
            A.close(got[rs, c], ref["out"], ref["out_tol"], "out of request %d head %d" % (r, h))
            A.close(lse[rs, h], ref["lse"], ref["lse_tol"], "lse")


@pytest.mark.parametrize("dh", [16, 32, 48, 64, 80, 96, 112, 128])
def test_attention_head_sizes(cuda, dh):
    _attn_check(cuda, [130, 1, 64, 200], [1, 1, 1, 1], 4, 2, dh)
    _attn_check(cuda, [130, 40, 64, 200], [3, 40, 1, 20], 2, 2, dh)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,m", [([1], [1]), ([63, 64, 65], [1, 1, 1]), ([127, 128, 129], [1, 2, 3]), ([0, 5], [1, 1]), ([10, 20], [0, 2]),
                                    ([70], [70]), ([300], [33]), ([3000, 1, 700], [1, 1, 1]), ([2], [5]), ([500, 66], [100, 17])])
def test_attention_lengths(cuda, lens, m, causal):
    """row counts over the request's length: the first rows of a causal step see nothing"""
    _attn_check(cuda, lens, m, 2, 1, 32, causal=causal)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (8, 1), (16, 2), (6, 2), (24, 1), (40, 1), (5, 1)])
@pytest.mark.parametrize("m", [1, 3])
def test_attention_shared_heads(cuda, H, Hkv, m):
    _attn_check(cuda, [150, 90], [m, m], H, Hkv, 64, slopes=[0.5 / (h + 1) for h in range(H)])


@pytest.mark.parametrize("kw", [dict(cap=5.0), dict(cap=20.0, slopes=[0.1, 0.0, 1.0, 0.01]), dict(slopes=[2.0, 0.0, -0.001, 0.3], causal=False),
                                dict(cap=0.5, causal=False), dict(scale=1.0, amp=2.0)])
def test_attention_shaped_scores(cuda, kw):
    _attn_check(cuda, [200, 65], [1, 4], 4, 2, 80, **kw)
    _attn_check(cuda, [200, 65], [30, 64], 4, 2, 80, **kw)


@pytest.mark.parametrize("m", [1, 20])
def test_attention_over_long_caches(cuda, m):
    """the length split over workgroups and joined; requests that end in the first piece beside it"""
    _attn_check(cuda, [20000, 3, 700], [m, 1, m], 4, 2, 64)
    _attn_check(cuda, [9000], [m], 2, 1, 128, slopes=[0.001, 0.0], causal=False)


def test_attention_launch_bounds(cuda):
    """bounds over the real sizes, a table wider than the lengths, rows of nobody left as they were"""
    _attn_check(cuda, [100, 30], [2, 1], 4, 2, 32, width=200, extra=3, max_q=64)
    _attn_check(cuda, [100, 30], [2, 1], 4, 2, 32, width=300, max_len=130, extra=1)


def test_attention_of_blocks_outside_the_pool(cuda):
    """a table entry outside the pool hides its tokens"""
    cache, table, dense = _cache_of(cuda, [200], 1, 32, 5)
    q = torch.randn((1, 32), generator=torch.Generator().manual_seed(3)).to(BF)
    for bad in (-1, cache.n_blocks, 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = bad
        out = KV.kv_attn(cache, q.to(cuda), t, _i([200], cuda), _i([0, 1], cuda), 1, 1)
        ok = torch.ones((1, 200), dtype=torch.bool)
        ok[0, 64:128] = False
        ref = A.head(q, dense[0][0][0], dense[0][1][0], ok, 199 - torch.arange(200)[None], 32 ** -0.5, 0.0, None, BF)
        A.close(out, ref["out"], ref["out_tol"], "out")


@pytest.mark.parametrize("m", [8, 40])
def test_stored_nan_reaches_the_rows_that_see_it(cuda, m):
    """NaN stored for the step's last token: earlier rows of the step are not touched by it"""
    cache, table, dense = _cache_of(cuda, [150], 1, 32, 6)
    blk = int(table[0, 149 // BS])
    cache.k.view(torch.uint8)[blk, 0, 149 % BS] = 0x7F
    cache.v.view(torch.uint8)[blk, 0, :, _place(149 % BS)] = 0x7F
    q = torch.randn((m, 32), generator=torch.Generator().manual_seed(3)).to(BF)
    out = KV.kv_attn(cache, q.to(cuda), table, _i([150], cuda), _i([0, m], cuda), 1, m)
    dist = 150 - m + torch.arange(m)[:, None] - torch.arange(150)[None]
    ref = A.head(q, dense[0][0][0], dense[0][1][0], dist >= 0, dist, 32 ** -0.5, 0.0, None, BF)
    A.close(out[:-1], ref["out"][:-1], ref["out_tol"][:-1], "out")
    assert out[-1].isnan().all()


def test_strides_of_rows(cuda):
    cache, table, _ = _cache_of(cuda, [100, 70], 2, 32, 7)
    wide = torch.randn((2, 64 + 64 + 8), generator=torch.Generator().manual_seed(3)).to(BF).to(cuda)
    q = wide[:, 64:128]
    args = (table, _i([100, 70], cuda), _i([0, 1, 2], cuda), 2, 1)
    a = KV.kv_attn(cache, q, *args)
    buf = torch.zeros((2, 80), dtype=BF, device=cuda)
    KV.kv_attn(cache, q.contiguous(), *args, out=buf[:, 8:72])
    assert torch.equal(a, buf[:, 8:72]) and (buf[:, :8] == 0).all() and (buf[:, 72:] == 0).all()
    with pytest.raises(ValueError, match="aligned"):
        KV.kv_attn(cache, wide[:, 1:65], *args)


# ------------------------------------------------------------------------------------------------ together
def test_a_serving_loop(cuda):
    """fill, steps of one event, a request that leaves and one that comes, against attention over the values that the cache holds; the
    same step captured in a graph and replayed equals the eager one"""
    n, H, Hkv, dh, width = 4, 8, 2, 64, 6
    g = torch.Generator().manual_seed(2)
    cache, host = KV.KVCache.empty(14, Hkv, dh, cuda), Host(14, Hkv, dh)
    lens, free, n_free = _i(np.zeros(n), cuda), _i(np.arange(14), cuda), _i([14], cuda)
    table = torch.full((n, width), -1, dtype=torch.int32, device=cuda)
    for step, new in enumerate([[100, 64, 3, 0], [1, 1, 1, 1], [1, 1, 1, 1], "release", [50, 1, 1, 1], [1, 1, 1, 1]]):
        if new == "release":
            KV.kv_release(_i([1, 0, 0, 0], cuda), lens, table, free, n_free)
            continue
        rows = sum(new)
        kr, vr = (torch.randn((rows, Hkv * dh), generator=g).to(BF) for _ in range(2))
        q = torch.randn((rows, H * dh), generator=g).to(BF)
        kd, vd, qd, nd = kr.to(cuda), vr.to(cuda), q.to(cuda), _i(new, cuda)

        def go():
            p = KV.kv_plan(lens, nd, table, free, n_free, rows)
            KV.kv_append(cache, kd, vd, p)
            return p, KV.kv_attn(cache, qd, table, p.lens, p.row_off, H, 100)

        plan, out = go()
        eager = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan2, out2 = go()
        for _ in range(3):
            out2.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(eager, out2) and all(torch.equal(a, b) for a, b in zip(plan, plan2))
            torch.cuda.synchronize()
        host.append((kr, vr), plan.slots.cpu().numpy(), torch.stack([plan.run_row, plan.run_len], 1).cpu().numpy())
        assert plan.refused.tolist() == [0]
        for r in range(n):
            m, L, o = new[r], int(plan.lens[r]), int(plan.row_off[r])
            if not m:
                continue
            tb = table[r, :-(-L // BS)].tolist()
            kk, vv = (torch.as_tensor(np.concatenate([host.val[w][b] * host.scale[w][b][:, None, None] for b in tb], 1)[:, :L]) for w in range(2))
            dist = L - m + torch.arange(m)[:, None] - torch.arange(L)[None]
            for h in range(H):
                ref = A.head(q[o:o + m, h * dh:(h + 1) * dh], kk[h // 4], vv[h // 4], dist >= 0, dist, dh ** -0.5, 0.0, None, BF)
                A.close(eager[o:o + m, h * dh:(h + 1) * dh], ref["out"], ref["out_tol"], "step %d request %d" % (step, r))
        lens, n_free = plan.lens.clone(), plan.n_free.clone()
    assert sorted(free[:int(n_free)].tolist() + [b for t, L in zip(table.tolist(), lens.tolist()) for b in t[:-(-L // BS)]]) == list(range(14))


def test_another_stream(cuda):
    cache, table, _ = _cache_of(cuda, [500, 70], 2, 32, 8)
    q = torch.randn((2, 128), generator=torch.Generator().manual_seed(3)).to(BF).to(cuda)
    args = (table, _i([500, 70], cuda), _i([0, 1, 2], cuda), 4, 1)
    a = KV.kv_attn(cache, q, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = KV.kv_attn(cache, q, *args)
    side.synchronize()
    assert torch.equal(a, b)


def test_two_graphs_two_streams_and_one_history_twice(cuda):
    """split lengths: two captured calls and an eager one on a side stream do not share a workspace; two requests that name the same blocks
    get the same rows"""
    lens, H = [9000, 9000, 64], 4
    cache, table, _ = _cache_of(cuda, lens, 2, 32, 8)
    table[1] = table[0]
    g = torch.Generator().manual_seed(3)
    one = torch.randn((2, H * 32), generator=g).to(BF)
    q1 = torch.cat([one, one, one]).to(cuda)
    q2 = torch.randn((6, H * 32), generator=g).to(BF).to(cuda)
    args = (table, _i(lens, cuda), _i([0, 2, 4, 6], cuda), H, 2)
    w1, w2 = KV.kv_attn(cache, q1, *args), KV.kv_attn(cache, q2, *args)
    assert torch.equal(w1[:2], w1[2:4])
    torch.cuda.synchronize()
    graphs = []
    for q in (q1, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, KV.kv_attn(cache, q, *args)))
    side = torch.cuda.Stream()
    for _ in range(3):
        for _g, o in graphs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            e = KV.kv_attn(cache, q2, *args)
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], w1) and torch.equal(graphs[1][1], w2) and torch.equal(e, w2)


def test_rows_of_a_refused_request(cuda):
    """nothing is stored for them, the others are served, and their attention reads only what they held"""
    cache = KV.KVCache.empty(2, 1, 32, cuda)
    lens, table = _i([0, 0], cuda), torch.full((2, 2), -1, dtype=torch.int32, device=cuda)
    free, n_free = _i([0, 1], cuda), _i([2], cuda)
    x = torch.randn((100, 32), generator=torch.Generator().manual_seed(1)).to(BF).to(cuda)
    plan = KV.kv_plan(lens, _i([30, 70], cuda), table, free, n_free, 100)        # one block for the first, two wanted by the second, one left
    assert plan.refused.tolist() == [1] and plan.lens.tolist() == [30, 0] and plan.n_free.tolist() == [1] and (plan.slots[30:] == -1).all()
    KV.kv_append(cache, x, x, plan)
    out, lse = KV.kv_attn(cache, x, table, plan.lens, plan.row_off, 1, 70, want_lse=True)
    assert (out[30:] == 0).all() and (lse[30:] == -np.inf).all() and (out[:30] != 0).any(-1).all()


def test_refusals_of_device_arguments(cuda):
    cache, table, _ = _cache_of(cuda, [70], 2, 32, 8)
    q = torch.zeros((3, 128), dtype=BF, device=cuda)
    lens, off = _i([70], cuda), _i([0, 3], cuda)
    ok = dict(q=q, table=table, lens=lens, row_off=off, H=4, max_q=3)
    for kw, msg in ((dict(H=3), "share"), (dict(q=q.float()), "bf16"), (dict(q=q[:, :64]), "bf16 rows"), (dict(table=table[0]), "table"),
                    (dict(lens=lens.long()), "lens"), (dict(row_off=lens), "row_off"), (dict(max_q=-1), "negative"), (dict(scale=0.0), "scale"),
                    (dict(cap=float("nan")), "scale"), (dict(out=q), "not be q"), (dict(out=q[:2].clone()), "out must be"),
                    (dict(slopes=torch.zeros(3, device=cuda)), "slopes"), (dict(max_len=-1), "negative"), (dict(table=table.cpu()), "table")):
        with pytest.raises(ValueError, match=msg):
            KV.kv_attn(cache, **{**ok, **kw})
    one = KV.kv_attn(cache, **ok)
    assert torch.equal(one, KV.kv_attn(cache, **{**ok, "max_q": 2 ** 40, "max_len": 2 ** 40}))   # bounds that say nothing
    n, i = _i([1], cuda), _i([3], cuda)
    for a in ((lens, i, table[0], n, n, 3), (lens[None], i, table, n, n, 3), (lens, i, table, n, n, -1), (lens, i, table, n, n.cpu(), 3)):
        with pytest.raises(ValueError):
            KV.kv_plan(*a)
    plan = KV.kv_plan(lens, i, table, n, n, 3)
    x = torch.zeros((3, 64), dtype=BF, device=cuda)
    for k, v in ((x[:2], x), (x, x[:, :32]), (x.float(), x), (x.cpu(), x)):
        with pytest.raises(ValueError):
            KV.kv_append(cache, k, v, plan)
    with pytest.raises(ValueError):
        KV.kv_read(cache, plan.slots.long())
    c = cache
    for a in ((c.k[:, :1], c.v, c.k_scale, c.v_scale), (c.k, c.v, c.k_scale[:1], c.v_scale), (c.k.view(torch.uint8), c.v, c.k_scale, c.v_scale),
              (c.k, c.v, c.k_scale.double(), c.v_scale), (c.k.cpu(), c.v.cpu(), c.k_scale.cpu(), c.v_scale.cpu())):
        with pytest.raises(ValueError):
            KV.KVCache(*a)


@pytest.mark.parametrize("m", [1, 30])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30])
def test_caps_far_over_the_scores(cuda, cap, m):
    """the bounds of scores without a cap hold: a cap of 1e4 and more changes scores of about 8 by less than 1e-6 of them"""
    lens, H, Hkv, dh = [200, 65], 4, 2, 80
    cache, table, dense = _cache_of(cuda, lens, Hkv, dh, 23)
    q = torch.randn((2 * m, H * dh), generator=torch.Generator().manual_seed(24)).to(BF)
    got, lse = KV.kv_attn(cache, q.to(cuda), table, _i(lens, cuda), _i([0, m, 2 * m], cuda), H, m, causal=False, cap=cap, want_lse=True)
    for r, L in enumerate(lens):
        ok, dist = torch.ones((m, L), dtype=torch.bool), torch.zeros((m, L), dtype=torch.int64)
        for h in range(H):
            c, hk = slice(h * dh, h * dh + dh), h // (H // Hkv)
            ref = A.head(q[r * m:r * m + m, c], dense[r][0][hk], dense[r][1][hk], ok, dist, dh ** -0.5, 0.0, None, BF)
            A.close(got[r * m:r * m + m, c], ref["out"], ref["out_tol"], "out")
            A.close(lse[r * m:r * m + m, h], ref["lse"], ref["lse_tol"], "lse")


@pytest.mark.parametrize("cap", [0.5, 30.0, 1e3, 1e6, 9e37])
def test_capped_scores_keep_their_bits(cuda, cap):
    """One cached token: lse is the score, whose dot product is exact; what is off is the tanh form and three roundings.  Caps of at most 64 take
    cap (1 - 2 r): r, at most 1, comes from a sum (2^-24), v_rcp_f32 (2^-23) and a power (v_exp_f32 and its argument, 2^-23 each of r (1 - r) <= 1/4
    where |a| is small and less where the argument is long): under 2^-22.4, doubled and rounded: 2^-21 of the cap.  Larger ones: 2^-20 of the value."""
    cache = KV.KVCache.empty(1, 1, 16, cuda)
    one = torch.zeros((1, 16), dtype=BF, device=cuda)
    one[0, 3] = 1.0
    plan = KV.kv_plan(_i([0], cuda), _i([1], cuda), _i([[-1]], cuda), _i([0], cuda), _i([1], cuda), 1)
    KV.kv_append(cache, one, one, plan)
    mags = torch.logspace(-6, 3, 301, dtype=F64).to(BF)
    if cap < 1e4:
        mags = torch.cat([mags, (torch.linspace(0.01, 4, 400, dtype=F64) * cap).to(BF)])
    x = torch.cat([mags, -mags])
    q = torch.zeros((len(x), 16), dtype=BF)
    q[:, 3] = x
    _, lse = KV.kv_attn(cache, q.to(cuda), _i([[0]], cuda), plan.lens, _i([0, len(x)], cuda), 1, len(x), causal=False, scale=1.0, cap=cap, want_lse=True)
    want = cap * torch.tanh(x.double() / cap)
    assert ((lse[:, 0].cpu().double() - want).abs() <= 2.0 ** -19 * want.abs() + (2.0 ** -21 * cap if cap <= 64 else 0.0)).all()


@pytest.mark.parametrize("m,max_q,L,max_len,causal", [(40, 16, 200, None, True), (40, 33, 200, None, True), (5, 1, 70, None, True), (3, 3, 300, 128, True),
                                                      (64, 10, 300, 256, True), (3, 2, 300, 100, False), (9, 4, 5, None, True)])
def test_rows_and_tokens_past_the_bounds_are_cut_where_they_stand(cuda, m, max_q, L, max_len, causal):
    """A replayed graph's requests may outgrow max_q / max_len: rows and tokens past them are cut, and row i still stands at lens - m + i, so it sees
    no token of the rows behind it, and its distances are those of the whole request"""
    H, Hkv, dh = 4, 2, 32
    cache, table, dense = _cache_of(cuda, [L], Hkv, dh, 21)
    q = torch.randn((m, H * dh), generator=torch.Generator().manual_seed(22)).to(BF)
    sl = torch.tensor([0.05, 0.0, 0.2, 0.01])
    out = torch.full_like(q, 7.0).to(cuda)
    got, lse = KV.kv_attn(cache, q.to(cuda), table, _i([L], cuda), _i([0, m], cuda), H, max_q, max_len, causal=causal, slopes=sl.to(cuda), out=out, want_lse=True)
    n, most = min(m, max_q), L if max_len is None else min(L, max_len)
    pos = L - m + torch.arange(n) if causal else torch.full((n,), L)
    dist = pos[:, None] - torch.arange(most)[None]
    ok = dist >= 0 if causal else torch.ones((n, most), dtype=torch.bool)
    for h in range(H):
        c, hk = slice(h * dh, h * dh + dh), h // (H // Hkv)
        ref = A.head(q[:n, c], dense[0][0][hk][:most], dense[0][1][hk][:most], ok, dist, dh ** -0.5, 0.0, sl[h].double(), BF)
        A.close(got[:n, c], ref["out"], ref["out_tol"], "out of head %d" % h)
        A.close(lse[:n, h], ref["lse"], ref["lse_tol"], "lse of head %d" % h)
    assert (got[n:] == 7.0).all()


def test_rows_of_nobody_are_zero(cuda):
    """without `out`, rows that belong to no request, rows past max_q and whole calls without requests give zeros (lse -inf), not what the memory
    held; with `out` they stay as they were"""
    H, Hkv, dh, rows = 4, 2, 32, 50
    lens, m = [100, 30, 70], [7, 0, 12]
    cache, table, dense = _cache_of(cuda, lens, Hkv, dh, 25)
    q = torch.randn((rows, H * dh), generator=torch.Generator().manual_seed(26)).to(BF).to(cuda)
    lens, off = _i(lens, cuda), _i([3, 10, 10, 22], cuda)                         # rows 0 .. 2 and 22 .. 49 are nobody's

    def poison():
        for shape, dt in (((rows, H * dh), BF), ((rows, H), torch.float32)):
            bad = torch.full(shape, float("nan"), dtype=dt, device=cuda)
            del bad                                                              # (the allocator hands the same memory out again)

    poison()
    want, wl = KV.kv_attn(cache, q, table, lens, off, H, 12, out=torch.full_like(q, 7.0), want_lse=True)
    assert (want[:3] == 7.0).all() and (want[22:] == 7.0).all() and (wl[:3] == -np.inf).all() and (wl[22:] == -np.inf).all()
    for max_q in (12, 5, 40):
        poison()
        got, lse = KV.kv_attn(cache, q, table, lens, off, H, max_q, want_lse=True)
        held = torch.zeros(rows, dtype=torch.bool, device=cuda)
        for a, b in ((3, 10), (10, 22)):
            held[a:min(b, a + max_q)] = True
        assert torch.equal(got[held], want[held]) and torch.equal(lse[held], wl[held])
        assert (got[~held] == 0).all() and (lse[~held] == -np.inf).all()
    for kw in (dict(max_q=0), dict(max_q=12, table=table[:0], lens=lens[:0], row_off=off[:1])):
        poison()
        a = {**dict(table=table, lens=lens, row_off=off, max_q=12), **kw}
        got, lse = KV.kv_attn(cache, q, a["table"], a["lens"], a["row_off"], H, a["max_q"], want_lse=True)
        assert (got == 0).all() and (lse == -np.inf).all()
    big, tb, _d = _cache_of(cuda, [5000, 1], Hkv, dh, 27)                         # the length split over workgroups and joined
    for max_q in (3, 2):
        poison()
        got, lse = KV.kv_attn(big, q, tb, _i([5000, 1], cuda), _i([1, 4, 6], cuda), H, max_q, want_lse=True)
        held = torch.zeros(rows, dtype=torch.bool, device=cuda)
        held[1:1 + max_q] = True
        held[4:6] = True
        assert (got[held] != 0).any(-1)[:max_q].all() and (got[~held] == 0).all() and (lse[~held] == -np.inf).all()


@pytest.mark.parametrize("m,L", [(1, 200), (20, 200), (40, 150), (2, 9000), (30, 9000)])
def test_stored_nan_of_single_dims(cuda, m, L):
    """NaN stored in single dims of V, of a token that all rows see and of the last one, which only the last row sees (also where the length is split
    and joined): those dims are NaN where they are seen, every other value holds its bound"""
    H, Hkv, dh = 4, 2, 80
    cache, table, dense = _cache_of(cuda, [L], Hkv, dh, 33)
    for pos, hk, dim in ((5, 0, 3), (5, 1, 79), (L - 1, 0, 64), (L - 1, 1, 0)):
        cache.v.view(torch.uint8)[int(table[0, pos // BS]), hk, dim, _place(pos % BS)] = 0x7F
    q = torch.randn((m, H * dh), generator=torch.Generator().manual_seed(34)).to(BF)
    got = KV.kv_attn(cache, q.to(cuda), table, _i([L], cuda), _i([0, m], cuda), H, m)
    dist = (L - m + torch.arange(m))[:, None] - torch.arange(L)[None]
    for h in range(H):
        hk, c = h // (H // Hkv), slice(h * dh, h * dh + dh)
        ref = A.head(q[:, c], dense[0][0][hk], dense[0][1][hk], dist >= 0, dist, dh ** -0.5, 0.0, None, BF)
        want = ref["out"].clone()
        want[:, 3 if hk == 0 else 79] = np.nan
        want[-1, 64 if hk == 0 else 0] = np.nan
        A.close(got[:, c], want, ref["out_tol"], "out of head %d" % h)


@pytest.mark.parametrize("dh", [16, 80, 128])
@pytest.mark.parametrize("cap", [64.0, 65.0, 400.0])
def test_caps_on_both_sides_of_the_short_form(cuda, cap, dh):
    """caps up to 64 take the short form, kernels of their own beyond: few rows and many, a length in pieces, scores that reach the cap"""
    _attn_check(cuda, [200, 65], [1, 4], 4, 2, dh, cap=cap, scale=4.0, slopes=[0.1, 0.0, 1.0, 0.01])
    _attn_check(cuda, [200, 65], [30, 64], 4, 2, dh, cap=cap, scale=4.0)
    _attn_check(cuda, [9000], [2], 2, 1, dh, cap=cap, causal=False)


def test_a_replay_with_other_rows_leaves_zeros_where_nobody_is(cuda):
    """one captured step, replayed with more, fewer and no rows of each request, and with other lengths: every replay as the eager call, the rest zero"""
    H, Hkv, dh, rows = 4, 2, 64, 24
    cache, table, _ = _cache_of(cuda, [300, 70, 129], Hkv, dh, 61)
    q = torch.randn((rows, H * dh), generator=torch.Generator().manual_seed(62)).to(BF).to(cuda)
    lens, off = _i([300, 70, 129], cuda), _i([0, 4, 8, 12], cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        KV.kv_attn(cache, q, table, lens, off, H, 8, want_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = KV.kv_attn(cache, q, table, lens, off, H, 8, want_lse=True)
    for L, o in (([300, 70, 129], [0, 8, 16, 24]), ([10, 70, 64], [2, 2, 7, 9]), ([300, 1, 0], [0, 0, 0, 0]), ([299, 69, 100], [5, 6, 7, 20])):
        lens.copy_(_i(L, cuda))
        off.copy_(_i(o, cuda))
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        want, wl = KV.kv_attn(cache, q, table, lens, off, H, 8, want_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wl)
        held = torch.zeros(rows, dtype=torch.bool, device=cuda)
        for a, b in zip(o, o[1:]):
            held[a:min(b, a + 8)] = True
        assert (out[~held] == 0).all() and (lse[~held] == -np.inf).all()
