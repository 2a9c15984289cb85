"""Serving from kept histories: CandidateScorer.remember / logits_of against the same decoder over the values that the cache holds, and
HistoryCache's bookkeeping."""
import numpy as np
import pytest
import torch

from cikm2020_dmt_amd import kv_cache as KV
from cikm2020_dmt_amd import ops
from cikm2020_dmt_amd import spec as S
from cikm2020_dmt_amd.data_feed.synthetic import make_batch
from cikm2020_dmt_amd.engine import AssembleFn, DeviceBatch, FeatureColumn, trans_prefix
from cikm2020_dmt_amd.serving import CandidateScorer, HistoryCache
from cikm2020_dmt_amd.train import Trainer

pytestmark = pytest.mark.gpu
ROWS = {"Sku": 3000, "Brand": 800, "Shopid": 900, "Cid3": 300, "Cid2": 50}


def _slots(table_row, n):
    pos = torch.arange(n, device=table_row.device)
    return (table_row[pos // 64] * 64 + pos % 64).to(torch.int32)


def _trainer(cuda, dtype=torch.bfloat16, **opt):
    sp = dict(S.scaled_spec(S.e64_spec(), ROWS), **opt)
    return sp, Trainer(sp, device=cuda, compute_dtype=dtype, init=True, dropout=False)


def _expected(sc, users, batch):
    """logits_of with the attention of the tiled request path over the rows that the cache holds for each candidate's user"""
    eng, spec = sc.engine, sc.spec
    d, H = spec["d_model"], spec["num_heads"]
    with torch.no_grad():
        tar, zbuf = eng.gather_pooled(batch)
        us = []
        for i, h in enumerate(sc.histories):
            y = eng.decoder_query(tar).unsqueeze(1)
            L = h.lens[torch.as_tensor(users, device=h.lens.device)].contiguous()
            T = int(L.max())
            for j, cache in enumerate(h.layers):
                blk = trans_prefix(i) + "num_blocks_%d/" % j
                a = blk + "vanilla_attention/"
                wl, bl, w = eng._lf(a + "qkv_kernel"), eng._lf(a + "qkv_bias"), eng._w(a + "qkv_kernel")
                q = ops.linear(y, wl[:, :d], bl[:d], eng._wslice(w, 0, d))
                pos = torch.arange(T, device=tar.device)
                slots = h.table[torch.as_tensor(users, device=tar.device)][:, pos // 64] * 64 + pos % 64
                k, v = KV.kv_read(cache, slots.to(torch.int32).reshape(-1).contiguous())
                kv = torch.cat([k, v], 1).reshape(len(users), T, 2 * d)
                s = ops.AttnFn.apply(q, kv, y, None, L, H, d, False, 0, 1.0, eng.kopts)
                s = ops.layer_norm(s, eng._lf(a + "ln/gamma"), eng._lf(a + "ln/beta"))
                y = eng.ff(s, blk + "positionwise_feedforward/")
            us.append(y.squeeze(1))
        z = AssembleFn.apply(zbuf, eng.plan.interest_off, d, *eng.interest_blocks(us, [tar] * len(us)))
        tasks = eng.expert_gate(z, z_is_engine_buffer=True)
        return [eng.build_tower(m, nm) for m, nm in zip(tasks, ("click", "order"))]


def _one_user_rows(sp, tr, seed, n):
    inputs, mask, label = make_batch(sp, n, seed=seed, lengths="ragged", weights="random")
    return tr.make_batch(inputs, mask, label)


@pytest.mark.parametrize("opt", [dict(), dict(num_blocks_decode=2)])
def test_candidates_of_remembered_users(cuda, opt):
    """several users at once, replaced and extended histories, users without candidates; tolerance: the bf16 one of the request path"""
    sp, tr = _trainer(cuda, **opt)
    sc = CandidateScorer(tr.engine)
    sc.keep_histories(9, 40)
    assert sc.remember([4, 0, 7, 2], _one_user_rows(sp, tr, 3, 4)) == 0
    assert sc.remember([7, 8], _one_user_rows(sp, tr, 4, 2)) == 0                # 7 again: replaced
    users = [0] * 5 + [2] * 1 + [7] * 33 + [8] * 2
    batch = _one_user_rows(sp, tr, 9, len(users))
    got, want = sc.logits_of(users, batch), _expected(sc, users, batch)
    for g, w in zip(got, want):
        assert torch.allclose(g.float(), w.float(), atol=4e-2, rtol=4e-2)
    for h in sc.histories:                                                        # every block is in one table or free
        held = [b for t, L in zip(h.table.tolist(), h.lens.tolist()) for b in t[:-(-L // 64)]]
        assert sorted(held + h.free[:int(h.n_free)].tolist()) == list(range(40))


def test_histories_follow_the_encoder(cuda):
    """the cached K / V are the decoder's projections of the encoded rows, each within half a step of e4m3 at its block's scale (2^-4 of the
    value, 2^-10 of the scale below the normal range)"""
    sp, tr = _trainer(cuda)
    eng, d = tr.engine, sp["d_model"]
    sc = CandidateScorer(eng)
    sc.keep_histories(3, 12)
    batch = _one_user_rows(sp, tr, 5, 3)
    users = [2, 0, 1]
    assert sc.remember(users, batch) == 0
    eng.packed_rows = False                                                       # [B, T, d] below
    with torch.no_grad():
        X, _t, _z = eng.gather(batch)
        for i, pairs in enumerate(sp["attention_embed_pairs"]):
            lens = batch.feats[pairs[-1][0]].lens
            kv = eng.memory_kv(eng.encode_prepared(X[i], lens, i), i, 0).float()
            h = sc.histories[i]
            for r, u in enumerate(users):
                L = int(lens[r])
                assert int(h.lens[u]) == L
                pos = torch.arange(L, device=cuda)
                slots = (h.table[u][pos // 64] * 64 + pos % 64).to(torch.int32)
                k, v = KV.kv_read(h.layers[0], slots)
                for got, want, sc_ in ((k, kv[r, :L, :d], h.layers[0].k_scale), (v, kv[r, :L, d:], h.layers[0].v_scale)):
                    step = sc_[(slots // 64).long()].repeat_interleave(d // sp["num_heads"], 1)
                    assert ((got.float() - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * step).all()


def test_no_room_and_refusals(cuda):
    sp, tr = _trainer(cuda)
    sc = CandidateScorer(tr.engine)
    sc.keep_histories(4, 2)
    assert sc.remember([0, 1, 2, 3], _one_user_rows(sp, tr, 5, 4)) == 6          # 2 blocks a sequence, 4 users of one block each, 3 sequences
    batch = _one_user_rows(sp, tr, 5, 2)
    with pytest.raises(RuntimeError, match="keep_histories"):
        CandidateScorer(tr.engine).logits_of([0, 0], batch)
    for bad in ([0, 0], [0], [0, 4], [-1, 0]):
        with pytest.raises(ValueError):
            sc.remember(bad, batch)
    for bad in ([1, 0], [0], [0, 4]):
        with pytest.raises(ValueError):
            sc.logits_of(bad, batch)
    with pytest.raises(ValueError, match="bf16"):
        CandidateScorer(_trainer(cuda, torch.float32)[1].engine).keep_histories(4, 2)
    with pytest.raises(ValueError, match="multiple of 16"):
        CandidateScorer(Trainer(S.scaled_spec(S.default_spec(), ROWS), device=cuda, compute_dtype=torch.bfloat16, dropout=False).engine).keep_histories(4, 2)
    with pytest.raises(ValueError):
        HistoryCache(0, 4, 64, 2, 32)
    h = HistoryCache(2, 4, 64, 2, 32, layers=2)
    x = torch.zeros((1, 64), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="2 layers"):
        h.append([(x, x)], torch.tensor([1, 0], dtype=torch.int32, device=cuda))


def test_a_cache_of_many_users(cuda):
    """attend for every place and for a few named ones (more places than one attention call takes): the same rows"""
    n, H, dh = 70000, 2, 32
    h = HistoryCache(n, 64, 100, H, dh, device=cuda)
    g = torch.Generator().manual_seed(4)
    new = torch.zeros(n, dtype=torch.int32)
    places = [3, 1500, 69999]
    new[places] = torch.tensor([100, 64, 1], dtype=torch.int32)
    k, v = (torch.randn((165, H * dh), generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    assert int(h.append([(k, v)], new.to(cuda)).refused) == 0
    at = torch.tensor(places, device=cuda)
    table, lens = h.of(at)
    assert lens.tolist() == [100, 64, 1] and (table[:, 0] >= 0).all() and h.max_len == 128
    q = torch.randn((3, H * dh), generator=g).to(torch.bfloat16).to(cuda)
    off = torch.arange(4, dtype=torch.int32, device=cuda)
    got = h.attend(0, q, off, H, 1, (table, lens), causal=False)
    for r, (a, b) in enumerate(((0, 100), (100, 164), (164, 165))):
        kk, vv = (x.float().reshape(-1, H, dh).transpose(0, 1) for x in KV.kv_read(h.layers[0], _slots(table[r], b - a)))
        p = torch.softmax((q[r].float().reshape(H, 1, dh) * kk).sum(-1) * dh ** -0.5, -1)
        want = (p[..., None] * vv).sum(1).reshape(-1)
        # weights and result are rounded once each: half a step of values of at most max |v|, twice
        assert (got[r].float() - want).abs().max() <= 2 * 2.0 ** -8 * float(vv.abs().max())
    with pytest.raises(Exception, match="65535"):
        h.attend(0, q, torch.zeros(n + 1, dtype=torch.int32, device=cuda), H, 1)
    h.drop((torch.arange(n) == 1500).to(torch.int32).to(cuda))
    assert h.of(at)[1].tolist() == [100, 0, 1] and int(h.n_free) == 64 - 4 + 1


def _emptied(batch, sp, rows):
    """the batch with empty histories: rows[i] have no event in sequence i"""
    for i, pairs in enumerate(sp["attention_embed_pairs"]):
        for uf, _item in pairs:
            c = batch.feats[uf]
            c.lens[torch.as_tensor(rows[i], dtype=torch.long, device=c.lens.device)] = 0
            c.lens_host[rows[i]] = 0
    return batch


def _row(batch, r, n):
    """row r of the batch n times over"""
    at = torch.full((n,), r, device=batch.dense.device)
    return DeviceBatch(n, {f: FeatureColumn(c.idx[at], c.wts[at] if c.wts is not None else None, c.lens[at], c.T) for f, c in batch.feats.items()},
                       batch.dense[at])


def test_an_empty_sequence_is_the_mean_of_its_padded_rows(cuda):
    """A user without events in a sequence: the model's attention gives every padded row the same weight, so what is kept is one row, the mean of
    K and of V over them, within the roundings (fp32 mean of bf16 rows to bf16: 2^-8 of the value; half a step of e4m3: 2^-4 of it, 2^-10 of the
    scale below the normal range)"""
    sp, tr = _trainer(cuda, num_blocks_decode=2)
    eng, d = tr.engine, sp["d_model"]
    sc = CandidateScorer(eng)
    sc.keep_histories(5, 12)
    batch = _emptied(_one_user_rows(sp, tr, 5, 4), sp, {0: [1], 1: [0, 1, 3], 2: [0, 1, 2, 3]})
    users = [4, 0, 1, 2]
    assert sc.remember(users, batch) == 0
    eng.packed_rows = False
    with torch.no_grad():
        X, _t, _z = eng.gather(batch)
        for i, pairs in enumerate(sp["attention_embed_pairs"]):
            lens = batch.feats[pairs[-1][0]].lens
            mem, h = eng.encode_prepared(X[i], lens, i), sc.histories[i]
            assert [int(h.lens[u]) for u in users] == [max(int(x), 1) for x in lens]
            for j, cache in enumerate(h.layers):
                mean = eng.memory_kv(mem, i, j).double().mean(1)
                for r, u in enumerate(users):
                    if int(lens[r]):
                        continue
                    slot = (h.table[u][:1] * 64).to(torch.int32)
                    k, v = KV.kv_read(cache, slot)
                    for got, want, scale in ((k, mean[r, :d], cache.k_scale), (v, mean[r, d:], cache.v_scale)):
                        step = scale[int(slot) // 64].repeat_interleave(d // sp["num_heads"])
                        assert ((got[0].double() - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + 2.0 ** -10 * step).all()


@pytest.mark.parametrize("opt", [dict(), dict(num_blocks_decode=2)])
def test_logits_of_users_with_empty_sequences(cuda, opt):
    """logits_of against logits, the request path that re-encodes the user: lengths of 0 in some sequences, in all, in none.  V is made the same
    for every row (its kernel 0, its bias of values that 8 bits hold), so that the cache rounds nothing that counts and every non-empty or
    empty attention gives that row: the tolerance is the bf16 one of the request path."""
    sp, tr = _trainer(cuda, **opt)
    state, rng = {}, np.random.default_rng(3)
    for name, arr in tr.store.dense_state_dict().items():
        if "vanilla_attention/dense_2/kernel" in name:
            state[name] = np.zeros_like(arr)
        elif "vanilla_attention/dense_2/bias" in name:
            state[name] = rng.integers(-14, 15, arr.shape) / 8.0                 # (14 / 8 = 1.75: four significant bits at most)
    tr.store.load_state(state)
    sc = CandidateScorer(tr.engine)
    sc.keep_histories(6, 24)
    hist = _emptied(_one_user_rows(sp, tr, 6, 5), sp, {0: [0, 2], 1: [2, 3], 2: [2, 4]})
    places = [0, 1, 3, 4, 5]
    assert sc.remember(places, hist) == 0
    for r, place in enumerate(places):
        batch = _row(hist, r, 3)
        for g, w in zip(sc.logits_of([place] * 3, batch), sc.logits(batch)):
            assert torch.allclose(g.float(), w.float(), atol=4e-2, rtol=4e-2), (r, g.flatten().tolist(), w.flatten().tolist())
