"""Serving path: score B candidate items for ONE user.

Mirrors /root/reference/DMT_code/saved_model/export_model.py:23-138 (online normalisation of the raw dense features,
sigmoid heads, weighted score) and model/inference_mlp.py:73-113 (`online_build_sparsetensor`: the user-side id features of
the request are tiled across the candidate batch and the ordinary predict graph runs on the tiled batch).

The reference re-encodes the user's behaviour sequences for every candidate row.  Here the three sequence encoders (self-
attention + FFN over [T, d]) and the K | V projections of their memories run ONCE per request; every candidate only pays for
its own embedding lookups, the single-query decoder attention against the shared memory (zero batch stride), MMoE and the
towers.  CandidateScorer.keep_histories holds the projected memories of many users between requests (HistoryCache, 8 bits), so
that candidates of several users are scored in one batch with no encoder in it.  Same numbers as Inference.inference(tiled batch, is_predict=True) -- checked in tests/test_gpu_serving.py.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence

import numpy as np
import torch

from .engine import AssembleFn, DeviceBatch, DMTEngine, FeatureColumn
from .kv_cache import BLOCK, KVCache, kv_append, kv_attn, kv_plan, kv_release


def normalisation_constants(mean: Sequence[float], std: Sequence[float]):
    """saved_model/preprocess.py:17-40 `vec_constant` (float64 there as well):
    c = mean*std / (3 (std+eps)^2) + mean*std / (std+eps) - mean."""
    m, s = np.asarray(mean, dtype=np.float64), np.asarray(std, dtype=np.float64)
    eps = 1e-7
    c = m * s / (np.square(s + eps) * 3.0) + m * s / (s + eps) - m
    return c.astype(np.float32), s.astype(np.float32)


def normalise_dense(raw: torch.Tensor, const_vec: torch.Tensor, std: torch.Tensor) -> torch.Tensor:
    """export_model.py:86-96: clip(x, 0, FLT_MAX) * std / (3 (std + 1e-7)^2) - c, clipped to [-0.99, 0.99] (fp32)."""
    x = torch.clamp(raw.float(), min=0.0)      # (the upper bound sys.float_info.max is no bound for float32)
    y = x * std / (torch.square(std + 1e-7) * 3.0) - const_vec
    return torch.clamp(y, min=-0.99, max=0.99)


class HistoryCache:
    """K / V of many users' histories in 8 bits between requests (kv_cache.py): `n_users` places, each holding up to max_len rows in 64-row
    blocks of one pool per layer; all layers share the block table.  Rows are appended for any set of users at a time, queries of any set of
    users attend in one launch, a user's place is given up and its blocks return to the pool -- all on the GPU, in stream order."""

    def __init__(self, n_users, n_blocks, max_len, num_heads, head_dim, layers=1, device="cuda"):
        if n_users <= 0 or n_blocks <= 0 or max_len <= 0 or layers <= 0:
            raise ValueError("HistoryCache needs at least one user, block, row and layer")
        self.layers = [KVCache.empty(n_blocks, num_heads, head_dim, device) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=self.layers[0].device)
        width = -(-max_len // BLOCK)
        self.n_users, self.max_len = int(n_users), width * BLOCK                 # (whole blocks)
        self.table = torch.full((n_users, width), -1, **i32)
        self.lens = torch.zeros((n_users,), **i32)
        self.free = torch.arange(n_blocks, **i32)
        self.n_free = torch.full((1,), n_blocks, **i32)

    def append(self, rows, new_lens):
        """rows: one (k_rows, v_rows) pair per layer, bf16 [R, num_heads * head_dim], the users' new rows in the order of their places; new_lens:
        int32 [n_users] (0: nothing).  Returns the KVPlan: plan.refused counts users whose rows found no room (their histories stay)."""
        if len(rows) != len(self.layers):
            raise ValueError("%d layers, got rows for %d" % (len(self.layers), len(rows)))
        plan = kv_plan(self.lens, new_lens, self.table, self.free, self.n_free, rows[0][0].shape[0])
        for cache, (k, v) in zip(self.layers, rows):
            kv_append(cache, k, v, plan)
        self.lens, self.n_free = plan.lens, plan.n_free
        return plan

    def of(self, places):
        """(table, lens) of the users in `places` (index tensor), in that order: what attend takes for a step that concerns these alone"""
        return self.table.index_select(0, places), self.lens.index_select(0, places)

    def attend(self, layer, q, row_off, num_heads, max_q, held=None, **kw):
        """kv_attn of one layer: query rows row_off[r] .. row_off[r + 1] of q belong to user r, or to the r-th of held = of(places) (at most
        65535 users a call)"""
        table, lens = (self.table, self.lens) if held is None else held
        return kv_attn(self.layers[layer], q, table, lens, row_off, num_heads, max_q, **kw)

    def drop(self, done):
        """done: int32 [n_users], non-zero: forget that user"""
        self.lens, self.n_free = self.lens.clone(), self.n_free.clone()          # (a plan of an earlier step keeps its own)
        kv_release(done, self.lens, self.table, self.free, self.n_free)


class CandidateScorer:
    def __init__(self, engine: DMTEngine, export_weight=(1.0, 1.0), mean: Optional[Sequence[float]] = None,
                 std: Optional[Sequence[float]] = None, optimizer=None):
        """optimizer: the TFAdam of a LIVE trainer sharing this engine's tables, or None for a frozen / restored model.  The exact lazy
        Adam leaves zero-gradient updates of untouched rows pending; scoring reads rows without replaying them, so with
        a live optimizer the tables are flushed before every request that follows a train step."""
        self.engine = engine
        self.optimizer = optimizer
        self._flushed_at = -1
        self.spec = engine.spec
        self.w = (float(export_weight[0]), float(export_weight[1]))
        dev = engine.store.device
        if mean is not None:
            c, s = normalisation_constants(mean, std)
            self.const_vec, self.std = torch.as_tensor(c).to(dev), torch.as_tensor(s).to(dev)
        else:
            self.const_vec = self.std = None
        self.user_feats = [f for (_n, _r, _d, f, side) in self.spec["embedding_list"] if side == "u"]

    # ------------------------------------------------------------------ request assembly
    def tile_request(self, user_inputs: dict, item_inputs: dict, dense_raw: np.ndarray) -> DeviceBatch:
        """user_inputs: {feature: (ids int[T], wts float[T] or None)} -- one list per user-side feature, as the
        emb_common_* placeholders of export_model.py:64-84;  item_inputs: {feature: (idx int[B, T], lens int[B], wts or None)}
        (already padded; item-side features carry one id per candidate in the reference data);  dense_raw: float[B, F]."""
        dev = self.engine.store.device
        B = int(np.asarray(dense_raw).shape[0])
        feats: Dict[str, FeatureColumn] = {}
        for f, (ids, wts) in user_inputs.items():
            ids = np.asarray(ids, dtype=np.int32).reshape(1, -1)
            T = max(ids.shape[1], 1)
            idx = torch.as_tensor(ids).to(dev).expand(B, T).contiguous()
            lens = torch.full((B,), ids.shape[1], dtype=torch.int32, device=dev)
            w = None
            if wts is not None and not np.all(np.asarray(wts) == 1.0):
                w = torch.as_tensor(np.asarray(wts, dtype=np.float32).reshape(1, -1)).to(dev).expand(B, T).contiguous()
            feats[f] = FeatureColumn(idx, w, lens, T)
        for f, (idx, lens, wts) in item_inputs.items():
            idx = np.asarray(idx, dtype=np.int32)
            w = None
            if wts is not None and not np.all(np.asarray(wts) == 1.0):
                w = torch.as_tensor(np.asarray(wts, dtype=np.float32)).to(dev)
            feats[f] = FeatureColumn(torch.as_tensor(idx).to(dev), w, torch.as_tensor(np.asarray(lens, dtype=np.int32)).to(dev), idx.shape[1])
        dense = torch.as_tensor(np.asarray(dense_raw, dtype=np.float32)).to(dev)
        if self.const_vec is not None:
            dense = normalise_dense(dense, self.const_vec, self.std)
        return DeviceBatch(B, feats, dense.contiguous())

    @staticmethod
    def _row0(batch: DeviceBatch) -> DeviceBatch:
        feats = {f: FeatureColumn(c.idx[:1], c.wts[:1] if c.wts is not None else None, c.lens[:1], c.T) for f, c in batch.feats.items()}
        return DeviceBatch(1, feats, batch.dense[:1])

    def _fresh_tables(self):
        if self.optimizer is not None and self.optimizer.global_step != self._flushed_at:
            self.optimizer.flush_tables()
            self._flushed_at = self.optimizer.global_step

    # ------------------------------------------------------------------ scoring
    @torch.no_grad()
    def logits(self, batch: DeviceBatch):
        """(click_logit, order_logit) [B, 1] for B candidate rows of one user; user-side columns are read from row 0."""
        eng, spec = self.engine, self.spec
        self._fresh_tables()
        saved_seed, eng.dropout_step_seed = eng.dropout_step_seed, None        # predict graph: is_train=False
        try:
            b1 = self._row0(batch)
            X1, _tar1, _z1 = eng.gather(b1)
            tar_g, zbuf = eng.gather_pooled(batch)
            in_mlp = bool(spec.get("is_trans_input_by_mlp"))      # (then both gathers hand out raw rows and every sequence has its own target)
            us, tars_scaled = [], []
            for i, pairs in enumerate(spec["attention_embed_pairs"]):
                lens1 = b1.feats[pairs[-1][0]].lens
                x1, tar_i = eng.input_mlp(i, X1[i], tar_g) if in_mlp else (X1[i], tar_g)
                tars_scaled.append(tar_i)
                mem1 = eng.encode_prepared(x1, lens1, i)                       # [1, T, d], once per request
                k_lens = lens1.expand(batch.B).contiguous()
                us.append(eng.decode_shared(eng.decoder_query(tar_i).unsqueeze(1), mem1, k_lens, i).squeeze(1))
            z = AssembleFn.apply(zbuf, eng.plan.interest_off, spec["d_model"], *eng.interest_blocks(us, tars_scaled))
            tasks = eng.expert_gate(z, z_is_engine_buffer=True)          # (z is gather_pooled's zero-initialised zbuf)
            return tuple(eng.build_tower(m, nm) for m, nm in zip(tasks, ("click", "order")))
        finally:
            eng.dropout_step_seed = saved_seed

    # ------------------------------------------------------------------ histories kept between requests
    def keep_histories(self, n_users, n_blocks):
        """Make room for the encoded histories of n_users users (n_blocks blocks of 64 rows a sequence): remember() encodes a user once,
        logits_of() then scores candidates of many users in one batch without running an encoder.  For bf16 engines with a head size that
        is a multiple of 16 (the E64 widths); the decoder's K / V are held in 8 bits, so its attention is that of the rounded rows."""
        eng, spec = self.engine, self.spec
        if eng.store.compute_dtype != torch.bfloat16:
            raise ValueError("histories are kept for bf16 engines")
        if spec.get("is_trans_input_by_mlp"):
            raise ValueError("histories are not kept for is_trans_input_by_mlp models")
        H, layers = spec["num_heads"], int(spec.get("num_blocks_decode", 1))
        self.histories = [HistoryCache(n_users, n_blocks, spec["maxlen_k"], H, spec["d_model"] // H, layers, eng.store.device)
                          for _ in spec["attention_embed_pairs"]]

    def _places(self, users, B):
        if not hasattr(self, "histories"):
            raise RuntimeError("keep_histories() first")
        users, n = np.asarray(users, dtype=np.int64), self.histories[0].n_users
        if users.shape != (B,) or B == 0:
            raise ValueError("one place for each row of the batch")
        if users.min() < 0 or users.max() >= n:
            raise ValueError("places lie in 0 .. %d" % (n - 1))
        return users, n

    @torch.no_grad()
    def remember(self, users, batch: DeviceBatch):
        """Encode row r of `batch` as the history of place users[r] (distinct places; what stood there is replaced).  A sequence without events
        is kept as one row, the mean of its T padded rows (T: the column's width in this batch): the model's attention gives those the
        same weight, in training and in logits().
        Returns the number of (user, sequence) histories that found no room: nothing is kept of them, and the attention over them gives
        zeros.  A history is as old as the weights that encoded it: after training steps, remember it again."""
        eng, spec = self.engine, self.spec
        users, n = self._places(users, batch.B)
        if len(np.unique(users)) != len(users):
            raise ValueError("the places of one call must be distinct")
        self._fresh_tables()
        dev, d = eng.store.device, spec["d_model"]
        order = np.argsort(users)                                # rows go in in the order of the places
        done = np.zeros(n, dtype=np.int32)
        done[users] = 1
        # (dense rows: without host lengths no sequence is packed)
        dense = DeviceBatch(batch.B, {f: FeatureColumn(c.idx, c.wts, c.lens, c.T) for f, c in batch.feats.items()}, batch.dense)
        saved_seed, eng.dropout_step_seed = eng.dropout_step_seed, None
        try:
            X, _tar, _z = eng.gather(dense)
            refused = 0
            for i, h in enumerate(self.histories):
                lens, T = eng.seq_lens(dense, i), X[i].shape[1]
                held = lens.cpu().numpy()
                empty = np.flatnonzero(held <= 0)
                if len(empty):
                    empty = torch.as_tensor(empty).to(dev)
                new = np.zeros(n, dtype=np.int32)
                new[users] = np.clip(held, 1, T)
                at = torch.as_tensor(np.concatenate([r * T + np.arange(new[users[r]]) for r in order])).to(dev)
                mem = eng.encode_prepared(X[i], lens, i)
                rows = []
                for j in range(len(h.layers)):
                    kv = eng.memory_kv(mem, i, j)
                    if len(empty):
                        kv[empty, 0] = kv[empty].float().mean(1).to(kv.dtype)
                    kv = kv.reshape(-1, 2 * d)[at]
                    rows.append((kv[:, :d], kv[:, d:]))
                h.drop(torch.as_tensor(done).to(dev))
                refused += int(h.append(rows, torch.as_tensor(new).to(dev)).refused)
            return refused
        finally:
            eng.dropout_step_seed = saved_seed

    @torch.no_grad()
    def logits_of(self, users, batch: DeviceBatch):
        """(click_logit, order_logit) [B, 1] for candidate rows of remembered users: users[r] is the place of row r's user, in ascending
        order (rows of one user side by side).  The sequence columns of `batch` are not read by the attention."""
        eng, spec = self.engine, self.spec
        users, _n = self._places(users, batch.B)
        if (np.diff(users) < 0).any():
            raise ValueError("the places must stand in ascending order")
        self._fresh_tables()
        asked, count = np.unique(users, return_counts=True)
        row_off = torch.as_tensor(np.concatenate([[0], np.cumsum(count)]).astype(np.int32)).to(eng.store.device)
        asked = torch.as_tensor(asked).to(eng.store.device)
        saved_seed, eng.dropout_step_seed = eng.dropout_step_seed, None
        try:
            tar, zbuf = eng.gather_pooled(batch)
            us = []
            for i, h in enumerate(self.histories):
                held = h.of(asked)
                attend = lambda j, q, h=h, held=held: h.attend(j, q, row_off, spec["num_heads"], int(count.max()), held, causal=False)  # noqa: E731
                us.append(eng.decode_cached(eng.decoder_query(tar), i, attend))
            z = AssembleFn.apply(zbuf, eng.plan.interest_off, spec["d_model"], *eng.interest_blocks(us, [tar] * len(us)))
            tasks = eng.expert_gate(z, z_is_engine_buffer=True)
            return tuple(eng.build_tower(m, nm) for m, nm in zip(tasks, ("click", "order")))
        finally:
            eng.dropout_step_seed = saved_seed

    @torch.no_grad()
    def score(self, batch: DeviceBatch):
        """export_model.py:106-114: Scores = (w0 sigmoid(click) + w1 sigmoid(order)) / (w0 + w1); also returns both heads."""
        c, o = self.logits(batch)
        pc, po = torch.sigmoid(c.float()).reshape(-1), torch.sigmoid(o.float()).reshape(-1)
        return (self.w[0] * pc + self.w[1] * po) / (self.w[0] + self.w[1]), pc, po


class GraphedScorer:
    """The kernel sequence of CandidateScorer.score for ONE request shape (candidate count, padded id-list lengths), captured
    once into a HIP graph and replayed per request: the eager path is bound by ~100 host-side launches (1.3 ms at any candidate
    count), the replay is not (0.63 ms at 256 candidates, 0.89 ms at 4096 on MI355X, scripts/serve_bench.py).
    Requests are written into the captured input buffers in place; shapes must match the template."""

    def __init__(self, scorer: CandidateScorer, template: DeviceBatch):
        self.scorer = scorer
        self.static = template
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                 # warm-up outside the capture (lazy library / allocator state)
            for _ in range(2):
                scorer.score(template)
        torch.cuda.current_stream().wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = scorer.score(template)

    def score(self, batch: DeviceBatch):
        st = self.static
        if batch.B != st.B or set(batch.feats) != set(st.feats):
            raise ValueError("request does not match the captured shape (B=%d)" % st.B)
        for f, col in batch.feats.items():
            dst = st.feats[f]
            if col.idx.shape != dst.idx.shape:
                raise ValueError("feature %s: id-list shape differs from the captured request" % f)
            # whether a weights column exists is a property of the captured graph, not of a request's values: a request whose weights
            # are all 1.0 arrives without the column (tile_request drops it) and is served by writing ones
            if dst.wts is None and col.wts is not None:
                raise ValueError("feature %s: the captured request has no weights column but this request has weights != 1" % f)
            dst.idx.copy_(col.idx); dst.lens.copy_(col.lens)
            if dst.wts is not None:
                if col.wts is not None:
                    dst.wts.copy_(col.wts)
                else:
                    dst.wts.fill_(1.0)
        st.dense.copy_(batch.dense)
        self.graph.replay()
        return self.out
