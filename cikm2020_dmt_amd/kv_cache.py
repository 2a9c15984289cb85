"""K / V of served histories in 8 bits: a pool of 64-token blocks, the GPU-side allocator that hands them out, the append that rounds new
rows into them and the attention that reads them.  Serving keeps a user's encoded history here between requests; serving.HistoryCache is
the object around these calls.

    plan = kv_plan(lens, new_lens, table, free, n_free, rows)      # blocks, slots of this step's rows; lens / n_free of the next step
    kv_append(cache, k_rows, v_rows, plan)                         # bf16 rows -> e4m3 bytes, one power-of-two scale a block and head
    out = kv_attn(cache, q_rows, table, plan.lens, plan.row_off, H, max_q)
    kv_release(done, lens, table, free, n_free)

Everything is computed by libdmt_hip kernels on the current stream; nothing is read back, so a step can be captured in a graph (the
workspaces come from torch's allocator in every call).  include/dmt_hip.h (dmt_kv_*) has the layouts and the rules."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .ops import BF16, F32, _cur_device, _raw_stream, p

BLOCK = L.DMT_KV_BLOCK
F8 = torch.float8_e4m3fn


def _call(device, name, *args):
    """one entry point on the device's current stream (with that device current)"""
    if _cur_device() == device.index:
        L.call(name, *args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            L.call(name, *args, _raw_stream(_cur_device()))


class KVCache:
    """The pools: k [n_blocks, Hkv, 64, dh], v [n_blocks, Hkv, dh, 64] (float8_e4m3fn), k_scale, v_scale fp32 [n_blocks, Hkv]."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.shape[2] != BLOCK or v.dim() != 4 or tuple(v.shape) != (k.shape[0], k.shape[1], k.shape[3], BLOCK):
            raise ValueError("k must be [n_blocks, Hkv, %d, dh] and v [n_blocks, Hkv, dh, %d], got %s and %s" % (BLOCK, BLOCK, tuple(k.shape), tuple(v.shape)))
        n, Hkv, _, dh = k.shape
        if dh % 16 or not 0 < dh <= 128 or n * BLOCK >= 2 ** 31 or n == 0 or Hkv == 0:
            raise ValueError("the cache takes dh a multiple of 16 up to 128 and 1 .. 2^31 / %d - 1 blocks: got dh = %d, %d blocks" % (BLOCK, dh, n))
        for t in (k, v):
            if t.dtype != F8 or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("the pools must be contiguous, 16-byte aligned %s tensors" % F8)
        for t in (k_scale, v_scale):
            if t.dtype != F32 or tuple(t.shape) != (n, Hkv) or not t.is_contiguous():
                raise ValueError("the scales must be contiguous fp32 [%d, %d]" % (n, Hkv))
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1 or not k.is_cuda:
            raise ValueError("the cache lives on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_blocks, self.Hkv, self.dh, self.device = n, Hkv, dh, k.device
        self._ws_bytes = {}
        self._args = (Hkv, dh, n, k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())

    @classmethod
    def empty(cls, n_blocks, Hkv, dh, device="cuda"):
        z = lambda *s: torch.zeros(s, dtype=torch.uint8, device=device).view(F8)  # noqa: E731
        return cls(z(n_blocks, Hkv, BLOCK, dh), z(n_blocks, Hkv, dh, BLOCK), torch.ones((n_blocks, Hkv), device=device),
                   torch.ones((n_blocks, Hkv), device=device))


class KVPlan(NamedTuple):
    """What kv_plan leaves: row_off [n + 1], lens [n] (after the step), slots [rows] (-1: not stored), the runs of kv_append, n_free [1] of
    the next step, refused [1] requests (their rows have slots -1 and their lens stay)."""
    row_off: torch.Tensor
    lens: torch.Tensor
    slots: torch.Tensor
    run_row: torch.Tensor
    run_len: torch.Tensor
    n_free: Optional[torch.Tensor]
    refused: Optional[torch.Tensor]


def _i32(t, shape, what, device):
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError("%s must be a contiguous int32 tensor %s on %s, got %s %s on %s" % (what, list(shape), device, t.dtype, list(t.shape), t.device))


def kv_plan(lens, new_lens, table, free, n_free, rows) -> KVPlan:
    """Block tables and slots of a step, on the GPU.  lens [n]: tokens held; new_lens [n]: rows that each request adds; table
    [n, width]: its blocks (the new ones are written into it); free: the stack of free block ids, n_free [1] of them; rows: rows of the
    step's matrices.  All int32.  Calling it again with the same arguments gives the same plan."""
    dev = lens.device
    if not lens.is_cuda:
        raise RuntimeError("libdmt_hip kernels need device tensors (got a %s tensor); there is no CPU path" % dev)
    if lens.dim() != 1 or table.dim() != 2:
        raise ValueError("lens is [n] and table [n, width], got %s and %s" % (list(lens.shape), list(table.shape)))
    n, width, rows = lens.shape[0], table.shape[1], int(rows)
    _i32(lens, (n,), "lens", dev)
    _i32(new_lens, (n,), "new_lens", dev)
    _i32(table, (n, width), "table", dev)
    _i32(free, (free.numel(),), "free", dev)
    _i32(n_free, (1,), "n_free", dev)
    if not 0 <= rows < 2 ** 30:
        raise ValueError("rows must lie in 0 .. 2^30 - 1, got %d" % rows)
    runs = min(rows, rows // BLOCK + 2 * n)
    need = 16 + 8 * n                                                            # dmt_kv_plan_ws_bytes
    sizes = (n + 1, n, rows, runs, runs, 1, 1)
    buf = lens.new_empty(need // 4 + sum(sizes))     # one allocation: the step is a matter of microseconds
    base = buf.data_ptr()
    out = torch.split_with_sizes(buf, (need // 4,) + sizes)
    a0 = base + need
    a1 = a0 + 4 * (n + 1)
    a2 = a1 + 4 * n
    a3 = a2 + 4 * rows
    a4 = a3 + 4 * runs
    _call(dev, "dmt_kv_plan", n, rows, lens.data_ptr(), new_lens.data_ptr(), table.data_ptr(), width, free.data_ptr(), free.shape[0],
          n_free.data_ptr(), a0, a1, a2, a3, a4, a4 + 4 * runs, base, need)
    return KVPlan(*out[1:])


def kv_release(done, lens, table, free, n_free):
    """Requests r with done[r] != 0 (int32 [n]) give their blocks back: pushed on `free`, n_free and lens are changed in place.  A block that
    two tables name is pushed once for each."""
    dev, n = lens.device, lens.shape[0]
    if not lens.is_cuda:
        raise RuntimeError("libdmt_hip kernels need device tensors (got a %s tensor); there is no CPU path" % dev)
    if lens.dim() != 1 or table.dim() != 2:
        raise ValueError("lens is [n] and table [n, width], got %s and %s" % (list(lens.shape), list(table.shape)))
    _i32(done, (n,), "done", dev)
    _i32(lens, (n,), "lens", dev)
    _i32(table, (n, table.shape[1]), "table", dev)
    _i32(free, (free.numel(),), "free", dev)
    _i32(n_free, (1,), "n_free", dev)
    _call(dev, "dmt_kv_release", n, p(done), p(lens), p(table), table.shape[1], p(free), p(n_free), free.numel())


def _rows(t, what, width, device):
    if t.dim() != 2 or t.dtype is not BF16 or t.shape[1] != width or t.device != device or t.stride(1) != 1:
        raise ValueError("%s must be bf16 rows [., %d] with unit inner stride on %s, got %s %s on %s" % (what, width, device, t.dtype, list(t.shape), t.device))
    rs = t.stride(0) if t.shape[0] > 1 else width
    if t.data_ptr() % 16 or rs % 8 or rs < width:
        raise ValueError("%s: rows must be 16-byte aligned and not overlap (stride %d)" % (what, rs))
    return rs


def kv_append(cache: KVCache, k_rows, v_rows, plan: KVPlan):
    """k_rows, v_rows (bf16 [rows, Hkv * dh]) into the slots of `plan`.  A block belongs to one request: two requests whose tables name the
    same block must not grow it in one call.  Doing it again with the same rows changes nothing."""
    rows, w, dev = plan.slots.shape[0], cache.Hkv * cache.dh, cache.device
    krs, vrs = _rows(k_rows, "k_rows", w, dev), _rows(v_rows, "v_rows", w, dev)
    if k_rows.shape[0] != rows or v_rows.shape[0] != rows:
        raise ValueError("the plan holds %d rows, k_rows %d and v_rows %d" % (rows, k_rows.shape[0], v_rows.shape[0]))
    runs = plan.run_row.shape[0]
    for t, s, what in ((plan.slots, rows, "slots"), (plan.run_row, runs, "run_row"), (plan.run_len, runs, "run_len")):
        _i32(t, (s,), what, dev)
    _call(dev, "dmt_kv_append", *cache._args, rows, k_rows.data_ptr(), krs, v_rows.data_ptr(), vrs, plan.slots.data_ptr(),
          plan.run_row.data_ptr(), plan.run_len.data_ptr(), runs)


def kv_read(cache: KVCache, slots):
    """(k_rows, v_rows) bf16 [n, Hkv * dh]: the values that stand in `slots` (int32 [n]), exactly; zeros for a slot outside the pool."""
    n, w = slots.shape[0], cache.Hkv * cache.dh
    _i32(slots, (n,), "slots", cache.device)
    k = torch.empty((n, w), dtype=BF16, device=cache.device)
    v = torch.empty_like(k)
    _call(cache.device, "dmt_kv_read", *cache._args, n, slots.data_ptr(), k.data_ptr(), w, v.data_ptr(), w)
    return k, v


def kv_attn(cache: KVCache, q, table, lens, row_off, H, max_q, max_len=None, *, causal=True, scale=None, cap=0.0, slopes=None, out=None,
            want_lse=False):
    """Attention of n requests' query rows over their cached tokens: q bf16 [rows, H * dh], request r owns rows row_off[r] .. row_off[r + 1]
    (int32 [n + 1]) and lens[r] tokens in the blocks table[r].  causal: its m rows stand at the positions lens - m .. lens - 1 (append
    them first; a request that the plan refused has nothing appended, so its rows stand over the last tokens that it held); otherwise
    every row stands behind the last token and sees all (candidates).  Scores as in ops.attn_var: scale, cap, slopes
    (fp32 [H]).  max_q bounds the rows of a request, max_len the lengths (default: what the table can hold): they size the launch, so
    keep them fixed for a captured graph and tight for speed.  Rows of no request (before row_off[0], past a request's max_q, past
    row_off[n]) are zeros, with `out` they stay as they were there; their lse is -inf."""
    dev, n = cache.device, lens.shape[0]
    if table.dim() != 2:
        raise ValueError("table is [n, width], got %s" % list(table.shape))
    if H <= 0 or H % cache.Hkv:
        raise ValueError("H = %d query heads cannot share Hkv = %d key heads evenly" % (H, cache.Hkv))
    w = H * cache.dh
    q_rs = _rows(q, "q", w, dev)
    _i32(table, (n, table.shape[1]), "table", dev)
    _i32(lens, (n,), "lens", dev)
    _i32(row_off, (n + 1,), "row_off", dev)
    if slopes is not None and (slopes.dtype != F32 or tuple(slopes.shape) != (H,) or not slopes.is_contiguous() or slopes.device != dev):
        raise ValueError("slopes must be a contiguous fp32 tensor [%d] on %s" % (H, dev))
    scale = 1.0 / float(cache.dh) ** 0.5 if scale is None else float(scale)
    if not (0.0 < scale <= 1e38) or not (0.0 <= cap <= 1e38):
        raise ValueError("scale must be positive, cap 0 or positive, both at most 1e38: got %r, %r" % (scale, cap))
    if max_q < 0 or (max_len is not None and max_len < 0):
        raise ValueError("max_q and max_len must not be negative")
    max_q = min(int(max_q), q.shape[0])                                          # (no request has more rows than there are)
    given = out is not None
    if not given:
        out = q.new_empty((q.shape[0], w))
    elif out.shape != q.shape:
        raise ValueError("out must be %s" % list(q.shape))
    elif out.data_ptr() == q.data_ptr() and q.shape[0]:
        raise ValueError("out must not be q")
    o_rs = _rows(out, "out", w, dev) if given else w
    lse = torch.empty((q.shape[0], H), dtype=F32, device=dev) if want_lse else None
    most = table.shape[1] * BLOCK
    max_len = most if max_len is None else min(int(max_len), most)
    key = (n, H, max_q, max_len)
    need = cache._ws_bytes.get(key)
    if need is None:                   # (a function of the sizes alone)
        if len(cache._ws_bytes) >= 4096:
            cache._ws_bytes.clear()
        d = L.KvAttnDesc()
        d.n, d.Hq, d.Hkv, d.dh, d.max_q, d.max_len = n, H, cache.Hkv, cache.dh, max_q, max_len
        need = cache._ws_bytes[key] = int(L.load().dmt_kv_attn_ws_bytes(C.byref(d)))
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    a = cache._args
    d = L.kv_attn_desc(n, H, a[0], a[1], a[2], max_q, max_len, table.shape[1], q.shape[0], a[3], a[4], a[5], a[6], q.data_ptr(), q_rs,
                       table.data_ptr(), lens.data_ptr(), row_off.data_ptr(), scale, cap, 1 if causal else 0, 2 if given else 3,
                       0 if slopes is None else slopes.data_ptr(), out.data_ptr(), o_rs, 0 if lse is None else lse.data_ptr(),
                       0 if ws is None else ws.data_ptr(), need)
    _call(dev, "dmt_kv_attn", C.byref(d))
    return (out, lse) if want_lse else out
