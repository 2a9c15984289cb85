// Attention over packed rows of any length: forward (include/dmt_hip.h: dmt_attn_var_desc has the formulas).
#include "dmt_attn_var.h"

using namespace attn_var;

namespace {

template <typename T>
__global__ __launch_bounds__(256) void rows_fwd_kernel(const Args a) {
  __shared__ float lds[4][ROW_LDS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.z, h = blockIdx.y;
  const Ex e = example(a, b);
  const int i = blockIdx.x * 4 + wave;
  if (i < e.ql) row_fwd<T>(a, e, h, i, lds[wave], lane);
}

__global__ void doc_ranges_kernel(const int* off, const int* lens, const int* doc, int most, long long rows, int nt, int B, int2* out) {
  const int t = blockIdx.x * blockDim.y + threadIdx.y, b = blockIdx.y, lane = threadIdx.x;
  if (t >= nt) return;
  const int len = clip_len(lens[b], most, off[b], rows);
  const int i = t * 64 + lane;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
  if (i < len) lo = hi = doc[(long long)off[b] + i];
  for (int s = 32; s; s >>= 1) {
    lo = min(lo, __shfl_xor(lo, s));
    hi = max(hi, __shfl_xor(hi, s));
  }
  if (lane == 0) out[(long long)b * nt + t] = make_int2(lo, hi);
}

}  // namespace

uint64_t up16(uint64_t x) { return (x + 15) & ~15ull; }

extern "C" int dmt_attn_var_supported(int32_t dtype, int32_t dh, int32_t Hq, int32_t Hkv) {
  if (dtype != DMT_F32 && dtype != DMT_BF16) return 0;
  if (dh <= 0 || dh > MAX_DH || dh % (dtype == DMT_F32 ? 4 : 8)) return 0;
  return Hq > 0 && Hkv > 0 && Hq % Hkv == 0;
}

namespace {
struct WsLayout { uint64_t qr, kr, D, sp, total; };
WsLayout ws_layout(const dmt_attn_var_desc* d, bool backward) {
  const uint64_t nqt = (uint64_t)cdiv64(d->max_q, 64), nkt = (uint64_t)cdiv64(d->max_k, 64);
  WsLayout w;
  uint64_t at = 0;
  w.qr = at;
  if (d->q_doc) at += up16(8 * nqt * (uint64_t)d->B);
  w.kr = at;
  if (d->q_doc) at += up16(8 * nkt * (uint64_t)d->B);
  w.D = at;
  if (backward) at += up16(4 * (uint64_t)d->rows_q * (uint64_t)d->Hq);
  w.sp = at;
  if (backward && d->dslopes) at += up16(4 * (uint64_t)d->Hq * (uint64_t)d->B * (uint64_t)cdiv64(d->max_q, 128));
  w.total = at;
  return w;
}
bool al16(const void* p, int64_t rs, int es) { return ((uintptr_t)p % 16) == 0 && (rs * es) % 16 == 0; }
}  // namespace

extern "C" uint64_t dmt_attn_var_ws_bytes(const dmt_attn_var_desc* d, int32_t backward) {
  if (!d || d->B <= 0 || d->max_q <= 0 || d->max_k <= 0) return 0;
  return ws_layout(d, backward != 0).total;
}

int dmt_attn_var_args(const dmt_attn_var_desc* d, Args* a, bool backward, const char* what) {
  DMT_CHECK_ARG(d, "%s: no descriptor", what);
  DMT_CHECK_ARG(d->B >= 0 && d->max_q >= 0 && d->max_k >= 0 && d->rows_q >= 0 && d->rows_k >= 0, "%s: negative size", what);
  DMT_CHECK_ARG(dmt_attn_var_supported(d->dtype, d->dh, d->Hq, d->Hkv),
                "%s: needs bf16 (dh %% 8 == 0) or fp32 (dh %% 4 == 0), dh <= 128 and Hq a multiple of Hkv: got dtype %d, dh %d, Hq %d, Hkv %d", what,
                d->dtype, d->dh, d->Hq, d->Hkv);
  DMT_CHECK_ARG(d->B <= 65535 && d->Hq <= 65535, "%s: B and Hq <= 65535", what);
  DMT_CHECK_ARG(d->rows_q < (1ll << 31) && d->rows_k < (1ll << 31), "%s: row numbers are int32", what);
  DMT_CHECK_ARG(d->scale > 0.f && d->scale < 3.4e38f, "%s: scale must be positive and finite", what);
  DMT_CHECK_ARG(d->cap >= 0.f && d->cap < 3.4e38f, "%s: cap must be 0 (none) or positive and finite", what);
  DMT_CHECK_ARG((d->q_doc == nullptr) == (d->k_doc == nullptr), "%s: q_doc and k_doc go together", what);
  if (d->B == 0 || d->max_q == 0 || d->rows_q == 0) {
    // no query row: the forward has nothing to do, the backward still owes dk = dv = 0
    if (!backward || d->B == 0 || d->max_k == 0 || d->rows_k == 0) return 1;
  }
  DMT_CHECK_ARG(d->q_off && d->q_lens && d->k_off && d->k_lens, "%s: NULL offsets or lengths", what);
  const int es = d->dtype == DMT_F32 ? 4 : 2;
  const int64_t wq = (int64_t)d->Hq * d->dh, wk = (int64_t)d->Hkv * d->dh;
  DMT_CHECK_ARG(d->rows_q == 0 || (d->Q && d->out), "%s: NULL Q / out", what);
  DMT_CHECK_ARG(d->rows_k == 0 || (d->K && d->V), "%s: NULL K / V", what);
  DMT_CHECK_ARG(d->q_rs >= wq && d->k_rs >= wk && d->v_rs >= wk && (d->rows_q == 0 || d->o_rs >= wq), "%s: row stride shorter than a row", what);
  DMT_CHECK_ARG(d->k_rs * es < (1ll << 24) && d->v_rs * es < (1ll << 24) && d->q_rs * es < (1ll << 24), "%s: row stride of 16 MB or more", what);
  DMT_CHECK_ARG(al16(d->Q, d->q_rs, es) && al16(d->K, d->k_rs, es) && al16(d->V, d->v_rs, es) && al16(d->out, d->o_rs, es),
                "%s: operand rows must be 16-byte aligned", what);
  if (backward) {
    DMT_CHECK_ARG(d->rows_q == 0 || (d->dout && d->lse && d->dQ), "%s: NULL dout / lse / dQ", what);
    DMT_CHECK_ARG(d->rows_k == 0 || (d->dK && d->dV), "%s: NULL dK / dV", what);
    DMT_CHECK_ARG((d->rows_q == 0 || (d->do_rs >= wq && d->dq_rs >= wq)) && d->dk_rs >= wk && d->dv_rs >= wk && d->do_rs * es < (1ll << 24),
                  "%s: bad gradient row stride", what);
    DMT_CHECK_ARG(al16(d->dout, d->do_rs, es) && al16(d->dQ, d->dq_rs, es) && al16(d->dK, d->dk_rs, es) && al16(d->dV, d->dv_rs, es),
                  "%s: gradient rows must be 16-byte aligned", what);
    DMT_CHECK_ARG(!d->dslopes || d->slopes, "%s: dslopes without slopes", what);
  }
  const WsLayout w = ws_layout(d, backward);
  DMT_CHECK_ARG(w.total == 0 || (d->ws && ((uintptr_t)d->ws % 16) == 0 && d->ws_bytes >= w.total), "%s: workspace of %llu bytes needed", what,
                (unsigned long long)w.total);
  char* ws = (char*)d->ws;
  a->B = d->B; a->Hq = d->Hq; a->Hkv = d->Hkv; a->dh = d->dh; a->G = d->Hq / d->Hkv;
  a->max_q = d->max_q; a->max_k = d->max_k; a->rows_q = d->rows_q; a->rows_k = d->rows_k;
  a->Q = d->Q; a->q_rs = d->q_rs; a->K = d->K; a->k_rs = d->k_rs; a->V = d->V; a->v_rs = d->v_rs;
  a->q_off = d->q_off; a->q_lens = d->q_lens; a->k_off = d->k_off; a->k_lens = d->k_lens;
  a->scale = d->scale; a->cap = d->cap; a->causal = d->causal != 0; a->slopes = d->slopes; a->prefix = d->prefix;
  a->q_doc = d->q_doc; a->k_doc = d->k_doc;
  a->out = d->out; a->o_rs = d->o_rs; a->lse = d->lse;
  a->dout = d->dout; a->do_rs = d->do_rs; a->dQ = d->dQ; a->dq_rs = d->dq_rs; a->dK = d->dK; a->dk_rs = d->dk_rs; a->dV = d->dV; a->dv_rs = d->dv_rs;
  a->dslopes = d->dslopes;
  a->nqt = (int)cdiv64(d->max_q, 64);
  a->nkt = (int)cdiv64(d->max_k, 64);
  a->q_rng = d->q_doc ? (const int2*)(ws + w.qr) : nullptr;
  a->k_rng = d->q_doc ? (const int2*)(ws + w.kr) : nullptr;
  a->D = backward ? (float*)(ws + w.D) : nullptr;
  a->slope_part = backward && d->dslopes ? (float*)(ws + w.sp) : nullptr;
  return DMT_OK;
}

int dmt_attn_var_doc_ranges(const Args& a, void* stream) {
  if (!a.q_doc) return DMT_OK;
  hipStream_t st = (hipStream_t)stream;
  if (a.nqt) doc_ranges_kernel<<<dim3((a.nqt + 3) / 4, a.B), dim3(64, 4), 0, st>>>(a.q_off, a.q_lens, a.q_doc, a.max_q, a.rows_q, a.nqt, a.B, (int2*)a.q_rng);
  if (a.nkt) doc_ranges_kernel<<<dim3((a.nkt + 3) / 4, a.B), dim3(64, 4), 0, st>>>(a.k_off, a.k_lens, a.k_doc, a.max_k, a.rows_k, a.nkt, a.B, (int2*)a.k_rng);
  DMT_CHECK_LAUNCH("dmt_attn_var(doc ranges)");
  return DMT_OK;
}

extern "C" int dmt_attn_var_fwd(const dmt_attn_var_desc* d, void* stream) {
  Args a;
  const int rc = dmt_attn_var_args(d, &a, false, "dmt_attn_var_fwd");
  if (rc) return rc < 0 ? rc : DMT_OK;
  const dim3 grid((a.max_q + 3) / 4, a.Hq, a.B);
  if (d->dtype == DMT_F32)
    rows_fwd_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    rows_fwd_kernel<bf16_t><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  DMT_CHECK_LAUNCH("dmt_attn_var_fwd(rows)");
  return DMT_OK;
}
