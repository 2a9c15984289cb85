// Attention over packed rows of any length: forward (include/dmt_hip.h: dmt_attn_var_desc has the formulas).
#include "dmt_attn_var.h"

using namespace attn_var;

namespace {

// One workgroup of NW wavefronts owns 32 NW queries of a head (rows_of) and walks over the keys in tiles of 64: bf16 has one tile in LDS and the next
// on its way there (loads into LDS, rows swizzled by exclusive or so that neither row nor transposing reads meet in a bank), fp32 has one tile
// and the next in registers.  S^T = K Q^T and O^T = V^T P^T: a lane owns a query, its statistics stay in the lane, and P packed is an operand.
// One pass: the running maximum m moves only when a row's scores pass it by more than 2^8 (the weights
// are then at most 256, exact in fp32 sums and without loss in bf16), so the output is rescaled a few times a row instead of every tile.
// What bounds it: the matrix pipe and, beside it, one power and about 4 other vector operations a score (2 x 4096 causal, 16 heads of 128: 171 us =
// 802 TFLOP/s of the products that the mask leaves); for short histories the rows (256 of up to 200, 4 heads of 80: 37 us, 57 MB).
// fp32 takes 32x32x2 products; past 64 dims its operands and sums do not fit the registers and part of them goes to scratch (64 histories of up to
// 200 with slopes, 4 heads of 20 / 80 / 128: 27 / 74 / 86 us, dQ 37 / 128 / 142, dK and dV 41 / 134 / 229).
template <typename T, int DHP, int SHAPE, bool DOCS, int NW>
__global__ __launch_bounds__(64 * NW, 2) void tile_fwd_kernel(const Args a, int nt) {
  typedef Tile<T, DHP> TL;
  constexpr int NB = sizeof(T) == 2 ? 2 : 1, ROWS = 32 * NW;               // tiles in LDS
  constexpr int PAD = sizeof(T) == 2 ? 0 : 32, KE = KT * TL::RS, VE = KT * TL::RS + PAD;      // (fp32: dims past the last row's end are read, not used)
  __shared__ __attribute__((aligned(16))) T lds[NB * (KE + VE)];
  __shared__ __attribute__((aligned(16))) int docs[DOCS ? NB : 1][KT];
  static_assert(sizeof(lds) >= NW * ROW_LDS * sizeof(float), "the row form works in the tiles' memory");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l31 = lane & 31;
  int head, qt;
  place(blockIdx.x, a.B * a.Hq, nt, a.causal, head, qt);
  const int b = head / a.Hq, h = head - b * a.Hq, hk = h / a.G;
  const Ex e = example(a, b);
  if (qt * ROWS >= e.ql) return;
  const int iw = qt * ROWS + wave * 32, i = iw + l31;
  const bool active = iw < e.ql;
  const T* K = (const T*)a.K + e.k0 * a.k_rs + (long long)hk * a.dh;
  const T* V = (const T*)a.V + e.k0 * a.v_rs + (long long)hk * a.dh;
  const Shape sh = shape_of<T>(a, h);
  // what the workgroup, the wavefront and the lane's row may see
  const int last = (qt * ROWS + ROWS < e.ql ? qt * ROWS + ROWS : e.ql) - 1;
  const int lim_wg = a.causal ? max(e.pre, min(e.kl, last + e.off + 1)) : e.kl;
  const int lim_w = a.causal ? max(e.pre, min(e.kl, min(iw + 31, e.ql - 1) + e.off + 1)) : e.kl;
  const int lim0 = a.causal ? min(e.kl, i + e.off + 1) : e.kl, lim = max(lim0, e.pre);
  const int nk = (lim_wg + KT - 1) / KT;
  int qd = 0;
  Walk<DOCS> wk;
  wk.hi = nk;
  if constexpr (DOCS) {
    wk.lo = 0;
    const int2* qr = a.q_rng + (long long)b * a.nqt;
    const int t0 = qt * ROWS / 64, t1 = NW > 2 && t0 + 1 < a.nqt ? t0 + 1 : t0;
    const int2 r0 = qr[t0], r1 = qr[t1], rw = wave < 2 ? r0 : r1;
    wk.rng = a.k_rng + (long long)b * a.nkt;
    wk.free_wg = wk.free_w = (e.pre + KT - 1) / KT;
    wk.glo = min(r0.x, r1.x);
    wk.ghi = max(r0.y, r1.y);
    wk.wlo = rw.x;
    wk.whi = rw.y;
    wk.chunk = -1;
    qd = i < e.ql ? a.q_doc[e.q0 + i] : 0;
  }
  Stage<T, DHP, NW> st;
  st.init(a.k_rs, a.v_rs, a.dh, tid);
  int kd = 0;
  const auto begin = [&](int t, int buf) {
    const int k0 = t * KT;
    st.begin(K + (long long)k0 * a.k_rs, a.k_rs, V + (long long)k0 * a.v_rs, a.v_rs, min(KT, e.kl - k0), a.dh, lds + buf * (KE + VE),
             lds + buf * (KE + VE) + KE);
    if (DOCS && tid < KT) kd = k0 + tid < e.kl ? a.k_doc[e.k0 + k0 + tid] : 0;
  };
  const auto end = [&](int buf) {
    st.end(lds + buf * (KE + VE), lds + buf * (KE + VE) + KE);
    if (DOCS && tid < KT) docs[buf][tid] = kd;
  };
  int flags = 0, buf = 0, t = wk.next(0, flags);
  if (t < nk) begin(t, 0);                                 // (its latency and that of the row's own loads pass together)
  typename TL::Frag q[TL::NS];
  own_row<T, DHP>(q, (const T*)a.Q + e.q0 * a.q_rs + (long long)h * a.dh, a.q_rs, e.ql, a.dh, iw, l31, half);
  f32x16_t o[TL::NDT];
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) o[dt] = zero16();
  // l: the sum of the weights, for lse; lr: of the weights as the product with V has them.  The output is divided by lr: a row of few keys then keeps
  // what the rounding of its large weight does out of rowsum(dout out), which the backward subtracts from nearly the same number (error of dQ
  // and dK: 0.0025 of their norm instead of 0.0028 in capped sessions; 164 -> 171 us at 2 x 4096 causal, 16 heads of 128)
  float m = -INFINITY, l = 0.f, lr = 0.f;
  if (t < nk) end(0);
  __syncthreads();
  while (t < nk) {
    int nflags = 0;
    const int tn = wk.next(t + 1, nflags), k0 = t * KT;
    if (tn < nk) begin(tn, NB == 2 ? buf ^ 1 : 0);
    const T* Kl = lds + buf * (KE + VE);
    const T* Vl = Kl + KE;
    const bool work = active && k0 < lim_w && (flags & 1), docs_differ = DOCS && (flags & 2) && k0 + KT > e.pre;
    if (work) {
      f32x16_t s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = zero16();
#pragma unroll
        for (int x = 0; x < TL::NS; ++x) s[u] = TL::mma(TL::natural(Kl, u, l31, x, half), q[x], s[u]);
      }
      settle(s[0], s[1]);
      if (SHAPE) {
        if (SHAPE >= 2) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = sh.cap.less<SHAPE == 3>(s[u][r], sh.cap.r(s[u][r]), 0.f);
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] *= sh.cap.c1;
        }
        if (SHAPE == 1 || sh.slope) {
          const float d0 = (float)(i + e.off - k0 - 4 * half);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = __builtin_fmaf(-sh.sl2, fabsf(d0 - (float)(32 * u + reg_row(r, 0))), s[u][r]);
        }
      }
      // masked places become -inf: only in the tiles that the lengths, the diagonal or a document boundary cross
      const bool cut = k0 + KT > e.kl || (a.causal && k0 + KT > e.pre && k0 + KT - 1 > iw + e.off);
      if (docs_differ && !cut && k0 >= e.pre) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4 d = *reinterpret_cast<const int4*>(&docs[buf][32 * u + 8 * g + 4 * half]);
            const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) s[u][4 * g + c] = dd[c] == qd ? s[u][4 * g + c] : -INFINITY;
          }
      } else if (docs_differ) {
        const int pre = e.pre - k0 - 4 * half, lm = lim0 - k0 - 4 * half;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4 d = *reinterpret_cast<const int4*>(&docs[buf][32 * u + 8 * g + 4 * half]);
            const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int key = 32 * u + 8 * g + c;
              s[u][4 * g + c] = (key < pre || (key < lm && dd[c] == qd)) ? s[u][4 * g + c] : -INFINITY;
            }
          }
      } else if (cut) {
        const int lm = lim - k0 - 4 * half;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + reg_row(r, 0) < lm ? s[u][r] : -INFINITY;
      }
      float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, fmaxf(s[0][r], s[1][r]));
      mx = fmaxf(mx, other_half(mx));
      const float c = SHAPE ? 1.f : sh.cap.c1;
      const float mt = mx * c;
      if (__any(mt > m + 8.f)) {
        const float mn = fmaxf(m, mt), f = m == -INFINITY ? 0.f : exp2_hw(m - mn);
        m = mn;
        l *= f;
        lr *= f;
#pragma unroll
        for (int dt = 0; dt < TL::NDT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= f;
      }
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[u][r] = exp2_hw(SHAPE ? s[u][r] - mu : __builtin_fmaf(s[u][r], c, -mu));
          l += s[u][r];
        }
        TL::accumulate(o, Vl, 32 * u, s[u], lane, sizeof(T) == 2 ? &lr : nullptr);
      }
    }
    if (NB == 1) __syncthreads();
    if (tn < nk) end(NB == 2 ? buf ^ 1 : 0);
    __syncthreads();
    if (NB == 2) buf ^= 1;
    t = tn;
    flags = nflags;
  }
  if (!active) return;
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) settle(o[dt]);
  l += other_half(l);
  lr = sizeof(T) == 2 ? lr + other_half(lr) : l;
  const float inv = lr == 0.f ? 0.f : 1.f / lr;
  float bad = 0.f;
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) bad += not_finite(o[dt], dt, half, a.dh);
  const long long row = e.q0 + i;
  const bool in = i < e.ql;
  if (in) {
    T* O = (T*)a.out + row * a.o_rs + (long long)h * a.dh;
#pragma unroll
    for (int dt = 0; dt < TL::NDT; ++dt) store_dims<T>(o[dt], inv, O, dt, half, a.dh);
    if (sizeof(T) == 2 && a.out_lo) {
      T* L = (T*)a.out_lo + (row * a.Hq + h) * a.dh;
#pragma unroll
      for (int dt = 0; dt < TL::NDT; ++dt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = o[dt][r] * inv;
          o[dt][r] = x - bf2f(f2bf(x));
        }
        store_dims<T>(o[dt], 1.f, L, dt, half, a.dh);
      }
    }
    if (a.lse && half == 0) a.lse[row * a.Hq + h] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
  }
  // (a sum that is NaN: so is a score that the row sees, and the whole row)
  unsigned long long again = __ballot(in && !(bad == 0.f) && l == l);
  again |= again >> 32;
  if (!again) return;
  const unsigned long long dims = not_finite_bits<TL::NDT>(o, half, a.dh);
  for (int r = 0; r < 32; ++r)
    if ((again >> r) & 1)
      row_fwd<T>(*args_again(), e, h, iw + r, dim_of_row(dims, r, 0, lane), dim_of_row(dims, r, 1, lane), (float*)lds + wave * ROW_LDS, lane);
}

// (least, largest) document id of every 64 rows, of the queries (blockIdx.z = 0) and of the keys: tiles that share no id are skipped, tiles of
// one id need no mask
__global__ __launch_bounds__(256) void doc_ranges_kernel(const Args a) {
  const bool keys = blockIdx.z == 1;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y, lane = threadIdx.x & 63, nt = keys ? a.nkt : a.nqt;
  if (t >= nt) return;
  const Ex e = example(a, b);
  const int i = t * 64 + lane, len = keys ? e.kl : e.ql;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
  if (i < len) lo = hi = keys ? a.k_doc[e.k0 + i] : a.q_doc[e.q0 + i];
  for (int s = 32; s; s >>= 1) {
    lo = min(lo, __shfl_xor(lo, s));
    hi = max(hi, __shfl_xor(hi, s));
  }
  if (lane == 0) (keys ? a.k_rng : a.q_rng)[(long long)b * nt + t] = make_int2(lo, hi);
}

template <typename T, int DHP, int NW> void launch_tile_as(const Args& a, hipStream_t st) {
  const int nt = (int)cdiv64(a.max_q, 32 * NW);
  const unsigned grid = (unsigned)((long long)nt * a.Hq * a.B);
  with_shape<T>(a, [&](auto shape, auto docs) { tile_fwd_kernel<T, DHP, decltype(shape)::value, decltype(docs)::value, NW><<<grid, 64 * NW, 0, st>>>(a, nt); });
}
template <typename T, int DHP> void launch_tile(const Args& a, hipStream_t st) {
  if constexpr (DHP <= 80) {
    if (rows_of(a, DHP) == 64) return launch_tile_as<T, DHP, 2>(a, st);
  }
  launch_tile_as<T, DHP, 4>(a, st);
}
template <typename T> int launch_fwd(const Args& a, hipStream_t st) {
  if (a.dh <= 32) launch_tile<T, 32>(a, st);
  else if (a.dh <= 64) launch_tile<T, 64>(a, st);
  else if (a.dh <= 80) launch_tile<T, 80>(a, st);
  else launch_tile<T, 128>(a, st);
  DMT_CHECK_LAUNCH("dmt_attn_var_fwd");
  return DMT_OK;
}

}  // namespace

static uint64_t up16(uint64_t x) { return (x + 15) & ~15ull; }

extern "C" int dmt_attn_var_supported(int32_t dtype, int32_t dh, int32_t Hq, int32_t Hkv) {
  if (dtype != DMT_F32 && dtype != DMT_BF16) return 0;
  if (dh <= 0 || dh > MAX_DH || dh % (dtype == DMT_F32 ? 4 : 8)) return 0;
  return Hq > 0 && Hkv > 0 && Hq % Hkv == 0;
}

namespace {
// dK, dV: a workgroup walks over the query heads of its group and over the queries.  When that leaves fewer than four workgroups a compute unit
// the walk is cut into pieces that run side by side and leave fp32 sums to be added in their order: first by head, then by ranges of at least
// 256 queries.  (Two, four, eight a unit: 4 histories of 2048 in sessions 116, 65, 89 us; 2 x 4096 causal, 16 heads of 128, dK: 288, 225, 225 us.)
int parts_of(const dmt_attn_var_desc* d, int* qparts) {
  const int64_t G = d->Hq / d->Hkv, base = (int64_t)d->B * d->Hkv * cdiv64(d->max_k, 128), want = 1024;
  const int64_t p = base > 0 ? cdiv64(want, base) : 1, hp = p < G ? p : G;
  int64_t qp = base > 0 ? cdiv64(want, base * hp) : 1;
  if (qp > d->max_q / 256) qp = d->max_q / 256;
  if (qp < 1) qp = 1;
  *qparts = (int)qp;
  return (int)(hp * qp);
}
struct WsLayout { uint64_t D, sp, pk, pv, total; };
WsLayout ws_layout(const dmt_attn_var_desc* d) {
  WsLayout w;
  uint64_t at = 0;
  w.D = at;
  at += up16(4 * (uint64_t)d->rows_q * (uint64_t)d->Hq);
  w.sp = at;
  if (d->dslopes) at += up16(4 * (uint64_t)d->Hq * (uint64_t)d->B * (uint64_t)cdiv64(d->max_q, 64));
  int qparts;
  const int parts = parts_of(d, &qparts);
  const uint64_t part = parts > 1 ? up16(4 * (uint64_t)parts * (uint64_t)d->rows_k * (uint64_t)d->Hkv * (uint64_t)d->dh) : 0;
  w.pk = at;
  at += part;
  w.pv = at;
  w.total = at + part;
  return w;
}
bool al16(const void* p, int64_t rs, int es) { return ((uintptr_t)p % 16) == 0 && (rs * es) % 16 == 0; }
}  // namespace

extern "C" uint64_t dmt_attn_var_ws_bytes(const dmt_attn_var_desc* d) {
  if (!d || d->B <= 0 || d->max_q < 0 || d->max_k < 0 || d->Hkv <= 0 || d->Hq < d->Hkv || d->dh <= 0 || d->rows_q < 0 || d->rows_k < 0) return 0;
  return ws_layout(d).total;
}
extern "C" uint64_t dmt_attn_var_doc_bytes(int32_t B, int32_t max_q, int32_t max_k) {
  if (B <= 0 || max_q < 0 || max_k < 0) return 0;
  return up16(8 * (uint64_t)B * (uint64_t)cdiv64(max_q, 64)) + up16(8 * (uint64_t)B * (uint64_t)cdiv64(max_k, 64));
}

int dmt_attn_var_args(const dmt_attn_var_desc* d, Args* a, bool backward, const char* what) {
  DMT_CHECK_ARG(d, "%s: no descriptor", what);
  DMT_CHECK_ARG(d->B >= 0 && d->max_q >= 0 && d->max_k >= 0 && d->rows_q >= 0 && d->rows_k >= 0, "%s: negative size", what);
  DMT_CHECK_ARG(dmt_attn_var_supported(d->dtype, d->dh, d->Hq, d->Hkv),
                "%s: needs bf16 (dh %% 8 == 0) or fp32 (dh %% 4 == 0), dh <= 128 and Hq a multiple of Hkv: got dtype %d, dh %d, Hq %d, Hkv %d", what,
                d->dtype, d->dh, d->Hq, d->Hkv);
  DMT_CHECK_ARG((int64_t)d->B * d->Hq * (cdiv64(d->max_q > d->max_k ? d->max_q : d->max_k, 64) + 1) < (1ll << 31), "%s: B * Hq * max length / 64 passes 2^31", what);
  DMT_CHECK_ARG(d->B <= 65535 && d->Hq <= 65535, "%s: B and Hq <= 65535", what);
  DMT_CHECK_ARG(d->rows_q < (1ll << 31) && d->rows_k < (1ll << 31), "%s: row numbers are int32", what);
  DMT_CHECK_ARG(d->scale > 0.f && d->scale <= 1e38f, "%s: scale must be positive and at most 1e38", what);
  DMT_CHECK_ARG(d->cap >= 0.f && d->cap <= 1e38f, "%s: cap must be 0 (none) or positive and at most 1e38", what);
  DMT_CHECK_ARG((d->q_doc == nullptr) == (d->k_doc == nullptr), "%s: q_doc and k_doc go together", what);
  if (d->B == 0) {                       // no example: only a slopes' gradient is owed, and nothing is read
    if (!backward || !d->dslopes) return 1;
    *a = Args{};
    a->Hq = d->Hq;
    a->dslopes = d->dslopes;
    return DMT_OK;
  }
  if (d->max_q == 0 || d->rows_q == 0) {
    // no query row: the forward has nothing to do, the backward still owes dk = dv = 0 and dslopes = 0
    if (!backward || ((d->max_k == 0 || d->rows_k == 0) && !d->dslopes)) return 1;
  }
  DMT_CHECK_ARG(d->q_off && d->q_lens && d->k_off && d->k_lens, "%s: NULL offsets or lengths", what);
  const int es = d->dtype == DMT_F32 ? 4 : 2;
  const int64_t wq = (int64_t)d->Hq * d->dh, wk = (int64_t)d->Hkv * d->dh;
  DMT_CHECK_ARG(d->rows_q == 0 || (d->Q && d->out), "%s: NULL Q / out", what);
  DMT_CHECK_ARG(d->rows_k == 0 || (d->K && d->V), "%s: NULL K / V", what);
  DMT_CHECK_ARG(d->q_rs >= wq && d->k_rs >= wk && d->v_rs >= wk && (d->rows_q == 0 || d->o_rs >= wq), "%s: row stride shorter than a row", what);
  DMT_CHECK_ARG(d->k_rs * es < (1ll << 24) && d->v_rs * es < (1ll << 24) && d->q_rs * es < (1ll << 24) && d->o_rs * es < (1ll << 24),
                "%s: row stride of 16 MB or more", what);
  DMT_CHECK_ARG(al16(d->Q, d->q_rs, es) && al16(d->K, d->k_rs, es) && al16(d->V, d->v_rs, es) && al16(d->out, d->o_rs, es),
                "%s: operand rows must be 16-byte aligned", what);
  if (backward) {
    DMT_CHECK_ARG(d->rows_q == 0 || (d->dout && d->lse && d->dQ), "%s: NULL dout / lse / dQ", what);
    DMT_CHECK_ARG(d->rows_k == 0 || (d->dK && d->dV), "%s: NULL dK / dV", what);
    DMT_CHECK_ARG((d->rows_q == 0 || (d->do_rs >= wq && d->dq_rs >= wq)) && d->dk_rs >= wk && d->dv_rs >= wk && d->do_rs * es < (1ll << 24),
                  "%s: bad gradient row stride", what);
    DMT_CHECK_ARG(al16(d->dout, d->do_rs, es) && al16(d->dQ, d->dq_rs, es) && al16(d->dK, d->dk_rs, es) && al16(d->dV, d->dv_rs, es),
                  "%s: gradient rows must be 16-byte aligned", what);
    DMT_CHECK_ARG((uintptr_t)d->out_lo % 16 == 0, "%s: out_lo must be 16-byte aligned", what);
    DMT_CHECK_ARG(!d->dslopes || d->slopes, "%s: dslopes without slopes", what);
  }
  DMT_CHECK_ARG(!d->q_doc || (d->doc_ranges && ((uintptr_t)d->doc_ranges % 16) == 0), "%s: documents need doc_ranges (16-byte aligned)", what);
  WsLayout w = {0, 0, 0, 0, 0};
  if (backward) {
    w = ws_layout(d);
    DMT_CHECK_ARG(w.total == 0 || (d->ws && ((uintptr_t)d->ws % 16) == 0 && d->ws_bytes >= w.total), "%s: workspace of %llu bytes needed", what,
                  (unsigned long long)w.total);
  }
  DMT_CHECK_ARG(d->rows_q == 0 || (d->out != d->Q && d->out != d->K && d->out != d->V), "%s: out must not be an operand", what);
  char* ws = (char*)d->ws;
  a->B = d->B; a->Hq = d->Hq; a->Hkv = d->Hkv; a->dh = d->dh; a->G = d->Hq / d->Hkv;
  a->max_q = d->max_q; a->max_k = d->max_k; a->rows_q = d->rows_q; a->rows_k = d->rows_k;
  a->Q = d->Q; a->q_rs = d->q_rs; a->K = d->K; a->k_rs = d->k_rs; a->V = d->V; a->v_rs = d->v_rs;
  a->q_off = d->q_off; a->q_lens = d->q_lens; a->k_off = d->k_off; a->k_lens = d->k_lens;
  a->scale = d->scale; a->cap = d->cap; a->causal = d->causal != 0; a->slopes = d->slopes; a->prefix = d->prefix;
  a->q_doc = d->q_doc; a->k_doc = d->k_doc;
  a->out = d->out; a->o_rs = d->o_rs; a->lse = d->lse; a->out_lo = d->dtype == DMT_BF16 ? d->out_lo : nullptr;
  a->dout = d->dout; a->do_rs = d->do_rs; a->dQ = d->dQ; a->dq_rs = d->dq_rs; a->dK = d->dK; a->dk_rs = d->dk_rs; a->dV = d->dV; a->dv_rs = d->dv_rs;
  a->dslopes = d->dslopes;
  a->nqt = (int)cdiv64(d->max_q, 64);
  a->nkt = (int)cdiv64(d->max_k, 64);
  a->q_rng = (int2*)d->doc_ranges;
  a->k_rng = d->q_doc ? (int2*)((char*)d->doc_ranges + up16(8 * (uint64_t)d->B * (uint64_t)a->nqt)) : nullptr;
  a->D = backward ? (float*)(ws + w.D) : nullptr;
  a->slope_part = backward && d->dslopes ? (float*)(ws + w.sp) : nullptr;
  a->parts = a->qparts = 1;
  if (backward) a->parts = parts_of(d, &a->qparts);
  a->part_k = backward ? (float*)(ws + w.pk) : nullptr;
  a->part_v = backward ? (float*)(ws + w.pv) : nullptr;
  return DMT_OK;
}

extern "C" int dmt_attn_var_fwd(const dmt_attn_var_desc* d, void* stream) {
  Args a;
  const int rc = dmt_attn_var_args(d, &a, false, "dmt_attn_var_fwd");
  if (rc) return rc < 0 ? rc : DMT_OK;
  if (a.q_doc) {
    const int nt = a.nqt > a.nkt ? a.nqt : a.nkt;
    doc_ranges_kernel<<<dim3((nt + 3) / 4, a.B, 2), 256, 0, (hipStream_t)stream>>>(a);
    DMT_CHECK_LAUNCH("dmt_attn_var_fwd(document ranges)");
  }
  return d->dtype == DMT_F32 ? launch_fwd<float>(a, (hipStream_t)stream) : launch_fwd<bf16_t>(a, (hipStream_t)stream);
}
