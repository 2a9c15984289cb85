// Attention over packed rows of any length: backward.  Two kernels recompute the weights from the saved row sums -- one owns query rows (dQ and
// the slopes' gradient), one owns key rows (dK, dV, over all query heads of the group) -- so that nothing is added by atomics.
// P and dX are rounded to bf16 as operands of the matrix instructions: measured error of dQ and dK 0.0024 of their norm, 0.0017 of it the rounding of
// the result itself; a second product with what the rounding took away would cost a third of the matrix time for that difference.  With documents,
// where few keys share a row and D (from the rounded weights of the output) adds to it, 0.0025 in capped sessions, it is done for dX: 0.0017 (4
// histories of 2048 in sessions, forward and backward: 166 instead of 161 us; the chain of a walk bounds them, not the matrix pipe).
#include "dmt_attn_var.h"

using namespace attn_var;

namespace {

// The scores of one 32 x 32 tile, in place: z2 minus the row statistic (kept in rows or, stat[], in registers).  d0: distance of register row 0
// and the lane's column; STEP: what a register row adds to it.  cr: what the cap's derivative needs.
template <int SHAPE, int STEP, typename STAT>
__device__ __forceinline__ void weights(f32x16_t& s, f32x16_t& cr, const Shape& sh, float d0, STAT stat) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float z;
    if (SHAPE >= 2) {
      cr[r] = sh.cap.r(s[r]);
      z = sh.cap.less<SHAPE == 3>(s[r], cr[r], stat(r));
    } else {
      z = __builtin_fmaf(s[r], sh.cap.c1, -stat(r));
    }
    if (SHAPE == 1 || (SHAPE >= 2 && sh.slope)) z = __builtin_fmaf(-sh.sl2, fabsf(d0 + (float)(STEP * reg_row(r, 0))), z);
    s[r] = exp2_hw(z);
  }
}

// dQ (and D): one workgroup owns 128 or 64 queries of a head, as in the forward: S^T and dP^T with lane = query, dX packed is the B operand of
// dQ^T += K^T dX.  Bound by the matrix pipe: 2 x 4096 causal, 16 heads of 128: 210 us = 977 TFLOP/s; 256 histories of up to 200, 4 heads of 80: 46 us.
template <typename T, int DHP, int SHAPE, bool DOCS, int NW>
__global__ __launch_bounds__(64 * NW, 2) void tile_dq_kernel(const Args a, int nt) {
  typedef Tile<T, DHP> TL;
  constexpr int NB = sizeof(T) == 2 ? 2 : 1, ROWS = 32 * NW;
  constexpr int PAD = sizeof(T) == 2 ? 0 : 32, KE = KT * TL::RS + PAD, VE = KT * TL::RS;
  __shared__ __attribute__((aligned(16))) T lds[NB * (KE + VE)];
  __shared__ __attribute__((aligned(16))) int docs[DOCS ? NB : 1][KT];
  __shared__ float part[NW];
  static_assert(sizeof(lds) >= NW * ROW_LDS * sizeof(float), "the row form works in the tiles' memory");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l31 = lane & 31;
  int head, qt;
  place(blockIdx.x, a.B * a.Hq, nt, a.causal, head, qt);
  const int b = head / a.Hq, h = head - b * a.Hq, hk = h / a.G;
  const Ex e = example(a, b);
  if (qt * ROWS >= e.ql) {
    if (a.slope_part && tid == 0) a.slope_part[((long long)h * a.B + b) * nt + qt] = 0.f;
    return;
  }
  const int iw = qt * ROWS + wave * 32, i = iw + l31;
  const bool active = iw < e.ql, in = i < e.ql;
  const T* K = (const T*)a.K + e.k0 * a.k_rs + (long long)hk * a.dh;
  const T* V = (const T*)a.V + e.k0 * a.v_rs + (long long)hk * a.dh;
  const Shape sh = shape_of<T>(a, h);
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
    qd = in ? a.q_doc[e.q0 + i] : 0;
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
  if (t < nk) begin(t, 0);                               // (its latency and that of the rows' own loads pass together)
  typename TL::Frag q[TL::NS], g[TL::NS];
  own_row<T, DHP>(q, (const T*)a.Q + e.q0 * a.q_rs + (long long)h * a.dh, a.q_rs, e.ql, a.dh, iw, l31, half);
  own_row<T, DHP>(g, (const T*)a.dout + e.q0 * a.do_rs + (long long)h * a.dh, a.do_rs, e.ql, a.dh, iw, l31, half);
  const long long stat = (e.q0 + (in ? i : 0)) * a.Hq + h;
  // (a row that sees nothing: lse = -inf; its weights 2^(z - inf) are 0)
  const float lse = a.lse[stat], lse2 = in && lse != -INFINITY ? lse * LOG2E : INFINITY;
  float D = 0.f;                                         // rowsum(dout * out), for this kernel and the next
  {
    typename TL::Frag ov[TL::NS];
    own_row<T, DHP>(ov, (const T*)a.out + e.q0 * a.o_rs + (long long)h * a.dh, a.o_rs, e.ql, a.dh, iw, l31, half);
#pragma unroll
    for (int x = 0; x < TL::NS; ++x) D = TL::dot(g[x], ov[x], D);
    if (sizeof(T) == 2 && a.out_lo) {
      const long long ls = (long long)a.Hq * a.dh;
      own_row<T, DHP>(ov, (const T*)a.out_lo + e.q0 * ls + (long long)h * a.dh, ls, e.ql, a.dh, iw, l31, half);
#pragma unroll
      for (int x = 0; x < TL::NS; ++x) D = TL::dot(g[x], ov[x], D);
    }
    D += other_half(D);
    if (in && half == 0) a.D[stat] = D;
  }
  f32x16_t o[TL::NDT];
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) o[dt] = zero16();
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, sp = 0.f;
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
      const bool cut = k0 + KT > e.kl || (a.causal && k0 + KT > e.pre && k0 + KT - 1 > iw + e.off);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x16_t s = zero16(), dp = zero16(), cr;
#pragma unroll
        for (int x = 0; x < TL::NS; ++x) {
          s = TL::mma(TL::natural(Kl, u, l31, x, half), q[x], s);
          dp = TL::mma(TL::natural(Vl, u, l31, x, half), g[x], dp);
        }
        const float d0 = (float)(i + e.off - k0 - 32 * u - 4 * half);
        settle(s, dp);
        weights<SHAPE, -1>(s, cr, sh, d0, [&](int) { return lse2; });
        if (docs_differ || cut) {
          // (a masked place gives weight and gradient 0 whatever stands there)
          const int pre = e.pre - k0 - 32 * u - 4 * half, lm = (docs_differ ? lim0 : lim) - k0 - 32 * u - 4 * half;
#pragma unroll
          for (int gg = 0; gg < 4; ++gg) {
            int4 d = make_int4(qd, qd, qd, qd);
            if (docs_differ) d = *reinterpret_cast<const int4*>(&docs[buf][32 * u + 8 * gg + 4 * half]);
            const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int key = 8 * gg + c;
              const bool ok = key < pre || (key < lm && dd[c] == qd);
              s[4 * gg + c] = ok ? s[4 * gg + c] : 0.f;
              dp[4 * gg + c] = ok ? dp[4 * gg + c] : 0.f;
            }
          }
        }
        if (SHAPE && a.slope_part) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float ad = fabsf(d0 - (float)reg_row(r, 0)), pd = s[r] * dp[r];
            s0 += pd;
            s1 = __builtin_fmaf(pd, ad, s1);
            s2 = __builtin_fmaf(s[r], ad, s2);
            sp += s[r];
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] *= dp[r] - D;
          if (SHAPE >= 2) s[r] *= dmt_cap::derivative(cr[r]);
        }
        TL::template accumulate<DOCS>(o, Kl, 32 * u, s, lane);
      }
    }
    if (NB == 1) __syncthreads();
    if (tn < nk) end(NB == 2 ? buf ^ 1 : 0);
    __syncthreads();
    if (NB == 2) buf ^= 1;
    t = tn;
    flags = nflags;
  }
  float sl = 0.f;
  if (active) {
#pragma unroll
    for (int dt = 0; dt < TL::NDT; ++dt) settle(o[dt]);
    if (SHAPE && a.slope_part) {
      s0 += other_half(s0);
      s1 += other_half(s1);
      s2 += other_half(s2);
      sp += other_half(sp);
      sl = in ? slope_part(s0, s1, s2, sp) : 0.f;
    }
    float bad = 0.f;                                     // (sl holds: what is masked was zeroed in both of its factors)
#pragma unroll
    for (int dt = 0; dt < TL::NDT; ++dt) bad += not_finite(o[dt], dt, half, a.dh);
    if (in) {
      T* O = (T*)a.dQ + (e.q0 + i) * a.dq_rs + (long long)h * a.dh;
#pragma unroll
      for (int dt = 0; dt < TL::NDT; ++dt) store_dims<T>(o[dt], a.scale, O, dt, half, a.dh);
    }
    // (a row that sees something, and whose lse or D is NaN, is NaN)
    unsigned long long again = __ballot(in && !(bad == 0.f) && (lse == -INFINITY || (lse == lse && D == D)));
    again |= again >> 32;
    if (half) sl = 0.f;                                  // (both halves hold the row's)
    sl = wave_sum(sl);
    if (again) {
      const unsigned long long dims = not_finite_bits<TL::NDT>(o, half, a.dh);
      for (int r = 0; r < 32; ++r)
        if ((again >> r) & 1)
          row_dq<T>(*args_again(), e, h, iw + r, __shfl(D, r), dim_of_row(dims, r, 0, lane), dim_of_row(dims, r, 1, lane), (float*)lds + wave * ROW_LDS, lane);
    }
  }
  if (a.slope_part) {
    if (lane == 0) part[wave] = sl;
    __syncthreads();
    if (tid == 0) a.slope_part[((long long)h * a.B + b) * nt + qt] = NW == 4 ? (part[0] + part[1]) + (part[2] + part[NW - 1]) : part[0] + part[1];
  }
}

// dslopes[h] = sum of its parts, in their order (64 bits: the terms cancel)
__device__ void sum_slopes(const float* part, long long n, float* out, double* red) {
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += 256) s += (double)part[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) *out = (float)red[0];
}

__global__ __launch_bounds__(256) void slopes_kernel(const Args a, long long n) {
  __shared__ double red[256];
  sum_slopes(a.slope_part + (long long)blockIdx.x * n, n, a.dslopes + blockIdx.x, red);
}

// dK, dV: one workgroup owns 128 keys (a wavefront 32, their K and V rows in registers) and walks over the queries of every head of the group in
// tiles of 64: S and dP with lane = key, P and dX packed are the B operands of dV^T += dO^T P and dK^T += Q^T dX.  Nothing crosses wavefronts.
// WHAT: 1 = dK, 2 = dV, 3 = both.  Both accumulators and both operands' rows fit the 256 registers of two wavefronts a SIMD up to 80 dims (64 in
// fp32); wider heads take a kernel each -- one more product of scores, but at 4096 causal keys, 16 heads of 128 dims 221 + 164 us against 443 us
// for one kernel with one wavefront a SIMD (accumulators moved between register files) and 1033 us with spills.  (930 and 835 TFLOP/s; up to 80 dims
// two kernels would lose: 4 histories of 2048 in sessions 77 to 92 us against 71 to 84 for one.)  256 histories of up to 200, 4 heads of 80: 49 us.
template <typename T, int DHP, int SHAPE, bool DOCS, int WHAT>
__global__ __launch_bounds__(256, 2) void tile_dkv_kernel(const Args a, int nt, int nqt) {
  typedef Tile<T, DHP> TL;
  constexpr int NB = sizeof(T) == 2 ? 2 : 1;
  constexpr int QE = KT * TL::RS + (sizeof(T) == 2 ? 0 : 32);
  __shared__ __attribute__((aligned(16))) T lds[NB * 2 * QE];
  __shared__ __attribute__((aligned(16))) int docs[DOCS ? NB : 1][KT];
  __shared__ __attribute__((aligned(16))) float stats[NB][2][KT];
  static_assert(sizeof(lds) >= 4 * ROW_LDS * sizeof(float), "the row form works in the tiles' memory");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l31 = lane & 31;
  const int id = (int)blockIdx.x - (SHAPE && (WHAT & 1) && a.slope_part ? a.Hq : 0);
  if (SHAPE && (WHAT & 1) && id < 0) {                                 // the first workgroups finish the slopes' gradient that the dQ kernel left in parts
    const long long n = (long long)a.B * nqt;
    sum_slopes(a.slope_part + (long long)blockIdx.x * n, n, a.dslopes + blockIdx.x, (double*)lds);
    return;
  }
  int head, kt;
  place(id, a.B * a.Hkv * a.parts, nt, false, head, kt);
  const int part = head % a.parts, b = head / (a.parts * a.Hkv), hk = head / a.parts - b * a.Hkv;
  const int g0 = part_head(a, part / a.qparts), ng = part_head(a, part / a.qparts + 1) - g0;
  const Ex e = example(a, b);
  if (kt * 128 >= e.kl) return;
  const int jw = kt * 128 + wave * 32, j = jw + l31;
  const bool active = jw < e.kl;
  // queries that may see some key of the workgroup / wavefront / lane: from `lo` on (rows before it sit above the diagonal, unless the key
  // belongs to the prefix)
  const int lo_wg = a.causal && kt * 128 >= e.pre ? max(0, kt * 128 - e.off) : 0;
  const int lo_w = a.causal && jw >= e.pre ? max(0, jw - e.off) : 0;
  const int lo_l = j >= e.kl ? 0x7fffffff : (a.causal && j >= e.pre ? max(0, j - e.off) : 0);
  const int nq = (e.ql + KT - 1) / KT, tl = lo_wg / KT, span = nq > tl ? nq - tl : 0, qp = part % a.qparts;
  const int t0 = tl + (int)((long long)span * qp / a.qparts), t1 = tl + (int)((long long)span * (qp + 1) / a.qparts);
  int kd_l = 0;
  Walk<DOCS> wk;
  wk.hi = t1;
  if constexpr (DOCS) {
    wk.lo = t0;
    const int2* kr = a.k_rng + (long long)b * a.nkt;
    const int2 r0 = kr[kt * 2], r1 = kt * 2 + 1 < a.nkt ? kr[kt * 2 + 1] : r0, rw = wave < 2 ? r0 : r1;
    wk.rng = a.q_rng + (long long)b * a.nqt;
    wk.free_wg = kt * 128 < e.pre ? t1 : 0;              // (a key of the prefix: no document hides it from any query)
    wk.free_w = jw < e.pre ? t1 : 0;
    wk.glo = min(r0.x, r1.x);
    wk.ghi = max(r0.y, r1.y);
    wk.wlo = rw.x;
    wk.whi = rw.y;
    wk.chunk = -1;
    kd_l = j < e.kl ? a.k_doc[e.k0 + j] : 0;
  }
  Stage<T, DHP, 4> st;
  st.init(a.q_rs, a.do_rs, a.dh, tid);
  int qd = 0;
  float lse2 = 0.f;
  const auto begin = [&](int g, int t, int buf) {
    const int h = hk * a.G + g0 + g, i0 = t * KT;
    st.begin((const T*)a.Q + (e.q0 + i0) * a.q_rs + (long long)h * a.dh, a.q_rs, (const T*)a.dout + (e.q0 + i0) * a.do_rs + (long long)h * a.dh, a.do_rs,
             min(KT, e.ql - i0), a.dh, lds + buf * 2 * QE, lds + buf * 2 * QE + QE);
    if (tid < 2 * KT) {
      const int i = i0 + (tid & (KT - 1));
      const long long stat = (e.q0 + i) * a.Hq + h;
      if (tid < KT) {
        const float x = i < e.ql ? a.lse[stat] : -INFINITY;
        lse2 = x != -INFINITY ? x * LOG2E : INFINITY;     // (rows that see nothing, rows past the end: weight 0)
        if (DOCS) qd = i < e.ql ? a.q_doc[e.q0 + i] : 0;
      } else {
        lse2 = i < e.ql ? a.D[stat] : 0.f;
      }
    }
  };
  const auto end = [&](int buf) {
    st.end(lds + buf * 2 * QE, lds + buf * 2 * QE + QE);
    if (tid < 2 * KT) stats[buf][tid / KT][tid & (KT - 1)] = lse2;
    if (DOCS && tid < KT) docs[buf][tid] = qd;
  };
  f32x16_t dk[WHAT & 1 ? TL::NDT : 1], dv[WHAT & 2 ? TL::NDT : 1];
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) {
    if (WHAT & 1) dk[dt] = zero16();
    if (WHAT & 2) dv[dt] = zero16();
  }
  // the walk: the heads of the part one after the other, each over the tiles to visit
  int flags = 0, buf = 0, g = 0, t = wk.next(t0, flags);
  if (t >= t1) g = ng;
  const int first = t, first_flags = flags;
  if (g < ng) begin(0, t, 0);
  typename TL::Frag k[TL::NS], v[TL::NS];
  own_row<T, DHP>(k, (const T*)a.K + e.k0 * a.k_rs + (long long)hk * a.dh, a.k_rs, e.kl, a.dh, jw, l31, half);
  if (WHAT & 1) own_row<T, DHP>(v, (const T*)a.V + e.k0 * a.v_rs + (long long)hk * a.dh, a.v_rs, e.kl, a.dh, jw, l31, half);
  if (g < ng) end(0);
  __syncthreads();
  while (g < ng) {
    int nflags = 0, gn = g, tn = wk.next(t + 1, nflags);
    if (tn >= t1) {
      ++gn;
      tn = first;
      nflags = first_flags;
    }
    const int i0 = t * KT;
    if (gn < ng) begin(gn, tn, NB == 2 ? buf ^ 1 : 0);
    const T* Ql = lds + buf * 2 * QE;
    const T* Gl = Ql + QE;
    const Shape sh = shape_of<T>(a, hk * a.G + g0 + g);
    const bool work = active && i0 + KT > lo_w && (flags & 1), docs_differ = DOCS && (flags & 2) && jw + 32 > e.pre;
    if (work) {
      const bool cut = jw + 32 > e.kl || (a.causal && jw + 32 > e.pre && i0 + e.off < jw + 31);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x16_t s = zero16(), dp = zero16(), cr;
#pragma unroll
        for (int x = 0; x < TL::NS; ++x) {
          s = TL::mma(TL::natural(Ql, u, l31, x, half), k[x], s);
          if (WHAT & 1) dp = TL::mma(TL::natural(Gl, u, l31, x, half), v[x], dp);
        }
        if (WHAT & 1) settle(s, dp);
        else settle(s);
        f32x4_t ls[4];
#pragma unroll
        for (int gg = 0; gg < 4; ++gg) ls[gg] = *reinterpret_cast<const f32x4_t*>(&stats[buf][0][32 * u + 8 * gg + 4 * half]);
        weights<SHAPE, 1>(s, cr, sh, (float)(i0 + 32 * u + 4 * half + e.off - j), [&](int r) { return ls[r >> 2][r & 3]; });
        if (docs_differ || cut) {
          const int lo = lo_l - i0 - 32 * u - 4 * half;
#pragma unroll
          for (int gg = 0; gg < 4; ++gg) {
            int4 d = make_int4(kd_l, kd_l, kd_l, kd_l);
            if (docs_differ && j >= e.pre) d = *reinterpret_cast<const int4*>(&docs[buf][32 * u + 8 * gg + 4 * half]);
            const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const bool ok = 8 * gg + c >= lo && dd[c] == kd_l;
              s[4 * gg + c] = ok ? s[4 * gg + c] : 0.f;
              dp[4 * gg + c] = ok ? dp[4 * gg + c] : 0.f;
            }
          }
        }
        if (WHAT & 2) TL::accumulate(dv, Gl, 32 * u, s, lane);
        if (!(WHAT & 1)) continue;
#pragma unroll
        for (int gg = 0; gg < 4; ++gg) {
          const float4 ds = *reinterpret_cast<const float4*>(&stats[buf][1][32 * u + 8 * gg + 4 * half]);
          const float D[4] = {ds.x, ds.y, ds.z, ds.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[4 * gg + c] *= dp[4 * gg + c] - D[c];
            if (SHAPE >= 2) s[4 * gg + c] *= dmt_cap::derivative(cr[4 * gg + c]);
          }
        }
        TL::template accumulate<DOCS>(dk, Ql, 32 * u, s, lane);
      }
    }
    if (NB == 1) __syncthreads();
    if (gn < ng) end(NB == 2 ? buf ^ 1 : 0);
    __syncthreads();
    if (NB == 2) buf ^= 1;
    g = gn;
    t = tn;
    flags = nflags;
  }
  if (!active) return;
  const bool in = j < e.kl;
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) {
    if (WHAT & 1) settle(dk[dt]);
    if (WHAT & 2) settle(dv[dt]);
  }
  float bad = 0.f;
#pragma unroll
  for (int dt = 0; dt < TL::NDT; ++dt) {
    if (WHAT & 1) bad += not_finite(dk[dt], dt, half, a.dh);
    if (WHAT & 2) bad += not_finite(dv[dt], dt, half, a.dh);
  }
  if (in && a.parts > 1) {
    const long long at = (((long long)part * a.rows_k + e.k0 + j) * a.Hkv + hk) * a.dh;
#pragma unroll
    for (int dt = 0; dt < TL::NDT; ++dt) {
      if (WHAT & 1) store_dims<float>(dk[dt], 1.f, a.part_k + at, dt, half, a.dh);
      if (WHAT & 2) store_dims<float>(dv[dt], 1.f, a.part_v + at, dt, half, a.dh);
    }
  } else if (in) {
    T* pk = (T*)a.dK + (e.k0 + j) * a.dk_rs + (long long)hk * a.dh;
    T* pv = (T*)a.dV + (e.k0 + j) * a.dv_rs + (long long)hk * a.dh;
#pragma unroll
    for (int dt = 0; dt < TL::NDT; ++dt) {
      if (WHAT & 1) store_dims<T>(dk[dt], a.scale, pk, dt, half, a.dh);
      if (WHAT & 2) store_dims<T>(dv[dt], 1.f, pv, dt, half, a.dh);
    }
  }
  unsigned long long again = __ballot(in && !(bad == 0.f));
  again |= again >> 32;
  if (!again) return;
  unsigned long long bk = 0, bv = 0;
  if (WHAT & 1) bk = not_finite_bits<TL::NDT>(dk, half, a.dh);
  if (WHAT & 2) bv = not_finite_bits<TL::NDT>(dv, half, a.dh);
  for (int r = 0; r < 32; ++r)
    if ((again >> r) & 1)
      row_dkv<T>(*args_again(), e, hk, part, t0 * KT, min(e.ql, t1 * KT), jw + r, dim_of_row(bk, r, 0, lane), dim_of_row(bk, r, 1, lane),
                 dim_of_row(bv, r, 0, lane), dim_of_row(bv, r, 1, lane), (float*)lds + wave * ROW_LDS, lane);
}

// dK = scale (sum of its parts), dV = sum of its parts, in their order: 16 key rows of one example a workgroup.  Bound by the parts' bytes (4 x 2 x 4096
// rows of 512, 134 MB of K and V: 35 us; 4 histories of 2048: 12 us).
template <typename T>
__global__ __launch_bounds__(256) void join_parts_kernel(const Args a) {
  const Ex e = example(a, blockIdx.y);
  const int w = a.Hkv * a.dh, c4 = w / 4, j0 = blockIdx.x * 16;
  const int rows = e.kl - j0 < 16 ? e.kl - j0 : 16;
  for (int x = threadIdx.x; x < rows * c4 * 2; x += 256) {
    const bool is_v = x >= rows * c4;
    const int y = is_v ? x - rows * c4 : x, r = y / c4, c = (y - r * c4) * 4;
    const long long row = e.k0 + j0 + r;
    const float* p = (is_v ? a.part_v : a.part_k) + row * w + c;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < a.parts; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(p + (long long)i * a.rows_k * w);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float f = is_v ? 1.f : a.scale;
    T* o = is_v ? (T*)a.dV + row * a.dv_rs + c : (T*)a.dK + row * a.dk_rs + c;
    if (sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(dmt_pack_bf16(s.x * f, s.y * f), dmt_pack_bf16(s.z * f, s.w * f));
    else *reinterpret_cast<float4*>(o) = make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
  }
}

template <typename T, int DHP, int NW> void launch_dq_as(const Args& a, hipStream_t st) {
  const int nt = (int)cdiv64(a.max_q, 32 * NW);
  const unsigned grid = (unsigned)((long long)nt * a.Hq * a.B);
  with_shape<T>(a, [&](auto shape, auto docs) { tile_dq_kernel<T, DHP, decltype(shape)::value, decltype(docs)::value, NW><<<grid, 64 * NW, 0, st>>>(a, nt); });
}
template <typename T, int DHP> void launch_dq(const Args& a, hipStream_t st) {
  if constexpr (DHP <= 80) {
    if (rows_of(a, DHP) == 64) return launch_dq_as<T, DHP, 2>(a, st);
  }
  launch_dq_as<T, DHP, 4>(a, st);
}
template <typename T, int DHP> void launch_dkv(const Args& a, int nt, int nqt, hipStream_t st) {
  const unsigned grid = (unsigned)((long long)nt * a.Hkv * a.B * a.parts), more = a.slope_part ? a.Hq : 0;
  with_shape<T>(a, [&](auto shape, auto docs) {
    constexpr int S = decltype(shape)::value;
    constexpr bool D = decltype(docs)::value;
    if constexpr (DHP > (sizeof(T) == 2 ? 80 : 64)) {
      tile_dkv_kernel<T, DHP, S, D, 2><<<grid, 256, 0, st>>>(a, nt, nqt);
      tile_dkv_kernel<T, DHP, S, D, 1><<<grid + more, 256, 0, st>>>(a, nt, nqt);
    } else {
      tile_dkv_kernel<T, DHP, S, D, 3><<<grid + more, 256, 0, st>>>(a, nt, nqt);
    }
  });
}

template <typename T>
int launch_bwd(Args a, hipStream_t st) {
  const int dhp = a.dh <= 32 ? 32 : (a.dh <= 64 ? 64 : (a.dh <= 80 ? 80 : 128));
  const int nqt = (int)cdiv64(a.max_q, rows_of(a, dhp)), nkt = (int)cdiv64(a.max_k, 128);
  if (a.rows_q && nqt) {
    if (a.dh <= 32) launch_dq<T, 32>(a, st);
    else if (a.dh <= 64) launch_dq<T, 64>(a, st);
    else if (a.dh <= 80) launch_dq<T, 80>(a, st);
    else launch_dq<T, 128>(a, st);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(dq)");
  }
  if (a.dslopes && (!nkt || !a.rows_q || !nqt)) {      // (no dK / dV kernel to finish them, or no query or example at all: n = 0)
    slopes_kernel<<<a.Hq, 256, 0, st>>>(a, a.rows_q && nqt ? (long long)a.B * nqt : 0);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(slopes)");
    a.slope_part = nullptr;
  }
  if (nkt) {
    if (a.dh <= 32) launch_dkv<T, 32>(a, nkt, nqt, st);
    else if (a.dh <= 64) launch_dkv<T, 64>(a, nkt, nqt, st);
    else if (a.dh <= 80) launch_dkv<T, 80>(a, nkt, nqt, st);
    else launch_dkv<T, 128>(a, nkt, nqt, st);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(dkv)");
    if (a.parts > 1 && a.rows_k) {
      join_parts_kernel<T><<<dim3((unsigned)cdiv64(a.max_k, 16), a.B), 256, 0, st>>>(a);
      DMT_CHECK_LAUNCH("dmt_attn_var_bwd(join)");
    }
  }
  return DMT_OK;
}

}  // namespace

extern "C" int dmt_attn_var_bwd(const dmt_attn_var_desc* d, void* stream) {
  Args a;
  int rc = dmt_attn_var_args(d, &a, true, "dmt_attn_var_bwd");
  if (rc) return rc < 0 ? rc : DMT_OK;
  return d->dtype == DMT_F32 ? launch_bwd<float>(a, (hipStream_t)stream) : launch_bwd<bf16_t>(a, (hipStream_t)stream);
}
