// What the kernels of dmt_attn_var.hip (forward) and dmt_attn_var_bwd.hip share: the arguments, the scores and masks, and the row kernels.
//
// Scores are kept in log2 units (z2 = z log2 e), so that a weight is one v_exp_f32: p = 2^(z2 - m2).
#pragma once
#include "dmt_common.h"

namespace attn_var {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int KT = 64;              // keys (dQ and forward) or queries (dK, dV) of one tile
constexpr int MAX_DH = 128;

struct Args {
  int B, Hq, Hkv, dh, G;
  int max_q, max_k;
  long long rows_q, rows_k;
  const void* Q; long long q_rs;
  const void* K; long long k_rs;
  const void* V; long long v_rs;
  const int* q_off; const int* q_lens; const int* k_off; const int* k_lens;
  float scale, cap;
  int causal;
  const float* slopes;
  const int* prefix;
  const int* q_doc; const int* k_doc;
  void* out; long long o_rs;
  float* lse;
  void* out_lo;
  const void* dout; long long do_rs;
  void* dQ; long long dq_rs;
  void* dK; long long dk_rs;
  void* dV; long long dv_rs;
  float* dslopes;
  float* D;                         // [rows_q, Hq]: rowsum(dout * out)
  float* slope_part;                // [Hq][B * tiles of the dQ kernel]
  int parts, qparts;                // dK, dV: heads of a group x query ranges in `parts` pieces (qparts ranges), summed by a launch of their own
  float* part_k; float* part_v;     // [parts][rows_k][Hkv * dh] when parts > 1
  int2* q_rng; int2* k_rng;         // (least, largest) document id of every 64-row tile: [B][ceil(max / 64)]
  int nqt, nkt;                     // 64-row tiles of max_q, max_k
};

// The arguments once more, for the part behind a kernel's loop that hardly ever runs: read from the argument segment there and then, so that
// they do not occupy (and spill) scalar registers in the loop.  Args is the first argument of every kernel that asks.
__device__ __forceinline__ const Args* args_again() {
  const void* p = (const void*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (const Args*)p;
}

// one example's lengths (as far as they are computed), the distance of its last key and last query, and what its queries may see
struct Ex {
  int ql, kl, off, pre;
  long long q0, k0;
};
// (a length is cut where its rows would leave the matrix, a start outside it leaves nothing: no index of a caller reaches past the operands)
__device__ __forceinline__ int clip_len(int len, int most, int first, long long rows) {
  if (first < 0 || len <= 0) return 0;
  long long m = len < most ? len : most;
  if (first + m > rows) m = rows - first;
  return m > 0 ? (int)m : 0;
}
__device__ __forceinline__ Ex example(const Args& a, int b) {
  Ex e;
  e.q0 = a.q_off[b];
  e.k0 = a.k_off[b];
  e.ql = clip_len(a.q_lens[b], a.max_q, (int)e.q0, a.rows_q);
  e.kl = clip_len(a.k_lens[b], a.max_k, (int)e.k0, a.rows_k);
  // positions are those of the lengths as they stand: what is cut off moves nothing that stays (the last 4096 numbers below 2^31 are kept free for the
  // rows and keys that a tile has beyond its example)
  const auto whole = [](int n) { return n < 0 ? 0 : (n < 0x7fffefff ? n : 0x7fffefff); };
  e.off = whole(a.k_lens[b]) - whole(a.q_lens[b]);
  const int p = a.prefix ? a.prefix[b] : 0;
  e.pre = p < 0 ? 0 : (p > e.kl ? e.kl : p);
  return e;
}

// constants of one head's scores: z2 = (capped ? cap(s) : cap.c1 s) - sl2 |distance|
struct Shape {
  dmt_cap cap;
  float sl2;       // slope log2e
  bool capped, slope;
};
template <typename T> __device__ __forceinline__ Shape shape_of(const Args& a, int h) {
  const bool slope = a.slopes != nullptr;
  return {dmt_cap(a.scale, a.cap, sizeof(T) == 2), slope ? a.slopes[h] * LOG2E : 0.f, a.cap > 0.f, slope};
}
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float z2_of(const Shape& s, float x, float dist) {
  float y = s.capped ? s.cap(x) : s.cap.c1 * x;
  if (s.slope) y = __builtin_fmaf(-s.sl2, fabsf(dist), y);
  return y;
}

template <typename T> __device__ __forceinline__ float dot_rows(const float* __restrict__ q, const T* __restrict__ k, int dh) {
  float s = 0.f;
  for (int c = 0; c < dh; ++c) s = __builtin_fmaf(q[c], ldf<T>(k + c), s);
  return s;
}

// ---------------------------------------------------------------------------------------------------------------- rows, one at a time
// One wavefront computes one row with plain arithmetic: 64 keys at a time, a lane per key for the scores, a lane per dim for the sums; only
// what the row may see is ever read into a sum.  It is the form that holds whatever the operands hold: the tile kernels multiply the
// weight 0 of a masked place into what stands there, so the dims of a row that come out of them not finite (s0, s1: of the lane's two) are computed
// again here.  NaN stays NaN: once all of them are, what the row may see has decided it and the rest is not looked at (a step whose operands
// hold NaN in every row pays for 64 keys a row, not for all: 2 x 2048 causal, 8 heads of 64, forward and backward: 2.7 ms; 48 without; 0.23 clean).
// lds: [2 * MAX_DH + 2 * 64] floats of the wavefront's own.
__device__ __forceinline__ bool all_nan(bool s0, float o0, bool s1, float o1) { return !__any((s0 && o0 == o0) || (s1 && o1 == o1)); }
__device__ __forceinline__ void lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
constexpr int ROW_LDS = 2 * MAX_DH + 2 * 64;

__device__ __forceinline__ bool may_see(const Args& a, const Ex& e, int i, int j, int qd) {
  if (j >= e.kl) return false;
  if (j < e.pre) return true;
  if (a.causal && j > i + e.off) return false;
  return a.q_doc == nullptr || a.k_doc[e.k0 + j] == qd;
}

template <typename T>
__device__ void row_fwd(const Args& a, const Ex& e, int h, int i, bool s0, bool s1, float* lds, int lane) {
  float* q = lds;
  float* pl = lds + 2 * MAX_DH;
  const int dh = a.dh, hk = h / a.G;
  const T* Q = (const T*)a.Q + (e.q0 + i) * a.q_rs + (long long)h * dh;
  const T* K = (const T*)a.K + e.k0 * a.k_rs + (long long)hk * dh;
  const T* V = (const T*)a.V + e.k0 * a.v_rs + (long long)hk * dh;
  for (int c = lane; c < dh; c += 64) q[c] = ldf<T>(Q + c);
  lds_fence();
  const Shape s = shape_of<T>(a, h);
  const int qd = a.q_doc ? a.q_doc[e.q0 + i] : 0;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < e.kl; j0 += 64) {
    const int j = j0 + lane;
    const bool ok = may_see(a, e, i, j, qd);
    const unsigned long long vis = __ballot(ok);
    if (!vis) continue;
    float z = -INFINITY;
    if (ok) z = z2_of(s, dot_rows<T>(q, K + (long long)j * a.k_rs, dh), (float)(i + e.off - j));
    const float mn = fmaxf(m, wave_max(z));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float p = ok ? exp2_hw(z - mu) : 0.f;
    const float f = m == -INFINITY ? 0.f : exp2_hw(m - mu);
    m = mn;
    l = l * f + wave_sum(p);
    o0 *= f;
    o1 *= f;
    pl[lane] = p;
    lds_fence();
    for (int t = 0; t < 64; ++t) {
      if (!((vis >> t) & 1)) continue;
      const float pt = pl[t];
      const T* v = V + (long long)(j0 + t) * a.v_rs;
      if (lane < dh) o0 = __builtin_fmaf(pt, ldf<T>(v + lane), o0);
      if (lane + 64 < dh) o1 = __builtin_fmaf(pt, ldf<T>(v + lane + 64), o1);
    }
    lds_fence();
    if (all_nan(s0, o0, s1, o1)) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;            // (nothing seen: 0; NaN stays)
  const long long row = e.q0 + i;
  T* O = (T*)a.out + row * a.o_rs + (long long)h * dh;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = lane + 64 * u;
    if (u ? s1 : s0) {
      const float o = (u ? o1 : o0) * inv;
      stf<T>(O + c, o);
      if (sizeof(T) == 2 && a.out_lo) stf<T>((T*)a.out_lo + (row * a.Hq + h) * dh + c, o - bf2f(f2bf(o)));
    }
  }
}

// one row's part of dslopes[h]:
//     - sum_j |d_j| P_j (dP_j - D)  =  S0 S2 - S1,   S0 = sum P dP, S1 = sum P dP |d|, S2 = sum P |d|,  each over Sp = sum P
// with D = S0 from the same weights, not from the rounded output: the terms cancel, and dslopes is an fp32 result.
__device__ __forceinline__ float slope_part(float s0, float s1, float s2, float sp) {
  const float i = sp == 0.f ? 0.f : 1.f / sp;
  return i * __builtin_fmaf(s0 * i, s2, -s1);
}
// dq of one row
template <typename T>
__device__ void row_dq(const Args& a, const Ex& e, int h, int i, float D, bool s0, bool s1, float* lds, int lane) {
  float* q = lds;
  float* g = lds + MAX_DH;
  float* xl = lds + 2 * MAX_DH;
  const int dh = a.dh, hk = h / a.G;
  const long long row = e.q0 + i;
  const T* K = (const T*)a.K + e.k0 * a.k_rs + (long long)hk * dh;
  const T* V = (const T*)a.V + e.k0 * a.v_rs + (long long)hk * dh;
  for (int c = lane; c < dh; c += 64) {
    q[c] = ldf<T>((const T*)a.Q + row * a.q_rs + (long long)h * dh + c);
    g[c] = ldf<T>((const T*)a.dout + row * a.do_rs + (long long)h * dh + c);
  }
  lds_fence();
  const Shape s = shape_of<T>(a, h);
  const int qd = a.q_doc ? a.q_doc[e.q0 + i] : 0;
  const float lse2 = a.lse[row * a.Hq + h] * LOG2E;
  float o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < e.kl; j0 += 64) {
    const int j = j0 + lane;
    const bool ok = may_see(a, e, i, j, qd);
    const unsigned long long vis = __ballot(ok);
    if (!vis) continue;
    float dx = 0.f;
    if (ok) {
      const float x = dot_rows<T>(q, K + (long long)j * a.k_rs, dh);
      const float p = exp2_hw(z2_of(s, x, (float)(i + e.off - j)) - lse2);
      dx = p * (dot_rows<T>(g, V + (long long)j * a.v_rs, dh) - D);
      if (s.capped) dx *= dmt_cap::derivative(s.cap.r(x));
    }
    xl[lane] = dx;
    lds_fence();
    for (int t = 0; t < 64; ++t) {
      if (!((vis >> t) & 1)) continue;
      const float xt = xl[t];
      const T* k = K + (long long)(j0 + t) * a.k_rs;
      if (lane < dh) o0 = __builtin_fmaf(xt, ldf<T>(k + lane), o0);
      if (lane + 64 < dh) o1 = __builtin_fmaf(xt, ldf<T>(k + lane + 64), o1);
    }
    lds_fence();
    if (all_nan(s0, o0, s1, o1)) break;
  }
  T* O = (T*)a.dQ + row * a.dq_rs + (long long)h * dh;
  if (s0) stf<T>(O + lane, o0 * a.scale);
  if (s1) stf<T>(O + lane + 64, o1 * a.scale);
}

// dk (sk) and dv (sv) of one key row: over the query heads of its group (those of one part), then over the queries (of one range)
__device__ __forceinline__ int part_head(const Args& a, int hp) { return (int)((long long)a.G * hp / (a.parts / a.qparts)); }
template <typename T>
__device__ void row_dkv(const Args& a, const Ex& e, int hk, int part, int i_lo, int i_hi, int j, bool sk0, bool sk1, bool sv0, bool sv1, float* lds, int lane) {
  float* k = lds;
  float* v = lds + MAX_DH;
  float* pl = lds + 2 * MAX_DH;
  float* xl = pl + 64;
  const int dh = a.dh;
  const long long row = e.k0 + j;
  for (int c = lane; c < dh; c += 64) {
    k[c] = ldf<T>((const T*)a.K + row * a.k_rs + (long long)hk * dh + c);
    v[c] = ldf<T>((const T*)a.V + row * a.v_rs + (long long)hk * dh + c);
  }
  lds_fence();
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  bool done = false;
  for (int h = hk * a.G + part_head(a, part / a.qparts); h < hk * a.G + part_head(a, part / a.qparts + 1) && !done; ++h) {
    const Shape s = shape_of<T>(a, h);
    const T* Q = (const T*)a.Q + e.q0 * a.q_rs + (long long)h * dh;
    const T* O = (const T*)a.dout + e.q0 * a.do_rs + (long long)h * dh;
    for (int i0 = i_lo; i0 < i_hi && !done; i0 += 64) {
      const int i = i0 + lane;
      const bool ok = i < i_hi && may_see(a, e, i, j, a.q_doc ? a.q_doc[e.q0 + i] : 0);
      const unsigned long long vis = __ballot(ok);
      if (!vis) continue;
      float p = 0.f, dx = 0.f;
      if (ok) {
        const long long qr = (e.q0 + i) * a.Hq + h;
        const float x = dot_rows<T>(k, Q + (long long)i * a.q_rs, dh);
        p = exp2_hw(z2_of(s, x, (float)(i + e.off - j)) - a.lse[qr] * LOG2E);
        dx = p * (dot_rows<T>(v, O + (long long)i * a.do_rs, dh) - a.D[qr]);
        if (s.capped) dx *= dmt_cap::derivative(s.cap.r(x));
      }
      pl[lane] = p;
      xl[lane] = dx;
      lds_fence();
      for (int t = 0; t < 64; ++t) {
        if (!((vis >> t) & 1)) continue;
        const float pt = pl[t], xt = xl[t];
        const T* qr = Q + (long long)(i0 + t) * a.q_rs;
        const T* gr = O + (long long)(i0 + t) * a.do_rs;
        if (lane < dh) {
          k0 = __builtin_fmaf(xt, ldf<T>(qr + lane), k0);
          v0 = __builtin_fmaf(pt, ldf<T>(gr + lane), v0);
        }
        if (lane + 64 < dh) {
          k1 = __builtin_fmaf(xt, ldf<T>(qr + lane + 64), k1);
          v1 = __builtin_fmaf(pt, ldf<T>(gr + lane + 64), v1);
        }
      }
      lds_fence();
      done = all_nan(sk0, k0, sk1, k1) && all_nan(sv0, v0, sv1, v1);
    }
  }
  if (a.parts > 1) {
    const long long at = (((long long)part * a.rows_k + row) * a.Hkv + hk) * dh + lane;
    if (sk0) a.part_k[at] = k0;
    if (sk1) a.part_k[at + 64] = k1;
    if (sv0) a.part_v[at] = v0;
    if (sv1) a.part_v[at + 64] = v1;
    return;
  }
  T* dk = (T*)a.dK + row * a.dk_rs + (long long)hk * dh + lane;
  T* dv = (T*)a.dV + row * a.dv_rs + (long long)hk * dh + lane;
  if (sk0) stf<T>(dk, k0 * a.scale);
  if (sk1) stf<T>(dk + 64, k1 * a.scale);
  if (sv0) stf<T>(dv, v0);
  if (sv1) stf<T>(dv + 64, v1);
}

// ---------------------------------------------------------------------------------------------------------------- tiles
// 32 x 32 products (v_mfma_f32_32x32x16_bf16, v_mfma_f32_32x32x2_f32): a lane l holds column l % 32 of the result and the 16 rows
// 8 (r / 4) + 4 (l / 32) + r % 4, r = 0 .. 15.  Scores are computed with the OWNED row (a query in the forward and dQ kernels, a key in the
// dK / dV kernel) as the column: its statistics are one value of a lane, a softmax needs one exchange between the halves, and the weights
// are already the B operand of the next product -- the sum over the 16 register rows may run in any order, so the A operand is read in the
// registers' order (two transposing 8-byte LDS reads of 4 rows each in bf16; one element a register in fp32).
typedef __attribute__((ext_vector_type(8))) short bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short bf16x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;
typedef __attribute__((address_space(3))) bf16x4_t* lds_p4;

__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
__device__ __forceinline__ int reg_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }
__device__ __forceinline__ float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// The wait that the result of a product needs before plain instructions read it (11 cycles after a 32x32x16, 18 after a 32x32x2), stated here: the
// compiler counts it, but where a branch forks behind the product and joins before the read it has counted the longer way only, and the last
// register of a tile was read before it was written.  To be used behind every product whose result meets a branch.
__device__ __forceinline__ void settle(f32x16_t& a) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a)); }
__device__ __forceinline__ void settle(f32x16_t& a, f32x16_t& b) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a), "+v"(b)); }

typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
template <typename T, int DHP> struct Tile;
template <int DHP> struct Tile<bf16_t, DHP> {
  typedef bf16x8_t Frag;
  static constexpr int NS = DHP / 16;             // contraction steps of a head
  static constexpr int NDT = (DHP + 31) / 32;     // 32-dim tiles of a head
  static constexpr int CH = DHP / 8;              // 16-byte chunks of a row
  static constexpr int CHE = 8;                   // elements of a chunk
  // LDS rows: the 16-byte chunks of a row are permuted by its number, so that both ways of reading it spread over the banks: 16 bytes of 8
  // consecutive rows (natural), and 4 rows x 2 chunks (transposing; r a multiple of 4).
  static constexpr int SC = DHP == 80 ? 12 : CH;  // chunks of a row in LDS
  static constexpr int RS = SC * 8;
  static __device__ __forceinline__ int swz(int row) { return SC % 8 ? (row >> 2) & 1 : ((row & 3) << 1) | ((row >> 2) & 1); }
  static __device__ __forceinline__ int at(int row, int ch) { return row * RS + ((ch ^ swz(row)) * 8); }
  static __device__ __forceinline__ Frag natural(const bf16_t* X, int u, int l31, int s, int half) {     // row 32 u + l31
    return *reinterpret_cast<const bf16x8_t*>(X + 32 * u * RS + at(l31, 2 * s + half));
  }
  static __device__ __forceinline__ int col(int s, int half) { return 16 * s + 8 * half; }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_fmaf(bf2f((bf16_t)a[e]), bf2f((bf16_t)b[e]), c);
    return c;
  }
  static __device__ __forceinline__ f32x16_t mma(const Frag& a, const Frag& b, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // acc[dt] += X[row0 .. row0 + 31][dims dt]^T w; sum += the lane's w as they were rounded.  LO: what the rounding took away is multiplied too
  template <bool LO = false>
  static __device__ __forceinline__ void accumulate(f32x16_t* acc, const bf16_t* X, int row0, const f32x16_t& w, int lane, float* sum = nullptr) {
    const int half = lane >> 5, i16 = lane & 15, grp = (lane >> 4) & 1, r = 4 * half + (i16 >> 2);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      union { bf16x8_t v; unsigned d[4]; } b, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b.d[i] = dmt_pack_bf16(w[8 * u + 2 * i], w[8 * u + 2 * i + 1]);
        if (LO) l.d[i] = dmt_pack_bf16(w[8 * u + 2 * i] - __uint_as_float(b.d[i] << 16), w[8 * u + 2 * i + 1] - __uint_as_float(b.d[i] & 0xffff0000u));
        if (sum) *sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2_t, b.d[i]), __builtin_bit_cast(bf2_t, 0x3f803f80u), *sum, false);
      }
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const bf16_t* x = X + (row0 + 16 * u) * RS + at(r, 4 * dt + 2 * grp + ((i16 >> 1) & 1)) + 4 * (i16 & 1);
        const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p4)(x));
        const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p4)(x + 8 * RS));
        const bf16x8_t f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        acc[dt] = mma(f, b.v, acc[dt]);
        if (LO) acc[dt] = mma(f, l.v, acc[dt]);
      }
    }
  }
};
template <int DHP> struct Tile<float, DHP> {
  typedef f32x4_t Frag;
  static constexpr int NS = DHP / 8;
  static constexpr int NDT = (DHP + 31) / 32;
  static constexpr int CH = DHP / 4;
  static constexpr int CHE = 4;
  static constexpr int RS = DHP + 4;
  static __device__ __forceinline__ int at(int row, int ch) { return row * RS + ch * 4; }
  static __device__ __forceinline__ Frag natural(const float* X, int u, int l31, int s, int half) {
    return *reinterpret_cast<const f32x4_t*>(X + 32 * u * RS + at(l31, 2 * s + half));
  }
  static __device__ __forceinline__ int col(int s, int half) { return 8 * s + 4 * half; }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_fmaf(a[e], b[e], c);
    return c;
  }
  static __device__ __forceinline__ f32x16_t mma(const Frag& a, const Frag& b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  template <bool LO = false>
  static __device__ __forceinline__ void accumulate(f32x16_t* acc, const float* X, int row0, const f32x16_t& w, int lane, float* = nullptr) {
    const float* x = X + (row0 + 4 * (lane >> 5)) * RS + (lane & 31);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[(8 * (r >> 2) + (r & 3)) * RS + dt * 32], w[r], acc[dt], 0, 0, 0);
    }
  }
};

// A buffer descriptor over `rows` rows (at most 64) of one head: what lies past the last row or past dim dh reads as zero, so that neither a ragged end
// nor a padded head size needs a branch, and nothing outside the example is touched.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
template <typename T> __device__ __forceinline__ rsrc_t rows_rsrc(const T* base, long long rs, int rows, int dh) {
  const unsigned bytes = rows > 0 ? (unsigned)((rows - 1) * (int)(rs * (int)sizeof(T)) + dh * (int)sizeof(T)) : 0u;
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00027000);
}
constexpr int OUTSIDE = 0x7ffffff0;
__device__ __forceinline__ u32x4_t load16(rsrc_t r, int off) { return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); }

// One lane's fragments of its own row (the B operands that stay in registers): row row0 + l31 of the example that starts at `base`.  The descriptor
// starts at the wavefront's first row: its 32 rows of under 16 MB stay below 2^29 bytes, whatever the example's length times its stride.
template <typename T, int DHP>
__device__ __forceinline__ void own_row(typename Tile<T, DHP>::Frag* f, const T* base, long long rs, int rows, int dh, int row0, int l31, int half) {
  const rsrc_t r = rows_rsrc<T>(base + row0 * rs, rs, min(rows - row0, 32), dh);
  const int at = l31 * (int)(rs * (int)sizeof(T));
#pragma unroll
  for (int s = 0; s < Tile<T, DHP>::NS; ++s) {
    const int c = Tile<T, DHP>::col(s, half);
    f[s] = __builtin_bit_cast(typename Tile<T, DHP>::Frag, load16(r, c < dh ? at + c * (int)sizeof(T) : OUTSIDE));
  }
}

// The 64-row tiles of two operands on their way into LDS.  bf16: straight from memory (buffer_load ... lds: 64 lanes fill 1 KB of consecutive
// 16-byte chunks, each lane choosing what the row permutation wants there); issued a tile ahead, it costs no registers and no LDS-write
// instructions.  begin() and end() bracket the use of the tile before; the buffer that begin() names must be free.
template <typename T, int DHP, int NW> struct Stage;        // NW wavefronts
__device__ __forceinline__ u32x4_t rsrc_words(const void* base, unsigned bytes) {
  const unsigned long long p = (unsigned long long)(uintptr_t)base;
  u32x4_t r;
  r[0] = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)p);
  r[1] = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(p >> 32)) & 0xffffu;
  r[2] = (unsigned)__builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00027000u;
  return r;
}
// m0, the LDS address of the load, is a reserved register that an asm statement may not leave changed: it is put back behind the load, which has read
// it by then.  (No output register: nothing that a load in flight could write.)
__device__ __forceinline__ void load16_lds(const u32x4_t& rsrc, int off, unsigned lds) {
  unsigned kept;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(kept) : "s"(lds), "v"(off), "s"(rsrc) : "memory");
}
template <int DHP, int NW> struct Stage<bf16_t, DHP, NW> {
  typedef Tile<bf16_t, DHP> TL;
  static constexpr int NT = 64 * NW, IT = KT * TL::SC / NT;
  static_assert(KT * TL::SC % NT == 0, "whole 1 KB pieces");
  int off_a[IT], off_b[IT];              // byte offsets within a tile
  unsigned at;                           // LDS byte offset of the wavefront's first piece within a tile
  __device__ __forceinline__ void init(long long rs_a, long long rs_b, int dh, int tid) {
    at = (unsigned)__builtin_amdgcn_readfirstlane(tid >> 6) * 1024u;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = tid + i * NT, row = c / TL::SC, ch = (c - row * TL::SC) ^ TL::swz(row);
      const bool in = ch * 8 < dh;
      off_a[i] = in ? row * (int)(rs_a * 2) + ch * 16 : OUTSIDE;
      off_b[i] = in ? row * (int)(rs_b * 2) + ch * 16 : OUTSIDE;
    }
  }
  __device__ __forceinline__ void begin(const bf16_t* pa, long long rs_a, const bf16_t* pb, long long rs_b, int rows, int dh, bf16_t* la, bf16_t* lb) {
    const unsigned da = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)la + at;
    const unsigned db = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lb + at;
    const u32x4_t ra = rsrc_words(pa, (unsigned)((rows - 1) * (int)(rs_a * 2) + dh * 2)), rb = rsrc_words(pb, (unsigned)((rows - 1) * (int)(rs_b * 2) + dh * 2));
#pragma unroll
    for (int i = 0; i < IT; ++i) load16_lds(ra, off_a[i], (unsigned)__builtin_amdgcn_readfirstlane((int)(da + 1024u * NW * i)));
#pragma unroll
    for (int i = 0; i < IT; ++i) load16_lds(rb, off_b[i], (unsigned)__builtin_amdgcn_readfirstlane((int)(db + 1024u * NW * i)));
  }
  __device__ __forceinline__ void end(bf16_t*, bf16_t*) const { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
};
// fp32: through registers, one tile in LDS
template <int DHP, int NW> struct Stage<float, DHP, NW> {
  typedef Tile<float, DHP> TL;
  static constexpr int NT = 64 * NW, IT = (KT * TL::CH + NT - 1) / NT;
  u32x4_t a[IT], b[IT];
  int off_a[IT], off_b[IT], dst[IT];     // byte offsets within a tile; element in LDS
  __device__ __forceinline__ void init(long long rs_a, long long rs_b, int dh, int tid) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = tid + i * NT, row = c / TL::CH, ch = c - row * TL::CH;
      const bool in = row < KT && ch * 4 < dh;
      off_a[i] = in ? row * (int)(rs_a * 4) + ch * 16 : OUTSIDE;
      off_b[i] = in ? row * (int)(rs_b * 4) + ch * 16 : OUTSIDE;
      dst[i] = row < KT ? TL::at(row, ch) : -1;
    }
  }
  __device__ __forceinline__ void begin(const float* pa, long long rs_a, const float* pb, long long rs_b, int rows, int dh, float*, float*) {
    const rsrc_t ra = rows_rsrc<float>(pa, rs_a, rows, dh), rb = rows_rsrc<float>(pb, rs_b, rows, dh);
#pragma unroll
    for (int i = 0; i < IT; ++i) a[i] = load16(ra, off_a[i]);
#pragma unroll
    for (int i = 0; i < IT; ++i) b[i] = load16(rb, off_b[i]);
  }
  __device__ __forceinline__ void end(float* la, float* lb) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if ((KT * TL::CH) % NT != 0 && dst[i] < 0) continue;
      *reinterpret_cast<u32x4_t*>(la + dst[i]) = a[i];
      *reinterpret_cast<u32x4_t*>(lb + dst[i]) = b[i];
    }
  }
};

// The tiles lo .. hi - 1 that a workgroup has to visit.  With documents the ranges of 64 tiles are looked at together, a lane a tile: a walk that
// asked for one range after the other spent most of a workgroup's life waiting for them.
template <bool DOCS> struct Walk;
template <> struct Walk<false> {         // every tile, nothing masked
  int hi;
  __device__ __forceinline__ int next(int t, int& flags) {
    flags = 1;
    return t < hi ? t : hi;
  }
};
template <> struct Walk<true> {
  const int2* rng;
  int lo, hi, free_wg, free_w;           // tiles before free_wg (free_w) hold rows that no document hides from the workgroup (wavefront)
  int glo, ghi, wlo, whi;                // the ids of the workgroup's and of the wavefront's own rows
  int chunk;
  unsigned long long vis, visw, same;
  __device__ __forceinline__ void look(int c) {
    const int t = c * 64 + (threadIdx.x & 63);
    const bool in = t >= lo && t < hi;
    const int2 r = in ? rng[t] : make_int2(1, 0);
    vis = __ballot(in && (t < free_wg || (r.x <= ghi && r.y >= glo)));
    visw = __ballot(in && (t < free_w || (r.x <= whi && r.y >= wlo)));
    same = __ballot(in && r.x == r.y && wlo == whi && r.x == wlo);
    chunk = c;
  }
  // the first tile to visit from t on, or hi; flags: 1 = the wavefront has to look at it, 2 = documents may hide some of it
  __device__ __forceinline__ int next(int t, int& flags) {
    while (t < hi) {
      if ((t >> 6) != chunk) look(t >> 6);
      const unsigned long long m = vis >> (t & 63);
      if (m) {
        t += __ffsll((long long)m) - 1;
        flags = (int)((visw >> (t & 63)) & 1) | ((int)((same >> (t & 63)) & 1) ^ 1) << 1;
        return t;
      }
      t = (t | 63) + 1;
    }
    return hi;
  }
};

// one 32 x 32 result (lane = row of the matrix, registers = dims) to memory
template <typename T>
__device__ __forceinline__ void store_dims(const f32x16_t& o, float f, T* row, int dt, int half, int dh) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int j = dt * 32 + 8 * g + 4 * half;
    if (j + 4 > dh) continue;
    if (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(row + j) = make_uint2(dmt_pack_bf16(o[4 * g] * f, o[4 * g + 1] * f), dmt_pack_bf16(o[4 * g + 2] * f, o[4 * g + 3] * f));
    } else {
      *reinterpret_cast<float4*>(row + j) = make_float4(o[4 * g] * f, o[4 * g + 1] * f, o[4 * g + 2] * f, o[4 * g + 3] * f);
    }
  }
}
// 0 when every dim < dh of the lane's half row is finite, else not
__device__ __forceinline__ float not_finite(const f32x16_t& o, int dt, int half, int dh) {
  float t = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (dt * 32 + reg_row(r, half) < dh) t += o[r] * 0.f;
  return t;
}

// which dims < dh of the lane's half row are not finite (a bit for each register); then, from the two lanes that hold row r (the same for all lanes),
// whether dim lane + 64 u is one of them
template <int NDT> __device__ __forceinline__ unsigned long long not_finite_bits(const f32x16_t* o, int half, int dh) {
  unsigned long long m = 0;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (dt * 32 + reg_row(r, half) < dh && !(o[dt][r] * 0.f == 0.f)) m |= 1ull << (dt * 16 + r);
  return m;
}
__device__ __forceinline__ bool dim_of_row(unsigned long long m, int r, int u, int lane) {
  const int c = lane + 64 * u, w = c & 31, from = r + ((w >> 2) & 1) * 32, bit = (c >> 5) * 16 + (w >> 3) * 4 + (w & 3);
  const unsigned lo = __shfl((unsigned)m, from), hi = __shfl((unsigned)(m >> 32), from);
  return ((bit < 32 ? lo >> bit : hi >> (bit - 32)) & 1) != 0;
}

// which rows of which head a workgroup takes: workgroups go round the 8 dies, each with an L2 of its own, so a die gets whole heads (the
// heads that share keys side by side); the tiles with the longest rows of a causal mask start first.
__device__ __forceinline__ void place(int id, int heads, int nt, bool last_first, int& head, int& tile) {
  int t;
  if (heads % 8 == 0) {
    const int per = heads / 8, s = id >> 3;
    head = (id & 7) * per + s % per;
    t = s / per;
  } else {
    head = id % heads;
    t = id / heads;
  }
  tile = last_first ? nt - 1 - t : t;
}

}  // namespace attn_var

// Query rows of a workgroup of the forward and dQ kernels: 128 (the four wavefronts share each tile of keys), but 64 where that leaves two
// workgroups a compute unit or fewer, so that uneven rows even out (4 histories of 2048 in sessions, 8 heads of 64: forward 33 against 37 us, dQ 43
// against 48; 256 histories of up to 200, 4 heads of 80, would lose: 47 against 38 and 52 against 48).  Heads wider than 80 keep 128: their tiles
// of keys fill the LDS of half a compute unit either way.
inline int rows_of(const attn_var::Args& a, int dhp) {
  return dhp <= 80 && (long long)a.B * a.Hq * cdiv64(a.max_q, 128) <= 512 ? 64 : 128;
}

// The kernels' variants: scores as they are (0), with slopes alone (1), capped and perhaps with slopes (2; 3: near, see dmt_cap); documents or none.
// (One kernel with a branch between 2 and 3 takes the registers of both: 128 dims causal with a cap of 20 took 669 instead of 542 us.)
template <int V> struct Const { static constexpr int value = V; };
template <typename T, typename DOCS, typename F> void with_score(const attn_var::Args& a, DOCS docs, F f) {
  if (!(a.cap > 0.f)) {
    if (a.slopes) f(Const<1>(), docs);
    else f(Const<0>(), docs);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (!dmt_cap(a.scale, a.cap, true).near) return f(Const<2>(), docs);
  }
  f(Const<3>(), docs);
}
template <typename T, typename F> void with_shape(const attn_var::Args& a, F f) {
  if (a.q_doc) with_score<T>(a, Const<1>(), f);
  else with_score<T>(a, Const<0>(), f);
}

int dmt_attn_var_args(const dmt_attn_var_desc* d, attn_var::Args* a, bool backward, const char* what);
