// K / V cache in 8 bits for served histories: block tables and slots, append, read back, attention (include/dmt_hip.h: dmt_kv_*).
//
// Layout of a block (64 tokens of one request) for one key / value head:
//   K [64 tokens][dh]       the A operand of S^T = K Q^T: a lane's 8 (or 16) contraction values lie side by side;
//   V [dh][64 places]       the A operand of O^T = V^T P^T.  A 16x16 product leaves lane group b = lane / 16 with the weights of tokens
//                           16 a + 4 b + r (a = tile, r = register): place 16 b + 4 a + r puts the 16 tokens of a group side by side.
#include "dmt_common.h"

namespace {

constexpr int BS = DMT_KV_BLOCK;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int MAX_DH = 128;
constexpr float F8_MAX = 448.f;

typedef float f32x2_t __attribute__((ext_vector_type(2)));

__host__ __device__ __forceinline__ int place_of(int t) { return 16 * ((t >> 2) & 3) + 4 * (t >> 4) + (t & 3); }
__device__ __forceinline__ float f8_to_f32(unsigned byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }
// nearest e4m3, ties to even; infinities and what is past the largest value -> +-448, NaN stays
__device__ __forceinline__ float f8_clamp(float x) { return x > F8_MAX ? F8_MAX : (x < -F8_MAX ? -F8_MAX : x); }
__device__ __forceinline__ unsigned f32_to_f8x2(float a, float b) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(a), f8_clamp(b), 0, false) & 0xffffu;
}
// least power of two s >= 2^-100 with a <= 448 s  (448 = 1.75 * 2^8; a finite, >= 0)
__device__ __forceinline__ int scale_exp(float a) {
  const unsigned u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 127;
  const int s = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return s < -100 ? -100 : s;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// ================================================================================================================ plan
// The sums run over the requests in chunks of one workgroup (1024): rows, blocks wanted, runs.  What a row needs -- its request, position,
// block -- it then finds by itself (a binary search over row_off), so the second part is as wide as there are rows; with few rows and
// requests the first workgroup does it too and there is one launch.  Latency bounds it: 64 requests of one event 4.8 us; 2000 requests with 270000
// rows 5.7 + 7.1 us.
constexpr int PLAN_NT = 1024;
constexpr int PLAN_SMALL_ROWS = 4096;

struct PlanArgs {
  int n, rows, width, max_runs;
  const int* lens; const int* new_lens; int* table; const int* free_ids; const int* n_free;
  int* row_off; int* lens_out; int* slots; int* run_row; int* run_len; int* state;
  int free_cap;
  int2* req;        // [n]: (index of the request's first new block among the step's new blocks, or -1 when refused; first run)
  int* totals;      // {runs}
};
__device__ __forceinline__ int free_count(const PlanArgs& a) { return a.n_free[0] < a.free_cap ? a.n_free[0] : a.free_cap; }

// Inclusive sums of two values over the workgroup: a Kogge-Stone scan by DPP within a wavefront, the wavefronts' sums through LDS (each wavefront
// scans the 16 of them itself: one barrier).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1, 3; row_bcast:31 into rows 2, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
struct Pair { int a, b, ta, tb; };     // inclusive sums, totals
__device__ __forceinline__ Pair wg_scan(int a, int b, int (*red)[2][PLAN_NT / 64], int& turn, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  Pair p;
  p.a = wave_scan(a);
  p.b = wave_scan(b);
  int (*rd)[PLAN_NT / 64] = red[turn];
  turn ^= 1;                           // (two sets of slots: one barrier a scan)
  if (lane == 63) {
    rd[0][wave] = p.a;
    rd[1][wave] = p.b;
  }
  __syncthreads();
  const int l16 = lane & 15, sa = wave_scan(lane < 16 ? rd[0][l16] : 0), sb = wave_scan(lane < 16 ? rd[1][l16] : 0);
  p.ta = __builtin_amdgcn_readlane(sa, 15);
  p.tb = __builtin_amdgcn_readlane(sb, 15);
  if (wave > 0) {
    p.a += __builtin_amdgcn_readlane(sa, wave - 1);
    p.b += __builtin_amdgcn_readlane(sb, wave - 1);
  }
  return p;
}

__device__ void plan_rows(const PlanArgs& a, int t, int step, int total, int runs) {
  const int n_free = free_count(a);
  for (; t < a.rows; t += step) {
    int slot = -1;
    if (t < total) {
      int lo = 0, hi = a.n;                       // request r: row_off[r] <= t < row_off[r + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_off[mid] <= t) lo = mid; else hi = mid;
      }
      const int r = lo;
      const int2 rq = a.req[r];
      if (rq.x >= 0) {
        const int first = a.row_off[r], len = a.lens[r];
        const int pos = len + t - first, bi = pos / BS, have = (len + BS - 1) / BS;
        const int block = bi < have ? a.table[(long long)r * a.width + bi] : a.free_ids[n_free - 1 - (rq.x + bi - have)];
        slot = block * BS + pos % BS;
        if (t == first || pos % BS == 0) {
          const int run = rq.y + bi - len / BS;
          const int left = a.row_off[r + 1] - t, room = BS - pos % BS;
          a.run_row[run] = t;
          a.run_len[run] = left < room ? left : room;
          if (bi >= have) a.table[(long long)r * a.width + bi] = block;
        }
      }
    }
    a.slots[t] = slot;
    if (t >= runs && t < a.max_runs) {
      a.run_row[t] = -1;
      a.run_len[t] = 0;
    }
  }
}

// (The row counts are scanned in two halves of 16 bits: 1024 of them cannot pass 31 bits then.  Blocks and runs of requests that fit are bounded by
// the rows, fewer than 2^30.)
__global__ __launch_bounds__(PLAN_NT) void plan_kernel(const PlanArgs a, int small) {
  __shared__ int red[2][2][PLAN_NT / 64];
  const int tid = threadIdx.x;
  int turn = 0;
  long long row_base = 0, need_base = 0;
  int run_base = 0, taken = 0, refused = 0;
  const int n_free = free_count(a);
  for (int r0 = 0; r0 < a.n; r0 += PLAN_NT) {
    const int r = r0 + tid;
    const bool in = r < a.n;
    const int len = in ? a.lens[r] : 0, nw = in ? a.new_lens[r] : 0;
    const int rows = nw > 0 ? nw : 0;
    long long row_end;
    Pair p;
    {
      p = wg_scan(rows & 0xffff, rows >> 16, red, turn, tid);
      row_end = row_base + p.a + ((long long)p.b << 16);
      row_base += p.ta + ((long long)p.tb << 16);
    }
    const bool fits = in && nw >= 0 && len >= 0 && (long long)len + nw <= (long long)a.width * BS && row_end <= a.rows;
    // (fits: len + nw <= 64 width < 2^37, so blocks < 2^31 / 64 when it matters; rows <= a.rows < 2^30)
    const int blocks_end = fits ? (int)(((long long)len + nw + BS - 1) / BS) : 0, have = fits ? (int)(((long long)len + BS - 1) / BS) : 0;
    const int need = blocks_end - have;
    p = wg_scan(need, 0, red, turn, tid);
    const long long need_end = need_base + p.a;
    need_base += p.ta;
    const bool ok = fits && (need == 0 || need_end <= n_free);
    const int runs = ok && nw > 0 ? blocks_end - len / BS : 0;
    p = wg_scan(runs, (ok ? need : 0), red, turn, tid);
    const int run_first = run_base + p.a - runs;
    run_base += p.ta;
    taken += p.tb;
    refused += __syncthreads_count(in && !ok);
    if (in) {
      const long long row_first = row_end - rows;
      a.row_off[r] = (int)(row_first < 0x7fffffffll ? row_first : 0x7fffffffll);
      if (r == a.n - 1) a.row_off[a.n] = (int)(row_end < 0x7fffffffll ? row_end : 0x7fffffffll);
      a.lens_out[r] = ok ? len + nw : len;
      a.req[r] = make_int2(ok ? (int)(need_end - need) : -1, run_first);
    }
  }
  if (tid == 0) {
    if (a.n == 0) a.row_off[0] = 0;
    a.state[0] = n_free - taken;
    a.state[1] = refused;
    a.totals[0] = run_base;
  }
  if (small) {
    __threadfence_block();
    __syncthreads();
    plan_rows(a, tid, PLAN_NT, row_base < 0x7fffffffll ? (int)row_base : 0x7fffffff, run_base);
  }
}

__global__ __launch_bounds__(256) void plan_rows_kernel(const PlanArgs a) {
  plan_rows(a, blockIdx.x * 256 + threadIdx.x, 0x40000000, a.row_off[a.n], a.totals[0]);
}

__global__ __launch_bounds__(PLAN_NT) void release_kernel(int n, const int* done, int* lens, const int* table, int width, int* free_ids, int* n_free,
                                                          int cap) {
  __shared__ int red[2][2][PLAN_NT / 64];
  const int tid = threadIdx.x;
  int turn = 0;
  long long base = n_free[0];
  for (int r0 = 0; r0 < n; r0 += PLAN_NT) {
    const int r = r0 + tid;
    const bool in = r < n && done[r] != 0 && lens[r] > 0;
    long long held = in ? ((long long)lens[r] + BS - 1) / BS : 0;
    const int mine = (int)(held > width ? width : held);
    const Pair p = wg_scan(mine & 0xffff, mine >> 16, red, turn, tid);
    const long long end = base + p.a + ((long long)p.b << 16);
    base += p.ta + ((long long)p.tb << 16);
    if (in) {
      long long at = end - mine;
      for (int j = 0; j < mine; ++j, ++at)
        if (at >= 0 && at < cap) free_ids[at] = table[(long long)r * width + j];
      lens[r] = 0;
    }
  }
  __syncthreads();
  if (tid == 0) n_free[0] = (int)(base < cap ? base : cap);
}

// ================================================================================================================ append / read
struct Cache {
  int Hkv, dh, n_blocks;
  uint8_t* k; uint8_t* v;
  float* ks; float* vs;
};

// One workgroup owns a (run, head): its rows are held in registers between the maximum and the rounding.  What bounds it is the rows' bytes; the
// bytes of V pass through LDS because they lie across the tokens (68 bytes a dim there: the 16 chunks of a row would meet in one bank at 64).
// 256 requests of one event, 8 heads of 128: 11 us; 16 fills of up to 2500 rows: 36 us.  (A thread with 4 side-by-side tokens, whole words of V instead of
// bytes: 33 us for the rows, but 12 to 15 for the events; bytes of V straight to memory for short runs did not help.)
constexpr int VLD = BS + 4;
__global__ __launch_bounds__(256) void append_kernel(const Cache c, int rows, const bf16_t* kr, long long k_rs, const bf16_t* vr, long long v_rs,
                                                     const int* slots, const int* run_row, const int* run_len) {
  __shared__ float red[2][4];
  __shared__ __attribute__((aligned(16))) unsigned char vt[MAX_DH * VLD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hk = blockIdx.y, dh = c.dh, ch = dh / 8;
  const int row0 = run_row[blockIdx.x];
  int len = run_len[blockIdx.x];
  if (row0 < 0 || row0 >= rows || len <= 0) return;
  const int slot = slots[row0], block = slot / BS, first = slot % BS;
  if (slot < 0 || block >= c.n_blocks) return;
  if (len > BS - first) len = BS - first;
  if (len > rows - row0) len = rows - row0;
  const long long bh = (long long)block * c.Hkv + hk;
  uint8_t* kb = c.k + bh * BS * dh;
  uint8_t* vb = c.v + bh * BS * dh;
  uint4 kx[4], vx[4];
  float ka = 0.f, va = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int cc = tid + i * 256, t = cc / ch, q = cc - t * ch;
    if (t < len) {
      kx[i] = *reinterpret_cast<const uint4*>(kr + (row0 + t) * k_rs + (long long)hk * dh + q * 8);
      vx[i] = *reinterpret_cast<const uint4*>(vr + (row0 + t) * v_rs + (long long)hk * dh + q * 8);
      const unsigned* kw = reinterpret_cast<const unsigned*>(&kx[i]);
      const unsigned* vw = reinterpret_cast<const unsigned*>(&vx[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float x = fabsf(__uint_as_float(s ? (kw[e] & 0xffff0000u) : (kw[e] << 16)));
          const float y = fabsf(__uint_as_float(s ? (vw[e] & 0xffff0000u) : (vw[e] << 16)));
          if (x < INFINITY) ka = fmaxf(ka, x);
          if (y < INFINITY) va = fmaxf(va, y);
        }
      }
    }
  }
  ka = wave_max(ka);
  va = wave_max(va);
  if (lane == 0) { red[0][wave] = ka; red[1][wave] = va; }
  __syncthreads();
  ka = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  va = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  float ks = pow2(scale_exp(ka)), vs = pow2(scale_exp(va));
  const float ks0 = c.ks[bh], vs0 = c.vs[bh];
  const bool older = first > 0;
  const bool k_grow = older && ks > ks0, v_grow = older && vs > vs0;
  if (older) {
    ks = fmaxf(ks, ks0);
    vs = fmaxf(vs, vs0);
  }
  const float ki = 1.f / ks, vi = 1.f / vs;       // (powers of two: exact)
  __syncthreads();                                // (every thread has read the old scales)
  if (tid == 0) { c.ks[bh] = ks; c.vs[bh] = vs; }
  if (k_grow) {
    const float f = ks0 * ki;
    for (int x = tid * 4; x < first * dh; x += 1024) {
      const unsigned w = *reinterpret_cast<unsigned*>(kb + x);
      const unsigned lo = f32_to_f8x2(f8_to_f32(w & 255) * f, f8_to_f32((w >> 8) & 255) * f);
      const unsigned hi = f32_to_f8x2(f8_to_f32((w >> 16) & 255) * f, f8_to_f32(w >> 24) * f);
      *reinterpret_cast<unsigned*>(kb + x) = lo | (hi << 16);
    }
  }
  // V: the block passes through LDS (its bytes lie across the tokens)
  if (len < BS) {
    for (int x = tid * 16; x < dh * BS; x += 4096) {
      const uint4 w = *reinterpret_cast<const uint4*>(vb + x);
      unsigned* d = reinterpret_cast<unsigned*>(vt + (x / BS) * VLD + x % BS);
      d[0] = w.x;
      d[1] = w.y;
      d[2] = w.z;
      d[3] = w.w;
    }
    __syncthreads();
  }
  if (v_grow) {
    const float f = vs0 * vi;
    for (int x = tid; x < dh * first; x += 256) {
      const int dd = x / first, at = dd * VLD + place_of(x - dd * first);
      vt[at] = (unsigned char)f32_to_f8x2(f8_to_f32(vt[at]) * f, 0.f);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int cc = tid + i * 256, t = cc / ch, q = cc - t * ch;
    if (t < len) {
      const unsigned* kw = reinterpret_cast<const unsigned*>(&kx[i]);
      const unsigned* vw = reinterpret_cast<const unsigned*>(&vx[i]);
      unsigned o[2] = {0u, 0u};
      const int pl = place_of(first + t);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e >> 1] |= f32_to_f8x2(__uint_as_float(kw[e] << 16) * ki, __uint_as_float(kw[e] & 0xffff0000u) * ki) << (16 * (e & 1));
        const unsigned y = f32_to_f8x2(__uint_as_float(vw[e] << 16) * vi, __uint_as_float(vw[e] & 0xffff0000u) * vi);
        vt[(q * 8 + 2 * e) * VLD + pl] = (unsigned char)y;
        vt[(q * 8 + 2 * e + 1) * VLD + pl] = (unsigned char)(y >> 8);
      }
      *reinterpret_cast<uint2*>(kb + (long long)(first + t) * dh + q * 8) = make_uint2(o[0], o[1]);
    }
  }
  __syncthreads();
  for (int x = tid * 16; x < dh * BS; x += 4096) {
    const unsigned* d = reinterpret_cast<const unsigned*>(vt + (x / BS) * VLD + x % BS);
    *reinterpret_cast<uint4*>(vb + x) = make_uint4(d[0], d[1], d[2], d[3]);
  }
}

// A workgroup reads 64 listed slots of one head.  V lies across the tokens: when the slots are a whole block in order (how a caller looks at a
// block) its bytes come in 16-byte loads, 4 x 4 tokens of one dim each, and are turned around in LDS; else a lane per slot gathers bytes.
// Bound by the bytes, two thirds of them the bf16 rows: 256 blocks, 8 heads of 128: 24 us.
__global__ __launch_bounds__(256) void read_kernel(const Cache c, int n, const int* slots, bf16_t* kr, long long k_rs, bf16_t* vr, long long v_rs) {
  __shared__ __attribute__((aligned(16))) bf16_t tile[64 * (MAX_DH + 8)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hk = blockIdx.y, dh = c.dh, ch = dh / 8, ld = dh + 8;
  const int i0 = blockIdx.x * 64;
  const int cnt = n - i0 < 64 ? n - i0 : 64;
  const int slot = lane < cnt ? slots[i0 + lane] : -1, block = slot >= 0 ? slot / BS : -1;
  const bool ok = slot >= 0 && block < c.n_blocks;
  const long long bh = ok ? (long long)block * c.Hkv + hk : 0;
  const int slot0 = __builtin_amdgcn_readfirstlane(slot);
  const bool whole = slot0 % BS == 0 && __all(ok && slot == slot0 + lane);
  const float vs = ok ? c.vs[bh] : 0.f;
  if (whole) {
    const uint8_t* src = c.v + bh * BS * dh;
    for (int x = tid; x < dh * 4; x += 256) {
      const int j = x >> 2, b = x & 3;
      const uint4 w = *reinterpret_cast<const uint4*>(src + j * BS + 16 * b);
      const unsigned d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[(16 * q + 4 * b + e) * ld + j] = f2bf(f8_to_f32((d[q] >> (8 * e)) & 255) * vs);
    }
  } else {
    const uint8_t* src = c.v + bh * BS * dh + (ok ? place_of(slot % BS) : 0);
    for (int j = wave; j < dh; j += 4) tile[lane * ld + j] = ok ? f2bf(f8_to_f32(src[(long long)j * BS]) * vs) : (bf16_t)0;
  }
  for (int x = tid; x < cnt * ch; x += 256) {
    const int i = x / ch, q = x - i * ch, sl = slots[i0 + i], bl = sl >= 0 ? sl / BS : -1;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (sl >= 0 && bl < c.n_blocks) {
      const long long b2 = (long long)bl * c.Hkv + hk;
      const uint2 w = *reinterpret_cast<const uint2*>(c.k + (b2 * BS + sl % BS) * dh + q * 8);
      const float s = c.ks[b2];
      const unsigned lo = w.x, hi = w.y;
      o.x = dmt_pack_bf16(f8_to_f32(lo & 255) * s, f8_to_f32((lo >> 8) & 255) * s);
      o.y = dmt_pack_bf16(f8_to_f32((lo >> 16) & 255) * s, f8_to_f32(lo >> 24) * s);
      o.z = dmt_pack_bf16(f8_to_f32(hi & 255) * s, f8_to_f32((hi >> 8) & 255) * s);
      o.w = dmt_pack_bf16(f8_to_f32((hi >> 16) & 255) * s, f8_to_f32(hi >> 24) * s);
    }
    *reinterpret_cast<uint4*>(kr + (long long)(i0 + i) * k_rs + (long long)hk * dh + q * 8) = o;
  }
  __syncthreads();
  for (int x = tid; x < cnt * ch; x += 256) {
    const int i = x / ch, q = x - i * ch;
    *reinterpret_cast<uint4*>(vr + (long long)(i0 + i) * v_rs + (long long)hk * dh + q * 8) = *reinterpret_cast<const uint4*>(tile + i * ld + q * 8);
  }
}

// ================================================================================================================ attention
struct KvArgs {
  Cache c;
  int n, Hq, G, max_q, max_len, width, causal, rest;
  long long rows;
  const bf16_t* Q; long long q_rs;
  const int* table; const int* lens; const int* row_off;
  float scale, cap;
  const float* slopes;
  bf16_t* out; long long o_rs;
  float* lse;
};

// A request's rows and tokens as far as they are computed (m, L: cut at max_q, max_len, the table's width and the matrix), and `at`, the position
// of its first row (causal) or of all of them, from the lengths as they stand: what is cut off moves nothing that stays.
struct Req { int m, L, at; long long row0; };
__device__ __forceinline__ Req request(const KvArgs& a, int r) {
  Req q;
  const long long lo = a.row_off[r], hi = a.row_off[r + 1], held = a.lens[r];
  q.row0 = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
  long long m = (hi > a.rows ? a.rows : hi) - q.row0;
  q.m = m < 0 ? 0 : (int)(m > a.max_q ? a.max_q : m);
  const long long most = (long long)a.width * BS;
  long long L = held;
  if (L > a.max_len) L = a.max_len;
  if (L > most) L = most;
  q.L = L < 0 ? 0 : (int)L;
  const long long at = a.causal ? held - (hi - q.row0) : held;
  q.at = (int)(at < -0x7fffffffll ? -0x7fffffffll : at);       // (held < 2^31 and hi >= row0 where there is a row)
  return q;
}
// position of row i, and the number of tokens that it sees
__device__ __forceinline__ int position(const KvArgs& a, const Req& q, int i) { return a.causal ? q.at + i : q.at; }
__device__ __forceinline__ int sees(const KvArgs& a, const Req& q, int i) {
  const int s = a.causal ? q.at + i + 1 : q.L;
  return s < 0 ? 0 : (s < q.L ? s : q.L);
}

__device__ __forceinline__ float kv_z2(const KvArgs& a, float x, float slope2, float dist) {
  const float y = a.cap > 0.f ? dmt_cap(a.scale, a.cap, true)(x) : a.scale * LOG2E * x;
  return a.slopes ? __builtin_fmaf(-slope2, fabsf(dist), y) : y;
}
__device__ __forceinline__ void lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// rows r0 .. r1 - 1 of the heads h0 .. h0 + heads - 1 that no request's row is: zeros in out, -inf in lse, as a.rest asks
__device__ __forceinline__ void rest_rows(const KvArgs& a, long long r0, long long r1, int h0, int heads) {
  const int c8 = heads * a.c.dh / 8;
  if (a.rest & 1)
    for (long long x = threadIdx.x; x < (r1 - r0) * c8; x += blockDim.x)
      *reinterpret_cast<uint4*>(a.out + (r0 + x / c8) * a.o_rs + (long long)h0 * a.c.dh + x % c8 * 8) = make_uint4(0u, 0u, 0u, 0u);
  if ((a.rest & 2) && a.lse)
    for (long long x = threadIdx.x; x < (r1 - r0) * heads; x += blockDim.x) a.lse[(r0 + x / heads) * a.Hq + h0 + x % heads] = -INFINITY;
}
// ... as workgroup `part` of `parts` of key head hk finds them: what of request r (part `first` of its own) lies past max_q, the rows before the first
// request's, and its share of those behind the last one's
__device__ __forceinline__ void rest_of(const KvArgs& a, const Req& rq, int r, int hk, bool first, long long part, long long parts) {
  const long long hi = a.row_off[r + 1], end = hi < a.rows ? hi : a.rows, last = a.row_off[a.n], tail = last < 0 ? 0 : (last < a.rows ? last : a.rows);
  if (first && r == 0 && rq.row0 > 0) rest_rows(a, 0, rq.row0, hk * a.G, a.G);
  if (first && rq.row0 + rq.m < end) rest_rows(a, rq.row0 + rq.m, end, hk * a.G, a.G);
  if (tail < a.rows) {
    const long long each = (a.rows - tail + parts - 1) / parts, r0 = tail + part * each;
    if (r0 < a.rows) rest_rows(a, r0, r0 + each < a.rows ? r0 + each : a.rows, hk * a.G, a.G);
  }
}
// ... of a call without requests
__global__ __launch_bounds__(256) void kv_rest_kernel(const KvArgs a) {
  rest_rows(a, a.rows * blockIdx.x / gridDim.x, a.rows * (blockIdx.x + 1ll) / gridDim.x, 0, a.Hq);
}

// One wavefront, one (row, head), plain arithmetic: a lane per token for the scores, a lane per dim for the sums -- of the dims that the tiles left
// not finite (s0, s1: of the lane's two), until all of them are NaN, which nothing after them changes.
__device__ void kv_row(const KvArgs& a, const Req& rq, int r, int h, int i, bool s0, bool s1, float* lds, int lane) {
  float* q = lds;
  float* pl = lds + MAX_DH;
  const int dh = a.c.dh, hk = h / a.G;
  const long long row = rq.row0 + i;
  for (int x = lane; x < dh; x += 64) q[x] = bf2f(a.Q[row * a.q_rs + (long long)h * dh + x]);
  lds_fence();
  const float slope2 = a.slopes ? a.slopes[h] * LOG2E : 0.f;
  const int lim = sees(a, rq, i), pos = position(a, rq, i);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < lim; j0 += BS) {
    const int block = a.table[(long long)r * a.width + j0 / BS];
    if (block < 0 || block >= a.c.n_blocks) continue;
    const long long bh = (long long)block * a.c.Hkv + hk;
    const uint8_t* kb = a.c.k + (bh * BS + lane) * dh;
    const uint8_t* vb = a.c.v + bh * BS * dh;
    const float ks = a.c.ks[bh], vs = a.c.vs[bh];
    const int j = j0 + lane;
    const bool ok = j < lim;
    float z = -INFINITY;
    if (ok) {
      float s = 0.f;
      for (int x = 0; x < dh; ++x) s = __builtin_fmaf(q[x], f8_to_f32(kb[x]) * ks, s);
      z = kv_z2(a, s, slope2, (float)(pos - j));
    }
    const float mn = fmaxf(m, wave_max(z));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float p = ok ? __builtin_amdgcn_exp2f(z - mu) : 0.f;
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    l = l * f + wave_sum(p);
    o0 *= f;
    o1 *= f;
    pl[lane] = p;
    lds_fence();
    const int last = lim - j0 < BS ? lim - j0 : BS;
    for (int t = 0; t < last; ++t) {
      const float pt = pl[t] * vs;
      const int pc = place_of(t);
      if (lane < dh) o0 = __builtin_fmaf(pt, f8_to_f32(vb[(long long)lane * BS + pc]), o0);
      if (lane + 64 < dh) o1 = __builtin_fmaf(pt, f8_to_f32(vb[(long long)(lane + 64) * BS + pc]), o1);
    }
    lds_fence();
    if (!__any((s0 && o0 == o0) || (s1 && o1 == o1))) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf16_t* O = a.out + row * a.o_rs + (long long)h * dh;
  if (s0) O[lane] = f2bf(o0 * inv);
  if (s1) O[lane + 64] = f2bf(o1 * inv);
}
// which of 8 values are not finite
__device__ __forceinline__ unsigned not_finite8(const float* x) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m |= x[e] * 0.f == 0.f ? 0u : 1u << e;
  return m;
}

// Tiles.  A wavefront takes a block of 64 tokens at a time and the columns of a tile -- 16 NQ (row, head of the group) pairs: heads that share a
// key head read its bytes together -- and keeps its own running maximum, sum and output; the four wavefronts of a workgroup walk over every
// fourth block of the workgroup's piece of the length.  K and V go from memory to registers in 16-byte loads (each byte once a tile of columns)
// and become bf16 by v_cvt_scalef32_pk_bf16_fp8, which takes the block's scale along: the products see the stored values exactly.
//   S^T = K Q^T   (16x16x32, tokens x columns): the contraction runs over the dims in the order in which a lane loads them -- 16 bytes of a
//                 row are two steps of 8 -- and Q is laid out the same way; a remainder of 16 dims is a step whose upper half is zero
//                 (a 16x16x16 product that adds to the result of a 16x16x32 one just before it came out wrong here).
//   O^T = V^T P^T (dims x columns): the weights of S^T, packed, are the B operand; the places of V are in that order.
// What bounds it: the cache's bytes for few columns (64 ragged requests of up to 8192 tokens, 32 heads on 8 of 128, one row each: 117 to 121 us, 4.6 TB/s);
// with many columns the walk of a wavefront over its blocks, load after load (16 requests of up to 1000 tokens, 300 rows, 4 heads of 80: 24 us;
// requesting the next block ahead takes the registers of a third workgroup: 30; 48 columns a tile: 34); for a single short request the launch (4.8 us).
typedef __attribute__((ext_vector_type(8))) short bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short bf16x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));

// 4 bytes -> 4 bf16 (two registers)
__device__ __forceinline__ uint2 f8x4_bf16(unsigned w, float scale) {
  return make_uint2(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)));
}
__device__ __forceinline__ bf16x8_t f8x8_bf16(unsigned lo, unsigned hi, float scale) {
  union { bf16x8_t v; uint2 d[2]; } u;
  u.d[0] = f8x4_bf16(lo, scale);
  u.d[1] = f8x4_bf16(hi, scale);
  return u.v;
}
__device__ __forceinline__ bf16x8_t f8x4_frag(unsigned w, float scale) {
  union { bf16x8_t v; uint2 d[2]; } u;
  u.d[0] = f8x4_bf16(w, scale);
  u.d[1] = make_uint2(0u, 0u);
  return u.v;
}

// max / sum over the four 16-lane groups (the tokens of one column)
__device__ __forceinline__ float xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float col_max(float x) {
  x = fmaxf(x, xor16(x));
  return fmaxf(x, xor32(x));
}
__device__ __forceinline__ float col_sum(float x) {
  x += xor16(x);
  return x + xor32(x);
}

struct Split { int pieces, chunk, nqt; };          // pieces of the length, blocks of a piece, tiles of columns

template <int DH> struct Dims {
  static constexpr int N64 = DH / 64, R = DH % 64, N32 = R / 32, N16 = (R % 32) / 16;    // 16-byte, 8-byte and 4-byte loads of a row
  static constexpr int KW = 4 * N64 + 2 * N32 + N16;                                       // dwords of a lane
};

// SHAPE: 0 the scores as they are, 1 with a cap and / or slopes, 2 with a cap that takes the longer form (dmt_cap: near)
template <int DH, int NQ, int SHAPE>
__global__ __launch_bounds__(256, 2) void kv_tile_kernel(const KvArgs a, const Split sp, float* __restrict__ part_o, float2* __restrict__ part_ml) {
  typedef Dims<DH> DM;
  constexpr int NC = 16 * NQ, NDT = DH / 16, LO = DH + 4;
  __shared__ __attribute__((aligned(16))) float lo[4][NC * LO];
  __shared__ float lm[4][NC], ll[4][NC];
  __shared__ unsigned char dims[NC][16];       // a bit for each dim of a column that came out not finite
  static_assert(sizeof(lo[0]) >= (MAX_DH + 64) * sizeof(float), "the row form works in a wavefront's part");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = lane >> 4, l15 = lane & 15;
  const int pairs = a.n * a.c.Hkv, items = pairs * sp.pieces, id = blockIdx.x;
  // the column tiles of one piece read the same bytes: side by side on one die (workgroups go round the 8 dies)
  int item, qt;
  if (items % 8 == 0) {
    item = (id & 7) * (items / 8) + (id >> 3) / sp.nqt;
    qt = (id >> 3) % sp.nqt;
  } else {
    item = id / sp.nqt;
    qt = id % sp.nqt;
  }
  const int piece = item % sp.pieces, pair = item / sp.pieces, hk = pair % a.c.Hkv, r = pair / a.c.Hkv;
  const Req rq = request(a, r);
  const int cols = rq.m * a.G, nb = (rq.L + BS - 1) / BS;
  if (a.rest) rest_of(a, rq, r, hk, qt == 0 && piece == 0, ((long long)r * sp.pieces + piece) * sp.nqt + qt, (long long)a.n * sp.pieces * sp.nqt);
  if (qt * NC >= cols || (piece > 0 && piece * sp.chunk >= nb)) return;
  int lim[NQ], pos[NQ], lim_wg = 0;
  float sl2[NQ];
  constexpr int NF = 2 * DM::N64 + DM::N32;
  bf16x8_t q[NQ][NF ? NF : 1];
  bf16x8_t q16[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int c = qt * NC + 16 * x + l15;
    const bool in = c < cols;
    const int i = in ? c / a.G : 0, g = in ? c - i * a.G : 0, h = hk * a.G + g;
    lim[x] = in ? sees(a, rq, i) : 0;
    pos[x] = position(a, rq, i);
    sl2[x] = SHAPE && a.slopes ? a.slopes[h] * LOG2E : 0.f;
    const bf16_t* Q = a.Q + (rq.row0 + i) * a.q_rs + (long long)h * DH;
    const bf16x8_t z8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < DM::N64; ++s) {
      q[x][2 * s] = in ? *reinterpret_cast<const bf16x8_t*>(Q + 64 * s + 16 * grp) : z8;
      q[x][2 * s + 1] = in ? *reinterpret_cast<const bf16x8_t*>(Q + 64 * s + 16 * grp + 8) : z8;
    }
    if (DM::N32) q[x][2 * DM::N64] = in ? *reinterpret_cast<const bf16x8_t*>(Q + 64 * DM::N64 + 8 * grp) : z8;
    q16[x] = z8;
    if (DM::N16 && in) {
      const bf16x4_t w = *reinterpret_cast<const bf16x4_t*>(Q + DH - 16 + 4 * grp);
      q16[x] = bf16x8_t{w[0], w[1], w[2], w[3], 0, 0, 0, 0};
    }
  }
  {
    const int last = min(qt * NC + NC, cols) - 1;
    lim_wg = sees(a, rq, last / a.G);
  }
  const int b0 = piece * sp.chunk, b1 = min(min(b0 + sp.chunk, nb), (lim_wg + BS - 1) / BS);
  f32x4_t o[NQ][NDT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[x][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const dmt_cap cap(a.scale, a.cap, true);
  const float c1 = cap.c1;
  const int* tb = a.table + (long long)r * a.width;
  int block = b0 + wave < b1 ? tb[b0 + wave] : 0;
  for (int t = b0 + wave; t < b1; t += 4) {
    const int cur = __builtin_amdgcn_readfirstlane(block), j0 = t * BS;
    if (t + 4 < b1) block = tb[t + 4];
    if (cur < 0 || cur >= a.c.n_blocks) continue;
    const long long bh = (long long)cur * a.c.Hkv + hk;
    const uint8_t* kb = a.c.k + bh * BS * DH;
    const uint8_t* vb = a.c.v + bh * BS * DH;
    const float ks = a.c.ks[bh], vs = a.c.vs[bh];
    unsigned kw[4][DM::KW];
    unsigned vw[NDT][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint8_t* row = kb + (16 * u + l15) * DH;
#pragma unroll
      for (int s = 0; s < DM::N64; ++s) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + 64 * s + 16 * grp);
        kw[u][4 * s] = w.x;
        kw[u][4 * s + 1] = w.y;
        kw[u][4 * s + 2] = w.z;
        kw[u][4 * s + 3] = w.w;
      }
      if (DM::N32) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 64 * DM::N64 + 8 * grp);
        kw[u][4 * DM::N64] = w.x;
        kw[u][4 * DM::N64 + 1] = w.y;
      }
      if (DM::N16) kw[u][DM::KW - 1] = *reinterpret_cast<const unsigned*>(row + DH - 16 + 4 * grp);
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const uint4 w = *reinterpret_cast<const uint4*>(vb + (16 * dt + l15) * BS + 16 * grp);
      vw[dt][0] = w.x;
      vw[dt][1] = w.y;
      vw[dt][2] = w.z;
      vw[dt][3] = w.w;
    }
    f32x4_t s[NQ][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) s[x][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const bf16x8_t k = f8x8_bf16(kw[u][2 * f], kw[u][2 * f + 1], ks);
#pragma unroll
        for (int x = 0; x < NQ; ++x) s[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[x][f], s[x][u], 0, 0, 0);
      }
      if (DM::N16) {
        const bf16x8_t k = f8x4_frag(kw[u][DM::KW - 1], ks);
#pragma unroll
        for (int x = 0; x < NQ; ++x) s[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q16[x], s[x][u], 0, 0, 0);
      }
    }
    if (j0 + BS > rq.L) {       // the last block: what stands behind the last token may be anything, and its weight 0 does not silence NaN
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int n = rq.L - j0 - 16 * u - 4 * grp;
        const unsigned keep = n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) vw[dt][u] &= keep;
      }
    }
    bf16x8_t p[NQ][2];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int lx = lim[x] - j0 - 4 * grp;
      const float d0 = (float)(pos[x] - j0 - 4 * grp);
      float mx = -INFINITY;
      if (SHAPE) {
        const auto each = [&](auto score) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][u][e] = score(s[x][u][e]);
        };
        if (SHAPE == 1 && !(a.cap > 0.f)) each([&](float z) { return c1 * z; });
        else each([&](float z) { return cap.less<SHAPE == 2>(z, cap.r(z), 0.f); });
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float z = s[x][u][e];
          if (SHAPE) z = __builtin_fmaf(-sl2[x], fabsf(d0 - (float)(16 * u + e)), z);
          z = 16 * u + e < lx ? z : -INFINITY;
          s[x][u][e] = z;
          mx = fmaxf(mx, z);
        }
      mx = col_max(mx) * (SHAPE ? 1.f : c1);
      if (__any(mx > m[x] + 8.f)) {               // (as in the tile kernels of attn_var: weights up to 2^8 before the output is rescaled)
        const float mn = fmaxf(m[x], mx), f = m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[x] - mn);
        m[x] = mn;
        l[x] *= f;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x][dt][e] *= f;
      }
      const float mu = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[x][u][e] = __builtin_amdgcn_exp2f(SHAPE ? s[x][u][e] - mu : __builtin_fmaf(s[x][u][e], c1, -mu));
          l[x] += s[x][u][e];
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        union { bf16x8_t v; unsigned d[4]; } w;
        w.d[0] = dmt_pack_bf16(s[x][2 * u][0], s[x][2 * u][1]);
        w.d[1] = dmt_pack_bf16(s[x][2 * u][2], s[x][2 * u][3]);
        w.d[2] = dmt_pack_bf16(s[x][2 * u + 1][0], s[x][2 * u + 1][1]);
        w.d[3] = dmt_pack_bf16(s[x][2 * u + 1][2], s[x][2 * u + 1][3]);
        p[x][u] = w.v;
      }
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const bf16x8_t v0 = f8x8_bf16(vw[dt][0], vw[dt][1], vs), v1 = f8x8_bf16(vw[dt][2], vw[dt][3], vs);
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        o[x][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, p[x][0], o[x][dt], 0, 0, 0);
        o[x][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, p[x][1], o[x][dt], 0, 0, 0);
      }
    }
  }
  // the four wavefronts' parts, joined in their order
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    l[x] = col_sum(l[x]);
    if (grp == 0) {
      lm[wave][16 * x + l15] = m[x];
      ll[wave][16 * x + l15] = l[x];
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4_t*>(&lo[wave][(16 * x + l15) * LO + 16 * dt + 4 * grp]) = o[x][dt];
  }
  __syncthreads();
  const long long part = ((long long)item * sp.nqt + qt) * NC;
  unsigned long long again = 0;
  for (int y = tid; y < NC * (DH / 8); y += 256) {
    const int cl = y / (DH / 8), d8 = (y - cl * (DH / 8)) * 8, c = qt * NC + cl;
    if (c >= cols) continue;
    float M = fmaxf(fmaxf(lm[0][cl], lm[1][cl]), fmaxf(lm[2][cl], lm[3][cl])), Ls = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(lm[w][cl] - mu);
      Ls = __builtin_fmaf(ll[w][cl], f, Ls);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(lo[w][cl * LO + d8 + e], f, acc[e]);
    }
    if (sp.pieces > 1) {
      float* po = part_o + (part + cl) * DH + d8;
      *reinterpret_cast<float4*>(po) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(po + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (d8 == 0) part_ml[part + cl] = make_float2(M, Ls);
      continue;
    }
    const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
    const int i = c / a.G, h = hk * a.G + c - i * a.G;
    const long long row = rq.row0 + i;
    *reinterpret_cast<uint4*>(a.out + row * a.o_rs + (long long)h * DH + d8) =
        make_uint4(dmt_pack_bf16(acc[0] * inv, acc[1] * inv), dmt_pack_bf16(acc[2] * inv, acc[3] * inv), dmt_pack_bf16(acc[4] * inv, acc[5] * inv),
                   dmt_pack_bf16(acc[6] * inv, acc[7] * inv));
    if (a.lse && d8 == 0) a.lse[row * a.Hq + h] = Ls == 0.f ? -INFINITY : (M + __log2f(Ls)) * LN2;
    // (a sum that is NaN: so is a score that the row sees, and the whole row)
    const unsigned bad = Ls == Ls ? not_finite8(acc) : 0u;
    dims[cl][d8 / 8] = (unsigned char)bad;
    if (bad) again |= 1ull << cl;
  }
  if (sp.pieces > 1) return;
  // columns that came out not finite once more, by what they may see alone
  __shared__ unsigned long long redo;
  if (tid == 0) redo = 0;
  __syncthreads();
  if (again) atomicOr(&redo, again);
  __syncthreads();
  if (redo)
    for (int cl = wave; cl < NC; cl += 4)
      if ((redo >> cl) & 1) {
        const int c = qt * NC + cl, i = c / a.G;
        kv_row(a, rq, r, hk * a.G + c - i * a.G, i, lane < DH && ((dims[cl][lane / 8] >> (lane % 8)) & 1),
               lane + 64 < DH && ((dims[cl][8 + lane / 8] >> (lane % 8)) & 1), lo[wave], lane);
      }
}

// Joins the pieces of a (row, head), in their order: 16 lanes a column and 8 dims a lane; with many pieces `gpc` such groups take every
// gpc-th piece of one column and meet in LDS (one group alone would wait for one piece after the other: 400 of them took 230 us; now 7).
template <int NQ>
__global__ __launch_bounds__(256) void kv_join_kernel(const KvArgs a, const Split sp, int gpc, const float* __restrict__ part_o,
                                                      const float2* __restrict__ part_ml) {
  __shared__ __attribute__((aligned(16))) float lo[16][MAX_DH];
  __shared__ float lm[16], ll[16];
  constexpr int NC = 16 * NQ;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, grp = threadIdx.x >> 4, r = blockIdx.z, hk = blockIdx.y, dh = a.c.dh;
  const Req rq = request(a, r);
  const int per = 16 / gpc, c = blockIdx.x * per + grp / gpc, g0 = grp % gpc, nb = (rq.L + BS - 1) / BS;
  if ((int)blockIdx.x * per >= rq.m * a.G) return;
  const bool in = c < rq.m * a.G;
  const int i = in ? c / a.G : 0, h = hk * a.G + (in ? c - i * a.G : 0);
  const int np = in ? max(1, (nb + sp.chunk - 1) / sp.chunk) : 0;
  const long long item0 = ((long long)r * a.c.Hkv + hk) * sp.pieces;
  float M = -INFINITY, Ls = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = g0; p < np; p += gpc) {
    const long long at = ((item0 + p) * sp.nqt + c / NC) * NC + c % NC;
    const float2 ml = part_ml[at];
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (l15 * 8 < dh) {
      const float* po = part_o + at * dh + l15 * 8;
      const float4 x = *reinterpret_cast<const float4*>(po), y = *reinterpret_cast<const float4*>(po + 4);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    }
    const float mn = fmaxf(M, ml.x), mu = mn == -INFINITY ? 0.f : mn;
    const float f0 = __builtin_amdgcn_exp2f(M - mu), f1 = __builtin_amdgcn_exp2f(ml.x - mu);
    M = mn;
    Ls = __builtin_fmaf(Ls, f0, ml.y * f1);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(acc[e], f0, v[e] * f1);
  }
  if (gpc > 1) {
    if (l15 == 0) { lm[grp] = M; ll[grp] = Ls; }
    *reinterpret_cast<float4*>(&lo[grp][l15 * 8]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    *reinterpret_cast<float4*>(&lo[grp][l15 * 8 + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    __syncthreads();
    if (g0 == 0) {
      M = -INFINITY;
      for (int g = 0; g < gpc; ++g) M = fmaxf(M, lm[grp + g]);
      const float mu = M == -INFINITY ? 0.f : M;
      Ls = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      for (int g = 0; g < gpc; ++g) {
        const float f = __builtin_amdgcn_exp2f(lm[grp + g] - mu);
        Ls = __builtin_fmaf(ll[grp + g], f, Ls);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(lo[grp + g][l15 * 8 + e], f, acc[e]);
      }
    }
    __syncthreads();
  }
  const bool mine = in && g0 == 0;
  const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
  const long long row = rq.row0 + i;
  const unsigned bad = mine && Ls == Ls && l15 * 8 < dh ? not_finite8(acc) : 0u;       // (as above)
  if (mine && l15 * 8 < dh)
    *reinterpret_cast<uint4*>(a.out + row * a.o_rs + (long long)h * dh + l15 * 8) =
        make_uint4(dmt_pack_bf16(acc[0] * inv, acc[1] * inv), dmt_pack_bf16(acc[2] * inv, acc[3] * inv), dmt_pack_bf16(acc[4] * inv, acc[5] * inv),
                   dmt_pack_bf16(acc[6] * inv, acc[7] * inv));
  if (mine && a.lse && l15 == 0) a.lse[row * a.Hq + h] = Ls == 0.f ? -INFINITY : (M + __log2f(Ls)) * LN2;
  const unsigned long long again = __ballot(bad != 0u);
  for (int g = 0; g < 4; ++g)
    if ((again >> (16 * g)) & 0xffff) {
      const int cc = blockIdx.x * per + (wave * 4 + g) / gpc, ii = cc / a.G;
      const unsigned b0 = __shfl(bad, 16 * g + lane / 8), b1 = __shfl(bad, 16 * g + 8 + lane / 8);
      kv_row(a, rq, r, hk * a.G + cc - ii * a.G, ii, (b0 >> (lane % 8)) & 1, (b1 >> (lane % 8)) & 1, lo[wave * 4], lane);
    }
}

// How a call is cut up.  Columns: 16 a tile up to 32 of them, else 32 (each conversion of a block then serves twice the columns): 4 rows x 8 heads of
// 64 requests of 1000 tokens 17.5 us in tiles of 16, 21.6 in tiles of 32; 64 rows x 8 heads over 16000 tokens 93 against 60 us.
// Length: 512 workgroups -- two for each compute unit -- but at least 4 blocks, one for each wavefront, a piece; a length that one piece holds
// needs no joining launch.  (64 ragged requests of up to 8192 tokens, 8 key heads: 120 us in 512 whole-length workgroups, 130 us in 1024 and
// more pieces; one of 100001 tokens, 2 key heads: 21 us at 512, 24 us at 1024; 16 x 300 candidates over 1000 tokens: 23 against 34 us.)

constexpr long long WANT_WG = 512;
Split split_of(int n, int Hkv, int G, int max_q, int max_len, int& nq) {
  Split s;
  const long long cols = (long long)max_q * G;
  nq = cols <= 32 ? 1 : 2;
  s.nqt = (int)cdiv64(cols, 16 * nq);
  const long long base = (long long)n * Hkv * s.nqt, nb = cdiv64(max_len, BS);
  long long chunk = cdiv64(nb * base, WANT_WG);
  if (chunk < 4) chunk = 4;
  if (chunk > nb) chunk = nb > 0 ? nb : 1;
  s.chunk = (int)chunk;
  s.pieces = (int)(nb > 0 ? cdiv64(nb, chunk) : 1);
  return s;
}

template <int DH, int NQ> void launch_kv(const KvArgs& a, const Split& s, float* po, float2* ml, hipStream_t st) {
  const unsigned grid = (unsigned)((long long)a.n * a.c.Hkv * s.pieces * s.nqt);
  if (a.cap > 0.f && dmt_cap(a.scale, a.cap, true).near) kv_tile_kernel<DH, NQ, 2><<<grid, 256, 0, st>>>(a, s, po, ml);
  else if (a.cap > 0.f || a.slopes) kv_tile_kernel<DH, NQ, 1><<<grid, 256, 0, st>>>(a, s, po, ml);
  else kv_tile_kernel<DH, NQ, 0><<<grid, 256, 0, st>>>(a, s, po, ml);
}
template <int NQ> void launch_kv_dh(const KvArgs& a, const Split& s, float* po, float2* ml, hipStream_t st) {
  switch (a.c.dh) {
    case 16: launch_kv<16, NQ>(a, s, po, ml, st); break;
    case 32: launch_kv<32, NQ>(a, s, po, ml, st); break;
    case 48: launch_kv<48, NQ>(a, s, po, ml, st); break;
    case 64: launch_kv<64, NQ>(a, s, po, ml, st); break;
    case 80: launch_kv<80, NQ>(a, s, po, ml, st); break;
    case 96: launch_kv<96, NQ>(a, s, po, ml, st); break;
    case 112: launch_kv<112, NQ>(a, s, po, ml, st); break;
    default: launch_kv<128, NQ>(a, s, po, ml, st); break;
  }
}

bool cache_ok(int Hkv, int dh, int n_blocks, const void* k, const void* v, const float* ks, const float* vs) {
  return Hkv > 0 && Hkv <= 65535 && dh > 0 && dh <= MAX_DH && dh % 16 == 0 && n_blocks > 0 && n_blocks <= 0x7fffffff / BS && k && v && ks && vs &&
         (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0;
}
const char* CACHE_MSG = "%s: bad cache (Hkv %d, dh %d -- a multiple of 16 up to 128 -- , %d blocks; 16-byte aligned pools, slots below 2^31)";

}  // namespace

extern "C" uint64_t dmt_kv_plan_ws_bytes(int32_t n) { return n < 0 ? 0 : 16 + 8ull * (uint64_t)n; }

extern "C" int dmt_kv_plan(int32_t n, int32_t rows, const int32_t* lens, const int32_t* new_lens, int32_t* table, int32_t width,
                           const int32_t* free_ids, int32_t free_cap, const int32_t* n_free, int32_t* row_off, int32_t* lens_out, int32_t* slots, int32_t* run_row,
                           int32_t* run_len, int32_t* state, void* ws, uint64_t ws_bytes, void* stream) {
  DMT_CHECK_ARG(n >= 0 && rows >= 0 && width >= 0 && rows <= 0x3fffffff, "dmt_kv_plan: n %d, rows %d (at most 2^30), width %d", n, rows, width);
  DMT_CHECK_ARG(n_free && row_off && state && free_cap >= 0, "dmt_kv_plan: NULL n_free / row_off / state");
  DMT_CHECK_ARG(n == 0 || (lens && new_lens && lens_out && table && free_ids), "dmt_kv_plan: NULL lens / new_lens / lens_out / table / free_ids");
  DMT_CHECK_ARG(rows == 0 || (slots && run_row && run_len), "dmt_kv_plan: NULL slots / run_row / run_len");
  DMT_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= dmt_kv_plan_ws_bytes(n), "dmt_kv_plan: workspace of %llu bytes needed",
                (unsigned long long)dmt_kv_plan_ws_bytes(n));
  DMT_CHECK_ARG(state != n_free && (n == 0 || lens_out != lens), "dmt_kv_plan: lens_out and state are written before lens and n_free were read");
  PlanArgs a;
  a.n = n; a.rows = rows; a.width = width;
  const long long mr = (long long)rows / BS + 2ll * n;
  a.max_runs = (int)(mr < rows ? mr : rows);
  a.lens = lens; a.new_lens = new_lens; a.table = table; a.free_ids = free_ids; a.free_cap = free_cap; a.n_free = n_free;
  a.row_off = row_off; a.lens_out = lens_out; a.slots = slots; a.run_row = run_row; a.run_len = run_len; a.state = state;
  a.totals = (int*)ws;
  a.req = (int2*)((char*)ws + 16);
  const int small = rows <= PLAN_SMALL_ROWS;
  plan_kernel<<<1, PLAN_NT, 0, (hipStream_t)stream>>>(a, small);
  DMT_CHECK_LAUNCH("dmt_kv_plan");
  if (!small) {
    plan_rows_kernel<<<(unsigned)cdiv64(rows, 256), 256, 0, (hipStream_t)stream>>>(a);
    DMT_CHECK_LAUNCH("dmt_kv_plan(rows)");
  }
  return DMT_OK;
}

extern "C" int dmt_kv_release(int32_t n, const int32_t* done, int32_t* lens, const int32_t* table, int32_t width, int32_t* free_ids, int32_t* n_free,
                              int32_t cap, void* stream) {
  DMT_CHECK_ARG(n >= 0 && width >= 0 && cap >= 0, "dmt_kv_release: negative size");
  if (n == 0) return DMT_OK;
  DMT_CHECK_ARG(done && lens && table && free_ids && n_free, "dmt_kv_release: NULL pointer");
  release_kernel<<<1, PLAN_NT, 0, (hipStream_t)stream>>>(n, done, lens, table, width, free_ids, n_free, cap);
  DMT_CHECK_LAUNCH("dmt_kv_release");
  return DMT_OK;
}

extern "C" int dmt_kv_append(int32_t Hkv, int32_t dh, int32_t n_blocks, uint8_t* k, uint8_t* v, float* k_scale, float* v_scale, int32_t rows,
                             const void* k_rows, int64_t k_rs, const void* v_rows, int64_t v_rs, const int32_t* slots, const int32_t* run_row,
                             const int32_t* run_len, int32_t max_runs, void* stream) {
  DMT_CHECK_ARG(cache_ok(Hkv, dh, n_blocks, k, v, k_scale, v_scale), CACHE_MSG, "dmt_kv_append", Hkv, dh, n_blocks);
  DMT_CHECK_ARG(rows >= 0 && max_runs >= 0, "dmt_kv_append: negative size");
  if (rows == 0 || max_runs == 0) return DMT_OK;
  DMT_CHECK_ARG(k_rows && v_rows && slots && run_row && run_len, "dmt_kv_append: NULL rows / slots / runs");
  DMT_CHECK_ARG(k_rs >= (int64_t)Hkv * dh && v_rs >= (int64_t)Hkv * dh && k_rs % 8 == 0 && v_rs % 8 == 0 && (uintptr_t)k_rows % 16 == 0 &&
                    (uintptr_t)v_rows % 16 == 0, "dmt_kv_append: rows of at least Hkv * dh, 16-byte aligned");
  const Cache c = {Hkv, dh, n_blocks, k, v, k_scale, v_scale};
  append_kernel<<<dim3(max_runs, Hkv), 256, 0, (hipStream_t)stream>>>(c, rows, (const bf16_t*)k_rows, k_rs, (const bf16_t*)v_rows, v_rs, slots, run_row,
                                                                      run_len);
  DMT_CHECK_LAUNCH("dmt_kv_append");
  return DMT_OK;
}

extern "C" int dmt_kv_read(int32_t Hkv, int32_t dh, int32_t n_blocks, const uint8_t* k, const uint8_t* v, const float* k_scale, const float* v_scale,
                           int32_t n, const int32_t* slots, void* k_rows, int64_t k_rs, void* v_rows, int64_t v_rs, void* stream) {
  DMT_CHECK_ARG(cache_ok(Hkv, dh, n_blocks, k, v, k_scale, v_scale), CACHE_MSG, "dmt_kv_read", Hkv, dh, n_blocks);
  DMT_CHECK_ARG(n >= 0, "dmt_kv_read: negative size");
  if (n == 0) return DMT_OK;
  DMT_CHECK_ARG(k_rows && v_rows && slots, "dmt_kv_read: NULL rows / slots");
  DMT_CHECK_ARG(k_rs >= (int64_t)Hkv * dh && v_rs >= (int64_t)Hkv * dh && k_rs % 8 == 0 && v_rs % 8 == 0 && (uintptr_t)k_rows % 16 == 0 &&
                    (uintptr_t)v_rows % 16 == 0, "dmt_kv_read: rows of at least Hkv * dh, 16-byte aligned");
  const Cache c = {Hkv, dh, n_blocks, (uint8_t*)k, (uint8_t*)v, (float*)k_scale, (float*)v_scale};
  read_kernel<<<dim3((unsigned)cdiv64(n, 64), Hkv), 256, 0, (hipStream_t)stream>>>(c, n, slots, (bf16_t*)k_rows, k_rs, (bf16_t*)v_rows, v_rs);
  DMT_CHECK_LAUNCH("dmt_kv_read");
  return DMT_OK;
}

static uint64_t kv_ws(const dmt_kv_attn_desc* d, Split* s, int* nq, uint64_t* ml_at) {
  *s = split_of(d->n, d->Hkv, d->Hq / d->Hkv, d->max_q, d->max_len, *nq);
  const uint64_t cols = (uint64_t)d->n * d->Hkv * s->pieces * s->nqt * 16 * (uint64_t)*nq;
  *ml_at = cols * (uint64_t)d->dh * 4;
  return s->pieces > 1 ? cols * ((uint64_t)d->dh * 4 + 8) : 0;
}

// (split_of and kv_ws count in 64 bits: n Hkv and the tiles of columns stay below 2^31 each and together)
static bool launch_fits(const dmt_kv_attn_desc* d) {
  const int64_t cols = (int64_t)d->max_q * (d->Hq / d->Hkv), heads = (int64_t)d->n * d->Hkv;
  return cols < (1ll << 31) && heads < (1ll << 31) && heads * cdiv64(cols, cols <= 32 ? 16 : 32) < (1ll << 31);
}

extern "C" uint64_t dmt_kv_attn_ws_bytes(const dmt_kv_attn_desc* d) {
  if (!d || d->n <= 0 || d->Hkv <= 0 || d->Hq < d->Hkv || d->max_q <= 0 || d->max_len <= 0 || d->dh <= 0 || !launch_fits(d)) return 0;
  Split s;
  int nq;
  uint64_t ml;
  return kv_ws(d, &s, &nq, &ml);
}

extern "C" int dmt_kv_attn(const dmt_kv_attn_desc* d, void* stream) {
  DMT_CHECK_ARG(d, "dmt_kv_attn: no descriptor");
  DMT_CHECK_ARG(cache_ok(d->Hkv, d->dh, d->n_blocks, d->k, d->v, d->k_scale, d->v_scale), CACHE_MSG, "dmt_kv_attn", d->Hkv, d->dh, d->n_blocks);
  DMT_CHECK_ARG(d->Hq > 0 && d->Hq <= 65535 && d->Hq % d->Hkv == 0, "dmt_kv_attn: Hq %d is not a multiple of Hkv %d", d->Hq, d->Hkv);
  DMT_CHECK_ARG(d->n >= 0 && d->n <= 65535 && d->max_q >= 0 && d->max_len >= 0 && d->width >= 0 && d->rows >= 0 && d->rows < (1ll << 31),
                "dmt_kv_attn: n %d (at most 65535), max_q %d, max_len %d, width %d", d->n, d->max_q, d->max_len, d->width);
  DMT_CHECK_ARG(d->scale > 0.f && d->scale <= 1e38f && d->cap >= 0.f && d->cap <= 1e38f,
                "dmt_kv_attn: scale must be positive, cap 0 or positive, both at most 1e38");
  const bool none = d->n == 0 || d->max_q == 0;
  if (d->rows == 0 || (none && !d->rest)) return DMT_OK;
  DMT_CHECK_ARG(d->Q && d->out && (none || (d->lens && d->row_off && (d->table || d->width == 0))), "dmt_kv_attn: NULL pointer");
  const int64_t wq = (int64_t)d->Hq * d->dh;
  DMT_CHECK_ARG(d->q_rs >= wq && d->o_rs >= wq && d->q_rs % 8 == 0 && d->o_rs % 8 == 0 && (uintptr_t)d->Q % 16 == 0 && (uintptr_t)d->out % 16 == 0,
                "dmt_kv_attn: rows of at least Hq * dh, 16-byte aligned");
  KvArgs a;
  a.c = {d->Hkv, d->dh, d->n_blocks, (uint8_t*)d->k, (uint8_t*)d->v, (float*)d->k_scale, (float*)d->v_scale};
  a.n = d->n; a.Hq = d->Hq; a.G = d->Hq / d->Hkv; a.max_q = d->max_q; a.max_len = d->max_len; a.width = d->width; a.causal = d->causal != 0;
  a.rest = d->rest;
  a.rows = d->rows; a.Q = (const bf16_t*)d->Q; a.q_rs = d->q_rs; a.table = d->table; a.lens = d->lens; a.row_off = d->row_off;
  a.scale = d->scale; a.cap = d->cap; a.slopes = d->slopes; a.out = (bf16_t*)d->out; a.o_rs = d->o_rs; a.lse = d->lse;
  if (none) {
    kv_rest_kernel<<<(unsigned)(d->rows < 4096 ? d->rows : 4096), 256, 0, (hipStream_t)stream>>>(a);
    DMT_CHECK_LAUNCH("dmt_kv_attn(no request)");
    return DMT_OK;
  }
  DMT_CHECK_ARG(launch_fits(d), "dmt_kv_attn: the launch passes 2^31 workgroups");
  Split s;
  int nq;
  uint64_t ml_at;
  const uint64_t need = kv_ws(d, &s, &nq, &ml_at);
  DMT_CHECK_ARG(need == 0 || (d->ws && (uintptr_t)d->ws % 16 == 0 && d->ws_bytes >= need), "dmt_kv_attn: workspace of %llu bytes needed",
                (unsigned long long)need);
  DMT_CHECK_ARG((long long)d->n * d->Hkv * s.nqt * s.pieces < (1ll << 31), "dmt_kv_attn: the launch passes 2^31 workgroups");
  DMT_CHECK_ARG(d->out != d->Q, "dmt_kv_attn: out must not be Q");
  float* po = (float*)d->ws;
  float2* ml = need ? (float2*)((char*)d->ws + ml_at) : nullptr;
  if (nq == 1) launch_kv_dh<1>(a, s, po, ml, (hipStream_t)stream);
  else launch_kv_dh<2>(a, s, po, ml, (hipStream_t)stream);
  DMT_CHECK_LAUNCH(s.pieces > 1 ? "dmt_kv_attn(pieces)" : "dmt_kv_attn");
  if (s.pieces > 1) {
    const int gpc = s.pieces <= 4 ? 1 : (s.pieces <= 16 ? 4 : 16);
    const dim3 grid((unsigned)cdiv64((long long)a.max_q * a.G, 16 / gpc), a.c.Hkv, a.n);
    if (nq == 1) kv_join_kernel<1><<<grid, 256, 0, (hipStream_t)stream>>>(a, s, gpc, po, ml);
    else kv_join_kernel<2><<<grid, 256, 0, (hipStream_t)stream>>>(a, s, gpc, po, ml);
    DMT_CHECK_LAUNCH("dmt_kv_attn(join)");
  }
  return DMT_OK;
}
