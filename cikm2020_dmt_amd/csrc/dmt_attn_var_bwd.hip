// Attention over packed rows of any length: backward.  Two kernels recompute the weights from the saved row sums -- one owns query rows (dQ and
// the slopes' gradient), one owns key rows (dK, dV, over all query heads of the group) -- so that nothing is added by atomics.
#include "dmt_attn_var.h"

using namespace attn_var;

namespace {

// D[row, h] = sum_c dout[row, h, c] out[row, h, c]; a row per 16 lanes
template <typename T>
__global__ __launch_bounds__(256) void rowsum_kernel(const Args a) {
  const long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int l16 = threadIdx.x & 15;
  if (item >= a.rows_q * a.Hq) return;
  const long long row = item / a.Hq;
  const int h = (int)(item - row * a.Hq);
  const T* g = (const T*)a.dout + row * a.do_rs + (long long)h * a.dh;
  float s = 0.f;
  const T* o = (const T*)a.out + row * a.o_rs + (long long)h * a.dh;
  for (int c = l16; c < a.dh; c += 16) s = __builtin_fmaf(ldf<T>(g + c), ldf<T>(o + c), s);
  s += __shfl_xor(s, 8);
  s += __shfl_xor(s, 4);
  s += __shfl_xor(s, 2);
  s += __shfl_xor(s, 1);
  if (l16 == 0) a.D[item] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void rows_dq_kernel(const Args a) {
  __shared__ float lds[4][ROW_LDS];
  __shared__ float part[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.z, h = blockIdx.y;
  const Ex e = example(a, b);
  float sl = 0.f;
  for (int i = blockIdx.x * 128 + wave; i < e.ql && i < (int)blockIdx.x * 128 + 128; i += 4) sl += row_dq<T>(a, e, h, i, lds[wave], lane);
  if (a.slope_part) {
    if (lane == 0) part[wave] = sl;
    __syncthreads();
    if (threadIdx.x == 0) a.slope_part[((long long)h * a.B + b) * gridDim.x + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void rows_dkv_kernel(const Args a) {
  __shared__ float lds[4][ROW_LDS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.z, hk = blockIdx.y;
  const Ex e = example(a, b);
  const int j = blockIdx.x * 4 + wave;
  if (j < e.kl) row_dkv<T>(a, e, hk, j, lds[wave], lane);
}

// dslopes[h] += sum of its parts, in their order (64 bits: the terms cancel)
__global__ __launch_bounds__(256) void slopes_kernel(const float* part, long long n, float* out) {
  __shared__ double red[256];
  const float* p = part + (long long)blockIdx.x * n;
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += 256) s += (double)p[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] += (float)red[0];
}

template <typename T>
int launch_bwd(const Args& a, hipStream_t st) {
  const long long items = a.rows_q * a.Hq;
  if (items && a.max_q) {
    rowsum_kernel<T><<<(unsigned)cdiv64(items, 16), 256, 0, st>>>(a);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(row sums)");
    const int nt = (int)cdiv64(a.max_q, 128);
    rows_dq_kernel<T><<<dim3(nt, a.Hq, a.B), 256, 0, st>>>(a);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(dq rows)");
    if (a.slope_part) {
      slopes_kernel<<<a.Hq, 256, 0, st>>>(a.slope_part, (long long)a.B * nt, a.dslopes);
      DMT_CHECK_LAUNCH("dmt_attn_var_bwd(slopes)");
    }
  }
  if (a.rows_k && a.max_k) {
    rows_dkv_kernel<T><<<dim3((a.max_k + 3) / 4, a.Hkv, a.B), 256, 0, st>>>(a);
    DMT_CHECK_LAUNCH("dmt_attn_var_bwd(dkv rows)");
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
