// attention.cu — softmax attention and its gradient: entry points, argument checks and the kernels.
#include <cmath>

#include "attention.cuh"
#include "conv_plan.h"

namespace wb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

WB_DEV float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// A warp holds a row of up to 128 values, 4 a lane.
template <typename T>
WB_DEV void row4(const T* p, int D, int lane, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lane * 4 + i < D ? to_float(p[lane * 4 + i]) : 0.f;
}
template <typename T>
WB_DEV void put4(T* p, int D, int lane, const float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane * 4 + i < D) p[lane * 4 + i] = from_float<T>(v[i]);
}
WB_DEV float dot4(const float* x, const float* y) {
  return warp_sum(x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3]);
}

// delta = rowsum(dO * O) and the log-sum-exp in units of log 2, padded with what gives probability 0
template <typename T>
__global__ void __launch_bounds__(128) attn_delta_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + threadIdx.x / 32, h = blockIdx.y, b = blockIdx.z;
  if (i >= p.t_pad) return;
  const AttnItem it(a, b);
  float d = 0.f, l = INFINITY;
  if (i < it.ql) {
    float x[4], y[4];
    row4(at<T>(a.dout, b, i, h), a.D, lane, x);
    row4(at<T>(a.out, b, i, h), a.D, lane, y);
    d = dot4(x, y);
    l = a.lse[((long long)b * a.Hq + h) * a.Tq + i] * kLog2e;
    if (l == -INFINITY) l = INFINITY;
  }
  if (lane == 0) {
    const long long r = ((long long)b * a.Hq + h) * p.t_pad + i;
    p.delta[r] = d;
    p.lse2[r] = l;
  }
}

// dQ, a warp per query
template <typename T>
__global__ void __launch_bounds__(128) attn_dq_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + threadIdx.x / 32, h = blockIdx.y, b = blockIdx.z;
  if (i >= a.Tq) return;
  const AttnItem it(a, b);
  float q[4], g[4], acc[4] = {}, k[4], v[4];
  row4(at<T>(a.q, b, i, h), a.D, lane, q);
  row4(at<T>(a.dout, b, i, h), a.D, lane, g);
  const long long r = ((long long)b * a.Hq + h) * p.t_pad + i;
  const float l2 = p.lse2[r], delta = p.delta[r];
  for (int j = it.key_lo(a, i); j < it.key_hi(a, i); ++j) {
    row4(at<T>(a.k, b, j, h / p.group), a.D, lane, k);
    row4(at<T>(a.v, b, j, h / p.group), a.D, lane, v);
    const float w = exp2f(dot4(q, k) * a.scale * kLog2e - l2);
    const float ds = w * (dot4(g, v) - delta) * a.scale;
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[d] += ds * k[d];
  }
  put4(at<T>(a.dq, b, i, h), a.D, lane, acc);
}

// dK and dV, a warp per key, over the query heads that share it
template <typename T>
__global__ void __launch_bounds__(128) attn_dkv_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int lane = threadIdx.x & 31, j = blockIdx.x * 4 + threadIdx.x / 32, hk = blockIdx.y, b = blockIdx.z;
  if (j >= a.Tk) return;
  const AttnItem it(a, b);
  float k[4] = {}, v[4] = {}, dk[4] = {}, dv[4] = {}, q[4], g[4];
  if (j < it.kl) {
    row4(at<T>(a.k, b, j, hk), a.D, lane, k);
    row4(at<T>(a.v, b, j, hk), a.D, lane, v);
  }
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    for (int i = it.query_lo(a, j); i < it.query_hi(a, j); ++i) {
      row4(at<T>(a.q, b, i, h), a.D, lane, q);
      row4(at<T>(a.dout, b, i, h), a.D, lane, g);
      const long long r = ((long long)b * a.Hq + h) * p.t_pad + i;
      const float w = exp2f(dot4(q, k) * a.scale * kLog2e - p.lse2[r]);
      const float ds = w * (dot4(g, v) - p.delta[r]) * a.scale;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        dv[d] += w * g[d];
        dk[d] += ds * q[d];
      }
    }
  }
  put4(at<T>(a.dk, b, j, hk), a.D, lane, dk);
  put4(at<T>(a.dv, b, j, hk), a.D, lane, dv);
}

}  // namespace

bool attn_map(CUtensorMap* m, const WubuB200View& v, int B, int T, int H, int D) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)T, (uint64_t)H, (uint64_t)B};
  // the stride of a unit extent is never applied, but has to be a positive multiple of 16
  const uint64_t strides[3] = {v.token ? (uint64_t)v.token * 2 : 16, v.head ? (uint64_t)v.head * 2 : 16,
                               v.batch ? (uint64_t)v.batch * 2 : 16};
  return make_map_16bit_4d(m, v.data, dims, strides, 64, kTile);
}

int attn_backward(const AttnParams& p, cudaStream_t st) {
  const WubuB200Attn& a = p.a;
  with_dtype(a.dtype, [&](auto t) {
    typedef decltype(t) T;
    if (a.Tq) {
      attn_delta_kernel<T><<<dim3(p.t_pad / 4, a.Hq, a.B), 128, 0, st>>>(p);
      attn_dq_kernel<T><<<dim3((a.Tq + 3) / 4, a.Hq, a.B), 128, 0, st>>>(p);
    }
    if (a.Tk) attn_dkv_kernel<T><<<dim3((a.Tk + 3) / 4, a.Hkv, a.B), 128, 0, st>>>(p);
  });
  return ops_launched("attn_backward");
}

namespace {

// 1 = nothing to do
int check_shape(const WubuB200Attn* a) {
  if (!a || (a->dtype != WUBU_B200_BF16 && a->dtype != WUBU_B200_F16) || a->B < 0 || a->Hq < 0 || a->Hkv < 0 ||
      a->Tq < 0 || a->Tk < 0 || a->window < 0 || !(a->scale >= 0.f) || a->scale == INFINITY)
    return WUBU_B200_ERR_ARG;
  if (a->D < 8 || a->D > 128 || a->D % 8 || a->B > 65535 || a->Hq > 65535 || a->Tq > (1 << 28) || a->Tk > (1 << 28))
    return WUBU_B200_ERR_SHAPE;
  if (a->B == 0 || a->Hq == 0) return a->Hq == 0 && a->Hkv != 0 ? WUBU_B200_ERR_SHAPE : 1;
  if (a->Hkv == 0 || a->Hq % a->Hkv) return WUBU_B200_ERR_SHAPE;
  return a->Tq == 0 && a->Tk == 0 ? 1 : WUBU_B200_OK;
}

// Alignment and strides of a view of T x H rows; strides of unit extents mean nothing and become 0.
bool check_view(WubuB200View& v, int B, int T, int H, int D) {
  if (T == 0) return true;
  if (!v.data || !aligned16(v.data)) return false;
  const int n[3] = {B, T, H};
  long long* s[3] = {&v.batch, &v.token, &v.head};
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) *s[i] = 0;
    else if (*s[i] < D || *s[i] % 8 || *s[i] >= (1ll << 38)) return false;  // 40 bits of bytes in a tensor map
  }
  return true;
}

int padded(int T) { return (T + 127) / 128 * 128; }

long long backward_bytes(const WubuB200Attn& a) { return 2ll * a.B * a.Hq * padded(a.Tq) * (long long)sizeof(float); }

int prepare(const WubuB200Attn* in, AttnParams& p) {
  const int rc = check_shape(in);
  if (rc != WUBU_B200_OK) return rc;
  p.a = *in;
  WubuB200Attn& a = p.a;
  if (a.scale == 0.f) a.scale = 1.f / sqrtf((float)a.D);
  p.group = a.Hq / a.Hkv;
  p.t_pad = padded(a.Tq);
  if (!check_view(a.q, a.B, a.Tq, a.Hq, a.D) || !check_view(a.k, a.B, a.Tk, a.Hkv, a.D) ||
      !check_view(a.v, a.B, a.Tk, a.Hkv, a.D) || !check_view(a.out, a.B, a.Tq, a.Hq, a.D) || (a.Tq && !a.lse))
    return WUBU_B200_ERR_ARG;
  p.wait_ns = wait_limit_ns();
  return WUBU_B200_OK;
}

}  // namespace
}  // namespace wb

using namespace wb;

extern "C" {

long long wubu_b200_attn_workspace(const WubuB200Attn* a, int backward) {
  const int rc = check_shape(a);
  if (rc != WUBU_B200_OK) return rc == 1 ? 0 : rc;
  return backward ? backward_bytes(*a) : attn_fwd_bytes(*a);
}

int wubu_b200_attn_forward(const WubuB200Attn* in, void* stream) {
  AttnParams p{};
  const int rc = prepare(in, p);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  if (p.a.Tq == 0) return WUBU_B200_OK;
  if (const long long n = attn_fwd_bytes(p.a)) {
    if (!p.a.workspace || !aligned16(p.a.workspace)) return WUBU_B200_ERR_ARG;
    if (p.a.workspace_bytes < n) return WUBU_B200_ERR_NOMEM;
  }
  p.err = ops_status_word();
  if (!p.err) return WUBU_B200_ERR_CUDA;
  return attn_forward(p, (cudaStream_t)stream);
}

int wubu_b200_attn_backward(const WubuB200Attn* in, void* stream) {
  AttnParams p{};
  const int rc = prepare(in, p);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  WubuB200Attn& a = p.a;
  if (!check_view(a.dout, a.B, a.Tq, a.Hq, a.D) || !check_view(a.dq, a.B, a.Tq, a.Hq, a.D) ||
      !check_view(a.dk, a.B, a.Tk, a.Hkv, a.D) || !check_view(a.dv, a.B, a.Tk, a.Hkv, a.D))
    return WUBU_B200_ERR_ARG;
  if (a.Tq) {
    if (!a.workspace || !aligned16(a.workspace)) return WUBU_B200_ERR_ARG;
    if (a.workspace_bytes < backward_bytes(a)) return WUBU_B200_ERR_NOMEM;
  }
  p.delta = static_cast<float*>(a.workspace);
  p.lse2 = p.delta + (long long)a.B * a.Hq * p.t_pad;
  p.err = ops_status_word();
  if (!p.err) return WUBU_B200_ERR_CUDA;
  return attn_backward(p, (cudaStream_t)stream);
}

}  // extern "C"
