// attention.cu — softmax attention and its gradient: entry points and argument checks.
#include <cmath>

#include "attention.cuh"
#include "conv_plan.h"

namespace wb {

bool attn_map(CUtensorMap* m, const WubuB200View& v, int B, int T, int H, int D) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)T, (uint64_t)H, (uint64_t)B};
  // the stride of a unit extent is never applied, but has to be a positive multiple of 16
  const uint64_t strides[3] = {v.token ? (uint64_t)v.token * 2 : 16, v.head ? (uint64_t)v.head * 2 : 16,
                               v.batch ? (uint64_t)v.batch * 2 : 16};
  return make_map_16bit_4d(m, v.data, dims, strides, 64, kTile);
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

int prepare(const WubuB200Attn* in, AttnParams& p) {
  const int rc = check_shape(in);
  if (rc != WUBU_B200_OK) return rc;
  p.a = *in;
  WubuB200Attn& a = p.a;
  if (a.scale == 0.f) a.scale = 1.f / sqrtf((float)a.D);
  p.group = a.Hq / a.Hkv;
  p.t_pad = (a.Tq + kTile - 1) / kTile * kTile;
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
  return backward ? attn_bwd_bytes(*a) : attn_fwd_bytes(*a);
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
  if (!a.workspace || !aligned16(a.workspace)) return WUBU_B200_ERR_ARG;
  if (a.workspace_bytes < attn_bwd_bytes(a)) return WUBU_B200_ERR_NOMEM;
  p.err = ops_status_word();
  if (!p.err) return WUBU_B200_ERR_CUDA;
  return attn_backward(p, (cudaStream_t)stream);
}

}  // extern "C"
