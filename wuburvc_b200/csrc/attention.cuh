// attention.cuh — softmax attention and its gradient: parameters and index arithmetic of the kernels.
#pragma once
#include "ops.cuh"

namespace wb {

struct AttnParams {
  WubuB200Attn a;    // with scale resolved and strides of unit extents cleared
  int group;         // query heads to a key / value head
  float* delta;      // backward: [B][Hq][t_pad] rowsum(dO * O)
  float* lse2;       // backward: [B][Hq][t_pad] lse in units of log 2; +infinity where a query sees nothing
  int t_pad;
  int* err;
  unsigned long long wait_ns;
};

// One item's lengths, and the range of keys that a query sees: query i sits at place i + off.
struct AttnItem {
  int ql, kl, off;
  WB_DEV AttnItem(const WubuB200Attn& a, int b) {
    ql = a.q_lens ? min(max(__ldg(a.q_lens + b), 0), a.Tq) : a.Tq;
    kl = a.k_lens ? min(max(__ldg(a.k_lens + b), 0), a.Tk) : a.Tk;
    off = kl - ql;
  }
  // keys [lo, hi) of query i (hi <= lo: none)
  WB_DEV int key_lo(const WubuB200Attn& a, int i) const {
    return a.window > 0 && a.window < a.Tq + a.Tk ? max(0, i + off - a.window + 1) : 0;
  }
  WB_DEV int key_hi(const WubuB200Attn& a, int i) const {
    if (i >= ql) return 0;
    if (a.causal) return min(kl, i + off + 1);
    return a.window > 0 && a.window < a.Tq + a.Tk ? min(kl, i + off + a.window) : kl;
  }
  // queries [lo, hi) that see key j
  WB_DEV int query_lo(const WubuB200Attn& a, int j) const {
    if (a.causal) return max(0, j - off);
    return a.window > 0 && a.window < a.Tq + a.Tk ? max(0, j - off - a.window + 1) : 0;
  }
  WB_DEV int query_hi(const WubuB200Attn& a, int j) const {
    if (j >= kl) return 0;
    return a.window > 0 && a.window < a.Tq + a.Tk ? min(ql, j - off + a.window) : ql;
  }
};

template <typename T>
WB_DEV T* at(const WubuB200View& v, int b, int t, int h) {
  return static_cast<T*>(v.data) + b * v.batch + t * v.token + h * v.head;
}

int attn_forward(const AttnParams& p, cudaStream_t st);
int attn_backward(const AttnParams& p, cudaStream_t st);

}  // namespace wb
