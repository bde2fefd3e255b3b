// attention_bwd.cu — the gradient of softmax attention on the tensor cores.
//
// With P = 2^(c S - L) recomputed from the scores and the log-sum-exp L (c = scale log2 e, L in units of
// log 2), D_i = sum_d dO_id O_id and dS = P (dO V^T - D):
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K.
// dK and dV are sums over queries and dQ is a sum over keys.  One grid does both, in two roles: a CTA of the
// first owns 128 keys and runs over the queries that see them (and over the query heads that share
// the key head), a CTA of the second owns 128 queries and runs over their keys.  S and dO V^T are formed in
// both (7 products where 5 are the least), and in return no sum crosses CTAs: there are no atomics
// and the result does not depend on the order in which CTAs run.
//
// Everything between the products stays in tensor memory.  The first role forms the transposed scores
// (rows are keys), so that P^T and dS^T are written over them as the A operands of the next products.
// Eight warps do the exponentials, two to a row quadrant, 64 columns a thread; one warp loads, one
// issues.  A step's products and its elementwise halves alternate:
//   keys' role:     tensor  dV(n) S(n+1) | dK(n) dP(n+1)      warps  dS(n) | P(n+1)
//   queries' role:  tensor  dQ(n) dP(n+1) S(n+2)              warps  P(n+1) dS(n+1)
//
// fp16 has few small numbers and a low ceiling, so its P is scaled by 2^14 (P <= 1) and its dS by the
// power of two that the norms of dO and V allow: |dS| <= P (|dO_i| |V_j| + |D_i|) <= 2 max|dO| max|V|.
#include <type_traits>

#include "attention.cuh"

namespace wb {
namespace {

constexpr int kStagesA = 3, kStagesB = 2;  // the keys' role uses two of the first ring
constexpr int kProducer = 8, kMma = 9, kThreads = 384;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnBwdMaps {
  CUtensorMap q, k, v, dout;
};

template <typename T>
struct BwdShift {
  static constexpr float value = 0.f;
};
template <>
struct BwdShift<f16> {
  static constexpr float value = 14.f;
};

struct Barriers {
  uint64_t res_full, a_full[kStagesA], a_empty[kStagesA], b_full[kStagesB], b_empty[kStagesB], s_full[2], dp_full, p_ready,
      ds_ready, acc_full, mma_done;
};

// the power of two that dS is scaled by (fp16), from the bits of the largest squared row norms
template <typename T>
WB_DEV float ds_scale(const AttnParams& p, int b, int hk) {
  if (!std::is_same<T, f16>::value) return 1.f;
  const int n = p.a.B * p.a.Hkv, i = b * p.a.Hkv + hk;
  const float m = sqrtf(__uint_as_float(p.norm_bits[i])) * sqrtf(__uint_as_float(p.norm_bits[n + i]));
  if (!(m > 0.f) || m > 1e30f) return 1.f;
  return exp2f(fminf(floorf(log2f(16384.f / m)), 100.f));
}

WB_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
attn_bwd_tc_kernel(const __grid_constant__ AttnBwdMaps maps, const __grid_constant__ AttnParams p, int kv_ctas) {
  constexpr int kBoxes = DP / 64;
  constexpr uint32_t kTileBytes = kBoxes * kBox;
  constexpr float kShift = BwdShift<T>::value;
  constexpr int kBf16 = std::is_same<T, bf16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* res0 = smem;                  // K or Q, for the whole CTA
  uint8_t* res1 = smem + kTileBytes;     // V or dO
  uint8_t* ra = smem + 2 * kTileBytes;   // ring of Q or K
  uint8_t* rb = ra + kStagesA * kTileBytes;  // ring of dO or V
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_slot;
  // keys' role: the log-sum-exp and D of a step's 128 queries, two steps, in the first ring's third tile
  float* rows = reinterpret_cast<float*>(ra + 2 * kTileBytes);

  const WubuB200Attn& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool kv = (int)blockIdx.x < kv_ctas;
  // this CTA's tile: keys in order (causal: the first have the most queries), queries from the last on
  int tile, hq, hk, b, t0 = 0, t1 = 0, heads;
  {
    const int heads_all = (kv ? a.Hkv : a.Hq) * a.B;
    const int id = kv ? (int)blockIdx.x : (int)blockIdx.x - kv_ctas;
    const int r = id / heads_all, hb = id - r * heads_all;
    const int h = hb % (kv ? a.Hkv : a.Hq);
    b = hb / (kv ? a.Hkv : a.Hq);
    tile = kv ? r : (a.Tq + kTile - 1) / kTile - 1 - r;
    hk = kv ? h : h / p.group;
    hq = kv ? h * p.group : h;
    heads = kv ? p.group : 1;
  }
  const AttnItem it(a, b);
  const int own0 = tile * kTile;
  {  // the other side's tiles [t0, t1) that any of this tile's rows meets
    const int last = min(own0 + kTile, kv ? it.kl : it.ql) - 1;
    if (last >= own0) {
      const int lo = kv ? it.query_lo(a, own0) : it.key_lo(a, own0), hi = kv ? it.query_hi(a, last) : it.key_hi(a, last);
      if (hi > lo) {
        t0 = lo / kTile;
        t1 = (hi + kTile - 1) / kTile;
      }
    }
  }
  const int per_head = t1 - t0, steps = per_head * heads;
  // slot and phase of step n in the rings
  const int na = kv ? 2 : kStagesA;
  auto slot_a = [&](int n) { return kv ? n & 1 : n % kStagesA; };
  auto phase_a = [&](int n) { return (uint32_t)(kv ? n >> 1 : n / kStagesA) & 1u; };
  auto slot_b = [&](int n) { return n % kStagesB; };
  auto phase_b = [&](int n) { return (uint32_t)(n / kStagesB) & 1u; };

  if (threadIdx.x == 0) {
    mbar_init(&bar.res_full, 1);
    for (int i = 0; i < kStagesA; ++i) {
      mbar_init(&bar.a_full[i], 1);
      mbar_init(&bar.a_empty[i], 1);
    }
    for (int i = 0; i < kStagesB; ++i) {
      mbar_init(&bar.b_full[i], 1);
      mbar_init(&bar.b_empty[i], 1);
    }
    mbar_init(&bar.s_full[0], 1);
    mbar_init(&bar.s_full[1], 1);
    mbar_init(&bar.dp_full, 1);
    mbar_init(&bar.p_ready, 8);
    mbar_init(&bar.ds_ready, 8);
    mbar_init(&bar.acc_full, 1);
    mbar_init(&bar.mma_done, 1);
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc(&tmem_slot, 512);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // keys' role: S at 0, dP at 128, dV at 256, dK at 384; queries' role: S at 0 and 128, dP at 256, dQ at 384
  const uint32_t tDP = tmem + (kv ? 128 : 256), tAcc0 = tmem + 256, tAcc1 = tmem + 384;

  if (warp >= kProducer) {
    regs_dec<72>();
    if (warp == kProducer) {
      bool ok = true;
      FillTrack fr, fa, fb;
      if (steps > 0) {
        fr.fill(0, 0);
        mbar_expect_tx_warp(&bar.res_full, 2 * kTileBytes);
        load_tile(res0, kv ? &maps.k : &maps.q, &bar.res_full, own0, kv ? hk : hq, b, kBoxes);
        load_tile(res1, kv ? &maps.v : &maps.dout, &bar.res_full, own0, kv ? hk : hq, b, kBoxes);
      }
      int t = t0, h = kv ? hq : hk;
      for (int n = 0; n < steps; ++n) {
        const int sa = slot_a(n), sb = slot_b(n);
        if (ok && n >= na) ok = bar_wait(&bar.a_empty[sa], phase_a(n) ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        if (ok) {
          fa.fill(sa, phase_a(n));
          mbar_expect_tx_warp(&bar.a_full[sa], kTileBytes + (kv ? 2 * kTile * 4 : 0));
          load_tile(ra + sa * kTileBytes, kv ? &maps.q : &maps.k, &bar.a_full[sa], t * kTile, h, b, kBoxes);
          if (kv) {
            const long long r = ((long long)b * a.Hq + h) * p.t_pad + t * kTile;
            bulk_load(rows + sa * 2 * kTile, p.lse2 + r, kTile * 4, &bar.a_full[sa]);
            bulk_load(rows + sa * 2 * kTile + kTile, p.delta + r, kTile * 4, &bar.a_full[sa]);
          }
        }
        if (ok && n >= kStagesB) ok = bar_wait(&bar.b_empty[sb], phase_b(n) ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        if (ok) {
          fb.fill(sb, phase_b(n));
          mbar_expect_tx_warp(&bar.b_full[sb], kTileBytes);
          load_tile(rb + sb * kTileBytes, kv ? &maps.dout : &maps.v, &bar.b_full[sb], t * kTile, h, b, kBoxes);
        }
        if (++t == t1) {
          t = t0;
          ++h;
        }
      }
      fr.drain(&bar.res_full, p.err, p.wait_ns);  // no copy of this CTA may land after it exits
      fa.drain(bar.a_full, p.err, p.wait_ns);
      fb.drain(bar.b_full, p.err, p.wait_ns);
    } else if (warp == kMma) {
      const uint32_t id_s = make_idesc(128, 128, 0, 0, kBf16);
      const uint32_t id_o = make_idesc(128, (a.D + 15) / 16 * 16, 0, 1, kBf16);
      const int ksteps = (a.D + 15) / 16;
      const uint64_t dr0 = desc_k(res0), dr1 = desc_k(res1);
      bool ok = steps > 0 ? bar_wait(&bar.res_full, 0, p.err, ERR_WAIT_FULL, p.wait_ns) : true;
      // rows of step n's tiles beyond the item's length
      auto valid = [&](int n) { return (kv ? it.ql : it.kl) - (t0 + n % per_head) * kTile; };
      auto wait_a = [&](int n) {
        const int st = slot_a(n);
        if (ok) ok = bar_wait(&bar.a_full[st], phase_a(n), p.err, ERR_WAIT_FULL, p.wait_ns);
        if (ok && valid(n) < kTile) zero_rows(ra + st * kTileBytes, max(valid(n), 0), kBoxes);
      };
      auto wait_b = [&](int n) {
        const int st = slot_b(n);
        if (ok) ok = bar_wait(&bar.b_full[st], phase_b(n), p.err, ERR_WAIT_FULL, p.wait_ns);
        if (ok && valid(n) < kTile) zero_rows(rb + st * kTileBytes, max(valid(n), 0), kBoxes);
      };
      auto issue_s = [&](int n) {
        wait_a(n);
        const int buf = kv ? 0 : n & 1;
        if (ok) {
          mma_values<DP>(tmem + 128 * buf, dr0, desc_k(ra + slot_a(n) * kTileBytes), id_s, ksteps);
          umma_commit_warp(&bar.s_full[buf]);
        }
      };
      auto issue_dp = [&](int n) {
        wait_b(n);
        if (ok) {
          mma_values<DP>(tDP, dr1, desc_k(rb + slot_b(n) * kTileBytes), id_s, ksteps);
          umma_commit_warp(&bar.dp_full);
          if (!kv) umma_commit_warp(&bar.b_empty[slot_b(n)]);  // nothing else reads V
        }
      };
      // acc += (A in tensor memory, 128 x 128, its halves 64 columns apart) x tile
      auto issue_acc = [&](uint32_t acc, uint32_t src, const uint8_t* tile_, int n) {
        const uint64_t d = desc_mn(tile_);
        mma4_ts(acc, src, d, id_o, n > 0);
        mma4_ts(acc, src + 64, d + (4 * 2048u >> 4), id_o, 1);
      };
      if (steps > 0) {
        issue_s(0);
        issue_dp(0);
        if (!kv && steps > 1) issue_s(1);
      }
      for (int n = 0; n < steps; ++n) {
        const uint32_t ph = n & 1;
        if (kv) {
          if (ok) ok = bar_wait(&bar.p_ready, ph, p.err, ERR_WAIT_ACC, p.wait_ns);
          tc_fence_after();
          if (ok) issue_acc(tAcc0, tmem, rb + slot_b(n) * kTileBytes, n);
          if (n + 1 < steps) issue_s(n + 1);
        }
        if (ok) ok = bar_wait(&bar.ds_ready, ph, p.err, ERR_WAIT_ACC, p.wait_ns);
        tc_fence_after();
        if (ok) {
          issue_acc(tAcc1, tDP, ra + slot_a(n) * kTileBytes, n);
          umma_commit_warp(&bar.a_empty[slot_a(n)]);
          if (kv) umma_commit_warp(&bar.b_empty[slot_b(n)]);
        }
        if (n + 1 < steps) issue_dp(n + 1);
        if (!kv && n + 2 < steps) issue_s(n + 2);
      }
      if (ok) umma_commit_warp(&bar.acc_full);
      // every MMA this warp issued has completed before TMEM is released (also after a timed-out wait)
      umma_commit_warp(&bar.mma_done);
      bar_wait(&bar.mma_done, 0, p.err, ERR_WAIT_ACC, p.wait_ns);
    }
  } else {
    regs_inc<216>();
    const int half = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int row = own0 + (warp & 3) * 32 + lane;  // a key or a query
    const float c = a.scale * kLog2e;
    const float f = ds_scale<T>(p, b, hk) * exp2f(-kShift);  // on P 2^shift (dP - D)
    const int lo = kv ? it.query_lo(a, row) : it.key_lo(a, row), hi = kv ? it.query_hi(a, row) : it.key_hi(a, row);
    // tiles that all of this tile's live rows meet whole need no mask
    const int last = min(own0 + kTile, kv ? it.kl : it.ql) - 1;
    const int all_lo = last >= own0 ? (kv ? it.query_lo(a, last) : it.key_lo(a, last)) : 0;
    const int all_hi = kv ? it.query_hi(a, own0) : it.key_hi(a, own0);
    float l2 = 0.f, delta = 0.f;
    if (!kv && steps > 0) {
      const long long r = ((long long)b * a.Hq + hq) * p.t_pad + row;
      l2 = p.lse2[r];
      delta = p.delta[r];
    }
    const uint32_t DPc = tDP + lanes + 64 * half;
    bool ok = true;
    for (int n = 0; n < steps; ++n) {
      const int st = slot_a(n), col0 = (t0 + n % per_head) * kTile + 64 * half;
      const uint32_t S = tmem + (kv ? 0 : 128 * (n & 1)) + lanes + 64 * half;
      if (kv && ok) ok = bar_wait(&bar.a_full[st], phase_a(n), p.err, ERR_WAIT_FULL, p.wait_ns);
      if (ok)
        ok = kv ? bar_wait(&bar.s_full[0], n & 1, p.err, ERR_WAIT_ACC, p.wait_ns)
                : bar_wait(&bar.s_full[n & 1], (n >> 1) & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
      if (!ok) continue;
      tc_fence_after();
      float x[64];
      tmem_load<64>(S, x);
      if (kv) {
        const float4* ls = reinterpret_cast<const float4*>(rows + st * 2 * kTile + 64 * half);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float4 v = ls[k];
          x[4 * k] = ex2(fmaf(x[4 * k], c, kShift - v.x));
          x[4 * k + 1] = ex2(fmaf(x[4 * k + 1], c, kShift - v.y));
          x[4 * k + 2] = ex2(fmaf(x[4 * k + 2], c, kShift - v.z));
          x[4 * k + 3] = ex2(fmaf(x[4 * k + 3], c, kShift - v.w));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 64; ++k) x[k] = ex2(fmaf(x[k], c, kShift - l2));
      }
      if (col0 - 64 * half < all_lo || col0 - 64 * half + kTile > all_hi) {
        const int r0 = lo - col0, r1 = hi - col0;
#pragma unroll
        for (int k = 0; k < 64; ++k) x[k] = k >= r0 && k < r1 ? x[k] : 0.f;
      }
      uint32_t w[32];
      if (kv) {
#pragma unroll
        for (int k = 0; k < 32; ++k) w[k] = pack2(x[2 * k], x[2 * k + 1], T());
        tmem_st32(S, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_ready);
      }
      ok = bar_wait(&bar.dp_full, n & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
      if (!ok) continue;
      tc_fence_after();
      float y[64];
      tmem_load<64>(DPc, y);
      const float4* ds = reinterpret_cast<const float4*>(rows + st * 2 * kTile + kTile + 64 * half);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float4 v = make_float4(delta, delta, delta, delta);
        if (kv) v = ds[k];
        float g[4] = {y[4 * k] - v.x, y[4 * k + 1] - v.y, y[4 * k + 2] - v.z, y[4 * k + 3] - v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] *= x[4 * k + e];
          if (!kBf16) g[e] *= f;
        }
        w[2 * k] = pack2(g[0], g[1], T());
        w[2 * k + 1] = pack2(g[2], g[3], T());
      }
      tmem_st32(DPc, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.ds_ready);
    }
    if (steps > 0 && ok) ok = bar_wait(&bar.acc_full, 0, p.err, ERR_WAIT_ACC, p.wait_ns);
    tc_fence_after();
    // the accumulators, half of the columns to each warpgroup
    const bool live = hi > lo && steps > 0 && ok;
    const float ds_out = a.scale / (kBf16 ? 1.f : f * exp2f(kShift));
    const float p_out = exp2f(-kShift);
#pragma unroll
    for (int g = 0; g < DP / 64; ++g) {
      const int d0 = half * (DP / 2) + 32 * g;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if (!kv && which == 0) continue;
        float o[32];
        if (steps > 0) tmem_load<32>((which ? tAcc1 : tAcc0) + lanes + d0, o);
        const float sc = which ? ds_out : p_out;
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = live ? o[k] * sc : 0.f;
        if (row >= (kv ? a.Tk : a.Tq)) continue;
        T* out = kv ? (which ? at<T>(a.dk, b, row, hk) : at<T>(a.dv, b, row, hk)) : at<T>(a.dq, b, row, hq);
#pragma unroll
        for (int k = 0; k < 32; k += 8)
          if (d0 + k < a.D) store8(out + d0 + k, o + k);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, 512);
}

template <typename T>
WB_DEV float dot8(const T* x, const T* y) {
  float u[8], v[8], s = 0.f;
  load8(x, u);
  load8(y, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) s += u[k] * v[k];
  return s;
}

// delta = rowsum(dO * O) and the log-sum-exp in units of log 2, padded to whole tiles with what gives
// probability 0; for fp16 also the largest squared norms of dO's and V's rows (an integer maximum over
// the bits of non-negative floats: its order does not matter).  16 threads a row.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int t = threadIdx.x & 15, i = blockIdx.x * 16 + threadIdx.x / 16, h = blockIdx.y, b = blockIdx.z;
  const AttnItem it(a, b);
  float d = 0.f, g = 0.f, v = 0.f;
  if (i < it.ql && t * 8 < a.D) {
    const T* x = at<T>(a.dout, b, i, h) + t * 8;
    d = dot8(x, at<T>(a.out, b, i, h) + t * 8);
    if (std::is_same<T, f16>::value) g = dot8(x, x);
  }
  const bool keys = std::is_same<T, f16>::value && h % p.group == 0;
  if (keys && i < it.kl && t * 8 < a.D) {
    const T* x = at<T>(a.v, b, i, h / p.group) + t * 8;
    v = dot8(x, x);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, m);
    if (std::is_same<T, f16>::value) {
      g += __shfl_xor_sync(0xffffffffu, g, m);
      v += __shfl_xor_sync(0xffffffffu, v, m);
    }
  }
  if (t == 0 && i < p.t_pad) {
    const long long r = ((long long)b * a.Hq + h) * p.t_pad + i;
    const float l = i < it.ql ? a.lse[((long long)b * a.Hq + h) * a.Tq + i] * kLog2e : INFINITY;
    p.delta[r] = d;
    p.lse2[r] = l == -INFINITY ? INFINITY : l;
  }
  if (std::is_same<T, f16>::value) {
    const int n = a.B * a.Hkv, at_ = b * a.Hkv + h / p.group;
    const uint32_t gm = __reduce_max_sync(0xffffffffu, __float_as_uint(g));
    const uint32_t vm = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if ((threadIdx.x & 31) == 0) {
      if (gm) atomicMax(p.norm_bits + at_, gm);
      if (vm) atomicMax(p.norm_bits + n + at_, vm);
    }
  }
}

template <typename T, int DP>
int launch_bwd(const AttnBwdMaps& maps, const AttnParams& p, cudaStream_t st) {
  const WubuB200Attn& a = p.a;
  constexpr int smem = (2 + kStagesA + kStagesB) * (DP / 64) * (int)kBox + 1024;
  static std::atomic<uint64_t> devices{0};
  if (!ops_smem_limit((const void*)attn_bwd_tc_kernel<T, DP>, smem, devices)) return WUBU_B200_ERR_CUDA;
  if (std::is_same<T, f16>::value &&
      cudaMemsetAsync(p.norm_bits, 0, 2ull * a.B * a.Hkv * sizeof(unsigned), st) != cudaSuccess)
    return WUBU_B200_ERR_CUDA;
  const int rows = std::is_same<T, f16>::value && a.Tk > p.t_pad ? a.Tk : p.t_pad;
  if (rows) attn_delta_kernel<T><<<dim3((rows + 15) / 16, a.Hq, a.B), 256, 0, st>>>(p);
  int rc = ops_launched("attn_backward rows");
  if (rc != WUBU_B200_OK) return rc;
  const long long kv = (long long)((a.Tk + kTile - 1) / kTile) * a.Hkv * a.B;
  const long long qs = (long long)((a.Tq + kTile - 1) / kTile) * a.Hq * a.B;
  if (kv + qs > 0x7FFFFFFFll) return WUBU_B200_ERR_SHAPE;
  attn_bwd_tc_kernel<T, DP><<<(unsigned)(kv + qs), kThreads, smem, st>>>(maps, p, (int)kv);
  return ops_launched("attn_backward");
}

}  // namespace

long long attn_bwd_bytes(const WubuB200Attn& a) {
  const long long t_pad = (a.Tq + kTile - 1) / kTile * kTile;
  return 2ll * a.B * a.Hq * t_pad * (long long)sizeof(float) + 2ll * a.B * a.Hkv * (long long)sizeof(unsigned);
}

int attn_backward(const AttnParams& in, cudaStream_t st) {
  AttnParams p = in;
  const WubuB200Attn& a = p.a;
  const long long rows = (long long)a.B * a.Hq * p.t_pad;
  p.delta = static_cast<float*>(a.workspace);
  p.lse2 = p.delta + rows;
  p.norm_bits = reinterpret_cast<unsigned*>(p.lse2 + rows);
  AttnBwdMaps maps{};
  if (a.Tq && (!attn_map(&maps.q, a.q, a.B, a.Tq, a.Hq, a.D) || !attn_map(&maps.dout, a.dout, a.B, a.Tq, a.Hq, a.D)))
    return WUBU_B200_ERR_CUDA;
  if (a.Tk && (!attn_map(&maps.k, a.k, a.B, a.Tk, a.Hkv, a.D) || !attn_map(&maps.v, a.v, a.B, a.Tk, a.Hkv, a.D)))
    return WUBU_B200_ERR_CUDA;
  if (a.dtype == WUBU_B200_BF16)
    return a.D <= 64 ? launch_bwd<bf16, 64>(maps, p, st) : launch_bwd<bf16, 128>(maps, p, st);
  return a.D <= 64 ? launch_bwd<f16, 64>(maps, p, st) : launch_bwd<f16, 128>(maps, p, st);
}

}  // namespace wb
