// attention_fwd.cu — softmax attention, forward, on the tensor cores.
//
// For a query row with scores s_j = scale q.k_j the output is sum_j e^(s_j - m) v_j / sum_j e^(s_j - m) for any
// m; keys arrive in tiles of 128 and m follows the running maximum.  The sums may keep an older m as
// long as e^(s - m) stays small: only when the maximum has moved by more than 2^8 are the accumulator
// and the sum scaled down (rarely after the first tiles), which keeps that pass over the accumulator
// out of the steady state.  P is rounded to the inputs' type for its product with V; the row sum is
// taken from the unrounded float32 values.
//
// A CTA owns two query tiles of 128 rows of one head (two streams).  Per stream the scores S (128 x 128
// fp32) and the output accumulator live in tensor memory; four warps read S, one row a thread, and
// write P back in two halves, from where the second product reads it as its A operand; a warp of its
// own issues the stream's products.  While the warps of one stream work on their exponentials, the
// tensor core runs the other stream's products.  K and V tiles arrive by TMA in rings and serve both.
// Up to 64 values a row, tensor memory has room for P beside S: the next scores are then issued as soon
// as S has been read and the streams never wait for a product.  At 128 values P lies over S.
#include <type_traits>

#include "attention.cuh"

namespace wb {
namespace {

// Eight softmax warps (a row of 128 scores in registers each thread), and a warpgroup of which one warp
// loads and one issues the products.  384 threads are launched with 168 registers; the split 256 x 216 +
// 128 x 72 is the same 64512.
constexpr int kProducer = 8, kMma = 9, kThreads = 384;  // kMma + s issues stream s

struct AttnFwdMaps {
  CUtensorMap q, k, v;
};

template <typename T>
struct FwdShift {  // P = 2^(x + value): fp16 runs out of small numbers, so its P is scaled up
  static constexpr float value = 0.f;
};
template <>
struct FwdShift<f16> {
  static constexpr float value = 6.f;
};

template <int DP>
constexpr int kFwdStages = DP == 64 ? 3 : 2;  // tiles in each of the two rings

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
attn_fwd_tc_kernel(const __grid_constant__ AttnFwdMaps maps, const __grid_constant__ AttnParams p) {
  constexpr int kBoxes = DP / 64;
  constexpr uint32_t kTileBytes = kBoxes * kBox;
  constexpr int kStages = kFwdStages<DP>;
  constexpr float kShift = FwdShift<T>::value;
  constexpr bool kApart = DP == 64;  // P has columns of its own
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qt = smem;
  uint8_t* kt = qt + 2 * kTileBytes;
  uint8_t* vt = kt + kStages * kTileBytes;
  // per stream: S complete; S read (kApart); the halves of P written; the product that read P done
  __shared__ uint64_t q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2],
      s_read[2], p_ready[2][2], pv_done[2], mma_done[2];
  __shared__ uint32_t tmem_slot;

  const WubuB200Attn& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int npairs = (a.Tq + 2 * kTile - 1) / (2 * kTile);
  // causal: the last pair has the most keys and goes first
  const int pair = npairs - 1 - (int)(blockIdx.x / p.splits), split = blockIdx.x % p.splits;
  const int h = blockIdx.y, b = blockIdx.z;
  const AttnItem it(a, b);
  // key tiles [t0, t1) of each stream, their union, and this CTA's part of it
  int q0[2], t0[2], t1[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    q0[s] = (2 * pair + s) * kTile;
    const int last = min(q0[s] + kTile, it.ql) - 1;
    const int lo = it.key_lo(a, q0[s]), hi = last >= q0[s] ? it.key_hi(a, last) : 0;
    t0[s] = hi > lo ? lo / kTile : 0;
    t1[s] = hi > lo ? (hi + kTile - 1) / kTile : 0;
  }
  int u0 = t1[0] > t0[0] ? (t1[1] > t0[1] ? min(t0[0], t0[1]) : t0[0]) : t0[1], u1 = max(t1[0], t1[1]);
  {
    const int n = max(0, u1 - u0);
    const int c0 = u0 + (int)((long long)n * split / p.splits), c1 = u0 + (int)((long long)n * (split + 1) / p.splits);
    u0 = c0;
    u1 = c1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      t0[s] = max(t0[s], u0);
      t1[s] = max(t0[s], min(t1[s], u1));
    }
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_read[i], 4);
      mbar_init(&p_ready[i][0], 4);
      mbar_init(&p_ready[i][1], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&mma_done[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {  // a tile is free once both streams are done with it
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc(&tmem_slot, 512);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // columns: S at 0 and 128; apart, P at 256 and 320 and O at 384 and 448; else P over S and O at 256 and 384
  auto col_p = [&](int s) { return tmem + (kApart ? 256 + 64 * s : 128 * s); };
  auto col_o = [&](int s) { return tmem + (kApart ? 384 + 64 * s : 256 + 128 * s); };

  if (warp >= kProducer) {
    regs_dec<72>();
    if (warp == kProducer) {
      bool ok = true;
      FillTrack fq, fk, fv;
      const int hk = h / p.group;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (t1[s] > t0[s]) {
          fq.fill(s, 0);
          mbar_expect_tx_warp(&q_full[s], kTileBytes);
          load_tile(qt + s * kTileBytes, &maps.q, &q_full[s], q0[s], h, b, kBoxes);
        }
      for (int j = u0; j < u1; ++j) {
        const int n = j - u0, st = n % kStages;
        const uint32_t ph = (n / kStages) & 1;
        if (ok && n >= kStages) ok = bar_wait(&k_empty[st], ph ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        if (ok) {
          fk.fill(st, ph);
          mbar_expect_tx_warp(&k_full[st], kTileBytes);
          load_tile(kt + st * kTileBytes, &maps.k, &k_full[st], j * kTile, hk, b, kBoxes);
        }
        if (ok && n >= kStages) ok = bar_wait(&v_empty[st], ph ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        if (ok) {
          fv.fill(st, ph);
          mbar_expect_tx_warp(&v_full[st], kTileBytes);
          load_tile(vt + st * kTileBytes, &maps.v, &v_full[st], j * kTile, hk, b, kBoxes);
        }
      }
      fq.drain(q_full, p.err, p.wait_ns);  // no copy of this CTA may land after it exits
      fk.drain(k_full, p.err, p.wait_ns);
      fv.drain(v_full, p.err, p.wait_ns);
    } else if (warp < kMma + 2) {
      const int s = warp - kMma;
      const int st0 = s ? t0[1] : t0[0], st1 = s ? t1[1] : t1[0];
      constexpr int kBf16 = std::is_same<T, bf16>::value;
      const uint32_t id_s = make_idesc(128, 128, 0, 0, kBf16);
      const uint32_t id_o = make_idesc(128, (a.D + 15) / 16 * 16, 0, 1, kBf16);
      const int ksteps = (a.D + 15) / 16;
      const uint64_t dq = desc_k(qt + s * kTileBytes);
      const uint32_t P = col_p(s), O = col_o(s), S = tmem + 128 * s;
      bool ok = true;
      uint32_t ph = 0;
      // the scores against key tile j, or a pass by a tile that the stream does not meet
      auto issue_s = [&](int j) {
        const int n = j - u0, sl = n % kStages;
        if (ok) ok = bar_wait(&k_full[sl], (n / kStages) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
        if (!ok) return;
        if (j < st0 || j >= st1) {
          if (lane == 0) mbar_arrive(&k_empty[sl]);
          return;
        }
        mma_values<DP>(S, dq, desc_k(kt + sl * kTileBytes), id_s, ksteps);
        umma_commit_warp(&s_full[s]);
        umma_commit_warp(&k_empty[sl]);
      };
      if (st1 > st0) ok = bar_wait(&q_full[s], 0, p.err, ERR_WAIT_FULL, p.wait_ns);
      if (u0 < u1) issue_s(u0);
      for (int j = u0; j < u1; ++j) {
        const int n = j - u0, sl = n % kStages;
        const bool mine = j >= st0 && j < st1;
        if (kApart) {
          if (mine && ok) ok = bar_wait(&s_read[s], ph, p.err, ERR_WAIT_ACC, p.wait_ns);
          tc_fence_after();
          if (j + 1 < u1) issue_s(j + 1);
        }
        if (ok) ok = bar_wait(&v_full[sl], (n / kStages) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
        if (mine) {
          uint8_t* tile = vt + sl * kTileBytes;
          const int valid = it.kl - j * kTile;  // both streams may clear the same rows
          if (ok && valid < kTile) zero_rows(tile, max(valid, 0), kBoxes);
          const uint64_t dv = desc_mn(tile);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (ok) ok = bar_wait(&p_ready[s][half], ph, p.err, ERR_WAIT_ACC, p.wait_ns);
            tc_fence_after();
            if (ok) mma4_ts(O, P + 32 * half, dv + half * (4 * 2048u >> 4), id_o, (j > st0) | half);
          }
          ph ^= 1u;
          if (ok) {
            umma_commit_warp(&pv_done[s]);
            umma_commit_warp(&v_empty[sl]);
          }
        } else if (ok && lane == 0) {
          mbar_arrive(&v_empty[sl]);
        }
        if (!kApart && j + 1 < u1) issue_s(j + 1);
      }
      // every MMA this warp issued has completed before TMEM is released (also after a timed-out wait)
      umma_commit_warp(&mma_done[s]);
      bar_wait(&mma_done[s], 0, p.err, ERR_WAIT_ACC, p.wait_ns);
    }
  } else {
    regs_inc<216>();
    const int s = warp >> 2;
    const int sq0 = s ? q0[1] : q0[0], st0 = s ? t0[1] : t0[0], st1 = s ? t1[1] : t1[0];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t S = tmem + 128 * s + lanes, O = col_o(s) + lanes, P = col_p(s) + lanes;
    const int i = sq0 + (warp & 3) * 32 + lane;
    const int lo = it.key_lo(a, i), hi = it.key_hi(a, i);
    // key tiles that every live row of the query tile sees whole need no mask
    const int tile_last = min(sq0 + kTile, it.ql) - 1;
    const int all_lo = tile_last >= sq0 ? it.key_lo(a, tile_last) : 0, all_hi = it.key_hi(a, sq0);
    const float c = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    uint32_t ph = 0;
    for (int j = st0; j < st1; ++j) {
      if (ok) ok = bar_wait(&s_full[s], ph, p.err, ERR_WAIT_ACC, p.wait_ns);
      if (!ok) continue;
      tc_fence_after();
      float x[128];
      tmem_load<128>(S, x);
      if (kApart) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_read[s]);
      }
      const int j0 = j * kTile;
      if (j0 < all_lo || j0 + kTile > all_hi) {
        const int r0 = lo - j0, r1 = hi - j0;
#pragma unroll
        for (int k = 0; k < 128; ++k) x[k] = k >= r0 && k < r1 ? x[k] : -INFINITY;
      }
      float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int k = 4; k < 124; k += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[k + e], x[k + 4 + e]);
      const float mt = max3(max3(mx[0], mx[1], x[124]), max3(mx[2], mx[3], x[125]), fmaxf(x[126], x[127]));
      // move m when the maximum has outgrown it by 2^8 (or was not set)
      const bool move = mt > m && (m == -INFINITY || (mt - m) * c > 8.f);
      const bool any_move = __any_sync(0xffffffffu, move);
      // apart, S may be ahead of the product that last read P and added to O; over S it cannot be
      if (kApart && j > st0) ok = bar_wait(&pv_done[s], ph ^ 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
      ph ^= 1u;
      if (!ok) continue;
      if (any_move) {
        const float f = !move ? 1.f : m == -INFINITY ? 0.f : ex2((m - mt) * c);
        if (move) m = mt;
        l *= f;
        if (j > st0) {
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < DP / 32; ++g) {
            float o[32];
            tmem_load<32>(O + 32 * g, o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= f;
            tmem_st32(O + 32 * g, reinterpret_cast<const uint32_t*>(o));
          }
        }
      }
      const float mc = (m == -INFINITY ? 0.f : m * c) - kShift;
      const uint64_t cc = two(c, c), mm = two(-mc, -mc);
      uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float* y = x + 64 * g;
        uint32_t w[32];
#pragma unroll
        for (int k = 0; k < 64; k += 2) each(fma2(two(y[k], y[k + 1]), cc, mm), y[k], y[k + 1]);
#pragma unroll
        for (int k = 0; k < 64; ++k) y[k] = ex2(y[k]);
#pragma unroll
        for (int k = 0; k < 64; k += 2) sum[k / 2 & 3] = add2(sum[k / 2 & 3], two(y[k], y[k + 1]));
#pragma unroll
        for (int k = 0; k < 32; ++k) w[k] = pack2(y[2 * k], y[2 * k + 1], T());
        tmem_st32(P + 32 * g, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[s][g]);
      }
      float l0, l1;
      each(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
      l += l0 + l1;
    }
    // the last product: its phase is that of the number of tiles before it
    if (st1 > st0 && ok) ok = bar_wait(&pv_done[s], ph ^ 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
    tc_fence_after();
    const bool live = l > 0.f && hi > lo && st1 > st0 && ok;
    const bool bad = hi > lo && st1 > st0 && !(l == l);  // a NaN among the scores stays visible
    const float inv = live ? 1.f / l : 0.f;
    const float lse = live ? m * a.scale + (logf(l) - kShift * 0.69314718055994531f) : bad ? l : -INFINITY;
    const long long row = ((long long)b * a.Hq + h) * a.Tq + i;
    if (i < a.Tq) (p.splits > 1 ? p.part_lse + (long long)split * a.B * a.Hq * a.Tq : a.lse)[row] = lse;
#pragma unroll
    for (int g = 0; g < DP / 32; ++g) {
      float o[32];
      if (st1 > st0) tmem_load<32>(O + 32 * g, o);
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = live ? o[k] * inv : bad ? l : 0.f;
      if (i >= a.Tq) continue;
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        if (32 * g + k >= a.D) continue;
        if (p.splits > 1)
          store8(p.part + ((long long)split * a.B * a.Hq * a.Tq + row) * a.D + 32 * g + k, o + k);
        else
          store8(at<T>(a.out, b, i, h) + 32 * g + k, o + k);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, 512);
}

// Joins the parts of a query's keys: out = sum_s w_s out_s with w_s = e^(lse_s - lse).  A warp per row.
template <typename T>
__global__ void __launch_bounds__(128) attn_fwd_join_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.B * a.Hq * a.Tq, row = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_lse[s * rows + row]);
  const float base = m == -INFINITY ? 0.f : m;
  float total = 0.f, o[4] = {};
  const bool on = lane * 4 < a.D;
  for (int s = 0; s < p.splits; ++s) {
    const float w = expf(p.part_lse[s * rows + row] - base);
    total += w;
    if (!on || w == 0.f) continue;
    const float4 v = *reinterpret_cast<const float4*>(p.part + (s * rows + row) * a.D + lane * 4);
    o[0] += w * v.x;
    o[1] += w * v.y;
    o[2] += w * v.z;
    o[3] += w * v.w;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane == 0) a.lse[row] = total == 0.f ? -INFINITY : base + logf(total);
  const int i = (int)(row % a.Tq), h = (int)(row / a.Tq % a.Hq), b = (int)(row / a.Tq / a.Hq);
  if (on)
    *reinterpret_cast<uint2*>(at<T>(a.out, b, i, h) + lane * 4) =
        make_uint2(pack2(o[0] * inv, o[1] * inv, T()), pack2(o[2] * inv, o[3] * inv, T()));
}

template <typename T, int DP>
int launch_fwd(const AttnFwdMaps& maps, const AttnParams& p, cudaStream_t st) {
  const WubuB200Attn& a = p.a;
  constexpr int smem = (2 + 2 * kFwdStages<DP>) * (DP / 64) * (int)kBox + 1024;
  static std::atomic<uint64_t> devices{0};
  if (!ops_smem_limit((const void*)attn_fwd_tc_kernel<T, DP>, smem, devices)) return WUBU_B200_ERR_CUDA;
  const int npairs = (a.Tq + 2 * kTile - 1) / (2 * kTile);
  attn_fwd_tc_kernel<T, DP><<<dim3(npairs * p.splits, a.Hq, a.B), kThreads, smem, st>>>(maps, p);
  int rc = ops_launched("attn_forward");
  if (rc != WUBU_B200_OK || p.splits == 1) return rc;
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  attn_fwd_join_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(p);
  return ops_launched("attn_forward join");
}

}  // namespace

// Few query rows and many keys: the keys of a row are split over CTAs, as many as fill the SMs once.
int attn_fwd_splits(const WubuB200Attn& a) {
  const long long ctas = (long long)((a.Tq + 2 * kTile - 1) / (2 * kTile)) * a.Hq * a.B;
  const int tiles = (a.Tk + kTile - 1) / kTile;
  if (ctas == 0 || tiles < 2 || ctas > 74) return 1;
  const long long s = 148 / ctas;
  return (int)(s < tiles ? s : tiles);
}
long long attn_fwd_bytes(const WubuB200Attn& a) {
  const int s = attn_fwd_splits(a);
  return s == 1 ? 0 : (long long)s * a.B * a.Hq * a.Tq * (a.D + 4) * (long long)sizeof(float);
}

int attn_forward(const AttnParams& in, cudaStream_t st) {
  AttnParams p = in;
  const WubuB200Attn& a = p.a;
  p.splits = attn_fwd_splits(a);
  p.part = static_cast<float*>(a.workspace);
  p.part_lse = p.part + (long long)p.splits * a.B * a.Hq * a.Tq * a.D;
  AttnFwdMaps maps{};
  if (!attn_map(&maps.q, a.q, a.B, a.Tq, a.Hq, a.D)) return WUBU_B200_ERR_CUDA;
  if (a.Tk && (!attn_map(&maps.k, a.k, a.B, a.Tk, a.Hkv, a.D) || !attn_map(&maps.v, a.v, a.B, a.Tk, a.Hkv, a.D)))
    return WUBU_B200_ERR_CUDA;
  if (a.dtype == WUBU_B200_BF16)
    return a.D <= 64 ? launch_fwd<bf16, 64>(maps, p, st) : launch_fwd<bf16, 128>(maps, p, st);
  return a.D <= 64 ? launch_fwd<f16, 64>(maps, p, st) : launch_fwd<f16, 128>(maps, p, st);
}

}  // namespace wb
