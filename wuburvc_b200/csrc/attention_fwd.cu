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
// Measured (B200): 16 heads on 4, 6000 tokens causal, 128 values: 159 us with its inputs in L2, 930
// TFLOP/s of visible work, 170 without (floor 91 us at the measured product rate); 4 x 16 heads, 2048 x 64: 117 us; 16 x up to 499, 12 heads of 64:
// 31 us (floor 4.9): items of four steps, whose filling and draining nothing overlaps.
// Up to 64 values a row, tensor memory has room for P beside S: the next scores are then issued as soon
// as S has been read and the streams never wait for a product.  At 128 values P lies over S.
#include <type_traits>

#include "attention.cuh"

namespace wb {
namespace {

// Eight softmax warps (a row of 128 scores in registers each thread), and a warpgroup of which one warp
// loads and two issue the products.  384 threads are launched with 168 registers; the split 256 x 216 +
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

// A work item: a pair of query tiles of one head, and a part of their keys.
struct FwdWork {
  AttnItem it;
  int b, h, split;
  int q0[2], t0[2], t1[2];  // per stream: first query, key tiles [t0, t1)
  int u0, u1;               // the tiles that either stream meets
  bool none;                // no item: the work is done
  FwdWork() = default;
  WB_DEV FwdWork(const AttnParams& p, int id) {
    const WubuB200Attn& a = p.a;
    none = false;
    const unsigned t = (unsigned)id / (unsigned)a.Hq;
    h = id - t * a.Hq;
    unsigned r = t / (unsigned)a.B;
    b = t - r * a.B;
    it = AttnItem(a, b);
    split = 0;
    if (p.splits > 1) {
      split = r % (unsigned)p.splits;
      r /= (unsigned)p.splits;
    }
    const int pair = (a.Tq + 2 * kTile - 1) / (2 * kTile) - 1 - (int)r;  // causal: the last has the most keys and goes first
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      q0[s] = (2 * pair + s) * kTile;
      const int last = min(q0[s] + kTile, it.ql) - 1;
      const int lo = it.key_lo(a, q0[s]), hi = last >= q0[s] ? it.key_hi(a, last) : 0;
      t0[s] = hi > lo ? lo / kTile : 0;
      t1[s] = hi > lo ? (hi + kTile - 1) / kTile : 0;
    }
    u0 = t1[0] > t0[0] ? (t1[1] > t0[1] ? min(t0[0], t0[1]) : t0[0]) : t0[1];
    u1 = max(t1[0], t1[1]);
    if (p.splits > 1) {
      const int n = max(0, u1 - u0), first = u0;
      u0 = first + n * split / p.splits;
      u1 = first + n * (split + 1) / p.splits;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        t0[s] = max(t0[s], u0);
        t1[s] = max(t0[s], min(t1[s], u1));
      }
    }
  }
};

template <int DP>
constexpr int kFwdStages = DP == 64 ? 3 : 2;  // tiles in each of the two rings

// SPLIT: the keys of a row are split over work items, whose results go to the workspace.
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
attn_fwd_tc_kernel(const __grid_constant__ AttnFwdMaps maps, const __grid_constant__ AttnParams p) {
  constexpr int kBoxes = DP / 64;
  constexpr uint32_t kTileBytes = kBoxes * kBox;
  constexpr int kStages = kFwdStages<DP>;
  constexpr float kShift = FwdShift<T>::value;
  constexpr bool kApart = DP == 64;  // P has columns of its own
  // Of 32 exponentials, so many on the FMA units.  Up to 64 values a row the function unit is what the warps
  // wait for (4 x 16 heads, 4096 tokens of 64: 391 us with 8, 417 with 0); at 128 values a step is bound
  // by its chain of products, and the additional instructions only lengthen it (203 us against 188).
  constexpr int kPoly = DP == 64 ? 8 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qt = smem;
  uint8_t* kt = qt + 2 * kTileBytes;
  uint8_t* vt = kt + kStages * kTileBytes;
  uint8_t* stage = vt + kStages * kTileBytes;  // 2 KB a softmax warp
  // per stream: S complete; S read (kApart); the halves of P written; the product that read P done
  __shared__ FwdWork items[2];  // worked out by the loading warp (about a thousand cycles), behind the last item
  __shared__ uint64_t item_full[2], item_empty[2], q_full[2], q_empty[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2],
      s_read[2], p_ready[2][2], pv_done[2], turn[2], mma_done[2];
  __shared__ uint32_t tmem_slot;

  const WubuB200Attn& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int work = (a.Tq + 2 * kTile - 1) / (2 * kTile) * p.splits * a.Hq * a.B;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kProducer + 2);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_read[i], 4);
      mbar_init(&p_ready[i][0], 4);
      mbar_init(&p_ready[i][1], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&turn[i], 4);
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
  // item n's slot: false at the end of the work
  auto take = [&](int n) {
    return bar_wait(&item_full[n & 1], (n >> 1) & 1, p.err, ERR_WAIT_FULL, p.wait_ns) && !items[n & 1].none;
  };
  auto done = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[n & 1]);
  };
  // columns: S at 0 and 128; apart, P at 256 and 320 and O at 384 and 448; else P over S and O at 256 and 384
  auto col_p = [&](int s) { return tmem + (kApart ? 256 + 64 * s : 128 * s); };
  auto col_o = [&](int s) { return tmem + (kApart ? 384 + 64 * s : 256 + 128 * s); };

  if (warp >= kProducer) {
    regs_dec<72>();
    if (warp == kProducer) {
      bool ok = true;
      FillTrack fq, fk, fv;
      int n = 0, nq[2] = {0, 0};  // tiles loaded so far
      int count = 0;
      for (AttnRounds r(work);; r.advance(), ++count) {
        if (ok && count >= 2) ok = bar_wait(&item_empty[count & 1], ((count >> 1) & 1) ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        const bool none = !ok || !r.more();
        FwdWork k(p, none ? 0 : r.next);
        k.none = none;
        if (lane == 0) {
          items[count & 1] = k;
          mbar_arrive(&item_full[count & 1]);
        }
        __syncwarp();
        if (none) break;
        const int hk = k.h / p.group;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (k.t1[s] <= k.t0[s]) continue;
          if (ok && nq[s]) ok = bar_wait(&q_empty[s], (nq[s] - 1) & 1, p.err, ERR_WAIT_EMPTY, p.wait_ns);
          if (ok) {
            fq.fill(s, nq[s]);
            mbar_expect_tx_warp(&q_full[s], kTileBytes);
            load_tile(qt + s * kTileBytes, &maps.q, &q_full[s], k.q0[s], k.h, k.b, kBoxes);
          }
          ++nq[s];
        }
        for (int j = k.u0; j < k.u1; ++j, ++n) {
          const int st = n % kStages;
          const uint32_t ph = (n / kStages) & 1;
          if (ok && n >= kStages) ok = bar_wait(&k_empty[st], ph ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
          if (ok) {
            fk.fill(st, ph);
            mbar_expect_tx_warp(&k_full[st], kTileBytes);
            load_tile(kt + st * kTileBytes, &maps.k, &k_full[st], j * kTile, hk, k.b, kBoxes);
          }
          if (ok && n >= kStages) ok = bar_wait(&v_empty[st], ph ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
          if (ok) {
            fv.fill(st, ph);
            mbar_expect_tx_warp(&v_full[st], kTileBytes);
            load_tile(vt + st * kTileBytes, &maps.v, &v_full[st], j * kTile, hk, k.b, kBoxes);
          }
        }
      }
      fq.drain(q_full, p.err, p.wait_ns);  // no copy of this CTA may land after it exits
      fk.drain(k_full, p.err, p.wait_ns);
      fv.drain(v_full, p.err, p.wait_ns);
    } else if (warp < kMma + 2) {
      const int s = warp - kMma;
      constexpr int kBf16 = std::is_same<T, bf16>::value;
      const uint32_t id_s = make_idesc(128, 128, 0, 0, kBf16);
      const uint32_t id_o = make_idesc(128, (a.D + 15) / 16 * 16, 0, 1, kBf16);
      const int ksteps = (a.D + 15) / 16;
      const uint64_t dq = desc_k(qt + s * kTileBytes);
      const uint32_t P = col_p(s), O = col_o(s), S = tmem + 128 * s;
      bool ok = true;
      uint32_t ph = 0;     // of the stream's tiles
      int n0 = 0, nq = 0;  // tiles in the rings before this item; the stream's query tiles
      for (int count = 0; take(count); ++count) {
        const FwdWork k = items[count & 1];
        done(count);
        const int st0 = s ? k.t0[1] : k.t0[0], st1 = s ? k.t1[1] : k.t1[0], u0 = k.u0, u1 = k.u1;
        // the scores against key tile j, or a pass by a tile that the stream does not meet
        auto issue_s = [&](int j) {
          const int n = n0 + j - u0, sl = n % kStages;
          if (ok) ok = bar_wait(&k_full[sl], (n / kStages) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
          if (!ok) return;
          if (j < st0 || j >= st1) {
            if (lane == 0) mbar_arrive(&k_empty[sl]);
            return;
          }
          mma_values<DP>(S, dq, desc_k(kt + sl * kTileBytes), id_s, ksteps);
          umma_commit_warp(&s_full[s]);
          umma_commit_warp(&k_empty[sl]);
          if (j == st1 - 1) umma_commit_warp(&q_empty[s]);
        };
        if (st1 > st0) {
          if (ok) ok = bar_wait(&q_full[s], nq & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
          ++nq;
        }
        if (u0 < u1) issue_s(u0);
        for (int j = u0; j < u1; ++j) {
          const int n = n0 + j - u0, sl = n % kStages;
          const bool mine = j >= st0 && j < st1;
          if (kApart) {
            if (mine && ok) ok = bar_wait(&s_read[s], ph, p.err, ERR_WAIT_ACC, p.wait_ns);
            tc_fence_after();
            if (j + 1 < u1) issue_s(j + 1);
          }
          if (ok) ok = bar_wait(&v_full[sl], (n / kStages) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
          if (mine) {
            uint8_t* tile = vt + sl * kTileBytes;
            const int valid = k.it.kl - j * kTile;  // both streams may clear the same rows
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
        n0 += max(0, u1 - u0);
      }
      // every MMA this warp issued has completed before TMEM is released (also after a timed-out wait)
      umma_commit_warp(&mma_done[s]);
      bar_wait(&mma_done[s], 0, p.err, ERR_WAIT_ACC, p.wait_ns);
    }
  } else {
    regs_inc<216>();
    const int s = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t S = tmem + 128 * s + lanes, O = col_o(s) + lanes, P = col_p(s) + lanes;
    const float c = a.scale * 1.4426950408889634f;
    bool ok = true;
    uint32_t ph = 0;
    // P over S (128 values): the streams take turns with their exponentials, so that one's products run beside the
    // other's exponentials instead of both waiting for the tensor core at once (3840 tokens, 16 heads:
    // 140 us against 164; with P apart it only costs).  Stream 1's turn g follows stream 0's, whose turn
    // g + 1 follows it; a stream passes its turn on half way.  The streams' tile counts differ by one at
    // most where both have tiles, and the shorter then takes an empty turn.
    uint32_t g_turn = 0;
    auto wait_turn = [&] {
      if (s == 1 && ok) ok = bar_wait(&turn[0], g_turn & 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
      if (s == 0 && ok && g_turn) ok = bar_wait(&turn[1], (g_turn - 1) & 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
      ++g_turn;
    };
    for (int count = 0; take(count); ++count) {
      const FwdWork& next = items[count & 1];
      const int n_s0 = next.t1[0] - next.t0[0], n_s1 = next.t1[1] - next.t0[1];
      const bool turns = !kApart && n_s0 > 0 && n_s1 > 0;
      const bool empty_turn = turns && (s ? n_s1 < n_s0 : n_s0 < n_s1);
      const AttnItem it = next.it;
      const int h = next.h, b = next.b, split = next.split;
      const int sq0 = s ? next.q0[1] : next.q0[0], st0 = s ? next.t0[1] : next.t0[0], st1 = s ? next.t1[1] : next.t1[0];
      const int i = sq0 + (warp & 3) * 32 + lane;
      const int lo = it.key_lo(a, i), hi = it.key_hi(a, i);
      // key tiles that every live row of the query tile sees whole need no mask
      const int tile_last = min(sq0 + kTile, it.ql) - 1;
      const int all_lo = tile_last >= sq0 ? it.key_lo(a, tile_last) : 0, all_hi = it.key_hi(a, sq0);
      float m = -INFINITY, l = 0.f;
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
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t see = see_bits(lo - j0 - 32 * g, hi - j0 - 32 * g);
#pragma unroll
            for (int k = 0; k < 32; ++k) x[32 * g + k] = see >> k & 1 ? x[32 * g + k] : -INFINITY;
          }
        }
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int k = 4; k < 124; k += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[k + e], x[k + 4 + e]);
        const float mt = max3(max3(mx[0], mx[1], x[124]), max3(mx[2], mx[3], x[125]), max3(x[126], x[127], x[127]));
        // Move m when the maximum has outgrown it by 2^8 (or was not set), and where a score is NaN: the row's m is
        // NaN from there on, and with it all that follows.  An infinite maximum makes it NaN too (infinity less
        // itself is), as it does in the formula.
        const bool move = !(mt <= m) && (m == -INFINITY || !((mt - m) * c <= 8.f));
        const bool any_move = __any_sync(0xffffffffu, move);
        // apart, S may be ahead of the product that last read P and added to O; over S it cannot be
        if (kApart && j > st0) ok = bar_wait(&pv_done[s], ph ^ 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
        ph ^= 1u;
        if (!ok) continue;
        if (any_move) {
          const float f = !move ? 1.f : m == -INFINITY ? 0.f : ex2((m - mt) * c);
          if (move) m = mt + (mt - mt);
          l *= f;
          if (j > st0) {
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < DP / 16; ++g) {  // (few registers beside the scores)
              float o[16];
              tmem_load16(O + 16 * g, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] *= f;
              tmem_st16(O + 16 * g, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        if (turns) wait_turn();
        if (!ok) continue;
        const float mc = (m == -INFINITY ? 0.f : m * c) - kShift;
        const uint64_t cc = two(c, c), mm = two(-mc, -mc);
        uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float* y = x + 64 * g + 32 * q;
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) each(fma2(two(y[k], y[k + 1]), cc, mm), y[k], y[k + 1]);
#pragma unroll
            for (int k = 0; k < 32 - kPoly; ++k) y[k] = ex2(y[k]);
#pragma unroll
            for (int k = 32 - kPoly; k < 32; k += 2) each(ex2_poly2(two(y[k], y[k + 1])), y[k], y[k + 1]);
#pragma unroll
            for (int k = 0; k < 32; k += 2) sum[k / 2 & 3] = add2(sum[k / 2 & 3], two(y[k], y[k + 1]));
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = pack2(y[2 * k], y[2 * k + 1], T());
            tmem_st16(P + 32 * g + 16 * q, w);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&p_ready[s][g]);
            if (turns && g == 0) mbar_arrive(&turn[s]);
          }
        }
        float l0, l1;
        each(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
        l += l0 + l1;
      }
      if (empty_turn) {
        wait_turn();
        if (ok && lane == 0) mbar_arrive(&turn[s]);
      }
      // the last product: its phase is that of the number of tiles before it
      if (st1 > st0 && ok) ok = bar_wait(&pv_done[s], ph ^ 1u, p.err, ERR_WAIT_ACC, p.wait_ns);
      tc_fence_after();
      // (without a score above -infinity m is not set, and l holds what the polynomial's 2^-125 add up to)
      const bool live = l > 0.f && m > -INFINITY && hi > lo && st1 > st0 && ok;
      const bool bad = hi > lo && st1 > st0 && !(l == l);  // a NaN among the scores stays visible
      const float inv = live ? 1.f / l : 0.f;
      const float lse = live ? m * a.scale + (logf(l) - kShift * 0.69314718055994531f) : bad ? l : -INFINITY;
      const long long row = ((long long)b * a.Hq + h) * a.Tq + i;
      if (i < a.Tq) (SPLIT ? p.part_lse + (long long)split * a.B * a.Hq * a.Tq : a.lse)[row] = lse;
      auto values = [&](int d0, float* o) {  // 32 of the row's results
        if (st1 > st0) tmem_load<32>(O + d0, o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = live ? o[k] * inv : bad ? l : 0.f;
      };
      if (SPLIT) {
        float* part = p.part + ((long long)split * a.B * a.Hq * a.Tq + row) * a.D;
#pragma unroll
        for (int d0 = 0; d0 < DP; d0 += 32) {
          float o[32];
          values(d0, o);
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (i < a.Tq && d0 + k < a.D) store8(part + d0 + k, o + k);
          __syncwarp();
        }
      } else {
        const int r0 = sq0 + (warp & 3) * 32;
        T* out = at<T>(a.out, b, r0, h);
#pragma unroll
        for (int d0 = 0; d0 < DP; d0 += 32) {
          float o[32];
          values(d0, o);
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) w[k] = pack2(o[2 * k], o[2 * k + 1], T());
          store_rows<4>(stage + warp * 2048, w, out + d0, a.out.token, a.Tq - r0, a.D - d0);
        }
      }
      done(count);
      tc_fence_before();  // O is read before the next item's first product may be issued
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kMma) tmem_dealloc(tmem, 512);
}

// Joins the parts of a query's keys: out = sum_s w_s out_s with w_s = e^(lse_s - lse).  A warp per row; lane s
// holds part s's weight (at most 32 parts).
constexpr int kMaxSplits = 32;
template <typename T>
__global__ void __launch_bounds__(128) attn_fwd_join_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.B * a.Hq * a.Tq, row = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  griddep_wait();
  if (row >= rows) return;
  const float lse = lane < p.splits ? p.part_lse[lane * rows + row] : -INFINITY;
  float m = lse;
#pragma unroll
  for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  const float base = m == -INFINITY ? 0.f : m, w = expf(lse - base);
  float total = w;
#pragma unroll
  for (int k = 16; k; k >>= 1) total += __shfl_xor_sync(0xffffffffu, total, k);
  const bool on = lane * 4 < a.D;
  const float* part = p.part + row * a.D + (on ? lane * 4 : 0);
  float o[4] = {};
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s);
    const float4 v = *reinterpret_cast<const float4*>(part + s * rows * a.D);
    o[0] += ws * v.x;
    o[1] += ws * v.y;
    o[2] += ws * v.z;
    o[3] += ws * v.w;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane == 0) a.lse[row] = total == 0.f ? -INFINITY : base + logf(total);
  const int i = (int)(row % a.Tq), h = (int)(row / a.Tq % a.Hq), b = (int)(row / a.Tq / a.Hq);
  if (on)
    *reinterpret_cast<uint2*>(at<T>(a.out, b, i, h) + lane * 4) =
        make_uint2(pack2(o[0] * inv, o[1] * inv, T()), pack2(o[2] * inv, o[3] * inv, T()));
}

template <typename T, int DP, bool SPLIT>
int launch_fwd(const AttnFwdMaps& maps, const AttnParams& p, cudaStream_t st) {
  const WubuB200Attn& a = p.a;
  constexpr int smem = (2 + 2 * kFwdStages<DP>) * (DP / 64) * (int)kBox + 8 * 2048 + 1024;
  static std::atomic<uint64_t> devices{0};
  if (!ops_smem_limit((const void*)attn_fwd_tc_kernel<T, DP, SPLIT>, smem, devices)) return WUBU_B200_ERR_CUDA;
  const long long work = (long long)((a.Tq + 2 * kTile - 1) / (2 * kTile)) * p.splits * a.Hq * a.B;
  const int sms = ops_sms();
  if (work > 0x3FFFFFFF || !sms) return sms ? WUBU_B200_ERR_SHAPE : WUBU_B200_ERR_CUDA;
  attn_fwd_tc_kernel<T, DP, SPLIT><<<(unsigned)(work < sms ? work : sms), kThreads, smem, st>>>(maps, p);
  const int rc = ops_launched("attn_forward");
  if (rc != WUBU_B200_OK || !SPLIT) return rc;
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  return ops_launch_after(attn_fwd_join_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st,
                          "attn_forward join", p);
}
template <typename T>
int launch_fwd(const AttnFwdMaps& maps, const AttnParams& p, cudaStream_t st) {
  if (p.splits > 1)
    return p.a.D <= 64 ? launch_fwd<T, 64, true>(maps, p, st) : launch_fwd<T, 128, true>(maps, p, st);
  return p.a.D <= 64 ? launch_fwd<T, 64, false>(maps, p, st) : launch_fwd<T, 128, false>(maps, p, st);
}

}  // namespace

// Few query rows and many keys: the keys of a row are split over CTAs, as many as fill the SMs once, where that
// takes more than three tiles off a CTA's chain: a tile is about 1.1 us of it, the join about 3 us.  (One query,
// 64 values, us split / whole: 12 heads, 1500 keys 12.9 / 18.7, 600 keys 11.4 / 11.5, 400 keys 10.3 / 10.0, 200
// keys 9.1 / 7.5; 72 heads, 1500 keys 17.1 / 19.3, 900 keys 14.8 / 15.8, 300 keys 12.8 / 9.7; 84 heads in two
// parts, more than fill the SMs once, 1500 keys 27 / 19.4.)
int attn_fwd_splits(const WubuB200Attn& a) {
  const long long ctas = (long long)((a.Tq + 2 * kTile - 1) / (2 * kTile)) * a.Hq * a.B;
  const int tiles = (a.Tk + kTile - 1) / kTile, sms = ops_sms();
  if (ctas == 0 || 2 * ctas > sms) return 1;
  const long long most = sms / ctas < kMaxSplits ? sms / ctas : kMaxSplits;
  const int s = (int)(most < tiles ? most : tiles);
  return s > 1 && tiles - (tiles + s - 1) / s > 3 ? s : 1;
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
  return a.dtype == WUBU_B200_BF16 ? launch_fwd<bf16>(maps, p, st) : launch_fwd<f16>(maps, p, st);
}

}  // namespace wb
