// attention_bwd.cu — the gradient of softmax attention on the tensor cores.
//
// With P = 2^(c S - L) recomputed from the scores and the log-sum-exp L (c = scale log2 e, L in units of
// log 2), D_i = sum_j P_ij (dO V^T)_ij and dS = P (dO V^T - D):
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K.
// D is also sum_d dO_id O_id, which takes one pass over the rows where the sum over keys takes two more products.
// But O is the forward's result, rounded to 16 bits, and where a row sees few keys that rounding shows beside the
// one of dS (dQ and dK: 2.3 times the error of a single rounding for 2 keys, 1.5-2 for 4 to 16, 1.4 from 32
// on).  So rows of up to 16 keys sum over them, in float32 (1.3-1.5 times for any length).
// dK and dV are sums over queries and dQ is a sum over keys.  One grid does both, in two roles: a CTA of the
// first owns 128 keys and runs over the queries that see them (and over the query heads that share
// the key head), a CTA of the second owns 128 queries and runs over their keys.  S and dO V^T are formed in
// both (7 products where 5 are the least), and in return no sum crosses CTAs: there are no atomics
// and the result does not depend on the order in which CTAs run.
//
// Everything between the products stays in tensor memory.  The first role forms the transposed scores
// (rows are keys), so that P^T and dS^T are written over them as the A operands of the next products.
// Sixteen warps do the exponentials, four to a row quadrant, 32 columns a thread; one warp loads, one
// issues.  A CTA an SM works through the items of both roles, loading the next one's tiles behind the last
// one's steps; where one item would outlast the rest, its steps are split and float32 parts joined.  A
// step's products and its elementwise halves alternate:
//   keys' role:     tensor  dV(n) S(n+1) | dK(n) dP(n+1)      warps  dS(n) | P(n+1)        at 128 values a row
//                           dV(n) | dK(n) dP(n+1) S(n+2)             dS(n) | P(n+1)        up to 64
//   queries' role:  tensor  dQ(n) dP(n+1) S(n+2)              warps  P(n+1) dS(n+1)
//
// Measured (B200): 16 heads on 4, 4001 tokens causal, 128 values: 263 us with its inputs in L2 (floor 101 us for 5
// products, 141 for the 7); 4 x 16 heads, 2048 x 64: 318 us; 16 x up to 499, 12 heads of 64: 77 us (floor 9.8).  What bounds
// it is the chain product - exponentials - product of a step: without any exponential it is 5 % faster.
//
// fp16 has few small numbers and a low ceiling, so its P is scaled by 2^14 (P <= 1) and its dS by the
// power of two that the norms of dO and V allow: |dS| <= P (|dO_i| |V_j| + |D_i|) <= 2 max|dO| max|V|.
#include <type_traits>

#include "attention.cuh"

namespace wb {
namespace {

constexpr int kProducer = 16, kMma = 17, kThreads = 640;  // 640 x 96 registers = 512 x 104 + 128 x 64
constexpr float kLog2e = 1.4426950408889634f;
// Tiles in the ring of Q or K, and of dO or V.  (Of K the second role wants a third, which 128 values a row
// leave no room for beside the store staging.)
template <int DP>
constexpr int kStagesA = DP == 64 ? 3 : 2;
constexpr int kStagesB = 2;

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
  uint64_t item_full[2], item_empty[2], res_full, res_empty, a_full[3], a_empty[3], b_full[kStagesB], b_empty[kStagesB], s_full[2], dp_full, p_ready[2],
      ds_ready, acc_full, acc_read, mma_done;
};

// A work item: 128 keys or 128 queries of one head, and a part of the steps over the other side's tiles.
struct BwdWork {
  AttnItem it;
  bool kv;
  int b, hk, hq, own0, split;
  int t0, per_head;      // the other side's first tile and their count, for each head
  int steps, t, h;       // of this part: steps, and where they start
  bool none;             // no item: the work is done
  BwdWork() = default;
  WB_DEV BwdWork(const AttnParams& p, int id, int kv_work) {
    const WubuB200Attn& a = p.a;
    none = false;
    kv = id < kv_work;
    unsigned r = kv ? id : id - kv_work;
    const unsigned heads = kv ? a.Hkv : a.Hq, splits = kv ? p.kv_splits : p.q_splits;
    const unsigned u = r / heads;
    const int head = r - u * heads;
    r = u / (unsigned)a.B;
    b = u - r * a.B;
    it = AttnItem(a, b);
    split = 0;
    if (splits > 1) {
      split = r % splits;
      r /= splits;
    }
    // keys in order (causal: the first have the most queries), queries from the last on
    own0 = (kv ? (int)r : (a.Tq + kTile - 1) / kTile - 1 - (int)r) * kTile;
    hk = kv ? head : head / p.group;
    hq = kv ? head * p.group : head;
    t0 = per_head = 0;
    const int last = min(own0 + kTile, kv ? it.kl : it.ql) - 1;
    if (last >= own0) {
      const int lo = kv ? it.query_lo(a, own0) : it.key_lo(a, own0), hi = kv ? it.query_hi(a, last) : it.key_hi(a, last);
      if (hi > lo) {
        t0 = lo / kTile;
        per_head = (hi + kTile - 1) / kTile - t0;
      }
    }
    steps = kv ? per_head * p.group : per_head;
    t = t0;
    h = kv ? hq : hk;
    if (splits > 1 && steps) {
      const int n0 = (int)((long long)steps * split / splits), n1 = (int)((long long)steps * (split + 1) / splits);
      steps = n1 - n0;
      h += n0 / per_head;
      t += n0 % per_head;
    }
  }
  WB_DEV void advance(int& tt, int& hh) const {
    if (++tt == t0 + per_head) {
      tt = t0;
      ++hh;
    }
  }
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

// The CTAs take items in order as they come free (the lengths and causal order make items unequal): the first by
// their number, the rest from a counter that the kernel before has cleared.  The loading warp draws, works
// the item out (divisions and the item's lengths: about a thousand cycles, behind the last item's steps) and hands
// it to the other warps.  Which CTA works on an item does not change its result.
struct Items {
  Barriers& bar;
  const BwdWork* slots;
  int n;  // taken so far
  WB_DEV bool take(BwdWork& k, const AttnParams& p) {
    const int s = n & 1;
    const bool ok = bar_wait(&bar.item_full[s], (n >> 1) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
    k = slots[s];
    if (!ok) k.none = true;
    return !k.none;
  }
  WB_DEV void done() {  // with the item as it lies in the slot
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bar.item_empty[n & 1]);
    ++n;
  }
};

// SPLIT: in one role at least the steps of an item are split.
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
attn_bwd_tc_kernel(const __grid_constant__ AttnBwdMaps maps, const __grid_constant__ AttnParams p, int kv_work, int work) {
  constexpr int kBoxes = DP / 64;
  constexpr uint32_t kTileBytes = kBoxes * kBox;
  constexpr int kA = kStagesA<DP>;
  // Up to 64 values a row two S fit beside the accumulators in the keys' role too, and S(n+2) is issued behind step
  // n's last product; at 128 its single S has to wait for dV(n), which reads P from it.
  constexpr bool kTwoS = DP == 64;
  constexpr float kShift = BwdShift<T>::value;
  constexpr int kBf16 = std::is_same<T, bf16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* res0 = smem;                    // K or Q, for a whole item
  uint8_t* res1 = smem + kTileBytes;       // V or dO
  uint8_t* ra = smem + 2 * kTileBytes;     // ring of Q or K
  uint8_t* rb = ra + kA * kTileBytes;      // ring of dO or V
  uint8_t* stage = rb + kStagesB * kTileBytes;  // 1 KB a warp
  // keys' role: the log-sum-exp and row sum of a step's 128 queries, with the first ring's tiles
  float* rows = reinterpret_cast<float*>(stage + kProducer * 1024);
  __shared__ Barriers bar;
  __shared__ BwdWork item_slots[2];
  __shared__ uint32_t tmem_slot;

  const WubuB200Attn& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.item_full[i], 1);
      mbar_init(&bar.item_empty[i], kProducer + 1);
    }
    mbar_init(&bar.res_full, 1);
    mbar_init(&bar.res_empty, 1);
    for (int i = 0; i < kA; ++i) {
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
    mbar_init(&bar.p_ready[0], kProducer);
    mbar_init(&bar.p_ready[1], kProducer);
    mbar_init(&bar.ds_ready, kProducer);
    mbar_init(&bar.acc_full, 1);
    mbar_init(&bar.acc_read, kProducer);
    mbar_init(&bar.mma_done, 1);
    fence_barrier_init();
  }
  if (warp == kMma) tmem_alloc(&tmem_slot, 512);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // columns: S at 0 (every second step's at 256, but for the keys' role at 128 values), dP at 128; dV at 384 and dK or
  // dQ at 448, at 128 values at 256 and 384
  const uint32_t tDP = tmem + 128, tAcc0 = tmem + (kTwoS ? 384 : 256), tAcc1 = tmem + (kTwoS ? 448 : 384);

  if (warp >= kProducer) {
    regs_dec<64>();
    if (warp == kProducer) {
      bool ok = true;
      FillTrack fr, fa, fb;
      int n = 0, items = 0, drawn = 0;  // steps, items with steps, and all items so far
      int next = blockIdx.x;
      for (;;) {
        const int id = __shfl_sync(0xffffffffu, next, 0);
        if (ok && drawn >= 2) ok = bar_wait(&bar.item_empty[drawn & 1], ((drawn >> 1) & 1) ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        const bool none = !ok || id >= work;
        BwdWork k(p, none ? 0 : id, kv_work);
        k.none = none;
        if (lane == 0) {
          item_slots[drawn & 1] = k;
          mbar_arrive(&bar.item_full[drawn & 1]);
        }
        __syncwarp();
        if (none) break;
        if (drawn++ == 0) griddep_wait();  // the counter, the row sums and log-sum-exps come from the kernel before
        // (drawn here, looked at when the item's loads are out)
        next = lane == 0 ? (int)gridDim.x + (int)atomicAdd(p.counter, 1u) : 0;
        if (k.steps == 0) continue;
        if (ok && items) ok = bar_wait(&bar.res_empty, (items - 1) & 1, p.err, ERR_WAIT_EMPTY, p.wait_ns);
        if (ok) {
          fr.fill(0, items);
          mbar_expect_tx_warp(&bar.res_full, 2 * kTileBytes);
          load_tile(res0, k.kv ? &maps.k : &maps.q, &bar.res_full, k.own0, k.kv ? k.hk : k.hq, k.b, kBoxes);
          load_tile(res1, k.kv ? &maps.v : &maps.dout, &bar.res_full, k.own0, k.kv ? k.hk : k.hq, k.b, kBoxes);
        }
        ++items;
        int t = k.t, h = k.h;
        for (int i = 0; i < k.steps; ++i, ++n) {
          const int sa = n % kA, sb = n % kStagesB;
          const uint32_t pa = (n / kA) & 1, pb = (n / kStagesB) & 1;
          if (ok && n >= kA) ok = bar_wait(&bar.a_empty[sa], pa ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
          if (ok) {
            fa.fill(sa, pa);
            mbar_expect_tx_warp(&bar.a_full[sa], kTileBytes + (k.kv ? 2 * kTile * 4 : 0));
            load_tile(ra + sa * kTileBytes, k.kv ? &maps.q : &maps.k, &bar.a_full[sa], t * kTile, h, k.b, kBoxes);
            if (k.kv) {
              const long long q = ((long long)k.b * a.Hq + h) * p.t_pad + t * kTile;
              bulk_load(rows + sa * 2 * kTile, p.lse2 + q, kTile * 4, &bar.a_full[sa]);
              bulk_load(rows + sa * 2 * kTile + kTile, p.delta + q, kTile * 4, &bar.a_full[sa]);
            }
          }
          if (ok && n >= kStagesB) ok = bar_wait(&bar.b_empty[sb], pb ^ 1u, p.err, ERR_WAIT_EMPTY, p.wait_ns);
          if (ok) {
            fb.fill(sb, pb);
            mbar_expect_tx_warp(&bar.b_full[sb], kTileBytes);
            load_tile(rb + sb * kTileBytes, k.kv ? &maps.dout : &maps.v, &bar.b_full[sb], t * kTile, h, k.b, kBoxes);
          }
          k.advance(t, h);
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
      bool ok = true;
      int n0 = 0, items = 0;           // steps and items (with steps) so far
      uint32_t p_phase[2] = {0, 0};    // of P, by the buffer of its S
      Items take{bar, item_slots, 0};
      for (BwdWork k; take.take(k, p);) {
        take.done();
        if (k.steps == 0) continue;
        const bool kv = k.kv;
        if (ok) ok = bar_wait(&bar.res_full, items & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
        ++items;
        const bool two_s = kTwoS || !kv;
        int ta = k.t, tb = k.t, unused = 0;  // tiles of the next S and dP
        // step n's tile in a ring, its rows beyond the item's length cleared
        auto clear = [&](uint8_t* tile, int tt) {
          const int valid = (kv ? k.it.ql : k.it.kl) - tt * kTile;
          if (ok && valid < kTile) zero_rows(tile, max(valid, 0), kBoxes);
        };
        auto issue_s = [&](int i) {
          const int n = n0 + i, sa = n % kA, buf = two_s ? i & 1 : 0;
          if (ok) ok = bar_wait(&bar.a_full[sa], (n / kA) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
          clear(ra + sa * kTileBytes, ta);
          k.advance(ta, unused);
          if (ok) {
            mma_values<DP>(tmem + 256 * buf, dr0, desc_k(ra + sa * kTileBytes), id_s, ksteps);
            umma_commit_warp(&bar.s_full[buf]);
          }
        };
        auto issue_dp = [&](int i) {
          const int n = n0 + i, sb = n % kStagesB;
          if (ok) ok = bar_wait(&bar.b_full[sb], (n / kStagesB) & 1, p.err, ERR_WAIT_FULL, p.wait_ns);
          clear(rb + sb * kTileBytes, tb);
          k.advance(tb, unused);
          if (ok) {
            mma_values<DP>(tDP, dr1, desc_k(rb + sb * kTileBytes), id_s, ksteps);
            umma_commit_warp(&bar.dp_full);
            if (!kv) umma_commit_warp(&bar.b_empty[sb]);  // nothing else reads V
            if (i == k.steps - 1) umma_commit_warp(&bar.res_empty);
          }
        };
        // acc += (A in tensor memory, 128 x 128, its quarters 32 columns apart) x tile
        auto issue_acc = [&](uint32_t acc, uint32_t src, const uint8_t* tile, int i) {
          const uint64_t d = desc_mn(tile);
          mma4_ts<32>(acc, src, d, id_o, i > 0);
          mma4_ts<32>(acc, src + 64, d + (4 * 2048u >> 4), id_o, 1);
        };
        issue_s(0);
        issue_dp(0);
        if (two_s && k.steps > 1) {
          // At 128 values the second S lies where the last item's dV may still be read.  Items without steps do not
          // count on either side: the warps gave the last item's P and dS only after they had read the accumulators
          // of the one before it, so the barrier is at most one phase behind and its parity tells which.
          if (!kTwoS && ok && items > 1) ok = bar_wait(&bar.acc_read, (items - 2) & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
          tc_fence_after();
          issue_s(1);
        }
        for (int i = 0; i < k.steps; ++i) {
          const int n = n0 + i, sa = n % kA, sb = n % kStagesB;
          if (kv) {
            // (with two S the warps may be done with P(i + 1) before this warp looks for P(i): a single barrier, two
            // phases on, would never show it)
            const int buf = two_s ? i & 1 : 0;
            if (ok) ok = bar_wait(&bar.p_ready[buf], buf ? p_phase[1] : p_phase[0], p.err, ERR_WAIT_ACC, p.wait_ns);
            if (buf) p_phase[1] ^= 1u;
            else p_phase[0] ^= 1u;
            tc_fence_after();
            if (ok) {
              issue_acc(tAcc0, tmem + 256 * buf, rb + sb * kTileBytes, i);
              umma_commit_warp(&bar.b_empty[sb]);
            }
            if (!two_s && i + 1 < k.steps) issue_s(i + 1);
          }
          if (ok) ok = bar_wait(&bar.ds_ready, n & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
          tc_fence_after();
          if (ok) {
            issue_acc(tAcc1, tDP, ra + sa * kTileBytes, i);
            umma_commit_warp(&bar.a_empty[sa]);
            if (i == k.steps - 1) umma_commit_warp(&bar.acc_full);
          }
          if (i + 1 < k.steps) issue_dp(i + 1);
          if (two_s && i + 2 < k.steps) issue_s(i + 2);
        }
        n0 += k.steps;
      }
      // every MMA this warp issued has completed before TMEM is released (also after a timed-out wait)
      umma_commit_warp(&bar.mma_done);
      bar_wait(&bar.mma_done, 0, p.err, ERR_WAIT_ACC, p.wait_ns);
    }
  } else {
    regs_inc<104>();
    const int quarter = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t DPc = tDP + lanes + 32 * quarter;
    const float c = a.scale * kLog2e;
    bool ok = true;
    int n0 = 0, items = 0;         // steps and items (with steps) so far
    uint32_t s_phase[2] = {0, 0};  // of the two buffers of S
    griddep_wait();                // the queries' role reads row sums and log-sum-exps itself
    Items take{bar, item_slots, 0};
    for (;;) {
      bool kv;
      int steps, t, t0, t_end;             // steps; the next step's tile, and the range that it runs through
      int lo, hi, whole0, whole1;          // the row's range, and the tiles that need no mask
      float l2 = 0.f, delta = 0.f, f = 1.f;  // queries' role: the row's values; the scale of P 2^shift (dP - D)
      {
        BwdWork k;
        if (!take.take(k, p)) break;
        kv = k.kv;
        steps = k.steps;
        t = k.t;
        t0 = k.t0;
        t_end = k.t0 + k.per_head;
        const int row = k.own0 + (warp & 3) * 32 + lane;  // a key or a query
        lo = kv ? k.it.query_lo(a, row) : k.it.key_lo(a, row);
        hi = kv ? k.it.query_hi(a, row) : k.it.key_hi(a, row);
        // tiles that all of this tile's live rows meet whole
        const int last = min(k.own0 + kTile, kv ? k.it.kl : k.it.ql) - 1;
        const int all_lo = last >= k.own0 ? (kv ? k.it.query_lo(a, last) : k.it.key_lo(a, last)) : 0;
        const int all_hi = kv ? k.it.query_hi(a, k.own0) : k.it.key_hi(a, k.own0);
        whole0 = (all_lo + kTile - 1) / kTile;
        whole1 = all_hi / kTile;
        if (!kBf16) f = ds_scale<T>(p, k.b, k.hk) * exp2f(-kShift);
        if (!kv && steps > 0) {
          const long long q = ((long long)k.b * a.Hq + k.hq) * p.t_pad + row;
          l2 = p.lse2[q];
          delta = p.delta[q];
        }
      }
      // the steps of one role (compiled for each: choices inside would cost an instruction a value)
      auto run = [&](auto role) {
        constexpr bool KV = decltype(role)::value;
        int sa = n0 % kA;
        uint32_t pa = (n0 / kA) & 1;
        for (int i = 0; i < steps; ++i) {
          const int buf = KV && !kTwoS ? 0 : i & 1;
          const bool masked = t < whole0 || t >= whole1;
          const int col0 = t * kTile + 32 * quarter;
          if (++t == t_end) t = t0;
          const uint32_t S = tmem + 256 * buf + lanes + 32 * quarter;
          const float* step_rows = rows + sa * 2 * kTile + 32 * quarter;
          if (KV) {
            if (ok) ok = bar_wait(&bar.a_full[sa], pa, p.err, ERR_WAIT_FULL, p.wait_ns);
            if (++sa == kA) {
              sa = 0;
              pa ^= 1u;
            }
          }
          if (ok) ok = bar_wait(&bar.s_full[buf], buf ? s_phase[1] : s_phase[0], p.err, ERR_WAIT_ACC, p.wait_ns);
          if (buf) s_phase[1] ^= 1u;
          else s_phase[0] ^= 1u;
          if (!ok) continue;
          tc_fence_after();
          float x[32];
          tmem_load<32>(S, x);
          const uint64_t cc = two(c, c), ll = two(l2, l2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint64_t l01 = ll, l23 = ll;
            if (KV) {
              const float4 v = lds4(step_rows + 4 * e);
              l01 = two(v.x, v.y);
              l23 = two(v.z, v.w);
            }
            each(fma2(two(x[4 * e], x[4 * e + 1]), cc, l01), x[4 * e], x[4 * e + 1]);
            each(fma2(two(x[4 * e + 2], x[4 * e + 3]), cc, l23), x[4 * e + 2], x[4 * e + 3]);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = ex2(x[e]);
          if (masked) {
            const uint32_t see = see_bits(lo - col0, hi - col0);
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = see >> e & 1 ? x[e] : 0.f;
          }
          if (KV) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack2(x[16 * g + 2 * e], x[16 * g + 2 * e + 1], T());
              tmem_st8(S + 8 * g, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.p_ready[buf]);
          }
          ok = bar_wait(&bar.dp_full, (n0 + i) & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
          if (!ok) continue;
          tc_fence_after();
          const uint64_t dd = two(delta, delta), ff = two(f, f);
#pragma unroll
          for (int g = 0; g < 2; ++g) {  // 16 columns at a time, written over columns that have been read
            float y[16];
            uint32_t w[8];
            tmem_load16(DPc + 16 * g, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float* xe = x + 16 * g + 4 * e;
              uint64_t d01 = dd, d23 = dd;
              if (KV) {
                const float4 v = lds4(step_rows + kTile + 16 * g + 4 * e);
                d01 = two(v.x, v.y);
                d23 = two(v.z, v.w);
              }
              uint64_t g0 = mul2(add2(two(y[4 * e], y[4 * e + 1]), d01), two(xe[0], xe[1]));
              uint64_t g1 = mul2(add2(two(y[4 * e + 2], y[4 * e + 3]), d23), two(xe[2], xe[3]));
              if (!kBf16) {
                g0 = mul2(g0, ff);
                g1 = mul2(g1, ff);
              }
              float u0, u1, u2, u3;
              each(g0, u0, u1);
              each(g1, u2, u3);
              w[2 * e] = pack2(u0, u1, T());
              w[2 * e + 1] = pack2(u2, u3, T());
            }
            tmem_st8(DPc + 8 * g, w);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.ds_ready);
        }
      };
      if (kv) run(std::true_type());
      else run(std::false_type());
      const BwdWork k = item_slots[take.n & 1];  // (read again rather than held in registers over the steps)
      take.done();
      n0 += k.steps;
      if (k.steps > 0) {
        if (ok) ok = bar_wait(&bar.acc_full, items & 1, p.err, ERR_WAIT_ACC, p.wait_ns);
        ++items;
        tc_fence_after();
      }
      // the accumulators, a quarter of the columns to each warpgroup
      const int row = k.own0 + (warp & 3) * 32 + lane;
      const bool live = hi > lo && k.steps > 0 && ok;
      const float ds_out = a.scale / (kBf16 ? 1.f : f * exp2f(kShift)), p_out = exp2f(-kShift);
      constexpr int kCols = DP / 4;
      const int d0 = kCols * quarter;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if (!kv && which == 0) continue;
        const float sc = which ? ds_out : p_out;
        const int tokens = kv ? a.Tk : a.Tq, H = kv ? a.Hkv : a.Hq, head = kv ? k.hk : k.hq;
#pragma unroll 1
        for (int d = d0; d < d0 + kCols; d += 16) {  // (one after the other: few registers)
          float o[16];
          if (k.steps > 0) tmem_load16((which ? tAcc1 : tAcc0) + lanes + d, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = live ? o[e] * sc : 0.f;
          if (SPLIT && (kv ? p.kv_splits : p.q_splits) > 1) {
            float* part = (!kv ? p.part_dq : which ? p.part_dk : p.part_dv) +
                          ((((long long)k.split * a.B + k.b) * H + head) * tokens + row) * a.D + d;
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              if (row < tokens && d + e < a.D) store8(part + e, o + e);
            __syncwarp();
          } else {
            const int r0 = k.own0 + (warp & 3) * 32;
            const WubuB200View& view = !kv ? a.dq : which ? a.dk : a.dv;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack2(o[2 * e], o[2 * e + 1], T());
            store_rows<2>(stage + warp * 1024, w, at<T>(view, k.b, r0, head) + d, view.token, tokens - r0, a.D - d);
          }
        }
      }
      if (k.steps == 0) continue;
      tc_fence_before();  // the accumulators are read before the next item's products may be issued
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_read);
    }
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

// - rowsum(dO * O) and the negative log-sum-exp in units of log 2 (with P's shift), padded to whole tiles with
// what gives probability 0; for fp16 also the largest squared norms of dO's and V's rows (an integer maximum over
// the bits of non-negative floats: its order does not matter).  N threads a row, 8 values each.
template <typename T, int N>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  griddep_launch();  // (for the kernel of the rows of few keys)
  const int t = threadIdx.x % N, i = blockIdx.x * (256 / N) + threadIdx.x / N, h = blockIdx.y, b = blockIdx.z;
  if (threadIdx.x == 0 && blockIdx.x == 0 && h == 0 && b == 0) *p.counter = 0;
  const AttnItem it(a, b);
  constexpr bool kNorms = std::is_same<T, f16>::value;
  float d = 0.f, g = 0.f, v = 0.f;
  if (i < it.ql && t * 8 < a.D) {
    const T* x = at<T>(a.dout, b, i, h) + t * 8;
    d = dot8(x, at<T>(a.out, b, i, h) + t * 8);
    if (kNorms) g = dot8(x, x);
  }
  if (kNorms && h % p.group == 0 && i < it.kl && t * 8 < a.D) {
    const T* x = at<T>(a.v, b, i, h / p.group) + t * 8;
    v = dot8(x, x);
  }
#pragma unroll
  for (int m = 1; m < N; m <<= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, m);
    if (kNorms) {
      g += __shfl_xor_sync(0xffffffffu, g, m);
      v += __shfl_xor_sync(0xffffffffu, v, m);
    }
  }
  if (t == 0 && i < p.t_pad) {
    const long long r = ((long long)b * a.Hq + h) * p.t_pad + i;
    const float l = i < it.ql ? a.lse[((long long)b * a.Hq + h) * a.Tq + i] * kLog2e : INFINITY;
    p.delta[r] = -d;
    p.lse2[r] = l == -INFINITY ? -INFINITY : BwdShift<T>::value - l;
  }
  if (kNorms) {
    const int n = a.B * a.Hkv, at_ = b * a.Hkv + h / p.group;
    const uint32_t gm = __reduce_max_sync(0xffffffffu, __float_as_uint(g));
    const uint32_t vm = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if ((threadIdx.x & 31) == 0) {
      if (gm) atomicMax(p.norm_bits + at_, gm);
      if (vm) atomicMax(p.norm_bits + n + at_, vm);
    }
  }
}

// Rows of up to kFewKeys keys have their D from the keys.  They lie in the rows [first, last) of an item: any of them
// where the window is no wider or the item has no more keys, else the 16 rows whose order or window ends at
// keys 1 to 16.
constexpr int kFewKeys = 16;
WB_DEV void few_key_range(const WubuB200Attn& a, const AttnItem& it, int& first, int& last) {
  first = 0;
  last = it.ql;
  if ((a.window > 0 && a.window <= kFewKeys) || it.kl <= kFewKeys) return;
  const int ahead = a.causal ? 0 : a.window - 1;  // a row at place p sees keys up to p + ahead
  first = max(0, -ahead - it.off);
  last = a.causal || a.window > 0 ? min(it.ql, kFewKeys - ahead - it.off) : 0;
}

// D[16 x 8] += A[16 x 16] B[8 x 16]^T, fragments as mma.sync has them
WB_DEV void mma_16x8(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bf16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
WB_DEV void mma_16x8(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, f16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// - D of the rows of few keys, over what the kernel before wrote for them; 16 rows to a warp.  Their keys lie within 31 in
// a row; S and dP are formed 16 x 16 at a time with fragments straight from memory: a tile this small is all
// latency, and the other tensor path would need it in shared memory first.  The order of a product's values
// being free, a lane's 8 of every 32 are those that lie together.  Cost (us with / without): 4001 tokens causal, 16
// heads on 4, 128 values 262 / 260; 16 x 499 causal, 12 heads of 64 76 / 74; with a window of 16 all rows are
// such: 4 x 4000, 16 heads on 4, 128 values 234 / 189.
template <typename T>
__global__ void __launch_bounds__(128) attn_few_keys_kernel(const AttnParams p) {
  const WubuB200Attn& a = p.a;
  const int h = blockIdx.y, b = blockIdx.z, warps = blockDim.x / 32;
  griddep_launch();
  const AttnItem it(a, b);
  int start, stop;
  few_key_range(a, it, start, stop);
  const int lane = threadIdx.x & 31, g = lane >> 2, t2 = (lane & 3) * 2;
  const float c = a.scale * kLog2e;
  bool waited = false;
  for (int r0 = start + (blockIdx.x * warps + threadIdx.x / 32) * 16; r0 < stop; r0 += gridDim.x * warps * 16) {
    int lo[2], hi[2], first = a.Tk, end = 0;
    float l[2], sum[2] = {0.f, 0.f};
    const T *q[2], *dout[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      int i = r0 + g + 8 * r;
      lo[r] = it.key_lo(a, i);
      hi[r] = it.key_hi(a, i);
      if (hi[r] - lo[r] > kFewKeys) hi[r] = lo[r];  // not one of them
      if (hi[r] > lo[r]) {
        first = min(first, lo[r]);
        end = max(end, hi[r]);
      }
      i = min(i, it.ql - 1);  // (beyond the item any row will do)
      l[r] = a.lse[((long long)b * a.Hq + h) * a.Tq + i] * kLog2e;
      q[r] = at<T>(a.q, b, i, h) + 4 * t2;
      dout[r] = at<T>(a.dout, b, i, h) + 4 * t2;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    end = __reduce_max_sync(0xffffffffu, end);
    for (int j0 = first; j0 < end; j0 += 16) {
      const T *k[2], *v[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j = min(j0 + 8 * n + g, end - 1);
        k[n] = at<T>(a.k, b, j, h / p.group) + 4 * t2;
        v[n] = at<T>(a.v, b, j, h / p.group) + 4 * t2;
      }
      float s[2][4] = {}, dp[2][4] = {};
#pragma unroll 1
      for (int d = 0; d < a.D; d += 32) {
        const bool on = d + 4 * t2 < a.D;
        auto eight = [&](const T* x) { return on ? __ldg(reinterpret_cast<const uint4*>(x + d)) : make_uint4(0, 0, 0, 0); };
        const uint4 q0 = eight(q[0]), q1 = eight(q[1]), g0 = eight(dout[0]), g1 = eight(dout[1]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint4 kn = eight(k[n]), vn = eight(v[n]);
          mma_16x8(s[n], q0.x, q1.x, q0.y, q1.y, kn.x, kn.y, T());
          mma_16x8(s[n], q0.z, q1.z, q0.w, q1.w, kn.z, kn.w, T());
          mma_16x8(dp[n], g0.x, g1.x, g0.y, g1.y, vn.x, vn.y, T());
          mma_16x8(dp[n], g0.z, g1.z, g0.w, g1.w, vn.z, vn.w, T());
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int n = x >> 2, r = x >> 1 & 1, j = j0 + 8 * n + t2 + (x & 1);
        if (j >= lo[r] && j < hi[r] && l[r] != -INFINITY) sum[r] += ex2(s[n][x & 3] * c - l[r]) * dp[n][x & 3];
      }
    }
    if (!waited) griddep_wait();
    waited = true;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      if (hi[r] > lo[r] && (lane & 3) == 0) p.delta[((long long)b * a.Hq + h) * p.t_pad + r0 + g + 8 * r] = -sum[r];
    }
  }
  if (!waited) griddep_wait();  // what waits for this kernel waits for the one before it too
}

// A gradient from the float32 sums of its parts, in order; 8 values a thread.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const float* part, int splits, WubuB200View out, int B, int H,
                                                        int tokens, int D) {
  griddep_wait();
  const long long all = (long long)B * H * tokens * D, at8 = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at8 >= all) return;
  float o[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 u = *reinterpret_cast<const float4*>(part + s * all + at8), v = *reinterpret_cast<const float4*>(part + s * all + at8 + 4);
    o[0] += u.x; o[1] += u.y; o[2] += u.z; o[3] += u.w;
    o[4] += v.x; o[5] += v.y; o[6] += v.z; o[7] += v.w;
  }
  const int d = (int)(at8 % D);
  const long long r = at8 / D;
  const int i = (int)(r % tokens), h = (int)(r / tokens % H), b = (int)(r / tokens / H);
  store8(at<T>(out, b, i, h) + d, o);
}

long long tiles_of(int T) { return (T + kTile - 1) / kTile; }

// Into how many parts the steps of a key tile's and of a query tile's item are split.  The grid is as long as its
// longest item: where that (4 products a step in the keys' role, 3 in the other) is longer than an even
// share of all the work, which happens with few heads or many that share a key head, it is cut to about
// that share.  Causal order halves the work but not the longest item.  Joining the parts costs what some 16
// products do, and parts of fewer than six steps lose (12 heads on 1, 700 tokens, 64 values: 34 us with two steps
// at least, 30 with six; at 400 tokens 31 and 27, four steps 25).  (us split / whole: 16 heads on 4,
// 4001 tokens causal, 128 values, 2 parts: 258 / 309; 12 heads on 1, 1500 tokens, 64 values: 60 / 207; 12 heads,
// 1500 causal, 64 values, the longest item 1.2 shares, so not split: 55 / 39; 2 heads of 96, 300 tokens, not split
// either: 25 / 18.)
void bwd_splits(const WubuB200Attn& a, int sms, int& kv, int& q) {
  const long long nq = tiles_of(a.Tq), nk = tiles_of(a.Tk), group = a.Hkv ? a.Hq / a.Hkv : 1;
  const long long kv_item = 4 * nq * group, q_item = 3 * nk;
  const long long share = (kv_item * nk * a.Hkv + q_item * nq * a.Hq) * a.B / (a.causal ? 2 : 1) / (sms > 0 ? sms : 1) + 1;
  auto parts = [&](long long item, long long steps) {
    long long s = (item + share - 1) / share;
    if (s > steps / 6) s = steps / 6;
    if (s > 16) s = 16;
    if (s < 2) return 1;
    const long long part = (item + s - 1) / s;
    return item - (part > share ? part : share) > 16 ? (int)s : 1;
  };
  kv = parts(kv_item, nq * group);
  q = parts(q_item, nk);
}

template <typename T, int DP>
int launch_bwd(const AttnBwdMaps& maps, const AttnParams& p, int sms, cudaStream_t st) {
  const WubuB200Attn& a = p.a;
  constexpr int smem = (2 + kStagesA<DP> + kStagesB) * (DP / 64) * (int)kBox + kProducer * 1024 + kStagesA<DP> * 2 * kTile * 4 + 1024;
  static std::atomic<uint64_t> devices[2];
  auto* kernel = p.kv_splits > 1 || p.q_splits > 1 ? attn_bwd_tc_kernel<T, DP, true> : attn_bwd_tc_kernel<T, DP, false>;
  if (!ops_smem_limit((const void*)attn_bwd_tc_kernel<T, DP, true>, smem, devices[0]) ||
      !ops_smem_limit((const void*)attn_bwd_tc_kernel<T, DP, false>, smem, devices[1]))
    return WUBU_B200_ERR_CUDA;
  if (std::is_same<T, f16>::value &&
      cudaMemsetAsync(p.norm_bits, 0, 2ull * a.B * a.Hkv * sizeof(unsigned), st) != cudaSuccess)
    return WUBU_B200_ERR_CUDA;
  const int rows = std::is_same<T, f16>::value && a.Tk > p.t_pad ? a.Tk : p.t_pad;
  constexpr int kRows = 256 / (DP / 8);
  attn_delta_kernel<T, DP / 8><<<dim3(rows ? (rows + kRows - 1) / kRows : 1, a.Hq, a.B), 256, 0, st>>>(p);
  int rc = ops_launched("attn_backward rows");
  if (rc != WUBU_B200_OK) return rc;
  // rows of few keys: all may be such, or 16 of an order or a window, or those of short items
  const bool all_few = (a.window > 0 && a.window <= kFewKeys) || a.Tk <= kFewKeys;
  if (a.Tq && a.Tk && (all_few || a.causal || a.window || a.k_lens)) {
    const bool one = !all_few && !a.k_lens;
    rc = ops_launch_after(attn_few_keys_kernel<T>, dim3(all_few ? p.t_pad / 64 : 1, a.Hq, a.B), dim3(one ? 32 : 128), 0, st,
                          "attn_backward few keys", p);
    if (rc != WUBU_B200_OK) return rc;
  }
  const long long kv = tiles_of(a.Tk) * a.Hkv * a.B * p.kv_splits, qs = tiles_of(a.Tq) * a.Hq * a.B * p.q_splits;
  if (kv + qs > 0x3FFFFFFF) return WUBU_B200_ERR_SHAPE;
  const int work = (int)(kv + qs);
  rc = ops_launch_after(kernel, dim3(work < sms ? work : sms), dim3(kThreads), smem, st,
                        "attn_backward", maps, p, (int)kv, work);
  auto join = [&](const float* part, int splits, const WubuB200View& out, int H, int tokens) {
    const long long n8 = (long long)a.B * H * tokens * a.D / 8;
    if (rc == WUBU_B200_OK && splits > 1 && n8)
      rc = ops_launch_after(attn_join_kernel<T>, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, st, "attn_backward join",
                            part, splits, out, a.B, H, tokens, a.D);
  };
  join(p.part_dk, p.kv_splits, a.dk, a.Hkv, a.Tk);
  join(p.part_dv, p.kv_splits, a.dv, a.Hkv, a.Tk);
  join(p.part_dq, p.q_splits, a.dq, a.Hq, a.Tq);
  return rc;
}

// The workspace: delta, lse2, counter and norm bits (to a multiple of 16 bytes), then the parts of dk, dv and dq.
long long bwd_layout(const WubuB200Attn& a, AttnParams* p) {
  int kv = 1, q = 1;
  bwd_splits(a, ops_sms(), kv, q);
  const long long rows = (long long)a.B * a.Hq * tiles_of(a.Tq) * kTile, bits = (1 + 2ll * a.B * a.Hkv + 3) / 4 * 4;
  const long long dkv = kv > 1 ? (long long)kv * a.B * a.Hkv * a.Tk * a.D : 0;
  const long long dq = q > 1 ? (long long)q * a.B * a.Hq * a.Tq * a.D : 0;
  if (p) {
    float* w = static_cast<float*>(a.workspace);
    p->delta = w;
    p->lse2 = w + rows;
    p->counter = reinterpret_cast<unsigned*>(w + 2 * rows);
    p->norm_bits = p->counter + 1;
    p->part_dk = w + 2 * rows + bits;
    p->part_dv = p->part_dk + dkv;
    p->part_dq = p->part_dv + dkv;
    p->kv_splits = kv;
    p->q_splits = q;
  }
  return (2 * rows + bits + 2 * dkv + dq) * (long long)sizeof(float);
}

}  // namespace

long long attn_bwd_bytes(const WubuB200Attn& a) { return bwd_layout(a, nullptr); }

int attn_backward(const AttnParams& in, cudaStream_t st) {
  AttnParams p = in;
  const WubuB200Attn& a = p.a;
  bwd_layout(a, &p);
  const int sms = ops_sms();
  if (!sms) return WUBU_B200_ERR_CUDA;
  AttnBwdMaps maps{};
  if (a.Tq && (!attn_map(&maps.q, a.q, a.B, a.Tq, a.Hq, a.D) || !attn_map(&maps.dout, a.dout, a.B, a.Tq, a.Hq, a.D)))
    return WUBU_B200_ERR_CUDA;
  if (a.Tk && (!attn_map(&maps.k, a.k, a.B, a.Tk, a.Hkv, a.D) || !attn_map(&maps.v, a.v, a.B, a.Tk, a.Hkv, a.D)))
    return WUBU_B200_ERR_CUDA;
  if (a.dtype == WUBU_B200_BF16)
    return a.D <= 64 ? launch_bwd<bf16, 64>(maps, p, sms, st) : launch_bwd<bf16, 128>(maps, p, sms, st);
  return a.D <= 64 ? launch_bwd<f16, 64>(maps, p, sms, st) : launch_bwd<f16, 128>(maps, p, sms, st);
}

}  // namespace wb
