// attention.cuh — softmax attention and its gradient: parameters and index arithmetic of the kernels.
#pragma once
#include "ops.cuh"

namespace wb {

struct AttnParams {
  WubuB200Attn a;    // with scale resolved and strides of unit extents cleared
  int group;         // query heads to a key / value head
  float* delta;      // backward: [B][Hq][t_pad] - rowsum(P * dP)
  float* lse2;       //           the negative log-sum-exp in units of log 2; -infinity where a query sees nothing
  unsigned* counter;    // backward: items drawn
  unsigned* norm_bits;  // backward, fp16: [2][B][Hkv] bits of the largest squared row norms of dO and of V
  int t_pad;
  int splits;        // forward: parts that the keys are split into, each with an out and an lse of its own
  float* part;       // [splits][B][Hq][Tq][D]
  float* part_lse;   // [splits][B][Hq][Tq]
  int kv_splits, q_splits;             // backward: parts of the steps of a key tile's and of a query tile's item
  float *part_dk, *part_dv, *part_dq;  // [splits][B][H][T][D]
  int* err;
  unsigned long long wait_ns;
};

// One item's lengths, and the range of keys that a query sees: query i sits at place i + off.
struct AttnItem {
  int ql, kl, off;
  AttnItem() = default;
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

// The CTAs of a grid no larger than the SMs work through `work` items, heaviest first where that is known:
// there and back over the CTAs, so that who had the heaviest item of a round has the lightest of the next.
struct AttnRounds {
  int work, next, round;
  WB_DEV AttnRounds(int work_) : work(work_), next(blockIdx.x), round(0) {}
  WB_DEV bool more() const { return next < work; }
  WB_DEV void advance() {
    ++round;
    next = round * (int)gridDim.x + ((round & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  }
};

int attn_forward(const AttnParams& p, cudaStream_t st);
long long attn_fwd_bytes(const WubuB200Attn& a);  // the forward's workspace
long long attn_bwd_bytes(const WubuB200Attn& a);  // the backward's
int attn_backward(const AttnParams& p, cudaStream_t st);

// bits [lo, hi) of 32
WB_DEV uint32_t see_bits(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? ~0u : hi <= 0 ? 0u : (1u << hi) - 1u;
  const uint32_t below_lo = lo >= 32 ? ~0u : lo <= 0 ? 0u : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}

// ---- tensor-core tiles ---------------------------------------------------------------------------
// A tile is 128 tokens of one head in shared memory, as one box of 64 values a row (DP = 64) or two
// (DP = 128), 16 KB each with 128-byte swizzle; columns from D on and tokens from T on are filled with zeros by
// the copy.  The same tile serves as an operand along its values (K-major: q k^T, dO V^T) and along its
// tokens (MN-major: P V, P^T dO, dS K, dS^T Q).
constexpr int kTile = 128;
constexpr uint32_t kBox = 128 * 128;  // bytes

// The map of a view's tokens x values; false (with a message) if it cannot be encoded.
bool attn_map(CUtensorMap* m, const WubuB200View& v, int B, int T, int H, int D);

WB_DEV void load_tile(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int t0, int h, int b, int boxes) {
  for (int i = 0; i < boxes; ++i) tma_load_4d_warp(dst + i * kBox, m, bar, i * 64, t0, h, b);
}
WB_DEV uint64_t desc_k(const uint8_t* tile) { return make_sdesc(smem_u32(tile), 16, 1024, 2); }
WB_DEV uint64_t desc_mn(const uint8_t* tile) { return make_sdesc(smem_u32(tile), kBox, 1024, 2); }

// Four steps of 16 in one go (one election, the later steps' operands by constant offsets): D[tmem] (+)= A B^T
// with both operands in shared memory along their rows.
WB_DEV void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "add.u64 a1, %1, 2;\n\tadd.u64 b1, %2, 2;\n\t"
      "add.u64 a2, %1, 4;\n\tadd.u64 b2, %2, 4;\n\t"
      "add.u64 a3, %1, 6;\n\tadd.u64 b3, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, 1;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in tensor memory (128 rows, two 16-bit values a column, the second pair of steps at column A2)
// and B along its tokens (16 tokens are 2 KB).
template <int A2 = 16>
WB_DEV void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u64 b1, %2, 128;\n\t"
      "add.u32 a2, %1, %5;\n\tadd.u64 b2, %2, 256;\n\t"
      "add.u32 a3, a2, 8;\n\tadd.u64 b3, %2, 384;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(A2)
      : "memory");
}
// D[tmem] = A B^T over the values of two tiles; `ksteps` (at most DP / 16) steps of 16
template <int DP>
WB_DEV void mma_values(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int ksteps) {
#pragma unroll
  for (int box = 0; box < DP / 64; ++box) {
    const uint64_t ab = a + box * (kBox >> 4), bb = b + box * (kBox >> 4);
    if (ksteps >= 4 * box + 4) {
      mma4_ss(d, ab, bb, idesc, box);
    } else {
      for (int k = 4 * box; k < ksteps; ++k) umma_f16_warp(d, ab + 2 * (k & 3), bb + 2 * (k & 3), idesc, k != 0);
    }
  }
}

WB_DEV void tmem_ld32_async(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
WB_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// After tmem_wait_ld: ties 32 loaded values to this point, so that no use of them is moved above the wait.
WB_DEV void tmem_use32(float* v) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]),
                 "+f"(v[i + 6]), "+f"(v[i + 7]));
}
template <int N>
WB_DEV void tmem_load(uint32_t taddr, float* v) {  // N columns, a multiple of 32
#pragma unroll
  for (int g = 0; g < N; g += 32) tmem_ld32_async(taddr + g, v + g);
  tmem_wait_ld();
#pragma unroll
  for (int g = 0; g < N; g += 32) tmem_use32(v + g);
}
WB_DEV void tmem_load16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]),
                 "+f"(v[i + 6]), "+f"(v[i + 7]));
}
WB_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
WB_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
WB_DEV void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
WB_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// mbar_wait_warp with a first test in line: most waits of the pipeline are for phases that are long complete.
WB_DEV bool bar_wait(uint64_t* bar, uint32_t parity, int* err, int code, unsigned long long limit_ns) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, done)) return true;
  return mbar_wait_warp(bar, parity, err, code, limit_ns);
}
// A warp writes 32 rows x 8 N values, a row in each lane (packed pairs w[4 N]), 16 N bytes to a row at a time:
// through 512 N bytes of shared memory, 16-byte pieces swizzled by row, then N lanes to a row.  `row` is the
// first row's address, rows are `stride` elements apart; rows from `rows` and values from `cols` on are
// left out.  (Each lane storing its own row touched 32 lines an instruction and took several thousand
// cycles a tile.)
template <int N, typename T>
WB_DEV void store_rows(uint8_t* stage, const uint32_t* w, T* row, long long stride, int rows, int cols) {
  static_assert(N == 2 || N == 4, "");
  constexpr int kSkew = N == 4 ? 1 : 2;  // rows apart by 128 bytes take other pieces
  const int lane = threadIdx.x & 31;
  uint4* st = reinterpret_cast<uint4*>(stage);
#pragma unroll
  for (int c = 0; c < N; ++c)
    st[lane * N + (c ^ (lane >> kSkew & (N - 1)))] = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
  const int c = lane & (N - 1);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = 32 / N * i + lane / N;
    const uint4 v = st[r * N + (c ^ (r >> kSkew & (N - 1)))];
    if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(row + r * stride + c * 8) = v;
  }
  __syncwarp();
}
// Four floats from shared memory, in program order with the other volatile accesses (the compiler would load all
// of a step's row values at its start and run out of registers).
WB_DEV float4 lds4(const float* p) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(p)));
  return v;
}
WB_DEV void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A warp writes zeros over the tokens [from, 128) of a tile (what lies beyond an item's length may be
// anything, and 0 x NaN is NaN), visibly to the tensor core.
WB_DEV void zero_rows(uint8_t* tile, int from, int boxes) {
  const int lane = threadIdx.x & 31;
  for (int i = 0; i < boxes; ++i)
    for (int o = from * 128 + lane * 16; o < (int)kBox; o += 512)
      *reinterpret_cast<uint4*>(tile + i * kBox + o) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// Moves registers between the warpgroups of a CTA (executed by whole warpgroups); the shares must add up
// to no more than what the CTA was launched with.
template <int N>
WB_DEV void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
WB_DEV void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The largest of three, NaN if one of them is.
WB_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two values on the FMA units, for x up to 120: x = n + f with n a whole number and |f| <= 1/2 (adding and
// subtracting 1.5 * 2^23 rounds to n), 2^f by a polynomial of degree 4 whose largest relative error is
// least (2.7e-6 in float32, far below the rounding of P; fitted by reweighted least squares), and n added
// to the exponent.  Below -125, and for NaN, it returns about 2^-125, which stands for 0: a caller whose
// values may be NaN looks for that elsewhere.
WB_DEV uint64_t ex2_poly2(uint64_t x) {
  float a, b;
  each(x, a, b);
  x = two(fmaxf(a, -125.f), fmaxf(b, -125.f));
  const uint64_t big = two(12582912.f, 12582912.f), t = add2(x, big);
  const uint64_t f = add2(x, fma2(t, two(-1.f, -1.f), big));  // x - (t - big)
  uint64_t p = two(0.009570102f, 0.009570102f);
  p = fma2(p, f, two(0.05591786f, 0.05591786f));
  p = fma2(p, f, two(0.24024744f, 0.24024744f));
  p = fma2(p, f, two(0.6931218f, 0.6931218f));
  p = fma2(p, f, two(0.9999993f, 0.9999993f));
  float ta, tb;
  each(t, ta, tb);
  each(p, a, b);
  return two(__uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23)),
             __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23)));
}
WB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace wb
