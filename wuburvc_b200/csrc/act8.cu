// act8.cu — an activation whose input is kept in 8 bits for the backward pass.
//
// Training a layer y = act(x) needs x again in the backward pass, and the next layer's weight
// gradient needs y.  Kept as 16-bit tensors that is 4 bytes a value; here x is kept as int8 with one fp32
// scale per 128 values of a row (1.03 bytes) and the backward forms both act'(x') and act(x') from it.
// The step of a block is max|x| / 127, so |x' - x| <= max|x| / 254 over the block.
//
// Both kernels move each byte once: forward 2 + 2 + 1 bytes a 16-bit value,
// backward 1 + 2 + 2 (+ 2 for y').  Eight threads own a block, 16 values each, as two 16-byte pieces
// 64 values apart, so that a warp's load covers whole 128-byte lines.  Measured (B200, 7984 x 2048 bf16, GELU):
// forward 18-20 us for 82 MB (65 % of the measured copy rate; bound by instruction issue: 26 a value, 75 % of the
// slots), backward with y' 22-24 us for 115 MB (76 %; 25 a value, 57 %, half the warps of an SM).
#include <type_traits>

#include "ops.cuh"

namespace wb {
namespace {

constexpr int kBlock = 128;        // values that share a scale
constexpr int kThreads = 256;
constexpr int kMaxCols = 0x7FFFFFFF - 2 * kBlock;  // columns are numbered in 32 bits, to the end of a block
constexpr float kTiny = 0x1p-100f;  // below this a block is kept as zeros (127 / max|x| must not overflow), but see block_scale

struct Act8 {
  float slope;
  const void* in;  // x (forward) or dy (backward)
  long long in_stride;
  void* out;       // y (forward) or dx (backward)
  void* again;     // y' (backward)
  signed char* q;
  float* scale;
  long long rows, blocks;  // blocks = rows * nblk
  int cols, nblk;
};

// Approximations of the hardware's function units (relative error near 2^-22).
WB_DEV float fast_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
WB_DEV float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

WB_DEV uint64_t both(float v) { return two(v, v); }
WB_DEV uint64_t abs2(uint64_t x) { return x & 0x7FFFFFFF7FFFFFFFull; }
WB_DEV uint64_t rcp2(uint64_t x) {
  float a, b;
  each(x, a, b);
  return two(fast_rcp(a), fast_rcp(b));
}
WB_DEV uint64_t ex22(uint64_t x) {
  float a, b;
  each(x, a, b);
  return two(fast_ex2(a), fast_ex2(b));
}

// Phi(-|x|) and e^(-x^2/2) of two values: the first is the second times a polynomial in t = 1 / (1 + p |x| / sqrt 2)
// (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26, halved; absolute error below 1e-7).
// Straight-line code with one exponential and one reciprocal a value: a library erff in two ranges with expf
// beside it took twice the time of the memory traffic, and one value at a time these kernels were still
// bound by instruction issue (31 a value).
WB_DEV uint64_t normal_tail2(uint64_t x, uint64_t& e) {
  const uint64_t t = rcp2(fma2(both(0.3275911f * 0.70710678118654752f), abs2(x), both(1.f)));
  e = ex22(mul2(mul2(x, x), both(-0.72134752044448170f)));
  uint64_t s = fma2(both(0.5f * 1.061405429f), t, both(-0.5f * 1.453152027f));
  s = fma2(s, t, both(0.5f * 1.421413741f));
  s = fma2(s, t, both(-0.5f * 0.284496736f));
  s = fma2(s, t, both(0.5f * 0.254829592f));
  return mul2(mul2(s, t), e);
}

template <int ACT>
WB_DEV uint64_t act_value2(uint64_t x, float slope) {
  float a, b;
  each(x, a, b);
  if (ACT == WUBU_B200_ACT_LRELU || ACT == WUBU_B200_ACT_LRELU_SIGN)
    return two(a > 0.f ? a : slope * a, b > 0.f ? b : slope * b);
  if (ACT == WUBU_B200_ACT_GELU) {
    // x Phi(x) = max(x, 0) - |x| Phi(-|x|), whose second term is 0 from |x| = 64 on (so that infinity stays)
    uint64_t e;
    const uint64_t tail = normal_tail2(x, e);
    return fma2(two(-fminf(fabsf(a), 64.f), -fminf(fabsf(b), 64.f)), tail, two(fmaxf(a, 0.f), fmaxf(b, 0.f)));
  }
  if (ACT == WUBU_B200_ACT_SILU) return mul2(x, rcp2(add2(both(1.f), ex22(mul2(x, both(-1.4426950408889634f))))));
  return x;
}
// The slope that the backward of a block with this scale takes: NaN where the block is kept as NaN, so that the
// leaky ReLU's derivative, which looks at x' > 0 alone, is NaN there as the others' are.
WB_DEV float slope_of(float slope, float scale) { return scale == scale ? slope : scale; }
// act(x) and act'(x)
template <int ACT>
WB_DEV void act_both2(uint64_t x, float slope, uint64_t& y, uint64_t& d) {
  if (ACT == WUBU_B200_ACT_LRELU || ACT == WUBU_B200_ACT_LRELU_SIGN) {
    float a, b;
    each(x, a, b);
    d = two(a > 0.f ? 1.f : slope, b > 0.f ? 1.f : slope);
    y = mul2(x, d);
  } else if (ACT == WUBU_B200_ACT_GELU) {
    uint64_t e;
    const uint64_t tail = normal_tail2(x, e);
    // Phi(x) = 1/2 + (1/2 - Phi(-|x|)) with x's sign
    const uint64_t h = fma2(tail, both(-1.f), both(0.5f));
    const uint64_t cdf = add2(both(0.5f), abs2(h) | (x & 0x8000000080000000ull));
    y = mul2(x, cdf);
    d = fma2(mul2(x, both(0.39894228040143268f)), e, cdf);
  } else if (ACT == WUBU_B200_ACT_SILU) {
    const uint64_t t = rcp2(add2(both(1.f), ex22(mul2(x, both(-1.4426950408889634f)))));
    y = mul2(x, t);
    d = fma2(y, fma2(t, both(-1.f), both(1.f)), t);
  } else {
    y = x;
    d = both(1.f);
  }
}

// max|x| as float bits: the order of non-negative floats is that of their bits, and infinities and
// NaN come out above every finite value (a floating-point maximum would drop a NaN).
WB_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The same of 8 values in memory form; 16-bit values two at a time.
WB_DEV uint32_t abs_bits8(const uint4* r, float) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m = max(max(m, r[i].x & 0x7FFFFFFFu), r[i].y & 0x7FFFFFFFu);
    m = max(max(m, r[i].z & 0x7FFFFFFFu), r[i].w & 0x7FFFFFFFu);
  }
  return m;
}
WB_DEV uint32_t abs_halves(const uint4* r) {
  constexpr uint32_t k = 0x7FFF7FFFu;
  const uint32_t m = __vmaxu2(__vmaxu2(r->x & k, r->y & k), __vmaxu2(r->z & k, r->w & k));
  return max(m >> 16, m & 0xFFFFu);
}
WB_DEV uint32_t abs_bits8(const uint4* r, bf16) { return abs_halves(r) << 16; }
WB_DEV uint32_t abs_bits8(const uint4* r, f16) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)abs_halves(r))));
}

// ACT_LRELU_SIGN keeps the positive values of a tiny block too, as one step of kTiny / 127.
template <int ACT>
WB_DEV void block_scale(uint32_t top, float& inv, float& scale) {
  const float m = __uint_as_float(top);
  inv = m < kTiny ? 0.f : __fdiv_rn(127.f, m);
  scale = m < kTiny ? (ACT == WUBU_B200_ACT_LRELU_SIGN && m > 0.f ? kTiny / 127.f : 0.f) : __fdiv_rn(m, 127.f);
  if (top >= 0x7F800000u) {  // an infinity or a NaN in the block
    inv = 0.f;
    scale = __uint_as_float(0x7FC00000u);
  }
}

// round-to-even(x * inv) as an int8 in the low byte: adding 1.5 * 2^23 leaves the integer in the low bits of
// the float.  ACT_LRELU_SIGN: what is positive stays so.
// One value at a time: the assembler joins a product and a sum of two values into one rounding.
template <int ACT>
WB_DEV uint32_t quantise(float x, float inv) {
  float v = __fmul_rn(x, inv);
  if (ACT == WUBU_B200_ACT_LRELU_SIGN && x > 0.f) v = fmaxf(v, 1.f);
  return __float_as_uint(__fadd_rn(v, 12582912.f));
}
WB_DEV uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// byte k of w, offset by 128, as a float: the byte becomes the low mantissa bits of 2^23
WB_DEV float dequantise(uint32_t w_offset, int k) {
  return __uint_as_float(__byte_perm(w_offset, 0x4B000000u, 0x7440u | (uint32_t)k)) - 8388736.f;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) act8_forward_kernel(const Act8 a) {
  const int t = threadIdx.x & 7;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  const bool on = blk < a.blocks;
  const long long row = !on ? 0 : a.nblk == 1 ? blk : blk / a.nblk;
  const int c0 = on ? (int)(blk - row * a.nblk) * kBlock + t * 8 : a.cols;
  const T* x = static_cast<const T*>(a.in) + row * a.in_stride;
  uint4 raw[2][sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      raw[i][k] = c0 + 64 * i < a.cols ? __ldg(reinterpret_cast<const uint4*>(x + c0 + 64 * i) + k) : make_uint4(0, 0, 0, 0);
  uint32_t top = max(abs_bits8(raw[0], T()), abs_bits8(raw[1], T()));
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
  if (!on) return;
  float inv, scale;
  block_scale<ACT>(top, inv, scale);
  if (t == 0) a.scale[blk] = scale;
  const bool bad = top >= 0x7F800000u;  // q = 0 there (x * 0 may be NaN)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (c0 + 64 * i >= a.cols) continue;
    float w[8];
    const T* e = reinterpret_cast<const T*>(raw[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = to_float(e[k]);
    const long long at = row * a.cols + c0 + 64 * i;
    uint32_t q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = quantise<ACT>(w[k], inv);
    const uint2 packed = make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
    *reinterpret_cast<uint2*>(a.q + at) = bad ? make_uint2(0, 0) : packed;
    if (a.out) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) each(act_value2<ACT>(two(w[k], w[k + 1]), a.slope), w[k], w[k + 1]);
      store8(static_cast<T*>(a.out) + at, w);
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) act8_backward_kernel(const Act8 a) {
  const int t = threadIdx.x & 7;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  if (blk >= a.blocks) return;
  const long long row = a.nblk == 1 ? blk : blk / a.nblk;
  const int c0 = (int)(blk - row * a.nblk) * kBlock + t * 8;
  const float scale = __ldg(a.scale + blk), slope = slope_of(a.slope, scale);
  const long long at = row * a.cols + c0;
  uint2 q[2];
  float g[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (c0 + 64 * i >= a.cols) continue;
    q[i] = __ldg(reinterpret_cast<const uint2*>(a.q + at + 64 * i));
    if (a.in) load8(static_cast<const T*>(a.in) + row * a.in_stride + c0 + 64 * i, g[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (c0 + 64 * i >= a.cols) continue;
    float y[8];
    const uint32_t lo = q[i].x ^ 0x80808080u, hi = q[i].y ^ 0x80808080u;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const uint32_t w = k < 4 ? lo : hi;
      const uint64_t x = mul2(two(dequantise(w, k & 3), dequantise(w, (k & 3) + 1)), both(scale));
      uint64_t yy, d;
      act_both2<ACT>(x, slope, yy, d);
      each(yy, y[k], y[k + 1]);
      each(mul2(two(g[i][k], g[i][k + 1]), d), g[i][k], g[i][k + 1]);
    }
    if (a.out) store8(static_cast<T*>(a.out) + at + 64 * i, g[i]);
    if (a.again) store8(static_cast<T*>(a.again) + at + 64 * i, y);
  }
}

// Rows whose length, stride or address rules out 16-byte pieces: a warp owns a block, 4 values a lane.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) act8_forward_any_kernel(const Act8 a) {
  const int lane = threadIdx.x & 31;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (blk >= a.blocks) return;
  const long long row = blk / a.nblk;
  const int c0 = (int)(blk - row * a.nblk) * kBlock + lane;
  const T* x = static_cast<const T*>(a.in) + row * a.in_stride;
  float v[4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = c0 + 32 * i < a.cols ? to_float(x[c0 + 32 * i]) : 0.f;
    top = max(top, abs_bits(v[i]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  float inv, scale;
  block_scale<ACT>(top, inv, scale);
  if (lane == 0) a.scale[blk] = scale;
  const bool bad = top >= 0x7F800000u;
  uint32_t q[4];
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {  // (the same operations as above, value for value)
    q[i] = quantise<ACT>(v[i], inv);
    q[i + 1] = quantise<ACT>(v[i + 1], inv);
    each(act_value2<ACT>(two(v[i], v[i + 1]), a.slope), y[i], y[i + 1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c0 + 32 * i >= a.cols) continue;
    const long long at = row * a.cols + c0 + 32 * i;
    a.q[at] = bad ? (signed char)0 : (signed char)q[i];
    if (a.out) static_cast<T*>(a.out)[at] = from_float<T>(y[i]);
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) act8_backward_any_kernel(const Act8 a) {
  const int lane = threadIdx.x & 31;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (blk >= a.blocks) return;
  const long long row = blk / a.nblk;
  const int c0 = (int)(blk - row * a.nblk) * kBlock + lane;
  const float scale = a.scale[blk], slope = slope_of(a.slope, scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 32 * i;
    if (c >= a.cols) continue;
    const long long at = row * a.cols + c;
    uint64_t yy, dd;
    float y, d, unused;
    act_both2<ACT>(two((float)a.q[at] * scale, 0.f), slope, yy, dd);
    each(yy, y, unused);
    each(dd, d, unused);
    if (a.out)
      static_cast<T*>(a.out)[at] =
          from_float<T>(to_float(static_cast<const T*>(a.in)[row * a.in_stride + c]) * d);
    if (a.again) static_cast<T*>(a.again)[at] = from_float<T>(y);
  }
}

template <typename F>
void with_act(int act, F f) {
  if (act == WUBU_B200_ACT_LRELU) f(std::integral_constant<int, WUBU_B200_ACT_LRELU>());
  else if (act == WUBU_B200_ACT_GELU) f(std::integral_constant<int, WUBU_B200_ACT_GELU>());
  else if (act == WUBU_B200_ACT_SILU) f(std::integral_constant<int, WUBU_B200_ACT_SILU>());
  else if (act == WUBU_B200_ACT_LRELU_SIGN) f(std::integral_constant<int, WUBU_B200_ACT_LRELU_SIGN>());
  else f(std::integral_constant<int, WUBU_B200_ACT_IDENTITY>());
}

// Everything but the pointers; 1 = nothing to do.
int check_act8(int dtype, int act, long long rows, int cols) {
  if (!ops_dtype_ok(dtype) || act < WUBU_B200_ACT_IDENTITY || act > WUBU_B200_ACT_LRELU_SIGN) return WUBU_B200_ERR_ARG;
  if (rows < 0 || cols < 0) return WUBU_B200_ERR_ARG;
  if (rows == 0 || cols == 0) return 1;
  if (cols > kMaxCols) return WUBU_B200_ERR_SHAPE;
  const long long nblk = (cols + kBlock - 1) / kBlock;
  // one warp per block in the general kernels, grid.x below 2^31
  if (rows > (((long long)1 << 31) - 1) * (kThreads / 32) / nblk) return WUBU_B200_ERR_SHAPE;
  return WUBU_B200_OK;
}

// 16-byte pieces of x / y and 8-byte pieces of q
bool whole_pieces(const Act8& a) {
  return a.cols % 8 == 0 && a.in_stride % 8 == 0 && aligned16(a.in) && aligned16(a.out) && aligned16(a.again) &&
         (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
}

}  // namespace
}  // namespace wb

using namespace wb;

extern "C" {

int wubu_b200_act8_forward(int dtype, int act, float slope, const void* x, long long x_stride, void* y, signed char* q,
                           float* scale, long long rows, int cols, void* stream) {
  const int rc = check_act8(dtype, act, rows, cols);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  if (!x || !q || !scale || (rows > 1 && x_stride < cols)) return WUBU_B200_ERR_ARG;
  Act8 a{slope, x, rows > 1 ? x_stride : 0, y, nullptr, q, scale, rows, 0, cols, (cols + kBlock - 1) / kBlock};
  a.blocks = rows * a.nblk;
  cudaStream_t st = (cudaStream_t)stream;
  const int per = whole_pieces(a) ? kThreads / 8 : kThreads / 32;
  const unsigned grid = (unsigned)((a.blocks + per - 1) / per);
  with_dtype(dtype, [&](auto t) {
    with_act(act, [&](auto k) {
      typedef decltype(t) T;
      constexpr int A = decltype(k)::value;
      if (per == kThreads / 8) act8_forward_kernel<T, A><<<grid, kThreads, 0, st>>>(a);
      else act8_forward_any_kernel<T, A><<<grid, kThreads, 0, st>>>(a);
    });
  });
  return ops_launched("act8_forward");
}

int wubu_b200_act8_backward(int dtype, int act, float slope, const void* dy, long long dy_stride, const signed char* q,
                            const float* scale, void* dx, void* y_again, long long rows, int cols, void* stream) {
  const int rc = check_act8(dtype, act, rows, cols);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  if (!q || !scale || !dy != !dx || (!dx && !y_again) || (dy && rows > 1 && dy_stride < cols)) return WUBU_B200_ERR_ARG;
  Act8 a{slope, dy, dy && rows > 1 ? dy_stride : 0, dx, y_again, const_cast<signed char*>(q),
         const_cast<float*>(scale), rows, 0, cols, (cols + kBlock - 1) / kBlock};
  a.blocks = rows * a.nblk;
  cudaStream_t st = (cudaStream_t)stream;
  const int per = whole_pieces(a) ? kThreads / 8 : kThreads / 32;
  const unsigned grid = (unsigned)((a.blocks + per - 1) / per);
  with_dtype(dtype, [&](auto t) {
    with_act(act, [&](auto k) {
      typedef decltype(t) T;
      constexpr int A = decltype(k)::value;
      if (per == kThreads / 8) act8_backward_kernel<T, A><<<grid, kThreads, 0, st>>>(a);
      else act8_backward_any_kernel<T, A><<<grid, kThreads, 0, st>>>(a);
    });
  });
  return ops_launched("act8_backward");
}

}  // extern "C"
