// act8.cu — an activation whose input is kept in 8 bits for the backward pass.
//
// Training a layer y = act(x) needs x again in the backward pass, and the next layer's weight
// gradient needs y.  Kept as 16-bit tensors that is 4 bytes a value; here x is kept as int8 with one fp32
// scale per 128 values of a row (1.03 bytes) and the backward forms both act'(x') and act(x') from it.
// The step of a block is max|x| / 127, so |x' - x| <= max|x| / 254 over the block.
//
// Both kernels move each byte once and are bound by HBM: forward 2 + 2 + 1 bytes a 16-bit value,
// backward 1 + 2 + 2 (+ 2 for y').  Eight threads own a block, 16 values each, as two 16-byte pieces
// 64 values apart, so that a warp's load covers whole 128-byte lines.
#include "ops.cuh"

namespace wb {
namespace {

constexpr int kBlock = 128;        // values that share a scale
constexpr int kThreads = 256;
constexpr float kTiny = 0x1p-100f;  // below this a block is kept as zeros (127 / max|x| must not overflow)

struct Act8 {
  int act;
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

WB_DEV float exp2f_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(x) and the density phi(x) of the normal distribution from one exponential and one reciprocal:
// Phi(-|x|) is e^(-x^2/2) times a polynomial in t = 1 / (1 + p |x| / sqrt 2) (Abramowitz and Stegun,
// Handbook of Mathematical Functions, 7.1.26; absolute error below 1e-7).  Straight-line code: a
// library erff in two ranges, with expf beside it, made the backward twice as slow as its memory traffic.
WB_DEV void normal(float x, float& cdf, float& density) {
  const float z = fabsf(x);
  const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, z, 1.f));
  const float e = exp2f_fast(x * x * -0.72134752044448170f);  // e^(-x^2/2)
  float s = fmaf(1.061405429f, t, -1.453152027f);
  s = fmaf(s, t, 1.421413741f);
  s = fmaf(s, t, -0.284496736f);
  s = fmaf(s, t, 0.254829592f);
  const float tail = 0.5f * s * t * e;
  cdf = x > 0.f ? 1.f - tail : tail;
  density = e * 0.39894228040143268f;
}

WB_DEV float act_value(float x, int act, float slope) {
  if (act == WUBU_B200_ACT_LRELU) return x > 0.f ? x : slope * x;
  if (act == WUBU_B200_ACT_GELU) {
    float cdf, density;
    normal(x, cdf, density);
    return x * cdf;
  }
  if (act == WUBU_B200_ACT_SILU) return __fdividef(x, 1.f + __expf(-x));
  return x;
}
// act(x) and act'(x)
WB_DEV void act_both(float x, int act, float slope, float& y, float& d) {
  if (act == WUBU_B200_ACT_LRELU) {
    d = x > 0.f ? 1.f : slope;
    y = x * d;
  } else if (act == WUBU_B200_ACT_GELU) {
    float cdf, density;
    normal(x, cdf, density);
    y = x * cdf;
    d = fmaf(x, density, cdf);
  } else if (act == WUBU_B200_ACT_SILU) {
    const float t = __fdividef(1.f, 1.f + __expf(-x));
    y = x * t;
    d = t * (1.f + x * (1.f - t));
  } else {
    y = x;
    d = 1.f;
  }
}

// max|x| as float bits: the order of non-negative floats is that of their bits, and infinities and
// NaN come out above every finite value (a floating-point maximum would drop a NaN).
WB_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

WB_DEV void block_scale(uint32_t top, float& inv, float& scale) {
  const float m = __uint_as_float(top);
  inv = m < kTiny ? 0.f : __fdiv_rn(127.f, m);
  scale = m < kTiny ? 0.f : __fdiv_rn(m, 127.f);
  if (top >= 0x7F800000u) {  // an infinity or a NaN in the block
    inv = 0.f;
    scale = __uint_as_float(0x7FC00000u);
  }
}

// round-to-even(x * inv) as an int8: adding 1.5 * 2^23 leaves the integer in the low bits of the float
WB_DEV uint32_t quantise(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)) & 0xFFu;
}
// byte k of w, offset by 128, as a float: the byte becomes the low mantissa bits of 2^23
WB_DEV float dequantise(uint32_t w_offset, int k) {
  return __uint_as_float(__byte_perm(w_offset, 0x4B000000u, 0x7440u | (uint32_t)k)) - 8388736.f;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) act8_forward_kernel(const Act8 a) {
  const int t = threadIdx.x & 7;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  const bool on = blk < a.blocks;
  const long long row = on ? blk / a.nblk : 0;
  const int c0 = on ? (int)(blk - row * a.nblk) * kBlock + t * 8 : a.cols;
  const T* x = static_cast<const T*>(a.in) + row * a.in_stride;
  float v[16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float* w = v + 8 * i;
    if (c0 + 64 * i < a.cols) {
      load8(x + c0 + 64 * i, w);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) top = max(top, abs_bits(v[k]));
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
  if (!on) return;
  float inv, scale;
  block_scale(top, inv, scale);
  if (t == 0) a.scale[blk] = scale;
  const bool bad = top >= 0x7F800000u;  // q = 0 there (x * 0 may be NaN)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (c0 + 64 * i >= a.cols) continue;
    const float* w = v + 8 * i;
    const long long at = row * a.cols + c0 + 64 * i;
    uint32_t lo = 0, hi = 0;
    if (!bad) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lo |= quantise(w[k], inv) << (8 * k);
        hi |= quantise(w[k + 4], inv) << (8 * k);
      }
    }
    *reinterpret_cast<uint2*>(a.q + at) = make_uint2(lo, hi);
    if (a.out) {
      float y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = act_value(w[k], a.act, a.slope);
      store8(static_cast<T*>(a.out) + at, y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) act8_backward_kernel(const Act8 a) {
  const int t = threadIdx.x & 7;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;
  if (blk >= a.blocks) return;
  const long long row = blk / a.nblk;
  const int c0 = (int)(blk - row * a.nblk) * kBlock + t * 8;
  const float scale = __ldg(a.scale + blk);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + 64 * i;
    if (c >= a.cols) continue;
    const long long at = row * a.cols + c;
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(a.q + at));
    float g[8], y[8];
    if (a.in) load8(static_cast<const T*>(a.in) + row * a.in_stride + c, g);
    const uint32_t lo = q.x ^ 0x80808080u, hi = q.y ^ 0x80808080u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = dequantise(k < 4 ? lo : hi, k & 3) * scale;
      float d;
      act_both(x, a.act, a.slope, y[k], d);
      g[k] = a.in ? g[k] * d : 0.f;
    }
    if (a.out) store8(static_cast<T*>(a.out) + at, g);
    if (a.again) store8(static_cast<T*>(a.again) + at, y);
  }
}

// Rows whose length, stride or address rules out 16-byte pieces: a warp owns a block, 4 values a lane.
template <typename T>
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
  block_scale(top, inv, scale);
  if (lane == 0) a.scale[blk] = scale;
  const bool bad = top >= 0x7F800000u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c0 + 32 * i >= a.cols) continue;
    const long long at = row * a.cols + c0 + 32 * i;
    a.q[at] = bad ? (signed char)0 : (signed char)quantise(v[i], inv);
    if (a.out) static_cast<T*>(a.out)[at] = from_float<T>(act_value(v[i], a.act, a.slope));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) act8_backward_any_kernel(const Act8 a) {
  const int lane = threadIdx.x & 31;
  const long long blk = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (blk >= a.blocks) return;
  const long long row = blk / a.nblk;
  const int c0 = (int)(blk - row * a.nblk) * kBlock + lane;
  const float scale = a.scale[blk];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 32 * i;
    if (c >= a.cols) continue;
    const long long at = row * a.cols + c;
    float y, d;
    act_both((float)a.q[at] * scale, a.act, a.slope, y, d);
    if (a.out)
      static_cast<T*>(a.out)[at] =
          from_float<T>(to_float(static_cast<const T*>(a.in)[row * a.in_stride + c]) * d);
    if (a.again) static_cast<T*>(a.again)[at] = from_float<T>(y);
  }
}

// Everything but the pointers; 1 = nothing to do.
int check_act8(int dtype, int act, long long rows, int cols) {
  if (!ops_dtype_ok(dtype) || act < WUBU_B200_ACT_IDENTITY || act > WUBU_B200_ACT_SILU) return WUBU_B200_ERR_ARG;
  if (rows < 0 || cols < 0) return WUBU_B200_ERR_ARG;
  if (rows == 0 || cols == 0) return 1;
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
  Act8 a{act, slope, x, rows > 1 ? x_stride : 0, y, nullptr, q, scale, rows, 0, cols, (cols + kBlock - 1) / kBlock};
  a.blocks = rows * a.nblk;
  cudaStream_t st = (cudaStream_t)stream;
  const int per = whole_pieces(a) ? kThreads / 8 : kThreads / 32;
  const unsigned grid = (unsigned)((a.blocks + per - 1) / per);
  with_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (per == kThreads / 8) act8_forward_kernel<T><<<grid, kThreads, 0, st>>>(a);
    else act8_forward_any_kernel<T><<<grid, kThreads, 0, st>>>(a);
  });
  return ops_launched("act8_forward");
}

int wubu_b200_act8_backward(int dtype, int act, float slope, const void* dy, long long dy_stride, const signed char* q,
                            const float* scale, void* dx, void* y_again, long long rows, int cols, void* stream) {
  const int rc = check_act8(dtype, act, rows, cols);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  if (!q || !scale || !dy != !dx || (!dx && !y_again) || (dy && rows > 1 && dy_stride < cols)) return WUBU_B200_ERR_ARG;
  Act8 a{act, slope, dy, dy && rows > 1 ? dy_stride : 0, dx, y_again, const_cast<signed char*>(q),
         const_cast<float*>(scale), rows, 0, cols, (cols + kBlock - 1) / kBlock};
  a.blocks = rows * a.nblk;
  cudaStream_t st = (cudaStream_t)stream;
  const int per = whole_pieces(a) ? kThreads / 8 : kThreads / 32;
  const unsigned grid = (unsigned)((a.blocks + per - 1) / per);
  with_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (per == kThreads / 8) act8_backward_kernel<T><<<grid, kThreads, 0, st>>>(a);
    else act8_backward_any_kernel<T><<<grid, kThreads, 0, st>>>(a);
  });
  return ops_launched("act8_backward");
}

}  // extern "C"
