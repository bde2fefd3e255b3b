// resnorm.cu — the norms before and after a block fused with its gate and the residual scale:
//   u = post(f),  r = a x + gate * u,  h = norm(r)
// and the gradients of everything that goes in.  With n = (v - mean) / sigma (layer; the RMS form
// has no mean), y = w n + b and g = w dy, a norm's gradient is
//   dv = (g - mean(g) - n mean(g n)) / sigma        (no mean(g) in the RMS form)
//   dw = sum over rows of dy n,  db = sum over rows of dy.
// The backward recomputes both norms from x and f, so that the forward keeps no statistics.
//
// A group of threads owns a row and holds it in registers, 8 values a thread, so each tensor is read
// once and written once (bound by HBM).  In the backward a thread meets the same columns in every
// row of its block's range and sums the parameter gradients in registers; the blocks' partial sums
// are added in a fixed order by a second kernel.
#include "ops.cuh"

namespace wb {
namespace {

constexpr int kMaxCols = 8192;  // 1024 threads x 8 values

struct RowReduce {  // sums over a row's group of warps; four buffers in turn need one barrier a sum
  float2* buf;      // [4][rows][warps]
  int warps, rows, row, warp, lane, turn;
  WB_DEV float2 operator()(float a, float b) {
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, m);
      b += __shfl_xor_sync(0xffffffffu, b, m);
    }
    if (warps == 1) return make_float2(a, b);
    float2* mine = buf + (turn * rows + row) * warps;
    turn = (turn + 1) & 3;
    if (lane == 0) mine[warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int i = 0; i < warps; ++i) {
      a += mine[i].x;
      b += mine[i].y;
    }
    return make_float2(a, b);
  }
};

// A thread's 8 columns of a row: one run of 8 (VEC) or every G-th column from `tid`.
template <bool VEC>
struct Cols {
  int c, cols, G;
  WB_DEV int at(int k) const { return VEC ? c + k : c + k * G; }
  WB_DEV bool on(int k) const { return at(k) < cols; }
  template <typename T>
  WB_DEV void load(const T* p, float* v) const {
    if (VEC) {
      if (on(0)) load8(p + c, v);
      else
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = on(k) ? to_float(p[at(k)]) : 0.f;
    }
  }
  WB_DEV void vector(const float* p, float* v, float none) const {  // a parameter vector, or `none` without one
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = p && on(k) ? __ldg(p + at(k)) : none;
  }
  template <typename T>
  WB_DEV void store(T* p, const float* v) const {
    if (VEC) {
      if (on(0)) store8(p + c, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (on(k)) p[at(k)] = from_float<T>(v[k]);
    }
  }
};

// v <- (v - mean) / sigma in place; returns 1 / sigma.  The variance is taken from the centred values
// (a second sum), not as a difference of two large sums.
template <bool VEC>
WB_DEV float normalise(float* v, int kind, const Cols<VEC>& cc, float inv_cols, float eps, RowReduce& sum) {
  if (kind == WUBU_B200_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k];
    const float mean = sum(s, 0.f).x * inv_cols;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = cc.on(k) ? v[k] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) q += v[k] * v[k];
  const float inv = rsqrtf(sum(q, 0.f).x * inv_cols + eps);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] *= inv;
  return inv;
}

// g <- gradient of the normalised values n's source, for g = gradient of n
template <bool VEC>
WB_DEV void normalise_backward(float* g, const float* n, float inv, int kind, const Cols<VEC>& cc, float inv_cols,
                               RowReduce& sum) {
  float s = 0.f, p = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    s += g[k];
    p += g[k] * n[k];
  }
  const float2 t = sum(s, p);
  const float mg = kind == WUBU_B200_NORM_LAYER ? t.x * inv_cols : 0.f, mp = t.y * inv_cols;
#pragma unroll
  for (int k = 0; k < 8; ++k) g[k] = cc.on(k) ? (g[k] - mg - n[k] * mp) * inv : 0.f;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(1024) resnorm_forward_kernel(const WubuB200ResNorm a, long long rows) {
  extern __shared__ float2 red[];
  const int G = blockDim.x, R = blockDim.y;
  RowReduce sum{red, G / 32, R, (int)threadIdx.y, (int)threadIdx.x / 32, (int)threadIdx.x & 31, 0};
  const Cols<VEC> cc{VEC ? (int)threadIdx.x * 8 : (int)threadIdx.x, a.cols, G};
  const float inv_cols = 1.f / (float)a.cols;
  const long long row = (long long)blockIdx.x * R + threadIdx.y;
  const bool on = row < rows;
  const long long at = on ? row : rows - 1;  // the last block's idle groups repeat the last row, unstored
  float x[8], f[8], t[8];
  cc.load(static_cast<const T*>(a.x) + at * a.x_stride, x);
  cc.load(static_cast<const T*>(a.f) + at * a.f_stride, f);
  if (a.post) {
    normalise(f, a.post, cc, inv_cols, a.eps, sum);
    cc.vector(a.post_weight, t, 1.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= t[k];
    cc.vector(a.post_bias, t, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += t[k];
  }
  if (a.gate) {
    cc.vector(a.gate_values + (a.gate == WUBU_B200_GATE_ITEM ? at / a.rows_per_item * a.cols : 0), t, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= t[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = fmaf(a.res_scale, x[k], f[k]);
  if (a.r && on) cc.store(static_cast<T*>(a.r) + at * a.cols, x);
  if (!a.norm) return;
  normalise(x, a.norm, cc, inv_cols, a.eps, sum);
  cc.vector(a.weight, t, 1.f);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] *= t[k];
  cc.vector(a.bias, t, 0.f);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] += t[k];
  if (on) cc.store(static_cast<T*>(a.h) + at * a.cols, x);
}

// The column sums a block hands on, in this order; partials are [vector][block][cols].
enum { kDWeight, kDBias, kDPostWeight, kDPostBias, kDGate, kVectors };

struct ResNormGrid {
  int blocks_per_item, rows_per_block;
  long long blocks;
  float* part;
};

// MAXT: 256 threads may use all the registers that the sums and the row want; rows of more than 2048
// columns take up to 1024 threads.
template <typename T, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) resnorm_backward_kernel(const WubuB200ResNorm a, const ResNormGrid gr) {
  extern __shared__ float2 red[];
  const int G = blockDim.x, R = blockDim.y;
  RowReduce sum{red, G / 32, R, (int)threadIdx.y, (int)threadIdx.x / 32, (int)threadIdx.x & 31, 0};
  const Cols<VEC> cc{VEC ? (int)threadIdx.x * 8 : (int)threadIdx.x, a.cols, G};
  const float inv_cols = 1.f / (float)a.cols;
  const long long item = blockIdx.x / gr.blocks_per_item;
  const long long t0 = (long long)(blockIdx.x - item * gr.blocks_per_item) * gr.rows_per_block;
  const long long t1 = min(t0 + gr.rows_per_block, a.rows_per_item);
  const float* gate = a.gate ? a.gate_values + (a.gate == WUBU_B200_GATE_ITEM ? item * a.cols : 0) : nullptr;
  float dw[8], db[8], dpw[8], dpb[8], dg[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) dw[k] = db[k] = dpw[k] = dpb[k] = dg[k] = 0.f;
  for (long long t = t0; t < t1; t += R) {  // the same count for all groups of the block (barriers inside)
    const bool on = t + threadIdx.y < t1;
    const long long row = item * a.rows_per_item + (on ? t + threadIdx.y : t);
    float x[8], n[8], d[8], g[8], v[8];
    cc.load(static_cast<const T*>(a.x) + row * a.x_stride, x);
    cc.load(static_cast<const T*>(a.f) + row * a.f_stride, n);
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k] = g[k] = 0.f;
    if (a.dr) cc.load(static_cast<const T*>(a.dr) + row * a.dr_stride, d);
    if (a.dh) cc.load(static_cast<const T*>(a.dh) + row * a.dh_stride, g);
    // forward again: n = normalised f, u = its affine form, x <- r <- normalised r
    const float post_inv = a.post ? normalise(n, a.post, cc, inv_cols, a.eps, sum) : 1.f;
    float u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = n[k];
    if (a.post) {
      cc.vector(a.post_weight, v, 1.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] *= v[k];
      cc.vector(a.post_bias, v, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] += v[k];
    }
    cc.vector(gate, v, 1.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = fmaf(a.res_scale, x[k], v[k] * u[k]);
    // d <- gradient of r
    if (a.norm && a.dh) {
      const float inv = normalise(x, a.norm, cc, inv_cols, a.eps, sum);
      float w[8];
      cc.vector(a.weight, w, 1.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (on) {
          dw[k] += g[k] * x[k];
          db[k] += g[k];
        }
        g[k] *= w[k];
      }
      normalise_backward(g, x, inv, a.norm, cc, inv_cols, sum);
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] += g[k];
    }
    // x <- dx, d <- gradient of u
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = a.res_scale * d[k];
      if (on) dg[k] += d[k] * u[k];
      d[k] *= v[k];
    }
    if (a.dx && on) cc.store(static_cast<T*>(a.dx) + row * a.cols, x);
    if (a.post) {
      cc.vector(a.post_weight, v, 1.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (on) {
          dpw[k] += d[k] * n[k];
          dpb[k] += d[k];
        }
        d[k] *= v[k];
      }
      normalise_backward(d, n, post_inv, a.post, cc, inv_cols, sum);
    }
    if (a.df && on) cc.store(static_cast<T*>(a.df) + row * a.cols, d);
  }
  // the block's R groups in order, then one partial row per block
  float* acc = reinterpret_cast<float*>(red);
  const float* mine[kVectors] = {dw, db, dpw, dpb, dg};
  float* const want[kVectors] = {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dgate};
#pragma unroll
  for (int q = 0; q < kVectors; ++q) {
    if (!want[q]) continue;
    float* part = gr.part + ((long long)q * gr.blocks + blockIdx.x) * a.cols;
    if (R > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (cc.on(k)) acc[threadIdx.y * a.cols + cc.at(k)] = mine[q][k];
      __syncthreads();
      for (int c = threadIdx.y * G + threadIdx.x; c < a.cols; c += G * R) {
        float s = 0.f;
        for (int r = 0; r < R; ++r) s += acc[r * a.cols + c];
        part[c] = s;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (cc.on(k)) part[cc.at(k)] = mine[q][k];
    }
  }
}

// out[item][c] = sum over `n` partial rows from item * n on, in order (8 threads a column, each a run of
// rows, then the 8 in order).
constexpr int kReduceCols = 32, kReduceRuns = 8;
struct ColumnSums {
  const float* part[kVectors];
  float* out[kVectors];
  long long n[kVectors];
  int items[kVectors];
};
__global__ void __launch_bounds__(kReduceCols* kReduceRuns) resnorm_sums_kernel(const ColumnSums s, int cols) {
  __shared__ float run[kReduceRuns][kReduceCols];
  const int q = blockIdx.z;
  if ((int)blockIdx.y >= s.items[q]) return;
  const int c = blockIdx.x * kReduceCols + threadIdx.x;
  const long long n = s.n[q], per = (n + kReduceRuns - 1) / kReduceRuns;
  const long long i0 = min(n, per * threadIdx.y), i1 = min(n, i0 + per);
  const float* p = s.part[q] + (long long)blockIdx.y * n * cols + c;
  float acc = 0.f;
  if (c < cols)
    for (long long i = i0; i < i1; ++i) acc += p[i * cols];
  run[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y || c >= cols) return;
  acc = 0.f;
#pragma unroll
  for (int i = 0; i < kReduceRuns; ++i) acc += run[i][threadIdx.x];
  s.out[q][(long long)blockIdx.y * cols + c] = acc;
}

bool strides_ok(const WubuB200ResNorm& a, long long stride, const void* p) {
  return !p || a.items * a.rows_per_item <= 1 || stride >= a.cols;
}

// 1 = nothing to do
int check_resnorm(const WubuB200ResNorm* a) {
  if (!a || !ops_dtype_ok(a->dtype) || a->norm < 0 || a->norm > WUBU_B200_NORM_RMS || a->post < 0 ||
      a->post > WUBU_B200_NORM_RMS || a->gate < 0 || a->gate > WUBU_B200_GATE_ITEM || a->items < 0 ||
      a->rows_per_item < 0 || !(a->eps >= 0.f))
    return WUBU_B200_ERR_ARG;
  if (a->cols < 1 || a->cols > kMaxCols) return WUBU_B200_ERR_SHAPE;
  if (a->items == 0 || a->rows_per_item == 0) return 1;
  if (a->rows_per_item > 0x7FFFFFFFll / a->items || (a->gate == WUBU_B200_GATE_ITEM && a->items > 65535))
    return WUBU_B200_ERR_SHAPE;
  if (!a->x || !a->f || (a->gate && !a->gate_values) || !strides_ok(*a, a->x_stride, a->x) ||
      !strides_ok(*a, a->f_stride, a->f))
    return WUBU_B200_ERR_ARG;
  return WUBU_B200_OK;
}

bool vec_ok(const WubuB200ResNorm& a, const void* p, long long stride) { return aligned16(p) && stride % 8 == 0; }

// threads a row (a multiple of 32), rows at a time
dim3 group_of(int cols) {
  const int G = (((cols + 7) / 8) + 31) / 32 * 32;
  return dim3(G, G >= 128 ? 1 : 128 / G);
}

// Row ranges of the backward's blocks: enough blocks to fill the SMs several times over, few enough
// that their partial sums stay small beside the tensors.
ResNormGrid grid_of(const WubuB200ResNorm& a, const dim3& g) {
  const long long want = 148 * 4;
  ResNormGrid r{};
  long long per_item = (want + a.items - 1) / a.items;
  const long long most = (a.rows_per_item + g.y - 1) / g.y;
  per_item = per_item < 1 ? 1 : per_item > most ? most : per_item;
  long long rows = (a.rows_per_item + per_item - 1) / per_item;
  rows = (rows + g.y - 1) / g.y * g.y;
  r.rows_per_block = (int)rows;
  r.blocks_per_item = (int)((a.rows_per_item + rows - 1) / rows);
  r.blocks = r.blocks_per_item * a.items;
  return r;
}

size_t reduce_bytes(const dim3& g) { return sizeof(float2) * 4 * g.y * (g.x / 32); }

}  // namespace
}  // namespace wb

using namespace wb;

extern "C" {

int wubu_b200_resnorm_forward(const WubuB200ResNorm* p, void* stream) {
  const int rc = check_resnorm(p);
  if (rc != WUBU_B200_OK) return rc == 1 ? WUBU_B200_OK : rc;
  WubuB200ResNorm a = *p;
  if (!a.norm != !a.h || (!a.r && !a.h)) return WUBU_B200_ERR_ARG;
  const long long rows = a.items * a.rows_per_item;
  if (rows == 1) a.x_stride = a.f_stride = 0;
  const bool vec = a.cols % 8 == 0 && vec_ok(a, a.x, a.x_stride) && vec_ok(a, a.f, a.f_stride) && aligned16(a.r) &&
                   aligned16(a.h);
  const dim3 g = group_of(a.cols);
  const unsigned grid = (unsigned)((rows + g.y - 1) / g.y);
  cudaStream_t st = (cudaStream_t)stream;
  with_dtype(a.dtype, [&](auto t) {
    typedef decltype(t) T;
    if (vec) resnorm_forward_kernel<T, true><<<grid, g, reduce_bytes(g), st>>>(a, rows);
    else resnorm_forward_kernel<T, false><<<grid, g, reduce_bytes(g), st>>>(a, rows);
  });
  return ops_launched("resnorm_forward");
}

long long wubu_b200_resnorm_workspace(const WubuB200ResNorm* a) {
  const int rc = check_resnorm(a);
  if (rc != WUBU_B200_OK) return rc == 1 ? 0 : rc;
  return grid_of(*a, group_of(a->cols)).blocks * kVectors * a->cols * (long long)sizeof(float);
}

int wubu_b200_resnorm_backward(const WubuB200ResNorm* p, void* stream) {
  int rc = check_resnorm(p);
  cudaStream_t st = (cudaStream_t)stream;
  if (rc < 0) return rc;
  WubuB200ResNorm a = *p;
  float* const out[kVectors] = {a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dgate};
  if (rc == 1) {  // no rows: the sums over them are zero
    for (int q = 0; q < kVectors; ++q) {
      const long long n = q == kDGate && a.gate == WUBU_B200_GATE_ITEM ? a.items * a.cols : a.cols;
      if (out[q] && n && cudaMemsetAsync(out[q], 0, n * sizeof(float), st) != cudaSuccess) return WUBU_B200_ERR_CUDA;
    }
    return WUBU_B200_OK;
  }
  if ((a.dh && !a.norm) || (a.dgate && !a.gate) || ((a.dweight || a.dbias) && !a.norm) ||
      ((a.dpost_weight || a.dpost_bias) && !a.post) || !strides_ok(a, a.dr_stride, a.dr) ||
      !strides_ok(a, a.dh_stride, a.dh))
    return WUBU_B200_ERR_ARG;
  const dim3 g = group_of(a.cols);
  ResNormGrid gr = grid_of(a, g);
  bool sums = false;
  for (int q = 0; q < kVectors; ++q) sums = sums || out[q];
  if (sums) {
    if (!a.workspace) return WUBU_B200_ERR_ARG;
    if (a.workspace_bytes < gr.blocks * kVectors * a.cols * (long long)sizeof(float)) return WUBU_B200_ERR_NOMEM;
    gr.part = static_cast<float*>(a.workspace);
  }
  if (a.items * a.rows_per_item == 1) a.x_stride = a.f_stride = a.dr_stride = a.dh_stride = 0;
  const bool vec = a.cols % 8 == 0 && vec_ok(a, a.x, a.x_stride) && vec_ok(a, a.f, a.f_stride) &&
                   (!a.dr || vec_ok(a, a.dr, a.dr_stride)) && (!a.dh || vec_ok(a, a.dh, a.dh_stride)) &&
                   aligned16(a.dx) && aligned16(a.df);
  size_t smem = reduce_bytes(g);
  if (g.y > 1 && smem < sizeof(float) * g.y * a.cols) smem = sizeof(float) * g.y * a.cols;
  with_dtype(a.dtype, [&](auto t) {
    typedef decltype(t) T;
    auto* kernel = g.x <= 256 ? (vec ? resnorm_backward_kernel<T, true, 256> : resnorm_backward_kernel<T, false, 256>)
                              : (vec ? resnorm_backward_kernel<T, true, 1024> : resnorm_backward_kernel<T, false, 1024>);
    kernel<<<(unsigned)gr.blocks, g, smem, st>>>(a, gr);
  });
  rc = ops_launched("resnorm_backward");
  if (rc != WUBU_B200_OK || !sums) return rc;
  ColumnSums s{};
  int items = 1;
  for (int q = 0; q < kVectors; ++q) {
    if (!out[q]) continue;
    const bool by_item = q == kDGate && a.gate == WUBU_B200_GATE_ITEM;
    s.part[q] = gr.part + (long long)q * gr.blocks * a.cols;
    s.out[q] = out[q];
    s.items[q] = by_item ? (int)a.items : 1;
    s.n[q] = by_item ? gr.blocks_per_item : gr.blocks;
    if (s.items[q] > items) items = s.items[q];
  }
  resnorm_sums_kernel<<<dim3((a.cols + kReduceCols - 1) / kReduceCols, items, kVectors), dim3(kReduceCols, kReduceRuns),
                        0, st>>>(s, a.cols);
  return ops_launched("resnorm_sums");
}

}  // extern "C"
