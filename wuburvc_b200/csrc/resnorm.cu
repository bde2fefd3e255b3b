// resnorm.cu — the norms before and after a block fused with its gate and the residual scale:
//   u = post(f),  r = a x + gate * u,  h = norm(r)
// and the gradients of everything that goes in.  With n = (v - mean) / sigma (layer; the RMS form
// has no mean), y = w n + b and g = w dy, a norm's gradient is
//   dv = (g - mean(g) - n mean(g n)) / sigma        (no mean(g) in the RMS form)
//   dw = sum over rows of dy n,  db = sum over rows of dy.
// The backward recomputes both norms from x and f, so that the forward keeps no statistics.
//
// A group of threads owns a row and holds it in registers, 8 values a thread, so each tensor is read
// once and written once.  A block runs several groups, each with a barrier of its own, over
// a range of one item's rows: the parameter vectors stay in registers, the next row is loaded before the
// current one's sums are taken, and in the backward a thread meets the same columns in every row and
// adds up the parameter gradients in registers; the blocks' partial sums are added in a fixed order by a
// second kernel.  Measured (B200): 7984 x 768 bf16, rms / gate / rms: forward 13.4 us (49 MB: 56 % of the
// measured copy rate), backward 30 + 6 us (74 MB); 6000 x 768 fp16 LayerNorm backward 18 + 5 us (46 MB).  The
// backward's rows are bound by the latency of their four sums: 12 warps an SM hold all the registers.  Rows of
// more than kThreads * 8 columns have 64 registers a thread and spill in the backward: 4096 rows of 4000 bf16,
// LayerNorm, 52 us forward (98 MB), 200 backward (164 MB), against 23 and 60 at 3000 columns.
// A mean is a sum times 1 / cols, and a gate is multiplied into the affine weights before they meet a row: each is off by
// an ulp of float32 from the formula's order, which shows in float32 results alone.
#include <type_traits>

#include "ops.cuh"

namespace wb {
namespace {

constexpr int kMaxCols = 8192;   // 1024 threads x 8 values
constexpr int kThreads = 384;    // threads a block, where a row needs no more
// Rows are numbered in 32 bits: up to 12 are added to a number within the range (as many as a block takes at a time).
constexpr long long kMaxRows = 0x7FFFFFFFll - 32;

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
    asm volatile("bar.sync %0, %1;" ::"r"(row + 1), "r"(warps * 32) : "memory");
    a = mine[0].x + mine[1].x;
    b = mine[0].y + mine[1].y;
    if (warps > 2) {
      a += mine[2].x;
      b += mine[2].y;
    }
    for (int i = 3; i < warps; ++i) {
      a += mine[i].x;
      b += mine[i].y;
    }
    return make_float2(a, b);
  }
  WB_DEV float operator()(float a) {
#pragma unroll
    for (int m = 16; m; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
    if (warps == 1) return a;
    float2* mine = buf + (turn * rows + row) * warps;
    turn = (turn + 1) & 3;
    if (lane == 0) mine[warp].x = a;
    asm volatile("bar.sync %0, %1;" ::"r"(row + 1), "r"(warps * 32) : "memory");
    a = mine[0].x + mine[1].x;
    if (warps > 2) a += mine[2].x;
    for (int i = 3; i < warps; ++i) a += mine[i].x;
    return a;
  }
};

// 8 values as they lie in memory
template <typename T>
struct Raw {
  uint4 a[sizeof(T) / 2];
};

// A thread's 8 columns of a row: one run of 8 (VEC) or every G-th column from `tid`.
template <bool VEC>
struct Cols {
  int c, cols, G;
  bool any;  // c < cols; with VEC that goes for all 8 (cols is a multiple of 8)
  WB_DEV Cols(int tid, int cols_, int G_) : c(VEC ? tid * 8 : tid), cols(cols_), G(G_), any(c < cols_) {}
  WB_DEV int at(int k) const { return VEC ? c + k : c + k * G; }
  WB_DEV bool on(int k) const { return VEC ? any : at(k) < cols; }
  template <typename T>
  WB_DEV void fetch(const T* p, Raw<T>& r) const {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        r.a[i] = on(0) ? __ldg(reinterpret_cast<const uint4*>(p + c) + i) : make_uint4(0, 0, 0, 0);
    } else {
      T* v = reinterpret_cast<T*>(r.a);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = on(k) ? p[at(k)] : from_float<T>(0.f);
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
template <typename T>
WB_DEV void widen(const Raw<T>& r, float* v) {
  const T* p = reinterpret_cast<const T*>(r.a);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = to_float(p[k]);
}

// v <- (v - mean) / sigma in place; returns 1 / sigma.  The variance is taken from the centred values
// (a second sum), not as a difference of two large sums.
template <bool VEC>
WB_DEV float normalise(float* v, int kind, const Cols<VEC>& cc, float inv_cols, float eps, RowReduce& sum) {
  if (kind == WUBU_B200_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k];
    const float mean = sum(s) * inv_cols;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = cc.on(k) ? v[k] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) q += v[k] * v[k];
  const float inv = rsqrtf(sum(q) * inv_cols + eps);
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
  const float2 t = kind == WUBU_B200_NORM_LAYER ? sum(s, p) : make_float2(0.f, sum(p));
  const float mg = t.x * inv_cols, mp = t.y * inv_cols;
#pragma unroll
  for (int k = 0; k < 8; ++k) g[k] = cc.on(k) ? (g[k] - mg - n[k] * mp) * inv : 0.f;
}

// A block's rows [t0, t1) of one item.
struct ResNormGrid {
  int blocks_per_item, rows_per_block;
  long long blocks;
  float* part;
};

// MAXT: rows of more than kThreads * 8 columns take up to 1024 threads.
template <typename T, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == kThreads ? 2 : 1)
resnorm_forward_kernel(const WubuB200ResNorm a, const ResNormGrid gr) {
  extern __shared__ float2 red[];
  const int G = blockDim.x, R = blockDim.y;
  RowReduce sum{red, G / 32, R, (int)threadIdx.y, (int)threadIdx.x / 32, (int)threadIdx.x & 31, 0};
  const Cols<VEC> cc((int)threadIdx.x, a.cols, G);
  const float inv_cols = 1.f / (float)a.cols;
  const int item = blockIdx.x / gr.blocks_per_item;
  const int t0 = (int)(blockIdx.x - item * gr.blocks_per_item) * gr.rows_per_block + threadIdx.y;
  const int t1 = (int)min((long long)t0 - threadIdx.y + gr.rows_per_block, a.rows_per_item);
  const long long row0 = item * a.rows_per_item;
  // the next row to load, and the next to store
  const T *xp = static_cast<const T*>(a.x) + (row0 + t0) * a.x_stride,
          *fp = static_cast<const T*>(a.f) + (row0 + t0) * a.f_stride;
  const long long xs = R * a.x_stride, fs = R * a.f_stride, os = (long long)R * a.cols;
  T *rp = static_cast<T*>(a.r) + (row0 + t0) * a.cols, *hp = static_cast<T*>(a.h) + (row0 + t0) * a.cols;
  Raw<T> rx, rf;
  if (t0 < t1) {
    cc.fetch(xp, rx);
    cc.fetch(fp, rf);
  }
  float w[8], wb_[8], pw[8], pb[8];
  cc.vector(a.weight, w, 1.f);
  cc.vector(a.bias, wb_, 0.f);
  cc.vector(a.post_weight, pw, 1.f);
  cc.vector(a.post_bias, pb, 0.f);
  if (a.gate) {  // folded into the affine form: gate * (n pw + pb)
    float gt[8];
    cc.vector(a.gate_values + (a.gate == WUBU_B200_GATE_ITEM ? (long long)item * a.cols : 0), gt, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      pw[k] *= gt[k];
      pb[k] *= gt[k];
    }
  }
  for (int t = t0; t < t1; t += R, rp += os, hp += os) {
    float x[8], f[8];
    widen(rx, x);
    widen(rf, f);
    if (t + R < t1) {
      cc.fetch(xp += xs, rx);
      cc.fetch(fp += fs, rf);
    }
    if (a.post) normalise(f, a.post, cc, inv_cols, a.eps, sum);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = fmaf(a.res_scale, x[k], fmaf(f[k], pw[k], pb[k]));
    if (a.r) cc.store(rp, x);
    if (!a.norm) continue;
    normalise(x, a.norm, cc, inv_cols, a.eps, sum);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = fmaf(x[k], w[k], wb_[k]);
    cc.store(hp, x);
  }
}

// The column sums a block hands on, in this order; partials are [vector][block][cols].
enum { kDWeight, kDBias, kDPostWeight, kDPostBias, kDGate, kVectors };

// POST, GATE: without a post norm or a gate their vectors and sums take no registers (true also serves
// their absence).
template <typename T, bool VEC, int MAXT, bool POST, bool GATE>
__global__ void __launch_bounds__(MAXT, 1) resnorm_backward_kernel(const WubuB200ResNorm a, const ResNormGrid gr) {
  extern __shared__ float2 red[];
  const int G = blockDim.x, R = blockDim.y;
  RowReduce sum{red, G / 32, R, (int)threadIdx.y, (int)threadIdx.x / 32, (int)threadIdx.x & 31, 0};
  const Cols<VEC> cc((int)threadIdx.x, a.cols, G);
  const float inv_cols = 1.f / (float)a.cols;
  const int item = blockIdx.x / gr.blocks_per_item;
  const int t0 = (int)(blockIdx.x - item * gr.blocks_per_item) * gr.rows_per_block + threadIdx.y;
  const int t1 = (int)min((long long)t0 - threadIdx.y + gr.rows_per_block, a.rows_per_item);
  const long long row0 = item * a.rows_per_item;
  const T *xp = static_cast<const T*>(a.x) + (row0 + t0) * a.x_stride,
          *fp = static_cast<const T*>(a.f) + (row0 + t0) * a.f_stride,
          *dp = static_cast<const T*>(a.dr) + (row0 + t0) * a.dr_stride,
          *hp = static_cast<const T*>(a.dh) + (row0 + t0) * a.dh_stride;
  T *dxp = static_cast<T*>(a.dx) + (row0 + t0) * a.cols, *dfp = static_cast<T*>(a.df) + (row0 + t0) * a.cols;
  const bool norm = a.norm && a.dh;
  Raw<T> rx, rf, rd, rh;
  auto fetch = [&] {  // the row at the pointers, which move on
    cc.fetch(xp, rx);
    cc.fetch(fp, rf);
    if (a.dr) cc.fetch(dp, rd);
    if (a.dh) cc.fetch(hp, rh);
    xp += R * a.x_stride;
    fp += R * a.f_stride;
    dp += R * a.dr_stride;
    hp += R * a.dh_stride;
  };
  if (t0 < t1) fetch();
  float w[8], pw[8], pb[8], gt[8];
  cc.vector(a.weight, w, 1.f);
  if (POST) {
    cc.vector(a.post_weight, pw, 1.f);
    cc.vector(a.post_bias, pb, 0.f);
  }
  if (GATE) cc.vector(a.gate ? a.gate_values + (a.gate == WUBU_B200_GATE_ITEM ? (long long)item * a.cols : 0) : nullptr, gt, 1.f);
  float dw[8], db[8], dpw[8], dpb[8], dg[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) dw[k] = db[k] = dpw[k] = dpb[k] = dg[k] = 0.f;
  for (int t = t0; t < t1; t += R, dxp += (long long)R * a.cols, dfp += (long long)R * a.cols) {
    float x[8], n[8], d[8], g[8];
    widen(rx, x);
    widen(rf, n);
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k] = g[k] = 0.f;
    if (a.dr) widen(rd, d);
    if (a.dh) widen(rh, g);
    if (t + R < t1) fetch();
    // forward again: n = normalised f, x <- r <- normalised r
    const float post_inv = POST && a.post ? normalise(n, a.post, cc, inv_cols, a.eps, sum) : 1.f;
    auto u = [&](int k) { return POST ? fmaf(n[k], pw[k], pb[k]) : n[k]; };
    // d <- gradient of r
    if (norm) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = fmaf(a.res_scale, x[k], GATE ? gt[k] * u(k) : u(k));
      const float inv = normalise(x, a.norm, cc, inv_cols, a.eps, sum);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        dw[k] += g[k] * x[k];
        db[k] += g[k];
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
      if (GATE) {
        dg[k] += d[k] * u(k);
        d[k] *= gt[k];
      }
    }
    if (a.dx) cc.store(dxp, x);
    if (POST && a.post) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        dpw[k] += d[k] * n[k];
        dpb[k] += d[k];
        d[k] *= pw[k];
      }
      normalise_backward(d, n, post_inv, a.post, cc, inv_cols, sum);
    }
    if (a.df) cc.store(dfp, d);
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

// out[c] = sum over n partial rows, in order: 8 threads a column, each a run of rows, then the 8 in order.
// blockIdx.y counts the sums that are asked for, the gate's one to an item.
constexpr int kReduceCols = 32, kReduceRuns = 8;
struct ColumnSums {
  const float* part[kVectors];
  float* out[kVectors];
  int n[kVectors];
  int count;  // sums before the last entry, which holds the items' gates
};
__global__ void __launch_bounds__(kReduceCols* kReduceRuns) resnorm_sums_kernel(const ColumnSums s, int cols) {
  __shared__ float run[kReduceRuns][kReduceCols];
  griddep_wait();
  const int q = min((int)blockIdx.y, s.count), item = blockIdx.y - q;
  const int c = blockIdx.x * kReduceCols + threadIdx.x;
  const int n = s.n[q], per = (n + kReduceRuns - 1) / kReduceRuns;
  const int i0 = min(n, per * (int)threadIdx.y), i1 = min(n, i0 + per);
  const float* p = s.part[q] + (long long)item * n * cols + c;
  float acc = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int i = i0; i < i1; ++i) acc += __ldg(p + (long long)i * cols);
  }
  run[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y || c >= cols) return;
  acc = 0.f;
#pragma unroll
  for (int i = 0; i < kReduceRuns; ++i) acc += run[i][threadIdx.x];
  s.out[q][(long long)item * cols + c] = acc;
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
  if (a->rows_per_item > kMaxRows / a->items || (a->gate == WUBU_B200_GATE_ITEM && a->items > 65000))
    return WUBU_B200_ERR_SHAPE;
  if (!a->x || !a->f || (a->gate && !a->gate_values) || !strides_ok(*a, a->x_stride, a->x) ||
      !strides_ok(*a, a->f_stride, a->f))
    return WUBU_B200_ERR_ARG;
  return WUBU_B200_OK;
}

bool vec_ok(const WubuB200ResNorm& a, const void* p, long long stride) { return aligned16(p) && stride % 8 == 0; }

// Items matter to their gates alone: without such gates the rows are one item's, and the row ranges (and
// the partial sums, one row of them to a range) do not depend on how the rows were numbered.
WubuB200ResNorm as_ranges(const WubuB200ResNorm& in) {
  WubuB200ResNorm a = in;
  if (a.gate != WUBU_B200_GATE_ITEM) {
    a.rows_per_item *= a.items;
    a.items = 1;
  }
  return a;
}

// threads a row (a multiple of 32), rows at a time (a barrier each: at most 15)
dim3 group_of(int cols) {
  const int G = (((cols + 7) / 8) + 31) / 32 * 32;
  const int R = G >= kThreads ? 1 : kThreads / G;
  return dim3(G, R);
}

// Row ranges of the blocks: as many blocks as run at once (`resident` an SM), within an item.
ResNormGrid grid_of(const WubuB200ResNorm& a, const dim3& g, int resident) {
  const int sms = ops_sms();
  const long long want = (long long)(sms > 0 ? sms : 1) * resident;
  ResNormGrid r{};
  long long per_item = want / a.items;
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
  WubuB200ResNorm a = as_ranges(*p);
  if (!a.norm != !a.h || (!a.r && !a.h)) return WUBU_B200_ERR_ARG;
  const long long rows = a.items * a.rows_per_item;
  if (rows == 1) a.x_stride = a.f_stride = 0;
  const bool vec = a.cols % 8 == 0 && vec_ok(a, a.x, a.x_stride) && vec_ok(a, a.f, a.f_stride) && aligned16(a.r) &&
                   aligned16(a.h);
  const dim3 g = group_of(a.cols);
  const ResNormGrid gr = grid_of(a, g, g.x * g.y <= kThreads ? 2 : 1);
  const size_t smem = reduce_bytes(g);
  cudaStream_t st = (cudaStream_t)stream;
  with_dtype(a.dtype, [&](auto t) {
    typedef decltype(t) T;
    auto* kernel = g.x <= kThreads ? (vec ? resnorm_forward_kernel<T, true, kThreads> : resnorm_forward_kernel<T, false, kThreads>)
                                   : (vec ? resnorm_forward_kernel<T, true, 1024> : resnorm_forward_kernel<T, false, 1024>);
    kernel<<<(unsigned)gr.blocks, g, smem, st>>>(a, gr);
  });
  return ops_launched("resnorm_forward");
}

long long wubu_b200_resnorm_workspace(const WubuB200ResNorm* a) {
  const int rc = check_resnorm(a);
  if (rc != WUBU_B200_OK) return rc == 1 ? 0 : rc;
  return grid_of(as_ranges(*a), group_of(a->cols), 1).blocks * kVectors * a->cols * (long long)sizeof(float);
}

int wubu_b200_resnorm_backward(const WubuB200ResNorm* p, void* stream) {
  int rc = check_resnorm(p);
  cudaStream_t st = (cudaStream_t)stream;
  if (rc < 0) return rc;
  WubuB200ResNorm a = rc == 1 ? *p : as_ranges(*p);
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
  ResNormGrid gr = grid_of(a, g, 1);
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
    auto pick = [&](auto v) {
      constexpr bool V = decltype(v)::value;
      if (g.x > kThreads) return resnorm_backward_kernel<T, V, 1024, true, true>;  // (gate and post may be absent)
      if (a.post) return a.gate ? resnorm_backward_kernel<T, V, kThreads, true, true> : resnorm_backward_kernel<T, V, kThreads, true, false>;
      return a.gate ? resnorm_backward_kernel<T, V, kThreads, false, true> : resnorm_backward_kernel<T, V, kThreads, false, false>;
    };
    auto* kernel = vec ? pick(std::true_type()) : pick(std::false_type());
    kernel<<<(unsigned)gr.blocks, g, smem, st>>>(a, gr);
  });
  rc = ops_launched("resnorm_backward");
  if (rc != WUBU_B200_OK || !sums) return rc;
  ColumnSums s{};
  int k = 0, sums_y = 0;
  for (int q = 0; q < kVectors; ++q) {  // the gate's comes last
    if (!out[q]) continue;
    const bool by_item = q == kDGate && a.gate == WUBU_B200_GATE_ITEM;
    s.part[k] = gr.part + (long long)q * gr.blocks * a.cols;
    s.out[k] = out[q];
    s.n[k] = by_item ? gr.blocks_per_item : (int)gr.blocks;
    s.count = k++;
    sums_y += by_item ? (int)a.items : 1;
  }
  return ops_launch_after(resnorm_sums_kernel, dim3((a.cols + kReduceCols - 1) / kReduceCols, sums_y),
                          dim3(kReduceCols, kReduceRuns), 0, st, "resnorm_sums", s, a.cols);
}

}  // extern "C"
