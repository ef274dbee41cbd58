// Group norm with an activation on channels-last maps, y = act(xh gamma + beta), xh = (x - mean) rstd over the
// S rows and C / G channels of a (sample, group), and its backward pass
//   dz = dy act'(z);  d_beta = sum dz;  d_gamma = sum dz xh;
//   dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh)).
//
// Bound by memory in the statistics and in fp32, by the activation's vector instructions in 16 bits.  Two forms:
//  * one block per (sample, group) that keeps the whole group in registers (x read once, y written once): one launch,
//    for groups of up to kHeld vectors a thread whose row segments are at least 32 bytes;
//  * chunks of rows: one pass writes sums per (sample, chunk, group), a second folds the sums of its sample and
//    writes y.  The second pass takes the chunks in the opposite order, so that what the first read last is still in
//    the 256 MB memory-side cache.  14 x 65536 rows of 256 in bf16 (470 MB), 32 groups, gelu: sums 132 us (3.6 TB/s),
//    y 209 (166 of them its 22 vector instructions an element, two transcendental), gradient's sums 257 (29 an element:
//    208), dx 275 (29: 211).  Passing a few samples at a time
//    through both passes, all of them from the cache, took 1716 us: launches that small do not fill the memory.
// Sums over x and x^2 are held in 64 bits: E[x^2] - mean^2 then needs no pivot, whatever the mean is, and the double
// adds hide under the loads.  The backward's sums are fp32 within a thread (at most 256 rows) and 64 bits across threads and
// chunks, whose sums are rounded to fp32 once each.  Every sum has a fixed order: results repeat bit for bit.
#include "elem.h"
#include "pixelsplat_ops.h"

namespace ps {
namespace {

constexpr int kThreads = 256;
constexpr int kHeldForward = 8;    // 16-byte vectors of x a thread keeps in the one-launch form
constexpr int kHeldBackward = 4;   // of x and of dy

struct Rows {                      // [n][s][c] with unit channel stride
  int64_t sample, row;
};

struct Shape {
  int n, s, c, groups, cg;
  float eps;
  int act, param_f32;
};

__device__ __forceinline__ double2 wave_sum(double2 v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    v.x += __shfl_xor(v.x, m);
    v.y += __shfl_xor(v.y, m);
  }
  return v;
}

// sum over the block's threads, known to all of them; lds holds one double2 per wave
__device__ __forceinline__ double2 block_sum(double2 v, double2* lds) {
  v = wave_sum(v);
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double2 t = lds[0];
  for (int w = 1; w < waves; ++w) t = t + lds[w];
  __syncthreads();
  return t;
}

__device__ __forceinline__ void moments(double2 sums, double count, float eps, float& mean, float& rstd) {
  const double m = sums.x / count;
  const double var = sums.y / count - m * m;
  mean = (float)m;
  rstd = (float)(1.0 / sqrt((var > 0.0 ? var : (var == var ? 0.0 : var)) + (double)eps));
}

template <typename T> constexpr bool exact_act() { return sizeof(T) == 4; }

// ---------------------------------------------------------------------------------------------------------------
// one launch: a block holds the (sample, group) in registers
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int V, int HELD>
__global__ void __launch_bounds__(1024) group_norm_held_forward_kernel(
    Shape sh, const T* __restrict__ x, Rows rx, const void* __restrict__ gamma, const void* __restrict__ beta,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ double2 lds[16];
  const int g = blockIdx.x, n = blockIdx.y, at = n * sh.groups + g;
  const int per_row = sh.cg / V, count = sh.s * per_row;
  const T* xg = x + n * rx.sample + (int64_t)g * sh.cg;
  T* yg = y + ((int64_t)n * sh.s * sh.groups + g) * sh.cg;
  Pack<T, V> held[HELD];
  double2 sum = make_double2(0, 0);
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    if (i < count) held[j] = *reinterpret_cast<const Pack<T, V>*>(xg + (i / per_row) * rx.row + (i % per_row) * V);
  }
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    if ((int)(threadIdx.x + j * blockDim.x) < count) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double v = to_f32(held[j].v[e]);
        sum.x += v;
        sum.y = fma(v, v, sum.y);
      }
    }
  }
  float mean, rstd;
  moments(block_sum(sum, lds), (double)sh.s * sh.cg, sh.eps, mean, rstd);
  if (threadIdx.x == 0) {
    mean_out[at] = mean;
    rstd_out[at] = rstd;
  }
  with_act(sh.act, [&](auto tag) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = threadIdx.x + j * blockDim.x;
      if (i < count) {
        const int ch = (i % per_row) * V;
        Pack<T, V> out;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = g * sh.cg + ch + e;
          const float ga = gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f;
          const float be = beta ? load_param<T>(beta, sh.param_f32, c) : 0.f;
          out.v[e] = from_f32<T>(act_value<decltype(tag)::act, exact_act<T>()>(fmaf((to_f32(held[j].v[e]) - mean) * rstd, ga, be)));
        }
        *reinterpret_cast<Pack<T, V>*>(yg + (int64_t)(i / per_row) * sh.c + ch) = out;
      }
    }
  });
}

// blockDim.x is a multiple of the vectors per row: a thread's channels are the same in all its rows.
// partial: [n][2][c] (d_beta | d_gamma of the sample)
template <typename T, int V, int HELD>
__global__ void __launch_bounds__(1024) group_norm_held_backward_kernel(
    Shape sh, const T* __restrict__ x, Rows rx, const T* __restrict__ dy, Rows rdy, const void* __restrict__ gamma,
    const void* __restrict__ beta, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
    T* __restrict__ dx, float* __restrict__ partial) {
  extern __shared__ float chan[];                     // [rows in flight][2][cg]
  __shared__ double2 lds[16];
  const int g = blockIdx.x, n = blockIdx.y, at = n * sh.groups + g;
  const int per_row = sh.cg / V, count = sh.s * per_row;
  const int col = (threadIdx.x % per_row) * V, row0 = threadIdx.x / per_row, step = blockDim.x / per_row;
  const T* xg = x + n * rx.sample + (int64_t)g * sh.cg + col;
  const T* dyg = dy + n * rdy.sample + (int64_t)g * sh.cg + col;
  T* dxg = dx + ((int64_t)n * sh.s * sh.groups + g) * sh.cg + col;
  Pack<T, V> hx[HELD], hd[HELD];
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    if ((int)(threadIdx.x + j * blockDim.x) < count) {
      hx[j] = *reinterpret_cast<const Pack<T, V>*>(xg + (row0 + j * step) * rx.row);
      hd[j] = *reinterpret_cast<const Pack<T, V>*>(dyg + (row0 + j * step) * rdy.row);
    }
  }
  const float mean = mean_in[at], rstd = rstd_in[at];
  float ga[V], be[V], sb[V], sg[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = g * sh.cg + col + e;
    ga[e] = gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f;
    be[e] = beta ? load_param<T>(beta, sh.param_f32, c) : 0.f;
    sb[e] = sg[e] = 0.f;
  }
  float dz[HELD][V];
  with_act(sh.act, [&](auto tag) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if ((int)(threadIdx.x + j * blockDim.x) < count) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = (to_f32(hx[j].v[e]) - mean) * rstd;
          float value;
          const float d = to_f32(hd[j].v[e]) * act_slope<decltype(tag)::act, exact_act<T>()>(fmaf(xh, ga[e], be[e]), &value);
          dz[j][e] = d;
          sb[e] += d;
          sg[e] = fmaf(d, xh, sg[e]);
        }
      }
    }
  });
  double2 sum = make_double2(0, 0);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sum.x += (double)ga[e] * sb[e];
    sum.y += (double)ga[e] * sg[e];
    chan[(row0 * 2 + 0) * sh.cg + col + e] = sb[e];
    chan[(row0 * 2 + 1) * sh.cg + col + e] = sg[e];
  }
  sum = block_sum(sum, lds);                          // (also the barrier for chan)
  const double inv = 1.0 / ((double)sh.s * sh.cg);
  const float m1 = (float)(sum.x * inv), m2 = (float)(sum.y * inv);
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    if ((int)(threadIdx.x + j * blockDim.x) < count) {
      Pack<T, V> out;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (to_f32(hx[j].v[e]) - mean) * rstd;
        out.v[e] = from_f32<T>(rstd * (fmaf(dz[j][e], ga[e], -m1) - xh * m2));
      }
      *reinterpret_cast<Pack<T, V>*>(dxg + (int64_t)(row0 + j * step) * sh.c) = out;
    }
  }
  for (int i = threadIdx.x; i < 2 * sh.cg; i += blockDim.x) {
    const int k = i / sh.cg, c = i % sh.cg;
    double t = 0;
    for (int r = 0; r < step; ++r) t += chan[(r * 2 + k) * sh.cg + c];
    partial[((int64_t)n * 2 + k) * sh.c + g * sh.cg + c] = (float)t;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// chunks of rows
// ---------------------------------------------------------------------------------------------------------------
// A block takes a chunk of rows of a block of at most 256 vectors of columns; thread t owns vector t % tc of the rows
// t / tc, t / tc + tr, ...  (tc vectors a row, tr = 256 / tc rows at a time).
struct Columns {
  int c0, nc, tc, tr, vec, row0;
  bool on;
  __device__ Columns(int c, int V, int block) {
    const int all = c / V;
    c0 = block * kThreads * V;
    tc = min(all - block * kThreads, kThreads);
    nc = tc * V;
    tr = kThreads / tc;
    vec = (threadIdx.x % tc) * V;
    row0 = threadIdx.x / tc;
    on = row0 < tr;
  }
};

// The rows of a chunk.  A sample may have up to 2^31 - 1: the end of the last chunk does not fit 32 bits, so rows are
// counted from the chunk's first.
struct Chunk {
  int64_t first;
  int count;
  __device__ Chunk(int s, int rows, int chunk) : first((int64_t)chunk * rows), count((int)min((int64_t)rows, s - first)) {}
};

// sums: [n][chunks * column blocks][groups] of (sum x, sum x^2)
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) group_norm_sums_kernel(Shape sh, int rows, const T* __restrict__ x, Rows rx,
                                                                  double2* __restrict__ sums) {
  __shared__ double2 lds[kThreads * V];
  const Columns q(sh.c, V, blockIdx.z);
  const Chunk k(sh.s, rows, blockIdx.x);
  const int n = blockIdx.y;
  double2 acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = make_double2(0, 0);
  if (q.on) {
    const T* p = x + n * rx.sample + k.first * rx.row + q.c0 + q.vec;
#pragma unroll 4
    for (int r = q.row0; r < k.count; r += q.tr) {
      const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p + r * rx.row);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double d = to_f32(v.v[e]);
        acc[e].x += d;
        acc[e].y = fma(d, d, acc[e].y);
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) lds[q.row0 * q.nc + q.vec + e] = acc[e];
  }
  __syncthreads();
  // per channel over the rows in flight (in place: row 0 receives), then per group
  for (int c = threadIdx.x; c < q.nc; c += kThreads) {
    double2 t = lds[c];
    for (int r = 1; r < q.tr; ++r) t = t + lds[r * q.nc + c];
    lds[c] = t;
  }
  __syncthreads();
  // a group's channels to as many lanes, up to a wave's
  int lanes = 1;
  while (lanes < sh.cg && lanes < 64) lanes *= 2;
  const int l = threadIdx.x & (lanes - 1), at_once = kThreads / lanes;
  double2* out = sums + ((int64_t)n * gridDim.x * gridDim.z + blockIdx.x * gridDim.z + blockIdx.z) * sh.groups;
  for (int g0 = 0; g0 < sh.groups; g0 += at_once) {
    const int g = g0 + threadIdx.x / lanes;
    const int a = max(g * sh.cg - q.c0, 0), b = min((g + 1) * sh.cg - q.c0, q.nc);
    double2 t = make_double2(0, 0);
    for (int c = a + l; c < b; c += lanes) t = t + lds[c];
    for (int m = lanes >> 1; m >= 1; m >>= 1) {
      t.x += __shfl_xor(t.x, m);
      t.y += __shfl_xor(t.y, m);
    }
    if (l == 0 && g < sh.groups) out[g] = t;
  }
}

// the sums of the sample's parts, per group: stats[g] = (mean, rstd)
__device__ __forceinline__ void fold_moments(const Shape& sh, int parts, const double2* __restrict__ sums, double2* scratch,
                                             float2* stats) {
  for (int g0 = 0; g0 < sh.groups; g0 += kThreads) {
    const int ng = min(sh.groups - g0, kThreads), lanes = kThreads / ng;
    const int g = threadIdx.x % ng, l = threadIdx.x / ng;
    double2 t = make_double2(0, 0);
    if (l < lanes)
#pragma unroll 4
      for (int p = l; p < parts; p += lanes) t = t + sums[(int64_t)p * sh.groups + g0 + g];
    scratch[threadIdx.x] = t;
    __syncthreads();
    if (l == 0) {
      for (int k = 1; k < lanes; ++k) t = t + scratch[k * ng + g];
      float mean, rstd;
      moments(t, (double)sh.s * sh.cg, sh.eps, mean, rstd);
      stats[g0 + g] = make_float2(mean, rstd);
    }
    __syncthreads();
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) group_norm_apply_kernel(
    Shape sh, int rows, int parts, const T* __restrict__ x, Rows rx, const double2* __restrict__ sums,
    const void* __restrict__ gamma, const void* __restrict__ beta, T* __restrict__ y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out) {
  extern __shared__ float2 stats[];                   // [groups]
  __shared__ double2 scratch[kThreads];
  const Columns q(sh.c, V, blockIdx.z);
  // opposite order of the sums kernel: what it read last comes first
  const int n = gridDim.y - 1 - blockIdx.y, chunk = gridDim.x - 1 - blockIdx.x;
  const Chunk k(sh.s, rows, chunk);
  fold_moments(sh, parts, sums + (int64_t)n * parts * sh.groups, scratch, stats);
  if (chunk == 0 && blockIdx.z == 0)
    for (int g = threadIdx.x; g < sh.groups; g += kThreads) {
      mean_out[n * sh.groups + g] = stats[g].x;
      rstd_out[n * sh.groups + g] = stats[g].y;
    }
  if (!q.on) return;
  float mean[V], scale[V], be[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = q.c0 + q.vec + e;
    const float2 st = stats[c / sh.cg];
    mean[e] = st.x;
    scale[e] = st.y * (gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f);
    be[e] = beta ? load_param<T>(beta, sh.param_f32, c) : 0.f;
  }
  const T* p = x + n * rx.sample + k.first * rx.row + q.c0 + q.vec;
  T* o = y + ((int64_t)n * sh.s + k.first) * sh.c + q.c0 + q.vec;
  with_act(sh.act, [&](auto tag) {
#pragma unroll 8
    for (int r = q.row0; r < k.count; r += q.tr) {
      const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p + r * rx.row);
      Pack<T, V> out;
#pragma unroll
      for (int e = 0; e < V; ++e)
        out.v[e] = from_f32<T>(act_value<decltype(tag)::act, exact_act<T>()>(fmaf(to_f32(v.v[e]) - mean[e], scale[e], be[e])));
      *reinterpret_cast<Pack<T, V>*>(o + (int64_t)r * sh.c) = out;
    }
  });
}

// partial: [n][chunks][2][c] (sum dz | sum dz xh)
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) group_norm_grad_sums_kernel(
    Shape sh, int rows, const T* __restrict__ x, Rows rx, const T* __restrict__ dy, Rows rdy,
    const void* __restrict__ gamma, const void* __restrict__ beta, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ partial) {
  __shared__ float lds[2][kThreads * V];
  const Columns q(sh.c, V, blockIdx.z);
  const Chunk k(sh.s, rows, blockIdx.x);
  const int n = blockIdx.y;
  if (q.on) {
    float mean[V], rstd[V], ga[V], be[V], sb[V], sg[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = q.c0 + q.vec + e, g = n * sh.groups + c / sh.cg;
      mean[e] = mean_in[g];
      rstd[e] = rstd_in[g];
      ga[e] = gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f;
      be[e] = beta ? load_param<T>(beta, sh.param_f32, c) : 0.f;
      sb[e] = sg[e] = 0.f;
    }
    const T* p = x + n * rx.sample + k.first * rx.row + q.c0 + q.vec;
    const T* d = dy + n * rdy.sample + k.first * rdy.row + q.c0 + q.vec;
    with_act(sh.act, [&](auto tag) {
#pragma unroll 4
      for (int r = q.row0; r < k.count; r += q.tr) {
        const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p + r * rx.row);
        const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(d + r * rdy.row);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = (to_f32(v.v[e]) - mean[e]) * rstd[e];
          float value;
          const float dz = to_f32(u.v[e]) * act_slope<decltype(tag)::act, exact_act<T>()>(fmaf(xh, ga[e], be[e]), &value);
          sb[e] += dz;
          sg[e] = fmaf(dz, xh, sg[e]);
        }
      }
    });
#pragma unroll
    for (int e = 0; e < V; ++e) {
      lds[0][q.row0 * q.nc + q.vec + e] = sb[e];
      lds[1][q.row0 * q.nc + q.vec + e] = sg[e];
    }
  }
  __syncthreads();
  float* out = partial + ((int64_t)n * gridDim.x + blockIdx.x) * 2 * sh.c;
  for (int c = threadIdx.x; c < q.nc; c += kThreads) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      double t = 0;
      for (int r = 0; r < q.tr; ++r) t += lds[j][r * q.nc + c];
      out[j * sh.c + q.c0 + c] = (float)t;
    }
  }
}

// Blocks 0 .. group_blocks - 1: (sample, group)s in turn, group_sums = (mean(gamma dz), mean(gamma dz xh)).
// The blocks behind them: 8 columns of d_beta | d_gamma each, 32 threads a column.
template <typename T>
__global__ void __launch_bounds__(kThreads) group_norm_fold_kernel(
    Shape sh, int chunks, int group_blocks, const float* __restrict__ partial, const void* __restrict__ gamma,
    float2* __restrict__ group_sums, void* __restrict__ d_gamma, void* __restrict__ d_beta) {
  __shared__ double lds[32][9];
  if ((int)blockIdx.x < group_blocks) {
    __shared__ double2 waves[kThreads / 64];
    const int items = chunks * sh.cg;
    for (int at = blockIdx.x; at < sh.n * sh.groups; at += group_blocks) {
      const int n = at / sh.groups, c0 = (at % sh.groups) * sh.cg;
      const float* p = partial + (int64_t)n * chunks * 2 * sh.c;
      double2 t = make_double2(0, 0);
#pragma unroll 4
      for (int j = threadIdx.x; j < items; j += kThreads) {
        const int chunk = j / sh.cg, c = c0 + j % sh.cg;
        const double ga = gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f;
        t.x += ga * p[(int64_t)(2 * chunk) * sh.c + c];
        t.y += ga * p[(int64_t)(2 * chunk + 1) * sh.c + c];
      }
      t = block_sum(t, waves);
      const double inv = 1.0 / ((double)sh.s * sh.cg);
      if (threadIdx.x == 0) group_sums[at] = make_float2((float)(t.x * inv), (float)(t.y * inv));
    }
    return;
  }
  const int col = (blockIdx.x - group_blocks) * 8 + (threadIdx.x & 7), l = threadIdx.x >> 3;
  double t = 0;
  if (col < 2 * sh.c)
#pragma unroll 8
    for (int64_t p = l; p < (int64_t)sh.n * chunks; p += 32) t += partial[p * 2 * sh.c + col];
  lds[l][threadIdx.x & 7] = t;
  __syncthreads();
  if (l == 0 && col < 2 * sh.c) {
    for (int k = 1; k < 32; ++k) t += lds[k][threadIdx.x];
    void* out = col < sh.c ? d_beta : d_gamma;
    if (out) store_param<T>(out, sh.param_f32, col < sh.c ? col : col - sh.c, (float)t);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) group_norm_grad_apply_kernel(
    Shape sh, int rows, const T* __restrict__ x, Rows rx, const T* __restrict__ dy, Rows rdy,
    const void* __restrict__ gamma, const void* __restrict__ beta, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const float2* __restrict__ group_sums, T* __restrict__ dx) {
  const Columns q(sh.c, V, blockIdx.z);
  const int n = gridDim.y - 1 - blockIdx.y, chunk = gridDim.x - 1 - blockIdx.x;
  const Chunk k(sh.s, rows, chunk);
  if (!q.on) return;
  float mean[V], rstd[V], ga[V], be[V], m1[V], m2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = q.c0 + q.vec + e, g = n * sh.groups + c / sh.cg;
    mean[e] = mean_in[g];
    rstd[e] = rstd_in[g];
    ga[e] = gamma ? load_param<T>(gamma, sh.param_f32, c) : 1.f;
    be[e] = beta ? load_param<T>(beta, sh.param_f32, c) : 0.f;
    m1[e] = group_sums[g].x;
    m2[e] = group_sums[g].y;
  }
  const T* p = x + n * rx.sample + k.first * rx.row + q.c0 + q.vec;
  const T* d = dy + n * rdy.sample + k.first * rdy.row + q.c0 + q.vec;
  T* o = dx + ((int64_t)n * sh.s + k.first) * sh.c + q.c0 + q.vec;
  with_act(sh.act, [&](auto tag) {
#pragma unroll 4
    for (int r = q.row0; r < k.count; r += q.tr) {
      const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p + r * rx.row);
      const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(d + r * rdy.row);
      Pack<T, V> out;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (to_f32(v.v[e]) - mean[e]) * rstd[e];
        float value;
        const float dz = to_f32(u.v[e]) * act_slope<decltype(tag)::act, exact_act<T>()>(fmaf(xh, ga[e], be[e]), &value);
        out.v[e] = from_f32<T>(rstd[e] * (fmaf(dz, ga[e], -m1[e]) - xh * m2[e]));
      }
      *reinterpret_cast<Pack<T, V>*>(o + (int64_t)r * sh.c) = out;
    }
  });
}

// ---------------------------------------------------------------------------------------------------------------
struct Plan {
  int vec;               // elements of a vector access: 16 bytes of them, or 1
  int held, threads;     // the one-launch form: vectors a thread keeps (0: chunks)
  int chunks, rows, column_blocks;
};

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

Plan plan(const PsGroupNormDesc& d, const void* x, const void* dy, bool backward) {
  Plan p = {};
  const int e = d.dtype == PS_DTYPE_F32 ? 4 : 2, wide = 16 / e;
  auto fits = [&](const void* t, int64_t sample, int64_t row) {
    return !t || ((reinterpret_cast<uintptr_t>(t) & 15) == 0 && sample % wide == 0 && row % wide == 0);
  };
  const bool aligned = d.channels % wide == 0 && fits(x, d.x_sample_stride, d.x_row_stride) &&
                       fits(dy, d.dy_sample_stride, d.dy_row_stride);
  p.vec = aligned ? wide : 1;
  const int cg = d.channels / d.groups;
  const int most = backward ? kHeldBackward : kHeldForward;
  if (aligned && cg % wide == 0 && cg * e >= 32) {
    const int per_row = cg / wide;
    const int64_t vectors = (int64_t)d.rows * per_row;
    int threads = vectors <= 256 * 2 ? 256 : vectors <= 512 * 2 ? 512 : 1024;
    if (backward) {
      if (threads * wide > 4096) threads = 4096 / wide;   // 32 KB of LDS for the channels' sums
      threads -= threads % per_row;                       // a thread keeps its channels (0: a row is wider than the block)
    }
    if (threads >= 256 / 2 && vectors <= (int64_t)threads * most && threads % 64 == 0) {
      p.held = (int)((vectors + threads - 1) / threads);
      p.threads = threads;
      p.chunks = 1;
      return p;
    }
  }
  const int vectors = d.channels / p.vec;
  p.column_blocks = (vectors + kThreads - 1) / kThreads;
  const int at_once = kThreads / (vectors < kThreads ? vectors : kThreads);   // rows a block takes at a time
  // Blocks: four a CU, and up to 16 of 32 steps or more each, so that a CU always has some that read while others end
  // (14 x 256 x 256 x 256 in bf16: 1040 us at 1024 blocks, 890 at 3584).
  const int64_t steps = (int64_t)d.samples * p.column_blocks * (d.rows / at_once);
  const int blocks = steps >= 4096 * 32 ? 4096 : steps >= 1024 * 32 ? (int)(steps / 32) : 1024;
  int want = (int)((blocks + (int64_t)d.samples * p.column_blocks - 1) / ((int64_t)d.samples * p.column_blocks));
  if (want > 256) want = 256;
  // the gradient's sums are fp32 within a thread: no more than 256 rows of it, however long the sample
  const int64_t least = ((int64_t)d.rows + (int64_t)at_once * 256 - 1) / ((int64_t)at_once * 256);
  if (backward && want < least) want = (int)least;
  int64_t rows = ((int64_t)d.rows + want - 1) / want;
  rows = round_up(rows < 2 * at_once ? 2 * at_once : rows, at_once);
  p.rows = (int)(rows < d.rows ? rows : d.rows);
  p.chunks = (int)((d.rows + rows - 1) / rows);
  return p;
}

Shape shape_of(const PsGroupNormDesc& d) {
  Shape s;
  s.n = d.samples; s.s = d.rows; s.c = d.channels; s.groups = d.groups; s.cg = d.channels / d.groups;
  s.eps = d.eps; s.act = d.activation; s.param_f32 = d.param_f32;
  return s;
}

template <typename T, int V>
void forward_chunks(const PsGroupNormDesc& d, const Plan& p, const void* x, const void* gamma, const void* beta, void* y,
                    float* mean, float* rstd, void* workspace, hipStream_t st) {
  const Shape sh = shape_of(d);
  const Rows rx = {d.x_sample_stride, d.x_row_stride};
  const dim3 grid(p.chunks, d.samples, p.column_blocks);
  double2* sums = reinterpret_cast<double2*>(workspace);
  group_norm_sums_kernel<T, V><<<grid, kThreads, 0, st>>>(sh, p.rows, (const T*)x, rx, sums);
  group_norm_apply_kernel<T, V><<<grid, kThreads, sizeof(float2) * d.groups, st>>>(
      sh, p.rows, p.chunks * p.column_blocks, (const T*)x, rx, sums, gamma, beta, (T*)y, mean, rstd);
}

template <typename T, int V>
void backward_chunks(const PsGroupNormDesc& d, const Plan& p, const void* x, const void* dy, const void* gamma,
                     const void* beta, const float* mean, const float* rstd, void* dx, void* d_gamma, void* d_beta,
                     void* workspace, hipStream_t st) {
  const Shape sh = shape_of(d);
  const Rows rx = {d.x_sample_stride, d.x_row_stride}, rdy = {d.dy_sample_stride, d.dy_row_stride};
  const dim3 grid(p.chunks, d.samples, p.column_blocks);
  float2* group_sums = reinterpret_cast<float2*>(workspace);
  float* partial = reinterpret_cast<float*>(group_sums + (size_t)d.samples * d.groups);
  group_norm_grad_sums_kernel<T, V><<<grid, kThreads, 0, st>>>(sh, p.rows, (const T*)x, rx, (const T*)dy, rdy, gamma,
                                                               beta, mean, rstd, partial);
  // a launch holds 2^32 threads, a batch up to 2^29 groups
  const int group_blocks = d.samples * d.groups < 1 << 20 ? d.samples * d.groups : 1 << 20;
  group_norm_fold_kernel<T><<<group_blocks + (2 * d.channels + 7) / 8, kThreads, 0, st>>>(
      sh, p.chunks, group_blocks, partial, gamma, group_sums, d_gamma, d_beta);
  group_norm_grad_apply_kernel<T, V><<<grid, kThreads, 0, st>>>(sh, p.rows, (const T*)x, rx, (const T*)dy, rdy, gamma,
                                                                beta, mean, rstd, group_sums, (T*)dx);
}

template <typename T>
void forward_typed(const PsGroupNormDesc& d, const void* x, const void* gamma, const void* beta, void* y, float* mean,
                   float* rstd, void* workspace, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const Plan p = plan(d, x, nullptr, false);
  if (p.held) {
    const Shape sh = shape_of(d);
    const Rows rx = {d.x_sample_stride, d.x_row_stride};
    const dim3 grid(d.groups, d.samples);
    if (p.held <= 2)
      group_norm_held_forward_kernel<T, V, 2><<<grid, p.threads, 0, st>>>(sh, (const T*)x, rx, gamma, beta, (T*)y, mean, rstd);
    else
      group_norm_held_forward_kernel<T, V, kHeldForward><<<grid, p.threads, 0, st>>>(sh, (const T*)x, rx, gamma, beta, (T*)y, mean, rstd);
  } else if (p.vec > 1) {
    forward_chunks<T, V>(d, p, x, gamma, beta, y, mean, rstd, workspace, st);
  } else {
    forward_chunks<T, 1>(d, p, x, gamma, beta, y, mean, rstd, workspace, st);
  }
}

template <typename T>
void backward_typed(const PsGroupNormDesc& d, const void* x, const void* dy, const void* gamma, const void* beta,
                    const float* mean, const float* rstd, void* dx, void* d_gamma, void* d_beta, void* workspace,
                    hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const Plan p = plan(d, x, dy, true);
  if (p.held) {
    const Shape sh = shape_of(d);
    const Rows rx = {d.x_sample_stride, d.x_row_stride}, rdy = {d.dy_sample_stride, d.dy_row_stride};
    const dim3 grid(d.groups, d.samples);
    const size_t lds = (size_t)p.threads * V * 2 * sizeof(float);   // threads / (cg / V) rows of 2 cg floats
    float* partial = reinterpret_cast<float*>(workspace);
    if (p.held <= 2)
      group_norm_held_backward_kernel<T, V, 2><<<grid, p.threads, lds, st>>>(
          sh, (const T*)x, rx, (const T*)dy, rdy, gamma, beta, mean, rstd, (T*)dx, partial);
    else
      group_norm_held_backward_kernel<T, V, kHeldBackward><<<grid, p.threads, lds, st>>>(
          sh, (const T*)x, rx, (const T*)dy, rdy, gamma, beta, mean, rstd, (T*)dx, partial);
    if (d_gamma || d_beta)
      group_norm_fold_kernel<T><<<(2 * d.channels + 7) / 8, kThreads, 0, st>>>(sh, 1, 0, partial, gamma, nullptr,
                                                                                 d_gamma, d_beta);
  } else if (p.vec > 1) {
    backward_chunks<T, V>(d, p, x, dy, gamma, beta, mean, rstd, dx, d_gamma, d_beta, workspace, st);
  } else {
    backward_chunks<T, 1>(d, p, x, dy, gamma, beta, mean, rstd, dx, d_gamma, d_beta, workspace, st);
  }
}

bool desc_ok(const PsGroupNormDesc* d) {
  return d && d->samples > 0 && d->rows > 0 && d->channels > 0 && d->groups > 0 && d->channels % d->groups == 0 &&
         d->eps >= 0.f && d->x_row_stride >= d->channels && d->x_sample_stride >= 0;
}
int unsupported(const PsGroupNormDesc& d) {
  return d.channels > 8192 || d.samples > 65535 || (int64_t)d.rows * d.channels >= (int64_t)1 << 31 ||
         d.dtype < PS_DTYPE_F32 || d.dtype > PS_DTYPE_F16 ||
         d.activation < PS_ACT_NONE || d.activation > PS_ACT_SIGMOID;
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" {

size_t ps_group_norm_workspace_bytes(const PsGroupNormDesc* d, int32_t backward) {
  if (!desc_ok(d) || unsupported(*d)) return 0;
  // the chunked form at its most (unaligned tensors have more column blocks, and each of those has fewer chunks)
  PsGroupNormDesc q = *d;
  size_t most = 0;
  for (int form = 0; form < 2; ++form) {
    const Plan p = plan(q, form ? (const void*)1 : nullptr, nullptr, backward != 0);
    const size_t parts = (size_t)d->samples * p.chunks;
    const size_t bytes = backward ? sizeof(float2) * d->samples * d->groups + sizeof(float) * parts * 2 * d->channels
                                  : p.held ? 0 : sizeof(double2) * parts * p.column_blocks * d->groups;
    if (bytes > most) most = bytes;
  }
  return most + 256;
}

int ps_group_norm_forward(const PsGroupNormDesc* d, const void* x, const void* gamma, const void* beta, void* y,
                          float* mean, float* rstd, void* workspace, size_t workspace_bytes, void* stream) {
  if (!desc_ok(d) || !x || !y || !mean || !rstd || !workspace) return PS_ERR_BAD_ARG;
  if (unsupported(*d)) return PS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(y) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return PS_ERR_BAD_ARG;
  if (workspace_bytes < ps_group_norm_workspace_bytes(d, 0)) return PS_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case PS_DTYPE_F32: forward_typed<float>(*d, x, gamma, beta, y, mean, rstd, workspace, st); break;
    case PS_DTYPE_BF16: forward_typed<bf16>(*d, x, gamma, beta, y, mean, rstd, workspace, st); break;
    default: forward_typed<f16>(*d, x, gamma, beta, y, mean, rstd, workspace, st); break;
  }
  return hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

int ps_group_norm_backward(const PsGroupNormDesc* d, const void* x, const void* dy, const void* gamma, const void* beta,
                           const float* mean, const float* rstd, void* dx, void* d_gamma, void* d_beta, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (!desc_ok(d) || !x || !dy || !mean || !rstd || !dx || !workspace || d->dy_row_stride < 0 || d->dy_sample_stride < 0)
    return PS_ERR_BAD_ARG;
  if (unsupported(*d)) return PS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(dx) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return PS_ERR_BAD_ARG;
  if (workspace_bytes < ps_group_norm_workspace_bytes(d, 1)) return PS_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case PS_DTYPE_F32: backward_typed<float>(*d, x, dy, gamma, beta, mean, rstd, dx, d_gamma, d_beta, workspace, st); break;
    case PS_DTYPE_BF16: backward_typed<bf16>(*d, x, dy, gamma, beta, mean, rstd, dx, d_gamma, d_beta, workspace, st); break;
    default: backward_typed<f16>(*d, x, dy, gamma, beta, mean, rstd, dx, d_gamma, d_beta, workspace, st); break;
  }
  return hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

}  // extern "C"
