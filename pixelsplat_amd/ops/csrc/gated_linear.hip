// Gated projection of a feed-forward block, h = act(x Wg^T + bg) * (x Wu^T + bu), and its backward pass
//   du = dh act(a), da = dh u act'(a)   (a, u the two projections)
//   dx = da Wg + du Wu;  dWg = da^T x;  dWu = du^T x;  dbg, dbu = column sums of da, du.
//
// Bound by the matrix instructions (4 M D F flop forward, 8 M D F backward), except for a few rows, where the two
// weight matrices are all there is to read.
//
// One tiled product serves all of it.  A block computes a BM x BN tile; both operands go from global memory straight
// into LDS in slices of 128 bytes of the contraction index, double buffered, and from there as MFMA fragments.
// Operands lie along the contraction index (x, W in the forward) or across it (W in dx, both in dW: transposing LDS
// reads, no copies).  In the forward a block's columns are gate and up columns of the same hidden units in
// alternating runs of 32, so that the wave that holds a also holds u and the activation is its epilogue: neither
// projection reaches memory.
//
// 16384 x 1024 -> 4096 in bf16, silu: forward 342 us (275 GFLOP, 800 TFLOP/s; the fastest of 23 passes 322: its copies alone
// 246, its matrix instructions alone 249), da and du 417, dx 350, both weight gradients 331.  One token of it: 4.4 us for 17 MB of
// weights.
//
// What the backward needs of a and u: fp32 tensors keep both (8 bytes a hidden value, against 4 D flop at 150
// TFLOP/s); 16-bit tensors compute them again (the products are 8 times as fast, and keeping them rounded to 16 bits
// would put a second rounding into every gradient).  da and du are rounded to the tensors' type before they enter
// their products, as h is before its own; in fp16 they are first brought into its range (range_kernel).
#include "mfma_tile.h"
#include "pixelsplat_ops.h"

namespace ps {
namespace {

__device__ const uint4 kZeros[1] = {{0, 0, 0, 0}};   // what a copy reads for a chunk outside its operand

constexpr int kSliceBytes = 128;
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

struct Operand {
  const void* p[2];       // two matrices: the halves of the contraction (dx), or of the columns (forward)
  int64_t ld;             // elements
};

struct Product {
  int m, n, k;            // n: columns of the result (forward: hidden units); k: of one half
  int halves;             // of the contraction index
  int first;              // blockIdx.z + first: which of a's matrices, where halves is 1
  Operand a, b;
  int tiles_m, tiles_n, slices_per_split;
};

// which columns of a forward block belong to which projection
__device__ __forceinline__ int pair_unit(int col) { return (col >> 6) * 32 + (col & 31); }
__device__ __forceinline__ int pair_half(int col) { return (col >> 5) & 1; }

// blocks go to the 8 dies in turn: each die gets a run of neighbouring tiles, and its L2 the operands they share
__device__ __forceinline__ int die_order(int id, int count) {
  const int per = count >> 3, extra = count & 7, die = id & 7, at = id >> 3;
  return die * per + min(die, extra) + at;
}

// A copier owns what a wave copies of one operand: kPieces pieces of 1 KB of its tile every slice.
template <typename T, int ROWS, int WAVES, bool ACROSS>
struct Copier {
  static constexpr int kPieces = ROWS * kSliceBytes / 1024 / WAVES;
  const T* at[kPieces];     // at contraction index 0; NULL: outside the operand
  int kk[kPieces];          // contraction index within the slice
  int64_t other, step;      // from the first matrix to the second; elements of a contraction index

  template <bool PAIRED>
  __device__ __forceinline__ void init(const Operand& o, int which, int row0, int rows, int wave, int lane) {
    const T* p0 = reinterpret_cast<const T*>(which ? o.p[1] : o.p[0]);
    const T* p1 = reinterpret_cast<const T*>(o.p[1]);
    other = (reinterpret_cast<const char*>(p1) - reinterpret_cast<const char*>(p0)) / (int)sizeof(T);
    step = ACROSS ? o.ld : 1;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int piece = j * WAVES + wave, pos = piece * 64 + lane;
      if (ACROSS) {
        constexpr int kChunks = ROWS / kVec<T>;                  // of a row of the tile
        const int k = pos / kChunks;
        const int row = row0 + ((pos % kChunks) ^ across_swizzle<T, ROWS>(k)) * kVec<T>;
        at[j] = row < rows ? p0 + k * o.ld + row : nullptr;
        kk[j] = k;
      } else {
        const int r = pos >> 3, chunk = (pos & 7) ^ ((r >> 1) & 7);
        const int row = PAIRED ? row0 / 2 + pair_unit(r) : row0 + r;
        at[j] = row < rows ? (PAIRED && pair_half(piece * 8) ? p1 : p0) + row * o.ld + chunk * kVec<T> : nullptr;
        kk[j] = chunk * kVec<T>;
      }
    }
  }
  // slice [k0, ...) of a contraction of length k, in the first or second matrix
  __device__ __forceinline__ void copy(int which, int k0, int k, char* tile, int wave) const {
    const int64_t delta = k0 * step + (which ? other : 0);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const bool inside = at[j] != nullptr && k0 + kk[j] < k;
      copy_to_lds(inside ? (const void*)(at[j] + delta) : (const void*)kZeros, tile + (j * WAVES + wave) * 1024);
    }
  }
};

// A 16-bit tile on its way from result registers to memory: a register's 32 lanes are 64 bytes of a row, memory wants
// 16 bytes a lane.  Rows are 16 bytes longer than they are, so that the halves of a wave, 4 rows apart, differ in banks.
template <typename T, int ROWS, int COLS, int THREADS>
struct Staged {
  static constexpr int kPitch = COLS * 2 + 16, kBytes = ROWS * kPitch, kChunks = ROWS * COLS / 8 / THREADS;
  static __device__ __forceinline__ T* at(char* tile, int row, int col) { return reinterpret_cast<T*>(tile + row * kPitch) + col; }
  // f(chunk of the thread, row, first column)
  template <typename F>
  static __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int pos = i * THREADS + threadIdx.x;
      f(i, pos / (COLS / 8), pos % (COLS / 8) * 8);
    }
  }
  // rows of out from (row0, col0): rows and columns (a multiple of 8) that there are
  static __device__ __forceinline__ void flush(char* tile, T* out, int64_t ld, int row0, int rows, int col0, int cols) {
    each([&](int, int row, int col) {
      if (row0 + row < rows && col0 + col < cols)
        *reinterpret_cast<uintx4*>(out + (row0 + row) * ld + col0 + col) = *reinterpret_cast<uintx4*>(at(tile, row, col));
    });
  }
};

// what an epilogue knows of its block
template <typename T_, int BM_, int BN_, int WM_, int WN_>
struct Tile {
  typedef T_ T;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, THREADS = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
  char* lds;
  int m0, n0, wm, wn, lane, row_part;
};

// BM x BN tile of WM x WN waves; EP writes the result
template <typename T, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS, bool PAIRED, typename EP>
__global__ void __launch_bounds__(WM * WN * 64, 2)
product_kernel(Product g, EP ep) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, kK = kSliceBytes / sizeof(T);
  constexpr int kA = BM * kSliceBytes, kB = BN * kSliceBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];    // 2 x (A | B)
  if (ep.done()) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, hi = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  // tiles of 8 rows of tiles at a time, column by column: neighbours share their operands in the die's L2
  const int id = die_order(blockIdx.x, g.tiles_m * g.tiles_n);
  const int group = id / (8 * g.tiles_n), rows_in = min(8, g.tiles_m - group * 8), in = id - group * 8 * g.tiles_n;
  const int tm = group * 8 + in % rows_in, tn = in / rows_in;
  const int m0 = tm * BM, n0 = tn * BN;

  const Tile<T, BM, BN, WM, WN> tile = {lds, m0, n0, wm, wn, lane, tm * WM + wm};
  Copier<T, BM, WAVES, A_ACROSS> ca;
  Copier<T, BN, WAVES, B_ACROSS> cb;
  ca.template init<false>(g.a, blockIdx.z + g.first, m0, g.m, wave, lane);
  cb.template init<PAIRED>(g.b, 0, n0, g.n, wave, lane);

  floatx16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = zero16();

  const int per_half = (g.k + kK - 1) / kK, slices = per_half * g.halves;
  const int s0 = blockIdx.y * g.slices_per_split, s1 = min(s0 + g.slices_per_split, slices);
  auto load = [&](int s, int buf) {
    const int which = s >= per_half ? 1 : 0, k0 = (s - which * per_half) * kK;
    ca.copy(which, k0, g.k, lds + buf * (kA + kB), wave);
    cb.copy(which, k0, g.k, lds + buf * (kA + kB) + kA, wave);
  };
  if (s0 < s1) load(s0, 0);
  wait_for_copies();
  __syncthreads();
  for (int s = s0; s < s1; ++s) {
    const int buf = (s - s0) & 1;
    if (s + 1 < s1) load(s + 1, buf ^ 1);
    const char* ta = lds + buf * (kA + kB);
    const char* tb = ta + kA;
#pragma unroll
    for (int c = 0; c < 4; ++c) {                    // 32 bytes of the contraction index a step
      Frag<T> fa[TM], fb[TN];
      const int k0 = (2 * c + hi) * kVec<T>;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = (wm * TM + i) * 32;
        fa[i] = A_ACROSS ? across_fragment<T, BM>(ta, row, k0, k0 + 4, lane)
                         : along_fragment<T>(ta, row + (lane & 31), 2 * c + hi);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = (wn * TN + j) * 32;
        fb[j] = B_ACROSS ? across_fragment<T, BN>(tb, row, k0, k0 + 4, lane)
                         : along_fragment<T>(tb, row + (lane & 31), 2 * c + hi);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j]);
    }
    wait_for_copies();
    __syncthreads();                                 // the next slice has arrived, this one has been read
  }
  ep.store(acc, tile, g);                      // LDS is free
}

// ---- epilogues --------------------------------------------------------------------------------------------------
// h, and (fp32 training) a and u
struct NotDone {
  __device__ __forceinline__ bool done() const { return false; }
};
struct StoreGated : NotDone {
  void* h;
  const void *bg, *bu;
  float *a, *u;           // NULL: not kept
  int act;
  template <typename TL>
  __device__ __forceinline__ void store(const floatx16 (&acc)[TL::TM][TL::TN], const TL& t, const Product& g) const {
    typedef typename TL::T T;
    typedef Staged<T, TL::BM, TL::BN / 2, TL::THREADS> St;
    const bool staged = sizeof(T) == 2 && g.n % 8 == 0;
    const int u0 = t.n0 / 2;
    with_act(act, [&](auto tag) {
#pragma unroll
      for (int j = 0; j < TL::TN; j += 2) {
        const int col = (t.wn * TL::TN + j) * 16 + (t.lane & 31), f = u0 + col;
        if (f >= g.n) continue;
        const float wg = bg ? to_f32(reinterpret_cast<const T*>(bg)[f]) : 0.f;
        const float wu = bu ? to_f32(reinterpret_cast<const T*>(bu)[f]) : 0.f;
#pragma unroll
        for (int i = 0; i < TL::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int in = (t.wm * TL::TM + i) * 32 + result_row(r, t.lane >> 5), row = t.m0 + in;
            const float za = acc[i][j][r] + wg, zu = acc[i][j + 1][r] + wu;
            const T v = from_f32<T>(act_value<decltype(tag)::act, sizeof(T) == 4>(za) * zu);
            if (staged) {
              *St::at(t.lds, in, col) = v;
            } else if (row < g.m) {
              const int64_t at = (int64_t)row * g.n + f;
              reinterpret_cast<T*>(h)[at] = v;
              if (a) { a[at] = za; u[at] = zu; }
            }
          }
      }
    });
    if (staged) {
      __syncthreads();
      if constexpr (sizeof(T) == 2) St::flush(t.lds, (T*)h, g.n, t.m0, g.m, u0, g.n);
    }
  }
};

// fp16: what da and du are multiplied by before they are rounded, and its inverse; powers of two.
struct Range { float scale, inverse; };

// da and du (16-bit) from the recomputed projections; with biases, their column sums over the wave's rows.  dh comes
// through LDS where it lies in whole aligned chunks; da takes its place there.
struct StoreGatedGrad {
  const void* dh;
  int64_t ld_dh;
  int dh_chunks;          // rows of dh are whole 16-byte chunks
  const void *bg, *bu;
  void *da, *du;          // [m][ld]
  int ld;
  float* sums;            // [row parts][2][ld] or NULL
  int act;
  float* peaks;           // fp16: the largest finite |da| and |du| of every wave
  const Range* range;     // fp16, the second time: see range_kernel
  __device__ __forceinline__ bool done() const { return range != nullptr && range->scale == 1.f; }
  template <typename TL>
  __device__ __forceinline__ void store(const floatx16 (&acc)[TL::TM][TL::TN], const TL& t, const Product& g) const {
    typedef typename TL::T T;
    typedef Staged<T, TL::BM, TL::BN / 2, TL::THREADS> St;
    const float by = kNarrow<T> && range ? range->scale : 1.f;
    float peak = 0.f;
    char *ta = t.lds, *tu = t.lds + St::kBytes;
    const int u0 = t.n0 / 2;
    if (dh_chunks) {
      uintx4 v[St::kChunks];
      St::each([&](int i, int row, int col) {
        const bool there = t.m0 + row < g.m && u0 + col < g.n;
        v[i] = *reinterpret_cast<const uintx4*>(there ? (const void*)((const T*)dh + (t.m0 + row) * ld_dh + u0 + col)
                                                      : (const void*)kZeros);
      });
      St::each([&](int i, int row, int col) { *reinterpret_cast<uintx4*>(St::at(ta, row, col)) = v[i]; });
      __syncthreads();
    }
    with_act(act, [&](auto tag) {
#pragma unroll
      for (int j = 0; j < TL::TN; j += 2) {
        const int col = (t.wn * TL::TN + j) * 16 + (t.lane & 31), f = u0 + col;
        if (f >= ld) continue;
        const bool on = f < g.n;                        // the columns behind the last are zero
        const float wg = on && bg ? to_f32(reinterpret_cast<const T*>(bg)[f]) : 0.f;
        const float wu = on && bu ? to_f32(reinterpret_cast<const T*>(bu)[f]) : 0.f;
        float sa = 0.f, su = 0.f;
#pragma unroll
        for (int i = 0; i < TL::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int in = (t.wm * TL::TM + i) * 32 + result_row(r, t.lane >> 5), row = t.m0 + in;
            float va = 0.f, vu = 0.f;
            if (on && row < g.m) {
              const float d = to_f32(dh_chunks ? *St::at(ta, in, col) : reinterpret_cast<const T*>(dh)[row * ld_dh + f]);
              float value;
              const float slope = act_slope<decltype(tag)::act, false>(acc[i][j][r] + wg, &value);
              va = d * (acc[i][j + 1][r] + wu) * slope;
              vu = d * value;
            }
            if constexpr (kNarrow<T>) {
              const float top = fmaxf(fabsf(va), fabsf(vu));
              if (top < __builtin_inff()) peak = fmaxf(peak, top);
              *St::at(ta, in, col) = from_f32<T>(va * by);
              *St::at(tu, in, col) = from_f32<T>(vu * by);
            } else {
              *St::at(ta, in, col) = from_f32<T>(va);
              *St::at(tu, in, col) = from_f32<T>(vu);
            }
            sa += va;
            su += vu;
          }
        if (sums) {
          sa += __shfl_xor(sa, 32);
          su += __shfl_xor(su, 32);
          if (t.lane < 32) {
            sums[((int64_t)t.row_part * 2 + 0) * ld + f] = sa;
            sums[((int64_t)t.row_part * 2 + 1) * ld + f] = su;
          }
        }
      }
    });
    if constexpr (kNarrow<T>) {
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) peak = fmaxf(peak, __shfl_xor(peak, m));
      if (t.lane == 0) peaks[blockIdx.x * (TL::THREADS / 64) + (threadIdx.x >> 6)] = peak;
    }
    __syncthreads();
    St::flush(ta, (T*)da, ld, t.m0, g.m, u0, ld);
    St::flush(tu, (T*)du, ld, t.m0, g.m, u0, ld);
  }
};

// the product itself, or this split's part of it in fp32
struct StoreMatrix : NotDone {
  void* c[2];             // by blockIdx.z
  float* parts;           // [blockIdx.z][splits][m][n] or NULL
  const Range* range;     // fp16: what its first operand was multiplied by
  template <typename TL>
  __device__ __forceinline__ void store(const floatx16 (&acc)[TL::TM][TL::TN], const TL& t, const Product& g) const {
    typedef typename TL::T T;
    typedef Staged<T, TL::BM, TL::BN, TL::THREADS> St;
    T* out = reinterpret_cast<T*>(blockIdx.z ? c[1] : c[0]);
    const bool staged = sizeof(T) == 2 && !parts;       // n is a multiple of 8
    const float by = kNarrow<T> ? range->inverse : 1.f;
#pragma unroll
    for (int j = 0; j < TL::TN; ++j) {
      const int in_col = (t.wn * TL::TN + j) * 32 + (t.lane & 31), col = t.n0 + in_col;
      if (col >= g.n) continue;
#pragma unroll
      for (int i = 0; i < TL::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int in = (t.wm * TL::TM + i) * 32 + result_row(r, t.lane >> 5), row = t.m0 + in;
          const float v = kNarrow<T> ? acc[i][j][r] * by : acc[i][j][r];
          if (staged) *St::at(t.lds, in, in_col) = from_f32<T>(v);
          else if (row < g.m && parts) parts[(((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * g.m + row) * g.n + col] = v;
          else if (row < g.m) out[(int64_t)row * g.n + col] = from_f32<T>(v);
        }
    }
    if (staged) {
      __syncthreads();
      if constexpr (sizeof(T) == 2) St::flush(t.lds, out, g.n, t.m0, g.m, t.n0, g.n);
    }
  }
};

// ---- small kernels ----------------------------------------------------------------------------------------------
// fp16 holds less than the products it is an operand of: da = dh u act'(a) of 2^17 is infinite in it though dx is not, and
// below 2^-14 it has few bits.  So da and du are computed twice where their largest value lies outside 2^-6 .. 65504, the
// second time multiplied by the power of two that takes it to 2^14 .. 2^15; the products' results are divided by it.  Where it
// lies inside (what is smaller is off by 2^-25 at most, 2^-19 of the largest), the second launch ends at once.  A scale a row
// would do for dx, but rows are what dW sums over.  The training pass of 16384 x 1024 -> 4096: 1443 us without either, 1476 as it
// is, 1871 where it computes them twice.
__global__ void __launch_bounds__(1024) range_kernel(int64_t n, const float* __restrict__ peaks, Range* __restrict__ range) {
  __shared__ float lds[16];
  float peak = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) peak = fmaxf(peak, peaks[i]);
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) peak = fmaxf(peak, __shfl_xor(peak, m));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = peak;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) peak = fmaxf(peak, lds[w]);
    int up = 0;
    if (peak > 65504.f || (peak > 0.f && peak < 0.015625f)) up = max(-100, min(100, 14 - ilogbf(peak)));
    *range = {ldexpf(1.f, up), ldexpf(1.f, -up)};
  }
}

// fp32: da, du of the kept projections.  A block takes `rows` rows of 256 columns and leaves their column sums.
__global__ void __launch_bounds__(256) gated_slope_kernel(int m, int n, int ld, int rows, int act, const float* __restrict__ a,
                                                          const float* __restrict__ u, const float* __restrict__ dh,
                                                          int64_t ld_dh, float* __restrict__ da, float* __restrict__ du,
                                                          float* __restrict__ sums) {
  const int f = blockIdx.x * 256 + threadIdx.x;
  if (f >= ld) return;
  const int r0 = blockIdx.y * rows, r1 = min(r0 + rows, m);
  const int fc = min(f, n - 1);                      // the columns behind the last are zero
  const bool on = f < n;
  float sa = 0.f, su = 0.f;
  with_act(act, [&](auto tag) {
    for (int r = r0; r < r1; r += 4) {
      float za[4], zu[4], d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = min(r + i, m - 1);
        za[i] = a[row * n + fc];
        zu[i] = u[row * n + fc];
        d[i] = dh[row * ld_dh + fc];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + i >= r1) continue;
        float value;
        const float slope = act_slope<decltype(tag)::act, true>(za[i], &value);
        const float va = on ? d[i] * zu[i] * slope : 0.f, vu = on ? d[i] * value : 0.f;
        da[(int64_t)(r + i) * ld + f] = va;
        du[(int64_t)(r + i) * ld + f] = vu;
        sa += va;
        su += vu;
      }
    }
  });
  if (sums) {
    sums[((int64_t)blockIdx.y * 2 + 0) * ld + f] = sa;
    sums[((int64_t)blockIdx.y * 2 + 1) * ld + f] = su;
  }
}

// What is left of a backward pass, in one launch: sums of the splits' parts (each in their order), and the biases'
// gradients from the column sums of all rows' parts (16 columns a block, 16 threads a column).
struct Join {
  int64_t count;          // elements (a multiple of 4) of one matrix
  int splits, matrices, blocks;
  const float* parts;     // [matrices][splits][count]
  void* c[2];
};
struct Finish {
  Join join[2];
  int sum_parts, hidden, ld, bias_blocks;
  const float* sums;
  void* db[2];
};
template <typename T>
__global__ void __launch_bounds__(256) gated_finish_kernel(Finish f) {
  __shared__ double lds[16][17];
  int block = blockIdx.x;
  for (int k = 0; k < 2; ++k) {
    const Join& q = f.join[k];
    if (block < q.blocks) {
      const int64_t i = ((int64_t)block * 256 + threadIdx.x) * 4;
      if (i >= q.count * q.matrices) return;
      const int which = i >= q.count;
      const float* p = q.parts + which * (q.splits - 1) * q.count + i;
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < q.splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(p + s * q.count);
        t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
      }
      Pack<T, 4> out = {{from_f32<T>(t.x), from_f32<T>(t.y), from_f32<T>(t.z), from_f32<T>(t.w)}};
      *reinterpret_cast<Pack<T, 4>*>((T*)(which ? q.c[1] : q.c[0]) + (i - which * q.count)) = out;
      return;
    }
    block -= q.blocks;
  }
  const int col = block * 16 + (threadIdx.x & 15), l = threadIdx.x >> 4;
  double t = 0;
  if (col < 2 * f.ld)
#pragma unroll 4
    for (int p = l; p < f.sum_parts; p += 16) t += f.sums[(int64_t)p * 2 * f.ld + col];
  lds[l][threadIdx.x & 15] = t;
  __syncthreads();
  if (l == 0 && col < 2 * f.ld) {
    for (int k = 1; k < 16; ++k) t += lds[k][threadIdx.x];
    const int u = col < f.ld ? col : col - f.ld;
    T* out = (T*)(col < f.ld ? f.db[0] : f.db[1]);
    if (out && u < f.hidden) out[u] = from_f32<T>((float)t);
  }
}

// ---- a few rows: a wave takes a hidden unit, its lanes the contraction index --------------------------------------
template <typename T, int M>
__global__ void __launch_bounds__(256) gated_rows_kernel(int m, int d, int n, int act, const T* __restrict__ x, int64_t ldx,
                                                         const T* __restrict__ wg, const T* __restrict__ wu, int64_t ldw,
                                                         const T* __restrict__ bg, const T* __restrict__ bu, T* __restrict__ h,
                                                         float* __restrict__ a, float* __restrict__ u) {
  const int f = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (f >= n) return;
  constexpr int V = kVec<T>;
  float sa[M], su[M];
#pragma unroll
  for (int i = 0; i < M; ++i) sa[i] = su[i] = 0.f;
  const T* rg = wg + f * ldw;
  const T* ru = wu + f * ldw;
#pragma unroll 2
  for (int k = lane * V; k < d; k += 64 * V) {
    const Pack<T, V> g = *reinterpret_cast<const Pack<T, V>*>(rg + k);
    const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(ru + k);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (i < m) {
        const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + i * ldx + k);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sa[i] = fmaf(to_f32(v.v[e]), to_f32(g.v[e]), sa[i]);
          su[i] = fmaf(to_f32(v.v[e]), to_f32(w.v[e]), su[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      sa[i] += __shfl_xor(sa[i], s);
      su[i] += __shfl_xor(su[i], s);
    }
  if (lane == 0) {
    const float b0 = bg ? to_f32(bg[f]) : 0.f, b1 = bu ? to_f32(bu[f]) : 0.f;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (i < m) {
        const float za = sa[i] + b0, zu = su[i] + b1;
        const int64_t at = (int64_t)i * n + f;
        with_act(act, [&](auto tag) { h[at] = from_f32<T>(act_value<decltype(tag)::act, sizeof(T) == 4>(za) * zu); });
        if (a) { a[at] = za; u[at] = zu; }
      }
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------
constexpr int kCus = 256;
constexpr int kFewRows = 8;

struct Tiling { int bm, bn, splits, slices_per_split, tiles_m, tiles_n; };

// columns: of the tiles (forward: 2 n); products: in the launch.  The largest tile that still fills the machine, twice
// where a tile is big; a contraction is split where even small tiles do not, into 4 slices of it at least.
Tiling tiling(int dtype, int m, int columns, int k, int halves, int products, bool may_split) {
  Tiling t;
  const int kk = kSliceBytes / (dtype == PS_DTYPE_F32 ? 4 : 2);
  auto count = [](int a, int b) { return (a + b - 1) / b; };
  auto tiles = [&](int size) { return (int64_t)count(m, size) * count(columns, size) * products; };
  t.bm = dtype != PS_DTYPE_F32 && tiles(256) >= 2 * kCus ? 256 : tiles(128) >= kCus ? 128 : 64;
  t.bn = t.bm;
  t.tiles_m = count(m, t.bm);
  t.tiles_n = count(columns, t.bn);
  const int slices = count(k, kk) * halves;
  t.splits = 1;
  if (may_split && tiles(t.bm) < 2 * kCus) {
    int s = (int)(4 * kCus / tiles(t.bm));
    if (s > slices / 4) s = slices / 4;
    t.splits = s < 1 ? 1 : s;
  }
  t.slices_per_split = count(slices, t.splits);
  t.splits = count(slices, t.slices_per_split);
  return t;
}

template <typename T, bool A_ACROSS, bool B_ACROSS, bool PAIRED, typename EP>
int launch_product(Product g, const Tiling& t, const EP& ep, hipStream_t st, int products = 1) {
  g.tiles_m = t.tiles_m;
  g.tiles_n = t.tiles_n;
  g.slices_per_split = t.slices_per_split;
  const dim3 grid((unsigned)(t.tiles_m * t.tiles_n), (unsigned)t.splits, (unsigned)products);
  // two buffers of slices; then at most two staged tiles of half the columns, or one of all
  const size_t slices = (size_t)2 * (t.bm + t.bn) * kSliceBytes, staged = (size_t)t.bm * (2 * t.bn + 32);
  const size_t lds = sizeof(T) == 2 && staged > slices ? staged : slices;
  if constexpr (sizeof(T) == 2) {
    if (t.bm == 256) {
      auto kernel = product_kernel<T, 256, 256, 2, 4, A_ACROSS, B_ACROSS, PAIRED, EP>;
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) !=
          hipSuccess)
        return PS_ERR_LAUNCH;
      kernel<<<grid, 512, lds, st>>>(g, ep);
      return PS_OK;
    }
  }
  if (t.bm == 128) {
    product_kernel<T, 128, 128, 2, 2, A_ACROSS, B_ACROSS, PAIRED, EP><<<grid, 256, lds, st>>>(g, ep);
  } else {
    constexpr int WN = PAIRED ? 1 : 2;               // a wave of a pair holds 32 columns of each
    product_kernel<T, 64, 64, 2, WN, A_ACROSS, B_ACROSS, PAIRED, EP><<<grid, 128 * WN, lds, st>>>(g, ep);
  }
  return PS_OK;
}

int pad8(int n) { return (n + 7) & ~7; }
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct BackwardPlan {
  int ld, sum_parts, slope_rows;
  Tiling again, dx, dw;
  size_t da, du, sums, peaks, range, parts_x, parts_w, total;
};

BackwardPlan backward_plan(const PsGatedLinearDesc& d) {
  BackwardPlan p = {};
  const size_t e = d.dtype == PS_DTYPE_F32 ? 4 : 2;
  p.ld = pad8(d.hidden);
  p.again = tiling(d.dtype, d.rows, 2 * p.ld, d.dim, 1, 1, false);
  p.dx = tiling(d.dtype, d.rows, d.dim, d.hidden, 2, 1, true);
  p.dw = tiling(d.dtype, d.hidden, d.dim, d.rows, 1, 2, true);
  p.slope_rows = 8;
  while (p.slope_rows < 64 && (int64_t)d.rows * p.ld > (int64_t)p.slope_rows * 256 * 8 * kCus) p.slope_rows *= 2;
  while (d.rows / p.slope_rows >= 32768) p.slope_rows *= 2;   // blocks along a grid's second axis
  p.sum_parts = d.dtype == PS_DTYPE_F32 ? (d.rows + p.slope_rows - 1) / p.slope_rows : p.again.tiles_m * 2;
  size_t at = 0;
  p.da = at; at += align256(e * d.rows * p.ld);
  p.du = at; at += align256(e * d.rows * p.ld);
  p.sums = at; at += align256(sizeof(float) * p.sum_parts * 2 * p.ld);
  if (d.dtype == PS_DTYPE_F16) {
    p.peaks = at; at += align256(sizeof(float) * 8 * p.again.tiles_m * (size_t)p.again.tiles_n);   // 8 waves a tile at most
    p.range = at; at += align256(sizeof(Range));
  }
  p.parts_x = at; at += p.dx.splits > 1 ? align256(sizeof(float) * p.dx.splits * (size_t)d.rows * d.dim) : 0;
  p.parts_w = at; at += p.dw.splits > 1 ? align256(sizeof(float) * 2 * p.dw.splits * (size_t)d.hidden * d.dim) : 0;
  p.total = at;
  return p;
}

template <typename T>
int forward_typed(const PsGatedLinearDesc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                  void* h, float* a, float* u, hipStream_t st) {
  if (d.rows <= kFewRows) {
    const unsigned grid = (unsigned)((d.hidden + 3) / 4);
    auto run = [&](auto kernel) {
      kernel<<<grid, 256, 0, st>>>(d.rows, d.dim, d.hidden, d.activation, (const T*)x, d.x_row_stride, (const T*)wg,
                                   (const T*)wu, d.w_row_stride, (const T*)bg, (const T*)bu, (T*)h, a, u);
    };
    if (d.rows == 1) run(gated_rows_kernel<T, 1>);
    else if (d.rows == 2) run(gated_rows_kernel<T, 2>);
    else if (d.rows <= 4) run(gated_rows_kernel<T, 4>);
    else run(gated_rows_kernel<T, kFewRows>);
    return PS_OK;
  }
  Product g = {};
  g.m = d.rows; g.n = d.hidden; g.k = d.dim; g.halves = 1;
  g.a.p[0] = x; g.a.ld = d.x_row_stride;
  g.b.p[0] = wg; g.b.p[1] = wu; g.b.ld = d.w_row_stride;
  StoreGated ep = {{}, h, bg, bu, a, u, d.activation};
  return launch_product<T, false, false, true>(g, tiling(d.dtype, d.rows, 2 * d.hidden, d.dim, 1, 1, false), ep, st);
}

template <typename T>
int backward_typed(const PsGatedLinearDesc& d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu,
                   const float* a, const float* u, const void* dh, void* dx, void* dwg, void* dwu, void* dbg, void* dbu,
                   char* ws, hipStream_t st) {
  const BackwardPlan p = backward_plan(d);
  T* da = (T*)(ws + p.da);
  T* du = (T*)(ws + p.du);
  float* sums = dbg || dbu ? (float*)(ws + p.sums) : nullptr;
  float* parts_x = p.dx.splits > 1 ? (float*)(ws + p.parts_x) : nullptr;
  float* parts_w = p.dw.splits > 1 ? (float*)(ws + p.parts_w) : nullptr;
  const Range* range = kNarrow<T> ? (const Range*)(ws + p.range) : nullptr;
  Finish f = {};
  if constexpr (sizeof(T) == 4) {
    const dim3 grid((unsigned)((p.ld + 255) / 256), (unsigned)p.sum_parts);
    gated_slope_kernel<<<grid, 256, 0, st>>>(d.rows, d.hidden, p.ld, p.slope_rows, d.activation, a, u, (const float*)dh,
                                             d.dh_row_stride, da, du, sums);
  } else {
    Product g = {};
    g.m = d.rows; g.n = d.hidden; g.k = d.dim; g.halves = 1;
    g.a.p[0] = x; g.a.ld = d.x_row_stride;
    g.b.p[0] = wg; g.b.p[1] = wu; g.b.ld = d.w_row_stride;
    const int chunks = d.hidden % 8 == 0 && d.dh_row_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(dh) & 15) == 0;
    StoreGatedGrad ep = {dh, d.dh_row_stride, chunks, bg, bu, da, du, p.ld, sums, d.activation, (float*)(ws + p.peaks), nullptr};
    if (int rc = launch_product<T, false, false, true>(g, p.again, ep, st)) return rc;
    if (kNarrow<T>) {
      const int waves = p.again.bm == 256 ? 8 : p.again.bm == 128 ? 4 : 2;
      range_kernel<<<1, 1024, 0, st>>>((int64_t)p.again.tiles_m * p.again.tiles_n * waves, ep.peaks, (Range*)range);
      ep.range = range;
      if (int rc = launch_product<T, false, false, true>(g, p.again, ep, st)) return rc;
    }
  }
  auto join = [](const Tiling& t, int64_t count, const float* parts, int matrices, void* c0, void* c1) {
    Join j = {count, t.splits, matrices, (int)((count * matrices / 4 + 255) / 256), parts, {c0, c1}};
    return j;
  };
  if (dx) {
    Product g = {};
    g.m = d.rows; g.n = d.dim; g.k = d.hidden; g.halves = 2;
    g.a.p[0] = da; g.a.p[1] = du; g.a.ld = p.ld;
    g.b.p[0] = wg; g.b.p[1] = wu; g.b.ld = d.w_row_stride;
    StoreMatrix ep = {{}, {dx, nullptr}, parts_x, range};
    if (int rc = launch_product<T, false, true, false>(g, p.dx, ep, st)) return rc;
    if (parts_x) f.join[0] = join(p.dx, (int64_t)d.rows * d.dim, parts_x, 1, dx, nullptr);
  }
  if (dwg || dwu) {                                  // both in one launch
    const int products = dwg && dwu ? 2 : 1;
    Product g = {};
    g.m = d.hidden; g.n = d.dim; g.k = d.rows; g.halves = 1; g.first = dwg ? 0 : 1;
    g.a.p[0] = da; g.a.p[1] = du; g.a.ld = p.ld;
    g.b.p[0] = x; g.b.ld = d.x_row_stride;
    StoreMatrix ep = {{}, {dwg ? dwg : dwu, dwu}, parts_w, range};
    if (int rc = launch_product<T, true, true, false>(g, p.dw, ep, st, products)) return rc;
    if (parts_w) f.join[1] = join(p.dw, (int64_t)d.hidden * d.dim, parts_w, products, dwg ? dwg : dwu, dwu);
  }
  f.sum_parts = p.sum_parts; f.hidden = d.hidden; f.ld = p.ld; f.sums = sums;
  f.bias_blocks = sums ? (2 * p.ld + 15) / 16 : 0;
  f.db[0] = dbg; f.db[1] = dbu;
  const int blocks = f.join[0].blocks + f.join[1].blocks + f.bias_blocks;
  if (blocks) gated_finish_kernel<T><<<blocks, 256, 0, st>>>(f);
  return PS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// both operands of every product are copied in 16-byte chunks: rows start on 16 bytes and hold whole chunks
int check(const PsGatedLinearDesc* d, const void* x, const void* wg, const void* wu) {
  if (!d || !x || !wg || !wu || d->rows <= 0 || d->dim <= 0 || d->hidden <= 0) return PS_ERR_BAD_ARG;
  if (d->dtype < PS_DTYPE_F32 || d->dtype > PS_DTYPE_F16 || d->activation < PS_ACT_NONE || d->activation > PS_ACT_SIGMOID)
    return PS_ERR_UNSUPPORTED;
  if (d->rows > (1 << 28) || d->dim > (1 << 24) || d->hidden > (1 << 24)) return PS_ERR_UNSUPPORTED;
  const int chunk = d->dtype == PS_DTYPE_F32 ? 4 : 8;
  if (d->dim % chunk || d->x_row_stride < d->dim || d->w_row_stride < d->dim || d->x_row_stride % chunk ||
      d->w_row_stride % chunk || !aligned16(x) || !aligned16(wg) || !aligned16(wu))
    return PS_ERR_BAD_ARG;
  const int64_t tiles = ((int64_t)d->rows + 127) / 128 * ((2 * (int64_t)d->hidden + 127) / 128 + (d->dim + 127) / 128);
  return tiles < (int64_t)1 << 31 ? PS_OK : PS_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" {

int ps_gated_linear_forward(const PsGatedLinearDesc* d, const void* x, const void* w_gate, const void* w_up,
                            const void* b_gate, const void* b_up, void* h, float* gate, float* up, void* stream) {
  if (int rc = check(d, x, w_gate, w_up)) return rc;
  if (!h || !aligned16(h) || (gate == nullptr) != (up == nullptr)) return PS_ERR_BAD_ARG;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d->dtype) {
    case PS_DTYPE_F32: rc = forward_typed<float>(*d, x, w_gate, w_up, b_gate, b_up, h, gate, up, st); break;
    case PS_DTYPE_BF16: rc = forward_typed<bf16>(*d, x, w_gate, w_up, b_gate, b_up, h, gate, up, st); break;
    default: rc = forward_typed<f16>(*d, x, w_gate, w_up, b_gate, b_up, h, gate, up, st); break;
  }
  return rc ? rc : hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

size_t ps_gated_linear_backward_workspace_bytes(const PsGatedLinearDesc* d) {
  const void* p = reinterpret_cast<const void*>(16);
  return check(d, p, p, p) ? 0 : backward_plan(*d).total;
}

int ps_gated_linear_backward(const PsGatedLinearDesc* d, const void* x, const void* w_gate, const void* w_up,
                             const void* b_gate, const void* b_up, const float* gate, const float* up, const void* dh,
                             void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (int rc = check(d, x, w_gate, w_up)) return rc;
  if (!dh || !workspace || !aligned16(workspace) || d->dh_row_stride < d->hidden) return PS_ERR_BAD_ARG;
  if (d->dtype == PS_DTYPE_F32 && (!gate || !up)) return PS_ERR_BAD_ARG;
  if (!aligned16(dx) || !aligned16(dw_gate) || !aligned16(dw_up)) return PS_ERR_BAD_ARG;
  if (workspace_bytes < backward_plan(*d).total) return PS_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  int rc;
  switch (d->dtype) {
    case PS_DTYPE_F32: rc = backward_typed<float>(*d, x, w_gate, w_up, b_gate, b_up, gate, up, dh, dx, dw_gate, dw_up, db_gate, db_up, ws, st); break;
    case PS_DTYPE_BF16: rc = backward_typed<bf16>(*d, x, w_gate, w_up, b_gate, b_up, gate, up, dh, dx, dw_gate, dw_up, db_gate, db_up, ws, st); break;
    default: rc = backward_typed<f16>(*d, x, w_gate, w_up, b_gate, b_up, gate, up, dh, dx, dw_gate, dw_up, db_gate, db_up, ws, st); break;
  }
  return rc ? rc : hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

}  // extern "C"
