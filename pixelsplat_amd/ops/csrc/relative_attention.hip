// Attention over a token grid with a learned relative position bias,
//   s = scale q.k + table[bucket[key - query]][head];  p = softmax(s) over the keys that are there;  o = p v,
// and its backward pass
//   dp = do.v;  ds = p (dp - do.o);  dq = scale ds k;  dk = scale ds^T q;  dv = p^T do;
//   d_table[b][head] = sum of ds over the batch and the pairs whose offset has bucket b.
//
// Tokens of a gh x gw grid are numbered by rows; code(t) = row (2 gw - 1) + column, so that the flattened (row, column)
// offset of a pair is code(key) - code(query) + origin.  A first small kernel spreads the table over the offsets, per
// head; a block then needs, for a tile of keys, one contiguous window of that, which it copies to LDS with the keys.
//
// Layout of the work.  A wave owns 32 queries (forward, dq) or 32 keys (dk, dv) as the COLUMNS of its products -- their
// operands stay in registers for the whole pass -- and streams the other side through LDS, double buffered, copied
// straight from global memory.  With columns in lanes, the 32 x 32 result of the first product has its rows in
// registers, which is what the second product contracts over: probabilities and ds go from the result registers into
// operand registers with no shuffle and no LDS (the order of the contraction index follows the registers', and the other
// operand is read in that order).  Softmax statistics are one value a lane.
//
// Logits are kept times log2(e): one exp2 an element.  Sums, statistics and do.o are fp32.  In 16-bit types the forward
// multiplies v by p rounded and by the rounded remainder, and for the backward it keeps o in fp32 too: a rounding in o
// would be the same in every ds of its row through do.o, and does not average out of sums over pairs (the table's
// gradient: 2.4 times the error of its own rounding at 8 buckets of 1785 tokens; forward 138 -> 173 us at 2 x 8 heads of
// 64 x 64 tokens of 64 in bf16).  The backward rounds ds, and p for dv, to the tensors' type as operands: these roundings
// are independent, as large as the results' own (the remainders here too: 447 -> 543 us).  A row's maximum and the inverse of
// its sum are kept apart: their sum as a logarithm would lose the second where all biases of a row are at the lowest value.
//
// d_table without atomics, in a fixed order.  In a row-numbered grid the pairs of one difference key - query have just two
// offsets: key and query in columns that ascend (key column >= query column), or that wrap.  So in the dq pass a wave
// writes a 32 x 32 tile of ds to LDS, in rows of 65 words with 33 zeros before each, and reads it along the diagonals:
// one difference a lane, neighbouring lanes in neighbouring banks, two sums; one where the tile's keys and queries each lie
// in one row of the grid, where a difference is one offset.  A tile's
// 63 differences are 32 final ones and 31 that the next tile of keys adds to, which stay in registers; the final ones
// go to the wave's row in memory.  Two small kernels add the rows by offset and the offsets by bucket.  (LDS float
// atomics on a table of offsets measured 1487 us for the dq pass at 2 x 8 heads, 64 x 64 tokens of 64.)
//
// Bound by the matrix instructions in fp32, by the vector instructions of the softmax in 16 bits, by the keys' and
// values' bytes for a few queries, which split the keys over blocks and join their partial results.  2 x 8 heads of 64 x 64
// tokens of 64 in bf16: forward 176 us, dq and the table's rows 254, dk and dv 201, the table's joins 45.  14 x 4 heads of
// 16 x 16 tokens of 128 in fp32: 35, 58, 53 and 23.  One query of 4 x 8 heads over 16384 keys of 64 in bf16: 28 us, 4.8 TB/s.
#include "mfma_tile.h"
#include "pixelsplat_ops.h"

namespace ps {
namespace {

__device__ const uint4 kZeros[1] = {{0, 0, 0, 0}};
__device__ const uint8_t kOnes[1] = {1};
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

typedef int intx4 __attribute__((ext_vector_type(4)));

struct Strides { int64_t b, h, t; };

struct Args {
  const void *q, *k, *v;
  Strides sq, sk, sv;
  const uint8_t* mask;            // [batch][nk] or NULL
  int64_t mask_b;
  const float* bias;              // [heads][offsets], times log2(e)
  int batch, heads, nq, nk, dim, gw, origin, offsets, q_start, nq_pad;
  float scale;
  int window;                     // floats of a window in LDS, a multiple of 64
  int col_tiles, splits, tiles_per_split;
  // forward
  void* out;                      // [batch][nq][heads][dim]
  float* o32;                     // the same in fp32 or NULL
  float* stats;                   // [2][batch heads][nq_pad] or NULL: maximum (log2, or up to 15 less; +inf: no keys), 1 / sum (0)
  float *part_o, *part_ml;        // [splits][batch heads nq][dim], [..][2]
  int join_lanes;                 // threads that share a row's splits
  // backward
  const void* dout;
  Strides sdo;
  const float* o_kept;            // fp32 o
  float* delta;                   // [batch heads][nq_pad]: do.o / sum
  void *dq, *dk, *dv;
  float *part_q, *part_k, *part_v;   // [splits][like dq, dk, dv] fp32, where there are splits
  float* diag_rows;               // [batch heads][nq_pad / 32][splits of dq][1 or 2][diag_pitch]
  int diag_pitch, diag_end;       // words of a row; differences that all splits' rows hold
};

__device__ __forceinline__ int code_of(int t, int gw) { return t + (int)((unsigned)t / (unsigned)gw) * (gw - 1); }

// whether the tokens first .. first + n - 1 all exist and lie in one row of the grid
__device__ __forceinline__ bool in_a_row(int first, int n, int tokens, int gw) {
  return first + n <= tokens && (int)((unsigned)first % (unsigned)gw) + n <= gw;
}

template <typename T> constexpr int kRows = sizeof(T) == 2 ? 64 : 32;   // rows of a streamed tile

// ---- streamed tiles: [rows][PITCH bytes], 16-byte chunk c of row r at c ^ swizzle(r) -----------------------------
// Both reads are free of bank conflicts: 16 rows at one chunk (the swizzle takes all values over 16 rows that do not
// differ in their bank already), and 4 rows at four neighbouring chunks (its high bits come from r & 3).
template <int PITCH>
__device__ __forceinline__ int swizzle(int r) {
  if (PITCH % 256 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
  if (PITCH % 256 == 128) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  return (r >> 2) & 3;
}

template <typename T, int PITCH>
__device__ __forceinline__ Frag<T> along(const char* tile, int row, int chunk) {
  return *reinterpret_cast<const Frag<T>*>(tile + row * PITCH + ((chunk ^ swizzle<PITCH>(row)) << 4));
}

// columns d0 .. d0 + 31 of the rows that registers kVec * s .. of a result hold
template <typename T, int PITCH>
__device__ __forceinline__ Frag<T> across(const char* tile, int row0, int s, int d0, int lane) {
  const int hi = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
    const int i = lane & 15, kr = i >> 2, col = (lane & 16) + (i & 3) * 4;
    const int r0 = row0 + 16 * s + 4 * hi + kr, r1 = r0 + 8, chunk = (d0 + col) >> 3, in = (col & 4) * 2;
    const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_shortx4*)(tile + r0 * PITCH + ((chunk ^ swizzle<PITCH>(r0)) << 4) + in));
    const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_shortx4*)(tile + r1 * PITCH + ((chunk ^ swizzle<PITCH>(r1)) << 4) + in));
    return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const int col = d0 + (lane & 31);
    Frag<T> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = row0 + 8 * s + 4 * hi + j;
      v[j] = *reinterpret_cast<const float*>(tile + r * PITCH + (((col >> 2) ^ swizzle<PITCH>(r)) << 4) + (col & 3) * 4);
    }
    return v;
  }
}

// registers kVec * s .. of a result as an operand
template <typename T>
__device__ __forceinline__ Frag<T> as_operand(const floatx16& r, int s) {
  Frag<T> f;
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e) f[e] = from_f32<T>(r[s * kVec<T> + e]);
  return f;
}

// fp16 holds less than ds = p (dp - do.o) can be, and few bits of what p leaves of it over many keys.  So ds enters its
// products times 2^up, a column's own, and the result is divided by it.  2^up takes the largest |ds| of the column so far to
// 2^15 at most, and to 2^14 when it is chosen; when a larger one comes, what was accumulated shrinks, as it does for a new maximum of a
// softmax.  Infinities stay infinities and are not counted.  p for dv, at most 1, enters times 2^kUpOfP.
// (Backward of 2 x 8 heads of 64 x 64 tokens of 64: 498 us without, 552 with it, 435 in bf16, which needs none of it.)
constexpr int kUpFirst = 80;             // of a column that has seen zeros only
constexpr int kUpOfP = 14;
template <int N>
__device__ __forceinline__ void into_range(floatx16& ds, int& up, floatx16 (&acc)[N]) {
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
  top = fmaxf(top, __shfl_xor(top, 32));
  if (__any(ldexpf(top, up) > 32768.f)) {
    top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]) < kInf ? fabsf(ds[r]) : 0.f);
    top = fmaxf(top, __shfl_xor(top, 32));
    const int to = ldexpf(top, up) > 32768.f ? 14 - ilogbf(top) : up;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][r] = ldexpf(acc[t][r], to - up);
    up = to;
  }
  const float by = ldexpf(1.f, up);
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] *= by;
}

// what as_operand left of them
template <typename T>
__device__ __forceinline__ Frag<T> remainder(const floatx16& r, int s, const Frag<T>& of) {
  Frag<T> f;
#pragma unroll
  for (int e = 0; e < kVec<T>; ++e) f[e] = from_f32<T>(r[s * kVec<T> + e] - to_f32(of[e]));
  return f;
}

// rows `bits` of the tile at `base` (row stride `stride` elements); rows that are not there become zeros
template <typename T, int PITCH, int ROWS, int WAVES>
__device__ __forceinline__ void copy_tile(const T* base, int64_t stride, int dim, uint64_t bits, char* tile, int wave,
                                          int lane) {
  constexpr int kChunks = PITCH / 16, kPieces = ROWS * PITCH / 1024;
#pragma unroll
  for (int j = 0; j < kPieces / WAVES; ++j) {
    const int pos = (j * WAVES + wave) * 64 + lane, row = pos / kChunks;
    const int d = ((pos % kChunks) ^ swizzle<PITCH>(row)) * kVec<T>;
    const bool on = ((bits >> row) & 1) && d < dim;
    copy_known(on ? (const void*)(base + (row * (int)stride + d)) : (const void*)kZeros, tile + (j * WAVES + wave) * 1024);
  }
}

// offsets first .. first + window of the head's bias
template <int WAVES>
__device__ __forceinline__ void copy_window(const float* bias, int offsets, int first, int window, float* lds, int wave,
                                            int lane) {
  for (int i = wave * 64; i < window; i += WAVES * 64)
    copy_word_known(bias + min(max(first + i + lane, 0), offsets - 1), lds + i);
}

// a lane's column operand: 16-byte chunks 2 s + hi of its row
template <typename T, int DP>
__device__ __forceinline__ void load_columns(Frag<T> (&f)[DP / kFragK<T>], const T* row, bool on, int dim, int hi) {
#pragma unroll
  for (int s = 0; s < DP / kFragK<T>; ++s) {
    const int d = (2 * s + hi) * kVec<T>;
    f[s] = *reinterpret_cast<const Frag<T>*>(on && d < dim ? (const void*)(row + d) : (const void*)kZeros);
  }
}

// Order of a product's LDS reads and matrix instructions in fp32: reads run AHEAD of them.  Left alone, the compiler puts
// each read in front of its use and waits for it, 64 cycles of matrix work at a time (forward 38 -> 34 us, dq 62 -> 57
// at 14 x 4 heads of 256 tokens of 128).
template <int READS, int PRODUCTS, int AHEAD>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < READS - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / READS, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS - (READS - AHEAD) * (PRODUCTS / READS), 0);
}

// s = s scale + bias for 32 rows.  codes: the rows' distances in the window; `line`: they are consecutive, `base` is the
// first row's entry and `step` + or - 1 (addresses are then the lane's and a constant: an instruction an element less).
template <int STEP>
__device__ __forceinline__ void add_bias(floatx16& s, float scale, const float* window, const int* codes, bool line,
                                         const float* base, int u, int hi) {
  if (line) {
    const float* from = base + STEP * 4 * hi;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], scale, from[STEP * (u * 32 + 8 * (r >> 2) + (r & 3))]);
  } else {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const intx4 c = *reinterpret_cast<const intx4*>(codes + u * 32 + 8 * a + 4 * hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * a + j] = fmaf(s[4 * a + j], scale, window[c[j]]);
    }
  }
}

// the columns' result [DP x 32], transposed into rows of `out` (dim elements each), times `by`
template <typename T, int DP>
__device__ __forceinline__ void store_columns(const floatx16 (&acc)[DP / 32], float by, T* row, int dim, int hi) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = t * 32 + 8 * a + 4 * hi;
      if (d < dim) {                                   // dim is a multiple of 4
        Pack<T, 4> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v.v[j] = from_f32<T>(acc[t][4 * a + j] * by);
        *reinterpret_cast<Pack<T, 4>*>(row + d) = v;
      }
    }
}

template <typename T, int DP, int WAVES>
struct Lds {                                            // bytes
  static constexpr int kTile = kRows<T> * DP * (int)sizeof(T);
  static constexpr int kRowData = 64 * 4;               // one word a row
  static constexpr int kWindow = 2 * kTile + 4 * kRowData;
  // [2][first tile | second tile | codes | row data 1 | 2 | 3 | window]
  __host__ __device__ static int buffer(int window) { return kWindow + window * 4; }
};

// what the wave wrote to LDS before is what its lanes read after
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The byte that says whether a row of a tile is there: loaded a tile ahead and without a branch, so that nothing waits for
// it before it is used.
__device__ __forceinline__ uint8_t mask_byte(const uint8_t* mask, int row, int count) {
  return *(mask ? mask + min(row, count - 1) : kOnes);
}

// ---------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) spread_table_kernel(int heads, int offsets, int buckets, const int32_t* __restrict__ map,
                                                           const void* __restrict__ table, int table_f32,
                                                           float* __restrict__ bias) {
  const int o = blockIdx.x * 256 + threadIdx.x;
  if (o >= offsets) return;
  const int bucket = map[o];
  const bool on = bucket >= 0 && bucket < buckets;
  for (int h = blockIdx.y; h < heads; h += gridDim.y) {
    const float v = on ? load_param<T>(table, table_f32, (int64_t)bucket * heads + h) : 0.f;
    // a bias at the types' lowest value stays finite after the factor: a row of nothing else is uniform, not empty
    float b = v * kLog2e;
    if (b < -3e38f && v != -kInf) b = -3e38f;
    if (b > 3e38f && v != kInf) b = 3e38f;
    bias[(int64_t)h * offsets + o] = b;
  }
}

template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, DP == 128 && (sizeof(T) == 4 || WAVES == 1) ? 1 : 2) attention_forward_kernel(Args p) {
  constexpr int PITCH = DP * sizeof(T), ROWS = kRows<T>, SUBS = ROWS / 32, KF = DP / kFragK<T>, PF = 32 / kFragK<T>;
  constexpr float kLift = kNarrow<T> ? 7.f : 0.f;
  typedef Lds<T, DP, WAVES> L;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, hi = lane >> 5;
  const int tile = blockIdx.x % p.col_tiles, bh = blockIdx.x / p.col_tiles, split = blockIdx.y;
  const int b = bh / p.heads, h = bh % p.heads;
  const int first = tile * WAVES * 32, last = min(first + WAVES * 32, p.nq) - 1;
  const int qi = first + wave * 32 + (lane & 31);
  const bool q_on = qi < p.nq;
  const int code_last = code_of(p.q_start + max(last, 0), p.gw);
  const int q_off = code_last - code_of(p.q_start + min(qi, max(last, 0)), p.gw);

  Frag<T> qf[KF];
  load_columns<T, DP>(qf, (const T*)p.q + b * p.sq.b + h * p.sq.h + qi * p.sq.t, q_on, p.dim, hi);
  const T* kb = (const T*)p.k + b * p.sk.b + h * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + h * p.sv.h;
  const uint8_t* mask = p.mask ? p.mask + b * p.mask_b : nullptr;
  const float* bias = p.bias + (int64_t)h * p.offsets;
  const int bytes = L::buffer(p.window);

  floatx16 o[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) o[t] = zero16();
  float m = -kInf, l = 0.f;

  const int tiles = (p.nk + ROWS - 1) / ROWS;
  const int t0 = split * p.tiles_per_split, t1 = min(t0 + p.tiles_per_split, tiles);
  uint64_t bits = 0, next_bits = 0;
  uint8_t there = mask_byte(mask, t0 * ROWS + lane, p.nk);
  auto load = [&](int kt, int buf) {
    char* at = lds + buf * bytes;
    const int k0 = kt * ROWS;
    next_bits = __ballot(there != 0 && lane < ROWS && k0 + lane < p.nk);
    there = mask_byte(mask, k0 + ROWS + lane, p.nk);
    copy_tile<T, PITCH, ROWS, WAVES>(kb + k0 * p.sk.t, p.sk.t, p.dim, next_bits, at, wave, lane);
    copy_tile<T, PITCH, ROWS, WAVES>(vb + k0 * p.sv.t, p.sv.t, p.dim, next_bits, at + L::kTile, wave, lane);
    int* codes = reinterpret_cast<int*>(at + 2 * L::kTile);
    const int c0 = code_of(k0, p.gw);
    if ((int)threadIdx.x < ROWS) codes[threadIdx.x] = code_of(min(k0 + (int)threadIdx.x, p.nk - 1), p.gw) - c0;
    copy_window<WAVES>(bias, p.offsets, c0 - code_last + p.origin, p.window,
                       reinterpret_cast<float*>(at + L::kWindow), wave, lane);
  };
  if (t0 < t1) load(t0, 0);
  __syncthreads();
  for (int kt = t0; kt < t1; ++kt) {
    const int buf = (kt - t0) & 1;
    bits = next_bits;
    if (kt + 1 < t1) load(kt + 1, buf ^ 1);
    const char* tk = lds + buf * bytes;
    const char* tv = tk + L::kTile;
    const int* codes = reinterpret_cast<const int*>(tk + 2 * L::kTile);
    const float* window = reinterpret_cast<const float*>(tk + L::kWindow) + q_off;

    floatx16 s[SUBS];
    float top = -kInf;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      s[u] = zero16();
#pragma unroll
      for (int f = 0; f < KF; ++f)
        s[u] = mfma(along<T, PITCH>(tk, u * 32 + (lane & 31), 2 * f + hi), qf[f], s[u]);
      if (sizeof(T) == 4) reads_ahead<KF, 4 * KF, 4>();
    }
    const bool line = in_a_row(kt * ROWS, ROWS, p.nk, p.gw);
#pragma unroll
    for (int u = 0; u < SUBS; ++u) add_bias<1>(s[u], p.scale, window, codes, line, window, u, hi);
    if (bits != (ROWS == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const uint32_t mine = (uint32_t)(bits >> (32 * u)) >> (4 * hi);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((mine >> (8 * (r >> 2) + (r & 3))) & 1)) s[u][r] = -kInf;
      }
    }
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    top = fmaxf(top, __shfl_xor(top, 32));
    // A new maximum: what there is shrinks.  Not for every one: terms of up to 2^8 are as exact as those of up to 1.  In fp16,
    // which ends at 2^-24 and 2^16, the largest term is 2^7 .. 2^15: a term 2^-25 of it is lost, and 2^18 keys of those are
    // a hundredth of the result; 2^-32 of it is not missed.
    if (__any(top > m + (8.f + kLift))) {
      const float nm = fmaxf(m, top - kLift);
      const float by = __builtin_amdgcn_exp2f(m - (nm == -kInf ? 0.f : nm));
      m = nm;
      l *= by;
#pragma unroll
      for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= by;
    }
    const float base = m == -kInf ? 0.f : m;           // nothing yet: exp2(-inf) = 0
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - base);
        l += s[u][r];
      }
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
      for (int f = 0; f < PF; ++f) {
        const Frag<T> pf = as_operand<T>(s[u], f);
        Frag<T> v[DP / 32];
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) v[t] = across<T, PITCH>(tv, u * 32, f, t * 32, lane);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) o[t] = mfma(v[t], pf, o[t]);
        if (sizeof(T) == 2) {
          const Frag<T> rest = remainder<T>(s[u], f, pf);
#pragma unroll
          for (int t = 0; t < DP / 32; ++t) o[t] = mfma(v[t], rest, o[t]);
        }
      }
    if (sizeof(T) == 4) reads_ahead<4 * PF * (DP / 32), 4 * PF * (DP / 32), 8>();
    __syncthreads();
  }
  l += __shfl_xor(l, 32);
  if (p.splits > 1) {
    if (!q_on) return;
    const int64_t row = ((int64_t)split * p.batch * p.heads + bh) * p.nq + qi;
    if (hi == 0) {
      p.part_ml[row * 2] = m;
      p.part_ml[row * 2 + 1] = l;
    }
    store_columns<float, DP>(o, 1.f, p.part_o + row * p.dim, p.dim, hi);
    return;
  }
  const float by = q_on && l != 0.f ? 1.f / l : 0.f;   // a row without keys is zero
  if (p.stats && hi == 0 && qi < p.nq_pad) {
    const int64_t at = (int64_t)bh * p.nq_pad + qi;
    p.stats[at] = q_on && l != 0.f ? m : kInf;
    p.stats[(int64_t)p.batch * p.heads * p.nq_pad + at] = by;
  }
  if (!q_on) return;
  const int64_t row = (((int64_t)b * p.nq + qi) * p.heads + h) * p.dim;
  store_columns<T, DP>(o, by, (T*)p.out + row, p.dim, hi);
  if (p.o32) store_columns<float, DP>(o, by, p.o32 + row, p.dim, hi);
}

// The splits of a row, joined.  A thread takes 4 columns and every join_lanes-th split; those of a row meet in LDS.
template <typename T>
__global__ void __launch_bounds__(256) join_splits_kernel(Args p) {
  __shared__ float lds[256][7];
  const int per = p.dim / 4, lanes = p.join_lanes, row_threads = per * lanes, in_block = 256 / row_threads;
  const int in = threadIdx.x % row_threads, part = in / per, d = (in % per) * 4;
  const int64_t at = (int64_t)blockIdx.x * in_block + threadIdx.x / row_threads, rows = (int64_t)p.batch * p.heads * p.nq_pad;
  const int bh = (int)(at / p.nq_pad), qi = (int)(at % p.nq_pad);
  const bool on = (int)threadIdx.x < in_block * row_threads && at < rows && qi < p.nq;
  const int64_t all = (int64_t)p.batch * p.heads * p.nq, row = (int64_t)bh * p.nq + qi;
  float m = -kInf, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  if (on) {
#pragma unroll 4
    for (int s = part; s < p.splits; s += lanes) m = fmaxf(m, p.part_ml[(s * all + row) * 2]);
    const float base = m == -kInf ? 0.f : m;
#pragma unroll 4
    for (int s = part; s < p.splits; s += lanes) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * all + row) * 2);
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * all + row) * p.dim + d);
      const float by = __builtin_amdgcn_exp2f(ml.x - base);
      l = fmaf(ml.y, by, l);
      o[0] = fmaf(v.x, by, o[0]);
      o[1] = fmaf(v.y, by, o[1]);
      o[2] = fmaf(v.z, by, o[2]);
      o[3] = fmaf(v.w, by, o[3]);
    }
  }
  if (lanes > 1) {
    float* mine = lds[threadIdx.x];
    mine[0] = m;
    mine[1] = l;
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[2 + j] = o[j];
    __syncthreads();
    if (on && part == 0) {
      float top = m;
      for (int k = 1; k < lanes; ++k) top = fmaxf(top, lds[threadIdx.x + k * per][0]);
      const float base = top == -kInf ? 0.f : top;
      l = o[0] = o[1] = o[2] = o[3] = 0.f;
      for (int k = 0; k < lanes; ++k) {
        const float* other = lds[threadIdx.x + k * per];
        const float by = __builtin_amdgcn_exp2f(other[0] - base);
        l = fmaf(other[1], by, l);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(other[2 + j], by, o[j]);
      }
      m = top;
    }
  }
  if (part != 0 || (int)threadIdx.x >= in_block * row_threads || at >= rows) return;
  const float by = on && l != 0.f ? 1.f / l : 0.f;
  if (p.stats && d == 0) {
    p.stats[at] = by != 0.f ? m : kInf;
    p.stats[rows + at] = by;
  }
  if (!on) return;
  const int64_t to = (((int64_t)(bh / p.heads) * p.nq + qi) * p.heads + bh % p.heads) * p.dim + d;
  Pack<T, 4> v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v.v[j] = from_f32<T>(o[j] * by);
    if (p.o32) p.o32[to + j] = o[j] * by;
  }
  *reinterpret_cast<Pack<T, 4>*>((T*)p.out + to) = v;
}

// ---------------------------------------------------------------------------------------------------------------
constexpr int kDiagRow = 65, kDiagZeros = 33, kDiag = 33 * kDiagRow + 3;      // words; of a wave: 33 rows, a multiple of 4

// dq, do.o and the diagonals of ds (SUMS a difference; 0: none).  Columns are queries, rows are keys, as in the forward.
template <typename T, int DP, int WAVES, int SUMS>
__global__ void __launch_bounds__(WAVES * 64, sizeof(T) == 4 || (SUMS && DP == 128) ? 1 : 2) attention_dq_kernel(Args p) {
  constexpr int PITCH = DP * sizeof(T), ROWS = kRows<T>, SUBS = ROWS / 32, KF = DP / kFragK<T>, PF = 32 / kFragK<T>;
  typedef Lds<T, DP, WAVES> L;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, hi = lane >> 5;
  const int tile = blockIdx.x % p.col_tiles, bh = blockIdx.x / p.col_tiles, split = blockIdx.y;
  const int b = bh / p.heads, h = bh % p.heads;
  const int first = tile * WAVES * 32, last = max(min(first + WAVES * 32, p.nq) - 1, 0);
  const int qi = first + wave * 32 + (lane & 31);
  const bool q_on = qi < p.nq;
  const int code_last = code_of(p.q_start + last, p.gw);
  const int code_mine = code_of(p.q_start + min(qi, last), p.gw);
  const int q_off = code_last - code_mine;
  const int bytes = L::buffer(p.window);

  Frag<T> qf[KF], df[KF];
  load_columns<T, DP>(qf, (const T*)p.q + b * p.sq.b + h * p.sq.h + qi * p.sq.t, q_on, p.dim, hi);
  load_columns<T, DP>(df, (const T*)p.dout + b * p.sdo.b + h * p.sdo.h + qi * p.sdo.t, q_on, p.dim, hi);
  float delta = 0.f;
  if (q_on) {
    const float* o = p.o_kept + (((int64_t)b * p.nq + qi) * p.heads + h) * p.dim;
#pragma unroll
    for (int f = 0; f < KF; ++f)
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e) {
        const int d = (2 * f + hi) * kVec<T> + e;
        if (d < p.dim) delta = fmaf(to_f32(df[f][e]), o[d], delta);
      }
  }
  delta += __shfl_xor(delta, 32);
  float m = kInf, inv = 0.f;
  if (qi < p.nq_pad) {
    const int64_t at = (int64_t)bh * p.nq_pad + qi;
    m = p.stats[at];
    inv = p.stats[(int64_t)p.batch * p.heads * p.nq_pad + at];
    delta *= inv;
    if (hi == 0 && split == 0) p.delta[at] = delta;
  }

  // The wave's tile of ds and its row: entry i holds the difference i - 31 + (first key's token) - (first query's token).
  const int tiles = (p.nk + ROWS - 1) / ROWS;
  const int t0 = split * p.tiles_per_split, t1 = min(t0 + p.tiles_per_split, tiles);
  const bool wave_on = first + wave * 32 < p.nq;
  float* diag = reinterpret_cast<float*>(lds + 2 * bytes) + wave * kDiag;
  float* diag_row = nullptr;
  bool wave_line = false;                               // the wave's queries lie in one row of the grid
  int wave_col = 0, diff_col = 0, step_col = 0;         // columns: of the first query, of the lane's difference, 32 more
  float carry[2] = {0.f, 0.f};
  if (SUMS) {
    diag_row = p.diag_rows + (((int64_t)bh * (p.nq_pad / 32) + (first / 32 + wave)) * p.splits + split) * SUMS * p.diag_pitch;
    for (int i = lane; i < kDiag; i += 64) diag[i] = 0.f;
    if (SUMS == 2) {
      const int token = p.q_start + first + wave * 32;
      wave_col = __builtin_amdgcn_readfirstlane((unsigned)token % (unsigned)p.gw);
      wave_line = wave_col + 32 <= p.gw;
      step_col = 32 % p.gw;
      diff_col = (t0 * ROWS + lane - 31 - token) % p.gw;
      if (diff_col < 0) diff_col += p.gw;
    }
  }

  const T* kb = (const T*)p.k + b * p.sk.b + h * p.sk.h;
  const T* vb = (const T*)p.v + b * p.sv.b + h * p.sv.h;
  const uint8_t* mask = p.mask ? p.mask + b * p.mask_b : nullptr;
  const float* bias = p.bias + (int64_t)h * p.offsets;
  floatx16 dq[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) dq[t] = zero16();
  int up = kNarrow<T> ? kUpFirst : 0;

  uint64_t bits = 0, next_bits = 0;
  uint8_t there = mask_byte(mask, t0 * ROWS + lane, p.nk);
  auto load = [&](int kt, int buf) {
    char* at = lds + buf * bytes;
    const int k0 = kt * ROWS;
    next_bits = __ballot(there != 0 && lane < ROWS && k0 + lane < p.nk);
    there = mask_byte(mask, k0 + ROWS + lane, p.nk);
    copy_tile<T, PITCH, ROWS, WAVES>(kb + k0 * p.sk.t, p.sk.t, p.dim, next_bits, at, wave, lane);
    copy_tile<T, PITCH, ROWS, WAVES>(vb + k0 * p.sv.t, p.sv.t, p.dim, next_bits, at + L::kTile, wave, lane);
    int* codes = reinterpret_cast<int*>(at + 2 * L::kTile);
    const int c0 = code_of(k0, p.gw);
    if ((int)threadIdx.x < ROWS) codes[threadIdx.x] = code_of(min(k0 + (int)threadIdx.x, p.nk - 1), p.gw) - c0;
    copy_window<WAVES>(bias, p.offsets, c0 - code_last + p.origin, p.window,
                       reinterpret_cast<float*>(at + L::kWindow), wave, lane);
  };
  load(t0, 0);
  __syncthreads();
  for (int kt = t0; kt < t1; ++kt) {
    const int buf = (kt - t0) & 1;
    bits = next_bits;
    if (kt + 1 < t1) load(kt + 1, buf ^ 1);
    const char* tk = lds + buf * bytes;
    const char* tv = tk + L::kTile;
    const int* codes = reinterpret_cast<const int*>(tk + 2 * L::kTile);
    const float* window = reinterpret_cast<const float*>(tk + L::kWindow) + q_off;
    const bool whole = bits == (ROWS == 64 ? ~0ull : 0xffffffffull);
    const bool line = in_a_row(kt * ROWS, ROWS, p.nk, p.gw);
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      floatx16 s = zero16(), ds = zero16();
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        s = mfma(along<T, PITCH>(tk, u * 32 + (lane & 31), 2 * f + hi), qf[f], s);
        ds = mfma(along<T, PITCH>(tv, u * 32 + (lane & 31), 2 * f + hi), df[f], ds);
      }
      if (sizeof(T) == 4) reads_ahead<2 * KF, 8 * KF, 4>();
      add_bias<1>(s, p.scale, window, codes, line, window, u, hi);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(s[r] - m) * fmaf(ds[r], inv, -delta);
      if (!whole) {
        const uint32_t mine = (uint32_t)(bits >> (32 * u)) >> (4 * hi);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((mine >> (8 * (r >> 2) + (r & 3))) & 1)) ds[r] = 0.f;
      }
      if (SUMS && wave_on) {
#pragma unroll
        for (int r = 0; r < 16; ++r) diag[(lane & 31) * kDiagRow + kDiagZeros + result_row(r, hi)] = ds[r];
        wave_order();
        float sum[2] = {0.f, 0.f};
        const float* at = diag + lane + (kDiagZeros - 31);  // query i of the wave, key i + lane - 31 of the tile
        if (SUMS == 1 || (wave_line && in_a_row(kt * ROWS + u * 32, 32, p.nk, p.gw))) {
          // both in one row of the grid: a difference is one offset, which the first query that has it tells
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[0] += at[i * (kDiagRow + 1)];
          if (SUMS == 2 && wave_col + max(31 - lane, 0) + diff_col >= p.gw) {
            sum[1] = sum[0];
            sum[0] = 0.f;
          }
        } else {
          int col = wave_col;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = at[i * (kDiagRow + 1)];
            const bool wraps = col + diff_col >= p.gw;
            sum[0] += wraps ? 0.f : v;
            sum[1] += wraps ? v : 0.f;
            col = col + 1 == p.gw ? 0 : col + 1;
          }
        }
        wave_order();
        if (SUMS == 2) {
          diff_col += step_col;
          if (diff_col >= p.gw) diff_col -= p.gw;
        }
#pragma unroll
        for (int c = 0; c < SUMS; ++c) {
          if (lane < 32) diag_row[c * p.diag_pitch + (kt - t0) * ROWS + u * 32 + lane] = sum[c] + carry[c];
          carry[c] = __shfl_xor(sum[c], 32);
        }
      }
      if constexpr (kNarrow<T>) into_range(ds, up, dq);
#pragma unroll
      for (int f = 0; f < PF; ++f) {
        const Frag<T> sf = as_operand<T>(ds, f);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) dq[t] = mfma(across<T, PITCH>(tk, u * 32, f, t * 32, lane), sf, dq[t]);
      }
      if (sizeof(T) == 4) reads_ahead<4 * PF * (DP / 32), 4 * PF * (DP / 32), 8>();
    }
    __syncthreads();
  }
  if (SUMS && wave_on && lane < 32) {
#pragma unroll
    for (int c = 0; c < SUMS; ++c) diag_row[c * p.diag_pitch + (t1 - t0) * ROWS + lane] = carry[c];
  }
  if (q_on && p.dq) {
    const int64_t row = (((int64_t)b * p.nq + qi) * p.heads + h) * p.dim;
    const float by = ldexpf(p.scale * (1.f / kLog2e), -up);
    if (p.splits > 1)
      store_columns<float, DP>(dq, by, p.part_q + split * ((int64_t)p.batch * p.nq * p.heads * p.dim) + row, p.dim, hi);
    else
      store_columns<T, DP>(dq, by, (T*)p.dq + row, p.dim, hi);
  }
}

// dk, dv.  Columns are keys, rows are queries.
template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, DP == 128 ? 1 : 2) attention_dkv_kernel(Args p) {
  constexpr int PITCH = DP * sizeof(T), ROWS = kRows<T>, SUBS = ROWS / 32, KF = DP / kFragK<T>, PF = 32 / kFragK<T>;
  typedef Lds<T, DP, WAVES> L;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, hi = lane >> 5;
  const int tile = blockIdx.x % p.col_tiles, bh = blockIdx.x / p.col_tiles, split = blockIdx.y;
  const int b = bh / p.heads, h = bh % p.heads;
  const int first = tile * WAVES * 32, last = min(first + WAVES * 32, p.nk) - 1;
  const int ki = first + wave * 32 + (lane & 31);
  const bool in = ki < p.nk;
  const bool k_on = in && (p.mask == nullptr || p.mask[b * p.mask_b + ki] != 0);
  const int code_first = code_of(first, p.gw);
  const int k_off = code_of(min(ki, last), p.gw) - code_first;
  const int bytes = L::buffer(p.window);

  Frag<T> kf[KF], vf[KF];
  load_columns<T, DP>(kf, (const T*)p.k + b * p.sk.b + h * p.sk.h + ki * p.sk.t, k_on, p.dim, hi);
  load_columns<T, DP>(vf, (const T*)p.v + b * p.sv.b + h * p.sv.h + ki * p.sv.t, k_on, p.dim, hi);
  const T* qb = (const T*)p.q + b * p.sq.b + h * p.sq.h;
  const T* db = (const T*)p.dout + b * p.sdo.b + h * p.sdo.h;
  const float* bias = p.bias + (int64_t)h * p.offsets;
  const float* stat_rows[3] = {p.stats + (int64_t)bh * p.nq_pad, p.stats + ((int64_t)p.batch * p.heads + bh) * p.nq_pad,
                               p.delta + (int64_t)bh * p.nq_pad};

  floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) dk[t] = dv[t] = zero16();
  int up = kNarrow<T> ? kUpFirst : 0;

  const int tiles = (p.nq + ROWS - 1) / ROWS;
  const int t0 = split * p.tiles_per_split, t1 = min(t0 + p.tiles_per_split, tiles);
  auto load = [&](int qt, int buf) {
    char* at = lds + buf * bytes;
    const int q0 = qt * ROWS, end = min(q0 + ROWS, p.nq) - 1;
    const uint64_t bits = __ballot(lane < ROWS && q0 + lane < p.nq);
    copy_tile<T, PITCH, ROWS, WAVES>(qb + q0 * p.sq.t, p.sq.t, p.dim, bits, at, wave, lane);
    copy_tile<T, PITCH, ROWS, WAVES>(db + q0 * p.sdo.t, p.sdo.t, p.dim, bits, at + L::kTile, wave, lane);
    // codes count down from the tile's last query, whose window entry is the first
    int* codes = reinterpret_cast<int*>(at + 2 * L::kTile);
    float* rows = reinterpret_cast<float*>(at + 2 * L::kTile + L::kRowData);
    const int c1 = code_of(p.q_start + end, p.gw);
    if ((int)threadIdx.x < ROWS)
      codes[threadIdx.x] = c1 - code_of(p.q_start + min(q0 + (int)threadIdx.x, end), p.gw);
    for (int i = wave; i < 3; i += WAVES)                          // nq_pad holds whole tiles
      copy_word_known(stat_rows[i] + q0 + min(lane, ROWS - 1), rows + 64 * i);
    copy_window<WAVES>(bias, p.offsets, code_first - c1 + p.origin, p.window,
                       reinterpret_cast<float*>(at + L::kWindow), wave, lane);
  };
  load(t0, 0);
  __syncthreads();
  for (int qt = t0; qt < t1; ++qt) {
    const int buf = (qt - t0) & 1;
    if (qt + 1 < t1) load(qt + 1, buf ^ 1);
    const char* tq = lds + buf * bytes;
    const char* td = tq + L::kTile;
    const int* codes = reinterpret_cast<const int*>(tq + 2 * L::kTile);
    const float* rows = reinterpret_cast<const float*>(tq + 2 * L::kTile + L::kRowData);
    const float* window = reinterpret_cast<const float*>(tq + L::kWindow) + k_off;
    // whole tiles of queries in one row of the grid: the last one's entry is the first
    const bool line = qt * ROWS + ROWS <= p.nq && in_a_row(p.q_start + qt * ROWS, ROWS, p.nk, p.gw);
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      floatx16 s = zero16(), ds = zero16();
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        s = mfma(along<T, PITCH>(tq, u * 32 + (lane & 31), 2 * f + hi), kf[f], s);
        ds = mfma(along<T, PITCH>(td, u * 32 + (lane & 31), 2 * f + hi), vf[f], ds);
      }
      add_bias<-1>(s, p.scale, window, codes, line, window + ROWS - 1, u, hi);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx4 e = *reinterpret_cast<const floatx4*>(rows + u * 32 + 8 * a + 4 * hi);
        const floatx4 w = *reinterpret_cast<const floatx4*>(rows + 64 + u * 32 + 8 * a + 4 * hi);
        const floatx4 g = *reinterpret_cast<const floatx4*>(rows + 128 + u * 32 + 8 * a + 4 * hi);
        const float es[4] = {e.x, e.y, e.z, e.w}, ws[4] = {w.x, w.y, w.z, w.w}, gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * a + j;
          const float pr = __builtin_amdgcn_exp2f(s[r] - es[j]);
          s[r] = kNarrow<T> ? pr * ws[j] * (float)(1 << kUpOfP) : pr * ws[j];
          ds[r] = pr * fmaf(ds[r], ws[j], -gs[j]);
        }
      }
      if constexpr (kNarrow<T>) into_range(ds, up, dk);
#pragma unroll
      for (int f = 0; f < PF; ++f) {
        const Frag<T> pf = as_operand<T>(s, f), sf = as_operand<T>(ds, f);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
          dv[t] = mfma(across<T, PITCH>(td, u * 32, f, t * 32, lane), pf, dv[t]);
          dk[t] = mfma(across<T, PITCH>(tq, u * 32, f, t * 32, lane), sf, dk[t]);
        }
      }
    }
    __syncthreads();
  }
  if (in) {
    const int64_t row = (((int64_t)b * p.nk + ki) * p.heads + h) * p.dim;
    if (!k_on) {                                        // a key that is not there: its column held what no row saw
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) dk[t] = dv[t] = zero16();
    }
    const float by = ldexpf(p.scale * (1.f / kLog2e), -up), by_v = kNarrow<T> ? 1.f / (1 << kUpOfP) : 1.f;
    const int64_t part = split * ((int64_t)p.batch * p.nk * p.heads * p.dim) + row;
    if (p.dk && p.splits > 1) store_columns<float, DP>(dk, by, p.part_k + part, p.dim, hi);
    else if (p.dk) store_columns<T, DP>(dk, by, (T*)p.dk + row, p.dim, hi);
    if (p.dv && p.splits > 1) store_columns<float, DP>(dv, by_v, p.part_v + part, p.dim, hi);
    else if (p.dv) store_columns<T, DP>(dv, by_v, (T*)p.dv + row, p.dim, hi);
  }
}

// d_offsets[head][o] = the sum of the waves' rows at the offset's difference: 16 offsets a block, 16 threads an offset take
// every 16th row
__global__ void __launch_bounds__(256) join_diagonals_kernel(Args p, int sums, double* __restrict__ d_offsets) {
  __shared__ double lds[16][17];
  const int o = blockIdx.x * 16 + (threadIdx.x & 15), h = blockIdx.y, part = threadIdx.x >> 4;
  const int waves = (p.nq + 31) / 32, pitch = 2 * p.gw - 1, per = p.nq_pad / 32;
  double t = 0;
  if (o < p.offsets) {
    const int dy = o / pitch - p.origin / pitch, dx = o % pitch - (p.gw - 1);
    const int at = dy * p.gw + dx + 31 + p.q_start;     // at the first wave; 32 more at each next
    const float* rows = p.diag_rows + (dx < 0 ? p.diag_pitch : 0) * (sums - 1);
    const int len = p.diag_pitch - 32, end = p.diag_end;        // a split's keys; what the waves' rows hold
    // the waves whose rows hold the difference
    const int w0 = at < 0 ? (-at + 31) / 32 : 0, w1 = at >= end ? 0 : min(waves, (end - 1 - at) / 32 + 1);
    const int n = max(w1 - w0, 1), all = w1 > w0 ? p.batch * n : 0;
    const int64_t pitch_w = (int64_t)p.splits * sums * p.diag_pitch;
    // (batch, wave) number part, part + 16, ..: a division here, none in the loop
    int b = part / n, w = part - b * n;
    const int step_b = 16 / n, step_w = 16 - step_b * n;
    const float* of_h = rows + (int64_t)h * per * pitch_w;
    const int64_t pitch_b = (int64_t)p.heads * per * pitch_w;
#pragma unroll 4
    for (int i = part; i < all; i += 16) {
      const float* row = of_h + b * pitch_b + (w0 + w) * pitch_w;
      const int u = at + 32 * (w0 + w);
      if (p.splits == 1) {
        t += row[u];
      } else {
        const int s = min(u / len, p.splits - 1), in = u - s * len;
        row += (int64_t)s * sums * p.diag_pitch;
        t += row[in];
        if (s > 0 && in < 32) t += row[in + len - (int64_t)sums * p.diag_pitch];   // the end of the split before
      }
      b += step_b;
      w += step_w;
      if (w >= n) {
        w -= n;
        ++b;
      }
    }
  }
  lds[part][threadIdx.x & 15] = t;
  __syncthreads();
  if (part == 0 && o < p.offsets) {
    for (int k = 1; k < 16; ++k) t += lds[k][threadIdx.x];
    d_offsets[(int64_t)h * p.offsets + o] = t;
  }
}

// dq, dk, dv of their splits' parts, in order
struct Parts {
  const float* from;
  void* to;
  int64_t count;          // elements, a multiple of 4
  int splits, blocks;
};
struct Gradients { Parts g[3]; };
template <typename T>
__global__ void __launch_bounds__(256) join_gradients_kernel(Gradients a) {
  int block = blockIdx.x;
  for (int k = 0; k < 3; ++k) {
    const Parts& q = a.g[k];
    if (block < q.blocks) {
      const int64_t i = ((int64_t)block * 256 + threadIdx.x) * 4;
      if (i >= q.count) return;
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < q.splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(q.from + s * q.count + i);
        t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
      }
      Pack<T, 4> out = {{from_f32<T>(t.x), from_f32<T>(t.y), from_f32<T>(t.z), from_f32<T>(t.w)}};
      *reinterpret_cast<Pack<T, 4>*>((T*)q.to + i) = out;
      return;
    }
    block -= q.blocks;
  }
}

constexpr int kJoinHeads = 8, kJoinList = 8192;
constexpr int kJoinLists = 512;          // of the longest map: a grid of 2^20 tokens has less than 2^22 offsets

// ranges[i] = lowest and highest bucket of entries kJoinList i .. of the map
__global__ void __launch_bounds__(256) bucket_ranges_kernel(int offsets, const int32_t* __restrict__ map, int2* __restrict__ ranges) {
  __shared__ int2 lds[4];
  const int end = min((int)(blockIdx.x + 1) * kJoinList, offsets);
  int lo = INT32_MAX, hi = INT32_MIN;
  for (int i = blockIdx.x * kJoinList + threadIdx.x; i < end; i += 256) {
    lo = min(lo, map[i]);
    hi = max(hi, map[i]);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    lo = min(lo, __shfl_xor(lo, m));
    hi = max(hi, __shfl_xor(hi, m));
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_int2(lo, hi);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) {
      lo = min(lo, lds[w].x);
      hi = max(hi, lds[w].y);
    }
    ranges[blockIdx.x] = make_int2(lo, hi);
  }
}

// d_table[bucket][head]: a block a bucket and 8 heads.  It lists the offsets of its bucket, in order -- kJoinList entries
// of the map at a time, a run of them a wave -- then 32 threads a head take the list's entries.  With `ranges` it passes over
// runs of entries that cannot hold its bucket.
template <typename T>
__global__ void __launch_bounds__(256) join_offsets_kernel(int heads, int offsets, int buckets, const int32_t* __restrict__ map,
                                                           const int2* __restrict__ ranges, const double* __restrict__ d_offsets,
                                                           void* __restrict__ d_table, int table_f32) {
  constexpr int kRun = kJoinList / 4;
  __shared__ int list[4][kRun];
  __shared__ int found[4];
  __shared__ double lds[32][kJoinHeads + 1];
  __shared__ uint64_t held[kJoinLists / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int j = threadIdx.x & (kJoinHeads - 1), h = blockIdx.y * kJoinHeads + j, part = threadIdx.x / kJoinHeads;
  const double* of_h = d_offsets + (int64_t)min(h, heads - 1) * offsets;
  for (int bucket = blockIdx.x; bucket < buckets; bucket += gridDim.x) {      // a launch has no 2^24 blocks of 256
    if (ranges) {
      for (int i = threadIdx.x; i < kJoinLists; i += 256) {
        const int2 r = i * kJoinList < offsets ? ranges[i] : make_int2(1, 0);
        const uint64_t hits = __ballot(r.x <= bucket && bucket <= r.y);
        if (lane == 0) held[i >> 6] = hits;
      }
      __syncthreads();
    }
    double t = 0;
    for (int base = 0; base < offsets; base += kJoinList) {
      const int at = base / kJoinList;
      if (ranges && !((held[at >> 6] >> (at & 63)) & 1)) continue;
      int mine[kRun / 64], n = 0;
      const int from = base + wave * kRun + lane;
#pragma unroll
      for (int i = 0; i < kRun / 64; ++i) mine[i] = from + i * 64 < offsets ? map[from + i * 64] : -1;
#pragma unroll
      for (int i = 0; i < kRun / 64; ++i) {
        const uint64_t hits = __ballot(mine[i] == bucket);
        if (mine[i] == bucket) list[wave][n + __popcll(hits & ((1ull << lane) - 1))] = from + i * 64;
        n += __popcll(hits);
      }
      if (lane == 0) found[wave] = n;
      __syncthreads();
      for (int w = 0; w < 4; ++w)
#pragma unroll 4
        for (int i = part; i < found[w]; i += 32) t += of_h[list[w][i]];
      __syncthreads();
    }
    lds[part][j] = t;
    __syncthreads();
    if (part == 0 && h < heads) {
      for (int k = 1; k < 32; ++k) t += lds[k][j];
      store_param<T>(d_table, table_f32, (int64_t)bucket * heads + h, (float)t);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
int count(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// codes that n neighbouring tokens span, less one, at most: a token a code, and gw - 1 more at the end of a row
int span_of(int n, int gh, int gw) {
  n = n < gh * gw ? n : gh * gw;
  int crossings = count(n - 1, gw);
  if (crossings > gh - 1) crossings = gh - 1;
  return (n - 1) + crossings * (gw - 1);
}

struct Split { int splits, tiles; };     // tiles of each

// Few blocks: split the streamed side, two tiles a split at least.  Blocks that leave most CUs idle in their last round:
// split it if the longest CU then has 15 % less to do, 16 tiles a split at least: forward and backward of 16 heads of
// 48 x 48 tokens of 128 in fp32 3330 -> 2340 us, of 14 heads of 50 x 60 of 32 in fp16 401 -> 337, but of 27 heads of
// 33 x 40 of 64 in bf16, 10 tiles a split, 234 -> 243.
Split split_of(int64_t blocks, int want, int tiles) {
  int s = blocks < want ? (int)(want / blocks) : 1;
  if (s > tiles / 2) s = tiles / 2;
  if (s < 1) s = 1;
  if (s == 1 && blocks <= 768) {
    auto load = [&](int n) { return (double)((blocks * n + 255) / 256) / n; };
    for (int n = 2; n <= 4 && tiles / n >= 16; ++n)
      if (load(n) < 0.85 * load(s)) s = n;
  }
  const int per = count(tiles, s);
  return {count(tiles, per), per};
}

constexpr int64_t kManyReads = (int64_t)1 << 28;

struct Plan {
  int waves, rows, nq_pad, window, window_b, sums, diag_pitch, offsets, dp;
  Split forward, dq, dkv;
  size_t part_o, part_ml, forward_total;
  size_t delta, diag_rows, d_offsets, ranges, part_q, part_k, part_v, backward_total;
};

// Every bucket's block reads the whole map, unless a launch more tells it where its bucket cannot be.  The whole training
// pass of 64 queries of 8 heads with a bucket for every offset, with it / without: 96 x 96 keys (2^30.3 reads) 239 / 529 us,
// 256 x 256 (2^36) 1.8 / 18.3 ms; below 2^28 reads the join is 10 us of 100 - 170 and another launch takes 3.  A map whose
// buckets lie anywhere gains nothing from it, and its join stays at buckets times offsets: 18.7 ms at 256 x 256.
bool many_reads(const PsRelativeAttentionDesc& d, int offsets) { return (int64_t)d.buckets * offsets >= kManyReads; }

// table: its gradient is wanted, whose sums are all that grows with queries times keys
Plan plan(const PsRelativeAttentionDesc& d, bool training, bool table = false) {
  Plan p = {};
  const int nk = d.grid_h * d.grid_w, e = d.dtype == PS_DTYPE_F32 ? 4 : 2;
  p.rows = e == 2 ? 64 : 32;
  p.dp = d.dim <= 32 ? 32 : d.dim <= 64 ? 64 : 128;
  p.offsets = (2 * d.grid_h - 1) * (2 * d.grid_w - 1);
  p.nq_pad = count(d.queries, 64) * 64;
  p.waves = d.queries <= 32 ? 1 : 4;
  auto window = [&](int columns) {
    return count(span_of(columns, d.grid_h, d.grid_w) + span_of(p.rows, d.grid_h, d.grid_w) + 1, 64) * 64;
  };
  p.window = window(p.waves * 32);
  p.window_b = window(128);
  const int64_t bh = (int64_t)d.batch * d.heads;
  const int tiles = count(nk, p.rows), q_tiles = count(d.queries, p.rows);
  // As many blocks as are resident at once, in one round: of one wave, their LDS decides; of four, their registers (one
  // block a CU for rows of 512 bytes, else two are enough to fill the vector pipes).
  const int fill = p.dp * e == 512 ? 256 : 512;
  const int resident = 160 * 1024 / (2 * (2 * p.rows * p.dp * e + 4 * 256 + 4 * p.window));
  const int64_t blocks = bh * count(training ? p.nq_pad : d.queries, p.waves * 32);
  p.forward = p.waves == 1 ? split_of(blocks, 256 * (resident < 1 ? 1 : resident > 8 ? 8 : resident), tiles)
                           : split_of(blocks, fill, tiles);
  p.dq = split_of(bh * count(p.nq_pad, 128), fill, tiles);
  p.dkv = split_of(bh * count(nk, 128), fill, q_tiles);
  p.sums = d.grid_h == 1 ? 1 : 2;
  p.diag_pitch = p.dq.tiles * p.rows + 32;
  const size_t rows = (size_t)bh * d.queries;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
  if (p.forward.splits > 1) {
    p.part_o = take(sizeof(float) * p.forward.splits * rows * d.dim);
    p.part_ml = take(sizeof(float) * p.forward.splits * rows * 2);
  }
  p.forward_total = at + 256;
  at = 0;
  p.delta = take(sizeof(float) * bh * p.nq_pad);
  if (table) {
    p.diag_rows = take(sizeof(float) * bh * (p.nq_pad / 32) * p.dq.splits * p.sums * p.diag_pitch);
    p.d_offsets = take(sizeof(double) * d.heads * p.offsets);
    if (many_reads(d, p.offsets)) p.ranges = take(sizeof(int2) * kJoinLists);
  }
  if (p.dq.splits > 1) p.part_q = take(sizeof(float) * p.dq.splits * rows * d.dim);
  if (p.dkv.splits > 1) {
    p.part_k = take(sizeof(float) * p.dkv.splits * bh * nk * d.dim);
    p.part_v = take(sizeof(float) * p.dkv.splits * bh * nk * d.dim);
  }
  p.backward_total = at + 256;
  return p;
}

Args args_of(const PsRelativeAttentionDesc& d, const Plan& p) {
  Args a = {};
  a.sq = {d.q_strides[0], d.q_strides[1], d.q_strides[2]};
  a.sk = {d.k_strides[0], d.k_strides[1], d.k_strides[2]};
  a.sv = {d.v_strides[0], d.v_strides[1], d.v_strides[2]};
  a.sdo = {d.do_strides[0], d.do_strides[1], d.do_strides[2]};
  a.mask_b = d.mask_stride;
  a.batch = d.batch; a.heads = d.heads; a.nq = d.queries; a.nk = d.grid_h * d.grid_w; a.dim = d.dim;
  a.gw = d.grid_w; a.origin = (d.grid_h - 1) * (2 * d.grid_w - 1) + d.grid_w - 1; a.offsets = p.offsets;
  a.q_start = d.query_start; a.nq_pad = p.nq_pad; a.scale = d.scale * kLog2e;
  a.diag_pitch = p.diag_pitch; a.diag_end = count(a.nk, p.rows) * p.rows + 32;
  return a;
}

template <typename K>
bool allow_lds(K kernel, size_t bytes) {
  return bytes <= 64 * 1024 || hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

template <typename T, int DP, int WAVES>
int run_forward(Args a, const Plan& p, hipStream_t st) {
  a.col_tiles = count(a.stats ? a.nq_pad : a.nq, WAVES * 32);
  a.splits = p.forward.splits;
  a.tiles_per_split = p.forward.tiles;
  a.window = p.window;
  const size_t lds = 2 * (size_t)Lds<T, DP, WAVES>::buffer(p.window);
  auto kernel = attention_forward_kernel<T, DP, WAVES>;
  if (!allow_lds(kernel, lds)) return PS_ERR_LAUNCH;
  kernel<<<dim3((unsigned)(a.col_tiles * a.batch * a.heads), (unsigned)a.splits), WAVES * 64, lds, st>>>(a);
  if (a.splits > 1) {
    a.join_lanes = a.splits >= 8 ? 8 : 1;                // dim <= 128: a row's threads fit a block
    const int in_block = 256 / (a.dim / 4 * a.join_lanes);
    join_splits_kernel<T><<<(unsigned)(((int64_t)a.batch * a.heads * a.nq_pad + in_block - 1) / in_block), 256, 0, st>>>(a);
  }
  return PS_OK;
}

template <typename T, int DP>
int run_backward(Args a, const Plan& p, bool table, hipStream_t st) {
  constexpr int WAVES = 4;
  const size_t lds = 2 * (size_t)Lds<T, DP, WAVES>::buffer(p.window_b);
  a.window = p.window_b;
  const unsigned bh = (unsigned)(a.batch * a.heads);
  a.col_tiles = count(a.nq_pad, WAVES * 32);
  a.splits = p.dq.splits;
  a.tiles_per_split = p.dq.tiles;
  auto dq = [&](auto kernel, size_t bytes) {
    if (!allow_lds(kernel, bytes)) return false;
    kernel<<<dim3(a.col_tiles * bh, (unsigned)a.splits), WAVES * 64, bytes, st>>>(a);
    return true;
  };
  const size_t with = lds + (size_t)WAVES * kDiag * sizeof(float);
  const bool ok = !table ? dq(attention_dq_kernel<T, DP, WAVES, 0>, lds)
                  : p.sums == 1 ? dq(attention_dq_kernel<T, DP, WAVES, 1>, with)
                                : dq(attention_dq_kernel<T, DP, WAVES, 2>, with);
  if (!ok) return PS_ERR_LAUNCH;
  if (a.dk || a.dv) {
    a.col_tiles = count(a.nk, WAVES * 32);
    a.splits = p.dkv.splits;
    a.tiles_per_split = p.dkv.tiles;
    auto kernel = attention_dkv_kernel<T, DP, WAVES>;
    if (!allow_lds(kernel, lds)) return PS_ERR_LAUNCH;
    kernel<<<dim3(a.col_tiles * bh, (unsigned)a.splits), WAVES * 64, lds, st>>>(a);
  }
  Gradients g = {};
  unsigned blocks = 0;
  auto add = [&](int i, void* to, const float* from, int tokens, int splits) {
    const int64_t n = (int64_t)bh * tokens * a.dim;
    if (!to || splits <= 1) return;
    g.g[i] = {from, to, n, splits, count(n, 1024)};
    blocks += g.g[i].blocks;
  };
  add(0, a.dq, a.part_q, a.nq, p.dq.splits);
  add(1, a.dk, a.part_k, a.nk, p.dkv.splits);
  add(2, a.dv, a.part_v, a.nk, p.dkv.splits);
  if (blocks) join_gradients_kernel<T><<<blocks, 256, 0, st>>>(g);
  return PS_OK;
}

template <typename T>
int forward_typed(const PsRelativeAttentionDesc& d, Args a, const Plan& p, const int32_t* map, const void* table,
                  float* bias, hipStream_t st) {
  spread_table_kernel<T><<<dim3((unsigned)count(p.offsets, 256), (unsigned)d.heads), 256, 0, st>>>(
      d.heads, p.offsets, d.buckets, map, table, d.table_f32, bias);
  if (p.waves == 1)
    return p.dp == 32 ? run_forward<T, 32, 1>(a, p, st) : p.dp == 64 ? run_forward<T, 64, 1>(a, p, st)
                                                                     : run_forward<T, 128, 1>(a, p, st);
  return p.dp == 32 ? run_forward<T, 32, 4>(a, p, st) : p.dp == 64 ? run_forward<T, 64, 4>(a, p, st)
                                                                   : run_forward<T, 128, 4>(a, p, st);
}

template <typename T>
int backward_typed(const PsRelativeAttentionDesc& d, Args a, const Plan& p, const int32_t* map, void* d_table, char* ws,
                   hipStream_t st) {
  const int rc = p.dp == 32 ? run_backward<T, 32>(a, p, d_table != nullptr, st)
               : p.dp == 64 ? run_backward<T, 64>(a, p, d_table != nullptr, st)
                            : run_backward<T, 128>(a, p, d_table != nullptr, st);
  if (rc || !d_table) return rc;
  a.splits = p.dq.splits;
  double* d_offsets = (double*)(ws + p.d_offsets);
  join_diagonals_kernel<<<dim3((unsigned)count(p.offsets, 16), (unsigned)d.heads), 256, 0, st>>>(a, p.sums, d_offsets);
  int2* ranges = many_reads(d, p.offsets) ? (int2*)(ws + p.ranges) : nullptr;
  if (ranges) bucket_ranges_kernel<<<(unsigned)count(p.offsets, kJoinList), 256, 0, st>>>(p.offsets, map, ranges);
  const unsigned blocks = (unsigned)(d.buckets < 1 << 20 ? d.buckets : 1 << 20);
  join_offsets_kernel<T><<<dim3(blocks, (unsigned)count(d.heads, kJoinHeads)), 256, 0, st>>>(
      d.heads, p.offsets, d.buckets, map, ranges, d_offsets, d_table, d.table_f32);
  return PS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const PsRelativeAttentionDesc* d) {
  if (!d || d->batch <= 0 || d->heads <= 0 || d->queries <= 0 || d->grid_h <= 0 || d->grid_w <= 0 || d->dim <= 0 ||
      d->buckets <= 0 || d->query_start < 0)
    return PS_ERR_BAD_ARG;
  if (d->dtype < PS_DTYPE_F32 || d->dtype > PS_DTYPE_F16) return PS_ERR_UNSUPPORTED;
  const int64_t nk = (int64_t)d->grid_h * d->grid_w;
  if (nk > 1 << 20 || (d->grid_h > 1 && d->grid_w > 512) || d->dim > 128 || d->heads > 65535 ||
      (int64_t)d->batch * d->heads >= 1 << 24 || d->buckets > 1 << 24)
    return PS_ERR_UNSUPPORTED;
  if (d->query_start + (int64_t)d->queries > nk) return PS_ERR_BAD_ARG;
  // threads of a launch: 64 for 32 tokens, 256 at least for a head, 2^32 at most
  if ((int64_t)d->batch * d->heads * ((d->queries + 63) / 64 * 2) >= 1 << 26 ||
      (int64_t)d->batch * d->heads * ((nk + 31) / 32) >= 1 << 26)
    return PS_ERR_UNSUPPORTED;
  const int chunk = d->dtype == PS_DTYPE_F32 ? 4 : 8;
  if (d->dim % chunk) return PS_ERR_BAD_ARG;
  return PS_OK;
}
// rows start on 16 bytes; 64 of them are within 32-bit offsets of each other
int check_rows(const PsRelativeAttentionDesc& d, const void* p, const int64_t* strides) {
  const int chunk = d.dtype == PS_DTYPE_F32 ? 4 : 8;
  if (!p || !aligned16(p)) return PS_ERR_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (strides[i] % chunk || strides[i] < 0) return PS_ERR_BAD_ARG;
  return strides[2] < (int64_t)1 << 24 ? PS_OK : PS_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" {

size_t ps_relative_attention_workspace_bytes(const PsRelativeAttentionDesc* d, int32_t pass) {
  if (check(d)) return 0;
  if (pass != PS_FORWARD) return plan(*d, true, pass != PS_BACKWARD_NO_TABLE).backward_total;
  const size_t a = plan(*d, false).forward_total, b = plan(*d, true).forward_total;
  return a > b ? a : b;
}

int ps_relative_attention_forward(const PsRelativeAttentionDesc* d, const void* q, const void* k, const void* v,
                                  const uint8_t* key_mask, const int32_t* bucket_map, const void* table, void* out,
                                  float* out_f32, float* stats, float* bias, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check(d)) return rc;
  if (int rc = check_rows(*d, q, d->q_strides)) return rc;
  if (int rc = check_rows(*d, k, d->k_strides)) return rc;
  if (int rc = check_rows(*d, v, d->v_strides)) return rc;
  if (!bucket_map || !table || !out || !aligned16(out) || !bias || !workspace || !aligned16(workspace) ||
      (out_f32 && !aligned16(out_f32)))
    return PS_ERR_BAD_ARG;
  if (workspace_bytes < ps_relative_attention_workspace_bytes(d, PS_FORWARD)) return PS_ERR_WORKSPACE;
  const Plan p = plan(*d, stats != nullptr);
  Args a = args_of(*d, p);
  a.q = q; a.k = k; a.v = v; a.mask = key_mask; a.bias = bias;
  a.out = out; a.o32 = out_f32; a.stats = stats;
  a.part_o = (float*)((char*)workspace + p.part_o);
  a.part_ml = (float*)((char*)workspace + p.part_ml);
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d->dtype) {
    case PS_DTYPE_F32: rc = forward_typed<float>(*d, a, p, bucket_map, table, bias, st); break;
    case PS_DTYPE_BF16: rc = forward_typed<bf16>(*d, a, p, bucket_map, table, bias, st); break;
    default: rc = forward_typed<f16>(*d, a, p, bucket_map, table, bias, st); break;
  }
  return rc ? rc : hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

int ps_relative_attention_backward(const PsRelativeAttentionDesc* d, const void* q, const void* k, const void* v,
                                   const uint8_t* key_mask, const int32_t* bucket_map, const float* bias,
                                   const float* out_f32, const float* stats, const void* d_out, void* dq, void* dk, void* dv,
                                   void* d_table, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check(d)) return rc;
  if (int rc = check_rows(*d, q, d->q_strides)) return rc;
  if (int rc = check_rows(*d, k, d->k_strides)) return rc;
  if (int rc = check_rows(*d, v, d->v_strides)) return rc;
  if (int rc = check_rows(*d, d_out, d->do_strides)) return rc;
  if (!bucket_map || !bias || !out_f32 || !stats || !workspace || !aligned16(workspace)) return PS_ERR_BAD_ARG;
  if (!aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return PS_ERR_BAD_ARG;
  const Plan p = plan(*d, true, d_table != nullptr);
  if (workspace_bytes < p.backward_total) return PS_ERR_WORKSPACE;
  Args a = args_of(*d, p);
  char* ws = (char*)workspace;
  a.q = q; a.k = k; a.v = v; a.mask = key_mask; a.bias = bias; a.dout = d_out;
  a.o_kept = out_f32; a.stats = const_cast<float*>(stats); a.delta = (float*)(ws + p.delta);
  a.diag_rows = (float*)(ws + p.diag_rows);
  a.part_q = (float*)(ws + p.part_q); a.part_k = (float*)(ws + p.part_k); a.part_v = (float*)(ws + p.part_v);
  a.dq = dq; a.dk = dk; a.dv = dv;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d->dtype) {
    case PS_DTYPE_F32: rc = backward_typed<float>(*d, a, p, bucket_map, d_table, ws, st); break;
    case PS_DTYPE_BF16: rc = backward_typed<bf16>(*d, a, p, bucket_map, d_table, ws, st); break;
    default: rc = backward_typed<f16>(*d, a, p, bucket_map, d_table, ws, st); break;
  }
  return rc ? rc : hipGetLastError() == hipSuccess ? PS_OK : PS_ERR_LAUNCH;
}

}  // extern "C"
