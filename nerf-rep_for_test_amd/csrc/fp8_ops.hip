// 8-bit block-scaled products: e4m3 values with one power-of-two scale (E8M0)
// for 1 x 128 of the activations and for 128 x 128 of the weights,
//   y[m][n] = sum_k x[m][k] w[n][k]  (+ bias[n], ReLU),
// dense, or with rows sorted by expert and a weight matrix for each expert.
//
// A block's scale is the smallest 2^e that brings its largest magnitude to 448
// (e4m3's largest value) or less. Scaling by a power of two is exact, so a
// value is rounded once, to e4m3, whatever computes it, and the matrix
// instruction applies the scales itself (v_mfma_scale_f32_16x16x128: one
// instruction is one block). Sums are FP32 in the matrix accumulators; the
// result is rounded once, to the output's type. The 8-bit instruction adds 8
// neighbouring products at the scale of the largest, with 13 bits below it: off
// by 1.3e-5 of a product's norm (measured, normal values), and by 7 2^-13 of the
// largest product at most, where it outweighs its seven neighbours: below BF16's
// half step of 2^-8, up to 1.75 of FP16's 2^-11. Kept for 16-bit results, which it
// gives at twice the rate. An FP32 result takes the FP16 instruction instead
// (Fp8Wide: exact products; 8192 x 8192 x 8192 in 1260 us against 520, 262144 rows
// through 256 x 256 in 108 against 60, few rows in the same time).
#include "tile_product.h"

namespace nerfhip {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

// The biased exponent (E8M0) of a block whose largest |x| has these bits; 255 (NaN:
// the block's products are NaN) where a value is not finite.
__device__ __forceinline__ int block_scale(unsigned amax) {
  if (amax >= 0x7f800000u) return 255;
  const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (e < -127 ? -127 : e) + 127;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ int pack4(float a, float b, float c, float d) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

// The largest value of 16 neighbouring lanes, by DPP.
__device__ __forceinline__ unsigned max16(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));    // lane ^ 1
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));    // lane ^ 2
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));   // the other four of 8
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
}

// The largest value of the 4 lanes that are 16 apart.
__device__ __forceinline__ unsigned max4(unsigned v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// N values of a row from column k on; zeros from K on. VEC: 16-byte loads (whole
// pieces lie inside or outside of the row).
template <class T, int N, bool VEC>
__device__ __forceinline__ void load_row(float (&f)[N], const T* row, int64_t k, int64_t K) {
  constexpr int W = 16 / sizeof(T);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
      Vec<T, W> v = {};
      if (k + i < K) v = *(const Vec<T, W>*)(row + k + i);
#pragma unroll
      for (int j = 0; j < W; ++j) f[i + j] = (float)v.v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = k + i < K ? (float)row[k + i] : 0.0f;
  }
}

// 8 values of a row from column k on as they are; zeros from K on.
template <class T, bool VEC>
__device__ __forceinline__ void load_raw(T (&v)[8], const T* row, int64_t k, int64_t K) {
  constexpr int W = 16 / sizeof(T);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      Vec<T, W> q = {};
      if (k + i < K) q = *(const Vec<T, W>*)(row + k + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = q.v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : (T)0.0f;
  }
}

// A row of the activations: row i itself, or where `order` is given the row that
// slot order[i] (of `div` slots for each row) came from; -1: no row of x (zeros).
__device__ __forceinline__ int64_t source_row(const int* order, int div, int64_t rows, int64_t i) {
  if (!order) return i;
  const int s = order[i];
  return s < 0 || s / div >= rows ? -1 : s / div;
}

// Rows of x (row m: source_row, zeros from `live` on) to e4m3 q [M][KB * 128] and packed scales s [ceil(KB / 4)][M] (the bytes of 4
// neighbouring blocks of one row in one word). 16 lanes take one block of 128: 8 values
// each, the largest magnitude by 4 steps inside the 16 lanes. Bound by HBM: every byte
// is read and written once, 8192 x 8192 in 16 bits (201 MB) in 41 us, 4.9 TB/s.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t ldx, const int* __restrict__ order,
                                                       int div, int64_t rows, int64_t live, int64_t M, int64_t K, int KB,
                                                       unsigned char* __restrict__ q,
                                                       unsigned char* __restrict__ s) {
  const int l = threadIdx.x & 15;
  const int64_t blocks = M * KB;
  for (int64_t b = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); b < blocks; b += (int64_t)gridDim.x * 16) {
    const int64_t m = b / KB;
    const int kb = (int)(b - m * KB);
    const int64_t src = m < live ? source_row(order, div, rows, m) : -1;
    float f[8] = {};
    if (src >= 0) load_row<T, 8, VEC>(f, x + src * ldx, (int64_t)kb * 128 + l * 8, K);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(f[i]));
    top = max16(top);
    const int sc = block_scale(top), e = 127 - sc;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __builtin_ldexpf(f[i], e);
    int2 v;
    v.x = pack4(f[0], f[1], f[2], f[3]);
    v.y = pack4(f[4], f[5], f[6], f[7]);
    *(int2*)(q + (m * KB + kb) * 128 + l * 8) = v;
    if (l == 0) s[((kb >> 2) * M + m) * 4 + (kb & 3)] = (unsigned char)sc;
  }
}

// Blocks of 128 x 128 of weights (stack [E][N][K], rows ldw apart, matrices sw apart) to
// e4m3 q [E][N][KB * 128] and scales [E][NB][KB]. One workgroup for each block.
template <class T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ w, int64_t sw, int64_t ldw,
                                                              int64_t N, int64_t K, int NB, int KB, int64_t first,
                                                              unsigned char* __restrict__ q,
                                                              unsigned char* __restrict__ s) {
  const int64_t id = first + blockIdx.x;
  const int kb = (int)(id % KB);
  const int nb = (int)(id / KB % NB);
  const int64_t e = id / KB / NB;
  const int t = threadIdx.x, l = t & 15, r0 = t >> 4;
  const T* base = w + e * sw;
  float f[8][8];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = (int64_t)nb * 128 + i * 16 + r0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t k = (int64_t)kb * 128 + l * 8 + j;
      f[i][j] = n < N && k < K ? (float)base[n * ldw + k] : 0.0f;
      top = max(top, abs_bits(f[i][j]));
    }
  }
  for (int d = 1; d < 64; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
  __shared__ unsigned part[4];
  if ((t & 63) == 0) part[t >> 6] = top;
  __syncthreads();
  top = max(max(part[0], part[1]), max(part[2], part[3]));
  const int sc = block_scale(top), ex = 127 - sc;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = (int64_t)nb * 128 + i * 16 + r0;
    if (n < N) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = __builtin_ldexpf(f[i][j], ex);
      int2 v;
      v.x = pack4(f[i][0], f[i][1], f[i][2], f[i][3]);
      v.y = pack4(f[i][4], f[i][5], f[i][6], f[i][7]);
      *(int2*)(q + ((e * N + n) * KB + kb) * 128 + l * 8) = v;
    }
  }
  if (t == 0) s[id] = (unsigned char)sc;
}

struct LinearArgs {
  const void* x;              // the activations' rows (skinny form)
  int64_t ldx, x_rows;
  const int* order;           // or null
  int div;
  const unsigned char* q;     // quantised rows [q_rows][KB * 128] (tiled form)
  const unsigned* s;          // [ceil(KB / 4)][q_rows]
  int64_t q_rows;
  int gather;                 // q holds x's rows and one of zeros; else the M rows as they are taken
  const unsigned char* wq;    // [E][N][KB * 128]
  const unsigned char* ws;    // [E][NB][KB]
  const int* offsets;         // [E + 1], or null (dense: E = 1)
  int E;
  const float* bias;          // [E][N], or null
  int relu;
  int64_t M, N, K;
  int KB, NB;
  void* out;                  // [M][N], rows ldo apart
  int64_t ldo;
};

// Rows [lo, hi) of expert e; e == E: the rows behind the last expert's (no weights: zeros).
__device__ __forceinline__ void expert_rows(const LinearArgs& a, int e, int64_t& lo, int64_t& hi) {
  if (!a.offsets) {
    lo = 0;
    hi = a.M;
    return;
  }
  lo = a.offsets[e];
  hi = e < a.E ? a.offsets[e + 1] : a.M;
  lo = lo < 0 ? 0 : (lo > a.M ? a.M : lo);
  hi = hi < lo ? lo : (hi > a.M ? a.M : hi);
}

template <class T, int N>
__device__ __forceinline__ void store_run(T* at, const float (&v)[N], int64_t room, bool vec) {
  constexpr int W = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  if (vec && room >= N) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
      Vec<T, W> o;
#pragma unroll
      for (int j = 0; j < W; ++j) o.v[j] = (T)v[i + j];
      *(Vec<T, W>*)(at + i) = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < room) at[i] = (T)v[i];
  }
}

// max(v, 0) that keeps NaN
__device__ __forceinline__ float relu_of(float v) { return v < 0.0f ? 0.0f : v; }

// ---------------------------------------------------------------- tiled form

// Rows rounded to 8 bits by quantize_kernel, then tiles of 64 x 64, 128 x 128 or 256 x 256
// (tile_product.h). Large products are bound by the matrix cores and the power they may draw
// (8192 x 8192 x 8192: a call 507 to 512 us, 42 of them the rounding of x, so 2.3 PFLOP/s; 521 to 565 us for the
// product under a kernel trace; the library's own 8-bit product reaches 2.5 to 2.7), those of experts by their
// short rows: 32768 of 2048 in 242 to 257 us, 1.1 PFLOP/s, a third of it starts and ends of tiles.

// Workgroup -> (expert, row tile): experts' row tiles one after another. Every wave sums the
// experts' tile counts 64 at a time until the tile is met.
template <int BM>
__device__ __forceinline__ bool find_tile(const LinearArgs& a, int tile, int& e, int64_t& m0, int64_t& hi) {
  if (!a.offsets) {
    e = 0;
    m0 = (int64_t)tile * BM;
    hi = a.M;
    return m0 < a.M;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base <= a.E; base += 64) {
    const int mine = base + lane;
    int64_t l = 0, h = 0;
    if (mine <= a.E) expert_rows(a, mine, l, h);
    const int n = (int)cdiv(h - l, BM);
    int sum = n;
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned long long met = __ballot(before + sum > tile);
    if (met) {
      const int at = __builtin_ctzll(met);
      e = base + at;
      const int first = before + __shfl(sum - n, at);
      m0 = __shfl((int)l, at) + (int64_t)(tile - first) * BM;   // (rows are below 2^31)
      hi = __shfl((int)h, at);
      return true;
    }
    before += __shfl(sum, 63);
  }
  return false;
}

// This lane's columns' bias (zeros without) in a tile from column n0 on.
template <class S>
__device__ __forceinline__ void load_bias(const LinearArgs& a, const TileProduct<S>& p, int64_t e, int64_t n0,
                                          float (&bias)[4 * S::TN]) {
#pragma unroll
  for (int c = 0; c < 4 * S::TN; ++c) {
    const int64_t n = n0 + p.n(c / 8) + c % 8;
    bias[c] = a.bias && n < a.N ? a.bias[e * a.N + n] : 0.0f;
  }
}

// The tile's results: bias, ReLU, one rounding, rows below hi.
template <class S, class T>
__device__ __forceinline__ void store_tile(const LinearArgs& a, const TileProduct<S>& p, const float (&bias)[4 * S::TN],
                                           int64_t m0, int64_t hi, int64_t n0) {
  const bool vec = ((uintptr_t)a.out | (uintptr_t)(a.ldo * sizeof(T))) % 16 == 0;
  auto value = [&](int i, int h, float (&v)[8]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      v[c] = p.acc[i][2 * h + c / 4][c % 4] + bias[8 * h + c];
      if (a.relu) v[c] = relu_of(v[c]);
    }
  };
  // whole rows of the tile: no question but the row's (a branch around every store cost 76 us against 62 over
  // 2^18 rows through 256 x 256)
  if (vec && n0 + S::BN <= a.N) {
#pragma unroll
    for (int i = 0; i < S::TM; ++i) {
      const int64_t m = m0 + p.m(i);
      T* row = (T*)a.out + m * a.ldo + n0;
      if (m < hi) {
#pragma unroll
        for (int h = 0; h < S::TN / 2; ++h) {
          float v[8];
          value(i, h, v);
          store_run(row + p.n(h), v, 8, true);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < S::TM; ++i) {
    const int64_t m = m0 + p.m(i);
#pragma unroll
    for (int h = 0; h < S::TN / 2; ++h) {
      const int64_t n = n0 + p.n(h);
      if (m < hi && n < a.N) {
        float v[8];
        value(i, h, v);
        store_run((T*)a.out + m * a.ldo + n, v, a.N - n, vec);
      }
    }
  }
}

constexpr int kScaleRun = 512;   // blocks of K whose weights' scales are in LDS at a time

// A stage with its rows' scale words, two of them, and the weights' scale bytes.
template <class S>
struct ProductLds {
  static constexpr int kAll = S::kStage + (S::BM > S::NT ? S::BM : S::NT) * 4;
  static constexpr size_t kBytes = S::NS * kAll + (S::BN / 128 > 0 ? S::BN / 128 : 1) * kScaleRun;
};

template <class S, class T>
__global__ __launch_bounds__(S::NT) void product_kernel(const LinearArgs a, int mtiles, int ntiles) {
  using L = ProductLds<S>;
  static_assert(128 % (16 * S::TN) == 0 && (S::BN % 128 == 0 || 128 % S::BN == 0), "one scale for a wave's columns");
  constexpr int kBlocksN = S::BN > 128 ? S::BN / 128 : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int64_t id = xcd_tile(blockIdx.x, gridDim.x);
  int e, mt, nt;
  band_tile(id, mtiles, ntiles, 8, mt, nt);
  int64_t m0, hi;
  if (!find_tile<S::BM>(a, mt, e, m0, hi)) return;
  const int64_t n0 = (int64_t)nt * S::BN;
  TileProduct<S> p;
  const bool none = e == a.E && a.offsets;
  const int64_t ld = (int64_t)a.KB * 128;
  const int eb = none ? 0 : e;
  // a tile's rows among the quantised ones: neighbours, or x's rows where `order` says (the row of zeros
  // behind them for none)
  const int64_t first = a.gather ? 0 : m0;
  const auto row = [&](int r) {
    const int64_t m = m0 + r < hi ? m0 + r : hi - 1;
    if (!a.gather) return (unsigned)(m - m0);
    const int64_t src = source_row(a.order, a.div, a.x_rows, m);
    return (unsigned)(src < 0 ? a.x_rows : src);
  };
  p.init_rows((const char*)a.q + first * ld, (unsigned)ld, row, (const char*)a.wq + (int64_t)eb * a.N * ld, ld, n0, a.N);
  if (!none) {
    // Scales reach the loop through LDS only, so nothing in it waits for a load into registers:
    // the rows' words (4 blocks) with each stage, the weights' bytes kScaleRun blocks at a time.
    const int t = threadIdx.x, w = t >> 6;
    const unsigned char* ws = a.ws + (int64_t)eb * a.NB * a.KB;
    const int64_t nb0 = n0 / 128;
    const unsigned* s0 = (const unsigned*)uniform((int64_t)(a.s + first));
    char* bytes = lds + S::NS * L::kAll;
    const unsigned char* mine = (const unsigned char*)bytes + (S::BN > 128 ? (w % S::WC) * 16 * S::TN / 128 : 0) * kScaleRun;
    constexpr int NS = S::NS, kScaleLoads = (S::BM + S::NT - 1) / S::NT;
    constexpr int kLoads = S::LA + S::LB + kScaleLoads;   // of one wave for one stage
    unsigned srow[kScaleLoads];
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) srow[i] = row(i * S::NT + t) * 4u;
    struct Plan {
      typename TileProduct<S>::Loads l;
      i32x4 rs;
      unsigned at;
    };
    auto plan = [&](int k) {
      Plan x;
      char* stage = lds + (k % NS) * L::kAll;
      x.l = p.loads(stage, k, k < a.KB);
      x.rs = make_rsrc(s0 + (int64_t)(k >> 2) * a.q_rows, k < a.KB);
      x.at = lds_offset(stage) + S::kStage + (unsigned)__builtin_amdgcn_readfirstlane(w * 64) * 4u;
      return x;
    };
    auto load = [&](const Plan& x, int q) {
      p.load_one(x.l, q);
      if (q >= S::LA + S::LB) {   // (a wave behind the last row loads into the room after it)
        const int i = q - S::LA - S::LB;
        load_lds4(x.rs, srow[i], x.at + i * S::NT * 4u);
      }
    };
    auto chunk = [&](int k, auto part) {
      const char* stage = lds + (k % NS) * L::kAll;
      int word[S::TM];   // (read first: they are needed first)
#pragma unroll
      for (int i = 0; i < S::TM; ++i) word[i] = ((const int*)(stage + S::kStage))[p.m(i)];
      const int sn = mine[k % kScaleRun];
      p.chunk(stage, stage + S::BM * 128, word, 8 * (k & 3), sn, kLoads, part);
    };
    auto scales = [&](int k) {   // the weights' scales of the next run of blocks
      if (k % kScaleRun != 0 || k >= a.KB) return;
      if (k) __syncthreads();
      for (int q = t; q < kBlocksN * kScaleRun; q += S::NT) {
        const int64_t nb = nb0 + q / kScaleRun;
        const int kb = k + q % kScaleRun;
        if (kb < a.KB && nb < a.NB) bytes[q] = (char)ws[nb * a.KB + kb];
      }
    };
    tile_steps<S, kLoads>(a.KB, plan, load, chunk, scales, [] {});
  }
  float bias[4 * S::TN] = {};
  if (!none) load_bias<S>(a, p, eb, n0, bias);
  store_tile<S, T>(a, p, bias, m0, hi, n0);
}

// ---------------------------------------------------------------- resident form

// Many rows through one small matrix (N <= 256, K <= 256: the width of the framework's networks): bound
// by reading x and writing y. One workgroup on each CU holds the 8-bit weights in LDS and walks over
// tiles of 128 rows: the next tile's rows are on their way into registers while this one's products run
// and its results are stored; a tile is rounded to 8 bits straight into LDS (two buffers, one barrier
// for each tile), so the activations' 8-bit form never goes to memory. 2^18 rows of 256 in 16 bits
// (268 MB) in 58 us, 4.6 TB/s; rounded and multiplied in two launches: 109 us.
constexpr int kResident = 256;

template <class S>
constexpr size_t resident_lds(int KB) {
  return (size_t)KB * (S::BN * 128 + 2 * S::BM * 129) + 4 * KB;
}

template <class S, class X, class T, int KB, bool VEC>
__global__ __launch_bounds__(S::NT) void resident_kernel(const LinearArgs a, int mtiles) {
  static_assert(S::BN == kResident, "all columns in one tile");
  constexpr int IT = S::BM * KB * 16 / S::NT;   // blocks of 128 for each 16 lanes
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int t = threadIdx.x, w = t >> 6, l = t & 15;
  const int64_t ld = KB * 128;
  const char* W = (const char*)a.wq;
  char* rows = lds + KB * S::BN * 128;                                      // [2][KB][BM][128]
  unsigned char* sx = (unsigned char*)rows + 2 * KB * S::BM * 128;          // [2][KB][BM]
  TileProduct<S> p;
  p.init(W, ld, 0, 1, W, ld, 0, a.N);
  for (int k = 0; k < KB; ++k) p.load_n(lds + k * S::BN * 128, k);
  int sn[KB];
  float bias[4 * S::TN];
  const int nb = (w % S::WC) * 16 * S::TN / 128;
#pragma unroll
  for (int k = 0; k < KB; ++k) sn[k] = a.ws[(nb < a.NB ? nb : a.NB - 1) * KB + k];
  load_bias<S>(a, p, 0, 0, bias);
  X x[IT][8];
  auto fetch = [&](int64_t tile) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int b = i * (S::NT / 16) + (t >> 4), r = b % S::BM, kb = b / S::BM;
      const int64_t m = tile * S::BM + r;
      load_raw<X, VEC>(x[i], (const X*)a.x + (m < a.M ? m : a.M - 1) * a.ldx, kb * 128 + l * 8, a.K);
    }
  };
  int64_t tile = blockIdx.x;
  fetch(tile);
  for (int at = 0; tile < mtiles; tile += gridDim.x, at ^= 1) {
    char* mine = rows + at * KB * S::BM * 128;
    unsigned char* smine = sx + at * KB * S::BM;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int b = i * (S::NT / 16) + (t >> 4), r = b % S::BM, kb = b / S::BM;
      float f[8];
      unsigned top = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        f[c] = (float)x[i][c];
        top = max(top, abs_bits(f[c]));
      }
      top = max16(top);
      const int sc = block_scale(top), ex = 127 - sc;
#pragma unroll
      for (int c = 0; c < 8; ++c) f[c] = __builtin_ldexpf(f[c], ex);
      int2 v;
      v.x = pack4(f[0], f[1], f[2], f[3]);
      v.y = pack4(f[4], f[5], f[6], f[7]);
      *(int2*)(mine + kb * S::BM * 128 + r * 128 + (((l >> 1) ^ swz<S::R>(r)) << 4) + (l & 1) * 8) = v;
      if (l == 0) smine[kb * S::BM + r] = (unsigned char)sc;
    }
    const int64_t next = tile + gridDim.x;
    if (at == 0 && tile == blockIdx.x) stage_ready();   // (the weights, too)
    else __syncthreads();
    fetch(next < mtiles ? next : tile);
    p.clear();
#pragma unroll 1   // (the fragments of one block at a time)
    for (int k = 0; k < KB; ++k) {
      int word[S::TM];
#pragma unroll
      for (int i = 0; i < S::TM; ++i) word[i] = smine[k * S::BM + p.m(i)];
      p.chunk(mine + k * S::BM * 128, lds + k * S::BN * 128, word, 0, KB == 1 || k == 0 ? sn[0] : sn[KB - 1], 0,
              [](int) {});
    }
    store_tile<S, T>(a, p, bias, tile * S::BM, a.M, 0);
  }
}

// ---------------------------------------------------------------- skinny form

// Tile `tile` of the tiles of 16 rows behind each expert's first: a lane counts those of a run of experts.
__device__ __forceinline__ bool find_further(const LinearArgs& a, int tile, int& e, int64_t& m0, int64_t& hi) {
  const int lane = threadIdx.x & 63, n = a.offsets ? a.E + 1 : 1, per = (n + 63) / 64;
  const auto tiles = [&](int at) {
    int64_t lo = 0, end = 0;
    if (at < n) expert_rows(a, at, lo, end);
    return end > lo ? (int)((end - lo - 1) / 16) : 0;
  };
  int mine = 0;
#pragma unroll 4
  for (int i = 0; i < per; ++i) mine += tiles(lane * per + i);
  int sum = mine;
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  const unsigned long long met = __ballot(sum > tile);
  if (!met) return false;
  const int at = __builtin_ctzll(met);
  int left = tile - __builtin_amdgcn_readlane(sum - mine, at);
  e = at * per;
  for (int c; e + 1 < n && (c = tiles(e)) <= left; ++e) left -= c;   // (that lane counted more than `left`)
  e = __builtin_amdgcn_readfirstlane(e);
  expert_rows(a, e, m0, hi);
  m0 += 16 * (int64_t)(__builtin_amdgcn_readfirstlane(left) + 1);
  return true;
}

// Few rows for each weight matrix: bound by the weights' bytes. A workgroup of 8 waves
// takes 16 rows of x (blockIdx.y: the first 16 of each expert, then the further 16s of
// whatever experts have them) and 16 TN weight rows; the waves share the blocks of K
// between them, U at a time (all of their loads in flight), read the weights straight into
// the matrix operands (16 rows x 128 B lines, no LDS) and quantise the activations in
// registers (a row's block lies in 4 lanes), so one launch reads each weight once for every
// 16 rows. The 8 partial sums are added in wave order.
// Rows that a gate spreads unevenly (64 experts of 1024 x 2048, 1024 rows; 256 of 512 x 1024, 4096): all on one
// expert 30 and 43 us (one workgroup walking them all: 415 and 990), at random 40 and 52 (48 and 47), evenly 30
// and 41 (28 and 35: the further 16s' workgroups start and find nothing).
// 4096 x 4096 for one row in 7.1 us (2.4 TB/s: its start and end are half of that), 64 experts of
// 1024 x 2048 with 96 rows in 21 us (5 TB/s).
template <class T, class O, int TN, bool VEC>
__global__ __launch_bounds__(512) void skinny_kernel(const LinearArgs a) {
  constexpr int W = 8, U = TN == 4 ? 1 : 2;
  __shared__ float part[W][TN][16][17];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, g = lane >> 4, r = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * TN;
  const int firsts = a.offsets ? a.E + 1 : 1;
  int e = blockIdx.y;
  int64_t m0, hi;
  if (e < firsts) {
    expert_rows(a, e, m0, hi);
    if (m0 >= hi) return;
  } else if (!find_further(a, e - firsts, e, m0, hi)) {
    return;
  }
  const bool none = a.offsets && e == a.E;
  const int eb = none ? 0 : e;
  const unsigned char* wrow[TN];
  const unsigned char* ws = a.ws + ((int64_t)eb * a.NB + n0 / 128) * a.KB;   // (16 TN divides 128)
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int64_t n = n0 + 16 * j + r;
    wrow[j] = a.wq + ((int64_t)eb * a.N + (n < a.N ? n : a.N - 1)) * a.KB * 128 + g * 16;
  }
  f32x4 acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = f32x4(0.0f);
  const int64_t src = source_row(a.order, a.div, a.x_rows, m0 + r < hi ? m0 + r : hi - 1);
  const T* xrow = src < 0 ? nullptr : (const T*)a.x + src * a.ldx;
  for (int k0 = w; k0 < a.KB && !none; k0 += W * U) {
    i32x4 wf[U][TN][2];
    int sn[U];
    T x[U][2][16];
#pragma unroll
    for (int u = 0; u < U; ++u) {   // (blocks behind the last one: the last one again, not used)
      const int64_t k = k0 + u * W < a.KB ? k0 + u * W : a.KB - 1;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        wf[u][j][0] = *(const i32x4*)(wrow[j] + k * 128);
        wf[u][j][1] = *(const i32x4*)(wrow[j] + k * 128 + 64);
      }
      sn[u] = ws[k];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 16; c += 8) {
          T v[8] = {};
          if (xrow) load_raw<T, VEC>(v, xrow, k * 128 + h * 64 + g * 16 + c, a.K);
#pragma unroll
          for (int q = 0; q < 8; ++q) x[u][h][c + q] = v[q];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[2][16];
      unsigned top = 0;
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        f[c >> 4][c & 15] = (float)x[u][c >> 4][c & 15];
        top = max(top, abs_bits(f[c >> 4][c & 15]));
      }
      top = max4(top);
      const int sc = block_scale(top), ex = 127 - sc;
      i32x8 xf;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float* v = &f[c >> 2][(c & 3) * 4];
        xf[c] = pack4(__builtin_ldexpf(v[0], ex), __builtin_ldexpf(v[1], ex), __builtin_ldexpf(v[2], ex),
                      __builtin_ldexpf(v[3], ex));
      }
      if (k0 + u * W < a.KB) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const i32x8 wj = __builtin_shufflevector(wf[u][j][0], wf[u][j][1], 0, 1, 2, 3, 4, 5, 6, 7);
          if constexpr (sizeof(O) == 4)
            acc[j] = wide_block(wj, xf, sn[u], sc, acc[j]);
          else
            acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wj, xf, acc[j], 0, 0, 0, sn[u], 0, sc);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) part[w][j][r][g * 4 + c] = acc[j][c];   // [row m][column n]
  __syncthreads();
  for (int o = t; o < TN * 256; o += 512) {
    const int j = (o >> 4) % TN, m = (o >> 4) / TN, c = o & 15;
    float v = part[0][j][m][c];
#pragma unroll
    for (int u = 1; u < W; ++u) v += part[u][j][m][c];
    const int64_t row = m0 + m, n = n0 + 16 * j + c;
    if (row < hi && n < a.N) {
      if (a.bias && !none) v += a.bias[(int64_t)eb * a.N + n];
      if (a.relu) v = relu_of(v);
      ((O*)a.out)[row * a.ldo + n] = (O)v;
    }
  }
}

// ---------------------------------------------------------------- launches

bool aligned16(const void* p, int64_t ld, int size) {
  return (uintptr_t)p % 16 == 0 && (uint64_t)ld * size % 16 == 0;
}

template <class T>
void launch_quantize(const LinearArgs& a, unsigned char* q, unsigned char* s, hipStream_t st) {
  const int64_t groups = cdiv(a.q_rows * a.KB, 16);
  const unsigned grid = (unsigned)(groups < 65536 ? groups : 65536);
  const bool vec = aligned16(a.x, a.ldx, sizeof(T)) && a.K % (16 / sizeof(T)) == 0;
  auto* kern = vec ? quantize_kernel<T, true> : quantize_kernel<T, false>;
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, st, (const T*)a.x, a.ldx, a.gather ? nullptr : a.order, a.div, a.x_rows,
                     a.gather ? a.x_rows : a.q_rows, a.q_rows, a.K, a.KB, q, s);
}

template <class S, class T>
void launch_product(const LinearArgs& a, hipStream_t st) {
  const int64_t mt = a.offsets ? a.M / S::BM + a.E + 1 : cdiv(a.M, S::BM), nt = cdiv(a.N, S::BN);
  hipLaunchKernelGGL((product_kernel<S, T>), dim3((unsigned)(mt * nt)), dim3(S::NT), ProductLds<S>::kBytes, st, a,
                     (int)mt, (int)nt);
}

template <class S, class X, class T, int KB>
void launch_resident(const LinearArgs& a, hipStream_t st) {
  const int64_t mt = cdiv(a.M, S::BM), cus = stream_cu_count(st);
  const bool vec = aligned16(a.x, a.ldx, sizeof(X)) && a.K % (16 / sizeof(X)) == 0;
  auto* kern = vec ? resident_kernel<S, X, T, KB, true> : resident_kernel<S, X, T, KB, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(mt < cus ? mt : cus)), dim3(S::NT), resident_lds<S>(KB), st, a, (int)mt);
}

template <class X, class T>
void launch_resident_k(const LinearArgs& a, hipStream_t st) {
  // (the wide products' registers: half the rows)
  using S = typename std::conditional<sizeof(T) == 4, TileShape<Fp8Wide, 2, 4, 2, 4>, TileShape<Fp8, 4, 4, 2, 4>>::type;
  if (a.KB == 1) launch_resident<S, X, T, 1>(a, st);
  else launch_resident<S, X, T, 2>(a, st);
}

template <class X>
void launch_resident_out(const LinearArgs& a, int out_type, hipStream_t st) {
  if (out_type == NERF_F32) launch_resident_k<X, float>(a, st);
  else if (out_type == NERF_BF16) launch_resident_k<X, bf16>(a, st);
  else launch_resident_k<X, f16>(a, st);
}

template <class T, class O, int TN>
void launch_skinny(const LinearArgs& a, hipStream_t st) {
  const bool vec = aligned16(a.x, a.ldx, sizeof(T)) && a.K % (16 / sizeof(T)) == 0;
  // (further 16s: a matrix with r rows has (r - 1) / 16 of them, all together (M - 1) / 16 at most)
  const int64_t tiles = (a.offsets ? a.E + 1 : 1) + (a.M - 1) / 16;
  auto* kern = vec ? skinny_kernel<T, O, TN, true> : skinny_kernel<T, O, TN, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)cdiv(a.N, 16 * TN), (unsigned)tiles), dim3(512), 0, st, a);
}

template <class T, class O>
void launch_skinny_n(const LinearArgs& a, hipStream_t st) {
  // 16-row tiles with work. Wider workgroups round the activations once for more of the weights and
  // need fewer starts (64 experts of 1024 x 2048, 96 rows: 24 us with 4 tiles, 34 with 2, 34 with 1; one
  // row, 16384 x 4096: 14, 19, 21), where there are enough of them (6 experts with a row each: 12, 9, 10;
  // one row, 8192 x 8192: 20, 18, 19; 16 rows, 4096 x 4096: -, 12, 10).
  const int64_t tiles = cdiv(a.N, 16) * (a.offsets ? (a.M < a.E ? a.M : a.E) : 1);
  if (tiles >= 1024) launch_skinny<T, O, 4>(a, st);
  else if (tiles > 256) launch_skinny<T, O, 2>(a, st);
  else launch_skinny<T, O, 1>(a, st);
}

template <class T>
void launch_skinny_out(const LinearArgs& a, int out_type, hipStream_t st) {
  if (out_type == NERF_F32) launch_skinny_n<T, float>(a, st);
  else if (out_type == NERF_BF16) launch_skinny_n<T, bf16>(a, st);
  else launch_skinny_n<T, f16>(a, st);
}

// Few rows for each weight matrix: the skinny form, which takes 16 rows (one matrix operand) at a time and
// reads the weights again for the next 16 (4096 x 4096, 16-bit rows: 32 of them 17 us, tiled 21; 48: 23
// and 21; 16 experts of 1024 x 2048 with 256 rows: 14 and 18 us, with 512: 23 and 19). However the rows are spread:
// the host does not know it.
bool is_skinny(int64_t M, int E, bool grouped) {
  return grouped ? M <= 16 * (int64_t)E && E < 32767 : M <= 32;   // (2 E + 1 workgroups along y)
}

// Many rows through one small matrix: the resident form (a tile for every CU at least).
bool is_resident(int64_t M, int64_t N, int64_t K, bool grouped) {
  return !grouped && N <= kResident && K <= kResident && M >= 256 * 128;
}

int check(const NerfFp8Linear* d) {
  NERF_REQUIRE(d && d->x && d->wq && d->ws && d->out, "nerf_fp8_linear: null pointer");
  NERF_REQUIRE(d->M >= 1 && d->N >= 1 && d->K >= 1 && d->M < (1ll << 31) && d->N < (1ll << 31) && d->K <= (1ll << 23),
               "nerf_fp8_linear: bad size");
  NERF_REQUIRE(d->x_type >= NERF_F32 && d->x_type <= NERF_F16 && d->out_type >= NERF_F32 && d->out_type <= NERF_F16,
               "nerf_fp8_linear: bad type");
  NERF_REQUIRE(d->E >= 1 && d->E <= 65534 && (d->offsets || d->E == 1), "nerf_fp8_linear: E matrices need offsets");
  NERF_REQUIRE(d->order ? d->slots >= 1 && d->x_rows >= 1 : d->x_rows == d->M, "nerf_fp8_linear: slots or rows of x");
  NERF_REQUIRE(d->offsets || !d->order, "nerf_fp8_linear: order without offsets");
  NERF_REQUIRE(d->ldx >= 0 && d->ldo >= d->N, "nerf_fp8_linear: row pitch");
  NERF_REQUIRE((uintptr_t)d->wq % 16 == 0, "nerf_fp8_linear: weights need 16-byte alignment");
  return 0;
}

}  // namespace
}  // namespace nerfhip

using namespace nerfhip;

extern "C" {

size_t nerf_fp8_linear_workspace(int64_t M, int64_t N, int64_t K, int E, int grouped) {
  if (M < 1 || N < 1 || K < 1 || is_skinny(M, E, grouped != 0) || is_resident(M, N, K, grouped != 0)) return 0;
  const int64_t KB = cdiv(K, 128);
  return (size_t)((M + 1) * KB * 128 + cdiv(KB, 4) * (M + 1) * 4);   // (a row of zeros behind the others)
}

int nerf_fp8_linear(const NerfFp8Linear* d, void* workspace, size_t workspace_bytes, nerf_stream_t stream) {
  if (const int rc = check(d)) return rc;
  const hipStream_t st = as_stream(stream);
  LinearArgs a;
  a.x = d->x;
  a.ldx = d->ldx;
  a.x_rows = d->x_rows;
  a.order = d->order;
  a.div = d->order ? d->slots : 1;
  a.wq = (const unsigned char*)d->wq;
  a.ws = (const unsigned char*)d->ws;
  a.offsets = d->offsets;
  a.E = d->E;
  a.bias = d->bias;
  a.relu = d->relu;
  a.M = d->M;
  a.N = d->N;
  a.K = d->K;
  a.KB = (int)cdiv(d->K, 128);
  a.NB = (int)cdiv(d->N, 128);
  a.out = d->out;
  a.ldo = d->ldo;
  a.q = nullptr;
  a.s = nullptr;
  a.q_rows = 0;
  a.gather = 0;
  if (is_skinny(d->M, d->E, d->offsets != nullptr)) {
    NERF_REQUIRE(launch_fits(cdiv(d->N, 64), 512), "nerf_fp8_linear: too many columns");
    if (d->x_type == NERF_F32) launch_skinny_out<float>(a, d->out_type, st);
    else if (d->x_type == NERF_BF16) launch_skinny_out<bf16>(a, d->out_type, st);
    else launch_skinny_out<f16>(a, d->out_type, st);
    return check_launch("nerf_fp8_linear");
  }
  if (is_resident(d->M, d->N, d->K, d->offsets != nullptr)) {
    if (d->x_type == NERF_F32) launch_resident_out<float>(a, d->out_type, st);
    else if (d->x_type == NERF_BF16) launch_resident_out<bf16>(a, d->out_type, st);
    else launch_resident_out<f16>(a, d->out_type, st);
    return check_launch("nerf_fp8_linear");
  }
  NERF_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                   workspace_bytes >= nerf_fp8_linear_workspace(d->M, d->N, d->K, d->E, d->offsets != nullptr),
               "nerf_fp8_linear: workspace too small or unaligned");
  unsigned char* q = (unsigned char*)workspace;
  // experts' rows: x is rounded once, not once for each of its slots, and the tiles take its rows where
  // they are (32-bit offsets)
  a.gather = d->order && (d->x_rows + 1) * a.KB * 128 < (1ll << 32) && d->x_rows <= d->M;
  a.q_rows = a.gather ? d->x_rows + 1 : d->M;
  unsigned char* s = q + a.q_rows * a.KB * 128;
  a.q = q;
  a.s = (const unsigned*)s;
  using S = TileShape<Fp8, 4, 4, 2, 2>;
  using SW = TileShape<Fp8Wide, 4, 4, 2, 2>;
  // 256 x 256 (128 x 128 for a wave, the whole register file) reads half as much LDS for each product,
  // but one workgroup on a CU has nobody to cover its start and end: for long rows and many tiles
  // (8192 x 8192 x 8192: 484 us against 632; 32768 rows of 2048 over 32 experts: 256 against 235).
  using SL = TileShape<Fp8, 8, 8, 2, 2>;
  const bool large = d->K >= 4096 && cdiv(d->M, 256) * cdiv(d->N, 256) >= 512;
  // 64 x 64 where the larger tiles would leave CUs without one.
  using SS = TileShape<Fp8, 2, 2, 2, 2>;
  using SWS = TileShape<Fp8Wide, 2, 2, 2, 2>;
  const bool small = (cdiv(d->M, 128) + (d->offsets ? (d->M < d->E ? d->M : d->E) : 0)) * cdiv(d->N, 128) <= 256;
  const int side = small ? SS::BM : S::BM;   // (the largest tiles are fewer)
  NERF_REQUIRE(launch_fits((d->M / side + d->E + 1) * cdiv(d->N, side), S::NT), "nerf_fp8_linear: too many tiles");
  if (d->x_type == NERF_F32) launch_quantize<float>(a, q, s, st);
  else if (d->x_type == NERF_BF16) launch_quantize<bf16>(a, q, s, st);
  else launch_quantize<f16>(a, q, s, st);
  if (const int rc = check_launch("nerf_fp8_linear")) return rc;
  if (small) {
    if (d->out_type == NERF_F32) launch_product<SWS, float>(a, st);
    else if (d->out_type == NERF_BF16) launch_product<SS, bf16>(a, st);
    else launch_product<SS, f16>(a, st);
  } else if (d->out_type == NERF_F32) launch_product<SW, float>(a, st);
  else if (d->out_type == NERF_BF16) large ? launch_product<SL, bf16>(a, st) : launch_product<S, bf16>(a, st);
  else large ? launch_product<SL, f16>(a, st) : launch_product<S, f16>(a, st);
  return check_launch("nerf_fp8_linear");
}

int nerf_fp8_quantize_weight(const void* w, int type, int64_t stack_stride, int64_t ldw, int E, int64_t N, int64_t K,
                             void* q, void* scale, nerf_stream_t stream) {
  NERF_REQUIRE(w && q && scale, "nerf_fp8_quantize_weight: null pointer");
  NERF_REQUIRE(E >= 1 && N >= 1 && K >= 1 && type >= NERF_F32 && type <= NERF_F16,
               "nerf_fp8_quantize_weight: bad size or type");
  const int64_t KB = cdiv(K, 128), NB = cdiv(N, 128);
  NERF_REQUIRE(KB < (1ll << 24) && NB < (1ll << 24) && E * NB * KB < (1ll << 31),
               "nerf_fp8_quantize_weight: too many blocks");
  NERF_REQUIRE((uintptr_t)q % 8 == 0, "nerf_fp8_quantize_weight: q needs 8-byte alignment");
  const int64_t blocks = E * NB * KB, most = 1 << 22;   // (of one launch)
  const hipStream_t st = as_stream(stream);
  for (int64_t first = 0; first < blocks; first += most) {
    const dim3 grid((unsigned)(blocks - first < most ? blocks - first : most)), block(256);
#define NERF_QW(T)                                                                                          \
  hipLaunchKernelGGL(quantize_weight_kernel<T>, grid, block, 0, st, (const T*)w, stack_stride, ldw, N, K,   \
                     (int)NB, (int)KB, first, (unsigned char*)q, (unsigned char*)scale)
    if (type == NERF_F32) NERF_QW(float);
    else if (type == NERF_BF16) NERF_QW(bf16);
    else NERF_QW(f16);
#undef NERF_QW
  }
  return check_launch("nerf_fp8_quantize_weight");
}

}  // extern "C"
