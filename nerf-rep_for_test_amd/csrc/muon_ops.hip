// Muon's update: momentum, Newton-Schulz orthogonalisation, weight decay and the step.
//   buf = mu buf + g,  u = g + mu buf (Nesterov; else u = buf),  X = u / (|u| + eps),
//   steps times:  A = X X^T,  B = b A + c A A,  X = a X + B X,
//   p = p (1 - lr wd) - lr sqrt(max(1, m / n)) X;
// or X alone (orthogonalisation). X is worked on with its short side r as rows ([r][c],
// the transpose of a tall matrix). The quintic a s + b s^3 + c s^5 keeps singular values
// within [0, 1.21] (its maximum on [0, 1.21] is 1.2024), which bounds every entry:
// |X| <= 1.21, |A| <= 1.45, |B| <= 2.81.
//
// Products are FP32-accurate on the FP16 matrix cores (tile_product.h, Split): operands
// as hi + lo FP16, x = hi + lo to 22 bits, three terms in FP32 accumulators. The bounds
// above let X be held times S (a power of two near sqrt(r c), at most 2^15), A times 2^15
// and B times 2^14, so lo parts stay clear of FP16's least numbers and nothing overflows.
// Where |u| is small beside eps, X starts at t = |u| / (|u| + eps) and grows by a = 3.4445 a step at
// most: it is held times S 2^j with the largest j that keeps t a^k 2^j within the same bound, from t, on the
// device, for each matrix and step (grown_shift; j is 0 from t = 0.6 on). Without it X's FP16 parts ran
// out of bits (relative errors of 2e-5 at t = 1e-3, all of it at 1e-9).
// The three products of a step are one launch each over all matrices. A and B are
// symmetric: only tiles on and below the diagonal are computed and each is stored twice.
// Large matrices are bound by the matrix cores (B X for two of 2048 x 4096 and one of 2048 x 2048: 242 to 262 us,
// 1.0 to 1.07 PFLOP/s in FP16; the library's FP16 product reaches 1.15), small ones by the latency of 17
// launches (the trainer's 20 matrices: 150 us, 8 to 13 a launch), those between by HBM (32 of
// 512 x 1024: B X moves 300 MB in 77 to 84 us).
// All sums have a fixed order. X is kept in both layouts (rows for A, its transpose for
// B X), since the product takes both operands with the reduction axis contiguous.
#include "tile_product.h"

namespace nerfhip {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScaleA = 32768.0f, kScaleB = 16384.0f;
constexpr int kMaxGroups = 32;    // stacks of equal matrices in one launch
constexpr int kNormBlocks = 512;  // partial sums of one matrix's norm, at most
// .. and behind them t, as a float. (128 bytes, a cache line: rows of the buffers that follow keep to lines, 2430 us
// against 3010 for the large matrices)
constexpr int kNormSlots = kNormBlocks + 16;
constexpr float kBound = 1.2024f; // singular values of X
constexpr int kMaxShift = 110;    // (1 / (S 2^j) stays a normal number)

struct Group {
  void* out;           // parameters (FP32) or results, [count] matrices out_stride apart
  const void* g;       // [count][m][n], g_stride apart
  float* buf;          // momentum, contiguous, or null
  int64_t out_stride, g_stride;
  char* work;          // per matrix: Xs, Xt, Xt', A, B (split rows)
  double* norm;        // [count][kNormSlots]
  int m, n, r, c, count;
  int norm_blocks;
  float s;             // S of X's scale S 2^j
  float adjust;        // sqrt(max(1, m / n))
};

struct Batch {
  Group g[kMaxGroups];
  int end[kMaxGroups];   // prefix sums of the groups' workgroups
  int count;
  float mu, clip, eps, decay, lr;
  const float* lr_dev;
  int nesterov, type;
};

// Bytes of a row of `n` values as split chunks.
__host__ __device__ inline int64_t row_bytes(int n) { return cdiv(n, 32) * 128; }

struct Work {   // one matrix's buffers
  char *xs, *xt0, *xt1, *a, *b;
};
__host__ __device__ inline int64_t work_bytes(int r, int c) {
  return r * row_bytes(c) + 2 * (int64_t)c * row_bytes(r) + 2 * (int64_t)r * row_bytes(r);
}
__device__ __forceinline__ Work work_of(const Group& g, int i) {
  Work w;
  w.xs = g.work + i * work_bytes(g.r, g.c);
  w.xt0 = w.xs + g.r * row_bytes(g.c);
  w.xt1 = w.xt0 + g.c * row_bytes(g.r);
  w.a = w.xt1 + g.c * row_bytes(g.r);
  w.b = w.a + g.r * row_bytes(g.r);
  return w;
}

__device__ __forceinline__ int find_group(const Batch& b, int& blk) {
  int k = 0;
#pragma unroll
  for (int step = kMaxGroups / 2; step >= 1; step /= 2)   // the first group that ends behind blk
    if (k + step <= b.count - 1 && blk >= b.end[k + step - 1]) k += step;
  blk -= k ? b.end[k - 1] : 0;
  return k;
}

// j of a matrix whose singular values are t grow at most (grow = a^k: infinity for large k).
__device__ __forceinline__ int grown_shift(float t, float grow) {
  const float m = fminf(t * grow, kBound) * (1.0f / kBound);   // (0 inf, NaN: kBound)
  int e;
  __builtin_frexpf(m, &e);
  return e > 0 ? 0 : (e < -kMaxShift ? kMaxShift : -e);
}
__device__ __forceinline__ float size_of(const Group& g, int i) {
  return *(const float*)(g.norm + (int64_t)i * kNormSlots + kNormBlocks);
}

struct HiLo {
  f16 hi, lo;
};
__device__ __forceinline__ HiLo split(float v) {
  HiLo s;
  s.hi = (f16)v;
  s.lo = (f16)(v - (float)s.hi);
  return s;
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
  if (type == NERF_F32) return ((const float*)p)[i];
  if (type == NERF_BF16) return (float)((const bf16*)p)[i];
  return (float)((const f16*)p)[i];
}

__device__ __forceinline__ float clipped(float g, float clip) {   // (NaN stays)
  if (clip < 0.0f) return g;
  return g > clip ? clip : (g < -clip ? -clip : g);
}

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// W (4 or 1) neighbours from element i on as FP32.
template <int W>
__device__ __forceinline__ void load_w(float (&f)[W], const void* p, int type, int64_t i) {
  if (W == 1) {
    f[0] = load_any(p, type, i);
  } else if (type == NERF_F32) {
    const Vec<float, W> v = *(const Vec<float, W>*)((const float*)p + i);
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = v.v[e];
  } else if (type == NERF_BF16) {
    const Vec<bf16, W> v = *(const Vec<bf16, W>*)((const bf16*)p + i);
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = (float)v.v[e];
  } else {
    const Vec<f16, W> v = *(const Vec<f16, W>*)((const f16*)p + i);
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = (float)v.v[e];
  }
}

// The momentum is advanced and the matrices' squares are summed (64 bits: no overflow, a fixed
// order). 4 runs of W values of a thread are in flight together: bound by HBM, 252 MB in 44 us
// (5.7 TB/s, part of it from the last-level cache).
template <int W>
__device__ __forceinline__ double norm_part(const Batch& b, const char* src, float* buf, int64_t n, int part, int parts) {
  double sum = 0.0;
  const int64_t step = (int64_t)parts * 256 * W;
  for (int64_t k0 = ((int64_t)part * 256 + threadIdx.x) * W; k0 < n; k0 += 4 * step) {
    float v[4][W], m[4][W] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t k = k0 + u * step;
      if (k < n) {
        load_w<W>(v[u], src, b.type, k);
        if (buf) load_w<W>(m[u], buf, NERF_F32, k);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t k = k0 + u * step;
      if (k < n) {
        Vec<float, W> o;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          float x = clipped(v[u][e], b.clip);
          if (buf) {
            o.v[e] = m[u][e] * b.mu + x;
            x = b.nesterov ? x + b.mu * o.v[e] : o.v[e];
          }
          sum += (double)x * x;
        }
        if (buf) *(Vec<float, W>*)(buf + k) = o;
      }
    }
  }
  return sum;
}

__global__ __launch_bounds__(256) void muon_norm_kernel(const Batch b) {
  int blk = blockIdx.x;
  const Group& g = b.g[find_group(b, blk)];
  const int i = blk / g.norm_blocks, part = blk - i * g.norm_blocks;
  const int64_t n = (int64_t)g.m * g.n;
  const int size = b.type == NERF_F32 ? 4 : 2;
  const char* src = (const char*)g.g + i * g.g_stride * size;
  float* buf = g.buf ? g.buf + i * n : nullptr;
  const bool vec = n % 4 == 0 && ((uintptr_t)src % (4 * size) | (uintptr_t)buf % 16) == 0;
  double sum = vec ? norm_part<4>(b, src, buf, n, part, g.norm_blocks) : norm_part<1>(b, src, buf, n, part, g.norm_blocks);
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  __shared__ double w[4];
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) g.norm[(int64_t)i * kNormSlots + part] = (w[0] + w[1]) + (w[2] + w[3]);
}

__device__ __forceinline__ void put8(char* row, int k, const HiLo (&v)[8]) {   // columns k .. k + 8 of a split row
  f16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = v[i].hi;
    l[i] = v[i].lo;
  }
  char* at = row + (k >> 5) * 128 + (k & 31) * 2;
  *(f16x8*)at = h;
  *(f16x8*)(at + 64) = l;
}

// u / (|u| + eps) times S 2^j in both layouts. A workgroup takes 64 x 64 of [m][n]. Bound by HBM: 336 MB in
// 59 to 69 us (5.7 to 4.9 TB/s) for 21 M elements with their momentum.
__global__ __launch_bounds__(256) void muon_split_kernel(const Batch b) {
  __shared__ float tile[64][65];
  __shared__ double wsum[4];
  int blk = blockIdx.x;
  const Group& g = b.g[find_group(b, blk)];
  const int tn = (g.n + 63) / 64, tm = (g.m + 63) / 64;
  const int i = blk / (tm * tn), t = blk - i * tm * tn, m0 = t / tn * 64, n0 = t % tn * 64;
  double sum = 0.0;
  for (int k = threadIdx.x; k < g.norm_blocks; k += 256) sum += g.norm[(int64_t)i * kNormSlots + k];
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double norm = __builtin_sqrt((wsum[0] + wsum[1]) + (wsum[2] + wsum[3]));
  const float size0 = (float)(norm / (norm + (double)b.eps));
  if (t == 0 && threadIdx.x == 0) *(float*)(g.norm + (int64_t)i * kNormSlots + kNormBlocks) = size0;
  // (64 bits: beyond 32 for a small |u| or eps)
  const double inv = __builtin_ldexp((double)g.s, grown_shift(size0, 1.0f)) / (norm + (double)b.eps);
  const int64_t size = (int64_t)g.m * g.n;
  const char* src = (const char*)g.g + i * g.g_stride * (b.type == NERF_F32 ? 4 : 2);
  const float* buf = g.buf ? g.buf + i * size : nullptr;
  float v[16], mo[16] = {};
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int y = u * 4 + (threadIdx.x >> 6), x = threadIdx.x & 63;
    v[u] = 0.0f;
    if (m0 + y < g.m && n0 + x < g.n) {
      const int64_t k = (int64_t)(m0 + y) * g.n + n0 + x;
      v[u] = load_any(src, b.type, k);
      if (buf) mo[u] = buf[k];
    }
  }
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    float x = clipped(v[u], b.clip);
    if (buf) x = b.nesterov ? x + b.mu * mo[u] : mo[u];
    tile[u * 4 + (threadIdx.x >> 6)][threadIdx.x & 63] = (float)((double)x * inv);
  }
  __syncthreads();
  const Work w = work_of(g, i);
  const bool tall = g.m > g.n;
  char* mat = tall ? w.xt0 : w.xs;   // rows like [m][n]
  char* tra = tall ? w.xs : w.xt0;   // rows like [n][m]
  const int64_t lm = row_bytes(g.n), ln = row_bytes(g.m);
  const int pn = (g.n + 31) & ~31, pm = (g.m + 31) & ~31;
  for (int q = threadIdx.x; q < 512; q += 256) {
    const int row = q >> 3, k = (q & 7) * 8;
    HiLo v[8];
    if (m0 + row < g.m && n0 + k < pn) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = split(tile[row][k + e]);
      put8(mat + (m0 + row) * lm, n0 + k, v);
    }
    if (n0 + row < g.n && m0 + k < pm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = split(tile[k + e][row]);
      put8(tra + (n0 + row) * ln, m0 + k, v);
    }
  }
}

// 8 neighbours of the result (room: how many exist): the step on the parameters, or X itself.
template <class T>
__device__ __forceinline__ void finish(T* at, const float (&f)[8], int room, bool update, float keep, float rate) {
  constexpr int W = 16 / sizeof(T);
  if (room >= 8 && (uintptr_t)at % 16 == 0) {
    Vec<T, W> o[8 / W];
    if (update) {
#pragma unroll
      for (int h = 0; h < 8 / W; ++h) o[h] = *(const Vec<T, W>*)(at + h * W);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      T& v = o[e / W].v[e % W];
      v = update ? (T)((float)v * keep - f[e] * rate) : (T)f[e];
    }
#pragma unroll
    for (int h = 0; h < 8 / W; ++h) *(Vec<T, W>*)(at + h * W) = o[h];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < room) at[e] = update ? (T)((float)at[e] * keep - f[e] * rate) : (T)f[e];
  }
}

enum { kStepA = 0, kStepB = 1, kStepX = 2, kStepLast = 3 };

// One product of a step for every matrix of the batch; flip: which of the two transposes is read; grow: a^k of
// step k. (Two
// waves on a SIMD: the accumulators stay in place in the VGPRs; with the whole register file the compiler
// put them into AGPRs and moved them every step, 2690 us against 2520 for the large matrices.)
template <class S, int STEP, class T>
__global__ __launch_bounds__(S::NT, 2) void muon_product_kernel(const Batch bt, int flip, float grow) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int TM = S::TM, TN = S::TN;
  int blk = blockIdx.x;
  const Group& g = bt.g[find_group(bt, blk)];
  const int rows = g.r, cols = STEP >= kStepX ? g.c : g.r;
  const int tm = (rows + S::BM - 1) / S::BM, tn = (cols + S::BN - 1) / S::BN;
  const int tiles = STEP >= kStepX ? tm * tn : tm * (tm + 1) / 2;
  const int i = blk / tiles, t = blk - i * tiles;
  int mt, nt;
  if (STEP >= kStepX) {
    mt = t % tm;
    nt = t / tm;
  } else {   // the tiles on and below the diagonal, row by row
    mt = (int)((__builtin_sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
    while (mt * (mt + 1) / 2 > t) --mt;
    while ((mt + 1) * (mt + 2) / 2 <= t) ++mt;
    nt = t - mt * (mt + 1) / 2;
  }
  const Work w = work_of(g, i);
  const char* xt = flip ? w.xt1 : w.xt0;
  const char* M = STEP == kStepA ? w.xs : (STEP == kStepB ? w.a : w.b);
  const char* N = STEP == kStepA ? w.xs : (STEP == kStepB ? w.a : xt);
  const int kdim = STEP == kStepA ? g.c : g.r;
  const int64_t ld = row_bytes(kdim);
  const int m0 = mt * S::BM, n0 = nt * S::BN, steps = (kdim + 31) / 32;
  const float size = STEP == kStepB ? 0.0f : size_of(g, i);   // (on its way during the product)
  TileProduct<S> p;
  p.init(M, ld, m0, rows, N, ld, n0, cols);
  using P = TileProduct<S>;
  constexpr int kLoads = S::LA + S::LB;
  tile_steps<S, kLoads>(
      steps, [&](int k) { return p.loads(lds + k % S::NS * S::kStage, k, k < steps); },
      [&](const typename P::Loads& l, int q) { p.load_one(l, q); },
      [&](int k, auto part) {
        const char* stage = lds + k % S::NS * S::kStage;
        p.chunk(stage, stage + S::BM * 128, kLoads, part);
      },
      [](int) {},
      // (its wait here, behind the first loads: a scalar load still open in the loop would make every wait for an
      // operand from LDS one for all of them)
      [&] { asm volatile("" ::"s"(size)); });
  char* to = STEP == kStepA ? w.a : (STEP == kStepB ? w.b : w.xs);
  const char* add = STEP == kStepB ? w.a : w.xs;   // the term beside the product
  const int64_t lto = row_bytes(cols);
  constexpr int PITCH = S::BM + 4;   // LDS row of the transposed tile, words
  unsigned* tr = (unsigned*)lds;
  // X comes times g.s 2^j and goes on times g.s 2^(j + next) (A of a large j is nothing beside 1: 0)
  const int j = STEP == kStepB ? 0 : grown_shift(size, grow);
  const float unscale = STEP == kStepA ? __builtin_ldexpf(kScaleA / (g.s * g.s), -2 * j) : 1.0f;
  const float next = STEP == kStepX ? __builtin_ldexpf(1.0f, grown_shift(size, grow * kA) - j) : 1.0f;
  const float beside_x = kA * next, acc_x = 1.0f / kScaleB * next, unscale_x = __builtin_ldexpf(1.0f / g.s, -j);
  const float lr = STEP == kStepLast ? (bt.lr_dev ? *bt.lr_dev : bt.lr) : 0.0f;
  const float keep = 1.0f - lr * bt.decay, rate = lr * g.adjust;
  const bool tall = g.m > g.n, once = STEP < kStepX && mt == nt;   // (on the diagonal: no transposed tile)
  const bool whole = m0 + S::BM <= rows && n0 + S::BN <= cols;
  // (whole tiles without a question around each access: the trainer's matrices 150 us against 157, 32 of
  // 512 x 1024 827 against 843)
  auto epilogue = [&](auto all) {
    constexpr bool ALL = decltype(all)::value;
#pragma unroll
    for (int q = 0; q < TM; ++q) {
      const int ml = p.m(q), m = m0 + ml;
#pragma unroll
      for (int h = 0; h < 4 * TN; h += 8) {
        HiLo v[8];
        float f[8];
        const int nl = p.n(h / 8), nn = n0 + nl;
        f16x8 ah = {}, al = {};
        if (STEP != kStepA && (ALL || (m < rows && nn < cols))) {
          const char* at = add + m * lto + (nn >> 5) * 128 + (nn & 31) * 2;
          ah = *(const f16x8*)at;
          al = *(const f16x8*)(at + 64);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float acc = p.acc[q][(h + e) / 4][(h + e) % 4];
          float x = acc;
          const float beside = (float)ah[e] + (float)al[e];
          if (STEP == kStepA) x = acc * unscale;
          if (STEP == kStepB) x = kB * (kScaleB / kScaleA) * beside + kC * (kScaleB / (kScaleA * kScaleA)) * acc;
          if (STEP >= kStepX) x = beside_x * beside + acc_x * acc;
          f[e] = ALL || nn + e < cols ? x : 0.0f;
          if (STEP != kStepLast) v[e] = split(f[e]);
        }
        if (STEP == kStepLast) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= unscale_x;
          if (tall) {
#pragma unroll
            for (int e = 0; e < 8; ++e) tr[(nl + e) * PITCH + ml] = __float_as_uint(f[e]);
          } else if (ALL || m < rows) {
            finish<T>((T*)g.out + i * g.out_stride + (int64_t)m * g.n + nn, f, ALL ? 8 : cols - nn, g.buf != nullptr, keep, rate);
          }
        } else {
          if (ALL || (m < rows && nn < ((cols + 31) & ~31))) put8(to + m * lto, nn, v);
          if (!once) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              tr[(nl + e) * PITCH + ml] =
                  (unsigned)__builtin_bit_cast(unsigned short, v[e].hi) | (unsigned)__builtin_bit_cast(unsigned short, v[e].lo) << 16;
          }
        }
      }
    }
    if (once || (STEP == kStepLast && !tall)) return;
    __syncthreads();
    // the transposed tile: rows n, 8 columns m at a time
    char* tt = STEP == kStepA ? w.a : (STEP == kStepB ? w.b : (flip ? w.xt0 : w.xt1));
    const int64_t ltt = row_bytes(rows);
    for (int q = threadIdx.x; q < S::BN * S::BM / 8; q += S::NT) {
      const int nl = q / (S::BM / 8), k = q % (S::BM / 8) * 8, nn = n0 + nl, m = m0 + k;
      if (!ALL && (nn >= cols || m >= ((rows + 31) & ~31))) continue;
      const unsigned* at = tr + nl * PITCH + k;
      if (STEP == kStepLast) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(at[e]);
        finish<T>((T*)g.out + i * g.out_stride + (int64_t)nn * g.n + m, f, ALL ? 8 : rows - m, g.buf != nullptr, keep, rate);
      } else {
        HiLo v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned u = ALL || m + e < rows ? at[e] : 0u;
          v[e].hi = __builtin_bit_cast(f16, (unsigned short)(u & 0xffffu));
          v[e].lo = __builtin_bit_cast(f16, (unsigned short)(u >> 16));
        }
        put8(tt + nn * ltt, m, v);
      }
    }
  };
  if (whole) epilogue(std::true_type());
  else epilogue(std::false_type());
}

// ---------------------------------------------------------------- launches

int check_group(const NerfMuonGroup& g, bool update) {
  NERF_REQUIRE(g.out && g.g && (!update || g.momentum), "nerf_muon: null pointer");
  NERF_REQUIRE(g.m >= 1 && g.n >= 1 && g.count >= 1 && g.m <= (1 << 20) && g.n <= (1 << 20) &&
                   g.count < (1 << 20) && g.g_stride >= 0 && g.out_stride >= 0,
               "nerf_muon: bad size");
  return 0;
}

int64_t group_bytes(const NerfMuonGroup& g) {
  const int r = (int)(g.m < g.n ? g.m : g.n), c = (int)(g.m < g.n ? g.n : g.m);
  return g.count * (work_bytes(r, c) + (int64_t)kNormSlots * 8);
}

int64_t count_tiles(const Group& g, int bm, int bn, bool square) {
  const int64_t tm = cdiv(g.r, bm), tn = cdiv(g.c, bn);
  return g.count * (square ? tm * (tm + 1) / 2 : tm * tn);
}

template <class S>
constexpr size_t lds_bytes() {
  const size_t a = S::NS * S::kStage, b = (size_t)S::BN * (S::BM + 4) * 4;
  return a > b ? a : b;
}

template <class S, int STEP, class T>
int launch_step(Batch& b, int flip, float grow, hipStream_t st) {
  int64_t end = 0;
  for (int k = 0; k < b.count; ++k) {
    end += count_tiles(b.g[k], S::BM, S::BN, STEP < kStepX);
    NERF_REQUIRE(launch_fits(end, S::NT), "nerf_muon: too many tiles");
    b.end[k] = (int)end;
  }
  hipLaunchKernelGGL((muon_product_kernel<S, STEP, T>), dim3((unsigned)end), dim3(S::NT), lds_bytes<S>(),
                     st, b, flip, grow);
  return check_launch("nerf_muon");
}

template <class S>
int run_steps(Batch& b, int steps, bool update, hipStream_t st) {
  float grow = 1.0f;
  for (int k = 0; k < steps; ++k, grow *= kA) {
    const int flip = k & 1;
    if (const int rc = launch_step<S, kStepA, float>(b, flip, grow, st)) return rc;
    if (const int rc = launch_step<S, kStepB, float>(b, flip, grow, st)) return rc;
    int rc;
    if (k + 1 < steps) rc = launch_step<S, kStepX, float>(b, flip, grow, st);
    else if (update || b.type == NERF_F32) rc = launch_step<S, kStepLast, float>(b, flip, grow, st);
    else if (b.type == NERF_BF16) rc = launch_step<S, kStepLast, bf16>(b, flip, grow, st);
    else rc = launch_step<S, kStepLast, f16>(b, flip, grow, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace
}  // namespace nerfhip

using namespace nerfhip;

extern "C" {

size_t nerf_muon_workspace(const NerfMuonGroup* groups, int n) {
  size_t s = 0;
  for (int k = 0; groups && k < n; ++k) s += (size_t)group_bytes(groups[k]);
  return s;
}

int nerf_muon(const NerfMuonGroup* groups, int n, const NerfMuonOptions* o, void* workspace, size_t workspace_bytes,
              nerf_stream_t stream) {
  NERF_REQUIRE(groups && o, "nerf_muon: null pointer");
  NERF_REQUIRE(n >= 1 && o->steps >= 1 && o->type >= NERF_F32 && o->type <= NERF_F16 &&
                   (!o->update || o->type == NERF_F32),
               "nerf_muon: bad count, steps or type");
  NERF_REQUIRE(o->eps > 0.0f && o->eps <= 3.402823466e+38f, "nerf_muon: eps must be positive and finite");
  for (int k = 0; k < n; ++k)
    if (const int rc = check_group(groups[k], o->update != 0)) return rc;
  NERF_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= nerf_muon_workspace(groups, n),
               "nerf_muon: workspace too small or unaligned");
  const hipStream_t st = as_stream(stream);
  char* at = (char*)workspace;
  for (int first = 0; first < n; first += kMaxGroups) {
    Batch b;
    b.count = n - first < kMaxGroups ? n - first : kMaxGroups;
    b.mu = o->momentum;
    b.clip = o->clip;
    b.eps = o->eps;
    b.decay = o->weight_decay;
    b.lr = o->lr;
    b.lr_dev = o->lr_device;
    b.nesterov = o->nesterov;
    b.type = o->type;
    int64_t end = 0, split_end[kMaxGroups], tiles64 = 0, tiles = 0;
    for (int k = 0; k < b.count; ++k) {
      const NerfMuonGroup& s = groups[first + k];
      Group& g = b.g[k];
      g.out = s.out;
      g.g = s.g;
      g.buf = o->update ? s.momentum : nullptr;
      g.out_stride = s.out_stride;
      g.g_stride = s.g_stride;
      g.m = (int)s.m;
      g.n = (int)s.n;
      g.count = (int)s.count;
      g.r = g.m < g.n ? g.m : g.n;
      g.c = g.m < g.n ? g.n : g.m;
      const int64_t size = s.m * s.n;
      const int64_t nb = cdiv(size, 2048);
      g.norm_blocks = (int)(nb < kNormBlocks ? nb : kNormBlocks);
      int e = 0;
      while (e < 15 && (1ll << (2 * e)) < size) ++e;
      g.s = (float)(1 << e);
      g.adjust = s.m > s.n ? (float)__builtin_sqrt((double)s.m / (double)s.n) : 1.0f;
      g.norm = (double*)at;
      at += g.count * (int64_t)kNormSlots * 8;
      g.work = at;
      at += g.count * work_bytes(g.r, g.c);
      end += (int64_t)g.count * g.norm_blocks;
      b.end[k] = (int)end;
      tiles += g.count * cdiv(s.m, 64) * cdiv(s.n, 64);
      split_end[k] = tiles;
      tiles64 += count_tiles(g, 128, 128, false);
      NERF_REQUIRE(launch_fits(end, 256) && launch_fits(tiles, 256), "nerf_muon: too many tiles");
    }
    hipLaunchKernelGGL(muon_norm_kernel, dim3((unsigned)end), dim3(256), 0, st, b);
    for (int k = 0; k < b.count; ++k) b.end[k] = (int)split_end[k];
    hipLaunchKernelGGL(muon_split_kernel, dim3((unsigned)tiles), dim3(256), 0, st, b);
    if (const int rc = check_launch("nerf_muon")) return rc;
    // 128 x 128 tiles read each operand half as often; 64 x 64 ones fill the CUs where there are few
    using Large = TileShape<Split, 4, 4, 2, 2>;
    using Small = TileShape<Split, 2, 2, 2, 2>;
    const int rc = tiles64 >= 256 ? run_steps<Large>(b, o->steps, o->update != 0, st)
                                  : run_steps<Small>(b, o->steps, o->update != 0, st);
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
