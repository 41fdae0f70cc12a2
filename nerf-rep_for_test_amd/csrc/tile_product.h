// The tiled product C[m][n] = sum_k M[m][k] N[n][k] of two row-major operands
// (the reduction axis contiguous in both), shared by the 8-bit block-scaled
// product (fp8_ops.hip) and the FP16-split products of the orthogonalisation
// (muon_ops.hip). Both operands are byte rows cut into chunks of 128 bytes, one
// chunk per K step:
//   Fp8:    128 e4m3 values, one v_mfma_scale_f32_16x16x128 per 16x16 tile;
//   Fp8Wide: the same values turned into FP16 (exact) in registers, four
//           v_mfma_f32_16x16x32_f16, the scale on their sum: the 8-bit instructions
//           add 8 neighbouring products with 13 bits below the largest one (seen
//           on the device), which a 16-bit result hides and an FP32 one does not;
//   Split:  32 values as 32 FP16 high parts then 32 FP16 low parts (x = hi + lo),
//           three v_mfma_f32_16x16x32_f16 (hi hi, hi lo, lo hi) per tile.
// A lane's two 16-byte pieces of a chunk (piece g and g + 4, g = lane / 16) are
// then the whole operand of either form, so staging and reading are the same.
//
// Staging: buffer loads into LDS (16 B per lane, no VGPRs) into two LDS stages; the
// next stage's loads are issued after this stage's fragment reads (the compiler
// waits for every outstanding LDS load before an LDS read) and land under its
// MFMAs. Piece p of row r lies at p ^ swz(r), so the 16 rows that a fragment
// read touches fall into the 16 different 16-byte slots of the 64 banks.
#pragma once

#include <type_traits>

#include "common.h"

namespace nerfhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Fp8 {};
struct Fp8Wide {};
struct Split {};

// 8 e4m3 values as FP16.
__device__ __forceinline__ f16x8 widen(int lo, int hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// acc + n m 2^(sn + sm - 254) for one block of 128 (a lane's 32 values of either), exact
// products; a scale of 255 is NaN.
__device__ __forceinline__ f32x4 wide_block(const i32x8& n, const i32x8& m, int sn, int sm, f32x4 acc) {
  f32x4 c = f32x4(0.0f);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(n[2 * q], n[2 * q + 1]), widen(m[2 * q], m[2 * q + 1]), c, 0, 0,
                                               0);
  const int e = sn + sm - 254;
  const float none = sn == 255 || sm == 255 ? __builtin_nanf("") : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += __builtin_ldexpf(c[i], e) + none;
  return acc;
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)v);
  const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// A buffer's range: everything, or nothing. (Opaque to the compiler, which would branch over the
// loads otherwise.)
__device__ __forceinline__ int range_of(bool live) { return __builtin_amdgcn_readfirstlane(live ? -1 : 0); }

// TM x TN tiles of 16 x 16 per wave, WR x WC waves.
template <class MODE, int TM_, int TN_, int WR_, int WC_>
struct TileShape {
  using Mode = MODE;
  static constexpr int TM = TM_, TN = TN_, WR = WR_, WC = WC_;
  static constexpr int BM = 16 * TM * WR, BN = 16 * TN * WC, NT = 64 * WR * WC;
  static constexpr int kStage = (BM + BN) * 128;   // bytes of one stage
  static constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;   // 16-byte pieces per thread
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole pieces per thread");
};

// Tile t, index a (0..15) of a wave's 16 T rows <-> row (a / 4) 4 T + 4 t + a % 4: a lane's
// results of all its tiles are then 4 T neighbours.
template <int T>
__device__ __forceinline__ constexpr int tile_row(int t, int a) {
  return (a >> 2) * 4 * T + 4 * t + (a & 3);
}
template <int T>
__device__ __forceinline__ constexpr int swz(int r) {
  return ((r / (4 * T)) & 3) * 2 + ((r >> 1) & 1);
}

template <class S>
struct TileProduct {
  static constexpr int TM = S::TM, TN = S::TN;
  f32x4 acc[TM][TN];
  const char* a0;          // the tile's first rows
  const char* b0;
  unsigned va[S::LA];      // this thread's pieces: byte offsets from them
  unsigned vb[S::LB];

  // Rows m0 .. (below M) of A and n0 .. (below N) of B; rows behind the last one read the last one
  // again (their results are not stored). lda, ldb: bytes, 2^24 at most.
  __device__ __forceinline__ void init(const char* A, int64_t lda, int64_t m0, int64_t M, const char* B,
                                       int64_t ldb, int64_t n0, int64_t N) {
    const int t = threadIdx.x;
    a0 = (const char*)uniform((int64_t)(A + m0 * lda));
    const int am = (int)(M - 1 - m0 < S::BM ? M - 1 - m0 : S::BM);
#pragma unroll
    for (int i = 0; i < S::LA; ++i) {
      const int idx = i * S::NT + t, r = idx >> 3, p = (idx & 7) ^ swz<TM>(r);
      va[i] = (unsigned)(r < am ? r : am) * (unsigned)lda + p * 16;
    }
    set_n(B, ldb, n0, N);
    clear();
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4(0.0f);
  }

  // The N rows n0 .. (below N) of B instead.
  __device__ __forceinline__ void set_n(const char* B, int64_t ldb, int64_t n0, int64_t N) {
    const int t = threadIdx.x;
    b0 = (const char*)uniform((int64_t)(B + n0 * ldb));
    const int bm = (int)(N - 1 - n0 < S::BN ? N - 1 - n0 : S::BN);
#pragma unroll
    for (int i = 0; i < S::LB; ++i) {
      const int idx = i * S::NT + t, r = idx >> 3, p = (idx & 7) ^ swz<TN>(r);
      vb[i] = (unsigned)(r < bm ? r : bm) * (unsigned)ldb + p * 16;
    }
  }

  // Starts the loads of chunk k of an operand (M's rows, N's rows) into LDS. `live` false: nothing
  // is read (an empty range: zeros arrive), so that a loop's last step needs no branch around its
  // loads; wait for them all the same before the LDS is used again or the wave ends.
  __device__ __forceinline__ void load_m(char* to, int k, bool live) const { pieces<S::LA>(a0, va, to, k, live); }
  __device__ __forceinline__ void load_n(char* to, int k, bool live) const { pieces<S::LB>(b0, vb, to, k, live); }
  __device__ __forceinline__ void load(char* stage, int k, bool live) const {
    load_m(stage, k, live);
    load_n(stage + S::BM * 128, k, live);
  }
  template <int L>
  static __device__ __forceinline__ void pieces(const char* base, const unsigned (&v)[L], char* to, int k, bool live) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)k * 128), 0, range_of(live), 0x00020000);
#pragma unroll
    for (int i = 0; i < L; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(to + (i * S::NT + w * 64) * 16), 16, (int)v[i], 0, 0, 0);
  }

  struct Frags {
    i32x4 m[TM][2], n[TN][2];
  };
  __device__ __forceinline__ void read(Frags& f, const char* stage) const { read(f, stage, stage + S::BM * 128); }
  __device__ __forceinline__ void read(Frags& f, const char* sa, const char* sb) const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, a = lane & 15;
    const int wr = (w / S::WC) * 16 * TM, wc = (w % S::WC) * 16 * TN;
    // one N and one M tile in turn: the first products need only the first of each
#pragma unroll
    for (int d = 0; d < (TM > TN ? TM : TN); ++d) {
      if (d < TN) {
        const int r = wc + tile_row<TN>(d, a);
        f.n[d][0] = *(const i32x4*)(sb + r * 128 + ((g ^ swz<TN>(r)) << 4));
        f.n[d][1] = *(const i32x4*)(sb + r * 128 + (((g + 4) ^ swz<TN>(r)) << 4));
      }
      if (d < TM) {
        const int r = wr + tile_row<TM>(d, a);
        f.m[d][0] = *(const i32x4*)(sa + r * 128 + ((g ^ swz<TM>(r)) << 4));
        f.m[d][1] = *(const i32x4*)(sa + r * 128 + (((g + 4) ^ swz<TM>(r)) << 4));
      }
    }
  }

  // The products in growing squares (i, j <= d), as their operands arrive.
  template <class F>
  static __device__ __forceinline__ void squares(F f) {
#pragma unroll
    for (int d = 0; d < (TM > TN ? TM : TN); ++d) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (j < d && d < TM) f(d, j);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i <= d && d < TN) f(i, d);
    }
  }

  static __device__ __forceinline__ i32x8 join(const i32x4* p) {
    return __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // Fp8, Fp8Wide: sm[i] / sn: the rows' scales in the lowest byte (E8M0).
  __device__ __forceinline__ void mul(const Frags& f, const int (&sm)[TM], int sn) {
    squares([&](int i, int j) {
      if constexpr (std::is_same<typename S::Mode, Fp8Wide>::value)
        acc[i][j] = wide_block(join(f.n[j]), join(f.m[i]), sn & 255, sm[i] & 255, acc[i][j]);
      else
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(f.n[j]), join(f.m[i]), acc[i][j], 0, 0, 0,
                                                                     sn, 0, sm[i]);
    });
  }

  __device__ __forceinline__ void mul(const Frags& f) {
    squares([&](int i, int j) {
      const f16x8 mh = __builtin_bit_cast(f16x8, f.m[i][0]), ml = __builtin_bit_cast(f16x8, f.m[i][1]);
      const f16x8 nh = __builtin_bit_cast(f16x8, f.n[j][0]), nl = __builtin_bit_cast(f16x8, f.n[j][1]);
      f32x4 c = acc[i][j];
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nh, mh, c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nl, mh, c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nh, ml, c, 0, 0, 0);
      acc[i][j] = c;
    });
  }

  // This lane's result rows and columns within the workgroup's tile: tile i -> row m(i),
  // columns n() .. n() + 4 TN (acc[i][j][r] is column n() + 4 j + r).
  __device__ __forceinline__ int m(int i) const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    return (w / S::WC) * 16 * TM + tile_row<TM>(i, lane & 15);
  }
  __device__ __forceinline__ int n() const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    return (w % S::WC) * 16 * TN + (lane >> 4) * 4 * TN;
  }
};

// Every wave's outstanding loads have landed and every wave is here.
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Workgroup p of `total` -> the tile it takes: workgroups go round-robin over the 8 XCDs, so
// the ones on one XCD (and its L2) take a run of neighbouring tiles.
__device__ __forceinline__ int64_t xcd_tile(int64_t p, int64_t total) {
  const int64_t q = total / 8, rem = total % 8, x = p % 8, i = p / 8;
  return x * q + (x < rem ? x : rem) + i;
}

// The order in which an XCD walks mtiles x ntiles: bands of `band` row tiles, down a band's
// column before the next one, so that the tiles in flight form a patch and share both operands in L2.
__device__ __forceinline__ void band_tile(int64_t id, int mtiles, int ntiles, int band, int& mt, int& nt) {
  const int64_t per = (int64_t)band * ntiles;
  const int b = (int)(id / per), m0 = b * band, h = mtiles - m0 < band ? mtiles - m0 : band;
  const int r = (int)(id - b * per);
  nt = r / h;
  mt = m0 + r - nt * h;
}

}  // namespace nerfhip
