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
// Staging: buffer loads straight into LDS (16 B per lane, no VGPRs), S::NS stages. They
// are issued by inline assembly: the compiler, which cannot tell the stages apart, would
// make every LDS read wait for all of them, while here a step waits for its own stage
// only (stage_ready) and the loads of the next NS - 1 stages stay in flight. They write
// no registers. Counts that the compiler takes of its own loads remain right: more loads
// in flight only make its waits longer.
// Piece p of row r lies at p ^ swz(r), so the 16 rows that a fragment read touches fall
// into the 16 different 16-byte slots of the 64 banks.
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

// 16 or 4 bytes of each lane, at base + voff, to LDS at lds + 16 (4) lane: `rsrc` as make_rsrc gives it.
__device__ __forceinline__ void load_lds16(i32x4 rsrc, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc)
               : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(i32x4 rsrc, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc)
               : "memory", "m0");
}
// A buffer from `base` (the same in all lanes) on: everything, or (live false) an empty range, whose
// loads give zeros.
__device__ __forceinline__ i32x4 make_rsrc(const void* base, bool live) {
  const uint64_t b = (uint64_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)b);
  r[1] = __builtin_amdgcn_readfirstlane((int)((b >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane(live ? -1 : 0);
  r[3] = 0x00020000;
  // (a vector instruction's scalar result needs 5 cycles before a load reads it; the compiler keeps
  // them for its own loads only)
  asm volatile("s_nop 4" ::"s"(r));
  return r;
}
__device__ __forceinline__ unsigned lds_offset(const void* p) {
  return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

// TM x TN tiles of 16 x 16 per wave, WR x WC waves, NS stages.
template <class MODE, int TM_, int TN_, int WR_, int WC_, int NS_ = 2>
struct TileShape {
  using Mode = MODE;
  static constexpr int NS = NS_;
  static constexpr int TM = TM_, TN = TN_, WR = WR_, WC = WC_;
  static constexpr int R = TM == 4 && TN == 4 && !std::is_same<MODE, Split>::value ? 4 : 2;   // see tile_row
  static constexpr int BM = 16 * TM * WR, BN = 16 * TN * WC, NT = 64 * WR * WC;
  static constexpr int kStage = (BM + BN) * 128;   // bytes of one stage
  static constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;   // 16-byte pieces per thread
  static_assert(TM % 2 == 0 && TN % 2 == 0, "tiles in pairs");
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole pieces per thread");
};

// Tile t, index a (0..15) of a wave's 16 T rows <-> row: the rows of R tiles are mixed so that a lane's
// results of them are 4 R neighbours, (a / 4) 4 R + 4 (t % R) + a % 4, the next R tiles 16 R rows on.
// R = 2: the 4 lanes of a row write 64 bytes of 16-bit results with each store; R = 4: each lane 32
// neighbouring bytes with two. Measured both ways: 8 x 8 tiles of 8-bit products (8192 x 8192 x 8192) 534 us with
// 2, 567 with 8; 4 x 4 tiles (2^18 rows through 256 x 256) 65 us with 2, 62 with 4; the FP16-split
// ones 832 us with 2, 863 with 4 (32 matrices of 512 x 1024).
template <int R>
__device__ __forceinline__ constexpr int tile_row(int t, int a) {
  return (t / R) * 16 * R + (a >> 2) * 4 * R + (t % R) * 4 + (a & 3);
}
template <int R>
__device__ __forceinline__ constexpr int swz(int r) {
  return ((r / (4 * R)) & 3) * 2 + ((r >> 1) & 1);
}

template <class S>
struct TileProduct {
  static constexpr int TM = S::TM, TN = S::TN, R = S::R;
  f32x4 acc[TM][TN];
  const char* a0;          // the tile's first rows
  const char* b0;
  unsigned va[S::LA];      // this thread's pieces: byte offsets from them
  unsigned vb[S::LB];

  // Rows m0 .. (below M) of A and n0 .. (below N) of B; rows behind the last one read the last one
  // again (their results are not stored). lda, ldb: bytes, 2^24 at most.
  __device__ __forceinline__ void init(const char* A, int64_t lda, int64_t m0, int64_t M, const char* B,
                                       int64_t ldb, int64_t n0, int64_t N) {
    const int am = (int)(M - 1 - m0 < S::BM ? M - 1 - m0 : S::BM);
    init_rows(A + m0 * lda, (unsigned)lda, [&](int r) { return (unsigned)(r < am ? r : am); }, B, ldb, n0, N);
  }
  // Tile row r of A is row row(r) from `base` on (below 4 GiB).
  template <class ROW>
  __device__ __forceinline__ void init_rows(const char* base, unsigned lda, ROW row, const char* B, int64_t ldb, int64_t n0,
                                            int64_t N) {
    a0 = (const char*)uniform((int64_t)base);
#pragma unroll
    for (int i = 0; i < S::LA; ++i) {
      const int idx = i * S::NT + (int)threadIdx.x, r = idx >> 3, p = (idx & 7) ^ swz<R>(r);
      va[i] = row(r) * lda + p * 16;
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
      const int idx = i * S::NT + t, r = idx >> 3, p = (idx & 7) ^ swz<R>(r);
      vb[i] = (unsigned)(r < bm ? r : bm) * (unsigned)ldb + p * 16;
    }
  }

  // The loads of chunk k of both operands into a stage, S::LA + S::LB in each wave, one at a time.
  // `live` false: nothing is read (an empty range: zeros arrive), so that a loop's last steps need no
  // branch around their loads; wait for them all the same before the LDS is used again or the wave ends.
  struct Loads {
    i32x4 ra, rb;
    unsigned at;
  };
  __device__ __forceinline__ Loads loads(char* stage, int k, bool live) const {
    Loads l;
    l.at = lds_offset(stage) + (unsigned)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024u;
    l.ra = make_rsrc(a0 + (int64_t)k * 128, live);
    l.rb = make_rsrc(b0 + (int64_t)k * 128, live);
    return l;
  }
  __device__ __forceinline__ void load_one(const Loads& l, int q) const {
    if (q < S::LA) load_lds16(l.ra, va[q < S::LA ? q : 0], l.at + q * S::NT * 16);
    else if (q < S::LA + S::LB) load_lds16(l.rb, vb[q < S::LA ? 0 : q - S::LA], l.at + S::BM * 128 + (q - S::LA) * S::NT * 16);
  }
  // Chunk k of B alone, at once.
  __device__ __forceinline__ void load_n(char* to, int k) const {
    const Loads l = loads(to - S::BM * 128, k, true);
#pragma unroll
    for (int q = 0; q < S::LB; ++q) load_one(l, S::LA + q);
  }

  struct Frags {
    i32x4 m[TM][2], n[TN][2];
  };
  // N tile d and M tile d of a chunk.
  __device__ __forceinline__ void read(Frags& f, const char* sa, const char* sb, int d) const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, a = lane & 15;
    if (d < TN) {
      const int r = (w % S::WC) * 16 * TN + tile_row<R>(d, a);
      f.n[d][0] = *(const i32x4*)(sb + r * 128 + ((g ^ swz<R>(r)) << 4));
      f.n[d][1] = *(const i32x4*)(sb + r * 128 + (((g + 4) ^ swz<R>(r)) << 4));
    }
    if (d < TM) {
      const int r = (w / S::WC) * 16 * TM + tile_row<R>(d, a);
      f.m[d][0] = *(const i32x4*)(sa + r * 128 + ((g ^ swz<R>(r)) << 4));
      f.m[d][1] = *(const i32x4*)(sa + r * 128 + (((g + 4) ^ swz<R>(r)) << 4));
    }
  }

  static __device__ __forceinline__ i32x8 join(const i32x4* p) {
    return __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // One chunk's products, from its rows in LDS, in growing squares (tiles i, j <= d), with part(0) ..
  // part(parts - 1), the next chunks' loads, along the way.
  // Large wave tiles (one wave on a SIMD): the operands of square d + 2 are read ahead of square d, so
  // that the first products wait for the first operands only, and the loads are spread evenly (issued
  // together they hold up the wave for as long as the memory path takes their addresses). Small ones:
  // other workgroups cover all that, and the loads are wanted early. 8192 x 8192 x 8192 in 8 bits with
  // 8 x 8 tiles a wave: 484 us spread, 549 together; 32768 rows of 2048 over 32 experts with 4 x 4: 246 and 226.
  template <class F, class P>
  __device__ __forceinline__ void squares(const char* sa, const char* sb, F f, int parts, P part) {
    constexpr int D = TM > TN ? TM : TN;
    constexpr bool kLarge = TM * TN > 16;
    Frags x;
    int done = 0, at = 0;
    if (!kLarge) {
#pragma unroll
      for (; at < parts; ++at) part(at);
    }
    auto one = [&](int i, int j) {
      f(x, i, j);
      ++done;
      bool any = false;
#pragma unroll
      for (; at * TM * TN < done * parts; ++at) {
        part(at);
        any = true;
      }
      if (any) __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int d = 0; d < (kLarge ? 2 : D); ++d) read(x, sa, sb, d);
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (kLarge) {
        if (d + 2 < D) read(x, sa, sb, d + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (j < d && d < TM) one(d, j);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i <= d && d < TN) one(i, d);
    }
  }

  // Fp8, Fp8Wide: word[i] >> shift / sn: the rows' scales in the lowest byte (E8M0).
  template <class P>
  __device__ __forceinline__ void chunk(const char* sa, const char* sb, const int (&word)[TM], int shift, int sn, int parts,
                                        P part) {
    squares(sa, sb, [&](const Frags& f, int i, int j) {
      const int sm = (int)((unsigned)word[i] >> shift);
      if constexpr (std::is_same<typename S::Mode, Fp8Wide>::value)
        acc[i][j] = wide_block(join(f.n[j]), join(f.m[i]), sn & 255, sm & 255, acc[i][j]);
      else
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(f.n[j]), join(f.m[i]), acc[i][j], 0, 0, 0,
                                                                     sn, 0, sm);
    }, parts, part);
  }

  template <class P>
  __device__ __forceinline__ void chunk(const char* sa, const char* sb, int parts, P part) {
    squares(sa, sb, [&](const Frags& f, int i, int j) {
      const f16x8 mh = __builtin_bit_cast(f16x8, f.m[i][0]), ml = __builtin_bit_cast(f16x8, f.m[i][1]);
      const f16x8 nh = __builtin_bit_cast(f16x8, f.n[j][0]), nl = __builtin_bit_cast(f16x8, f.n[j][1]);
      f32x4 c = acc[i][j];
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nh, mh, c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nl, mh, c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nh, ml, c, 0, 0, 0);
      acc[i][j] = c;
    }, parts, part);
  }

  // This lane's results within the workgroup's tile: tile i's are of row m(i); columns n(h) .. n(h) + 8 are
  // acc[i][2 h][0 .. 4], acc[i][2 h + 1][0 .. 4].
  __device__ __forceinline__ int m(int i) const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    return (w / S::WC) * 16 * TM + tile_row<R>(i, lane & 15);
  }
  __device__ __forceinline__ int n(int h) const {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    return (w % S::WC) * 16 * TN + (h / (R / 2)) * 16 * R + (lane >> 4) * 4 * R + h % (R / 2) * 8;
  }
};

// Every wave's loads but the last LEFT have landed, its LDS accesses are done, and every wave is here.
template <int LEFT = 0>
__device__ __forceinline__ void stage_ready() {
  static_assert(LEFT < 64, "the counter's range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(LEFT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The steps k = 0 .. n of a product over S::NS stages. plan(k): what the loads of chunk k into stage
// k % NS need (nothing that counts behind the last chunk); load(plan, q): one of them, q = 0 .. kLoads - 1 in
// each wave; chunk(k, part): its products, with part(0) .. part(kLoads - 1) between them. before(k) runs
// ahead of the barrier behind which chunk k is in LDS; started() when the first stages' loads are on their way.
template <class S, int kLoads, class PLAN, class LOAD, class CHUNK, class BEFORE, class STARTED>
__device__ __forceinline__ void tile_steps(int n, PLAN plan, LOAD load, CHUNK chunk, BEFORE before, STARTED started) {
  constexpr int NS = S::NS;
#pragma unroll
  for (int k = 0; k < NS - 1; ++k) {
    const auto l = plan(k);
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load(l, q);
  }
  started();
  for (int k = 0; k < n; ++k) {
    before(k);
    const auto l = plan(k + NS - 1);
    stage_ready<(NS - 2) * kLoads>();
    chunk(k, [&](int q) { load(l, q); });
  }
  stage_ready();   // (nothing is on its way into LDS any more)
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
