// Linear layers over a few rows with 4-bit weights (gfx950): y = act(x) W^T +
// bias for x [M <= 16, K <= 4096], W = e2m1 code * bf16 scale of its group of 32,
// 64 or 128 columns: the timestep MLPs' linears with a quarter of the bytes.
//
// Bound by the read of W, once: 50 MB of codes and 6 MB of scales (groups of
// 32) for 4096 -> 24576.  Vector products (one conversion per two weights, then
// a dot product per row of x) would pass the read's time from about 4 rows on, so
// the products run on the bf16 matrix cores, whose tile of 16 rows costs the
// same for 1 row and for 16: a code is exact in bf16, v_cvt_scalef32_pk_bf16_fp4
// makes two per instruction, and one v_mfma_f32_16x16x32_bf16 multiplies 16 rows
// of W with all rows of x over the 32 columns of one group (w is the second
// operand: a lane's four results all belong to one row of W, so the group's
// scale is one float32 FMA each, unrounded).  The packed order puts what a wave
// reads for 16 rows and 128 columns into one contiguous kilobyte, a lane's 16 bytes
// holding its 8 columns of four blocks of 32 (codes row after row, 64 bytes of 16
// rows per load, reached 3.7 TB/s over long weights).  Rows of x that do not exist
// repeat the last one: their results are not stored.
//
// A workgroup has 8 waves: KS of them share a tile of 16 rows of W, each with up
// to 4 chunks of 128 columns in flight, and meet in LDS; 8 / KS tiles at a time.
// x is staged in LDS once per workgroup, which then strides over the tiles.  SiLU(x)
// is held to 2^-16 as two rows of the matrix cores' 16: its bf16 and the bf16 of what
// that leaves, whose sums meet in the epilogue.  (Rounded to bf16 once it would add
// as much error again as the result's own rounding.)  That costs no products up to 8
// rows; more go by halves, two workgroups of one XCD over the same tiles, so that the
// second read of W comes from their L2 (16 rows of 4096 -> 24576: 25.7 us; rounded
// once 20.8).  2 rows of 4096 -> 24576 with groups of 32 and SiLU: 13.8 us (4.1 TB/s
// of 57 MB; 5.5 TB/s at the end of longer weights), 8 rows of 2048 -> 12288 with groups
// of 128: 7.5 us, of which computing SiLU(x) in every workgroup takes about 1.

#include <type_traits>

#include "ltx_common.h"

namespace ltx {

constexpr int kG4Waves = 8, kG4Chunks = 4;

typedef __bf16 g4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float g4_f4 __attribute__((ext_vector_type(4)));

struct Group4Args {
  const uint16_t* x;
  int64_t x_ls;
  const uint8_t* codes;
  const uint16_t* scales;
  const uint16_t* bias;  // null: none
  uint16_t* y;
  int64_t y_ls;
  int64_t N;
  int M, K;
};

// SiLU through one exp2 and one reciprocal (1 ulp each).
__device__ __forceinline__ float g4_silu(float v) {
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// 8 codes (lower half of byte 0 first) as bf16.
__device__ __forceinline__ g4_bf16x8 g4_decode(uint32_t w) {
  const ltx_bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0);
  const ltx_bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1);
  const ltx_bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2);
  const ltx_bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3);
  const auto ab = __builtin_shufflevector(a, b, 0, 1, 2, 3), cd = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(ab, cd, 0, 1, 2, 3, 4, 5, 6, 7);
}

// KS waves per tile, GROUP columns per scale.  With SILU, rows 4 i + 2 h + l of the
// matrix cores' 16 (h, l of {0, 1}) are part h of row 2 i + l of x: a lane has both sums.
template <int KS, int GROUP, bool SILU>
__global__ void __launch_bounds__(64 * kG4Waves) group4_linear_kernel(const Group4Args a) {
  constexpr int kTiles = kG4Waves / KS, kPer = 128 / GROUP;  // tiles per workgroup; scales per chunk and row
  extern __shared__ uint4 xs[];                              // [M, with SiLU 2 M][chunks * 16 + 1]
  __shared__ float part[2][kG4Waves][SILU ? 8 : 16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, p = lane >> 4, kw = wave % KS;
  const int chunks = (a.K + 127) / 128, row_words = chunks * 16 + 1;
  const int64_t tiles = (a.N + 15) / 16;
  const int own = (chunks + KS - 1) / KS, c0 = kw * own, c1 = min(c0 + own, chunks);  // this wave's chunks

  // One tile's rows of W in registers: 4 chunks of codes and their scales.  Every
  // load of a round is unconditional (a wave with fewer chunks reads its last one
  // again, one without a tile the last tile): loads that may not have been issued
  // would make the waits for older ones wait for all.
  struct Rows {
    uint4 w[kG4Chunks];
    uint16_t s[kG4Chunks][kPer];
  };
  auto load = [&](Rows& t, int64_t tile) {
    const int64_t at = (tile < tiles ? tile : tiles - 1) * chunks;
#pragma unroll
    for (int i = 0; i < kG4Chunks; ++i) {
      const int64_t c = at + max(min(c0 + i, c1 - 1), 0);
      t.w[i] = *reinterpret_cast<const uint4*>(a.codes + c * 1024 + lane * 16);
      __builtin_memcpy(t.s[i], __builtin_assume_aligned(a.scales + (c * 16 + r16) * kPer, kPer * 2), sizeof(t.s[i]));
    }
  };
  int m_first = 0, M = a.M, block = blockIdx.x, blocks = gridDim.x;
  if (SILU && a.M > 8) {  // halves of the rows: workgroups 8 apart, of one XCD
    const int per = (a.M + 1) >> 1;
    m_first = block & 8 ? per : 0;
    M = min(a.M - m_first, per);
    block = (block >> 4) * 8 + (block & 7);
    blocks >>= 1;
  }
  const uint16_t* x = a.x + m_first * a.x_ls;
  const int64_t stride = (int64_t)blocks * kTiles, first = (int64_t)block * kTiles;
  const int64_t tile = first + wave / KS;
  const int64_t rounds = (tiles - first + stride - 1) / stride;
  Rows rows[2];

  // x: a thread keeps its column, rows go by in fours.  Loads return in order, so
  // the last of them are issued ahead of the first rows of W, which then travel
  // while x is staged.
  const int words = chunks * 16, xrows = 64 * kG4Waves / words;
  const int xm = threadIdx.x / words, xc = threadIdx.x - xm * words;
  for (int m0 = 0; m0 < M; m0 += 4 * xrows) {
    uint4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = m0 + q * xrows + xm;
      v[q] = make_uint4(0, 0, 0, 0);  // columns past K: their codes are 0, so x must be finite there
      if (xm < xrows && m < M && xc * 8 < a.K) v[q] = *reinterpret_cast<const uint4*>(x + m * a.x_ls + xc * 8);
    }
    if (m0 + 4 * xrows >= M) {
      load(rows[0], tile);
      if (rounds > 1) load(rows[1], tile + stride);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = m0 + q * xrows + xm;
      if (xm >= xrows || m >= M) break;
      if constexpr (SILU) {
        uint4 rest;
        uint32_t *t = &v[q].x, *d = &rest.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo = g4_silu(bf16_bits_to_f32(t[e] & 0xFFFFu)), hi = g4_silu(bf16_bits_to_f32(t[e] >> 16));
          t[e] = pack_bf16x2(lo, hi);
          const float blo = bf16_bits_to_f32(t[e] & 0xFFFFu), bhi = bf16_bits_to_f32(t[e] >> 16);
          d[e] = pack_bf16x2(lo == blo ? 0.0f : lo - blo, hi == bhi ? 0.0f : hi - bhi);  // infinity leaves nothing
        }
        xs[(M + m) * row_words + xc] = rest;
      }
      xs[m * row_words + xc] = v[q];
    }
  }
  __syncthreads();
  const int xrow = SILU ? (r16 >> 1 & 1) * M + min((r16 >> 2) * 2 + (r16 & 1), M - 1) : min(r16, M - 1);
  const uint4* xr = xs + xrow * row_words + p;

  // the result that this thread stores in a round: row ym of x, column yc of tile yt
  const int yt = threadIdx.x >> 8, ym = (threadIdx.x >> 4) & 15, yc = threadIdx.x & 15;
  auto round = [&](Rows& t, int64_t r, auto prefetch) {
    const int64_t t0 = first + r * stride;
    float bias[(kTiles + 1) / 2] = {};
#pragma unroll
    for (int h = 0; h < (kTiles + 1) / 2; ++h) {
      const int64_t n = (t0 + h * 2 + yt) * 16 + yc;
      if (a.bias != nullptr) bias[h] = bf16_bits_to_f32(a.bias[n < a.N ? n : a.N - 1]);
    }
    g4_f4 acc = {};
#pragma unroll
    for (int i = 0; i < kG4Chunks; ++i) {
      const int c = c0 + i;
      if (c < c1) {
        const uint32_t* wp = &t.w[i].x;
        g4_f4 d = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const g4_bf16x8 xv = __builtin_bit_cast(g4_bf16x8, xr[c * 16 + j * 4]);
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, g4_decode(wp[j]), d, 0, 0, 0);
          if ((j + 1) * 32 % GROUP == 0) {
            const float sc = bf16_bits_to_f32(t.s[i][j * 32 / GROUP]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(d[e], sc, acc[e]);
            d = g4_f4{};
          }
        }
      }
    }
    if (prefetch) load(t, tile + (r + 2) * stride);
    // lane: rows 4 p .. + 3 of x (with SILU 2 p and 2 p + 1), row r16 of the tile
    const int buf = (int)(r & 1);
    constexpr int kOwn = SILU ? 2 : 4;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) part[buf][wave][p * kOwn + e][r16] = SILU ? acc[e] + acc[e + 4 - kOwn] : acc[e];
    __syncthreads();  // the other buffer's sums, read a round ago, may be overwritten after it
#pragma unroll
    for (int h = 0; h < (kTiles + 1) / 2; ++h) {
      const int tw = h * 2 + yt;
      const int64_t n = (t0 + tw) * 16 + yc;
      if (tw < kTiles && ym < M && n < a.N) {
        float v = bias[h];
#pragma unroll
        for (int k = 0; k < KS; ++k) v += part[buf][tw * KS + k][ym][yc];
        a.y[(m_first + ym) * a.y_ls + n] = f32_to_bf16_bits(v);
      }
    }
  };
  // every wave of a workgroup runs the same rounds; one without a tile adds to no stored result
  const std::true_type more;
  const std::false_type last;
  int64_t r = 0;
  for (; r + 3 < rounds; r += 2) {
    round(rows[0], r, more);
    round(rows[1], r + 1, more);
  }
  if (r + 2 < rounds) {
    round(rows[0], r, more);
    round(rows[1], r + 1, last);
    round(rows[0], r + 2, last);
  } else {
    round(rows[0], r, last);
    if (r + 1 < rounds) round(rows[1], r + 1, last);
  }
}

template <int KS, int GROUP, bool SILU>
void launch_group4(const Group4Args& a, hipStream_t st) {
  const int chunks = (a.K + 127) / 128;
  const size_t lds = (size_t)(!SILU ? a.M : a.M > 8 ? a.M + 1 : 2 * a.M) * (chunks * 16 + 1) * 16;
  const size_t all = lds + sizeof(float) * 2 * kG4Waves * (SILU ? 8 : 16) * 17;
  // Resident workgroups per CU: two (16 waves) where the LDS holds them (weights from HBM,
  // groups of 128, SiLU: 4 rows of 4096 -> 24576 in 15.8 us, one 17.9); two that do not fit take turns
  // and stage x twice (8 rows of it 23.6, one 19.4).  One also where SiLU of a large x is what a
  // workgroup does most and two would have no more than a round each: 8 rows of 2048 -> 12288
  // in 8.1, two 8.6; 7 rows 7.7 and 8.1.  Not without SiLU (8 rows 7.1, two 6.8), nor by halves
  // (12 rows of 2048 -> 16384 10.5, two 10.0), nor for longer weights (7 rows of 2048 -> 24576
  // 10.6, two 10.4).
  const int64_t want = ceil_div(ceil_div(a.N, 16), kG4Waves / KS);
  const bool one = all > 80 * 1024 || (SILU && a.M <= 8 && all > 48 * 1024 && want <= 512);
  const int64_t most = one ? 256 : 512;
  int64_t grid = want < most ? want : most;
  if (SILU && a.M > 8) grid = 2 * (want < most / 2 ? ceil_div(want, 8) * 8 : most / 2);  // whole groups of 8, 8 apart
  hipLaunchKernelGGL((group4_linear_kernel<KS, GROUP, SILU>), dim3((unsigned)grid), dim3(64 * kG4Waves), lds, st, a);
}

template <int GROUP, bool SILU>
void launch_group4(const Group4Args& a, hipStream_t st) {
  // as few waves per tile as hold its columns in flight (4 chunks of 128 each)
  const int chunks = (a.K + 127) / 128;
  if (chunks <= kG4Chunks)
    launch_group4<1, GROUP, SILU>(a, st);
  else if (chunks <= 2 * kG4Chunks)
    launch_group4<2, GROUP, SILU>(a, st);
  else if (chunks <= 4 * kG4Chunks)
    launch_group4<4, GROUP, SILU>(a, st);
  else
    launch_group4<8, GROUP, SILU>(a, st);
}
static_assert(LTX_SKINNY_MAX_K <= 8 * kG4Chunks * 128, "8 waves hold a row of W");

}  // namespace ltx

using namespace ltx;

extern "C" int ltx_group4_linear(int64_t M, int64_t N, int64_t K, int64_t group, const void* x, int64_t x_ls,
                                 int silu, const void* codes, const void* scales, const void* bias, void* y,
                                 int64_t y_ls, void* stream) {
  clear_error();
  LTX_REQUIRE(M >= 0 && M <= LTX_GROUP4_MAX_ROWS, "ltx_group4_linear: M must be at most %d", LTX_GROUP4_MAX_ROWS);
  LTX_REQUIRE(group == 32 || group == 64 || group == 128, "ltx_group4_linear: group must be 32, 64 or 128");
  LTX_REQUIRE(K >= group && K <= LTX_SKINNY_MAX_K && K % group == 0,
              "ltx_group4_linear: K must be a multiple of the group, at most %d", LTX_SKINNY_MAX_K);
  LTX_REQUIRE(N >= 0 && N <= 0x7FFFFFFF, "ltx_group4_linear: bad N");
  if (M * N == 0) return LTX_OK;
  LTX_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr && y != nullptr,
              "ltx_group4_linear: null pointer");
  LTX_REQUIRE((uintptr_t)x % 16 == 0 && x_ls % 8 == 0 && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 8 == 0,
              "ltx_group4_linear: x rows and codes must be 16-byte aligned, scales 8-byte");
  LTX_REQUIRE(M == 1 || y_ls >= N, "ltx_group4_linear: rows of y overlap");
  Group4Args a{(const uint16_t*)x, x_ls, (const uint8_t*)codes, (const uint16_t*)scales, (const uint16_t*)bias,
               (uint16_t*)y, y_ls, N, (int)M, (int)K};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (group == 32)
    silu ? launch_group4<32, true>(a, st) : launch_group4<32, false>(a, st);
  else if (group == 64)
    silu ? launch_group4<64, true>(a, st) : launch_group4<64, false>(a, st);
  else
    silu ? launch_group4<128, true>(a, st) : launch_group4<128, false>(a, st);
  LTX_LAUNCH_CHECK("ltx_group4_linear");
  return LTX_OK;
}
