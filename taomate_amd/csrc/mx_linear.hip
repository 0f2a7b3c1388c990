// Linear layers of 8-bit rows with 8-bit weights (gfx950): y = act(a w^T + bias)
// on the scaled matrix cores (v_mfma_scale_f32_16x16x128_f8f6f4).
//
// One MFMA takes 16 rows of w and 16 rows of a over 128 columns, every lane
// with the E8M0 scale of one row's block of 32, and adds 16 x 16 products into
// float32 accumulators at the rate of unscaled e4m3: the block scales cost no
// vector work.  Its operands, as measured: lane l holds row l % 16, columns
// 16 (l / 16) .. + 15 in its first 16 bytes and 64 more in its second, and the
// scale of block l / 16 (columns 32 (l / 16) .. + 31) of that row.  The result's
// lane l holds, for row l % 16 of the second operand, rows 4 (l / 16) .. + 3 of the
// first: w is the first operand, so that a lane ends with neighbouring outputs
// of one row of y.
//
// The instruction adds the products of up to 8 neighbouring columns after shifting them
// to the largest and keeps 13 bits below it; all further sums are float32.  So a sum
// may be off by 7 * 2^-13 of its products' magnitudes.  In sums that do not cancel
// that stays under the rounding of either result (bf16 2^-8, e4m3 2^-4); in one that
// does it can be all of it: neighbouring products 1, -1, 2^-14 give 0.  It is taken
// because the operands themselves are rounded to 2^-4 and the results to 2^-8 or 2^-4, and
// because every product at this rate has it: the library's fp8 products cut at the same
// bit (1.3e-5 of a result's norm for normal operands).  Of the 8-bit results of real sizes 0.2 %
// of the codes become their neighbour, and the error against results that are not
// rounded is 0.02645 of their norm with the cut and without.
//
// Large sizes: 8192 x 8192 x 8192 in 371-400 us by box (2.75-2.96 PFLOP/s of 5.0; the matrix
// cores busy 75-81 % of the cycles), 2304 x 4096 -> 16384 with GELU and an 8-bit result in
// 126-143 us, 2304 x 16384 -> 4096 in 122-147 (busy 74 % of the cycles of the CUs with a tile).  The
// loop loses what the two waves of a SIMD do not hide of its loads and LDS reads:
// 2304 x 16384 -> 4096 takes 123 us, without the loads 98, without the reads 104, without
// either 93 (8192^3 371, 335, 341 and 306).  Where the chip is full of tiles for long, power
// comes on top: 1.63-1.74 GHz at 8192^3, 2.0-2.1 at the others.  By the weight's read at few rows
// (2 of 4096 -> 16384: 12.7 us, 5.4 TB/s), between them by latency.
//
// Tiles of a and w travel HBM -> LDS without registers, 128 columns (one MFMA's
// depth) per step, in rows of 128 bytes whose 16-byte chunks are exchanged by
// chunk ^= (row / 2) % 8: the 16 rows that a fragment read touches then lie in
// 16 different 16-byte columns of the LDS.  Tile t of a wave's w rows holds the
// channels 4 NT i + 4 t + r (i, r in [0, 4)) in its rows 4 i + r, so that lane
// group i ends with the 4 NT neighbouring channels 4 NT i ..: contiguous stores,
// and blocks of 32 for an 8-bit result inside a pair of lanes (NT = 4) or four (NT = 2).

#include <math.h>

#include <type_traits>

#include "mx_common.h"

namespace ltx {

typedef int mx_i4 __attribute__((ext_vector_type(4)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
#define MX_LDS __attribute__((address_space(3)))
typedef MX_LDS void* mx_lds_ptr;
// 16 (4) bytes per lane from a buffer's offset straight into LDS: lane l's land at `to` + 16 l (4 l).
__device__ __forceinline__ void mx_lds_load16(__amdgpu_buffer_rsrc_t r, uint32_t to, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (mx_lds_ptr)(uintptr_t)to, 16, offset, 0, 0, 0);
}
__device__ __forceinline__ void mx_lds_load4(__amdgpu_buffer_rsrc_t r, uint32_t to, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (mx_lds_ptr)(uintptr_t)to, 4, offset, 0, 0, 0);
}
// The byte column that lane l of a load of 8 rows from `row` on reads: its chunk, exchanged.
__device__ __forceinline__ int mx_chunk(int l, int row) { return ((l & 7) ^ (((row + (l >> 3)) >> 1) & 7)) * 16; }
__device__ __forceinline__ const MX_LDS uint8_t* mx_lds(uint32_t at) { return (const MX_LDS uint8_t*)(uintptr_t)at; }
// A lane's 32 bytes of a fragment: 16 of the row's first 64, 16 of its last.
__device__ __forceinline__ mx_i8 mx_fragment(const MX_LDS uint8_t* lo, const MX_LDS uint8_t* hi) {
  const mx_i4 x = *(const MX_LDS mx_i4*)lo, y = *(const MX_LDS mx_i4*)hi;
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ mx_i8 mx_fragment(__amdgpu_buffer_rsrc_t r, int lo, int hi) {
  const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, lo, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b128(r, hi, 0, 0);
  return __builtin_shufflevector(__builtin_bit_cast(mx_i4, x), __builtin_bit_cast(mx_i4, y), 0, 1, 2, 3, 4, 5, 6, 7);
}

struct MxLinearArgs {
  const uint8_t* a;
  const uint8_t* as;
  const uint8_t* w;
  const uint8_t* ws;
  const uint16_t* bias;  // null: none
  void* y;
  uint8_t* ys;           // null: y is bf16
  int64_t y_ls;
  int M, N, K;
};

// tanh-GELU: y sigmoid(2 u), u = sqrt(2 / pi) (y + 0.044715 y^3).  The sigmoid
// through one exp2 and one reciprocal (1 ulp each).
__device__ __forceinline__ float mx_gelu(float y) {
  const float c = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  const float u = y * fmaf(y * y, 0.044715f * c, c);
  return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u));
}

constexpr int kGroupM = 4;

// MT x NT tiles of 16 x 16 per wave, WM x WN waves per group, ST buffers of one step each,
// KG groups that split the columns of K and meet at the end.
template <int MT, int NT, int WM, int WN, int ST, int KG>
struct MxTile {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves * KG;  // waves of a group
  static constexpr int kBM = 16 * MT * WM, kBN = 16 * NT * WN, kRows = kBM + kBN;
  static constexpr int kARows = (kBM + 63) / 64 * 64, kWRows = (kBN + 63) / 64 * 64;  // of scales: whole loads
  static constexpr int kCodes = kRows * 128, kStage = kCodes + (kARows + kWRows) * 4;
  // 1 KB loads (8 rows) per step and wave, of each operand
  static constexpr int kPerA = (kBM / 8 + kWaves - 1) / kWaves, kPerW = (kBN / 8 + kWaves - 1) / kWaves;
  static constexpr int kScaleLoads = (kARows + kWRows) / 64;     // 256 byte loads (64 rows' words) per step
  static constexpr int kScalePer = (kScaleLoads + kWaves - 1) / kWaves, kParts = kPerA + kPerW + kScalePer;
  static_assert(KG == 1 || kWaves * MT * NT * 1024 <= ST * kStage, "LDS");
  static_assert(ST >= 2 && KG * ST * kStage <= 160 * 1024, "LDS");
};

template <int MT, int NT, int WM, int WN, int ST, int KG, bool GELU>
__global__ void __launch_bounds__(64 * WM * WN * KG, 2) mx_linear_kernel(const MxLinearArgs p) {
  using T = MxTile<MT, NT, WM, WN, ST, KG>;
  __shared__ __attribute__((aligned(128))) uint8_t lds[KG * ST * T::kStage];
  const int lane = threadIdx.x & 63, wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_of_all % T::kWaves, kg = wave_of_all / T::kWaves;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mx_lds_ptr)lds + kg * ST * T::kStage;
  const int wm = wave % WM, wn = wave / WM;
  const int g = lane >> 4, r16 = lane & 15;
  // Workgroups go round-robin to the 8 XCDs: each gets a contiguous run of tiles, walked in
  // groups of kGroupM rows of tiles, so that those resident on one L2 share rows of a and w.
  const int tm = (p.M + T::kBM - 1) / T::kBM, tn = gridDim.x / tm;
  const int per = gridDim.x / 8, rem = gridDim.x % 8, xcd = blockIdx.x % 8;
  const int tile = xcd * per + min(xcd, rem) + blockIdx.x / 8;
  const int group = tile / (kGroupM * tn), in = tile - group * kGroupM * tn, gm = min(kGroupM, tm - group * kGroupM);
  const int m0 = __builtin_amdgcn_readfirstlane((group * kGroupM + in % gm) * T::kBM);
  const int n0 = __builtin_amdgcn_readfirstlane(in / gm * T::kBN);
  // A group's steps; the last group's end with K, and what the first ones have before column 0 reads as zeros.
  const int all = (p.K + 127) / 128, steps = (all + KG - 1) / KG, first = all - (KG - kg) * steps;

  // The channel of the tile that row r of its w rows holds.
  auto channel = [](int r) {
    const int s = r % (16 * NT);
    return r - s + (s % 16 / 4) * 4 * NT + (s / 16) * 4 + s % 4;
  };
  // This lane's part of the wave's loads: rows 8 j .. + 7 of load j, a chunk each
  const int mrows = min(p.M - m0, T::kBM), nrows = max(min(p.N - n0, T::kBN), 0);
  // (a wave whose part lies past an operand's loads repeats the last one: no branch).
  int aoff[T::kPerA], woff[T::kPerW];
#pragma unroll
  for (int q = 0; q < T::kPerA; ++q) aoff[q] = (min(q * T::kWaves + wave, T::kBM / 8 - 1) * 8 + (lane >> 3)) * p.K;
#pragma unroll
  for (int q = 0; q < T::kPerW; ++q)
    woff[q] = channel(min(q * T::kWaves + wave, T::kBN / 8 - 1) * 8 + (lane >> 3)) * p.K;
  int soff[T::kScalePer];
#pragma unroll
  for (int i = 0; i < T::kScalePer; ++i) {
    const int row = min(i * T::kWaves + wave, T::kScaleLoads - 1) * 64 + lane;
    soff[i] = (row < T::kARows ? row : channel(row - T::kARows)) * 4;
  }
  const uint8_t* abase = p.a + (int64_t)m0 * p.K;
  const uint8_t* wbase = p.w + (int64_t)n0 * p.K;
  const uint8_t* asbase = p.as + (int64_t)m0 * 4;
  const uint8_t* wsbase = p.ws + (int64_t)n0 * 4;

  // The loads of a step.  Their buffer descriptors end with the
  // tile's last row, so rows past M or N, columns past K (by their offset) and steps
  // past the last (by the descriptor) read as zeros: the loop issues them without a
  // branch.
  struct Step {
    uint32_t base;
    __amdgpu_buffer_rsrc_t a, w, as, ws;
    int left;
  };
  auto step = [&](int ks, int at) {
    Step r;
    r.base = lds0 + at;
    const int k0 = (first + ks) * 128, left = k0 < 0 || ks >= steps ? 0 : max(p.K - k0, 0);
    r.a = __builtin_amdgcn_make_buffer_rsrc((void*)(abase + k0), (short)0, left > 0 ? mrows * p.K - k0 : 0, 0x00020000);
    r.w = __builtin_amdgcn_make_buffer_rsrc((void*)(wbase + k0), (short)0, left > 0 ? max(nrows * p.K - k0, 0) : 0,
                                            0x00020000);
    r.as = __builtin_amdgcn_make_buffer_rsrc((void*)(asbase + (int64_t)(first + ks) * p.M * 4), (short)0,
                                             left > 0 ? mrows * 4 : 0, 0x00020000);
    r.ws = __builtin_amdgcn_make_buffer_rsrc((void*)(wsbase + (int64_t)(first + ks) * p.N * 4), (short)0,
                                             left > 0 ? nrows * 4 : 0, 0x00020000);
    r.left = left;
    return r;
  };
  auto issue_a = [&](const Step& r, int q) {
    const int j = min(q * T::kWaves + wave, T::kBM / 8 - 1), col = mx_chunk(lane, j * 8);
    mx_lds_load16(r.a, r.base + j * 1024, aoff[q] + col + (col < r.left ? 0 : 0x40000000));
  };
  auto issue_w = [&](const Step& r, int q) {
    const int j = min(q * T::kWaves + wave, T::kBN / 8 - 1), col = mx_chunk(lane, T::kBM + j * 8);
    mx_lds_load16(r.w, r.base + T::kBM * 128 + j * 1024, woff[q] + col + (col < r.left ? 0 : 0x40000000));
  };
  auto issue_scales = [&](const Step& r, int q) {
    const int j = min(q * T::kWaves + wave, T::kScaleLoads - 1);
    mx_lds_load4(j * 64 < T::kARows ? r.as : r.ws, r.base + T::kCodes + j * 256, soff[q]);
  };
  auto issue_all = [&](int ks) {
    const Step r = step(ks, ks * T::kStage);
#pragma unroll
    for (int q = 0; q < T::kPerW; ++q) issue_w(r, q);
#pragma unroll
    for (int q = 0; q < T::kPerA; ++q) issue_a(r, q);
#pragma unroll
    for (int q = 0; q < T::kScalePer; ++q) issue_scales(r, q);
  };

  // Fragments and their scales from a step's buffer: rows 16 apart share their chunk exchange.
  const int sx = (r16 >> 1) & 7;
  const uint32_t alo = lds0 + (wm * MT * 16 + r16) * 128 + (g ^ sx) * 16;
  const uint32_t wlo = lds0 + (T::kBM + wn * NT * 16 + r16) * 128 + (g ^ sx) * 16;
  const uint32_t asc = lds0 + T::kCodes + (wm * MT * 16 + r16) * 4 + g;
  const uint32_t wsc = lds0 + T::kCodes + (T::kARows + wn * NT * 16 + r16) * 4 + g;
  struct Buffer {
    const MX_LDS uint8_t *alo, *ahi, *wlo, *whi, *asc, *wsc;
  };
  auto buffer = [&](int at) {
    return Buffer{mx_lds(alo + at), mx_lds((alo + at) ^ 64), mx_lds(wlo + at), mx_lds((wlo + at) ^ 64),
                  mx_lds(asc + at), mx_lds(wsc + at)};
  };

  // One step of a wave.  The fragments of w are held.  The first H tiles of a are
  // multiplied column by column; after them every wave has its w in registers, and
  // the loads of the w of the step ST later go out into its place.  The middle tiles
  // go one by one, those after them read meanwhile.  When the last S are in
  // registers the waves meet: the next step's data have landed, a's place is free, and
  // the loads of the a of the step ST later go out.  The last S tiles go column by
  // column again, and each fragment of w, done after S products, is read for the
  // next step, as are its first H tiles of a: every read has several products to
  // arrive in, its own wave's and those of the SIMD's other wave, and w's loads,
  // which come from further away, more than a step.
  constexpr int H = MT > 3 ? 2 : 1, S = MT > 4 ? 3 : MT - H, kMid = MT - H - S;
  mx_f4 acc[MT][NT] = {};
  mx_i8 fw[NT], fa[MT];
  int sw[NT], sa[MT];
  // all but the latest `later` loads of this wave have landed, all its reads too
  auto meet = [&](auto later) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(later)::value) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto read_a = [&](const Buffer& b, int t, int mask) {
    fa[t] = mx_fragment(b.alo + t * 2048, b.ahi + t * 2048);
    sa[t] = b.asc[t * 64] & mask;
  };
  auto read_w = [&](const Buffer& b, int u, int mask) {
    fw[u] = mx_fragment(b.wlo + u * 2048, b.whi + u * 2048);
    sw[u] = b.wsc[u * 64] & mask;
  };
  auto product = [&](int t, int u) {
    acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u], fa[t], acc[t][u], 0, 0, 0, sw[u], 0, sa[t]);
  };
  auto first_tiles = [&](const Buffer& b, int mask, const Step* after) {
#pragma unroll
    for (int r = 0; r <= kMid; ++r) {
#pragma unroll
      for (int t = H + (r * (MT - H) + kMid) / (kMid + 1); t < H + ((r + 1) * (MT - H) + kMid) / (kMid + 1); ++t)
        read_a(b, t, mask);
      if (r == 0) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int t = 0; t < H; ++t) product(t, u);
      } else {
#pragma unroll
        for (int u = 0; u < NT; ++u) product(H + r - 1, u);
        if (after != nullptr)
#pragma unroll
          for (int q = (r - 1) * T::kPerW / max(kMid, 1); q < r * T::kPerW / max(kMid, 1); ++q) issue_w(*after, q);
      }
#pragma unroll
      for (int i = 0; i < NT * (r == 0 ? H : 1); ++i) {  // reads and loads between the products
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
        if (r == 0)
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        else
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (r == 0 && after != nullptr) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kMid == 0)
#pragma unroll
          for (int q = 0; q < T::kPerW; ++q) issue_w(*after, q);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < ST; ++i) issue_all(i);
  meet(std::integral_constant<int, (ST - 1) * T::kParts>{});
  {
    const Buffer b = buffer(0);
    const int live = first * 128 + g * 32 < p.K ? 0xFF : 0;  // the scale bytes of blocks past K are not looked at
#pragma unroll
    for (int t = 0; t < H; ++t) read_a(b, t, live);
#pragma unroll
    for (int u = 0; u < NT; ++u) read_w(b, u, live);
  }
  int at = 0;  // the step's buffer
  for (int ks = 0; ks + 1 < steps; ++ks) {
    const int next_at = at + T::kStage == ST * T::kStage ? 0 : at + T::kStage;
    const Step after = step(ks + ST, at);
    first_tiles(buffer(at), 0xFF, &after);
    __builtin_amdgcn_s_setprio(1);
    meet(std::integral_constant<int, (ST - 2) * T::kParts + T::kPerW>{});
    const Buffer next = buffer(next_at);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int t = MT - S; t < MT; ++t) product(t, u);
#pragma unroll
      for (int q = u * T::kPerA / NT; q < (u + 1) * T::kPerA / NT; ++q) issue_a(after, q);
      if (u == NT - 1)
#pragma unroll
        for (int q = 0; q < T::kScalePer; ++q) issue_scales(after, q);
      read_w(next, u, 0xFF);
      if (u < H) read_a(next, u, 0xFF);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    at = next_at;
  }
  // the bias travels during the last step, as pairs of bf16
  const int n = n0 + wn * 16 * NT + g * 4 * NT;
  uint32_t bias[2 * NT] = {};
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4 * NT; i += 8) {
      if (n + i + 8 <= p.N) {
        __builtin_memcpy(bias + i / 2, p.bias + n + i, 16);
      } else {
#pragma unroll
        for (int e = i; e < i + 8; ++e)
          if (n + e < p.N) bias[e / 2] |= (uint32_t)p.bias[n + e] << (16 * (e % 2));
      }
    }
  }
  const int live = (first + steps - 1) * 128 + g * 32 < p.K ? 0xFF : 0;
#pragma unroll
  for (int u = 0; u < NT; ++u) sw[u] &= live;
#pragma unroll
  for (int t = 0; t < H; ++t) sa[t] &= live;
  first_tiles(buffer(at), live, nullptr);
#pragma unroll
  for (int t = MT - S; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) product(t, u);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may land in the LDS of the next workgroup
  // The groups' sums meet in LDS; group kg takes every KG-th row of tiles from there on
  // (the first group alone: 10.7 us for 150 x 2048 -> 8192 with GELU, 9.3 so).
  mx_f4* const part = reinterpret_cast<mx_f4*>(lds) + lane;
  auto part_at = [&](int k, int t, int u) { return (((k * T::kWaves + wave) * MT + t) * NT + u) * 64; };
  if constexpr (KG > 1) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
      if (t % KG != kg)
#pragma unroll
        for (int u = 0; u < NT; ++u) part[part_at(kg, t, u)] = acc[t][u];
    __syncthreads();
  }

  // Epilogue: lane group g holds channels n .. n + 4 NT - 1 of row m for every tile row.
  // Channels past N are zeros (NaN beside one in a): they count in no block's maximum.
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (KG > 1 && t % KG != kg) continue;
#pragma unroll
    for (int k = 1; k < KG; ++k)
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[t][u] += part[part_at((t + k) % KG, t, u)];
    const int m = m0 + (wm * MT + t) * 16 + r16;
    float v[4 * NT];
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) {
      const uint32_t b = bias[i / 2];
      v[i] = acc[t][i / 4][i % 4] + __uint_as_float(i % 2 ? b & 0xFFFF0000u : b << 16);
      if (GELU) v[i] = mx_gelu(v[i]);
    }
    if (p.ys != nullptr) {
      static_assert(NT == 2 || NT == 4, "a block of 32 lies in two or four lanes");
      float top = mx_top(v);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      if (NT == 2) top = fmaxf(top, __shfl_xor(top, 32, 64));
      const uint32_t code = mx_scale_code(top);
      const float inv = mx_inverse(code);
      if (m < p.M) {
        uint8_t* yp = (uint8_t*)p.y + (int64_t)m * p.N + n;
        constexpr int kStore = NT == 2 ? 8 : 16;  // N is a multiple of 32, n one of 4 NT: whole stores
        uint32_t c[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i)
          c[i] = mx_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
#pragma unroll
        for (int i = 0; i < 4 * NT; i += kStore)
          if (n + i < p.N) __builtin_memcpy(__builtin_assume_aligned(yp + i, kStore), c + i / 4, kStore);
        // blocks past N up to the next 128 columns are written as 0
        if (n / 128 < (p.N + 127) / 128 && n % 32 == 0)
          p.ys[((int64_t)(n / 128) * p.M + m) * 4 + n / 32 % 4] = (uint8_t)code;
      }
    } else if (m < p.M) {
      uint16_t* yp = (uint16_t*)p.y + (int64_t)m * p.y_ls + n;
#pragma unroll
      for (int i = 0; i < 4 * NT; i += 8) {
        if (n + i + 8 <= p.N) {
          const uint4 w = make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                                     pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
          // one store, also where the row is aligned to 2 bytes only (331 x 1056 -> 4099: 9.0 us; by 2 bytes 11.3)
          __builtin_memcpy(yp + i, &w, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + i + e < p.N) yp[i + e] = f32_to_bf16_bits(v[i + e]);
        }
      }
    }
  }
}

template <int MT, int NT, int WM, int WN, int ST, int KG, bool GELU>
void launch_mx_linear(const MxLinearArgs& p, hipStream_t st) {
  using T = MxTile<MT, NT, WM, WN, ST, KG>;
  // an 8-bit result's scales are written up to the next 128 columns
  const int64_t cols = p.ys != nullptr ? ceil_div(p.N, 128) * 128 : p.N;
  const dim3 grid((unsigned)(ceil_div(cols, T::kBN) * ceil_div(p.M, T::kBM)));
  hipLaunchKernelGGL((mx_linear_kernel<MT, NT, WM, WN, ST, KG, GELU>), grid, dim3(T::kThreads), 0, st, p);
}

// Few rows: a workgroup's 8 waves share a tile of 16 MT rows of y by 16 NT channels and
// split its columns of K.  They have no operand in common, so fragments go from HBM
// straight to registers, the next step's while this one's are multiplied; a
// problem whose steps one after the other would each wait for memory waits an eighth as
// often.  The partial sums meet in LDS: the upper four waves' are added to the lower
// four's, then 512 threads add four each, 8 neighbouring channels of a row at a time.
constexpr int kRowWaves = 8;

template <int MT, int NT, bool GELU>
__global__ void __launch_bounds__(64 * kRowWaves, 2) mx_linear_rows_kernel(const MxLinearArgs p) {
  constexpr int kBM = 16 * MT, kBN = 16 * NT, kLine = kBN + 4;
  __shared__ __attribute__((aligned(16))) float part[kRowWaves / 2][kBM][kLine];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  // workgroups of one XCD share channels: the rows of y go by first
  const int tm = (p.M + kBM - 1) / kBM;
  const int per = gridDim.x / 8, rem = gridDim.x % 8, xcd = blockIdx.x % 8;
  const int tile = xcd * per + min(xcd, rem) + blockIdx.x / 8;
  const int m0 = __builtin_amdgcn_readfirstlane(tile % tm * kBM), n0 = __builtin_amdgcn_readfirstlane(tile / tm * kBN);
  const int steps = (p.K + 127) / 128, own = (steps + kRowWaves - 1) / kRowWaves;
  const int first = wave * own, last = min(first + own, steps);

  const int mrows = min(p.M - m0, kBM), nrows = max(min(p.N - n0, kBN), 0);
  const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + (int64_t)m0 * p.K), (short)0, mrows * p.K, 0x00020000);
  const auto rw = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + (int64_t)n0 * p.K), (short)0, nrows * p.K, 0x00020000);
  struct Fragments {
    mx_i8 a[MT], w[NT];
    int sa[MT], sw[NT];
  };
  // rows past the operand's last, and columns past K by their offset, read as zeros
  auto load = [&](Fragments& f, int ks) {
    const int lo = ks * 128 + g * 16, hi = lo + 64;
    const int plo = lo < p.K ? lo : 0x40000000, phi = hi < p.K ? hi : 0x40000000;
#pragma unroll
    for (int t = 0; t < MT; ++t) f.a[t] = mx_fragment(ra, (t * 16 + r16) * p.K + plo, (t * 16 + r16) * p.K + phi);
#pragma unroll
    for (int u = 0; u < NT; ++u) f.w[u] = mx_fragment(rw, (u * 16 + r16) * p.K + plo, (u * 16 + r16) * p.K + phi);
    const bool live = ks * 128 + g * 32 < p.K;  // the scale bytes of blocks past K are not looked at
    const uint8_t* as = p.as + ((int64_t)ks * p.M + m0) * 4 + g;
    const uint8_t* ws = p.ws + ((int64_t)ks * p.N + n0) * 4 + g;
#pragma unroll
    for (int t = 0; t < MT; ++t) f.sa[t] = live && t * 16 + r16 < mrows ? as[(t * 16 + r16) * 4] : 0;
#pragma unroll
    for (int u = 0; u < NT; ++u) f.sw[u] = live && u * 16 + r16 < nrows ? ws[(u * 16 + r16) * 4] : 0;
  };
  mx_f4 acc[MT][NT] = {};
  auto products = [&](const Fragments& f) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u)
        acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f.w[u], f.a[t], acc[t][u], 0, 0, 0, f.sw[u], 0, f.sa[t]);
  };
  Fragments f[2];
  if (first < last) load(f[0], first);
  int ks = first;
  for (; ks + 2 < last; ks += 2) {
    load(f[1], ks + 1);
    products(f[0]);
    load(f[0], ks + 2);
    products(f[1]);
  }
  if (ks + 1 < last) {
    load(f[1], ks + 1);
    products(f[0]);
    products(f[1]);
  } else if (ks < last) {
    products(f[0]);
  }

  // lane: channels 16 u + 4 g .. + 3 of row 16 t + r16
  if (wave >= kRowWaves / 2)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u)
        *reinterpret_cast<mx_f4*>(&part[wave - kRowWaves / 2][t * 16 + r16][u * 16 + g * 4]) = acc[t][u];
  __syncthreads();
  if (wave < kRowWaves / 2)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        mx_f4* to = reinterpret_cast<mx_f4*>(&part[wave][t * 16 + r16][u * 16 + g * 4]);
        *to = *to + acc[t][u];
      }
  __syncthreads();
  constexpr int kItems = kBM * kBN / 8, kCols = kBN / 8;
#pragma unroll
  for (int i0 = 0; i0 < kItems; i0 += 64 * kRowWaves) {
    const int i = i0 + threadIdx.x;
    if (kItems % (64 * kRowWaves) != 0 && i >= kItems) break;  // whole blocks of 4 threads
    const int row = i / kCols, c = i % kCols * 8, m = m0 + row, n = n0 + c;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const mx_f4 x = *reinterpret_cast<const mx_f4*>(&part[0][row][c + e]), y = *reinterpret_cast<const mx_f4*>(&part[1][row][c + e]);
      const mx_f4 z = *reinterpret_cast<const mx_f4*>(&part[2][row][c + e]), w = *reinterpret_cast<const mx_f4*>(&part[3][row][c + e]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[e + k] = (x[k] + y[k]) + (z[k] + w[k]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] += p.bias != nullptr && n + e < p.N ? bf16_bits_to_f32(p.bias[n + e]) : 0.0f;
      if (GELU) v[e] = mx_gelu(v[e]);
    }
    if (p.ys != nullptr) {
      if constexpr (NT % 2 == 0) {
        float top = mx_top(v);
        top = fmaxf(top, __shfl_xor(top, 1, 64));
        top = fmaxf(top, __shfl_xor(top, 2, 64));
        const uint32_t code = mx_scale_code(top);
        const float inv = mx_inverse(code);
        if (m < p.M) {
          if (n < p.N)
            *reinterpret_cast<uint2*>((uint8_t*)p.y + (int64_t)m * p.N + n) =
                make_uint2(mx_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                           mx_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
          // blocks past N up to the next 128 columns are written as 0
          if (n % 32 == 0 && n / 128 < (p.N + 127) / 128)
            p.ys[((int64_t)(n / 128) * p.M + m) * 4 + n / 32 % 4] = (uint8_t)code;
        }
      }
    } else if (m < p.M) {
      uint16_t* yp = (uint16_t*)p.y + (int64_t)m * p.y_ls + n;
      if (n + 8 <= p.N) {
        const uint4 w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                   pack_bf16x2(v[6], v[7]));
        __builtin_memcpy(yp, &w, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < p.N) yp[e] = f32_to_bf16_bits(v[e]);
      }
    }
  }
}

template <int MT, int NT, bool GELU>
void launch_mx_rows(const MxLinearArgs& p, hipStream_t st) {
  const int64_t cols = p.ys != nullptr ? ceil_div(p.N, 128) * 128 : p.N;
  const dim3 grid((unsigned)(ceil_div(cols, 16 * NT) * ceil_div(p.M, 16 * MT)));
  hipLaunchKernelGGL((mx_linear_rows_kernel<MT, NT, GELU>), grid, dim3(64 * kRowWaves), 0, st, p);
}

// The kernels by their tile of y and the groups that split K, with an estimate of
// their time in us, fitted to 75 shapes of 1 to 2304 rows, 128 to 16384 columns and 32
// to 16384 channels: `once`, then for every round of workgroups `round` plus `step` for
// each step of a group (`each` per 256 tiles and step instead where many tiles
// share a CU), never below what the bytes take at 5.3 TB/s.  Over those shapes the
// choice is within 1 % of the fastest of 19 tiles in the mean.  What each is for, the
// next best beside it: 1 row of 8256 -> 195 16 x 16 7.0 us (16 x 32, whose tiles hold the blocks
// of an 8-bit result, and 32 x 32 9.8); 8 rows of 4096 -> 4096 32 x 32 6.9 (16 x 16 7.1); 75 rows of 2048 -> 8192 48 x 64 7.4 (80 x 64 8.6),
// 150 rows 80 x 64 9.2 (160 x 64 10.7), of 8192 -> 2048 48 x 32 12.0 (32 x 64 14.3); 331 rows of
// 1056 -> 4099 160 x 64 9.2 (128 x 128 11.2); 768 rows of 16384 -> 4096 128 x 128 64 (48 x 64 and
// 80 x 64 88 and more); 384 rows of 4096 -> 16384 128 x 256 34.6 (192 x 256 36.8); 2304 rows 192 x 256
// 146 (256 x 256 150), to 12288 channels 256 x 256 111 (192 x 256 121).
struct MxShape {
  int rows, cols, groups;
  float once, round, step, each;
  void (*launch[2])(const MxLinearArgs&, hipStream_t);  // plain, with GELU
};
constexpr MxShape kMxShapes[] = {
    // bf16 results
    {16, 16, 8, 3.13f, 0.0f, 0.37f, 0.76f, {launch_mx_rows<1, 1, false>, launch_mx_rows<1, 1, true>}},
    // 8-bit ones: whole blocks
    {16, 32, 8, 2.98f, 0.0f, 0.65f, 1.32f, {launch_mx_rows<1, 2, false>, launch_mx_rows<1, 2, true>}},
    {32, 32, 4, 1.84f, 2.06f, 0.39f, 0.0f, {launch_mx_linear<2, 2, 1, 1, 3, 4, false>, launch_mx_linear<2, 2, 1, 1, 3, 4, true>}},
    {32, 64, 4, 1.66f, 2.59f, 0.60f, 0.0f, {launch_mx_linear<2, 2, 1, 2, 3, 4, false>, launch_mx_linear<2, 2, 1, 2, 3, 4, true>}},
    {48, 32, 4, 1.70f, 2.38f, 0.47f, 0.0f, {launch_mx_linear<3, 2, 1, 1, 3, 4, false>, launch_mx_linear<3, 2, 1, 1, 3, 4, true>}},
    {48, 64, 4, 1.48f, 2.38f, 0.68f, 0.0f, {launch_mx_linear<3, 2, 1, 2, 2, 4, false>, launch_mx_linear<3, 2, 1, 2, 2, 4, true>}},
    {80, 64, 4, 1.19f, 3.14f, 0.85f, 0.0f, {launch_mx_linear<5, 2, 1, 2, 2, 4, false>, launch_mx_linear<5, 2, 1, 2, 2, 4, true>}},
    {160, 64, 2, 0.0f, 4.16f, 0.70f, 0.0f, {launch_mx_linear<5, 2, 2, 2, 2, 2, false>, launch_mx_linear<5, 2, 2, 2, 2, 2, true>}},
    {128, 128, 2, 0.0f, 4.95f, 0.86f, 0.0f, {launch_mx_linear<4, 4, 2, 2, 2, 2, false>, launch_mx_linear<4, 4, 2, 2, 2, 2, true>}},
    {128, 256, 1, 0.0f, 5.39f, 0.77f, 0.0f, {launch_mx_linear<4, 4, 2, 4, 3, 1, false>, launch_mx_linear<4, 4, 2, 4, 3, 1, true>}},
    {192, 256, 1, 0.0f, 5.22f, 0.91f, 0.0f, {launch_mx_linear<6, 4, 2, 4, 2, 1, false>, launch_mx_linear<6, 4, 2, 4, 2, 1, true>}},
    {256, 256, 1, 0.0f, 6.34f, 1.05f, 0.0f, {launch_mx_linear<8, 4, 2, 4, 2, 1, false>, launch_mx_linear<8, 4, 2, 4, 2, 1, true>}},
};

// Whether a tile can hold such a result: the smallest exist once for either kind.
bool mx_admits(const MxShape& h, bool quantized) { return h.each == 0.0f || h.cols == (quantized ? 32 : 16); }

// Null if every tile makes more workgroups than a grid of 512 threads each may have (2^32 threads).
const MxShape* choose_mx(int64_t M, int64_t N, int64_t K, bool quantized) {
  const float bytes = ((float)M + N) * K * 1.03f + 2.0f * M * N, floor = 2.5f + bytes / 5.3e6f;
  const int64_t cols = quantized ? ceil_div(N, 128) * 128 : N;
  const MxShape* best = nullptr;
  float least = 0.0f;
  for (const MxShape& h : kMxShapes) {
    if (!mx_admits(h, quantized)) continue;
    const int64_t count = ceil_div(M, h.rows) * ceil_div(cols, h.cols);
    if (count >= (int64_t{1} << 32) / 512) continue;
    const float tiles = (float)count;
    const float steps = (float)ceil_div(ceil_div(K, 128), h.groups);
    const float rounds = h.each > 0.0f ? 1.0f : ceilf(tiles / 256.0f);
    const float own = h.once + rounds * (h.round + steps * h.step) + tiles / 256.0f * steps * h.each;
    const float t = fmaxf(own, floor) + 0.1f * own;  // between those at the floor, the one with least of its own
    if (best == nullptr || t < least) best = &h, least = t;
  }
  return best;
}

}  // namespace ltx

using namespace ltx;

#define LTX_REQUIRE_MX_SIZES(name)                                                                               \
  LTX_REQUIRE(M >= 0 && M <= 0x3FFFFFFF && N >= 0 && N <= 0x3FFFFFFF, name ": bad M or N");                       \
  LTX_REQUIRE(K >= kMxBlock && K % kMxBlock == 0 && K <= LTX_MX_MAX_K,                                            \
              name ": K must be a multiple of %d, at most %d", kMxBlock, LTX_MX_MAX_K)

extern "C" int ltx_mx_linear_tile(int64_t M, int64_t N, int64_t K, int quantized, int64_t* tile) {
  clear_error();
  LTX_REQUIRE_MX_SIZES("ltx_mx_linear_tile");
  LTX_REQUIRE(tile != nullptr, "ltx_mx_linear_tile: null pointer");
  const MxShape* const h = M * N == 0 ? nullptr : choose_mx(M, N, K, quantized != 0);
  LTX_REQUIRE(h != nullptr, "ltx_mx_linear_tile: the result is empty or too large");
  tile[0] = h->rows, tile[1] = h->cols, tile[2] = h->groups, tile[3] = tile[4] = 0;
  for (const MxShape& o : kMxShapes) {
    if (!mx_admits(o, quantized != 0)) continue;
    tile[3] += &o < h;
    tile[4] += 1;
  }
  return LTX_OK;
}

extern "C" int ltx_mx_linear(int64_t M, int64_t N, int64_t K, const void* a_codes, const void* a_scales,
                             const void* w_codes, const void* w_scales, const void* bias, int act, void* y,
                             int64_t y_ls, void* y_scales, void* stream) {
  clear_error();
  LTX_REQUIRE_MX_SIZES("ltx_mx_linear");
  LTX_REQUIRE(act == 0 || act == 1, "ltx_mx_linear: unknown activation %d", act);
  LTX_REQUIRE(y_scales == nullptr || N % kMxBlock == 0, "ltx_mx_linear: 8-bit output needs N a multiple of %d", kMxBlock);
  if (M * N == 0) return LTX_OK;
  LTX_REQUIRE(a_codes != nullptr && a_scales != nullptr && w_codes != nullptr && w_scales != nullptr && y != nullptr,
              "ltx_mx_linear: null pointer");
  LTX_REQUIRE((uintptr_t)a_codes % 16 == 0 && (uintptr_t)w_codes % 16 == 0 && (uintptr_t)a_scales % 4 == 0 &&
                  (uintptr_t)w_scales % 4 == 0 && (y_scales == nullptr || ((uintptr_t)y % 16 == 0 && (uintptr_t)y_scales % 4 == 0)),
              "ltx_mx_linear: codes must be 16-byte aligned, scales 4-byte");
  LTX_REQUIRE(y_scales != nullptr || M == 1 || y_ls >= N, "ltx_mx_linear: rows of y overlap");
  MxLinearArgs p{(const uint8_t*)a_codes, (const uint8_t*)a_scales, (const uint8_t*)w_codes, (const uint8_t*)w_scales,
                 (const uint16_t*)bias, y, (uint8_t*)y_scales, y_ls, (int)M, (int)N, (int)K};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const MxShape* const h = choose_mx(M, N, K, y_scales != nullptr);
  LTX_REQUIRE(h != nullptr, "ltx_mx_linear: the result is too large");
  h->launch[act](p, st);
  LTX_LAUNCH_CHECK("ltx_mx_linear");
  return LTX_OK;
}
