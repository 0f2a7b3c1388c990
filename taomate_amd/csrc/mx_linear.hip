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
// Tiles of a and w travel HBM -> LDS without registers, 128 columns (one MFMA's
// depth) per step, in rows of 128 bytes whose 16-byte chunks are exchanged by
// chunk ^= (row / 2) % 8: the 16 rows that a fragment read touches then lie in
// 16 different 16-byte columns of the LDS.  Tile t of a wave's w rows holds the
// channels 4 NT i + 4 t + r (i, r in [0, 4)) in its rows 4 i + r, so that lane
// group i ends with the 4 NT neighbouring channels 4 NT i ..: contiguous stores,
// and blocks of 32 for an 8-bit result inside one lane (NT = 8) or a pair (NT = 4).

#include "mx_common.h"

namespace ltx {

typedef int mx_i4 __attribute__((ext_vector_type(4)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* mx_lds_ptr;

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
  int vec;               // bf16 rows of y take 16-byte stores
};

// tanh-GELU: y sigmoid(2 u), u = sqrt(2 / pi) (y + 0.044715 y^3).  The sigmoid
// through one exp2 and one reciprocal (1 ulp each).
__device__ __forceinline__ float mx_gelu(float y) {
  const float c = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  const float u = c * (y + 0.044715f * y * y * y);
  return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u));
}

// MT x NT tiles of 16 x 16 per wave, WM x WN waves, ST buffers of one step.
template <int MT, int NT, int WM, int WN, int ST>
struct MxTile {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kBM = 16 * MT * WM, kBN = 16 * NT * WN, kRows = kBM + kBN;
  static constexpr int kCodes = kRows * 128, kStage = kCodes + kRows * 4;
  static constexpr int kPer = (kRows / 8 + kWaves - 1) / kWaves;  // 1 KB loads (8 rows) per wave and step
  static constexpr int kScalesPer = (kRows + kWaves - 1) / kWaves;
  static_assert(kScalesPer <= 64 && kRows % 8 == 0, "one scale load per wave");
  static_assert(ST * kStage <= 160 * 1024, "LDS");
};

template <int MT, int NT, int WM, int WN, int ST, bool GELU>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4 > 0 ? WM * WN / 4 : 1) mx_linear_kernel(const MxLinearArgs p) {
  using T = MxTile<MT, NT, WM, WN, ST>;
  __shared__ __attribute__((aligned(128))) uint8_t lds[ST * T::kStage];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mx_lds_ptr)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int g = lane >> 4, r16 = lane & 15;
  const int m0 = blockIdx.y * T::kBM, n0 = blockIdx.x * T::kBN;
  const int steps = (p.K + 127) / 128;

  // Buffer descriptors of the tile's rows: rows past M or N lie past the end and read as zeros.
  const int mrows = min(p.M - m0, T::kBM), nrows = max(min(p.N - n0, T::kBN), 0);
  const auto ra =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.a + (int64_t)m0 * p.K), (short)0, mrows * p.K, 0x00020000);
  const auto rw =
      __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + (int64_t)n0 * p.K), (short)0, nrows * p.K, 0x00020000);

  // This lane's part of the wave's loads: LDS rows 8 j .. of load j, a chunk each.
  uint32_t voff[T::kPer];
  uint32_t col[T::kPer];
#pragma unroll
  for (int q = 0; q < T::kPer; ++q) {
    const int row = (q * T::kWaves + wave) * 8 + (lane >> 3);
    const int c = (lane & 7) ^ ((row >> 1) & 7);
    int src = row;
    if (row >= T::kBM) {  // w: channel order of the wave's block
      const int s = (row - T::kBM) % (16 * NT), b = (row - T::kBM) / (16 * NT);
      src = b * 16 * NT + (s % 16 / 4) * 4 * NT + (s / 16) * 4 + s % 4;
    }
    col[q] = (uint32_t)c * 16;
    voff[q] = (uint32_t)src * (uint32_t)p.K + col[q];
  }
  // and of the scales: one word (four blocks) per row of the tile
  const int srow = wave * T::kScalesPer + lane;
  const bool sload = lane < T::kScalesPer && srow < T::kRows;
  const bool sa = srow < T::kBM;
  int ssrc = srow;
  if (!sa) {
    const int s = (srow - T::kBM) % (16 * NT), b = (srow - T::kBM) / (16 * NT);
    ssrc = b * 16 * NT + (s % 16 / 4) * 4 * NT + (s / 16) * 4 + s % 4;
  }
  const uint8_t* sp = sa ? p.as + (int64_t)min(m0 + ssrc, p.M - 1) * 4 : p.ws + (int64_t)min(n0 + ssrc, p.N - 1) * 4;
  const int64_t sstep = (int64_t)(sa ? p.M : p.N) * 4;

  auto load = [&](int ks) {
    const uint32_t base = lds0 + (uint32_t)(ks % ST) * T::kStage;
    const uint32_t k0 = (uint32_t)ks * 128;
#pragma unroll
    for (int q = 0; q < T::kPer; ++q) {
      const int j = q * T::kWaves + wave;
      if (T::kPer * T::kWaves * 8 == T::kRows || j * 8 < T::kRows) {
        // columns past K read as zeros: an offset past the end of either operand
        const uint32_t off = k0 + col[q] < (uint32_t)p.K ? voff[q] + k0 : 0x80000000u;
        const mx_lds_ptr to = (mx_lds_ptr)(uintptr_t)(base + (uint32_t)j * 1024);
        if (j * 8 < T::kBM)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, to, 16, off, 0, 0, 0);
        else
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, to, 16, off, 0, 0, 0);
      }
    }
  };
  auto load_scales = [&](int ks) { return sload ? *reinterpret_cast<const uint32_t*>(sp + ks * sstep) : 0u; };
  auto put_scales = [&](int ks, uint32_t word) {
    // the scale bytes of blocks past K are not looked at
    const int left = p.K / 32 - ks * 4;
    if (left < 4) word &= (1u << (8 * left)) - 1u;
    if (sload) *reinterpret_cast<uint32_t*>(lds + (ks % ST) * T::kStage + T::kCodes + srow * 4) = word;
  };

  mx_f4 acc[MT][NT] = {};
  load(0);
  put_scales(0, load_scales(0));
  for (int ks = 0; ks < steps; ++ks) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t next_scales = 0;
    if (ks + 1 < steps) {
      next_scales = load_scales(ks + 1);
      load(ks + 1);
    }
    const uint8_t* st = lds + (ks % ST) * T::kStage;
    auto fragment = [&](int row) {
      const int sw = (row >> 1) & 7;
      const mx_i4 lo = *reinterpret_cast<const mx_i4*>(st + row * 128 + ((g ^ sw) * 16));
      const mx_i4 hi = *reinterpret_cast<const mx_i4*>(st + row * 128 + (((g + 4) ^ sw) * 16));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto scale = [&](int row) { return (int)st[T::kCodes + row * 4 + g]; };
    mx_i8 fw[NT];
    int sw[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = T::kBM + (wn * NT + t) * 16 + r16;
      fw[t] = fragment(row);
      sw[t] = scale(row);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = (wm * MT + t) * 16 + r16;
      const mx_i8 fa = fragment(row);
      const int sc = scale(row);
#pragma unroll
      for (int u = 0; u < NT; ++u)
        acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u], fa, acc[t][u], 0, 0, 0, sw[u], 0, sc);
    }
    if (ks + 1 < steps) put_scales(ks + 1, next_scales);
  }

  // Epilogue: lane group g holds channels n .. n + 4 NT - 1 of row m for every tile row.
  const int n = n0 + wn * 16 * NT + g * 4 * NT;
  float bias[4 * NT];
#pragma unroll
  for (int i = 0; i < 4 * NT; ++i)
    bias[i] = p.bias != nullptr && n + i < p.N ? bf16_bits_to_f32(p.bias[n + i]) : 0.0f;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = m0 + (wm * MT + t) * 16 + r16;
    float v[4 * NT];
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) {
      v[i] = acc[t][i / 4][i % 4] + bias[i];
      if (GELU) v[i] = mx_gelu(v[i]);
    }
    if (p.ys != nullptr) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        if (n + i >= p.N) v[i] = 0.0f;
        top = fmaxf(top, mx_magnitude(v[i]));
      }
      if (NT < 8) top = fmaxf(top, __shfl_xor(top, 16, 64));
      static_assert(NT == 4 || NT == 8, "a block of 32 lies in one lane or a pair of lanes");
      const uint32_t code = mx_scale_code(top);
      const float inv = mx_inverse(code);
      if (m < p.M) {
        uint8_t* yp = (uint8_t*)p.y + (int64_t)m * p.N + n;
#pragma unroll
        for (int i = 0; i < 4 * NT; i += 16) {
          const uint4 c = make_uint4(mx_pack4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv),
                                     mx_pack4(v[i + 4] * inv, v[i + 5] * inv, v[i + 6] * inv, v[i + 7] * inv),
                                     mx_pack4(v[i + 8] * inv, v[i + 9] * inv, v[i + 10] * inv, v[i + 11] * inv),
                                     mx_pack4(v[i + 12] * inv, v[i + 13] * inv, v[i + 14] * inv, v[i + 15] * inv));
          if (n + i < p.N) *reinterpret_cast<uint4*>(yp + i) = c;
        }
        // blocks past N up to the next 128 columns are written as 0
        if (n / 128 < (p.N + 127) / 128 && n % 32 == 0)
          p.ys[((int64_t)(n / 128) * p.M + m) * 4 + n / 32 % 4] = (uint8_t)code;
      }
    } else if (m < p.M) {
      uint16_t* yp = (uint16_t*)p.y + (int64_t)m * p.y_ls + n;
#pragma unroll
      for (int i = 0; i < 4 * NT; i += 8) {
        if (p.vec && n + i + 8 <= p.N) {
          *reinterpret_cast<uint4*>(yp + i) = make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                                                         pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + i + e < p.N) yp[i + e] = f32_to_bf16_bits(v[i + e]);
        }
      }
    }
  }
}

template <int MT, int NT, int WM, int WN, int ST, bool GELU>
void launch_mx_linear(const MxLinearArgs& p, hipStream_t st) {
  using T = MxTile<MT, NT, WM, WN, ST>;
  // an 8-bit result's scales are written up to the next 128 columns
  const int64_t cols = p.ys != nullptr ? ceil_div(p.N, 128) * 128 : p.N;
  const dim3 grid((unsigned)ceil_div(cols, T::kBN), (unsigned)ceil_div(p.M, T::kBM));
  hipLaunchKernelGGL((mx_linear_kernel<MT, NT, WM, WN, ST, GELU>), grid, dim3(T::kThreads), 0, st, p);
}

}  // namespace ltx

using namespace ltx;

extern "C" int ltx_mx_linear(int64_t M, int64_t N, int64_t K, const void* a_codes, const void* a_scales,
                             const void* w_codes, const void* w_scales, const void* bias, int act, void* y,
                             int64_t y_ls, void* y_scales, void* stream) {
  clear_error();
  LTX_REQUIRE(M >= 0 && M <= 0x3FFFFFFF && N >= 0 && N <= 0x3FFFFFFF, "ltx_mx_linear: bad M or N");
  LTX_REQUIRE(K >= kMxBlock && K % kMxBlock == 0 && K <= LTX_MX_MAX_K,
              "ltx_mx_linear: K must be a multiple of %d, at most %d", kMxBlock, LTX_MX_MAX_K);
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
                 (const uint16_t*)bias, y, (uint8_t*)y_scales, y_ls, (int)M, (int)N, (int)K,
                 (uintptr_t)y % 16 == 0 && y_ls % 8 == 0};
  LTX_REQUIRE(ceil_div(M, 128) <= 65535, "ltx_mx_linear: too many rows");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (act)
    launch_mx_linear<4, 4, 2, 2, 2, true>(p, st);
  else
    launch_mx_linear<4, 4, 2, 2, 2, false>(p, st);
  LTX_LAUNCH_CHECK("ltx_mx_linear");
  return LTX_OK;
}
