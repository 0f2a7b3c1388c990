// Linear layers over a few rows with 4-bit weights (gfx950): y = act(x) W^T +
// bias, W = e2m1 code * bf16 scale of its group of 32, 64 or 128 columns.
#include "ltx_common.h"

namespace ltx {

constexpr int kG4Threads = 256;

struct Group4Args {
  const uint16_t* x;
  int64_t x_ls;
  const uint8_t* codes;
  const uint16_t* scales;
  const uint16_t* bias;  // null: none
  uint16_t* y;
  int64_t y_ls;
  int64_t N;
  int M, K, group, silu;
};

// One wave per row of W: lanes stride over its 16-byte pieces.
__global__ void __launch_bounds__(kG4Threads) group4_linear_kernel(const Group4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * (kG4Threads / 64) + (threadIdx.x >> 6);
  if (n >= a.N) return;
  const int chunks = (a.K + 127) / 128;
  float acc[LTX_GROUP4_MAX_ROWS] = {};
  for (int i = lane; i < chunks * 4; i += 64) {
    const uint4 w = *reinterpret_cast<const uint4*>(a.codes + n * chunks * 64 + (int64_t)i * 16);
    for (int j = 0; j < 4; ++j) {
      const int k = (i >> 2) * 128 + j * 32 + (i & 3) * 8;
      if (k >= a.K) break;
      const float s = bf16_bits_to_f32(a.scales[n * (a.K / a.group) + k / a.group]);
      const uint32_t word = (&w.x)[j];
      float v[8];
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = (word >> (4 * e)) & 15u, m = c & 7u;
        const float mag = m < 2u ? 0.5f * m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
        v[e] = (c & 8u) ? -mag * s : mag * s;
      }
      for (int m = 0; m < a.M; ++m)
        for (int e = 0; e < 8; ++e) {
          float xv = bf16_bits_to_f32(a.x[m * a.x_ls + k + e]);
          if (a.silu) xv = bf16_bits_to_f32(f32_to_bf16_bits(xv / (1.0f + expf(-xv))));
          acc[m] = fmaf(xv, v[e], acc[m]);
        }
    }
  }
  for (int m = 0; m < a.M; ++m) {
    float t = acc[m];
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    if (lane == 0) {
      if (a.bias != nullptr) t += bf16_bits_to_f32(a.bias[n]);
      a.y[m * a.y_ls + n] = f32_to_bf16_bits(t);
    }
  }
}

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
  LTX_REQUIRE((uintptr_t)x % 16 == 0 && x_ls % 8 == 0 && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 2 == 0,
              "ltx_group4_linear: x rows and codes must be 16-byte aligned");
  Group4Args a{(const uint16_t*)x, x_ls, (const uint8_t*)codes, (const uint16_t*)scales, (const uint16_t*)bias,
               (uint16_t*)y, y_ls, N, (int)M, (int)K, (int)group, silu};
  hipLaunchKernelGGL(group4_linear_kernel, dim3((unsigned)ceil_div(N, kG4Threads / 64)), dim3(kG4Threads), 0,
                     reinterpret_cast<hipStream_t>(stream), a);
  LTX_LAUNCH_CHECK("ltx_group4_linear");
  return LTX_OK;
}
