// Gated residual update + modulated RMSNorm with 8-bit output rows (gfx950): the
// producer of the block-scaled linears' activations.
//
//   x' = x + y * g,  n = x' * rsqrt(mean x'^2 + eps) * (1 + scale) + shift
//   codes, scales = 8-bit rows of n (mx_common.h); x_out = bf16(x')
//
// Everything between the loads and the two outputs is float32; x' is rounded
// to bf16 for the residual stream only, n once, to its code.
//
// Bound by HBM: one read of x, y and the modulation rows, one write of x_out
// and of the codes (half of the bf16 row that ltx_adaln writes): 13.7 us at
// 2304 x 4096 (66 MB, 4.8 TB/s), 19.5 at 1980 x 4096 with modulation rows per token.  One workgroup
// per row, 8 channels per chunk of a thread, so that the four lanes of a quad
// hold a block: its maximum is two quad exchanges, the row's sum of squares
// the only reduction across the workgroup.  Threads past the row's last chunk
// carry zeros, so every exchange is between live lanes.

#include "mx_common.h"

namespace ltx {

struct MxNormArgs {
  const uint16_t* x;
  int64_t x_bs, x_ls;
  const uint16_t* y;      // null: x' = x
  int64_t y_bs, y_ls;
  const uint16_t* gate;   // null: x' = x + y
  int64_t g_bs, g_ls;
  uint16_t* x_out;        // null: not written
  int64_t xo_bs, xo_ls;
  const uint16_t* scale;  // null: no modulation
  int64_t s_bs, s_ls;
  const uint16_t* shift;
  int64_t h_bs, h_ls;
  uint8_t* codes;
  uint8_t* scales;
  int64_t B, rows;        // rows = B * L
  int C;
  float eps;              // < 0: no norm
};

constexpr int kMxMaxBatchY = 65535;

template <int NV>
__global__ void __launch_bounds__(1024 / NV) adaln_mx_kernel(const MxNormArgs a) {
  const int64_t l = blockIdx.x, b = (int64_t)blockIdx.z * kMxMaxBatchY + blockIdx.y;
  if (b >= a.B) return;  // uniform across the block
  const bool has_y = a.y != nullptr, has_gate = a.gate != nullptr, modulate = a.scale != nullptr;
  const int nch = a.C / 8;
  int ch[NV];
  bool live[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ch[i] = threadIdx.x + i * blockDim.x;
    live[i] = ch[i] < nch;
  }
  auto ld = [&](const uint16_t* p, int64_t bs, int64_t ls, int i) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live[i]) v = *reinterpret_cast<const uint4*>(p + (b * bs + l * ls) + (int64_t)ch[i] * 8);
    return v;
  };
  auto get = [](const uint4& r, int e) {
    const uint32_t w = (&r.x)[e >> 1];
    return (e & 1) ? __uint_as_float(w & 0xFFFF0000u) : __uint_as_float(w << 16);
  };
  uint4 xv[NV], yv[NV], gv[NV], sv[NV], hv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) xv[i] = ld(a.x, a.x_bs, a.x_ls, i);
  if (has_y)
#pragma unroll
    for (int i = 0; i < NV; ++i) yv[i] = ld(a.y, a.y_bs, a.y_ls, i);
  if (has_gate)
#pragma unroll
    for (int i = 0; i < NV; ++i) gv[i] = ld(a.gate, a.g_bs, a.g_ls, i);
  if (modulate)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      sv[i] = ld(a.scale, a.s_bs, a.s_ls, i);
      hv[i] = ld(a.shift, a.h_bs, a.h_ls, i);
    }

  float x[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = get(xv[i], e);
      if (has_y) v = has_gate ? fmaf(get(yv[i], e), get(gv[i], e), v) : v + get(yv[i], e);
      x[i][e] = v;
      ss = fmaf(v, v, ss);
    }
    if (a.x_out != nullptr && live[i])
      *reinterpret_cast<uint4*>(a.x_out + (b * a.xo_bs + l * a.xo_ls) + (int64_t)ch[i] * 8) =
          make_uint4(pack_bf16x2(x[i][0], x[i][1]), pack_bf16x2(x[i][2], x[i][3]), pack_bf16x2(x[i][4], x[i][5]),
                     pack_bf16x2(x[i][6], x[i][7]));
  }
  if (a.eps >= 0.0f) {  // uniform across the grid
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
    __shared__ float red[16];
    const int nwaves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    float tot = 0.0f;
    for (int w = 0; w < nwaves; ++w) tot += red[w];
    const float rs = 1.0f / sqrtf(__fadd_rn(__fdiv_rn(tot, (float)a.C), a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[i][e] *= rs;
        if (modulate) x[i][e] = fmaf(x[i][e], 1.0f + get(sv[i], e), get(hv[i], e));
      }
  }
  const int64_t row = b * gridDim.x + l;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float top = mx_top(x[i]);
    top = fmaxf(top, __shfl_xor(top, 1, 64));
    top = fmaxf(top, __shfl_xor(top, 2, 64));
    const uint32_t code = mx_scale_code(top);
    const float inv = mx_inverse(code);
    if (live[i])
      *reinterpret_cast<uint2*>(a.codes + row * a.C + (int64_t)ch[i] * 8) =
          make_uint2(mx_pack4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv),
                     mx_pack4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv));
    // the four scales of 128 columns in one word; blocks past the row hold zeros, whose code is 0
    uint32_t word = code << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor(word, 4, 64);
    word |= __shfl_xor(word, 8, 64);
    if (live[i] && (lane & 15) == 0)
      *reinterpret_cast<uint32_t*>(a.scales + ((int64_t)(ch[i] >> 4) * a.rows + row) * 4) = word;
  }
}

}  // namespace ltx

using namespace ltx;

extern "C" int ltx_adaln_mx(int64_t B, int64_t L, int64_t C, const void* x, int64_t x_bs, int64_t x_ls,
                            const void* y, int64_t y_bs, int64_t y_ls, const void* gate, int64_t g_bs,
                            int64_t g_ls, void* x_out, int64_t xo_bs, int64_t xo_ls, const void* scale,
                            int64_t s_bs, int64_t s_ls, const void* shift, int64_t h_bs, int64_t h_ls, float eps,
                            void* codes, void* scales, void* stream) {
  clear_error();
  LTX_REQUIRE(B >= 0 && L >= 0 && C >= kMxBlock && C % kMxBlock == 0 && C <= 8192,
              "ltx_adaln_mx: C must be a multiple of %d in [%d, 8192]", kMxBlock, kMxBlock);
  // a grid holds fewer than 2^32 threads along L, at most 512 a row
  LTX_REQUIRE(B <= 0x7FFFFFFF && L < (int64_t{1} << 32) / 512 && B * L <= 0x7FFFFFFF, "ltx_adaln_mx: too many rows");
  if (B * L == 0) return LTX_OK;
  LTX_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "ltx_adaln_mx: null pointer");
  LTX_REQUIRE(gate == nullptr || y != nullptr, "ltx_adaln_mx: a gate needs a residual branch y");
  LTX_REQUIRE((scale == nullptr) == (shift == nullptr), "ltx_adaln_mx: scale and shift go together");
  LTX_REQUIRE(scale == nullptr || eps >= 0.0f, "ltx_adaln_mx: modulation needs the norm");
  LTX_REQUIRE(x_out == nullptr || y != nullptr, "ltx_adaln_mx: x_out without a residual branch");
  // one sample after the other, or one token's samples after the other's
  const auto apart = [&](int64_t n, int64_t step) { return n == 1 || step >= C; };
  const auto nested = [&](int64_t n, int64_t inner, int64_t outer) { return (outer - C) / (n - 1) >= inner; };
  LTX_REQUIRE(x_out == nullptr || (apart(L, xo_ls) && apart(B, xo_bs) &&
                                   (L == 1 || B == 1 || nested(L, xo_ls, xo_bs) || nested(B, xo_bs, xo_ls))),
              "ltx_adaln_mx: rows of x_out overlap");
  auto ok = [](const void* p, int64_t bs, int64_t ls) {
    return p == nullptr || (((uintptr_t)p % 16) == 0 && bs % 8 == 0 && ls % 8 == 0);
  };
  LTX_REQUIRE(ok(x, x_bs, x_ls) && ok(y, y_bs, y_ls) && ok(gate, g_bs, g_ls) && ok(x_out, xo_bs, xo_ls) &&
                  ok(scale, s_bs, s_ls) && ok(shift, h_bs, h_ls) && (uintptr_t)codes % 16 == 0 &&
                  (uintptr_t)scales % 4 == 0,
              "ltx_adaln_mx: rows and codes must be 16-byte aligned, scales 4-byte");
  MxNormArgs a{(const uint16_t*)x, x_bs, x_ls, (const uint16_t*)y, y_bs, y_ls, (const uint16_t*)gate, g_bs, g_ls,
               (uint16_t*)x_out, xo_bs, xo_ls, (const uint16_t*)scale, s_bs, s_ls, (const uint16_t*)shift, h_bs,
               h_ls, (uint8_t*)codes, (uint8_t*)scales, B, B * L, (int)C, eps};
  const dim3 grid((unsigned)L, (unsigned)(B < kMxMaxBatchY ? B : kMxMaxBatchY), (unsigned)ceil_div(B, kMxMaxBatchY));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto threads = [&](int nv) { return dim3((unsigned)(ceil_div(C, 8 * nv * 64) * 64)); };
  if (C >= 2048)
    hipLaunchKernelGGL(adaln_mx_kernel<2>, grid, threads(2), 0, st, a);
  else
    hipLaunchKernelGGL(adaln_mx_kernel<1>, grid, threads(1), 0, st, a);
  LTX_LAUNCH_CHECK("ltx_adaln_mx");
  return LTX_OK;
}
