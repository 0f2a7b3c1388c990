// A KV cache in blocks for requests of different lengths: the block tables
// (which blocks a request holds, taken from and put back on a stack of free
// blocks) and the writes of new tokens into their slots.
//
// Blocks are `block` tokens (a power of two); token position p of a request
// lies in slot table[p / block] * block + p % block.

#include <initializer_list>

#include "ltx_common.h"

namespace ltx {

// --------------------------------------------------------------------------
// Block tables.
//
// Growing: request b needs take_b = ceil((len_b + new_b) / block) -
// ceil(len_b / block) more blocks and gets them from the top of the stack in
// the order of the requests: with P_b = take_0 + ... + take_{b-1} its j-th new
// block is free[top - 1 - P_b - j].  Token t belongs to the request whose new
// tokens start at S_b = new_0 + ... + new_{b-1} <= t.  Both sums are one scan
// over the requests, so every workgroup does the scan for itself (a few loads
// a thread) and a table entry or a slot is then found by a binary search over
// the sums in LDS, with no order between workgroups: a token in a new block
// reads its id from the stack, not from the table that another workgroup
// writes.  Releasing is the same scan over the blocks of the requests that
// are done.  Nothing is given or taken when the whole call does not fit.
//
// What bounds it is latency: loads of the lengths, the scan, one dependent
// load (block id), the stores.
// --------------------------------------------------------------------------
constexpr int kTableThreads = 256;
constexpr int kTableTokens = 4 * kTableThreads;  // tokens (or returned blocks) of one workgroup

struct TableParams {
  int32_t* tables;
  int64_t t_bs;  // elements from one request's row to the next
  const int32_t* lens;
  const int32_t* fresh;  // new tokens of each request
  const uint8_t* done;
  int32_t* free_list;
  const int32_t* top;
  int32_t* status;
  int32_t *lens_out, *top_out, *starts, *positions;
  int64_t* slots;
  int64_t tokens, n_free;
  int B, width, shift;
  int place, books;  // whether the launch moves blocks and places tokens; whether workgroup 0 keeps the books
};

template <bool GROW>
__global__ void __launch_bounds__(kTableThreads) block_table_kernel(const TableParams p) {
  __shared__ int s_blocks[LTX_MAX_REQUESTS], s_tokens[LTX_MAX_REQUESTS], s_len[LTX_MAX_REQUESTS];
  __shared__ uint32_t s_wave[2][kTableThreads / 64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int top = *p.top;
  const int64_t block = (int64_t)1 << p.shift;
  const int per = (p.B + kTableThreads - 1) / kTableThreads;
  const int b0 = tid * per, b1 = min(b0 + per, p.B);
  auto blocks_of = [&](int64_t n) { return (n + block - 1) >> p.shift; };

  // ---- this thread's requests: their blocks and tokens, and what is wrong ----
  int bad = (top < 0 || top > p.n_free) ? LTX_BLOCKS_FREE : 0;
  uint32_t blocks = 0, tokens = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t len = p.lens[b], add = GROW ? p.fresh[b] : 0;
    const bool mine = GROW || p.done[b] != 0;
    if (len < 0 || add < 0) {
      bad |= LTX_BLOCKS_LENGTH;
    } else {
      if (mine && blocks_of(len + add) > p.width) bad |= LTX_BLOCKS_WIDTH;
      blocks = add_sat(blocks, (uint32_t)(GROW ? blocks_of(len + add) - blocks_of(len) : mine ? blocks_of(len) : 0));
      tokens = add_sat(tokens, (uint32_t)add);
    }
  }
  uint32_t sum_b = wave_scan(blocks), sum_t = wave_scan(tokens);
  if (lane == 63) s_wave[0][wave] = sum_b, s_wave[1][wave] = sum_t;
  __syncthreads();
  uint32_t all_b = 0, all_t = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / 64; ++w) {
    if (w < wave) sum_b = add_sat(sum_b, s_wave[0][w]), sum_t = add_sat(sum_t, s_wave[1][w]);
    all_b = add_sat(all_b, s_wave[0][w]);
    all_t = add_sat(all_t, s_wave[1][w]);
  }
  if (GROW ? all_b > (int64_t)top : top + (int64_t)all_b > p.n_free) bad |= LTX_BLOCKS_FREE;
  if (GROW && all_t > p.tokens) bad |= LTX_BLOCKS_TOKENS;
  const bool keeper = p.books && blockIdx.x == 0;

  if (__syncthreads_or(bad)) {  // everything stays as it is, no token has a slot
    int all = 0;
    for (int bit : {LTX_BLOCKS_FREE, LTX_BLOCKS_WIDTH, LTX_BLOCKS_TOKENS, LTX_BLOCKS_LENGTH})
      all |= __syncthreads_or(bad & bit) ? bit : 0;
    for (int b = b0; keeper && b < b1; ++b) {
      if (p.lens_out != p.lens) p.lens_out[b] = p.lens[b];
      if (GROW) p.starts[b] = 0;
    }
    if (keeper && tid == 0) {
      if (GROW) p.starts[p.B] = 0;
      *p.top_out = top;
      *p.status |= all;
    }
    if (GROW && p.place)
      for (int i = 0; i < kTableTokens / kTableThreads; ++i) {
        const int64_t t = (int64_t)blockIdx.x * kTableTokens + i * kTableThreads + tid;
        if (t < p.tokens) p.slots[t] = -1, p.positions[t] = 0;
      }
    return;
  }

  // from here on every sum is at most n_free or tokens, both below 2^31
  int at_b = (int)(sum_b - blocks), at_t = (int)(sum_t - tokens);
  for (int b = b0; b < b1; ++b) {
    const int len = p.lens[b], add = GROW ? p.fresh[b] : 0;
    const bool mine = GROW || p.done[b] != 0;
    s_blocks[b] = at_b;
    s_tokens[b] = at_t;
    s_len[b] = len;
    if (keeper) {
      if (GROW) p.starts[b] = at_t;
      p.lens_out[b] = GROW ? len + add : mine ? 0 : len;
    }
    at_b += (int)(GROW ? blocks_of((int64_t)len + add) - blocks_of(len) : mine ? blocks_of(len) : 0);
    at_t += add;
  }
  if (keeper && tid == 0) {
    if (GROW) p.starts[p.B] = (int)all_t;
    *p.top_out = GROW ? top - (int)all_b : top + (int)all_b;
  }
  __syncthreads();

  if (!p.place) return;

  if (GROW) {
    // ---- new table entries, shared by all workgroups ----
    for (int64_t e = (int64_t)blockIdx.x * kTableThreads + tid; e < all_b; e += (int64_t)gridDim.x * kTableThreads) {
      const int b = last_at_most(s_blocks, p.B, (int)e);
      const int j = (int)blocks_of(s_len[b]) + (int)e - s_blocks[b];
      p.tables[b * p.t_bs + j] = p.free_list[top - 1 - e];
    }
    // ---- slots and positions of this workgroup's tokens ----
    const int64_t t0 = (int64_t)blockIdx.x * kTableTokens + tid;
#pragma unroll
    for (int i = 0; i < kTableTokens / kTableThreads; ++i) {
      const int64_t t = t0 + i * kTableThreads;
      if (t >= p.tokens) break;
      int64_t slot = -1;
      int pos = 0;
      if (t < all_t) {
        const int b = last_at_most(s_tokens, p.B, (int)t);
        pos = s_len[b] + (int)t - s_tokens[b];
        const int j = pos >> p.shift, held = (int)blocks_of(s_len[b]);
        const int id = j < held ? p.tables[b * p.t_bs + j] : p.free_list[top - 1 - s_blocks[b] - (j - held)];
        slot = ((int64_t)id << p.shift) + (pos & (block - 1));
      }
      p.slots[t] = slot;
      p.positions[t] = pos;
    }
  } else {
    for (int64_t e = (int64_t)blockIdx.x * kTableThreads + tid; e < all_b; e += (int64_t)gridDim.x * kTableThreads) {
      const int b = last_at_most(s_blocks, p.B, (int)e);
      p.free_list[top + e] = p.tables[b * p.t_bs + (e - s_blocks[b])];
    }
  }
}

// --------------------------------------------------------------------------
// Writes of new tokens into their slots.
//
// A row is one token's D values of one head, D / 8 lanes of 8 values each.
// Rows run over the tokens of a head first: consecutive tokens mostly lie in
// one block, whose rows of a head are consecutive in the usual layout, so a
// wave's stores cover whole lines.  8-bit rows carry a float32 scale each,
// maximum / 448 (1 for a row of zeros): the maximum is taken over the row's
// lanes by lane exchanges, and the quotient is rounded once to e4m3.
// Bound by HBM: every value is read once and written once.
// --------------------------------------------------------------------------
struct PagedAppend {
  const uint16_t* src[2];
  int64_t s_ls[2], s_hs[2];
  void* dst[2];
  int64_t d_ps[2], d_ts[2], d_hs[2];
  float* scales[2];
  int64_t sc_ps[2], sc_ts[2], sc_hs[2];
  const int64_t* slots;
  int64_t T, n_slots;
  int H, shift;
};

// Largest value of N neighbouring lanes (N a power of two up to 16), in all of them.
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
  for (int d = 1; d < N; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

template <int D, bool FP8>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppend a) {
  constexpr int CPR = D / 8, ROWS = 256 / CPR;
  const int h = blockIdx.y, c = threadIdx.x % CPR;
  const int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / CPR;
  if (t >= a.T) return;  // whole rows leave: the lanes of a row stay together
  const int64_t slot = a.slots[t];
  uint4 raw[2];
#pragma unroll
  for (int w = 0; w < 2; ++w)
    raw[w] = *reinterpret_cast<const uint4*>(a.src[w] + t * a.s_ls[w] + h * a.s_hs[w] + c * 8);
  if (slot < 0 || slot >= a.n_slots) return;
  const int64_t page = slot >> a.shift, off = slot & (((int64_t)1 << a.shift) - 1);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int64_t at = page * a.d_ps[w] + off * a.d_ts[w] + h * a.d_hs[w] + c * 8;
    if constexpr (!FP8) {
      store_stream(static_cast<uint16_t*>(a.dst[w]) + at, raw[w]);
    } else {
      const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[2 * i] = bf16_bits_to_f32(u[i]), x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      // the largest finite magnitude; NaN and infinities become NaN in their places
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]) < __builtin_inff() ? fabsf(x[i]) : 0.0f);
      top = lanes_max<CPR>(top);
      const float sc = top > 0.0f ? __fdiv_rn(top, 448.0f) : 1.0f;
      float q[8];
      quotients_e4m3_bf16(x, sc, __fdiv_rn(1.0f, sc), top >= kCorrectedMinMax, q);
      uint2 codes;
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      codes.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
      int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
      codes.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
      store_stream(static_cast<uint8_t*>(a.dst[w]) + at, codes);
      if (c == 0) a.scales[w][page * a.sc_ps[w] + off * a.sc_ts[w] + h * a.sc_hs[w]] = sc;
    }
  }
}

}  // namespace ltx

using namespace ltx;

static int block_shift(int64_t block) {
  for (int s = 4; s <= 8; ++s)
    if (block == (int64_t)1 << s) return s;
  return -1;
}

static int check_tables(const char* name, int64_t B, int64_t width, int64_t t_bs, int64_t block, int64_t n_free,
                        int64_t tokens) {
  LTX_REQUIRE(B >= 0 && B <= LTX_MAX_REQUESTS, "%s: %lld requests, at most %d", name, (long long)B, LTX_MAX_REQUESTS);
  LTX_REQUIRE(block_shift(block) > 0, "%s: block of %lld tokens (16, 32, 64, 128 or 256)", name, (long long)block);
  LTX_REQUIRE(width >= 0 && width * block <= 0x7FFFFFFF, "%s: %lld blocks a request hold more than 2^31 - 1 tokens", name,
              (long long)width);
  LTX_REQUIRE(B <= 1 || t_bs >= width, "%s: table rows overlap", name);
  LTX_REQUIRE(n_free >= 0 && n_free <= 0x7FFFFFFF, "%s: bad number of blocks", name);
  LTX_REQUIRE(tokens >= 0 && tokens <= 0x7FFFFFFF, "%s: bad number of tokens", name);
  return LTX_OK;
}

// lens_out and top_out may be the inputs themselves: workgroup 0 would then
// change what others still read, so where there are others the books are kept
// by a second launch after them.
template <bool GROW>
static int run_tables(TableParams p, int64_t groups, hipStream_t st, const char* name) {
  const bool in_place = p.lens_out == p.lens || p.top_out == p.top;
  const dim3 grid((unsigned)(groups > 1 ? groups : 1)), threads(kTableThreads);
  const bool two = groups > 1 && in_place;
  p.place = 1, p.books = !two;
  hipLaunchKernelGGL((block_table_kernel<GROW>), grid, threads, 0, st, p);
  if (two) {
    p.place = 0, p.books = 1;
    hipLaunchKernelGGL((block_table_kernel<GROW>), dim3(1), threads, 0, st, p);
  }
  LTX_LAUNCH_CHECK(name);
  return LTX_OK;
}

extern "C" int ltx_kv_block_grow(int64_t B, int64_t width, int64_t block, int32_t* tables, int64_t t_bs,
                                 const int32_t* lens, const int32_t* fresh, const int32_t* free_list, int64_t n_free,
                                 const int32_t* top, int32_t* status, int64_t tokens, int32_t* lens_out,
                                 int32_t* top_out, int32_t* starts, int64_t* slots, int32_t* positions, void* stream) {
  clear_error();
  if (const int rc = check_tables("ltx_kv_block_grow", B, width, t_bs, block, n_free, tokens)) return rc;
  LTX_REQUIRE(top && status && top_out && starts && (B == 0 || (lens && fresh && lens_out)) &&
                  (B == 0 || width == 0 || tables) && (n_free == 0 || free_list) && (tokens == 0 || (slots && positions)),
              "ltx_kv_block_grow: null pointer");
  TableParams p{};
  p.tables = tables, p.t_bs = t_bs, p.lens = lens, p.fresh = fresh;
  p.free_list = const_cast<int32_t*>(free_list), p.top = top, p.status = status;
  p.lens_out = lens_out, p.top_out = top_out, p.starts = starts, p.slots = slots, p.positions = positions;
  p.tokens = tokens, p.n_free = n_free, p.B = (int)B, p.width = (int)width, p.shift = block_shift(block);
  return run_tables<true>(p, ceil_div(tokens, kTableTokens), reinterpret_cast<hipStream_t>(stream), "ltx_kv_block_grow");
}

extern "C" int ltx_kv_block_release(int64_t B, int64_t width, int64_t block, const int32_t* tables, int64_t t_bs,
                                    const int32_t* lens, const uint8_t* done, int32_t* free_list, int64_t n_free,
                                    const int32_t* top, int32_t* status, int32_t* lens_out, int32_t* top_out,
                                    void* stream) {
  clear_error();
  if (const int rc = check_tables("ltx_kv_block_release", B, width, t_bs, block, n_free, 0)) return rc;
  LTX_REQUIRE(top && status && top_out && (B == 0 || (lens && done && lens_out)) && (B == 0 || width == 0 || tables) &&
                  (n_free == 0 || free_list),
              "ltx_kv_block_release: null pointer");
  TableParams p{};
  p.tables = const_cast<int32_t*>(tables), p.t_bs = t_bs, p.lens = lens, p.done = done;
  p.free_list = free_list, p.top = top, p.status = status, p.lens_out = lens_out, p.top_out = top_out;
  p.n_free = n_free, p.B = (int)B, p.width = (int)width, p.shift = block_shift(block);
  // how many blocks come back is known on the device only: at most all of the
  // tables; 64 workgroups take turns where there are more than one round of them
  const int64_t most = ceil_div(B * width < n_free ? B * width : n_free, kTableTokens);
  return run_tables<false>(p, most < 64 ? most : 64, reinterpret_cast<hipStream_t>(stream), "ltx_kv_block_release");
}

extern "C" int ltx_kv_paged_append(int kv_dtype, int64_t T, int64_t H, int64_t D, const void* k, int64_t k_ls,
                                   int64_t k_hs, const void* v, int64_t v_ls, int64_t v_hs, void* k_pool, int64_t kp_ps,
                                   int64_t kp_ts, int64_t kp_hs, void* v_pool, int64_t vp_ps, int64_t vp_ts,
                                   int64_t vp_hs, float* k_scales, int64_t ks_ps, int64_t ks_ts, int64_t ks_hs,
                                   float* v_scales, int64_t vs_ps, int64_t vs_ts, int64_t vs_hs, int64_t n_blocks,
                                   int64_t block, const int64_t* slots, void* stream) {
  clear_error();
  const char* const name = "ltx_kv_paged_append";
  LTX_REQUIRE(T >= 0 && H >= 1 && H <= 65535 && (D == 64 || D == 128), "%s: bad shape (D 64 or 128)", name);
  LTX_REQUIRE(kv_dtype == LTX_BF16 || kv_dtype == LTX_F8E4M3, "%s: pools are bf16 or e4m3", name);
  LTX_REQUIRE(block_shift(block) > 0, "%s: block of %lld tokens (16, 32, 64, 128 or 256)", name, (long long)block);
  LTX_REQUIRE(n_blocks >= 0 && n_blocks <= 0x7FFFFFFF, "%s: bad number of blocks", name);
  if (T == 0 || n_blocks == 0) return LTX_OK;
  const bool fp8 = kv_dtype == LTX_F8E4M3;
  LTX_REQUIRE(k && v && k_pool && v_pool && slots && (!fp8 || (k_scales && v_scales)), "%s: null pointer", name);
  auto al = [](const void* p, int64_t bytes, std::initializer_list<int64_t> strides, int64_t elems) {
    bool ok = (uintptr_t)p % bytes == 0;
    for (int64_t s : strides) ok = ok && s % elems == 0;
    return ok;
  };
  LTX_REQUIRE(al(k, 16, {k_ls, k_hs}, 8) && al(v, 16, {v_ls, v_hs}, 8), "%s: rows of k and v must be 16-byte aligned", name);
  LTX_REQUIRE(al(k_pool, fp8 ? 8 : 16, {kp_ps, kp_ts, kp_hs}, 8) && al(v_pool, fp8 ? 8 : 16, {vp_ps, vp_ts, vp_hs}, 8),
              "%s: rows of the pools must be %d-byte aligned", name, fp8 ? 8 : 16);
  PagedAppend a{};
  a.src[0] = static_cast<const uint16_t*>(k), a.s_ls[0] = k_ls, a.s_hs[0] = k_hs;
  a.src[1] = static_cast<const uint16_t*>(v), a.s_ls[1] = v_ls, a.s_hs[1] = v_hs;
  a.dst[0] = k_pool, a.d_ps[0] = kp_ps, a.d_ts[0] = kp_ts, a.d_hs[0] = kp_hs;
  a.dst[1] = v_pool, a.d_ps[1] = vp_ps, a.d_ts[1] = vp_ts, a.d_hs[1] = vp_hs;
  a.scales[0] = k_scales, a.sc_ps[0] = ks_ps, a.sc_ts[0] = ks_ts, a.sc_hs[0] = ks_hs;
  a.scales[1] = v_scales, a.sc_ps[1] = vs_ps, a.sc_ts[1] = vs_ts, a.sc_hs[1] = vs_hs;
  a.slots = slots, a.T = T, a.n_slots = n_blocks * block, a.H = (int)H, a.shift = block_shift(block);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t groups = ceil_div(T, 256 / (D / 8));
  LTX_REQUIRE(groups < (1 << 24), "%s: too many tokens", name);  // 2^32 threads
  const dim3 grid((unsigned)groups, (unsigned)H), threads(256);
  if (D == 128) {
    if (fp8) hipLaunchKernelGGL((paged_append_kernel<128, true>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<128, false>), grid, threads, 0, st, a);
  } else {
    if (fp8) hipLaunchKernelGGL((paged_append_kernel<64, true>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<64, false>), grid, threads, 0, st, a);
  }
  LTX_LAUNCH_CHECK(name);
  return LTX_OK;
}
