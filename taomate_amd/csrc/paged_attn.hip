// Attention of one new token of each request over its blocks of a paged KV cache.
//
// out[b, h] = sum_j softmax_j(scale q[b, h] . k[b, j, h / G]) v[b, j, h / G]
// over the len[b] tokens that the request's blocks hold, G query heads to a
// key head.  Every cached byte is read once, so HBM bounds it.
//
// Matrix-core mapping (v_mfma_f32_16x16x32_bf16; lane l, c = l % 16, g = l / 16).
// The up to 16 query heads of one key head are the columns; a wave takes 32
// keys at a time, straight from memory to registers, nothing through LDS:
//   S = K Q^T: A = K rows (lane: row c of a 16-key half, 8 channels of group
//   g), B = Q^T.  The accumulator gives lane (c, g) head c and the keys
//   4 g + i of each half.
//   O^T += V^T P^T: B = P from the softmax registers: the product sums over
//   keys, so its k index (g, 4 half + i) may stand for key 16 half + 4 g + i,
//   which the lane has.  A = V^T wants 8 keys of one channel in a lane; lane
//   (c, g) loads its D / 16 channels of those 8 keys (a load instruction covers
//   four whole rows) and v_perm_b32 turns the 8 x D/16 block in registers.
// Wide loads of whole rows, no barrier in the key loop, the next 32 keys'
// loads in flight under this one's arithmetic: 32 KB a wave, 256 KB a CU.
//
// 8-bit caches: codes are decoded to bf16 (exact) in registers, the K scales
// multiply the scores and the V scales P, both in float32.
//
// Softmax statistics, P's sum and O are float32; P goes into its product as two
// bf16 parts (2^-16 of each weight; one part, 2^-8, is at most 1 % faster where
// memory bounds the kernel).

#include "attn_common.h"

namespace ltx {

constexpr int kTokenWaves = 4;                // waves of a workgroup (1 where no request holds many tokens)
constexpr int kTokenTile = 32 * kTokenWaves;  // keys of one step of such a workgroup

struct PagedAttn {
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  int64_t q_bs, q_hs, o_bs, o_hs;
  const char *k, *v;           // pools; strides in bytes
  int64_t k_ps, k_hs, v_ps, v_hs;
  int k_ts, v_ts;
  const float *k_sc, *v_sc;    // scales: tokens of a block contiguous
  int64_t sc_ps, sc_hs;
  const int32_t *tables, *lens;
  int64_t t_bs;
  int B, Hk, G, groups;        // groups of up to 16 query heads to a key head
  int width, shift, n_blocks;
  float scale_log2;
  // split form: `ranges` equal shares of all requests' tiles, each at least min_tiles
  int ranges, min_tiles, part_heads;
  float *part_o, *part_ml;     // [range][key head group][2][part_heads][D], [..][2]
  int4* joins;                 // [range]: the request that range continues first (-1: none), its ranges, its first slot
};

// Reads of the cache.  NT: the tables could name more than the last-level cache
// holds: non-temporal loads, which pass the caches by (a plain read of 1 GiB runs at 7.0
// TB/s with them and at 6.2 without; 64 requests over 375 MB 68.8 us and
// 76.3, four over 840 MB of e4m3 139 and 150).  A smaller cache that the last
// step left in the last-level cache is slower so (10 MB: 10.5 us and 8.2).
// The tables' width bounds what is read, and mostly from far above; a bound by the
// pool as well would be closer and is not better, since the layers of a model take
// turns and none finds its blocks in that cache again (tables of 16384 tokens, 8
// heads x 128: 64 requests of 900, 243 MB, six layers in turn 44 us and 49, one
// layer alone 43 and 40; 64 of 300, twelve layers 19 and 21, one 18 and 18.5).
// Rows that share blocks (64 rows over 4096 tokens) take 96 us either way.
constexpr int64_t kLastLevelBytes = 256 << 20;
template <bool NT, typename T>
__device__ __forceinline__ T load_cached(const char* p) {
  typedef unsigned int vec_t __attribute__((ext_vector_type(sizeof(T) / 4)));
  const vec_t* const v = reinterpret_cast<const vec_t*>(p);
  return __builtin_bit_cast(T, NT ? __builtin_nontemporal_load(v) : *v);
}

template <int D, bool FP8>
struct TokenTile {
  static constexpr int KN = FP8 ? D / 64 : D / 32;        // 16-byte loads of a K row's lane
  static constexpr int VW = (D / 16) * (FP8 ? 1 : 2) / 4;  // words of a V row's lane
  uint4 k[2][KN];
  uint32_t v[2][4][VW];
  f32x4_t ks[2], vs[2];
};

// The first tile of every request among all requests' tiles (one at least a
// request, so that an empty one's result is written too), first[B] their
// number: a scan by 256 threads.
__device__ __forceinline__ int first_tiles(const PagedAttn& p, int* first) {
  __shared__ uint32_t s_wave[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (p.B + 255) / 256, b0 = tid * each, b1 = min(b0 + each, p.B);
  const int capacity = p.width << p.shift;
  auto tiles = [&](int b) { return max(1, (min(max(p.lens[b], 0), capacity) + kTokenTile - 1) / kTokenTile); };
  uint32_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles(b);
  uint32_t sum = wave_scan(mine);
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) sum += s_wave[w];
    all += s_wave[w];
  }
  int at = (int)(sum - mine);
  for (int b = b0; b < b1; ++b) {
    first[b] = at;
    at += tiles(b);
  }
  if (tid == 0) first[p.B] = all;
  __syncthreads();
  return all;
}

// e4m3 codes of bytes 0-1 / 2-3 of a word as a bf16 pair (exact).
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}

template <int D, bool FP8, bool SPLIT, bool NT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) paged_attn_kernel(const PagedAttn p) {
  using Tile = TokenTile<D, FP8>;
  static_assert(!SPLIT || WAVES == kTokenWaves, "shares are counted in kTokenTile");
  constexpr int TILE = 32 * WAVES;  // keys of one step
  constexpr int KS = D / 32;        // 32-channel steps of a score
  constexpr int DV = D / 16;        // channels of a lane's V block = 16-channel tiles of O
  constexpr int OS = D + 4;         // row stride of the joined O in LDS
  constexpr int EB = FP8 ? 1 : 2;   // bytes of a cached value
  __shared__ __attribute__((aligned(16))) float s_o[WAVES][16][OS];
  __shared__ float s_ml[WAVES][16][2];
  extern __shared__ int s_first[];  // SPLIT: first tile of each request

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = (int)blockIdx.x / p.groups, grp = (int)blockIdx.x % p.groups;
  const int h0 = kvh * p.G + grp * 16, nh = min(16, p.G - grp * 16);
  const int capacity = p.width << p.shift;
  const int block_mask = (1 << p.shift) - 1;

  const char* const kh = p.k + kvh * p.k_hs;
  const char* const vh = p.v + kvh * p.v_hs;
  const int k_lane = c * p.k_ts + g * 16;
  const int v_lane = 4 * g * p.v_ts + c * (DV * EB);

  auto length = [&](int b) { return min(max(p.lens[b], 0), capacity); };

  // keys [t0, t1) tiles of request b: the four waves' shares joined, then
  // written as the result (slot < 0) or as a partial one
  auto attend = [&](int b, int t0, int t1, int slot) {
    const int32_t* const row = p.tables + b * p.t_bs;
    const int key_w = t0 * TILE + wave * 32;  // this wave's first key
    // the block ids of this wave's next 32 tiles, two halves each, one a lane
    auto ids_of = [&](int i) {
      const int64_t key = (int64_t)key_w + (int64_t)(i + (lane >> 1)) * TILE + (lane & 1) * 16;
      const int64_t j = key >> p.shift;
      return row[j < p.width ? j : p.width - 1];
    };
    int ids = ids_of(0), ids_next = 0;  // before the length is known: one wait for both

    bf16x8_t qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = FP8 ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (c < nh) x = *reinterpret_cast<const uint4*>(p.q + b * p.q_bs + (h0 + c) * p.q_hs + d);
      qf[s] = __builtin_bit_cast(bf16x8_t, x);
    }

    const int len = __builtin_amdgcn_readfirstlane(length(b));
    const int end = min(len, t1 * TILE);
    const int n = end > key_w ? (end - key_w + TILE - 1) / TILE : 0;
    if (n > 32) ids_next = ids_of(32);

    // tile i's loads; lim[t]: how many keys of half t take part
    auto load = [&](Tile& x, int (&lim)[2], int i) {
      if (i > 0 && (i & 31) == 0) {
        ids = ids_next;
        if (i + 32 < n) ids_next = ids_of(i + 32);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key0 = key_w + i * TILE + t * 16;
        int id = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + t);
        const bool there = (unsigned)id < (unsigned)p.n_blocks;  // an id outside the pool: keys that take no part
        lim[t] = there ? min(max(end - key0, 0), 16) : 0;
        id = there ? id : 0;
        const int off = key0 & block_mask;
        const char* const kb = kh + (int64_t)id * p.k_ps + (int64_t)off * p.k_ts;
        const char* const vb = vh + (int64_t)id * p.v_ps + (int64_t)off * p.v_ts;
#pragma unroll
        for (int s = 0; s < Tile::KN; ++s) x.k[t][s] = load_cached<NT, uint4>(kb + k_lane + s * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char* const a = vb + v_lane + r * p.v_ts;
          if constexpr (Tile::VW == 4) {
            const uint4 y = load_cached<NT, uint4>(a);
            x.v[t][r][0] = y.x, x.v[t][r][1] = y.y, x.v[t][r][2] = y.z, x.v[t][r][3] = y.w;
          } else if constexpr (Tile::VW == 2) {
            const uint2 y = load_cached<NT, uint2>(a);
            x.v[t][r][0] = y.x, x.v[t][r][1] = y.y;
          } else {
            x.v[t][r][0] = *reinterpret_cast<const uint32_t*>(a);
          }
        }
        if constexpr (FP8) {
          const int64_t sc = (int64_t)id * p.sc_ps + kvh * p.sc_hs + off + 4 * g;
          x.ks[t] = *reinterpret_cast<const f32x4_t*>(p.k_sc + sc);
          x.vs[t] = *reinterpret_cast<const f32x4_t*>(p.v_sc + sc);
        }
      }
    };

    f32x4_t o[DV];
#pragma unroll
    for (int e = 0; e < DV; ++e) o[e] = f32x4_t{};
    float m = -INFINITY, l = 0.0f;

    auto compute = [&](Tile& x, const int (&lim)[2]) {
#pragma clang fp contract(off)  // a score minus the maximum: both rounded alike, so that equal scores give 0
      f32x4_t s[2] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint4 a;
          if constexpr (FP8) {
            const uint4 w = x.k[t][k >> 1];
            const uint32_t lo = (k & 1) ? w.z : w.x, hi = (k & 1) ? w.w : w.y;
            a = make_uint4(fp8_pair(lo, false), fp8_pair(lo, true), fp8_pair(hi, false), fp8_pair(hi, true));
          } else {
            a = x.k[t][k];
          }
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), qf[k], s[t], 0, 0, 0);
        }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] *= p.scale_log2;
        if constexpr (FP8) s[t] *= x.ks[t];
      }
      if (lim[0] < 16 || lim[1] < 16) {
        // keys past the end: no score, and no value (memory that no token was
        // written to may hold anything, and 0 * inf is no 0)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (4 * g + r >= lim[t]) {
              s[t][r] = -INFINITY;
              if constexpr (FP8) x.vs[t][r] = 0.0f;
#pragma unroll
              for (int w = 0; w < Tile::VW; ++w) x.v[t][r][w] = 0;
            }
      }
      float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                        fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      top = quad_max(top);
      if (__builtin_amdgcn_ballot_w64(top > m)) {
        const float m_new = fmaxf(m, top);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < DV; ++e) o[e] *= alpha;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      // P in two bf16 parts, the second holding what the first rounds away
      uint32_t pw[4], pr[4];
      auto split = [&](float a, float b, uint32_t& hi, uint32_t& lo) {
        hi = pack_bf16x2(a, b);
        lo = pack_bf16x2(a - bf16_bits_to_f32(hi & 0xFFFFu), b - __uint_as_float(hi & 0xFFFF0000u));
      };
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - base);
          l += s[t][r];
        }
        if constexpr (FP8) s[t] *= x.vs[t];
        split(s[t][0], s[t][1], pw[2 * t], pr[2 * t]);
        split(s[t][2], s[t][3], pw[2 * t + 1], pr[2 * t + 1]);
      }
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, make_uint4(pw[0], pw[1], pw[2], pw[3]));
      const bf16x8_t rf = __builtin_bit_cast(bf16x8_t, make_uint4(pr[0], pr[1], pr[2], pr[3]));
#pragma unroll
      for (int e2 = 0; e2 < DV / 2; ++e2) {  // two channels at a time: the halves of one word
        uint32_t w[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) w[t][r] = FP8 ? fp8_pair(x.v[t][r][e2 >> 1], e2 & 1) : x.v[t][r][FP8 ? 0 : e2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t sel = u ? 0x07060302u : 0x05040100u;
          const uint4 a = make_uint4(
              __builtin_amdgcn_perm(w[0][1], w[0][0], sel), __builtin_amdgcn_perm(w[0][3], w[0][2], sel),
              __builtin_amdgcn_perm(w[1][1], w[1][0], sel), __builtin_amdgcn_perm(w[1][3], w[1][2], sel));
          f32x4_t& oe = o[2 * e2 + u];
          oe = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), rf, oe, 0, 0, 0);
          oe = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), pf, oe, 0, 0, 0);
        }
      }
    };

    if (n > 0) {
      Tile x, y;
      int lx[2], ly[2];
      load(x, lx, 0);
      for (int i = 0;;) {
        if (i + 1 < n) load(y, ly, i + 1);
        __builtin_amdgcn_sched_barrier(0);
        compute(x, lx);
        if (++i >= n) break;
        if (i + 1 < n) load(x, lx, i + 1);
        __builtin_amdgcn_sched_barrier(0);
        compute(y, ly);
        if (++i >= n) break;
      }
    }
    l = quad_sum(l);

    // ---- the four waves' shares: lane (c, g) holds head c, channels 4 DV g + DV r + e ----
    if (c < nh) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < DV; e += 4)
          *reinterpret_cast<f32x4_t*>(&s_o[wave][c][4 * DV * g + DV * r + e]) =
              f32x4_t{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
      if (g == 0) s_ml[wave][c][0] = m, s_ml[wave][c][1] = l;
    }
    __syncthreads();
    for (int i = tid; i < nh * (D / 4); i += 64 * WAVES) {
      const int h = i / (D / 4), d = i % (D / 4) * 4;
      float mm = s_ml[0][h][0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, s_ml[w][h][0]);
      f32x4_t acc{};
      float ll = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = mm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][h][0] - mm);
        ll += f * s_ml[w][h][1];
        acc += f * *reinterpret_cast<const f32x4_t*>(&s_o[w][h][d]);
      }
      if (SPLIT && slot >= 0) {
        const int64_t at = (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + slot) * p.part_heads + h;
        *reinterpret_cast<f32x4_t*>(p.part_o + at * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mm, ll);
      } else {
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        *reinterpret_cast<uint2*>(p.o + b * p.o_bs + (h0 + h) * p.o_hs + d) =
            make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
        if (d == 0 && p.lse != nullptr)
          p.lse[(int64_t)b * (p.Hk * p.G) + h0 + h] = (mm + __log2f(ll)) / kLog2e;
      }
    }
    __syncthreads();
  };

  if constexpr (!SPLIT) {
    attend((int)blockIdx.y, 0, (capacity + TILE - 1) / TILE, -1);
  } else {
    const int total = first_tiles(p, s_first);
    const int per = max(p.min_tiles, (total + p.ranges - 1) / p.ranges);
    const int x = (int)blockIdx.y;
    const int64_t r0 = (int64_t)x * per;
    const bool keeper = blockIdx.x == 0 && tid == 0;
    if (r0 >= total) {
      if (keeper) p.joins[x] = make_int4(-1, 0, 0, 0);
      return;
    }
    const int r1 = (int)min(r0 + per, (int64_t)total);
    int b = last_at_most(s_first, p.B, (int)r0);
    if (keeper) {  // the join's work: a request that the range before this one began
      const int st = s_first[b], xa = st / per;
      p.joins[x] = make_int4(st < r0 && xa + 1 == x ? b : -1, xa, (s_first[b + 1] - 1) / per, st == xa * per ? 0 : 1);
    }
    for (int r = (int)r0; r < r1; ++b) {
      const int st = s_first[b], en = s_first[b + 1], to = min(r1, en);
      attend(b, r - st, to - st, r == st && to == en ? -1 : r == r0 ? 0 : 1);
      r = to;
    }
  }
}

// Joins the partial results of the requests that several ranges share:
// workgroup (x, key head group, head) takes the request that range x is the
// first to continue, if there is one.  Eight teams of threads take every
// eighth partial result each.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttn p) {
  constexpr int TEAM = D / 4, TEAMS = 256 / TEAM;
  __shared__ __attribute__((aligned(16))) float s_o[TEAMS][D];
  __shared__ float s_ml[TEAMS][2];
  const int grp = (int)blockIdx.y % p.groups, kvh = (int)blockIdx.y / p.groups, h = blockIdx.z;
  const int4 job = p.joins[blockIdx.x + 1];
  const int b = job.x, xa = job.y, xb = job.z;
  if (b < 0 || grp * 16 + h >= p.G) return;

  const int team = threadIdx.x / TEAM, d = threadIdx.x % TEAM * 4;
  float m = -INFINITY, l = 0.0f;
  f32x4_t acc{};
#pragma unroll 4
  for (int i = xa + team; i <= xb; i += TEAMS) {
    const int slot = i == xa ? job.w : 0;
    const int64_t at = (((int64_t)i * gridDim.y + blockIdx.y) * 2 + slot) * p.part_heads + h;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(p.part_o + at * D + d);
    const float m_new = fmaxf(m, ml.x);
    const float fa = m_new == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
    const float fb = m_new == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m_new);
    l = l * fa + ml.y * fb;
    acc = acc * fa + o * fb;
    m = m_new;
  }
  *reinterpret_cast<f32x4_t*>(&s_o[team][d]) = acc;
  if (d == 0) s_ml[team][0] = m, s_ml[team][1] = l;
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int w = 1; w < TEAMS; ++w) m = fmaxf(m, s_ml[w][0]);
  acc = f32x4_t{};
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < TEAMS; ++w) {
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][0] - m);
    l += f * s_ml[w][1];
    acc += f * *reinterpret_cast<const f32x4_t*>(&s_o[w][d]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int head = kvh * p.G + grp * 16 + h;
  *reinterpret_cast<uint2*>(p.o + b * p.o_bs + head * p.o_hs + d) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (d == 0 && p.lse != nullptr) p.lse[(int64_t)b * (p.Hk * p.G) + head] = (m + __log2f(l)) / kLog2e;
}

}  // namespace ltx

using namespace ltx;

struct TokenPlan {
  int64_t y, ranges, min_tiles, part_heads;  // ranges 0: one workgroup a request and key head group
  bool one_wave;                             // of one wave
  int64_t parts() const { return ranges * y * 2 * part_heads; }
  int64_t bytes(int64_t D) const { return parts() * (D + 2) * 4 + ranges * 16; }
};

// Requests that can hold few tokens only take a workgroup each, one launch.  Up
// to 1024 tokens, or 512 where there are few workgroups (a CU reads no more than 60
// GB/s: one request of 1000 tokens with 8 key heads takes 12.7 us whole and 8.1 in
// shares).  Of one wave where there are more than fit at once and few steps'
// keys in each, for which four waves would mostly idle (123 requests of up to
// 60 tokens, 32 key heads: 24.9 us with four and 12.2 with one; of 250 tokens 58
// and 51; 256 of 500, 8 key heads, 83 and 94).
// Otherwise all requests' tiles are cut into equal ranges: as many as are
// resident at once (two workgroups a CU), or one a CU and down to a tile each where
// there is little to share.
// The key heads of a request start next to each other: their rows lie side by
// side in a block (256 requests of up to 1000 tokens, 32 heads, e4m3: 117 us, and
// 180 with the requests side by side).
static TokenPlan plan_token(int64_t B, int64_t Hk, int64_t G, int64_t capacity) {
  const int64_t tiles = ceil_div(capacity, kTokenTile), groups = ceil_div(G, 16), y = Hk * groups;
  TokenPlan t{y, 0, 1, G < 16 ? G : 16, B * y > 512 && capacity <= (B * y >= 2048 ? 256 : 128)};
  const bool little = B * tiles * y <= 1024;
  const int64_t resident = little ? 256 : 512;
  if (tiles <= (B * y <= 64 ? 4 : 8) || y >= resident) return t;
  t.min_tiles = little ? 1 : 2;
  const int64_t most = ceil_div(B * tiles, t.min_tiles);
  t.ranges = resident / y < most ? resident / y : most;
  return t;
}

extern "C" int ltx_paged_attn_workspace_size(int64_t B, int64_t Hk, int64_t G, int64_t D, int64_t width, int64_t block,
                                             int64_t* bytes) {
  clear_error();
  LTX_REQUIRE(bytes != nullptr && B >= 0 && Hk >= 1 && G >= 1 && D >= 1 && width >= 0 && block >= 1,
              "ltx_paged_attn_workspace_size: bad argument");
  const TokenPlan t = plan_token(B, Hk, G, width * block);
  *bytes = t.bytes(D);
  return LTX_OK;
}

template <int D, bool FP8, bool NT>
static void launch_token(const PagedAttn& p, const TokenPlan& t, hipStream_t st) {
  const dim3 threads(64 * kTokenWaves);
  const unsigned y = (unsigned)t.y;
  const dim3 each(y, (unsigned)p.B);
  if (t.one_wave) {
    hipLaunchKernelGGL((paged_attn_kernel<D, FP8, false, NT, 1>), each, dim3(64), 0, st, p);
    return;
  }
  if (t.ranges == 0) {
    hipLaunchKernelGGL((paged_attn_kernel<D, FP8, false, NT, kTokenWaves>), each, threads, 0, st, p);
    return;
  }
  hipLaunchKernelGGL((paged_attn_kernel<D, FP8, true, NT, kTokenWaves>), dim3(y, (unsigned)t.ranges), threads,
                     (unsigned)(p.B + 1) * 4, st, p);
  if (t.ranges > 1)
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3((unsigned)t.ranges - 1, y, (unsigned)t.part_heads), dim3(256), 0,
                       st, p);
}
template <int D, bool FP8>
static void launch_token(const PagedAttn& p, const TokenPlan& t, hipStream_t st) {
  const int64_t most = (int64_t)p.B * (p.width << p.shift) * p.Hk * 2 * D * (FP8 ? 1 : 2);
  if (most > kLastLevelBytes && p.groups == 1) launch_token<D, FP8, true>(p, t, st);
  else launch_token<D, FP8, false>(p, t, st);
}

extern "C" int ltx_paged_attn(int kv_dtype, int64_t B, int64_t Hk, int64_t G, int64_t D, const void* q, int64_t q_bs,
                              int64_t q_hs, const void* k_pool, int64_t k_ps, int64_t k_ts, int64_t k_hs,
                              const void* v_pool, int64_t v_ps, int64_t v_ts, int64_t v_hs, const float* k_scales,
                              const float* v_scales, int64_t sc_ps, int64_t sc_hs, int64_t n_blocks, int64_t block,
                              const int32_t* tables, int64_t t_bs, int64_t width, const int32_t* lens, void* out,
                              int64_t o_bs, int64_t o_hs, float* lse, float scale, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* const name = "ltx_paged_attn";
  LTX_REQUIRE(B >= 0 && B <= LTX_MAX_REQUESTS, "%s: %lld requests, at most %d", name, (long long)B, LTX_MAX_REQUESTS);
  LTX_REQUIRE(Hk >= 1 && G >= 1 && Hk * G <= 65535 && (D == 64 || D == 128), "%s: bad head layout (D 64 or 128)", name);
  LTX_REQUIRE(kv_dtype == LTX_BF16 || kv_dtype == LTX_F8E4M3, "%s: pools are bf16 or e4m3", name);
  int shift = -1;
  for (int s = 4; s <= 8; ++s)
    if (block == (int64_t)1 << s) shift = s;
  LTX_REQUIRE(shift > 0, "%s: block of %lld tokens (16, 32, 64, 128 or 256)", name, (long long)block);
  LTX_REQUIRE(n_blocks >= 1 && n_blocks <= 0x7FFFFFFF, "%s: a pool holds at least one block", name);
  LTX_REQUIRE(width >= 1 && width * block <= 0x40000000, "%s: a table row holds 1 to 2^30 tokens", name);
  LTX_REQUIRE(B * ceil_div(width * block, kTokenTile) <= 0x40000000, "%s: the tables hold too many tokens", name);
  if (B == 0) return LTX_OK;
  const bool fp8 = kv_dtype == LTX_F8E4M3;
  LTX_REQUIRE(q && k_pool && v_pool && tables && lens && out && (!fp8 || (k_scales && v_scales)), "%s: null pointer", name);
  LTX_REQUIRE((uintptr_t)q % 16 == 0 && q_bs % 8 == 0 && q_hs % 8 == 0 && (uintptr_t)out % 8 == 0 && o_bs % 4 == 0 &&
                  o_hs % 4 == 0,
              "%s: rows of q must be 16-byte and of out 8-byte aligned", name);
  const int64_t per = fp8 ? 16 : 8;
  for (int64_t s : {k_ps, k_ts, k_hs, v_ps, v_ts, v_hs})
    LTX_REQUIRE(s % per == 0, "%s: rows of the pools must be 16-byte aligned", name);
  LTX_REQUIRE((uintptr_t)k_pool % 16 == 0 && (uintptr_t)v_pool % 16 == 0, "%s: rows of the pools must be 16-byte aligned", name);
  // offsets inside a block are 32-bit
  LTX_REQUIRE(k_ts >= 0 && v_ts >= 0 && k_ts <= 0x7FFFFFFF / 64 && v_ts <= 0x7FFFFFFF / 64, "%s: bad token stride", name);
  LTX_REQUIRE(!fp8 || ((uintptr_t)k_scales % 16 == 0 && (uintptr_t)v_scales % 16 == 0 && sc_ps % 4 == 0 && sc_hs % 4 == 0),
              "%s: scales of a block and head must be 16-byte aligned", name);
  const TokenPlan t = plan_token(B, Hk, G, width * block);
  const int64_t need = t.bytes(D);
  LTX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
              "%s: needs %lld bytes of workspace", name, (long long)need);
  PagedAttn p{};
  p.q = static_cast<const uint16_t*>(q), p.q_bs = q_bs, p.q_hs = q_hs;
  p.o = static_cast<uint16_t*>(out), p.o_bs = o_bs, p.o_hs = o_hs, p.lse = lse;
  const int64_t eb = fp8 ? 1 : 2;
  p.k = static_cast<const char*>(k_pool), p.k_ps = k_ps * eb, p.k_hs = k_hs * eb, p.k_ts = (int)(k_ts * eb);
  p.v = static_cast<const char*>(v_pool), p.v_ps = v_ps * eb, p.v_hs = v_hs * eb, p.v_ts = (int)(v_ts * eb);
  p.k_sc = k_scales, p.v_sc = v_scales, p.sc_ps = sc_ps, p.sc_hs = sc_hs;
  p.tables = tables, p.t_bs = t_bs, p.lens = lens;
  p.B = (int)B, p.Hk = (int)Hk, p.G = (int)G, p.groups = (int)ceil_div(G, 16);
  p.width = (int)width, p.shift = shift, p.n_blocks = (int)n_blocks;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)D)) * kLog2e;
  p.ranges = (int)t.ranges, p.min_tiles = (int)t.min_tiles, p.part_heads = (int)t.part_heads;
  if (t.ranges > 0) {
    p.joins = static_cast<int4*>(workspace);
    p.part_o = reinterpret_cast<float*>(p.joins + t.ranges);
    p.part_ml = p.part_o + t.parts() * D;
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (D == 128) {
    if (fp8) launch_token<128, true>(p, t, st);
    else launch_token<128, false>(p, t, st);
  } else {
    if (fp8) launch_token<64, true>(p, t, st);
    else launch_token<64, false>(p, t, st);
  }
  LTX_LAUNCH_CHECK(name);
  return LTX_OK;
}
