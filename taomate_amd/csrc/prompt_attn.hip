// Attention over whole prompts: packed rows, grouped heads, causal or not.
//
// out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys of row i's own
// prompt; causal: j <= i + Lk - Lq.  4 D multiply-adds a (row, key, head), so
// the matrix cores bound it.
//
// Work decomposition.  A workgroup of 4 waves owns 128 rows of one prompt and
// head, 32 rows a wave; keys stream through LDS in tiles of 64 (double
// buffered, loaded straight to LDS).  The prompts' lengths lie on the device:
// every wave finds its workgroup's prompt and rows by a scan over the starts,
// and the grid is as large as any lengths of that sum can need.
//
// Matrix-core mapping (v_mfma_f32_16x16x32_bf16; lane l, li = l % 16, lg = l / 16):
//   S^T = K Q^T: A = K rows (LDS), B = Q^T (registers, loaded once): a lane has
//   two queries and, with K rows in the order key_of_row, 8 consecutive keys of
//   each 32: the softmax statistics are per-lane scalars.
//   O^T += V^T P^T: B = P straight from the softmax registers, A = V^T by
//   transposing LDS reads of the tile's rows.
// Softmax: base 2, log2(e) folded into the scale, running maximum and sum per
// query in float32; the maximum is raised only when a tile's sum passes 2^16
// (P then needs no rescaling of O for most tiles).  P is rounded to bf16 for
// its product (half a step, 2^-8, of each weight), its sum is not.

#include <type_traits>

#include "attn_common.h"

namespace ltx {

constexpr int kRows = 128;  // rows of a workgroup
constexpr int kKeys = 64;   // keys of a tile
constexpr int kResident = 512;  // workgroups that run at once: two a CU (64 channels: three)

struct PromptAttn {
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  int64_t q_ls, q_hs, o_ls, o_hs;
  const char *k, *v;  // strides in bytes
  int64_t k_hs, v_hs;
  int k_ls, v_ls;
  const int32_t *q_starts, *k_starts;
  int B, Tq, Tk, Hk, G, causal, zero_rest, sorted, tiles;
  float scale_log2;
  // SPLIT: a row tile's key tiles are shared by up to `split` workgroups, whose
  // results [workgroup][range][row][D] and (maximum, sum) are joined afterwards
  int split;
  float *part_o, *part_ml;
};

// Where a workgroup works: rows from row0 of a prompt whose Lq rows start at q0 and
// whose Lk keys start at k0 of the packed tensors; begin, end: the first row of
// all prompts and the first one behind them.
struct PromptRows {
  int q0, k0, row0, Lq, Lk, begin, end;
};

// Row tile t in the order in which the workgroups start: a prompt's last tile
// first (late rows of a causal prompt see the most keys), the last prompt first;
// with `sorted` (up to 64 prompts) the prompts with the most keys first, so that a
// grid of several rounds ends with its short tiles.
// False: there are fewer tiles.
__device__ __forceinline__ bool find_rows(const PromptAttn& p, int t, PromptRows& r) {
  const int lane = threadIdx.x & 63;
  r.begin = r.end = 0;
  if (p.B == 1) {  // no search: scalar loads
    r.begin = r.q0 = min(max(p.q_starts[0], 0), p.Tq);
    r.end = min(max(p.q_starts[1], r.q0), p.Tq);
    r.k0 = min(max(p.k_starts[0], 0), p.Tk);
    r.Lk = min(max(p.k_starts[1], r.k0), p.Tk) - r.k0;
    r.Lq = r.end - r.q0;
    r.row0 = ((r.Lq + kRows - 1) / kRows - 1 - t) * kRows;
    return r.row0 >= 0;
  }
  for (int b0 = p.B - 1; b0 >= 0; b0 -= 64) {
    const int b = b0 - lane;
    int s = 0, n = 0, ks = 0, m = 0;
    if (b >= 0) {
      const int s0 = p.q_starts[b], s1 = p.q_starts[b + 1], k0 = p.k_starts[b], k1 = p.k_starts[b + 1];
      s = min(max(s0, 0), p.Tq);
      n = min(max(s1, s), p.Tq) - s;
      ks = min(max(k0, 0), p.Tk);
      m = min(max(k1, ks), p.Tk) - ks;
    }
    if (b0 == p.B - 1) {
      r.end = __builtin_amdgcn_readfirstlane(s + n);
      r.begin = p.B <= 64 ? __builtin_amdgcn_readlane(s, p.B - 1) : min(max(p.q_starts[0], 0), p.Tq);
    }
    if (p.sorted) {
      // by powers of two of their number of key tiles: the longest three, then the others
      const int mine = lane < p.B ? 32 - __builtin_clz(m / kKeys + 1) : 0;
      const int longest = wave_max(mine);
      int rank = lane, before = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool here = lane < p.B && (c < 3 ? mine == longest - c : mine < longest - 2);
        const uint64_t all = __builtin_amdgcn_ballot_w64(here);
        const int at = before + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        rank = here ? at : rank;
        before += __builtin_popcountll(all);
      }
      s = __builtin_amdgcn_ds_permute(rank * 4, s);
      n = __builtin_amdgcn_ds_permute(rank * 4, n);
      ks = __builtin_amdgcn_ds_permute(rank * 4, ks);
      m = __builtin_amdgcn_ds_permute(rank * 4, m);
    }
    const int tiles = (n + kRows - 1) / kRows;
    const int sum = (int)wave_scan((uint32_t)tiles);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum > t);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int before = __builtin_amdgcn_readlane(sum - tiles, at);
      r.q0 = __builtin_amdgcn_readlane(s, at);
      r.Lq = __builtin_amdgcn_readlane(n, at);
      r.k0 = __builtin_amdgcn_readlane(ks, at);
      r.Lk = __builtin_amdgcn_readlane(m, at);
      r.row0 = (__builtin_amdgcn_readlane(tiles, at) - 1 - (t - before)) * kRows;
      return true;
    }
    t -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The row tile and heads of a workgroup.  Workgroups are dispatched round-robin
// over the 8 XCDs.  The G heads that share a key head's keys run side by side on
// one XCD (one L2), and the XCDs take the (row tile, key head) pairs in turn, so
// each gets long and short ones.
__device__ __forceinline__ int unit_of(const PromptAttn& p, int& kvh, int& h) {
  const int slot = (int)blockIdx.x >> 3;
  const int unit = slot / p.G * 8 + ((int)blockIdx.x & 7);
  kvh = unit % p.Hk;
  h = kvh * p.G + slot % p.G;
  return unit / p.Hk;
}

// keys that some row of the tile sees
__device__ __forceinline__ int seen_keys(const PromptAttn& p, const PromptRows& w) {
  const int seen = p.causal ? min(w.Lk, min(w.Lq, w.row0 + kRows) + w.Lk - w.Lq) : w.Lk;
  return max(seen, 0);
}

// How many workgroups share a row tile that sees `seen` keys, and the key tiles of each.
constexpr int kMinPart = 4;
__device__ __forceinline__ int parts_of(const PromptAttn& p, int seen, int& tiles) {
  const int all = (seen + kKeys - 1) / kKeys;
  const int parts = max(1, min(p.split, all / kMinPart));
  tiles = (all + parts - 1) / parts;
  return tiles > 0 ? (all + tiles - 1) / tiles : 1;
}

// x where i < lim, else -inf, by bit selection: comparisons would hold a pair
// of scalar registers each, and the key loop's own would be moved out and back
// in every tile to make room.
__device__ __forceinline__ float keep_below(float x, int i, int lim) {
  const uint32_t keep = (uint32_t)((i - lim) >> 31);
  return __uint_as_float((__float_as_uint(x) & keep) | (0xFF800000u & ~keep));
}

template <int D, bool SPLIT>
__device__ __forceinline__ void prompt_body(const PromptAttn& p) {
  constexpr int BN = kKeys;
  constexpr int NKC = D / 8;             // 16-byte chunks of a row
  constexpr int BUF = BN * D;            // elements of a K or V tile buffer
  constexpr int SLOTS = BUF / 512 / 4;   // load instructions (64 chunks) per wave and tile
  constexpr int CB = D / 16;             // 16-channel blocks of O
  constexpr int KS = D / 32;             // 32-channel steps of a score
  constexpr float kOver = 65536.0f;      // largest per-lane tile sum kept without raising m
  // 64 channels: P(j) takes the registers of P(j-1), each word once its product
  // is issued, so that three workgroups fit a CU (168 registers): 24 prompts of
  // up to 1023 rows, 32 heads, 44.7 us and 51.5 with two (at the start of a run; 37.7
  // once the clock has risen); 128 channels have no use for it
  constexpr bool ONE_P = D == 64;
  constexpr float kHuge = 0x1p28f;       // |m| whose last place is 2^4 or more (exp_all)

  // K(0), K(1), V(0), V(1), one array: the output staging spans them
  __shared__ __attribute__((aligned(16))) uint16_t smem[4 * BUF];
  uint16_t* const kbuf = smem;
  uint16_t* const vbuf = smem + 2 * BUF;

  int kvh, h;
  const int unit = unit_of(p, kvh, h);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int li = lane & 15, lg = lane >> 4;
  PromptRows w;
  const bool works = find_rows(p, unit, w);
  const int rest = w.begin + p.Tq - w.end;
  if (p.zero_rest && rest > 0 && (!SPLIT || blockIdx.y == 0)) {
    // rows before and behind the prompts, shared by all row tiles
    for (int64_t row0 = (int64_t)unit * kRows; row0 < rest; row0 += (int64_t)p.tiles * kRows)
      for (int i = threadIdx.x; i < kRows * NKC; i += 256) {
        int64_t row = row0 + i / NKC;
        if (row >= rest) break;
        if (row >= w.begin) row += w.end - w.begin;
        *reinterpret_cast<uint4*>(p.o + row * p.o_ls + h * p.o_hs + i % NKC * 8) = make_uint4(0, 0, 0, 0);
        if (p.lse != nullptr && i % NKC == 0) p.lse[(int64_t)h * p.Tq + row] = -INFINITY;
      }
  }
  if (!works) return;
  const int q0 = w.row0 + wave * 32 + li;  // this lane's queries: q0 and q0 + 16
  int shift = w.Lk - w.Lq;                 // causal: row i sees keys up to i + shift
  int seen = seen_keys(p, w);
  int parts = 1;
  if constexpr (SPLIT) {
    // this workgroup's share: the prompt without the keys before and after it
    int tiles;
    parts = parts_of(p, seen, tiles);
    if ((int)blockIdx.y >= parts) return;
    const int skip = (int)blockIdx.y * tiles * BN;
    w.k0 += skip;
    w.Lk -= skip;
    shift -= skip;
    seen = min(seen - skip, tiles * BN);
  }
  const int ntiles = (seen + BN - 1) / BN;
  // of this wave: past the last key of its rows, or without rows, it only
  // takes part in the loads
  const int row_w = w.row0 + wave * 32;
  const int wave_seen = row_w >= w.Lq ? 0 : p.causal ? min(seen, row_w + 32 + shift) : seen;
  const int wtiles = max(1, (max(wave_seen, 0) + BN - 1) / BN);

  // ---- per-lane load offsets (bytes from a tile's first key), loop invariant:
  // slot i of wave w fills LDS chunks (w + 4 i) * 64 + lane, a uniform number
  // of keys further than slot 0 ----
  const int krow0 = (wave * 64 + lane) / NKC;
  const int koff = key_of_row(krow0) * p.k_ls + ((lane % NKC) ^ row_swizzle<NKC>(krow0)) * 16;
  const int voff = krow0 * p.v_ls + ((lane % NKC) ^ key_swizzle<NKC>(krow0)) * 16;
  const char* kptr = p.k + kvh * p.k_hs + (int64_t)w.k0 * p.k_ls;
  const char* vptr = p.v + kvh * p.v_hs + (int64_t)w.k0 * p.v_ls;
  int krem = seen, vrem = seen;  // seen keys from the next K (V) tile on
  auto lds_slot0 = [&](uint16_t* buf0) {
    uint32_t a = (uint32_t)(uintptr_t)(lds_ptr_t)(buf0 + wave * 512);
    asm volatile("" : "+s"(a));  // one address, not one scalar register for each slot and buffer
    return a;
  };
  // A tile's loads.  Rows past the last key that any row here sees lie outside the
  // partial tile's buffer range: those lanes load zeros, so nothing of later keys, of
  // the next prompt or of memory behind the tensor is read, and their scores are
  // masked.  A whole
  // tile's slots take their uniform offset from a scalar register; a partial
  // tile adds it per lane, so that the range check sees all of it.
  auto issue = [&](uint16_t* buf0, const char*& ptr, int& rem, int off0, int row_bytes, auto keys_of_slot) {
    const uint32_t l0 = lds_slot0(buf0);
    if (rem >= BN) {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)ptr, (short)0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(uintptr_t)(l0 + i * 4096), 16, off0,
                                                 keys_of_slot(i) * row_bytes, 0, 0);
    } else {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)ptr, (short)0, max(rem, 0) * row_bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(uintptr_t)(l0 + i * 4096), 16,
                                                 off0 + keys_of_slot(i) * row_bytes, 0, 0, 0);
    }
    rem -= BN;
    ptr += (int64_t)BN * row_bytes;
  };
  auto issue_k = [&](int buf) {
    issue(kbuf + buf * BUF, kptr, krem, koff, p.k_ls, [](int i) { return key_of_row(i * (256 / NKC)); });
  };
  auto issue_v = [&](int buf) {
    issue(vbuf + buf * BUF, vptr, vrem, voff, p.v_ls, [](int i) { return i * (256 / NKC); });
  };

  // ---- Q^T fragments, resident for the whole key loop ----
  bf16x8_t qf[2][KS];
  auto load_q = [&]() {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int qi = q0 + 16 * n;
      const bool ok = qi < w.Lq;
      const uint16_t* qp = p.q + (int64_t)(w.q0 + (ok ? qi : 0)) * p.q_ls + h * p.q_hs + lg * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint4 v = ok ? *reinterpret_cast<const uint4*>(qp + s * 32) : make_uint4(0, 0, 0, 0);
        qf[n][s] = __builtin_bit_cast(bf16x8_t, v);
      }
    }
  };

  f32x4_t oacc[CB][2];
#pragma unroll
  for (int d = 0; d < CB; ++d) oacc[d][0] = oacc[d][1] = f32x4_t{};
  const float c = p.scale_log2;  // > 0
  float m_run[2] = {-INFINITY, -INFINITY};  // per query, base-2 logit units
  float l_run[2] = {0.0f, 0.0f};            // this lane's share of the row sums

  // Scores: s[kb][n][r] is query q0 + 16 n over key 32 (kb / 2) + 8 lg + 4 (kb % 2) + r
  // of the tile; score pair q (two adjacent r) of the softmax and of P is
  // kb = 2 (q / 8) + (q % 4) / 2, n = (q / 4) % 2, r = 2 (q % 2) + {0, 1},
  // so P words 8 k2 + 4 n .. + 3 are the B operand of key half k2.
  // Tile j's keys that a query does not see drop out of its softmax.  Only a
  // prompt's last tile and the tiles on the diagonal of this wave's rows need it.
  auto mask = [&](f32x4_t (&s)[4][2], int j) {
    const int end = w.Lk - j * BN, first = w.row0 + wave * 32 + shift + 1 - j * BN;  // of the wave's first row
    if (end >= BN && (!p.causal || first >= BN)) return;
    const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));  // rare: no register held for it
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int lim = (p.causal ? min(end, first + (ln & 15) + 16 * n) : end) - 8 * (ln >> 4);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[kb][n][r] = keep_below(s[kb][n][r], 32 * (kb >> 1) + 4 * (kb & 1) + r, lim);
    }
  };
  // Largest base-2 logit of a tile for this lane's query n; a row that sees
  // no key of it has the lowest number: its weights are 2^-inf = 0, and the
  // first key that it does see passes any sum and raises it.
  auto tile_max = [&](const f32x4_t (&s)[4][2], int n) {
    float mt = s[0][n][0];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[kb][n][r]);
    return fmaxf(quad_max(mt) * c, -3.0e38f);
  };
  // P = 2^(S*c + neg_m) of query n packed to bf16 pairs; returns this lane's
  // sum of the values before they are rounded.  Used outside the slot program
  // (first tile, raised maximum).  S*c - m in one rounding is the better
  // difference, but m is a rounded S*c itself: where its last place is worth more than
  // kOver's exponent, equal scores would weigh 0 or infinity.  There the
  // product is rounded first, as m was (and `over` sends every tile here).
  auto exp_all = [&](const f32x4_t (&s)[4][2], uint32_t (&pw)[16], int n, float neg_m) {
#pragma clang fp contract(off)
    float ps = 0.0f;
    const bool huge = fabsf(neg_m) > kHuge;
    auto arg = [&](float x) {
      const float rounded = x * c;
      return huge ? rounded + neg_m : __builtin_fmaf(x, c, neg_m);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int q = (i >> 2) * 8 + n * 4 + (i & 3), kb = 2 * (q >> 3) + ((q & 3) >> 1), r = 2 * (q & 1);
      const float p0 = __builtin_amdgcn_exp2f(arg(s[kb][n][r]));
      const float p1 = __builtin_amdgcn_exp2f(arg(s[kb][n][r + 1]));
      pw[q] = pack_bf16x2(p0, p1);
      ps += p0 + p1;
    }
    return ps;
  };
  // Fragments: lane (li, lg) reads row li of a 16-row block, 16-byte chunk
  // 4 * step + lg, stored at the chunk index xor the row's swizzle.  The
  // blocks' row offsets are multiples of 16 rows and a step only flips offset
  // bits (4 chunks = 32 elements), so one offset per operand serves every
  // fragment.
  const int kofs = li * D + (lg ^ row_swizzle<NKC>(li)) * 8;
  auto kfrag = [&](int buf, int kb, int s) -> bf16x8_t {
    return *reinterpret_cast<const bf16x8_t*>(kbuf + buf * BUF + kb * 16 * D + (kofs ^ (s * 32)));
  };
  // V tiles hold keys in rows, so a V^T fragment is read with the
  // transposing LDS read: the 16 lanes of one lg read a block of 4 keys x 16
  // channels (8 bytes per lane) and lane li receives its channel of the 4
  // keys; two reads give the lane's 8 keys.
  const int tofs = (8 * lg + (li >> 2)) * D + (((li >> 1) & 1) ^ key_swizzle<NKC>(8 * lg + (li >> 2))) * 8 +
                   (li & 1) * 4;
  auto vfrag = [&](int buf, int d, int k2) -> bf16x8_t {
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef short s16x8_t __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;
    uint16_t* v0 = vbuf + buf * BUF + 32 * k2 * D + (tofs ^ (16 * d));
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)v0);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(v0 + 4 * D));
    return __builtin_bit_cast(bf16x8_t, (s16x8_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto pfrag = [](const uint32_t (&pw)[16], int k2, int n) {
    const int q = 8 * k2 + 4 * n;
    return __builtin_bit_cast(bf16x8_t, make_uint4(pw[q], pw[q + 1], pw[q + 2], pw[q + 3]));
  };
  // S = K Q^T of a whole tile (first tiles only)
  auto qk_tile = [&](int buf, f32x4_t (&s)[4][2]) {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const bf16x8_t a = kfrag(buf, kb, k);
#pragma unroll
        for (int n = 0; n < 2; ++n)
          s[kb][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[n][k], k == 0 ? f32x4_t{} : s[kb][n], 0, 0, 0);
      }
  };
  // O^T += V^T P^T of a whole tile (last tile only)
  auto pv_tile = [&](int buf, const uint32_t (&pw)[16]) {
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int d = 0; d < CB; ++d) {
        const bf16x8_t a = vfrag(buf, d, k2);
#pragma unroll
        for (int n = 0; n < 2; ++n)
          oacc[d][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pfrag(pw, k2, n), oacc[d][n], 0, 0, 0);
      }
  };
  // the tile loads go straight to LDS and are counted by vmcnt, so they must
  // land before the barrier publishes them
  auto publish = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // ---- the slot program of one tile ----
  // NS slots: PV(j-1) (2*CB fragments of V(j-1)) then S(j+1) (4*KS fragments
  // of K(j+1)).  Each slot issues the two MFMAs of its fragment (the lane's
  // two queries), the LDS read of the fragment PREF slots ahead, and a slice
  // of the softmax of S(j).  With 32 slots (D = 128) that is one score per
  // slot: score i has its fma at slot i, its exp at i + 1 and its row-sum add
  // at i + 2, and pair q its bf16 pack at 2q + 3 (whole pairs per slot, fma
  // of both at 2q and the rest at 2q + 1 and 2q + 3, measured 1 % slower: the
  // odd slots then carry two exps, the adds and the pack).  With 16 slots
  // (D = 64) score pair p has its fma at slot p, its exp at p + 1 and its
  // pack and adds at p + 2.  A scheduling fence closes every slot, so the exp
  // work stays spread under the MFMAs.  The row sum adds the fp32 P
  // values: v_dot2c_f32_bf16 over the packed pair (one instruction instead
  // of two) waits for the SIMD's matrix pipeline on gfx950, about one MFMA
  // per instruction while the other wave's MFMAs run, where adds issue
  // beside them.
  constexpr int NPV = 2 * CB, NS = NPV + 4 * KS;
  constexpr int PREF = ONE_P ? 2 : 3;
  auto tile = [&](int vb, int kbf, const f32x4_t (&scur)[4][2], f32x4_t (&snext)[4][2], const uint32_t (&pprev)[16],
                  uint32_t (&pcur)[16], float (&ps)[2], const float (&neg_m)[2], auto&& loads) {
    auto frag = [&](int t) -> bf16x8_t {
      if (t < NPV) return vfrag(vb, t % CB, t / CB);
      return kfrag(kbf, (t - NPV) & 3, (t - NPV) >> 2);
    };
    bf16x8_t ring[PREF + 1];
#pragma unroll
    for (int t = 0; t < PREF; ++t) ring[t] = frag(t);
    float e0[16], e1[16];
    ps[0] = ps[1] = 0.0f;
#pragma unroll
    for (int t = 0; t < NS + 2; ++t) {
      if (t < NS) {
        if (t + PREF < NS) ring[(t + PREF) % (PREF + 1)] = frag(t + PREF);
        const bf16x8_t a = ring[t % (PREF + 1)];
        if (t == NPV - PREF) loads();
        // the query blocks alternate (0 1, 1 0, ...): consecutive MFMAs share an operand
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = i ^ (t & 1);
          if (t < NPV) {
            oacc[t % CB][n] =
                __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pfrag(pprev, t / CB, n), oacc[t % CB][n], 0, 0, 0);
          } else {
            const int kb = (t - NPV) & 3, kk = (t - NPV) >> 2;  // the four key blocks' chains alternate
            snext[kb][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[n][kk], kk == 0 ? f32x4_t{} : snext[kb][n],
                                                                   0, 0, 0);
          }
        }
      }
      if constexpr (NS == 32) {
        // one score per slot: its fma at slot i, its exp at i + 1, its
        // row-sum add at i + 2, and the bf16 pack of pair q at 2q + 3, so
        // every slot carries the same vector work
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int q = i >> 1, n = (q >> 2) & 1, kb = 2 * (q >> 3) + ((q & 3) >> 1), r = 2 * (q & 1) + (i & 1);
          float* e = (i & 1) ? e1 : e0;
          if (t == i) e[q] = __builtin_fmaf(scur[kb][n][r], c, neg_m[n]);
          if (t == i + 1) e[q] = __builtin_amdgcn_exp2f(e[q]);
          if (t == i + 2) ps[n] = ps[n] + e[q];
        }
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (t == 2 * q + 3) {
            pcur[q] = pack_bf16x2(e0[q], e1[q]);
            // with no use left in this slot the compiler would sink the pack
            // to the next tile's PV and issue all sixteen back to back after
            // the slot program; pin it here, under this slot's MFMAs
            asm volatile("" : "+v"(pcur[q]));
          }
      } else {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const int n = (q >> 2) & 1, kb = 2 * (q >> 3) + ((q & 3) >> 1), r = 2 * (q & 1);
          if ((2 * q * NS) / 32 == t) {
            e0[q] = __builtin_fmaf(scur[kb][n][r], c, neg_m[n]);
            e1[q] = __builtin_fmaf(scur[kb][n][r + 1], c, neg_m[n]);
          }
          if ((2 * q * NS) / 32 + 1 == t) {
            e0[q] = __builtin_amdgcn_exp2f(e0[q]);
            e1[q] = __builtin_amdgcn_exp2f(e1[q]);
          }
          if (t == (q < 2 ? 4 : q + 2)) {  // from slot 4 on the words of P(j-1) below 8 are free, from slot 8 on all
            pcur[q] = pack_bf16x2(e0[q], e1[q]);
            ps[n] = ps[n] + e0[q];
            ps[n] = ps[n] + e1[q];
            asm volatile("" : "+v"(pcur[q]));
          }
        }
      }
      // the slot's order: MFMA, exp, MFMA, fragment read, other vector work
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      if (t + PREF < NPV)
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      else
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (ntiles > 0) {
    f32x4_t sa[4][2], sb[4][2];
    uint32_t pa[16], pb[16];  // P(j) of even / odd j
    // ---- prologue: S(0) sets m from its own maximum; P(0); S(1) ----
    issue_k(0);
    if (ntiles > 1) issue_k(1);
    issue_v(0);
    load_q();  // its latency overlaps the first tiles' loads
    publish();
    qk_tile(0, sa);
    mask(sa, 0);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      m_run[n] = tile_max(sa, n);
      l_run[n] = exp_all(sa, pa, n, -m_run[n]);
    }
    if (ntiles > 1) qk_tile(1, sb);
    if (ntiles > 2) {
      __syncthreads();  // every wave is done with K(0)
      issue_k(0);       // K(2)
    }
    // ---- iteration j (1 <= j < ntiles), of parity jp: the slot program
    //      computes O += V(j-1)^T P(j-1), S(j+1) = K(j+1) Q^T and
    //      P(j) = 2^(S(j)c - m).  On the last tile S(j+1) is computed from
    //      stale LDS and dropped. ----
    auto step = [&](int j, auto jpar, f32x4_t (&scur)[4][2], f32x4_t (&snext)[4][2], const uint32_t (&pprev)[16],
                    uint32_t (&pcur)[16]) {
      constexpr int jp = decltype(jpar)::value;
      publish();  // K(j+1) and V(j-1) have landed; the buffers of K(j) and V(j-2) are free
      // after the tile's last V fragment read: the compiler waits for every
      // load to LDS in flight before a transposing read
      auto loads = [&]() {
        if (j + 2 < ntiles) issue_k(jp);  // K(j+2)
        issue_v(jp);                      // V(j)
      };
      mask(scur, j);
      const float neg_m[2] = {-m_run[0], -m_run[1]};
      const float over[2] = {fabsf(m_run[0]) > kHuge ? -1.0f : kOver, fabsf(m_run[1]) > kHuge ? -1.0f : kOver};
      float ps[2];
      tile(1 - jp, 1 - jp, scur, snext, pprev, pcur, ps, neg_m, loads);
      if (__builtin_amdgcn_ballot_w64(ps[0] > over[0] || ps[1] > over[1])) {
        // raise m to the tile maximum, rescale O and l, redo P(j) from S(j)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float m_new = fmaxf(m_run[n], tile_max(scur, n));
          const float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_new);
          m_run[n] = m_new;
          l_run[n] *= alpha;
#pragma unroll
          for (int d = 0; d < CB; ++d) oacc[d][n] *= alpha;
          ps[n] = exp_all(scur, pcur, n, -m_run[n]);
        }
      }
      l_run[0] += ps[0];
      l_run[1] += ps[1];
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    int j = 1;
    for (; j + 1 < wtiles; j += 2) {
      step(j, odd, sb, sa, pa, ONE_P ? pa : pb);
      step(j + 1, even, sa, sb, ONE_P ? pa : pb, pa);
    }
    if (j < wtiles) step(j, odd, sb, sa, pa, ONE_P ? pa : pb);
    // ---- the wave's last tile: O += V(n-1)^T P(n-1); then only loads for the
    //      waves whose rows see further ----
    publish();
    if ((wtiles - 1) & 1)
      pv_tile(1, ONE_P ? pa : pb);
    else
      pv_tile(0, pa);
    for (j = wtiles; j < ntiles; ++j) {
      if (j + 2 < ntiles) issue_k(j & 1);
      issue_v(j & 1);
      publish();
    }
  }

  if constexpr (SPLIT) {
    if (parts > 1) {
      const int64_t at = ((int64_t)blockIdx.x * p.split + blockIdx.y) * kRows + wave * 32 + li;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float l = quad_sum(l_run[n]);
        if (q0 + 16 * n >= w.Lq) continue;
#pragma unroll
        for (int d = 0; d < CB; ++d)
          *reinterpret_cast<f32x4_t*>(p.part_o + (at + 16 * n) * D + 16 * d + 4 * lg) = oacc[d][n];
        if (lg == 0) *reinterpret_cast<float2*>(p.part_ml + (at + 16 * n) * 2) = make_float2(m_run[n], l);
      }
      return;
    }
  }

  // ---- normalise and store: the wave's 32 rows go through LDS (16-byte chunks
  // xor-swizzled by row), so that a store instruction covers whole rows ----
  const float l_tot[2] = {quad_sum(l_run[0]), quad_sum(l_run[1])};
  const float inv[2] = {l_tot[0] == 0.0f ? 0.0f : 1.0f / l_tot[0], l_tot[1] == 0.0f ? 0.0f : 1.0f / l_tot[1]};
  static_assert(4 * 32 * D <= 4 * BUF, "output staging region");
  uint16_t* const stage = smem + wave * 32 * D;
  __syncthreads();  // every wave is done reading the K/V tiles
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int d = 0; d < CB; ++d)
      *reinterpret_cast<uint2*>(stage + (16 * n + li) * D + ((2 * d + (lg >> 1)) ^ row_swizzle<NKC>(li)) * 8 +
                                (lg & 1) * 4) =
          make_uint2(pack_bf16x2(oacc[d][n][0] * inv[n], oacc[d][n][1] * inv[n]),
                     pack_bf16x2(oacc[d][n][2] * inv[n], oacc[d][n][3] * inv[n]));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int ch = i * 64 + lane, r = ch / NKC, cc = ch % NKC;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * D + (cc ^ row_swizzle<NKC>(r & 15)) * 8);
    if (row_w + r < w.Lq) store_stream(p.o + (int64_t)(w.q0 + row_w + r) * p.o_ls + h * p.o_hs + cc * 8, v);
  }
  if (p.lse == nullptr || lg != 0) return;
#pragma unroll
  for (int n = 0; n < 2; ++n)
    if (q0 + 16 * n < w.Lq)
      p.lse[(int64_t)h * p.Tq + w.q0 + q0 + 16 * n] =
          l_tot[n] == 0.0f ? -INFINITY : (m_run[n] + __log2f(l_tot[n])) / kLog2e;
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) prompt_attn_kernel(const PromptAttn p) {
  prompt_body<D, SPLIT>(p);
}

// Joins the key ranges of a row tile: a thread takes 4 channels of a row.
template <int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptAttn p) {
  int kvh, h;
  PromptRows w;
  if (!find_rows(p, unit_of(p, kvh, h), w)) return;
  int tiles;
  const int parts = parts_of(p, seen_keys(p, w), tiles);
  const int i = (int)blockIdx.y * 256 + threadIdx.x, row = i / (D / 4), d = i % (D / 4) * 4;
  if (parts <= 1 || w.row0 + row >= w.Lq) return;
  const int64_t first = (int64_t)blockIdx.x * p.split;
  float m = -INFINITY, l = 0.0f;
  f32x4_t acc{};
#pragma unroll 4
  for (int r = 0; r < parts; ++r) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + ((first + r) * kRows + row) * 2);
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(p.part_o + ((first + r) * kRows + row) * D + d);
    const float m_new = fmaxf(m, ml.x);
    const float fa = __builtin_amdgcn_exp2f(m - m_new), fb = __builtin_amdgcn_exp2f(ml.x - m_new);
    l = l * fa + ml.y * fb;
    acc = acc * fa + o * fb;
    m = m_new;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = w.q0 + w.row0 + row;
  *reinterpret_cast<uint2*>(p.o + at * p.o_ls + h * p.o_hs + d) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (p.lse != nullptr && d == 0)
    p.lse[(int64_t)h * p.Tq + at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) / kLog2e;
}

}  // namespace ltx

using namespace ltx;

// Workgroups of a call and how many may share a row tile.  Few rows over many
// keys leave most CUs idle, so the keys are split where row tiles and heads (pairs of a
// row tile and a key head counted by eights, as the grid has them) fill
// at most a quarter of the resident workgroups (half of them run each almost
// twice as fast alone: 1024 rows over 4096 keys, 32 heads, 79 us split and 78
// whole) and the prompts have keys enough to pay for the join: 768 on average,
// 2048 above an eighth (32/8 heads x 128: 16 rows over 1024 keys 12.0 us and 20.6
// whole, over 512 no difference; 512 rows over 2048 34 and 41, over 1024 28 and 22).
// Up to 32 rows a prompt there is little to join: up to half of the workgroups, and 256 keys
// on average, of which some prompts have more (5 prompts of 8 rows over 2000 keys
// 21.7 us and 32.4 whole; 32 of up to 8 rows over up to 3000, 8 heads x 64, 20.3 and 27.1).
struct PromptPlan {
  int64_t tiles, grid, split;
  int64_t bytes(int64_t D) const { return split > 1 ? grid * split * kRows * (D + 2) * 4 : 0; }
};
static PromptPlan plan_prompt(int64_t B, int64_t Tq, int64_t Tk, int64_t Hk, int64_t G) {
  // the most row tiles of B prompts with Tq rows: B of one row, and full ones
  const int64_t some = B < Tq ? B : Tq, tiles = some + (Tq - some) / kRows;
  PromptPlan t{tiles, ceil_div((tiles > 0 ? tiles : 1) * Hk, 8) * 8 * G, 1};
  const bool few = Tq <= 32 * B;
  const int64_t least = few ? (B > 3 ? B * 256 : 768) : B * (t.grid * 8 <= kResident ? 768 : 2048);
  if (Tq > 0 && t.grid * (few ? 2 : 4) <= kResident && Tk >= least) {
    t.split = kResident / t.grid;
    if (t.split > 16) t.split = 16;
  }
  return t;
}

extern "C" int ltx_prompt_attn_workspace_size(int64_t B, int64_t Tq, int64_t Tk, int64_t Hk, int64_t G, int64_t D,
                                              int64_t* bytes) {
  clear_error();
  LTX_REQUIRE(bytes != nullptr && B >= 0 && B <= LTX_MAX_REQUESTS && Tq >= 0 && Tk >= 0 && Tq <= 0x40000000 &&
                  Tk <= 0x40000000 && Hk >= 1 && G >= 1 && Hk <= 65535 && G <= 65535 && D >= 1 && D <= 65535,
              "ltx_prompt_attn_workspace_size: bad argument");
  *bytes = plan_prompt(B, Tq, Tk, Hk, G).bytes(D);
  return LTX_OK;
}

template <int D>
static void launch_prompt(const PromptAttn& p, const PromptPlan& t, hipStream_t st) {
  const dim3 threads(256);
  if (t.split <= 1) {
    hipLaunchKernelGGL((prompt_attn_kernel<D, false>), dim3((unsigned)t.grid), threads, 0, st, p);
    return;
  }
  hipLaunchKernelGGL((prompt_attn_kernel<D, true>), dim3((unsigned)t.grid, (unsigned)t.split), threads, 0, st, p);
  hipLaunchKernelGGL((prompt_join_kernel<D>), dim3((unsigned)t.grid, kRows * (D / 4) / 256), threads, 0, st, p);
}

extern "C" int ltx_prompt_attn(int64_t B, int64_t Tq, int64_t Tk, int64_t Hk, int64_t G, int64_t D, const void* q,
                               int64_t q_ls, int64_t q_hs, const void* k, int64_t k_ls, int64_t k_hs, const void* v,
                               int64_t v_ls, int64_t v_hs, const int32_t* q_starts, const int32_t* k_starts, int causal,
                               void* out, int64_t o_ls, int64_t o_hs, int zero_rest, float* lse, float scale,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* const name = "ltx_prompt_attn";
  LTX_REQUIRE(B >= 0 && B <= LTX_MAX_REQUESTS, "%s: %lld prompts, at most %d", name, (long long)B, LTX_MAX_REQUESTS);
  LTX_REQUIRE(Hk >= 1 && G >= 1 && Hk * G <= 65535 && (D == 64 || D == 128), "%s: bad head layout (D 64 or 128)", name);
  LTX_REQUIRE(Tq >= 0 && Tk >= 0 && Tq <= 0x40000000 && Tk <= 0x40000000, "%s: more than 2^30 rows or keys", name);
  if (Tq == 0) return LTX_OK;
  LTX_REQUIRE(q && out && q_starts && k_starts && (Tk == 0 || (k && v)), "%s: null pointer", name);
  auto rows = [](const void* t, int64_t ls, int64_t hs) { return (uintptr_t)t % 16 == 0 && ls % 8 == 0 && hs % 8 == 0; };
  LTX_REQUIRE(rows(q, q_ls, q_hs) && rows(k, k_ls, k_hs) && rows(v, v_ls, v_hs) && rows(out, o_ls, o_hs),
              "%s: rows must be 16-byte aligned", name);
  // a tile's 64 rows are reached with 32-bit byte offsets, and cut by their number times the stride
  for (int64_t s : {k_ls, v_ls})
    LTX_REQUIRE(Tk <= 1 || (s >= D && s <= 0x7FFFFFFF / 256), "%s: k and v rows overlap or lie too far apart", name);
  PromptAttn p{};
  p.q = static_cast<const uint16_t*>(q), p.q_ls = q_ls, p.q_hs = q_hs;
  p.o = static_cast<uint16_t*>(out), p.o_ls = o_ls, p.o_hs = o_hs, p.lse = lse;
  p.k = static_cast<const char*>(k), p.k_ls = (int)(Tk > 1 ? k_ls : D) * 2, p.k_hs = k_hs * 2;
  p.v = static_cast<const char*>(v), p.v_ls = (int)(Tk > 1 ? v_ls : D) * 2, p.v_hs = v_hs * 2;
  p.q_starts = q_starts, p.k_starts = k_starts;
  p.B = (int)B, p.Tq = (int)Tq, p.Tk = (int)Tk, p.Hk = (int)Hk, p.G = (int)G;
  p.causal = causal != 0, p.zero_rest = zero_rest != 0;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)D)) * kLog2e;
  const PromptPlan t = plan_prompt(B, Tq, Tk, Hk, G);
  LTX_REQUIRE(t.grid < (1 << 24), "%s: too many rows and heads for one launch", name);  // 2^32 threads
  const int64_t need = t.bytes(D);
  LTX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
              "%s: needs %lld bytes of workspace", name, (long long)need);
  p.sorted = B > 1 && B <= 64 && t.grid > kResident;  // a grid that is resident at once needs no order
  p.tiles = (int)(t.tiles > 0 ? t.tiles : 1);
  if (t.split > 1) {
    p.split = (int)t.split;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + t.grid * t.split * kRows * D;
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (D == 128) launch_prompt<128>(p, t, st);
  else launch_prompt<64>(p, t, st);
  LTX_LAUNCH_CHECK(name);
  return LTX_OK;
}
