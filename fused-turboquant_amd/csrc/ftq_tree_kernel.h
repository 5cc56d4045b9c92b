// Attention of a tree of drafted tokens over the slot cache (speculative
// decoding): sequence b has n_b query tokens, stored at its last n_b positions
// c_b + j, and token i attends the context positions [start_i, c_b) and the
// tokens j whose bit is set in its mask row (without masks, a chain: j <= i).
//
// The decode kernels give one query token a sequence a wave's 16 matrix
// columns; n_b tokens through them would dequantise the cache n_b times.  Here a
// workgroup (4 waves) takes 64 CT columns, a column being a (token, head of the
// kv head's group) pair, dequantises each tile of TK positions once into LDS as
// matrix-core operands, and every wave reads these for its 16 CT columns:
//   S^T = K Q^T, softmax in the log2 domain with a lazily raised maximum,
//   O^T = V^T P^T (v_mfma_f32_16x16x32_f16, float32 sums).
// With a position's V = (code - mid) scale + (min + mid scale), the weight enters
// the product as w = p f, f the scale without the power of two that its operand
// (code - mid) 2^e carries, and the sums of the weights and of the minima are four
// more rows of it, 1 / f and (min + mid scale) / f in two parts each: two matrix
// instructions in place of 32 additions, and the rounding of w is in numerator and
// denominator alike.
// A sequence's tiles are cut into parts of about one length for all sequences, as
// many as the GPU holds workgroups (tree_share): sequences of 1000 and of 6000
// positions keep them busy alike (16 of them: 94 -> 75 us against as many parts for
// each).  The parts meet in tree_merge_kernel.
//
// Cost: a tile of 32 positions takes a wave some 230 vector and 36 matrix
// instructions at 32 columns of 128 dims, and 20 KB of LDS reads.  Two conversations of
// 98000 positions with 61 nodes of 32 heads, K4 V2: 390 us with the merge, 197 GFLOP at
// 504 TFLOP/s; vector units busy 58% of the time, matrix units 28%, LDS 38%, at two
// waves a SIMD (registers).  At 16 sequences of 1024-6000 positions with up to 32 nodes
// 67 us, of which a workgroup's start (its share, the queries' transform, the first
// bytes) is a tenth and the merge 5 us; at few columns (24 chains of 5 tokens, 64-wide
// heads: 48 us, 958 GB/s) the latency of start and tile bound it.
//
// Operands in LDS, in the order in which lane (m, g) (m = lane & 15, g = lane >> 4)
// reads its 16 bytes:
//   K  [16-position tile][32-dim step s][part]: position m, dims 32 s + 8 g + j
//   V  [32-position tile][block b][part]: dim NB m + b, positions 4 g + j and
//      16 + 4 g + j (j < 4) -- the rows of the S^T accumulators, so that the weights
//      go from the score registers into the product without a shuffle
//   X  [32-position tile]: rows 0 .. 3 the parts of 1 / f and of the minimum, the
//      others 0, positions as V
// (K and V with the exchanges of TreeGeo, which spread a dequantising wave's writes
// over the LDS banks) and 2 floats a position: K factor, weight factor f LIFT.
#pragma once

#include "ftq_attn_dev.h"
#include "ftq_chunk_kernel.h"  // f16 pairs, the butterflies across lane rows
#include "ftq_merge.h"
#include "ftq_v1_dev.h"

#include <type_traits>

namespace ftq {

struct TreeArgs {
  const void* q;            // [tokens][hq][D]
  int qt, tokens;
  const uint8_t* cache;
  int64_t nb, sblk, spos, shead;
  int lbs;                  // log2 of the block size
  const int32_t* bt;        // [B][max_blocks]
  int max_blocks;
  const int32_t *sl, *qsl;  // seq_lens [B], query_start_loc [B + 1]
  const int32_t* ks;        // first context position of each token, or null
  const uint64_t* mask;     // [tokens][words], or null (a chain)
  int words;
  int B, hq, hkv;
  const float* cent;
  int kb, vb, flags;
  float qscale;             // of the (unnormalised) rotated query: scale log2 e, and the rotation's norm
  int splits, nblk;         // most parts of a row; 1: a workgroup per column block (nblk a sequence)
  float *wo, *wl;           // partial outputs / log-sum-exps, or
  void* out;                // the output itself (wo == null)
  int ot, unrot;            // its type; whether V is taken back by H
  float oscale;
  float* lse;               // with a direct output, or null
  const float* rot;         // matrix of the rotation strategy, or null
};

typedef __bf16 TreeBf8 __attribute__((ext_vector_type(8)));
constexpr int TREE_RAW = 16;  // key_bits of raw fp16 slots

template <int D> struct TreeGeo {
  static constexpr int CT = D == 256 ? 1 : 2;     // 16-column tiles per wave, at most
  static constexpr int TK = D == 64 ? 64 : 32;    // positions of a tile
  static constexpr int NS = D / 32, NB = D / 16, NT = TK / 16, NP = TK / 32;
  // The dequantising lanes of one position write the steps and rows (s, g) of one m,
  // which are multiples of 256 bytes apart: m is exchanged with m ^ kx, which differs
  // among eight lanes that write together.
  __host__ __device__ static constexpr int kx(int s, int g) {
    return D == 64 ? 4 * s + 2 * (g >> 1) : D == 128 ? 2 * s + (g >> 1) : s;
  }
  __device__ __forceinline__ static int kunit(int ts, int m, int g) { return ts * 64 + g * 16 + (m ^ kx(ts % NS, g)); }
  // The upper half of the V blocks has the position groups 4 g + j and 16 + 4 g + j
  // exchanged: two lanes that write blocks NB / 2 apart fill 16 bytes together.
  __host__ __device__ static constexpr bool vx(int b) { return D != 64 && b >= NB / 2; }
};

// A sequence and kv head.
struct TreeUnit {
  int b, kvh;
  int q0, n, ctx, len;      // first query token, query tokens, context positions, all positions
  int t0, t1;               // its tiles: from its first token's start on, to the last position with a page
  __device__ __forceinline__ void of(const TreeArgs& a, int seq, int tk) { of(a, seq, a.qsl[seq], a.qsl[seq + 1], a.sl[seq], tk); }
  __device__ __forceinline__ void of(const TreeArgs& a, int seq, int begin, int end, int positions, int tk) {
    b = seq;
    q0 = min(max(begin, 0), a.tokens);
    n = max(min(end, a.tokens) - q0, 0);
    len = max(positions, n);
    ctx = len - n;
    const int held = (int)min((int64_t)len, (int64_t)a.max_blocks << a.lbs);
    t0 = a.ks != nullptr && n > 0 ? min(max(a.ks[q0], 0), ctx) / tk : 0;
    t1 = max((held + tk - 1) / tk, t0 + 1);
  }
};

// A workgroup's part of a sequence: tiles [tb0, tb1), of column blocks blk, blk +
// nblk, ...  Workgroups are dealt to the 8 XCDs in turn; with the kv head fastest and
// then the block, those that read the same slots at one time share an XCD's L2 when
// there are 8 heads or a multiple.
struct TreePart {
  int blk, tb0, tb1;
  int part, spare;          // which of the sequence's; spare: those behind it that do not exist, if it is the last (else 0)
};

// Over the 64 lanes of a wave, without LDS (the exchanges of wave_min_u32)
template <typename T>
__device__ __forceinline__ T tree_wave_sum(T x) {
  auto dpp = [](T v, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  x += dpp(x, std::integral_constant<int, 0xB1>{});
  x += dpp(x, std::integral_constant<int, 0x4E>{});
  x += dpp(x, std::integral_constant<int, 0x141>{});
  x += dpp(x, std::integral_constant<int, 0x128>{});
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = __builtin_bit_cast(T, (uint32_t)r[0]) + __builtin_bit_cast(T, (uint32_t)r[1]);
  r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(T, (uint32_t)r[0]) + __builtin_bit_cast(T, (uint32_t)r[1]);
}
// Sums of the lanes up to each
__device__ __forceinline__ int tree_wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // lane - 1, - 2, - 4, - 8 of a row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // rows 1, 3: the row before's last lane
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // rows 2, 3: lane 31
  return x;
}

// The parts: no longer than a length for which all sequences together have no more
// parts than there are workgroups (per head and column block; at least one per
// sequence), found by bisection to 1/16, a lane per sequence.  The tiles of a sequence
// are dealt evenly to its parts.  False: no part is left for this workgroup.
constexpr int TREE_PART_MIN = 2;  // tiles (one sequence of 900 positions: 25.9 us, with 4 27.0)
// What the lane's sequence is read from; apart from tree_share, so that other work can
// be done meanwhile.
struct TreeMine {
  int begin, end, positions;
  __device__ __forceinline__ TreeMine(const TreeArgs& a, int lane) {
    const int b = min(lane, a.B - 1);
    begin = a.qsl[b];
    end = a.qsl[b + 1];
    positions = a.sl[b];
  }
};
template <int TK>
__device__ __forceinline__ bool tree_share(const TreeArgs& a, const TreeMine& m, int lane, TreeUnit& u, TreePart& p) {
  u.kvh = blockIdx.x % a.hkv;
  const int id = blockIdx.x / a.hkv, w = id / a.nblk;
  p.blk = id % a.nblk;
  if (a.splits == 1) {
    u.of(a, w, TK);
    p.tb0 = u.t0; p.tb1 = u.t1; p.part = p.spare = 0;
    return true;
  }
  auto tiles = [&](int b) __attribute__((always_inline)) {
    if (b >= a.B) return 0;
    TreeUnit v;
    v.of(a, b, TK);
    return v.n > 0 ? v.t1 - v.t0 : 0;
  };
  TreeUnit v;
  v.of(a, min(lane, a.B - 1), m.begin, m.end, m.positions, TK);
  const int mine = lane < a.B && v.n > 0 ? v.t1 - v.t0 : 0;
  auto total = [&](auto f) __attribute__((always_inline)) {  // f(tiles) over the sequences
    auto x = f(mine);
    for (int b0 = 64; b0 < a.B; b0 += 64) x += f(tiles(b0 + lane));
    return tree_wave_sum(x);
  };
  const int workers = (int)gridDim.x / (a.hkv * a.nblk);  // >= B
  auto parts = [&](int len) __attribute__((always_inline)) {
    return __builtin_amdgcn_readfirstlane(total([&](int t) { return (int)((uint32_t)(t + len - 1) / (uint32_t)len); }));
  };
  int longest = mine;
  for (int b0 = 64; b0 < a.B; b0 += 64) longest = max(longest, tiles(b0 + lane));
  longest = __builtin_amdgcn_readfirstlane((int)~wave_min_u32(~(uint32_t)longest));
  const float sum = total([](int t) { return (float)t; });
  int lo = max(TREE_PART_MIN, max((longest + a.splits - 1) / a.splits, (int)(sum / (float)workers)));
  lo = __builtin_amdgcn_readfirstlane(lo);
  int hi = max(lo, longest);  // at most one part per sequence: fits
  if (parts(lo) <= workers) {
    hi = lo;
  } else {
    const int guess = __builtin_amdgcn_readfirstlane((int)min(sum / (float)max(workers - a.B, 1) + 2.f, (float)hi));
    if (guess > lo && guess < hi) {
      if (parts(guess) <= workers) hi = guess;
      else lo = guess;
    }
    while (hi - lo > 1 + (lo >> 4)) {
      const int mid = lo + ((hi - lo) >> 1);
      if (parts(mid) <= workers) hi = mid;
      else lo = mid;
    }
  }
  for (int b0 = 0, before = 0; b0 < a.B; b0 += 64) {
    const int own = (int)((uint32_t)((b0 == 0 ? mine : tiles(b0 + lane)) + hi - 1) / (uint32_t)hi);
    const int c = tree_wave_scan(own);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + c > w);
    if (past != 0) {
      const int l = __builtin_ctzll(past), n = __builtin_amdgcn_readlane(own, l);
      u.of(a, b0 + l, TK);
      p.part = w - before - (__builtin_amdgcn_readlane(c, l) - n);
      const uint32_t nt = u.t1 - u.t0, each = nt / (uint32_t)n, more = nt - each * n;  // the first parts: one more
      p.tb0 = u.t0 + (int)(p.part * each + min((uint32_t)p.part, more));
      p.tb1 = p.tb0 + (int)(each + ((uint32_t)p.part < more ? 1u : 0u));
      p.spare = p.part == n - 1 ? a.splits - n : 0;
      return true;
    }
    before += __builtin_amdgcn_readlane(c, 63);
  }
  return false;
}

// What the sequence's token r attends of the 32 positions from pos0 on: the context
// from its start on, and the tokens of its mask (null: those up to its own).
__device__ __forceinline__ uint32_t tree_visible(const TreeArgs& a, const TreeUnit& u, int r, int pos0) {
  auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; };  // bits 0 .. k - 1
  const int rel = pos0 - u.ctx;  // tree token of bit 0
  uint32_t v = below(-rel);
  if (a.ks != nullptr && v != 0) v &= ~below(a.ks[u.q0 + r] - pos0);
  uint32_t w = 0;
  if (rel > -32 && rel < u.n) {
    if (a.mask == nullptr) {
      w = below(r + 1 - rel) & ~below(-rel);
    } else {
      const uint64_t* row = a.mask + (int64_t)(u.q0 + r) * a.words;
      if (rel < 0) {
        w = (uint32_t)(row[0] << -rel);
      } else {
        const int i = rel >> 6, o = rel & 63;
        if (i < a.words) w = (uint32_t)(row[i] >> o);
        if (o > 32 && i + 1 < a.words) w |= (uint32_t)(row[i + 1] << (64 - o));
      }
      w &= below(u.n - rel);
    }
  }
  return v | w;
}

// What a position's V brings besides its codes.
struct TreeV {
  float f;              // weight factor, NaN where a field is not finite
  float mult;           // V operand: (code - mid) times this, a power of two (tiny scales: the scale)
  uint32_t hi, lo;      // 32 / f and minimum / (16 f): f16 parts (x | y << 16), the low ones times 2^11
};
// w = p f LIFT stays below 2^(TAU + 6) LIFT = 2^15
constexpr float TREE_LIFT = 32.f;
// f16 parts of x and y
__device__ __forceinline__ void tree_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pk_f16(x, y);
  lo = pk_f16(f16_rest(x, hi, 0) * 2048.f, f16_rest(y, hi, 1) * 2048.f);
}
// scale sc and minimum vm (with the middle of the codes times sc: not finite where
// either is not); operands of at most 2^(15 - top) before the power of two.  f is in
// [32, 64) where the exponent allows, so that the low parts of small weights are
// normal numbers.  A scale below f16's normal numbers is the multiplier itself.
__device__ __forceinline__ TreeV tree_v(float sc, float vm, int top) {
  TreeV r;
  const bool tiny = fabsf(sc) < 6.103515625e-05f, bad = !(fabsf(vm) < INFINITY);
  const int e = min(max((int)((__float_as_uint(sc) >> 23) & 255u) - 132, -14), top);
  r.mult = tiny ? sc : __uint_as_float((uint32_t)(127 + e) << 23);
  const float f = tiny ? 1.f : sc * __uint_as_float((uint32_t)(127 - e) << 23);
  const float inv = __builtin_amdgcn_rcpf(f);
  tree_parts(32.f * inv, vm * inv * 0.0625f, r.hi, r.lo);
  r.f = bad ? __builtin_nanf("") : f * TREE_LIFT;
  r.hi = bad ? 0u : r.hi;
  r.lo = bad ? 0u : r.lo;
  return r;
}
__device__ __forceinline__ float tree_max3(float a, float b, float c) {
  float r;  // (fmaxf would quiet each operand first)
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// row r (0 .. 3: x high, y high, x low, y low) of X at position p: its halfword
template <int D>
__device__ __forceinline__ uint16_t* tree_x(u32x4* xb, int p, int r) {
  return reinterpret_cast<uint16_t*>(xb + (p >> 5) * 64 + ((p >> 2) & 3) * 16 + r) + ((p >> 4) & 1) * 4 + (p & 3);
}

// The block of 16 positions from pos on, or -1 (uniform)
__device__ __forceinline__ int tree_page(const TreeArgs& a, const TreeUnit& u, int pos) {
  // (a scalar load: nothing writes the table meanwhile)
  const auto* bt = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.bt + (int64_t)u.b * a.max_blocks);
  const int page = pos >> a.lbs;
  const int phys = pos < u.len && page < a.max_blocks ? bt[page] : -1;
  return phys >= 0 && (int64_t)phys < a.nb ? phys : -1;
}
template <int TK>
__device__ __forceinline__ uint32_t tree_held(const TreeArgs& a, const TreeUnit& u, int pos0) {
  uint32_t on = 0;
#pragma unroll
  for (int k = 0; k < TK / 16; ++k) on |= tree_page(a, u, pos0 + 16 * k) >= 0 ? 1u << k : 0u;
  return on;
}

// The scale of a table of N values that table_scale finds, the 128 candidates dealt
// to the four waves (two lanes a candidate, half the table each).
template <int N>
struct TreeSigma {
  float c[N / 2], base;
  bool none;
  __device__ __forceinline__ void fetch(const float* cent, int lane) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) c[i] = cent[(lane >> 5) * (N / 2) + i];
  }
  __device__ __forceinline__ static void both(float x, float& lo, float& hi) {  // of lanes l and l ^ 32
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
  }
  // the wave's best: spread and number
  __device__ __forceinline__ uint32_t best(int lane, int wave) {
    float mx = 0.f, x, y;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) mx = fmaxf(mx, fabsf(c[i]));
    both(mx, x, y);
    mx = fmaxf(x, y);
    none = !(mx > 0.f) || !(mx < INFINITY);
    const int e = (int)((__float_as_uint(mx) >> 23) & 255u);  // mx in [2^(e-127), 2^(e-126))
    base = __uint_as_float((uint32_t)min(max(263 - e, 1), 254) << 23);  // 2^(136 - e)
    const int j = wave * 32 + (lane & 31);
    const float sg = base * (1.f + (float)j * (1.f / 128.f));
    float tlo = INFINITY, thi = -INFINITY;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float t = f16_bits_to_f32(f32_to_f16_bits(sg * c[i])) * __builtin_amdgcn_rcpf(c[i]);
      tlo = c[i] != 0.f ? fminf(tlo, t) : tlo;
      thi = c[i] != 0.f ? fmaxf(thi, t) : thi;
    }
    both(tlo, x, y);
    tlo = fminf(x, y);
    both(thi, x, y);
    thi = fmaxf(x, y);
    return wave_min_u32((__float_as_uint((thi - tlo) * __builtin_amdgcn_rcpf(sg)) & ~127u) | (uint32_t)j);
  }
  __device__ __forceinline__ float sigma(uint32_t of_all) const {
    return none ? 1.f : base * (1.f + (float)(of_all & 127u) * (1.f / 128.f));
  }
};

// One wave's columns.  KHL: K as f16 hi + lo, and float32 queries too (else 16-bit ones); NH: f16 parts of the query and of
// the weights; VHL: V as hi + lo (Lloyd-Max V).
template <int D, int CT, bool KHL, int NH, bool VHL>
struct TreeWave {
  using C = TreeGeo<D>;
  static constexpr int TK = C::TK, NS = C::NS, NB = C::NB, NT = C::NT, NP = C::NP;
  static constexpr int KP = KHL ? 2 : 1, VP = VHL ? 2 : 1;
  static constexpr int KU = NT * NS * KP * 64, VU = NP * NB * VP * 64;  // 16-byte units of a tile
  static constexpr float TAU = 4.f;        // weights stay below 2^TAU
  static constexpr float MINF = -3.0e38f;  // running maximum of a column with no position yet

  // (the scalars apart from each other: neighbours would be loaded together before
  // they are registers, and then never become any)
  int c0, nct;                             // the wave's first column; tiles of columns in use (uniform; 0: none)
  int qlarge;                              // some qs is not 1 (wave-uniform)
  half8 qh[CT][NS], ql[NH == 2 ? CT : 1][NH == 2 ? NS : 1];
  float qs[CT];                            // of the scores: 1, or what a query beyond f16's range was divided by
  floatx4 acc[CT][NB];
  float m_run[CT];
  floatx4 accx[CT];                        // lanes of row 0: the rows of X
  int row[CT];                             // query row in the sequence, or -1

  // The columns, and the first and last of their first context positions over the
  // workgroup (`none` and 0 for a wave without columns)
  __device__ __forceinline__ void columns(const TreeArgs& a, const TreeUnit& u, int blk, int lane, int wave, int (*red)[2],
                                          int none, int& first, int& last) {
    const int G = a.hq / a.hkv, n = lane & 15, begin = blk * 64 * CT;
    // a block of at most 64 columns is one tile of each wave
    const int each = CT > 1 && u.n * G - begin <= 64 ? 1 : CT;
    c0 = begin + wave * 16 * each;
    nct = __builtin_amdgcn_readfirstlane(min(max((u.n * G - c0 + 15) / 16, 0), each));
    first = none;
    last = 0;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int col = c0 + 16 * ct + n;
      row[ct] = ct < each && col < u.n * G ? col / G : -1;
      if (row[ct] >= 0) {
        const int start = a.ks != nullptr ? max(a.ks[u.q0 + row[ct]], 0) : 0;
        first = min(first, start);
        last = max(last, start);
      }
      m_run[ct] = MINF;
      accx[ct] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[ct][b] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    first = (int)wave_min_u32((uint32_t)first);
    last = (int)~wave_min_u32(~(uint32_t)last);
    if (lane == 0) {
      red[wave][0] = first;
      red[wave][1] = last;
    }
    __syncthreads();
    first = __builtin_amdgcn_readfirstlane(min(min(red[0][0], red[1][0]), min(red[2][0], red[3][0])));
    last = __builtin_amdgcn_readfirstlane(max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1])));
  }

  // The columns' queries as they are stored: lane (n, g) dims 32 s + 8 g + j of column n
  struct Raw {
    u32x4 x[CT][NS][KHL ? 2 : 1];  // float32: j < 4 and the others; 16 bits: all in the first
  };
  __device__ __forceinline__ void fetch(const TreeArgs& a, const TreeUnit& u, int lane, Raw& q) {
    const int G = a.hq / a.hkv;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int col = min(c0 + 16 * ct + (lane & 15), u.n * G - 1);  // behind the last: it again, for nobody
      const int r = col / G, h = u.kvh * G + (col - r * G);
      const int64_t off = ((int64_t)(u.q0 + r) * a.hq + h) * D + 8 * (lane >> 4);
      const char* src = static_cast<const char*>(a.q) + off * (a.qt == F32 ? 4 : 2);
      if (KHL && a.qt == F32) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int k = 0; k < KP; ++k) q.x[ct][s][k] = *reinterpret_cast<const u32x4*>(src + 128 * s + 16 * k);
      } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          q.x[ct][s][0] = *reinterpret_cast<const u32x4*>(src + 64 * s);
          if constexpr (KHL) q.x[ct][s][1] = u32x4{0, 0, 0, 0};
        }
      }
    }
  }

  // The columns' queries, rotated and scaled, as f16 hi + lo.  The transform is a matrix
  // product, its rows in the order in which the score products take a query's dims (block
  // b: dims 32 (b >> 1) + 8 g + 4 (b & 1) + i); a float32 query goes in as three bf16
  // numbers, which is exact.  A caller's matrix: through 16 rows of LDS of the wave's own.
  // RAW: 1 raw slots (no transform), 0 codes, -1 either.
  template <int RAW>
  __device__ __forceinline__ void queries(const TreeArgs& a, const TreeUnit& u, const Raw& q, int lane, float (*rows)[D + 4]) {
    const int g = lane >> 4, n = lane & 15;
    // signs of row n and dims 8 g + j (the parity of the bits that both have), ones of
    // the operand's type
    const uint32_t one = a.qt == F16 ? 0x3c003c00u : 0x3f803f80u;
    const int hg = __builtin_popcount((n >> 2) & g), n0 = n & 1, n1 = (n >> 1) & 1;
    auto pair = [&](int j0, int j1) { return one | (uint32_t)(j0 & 1) << 15 | (uint32_t)(j1 & 1) << 31; };
    const uint32_t e0 = pair(hg, hg + n0), e1 = pair(hg + n1, hg + n0 + n1), sgn = 0x80008000u;
    qlarge = 0;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float inv = 1.f;
      floatx4 y[NB];  // dims 32 (b >> 1) + 8 g + 4 (b & 1) + i of column n
#pragma unroll
      for (int b = 0; b < NB; ++b) y[b] = floatx4{0.f, 0.f, 0.f, 0.f};
      if (ct < nct) {
        if (RAW == 1 || (RAW < 0 && a.kb == TREE_RAW) || a.rot != nullptr) {
          if (KHL && a.qt == F32) {
#pragma unroll
            for (int b = 0; b < NB; ++b) y[b] = __builtin_bit_cast(floatx4, q.x[ct][b >> 1][KHL ? b & 1 : 0]);
          } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t w = q.x[ct][b >> 1][0][2 * (b & 1) + (i >> 1)];
                y[b][i] = half_bits_to_f32(a.qt == F16 ? F16 : BF16, i & 1 ? w >> 16 : w & 0xffffu);
              }
          }
          if (RAW != 1 && a.rot != nullptr) {
            const int d0 = 8 * g;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              *reinterpret_cast<floatx4*>(&rows[n][32 * (b >> 1) + d0 + 4 * (b & 1)]) = y[b];
              y[b] = floatx4{0.f, 0.f, 0.f, 0.f};
            }
            __asm__ volatile("" ::: "memory");  // a wave's LDS accesses run in order
            for (int k = 0; k < D; ++k) {
              const float xk = rows[n][k];
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                const floatx4 m = *reinterpret_cast<const floatx4*>(a.rot + (int64_t)k * D + 32 * (b >> 1) + d0 + 4 * (b & 1));
#pragma unroll
                for (int i = 0; i < 4; ++i) y[b][i] = __builtin_fmaf(xk, m[i], y[b][i]);
              }
            }
            __asm__ volatile("" ::: "memory");
          }
        } else {
          [[maybe_unused]] auto transform = [&](auto wide, auto part) __attribute__((always_inline)) {  // y += H x
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int s = 0; s < NS; ++s) {
                const uint32_t all = __builtin_popcount((b >> 1) & s) & 1 ? sgn : 0u, up = b & 1 ? sgn : 0u;
                const u32x4 h{e0 ^ all, e1 ^ all, e0 ^ all ^ up, e1 ^ all ^ up};
                if constexpr (decltype(wide)::value)
                  y[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(TreeBf8, h), __builtin_bit_cast(TreeBf8, part(s)), y[b], 0, 0, 0);
                else
                  y[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, h), __builtin_bit_cast(half8, part(s)), y[b], 0, 0, 0);
              }
          };
          if (a.qt == F16) {
            transform(std::false_type{}, [&](int s) { return q.x[ct][s][0]; });
          } else if (!KHL || a.qt == BF16) {
            transform(std::true_type{}, [&](int s) { return q.x[ct][s][0]; });
          } else if constexpr (KHL) {
            u32x4 rest[NS][2];
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
              for (int k = 0; k < 2; ++k) rest[s][k] = q.x[ct][s][k];
#pragma unroll 1
            for (int t = 0; t < 3; ++t) {
              u32x4 top[NS];  // the upper halves, and what they leave
#pragma unroll
              for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int i = 0; i < 4; i += 2) {
                    const uint32_t v0 = rest[s][k][i], v1 = rest[s][k][i + 1];
                    top[s][2 * k + i / 2] = __builtin_amdgcn_perm(v1, v0, 0x07060302u);
                    rest[s][k][i] = __float_as_uint(__uint_as_float(v0) - __uint_as_float(v0 & 0xffff0000u));
                    rest[s][k][i + 1] = __float_as_uint(__uint_as_float(v1) - __uint_as_float(v1 & 0xffff0000u));
                  }
              transform(std::true_type{}, [&](int s) { return top[s]; });
            }
          }
        }
        float mx = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          // (the compiler knows what to wait for before this product reads a matrix
          // instruction's result; before inline assembly it does not)
          y[b] *= a.qscale;
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float v0 = y[b][i], v1 = y[b][i + 1];
            asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(mx) : "v"(v0), "v"(v1));
          }
        }
        mx = warp_max_q(mx);
        // A query that f16 cannot hold is scaled to [2^13, 2^14).  Small ones need
        // no scale: what their low parts lose below f16's range is 2^-25 of a
        // score, an absolute error.
        const int e = (int)((__float_as_uint(mx) >> 23) & 255u);
        const int ue = e >= 127 + 14 && e < 255 ? 140 + 127 - e : 127;
        inv = __uint_as_float((uint32_t)(254 - ue) << 23);
        if (__builtin_amdgcn_ballot_w64(ue != 127) != 0) {
          qlarge = 1;
#pragma unroll
          for (int b = 0; b < NB; ++b) y[b] *= __uint_as_float((uint32_t)ue << 23);
        }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v0 = y[2 * s + (j >> 1)][2 * (j & 1)], v1 = y[2 * s + (j >> 1)][2 * (j & 1) + 1];
          h[j] = pk_f16(v0, v1);
          l[j] = NH == 2 ? pk_f16(f16_rest(v0, h[j], 0), f16_rest(v1, h[j], 1)) : 0u;
        }
        qh[ct][s] = __builtin_bit_cast(half8, u32x4{h[0], h[1], h[2], h[3]});
        if constexpr (NH == 2) ql[ct][s] = __builtin_bit_cast(half8, u32x4{l[0], l[1], l[2], l[3]});
      }
      qs[ct] = inv;
    }
  }

  // One tile of the positions from pos0 on: kb, vb, xb its operands ([k][part][NS],
  // [p][part][NB] and [p] units of 64), tb its factors.  edge (uniform): some column
  // does not attend all of it, or (bit k of `on`: positions 16 k .. have a page) nobody
  // some.  beside(0), beside(1): work to do under the score products and under the
  // value products.  USE: 16-column tiles in use.
  template <int USE, typename F>
  __device__ __forceinline__ void tile(const TreeArgs& a, const TreeUnit& u, const u32x4* kb, const u32x4* vb, const u32x4* xb,
                                       const float (*tb)[TK], int pos0, bool edge, uint32_t on, int lane, F beside) {
    const int g = lane >> 4;
    floatx4 s[NT][USE];
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int ct = 0; ct < USE; ++ct) s[k][ct] = floatx4{0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = KHL ? 1 : NS;  // steps whose K operands are requested together
#pragma unroll
    for (int d0 = 0; d0 < NS; d0 += AHEAD) {
      half8 xh[AHEAD][NT], xl[AHEAD][NT];
#pragma unroll
      for (int d = 0; d < AHEAD; ++d)
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          const int at = C::kunit(d0 + d, lane & 15, g);
          xh[d][k] = __builtin_bit_cast(half8, kb[(k * KP) * NS * 64 + at]);
          if constexpr (KHL) xl[d][k] = __builtin_bit_cast(half8, kb[(k * KP + 1) * NS * 64 + at]);
        }
      if constexpr (!KHL) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        // the low products first: what they add is not lost beside the high ones' sum
        if constexpr (NH == 2) {
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int ct = 0; ct < USE; ++ct) s[k][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh[d][k], ql[ct][d0 + d], s[k][ct], 0, 0, 0);
        }
        if constexpr (KHL) {
#pragma unroll
          for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int ct = 0; ct < USE; ++ct) s[k][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl[d][k], qh[ct][d0 + d], s[k][ct], 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int ct = 0; ct < USE; ++ct) s[k][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh[d][k], qh[ct][d0 + d], s[k][ct], 0, 0, 0);
      }
    }
    beside(std::integral_constant<int, 0>{});
    float tf[2][NT][4];  // the factors of this lane's positions 16 k + 4 g + i
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(&tb[f][16 * k + 4 * g]);
        tf[f][k][0] = x.x; tf[f][k][1] = x.y; tf[f][k][2] = x.z; tf[f][k][3] = x.w;
      }
    if (qlarge != 0) {
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int ct = 0; ct < USE; ++ct) s[k][ct] *= qs[ct];
    }
    floatx4 y[NT][USE];  // scores less the running maximum
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int ct = 0; ct < USE; ++ct)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[k][ct][i] = __builtin_fmaf(s[k][ct][i], tf[0][k][i], -m_run[ct]);
    if (edge) {
#pragma unroll
      for (int ct = 0; ct < USE; ++ct)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const uint32_t held = ((on >> (2 * p)) & 1u ? 0xffffu : 0u) | ((on >> (2 * p + 1)) & 1u ? 0xffff0000u : 0u);
          uint32_t vis = row[ct] >= 0 ? tree_visible(a, u, row[ct], pos0 + 32 * p) & held : 0u;
          vis >>= 4 * g;
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (((vis >> (16 * k + i)) & 1u) == 0) y[2 * p + k][ct][i] = -INFINITY;
        }
    }
    float tm = -INFINITY;
#pragma unroll
    for (int ct = 0; ct < USE; ++ct)
#pragma unroll
      for (int k = 0; k < NT; ++k) tm = tree_max3(tree_max3(tm, y[k][ct][0], y[k][ct][1]), y[k][ct][2], y[k][ct][3]);
    if (__builtin_amdgcn_ballot_w64(tm > TAU) != 0) {  // wave-uniform, rare: raise the maxima
#pragma unroll
      for (int ct = 0; ct < USE; ++ct) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[k][ct][i] = y[k][ct][i] == -INFINITY ? -INFINITY : s[k][ct][i] * tf[0][k][i];
            mx = fmaxf(mx, y[k][ct][i]);
          }
        const float mn = fmaxf(m_run[ct], warp_max_q(mx));
        const float al = __builtin_amdgcn_exp2f(m_run[ct] - mn);
        m_run[ct] = mn;
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[k][ct][i] -= mn;
        accx[ct] *= al;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[ct][b] *= al;
      }
    }
    // weights x V factor as f16 parts
    u32x4 ph[NP][USE], pl[NH == 2 ? NP : 1][NH == 2 ? USE : 1];
    auto weights = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
      for (int ct = 0; ct < USE; ++ct)
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool hid = decltype(masked)::value && y[k][ct][i] == -INFINITY;  // its factor may be NaN
            w[i] = __builtin_amdgcn_exp2f(y[k][ct][i]) * (hid ? 0.f : tf[1][k][i]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t hi = pk_f16(w[2 * h], w[2 * h + 1]);
            ph[k >> 1][ct][2 * (k & 1) + h] = hi;
            if constexpr (NH == 2) pl[k >> 1][ct][2 * (k & 1) + h] = pk_f16(f16_rest(w[2 * h], hi, 0), f16_rest(w[2 * h + 1], hi, 1));
          }
        }
    };
    if (edge) weights(std::true_type{});
    else weights(std::false_type{});
    auto of = [](const u32x4& w, bool swap) { return __builtin_bit_cast(half8, swap ? u32x4{w[2], w[3], w[0], w[1]} : w); };
    auto product = [&](half8 x, floatx4& c, int p, int ct, bool swap) __attribute__((always_inline)) {
      if constexpr (NH == 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, of(pl[p][ct], swap), c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, of(ph[p][ct], swap), c, 0, 0, 0);
    };
    half8 xx[NP], xv[NP * NB];
#pragma unroll
    for (int p = 0; p < NP; ++p) xx[p] = __builtin_bit_cast(half8, xb[p * 64 + lane]);
#pragma unroll
    for (int i = 0; i < NP * NB; ++i) xv[i] = __builtin_bit_cast(half8, vb[((i / NB) * VP * NB + i % NB) * 64 + lane]);
    __builtin_amdgcn_sched_barrier(0);
    beside(std::integral_constant<int, 1>{});
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int ct = 0; ct < USE; ++ct) product(xx[p], accx[ct], p, ct, false);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if constexpr (VHL) {
          const half8 lo = __builtin_bit_cast(half8, vb[((p * VP + 1) * NB + b) * 64 + lane]);
#pragma unroll
          for (int ct = 0; ct < USE; ++ct) acc[ct][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, of(ph[p][ct], C::vx(b)), acc[ct][b], 0, 0, 0);
        }
#pragma unroll
        for (int ct = 0; ct < USE; ++ct) product(xv[p * NB + b], acc[ct][b], p, ct, C::vx(b));
      }
    }
  }

  // tile<> for the tiles in use; a wave without columns does its share of the work beside
  template <typename F>
  __device__ __forceinline__ void step(const TreeArgs& a, const TreeUnit& u, const u32x4* kb, const u32x4* vb, const u32x4* xb,
                                       const float (*tb)[TK], int pos0, bool edge, uint32_t on, int lane, F beside) {
    if (CT > 1 && nct > 1) {
      tile<CT>(a, u, kb, vb, xb, tb, pos0, edge, on, lane, beside);
    } else if (nct == 1) {
      tile<1>(a, u, kb, vb, xb, tb, pos0, edge, on, lane, beside);
    } else {
      beside(std::integral_constant<int, 0>{});
      beside(std::integral_constant<int, 1>{});
    }
  }

  // Lane (n, g) holds dims NB (4 g + i) + b of column n.
  __device__ __forceinline__ void finish(const TreeArgs& a, const TreeUnit& u, const TreePart& part, int lane) {
    const int n = lane & 15, g = lane >> 4, G = a.hq / a.hkv;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      // sums of the weights and of the minima, both times LIFT, from the lanes g = 0
      const float L = __shfl(__builtin_fmaf(accx[ct][2], 1.f / 2048.f, accx[ct][0]), n) * (1.f / 32.f);
      const float Z = __shfl(__builtin_fmaf(accx[ct][3], 1.f / 2048.f, accx[ct][1]), n) * 16.f;
      const bool none = L == 0.f;  // no position; a NaN score makes L, and the output, NaN
      const float inv = none ? 0.f : 1.f / L;
      float y[4][NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i][b] = none ? 0.f : (acc[ct][b][i] + Z) * inv;
      const int64_t at = (int64_t)(u.q0 + row[ct]) * a.hq + u.kvh * G + (c0 + 16 * ct + n - row[ct] * G);
      if (a.wo != nullptr) {
        if (row[ct] >= 0) {
          const int64_t r = at * a.splits + part.part;
#pragma unroll
          for (int i = 0; i < 4; ++i) store_elems<F32, NB>(a.wo, r * D + NB * (4 * g + i), y[i]);
          if (g == 0) {
            a.wl[r] = none ? -INFINITY : m_run[ct] + __builtin_log2f(L * (1.f / TREE_LIFT));
            for (int k = 1; k <= part.spare; ++k) a.wl[r + k] = -INFINITY;
          }
        }
        continue;
      }
      if (a.unrot) {  // H o: the low dim bits in registers, the top two across the lane rows
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int st = 1; st < NB; st <<= 1)
#pragma unroll
            for (int b = 0; b < NB; ++b)
              if ((b & st) == 0) {
                const float v0 = y[i][b], v1 = y[i][b + st];
                y[i][b] = v0 + v1;
                y[i][b + st] = v0 - v1;
              }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float u0 = y[0][b] + y[1][b], u1 = y[0][b] - y[1][b], u2 = y[2][b] + y[3][b], u3 = y[2][b] - y[3][b];
          y[0][b] = u0 + u2; y[1][b] = u1 + u3; y[2][b] = u0 - u2; y[3][b] = u1 - u3;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i][b] = fwht_pair32(fwht_pair16(y[i][b], g & 1), g & 2) * a.oscale;
        }
      }
      if (row[ct] >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t off = at * D + NB * (4 * g + i);
          if (a.ot == F32) store_elems<F32, NB>(a.out, off, y[i]);
          else if (a.ot == F16) store_elems<F16, NB>(a.out, off, y[i]);
          else store_elems<BF16, NB>(a.out, off, y[i]);
        }
        if (a.lse != nullptr && g == 0) a.lse[at] = none ? -INFINITY : (m_run[ct] + __builtin_log2f(L * (1.f / TREE_LIFT))) * 0.69314718055994531f;
      }
    }
  }
};

// Partial outputs of a row -> the row: the parts' log-sum-exps (log2 domain), -inf
// behind the last, weigh them; then the output transform, MergeRot of ftq_merge.h.
// A wave per row; rows behind the last sequence stay as they are.
template <int D, int OT, int ROT>
__global__ __launch_bounds__(256) void tree_merge_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_lse,
                                                         const int32_t* __restrict__ tokens_end, int tokens, int hq, int splits,
                                                         const float* __restrict__ rot, float scale, void* __restrict__ out,
                                                         float* __restrict__ lse_out) {
  constexpr int E = D / 64;
  __shared__ float mrow[ROT == ROT_MATRIX ? 4 : 1][ROT == ROT_MATRIX ? D : 1];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * 4 + wv;
  if (r >= (int64_t)min(max(*tokens_end, 0), tokens) * hq) return;
  const float* lse = ws_lse + r * splits;
  float M = -INFINITY;
  bool nan = false;
  int np = 0;  // parts to add
  for (int s0 = 0; s0 < splits; s0 += 64) {
    const float l = s0 + lane < splits ? lse[s0 + lane] : -INFINITY;
    M = fmaxf(M, l);
    nan = nan || l != l;
    const uint64_t some = __builtin_amdgcn_ballot_w64(l > -INFINITY);
    if (some != 0) np = s0 + 64 - __builtin_clzll(some);
  }
  M = wave_max64(M);
  nan = __builtin_amdgcn_ballot_w64(nan) != 0;  // the maximum does not show it
  float y[E], W = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = 0.f;
  const float* po = ws_o + r * splits * D + lane * E;
  constexpr int CH = 8;
  for (int s0 = 0; s0 < np; s0 += CH) {
    float x[CH][E], l[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (s0 + k < np) {
        load_f32_small<E>(po + (int64_t)(s0 + k) * D, x[k]);
        l[k] = lse[s0 + k];
      }
#pragma unroll
    for (int k = 0; k < CH; ++k)
      if (s0 + k < np) {
        const float w = __builtin_amdgcn_exp2f(l[k] - M);
        W += w;
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = __builtin_fmaf(w, x[k][i], y[i]);
      }
  }
  if (nan) W = __builtin_nanf("");
  if (lse_out != nullptr && lane == 0) lse_out[r] = W == 0.f ? -INFINITY : (M + __builtin_log2f(W)) * 0.69314718055994531f;
  const float inv = W == 0.f ? 0.f : 1.f / W;
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] *= inv;
  if constexpr (ROT == ROT_MATRIX) {
#pragma unroll
    for (int i = 0; i < E; ++i) mrow[wv][lane * E + i] = y[i];
    __asm__ volatile("" ::: "memory");  // this wave's row; a wave's LDS accesses run in order
    float z[E];
#pragma unroll
    for (int i = 0; i < E; ++i) z[i] = 0.f;
    for (int j = 0; j < D; ++j) {
      const float oj = mrow[wv][j];
#pragma unroll
      for (int i = 0; i < E; ++i) z[i] = __builtin_fmaf(oj, rot[(int64_t)(lane * E + i) * D + j], z[i]);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = z[i];
  } else if constexpr (ROT == ROT_PLAIN) {
    fwht_wave64<E>(y, lane);
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] *= scale;
  }
  store_small<OT, E>(out, r * D + lane * E, y);
}

}  // namespace ftq
