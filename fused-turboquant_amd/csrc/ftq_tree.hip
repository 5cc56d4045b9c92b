// Attention of drafted-token trees over the vLLM v1 slot cache and the raw fp16
// slots of the boundary layers: every slot format, through rows of LDS.  The
// mathematics and the layouts: ftq_tree_kernel.h.
#include "ftq_internal.h"
#include "ftq_tree_kernel.h"

#include <algorithm>
#include <cmath>

namespace ftq {

float fwht_scale(int d);
bool v1_widths_ok(int kb, int vb, int flags);
hipError_t tree_fast_64(const TreeArgs& a, int ct, unsigned grid, hipStream_t st);
hipError_t tree_fast_128(const TreeArgs& a, int ct, unsigned grid, hipStream_t st);
hipError_t tree_fast_256(const TreeArgs& a, int ct, unsigned grid, hipStream_t st);

namespace {

// n <= 16 bits at bit offset p of a little-endian dword row (one pad dword)
__device__ __forceinline__ uint32_t row_bits(const uint32_t* row, int p, int n) {
  const int i = p >> 5;
  return __builtin_amdgcn_alignbit(row[i + 1], row[i], (uint32_t)p & 31u) & ((1u << n) - 1u);
}

__device__ __forceinline__ float e4m3_value(uint32_t b) {
  const uint32_t e = (b >> 3) & 15u, m = b & 7u;
  float v;
  if (e == 0) v = (float)m * (1.f / 512.f);
  else if (e == 15 && m == 7) v = __builtin_nanf("");
  else v = __uint_as_float(((e + 120u) << 23) | (m << 20));
  return (b & 0x80u) ? -v : v;
}

// Power of two that puts the largest finite |c| of a table in [1, 2); x in lanes
__device__ __forceinline__ float pow2_of(float mx) {
  mx = wave_max64(mx);
  if (!(mx > 0.f) || !(mx < INFINITY)) return 1.f;
  const int e = (int)((__float_as_uint(mx) >> 23) & 255u);
  return __uint_as_float((uint32_t)min(max(254 - e, 1), 253) << 23);
}

// Any slot format: the tile's slots as rows of LDS, from them the factors of each
// position, then the operands.  FULL: every product is float32-level (hi + lo parts
// of what f16 does not hold exactly); else, for bf16 outputs of 16-bit queries, one
// part (rounded by at most 2^-11 of a K table value, query or weight, beside 2^-8 of
// the output) and two workgroups a CU.  Bound by the LDS reads and bit extractions of its
// dequantisation: 16 sequences of 1024-5989 positions, 32 nodes, 128-wide heads, 8-bit
// codes: 333 us for bf16 (FULL: 530), where 4-bit ones take 88 in a kernel of the
// formats in everyday use.
template <int D, bool LM, bool FULL>
__global__ __launch_bounds__(256, FULL ? 1 : 2) void tree_any_kernel(const TreeArgs a) {
  using C = TreeGeo<D>;
  constexpr int CT = C::CT, TK = C::TK, NS = C::NS, NB = C::NB, NT = C::NT, NP = C::NP;
  using W = TreeWave<D, CT, FULL, FULL ? 2 : 1, LM && FULL>;
  constexpr int LPT = 256 / TK, DPL = D / LPT;  // lanes of a position, their dims
  extern __shared__ __attribute__((aligned(16))) uint32_t pool[];  // slots [TK][pitch]; before: query rows; both: operands behind
  __shared__ __attribute__((aligned(16))) float tb[2][TK];
  __shared__ u32x4 xb[NP * 64];
  __shared__ uint32_t tabk[256], tabv[16];  // f16 hi | lo << 16 of the scaled table
  __shared__ float tabn[256];
  __shared__ float vex[TK];                 // multiplier of the position's V operand
  __shared__ float table_scale_inv;
  __shared__ int red[4][2];

  const int G = a.hq / a.hkv, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  TreeUnit u;
  TreePart part;
  if (!tree_share<TK>(a, TreeMine(a, lane), lane, u, part)) return;
  const bool raw = a.kb == TREE_RAW, kf8 = (a.flags & V1F_KFP8) != 0;
  const V1Geom geo = raw ? V1Geom{2 * D, 2 * D, 2 * D, 4 * D} : v1_geom(D, a.kb, a.vb, kf8);
  const int nd = (geo.raw + 3) / 4, pitch = (nd + 1) | 1;
  uint32_t* rows = pool;
  u32x4* kf = reinterpret_cast<u32x4*>(pool + (TK * pitch + 3) / 4 * 4);
  u32x4* vf = kf + W::KU;
  const float mid = raw ? 0.f : 0.5f * (float)((1 << a.vb) - 1);
  for (int i = tid; i < NP * 64; i += 256) xb[i] = u32x4{0, 0, 0, 0};

  if (!raw && wave == 0) {  // tables
    const int nk = 1 << a.kb;
    float mx = 0.f;
    if (!kf8)
      for (int e = lane; e < nk; e += 64) mx = fmaxf(mx, fabsf(a.cent[e]));
    const float sg = kf8 ? 1.f : pow2_of(mx) * 512.f;
    for (int e = lane; e < nk; e += 64) {
      const float c = kf8 ? e4m3_value((uint32_t)e) : a.cent[e], x = sg * c;
      const uint32_t h = f32_to_f16_bits(x);
      tabk[e] = h | f32_to_f16_bits(x - f16_bits_to_f32(h)) << 16;
      tabn[e] = c;
    }
    if (LM && lane < 16) {  // V codes of 4 bits; those past the table, which are never stored, read its last entry
      const float x = sg * (1.f / 512.f) * a.cent[min(lane, nk - 1)];
      const uint32_t h = f32_to_f16_bits(x);
      tabv[lane] = h | f32_to_f16_bits(x - f16_bits_to_f32(h)) << 16;
    }
    if (lane == 0) table_scale_inv = 1.f / sg;
  }

  for (; part.blk * 64 * CT < u.n * G; part.blk += a.nblk) {
    W w;
    int first, last;
    w.columns(a, u, part.blk, lane, wave, red, u.len, first, last);  // its barrier: the pool is free, and the tables written
    typename W::Raw q;
    w.fetch(a, u, lane, q);
    w.template queries<-1>(a, u, q, lane, reinterpret_cast<float(*)[D + 4]>(pool) + 16 * wave);
    __syncthreads();
    first = min(first, u.ctx) / TK;  // the tree's own positions always
    const int tb0 = part.part == 0 ? first : max(part.tb0, first), tb1 = part.tb1;

    for (int t = tb0; t < tb1; ++t) {
      const int pos0 = t * TK;
      float beyond = 0.f;  // raw slots: whether this lane read a V element that is not finite
      {
        const int p = tid / LPT, sub = tid % LPT, pos = pos0 + p, page = pos >> a.lbs;
        const int phys = pos < u.len && page < a.max_blocks ? a.bt[(int64_t)u.b * a.max_blocks + page] : -1;
        const bool on = phys >= 0 && (int64_t)phys < a.nb;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(
            a.cache + (on ? (int64_t)phys * a.sblk + (int64_t)(pos & ((1 << a.lbs) - 1)) * a.spos + (int64_t)u.kvh * a.shead : 0));
        for (int c = sub; c < nd; c += LPT) {
          const uint32_t x = on ? src[c] : 0u;
          rows[p * pitch + c] = x;
          if (raw && c >= D / 2 && ((x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u)) beyond = 1.f;
        }
        if (sub == 0) rows[p * pitch + nd] = 0;
      }
      __syncthreads();
      {  // factors
        const int p = tid / LPT, sub = tid % LPT;
        const uint32_t* row = rows + p * pitch;
        float csq = 0.f, vsq = 0.f;
        if (!raw && !kf8) {
          for (int d = 0; d < DPL; ++d) {
            const float c = tabn[row_bits(row, (sub * DPL + d) * a.kb, a.kb)];
            csq = __builtin_fmaf(c, c, csq);
          }
          csq = group_sum<LPT>(csq);
        }
        if constexpr (LM) {
          for (int d = 0; d < DPL; ++d) {
            const float c = tabn[min((int)row_bits(row, 8 * geo.kps + (sub * DPL + d) * 4, 4), (1 << a.kb) - 1)];
            vsq = __builtin_fmaf(c, c, vsq);
          }
          vsq = group_sum<LPT>(vsq);
        }
        if (raw) beyond = group_sum<LPT>(beyond);
        if (sub == 0) {
          // A raw V that is not finite (as a scale or minimum): operands of 0 and a NaN
          // factor, so that the rows that attend it are NaN and the others, whose
          // products meet it with a weight of 0, are not.
          float fk = 1.f;
          TreeV v{beyond == 0.f ? TREE_LIFT : __builtin_nanf(""), beyond == 0.f ? 1.f : 0.f, beyond == 0.f ? 0x5000u : 0u, 0u};
          if (!raw) {
            if (!kf8) fk = f16_bits_to_f32(row_bits(row, 8 * geo.mse, 16)) / __builtin_sqrtf(csq + 1e-16f) * table_scale_inv;
            float sc = f16_bits_to_f32(row_bits(row, 8 * (geo.kps + geo.vdb), 16)), vm = 0.f;
            if constexpr (LM) {  // the norm's; a minimum of 0, or NaN where the norm is not finite
              sc = sc / __builtin_sqrtf(vsq + 1e-16f) * (512.f * table_scale_inv);
              vm = sc * 0.f;
            }
            else vm = __builtin_fmaf(mid, sc, f16_bits_to_f32(row_bits(row, 8 * (geo.kps + geo.vdb) + 16, 16)));
            // (codes of 128 at most times 2^8; Lloyd-Max values are below 2)
            v = tree_v(sc, vm, LM ? 14 : a.vb == 8 ? 8 : 11);
          }
          tb[0][p] = fk;
          tb[1][p] = v.f;
          *tree_x<D>(xb, p, 0) = (uint16_t)v.hi;
          *tree_x<D>(xb, p, 1) = (uint16_t)(v.hi >> 16);
          *tree_x<D>(xb, p, 2) = (uint16_t)v.lo;
          *tree_x<D>(xb, p, 3) = (uint16_t)(v.lo >> 16);
          vex[p] = v.mult;
        }
      }
      __syncthreads();
      for (int i = tid; i < NT * NS * 64; i += 256) {
        const int l = i & 63, ts = i >> 6, m = l & 15, g = l >> 4;
        const int d0 = (ts % NS) * 32 + 8 * g, at = (ts / NS) * W::KP * NS * 64 + C::kunit(ts % NS, m, g);
        const uint32_t* row = rows + ((ts / NS) * 16 + m) * pitch;
        uint32_t h[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (raw) {
            h[j] = row[d0 / 2 + j];
            lo[j] = 0;
          } else {
            const uint32_t x = tabk[row_bits(row, (d0 + 2 * j) * a.kb, a.kb)], y = tabk[row_bits(row, (d0 + 2 * j + 1) * a.kb, a.kb)];
            h[j] = (x & 0xffffu) | (y << 16);
            lo[j] = (x >> 16) | (y & 0xffff0000u);
          }
        }
        kf[at] = u32x4{h[0], h[1], h[2], h[3]};
        if constexpr (FULL) kf[at + NS * 64] = u32x4{lo[0], lo[1], lo[2], lo[3]};
      }
      for (int i = tid; i < NP * NB * 64; i += 256) {
        const int l = i & 63, pb = i >> 6, m = l & 15, g = l >> 4, d = NB * m + pb % NB;
        uint32_t h[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x[2], y[2];  // hi and lo of two positions
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int p = (pb / NB) * 32 + ((j >> 1) ^ (C::vx(pb % NB) ? 1 : 0)) * 16 + 4 * g + 2 * (j & 1) + k;
            const uint32_t* row = rows + p * pitch;
            y[k] = 0.f;
            if (raw) {
              x[k] = vex[p] != 0.f ? f16_bits_to_f32(row_bits(row, 16 * D + 16 * d, 16)) : 0.f;
            } else if constexpr (LM) {
              const uint32_t c = tabv[row_bits(row, 8 * geo.kps + d * 4, 4)];
              x[k] = f16_bits_to_f32(c & 0xffffu) * vex[p];
              if constexpr (FULL) y[k] = f16_bits_to_f32(c >> 16) * vex[p];
            } else {
              x[k] = ((float)row_bits(row, 8 * geo.kps + d * a.vb, a.vb) - mid) * vex[p];
            }
          }
          h[j] = pk_f16(x[0], x[1]);
          if constexpr (LM && FULL) lo[j] = pk_f16(y[0], y[1]);
        }
        const int at = ((pb / NB) * W::VP * NB + pb % NB) * 64 + l;
        vf[at] = u32x4{h[0], h[1], h[2], h[3]};
        if constexpr (LM && FULL) vf[at + NB * 64] = u32x4{lo[0], lo[1], lo[2], lo[3]};
      }
      __syncthreads();
      const uint32_t on = tree_held<TK>(a, u, pos0);  // bit k: positions 16 k .. of the tile have a page
      w.step(a, u, kf, vf, xb, tb, pos0, pos0 < last || pos0 + TK > u.ctx || on != (1u << NT) - 1u, on, lane, [](auto) {});
      __syncthreads();  // before the next tile's rows
    }
    w.finish(a, u, part, lane);
  }
}

template <int D, bool LM, bool FULL>
hipError_t any_launch(const TreeArgs& a, unsigned grid, hipStream_t st) {
  using C = TreeGeo<D>;
  using W = TreeWave<D, C::CT, FULL, FULL ? 2 : 1, LM && FULL>;
  const bool raw = a.kb == TREE_RAW;
  const V1Geom geo = raw ? V1Geom{2 * D, 2 * D, 2 * D, 4 * D} : v1_geom(D, a.kb, a.vb, (a.flags & V1F_KFP8) != 0);
  const int pitch = ((geo.raw + 3) / 4 + 1) | 1;
  const size_t rows = (size_t)(C::TK * pitch + 3) / 4 * 16;
  const size_t lds = std::max(rows + (size_t)(W::KU + W::VU) * 16, (size_t)64 * (D + 4) * 4);
  tree_any_kernel<D, LM, FULL><<<dim3(grid), dim3(256), lds, st>>>(a);
  return hipGetLastError();
}

template <int D>
hipError_t tree_merge(const TreeArgs& a, int64_t tokens, bool vrot, hipStream_t st) {
  const dim3 grid((unsigned)((tokens * a.hq + 3) / 4)), block(256);
  const int32_t* end = a.qsl + a.B;
  const float rs = fwht_scale(D);
#define FTQ_TREE_MERGE(R, S, F)                                                                                              \
  (a.ot == F32   ? tree_merge_kernel<D, F32, R><<<grid, block, 0, st>>>(a.wo, a.wl, end, a.tokens, a.hq, a.splits, S, F, a.out, a.lse) \
   : a.ot == F16 ? tree_merge_kernel<D, F16, R><<<grid, block, 0, st>>>(a.wo, a.wl, end, a.tokens, a.hq, a.splits, S, F, a.out, a.lse) \
                 : tree_merge_kernel<D, BF16, R><<<grid, block, 0, st>>>(a.wo, a.wl, end, a.tokens, a.hq, a.splits, S, F, a.out, a.lse))
  if (vrot && a.rot != nullptr) FTQ_TREE_MERGE(ROT_MATRIX, a.rot, 1.f);
  else if (vrot) FTQ_TREE_MERGE(ROT_PLAIN, nullptr, rs);
  else FTQ_TREE_MERGE(ROT_NONE, nullptr, rs);
  return hipGetLastError();
#undef FTQ_TREE_MERGE
}

// The formats of ftq_tree_fast.h: 16-bit queries and outputs, 2-4 bit codes or raw slots that
// 16-byte loads reach, and positions of a tile within 32-bit offsets.
bool tree_fast_takes(const TreeArgs& a) {
  if (a.ot == F32 || a.qt == F32 || a.spos > (1 << 26)) return false;
  if (a.kb == TREE_RAW) return (((uintptr_t)a.cache | (uintptr_t)a.sblk | (uintptr_t)a.spos | (uintptr_t)a.shead) & 15) == 0;
  return a.kb >= 2 && a.kb <= 4 && a.vb >= 2 && a.vb <= 4 && (a.flags & V1F_KFP8) == 0 && !((a.flags & V1F_VLM) != 0 && a.vb == 4);
}

template <int D>
hipError_t tree_launch(const TreeArgs& a, int ct, unsigned grid, int64_t tokens, bool vrot, hipStream_t st) {
  const bool lm = (a.flags & V1F_VLM) != 0 && a.vb == 4;
  const hipError_t e = tree_fast_takes(a) ? (D == 64 ? tree_fast_64(a, ct, grid, st) : D == 128 ? tree_fast_128(a, ct, grid, st) : tree_fast_256(a, ct, grid, st))
                       : a.ot == BF16 && a.qt != F32 ? (lm ? any_launch<D, true, false>(a, grid, st) : any_launch<D, false, false>(a, grid, st))
                       : lm ? any_launch<D, true, true>(a, grid, st) : any_launch<D, false, true>(a, grid, st);
  if (e != hipSuccess || a.wo == nullptr) return e;
  return tree_merge<D>(a, tokens, vrot, st);
}

// 16-column tiles of a wave for sequences of at most `cols` columns: one where 64
// columns do, and three workgroups a CU (24 sequences, 20 columns of 64-wide heads: 54
// us, with two column tiles 62, with one and two workgroups 61; 80 sequences, 32
// columns of 128-wide heads: 235, 279 and 276), else two (16 sequences of 1024-6000 positions, 128 columns of
// 128-wide heads: 91 us, with one 102; 98000 positions, 244 columns: 339 and 448).
int tree_ct(int d, int64_t cols) { return d == 256 || cols <= 64 ? 1 : 2; }
// Workgroups that the 256 CUs hold at once, by registers and LDS.
int64_t tree_resident(int d, int ct) { return 256 * (d != 256 && ct == 1 ? 3 : 2); }
// Parts (tree_share) of all sequences together, per kv head and column block: what the
// GPU holds.  (Half of it: 91 -> 124 us at 16 sequences of 1024-6000 positions; twice:
// 111 us, each part's start and end are work too.)  Where that is hardly more than the
// sequences, two each (48 sequences of 3000 positions, 128 columns: 201 us, with one
// each 206, with three 223).
int64_t tree_parts_all(int d, int ct, int hkv, int64_t nblk, int64_t batch) {
  const int64_t s = tree_resident(d, ct) / (hkv * nblk);
  return 3 * batch <= 2 * s ? s : std::max(s, 2 * batch);
}

}  // namespace
}  // namespace ftq

using namespace ftq;

extern "C" int ftq_v1_tree_choose_splits(int batch, int max_query_len, int num_q_heads, int num_kv_heads, int d,
                                         int key_bits, int value_bits, int v_flags, int max_seq_len) {
  (void)key_bits; (void)value_bits; (void)v_flags;
  if (batch <= 0 || max_query_len <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      max_seq_len <= 0)
    return 1;
  // An even share for each, and three times that when the others are shorter.
  const int64_t ncols = (int64_t)max_query_len * (num_q_heads / num_kv_heads);
  const int ct = tree_ct(d, ncols);
  const int64_t nblk = (ncols + 64 * ct - 1) / (64 * ct);
  // Two rounds of whole sequences need no parts: 200 sequences of 500-4480 positions,
  // 32 columns: 391 us, in parts 433; 128 sequences (1.3 rounds): 365 and 330.
  if (nblk * batch * num_kv_heads >= 2 * tree_resident(d, ct)) return 1;
  const int64_t tiles = ((int64_t)max_seq_len + (d == 64 ? 63 : 31)) / (d == 64 ? 64 : 32);
  const int64_t s = 3 * tree_parts_all(d, ct, num_kv_heads, nblk, batch) / batch + 1;
  return (int)std::max<int64_t>(std::min({s, tiles / TREE_PART_MIN, (int64_t)64}), 1);
}

extern "C" int ftq_v1_tree_attention(const void* query, int q_dtype, int64_t num_tokens, const uint8_t* kv_cache,
                                     int64_t num_blocks, int block_size, int64_t stride_block, int64_t stride_pos,
                                     int64_t stride_head, const int32_t* block_table, int max_blocks_per_seq,
                                     const int32_t* seq_lens, const int32_t* query_start_loc, const uint64_t* tree_mask,
                                     int mask_words, const int32_t* kv_start, int batch, int max_query_len,
                                     int num_q_heads, int num_kv_heads, int d, const float* centroids, int key_bits,
                                     int value_bits, float scale, int v_flags, int num_splits, void* workspace,
                                     int64_t workspace_bytes, void* out, int out_dtype, float* lse_out,
                                     const float* rotation, void* stream) {
  const bool raw = key_bits == TREE_RAW;
  FTQ_REQUIRE(d == 64 || d == 128 || d == 256, "tree attention: head_dim must be 64, 128 or 256");
  FTQ_REQUIRE(raw ? (value_bits == TREE_RAW && v_flags == 0 && rotation == nullptr)
                  : v1_widths_ok(key_bits, value_bits, v_flags),
              "tree attention: key_bits and value_bits must both be in 1..4, both 8 or both 16 (raw fp16 slots, no flags)");
  FTQ_REQUIRE((v_flags & ~(V1F_VROT | V1F_VLM | V1F_KFP8)) == 0,
              "tree attention: v_flags bits 0 (V rotated), 1 (Lloyd-Max V) and 2 (fp8 keys) only");
  FTQ_REQUIRE(block_size >= 16 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,
              "block_size must be a power of two in [16, 4096]");
  FTQ_REQUIRE(num_tokens >= 0 && batch >= 0 && max_query_len >= 0 && num_kv_heads > 0 && num_q_heads > 0 &&
                  num_blocks >= 0 && max_blocks_per_seq >= 0,
              "bad token / sequence / head / block counts");
  FTQ_REQUIRE(num_q_heads % num_kv_heads == 0, "num_q_heads must be a multiple of num_kv_heads");
  FTQ_REQUIRE(num_q_heads / num_kv_heads <= 16, "GQA group (num_q_heads / num_kv_heads) must be <= 16");
  FTQ_REQUIRE(q_dtype >= F32 && q_dtype <= BF16 && out_dtype >= F32 && out_dtype <= BF16,
              "dtype must be FTQ_F32, FTQ_F16 or FTQ_BF16");
  const int raw_bytes = raw ? 4 * d : v1_geom(d, key_bits, value_bits, (v_flags & V1F_KFP8) != 0).raw;
  FTQ_REQUIRE(stride_head >= raw_bytes, "stride_head is smaller than the slot bytes");
  FTQ_REQUIRE(cache_strides_ok(num_blocks, stride_block, stride_pos, stride_head, num_kv_heads, block_size),
              "kv_cache strides must describe [num_blocks][block_size][num_kv_heads][slot]");
  FTQ_REQUIRE(stride_head % 4 == 0 && stride_pos % 4 == 0 && stride_block % 4 == 0,
              "kv_cache strides must be multiples of 4 bytes");
  FTQ_REQUIRE(num_splits >= 1 && num_splits <= 1024, "num_splits must be in [1, 1024]");
  FTQ_REQUIRE(tree_mask == nullptr || mask_words >= 1, "tree_mask needs at least one word a token");
  if (num_tokens == 0 || batch == 0 || max_query_len == 0) return FTQ_OK;
  FTQ_REQUIRE(num_tokens <= (1 << 30) / num_q_heads, "tree attention: too many tokens");
  FTQ_REQUIRE(num_blocks >= 1, "kv_cache must hold at least one block");
  FTQ_REQUIRE(query && kv_cache && block_table && seq_lens && query_start_loc && out && workspace, "null pointer argument");
  FTQ_REQUIRE(centroids != nullptr || raw || (v_flags & V1F_KFP8) != 0, "null centroids");
  FTQ_REQUIRE(aligned16(query) && aligned16(out) && aligned16(workspace) && aligned4(kv_cache),
              "query, out and workspace must be 16-byte aligned, kv_cache 4-byte aligned");
  FTQ_REQUIRE(((uintptr_t)tree_mask & 7u) == 0, "tree_mask must be 8-byte aligned");
  const int64_t need = split_workspace_bytes((int)num_tokens, num_q_heads, d, num_splits);
  FTQ_REQUIRE(need >= 0 && workspace_bytes >= need, "workspace too small (see ftq_v1_workspace_bytes)");
  const int64_t ncols = std::min<int64_t>(max_query_len, num_tokens) * (num_q_heads / num_kv_heads);
  TreeArgs a{};
  a.qt = q_dtype; a.ot = out_dtype; a.kb = key_bits; a.vb = value_bits; a.flags = v_flags;
  a.cache = kv_cache; a.nb = num_blocks; a.sblk = stride_block; a.spos = stride_pos; a.shead = stride_head;
  const int ct = tree_fast_takes(a) ? tree_ct(d, ncols) : tree_ct(d, INT32_MAX);
  const int64_t nblk = (ncols + 64 * ct - 1) / (64 * ct);
  const int64_t parts = num_splits == 1 ? batch : tree_parts_all(d, ct, num_kv_heads, nblk, batch);
  int64_t grid = 0;
  FTQ_REQUIRE(!__builtin_mul_overflow(nblk * num_kv_heads, parts, &grid) && grid <= INT32_MAX, "tree attention: grid too large");
  const bool vrot = (v_flags & V1F_VROT) != 0;
  a.q = query; a.tokens = (int)num_tokens;
  while ((1 << a.lbs) < block_size) ++a.lbs;
  a.bt = block_table; a.max_blocks = max_blocks_per_seq;
  a.sl = seq_lens; a.qsl = query_start_loc; a.ks = kv_start;
  a.mask = tree_mask; a.words = mask_words;
  a.B = batch; a.hq = num_q_heads; a.hkv = num_kv_heads;
  a.cent = centroids;
  a.qscale = (raw || rotation != nullptr ? 1.f : fwht_scale(d)) * scale * 1.4426950408889634f;
  a.splits = num_splits; a.nblk = (int)nblk;
  const bool direct = num_splits == 1 && !(vrot && rotation != nullptr);
  a.wo = direct ? nullptr : static_cast<float*>(workspace);
  a.wl = direct ? nullptr : a.wo + num_tokens * num_q_heads * num_splits * d;
  a.out = out;
  a.unrot = vrot; a.oscale = vrot ? fwht_scale(d) : 1.f;
  a.lse = lse_out; a.rot = rotation;
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = d == 64 ? tree_launch<64>(a, ct, (unsigned)grid, num_tokens, vrot, st) : d == 128 ? tree_launch<128>(a, ct, (unsigned)grid, num_tokens, vrot, st)
                                                                                    : tree_launch<256>(a, ct, (unsigned)grid, num_tokens, vrot, st);
  return hip_status(e);
}
