// Tree attention for the formats in everyday use: 2-4 bit keys (codebook) with
// 2-4 bit uniform values, and raw fp16 slots, with 16-bit queries and outputs
// (float32 ones take the kernel of ftq_tree.hip, whose products are all float32-level).
//
// Two LDS buffers of operands: while the waves multiply one tile, each thread
// turns the bytes of the next, which it loaded a tile earlier, into operands, and
// requests the bytes of the one after.  One barrier a tile.  A wave takes TK / 4
// positions of a tile:
//   K  LPT lanes a position, EK consecutive dims each: pair table lookups, whose
//      squares give the norm correction, written as 16-byte operands
//   V  LPQ lanes four positions, DV consecutive dims of each: codes to f16 in
//      place (mantissa bits, one packed multiply-add), written as the four
//      positions of each dim, the transposition that the product needs
// Measured steps, 16 sequences of 1024-6000 positions, up to 32 nodes, 128-wide heads
// (us): through rows of LDS 580, this scheme 94, parts of one length 75, the table's
// scale searched by four waves and the queries four lanes each 70, their transform as a
// matrix product 67.  Measured and not kept:
// vector and matrix instructions interleaved by hand (98000 positions: 340 -> 362 us),
// wave priorities around the products (340 -> 344).
// Operands: K table values as f16 (a common scale that keeps their relative
// errors alike, TreeSigma), V codes exact (centred, times the scale's own power
// of two).  bf16 outputs: query and weights as one f16 number, 2^-11 beside the
// output's 2^-8; fp16 outputs: as hi + lo.
#pragma once

#include "ftq_internal.h"
#include "ftq_tree_kernel.h"

namespace ftq {

struct __attribute__((packed, aligned(2))) TreeU32 { uint32_t v; };
struct __attribute__((packed, aligned(2))) TreeU64 { uint64_t v; };

// N bytes (a multiple of 4) from an even offset
template <int N>
__device__ __forceinline__ void tree_bytes(const uint8_t* p, uint32_t (&w)[N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; i += 2) {
    if (i + 1 < N / 4) {
      const uint64_t x = reinterpret_cast<const TreeU64*>(p + 4 * i)->v;
      w[i] = (uint32_t)x;
      w[i + 1] = (uint32_t)(x >> 32);
    } else {
      w[i] = reinterpret_cast<const TreeU32*>(p + 4 * i)->v;
    }
  }
}

// All waves' LDS accesses before it are done; loads in flight stay in flight
__device__ __forceinline__ void tree_barrier() { __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A tile's operands: 16-byte units of K, V, X and the factors
template <int D> struct TreeBuf {
  using C = TreeGeo<D>;
  static constexpr int V = C::NT * C::NS * 64, X = V + C::NP * C::NB * 64, T = X + C::NP * 64, SIZE = T + 2 * C::TK / 4;
};

// KB = TREE_RAW: raw fp16 slots (16-byte aligned)
template <int D, int KB, int VB>
struct TreeFmt {
  using C = TreeGeo<D>;
  static constexpr bool RAW = KB == TREE_RAW;
  static constexpr V1Geom G = RAW ? V1Geom{2 * D, 2 * D, 2 * D, 4 * D} : v1_geom(D, KB, VB);
  static constexpr int TPW = C::TK / 4;                     // positions of a wave
  static constexpr int LPT = 64 / TPW, EK = D / LPT;        // K: lanes of a position, dims of a lane
  static constexpr int LPQ = 256 / TPW, DV = D / LPQ;       // V: lanes of four positions, dims of a lane
  // Loads are whole dwords from even offsets (16-bit ones would be converted, and
  // waited for, as they come); what they read past a lane's codes lies in the slot.
  static constexpr int KN = EK * KB / 8, KR = (KN + 3) / 4 * 4;  // bytes of a lane's K codes, and read
  static constexpr int VBITS = DV * VB;                     // a lane's V codes of one position
  static constexpr bool VSH = VBITS % 16 != 0;              // ... that may start inside a 16-bit unit
  static constexpr int VR = RAW ? VBITS / 8 : 4;            // bytes read for them
  static constexpr int ENTRIES = RAW ? 1 : 1 << (2 * KB);
  static constexpr float MID = 0.5f * (float)((1 << (RAW ? 0 : VB)) - 1);

  uint32_t k[KR / 4], v[4][VR / 4];
  uint32_t kn, sm;  // K norm of the lane's position; scale | minimum of V position lane % 4 of its four

  // base: slot of the wave's first position (uniform)
  __device__ __forceinline__ void load(const uint8_t* base, uint32_t s_pos, int lane) {
    const int e = lane % LPT, dq = lane % LPQ;
    uint32_t kn_at = (uint32_t)(lane / LPT) * s_pos, k_at = kn_at + e * KN;
    uint32_t v_at = (uint32_t)(lane / LPQ * 4) * s_pos, sm_at = v_at + (uint32_t)(dq & 3) * s_pos;
    v_at += (uint32_t)(dq * VBITS) >> 4 << 1;
    // (opaque here, so that each stays the 32-bit offset of a uniform address)
    __asm__ volatile("" : "+v"(kn_at), "+v"(k_at), "+v"(v_at), "+v"(sm_at));
    if constexpr (RAW) {
#pragma unroll
      for (int i = 0; i < KN / 16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(base + k_at + 16 * i);
        k[4 * i] = x.x; k[4 * i + 1] = x.y; k[4 * i + 2] = x.z; k[4 * i + 3] = x.w;
      }
    } else {
      tree_bytes<KR>(base + k_at, k);
      kn = reinterpret_cast<const TreeU32*>(base + kn_at + G.mse)->v;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint64_t row = (uint64_t)i * s_pos + G.kps;
      __asm__("" : "+s"(row));  // uniform, and added to the base first
      const uint8_t* pv = base + row;
      if constexpr (RAW) {
        if constexpr (VR == 8) {
          const uint2 x = *reinterpret_cast<const uint2*>(pv + v_at);
          v[i][0] = x.x; v[i][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(pv + v_at);
          v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
        }
      } else {
        tree_bytes<VR>(pv + v_at, v[i]);
      }
    }
    if constexpr (!RAW) sm = reinterpret_cast<const TreeU32*>(base + sm_at + (G.kps + G.vdb))->v;
  }

  // K operands and factors of the tile's positions TPW w .., to a buffer
  __device__ __forceinline__ void emit_k(const uint32_t* table, u32x4* buf, int w, int lane) const {
    constexpr int NS = C::NS;
    const int p = w * TPW + lane / LPT, e = lane % LPT, d0 = e * EK;
    float csq = 0.f;
#pragma unroll
    for (int u = 0; u < EK / 8; ++u) {
      u32x4 x;
      if constexpr (RAW) {
        x = u32x4{k[4 * u], k[4 * u + 1], k[4 * u + 2], k[4 * u + 3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = lds_dword_at(table, lut_field<2, 2 * KB>(k, (8 * u + 2 * j) * KB, 0u));
          const half2_t h = __builtin_bit_cast(half2_t, (uint32_t)x[j]);
          csq = __builtin_amdgcn_fdot2(h, h, csq, false);
        }
      }
      const int d = d0 + 8 * u;
      buf[(p >> 4) * NS * 64 + C::kunit(d / 32, p & 15, (d / 8) & 3)] = x;
    }
    // the lanes of a position all have its factor, and write it to one place
    float* tb = reinterpret_cast<float*>(buf + TreeBuf<D>::T);
    if constexpr (!RAW) tb[p] = f16_bits_to_f32(kn & 0xffffu) * __builtin_amdgcn_rsqf(group_sum<LPT>(csq) + 1e-16f);
    else tb[p] = 1.f;
  }

  // V and X operands and factors
  __device__ __forceinline__ void emit_v(u32x4* buf, int w, int lane) const {
    constexpr int NB = C::NB;
    u32x4 *vb = buf + TreeBuf<D>::V, *xb = buf + TreeBuf<D>::X;
    float* tb = reinterpret_cast<float*>(buf + TreeBuf<D>::T) + C::TK;
    // V: positions 4 q ..
    const int q = w * (TPW / 4) + lane / LPQ, dq = lane % LPQ;
    uint2* out = reinterpret_cast<uint2*>(vb + (q >> 3) * NB * 64 + (q & 3) * 16);
    const int half = (q >> 2) & 1;
    auto put = [&](int i, uint32_t lo, uint32_t hi) {  // the lane's dim i, four positions
      const int d = dq * DV + i, b = d % NB, m = d / NB;
      out[(b * 64 + m) * 2 + (C::vx(b) ? 1 - half : half)] = make_uint2(lo, hi);
    };
    if constexpr (RAW) {
      // a V that is not finite: operands of 0 and a NaN factor (as tree_any_kernel)
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < DV / 2; ++j) any |= ((v[i][j] & 0x7c00u) == 0x7c00u || (v[i][j] & 0x7c000000u) == 0x7c000000u) ? 1u : 0u;
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(any != 0);
        constexpr uint64_t ONE = LPQ == 32 ? 0xffffffffull : 0xffffull;
        bad |= (lanes >> (lane / LPQ * LPQ) & ONE) != 0 ? 1u << i : 0u;
      }
#pragma unroll
      for (int i = 0; i < DV; ++i) {
        const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
        uint32_t lo = __builtin_amdgcn_perm(v[1][i / 2], v[0][i / 2], sel), hi = __builtin_amdgcn_perm(v[3][i / 2], v[2][i / 2], sel);
        lo &= (bad & 1 ? 0u : 0xffffu) | (bad & 2 ? 0u : 0xffff0000u);
        hi &= (bad & 4 ? 0u : 0xffffu) | (bad & 8 ? 0u : 0xffff0000u);
        put(i, lo, hi);
      }
      const int own = dq & 3;  // lanes with the same write the same
      const bool b = (bad >> own) & 1;
      tb[4 * q + own] = b ? __builtin_nanf("") : TREE_LIFT;
      *tree_x<D>(xb, 4 * q + own, 0) = b ? 0 : 0x5000;  // 32
    } else {
      // the lane's own position; operand (code - mid) mult = (1 + code 2^-VB) 2^VB mult
      // - (2^VB + mid) mult
      const float sc = f16_bits_to_f32(sm & 0xffffu);
      const TreeV r = tree_v(sc, __builtin_fmaf(MID, sc, f16_bits_to_f32(sm >> 16)), 11);
      const int own_p = 4 * q + (dq & 3);  // lanes with the same write the same
      tb[own_p] = r.f;
      *tree_x<D>(xb, own_p, 0) = (uint16_t)r.hi;
      *tree_x<D>(xb, own_p, 1) = (uint16_t)(r.hi >> 16);
      *tree_x<D>(xb, own_p, 2) = (uint16_t)r.lo;
      *tree_x<D>(xb, own_p, 3) = (uint16_t)(r.lo >> 16);
      const uint32_t own = pk_f16(r.mult * (float)(1 << VB), r.mult * -((float)(1 << VB) + MID));
      uint32_t ec[4];  // of the four positions: from the four lanes of a quad
      ec[0] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0x00, 0xF, 0xF, true);
      ec[1] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0x55, 0xF, 0xF, true);
      ec[2] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0xAA, 0xF, 0xF, true);
      ec[3] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0xFF, 0xF, 0xF, true);
      uint32_t one = 0x3C003C00u;
      asm("" : "+v"(one));  // in a register: the mask and it then are one v_and_or_b32
      const uint32_t vsh = VSH ? (uint32_t)(dq * VBITS) & 15u : 0u;
      constexpr int PER = 16 / VB;  // codes of a 16-bit window
      constexpr uint32_t CM = (((1u << VB) - 1u) << (10 - VB)) * 0x10001u;
#pragma unroll
      for (int o = 0; o < DV; o += PER) {
        uint32_t x[2];
        half2_t e2[2], c2[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t a = v[2 * j][0], b = v[2 * j + 1][0];
          if constexpr (VSH) {
            a >>= vsh;
            b >>= vsh;
          }
          if (o * VB == 0) {
            x[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
          } else {
            const int s = o * VB;
            x[j] = __builtin_amdgcn_perm(b >> s, a >> s, 0x05040100u);
          }
          e2[j] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(ec[2 * j + 1], ec[2 * j], 0x05040100u));
          c2[j] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(ec[2 * j + 1], ec[2 * j], 0x07060302u));
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (o + i >= DV) continue;
          uint32_t r[2];
          const int sh = 10 - VB - i * VB;  // the code's bits to the top of the mantissa
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t y = ((sh >= 0 ? x[j] << (sh >= 0 ? sh : 0) : x[j] >> (sh >= 0 ? 0 : -sh)) & CM) | one;
            r[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, y), e2[j], c2[j]));
          }
          put(o + i, r[0], r[1]);
        }
      }
    }
  }
};

template <int D, int KB, int VB, int NH, int CT>
__global__ __launch_bounds__(256, D <= 128 && CT == 1 ? 3 : 2) void tree_fast_kernel(const TreeArgs a) {
  using C = TreeGeo<D>;
  using F = TreeFmt<D, KB, VB>;
  constexpr int TK = C::TK, NT = C::NT, NP = C::NP;
  using W = TreeWave<D, CT, false, NH, false>;
  using B = TreeBuf<D>;
  constexpr int QU = 64 * (D + 4) / 4;
  __shared__ u32x4 pool[2 * B::SIZE > QU ? 2 * B::SIZE : QU];  // two buffers; before: query rows
  __shared__ uint32_t table[F::ENTRIES];
  __shared__ int red[4][2];
  __shared__ uint32_t sigmas[4];

  const int G = a.hq / a.hkv, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TreeMine mine(a, lane);
  TreeSigma<F::RAW ? 2 : 1 << KB> scale;
  float pair[2];
  if constexpr (!F::RAW) {
    scale.fetch(a.cent, lane);
    pair[0] = a.cent[tid & ((1 << KB) - 1)];
    pair[1] = a.cent[(tid >> KB) & ((1 << KB) - 1)];
    const uint32_t best = scale.best(lane, wave);
    if (lane == 0) sigmas[wave] = best;
  }
  TreeUnit u;
  TreePart part;
  if (!tree_share<TK>(a, mine, lane, u, part)) return;
  const uint32_t s_pos = (uint32_t)a.spos;
  const int nb32 = (int)min(a.nb, (int64_t)0x7fffffff);
  // the wave's positions of a tile lie in one run of 16
  const int sub = wave * F::TPW / 16, within = wave * F::TPW % 16;
  const uint8_t* head = a.cache + (int64_t)u.kvh * a.shead + (int64_t)within * a.spos;

  for (; part.blk * 64 * CT < u.n * G; part.blk += a.nblk) {
    W w;
    int first, last;
    w.columns(a, u, part.blk, lane, wave, red, u.len, first, last);  // its barrier: the pool is free
    if constexpr (!F::RAW) {  // pairs of scaled table values (again for a further block)
      const float sg = scale.sigma(min(min(sigmas[0], sigmas[1]), min(sigmas[2], sigmas[3])));
      if (tid < F::ENTRIES) table[tid] = f32_to_f16_bits(sg * pair[0]) | f32_to_f16_bits(sg * pair[1]) << 16;
    }
    first = min(first, u.ctx) / TK;  // the tree's own positions always
    const int held = (int)min((int64_t)u.len, (int64_t)a.max_blocks << a.lbs);  // positions that can have a page
    const int tb0 = part.part == 0 ? first : max(part.tb0, first), tb1 = min(part.tb1, (held + TK - 1) / TK);

    F raw;
    // Block-table entries of the tile to load next, lane k: positions 16 k ..; a
    // vector load in line with the slots', so that nothing waits for it alone
    int entry = -1;
    uint32_t on = 0;  // runs of 16 with a page, of the tile in `raw`
    const int32_t* bt = a.bt + (int64_t)u.b * a.max_blocks;
    auto entries = [&](int t) __attribute__((always_inline)) {
      entry = bt[min((t * TK + 16 * (lane & (NT - 1))) >> a.lbs, a.max_blocks - 1)];
    };
    auto fetch = [&](int t) __attribute__((always_inline)) {  // tile t's bytes, and the next one's entries
      const int pos = t * TK + 16 * (lane & (NT - 1));
      const bool ok = pos < held && (uint32_t)entry < (uint32_t)nb32;
      on = (uint32_t)__builtin_amdgcn_ballot_w64(ok) & ((1u << NT) - 1u);
      const int page = __builtin_amdgcn_readlane(ok ? entry : 0, sub);  // positions without one read block 0
      const int64_t at = (int64_t)page * a.sblk + (int64_t)((t * TK + 16 * sub) & ((1 << a.lbs) - 1)) * a.spos;
      raw.load(head + at, s_pos, lane);
      entries(min(t + 1, tb1 - 1));
    };
    uint32_t now = 0;  // `on` of the tile that is multiplied
    // the queries and the first bytes are on their way together
    typename W::Raw q;
    if (tb0 < tb1) entries(tb0);
    w.fetch(a, u, lane, q);
    if (tb0 < tb1) fetch(tb0);
    w.template queries<F::RAW ? 1 : 0>(a, u, q, lane, reinterpret_cast<float(*)[D + 4]>(pool) + 16 * wave);
    __syncthreads();
    if (tid < 2 * 64 * NP) pool[tid / (64 * NP) * B::SIZE + B::X + tid % (64 * NP)] = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (tb0 < tb1) {
      raw.emit_k(table, pool, wave, lane);
      raw.emit_v(pool, wave, lane);
      now = on;
      fetch(min(tb0 + 1, tb1 - 1));
    }
    // A loop for each number of column tiles in use: every wave meets the others'
    // barriers in its own (a branch inside one loop costs copies of the accumulators).
    auto run = [&](auto use) __attribute__((always_inline)) {
      constexpr int USE = decltype(use)::value;
      int p = 0;
      for (int t = tb0; t < tb1; ++t, p ^= 1) {
        tree_barrier();
        const int pos0 = t * TK;
        const u32x4* buf = pool + p * B::SIZE;
        u32x4* to = pool + (p ^ 1) * B::SIZE;
        // (behind the last tile: it again, for nobody)
        auto beside = [&](auto part) __attribute__((always_inline)) {
          if constexpr (decltype(part)::value == 0) raw.emit_k(table, to, wave, lane);
          else raw.emit_v(to, wave, lane);
        };
        if constexpr (USE > 0) {
          w.template tile<USE>(a, u, buf, buf + B::V, buf + B::X, reinterpret_cast<const float(*)[TK]>(buf + B::T), pos0,
                               pos0 < last || pos0 + TK > u.ctx || now != (1u << NT) - 1u, now, lane, beside);
        } else {
          beside(std::integral_constant<int, 0>{});
          beside(std::integral_constant<int, 1>{});
        }
        now = on;
        fetch(min(t + 2, tb1 - 1));
      }
    };
    if (CT > 1 && w.nct > 1) run(std::integral_constant<int, CT>{});
    else if (w.nct == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 0>{});
    w.finish(a, u, part, lane);
  }
}

template <int D, int KB, int VB, int NH>
hipError_t tree_fast_ct(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) {
  if constexpr (D != 256) {
    if (ct == 2) {
      tree_fast_kernel<D, KB, VB, NH, 2><<<dim3(grid), dim3(256), 0, st>>>(a);
      return hipGetLastError();
    }
  }
  tree_fast_kernel<D, KB, VB, NH, 1><<<dim3(grid), dim3(256), 0, st>>>(a);
  return hipGetLastError();
}
template <int D, int KB, int VB>
hipError_t tree_fast_go(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) {
  return a.ot == BF16 ? tree_fast_ct<D, KB, VB, 1>(a, ct, grid, st) : tree_fast_ct<D, KB, VB, 2>(a, ct, grid, st);
}

// ct: 16-column tiles of a wave
template <int D>
hipError_t tree_fast_launch(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) {
  if (a.kb == TREE_RAW) return tree_fast_go<D, TREE_RAW, TREE_RAW>(a, ct, grid, st);
#define FTQ_TREE_VB(KB)                                         \
  return a.vb == 2   ? tree_fast_go<D, KB, 2>(a, ct, grid, st) \
         : a.vb == 3 ? tree_fast_go<D, KB, 3>(a, ct, grid, st) \
                     : tree_fast_go<D, KB, 4>(a, ct, grid, st)
  if (a.kb == 2) FTQ_TREE_VB(2);
  if (a.kb == 3) FTQ_TREE_VB(3);
  FTQ_TREE_VB(4);
#undef FTQ_TREE_VB
}

}  // namespace ftq
