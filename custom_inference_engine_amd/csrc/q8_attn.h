// Attention over 8-bit key tiles (q8_cache.h): tile loads, conversion and the
// 32-key step, shared by the decode and mixed kernels.
//
// As in attn_engine.h a wave computes S^T = K . Q^T and O^T = V^T . P^T with
// v_mfma_f32_16x16x32_f16, up to 16 query columns per column tile.  Operand layout
// (lane l, r16 = l % 16, grp = l / 16), chosen for byte rows:
//   K tile: lane holds bytes [64 j + 16 grp, + 16) of key r16, j < D / 64: one
//     16-byte load per 64 dims (a wave reads 1 KiB in one piece).  The order of the
//     dims in the dot product is free, so k-step 2 j + i takes bytes 8 i .. 8 i + 7 of
//     them, and Q is loaded in that order (q8_dim).
//   V tile: lane holds bytes [NT r16, + NT) of rows 4 grp + e, e < 4 (a group reads
//     whole rows).  Bytes of two rows are brought side by side (v_perm), so one
//     conversion gives the two keys of an operand register.
// The converted values are the cache's own, exactly (its scales are applied by the
// conversion), so what follows is the fp16 kernels' arithmetic: P rounded to fp16
// (2^-11 of each weight, the cache's own rounding is 2^-4), sums in fp32.
#pragma once

#include "attn_engine.h"
#include "q8_cache.h"

namespace cie {

// First dim of the 8 that k-step ks takes in lane group grp.
__device__ __forceinline__ int q8_dim(int ks, int grp) { return 64 * (ks >> 1) + 16 * grp + 8 * (ks & 1); }

// Raw bytes of one 16-key tile.
template <int D>
struct Q8Tile {
  static constexpr int NJ = D / 64;
  typedef uint32_t vrow_t __attribute__((ext_vector_type(NJ)));
  u32x4 k[NJ];
  vrow_t v[4];
};

// Lane's byte offsets in a tile.
template <int D>
struct Q8Lane {
  uint32_t k, v;
  __device__ __forceinline__ Q8Lane(int r16, int grp)
      : k((uint32_t)(r16 * D + 16 * grp)), v((uint32_t)(4 * grp * D + Geo<D>::NT * r16)) {}
};

// A tile's rows as a raw buffer (attn_engine.h, tile_rsrc): rows at or past `rows` read as zeros and
// touch no memory, so a sequence's last tile costs its rows only and an absent tile (0 rows) nothing.
// All arguments wave-uniform.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t q8_rsrc(const uint8_t* pool, int64_t off, int rows, int D) {
  return coherent_rsrc(pool + off, (uint32_t)__builtin_amdgcn_readfirstlane(rows * D));
}

// A call reads each K/V byte once per workgroup: past the caches' reuse (nt).
template <int D, int POL>
__device__ __forceinline__ void q8_load(Q8Tile<D>& t, __amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv,
                                        const Q8Lane<D>& lo) {
  typedef typename Q8Tile<D>::vrow_t vrow_t;
#pragma unroll
  for (int j = 0; j < Q8Tile<D>::NJ; ++j)
    t.k[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, lo.k + 64 * j, 0, POL));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (D == 64)
      t.v[e] = __builtin_bit_cast(vrow_t, __builtin_amdgcn_raw_buffer_load_b32(rv, lo.v + e * D, 0, POL));
    else
      t.v[e] = __builtin_bit_cast(vrow_t, __builtin_amdgcn_raw_buffer_load_b64(rv, lo.v + e * D, 0, POL));
  }
}

// A tile's K operands.
template <int D>
__device__ __forceinline__ void q8_k_operand(f16x8 (&k)[Geo<D>::KS], const Q8Tile<D>& t, float scale) {
#pragma unroll
  for (int j = 0; j < Q8Tile<D>::NJ; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) k[2 * j + i] = q8_values8(t.k[j][2 * i], t.k[j][2 * i + 1], scale);
}

// Rows 4 grp + e at or past n_rows become zeros: a masked key's weight is 0, but its bytes may hold
// anything (NaN among it).
template <int D>
__device__ __forceinline__ void q8_zero_rows(Q8Tile<D>& t, int n_rows, int grp) {
  typedef typename Q8Tile<D>::vrow_t vrow_t;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * grp + e >= n_rows) t.v[e] = vrow_t{};
}

// NaN among V where keys are masked.  A masked key's weight is 0, but 0 times NaN is NaN, in every column of the tile.
// So a tile that holds one takes part with zeros in its place, and leaves a map in LDS, [key][r16] a byte with a bit for
// each of dims NT r16 + 0 .. NT - 1; q8_nan_fix then makes NaN what the columns that attend such a key hold.  (Rare.)
constexpr int kQ8NanMap = kQ8Block * 16;  // bytes a tile

// The NaNs of a tile's V words, as the top bits of their bytes.
__device__ __forceinline__ uint32_t q8_nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Whether a V byte of the wave's tile is a NaN (uniform).
template <int D>
__device__ __forceinline__ bool q8_has_nan(const Q8Tile<D>& t) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < Q8Tile<D>::NJ; ++w) m |= q8_nan_bytes(t.v[e][w]);
  return __any(m != 0);
}

template <int D>
__device__ __forceinline__ void q8_nan_map(Q8Tile<D>& t, uint8_t* map, int r16, int grp) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t bits = 0;
#pragma unroll
    for (int w = 0; w < Q8Tile<D>::NJ; ++w) {
      const uint32_t m = q8_nan_bytes(t.v[e][w]) >> 7;
      bits |= (m * 0x10204080u >> 28) << (4 * w);
      t.v[e][w] &= ~(m * 0xffu);
    }
    map[(4 * grp + e) * 16 + r16] = (uint8_t)bits;
  }
}

// hit[c]: byte r the bits of dims NT (4 grp + r) + nt that hold a NaN among the keys that column c attends, of the tile
// of `map`, whose first key is key0.
template <int NCT>
__device__ __forceinline__ void q8_nan_hits(uint32_t (&hit)[NCT], const uint8_t* map, int key0, const int (&lim)[NCT],
                                            int grp) {
  for (int key = 0; key < kQ8Block; ++key) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(map + key * 16 + 4 * grp);
#pragma unroll
    for (int c = 0; c < NCT; ++c) hit[c] |= key0 + key < lim[c] ? word : 0u;
  }
}

template <int D, int NCT>
__device__ __forceinline__ void q8_nan_fix(SoftmaxAcc<D, NCT>& st, const uint32_t (&hit)[NCT]) {
#pragma unroll
  for (int c = 0; c < NCT; ++c)
#pragma unroll
    for (int nt = 0; nt < Geo<D>::NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        st.acc[c][nt][r] = hit[c] >> (8 * r + nt) & 1 ? __builtin_nanf("") : st.acc[c][nt][r];
}

// Keys 4 grp + 0 .. 3 of a tile as elements 4 half .. 4 half + 3 of the V^T operands (dim NT r16 + nt).
template <int D>
__device__ __forceinline__ void q8_v_operand(f16x8 (&va)[Geo<D>::NT], int half, const Q8Tile<D>& t, float scale) {
#pragma unroll
  for (int w = 0; w < Q8Tile<D>::NJ; ++w) {
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {  // keys 2 pr, 2 pr + 1
      const uint32_t a = t.v[2 * pr][w], b = t.v[2 * pr + 1][w];
      const uint32_t d01 = __builtin_amdgcn_perm(b, a, 0x05010400);  // {a0, b0, a1, b1}
      const uint32_t d23 = __builtin_amdgcn_perm(b, a, 0x07030602);
      const f16x2 x[4] = {q8_pair<false>(d01, scale), q8_pair<true>(d01, scale), q8_pair<false>(d23, scale),
                          q8_pair<true>(d23, scale)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        va[4 * w + i][4 * half + 2 * pr] = x[i][0];
        va[4 * w + i][4 * half + 2 * pr + 1] = x[i][1];
      }
    }
  }
}

// A state that saw no key (its sum is 0; a NaN among the attended values leaves a NaN, which is not).
__device__ __forceinline__ bool q8_no_key(float l) { return l == 0.f; }

// The larger of two, NaN if either is (v_maximum3_f32 takes operands as they are, where fmaxf's v_max_f32 needs each
// made canonical first).  A NaN score is its column's whole result, so no maximum has to look past it.
__device__ __forceinline__ float q8_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// As col_max4 and wave_max, so.
__device__ __forceinline__ float q8_col_max4(float x) {
  float a, b;
  swap16(x, a, b);
  swap32(q8_max(a, b), a, b);
  return q8_max(a, b);
}
__device__ __forceinline__ float q8_wave_max(float x) {
  x = q8_max(x, row_ror<8>(x));
  x = q8_max(x, row_ror<4>(x));
  x = q8_max(x, row_ror<2>(x));
  x = q8_max(x, row_ror<1>(x));
  return q8_col_max4(x);
}

// One step of NP 32-key pairs of tiles for NCT column tiles.  k(i, ka) gives the K operands of tile i (< 2 NP), whose
// first key is key0[i] (kNoKey: absent, all masked), v(p, va) the V^T operands of pair p once the weights are known;
// meanwhile() is work that needs nothing of the step, done while its S MFMAs run.
// lim[c]: keys the lane's column attends; mask: some key of the step may be at or past one of them.  Phase by phase,
// so that a wave overlaps the VALU work and the MFMAs of its column tiles and pairs; attend_pair_body's softmax.
template <int D, int NCT, int NP, bool LDS, class K, class V, class M>
__device__ __forceinline__ void q8_step(SoftmaxAcc<D, NCT>& st, K k, V v, M meanwhile, const f16x8 (&q)[NCT][Geo<D>::KS],
                                        const int (&key0)[2 * NP], const int (&lim)[NCT], bool mask, float scale_log2,
                                        int grp) {
  constexpr int KS = Geo<D>::KS;
  constexpr int NT = Geo<D>::NT;
  f32x4 s[NCT][2 * NP];
  // Waves of two workgroups share a SIMD: at D = 64, where a step is mostly VALU work, the one that has MFMAs to issue
  // goes first (4 x 2,048 rows, 14 / 2 heads: 49.4 -> 47.4 us, 300 rows over 8,192 keys 39.6 -> 36.3, 8,192 rows of 8 / 8
  // heads 136 -> 141; at D = 128 ragged chunks 150 -> 160).
  constexpr bool kFirst = LDS && D == 64;
  if (kFirst) __builtin_amdgcn_s_setprio(1);
  f16x8 ka[2][KS];  // a tile's operands are fetched while the one before it is multiplied
  k(0, ka[0]);
#pragma unroll
  for (int i = 0; i < 2 * NP; ++i) {
    if (i + 1 < 2 * NP) k(i + 1, ka[(i + 1) % 2]);
    if (LDS) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < NCT; ++c) s[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int c = 0; c < NCT; ++c) s[c][i] = mfma16x16x32(ka[i % 2][ks], q[c][ks], s[c][i]);
    if (LDS) __builtin_amdgcn_sched_barrier(0);
  }
  meanwhile();
  if (kFirst) __builtin_amdgcn_s_setprio(0);
  if (mask) {
#pragma unroll
    for (int c = 0; c < NCT; ++c)
#pragma unroll
      for (int i = 0; i < 2 * NP; ++i) {
        // (the asm keeps this a branch: most steps mask nothing, and selects nearly double a step's VALU work)
        asm volatile("" : "+v"(s[c][i]));
#pragma unroll
        for (int r = 0; r < 4; ++r) s[c][i][r] = key0[i] + 4 * grp + r < lim[c] ? s[c][i][r] : kNegInf;
      }
  }
  float xb[NCT];
  bool need = false;
#pragma unroll
  for (int c = 0; c < NCT; ++c) {
    xb[c] = s[c][0][0];
#pragma unroll
    for (int i = 1; i < 8 * NP; ++i) xb[c] = q8_max(xb[c], s[c][i / 4][i % 4]);
    need |= xb[c] > st.thr[c];
  }
  if (__any(need)) {  // rare: move the reference max
#pragma unroll
    for (int c = 0; c < NCT; ++c) {
      const float m_new = q8_max(st.m[c], q8_col_max4(xb[c]) * scale_log2);
      const float alpha = fast_exp2(st.m[c] - m_new);
      st.m[c] = m_new;
      st.thr[c] = (m_new + kRescaleSlack) / scale_log2;
      st.lsum[c][0] *= alpha;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) st.acc[c][nt] *= alpha;
    }
  }
  const f16x8 ones = {(f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f};
#pragma unroll
  for (int pr = 0; pr < NP; ++pr) {
    f16x8 va[NT];
    if (LDS) {
      v(pr, va);  // (from LDS: fetched while the exponentials run)
      __builtin_amdgcn_sched_barrier(0);
    }
    f16x8 p[NCT];
#pragma unroll
    for (int c = 0; c < NCT; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[c][e] = (f16)fast_exp2(__builtin_fmaf(s[c][2 * pr + e / 4][e % 4], scale_log2, -st.m[c]));
    if (!LDS) v(pr, va);
#pragma unroll
    for (int c = 0; c < NCT; ++c) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) st.acc[c][nt] = mfma16x16x32(va[nt], p[c], st.acc[c][nt]);
      st.lsum[c] = mfma16x16x32(ones, p[c], st.lsum[c]);
    }
  }
}

// The same for one column tile from raw tiles: NT2 = 2 NP of them with their K and V scales.
template <int D, int NT2>
__device__ __forceinline__ void q8_attend(SoftmaxAcc<D, 1>& st, const Q8Tile<D> (&t)[NT2], const f32x2 (&sc)[NT2],
                                          const f16x8 (&q)[1][Geo<D>::KS], const int (&key0)[NT2], const int (&lim)[1],
                                          bool mask, float scale_log2, int grp) {
  auto k = [&](int i, f16x8 (&ka)[Geo<D>::KS]) { q8_k_operand<D>(ka, t[i], sc[i][0]); };
  auto v = [&](int pr, f16x8 (&va)[Geo<D>::NT]) {
    q8_v_operand<D>(va, 0, t[2 * pr], sc[2 * pr][1]);
    q8_v_operand<D>(va, 1, t[2 * pr + 1], sc[2 * pr + 1][1]);
  };
  q8_step<D, 1, NT2 / 2, false>(st, k, v, [] {}, q, key0, lim, mask, scale_log2, grp);
}

// The same where several rows share the column tile, so that a key that one masks may be another's.  map: the wave's,
// kQ8NanMap bytes a tile.
template <int D, int NT2>
__device__ __forceinline__ void q8_attend_rows(SoftmaxAcc<D, 1>& st, Q8Tile<D> (&t)[NT2], const f32x2 (&sc)[NT2],
                                               const f16x8 (&q)[1][Geo<D>::KS], const int (&key0)[NT2],
                                               const int (&lim)[1], bool mask, float scale_log2, uint8_t* map, int r16,
                                               int grp) {
  uint32_t hit[1] = {0};
  if (mask) {
#pragma unroll
    for (int i = 0; i < NT2; ++i) {
      if (!q8_has_nan<D>(t[i])) continue;
      q8_nan_map<D>(t[i], map + i * kQ8NanMap, r16, grp);
      __builtin_amdgcn_wave_barrier();
      q8_nan_hits<1>(hit, map + i * kQ8NanMap, key0[i], lim, grp);
    }
  }
  q8_attend<D, NT2>(st, t, sc, q, key0, lim, mask, scale_log2, grp);
  if (__any(hit[0] != 0)) q8_nan_fix<D, 1>(st, hit);
}

// Where a wave's tiles live: kv head g of the pools and of the scales.
struct Q8Src {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* scales;
  int64_t page_stride, head_off;  // bytes
  int32_t H_kv, g, per;           // per: blocks a page
  __device__ __forceinline__ int64_t tile(int page, int block, int D) const {
    return (int64_t)page * page_stride + head_off + (int64_t)block * (kQ8Block * D);
  }
  __device__ __forceinline__ const float* scale(int page, int block) const {
    return scales + 2 * (((int64_t)page * H_kv + g) * per + block);
  }
};

}  // namespace cie
