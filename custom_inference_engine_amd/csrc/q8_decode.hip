// Split-KV decode over the 8-bit paged cache (q8_cache.h), one launch per call.
//
// For sequence b, query head h (kv head g = h / G): o = softmax(q . K^T * D^-0.5) . V
// over the first L tokens of slot slot_ids[b], o = 0 where L = 0.  Entry modes as
// for the fp16 pools (paged_decode.hip): plain (L = lens[b]); append (pos =
// lens[slot], the new row is written at pos and L = pos + 1); append from the fused
// QKV projection's row, q and the new K row rotated; each on its own or from a
// step's plan (cie_paged_decode_plan: it holds slots, lengths, splits and page ids,
// which do not depend on the pools' type).
//
// Work.  The ceil(L / 16) key tiles of a (sequence, kv head) are dealt round-robin to
// its S * 4 waves, wave gw taking tiles gw, gw + 4 S, ... (the plan's deal).  A tile is
// a block of the cache, so a wave's tile comes with one K and one V scale: lane k
// holds the byte offset and the scales of the wave's k-th tile, gathered 64 at a
// time, and a step of q8_tiles tiles reads as many lanes.  A ring of kQ8Pf + 1 steps of
// raw bytes keeps kQ8Pf steps of loads in flight; they are converted when their step
// comes.
// The new row's tile belongs to the wave that it would be dealt to: that wave loads
// the tile's bytes first of all, and after its other tiles rounds the new row under
// the block's new scale, rewrites the block's rows if the scale grew, and attends the
// tile from the registers it wrote; nobody else reads that block.  The result is the
// two-launch one (append, then attend), bit for bit.
// The waves fold through LDS; the last workgroup of a (sequence, kv head) to arrive
// merges the splits' states by log-sum-exp (arrive_last).
//
// What bounds it: the HBM reads of K and V, half the fp16 pools' (96 sequences of 2,048 to 16,384 keys, 32 / 8 heads, D
// = 128: 1.82 GB in 322 us, 5.7 TB/s; fp16 571 us); where those are few, the chain of launch, index, page, tile, fold,
// arrival and merge, about 7 us (32 sequences of 4,096 keys, 14 / 2 heads, D = 64: 12.0 us, 34 MB; 11.5 with a plan).
#include "q8_attn.h"

namespace cie {

constexpr int kQ8Waves = 4;
constexpr int kQ8Threads = kQ8Waves * kWave;
constexpr int kQ8MaxSplits = 64;
constexpr int kQ8PlanDesc = 8;  // a plan's words per workgroup (paged_decode.hip)
// Tiles of a step: its chain (scores, maximum, exponentials, P.V) is what a lone wave on its SIMD waits for, so four
// at D = 64; one step's loads are in flight ahead of the one at work (two: no faster at either D, 3 % slower at 96
// sequences of D = 128, whose second workgroup on a CU hides as much).
template <int D>
constexpr int q8_tiles() {
  return D == 64 ? 4 : 2;
}
constexpr int kQ8Pf = 1;

struct Q8DecodeParams {
  f16* o;
  const f16* q;
  int64_t q_row_stride;
  const f16* cos;
  const f16* sin;
  int64_t cs_stride;
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* scales;
  const f16* k_new;
  const f16* v_new;
  int64_t k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  const int64_t* lens;
  const int64_t* slot_ids;
  const int64_t* block_table;
  float* part_m;    // row (first workgroup of the group + split) * G + head of the group
  float* part_l;
  float* part_acc;  // [row][D]
  int32_t* counters;
  const int32_t* plan;
  int64_t pool_page_stride, pool_head_stride, bt_stride, n_pages;
  int32_t n_wg, bt_width, n_slots, B, H_q, H_kv, G, page_size, n_splits;
  float scale_log2;
  int32_t* err;
};

// 8 dims x from d0 of a row, rotated: y[d] = x[d] cos[d] -+ x[partner] sin[d] (rope8's rounding).
template <int D>
__device__ __forceinline__ f16x8 rope_dims(f16x8 x, f16x8 partner, f16x8 c, f16x8 s, bool low) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = (float)partner[j] * (float)s[j];
    float y = __builtin_fmaf((float)x[j], (float)c[j], low ? -t : t);
    asm volatile("" : "+v"(y));  // one rounding to fp32, then one to fp16, as rope8
    x[j] = (f16)y;
  }
  return x;
}

// A row's dims in the lane's K-operand order.
template <int D>
__device__ __forceinline__ void load_dims(f16x8 (&x)[Geo<D>::KS], const f16* row, int grp) {
#pragma unroll
  for (int ks = 0; ks < Geo<D>::KS; ++ks) x[ks] = *reinterpret_cast<const f16x8*>(row + q8_dim(ks, grp));
}
// Their rotate_half partners: at D = 128 the lane's own k-steps ks ^ 2, at D = 64 another lane's, loaded.
template <int D>
__device__ __forceinline__ void load_partners(f16x8 (&x)[Geo<D>::KS], const f16* row, int grp) {
  if constexpr (D == 64) {
#pragma unroll
    for (int ks = 0; ks < Geo<D>::KS; ++ks) x[ks] = *reinterpret_cast<const f16x8*>(row + (q8_dim(ks, grp) ^ 32));
  }
}
template <int D>
__device__ __forceinline__ void rope_row(f16x8 (&x)[Geo<D>::KS], const f16x8 (&xp)[Geo<D>::KS],
                                         const f16x8 (&c)[Geo<D>::KS], const f16x8 (&s)[Geo<D>::KS], int grp) {
  static_assert(D == 64 || D == 128, "partner layout");
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if constexpr (D == 64) {
      x[ks] = rope_dims<D>(x[ks], xp[ks], c[ks], s[ks], q8_dim(ks, grp) < 32);
    } else {
      rope8(x[ks], x[ks ^ 2], c[ks], c[ks ^ 2], s[ks], s[ks ^ 2]);
    }
  }
}

// Put the new row (kn: the lane's K dims, vn: its V dims) into the tile at row `row` under the block's new
// scales, and the bytes that changed into the pool.  sc: the scales of the block's rows, updated.
template <int D>
__device__ __forceinline__ void append_row(Q8Tile<D>& t, f16x8 (&kn)[Geo<D>::KS],
                                           const typename HVec<Geo<D>::NT>::type& vn, uint8_t* kt, uint8_t* vt,
                                           float* scale, f32x2& sc, int row, int r16, int grp,
                                           const Q8Lane<D>& lo) {
  constexpr int NJ = Q8Tile<D>::NJ;
  typedef typename Q8Tile<D>::vrow_t vrow_t;
  f16x8 v8 = {};
#pragma unroll
  for (int i = 0; i < Geo<D>::NT; ++i) v8[i] = vn[i];
  uint32_t km = 0, vm = q8_raw_max(v8, 0);
#pragma unroll
  for (int ks = 0; ks < Geo<D>::KS; ++ks) km = q8_raw_max(kn[ks], km);
  km = q8_wave_mag(km);
  vm = q8_wave_mag(vm);
  if (max(km, vm) > kQ8Limit) {  // uniform; rare
    km = 0;
#pragma unroll
    for (int ks = 0; ks < Geo<D>::KS; ++ks) {
      km = q8_mag8(kn[ks], km);
      q8_limit8(kn[ks]);
    }
    km = q8_wave_mag(km);
    vm = q8_wave_mag(q8_mag8(v8, 0));
    q8_limit8(v8);
  }
  const bool fresh = row == 0;
  const int k_old = fresh ? kQ8EMin : q8_scale_exponent(sc[0]);
  const int v_old = fresh ? kQ8EMin : q8_scale_exponent(sc[1]);
  const int ke = uniform(max(k_old, q8_exponent(km)));
  const int ve = uniform(max(v_old, q8_exponent(vm)));
  const bool k_all = !fresh && ke != k_old, v_all = !fresh && ve != v_old;  // the block's rows change
  if (k_all) {
    const float f = q8_pow2(k_old - ke);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) t.k[j][i] = q8_rescale4(t.k[j][i], f);
  }
  if (v_all) {
    const float f = q8_pow2(v_old - ve);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < NJ; ++i) t.v[e][i] = q8_rescale4(t.v[e][i], f);
  }
  const float ks = q8_pow2(ke), vs = q8_pow2(ve);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const u32x2 a = q8_round8(kn[2 * j], ks), b = q8_round8(kn[2 * j + 1], ks);
    const u32x4 kq = {a[0], a[1], b[0], b[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) t.k[j][i] = r16 == row ? kq[i] : t.k[j][i];
    if (k_all || r16 == row) *reinterpret_cast<u32x4*>(kt + lo.k + 64 * j) = t.k[j];
  }
  const u32x2 vq = q8_round8(v8, vs);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool mine = 4 * grp + e == row;
#pragma unroll
    for (int i = 0; i < NJ; ++i) t.v[e][i] = mine ? vq[i] : t.v[e][i];
    if (v_all || mine) *reinterpret_cast<vrow_t*>(vt + lo.v + e * D) = t.v[e];
  }
  sc = f32x2{ks, vs};
  if (r16 == 0 && grp == 0) *reinterpret_cast<f32x2*>(scale) = sc;
}

// Merge the S states of every head of a group (rows row0 + s * G + h) into o.  One workgroup does it, so
// memory round trips bound it: the first kLoads acc loads of a thread go out with the m and l loads, one
// split a lane; a wave reduces a head's maximum and sum across its lanes and leaves the splits' weights
// 2^(m - M) / l in LDS.  sm: 16 * kQ8MaxSplits floats, then a f32x4 a thread.
template <int D>
__device__ __forceinline__ void q8_merge(const Q8DecodeParams& p, int64_t row0, int b, int g, int S, int tid,
                                         f32x4* sm) {
  static_assert(kQ8MaxSplits == kWave, "a split per lane");
  constexpr int D4 = D / 4, kLoads = 16, kHeads = 16 / kQ8Waves;
  float* const sm_w = reinterpret_cast<float*>(sm);
  f32x4* const sm_sum = sm + 16 * kQ8MaxSplits / 4;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + row0 * D, (uint32_t)(p.G * S * D * sizeof(float)));
  float ms[kHeads], ls[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = wave + i * kQ8Waves;
    const bool live = h < p.G && lane < S;
    ms[i] = live ? agent_load(&p.part_m[row0 + lane * p.G + h]) : kEmptyMax;
    ls[i] = live ? agent_load(&p.part_l[row0 + lane * p.G + h]) : 0.f;
  }
  const int n_units = p.G * D4;
  const int R = max(1, kQ8Threads / n_units);  // threads a unit (4 dims of a head)
  for (int u0 = 0; u0 < n_units; u0 += kQ8Threads) {
    const int r = R > 1 ? tid / n_units : 0;
    const int unit = u0 + (R > 1 ? tid - r * n_units : tid);
    const bool live = unit < n_units && r < R;
    const int h = live ? unit / D4 : 0;
    const int d4 = unit - h * D4;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = r; s0 < S || s0 == r; s0 += R * kLoads) {
      f32x4 as[kLoads];
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int s = s0 + u * R;  // past the last split: beyond the descriptor, zeros
        const uint32_t off =
            live && s < S ? (uint32_t)(((s * p.G + h) * D + 4 * d4) * sizeof(float)) : 0x7ffffff0u;
        as[u] = agent_load4(racc, off);
      }
      if (u0 == 0 && s0 == r) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const int hh = wave + i * kQ8Waves;
          if (hh < p.G) {  // uniform in the wave
            const float M = q8_wave_max(ms[i]);
            const float a = fast_exp2(ms[i] - M);
            const float den = wave_sum(a * ls[i]);
            sm_w[hh * kQ8MaxSplits + lane] = q8_no_key(den) ? 0.f : a / den;  // no key at all: o = 0
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int s = s0 + u * R;
        num += (live && s < S ? sm_w[h * kQ8MaxSplits + s] : 0.f) * as[u];
      }
    }
    if (R > 1) {
      sm_sum[tid] = num;
      __syncthreads();
      if (live && r == 0)
        for (int i = 1; i < R; ++i) num += sm_sum[tid + i * n_units];
    }
    if (live && r == 0) {
      f16x4 o4;
#pragma unroll
      for (int i = 0; i < 4; ++i) o4[i] = (f16)num[i];
      *reinterpret_cast<f16x4*>(p.o + ((int64_t)b * p.H_q + g * p.G + h) * D + 4 * d4) = o4;
    }
  }
}

// The same for few states: a thread owns 4 dims of a head and takes kFewLoads states a round, each with its m and l, so
// that a round trip and no barrier serve kFewLoads splits (graph replays, 14 / 2 heads, D = 64: 32 sequences of 4,096
// keys, 4 splits, 12.4 us through q8_merge, 11.2 so; 1 of 1,000, 16 splits, 8.6 and 7.0; 4 of 8,000, 32 splits, 10.6 and
// 11.3).
constexpr int kFewLoads = 8, kFewStates = 16;
template <int D>
__device__ __forceinline__ void q8_merge_few(const Q8DecodeParams& p, int64_t row0, int b, int g, int S, int tid) {
  constexpr int D4 = D / 4;
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + row0 * D, (uint32_t)(p.G * S * D * sizeof(float)));
  for (int unit = tid; unit < p.G * D4; unit += kQ8Threads) {
    const int h = unit / D4, d4 = unit - h * D4;
    float M = kEmptyMax, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += kFewLoads) {
      float ms[kFewLoads], ls[kFewLoads];
      f32x4 as[kFewLoads];
#pragma unroll
      for (int u = 0; u < kFewLoads; ++u) {
        ms[u] = kEmptyMax;
        ls[u] = 0.f;
        as[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s0 + u < S) {  // uniform
          const int row = (s0 + u) * p.G + h;
          ms[u] = agent_load(&p.part_m[row0 + row]);
          ls[u] = agent_load(&p.part_l[row0 + row]);
          as[u] = agent_load4(racc, (uint32_t)((row * D + 4 * d4) * sizeof(float)));
        }
      }
      float Mn = M;
#pragma unroll
      for (int u = 0; u < kFewLoads; ++u) Mn = q8_max(Mn, ms[u]);
      const float c = fast_exp2(M - Mn);
      num *= c;
      den *= c;
      M = Mn;
#pragma unroll
      for (int u = 0; u < kFewLoads; ++u) {
        const float a = fast_exp2(ms[u] - M);
        num += a * as[u];
        den += a * ls[u];
      }
    }
    f16x4 o4;
#pragma unroll
    for (int i = 0; i < 4; ++i) o4[i] = (f16)(q8_no_key(den) ? 0.f : num[i] / den);
    *reinterpret_cast<f16x4*>(p.o + ((int64_t)b * p.H_q + g * p.G + h) * D + 4 * d4) = o4;
  }
}

// (leading arguments: preloaded into SGPRs, so the start's first loads need not wait for the argument load)
template <int D, bool kAppend, bool kRope, bool kPlanned>
__global__ __launch_bounds__(kQ8Threads) __attribute__((amdgpu_waves_per_eu(2)))
void q8_decode_kernel(const int64_t* __restrict__ a_slot_ids, const int32_t* __restrict__ a_plan, int32_t a_n_wg,
                      Q8DecodeParams p) {
  static_assert(kAppend || !kRope, "rope mode appends");
  constexpr int KS = Geo<D>::KS;
  constexpr int NT = Geo<D>::NT;
  constexpr int W = kQ8Waves;
  constexpr int PF = kQ8Pf, NS = q8_tiles<D>();
  typedef typename HVec<NT>::type vhalf_t;
  __shared__ float sm_m[W][16];
  __shared__ float sm_l[W][16];
  __shared__ f32x4 sm_acc[W][16][D / 4 + 1];  // (padded rows; the merge's scratch afterwards)
  static_assert(sizeof(sm_acc) >= (16 * kQ8MaxSplits / 4 + kQ8Threads) * sizeof(f32x4), "merge scratch");
  __shared__ int sm_last;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int r16 = lane & 15;
  const int grp = lane >> 4;
  const int tpp = p.page_size >> 4;  // tiles, that is blocks, a page
  const int row_tiles = p.bt_width * tpp;
  const Q8Lane<D> lo(r16, grp);

  // The workgroup's work (split `split` of the S of (b, g)), the L keys to attend, the new row's position,
  // and the page ids of this wave's first 64 tiles, a lane each.  Every load of the start goes out before
  // any check.
  int split, g, b, S, L, pos = -1, w_first, pages = 0;
  int64_t slot;
  f16x8 q[1][KS], qp[KS], cs[KS], sn[KS];
  auto load_q = [&]() {
    const f16* const row = p.q + (int64_t)b * p.q_row_stride + (int64_t)(g * p.G + (r16 < p.G ? r16 : 0)) * D;
    load_dims<D>(q[0], row, grp);
    if constexpr (kRope) {
      load_partners<D>(qp, row, grp);
      load_dims<D>(cs, p.cos + (int64_t)b * p.cs_stride, grp);
      load_dims<D>(sn, p.sin + (int64_t)b * p.cs_stride, grp);
    }
  };
  if constexpr (kPlanned) {
    const int w = blockIdx.x;
    const int32_t* const d = a_plan + (int64_t)w * kQ8PlanDesc;
    pages = a_plan[(int64_t)a_n_wg * kQ8PlanDesc + ((int64_t)w * W + wave) * kWave + lane];
    b = d[0];
    if (b < 0) return;  // idle in this plan (uniform)
    g = d[1];
    split = d[2];
    S = d[3];
    slot = d[4];
    L = d[5];
    pos = d[6];
    w_first = d[7];
    // A plan of another batch or of the other append mode: nothing of it is followed.  (Without partials, which the host
    // allows where the workgroups are as many as the call's (sequence, kv head) pairs, no pair is split; a plan of fewer
    // sequences may be as long and split them.)
    const bool fits = b < p.B && (uint32_t)g < (uint32_t)p.H_kv && (uint32_t)S <= (uint32_t)kQ8MaxSplits &&
                      (uint32_t)split < (uint32_t)S && w_first >= 0 && w_first <= a_n_wg - S &&
                      (uint32_t)d[4] < (uint32_t)p.n_slots && L >= 0 && L <= 16 * row_tiles &&
                      pos == (kAppend ? L - 1 : -1) && (S == 1 || a_n_wg > p.B * p.H_kv);
    // Descriptors come in order: the last live one has to be the call's last pair's, else the plan lacks sequences or
    // heads (theirs stay as they are).  (Past the last descriptor lie page ids, so the word may be read.)
    const int next_b = d[kQ8PlanDesc];
    const bool whole = (w + 1 < a_n_wg && next_b >= 0) || (b == p.B - 1 && g == p.H_kv - 1);
    if (!fits || !whole) set_err(p.err, CIE_ERRBIT_PLAN);
    if (!fits) return;
    load_q();
    if ((uint32_t)pages >= (uint32_t)p.n_pages) {
      set_err(p.err, CIE_ERRBIT_PAGE);
      pages = 0;
    }
  } else {
    split = blockIdx.x;
    g = blockIdx.y;
    b = blockIdx.z;
    S = p.n_splits;
    w_first = (b * p.H_kv + g) * S;
    slot = a_slot_ids[b];
    const bool slot_ok = slot >= 0 && slot < p.n_slots;
    if (!slot_ok) {
      set_err(p.err, CIE_ERRBIT_PAGE);
      slot = 0;
    }
    const int t = split * W + wave + lane * S * W;
    const int64_t page = t < row_tiles ? p.block_table[slot * p.bt_stride + t / tpp] : 0;
    const int64_t len = kAppend ? p.lens[slot] : p.lens[b];
    load_q();
    const int64_t cap = (int64_t)row_tiles * 16;
    L = 0;
    if constexpr (kAppend) {
      if (slot_ok && len >= 0 && len < cap) {
        pos = (int)len;
        L = pos + 1;
      } else if (slot_ok) {
        set_err(p.err, CIE_ERRBIT_LEN);
      }
    } else {
      if (len < 0 || len > cap) set_err(p.err, CIE_ERRBIT_LEN);
      if (slot_ok) L = (int)max((int64_t)0, min(len, cap));
    }
    // (page ids past the sequence may be anything: not used, not reported)
    if (t < ((L + 15) >> 4)) {
      if (page < 0 || page >= p.n_pages)
        set_err(p.err, CIE_ERRBIT_PAGE);
      else
        pages = (int)page;
    }
  }
  split = uniform(split);
  L = uniform(L);
  pos = uniform(pos);
  const int TW = S * W;
  const int gw = uniform(split * W + wave);
  const int n_tiles = (L + 15) >> 4;
  int n_mine = uniform(n_tiles > gw ? (n_tiles - gw + TW - 1) / TW : 0);
  const Q8Src src{p.k_pool, p.v_pool, p.scales, p.pool_page_stride, g * p.pool_head_stride, p.H_kv, g, tpp};

  // Lane k's tile (the wave's tile c0 + k): byte offset in the pools and scales.
  int64_t toff = 0;
  f32x2 tsc = {1.f, 1.f};
  auto lane_tiles = [&](int c0, int page) {
    const int t = gw + (c0 + lane) * TW;
    const int block = t % tpp;
    toff = src.tile(page, block, D);
    if (c0 + lane < n_mine) tsc = *reinterpret_cast<const f32x2*>(src.scale(page, block));
  };
  lane_tiles(0, pages);

  // The tile that holds the new row: its wave takes it out of its list, loads it now and attends it last.
  const bool own_new = kAppend && pos >= 0 && uniform((n_tiles - 1) % TW == gw);
  Q8Tile<D> nt;
  f16x8 kn[KS], knp[KS];
  vhalf_t vn;
  uint8_t *nk = nullptr, *nv = nullptr;
  float* nscale = nullptr;
  f32x2 nsc = {1.f, 1.f};
  if constexpr (kAppend) {
    if (own_new) {
      const int k = n_mine - 1;
      const int block = (n_tiles - 1) % tpp;
      int page;
      if (k < kWave) {
        page = __builtin_amdgcn_readlane(pages, k);
      } else {
        int64_t pg = p.block_table[slot * p.bt_stride + (n_tiles - 1) / tpp];
        if (pg < 0 || pg >= p.n_pages) {
          set_err(p.err, CIE_ERRBIT_PAGE);
          pg = 0;
        }
        page = uniform((int)pg);
      }
      const int64_t off = src.tile(page, block, D);
      nk = p.k_pool + off;
      nv = p.v_pool + off;
      nscale = p.scales + (src.scale(page, block) - p.scales);
      q8_load<D, 0>(nt, q8_rsrc(p.k_pool, off, 16, D), q8_rsrc(p.v_pool, off, 16, D), lo);
      nsc = *reinterpret_cast<const f32x2*>(nscale);
      const f16* const krow = p.k_new + (int64_t)b * p.k_tok_stride + (int64_t)g * p.k_head_stride;
      load_dims<D>(kn, krow, grp);
      if constexpr (kRope) load_partners<D>(knp, krow, grp);
      vn = *reinterpret_cast<const vhalf_t*>(p.v_new + (int64_t)b * p.v_tok_stride + (int64_t)g * p.v_head_stride +
                                             NT * r16);
      --n_mine;
    }
  }

  SoftmaxAcc<D, 1> st;
  st.init();
  const int lim[1] = {L};
  auto prepare_q = [&]() {
    if constexpr (kRope) {
      rope_row<D>(q[0], qp, cs, sn, grp);
      if (own_new) rope_row<D>(kn, knp, cs, sn, grp);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[0][ks] = r16 < p.G ? q[0][ks] : f16x8{};
  };
  // Rotated before the first steps' loads go out at D = 128, where q, k, cos and sin beside them do not fit 256
  // registers; else while those are in flight.
  constexpr bool kFirst = kRope && D == 128;
  if (kFirst || n_mine == 0) prepare_q();
  for (int c0 = 0; c0 < n_mine; c0 += kWave) {
    if (c0 > 0) {
      const int t = gw + (c0 + lane) * TW;
      int64_t pg = 0;
      if (c0 + lane < n_mine) {
        pg = p.block_table[slot * p.bt_stride + t / tpp];
        if (pg < 0 || pg >= p.n_pages) {
          set_err(p.err, CIE_ERRBIT_PAGE);
          pg = 0;
        }
      }
      lane_tiles(c0, (int)pg);
    }
    const int n_chunk = min(kWave, n_mine - c0);
    const int n_steps = (n_chunk + NS - 1) / NS;
    Q8Tile<D> ring[PF + 1][NS];
    // every iteration issues one step's loads (past the last tile: of no rows), so that the wait before a step
    // covers that step's loads only
    auto issue = [&](int i, int j) {
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const int k = NS * j + u;
        const int kk = min(k, n_chunk - 1);
        const int rows = k < n_chunk ? min(16, L - (gw + (c0 + kk) * TW) * 16) : 0;
        const int64_t off = readlane64(toff, kk);
        q8_load<D, kBufNt>(ring[i][u], q8_rsrc(p.k_pool, off, rows, D), q8_rsrc(p.v_pool, off, rows, D), lo);
      }
    };
#pragma unroll
    for (int j = 0; j < PF; ++j) issue(j, j);
    if (!kFirst && c0 == 0) prepare_q();
    for (int j0 = 0; j0 < n_steps; j0 += PF + 1) {
#pragma unroll
      for (int u = 0; u <= PF; ++u) {
        const int j = j0 + u;
        issue((u + PF) % (PF + 1), j + PF);
        if (j < n_steps) {
          int key0[NS];
          f32x2 sc[NS];
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const int k = NS * j + i, kk = min(k, n_chunk - 1);
            key0[i] = k < n_chunk ? (gw + (c0 + kk) * TW) * 16 : kNoKey;
#pragma unroll
            for (int w = 0; w < 2; ++w)
              sc[i][w] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(tsc[w]), kk));
          }
          q8_attend<D, NS>(st, ring[u], sc, q, key0, lim, key0[NS - 1] + 16 > L, p.scale_log2, grp);
        }
      }
    }
  }
  if constexpr (kAppend) {
    if (own_new) {
      const int row = pos & 15;
      append_row<D>(nt, kn, vn, nk, nv, nscale, nsc, row, r16, grp, lo);
      q8_zero_rows<D>(nt, row + 1, grp);
      const Q8Tile<D> pair[2] = {nt, nt};  // (the second copy masked)
      const f32x2 sc[2] = {nsc, nsc};
      const int key0[2] = {pos - row, kNoKey};
      q8_attend<D, 2>(st, pair, sc, q, key0, lim, true, p.scale_log2, grp);
    }
  }

  // Splits that hold a tile: dealt a tile a wave or less, those from this one on are empty (a plan has none).  They
  // arrive, but leave no state.
  const int S_used = kPlanned ? S : min(S, max(1, (n_tiles + W - 1) / W));
  const int64_t row0 = (int64_t)w_first * p.G;
  if (split < S_used) {  // (uniform)
  // Fold the workgroup's waves: a thread folds 4 dims of one head.
  if (grp == 0) {
    sm_m[wave][r16] = st.m[0];
    sm_l[wave][r16] = st.lsum[0][0];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n4 = 0; n4 < NT / 4; ++n4)
      sm_acc[wave][r16][(NT * (4 * grp + r)) / 4 + n4] = f32x4{st.acc[0][4 * n4][r], st.acc[0][4 * n4 + 1][r],
                                                              st.acc[0][4 * n4 + 2][r], st.acc[0][4 * n4 + 3][r]};
  __syncthreads();
  constexpr int D4 = D / 4;
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + row0 * D, S > 1 ? (uint32_t)(p.G * S * D * sizeof(float)) : 0);
  for (int it = threadIdx.x; it < p.G * D4; it += kQ8Threads) {
    const int h = it / D4;
    const int d4 = it - h * D4;
    float M = kEmptyMax;
#pragma unroll
    for (int w = 0; w < W; ++w) M = q8_max(M, sm_m[w][h]);
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float a = fast_exp2(sm_m[w][h] - M);  // (a wave that saw no key: l = 0, acc = 0)
      num += a * sm_acc[w][h][d4];
      den += a * sm_l[w][h];
    }
    if (S == 1) {
      f16x4 o4;
#pragma unroll
      for (int i = 0; i < 4; ++i) o4[i] = (f16)(q8_no_key(den) ? 0.f : num[i] / den);
      *reinterpret_cast<f16x4*>(p.o + ((int64_t)b * p.H_q + g * p.G + h) * D + 4 * d4) = o4;
    } else {
      const int row = split * p.G + h;
      agent_store4(racc, (uint32_t)((row * D + 4 * d4) * sizeof(float)), num);
      if (d4 == 0) {
        agent_store(&p.part_m[row0 + row], M);
        agent_store(&p.part_l[row0 + row], den);
      }
    }
  }
  }
  if (S == 1) return;
  int32_t* const arrival = p.counters + b * p.H_kv + g;
  if (!arrive_last(arrival, (int64_t)p.B * p.H_kv, S, &sm_last, p.err)) return;
  if (S_used <= kFewStates)
    q8_merge_few<D>(p, row0, b, g, S_used, threadIdx.x);
  else
    q8_merge<D>(p, row0, b, g, S_used, threadIdx.x, &sm_acc[0][0][0]);
  if (threadIdx.x == 0) counter_reset(arrival);
}

template <int D, bool kAppend, bool kRope>
static int q8_launch_decode(const Q8DecodeParams& p, hipStream_t stream) {
  if (p.plan)
    hipLaunchKernelGGL((q8_decode_kernel<D, kAppend, kRope, true>), dim3(p.n_wg), dim3(kQ8Threads), 0, stream,
                       p.slot_ids, p.plan, p.n_wg, p);
  else
    hipLaunchKernelGGL((q8_decode_kernel<D, kAppend, kRope, false>), dim3(p.n_splits, p.H_kv, p.B), dim3(kQ8Threads),
                       0, stream, p.slot_ids, p.plan, p.n_wg, p);
  return (int)hipGetLastError();
}

// n_splits: splits a (sequence, kv head), or with a plan its workgroups.
template <bool kAppend, bool kRope>
static int q8_decode_entry(Q8DecodeParams& p, void* partials, int32_t* counters, int64_t B, int64_t H_q, int64_t H_kv,
                           int64_t D, int64_t page_size, int64_t n_pages, int64_t pool_page_stride,
                           int64_t pool_head_stride, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                           int64_t n_splits, int32_t* err, void* stream) {
  if (B < 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || n_pages <= 0 || bt_width <= 0 || bt_stride < bt_width ||
      n_slots <= 0 || n_splits <= 0 || page_size <= 0)
    return CIE_EINVAL;
  if (B == 0) return CIE_OK;
  if (!p.o || !p.q || !p.k_pool || !p.v_pool || !p.scales || !p.block_table || (!p.plan && (!p.lens || !p.slot_ids)))
    return CIE_EINVAL;
  const int64_t G = H_q / H_kv;
  if (G > 16 || (D != 64 && D != 128) || page_size % 16 != 0 || B > 65535 || H_kv > 65535 ||
      (!p.plan && n_splits > kQ8MaxSplits) || n_splits > 0x7fffffff || bt_width > 0x7fffffff / page_size ||
      n_pages > 0x7fffffff)
    return CIE_EUNSUPPORTED;
  // (a plan gives every (sequence, kv head) one workgroup at least, kQ8MaxSplits at most)
  if (p.plan && (n_splits < B * H_kv || n_splits % H_kv != 0 || n_splits > B * H_kv * kQ8MaxSplits)) return CIE_EINVAL;
  const int64_t n_wg = p.plan ? n_splits : B * H_kv * n_splits;
  if (n_wg > 0x7fffffff) return CIE_EUNSUPPORTED;
  if (n_wg > B * H_kv && (!partials || !counters)) return CIE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k_pool) |
       reinterpret_cast<uintptr_t>(p.v_pool) | reinterpret_cast<uintptr_t>(p.scales) |
       reinterpret_cast<uintptr_t>(partials) | reinterpret_cast<uintptr_t>(counters)) & 15)
    return CIE_EINVAL;
  if (pool_page_stride % 16 != 0 || pool_head_stride % 16 != 0) return CIE_EINVAL;
  // partials as cie_paged_decode_planned_partials_bytes lays them out: m | l | acc, 256-byte regions
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  const int64_t rows = n_wg * G;
  char* const ws = static_cast<char*>(partials);
  p.part_m = reinterpret_cast<float*>(ws);
  p.part_l = reinterpret_cast<float*>(ws + up(rows * 4));
  p.part_acc = reinterpret_cast<float*>(ws + up(up(rows * 4) + rows * 4));
  p.counters = counters;
  p.pool_page_stride = pool_page_stride;
  p.pool_head_stride = pool_head_stride;
  p.bt_stride = bt_stride;
  p.n_pages = n_pages;
  p.bt_width = (int32_t)bt_width;
  p.n_slots = (int32_t)(n_slots > 0x7fffffff ? 0x7fffffff : n_slots);
  p.B = (int32_t)B;
  p.H_q = (int32_t)H_q;
  p.H_kv = (int32_t)H_kv;
  p.G = (int32_t)G;
  p.page_size = (int32_t)page_size;
  p.n_splits = (int32_t)n_splits;
  p.n_wg = (int32_t)n_wg;
  p.scale_log2 = kLog2e / __builtin_sqrtf((float)D);
  p.err = err;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return D == 64 ? q8_launch_decode<64, kAppend, kRope>(p, s) : q8_launch_decode<128, kAppend, kRope>(p, s);
}

static Q8DecodeParams q8_decode_params(void* o, const void* q, int64_t q_row_stride, void* k_pool, void* v_pool,
                                       void* scales, const int64_t* lens, const int64_t* slot_ids,
                                       const int64_t* block_table, const int32_t* plan) {
  Q8DecodeParams p{};
  p.o = static_cast<f16*>(o);
  p.q = static_cast<const f16*>(q);
  p.q_row_stride = q_row_stride;
  p.k_pool = static_cast<uint8_t*>(k_pool);
  p.v_pool = static_cast<uint8_t*>(v_pool);
  p.scales = static_cast<float*>(scales);
  p.lens = lens;
  p.slot_ids = slot_ids;
  p.block_table = block_table;
  p.plan = plan;
  return p;
}

static bool rows_aligned(const void* ptr, int64_t s0, int64_t s1) {
  return ptr && !(reinterpret_cast<uintptr_t>(ptr) & 15) && s0 % 8 == 0 && s1 % 8 == 0;
}

}  // namespace cie

using namespace cie;

extern "C" int cie_q8_decode(void* o, const void* q, const void* k_pool, const void* v_pool, const void* scales,
                             const int64_t* lens, const int64_t* slot_ids, const int64_t* block_table,
                             const int32_t* plan, void* partials, int32_t* counters, int64_t B, int64_t H_q,
                             int64_t H_kv, int64_t D, int64_t page_size, int64_t n_pages, int64_t pool_page_stride,
                             int64_t pool_head_stride, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                             int64_t n_splits, int32_t* err, void* stream) {
  Q8DecodeParams p = q8_decode_params(o, q, H_q * D, const_cast<void*>(k_pool), const_cast<void*>(v_pool),
                                      const_cast<void*>(scales), lens, slot_ids, block_table, plan);
  return q8_decode_entry<false, false>(p, partials, counters, B, H_q, H_kv, D, page_size, n_pages, pool_page_stride,
                                       pool_head_stride, bt_stride, bt_width, n_slots, n_splits, err, stream);
}

extern "C" int cie_q8_decode_append(void* o, const void* q, void* k_pool, void* v_pool, void* scales,
                                    const void* k_new, const void* v_new, int64_t k_tok_stride, int64_t k_head_stride,
                                    int64_t v_tok_stride, int64_t v_head_stride, const int64_t* lens,
                                    const int64_t* slot_ids, const int64_t* block_table, const int32_t* plan,
                                    void* partials, int32_t* counters, int64_t B, int64_t H_q, int64_t H_kv, int64_t D,
                                    int64_t page_size, int64_t n_pages, int64_t pool_page_stride,
                                    int64_t pool_head_stride, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                                    int64_t n_splits, int32_t* err, void* stream) {
  if (B > 0 && (!rows_aligned(k_new, k_tok_stride, k_head_stride) || !rows_aligned(v_new, v_tok_stride, v_head_stride)))
    return CIE_EINVAL;
  Q8DecodeParams p = q8_decode_params(o, q, H_q * D, k_pool, v_pool, scales, lens, slot_ids, block_table, plan);
  p.k_new = static_cast<const f16*>(k_new);
  p.v_new = static_cast<const f16*>(v_new);
  p.k_tok_stride = k_tok_stride;
  p.k_head_stride = k_head_stride;
  p.v_tok_stride = v_tok_stride;
  p.v_head_stride = v_head_stride;
  return q8_decode_entry<true, false>(p, partials, counters, B, H_q, H_kv, D, page_size, n_pages, pool_page_stride,
                                      pool_head_stride, bt_stride, bt_width, n_slots, n_splits, err, stream);
}

extern "C" int cie_q8_decode_qkv_rope(void* o, const void* qkv, int64_t qkv_row_stride, const void* cos,
                                      const void* sin, int64_t cs_row_stride, void* k_pool, void* v_pool, void* scales,
                                      const int64_t* lens, const int64_t* slot_ids, const int64_t* block_table,
                                      const int32_t* plan, void* partials, int32_t* counters, int64_t B, int64_t H_q,
                                      int64_t H_kv, int64_t D, int64_t page_size, int64_t n_pages,
                                      int64_t pool_page_stride, int64_t pool_head_stride, int64_t bt_stride,
                                      int64_t bt_width, int64_t n_slots, int64_t n_splits, int32_t* err,
                                      void* stream) {
  if (B < 0 || H_q <= 0 || H_kv <= 0 || D <= 0) return CIE_EINVAL;
  if (B > 0 && (!rows_aligned(qkv, qkv_row_stride, 0) || !rows_aligned(cos, cs_row_stride, 0) ||
                !rows_aligned(sin, cs_row_stride, 0) || qkv_row_stride < (H_q + 2 * H_kv) * D || cs_row_stride < D))
    return CIE_EINVAL;
  Q8DecodeParams p = q8_decode_params(o, qkv, qkv_row_stride, k_pool, v_pool, scales, lens, slot_ids, block_table, plan);
  const f16* const row = static_cast<const f16*>(qkv);
  p.k_new = row + H_q * D;
  p.v_new = row + (H_q + H_kv) * D;
  p.k_tok_stride = p.v_tok_stride = qkv_row_stride;
  p.k_head_stride = p.v_head_stride = D;
  p.cos = static_cast<const f16*>(cos);
  p.sin = static_cast<const f16*>(sin);
  p.cs_stride = cs_row_stride;
  return q8_decode_entry<true, true>(p, partials, counters, B, H_q, H_kv, D, page_size, n_pages, pool_page_stride,
                                     pool_head_stride, bt_stride, bt_width, n_slots, n_splits, err, stream);
}
