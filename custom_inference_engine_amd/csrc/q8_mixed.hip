// Varlen causal attention over the 8-bit paged cache (q8_cache.h): chunked prefill
// and decode rows in one launch, from a plan made once per step.
//
// Sequence b owns query rows [cu_seqlens[b], cu_seqlens[b + 1]); its row i sits at
// position kv_lens[b] + i and attends keys 0 .. kv_lens[b] + i of slot slot_ids[b].
// Rows outside every sequence are left untouched.
//
// Work.  A query tile is up to R rows of a sequence and one kv head: R * G <= kTileCols
// (row, head) columns, or half of that in small launches.  An item is a tile and a
// range of its key tiles.
//  * Wide items (more than 16 columns): every wave has one or two column tiles of 16
//    and all keys of the item.  Keys go by stages of 64: wave w loads the stage's
//    16-key tile w as bytes (so its page and its two scales are scalars), converts it
//    once and leaves it in LDS in MFMA operand order (K: slot [tile][k-step][lane];
//    V^T: [pair][dim tile][lane]), where a lane writes its own slots and every wave
//    reads the same ones: 16-byte accesses without bank conflicts.  Converting in the
//    loader costs each value once per workgroup instead of once per wave.  Two
//    buffers, one barrier a stage, the next stage's bytes in flight in registers.
//  * Narrow items (a decode row and its like: 16 columns or fewer): one column tile,
//    its keys dealt over the four waves, straight from registers as the decode
//    kernel does; the waves fold through LDS.
// A tile whose keys exceed the plan's share is split over several items; each
// leaves its state (m, l, acc) in `partials` and the last to arrive merges them.
//
// The plan (q8_mixed_plan_kernel, one workgroup) sizes that share so that the
// launch has about kQ8Slots items' worth of work, and lists the items, longest
// first.  It depends on the step's sequences only, so a step makes it once for all
// its layers.
//
// What bounds it: prefill of several rounds of items, the softmax's VALU work between
// the MFMAs (a step of 32 keys costs a wave 18 MFMAs and 16 exponentials at D = 64 and two
// column tiles): 4 x 8,192 rows, 14 / 2 heads, D = 64, 506 us, 950 TFLOP/s; 8,192 rows, 32 /
// 8 heads, D = 128, 505 us, 1,088 TFLOP/s (a large fp16 product reaches 1,135).  Launches
// whose items all start at once last as long as the longest: 8,192 rows, 8 / 8 heads, D =
// 64, 512 items of up to 128 stages, 65 on average, 131 us, 526 TFLOP/s.  Decode rows, the
// K/V reads and the chain around them (32 rows over 8,000 keys 15.8 us).
#include "q8_attn.h"

namespace cie {

constexpr int kMW = 4;  // waves a workgroup
constexpr int kMThreads = kMW * kWave;
constexpr int kQ8Slots = 256;        // items a launch's work is cut into, about
constexpr int kMaxSplitItems = 2 * kQ8Slots;  // (see the plan)
constexpr int kQ8MinShare = 32;  // key tiles (512 keys): below, an item's start costs more than its keys
constexpr int kQ8MaxSeqs = 2048;
constexpr int kItemWords = 12;
constexpr int kHeadWords = 12;
constexpr int kQ8MaxChunks = 48;  // items of a split tile at most (one workgroup merges them)
constexpr int kPlanThreadsM = 512;
constexpr int kPlanMagic = 0x71386d31;

// Column tiles of a wave, and columns of a wide tile, at most.
constexpr int kQ8Ct = 2;
constexpr int kTileCols = 16 * kMW * kQ8Ct;

struct Q8Item {
  int tok0;    // packed row of the tile's first row
  int rows;    // rows, negative: a narrow item
  int g, slot;
  int pos0;    // position of the first row
  int t0, t1;  // key tiles
  int chunk, n_chunks;
  int pbase;   // first partial row of the tile (split tiles): row pbase + chunk * columns + column
  int ctr;     // its arrival word
  int pad;
};
static_assert(sizeof(Q8Item) == kItemWords * 4, "item layout");

struct Q8MixedParams {
  f16* o;
  const f16* q;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* scales;
  const int64_t* block_table;
  const int32_t* plan;
  float* part_m;
  float* part_l;
  float* part_acc;
  int32_t* counters;
  int64_t pool_page_stride, pool_head_stride, bt_stride, n_pages, total_T;
  int32_t part_cap, n_ctr, plan_cap, B, bt_width, n_slots, H_q, H_kv, G, page_size;
  uint32_t g_magic;
  float scale_log2;
  int32_t* err;
};

// ---- the plan ----

struct Q8PlanParams {
  int32_t* plan;
  const int64_t* cu_seqlens;
  const int64_t* kv_lens;
  const int64_t* slot_ids;
  int64_t total_T, cap;  // cap: keys a block-table row holds
  int32_t B, bt_width, n_slots, H_q, H_kv, G, page_size, D, max_rows, part_cap, plan_cap;
  int32_t* err;
};

// What a plan was made for (its first words, after the item count): a call with other sizes writes nothing.
template <class P>
__device__ __forceinline__ int plan_word(const P& p, int i, int D) {
  const int w[kHeadWords - 1] = {kPlanMagic, p.B, (int)p.total_T, p.H_q, p.H_kv, D, p.page_size, p.bt_width,
                                 p.n_slots, p.part_cap, p.plan_cap};
  return w[i];
}

struct Q8Seq {
  int64_t t0;
  int slot, L, c;
};

__device__ __forceinline__ Q8Seq q8_seq(const Q8PlanParams& p, int b, bool report) {
  Q8Seq s{0, 0, 0, 0};
  const int64_t t0 = p.cu_seqlens[b], t1 = p.cu_seqlens[b + 1], slot = p.slot_ids[b], c = p.kv_lens[b];
  if (t1 == t0) return s;
  if (t0 < 0 || t1 < t0 || t1 > p.total_T || slot < 0 || slot >= p.n_slots) {
    if (report) set_err(p.err, CIE_ERRBIT_PAGE);
    return s;
  }
  if (c < 0 || c > p.cap || c + (t1 - t0) > p.cap) {
    if (report) set_err(p.err, CIE_ERRBIT_LEN);
    return s;
  }
  if (t1 - t0 > p.max_rows && report) set_err(p.err, CIE_ERRBIT_LEN);
  s.t0 = t0;
  s.slot = (int)slot;
  s.L = (int)min((int64_t)p.max_rows, t1 - t0);
  s.c = (int)c;
  return s;
}

// How a sequence is cut: its tiles' rows, and key tiles an item at most (once the launch's `want` is known).
struct Q8Cut {
  bool narrow;
  int R, n_rt, share;
  __device__ __forceinline__ Q8Cut(const Q8PlanParams& p, int L, int cols, int want) {
    narrow = (int64_t)L * p.G <= 16;
    R = narrow ? max(1, L) : cols / p.G;
    n_rt = (L + R - 1) / R;
    share = (max(kQ8MinShare, narrow ? 4 * want : want) + 3) & ~3;
  }
};

constexpr int kPlanWavesM = kPlanThreadsM / kWave;

// Exclusive prefix sums of N values over the workgroup's threads, and their sums, with one barrier; red: not read by
// anyone since the last.
template <int N>
__device__ __forceinline__ void plan_block_scan(const int (&v)[N], int (&before)[N], int (&all)[N],
                                                int (&red)[N][kPlanWavesM]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = wave_inclusive_sum(v[i]);
  if (lane == kWave - 1)
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][wave] = inc[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int base = 0;
    all[i] = 0;
#pragma unroll
    for (int w = 0; w < kPlanWavesM; ++w) {
      const int x = red[i][w];
      base += w < wave ? x : 0;
      all[i] += x;
    }
    before[i] = base + inc[i] - v[i];
  }
}

// One workgroup: a thread up to kSeqsPer sequences in order, then a thread a query tile.  Barriers are most of its time
// (five, where a batch has no more than kPlanThreadsM tiles).
//
// Columns of a wide tile: with W the launch's work in key tiles of wide items of kTileCols columns (a narrow item's
// key tile counts a quarter), a launch of W <= kSmallWork * kQ8Slots takes tiles of half as many, one column tile a
// wave: such a launch lasts as long as its items, whose stages are then shorter, and it has CUs for more of them (100
// rows over 900 keys, 14 / 2 heads, D = 64: 17 -> 14 us; 32 / 8 heads, D = 128: 24 -> 18; 512 over 4,096: 34 -> 32).
// Larger ones pay the K/V operands' conversion and LDS reads twice (4 x 8,192 rows: 568 us whole, 710 in halves).
//
// Key tiles an item holds at most: want = W / kQ8Slots (W in the tiles taken), 4 want for narrow items, and kQ8MinShare
// at least.  A tile of kt > share key tiles becomes ceil(kt / share) items, so the items beyond one a tile are at most
// kQ8Slots, split tiles at most that many, and their items at most kMaxSplitItems.  (W is taken from closed forms that
// are no smaller.)  Splitting costs partial rows written and read, so no more than about an item a CU is split off
// (4 x 2,048 rows: 49 us at 256 slots, 59 at 1,024).
//
// Items are listed the longest first, to kPlanLevels of length: the workgroups of a launch start in order, so what
// starts last is short.
constexpr int kSmallWork = 80;
constexpr int kPlanLevels = 64;
__global__ __launch_bounds__(kPlanThreadsM) void q8_mixed_plan_kernel(Q8PlanParams p) {
  __shared__ int64_t sm_t0[kQ8MaxSeqs];
  __shared__ int sm_slot[kQ8MaxSeqs], sm_L[kQ8MaxSeqs], sm_c[kQ8MaxSeqs];
  __shared__ int sm_first[kQ8MaxSeqs];  // a sequence's first tile
  __shared__ int sm_level[kPlanLevels];
  __shared__ int sm_seq[3][kPlanWavesM], sm_tile[2][kPlanWavesM];
  __shared__ float sm_work[2][kPlanWavesM];  // a wave's part of W in whole tiles, in half tiles
  __shared__ int sm_fits;
  constexpr int kSeqsPer = kQ8MaxSeqs / kPlanThreadsM;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  if (tid < kPlanLevels) sm_level[tid] = 0;
  const int per_thread = (p.B + kPlanThreadsM - 1) / kPlanThreadsM, b_first = tid * per_thread;
  float work[2] = {0.f, 0.f};
  int n_seq[3] = {0, 0, 0};  // tiles if they are whole, if they are half ones; ranges that run backwards
  int n_rt[2][kSeqsPer];
#pragma unroll
  for (int u = 0; u < kSeqsPer; ++u) {
    n_rt[0][u] = n_rt[1][u] = 0;
    const int b = b_first + u;
    if (u >= per_thread || b >= p.B) continue;
    const Q8Seq s = q8_seq(p, b, true);
    // (others may overlap such a range; the bounds below need disjoint ones)
    n_seq[2] |= p.cu_seqlens[b + 1] < p.cu_seqlens[b];
    sm_t0[b] = s.t0;
    sm_slot[b] = s.slot;
    sm_L[b] = s.L;
    sm_c[b] = s.c;
    if (s.L == 0) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Q8Cut cut(p, s.L, kTileCols >> i, 0);
      const float n = (float)cut.n_rt;
      work[i] += cut.narrow ? (float)((s.c + s.L) >> 6) + 1.f
                            : n * (float)((s.c >> 4) + 2) + (float)cut.R * n * (n + 1.f) * (1.f / 32) + 1.f;
      n_rt[i][u] = cut.n_rt;
      n_seq[i] += cut.n_rt;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float w = wave_sum(work[i]);
    if (lane == 0) sm_work[i][tid / kWave] = w;
  }
  int seq_before[3], seq_all[3];
  plan_block_scan(n_seq, seq_before, seq_all, sm_seq);
  if (seq_all[2]) {
    if (tid == 0) p.plan[0] = 0;
    if (tid > 0 && tid < kHeadWords) p.plan[tid] = plan_word(p, tid - 1, p.D);
    return;
  }
  float total[2] = {0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kPlanWavesM; ++w) {
    total[0] += sm_work[0][w];
    total[1] += sm_work[1][w];
  }
  // (fp32 sums of positive terms, each rounded by 2^-24 of itself a few times: 1e-3 more covers their errors)
  const float per_slot = 1.001f * (float)p.H_kv / kQ8Slots;
  const bool small = total[0] * per_slot <= (float)kSmallWork;
  const int cols = small ? kTileCols / 2 : kTileCols;
  const int want = (int)fminf(67108864.f, (small ? total[1] : total[0]) * per_slot + 1.f);
  const int n_tiles = small ? seq_all[1] : seq_all[0];
  int at_tile = small ? seq_before[1] : seq_before[0];
#pragma unroll
  for (int u = 0; u < kSeqsPer; ++u) {
    if (u < per_thread && b_first + u < p.B) sm_first[b_first + u] = at_tile;
    at_tile += small ? n_rt[1][u] : n_rt[0][u];
  }
  __syncthreads();

  // A thread's tile: sequence, rows, chunks, partial rows and arrival words before it.
  int b = 0, r = 0, n = 0, rows = 0, kt = 0, pbase = 0, ctr = 0, level = 0;
  int rows_at = 0, ctr_at = 0;
  auto tile = [&](int i0) {
    const int i = i0 + tid;
    n = rows = 0;
    int R = 1, share = 1;
    bool narrow = false;
    if (i < n_tiles) {
      int lo = 0, hi = p.B - 1;  // the last sequence whose first tile is at or before i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sm_first[mid] <= i)
          lo = mid;
        else
          hi = mid - 1;
      }
      b = lo;
      const Q8Cut cut(p, sm_L[b], cols, want);
      r = i - sm_first[b];
      R = cut.R;
      share = cut.share;
      narrow = cut.narrow;
      rows = min(R, sm_L[b] - r * R);
      kt = (sm_c[b] + r * R + rows + 15) >> 4;
      n = min(kQ8MaxChunks, (kt + share - 1) / share);
    }
    const int mine[2] = {n > 1 ? n * rows * p.G * p.H_kv : 0, n > 1 ? p.H_kv : 0};
    int before[2], all[2];
    plan_block_scan(mine, before, all, sm_tile);
    pbase = rows_at + before[0];
    ctr = ctr_at + before[1];
    rows_at += all[0];
    ctr_at += all[1];
    if ((int64_t)pbase + mine[0] > p.part_cap) n = 1;  // (a guard: partial rows past the buffer; q8_part_rows holds all)
    if (n > 0) {
      const int len = (kt + n - 1) / n;  // an item's key tiles, in a wide item's
      level = kPlanLevels - 1 - min(kPlanLevels - 1, (int)((int64_t)len * kPlanLevels / (share + 1)));
      if (narrow) rows = -rows;
    }
  };
  const bool once = n_tiles <= kPlanThreadsM;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreadsM) {
    if (i0 > 0) __syncthreads();
    tile(i0);
    if (n > 0) atomicAdd(&sm_level[level], n * p.H_kv);
  }
  __syncthreads();
  if (tid < kWave) {  // levels' first items
    const int v = sm_level[tid], inc = wave_inclusive_sum(v);
    sm_level[tid] = inc - v;
    const int n_items = __builtin_amdgcn_readlane(inc, kWave - 1);
    if (tid == 0) {
      const bool fits = n_items <= p.plan_cap;  // (a guard: q8_plan_items holds all)
      if (!fits) set_err(p.err, CIE_ERRBIT_PLAN);
      sm_fits = fits;
      p.plan[0] = fits ? n_items : 0;
#pragma unroll
      for (int i = 1; i < kHeadWords; ++i) p.plan[i] = plan_word(p, i - 1, p.D);
    }
  }
  __syncthreads();
  if (!sm_fits) return;
  Q8Item* const items = reinterpret_cast<Q8Item*>(p.plan + kHeadWords);
  rows_at = ctr_at = 0;
  for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreadsM) {
    if (!once) {
      if (i0 > 0) __syncthreads();
      tile(i0);
    }
    if (n == 0) continue;
    const int abs_rows = rows < 0 ? -rows : rows;
    const int R = rows < 0 ? 0 : cols / p.G;  // (a narrow sequence has one tile)
    int at = atomicAdd(&sm_level[level], n * p.H_kv);
    Q8Item it;
    it.tok0 = (int)sm_t0[b] + r * R;
    it.rows = rows;
    it.slot = sm_slot[b];
    it.pos0 = sm_c[b] + r * R;
    it.n_chunks = n;
    it.pad = 0;
    const int per = 4 * ((((kt + 3) >> 2) + n - 1) / n);  // near-equal chunks in whole stages (4 tiles)
    for (int g = 0; g < p.H_kv; ++g) {
      it.g = g;
      it.pbase = n > 1 ? pbase + g * n * abs_rows * p.G : 0;
      it.ctr = n > 1 ? ctr + g : 0;
      for (int c = 0; c < n; ++c) {
        it.chunk = c;
        it.t0 = min(kt, c * per);
        it.t1 = min(kt, it.t0 + per);
        items[at++] = it;
      }
    }
  }
}

// ---- the attention ----

template <int D>
struct Q8Lds {
  static constexpr int kK = 4 * Geo<D>::KS * kWave;  // operand slots of a stage
  static constexpr int kV = 2 * Geo<D>::NT * kWave;
  static constexpr int kStage = kK + kV;
  static constexpr int kFold = kMW * 16 * (D / 4 + 1) + 2 * kMW * 16 / 4;
  static constexpr int kMerge = (kTileCols * kQ8MaxChunks + 2 * kMThreads) / 4 + kMThreads;
  static constexpr int kNans = 4 * kQ8NanMap / 16;  // NaN maps of a stage
  static constexpr int kSlots = 2 * kStage + 2 * kNans;
  static_assert(kSlots >= kMerge, "the merge's scratch");
  static_assert(kSlots >= kFold + kMW * kNans, "the fold, and NaN maps for the waves' steps of narrow items");
  static_assert(kMThreads >= kTileCols && kTileCols * (D / 4) <= 16 * kMThreads, "the merge's threads");
};

// Column cc of an item: its row and head, and where its output goes.
struct Q8Col {
  int row, head;
  __device__ __forceinline__ Q8Col(const Q8MixedParams& p, int cc)
      : row(magic_div(cc, p.g_magic)), head(cc - magic_div(cc, p.g_magic) * p.G) {}
};
template <int D>
__device__ __forceinline__ int64_t out_row(const Q8MixedParams& p, const Q8Item& it, const Q8Col& c) {
  return ((int64_t)(it.tok0 + c.row) * p.H_q + it.g * p.G + c.head) * D;
}

// The wave's tiles: t0 + wave + 4 k, byte offsets and scales of 64 of them in its lanes.
template <int D>
struct WaveTiles {
  const Q8MixedParams& p;
  const Q8Src src;
  const int64_t* bt_row;
  int t0, n, tpp, lane;
  int64_t off;
  f32x2 sc;
  __device__ __forceinline__ WaveTiles(const Q8MixedParams& p_, const Q8Item& it, int wave, int lane_)
      : p(p_),
        src{p_.k_pool, p_.v_pool, p_.scales, p_.pool_page_stride, (int64_t)it.g * p_.pool_head_stride, p_.H_kv, it.g,
            p_.page_size >> 4},
        bt_row(p_.block_table + (int64_t)it.slot * p_.bt_stride),
        t0(uniform(it.t0 + wave)),
        n(uniform(max(0, (it.t1 - it.t0 - wave + 3) >> 2))),
        tpp(p_.page_size >> 4),
        lane(lane_),
        off(0),
        sc{1.f, 1.f} {}
  __device__ __forceinline__ void gather(int c0) {
    if (c0 + lane < n) {
      const int t = t0 + 4 * (c0 + lane);
      int64_t page = bt_row[t / tpp];
      if (page < 0 || page >= p.n_pages) {
        set_err(p.err, CIE_ERRBIT_PAGE);
        page = 0;
      }
      off = src.tile((int)page, t % tpp, D);
      sc = *reinterpret_cast<const f32x2*>(src.scale((int)page, t % tpp));
    }
  }
  // tile k (of the gathered 64), rows below key_end; a k past the last: no rows
  template <int POL>
  __device__ __forceinline__ void load(Q8Tile<D>& t, int c0, int k, int key_end, const Q8Lane<D>& lo) const {
    const bool real = c0 + k < n;
    const int rows = real ? min(16, key_end - 16 * (t0 + 4 * (c0 + k))) : 0;
    const int64_t o = readlane64(off, real ? k : 0);
    q8_load<D, POL>(t, q8_rsrc(p.k_pool, o, rows, D), q8_rsrc(p.v_pool, o, rows, D), lo);
  }
  __device__ __forceinline__ float scale(int i, int k) const {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc[i]), k));
  }
};

// A partial row's order: the 16-byte piece of dims 4 d4 .. 4 d4 + 3 sits at piece (d4 % NT) * 4 + d4 / NT, so that the
// four lanes of a column (each NT pieces of consecutive dims) write 64 bytes in one piece at a time.
template <int D>
__device__ __forceinline__ int part_piece(int d4) {
  return (d4 % Geo<D>::NT) * 4 + d4 / Geo<D>::NT;
}

// Merge a split tile's chunk states into o.  One workgroup does it, so memory round trips bound it.  A thread owns UN
// pieces (4 dims of a column; pieces tid + 256 i), kMergeLoads loads in flight; where the pieces are fewer than the
// threads, R threads share one, each taking every R-th chunk, and are summed through LDS.  The first loads go out
// ahead of the chunks' weights 2^(m - M) / l, which `weights` leaves in sm_w.
constexpr int kMergeLoads = 16;
template <int D, int UN, class Weights>
__device__ __forceinline__ void merge_pieces(const Q8MixedParams& p, const Q8Item& it, int cols, const float* sm_w,
                                             f32x4* sm_sum, Weights weights) {
  constexpr int D4 = D / 4, CG = kMergeLoads / UN;
  const int n = it.n_chunks, n_units = cols * D4;
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + (int64_t)it.pbase * D, (uint32_t)(n_units * n * sizeof(f32x4)));
  const int R = UN == 1 ? max(1, kMThreads / n_units) : 1;
  const int r = R > 1 ? (int)threadIdx.x / n_units : 0;
  const int u0 = threadIdx.x - r * n_units;
  f32x4 num[UN];
#pragma unroll
  for (int i = 0; i < UN; ++i) num[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 x[CG][UN];
  auto load = [&](int c0) {
#pragma unroll
    for (int k = 0; k < CG; ++k)
#pragma unroll
      for (int i = 0; i < UN; ++i) {  // (past the last piece or chunk: beyond the descriptor, zeros)
        const int u = u0 + i * kMThreads, c = c0 + k * R;
        x[k][i] = agent_load4(racc, r < R && u < n_units && c < n ? (uint32_t)((c * n_units + u) * sizeof(f32x4))
                                                                  : 0x7ffffff0u);
      }
  };
  load(r);
  weights();
  for (int c0 = r; c0 < n;) {
#pragma unroll
    for (int k = 0; k < CG; ++k)
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        const int u = u0 + i * kMThreads, c = c0 + k * R;
        if (u < n_units && c < n) num[i] += sm_w[c * cols + u / D4] * x[k][i];
      }
    c0 += R * CG;
    if (c0 < n) load(c0);
  }
  if (R > 1) {
    sm_sum[threadIdx.x] = num[0];
    __syncthreads();
    if (r == 0)
      for (int i = 1; i < R; ++i) num[0] += sm_sum[u0 + i * n_units];
  }
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    const int u = u0 + i * kMThreads;
    if (r == 0 && u < n_units) {
      const int cc = u / D4, piece = u % D4;
      const int d4 = (piece % 4) * Geo<D>::NT + piece / 4;
      f16x4 o4;
#pragma unroll
      for (int j = 0; j < 4; ++j) o4[j] = (f16)num[i][j];
      *reinterpret_cast<f16x4*>(p.o + out_row<D>(p, it, Q8Col(p, cc)) + 4 * d4) = o4;
    }
  }
}

// The chunks' weights of every column, in sm_w[chunk * cols + column]: tpc threads share a column's chunks.  sm_m:
// [2][thread], their maxima and sums.
__device__ __forceinline__ void merge_weights(const Q8MixedParams& p, const Q8Item& it, int cols, float* sm_w,
                                              float* sm_m) {
  constexpr int kGroup = 8;
  const int n = it.n_chunks;
  const int tpc = kMThreads / cols;
  const int j = (int)threadIdx.x / cols, cc = threadIdx.x - j * cols;
  float M = kEmptyMax, den = 0.f;
  if (j < tpc) {
    for (int c0 = j; c0 < n; c0 += kGroup * tpc) {
      float ms[kGroup], ls[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int row = it.pbase + min(c0 + i * tpc, n - 1) * cols + cc;
        ms[i] = agent_load(&p.part_m[row]);
        ls[i] = agent_load(&p.part_l[row]);
      }
      float Mn = M;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) Mn = q8_max(Mn, ms[i]);  // (the last chunk again past the end: no matter)
      den *= fast_exp2(M - Mn);
      M = Mn;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int c = c0 + i * tpc;
        if (c < n) {
          den += fast_exp2(ms[i] - M) * ls[i];
          sm_w[c * cols + cc] = ms[i];
        }
      }
    }
    sm_m[threadIdx.x] = M;
    sm_m[kMThreads + threadIdx.x] = den;
  }
  __syncthreads();
  if (j < tpc) {
    float top = kEmptyMax, sum = 0.f;
    for (int i = 0; i < tpc; ++i) top = q8_max(top, sm_m[i * cols + cc]);
    for (int i = 0; i < tpc; ++i) sum += fast_exp2(sm_m[i * cols + cc] - top) * sm_m[kMThreads + i * cols + cc];
    const float inv = q8_no_key(sum) ? 0.f : 1.f / sum;
    for (int c = j; c < n; c += tpc) {
      float* const w = &sm_w[c * cols + cc];
      *w = fast_exp2(*w - top) * inv;
    }
  }
  __syncthreads();
}

// The same for few chunks: a thread owns UN pieces (tid + 256 i) and takes CH chunks a round, each with its m and l: a
// round trip, no barrier (14 / 2 heads, D = 64, planned: 8 rows over 4,000 keys 12.2 us through merge_pieces, 9.2 so; 2 x
// 64 rows over 2,000 15.3 and 14.1).  Past 4 pieces a thread it is the slower: 8 of them take 24 more registers (4 x
// 8,192 rows 562 -> 620 us).
template <int D, int UN, int CH>
__device__ __forceinline__ void merge_few(const Q8MixedParams& p, const Q8Item& it, int cols) {
  constexpr int D4 = D / 4;
  const int n = it.n_chunks, n_units = cols * D4;
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + (int64_t)it.pbase * D, (uint32_t)(n_units * n * sizeof(f32x4)));
  float M[UN], den[UN];
  f32x4 num[UN];
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    M[i] = kEmptyMax;
    den[i] = 0.f;
    num[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int c0 = 0; c0 < n; c0 += CH) {
    float ms[CH][UN], ls[CH][UN];
    f32x4 as[CH][UN];
#pragma unroll
    for (int u = 0; u < CH; ++u) {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        ms[u][i] = kEmptyMax;
        ls[u][i] = 0.f;
        as[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int unit = threadIdx.x + i * kMThreads;
        if (c0 + u < n && unit < n_units) {
          const int row = (c0 + u) * cols + unit / D4;
          ms[u][i] = agent_load(&p.part_m[it.pbase + row]);
          ls[u][i] = agent_load(&p.part_l[it.pbase + row]);
          as[u][i] = agent_load4(racc, (uint32_t)((row * D + 4 * part_piece<D>(unit % D4)) * sizeof(float)));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      float Mn = M[i];
#pragma unroll
      for (int u = 0; u < CH; ++u) Mn = q8_max(Mn, ms[u][i]);
      const float a0 = fast_exp2(M[i] - Mn);
      num[i] *= a0;
      den[i] *= a0;
      M[i] = Mn;
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const float a = fast_exp2(ms[u][i] - Mn);
        num[i] += a * as[u][i];
        den[i] += a * ls[u][i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    const int unit = threadIdx.x + i * kMThreads;
    if (unit >= n_units) continue;
    const int cc = unit / D4, d4 = unit - cc * D4;
    f16x4 o4;
#pragma unroll
    for (int j = 0; j < 4; ++j) o4[j] = (f16)(q8_no_key(den[i]) ? 0.f : num[i][j] / den[i]);
    *reinterpret_cast<f16x4*>(p.o + out_row<D>(p, it, Q8Col(p, cc)) + 4 * d4) = o4;
  }
}

template <int D>
__device__ __forceinline__ void q8_mixed_merge(const Q8MixedParams& p, const Q8Item& it, int cols, f32x4* lds) {
  float* const sm_w = reinterpret_cast<float*>(lds);
  float* const sm_m = sm_w + kTileCols * kQ8MaxChunks;
  f32x4* const sm_sum = lds + (kTileCols * kQ8MaxChunks + 2 * kMThreads) / 4;
  auto weights = [&] { merge_weights(p, it, cols, sm_w, sm_m); };
  const int n_units = cols * (D / 4);
  if (it.n_chunks <= 16 && n_units <= kMThreads)
    merge_few<D, 1, 8>(p, it, cols);
  else if (it.n_chunks <= 8 && n_units <= 4 * kMThreads)
    merge_few<D, 4, 4>(p, it, cols);
  else if (n_units <= kMThreads)
    merge_pieces<D, 1>(p, it, cols, sm_w, sm_sum, weights);
  else if (n_units <= 2 * kMThreads)
    merge_pieces<D, 2>(p, it, cols, sm_w, sm_sum, weights);
  else if (D == 64 || n_units <= 8 * kMThreads)
    merge_pieces<D, 8>(p, it, cols, sm_w, sm_sum, weights);
  else if constexpr (D == 128)
    merge_pieces<D, 16>(p, it, cols, sm_w, sm_sum, weights);
}

template <int D>
__device__ __forceinline__ void load_col_q(f16x8 (&q)[Geo<D>::KS], int& lim, const Q8MixedParams& p, const Q8Item& it,
                                           int cols, int cc, int grp) {
  const bool live = cc < cols;
  const Q8Col c(p, live ? cc : 0);
  const f16* const row = p.q + out_row<D>(p, it, c);
#pragma unroll
  for (int ks = 0; ks < Geo<D>::KS; ++ks) {
    q[ks] = *reinterpret_cast<const f16x8*>(row + q8_dim(ks, grp));
    if (!live) q[ks] = f16x8{};
  }
  lim = live ? it.pos0 + c.row + 1 : kNoKey;  // (an absent column attends everything, for no one)
}

// Wide item, NA column tiles in this wave (0: it only loads).
template <int D, int NA>
__device__ __forceinline__ void wide_item(const Q8MixedParams& p, const Q8Item& it, int cols, f32x4* lds,
                                          uint32_t (*sm_nan)[kMW], int wave, int lane) {
  constexpr int KS = Geo<D>::KS, NT = Geo<D>::NT;
  constexpr int NC = NA > 0 ? NA : 1;
  const int r16 = lane & 15, grp = lane >> 4;
  const Q8Lane<D> lo(r16, grp);
  const int key_end = it.pos0 + it.rows;
  WaveTiles<D> tiles(p, it, wave, lane);
  f16x8 q[NC][KS];
  int lim[NC];
  tiles.gather(0);
  if constexpr (NA > 0) {
#pragma unroll
    for (int c = 0; c < NA; ++c) load_col_q<D>(q[c], lim[c], p, it, cols, 16 * (wave + kMW * c) + r16, grp);
  }
  int mask_from = kNoKey;
  if constexpr (NA > 0) {
#pragma unroll
    for (int c = 0; c < NA; ++c) mask_from = min(mask_from, lim[c]);
    for (int off = 1; off < kWave; off <<= 1) mask_from = min(mask_from, __shfl_xor(mask_from, off, kWave));
    mask_from = uniform(mask_from);
  }
  SoftmaxAcc<D, NC> st;
  st.init();
  const int n_stages = uniform((it.t1 - it.t0 + 3) >> 2);
  Q8Tile<D> raw;
  f16x8* const buf = reinterpret_cast<f16x8*>(lds);
  // Stages of which some row masks a key; their tiles' NaN maps.
  auto masked = [&](int sg) { return 16 * (it.t0 + 4 * (sg + 1)) > it.pos0 + 1; };
  auto nan_map = [&](int sg, int i) {
    return reinterpret_cast<uint8_t*>(lds + 2 * Q8Lds<D>::kStage + (sg & 1) * Q8Lds<D>::kNans) + i * kQ8NanMap;
  };
  // this wave's tile of stage sg (its bytes in raw), converted into operand slots; then stage sg + 1's loads
  auto stage = [&](int sg, bool look) {
    f16x8* const kbuf = buf + (sg & 1) * Q8Lds<D>::kStage;
    f16x8* const vbuf = kbuf + Q8Lds<D>::kK;
    const int k = sg & (kWave - 1);
    if (look && masked(sg)) {
      const bool nan = q8_has_nan<D>(raw);
      if (nan) q8_nan_map<D>(raw, nan_map(sg, wave), r16, grp);
      if (lane == 0) sm_nan[sg & 1][wave] = nan;
    }
    const float ks = tiles.scale(0, k), vs = tiles.scale(1, k);
    f16x8 ko[KS];
    q8_k_operand<D>(ko, raw, ks);
#pragma unroll
    for (int i = 0; i < KS; ++i) kbuf[(wave * KS + i) * kWave + lane] = ko[i];
    f16x8 va[NT];
    q8_v_operand<D>(va, 0, raw, vs);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      reinterpret_cast<f16x4*>(vbuf + ((wave >> 1) * NT + nt) * kWave + lane)[wave & 1] =
          f16x4{va[nt][0], va[nt][1], va[nt][2], va[nt][3]};
    const int next = (sg + 1) & (kWave - 1);
    if (next == 0) tiles.gather(sg + 1);
    tiles.template load<0>(raw, sg + 1 - next, next, key_end, lo);  // (past the last: no rows)
  };
  // stage sg; kLook: it, or the next one, holds masked keys (else no code for them: 4 x 2,048 rows, 14 / 2 heads, D =
  // 64, 48.0 us, 48.3 with it in every stage; 47.1 without a look at NaNs)
  auto step = [&](int sg, auto look) {
    constexpr bool kLook = decltype(look)::value;
    // stage sg is written, and stage sg - 1's buffer free: the next one is converted while sg's S MFMAs run
    __syncthreads();
    const f16x8* const kbuf = buf + (sg & 1) * Q8Lds<D>::kStage;
    const f16x8* const vbuf = kbuf + Q8Lds<D>::kK;
    if constexpr (NA > 0) {
      int key0[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) key0[i] = 16 * (it.t0 + 4 * sg + i);
      auto k = [&](int i, f16x8 (&ka)[KS]) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) ka[ks] = kbuf[(i * KS + ks) * kWave + lane];
      };
      auto v = [&](int pr, f16x8 (&va)[NT]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) va[nt] = vbuf[(pr * NT + nt) * kWave + lane];
      };
      q8_step<D, NC, 2, true>(st, k, v, [&] { stage(sg + 1, kLook); }, q, key0, lim,
                              kLook && key0[3] + 16 > mask_from, p.scale_log2, grp);
      if (kLook && masked(sg)) {
        uint32_t hit[NC] = {};
        for (int i = 0; i < 4; ++i)
          if (uniform((int)sm_nan[sg & 1][i])) q8_nan_hits<NC>(hit, nan_map(sg, i), key0[0] + 16 * i, lim, grp);
        bool any = false;
#pragma unroll
        for (int c = 0; c < NC; ++c) any |= hit[c] != 0;
        if (__any(any)) q8_nan_fix<D, NC>(st, hit);
      }
    } else {
      stage(sg + 1, kLook);
    }
  };
  tiles.template load<0>(raw, 0, 0, key_end, lo);
  stage(0, true);
  int sg = 0;
  for (; sg < n_stages && !masked(sg + 1); ++sg) step(sg, std::false_type{});
  for (; sg < n_stages; ++sg) step(sg, std::true_type{});
  __syncthreads();  // (the merge takes the buffers)
  if constexpr (NA > 0) {
    const __amdgpu_buffer_rsrc_t racc =
        coherent_rsrc(p.part_acc + (int64_t)it.pbase * D,
                      it.n_chunks > 1 ? (uint32_t)(cols * it.n_chunks * D * sizeof(float)) : 0);
#pragma unroll
    for (int c = 0; c < NA; ++c) {
      const int cc = 16 * (wave + kMW * c) + r16;
      if (cc >= cols) continue;
      const float l = st.lsum[c][0];
      if (it.n_chunks == 1) {
        const float inv = q8_no_key(l) ? 0.f : 1.f / l;
        f16* const o = p.o + out_row<D>(p, it, Q8Col(p, cc)) + NT * 4 * grp;
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {  // the lane's 4 NT dims, 8 at a time
          f16x8 x;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = (f16)(st.acc[c][(8 * i + j) % NT][(8 * i + j) / NT] * inv);
          *reinterpret_cast<f16x8*>(o + 8 * i) = x;
        }
      } else {
        const int row = it.chunk * cols + cc;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          agent_store4(racc, (uint32_t)((row * D + 4 * part_piece<D>(NT * grp + i)) * sizeof(float)),
                       f32x4{st.acc[c][(4 * i) % NT][(4 * i) / NT], st.acc[c][(4 * i + 1) % NT][(4 * i + 1) / NT],
                             st.acc[c][(4 * i + 2) % NT][(4 * i + 2) / NT],
                             st.acc[c][(4 * i + 3) % NT][(4 * i + 3) / NT]});
        if (grp == 0) {
          agent_store(&p.part_m[it.pbase + row], st.m[c]);
          agent_store(&p.part_l[it.pbase + row], l);
        }
      }
    }
  }
}

// Narrow item: one column tile, the keys dealt over the waves.
template <int D>
__device__ __forceinline__ void narrow_item(const Q8MixedParams& p, const Q8Item& it, int cols, f32x4* lds, int wave,
                                            int lane) {
  constexpr int KS = Geo<D>::KS, NT = Geo<D>::NT, D4 = D / 4;
  constexpr int PF = 1, NS = D == 64 ? 4 : 2;  // (as the decode kernel's)
  const int r16 = lane & 15, grp = lane >> 4;
  const Q8Lane<D> lo(r16, grp);
  const int key_end = it.pos0 - it.rows;  // (rows: negative here)
  WaveTiles<D> tiles(p, it, wave, lane);
  tiles.gather(0);
  f16x8 q[1][KS];
  int lim[1];
  load_col_q<D>(q[0], lim[0], p, it, cols, r16, grp);
  uint8_t* const map = reinterpret_cast<uint8_t*>(lds + Q8Lds<D>::kFold) + wave * NS * kQ8NanMap;
  const int mask_from = it.pos0 + 1;  // the first row's keys
  SoftmaxAcc<D, 1> st;
  st.init();
  for (int c0 = 0; c0 < tiles.n; c0 += kWave) {
    if (c0 > 0) tiles.gather(c0);
    const int n_chunk = min(kWave, tiles.n - c0);
    const int n_steps = (n_chunk + NS - 1) / NS;
    Q8Tile<D> ring[PF + 1][NS];
    auto issue = [&](int i, int j) {  // (tiles past the last: no rows)
#pragma unroll
      for (int u = 0; u < NS; ++u)
        tiles.template load<kBufNt>(ring[i][u], c0, NS * j + u < n_chunk ? NS * j + u : tiles.n, key_end, lo);
    };
#pragma unroll
    for (int j = 0; j < PF; ++j) issue(j, j);
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
            key0[i] = k < n_chunk ? 16 * (tiles.t0 + 4 * (c0 + kk)) : kNoKey;
            sc[i] = f32x2{tiles.scale(0, kk), tiles.scale(1, kk)};
          }
          q8_attend_rows<D, NS>(st, ring[u], sc, q, key0, lim, key0[NS - 1] + 16 > mask_from, p.scale_log2, map, r16,
                               grp);
        }
      }
    }
  }
  // fold the waves
  f32x4(*const sm_acc)[16][D4 + 1] = reinterpret_cast<f32x4(*)[16][D4 + 1]>(lds);
  float(*const sm_m)[16] = reinterpret_cast<float(*)[16]>(lds + kMW * 16 * (D4 + 1));
  float(*const sm_l)[16] = sm_m + kMW;
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
  const __amdgpu_buffer_rsrc_t racc =
      coherent_rsrc(p.part_acc + (int64_t)it.pbase * D,
                    it.n_chunks > 1 ? (uint32_t)(cols * it.n_chunks * D * sizeof(float)) : 0);
  for (int u = threadIdx.x; u < cols * D4; u += kMThreads) {
    const int cc = u / D4, d4 = u - cc * D4;
    float M = kEmptyMax, den = 0.f;
#pragma unroll
    for (int w = 0; w < kMW; ++w) M = q8_max(M, sm_m[w][cc]);
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kMW; ++w) {
      const float a = fast_exp2(sm_m[w][cc] - M);
      num += a * sm_acc[w][cc][d4];
      den += a * sm_l[w][cc];
    }
    if (it.n_chunks == 1) {
      f16x4 o4;
#pragma unroll
      for (int i = 0; i < 4; ++i) o4[i] = (f16)(q8_no_key(den) ? 0.f : num[i] / den);
      *reinterpret_cast<f16x4*>(p.o + out_row<D>(p, it, Q8Col(p, cc)) + 4 * d4) = o4;
    } else {
      const int row = it.chunk * cols + cc;
      agent_store4(racc, (uint32_t)((row * D + 4 * part_piece<D>(d4)) * sizeof(float)), num);
      if (d4 == 0) {
        agent_store(&p.part_m[it.pbase + row], M);
        agent_store(&p.part_l[it.pbase + row], den);
      }
    }
  }
}

template <int D>
__global__ __launch_bounds__(kMThreads) __attribute__((amdgpu_waves_per_eu(2)))
void q8_mixed_kernel(Q8MixedParams p) {
  __shared__ f32x4 lds[Q8Lds<D>::kSlots];
  __shared__ uint32_t sm_nan[2][kMW];  // whether a stage's V tile holds a NaN (stages of masked keys)
  __shared__ int sm_last;
  const int32_t* const head = p.plan;
  const Q8Item it = reinterpret_cast<const Q8Item*>(head + kHeadWords)[blockIdx.x];  // (read with the head)
  bool same = true;
#pragma unroll
  for (int i = 1; i < kHeadWords; ++i) same &= head[i] == plan_word(p, i - 1, D);
  if (!same) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_err(p.err, CIE_ERRBIT_PLAN);
    return;
  }
  if ((int)blockIdx.x >= head[0]) return;
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
  const bool narrow = it.rows < 0;
  const int cols = (narrow ? -it.rows : it.rows) * p.G;
  if (narrow) {
    narrow_item<D>(p, it, cols, lds, wave, lane);
  } else {
    const int n_ct = (cols + 15) >> 4;
    const int na = n_ct > wave ? (n_ct - wave + kMW - 1) / kMW : 0;  // column tiles wave, wave + 4, ..
    if (na == 2)
      wide_item<D, 2>(p, it, cols, lds, sm_nan, wave, lane);
    else if (na == 1)
      wide_item<D, 1>(p, it, cols, lds, sm_nan, wave, lane);
    else
      wide_item<D, 0>(p, it, cols, lds, sm_nan, wave, lane);
  }
  if (it.n_chunks == 1) return;
  int32_t* const arrival = p.counters + it.ctr;
  if (!arrive_last(arrival, p.n_ctr, it.n_chunks, &sm_last, p.err)) return;
  q8_mixed_merge<D>(p, it, cols, lds);
  if (threadIdx.x == 0) counter_reset(arrival);
}

// Items a plan can hold: one a query tile and kv head, and kQ8Slots more from splitting.  A launch of half tiles has W <=
// kSmallWork * kQ8Slots, and a sequence no more half tiles than its part of W: with n whole ones of R rows that part is
// 2 n + R n (n + 1) / 32 + 1 at least, 2.5 n + 1 as R >= 8, and its half ones are 2.25 n + 1 at most (13 and 14 heads a
// group: 9 rows a whole tile, 4 a half one).
static int64_t q8_plan_items(int64_t B, int64_t total_T, int64_t H_q, int64_t H_kv) {
  const int64_t R = kTileCols / (H_q / H_kv), half = kTileCols / 2 / (H_q / H_kv);
  const int64_t whole = H_kv * (total_T / R + B), small = H_kv * (total_T / half + B);
  const int64_t most = kSmallWork * kQ8Slots + H_kv * B;
  return kQ8Slots + (whole > most ? whole : small < most ? small : most);
}

// Partial rows a launch can need: its split items' columns, and no more than kQ8MaxChunks a query row and head.
static int64_t q8_part_rows(int64_t total_T, int64_t H_q) {
  const int64_t most = (int64_t)kMaxSplitItems * kTileCols;
  return total_T > most / (kQ8MaxChunks * H_q) ? most : kQ8MaxChunks * total_T * H_q;
}

static int q8_mixed_check(int64_t B, int64_t total_T, int64_t max_seqlen, int64_t H_q, int64_t H_kv, int64_t D,
                          int64_t page_size, int64_t bt_width, int64_t n_slots) {
  if (B < 0 || total_T < 0 || max_seqlen < 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || page_size <= 0 ||
      bt_width <= 0 || n_slots <= 0)
    return CIE_EINVAL;
  if (H_q / H_kv > 16 || (D != 64 && D != 128) || page_size % 16 != 0 || B > kQ8MaxSeqs || H_kv > 4096 ||
      total_T > (1 << 24) || bt_width > 0x3fffffff / page_size ||
      q8_plan_items(B, total_T, H_q, H_kv) > 0x7fffffff / kItemWords)
    return CIE_EUNSUPPORTED;
  return CIE_OK;
}

}  // namespace cie

using namespace cie;

extern "C" int64_t cie_q8_mixed_plan_bytes(int64_t B, int64_t total_T, int64_t H_q, int64_t H_kv) {
  if (B < 0 || total_T < 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || H_q / H_kv > 16 || B > kQ8MaxSeqs ||
      H_kv > 4096 || total_T > (1 << 24))
    return -1;
  return (kHeadWords + q8_plan_items(B, total_T, H_q, H_kv) * kItemWords) * 4;
}

extern "C" int64_t cie_q8_mixed_partials_bytes(int64_t total_T, int64_t H_q, int64_t D) {
  if (total_T < 0 || H_q <= 0 || H_q > 65536 || (D != 64 && D != 128)) return -1;
  const int64_t rows = q8_part_rows(total_T, H_q);
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  return 2 * up(rows * 4) + rows * D * 4;
}

extern "C" int64_t cie_q8_mixed_counters(void) { return 2 * kQ8Slots; }

extern "C" int cie_q8_mixed_plan(int32_t* plan, int64_t plan_bytes, const int64_t* cu_seqlens, const int64_t* kv_lens,
                                 const int64_t* slot_ids, int64_t B, int64_t total_T, int64_t max_seqlen, int64_t H_q,
                                 int64_t H_kv, int64_t D, int64_t page_size, int64_t bt_width, int64_t n_slots,
                                 int32_t* err, void* stream) {
  if (int rc = q8_mixed_check(B, total_T, max_seqlen, H_q, H_kv, D, page_size, bt_width, n_slots)) return rc;
  if (!plan || (reinterpret_cast<uintptr_t>(plan) & 15) || (B > 0 && (!cu_seqlens || !kv_lens || !slot_ids)) ||
      plan_bytes < cie_q8_mixed_plan_bytes(B, total_T, H_q, H_kv))
    return CIE_EINVAL;
  Q8PlanParams p{};
  p.plan = plan;
  p.cu_seqlens = cu_seqlens;
  p.kv_lens = kv_lens;
  p.slot_ids = slot_ids;
  p.total_T = total_T;
  p.cap = bt_width * page_size;
  p.B = (int32_t)B;
  p.n_slots = (int32_t)(n_slots > 0x7fffffff ? 0x7fffffff : n_slots);
  p.H_q = (int32_t)H_q;
  p.H_kv = (int32_t)H_kv;
  p.G = (int32_t)(H_q / H_kv);
  p.D = (int32_t)D;
  p.page_size = (int32_t)page_size;
  p.bt_width = (int32_t)bt_width;
  p.max_rows = (int32_t)(max_seqlen > total_T ? total_T : max_seqlen);
  p.part_cap = (int32_t)q8_part_rows(total_T, H_q);
  p.plan_cap = (int32_t)q8_plan_items(B, total_T, H_q, H_kv);
  p.err = err;
  hipLaunchKernelGGL(q8_mixed_plan_kernel, dim3(1), dim3(kPlanThreadsM), 0, static_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}

extern "C" int cie_q8_mixed(void* o, const void* q, const void* k_pool, const void* v_pool, const void* scales,
                            const int32_t* plan, int64_t plan_bytes, const int64_t* block_table, void* partials,
                            int64_t partials_bytes, int32_t* counters, int64_t B, int64_t total_T, int64_t H_q,
                            int64_t H_kv, int64_t D, int64_t page_size, int64_t n_pages, int64_t pool_page_stride,
                            int64_t pool_head_stride, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                            int32_t* err, void* stream) {
  if (int rc = q8_mixed_check(B, total_T, total_T, H_q, H_kv, D, page_size, bt_width, n_slots)) return rc;
  if (n_pages <= 0 || n_pages > 0x7fffffff || bt_stride < bt_width || pool_page_stride % 16 != 0 ||
      pool_head_stride % 16 != 0)
    return CIE_EINVAL;
  if (B == 0 || total_T == 0) return CIE_OK;
  if (!o || !q || !k_pool || !v_pool || !scales || !plan || !block_table || !partials || !counters ||
      plan_bytes < cie_q8_mixed_plan_bytes(B, total_T, H_q, H_kv) ||
      partials_bytes < cie_q8_mixed_partials_bytes(total_T, H_q, D))
    return CIE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) |
       reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(plan) |
       reinterpret_cast<uintptr_t>(partials) | reinterpret_cast<uintptr_t>(counters)) & 15)
    return CIE_EINVAL;
  Q8MixedParams p{};
  p.o = static_cast<f16*>(o);
  p.q = static_cast<const f16*>(q);
  p.k_pool = static_cast<const uint8_t*>(k_pool);
  p.v_pool = static_cast<const uint8_t*>(v_pool);
  p.scales = static_cast<const float*>(scales);
  p.block_table = block_table;
  p.plan = plan;
  const int64_t rows = q8_part_rows(total_T, H_q);
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  char* const ws = static_cast<char*>(partials);
  p.part_m = reinterpret_cast<float*>(ws);
  p.part_l = reinterpret_cast<float*>(ws + up(rows * 4));
  p.part_acc = reinterpret_cast<float*>(ws + 2 * up(rows * 4));
  p.counters = counters;
  p.pool_page_stride = pool_page_stride;
  p.pool_head_stride = pool_head_stride;
  p.bt_stride = bt_stride;
  p.n_pages = n_pages;
  p.total_T = total_T;
  p.part_cap = (int32_t)rows;
  p.n_ctr = kQ8Slots;
  p.plan_cap = (int32_t)q8_plan_items(B, total_T, H_q, H_kv);
  p.B = (int32_t)B;
  p.bt_width = (int32_t)bt_width;
  p.n_slots = (int32_t)(n_slots > 0x7fffffff ? 0x7fffffff : n_slots);
  p.H_q = (int32_t)H_q;
  p.H_kv = (int32_t)H_kv;
  p.G = (int32_t)(H_q / H_kv);
  p.page_size = (int32_t)page_size;
  p.g_magic = div_magic((uint32_t)p.G);
  p.scale_log2 = kLog2e / __builtin_sqrtf((float)D);
  p.err = err;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (D == 64)
    hipLaunchKernelGGL(q8_mixed_kernel<64>, dim3((unsigned)p.plan_cap), dim3(kMThreads), 0, s, p);
  else
    hipLaunchKernelGGL(q8_mixed_kernel<128>, dim3((unsigned)p.plan_cap), dim3(kMThreads), 0, s, p);
  return (int)hipGetLastError();
}
