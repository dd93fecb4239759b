// Writing the 8-bit paged cache (q8_cache.h) and reading it back.
//
// Append.  The unit of work is a block: 16 rows of one kv head, K or V, with one
// scale.  A wave takes one (block, head, K or V) at a time, a lane 16 values of a
// row (8 dims and their rotate_half partners, D / 2 further on), so RoPE, the
// block's amax (one wave maximum) and the rounding stay in registers: new rows are
// read once and written once, and the block's other rows are read only where it is
// not started anew, written only where its scale grows.
//
// Which rows of a call fall into a block: token mode takes any list of (page,
// offset) pairs.  A workgroup belongs to a token and goes on only if the token's
// block is not the one before its (a run's first token).  It then looks through the
// whole list for the block: an earlier token with it makes that one's workgroup the
// owner; otherwise the last token of each row is the one written.  So a list in any
// order, or with the same index twice, gives one result, with no race on a block.
// The search reads T page ids (L2 hits) and is shared by all heads of the block: T^2 / 16
// ids in all, which shows from some 32,000 rows on.
//
// What bounds it: memory at many tokens (8,192 rows of 8 heads, D = 128: 50 MB in 14.8
// us, 3.4 TB/s; from the projection, 32 / 8 heads, 189 MB in 42 us, 4.5 TB/s), the
// start's chain (index, search, rows) at few (3 rows of 2 heads, D = 64: 3.7 us).  Decode
// rows: 32 of 2 heads, D = 64, 3.7 us, 256 3.9, of 8 heads, D = 128, 5.1 and 6.3: slot,
// length, page and rows, one after the other (the fp16 append's 2.4 to 2.7, which needs
// no block's other rows), and with 8 heads two (head, K or V) pairs a wave in turn.
#include "q8_cache.h"

namespace cie {

// Waves a workgroup: 8 where a block has more than 4 (head, K or V) pairs to write, else 4; a wave holds one pair at a
// time.  (Two in flight: 137 registers at D = 128, one 8-wave workgroup a CU instead of two, 19.4 us for 8,192 rows of 8
// heads against 15.1; 4 waves 20.2.  464 rows of 2 heads with RoPE: 5.0 us, 5.4 with 8 waves.)  The rope form's 144
// registers leave one 8-wave workgroup a CU: past kEachRow rows, whose blocks no longer have a CU each, it takes 4
// (8,192 rows, 32 / 8 heads, D = 128: 42 us, 46 with 8; 300 rows: 9.5 with 4, 7.0 with 8).
constexpr int kFewWaves = 4, kManyWaves = 8;
constexpr int64_t kEachRow = 1024;  // rows up to which each has a workgroup of its own
constexpr int kScan = 8;
struct __attribute__((aligned(8))) PagePair {
  int64_t a, b;
};

struct Q8Params {
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* scales;
  const f16* k_new;
  const f16* v_new;
  int64_t k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  // decode mode
  const int64_t* slot_ids;
  const int64_t* lens;
  const int64_t* block_table;
  int64_t bt_stride, bt_width, n_slots;
  // token mode
  const int64_t* pages;
  const int64_t* offsets;
  // rope (token mode from the fused QKV projection): k_new / v_new point into its rows
  f16* q_out;
  const f16* qkv;
  const f16* cos;
  const f16* sin;
  int64_t qkv_stride, cs_stride;
  int32_t H_q;
  int32_t n_append_wg;  // workgroups that append; those after them rotate q
  // common
  int64_t n_rows, n_pages, pool_page_stride, pool_head_stride;
  int32_t H_kv, page_size, tokens_per_wg;
  int32_t* err;
};

// Rows of one block, and where the rows written come from.
struct Q8Rows {
  int64_t page;
  int block;        // block of the page
  bool fresh;       // row 0 is written: the block starts anew
  const int* last;  // [16] token of each row, -1: not written
};

// One wave's (block, head, K or V): loaded, then rounded and stored.
template <int D, bool kRope>
struct BlockTask {
  static constexpr int NU = D / 64;    // units of 16 values a lane
  static constexpr int kPer = D / 16;  // units a row
  uint8_t* pool;
  float* scale;
  float old_scale;
  f16x8 x[NU][2];
  f16x8 cs[kRope ? NU : 1][4];  // cos and sin of the dims, of their partners
  u32x2 old[NU][2];
  bool written[NU], rope;

  __device__ __forceinline__ void load(const Q8Params& p, const Q8Rows& b, int task, int lane) {
    const int h = task >> 1;
    const bool is_v = task & 1;
    pool = (is_v ? p.v_pool : p.k_pool) + b.page * p.pool_page_stride + h * p.pool_head_stride +
           (int64_t)b.block * kQ8Block * D;
    scale = p.scales + 2 * ((b.page * p.H_kv + h) * (p.page_size / kQ8Block) + b.block) + (is_v ? 1 : 0);
    const f16* const src = is_v ? p.v_new + h * p.v_head_stride : p.k_new + h * p.k_head_stride;
    const int64_t stride = is_v ? p.v_tok_stride : p.k_tok_stride;
    rope = kRope && !is_v;
    old_scale = 0.f;
    if (!b.fresh) old_scale = *scale;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int unit = lane + u * kWave;
      const int row = unit / kPer, d0 = 8 * (unit % kPer);
      const int t = b.last[row];
      written[u] = t >= 0;
      if (written[u]) {
        const f16* const r = src + t * stride + d0;
        x[u][0] = *reinterpret_cast<const f16x8*>(r);
        x[u][1] = *reinterpret_cast<const f16x8*>(r + D / 2);
        if (rope) {
          const f16* const c = p.cos + t * p.cs_stride + d0;
          const f16* const s = p.sin + t * p.cs_stride + d0;
          cs[u][0] = *reinterpret_cast<const f16x8*>(c);
          cs[u][1] = *reinterpret_cast<const f16x8*>(c + D / 2);
          cs[u][2] = *reinterpret_cast<const f16x8*>(s);
          cs[u][3] = *reinterpret_cast<const f16x8*>(s + D / 2);
        }
      } else if (!b.fresh) {
        old[u][0] = *reinterpret_cast<const u32x2*>(pool + row * D + d0);
        old[u][1] = *reinterpret_cast<const u32x2*>(pool + row * D + d0 + D / 2);
      }
    }
  }

  __device__ __forceinline__ void store(bool fresh, int lane) {
    uint32_t mag = 0;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (written[u]) {
        if (rope) rope8(x[u][0], x[u][1], cs[u][0], cs[u][1], cs[u][2], cs[u][3]);
        mag = q8_raw_max(x[u][0], q8_raw_max(x[u][1], mag));
      }
    }
    mag = q8_wave_mag(mag);
    if (mag > kQ8Limit) {  // uniform; rare
      mag = 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        if (written[u]) {
          mag = q8_mag8(x[u][0], q8_mag8(x[u][1], mag));
          q8_limit8(x[u][0]);
          q8_limit8(x[u][1]);
        }
      }
      mag = q8_wave_mag(mag);
    }
    const int e_old = fresh ? kQ8EMin : q8_scale_exponent(old_scale);
    const int e = max(e_old, q8_exponent(mag));
    const float s = q8_pow2(e), factor = q8_pow2(e_old - e);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int unit = lane + u * kWave;
      uint8_t* const dst = pool + (unit / kPer) * D + 8 * (unit % kPer);
      if (written[u]) {
        *reinterpret_cast<u32x2*>(dst) = q8_round8(x[u][0], s);
        *reinterpret_cast<u32x2*>(dst + D / 2) = q8_round8(x[u][1], s);
      } else if (!fresh && e != e_old) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<u32x2*>(dst + i * (D / 2)) =
              u32x2{q8_rescale4(old[u][i][0], factor), q8_rescale4(old[u][i][1], factor)};
      }
    }
    if (lane == 0) *scale = s;
  }
};

// The q heads of the rope form: a lane rotates 8 dims and their partners.
template <int D>
__device__ __forceinline__ void rotate_q(const Q8Params& p, int64_t gid) {
  constexpr int kPer = D / 16;
  if (gid >= p.n_rows * p.H_q * kPer) return;
  const int d0 = 8 * (int)(gid % kPer);
  const int64_t row = gid / kPer;
  const int h = (int)(row % p.H_q);
  const int64_t t = row / p.H_q;
  const f16* const x = p.qkv + t * p.qkv_stride + (int64_t)h * D + d0;
  const f16* const c = p.cos + t * p.cs_stride + d0;
  const f16* const s = p.sin + t * p.cs_stride + d0;
  f16x8 lo = *reinterpret_cast<const f16x8*>(x), hi = *reinterpret_cast<const f16x8*>(x + D / 2);
  rope8(lo, hi, *reinterpret_cast<const f16x8*>(c), *reinterpret_cast<const f16x8*>(c + D / 2),
        *reinterpret_cast<const f16x8*>(s), *reinterpret_cast<const f16x8*>(s + D / 2));
  f16* const dst = p.q_out + row * D + d0;
  *reinterpret_cast<f16x8*>(dst) = lo;
  *reinterpret_cast<f16x8*>(dst + D / 2) = hi;
}

template <int D, int W, bool kDecode, bool kRope>
__global__ __launch_bounds__(W * kWave)
void q8_append_kernel(Q8Params p) {
  constexpr int kAppendThreads = W * kWave;
  __shared__ int last[kQ8Block];
  __shared__ int earlier;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  if constexpr (kRope) {
    if ((int)blockIdx.x >= p.n_append_wg) {
      rotate_q<D>(p, (int64_t)(blockIdx.x - p.n_append_wg) * kAppendThreads + threadIdx.x);
      return;
    }
  }
  // The workgroup's tokens, a lane each (every wave the same): which of them start a run.
  // A prompt's run starts lie 16 tokens apart.  Workgroups go round the XCDs and their CUs in turn, so dealt in order
  // the ones with work would share a few CUs: the list is dealt with stride 16 tokens instead, which makes them
  // neighbours (4 x 2,048 rows of 8 heads, D = 128: 29 us dealt in order, 19 so, both before other steps).
  const int stride = kQ8Block / p.tokens_per_wg, per = p.n_append_wg / stride;
  const int64_t t0 = (int64_t)(stride * ((int)blockIdx.x % per) + (int)blockIdx.x / per) * p.tokens_per_wg;
  int64_t page = 0, off = 0;
  bool head = false;
  if (lane < p.tokens_per_wg && t0 + lane < p.n_rows) {
    const int64_t t = t0 + lane;
    int bad = 0;
    if constexpr (kDecode) {
      const int64_t slot = p.slot_ids[t];
      if (slot < 0 || slot >= p.n_slots) {
        bad = CIE_ERRBIT_PAGE;
      } else {
        const int64_t pos = p.lens[slot];
        if (pos < 0 || pos >= p.bt_width * p.page_size) {
          bad = CIE_ERRBIT_LEN;
        } else {
          page = p.block_table[slot * p.bt_stride + pos / p.page_size];
          off = pos % p.page_size;
        }
      }
      head = true;
    } else {
      page = p.pages[t];
      off = p.offsets[t];
      const int64_t page1 = t > 0 ? p.pages[t - 1] : -1, off1 = t > 0 ? p.offsets[t - 1] : -1;
      if (off < 0 || off >= p.page_size) bad = CIE_ERRBIT_OFFSET;
      head = page1 != page || off1 < 0 || off1 >= p.page_size || (int)off1 / kQ8Block != (int)off / kQ8Block;
    }
    if (!bad && (page < 0 || page >= p.n_pages)) bad = CIE_ERRBIT_PAGE;
    if (bad) {
      head = false;
      if (wave == 0) set_err(p.err, bad);
    }
  }
  for (uint64_t heads = __ballot(head); heads; heads &= heads - 1) {  // (uniform in the workgroup)
    const int i = __builtin_ctzll(heads);
    const int64_t t = t0 + i;
    const int64_t pg = readlane64(page, i), o = readlane64(off, i);
    const int block = (int)o / kQ8Block;
    __syncthreads();  // (the last token's block is done with `last`)
    if (threadIdx.x < kQ8Block) last[threadIdx.x] = -1;
    if (threadIdx.x == 0) earlier = 0;
    __syncthreads();
    if constexpr (kDecode) {
      // a slot that comes again later in the batch writes the row
      const int64_t slot = p.slot_ids[t];
      bool again = false;
      for (int64_t k = t + 1 + threadIdx.x; k < p.n_rows; k += kAppendThreads) again |= p.slot_ids[k] == slot;
      if (again) earlier = 1;
      if (threadIdx.x == 0) last[o % kQ8Block] = (int)t;
    } else {
      // The list's tokens of this block: kScan loads of two page ids a thread in flight, what they hit as a bit each.
      const int64_t last_pair = max((int64_t)0, p.n_rows - 2);
      for (int64_t k0 = 2 * threadIdx.x; k0 < p.n_rows; k0 += 2 * kScan * kAppendThreads) {
        uint32_t hits = 1;
        if (p.n_rows >= 2) {
          PagePair q[kScan];
#pragma unroll
          for (int u = 0; u < kScan; ++u)  // (past the list: its last two again)
            q[u] = *reinterpret_cast<const PagePair*>(p.pages + min(k0 + 2 * u * kAppendThreads, last_pair));
          hits = 0;
#pragma unroll
          for (int u = 0; u < kScan; ++u) {
            const uint32_t h = (q[u].a == pg ? 1u : 0u) | (q[u].b == pg ? 2u : 0u);
            hits |= k0 + 2 * u * kAppendThreads < p.n_rows ? h << (2 * u) : 0u;
          }
        }
        for (; hits; hits &= hits - 1) {
          const int bit = __builtin_ctz(hits);
          const int64_t k = min(k0 + (bit & ~1) * kAppendThreads, last_pair) + (bit & 1);
          const int64_t ko = p.offsets[k];
          if (ko < 0 || ko >= p.page_size || (int)ko / kQ8Block != block) continue;
          if (k < t) earlier = 1;
          atomicMax(&last[ko % kQ8Block], (int)k);
        }
      }
    }
    __syncthreads();
    if (earlier) continue;
    const Q8Rows rows{pg, block, last[0] >= 0, last};
    const int n_tasks = 2 * p.H_kv;
    BlockTask<D, kRope> task;
    for (int k = wave; k < n_tasks; k += W) {
      task.load(p, rows, k, lane);
      task.store(rows.fresh, lane);
    }
  }
}

// ---- reading back ----

struct Q8ReadParams {
  f16* k_out;  // (T, H_kv, D) dense
  f16* v_out;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* scales;
  const int64_t* pages;
  const int64_t* offsets;
  int64_t T, n_pages, pool_page_stride, pool_head_stride;
  int32_t H_kv, page_size;
  int32_t* err;
};

// Row t of the outputs = the cache's row (pages[t], offsets[t]): a lane converts 8 values of K and of V, so that a wave
// writes whole lines, past the caches (the rows are read by other kernels, later).  Bound by memory: 105,537 rows of 8
// heads, D = 128, 648 MB in 120 us, 5.4 TB/s.  A bad index reads as zeros and is reported.
template <int D>
__global__ __launch_bounds__(256) void q8_read_kernel(Q8ReadParams p) {
  constexpr int kPer = D / 8;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (gid >= p.T * p.H_kv * kPer) return;
  const int d0 = 8 * (int)(gid % kPer);
  const int64_t row = gid / kPer;
  const int h = (int)(row % p.H_kv);
  const int64_t t = row / p.H_kv;
  const int64_t page = p.pages[t], off = p.offsets[t];
  f16x8 k = {}, v = {};
  const bool off_ok = off >= 0 && off < p.page_size, page_ok = page >= 0 && page < p.n_pages;
  if (off_ok && page_ok) {
    const int64_t at = page * p.pool_page_stride + h * p.pool_head_stride + off * D + d0;
    const u32x2 kb = stream_load(reinterpret_cast<const u32x2*>(p.k_pool + at));
    const u32x2 vb = stream_load(reinterpret_cast<const u32x2*>(p.v_pool + at));
    const f32x2 s = *reinterpret_cast<const f32x2*>(
        p.scales + 2 * ((page * p.H_kv + h) * (p.page_size / kQ8Block) + off / kQ8Block));
    k = q8_values8(kb[0], kb[1], s[0]);
    v = q8_values8(vb[0], vb[1], s[1]);
  } else {
    set_err(p.err, off_ok ? CIE_ERRBIT_PAGE : CIE_ERRBIT_OFFSET);
  }
  __builtin_nontemporal_store(k, reinterpret_cast<f16x8*>(p.k_out + row * D + d0));
  __builtin_nontemporal_store(v, reinterpret_cast<f16x8*>(p.v_out + row * D + d0));
}

static bool q8_aligned(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

// What every entry point asks of the pools (D: 64 or 128, the attention kernels').
static int q8_check_pools(const void* k_pool, const void* v_pool, const void* scales, int64_t H_kv,
                          int64_t page_size, int64_t D, int64_t n_pages, int64_t page_stride, int64_t head_stride) {
  if (H_kv <= 0 || page_size <= 0 || D <= 0 || n_pages <= 0) return CIE_EINVAL;
  if ((D != 64 && D != 128) || page_size % kQ8Block != 0 || H_kv > 65535 || page_size > (1 << 20))
    return CIE_EUNSUPPORTED;
  if (!k_pool || !v_pool || !scales || !q8_aligned(k_pool) || !q8_aligned(v_pool) || !q8_aligned(scales) ||
      page_stride % 16 != 0 || head_stride % 16 != 0)
    return CIE_EINVAL;
  return CIE_OK;
}

template <int D, int W, bool kDecode, bool kRope>
static int q8_launch(const Q8Params& p, hipStream_t stream) {
  constexpr int n = W * kWave;
  int64_t blocks = p.n_append_wg;
  if (kRope) blocks += (p.n_rows * p.H_q * (D / 16) + n - 1) / n;
  if (blocks > 0x7fffffff) return CIE_EUNSUPPORTED;
  hipLaunchKernelGGL((q8_append_kernel<D, W, kDecode, kRope>), dim3((unsigned)blocks), dim3(n), 0, stream, p);
  return (int)hipGetLastError();
}

// Tokens a workgroup looks at (a power of two, 16 at most): one up to kEachRow rows, about the workgroups that the chip
// holds at once, so that the rows of a decode batch, each a block of its own, run side by side; more where it would
// take more rounds of workgroups, most of whose tokens belong to a run that another owns (8,192 rows of 2 heads with
// RoPE, D = 64: 9.8 us, 10.5 from 2,048; 1,500 rows, a block each: 7.6, and 10.8 from 512).
template <bool kDecode, bool kRope>
static int q8_launch_append(Q8Params& p, int64_t D, hipStream_t stream) {
  if (p.n_rows > 0x7fffffff / 512) return CIE_EUNSUPPORTED;
  p.tokens_per_wg = 1;
  while (!kDecode && p.tokens_per_wg < kQ8Block && p.n_rows > kEachRow * p.tokens_per_wg) p.tokens_per_wg *= 2;
  const int32_t stride = kQ8Block / p.tokens_per_wg;
  p.n_append_wg = (int32_t)((p.n_rows + kQ8Block - 1) / kQ8Block) * stride;
  const bool many = 2 * p.H_kv > kFewWaves && (!kRope || p.n_rows <= kEachRow);
  return D == 64 ? (many ? q8_launch<64, kManyWaves, kDecode, kRope>(p, stream)
                         : q8_launch<64, kFewWaves, kDecode, kRope>(p, stream))
                 : (many ? q8_launch<128, kManyWaves, kDecode, kRope>(p, stream)
                         : q8_launch<128, kFewWaves, kDecode, kRope>(p, stream));
}

static Q8Params q8_params(void* k_pool, void* v_pool, void* scales, int64_t n_rows, int64_t H_kv, int64_t page_size,
                          int64_t n_pages, int64_t page_stride, int64_t head_stride, int32_t* err) {
  Q8Params p{};
  p.k_pool = static_cast<uint8_t*>(k_pool);
  p.v_pool = static_cast<uint8_t*>(v_pool);
  p.scales = static_cast<float*>(scales);
  p.n_rows = n_rows;
  p.H_kv = (int32_t)H_kv;
  p.page_size = (int32_t)page_size;
  p.n_pages = n_pages;
  p.pool_page_stride = page_stride;
  p.pool_head_stride = head_stride;
  p.err = err;
  return p;
}

static int q8_new_rows(Q8Params& p, const void* k_new, const void* v_new, int64_t k_tok, int64_t k_head,
                       int64_t v_tok, int64_t v_head) {
  if (!k_new || !v_new || !q8_aligned(k_new) || !q8_aligned(v_new) || k_tok % 8 != 0 || k_head % 8 != 0 ||
      v_tok % 8 != 0 || v_head % 8 != 0)
    return CIE_EINVAL;
  p.k_new = static_cast<const f16*>(k_new);
  p.v_new = static_cast<const f16*>(v_new);
  p.k_tok_stride = k_tok;
  p.k_head_stride = k_head;
  p.v_tok_stride = v_tok;
  p.v_head_stride = v_head;
  return CIE_OK;
}

}  // namespace cie

using namespace cie;

extern "C" int cie_q8_append_decode(void* k_pool, void* v_pool, void* scales, const void* k_new, const void* v_new,
                                    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride,
                                    int64_t v_head_stride, const int64_t* slot_ids, const int64_t* lens,
                                    const int64_t* block_table, int64_t B, int64_t H_kv, int64_t page_size, int64_t D,
                                    int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
                                    int64_t bt_stride, int64_t bt_width, int64_t n_slots, int32_t* err, void* stream) {
  if (B < 0 || bt_width <= 0 || bt_stride < bt_width || n_slots <= 0) return CIE_EINVAL;
  if (int rc = q8_check_pools(k_pool, v_pool, scales, H_kv, page_size, D, n_pages, pool_page_stride, pool_head_stride))
    return rc;
  if (bt_width > 0x7fffffff / page_size) return CIE_EUNSUPPORTED;
  if (B == 0) return CIE_OK;
  if (!slot_ids || !lens || !block_table) return CIE_EINVAL;
  Q8Params p = q8_params(k_pool, v_pool, scales, B, H_kv, page_size, n_pages, pool_page_stride, pool_head_stride, err);
  if (int rc = q8_new_rows(p, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride)) return rc;
  p.slot_ids = slot_ids;
  p.lens = lens;
  p.block_table = block_table;
  p.bt_stride = bt_stride;
  p.bt_width = bt_width;
  p.n_slots = n_slots;
  return q8_launch_append<true, false>(p, D, static_cast<hipStream_t>(stream));
}

extern "C" int cie_q8_append_tokens(void* k_pool, void* v_pool, void* scales, const void* k_new, const void* v_new,
                                    int64_t k_tok_stride, int64_t k_head_stride, int64_t v_tok_stride,
                                    int64_t v_head_stride, const int64_t* pages, const int64_t* offsets, int64_t T,
                                    int64_t H_kv, int64_t page_size, int64_t D, int64_t n_pages,
                                    int64_t pool_page_stride, int64_t pool_head_stride, int32_t* err, void* stream) {
  if (T < 0) return CIE_EINVAL;
  if (int rc = q8_check_pools(k_pool, v_pool, scales, H_kv, page_size, D, n_pages, pool_page_stride, pool_head_stride))
    return rc;
  if (T == 0) return CIE_OK;
  if (!pages || !offsets) return CIE_EINVAL;
  Q8Params p = q8_params(k_pool, v_pool, scales, T, H_kv, page_size, n_pages, pool_page_stride, pool_head_stride, err);
  if (int rc = q8_new_rows(p, k_new, v_new, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride)) return rc;
  p.pages = pages;
  p.offsets = offsets;
  return q8_launch_append<false, false>(p, D, static_cast<hipStream_t>(stream));
}

extern "C" int cie_q8_append_tokens_qkv_rope(void* q_out, void* k_pool, void* v_pool, void* scales, const void* qkv,
                                             int64_t qkv_row_stride, const void* cos, const void* sin,
                                             int64_t cs_row_stride, const int64_t* pages, const int64_t* offsets,
                                             int64_t T, int64_t H_q, int64_t H_kv, int64_t page_size, int64_t D,
                                             int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
                                             int32_t* err, void* stream) {
  if (T < 0 || H_q <= 0) return CIE_EINVAL;
  if (int rc = q8_check_pools(k_pool, v_pool, scales, H_kv, page_size, D, n_pages, pool_page_stride, pool_head_stride))
    return rc;
  if (H_q > 65535) return CIE_EUNSUPPORTED;
  if (T == 0) return CIE_OK;
  if (!q_out || !qkv || !cos || !sin || !pages || !offsets || !q8_aligned(q_out) || !q8_aligned(qkv) ||
      !q8_aligned(cos) || !q8_aligned(sin) || qkv_row_stride % 8 != 0 || cs_row_stride % 8 != 0 ||
      qkv_row_stride < (H_q + 2 * H_kv) * D || cs_row_stride < D)
    return CIE_EINVAL;
  Q8Params p = q8_params(k_pool, v_pool, scales, T, H_kv, page_size, n_pages, pool_page_stride, pool_head_stride, err);
  const f16* const row = static_cast<const f16*>(qkv);
  p.k_new = row + H_q * D;
  p.v_new = row + (H_q + H_kv) * D;
  p.k_tok_stride = p.v_tok_stride = qkv_row_stride;
  p.k_head_stride = p.v_head_stride = D;
  p.q_out = static_cast<f16*>(q_out);
  p.qkv = row;
  p.cos = static_cast<const f16*>(cos);
  p.sin = static_cast<const f16*>(sin);
  p.qkv_stride = qkv_row_stride;
  p.cs_stride = cs_row_stride;
  p.pages = pages;
  p.offsets = offsets;
  p.H_q = (int32_t)H_q;
  return q8_launch_append<false, true>(p, D, static_cast<hipStream_t>(stream));
}

extern "C" int cie_q8_read_tokens(void* k_out, void* v_out, const void* k_pool, const void* v_pool,
                                  const void* scales, const int64_t* pages, const int64_t* offsets, int64_t T,
                                  int64_t H_kv, int64_t page_size, int64_t D, int64_t n_pages,
                                  int64_t pool_page_stride, int64_t pool_head_stride, int32_t* err, void* stream) {
  if (T < 0) return CIE_EINVAL;
  if (int rc = q8_check_pools(k_pool, v_pool, scales, H_kv, page_size, D, n_pages, pool_page_stride, pool_head_stride))
    return rc;
  if (T == 0) return CIE_OK;
  if (!k_out || !v_out || !pages || !offsets || !q8_aligned(k_out) || !q8_aligned(v_out)) return CIE_EINVAL;
  Q8ReadParams p{static_cast<f16*>(k_out), static_cast<f16*>(v_out), static_cast<const uint8_t*>(k_pool),
                 static_cast<const uint8_t*>(v_pool), static_cast<const float*>(scales), pages, offsets, T, n_pages,
                 pool_page_stride, pool_head_stride, (int32_t)H_kv, (int32_t)page_size, err};
  if (T > 0x7fffffffLL * 256 / (H_kv * (D / 8))) return CIE_EUNSUPPORTED;
  const int64_t blocks = (T * H_kv * (D / 8) + 255) / 256;
  if (D == 64)
    hipLaunchKernelGGL(q8_read_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), p);
  else
    hipLaunchKernelGGL(q8_read_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}
