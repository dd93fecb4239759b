// Low-rank adapters of many requests beside a shared projection:
//   y[t, s] += scale_i * B_is (A_is x_t),   i = the adapter of row t's request,
// for the slices s of y's columns (a fused projection has one a part).
//
// cie_adapter_plan sorts a step's rows by adapter into tiles of up to M rows of
// one adapter (M = 16 or 32), once for all of the step's projections.
// cie_adapter_add is one launch: a workgroup takes a tile and a range of y's
// columns.  Its eight waves share the sum over d_in (64 values of x at a time each,
// MFMA 16x16x32, ranks as rows and tokens as columns), their partial sums meet in
// LDS, and then each wave takes 64 columns of y at a time.  So x is read once and y
// read and written once, and nothing goes through memory between the two products.
//
// u = A x is fp32.  It enters the second product as values of the element type, u = hi +
// lo, side by side in the MFMA's K: 16 ranks fill K = 32, and B's values serve both
// halves.  In bf16 a third value, in an MFMA of its own, takes what the 16 bits of the two
// leave: the three hold all 24 bits of u.  In fp16 each row of a slice's u is first scaled by
// a power of two to below 2^15, so that no u overflows or loses bits to fp16's range; what is
// left of its rounding is 2^-22 of it, or 2^-39 of the row's largest in its slice.  The sum
// with y rounds once, as the plain form does.
//
// Bound by memory where rows are many: r <= 128 ranks are 2 r flops for each value of x
// and y, far from what the matrix cores could do.  8,192 rows of 4,096 take 45.9 us at
// rank 16 (4.4 TB/s), 54 at 64 and 80 at 128 (a workgroup fills a CU's LDS, so that its reads
// of x and its work on y take turns); in bf16, with the third value's MFMAs, 45.9, 56.4 and
// 84.  Few rows are bound by the stages in series, header ->
// tile -> x and A -> sums -> y: 6.2 us for one row into three slices.
#include "cie_common.h"

namespace cie {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class E>
struct Lane8;
template <>
struct Lane8<f16> {
  typedef f16x8 type;
};
template <>
struct Lane8<bf16> {
  typedef bf16x8 type;
};
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// ---- the plan ----

constexpr int kAdMaxAdapters = 1024;
constexpr int64_t kAdMaxRows = 1 << 24;
constexpr int kAdMaxSlices = 4;
constexpr int kAdMagic = 0x61647031;
// Header words: tiles, T, N, M, kAdMagic; then tiles of kAdTileHead + M words:
// adapter, rows, two unused, the rows' indexes.
constexpr int kAdHead = 8, kAdTileHead = 4;
constexpr int kPlanWaves = 16;
constexpr int kPlanThreads = kPlanWaves * kWave;
constexpr int kPlanBatch = 8;  // rows of a lane whose loads are in flight
constexpr int kPlanKept = 16;  // and that are kept from the count for the writing

// Rows of a tile: more share A's and B's reads, fewer fill the chip.  (1,052 rows of
// 1,000 at rank 64: 9.3 us with 16, 9.7 with 32; 2,048 rows of 4,096 31.2 and 22.1.)
__host__ __device__ static inline int tile_rows(int64_t T) { return T <= 1536 ? 16 : 32; }
static inline int64_t max_tiles(int64_t T, int64_t N, int M) {
  const int64_t groups = T < N ? T : N;  // (a group of c rows has ceil(c / M) <= (c - 1) / M + 1 tiles)
  return groups + (T - groups) / M;
}

struct PlanParams {
  int32_t* plan;
  const int64_t* row_slots;
  const int64_t* slot_adapters;
  int64_t T, n_slots;
  int64_t rows, share;  // of a workgroup, of a wave
  int32_t* counts;      // [groups][N] rows of a workgroup, where there are several
  int32_t N, M, log_m, groups;
  int32_t* err;
};

// Many rows are planned by several workgroups in two launches: each counts its rows,
// then each writes its rows behind those of the workgroups before it.  One workgroup
// does both at once, bound by a CU's loads and the rounds of its waves: 32 rows 4.0 us,
// 1,052 rows 5.0, 8,192 rows of four prompts 9.1 (two launches 10.2), of eight adapters at
// random 12.3 (10.8); 16,384 rows of four prompts 15.3 and 11.1, 65,536 rows 77 and 16.6.
// (Prompts decide: thousands of rows are prompts, each with one adapter, as a decoding
// request has a row or a few.)
constexpr int64_t kPlanAlone = 8192;
constexpr int kPlanGroups = 64;
static inline int64_t group_rows(int64_t T) {
  if (T <= kPlanAlone) return T;
  const int64_t rows = (T + kPlanGroups - 1) / kPlanGroups;
  return (rows + kPlanThreads - 1) / kPlanThreads * kPlanThreads;
}
enum PlanPhase { kPlanAll, kPlanCount, kPlanWrite };

// Rows are dealt to the waves in order, 64 adjacent rows at a time, and each wave
// counts its own, so that a group's rows keep their order and the plan is the same
// every time.  Lanes of one adapter find each other by a ballot a bit of its number,
// and the first of them takes as many places as they are (64 rows of one adapter need no
// ballots: 8,192 rows of four prompts 12.2 us with, 10.3 without; and 9.1 with tiles' heads
// written along with their first rows, not at the end).  Two dependent loads, the count, a
// scan over adapters, the rows.  The code is kept short (loops are not
// unrolled but for the loads'): it runs once, from a cold instruction cache.
template <PlanPhase kPhase>
__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(PlanParams p) {
  __shared__ int count[kPlanWaves * kAdMaxAdapters];  // [wave][N]: rows of a wave, then their first place
  __shared__ int tile0[kAdMaxAdapters], rows_of[kAdMaxAdapters], sums[kPlanWaves];
  __shared__ int seen[kPlanWaves][kPlanKept][kWave];   // rows' adapters and places (kPlaceBits), -1: none
  constexpr int kPlaceBits = 21;                       // (a wave has 2^20 rows at most)
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row0 = kPhase == kPlanAll ? 0 : blockIdx.x * p.rows, row1 = min(row0 + p.rows, p.T);
  const int64_t share = p.share, first = row0 + wave * share, end = min(first + share, row1);
  const int waves = (int)((row1 - row0 + share - 1) / share);  // that have rows
  const int bits = 32 - __builtin_clz(p.N);
  const uint64_t below = (1ull << lane) - 1;
  int* const mine = count + wave * p.N;

  int mistakes = 0, total = 0, n = 0;
  int* const out = p.plan + kAdHead;
  const int words = kAdTileHead + p.M;
  const bool again = share > kPlanKept * kWave;  // (else a wave's places are still there the second time)
  for (int i = tid; i < waves * p.N; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  for (int pass = 0; pass < 2; ++pass) {  // counted, then written
    for (int64_t at = first; at < end; at += kPlanBatch * kWave) {
      const int batch = (int)min((end - at + kWave - 1) / kWave, (int64_t)kPlanBatch);
      int(*const kept)[kWave] = seen[wave] + (again ? 0 : (int)(at - first) / kWave);
      if (pass == 0 || again) {
        int64_t slot[kPlanBatch];
#pragma unroll
        for (int i = 0; i < kPlanBatch; ++i) {
          const int64_t row = at + lane + i * kWave;
          slot[i] = row < end ? (p.row_slots ? p.row_slots[row] : row) : -1;
          if (row < end && (slot[i] < 0 || slot[i] >= p.n_slots)) {
            mistakes |= CIE_ERRBIT_PAGE;
            slot[i] = -1;
          }
        }
#pragma unroll
        for (int i = 0; i < kPlanBatch; ++i) {
          const int64_t a = p.slot_adapters[max(slot[i], (int64_t)0)];
          const bool none = slot[i] < 0 || a < 0 || a >= p.N;
          if (slot[i] >= 0 && a >= p.N) mistakes |= CIE_ERRBIT_ADAPTER;
          if (i < batch) kept[i][lane] = none ? -1 : (int)a << kPlaceBits;
        }
      }
#pragma unroll 1
      for (int i = 0; i < batch; ++i) {
        const int was = kept[i][lane], id = was >> kPlaceBits;
        const bool live = was >= 0;
        int place = was & ((1 << kPlaceBits) - 1);
        if (pass == 0 || again) {
          uint64_t same = __ballot(live);
          if (__ballot(id != uniform(id)) != 0)  // (a prompt's rows: all of one)
#pragma unroll 1
            for (int k = 0; k < bits; ++k) {
              const uint64_t ones = __ballot(id >> k & 1);
              same &= id >> k & 1 ? ones : ~ones;
            }
          int from = 0;
          if (live && (same & below) == 0) from = atomicAdd(&mine[id], __popcll(same));
          place = __shfl(from, live ? __builtin_ctzll(same) : 0, kWave) + __popcll(same & below);
          if (pass == 0 && !again && live) kept[i][lane] = id << kPlaceBits | place;
        }
        if (pass == 1 && live) {
          const int k = place + (again ? 0 : mine[id]);
          int* const tile = out + (int64_t)(tile0[id] + (k >> p.log_m)) * words;
          const int nth = k & (p.M - 1);
          tile[kAdTileHead + nth] = (int)(at + i * kWave + lane);
          if (nth == 0) {  // a tile's first row writes its head
            tile[0] = id;
            tile[1] = min(rows_of[id] - k, p.M);
          }
        }
      }
    }
    if (pass == 1) break;
    __syncthreads();
    // Adapter a's rows before each wave's, and its tiles.
    int rest = 0;  // rows of the workgroups from this one on
    if (kPhase == kPlanWrite && tid < p.N) {
#pragma unroll 8
      for (int w = 0; w < p.groups; ++w) {
        const int c = p.counts[w * p.N + tid];
        if (w < (int)blockIdx.x)
          n += c;
        else
          rest += c;
      }
      rest += n;
    }
    if (tid < p.N) {
#pragma unroll 1
      for (int w0 = 0; w0 < waves; w0 += 4) {  // (four reads, then four writes: one wait for each four)
        int c[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) c[w] = w0 + w < waves ? count[(w0 + w) * p.N + tid] : 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (w0 + w < waves) count[(w0 + w) * p.N + tid] = n;
          n += c[w];
        }
      }
    }
    if constexpr (kPhase == kPlanCount) {
      if (tid < p.N) p.counts[blockIdx.x * p.N + tid] = n;
      break;
    }
    if (kPhase == kPlanWrite) n = rest;  // (all its rows)
    const int tiles = (n + p.M - 1) >> p.log_m;
    const int incl = wave_inclusive_sum(tiles);
    if (lane == kWave - 1) sums[wave] = incl;
    __syncthreads();
    const int before = incl - tiles + waves_before<kPlanWaves>(sums[lane % kPlanWaves], wave, total);
    if (tid < p.N) {
      tile0[tid] = before;
      rows_of[tid] = n;
    }
    __syncthreads();
  }
  if (mistakes && kPhase != kPlanWrite) set_err(p.err, mistakes);  // (counted rows have been looked at)
  if (kPhase == kPlanCount || blockIdx.x > 0) return;
  if (tid == 0) {
    p.plan[0] = total;
    p.plan[1] = (int)p.T;
    p.plan[2] = p.N;
    p.plan[3] = p.M;
    p.plan[4] = kAdMagic;
  }
}

// ---- the products ----

constexpr int kAdBlock = 64;   // values of x a wave takes at a time: two MFMAs
constexpr int kAdUnits = 8;    // 16-rank units of u held at once: one slice of 128 ranks, or several of fewer

constexpr int kCus = 256;
constexpr int kAdWaves = 8;
constexpr int kAdThreads = kAdWaves * kWave;

struct AddParams {
  void* y;
  const void* x;
  const void* a;
  const void* b;
  const float* scales;
  const int32_t* ranks;
  const int32_t* plan;
  int64_t y_stride, x_stride;
  int32_t T, N, R, d_in, d_out, n_slices, chunks, per_chunk, col_tiles, max_tiles;
  int32_t slice_col[kAdMaxSlices + 1];   // a slice's first column
  int32_t slice_tile[kAdMaxSlices + 1];  // and its first 64-column tile
  int32_t* err;
};

// Eight values from k on, zeros at and past n.  Rows at any 2-byte address: one load all
// the same (global memory may be read so), but for the last few values.
template <class E, bool kAligned>
__device__ __forceinline__ typename Lane8<E>::type load8(const E* row, int k, int n) {
  typedef typename Lane8<E>::type vec;
  typedef vec any_vec __attribute__((aligned(2)));
  vec v = {};
  if constexpr (kAligned) {
    if (k < n) v = *reinterpret_cast<const vec*>(row + k);
  } else if (k + 8 <= n) {
    v = *reinterpret_cast<const any_vec*>(row + k);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (k + e < n) v[e] = row[k + e];
  }
  return v;
}
template <class E, bool kAligned>
__device__ __forceinline__ void store8(E* row, int k, int n, typename Lane8<E>::type v) {
  typedef typename Lane8<E>::type vec;
  typedef vec any_vec __attribute__((aligned(2)));
  if constexpr (kAligned) {
    if (k < n) *reinterpret_cast<vec*>(row + k) = v;
  } else if (k + 8 <= n) {
    *reinterpret_cast<any_vec*>(row + k) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (k + e < n) row[k + e] = v[e];
  }
}

// 2^e that takes m (fp16: the largest |u| of a row's slice) to [2^14, 2^15); 1 where there is no such.
template <class E>
__device__ __forceinline__ int row_shift(float m) {
  if constexpr (sizeof(E) == 2 && __is_same(E, f16)) {
    if (!(m > 0.f)) return 0;
    return min(15 - __builtin_amdgcn_frexp_expf(m), 100);
  }
  return 0;
}

// The largest of a row of 16 lanes (v >= 0), in each of them: rotations by 8, 4, 2 and 1, no LDS.
__device__ __forceinline__ float max_of_16(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, true)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true)));
}

// Copies 16 bytes a lane from p to the wave's KiB at dst (LDS, lane order), without
// passing through registers.  Assembly, as the compiler would make every later LDS
// read wait for all copies in flight; wait_copies publishes them to the wave.
__device__ __forceinline__ void copy16(void* dst, const void* p) {
  typedef __attribute__((address_space(3))) char lds_char;
  const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
// Every LDS read of this wave has returned: what it read may be overwritten.
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// Lanes of a wave read what others of it wrote: LDS accesses run in order, and the compiler keeps theirs here.
__device__ __forceinline__ void lds_order() { asm volatile("" : : : "memory"); }

// LDS of an instance.  A wave has a region of its own: a stage, which holds kDepth
// blocks of x and A on their way to the matrix cores, then the wave's partial sums of
// u, then the products for 16 rows of 64 columns; and room for B's values.
template <class E, int MR, int NT>
struct AddLds {
  static constexpr int M = 16 * MR;
  static constexpr int kDepth = MR == 1 ? (NT == 1 ? 4 : NT < 4 ? 2 : 1) : (NT == 1 ? 2 : 1);
  static constexpr int kSlab = 2048;                // 16 rows of 64 values
  static constexpr int kBlock = (MR + NT) * kSlab;  // a block: x's rows, then A's
  static constexpr int kStage = kDepth * kBlock;
  static constexpr int kSumRow = NT * 16 + 4;       // floats (padded: rows start in other banks)
  static constexpr int kOutRow = 64 + 4;
  static constexpr int kOut = 16 * kOutRow * 4;
  // B's values for 64 columns: 2 KiB a unit.  One or two units have room beside the
  // stage, and come in while it is in use; more (up to 8 KiB) lie behind the products.
  static constexpr int kB = NT == 1 || (NT == 3 && MR == 1) ? 2048 : 4096;
  static constexpr int kGroup = NT < 4 ? NT : 4;    // units whose B values are in LDS at once
  static constexpr int kRegion = kStage + kB;
  static_assert(M * kSumRow * 4 <= kStage && kOut <= kStage, "sums and products fit the stage");
  static_assert((kGroup < 3 ? kGroup * 2048 : 8192) <= (kGroup < 3 ? kB : kRegion - kOut), "B's values fit");
  // 16 ranks of u a unit: in fp32, then hi and lo, and in bf16 what these leave.
  static constexpr bool kThird = __is_same(E, bf16);
  static constexpr int kURow = kThird ? 96 : 64;
  static constexpr int kU = kAdUnits * M * kURow;
  static constexpr int kBytes = kAdWaves * kRegion + kU + kAdMaxSlices * M * 4;
  static_assert(kBytes <= 160 * 1024, "a workgroup's LDS");
};

// The code of small launches is kept short: each runs once, and a workgroup waits
// some 0.25 us for each further KiB of instructions (one row into three slices: 7.3 us
// with loops unrolled, 16 KB; 6.2 so).
template <class E, int MR, int NT, bool kAligned>
__global__ __launch_bounds__(kAdThreads) void adapter_add_kernel(AddParams p) {
  typedef typename Lane8<E>::type vec;
  typedef AddLds<E, MR, NT> L;
  constexpr int M = L::M, NW = kAdWaves, kDepth = L::kDepth;
  constexpr int kLanes = NT == 3 ? 16 : NT * 4;  // threads that sum a row of u, four ranks each
  constexpr int kHeld = NT < 4 ? NT : kAdUnits;  // units of u (fewer than four in all: the host's choice)
  static_assert(M * 16 <= kAdThreads, "a thread sums four values of u at most, and splits one a unit");
  __shared__ __align__(16) char lds[L::kBytes];
  char* const u_lds = lds + NW * L::kRegion;  // [unit][token]: 16 floats, or 16 his, 16 los (and 16 thirds)
  float* const factor = reinterpret_cast<float*>(u_lds + L::kU);  // [slice][token], of the slices at once

  // Which tile, and its rows.  Small launches deal tiles to the XCDs (workgroups go
  // to the eight in turn) one by one and read the tile's words along with the
  // header; large ones give an XCD adjacent tiles, mostly of one adapter, whose A
  // and B then come from its L2.
  // (Words that are no plan are found out below, after they have been used as one: the
  // count is kept to what there can be, so that no index leaves the buffer.)
  const int32_t* const head = p.plan;
  const int n_tiles = min(max(head[0], 0), p.max_tiles);
  const int xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
  int tile, chunk, per_chunk = p.per_chunk;
  if constexpr (MR == 1) {
    chunk = nth % p.chunks;
    tile = nth / p.chunks * 8 + xcd;
  } else {
    // Whole rounds of the CUs, a tile a workgroup; the tiles of the last round share
    // their columns among the CUs left (258 tiles of 32 rows of 4,096 at rank 64: 87 us
    // without this, 52 for 256).
    const int n = n_tiles, round = n / kCus * (kCus / 8), left = n % kCus;
    const int chunks = left ? min(p.chunks, kCus / left) : 1, items = left * chunks, share = (items + 7) / 8;
    if (nth < round) {
      tile = xcd * round + nth;
      chunk = 0;
      per_chunk = p.col_tiles;
    } else {
      const int item = nth - round < share ? xcd * share + nth - round : items;
      tile = item < items ? round * 8 + item / chunks : n;
      chunk = item % chunks;
      per_chunk = (p.col_tiles + chunks - 1) / chunks;
    }
  }
  const int32_t* const desc = p.plan + kAdHead + (int64_t)min(tile, p.max_tiles - 1) * (kAdTileHead + M);
  const int tid = threadIdx.x, lane = tid % kWave, wave = uniform(tid / kWave), m = lane % 16, g = lane / 16;
  const int r8 = lane / 8, c8 = lane % 8;  // memory order: eight rows of eight 16-byte pieces
  const int adapter = uniform(desc[0]), rows = uniform(desc[1]);
  int row_of[2 * MR];  // rows r8, 8 + r8, ... of the tile
#pragma unroll
  for (int r = 0; r < 2 * MR; ++r) row_of[r] = desc[kAdTileHead + 8 * r + r8];
  if (head[1] != p.T || head[2] != p.N || head[3] != M || head[4] != kAdMagic) {
    if (tid == 0 && blockIdx.x == 0) set_err(p.err, CIE_ERRBIT_PLAN);
    return;
  }
  if (tile >= n_tiles) return;
  const int ct0 = chunk * per_chunk, ct1 = min(ct0 + per_chunk, p.col_tiles);
  if (ct0 >= ct1) return;
  // The slices' first columns and column tiles, by index: not by a load each time.
  const auto slice_of = [&](int ct) {
    return (int)(ct >= p.slice_tile[1]) + (int)(ct >= p.slice_tile[2]) + (int)(ct >= p.slice_tile[3]);
  };
  const auto pick = [](const int32_t* v, int i) {
    return i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : i == 3 ? v[3] : v[4];
  };
  // (a tile's last rows: its first again, not written)
  const int row0 = uniform(row_of[0]);
#pragma unroll
  for (int r = 0; r < 2 * MR; ++r)
    if (8 * r + r8 >= rows) row_of[r] = row0;
  const int rank = p.ranks[adapter];
  const float scale = p.scales[adapter];
  // With one unit a slice the loads need not wait for the rank: an empty place is left at the end.
  const int units = p.R == 16 ? 1 : min(uniform((rank + 15) / 16), p.R / 16);
  if (units <= 0) return;
  const int at_once = units > kAdUnits / 2 ? 1 : units > 2 ? 2 : 4;  // slices whose u is held
  const int s_end = slice_of(ct1 - 1) + 1;

  char* const mine = lds + wave * L::kRegion;
  const E* x_row[2 * MR];
#pragma unroll
  for (int r = 0; r < 2 * MR; ++r) x_row[r] = static_cast<const E*>(p.x) + row_of[r] * p.x_stride;
  const int blocks = (p.d_in + kAdBlock - 1) / kAdBlock;
  // Slabs hold piece c of row r in place c ^ (r % 8): the lanes that read a piece of 16 rows meet no bank twice.
  const int k8 = 8 * (c8 ^ r8);
  const int64_t unit_step = (int64_t)16 * p.d_in, slice_step = (int64_t)p.R * p.d_in;

#pragma unroll 1
  for (int s0 = slice_of(ct0); s0 < s_end; s0 += at_once) {
    const int s1 = min(s0 + at_once, s_end);  // slices [s0, s1) of this workgroup's columns
    const int n_units = (s1 - s0) * units;

    // The 64 columns that come next: their slice, first and last column, y's values (in
    // memory order) and B's first units.
    const int first = max(ct0, pick(p.slice_tile, s0)), last = min(ct1, pick(p.slice_tile, s1));
    const int b_first = min(units, L::kGroup);
    const bool beside = (b_first == 1 ? 2048 : b_first == 2 ? 4096 : 8192) <= L::kB;
    char* const b_room = mine + (beside ? L::kStage : L::kOut);
    float* const out = reinterpret_cast<float*>(mine);
    int cs = 0, c0 = 0, c1 = 0;
    vec y_in[2 * MR];
    // Columns of 2, 4 or 8 pieces, piece c of column d in place c ^ (d / (8 / pieces) % pieces).
    const auto fetch_b = [&](int i0) {
      const int n = min(units - i0, L::kGroup);
      const int shift = n == 1 ? 1 : n == 2 ? 2 : 3, pieces = 1 << shift;
      const E* const from = static_cast<const E*>(p.b) + ((int64_t)adapter * p.d_out + c0) * p.R + 16 * i0;
#pragma unroll 1
      for (int k = 0; k < pieces; ++k) {
        const int d = (64 * k + lane) >> shift, c = lane % pieces ^ (d >> (3 - shift)) % pieces;
        if (c < 2 * n) copy16(b_room + 1024 * k, from + (int64_t)min(d, c1 - 1 - c0) * p.R + 8 * c);
      }
    };
    const auto open = [&](int ct) {
      cs = slice_of(ct);
      c0 = pick(p.slice_col, cs) + (ct - pick(p.slice_tile, cs)) * 64;
      c1 = pick(p.slice_col, cs + 1);
#pragma unroll
      for (int r = 0; r < 2 * MR; ++r)
        y_in[r] = load8<E, kAligned>(static_cast<const E*>(p.y) + row_of[r] * p.y_stride, c0 + 8 * c8, c1);
      fetch_b(0);
    };

    // u = A x, NT units at a time.
    int in_slice = 0;
    const E* a_unit = static_cast<const E*>(p.a) + ((int64_t)adapter * p.n_slices + s0) * slice_step + (int64_t)r8 * p.d_in;
#pragma unroll 1
    for (int u0 = 0; u0 < n_units; u0 += NT) {
      const int now = min(n_units - u0, NT);
      f32x4 acc[MR][NT] = {};
      // Block b's rows into place d of the wave's stage.
      const auto fetch = [&](int b, int d) {
        char* to = mine + d * L::kBlock;
        const int k = b * kAdBlock + k8;
        // (a row's last block: zeros past its end)
        const bool in = k < p.d_in;
#pragma unroll
        for (int r = 0; r < 2 * MR; ++r, to += 1024) {
          if (!kAligned)
            reinterpret_cast<vec*>(to)[lane] = load8<E, false>(x_row[r], k, p.d_in);
          else if (in)
            copy16(to, x_row[r] + k);
          else
            reinterpret_cast<vec*>(to)[lane] = vec{};
        }
        const E* row = a_unit;
        int i = in_slice;
#pragma unroll 1
        for (int n = 0; n < 2 * now; ++n, to += 1024) {
          if (!kAligned)
            reinterpret_cast<vec*>(to)[lane] = load8<E, false>(row, k, p.d_in);
          else if (in)
            copy16(to, row + k);
          else
            reinterpret_cast<vec*>(to)[lane] = vec{};
          row += unit_step / 2;
          if (n % 2 && ++i == units) {
            i = 0;
            row += slice_step - units * unit_step;
          }
        }
      };
      // Each place's next block is on its way while the matrix cores have the others.
#pragma unroll 1
      for (int d = 0; d < kDepth; ++d)
        if (wave + d * NW < blocks) fetch(wave + d * NW, d);
      if (MR == 1 && u0 == 0 && beside && first + wave < last) open(first + wave);
#pragma unroll 1
      for (int b = wave, d = 0; b < blocks; b += NW, d = d + 1 == kDepth ? 0 : d + 1) {
        vec xv[MR][2], av[NT][2];
        if (kDepth == 1 || d == 0) wait_copies();
        const char* const from = mine + d * L::kBlock + m * 128;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = 16 * ((4 * j + g) ^ (m % 8));
#pragma unroll
          for (int r = 0; r < MR; ++r) xv[r][j] = *reinterpret_cast<const vec*>(from + r * L::kSlab + at);
#pragma unroll
          for (int n = 0; n < NT; ++n) av[n][j] = *reinterpret_cast<const vec*>(from + (MR + n) * L::kSlab + at);
        }
        wait_lds_reads();
        if (b + NW * kDepth < blocks) fetch(b + NW * kDepth, d);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < MR; ++r) acc[r][n] = mma(av[n][j], xv[r][j], acc[r][n]);  // (n >= now: not used)
      }
      for (int n = 0; n < now; ++n) {
        a_unit += unit_step;
        if (++in_slice == units) {
          in_slice = 0;
          a_unit += slice_step - units * unit_step;
        }
      }
      // A lane has ranks 4g .. 4g + 3 of token m.
      float* const sums = reinterpret_cast<float*>(mine) + m * L::kSumRow + 4 * g;
#pragma unroll
      for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          *reinterpret_cast<f32x4*>(sums + 16 * r * L::kSumRow + 16 * n) = acc[r][n];
      __syncthreads();
      if (tid < M * kLanes && tid % kLanes < 4 * now) {
        const int t = tid / kLanes, q = tid % kLanes;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
          sum += reinterpret_cast<const f32x4*>(lds + w * L::kRegion)[t * (L::kSumRow / 4) + q];
        reinterpret_cast<f32x4*>(u_lds + ((u0 + q / 4) * M + t) * L::kURow)[q % 4] = sum;
      }
      __syncthreads();
    }

    // u's parts, slice by slice: sixteen lanes a row, one rank of each unit.
    if (tid < M * 16) {
      const int t = tid / 16, q = tid % 16;
#pragma unroll 1
      for (int s = 0; s < s1 - s0; ++s) {
        char* const row = u_lds + (s * units * M + t) * L::kURow;
        float v[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i)  // (past the slice's units: its last again, so that all loads go at once)
          v[i] = reinterpret_cast<const float*>(row + min(i, units - 1) * M * L::kURow)[q];
        int shift = 0;
        if constexpr (__is_same(E, f16)) {
          // The largest finite |u| of the row's slice decides its scale: an infinity stays one.
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (__builtin_fabsf(v[i]) < __builtin_huge_valf()) top = fmaxf(top, __builtin_fabsf(v[i]));
          shift = row_shift<E>(max_of_16(top));
        }
        lds_order();  // (the row's lanes are one wave's: all have read)
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          if (i >= units) break;
          E* const at = reinterpret_cast<E*>(row + i * M * L::kURow);
          const float u = __builtin_ldexpf(v[i], shift), left = u - (float)(E)u;
          const float lo = __builtin_isfinite(left) ? left : 0.f;  // (of an infinity, a NaN: hi says it)
          at[q] = (E)u;
          at[16 + q] = (E)lo;
          if constexpr (L::kThird) at[32 + q] = (E)(lo - (float)(E)lo);
        }
        if (q == 0) factor[s * M + t] = __builtin_ldexpf(scale, -shift);
      }
    }
    __syncthreads();
    if (rank <= 0) return;

    // y += scale B u: 64 columns at a time, B's rows as rows and tokens as columns of
    // the product, which goes through LDS to the memory's order.
    if (!(MR == 1 && beside) && first + wave < last) open(first + wave);
#pragma unroll 1
    for (int ct = first + wave; ct < last; ct += NW) {
      const int s = cs, col = c0, end = c1;
      vec yv[2 * MR];
#pragma unroll
      for (int r = 0; r < 2 * MR; ++r) yv[r] = y_in[r];
      f32x4 acc[MR][4] = {};
#pragma unroll 1
      for (int i0 = 0; i0 < units; i0 += L::kGroup) {
        const int n = min(units - i0, L::kGroup);
        const int shift = n == 1 ? 1 : n == 2 ? 2 : 3, pieces = 1 << shift;
        if (i0 > 0) fetch_b(i0);
        wait_copies();
        // 16 ranks at a time: hi and lo in one K of 32, B's values twice
#pragma unroll 2
        for (int i = 0; i < n; ++i) {
          vec bv[4], uv[MR], third[MR] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d = 16 * j + m, c = 2 * i + g % 2;
            bv[j] = *reinterpret_cast<const vec*>(b_room + ((d << shift) + (c ^ (d >> (3 - shift)) % pieces)) * 16);
          }
#pragma unroll
          for (int r = 0; r < MR; ++r) {
            const char* const at = u_lds + (((s - s0) * units + i0 + i) * M + 16 * r + m) * L::kURow + 16 * g;
            uv[r] = *reinterpret_cast<const vec*>(at);
            if (L::kThird && g < 2) third[r] = *reinterpret_cast<const vec*>(at + 64);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < MR; ++r) {
              if constexpr (L::kThird) acc[r][j] = mma(bv[j], third[r], acc[r][j]);  // (half of K: zeros)
              acc[r][j] = mma(bv[j], uv[r], acc[r][j]);
            }
        }
        wait_lds_reads();
      }
      if (ct + NW < last) open(ct + NW);
#pragma unroll
      for (int r = 0; r < MR; ++r) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(out + m * L::kOutRow + 16 * j + 4 * g) = acc[r][j];
        lds_order();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = 8 * h + r8, c = col + 8 * c8;
          const f32x4* const got = reinterpret_cast<const f32x4*>(out + t * L::kOutRow + 8 * c8);
          const f32x4 lo = got[0], hi = got[1];
          if (16 * r + t >= rows) continue;
          const float f = factor[(s - s0) * M + 16 * r + t];
          E* const to = static_cast<E*>(p.y) + row_of[2 * r + h] * p.y_stride;
          vec v;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float sum = __builtin_fmaf(e < 4 ? lo[e % 4] : hi[e % 4], f, (float)yv[2 * r + h][e]);
            asm volatile("" : "+v"(sum));  // (to fp32 first, in every variant: no v_fma_mixlo_f16)
            v[e] = (E)sum;
          }
          store8<E, kAligned>(to, c, end, v);
        }
        lds_order();
      }
    }
    if (s1 < s_end) __syncthreads();  // (the regions and u are used again)
  }
}

static bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

template <class E, int MR, bool kAligned>
static void launch_add(const AddParams& p, int units, dim3 grid, hipStream_t stream) {
  // Few units in all: no registers or partial sums for more.  (Unaligned rows: one, or any.)
  const dim3 block(kAdThreads);
  if (units == 1)
    hipLaunchKernelGGL((adapter_add_kernel<E, MR, 1, kAligned>), grid, block, 0, stream, p);
  else if (kAligned && units == 2)
    hipLaunchKernelGGL((adapter_add_kernel<E, MR, kAligned ? 2 : 4, kAligned>), grid, block, 0, stream, p);
  else if (kAligned && units == 3)
    hipLaunchKernelGGL((adapter_add_kernel<E, MR, kAligned ? 3 : 4, kAligned>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((adapter_add_kernel<E, MR, 4, kAligned>), grid, block, 0, stream, p);
}

template <class E>
static int dispatch_add(const AddParams& p, int units, bool aligned, dim3 grid, hipStream_t stream) {
  if (tile_rows(p.T) == 16)
    aligned ? launch_add<E, 1, true>(p, units, grid, stream) : launch_add<E, 1, false>(p, units, grid, stream);
  else
    aligned ? launch_add<E, 2, true>(p, units, grid, stream) : launch_add<E, 2, false>(p, units, grid, stream);
  return (int)hipGetLastError();
}

}  // namespace cie

using namespace cie;

extern "C" int64_t cie_adapter_plan_bytes(int64_t T, int64_t N) {
  if (T < 0 || N <= 0 || T > kAdMaxRows || N > kAdMaxAdapters) return -1;
  const int M = tile_rows(T);
  const int64_t groups = T > kPlanAlone ? (T + group_rows(T) - 1) / group_rows(T) : 0;
  return 4 * (kAdHead + max_tiles(T, N, M) * (kAdTileHead + M) + groups * N);
}

extern "C" int cie_adapter_plan(int32_t* plan, int64_t plan_bytes, const int64_t* row_slots,
                                const int64_t* slot_adapters, int64_t T, int64_t n_slots, int64_t N, int32_t* err,
                                void* stream) {
  if (T < 0 || N <= 0 || n_slots <= 0) return CIE_EINVAL;
  if (T > kAdMaxRows || N > kAdMaxAdapters) return CIE_EUNSUPPORTED;
  if (!plan || !aligned16(plan) || plan_bytes < cie_adapter_plan_bytes(T, N) || !slot_adapters ||
      (!row_slots && n_slots < T))
    return CIE_EINVAL;
  PlanParams p{};
  p.plan = plan;
  p.row_slots = row_slots;
  p.slot_adapters = slot_adapters;
  p.T = T;
  p.n_slots = n_slots;
  p.N = (int32_t)N;
  p.M = tile_rows(T);
  p.log_m = p.M == 16 ? 4 : 5;
  p.err = err;
  p.rows = group_rows(T);
  p.share = (p.rows + kPlanThreads - 1) / kPlanThreads * kWave;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (T == 0) return CIE_OK;
  if (T <= kPlanAlone) {
    hipLaunchKernelGGL(adapter_plan_kernel<kPlanAll>, dim3(1), dim3(kPlanThreads), 0, st, p);
    return (int)hipGetLastError();
  }
  p.groups = (int32_t)((T + p.rows - 1) / p.rows);
  p.counts = plan + kAdHead + max_tiles(T, N, p.M) * (kAdTileHead + p.M);
  hipLaunchKernelGGL(adapter_plan_kernel<kPlanCount>, dim3((unsigned)p.groups), dim3(kPlanThreads), 0, st, p);
  const int status = (int)hipGetLastError();
  if (status) return status;
  hipLaunchKernelGGL(adapter_plan_kernel<kPlanWrite>, dim3((unsigned)p.groups), dim3(kPlanThreads), 0, st, p);
  return (int)hipGetLastError();
}

extern "C" int cie_adapter_add(void* y, int64_t y_row_stride, const void* x, int64_t x_row_stride, const void* a,
                               const void* b, const float* scales, const int32_t* ranks, const int32_t* plan,
                               int64_t plan_bytes, int64_t T, int64_t N, int64_t R, int64_t d_in,
                               const int64_t* slice_widths, int64_t n_slices, int dtype, int32_t* err, void* stream) {
  if (T < 0 || N <= 0 || R <= 0 || d_in <= 0 || n_slices <= 0 || !slice_widths) return CIE_EINVAL;
  if (T > kAdMaxRows || N > kAdMaxAdapters || R % 16 || R > 16 * kAdUnits || d_in > 1 << 24 ||
      n_slices > kAdMaxSlices || (dtype != CIE_F16 && dtype != CIE_BF16))
    return CIE_EUNSUPPORTED;
  AddParams p{};
  bool aligned = d_in % 8 == 0 && x_row_stride % 8 == 0 && y_row_stride % 8 == 0 && aligned16(x) && aligned16(y) &&
                 aligned16(a);
  int64_t d_out = 0, tiles = 0;
  for (int s = 0; s < n_slices; ++s) {
    if (slice_widths[s] <= 0) return CIE_EINVAL;
    if (slice_widths[s] > 1 << 24) return CIE_EUNSUPPORTED;
    p.slice_col[s] = (int32_t)d_out;
    p.slice_tile[s] = (int32_t)tiles;
    d_out += slice_widths[s];
    tiles += (slice_widths[s] + 63) / 64;
    aligned = aligned && slice_widths[s] % 8 == 0;
  }
  for (int s = (int)n_slices; s <= kAdMaxSlices; ++s) {
    p.slice_col[s] = (int32_t)d_out;
    p.slice_tile[s] = (int32_t)tiles;
  }
  if (T == 0) return CIE_OK;
  if (!y || !x || !a || !b || !scales || !ranks || !plan || !aligned16(b) || !aligned16(plan) ||
      (T > 1 && (x_row_stride < d_in || y_row_stride < d_out)) || plan_bytes < cie_adapter_plan_bytes(T, N))
    return CIE_EINVAL;
  p.y = y;
  p.x = x;
  p.a = a;
  p.b = b;
  p.scales = scales;
  p.ranks = ranks;
  p.plan = plan;
  p.y_stride = y_row_stride;
  p.x_stride = x_row_stride;
  p.T = (int32_t)T;
  p.N = (int32_t)N;
  p.max_tiles = (int32_t)max_tiles(T, N, tile_rows(T));
  p.R = (int32_t)R;
  p.d_in = (int32_t)d_in;
  p.d_out = (int32_t)d_out;
  p.n_slices = (int32_t)n_slices;
  p.col_tiles = (int32_t)tiles;
  p.err = err;
  // Few tiles: several workgroups share one's columns (each computes u again), down to a
  // column tile a wave and a workgroup a CU.  Tiles of 16 rows go by how many tiles there
  // can be (their workgroups read their tile before they know how many there are).
  const int64_t most = (tiles + kAdWaves - 1) / kAdWaves;
  int64_t blocks;
  if (tile_rows(T) == 16) {
    int64_t chunks = kCus / p.max_tiles;
    chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
    p.per_chunk = (int32_t)((tiles + chunks - 1) / chunks);
    p.chunks = (int32_t)((tiles + p.per_chunk - 1) / p.per_chunk);
    blocks = (int64_t)(p.max_tiles + 7) / 8 * 8 * p.chunks;
  } else {
    p.chunks = (int32_t)most;
    blocks = (int64_t)kCus * (p.max_tiles / kCus + 1);
  }
  if (blocks > 0x7fffffff) return CIE_EUNSUPPORTED;
  const dim3 grid((unsigned)blocks);
  const int units = (int)(n_slices * (R / 16) < 5 ? n_slices * (R / 16) : 4);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CIE_F16 ? dispatch_add<f16>(p, units, aligned, grid, st) : dispatch_add<bf16>(p, units, aligned, grid, st);
}
