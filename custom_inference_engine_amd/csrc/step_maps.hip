// Block tables and slot maps from request lengths, on the GPU.
//
// A step has B sequences: slot s_b with l_b = lens[s_b] tokens held and n_b new
// ones, packed one after another.  cie_step_maps writes the packed offsets
// cu[b + 1] = cu[b] + n_b and, for row t of sequence b, its slot, its position
// l_b + t - cu[b], the page block_table[s_b, position / P] and the offset
// position % P.  With a free list it first gives each sequence the pages its new
// tokens need, ceil((l_b + n_b) / P) - ceil(l_b / P) of them.  cie_release_pages
// gives pages back.
//
// A free list is n_pages + 2 words: the count of free pages, a word that only
// these kernels use (zero between calls), and the pages, a stack whose top is the
// page handed out next.  Pages are handed out in the order of the sequences and,
// within one, of its positions, and taken back in the reverse order: giving back
// what a call was given leaves the list as it was.  Table entries that hold no page
// (0: a call whose pages the list did not have) are not given back: the last workgroup
// to arrive closes the gaps that they leave.
//
// Both are bound by latency, not by bytes: 40 bytes a row are written once.  So
// one launch does it all.  Every workgroup reads the B sequences and scans them
// for itself (two dependent round trips: slots and new lengths, then the held
// lengths), and no workgroup waits for what another writes: a row on a new page
// reads the page's id from the stack, at the place that the scan gives it, not
// from the table.  Words that other workgroups still read (the count, and a
// release's lengths) are changed by the last workgroup to arrive.
// Times of one call, replayed from a graph: one row 2.9 us, 32 sequences and 1,056
// rows 3.5 us, 496 sequences and 16,480 rows 4.2 us; with pages and their release
// 6.2 us for one sequence, 8.3 for 32, 14.9 for 496 with 16,480 rows and 1,480 new pages.
#include "cie_common.h"

namespace cie {

constexpr int kMapMaxSeqs = 2048;          // (scans and hash table of a batch: at most 74 KB of LDS)
constexpr int64_t kMapMaxRows = 1 << 24;   // sums over a batch stay below 2^31
constexpr int64_t kMapMaxPages = 1 << 24;
constexpr int64_t kMapMaxPage = 1 << 30;   // tokens a page: a page and a step's rows stay below 2^32

struct MapParams {
  int64_t* cu;         // (B + 1) or null
  int64_t* slots;      // (T) each, or null
  int64_t* positions;
  int64_t* pages;
  int64_t* offsets;
  const int64_t* slot_ids;
  const int64_t* counts;  // new tokens; release: tokens kept, or null (none)
  const int64_t* held;    // release: tokens whose pages are held, or null (lens)
  int64_t* lens;
  int64_t* block_table;
  int64_t* free_list;
  int64_t bt_stride, bt_width, n_slots, n_pages, T;
  double per_page;        // 1 / page_size
  int32_t B, page_size, hash_size;
  int32_t* err;
};

// Whole pages of n tokens, and the rest: 0 <= n <= 2^24 pages.  (The product is off by
// far less than one, so the quotient by one at most.)
__device__ __forceinline__ int whole_pages(int64_t n, const MapParams& p, uint32_t& rest) {
  int q = (int)((double)n * p.per_page);
  int64_t r = n - (int64_t)q * p.page_size;
  if (r < 0) {
    --q;
    r += p.page_size;
  } else if (r >= p.page_size) {
    ++q;
    r -= p.page_size;
  }
  rest = (uint32_t)r;
  return q;
}
__device__ __forceinline__ int pages_of(int64_t n, const MapParams& p) {
  uint32_t rest;
  const int q = whole_pages(n, p, rest);
  return q + (rest > 0);
}

// A batch's scans, in LDS.
struct Batch {
  int64_t* len;    // [B] held tokens
  int32_t* cu;     // [B + 1] rows before sequence b
  int32_t* rank;   // [B + 1] pages handed out (or given back) before sequence b
  int32_t* slot;   // [B] -1: not a slot
  int32_t* page;   // [B] whole pages held (release: pages kept)
  uint32_t* rest;  // [B] tokens held past them
  int32_t* hash;   // [hash_size] the slots that get (or give back) pages
};

__device__ __forceinline__ Batch batch_in(char* lds, int B) {
  Batch s;
  s.len = reinterpret_cast<int64_t*>(lds);
  s.cu = reinterpret_cast<int32_t*>(s.len + B);
  s.rank = s.cu + B + 1;
  s.slot = s.rank + B + 1;
  s.page = s.slot + B;
  s.rest = reinterpret_cast<uint32_t*>(s.page + B);
  s.hash = reinterpret_cast<int32_t*>(s.rest + B);
  return s;
}
static inline size_t batch_bytes(int B, int hash_size) {
  return (size_t)B * 8 + (size_t)(B + 1) * 8 + (size_t)B * 12 + (size_t)hash_size * 4;
}

// Exclusive prefix sums of two values over the workgroup's threads, and their totals,
// saturated at the caps (< 2^25: a wave's sum fits 31 bits).
template <int kThreads>
__device__ __forceinline__ void block_exclusive(int& a, int& b, int cap_a, int cap_b, int (*sm)[2], int& total_a,
                                                int& total_b) {
  a = min(a, cap_a);
  b = min(b, cap_b);
  const int in_a = wave_inclusive_sum(a), in_b = wave_inclusive_sum(b);
  const int wave = threadIdx.x / kWave;
  __syncthreads();  // (a former call's words are read)
  if (threadIdx.x % kWave == kWave - 1) {
    sm[wave][0] = min(in_a, cap_a);
    sm[wave][1] = min(in_b, cap_b);
  }
  __syncthreads();
  constexpr int kWaves = kThreads / kWave;
  const int from = threadIdx.x % kWaves;  // (of 16 waves at most: the caps' sums fit 31 bits)
  const int before_a = min(waves_before<kWaves>(sm[from][0], wave, total_a), cap_a);
  const int before_b = min(waves_before<kWaves>(sm[from][1], wave, total_b), cap_b);
  total_a = min(total_a, cap_a);
  total_b = min(total_b, cap_b);
  a = min(before_a + min(in_a - a, cap_a), cap_a);
  b = min(before_b + min(in_b - b, cap_b), cap_b);
}

// Adds slot to the set; false if it was there.  At most half of the set is filled.
__device__ __forceinline__ bool add_slot(int32_t* hash, int size, int slot) {
  uint32_t h = ((uint32_t)slot * 2654435761u) >> 8 & (uint32_t)(size - 1);
  while (true) {
    const int old = atomicCAS(&hash[h], -1, slot);
    if (old == -1) return true;
    if (old == slot) return false;
    h = (h + 1) & (uint32_t)(size - 1);
  }
}

// The sequence that element j of a scan belongs to: the last b with scan[b] <= j.
__device__ __forceinline__ int find(const int32_t* scan, int B, int j) {
  int lo = 0, hi = B;  // scan[lo] <= j < scan[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (scan[mid] <= j)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// True in the last of the grid's workgroups to come here, which finds all others past their reads.
__device__ __forceinline__ bool last_of_grid(int64_t* word, int* flag) {
  if (gridDim.x == 1) return true;
  __syncthreads();
  if (threadIdx.x == 0)
    *flag = __hip_atomic_fetch_add(word, (int64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
            (int64_t)gridDim.x - 1;
  __syncthreads();
  return *flag != 0;
}

template <bool kReserve, int kThreads>
__global__ __launch_bounds__(kThreads) void step_maps_kernel(MapParams p) {
  extern __shared__ __align__(8) char lds[];
  __shared__ int sm[kThreads / kWave][2], flag, bad;
  const Batch s = batch_in(lds, p.B);
  const int tid = threadIdx.x, B = p.B, T = (int)p.T;
  const uint32_t P = (uint32_t)p.page_size;
  const int each = (B + kThreads - 1) / kThreads, b0 = min(tid * each, B), b1 = min(b0 + each, B);
  const int64_t capacity = p.bt_width * P;

  int64_t avail = 0;
  if constexpr (kReserve) {
    avail = p.free_list[0];
    for (int i = tid; i < p.hash_size; i += kThreads) s.hash[i] = -1;
    if (tid == 0) bad = 0;
  }
  // New pages of a sequence whose n tokens are all mapped; 0 for the padding rows' slot and where they do not fit.
  const auto more_pages = [&](int b, int n) {
    const int64_t len = s.len[b];
    if (s.slot[b] <= 0 || n == 0 || len < 0 || len > capacity - n) return 0;  // (len: any word)
    const uint32_t rest = s.rest[b];
    return (int)((rest + (uint32_t)n + P - 1) / P) - (rest > 0);
  };
  int rows = 0, need = 0, mistakes = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const int64_t slot = p.slot_ids[b], n = p.counts[b];
    const bool ok = slot >= 0 && slot < p.n_slots;
    const int64_t len = ok ? p.lens[slot] : 0;
    if (!ok) mistakes |= CIE_ERRBIT_PAGE;
    if (n < 0 || len < 0) mistakes |= CIE_ERRBIT_LEN;
    s.slot[b] = ok ? (int)slot : -1;
    s.len[b] = len;
    uint32_t rest;
    s.page[b] = whole_pages(min(max(len, (int64_t)0), capacity), p, rest);
    s.rest[b] = rest;
    s.cu[b] = rows;  // (within the thread, completed below)
    s.rank[b] = need;
    const int take = (int)min(max(n, (int64_t)0), p.T);
    rows = min(rows + take, T + 1);
    if constexpr (kReserve) need += more_pages(b, take);
  }
  int total, need_total;
  int first_row = rows, first_page = need;
  block_exclusive<kThreads>(first_row, first_page, T + 1, 1 << 25, sm, total, need_total);
  for (int b = b0; b < b1; ++b) {
    s.cu[b] = min(s.cu[b] + first_row, T);
    s.rank[b] += first_page;
  }
  const bool cut = total > T;
  if (cut) mistakes |= CIE_ERRBIT_LEN;
  total = min(total, T);
  if (tid == 0) {
    s.cu[B] = total;
    s.rank[B] = need_total;
  }
  __syncthreads();

  bool granted = false;
  if constexpr (kReserve) {
    if (cut) {  // pages for the rows that are mapped only
      need = 0;
      for (int b = b0; b < b1; ++b) {
        s.rank[b] = need;
        need += more_pages(b, s.cu[b + 1] - s.cu[b]);
      }
      int none = 0, no_total;
      block_exclusive<kThreads>(need, none, 1 << 25, 1, sm, need_total, no_total);
      for (int b = b0; b < b1; ++b) s.rank[b] += need;
      if (tid == 0) s.rank[B] = need_total;
    }
    for (int b = b0; b < b1; ++b) {
      const int n = s.cu[b + 1] - s.cu[b];
      const int64_t len = s.len[b];
      if (s.slot[b] <= 0 || n == 0 || len < 0) continue;
      if (len > capacity - n)
        mistakes |= CIE_ERRBIT_LEN;
      else if (!add_slot(s.hash, p.hash_size, s.slot[b]))
        bad = 1;
    }
    __syncthreads();
    granted = !bad && need_total <= avail && avail <= p.n_pages;
    if (!granted) mistakes |= CIE_ERRBIT_FREE;
    if (granted) {
#pragma unroll 1
      for (int j = blockIdx.x * kThreads + tid; j < need_total; j += gridDim.x * kThreads) {
        const int b = find(s.rank, B, j);
        int64_t id = p.free_list[2 + avail - 1 - j];
        if (id <= 0 || id >= p.n_pages) {
          mistakes |= CIE_ERRBIT_PAGE;
          id = 0;
        }
        p.block_table[(int64_t)s.slot[b] * p.bt_stride + s.page[b] + (s.rest[b] > 0) + (j - s.rank[b])] = id;
      }
    }
  }

#pragma unroll 1
  for (int t = blockIdx.x * kThreads + tid; t < T; t += gridDim.x * kThreads) {
    int64_t slot = 0, pos = 0, page = 0, off = 0;
    if (t < total) {
      const int b = find(s.cu, B, t);
      if (s.slot[b] >= 0) {
        slot = s.slot[b];
        const int64_t len = s.len[b];
        pos = (int64_t)((uint64_t)len + (uint64_t)(t - s.cu[b]));  // (past 2^63: negative)
        if (pos < 0 || pos >= capacity) {
          mistakes |= CIE_ERRBIT_LEN;
        } else {
          // (past the whole pages held, or from a negative length on: below 2^32)
          const uint32_t past = len < 0 ? (uint32_t)pos : s.rest[b] + (uint32_t)(t - s.cu[b]), more = past / P;
          const int64_t at = s.page[b] + (int64_t)more;
          off = past - more * P;
          bool fresh = false;
          if constexpr (kReserve) {
            const int have = s.page[b] + (s.rest[b] > 0);
            fresh = slot > 0 && at >= have;
            if (fresh && granted && s.rank[b + 1] > s.rank[b]) {
              page = p.free_list[2 + avail - 1 - (s.rank[b] + (at - have))];
              if (page <= 0 || page >= p.n_pages) page = 0;
            }
          }
          if (!fresh) page = p.block_table[slot * p.bt_stride + at];
        }
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.pages[t] = page;
    p.offsets[t] = off;
  }
  if (blockIdx.x == 0)
    for (int b = tid; b <= B; b += kThreads) p.cu[b] = s.cu[b];
  if (mistakes) set_err(p.err, mistakes);
  if constexpr (kReserve) {
    if (last_of_grid(p.free_list + 1, &flag) && tid == 0) {
      if (granted) p.free_list[0] = avail - need_total;
      p.free_list[1] = 0;
    }
  }
}

constexpr int64_t kNoPage = -1;  // on the stack, until the gaps are closed

template <int kThreads>
__global__ __launch_bounds__(kThreads) void release_pages_kernel(MapParams p) {
  extern __shared__ __align__(8) char lds[];
  __shared__ int sm[kThreads / kWave][2], flag, bad, gaps;
  const Batch s = batch_in(lds, p.B);
  const int tid = threadIdx.x, B = p.B;
  const int each = (B + kThreads - 1) / kThreads, b0 = min(tid * each, B), b1 = min(b0 + each, B);
  const int64_t capacity = p.bt_width * p.page_size, avail = p.free_list[0];

  for (int i = tid; i < p.hash_size; i += kThreads) s.hash[i] = -1;
  if (tid == 0) bad = gaps = 0;
  __syncthreads();
  int gone = 0, mistakes = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const int64_t slot = p.slot_ids[b];
    const int64_t keep = p.counts ? p.counts[b] : 0;
    int64_t held = p.held ? p.held[b] : 0;
    s.rank[b] = gone;
    s.slot[b] = -1;
    if (slot == 0) continue;  // the padding rows' slot holds no pages
    if (slot < 0 || slot >= p.n_slots) {
      mistakes |= CIE_ERRBIT_PAGE;
      continue;
    }
    const int64_t len = p.lens[slot];
    if (!p.held) held = len;
    if (held < len || held < 0 || held > capacity || keep < 0 || keep > held) {
      mistakes |= CIE_ERRBIT_LEN;
      continue;
    }
    if (!add_slot(s.hash, p.hash_size, (int)slot)) bad = 1;
    s.slot[b] = (int)slot;
    s.len[b] = keep;
    s.page[b] = pages_of(keep, p);
    gone = (int)min((int64_t)gone + pages_of(held, p) - s.page[b], kMapMaxPages + 1);
  }
  int total, none = 0, no_total;
  int before = gone;
  block_exclusive<kThreads>(before, none, (int)kMapMaxPages + 1, 1, sm, total, no_total);
  for (int b = b0; b < b1; ++b) s.rank[b] = min(s.rank[b] + before, (int)kMapMaxPages + 1);
  if (tid == 0) s.rank[B] = total;
  __syncthreads();
  // (a list of all pages but page 0 is full)
  const bool taken = !bad && avail >= 0 && avail + total < p.n_pages;
  if (!taken) mistakes |= CIE_ERRBIT_FREE;
  int64_t* const stack = p.free_list + 2 + avail;
  if (taken) {
#pragma unroll 1
    for (int j = blockIdx.x * kThreads + tid; j < total; j += gridDim.x * kThreads) {
      const int b = find(s.rank, B, j);
      int64_t* const entry = p.block_table + (int64_t)s.slot[b] * p.bt_stride + s.page[b] + (j - s.rank[b]);
      int64_t id = *entry;
      if (id <= 0 || id >= p.n_pages) {
        mistakes |= CIE_ERRBIT_PAGE;
        if (id == 0) gaps = 1;
        id = id == 0 ? kNoPage : 0;
      }
      *entry = 0;
      // (agent scope: another CU's workgroup may close the gaps)
      __hip_atomic_store(&stack[total - 1 - j], id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (mistakes) set_err(p.err, mistakes);
  // The last workgroup to arrive, and whether any met an entry without a page (above the arrivals' 32 bits).
  __syncthreads();
  bool any_gaps = gaps != 0;
  if (gridDim.x > 1) {
    wait_stores();
    __syncthreads();
    if (tid == 0) {
      const int64_t old = __hip_atomic_fetch_add(p.free_list + 1, (int64_t)1 + ((int64_t)any_gaps << 32),
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      flag = (int)(old & 0xffffffff) == (int)gridDim.x - 1 ? 1 + (any_gaps || old >> 32 != 0) : 0;
    }
    __syncthreads();
    if (flag == 0) return;
    any_gaps = flag == 2;
  }
  if (taken) {
    for (int b = tid; b < B; b += kThreads)
      if (s.slot[b] > 0) p.lens[s.slot[b]] = s.len[b];
    int given = total;
    if (any_gaps) {
      wait_stores();
      __syncthreads();
      given = 0;
      for (int k0 = 0; k0 < total; k0 += kThreads) {  // (a word's new place is never behind its old one)
        const int k = k0 + tid;
        const int64_t id =
            k < total ? __hip_atomic_load(&stack[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : kNoPage;
        int place = id != kNoPage, none = 0, n, no_n;
        block_exclusive<kThreads>(place, none, kThreads, 1, sm, n, no_n);
        if (id != kNoPage) stack[given + place] = id;
        given += n;
      }
      for (int k = given + tid; k < total; k += kThreads) stack[k] = 0;
    }
    if (tid == 0) p.free_list[0] = avail + given;
  }
  if (tid == 0) p.free_list[1] = 0;
}

static int hash_size_of(int64_t B) {
  int n = 2;
  while (n < 2 * B) n *= 2;
  return n;
}

}  // namespace cie

using namespace cie;

extern "C" int cie_step_maps(int64_t* cu_seqlens, int64_t* slots, int64_t* positions, int64_t* pages,
                             int64_t* offsets, const int64_t* slot_ids, const int64_t* new_tokens,
                             const int64_t* lens, int64_t* block_table, int64_t* free_list, int64_t B, int64_t T,
                             int64_t page_size, int64_t n_pages, int64_t bt_stride, int64_t bt_width,
                             int64_t n_slots, int32_t* err, void* stream) {
  if (B < 0 || T < 0 || page_size <= 0 || bt_width <= 0 || bt_stride < bt_width || n_slots <= 0 ||
      (free_list && n_pages <= 0))
    return CIE_EINVAL;
  if (B > kMapMaxSeqs || T > kMapMaxRows || page_size > kMapMaxPage || bt_width > kMapMaxPages ||
      n_slots > 0x7fffffff || (free_list && n_pages > kMapMaxPages))
    return CIE_EUNSUPPORTED;
  if (!cu_seqlens || (T > 0 && (!slots || !positions || !pages || !offsets)) ||
      (B > 0 && (!slot_ids || !new_tokens || !lens || !block_table)))
    return CIE_EINVAL;
  MapParams p{};
  p.cu = cu_seqlens;
  p.slots = slots;
  p.positions = positions;
  p.pages = pages;
  p.offsets = offsets;
  p.slot_ids = slot_ids;
  p.counts = new_tokens;
  p.lens = const_cast<int64_t*>(lens);
  p.block_table = block_table;
  p.free_list = free_list;
  p.bt_stride = bt_stride;
  p.bt_width = bt_width;
  p.n_slots = n_slots;
  p.n_pages = n_pages;
  p.T = T;
  p.B = (int32_t)B;
  p.page_size = (int32_t)page_size;
  p.hash_size = free_list ? hash_size_of(B) : 0;
  p.err = err;
  p.per_page = 1.0 / (double)page_size;
  const size_t lds = batch_bytes((int)B, p.hash_size);
  const auto grid = [&](int64_t rows) {  // of a workgroup's rows; to one workgroup a CU, further rows are a loop
    const int64_t blocks = (T + rows - 1) / rows;
    return dim3((unsigned)(blocks < 1 ? 1 : blocks < 256 ? blocks : 256));
  };
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Scans want a sequence a thread; four times the threads start 0.5 us later.  Where pages are handed out, further workgroups
  // cost an arrival (1 us): two rows a thread, so that most steps are one workgroup.
  if (free_list && B <= 256 && T <= 256)
    hipLaunchKernelGGL((step_maps_kernel<true, 256>), dim3(1), dim3(256), lds, st, p);
  else if (free_list)
    hipLaunchKernelGGL((step_maps_kernel<true, 1024>), grid(2048), dim3(1024), lds, st, p);
  else if (B > 256)
    hipLaunchKernelGGL((step_maps_kernel<false, 1024>), grid(1024), dim3(1024), lds, st, p);
  else
    hipLaunchKernelGGL((step_maps_kernel<false, 256>), grid(256), dim3(256), lds, st, p);
  return (int)hipGetLastError();
}

extern "C" int cie_release_pages(int64_t* free_list, const int64_t* slot_ids, int64_t* lens, int64_t* block_table,
                                 const int64_t* keep, const int64_t* held, int64_t B, int64_t page_size,
                                 int64_t n_pages, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                                 int32_t* err, void* stream) {
  if (B < 0 || page_size <= 0 || n_pages <= 0 || bt_width <= 0 || bt_stride < bt_width || n_slots <= 0)
    return CIE_EINVAL;
  if (B > kMapMaxSeqs || page_size > kMapMaxPage || bt_width > kMapMaxPages || n_slots > 0x7fffffff ||
      n_pages > kMapMaxPages)
    return CIE_EUNSUPPORTED;
  if (B == 0) return CIE_OK;
  if (!free_list || !slot_ids || !lens || !block_table) return CIE_EINVAL;
  MapParams p{};
  p.slot_ids = slot_ids;
  p.counts = keep;
  p.held = held;
  p.lens = lens;
  p.block_table = block_table;
  p.free_list = free_list;
  p.bt_stride = bt_stride;
  p.bt_width = bt_width;
  p.n_slots = n_slots;
  p.n_pages = n_pages;
  p.B = (int32_t)B;
  p.page_size = (int32_t)page_size;
  p.hash_size = hash_size_of(B);
  p.err = err;
  p.per_page = 1.0 / (double)page_size;
  // The pages given back are known on the device only: as many workgroups as would
  // empty the pool in 32 rounds (an arrival costs 1.5 us, a round 0.5).
  const int64_t blocks = n_pages / 32768;
  const size_t lds = batch_bytes((int)B, p.hash_size);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (B <= 256 && n_pages <= 8192)
    hipLaunchKernelGGL(release_pages_kernel<256>, dim3(1), dim3(256), lds, st, p);
  else
    hipLaunchKernelGGL(release_pages_kernel<1024>, dim3((unsigned)(blocks < 1 ? 1 : blocks < 32 ? blocks : 32)),
                       dim3(1024), lds, st, p);
  return (int)hipGetLastError();
}
