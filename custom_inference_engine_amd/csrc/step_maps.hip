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
// what a call was given leaves the list as it was.
//
// Both are bound by latency, not by bytes: 40 bytes a row are written once.  So
// one launch does it all.  Every workgroup reads the B sequences and scans them
// for itself (two dependent round trips: slots and new lengths, then the held
// lengths), and no workgroup waits for what another writes: a row on a new page
// reads the page's id from the stack, at the place that the scan gives it, not
// from the table.  Words that other workgroups still read (the count, and a
// release's lengths) are changed by the last workgroup to arrive.
// Times of one call, replayed from a graph: one row 2.9 us, 32 sequences and
// 1,056 rows 3.9 us, 496 sequences and 16,480 rows with 1,480 new pages 8 us.
#include "cie_common.h"

namespace cie {

constexpr int kMapThreads = 256;
constexpr int kMapMaxSeqs = 2048;          // (scans and hash table of a batch: 56 KB of LDS)
constexpr int64_t kMapMaxRows = 1 << 24;   // sums over a batch stay below 2^31
constexpr int64_t kMapMaxPages = 1 << 24;

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
  int32_t B, page_size, hash_size;
  int32_t* err;
};

// a / d for 0 <= a, 0 < d < 2^31.
__device__ __forceinline__ int64_t div_by(int64_t a, int32_t d) {
  return (uint64_t)a >> 32 ? a / d : (int64_t)((uint32_t)a / (uint32_t)d);
}

// A batch's scans, in LDS.
struct Batch {
  int32_t* cu;     // [B + 1] rows before sequence b
  int32_t* rank;   // [B + 1] pages handed out (or given back) before sequence b
  int32_t* slot;   // [B] -1: not a slot
  int64_t* len;    // [B] held tokens; release: the first page given back
  int32_t* hash;   // [hash_size] the slots that get (or give back) pages
};

__device__ __forceinline__ Batch batch_in(char* lds, int B) {
  Batch s;
  s.len = reinterpret_cast<int64_t*>(lds);
  s.cu = reinterpret_cast<int32_t*>(s.len + B);
  s.rank = s.cu + B + 1;
  s.slot = s.rank + B + 1;
  s.hash = s.slot + B;
  return s;
}
static inline size_t batch_bytes(int B, int hash_size) {
  return (size_t)B * 8 + (size_t)(B + 1) * 8 + (size_t)B * 4 + (size_t)hash_size * 4;
}

// Exclusive prefix sum over the workgroup's threads, saturated at cap (< 2^25:
// a wave's sum fits 31 bits), and the total.  sm: a word a wave.
__device__ __forceinline__ int block_exclusive(int v, int cap, int* sm, int& total) {
  v = min(v, cap);
  const int incl = wave_inclusive_sum(v);
  const int wave = threadIdx.x / kWave;
  __syncthreads();  // (a former call's words are read)
  if (threadIdx.x % kWave == kWave - 1) sm[wave] = min(incl, cap);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kMapThreads / kWave; ++w) {
    if (w == wave) before = total;
    total = min(total + sm[w], cap);
  }
  return min(before + min(incl - v, cap), cap);
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

template <bool kReserve>
__global__ __launch_bounds__(kMapThreads) void step_maps_kernel(MapParams p) {
  extern __shared__ __align__(8) char lds[];
  __shared__ int sm[kMapThreads / kWave], flag, bad;
  const Batch s = batch_in(lds, p.B);
  const int tid = threadIdx.x, B = p.B, P = p.page_size;
  const int each = (B + kMapThreads - 1) / kMapThreads, b0 = min(tid * each, B), b1 = min(b0 + each, B);
  const int64_t capacity = p.bt_width * P;
  const int T = (int)p.T;

  int64_t avail = 0;
  if constexpr (kReserve) {
    avail = p.free_list[0];
    for (int i = tid; i < p.hash_size; i += kMapThreads) s.hash[i] = -1;
    if (tid == 0) bad = 0;
  }
  int rows = 0, mistakes = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t slot = p.slot_ids[b], n = p.counts[b];
    const bool ok = slot >= 0 && slot < p.n_slots;
    const int64_t len = ok ? p.lens[slot] : 0;
    if (!ok) mistakes |= CIE_ERRBIT_PAGE;
    if (n < 0 || len < 0) mistakes |= CIE_ERRBIT_LEN;
    s.slot[b] = ok ? (int)slot : -1;
    s.len[b] = len;
    s.cu[b] = rows;  // (within the thread, completed below)
    rows = min(rows + (int)min(max(n, (int64_t)0), p.T), T + 1);
  }
  int total;
  const int before = block_exclusive(rows, T + 1, sm, total);
  for (int b = b0; b < b1; ++b) s.cu[b] = min(s.cu[b] + before, T);
  if (total > T) mistakes |= CIE_ERRBIT_LEN;
  total = min(total, T);
  if (tid == 0) s.cu[B] = total;
  __syncthreads();

  int need_total = 0;
  bool granted = false;
  if constexpr (kReserve) {
    int need = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = s.cu[b + 1] - s.cu[b], slot = s.slot[b];
      const int64_t len = s.len[b];
      s.rank[b] = need;
      if (slot <= 0 || n == 0 || len < 0) continue;  // (slot 0 is the padding rows')
      if (len + n > capacity) {
        mistakes |= CIE_ERRBIT_LEN;
        continue;
      }
      const int more = (int)(div_by(len + n + P - 1, P) - div_by(len + P - 1, P));
      if (!add_slot(s.hash, p.hash_size, slot)) bad = 1;
      need += more;
    }
    const int first = block_exclusive(need, 1 << 25, sm, need_total);
    for (int b = b0; b < b1; ++b) s.rank[b] += first;
    if (tid == 0) s.rank[B] = need_total;
    __syncthreads();
    granted = !bad && need_total <= avail && avail <= p.n_pages;
    if (!granted) mistakes |= CIE_ERRBIT_FREE;
    if (granted) {
      for (int j = blockIdx.x * kMapThreads + tid; j < need_total; j += gridDim.x * kMapThreads) {
        const int b = find(s.rank, B, j);
        int64_t id = p.free_list[2 + avail - 1 - j];
        if (id <= 0 || id >= p.n_pages) {
          mistakes |= CIE_ERRBIT_PAGE;
          id = 0;
        }
        p.block_table[(int64_t)s.slot[b] * p.bt_stride + div_by(s.len[b] + P - 1, P) + (j - s.rank[b])] = id;
      }
    }
  }

  for (int t = blockIdx.x * kMapThreads + tid; t < T; t += gridDim.x * kMapThreads) {
    int64_t slot = 0, pos = 0, page = 0, off = 0;
    if (t < total) {
      const int b = find(s.cu, B, t);
      if (s.slot[b] >= 0) {
        slot = s.slot[b];
        const int64_t len = s.len[b];
        pos = len + (t - s.cu[b]);
        if (pos < 0 || pos >= capacity) {
          mistakes |= CIE_ERRBIT_LEN;
        } else {
          const int64_t at = div_by(pos, P);
          off = pos - at * P;
          bool fresh = false;
          if constexpr (kReserve) {
            const int64_t have = div_by(max(len, (int64_t)0) + P - 1, P);
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
    for (int b = tid; b <= B; b += kMapThreads) p.cu[b] = s.cu[b];
  if (mistakes) set_err(p.err, mistakes);
  if constexpr (kReserve) {
    if (last_of_grid(p.free_list + 1, &flag) && tid == 0) {
      if (granted) p.free_list[0] = avail - need_total;
      p.free_list[1] = 0;
    }
  }
}

__global__ __launch_bounds__(kMapThreads) void release_pages_kernel(MapParams p) {
  extern __shared__ __align__(8) char lds[];
  __shared__ int sm[kMapThreads / kWave], flag, bad;
  const Batch s = batch_in(lds, p.B);
  const int tid = threadIdx.x, B = p.B, P = p.page_size;
  const int each = (B + kMapThreads - 1) / kMapThreads, b0 = min(tid * each, B), b1 = min(b0 + each, B);
  const int64_t capacity = p.bt_width * P, avail = p.free_list[0];

  for (int i = tid; i < p.hash_size; i += kMapThreads) s.hash[i] = -1;
  if (tid == 0) bad = 0;
  __syncthreads();
  int gone = 0, mistakes = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t slot = p.slot_ids[b];
    s.rank[b] = gone;
    s.slot[b] = -1;
    if (slot == 0) continue;  // the padding rows' slot holds no pages
    if (slot < 0 || slot >= p.n_slots) {
      mistakes |= CIE_ERRBIT_PAGE;
      continue;
    }
    const int64_t len = p.lens[slot];
    const int64_t held = p.held ? p.held[b] : len;
    const int64_t keep = p.counts ? p.counts[b] : 0;
    if (held < len || held < 0 || held > capacity || keep < 0 || keep > held) {
      mistakes |= CIE_ERRBIT_LEN;
      continue;
    }
    if (!add_slot(s.hash, p.hash_size, (int)slot)) bad = 1;
    s.slot[b] = (int)slot;
    s.len[b] = div_by(keep + P - 1, P);
    gone = (int)min(gone + div_by(held + P - 1, P) - s.len[b], kMapMaxPages + 1);
  }
  int total;
  const int before = block_exclusive(gone, (int)kMapMaxPages + 1, sm, total);
  for (int b = b0; b < b1; ++b) s.rank[b] = min(s.rank[b] + before, (int)kMapMaxPages + 1);
  if (tid == 0) s.rank[B] = total;
  __syncthreads();
  // (a list of all pages but page 0 is full)
  const bool taken = !bad && avail >= 0 && avail + total < p.n_pages;
  if (!taken) mistakes |= CIE_ERRBIT_FREE;
  if (taken) {
    for (int j = blockIdx.x * kMapThreads + tid; j < total; j += gridDim.x * kMapThreads) {
      const int b = find(s.rank, B, j);
      int64_t* const entry = p.block_table + (int64_t)s.slot[b] * p.bt_stride + s.len[b] + (j - s.rank[b]);
      int64_t id = *entry;
      if (id <= 0 || id >= p.n_pages) {
        mistakes |= CIE_ERRBIT_PAGE;
        id = 0;
      }
      *entry = 0;
      p.free_list[2 + avail + total - 1 - j] = id;
    }
  }
  if (mistakes) set_err(p.err, mistakes);
  if (last_of_grid(p.free_list + 1, &flag)) {
    if (taken) {
      for (int b = tid; b < B; b += kMapThreads)
        if (s.slot[b] > 0) p.lens[s.slot[b]] = p.counts ? p.counts[b] : 0;
      if (tid == 0) p.free_list[0] = avail + total;
    }
    if (tid == 0) p.free_list[1] = 0;
  }
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
  if (B > kMapMaxSeqs || T > kMapMaxRows || page_size > 0x7fffffff || bt_width > kMapMaxPages ||
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
  // A row a thread, to one workgroup a CU: further rows are a loop.
  const int64_t blocks = (T + kMapThreads - 1) / kMapThreads;
  const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks < 256 ? blocks : 256));
  const size_t lds = batch_bytes((int)B, p.hash_size);
  if (free_list)
    hipLaunchKernelGGL(step_maps_kernel<true>, grid, dim3(kMapThreads), lds, static_cast<hipStream_t>(stream), p);
  else
    hipLaunchKernelGGL(step_maps_kernel<false>, grid, dim3(kMapThreads), lds, static_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}

extern "C" int cie_release_pages(int64_t* free_list, const int64_t* slot_ids, int64_t* lens, int64_t* block_table,
                                 const int64_t* keep, const int64_t* held, int64_t B, int64_t page_size,
                                 int64_t n_pages, int64_t bt_stride, int64_t bt_width, int64_t n_slots,
                                 int32_t* err, void* stream) {
  if (B < 0 || page_size <= 0 || n_pages <= 0 || bt_width <= 0 || bt_stride < bt_width || n_slots <= 0)
    return CIE_EINVAL;
  if (B > kMapMaxSeqs || page_size > 0x7fffffff || bt_width > kMapMaxPages || n_slots > 0x7fffffff ||
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
  // Four sequences' pages a wave or so; the page counts are known on the device only.
  const int64_t blocks = (B + 15) / 16;
  hipLaunchKernelGGL(release_pages_kernel, dim3((unsigned)(blocks < 32 ? blocks : 32)), dim3(kMapThreads),
                     batch_bytes((int)B, p.hash_size), static_cast<hipStream_t>(stream), p);
  return (int)hipGetLastError();
}
