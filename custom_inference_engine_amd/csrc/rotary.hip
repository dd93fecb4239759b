// Rows turned by their positions.
//
// Pair i of a head's first `rot` dims, (x, y), at position p turns by the angle
// p * f_i:  (x, y) -> s * (x cos - y sin, y cos + x sin).  "Half" layout pairs dim
// i with i + rot / 2, "interleaved" 2i with 2i + 1; the dims from rot on are
// copied.  The f_i are radians a position in fp64, so any base and any stretching
// for long contexts is a table of them.
//
// Angles: p * f_i in fp64, in turns, less the nearest whole turn (exact): at position
// 2^31 the angle is off by 2^-20 rad, where an fp32 product is off by whole turns.  cos
// and sin of what is left are taken in fp32 for 16-bit rows, whose rounding hides the 2^-22
// that this costs, and in fp64 for fp32 rows, rounded once.  Products and sums are fp32.
//
// Bound by memory: each row is read and written once.  A thread takes 16 bytes of
// each half of a pair's dims (two vectors of V values) and computes their V
// angles once for several heads of the token, whose loads it issues together.
// Few rows get a head a thread; many get fewer threads, down to a few rounds of
// the chip, so that the angles (some 60 instructions a pair) are spread over
// more heads.  8,192 rows of 48 heads of 128 into the pools: 40.7 us, 5.0 TB/s, what a copy
// reaches; 8,192 rows of 40 heads of 128 in fp32 61.4 us, 5.5 TB/s (their tables 3.9 us, with cos
// and sin in fp32 3.7).  Rows at any address and odd widths take the same vectors, unaligned;
// only heads that turn or copy less than a vector go value by value.
#include "cie_common.h"

namespace cie {

typedef __bf16 bf16;

template <class E>
struct VecOf;
template <>
struct VecOf<f16> {
  static constexpr int kWide = 8;
};
template <>
struct VecOf<bf16> {
  static constexpr int kWide = 8;
};
template <>
struct VecOf<float> {
  static constexpr int kWide = 4;
};

struct RotaryParams {
  void* q_out;         // (T, H_q, D) dense
  void* k_out;         // (T, H_kv, D) dense, or the K pool
  void* v_out;         // the V pool
  const void* q;
  const void* k;
  const void* v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const int64_t* positions;
  const double* freqs;
  const int64_t* pages;    // pools only
  const int64_t* offsets;
  int64_t pool_page_stride, pool_head_stride, n_pages;
  int64_t T;
  double scale;
  int32_t H_q, H_kv, D, rot, units, head_groups, page_size;
  int32_t* err;
};

// cos and sin of position p at V pairs from pair i on, times scale, for rows of E.
template <class E, int V>
__device__ __forceinline__ void angles(double p, const double* f, double scale, float* c, float* s) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const double turns = p * f[j] * 0.15915494309189533577;  // 1 / 2 pi
    const double left = turns - __builtin_rint(turns);
    if constexpr (sizeof(E) == 4) {
      double sin, cos;
      sincospi(2.0 * left, &sin, &cos);
      c[j] = (float)(cos * scale);
      s[j] = (float)(sin * scale);
    } else {
      sincospif(2.0f * (float)left, &s[j], &c[j]);
      c[j] *= (float)scale;
      s[j] *= (float)scale;
    }
  }
}

// V values side by side, at a multiple of their size or (global memory may be read so) of one's.
template <class E, int V, bool kAligned>
struct Pack {
  E v[V] __attribute__((aligned(sizeof(E) * (kAligned ? V : 1))));
};

// Two vectors of a head's dims (V pairs), turned.
template <class E, int V, bool kInterleaved, bool kAligned>
__device__ __forceinline__ void turn(Pack<E, V, kAligned>& lo, Pack<E, V, kAligned>& hi, const float* c, const float* s) {
  float x[2 * V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    x[j] = (float)lo.v[j];
    x[V + j] = (float)hi.v[j];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i0 = kInterleaved ? 2 * j : j, i1 = kInterleaved ? 2 * j + 1 : V + j;
    const float a = x[i0], b = x[i1];
    x[i0] = __builtin_fmaf(a, c[j], -(b * s[j]));
    x[i1] = __builtin_fmaf(b, c[j], a * s[j]);
    asm volatile("" : "+v"(x[i0]), "+v"(x[i1]));  // (to fp32 first, in every variant: no v_fma_mixlo_f16)
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    lo.v[j] = (E)x[j];
    hi.v[j] = (E)x[V + j];
  }
}

constexpr int kRotHeads = 4;  // heads whose loads a thread has in flight

template <class E, int V, bool kInterleaved, bool kPools, bool kAligned>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  typedef Pack<E, V, kAligned> vec;
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;  // (the host keeps the grid under 2^32 threads)
  const uint32_t rest = gid / (uint32_t)p.units;
  const int u = (int)(gid - rest * (uint32_t)p.units);
  const int64_t t = rest / (uint32_t)p.head_groups;
  const int group = (int)(rest - (uint32_t)t * (uint32_t)p.head_groups);
  if (t >= p.T) return;
  // Units of V pairs turn, then units of 2 V dims copy.  Where they do not come out even
  // the last unit of either kind lies back over the one before it: both write the same.
  const int half = p.rot / 2, turning = (half + V - 1) / V;
  const bool turns = u < turning;
  int d0, d1, pair = 0;
  if (!turns) {
    d0 = p.rot + min(2 * V * (u - turning), max(p.D - p.rot - 2 * V, 0));
    d1 = min(d0 + V, p.D - V);
  } else {
    pair = min(V * u, half - V);
    d0 = kInterleaved ? 2 * pair : pair;
    d1 = kInterleaved ? d0 + V : d0 + half;
  }
  int64_t page = 0, off = 0;
  bool kept = true;
  if constexpr (kPools) {
    page = p.pages[t];
    off = p.offsets[t];
  }
  float c[V], s[V];
  // (Before the rows' loads: behind them their registers leave three waves a SIMD, and
  // 2,048 rows of 40 heads take 11.7 us, not 9.6.)
  if (turns) angles<E, V>((double)p.positions[t], p.freqs + pair, p.scale, c, s);
  if constexpr (kPools) {
    kept = false;
    if (off < 0 || off >= p.page_size)
      set_err(p.err, CIE_ERRBIT_OFFSET);
    else if (page < 0 || page >= p.n_pages)
      set_err(p.err, CIE_ERRBIT_PAGE);
    else
      kept = true;
  }

  // Heads of q, of k and (into pools) of v, which is copied.
  const int keys = p.H_q, values = p.H_q + p.H_kv, heads = kPools ? values + p.H_kv : values;
  const E* const q = static_cast<const E*>(p.q) + t * p.q_tok;
  const E* const k = static_cast<const E*>(p.k) + t * p.k_tok;
  const E* const v = static_cast<const E*>(p.v) + t * p.v_tok;
  const int64_t at = page * p.pool_page_stride + off * p.D;
  for (int h0 = group; h0 < heads; h0 += kRotHeads * p.head_groups) {
    vec x[kRotHeads][2];
#pragma unroll
    for (int i = 0; i < kRotHeads; ++i) {
      const int h = h0 + i * p.head_groups;
      if (h >= heads) continue;
      const E* const row = h < keys                ? q + h * p.q_head
                           : !kPools || h < values ? k + (h - keys) * p.k_head
                                                   : v + (h - values) * p.v_head;
      x[i][0] = *reinterpret_cast<const vec*>(row + d0);
      x[i][1] = *reinterpret_cast<const vec*>(row + d1);
    }
#pragma unroll
    for (int i = 0; i < kRotHeads; ++i) {
      const int h = h0 + i * p.head_groups;
      if (h >= heads) continue;
      if (turns && (!kPools || h < values)) turn<E, V, kInterleaved, kAligned>(x[i][0], x[i][1], c, s);
      E* to;
      if (h < keys)
        to = static_cast<E*>(p.q_out) + (t * p.H_q + h) * p.D;
      else if (!kPools)
        to = static_cast<E*>(p.k_out) + (t * p.H_kv + (h - keys)) * p.D;
      else if (!kept)
        continue;
      else if (h < values)
        to = static_cast<E*>(p.k_out) + at + (h - keys) * p.pool_head_stride;
      else
        to = static_cast<E*>(p.v_out) + at + (h - values) * p.pool_head_stride;
      *reinterpret_cast<vec*>(to + d0) = x[i][0];
      *reinterpret_cast<vec*>(to + d1) = x[i][1];
    }
  }
}

// cos and sin of a step's positions, a value for each of the rot dims (as the
// fused append and decode calls take them).  A thread computes V pairs.
template <class E, int V, bool kInterleaved, bool kAligned>
__global__ __launch_bounds__(256) void rotary_tables_kernel(E* cos, E* sin, const int64_t* positions,
                                                            const double* freqs, double scale, int64_t T, int rot) {
  typedef Pack<E, V, kAligned> vec;
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
  const int half = rot / 2;
  const uint32_t units = (uint32_t)(half + V - 1) / V;
  const int64_t t = gid / units;
  if (t >= T) return;
  const int pair = min(V * (int)(gid % units), half - V);
  float c[V], s[V];
  angles<E, V>((double)positions[t], freqs + pair, scale, c, s);
#pragma unroll
  for (int j = 0; j < V; ++j) asm volatile("" : "+v"(c[j]), "+v"(s[j]));  // (to fp32 first, as above)
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const float* const from = part ? s : c;
    E* const row = (part ? sin : cos) + t * rot;
    vec a, b;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a.v[j] = (E)from[kInterleaved && V > 1 ? j / 2 : j];
      b.v[j] = (E)from[kInterleaved && V > 1 ? V / 2 + j / 2 : j];
    }
    *reinterpret_cast<vec*>(row + (kInterleaved ? 2 * pair : pair)) = a;
    *reinterpret_cast<vec*>(row + (kInterleaved ? 2 * pair + V : pair + half)) = b;
  }
}

static bool multiple_of(int64_t n, int64_t a) { return n % a == 0; }
static bool aligned_to(const void* ptr, int64_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; }

// Threads of a token's heads: enough to half fill the chip (256 CUs of 2,048), with no
// more than six heads a thread, and a power of two, so that a wave's rows lie side by
// side.  8,192 rows of 40 heads of 128: 31 us (5.4 TB/s) with five heads a thread, 43
// with all 40; 2,048 rows 9.6 us with three, 11.3 with one; 8,192 rows of 16 heads of 64
// 8.3 us with two, 10.1 with one.
constexpr int64_t kRotThreads = 256 * 1024;
constexpr int kRotMost = 6;
constexpr int64_t kRotMaxBlocks = (1 << 24) - 1;  // thread indexes in 32 bits

template <class E, int V, bool kPools, bool kAligned>
static int launch_rotary(RotaryParams p, bool interleaved, hipStream_t stream) {
  p.units = (p.rot / 2 + V - 1) / V + (p.D - p.rot + 2 * V - 1) / (2 * V);
  const int64_t heads = (int64_t)p.H_q + (kPools ? 2 : 1) * p.H_kv, row = p.T * p.units;
  int64_t groups = 1;
  while (groups * row < kRotThreads || groups * kRotMost < heads) groups *= 2;
  p.head_groups = (int32_t)(groups < heads ? groups : heads);
  const int64_t blocks = (row * p.head_groups + 255) / 256;
  if (blocks > kRotMaxBlocks) return CIE_EUNSUPPORTED;
  const dim3 grid((unsigned)blocks), block(256);
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<E, V, true, kPools, kAligned>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((rotary_kernel<E, V, false, kPools, kAligned>), grid, block, 0, stream, p);
  return (int)hipGetLastError();
}

// Vectors of 16 bytes where both parts of a head hold one, aligned or not (4,000 rows of
// 32 heads of 64, 20 dims turned: 12.0 us value by value, 9.5 so).
template <class E, bool kPools>
static int dispatch_rotary(const RotaryParams& p, bool interleaved, hipStream_t stream) {
  constexpr int V = VecOf<E>::kWide;
  if (p.rot / 2 < V || (p.D > p.rot && p.D - p.rot < V)) return launch_rotary<E, 1, kPools, true>(p, interleaved, stream);
  bool aligned = multiple_of(p.rot, 2 * V) && multiple_of(p.D, V) && aligned_to(p.q, 16) && aligned_to(p.k, 16) &&
                 aligned_to(p.q_out, 16) && aligned_to(p.k_out, 16) &&
                 multiple_of(p.q_tok | p.q_head | p.k_tok | p.k_head, V);
  if (kPools)
    aligned = aligned && aligned_to(p.v, 16) && aligned_to(p.v_out, 16) &&
              multiple_of(p.v_tok | p.v_head | p.pool_page_stride | p.pool_head_stride, V);
  return aligned ? launch_rotary<E, V, kPools, true>(p, interleaved, stream)
                 : launch_rotary<E, V, kPools, false>(p, interleaved, stream);
}

static int check_sizes(int64_t T, int64_t H_q, int64_t H_kv, int64_t D, int64_t rot, int dtype) {
  if (T < 0 || H_q < 0 || H_kv < 0 || H_q + H_kv <= 0 || D <= 0 || rot < 2 || rot > D || rot % 2 || D % 2)
    return CIE_EINVAL;
  if (dtype < 0 || dtype > 2 || H_q + H_kv > 65536 || D > 65536 || T > 0x7fffffff) return CIE_EUNSUPPORTED;
  return CIE_OK;
}

template <class E, int V, bool kAligned>
static int launch_tables(E* cos, E* sin, const int64_t* positions, const double* freqs, double scale, int64_t T,
                         int64_t rot, bool interleaved, hipStream_t stream) {
  const int64_t blocks = (T * ((rot / 2 + V - 1) / V) + 255) / 256;
  if (blocks > kRotMaxBlocks) return CIE_EUNSUPPORTED;
  const dim3 grid((unsigned)blocks), block(256);
  if (interleaved)
    hipLaunchKernelGGL((rotary_tables_kernel<E, V, true, kAligned>), grid, block, 0, stream, cos, sin, positions, freqs,
                       scale, T, (int)rot);
  else
    hipLaunchKernelGGL((rotary_tables_kernel<E, V, false, kAligned>), grid, block, 0, stream, cos, sin, positions, freqs,
                       scale, T, (int)rot);
  return (int)hipGetLastError();
}

template <class E>
static int dispatch_tables(void* cos, void* sin, const int64_t* positions, const double* freqs, double scale, int64_t T,
                           int64_t rot, bool interleaved, hipStream_t stream) {
  constexpr int V = VecOf<E>::kWide;
  E* const c = static_cast<E*>(cos);
  E* const s = static_cast<E*>(sin);
  if (rot / 2 < V) return launch_tables<E, 1, true>(c, s, positions, freqs, scale, T, rot, interleaved, stream);
  return multiple_of(rot, 2 * V) && aligned_to(cos, 16) && aligned_to(sin, 16)
             ? launch_tables<E, V, true>(c, s, positions, freqs, scale, T, rot, interleaved, stream)
             : launch_tables<E, V, false>(c, s, positions, freqs, scale, T, rot, interleaved, stream);
}

}  // namespace cie

using namespace cie;

extern "C" int cie_rotary(void* q_out, void* k_out, const void* q, const void* k, int64_t q_tok_stride,
                          int64_t q_head_stride, int64_t k_tok_stride, int64_t k_head_stride,
                          const int64_t* positions, const double* freqs, double scale, int64_t T, int64_t H_q,
                          int64_t H_kv, int64_t D, int64_t rot, int interleaved, int dtype, void* stream) {
  const int bad = check_sizes(T, H_q, H_kv, D, rot, dtype);
  if (bad) return bad;
  if (T == 0) return CIE_OK;
  if (!positions || !freqs || (H_q > 0 && (!q || !q_out)) || (H_kv > 0 && (!k || !k_out))) return CIE_EINVAL;
  RotaryParams p{};
  p.q_out = q_out;
  p.k_out = k_out;
  p.q = q;
  p.k = k;
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.k_tok = k_tok_stride;
  p.k_head = k_head_stride;
  p.positions = positions;
  p.freqs = freqs;
  p.T = T;
  p.scale = scale;
  p.H_q = (int32_t)H_q;
  p.H_kv = (int32_t)H_kv;
  p.D = (int32_t)D;
  p.rot = (int32_t)rot;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CIE_F16    ? dispatch_rotary<f16, false>(p, interleaved, st)
         : dtype == CIE_BF16 ? dispatch_rotary<bf16, false>(p, interleaved, st)
                             : dispatch_rotary<float, false>(p, interleaved, st);
}

extern "C" int cie_kv_append_tokens_qkv_rotary(
    void* q_out, void* k_pool, void* v_pool, const void* qkv, int64_t qkv_row_stride, const int64_t* positions,
    const double* freqs, double scale, const int64_t* pages, const int64_t* offsets, int64_t T, int64_t H_q,
    int64_t H_kv, int64_t page_size, int64_t D, int64_t n_pages, int64_t pool_page_stride, int64_t pool_head_stride,
    int64_t rot, int interleaved, int dtype, int32_t* err, void* stream) {
  const int bad = check_sizes(T, H_q, H_kv, D, rot, dtype);
  if (bad) return bad;
  if (H_q <= 0 || H_kv <= 0 || page_size <= 0 || n_pages <= 0) return CIE_EINVAL;
  if (page_size > 0x7fffffff || dtype == CIE_F32) return CIE_EUNSUPPORTED;
  if (T == 0) return CIE_OK;
  if (!q_out || !k_pool || !v_pool || !qkv || !positions || !freqs || !pages || !offsets ||
      qkv_row_stride < (H_q + 2 * H_kv) * D)
    return CIE_EINVAL;
  RotaryParams p{};
  const char* const rows = static_cast<const char*>(qkv);
  p.q_out = q_out;
  p.k_out = k_pool;
  p.v_out = v_pool;
  p.q = rows;
  p.k = rows + 2 * H_q * D;
  p.v = rows + 2 * (H_q + H_kv) * D;
  p.q_tok = p.k_tok = p.v_tok = qkv_row_stride;
  p.q_head = p.k_head = p.v_head = D;
  p.positions = positions;
  p.freqs = freqs;
  p.pages = pages;
  p.offsets = offsets;
  p.pool_page_stride = pool_page_stride;
  p.pool_head_stride = pool_head_stride;
  p.n_pages = n_pages;
  p.T = T;
  p.scale = scale;
  p.H_q = (int32_t)H_q;
  p.H_kv = (int32_t)H_kv;
  p.D = (int32_t)D;
  p.rot = (int32_t)rot;
  p.page_size = (int32_t)page_size;
  p.err = err;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CIE_F16 ? dispatch_rotary<f16, true>(p, interleaved, st)
                          : dispatch_rotary<bf16, true>(p, interleaved, st);
}

extern "C" int cie_rotary_tables(void* cos, void* sin, const int64_t* positions, const double* freqs, double scale,
                                 int64_t T, int64_t rot, int interleaved, int dtype, void* stream) {
  if (T < 0 || rot < 2 || rot % 2) return CIE_EINVAL;
  if (dtype < 0 || dtype > 2 || rot > 65536 || T > 0x7fffffff) return CIE_EUNSUPPORTED;
  if (T == 0) return CIE_OK;
  if (!cos || !sin || !positions || !freqs) return CIE_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CIE_F16    ? dispatch_tables<f16>(cos, sin, positions, freqs, scale, T, rot, interleaved, st)
         : dtype == CIE_BF16 ? dispatch_tables<bf16>(cos, sin, positions, freqs, scale, T, rot, interleaved, st)
                             : dispatch_tables<float>(cos, sin, positions, freqs, scale, T, rot, interleaved, st);
}
