// urb_sample.hip -- drawing a token per row of logits under temperature, top-k, top-p and min-p.
//
// All three filters keep a beginning of one order (logit descending, index ascending), so a row's
// kept tokens are those above a threshold logit plus the first few of those equal to it, and no row
// is ever sorted.  Logits are compared as 32-bit keys in their order; masses e = exp((l - m) / tau) are
// computed in f64 and summed as integers of 2^-shift (shift 42 to 61, by the vocabulary), so sums do not depend
// on their order and a row's result is the same whatever workgroups share it.
#include "urb_device.hpp"
#include "urb_step.hpp"

#include <type_traits>

namespace urb {

namespace {

typedef unsigned long long u64;

constexpr uint32_t kMinusInf = 0x007fffffu;  // key of -inf; NaN keys are 0

// Order-preserving key of a logit: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) return 0;
  const uint32_t b = f2u(l + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return u2f(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* p, size_t i) {
  if constexpr (BF16) return u2f((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  else return reinterpret_cast<const float*>(p)[i];
}

// exp(x) for x <= 0 in f64, 0 below 2^-63 (half of the finest unit that masses are summed in).
// x = n ln 2 + r with |r| <= ln(2) / 2; the Taylor series to r^13 leaves out less than 5e-18.
__device__ __forceinline__ double exp_down(double x) {
  if (!(x > -43.7)) return 0.0;
  const double n = rint(x * 1.4426950408889634074);
  double r = fma(-n, 0x1.62e42fefa39efp-1, x);  // ln 2, high and low part
  r = fma(-n, 0x1.abc9e3b39803fp-56, r);
  double s = 1.0 / 6227020800.0;
  s = fma(s, r, 1.0 / 479001600.0);
  s = fma(s, r, 1.0 / 39916800.0);
  s = fma(s, r, 1.0 / 3628800.0);
  s = fma(s, r, 1.0 / 362880.0);
  s = fma(s, r, 1.0 / 40320.0);
  s = fma(s, r, 1.0 / 5040.0);
  s = fma(s, r, 1.0 / 720.0);
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  s = fma(s, r, 1.0);
  return ldexp(s, (int)n);
}

// e of a logit key, and e as an integer.
struct Mass {
  double top, inv, scale;  // largest logit, 1 / temperature, 2^shift
  uint32_t top_key;
  float topf, bins;  // kBins / kBinRange / temperature
  __device__ __forceinline__ Mass(uint32_t key, float tau, double scale_)
      : top((double)key_value(key)), inv(1.0 / (double)tau), scale(scale_), top_key(key),
        topf(key_value(key)), bins((kBins / kBinRange) / tau) {}
  __device__ __forceinline__ double e(uint32_t key) const {
    if (key == top_key) return 1.0;  // also where both are +inf
    return exp_down(((double)key_value(key) - top) * inv);
  }
  __device__ __forceinline__ u64 fixed(double e) const { return (u64)(e * scale + 0.5); }
  // Bins of (m - l) / tau over [0, kBinRange), the last one open; the f32 steps keep the logits' order.
  static constexpr int kBins = 2048;
  static constexpr float kBinRange = 44.5f;  // beyond it masses are zero
  __device__ __forceinline__ int bin(uint32_t key) const {
    if (key == top_key) return 0;
    const float z = (topf - key_value(key)) * bins;
    return z < (float)(kBins - 1) ? (int)z : kBins - 1;
  }
};
constexpr int kBins = Mass::kBins;

// The sum that a beginning of the order must reach for top_p of `total` (an integer: sums are).
__device__ __forceinline__ u64 mass_wanted(float top_p, u64 total) {
  const u64 want = (u64)ceil((double)top_p * (double)total);
  return want < 1 ? 1 : want > total ? total : want;
}

// Block-wide helpers of the one-workgroup kernel.
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;

template <class T>
__device__ __forceinline__ T wave_sum(T v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int WAVES = kRowWaves, class T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  T s = 0;
  for (int w = 0; w < WAVES; ++w) s += slots[w];
  return s;
}
// Sum over the threads before this one; *total over all.
template <int WAVES = kRowWaves, class T>
__device__ __forceinline__ T block_before(T v, T* slots, T* total) {
  T inc = v;
  const int lane = threadIdx.x & 63;
  for (int o = 1; o < 64; o <<= 1) {
    const T up = __shfl_up(inc, o, 64);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 63) slots[threadIdx.x >> 6] = inc;
  __syncthreads();
  T before = 0, all = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += slots[w];
    all += slots[w];
  }
  *total = all;
  return before + inc - v;
}

// The bin where the running sum of `hist` from the highest bin down reaches `want` (1 <= want <= the
// sum of all), and the sum above it.  All threads get both.
__device__ void find_bin(const u64* hist, u64 want, u64* slots, int* bin, u64* above) {
  __shared__ int s_bin;
  __shared__ u64 s_above;
  constexpr int PER = kBins / kRowThreads;
  u64 mine[PER], sum = 0;
  const int first = kBins - 1 - (int)threadIdx.x * PER;  // highest bins first
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    mine[i] = hist[first - i];
    sum += mine[i];
  }
  u64 total;
  u64 run = block_before(sum, slots, &total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (run < want && run + mine[i] >= want) {
      s_bin = first - i;
      s_above = run;
    }
    run += mine[i];
  }
  __syncthreads();
  *bin = s_bin;
  *above = s_above;
  __syncthreads();
}

struct RowParams {
  float tau, top_p, min_p, uniform;
  int top_k;
  bool ok;
};
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row) {
  RowParams p;
  p.tau = a.temperature ? a.temperature[row] : 1.0f;
  p.top_k = a.top_k ? a.top_k[row] : 0;
  p.top_p = a.top_p ? a.top_p[row] : 1.0f;
  p.min_p = a.min_p ? a.min_p[row] : 0.0f;
  p.uniform = a.uniform[row];
  p.ok = finite(p.tau) && p.tau >= 0.0f && p.top_p > 0.0f && p.min_p >= 0.0f &&
         p.min_p <= 1.0f && p.uniform >= 0.0f && p.uniform < 1.0f;
  return p;
}

// ---- a row in one workgroup, whatever it holds: the thresholds by radix selection over the keys ----

struct RowLds {
  u64 hist[kBins];
  u64 slots[kRowWaves];
  int islots[kRowWaves];
  int found;
};

// -> (id, e of it, sum over the kept tokens); all threads.
template <bool BF16>
__device__ __noinline__ int draw_by_radix(const uint8_t* base, int V, const RowParams& p,
                                          const Mass& mass, RowLds& lds, u64* sum_kept) {
  u64* const hist = lds.hist;
  u64* const slots = lds.slots;
  int* const islots = lds.islots;
  const int tid = threadIdx.x;
  auto key = [&](int i) { return key_of(load_logit<BF16>(base, i)); };

  // Radix selection: the key at which the running sum of value(key) from the highest key down
  // reaches want, among keys for which `in`; *above = the sum over the keys beyond it.
  auto select = [&](auto value, auto in, u64 want, u64* above) -> uint32_t {
    uint32_t prefix = 0;
    u64 over = 0;
    for (int level = 0; level < 3; ++level) {
      const int low = level == 0 ? 21 : level == 1 ? 10 : 0;   // digits of 11, 11 and 10 bits
      const int bits = level == 2 ? 10 : 11;
      for (int b = tid; b < kBins; b += kRowThreads) hist[b] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kRowThreads) {
        const uint32_t k = key(i);
        if (!in(k)) continue;
        if (level && (k >> (low + bits)) != (prefix >> (low + bits))) continue;
        const u64 v = value(k);
        if (v) atomicAdd(&hist[(k >> low) & ((1u << bits) - 1)], v);
      }
      __syncthreads();
      int bin;
      u64 up;
      find_bin(hist, want - over, slots, &bin, &up);
      prefix |= (uint32_t)bin << low;
      over += up;
    }
    *above = over;
    return prefix;
  };
  auto valid = [&](uint32_t k) { return k > kMinusInf; };

  // kept: keys above `cut`, and the first `ties` of those equal to it
  uint32_t cut = kMinusInf;
  long long ties = 0;
  u64 tied = 0;  // mass of one of them
  if (p.top_k > 0 && p.top_k < V) {
    int n = 0;
    for (int i = tid; i < V; i += kRowThreads) n += valid(key(i));
    n = block_sum(n, islots);
    if (p.top_k < n) {
      u64 above;
      cut = select([](uint32_t) { return (u64)1; }, valid, (u64)p.top_k, &above);
      ties = p.top_k - (long long)above;
      tied = mass.fixed(mass.e(cut));
    }
  }
  if (p.top_p < 1.0f) {
    u64 sum = 0;
    for (int i = tid; i < V; i += kRowThreads) {
      const uint32_t k = key(i);
      if (k > cut) sum += mass.fixed(mass.e(k));
    }
    const u64 higher = block_sum(sum, slots);
    const u64 want = mass_wanted(p.top_p, higher + (u64)ties * tied);
    u64 above = higher;
    if (higher >= want) {  // reached above the ties of top_k
      cut = select([&](uint32_t q) { return mass.fixed(mass.e(q)); },
                   [&, from = cut](uint32_t q) { return q > from; }, want, &above);
      tied = mass.fixed(mass.e(cut));
    }
    ties = (long long)((want - above + tied - 1) / tied);
  }
  const double min_e = (double)p.min_p;
  u64 sum = 0;
  for (int i = tid; i < V; i += kRowThreads) {
    const uint32_t k = key(i);
    if (k > cut) {
      const double e = mass.e(k);
      if (e >= min_e) sum += mass.fixed(e);
    }
  }
  u64 total = block_sum(sum, slots);
  if (ties && mass.e(cut) >= min_e) total += (u64)ties * tied;
  else ties = 0;
  const double target = (double)p.uniform * (double)total;

  // the draw, tile by tile in index order
  if (tid == 0) lds.found = -1;
  constexpr int PER = 4;
  u64 before = 0;
  long long tie_count = 0;
  for (int i0 = 0; i0 < V; i0 += kRowThreads * PER) {
    uint32_t k[PER];
    int eq = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = i0 + tid * PER + u;
      k[u] = i < V ? key(i) : 0;
      eq += ties && k[u] == cut;
    }
    int all_eq;
    long long tie = tie_count + block_before(eq, islots, &all_eq);
    tie_count += all_eq;
    u64 w[PER], mine = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      bool kept = k[u] > cut;
      if (ties && k[u] == cut) kept = tie++ < ties;
      w[u] = 0;
      if (kept) {
        const double e = mass.e(k[u]);
        if (e >= min_e) w[u] = mass.fixed(e);
      }
      mine += w[u];
    }
    u64 tile;
    u64 run = before + block_before(mine, slots, &tile);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (!((double)run > target) && (double)(run + w[u]) > target) lds.found = i0 + tid * PER + u;
      run += w[u];
    }
    before += tile;
    if ((double)before > target) break;  // the same in all threads
  }
  __syncthreads();
  *sum_kept = total;
  return lds.found;
}

// ---- rows shared by many workgroups ----
//
// Four launches: the largest logit of every chunk; a histogram of the row in bins of (m - l) / tau,
// whose last workgroup finds the bin in which the kept tokens end; the sums of the chunks' tokens
// before that bin, and a list of the tokens in it; and one workgroup per row that orders the list,
// finds the last kept token, the chunk of the draw and the token in it.  A list too long for LDS
// (many equal logits) sends its row to draw_by_radix.
//
// Where the kept tokens are few, the list holds all of them and no sums are needed.  The row is read up
// to three times, after the first time from the Infinity Cache where a batch's logits fit it.

constexpr int kList = 2048;       // tokens that the last launch orders in LDS
constexpr int kChunkUnit = 2048;  // values per chunk and 256 threads: eight per thread
constexpr int kThreads = 256;

enum RowMode {
  kNoCut = 1,     // no top_k, no top_p: everything (that min_p leaves)
  kAllListed,     // the list holds every token of the bins up to the cut
  kBinListed,     // the list holds the cut's bin
  kByRadix,       // too many for a list
};

struct RowRecord {
  int mode, bin;
  int listed;     // tokens in the list
  int arrived;    // workgroups of the histogram that are through
  int above_n;    // tokens before the cut's bin
  int pad;
  u64 above, want;  // their mass; the mass that top_p asks for
};

struct Work {
  int chunks, chunk;  // of every row; values per chunk
  u64* best;          // [rows][chunks] largest key << 32 | ~lowest index
  u64* sums;          // [rows][chunks]
  u64* mass;          // [rows][kBins]
  int* count;         // [rows][kBins]
  u64* list;          // [rows][kList] key << 32 | ~index
  RowRecord* record;  // [rows]
};

template <bool BF16>
struct Row {
  const uint8_t* base;
  int V, lead;  // values from the 16-byte boundary at or before the row to its start
  __device__ __forceinline__ Row(const SampleArgs& a, int row)
      : base(reinterpret_cast<const uint8_t*>(a.logits) +
             (size_t)row * a.row_stride * (BF16 ? 2 : 4)),
        V(a.vocab), lead((int)(reinterpret_cast<uintptr_t>(base) % 16) / (BF16 ? 2 : 4)) {}
  // Keys of the eight values at place v (from the boundary; v % 8 == 0), 0 outside the row; returns
  // the index of the first.
  __device__ __forceinline__ int keys(int v, uint32_t (&k)[8]) const {
    const int i = v - lead;
    if (i >= 0 && i + 8 <= V) {
      if constexpr (BF16) {
        const uint4 q = ldg16(base + 2 * (size_t)i);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          k[2 * u] = key_of(bf16_lo(w[u]));
          k[2 * u + 1] = key_of(bf16_hi(w[u]));
        }
      } else {
        const float4 q = u2f4(ldg16(base + 4 * (size_t)i)), r = u2f4(ldg16(base + 4 * (size_t)i + 16));
        k[0] = key_of(q.x); k[1] = key_of(q.y); k[2] = key_of(q.z); k[3] = key_of(q.w);
        k[4] = key_of(r.x); k[5] = key_of(r.y); k[6] = key_of(r.z); k[7] = key_of(r.w);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        k[u] = i + u >= 0 && i + u < V ? key_of(load_logit<BF16>(base, i + u)) : 0;
    }
    return i;
  }
};

__device__ __forceinline__ u64 wave_max(u64 v) {
  for (int o = 32; o > 0; o >>= 1) {
    const u64 c = __shfl_xor(v, o, 64);
    v = c > v ? c : v;
  }
  return v;
}
template <int WAVES>
__device__ __forceinline__ u64 block_max(u64 v, u64* slots) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v = slots[w] > v ? slots[w] : v;
  return v;
}

// Largest key of each chunk; clears what the next launches add to.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_best_kernel(SampleArgs a, Work w) {
  __shared__ u64 slots[kThreads / 64];
  const int row = blockIdx.y, c = blockIdx.x;
  const Row<BF16> r(a, row);
  u64 best = 0;
  for (int j = 0; j < w.chunk; j += kChunkUnit) {
    uint32_t k[8];
    const int i = r.keys(c * w.chunk + j + 8 * threadIdx.x, k);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const u64 v = ((u64)k[u] << 32) | (0xffffffffu - (uint32_t)(i + u));
      best = v > best ? v : best;
    }
  }
  best = block_max<kThreads / 64>(best, slots);
  if (threadIdx.x == 0) w.best[(size_t)row * w.chunks + c] = best;
  for (int b = c * kThreads + threadIdx.x; b < kBins; b += w.chunks * kThreads) {
    w.mass[(size_t)row * kBins + b] = 0;
    w.count[(size_t)row * kBins + b] = 0;
  }
  if (c == 0 && threadIdx.x == 0) w.record[row] = RowRecord{};
}

// The row's largest key and its lowest index.
template <int WAVES>
__device__ __forceinline__ u64 row_best(const Work& w, int row, u64* slots) {
  u64 best = 0;
  for (int c = threadIdx.x; c < w.chunks; c += 64 * WAVES) {
    const u64 v = w.best[(size_t)row * w.chunks + c];
    best = v > best ? v : best;
  }
  return block_max<WAVES>(best, slots);
}

// A row that needs no sums at all: parameters out of range, nothing to draw, or the largest asked for.
__device__ __forceinline__ bool trivial(const RowParams& p, u64 best) {
  return !p.ok || (uint32_t)(best >> 32) <= kMinusInf || p.tau == 0.0f;
}

// The row's histogram, and by its last workgroup the bin where the kept tokens end.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a, Work w, double scale) {
  __shared__ u64 mass_lds[kBins];
  __shared__ int count_lds[kBins];
  __shared__ u64 slots[kThreads / 64];
  __shared__ int last;
  const int row = blockIdx.y, tid = threadIdx.x;
  const RowParams p = row_params(a, row);
  const u64 best = row_best<kThreads / 64>(w, row, slots);
  const bool by_count = p.top_k > 0 && p.top_k < a.vocab, by_mass = p.top_p < 1.0f;
  if (trivial(p, best)) return;
  RowRecord& rec = w.record[row];
  if (!by_count && !by_mass) {
    if (blockIdx.x == 0 && tid == 0) rec.mode = kNoCut;
    return;
  }
  const Row<BF16> r(a, row);
  const Mass m((uint32_t)(best >> 32), p.tau, scale);
  for (int b = tid; b < kBins; b += kThreads) {
    mass_lds[b] = 0;
    count_lds[b] = 0;
  }
  __syncthreads();
  for (int j = 0; j < w.chunk; j += kChunkUnit) {
    uint32_t k[8];
    r.keys(blockIdx.x * w.chunk + j + 8 * tid, k);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (k[u] <= kMinusInf) continue;
      const int b = m.bin(k[u]);
      atomicAdd(&count_lds[b], 1);
      if (!by_count) {
        const u64 f = m.fixed(m.e(k[u]));
        if (f) atomicAdd(&mass_lds[b], f);
      }
    }
  }
  __syncthreads();
  u64* const mass = w.mass + (size_t)row * kBins;
  int* const count = w.count + (size_t)row * kBins;
  for (int b = tid; b < kBins; b += kThreads) {
    if (count_lds[b]) atomicAdd(&count[b], count_lds[b]);
    if (mass_lds[b]) atomicAdd(&mass[b], mass_lds[b]);
  }
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(&rec.arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           w.chunks - 1;
  __syncthreads();
  if (!last) return;

  // 8 bins per thread, in order
  constexpr int PER = kBins / kThreads;
  int n[PER], n_sum = 0;
  u64 f[PER], f_sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    n[i] = __hip_atomic_load(&count[tid * PER + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    f[i] = by_count ? 0
                    : __hip_atomic_load(&mass[tid * PER + i], __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
    n_sum += n[i];
    f_sum += f[i];
  }
  __shared__ int n_slots[kThreads / 64];
  int n_all;
  u64 f_all;
  int n_run = block_before<kThreads / 64>(n_sum, n_slots, &n_all);
  u64 f_run = block_before<kThreads / 64>(f_sum, slots, &f_all);
  const u64 want = by_count ? 0 : mass_wanted(p.top_p, f_all);
  const int k = min(p.top_k, n_all);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool here = by_count ? n_run < k && n_run + n[i] >= k : f_run < want && f_run + f[i] >= want;
    if (here) {
      rec.bin = tid * PER + i;
      rec.above_n = n_run;
      rec.above = f_run;
      rec.want = want;
      rec.mode = n_run + n[i] <= kList                        ? kAllListed
                 : n[i] <= kList && !(by_count && by_mass) ? kBinListed
                                                              : kByRadix;
    }
    n_run += n[i];
    f_run += f[i];
  }
}

// The chunks' sums over the tokens before the cut's bin, and the list.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_list_kernel(SampleArgs a, Work w, double scale) {
  __shared__ u64 slots[kThreads / 64];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  RowRecord& rec = w.record[row];
  const int mode = rec.mode, cut = rec.bin;
  if (mode == 0 || mode == kByRadix) return;
  const RowParams p = row_params(a, row);
  const Mass m((uint32_t)(row_best<kThreads / 64>(w, row, slots) >> 32), p.tau, scale);
  const Row<BF16> r(a, row);
  const double min_e = (double)p.min_p;
  u64 sum = 0;
  for (int j = 0; j < w.chunk; j += kChunkUnit) {
    uint32_t k[8];
    const int i = r.keys(blockIdx.x * w.chunk + j + 8 * tid, k);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool valid = k[u] > kMinusInf;
      const int b = m.bin(k[u]);
      if (valid && (mode == kNoCut || (mode == kBinListed && b < cut))) {
        const double e = m.e(k[u]);
        if (e >= min_e) sum += m.fixed(e);
      }
      const bool listed = valid && (mode == kBinListed ? b == cut : mode == kAllListed && b <= cut);
      const u64 vote = __ballot(listed);
      if (vote) {
        int at = 0;
        if (lane == 0) at = atomicAdd(&rec.listed, __popcll(vote));
        at = __shfl(at, 0, 64) + __popcll(vote & ((1ull << lane) - 1));
        if (listed && at < kList)  // (at most kList: the histogram counted them)
          w.list[(size_t)row * kList + at] = ((u64)k[u] << 32) | (0xffffffffu - (uint32_t)(i + u));
      }
    }
  }
  if (mode != kAllListed) {
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) slots[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
      for (int v = 1; v < kThreads / 64; ++v) sum += slots[v];
      w.sums[(size_t)row * w.chunks + blockIdx.x] = sum;
    }
  }
}

// Sorts the first n values of v (padded with zeros to a power of two of at least 64 within kList):
// descending.
__device__ void sort_descending(u64* v, int n) {
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += kRowThreads) v[i] = 0;
  for (int width = 2; width <= size; width *= 2)
    for (int gap = width / 2; gap > 0; gap /= 2) {
      __syncthreads();
      for (int t = threadIdx.x; t < size / 2; t += kRowThreads) {
        const int i = 2 * t - (t & (gap - 1)), j = i + gap;
        const u64 x = v[i], y = v[j];
        if ((x < y) == ((i & width) == 0)) {
          v[i] = y;
          v[j] = x;
        }
      }
    }
  __syncthreads();
}

// One workgroup per row: the last kept token of the list, then the draw.  SMALL: a vocabulary that fits
// the list, in this launch alone.
template <bool BF16, bool SMALL>
__global__ __launch_bounds__(kRowThreads) void sample_draw_kernel(SampleArgs a, Work w,
                                                                  double scale) {
  __shared__ union {
    RowLds radix;
    struct {
      u64 list[kList];
      u64 slots[kRowWaves];
      int islots[kRowWaves];
    } s;
  } lds;
  __shared__ int s_n, s_found;
  __shared__ u64 s_cut, s_before;
  const int row = blockIdx.x, tid = threadIdx.x;
  const RowParams p = row_params(a, row);
  const Row<BF16> r(a, row);
  u64 best = 0;
  int mode = kAllListed, n = 0;
  if constexpr (SMALL) {
    if (tid == 0) s_n = 0;
    __syncthreads();
    uint32_t k[8];
    const int i = r.keys(8 * tid, k);   // (a row of kList values starts at most 7 past a boundary)
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k[u] > kMinusInf) {
        const u64 v = ((u64)k[u] << 32) | (0xffffffffu - (uint32_t)(i + u));
        best = v > best ? v : best;
        lds.s.list[atomicAdd(&s_n, 1)] = v;
      }
    best = block_max<kRowWaves>(best, lds.s.slots);
    n = s_n;
  } else {
    best = row_best<kRowWaves>(w, row, lds.s.slots);
  }
  auto done = [&](int id, float prob) {
    if (tid == 0) {
      a.ids[row] = id;
      if (a.probs) a.probs[row] = prob;
    }
  };
  if (trivial(p, best)) {
    if (!p.ok && tid == 0) flag(a.status, kStepArgument);
    const bool greedy = p.ok && (uint32_t)(best >> 32) > kMinusInf;
    done(greedy ? (int)(0xffffffffu - (uint32_t)best) : -1, greedy ? 1.0f : 0.0f);
    return;
  }
  const Mass m((uint32_t)(best >> 32), p.tau, scale);
  const double min_e = (double)p.min_p, uniform = (double)p.uniform;
  auto prob_of = [&](uint32_t key, u64 total) {
    return (float)(m.e(key) / ((double)total / scale));
  };
  RowRecord rec{};
  if constexpr (!SMALL) {
    rec = w.record[row];
    mode = rec.mode;
    n = min(rec.listed, kList);
    if (mode == kByRadix) {
      u64 total;
      __syncthreads();
      const int id = draw_by_radix<BF16>(r.base, r.V, p, m, lds.radix, &total);
      done(id, prob_of(key_of(load_logit<BF16>(r.base, id)), total));
      return;
    }
    for (int i = tid; i < n; i += kRowThreads) lds.s.list[i] = w.list[(size_t)row * kList + i];
  }
  // the list's kept tokens are its first `kept` in order
  int kept = 0;
  u64 kept_mass = 0;
  if (mode != kNoCut) {
    sort_descending(lds.s.list, n);
    const bool by_count = p.top_k > 0 && p.top_k < r.V;
    // (with every kept token in the list nothing comes before it)
    const int above_n = mode == kBinListed ? rec.above_n : 0;
    const int most = by_count ? min(n, p.top_k - above_n) : n;
    u64 f[2], mine = 0;
    double e[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = 2 * tid + u;
      e[u] = i < most ? m.e((uint32_t)(lds.s.list[i] >> 32)) : 0.0;
      f[u] = i < most ? m.fixed(e[u]) : 0;
      mine += f[u];
    }
    u64 all;
    u64 run = (mode == kBinListed ? rec.above : 0) + block_before<kRowWaves>(mine, lds.s.slots, &all);
    u64 want = ~0ull;
    if (p.top_p < 1.0f) want = by_count || SMALL ? mass_wanted(p.top_p, all) : rec.want;
    int mine_n = 0;
    u64 mine_f = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // (with equal logits e >= min_p holds for all or none, so the kept ones stay a beginning)
      if (2 * tid + u < most && run < want && e[u] >= min_e) {
        ++mine_n;
        mine_f += f[u];
      }
      run += f[u];
    }
    kept = block_sum<kRowWaves>(mine_n, lds.s.islots);
    kept_mass = block_sum<kRowWaves>(mine_f, lds.s.slots);
  }
  if (mode == kAllListed) {
    // the draw among the kept tokens by index: sorted by it, the key in the low half
    const double target = uniform * (double)kept_mass;
    for (int i = tid; i < kept; i += kRowThreads) {
      const u64 v = lds.s.list[i];
      lds.s.list[i] = (v << 32) | (v >> 32);   // ~index descending
    }
    sort_descending(lds.s.list, kept);
    u64 f[2];
    uint32_t key[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = 2 * tid + u;
      key[u] = i < kept ? (uint32_t)lds.s.list[i] : 0;
      f[u] = i < kept ? m.fixed(m.e(key[u])) : 0;
    }
    u64 all;
    u64 run = block_before<kRowWaves>(f[0] + f[1], lds.s.slots, &all);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!((double)run > target) && (double)(run + f[u]) > target) {
        a.ids[row] = (int)(0xffffffffu - (uint32_t)(lds.s.list[2 * tid + u] >> 32));
        if (a.probs) a.probs[row] = prob_of(key[u], kept_mass);
      }
      run += f[u];
    }
    return;
  }
  // the draw among the chunks' sums and the kept tokens of the list, which are added to theirs
  if (tid == 0) {
    s_cut = mode == kNoCut ? 0 : kept ? lds.s.list[kept - 1] : ~0ull;
    s_found = 0;
    s_before = 0;
  }
  __syncthreads();
  const u64 cut = s_cut;
  // tokens kept: valid, not after the cut in order, e >= min_p.  (Nothing kept of the list, because
  // of min_p: then nothing below its bin is kept and e decides.)
  u64 list_mine[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) list_mine[u] = 2 * tid + u < kept ? lds.s.list[2 * tid + u] : 0;
  __syncthreads();
  u64* const sums = lds.s.list;  // at most kList chunks
  for (int c = tid; c < w.chunks; c += kRowThreads) sums[c] = w.sums[(size_t)row * w.chunks + c];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (list_mine[u]) {
      const int i = (int)(0xffffffffu - (uint32_t)list_mine[u]);
      atomicAdd(&sums[(i + r.lead) / w.chunk], m.fixed(m.e((uint32_t)(list_mine[u] >> 32))));
    }
  __syncthreads();
  const u64 s0 = 2 * tid < w.chunks ? sums[2 * tid] : 0;
  const u64 s1 = 2 * tid + 1 < w.chunks ? sums[2 * tid + 1] : 0;
  u64 total;
  const u64 before = block_before<kRowWaves>(s0 + s1, lds.s.slots, &total);
  const double target = uniform * (double)total;
  if (!((double)before > target)) {
    if ((double)(before + s0) > target) {
      s_found = 2 * tid;
      s_before = before;
    } else if ((double)(before + s0 + s1) > target) {
      s_found = 2 * tid + 1;
      s_before = before + s0;
    }
  }
  __syncthreads();
  const int c = s_found;
  u64 run = s_before;
  for (int j = 0; j < w.chunk; j += 8 * kRowThreads) {
    uint32_t k[8];
    const int v = j + 8 * tid;
    const bool inside = v < w.chunk;
    const int i = r.keys(c * w.chunk + (inside ? v : 0), k);
    u64 f[8], mine = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const u64 at = ((u64)k[u] << 32) | (0xffffffffu - (uint32_t)(i + u));
      f[u] = 0;
      const bool in_order = cut == ~0ull ? m.bin(k[u]) < rec.bin : at >= cut;
      if (inside && k[u] > kMinusInf && in_order) {
        const double e = m.e(k[u]);
        if (e >= min_e) f[u] = m.fixed(e);
      }
      mine += f[u];
    }
    u64 all;
    u64 at = run + block_before<kRowWaves>(mine, lds.s.slots, &all);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (!((double)at > target) && (double)(at + f[u]) > target) {
        a.ids[row] = i + u;
        if (a.probs) a.probs[row] = prob_of(k[u], total);
      }
      at += f[u];
    }
    run += all;
    if ((double)run > target) break;  // the same in all threads
  }
}

size_t row_bytes(int chunks) {
  return (size_t)chunks * 16 + kBins * 12 + kList * 8 + sizeof(RowRecord);
}
int most_chunks(int vocab) { return (vocab + 7 + kChunkUnit - 1) / kChunkUnit; }

template <bool BF16>
void launch_rows(const SampleArgs& a, const Work& w, double scale, hipStream_t s) {
  if (a.vocab <= kList) {
    sample_draw_kernel<BF16, true><<<a.rows, kRowThreads, 0, s>>>(a, w, scale);
    return;
  }
  const dim3 grid(w.chunks, a.rows);
  sample_best_kernel<BF16><<<grid, kThreads, 0, s>>>(a, w);
  sample_bins_kernel<BF16><<<grid, kThreads, 0, s>>>(a, w, scale);
  sample_list_kernel<BF16><<<grid, kThreads, 0, s>>>(a, w, scale);
  sample_draw_kernel<BF16, false><<<a.rows, kRowThreads, 0, s>>>(a, w, scale);
}

}  // namespace

size_t sample_work_bytes(int vocab, int rows) {
  return vocab <= kList ? 0 : (size_t)std::min(rows, kSamplePass) * row_bytes(most_chunks(vocab));
}

void launch_sample(const SampleArgs& a, bool bf16, hipStream_t s) {
  int log = 0;
  while ((1 << log) < a.vocab) ++log;
  const double scale = (double)(1ull << (62 - (log < 1 ? 1 : log)));
  for (int row = 0; row < a.rows; row += kSamplePass) {
    SampleArgs p = a;
    p.rows = std::min(kSamplePass, a.rows - row);
    p.logits = static_cast<const char*>(a.logits) + (size_t)row * a.row_stride * (bf16 ? 2 : 4);
    if (a.temperature) p.temperature += row;
    if (a.top_k) p.top_k += row;
    if (a.top_p) p.top_p += row;
    if (a.min_p) p.min_p += row;
    p.uniform += row;
    p.ids += row;
    if (a.probs) p.probs += row;
    Work w{};
    if (a.vocab > kList) {
      // chunks of 2048 values for few rows, up to 8192 where that still leaves 16 workgroups per CU
      int units = 1;
      while (units < 4 && (long long)p.rows * ((a.vocab + 7) / (kChunkUnit * units)) > 4096) units *= 2;
      w.chunk = kChunkUnit * units;
      w.chunks = (a.vocab + 7 + w.chunk - 1) / w.chunk;
      const size_t rows = p.rows, most = most_chunks(a.vocab);
      char* at = static_cast<char*>(a.work);
      auto take = [&](auto** q, size_t n) {
        *q = reinterpret_cast<std::remove_reference_t<decltype(*q)>>(at);
        at += n * sizeof(**q);
      };
      take(&w.best, rows * most);
      take(&w.sums, rows * most);
      take(&w.mass, rows * kBins);
      take(&w.list, rows * kList);
      take(&w.record, rows);
      take(&w.count, rows * kBins);
    }
    if (bf16) launch_rows<true>(p, w, scale, s);
    else launch_rows<false>(p, w, scale, s);
  }
}

}  // namespace urb
