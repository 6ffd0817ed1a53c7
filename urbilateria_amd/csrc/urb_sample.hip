// urb_sample.hip -- drawing a token per row of logits under temperature, top-k, top-p and min-p.
//
// All three filters keep a beginning of one order (logit descending, index ascending), so a row's
// kept tokens are those above a threshold logit plus the first few of those equal to it, and no row
// is ever sorted.  Logits are compared as 32-bit keys in their order; masses e = exp((l - m) / tau) are
// computed in f64 and summed as integers of 2^-shift (shift 42 to 51, by the vocabulary), so sums do not
// depend on their order and a row's result is the same whatever workgroups share it.
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

// exp(x) for x <= 0 in f64, 0 below 2^-52.  x = n ln 2 / 16 + r with |r| <= ln(2) / 32, 2^(n / 16) by a table
// of sixteenth powers of two; the Taylor series to r^6 leaves out less than 5e-16.
constexpr int kPowers = 16;
__device__ const double kPower[kPowers] = {
    1.0,                    1.0442737824274138403, 1.0905077326652576592, 1.1387886347566916537,
    1.1892071150027210667,  1.2418578120734840486, 1.2968395546510096659, 1.3542555469368927283,
    1.4142135623730950488,  1.4768261459394993114, 1.5422108254079408236, 1.6104903319492543082,
    1.6817928305074290861,  1.7562521603732994831, 1.8340080864093424635, 1.9152065613971472939};
// The table in LDS (a barrier follows before its first use).
__device__ __forceinline__ void fill_powers(double* powers) {
  if (threadIdx.x < kPowers) powers[threadIdx.x] = kPower[threadIdx.x];
}
__device__ __forceinline__ double exp_down(double x, const double* powers) {
  if (!(x > -36.1)) return 0.0;
  const double magic = 0x1.8p52;  // adding it leaves an integer in the low bits
  const double t = fma(x, 23.083120654223414518, magic);  // 16 / ln 2
  const int n = (int)__double_as_longlong(t);
  const double d = t - magic;
  double r = fma(-d, 0x1.62e42fefa39efp-5, x);  // ln 2 / 16, high and low part
  r = fma(-d, 0x1.abc9e3b39803fp-60, r);
  double s = 1.0 / 720.0;
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  const double p = powers[n & (kPowers - 1)];
  return ldexp(fma(s * r, p, p), n >> 4);
}

// e of a logit, e as an integer, and the bin it falls into.
struct Mass {
  double top, inv, scale;  // largest logit, 1 / temperature, 2^shift
  float topf, bins;        // kBins / kBinRange / temperature
  const double* powers;
  __device__ __forceinline__ Mass(uint32_t key, float tau, double scale_, const double* powers_)
      : top((double)key_value(key)), inv(1.0 / (double)tau), scale(scale_), topf(key_value(key)),
        bins((kBins / kBinRange) / tau), powers(powers_) {}
  __device__ __forceinline__ double e(float l) const {
    if (l == topf) return 1.0;  // also where both are +inf
    return exp_down(((double)l - top) * inv, powers);
  }
  __device__ __forceinline__ double e(uint32_t key) const { return e(key_value(key)); }
  // (scale <= 2^51: the sum's low bits are the integer)
  __device__ __forceinline__ u64 fixed(double e) const {
    return (u64)__double_as_longlong(fma(e, scale, 0x1p52)) & 0xfffffffffffffull;
  }
  // (m - l) / tau in bins of 36.25 / 4096; from the last one on masses are zero.  The f32 steps keep the
  // logits' order; a NaN logit gives NaN.  For temperatures in `usual`: beyond, the difference of two
  // logits or its multiple may overflow f32 though the token has mass, and rows go by radix.
  static __device__ __forceinline__ bool usual(float tau) { return tau > 1e-30f && tau < 1e30f; }
  static constexpr int kBins = 4096;
  static constexpr float kBinRange = 36.25f;
  __device__ __forceinline__ float place(float l) const {
    return l == topf ? 0.0f : (topf - l) * bins;
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

// Running sums and maxima over a wave's lanes by DPP moves (a shuffle goes through the LDS, some ten times
// the latency).  All 64 lanes take part.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
  return (u64)(uint32_t)moved<CTRL, ROWS>((int)(uint32_t)v) |
         (u64)(uint32_t)moved<CTRL, ROWS>((int)(v >> 32)) << 32;
}
template <class T, class F>
__device__ __forceinline__ T wave_running(T v, F op) {
  v = op(v, moved<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8: rows of 16
  v = op(v, moved<0x112, 0xf>(v));
  v = op(v, moved<0x114, 0xf>(v));
  v = op(v, moved<0x118, 0xf>(v));
  v = op(v, moved<0x142, 0xa>(v));  // row 0's last into row 1, row 2's into row 3
  v = op(v, moved<0x143, 0xc>(v));  // row 1's last into rows 2 and 3
  return v;
}
template <class T>
__device__ __forceinline__ T wave_upto(T v) {
  return wave_running(v, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
  return (u64)(uint32_t)lane_of((int)(uint32_t)v, lane) | (u64)(uint32_t)lane_of((int)(v >> 32), lane) << 32;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
  return lane_of(wave_upto(v), 63);
}
__device__ __forceinline__ u64 wave_max(u64 v) {
  return lane_of(wave_running(v, [](u64 a, u64 b) { return a > b ? a : b; }), 63);
}
// Sum over the threads before this one; *total over all.
template <class T>
__device__ __forceinline__ T block_before(T v, T* slots, T* total) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T upto = wave_upto(v);
  __syncthreads();
  if (lane == 63) slots[wave] = upto;
  __syncthreads();
  const T all = wave_upto(lane < kRowWaves ? slots[lane] : T(0));
  *total = lane_of(all, kRowWaves - 1);
  return (wave ? lane_of(all, wave - 1) : T(0)) + upto - v;
}
template <class T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
  T total;
  block_before(v, slots, &total);
  return total;
}

constexpr int kDigits = 2048;  // of a radix pass

// The digit where the running sum of `hist` from the highest bin down reaches `want` (1 <= want <= the
// sum of all), and the sum above it.  All threads get both.
__device__ void find_bin(const u64* hist, u64 want, u64* slots, int* bin, u64* above) {
  __shared__ int s_bin;
  __shared__ u64 s_above;
  constexpr int PER = kDigits / kRowThreads;
  u64 mine[PER], sum = 0;
  const int first = kDigits - 1 - (int)threadIdx.x * PER;  // highest bins first
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
  u64 hist[kDigits];
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
      for (int b = tid; b < kDigits; b += kRowThreads) hist[b] = 0;
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
// Four launches: the largest logit of every part; a histogram of the row in bins of (m - l) / tau; the
// sums of the chunks' tokens before the bin in which the kept tokens end, and a list of the tokens in
// it; and one workgroup per row that orders the list, finds the last kept token, the chunk of the draw
// and the token in it.  A list too long for LDS (many equal logits) sends its row to draw_by_radix.
// (With the bin found by the histogram's last workgroup, behind a device-scope fence in each, that launch
// took 66 us for 256 rows, 53 of them without any sums: the fences write back and drop the L2s.)
//
// The row is read up to three times, after the first time from the Infinity Cache where a batch's logits
// fit it.  256 rows of 129280 f32 logits, a mixture of all filters: 24, 37, 40 and 14 us for the four
// launches; the first reads 132 MB at 5.3 TB/s, the next two are bound by the f64 exponentials of the tokens
// within 36 temperatures of the largest and by LDS atomics.  One row: 4, 6, 5 and 7 us, all latency.  A row
// by radix (129280 logits within 0.1 temperatures, top-p 0.9) takes 450 us alone and 256 of them 780: many
// passes of one workgroup.

constexpr int kList = 1024;                 // tokens that the last launch orders, one per thread
constexpr int kChunk = 8 * kRowThreads;     // values per chunk: eight per thread
constexpr int kSpan = kChunk / kRowWaves;   // values per sum: a wave's of a chunk
constexpr int kMaxSpans = ((1 << 20) / kChunk + 1) * kRowWaves;

enum RowMode {
  kNoCut = 1,     // no top_k, no top_p: everything (that min_p leaves)
  kAllListed,     // the list holds every token of the bins up to the cut
  kBinListed,     // the list holds the cut's bin
  kByRadix,       // too many for a list
};

struct RowRecord {
  int mode, bin;
  int few;        // kBinListed: the tokens up to the cut's bin fit a list too
  int above_n;    // tokens before the cut's bin
  u64 above, want;  // their mass; the mass that top_p asks for
  u64 best;         // the row's largest logit (order_of)
};

constexpr int kGroup = 64, kAllBins = kBins + kBins / kGroup;

struct Work {
  int chunks;            // of a row
  int parts;             // workgroups that share them
  u64* best;          // [rows][parts] largest key << 32 | ~lowest index
  u64* sums;          // [rows][chunks * kRowWaves]: one per span
  u64* mass;          // [rows][kAllBins]: the bins, then groups of kGroup of them
  int* count;         // [rows][kAllBins]
  u64* list;          // [rows][kList] key << 32 | ~index
  RowRecord* record;  // [rows]
  int* listed;        // [rows] tokens in the list
};

template <bool BF16>
struct Row {
  const uint8_t* base;
  int V, lead;  // values from the 16-byte boundary at or before the row to its start
  __device__ __forceinline__ Row(const SampleArgs& a, int row)
      : base(reinterpret_cast<const uint8_t*>(a.logits) +
             (size_t)row * a.row_stride * (BF16 ? 2 : 4)),
        V(a.vocab), lead((int)(reinterpret_cast<uintptr_t>(base) % 16) / (BF16 ? 2 : 4)) {}
  // The eight values at place v (from the boundary; v % 8 == 0), -inf outside the row; returns the
  // index of the first.
  __device__ __forceinline__ int values(int v, float (&l)[8]) const {
    const int i = v - lead;
    if (i >= 0 && i + 8 <= V) {
      if constexpr (BF16) {
        const uint4 q = ldg16(base + 2 * (size_t)i);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          l[2 * u] = bf16_lo(w[u]);
          l[2 * u + 1] = bf16_hi(w[u]);
        }
      } else {
        const float4 q = u2f4(ldg16(base + 4 * (size_t)i)), r = u2f4(ldg16(base + 4 * (size_t)i + 16));
        l[0] = q.x; l[1] = q.y; l[2] = q.z; l[3] = q.w;
        l[4] = r.x; l[5] = r.y; l[6] = r.z; l[7] = r.w;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        l[u] = i + u >= 0 && i + u < V ? load_logit<BF16>(base, i + u) : -__builtin_inff();
    }
    return i;
  }
};

// A logit and its index as one number: larger logits first, then lower indexes.
__device__ __forceinline__ u64 order_of(float l, int i) {
  return ((u64)key_of(l) << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ int index_of(u64 order) { return (int)(0xffffffffu - (uint32_t)order); }
__device__ __forceinline__ uint32_t key_in(u64 order) { return (uint32_t)(order >> 32); }

__device__ __forceinline__ u64 block_max(u64 v, u64* slots) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) v = slots[w] > v ? slots[w] : v;
  return v;
}

// The chunks of a part: [first, last).
struct Part {
  int first, last;
  __device__ __forceinline__ Part(const Work& w, int part)
      : first(w.chunks * part / w.parts), last(w.chunks * (part + 1) / w.parts) {}
};

// Largest key of each part; clears what the next launches add to.
template <bool BF16>
__global__ __launch_bounds__(kRowThreads, 8) void sample_best_kernel(SampleArgs a, Work w) {
  __shared__ u64 slots[kRowWaves];
  const int row = blockIdx.y, tid = threadIdx.x;
  const Row<BF16> r(a, row);
  const Part part(w, blockIdx.x);
  u64 best = 0;
  for (int c = part.first; c < part.last; ++c) {
    float l[8];
    const int i = r.values(c * kChunk + 8 * tid, l);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const u64 v = order_of(l[u], i + u);
      best = v > best ? v : best;
    }
  }
  best = block_max(best, slots);
  if (tid == 0) w.best[(size_t)row * w.parts + blockIdx.x] = best;
  for (int b = blockIdx.x * kRowThreads + tid; b < kAllBins; b += w.parts * kRowThreads) {
    w.mass[(size_t)row * kAllBins + b] = 0;
    w.count[(size_t)row * kAllBins + b] = 0;
  }
  if (blockIdx.x == 0 && tid == 0) w.listed[row] = 0;
}

// The row's largest key and its lowest index.
__device__ __forceinline__ u64 row_best(const Work& w, int row) {
  u64 best = 0;
  for (int c = threadIdx.x & 63; c < w.parts; c += 64) {
    const u64 v = w.best[(size_t)row * w.parts + c];
    best = v > best ? v : best;
  }
  return wave_max(best);
}

// A row that needs no sums at all: parameters out of range, nothing to draw, or the largest asked for.
__device__ __forceinline__ bool trivial(const RowParams& p, u64 best) {
  return !p.ok || (uint32_t)(best >> 32) <= kMinusInf || p.tau == 0.0f;
}

// The row's histogram, of counts and, for top_p alone, of masses.
template <bool BF16>
__global__ __launch_bounds__(kRowThreads, 8) void sample_bins_kernel(SampleArgs a, Work w,
                                                                     double scale) {
  __shared__ u64 mass_lds[kBins];
  __shared__ int count_lds[kBins];
  __shared__ double powers[kPowers];
  const int row = blockIdx.y, tid = threadIdx.x;
  const RowParams p = row_params(a, row);
  const u64 best = row_best(w, row);
  const bool by_count = p.top_k > 0 && p.top_k < a.vocab;
  if (trivial(p, best) || !(by_count || p.top_p < 1.0f)) return;
  const Row<BF16> r(a, row);
  const Mass m(key_in(best), p.tau, scale, powers);
  const Part part(w, blockIdx.x);
  float next[8];
  r.values(part.first * kChunk + 8 * tid, next);
  fill_powers(powers);
  for (int b = tid; b < kBins; b += kRowThreads) {
    mass_lds[b] = 0;
    count_lds[b] = 0;
  }
  __syncthreads();
  for (int c = part.first; c < part.last; ++c) {
    float l[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) l[u] = next[u];
    if (c + 1 < part.last) r.values((c + 1) * kChunk + 8 * tid, next);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      // (logits without mass count for nothing: top_k ends before them or does not matter)
      const float z = m.place(l[u]);
      if (!(z < (float)(kBins - 1))) continue;
      atomicAdd(&count_lds[(int)z], 1);
      if (!by_count) atomicAdd(&mass_lds[(int)z], m.fixed(m.e(l[u])));
    }
  }
  __syncthreads();
  u64* const mass = w.mass + (size_t)row * kAllBins;
  int* const count = w.count + (size_t)row * kAllBins;
  for (int b = tid; b < kBins; b += kRowThreads) {
    int n = count_lds[b];
    u64 f = mass_lds[b];
    if (n) atomicAdd(&count[b], n);
    if (f) atomicAdd(&mass[b], f);
    // a wave holds a group
    n = wave_sum(n);
    f = wave_sum(f);
    if (b % kGroup == 0) {
      if (n) atomicAdd(&count[kBins + b / kGroup], n);
      if (f) atomicAdd(&mass[kBins + b / kGroup], f);
    }
  }
}

// Where the row's kept tokens end, by the histogram: every wave for itself.
__device__ __forceinline__ RowRecord find_cut(const Work& w, int row, const RowParams& p, int V) {
  static_assert(kBins == kGroup * 64 && kGroup == 64, "a lane per group, then one per bin");
  RowRecord rec{};
  const bool by_count = p.top_k > 0 && p.top_k < V, by_mass = p.top_p < 1.0f;
  if (!Mass::usual(p.tau)) {
    rec.mode = kByRadix;
    return rec;
  }
  if (!by_count && !by_mass) {
    rec.mode = kNoCut;
    return rec;
  }
  const int lane = threadIdx.x & 63;
  const u64* const mass = w.mass + (size_t)row * kAllBins;
  const int* const count = w.count + (size_t)row * kAllBins;
  int n = count[kBins + lane];
  u64 f = mass[kBins + lane];
  int n_upto = wave_upto(n);
  u64 f_upto = wave_upto(f);
  const int k = min(p.top_k, lane_of(n_upto, 63));
  rec.want = by_count ? 0 : mass_wanted(p.top_p, lane_of(f_upto, 63));
  // the first lane whose sums reach what is asked for, and the sums before it
  auto cross = [&] {
    const bool reached = by_count ? rec.above_n + n_upto >= k : rec.above + f_upto >= rec.want;
    const int at = __ffsll(__ballot(reached)) - 1;
    rec.above_n += lane_of(n_upto - n, at);
    rec.above += lane_of(f_upto - f, at);
    return at;
  };
  const int group = cross();
  n = count[group * kGroup + lane];
  f = mass[group * kGroup + lane];
  n_upto = wave_upto(n);
  f_upto = wave_upto(f);
  const int at = cross();
  rec.bin = group * kGroup + at;
  const int here = lane_of(n, at);
  rec.few = rec.above_n + here <= kList;
  // (top_p of top_k's tokens needs all of them in order)
  if (by_count && by_mass) rec.mode = rec.few ? kAllListed : kByRadix;
  else rec.mode = here <= kList ? kBinListed : kByRadix;
  return rec;
}

// The chunks' sums over the tokens before the cut's bin, and the list.  Each workgroup gathers both in
// LDS and adds its part of the list with one atomic, so its chunks follow one another without barriers.
// Where the tokens up to the cut are few, they are gathered first and their masses computed from there:
// inside the loop any one of them costs its whole wave an exponential.
template <bool BF16>
__global__ __launch_bounds__(kRowThreads, 8) void sample_list_kernel(SampleArgs a, Work w,
                                                                     double scale) {
  __shared__ u64 list[kList];
  __shared__ u64 sums[kMaxSpans];
  __shared__ int s_n, s_at;
  __shared__ double powers[kPowers];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const RowParams p = row_params(a, row);
  const u64 best = row_best(w, row);
  if (trivial(p, best)) {
    if (blockIdx.x == 0 && tid == 0) w.record[row].best = best;
    return;
  }
  const Row<BF16> r(a, row);
  const Part part(w, blockIdx.x);
  float next[8];
  int at_next = r.values(part.first * kChunk + 8 * tid, next);
  RowRecord rec = find_cut(w, row, p, a.vocab);
  rec.best = best;
  if (blockIdx.x == 0 && tid == 0) w.record[row] = rec;
  if (rec.mode == kByRadix) return;
  const Mass m(key_in(best), p.tau, scale, powers);
  const double min_e = (double)p.min_p;
  fill_powers(powers);
  const int spans = (part.last - part.first) * kRowWaves;
  for (int i = tid; i < spans; i += kRowThreads) sums[i] = 0;
  if (tid == 0) s_n = 0;
  __syncthreads();
  // places below `sum_to` are summed in the loop, those from there to below `list_to` listed
  const bool dense = rec.mode == kAllListed || rec.few;
  const float sum_to = rec.mode == kNoCut ? (float)(kBins - 1) : dense ? 0.0f : (float)rec.bin;
  const float list_to = rec.mode == kNoCut ? 0.0f : (float)(rec.bin + 1);
  for (int c = part.first; c < part.last; ++c) {
    float l[8];
    const int i = at_next;
#pragma unroll
    for (int u = 0; u < 8; ++u) l[u] = next[u];
    if (c + 1 < part.last) at_next = r.values((c + 1) * kChunk + 8 * tid, next);
    u64 sum = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float z = m.place(l[u]);
      if (z < sum_to) {
        const double e = m.e(l[u]);
        if (e >= min_e) sum += m.fixed(e);
      } else if (z < list_to) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kList) list[at] = order_of(l[u], i + u);  // (it is: the histogram counted them)
      }
    }
    if (!dense) {
      sum = wave_sum(sum);
      if (lane == 0) sums[(c - part.first) * kRowWaves + tid / 64] = sum;
    }
  }
  __syncthreads();
  const int n = min(s_n, kList);
  const u64 mine = tid < n ? list[tid] : 0;
  bool listed = tid < n;
  if (rec.mode == kBinListed && rec.few) {
    if (listed && m.place(key_value(key_in(mine))) < (float)rec.bin) {
      listed = false;
      const double e = m.e(key_in(mine));
      if (e >= min_e) atomicAdd(&sums[(index_of(mine) + r.lead) / kSpan - part.first * kRowWaves], m.fixed(e));
    }
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    int at = 0;
    if (listed) at = atomicAdd(&s_n, 1);
    __syncthreads();
    if (listed) list[at] = mine;
    __syncthreads();
  }
  const int out = min(s_n, kList);
  if (tid == 0 && out) s_at = atomicAdd(&w.listed[row], out);
  __syncthreads();
  if (tid < out && s_at + tid < kList) w.list[(size_t)row * kList + s_at + tid] = list[tid];
  if (rec.mode != kAllListed)
    for (int i = tid; i < spans; i += kRowThreads)
      w.sums[((size_t)row * w.chunks + part.first) * kRowWaves + i] = sums[i];
}

// The value of lane (this ^ GAP), by moves between lanes where the hardware has one: within four
// lanes, rotation by half a row of 16, swaps of rows and of half waves.
template <int GAP>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (GAP == 1) return __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false);
  if constexpr (GAP == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false);
  if constexpr (GAP == 4) {  // mirrored in eight lanes, then in four
    const uint32_t m = __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false);
    return __builtin_amdgcn_update_dpp(0, m, 0x1b, 0xf, 0xf, false);
  }
  if constexpr (GAP == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);
  if constexpr (GAP == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  if constexpr (GAP == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int GAP>
__device__ __forceinline__ u64 lane_xor(u64 v) {
  return (u64)lane_xor<GAP>((uint32_t)v) | (u64)lane_xor<GAP>((uint32_t)(v >> 32)) << 32;
}

// Waves that hold the first n of a block's values, one per thread, as a power of two.
__device__ __forceinline__ int waves_for(int n) {
  int waves = 1;
  while (64 * waves < n) waves *= 2;
  return waves;
}

// Sorts the values of the block's first `waves` waves, one per thread: descending by thread.  A bitonic
// network; the waves beyond keep to the barriers.
__device__ __forceinline__ u64 sort_descending(u64 v, int waves, u64* lds) {
  const int tid = threadIdx.x;
  const bool part = __builtin_amdgcn_readfirstlane(tid >> 6) < waves;
  int width;
  auto take = [&](u64 o, int gap) {
    const bool larger = ((tid & gap) == 0) == ((tid & width) == 0);
    v = (o > v) == larger ? o : v;
  };
  for (width = 2; width <= 64 * waves; width *= 2) {
    for (int gap = width / 2; gap >= 64; gap /= 2) {
      __syncthreads();
      if (part) lds[tid] = v;
      __syncthreads();
      if (part) take(lds[tid ^ gap], gap);
    }
    if (!part) continue;
    if (width >= 64) take(lane_xor<32>(v), 32);
    if (width >= 32) take(lane_xor<16>(v), 16);
    if (width >= 16) take(lane_xor<8>(v), 8);
    if (width >= 8) take(lane_xor<4>(v), 4);
    if (width >= 4) take(lane_xor<2>(v), 2);
    take(lane_xor<1>(v), 1);
  }
  return v;
}

// block_before for values of the first `waves` waves; the others get nothing but the total.
__device__ __forceinline__ u64 first_before(u64 v, int waves, u64* slots, u64* total) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u64 upto = 0;
  if (wave < waves) {
    upto = wave_upto(v);
    if (lane == 63) slots[wave] = upto;
  }
  __syncthreads();
  const u64 all = wave_upto(lane < waves ? slots[lane] : 0);
  *total = lane_of(all, 63);
  return (wave && wave < waves ? lane_of(all, wave - 1) : 0) + upto - v;
}

// One workgroup per row: the last kept token of the list, then the draw.  SMALL: a vocabulary that fits
// the list, in this launch alone.  Bound by latency, 7 to 14 us of one step after another, so waves without
// a value skip what only the others need.
template <bool BF16, bool SMALL>
__global__ __launch_bounds__(kRowThreads) void sample_draw_kernel(SampleArgs a, Work w,
                                                                  double scale) {
  __shared__ union {
    RowLds radix;
    struct {
      u64 list[kList];
      u64 sums[kMaxSpans];
      u64 slots[4][kRowWaves];  // one per exchange: none is written again while a wave may still read it
    } s;
  } lds;
  __shared__ int s_n, s_found;
  __shared__ u64 s_cut, s_before;
  __shared__ double powers[kPowers];
  const int row = blockIdx.x, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RowParams p = row_params(a, row);
  const Row<BF16> r(a, row);
  RowRecord rec{};
  int n = 0;
  u64 mine = 0;
  if constexpr (!SMALL) {
    rec = w.record[row];
    n = min(w.listed[row], kList);
    mine = w.list[(size_t)row * kList + tid];
  }
  fill_powers(powers);
  if (tid == 0) s_n = 0;
  __syncthreads();
  if constexpr (SMALL) {
    const u64 v = tid < r.V ? order_of(load_logit<BF16>(r.base, tid), tid) : 0;
    if (key_in(v) > kMinusInf) {
      rec.best = v;
      lds.s.list[atomicAdd(&s_n, 1)] = v;
    }
    rec.best = block_max(rec.best, lds.s.slots[3]);
    rec.mode = kAllListed;
    n = s_n;
    mine = lds.s.list[tid];
  }
  auto done = [&](int id, float prob) {
    if (tid == 0) {
      a.ids[row] = id;
      if (a.probs) a.probs[row] = prob;
    }
  };
  if (trivial(p, rec.best)) {
    if (!p.ok && tid == 0) flag(a.status, kStepArgument);
    const bool greedy = p.ok && key_in(rec.best) > kMinusInf;
    done(greedy ? index_of(rec.best) : -1, greedy ? 1.0f : 0.0f);
    return;
  }
  const Mass m(key_in(rec.best), p.tau, scale, powers);
  const double min_e = (double)p.min_p, uniform = (double)p.uniform;
  if constexpr (!SMALL) {
    if (rec.mode == kByRadix) {
      u64 total;
      const int id = draw_by_radix<BF16>(r.base, r.V, p, m, lds.radix, &total);
      done(id, (float)(m.e(load_logit<BF16>(r.base, id)) / ((double)total / scale)));
      return;
    }
  }
  if (tid >= n) mine = 0;
  const int spans = SMALL ? (kList + 7 + kSpan - 1) / kSpan : w.chunks * kRowWaves;
  for (int i = tid; i < spans; i += kRowThreads)
    lds.s.sums[i] =
        rec.mode == kAllListed ? 0 : w.sums[(size_t)row * w.chunks * kRowWaves + i];
  // Kept are the valid tokens not after the cut in order, of e >= min_p: the cut is the list's last
  // kept one.  (None of the list, because of min_p: then those of the bins before it, as far as min_p
  // keeps them.)  The list's kept tokens are added to their spans' sums.
  u64 cut = 0;
  if (rec.mode != kNoCut) {
    const int waves = waves_for(n);
    mine = sort_descending(mine, waves, lds.s.list);
    const bool by_count = p.top_k > 0 && p.top_k < r.V;
    // (with every kept token in the list nothing comes before it)
    const bool part = rec.mode == kBinListed;
    const int most = by_count ? min(n, p.top_k - (part ? rec.above_n : 0)) : n;
    double e = 0.0;
    u64 f = 0;
    if (tid < most) {
      e = m.e(key_in(mine));
      f = m.fixed(e);
    }
    u64 all;
    const u64 run = (part ? rec.above : 0) + first_before(f, waves, lds.s.slots[0], &all);
    u64 want = ~0ull;
    if (p.top_p < 1.0f) want = SMALL || by_count ? mass_wanted(p.top_p, all) : rec.want;
    // (with equal logits e >= min_p holds for all or none, so the kept ones stay a beginning)
    const bool keep = tid < most && run < want && e >= min_e;
    const int kept = __syncthreads_count(keep);
    if (keep) atomicAdd(&lds.s.sums[(index_of(mine) + r.lead) / kSpan], f);
    if (kept == 0 && tid == 0) s_cut = ~0ull;
    if (keep && tid == kept - 1) s_cut = mine;
  }
  __syncthreads();
  if (rec.mode != kNoCut) cut = s_cut;
  // the span of the draw: up to three per thread, in order
  const int per = (spans + kRowThreads - 1) / kRowThreads;
  const int span_waves = (spans + 64 * per - 1) / (64 * per);
  u64 own[3] = {}, sum = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    const int i = tid * per + j;
    if (j < per && i < spans) own[j] = lds.s.sums[i];
    sum += own[j];
  }
  u64 total;
  u64 before = first_before(sum, span_waves, lds.s.slots[1], &total);
  const double target = uniform * (double)total;
  if (!((double)before > target) && (double)(before + sum) > target) {
    int j = 0;
    if (!((double)(before + own[0]) > target)) {
      before += own[0];
      j = 1;
      if (!((double)(before + own[1]) > target)) {
        before += own[1];
        j = 2;
      }
    }
    s_found = tid * per + j;
    s_before = before;
  }
  __syncthreads();
  // the draw in it, a value per thread
  u64 f = 0;
  double e = 0.0;
  const int i = s_found * kSpan + tid - r.lead;
  if (tid < kSpan && i >= 0 && i < r.V) {
    const float l = load_logit<BF16>(r.base, i);
    // (a whole list has a cut: its first token is kept)
    const float z = SMALL ? 0.0f : m.place(l);
    if (z < (float)(kBins - 1) && (cut == ~0ull ? z < (float)rec.bin : order_of(l, i) >= cut)) {
      e = m.e(l);
      if (e >= min_e) f = m.fixed(e);
    }
  }
  u64 all;
  const u64 run = s_before + first_before(f, kSpan / 64, lds.s.slots[2], &all);
  if (wave < kSpan / 64 && !((double)run > target) && (double)(run + f) > target) {
    a.ids[row] = i;
    if (a.probs) a.probs[row] = (float)(e / ((double)total / scale));
  }
}

// Workgroups of a launch that shares rows, about: enough that rows which cost more than others are spread
// over the chip, few enough that the histograms they add up do not take over (256 rows of 129280: 122.6 us;
// with 2048 for all but the histograms 125.4, with 4096 137; with 512 or 2048 for the histograms 130).
constexpr int kParts = 1024;
size_t row_bytes(int chunks) {
  return (size_t)chunks * 8 * (1 + kRowWaves) + kAllBins * 12 + kList * 8 + sizeof(RowRecord) + 4;
}
// (a row may start up to 7 values past a 16-byte boundary)
int row_chunks(int vocab) { return (vocab + 7 + kChunk - 1) / kChunk; }

template <bool BF16>
void launch_rows(const SampleArgs& a, const Work& w, double scale, hipStream_t s) {
  if (a.vocab <= kList) {
    sample_draw_kernel<BF16, true><<<a.rows, kRowThreads, 0, s>>>(a, w, scale);
    return;
  }
  const dim3 grid(w.parts, a.rows);
  sample_best_kernel<BF16><<<grid, kRowThreads, 0, s>>>(a, w);
  sample_bins_kernel<BF16><<<grid, kRowThreads, 0, s>>>(a, w, scale);
  sample_list_kernel<BF16><<<grid, kRowThreads, 0, s>>>(a, w, scale);
  sample_draw_kernel<BF16, false><<<a.rows, kRowThreads, 0, s>>>(a, w, scale);
}

}  // namespace

size_t sample_work_bytes(int vocab, int rows) {
  return vocab <= kList ? 0 : (size_t)std::min(rows, kSamplePass) * row_bytes(row_chunks(vocab));
}

void launch_sample(const SampleArgs& a, bool bf16, hipStream_t s) {
  int log = 0;
  while ((1 << log) < a.vocab) ++log;
  const double scale = (double)(1ull << std::min(51, 62 - log));
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
      w.chunks = row_chunks(a.vocab);
      w.parts = std::min(w.chunks, std::max(1, kParts / p.rows));
      const size_t rows = p.rows, most = w.chunks;
      char* at = static_cast<char*>(a.work);
      auto take = [&](auto** q, size_t n) {
        *q = reinterpret_cast<std::remove_reference_t<decltype(*q)>>(at);
        at += n * sizeof(**q);
      };
      take(&w.best, rows * most);
      take(&w.sums, rows * most * kRowWaves);
      take(&w.mass, rows * kAllBins);
      take(&w.list, rows * kList);
      take(&w.record, rows);
      take(&w.count, rows * kAllBins);
      take(&w.listed, rows);
    }
    if (bf16) launch_rows<true>(p, w, scale, s);
    else launch_rows<false>(p, w, scale, s);
  }
}

}  // namespace urb
