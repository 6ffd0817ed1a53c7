// urb_sample.hip -- drawing a token per row of logits under temperature, top-k, top-p and min-p.
//
// All three filters keep a beginning of one order (logit descending, index ascending), so a row's
// kept tokens are those above a threshold logit plus the first few of those equal to it, and no row
// is ever sorted.  Logits are compared as 32-bit keys in their order; masses e = exp((l - m) / tau) are
// computed in f64 and summed as integers of 2^-shift (shift 42 to 61, by the vocabulary), so sums do not depend
// on their order and a row's result is the same whatever workgroups share it.
#include "urb_device.hpp"
#include "urb_step.hpp"

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

// e of a logit key, and e as an integer.
struct Mass {
  double top, tau, scale;  // largest logit, temperature, 2^shift
  uint32_t top_key;
  __device__ __forceinline__ double e(uint32_t key) const {
    if (key == top_key) return 1.0;  // also where both are +inf
    return exp(((double)key_value(key) - top) / tau);
  }
  __device__ __forceinline__ u64 fixed(double e) const { return (u64)(e * scale + 0.5); }
};

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
template <class T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  T s = 0;
  for (int w = 0; w < kRowWaves; ++w) s += slots[w];
  return s;
}
// Sum over the threads before this one; *total over all.
template <class T>
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
  for (int w = 0; w < kRowWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += slots[w];
    all += slots[w];
  }
  *total = all;
  return before + inc - v;
}

constexpr int kBins = 2048;

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

// One workgroup per row, whatever the row holds: the thresholds by radix selection over the keys.
template <bool BF16>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a, double scale) {
  __shared__ u64 hist[kBins];
  __shared__ u64 slots[kRowWaves];
  __shared__ int islots[kRowWaves];
  const int row = blockIdx.x, tid = threadIdx.x;
  const int V = a.vocab;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(a.logits) +
                        (size_t)row * a.row_stride * (BF16 ? 2 : 4);
  auto key = [&](int i) { return key_of(load_logit<BF16>(base, i)); };
  const RowParams p = row_params(a, row);
  auto done = [&](int id, float prob) {
    if (tid == 0) {
      a.ids[row] = id;
      if (a.probs) a.probs[row] = prob;
    }
  };
  if (!p.ok) {
    if (tid == 0) flag(a.status, kStepArgument);
    done(-1, 0.0f);
    return;
  }
  // the largest key and its lowest index, as one number
  u64 best = 0;
  for (int i = tid; i < V; i += kRowThreads) {
    const u64 c = ((u64)key(i) << 32) | (uint32_t)(V - 1 - i);
    best = c > best ? c : best;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const u64 c = __shfl_xor(best, o, 64);
    best = c > best ? c : best;
  }
  if ((tid & 63) == 0) slots[tid >> 6] = best;
  __syncthreads();
  for (int w = 0; w < kRowWaves; ++w) best = slots[w] > best ? slots[w] : best;
  __syncthreads();
  const uint32_t top_key = (uint32_t)(best >> 32);
  if (top_key <= kMinusInf) {
    done(-1, 0.0f);
    return;
  }
  if (p.tau == 0.0f) {
    done(V - 1 - (int)(uint32_t)best, 1.0f);
    return;
  }
  const Mass mass{(double)key_value(top_key), (double)p.tau, scale, top_key};

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
  __shared__ int found;
  if (tid == 0) found = -1;
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
      if (!((double)run > target) && (double)(run + w[u]) > target) found = i0 + tid * PER + u;
      run += w[u];
    }
    before += tile;
    if ((double)before > target) break;  // the same in all threads
  }
  __syncthreads();
  const int id = found;
  float prob = 0.0f;
  if (id >= 0) prob = (float)(mass.e(key(id)) / ((double)total / scale));
  done(id, prob);
}

}  // namespace

void launch_sample(const SampleArgs& a, bool bf16, hipStream_t s) {
  int log = 0;
  while ((1 << log) < a.vocab) ++log;
  const double scale = (double)(1ull << (62 - (log < 1 ? 1 : log)));
  if (bf16) sample_row_kernel<true><<<a.rows, kRowThreads, 0, s>>>(a, scale);
  else sample_row_kernel<false><<<a.rows, kRowThreads, 0, s>>>(a, scale);
}

}  // namespace urb
