// urb_beam.hip -- beam search's selection: the best of width * vocab candidates of each request.
//
// The logits are read once.  A workgroup takes a slice of a beam's row: its largest logit and the sum of
// exp(l - m) in f64 (two candidates of different beams are told apart by the logarithms of such sums), and its
// best `picks` logits, for more cannot be taken from one beam.  They are found with a threshold: the
// picks-th largest of the threads' own largest is no more than the picks-th largest of all, and few others
// lie above it.  The second kernel joins a request's slices the same way over their candidates' scores.
#include "urb_device.hpp"
#include "urb_step.hpp"

#include <algorithm>

namespace urb {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kJoinThreads = 1024;

// Order-preserving key of a logit: NaN and -inf, which are never picked, 0; -0 as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -__builtin_inff())) return 0;
  const uint32_t b = f2u(l + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return u2f(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

}  // namespace

struct BeamSum {
  double z;  // of exp(l - m)
  float m;
  int pad;
};

namespace {

// Four neighbours of a row from i on; those past the end are -inf.
template <bool BF16>
__device__ __forceinline__ void load4(float (&v)[4], const uint8_t* row, int i, int vocab, bool wide) {
  if (wide && i + 4 <= vocab) {
    if constexpr (BF16) {
      const uint2 q = *reinterpret_cast<const uint2*>(row + 2 * (size_t)i);
      v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
    } else {
      const float4 q = u2f4(ldg16(row + 4 * (size_t)i));
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = -__builtin_inff();
    if (i + j < vocab) {
      if constexpr (BF16) v[j] = u2f((uint32_t)reinterpret_cast<const uint16_t*>(row)[i + j] << 16);
      else v[j] = reinterpret_cast<const float*>(row)[i + j];
    }
  }
}

// exp(l - m) for l <= m, 1 where both are +inf.
__device__ __forceinline__ double mass(float l, float m) {
  if (l == m) return 1.0;
  if (!(l > -__builtin_inff())) return 0.0;
  return exp((double)l - (double)m);
}

// A workgroup per slice and beam.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(BeamArgs a) {
  constexpr int PER = kBeamSlice / kThreads;
  __shared__ u64 best[kThreads];
  __shared__ u64 list[kBeamPicks * PER];
  __shared__ double s_z[kThreads / 64];
  __shared__ u64 s_key[kThreads / 64];
  __shared__ int n_list;
  __shared__ u64 s_least;
  const int slice = blockIdx.x, beam = blockIdx.y, tid = threadIdx.x;
  if (a.ended && a.ended[beam]) return;  // its logits count for nothing
  const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + beam * a.row_stride * (BF16 ? 2 : 4);
  const bool wide = reinterpret_cast<uintptr_t>(row) % (BF16 ? 8 : 16) == 0;
  const int base = slice * kBeamSlice + 4 * tid;
  float v[PER / 4][4];
#pragma unroll
  for (int k = 0; k < PER / 4; ++k) load4<BF16>(v[k], row, base + k * 4 * kThreads, a.vocab, wide);
  // keys: the larger logit, then the lower index
  u64 top = 0;
#pragma unroll
  for (int k = 0; k < PER / 4; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = key_of(v[k][j]);
      const uint32_t at = (uint32_t)(base + k * 4 * kThreads + j);
      const u64 both = (u64)key << 32 | (uint32_t)~at;
      if (key && both > top) top = both;
    }
  best[tid] = top;
  u64 most = top;
  for (int o = 32; o > 0; o >>= 1) most = max(most, (u64)__shfl_xor((long long)most, o, 64));
  if ((tid & 63) == 0) s_key[tid >> 6] = most;
  if (tid == 0) {
    n_list = 0;
    s_least = 0;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = max(most, s_key[w]);
  const bool any = most != 0;
  const float m = any ? key_value((uint32_t)(most >> 32)) : -__builtin_inff();
  double z = 0.0;
  if (any)
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) z += mass(v[k][j], m);
  for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
  if ((tid & 63) == 0) s_z[tid >> 6] = z;
  // the picks-th largest of the threads' best
  if (top) {
    int above = 0;
    for (int i = 0; i < kThreads; ++i) above += best[i] > top;
    if (above == a.picks - 1) s_least = top;
  }
  __syncthreads();
  const u64 least = s_least;  // 0: fewer threads than that have any
#pragma unroll
  for (int k = 0; k < PER / 4; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = key_of(v[k][j]);
      const uint32_t at = (uint32_t)(base + k * 4 * kThreads + j);
      const u64 both = (u64)key << 32 | (uint32_t)~at;
      if (key && both >= least) list[atomicAdd(&n_list, 1)] = both;
    }
  __syncthreads();
  const int n = n_list;
  u64* out = a.keys + ((size_t)beam * a.slices + slice) * a.picks;
  for (int i = tid; i < n; i += kThreads) {
    const u64 mine = list[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += list[j] > mine;
    if (above < a.picks) out[above] = mine;
  }
  for (int i = n + tid; i < a.picks; i += kThreads) out[i] = 0;
  if (tid == 0) {
    double sum = 0.0;
    for (int w = 0; w < kThreads / 64; ++w) sum += s_z[w];
    a.sums[(size_t)beam * a.slices + slice] = BeamSum{sum, m, 0};
  }
}

struct Candidate {
  double score;
  uint32_t at;  // beam * vocab + token
};
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) {
  return x.score > y.score || (x.score == y.score && x.at < y.at);
}

// A workgroup per request; a thread per slice of a beam, whose candidates are in order.
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a) {
  __shared__ Candidate head[kJoinThreads];
  __shared__ Candidate list[kBeamPicks * kBeamPicks];
  __shared__ double s_base[kBeamWidth];  // score and logarithm of a beam: what a logit - m is added to
  __shared__ float s_top[kBeamWidth];
  __shared__ int s_live[kBeamWidth];     // 0: no candidates, 1: its slices', 2: ended
  __shared__ int n_list, s_bad;
  __shared__ Candidate s_least;
  const int r = blockIdx.x, tid = threadIdx.x, width = a.width;
  if (tid == 0) {
    n_list = 0;
    s_bad = 0;
    s_least = Candidate{-__builtin_inf(), 0xffffffffu};
  }
  __syncthreads();
  // (a wave per beam in turn)
  for (int b = tid >> 6; b < width; b += kJoinThreads / 64) {
    const int lane = tid & 63, beam = r * width + b;
    const float c = a.scores[beam];
    const bool end = a.ended && a.ended[beam];
    float m = -__builtin_inff();
    double z = 0.0;
    if (!end) {
      const BeamSum* sums = a.sums + (size_t)beam * a.slices;
      const BeamSum mine = lane < a.slices ? sums[lane] : BeamSum{0.0, -__builtin_inff(), 0};
      m = mine.m;
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      z = mine.z * mass(mine.m, m);
      for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
    }
    if (lane == 0) {
      const bool bad = !(c <= 3.4028235e38f);  // NaN, +inf
      if (bad) s_bad = 1;
      const bool live = !bad && c > -__builtin_inff();
      s_live[b] = !live ? 0 : end ? 2 : m > -__builtin_inff() ? 1 : 0;
      s_top[b] = m;
      s_base[b] = end ? (double)c : (double)c - log(z);
    }
  }
  __syncthreads();
  // this thread's list
  const int b = tid / a.slices, slice = tid - b * a.slices;
  const bool mine = b < width && (s_live[b] == 1 || (s_live[b] == 2 && slice == 0));
  const u64* keys = a.keys + ((size_t)(r * width + b) * a.slices + slice) * a.picks;
  auto candidate = [&](int i) -> Candidate {
    const Candidate none{-__builtin_inf(), 0xffffffffu};
    if (s_live[b] == 2)
      return i == 0 ? Candidate{s_base[b], (uint32_t)b * a.vocab + a.end_token} : none;
    const u64 key = keys[i];
    if (!key) return none;
    const float l = key_value((uint32_t)(key >> 32));
    const double gap = l == s_top[b] ? 0.0 : (double)l - (double)s_top[b];
    const double score = s_base[b] + gap;
    return score > -__builtin_inf() ? Candidate{score, (uint32_t)b * a.vocab + ~(uint32_t)key} : none;
  };
  Candidate first{-__builtin_inf(), 0xffffffffu};
  if (mine) first = candidate(0);
  head[tid] = first;
  __syncthreads();
  const int lists = width * a.slices;
  if (first.at != 0xffffffffu) {
    int above = 0;
    for (int i = 0; i < lists; ++i) above += better(head[i], first);
    if (above == a.picks - 1) s_least = first;
  }
  __syncthreads();
  const Candidate least = s_least;
  if (first.at != 0xffffffffu)
    for (int i = 0; i < a.picks; ++i) {
      const Candidate c = i ? candidate(i) : first;
      if (c.at == 0xffffffffu || better(least, c)) break;
      list[atomicAdd(&n_list, 1)] = c;
    }
  __syncthreads();
  const int n = n_list;
  const size_t out = (size_t)r * a.picks;
  for (int i = tid; i < n; i += kJoinThreads) {
    const Candidate c = list[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += better(list[j], c);
    if (above < a.picks) {
      const int parent = (int)(c.at / (uint32_t)a.vocab);
      const int token = (int)(c.at - (uint32_t)parent * a.vocab);
      a.scores_out[out + above] = (float)c.score;
      a.tokens[out + above] = token;
      a.parents[out + above] = parent;
      if (a.ended_out) a.ended_out[out + above] = s_live[parent] == 2 || token == a.end_token;
    }
  }
  for (int i = n + tid; i < a.picks; i += kJoinThreads) {
    a.scores_out[out + i] = -__builtin_inff();
    a.tokens[out + i] = -1;
    a.parents[out + i] = -1;
    if (a.ended_out) a.ended_out[out + i] = 1;
  }
  if (tid == 0 && s_bad) flag(a.status, kStepArgument);
}

size_t keys_bytes(int vocab, int width, int picks, int requests) {
  return (size_t)requests * width * beam_slices(vocab) * picks * sizeof(u64);
}

}  // namespace

size_t beam_work_bytes(int vocab, int width, int picks, int requests) {
  return keys_bytes(vocab, width, picks, requests) +
         (size_t)requests * width * beam_slices(vocab) * sizeof(BeamSum);
}

void launch_beam(BeamArgs a, bool bf16, int max_requests, void* work, hipStream_t s) {
  a.slices = beam_slices(a.vocab);
  a.keys = static_cast<u64*>(work);
  a.sums = reinterpret_cast<BeamSum*>(static_cast<char*>(work) +
                                      keys_bytes(a.vocab, a.width, a.picks, max_requests));
  // requests of a launch: blockIdx.y is below 2^16
  const int most = 65535 / a.width;
  for (int r = 0; r < a.requests; r += most) {
    BeamArgs c = a;
    c.requests = std::min(most, a.requests - r);
    const size_t beams = (size_t)r * a.width, picks = (size_t)r * a.picks;
    c.logits = static_cast<const char*>(a.logits) + beams * a.row_stride * (bf16 ? 2 : 4);
    c.scores += beams;
    if (a.ended) c.ended += beams;
    c.scores_out += picks;
    c.tokens += picks;
    c.parents += picks;
    if (a.ended_out) c.ended_out += picks;
    c.keys += beams * a.slices * a.picks;
    c.sums += beams * a.slices;
    const dim3 grid(a.slices, c.requests * a.width);
    if (bf16) beam_slice_kernel<true><<<grid, kThreads, 0, s>>>(c);
    else beam_slice_kernel<false><<<grid, kThreads, 0, s>>>(c);
    beam_join_kernel<<<c.requests, kJoinThreads, 0, s>>>(c);
  }
}

}  // namespace urb
