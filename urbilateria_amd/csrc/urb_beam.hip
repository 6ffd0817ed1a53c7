// urb_beam.hip -- beam search's selection: the best of width * vocab candidates of each request.
//
// The logits are read once.  A workgroup takes a slice of a beam's row: its largest logit and the sum of
// exp(l - m) in f64 (two candidates of different beams are told apart by the logarithms of such sums), and its
// best `picks` logits, for more cannot be taken from one beam.  They are found with a threshold: the
// picks-th largest of the threads' own largest is no more than the picks-th largest of all, and few others
// lie above it.  The second kernel joins a request's slices the same way over their candidates' scores.
// 256 rows of 129280 f32 logits (132 MB) take 39 us, bound by the vector units, which are busy for 78 % of it (an
// exponential in f64 for each; LDS, with its table, for 23 %); the second kernel 8 to 13 for 32 requests, latency of
// its steps; 4 rows of 50257 take 6 and 5.
#include "urb_device.hpp"
#include "urb_step.hpp"

#include <algorithm>

namespace urb {

struct BeamSum {
  double z;  // of exp(l - m)
  float m;
  int pad;
};

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr float kInf = __builtin_inff();

// Order-preserving key of a logit: NaN and -inf, which are never picked, 0; -0 as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -kInf)) return 0;
  const uint32_t b = f2u(l + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return u2f(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// A logit's key and its index: the larger logit, then the lower index.
__device__ __forceinline__ u64 with_index(uint32_t key, int at) {
  return (u64)key << 32 | (uint32_t)~at;
}

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
    v[j] = -kInf;
    if (i + j < vocab) {
      if constexpr (BF16) v[j] = u2f((uint32_t)reinterpret_cast<const uint16_t*>(row)[i + j] << 16);
      else v[j] = reinterpret_cast<const float*>(row)[i + j];
    }
  }
}

// z + exp(l - m) for l <= m finite: l - m = n ln 2 / 64 + r with |r| <= ln(2) / 128, 2^(n / 64) by a table in LDS
// and the Taylor series to r^4, which leaves out 4e-14 of it.  Logits far below, of -inf and NaN count as
// exp(-60): all the vocabulary's together are no 2^-50 of the largest's 1.
constexpr int kPowers = 64;
__device__ __forceinline__ void fill_powers(double* powers) {
  if (threadIdx.x < kPowers) powers[threadIdx.x] = exp2((double)threadIdx.x / kPowers);
}
__device__ __forceinline__ double add_mass(double z, float l, double m, const double* powers) {
  const double x = fmax((double)l - m, -60.0);
  const double magic = 0x1.8p52;  // adding it leaves an integer in the low bits
  const double t = fma(x, 0x1.71547652b82fep+6, magic);  // 64 / ln 2
  const int n = (int)__double_as_longlong(t);
  const double r = fma(magic - t, 0x1.62e42fefa39efp-7, x);
  double s = fma(1.0 / 24.0, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  // the table's value times 2^(n / 64): a sum in its exponent
  const long long p = __double_as_longlong(powers[n & (kPowers - 1)]) + ((long long)(n >> 6) << 52);
  const double q = __longlong_as_double(p);
  return fma(q, fma(s, r, 1.0), z);
}

// The upper half of the n-th largest key of a wave's lanes; 0 where fewer lanes have one.
__device__ __forceinline__ uint32_t wave_nth(uint32_t key, int n) {
  uint32_t t = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit > 0xffffu; bit >>= 1)
    if (__popcll(__ballot(key >= (t | bit))) >= n) t |= bit;
  return t;
}

// Calls with(item, how many of list[0 .. n - 1] are before it) for every item, in a lane 0: a wave per item in
// turn, a lane for each of the others.
template <int WAVES, class T, class Before, class With>
__device__ __forceinline__ void rank_all(const T* list, int n, Before before, With with) {
  const int lane = threadIdx.x & 63;
  T others = lane < n ? list[lane] : T{};
#pragma unroll 2
  for (int i = threadIdx.x >> 6; i < n; i += WAVES) {
    const T mine = list[i];
    int above = __popcll(__ballot(lane < n && before(others, mine)));
    for (int j = 64 + lane; j - lane < n; j += 64) above += __popcll(__ballot(j < n && before(list[j], mine)));
    if (lane == 0) with(mine, above);
  }
}

// A workgroup per slice (of PER logits per thread) and beam.
template <bool BF16, int PER>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(BeamArgs a) {
  constexpr int WAVES = kThreads / 64;
  __shared__ double powers[kPowers];
  __shared__ u64 list[kBeamPicks * PER > kThreads ? kBeamPicks * PER : kThreads];
  __shared__ double s_z[WAVES];
  __shared__ float s_top[WAVES];
  __shared__ uint32_t s_nth[WAVES];
  __shared__ int n_heads, n_list;
  __shared__ u64 s_least;
  const int slice = blockIdx.x, beam = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
  if (a.ended && a.ended[beam]) return;  // its logits count for nothing
  const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + beam * a.row_stride * (BF16 ? 2 : 4);
  const bool wide = reinterpret_cast<uintptr_t>(row) % (BF16 ? 8 : 16) == 0;
  const int base = slice * (PER * kThreads) + 4 * tid, item = beam * a.slices + slice;
  auto index = [&](int k, int j) { return base + k * 4 * kThreads + j; };
  float v[PER / 4][4];
#pragma unroll
  for (int k = 0; k < PER / 4; ++k) load4<BF16>(v[k], row, index(k, 0), a.vocab, wide);
  fill_powers(powers);
  if (tid == 0) {
    n_heads = n_list = 0;
    s_least = 0;
  }
  // the largest of the thread (fmaxf passes NaNs over) and of the slice
  float top = -kInf;
#pragma unroll
  for (int k = 0; k < PER / 4; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, v[k][j]);
  const uint32_t key = key_of(top);
  float m = top;
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const uint32_t nth = wave_nth(key, (a.picks + WAVES - 1) / WAVES);
  if ((tid & 63) == 0) {
    s_top[wave] = m;
    s_nth[wave] = nth;
  }
  __syncthreads();
  // What every wave has its part of `picks` above is a bound (32 x 8 beams of 129280 logits take 49 us with it and
  // 50.6 with the picks-th of one wave, 16 x 32 with 64 picks 299 and 412); among the few bests that reach it,
  // the picks-th itself is found by counting.
  uint32_t bound = s_nth[0];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    m = fmaxf(m, s_top[w]);
    bound = min(bound, s_nth[w]);
  }
  const bool head = key && key >= bound;
  u64 best = 0;  // the thread's, if it is among them: the first of equal ones
  if (head) {
    int at = 0;
#pragma unroll
    for (int k = PER / 4; k-- > 0;)
#pragma unroll
      for (int j = 4; j-- > 0;)
        if (v[k][j] == top) at = index(k, j);
    best = with_index(key, at);
    list[atomicAdd(&n_heads, 1)] = best;
  }
  double z = 0.0;
  if (m == kInf) {  // as many as there are of it share all
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) z += v[k][j] == kInf ? 1.0 : 0.0;
  } else if (m > -kInf) {
    const double md = (double)m;
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) z = add_mass(z, v[k][j], md, powers);
  }
  for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
  if ((tid & 63) == 0) s_z[wave] = z;
  __syncthreads();
  auto above = [](u64 x, u64 y) { return x > y; };
  rank_all<WAVES>(list, n_heads, above, [&](u64 x, int n) {
    if (n == a.picks - 1) s_least = x;
  });
  __syncthreads();
  const u64 least = s_least;  // 0: fewer threads than that have any
  const float least_value = least ? key_value((uint32_t)(least >> 32)) : -kInf;
  if (head && best >= least)  // (others have nothing that does)
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[k][j] >= least_value) {
          const uint32_t one = key_of(v[k][j]);
          const u64 both = with_index(one, index(k, j));
          if (one && both >= least) list[atomicAdd(&n_list, 1)] = both;
        }
  __syncthreads();
  const int n = n_list;
  u64* out = a.keys + (size_t)item * a.picks;
  rank_all<WAVES>(list, n, above, [&](u64 x, int place) {
    if (place < a.picks) out[place] = x;
  });
  for (int i = n + tid; i < a.picks; i += kThreads) out[i] = 0;
  if (tid == 0) {
    double sum = 0.0;
    for (int w = 0; w < WAVES; ++w) sum += s_z[w];
    a.sums[item] = BeamSum{sum, m, 0};
  }
}

struct Candidate {
  double score;
  uint32_t at;   // beam << kTokenBits | token
  uint32_t key;  // of its logit
};
constexpr int kTokenBits = 18;
static_assert(kBeamVocab <= 1 << kTokenBits && kBeamWidth < 1 << (31 - kTokenBits), "beam and token in 32 bits");
constexpr uint32_t kNone = 0xffffffffu;
// The order of the picks.
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) {
  return x.score > y.score || (x.score == y.score && x.at < y.at);
}
// The order that the lists are in: a beam's candidates of one score by their logits first, which may differ in less
// than a score shows.
__device__ __forceinline__ bool ahead(const Candidate& x, const Candidate& y) {
  if (x.score != y.score) return x.score > y.score;
  return (x.at ^ y.at) >> kTokenBits || x.key == y.key ? x.at < y.at : x.key > y.key;
}

// What a beam's logits are scored with: c + ((l - m) - log z).
struct Scored {
  double c, log_z;
  float m;
  __device__ __forceinline__ double of(float v) const {
    return c + ((v == m ? 0.0 : (double)v - (double)m) - log_z);
  }
  // Logits above this in size have scores of their own: they lie 2^-24 of their size apart, and the three roundings of
  // two scores are off by less than 2^-52 (3 |v| + 3 |m| + |c| + 26), log z being below 13.
  __device__ __forceinline__ float own_scores() const {
    return (float)((fabs(c) + fabs((double)m) + 32.0) * 0x1p-25);
  }
  // whether a logit next to this one has its score too
  __device__ __forceinline__ bool shared(uint32_t key) const {
    const float v = key_value(key);
    const double score = of(v);
    return of(key_value(key - 1)) == score || (v < m && of(key_value(key + 1)) == score);
  }
};

// The picks from place `from` on: the lowest tokens of beam b with this score, of its row of logits.  All threads.
template <int THREADS>
__device__ __forceinline__ void pick_lowest(const BeamArgs& a, int r, int b, const Scored& beam, double score, int from,
                                            uint32_t* counts) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t size = a.bf16 ? 2 : 4, out = (size_t)r * a.picks;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + (r * a.width + b) * a.row_stride * size;
  const bool wide = reinterpret_cast<uintptr_t>(row) % (4 * size) == 0;
  for (int i0 = 0; i0 < a.vocab && from < a.picks; i0 += 4 * THREADS) {
    const int i = i0 + 4 * tid;
    float v[4];
    if (a.bf16) load4<true>(v, row, i, a.vocab, wide);
    else load4<false>(v, row, i, a.vocab, wide);
    bool hit[4];
    int before = 0, mine = 0, all = 0;  // of lower lanes, of this, of the wave
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hit[j] = beam.of(v[j]) == score;
      const uint64_t hits = __ballot(hit[j]);
      before += __popcll(hits & ((1ull << lane) - 1));
      all += __popcll(hits);
      mine += hit[j];
    }
    __syncthreads();
    if (lane == 0) counts[wave] = (uint32_t)all;
    __syncthreads();
    int place = from + before;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) place += (int)counts[w];
      from += (int)counts[w];
    }
    if (mine == 0) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (hit[j] && place < a.picks) {
        a.scores_out[out + place] = (float)score;
        a.tokens[out + place] = i + j;
        a.parents[out + place] = b;
        if (a.ended_out) a.ended_out[out + place] = i + j == a.end_token;
        ++place;
      }
  }
}

// A workgroup per request; each slice of each of its beams is a list in order.  `span` lists (a power of two)
// are counted for a beam, `team` threads go through a list.
//
// Logits that differ may share a score: close ones of a beam whose score is large, or of nearly 0.  Where a candidate
// that counts may be one of them, the lists are gone through again in the order that they are in.  A list has the
// largest logits of its slice, so it has all candidates above the last pick's score; of those with that very score
// lower tokens may be missing in the last pick's beam (lists of beams before it that end at that score would fill the
// picks by themselves).  They are looked up in the row, which only such calls read again.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void beam_join_kernel(BeamArgs a, int span, int team) {
  constexpr int WAVES = THREADS / 64, EARLY = 8;
  __shared__ double powers[kPowers];
  __shared__ Candidate list[kBeamPicks * kBeamPicks];
  __shared__ int s_live[kBeamWidth];  // 0: no candidates, 1: its slices', 2: ended
  __shared__ Scored s_beams[kBeamWidth];
  __shared__ uint32_t s_nth[WAVES];
  __shared__ int n_heads, n_list, s_bad, s_close;
  __shared__ Candidate s_least, s_last;
  static_assert(kBeamPicks * kBeamPicks >= THREADS, "a place for every list's first");
  const int r = blockIdx.x, tid = threadIdx.x;
  const int b = tid / (span * team), slice = tid / team & (span - 1), place = tid & (team - 1);
  const bool mine = b < a.width && slice < a.slices;
  const int beam = r * a.width + (mine ? b : 0);
  const size_t at = (size_t)beam * a.slices + (mine ? slice : 0);
  const u64* keys = a.keys + at * a.picks;
  // (all that is read is read at once: of a beam that has ended, keys and sum are what was there)
  u64 early[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) early[i] = mine && place + i * team < a.picks ? keys[place + i * team] : 0;
  const BeamSum sum = a.sums[at];
  const float score = a.scores[beam];
  const bool end = a.ended && a.ended[beam];
  fill_powers(powers);
  const Candidate none{-__builtin_inf(), kNone, 0};
  if (tid == 0) {
    n_heads = n_list = s_bad = s_close = 0;
    s_least = s_last = none;
  }
  __syncthreads();
  float m = mine && !end ? sum.m : -kInf;
  const float own = m;
  for (int o = span * team / 2; o >= team; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  double z = 0.0;
  if (m == kInf) z = own == kInf ? sum.z : 0.0;
  else if (own > -kInf) z = sum.z * add_mass(0.0, own, (double)m, powers);
  for (int o = span * team / 2; o >= team; o >>= 1) z += __shfl_xor(z, o, 64);
  const bool bad = !(score <= 3.4028235e38f);  // NaN, +inf
  const int live = bad || !(score > -kInf) ? 0 : end ? 2 : m > -kInf ? 1 : 0;
  const Scored scored{(double)score, end ? 0.0 : log(z), m};
  if (mine && slice == 0 && place == 0) {
    s_live[b] = live;
    s_beams[b] = scored;
    if (bad) s_bad = 1;
  }
  // candidate i of this list
  auto candidate = [&](int i, u64 both) -> Candidate {
    const uint32_t first = (uint32_t)b << kTokenBits, key = (uint32_t)(both >> 32);
    if (live == 2) return slice == 0 && i == 0 ? Candidate{scored.c, first | (uint32_t)a.end_token, 0} : none;
    if (live == 0 || !both) return none;
    const double c = scored.of(key_value(key));
    return (float)c > -kInf ? Candidate{c, first | ~(uint32_t)both, key} : none;
  };
  const float own_scores = scored.own_scores();
  auto collect = [&](auto before) __attribute__((always_inline)) {
    // the picks-th of the lists' first ones, as in the slices (a score's f32 keeps the order)
    Candidate first = none;
    if (mine && place == 0) first = candidate(0, early[0]);
    const uint32_t key = first.at == kNone ? 0 : key_of((float)first.score);
    const uint32_t nth = wave_nth(key, a.picks);
    if ((tid & 63) == 0) s_nth[tid >> 6] = nth;
    __syncthreads();
    uint32_t bound = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) bound = max(bound, s_nth[w]);
    const bool head = key && key >= bound;
    if (head) list[atomicAdd(&n_heads, 1)] = first;
    __syncthreads();
    rank_all<WAVES>(list, n_heads, before, [&](const Candidate& c, int above) {
      if (above == a.picks - 1) s_least = c;
    });
    __syncthreads();
    const Candidate least = s_least;
    // (lists are in order: behind one that falls short there is nothing)
    auto take = [&](int i, u64 k) {
      const Candidate c = candidate(i, k);
      const bool in = c.at != kNone && !before(least, c);
      if (in) list[atomicAdd(&n_list, 1)] = c;
      if (fabsf(key_value(c.key)) <= own_scores) s_close = 1;  // (NaN where there is no logit)
      return in;
    };
    if (mine) {
      bool more = true;
#pragma unroll
      for (int i = 0; i < EARLY; ++i) more = more && place + i * team < a.picks && take(place + i * team, early[i]);
      for (int i = place + EARLY * team; more && i < a.picks; i += team) more = take(i, keys[i]);
    }
    __syncthreads();
  };
  collect([](const Candidate& x, const Candidate& y) { return better(x, y); });
  const bool close = s_close;
  if (close) {
    __syncthreads();
    if (tid == 0) {
      n_heads = n_list = 0;
      s_least = none;
    }
    __syncthreads();
    collect([](const Candidate& x, const Candidate& y) { return ahead(x, y); });
  }
  const int n = n_list;
  const size_t out = (size_t)r * a.picks;
  rank_all<WAVES>(list, n, better, [&](const Candidate& c, int place) {
    if (place >= a.picks) return;
    const int parent = (int)(c.at >> kTokenBits), token = (int)(c.at & ((1u << kTokenBits) - 1));
    a.scores_out[out + place] = (float)c.score;
    a.tokens[out + place] = token;
    a.parents[out + place] = parent;
    if (a.ended_out) a.ended_out[out + place] = s_live[parent] == 2 || token == a.end_token;
    if (close && place == a.picks - 1 && s_live[parent] == 1 && s_beams[parent].shared(c.key)) s_last = c;
  });
  for (int i = n + tid; i < a.picks; i += THREADS) {
    a.scores_out[out + i] = -kInf;
    a.tokens[out + i] = -1;
    a.parents[out + i] = -1;
    if (a.ended_out) a.ended_out[out + i] = 1;
  }
  if (tid == 0 && s_bad) flag(a.status, kStepArgument);
  if (!close) return;
  __syncthreads();
  const Candidate last = s_last;
  if (last.at == kNone) return;
  const uint32_t parent = last.at >> kTokenBits;
  int from = 0;  // picks before those of the last one's beam and score
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + tid;
    from += __syncthreads_count(i < n && (list[i].score > last.score || (list[i].score == last.score &&
                                                                         list[i].at >> kTokenBits < parent)));
  }
  pick_lowest<THREADS>(a, r, (int)parent, s_beams[parent], last.score, from, s_nth);
}

int slices_of(int vocab, int slice) { return (vocab + slice - 1) / slice; }

// Lists that the join counts for a beam: a power of two, for shuffles.
int span_of(int slices) {
  int span = 1;
  while (span < slices) span *= 2;
  return span;
}

// Short slices while they are no more workgroups than eight per CU, or four where the join takes its large
// workgroups for them (and a request's fit the join, a beam's a wave of it): 4 beams over 50257 BF16 logits take
// 11.9 us with them and 16.4 without, 64 of them 15.8 and 18.5, 128 (with more workgroups) 21.4 and 23.8, but 64 over
// 129280 f32 logits 22.6 and 21.0; 24 beams of 3 requests over 129280 take 19.5 and 19.1.
constexpr int kBeamShortWork = 2048;
bool short_slices(int vocab, int width, int requests) {
  const int64_t slices = slices_of(vocab, kBeamShortSlice);
  const int64_t lists = span_of((int)slices) * width;
  return slices <= 64 && lists <= 1024 && slices * width * requests <= (lists <= 256 ? kBeamShortWork : 1024);
}

size_t lists_bytes(size_t lists, int picks) { return lists * (picks * sizeof(u64) + sizeof(BeamSum)); }

}  // namespace

size_t beam_work_bytes(int vocab, int width, int picks, int requests) {
  // (short slices of few requests may be more than long ones of all)
  const size_t many = (size_t)requests * width * slices_of(vocab, kBeamSlice);
  return lists_bytes(std::max<size_t>(many, kBeamShortWork), picks);
}

void launch_beam(BeamArgs a, bool bf16, void* work, hipStream_t s) {
  const bool brief = short_slices(a.vocab, a.width, a.requests);
  a.slices = slices_of(a.vocab, brief ? kBeamShortSlice : kBeamSlice);
  a.sums = static_cast<BeamSum*>(work);
  a.keys = reinterpret_cast<u64*>(a.sums + (size_t)a.requests * a.width * a.slices);
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
    c.bf16 = bf16;
    c.keys += beams * a.slices * a.picks;
    c.sums += beams * a.slices;
    const dim3 grid(a.slices, c.requests * a.width);
    constexpr int LONG = kBeamSlice / kThreads, SHORT = kBeamShortSlice / kThreads;
    if (bf16 && brief) beam_slice_kernel<true, SHORT><<<grid, kThreads, 0, s>>>(c);
    else if (bf16) beam_slice_kernel<true, LONG><<<grid, kThreads, 0, s>>>(c);
    else if (brief) beam_slice_kernel<false, SHORT><<<grid, kThreads, 0, s>>>(c);
    else beam_slice_kernel<false, LONG><<<grid, kThreads, 0, s>>>(c);
    // a thread for every list, or several where 256 suffice; a beam's are in one wave
    const int span = span_of(a.slices), lists = span * a.width;
    int team = 1;
    while (2 * team * lists <= 256 && 2 * team * span <= 64) team *= 2;
    if (lists <= 256) beam_join_kernel<256><<<c.requests, 256, 0, s>>>(c, span, team);
    else beam_join_kernel<1024><<<c.requests, 1024, 0, s>>>(c, span, team);
  }
}

}  // namespace urb
