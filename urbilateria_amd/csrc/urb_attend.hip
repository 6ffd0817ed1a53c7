// urb_attend.hip -- attention of a few new tokens per row over a paged cache, split over its length.
//
// One pass with a running maximum m and sum z: for a tile of tokens with scores s,
//   m' = max(m, max s),  z' = z e(m - m') + sum e(s - m'),  o' = o e(m - m') + sum e(s - m') v
// with e(x) = exp(scale x), and two parts of a row join by the same rule.  (The maximum is of the products
// before the scale, so that rounding errs by their distance to it and not by their size.)  A cached row is read
// once for up to sixteen queries of its head, 4 operations per value and query, so HBM bounds all but the shortest
// calls of so many: 64 rows of 4096 tokens of 8 heads of 128 are read at 6.4 TB/s (166 us), in E4M3 at 5.7 (95 us;
// f32 rows 6.1 and 5.3), 200 rows of lengths from 8 to 12000 at 5.5 (178 us); one row of 500 tokens takes 15 us,
// latencies of its two kernels.  More queries (drafted tokens of wide groups) read it again for every sixteen: 24 of
// a head take 368 us and 193 where 16 take 167 and 96.
//
// Work: a pair is a row and up to sixteen of its query heads (of all its new tokens) that share a cache head;
// a unit is kUnit tokens of a pair.  All units lie in one line, of which every workgroup takes an equal
// share, so ragged lengths and one long row fill the chip alike; a workgroup goes through its units pair by
// pair, the four waves taking 32 tokens each.  A pair inside one share is finished there; of the others every
// share leaves a part (m, z, o), which the second kernel joins in the order of the shares.
//
// A tile: S = K Q^T on 16x16x32 MFMAs (rows: tokens, columns: queries) leaves in every lane eight scores of
// one query, which as they stand are the B operand of o = V^T P^T, tokens 4g .. 4g + 3 of either half of the
// tile in lane group g.  V's A operand needs the tokens of a column side by side: the tile goes through
// LDS, from where ds_read_b64_tr_b16 turns it.  Only the loads of the next tile cross an iteration: K's
// are issued when the products with K are done, V's when V is in LDS.
#include "urb_cache.hpp"
#include "urb_device.hpp"
#include "urb_panel.hpp"

#include <algorithm>
#include <type_traits>

namespace urb {

namespace {

constexpr int kUnit = 128;       // tokens
// A pair's start and end (its queries, the waves' join, an output) cost about what a unit does: counted as one,
// 200 rows of log-spread lengths up to 12000 take 178 us and not 183, and of 2 185.
constexpr int kStart = 1;
constexpr int kTile = 32;        // tokens of a wave's step
constexpr int kWaves = 4;
constexpr int kStep = kTile * kWaves;  // tokens of a workgroup's step
constexpr int kAttendRows = 1024;  // of a launch
constexpr int kCus = 256;
// Loads that leave the caches alone are faster (200 ragged rows, 985 MB: 178 us and 194; a row of 131071 tokens
// of E4M3, 268 MB: 56.7 and 61.1) but for a cache that a later call finds in the 256 MB of the last level (24
// rows, 35 MB, one call after another: 21.9 and 20.1).
constexpr float kCachedBytes = 128.0f * 1048576.0f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kMinusInf = -__builtin_inff();

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Query planes and weight planes (BF16 parts whose sum is the f32 value): a BF16 query is one; weights of
// two have 16 bits, of three 24.
template <bool BF16> constexpr int kQueryPlanes = BF16 ? 1 : 3;
template <bool BF16> constexpr int kWeightPlanes = BF16 ? 2 : 3;

// floats of a part: o [16][dim], then m and z of each of the sixteen
constexpr __host__ __device__ int part_floats(int dim) { return 16 * (dim + 2); }

// What there is to join: parts of `n` shares from `first` on (n 0: nothing), kept by pairs of the launch or
// by the share that the pair's second part begins, whichever are fewer.
struct Join {
  uint32_t row, pair, first, n;
};

struct Line {
  uint32_t pairs, tiles;  // of a row; of a cache head's queries
  uint32_t group;         // query heads of a cache head
  float inv_group;
  uint32_t shares;        // workgroups that can have units
  bool by_pair;           // how joins are kept
  Join* joins;            // [shares]
  PageDivision page;
  uint32_t page16, token16;  // strides in units of 16 bytes
};

// The tokens in reach of any query of a row, [first, end), and first rounded down to a tile; a length that
// cannot be counts as 0.
struct Reach {
  int begin, first, end;
};
__device__ __forceinline__ Reach reach_of(const AttendArgs& a, int length) {
  if (length < 0 || (uint32_t)length > a.max_length) length = 0;
  int first = 0;
  if (a.window) first = (int)max<int64_t>(0, (int64_t)length - (a.queries - 1) - a.window);
  return Reach{first & ~(kTile - 1), first, length};
}
__device__ __forceinline__ uint32_t units_of(Reach r) {
  return kStart + (uint32_t)max(1, (r.end - r.begin + kUnit - 1) / kUnit);
}

// upto[i] = units per pair of rows 0 .. i, and the rows' lengths; all threads, ends with a barrier.
__device__ __forceinline__ void fill_line(const AttendArgs& a, uint32_t* upto, int* lengths, uint32_t* sums) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t base = 0;
  bool bad = false;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += 64 * kWaves) {
    const uint32_t r = r0 + tid;
    uint32_t u = 0;
    if (r < a.rows) {
      const int length = a.lengths[r];
      lengths[r] = length;
      bad |= length < 0 || (uint32_t)length > a.max_length;
      u = units_of(reach_of(a, length));
    }
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t w = (uint32_t)__shfl_up((int)u, o, 64);
      if (lane >= o) u += w;
    }
    if (lane == 63) sums[wave] = u;
    __syncthreads();
    uint32_t below = base;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) below += sums[w];
      base += sums[w];
    }
    if (r < a.rows) upto[r] = below + u;
    __syncthreads();
  }
  if (blockIdx.x == 0 && bad) flag(a.status, kCacheArgument);
}

// A value of LDS that all lanes read alike, as a scalar.
template <class T>
__device__ __forceinline__ T same(T v) {
  return (T)__builtin_amdgcn_readfirstlane((int)v);
}

// n / d for quotients below 2^20, as a scalar.
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d) {
  int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
  // (the product is off by less than one)
  const int left = (int)(n - (uint32_t)q * d);
  q += left < 0 ? -1 : (uint32_t)left >= d ? 1 : 0;
  return same((uint32_t)q);
}

// The place of a unit: row, pair of it, units of a pair of the row, the pair's first unit of tokens and the
// end of its units.
struct Place {
  uint32_t row, pair, units, first, end;
};
// (A whole wave searches: the last of every sixteen rows, then the rows of one sixteen.)
__device__ __forceinline__ Place place_of(const uint32_t* upto, uint32_t rows, uint32_t pairs, uint32_t unit) {
  const uint32_t lane = threadIdx.x & 63;
  static_assert(kAttendRows == 64 * 16, "two steps");
  // rows whose units all lie before
  const uint32_t whole = __popcll(__ballot(16 * lane + 15 < rows && upto[16 * lane + 15] * pairs <= unit)) * 16;
  const uint32_t row = whole + lane;
  const uint32_t mine = lane < 16 && row < rows ? upto[row] : 0xffffffffu;
  const uint32_t more = __popcll(__ballot(mine != 0xffffffffu && mine * pairs <= unit));
  Place p;
  p.row = whole + more;
  const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)more);
  const uint32_t under = more ? (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)more - 1)
                              : whole ? same(upto[whole - 1]) : 0;
  p.units = to - under;
  const uint32_t start = under * pairs;
  p.pair = quotient(unit - start, p.units);
  p.end = start + (p.pair + 1) * p.units;
  p.first = p.end - p.units + kStart;
  return p;
}
// The place behind a pair, if there is one.
__device__ __forceinline__ Place place_after(const uint32_t* upto, uint32_t pairs, const Place& at) {
  Place p = at;
  if (at.pair + 1 < pairs) {
    ++p.pair;
  } else {
    p.pair = 0;
    p.row = at.row + 1;
    p.units = same(upto[p.row]) - same(upto[at.row]);
  }
  p.end = at.end + p.units;
  p.first = at.end + kStart;
  return p;
}

// n shares of all the units: the first `more` of them have one unit more than the others' `each`.
struct Shares {
  uint32_t n, each, more;
  __device__ __forceinline__ Shares(uint32_t total, uint32_t most)
      : n(min(most, total)), each(same(total / n)), more(total - each * n) {}
  __device__ __forceinline__ uint32_t begin(uint32_t g) const { return g * each + min(g, more); }
  // the share that a unit lies in
  __device__ __forceinline__ uint32_t of(uint32_t unit) const {
    const uint32_t longer = more * (each + 1);
    return same(unit < longer ? unit / (each + 1) : more + (unit - longer) / each);
  }
};

// Query c of a pair's sixteen: new token and head.
struct Query {
  uint32_t token, head;
  bool there;
};
__device__ __forceinline__ Query query_of(const AttendArgs& a, const Line& line, uint32_t head, uint32_t pair,
                                          int c) {
  const uint32_t i = (pair - head * line.tiles) * 16 + c;
  Query q;
  // (i < 2^18: the quotient is off by less than the half that is added)
  q.token = (uint32_t)(((float)i + 0.5f) * line.inv_group);
  q.head = head * line.group + (i - q.token * line.group);
  q.there = q.token < a.queries;
  return q;
}

// Eight floats as BF16 planes that add up to them.
template <int PLANES>
__device__ __forceinline__ void planes_of(float (&v)[8], bf16x8 (&out)[PLANES]) {
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pk_bf16(v[2 * j], v[2 * j + 1]);
      v[2 * j] -= bf16_lo(w[j]);
      v[2 * j + 1] -= bf16_hi(w[j]);
    }
    out[p] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Eight E4M3 codes times a power of two, as BF16.
__device__ __forceinline__ uint4 decode8(uint32_t lo, uint32_t hi, float scale) {
  return make_uint4(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)));
}

// Stores four consecutive outputs.
template <bool BF16>
__device__ __forceinline__ void store4(uint8_t* p, float4 v) {
  if constexpr (BF16) *reinterpret_cast<uint2*>(p) = make_uint2(pk_bf16(v.x, v.y), pk_bf16(v.z, v.w));
  else *reinterpret_cast<float4*>(p) = v;
}

// The end of a pair: four values of query q of it from their sum o under the maximum m, and once per query
// the logarithm.
template <bool BF16>
__device__ __forceinline__ void finish4(const AttendArgs& a, uint32_t row, const Query& q, int d, float4 o,
                                        float m, float z) {
  if (!q.there) return;
  m *= a.scale;
  const float s = a.sinks ? a.sinks[q.head] : kMinusInf;
  if (s != kMinusInf) {
    // the sink as one more score, with no value: all of it where it is +inf, and nothing of it where the largest
    // score has left f32's range
    const float top = fmaxf(m, s);
    const float f = s == -kMinusInf ? 0.0f : m == top ? 1.0f : exp2f((m - top) * kLog2e);
    z = z * f + (s == top ? 1.0f : exp2f((s - top) * kLog2e));
    o.x *= f; o.y *= f; o.z *= f; o.w *= f;
    m = top;
  }
  if (a.lse && d == 0)
    a.lse[((uint64_t)row * a.queries + q.token) * a.q_heads + q.head] =
        z == 0.0f ? kMinusInf : fmaf(log2f(z), kLn2, m);
  if (d >= (int)a.cache.dim) return;
  const float inv = z == 0.0f ? 0.0f : 1.0f / z;
  const float4 r = z == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                             : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  store4<BF16>(a.out + row * a.out_row + q.token * a.out_token + q.head * a.out_head + d * (BF16 ? 2 : 4), r);
}

// Workgroups per CU, and with it shares: what the registers hold without spilling.  (64 rows of 4096 tokens of 8
// heads of 128 in E4M3 take 93 us with two per CU and 102 with three; f32 rows over BF16 have 6.1 TB/s with one.)
template <int DS, bool F8, bool BF16>
constexpr int kPerCu = DS == 2 && F8 ? 3 : DS <= 3 || (DS == 4 && (F8 || BF16)) || (DS == 6 && F8) ? 2 : 1;

// DS: head_dim in steps of 32, rounded up.
template <int DS, bool F8, bool BF16>
__global__ __launch_bounds__(64 * kWaves, (kPerCu<DS, F8, BF16>)) void attend_kernel(AttendArgs a, Line line) {
  constexpr int QP = kQueryPlanes<BF16>, PP = kWeightPlanes<BF16>;
  constexpr int KS = F8 ? 2 * ((DS + 1) / 2) : DS;  // MFMA steps over head_dim
  constexpr int KL = F8 ? KS / 2 : KS;              // 16-byte loads of 16 K rows per lane
  constexpr int VL = F8 ? DS : 2 * DS;              // 16-byte loads of a V tile per lane
  constexpr int VP = (F8 ? 2 : 4) * DS;             // 16-byte pieces of a V row
  constexpr int VSTRIDE = 64 * DS + 32;             // bytes of a V row in LDS: no bank conflicts
  constexpr int OSTRIDE = 32 * DS + 4;              // floats of a query's sums in LDS
  constexpr int STAGE = kTile * VSTRIDE;
  static_assert(16 * OSTRIDE * 4 <= STAGE, "a wave's sums fit its stage");
  __shared__ __attribute__((aligned(16))) uint8_t stage[kWaves][STAGE];
  __shared__ __attribute__((aligned(16))) uint4 q_lds[QP][KS][64];
  __shared__ float s_m[kWaves][16], s_z[kWaves][16];
  __shared__ uint32_t upto[kAttendRows], sums[kWaves];
  __shared__ int lengths[kAttendRows];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  fill_line(a, upto, lengths, sums);
  const uint32_t total = same(upto[a.rows - 1]) * line.pairs;
  const Shares shares(total, line.shares);
  if (blockIdx.x >= shares.n) {
    if (!line.by_pair && tid == 0) line.joins[blockIdx.x].n = 0;
    return;
  }
  const uint32_t unit_begin = shares.begin(blockIdx.x), unit_end = shares.begin(blockIdx.x + 1);
  const float scale2 = a.scale * kLog2e;
  const uint32_t dim = a.cache.dim;
  // Whether K and V pass the caches by: what one call reads once, a line in one load (rows of 160 bytes have 5.6
  // TB/s and so 5.3), and is too much to be there at the next.
  constexpr int B = F8 ? 1 : 2;
  const bool once = line.tiles == 1 && dim * B % 64 == 0 &&
                    (float)total * (float)(kUnit * 2 * B) * (float)dim > kCachedBytes;
  const bool full = dim == (F8 ? 32 * KS : 32 * DS);
  uint8_t* const mine = stage[wave];

  // What of a pair lies in this share: tokens t0 .. t1 - 1 of row `row`, units up to `stop`; none past the
  // share's last token.
  struct Segment {
    Place at;
    Reach reach;
    uint32_t stop;
    int t0, t1;
    uint32_t head;
    bool begins, there;
  };
  auto segment_of = [&](const Place& at, uint32_t unit) -> Segment {
    Segment g;
    g.at = at;
    g.there = unit_end > g.at.first;
    g.reach = reach_of(a, same(lengths[g.at.row]));
    g.begins = unit <= g.at.first;
    g.stop = min(unit_end, g.at.end);
    g.t0 = g.reach.begin + (g.begins ? 0 : (int)(unit - g.at.first) * kUnit);
    g.t1 = min(g.reach.end, g.reach.begin + (int)(g.stop - g.at.first) * kUnit);
    g.head = quotient(g.at.pair, line.tiles);
    return g;
  };

  // The tile's token of this lane: lanes l and l + 32 have token l.
  auto page_of = [&](const Segment& g, int tile) -> int {
    const int t = tile + (lane & 31);
    return t >= g.reach.first && t < g.t1 ? a.tables[g.at.row * a.table_stride + line.page.of((uint32_t)t)] : -1;
  };
  uint4 kr[2][KL], vr[VL];
  uint32_t valid = 0, code = 0;  // tokens of the tile that there are; the scale code of the lane's token
  // Starts the loads of a tile whose pages are known.
  auto load = [&](const Segment& g, int tile, int page) __attribute__((always_inline)) {
    const int t = tile + (lane & 31);
    const bool fine = (uint32_t)page < a.cache.pages;
    if (t >= g.reach.first && t < g.t1 && !fine) flag(a.status, kCacheArgument);
    valid = (uint32_t)__ballot(fine);
    const uint32_t slot = (uint32_t)t - line.page.of((uint32_t)t) * line.page.size;
    // 16-byte units from the head's base to the lane's token
    const uint32_t off = fine ? (uint32_t)page * line.page16 + slot * line.token16 : 0;
    if constexpr (F8) {
      const uint8_t* const scales = lane < 32 ? a.cache.k_scales : a.cache.v_scales;
      code = fine ? ldg_u8(scales + ((uint64_t)page * a.cache.heads + g.head) * a.cache.page + slot) : 127;
    }
    const uint8_t* const kbase = a.cache.k + g.head * a.cache.head_stride;
    const uint8_t* const vbase = a.cache.v + g.head * a.cache.head_stride;
    // (values past the head's are not read; V's of tokens that are not there are zero, for a weight of zero
    // does not undo a NaN)
    auto both = [&](auto check, auto once) __attribute__((always_inline)) {
      auto get = [](const uint8_t* p) { return decltype(once)::value ? ldg16_stream(p) : ldg16(p); };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = kbase + ((uint64_t)(uint32_t)__shfl((int)off, 16 * h + col, 64) << 4);
#pragma unroll
        for (int s = 0; s < KL; ++s) {
          const uint32_t d = (F8 ? 64 : 32) * s + (F8 ? 16 : 8) * grp;
          const bool in = !decltype(check)::value || d < dim;
          kr[h][s] = in ? get(p + (F8 ? d : 2 * d)) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int n = i * 64 + lane, u = n / VP, piece = n - u * VP;
        const uint8_t* p = vbase + ((uint64_t)(uint32_t)__shfl((int)off, u, 64) << 4) + 16 * piece;
        const bool in = !decltype(check)::value || (valid >> u & 1 && piece * (F8 ? 16u : 8u) < dim);
        vr[i] = in ? get(p) : make_uint4(0, 0, 0, 0);
      }
    };
    const bool check = !full || valid != 0xffffffffu;
    if (once) {
      if (check) both(std::true_type{}, std::true_type{});
      else both(std::false_type{}, std::true_type{});
    } else {
      if (check) both(std::true_type{}, std::false_type{});
      else both(std::false_type{}, std::false_type{});
    }
  };

  // Queries, in the order of the operand (an E4M3 step takes eight of sixteen neighbours): read ahead, put
  // into LDS when the products with the last ones are done.
  constexpr int QL = (KS + kWaves - 1) / kWaves;
  uint4 qr[QL][BF16 ? 1 : 2];
  auto load_q = [&](const Segment& g) {
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int s = i * kWaves + wave;
      const int d = F8 ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 32 * s + 8 * grp;
      const Query q = query_of(a, line, g.head, g.at.pair, col);
      const uint8_t* from = a.q + g.at.row * a.q_row + q.token * a.q_token + q.head * a.q_head;
#pragma unroll
      for (int k = 0; k < (BF16 ? 1 : 2); ++k) {
        qr[i][k] = make_uint4(0, 0, 0, 0);
        if (q.there && s < KS && d < (int)dim) qr[i][k] = ldg16(from + (BF16 ? 2 : 4) * d + 16 * k);
      }
    }
  };
  auto stage_q = [&]() {
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      const int s = i * kWaves + wave;
      if (s >= KS) break;
      if constexpr (BF16) {
        q_lds[0][s][lane] = qr[i][0];
      } else {
        const float4 x = u2f4(qr[i][0]), y = u2f4(qr[i][1]);
        float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        bf16x8 p[QP];
        planes_of<QP>(v, p);
#pragma unroll
        for (int k = 0; k < QP; ++k) q_lds[k][s][lane] = __builtin_bit_cast(uint4, p[k]);
      }
    }
  };

  Segment g = segment_of(place_of(upto, a.rows, line.pairs, unit_begin), unit_begin);
  // Pages are known a segment, or two tiles, before their loads begin.
  int tile = g.t0 + kTile * wave;
  const int first_page = g.there ? page_of(g, tile) : -1;
  if (!line.by_pair && tid == 0) {
    // the share's first boundary, for the second kernel
    const uint32_t last = shares.of(g.at.end - 1);
    const bool second = !g.begins && shares.of(g.at.first) == blockIdx.x - 1;
    line.joins[blockIdx.x] = Join{g.at.row, g.at.pair, blockIdx.x - 1, second ? last - blockIdx.x + 2 : 0};
  }
  if (!g.there) return;
  int next_page = page_of(g, tile + kStep);
  load_q(g);
  auto segment_after = [&](const Segment& g) -> Segment {
    if (g.stop < unit_end) return segment_of(place_after(upto, line.pairs, g.at), g.stop);
    Segment none = g;
    none.there = false;
    return none;
  };
  Segment next = segment_after(g);
  int page0 = -1, page1 = -1, next_tile = 0;
  auto pages_of_next = [&]() {
    if (!next.there) return;
    next_tile = next.t0 + kTile * wave;
    page0 = page_of(next, next_tile);
    page1 = page_of(next, next_tile + kStep);
  };
  pages_of_next();
  if (tile < g.t1) load(g, tile, first_page);
  stage_q();
  __syncthreads();

  for (;;) {
    const bool whole = g.begins && g.stop == g.at.end, goes_on = next.there;
    if (line.by_pair && g.begins && tid == 0) {
      const uint32_t last = shares.of(g.at.end - 1);
      line.joins[g.at.row * line.pairs + g.at.pair] =
          Join{g.at.row, g.at.pair, blockIdx.x, whole ? 0 : last - blockIdx.x + 1};
    }
    if (goes_on) load_q(next);

    const Query mine_q = query_of(a, line, g.head, g.at.pair, col);
    const int my_end = mine_q.there ? g.reach.end - (int)(a.queries - 1 - mine_q.token) : 0;
    const int my_begin = a.window ? (int)max<int64_t>(0, (int64_t)my_end - a.window) : 0;
    // tiles inside these bounds need no mask for any query
    const int all_begin = a.window ? (int)max<int64_t>(0, (int64_t)g.reach.end - a.window) : 0;
    const int all_end = g.reach.end - (int)(a.queries - 1);

    float m = kMinusInf, z = 0.0f;
    f32x4 o[2 * DS];
#pragma unroll
    for (int j = 0; j < 2 * DS; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    do {
      // (a wave without a tile in the segment comes here once, for the loads)
      const bool have = tile < g.t1, stay = tile + kStep < g.t1;
      const uint32_t now = valid, now_code = code;
      // scores
      f32x4 s[2];
      if (have) {
        float ks[2] = {0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (F8) ks[h] = e8m0_to_f32((uint32_t)__shfl((int)now_code, 16 * h + col, 64));
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          bf16x8 q[QP];
#pragma unroll
          for (int p = 0; p < QP; ++p) q[p] = __builtin_bit_cast(bf16x8, q_lds[p][j][lane]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 w;
            if constexpr (F8)
              w = j & 1 ? decode8(kr[h][j / 2].z, kr[h][j / 2].w, ks[h])
                        : decode8(kr[h][j / 2].x, kr[h][j / 2].y, ks[h]);
            else w = kr[h][j];
            const bf16x8 k = __builtin_bit_cast(bf16x8, w);
#pragma unroll
            for (int p = QP - 1; p >= 0; --p)
              s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[p], s[h], 0, 0, 0);
          }
        }
        // V into LDS, then the loads of the next tile
        if constexpr (F8) {
#pragma unroll
          for (int i = 0; i < VL; ++i) {
            const int n = i * 64 + lane, t = n / VP, piece = n - t * VP;
            const float vs = e8m0_to_f32((uint32_t)__shfl((int)now_code, 32 + t, 64));
            uint4* to = reinterpret_cast<uint4*>(mine + t * VSTRIDE + 32 * piece);
            to[0] = decode8(vr[i].x, vr[i].y, vs);
            to[1] = decode8(vr[i].z, vr[i].w, vs);
          }
        } else {
#pragma unroll
          for (int i = 0; i < VL; ++i) {
            const int n = i * 64 + lane, t = n / VP, piece = n - t * VP;
            *reinterpret_cast<uint4*>(mine + t * VSTRIDE + 16 * piece) = vr[i];
          }
        }
      }
      if (stay || goes_on) {
        const Segment& to = stay ? g : next;
        const int to_tile = stay ? tile + kStep : next_tile;
        const int page = stay ? next_page : page0;
        next_page = stay ? page_of(g, tile + 2 * kStep) : page1;
        if (to_tile < to.t1) load(to, to_tile, page);
      }
      if (!have) break;
      // weights
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = s[j >> 2][j & 3];
      if (now != 0xffffffffu || tile < all_begin || tile + kTile > all_end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = 16 * (j >> 2) + 4 * grp + (j & 3), t = tile + i;
          if (!(now >> i & 1) || t < my_begin || t >= my_end) e[j] = kMinusInf;
        }
      }
      float top = e[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, e[j]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__ballot(top > m)) {
        const float up = fmaxf(m, top);
        const float f = up == kMinusInf ? 1.0f : exp2f((m - up) * scale2);
        m = up;
        z *= f;
#pragma unroll
        for (int j = 0; j < 2 * DS; ++j) {
          o[j][0] *= f; o[j][1] *= f; o[j][2] *= f; o[j][3] *= f;
        }
      }
      const float base = m == kMinusInf ? 0.0f : m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = exp2f((e[j] - base) * scale2);
        z += e[j];
      }
      bf16x8 w[PP];
      planes_of<PP>(e, w);
      // values (of the whole wave's stores: LDS takes a wave's operations in their order)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int j = 0; j < 2 * DS; ++j) {
        const uint8_t* p = mine + (4 * grp + col / 4) * VSTRIDE + 32 * j + 8 * (col & 3);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(p + 16 * VSTRIDE));
        const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int k = PP - 1; k >= 0; --k)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w[k], o[j], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      tile += kStep;
    } while (tile < g.t1);

    // the waves' sums, joined
    z += __shfl_xor(z, 16, 64);
    z += __shfl_xor(z, 32, 64);
    float* const sum = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int j = 0; j < 2 * DS; ++j)
      *reinterpret_cast<f32x4*>(sum + col * OSTRIDE + 16 * j + 4 * grp) = o[j];
    if (lane < 16) {
      s_m[wave][lane] = m;
      s_z[wave][lane] = z;
    }
    __syncthreads();
    if (goes_on) stage_q();
    const int c = tid >> 4;
    float mm = s_m[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, s_m[w][c]);
    float f[kWaves], zz = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      f[w] = mm == kMinusInf ? 0.0f : exp2f((s_m[w][c] - mm) * scale2);
      zz = fmaf(s_z[w][c], f[w], zz);
    }
    const Query q = query_of(a, line, g.head, g.at.pair, c);
    // the first part of a pair that goes on in the next share is this one's second
    float* const part = a.parts + (size_t)(2 * blockIdx.x + g.begins) * part_floats(32 * DS);
    for (int d = 4 * (tid & 15); d < 32 * DS; d += 64) {
      float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(
            reinterpret_cast<const float*>(stage[w]) + c * OSTRIDE + d);
        r.x = fmaf(v.x, f[w], r.x);
        r.y = fmaf(v.y, f[w], r.y);
        r.z = fmaf(v.z, f[w], r.z);
        r.w = fmaf(v.w, f[w], r.w);
      }
      if (whole) finish4<BF16>(a, g.at.row, q, d, r, mm, zz);
      else *reinterpret_cast<float4*>(part + 32 * DS * c + d) = r;
    }
    if (!whole && (tid & 15) == 0)
      *reinterpret_cast<float2*>(part + 16 * 32 * DS + 2 * c) = make_float2(mm, zz);
    if (!goes_on) break;
    __syncthreads();
    g = next;
    tile = next_tile;
    next = segment_after(g);
    pages_of_next();
  }
}

// Two parts of a query as one: (m, z, o) takes in (pm, pz, po).  (Scores of NaN alone leave a maximum of -inf, and
// sums of NaN that stay so.)
__device__ __forceinline__ void take_in(float& m, float& z, float4& o, float pm, float pz, const float4& po,
                                        float scale2) {
  const float top = fmaxf(m, pm), base = top == kMinusInf ? 0.0f : top;
  const float f = exp2f((m - base) * scale2), g = exp2f((pm - base) * scale2);
  m = top;
  z = fmaf(pz, g, z * f);
  o.x = fmaf(po.x, g, o.x * f);
  o.y = fmaf(po.y, g, o.y * f);
  o.z = fmaf(po.z, g, o.z * f);
  o.w = fmaf(po.w, g, o.w * f);
}

// Workgroup (j, y) joins the parts of join j.  `lanes` threads hold a query's row, four values each; `groups`
// of them take the parts in turn, so a row of many parts has many loads on their way.
template <bool BF16>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, Line line, int width, int lanes, int groups) {
  __shared__ float4 s_o[256];
  __shared__ float2 s_mz[256];
  const Join join = line.joins[blockIdx.x + (line.by_pair ? 0 : 1)];
  if (join.n == 0) return;
  const int tid = threadIdx.x, set = tid / lanes, d = 4 * (tid - set * lanes);
  const int queries = 256 / lanes / groups, group = set % groups;
  const int c = blockIdx.y * queries + set / groups;
  const float scale2 = a.scale * kLog2e;
  const size_t size = part_floats(width);
  float m = kMinusInf, z = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const bool in = d < width;
  constexpr int AHEAD = 4;
  for (uint32_t k0 = group; k0 < join.n; k0 += AHEAD * groups) {
    float2 mz[AHEAD];
    float4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t k = k0 + i * groups;
      mz[i] = make_float2(kMinusInf, 0.0f);
      v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (k < join.n && in) {
        // a pair's first part is its share's second, the others are first
        const float* p = a.parts + (2 * (size_t)(join.first + k) + (k == 0)) * size;
        mz[i] = *reinterpret_cast<const float2*>(p + 16 * width + 2 * c);
        v[i] = *reinterpret_cast<const float4*>(p + width * c + d);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) take_in(m, z, o, mz[i].x, mz[i].y, v[i], scale2);
  }
  if (groups > 1) {
    s_o[tid] = o;
    s_mz[tid] = make_float2(m, z);
    __syncthreads();
    if (group) return;
    for (int g = 1; g < groups; ++g) {
      const float2 mz = s_mz[tid + g * lanes];
      take_in(m, z, o, mz.x, mz.y, s_o[tid + g * lanes], scale2);
    }
  }
  if (in) finish4<BF16>(a, join.row, query_of(a, line, join.pair / line.tiles, join.pair, c), d, o, m, z);
}

// The most units of a pair.
uint32_t most_units(const AttendArgs& a) { return kStart + (a.max_length + kUnit - 1) / kUnit + 1; }

template <int DS, bool F8, bool BF16>
void launch_pass(const AttendArgs& a, Line line, hipStream_t s) {
  constexpr uint32_t most = kPerCu<DS, F8, BF16> * kCus;
  // no more shares than there can be units
  line.shares = (uint32_t)std::min<uint64_t>(most, (uint64_t)a.rows * line.pairs * most_units(a));
  line.by_pair = (uint64_t)a.rows * line.pairs < line.shares;
  line.joins = reinterpret_cast<Join*>(a.parts + (size_t)2 * most * part_floats(32 * DS));
  attend_kernel<DS, F8, BF16><<<line.shares, 64 * kWaves, 0, s>>>(a, line);
  const uint32_t joins = line.by_pair ? a.rows * line.pairs : line.shares - 1;
  if (joins == 0) return;
  // threads per query, and how many sets of them go through its parts: about four parts each
  const int lanes = DS <= 2 ? 16 : DS <= 4 ? 32 : 64;
  int groups = 1;
  while (groups < 256 / lanes && 4 * groups * joins < line.shares) groups *= 2;
  const int queries = 256 / lanes / groups;
  join_kernel<BF16><<<dim3(joins, (16 + queries - 1) / queries), 256, 0, s>>>(a, line, 32 * DS, lanes, groups);
}

template <int DS, bool F8, bool BF16>
constexpr size_t work_of() {
  return (size_t)kPerCu<DS, F8, BF16> * kCus * (2 * part_floats(32 * DS) * sizeof(float) + sizeof(Join));
}

// Calls f with the kernel's constants as types.
template <class F>
auto with_kernel(uint32_t dim, bool f8, bool bf16, F f) {
  auto rows = [&](auto ds, auto f8_) {
    return bf16 ? f(ds, f8_, std::true_type{}) : f(ds, f8_, std::false_type{});
  };
  auto types = [&](auto ds) { return f8 ? rows(ds, std::true_type{}) : rows(ds, std::false_type{}); };
  switch (((int)dim + 31) / 32) {
    case 1:
    case 2: return types(std::integral_constant<int, 2>{});
    case 3: return types(std::integral_constant<int, 3>{});
    case 4: return types(std::integral_constant<int, 4>{});
    case 5:
    case 6: return types(std::integral_constant<int, 6>{});
    default: return types(std::integral_constant<int, 8>{});
  }
}

Line line_of(const AttendArgs& a) {
  Line line{};
  line.group = a.q_heads / a.cache.heads;
  line.inv_group = 1.0f / (float)line.group;
  line.tiles = (a.queries * line.group + 15) / 16;
  line.pairs = a.cache.heads * line.tiles;
  line.page = PageDivision::by(a.cache.page);
  line.page16 = (uint32_t)(a.cache.page_stride >> 4);
  line.token16 = (uint32_t)(a.cache.token_stride >> 4);
  return line;
}

}  // namespace

size_t attend_work_bytes(uint32_t dim, bool f8, bool rows_bf16) {
  return with_kernel(dim, f8, rows_bf16, [](auto ds, auto f8_, auto bf16) {
    return work_of<decltype(ds)::value, decltype(f8_)::value, decltype(bf16)::value>();
  });
}

void launch_attend(const AttendArgs& a, bool rows_bf16, hipStream_t s) {
  const Line line = line_of(a);
  // rows of a launch: their units have 32 bits (a row has fewer than 2^31)
  const uint32_t most = (uint32_t)std::min<uint64_t>(kAttendRows, 0xffffffffu / (line.pairs * most_units(a)));
  for (uint32_t r = 0; r < a.rows; r += most) {
    AttendArgs c = a;
    c.rows = std::min(most, a.rows - r);
    c.q += r * a.q_row;
    c.out += r * a.out_row;
    c.tables += r * a.table_stride;
    c.lengths += r;
    if (a.lse) c.lse += (uint64_t)r * a.queries * a.q_heads;
    with_kernel(a.cache.dim, a.cache.k_scales != nullptr, rows_bf16, [&](auto ds, auto f8, auto bf16) {
      launch_pass<decltype(ds)::value, decltype(f8)::value, decltype(bf16)::value>(c, line, s);
      return 0;
    });
  }
}

}  // namespace urb
