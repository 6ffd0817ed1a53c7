// urb_attend.hip -- attention of a few new tokens per row over a paged cache, split over its length.
//
// One pass with a running maximum m and sum z: for a tile of tokens with scores s,
//   m' = max(m, max s),  z' = z e(m - m') + sum e(s - m'),  o' = o e(m - m') + sum e(s - m') v
// with e(x) = exp(scale x), and two parts of a row join by the same rule.  (The maximum is of the products
// before the scale, so that rounding errs by their distance to it and not by their size.)  Every cached row is read once, 4
// operations per value and query head that shares it, so HBM bounds all but the shortest calls.
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

namespace urb {

namespace {

constexpr int kUnit = 128;       // tokens
constexpr int kTile = 32;        // tokens of a wave's step
constexpr int kWaves = 4;
constexpr int kAttendRows = 1024;  // of a launch
constexpr int kShares = 768;     // most workgroups of a launch
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kMinusInf = -__builtin_inff();

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Query planes and weight planes (BF16 parts whose sum is the f32 value): a BF16 query is one; weights of
// two have 16 bits, of three 24.
template <bool BF16> constexpr int kQueryPlanes = BF16 ? 1 : 3;
template <bool BF16> constexpr int kWeightPlanes = BF16 ? 2 : 3;

// floats of a part: o [16][dim], m [16], z [16]
constexpr __host__ __device__ int part_floats(int dim) { return 16 * (dim + 2); }

struct Line {
  uint32_t pairs;   // of a row
  uint32_t shares;  // workgroups that can have units
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
  return (uint32_t)max(1, (r.end - r.begin + kUnit - 1) / kUnit);
}

// upto[i] = units per pair of rows 0 .. i; all threads, ends with a barrier.
__device__ __forceinline__ void fill_line(const AttendArgs& a, uint32_t* upto, uint32_t* sums, bool flags) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t base = 0;
  bool bad = false;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += 256) {
    const uint32_t r = r0 + tid;
    uint32_t u = 0;
    if (r < a.rows) {
      const int length = a.lengths[r];
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
  if (flags && bad) flag(a.status, kCacheArgument);
}

// The place of a unit: row, pair of it, first unit of that pair, units of a pair of the row.
struct Place {
  uint32_t row, pair, units;
  uint64_t first;
};
__device__ __forceinline__ Place place_of(const uint32_t* upto, uint32_t rows, uint32_t pairs, uint64_t unit) {
  uint32_t lo = 0, hi = rows - 1;  // the first row whose units end beyond
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if ((uint64_t)upto[mid] * pairs > unit) hi = mid;
    else lo = mid + 1;
  }
  const uint32_t under = lo ? upto[lo - 1] : 0;
  Place p;
  p.row = lo;
  p.units = upto[lo] - under;
  const uint64_t start = (uint64_t)under * pairs;
  p.pair = (uint32_t)((unit - start) / p.units);
  p.first = start + (uint64_t)p.pair * p.units;
  return p;
}

// Units of share g of n: [total g / n, total (g + 1) / n).
__device__ __forceinline__ uint64_t share_begin(uint64_t total, uint32_t g, uint32_t n) {
  return total * g / n;
}
// The share that unit u lies in.
__device__ __forceinline__ uint32_t share_of(uint64_t total, uint64_t u, uint32_t n) {
  return (uint32_t)(((u + 1) * n - 1) / total);
}

// Query c of a pair's sixteen: new token and head.
struct Query {
  uint32_t token, head;
  bool there;
};
__device__ __forceinline__ Query query_of(const AttendArgs& a, uint32_t pair, uint32_t tiles, int c) {
  const uint32_t group = a.q_heads / a.cache.heads;
  const uint32_t h = pair / tiles, i = (pair - h * tiles) * 16 + c;
  Query q;
  q.token = i / group;
  q.head = h * group + (i - q.token * group);
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
  if (a.sinks) {
    // the sink as one more score, with no value
    const float s = a.sinks[q.head];
    const float top = fmaxf(m, s), t = top == kMinusInf ? 0.0f : top;
    const float f = exp2f((m - t) * kLog2e);
    z = z * f + exp2f((s - t) * kLog2e);
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

// DS: head_dim in steps of 32, rounded up.
template <int DS, bool F8, bool BF16>
__global__ __launch_bounds__(64 * kWaves) void attend_kernel(AttendArgs a, Line line) {
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

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  fill_line(a, upto, sums, blockIdx.x == 0);
  const uint64_t total = (uint64_t)upto[a.rows - 1] * line.pairs;
  const uint32_t shares = (uint32_t)min<uint64_t>(line.shares, total);
  if (blockIdx.x >= shares) return;
  uint64_t unit = share_begin(total, blockIdx.x, shares);
  const uint64_t unit_end = share_begin(total, blockIdx.x + 1, shares);
  const uint32_t tiles = line.pairs / a.cache.heads;
  const float scale2 = a.scale * kLog2e;
  const uint32_t dim = a.cache.dim;
  uint8_t* const mine = stage[wave];

  while (unit < unit_end) {
    const Place at = place_of(upto, a.rows, line.pairs, unit);
    const uint64_t stop = min(unit_end, at.first + at.units);
    const Reach reach = reach_of(a, a.lengths[at.row]);
    const int t0 = reach.begin + (int)(unit - at.first) * kUnit;
    const int t1 = min(reach.end, reach.begin + (int)(stop - at.first) * kUnit);
    const uint32_t head = at.pair / tiles;
    const Query mine_q = query_of(a, at.pair, tiles, col);

    // queries, in the order of the operand (an E4M3 step takes eight of sixteen neighbours)
    __syncthreads();
    for (int i = tid; i < KS * 64; i += 64 * kWaves) {
      const int s = i >> 6, l = i & 63, g = l >> 4;
      const int d = F8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
      const Query q = query_of(a, at.pair, tiles, l & 15);
      float v[8] = {};
      bf16x8 p[QP];
      const bool in = q.there && d < (int)dim;
      const uint8_t* from = a.q + at.row * a.q_row + q.token * a.q_token + q.head * a.q_head;
      if constexpr (BF16) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (in) w = ldg16(from + 2 * d);
        q_lds[0][s][l] = w;
      } else {
        if (in) {
          const float4 x = u2f4(ldg16(from + 4 * d)), y = u2f4(ldg16(from + 4 * d + 16));
          v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
          v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
        }
        planes_of<QP>(v, p);
#pragma unroll
        for (int k = 0; k < QP; ++k) q_lds[k][s][l] = __builtin_bit_cast(uint4, p[k]);
      }
    }
    __syncthreads();

    const int my_end = mine_q.there ? reach.end - (int)(a.queries - 1 - mine_q.token) : 0;
    const int my_begin = a.window ? (int)max<int64_t>(0, (int64_t)my_end - a.window) : 0;
    // tiles inside these bounds need no mask for any query
    const int all_begin = a.window ? (int)max<int64_t>(0, (int64_t)reach.end - a.window) : 0;
    const int all_end = reach.end - (int)(a.queries - 1);

    float m = kMinusInf, z = 0.0f;
    f32x4 o[2 * DS];
#pragma unroll
    for (int j = 0; j < 2 * DS; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const int32_t* table = a.tables + at.row * a.table_stride;
    const uint8_t* const kbase = a.cache.k + head * a.cache.head_stride;
    const uint8_t* const vbase = a.cache.v + head * a.cache.head_stride;
    const uint8_t* const scales = (lane < 32 ? a.cache.k_scales : a.cache.v_scales);

    // The tile's token of this lane: lanes l and l + 32 have token l.
    auto page_of = [&](int tile) -> int {
      const int t = tile + (lane & 31);
      return t >= reach.first && t < t1 ? table[(uint32_t)t / a.cache.page] : -1;
    };
    uint4 kr[2][KL], vr[VL];
    uint32_t valid = 0, code = 0;  // tokens of the tile that there are; the scale code of the lane's token
    uint32_t off = 0;              // 16-byte units from the head's base to the lane's token
    auto place_tile = [&](int tile, int page) {
      const int t = tile + (lane & 31);
      const bool fine = (uint32_t)page < a.cache.pages;
      if (t >= reach.first && t < t1 && !fine) flag(a.status, kCacheArgument);
      valid = (uint32_t)__ballot(fine);
      const uint32_t slot = (uint32_t)t % a.cache.page;
      off = fine ? (uint32_t)((page * a.cache.page_stride + slot * a.cache.token_stride) >> 4) : 0;
      if constexpr (F8)
        code = fine ? ldg_u8(scales + ((uint64_t)page * a.cache.heads + head) * a.cache.page + slot) : 127;
    };
    auto load_k = [&]() {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = kbase + ((uint64_t)(uint32_t)__shfl((int)off, 16 * h + col, 64) << 4);
#pragma unroll
        for (int s = 0; s < KL; ++s) {
          const uint32_t d = (F8 ? 64 : 32) * s + (F8 ? 16 : 8) * grp;
          kr[h][s] = make_uint4(0, 0, 0, 0);
          if (d < dim) kr[h][s] = ldg16(p + (F8 ? d : 2 * d));
        }
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int n = i * 64 + lane, t = n / VP, piece = n - t * VP;
        const uint8_t* p = vbase + ((uint64_t)(uint32_t)__shfl((int)off, t, 64) << 4);
        vr[i] = make_uint4(0, 0, 0, 0);
        // (values that are not there stay zero: a weight of zero does not undo a NaN)
        if (valid >> t & 1 && piece * (F8 ? 16u : 8u) < dim) vr[i] = ldg16(p + 16 * piece);
      }
    };

    int tile = t0 + kTile * wave;
    int next_page = -1;
    if (tile < t1) {
      place_tile(tile, page_of(tile));
      next_page = page_of(tile + kUnit);
      load_k();
      load_v();
    }
    for (; tile < t1; tile += kUnit) {
      const uint32_t now = valid, now_code = code;
      const bool more = tile + kUnit < t1;
      // scores
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float ks = 0.0f;
        if constexpr (F8) ks = e8m0_to_f32((uint32_t)__shfl((int)now_code, 16 * h + col, 64));
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          uint4 w;
          if constexpr (F8)
            w = j & 1 ? decode8(kr[h][j / 2].z, kr[h][j / 2].w, ks) : decode8(kr[h][j / 2].x, kr[h][j / 2].y, ks);
          else w = kr[h][j];
          const bf16x8 k = __builtin_bit_cast(bf16x8, w);
#pragma unroll
          for (int p = QP - 1; p >= 0; --p)
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8, q_lds[p][j][lane]),
                                                           s[h], 0, 0, 0);
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
      if (more) {
        place_tile(tile + kUnit, next_page);
        next_page = page_of(tile + 2 * kUnit);
        load_k();
        load_v();
      }
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
    }

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
    const bool whole = unit == at.first && stop == at.first + at.units;
    const Query q = query_of(a, at.pair, tiles, c);
    // the first part of a pair that goes on in the next share is this one's second
    float* const part = a.parts + (size_t)(2 * blockIdx.x + (unit == at.first)) * part_floats(32 * DS);
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
      if (whole) finish4<BF16>(a, at.row, q, d, r, mm, zz);
      else *reinterpret_cast<float4*>(part + 32 * DS * c + d) = r;
    }
    if (!whole && (tid & 15) == 0) {
      part[16 * 32 * DS + c] = mm;
      part[16 * 32 * DS + 16 + c] = zz;
    }
    unit = stop;
  }
}

// Workgroup (g, y) joins the pair that share g begins inside of, if share g - 1 holds its first unit:
// dimensions 64 y .. 64 y + 63 of its sixteen queries.
template <bool BF16>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, Line line, int width) {
  __shared__ uint32_t upto[kAttendRows], sums[kWaves];
  fill_line(a, upto, sums, false);
  const uint64_t total = (uint64_t)upto[a.rows - 1] * line.pairs;
  const uint32_t shares = (uint32_t)min<uint64_t>(line.shares, total);
  const uint32_t g = blockIdx.x + 1;
  if (g >= shares) return;
  const uint64_t unit = share_begin(total, g, shares);
  const Place at = place_of(upto, a.rows, line.pairs, unit);
  if (at.first == unit || share_of(total, at.first, shares) != g - 1) return;
  const uint32_t last = share_of(total, at.first + at.units - 1, shares);
  const int c = threadIdx.x >> 4, d = 64 * blockIdx.y + 4 * (threadIdx.x & 15);
  const size_t size = part_floats(width);
  // the pair's first part is its share's second, the others are first
  auto part = [&](uint32_t k) { return a.parts + (2 * (size_t)k + (k == g - 1)) * size; };
  float m = kMinusInf;
  for (uint32_t k = g - 1; k <= last; ++k) m = fmaxf(m, part(k)[16 * width + c]);
  const float scale2 = a.scale * kLog2e;
  float z = 0.0f;
  float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const bool in = d < width;
  for (uint32_t k = g - 1; k <= last; ++k) {
    const float* p = part(k);
    const float f = m == kMinusInf ? 0.0f : exp2f((p[16 * width + c] - m) * scale2);
    z = fmaf(p[16 * width + 16 + c], f, z);
    if (in) {
      const float4 v = *reinterpret_cast<const float4*>(p + width * c + d);
      r.x = fmaf(v.x, f, r.x);
      r.y = fmaf(v.y, f, r.y);
      r.z = fmaf(v.z, f, r.z);
      r.w = fmaf(v.w, f, r.w);
    }
  }
  if (in) finish4<BF16>(a, at.row, query_of(a, at.pair, line.pairs / a.cache.heads, c), d, r, m, z);
}

// head_dim in steps of 32 as the kernels are built for
int steps_of(uint32_t dim) {
  const int s = ((int)dim + 31) / 32;
  return s <= 2 ? 2 : s == 5 ? 6 : s == 7 ? 8 : s;
}

template <int DS, bool BF16>
void launch_steps(const AttendArgs& a, const Line& line, hipStream_t s) {
  if (a.cache.k_scales) attend_kernel<DS, true, BF16><<<line.shares, 64 * kWaves, 0, s>>>(a, line);
  else attend_kernel<DS, false, BF16><<<line.shares, 64 * kWaves, 0, s>>>(a, line);
  if (line.shares > 1) join_kernel<BF16><<<dim3(line.shares - 1, (DS + 1) / 2), 256, 0, s>>>(a, line, 32 * DS);
}

template <bool BF16>
void launch_rows(const AttendArgs& a, hipStream_t s) {
  const uint32_t group = a.q_heads / a.cache.heads;
  Line line;
  line.pairs = a.cache.heads * ((a.queries * group + 15) / 16);
  // as many shares as there can be units
  const uint64_t most = (uint64_t)a.rows * line.pairs * ((a.max_length + kUnit - 1) / kUnit + 1);
  line.shares = (uint32_t)std::min<uint64_t>(kShares, most);
  switch (steps_of(a.cache.dim)) {
    case 2: launch_steps<2, BF16>(a, line, s); break;
    case 3: launch_steps<3, BF16>(a, line, s); break;
    case 4: launch_steps<4, BF16>(a, line, s); break;
    case 6: launch_steps<6, BF16>(a, line, s); break;
    default: launch_steps<8, BF16>(a, line, s);
  }
}

}  // namespace

size_t attend_work_bytes(uint32_t dim) {
  return (size_t)2 * kShares * part_floats(32 * steps_of(dim)) * sizeof(float);
}

void launch_attend(const AttendArgs& a, bool rows_bf16, hipStream_t s) {
  for (uint32_t r = 0; r < a.rows; r += kAttendRows) {
    AttendArgs c = a;
    c.rows = std::min<uint32_t>(kAttendRows, a.rows - r);
    c.q += r * a.q_row;
    c.out += r * a.out_row;
    c.tables += r * a.table_stride;
    c.lengths += r;
    if (a.lse) c.lse += (uint64_t)r * a.queries * a.q_heads;
    if (rows_bf16) launch_rows<true>(c, s);
    else launch_rows<false>(c, s);
  }
}

}  // namespace urb
