// urb_rotate.hip -- RMS norm of every query and key head with the position rotation, one pass.
//
// A head's row h of D values: n = h / sqrt(mean(h^2) + eps) * w, then the first R values turned in
// pairs by position * inv_freq.  Every value is read once and written once, so the kernel is bound by
// HBM; the norm's sum stays in the lanes that hold the row.  32768 tokens of 18 heads of 256 in BF16 (604 MB):
// 128 us, 4.7 TB/s, where a large copy reaches 5.0; 2000 tokens in f32 (61 MB): 14.5 us; a token 3.6.
//
// The angle is the f64 product of position and frequency (an f32 product has lost the fraction of a
// turn at position 2^24), reduced to [-pi/4, pi/4] with a two-part pi/2 and evaluated by the Taylor
// series in f64: below one rounding of the f32 cosine and sine that the rotation uses.
#include "urb_device.hpp"
#include "urb_panel.hpp"
#include "urb_step.hpp"

namespace urb {

namespace {

__device__ __forceinline__ float2 turn_of(int64_t position, float freq) {
  const double angle = (double)position * (double)freq;
  const double n = rint(angle * 0.63661977236758134308);  // 2 / pi
  double r = fma(-n, 0x1.921fb54442d18p+0, angle);        // pi / 2, high and low part
  r = fma(-n, 0x1.1a62633145c07p-54, r);
  const double q = r * r;
  // |r| <= pi/4: the first terms left out are below 2e-14
  double s = -1.0 / 1307674368000.0;
  s = fma(s, q, 1.0 / 6227020800.0);
  s = fma(s, q, -1.0 / 39916800.0);
  s = fma(s, q, 1.0 / 362880.0);
  s = fma(s, q, -1.0 / 5040.0);
  s = fma(s, q, 1.0 / 120.0);
  s = fma(s, q, -1.0 / 6.0);
  s = fma(s * q, r, r);
  double c = 1.0 / 20922789888000.0;
  c = fma(c, q, -1.0 / 87178291200.0);
  c = fma(c, q, 1.0 / 479001600.0);
  c = fma(c, q, -1.0 / 3628800.0);
  c = fma(c, q, 1.0 / 40320.0);
  c = fma(c, q, -1.0 / 720.0);
  c = fma(c, q, 1.0 / 24.0);
  c = fma(c, q, -0.5);
  c = fma(c, q, 1.0);
  // n modulo 4, also where n has more bits than an int (its f64 is then a multiple of 4 or exact)
  const int k = (int)(n - 4.0 * floor(n * 0.25));
  const float cf = (float)((k & 1) ? s : c), sf = (float)((k & 1) ? c : s);
  return make_float2(k == 1 || k == 2 ? -cf : cf, k >= 2 ? -sf : sf);
}

template <bool BF16>
__device__ __forceinline__ float load_one(const void* p, size_t i) {
  if constexpr (BF16) return u2f((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  else return reinterpret_cast<const float*>(p)[i];
}
template <bool BF16>
__device__ __forceinline__ void store_one(void* p, size_t i, float v) {
  if constexpr (BF16) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)pk_bf16(v, 0.0f);
  else reinterpret_cast<float*>(p)[i] = v;
}

// Any head_dim, alignment and stride: one wave per head row, a value or a pair per lane and step (18 heads of
// 256 in BF16, a value off the boundary that the wide kernel asks for: 3.6 us against its 3.4 for a token, 9.0
// against 6.2 for 515, 533 against 130 for 32768).
template <bool BF16>
__global__ __launch_bounds__(256) void rotate_any_kernel(RotateArgs a) {
  const uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (uint64_t)a.tokens * a.heads) return;
  const int lane = threadIdx.x & 63;
  const uint32_t t = (uint32_t)(row / a.heads);
  const int head = (int)(row % a.heads);
  const bool is_k = head >= a.q_heads;
  const HeadRows& m = is_k ? a.k : a.q;
  const int h = is_k ? head - a.q_heads : head;
  const size_t in = (size_t)t * m.in_token + (size_t)h * m.in_head;
  const size_t out = (size_t)t * m.out_token + (size_t)h * m.out_head;
  float sum = 0.0f;
  for (int i = lane; i < a.dim; i += 64) {
    const float v = load_one<BF16>(m.in, in + i);
    sum = fmaf(v, v, sum);
  }
  sum = wave_sum_f32(sum);
  const float inv = 1.0f / sqrtf(sum / (float)a.dim + a.eps);
  auto normed = [&](int i) {
    return load_one<BF16>(m.in, in + i) * inv * (m.weight[i] + a.offset);
  };
  const int half = a.rotary / 2;
  for (int i = lane; i < half; i += 64) {
    const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
    const float2 cs = turn_of(a.positions[t], a.inv_freq[i]);
    const float x = normed(i0), y = normed(i1);
    store_one<BF16>(m.out, out + i0, fmaf(x, cs.x, -(y * cs.y)));
    store_one<BF16>(m.out, out + i1, fmaf(y, cs.x, x * cs.y));
  }
  for (int i = a.rotary + lane; i < a.dim; i += 64) store_one<BF16>(m.out, out + i, normed(i));
}

// Eight values of a row.
template <bool BF16>
__device__ __forceinline__ void load8(float (&v)[8], const uint8_t* p) {
  if constexpr (BF16) {
    const uint4 q = ldg16(p);
    v[0] = bf16_lo(q.x); v[1] = bf16_hi(q.x); v[2] = bf16_lo(q.y); v[3] = bf16_hi(q.y);
    v[4] = bf16_lo(q.z); v[5] = bf16_hi(q.z); v[6] = bf16_lo(q.w); v[7] = bf16_hi(q.w);
  } else {
    const float4 a = u2f4(ldg16(p)), b = u2f4(ldg16(p + 16));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}
template <bool BF16>
__device__ __forceinline__ void store8(uint8_t* p, const float (&v)[8]) {
  if constexpr (BF16) {
    const uint4 q = make_uint4(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]),
                               pk_bf16(v[6], v[7]));
    *reinterpret_cast<uint4*>(p) = q;
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Sixteen-byte heads: `span` (a power of two) lanes hold a head row, 16 values each, loaded as two
// eights that hold both values of every pair: eights u and R / 16 + u of the turned part, or neighbours.
// A lane's place in its row is the same for all its rows, so its weights stay in registers; a workgroup
// takes all heads of `group` tokens (blockIdx.y: a part of them), whose cosines and sines it computes once
// into LDS.
template <bool BF16, bool INTER>
__global__ __launch_bounds__(256) void rotate_wide_kernel(RotateArgs a, int span, int group,
                                                          int parts) {
  extern __shared__ float2 turns[];  // [group][rotary / 2]
  const uint32_t t0 = blockIdx.x * group;
  const int tokens = (int)min((uint32_t)group, a.tokens - t0);
  const int half = a.rotary / 2, lanes = a.dim / 16;
  const int u = threadIdx.x & (span - 1), row0 = threadIdx.x / span, rows = 256 / span;
  const bool active = u < lanes;
  const int turned = a.rotary / 16;  // lanes that hold pairs (not interleaved)
  int o0 = 16 * u, o1 = 16 * u + 8;
  if (!INTER && u < turned) {
    o0 = 8 * u;
    o1 = half + 8 * u;
  }
  if (!active) o0 = o1 = 0;
  float wq[2][8], wk[2][8];
  load8<false>(wq[0], reinterpret_cast<const uint8_t*>(a.q.weight + o0));
  load8<false>(wq[1], reinterpret_cast<const uint8_t*>(a.q.weight + o1));
  const float* kw = a.k.weight ? a.k.weight : a.q.weight;
  load8<false>(wk[0], reinterpret_cast<const uint8_t*>(kw + o0));
  load8<false>(wk[1], reinterpret_cast<const uint8_t*>(kw + o1));
  for (int i = threadIdx.x; i < tokens * half; i += 256)
    turns[i] = turn_of(a.positions[t0 + i / half], a.inv_freq[i % half]);
  constexpr size_t B = BF16 ? 2 : 4;
  const int items = tokens * a.heads;
  const float mean = 1.0f / (float)a.dim;
  for (int r = rows * blockIdx.y; r < items; r += rows * parts) {
    // (lanes past the last row or value take part in the barrier and the sums alone)
    const int i = min(r + row0, items - 1);
    const bool there = r + row0 < items && active;
    const int tl = i / a.heads, head = i - tl * a.heads;
    const bool is_k = head >= a.q_heads;
    const HeadRows& m = is_k ? a.k : a.q;
    const int h = is_k ? head - a.q_heads : head;
    float x[2][8] = {};
    if (there) {
      const uint8_t* in = reinterpret_cast<const uint8_t*>(m.in) +
                          ((size_t)(t0 + tl) * m.in_token + (size_t)h * m.in_head) * B;
      load8<BF16>(x[0], in + o0 * B);
      load8<BF16>(x[1], in + o1 * B);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(x[0][j], x[0][j], fmaf(x[1][j], x[1][j], sum));
    for (int o = span / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float inv = 1.0f / sqrtf(fmaf(sum, mean, a.eps));
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[v][j] = x[v][j] * inv * ((is_k ? wk[v][j] : wq[v][j]) + a.offset);
    if (r == rows * (int)blockIdx.y) __syncthreads();  // the turns are there
    const float2* cs = turns + tl * half + 8 * u;
    if constexpr (INTER) {
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (8 * u + 4 * v + j < half) {
            const float2 c = cs[4 * v + j];
            const float p = x[v][2 * j], q = x[v][2 * j + 1];
            x[v][2 * j] = fmaf(p, c.x, -(q * c.y));
            x[v][2 * j + 1] = fmaf(q, c.x, p * c.y);
          }
    } else if (u < turned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 c = cs[j];
        const float p = x[0][j], q = x[1][j];
        x[0][j] = fmaf(p, c.x, -(q * c.y));
        x[1][j] = fmaf(q, c.x, p * c.y);
      }
    }
    if (there) {
      uint8_t* out = reinterpret_cast<uint8_t*>(m.out) +
                     ((size_t)(t0 + tl) * m.out_token + (size_t)h * m.out_head) * B;
      store8<BF16>(out + o0 * B, x[0]);
      store8<BF16>(out + o1 * B, x[1]);
    }
  }
}

// Whether every head of m starts at a multiple of 16 bytes.
bool wide_rows(const HeadRows& m, size_t b) {
  const auto fits = [&](const void* p, uint64_t token, uint64_t head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token * b % 16 == 0 && head * b % 16 == 0;
  };
  return fits(m.in, m.in_token, m.in_head) && fits(m.out, m.out_token, m.out_head) &&
         reinterpret_cast<uintptr_t>(m.weight) % 16 == 0;
}

template <bool BF16>
void launch_wide(const RotateArgs& a, hipStream_t s) {
  int span = 1;
  while (span < a.dim / 16) span *= 2;
  const int rows = 256 / span;  // head rows that a workgroup holds at a time
  // Tokens per workgroup: up to eight, the fewest whose rows fill its last round to nine tenths,
  // while that leaves four workgroups per CU.
  int group = 1;
  auto full = [&](int g) { return 10 * g * a.heads >= 9 * ((g * a.heads + rows - 1) / rows) * rows; };
  for (int g = 1; g <= 8; ++g) {
    if ((a.tokens + g - 1) / g < 1024) break;
    group = g;
    if (g * a.heads >= 4 * rows && full(g)) break;
  }
  // Few tokens: a workgroup per round of rows, until the chip has four per CU.
  const int rounds = (group * a.heads + rows - 1) / rows;
  const int blocks = (int)((a.tokens + group - 1) / group);
  const int parts = std::max(1, std::min(rounds, 1024 / blocks));
  const dim3 grid(blocks, parts);
  const size_t lds = (size_t)group * (a.rotary / 2) * sizeof(float2);
  if (a.interleaved) rotate_wide_kernel<BF16, true><<<grid, 256, lds, s>>>(a, span, group, parts);
  else rotate_wide_kernel<BF16, false><<<grid, 256, lds, s>>>(a, span, group, parts);
}

// Head rows per launch (longer calls take several): a launch may have no more than 2^32 threads, and either
// kernel has at most 256 of them per head row.
constexpr uint32_t kMostRows = 1u << 23;

// The same call from token t on.
HeadRows rows_from(const HeadRows& m, uint32_t t, size_t b) {
  HeadRows r = m;
  if (!m.in) return r;
  r.in = static_cast<const char*>(m.in) + t * m.in_token * b;
  r.out = static_cast<char*>(m.out) + t * m.out_token * b;
  return r;
}

}  // namespace

void launch_rotate(const RotateArgs& a, bool bf16, hipStream_t s) {
  const uint32_t most = std::max(1u, kMostRows / (uint32_t)a.heads);
  if (a.tokens > most) {
    const size_t b = bf16 ? 2 : 4;
    for (uint32_t t = 0; t < a.tokens; t += most) {
      RotateArgs c = a;
      c.q = rows_from(a.q, t, b);
      c.k = rows_from(a.k, t, b);
      if (a.positions) c.positions = a.positions + t;
      c.tokens = std::min(most, a.tokens - t);
      launch_rotate(c, bf16, s);
    }
    return;
  }
  const bool eights = a.dim % 16 == 0 && (a.interleaved || a.rotary % 16 == 0);
  if (eights && wide_rows(a.q, bf16 ? 2 : 4) && (!a.k.in || wide_rows(a.k, bf16 ? 2 : 4))) {
    if (bf16) launch_wide<true>(a, s);
    else launch_wide<false>(a, s);
    return;
  }
  const uint64_t rows = (uint64_t)a.tokens * a.heads;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (bf16) rotate_any_kernel<true><<<grid, 256, 0, s>>>(a);
  else rotate_any_kernel<false><<<grid, 256, 0, s>>>(a);
}

}  // namespace urb
