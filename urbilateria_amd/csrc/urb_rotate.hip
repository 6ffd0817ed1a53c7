// urb_rotate.hip -- RMS norm of every query and key head with the position rotation, one pass.
//
// A head's row h of D values: n = h / sqrt(mean(h^2) + eps) * w, then the first R values turned in
// pairs by position * inv_freq.  Every value is read once and written once, so the kernel is bound by
// HBM; the norm's sum stays in the lanes that hold the row.
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

// Any head_dim, alignment and stride: one wave per head row, a value or a pair per lane and step.
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

}  // namespace

void launch_rotate(const RotateArgs& a, bool bf16, hipStream_t s) {
  const uint64_t rows = (uint64_t)a.tokens * a.heads;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (bf16) rotate_any_kernel<true><<<grid, 256, 0, s>>>(a);
  else rotate_any_kernel<false><<<grid, 256, 0, s>>>(a);
}

}  // namespace urb
