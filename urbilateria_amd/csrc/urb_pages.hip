// urb_pages.hip -- the pages of a cache: what a step's new tokens need, rows into slots, and tables that
// follow the beams of a search.
#include "urb_cache.hpp"
#include "urb_device.hpp"
#include "urb_panel.hpp"

#include <algorithm>

namespace urb {

namespace {

// ---- rows into slots ----
//
// Every value is read once and written once: bound by HBM (8190 tokens of 8 heads of 128, BF16 to E4M3: 50 MB in
// 10.4 us, 4.85 TB/s, the vector units busy for 88 %), or for a few tokens by the launch (33 of 2 heads of 256:
// 3 us).  A row of a head is held by dim / 16 lanes (of `span`, a power of two), sixteen values each, so an E4M3 row's largest
// value is a few shuffles away and its codes leave in one 16-byte store per lane.
template <bool BF16>
__device__ __forceinline__ void load16(float (&v)[16], const uint8_t* p) {
  if constexpr (BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 q = ldg16(p + 16 * i);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[8 * i + 2 * j] = bf16_lo(w[j]);
        v[8 * i + 2 * j + 1] = bf16_hi(w[j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q = u2f4(ldg16(p + 16 * i));
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  }
}

template <bool BF16, bool F8>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a, int span) {
  const uint32_t row = blockIdx.x * (256 / span) + threadIdx.x / span;
  const int u = threadIdx.x & (span - 1);
  const uint32_t per_token = 2 * a.cache.heads;
  const uint32_t t = row / per_token;
  if (t >= a.tokens) return;
  const uint32_t h2 = row - t * per_token;
  const bool is_v = h2 >= a.cache.heads;
  const uint32_t h = is_v ? h2 - a.cache.heads : h2;
  const int64_t slot = a.slots[t];
  if ((uint64_t)slot >= (uint64_t)a.cache.pages * a.cache.page) return;
  const uint32_t page = (uint32_t)slot / a.cache.page, at = (uint32_t)slot - page * a.cache.page;
  const bool there = u < (int)a.cache.dim / 16;
  constexpr int B = BF16 ? 2 : 4;
  const uint8_t* in = (is_v ? a.v + t * a.v_token + h * a.v_head : a.k + t * a.k_token + h * a.k_head) +
                      16 * B * u;
  uint8_t* out = (is_v ? a.cache.v : a.cache.k) + page * a.cache.page_stride +
                 h * a.cache.head_stride + at * a.cache.token_stride;
  if constexpr (!F8) {
    if (!there) return;
    out += 32 * u;
    if constexpr (BF16) {
      const uint4 lo = ldg16(in), hi = ldg16(in + 16);
      reinterpret_cast<uint4*>(out)[0] = lo;
      reinterpret_cast<uint4*>(out)[1] = hi;
    } else {
      float v[16];
      load16<false>(v, in);
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pk_bf16(v[2 * j], v[2 * j + 1]);
      reinterpret_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  } else {
    float v[16] = {};
    if (there) load16<BF16>(v, in);
    // the largest magnitude, as bits: those of infinities and NaNs are above all others'
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, f2u(v[j]) & 0x7fffffffu);
    for (int o = span / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (!there) return;
    // 448 is 1.75 * 2^8: the power of two at or above a 448th is found from exponent and mantissa
    const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);
    const bool bad = top >= 0x7f800000u;
    const uint32_t scale = bad ? 127 : (uint32_t)max(e, 27);
    const float inv = u2f((254 - scale) << 23);  // exact, as the products are
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j] * inv, v[4 * j + 1] * inv, 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2] * inv, v[4 * j + 3] * inv, c, true);
      w[j] = bad ? 0x7f7f7f7fu : (uint32_t)c;
    }
    *reinterpret_cast<uint4*>(out + 16 * u) = make_uint4(w[0], w[1], w[2], w[3]);
    if (u == 0)
      (is_v ? a.cache.v_scales : a.cache.k_scales)[((uint64_t)page * a.cache.heads + h) *
                                                       a.cache.page + at] = (uint8_t)scale;
  }
}

// ---- block-wide helpers ----

// Sum over the threads before this one; *total over all THREADS of them.  All threads take part.
template <int THREADS>
__device__ __forceinline__ int64_t before(int64_t v, int64_t* slots, int64_t* total) {
  constexpr int WAVES = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t upto = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t w = __shfl_up((long long)upto, o, 64);
    if (lane >= o) upto += w;
  }
  __syncthreads();
  if (lane == 63) slots[wave] = upto;
  __syncthreads();
  int64_t base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) base += slots[w];
    all += slots[w];
  }
  *total = all;
  return base + upto - v;
}

// Free pages that the stack's count stands for.
__device__ __forceinline__ int stack_size(const int32_t* count, uint32_t pages, int* bits) {
  const int n = *count;
  if (n >= 0 && (uint32_t)n <= pages) return n;
  *bits |= kCacheArgument;
  return 0;
}

// ---- the pages and slots of a step ----
//
// Two sums over the rows say all: the tokens and the pages that the rows before a row bring.  They are one
// workgroup's work (a row is 8 bytes, four of them a thread's); the tokens follow in the same launch while they
// are few, in a grid of their own otherwise.  Latency bounds both: loads, two sums, the stack or the table,
// stores: 4 us for a token of each of 200 rows, 6 and 7 for 300 000 tokens of 1500 rows (6 MB written).
constexpr int kPlanThreads = 1024, kPlanPer = 4;
constexpr int kPlanWindow = 1024;  // rows of a search in LDS
constexpr int kPlanTokens = 1024;  // tokens of a workgroup of their own

// The sums over the lanes up to this one, no more than `most` (such sums do not depend on their order).
__device__ __forceinline__ uint32_t wave_upto(uint32_t v, uint32_t most) {
  auto add = [&](int moved) { v = min(v + (uint32_t)moved, most); };
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8: rows of 16
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row 0's last into 1, 2's into 3
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // row 1's last into 2 and 3
  return v;
}
// The sums over the threads before this one and over all, no more than `most` (below 2^31).
__device__ __forceinline__ uint32_t plan_before(uint32_t v, uint32_t most, uint32_t* slots, uint32_t* all) {
  constexpr int WAVES = kPlanThreads / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t upto = wave_upto(v, most);
  __syncthreads();
  if (lane == 63) slots[wave] = upto;
  __syncthreads();
  const uint32_t sums = wave_upto(lane < WAVES ? slots[lane] : 0, most);
  *all = (uint32_t)__builtin_amdgcn_readlane((int)sums, WAVES - 1);
  const uint32_t before = wave ? (uint32_t)__builtin_amdgcn_readlane((int)sums, wave - 1) : 0;
  const uint32_t lower = (uint32_t)__shfl_up((int)upto, 1, 64);
  return min(before + (lane ? lower : 0), most);
}

// The tokens t0 .. t1 - 1 (total of them real), whose rows are among the n from `first` on: rows[i] is row
// first + i, in LDS or not.
__device__ __forceinline__ void plan_tokens(const PlanArgs& a, uint32_t t0, uint32_t t1, uint32_t total,
                                            const PlanRow* rows, uint32_t first, uint32_t n) {
  int bits = 0;
  for (uint32_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    int row = -1;
    int64_t position = 0, slot = -1;
    if (t < total) {
      uint32_t lo = 0, hi = n;  // the last row that starts at t or before
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (rows[mid].start <= (int)t) lo = mid;
        else hi = mid;
      }
      const PlanRow r = rows[lo];
      row = (int)(first + lo);
      position = (int64_t)r.have + (int)t - r.start;
      if (r.top >= 0) {
        const uint32_t p = (uint32_t)position, block = a.page.of(p), at = p - block * a.page.size;
        const uint32_t held = a.page.up((uint32_t)r.have);
        int32_t* entry = a.tables + row * a.table_stride + block;
        int page;
        if (block < held) {
          page = *entry;
        } else {
          page = a.free_pages[r.top - (int)(block - held)];
          if (at == 0) *entry = page;
        }
        if ((uint32_t)page < a.pages) slot = (int64_t)page * a.page.size + at;
        else bits |= kCacheArgument;
      }
    }
    a.slots[t] = slot;
    if (a.token_rows) a.token_rows[t] = row;
    if (a.positions) a.positions[t] = position;
  }
  if (bits) flag(a.status, bits);
}

template <bool ALL>
__global__ __launch_bounds__(kPlanThreads) void plan_rows_kernel(PlanArgs a) {
  __shared__ uint32_t slots[kPlanThreads / 64];
  __shared__ int s_used;
  __shared__ PlanRow rows[ALL ? kPlanWindow : 1];
  constexpr int PER = ALL ? 1 : kPlanPer;  // rows of a thread
  const uint32_t most_tokens = a.tokens + 1, most_pages = a.pages + 1;
  const int tid = threadIdx.x;
  int bits = 0;
  if (tid == 0) s_used = 0;
  const int count = stack_size(a.free_count, a.pages, &bits);
  uint32_t tokens_before = 0, pages_before = 0;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += PER * kPlanThreads) {
    const uint32_t first_row = r0 + PER * tid;
    int have[PER], tokens[PER];
    bool ok[PER];
    uint32_t sum = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t r = first_row + i;
      have[i] = r < a.rows ? a.lengths[r] : 0;
      tokens[i] = r < a.rows ? a.added ? a.added[r] : 1 : 0;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      ok[i] = have[i] >= 0 && tokens[i] >= 0 &&
              (int64_t)have[i] + tokens[i] <= (int64_t)a.max_blocks * a.page.size;
      if (!ok[i]) tokens[i] = 0;
      sum = min(sum + (uint32_t)tokens[i], most_tokens);
    }
    uint32_t start[PER];
    start[0] = min(tokens_before + plan_before(sum, most_tokens, slots, &all), most_tokens);
    tokens_before = min(tokens_before + all, most_tokens);
#pragma unroll
    for (int i = 1; i < PER; ++i) start[i] = min(start[i - 1] + (uint32_t)tokens[i - 1], most_tokens);
    // pages, of the rows whose tokens have their places
    int need[PER];
    bool over[PER];
    sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      over[i] = start[i] + (uint32_t)tokens[i] > a.tokens;
      need[i] = ok[i] && !over[i]
                    ? (int)(a.page.up((uint32_t)(have[i] + tokens[i])) - a.page.up((uint32_t)have[i]))
                    : 0;
      sum = min(sum + (uint32_t)need[i], most_pages);
    }
    uint32_t page = min(pages_before + plan_before(sum, most_pages, slots, &all), most_pages);
    pages_before = min(pages_before + all, most_pages);
    int used = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t r = first_row + i;
      const bool enough = need[i] == 0 || page + (uint32_t)need[i] <= (uint32_t)count;
      const bool served = ok[i] && !over[i] && enough;
      if (served && need[i]) used = (int)page + need[i];
      if (r < a.rows) {
        if (!ok[i] || over[i]) bits |= kCacheArgument;
        if (!enough) bits |= kCacheMemory;
        const int at = (int)min(start[i], a.tokens);
        const PlanRow row{at, have[i], !served ? -1 : need[i] ? count - 1 - (int)page : 0, 0};
        if constexpr (ALL) rows[r] = row;
        else a.row_plans[r] = row;
        a.lengths_out[r] = served ? have[i] + tokens[i] : have[i];
        if (a.starts) a.starts[r] = at;
      }
      page = min(page + (uint32_t)need[i], most_pages);
    }
    // (of the rows that need pages, those that are served come first)
    if (used) atomicMax(&s_used, used);
  }
  __syncthreads();
  const uint32_t total = min(tokens_before, a.tokens);
  if (tid == 0) {
    if (a.starts) a.starts[a.rows] = (int)total;
    *a.free_count_out = count - s_used;
    if constexpr (!ALL) a.row_plans[a.rows] = PlanRow{(int)total, 0, -1, 0};
  }
  if (bits) flag(a.status, bits);
  if constexpr (ALL) plan_tokens(a, 0, a.tokens, total, rows, 0, a.rows);
}

__global__ __launch_bounds__(256) void plan_tokens_kernel(PlanArgs a) {
  __shared__ PlanRow rows[kPlanWindow];
  const uint32_t t0 = blockIdx.x * kPlanTokens, t1 = min(t0 + kPlanTokens, a.tokens);
  const uint32_t total = (uint32_t)a.row_plans[a.rows].start;
  // The rows from that of the first token to that of the last: all of them, cut down by probes of every
  // step-th while they are too many for LDS (and the probes tell: many rows may bring no token).
  uint32_t first = 0, n = a.rows;
  while (n > kPlanWindow) {
    const uint32_t step = (n + 255) / 256, at = threadIdx.x * step;
    const int start = at < n ? a.row_plans[first + at].start : 0x7fffffff;
    const uint32_t lower = (uint32_t)max(1, __syncthreads_count(start <= (int)t0));
    const uint32_t upper = (uint32_t)max(1, __syncthreads_count(start < (int)t1));
    const uint32_t skip = (lower - 1) * step, left = min(n, upper * step) - skip;
    first += skip;
    if (left == n) break;
    n = left;
  }
  const PlanRow* from = a.row_plans + first;
  if (n <= kPlanWindow) {
    for (uint32_t i = threadIdx.x; i < n; i += 256) rows[i] = from[i];
    from = rows;
  }
  __syncthreads();
  plan_tokens(a, t0, t1, total, from, first, n);
}

// ---- tables that follow their beams ----

// The rows of a request that take a copy of their parent's last page, one filled in part that stays with a
// lower child; a whole wave, one row per lane.
__device__ __forceinline__ uint64_t copying_rows(const int* parent, const int* length, int width,
                                                 const PageDivision& page) {
  const int i = threadIdx.x & 63;
  const int p = i < width ? parent[i] : -1;
  bool lower = false;
  for (int j = 0; j < width; ++j) lower |= j < i && parent[j] == p;
  const uint32_t n = (uint32_t)length[p < 0 ? 0 : p];
  return __ballot(p >= 0 && lower && page.of(n) * page.size != n);
}

// The pages, lengths and stack of a request's rows, when all requests' dropped pages and copies are known:
// dropped ones go on the stack, copies take theirs off it.  What a page on top is, when it is one that a
// request has just dropped, is looked up in that request's list and not on the stack, which another workgroup
// may not have written yet.  A single request's (ALONE) count, dropped pages, put on the stack already, and, in the
// first wave, rows that copy are known.
template <bool ALONE>
__device__ __forceinline__ void fork_books(const ForkArgs& a, const int* parent, const int* length,
                                           int64_t* slots, int* s_upto, int count, int dropped, uint64_t copying) {
  const uint32_t r = blockIdx.x, row0 = r * a.width;
  const int tid = threadIdx.x, width = (int)a.width;
  int copies_before = 0, copies_all = 0;
  if constexpr (!ALONE) {
    // pages dropped by requests 0 .. q, and copies before this request and in all (fewer than 2^20)
    int64_t copies = 0, all;
    for (uint32_t q0 = 0; q0 < a.requests; q0 += 256) {
      const uint32_t q = q0 + tid;
      const int d = q < a.requests ? a.drops[q] : 0;
      const int64_t c = q < a.requests ? a.copies[q] : 0;
      copies += c << 32 | (q < r ? c : 0);
      const int upto = dropped + (int)before<256>(d, slots, &all) + d;
      if (q < a.requests) s_upto[q] = upto;
      dropped += (int)all;
    }
    (void)before<256>(copies, slots, &all);
    copies_before = (int)(all & 0xffffffff);
    copies_all = (int)(all >> 32);
    const int32_t* list = a.dropped + (uint64_t)row0 * a.max_blocks;
    const int before_r = r ? s_upto[r - 1] : 0, n = s_upto[r] - before_r;
    const int64_t first = (int64_t)count + before_r;
    for (int j = tid; j < n; j += 256)
      if (first + j < a.pages) a.free_pages[first + j] = list[j];
  }
  if (tid >= 64) return;
  if constexpr (ALONE) copies_all = __popcll(copying);
  else copying = copying_rows(parent, length, width, a.page);
  const int64_t room = (int64_t)a.pages - count;  // of the stack
  const int64_t size = count + min((int64_t)dropped, room);
  if (r == 0 && tid == 0) {
    *a.free_count_out = (int)max(size - copies_all, (int64_t)0);
    if (dropped > room) flag(a.status, kCacheArgument);
  }
  if (tid >= width) return;
  const int p = parent[tid];
  int kept = p >= 0 ? length[p] : 0;
  ForkCopy copy{0, 0, 0};
  if (copying >> tid & 1) {
    const int64_t at = size - 1 - copies_before - __popcll(copying & ((1ull << tid) - 1));
    if (at < 0) {
      kept = 0;
      flag(a.status, kCacheMemory);
    } else {
      int to;
      if (at < count) {
        to = a.free_pages[at];
      } else {
        const int want = (int)(at - count);
        uint32_t q = 0, end = ALONE ? 0 : a.requests - 1;  // the first request whose dropped pages end beyond
        while (q < end) {
          const uint32_t mid = (q + end) / 2;
          if (s_upto[mid] > want) end = mid;
          else q = mid + 1;
        }
        to = a.dropped[(uint64_t)q * a.width * a.max_blocks + (want - (q ? s_upto[q - 1] : 0))];
      }
      const uint32_t last = a.page.of((uint32_t)length[p]);
      const int from = a.tables[(uint64_t)(row0 + p) * a.table_stride + last];
      a.tables_out[(uint64_t)(row0 + tid) * a.table_out_stride + last] = to;
      if ((uint32_t)to >= a.pages || (uint32_t)from >= a.pages) flag(a.status, kCacheArgument);
      else copy = ForkCopy{(uint32_t)from, (uint32_t)to, (uint32_t)length[p] - last * a.page.size};
    }
  }
  a.page_copies[row0 + tid] = copy;
  a.lengths_out[row0 + tid] = kept;
}

// One request per workgroup: its rows' tables, and the pages that none of them holds any more.  A page can
// stand in several rows only in one column, so a column is one thread's work.  Latency bounds it (parents and
// lengths, the column, the pages' places): 7 us for 4 rows of 59 pages, 11 for 32 requests of 8 rows of 43.
template <bool ALONE>
__global__ __launch_bounds__(256) void fork_tables_kernel(ForkArgs a) {
  extern __shared__ int column[];  // [width][256]
  __shared__ int parent[kForkWidth], length[kForkWidth];
  __shared__ uint32_t blocks[kForkWidth];
  __shared__ unsigned long long s_used;  // rows with a child
  __shared__ uint32_t s_columns;
  __shared__ int64_t slots[4];
  const uint32_t r = blockIdx.x, row0 = r * a.width;
  const int tid = threadIdx.x, width = (int)a.width;
  int bits = 0;
  if (tid == 0) {
    s_used = 0;
    s_columns = 0;
  }
  __syncthreads();
  // (read with the parents, and written at the end)
  const int count = ALONE || (r == 0 && tid == 0) ? stack_size(a.free_count, a.pages, &bits) : 0;
  if (tid < width) {
    int p = a.parents[row0 + tid];
    if (p >= width) bits |= kCacheArgument;
    parent[tid] = p < 0 || p >= width ? -1 : p;
    int n = a.lengths[row0 + tid];
    if (n < 0 || (int64_t)n > (int64_t)a.max_blocks * a.page.size) {
      bits |= kCacheArgument;
      n = 0;
    }
    length[tid] = n;
    a.old_lengths[row0 + tid] = n;
    blocks[tid] = a.page.up((uint32_t)n);
    if (parent[tid] >= 0) atomicOr(&s_used, 1ull << parent[tid]);
    atomicMax(&s_columns, blocks[tid]);
  }
  __syncthreads();
  uint64_t copying = 0;
  if (tid < 64) {
    copying = copying_rows(parent, length, width, a.page);
    if (!ALONE && tid == 0) a.copies[r] = __popcll(copying);
  }
  const uint64_t used = s_used;
  const uint32_t columns = s_columns;
  const int32_t* in = a.tables + row0 * a.table_stride;
  // Two rows with children that hold the last page of one of them, filled in part, would write over each other's
  // tokens: pair q of rows is compared by its entries in that column.
  struct Pair {
    int mine, other;
  };
  auto entries = [&](int q) -> Pair {
    const int i = q / width, j = q - i * width;
    if (i >= width || i == j || !(used >> i & 1) || !(used >> j & 1)) return Pair{-1, -1};
    const uint32_t last = a.page.of((uint32_t)length[i]);
    if (last == blocks[i] || last >= blocks[j]) return Pair{-1, -1};
    return Pair{in[i * a.table_stride + last], in[j * a.table_stride + last]};
  };
  auto shared = [&](Pair p) { return p.mine == p.other && (uint32_t)p.mine < a.pages; };
  const Pair first_pair = entries(tid);  // (read with the first columns)
  int32_t* out = a.tables_out + row0 * a.table_out_stride;
  int32_t* list = a.dropped + (uint64_t)row0 * a.max_blocks;
  int n_dropped = 0;
  for (uint32_t c0 = 0; c0 < columns; c0 += 256) {
    const uint32_t c = c0 + tid;
    uint64_t held = 0, drop = 0;
#pragma unroll 8
    for (int i = 0; i < width; ++i) held |= (uint64_t)(c < blocks[i]) << i;
    if (held) {
      // the column in LDS (each thread its own): eight loads on their way at a time
      for (int i0 = 0; i0 < width; i0 += 8) {
        int e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = held >> (i0 + i) & 1 ? in[(i0 + i) * a.table_stride + c] : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < width) column[(i0 + i) * 256 + tid] = e[i];
      }
      for (int i = 0; i < width; ++i) {
        const int p = parent[i];
        if (p >= 0 && held >> p & 1) out[i * a.table_out_stride + c] = column[p * 256 + tid];
      }
      for (uint64_t rest = held & ~used; rest; rest &= rest - 1) {
        const int i = __ffsll((unsigned long long)rest) - 1, page = column[i * 256 + tid];
        if ((uint32_t)page >= a.pages) {
          bits |= kCacheArgument;
          continue;
        }
        // held by no row with children, and by no lower row without
        const uint64_t others = held & (used | ((1ull << i) - 1));
        bool gone = true;
        for (int j0 = 0; j0 < width; j0 += 8) {
          int e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = column[min(j0 + j, width - 1) * 256 + tid];
#pragma unroll
          for (int j = 0; j < 8; ++j) gone = gone && !(others >> (j0 + j) & 1 && e[j] == page);
        }
        if (gone) drop |= 1ull << i;
      }
    }
    int64_t all;
    int at = n_dropped + (int)before<256>(__popcll(drop), slots, &all);
    n_dropped += (int)all;
    for (; drop; drop &= drop - 1, ++at) {
      const int page = column[(__ffsll((unsigned long long)drop) - 1) * 256 + tid];
      list[at] = page;
      if (ALONE && (int64_t)count + at < a.pages) a.free_pages[count + at] = page;
    }
  }
  bool twice = shared(first_pair);
  for (int q = 256 + tid; q < width * width; q += 256) twice |= shared(entries(q));
  if (twice) bits |= kCacheArgument;
  if (!ALONE && tid == 0) {
    a.drops[r] = n_dropped;
    if (r == 0) *a.count = count;
  }
  if (bits) flag(a.status, bits);
  if constexpr (ALONE) {
    // a single request has its books done here
    __syncthreads();
    fork_books<true>(a, parent, length, slots, nullptr, count, n_dropped, copying);
  }
}

__global__ __launch_bounds__(256) void fork_books_kernel(ForkArgs a) {
  __shared__ int parent[kForkWidth], length[kForkWidth];
  __shared__ int64_t slots[4];
  __shared__ int s_upto[kForkRequests];
  const int tid = threadIdx.x, width = (int)a.width, count = *a.count;
  if (tid < width) {
    const int p = a.parents[blockIdx.x * a.width + tid];
    parent[tid] = p < 0 || p >= width ? -1 : p;
    length[tid] = a.old_lengths[blockIdx.x * a.width + tid];
  }
  fork_books<false>(a, parent, length, slots, s_upto, count, 0, 0);
}

// Copies the first tokens of one page per blockIdx.x in the cache blockIdx.z; blockIdx.y takes the pieces of
// 16 bytes in turn, four at a time so that a lane has four loads on their way.  Bound by the way to HBM and back, with
// the rows that copy nothing in the grid too, and by the arithmetic of addresses (vector units are busy for 43 % of
// it): 67 MB of 32 x 8 beams in six caches in 20 to 23 us, 2.9 TB/s.
__global__ __launch_bounds__(256) void fork_copy_kernel(const ForkCopy* copies, ForkCaches caches) {
  const ForkCopy copy = copies[blockIdx.x];
  const uint32_t tokens = copy.tokens;
  if (tokens == 0) return;
  const KvCache& c = caches.c[blockIdx.z];
  const bool f8 = c.k_scales != nullptr;
  const uint32_t row16 = c.dim * (f8 ? 1 : 2) / 16;  // pieces of a row
  const uint32_t rows = 2 * c.heads * tokens, items = rows * row16;
  const uint64_t from = copy.from * c.page_stride, to = copy.to * c.page_stride;
  const uint32_t step = gridDim.y * 256;
  constexpr int AHEAD = 4;
  for (uint32_t j0 = blockIdx.y * 256 + threadIdx.x; j0 < items; j0 += AHEAD * step) {
    uint8_t* base[AHEAD];
    uint4 v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const uint32_t j = min(j0 + u * step, items - 1);
      const uint32_t row = j / row16, piece = j - row * row16;
      const uint32_t h2 = row / tokens, t = row - h2 * tokens;
      const bool is_v = h2 >= c.heads;
      base[u] = (is_v ? c.v : c.k) + (is_v ? h2 - c.heads : h2) * c.head_stride + t * c.token_stride + 16 * piece;
      v[u] = ldg16(base[u] + from);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (j0 + u * step < items) *reinterpret_cast<uint4*>(base[u] + to) = v[u];
  }
  if (!f8) return;
  for (uint32_t row = blockIdx.y * 256 + threadIdx.x; row < rows; row += step) {
    const uint32_t h2 = row / tokens, t = row - h2 * tokens;
    const bool is_v = h2 >= c.heads;
    const uint32_t h = is_v ? h2 - c.heads : h2;
    uint8_t* s = is_v ? c.v_scales : c.k_scales;
    s[((uint64_t)copy.to * c.heads + h) * c.page + t] = s[((uint64_t)copy.from * c.heads + h) * c.page + t];
  }
}

}  // namespace

void launch_append(const AppendArgs& a, bool rows_bf16, hipStream_t s) {
  int span = 1;
  while (span < (int)a.cache.dim / 16) span *= 2;
  // tokens of a launch: row numbers of 32 bits, fewer than 2^31 threads
  const uint32_t most = std::max(1u, (1u << 26) / a.cache.heads);
  for (uint32_t t = 0; t < a.tokens; t += most) {
    AppendArgs c = a;
    c.k += t * a.k_token;
    c.v += t * a.v_token;
    c.slots += t;
    c.tokens = std::min(most, a.tokens - t);
    const uint64_t threads = (uint64_t)c.tokens * 2 * a.cache.heads * span;
    const dim3 grid((unsigned)((threads + 255) / 256));
    const bool f8 = a.cache.k_scales != nullptr;
    if (rows_bf16 && f8) append_kernel<true, true><<<grid, 256, 0, s>>>(c, span);
    else if (rows_bf16) append_kernel<true, false><<<grid, 256, 0, s>>>(c, span);
    else if (f8) append_kernel<false, true><<<grid, 256, 0, s>>>(c, span);
    else append_kernel<false, false><<<grid, 256, 0, s>>>(c, span);
  }
}

void launch_plan(const PlanArgs& a, hipStream_t s) {
  // One launch while its workgroup has a few tokens per thread.
  if (a.rows <= kPlanWindow && a.tokens <= 4 * kPlanThreads) {
    plan_rows_kernel<true><<<1, kPlanThreads, 0, s>>>(a);
    return;
  }
  plan_rows_kernel<false><<<1, kPlanThreads, 0, s>>>(a);
  plan_tokens_kernel<<<(a.tokens + kPlanTokens - 1) / kPlanTokens, 256, 0, s>>>(a);
}

void launch_fork(const ForkArgs& a, hipStream_t s) {
  const size_t lds = a.width * 256 * sizeof(int);
  if (a.requests == 1) {
    fork_tables_kernel<true><<<1, 256, lds, s>>>(a);
  } else {
    fork_tables_kernel<false><<<a.requests, 256, lds, s>>>(a);
    fork_books_kernel<<<a.requests, 256, 0, s>>>(a);
  }
}

void launch_fork_copies(const ForkArgs& a, const ForkCaches& caches, uint32_t n, hipStream_t s) {
  uint64_t bytes = 0;
  for (uint32_t i = 0; i < n; ++i)
    bytes = std::max<uint64_t>(bytes, 2ull * caches.c[i].heads * a.page.size * caches.c[i].dim);
  // parts of a page: four pieces for every lane in the largest of E4M3 caches, eight of BF16, while that is no more
  // than 64 workgroups per CU
  const uint32_t rows = a.requests * a.width;
  const uint32_t parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(bytes / 16384, 16384 / (rows * n)));
  fork_copy_kernel<<<dim3(rows, parts, n), 256, 0, s>>>(a.page_copies, caches);
}

}  // namespace urb
