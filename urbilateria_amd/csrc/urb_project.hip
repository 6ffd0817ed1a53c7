// urb_project.hip -- projections of token rows by one packed matrix with a low-rank adapter per row.
//
//   y[t] = W x[t] + scale_a B_a (A_a x[t])
//
// The adapters' first products u = A x come first, into the workspace; then W x, with the second products
// added to the accumulators before they are rounded (without adapters only the latter).
//
// Operands.  W streams in the panel layout (urb_kernels.hpp) straight into MFMA operands, MX codes
// decoded to BF16 in registers (exact).  f32 rows are carried as three BF16 planes: truncating v to
// 8 significant bits, then the rest, then the rest of that, loses none of its 24 bits; planes that are
// zero for a whole operand (rows whose values are BF16 already) are skipped.  u is carried the
// same way, whatever the outputs' type: cut to two planes, 2^-17 of it were lost, ten times what the f32 sums
// lose, and BF16 outputs would round to the other neighbour that much more often.
//
// A tile may hold rows of any adapters: each distinct adapter of a block of 16 rows multiplies the block's
// u with the other adapters' rows set to zero.  A row has one adapter, so the order in which a tile takes
// its adapters changes no sum, and a row's result does not depend on the rows beside it.
//
// What bounds it.  Few rows: the weights' bytes (1 BF16 row, 16384 x 8192: 44.3 us without adapters, 6.1
// TB/s); with adapters the launch of the first products before it and its latency.  Many: the matrix
// instructions (4096 rows of 7168 -> 7168, BF16: 346 to 358 us without adapters, 1.2 PFLOP/s).  f32 rows whose
// values need all 24 bits cost three products.
#include "urb_panel.hpp"
#include "urb_step.hpp"

namespace urb {

namespace {

// Rows of a call that takes tiles.  Below, one block of 16 rows per workgroup and the weights read once; a
// second block reads them again (24 BF16 rows, 8192 -> 16384: 82.2 us, tiles 47.2; MXFP8, 6144 -> 9232: 31 and
// 17.4; only of 16 M values in BF16 10.3 and 12.3).
constexpr int kTileTokens = 17;
constexpr int kMaxSlices = 16;    // most slices of K

// __builtin_amdgcn_sched_barrier: VALU, SALU and LDS reads may cross; loads, LDS stores, MFMAs stay.
constexpr int kHoldLoads = 0x106;

// v as BF16 planes by truncation, v = hi + mid + lo exactly (v finite and not subnormal in the
// lower planes); an infinity keeps its first plane alone.
__device__ __forceinline__ float plane_rest(float v, float hi) { return v == hi ? 0.0f : v - hi; }
__device__ __forceinline__ float trunc_bf16(float v) { return u2f(f2u(v) & 0xffff0000u); }
// the upper halves of two words: a's in the low half
__device__ __forceinline__ uint32_t high_halves(float a, float b) {
  return __builtin_amdgcn_perm(f2u(b), f2u(a), 0x07060302u);
}

// Eight values in P BF16 planes: one for BF16 values, kF32Planes for f32 ones.
constexpr int kF32Planes = 3;
template <int P>
struct Planes {
  uint32_t w[P][4];
  __device__ __forceinline__ bf16x8 operand(int p) const {
    return __builtin_bit_cast(bf16x8, make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]));
  }
};
__device__ __forceinline__ Planes<kF32Planes> split_planes(const float (&v)[8]) {
  Planes<kF32Planes> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < kF32Planes; ++p) {
      r.w[p][i] = high_halves(a, b);
      a = plane_rest(a, trunc_bf16(a));
      b = plane_rest(b, trunc_bf16(b));
    }
  }
  return r;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The eight values at `k` of a token row as MFMA planes: one for BF16 rows, three for f32 ones.
template <bool XB>
constexpr int x_planes() { return XB ? 1 : kF32Planes; }
template <bool XB>
__device__ __forceinline__ Planes<x_planes<XB>()> load_x(const uint8_t* row, int k) {
  if constexpr (XB) {
    const uint4 q = ldg16(row + 2 * (size_t)k);
    return {{{q.x, q.y, q.z, q.w}}};
  } else {
    const float4 a = u2f4(ldg16(row + 4 * (size_t)k)), b = u2f4(ldg16(row + 4 * (size_t)k + 16));
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return split_planes(v);
  }
}
// The same as loaded, for loads ahead of their use.
template <bool XB>
struct XRaw {
  uint4 q[XB ? 1 : 2];
  __device__ __forceinline__ void load(const uint8_t* row, int k) {
    q[0] = ldg16(row + (XB ? 2 : 4) * (size_t)k);
    if constexpr (!XB) q[1] = ldg16(row + 4 * (size_t)k + 16);
  }
  __device__ __forceinline__ Planes<x_planes<XB>()> planes() const {
    if constexpr (XB) {
      return {{{q[0].x, q[0].y, q[0].z, q[0].w}}};
    } else {
      const float4 a = u2f4(q[0]), b = u2f4(q[1]);
      const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      return split_planes(v);
    }
  }
};
// acc += w * x over the planes of x that hold anything for some lane.
template <int P>
__device__ __forceinline__ f32x4 mma_planes(bf16x8 w, const Planes<P>& x, f32x4 acc) {
  acc = mfma(w, x.operand(0), acc);
  if constexpr (P == kF32Planes) {
    if (__ballot((x.w[1][0] | x.w[1][1] | x.w[1][2] | x.w[1][3]) != 0)) {
      acc = mfma(w, x.operand(1), acc);
      acc = mfma(w, x.operand(2), acc);
    }
  }
  return acc;
}

// ---- u = A x for every row with an adapter ----

constexpr int kFew = 64;  // rows whose adapters a wave sorts out by itself

constexpr int kOrderThreads = 1024;
constexpr int kMaxPass = 8192;   // most rows of a pass
constexpr int kMaxSlots = 4096;
static_assert(kMaxSlots == 4 * kOrderThreads, "four slots per thread");

// Adds one to count[id] for every lane with id >= 0; returns what was there before the lane's own (lanes of
// one id get consecutive values).  Ids that many lanes share, as in a batch sorted by request, are
// counted by one atomic: 64 on one address take turns.
__device__ __forceinline__ int count_up(int* count, int id) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  for (int round = 0; round < 4; ++round) {
    const uint64_t open = __ballot(id >= 0);
    if (!open) return at;
    const int some = __shfl(id, __ffsll((unsigned long long)open) - 1, 64);
    const uint64_t same = __ballot(id == some);
    if (__popcll(same) < 8) break;
    int first = 0;
    if (lane == __ffsll((unsigned long long)same) - 1) first = atomicAdd(&count[some], __popcll(same));
    first = __shfl(first, __ffsll((unsigned long long)same) - 1, 64);
    if (id == some) {
      at = first + __popcll(same & ((1ull << lane) - 1));
      id = -1;
    }
  }
  return id >= 0 ? atomicAdd(&count[id], 1) : at;
}

// The rows in order of their adapters, those without one last, and the blocks of up to 16 rows of one
// adapter: slot, first place in the order, rows.  One workgroup; `order` holds `tokens` entries, `blocks`
// (3 ints each) at most order_blocks().  Which row of an adapter comes first is left to chance: no sum goes
// over rows.
__global__ __launch_bounds__(kOrderThreads) void order_kernel(ProjArgs p, int* order, int* blocks,
                                                              int* n_blocks) {
  __shared__ int count[kMaxSlots];  // rows per slot, then the place of its next one (-1: an empty slot)
  __shared__ int row_at[kMaxSlots + 1], tile_at[kMaxSlots];  // first row and block of each slot
  __shared__ int s_blocks, s_idle;
  __shared__ int waves[2][kOrderThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < p.slots; i += kOrderThreads) count[i] = 0;
  __syncthreads();
  // (all ids at once: the loads of a loop would wait for the atomics before them)
  constexpr int PER = kMaxPass / kOrderThreads;
  int ids[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int t = j * kOrderThreads + tid;
    ids[j] = t < p.tokens ? p.ids[t] : -1;
  }
  bool bad = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (ids[j] >= p.slots) {
      bad = true;
      ids[j] = -1;
    }
    if (j * kOrderThreads < p.tokens) count_up(count, ids[j]);
  }
  __syncthreads();
  // four slots per thread, in order: running sums of rows and of blocks
  int n[4], rows = 0, tiles = 0;
  bool filled[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int slot = 4 * tid + j;
    n[j] = slot < p.slots ? count[slot] : 0;
    filled[j] = n[j] && p.table[slot].rank > 0;
    if (n[j] && !filled[j]) {
      bad = true;
      n[j] = 0;
    }
    rows += n[j];
    tiles += (n[j] + 15) / 16;
  }
  if (bad) flag(p.status, kStepArgument);
  int row = rows, tile = tiles;
  for (int o = 1; o < 64; o <<= 1) {
    const int r = __shfl_up(row, o, 64), b = __shfl_up(tile, o, 64);
    if (lane >= o) {
      row += r;
      tile += b;
    }
  }
  if (lane == 63) {
    waves[0][wave] = row;
    waves[1][wave] = tile;
  }
  __syncthreads();
  row -= rows;
  tile -= tiles;
  for (int w = 0; w < wave; ++w) {
    row += waves[0][w];
    tile += waves[1][w];
  }
  if (tid == kOrderThreads - 1) {
    *n_blocks = tile + tiles;
    s_blocks = tile + tiles;
    s_idle = row + rows;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int slot = 4 * tid + j;
    if (slot < p.slots) count[slot] = filled[j] ? row : -1;
    row_at[slot] = row;
    tile_at[slot] = tile;
    row += n[j];
    tile += (n[j] + 15) / 16;
  }
  if (tid == kOrderThreads - 1) row_at[kMaxSlots] = row;
  __syncthreads();
  // the slot of each block: the last whose blocks begin at or before it
  for (int b = tid; b < s_blocks; b += kOrderThreads) {
    int lo = 0;
#pragma unroll
    for (int step = kMaxSlots / 2; step > 0; step /= 2)
      if (tile_at[lo + step] <= b) lo += step;
    const int from = row_at[lo] + 16 * (b - tile_at[lo]);
    blocks[3 * b] = lo;
    blocks[3 * b + 1] = from;
    blocks[3 * b + 2] = min(16, row_at[lo + 1] - from);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kOrderThreads >= p.tokens) break;
    const int t = j * kOrderThreads + tid;
    const int id = ids[j] >= 0 && count[ids[j]] >= 0 ? ids[j] : -1;
    int at = count_up(count, id);
    const uint64_t idle = __ballot(id < 0 && t < p.tokens);
    int first = 0;
    if (lane == 0 && idle) first = atomicAdd(&s_idle, (int)__popcll(idle));
    first = __shfl(first, 0, 64);
    if (id < 0) at = first + (int)__popcll(idle & ((1ull << lane) - 1));
    if (t < p.tokens) order[at] = t;
  }
}

// Rank r's value of an adapter's first product, scaled.  Ranks past the adapter's own pad it to a whole panel
// with rows of A that are zero, whose products with an infinite or NaN x are NaN: they are zeros here.
__device__ __forceinline__ float scaled(const AdapterEntry& e, int r, float v) {
  return r < e.rank ? v * e.scale : 0.0f;
}

// The adapters' first products, as the planes that the second ones multiply: planes[(t * kF32Planes + plane) *
// ld + rank], scaled.
struct FirstProduct {
  uint16_t* planes;
  int ld;
};
// The rows in order of their adapters (NULL: few rows), and order_kernel's blocks (NULL: each workgroup finds
// its own and writes its part of the order).
struct Order {
  int* order;
  const int* blocks;
  const int* n_blocks;
};

constexpr int kPrepareWaves = 16;
constexpr int kOwnBlocks = 64 * kPrepareWaves;  // most rows whose blocks each workgroup finds for itself

// The unit-th block of up to 16 rows of one adapter (slots ascending, rows ascending, at last the blocks
// of rows without an adapter) of at most kOwnBlocks rows: what order_kernel finds for all, by each workgroup
// for itself, which costs less than that launch (calls of 131 and of 1000 rows: 68.6 -> 66.0 and 77.1 -> 74.2
// us).  Returns the rows in it (0: no such block), their numbers in rows[], its slot (-1: none) and
// its first place in the order.
__device__ __forceinline__ int find_block(const ProjArgs& p, int unit, int* count, int* rows, int* slot,
                                          int* place) {
  __shared__ int waves[kPrepareWaves], s_slot, s_z, s_place;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = tid < p.tokens ? p.ids[tid] : -1;
  constexpr int PER = kMaxSlots / (64 * kPrepareWaves);
  bool filled[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = PER * tid + j;
    filled[j] = i < p.slots && p.table[i].rank > 0;
    if (i < p.slots) count[i] = 0;
  }
  if (tid == 0) s_slot = -1;
  bool bad = id >= p.slots;
  if (bad || id < 0) id = -1;
  __syncthreads();
  count_up(count, id);
  __syncthreads();
  // running sums of rows (high half) and of blocks (low half)
  int n[PER], sums = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = PER * tid + j;
    n[j] = i < p.slots ? count[i] : 0;
    if (!filled[j]) {
      bad |= n[j] != 0;
      n[j] = 0;
      if (i < p.slots) count[i] = -1;
    }
    sums += (n[j] << 16) + (n[j] + 15) / 16;
  }
  if (bad && blockIdx.x == 0 && blockIdx.y == 0) flag(p.status, kStepArgument);
  int upto = sums;
  for (int o = 1; o < 64; o <<= 1) {
    const int b = __shfl_up(upto, o, 64);
    if (lane >= o) upto += b;
  }
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  int at = upto - sums, all = 0;
#pragma unroll
  for (int w = 0; w < kPrepareWaves; ++w) {
    if (w < wave) at += waves[w];
    all += waves[w];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int next = at + (n[j] << 16) + (n[j] + 15) / 16;
    if (unit >= (at & 0xffff) && unit < (next & 0xffff)) {
      s_slot = PER * tid + j;
      s_z = unit - (at & 0xffff);
      s_place = at >> 16;
    }
    at = next;
  }
  if (id >= 0 && count[id] < 0) id = -1;
  __syncthreads();
  *slot = s_slot;
  const bool idle = *slot < 0;
  const int z = idle ? unit - (all & 0xffff) : s_z;
  *place = (idle ? all >> 16 : s_place) + 16 * z;
  const bool mine = tid < p.tokens && id == *slot;
  const uint64_t same = __ballot(mine);
  if (lane == 0) waves[wave] = (int)__popcll(same);
  __syncthreads();
  int first = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kPrepareWaves; ++w) {
    total += waves[w];
    if (w < wave) first += waves[w];
  }
  first += (int)__popcll(same & ((1ull << lane) - 1)) - 16 * z;
  if (mine && first >= 0 && first < 16) rows[first] = tid;
  __syncthreads();
  return max(0, min(16, total - 16 * z));
}

// One row of f32 values as planes [3][tokens][cols], and how many of them it needs (1: its values are
// BF16).  All threads of a workgroup.
__device__ __forceinline__ void row_planes(const ProjArgs& p, int t, uint16_t* x_planes, int* needed) {
  const uint8_t* row = reinterpret_cast<const uint8_t*>(p.x) + (size_t)t * p.x_stride * 4;
  bool more = false;
  for (int c = 8 * threadIdx.x; c < p.cols; c += 8 * blockDim.x) {
    const Planes<kF32Planes> v = load_x<false>(row, c);
#pragma unroll
    for (int pl = 0; pl < kF32Planes; ++pl)
      *reinterpret_cast<uint4*>(x_planes + ((size_t)pl * p.tokens + t) * p.cols + c) =
          make_uint4(v.w[pl][0], v.w[pl][1], v.w[pl][2], v.w[pl][3]);
    more |= (v.w[1][0] | v.w[1][1] | v.w[1][2] | v.w[1][3]) != 0;
  }
  more = __syncthreads_or(more);
  if (threadIdx.x == 0) needed[t] = more ? kF32Planes : 1;
}

// What the products of a call need beforehand, in one launch.  Workgroups below `firsts`: the first product
// of up to 16 rows of one adapter with up to `per` of its 16-rank panels (per 1 or 4), the waves' parts of K
// summed in order.  With an order, a workgroup takes a block of it, or of up to 1024 rows finds its own
// (find_block); of up to 64 rows workgroup (who, panels, z) takes the z-th 16 rows of slot `who`, or (by_token) of the
// slot of row `who` if no row before has it.
// In a grid of several rows each takes a slice of K and writes its sum to u_parts [slice][tokens][ld]
// for finish_kernel.  The other workgroups: a row of f32 values each (row_planes).
template <bool XB>
__global__ __launch_bounds__(64 * kPrepareWaves) void prepare_kernel(
    ProjArgs p, FirstProduct u, float* u_parts, Order order, int firsts, int groups, int per,
    bool by_token, uint16_t* x_planes, int* needed) {
  __shared__ f32x4 red[kPrepareWaves][4][64];
  __shared__ int s_rows[kFew];
  static_assert(sizeof(red) >= kMaxSlots * 4, "counts before, sums after");
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if ((int)blockIdx.x >= firsts) {
    if constexpr (!XB) row_planes(p, blockIdx.x - firsts, x_planes, needed);
    return;
  }
  const int group = blockIdx.x % groups, unit = blockIdx.x / groups;
  int slot, n, t;
  if (order.blocks) {
    if (unit >= *order.n_blocks) return;
    slot = order.blocks[3 * unit];
    n = order.blocks[3 * unit + 2];
    t = order.order[order.blocks[3 * unit + 1] + min(ln, n - 1)];
  } else if (p.tokens > kFew) {
    int place;
    n = find_block(p, unit, reinterpret_cast<int*>(red), s_rows, &slot, &place);
    if (group == 0 && blockIdx.y == 0 && tid < n) order.order[place + tid] = s_rows[tid];
    if (n == 0 || slot < 0) return;
    t = s_rows[min(ln, n - 1)];
  } else {
    const int tiles = (p.tokens + 15) / 16, who = unit / tiles, z = unit % tiles;
    const int id = lane < p.tokens ? p.ids[lane] : -1;
    if (blockIdx.x == 0 && blockIdx.y == 0 && wave == 0 && id >= 0 &&
        (id >= p.slots || p.table[id].rank == 0))
      flag(p.status, kStepArgument);
    slot = by_token ? __builtin_amdgcn_readlane(id, who) : who;
    if (slot < 0 || slot >= p.slots) return;
    const uint64_t same = __ballot(id == slot);
    if (by_token && __ffsll((unsigned long long)same) - 1 != who) return;
    n = min(16, (int)__popcll(same) - 16 * z);  // (unsigned, it would never be negative)
    if (n <= 0) return;
    if (id == slot) s_rows[__popcll(same & ((1ull << lane) - 1))] = lane;  // (the same from every wave)
    __syncthreads();
    t = s_rows[16 * z + min(ln, n - 1)];
  }
  const AdapterEntry e = p.table[slot];
  const int steps = p.cols / 32, panels = (e.rank + 15) / 16;
  const int q0 = group * per, nq = min(per, panels - q0);
  if (nq <= 0) return;
  const int waves = kPrepareWaves * gridDim.y, part = kPrepareWaves * blockIdx.y + wave;
  const int s0 = steps * part / waves, s1 = steps * (part + 1) / waves;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(p.x) + (size_t)t * p.x_stride * (XB ? 2 : 4);
  const uint16_t* a = p.a + (size_t)slot * p.a_slot + 8 * lane;
  f32x4 acc[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
  // (loads in batches: the check for empty planes is a branch, across which none would be moved)
  auto sweep = [&](auto count) {
    constexpr int NQ = decltype(count)::value, BATCH = XB || NQ <= 2 ? 4 : 2;
    for (int s = s0; s < s1; s += BATCH) {
      XRaw<XB> xv[BATCH];
      uint4 w[BATCH][NQ];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int si = min(s + i, s1 - 1);
        xv[i].load(row, 32 * si + 8 * lq);
#pragma unroll
        for (int q = 0; q < NQ; ++q) w[i][q] = ldg16(a + ((size_t)(q0 + q) * steps + si) * 512);
      }
      __builtin_amdgcn_sched_barrier(kHoldLoads);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (s + i >= s1) break;
        const auto x = xv[i].planes();
#pragma unroll
        for (int q = 0; q < NQ; ++q)
          acc[q] = mma_planes(__builtin_bit_cast(bf16x8, w[i][q]), x, acc[q]);
      }
    }
  };
  if (nq == 1) sweep(Int<1>{});
  else if (nq == 2) sweep(Int<2>{});
  else if (nq == 3) sweep(Int<3>{});
  else sweep(Int<4>{});
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (q < nq) red[wave][q][lane] = acc[q];
  __syncthreads();
  if (wave < nq && ln < n) {
    // lane (ln, lq) holds ranks 4 lq + [0, 4) of row ln
    f32x4 v = red[0][wave][lane];
#pragma unroll
    for (int z = 1; z < kPrepareWaves; ++z) v += red[z][wave][lane];
    if (gridDim.y > 1) {
      *reinterpret_cast<f32x4*>(u_parts + ((size_t)blockIdx.y * p.tokens + t) * u.ld +
                                16 * (q0 + wave) + 4 * lq) = v;
      return;
    }
    const int r = 16 * (q0 + wave) + 4 * lq;
    const float w[8] = {scaled(e, r, v[0]), scaled(e, r + 1, v[1]), scaled(e, r + 2, v[2]),
                        scaled(e, r + 3, v[3])};
    const Planes<kF32Planes> planes = split_planes(w);
#pragma unroll
    for (int pl = 0; pl < kF32Planes; ++pl)
      *reinterpret_cast<uint2*>(u.planes + ((size_t)t * kF32Planes + pl) * u.ld + r) =
          make_uint2(planes.w[pl][0], planes.w[pl][1]);
  }
}

// (a thread per eight values of a row of 8192: 131 rows of 7168 in 6.6 us; with 256 threads 7.7)
constexpr int kFinishThreads = 1024;
// The slices' sums of a row's first product, in order, as planes; and the row's own planes (x_planes).
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(
    ProjArgs p, FirstProduct u, const float* u_parts, int slices, uint16_t* x_planes, int* needed) {
  const int t = blockIdx.x;
  const int id = p.ids[t], r = 8 * threadIdx.x;
  AdapterEntry e{0, 0.0f};
  if (id >= 0 && id < p.slots) e = p.table[id];
  if (r < 16 * ((e.rank + 15) / 16)) {  // (as many as the panels wrote)
    float v[8] = {};
    const float* from = u_parts + (size_t)t * u.ld + r;
#pragma unroll 8
    for (int z = 0; z < slices; ++z) {
      const float4 c = *reinterpret_cast<const float4*>(from);
      const float4 d = *reinterpret_cast<const float4*>(from + 4);
      v[0] += c.x; v[1] += c.y; v[2] += c.z; v[3] += c.w;
      v[4] += d.x; v[5] += d.y; v[6] += d.z; v[7] += d.w;
      from += (size_t)p.tokens * u.ld;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = scaled(e, r + j, v[j]);
    const Planes<kF32Planes> out = split_planes(v);
#pragma unroll
    for (int pl = 0; pl < kF32Planes; ++pl)
      *reinterpret_cast<uint4*>(u.planes + ((size_t)t * kF32Planes + pl) * u.ld + r) =
          make_uint4(out.w[pl][0], out.w[pl][1], out.w[pl][2], out.w[pl][3]);
  }
  if (x_planes) row_planes(p, t, x_planes, needed);
}

// ---- the second products, added to a tile's accumulators ----

// The slots of a tile's rows (-1: none) and its distinct filled ones, in LDS.
template <int MAX>
struct TileSlots {
  int ids[MAX], rows[MAX];
  int2 list[MAX];  // slot, rank units
  int n;
  uint32_t seen[kMaxSlots / 32];
};
template <int MAX>
__device__ __forceinline__ void find_slots(const ProjArgs& p, const int* order, int t0, int count,
                                           TileSlots<MAX>& s) {
  const int tid = threadIdx.x;
  if (tid == 0) s.n = 0;
  for (int i = tid; i < kMaxSlots / 32; i += blockDim.x) s.seen[i] = 0;
  __syncthreads();
  for (int i = tid; i < MAX; i += blockDim.x) {
    const int t = t0 + min(i, count - 1), row = order ? order[t] : t;
    s.rows[i] = row;
    int id = i < count ? p.ids[row] : -1;
    int rank = 0;
    if (id >= p.slots || (id >= 0 && (rank = p.table[id].rank) == 0)) id = -1;
    s.ids[i] = id;
    if (id < 0) continue;
    const uint32_t bit = 1u << (id & 31);
    if (!(atomicOr(&s.seen[id >> 5], bit) & bit))
      s.list[atomicAdd(&s.n, 1)] = make_int2(id, (rank + 7) / 8);
  }
  __syncthreads();
}

// The B operands of `units` rank units from r on, of a panel (zero past the last).
__device__ __forceinline__ bf16x8 load_up(const uint16_t* b, int r, int units) {
  const int lane = threadIdx.x & 63, lq = lane >> 4;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (r + lq < units) w = ldg16(b + (size_t)r * 128 + 8 * lane);
  return __builtin_bit_cast(bf16x8, w);
}

// acc[q][m] (lane (ln, lq): rows 16 (panel0 + q) + 4 lq + [0, 4) of the tile's row 16 m + ln) +=
// the adapters' parts.  Of `parts` accumulators that are added up afterwards, each takes the slots with
// slot % parts == part: a row's sum then has the same order in any batch.  B comes from HBM the first
// time, so the next operands are loaded before the present ones are used.
template <int MAX, int NP, int MB>
__device__ __forceinline__ void add_adapters(const ProjArgs& p, const TileSlots<MAX>& s,
                                             const FirstProduct& u, int panel0, int panels,
                                             int part, int parts, f32x4 (&acc)[NP][MB]) {
  const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
  int i = -1, r = 0, slot = 0, units = 0;
  // the next 32 ranks: of this slot or the next of this part; false past the last
  auto advance = [&] {
    r += 4;
    if (r < units) return true;
    r = 0;
    while (++i < s.n) {
      slot = __builtin_amdgcn_readfirstlane(s.list[i].x);
      units = __builtin_amdgcn_readfirstlane(s.list[i].y);
      if (slot % parts == part) return true;
    }
    return false;
  };
  auto load = [&](bf16x8* w) {
    const uint16_t* b = p.b + (size_t)slot * p.b_slot;
#pragma unroll
    for (int q = 0; q < NP; ++q)
      w[q] = load_up(b + (size_t)min(panel0 + q, panels - 1) * units * 128, r, units);
  };
  bf16x8 next[NP];
  bool more = advance();
  if (more) load(next);
  while (more) {
    bf16x8 w[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) w[q] = next[q];
    const int now = slot, from = r, to = units;
    more = advance();
    if (more) load(next);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int local = 16 * m + ln;
      const bool mine = s.ids[local] == now;
      if (!__ballot(mine)) continue;
      bf16x8 v[kF32Planes];
#pragma unroll
      for (int pl = 0; pl < kF32Planes; ++pl) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (mine && from + lq < to)
          x = ldg16(u.planes + ((size_t)s.rows[local] * kF32Planes + pl) * u.ld + 8 * (from + lq));
        v[pl] = __builtin_bit_cast(bf16x8, x);
      }
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int pl = 0; pl < kF32Planes; ++pl) acc[q][m] = mfma(w[q], v[pl], acc[q][m]);
    }
  }
}

// Four consecutive outputs of a token.
template <bool YB>
__device__ __forceinline__ void store_y(const ProjArgs& p, int t, int row, f32x4 v) {
  const size_t at = (size_t)t * p.y_stride + row;
  if constexpr (YB) {
    uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + at;
    const uint32_t a = pk_bf16(v[0], v[1]), b = pk_bf16(v[2], v[3]);
    if (reinterpret_cast<uintptr_t>(y) % 8 == 0) {
      *reinterpret_cast<uint2*>(y) = make_uint2(a, b);
    } else {
      y[0] = (uint16_t)a; y[1] = (uint16_t)(a >> 16);
      y[2] = (uint16_t)b; y[3] = (uint16_t)(b >> 16);
    }
  } else {
    float* y = reinterpret_cast<float*>(p.y) + at;
    if (reinterpret_cast<uintptr_t>(y) % 16 == 0) {
      *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      y[0] = v[0]; y[1] = v[1]; y[2] = v[2]; y[3] = v[3];
    }
  }
}

// ---- W x for up to 16 tokens: eight waves split K of one panel ----
constexpr int kSplitWaves = 8;

// ALONE: the tile computes its rows' first products itself, every workgroup all of them (kAloneRanks of at
// most: rows times ranks), its waves over the K they have anyway.
constexpr int kAloneRanks = 32;
constexpr double kAloneBytes = 50e6;

template <int FMT, bool XB, bool YB, bool ALONE>
__global__ __launch_bounds__(64 * kSplitWaves) void split_kernel(ProjArgs p, FirstProduct u) {
  constexpr int UP = kAloneRanks / 16;
  __shared__ f32x4 red_u[ALONE ? kSplitWaves : 1][UP][64];
  __shared__ f32x4 red[kSplitWaves][64];
  __shared__ TileSlots<16> slots;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lq = lane >> 4;
  const int count = p.tokens, panel = blockIdx.x;
  const int steps = p.cols / kGemmKStep;
  const int s0 = steps * wave / kSplitWaves, s1 = steps * (wave + 1) / kSplitWaves;
  const size_t pbytes = kPanelRows * panel_row_bytes<FMT>(p.cols);
  const size_t pscales = (size_t)kPanelRows * (p.cols / 32);
  const uint8_t* const pd = p.data + panel * pbytes;
  const uint8_t* const ps = FMT == kFmtBF16 ? nullptr : p.scales + panel * pscales;
  const uint8_t* const row =
      reinterpret_cast<const uint8_t*>(p.x) + (size_t)min(ln, count - 1) * p.x_stride * (XB ? 2 : 4);
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  // Weights DW steps ahead in a ring of R slots, rows one step ahead (loaded where they are used, every
  // step waits for the L2).
  constexpr int R = FMT == kFmtBF16 ? 2 : 4, DW = R - 1;
  BRaw<FMT> ring[R];
  XRaw<XB> xr[2][4];
  auto fetch = [&](int slot, int s) { load_b<FMT>(ring[slot], pd, 16u * lane, ps, lane, s); };
  auto fetch_rows = [&](int half, int s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) xr[half][j].load(row, kGemmKStep * s + frag_k<FMT>(j, lq));
  };
#pragma unroll
  for (int d = 0; d < DW; ++d)
    if (s0 + d < s1) fetch(d, s0 + d);
  if (s0 < s1) fetch_rows(0, s0);
  if (p.ids) {
    find_slots(p, nullptr, 0, count, slots);
    if constexpr (ALONE) {
      if (blockIdx.x == 0 && (int)threadIdx.x < count) {
        const int id = p.ids[threadIdx.x];
        if (id >= 0 && slots.ids[threadIdx.x] < 0) flag(p.status, kStepArgument);
      }
      int at = 0;
      for (int i = 0; i < slots.n; ++i) {
        const int slot = slots.list[i].x;
        const uint16_t* a = p.a + (size_t)slot * p.a_slot + 8 * lane;
        for (int q = 0; 2 * q < slots.list[i].y; ++q, ++at) {
          f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
          for (int s = s0; s < s1; ++s) {
            XRaw<XB> xv[4];
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              xv[j].load(row, kGemmKStep * s + 32 * j + 8 * lq);
              w[j] = ldg16(a + ((size_t)q * (4 * steps) + 4 * s + j) * 512);
            }
            __builtin_amdgcn_sched_barrier(kHoldLoads);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v = mma_planes(__builtin_bit_cast(bf16x8, w[j]), xv[j].planes(), v);
          }
          red_u[wave][at][lane] = v;
        }
      }
    } else {
      add_adapters(p, slots, u, panel, panel + 1, wave, kSplitWaves, acc);
    }
  }
  for (int i0 = s0; i0 < s1; i0 += R) {
#pragma unroll
    for (int d = 0; d < R; ++d) {
      const int s = i0 + d;
      if (s >= s1) break;
      if (s + DW < s1) fetch((d + DW) % R, s + DW);
      if (s + 1 < s1) fetch_rows((d + 1) & 1, s + 1);
      __builtin_amdgcn_sched_barrier(kHoldLoads);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 w = decode_b<FMT>(ring[d], j);
        acc[0][0] = mma_planes(w, xr[d & 1][j].planes(), acc[0][0]);
      }
    }
  }
  red[wave][lane] = acc[0][0];
  __syncthreads();
  if (wave > 0) return;
  f32x4 v = red[0][lane];
#pragma unroll
  for (int z = 1; z < kSplitWaves; ++z) v += red[z][lane];  // K parts in order
  if constexpr (ALONE) {
    int at = 0;
    for (int j = 0; p.ids && j < slots.n; ++j) {
      // the lane's eight ranks: of panel lq / 2, held four each by two lanes of its row
      const int slot = slots.list[j].x, units = slots.list[j].y;
      const bf16x8 w = load_up(p.b + (size_t)slot * p.b_slot + (size_t)panel * units * 128, 0, units);
      float uv[8] = {};
      if (slots.ids[ln] == slot && lq < units) {
        const int from = 32 * (lq & 1) + ln;
        f32x4 lo = red_u[0][at + lq / 2][from], hi = red_u[0][at + lq / 2][from + 16];
#pragma unroll
        for (int z = 1; z < kSplitWaves; ++z) {
          lo += red_u[z][at + lq / 2][from];
          hi += red_u[z][at + lq / 2][from + 16];
        }
        const AdapterEntry e = p.table[slot];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uv[r] = scaled(e, 8 * lq + r, lo[r]);
          uv[4 + r] = scaled(e, 8 * lq + 4 + r, hi[r]);
        }
      }
      const Planes<kF32Planes> planes = split_planes(uv);
#pragma unroll
      for (int pl = 0; pl < kF32Planes; ++pl) v = mfma(w, planes.operand(pl), v);
      at += (units + 1) / 2;
    }
  }
  if (ln < count) store_y<YB>(p, ln, panel * kPanelRows + 4 * lq, v);
}

// ---- W x for many tokens: tiles of MB 16-token blocks by kTileWaves x NP panels ----
//
// Each wave multiplies NP panels by all MB blocks.  Weights go from L2 straight into registers
// (a panel's slab is an MFMA operand as it lies), two slabs ahead; rows go through registers into LDS,
// one step of 128 values ahead, in two halves between the step's MFMAs.  Row m's chunk c (16 bytes) of a
// step lies at position c ^ x_swizzle(m) of the row's 256 bytes: a wave stores 1 KiB in a run, and the 16
// lanes that an LDS read serves at a time hit 16 distinct bank groups.  Scheduling fences hold the loads
// where they are written; left alone, the compiler sinks them to just before their use.
constexpr int kTileStep = kGemmKStep;
constexpr int kTileWaves = 4;

template <int FMT>
__device__ __forceinline__ int x_swizzle(int m) {
  // chunks read together: c and c ^ 1 (BF16), c and c ^ 4 (MX: frag_k)
  return FMT == kFmtBF16 ? m & 15 : (m & 3) | ((m & 8) ? 12 : 0);
}

// Slabs of a panel per step, and the operands in each.
template <int FMT>
constexpr int tile_slabs() { return FMT == kFmtMXFP4 ? 1 : FMT == kFmtMXFP8 ? 2 : 4; }
template <int FMT>
__device__ __forceinline__ bf16x8 tile_operand(const uint4& q, float sc, int part) {
  if constexpr (FMT == kFmtBF16) {
    return __builtin_bit_cast(bf16x8, q);
  } else if constexpr (FMT == kFmtMXFP4) {
    const uint32_t w = part == 0 ? q.x : part == 1 ? q.y : part == 2 ? q.z : q.w;
    return pack8(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
  } else {
    const uint32_t w0 = part ? q.z : q.x, w1 = part ? q.w : q.y;
    return pack8(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, false),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, sc, true),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, false),
                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, sc, true));
  }
}

// Rows in BF16 planes: plane i of row t is `plane` bytes after plane i - 1 of it; `planes`: how many of them
// each row needs (NULL: one).  `order`: the rows by adapter (NULL: as they lie), so that a block of 16 holds
// rows of one or two adapters instead of as many as the batch has: each adapter of a block multiplies all
// of it (16 adapters of rank 64 mixed over 1000 rows, BF16, 4096 -> 4096: 96.7 -> 71.7 us; 32 over 3000 178 ->
// 132; already in order 71.0 and 71.2).
struct TileRows {
  size_t plane;
  const int* planes;
  const int* order;
};

// Tiles by workgroup.  Workgroup b runs on XCD b % 8, which has an L2 of its own: the tiles are cut into
// 8 rectangles of by_rows x by_cols XCDs, so that an XCD reads a part of the rows and a part of the weights
// (all of both otherwise).  Within it, bands of `band` row tiles are walked column by column.
struct TileGrid {
  int rows, cols;        // tiles
  int by_rows, by_cols;  // XCDs
  int band;
  __host__ __device__ int tall() const { return (rows + by_rows - 1) / by_rows; }
  __host__ __device__ int wide() const { return (cols + by_cols - 1) / by_cols; }
  __device__ bool place(int block, int* row, int* col) const {
    const int xcd = block % 8, i = block / 8, h = tall(), w = wide();
    const int b = i / (band * w), in = i - b * band * w;
    const int here = min(band, h - b * band);  // rows of this band
    const int r = b * band + in % here, c = in / here;
    *row = xcd % by_rows * h + r;
    *col = xcd / by_rows * w + c;
    return r < h && c < w && *row < rows && *col < cols;
  }
};

template <int FMT, bool YB, int MB, int NP>
__global__ __launch_bounds__(64 * kTileWaves, 2) void tile_kernel(
    ProjArgs p, TileRows rows, FirstProduct u, TileGrid grid, float* parts) {
  constexpr int TM = 16 * MB, TN = kTileWaves * NP;  // tokens, panels
  constexpr int COPIES = TM * 16 / (64 * kTileWaves), HALF = COPIES / 2;  // per thread and step
  constexpr int SL = tile_slabs<FMT>(), PARTS = 4 / SL;
  constexpr bool MX = FMT != kFmtBF16;
  __shared__ __attribute__((aligned(16))) u16 x0[TM * kTileStep];
  __shared__ __attribute__((aligned(16))) u16 x1[TM * kTileStep];
  __shared__ TileSlots<TM> slots;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lq = lane >> 4;
  int row_tile, col_tile;
  if (!grid.place(blockIdx.x, &row_tile, &col_tile)) return;
  const int t0 = row_tile * TM, count = min(TM, p.tokens - t0);
  const int panels = p.rows / kPanelRows;
  const int panel0 = col_tile * TN + wave * NP;
  // this slice's steps
  const int all_steps = p.cols / kTileStep;
  const int begin = all_steps * (int)blockIdx.y / (int)gridDim.y;
  const int steps = all_steps * ((int)blockIdx.y + 1) / (int)gridDim.y - begin;
  const size_t pbytes = kPanelRows * panel_row_bytes<FMT>(p.cols);
  const size_t pscales = (size_t)kPanelRows * (p.cols / 32);
  const uint8_t* pd[NP];
  const uint8_t* ps[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q) {  // a panel past the last reads the last again and stores nothing
    const int panel = min(panel0 + q, panels - 1);
    pd[q] = p.data + panel * pbytes + (size_t)begin * (SL * 1024);
    ps[q] = MX ? p.scales + panel * pscales + (size_t)begin * 64 : nullptr;
  }
  int planes = 1;
  if (rows.planes) {
    for (int i = lane; i < count; i += 64)
      planes = max(planes, rows.planes[rows.order ? rows.order[t0 + i] : t0 + i]);
    for (int o = 32; o > 0; o >>= 1) planes = max(planes, __shfl_xor(planes, o, 64));
    planes = __builtin_amdgcn_readfirstlane(planes);
  }
  // this lane's copies: rows 4 (wave + kTileWaves i) + lane / 16, the same chunk of each
  const int copy_row = 4 * wave + lane / 16;
  const int copy_chunk = (lane & 15) ^ x_swizzle<FMT>(copy_row);
  const uint8_t* const xt = reinterpret_cast<const uint8_t*>(p.x) +
                            (rows.order ? 0 : (size_t)t0 * p.x_stride * 2) +
                            (size_t)begin * (2 * kTileStep);
  uint32_t copy_off[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int at = min(copy_row + 4 * kTileWaves * i, count - 1);
    copy_off[i] = (uint32_t)(rows.order ? rows.order[t0 + at] : at) * (uint32_t)(p.x_stride * 2) +
                  16u * copy_chunk;
  }
  // the rows of step s, plane pl: copies `first` .. first + HALF
  auto load_rows = [&](uint4* st, int first, int s, int pl) {
    const uint8_t* from = xt + pl * rows.plane + (size_t)s * (2 * kTileStep);
#pragma unroll
    for (int i = 0; i < HALF; ++i) st[i] = ldg16(from + copy_off[first + i]);
  };
  auto store_rows = [&](const uint4* st, int first, u16* to) {
#pragma unroll
    for (int i = 0; i < HALF; ++i)
      *reinterpret_cast<uint4*>(to + (wave + kTileWaves * (first + i)) * 512 + 8 * lane) = st[i];
  };
  // fragment reads: byte offsets of MFMA j's operand in block 0 of the rows
  uint32_t fo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    fo[j] = (uint32_t)ln * 256u +
            16u * ((frag_k<FMT>(j, lq) >> 3) ^ x_swizzle<FMT>(ln));

  f32x4 acc[NP][MB];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[q][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  uint4 slab[2][NP];
  uint32_t sc[2][NP];
  const uint32_t doff = 16u * lane;
  auto fetch = [&](uint4* to, int u) {
#pragma unroll
    for (int q = 0; q < NP; ++q) to[q] = ldg16(pd[q] + (doff + (uint32_t)u * 1024u));
  };
  auto fetch_scales = [&](uint32_t* to, int s) {
    if constexpr (MX) {
#pragma unroll
      for (int q = 0; q < NP; ++q) to[q] = ldg_u8(ps[q] + ((uint32_t)lane + (uint32_t)s * 64u));
    }
  };
  // One step: rows in `from`, the next step's (s1, pl1) into `to`.  PAR: parity of the step.
  auto step = [&](auto par, const u16* from, u16* to, int s, int s1, int pl1) {
    constexpr int PAR = decltype(par)::value;
    const uint8_t* base = reinterpret_cast<const uint8_t*>(from);
    uint4 st[HALF];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int part = j % PARTS, slot = FMT == kFmtMXFP4 ? PAR : (j / PARTS) & 1;
      if (j == 0) {
        load_rows(st, 0, s1, pl1);
        if constexpr (FMT == kFmtMXFP4) fetch(slab[PAR ^ 1], s1);
        fetch_scales(sc[PAR ^ 1], s1);
      }
      if (j == 2) {
        store_rows(st, 0, to);
        load_rows(st, HALF, s1, pl1);
      }
      __builtin_amdgcn_sched_barrier(kHoldLoads);
      bf16x8 a[MB];
#pragma unroll
      for (int m = 0; m < MB; ++m)
        a[m] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(base + fo[j] + m * 4096));
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const bf16x8 w =
            tile_operand<FMT>(slab[slot][q], MX ? e8m0_to_f32(sc[PAR][q]) : 1.0f, part);
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[q][m] = mfma(w, a[m], acc[q][m]);
      }
      __builtin_amdgcn_sched_barrier(kHoldLoads);
      if constexpr (FMT != kFmtMXFP4) {
        // the slab two on takes this one's place: of this step or the next
        if (part == PARTS - 1) {
          const int k = j / PARTS + 2;
          fetch(slab[slot], k < SL ? s * SL + k : s1 * SL + k - SL);
        }
      }
    }
    store_rows(st, HALF, to);
    __syncthreads();
  };

  fetch(slab[0], 0);
  if (p.ids) find_slots(p, rows.order, t0, count, slots);
  if constexpr (FMT != kFmtMXFP4) fetch(slab[1], 1);  // (a step has two slabs at least)
  fetch_scales(sc[0], 0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 st[HALF];
    load_rows(st, h * HALF, 0, 0);
    store_rows(st, h * HALF, x0);
  }
  __syncthreads();
  // steps in order, each over its planes; the one after the last reads the last again
  int s = 0, pl = 0;
  auto advance = [&](auto par, const u16* from, u16* to) {
    int s1 = s, pl1 = pl + 1;
    if (pl1 == planes) {
      pl1 = 0;
      s1 = s + 1;
    }
    step(par, from, to, s, min(s1, steps - 1), pl1);
    s = s1;
    pl = pl1;
  };
  while (true) {
    advance(Int<0>{}, x0, x1);
    if (s == steps) break;
    advance(Int<1>{}, x1, x0);
    if (s == steps) break;
  }
  if (p.ids)
    add_adapters(p, slots, u, panel0, panels, (int)blockIdx.y, (int)gridDim.y, acc);
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int local = 16 * m + ln;
    if (16 * m >= count) break;
    const int t = p.ids ? slots.rows[local] : t0 + local;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int panel = panel0 + q;
      if (panel >= panels) break;
      if (local >= count) continue;
      const int row = panel * kPanelRows + 4 * lq;
      if (parts)
        *reinterpret_cast<f32x4*>(parts + ((size_t)blockIdx.y * p.tokens + t) * p.rows + row) = acc[q][m];
      else
        store_y<YB>(p, t, row, acc[q][m]);
    }
  }
}

// y from the slices' sums, in order; four outputs per thread.
template <bool YB>
__global__ __launch_bounds__(256) void join_kernel(ProjArgs p, const float* parts, int slices) {
  const size_t quads = (size_t)p.tokens * p.rows / 4;
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i >= quads) return;
  f32x4 v = reinterpret_cast<const f32x4*>(parts)[i];
#pragma unroll 4
  for (int z = 1; z < slices; ++z) v += reinterpret_cast<const f32x4*>(parts)[z * quads + i];
  const int t = (int)(i / (p.rows / 4));
  store_y<YB>(p, t, (int)(i - (size_t)t * (p.rows / 4)) * 4, v);
}

// ---- laying an adapter out ----
// A: 16-rank panels of the BF16 panel layout; B: units of 8 ranks, [panel of 16 rows][unit][row].
__global__ void pack_adapter_kernel(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b,
                                    int rank, int rows, int cols, uint16_t* __restrict__ pa,
                                    uint16_t* __restrict__ pb, int* flag_word) {
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  const size_t at = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  bool bad = false;
  auto take = [&](uint16_t v) {
    bad |= (v & 0x7f80u) == 0x7f80u;
    return v;
  };
  const int panels = (rank + 15) / 16, slabs = cols / 32;
  for (size_t i = at; i < (size_t)panels * 16 * cols; i += stride) {
    const size_t unit = i / 8;
    const int l = (int)(unit % 64), slab = (int)(unit / 64 % slabs), panel = (int)(unit / 64 / slabs);
    const int r = 16 * panel + (l & 15), c = 32 * slab + 8 * (l >> 4) + (int)(i % 8);
    pa[i] = r < rank ? take(a[(size_t)r * cols + c]) : 0;
  }
  const int units = (rank + 7) / 8;
  for (size_t i = at; i < (size_t)rows * units * 8; i += stride) {
    const size_t unit = i / 8;
    const int ln = (int)(unit % 16), ru = (int)(unit / 16 % units);
    const size_t row = unit / 16 / units * 16 + ln;
    const int r = 8 * ru + (int)(i % 8);
    pb[i] = r < rank ? take(b[row * rank + r]) : 0;
  }
  if (bad) atomicOr(flag_word, 1);
}
__global__ void enter_adapter_kernel(int rank, float scale, AdapterEntry* entry, int* flag_word,
                                     int* status) {
  if (*flag_word) {
    flag(status, kStepNonFinite);
    rank = 0;
  }
  *flag_word = 0;
  *entry = AdapterEntry{rank, scale};
}

template <int FMT, bool XB, bool YB>
void launch_rows(const ProjArgs& p, const FirstProduct& u, bool alone, hipStream_t s) {
  const int panels = p.rows / kPanelRows;
  if (alone) split_kernel<FMT, XB, YB, true><<<panels, 64 * kSplitWaves, 0, s>>>(p, u);
  else split_kernel<FMT, XB, YB, false><<<panels, 64 * kSplitWaves, 0, s>>>(p, u);
}

template <int FMT>
constexpr double kWeightBits = FMT == kFmtBF16 ? 16 : FMT == kFmtMXFP8 ? 8.25 : 4.25;

// How a call of many rows is cut: 16-row blocks per tile (of 256 outputs), tiles, and slices of K.
struct TileShape {
  int blocks, panels, row_tiles, col_tiles, slices;
};
constexpr long kMostSliced = 512;  // workgroups beyond which K is not cut (bounds the slices' sums)
TileShape tile_shape(int tokens, int rows, int cols, int planes) {
  // tiles of equal height, at most 128 rows, an even number of blocks
  TileShape t{};
  t.row_tiles = (tokens + 127) / 128;
  const int blocks = ((tokens + t.row_tiles - 1) / t.row_tiles + 15) / 16;
  t.blocks = blocks <= 2 ? 2 : (blocks + 1) / 2 * 2;
  t.row_tiles = (tokens + 16 * t.blocks - 1) / (16 * t.blocks);
  // Panels per wave and slices of K by the time of the CU with the most workgroups.  Measured: a step of
  // 128 x 256 x 128 takes a workgroup 2.0 us alone on its CU (192 outputs 1.62) and two 1.72 each, smaller
  // ones 0.9 at least (loads' latency); 2 us to fill and drain a workgroup; joining slices 4 us and their
  // traffic.  (1000 rows of 4096 -> 6144: 192 tiles of 256 outputs 66 us, 256 of 192 outputs 56; 4096 rows of
  // 7168 -> 7168: 349 and 371.)
  const int steps = cols / kTileStep;
  double best = 0;
  for (int np = 4; np >= 3; --np) {
    const int col_tiles = (rows / kPanelRows + kTileWaves * np - 1) / (kTileWaves * np);
    const long tiles = (long)t.row_tiles * col_tiles;
    const double step = std::max(0.9, (np == 4 ? 2.0 : 1.62) * t.blocks / 8);
    for (int slices = 1; slices <= std::min(steps, kMaxSlices); ++slices) {
      if (slices > 1 && tiles * slices > kMostSliced) break;
      const long per_cu = (tiles * slices + 255) / 256;
      const int each = (steps + slices - 1) / slices * planes;
      double us = per_cu * (each * step * (per_cu > 1 ? 0.86 : 1.0) + 2.0);
      if (slices > 1) us += 4.0 + (double)slices * tokens * rows * 8 / 3.5e6;
      if (t.slices == 0 || us < best) {
        best = us;
        t.panels = kTileWaves * np;
        t.col_tiles = col_tiles;
        t.slices = slices;
      }
    }
  }
  return t;
}

template <int FMT, bool YB>
void launch_tiles(const ProjArgs& p, const TileRows& rows, const FirstProduct& u, const TileShape& t,
                  float* parts, hipStream_t s) {
  TileGrid grid{};
  grid.cols = t.col_tiles;
  grid.rows = t.row_tiles;
  // the cut that leaves an XCD the fewest tiles, then the fewest bytes to read
  const double row_bytes = 16.0 * t.blocks * 2, col_bytes = 16.0 * t.panels * kWeightBits<FMT> / 8;
  long best = -1;
  double bytes = 0;
  for (int r = 1; r <= 8; r *= 2) {
    TileGrid g = grid;
    g.by_rows = r;
    g.by_cols = 8 / r;
    const long tiles = (long)g.tall() * g.wide();
    const double read = g.tall() * row_bytes + g.wide() * col_bytes;
    if (best < 0 || tiles < best || (tiles == best && read < bytes)) {
      best = tiles;
      bytes = read;
      grid = g;
    }
  }
  grid.band = std::min(8, grid.tall());
  const dim3 blocks(8 * grid.tall() * grid.wide(), t.slices);
  float* const out = t.slices > 1 ? parts : nullptr;
  auto go = [&](auto mb, auto np) {
    tile_kernel<FMT, YB, decltype(mb)::value, decltype(np)::value>
        <<<blocks, 64 * kTileWaves, 0, s>>>(p, rows, u, grid, out);
  };
  auto tall = [&](auto np) {
    if (t.blocks == 2) go(Int<2>{}, np);
    else if (t.blocks == 4) go(Int<4>{}, np);
    else if (t.blocks == 6) go(Int<6>{}, np);
    else go(Int<8>{}, np);
  };
  if (t.panels == 3 * kTileWaves) tall(Int<3>{});
  else tall(Int<4>{});
  if (out) {
    const size_t quads = (size_t)p.tokens * p.rows / 4;
    join_kernel<YB><<<(unsigned)((quads + 255) / 256), 256, 0, s>>>(p, parts, t.slices);
  }
}

// What a call's launches share.
struct Pass {
  bool tiles, alone;
  TileShape shape;
  TileRows rows;
  FirstProduct u;
  float* parts;
};

template <int FMT>
void launch_types(const ProjArgs& p, const Pass& a, hipStream_t s) {
  if (a.tiles) {
    if (p.y_bf16) launch_tiles<FMT, true>(p, a.rows, a.u, a.shape, a.parts, s);
    else launch_tiles<FMT, false>(p, a.rows, a.u, a.shape, a.parts, s);
  } else if (p.x_bf16) {
    if (p.y_bf16) launch_rows<FMT, true, true>(p, a.u, a.alone, s);
    else launch_rows<FMT, true, false>(p, a.u, a.alone, s);
  } else {
    if (p.y_bf16) launch_rows<FMT, false, true>(p, a.u, a.alone, s);
    else launch_rows<FMT, false, false>(p, a.u, a.alone, s);
  }
}

// Most blocks of 16 rows of one adapter or of none.
int order_blocks(int tokens, int slots) { return tokens / 16 + std::min(tokens, slots + 1); }

// Slices of K of the first products (1: whole).  One workgroup pulls its rows and A at what a CU can, so
// long rows of f32 are cut, where the launch that adds the slices also makes the rows' planes.  Calls of 20,
// 64, 131, 400 rows to 4096 outputs, MXFP4, whole and cut, in us: of 4096 values 24.5, 34.1, 48.7, 77.2 and
// 25.4, 35.4, 49.1, 77.5; of 5120 values 27.1, 37.3, 56.9, 91.5 and 27.1, 36.4, 53.2, 88.1; of 8192 values 33.6,
// 44.9, 73.0, 125.4 and 30.7, 44.3, 63.1, 116.8.  (BF16 rows lose as much by the launch as they gain.)
int first_slices(int tokens, const ProjArgs& p) {
  if (p.x_bf16 || tokens < kTileTokens || tokens > 512) return 1;
  return p.cols >= 5120 ? std::min(8, p.cols / 1024) : 1;
}

// The workspace of a pass: the adapters' first products and their slices' sums, the order and its
// blocks, f32 rows' planes and their counts, the slices' sums.
struct WorkLayout {
  size_t u, u_parts, order, n_blocks, blocks, planes, needed, parts, total;
  WorkLayout(int tokens, const ProjArgs& p) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    const bool tiles = tokens >= kTileTokens, sorted = tokens > kFew;
    u = take(p.slots ? (size_t)tokens * 16 * rank_panels(p.max_rank) * 2 * kF32Planes : 0);
    u_parts = take(p.slots ? (size_t)first_slices(tokens, p) * tokens * 16 * rank_panels(p.max_rank) * 4 : 0);
    order = take(sorted ? (size_t)tokens * 4 : 0);
    n_blocks = take(16);
    blocks = take(sorted ? (size_t)order_blocks(tokens, p.slots) * 12 : 0);
    planes = take(!p.x_bf16 && tiles ? (size_t)tokens * p.cols * 2 * kF32Planes : 0);
    needed = take(!p.x_bf16 && tiles ? (size_t)tokens * 4 : 0);
    const int slices = tiles ? tile_shape(tokens, p.rows, p.cols, p.x_bf16 ? 1 : kF32Planes).slices : 1;
    parts = take(slices > 1 ? (size_t)slices * tokens * p.rows * 4 : 0);
    total = at;
  }
};

// Tokens per pass of a call (longer calls run in passes of this many): f32 rows are held in planes.
int pass_tokens(const ProjArgs& p) { return p.x_bf16 ? kMaxPass : 2048; }

}  // namespace

size_t proj_work_bytes(const ProjArgs& p, int max_tokens) {
  // (not monotonic in the rows: fewer may take more slices)
  size_t most = 0;
  for (int t = 1; t <= std::min(max_tokens, pass_tokens(p)); ++t)
    most = std::max(most, WorkLayout(t, p).total);
  return most;
}

void launch_project(const ProjArgs& p, hipStream_t s) {
  // (tiles address their rows by 32-bit offsets: a wider stride takes passes of few rows)
  const bool tiles = p.tokens >= kTileTokens && p.x_stride < (1u << 22);
  const int most = tiles ? pass_tokens(p) : kTileTokens - 1;
  if (p.tokens > most) {
    for (int t = 0; t < p.tokens; t += most) {
      ProjArgs q = p;
      q.tokens = std::min(most, p.tokens - t);
      q.x = static_cast<const char*>(p.x) + (size_t)t * p.x_stride * (p.x_bf16 ? 2 : 4);
      q.y = static_cast<char*>(p.y) + (size_t)t * p.y_stride * (p.y_bf16 ? 2 : 4);
      if (p.ids) q.ids = p.ids + t;
      launch_project(q, s);
    }
    return;
  }
  const WorkLayout w(p.tokens, p);
  char* const work = static_cast<char*>(p.work);
  auto ints = [&](size_t at) { return reinterpret_cast<int*>(work + at); };
  const int max_panels = rank_panels(p.max_rank);
  const FirstProduct u{reinterpret_cast<uint16_t*>(work + w.u), 16 * max_panels};
  // A token or two of low rank: every workgroup reads all of its adapters' A from L2, which must stay
  // under what a launch and its wait cost (5 us: 4096 -> 2048, BF16, rank 16, 11.9 -> 9.3 us).
  const bool alone = p.ids && p.slots && p.tokens * 16 * max_panels <= kAloneRanks &&
                     (double)p.rows / 16 * p.tokens * 32 * max_panels * p.cols <= kAloneBytes;
  Pass a{tiles, alone, {}, {}, u, reinterpret_cast<float*>(work + w.parts)};
  if (tiles) a.shape = tile_shape(p.tokens, p.rows, p.cols, p.x_bf16 ? 1 : kF32Planes);
  // the first products (of ids without any slot: one workgroup or the order, which report them)
  Order order{};
  int firsts = 0, groups = 1, per = 1;
  bool by_token = false;
  if (p.ids && p.tokens > kFew) {
    order.order = ints(w.order);
    if (p.tokens > kOwnBlocks) {
      order = Order{ints(w.order), ints(w.blocks), ints(w.n_blocks)};
      order_kernel<<<1, kOrderThreads, 0, s>>>(p, ints(w.order), ints(w.blocks), ints(w.n_blocks));
    }
    // (four panels per workgroup share the rows' loads)
    per = 4;
    groups = std::max(1, (max_panels + 3) / 4);
    firsts = order_blocks(p.tokens, p.slots) * groups;
  } else if (p.ids && !alone) {
    by_token = p.tokens < p.slots;
    groups = std::max(1, max_panels);
    firsts = std::max(1, std::min(p.tokens, p.slots)) * groups * ((p.tokens + 15) / 16);
  }
  uint16_t* const planes =
      tiles && !p.x_bf16 ? reinterpret_cast<uint16_t*>(work + w.planes) : nullptr;
  const int slices = firsts ? first_slices(p.tokens, p) : 1;
  float* const u_parts = reinterpret_cast<float*>(work + w.u_parts);
  const dim3 grid(firsts + (planes && slices == 1 ? p.tokens : 0), slices);
  if (grid.x) {
    auto go = [&](auto xb) {
      prepare_kernel<decltype(xb)::value><<<grid, 64 * kPrepareWaves, 0, s>>>(
          p, u, u_parts, order, firsts, groups, per, by_token, planes, ints(w.needed));
      if (slices > 1)
        finish_kernel<<<p.tokens, kFinishThreads, 0, s>>>(p, u, u_parts, slices, planes, ints(w.needed));
    };
    if (p.x_bf16) go(std::true_type{});
    else go(std::false_type{});
  }
  ProjArgs q = p;
  if (planes) {
    q.x = planes;
    q.x_stride = p.cols;
    a.rows = TileRows{(size_t)p.tokens * p.cols * 2, ints(w.needed), nullptr};
  }
  // (in order a tile's rows may lie anywhere: their offsets of 32 bits must reach all of them)
  if (tiles && (uint64_t)p.tokens * q.x_stride < (1ull << 31)) a.rows.order = order.order;
  if (p.format == kFmtBF16) launch_types<kFmtBF16>(q, a, s);
  else if (p.format == kFmtMXFP4) launch_types<kFmtMXFP4>(q, a, s);
  else launch_types<kFmtMXFP8>(q, a, s);
}

void launch_set_adapter(const uint16_t* a, const uint16_t* b, int rank, float scale, int rows,
                        int cols, uint16_t* slot_a, uint16_t* slot_b, AdapterEntry* entry,
                        int* flag_word, int* status, hipStream_t s) {
  if (rank > 0) {
    const size_t n = (size_t)rank_panels(rank) * 16 * cols + (size_t)rows * rank_units(rank) * 8;
    const int blocks = (int)std::min<size_t>((n + 255) / 256, 2048);
    pack_adapter_kernel<<<blocks, 256, 0, s>>>(a, b, rank, rows, cols, slot_a, slot_b, flag_word);
  }
  enter_adapter_kernel<<<1, 1, 0, s>>>(rank, scale, entry, flag_word, status);
}

}  // namespace urb
