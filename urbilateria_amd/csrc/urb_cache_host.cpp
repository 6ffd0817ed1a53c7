// urb_cache_host.cpp -- the C ABI of the paged cache (include/urb_cache.h): checks, contexts and the launches
// of each call.
#include "../../include/urb_cache.h"

#include <algorithm>
#include <new>

#include "urb_cache.hpp"
#include "urb_step_host.hpp"

struct urb_pager {
  urb_pager_desc desc{};
  int device = 0;
  void* work = nullptr;
  int* status = nullptr;
  urb::PlanRow* row_plans = nullptr;  // [max_rows + 1]
  // forks: [max_rows], [kForkRequests] twice, [1], [max_rows * max_blocks]
  int32_t *old_lengths = nullptr, *drops = nullptr, *copies = nullptr, *count = nullptr, *dropped = nullptr;
  urb::ForkCopy* page_copies = nullptr;  // [max_rows]
};

struct urb_attention {
  urb_attention_desc desc{};
  int device = 0;
  void* work = nullptr;
  int* status = nullptr;
  float* parts = nullptr;
};

namespace {

bool cache_type(urb_dtype t) { return t == URB_DTYPE_BF16 || t == URB_DTYPE_F8_E4M3; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Axis {
  uint64_t n, stride;
  // in bytes; the stride of an axis of one is not used
  uint64_t bytes(uint64_t b) const { return n > 1 ? stride * b : 0; }
};
// The values from the first to behind the last of rows of dim values along three axes; 0 if a stride is less than
// what the axes of smaller ones span, as it is where rows overlap, or if it is 2^40 or more.
uint64_t span_of(Axis a, Axis b, Axis c, uint64_t dim) {
  Axis axes[3] = {a, b, c};
  std::sort(axes, axes + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
  unsigned __int128 span = dim;
  for (const Axis& x : axes) {
    if (x.n <= 1) continue;
    if (x.stride < span) return 0;
    span += (unsigned __int128)(x.n - 1) * x.stride;
    if (span >> 40) return 0;
  }
  return (uint64_t)span;
}

// Whether two tables' rows of n entries, each one's rows apart, have an entry in common.
bool tables_meet(const int32_t* a, uint64_t a_stride, const int32_t* b, uint64_t b_stride, uint64_t rows,
                 uint64_t n) {
  typedef unsigned __int128 Wide;  // (strides may be anything)
  const Wide size = (Wide)n * sizeof(int32_t);
  auto at = [](const int32_t* p, uint64_t stride, uint64_t row) {
    return (Wide) reinterpret_cast<uintptr_t>(p) + (Wide)row * stride * sizeof(int32_t);
  };
  // the rows of both in their order (one table behind the other: no step)
  if (at(a, a_stride, rows - 1) + size <= at(b, b_stride, 0) || at(b, b_stride, rows - 1) + size <= at(a, a_stride, 0))
    return false;
  for (uint64_t i = 0, j = 0; i < rows && j < rows;) {
    const Wide x = at(a, a_stride, i), y = at(b, b_stride, j);
    if (x + size <= y) ++i;
    else if (y + size <= x) ++j;
    else return true;
  }
  return false;
}

bool geometry(uint32_t heads, uint32_t page_size, uint32_t head_dim) {
  return heads >= 1 && heads <= 1024 && page_size >= 1 && page_size <= 1024 && head_dim >= 16 &&
         head_dim <= 256 && head_dim % 16 == 0;
}

// Checks a cache's description and fills in what the kernels take.
urb_status take_cache(const urb_kv_cache* c, urb::KvCache* out) {
  if (!c || !c->k || !c->v || !cache_type(c->dtype)) return URB_ERR_ARGUMENT;
  const bool f8 = c->dtype == URB_DTYPE_F8_E4M3;
  if (f8 ? !c->k_scales || !c->v_scales : c->k_scales || c->v_scales) return URB_ERR_ARGUMENT;
  if (!geometry(c->heads, c->page_size, c->head_dim) || c->pages == 0 || c->pages > (1u << 24))
    return URB_ERR_SHAPE;
  const uint64_t b = f8 ? 1 : 2;
  const Axis pages{c->pages, c->page_stride}, heads{c->heads, c->head_stride},
      tokens{c->page_size, c->token_stride};
  const uint64_t span = span_of(pages, heads, tokens, c->head_dim);
  if (span == 0 || span * b >= (1ull << 36)) return URB_ERR_SHAPE;
  *out = urb::KvCache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scales, c->v_scales,
                      c->pages, c->heads, c->page_size, c->head_dim,
                      pages.bytes(b), heads.bytes(b), tokens.bytes(b)};
  return aligned16(c->k) && aligned16(c->v) && (out->page_stride | out->head_stride | out->token_stride) % 16 == 0
             ? URB_OK
             : URB_ERR_ARGUMENT;
}

template <class T>
T* carve(char*& p, size_t n) {
  T* at = reinterpret_cast<T*>(p);
  p += align_up(n * sizeof(T));
  return at;
}

// Allocates a context's workspace and clears its status word, which lies at its start.
urb_status make_work(size_t bytes, void** work, int* device, int** status) {
  URB_HIP(hipGetDevice(device));
  URB_HIP(hipMalloc(work, kAlign + bytes));
  *status = static_cast<int*>(*work);
  urb::launch_fill_i32(*status, 0, kAlign / 4, nullptr);
  URB_HIP(hipGetLastError());
  URB_HIP(hipDeviceSynchronize());
  return URB_OK;
}

template <class C>
void drop(C* c) {
  int now = 0;
  const bool other = hipGetDevice(&now) == hipSuccess && now != c->device;
  if (other) (void)hipSetDevice(c->device);
  (void)hipDeviceSynchronize();
  if (c->work) (void)hipFree(c->work);
  delete c;
  if (other) (void)hipSetDevice(now);
}

}  // namespace

extern "C" {

urb_status urb_kv_append(const urb_kv_cache* cache, const urb_kv_rows* rows, const int64_t* slots,
                         uint32_t tokens, void* stream) {
  urb::AppendArgs a{};
  if (const urb_status st = take_cache(cache, &a.cache)) return st;
  if (!rows || !rows->k || !rows->v || !slots || !row_type(rows->dtype)) return URB_ERR_ARGUMENT;
  if (tokens == 0 || tokens >= (1u << 24)) return URB_ERR_SHAPE;
  const uint64_t b = value_bytes(rows->dtype);
  a.k = static_cast<const uint8_t*>(rows->k);
  a.v = static_cast<const uint8_t*>(rows->v);
  a.k_token = Axis{tokens, rows->k_token_stride}.bytes(b);
  a.k_head = Axis{cache->heads, rows->k_head_stride}.bytes(b);
  a.v_token = Axis{tokens, rows->v_token_stride}.bytes(b);
  a.v_head = Axis{cache->heads, rows->v_head_stride}.bytes(b);
  if (!aligned16(a.k) || !aligned16(a.v) || (a.k_token | a.k_head | a.v_token | a.v_head) % 16)
    return URB_ERR_ARGUMENT;
  a.slots = slots;
  a.tokens = tokens;
  urb::launch_append(a, rows->dtype == URB_DTYPE_BF16, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_pager_create(const urb_pager_desc* d, urb_pager** out) {
  if (!d || !out) return URB_ERR_ARGUMENT;
  *out = nullptr;
  if (d->pages == 0 || d->pages > (1u << 24) || d->page_size == 0 || d->page_size > 1024 ||
      d->max_rows == 0 || d->max_rows > (1u << 20) || d->max_blocks == 0 || d->max_blocks > (1u << 20) ||
      d->max_tokens >= (1u << 30) || (uint64_t)d->max_rows * d->max_blocks >= (1ull << 31) ||
      (uint64_t)d->max_blocks * d->page_size >= (1ull << 30))
    return URB_ERR_SHAPE;
  urb_pager* c = new (std::nothrow) urb_pager();
  if (!c) return URB_ERR_OUT_OF_MEMORY;
  c->desc = *d;
  const size_t rows = d->max_rows, table = rows * d->max_blocks;
  const size_t requests = std::min<size_t>(urb::kForkRequests, rows);
  char* p = nullptr;  // (offsets first, addresses when the memory is there)
  auto lay = [&]() {
    c->row_plans = carve<urb::PlanRow>(p, rows + 1);
    c->old_lengths = carve<int32_t>(p, rows);
    c->drops = carve<int32_t>(p, requests);
    c->copies = carve<int32_t>(p, requests);
    c->count = carve<int32_t>(p, 1);
    c->dropped = carve<int32_t>(p, table);
    c->page_copies = carve<urb::ForkCopy>(p, rows);
  };
  lay();
  if (const urb_status st = make_work(reinterpret_cast<size_t>(p), &c->work, &c->device, &c->status)) {
    (void)hipGetLastError();
    if (c->work) (void)hipFree(c->work);
    delete c;
    return st;
  }
  p = static_cast<char*>(c->work) + kAlign;
  lay();
  *out = c;
  return URB_OK;
}

void urb_pager_destroy(urb_pager* c) {
  if (c) drop(c);
}

urb_status urb_pager_plan(urb_pager* c, const urb_page_plan* p, void* stream) {
  if (!c || !p || !on_device(c->device) || !p->lengths || !p->tables || !p->free_pages ||
      !p->free_count || !p->lengths_out || !p->slots || !p->free_count_out)
    return URB_ERR_ARGUMENT;
  const urb_pager_desc& d = c->desc;
  if (p->rows == 0 || p->rows > d.max_rows || p->tokens == 0 || p->tokens > d.max_tokens ||
      p->table_stride < d.max_blocks)
    return URB_ERR_SHAPE;
  urb::PlanArgs a{};
  a.rows = p->rows;
  a.tokens = p->tokens;
  a.page = urb::PageDivision::by(d.page_size);
  a.pages = d.pages;
  a.max_blocks = d.max_blocks;
  a.table_stride = p->table_stride;
  a.lengths = p->lengths;
  a.added = p->added;
  a.tables = p->tables;
  a.free_pages = p->free_pages;
  a.free_count = p->free_count;
  a.lengths_out = p->lengths_out;
  a.starts = p->starts;
  a.token_rows = p->token_rows;
  a.positions = p->positions;
  a.slots = p->slots;
  a.free_count_out = p->free_count_out;
  a.row_plans = c->row_plans;
  a.status = c->status;
  urb::launch_plan(a, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_pager_fork(urb_pager* c, const urb_page_fork* f, void* stream) {
  if (!c || !f || !on_device(c->device) || !f->parents || !f->tables || !f->lengths || !f->tables_out ||
      !f->lengths_out || !f->free_pages || !f->free_count || !f->free_count_out ||
      f->tables == f->tables_out || (f->n_caches && !f->caches))
    return URB_ERR_ARGUMENT;
  const urb_pager_desc& d = c->desc;
  if (f->requests == 0 || f->requests > urb::kForkRequests || f->width == 0 || f->width > urb::kForkWidth ||
      (uint64_t)f->requests * f->width > d.max_rows || f->table_stride < d.max_blocks ||
      f->table_out_stride < d.max_blocks || f->n_caches > 4096)
    return URB_ERR_SHAPE;
  if (tables_meet(f->tables, f->table_stride, f->tables_out, f->table_out_stride, (uint64_t)f->requests * f->width,
                  d.max_blocks))
    return URB_ERR_ARGUMENT;
  // (all caches are checked before the first launch)
  for (uint32_t i = 0; i < f->n_caches; ++i) {
    urb::KvCache c;
    if (const urb_status st = take_cache(f->caches + i, &c)) return st;
    if (c.pages != d.pages || c.page != d.page_size) return URB_ERR_SHAPE;
  }
  urb::ForkArgs a{};
  a.requests = f->requests;
  a.width = f->width;
  a.page = urb::PageDivision::by(d.page_size);
  a.pages = d.pages;
  a.max_blocks = d.max_blocks;
  a.table_stride = f->table_stride;
  a.table_out_stride = f->table_out_stride;
  a.parents = f->parents;
  a.tables = f->tables;
  a.lengths = f->lengths;
  a.tables_out = f->tables_out;
  a.lengths_out = f->lengths_out;
  a.free_pages = f->free_pages;
  a.free_count = f->free_count;
  a.free_count_out = f->free_count_out;
  a.old_lengths = c->old_lengths;
  a.drops = c->drops;
  a.copies = c->copies;
  a.dropped = c->dropped;
  a.page_copies = c->page_copies;
  a.count = c->count;
  a.status = c->status;
  urb::launch_fork(a, static_cast<hipStream_t>(stream));
  for (uint32_t done = 0; done < f->n_caches;) {
    urb::ForkCaches some;
    const uint32_t n = std::min<uint32_t>(urb::kForkCaches, f->n_caches - done);
    for (uint32_t i = 0; i < n; ++i) (void)take_cache(f->caches + done + i, &some.c[i]);
    urb::launch_fork_copies(a, some, n, static_cast<hipStream_t>(stream));
    done += n;
  }
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_pager_sync(urb_pager* c, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  int bits = 0;
  const urb_status st = take_status(c->status, static_cast<hipStream_t>(stream), &bits);
  if (st) return st;
  if (bits & urb::kCacheArgument) return URB_ERR_ARGUMENT;
  return bits & urb::kCacheMemory ? URB_ERR_OUT_OF_MEMORY : URB_OK;
}

urb_status urb_attention_create(const urb_attention_desc* d, urb_attention** out) {
  if (!d || !out) return URB_ERR_ARGUMENT;
  *out = nullptr;
  if (!row_type(d->dtype) || !cache_type(d->cache_dtype)) return URB_ERR_ARGUMENT;
  if (!geometry(d->heads, d->page_size, d->head_dim) || d->q_heads == 0 || d->q_heads > 8192 ||
      d->q_heads % d->heads || d->queries == 0 || d->queries > 16 || d->max_rows == 0 ||
      d->max_rows > (1u << 20) || d->max_length == 0 || d->max_length > (1u << 24))
    return URB_ERR_SHAPE;
  // (times log2(e) it is finite)
  if (!(d->scale > 0.0f) || d->scale > 0x1p127f) return URB_ERR_INVALID_GEOMETRY;
  urb_attention* c = new (std::nothrow) urb_attention();
  if (!c) return URB_ERR_OUT_OF_MEMORY;
  c->desc = *d;
  if (const urb_status st =
          make_work(urb::attend_work_bytes(d->head_dim, d->cache_dtype == URB_DTYPE_F8_E4M3,
                                           d->dtype == URB_DTYPE_BF16),
                    &c->work, &c->device, &c->status)) {
    (void)hipGetLastError();
    if (c->work) (void)hipFree(c->work);
    delete c;
    return st;
  }
  c->parts = reinterpret_cast<float*>(static_cast<char*>(c->work) + kAlign);
  *out = c;
  return URB_OK;
}

void urb_attention_destroy(urb_attention* c) {
  if (c) drop(c);
}

urb_status urb_attend(urb_attention* c, const urb_kv_cache* cache, const urb_attention_call* p,
                      void* stream) {
  if (!c || !p || !on_device(c->device)) return URB_ERR_ARGUMENT;
  urb::AttendArgs a{};
  if (const urb_status st = take_cache(cache, &a.cache)) return st;
  if (!p->q || !p->out || !p->tables || !p->lengths) return URB_ERR_ARGUMENT;
  const urb_attention_desc& d = c->desc;
  if (cache->heads != d.heads || cache->head_dim != d.head_dim || cache->page_size != d.page_size ||
      cache->dtype != d.cache_dtype)
    return URB_ERR_SHAPE;
  if (p->rows == 0 || p->rows > d.max_rows ||
      p->table_stride < ((uint64_t)d.max_length + d.page_size - 1) / d.page_size)
    return URB_ERR_SHAPE;
  const uint64_t b = value_bytes(d.dtype);
  const Axis rows{p->rows, p->out_row_stride}, tokens{d.queries, p->out_token_stride},
      heads{d.q_heads, p->out_head_stride};
  if (span_of(rows, tokens, heads, d.head_dim) == 0) return URB_ERR_SHAPE;
  a.rows = p->rows;
  a.queries = d.queries;
  a.q_heads = d.q_heads;
  a.window = d.window;
  a.max_length = d.max_length;
  a.scale = d.scale;
  a.q = static_cast<const uint8_t*>(p->q);
  a.out = static_cast<uint8_t*>(p->out);
  a.q_row = Axis{p->rows, p->q_row_stride}.bytes(b);
  a.q_token = Axis{d.queries, p->q_token_stride}.bytes(b);
  a.q_head = Axis{d.q_heads, p->q_head_stride}.bytes(b);
  a.out_row = rows.bytes(b);
  a.out_token = tokens.bytes(b);
  a.out_head = heads.bytes(b);
  if (!aligned16(a.q) || !aligned16(a.out) ||
      (a.q_row | a.q_token | a.q_head | a.out_row | a.out_token | a.out_head) % 16)
    return URB_ERR_ARGUMENT;
  a.tables = p->tables;
  a.table_stride = p->table_stride;
  a.lengths = p->lengths;
  a.sinks = p->sinks;
  a.lse = p->lse;
  a.parts = c->parts;
  a.status = c->status;
  urb::launch_attend(a, d.dtype == URB_DTYPE_BF16, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_attention_sync(urb_attention* c, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  int bits = 0;
  const urb_status st = take_status(c->status, static_cast<hipStream_t>(stream), &bits);
  if (st) return st;
  return bits ? URB_ERR_ARGUMENT : URB_OK;
}

}  // extern "C"
