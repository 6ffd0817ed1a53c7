// urb_step_host.cpp -- the C ABI of the decoder steps (include/urb_step.h): checks, contexts and
// the launches of each call.
#include "../../include/urb_step.h"

#include <algorithm>
#include <new>

#include "urb_step.hpp"
#include "urb_step_host.hpp"

struct urb_proj_ctx {
  urb_proj_desc desc{};
  int device = 0;
  void* weights = nullptr;   // own copy, panel layout
  void* adapters = nullptr;  // A and B of every slot
  void* work = nullptr;      // status words, table, a pass's workspace
  size_t weight_bytes = 0, adapter_bytes = 0, work_bytes = 0;
  const uint8_t* data = nullptr;
  const uint8_t* scales = nullptr;
  uint16_t* a = nullptr;
  uint16_t* b = nullptr;
  size_t a_slot = 0, b_slot = 0;
  int* status = nullptr;  // [0] latched failures, [1] an adapter being entered, [2] validation
  urb::AdapterEntry* table = nullptr;
  void* pass = nullptr;
};

struct urb_beams {
  urb_beams_desc desc{};
  int device = 0;
  void* work = nullptr;
  int* status = nullptr;
};

struct urb_sampler {
  urb_sampler_desc desc{};
  int device = 0;
  void* work = nullptr;
  int* status = nullptr;
};

namespace {

void free_proj(urb_proj_ctx* c) {
  if (c->weights) (void)hipFree(c->weights);
  if (c->adapters) (void)hipFree(c->adapters);
  if (c->work) (void)hipFree(c->work);
  delete c;
}

struct DeviceBuffer {
  void* p = nullptr;
  ~DeviceBuffer() {
    if (p) (void)hipFree(p);
  }
};

// The part of a call's arguments that the context fixes.
urb::ProjArgs proj_args(const urb_proj_desc& d) {
  urb::ProjArgs p{};
  p.format = (int)d.format;
  p.rows = (int)d.rows;
  p.cols = (int)d.cols;
  p.x_bf16 = d.x_dtype == URB_DTYPE_BF16;
  p.y_bf16 = d.y_dtype == URB_DTYPE_BF16;
  p.slots = (int)d.adapter_slots;
  p.max_rank = (int)d.max_rank;
  return p;
}

urb_status create_proj(const urb_proj_desc* d, const urb_matrix* w, urb_weight_source source,
                       urb_proj_ctx* c) {
  const size_t rows = d->rows, cols = d->cols;
  const bool mx = d->format != URB_FMT_BF16;
  const size_t data_bytes = d->format == URB_FMT_BF16    ? rows * cols * 2
                            : d->format == URB_FMT_MXFP4 ? rows * cols / 2
                                                         : rows * cols;
  const size_t scale_bytes = mx ? rows * (cols / 32) : 0;
  URB_HIP(hipGetDevice(&c->device));
  c->desc = *d;
  // ---- table, status words and what a pass holds between its launches
  const size_t slots = d->adapter_slots;
  const size_t table_at = align_up(4 * sizeof(int));
  const size_t pass_at = table_at + align_up(slots * sizeof(urb::AdapterEntry));
  c->work_bytes = pass_at + urb::proj_work_bytes(proj_args(*d), (int)d->max_tokens);
  URB_HIP(hipMalloc(&c->work, c->work_bytes));
  char* work = static_cast<char*>(c->work);
  c->status = reinterpret_cast<int*>(work);
  c->table = reinterpret_cast<urb::AdapterEntry*>(work + table_at);
  c->pass = work + pass_at;
  urb::launch_fill_i32(c->status, 0, pass_at / 4, nullptr);
  if (slots) {
    c->a_slot = (size_t)urb::rank_panels((int)d->max_rank) * 16 * cols;
    c->b_slot = rows * urb::rank_units((int)d->max_rank) * urb::kRankUnit;
    c->adapter_bytes = slots * (c->a_slot + c->b_slot) * 2;
    URB_HIP(hipMalloc(&c->adapters, c->adapter_bytes));
    c->a = static_cast<uint16_t*>(c->adapters);
    c->b = c->a + slots * c->a_slot;
  }
  // ---- the matrix
  if (source != URB_SOURCE_HOST)
    URB_HIP(hipDeviceSynchronize());  // it may come from any stream, the borrowed one too: it is validated
  if (source == URB_SOURCE_DEVICE_BORROW) {
    c->data = static_cast<const uint8_t*>(w->data);
    c->scales = mx ? w->scales : nullptr;
  } else {
    c->weight_bytes = align_up(data_bytes) + scale_bytes;
    URB_HIP(hipMalloc(&c->weights, c->weight_bytes));
    uint8_t* data = static_cast<uint8_t*>(c->weights);
    uint8_t* scales = mx ? data + align_up(data_bytes) : nullptr;
    DeviceBuffer staging;
    const uint8_t* from = static_cast<const uint8_t*>(w->data);
    const uint8_t* from_scales = w->scales;
    if (source == URB_SOURCE_HOST) {
      URB_HIP(hipMalloc(&staging.p, c->weight_bytes));
      uint8_t* st = static_cast<uint8_t*>(staging.p);
      URB_HIP(hipMemcpy(st, w->data, data_bytes, hipMemcpyHostToDevice));
      if (mx)
        URB_HIP(hipMemcpy(st + align_up(data_bytes), w->scales, scale_bytes,
                          hipMemcpyHostToDevice));
      from = st;
      from_scales = mx ? st + align_up(data_bytes) : nullptr;
    }
    urb::launch_pack(d->format, from, from_scales, (int)rows, (int)cols, data, scales, nullptr);
    URB_HIP(hipGetLastError());
    URB_HIP(hipDeviceSynchronize());
    c->data = data;
    c->scales = scales;
  }
  urb::launch_validate(d->format, c->data, data_bytes, c->scales, scale_bytes, c->status + 2,
                       nullptr);
  URB_HIP(hipGetLastError());
  URB_HIP(hipDeviceSynchronize());
  int flags = 0;
  URB_HIP(hipMemcpy(&flags, c->status + 2, sizeof(int), hipMemcpyDeviceToHost));
  if (flags & 1) return URB_ERR_NONFINITE;
  if (flags & 2) return URB_ERR_INVALID_SCALE;
  return URB_OK;
}

}  // namespace

extern "C" {

urb_status urb_proj_create(const urb_proj_desc* d, const urb_matrix* weight,
                           urb_weight_source source, urb_proj_ctx** out) {
  if (!d || !weight || !out) return URB_ERR_ARGUMENT;
  *out = nullptr;
  if (d->format != URB_FMT_BF16 && d->format != URB_FMT_MXFP4 && d->format != URB_FMT_MXFP8)
    return URB_ERR_ARGUMENT;
  if (!row_type(d->x_dtype) || !row_type(d->y_dtype)) return URB_ERR_ARGUMENT;
  if (source != URB_SOURCE_HOST && source != URB_SOURCE_DEVICE_COPY &&
      source != URB_SOURCE_DEVICE_BORROW)
    return URB_ERR_ARGUMENT;
  if (!weight->data || (d->format != URB_FMT_BF16 && !weight->scales)) return URB_ERR_ARGUMENT;
  if (!urb::panel_shape_ok(d->rows, d->cols) || d->rows > (1u << 20) || d->cols > 32768)
    return URB_ERR_SHAPE;
  if (d->max_tokens == 0 || d->max_tokens > (1u << 30) || d->adapter_slots > 4096 ||
      d->max_rank > 256 || (d->adapter_slots == 0) != (d->max_rank == 0))
    return URB_ERR_SHAPE;
  urb_proj_ctx* c = new (std::nothrow) urb_proj_ctx();
  if (!c) return URB_ERR_OUT_OF_MEMORY;
  const urb_status st = create_proj(d, weight, source, c);
  if (st) {
    (void)hipDeviceSynchronize();
    (void)hipGetLastError();
    free_proj(c);
    return st;
  }
  *out = c;
  return URB_OK;
}

void urb_proj_destroy(urb_proj_ctx* c) {
  if (!c) return;
  int now = 0;
  const bool other = hipGetDevice(&now) == hipSuccess && now != c->device;
  const int device = c->device;
  if (other) (void)hipSetDevice(device);
  (void)hipDeviceSynchronize();
  free_proj(c);
  if (other) (void)hipSetDevice(now);
}

urb_status urb_proj_set_adapter(urb_proj_ctx* c, uint32_t slot, const urb_adapter* adapter,
                                urb_weight_source source, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  if (slot >= c->desc.adapter_slots) return URB_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint16_t* slot_a = c->a + slot * c->a_slot;
  uint16_t* slot_b = c->b + slot * c->b_slot;
  const int rows = (int)c->desc.rows, cols = (int)c->desc.cols;
  if (!adapter) {
    urb::launch_set_adapter(nullptr, nullptr, 0, 0.0f, rows, cols, slot_a, slot_b,
                            c->table + slot, c->status + 1, c->status, s);
    URB_HIP(hipGetLastError());
    return URB_OK;
  }
  if (!adapter->a || !adapter->b) return URB_ERR_ARGUMENT;
  if (source != URB_SOURCE_HOST && source != URB_SOURCE_DEVICE_COPY) return URB_ERR_ARGUMENT;
  if (adapter->rank == 0 || adapter->rank > c->desc.max_rank) return URB_ERR_SHAPE;
  if (!finite_host(adapter->scale)) return URB_ERR_NONFINITE;
  const uint16_t* a = adapter->a;
  const uint16_t* b = adapter->b;
  const size_t a_bytes = (size_t)adapter->rank * cols * 2, b_bytes = (size_t)adapter->rank * rows * 2;
  DeviceBuffer staging;
  if (source == URB_SOURCE_HOST) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    URB_HIP(hipStreamIsCapturing(s, &cs));
    if (cs != hipStreamCaptureStatusNone) return URB_ERR_ARGUMENT;
    URB_HIP(hipMalloc(&staging.p, align_up(a_bytes) + b_bytes));
    char* st = static_cast<char*>(staging.p);
    URB_HIP(hipMemcpy(st, a, a_bytes, hipMemcpyHostToDevice));
    URB_HIP(hipMemcpy(st + align_up(a_bytes), b, b_bytes, hipMemcpyHostToDevice));
    a = reinterpret_cast<const uint16_t*>(st);
    b = reinterpret_cast<const uint16_t*>(st + align_up(a_bytes));
  }
  urb::launch_set_adapter(a, b, (int)adapter->rank, adapter->scale, rows, cols, slot_a, slot_b,
                          c->table + slot, c->status + 1, c->status, s);
  URB_HIP(hipGetLastError());
  if (staging.p) URB_HIP(hipStreamSynchronize(s));
  return URB_OK;
}

urb_status urb_proj_forward(urb_proj_ctx* c, const void* x, uint64_t x_stride,
                            const int32_t* adapter_ids, uint32_t tokens, void* y,
                            uint64_t y_stride, void* stream) {
  if (!c || !x || !y || !on_device(c->device)) return URB_ERR_ARGUMENT;
  const urb_proj_desc& d = c->desc;
  if (tokens == 0 || tokens > d.max_tokens || x_stride < d.cols || y_stride < d.rows)
    return URB_ERR_SHAPE;
  const size_t xb = value_bytes(d.x_dtype), yb = value_bytes(d.y_dtype);
  if (reinterpret_cast<uintptr_t>(x) % 16 || x_stride * xb % 16 ||
      reinterpret_cast<uintptr_t>(y) % yb)
    return URB_ERR_ARGUMENT;
  urb::ProjArgs p = proj_args(d);
  p.data = c->data;
  p.scales = c->scales;
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.table = c->table;
  p.a = c->a;
  p.b = c->b;
  p.a_slot = c->a_slot;
  p.b_slot = c->b_slot;
  p.work = c->pass;
  p.status = c->status;
  p.tokens = (int)tokens;
  p.x = x;
  p.y = y;
  p.ids = adapter_ids;
  urb::launch_project(p, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_proj_sync(urb_proj_ctx* c, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  int bits = 0;
  const urb_status st = take_status(c->status, static_cast<hipStream_t>(stream), &bits);
  if (st) return st;
  if (bits & urb::kStepNonFinite) return URB_ERR_NONFINITE;
  return bits & urb::kStepArgument ? URB_ERR_ARGUMENT : URB_OK;
}

urb_status urb_proj_memory(const urb_proj_ctx* c, size_t* weight_bytes, size_t* adapter_bytes,
                           size_t* workspace_bytes) {
  if (!c) return URB_ERR_ARGUMENT;
  if (weight_bytes) *weight_bytes = c->weight_bytes;
  if (adapter_bytes) *adapter_bytes = c->adapter_bytes;
  if (workspace_bytes) *workspace_bytes = c->work_bytes;
  return URB_OK;
}

urb_status urb_qk_norm_rope(const urb_qk_desc* d, const void* q, const void* k,
                            const float* q_weight, const float* k_weight,
                            const int64_t* positions, const float* inv_freq, uint32_t tokens,
                            void* q_out, void* k_out, void* stream) {
  if (!d || !q || !q_weight || !q_out) return URB_ERR_ARGUMENT;
  if (d->k_heads && (!k || !k_weight || !k_out)) return URB_ERR_ARGUMENT;
  if (d->rotary_dim && (!positions || !inv_freq)) return URB_ERR_ARGUMENT;
  if (!row_type(d->dtype)) return URB_ERR_ARGUMENT;
  const uint64_t heads = (uint64_t)d->q_heads + d->k_heads;
  if (tokens == 0 || d->q_heads == 0 || heads > 65535 || heads * tokens > 0x7fffffffu)
    return URB_ERR_SHAPE;
  if (d->head_dim < 2 || d->head_dim > 1024 || d->head_dim % 2 || d->rotary_dim % 2 ||
      d->rotary_dim > d->head_dim)
    return URB_ERR_SHAPE;
  if (!finite_host(d->eps) || !(d->eps > 0.0f)) return URB_ERR_INVALID_GEOMETRY;
  const size_t vb = value_bytes(d->dtype);
  auto aligned = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % vb == 0; };
  if (!aligned(q) || !aligned(q_out) || (d->k_heads && (!aligned(k) || !aligned(k_out))))
    return URB_ERR_ARGUMENT;
  if (!heads_apart(tokens, d->q_out_token_stride, d->q_heads, d->q_out_head_stride, d->head_dim) ||
      (d->k_heads &&
       !heads_apart(tokens, d->k_out_token_stride, d->k_heads, d->k_out_head_stride, d->head_dim)))
    return URB_ERR_SHAPE;
  urb::RotateArgs a{};
  a.q = urb::HeadRows{q, q_out, q_weight, d->q_token_stride, d->q_head_stride,
                      d->q_out_token_stride, d->q_out_head_stride};
  if (d->k_heads)
    a.k = urb::HeadRows{k, k_out, k_weight, d->k_token_stride, d->k_head_stride,
                        d->k_out_token_stride, d->k_out_head_stride};
  a.q_heads = (int)d->q_heads;
  a.heads = (int)heads;
  a.dim = (int)d->head_dim;
  a.rotary = (int)d->rotary_dim;
  a.interleaved = d->interleaved != 0;
  a.offset = d->zero_centered ? 1.0f : 0.0f;
  a.eps = d->eps;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.tokens = tokens;
  urb::launch_rotate(a, d->dtype == URB_DTYPE_BF16, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_sampler_create(const urb_sampler_desc* d, urb_sampler** out) {
  if (!d || !out) return URB_ERR_ARGUMENT;
  *out = nullptr;
  if (!row_type(d->dtype)) return URB_ERR_ARGUMENT;
  if (d->vocab == 0 || d->vocab > (1u << 20) || d->max_rows == 0 || d->max_rows > (1u << 24))
    return URB_ERR_SHAPE;
  urb_sampler* c = new (std::nothrow) urb_sampler();
  if (!c) return URB_ERR_OUT_OF_MEMORY;
  c->desc = *d;
  const urb_status st = [&]() -> urb_status {
    URB_HIP(hipGetDevice(&c->device));
    URB_HIP(hipMalloc(&c->work, kAlign + urb::sample_work_bytes((int)d->vocab, (int)d->max_rows)));
    c->status = static_cast<int*>(c->work);
    urb::launch_fill_i32(c->status, 0, kAlign / 4, nullptr);
    URB_HIP(hipGetLastError());
    URB_HIP(hipDeviceSynchronize());
    return URB_OK;
  }();
  if (st) {
    (void)hipGetLastError();
    if (c->work) (void)hipFree(c->work);
    delete c;
    return st;
  }
  *out = c;
  return URB_OK;
}

void urb_sampler_destroy(urb_sampler* c) {
  if (!c) return;
  int now = 0;
  const bool other = hipGetDevice(&now) == hipSuccess && now != c->device;
  if (other) (void)hipSetDevice(c->device);
  (void)hipDeviceSynchronize();
  if (c->work) (void)hipFree(c->work);
  delete c;
  if (other) (void)hipSetDevice(now);
}

urb_status urb_sample(urb_sampler* c, const void* logits, uint64_t row_stride, uint32_t rows,
                      const urb_sample_params* params, const float* uniform, int32_t* ids,
                      float* probs, void* stream) {
  if (!c || !logits || !uniform || !ids || !on_device(c->device)) return URB_ERR_ARGUMENT;
  const urb_sampler_desc& d = c->desc;
  if (rows == 0 || rows > d.max_rows || row_stride < d.vocab) return URB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(logits) % value_bytes(d.dtype)) return URB_ERR_ARGUMENT;
  const urb_sample_params none{};
  if (!params) params = &none;
  urb::SampleArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = (int)d.vocab;
  a.rows = (int)rows;
  a.temperature = params->temperature;
  a.top_k = params->top_k;
  a.top_p = params->top_p;
  a.min_p = params->min_p;
  a.uniform = uniform;
  a.ids = ids;
  a.probs = probs;
  a.status = c->status;
  a.work = static_cast<char*>(c->work) + kAlign;
  urb::launch_sample(a, d.dtype == URB_DTYPE_BF16, static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_sampler_sync(urb_sampler* c, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  int bits = 0;
  const urb_status st = take_status(c->status, static_cast<hipStream_t>(stream), &bits);
  if (st) return st;
  return bits ? URB_ERR_ARGUMENT : URB_OK;
}

urb_status urb_beams_create(const urb_beams_desc* d, urb_beams** out) {
  if (!d || !out) return URB_ERR_ARGUMENT;
  *out = nullptr;
  if (!row_type(d->dtype)) return URB_ERR_ARGUMENT;
  if (d->vocab == 0 || d->vocab > (uint32_t)urb::kBeamVocab || d->width == 0 ||
      d->width > (uint32_t)urb::kBeamWidth || d->picks == 0 || d->picks > (uint32_t)urb::kBeamPicks ||
      d->max_requests == 0 || d->max_requests > 65535)
    return URB_ERR_SHAPE;
  urb_beams* c = new (std::nothrow) urb_beams();
  if (!c) return URB_ERR_OUT_OF_MEMORY;
  c->desc = *d;
  const urb_status st = [&]() -> urb_status {
    URB_HIP(hipGetDevice(&c->device));
    URB_HIP(hipMalloc(&c->work, kAlign + urb::beam_work_bytes((int)d->vocab, (int)d->width, (int)d->picks,
                                                              (int)d->max_requests)));
    c->status = static_cast<int*>(c->work);
    urb::launch_fill_i32(c->status, 0, kAlign / 4, nullptr);
    URB_HIP(hipGetLastError());
    URB_HIP(hipDeviceSynchronize());
    return URB_OK;
  }();
  if (st) {
    (void)hipGetLastError();
    if (c->work) (void)hipFree(c->work);
    delete c;
    return st;
  }
  *out = c;
  return URB_OK;
}

void urb_beams_destroy(urb_beams* c) {
  if (!c) return;
  int now = 0;
  const bool other = hipGetDevice(&now) == hipSuccess && now != c->device;
  if (other) (void)hipSetDevice(c->device);
  (void)hipDeviceSynchronize();
  if (c->work) (void)hipFree(c->work);
  delete c;
  if (other) (void)hipSetDevice(now);
}

urb_status urb_beams_select(urb_beams* c, const urb_beams_call* p, void* stream) {
  if (!c || !p || !p->logits || !p->scores || !p->scores_out || !p->tokens || !p->parents ||
      !on_device(c->device))
    return URB_ERR_ARGUMENT;
  const urb_beams_desc& d = c->desc;
  if (p->requests == 0 || p->requests > d.max_requests || p->row_stride < d.vocab) return URB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(p->logits) % value_bytes(d.dtype)) return URB_ERR_ARGUMENT;
  if (p->end_token < (p->ended ? 0 : -1) || p->end_token >= (int64_t)d.vocab) return URB_ERR_ARGUMENT;
  if (d.picks != d.width && (p->scores_out == p->scores || (p->ended && p->ended_out == p->ended)))
    return URB_ERR_ARGUMENT;
  urb::BeamArgs a{};
  a.logits = p->logits;
  a.row_stride = p->row_stride;
  a.vocab = (int)d.vocab;
  a.width = (int)d.width;
  a.picks = (int)d.picks;
  a.requests = (int)p->requests;
  a.end_token = p->end_token;
  a.scores = p->scores;
  a.ended = p->ended;
  a.scores_out = p->scores_out;
  a.tokens = p->tokens;
  a.parents = p->parents;
  a.ended_out = p->ended_out;
  a.status = c->status;
  urb::launch_beam(a, d.dtype == URB_DTYPE_BF16, static_cast<char*>(c->work) + kAlign,
                   static_cast<hipStream_t>(stream));
  URB_HIP(hipGetLastError());
  return URB_OK;
}

urb_status urb_beams_sync(urb_beams* c, void* stream) {
  if (!c || !on_device(c->device)) return URB_ERR_ARGUMENT;
  int bits = 0;
  const urb_status st = take_status(c->status, static_cast<hipStream_t>(stream), &bits);
  if (st) return st;
  return bits ? URB_ERR_ARGUMENT : URB_OK;
}

}  // extern "C"
