// C entry points of the operators on rows of class logits (logits.h): the
// argument checks, the context's device and the launch.  Nothing here
// allocates, waits or keeps state, so calls may run at once and be captured.
#include <algorithm>
#include <cmath>

#include "logits.h"
#include "runtime.h"

namespace ppocr {
namespace {

// Grids take a row per workgroup of up to 1024 threads, with fewer than 2^32
// threads in all.
constexpr size_t kMaxLogitRows = (size_t)1 << 21;

// Makes a context's device current for a call and restores the caller's.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    HIP_OK(hipGetDevice(&before_));
    if (before_ == device) return;
    HIP_OK(hipSetDevice(device));
    changed_ = true;
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

// Rejects memory that kernels of `device` may not touch: null, host memory,
// another device's.
void check_device(const void* ptr, int device, const char* what) {
  hipPointerAttribute_t a{};
  if (hipPointerGetAttributes(&a, ptr) != hipSuccess) {
    (void)hipGetLastError();
    raise(PPOCR_ERR_INVALID_INPUT, std::string(what) + " is not device memory");
  }
  if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged)
    raise(PPOCR_ERR_INVALID_INPUT, std::string(what) + " is not device memory");
  if (a.type == hipMemoryTypeDevice && a.device != device)
    raise(PPOCR_ERR_INVALID_INPUT, std::string(what) + " is on device " + std::to_string(a.device) +
                                       ", the context on device " + std::to_string(device));
}
void check_optional(const void* ptr, int device, const char* what) {
  if (ptr) check_device(ptr, device, what);
}

void check_aligned(const void* ptr, size_t size, const char* what) {
  if (reinterpret_cast<uintptr_t>(ptr) % size)
    raise(PPOCR_ERR_INVALID_INPUT, std::string(what) + " is not aligned to its elements");
}

LogitRows rows_of(const ppocr_logits* l, const char* what) {
  const std::string name(what);
  if (!l) raise(PPOCR_ERR_INVALID_INPUT, name + " is null");
  if (l->type != PPOCR_F32 && l->type != PPOCR_BF16) raise(PPOCR_ERR_INVALID_INPUT, name + ": unknown element type");
  if (l->classes == 0 || l->classes > (size_t)kMaxLogitClasses)
    raise(PPOCR_ERR_INVALID_INPUT, name + ": " + std::to_string(l->classes) + " classes; 1 to " +
                                       std::to_string(kMaxLogitClasses) + " are supported");
  if (l->rows > kMaxLogitRows)
    raise(PPOCR_ERR_INVALID_INPUT, name + ": " + std::to_string(l->rows) + " rows; at most " +
                                       std::to_string(kMaxLogitRows) + " are supported");
  if (l->stride < l->classes || l->stride > (size_t)1 << 40)
    raise(PPOCR_ERR_INVALID_INPUT, name + ": the row stride is smaller than the row, or over 2^40");
  if (l->rows && !l->data) raise(PPOCR_ERR_INVALID_INPUT, name + ": data is null");
  LogitRows r{};
  r.x = l->data;
  r.rows = (int64_t)l->rows;
  r.classes = (int)l->classes;
  r.stride = (int64_t)l->stride;
  r.dt = l->type == PPOCR_BF16 ? DT_BF16 : DT_F32;
  check_aligned(l->data, dtype_size(r.dt), what);
  return r;
}

// Rows written by a call: in place (the same memory and stride) or apart.
void check_output(const LogitRows& in, const void* out, size_t stride, const char* what) {
  const std::string name(what);
  if (!out) raise(PPOCR_ERR_INVALID_INPUT, name + " is null");
  const size_t es = dtype_size(in.dt);
  check_aligned(out, es, what);
  if (stride < (size_t)in.classes || stride > (size_t)1 << 40)
    raise(PPOCR_ERR_INVALID_INPUT, name + ": the row stride is smaller than the row, or over 2^40");
  if (out == in.x && (stride == (size_t)in.stride || in.rows == 1)) return;
  const uintptr_t a = reinterpret_cast<uintptr_t>(in.x), b = reinterpret_cast<uintptr_t>(out);
  const uintptr_t na = ((size_t)(in.rows - 1) * in.stride + in.classes) * es;
  const uintptr_t nb = ((size_t)(in.rows - 1) * stride + in.classes) * es;
  if (a < b + nb && b < a + na) raise(PPOCR_ERR_INVALID_INPUT, name + " overlaps the logits without being in place");
}

void check_table(const void* table, size_t n, const int32_t* index, size_t rows, const char* what) {
  const std::string name(what);
  if (!table) {
    if (n || index) raise(PPOCR_ERR_INVALID_INPUT, name + ": a table's rows or index without the table");
    return;
  }
  if (n == 0 || n > (size_t)INT32_MAX) raise(PPOCR_ERR_INVALID_INPUT, name + ": the table has no rows, or over 2^31 - 1");
  if (!index && n != 1 && n != rows)
    raise(PPOCR_ERR_INVALID_INPUT, name + ": " + std::to_string(n) + " tables for " + std::to_string(rows) +
                                       " rows need an index (or one table, or one a row)");
}

RuleParams rules_of(const ppocr_logit_rules* r, const LogitRows& rows) {
  RuleParams p{};
  if (!r) return p;
  if (r->classes != (size_t)rows.classes)
    raise(PPOCR_ERR_INVALID_INPUT, "rules for " + std::to_string(r->classes) + " classes on logits of " +
                                       std::to_string(rows.classes));
  check_table(r->bias, r->n_bias, r->row_bias, (size_t)rows.rows, "bias");
  check_table(r->masks, r->n_masks, r->row_mask, (size_t)rows.rows, "masks");
  if (!r->history_offsets && (r->history || r->history_len || r->repetition || r->frequency || r->presence))
    raise(PPOCR_ERR_INVALID_INPUT, "penalties need the histories' offsets");
  if (r->history_offsets && r->history_len && !r->history) raise(PPOCR_ERR_INVALID_INPUT, "history is null");
  if (r->history_len > (size_t)1 << 40) raise(PPOCR_ERR_INVALID_INPUT, "the history is longer than 2^40");
  check_aligned(r->bias, 4, "bias");
  check_aligned(r->row_bias, 4, "row_bias");
  check_aligned(r->masks, 4, "masks");
  check_aligned(r->row_mask, 4, "row_mask");
  check_aligned(r->history, 4, "history");
  check_aligned(r->history_offsets, 8, "history_offsets");
  check_aligned(r->repetition, 4, "repetition");
  check_aligned(r->frequency, 4, "frequency");
  check_aligned(r->presence, 4, "presence");
  p.bias = r->bias;
  p.n_bias = (int64_t)r->n_bias;
  p.row_bias = r->row_bias;
  p.masks = r->masks;
  p.n_masks = (int64_t)r->n_masks;
  p.row_mask = r->row_mask;
  if (r->history_len) {
    p.history = r->history;
    p.history_len = (int64_t)r->history_len;
    p.offsets = r->history_offsets;
    p.repetition = r->repetition;
    p.frequency = r->frequency;
    p.presence = r->presence;
  }
  return p;
}

void check_rules_device(const RuleParams& p, int device) {
  check_optional(p.bias, device, "bias");
  check_optional(p.row_bias, device, "row_bias");
  check_optional(p.masks, device, "masks");
  check_optional(p.row_mask, device, "row_mask");
  check_optional(p.history, device, "history");
  check_optional(p.offsets, device, "history_offsets");
  check_optional(p.repetition, device, "repetition");
  check_optional(p.frequency, device, "frequency");
  check_optional(p.presence, device, "presence");
}

void check_top_count(size_t k, const char* what) {
  if (k == 0 || k > (size_t)kMaxTop)
    raise(PPOCR_ERR_INVALID_INPUT, std::string(what) + " must be 1 to " + std::to_string(kMaxTop) + ", got " +
                                       std::to_string(k));
}

void check_temperature(float t) {
  if (!(t >= 1e-3f && t <= 1e3f)) raise(PPOCR_ERR_INVALID_INPUT, "the temperature must be 0.001 to 1000");
}

DistillParams teacher_of(const ppocr_teacher* t, float temperature) {
  if (!t) raise(PPOCR_ERR_INVALID_INPUT, "teacher is null");
  check_top_count(t->k, "the teacher's k");
  check_temperature(temperature);
  check_aligned(t->values, 4, "the teacher's values");
  check_aligned(t->indices, 4, "the teacher's indices");
  check_aligned(t->rest, 4, "the teacher's rest");
  DistillParams p{};
  p.values = t->values;
  p.indices = t->indices;
  p.rest = t->rest;
  p.k = (int)t->k;
  p.temperature = temperature;
  return p;
}

void check_teacher_pointers(const DistillParams& p) {
  if (!p.values || !p.indices) raise(PPOCR_ERR_INVALID_INPUT, "the teacher's values or indices are null");
}

void check_distill_device(const LogitRows& rows, const DistillParams& p, int device) {
  check_device(rows.x, device, "student");
  check_device(p.values, device, "the teacher's values");
  check_device(p.indices, device, "the teacher's indices");
  check_optional(p.rest, device, "the teacher's rest");
  check_optional(p.grad_loss, device, "grad_loss");
  check_optional(p.loss, device, "loss");
  check_optional(p.state, device, "state");
  check_optional(p.grad, device, "grad");
}

int device_of(const ppocr_hip_ctx* ctx) {
  if (!ctx) raise(PPOCR_ERR_INVALID_INPUT, "context is null");
  return context_device(ctx);
}

}  // namespace
}  // namespace ppocr

using namespace ppocr;

extern "C" {

ppocr_status ppocr_hip_logit_rules(ppocr_hip_ctx* ctx, const ppocr_logits* logits, const ppocr_logit_rules* rules,
                                   void* out, size_t out_stride, void* stream) {
  return guarded([&] {
    const LogitRows rows = rows_of(logits, "logits");
    if (!rules) raise(PPOCR_ERR_INVALID_INPUT, "rules are null");
    const RuleParams p = rules_of(rules, rows);
    if (rows.rows) check_output(rows, out, out_stride, "out");
    const int device = device_of(ctx);
    if (rows.rows == 0) return;
    DeviceScope scope(device);
    check_device(rows.x, device, "logits");
    check_device(out, device, "out");
    check_rules_device(p, device);
    launch_logit_rules(rows, p, out, (int64_t)out_stride, static_cast<hipStream_t>(stream));
    HIP_OK(hipGetLastError());
  });
}

ppocr_status ppocr_hip_top_logits(ppocr_hip_ctx* ctx, const ppocr_logits* logits, const ppocr_logit_rules* rules,
                                  size_t k, float temperature, float* values, int32_t* indices, float* rest,
                                  void* stream) {
  return guarded([&] {
    const LogitRows rows = rows_of(logits, "logits");
    check_top_count(k, "k");
    check_temperature(temperature);
    TopParams p{};
    p.rules = rules_of(rules, rows);
    p.k = (int)k;
    p.temperature = temperature;
    p.values = values;
    p.indices = indices;
    p.rest = rest;
    if (rows.rows && (!values || !indices)) raise(PPOCR_ERR_INVALID_INPUT, "values or indices are null");
    check_aligned(values, 4, "values");
    check_aligned(indices, 4, "indices");
    check_aligned(rest, 4, "rest");
    const int device = device_of(ctx);
    if (rows.rows == 0) return;
    DeviceScope scope(device);
    check_device(rows.x, device, "logits");
    check_device(values, device, "values");
    check_device(indices, device, "indices");
    check_optional(rest, device, "rest");
    check_rules_device(p.rules, device);
    launch_top_logits(rows, p, static_cast<hipStream_t>(stream));
    HIP_OK(hipGetLastError());
  });
}

ppocr_status ppocr_hip_distill_loss(ppocr_hip_ctx* ctx, const ppocr_logits* student, const ppocr_teacher* teacher,
                                    float temperature, float* loss, float* state, void* stream) {
  return guarded([&] {
    const LogitRows rows = rows_of(student, "student");
    DistillParams p = teacher_of(teacher, temperature);
    check_aligned(loss, 4, "loss");
    check_aligned(state, 4, "state");
    p.loss = loss;
    p.state = state;
    if (rows.rows) {
      check_teacher_pointers(p);
      if (!loss) raise(PPOCR_ERR_INVALID_INPUT, "loss is null");
    }
    const int device = device_of(ctx);
    if (rows.rows == 0) return;
    DeviceScope scope(device);
    check_distill_device(rows, p, device);
    launch_distill(rows, p, static_cast<hipStream_t>(stream));
    HIP_OK(hipGetLastError());
  });
}

ppocr_status ppocr_hip_distill_grad(ppocr_hip_ctx* ctx, const ppocr_logits* student, const ppocr_teacher* teacher,
                                    const float* state, float temperature, const float* grad_loss, void* grad,
                                    size_t grad_stride, void* stream) {
  return guarded([&] {
    const LogitRows rows = rows_of(student, "student");
    DistillParams p = teacher_of(teacher, temperature);
    check_aligned(state, 4, "state");
    check_aligned(grad_loss, 4, "grad_loss");
    p.state = const_cast<float*>(state);  // only read by the gradient
    p.grad_loss = grad_loss;
    p.grad = grad;
    p.grad_stride = (int64_t)grad_stride;
    if (rows.rows) {
      check_teacher_pointers(p);
      if (!state) raise(PPOCR_ERR_INVALID_INPUT, "state is null");
      check_output(rows, grad, grad_stride, "grad");
    }
    const int device = device_of(ctx);
    if (rows.rows == 0) return;
    DeviceScope scope(device);
    check_distill_device(rows, p, device);
    launch_distill_grad(rows, p, static_cast<hipStream_t>(stream));
    HIP_OK(hipGetLastError());
  });
}

ppocr_status ppocr_hip_distill(ppocr_hip_ctx* ctx, const ppocr_logits* student, const ppocr_teacher* teacher,
                               float temperature, const float* grad_loss, float* loss, void* grad, size_t grad_stride,
                               void* stream) {
  return guarded([&] {
    const LogitRows rows = rows_of(student, "student");
    DistillParams p = teacher_of(teacher, temperature);
    check_aligned(grad_loss, 4, "grad_loss");
    check_aligned(loss, 4, "loss");
    p.loss = loss;
    p.grad_loss = grad_loss;
    p.grad = grad;
    p.grad_stride = (int64_t)grad_stride;
    if (rows.rows) {
      check_teacher_pointers(p);
      if (!loss) raise(PPOCR_ERR_INVALID_INPUT, "loss is null");
      check_output(rows, grad, grad_stride, "grad");
    }
    const int device = device_of(ctx);
    if (rows.rows == 0) return;
    DeviceScope scope(device);
    check_distill_device(rows, p, device);
    launch_distill(rows, p, static_cast<hipStream_t>(stream));
    HIP_OK(hipGetLastError());
  });
}

}  // extern "C"
