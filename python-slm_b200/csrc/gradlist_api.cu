// C ABI of gradient lists (include/slmopt.h): lifetime and checks of a list, the
// norm, clip and accumulate calls, and the optimizer step on a list.
#include "handle.h"

#include <algorithm>
#include <atomic>
#include <exception>
#include <new>
#include <numeric>
#include <utility>

using namespace slmopt;

namespace {

struct Extent {
  uintptr_t lo, hi;  // bytes
  uint32_t tensor;
};

// What depends on the tensors' addresses.
struct Addresses {
  std::vector<Extent> extents;  // non-empty tensors by address
  bool overlapping = false;     // two tensors share an element
  uint32_t off_runs = 0;        // see GradListView
};

uint32_t type_bytes(uint32_t type) { return type == kGradF32 ? 4u : 2u; }

}  // namespace

struct slm_grad_list {
  int device = 0;
  std::vector<GradTensor> tensors;
  std::vector<uint64_t> rows;  // 1 for contiguous tensors
  Addresses at;
  uint32_t pitched = 0;  // whether any tensor is rows with a pitch
  uint32_t off_vectors = 0, types = 0;  // see GradListView; bit per type of a tensor with elements
  uint64_t elements = 0;
  uint32_t unit_elems = kGradUnitMin;
  uint32_t n_units = 0;
  uint32_t keep = 0, cluster = 0, sms = 1;  // see GradListView
  GradTensor* d_tensors = nullptr;
  GradUnit* d_units = nullptr;
  // The owner, and one for every handle between its norm pass and update pass.
  std::atomic<int> holders{1};

  GradListView view() const {
    return GradListView{d_units, d_tensors, n_units, uint32_t(tensors.size()), unit_elems, pitched,
                        at.off_runs, off_vectors, types, cluster, sms, keep};
  }
};

namespace {

uint64_t span_bytes(const GradTensor& t, uint64_t rows) {
  const uint64_t size = type_bytes(t.flags & kGradTypeMask);
  return ((t.flags & kGradPitched) ? (rows - 1) * t.row_stride + t.columns : t.elements) * size;
}

uint32_t layout_flags(uint32_t type, bool pitched, const void* ptr, uint64_t columns,
                      uint64_t row_stride) {
  uint32_t f = type | (pitched ? kGradPitched : 0u);
  const uint64_t size = type_bytes(type), vec = kVec * size;
  if (reinterpret_cast<uintptr_t>(ptr) % vec == 0 &&
      (!pitched || (columns % kVec == 0 && row_stride * size % vec == 0)))
    f |= kGradVector;
  return f;
}

// Whether two tensors whose extents overlap share an element.  In rows as far
// apart as the two pitches allow (their greatest common divisor; a contiguous tensor
// is one row and goes with any pitch) they do not when their columns differ;
// other pairs count as sharing.
bool share_elements(const GradTensor& a, const GradTensor& b) {
  const bool ordered = uintptr_t(a.ptr) <= uintptr_t(b.ptr);
  const GradTensor &x = ordered ? a : b, &y = ordered ? b : a;
  const uint64_t sx = type_bytes(x.flags & kGradTypeMask), sy = type_bytes(y.flags & kGradTypeMask);
  const bool px = x.flags & kGradPitched, py = y.flags & kGradPitched;
  const uint64_t pitch = std::gcd(px ? x.row_stride * sx : 0u, py ? y.row_stride * sy : 0u);
  const uint64_t wide_x = (px ? x.columns : x.elements) * sx;  // of a row
  const uint64_t wide_y = (py ? y.columns : y.elements) * sy;
  if (pitch == 0u) return true;
  const uint64_t delta = uintptr_t(y.ptr) - uintptr_t(x.ptr);
  const uint64_t col = delta % pitch;  // y's first column within x's rows
  return col < wide_x || col + wide_y > pitch;
}

Addresses look_at_addresses(const std::vector<GradTensor>& tensors,
                            const std::vector<uint64_t>& rows) {
  Addresses at;
  for (uint32_t k = 0; k < tensors.size(); ++k) {
    const GradTensor& t = tensors[k];
    if (!t.elements) continue;
    if (!(t.flags & kGradVector)) at.off_runs = 1;
    at.extents.push_back(Extent{uintptr_t(t.ptr), uintptr_t(t.ptr) + span_bytes(t, rows[k]), k});
  }
  std::sort(at.extents.begin(), at.extents.end(),
            [](const Extent& a, const Extent& b) { return a.lo < b.lo; });
  for (size_t i = 0; i < at.extents.size() && !at.overlapping; ++i)
    for (size_t j = i + 1; j < at.extents.size() && at.extents[j].lo < at.extents[i].hi; ++j)
      if (share_elements(tensors[at.extents[i].tensor], tensors[at.extents[j].tensor])) {
        at.overlapping = true;
        break;
      }
  return at;
}

// Device memory of the list's device, aligned to its element size.
int check_pointer(const void* p, uint32_t type, int device) {
  if (!p) return fail(SLM_ERR_INVALID_ARGUMENT, "a gradient tensor with elements has no address");
  if (reinterpret_cast<uintptr_t>(p) % type_bytes(type) != 0)
    return fail(SLM_ERR_INVALID_ARGUMENT, "gradients must be aligned to their element size");
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return fail(SLM_ERR_INVALID_ARGUMENT, "a gradient tensor's address is unknown to CUDA");
  }
  if ((a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) ||
      (a.type == cudaMemoryTypeDevice && a.device != device))
    return fail(SLM_ERR_INVALID_ARGUMENT,
                "gradient tensors must lie in the memory of the list's device");
  return SLM_OK;
}

int cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return SLM_OK;
  return fail(e == cudaErrorMemoryAllocation ? SLM_ERR_OUT_OF_MEMORY : SLM_ERR_CUDA,
              std::string(what) + ": " + cudaGetErrorString(e));
}

int fill_list(slm_grad_list* l, const slm_grad_view* views, uint32_t n) {
  l->tensors.resize(n);
  l->rows.resize(n);
  for (uint32_t k = 0; k < n; ++k) {
    const slm_grad_view& v = views[k];
    if (v.dtype != SLM_DTYPE_F32 && v.dtype != SLM_DTYPE_BF16 && v.dtype != SLM_DTYPE_F16)
      return fail(SLM_ERR_INVALID_ARGUMENT, "unknown gradient dtype");
    constexpr uint64_t kMost = 1ull << 48;
    if (v.rows > kMost || v.columns > kMost || v.row_stride > kMost ||
        (v.rows && v.columns > kMost / v.rows) || (v.rows && v.row_stride > kMost / v.rows))
      return fail(SLM_ERR_SIZE_LIMIT, "a gradient tensor is larger than any memory");
    GradTensor& t = l->tensors[k];
    t = GradTensor{};
    t.ptr = v.data;
    t.elements = v.rows * v.columns;
    t.columns = v.columns ? v.columns : 1;
    t.row_stride = v.row_stride;
    const bool pitched = t.elements && v.rows > 1 && v.row_stride != v.columns;
    if (pitched && v.row_stride < v.columns)
      return fail(SLM_ERR_INVALID_ARGUMENT, "a gradient tensor's rows overlap");
    if (pitched && v.columns > (1u << 30))
      return fail(SLM_ERR_SIZE_LIMIT, "rows with a pitch have at most 2^30 columns");
    l->rows[k] = pitched ? v.rows : 1;
    if (pitched) l->pitched = 1;
    if (t.elements) l->types |= 1u << uint32_t(v.dtype);
    t.flags = layout_flags(uint32_t(v.dtype), pitched, v.data, t.columns, t.row_stride);
    t.offset = l->elements;
    if (t.elements && t.offset % kVec) l->off_vectors = 1;
    l->elements += t.elements;
    if (l->elements > kMost) return fail(SLM_ERR_SIZE_LIMIT, "the list is larger than any memory");
  }
  return SLM_OK;
}

int upload_list(slm_grad_list* l) {
  l->unit_elems = grad_unit_elems(l->elements);
  l->cluster = list_small_cluster();
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, l->device) == cudaSuccess &&
      sms > 0)
    l->sms = uint32_t(sms);
  uint64_t units = 0;
  for (GradTensor& t : l->tensors) {
    t.first_unit = uint32_t(units);
    units += (t.elements + l->unit_elems - 1) / l->unit_elems;
    if (units > 0x7fffffffull) return fail(SLM_ERR_SIZE_LIMIT, "the list has too many units");
  }
  l->n_units = uint32_t(units);
  std::vector<GradUnit> table(units);
  for (uint32_t k = 0; k < l->tensors.size(); ++k) {
    const GradTensor& t = l->tensors[k];
    const uint64_t size = type_bytes(t.flags & kGradTypeMask);
    for (uint64_t e = 0, i = 0; e < t.elements; e += l->unit_elems, ++i) {
      GradUnit& u = table[t.first_unit + i];
      uint64_t at = e;
      if (t.flags & kGradPitched) {
        u.row_stride = t.row_stride;
        u.columns = uint32_t(t.columns);
        u.column = uint32_t(e % t.columns);
        at = e / t.columns * t.row_stride + u.column;
      }
      u.ptr = static_cast<const uint8_t*>(t.ptr) + at * size;
      u.count = uint32_t(std::min<uint64_t>(l->unit_elems, t.elements - e));
      u.tensor = k;
      u.index = uint32_t(i);
      u.flags = t.flags;
      u.offset = t.offset + e;
    }
  }
  l->keep = l->n_units;
  for (uint64_t bytes = 0; l->keep > 0; --l->keep) {
    const GradUnit& u = table[l->keep - 1];
    bytes += uint64_t(u.count) * type_bytes(u.flags & kGradTypeMask);
    if (bytes > kGradKeepBytes) break;
  }
  int st;
  const size_t tensor_bytes = l->tensors.size() * sizeof(GradTensor);
  if ((st = cuda_status(cudaMalloc(&l->d_tensors, tensor_bytes), "cudaMalloc list tensors")))
    return st;
  if ((st = cuda_status(cudaMalloc(&l->d_units, std::max<size_t>(1, units) * sizeof(GradUnit)),
                        "cudaMalloc list units")))
    return st;
  // Pageable copies: they have left the host when the calls return.
  if ((st = cuda_status(cudaMemcpy(l->d_tensors, l->tensors.data(), tensor_bytes,
                                   cudaMemcpyHostToDevice),
                        "upload list tensors")))
    return st;
  if (units && (st = cuda_status(cudaMemcpy(l->d_units, table.data(), units * sizeof(GradUnit),
                                            cudaMemcpyHostToDevice),
                                 "upload list units")))
    return st;
  return cuda_status(cudaStreamSynchronize(nullptr), "upload list");
}

uint64_t partial_bytes(uint64_t units) { return (units ? units : 1) * sizeof(GradPartial); }

bool positive(float v) { return v > 0.0f && finite_f32(v); }

// The checks that the norm and clip calls share.
int check_norm_call(const slm_grad_list* list, float loss_scale, float max_norm, int kind,
                    const slm_list_norm* result, const float* norms, const float* tops,
                    const double* sum_squares, const void* workspace, uint64_t bytes) {
  if (!list || !result || !workspace) return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  if (!positive(loss_scale) || !positive(max_norm))
    return fail(SLM_ERR_INVALID_ARGUMENT, "loss scale and max norm must be positive and finite");
  if (kind != SLM_NORM_L2 && kind != SLM_NORM_MAX)
    return fail(SLM_ERR_INVALID_ARGUMENT, "unknown norm kind");
  if (reinterpret_cast<uintptr_t>(result) % 4 != 0 || reinterpret_cast<uintptr_t>(norms) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(tops) % 4 != 0 || reinterpret_cast<uintptr_t>(sum_squares) % 8 != 0)
    return fail(SLM_ERR_INVALID_ARGUMENT, "results must be aligned to their element size");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(SLM_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  if (bytes < partial_bytes(list->n_units))
    return fail(SLM_ERR_INVALID_ARGUMENT,
                "the workspace is smaller than slm_grad_list_workspace_bytes(list)");
  return SLM_OK;
}

// Whether an element of `out` lies on an element of `list` other than, for the
// same tensor in the same layout and type, itself.
bool collides(const slm_grad_list& list, const slm_grad_list& out) {
  size_t i = 0;
  for (const Extent& o : out.at.extents) {
    while (i < list.at.extents.size() && list.at.extents[i].hi <= o.lo) ++i;
    for (size_t j = i; j < list.at.extents.size() && list.at.extents[j].lo < o.hi; ++j) {
      if (list.at.extents[j].hi <= o.lo) continue;
      const uint32_t a = list.at.extents[j].tensor, b = o.tensor;
      const GradTensor &x = list.tensors[a], &y = out.tensors[b];
      if (a == b && x.ptr == y.ptr && x.flags == y.flags &&
          (!(x.flags & kGradPitched) || (x.row_stride == y.row_stride && x.columns == y.columns)))
        continue;
      if (share_elements(x, y)) return true;
    }
  }
  return false;
}

// Whether one of n contiguous f32 values lies on an element of `list`.
bool collides(const slm_grad_list& list, const float* values, uint64_t n) {
  GradTensor run{};
  run.ptr = values;
  run.elements = n;
  run.flags = kGradF32;
  const uintptr_t lo = reinterpret_cast<uintptr_t>(values), hi = lo + n * sizeof(float);
  for (const Extent& x : list.at.extents)
    if (x.lo < hi && lo < x.hi && share_elements(list.tensors[x.tensor], run)) return true;
  return false;
}

// Checks of a list against an optimizer handle's tensor table.
int check_step_list(slm_opt_handle* h, const slm_grad_list* list) {
  if (h->sharded())
    return h->err(SLM_ERR_INVALID_ARGUMENT,
                  "a ZeRO-1 handle takes its gradients in one buffer (slm_opt_gradient_buffer)");
  if (list->device != h->device)
    return h->err(SLM_ERR_INVALID_ARGUMENT, "the list is on another device than the handle");
  bool same = list->tensors.size() + 1 == h->offsets.size();
  for (size_t k = 0; same && k < list->tensors.size(); ++k)
    same = list->tensors[k].elements == h->offsets[k + 1] - h->offsets[k];
  if (!same)
    return h->err(SLM_ERR_E1_PARAMETER_LAYOUT_MISMATCH,
                  "the list's tensors are not the handle's parameters");
  return SLM_OK;
}

// A list without holders, whose work has been waited for.
void free_list(slm_grad_list* list) {
  DeviceGuard guard(list->device);
  cudaFree(list->d_tensors);
  cudaFree(list->d_units);
  delete list;
}

}  // namespace

void slmopt::drop_norm_pass(slm_opt_handle* h, cudaStream_t s) {
  h->pass_grads = nullptr;
  slm_grad_list* list = h->pass_list;
  h->pass_list = nullptr;
  if (!list || list->holders.fetch_sub(1) != 1) return;
  // Its owner has destroyed it, which waited for what was enqueued then: an update
  // pass on s at most has come since.  A graph that captures that goes on to read
  // the list, which is kept as long as the handle.
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(s, &status) != cudaSuccess) cudaGetLastError();
  if (status != cudaStreamCaptureStatusNone) {
    try {
      h->parked_lists.push_back(list);
    } catch (const std::exception&) {  // without room to note it, it is kept for good
    }
    return;
  }
  cudaStreamSynchronize(s);
  free_list(list);
}

void slmopt::free_parked_lists(slm_opt_handle* h) {
  for (slm_grad_list* list : h->parked_lists) free_list(list);
  h->parked_lists.clear();
}

uint64_t slmopt::list_partial_bytes(const std::vector<uint64_t>& offsets) {
  const uint32_t unit = grad_unit_elems(offsets.back());
  uint64_t units = 0;
  for (size_t k = 0; k + 1 < offsets.size(); ++k)
    units += (offsets[k + 1] - offsets[k] + unit - 1) / unit;
  return partial_bytes(units);
}

int slmopt::enqueue_list_norm(slm_opt_handle* h, const slm_grad_list* list,
                              const slm_step_config* cfg, cudaStream_t s) {
  return h->cuda(launch_list_norm_decide(list->view(),
                                         static_cast<GradPartial*>(h->d_list_partials),
                                         h->d_scaler, h->d_state, finalize_params(h, cfg), s),
                 "list norm kernel");
}

int slmopt::enqueue_list_update(slm_opt_handle* h, const slm_grad_list* list,
                                const slm_step_config* cfg, bool chained, cudaStream_t s) {
  return h->cuda(launch_list_update(list->view(), h->master, h->m1, h->m2, h->w16, h->d_decay,
                                    adamw_params(cfg), h->d_state, chained, s),
                 "list update kernel");
}

extern "C" {

int slm_grad_list_create(const slm_grad_view* views, uint32_t n, int device,
                         slm_grad_list** out) {
  if (!out) return fail(SLM_ERR_INVALID_ARGUMENT, "out is NULL");
  *out = nullptr;
  if (!views || n == 0) return fail(SLM_ERR_INVALID_ARGUMENT, "the list contains no tensors");
  slm_grad_list* l = nullptr;
  int st = SLM_OK;
  try {
    l = new slm_grad_list();
    st = fill_list(l, views, n);
    if (!st) {
      int count = 0;
      if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0)
        st = fail(SLM_ERR_NO_DEVICE, "no CUDA device is visible");
      else if (device < 0 || device >= count)
        st = fail(SLM_ERR_INVALID_ARGUMENT, "device ordinal out of range");
    }
    for (uint32_t k = 0; k < n && !st; ++k)
      if (l->tensors[k].elements)
        st = check_pointer(l->tensors[k].ptr, l->tensors[k].flags & kGradTypeMask, device);
    if (!st) {
      l->device = device;
      l->at = look_at_addresses(l->tensors, l->rows);
      DeviceGuard guard(device);
      st = guard.ok ? upload_list(l) : fail(SLM_ERR_CUDA, "cudaSetDevice failed");
    }
  } catch (const std::exception&) {
    st = fail(SLM_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  if (st) {
    const std::string why = g_last_error;
    slm_grad_list_destroy(l);
    return fail(st, why);
  }
  *out = l;
  return SLM_OK;
}

int slm_grad_list_destroy(slm_grad_list* list) {
  if (!list) return SLM_OK;
  if (!list->d_tensors && !list->d_units) {  // never came to a device
    delete list;
    return SLM_OK;
  }
  DeviceGuard guard(list->device);
  // Work enqueued with the list (on any stream) has read its tables, and its
  // tensors, when this returns; an update pass to come may still read them.
  const cudaError_t e = cudaDeviceSynchronize();
  if (e >= cudaErrorStreamCaptureUnsupported && e <= cudaErrorStreamCaptureWrongThread) {
    cudaGetLastError();
    return fail(SLM_ERR_CUDA, "a gradient list cannot be destroyed while a stream is captured");
  }
  if (list->holders.fetch_sub(1) == 1) free_list(list);
  return SLM_OK;
}

uint64_t slm_grad_list_elements(const slm_grad_list* list) { return list ? list->elements : 0; }

uint64_t slm_grad_list_workspace_bytes(const slm_grad_list* list) {
  return list ? partial_bytes(list->n_units) : 0;
}

int slm_grad_list_bind(slm_grad_list* list, const void* const* data, uint32_t n, void* stream) {
  if (!list || !data) return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  if (n != list->tensors.size())
    return fail(SLM_ERR_INVALID_ARGUMENT, "one address per tensor of the list is needed");
  for (uint32_t k = 0; k < n; ++k)
    if (list->tensors[k].elements)
      if (int st = check_pointer(data[k], list->tensors[k].flags & kGradTypeMask, list->device))
        return st;
  // The list's own tables change only once the device's are going to.
  std::vector<GradTensor> tensors;
  Addresses at;
  try {
    tensors = list->tensors;
    for (uint32_t k = 0; k < n; ++k) {
      GradTensor& t = tensors[k];
      t.ptr = data[k];
      t.flags = layout_flags(t.flags & kGradTypeMask, (t.flags & kGradPitched) != 0u, t.ptr,
                             t.columns, t.row_stride);
    }
    at = look_at_addresses(tensors, list->rows);
  } catch (const std::exception&) {
    return fail(SLM_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  DeviceGuard guard(list->device);
  for (uint32_t begin = 0; begin < n; begin += kGradBindBatch) {
    GradBind b;
    const uint32_t m = std::min(kGradBindBatch, n - begin);
    for (uint32_t i = 0; i < kGradBindBatch; ++i) {
      b.ptr[i] = i < m ? tensors[begin + i].ptr : nullptr;
      b.flags[i] = i < m ? tensors[begin + i].flags : 0u;
    }
    if (int st = cuda_status(launch_list_bind(list->d_tensors, list->d_units, list->n_units,
                                              list->unit_elems, b, begin, m,
                                              static_cast<cudaStream_t>(stream)),
                             "list bind kernel"))
      return st;
  }
  list->tensors.swap(tensors);
  std::swap(list->at, at);
  return SLM_OK;
}

int slm_grad_list_norm(const slm_grad_list* list, float loss_scale, float max_norm, int kind,
                       slm_list_norm* result_device, float* tensor_norms_device,
                       float* tensor_max_device, double* sum_squares_device,
                       void* workspace_device, uint64_t workspace_bytes, void* stream) {
  int st = check_norm_call(list, loss_scale, max_norm, kind, result_device, tensor_norms_device,
                           tensor_max_device, sum_squares_device, workspace_device,
                           workspace_bytes);
  if (st) return st;
  DeviceGuard guard(list->device);
  const GradListOut out{&result_device->norm, tensor_norms_device, tensor_max_device,
                        sum_squares_device};
  return cuda_status(launch_list_norm(list->view(), loss_scale, max_norm, kind, out,
                                      static_cast<GradPartial*>(workspace_device),
                                      static_cast<cudaStream_t>(stream)),
                     "list norm kernels");
}

int slm_grad_list_clip(const slm_grad_list* list, const slm_grad_list* out, float loss_scale,
                       float max_norm, int kind, slm_list_norm* result_device,
                       float* tensor_norms_device, float* tensor_max_device,
                       double* sum_squares_device, void* workspace_device,
                       uint64_t workspace_bytes, void* stream) {
  int st = check_norm_call(list, loss_scale, max_norm, kind, result_device, tensor_norms_device,
                           tensor_max_device, sum_squares_device, workspace_device,
                           workspace_bytes);
  if (st) return st;
  const bool in_place = !out || out == list;
  const slm_grad_list* to = in_place ? list : out;
  if (to->device != list->device)
    return fail(SLM_ERR_INVALID_ARGUMENT, "the output list is on another device");
  if (to->at.overlapping)
    return fail(SLM_ERR_INVALID_ARGUMENT,
                "tensors of the list that is written share elements, which would be clipped twice");
  if (!in_place) {
    bool same = to->tensors.size() == list->tensors.size();
    for (size_t k = 0; same && k < to->tensors.size(); ++k)
      same = to->tensors[k].elements == list->tensors[k].elements;
    if (!same)
      return fail(SLM_ERR_INVALID_ARGUMENT, "the output list's tensors have other sizes");
    if (collides(*list, *to))
      return fail(SLM_ERR_INVALID_ARGUMENT,
                  "an output tensor overlaps a gradient tensor without being that tensor");
  }
  DeviceGuard guard(list->device);
  const GradListOut o{&result_device->norm, tensor_norms_device, tensor_max_device,
                      sum_squares_device};
  return cuda_status(launch_list_clip(list->view(), to->view(), in_place, loss_scale, max_norm,
                                      kind, o, static_cast<GradPartial*>(workspace_device),
                                      static_cast<cudaStream_t>(stream)),
                     "list clip kernels");
}

int slm_grad_list_accumulate(const slm_grad_list* list, float* acc_device, uint64_t n,
                             int overwrite, void* stream) {
  // An accumulator without elements may have no address.
  if (!list || (!acc_device && list->elements))
    return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  if (n != list->elements)
    return fail(SLM_ERR_INVALID_ARGUMENT, "the accumulator needs one value per list element");
  if (reinterpret_cast<uintptr_t>(acc_device) % 16 != 0)
    return fail(SLM_ERR_INVALID_ARGUMENT, "the accumulator must be 16-byte aligned");
  if (collides(*list, acc_device, n))
    return fail(SLM_ERR_INVALID_ARGUMENT, "the accumulator overlaps a gradient tensor");
  DeviceGuard guard(list->device);
  return cuda_status(launch_list_accumulate(list->view(), acc_device, overwrite,
                                            static_cast<cudaStream_t>(stream)),
                     "list accumulate kernel");
}

int slm_opt_step_list(slm_opt_handle* h, const slm_grad_list* list, const slm_step_config* cfg,
                      slm_step_result* out, void* stream) {
  if (!h || !list) return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  int st = check_config(h, cfg);
  if (!st) st = check_step_list(h, list);
  if (st) return st;
  if (h->broken) return h->err(SLM_ERR_INTERNAL, "a previous step failed inside a kernel");
  DeviceGuard guard(h->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  drop_norm_pass(h, s);
  if ((st = phase_begin(h, s))) return st;
  if ((st = enqueue_list_norm(h, list, cfg, s))) return st;
  if ((st = phase_mark(h, s))) return st;
  if ((st = enqueue_list_update(h, list, cfg, true, s))) return st;
  if ((st = phase_mark(h, s))) return st;
  phase_end(h);
  return finish_step(h, out, s);
}

int slm_opt_norm_pass_list(slm_opt_handle* h, slm_grad_list* list,
                           const slm_step_config* cfg, void* stream) {
  if (!h || !list) return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  int st = check_config(h, cfg);
  if (!st) st = check_step_list(h, list);
  if (st) return st;
  DeviceGuard guard(h->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  drop_norm_pass(h, s);
  if ((st = enqueue_list_norm(h, list, cfg, s))) return st;
  list->holders.fetch_add(1);
  h->pass_list = list;
  h->pending = true;
  h->pending_stream = s;
  return SLM_OK;
}

int slm_opt_norm_pass_accumulate_list(slm_opt_handle* h, float* acc_device,
                                      const slm_grad_list* list, int overwrite,
                                      const slm_step_config* cfg, void* stream) {
  if (!h || !acc_device || !list) return fail(SLM_ERR_INVALID_ARGUMENT, "NULL argument");
  int st = check_config(h, cfg);
  if (!st) st = check_step_list(h, list);
  if (st) return st;
  if (reinterpret_cast<uintptr_t>(acc_device) % 16 != 0)
    return h->err(SLM_ERR_INVALID_ARGUMENT, "the accumulator must be 16-byte aligned");
  if (collides(*list, acc_device, h->P))
    return h->err(SLM_ERR_INVALID_ARGUMENT, "the accumulator overlaps a gradient tensor");
  DeviceGuard guard(h->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  drop_norm_pass(h, s);
  const FinalizeParams fp = finalize_params(h, cfg);
  GradPartial* part = static_cast<GradPartial*>(h->d_list_partials);
  const GradListView v = list->view();
  if ((st = h->cuda(launch_list_accumulate_norm(v, acc_device, overwrite, fp.static_scale,
                                                fp.dynamic ? h->d_scaler : nullptr, part, s),
                    "list accumulate + norm kernel")))
    return st;
  if ((st = h->cuda(launch_list_decide(v, part, h->d_scaler, h->d_state, fp, s),
                    "list decide kernel")))
    return st;
  h->pass_grads = acc_device;
  h->pass_dtype = SLM_DTYPE_F32;
  h->pending = true;
  h->pending_stream = s;
  return SLM_OK;
}

}  // extern "C"
