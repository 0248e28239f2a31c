// wfe_decoder_capi.cpp -- the entry points of include/wfe.h for the decoder's vocabulary operators: argument checks
// and launches.  Everything they refuse is refused here, before any device call.
#include <hip/hip_runtime.h>

#include <cstring>

#include "../../include/wfe.h"
#include "wfe_capi_util.h"
#include "wfe_decoder.h"

namespace {

constexpr int64_t kMaxRows = 1 << 24, kMaxVocab = 1 << 24, kMaxDim = 16384;
constexpr int64_t kMaxStride = (int64_t)1 << 46;
constexpr int64_t kMaxLogits = (int64_t)1 << 37;       // a grid has fewer than 2^32 threads: 256 for 128 x 128 logits

bool known_dtype(int32_t t) { return t == WFE_F32 || t == WFE_F16 || t == WFE_BF16; }
int size_of(int32_t t) { return t == WFE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_ce(const wfe_linear_ce* d) {
  using wfe::fail;
  if (!d) return fail(nullptr, WFE_ERR_ARG, "linear_ce: null description");
  if (!known_dtype(d->dtype)) return fail(nullptr, WFE_ERR_ARG, "linear_ce: dtype %d", d->dtype);
  if (d->rows < 0 || d->rows > kMaxRows)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: %lld rows outside 0..%lld", (long long)d->rows, (long long)kMaxRows);
  if (d->dim < 1 || d->dim > kMaxDim)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: dim %d outside 1..%lld", d->dim, (long long)kMaxDim);
  if (d->vocab < 1 || d->vocab > kMaxVocab)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: vocab %d outside 1..%lld", d->vocab, (long long)kMaxVocab);
  if (d->rows * d->vocab > kMaxLogits)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: %lld rows by %d of the vocabulary are more than %lld logits",
                (long long)d->rows, d->vocab, (long long)kMaxLogits);
  if (d->rows > 0 && d->inner < 1) return fail(nullptr, WFE_ERR_ARG, "linear_ce: inner %lld", (long long)d->inner);
  if (d->outer_stride < 0 || d->inner_stride < 0 || d->weight_stride < 0 || d->outer_stride > kMaxStride ||
      d->inner_stride > kMaxStride || d->weight_stride > kMaxStride)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: stride outside 0..2^46");
  if (d->label_bits != 32 && d->label_bits != 64)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: labels of %d bits", d->label_bits);
  if (d->reduction < WFE_REDUCE_NONE || d->reduction > WFE_REDUCE_MEAN)
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: reduction %d", d->reduction);
  if ((d->grad_hidden_dtype != WFE_F32 && d->grad_hidden_dtype != d->dtype) ||
      (d->grad_weight_dtype != WFE_F32 && d->grad_weight_dtype != d->dtype))
    return fail(nullptr, WFE_ERR_ARG, "linear_ce: gradients are float32 or of the inputs' type");
  return WFE_OK;
}

int check_embedding(const wfe_embedding_desc* d) {
  using wfe::fail;
  if (!d) return fail(nullptr, WFE_ERR_ARG, "embedding: null description");
  if (!known_dtype(d->dtype)) return fail(nullptr, WFE_ERR_ARG, "embedding: dtype %d", d->dtype);
  if (d->rows < 0 || d->rows > kMaxRows)
    return fail(nullptr, WFE_ERR_ARG, "embedding: %lld rows outside 0..%lld", (long long)d->rows, (long long)kMaxRows);
  if (d->dim < 1 || d->dim > kMaxDim)
    return fail(nullptr, WFE_ERR_ARG, "embedding: dim %d outside 1..%lld", d->dim, (long long)kMaxDim);
  if (d->vocab < 1 || d->vocab > kMaxVocab)
    return fail(nullptr, WFE_ERR_ARG, "embedding: vocab %d outside 1..%lld", d->vocab, (long long)kMaxVocab);
  if (d->weight_stride < 0 || d->grad_stride < 0 || d->weight_stride > kMaxStride || d->grad_stride > kMaxStride)
    return fail(nullptr, WFE_ERR_ARG, "embedding: stride outside 0..2^46");
  if (d->id_bits != 32 && d->id_bits != 64)
    return fail(nullptr, WFE_ERR_ARG, "embedding: ids of %d bits", d->id_bits);
  if (d->grad_weight_dtype != WFE_F32 && d->grad_weight_dtype != d->dtype)
    return fail(nullptr, WFE_ERR_ARG, "embedding: the gradient is float32 or of the inputs' type");
  return WFE_OK;
}

// One look per process at what every device is
int check_device(int32_t device) {
  constexpr int kMost = 64;
  static const struct Devices {
    int count = 0;
    bool ok[kMost] = {};
    Devices() {
      if (hipGetDeviceCount(&count) != hipSuccess) count = 0;
      if (count > kMost) count = kMost;
      for (int i = 0; i < count; ++i) {
        hipDeviceProp_t prop;
        ok[i] = hipGetDeviceProperties(&prop, i) == hipSuccess && std::strncmp(prop.gcnArchName, "gfx950", 6) == 0;
      }
    }
  } devices;
  if (devices.count < 1) return wfe::fail(nullptr, WFE_ERR_HIP, "no HIP device available: there is no CPU path");
  if (device < 0 || device >= devices.count)
    return wfe::fail(nullptr, WFE_ERR_ARG, "device %d outside 0..%d", device, devices.count - 1);
  if (!devices.ok[device]) return wfe::fail(nullptr, WFE_ERR_HIP, "device %d is not a gfx950", device);
  return WFE_OK;
}

#define CHECKED(expr)               \
  do {                              \
    const int rc_ = (expr);         \
    if (rc_ != WFE_OK) return rc_;  \
  } while (0)

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? WFE_OK : wfe::fail(nullptr, WFE_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int check_workspace(const void* workspace, int64_t have, int64_t need, const char* what) {
  if (have < need)
    return wfe::fail(nullptr, WFE_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)have,
                     (long long)need);
  if (need > 0 && (!workspace || !aligned(workspace, 16)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "%s: workspace null or not on 16 bytes", what);
  return WFE_OK;
}

}  // namespace

extern "C" {

int64_t wfe_linear_ce_state_bytes(const wfe_linear_ce* d) {
  CHECKED(check_ce(d));
  return wfe::lce_state_bytes(*d);
}

int64_t wfe_linear_ce_workspace_bytes(const wfe_linear_ce* d, const void* weight, int32_t backward, int32_t grads) {
  CHECKED(check_ce(d));
  return wfe::lce_workspace_bytes(*d, weight, backward, grads);
}

int wfe_linear_ce_forward(const wfe_linear_ce* d, const void* hidden, const void* weight, const void* labels,
                          float* loss, void* state, void* workspace, int64_t workspace_bytes, void* stream) {
  CHECKED(check_ce(d));
  if (!weight || !state || (d->rows > 0 && (!hidden || !labels)) || (!loss && (d->rows > 0 || d->reduction)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "linear_ce: null device pointer");
  if (!aligned(state, 16) || !aligned(loss, 4) || !aligned(labels, d->label_bits / 8) ||
      !aligned(hidden, size_of(d->dtype)) || !aligned(weight, size_of(d->dtype)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "linear_ce: misaligned pointer");
  CHECKED(check_workspace(workspace, workspace_bytes, wfe::lce_workspace_bytes(*d, weight, 0, 0), "linear_ce"));
  CHECKED(check_device(d->device));
  wfe::DeviceGuard guard(d->device);
  if (!guard.ok) return wfe::fail(nullptr, WFE_ERR_HIP, "hipSetDevice(%d) failed", d->device);
  return launched(wfe::launch_lce_forward(*d, hidden, weight, labels, loss, state, workspace,
                                          static_cast<hipStream_t>(stream)), "linear_ce forward");
}

int wfe_linear_ce_backward(const wfe_linear_ce* d, const void* weight, const void* state, const float* upstream,
                           void* grad_hidden, void* grad_weight, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  CHECKED(check_ce(d));
  if (!grad_hidden && !grad_weight) return WFE_OK;
  if (!weight || !state || (!upstream && (d->rows > 0 || d->reduction)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "linear_ce: null device pointer");
  if (!aligned(state, 16) || !aligned(upstream, 4) || !aligned(weight, size_of(d->dtype)) ||
      !aligned(grad_hidden, 16) || !aligned(grad_weight, 16))
    return wfe::fail(nullptr, WFE_ERR_ARG, "linear_ce: misaligned pointer (gradients start on 16 bytes)");
  const int grads = (grad_hidden ? WFE_GRAD_HIDDEN : 0) | (grad_weight ? WFE_GRAD_WEIGHT : 0);
  CHECKED(check_workspace(workspace, workspace_bytes, wfe::lce_workspace_bytes(*d, weight, 1, grads), "linear_ce"));
  CHECKED(check_device(d->device));
  wfe::DeviceGuard guard(d->device);
  if (!guard.ok) return wfe::fail(nullptr, WFE_ERR_HIP, "hipSetDevice(%d) failed", d->device);
  return launched(wfe::launch_lce_backward(*d, weight, state, upstream, grad_hidden, grad_weight, workspace,
                                           static_cast<hipStream_t>(stream)), "linear_ce backward");
}

int wfe_embedding(const wfe_embedding_desc* d, const void* ids, const void* weight, void* out, void* stream) {
  CHECKED(check_embedding(d));
  if (d->rows == 0) return WFE_OK;
  if (!ids || !weight || !out) return wfe::fail(nullptr, WFE_ERR_ARG, "embedding: null device pointer");
  if (!aligned(ids, d->id_bits / 8) || !aligned(weight, size_of(d->dtype)) || !aligned(out, size_of(d->dtype)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "embedding: misaligned pointer");
  CHECKED(check_device(d->device));
  wfe::DeviceGuard guard(d->device);
  if (!guard.ok) return wfe::fail(nullptr, WFE_ERR_HIP, "hipSetDevice(%d) failed", d->device);
  return launched(wfe::launch_embedding(*d, ids, weight, out, static_cast<hipStream_t>(stream)), "embedding");
}

int64_t wfe_embedding_workspace_bytes(const wfe_embedding_desc* d) {
  CHECKED(check_embedding(d));
  return wfe::embedding_workspace_bytes(*d);
}

int wfe_embedding_backward(const wfe_embedding_desc* d, const void* ids, const void* grad_out, void* grad_weight,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  CHECKED(check_embedding(d));
  if (!wfe::embedding_backward_fits(*d))
    return wfe::fail(nullptr, WFE_ERR_ARG, "embedding: the gradient of %lld rows, %d of the vocabulary and dim %d is more than one "
                     "launch", (long long)d->rows, d->vocab, d->dim);
  if (!grad_weight || (d->rows > 0 && (!ids || !grad_out)))
    return wfe::fail(nullptr, WFE_ERR_ARG, "embedding: null device pointer");
  if (!aligned(ids, d->id_bits / 8) || !aligned(grad_out, size_of(d->dtype)) || !aligned(grad_weight, 16))
    return wfe::fail(nullptr, WFE_ERR_ARG, "embedding: misaligned pointer (the gradient starts on 16 bytes)");
  CHECKED(check_workspace(workspace, workspace_bytes, wfe::embedding_workspace_bytes(*d), "embedding"));
  CHECKED(check_device(d->device));
  wfe::DeviceGuard guard(d->device);
  if (!guard.ok) return wfe::fail(nullptr, WFE_ERR_HIP, "hipSetDevice(%d) failed", d->device);
  return launched(wfe::launch_embedding_backward(*d, ids, grad_out, grad_weight, workspace,
                                                 static_cast<hipStream_t>(stream)), "embedding backward");
}

}  // extern "C"
