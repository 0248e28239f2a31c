// wfe_decoder.h -- launch interface between the C ABI (wfe_decoder_capi.cpp) and the kernels of the decoder's
// vocabulary operators: the cross entropy (wfe_lce.hip) and the token embedding (wfe_embed.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/wfe.h"

namespace wfe {

// ---- cross entropy over the vocabulary -------------------------------------------------------------------
constexpr int kLceRowPad = 256;     // packed hidden rows are padded to this many (the largest row tile)

inline int lce_dim_pad(const wfe_linear_ce& d) {            // whole multiples of 128 bytes
  const int e = d.dtype == WFE_F32 ? 32 : 64;
  return (d.dim + e - 1) / e * e;
}
inline int64_t lce_row_pad(const wfe_linear_ce& d) {
  return ((d.rows > 0 ? d.rows : 1) + kLceRowPad - 1) / kLceRowPad * kLceRowPad;
}

// What the forward pass leaves for the backward pass; r counts kept rows, n all rows.
struct LceState {
  int* head;         // [0] kept rows
  int* index;        // n of kept row r, ascending
  int* label;        // label of kept row r; -1: outside 0..vocab-1
  float* lse;        // log sum exp of its logits
  float* zlab;       // its label's logit
  int* slot;         // r of row n, -1: ignored
  void* packed;      // the kept rows of hidden, (row_pad, dim_pad), zeros up to a multiple of 64 rows behind them
};
inline int64_t lce_state_bytes(const wfe_linear_ce& d) {
  return 256 + 5 * lce_row_pad(d) * 4 + lce_row_pad(d) * lce_dim_pad(d) * (d.dtype == WFE_F32 ? 4 : 2);
}
inline LceState lce_state(void* p, const wfe_linear_ce& d) {
  char* c = static_cast<char*>(p) + 256;
  const int64_t step = lce_row_pad(d) * 4;
  return {static_cast<int*>(p), reinterpret_cast<int*>(c), reinterpret_cast<int*>(c + step),
          reinterpret_cast<float*>(c + 2 * step), reinterpret_cast<float*>(c + 3 * step),
          reinterpret_cast<int*>(c + 4 * step), c + 5 * step};
}

hipError_t launch_lce_forward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* labels,
                              float* loss, void* state, void* workspace, hipStream_t stream);
hipError_t launch_lce_backward(const wfe_linear_ce& d, const void* weight, const void* state, const float* upstream,
                               void* grad_hidden, void* grad_weight, void* workspace, hipStream_t stream);
int64_t lce_workspace_bytes(const wfe_linear_ce& d, const void* weight, int backward, int grads);

// ---- token embedding -----------------------------------------------------------------------------------
hipError_t launch_embedding(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out,
                            hipStream_t stream);
hipError_t launch_embedding_backward(const wfe_embedding_desc& d, const void* ids, const void* grad_out,
                                     void* grad_weight, void* workspace, hipStream_t stream);
int64_t embedding_workspace_bytes(const wfe_embedding_desc& d);
bool embedding_backward_fits(const wfe_embedding_desc& d);      // a launch has fewer than 2^32 threads

}  // namespace wfe
