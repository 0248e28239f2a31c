// wfe_decoder.h -- launch interface between the C ABI (wfe_decoder_capi.cpp) and the kernels of the decoder's
// vocabulary operators: the cross entropy (wfe_lce.hip) and the token embedding (wfe_embed.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/wfe.h"

namespace wfe {

// ---- cross entropy over the vocabulary -------------------------------------------------------------------
constexpr int kLceRowPad = 256;     // packed hidden rows are padded to this many (the largest row tile)

// What the forward pass leaves for the backward pass, `rows` entries each; r counts kept rows, n all rows.
struct LceState {
  int* head;         // [0] kept rows
  int* index;        // n of kept row r, ascending
  int* label;        // label of kept row r; -1: outside 0..vocab-1
  float* lse;        // log sum exp of its logits
  float* zlab;       // its label's logit
  int* slot;         // r of row n, -1: ignored
};
inline int64_t lce_state_bytes(int64_t rows) { return 64 + 5 * ((rows * 4 + 63) / 64 * 64); }
inline LceState lce_state(void* p, int64_t rows) {
  char* c = static_cast<char*>(p);
  const int64_t step = (rows * 4 + 63) / 64 * 64;
  return {reinterpret_cast<int*>(c), reinterpret_cast<int*>(c + 64), reinterpret_cast<int*>(c + 64 + step),
          reinterpret_cast<float*>(c + 64 + 2 * step), reinterpret_cast<float*>(c + 64 + 3 * step),
          reinterpret_cast<int*>(c + 64 + 4 * step)};
}

hipError_t launch_lce_forward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* labels,
                              float* loss, void* state, void* workspace, hipStream_t stream);
hipError_t launch_lce_backward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* state,
                               const float* upstream, void* grad_hidden, void* grad_weight, void* workspace,
                               hipStream_t stream);
int64_t lce_workspace_bytes(const wfe_linear_ce& d, const void* weight, int backward, int grads);

// ---- token embedding -----------------------------------------------------------------------------------
hipError_t launch_embedding(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out,
                            hipStream_t stream);
hipError_t launch_embedding_backward(const wfe_embedding_desc& d, const void* ids, const void* grad_out,
                                     void* grad_weight, void* workspace, hipStream_t stream);
int64_t embedding_workspace_bytes(const wfe_embedding_desc& d);

}  // namespace wfe
