// wfe_embed.hip -- token embedding with a scale, and the gradient of the embedding matrix, for gfx950.
//
//   out_n = s W_{id_n}            dW_v = s sum_{n: id_n = v} dout_n
//
// Both move memory and compute next to nothing.  The gradient is (vocab, dim) however few tokens occur, so writing it
// is most of the work; it is written once, zeros and sums alike, by reading the tokens in sorted order.
#include <hip/hip_runtime.h>

#include "wfe_decoder.h"

namespace wfe {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ inline long long id_at(const void* ids, int bits, long long n) {
  return bits == 64 ? static_cast<const long long*>(ids)[n] : static_cast<const int*>(ids)[n];
}

// 16 bytes of T, or a ragged end
template <typename T>
struct Vec {
  static constexpr int kN = 16 / (int)sizeof(T);
  T x[kN];
  __device__ void load(const T* p, int left, bool wide) {
    if (wide && left >= kN) __builtin_memcpy(x, __builtin_assume_aligned(p, 16), 16);
    else
      for (int e = 0; e < kN; ++e) x[e] = e < left ? p[e] : static_cast<T>(0.f);
  }
  __device__ void store(T* p, int left, bool wide) const {
    if (wide && left >= kN) __builtin_memcpy(__builtin_assume_aligned(p, 16), x, 16);
    else
      for (int e = 0; e < kN && e < left; ++e) p[e] = x[e];
  }
};

// One wave per token.
template <typename T>
__global__ __launch_bounds__(256) void embed_kernel(const void* ids, int id_bits, long long rows, const T* weight,
                                                    long long ld, int dim, int vocab, float scale, T* out) {
  const long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= rows) return;
  const long long id = id_at(ids, id_bits, n);
  const bool known = id >= 0 && id < vocab;
  const T* in = weight + (known ? id : 0) * ld;
  T* to = out + n * dim;
  const bool wide = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(to)) & 15) == 0;
  for (int d = (threadIdx.x & 63) * Vec<T>::kN; d < dim; d += 64 * Vec<T>::kN) {
    Vec<T> v;
    v.load(in + d, dim - d, wide);
    for (int e = 0; e < Vec<T>::kN; ++e)
      v.x[e] = known ? static_cast<T>(static_cast<float>(v.x[e]) * scale) : static_cast<T>(__builtin_nanf(""));
    v.store(to + d, dim - d, wide);
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------
// Sorting by token, stable, in one launch: a block owns kBins rows of the vocabulary and reads all ids itself, once
// to count (tokens below its rows give the place where its part of the sorted list starts) and once to place.  No
// block needs another's result.
constexpr int kBins = 256, kSortWaves = 16;

__global__ __launch_bounds__(kSortWaves * 64) void embed_sort_kernel(const void* ids, int id_bits, long long rows,
                                                                     int vocab, long long padding, int* start,
                                                                     int* order) {
  __shared__ int place[kSortWaves][kBins];     // counts, then next places, per wave and row
  __shared__ int below_of[kSortWaves];
  __shared__ int scan[kBins];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long v0 = (long long)blockIdx.x * kBins;
  for (int i = threadIdx.x; i < kSortWaves * kBins; i += kSortWaves * 64) (&place[0][0])[i] = 0;
  __syncthreads();
  // wave w takes a contiguous run of the tokens
  const long long each = ((rows + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const long long first = wave * each, last = min(first + each, rows);
  int below = 0;
  for (long long n = first + lane; n < last; n += 64) {
    const long long id = id_at(ids, id_bits, n);
    const bool counted = id >= 0 && id < vocab && id != padding;
    if (counted && id < v0) ++below;
    else if (counted && id < v0 + kBins) atomicAdd(&place[wave][(int)(id - v0)], 1);
  }
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_of[wave] = below;
  __syncthreads();
  int total = 0;
  if (threadIdx.x < kBins) {
    for (int w = 0; w < kSortWaves; ++w) total += place[w][threadIdx.x];
    scan[threadIdx.x] = total;
  }
  __syncthreads();
  for (int d = 1; d < kBins; d <<= 1) {        // inclusive sums
    int add = 0;
    if (threadIdx.x < kBins && (int)threadIdx.x >= d) add = scan[threadIdx.x - d];
    __syncthreads();
    if (threadIdx.x < kBins) scan[threadIdx.x] += add;
    __syncthreads();
  }
  if (threadIdx.x < kBins) {
    int at = scan[threadIdx.x] - total;
    for (int w = 0; w < kSortWaves; ++w) at += below_of[w];
    if (v0 + threadIdx.x < vocab) start[v0 + threadIdx.x] = at;
    if (v0 + threadIdx.x == vocab - 1) start[vocab] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = place[w][threadIdx.x];
      place[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  for (long long n0 = first; n0 < last; n0 += 64) {
    const long long n = n0 + lane;
    const long long id = n < last ? id_at(ids, id_bits, n) : -1;
    const int bin = id >= v0 && id < v0 + kBins && id < vocab && id != padding ? (int)(id - v0) : -1;
    unsigned long long left = __ballot(bin >= 0);
    while (left) {                             // one step per distinct token of the 64
      const int b = __shfl(bin, __ffsll((unsigned long long)left) - 1);
      const unsigned long long same = __ballot(bin == b);
      const int at = place[wave][b];
      if (bin == b) order[at + __popcll(same & ((1ull << lane) - 1))] = (int)n;
      if (lane == 0) place[wave][b] = at + __popcll(same);
      left &= ~same;
    }
  }
}

// One wave per row of the vocabulary.
template <typename T>
__global__ __launch_bounds__(256) void embed_sum_kernel(const int* start, const int* order, const T* grad,
                                                        long long ld, int dim, int vocab, float scale, void* out,
                                                        int out_f32) {
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v >= vocab) return;
  const int first = start[v], last = start[v + 1];
  constexpr int kN = Vec<T>::kN;
  const bool wide = (reinterpret_cast<uintptr_t>(grad) & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0;
  for (int d = (threadIdx.x & 63) * kN; d < dim; d += 64 * kN) {
    float sum[kN];
    for (int e = 0; e < kN; ++e) sum[e] = 0.f;
    for (int i = first; i < last; ++i) {
      Vec<T> x;
      x.load(grad + (long long)order[i] * ld + d, dim - d, wide);
      for (int e = 0; e < kN; ++e) sum[e] += static_cast<float>(x.x[e]);
    }
    const long long at = (long long)v * dim + d;
    if (out_f32) {
      float* to = static_cast<float*>(out) + at;
      for (int e = 0; e < kN && d + e < dim; ++e) to[e] = sum[e] * scale;
    } else {
      Vec<T> x;
      for (int e = 0; e < kN; ++e) x.x[e] = static_cast<T>(sum[e] * scale);
      T* to = static_cast<T*>(out) + at;
      x.store(to, dim - d, (reinterpret_cast<uintptr_t>(to) & 15) == 0);
    }
  }
}

template <typename T>
hipError_t embed(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out, hipStream_t stream) {
  embed_kernel<T><<<dim3((unsigned)((d.rows + 3) / 4)), dim3(256), 0, stream>>>(
      ids, d.id_bits, d.rows, static_cast<const T*>(weight), d.weight_stride, d.dim, d.vocab, d.scale,
      static_cast<T*>(out));
  return hipGetLastError();
}

template <typename T>
hipError_t embed_backward(const wfe_embedding_desc& d, const void* ids, const void* grad, void* grad_weight,
                          void* workspace, hipStream_t stream) {
  int* start = static_cast<int*>(workspace);
  int* order = start + d.vocab + 1;
  embed_sort_kernel<<<dim3((unsigned)((d.vocab + kBins - 1) / kBins)), dim3(kSortWaves * 64), 0, stream>>>(
      ids, d.id_bits, d.rows, d.vocab, d.padding_idx, start, order);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  embed_sum_kernel<T><<<dim3((unsigned)((d.vocab + 3) / 4)), dim3(256), 0, stream>>>(
      start, order, static_cast<const T*>(grad), d.grad_stride, d.dim, d.vocab, d.scale, grad_weight,
      d.grad_weight_dtype == WFE_F32);
  return hipGetLastError();
}

}  // namespace

int64_t embedding_workspace_bytes(const wfe_embedding_desc& d) { return 4 * ((int64_t)d.vocab + 1 + d.rows); }

hipError_t launch_embedding(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out,
                            hipStream_t stream) {
  if (d.dtype == WFE_F32) return embed<float>(d, ids, weight, out, stream);
  if (d.dtype == WFE_F16) return embed<_Float16>(d, ids, weight, out, stream);
  return embed<__bf16>(d, ids, weight, out, stream);
}

hipError_t launch_embedding_backward(const wfe_embedding_desc& d, const void* ids, const void* grad_out,
                                     void* grad_weight, void* workspace, hipStream_t stream) {
  if (d.dtype == WFE_F32) return embed_backward<float>(d, ids, grad_out, grad_weight, workspace, stream);
  if (d.dtype == WFE_F16) return embed_backward<_Float16>(d, ids, grad_out, grad_weight, workspace, stream);
  return embed_backward<__bf16>(d, ids, grad_out, grad_weight, workspace, stream);
}

}  // namespace wfe
