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

// One wave per token and slab of columns: few tokens still make many waves, and no wave waits for a second load.
template <typename T>
__global__ __launch_bounds__(256) void embed_kernel(const void* ids, int id_bits, long long rows, const T* weight,
                                                    long long ld, int dim, int vocab, float scale, T* out) {
  constexpr int kSlab = 64 * Vec<T>::kN;
  const unsigned slabs = (unsigned)(dim + kSlab - 1) / kSlab;
  const unsigned long long wave = (unsigned long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const long long n = (long long)(wave / slabs);
  if (n >= rows) return;
  const long long id = id_at(ids, id_bits, n);
  const bool known = id >= 0 && id < vocab;
  const T* in = weight + (known ? id : 0) * ld;
  T* to = out + n * dim;
  const bool wide = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(to)) & 15) == 0;
  const int d = (int)(wave % slabs) * kSlab + (threadIdx.x & 63) * Vec<T>::kN;
  if (d >= dim) return;
  Vec<T> v;
  v.load(in + d, dim - d, wide);
  for (int e = 0; e < Vec<T>::kN; ++e)
    v.x[e] = known ? static_cast<T>(static_cast<float>(v.x[e]) * scale) : static_cast<T>(__builtin_nanf(""));
  v.store(to + d, dim - d, wide);
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

// The sums.  Rows of the vocabulary with at most kPiece tokens ("light") are summed and written by one wave; a
// common token's list ("heavy") is cut at multiples of kPiece positions of the sorted list, each piece is summed by one wave
// to float32 partial sums, and embed_join_kernel adds them up in order.  A piece holds parts of at most two heavy rows:
// slot 0 is the one at its first position, slot 1 one that begins behind it.
constexpr int kPiece = 64, kRowsPerWave = 8, kJoinWaves = 16;

struct SumArgs {
  const int* start;
  const int* order;
  const void* ids;
  int id_bits;
  const void* grad;
  long long ld;
  long long rows;
  int dim, vocab;
  float scale;
  void* out;
  int out_f32;
  float* partial;         // (pieces, 2, dim)
};

template <typename T>
__device__ inline void add_rows(float* sum, const int* order, int first, int last, const T* grad, long long ld, int d,
                                int left, bool wide) {
  constexpr int kN = Vec<T>::kN, kDeep = 8;
  int i = first;
  for (; i + kDeep <= last; i += kDeep) {       // kDeep rows in flight
    Vec<T> x[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) x[k].load(grad + (long long)order[i + k] * ld + d, left, wide);
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
#pragma unroll
      for (int e = 0; e < kN; ++e) sum[e] += static_cast<float>(x[k].x[e]);
  }
  for (; i < last; ++i) {
    Vec<T> x;
    x.load(grad + (long long)order[i] * ld + d, left, wide);
#pragma unroll
    for (int e = 0; e < kN; ++e) sum[e] += static_cast<float>(x.x[e]);
  }
}

template <typename T>
__device__ inline void write_sum(const float* sum, const SumArgs& p, int v, int d) {
  constexpr int kN = Vec<T>::kN;
  const long long at = (long long)v * p.dim + d;
  if (p.out_f32) {
    float* to = static_cast<float*>(p.out) + at;
    const bool wide = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
#pragma unroll
    for (int h = 0; h < kN; h += 4) {
      Vec<float> x;
      for (int e = 0; e < 4; ++e) x.x[e] = sum[h + e] * p.scale;
      if (d + h < p.dim) x.store(to + h, p.dim - d - h, wide);
    }
  } else {
    Vec<T> x;
#pragma unroll
    for (int e = 0; e < kN; ++e) x.x[e] = static_cast<T>(sum[e] * p.scale);
    T* to = static_cast<T*>(p.out) + at;
    x.store(to, p.dim - d, (reinterpret_cast<uintptr_t>(to) & 15) == 0);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs p, int piece_blocks) {
  constexpr int kN = Vec<T>::kN, kSlab = 64 * kN;
  const int lane = threadIdx.x & 63;
  const T* grad = static_cast<const T*>(p.grad);
  const bool wide = (reinterpret_cast<uintptr_t>(grad) & 15) == 0 && (p.ld * (long long)sizeof(T)) % 16 == 0;
  if ((int)blockIdx.x < piece_blocks) {
    const int slabs = (p.dim + kSlab - 1) / kSlab;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int piece = wave / slabs, d = (wave % slabs) * kSlab + lane * kN;
    const int total = p.start[p.vocab], i0 = piece * kPiece, i1 = min(i0 + kPiece, total);
    if (i0 >= total || d >= p.dim) return;
    const int v0 = (int)id_at(p.ids, p.id_bits, p.order[i0]), v1 = (int)id_at(p.ids, p.id_bits, p.order[i1 - 1]);
    for (int slot = 0; slot < 2; ++slot) {
      const int v = slot ? v1 : v0;
      if (slot && v1 == v0) break;
      const int first = p.start[v], last = p.start[v + 1];
      if (last - first <= kPiece) continue;
      float sum[kN];
      for (int e = 0; e < kN; ++e) sum[e] = 0.f;
      add_rows<T>(sum, p.order, max(first, i0), min(last, i1), grad, p.ld, d, p.dim - d, wide);
      float* to = p.partial + ((long long)piece * 2 + slot) * p.dim + d;
      for (int e = 0; e < kN && d + e < p.dim; ++e) to[e] = sum[e];
    }
    return;
  }
  const int v0 = __builtin_amdgcn_readfirstlane(((blockIdx.x - piece_blocks) * 4 + (threadIdx.x >> 6)) * kRowsPerWave);
  if (v0 >= p.vocab) return;
  const int bounds = lane <= kRowsPerWave ? p.start[min(v0 + lane, p.vocab)] : 0;
  for (int k = 0; k < kRowsPerWave && v0 + k < p.vocab; ++k) {
    const int first = __builtin_amdgcn_readlane(bounds, k), last = __builtin_amdgcn_readlane(bounds, k + 1);
    if (last - first > kPiece) continue;
    for (int d = lane * kN; d < p.dim; d += kSlab) {
      float sum[kN];
      for (int e = 0; e < kN; ++e) sum[e] = 0.f;
      add_rows<T>(sum, p.order, first, last, grad, p.ld, d, p.dim - d, wide);
      write_sum<T>(sum, p, v0 + k, d);
    }
  }
}

// One block per piece (in which a heavy row may begin) and slab; the row's partial sums go to the waves in turns of
// contiguous runs, then the waves' sums are added in order.
template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(const SumArgs p) {
  constexpr int kN = Vec<T>::kN, kSlab = 64 * kN;
  __shared__ float sums[kJoinWaves][kSlab];
  const int slabs = (p.dim + kSlab - 1) / kSlab;
  const int piece = blockIdx.x / slabs, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = (blockIdx.x % slabs) * kSlab + lane * kN;
  const int total = p.start[p.vocab], i0 = piece * kPiece, i1 = min(i0 + kPiece, total);
  if (i0 >= total) return;
  const int v = (int)id_at(p.ids, p.id_bits, p.order[i1 - 1]);
  const int first = p.start[v], last = p.start[v + 1];
  if (last - first <= kPiece || first < i0) return;
  const int pieces = (last - 1) / kPiece - piece + 1;
  const int each = (pieces + kJoinWaves - 1) / kJoinWaves;
  float sum[kN];
  for (int e = 0; e < kN; ++e) sum[e] = 0.f;
  if (d < p.dim)
    for (int i = wave * each; i < min((wave + 1) * each, pieces); ++i) {
      const float* from = p.partial + ((long long)(piece + i) * 2 + (i == 0 && first > i0)) * p.dim + d;
      for (int e = 0; e < kN; ++e) sum[e] += d + e < p.dim ? from[e] : 0.f;
    }
  for (int e = 0; e < kN; ++e) sums[wave][lane * kN + e] = sum[e];
  __syncthreads();
  if (wave > 0 || d >= p.dim) return;
  for (int w = 1; w < kJoinWaves; ++w)
    for (int e = 0; e < kN; ++e) sum[e] += sums[w][lane * kN + e];
  write_sum<T>(sum, p, v, d);
}

int64_t index_bytes(const wfe_embedding_desc& d) { return 4 * ((int64_t)d.vocab + 1 + d.rows + 15) / 64 * 64 + 64; }

template <typename T>
hipError_t embed(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out, hipStream_t stream) {
  const int64_t slabs = (d.dim + 64 * Vec<T>::kN - 1) / (64 * Vec<T>::kN);
  embed_kernel<T><<<dim3((unsigned)((d.rows * slabs + 3) / 4)), dim3(256), 0, stream>>>(
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
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  SumArgs p{};
  p.start = start;
  p.order = order;
  p.ids = ids;
  p.id_bits = d.id_bits;
  p.grad = grad;
  p.ld = d.grad_stride;
  p.rows = d.rows;
  p.dim = d.dim;
  p.vocab = d.vocab;
  p.scale = d.scale;
  p.out = grad_weight;
  p.out_f32 = d.grad_weight_dtype == WFE_F32;
  p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + index_bytes(d));
  // no row can be heavy with kPiece tokens or fewer
  const int64_t slabs = (d.dim + 64 * Vec<T>::kN - 1) / (64 * Vec<T>::kN);
  const int64_t pieces = d.rows > kPiece ? (d.rows + kPiece - 1) / kPiece : 0;
  const int64_t piece_blocks = (pieces * slabs + 3) / 4;
  const int64_t row_blocks = (d.vocab + 4 * kRowsPerWave - 1) / (4 * kRowsPerWave);
  embed_sum_kernel<T><<<dim3((unsigned)(piece_blocks + row_blocks)), dim3(256), 0, stream>>>(p, (int)piece_blocks);
  e = hipGetLastError();
  if (e != hipSuccess || pieces == 0) return e;
  embed_join_kernel<T><<<dim3((unsigned)(pieces * slabs)), dim3(kJoinWaves * 64), 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace

int64_t embedding_workspace_bytes(const wfe_embedding_desc& d) {
  return index_bytes(d) + (d.rows > kPiece ? (d.rows + kPiece - 1) / kPiece * 2 * (int64_t)d.dim * 4 : 0);
}

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
