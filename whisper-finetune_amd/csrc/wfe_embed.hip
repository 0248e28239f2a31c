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

__device__ inline long long id_at(const void* ids, int bits, int n) {
  return bits == 64 ? static_cast<const long long*>(ids)[n] : static_cast<const int*>(ids)[n];
}

// 16 bytes of T.  WIDE: every row starts on 16 bytes and is whole multiples of them (the host knows); otherwise value
// by value, with a ragged end.  The two are kernels of their own: what a wave executes for the first time comes from the
// L2 line by line, and a gather this short is bound by that (768 rows of 1280: 16 us with both ways and a 64-bit division
// in one kernel, 2.9 so).
template <typename T, bool WIDE>
struct Vec {
  static constexpr int kN = 16 / (int)sizeof(T);
  T x[kN];
  __device__ void load(const T* p, int left) {
    if constexpr (WIDE) __builtin_memcpy(x, __builtin_assume_aligned(p, 16), 16);
    else
#pragma unroll
      for (int e = 0; e < kN; ++e) x[e] = e < left ? p[e] : static_cast<T>(0.f);
  }
  __device__ void store(T* p, int left) const {
    if constexpr (WIDE) __builtin_memcpy(__builtin_assume_aligned(p, 16), x, 16);
    else
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < left) p[e] = x[e];
  }
};

// A wave takes kTokens tokens' share of one slab of columns (blockIdx.y), all their loads in flight.  Columns of 1280
// bfloat16: 16 tokens 2.4 us, 768 2.9, 28672 (147 MB, out of the caches in part) 26; one token to a wave 3.3, 5.4 and 29.
constexpr int kTokens = 4;

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void embed_kernel(const void* ids, int id_bits, int rows, const T* weight,
                                                    long long ld, int dim, int vocab, float scale, T* out) {
  using V = Vec<T, WIDE>;
  const int first = __builtin_amdgcn_readfirstlane((blockIdx.x * 4 + (threadIdx.x >> 6)) * kTokens);
  const int d = (blockIdx.y * 64 + (threadIdx.x & 63)) * V::kN;
  if (d >= dim) return;
  V v[kTokens];
  bool known[kTokens];
#pragma unroll
  for (int k = 0; k < kTokens; ++k) {
    const int n = first + k;
    const long long id = n < rows ? id_at(ids, id_bits, n) : -1;
    known[k] = id >= 0 && id < vocab;
    v[k].load(weight + (known[k] ? id : 0) * ld + d, dim - d);
  }
#pragma unroll
  for (int k = 0; k < kTokens; ++k) {
    if (first + k >= rows) break;
#pragma unroll
    for (int e = 0; e < V::kN; ++e)
      v[k].x[e] = known[k] ? static_cast<T>(static_cast<float>(v[k].x[e]) * scale) : static_cast<T>(__builtin_nanf(""));
    v[k].store(out + (long long)(first + k) * dim + d, dim - d);
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------
// Sorting by token, stable, in one launch: a block owns kBins rows of the vocabulary and reads all ids itself, once
// to count (tokens below its rows give the place where its part of the sorted list starts) and once to place.  No
// block needs another's result.
constexpr int kBins = 256, kSortWaves = 16, kSortDeep = 8;
// A wave keeps the tokens it counted, row and number in one word, so that placing them needs no second read of the ids;
// a wave that meets more than this reads them again.
constexpr int kKeep = 448;
static_assert(kBins <= 256, "row in 8 bits, number (below 2^24) in 24");

__global__ __launch_bounds__(kSortWaves * 64) void embed_sort_kernel(const void* ids, int id_bits, int rows, int vocab,
                                                                     long long padding, int* start, int* order) {
  __shared__ int place[kSortWaves][kBins];     // counts, then next places, per wave and row
  __shared__ int below_of[kSortWaves], sum_of[kBins / 64];
  __shared__ unsigned keep[kSortWaves][kKeep];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int v0 = blockIdx.x * kBins;
  for (int i = threadIdx.x; i < kSortWaves * kBins; i += kSortWaves * 64) (&place[0][0])[i] = 0;
  __syncthreads();
  // wave w takes a contiguous run of the tokens; kSortDeep loads in flight.  -> row within the block's (kBins: none),
  // -1: below
  const int each = ((rows + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int first = wave * each, last = min(first + each, rows);
  auto bins_of = [&](int n0, int* bin) {
    long long id[kSortDeep];
#pragma unroll
    for (int k = 0; k < kSortDeep; ++k) id[k] = n0 + 64 * k + lane < last ? id_at(ids, id_bits, n0 + 64 * k + lane) : -1;
#pragma unroll
    for (int k = 0; k < kSortDeep; ++k) {
      const bool counted = id[k] >= 0 && id[k] < min((long long)vocab, (long long)v0 + kBins) && id[k] != padding;
      bin[k] = !counted ? kBins : id[k] < v0 ? -1 : (int)(id[k] - v0);
    }
  };
  int below = 0, kept = 0, bin[kSortDeep];
  for (int n0 = first; n0 < last; n0 += 64 * kSortDeep) {
    bins_of(n0, bin);
#pragma unroll
    for (int k = 0; k < kSortDeep; ++k) {
      const bool here = bin[k] >= 0 && bin[k] < kBins;
      below += bin[k] < 0;
      const unsigned long long mask = __ballot(here);
      if (mask == 0) continue;
      const int at = kept + __popcll(mask & ((1ull << lane) - 1));
      if (here) {
        atomicAdd(&place[wave][bin[k]], 1);
        if (at < kKeep) keep[wave][at] = (unsigned)bin[k] << 24 | (unsigned)(n0 + 64 * k + lane);
      }
      kept += __popcll(mask);
    }
  }
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_of[wave] = below;
  __syncthreads();
  int total = 0, upto = 0;
  if (threadIdx.x < kBins) {
    for (int w = 0; w < kSortWaves; ++w) total += place[w][threadIdx.x];
    upto = total;                              // inclusive sums within the wave
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 63) sum_of[wave] = upto;
  }
  __syncthreads();
  if (threadIdx.x < kBins) {
    int at = upto - total;
    for (int w = 0; w < kSortWaves; ++w) at += below_of[w];
    for (int w = 0; w < wave; ++w) at += sum_of[w];
    const int v = v0 + threadIdx.x;
    if (v < vocab) start[v] = at;
    if (v == vocab - 1) start[vocab] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = place[w][threadIdx.x];
      place[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  // 64 tokens at a time to their places, in order
  auto put = [&](bool here, int row, int n) {
    unsigned long long left = __ballot(here);
    while (left) {                             // one step per distinct token of the 64
      const int b = __builtin_amdgcn_readlane(row, __ffsll(left) - 1);
      const unsigned long long same = __ballot(here && row == b);
      const int at = place[wave][b];
      if (here && row == b) order[at + __popcll(same & ((1ull << lane) - 1))] = n;
      if (lane == 0) place[wave][b] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the other lanes read it the next time
      left &= ~same;
    }
  };
  if (kept <= kKeep) {
    for (int i = lane; i - lane < kept; i += 64) {
      const unsigned x = i < kept ? keep[wave][i] : 0;
      put(i < kept, (int)(x >> 24), (int)(x & 0xffffff));
    }
  } else {
    for (int n0 = first; n0 < last; n0 += 64 * kSortDeep) {
      bins_of(n0, bin);
#pragma unroll 1
      for (int k = 0; k < kSortDeep; ++k) put(bin[k] >= 0 && bin[k] < kBins, bin[k], n0 + 64 * k + lane);
    }
  }
}

// The sums.  A wave takes a slab of columns of kRowsPerWave rows of the vocabulary (a wave for whole rows: 26 us instead
// of 19 for 768 tokens, 53 instead of 42 for 64 x 448).  Rows with at most kPiece tokens ("light") it sums and writes; a
// common token's list ("heavy") is cut at multiples of kPiece positions of the sorted list, each piece is summed by one wave
// to float32 partial sums, and embed_join_kernel adds them up in order.  A piece holds parts of at most two heavy rows:
// slot 0 is the one at its first position, slot 1 one that begins behind it.
// kPiece: a wave sums its tokens one after the other, so the longest list is the tail of the launch (64 x 448 tokens
// of text: 64 -> 118 us, 32 -> 80, 16 -> 67).
constexpr int kPiece = 16, kRowsPerWave = 8, kJoinWaves = 16, kJoinPieces = 8;

struct SumArgs {
  const int* start;
  const int* order;
  const void* ids;
  int id_bits;
  const void* grad;
  long long ld;
  int dim, vocab, pieces;
  float scale;
  void* out;
  int out_f32;
  float* partial;         // (pieces, 2, dim)
};

// Adds `count` (at most 64) rows of grad, whose numbers lanes 0.. hold in `mine`, in order.
template <typename T, bool WIDE>
__device__ inline void add_rows(float* sum, int mine, int count, const T* grad, long long ld, int d, int left) {
  constexpr int kN = Vec<T, WIDE>::kN, kDeep = WIDE ? 8 : 1;
  for (int i = 0; i < count; i += kDeep) {       // kDeep rows in flight
    Vec<T, WIDE> x[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (i + k < count) x[k].load(grad + (long long)__builtin_amdgcn_readlane(mine, i + k) * ld + d, left);
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (i + k < count)
#pragma unroll
        for (int e = 0; e < kN; ++e) sum[e] += static_cast<float>(x[k].x[e]);
  }
}

template <typename T, bool WIDE>
__device__ inline void write_sum(const float* sum, const SumArgs& p, int v, int d) {
  constexpr int kN = Vec<T, WIDE>::kN;
  const long long at = (long long)v * p.dim + d;
  if (p.out_f32) {
#pragma unroll
    for (int h = 0; h < kN; h += 4) {
      Vec<float, WIDE> x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x.x[e] = sum[h + e] * p.scale;
      x.store(static_cast<float*>(p.out) + at + h, p.dim - d - h);
    }
  } else {
    Vec<T, WIDE> x;
#pragma unroll
    for (int e = 0; e < kN; ++e) x.x[e] = static_cast<T>(sum[e] * p.scale);
    x.store(static_cast<T*>(p.out) + at, p.dim - d);
  }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void embed_sum_kernel(const SumArgs p, int piece_blocks, int slabs) {
  constexpr int kN = Vec<T, WIDE>::kN, kSlab = 64 * kN;
  const int lane = threadIdx.x & 63;
  const T* grad = static_cast<const T*>(p.grad);
  if ((int)blockIdx.x < piece_blocks) {
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int piece = wave / slabs, d = (wave % slabs) * kSlab + lane * kN;
    const int total = p.start[p.vocab], i0 = piece * kPiece, i1 = min(i0 + kPiece, total);
    if (i0 >= total) return;
    const int v0 = (int)id_at(p.ids, p.id_bits, p.order[i0]), v1 = (int)id_at(p.ids, p.id_bits, p.order[i1 - 1]);
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
      const int v = slot ? v1 : v0;
      if (slot && v1 == v0) break;
      const int first = p.start[v], last = p.start[v + 1];
      if (last - first <= kPiece) continue;
      float sum[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) sum[e] = 0.f;
      const int from = max(first, i0), count = min(last, i1) - from;
      const int mine = lane < count ? p.order[from + lane] : 0;
      if (d < p.dim) add_rows<T, WIDE>(sum, mine, count, grad, p.ld, d, p.dim - d);
      float* to = p.partial + ((long long)piece * 2 + slot) * p.dim + d;
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (d + e < p.dim) to[e] = sum[e];
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((blockIdx.x - piece_blocks) * 4 + (threadIdx.x >> 6));
  const int v0 = wave / slabs * kRowsPerWave, d = (wave % slabs) * kSlab + lane * kN;
  if (v0 >= p.vocab) return;
  const int rows = min(kRowsPerWave, p.vocab - v0);
  const int bounds = lane <= kRowsPerWave ? p.start[min(v0 + lane, p.vocab)] : 0;
  const int length = __shfl(bounds, lane + 1) - bounds;
  // the many rows without tokens first, the rest while those stores drain
  float zero[kN];
#pragma unroll
  for (int e = 0; e < kN; ++e) zero[e] = 0.f;
#pragma unroll 1
  for (int k = 0; k < rows; ++k)
    if (__builtin_amdgcn_readlane(length, k) == 0)
      if (d < p.dim) write_sum<T, WIDE>(zero, p, v0 + k, d);
  unsigned long long light = __ballot(lane < rows && length > 0 && length <= kPiece);
  while (light) {
    const int k = __ffsll(light) - 1;
    light &= light - 1;
    const int first = __builtin_amdgcn_readlane(bounds, k), count = __builtin_amdgcn_readlane(length, k);
    const int mine = lane < count ? p.order[first + lane] : 0;
    if (d < p.dim) {
      float sum[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) sum[e] = 0.f;
      add_rows<T, WIDE>(sum, mine, count, grad, p.ld, d, p.dim - d);
      write_sum<T, WIDE>(sum, p, v0 + k, d);
    }
  }
}

// A block looks through kJoinPieces pieces for heavy rows that begin there (blockIdx.y: the slab); such a row's
// partial sums go to the waves in contiguous runs, then the waves' sums are added in order.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(const SumArgs p) {
  constexpr int kN = Vec<T, WIDE>::kN, kSlab = 64 * kN;
  __shared__ float sums[kJoinWaves][kSlab];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int d = blockIdx.y * kSlab + lane * kN;
  const int total = p.start[p.vocab];
  const int mine = blockIdx.x * kJoinPieces + lane, i0 = mine * kPiece, i1 = min(i0 + kPiece, total);
  int v = 0, first = 0, last = 0;
  if (lane < kJoinPieces && i0 < total) {
    v = (int)id_at(p.ids, p.id_bits, p.order[i1 - 1]);
    first = p.start[v];
    last = p.start[v + 1];
  }
  unsigned long long starts = __ballot(last - first > kPiece && first >= i0);
  while (starts) {                             // the same in every wave
    const int k = __ffsll(starts) - 1;
    starts &= starts - 1;
    const int piece = blockIdx.x * kJoinPieces + k;
    const int from = __builtin_amdgcn_readlane(first, k), to = __builtin_amdgcn_readlane(last, k);
    const int pieces = (to - 1) / kPiece - piece + 1;
    const int each = (pieces + kJoinWaves - 1) / kJoinWaves;
    const int begin = wave * each, end = min(begin + each, pieces);
    float sum[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) sum[e] = 0.f;
    if (d < p.dim)
#pragma unroll 4
      for (int i = begin; i < end; ++i) {
        const float* at = p.partial + ((long long)(piece + i) * 2 + (i == 0 && from > piece * kPiece)) * p.dim + d;
#pragma unroll
        for (int e = 0; e < kN; ++e) sum[e] += WIDE || d + e < p.dim ? at[e] : 0.f;
      }
#pragma unroll
    for (int e = 0; e < kN; ++e) sums[wave][e * 64 + lane] = sum[e];
    __syncthreads();
    if (wave == 0 && d < p.dim) {
#pragma unroll 1
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int e = 0; e < kN; ++e) sum[e] += sums[w][e * 64 + lane];
      write_sum<T, WIDE>(sum, p, __builtin_amdgcn_readlane(v, k), d);
    }
    __syncthreads();
  }
}

int64_t index_bytes(const wfe_embedding_desc& d) { return (4 * ((int64_t)d.vocab + 1 + d.rows) + 63) / 64 * 64; }
int64_t pieces_of(const wfe_embedding_desc& d) {              // no row can be heavy with kPiece tokens or fewer
  return d.rows > kPiece ? (d.rows + kPiece - 1) / kPiece : 0;
}

// rows of `stride` elements from p on start on 16 bytes and are whole multiples of them
template <typename T>
bool wide(const void* p, int64_t stride, int dim) {
  constexpr int kN = 16 / (int)sizeof(T);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kN == 0 && dim % kN == 0;
}

template <typename T, bool WIDE>
hipError_t embed_as(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out, hipStream_t stream) {
  constexpr int kSlab = 64 * (16 / (int)sizeof(T));
  const unsigned slabs = (d.dim + kSlab - 1) / kSlab;
  embed_kernel<T, WIDE><<<dim3((unsigned)((d.rows + 4 * kTokens - 1) / (4 * kTokens)), slabs), dim3(256), 0, stream>>>(
      ids, d.id_bits, (int)d.rows, static_cast<const T*>(weight), d.weight_stride, d.dim, d.vocab, d.scale,
      static_cast<T*>(out));
  return hipGetLastError();
}

template <typename T>
hipError_t embed(const wfe_embedding_desc& d, const void* ids, const void* weight, void* out, hipStream_t stream) {
  return wide<T>(weight, d.weight_stride, d.dim) && wide<T>(out, d.dim, d.dim)
             ? embed_as<T, true>(d, ids, weight, out, stream)
             : embed_as<T, false>(d, ids, weight, out, stream);
}

// Blocks of the sums' launch: a wave per piece and slab, then a wave per kRowsPerWave rows of the vocabulary and slab
struct SumGrid {
  int64_t pieces, rows;
};
SumGrid sum_grid(int64_t pieces, int64_t vocab, int64_t slabs) {
  return {(pieces * slabs + 3) / 4, ((vocab + kRowsPerWave - 1) / kRowsPerWave * slabs + 3) / 4};
}

template <typename T, bool WIDE>
hipError_t sums_as(const SumArgs& p, hipStream_t stream) {
  constexpr int kSlab = 64 * (16 / (int)sizeof(T));
  const unsigned slabs = (p.dim + kSlab - 1) / kSlab;
  const SumGrid grid = sum_grid(p.pieces, p.vocab, slabs);
  embed_sum_kernel<T, WIDE><<<dim3((unsigned)(grid.pieces + grid.rows)), dim3(256), 0, stream>>>(
      p, (int)grid.pieces, (int)slabs);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.pieces == 0) return e;
  embed_join_kernel<T, WIDE><<<dim3((p.pieces + kJoinPieces - 1) / kJoinPieces, slabs), dim3(kJoinWaves * 64), 0,
                               stream>>>(p);
  return hipGetLastError();
}

template <typename T>
hipError_t embed_backward(const wfe_embedding_desc& d, const void* ids, const void* grad, void* grad_weight,
                          void* workspace, hipStream_t stream) {
  int* start = static_cast<int*>(workspace);
  int* order = start + d.vocab + 1;
  embed_sort_kernel<<<dim3((unsigned)((d.vocab + kBins - 1) / kBins)), dim3(kSortWaves * 64), 0, stream>>>(
      ids, d.id_bits, (int)d.rows, d.vocab, d.padding_idx, start, order);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  SumArgs p{};
  p.start = start;
  p.order = order;
  p.ids = ids;
  p.id_bits = d.id_bits;
  p.grad = grad;
  p.ld = d.grad_stride;
  p.dim = d.dim;
  p.vocab = d.vocab;
  p.pieces = (int)pieces_of(d);
  p.scale = d.scale;
  p.out = grad_weight;
  p.out_f32 = d.grad_weight_dtype == WFE_F32;
  p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + index_bytes(d));
  return wide<T>(grad, d.grad_stride, d.dim) && wide<T>(grad_weight, d.dim, d.dim) ? sums_as<T, true>(p, stream)
                                                                                  : sums_as<T, false>(p, stream);
}

}  // namespace

int64_t embedding_workspace_bytes(const wfe_embedding_desc& d) {
  return index_bytes(d) + pieces_of(d) * 2 * (int64_t)d.dim * 4;
}

bool embedding_backward_fits(const wfe_embedding_desc& d) {
  const int64_t slab = 64 * (d.dtype == WFE_F32 ? 4 : 8);
  const SumGrid grid = sum_grid(pieces_of(d), d.vocab, (d.dim + slab - 1) / slab);
  return (grid.pieces + grid.rows) * 256 < (int64_t)1 << 32;
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
