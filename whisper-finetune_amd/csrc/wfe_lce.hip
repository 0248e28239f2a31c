// wfe_lce.hip -- softmax cross entropy over the vocabulary without keeping the logits, and its gradients, for gfx950.
//
//   z[n][v] = h_n . W_v          lse_n = log sum_v exp z[n][v]          loss_n = lse_n - z[n][y_n]
//   d[n][v] = exp(z[n][v] - lse_n) - [v == y_n]
//   dh_n = g_n sum_v d[n][v] W_v          dW_v = sum_n g_n d[n][v] h_n          (g_n: upstream share of row n)
//
// Rows whose label is ignore_index are dropped first: lce_pack_kernel copies the kept ones together (and pads
// them with zeros to whole tiles), every product after it runs over the kept rows only, whose number stays on the
// device.  All four products are one tile kernel that multiplies 16-byte K fragments out of LDS:
//   STATS  z tiles, reduced in registers to a maximum and a sum of exponentials per row and vocabulary tile
//   PROB   z tiles again, written as d for a piece of the vocabulary
//   DHID   dh += d W over that piece, in float32
//   DWEI   the piece's rows of dW, each written once
// Recomputing z costs one product more than keeping (rows, vocab) logits would.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "wfe_decoder.h"

namespace wfe {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of K of one row (or column) per lane: 8 values of 2 bytes or 4 of 4
union Frag {
  i32x4 i;
  bf16x8 b;
  f16x8 h;
  f32x4 f;
  s16x4 s[2];
};

template <typename T> struct Elem;
template <> struct Elem<__bf16> {
  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
  }
  static constexpr float kScale = 1.0f;
};
template <> struct Elem<_Float16> {
  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
  }
  // d is in [-1, 1]: stored times 2^14 so that small probabilities stay clear of the subnormals
  static constexpr float kScale = 16384.0f;
};
template <> struct Elem<float> {
  // lane group g holds k = 4 g .. 4 g + 3 of a 16-deep step; the i-th instruction takes every group's i-th value,
  // the same on both sides
  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[i], b.f[i], c, 0, 0, 0);
    return c;
  }
  static constexpr float kScale = 1.0f;
};

constexpr int kKBytes = 128;                               // depth of a K tile in bytes
template <typename T> constexpr int kKElems = kKBytes / (int)sizeof(T);
constexpr float kLog2e = 1.44269504088896340736f;

__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// ---- operands -------------------------------------------------------------------------------------------
// An operand tile in LDS is either a rows x 128 bytes of K ("along": K contiguous in memory) or K rows x columns
// ("across": K strided in memory, transposed by the read).  16-byte chunks of a row are permuted by an exclusive or
// so that the lanes of a fragment read meet different banks:
//   along           chunk ^ (row & 7)
//   across, 2 byte  pairs of chunks (a transposing read takes 32 bytes of each of 4 rows); 8 rows 0..3, 8..11 apart
//   across, 4 byte  groups of four chunks; 4 rows 4 apart
template <typename T, bool ACROSS>
__device__ inline int swizzle(int row) {
  if constexpr (!ACROSS) return row & 7;
  else if constexpr (sizeof(T) == 2) return ((row & 3) | ((row >> 1) & 4)) << 1;
  else return ((row >> 2) & 3) << 2;
}

// Loads tiles of N rows (or columns) with NW waves, 1024 bytes per wave and instruction straight into LDS.
template <typename T, bool ACROSS, int N, int NW>
struct Loader {
  static constexpr int kRowBytes = ACROSS ? N * (int)sizeof(T) : kKBytes;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = N * kKBytes;
  static constexpr int kInstrs = kTileBytes / 1024;
  static constexpr int kPer = (kInstrs + NW - 1) / NW;
  const char* base;
  long long step;                 // bytes from one K tile to the next
  long long ld;                   // bytes
  int k_left;                     // across: K rows that exist from the current tile on
  unsigned off[kPer];
  int wave, lane;

  // first: row or column of the tile; limit: rows (along) or columns (across, a multiple of 16 bytes) that exist;
  // k0 / k_rows: the first K and (across) the K rows that exist
  __device__ void init(const T* p, long long ld_elems, int first, int limit, long long k0, long long k_rows, int w,
                       int l) {
    wave = w;
    lane = l;
    ld = ld_elems * (long long)sizeof(T);
    if constexpr (ACROSS) {
      base = reinterpret_cast<const char*>(p) + k0 * ld + (long long)first * sizeof(T);
      step = ld * kKElems<T>;
      k_left = (int)(k_rows - k0);
    } else {
      base = reinterpret_cast<const char*>(p) + (long long)first * ld + k0 * (long long)sizeof(T);
      step = kKBytes;
      k_left = 0;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = (i * NW + wave) * 64 + lane;
      int row = id / kChunks;
      int c = (id % kChunks) ^ swizzle<T, ACROSS>(row);
      if constexpr (ACROSS) {
        const int most = (int)((limit - first) * (int)sizeof(T) / 16) - 1;
        c = c < most ? c : most;          // columns past the end: any that exist, their products are not stored
      } else {
        const int most = limit - first - 1;
        row = row < most ? row : most;
      }
      off[i] = (unsigned)(row * ld) + (unsigned)c * 16u;
    }
  }
  __device__ void issue(char* lds) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int instr = i * NW + wave;
      if (kInstrs % NW != 0 && instr >= kInstrs) break;
      unsigned o = off[i];
      if constexpr (ACROSS) {
        if (k_left < kKElems<T>) {        // K rows past the end: the last one (its factors on the other side are 0)
          const int row = (instr * 64 + lane) / kChunks;
          if (row >= k_left) o -= (unsigned)((row - k_left + 1) * ld);
        }
      }
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(base + o),
          (__attribute__((address_space(3))) void*)(lds + instr * 1024), 16, 0, 0);
    }
    base += step;
    if constexpr (ACROSS) k_left -= kKElems<T>;
  }
};

// Fragment of 16 rows (or columns) from m0 on, K step ks (0 or 1) of the tile
template <typename T, bool ACROSS, int N>
__device__ inline Frag read_frag(const char* lds, int m0, int ks, int lane) {
  Frag r;
  if constexpr (!ACROSS) {
    const int row = m0 + (lane & 15);
    const int c = (ks * 4 + (lane >> 4)) ^ (row & 7);
    r.i = *reinterpret_cast<const i32x4*>(lds + row * kKBytes + c * 16);
  } else if constexpr (sizeof(T) == 2) {
    const int g = lane >> 4, j = (lane & 15) >> 2, q = lane & 3;
    const int chunk = m0 / 8 + (q >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = ks * 32 + 8 * g + 4 * h + j;
      r.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
          lds + row * (N * 2) + (chunk ^ swizzle<T, true>(row)) * 16 + (q & 1) * 8));
    }
  } else {
    const int col = m0 + (lane & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = ks * 16 + 4 * (lane >> 4) + i;
      r.f[i] = *reinterpret_cast<const float*>(lds + row * (N * 4) + ((col / 4) ^ swizzle<T, true>(row)) * 16 +
                                               (col & 3) * 4);
    }
  }
  return r;
}

// ---- the tile kernel ----------------------------------------------------------------------------------------
enum Mode { kStats, kProb, kDhid, kDwei };

struct TileArgs {
  const void* hidden;     // packed rows (row_pad, dim_pad); DWEI: the weighted ones
  const void* weight;     // (vocab, dim_pad) from row v0 on, weight_ld elements apart
  void* prob;             // d of the piece, (row_pad, prob_ld)
  long long weight_ld, prob_ld;
  int dim, dim_pad, v0, piece, vocab;      // the piece holds vocabulary rows v0 .. v0 + piece - 1
  long long row_pad;
  const int* head;        // [0] kept rows
  const int* label;
  float* zlab;
  const float* lse;
  float2* partial;        // STATS: (vocabulary tiles, row_pad) maximum and sum
  float* acc;             // DHID: (splits, row_pad, dim_pad)
  int splits, first;
  void* grad_weight;      // DWEI: (vocab, dim)
  int grad_f32;
  const float* factor;    // DWEI
  int a_tiles, b_tiles;   // tiles along the two axes; of rows: the most there can be
};

template <typename T, int MODE, int BA, int BB, int WA, int WB>
__global__ __launch_bounds__(WA * WB * 64) void lce_tile_kernel(const TileArgs p) {
  constexpr bool kAAcross = MODE == kDhid || MODE == kDwei;
  constexpr bool kBAcross = MODE == kDwei;
  constexpr int NW = WA * WB, TA = BA / WA, TB = BB / WB, FA = TA / 16, FB = TB / 16;
  constexpr int kStage = (BA + BB) * kKBytes;
  constexpr int KE = kKElems<T>;
  extern __shared__ __align__(1024) char smem[];

  const int count = p.head[0];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;

  // Which tile: blocks go to the 8 XCDs in turn; each XCD takes a contiguous run of the tiles, ordered so that a few
  // tiles of one axis are reused from its L2 while the other axis passes.
  const int a_tiles = p.a_tiles;
  const int b_tiles = MODE == kDwei ? p.b_tiles : (count + BB - 1) / BB;
  const int plane = a_tiles * b_tiles;
  const int total = plane * (MODE == kDhid ? p.splits : 1);
  const int per = (total + 7) / 8;
  const int slot = blockIdx.x >> 3;
  int id = (blockIdx.x & 7) * per + slot;
  if (slot >= per || id >= total) return;
  const int split = id / plane;
  id -= split * plane;
  constexpr int kGroup = 8;
  const int group = id / (kGroup * a_tiles);
  const int rest = id - group * kGroup * a_tiles;
  const int in_group = min(kGroup, b_tiles - group * kGroup);
  const int ta = rest / in_group, tb = group * kGroup + rest % in_group;
  const int a0 = ta * BA, b0 = tb * BB;

  // K range, in tiles
  int k_first = 0, k_tiles;
  if constexpr (MODE == kStats || MODE == kProb) k_tiles = p.dim_pad / KE;
  else if constexpr (MODE == kDwei) k_tiles = (count + KE - 1) / KE;
  else {
    const int all = (p.piece + KE - 1) / KE;
    const int each = (all + p.splits - 1) / p.splits;
    k_first = split * each;
    k_tiles = min(each, all - k_first);
    if (k_tiles < 0) k_tiles = 0;
  }

  Loader<T, kAAcross, BA, NW> la;
  Loader<T, kBAcross, BB, NW> lb;
  const T* hidden = static_cast<const T*>(p.hidden);
  const T* weight = static_cast<const T*>(p.weight);
  const T* prob = static_cast<const T*>(p.prob);
  if constexpr (MODE == kStats || MODE == kProb) {
    la.init(weight, p.weight_ld, a0, p.piece, 0, 0, wave, lane);
    lb.init(hidden, p.dim_pad, b0, b0 + BB, 0, 0, wave, lane);
  } else if constexpr (MODE == kDhid) {
    la.init(weight, p.weight_ld, a0, p.dim_pad, (long long)k_first * KE, p.piece, wave, lane);
    lb.init(prob, p.prob_ld, b0, b0 + BB, (long long)k_first * KE, 0, wave, lane);
  } else {
    la.init(hidden, p.dim_pad, a0, p.dim_pad, 0, p.row_pad, wave, lane);
    lb.init(prob, p.prob_ld, b0, (int)p.prob_ld, 0, p.row_pad, wave, lane);
  }

  const int wa = wave % WA, wb = wave / WA;
  f32x4 acc[FA][FB];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (k_tiles > 0) {
    la.issue(smem);
    lb.issue(smem + BA * kKBytes);
  }
  for (int t = 0; t < k_tiles; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < k_tiles) {
      char* next = smem + ((t + 1) & 1) * kStage;
      la.issue(next);
      lb.issue(next + BA * kKBytes);
    }
    const char* sa = smem + (t & 1) * kStage;
    const char* sb = sa + BA * kKBytes;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      Frag fa[FA], fb[FB];
#pragma unroll
      for (int i = 0; i < FA; ++i) fa[i] = read_frag<T, kAAcross, BA>(sa, wa * TA + i * 16, ks, lane);
#pragma unroll
      for (int j = 0; j < FB; ++j) fb[j] = read_frag<T, kBAcross, BB>(sb, wb * TB + j * 16, ks, lane);
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = Elem<T>::mma(fa[i], fb[j], acc[i][j]);
    }
  }

  // acc[i][j][e] belongs to a = a0 + wa TA + 16 i + 4 (lane / 16) + e and b = b0 + wb TB + 16 j + lane % 16
  const int a_lane = a0 + wa * TA + 4 * (lane >> 4), b_lane = b0 + wb * TB + (lane & 15);
  if constexpr (MODE == kStats) {
    __syncthreads();                                    // the last tile has been read: LDS is free
    float2* red = reinterpret_cast<float2*>(smem);
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int n = b_lane + j * 16;
      const int y = n < count ? p.label[n] : -1;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v = a_lane + i * 16 + e;
          if (v >= p.vocab) acc[i][j][e] = -INFINITY;
          else if (v == y) p.zlab[n] = acc[i][j][e];
          top = fmaxf(top, acc[i][j][e]);
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += exp_of(acc[i][j][e] - ref);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16) red[wa * BB + wb * TB + j * 16 + lane] = make_float2(top, sum);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < BB; b += NW * 64) {
      float top = red[b].x, sum = red[b].y;
#pragma unroll
      for (int w = 1; w < WA; ++w) {
        const float2 o = red[w * BB + b];
        const float m = fmaxf(top, o.x), ref = m == -INFINITY ? 0.f : m;
        sum = sum * exp_of(top - ref) + o.y * exp_of(o.x - ref);
        top = m;
      }
      p.partial[(long long)ta * p.row_pad + b0 + b] = make_float2(top, sum);
    }
  } else if constexpr (MODE == kProb) {
    // d rounded once to the type of the products that follow: half a step (2^-9 of itself in bfloat16), the same that
    // rounding the gradients themselves costs
    T* out = static_cast<T*>(p.prob);
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int n = b_lane + j * 16;
      const bool kept = n < count;
      const int y = kept ? p.label[n] : -1;
      const float lse = kept ? p.lse[n] : 0.f;
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        T d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int a = a_lane + i * 16 + e, v = p.v0 + a;
          float x = exp_of(acc[i][j][e] - lse);
          x = v == y ? x - 1.f : x;
          d[e] = static_cast<T>(kept && v < p.vocab ? x * Elem<T>::kScale : 0.f);
        }
        __builtin_memcpy(out + (long long)n * p.prob_ld + a_lane + i * 16, d, sizeof d);
      }
    }
  } else if constexpr (MODE == kDhid) {
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int n = b_lane + j * 16;
      if (n >= count) continue;
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        const int d = a_lane + i * 16;
        if (d >= p.dim_pad) continue;
        f32x4* at = reinterpret_cast<f32x4*>(p.acc + ((long long)split * p.row_pad + n) * p.dim_pad + d);
        *at = p.first ? acc[i][j] : *at + acc[i][j];
      }
    }
  } else {
    const float factor = count > 0 ? *p.factor * (1.f / Elem<T>::kScale) : 0.f;
    const bool whole = (p.dim & 3) == 0;
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int b = b_lane + j * 16;
      if (b >= p.piece) continue;
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        const int d = a_lane + i * 16;
        const long long at = (long long)(p.v0 + b) * p.dim + d;
        const f32x4 x = count > 0 ? acc[i][j] * factor : f32x4{0.f, 0.f, 0.f, 0.f};
        if (p.grad_f32) {
          float* out = static_cast<float*>(p.grad_weight) + at;
          if (whole && d < p.dim) *reinterpret_cast<f32x4*>(out) = x;
          else
            for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = x[e];
        } else {
          T* out = static_cast<T*>(p.grad_weight) + at;
          T r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = static_cast<T>(x[e]);
          if (whole && d < p.dim) __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), r, sizeof r);
          else
            for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = r[e];
        }
      }
    }
  }
}

// ---- packing ------------------------------------------------------------------------------------------------
struct PackArgs {
  const void* labels;
  int label_bits;
  long long rows, inner, outer_stride, inner_stride, ignore_index;
  int dim, dim_pad, vocab, per_block;
  const void* hidden;
  void* packed;
  LceState st;
  float* losses;          // per-row losses to clear for ignored rows, or null
};

__device__ inline long long label_at(const void* labels, int bits, long long n) {
  return bits == 64 ? static_cast<const long long*>(labels)[n] : static_cast<const int*>(labels)[n];
}

// one row of `dim` values to a packed row of `dim_pad`, zeros behind; factor: nullptr or the row's weight
template <typename T>
__device__ inline void copy_row(const T* in, T* out, int dim, int dim_pad, int lane, int lanes, float weight,
                                bool weighted) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool wide = (reinterpret_cast<uintptr_t>(in) & 15) == 0;
  for (int c = lane; c < dim_pad / kVec; c += lanes) {
    T x[kVec];
    const int d0 = c * kVec;
    if (wide && d0 + kVec <= dim) __builtin_memcpy(x, __builtin_assume_aligned(in + d0, 16), 16);
    else
      for (int e = 0; e < kVec; ++e) x[e] = d0 + e < dim ? in[d0 + e] : static_cast<T>(0.f);
    if (weighted)
      for (int e = 0; e < kVec; ++e) x[e] = static_cast<T>(static_cast<float>(x[e]) * weight);
    __builtin_memcpy(__builtin_assume_aligned(out + d0, 16), x, 16);
  }
}

// Block b takes rows [b per_block, ...): the kept rows before it are counted again by every block (a read of at most
// all labels, out of L2), which saves a pass and its launch.  Rows behind the last kept one stay as they are: they
// reach only sums that nobody reads.
constexpr int kPackRows = 16;

template <typename T>
__global__ __launch_bounds__(256) void lce_pack_kernel(const PackArgs p) {
  __shared__ int counts[4];
  __shared__ int slot_of[64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long first = (long long)blockIdx.x * p.per_block;
  const long long last = min(first + p.per_block, p.rows);
  int before = 0;
  for (long long n = threadIdx.x; n < first; n += 256) before += label_at(p.labels, p.label_bits, n) != p.ignore_index;
  for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
  if (lane == 0) counts[wave] = before;
  __syncthreads();
  int at = counts[0] + counts[1] + counts[2] + counts[3];
  for (long long n0 = first; n0 < last; n0 += 64) {
    __syncthreads();
    if (wave == 0) {
      const long long n = n0 + lane;
      const long long y = n < last ? label_at(p.labels, p.label_bits, n) : p.ignore_index;
      const bool kept = n < last && y != p.ignore_index;
      const unsigned long long mask = __ballot(kept);
      const int r = at + __popcll(mask & ((1ull << lane) - 1));
      slot_of[lane] = kept ? r : -1;
      if (n < last) p.st.slot[n] = kept ? r : -1;
      if (kept) {
        p.st.index[r] = (int)n;
        p.st.label[r] = y >= 0 && y < p.vocab ? (int)y : -1;
        p.st.zlab[r] = __builtin_nanf("");
      } else if (n < last && p.losses) {
        p.losses[n] = 0.f;
      }
      if (lane == 0) counts[0] = __popcll(mask);
    }
    __syncthreads();
    at += counts[0];
    for (int i = wave; i < min(64ll, last - n0); i += 4) {
      const int r = slot_of[i];
      if (r < 0) continue;
      const long long n = n0 + i;
      const T* in = static_cast<const T*>(p.hidden) + (n / p.inner) * p.outer_stride + (n % p.inner) * p.inner_stride;
      copy_row<T>(in, static_cast<T*>(p.packed) + (long long)r * p.dim_pad, p.dim, p.dim_pad, lane, 64, 1.f, false);
    }
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) p.st.head[0] = at;      // the number of kept rows
}

// The backward pass packs again from the index the forward pass left: plain rows for PROB, and for a loss that is
// weighted row by row (upstream of WFE_REDUCE_NONE) rows times g_n / max |g| for DWEI.
struct RepackArgs {
  const void* hidden;
  long long inner, outer_stride, inner_stride;
  int dim, dim_pad, mean, per_row;
  LceState st;
  const float* upstream;
  float* row_factor;      // g of kept row r
  float* factor;          // what DWEI multiplies with; per_row: max |g|, left by lce_top_kernel
  void* packed;
  void* weighted;         // null unless per_row
};

// max |g| over the kept rows
__global__ __launch_bounds__(1024) void lce_top_kernel(const float* upstream, LceState st, float* factor) {
  __shared__ float tops[16];
  const int count = st.head[0];
  float top = 0.f;
  for (int r = threadIdx.x; r < count; r += 1024) top = fmaxf(top, fabsf(upstream[st.index[r]]));
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) top = fmaxf(top, tops[i]);
    *factor = top;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void lce_repack_kernel(const RepackArgs p) {
  const int count = p.st.head[0];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // DWEI goes over the rows in whole K tiles: zeros up to there
  const long long end = ((long long)count + kKElems<T> - 1) / kKElems<T> * kKElems<T>;
  const long long r0 = (long long)blockIdx.x * kPackRows;
  if (r0 >= end && blockIdx.x > 0) return;
  const float shared = p.per_row ? *p.factor : p.mean ? p.upstream[0] / (float)count : p.upstream[0];
  if (!p.per_row && blockIdx.x == 0 && threadIdx.x == 0) *p.factor = shared;
  for (long long r = r0 + wave; r < min(r0 + kPackRows, end); r += 4) {
    const bool kept = r < count;
    const long long n = kept ? p.st.index[r] : 0;
    const T* in = static_cast<const T*>(p.hidden) + (n / p.inner) * p.outer_stride + (n % p.inner) * p.inner_stride;
    const int dim = kept ? p.dim : 0;
    const float g = !kept ? 0.f : p.per_row ? p.upstream[n] : shared;
    if (kept && lane == 0) p.row_factor[r] = g;
    copy_row<T>(in, static_cast<T*>(p.packed) + r * p.dim_pad, dim, p.dim_pad, lane, 64, 1.f, false);
    if (p.per_row && p.weighted)
      copy_row<T>(in, static_cast<T*>(p.weighted) + r * p.dim_pad, dim, p.dim_pad, lane, 64,
                  shared > 0.f ? g / shared : g, true);
  }
}

// W with rows that the tiles cannot read in place (odd sizes, strides or alignment): one padded copy
template <typename T>
__global__ __launch_bounds__(256) void lce_pad_weight_kernel(const T* weight, long long ld, T* out, int dim,
                                                             int dim_pad, int vocab) {
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v < vocab)
    copy_row<T>(weight + (long long)v * ld, out + (long long)v * dim_pad, dim, dim_pad, threadIdx.x & 63, 64, 1.f, false);
}

// ---- losses out of the tiles' statistics --------------------------------------------------------------------
// 16 rows per block, 16 threads per row over the vocabulary tiles.
__global__ __launch_bounds__(256) void lce_loss_kernel(const float2* partial, int tiles, long long row_pad,
                                                       LceState st, float* losses, float* row_loss) {
  const int count = st.head[0];
  if ((long long)blockIdx.x * 16 >= count) return;
  const int col = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int r = blockIdx.x * 16 + col;
  __shared__ float2 red[16][16];
  float top = -INFINITY, sum = 0.f;
  if (r < count) {
    const float2* from = partial + r;
    for (int t0 = part; t0 < tiles; t0 += 16 * 8) {           // 8 loads in flight
      float2 o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        o[k] = t0 + 16 * k < tiles ? from[(long long)(t0 + 16 * k) * row_pad] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float m = fmaxf(top, o[k].x), ref = m == -INFINITY ? 0.f : m;
        sum = sum * exp_of(top - ref) + o[k].y * exp_of(o[k].x - ref);
        top = m;
      }
    }
  }
  red[part][col] = make_float2(top, sum);
  __syncthreads();
  if (part > 0 || r >= count) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, red[i][col].x);
  const float ref = top == -INFINITY ? 0.f : top;
  sum = 0.f;
  for (int i = 0; i < 16; ++i) sum += red[i][col].y * exp_of(red[i][col].x - ref);
  const float lse = st.label[r] < 0 ? __builtin_nanf("") : top + logf(sum);
  const float loss = lse - st.zlab[r];
  st.lse[r] = lse;
  row_loss[r] = loss;
  if (losses) losses[st.index[r]] = loss;
}

// sum or mean of the kept rows' losses, in float64 and in a fixed order.  (A launch of its own: one block telling the
// last of the others by a counter needs every block's writes out of its XCD's L2 first, which took 50 us.)
__global__ __launch_bounds__(1024) void lce_total_kernel(const float* row_loss, LceState st, float* total, int mean) {
  __shared__ double sums[16];
  const int count = st.head[0];
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) s += row_loss[i];
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sums[i];
    *total = (float)(mean ? s / (double)count : s);
  }
}

// dh: the splits' sums, times g, to every row's place; zeros for ignored rows
template <typename T>
__global__ __launch_bounds__(256) void lce_dhid_kernel(const float* acc, int splits, long long row_pad, int dim,
                                                       int dim_pad, long long rows, LceState st,
                                                       const float* row_factor, void* out, int out_f32) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long n = (long long)blockIdx.x * 4 + wave;
  if (n >= rows) return;
  const int r = st.slot[n];
  const bool kept = r >= 0;
  const float g = kept ? row_factor[r] * (1.f / Elem<T>::kScale) : 0.f;
  for (int d = lane * 4; d < dim; d += 256) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (kept) {
      for (int i = 0; i < splits; ++i)
        s += *reinterpret_cast<const f32x4*>(acc + ((long long)i * row_pad + r) * dim_pad + d);
      s *= g;
    }
    for (int e = 0; e < 4 && d + e < dim; ++e) {
      if (out_f32) static_cast<float*>(out)[n * dim + d + e] = s[e];
      else static_cast<T*>(out)[n * dim + d + e] = static_cast<T>(s[e]);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------------------
constexpr int kBA = 128, kBB = 128, kWA = 2, kWB = 2;
constexpr long long kPieceBytes = 256ll << 20;     // most that the piece of d held at a time takes

struct Plan {
  int size, ke, dim_pad;
  long long row_pad;
  bool copy_weight;
  int piece, splits;
  // offsets into the workspace
  long long packed, weighted, weight, partial, row_loss, prob, acc, row_factor, factor, bytes;
};

long long up(long long x, long long to) { return (x + to - 1) / to * to; }

Plan make_plan(const wfe_linear_ce& d, const void* weight, bool backward, int grads) {
  Plan p{};
  p.size = d.dtype == WFE_F32 ? 4 : 2;
  p.ke = kKBytes / p.size;
  p.dim_pad = (int)up(d.dim, p.ke);
  p.row_pad = up(d.rows > 0 ? d.rows : 1, kLceRowPad);
  // in place: whole K tiles, 16-byte rows, offsets inside a tile in 32 bits
  p.copy_weight = !(d.dim == p.dim_pad && (d.weight_stride * p.size) % 16 == 0 &&
                    d.weight_stride * p.size < (1ll << 22) && (reinterpret_cast<uintptr_t>(weight) & 15) == 0);
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long o = at;
    at += up(bytes, 256);
    return o;
  };
  p.packed = take(p.row_pad * p.dim_pad * p.size);
  if (p.copy_weight) p.weight = take((long long)d.vocab * p.dim_pad * p.size);
  if (!backward) {
    p.partial = take(up(d.vocab, kBA) / kBA * p.row_pad * 8);
    p.row_loss = take(p.row_pad * 4);
  } else {
    const long long all = up(d.vocab, kLceRowPad);
    long long piece = kPieceBytes / (p.row_pad * p.size) / kLceRowPad * kLceRowPad;
    piece = piece < kLceRowPad ? kLceRowPad : piece > all ? all : piece;
    p.piece = (int)piece;
    // DHID has few tiles of its own: its K, the vocabulary, is split until there are two blocks for each of the 256 CUs,
    // each with at least 8 K tiles
    const long long tiles = up(p.dim_pad, kBA) / kBA * (up(d.rows > 0 ? d.rows : 1, kBB) / kBB);
    long long splits = (512 + tiles - 1) / tiles;
    const long long most = (p.piece / p.ke + 7) / 8;
    p.splits = (int)(splits > most ? most : splits);
    if (grads & WFE_GRAD_WEIGHT) {
      if (d.reduction == WFE_REDUCE_NONE) p.weighted = take(p.row_pad * p.dim_pad * p.size);
    }
    p.prob = take(p.row_pad * p.piece * p.size);
    if (grads & WFE_GRAD_HIDDEN) p.acc = take(p.splits * p.row_pad * p.dim_pad * 4);
    p.row_factor = take(p.row_pad * 4);
    p.factor = take(4);
  }
  p.bytes = at;
  return p;
}

template <typename T, int MODE>
hipError_t launch_tiles(const TileArgs& a, long long tiles, hipStream_t stream) {
  constexpr int kLds = 2 * (kBA + kBB) * kKBytes;
  auto* kernel = lce_tile_kernel<T, MODE, kBA, kBB, kWA, kWB>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (e != hipSuccess) return e;
  if (tiles > 0x7ffffff0ll) return hipErrorInvalidValue;
  kernel<<<dim3((unsigned)up(tiles, 8)), dim3(kWA * kWB * 64), kLds, stream>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t pad_weight(const wfe_linear_ce& d, const Plan& p, const void* weight, char* ws, hipStream_t stream) {
  lce_pad_weight_kernel<T><<<dim3((d.vocab + 3) / 4), dim3(256), 0, stream>>>(
      static_cast<const T*>(weight), d.weight_stride, reinterpret_cast<T*>(ws + p.weight), d.dim, p.dim_pad, d.vocab);
  return hipGetLastError();
}

void fill_tiles(TileArgs& a, const wfe_linear_ce& d, const Plan& p, const void* weight, char* ws, const LceState& st) {
  a.hidden = ws + p.packed;
  a.weight = p.copy_weight ? ws + p.weight : weight;
  a.weight_ld = p.copy_weight ? p.dim_pad : d.weight_stride;
  a.dim = d.dim;
  a.dim_pad = p.dim_pad;
  a.v0 = 0;
  a.piece = a.vocab = d.vocab;
  a.row_pad = p.row_pad;
  a.head = st.head;
  a.label = st.label;
  a.zlab = st.zlab;
  a.lse = st.lse;
}

#define LCE_TRY(expr)                      \
  do {                                     \
    const hipError_t e_ = (expr);          \
    if (e_ != hipSuccess) return e_;       \
  } while (0)

template <typename T>
hipError_t forward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* labels, float* loss,
                   void* state, char* ws, hipStream_t stream) {
  const Plan p = make_plan(d, weight, false, 0);
  const LceState st = lce_state(state, d.rows);
  const bool none = d.reduction == WFE_REDUCE_NONE;
  PackArgs k{};
  k.labels = labels;
  k.label_bits = d.label_bits;
  k.rows = d.rows;
  k.inner = d.inner;
  k.outer_stride = d.outer_stride;
  k.inner_stride = d.inner_stride;
  k.ignore_index = d.ignore_index;
  k.dim = d.dim;
  k.dim_pad = p.dim_pad;
  k.vocab = d.vocab;
  k.per_block = (int)(d.rows <= kPackRows * 1024 ? kPackRows : up((d.rows + 1023) / 1024, 64));
  k.hidden = hidden;
  k.packed = ws + p.packed;
  k.st = st;
  k.losses = none ? loss : nullptr;
  const long long blocks = d.rows > 0 ? (d.rows + k.per_block - 1) / k.per_block : 1;
  lce_pack_kernel<T><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(k);
  LCE_TRY(hipGetLastError());
  if (p.copy_weight) LCE_TRY(pad_weight<T>(d, p, weight, ws, stream));
  TileArgs a{};
  fill_tiles(a, d, p, weight, ws, st);
  a.partial = reinterpret_cast<float2*>(ws + p.partial);
  a.a_tiles = (d.vocab + kBA - 1) / kBA;
  a.b_tiles = (int)((d.rows + kBB - 1) / kBB);
  if (d.rows > 0) LCE_TRY((launch_tiles<T, kStats>(a, (long long)a.a_tiles * a.b_tiles, stream)));
  float* row_loss = reinterpret_cast<float*>(ws + p.row_loss);
  if (d.rows > 0) {
    lce_loss_kernel<<<dim3((unsigned)((d.rows + 15) / 16)), dim3(256), 0, stream>>>(
        a.partial, a.a_tiles, p.row_pad, st, none ? loss : nullptr, row_loss);
    LCE_TRY(hipGetLastError());
  }
  if (!none) lce_total_kernel<<<dim3(1), dim3(1024), 0, stream>>>(row_loss, st, loss, d.reduction == WFE_REDUCE_MEAN);
  return hipGetLastError();
}

template <typename T>
hipError_t backward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* state,
                    const float* upstream, void* grad_hidden, void* grad_weight, char* ws, hipStream_t stream) {
  const int grads = (grad_hidden ? WFE_GRAD_HIDDEN : 0) | (grad_weight ? WFE_GRAD_WEIGHT : 0);
  const Plan p = make_plan(d, weight, true, grads);
  const LceState st = lce_state(const_cast<void*>(state), d.rows);
  RepackArgs k{};
  k.hidden = hidden;
  k.inner = d.inner;
  k.outer_stride = d.outer_stride;
  k.inner_stride = d.inner_stride;
  k.dim = d.dim;
  k.dim_pad = p.dim_pad;
  k.mean = d.reduction == WFE_REDUCE_MEAN;
  k.per_row = d.reduction == WFE_REDUCE_NONE;
  k.st = st;
  k.upstream = upstream;
  k.row_factor = reinterpret_cast<float*>(ws + p.row_factor);
  k.factor = reinterpret_cast<float*>(ws + p.factor);
  k.packed = ws + p.packed;
  k.weighted = grad_weight && k.per_row ? ws + p.weighted : nullptr;
  if (k.per_row) {
    lce_top_kernel<<<dim3(1), dim3(1024), 0, stream>>>(upstream, st, k.factor);
    LCE_TRY(hipGetLastError());
  }
  lce_repack_kernel<T><<<dim3((unsigned)(p.row_pad / kPackRows)), dim3(256), 0, stream>>>(k);
  LCE_TRY(hipGetLastError());
  if (p.copy_weight) LCE_TRY(pad_weight<T>(d, p, weight, ws, stream));
  TileArgs a{};
  fill_tiles(a, d, p, weight, ws, st);
  const T* w = static_cast<const T*>(a.weight);
  a.prob = ws + p.prob;
  a.prob_ld = p.piece;
  a.acc = reinterpret_cast<float*>(ws + p.acc);
  a.splits = p.splits;
  a.grad_weight = grad_weight;
  a.grad_f32 = d.grad_weight_dtype == WFE_F32;
  a.factor = k.factor;
  const int row_tiles = (int)((d.rows + kBB - 1) / kBB);
  const int dim_tiles = (p.dim_pad + kBA - 1) / kBA;
  for (int v0 = 0; v0 < d.vocab; v0 += p.piece) {
    a.v0 = v0;
    a.piece = d.vocab - v0 < p.piece ? d.vocab - v0 : p.piece;
    a.weight = w + (long long)v0 * a.weight_ld;
    a.hidden = ws + p.packed;
    a.first = v0 == 0;
    if (d.rows > 0) {
      a.a_tiles = (a.piece + kBA - 1) / kBA;
      a.b_tiles = row_tiles;
      LCE_TRY((launch_tiles<T, kProb>(a, (long long)a.a_tiles * a.b_tiles, stream)));
      if (grad_hidden) {
        a.a_tiles = dim_tiles;
        LCE_TRY((launch_tiles<T, kDhid>(a, (long long)dim_tiles * row_tiles * p.splits, stream)));
      }
    }
    if (grad_weight) {
      if (k.weighted) a.hidden = k.weighted;
      a.a_tiles = dim_tiles;
      a.b_tiles = (a.piece + kBB - 1) / kBB;
      LCE_TRY((launch_tiles<T, kDwei>(a, (long long)dim_tiles * a.b_tiles, stream)));
    }
  }
  if (grad_hidden && d.rows > 0) {
    lce_dhid_kernel<T><<<dim3((unsigned)((d.rows + 3) / 4)), dim3(256), 0, stream>>>(
        a.acc, p.splits, p.row_pad, d.dim, p.dim_pad, d.rows, st, k.row_factor, grad_hidden,
        d.grad_hidden_dtype == WFE_F32);
    LCE_TRY(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace

int64_t lce_workspace_bytes(const wfe_linear_ce& d, const void* weight, int backward, int grads) {
  return make_plan(d, weight, backward != 0, grads).bytes;
}

hipError_t launch_lce_forward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* labels,
                              float* loss, void* state, void* workspace, hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  if (d.dtype == WFE_F32) return forward<float>(d, hidden, weight, labels, loss, state, ws, stream);
  if (d.dtype == WFE_F16) return forward<_Float16>(d, hidden, weight, labels, loss, state, ws, stream);
  return forward<__bf16>(d, hidden, weight, labels, loss, state, ws, stream);
}

hipError_t launch_lce_backward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* state,
                               const float* upstream, void* grad_hidden, void* grad_weight, void* workspace,
                               hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  if (d.dtype == WFE_F32)
    return backward<float>(d, hidden, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
  if (d.dtype == WFE_F16)
    return backward<_Float16>(d, hidden, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
  return backward<__bf16>(d, hidden, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
}

}  // namespace wfe
