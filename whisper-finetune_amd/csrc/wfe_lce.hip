// wfe_lce.hip -- softmax cross entropy over the vocabulary without keeping the logits, and its gradients, for gfx950.
//
//   z[n][v] = h_n . W_v          lse_n = log sum_v exp z[n][v]          loss_n = lse_n - z[n][y_n]
//   d[n][v] = exp(z[n][v] - lse_n) - [v == y_n]
//   dh_n = g_n sum_v d[n][v] W_v          dW_v = sum_n g_n d[n][v] h_n          (g_n: upstream share of row n)
//
// Rows whose label is ignore_index are dropped first: lce_pack_kernel copies the kept ones together, every product
// after it runs over the kept rows only, whose number stays on the device.  All four products are one tile routine that
// multiplies K fragments out of LDS:
//   STATS  z tiles, reduced in registers to a maximum and a sum of exponentials per row and vocabulary tile
//   PROB   z tiles again, written as d for a piece of the vocabulary and, where the rows are many, a share of them
//   DHID   dh += d W over that piece, in float32
//   DWEI   the piece's rows of dW, in float32 until the last share of the rows, then written once
// Recomputing z costs one product more than keeping (rows, vocab) logits would.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "wfe_decoder.h"

namespace wfe {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Element types.  Frag: 32 K of 16 rows (or columns), a lane's share; lane group g = lane / 16 holds k = 8 g .. 8 g + 7
// of 2-byte types, and k = 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 of float: any order does that is the same on both
// sides of a product.
template <typename T> struct Elem;
template <> struct Elem<__bf16> {
  union Frag { i32x4 i; bf16x8 b; s16x4 s[2]; };
  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
  }
  static constexpr float kScale = 1.0f;
};
template <> struct Elem<_Float16> {
  union Frag { i32x4 i; f16x8 h; s16x4 s[2]; };
  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
  }
  // d is in (-2, 2), rows' own weights included: stored times 2^14 so that small probabilities stay clear of the subnormals
  static constexpr float kScale = 16384.0f;
};
// float32 products on the bfloat16 matrix instructions, which do 16 times the work of the float32 ones per cycle: a
// value is the exact sum of three bfloat16 (8 + 8 + 8 of its 24 bits, each the rounding of what is left), and of the nine
// partial products the six down to 2^-16 of the whole are added up, smallest first.  What is left out, mid lo, lo mid and
// lo lo with |mid| <= 2^-8 and |lo| <= 2^-17 of a value, is at most 2^-24 (1 + 2^-10) of a product: what rounding it to float32
// may cost, once.  (Of random values 2^-26 and less in 96 of 100 products.  Two products more would take it to 2^-34, at a
// third more matrix work.)  Infinities (inf - inf while splitting) come out as NaN:
// run_tile repeats such a tile with the float32 instructions.
template <> struct Elem<float> {
  struct Frag { f32x4 x[2]; };
  struct Parts { bf16x8 hi, mid, lo; };
  static __device__ Parts split(const Frag& f) {
    u32x4 hi, mid, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {                // two at a time, as the conversion instruction takes them
      const float a = f.x[k >> 1][2 * (k & 1)], b = f.x[k >> 1][2 * (k & 1) + 1];
      hi[k] = pair(a, b);
      const float ra = a - __builtin_bit_cast(float, hi[k] << 16), rb = b - __builtin_bit_cast(float, hi[k] & 0xffff0000u);
      mid[k] = pair(ra, rb);
      lo[k] = pair(ra - __builtin_bit_cast(float, mid[k] << 16), rb - __builtin_bit_cast(float, mid[k] & 0xffff0000u));
    }
    return {__builtin_bit_cast(bf16x8, hi), __builtin_bit_cast(bf16x8, mid), __builtin_bit_cast(bf16x8, lo)};
  }
  static __device__ unsigned pair(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
  // the six, smallest first, each for a row of results in turn: no instruction waits for the one before it
  template <int N>
  static __device__ void mma(const Parts& a, const Parts (&b)[N], f32x4 (&c)[N]) {
    const auto each = [&](auto&& term) {
#pragma unroll
      for (int j = 0; j < N; ++j) c[j] = term(b[j], c[j]);
    };
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.lo, y.hi, z, 0, 0, 0); });
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, y.lo, z, 0, 0, 0); });
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.mid, y.mid, z, 0, 0, 0); });
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.mid, y.hi, z, 0, 0, 0); });
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, y.mid, z, 0, 0, 0); });
    each([&](const Parts& y, f32x4 z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.hi, y.hi, z, 0, 0, 0); });
  }
  static __device__ f32x4 mma_exact(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[h][i], b.x[h][i], c, 0, 0, 0);
    return c;
  }
  static constexpr float kScale = 1.0f;
};

constexpr int kKElems = 32;                                // depth of a K tile
template <typename T> constexpr int kKBytes = kKElems * (int)sizeof(T);
constexpr int kPadRows = 64;                               // zeros follow the kept rows up to a multiple of this
constexpr float kLog2e = 1.44269504088896340736f;

// (The argument's rounding, half a step of x log2(e), is what a logit's own rounding may be; the loss of 16-bit inputs is off
// by 0.7e-6 at a dim of 384 and 1.2e-6 at 1280, root mean square.)
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A row's own weight as m 2^e, 1 <= |m| < 2 (or 0, an infinity, NaN): m goes into d before that is rounded, 2^e where it costs no
// rounding.
__device__ inline float weight_m(float g) { return 2.f * __builtin_amdgcn_frexp_mantf(g); }
__device__ inline int weight_e(float g) { return __builtin_amdgcn_frexp_expf(g) - 1; }

// ---- operands -------------------------------------------------------------------------------------------
// An operand tile in LDS is either rows x 32 of K ("along": K contiguous in memory) or K rows x columns
// ("across": K strided in memory, transposed by the read).  16-byte chunks of a row are permuted by an exclusive or
// so that the lanes of a fragment read meet different banks:
//   along, 64 bytes rows of 4 chunks, 4 rows cover the banks: rows 4 apart take different pairs of chunks (a 16-byte
//                   read serves 8 lanes of one chunk number with 8 of the next at a time)
//   along, 128      rows of 8 chunks: chunk ^ (row & 7)
//   across, 2 byte  pairs of chunks (a transposing read takes 32 bytes of each of 4 rows); 8 rows 0..3, 8..11 apart
//   across, 4 byte  groups of four chunks; 4 rows 4 apart
template <typename T, bool ACROSS, int N, int KS>
__device__ inline int swizzle(int row) {
  if constexpr (!ACROSS) return KS * sizeof(T) == 2 ? (row >> 1) & 2 : row & 7;
  else if constexpr (sizeof(T) == 2) return (((row & 3) | ((row >> 1) & 4)) & (N / 16 - 1)) << 1;
  else return (((row >> 2) & 3) & (N / 16 - 1)) << 2;
}

// Loads tiles of N rows (or columns) with NW waves, 1024 bytes per wave and instruction straight into LDS.
template <typename T, bool ACROSS, int N, int NW, int KS>
struct Loader {
  static constexpr int kRowBytes = ACROSS ? N * (int)sizeof(T) : KS * kKBytes<T>;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTileBytes = N * KS * kKBytes<T>;
  static constexpr int kInstrs = kTileBytes / 1024;
  static constexpr int kPer = (kInstrs + NW - 1) / NW;
  const char* base;
  long long step;                 // bytes from one K tile to the next
  long long ld;                   // bytes
  int k_left;                     // K rows (across), or bytes of a row (along), that exist from the current tile on
  const char* zeros;              // along: 16 bytes of zeros, read in place of those that do not exist
  unsigned off[kPer];
  int wave, lane;

  // first: row or column of the tile; limit: rows (along) or columns (across, a multiple of 16 bytes) that exist;
  // k0: the first K; k_end: the K that exist (along: whole 16 bytes, from k0 = 0 on)
  __device__ void init(const T* p, long long ld_elems, int first, int limit, long long k0, long long k_end, int w,
                       int l, const T* zero = nullptr) {
    wave = w;
    lane = l;
    ld = ld_elems * (long long)sizeof(T);
    if constexpr (ACROSS) {
      base = reinterpret_cast<const char*>(p) + k0 * ld + (long long)first * sizeof(T);
      step = ld * kKElems * KS;
      k_left = (int)(k_end - k0);
    } else {
      base = reinterpret_cast<const char*>(p) + (long long)first * ld + k0 * (long long)sizeof(T);
      step = KS * kKBytes<T>;
      k_left = (int)k_end * (int)sizeof(T);
      zeros = reinterpret_cast<const char*>(zero);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int id = (i * NW + wave) % kInstrs * 64 + lane;     // (a small tile: some waves fetch the same again)
      int row = id / kChunks;
      int c = (id % kChunks) ^ swizzle<T, ACROSS, N, KS>(row);
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
  // LAST: the tile may reach past the K that exist.  Rows that do not are read as the last one that does (their factors on
  // the other side are 0); of a row, zeros in place of what does not (their factors are 0, but what lies there may be
  // infinite, or nobody's memory).
  template <bool LAST, bool TAIL>
  __device__ void issue(char* lds) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int instr = (i * NW + wave) % kInstrs;
      unsigned o = off[i];
      if constexpr (ACROSS && LAST) {
        const int row = (instr * 64 + lane) / kChunks;
        o -= (unsigned)(max(row - k_left + 1, 0) * ld);
      }
      const char* from = base + o;
      if constexpr (!ACROSS && LAST && TAIL) {
        const int id = instr * 64 + lane, c = (id % kChunks) ^ swizzle<T, false, N, KS>(id / kChunks);
        from = c * 16 < k_left ? from : zeros;
      }
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)from,
          (__attribute__((address_space(3))) void*)(lds + instr * 1024), 16, 0, 0);
    }
    base += step;
    k_left -= ACROSS ? KS * kKElems : KS * kKBytes<T>;
  }
};

// Fragment of 16 rows (or columns) from m0 on, step ks of the tile's KS
template <typename T, bool ACROSS, int N, int KS>
__device__ inline typename Elem<T>::Frag read_frag(const char* lds, int m0, int ks, int lane) {
  typename Elem<T>::Frag r;
  const int g = lane >> 4;
  if constexpr (!ACROSS) {
    const int row = m0 + (lane & 15), swz = swizzle<T, false, N, KS>(row);
    const char* at = lds + row * (KS * kKBytes<T>);
    if constexpr (sizeof(T) == 2) r.i = *reinterpret_cast<const i32x4*>(at + ((4 * ks + g) ^ swz) * 16);
    else
#pragma unroll
      for (int h = 0; h < 2; ++h) r.x[h] = *reinterpret_cast<const f32x4*>(at + ((8 * ks + 4 * h + g) ^ swz) * 16);
  } else if constexpr (sizeof(T) == 2) {
    const int j = (lane & 15) >> 2, q = lane & 3;
    const int chunk = m0 / 8 + (q >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 32 * ks + 8 * g + 4 * h + j;
      r.s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
          lds + row * (N * 2) + (chunk ^ swizzle<T, true, N, KS>(row)) * 16 + (q & 1) * 8));
    }
  } else {
    const int col = m0 + (lane & 15);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 32 * ks + 16 * h + 4 * g + i;
        r.x[h][i] = *reinterpret_cast<const float*>(lds + row * (N * 4) + ((col / 4) ^ swizzle<T, true, N, KS>(row)) * 16 +
                                                    (col & 3) * 4);
      }
  }
  return r;
}

// ---- the tile routine --------------------------------------------------------------------------------------
template <int N> struct Const { static constexpr int value = N; };
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
enum Mode { kStats, kProb, kDhid, kDwei };

// A block's tile: BA x BB results of WA x WB waves, S K tiles of KS steps of 32 in LDS, PER blocks on a CU at a time
template <int BA_, int BB_, int WA_, int WB_, int S_, int PER_, int KS_ = 1>
struct Cfg {
  static constexpr int BA = BA_, BB = BB_, WA = WA_, WB = WB_, S = S_, PER = PER_, KS = KS_;
  static constexpr int kThreads = WA * WB * 64;
  static constexpr int kWavesPerSimd = PER * WA * WB / 4;
  static constexpr int kSlots = 256 * PER;                 // blocks that run at once on 256 CUs
};
template <typename T, class C> constexpr int kStageBytes = (C::BA + C::BB) * C::KS * kKBytes<T>;
template <typename T, class C> constexpr int kLdsBytes = C::S * kStageBytes<T, C>;

struct TileArgs {
  const void* hidden;     // packed rows (row_pad, dim_pad)
  const void* weighted;   // DWEI: the same, or rows times 2^e of their own weight
  const void* weight;     // (vocab, weight_cols) from row v0 on, weight_ld elements apart
  void* prob;             // d of the piece, (share, prob_ld)
  long long weight_ld, prob_ld;
  int weight_cols;        // dim, or dim_pad with zeros behind dim; 16-byte rows either way
  int dim, dim_pad, v0, piece, vocab;      // the piece holds vocabulary rows v0 .. v0 + piece - 1
  long long row_pad;
  const int* head;        // [0] kept rows
  int row0, share;        // kept rows of this call: row0 .. row0 + share - 1, as many of them as there are; what belongs to
                          // rows (hidden, weighted, label, lse, index, acc) starts at row0
  const int* label;
  float* zlab;
  const float* lse;
  const float* own;       // PROB: the rows' own weights (upstream of WFE_REDUCE_NONE, by row of hidden), or null
  const int* index;       // rows of hidden
  float2* partial;        // STATS: (vocabulary tiles, row_pad) maximum and sum
  float* acc;             // DHID: (splits, row_pad, dim_pad)
  int first;              // DHID: acc starts with this piece
  float* wacc;            // DWEI: sums over the shares of the rows so far, (piece, dim_pad)
  int share_first, share_last;
  void* grad_weight;      // DWEI: (vocab, dim)
  int grad_f32;
  const float* factor;    // DWEI: multiplied with; mean: divided by the number of kept rows
  int mean;
};

__device__ inline int rows_of(const TileArgs& p) { return max(0, min(p.head[0] - p.row0, p.share)); }

// The id-th of `a_tiles` x `b_tiles` tiles, from column b_first on, of part `split` of `splits` of K.  smem: kLdsBytes.
template <typename T, class C, int MODE>
__device__ __forceinline__ void run_tile(const TileArgs& p, int count, int id, int a_tiles, int b_tiles, int b_first,
                                         int splits, char* smem) {
  constexpr bool kAAcross = MODE == kDhid || MODE == kDwei;
  constexpr bool kBAcross = MODE == kDwei;
  constexpr int BA = C::BA, BB = C::BB, WA = C::WA, WB = C::WB, kStages = C::S, kStage = kStageBytes<T, C>, KS = C::KS;
  constexpr int NW = WA * WB, TA = BA / WA, TB = BB / WB, FA = TA / 16, FB = TB / 16;
  constexpr int KE = kKElems * KS;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;

  const int plane = a_tiles * b_tiles;
  const int split = id / plane;
  id -= split * plane;
  constexpr int kGroup = 8;                                // tiles of one axis that stay in an XCD's L2 as the other passes
  const int group = id / (kGroup * a_tiles);
  const int rest = id - group * kGroup * a_tiles;
  const int in_group = min(kGroup, b_tiles - group * kGroup);
  const int ta = rest / in_group, tb = group * kGroup + rest % in_group;
  const int a0 = ta * BA, b0 = b_first + tb * BB;

  // K range, in tiles
  int k_first = 0, k_tiles;
  if constexpr (MODE == kStats || MODE == kProb) k_tiles = (p.dim + KE - 1) / KE;
  else if constexpr (MODE == kDwei) k_tiles = (count + KE - 1) / KE;
  else {
    const int all = (p.piece + KE - 1) / KE;
    const int each = (all + splits - 1) / splits;
    k_first = min(split * each, all);
    k_tiles = min(each, all - k_first);
  }

  const int wa = wave % WA, wb = wave / WA;
  f32x4 acc[FA][FB];
  auto product = [&](auto exact) {
    Loader<T, kAAcross, BA, NW, KS> la;
    Loader<T, kBAcross, BB, NW, KS> lb;
    const T* weight = static_cast<const T*>(p.weight);
    const T* prob = static_cast<const T*>(p.prob);
    if constexpr (MODE == kStats || MODE == kProb) {
      const T* hidden = static_cast<const T*>(p.hidden);      // its first row has zeros behind dim
      la.init(weight, p.weight_ld, a0, p.piece, 0, p.weight_cols, wave, lane, hidden + p.dim);
      lb.init(hidden, p.dim_pad, b0, b0 + BB, 0, 0, wave, lane);
    } else if constexpr (MODE == kDhid) {
      la.init(weight, p.weight_ld, a0, p.weight_cols, (long long)k_first * KE, p.piece, wave, lane);
      lb.init(prob, p.prob_ld, b0, b0 + BB, (long long)k_first * KE, 0, wave, lane);
    } else {
      la.init(static_cast<const T*>(p.weighted), p.dim_pad, a0, p.dim_pad, 0, p.share, wave, lane);
      lb.init(prob, p.prob_ld, b0, (int)p.prob_ld, 0, p.share, wave, lane);
    }

#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // kStages K tiles in LDS, all but one of them on their way while one is multiplied.  Per tile: wait until this wave's
    // part of the oldest has arrived (the younger ones may stay under way), one barrier -- now everybody's has, and
    // everybody has read the tile before it, whose place the next fetch takes -- then read fragments and multiply.
    // (The barrier is written out: __syncthreads would wait for every fetch.)
    constexpr int kFetches = decltype(la)::kPer + decltype(lb)::kPer;      // of every wave, per tile
    auto fetch = [&](auto last, int stage) {
      char* to = smem + stage * kStage;
      la.template issue<decltype(last)::value, true>(to);
      lb.template issue<decltype(last)::value, false>(to + BA * KS * kKBytes<T>);
    };
    typename Elem<T>::Frag fa[FA], fb[FB];
    auto read = [&](int stage, int ks) {
      const char* sa = smem + stage * kStage;
      const char* sb = sa + BA * KS * kKBytes<T>;
#pragma unroll
      for (int i = 0; i < FA; ++i) fa[i] = read_frag<T, kAAcross, BA, KS>(sa, wa * TA + i * 16, ks, lane);
#pragma unroll
      for (int j = 0; j < FB; ++j) fb[j] = read_frag<T, kBAcross, BB, KS>(sb, wb * TB + j * 16, ks, lane);
    };
    auto multiply = [&] {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int j = 0; j < FB; ++j) acc[i][j] = Elem<T>::mma(fa[i], fb[j], acc[i][j]);
      } else if constexpr (decltype(exact)::value) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int j = 0; j < FB; ++j) acc[i][j] = Elem<T>::mma_exact(fa[i], fb[j], acc[i][j]);
      } else {
        typename Elem<T>::Parts pb[FB];
#pragma unroll
        for (int j = 0; j < FB; ++j) pb[j] = Elem<T>::split(fb[j]);
#pragma unroll
        for (int i = 0; i < FA; ++i) Elem<T>::mma(Elem<T>::split(fa[i]), pb, acc[i]);
        // The order to issue them in: the splitting that the first products wait for, then one product to two vector
        // instructions.  Left to itself the compiler bunches them (201 x 384 x 51866: z 79 us, the gradients 143; so 74 and
        // 139; 384 rows: 105 and 220, so 99 and 210).
        __builtin_amdgcn_sched_group_barrier(0x002, 16 * (FA + FB), 0);
#pragma unroll
        for (int i = 0; i < 6 * FA * FB; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
        }
      }
    };
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t)
      if (t < k_tiles) {
        if (t + 1 < k_tiles) fetch(No{}, t);
        else fetch(Yes{}, t);
      }
    int stage = 0, free = kStages - 1;
    auto advance = [&] {
      free = stage;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    };
    if constexpr (NW == 8) {
      // Two waves per SIMD take turns: while one reads its fragments the other multiplies, one barrier per turn, the
      // second group half a tile behind the first.
      if (k_tiles >= kStages - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 2) * kFetches) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_barrier" ::: "memory");
      const bool second = wave >= 4;
      if (second) asm volatile("s_barrier" ::: "memory");
      auto turn = [&](auto more) {
        static_assert(KS == 1, "a turn is one step");
        read(stage, 0);
        if constexpr (decltype(more)::value == 2) fetch(No{}, free);
        if constexpr (decltype(more)::value == 1) fetch(Yes{}, free);
        if constexpr (decltype(more)::value > 0)
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kStages - 2) * kFetches) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        multiply();
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        advance();
      };
      int t = 0;
      for (; t + kStages < k_tiles; ++t) turn(Const<2>{});
      for (; t + kStages - 1 < k_tiles; ++t) turn(Const<1>{});
      for (; t < k_tiles; ++t) turn(Const<0>{});
      if (!second) asm volatile("s_barrier" ::: "memory");
    } else {
      auto tile = [&](auto more) {
        if constexpr (decltype(more)::value > 0)
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kStages - 2) * kFetches) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if constexpr (decltype(more)::value == 2) fetch(No{}, free);
        if constexpr (decltype(more)::value == 1) fetch(Yes{}, free);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          read(stage, ks);
          multiply();
        }
        advance();
      };
      int t = 0;
      for (; t + kStages < k_tiles; ++t) tile(Const<2>{});
      for (; t + kStages - 1 < k_tiles; ++t) tile(Const<1>{});
      for (; t < k_tiles; ++t) tile(Const<0>{});
    }
  };
  product(No{});
  if constexpr (sizeof(T) == 4) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= acc[i][j][e] != acc[i][j][e];
    if (__syncthreads_or(bad)) product(Yes{});
  }

  // acc[i][j][e] belongs to a = a0 + wa TA + 16 i + 4 (lane / 16) + e and b = b0 + wb TB + 16 j + lane % 16
  const int a_lane = a0 + wa * TA + 4 * (lane >> 4), b_lane = b0 + wb * TB + (lane & 15);
  if constexpr (MODE == kStats) {
    __syncthreads();                                    // the last tile has been read: LDS is free
    float2* red = reinterpret_cast<float2*>(smem);
    const bool ragged = a0 + BA > p.vocab;
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int n = b_lane + j * 16;
      const int y = n < count ? p.label[n] : -1;
      float top = -INFINITY;
      if (ragged) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (a_lane + i * 16 + e >= p.vocab) acc[i][j][e] = -INFINITY;
      }
      if (__any(y >= a0 + wa * TA && y < a0 + (wa + 1) * TA)) {      // seldom: the label is in this wave's part
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (a_lane + i * 16 + e == y) p.zlab[n] = acc[i][j][e];
      }
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
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
    // d rounded once to the type of the products that follow: at most half a step (2^-8 of itself in bfloat16), the same
    // that rounding the gradients themselves costs
    T* out = static_cast<T*>(p.prob);
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int n = b_lane + j * 16;
      const bool kept = n < count;
      const int y = kept ? p.label[n] : -1;
      const float lse = kept ? p.lse[n] : 0.f;
      const float m = Elem<T>::kScale * (kept && p.own ? weight_m(p.own[p.index[n]]) : 1.f);
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        T d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int a = a_lane + i * 16 + e, v = p.v0 + a;
          float x = exp_of(acc[i][j][e] - lse);
          x = v == y ? x - 1.f : x;
          d[e] = static_cast<T>(kept && v < p.vocab ? x * m : 0.f);
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
    const int all = p.head[0];
    const float factor = all > 0 ? *p.factor / (p.mean ? (float)all : 1.f) * (1.f / Elem<T>::kScale) : 0.f;
    const bool whole = (p.dim & 3) == 0;
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int b = b_lane + j * 16;
      if (b >= p.piece) continue;
#pragma unroll
      for (int i = 0; i < FA; ++i) {
        const int d = a_lane + i * 16;
        if (d >= p.dim) continue;
        f32x4 sum = acc[i][j];
        f32x4* so_far = reinterpret_cast<f32x4*>(p.wacc + (long long)b * p.dim_pad + d);
        if (!p.share_first) sum += *so_far;
        if (!p.share_last) {
          *so_far = sum;
          continue;
        }
        const long long at = (long long)(p.v0 + b) * p.dim + d;
        const f32x4 x = all > 0 ? sum * factor : f32x4{0.f, 0.f, 0.f, 0.f};
        if (p.grad_f32) {
          float* out = static_cast<float*>(p.grad_weight) + at;
          if (whole) *reinterpret_cast<f32x4*>(out) = x;
          else
            for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = x[e];
        } else {
          T* out = static_cast<T*>(p.grad_weight) + at;
          T r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = static_cast<T>(x[e]);
          if (whole) __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), r, sizeof r);
          else
            for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = r[e];
        }
      }
    }
  }
}

// Blocks go to the 8 XCDs in turn.  Block b of a run of `tiles` takes a tile such that each XCD has a contiguous part
// of the run; -1: none.  A run takes run_blocks of the grid.
__device__ __host__ inline int run_blocks(int tiles) { return (tiles + 7) / 8 * 8; }
__device__ inline int tile_of(int b, int tiles) {
  const int per = (tiles + 7) / 8, id = (b & 7) * per + (b >> 3);
  return id < tiles ? id : -1;
}

// The kept rows as strips of a tile's width; the rows that are left over, if they are few, take a narrower tile of the
// same threads (552 rows as 2 x 256 + 64 instead of 3 x 256: z of 552 x 768 x 51866 takes 62 us instead of 73, of 100 rows 18
// instead of 25, of 280 float32 rows of 384 97 us instead of 176).
template <class C>
struct Strips {
  static constexpr bool kNarrow = C::BB >= 128;
  static constexpr int kHalf = kNarrow ? C::BB / 2 : C::BB, kQuarter = kNarrow ? C::BB / 4 : C::BB;
  using Half = Cfg<C::BA, kHalf, C::WA, C::WB, C::S, C::PER>;
  using Quarter = Cfg<C::BA, kQuarter, C::WA, C::WB, C::S, C::PER>;
  int whole, rest;              // strips of C::BB rows; rows of the narrow strip: 0, a quarter or half of that
  __device__ explicit Strips(int count) {
    const int over = count % C::BB;
    rest = !kNarrow || over == 0 || over > kHalf ? 0 : over > kQuarter ? kHalf : kQuarter;
    whole = count / C::BB + (over > 0 && rest == 0);
  }
};

// Block b of the tiles over all strips, whole ones first; false: behind the last block
template <typename T, class C, int MODE>
__device__ __forceinline__ bool run_strips(const TileArgs& p, int count, int& b, int a_tiles, int splits, char* smem) {
  using S = Strips<C>;
  const S s(count);
  const int tiles = a_tiles * s.whole * splits;
  if (b < run_blocks(tiles)) {
    const int id = tile_of(b, tiles);
    if (id >= 0) run_tile<T, C, MODE>(p, count, id, a_tiles, s.whole, 0, splits, smem);
    return true;
  }
  b -= run_blocks(tiles);
  if constexpr (S::kNarrow) {
    const int narrow = s.rest > 0 ? a_tiles * splits : 0;
    if (b < run_blocks(narrow)) {
      const int id = tile_of(b, narrow);
      if (id >= 0) {
        if (s.rest == S::kQuarter) run_tile<T, typename S::Quarter, MODE>(p, count, id, a_tiles, 1, s.whole * C::BB, splits, smem);
        else run_tile<T, typename S::Half, MODE>(p, count, id, a_tiles, 1, s.whole * C::BB, splits, smem);
      }
      return true;
    }
    b -= run_blocks(narrow);
  }
  return false;
}

template <typename T, class C, int MODE>
__global__ __launch_bounds__(C::kThreads, C::kWavesPerSimd) void lce_logits_kernel(const TileArgs p) {
  extern __shared__ __align__(1024) char smem[];
  int b = blockIdx.x;
  run_strips<T, C, MODE>(p, rows_of(p), b, (p.piece + C::BA - 1) / C::BA, 1, smem);
}

// DHID has few tiles of its own, so its K, the vocabulary, is split.  Beside DWEI: parts of half a CU's share of all
// the work.  Alone: the number of parts (of up to 8, or about one round) that leaves the fewest CUs idle in the last
// round.  (480 x 1280 x 51866 bfloat16, 10 tiles: alone 69 us, unsplit 833; beside DWEI 173, unsplit 1071.)
struct SplitRule {
  int dim_tiles, bb, piece_steps, dwei_tiles, ke, slots, most;
};
__device__ inline int dhid_splits(const SplitRule& r, int count) {
  const int tiles = r.dim_tiles * ((count + r.bb - 1) / r.bb);
  if (tiles == 0) return 1;
  if (r.dwei_tiles > 0) {
    const long long work = (long long)r.dwei_tiles * ((count + r.ke - 1) / r.ke) + (long long)tiles * r.piece_steps;
    const long long part = max(work / (2 * r.slots), 8ll);
    return (int)min((long long)r.most, (r.piece_steps + part - 1) / part);
  }
  int best = 1;
  float left = 0.f;
  for (int k = 1; k <= min(r.most, max(8, r.slots / tiles)); ++k) {
    const int rounds = (tiles * k + r.slots - 1) / r.slots;
    const float busy = (float)(tiles * k) / (float)(rounds * r.slots);
    if (busy > left + 0.02f) {
      left = busy;
      best = k;
    }
  }
  return best;
}

// The gradients' products over one block of d (a piece of the vocabulary, a share of the rows), and the next block's d, in
// one grid: long tiles first, so that the short ones fill the CUs that run out of them.  (4500 x 1280 x 51866 bfloat16, all
// but the first of four blocks' d: 1.64 TFLOP in 1.56 ms, 1.06 PFLOP/s.)
struct GradArgs {
  TileArgs t;
  SplitRule rule;
  int dhid, dwei;
  TileArgs next;                // PROB's; piece 0: no next block
};

template <typename T, class C>
__global__ __launch_bounds__(C::kThreads, C::kWavesPerSimd) void lce_grads_kernel(const GradArgs g) {
  extern __shared__ __align__(1024) char smem[];
  const int count = rows_of(g.t);
  const int dim_tiles = g.rule.dim_tiles;
  int b = blockIdx.x;
  if (g.dwei) {
    const int b_tiles = (g.t.piece + C::BB - 1) / C::BB, tiles = dim_tiles * b_tiles;
    if (b < run_blocks(tiles)) {
      const int id = tile_of(b, tiles);
      if (id >= 0) run_tile<T, C, kDwei>(g.t, count, id, dim_tiles, b_tiles, 0, 1, smem);
      return;
    }
    b -= run_blocks(tiles);
  }
  if (g.dhid && run_strips<T, C, kDhid>(g.t, count, b, dim_tiles, dhid_splits(g.rule, count), smem)) return;
  if (g.next.piece > 0) run_strips<T, C, kProb>(g.next, rows_of(g.next), b, (g.next.piece + C::BA - 1) / C::BA, 1, smem);
}

// ---- packing ------------------------------------------------------------------------------------------------
// (These kernels take microseconds, which first fetches of instructions dominate: the aligned case of each is a kernel
// of its own, indices are 32 bits.)
struct PackArgs {
  const void* labels;
  int label_bits, rows, inner;
  long long outer_stride, inner_stride, ignore_index;
  int dim, dim_pad, vocab, per_block;
  const void* hidden;
  LceState st;
  float* losses;          // per-row losses to clear for ignored rows, or null
};

__device__ inline long long label_at(const void* labels, int bits, int n) {
  return bits == 64 ? static_cast<const long long*>(labels)[n] : static_cast<const int*>(labels)[n];
}

// one row of `dim` values to a packed row of `dim_pad`, zeros behind.  WIDE: dim == dim_pad and 16-byte rows
template <typename T, bool WIDE>
__device__ inline void copy_row(const T* in, T* out, int dim, int dim_pad, int lane) {
  constexpr int kVec = 16 / (int)sizeof(T);
  for (int d = lane * kVec; d < dim_pad; d += 64 * kVec) {
    T x[kVec];
    if constexpr (WIDE) __builtin_memcpy(x, __builtin_assume_aligned(in + d, 16), 16);
    else
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = d + e < dim ? in[d + e] : static_cast<T>(0.f);
    __builtin_memcpy(__builtin_assume_aligned(out + d, 16), x, 16);
  }
}

// Block b takes rows [b per_block, ...): the kept rows before it are counted again by every block (a read of at most
// all labels, out of L2), which saves a pass and its launch.  1 row 3.4 us, 768 of 1280 bfloat16 5.2, 7168 14.6 (some 4500
// kept, 23 MB read and written).
constexpr int kPackRows = 4;

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void lce_pack_kernel(const PackArgs p) {
  __shared__ int counts[4];
  __shared__ int slot_of[64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int first = blockIdx.x * p.per_block, last = min(first + p.per_block, p.rows);
  int before = 0;
#pragma unroll 4
  for (int n = threadIdx.x; n < first; n += 256) before += label_at(p.labels, p.label_bits, n) != p.ignore_index;
  for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
  if (lane == 0) counts[wave] = before;
  __syncthreads();
  int at = counts[0] + counts[1] + counts[2] + counts[3];
#pragma unroll 1
  for (int n0 = first; n0 < last; n0 += 64) {
    __syncthreads();
    if (wave == 0) {
      const int n = n0 + lane;
      const long long y = n < last ? label_at(p.labels, p.label_bits, n) : p.ignore_index;
      const bool kept = y != p.ignore_index;
      const unsigned long long mask = __ballot(kept);
      const int r = at + __popcll(mask & ((1ull << lane) - 1));
      slot_of[lane] = kept ? r : -1;
      if (n < last) p.st.slot[n] = kept ? r : -1;
      if (kept) {
        p.st.index[r] = n;
        p.st.label[r] = y >= 0 && y < p.vocab ? (int)y : -1;
        p.st.zlab[r] = __builtin_nanf("");
      } else if (n < last && p.losses) {
        p.losses[n] = 0.f;
      }
      if (lane == 0) counts[0] = __popcll(mask);
    }
    __syncthreads();
    at += counts[0];
#pragma unroll 1
    for (int i = wave; i < min(64, last - n0); i += 4) {
      const int r = slot_of[i];
      if (r < 0) continue;
      const unsigned n = n0 + i, outer = n / (unsigned)p.inner;
      const T* in = static_cast<const T*>(p.hidden) + outer * p.outer_stride + (n - outer * p.inner) * p.inner_stride;
      copy_row<T, WIDE>(in, static_cast<T*>(p.st.packed) + (long long)r * p.dim_pad, p.dim, p.dim_pad, lane);
    }
  }
  if (blockIdx.x == gridDim.x - 1) {         // knows the number of kept rows
    if (threadIdx.x == 0) p.st.head[0] = at;
    // DWEI goes over the rows in whole K tiles: zeros up to there (rows further on reach only sums that nobody reads)
    const int end = (at + kPadRows - 1) / kPadRows * kPadRows;
    const int vecs = (end - at) * (p.dim_pad / (16 / (int)sizeof(T)));
    f32x4* out = reinterpret_cast<f32x4*>(static_cast<T*>(p.st.packed) + (long long)at * p.dim_pad);
#pragma unroll 1
    for (int i = threadIdx.x; i < vecs; i += 256) out[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// 2^e of the largest weight of the kept rows (a few hundred: 4.5 us)
__global__ __launch_bounds__(1024) void lce_top_kernel(const float* upstream, LceState st, float* factor) {
  __shared__ int tops[16];
  constexpr int kNone = -1000;
  const int count = st.head[0];
  int top = kNone;
  for (int r = threadIdx.x; r < count; r += 1024) {
    const float g = upstream[st.index[r]];
    if (g != 0.f) top = max(top, weight_e(g));
  }
  for (int d = 32; d > 0; d >>= 1) top = max(top, __shfl_xor(top, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) top = max(top, tops[i]);
    *factor = top == kNone ? 1.f : __builtin_amdgcn_ldexpf(1.f, top);
  }
}

// A loss weighted row by row (upstream of WFE_REDUCE_NONE): rows times 2^e_n over the largest 2^e for DWEI, exact but for what
// leaves the type's range (half precision: below 2^-24 of the largest weight's rows).  A few hundred rows of 384 float32: 4.7 us.
template <typename T>
__global__ __launch_bounds__(256) void lce_weigh_kernel(const void* packed, void* weighted, int dim_pad, LceState st,
                                                        const float* upstream, const float* top) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int count = st.head[0];
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= (count + kPadRows - 1) / kPadRows * kPadRows) return;
  const bool kept = r < count;
  const int e = kept ? min(weight_e(upstream[st.index[r]]) - weight_e(*top), 0) : 0;      // (a weight of 0 has any exponent)
  for (int d = (threadIdx.x & 63) * kVec; d < dim_pad; d += 64 * kVec) {
    T x[kVec];
    __builtin_memcpy(x, __builtin_assume_aligned(static_cast<const T*>(packed) + (long long)r * dim_pad + d, 16), 16);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      x[k] = kept ? static_cast<T>(__builtin_amdgcn_ldexpf(static_cast<float>(x[k]), e)) : static_cast<T>(0.f);
    __builtin_memcpy(__builtin_assume_aligned(static_cast<T*>(weighted) + (long long)r * dim_pad + d, 16), x, 16);
  }
}

// W with rows that the tiles cannot read in place (odd sizes, strides or alignment): one padded copy (5003 x 250: 4.2 us)
template <typename T>
__global__ __launch_bounds__(256) void lce_pad_weight_kernel(const T* weight, long long ld, T* out, int dim,
                                                             int dim_pad, int vocab) {
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v < vocab)
    copy_row<T, false>(weight + (long long)v * ld, out + (long long)v * dim_pad, dim, dim_pad, threadIdx.x & 63);
}

// ---- losses out of the tiles' statistics --------------------------------------------------------------------
// 16 rows per block and step, 64 threads per row over the vocabulary tiles.  A grid of one block takes all rows and adds
// their losses up as well (total != null): up to 64 rows, 4 steps of at most 2 us, against 4.8 us of the launch that more
// rows take for it.  4 to 5 us in all, reads one after the other rather than bytes.
constexpr int kLossParts = 64, kLossSteps = 4;

__device__ inline void merge(float& top, float& sum, float2 o) {
  const float m = fmaxf(top, o.x), ref = m == -INFINITY ? 0.f : m;
  sum = sum * exp_of(top - ref) + o.y * exp_of(o.x - ref);
  top = m;
}

__device__ inline void sum_losses(const float* row_loss, int count, float* total, int mean) {
  __shared__ double sums[16];
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

__global__ __launch_bounds__(1024) void lce_loss_kernel(const float2* partial, int tiles, long long row_pad,
                                                        LceState st, float* losses, float* row_loss, float* total,
                                                        int mean) {
  const int count = st.head[0];
  const int col = threadIdx.x & 15, part = threadIdx.x >> 4;
  __shared__ float2 red[kLossParts][16];
  for (int r0 = blockIdx.x * 16; r0 < count; r0 += gridDim.x * 16) {
    const int r = r0 + col;
    float top = -INFINITY, sum = 0.f;
    if (r < count) {
      const float2* from = partial + r;
      for (int t0 = part; t0 < tiles; t0 += kLossParts * kLossSteps) {
        float2 o[kLossSteps];
#pragma unroll
        for (int k = 0; k < kLossSteps; ++k)
          o[k] = t0 + kLossParts * k < tiles ? from[(long long)(t0 + kLossParts * k) * row_pad]
                                             : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < kLossSteps; ++k) merge(top, sum, o[k]);
      }
      // the 4 threads of this row in the wave
      for (int d = 16; d < 64; d <<= 1) merge(top, sum, make_float2(__shfl_xor(top, d), __shfl_xor(sum, d)));
    }
    red[part][col] = make_float2(top, sum);
    __syncthreads();
    if (part == 0 && r < count) {
      for (int i = 4; i < kLossParts; i += 4) merge(top, sum, red[i][col]);
      const float lse = st.label[r] < 0 ? __builtin_nanf("") : top + logf(sum);
      const float loss = lse - st.zlab[r];
      st.lse[r] = lse;
      row_loss[r] = loss;
      if (losses) losses[st.index[r]] = loss;
    }
    __syncthreads();
  }
  if (total) sum_losses(row_loss, count, total, mean);
}

// sum or mean of the kept rows' losses, in float64 and in a fixed order.  (A launch of its own, 4.8 us: one block telling the
// last of the others by a counter needs every block's writes out of its XCD's L2 first, which took 50 us with fences;
// with every value written through 7.2 us for losses and total, as much as it saves where few rows are scored.)
__global__ __launch_bounds__(1024) void lce_total_kernel(const float* row_loss, LceState st, float* total, int mean) {
  sum_losses(row_loss, st.head[0], total, mean);
}

// dh: the splits' sums, times g, to every row's place; zeros for ignored rows.  A wave takes 256 columns of a row.  Reads what
// the splits wrote, 8 loads in flight: 480 kept rows of 1280 11.5 us, 4500 18.5.
struct DhidArgs {
  const float* acc;
  SplitRule rule;
  long long row_pad;
  int rows, dim, dim_pad, share;
  LceState st;
  const float* upstream;
  int reduction, out_f32;
  void* out;
};

template <typename T>
__global__ __launch_bounds__(256) void lce_dhid_kernel(const DhidArgs p) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int d = (blockIdx.y * 64 + (threadIdx.x & 63)) * 4;
  if (n >= p.rows || d >= p.dim) return;
  const int r = p.st.slot[n], count = p.st.head[0];
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (r >= 0) {
    const int splits = dhid_splits(p.rule, min(count - r / p.share * p.share, p.share));
    const bool none = p.reduction == WFE_REDUCE_NONE;
    float g = none ? 1.f / Elem<T>::kScale : *p.upstream * (1.f / Elem<T>::kScale);
    if (p.reduction == WFE_REDUCE_MEAN) g /= (float)count;
    const int e = none ? weight_e(p.upstream[n]) : 0;
    const float* from = p.acc + (long long)r * p.dim_pad + d;
    const long long step = p.row_pad * p.dim_pad;
#pragma unroll 8
    for (int i = 0; i < splits; ++i) s += *reinterpret_cast<const f32x4*>(from + i * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __builtin_amdgcn_ldexpf(s[i] * g, e);
  }
  const long long at = (long long)n * p.dim + d;
  const bool whole = (p.dim & 3) == 0;
  if (p.out_f32) {
    float* out = static_cast<float*>(p.out) + at;
    if (whole) *reinterpret_cast<f32x4*>(out) = s;
    else
      for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = s[e];
  } else {
    T* out = static_cast<T*>(p.out) + at;
    T x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<T>(s[e]);
    if (whole) __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), x, sizeof x);
    else
      for (int e = 0; e < 4 && d + e < p.dim; ++e) out[e] = x[e];
  }
}

// ---- host side ----------------------------------------------------------------------------------------------
// The tiles.  What bounds the large products is the clock under the matrix instructions' power (2.0 - 2.2 GHz of 2.4): z of
// 4096 x 1280 x 65536 bfloat16 takes 652 us (1054 TFLOP/s), the library's product of that shape 645, and zeros less than
// either.  A step of 32 of a 256 x 256 tile takes 0.785 us on its CU and a tile 7.7 us more (the first fetches, the
// results), so that tiles of 192, 224 or 320 columns cost more per product and won only where they saved a round of all CUs.
// Four K tiles in LDS (128 KB): with the two groups of waves taking turns no wave waits for a fetch.
using Large = Cfg<256, 256, 4, 2, 4, 1>;
// float32: six products for one, and 44 vector instructions per fragment to split it, from registers that 256 x 256 results
// would not leave.  z and gradients of 280 x 384 x 51866: 85 and 160 us; tiles of 128 x 256 with eight waves, one half splitting
// while the other multiplies: 100 and 202.
using Float = Cfg<128, 128, 2, 2, 2, 2>;
// The statistics of few rows, a read of W.  In 2-byte types in 128-byte pieces of its rows; 1280 x 51866, 133 MB:
// 16 rows 21 us (6.3 TB/s, part of it out of the caches), 24 with the large tile's quarter strip; 40 rows, two strips: 26 and 24.
using Stream = Cfg<128, 32, 4, 1, 3, 2, 2>;
// float32, 7 rows: 55 us, 57 with the tile above; 32 rows of 384: 20 and 21.  (Gradients of few rows take the usual tiles:
// 7 rows of 1280 68 us, narrow ones 71; float32 142, narrow ones 165.)
using FloatFew = Cfg<256, 32, 4, 1, 2, 2>;
template <typename T> using Tile = std::conditional_t<sizeof(T) == 4, Float, Large>;
template <typename T> using FewTile = std::conditional_t<sizeof(T) == 4, FloatFew, Stream>;

constexpr int kStatsRows = 128;                // fewest vocabulary rows of a tile: room for the statistics
// What one block of d takes; two are held.  Smaller ones are more launches of fewer tiles each, larger ones leave the cache
// that a block's two products read it from (gradients of 4500 x 1280 x 51866 bfloat16: 32 MB 2.30 ms, 128 MB 1.72, 512 MB
// 2.06).  A block is all rows of a piece of the vocabulary where that makes the piece wide enough: with narrow ones DWEI's
// tiles, all rows long, are few, and a piece is to be so wide that the three products of a launch keep all CUs busy 1.25
// times as long as one tile of DWEI takes.  More rows than that are cut into equal shares, over which DWEI's sums are kept in
// float32, and blocks may be twice as large, fewer shares then reading and writing those sums (loss and gradients of
// 28672 x 256 x 51866 bfloat16: 4.2 ms, with 128 MB 5.2; 7168 x 64: 0.86 and 0.97).  So d never takes more than 512 MB.
constexpr long long kBlockBytes = 128ll << 20;

long long up(long long x, long long to) { return (x + to - 1) / to * to; }

struct Plan {
  int size, ke, dim_pad;
  long long row_pad;
  bool copy_weight;
  int piece, pieces, splits;
  int share, shares;            // rows of a block
  // offsets into the workspace
  long long weighted, weight, partial, row_loss, prob[2], acc, wacc, top, bytes;
};

template <class C>
int tiles_of(long long x, bool a) { return (int)((x + (a ? C::BA : C::BB) - 1) / (a ? C::BA : C::BB)); }

Plan make_plan(const wfe_linear_ce& d, const void* weight, bool backward, int grads) {
  Plan p{};
  p.size = d.dtype == WFE_F32 ? 4 : 2;
  p.ke = kKElems;
  p.dim_pad = lce_dim_pad(d);
  p.row_pad = lce_row_pad(d);
  // in place: 16-byte rows of whole 16 bytes, offsets inside a tile in 32 bits
  p.copy_weight = !((d.dim * p.size) % 16 == 0 && (d.weight_stride * p.size) % 16 == 0 &&
                    d.weight_stride * p.size < (1ll << 22) && (reinterpret_cast<uintptr_t>(weight) & 15) == 0);
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long o = at;
    at += up(bytes, 256);
    return o;
  };
  if (p.copy_weight) p.weight = take((long long)d.vocab * p.dim_pad * p.size);
  if (!backward) {
    p.partial = take(up(d.vocab, kStatsRows) / kStatsRows * p.row_pad * 8);
    p.row_loss = take(p.row_pad * 4);
  } else {
    const long long all = up(d.vocab, kLceRowPad);
    const int edge = p.size == 4 ? Float::BB : Large::BB, slots = p.size == 4 ? Float::kSlots : Large::kSlots;
    const long long per_tile = 3 * ((p.dim_pad + edge - 1) / edge);       // tiles of a launch per `edge` of the piece
    const long long wide = (slots * 5 / 4 + per_tile - 1) / per_tile * edge;
    const long long columns = (wide < all ? wide : all) * p.size;
    const long long block = p.row_pad * columns <= kBlockBytes ? kBlockBytes : 2 * kBlockBytes;
    const long long most = block / columns / kLceRowPad * kLceRowPad;
    p.shares = (int)((p.row_pad + most - 1) / most);              // (`wide` is 27392 at most, `most` 2304 at least where it cuts)
    p.share = (int)up((p.row_pad + p.shares - 1) / p.shares, kLceRowPad);      // shares of one size, pieces of one size
    p.shares = (int)((p.row_pad + p.share - 1) / p.share);
    const long long piece = block / ((long long)p.share * p.size) / kLceRowPad * kLceRowPad;
    p.pieces = (int)((all + piece - 1) / piece);
    p.piece = (int)up((all + p.pieces - 1) / p.pieces, kLceRowPad);
    p.pieces = (int)((all + p.piece - 1) / p.piece);
    if ((grads & WFE_GRAD_WEIGHT) && d.reduction == WFE_REDUCE_NONE) {
      p.weighted = take(p.row_pad * p.dim_pad * p.size);
      p.top = take(4);
    }
    p.prob[0] = take((long long)p.share * p.piece * p.size);
    p.prob[1] = p.pieces * p.shares > 1 ? take((long long)p.share * p.piece * p.size) : p.prob[0];
    if ((grads & WFE_GRAD_WEIGHT) && p.shares > 1) p.wacc = take((long long)p.piece * p.dim_pad * 4);
    if (grads & WFE_GRAD_HIDDEN) {
      const long long one = p.row_pad * p.dim_pad * 4;
      // partial sums of dh: 64 MB; or up to 4 parts in 512 MB, behind which the tiles of one part fill the CUs twice
      const long long most = (64ll << 20) / one, parts = (512ll << 20) / one;
      p.splits = (int)(most > 64 ? 64 : most >= 4 ? most : parts > 4 ? 4 : parts > 1 ? parts : 1);
      p.acc = take(p.splits * one);
    }
  }
  p.bytes = at;
  return p;
}

#define LCE_TRY(expr)                      \
  do {                                     \
    const hipError_t e_ = (expr);          \
    if (e_ != hipSuccess) return e_;       \
  } while (0)

template <typename T, auto KERNEL, class C, class A>
hipError_t launch(const A& args, long long blocks, hipStream_t stream) {
  static unsigned long long done = 0;           // a bit per device: more than 64 KB of LDS has been asked for
  int device = 0;
  LCE_TRY(hipGetDevice(&device));
  const unsigned long long bit = 1ull << (device & 63);
  if (!(__atomic_load_n(&done, __ATOMIC_RELAXED) & bit)) {
    LCE_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize,
                                (kLdsBytes<T, C>)));
    __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  }
  if (blocks * C::kThreads > 0xffffffffll) return hipErrorInvalidValue;
  KERNEL<<<dim3((unsigned)blocks), dim3(C::kThreads), kLdsBytes<T, C>, stream>>>(args);
  return hipGetLastError();
}

template <typename T>
hipError_t pad_weight(const wfe_linear_ce& d, const Plan& p, const void* weight, char* ws, hipStream_t stream) {
  lce_pad_weight_kernel<T><<<dim3((d.vocab + 3) / 4), dim3(256), 0, stream>>>(
      static_cast<const T*>(weight), d.weight_stride, reinterpret_cast<T*>(ws + p.weight), d.dim, p.dim_pad, d.vocab);
  return hipGetLastError();
}

TileArgs tile_args(const wfe_linear_ce& d, const Plan& p, const void* weight, char* ws, const LceState& st) {
  TileArgs a{};
  a.hidden = a.weighted = st.packed;
  a.weight = p.copy_weight ? ws + p.weight : weight;
  a.weight_ld = p.copy_weight ? p.dim_pad : d.weight_stride;
  a.weight_cols = p.copy_weight ? p.dim_pad : d.dim;
  a.dim = d.dim;
  a.dim_pad = p.dim_pad;
  a.piece = a.vocab = d.vocab;
  a.row_pad = p.row_pad;
  a.share = (int)p.row_pad;
  a.head = st.head;
  a.label = st.label;
  a.zlab = st.zlab;
  a.lse = st.lse;
  a.index = st.index;
  return a;
}

// The most blocks that the strips of up to `rows` rows take with `tiles` tiles each
template <class C>
long long strip_blocks(long long tiles, int64_t rows) {
  return up(tiles * tiles_of<C>(rows, false), 8) + (Strips<C>::kNarrow ? up(tiles, 8) : 0);
}

template <typename T, class C>
hipError_t stats(const wfe_linear_ce& d, const TileArgs& a, int* tiles, hipStream_t stream) {
  static_assert(C::BA >= kStatsRows, "room for the statistics");
  *tiles = tiles_of<C>(d.vocab, true);
  return launch<T, lce_logits_kernel<T, C, kStats>, C>(a, strip_blocks<C>(*tiles, d.rows), stream);
}

template <typename T>
hipError_t forward(const wfe_linear_ce& d, const void* hidden, const void* weight, const void* labels, float* loss,
                   void* state, char* ws, hipStream_t stream) {
  const Plan p = make_plan(d, weight, false, 0);
  const LceState st = lce_state(state, d);
  const bool none = d.reduction == WFE_REDUCE_NONE;
  const int mean = d.reduction == WFE_REDUCE_MEAN;
  PackArgs k{};
  k.labels = labels;
  k.label_bits = d.label_bits;
  k.rows = (int)d.rows;
  k.inner = (int)(d.inner < d.rows ? d.inner : d.rows > 0 ? d.rows : 1);
  k.outer_stride = d.outer_stride;
  k.inner_stride = d.inner_stride;
  k.ignore_index = d.ignore_index;
  k.dim = d.dim;
  k.dim_pad = p.dim_pad;
  k.vocab = d.vocab;
  k.per_block = (int)up(d.rows > 0 ? (d.rows + 1023) / 1024 : 1, kPackRows);      // at most 1024 blocks
  k.hidden = hidden;
  k.st = st;
  k.losses = none ? loss : nullptr;
  const long long blocks = d.rows > 0 ? (d.rows + k.per_block - 1) / k.per_block : 1;
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool wide = d.dim == p.dim_pad && reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && d.outer_stride % kVec == 0 &&
                    d.inner_stride % kVec == 0;
  if (wide) lce_pack_kernel<T, true><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(k);
  else lce_pack_kernel<T, false><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(k);
  LCE_TRY(hipGetLastError());
  if (p.copy_weight) LCE_TRY(pad_weight<T>(d, p, weight, ws, stream));
  TileArgs a = tile_args(d, p, weight, ws, st);
  a.partial = reinterpret_cast<float2*>(ws + p.partial);
  int tiles = 0;
  if (d.rows > FewTile<T>::BB) LCE_TRY((stats<T, Tile<T>>(d, a, &tiles, stream)));
  else if (d.rows > 0) LCE_TRY((stats<T, FewTile<T>>(d, a, &tiles, stream)));
  float* row_loss = reinterpret_cast<float*>(ws + p.row_loss);
  float* total = none ? nullptr : loss;
  const bool one = d.rows <= 64;
  lce_loss_kernel<<<dim3((unsigned)(one ? 1 : (d.rows + 15) / 16)), dim3(1024), 0, stream>>>(
      a.partial, tiles, p.row_pad, st, none ? loss : nullptr, row_loss, one ? total : nullptr, mean);
  LCE_TRY(hipGetLastError());
  if (total && !one) lce_total_kernel<<<dim3(1), dim3(1024), 0, stream>>>(row_loss, st, total, mean);
  return hipGetLastError();
}

template <typename T>
hipError_t gradients(const wfe_linear_ce& d, const Plan& p, GradArgs& g, char* ws, hipStream_t stream) {
  using C = Tile<T>;
  // DWEI reads whole K tiles of rows, which PROB's narrowest strip has to have written
  static_assert(C::KS * kKElems <= Strips<C>::kQuarter, "rows of d");
  const char* w = static_cast<const char*>(g.t.weight);
  g.rule.dim_tiles = tiles_of<C>(p.dim_pad, true);
  g.rule.bb = C::BB;
  g.rule.piece_steps = (p.piece + p.ke - 1) / p.ke;
  g.rule.dwei_tiles = g.dwei ? g.rule.dim_tiles * tiles_of<C>(p.piece, false) : 0;
  g.rule.ke = p.ke;
  g.rule.slots = C::kSlots;
  g.rule.most = p.splits;
  g.t.prob_ld = p.piece;
  // Block i: share i % shares of the rows of piece i / shares
  const auto block = [&](int i) {
    TileArgs a = g.t;
    const int v0 = i / p.shares * p.piece, row0 = i % p.shares * p.share;
    a.v0 = v0;
    a.piece = d.vocab - v0 < p.piece ? d.vocab - v0 : p.piece;
    a.weight = w + (long long)v0 * g.t.weight_ld * p.size;
    a.prob = ws + p.prob[i & 1];
    a.row0 = row0;
    a.share = p.share;
    a.hidden = static_cast<const char*>(g.t.hidden) + (long long)row0 * p.dim_pad * p.size;
    a.weighted = static_cast<const char*>(g.t.weighted) + (long long)row0 * p.dim_pad * p.size;
    a.label += row0;
    a.lse += row0;
    a.index += row0;
    a.acc += (long long)row0 * p.dim_pad;
    a.first = v0 == 0;
    a.share_first = row0 == 0;
    a.share_last = i % p.shares == p.shares - 1;
    return a;
  };
  const auto rows_of = [&](const TileArgs& a) { return d.rows - a.row0 < a.share ? d.rows - a.row0 : (int64_t)a.share; };
  const int blocks = p.pieces * p.shares;
  if (d.rows > 0) {
    const TileArgs a = block(0);
    LCE_TRY((launch<T, lce_logits_kernel<T, C, kProb>, C>(a, strip_blocks<C>(tiles_of<C>(a.piece, true), rows_of(a)), stream)));
  }
  const TileArgs base = g.t;
  for (int i = 0; i < blocks; ++i) {           // block i's products beside block i + 1's d
    const TileArgs now = block(i);
    g.next = TileArgs{};
    if (i + 1 < blocks) g.next = block(i + 1);
    const long long grid =
        (g.dwei ? up((long long)g.rule.dim_tiles * tiles_of<C>(now.piece, false), 8) : 0) +
        (g.dhid ? strip_blocks<C>((long long)g.rule.dim_tiles * p.splits, rows_of(now)) : 0) +
        (g.next.piece > 0 ? strip_blocks<C>(tiles_of<C>(g.next.piece, true), rows_of(g.next)) : 0);
    g.t = now;
    if (grid > 0) LCE_TRY((launch<T, lce_grads_kernel<T, C>, C>(g, grid, stream)));
    g.t = base;
  }
  return hipSuccess;
}

template <typename T>
hipError_t backward(const wfe_linear_ce& d, const void* weight, const void* state, const float* upstream,
                    void* grad_hidden, void* grad_weight, char* ws, hipStream_t stream) {
  const int grads = (grad_hidden ? WFE_GRAD_HIDDEN : 0) | (grad_weight ? WFE_GRAD_WEIGHT : 0);
  const Plan p = make_plan(d, weight, true, grads);
  const LceState st = lce_state(const_cast<void*>(state), d);
  if (p.copy_weight) LCE_TRY(pad_weight<T>(d, p, weight, ws, stream));
  GradArgs g{};
  g.t = tile_args(d, p, weight, ws, st);
  g.t.acc = reinterpret_cast<float*>(ws + p.acc);
  g.t.wacc = reinterpret_cast<float*>(ws + p.wacc);
  g.t.grad_weight = grad_weight;
  g.t.grad_f32 = d.grad_weight_dtype == WFE_F32;
  g.t.mean = d.reduction == WFE_REDUCE_MEAN;
  g.t.factor = upstream;
  g.t.own = d.reduction == WFE_REDUCE_NONE ? upstream : nullptr;
  g.dhid = grad_hidden && d.rows > 0;
  g.dwei = grad_weight != nullptr;
  if (g.dwei && d.reduction == WFE_REDUCE_NONE) {
    float* top = reinterpret_cast<float*>(ws + p.top);
    lce_top_kernel<<<dim3(1), dim3(1024), 0, stream>>>(upstream, st, top);
    LCE_TRY(hipGetLastError());
    lce_weigh_kernel<T><<<dim3((unsigned)(p.row_pad / 4)), dim3(256), 0, stream>>>(st.packed, ws + p.weighted, p.dim_pad,
                                                                                st, upstream, top);
    LCE_TRY(hipGetLastError());
    g.t.weighted = ws + p.weighted;
    g.t.factor = top;
  }
  LCE_TRY(gradients<T>(d, p, g, ws, stream));
  if (g.dhid) {
    DhidArgs k{};
    k.acc = g.t.acc;
    k.rule = g.rule;
    k.row_pad = p.row_pad;
    k.rows = (int)d.rows;
    k.dim = d.dim;
    k.dim_pad = p.dim_pad;
    k.share = p.share;
    k.st = st;
    k.upstream = upstream;
    k.reduction = d.reduction;
    k.out_f32 = d.grad_hidden_dtype == WFE_F32;
    k.out = grad_hidden;
    lce_dhid_kernel<T><<<dim3((unsigned)((d.rows + 3) / 4), (d.dim + 255) / 256), dim3(256), 0, stream>>>(k);
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

hipError_t launch_lce_backward(const wfe_linear_ce& d, const void* weight, const void* state, const float* upstream,
                               void* grad_hidden, void* grad_weight, void* workspace, hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  if (d.dtype == WFE_F32) return backward<float>(d, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
  if (d.dtype == WFE_F16) return backward<_Float16>(d, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
  return backward<__bf16>(d, weight, state, upstream, grad_hidden, grad_weight, ws, stream);
}

}  // namespace wfe
