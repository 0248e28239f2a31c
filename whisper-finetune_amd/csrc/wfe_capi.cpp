// wfe_capi.cpp -- the C ABI declared in include/wfe.h.  Thin: argument checks,
// table upload at create time, kernel launches.  No torch types, no exceptions
// across the boundary.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <new>
#include <string>
#include <vector>

#include "../../include/wfe.h"
#include "wfe_capi_util.h"
#include "wfe_kernels.h"
#include "wfe_layout.h"

struct wfe_context {
  wfe_config cfg;
  float* d_dft = nullptr;
  float* d_mel = nullptr;
  wfe::Resolved* d_resolved = nullptr;  // grows on demand
  void* d_cops = nullptr;               // compiled ops, same capacity as d_resolved
  wfe::ChainHead* d_heads = nullptr;    // per utterance of a launch slice
  size_t resolved_cap = 0;
  double* d_noise_meansq = nullptr;     // grows on demand
  size_t noise_cap = 0;
  const float* noise_seen = nullptr;    // noise bank whose mean squares are cached
  const int64_t* noise_off_seen = nullptr;
  int n_noise_seen = 0;
  unsigned mel_mask[14];
  int bank = 0;                         // 1: 80-mel, 2: 128-mel compile-time masks, 0: run-time masks
  std::vector<double> mel_filters;      // (201, n_mel)
  // optional in-stream timing of the two kernels (wfe_kernel_timing)
  bool timing = false;
  std::vector<hipEvent_t> ev_pool;      // triples: before K1, after K1, after K2
  size_t ev_used = 0;
  unsigned* d_peaks = nullptr;              // reverb: max|x|, max|y| per utterance of a slice
  double* d_partials = nullptr;             // resolve pass: per-part sums of the batch slice
  unsigned* d_tickets = nullptr;            // resolve pass: one arrival counter per utterance of the slice, zero between launches
  struct RsTable {
    float* d = nullptr;
    int L = 0, M = 0, taps = 0, k0 = 0;
    // the same filter in the order resample_mfma_kernel reads it (ratios with >= 64 phases), else null
    float* d_frag = nullptr;
    int* d_meta = nullptr;
    int ptiles = 0, kspan = 0, nwaves = 0, group = 1;
  };
  std::map<std::pair<int, int>, RsTable> rs_tables;   // (in_rate, out_rate) -> filter on the device
  float* d_tile_stats = nullptr;            // per-tile minima / maxima of kernel 1, grows on demand
  size_t tile_stats_cap = 0;
  unsigned long long* d_stamps = nullptr;   // diagnostic builds only (wfe_debug_stamps)
  // augmented calls: the resolve pass (HBM-bound) of the second half of a batch runs on this stream under
  // kernel 1 (matrix-bound) of the first half; forked from and joined to the caller's stream with the two events
  // reverberation by FFT (wfe_reverb_fft.hip): twiddle tables, and the spectra of the impulse-response bank last seen
  float2* d_rv_tw = nullptr;
  float2* d_rv_H = nullptr;
  size_t rv_H_cap = 0;                      // float2 elements
  const float* rv_rir_seen = nullptr;
  const int64_t* rv_off_seen = nullptr;
  int rv_n_seen = 0, rv_p_max = 0, rv_max_taps = 0;
  float2* d_rv_ring = nullptr;              // the one-kernel form's ring, or the three-kernel form's Z then Y
  size_t rv_ring_cap = 0;                   // float2 elements
  hipStream_t side = nullptr;
  hipEvent_t ev_fork = nullptr, ev_join = nullptr;
  std::vector<char> ev_cont;                // per event triple: 1 = second half of the same call (not a launch of its own)
  int out_kind = WFE_OUT_F32;               // wfe_set_output_format
  int tune = 0;                             // WFE_TUNE (experiments)
  size_t rv_ws_limit = (size_t)4 << 30;     // bytes of FFT-reverb workspace per launch (WFE_RV_WS_MB): larger batches run in slices
  std::string err;
};

namespace {

constexpr int kMaxBatchPerLaunch = 4096;
thread_local std::string g_create_err;

// ---- wfe_logmel_static's scratch (include/wfe.h): the per-tile statistics kernel 1 leaves for
// kernel 2, for callers that cannot allocate.  One copy of the array per GPU, at its own address;
// host code never uses the array's name as an address, only the pointer hipGetSymbolAddress
// returned for the device (g_scratch_ptr, filled by wfe_create with that device current).
constexpr int kStaticTiles = 256 * 47;           // 256 utterances of 30 s (47 tiles of 64 frames each)
static __device__ __align__(256) float scratch[kStaticTiles * wfe::kTileStats];   // 1 732 608 bytes
constexpr int kMaxDevices = 64;
float* g_scratch_ptr[kMaxDevices] = {};
std::mutex g_scratch_mu;

// workspace sizes that wfe_create provides up front, so that the hot path of ordinary batches
// never reaches hipFree / hipMalloc (larger requests still grow on demand)
constexpr size_t kInitTiles = (size_t)kMaxBatchPerLaunch * 47;     // 4096 utterances of 30 s
constexpr size_t kInitOps = (size_t)kMaxBatchPerLaunch * 4;
constexpr size_t kInitNoise = 1024;
constexpr size_t kMaxTimedLaunches = 1 << 16;    // event triples kept while wfe_kernel_timing is on

using wfe::fail;

#define HIP_TRY(h, expr)                                                                 \
  do {                                                                                   \
    hipError_t e_ = (expr);                                                              \
    if (e_ != hipSuccess) return fail(h, WFE_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

using wfe::DeviceGuard;

int check_common(wfe_context* h, const void* wav, const int32_t* lengths, int32_t batch, int32_t n_samples,
                 const void* out) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  if (batch < 0) return fail(h, WFE_ERR_ARG, "batch %d < 0", batch);
  if (batch > 0 && (!wav || !lengths || !out)) return fail(h, WFE_ERR_ARG, "null device pointer");
  if (n_samples <= wfe::kHalf)
    return fail(h, WFE_ERR_ARG, "n_samples %d must exceed n_fft/2 = 200 (reflect padding)", n_samples);
  if (n_samples / wfe::kHop < 1) return fail(h, WFE_ERR_ARG, "n_samples %d gives no frame", n_samples);
  if ((long long)n_samples + wfe::kNfft >= (1LL << 30)) return fail(h, WFE_ERR_ARG, "n_samples too large");
  return WFE_OK;
}

// wav_or_pcm: float32 samples when channels == 0, interleaved int16 otherwise
void fill_args(wfe_context* h, wfe::FrontArgs& a, const void* wav_or_pcm, int channels, const int64_t* offsets,
               const int32_t* lengths, int64_t row_stride, int32_t n_samples) {
  std::memset(&a, 0, sizeof a);
  if (channels > 0) {
    a.pcm = static_cast<const short*>(wav_or_pcm);
    a.channels = channels;
  } else {
    a.wav = static_cast<const float*>(wav_or_pcm);
    a.channels = 1;
  }
  a.offsets = reinterpret_cast<const long long*>(offsets);
  a.lengths = lengths;
  a.row_stride = row_stride;
  a.n_samples = n_samples;
  a.n_frames = n_samples / wfe::kHop;
  a.n_mel = h->cfg.n_mel;
  a.dft_tab = h->d_dft;
  a.mel_tab = h->d_mel;
  std::memcpy(a.mel_mask, h->mel_mask, sizeof a.mel_mask);
  a.tile_stats = h->d_tile_stats;
  a.stamps = h->d_stamps;
  a.tune = h->tune;
}

// Batch sliced into launches of at most kMaxBatchPerLaunch utterances.
struct Slice {
  int begin, count;
};
std::vector<Slice> slices(int batch, int limit = kMaxBatchPerLaunch) {
  std::vector<Slice> v;
  for (int b = 0; b < batch; b += limit) v.push_back({b, batch - b < limit ? batch - b : limit});
  return v;
}

int ensure_aug_workspace(wfe_context* h, size_t total_ops, const float* noise, const int64_t* noise_off, int n_noise,
                         hipStream_t stream) {
  if (total_ops > h->resolved_cap) {
    if (h->d_resolved) HIP_TRY(h, hipFree(h->d_resolved));
    h->d_resolved = nullptr;
    h->resolved_cap = 0;
    size_t cap = total_ops < 1024 ? 1024 : total_ops * 2;
    HIP_TRY(h, hipMalloc(&h->d_resolved, cap * sizeof(wfe::Resolved)));
    if (h->d_cops) HIP_TRY(h, hipFree(h->d_cops));
    h->d_cops = nullptr;
    HIP_TRY(h, hipMalloc(&h->d_cops, cap * wfe::kCopBytes));
    h->resolved_cap = cap;
  }
  if (!h->d_partials)
    HIP_TRY(h, hipMalloc(&h->d_partials, sizeof(double) * 2 * wfe::kResolveParts * kMaxBatchPerLaunch));
  if (!h->d_tickets) {
    HIP_TRY(h, hipMalloc(&h->d_tickets, sizeof(unsigned) * kMaxBatchPerLaunch));
    HIP_TRY(h, hipMemsetAsync(h->d_tickets, 0, sizeof(unsigned) * kMaxBatchPerLaunch, stream));
  }
  if (!h->d_heads) HIP_TRY(h, hipMalloc(&h->d_heads, sizeof(wfe::ChainHead) * kMaxBatchPerLaunch));
  if (n_noise > 0) {
    if ((size_t)n_noise > h->noise_cap) {
      if (h->d_noise_meansq) HIP_TRY(h, hipFree(h->d_noise_meansq));
      h->d_noise_meansq = nullptr;
      h->noise_cap = 0;
      h->noise_seen = nullptr;
      size_t cap = (size_t)n_noise < 64 ? 64 : (size_t)n_noise * 2;
      HIP_TRY(h, hipMalloc(&h->d_noise_meansq, cap * wfe::kNoiseParts * sizeof(double)));
      h->noise_cap = cap;
    }
    // The mean squares of a bank are computed ONCE and kept while the caller keeps passing the same bank
    // (same clip pointer, same offsets pointer, same count): 0.012 ms and a read of the whole bank per call
    // otherwise.  A caller that refills a bank IN PLACE says so with wfe_noise_bank_changed.
    // (The kernel that fills them and the resolve pass that reads them run on the caller's streams in call
    // order; a handle's calls are ordered by contract, include/wfe.h.)
    if (h->noise_seen != noise || h->noise_off_seen != noise_off || h->n_noise_seen != n_noise) {
      HIP_TRY(h, wfe::launch_noise_meansq(noise, reinterpret_cast<const long long*>(noise_off), n_noise,
                                          h->d_noise_meansq, stream));
      h->noise_seen = noise;
      h->noise_off_seen = noise_off;
      h->n_noise_seen = n_noise;
    }
  }
  return WFE_OK;
}

int run_frontend(wfe_context* h, const void* wav, int channels, const int64_t* offsets, const int32_t* lengths,
                 int64_t row_stride, int32_t batch, int32_t n_samples, const wfe_aug_op* ops, const int32_t* op_begin, int64_t total_ops,
                 const float* noise, const int64_t* noise_off, int32_t n_noise, float* out, int mode, void* stream_) {
  int rc = check_common(h, wav, lengths, batch, n_samples, out);
  if (rc != WFE_OK) return rc;
  if (batch == 0) return WFE_OK;
  const bool aug = ops != nullptr;
  if (aug && !op_begin) return fail(h, WFE_ERR_ARG, "ops given without op_begin");
  if (aug && n_noise > 0 && (!noise || !noise_off)) return fail(h, WFE_ERR_ARG, "n_noise > 0 without a noise bank");
  if (aug && (total_ops < 0 || n_noise < 0)) return fail(h, WFE_ERR_ARG, "negative total_ops / n_noise");
  if (offsets == nullptr && row_stride < 0) return fail(h, WFE_ERR_ARG, "negative row_stride");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard(h->cfg.device);
  if (!guard.ok) return fail(h, WFE_ERR_HIP, "hipSetDevice(%d) failed", h->cfg.device);
  if (aug) {
    rc = ensure_aug_workspace(h, (size_t)total_ops, noise, noise_off, n_noise, stream);
    if (rc != WFE_OK) return rc;
  }
  const int T = n_samples / wfe::kHop;
  if (mode == 0) {
    const size_t per_slice = (size_t)(batch < kMaxBatchPerLaunch ? batch : kMaxBatchPerLaunch) *
                             ((T + wfe::kBlockFrames - 1) / wfe::kBlockFrames) * wfe::kTileStats;
    if (per_slice > h->tile_stats_cap) {
      if (h->d_tile_stats) HIP_TRY(h, hipFree(h->d_tile_stats));
      h->d_tile_stats = nullptr;
      h->tile_stats_cap = 0;
      HIP_TRY(h, hipMalloc(&h->d_tile_stats, per_slice * 2 * sizeof(float)));
      h->tile_stats_cap = per_slice * 2;
    }
  }
  const long long per_clip = (mode == 1) ? (long long)wfe::kNfreq * T : (long long)h->cfg.n_mel * T;
  const int nblk = (T + wfe::kBlockFrames - 1) / wfe::kBlockFrames;
  // One part of a launch slice: utterances [begin, begin + count) of the batch, whose per-utterance workspaces
  // (tile statistics, chain heads, partial sums, tickets) start at utterance `ws` of the slice's.
  auto part_args = [&](int begin, int count, int ws) {
    wfe::FrontArgs a;
    fill_args(h, a, wav, channels, offsets, lengths, row_stride, n_samples);
    // slice by pointer arithmetic so that blockIdx.y indexes the part
    if (offsets) a.offsets += begin;
    else if (a.pcm) a.pcm += (long long)begin * row_stride;
    else a.wav += (long long)begin * row_stride;
    a.lengths += begin;
    // (16-bit log-mel output: `out` counts 2-byte elements)
    const int kind = (mode == 0) ? h->out_kind : WFE_OUT_F32;
    a.out = (kind == WFE_OUT_F32) ? out + (long long)begin * per_clip
                                   : reinterpret_cast<float*>(reinterpret_cast<unsigned short*>(out) + (long long)begin * per_clip);
    a.out_kind = kind;
    if (a.tile_stats) a.tile_stats += (long long)ws * nblk * wfe::kTileStats;
    if (aug) {
      a.ops = ops;
      a.op_begin = op_begin + begin;
      a.noise = noise;
      a.noise_off = reinterpret_cast<const long long*>(noise_off);
      a.noise_meansq = h->d_noise_meansq;
      a.resolved = h->d_resolved;
      a.cops = h->d_cops;
      a.heads = h->d_heads + ws;
    }
    return a;
  };
  auto resolve_part = [&](const wfe::FrontArgs& a, int count, int ws, hipStream_t st) {
    return wfe::launch_resolve(a, count, h->d_partials + (size_t)ws * 2 * wfe::kResolveParts, h->d_tickets + ws, st);
  };
  // kernel 1 + clamp of one part, bracketed by timing events when asked for
  auto transform_part = [&](const wfe::FrontArgs& a, int count, bool continuation) -> int {
    hipEvent_t* ev = nullptr;
    if (h->timing && h->ev_used / 3 < kMaxTimedLaunches) {   // (beyond the cap launches go untimed)
      if (h->ev_used + 3 > h->ev_pool.size()) {
        for (int i = 0; i < 3; ++i) {
          hipEvent_t e;
          HIP_TRY(h, hipEventCreate(&e));
          h->ev_pool.push_back(e);
        }
        h->ev_cont.resize(h->ev_pool.size() / 3, 0);
      }
      ev = &h->ev_pool[h->ev_used];
      h->ev_cont[h->ev_used / 3] = continuation ? 1 : 0;
      h->ev_used += 3;
      HIP_TRY(h, hipEventRecord(ev[0], stream));
    }
    HIP_TRY(h, wfe::launch_frontend(a, count, mode, aug, h->bank, stream));
    if (ev) HIP_TRY(h, hipEventRecord(ev[1], stream));
    if (mode == 0)
      HIP_TRY(h, wfe::launch_clamp(a.out, a.out_kind, a.tile_stats, count, h->cfg.n_mel, T, stream));
    if (ev) HIP_TRY(h, hipEventRecord(ev[2], stream));
    return WFE_OK;
  };
  for (const Slice& s : slices(batch)) {
    // Experiment (WFE_TUNE & 128; OFF by default): augmented slices as two halves, the resolve pass -- a second read of
    // the waveform, HBM-bound -- of half B on the side stream under kernel 1 -- matrix-bound -- of half A (VERDICT r2
    // #3a).  Measured on 256 x 30 s: 0.853 ms per call against 0.810 in one part (kernel 1 0.732 against 0.672): the
    // augmented kernel holds every vector register of its SIMDs, so the resolve workgroups do not run UNDER it but
    // take whole workgroup slots from it, and two half-size launches have two ramps and two tails.
    const bool split = aug && s.count >= 64 && h->side && (h->tune & 128);
    const int na = split ? (s.count + 1) / 2 : s.count, nb = s.count - na;
    const wfe::FrontArgs a = part_args(s.begin, na, 0);
    if (aug) HIP_TRY(h, resolve_part(a, na, 0, stream));
    if (!split) {
      rc = transform_part(a, na, false);
      if (rc != WFE_OK) return rc;
      continue;
    }
    const wfe::FrontArgs b = part_args(s.begin + na, nb, na);
    HIP_TRY(h, hipEventRecord(h->ev_fork, stream));                      // B's inputs are ready where A's are
    HIP_TRY(h, hipStreamWaitEvent(h->side, h->ev_fork, 0));
    HIP_TRY(h, resolve_part(b, nb, na, h->side));
    HIP_TRY(h, hipEventRecord(h->ev_join, h->side));
    rc = transform_part(a, na, false);
    if (rc != WFE_OK) return rc;
    HIP_TRY(h, hipStreamWaitEvent(stream, h->ev_join, 0));               // the side stream rejoins the caller's
    rc = transform_part(b, nb, true);
    if (rc != WFE_OK) return rc;
  }
  return WFE_OK;
}

}  // namespace

int wfe::fail(wfe_context* h, int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  if (h) h->err = buf; else g_create_err = buf;
  return code;
}

extern "C" {

const char* wfe_version(void) { return "wfe-amd 0.1 (gfx950)"; }

int wfe_create(const wfe_config* cfg, wfe_handle* out) {
  if (!cfg || !out) return fail(nullptr, WFE_ERR_ARG, "null argument");
  *out = nullptr;
  if (cfg->n_fft != wfe::kNfft || cfg->hop_length != wfe::kHop)
    return fail(nullptr, WFE_ERR_ARG, "only n_fft=400 / hop_length=160 are implemented (got %d / %d)", cfg->n_fft,
                cfg->hop_length);
  if (cfg->sampling_rate != 16000)
    return fail(nullptr, WFE_ERR_SAMPLING, "only sampling_rate=16000 is implemented (got %d)", cfg->sampling_rate);
  if (cfg->n_mel < 1 || cfg->n_mel > wfe::kMaxMel)
    return fail(nullptr, WFE_ERR_ARG, "n_mel %d outside 1..%d", cfg->n_mel, wfe::kMaxMel);
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1)
    return fail(nullptr, WFE_ERR_HIP, "no HIP device available: the front end has no CPU path");
  if (cfg->device < 0 || cfg->device >= ndev)
    return fail(nullptr, WFE_ERR_ARG, "device %d outside 0..%d", cfg->device, ndev - 1);
  hipDeviceProp_t prop;
  if (hipGetDeviceProperties(&prop, cfg->device) != hipSuccess)
    return fail(nullptr, WFE_ERR_HIP, "hipGetDeviceProperties failed");
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    return fail(nullptr, WFE_ERR_HIP, "device %d is %s; this library is built for gfx950 only", cfg->device,
                prop.gcnArchName);

  wfe_context* h = new (std::nothrow) wfe_context();
  if (!h) return fail(nullptr, WFE_ERR_ALLOC, "out of host memory");
  h->cfg = *cfg;
  if (const char* t = std::getenv("WFE_TUNE")) h->tune = std::atoi(t);
  if (const char* t = std::getenv("WFE_RV_WS_MB"))
    if (std::atoll(t) > 0) h->rv_ws_limit = (size_t)std::atoll(t) << 20;
  h->mel_filters.resize((size_t)wfe::kNfreq * cfg->n_mel);
  wfe_build_mel_filters(cfg->n_mel, h->mel_filters.data());
  std::vector<float> dft((size_t)wfe::kDftTableFloats), mel((size_t)wfe::kMelTableFloats);
  wfe_build_dft_table(dft.data());
  wfe_build_mel_table(cfg->n_mel, mel.data(), h->mel_mask);
  if (cfg->n_mel == 80 && std::memcmp(h->mel_mask, wfe::kMelMask80, sizeof h->mel_mask) == 0) h->bank = 1;
  if (cfg->n_mel == 128 && std::memcmp(h->mel_mask, wfe::kMelMask128, sizeof h->mel_mask) == 0) h->bank = 2;


  DeviceGuard guard(cfg->device);
  hipError_t e = guard.ok ? hipSuccess : hipErrorInvalidDevice;
  if (e == hipSuccess) e = hipMalloc(&h->d_dft, dft.size() * sizeof(float));
  if (e == hipSuccess) e = hipMalloc(&h->d_mel, mel.size() * sizeof(float));
  if (e == hipSuccess) e = hipMemcpy(h->d_dft, dft.data(), dft.size() * sizeof(float), hipMemcpyHostToDevice);
  if (e == hipSuccess) e = hipMemcpy(h->d_mel, mel.data(), mel.size() * sizeof(float), hipMemcpyHostToDevice);
  // every workspace of the hot path at the size of an ordinary batch (<= 4096 utterances of 30 s,
  // <= 4 ops each, <= 1024 noise clips): ~11 MB; only larger requests ever reallocate
  if (e == hipSuccess) e = hipMalloc(&h->d_tile_stats, kInitTiles * wfe::kTileStats * sizeof(float));
  if (e == hipSuccess) h->tile_stats_cap = kInitTiles * wfe::kTileStats;
  if (e == hipSuccess) e = hipMalloc(&h->d_resolved, kInitOps * sizeof(wfe::Resolved));
  if (e == hipSuccess) e = hipMalloc(&h->d_cops, kInitOps * wfe::kCopBytes);
  if (e == hipSuccess) h->resolved_cap = kInitOps;
  if (e == hipSuccess) e = hipMalloc(&h->d_partials, sizeof(double) * 2 * wfe::kResolveParts * kMaxBatchPerLaunch);
  if (e == hipSuccess) e = hipMalloc(&h->d_tickets, sizeof(unsigned) * kMaxBatchPerLaunch);
  if (e == hipSuccess) e = hipMemset(h->d_tickets, 0, sizeof(unsigned) * kMaxBatchPerLaunch);
  if (e == hipSuccess) e = hipMalloc(&h->d_heads, sizeof(wfe::ChainHead) * kMaxBatchPerLaunch);
  if (e == hipSuccess) e = hipMalloc(&h->d_noise_meansq, kInitNoise * wfe::kNoiseParts * sizeof(double));
  if (e == hipSuccess) h->noise_cap = kInitNoise;
  if (e == hipSuccess) e = hipMalloc(&h->d_peaks, sizeof(unsigned) * 2 * kMaxBatchPerLaunch);
  if (e == hipSuccess) e = hipStreamCreateWithFlags(&h->side, hipStreamNonBlocking);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&h->ev_fork, hipEventDisableTiming);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&h->ev_join, hipEventDisableTiming);
  // wfe_logmel_static: this device's copy of the static scratch array (once per device)
  if (e == hipSuccess && cfg->device < kMaxDevices) {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (!g_scratch_ptr[cfg->device]) {
      float* ptr = nullptr;
      e = hipGetSymbolAddress(reinterpret_cast<void**>(&ptr), HIP_SYMBOL(scratch));
      if (e == hipSuccess) g_scratch_ptr[cfg->device] = ptr;
    }
  }
  if (e != hipSuccess) {
    fail(nullptr, WFE_ERR_HIP, "wfe_create: %s", hipGetErrorString(e));
    wfe_destroy(h);
    return WFE_ERR_HIP;
  }
  *out = h;
  return WFE_OK;
}

int wfe_destroy(wfe_handle h) {
  if (!h) return WFE_OK;
  DeviceGuard guard(h->cfg.device);
  if (h->d_dft) (void)hipFree(h->d_dft);
  if (h->d_mel) (void)hipFree(h->d_mel);
  if (h->d_resolved) (void)hipFree(h->d_resolved);
  if (h->d_cops) (void)hipFree(h->d_cops);
  if (h->d_heads) (void)hipFree(h->d_heads);
  if (h->d_noise_meansq) (void)hipFree(h->d_noise_meansq);
  if (h->d_tile_stats) (void)hipFree(h->d_tile_stats);
  for (auto& kv : h->rs_tables)
  {
    if (kv.second.d) (void)hipFree(kv.second.d);
    if (kv.second.d_frag) (void)hipFree(kv.second.d_frag);
    if (kv.second.d_meta) (void)hipFree(kv.second.d_meta);
  }
  if (h->d_partials) (void)hipFree(h->d_partials);
  if (h->d_tickets) (void)hipFree(h->d_tickets);
  if (h->d_rv_tw) (void)hipFree(h->d_rv_tw);
  if (h->d_rv_H) (void)hipFree(h->d_rv_H);
  if (h->d_rv_ring) (void)hipFree(h->d_rv_ring);
  if (h->d_peaks) (void)hipFree(h->d_peaks);
  for (hipEvent_t e : h->ev_pool) (void)hipEventDestroy(e);
  if (h->ev_fork) (void)hipEventDestroy(h->ev_fork);
  if (h->ev_join) (void)hipEventDestroy(h->ev_join);
  if (h->side) (void)hipStreamDestroy(h->side);
  delete h;
  return WFE_OK;
}

const char* wfe_last_error(wfe_handle h) { return h ? h->err.c_str() : g_create_err.c_str(); }

int wfe_mel_filters(wfe_handle h, double* host_out) {
  if (!h || !host_out) return fail(h, WFE_ERR_ARG, "null argument");
  std::memcpy(host_out, h->mel_filters.data(), h->mel_filters.size() * sizeof(double));
  return WFE_OK;
}

#ifdef WFE_STAMPS
// Diagnostic library only (not declared in include/wfe.h, not built by default).
int wfe_debug_stamps(wfe_handle h, unsigned long long* device_buf) {
  if (!h) return WFE_ERR_ARG;
  h->d_stamps = device_buf;
  return WFE_OK;
}
#endif

int wfe_set_output_format(wfe_handle h, int32_t format) {
  if (!h) return WFE_ERR_ARG;
  if (format != WFE_OUT_F32 && format != WFE_OUT_F16 && format != WFE_OUT_BF16)
    return fail(h, WFE_ERR_ARG, "output format %d is not WFE_OUT_F32 / WFE_OUT_F16 / WFE_OUT_BF16", format);
  h->out_kind = format;
  return WFE_OK;
}

int wfe_noise_bank_changed(wfe_handle h) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  h->noise_seen = nullptr;
  h->noise_off_seen = nullptr;
  h->n_noise_seen = 0;
  h->rv_rir_seen = nullptr;              // (and the impulse-response bank's cached spectra)
  h->rv_off_seen = nullptr;
  h->rv_n_seen = 0;
  return WFE_OK;
}

int wfe_kernel_timing(wfe_handle h, int32_t enable) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  h->timing = enable != 0;
  h->ev_used = 0;
  return WFE_OK;
}

int wfe_kernel_times(wfe_handle h, double* frontend_ms, double* clamp_ms, int64_t* launches) {
  if (!h || !frontend_ms || !clamp_ms || !launches) return fail(h, WFE_ERR_ARG, "null argument");
  DeviceGuard guard(h->cfg.device);
  double f = 0.0, c = 0.0;
  for (size_t i = 0; i + 2 < h->ev_used; i += 3) {
    HIP_TRY(h, hipEventSynchronize(h->ev_pool[i + 2]));
    float t1 = 0.f, t2 = 0.f;
    HIP_TRY(h, hipEventElapsedTime(&t1, h->ev_pool[i], h->ev_pool[i + 1]));
    HIP_TRY(h, hipEventElapsedTime(&t2, h->ev_pool[i + 1], h->ev_pool[i + 2]));
    f += t1;
    c += t2;
  }
  int64_t n = 0;
  for (size_t i = 0; i < h->ev_used / 3; ++i) n += h->ev_cont[i] ? 0 : 1;    // the halves of one call count once
  *frontend_ms = f;
  *clamp_ms = c;
  *launches = n;
  h->ev_used = 0;
  return WFE_OK;
}

int wfe_logmel(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths, int64_t row_stride,
               int32_t batch, int32_t n_samples, float* out, void* stream) {
  return run_frontend(h, wav, 0, offsets, lengths, row_stride, batch, n_samples, nullptr, nullptr, 0, nullptr, nullptr,
                      0, out, 0, stream);
}

// wfe_logmel for callers that cannot allocate: the same two kernels, their per-tile statistics in
// this GPU's copy of the static `scratch` array instead of the handle's workspace.  No hipMalloc,
// hipFree, event or host container on this path.
int wfe_logmel_static(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths,
                      int64_t row_stride, int32_t batch, int32_t n_samples, float* out, void* stream_) {
  int rc = check_common(h, wav, lengths, batch, n_samples, out);
  if (rc != WFE_OK) return rc;
  if (batch == 0) return WFE_OK;
  if (offsets == nullptr && row_stride < 0) return fail(h, WFE_ERR_ARG, "negative row_stride");
  const int T = n_samples / wfe::kHop;
  const long long tiles = (long long)batch * ((T + wfe::kBlockFrames - 1) / wfe::kBlockFrames);
  if (batch > kMaxBatchPerLaunch || tiles > kStaticTiles)
    return fail(h, WFE_ERR_ARG,
                "wfe_logmel_static: batch %d x %d tiles of 64 frames = %lld tiles exceeds the static scratch "
                "(%d tiles = 256 utterances of 30 s; at most %d utterances): split the batch or use wfe_logmel",
                batch, (T + wfe::kBlockFrames - 1) / wfe::kBlockFrames, tiles, kStaticTiles, kMaxBatchPerLaunch);
  if (h->cfg.device >= kMaxDevices || !g_scratch_ptr[h->cfg.device])
    return fail(h, WFE_ERR_HIP, "wfe_logmel_static: no scratch address for device %d", h->cfg.device);
  float* const stats = g_scratch_ptr[h->cfg.device];      // never the array's name: that is not a device address
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard(h->cfg.device);
  if (!guard.ok) return fail(h, WFE_ERR_HIP, "hipSetDevice(%d) failed", h->cfg.device);
  wfe::FrontArgs a;
  fill_args(h, a, wav, 0, offsets, lengths, row_stride, n_samples);
  a.tile_stats = stats;      // every tile's 12 statistics are written by kernel 1 before kernel 2 reads them: nothing to clear
  a.out = out;
  a.out_kind = h->out_kind;
  HIP_TRY(h, wfe::launch_frontend(a, batch, 0, false, h->bank, stream));
  HIP_TRY(h, wfe::launch_clamp(a.out, a.out_kind, stats, batch, h->cfg.n_mel, T, stream));
  return WFE_OK;
}

int wfe_power_spectrum(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths,
                       int64_t row_stride, int32_t batch, int32_t n_samples, float* out, void* stream) {
  return run_frontend(h, wav, 0, offsets, lengths, row_stride, batch, n_samples, nullptr, nullptr, 0, nullptr, nullptr,
                      0, out, 1, stream);
}

int wfe_augment_logmel(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths,
                       int64_t row_stride, int32_t batch, int32_t n_samples, const wfe_aug_op* ops,
                       const int32_t* op_begin, int64_t total_ops, const float* noise, const int64_t* noise_offsets,
                       int32_t n_noise, float* out, void* stream) {
  if (h && (!ops || !op_begin)) return fail(h, WFE_ERR_ARG, "ops / op_begin must not be null");
  return run_frontend(h, wav, 0, offsets, lengths, row_stride, batch, n_samples, ops, op_begin, total_ops, noise,
                      noise_offsets, n_noise, out, 0, stream);
}

int wfe_logmel_pcm16(wfe_handle h, const int16_t* pcm, const int64_t* offsets, const int32_t* lengths,
                     int64_t row_stride, int32_t channels, int32_t batch, int32_t n_samples, const wfe_aug_op* ops,
                     const int32_t* op_begin, int64_t total_ops, const float* noise, const int64_t* noise_offsets,
                     int32_t n_noise, float* out, void* stream) {
  if (h && (channels < 1 || channels > 256)) return fail(h, WFE_ERR_ARG, "channels %d outside 1..256", channels);
  if (!ops) return run_frontend(h, pcm, channels, offsets, lengths, row_stride, batch, n_samples, nullptr, nullptr, 0,
                                nullptr, nullptr, 0, out, 0, stream);
  return run_frontend(h, pcm, channels, offsets, lengths, row_stride, batch, n_samples, ops, op_begin, total_ops, noise,
                      noise_offsets, n_noise, out, 0, stream);
}

int wfe_augment_waveform(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths,
                         int64_t row_stride, int32_t batch, int32_t n_samples, const wfe_aug_op* ops,
                         const int32_t* op_begin, int64_t total_ops, const float* noise, const int64_t* noise_offsets,
                         int32_t n_noise, float* out, int32_t* out_lengths, void* stream_) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  if (batch < 0 || n_samples < 1) return fail(h, WFE_ERR_ARG, "bad batch / n_samples");
  if (batch == 0) return WFE_OK;
  if (!wav || !lengths || !out || !ops || !op_begin) return fail(h, WFE_ERR_ARG, "null device pointer");
  if (n_noise > 0 && (!noise || !noise_offsets)) return fail(h, WFE_ERR_ARG, "n_noise > 0 without a noise bank");
  if (total_ops < 0 || n_noise < 0) return fail(h, WFE_ERR_ARG, "negative total_ops / n_noise");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard(h->cfg.device);
  if (!guard.ok) return fail(h, WFE_ERR_HIP, "hipSetDevice(%d) failed", h->cfg.device);
  int rc = ensure_aug_workspace(h, (size_t)total_ops, noise, noise_offsets, n_noise, stream);
  if (rc != WFE_OK) return rc;
  for (const Slice& s : slices(batch)) {
    wfe::FrontArgs a;
    fill_args(h, a, wav, 0, offsets, lengths, row_stride, n_samples);
    if (offsets) a.offsets += s.begin; else a.wav += (long long)s.begin * row_stride;
    a.lengths += s.begin;
    a.ops = ops;
    a.op_begin = op_begin + s.begin;
    a.noise = noise;
    a.noise_off = reinterpret_cast<const long long*>(noise_offsets);
    a.noise_meansq = h->d_noise_meansq;
    a.resolved = h->d_resolved;
      a.cops = h->d_cops;
      a.heads = h->d_heads;
    HIP_TRY(h, wfe::launch_resolve(a, s.count, h->d_partials, h->d_tickets, stream));
    HIP_TRY(h, wfe::launch_waveform(a, s.count, out + (long long)s.begin * n_samples,
                                    out_lengths ? out_lengths + s.begin : nullptr, stream));
  }
  return WFE_OK;
}

int wfe_reverb(wfe_handle h, const float* wav, const int64_t* offsets, const int32_t* lengths, int64_t row_stride,
               int32_t batch, const float* rir, const int64_t* rir_offsets, int32_t n_rir, const int32_t* rir_index,
               float* out, int64_t out_stride, void* stream_) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  if (batch < 0) return fail(h, WFE_ERR_ARG, "batch %d < 0", batch);
  if (out_stride < 1 || out_stride >= (1LL << 30)) return fail(h, WFE_ERR_ARG, "bad out_stride");
  if (offsets == nullptr && row_stride < 0) return fail(h, WFE_ERR_ARG, "negative row_stride");
  if (batch == 0) return WFE_OK;
  if (!wav || !lengths || !out || !rir_index) return fail(h, WFE_ERR_ARG, "null device pointer");
  if (n_rir < 0 || (n_rir > 0 && (!rir || !rir_offsets))) return fail(h, WFE_ERR_ARG, "n_rir without impulse responses");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard(h->cfg.device);
  if (!guard.ok) return fail(h, WFE_ERR_HIP, "hipSetDevice(%d) failed", h->cfg.device);
  if (!h->d_peaks) HIP_TRY(h, hipMalloc(&h->d_peaks, sizeof(unsigned) * 2 * kMaxBatchPerLaunch));
  // Long impulse responses: the FFT form (wfe_reverb_fft.hip).  The bank's lengths are read back ONCE per bank (same
  // pointers and count; wfe_noise_bank_changed also forgets this one), its spectra are computed once and kept.
  // (WFE_TUNE & 8192: the direct sum for every length, for A/B and the tests.)
  bool use_fft = false;
  if (n_rir > 0 && !(h->tune & 8192)) {
    if (h->rv_rir_seen != rir || h->rv_off_seen != rir_offsets || h->rv_n_seen != n_rir) {
      h->rv_rir_seen = nullptr;                        // (nothing is cached until all of this has succeeded)
      h->rv_off_seen = nullptr;
      h->rv_n_seen = 0;
      h->rv_max_taps = 0;
      std::vector<int64_t> off((size_t)n_rir + 1);
      HIP_TRY(h, hipMemcpyAsync(off.data(), rir_offsets, off.size() * sizeof(int64_t), hipMemcpyDeviceToHost, stream));
      HIP_TRY(h, hipStreamSynchronize(stream));
      int max_taps = 0;
      for (int j = 0; j < n_rir; ++j) {
        const int64_t t = off[j + 1] - off[j];
        if (t < 0 || t >= (1LL << 30)) return fail(h, WFE_ERR_ARG, "impulse response %d: bad length", j);
        if (t > max_taps) max_taps = (int)t;
      }
      h->rv_p_max = (max_taps + wfe::kRvFftN / 2 - 1) / (wfe::kRvFftN / 2);
      if (max_taps >= wfe::kRvFftMinTaps) {
        if (!h->d_rv_tw) {
          std::vector<float2> tw(128);
          const double w = -2.0 * 3.14159265358979323846 / (double)wfe::kRvFftN;
          for (int i = 0; i < 64; ++i) {
            tw[i] = float2{(float)std::cos(w * 64.0 * i), (float)std::sin(w * 64.0 * i)};
            tw[64 + i] = float2{(float)std::cos(w * i), (float)std::sin(w * i)};
          }
          HIP_TRY(h, hipMalloc(&h->d_rv_tw, tw.size() * sizeof(float2)));
          HIP_TRY(h, hipMemcpy(h->d_rv_tw, tw.data(), tw.size() * sizeof(float2), hipMemcpyHostToDevice));
        }
        const size_t need = (size_t)n_rir * h->rv_p_max * wfe::kRvFftN;
        if (need > h->rv_H_cap) {
          if (h->d_rv_H) HIP_TRY(h, hipFree(h->d_rv_H));
          h->d_rv_H = nullptr;
          h->rv_H_cap = 0;
          HIP_TRY(h, hipMalloc(&h->d_rv_H, need * sizeof(float2)));
          h->rv_H_cap = need;
        }
        HIP_TRY(h, wfe::launch_reverb_spectra(rir, reinterpret_cast<const long long*>(rir_offsets), n_rir, h->rv_p_max,
                                              h->d_rv_tw, h->d_rv_H, stream));
      }
      h->rv_rir_seen = rir;
      h->rv_off_seen = rir_offsets;
      h->rv_n_seen = n_rir;
      h->rv_max_taps = max_taps;
    }
    use_fft = h->rv_max_taps >= wfe::kRvFftMinTaps;
  }
  // The three-kernel form keeps two spectra per block pair in its workspace (0.26 MB per second of audio): batches
  // whose workspace would exceed rv_ws_limit (4 GB: 512 utterances of 30 s) run in slices of as many as fit.
  int limit = kMaxBatchPerLaunch;
  if (use_fft && h->rv_p_max >= 3) {
    const long long blocks = (out_stride + wfe::kRvFftN / 2 - 1) / (wfe::kRvFftN / 2) + 1;
    const size_t per_utt = (size_t)(2 * ((blocks + 1) / 2) + h->rv_p_max - 1) * wfe::kRvFftN * sizeof(float2);
    const size_t fit = h->rv_ws_limit / per_utt;
    if (fit < (size_t)limit) limit = fit < 1 ? 1 : (int)fit;
  }
  for (const Slice& s : slices(batch, limit)) {
    wfe::ReverbArgs a;
    std::memset(&a, 0, sizeof a);
    a.wav = offsets ? wav : wav + (long long)s.begin * row_stride;
    a.offsets = offsets ? reinterpret_cast<const long long*>(offsets) + s.begin : nullptr;
    a.lengths = lengths + s.begin;
    a.row_stride = row_stride;
    a.rir = rir;
    a.rir_off = reinterpret_cast<const long long*>(rir_offsets);
    a.rir_index = rir_index + s.begin;
    a.out = out + (long long)s.begin * out_stride;
    a.out_stride = out_stride;
    a.peaks = h->d_peaks;
    a.tune = h->tune;
    HIP_TRY(h, hipMemsetAsync(h->d_peaks, 0, sizeof(unsigned) * 2 * kMaxBatchPerLaunch, stream));
    if (use_fft) {
      const int B = wfe::kRvFftN / 2, P = h->rv_p_max;
      const long long blocks = (out_stride + B - 1) / B + 1;                  // blocks of the full convolution per utterance, at most
      // three kernels from three partitions on (the products read every spectrum once instead of once per partition),
      // while the products' LDS fits; (WFE_TUNE & 16384: the one-kernel form for every length)
      const bool three = P >= 3 && !(h->tune & 16384) && wfe::reverb_mac_lds_bytes(P) <= wfe::kRvMacLdsMax;
      int segments = 1, seg_blocks = 1;
      const long long kh_cap = (blocks + 1) / 2, pairs_cap = kh_cap + P - 1;
      size_t need;
      if (three) {
        need = (size_t)s.count * (size_t)(pairs_cap + kh_cap) * wfe::kRvFftN;
      } else {
        // cut into segments so that a launch has ~4 workgroups per CU (a segment starts P - 1 pairs early)
        long long want = (1024 + s.count - 1) / s.count;
        const long long most = blocks / (2LL * P + 2) > 0 ? blocks / (2LL * P + 2) : 1;
        if (want > most) want = most;
        if (want < 1) want = 1;
        seg_blocks = (int)((blocks + want - 1) / want);
        segments = (int)((blocks + seg_blocks - 1) / seg_blocks);
        need = (size_t)s.count * segments * P * wfe::kRvFftN;
      }
      if (need > h->rv_ring_cap) {
        if (h->d_rv_ring) HIP_TRY(h, hipFree(h->d_rv_ring));
        h->d_rv_ring = nullptr;
        h->rv_ring_cap = 0;
        HIP_TRY(h, hipMalloc(&h->d_rv_ring, need * sizeof(float2)));
        h->rv_ring_cap = need;
      }
      HIP_TRY(h, hipMemsetAsync(a.out, 0, (size_t)s.count * out_stride * sizeof(float), stream));   // rows are zero behind their lengths
      if (three) {
        float2* Z = h->d_rv_ring;
        float2* Y = Z + (size_t)s.count * (size_t)pairs_cap * wfe::kRvFftN;
        HIP_TRY(h, wfe::launch_reverb_fft3(a, s.count, h->d_rv_tw, h->d_rv_H, P, Z, (int)pairs_cap, Y, (int)kh_cap, stream));
      } else {
        HIP_TRY(h, wfe::launch_reverb_fft(a, s.count, h->d_rv_tw, h->d_rv_H, P, h->d_rv_ring, segments, seg_blocks, stream));
      }
      HIP_TRY(h, wfe::launch_reverb_scale(a, s.count, stream));
      continue;
    }
    HIP_TRY(h, wfe::launch_reverb(a, s.count, stream));
  }
  return WFE_OK;
}

// The polyphase filter [taps][L] as the A operand of resample_mfma_kernel: T[p][c] = table[c - floor(p M / L)][(p M) mod L]
// (zero outside the taps), per tile of 16 phases only the k-steps (4 columns) its band touches, rounded to quads;
// lane l of a fragment holds row l % 16, column l / 16 of the k-step, 4 consecutive k-steps per float4.
// r > 1: groups of r L outputs (ratios with few phases: the same matrix, r times as tall, rows p >= L repeat the
// columns p mod L shifted by whole input steps).
static void build_resample_fragments(const std::vector<float>& table, int L0, int M0, int r, int taps,
                                     std::vector<float>& frag, std::vector<int>& meta, int& kspan) {
  const int L = L0 * r, M = M0 * r;
  const int ptiles = (L + 15) / 16;
  meta.assign(3 * (size_t)ptiles, 0);
  frag.clear();
  kspan = 0;
  long long foff = 0;
  for (int pt = 0; pt < ptiles; ++pt) {
    const int p0 = 16 * pt, p1 = (p0 + 16 < L ? p0 + 16 : L) - 1;
    const long long c_lo = (long long)p0 * M / L, c_hi = (long long)p1 * M / L + taps;   // [c_lo, c_hi)
    const int kb_lo = (int)(c_lo / 4), kb_hi = (int)((c_hi + 3) / 4), nq = (kb_hi - kb_lo + 3) / 4;
    meta[3 * pt] = kb_lo;
    meta[3 * pt + 1] = nq;
    meta[3 * pt + 2] = (int)foff;
    frag.resize((size_t)(foff + nq) * 256, 0.f);
    for (int q = 0; q < nq; ++q)
      for (int lane = 0; lane < 64; ++lane)
        for (int i = 0; i < 4; ++i) {
          const int p = p0 + (lane & 15);
          const long long c = 4LL * (kb_lo + 4 * q + i) + (lane >> 4);
          float v = 0.f;
          if (p < L) {
            const long long j = c - (long long)p * M / L;
            if (j >= 0 && j < taps) v = table[(size_t)j * L0 + (size_t)((long long)p * M0 % L0)];
          }
          frag[((size_t)(foff + q) * 64 + lane) * 4 + i] = v;
        }
    foff += nq;
    if (4 * (kb_lo + 4 * nq) > kspan) kspan = 4 * (kb_lo + 4 * nq);
  }
}

int wfe_resample(wfe_handle h, const void* in, int32_t pcm_channels, const int64_t* offsets, const int32_t* lengths,
                 int64_t row_stride, int32_t batch, int32_t in_rate, int32_t out_rate, float* out, int64_t out_stride,
                 const int32_t* out_lengths, void* stream_) {
  if (!h) return fail(nullptr, WFE_ERR_ARG, "null handle");
  if (batch < 0) return fail(h, WFE_ERR_ARG, "batch %d < 0", batch);
  if (pcm_channels < 0 || pcm_channels > 256) return fail(h, WFE_ERR_ARG, "pcm_channels %d outside 0..256", pcm_channels);
  if (in_rate < 1 || out_rate < 1) return fail(h, WFE_ERR_ARG, "bad rates %d -> %d", in_rate, out_rate);
  if (out_stride < 1 || out_stride >= (1LL << 30)) return fail(h, WFE_ERR_ARG, "bad out_stride");
  if (offsets == nullptr && row_stride < 0) return fail(h, WFE_ERR_ARG, "negative row_stride");
  if (batch == 0) return WFE_OK;
  if (!in || !lengths || !out || !out_lengths) return fail(h, WFE_ERR_ARG, "null device pointer");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard(h->cfg.device);
  if (!guard.ok) return fail(h, WFE_ERR_HIP, "hipSetDevice(%d) failed", h->cfg.device);
  auto key = std::make_pair((int)in_rate, (int)out_rate);
  auto it = h->rs_tables.find(key);
  if (it == h->rs_tables.end()) {
    wfe_context::RsTable t;
    if (wfe_resample_geometry(in_rate, out_rate, &t.L, &t.M, &t.taps, &t.k0) != WFE_OK)
      return fail(h, WFE_ERR_ARG, "unsupported resampling ratio %d -> %d", in_rate, out_rate);
    if (t.L > wfe::kRsChunkFloats)
      return fail(h, WFE_ERR_ARG, "resampling %d -> %d needs %d filter phases (> %d)", in_rate, out_rate, t.L,
                  wfe::kRsChunkFloats);
    if (t.taps + 2 + 256LL * t.M / t.L + 1 > wfe::kRsSpanFloats)
      return fail(h, WFE_ERR_ARG, "resampling %d -> %d decimates too steeply (%d taps)", in_rate, out_rate, t.taps);
    std::vector<float> host((size_t)t.taps * t.L);
    wfe_build_resample_table(in_rate, out_rate, host.data());
    HIP_TRY(h, hipMalloc(&t.d, host.size() * sizeof(float)));
    hipError_t e = hipMemcpy(t.d, host.data(), host.size() * sizeof(float), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      (void)hipFree(t.d);
      return fail(h, WFE_ERR_HIP, "resample table upload: %s", hipGetErrorString(e));
    }
    {                                                  // the GEMM form: the table as matrix-core fragments
      std::vector<float> frag;
      std::vector<int> meta;
      t.group = t.L >= 64 ? 1 : (160 + t.L - 1) / t.L;  // few phases: groups of about 160 outputs
      build_resample_fragments(host, t.L, t.M, t.group, t.taps, frag, meta, t.kspan);
      t.ptiles = (t.L * t.group + 15) / 16;
      int best = 1 << 30;
      for (int nw = 8; nw <= 16; ++nw) {               // waves per workgroup: the least idle tile slots, then the most waves
        const int waste = (t.ptiles + nw - 1) / nw * nw - t.ptiles;
        if (waste <= best) best = waste, t.nwaves = nw;
      }
      if (t.ptiles < 8) t.nwaves = t.ptiles;
      // round 3: 12 waves = three per SIMD, tiles dealt to the SIMDs in turn and the last ptiles % 4 tiles split
      // along the groups (resample_mfma_kernel); WFE_TUNE & 256 keeps round 2's count and assignment, for A/B
      else if (!(h->tune & 256)) t.nwaves = 12;
      if (15LL * t.M * t.group + t.kspan + 1024 <= wfe::kRsMfmaSpanFloats && frag.size() <= (64u << 20)) {
        hipError_t e1 = hipMalloc(&t.d_frag, frag.size() * sizeof(float));
        hipError_t e2 = e1 == hipSuccess ? hipMalloc(&t.d_meta, meta.size() * sizeof(int)) : e1;
        if (e2 == hipSuccess) e2 = hipMemcpy(t.d_frag, frag.data(), frag.size() * sizeof(float), hipMemcpyHostToDevice);
        if (e2 == hipSuccess) e2 = hipMemcpy(t.d_meta, meta.data(), meta.size() * sizeof(int), hipMemcpyHostToDevice);
        if (e2 != hipSuccess) {
          if (t.d_frag) (void)hipFree(t.d_frag);
          if (t.d_meta) (void)hipFree(t.d_meta);
          (void)hipFree(t.d);
          return fail(h, WFE_ERR_HIP, "resample fragment upload: %s", hipGetErrorString(e2));
        }
      }
    }
    it = h->rs_tables.emplace(key, t).first;
  }
  const wfe_context::RsTable& t = it->second;
  // outputs per workgroup: their input span (opb * M / L + taps + 1) must fit the LDS buffer
  long long opb = ((long long)wfe::kRsSpanFloats - t.taps - 2) * t.L / t.M;
  opb = opb / 256 * 256;
  if (opb > 2048) opb = 2048;
  if (opb < 256) return fail(h, WFE_ERR_ARG, "resampling %d -> %d decimates too steeply", in_rate, out_rate);
  for (const Slice& s : slices(batch)) {
    wfe::ResampleArgs a;
    std::memset(&a, 0, sizeof a);
    if (pcm_channels > 0) {
      a.pcm = static_cast<const short*>(in);
      a.channels = pcm_channels;
      if (!offsets) a.pcm += (long long)s.begin * row_stride;
    } else {
      a.wav = static_cast<const float*>(in);
      a.channels = 1;
      if (!offsets) a.wav += (long long)s.begin * row_stride;
    }
    a.offsets = offsets ? reinterpret_cast<const long long*>(offsets) + s.begin : nullptr;
    a.lengths = lengths + s.begin;
    a.row_stride = row_stride;
    a.out = out + (long long)s.begin * out_stride;
    a.out_stride = out_stride;
    a.out_lengths = out_lengths + s.begin;
    a.table = t.d;
    a.L = t.L;
    a.M = t.M;
    a.taps = t.taps;
    a.k0 = t.k0;
    a.out_per_block = (int)opb;
    a.tune = h->tune;
    a.frag = t.d_frag;
    a.frag_meta = t.d_meta;
    a.ptiles = t.ptiles;
    a.kspan = t.kspan;
    a.nwaves = t.nwaves;
    a.frag_group = t.group;
    HIP_TRY(h, wfe::launch_resample(a, s.count, stream));
  }
  return WFE_OK;
}

}  // extern "C"
