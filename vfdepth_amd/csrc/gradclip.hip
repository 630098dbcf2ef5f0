// Global gradient norm over a list of tensors, and clipping to a largest norm: what stands between the backward
// pass and the optimizer's step (trainer/vfdepth_trainer.py:63-66) when training.max_grad_norm is set.
//   n = sqrt(sum_t sum_i g_ti^2)      (or max_ti |g_ti|),      c = min(1, max_norm / (n + 1e-6)),      g <- c g
// The list travels in the kernels' arguments (pointer, length and type of up to CLIP_NORM_CAP tensors a launch), so
// a call copies nothing to the device and can be captured.  Squares are summed in fp64: an fp32 square overflows
// from |g| = 1.9e19 on.  The norm of 200 M values, call after call, reads fp32 at 5.1 TB/s (158 us) and bf16, with twice
// the conversions and fp64 operations a byte, at 4.2 (96 us).
// Every sum has a fixed order (block-strided chunks, one partial per block, no atomics): the same gradients give
// the same bits.
#include <algorithm>
#include <utility>
#include <vector>

#include "vfd_common.h"

namespace vfd {

constexpr int CLIP_CH = 16384;             // elements of one chunk: 64 per thread, 16 (fp32) or 8 (bf16) 16-B loads in flight
constexpr int CLIP_NORM_CAP = 176;         // tensors of one launch: the table stays under 4 KB of kernel arguments
constexpr int CLIP_SCALE_CAP = 120;
// Blocks of a launch at most.  Registers (86 and 94 a lane) leave five on a CU at a time, 1280 in all; the others start as
// those end.  200 M values, 291 tensors, with 1280, 2048 and 4096: bf16 norm 92, 96, 96 us, norm and scaling in place 313,
// 252, 277; fp32 155, 158, 157 and 588, 502, 523.
constexpr int CLIP_GRID = 2048;
constexpr int CLIP_MAX_PARTS = 4 * CLIP_GRID;

template <int CAP>
struct ClipTable {
  const void* p[CAP];
  long long n[CAP];
  int start[CAP];                          // first chunk of each tensor
  uint8_t dt[CAP];
  int count, chunks;
};
struct ScaleTable {
  ClipTable<CLIP_SCALE_CAP> t;
  void* out[CLIP_SCALE_CAP];
  uint8_t odt[CLIP_SCALE_CAP];
};
static_assert(sizeof(ClipTable<CLIP_NORM_CAP>) <= 3900 && sizeof(ScaleTable) <= 3900, "kernel arguments are 4 KB");

// Eight elements at any element boundary: gradients are often views of one all-reduce bucket, so neither their
// starts nor their lengths are multiples of 16 bytes.
template <typename T>
using clip_v8 __attribute__((ext_vector_type(8), aligned(sizeof(T)))) = T;

// The tensor of a chunk: every lane compares its share of the first chunks, kept in registers over all chunks
template <int CAP>
struct ClipFind {
  static constexpr int NS = (CAP + 63) / 64;
  int s[NS];
  __device__ __forceinline__ ClipFind(const ClipTable<CAP>& t) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int i = k * 64 + (int)(threadIdx.x & 63);
      s[k] = i < t.count ? t.start[i] : 0x7fffffff;
    }
  }
  __device__ __forceinline__ int operator()(int chunk) const {
    int c = 0;
#pragma unroll
    for (int k = 0; k < NS; ++k) c += __popcll(__ballot(s[k] <= chunk));
    return __builtin_amdgcn_readfirstlane(c - 1);
  }
};

template <bool INF>
__device__ __forceinline__ double norm_join(double a, double b) {
  if constexpr (INF) return a != a ? a : (b != b ? b : (a > b ? a : b));       // NaN wins
  return a + b;
}

template <bool INF>
__device__ __forceinline__ void norm_take(double& acc, float x) {
  const double v = (double)x;
  if constexpr (INF)
    acc = norm_join<true>(acc, v < 0 ? -v : v);
  else
    acc = fma(v, v, acc);
}

// Joined over the 256 threads of a block, in a fixed order; valid in every thread.
template <bool INF>
__device__ __forceinline__ double norm_block(double v, double* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = norm_join<INF>(v, __shfl_xor(v, off, WAVE));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return norm_join<INF>(norm_join<INF>(lds[0], lds[1]), norm_join<INF>(lds[2], lds[3]));
}

template <bool INF>
__device__ __forceinline__ double norm_total(const double* __restrict__ part, int parts, double* lds) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) v = norm_join<INF>(v, part[i]);
  v = norm_block<INF>(v, lds);
  return INF ? v : sqrt(v);
}

template <bool INF, typename T>
__device__ __forceinline__ void norm_chunk(double& acc, const T* __restrict__ p, long long left) {
  if (left >= CLIP_CH) {
    clip_v8<T> v[CLIP_CH / 2048];
#pragma unroll
    for (int u = 0; u < CLIP_CH / 2048; ++u) v[u] = *reinterpret_cast<const clip_v8<T>*>(p + u * 2048 + threadIdx.x * 8);
#pragma unroll
    for (int u = 0; u < CLIP_CH / 2048; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) norm_take<INF>(acc, (float)v[u][j]);
  } else {
    for (int i = threadIdx.x; i < (int)left; i += 256) norm_take<INF>(acc, ld1(p + i));
  }
}

template <bool INF>
__global__ __launch_bounds__(256) void grad_norm_k(const ClipTable<CLIP_NORM_CAP> t, double* __restrict__ part) {
  __shared__ double lds[4];
  const ClipFind<CLIP_NORM_CAP> find(t);
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int i = find(c);
    const long long at = (long long)(c - t.start[i]) * CLIP_CH, left = t.n[i] - at;
    if (t.dt[i] == 0)
      norm_chunk<INF>(acc, (const float*)t.p[i] + at, left);
    else
      norm_chunk<INF>(acc, (const __bf16*)t.p[i] + at, left);
  }
  const double s = norm_block<INF>(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// parts > CLIP_MAX_PARTS (thousands of tensors): joined to one before every scaling block would read them all
template <bool INF>
__global__ __launch_bounds__(256) void grad_norm_join_k(const double* __restrict__ part, int parts, double* __restrict__ one) {
  __shared__ double lds[4];
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) v = norm_join<INF>(v, part[i]);
  v = norm_block<INF>(v, lds);
  if (threadIdx.x == 0) *one = v;
}

template <bool INF>
__global__ __launch_bounds__(256) void grad_norm_fin_k(const double* __restrict__ part, int parts, float* __restrict__ norm) {
  __shared__ double lds[4];
  const double n = norm_total<INF>(part, parts, lds);
  if (threadIdx.x == 0) *norm = (float)n;
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* p, O* o, long long left, float c) {
  if (left >= CLIP_CH) {
    clip_v8<T> v[CLIP_CH / 2048];
#pragma unroll
    for (int u = 0; u < CLIP_CH / 2048; ++u) v[u] = *reinterpret_cast<const clip_v8<T>*>(p + u * 2048 + threadIdx.x * 8);
#pragma unroll
    for (int u = 0; u < CLIP_CH / 2048; ++u) {
      clip_v8<O> r;
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = (O)((float)v[u][j] * c);
      *reinterpret_cast<clip_v8<O>*>(o + u * 2048 + threadIdx.x * 8) = r;
    }
  } else {
    for (int i = threadIdx.x; i < (int)left; i += 256) st1(o + i, ld1(p + i) * c);
  }
}

// Every block joins the partials itself (16 KB of L2 at most per table, in one order for all: the same factor
// everywhere) instead of waiting for a launch that does; with nothing to clip an in-place call ends there.
template <bool INF>
__global__ __launch_bounds__(256) void grad_scale_k(const ScaleTable t, const double* __restrict__ part, int parts,
                                                    double max_norm, int in_place, float* __restrict__ norm) {
  __shared__ double lds[4];
  const double n = norm_total<INF>(part, parts, lds);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double f = max_norm / (n + 1e-6);
  const float c = f > 1.0 ? 1.f : (float)f;                  // NaN stays NaN: a bad gradient must not pass unseen
  if (in_place && c == 1.f) return;
  const ClipFind<CLIP_SCALE_CAP> find(t.t);
  for (int b = blockIdx.x; b < t.t.chunks; b += gridDim.x) {
    const int k = t.t.chunks - 1 - b;                        // backwards: what the norm read last is still cached
    const int i = find(k);
    const long long at = (long long)(k - t.t.start[i]) * CLIP_CH, left = t.t.n[i] - at;
    const void* p = t.t.p[i];
    void* o = t.out[i];
    if (t.t.dt[i] == 0) {
      if (t.odt[i] == 0) scale_chunk((const float*)p + at, (float*)o + at, left, c);
      else scale_chunk((const float*)p + at, (__bf16*)o + at, left, c);
    } else {
      if (t.odt[i] == 0) scale_chunk((const __bf16*)p + at, (float*)o + at, left, c);
      else scale_chunk((const __bf16*)p + at, (__bf16*)o + at, left, c);
    }
  }
}

static int clip_check(const char* what, int n, const void* const* grads, const int64_t* numel, const uint8_t* dt) {
  VFD_REQUIRE(n >= 0 && (n == 0 || (grads && numel && dt)), "%s: bad list", what);
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    VFD_REQUIRE(numel[i] >= 0 && numel[i] < (1ll << 42) && (numel[i] == 0 || grads[i]) && dt[i] <= 1,
                "%s: bad tensor %d", what, i);
    chunks += (numel[i] + CLIP_CH - 1) / CLIP_CH;
    VFD_REQUIRE(chunks < 0x7fffffffll - CLIP_GRID, "%s: too many elements", what);
  }
  return VFD_OK;
}

// Written memory must not be met twice: a block would read what another has already scaled.  `r` lists every written
// range, `ro` the ranges that are only read.
static int clip_overlap(const char* what, std::vector<std::pair<uintptr_t, uintptr_t>>& r,
                        std::vector<std::pair<uintptr_t, uintptr_t>>& ro) {
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    VFD_REQUIRE(r[i].first >= r[i - 1].second, "%s: two of the tensors written share memory", what);
  std::sort(ro.begin(), ro.end());
  size_t k = 0;
  uintptr_t far = 0;                                         // end of the furthest range that starts before this one
  for (const auto& w : r) {
    for (; k < ro.size() && ro[k].first < w.second; ++k) far = std::max(far, ro[k].second);
    VFD_REQUIRE(far <= w.first, "%s: an output shares memory with a gradient", what);
  }
  return VFD_OK;
}

// Fill one launch's table from tensor `i` on; returns the first tensor that did not fit.
template <int CAP>
static int clip_fill(ClipTable<CAP>& t, int i, int n, const void* const* grads, const int64_t* numel, const uint8_t* dt,
                     int* which) {
  t.count = t.chunks = 0;
  for (; i < n && t.count < CAP; ++i) {
    if (numel[i] == 0) continue;
    if (which) which[t.count] = i;
    t.p[t.count] = grads[i];
    t.n[t.count] = numel[i];
    t.start[t.count] = t.chunks;
    t.dt[t.count++] = dt[i];
    t.chunks += (int)((numel[i] + CLIP_CH - 1) / CLIP_CH);
  }
  return i;
}

// Blocks of a launch: as many rounds as CLIP_GRID blocks need, then as few blocks as do it in those rounds.
static int clip_grid(int chunks) {
  const int rounds = (chunks + CLIP_GRID - 1) / CLIP_GRID;
  return rounds ? (chunks + rounds - 1) / rounds : 0;
}

static int clip_parts(int n, const int64_t* numel) {
  int parts = 0, count = 0, chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (numel[i] == 0) continue;
    chunks += (int)((numel[i] + CLIP_CH - 1) / CLIP_CH);
    if (++count == CLIP_NORM_CAP) {
      parts += clip_grid(chunks);
      count = chunks = 0;
    }
  }
  return parts + clip_grid(chunks);
}

template <bool INF>
static int norm_launch(int n, const void* const* grads, const int64_t* numel, const uint8_t* dt, double* part, hipStream_t s) {
  ClipTable<CLIP_NORM_CAP> t;
  int parts = 0;
  for (int i = 0; i < n;) {
    i = clip_fill(t, i, n, grads, numel, dt, nullptr);
    if (t.chunks == 0) continue;
    const int grid = clip_grid(t.chunks);
    grad_norm_k<INF><<<grid, 256, 0, s>>>(t, part + parts);
    parts += grid;
  }
  return parts;
}

template <bool INF>
static int clip_run(int n, const void* const* grads, const int64_t* numel, const uint8_t* dt, bool scale, double max_norm,
                    void* const* outs, const uint8_t* odt, float* norm, double* part, hipStream_t s) {
  int parts = norm_launch<INF>(n, grads, numel, dt, part, s);
  if (parts > CLIP_MAX_PARTS) {
    grad_norm_join_k<INF><<<1, 256, 0, s>>>(part, parts, part + parts);
    part += parts;
    parts = 1;
  }
  if (!scale || parts == 0) {
    grad_norm_fin_k<INF><<<1, 256, 0, s>>>(part, parts, norm);
    return fail_launch("grad_norm");
  }
  ScaleTable t;
  int which[CLIP_SCALE_CAP];
  for (int first = (n - 1) / CLIP_SCALE_CAP * CLIP_SCALE_CAP; first >= 0; first -= CLIP_SCALE_CAP) {     // likewise
    clip_fill(t.t, first, std::min(n, first + CLIP_SCALE_CAP), grads, numel, dt, which);
    if (t.t.chunks == 0) continue;
    for (int k = 0; k < t.t.count; ++k) {
      t.out[k] = outs ? outs[which[k]] : const_cast<void*>(t.t.p[k]);
      t.odt[k] = outs ? odt[which[k]] : t.t.dt[k];
    }
    grad_scale_k<INF><<<clip_grid(t.t.chunks), 256, 0, s>>>(t, part, parts, max_norm, outs == nullptr, norm);
    norm = nullptr;                                          // written once
  }
  return fail_launch("clip_grads");
}

}  // namespace vfd

using namespace vfd;

extern "C" {

size_t vfd_grad_norm_workspace(int n, const int64_t* numel) {
  if (n < 0 || (n > 0 && numel == nullptr)) return 0;
  return sizeof(double) * ((size_t)clip_parts(n, numel) + 1);
}

int vfd_grad_norm(int n, const void* const* grads, const int64_t* numel, const uint8_t* dtypes, int inf_norm, float* norm,
                  void* workspace, size_t ws_bytes, void* stream) {
  if (int e = clip_check("grad_norm", n, grads, numel, dtypes)) return e;
  VFD_REQUIRE(norm && workspace && ws_bytes >= vfd_grad_norm_workspace(n, numel), "grad_norm: null output or workspace too small");
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_GRAD_CLIP, s);
  auto run = inf_norm ? clip_run<true> : clip_run<false>;
  return run(n, grads, numel, dtypes, false, 0.0, nullptr, nullptr, norm, (double*)workspace, s);
}

int vfd_clip_grads(int n, const void* const* grads, const int64_t* numel, const uint8_t* dtypes, int inf_norm, double max_norm,
                   void* const* outs, const uint8_t* out_dtypes, float* norm, void* workspace, size_t ws_bytes,
                   void* stream) {
  if (int e = clip_check("clip_grads", n, grads, numel, dtypes)) return e;
  VFD_REQUIRE(max_norm >= 0.0, "clip_grads: max_norm must be >= 0");
  VFD_REQUIRE(norm && workspace && ws_bytes >= vfd_grad_norm_workspace(n, numel), "clip_grads: null output or workspace too small");
  VFD_REQUIRE(outs == nullptr || out_dtypes != nullptr, "clip_grads: outputs without their types");
  for (int i = 0; outs != nullptr && i < n; ++i)
    VFD_REQUIRE((numel[i] == 0 || outs[i]) && out_dtypes[i] <= 1, "clip_grads: bad output %d", i);
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> r, ro;
    r.reserve(n);
    ro.reserve(outs ? n : 0);
    for (int i = 0; i < n; ++i) {
      if (numel[i] == 0) continue;
      const uintptr_t g = (uintptr_t)grads[i], ge = g + (uintptr_t)numel[i] * (dtypes[i] ? 2 : 4);
      if (outs == nullptr) {
        r.emplace_back(g, ge);
      } else {
        const uintptr_t o = (uintptr_t)outs[i];
        ro.emplace_back(g, ge);
        r.emplace_back(o, o + (uintptr_t)numel[i] * (out_dtypes[i] ? 2 : 4));
      }
    }
    if (int e = clip_overlap("clip_grads", r, ro)) return e;
  } catch (...) {
    set_error("clip_grads: out of host memory");
    return VFD_EINVAL;
  }
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_GRAD_CLIP, s);
  auto run = inf_norm ? clip_run<true> : clip_run<false>;
  return run(n, grads, numel, dtypes, true, max_norm, outs, out_dtypes, norm, (double*)workspace, s);
}

}  // extern "C"
