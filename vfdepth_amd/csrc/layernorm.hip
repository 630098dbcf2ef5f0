// Layer norm over the last dimension of a row-major map or token matrix, forward and backward, with the reduction of
// the weight's and bias's gradients: the sibling of the fused batch norm (bnact.hip) for channels-last maps.
//   m = mean_c x,  v = mean_c (x - m)^2,  r = 1 / sqrt(v + eps),  h = (x - m) r,  y = h w + b
//   d x = r (g w - mean_c(g w) - h mean_c(g w h)),   d w = sum_rows g h,   d b = sum_rows g
// x, y, g, d x fp32 or bf16; w, b, m, r, d w, d b and every sum fp32.
//
// Bound by HBM: forward reads x and writes y, backward reads x and g and writes d x.  A row stays in registers from its
// load to its store: L lanes of a wave (rows under 1025 values; several rows a wave when they are narrow) or a whole
// block of W waves hold it, 16 values a lane at most, so that the squared deviations are summed from the mean (a second
// pass over registers, not over memory).  Blocks walk over rows and load the next row while they work on this one.  The
// backward's column sums stay in registers over all rows of a block; blocks leave one partial row each, which a second
// launch adds in block order: no atomics, the same bits every time.
#include <algorithm>
#include <type_traits>

#include "vfd_common.h"

namespace vfd {

template <typename T>
struct LnV {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // rows start anywhere
};

// `cnt` of the V values at p (the rest 0)
template <typename T>
__device__ __forceinline__ typename LnV<T>::vec ln_load(const T* __restrict__ p, int cnt) {
  constexpr int V = LnV<T>::V;
  typename LnV<T>::vec v;
  if (cnt >= V) return *reinterpret_cast<const typename LnV<T>::vec*>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = (T)0.f;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < cnt) v[j] = p[j];
  return v;
}

template <typename T>
__device__ __forceinline__ void ln_store(T* __restrict__ p, const float* f, int cnt) {
  constexpr int V = LnV<T>::V;
  if (cnt >= V) {
    typename LnV<T>::vec v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)f[j];
    *reinterpret_cast<typename LnV<T>::vec*>(p) = v;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < cnt) p[j] = (T)f[j];
  }
}

// Sum over the L lanes (W = 1) or the W waves (L = 64) of a row's group; in every thread of the group.  W > 1: `lds`
// holds 2 W floats, and calls alternate `slot` so that one barrier a call is enough.
template <int L, int W>
__device__ __forceinline__ float ln_sum(float v, float* lds, int slot) {
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  if constexpr (W > 1) {
    float* s = lds + slot * W;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v += s[k];
  }
  return v;
}

template <typename T, int L, int W, int NV>
struct LnGroup {
  static constexpr int V = LnV<T>::V, G = L * W, BLOCK = G < 256 ? 256 : G, RB = BLOCK / G, E = NV * V;
  int cnt[NV];                                     // this lane's values of each vector
  int col;                                         // its first column
  __device__ __forceinline__ LnGroup(int C) {
    col = (int)(threadIdx.x % G) * V;
#pragma unroll
    for (int u = 0; u < NV; ++u) cnt[u] = min(max(C - col - u * G * V, 0), V);
  }
  __device__ __forceinline__ void params(const float* __restrict__ p, float other, float (&f)[E]) const {
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) f[u * V + j] = (p != nullptr && j < cnt[u]) ? p[col + u * G * V + j] : other;
  }
};

template <typename T, int L, int W, int NV>
__global__ __launch_bounds__((LnGroup<T, L, W, NV>::BLOCK)) void ln_fwd_k(
    const T* __restrict__ x, long long ldx, const float* __restrict__ w, const float* __restrict__ b, T* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, int rows, int C, float eps) {
  typedef LnGroup<T, L, W, NV> Gr;
  constexpr int V = Gr::V, E = Gr::E;
  __shared__ float lds[2 * W];
  const Gr gr(C);
  const int rib = threadIdx.x / Gr::G;
  float wv[E], bv[E];
  gr.params(w, 1.f, wv);
  gr.params(b, 0.f, bv);
  const long long step = (long long)gridDim.x * Gr::RB;
  typename LnV<T>::vec nx[NV];
  auto fetch = [&](long long base) {
    const long long r = base + rib < rows ? base + rib : rows - 1;
#pragma unroll
    for (int u = 0; u < NV; ++u) nx[u] = ln_load(x + r * ldx + gr.col + u * Gr::G * V, gr.cnt[u]);
  };
  fetch((long long)blockIdx.x * Gr::RB);
  for (long long base = (long long)blockIdx.x * Gr::RB; base < rows; base += step) {
    float f[E], s = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[u * V + j] = (float)nx[u][j];
        s += f[u * V + j];
      }
    if (base + step < rows) fetch(base + step);
    const float m = ln_sum<L, W>(s, lds, 0) / (float)C;
    s = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float& e = f[u * V + j];
        e = j < gr.cnt[u] ? e - m : 0.f;
        s = fmaf(e, e, s);
      }
    const float r = 1.f / sqrtf(ln_sum<L, W>(s, lds, 1) / (float)C + eps);
    const long long row = base + rib;
    if (row >= rows) continue;
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = fmaf(f[k] * r, wv[k], bv[k]);
#pragma unroll
    for (int u = 0; u < NV; ++u) ln_store(y + row * C + gr.col + u * Gr::G * V, f + u * V, gr.cnt[u]);
    if (mean != nullptr && threadIdx.x % Gr::G == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

template <typename T, int L, int W, int NV>
__global__ __launch_bounds__((LnGroup<T, L, W, NV>::BLOCK)) void ln_bwd_k(
    const T* __restrict__ g, const T* __restrict__ x, long long ldx, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ part, int rows,
    int C) {
  typedef LnGroup<T, L, W, NV> Gr;
  constexpr int V = Gr::V, E = Gr::E;
  __shared__ float lds[W > 1 ? 4 * W : 4 * L * E];
  const Gr gr(C);
  const int rib = threadIdx.x / Gr::G;
  float wv[E], dw[E], db[E];
  gr.params(w, 1.f, wv);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  const long long step = (long long)gridDim.x * Gr::RB;
  typename LnV<T>::vec nx[NV], ng[NV];
  float nm, nr;
  auto fetch = [&](long long base) {
    const long long r = base + rib < rows ? base + rib : rows - 1;
    nm = mean[r];
    nr = rstd[r];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      nx[u] = ln_load(x + r * ldx + gr.col + u * Gr::G * V, gr.cnt[u]);
      ng[u] = ln_load(g + r * C + gr.col + u * Gr::G * V, gr.cnt[u]);
    }
  };
  fetch((long long)blockIdx.x * Gr::RB);
  int slot = 0;
  for (long long base = (long long)blockIdx.x * Gr::RB; base < rows; base += step) {
    const long long row = base + rib;
    const float m = nm, r = nr;
    float h[E], gv[E], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int k = u * V + j;
        const bool ok = row < rows && j < gr.cnt[u];
        h[k] = ok ? ((float)nx[u][j] - m) * r : 0.f;
        gv[k] = ok ? (float)ng[u][j] : 0.f;
      }
    if (base + step < rows) fetch(base + step);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float gw = gv[k] * wv[k];
      s1 += gw;
      s2 = fmaf(gw, h[k], s2);
      dw[k] = fmaf(gv[k], h[k], dw[k]);
      db[k] += gv[k];
    }
    if (dx == nullptr) continue;
    // the two means in one exchange: their waves' sums lie beside each other
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) {
      s1 += __shfl_xor(s1, off, WAVE);
      s2 += __shfl_xor(s2, off, WAVE);
    }
    if constexpr (W > 1) {
      float* sl = lds + slot * 2 * W;
      slot ^= 1;
      if ((threadIdx.x & 63) == 0) {
        sl[threadIdx.x >> 6] = s1;
        sl[W + (threadIdx.x >> 6)] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        s1 += sl[k];
        s2 += sl[W + k];
      }
    }
    s1 /= (float)C;
    s2 /= (float)C;
    if (row < rows) {
#pragma unroll
      for (int k = 0; k < E; ++k) h[k] = r * (fmaf(gv[k], wv[k], -s1) - h[k] * s2);
#pragma unroll
      for (int u = 0; u < NV; ++u) ln_store(dx + row * C + gr.col + u * Gr::G * V, h + u * V, gr.cnt[u]);
    }
  }
  if (part == nullptr) return;
  float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float* a = half ? db : dw;
    if constexpr (W == 1) {
      // groups of a wave, then the block's four waves
#pragma unroll
      for (int off = L; off < WAVE; off <<= 1)
#pragma unroll
        for (int k = 0; k < E; ++k) a[k] += __shfl_xor(a[k], off, WAVE);
      __syncthreads();
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
      if (lane < L)
#pragma unroll
        for (int k = 0; k < E; ++k) lds[(wave * E + k) * L + lane] = a[k];
      __syncthreads();
      if (wave == 0 && lane < L)
#pragma unroll
        for (int k = 0; k < E; ++k)
          a[k] = (lds[k * L + lane] + lds[(E + k) * L + lane]) + (lds[(2 * E + k) * L + lane] + lds[(3 * E + k) * L + lane]);
      if (wave != 0 || lane >= L) continue;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < gr.cnt[u]) out[half * C + gr.col + u * Gr::G * V + j] = a[u * V + j];
  }
}

// Rows too wide for a block's registers (over 8192 values: sixteen waves of 16 values a lane would spill): a block a row,
// read again for each pass (from cache), 16 bytes a thread at a time.  4096 x 12 288 bf16: 53 us forward (3.8 TB/s), 140 its
// backward in three launches; blocks of 256 and a value a thread at a time took 169 and 231.
constexpr int LN_WIDE = 1024;
template <typename T, typename F>
__device__ __forceinline__ void ln_each(int C, F f) {       // f(first column, its values) over this thread's vectors of a row
  constexpr int V = LnV<T>::V;
  for (int c = (int)threadIdx.x * V; c < C; c += LN_WIDE * V) f(c, min(C - c, V));
}

// A vector's parameters from column c on; null: `other`
template <int V>
__device__ __forceinline__ void ln_wide_params(const float* __restrict__ p, int c, int cnt, float other, float (&f)[V]) {
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    LnV<float>::vec v = {other, other, other, other};
    if (p != nullptr) v = ln_load(p + c + h, cnt - h);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[h + j] = v[j];
  }
}

template <typename T>
__global__ __launch_bounds__(LN_WIDE) void ln_fwd_wide_k(const T* __restrict__ x, long long ldx, const float* __restrict__ w,
                                                         const float* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
                                                         float* __restrict__ rstd, int rows, int C, float eps) {
  constexpr int V = LnV<T>::V, W = LN_WIDE / 64;
  __shared__ float lds[2 * W];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.f;
    ln_each<T>(C, [&](int c, int cnt) {
      const auto v = ln_load(xr + c, cnt);
#pragma unroll
      for (int j = 0; j < V; ++j) s += (float)v[j];
    });
    const float m = ln_sum<64, W>(s, lds, 0) / (float)C;
    s = 0.f;
    ln_each<T>(C, [&](int c, int cnt) {
      const auto v = ln_load(xr + c, cnt);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = j < cnt ? (float)v[j] - m : 0.f;
        s = fmaf(e, e, s);
      }
    });
    const float r = 1.f / sqrtf(ln_sum<64, W>(s, lds, 1) / (float)C + eps);
    ln_each<T>(C, [&](int c, int cnt) {
      const auto v = ln_load(xr + c, cnt);
      float f[V], wv[V], bv[V];
      ln_wide_params(w, c, cnt, 1.f, wv);
      ln_wide_params(b, c, cnt, 0.f, bv);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = fmaf(((float)v[j] - m) * r, wv[j], bv[j]);
      ln_store(y + row * C + c, f, cnt);
    });
    if (mean != nullptr && threadIdx.x == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(LN_WIDE) void ln_bwd_wide_k(const T* __restrict__ g, const T* __restrict__ x, long long ldx,
                                                         const float* __restrict__ w, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, T* __restrict__ dx, int rows, int C) {
  constexpr int V = LnV<T>::V, W = LN_WIDE / 64;
  __shared__ float lds[2 * W];
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx, *gr = g + row * C;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    ln_each<T>(C, [&](int c, int cnt) {
      const auto xv = ln_load(xr + c, cnt), gv = ln_load(gr + c, cnt);
      float wv[V];
      ln_wide_params(w, c, cnt, 1.f, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gw = j < cnt ? (float)gv[j] * wv[j] : 0.f;
        s1 += gw;
        s2 = fmaf(gw, j < cnt ? ((float)xv[j] - m) * r : 0.f, s2);
      }
    });
    s1 = ln_sum<64, W>(s1, lds, 0) / (float)C;
    s2 = ln_sum<64, W>(s2, lds, 1) / (float)C;
    ln_each<T>(C, [&](int c, int cnt) {
      const auto xv = ln_load(xr + c, cnt), gv = ln_load(gr + c, cnt);
      float f[V], wv[V];
      ln_wide_params(w, c, cnt, 1.f, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = r * (fmaf((float)gv[j], wv[j], -s1) - ((float)xv[j] - m) * r * s2);
      ln_store(dx + row * C + c, f, cnt);
    });
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_cols_wide_k(const T* __restrict__ g, const T* __restrict__ x, long long ldx,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      float* __restrict__ part, int rows, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  constexpr int U = 4;                                       // rows in flight
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < rows; row += (long long)U * gridDim.y) {
    float gv[U], h[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long r = row + u * (long long)gridDim.y, q = r < rows ? r : rows - 1;
      gv[u] = ld1(g + q * C + c);
      h[u] = (ld1(x + q * ldx + c) - mean[q]) * rstd[q];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * (long long)gridDim.y < rows) {
        dw = fmaf(gv[u], h[u], dw);
        db += gv[u];
      }
  }
  part[(size_t)blockIdx.y * 2 * C + c] = dw;
  part[(size_t)blockIdx.y * 2 * C + C + c] = db;
}

// The kernel that holds a row of C values: F(L, W, NV), or F(0, 0, 0) for the wide form.
template <typename T, typename F>
static int ln_pick(int C, F f) {
  constexpr int V = LnV<T>::V;
  const int nv = (C + V - 1) / V;
#define LN_CASE(LIMIT, L, W, NV) \
  if (nv <= (LIMIT)) return f(std::integral_constant<int, L>(), std::integral_constant<int, W>(), std::integral_constant<int, NV>());
  LN_CASE(4, 4, 1, 1)
  LN_CASE(8, 8, 1, 1)
  LN_CASE(16, 16, 1, 1)
  LN_CASE(32, 32, 1, 1)
  LN_CASE(64, 64, 1, 1)
  LN_CASE(128, 64, 1, 2)
  if constexpr (V == 4) {
    LN_CASE(256, 64, 1, 4)
    LN_CASE(512, 64, 4, 2)
    LN_CASE(1024, 64, 4, 4)
    LN_CASE(2048, 64, 8, 4)
  } else {
    LN_CASE(256, 64, 4, 1)
    LN_CASE(512, 64, 4, 2)
    LN_CASE(1024, 64, 8, 2)
  }
#undef LN_CASE
  return f(std::integral_constant<int, 0>(), std::integral_constant<int, 0>(), std::integral_constant<int, 0>());
}

// Blocks that walk over the rows.  Forward, 23 040 x 4096 bf16: 91 us with 512, 77 with 1024, 85 with 2048, 150 with 8192
// (each loads the parameters); 5761 x 1021 fp32 14 with 1024, 17 with 2048.
constexpr int LN_FWD_GRID = 1024;

// Blocks of the backward = partial rows: enough to keep every CU loading, few enough that the partials (8 C bytes each,
// written and read) stay small beside the rows.  `w` waves and `e` values a lane hold a row: 23 040 x 4096 bf16 (4, 16) 131 us
// with 384, 115 with 512, 122 with 768; 5761 x 1021 fp32 (1, 16) 15.4 with 768, 18.4 with 1024; 368 640 x 64 bf16 (1, 8)
// 28.4 with 512, 26.6 with 1024.
static int ln_bwd_blocks(int rows, int rb, int w, int e) {
  const int most = w > 1 ? 512 : (e >= 16 ? 768 : 1024);
  const int need = (rows - 1) / rb + 1;                      // (rows up to 2^31 - 1: none added to them)
  return need < most ? need : most;
}

template <typename T>
static int ln_parts(int rows, int C) {
  return ln_pick<T>(C, [&](auto l, auto w, auto nv) {
    if constexpr (decltype(l)::value == 0)
      return std::max(1, std::min({rows, 128, (1 << 22) / C}));      // (partials of at most 32 MB up to 2^22 columns)
    else
      return ln_bwd_blocks(rows, LnGroup<T, l(), w(), nv()>::RB, w(), LnGroup<T, l(), w(), nv()>::E);
  });
}

template <typename T>
static int ln_fwd_run(const vfd_norm_desc* d, const void* x, const float* w, const float* b, void* y, float* mean,
                      float* rstd, hipStream_t s) {
  return ln_pick<T>(d->cols, [&](auto l, auto wv, auto nv) {
    if constexpr (decltype(l)::value == 0) {
      const int grid = d->rows < LN_FWD_GRID ? d->rows : LN_FWD_GRID;
      ln_fwd_wide_k<T><<<grid, LN_WIDE, 0, s>>>((const T*)x, d->ldx, w, b, (T*)y, mean, rstd, d->rows, d->cols, d->eps);
    } else {
      typedef LnGroup<T, l(), wv(), nv()> Gr;
      const int need = (d->rows - 1) / Gr::RB + 1, grid = need < LN_FWD_GRID ? need : LN_FWD_GRID;
      ln_fwd_k<T, l(), wv(), nv()><<<grid, Gr::BLOCK, 0, s>>>((const T*)x, d->ldx, w, b, (T*)y, mean, rstd, d->rows, d->cols, d->eps);
    }
    return fail_launch("layer_norm_fwd");
  });
}

template <typename T>
static int ln_bwd_run(const vfd_norm_desc* d, const void* g, const void* x, const float* w, const float* mean,
                      const float* rstd, void* dx, float* dw, float* db, float* part, hipStream_t s) {
  const bool cols = dw != nullptr || db != nullptr;
  const int nb = ln_parts<T>(d->rows, d->cols);
  const int e = ln_pick<T>(d->cols, [&](auto l, auto wv, auto nv) {
    if constexpr (decltype(l)::value == 0) {
      if (dx)
        ln_bwd_wide_k<T><<<d->rows < LN_FWD_GRID ? d->rows : LN_FWD_GRID, LN_WIDE, 0, s>>>((const T*)g, (const T*)x, d->ldx, w, mean,
                                                                              rstd, (T*)dx, d->rows, d->cols);
      if (cols)
        ln_cols_wide_k<T><<<dim3(cdiv(d->cols, 256), nb), 256, 0, s>>>((const T*)g, (const T*)x, d->ldx, mean, rstd, part,
                                                                       d->rows, d->cols);
    } else {
      ln_bwd_k<T, l(), wv(), nv()><<<nb, LnGroup<T, l(), wv(), nv()>::BLOCK, 0, s>>>(
          (const T*)g, (const T*)x, d->ldx, w, mean, rstd, (T*)dx, cols ? part : nullptr, d->rows, d->cols);
    }
    return fail_launch("layer_norm_bwd");
  });
  if (e != VFD_OK || !cols) return e;
  col_sums_k<float><<<col_sums_grid(2 * (size_t)d->cols), 1024, 0, s>>>(part, nb, 2 * d->cols, d->cols, dw, db);
  return fail_launch("layer_norm_bwd columns");
}

static int ln_check(const char* what, const vfd_norm_desc* d) {
  VFD_REQUIRE(d && d->rows >= 0 && d->cols >= 1 && d->cols <= (1 << 28) && d->ldx >= d->cols &&
                  (d->dtype == 0 || d->dtype == 1),
              "%s: bad descriptor", what);
  return VFD_OK;
}

}  // namespace vfd

using namespace vfd;

extern "C" {

int vfd_layer_norm_fwd(const vfd_norm_desc* d, const void* x, const float* w, const float* b, void* y, float* mean,
                       float* rstd, void* stream) {
  if (int e = ln_check("layer_norm_fwd", d)) return e;
  if (d->rows == 0) return VFD_OK;
  VFD_REQUIRE(x && y && (mean != nullptr) == (rstd != nullptr), "layer_norm_fwd: null tensor");
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_LN_FWD, s);
  return (d->dtype ? ln_fwd_run<__bf16> : ln_fwd_run<float>)(d, x, w, b, y, mean, rstd, s);
}

size_t vfd_layer_norm_bwd_workspace(const vfd_norm_desc* d) {
  if (ln_check("layer_norm_bwd", d) != VFD_OK || d->rows == 0) return 0;
  return (size_t)(d->dtype ? ln_parts<__bf16>(d->rows, d->cols) : ln_parts<float>(d->rows, d->cols)) * 2 * d->cols * sizeof(float);
}

int vfd_layer_norm_bwd(const vfd_norm_desc* d, const void* g, const void* x, const float* w, const float* mean,
                       const float* rstd, void* dx, float* dw, float* db, void* workspace, size_t ws_bytes, void* stream) {
  if (int e = ln_check("layer_norm_bwd", d)) return e;
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_LN_BWD, s);
  if (d->rows == 0) {
    if (dw) zero_async(dw, (size_t)d->cols * sizeof(float), s);
    if (db) zero_async(db, (size_t)d->cols * sizeof(float), s);
    return fail_launch("layer_norm_bwd");
  }
  VFD_REQUIRE(g && x && mean && rstd, "layer_norm_bwd: null tensor");
  VFD_REQUIRE((!dw && !db) || (workspace && ws_bytes >= vfd_layer_norm_bwd_workspace(d)), "layer_norm_bwd: workspace too small");
  if (!dx && !dw && !db) return VFD_OK;
  return (d->dtype ? ln_bwd_run<__bf16> : ln_bwd_run<float>)(d, g, x, w, mean, rstd, dx, dw, db, (float*)workspace, s);
}

}  // extern "C"
