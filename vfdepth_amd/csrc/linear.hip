// Matrix product with bias, activation and residual in its epilogue (a linear layer, or a 1x1 convolution of a
// channels-last map), forward and backward, on the matrix cores:
//   z = x W^T + b,   y = act(z) + r            x [M, K], W [N, K], y, z, r [M, N]
//   gz = g act'(z),  d x = gz W,  d W = gz^T x,  d b = column sums of gz,  d r = g
// fp32 (v_mfma_f32_32x32x2_f32) or bf16 (v_mfma_f32_32x32x16_bf16, fp32 sums, each output rounded once).
//
// One tile kernel serves the three products: an operand is read as [outer][contraction] (its contraction contiguous:
// x, W and gz forward) or as [contraction][outer] (W and gz, x in the gradients), and leaves LDS in the matrix
// instructions' order either way, so nothing is transposed in memory.
#include <algorithm>
#include <type_traits>

#include "vfd_common.h"

namespace vfd {

typedef float lin_f16 __attribute__((ext_vector_type(16)));
typedef float lin_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 lin_b8 __attribute__((ext_vector_type(8)));
typedef short lin_s4 __attribute__((ext_vector_type(4)));

enum LinAct { LIN_NONE = 0, LIN_RELU, LIN_LRELU, LIN_ELU, LIN_GELU, LIN_SILU, LIN_ACTS };
constexpr float LIN_SLOPE = 0.1f;            // the framework's LeakyReLU

// The activations run once per output, behind the matrix cores: a few instructions each.
__device__ __forceinline__ float lin_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2), by Abramowitz & Stegun 7.1.26 (Hastings): erfc(x) =
// t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + p x), within 1.5e-7 for x >= 0.
__device__ __forceinline__ float lin_phi(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
  e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504088896341f));
  const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f), 0.5f * -0.284496736f),
                       0.5f * 0.254829592f);
  const float q = t * p * e;
  return z > 0.f ? 1.f - q : q;
}

// exp(z) - 1 for z <= 0: its series where the subtraction would cancel
__device__ __forceinline__ float lin_expm1(float z) {
  const float s = z * fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 5040, 1.f / 720), 1.f / 120), 1.f / 24), 1.f / 6), 0.5f), 1.f);
  return z > -0.25f ? s : lin_exp(z) - 1.f;
}

template <int ACT>
__device__ __forceinline__ float lin_act(float z) {
  if constexpr (ACT == LIN_RELU) return z <= 0.f ? 0.f : z;               // NaN passes
  if constexpr (ACT == LIN_LRELU) return z > 0.f ? z : LIN_SLOPE * z;
  if constexpr (ACT == LIN_ELU) return z > 0.f ? z : lin_expm1(z);
  if constexpr (ACT == LIN_GELU) {
    float e;
    return z * lin_phi(z, e);
  }
  if constexpr (ACT == LIN_SILU) return z * __builtin_amdgcn_rcpf(1.f + lin_exp(-z));
  return z;
}

template <int ACT>
__device__ __forceinline__ float lin_slope(float z) {
  if constexpr (ACT == LIN_LRELU) return z > 0.f ? 1.f : LIN_SLOPE;
  if constexpr (ACT == LIN_ELU) return z > 0.f ? 1.f : lin_exp(z);
  if constexpr (ACT == LIN_GELU) {
    float e;
    const float phi = lin_phi(z, e);
    return fmaf(z, e * 0.39894228040143268f, phi);
  }
  if constexpr (ACT == LIN_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + lin_exp(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  return 1.f;
}

// g act'(z).  Where ReLU lets nothing through, an infinite or NaN g does not pass either.
template <int ACT>
__device__ __forceinline__ float lin_back(float g, float z) {
  if constexpr (ACT == LIN_RELU) return z <= 0.f ? 0.f : g;
  return g * lin_slope<ACT>(z);
}

template <typename F>
static int lin_with_act(int act, F f) {
  switch (act) {
    case LIN_RELU: return f(std::integral_constant<int, LIN_RELU>());
    case LIN_LRELU: return f(std::integral_constant<int, LIN_LRELU>());
    case LIN_ELU: return f(std::integral_constant<int, LIN_ELU>());
    case LIN_GELU: return f(std::integral_constant<int, LIN_GELU>());
    case LIN_SILU: return f(std::integral_constant<int, LIN_SILU>());
    default: return f(std::integral_constant<int, LIN_NONE>());
  }
}

// ---------------------------------------------------------------- tile kernel
template <typename T>
struct LinT {
  static constexpr int VE = 16 / (int)sizeof(T);        // values of a 16-byte chunk
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  typedef T avec __attribute__((ext_vector_type(16 / sizeof(T))));
};

__device__ __forceinline__ lin_f16 lin_mma(lin_b8 a, lin_b8 b, lin_f16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// four steps of two contraction values: lane halves hold values 4 h + j of each group of eight
__device__ __forceinline__ lin_f16 lin_mma(lin_f4 a, lin_f4 b, lin_f16 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// A chunk moved down by d >= 0 values, zeros behind it
template <typename T>
__device__ __forceinline__ typename LinT<T>::vec lin_down(typename LinT<T>::vec v, int d) {
  unsigned __int128 u;
  __builtin_memcpy(&u, &v, 16);
  u = d >= LinT<T>::VE ? (unsigned __int128)0 : u >> (d * 8 * (int)sizeof(T));
  __builtin_memcpy(&v, &u, 16);
  return v;
}

// One operand of a product: element (o, k) at p[o * ld + k] (MC = false) or p[k * ld + o] (MC = true).
template <typename T>
struct LinOp {
  const T* p;
  long long ld;
  int O, K;
};

// A tile of BO outer indices by RB bytes of contraction in LDS, filled by NT threads.
//   MC = false: rows of RB bytes, one per outer index.  A fragment's read takes one 16-byte chunk of 32 rows; the 16 lanes
//     that share a cycle (of 256 bytes) meet 16 different chunk places because a row's chunk numbers are exchanged by its
//     place among the rows that start at the same bank.
//   MC = true: rows of BO values, one per contraction index.  bf16: the transposing read takes 64 bytes of 4 rows in a
//     cycle, spread over 256 bytes by exchanging 64-byte groups by (row & 3); fp32: lanes read consecutive values.
template <typename T, bool MC, int BO, int NT, int RB>
struct LinTile {
  typedef LinT<T> X;
  static constexpr int BK = RB / (int)sizeof(T);        // contraction values of the tile
  static constexpr int BYTES = BO * RB, CK = RB / 16;   // its bytes, chunks of an outer index
  static constexpr int NCH = BO * CK / NT;              // chunks a thread stages
  static constexpr int CPR = MC ? BO / X::VE : CK;      // chunks of a row in LDS
  static constexpr int READS = !MC ? 1 : sizeof(T) == 2 ? 2 : 4;   // LDS instructions of a fragment
  static_assert(BO * CK % NT == 0 && (!MC || CPR == 8 || CPR % 16 == 0), "whole chunks a thread, exchanged within a row");

  static __device__ __forceinline__ int turn(int row) {            // what a row's chunk numbers are exchanged by
    if constexpr (!MC) return RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
    if constexpr (sizeof(T) != 2) return 0;
    return CPR == 8 ? (row & 2) << 1 : (row & 3) << 2;
  }
  static __device__ __forceinline__ int at(int row, int c) {       // byte offset of a chunk
    return row * (CPR * 16) + ((c ^ turn(row)) << 4);
  }
  // A tile through registers, at any alignment and with any edge: every load is unconditional and in bounds (a chunk that
  // would leave its row starts VE before the row's end and is shifted down, zeros behind it), so that they all fly together.
  static __device__ __forceinline__ void fetch(const LinOp<T>& op, int o0, int k0, typename X::vec (&v)[NCH]) {
    const int len = MC ? op.O : op.K;                   // of a row in memory
    const bool whole = k0 + BK <= op.K && (!MC || o0 + BO <= op.O);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e = (int)threadIdx.x + i * NT;
      const int row = e / CPR, c = (e % CPR) * X::VE;
      const int r = MC ? min(k0 + row, op.K - 1) : min(o0 + row, op.O - 1), at = (MC ? o0 : k0) + c;
      const T* p = op.p + (size_t)r * op.ld;
      if (whole) {
        v[i] = *reinterpret_cast<const typename X::vec*>(p + at);
      } else if (len >= X::VE) {
        const int from = min(at, len - X::VE);
        v[i] = lin_down<T>(*reinterpret_cast<const typename X::vec*>(p + from), at - from);
      } else {
#pragma unroll
        for (int j = 0; j < X::VE; ++j) {
          const T t = p[min(at + j, len - 1)];
          v[i][j] = at + j < len ? t : (T)0.f;
        }
      }
      if (MC && !whole && k0 + row >= op.K) v[i] = lin_down<T>(v[i], X::VE);
    }
  }
  static __device__ __forceinline__ void put(char* lds, const typename X::vec (&v)[NCH]) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e = (int)threadIdx.x + i * NT;
      *reinterpret_cast<typename X::avec*>(lds + at(e / CPR, e % CPR)) = v[i];
    }
  }
  // Whole tiles straight into LDS: a wave's 64 chunks land one after another, so each lane fetches the chunk whose place
  // that is.  Outer indices beyond the operand fetch its last chunk again (their products are not stored); a last chunk that
  // leaves its row goes on into the next one, which a ragged tile of the last rows must not (lin_tile_k).  Through a
  // buffer descriptor: a lane's offsets stay the same for every tile, and past the last tile an empty one loads nothing.
  struct Stream {
    const char* p;                                      // of the next tile (uniform)
    long long step;
    unsigned off[NCH];
  };
  static __device__ __forceinline__ void open(const LinOp<T>& op, int o0, int k0, Stream& s) {
    constexpr int ES = (int)sizeof(T);
    s.p = (const char*)(op.p + (MC ? (size_t)k0 * op.ld + o0 : (size_t)o0 * op.ld + k0));
    s.step = (long long)BK * ES * (MC ? op.ld : 1);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e = (int)threadIdx.x + i * NT;
      const int row = e / CPR, c = ((e % CPR) ^ turn(row)) * X::VE;
      s.off[i] = MC ? (unsigned)row * (unsigned)op.ld * ES + (unsigned)min(c, (op.O - 1 - o0) / X::VE * X::VE) * ES
                    : (unsigned)min(row, op.O - 1 - o0) * (unsigned)op.ld * ES + c * ES;
    }
  }
  static __device__ __forceinline__ void next(Stream& s, char* lds, bool live) {
    typedef __attribute__((address_space(3))) void lvoid;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)s.p, 0, live ? 0x7fffffff : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lvoid*)(lds + (i * NT + wave * 64) * 16), 16, s.off[i], 0, 0, 0);
    s.p += s.step;
  }
  // The 32 outer indices from o on, contraction step ks (32 bytes each): lane l holds outer l & 31, 16 bytes of contraction
  static __device__ __forceinline__ typename X::avec frag(const char* lds, int o, int ks) {
    const int lane = threadIdx.x & 63;
    typename X::avec r;
    if constexpr (!MC) {
      r = *reinterpret_cast<const typename X::avec*>(lds + at(o + (lane & 31), 2 * ks + (lane >> 5)));
    } else if constexpr (sizeof(T) == 2) {
      // transposing read: lane 4 q + p of 16-lane group gq supplies row q, columns 4 p .. of column half gq & 1
      const int gq = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
      const int col = o + 16 * (gq & 1) + 4 * p, k = 16 * ks + 8 * (gq >> 1) + q;
      typedef __attribute__((address_space(3))) lin_s4 lds_s4;
      const lin_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at(k, col >> 3) + (col & 7) * 2));
      const lin_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + at(k + 4, col >> 3) + (col & 7) * 2));
      __builtin_memcpy(&r, &a, 8);
      __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &b, 8);
    } else {
      const int k = 8 * ks + 4 * (lane >> 5);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = o + (lane & 31);
        r[j] = *reinterpret_cast<const float*>(lds + at(k + j, col >> 2) + (col & 3) * 4);
      }
    }
    return r;
  }
};

// Loads straight into LDS are counted with the loads from memory, and a barrier does not wait for them by itself: every
// wave waits until at most LEFT of its own are on their way (they arrive in order) and its LDS reads have ended, then all
// wait for each other.
template <int LEFT>
__device__ __forceinline__ void lin_arrived() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

template <typename T>
struct LinEpi {
  const T* bias;                 // [N], null
  const T* res;                  // [M, N], null
  T* z;                          // [M, N], null: pre-activation for the backward
  T* y;                          // [M, N]
  float* part;                   // [splits, M, N] where the contraction is split (then nothing else is used)
  int act;
};

// V consecutive values at any element boundary, `cnt` of them (the rest 0); null: 0; whole: all of them in every lane
template <int V, typename T>
__device__ __forceinline__ void lin_ld(const T* __restrict__ p, int cnt, float (&f)[V], bool whole = false) {
  typedef T vv __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if (whole) {
    const vv v = *reinterpret_cast<const vv*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)v[e];
  } else if (p != nullptr && cnt == V) {
    const vv v = *reinterpret_cast<const vv*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (p != nullptr && e < cnt) ? ld1(p + e) : 0.f;
  }
}
template <int V, typename T>
__device__ __forceinline__ void lin_st(T* __restrict__ p, int cnt, const float (&f)[V], bool whole = false) {
  typedef T vv __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vv v;
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (T)f[e];
  if (whole) {
    *reinterpret_cast<vv*>(p) = v;
  } else if (cnt == V) {
    *reinterpret_cast<vv*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < cnt) p[e] = v[e];
  }
}

// The epilogue of V consecutive outputs at element `at` of y
template <int ACT, int V, typename T>
__device__ __forceinline__ void lin_finish(const LinEpi<T>& ep, size_t at, int cnt, const float (&bias)[V], const float (&res)[V],
                                           float (&v)[V], bool whole = false) {
  if (ep.bias)
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += bias[e];
  if (ep.z) lin_st<V>(ep.z + at, cnt, v, whole);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = lin_act<ACT>(v[e]);
  if (ep.res)
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += res[e];
  lin_st<V>(ep.y + at, cnt, v, whole);
}

template <typename T, bool XMC, bool WMC, int BM, int BN, int WM, int WN, int OCC, int RB, int SLOTS, bool ASYNC, bool PART, int ACT>
__global__ __launch_bounds__(64 * WM * WN, OCC) void lin_tile_k(LinOp<T> x, LinOp<T> w, LinEpi<T> ep, int tm, int tn, int splits) {
  constexpr int NT = 64 * WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
  typedef LinT<T> X;
  typedef LinTile<T, XMC, BM, NT, RB> TX;
  typedef LinTile<T, WMC, BN, NT, RB> TW;
  constexpr int BK = TX::BK, KS = RB / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int STAGE = (BM + BN) * RB, LOADS = TX::NCH + TW::NCH;
  // tiles of one XCD (every eighth workgroup) are consecutive: column groups of 4 row tiles, splits outermost
  // (of 8: 16 384 x 2048 x 8192 bf16 461 us forward, 514 data gradient; 446 and 495 with 4)
  const int total = tm * tn * splits, xcd = blockIdx.x % 8, per = total / 8, rest = total % 8;
  int t = xcd * per + min(xcd, rest) + blockIdx.x / 8;
  const int split = t / (tm * tn);
  t -= split * tm * tn;
  constexpr int GM = 4;
  const int group = t / (GM * tn), g0 = group * GM, gm = min(GM, tm - g0);
  t -= group * GM * tn;
  const int m0 = (g0 + t % gm) * BM, n0 = (t / gm) * BN;
  const int kt = (x.K + BK - 1) / BK;
  int k_lo = (int)((long long)kt * split / splits);
  const int k_hi = (int)((long long)kt * (split + 1) / splits);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = (wave % WM) * FM * 32, wn = (wave / WM) * FN * 32;

  lin_f16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  typename X::avec fx[2][FM], fw[2][FN];
  auto load = [&](auto f, const char* cur, int ks) {
#pragma unroll
    for (int i = 0; i < FM; ++i) fx[f()][i] = TX::frag(cur, wm + 32 * i, ks);
#pragma unroll
    for (int j = 0; j < FN; ++j) fw[f()][j] = TW::frag(cur + TX::BYTES, wn + 32 * j, ks);
  };
  auto mma = [&](auto f) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = lin_mma(fw[f()][j], fx[f()][i], acc[i][j]);
  };
  const std::integral_constant<int, 0> f0;
  const std::integral_constant<int, 1> f1;
  // A step's instructions in turn: the reads of the next step's fragments (and the loads of another tile) between the
  // products of this one.  Left to itself the compiler reads fragments just before it needs them and waits.
  constexpr int READS = FM * TX::READS + FN * TW::READS, MMAS = FM * FN * (sizeof(T) == 2 ? 1 : 4);
  auto in_turn = [&](auto loads) {
    constexpr int PARTS = READS < MMAS ? READS : MMAS;
#pragma unroll
    for (int u = 0; u < PARTS; ++u) {
      constexpr int rd = 0x100, mm = 0x008, vm = 0x020;
      __builtin_amdgcn_sched_group_barrier(rd, READS / PARTS, 0);
      if constexpr (loads() > 0) __builtin_amdgcn_sched_group_barrier(vm, (loads() + PARTS - 1) / PARTS, 0);
      __builtin_amdgcn_sched_group_barrier(mm, MMAS / PARTS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const std::integral_constant<int, 0> no_loads;
  const std::integral_constant<int, LOADS> tile_loads;
  // all steps of a tile but the last's products; its first fragments are in f0, its last are left in f1
  auto steps = [&](const char* cur) {
#pragma unroll
    for (int ks = 0; ks + 1 < KS; ks += 2) {
      load(f1, cur, ks + 1);
      mma(f0);
      in_turn(no_loads);
      if (ks + 2 < KS) {
        load(f0, cur, ks + 2);
        mma(f1);
        in_turn(no_loads);
      }
    }
  };
  if constexpr (ASYNC) {
    // SLOTS tiles in LDS: one is worked on, the others are on their way.  The fragments of a step are read during the
    // products of the step before; a tile's last products run behind the barrier that frees its slot, while the next
    // tile's first fragments are read and another tile starts on its way.
    int k_end = min(k_hi, x.K / BK);
    if (k_end * BK == x.K && ((XMC && x.O % X::VE != 0 && m0 + BM > x.O) || (WMC && w.O % X::VE != 0 && n0 + BN > w.O)))
      --k_end;                                             // the last row of memory: no row behind it to go on into
    if (k_lo < k_end) {
      typename TX::Stream sx;
      typename TW::Stream sw;
      TX::open(x, m0, k_lo * BK, sx);
      TW::open(w, n0, k_lo * BK, sw);
      auto stage = [&](char* at, bool live) {
        TX::next(sx, at, live);
        TW::next(sw, at + TX::BYTES, live);
      };
#pragma unroll
      for (int u = 0; u < SLOTS; ++u) stage(lds + u * STAGE, k_lo + u < k_end);
      lin_arrived<LOADS * (SLOTS - 1)>();
      load(f0, lds, 0);
      int slot = 0;
#pragma unroll 1
      for (int k = k_lo; k < k_end; ++k) {
        char* cur = lds + slot * STAGE;
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
        steps(cur);
        lin_arrived<LOADS * (SLOTS - 2)>();                // the next tile is there
        stage(cur, k + SLOTS < k_end);
        load(f0, lds + slot * STAGE, 0);                   // (behind the last tile: read, not used)
        mma(f1);
        in_turn(tile_loads);
      }
      lin_arrived<0>();
    }
    k_lo = max(k_lo, min(k_end, k_hi));                  // a last tile that the contraction ends in: staged with masks
  }
  {
    typename X::vec vx[TX::NCH], vw[TW::NCH];
    if (k_lo < k_hi) {
      TX::fetch(x, m0, k_lo * BK, vx);
      TW::fetch(w, n0, k_lo * BK, vw);
      TX::put(lds, vx);
      TW::put(lds + TX::BYTES, vw);
    }
    __syncthreads();
    for (int k = k_lo; k < k_hi; ++k) {
      char* nxt = lds + ((k + 1 - k_lo) & 1) * STAGE;
      if (k + 1 < k_hi) {
        TX::fetch(x, m0, (k + 1) * BK, vx);
        TW::fetch(w, n0, (k + 1) * BK, vw);
      }
      const char* cur = lds + ((k - k_lo) & 1) * STAGE;
      load(f0, cur, 0);
      steps(cur);
      mma(f1);
      if (k + 1 < k_hi) {
        TX::put(nxt, vx);
        TW::put(nxt + TX::BYTES, vw);
      }
      __syncthreads();
    }
  }

  // D of a block: column (lane & 31) = row of y, 4 consecutive columns of y per group of 4 registers.  Each wave turns 32
  // rows at a time over in its own part of LDS, so that its lanes store (and load residuals) 16 bytes each, whole lines of
  // a row together: stored from registers, 32 bytes of 32 rows at a time, the same outputs took up to twice as long
  // (92 160 x 1024 bf16, contraction 256: 197 us, 120 this way).  The pitch of 4 more floats spreads the rows over the banks.
  constexpr int COLS = FN * 32, PITCH = COLS + 4;
  static_assert(WM * WN * 32 * PITCH * 4 <= SLOTS * STAGE, "the waves' output rows fit where the tiles were");
  float* turn = reinterpret_cast<float*>(lds) + wave * (32 * PITCH);
  const int M = x.O, N = w.O;
  auto turn_over = [&](auto i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        lin_f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i()][j][4 * q + e];
        *reinterpret_cast<lin_f4*>(turn + (lane & 31) * PITCH + 32 * j + 8 * q + 4 * (lane >> 5)) = v;
      }
  };
  constexpr int V = PART ? 4 : X::VE, LPR = COLS / V, PASS = 64 / LPR;
  const int col = n0 + wn + (lane % LPR) * V, cnt = min(max(N - col, 0), V);
  const bool whole = m0 + BM <= M && n0 + BN <= N;       // no edge in this tile (uniform)
  float bias[V];
  if constexpr (!PART)
    if (ep.bias) lin_ld<V>(ep.bias + col, cnt, bias, whole);
  size_t row = (size_t)(m0 + wm + lane / LPR) * N + col;
  const size_t down = (size_t)PASS * N;
  constexpr int FLY = OCC > 2 ? 2 : 4;                     // (three blocks a CU leave fewer registers)
#pragma unroll 1
  for (int i = 0; i < FM; ++i) {                         // one copy of the epilogue's code
    if (i == 0) turn_over(std::integral_constant<int, 0>());
    if constexpr (FM > 1)
      if (i == 1) turn_over(std::integral_constant<int, 1>());
    if constexpr (FM > 2) {
      if (i == 2) turn_over(std::integral_constant<int, 2>());
      if (i == 3) turn_over(std::integral_constant<int, 3>());
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += FLY * PASS) {        // rows a lane in flight
      float v[FLY][V], res[FLY][V];
      int c[FLY];
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        const int r = r0 + u * PASS + lane / LPR;
        c[u] = m0 + wm + 32 * i + r < M ? cnt : 0;
        if constexpr (!PART)
          if (ep.res) lin_ld<V>(ep.res + row + u * down, c[u], res[u], whole);
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
          const lin_f4 t = *reinterpret_cast<const lin_f4*>(turn + r * PITCH + (lane % LPR) * V + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][4 * h + e] = t[e];
        }
      }
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        if constexpr (PART)
          lin_st<V>(ep.part + (size_t)split * M * N + row + u * down, c[u], v[u], whole);
        else
          lin_finish<ACT>(ep, row + u * down, c[u], bias, res[u], v[u], whole);
      }
      row += FLY * down;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------- few rows
// At most 16 MB rows of x (a frame's tokens): bound by reading W once, so nothing is staged.  A block owns 16 rows of W,
// its eight waves take the contraction in turn (16 rows x 64 bytes of W a load, the x rows beside them from cache), and
// their sums meet in LDS.
constexpr int LIN_THIN = 64;
__device__ __forceinline__ lin_f4 lin_mma16(lin_b8 a, lin_b8 b, lin_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ lin_f4 lin_mma16(lin_f4 a, lin_f4 b, lin_f4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

template <typename T, int MB, int ACT>
__global__ __launch_bounds__(512) void lin_thin_k(LinOp<T> x, LinOp<T> w, LinEpi<T> ep) {
  typedef LinT<T> X;
  constexpr int W = 8, STEP = 4 * X::VE, U = 4;
  __shared__ lin_f4 sm[W][MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = x.K, M = x.O, N = w.O;
  const int n0 = blockIdx.x * 16, kl = (lane >> 4) * X::VE;
  const T* pw = w.p + (size_t)min(n0 + (lane & 15), N - 1) * w.ld;
  const T* px[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) px[i] = x.p + (size_t)min(16 * i + (lane & 15), M - 1) * x.ld;
  lin_f4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = lin_f4{0.f, 0.f, 0.f, 0.f};
  int k = wave * STEP;
  for (; k + (U - 1) * W * STEP + STEP <= K; k += U * W * STEP) {
    typename X::vec vw[U], vx[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + u * W * STEP + kl;
      vw[u] = *reinterpret_cast<const typename X::vec*>(pw + at);
#pragma unroll
      for (int i = 0; i < MB; ++i) vx[u][i] = *reinterpret_cast<const typename X::vec*>(px[i] + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i] = lin_mma16((typename X::avec)vw[u], (typename X::avec)vx[u][i], acc[i]);
  }
  auto edge = [&](const T* p, int at) {
    typename X::vec v;
    if (K >= X::VE) {
      const int from = min(at, K - X::VE);
      return lin_down<T>(*reinterpret_cast<const typename X::vec*>(p + from), at - from);
    }
#pragma unroll
    for (int j = 0; j < X::VE; ++j) {
      const T t = p[min(at + j, K - 1)];
      v[j] = at + j < K ? t : (T)0.f;
    }
    return v;
  };
  for (; k < K; k += W * STEP) {
    const typename X::vec vw = edge(pw, k + kl);
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = lin_mma16((typename X::avec)vw, (typename X::avec)edge(px[i], k + kl), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) sm[wave][i][lane] = acc[i];
  __syncthreads();
  if (threadIdx.x >= 64 * MB) return;
  // wave i finishes rows 16 i ..: a lane has row 16 i + (lane & 15), columns n0 + 4 (lane >> 4) ..
  const int m = 16 * wave + (lane & 15), n = n0 + 4 * (lane >> 4);
  lin_f4 v = sm[0][wave][lane];
#pragma unroll
  for (int r = 1; r < W; ++r) v += sm[r][wave][lane];
  if (m >= M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= N) continue;
    const size_t at = (size_t)m * N + n + e;
    float z = v[e] + (ep.bias ? ld1(ep.bias + n + e) : 0.f);
    if (ep.z) st1(ep.z + at, z);
    z = lin_act<ACT>(z);
    if (ep.res) z += ld1(ep.res + at);
    st1(ep.y + at, z);
  }
}

// A split contraction's partial products, added in a fixed order, and the epilogue.  SG threads share four columns of a row,
// each adds every SG-th partial: with one a product of few outputs and many splits waits for one load after another (a
// weight gradient of 64 x 256 in 256 splits: 53 us for the product and its sum, 22 with 16).
template <typename T, int ACT, int SG>
__global__ __launch_bounds__(256) void lin_join_k(LinEpi<T> ep, int splits, int M, int N) {
  constexpr int V = 4, U = 4, LANES = 256 / SG;            // columns a thread, partials in flight, column groups a block
  __shared__ float sm[SG > 1 ? SG : 1][SG > 1 ? LANES : 1][V];
  const int chunks = (N + V - 1) / V, lane = threadIdx.x % LANES, sg = threadIdx.x / LANES;
  const size_t mn = (size_t)M * N, all = (size_t)M * chunks;
  for (size_t base = (size_t)blockIdx.x * LANES; base < all; base += (size_t)gridDim.x * LANES) {
    const size_t i = base + lane < all ? base + lane : all - 1;
    const size_t m = i / chunks;
    const int col = (int)(i - m * chunks) * V, cnt = min(N - col, V);
    const float* p = ep.part + m * N + col;
    float v[V], a[U][V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    for (int k = sg; k < splits; k += U * SG) {
#pragma unroll
      for (int u = 0; u < U; ++u) lin_ld<V>(k + u * SG < splits ? p + (size_t)(k + u * SG) * mn : nullptr, cnt, a[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += a[u][e];
    }
    if constexpr (SG > 1) {
      __syncthreads();                                     // the round before has been read
#pragma unroll
      for (int e = 0; e < V; ++e) sm[sg][lane][e] = v[e];
      __syncthreads();
      if (sg != 0) continue;
#pragma unroll
      for (int r = 1; r < SG; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += sm[r][lane][e];
    }
    if (base + lane >= all) continue;
    lin_ld<V>(ep.bias ? ep.bias + col : nullptr, cnt, a[0]);
    lin_ld<V>(ep.res ? ep.res + m * N + col : nullptr, cnt, a[1]);
    lin_finish<ACT>(ep, m * N + col, cnt, a[0], a[1], v);
  }
}

// ---------------------------------------------------------------- gz = g act'(z) and its column sums
// A block owns 64 V columns of a strip of rows, four rows at a time (one per wave): gz written as it is read, the columns'
// sums kept in registers and left as one partial row per block (added in block order by col_sums_k).  gz has a pitch of
// its own, so that rows of an odd length become ones that the products can stream.
// Measured (16 384 x 8192 bf16, GELU): 176 us, 4.6 TB/s of the 805 MB it reads and writes.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void lin_act_bwd_k(const T* __restrict__ g, const T* __restrict__ z, T* __restrict__ gz,
                                                     long long ldg, float* __restrict__ part, int M, int N) {
  constexpr int V = LinT<T>::VE;
  typedef typename LinT<T>::vec vec;
  __shared__ float sm[4][64][V + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = (blockIdx.x * 64 + lane) * V, cnt = min(max(N - n, 0), V);
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (cnt > 0) {
    constexpr int U = 2;                                   // rows in flight a lane, and as many more being fetched
    const long long step = (long long)gridDim.y * 4;
    vec gv[U], zv[U];
    auto fetch = [&](long long m) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t at = (size_t)min(m + u * step, (long long)M - 1) * N + n;
        if (cnt == V) {
          gv[u] = *reinterpret_cast<const vec*>(g + at);
          if (ACT != LIN_NONE) zv[u] = *reinterpret_cast<const vec*>(z + at);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            gv[u][j] = j < cnt ? g[at + j] : (T)0.f;
            if (ACT != LIN_NONE) zv[u][j] = j < cnt ? z[at + j] : (T)0.f;
          }
        }
      }
    };
    long long m = (long long)blockIdx.y * 4 + wave;
    if (m < M) fetch(m);
    while (m < M) {
      float f[U][V], zf[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          f[u][j] = (float)gv[u][j];
          if (ACT != LIN_NONE) zf[u][j] = (float)zv[u][j];
        }
      const long long m0 = m;
      m += U * step;
      if (m < M) fetch(m);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (m0 + u * step >= M) continue;
        vec o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (ACT != LIN_NONE) f[u][j] = lin_back<ACT>(f[u][j], zf[u][j]);
          s[j] += f[u][j];
          o[j] = (T)f[u][j];
        }
        if (gz == nullptr) continue;                       // only the sums are wanted
        const size_t at = (size_t)(m0 + u * step) * ldg + n;
        if (cnt == V) {
          *reinterpret_cast<vec*>(gz + at) = o;
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < cnt) gz[at + j] = o[j];
        }
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int j = 0; j < V; ++j) sm[wave][lane][j] = s[j];
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < cnt)
        part[(size_t)blockIdx.y * N + n + j] = (sm[0][lane][j] + sm[1][lane][j]) + (sm[2][lane][j] + sm[3][lane][j]);
}

// Rows of an odd pitch or start laid out at a pitch of 16 bytes: read across (the gradients' products), 2-byte rows take 2.5
// times as long through registers (12 345 x 1001 x 1367 bf16, data and weight gradient 328 us, 145 with this).
template <typename T>
__global__ __launch_bounds__(256) void lin_pack_k(const T* __restrict__ src, long long lds, T* __restrict__ dst, long long ldd,
                                                  int rows, int cols) {
  const int chunks = (cols + 7) / 8;
  const size_t all = (size_t)rows * chunks;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
    const size_t r = i / chunks;
    const int c = (int)(i - r * chunks) * 8;
    float f[8];
    lin_ld<8>(src + r * lds + c, min(cols - c, 8), f);
    lin_st<8>(dst + r * ldd + c, min(cols - c, 8), f);
  }
}

// ---------------------------------------------------------------- host
constexpr int LIN_CUS = 256;

struct LinPlan {
  int tm, tn, splits;
};

// How often the contraction of a product of TILE x TILE tiles is split, and what it then costs in microseconds: the cheapest
// of splits that fill one to `resident` blocks a CU, of a few small ones and of none.  A block's 128 bytes of contraction
// take `lat` where it is alone on its CU and `thr` of the CU's time where it is not; a round starts and stores in 3, a second
// launch takes 6 and the partial sums their bytes at 8 TB/s (from cache).  Measured on operands that another kernel has just
// written (not in this XCD's L2), 128 x 128: fp32, bound by the matrix cores, 1.9 and 1.8; bf16 0.6 and 0.47, 0.25 and 0.03
// more for each operand that is read across; staged through registers 0.8 more, and 0.6 for each read across.  64 x 64: fp32
// 0.53 and 0.48; bf16 0.25 and 0.2, 0.4 with an operand read across; through registers 0.5 more, and 0.3.  Forward, small and
// large tiles: 1472 x 512 x 768 bf16 6.2 and 9.5 us, 512 x 1024 x 1024 6.8 and 13.3, 2000 x 512 x 512 fp32 13.3 and 23.7, but
// 2048^3 bf16 30 and 25.5.
template <typename T, bool XMC, bool WMC, int TILE>
static LinPlan lin_plan(int M, int N, int K, int resident, bool aligned, bool split, double& best) {
  static_assert(TILE == 64 || TILE == 128, "measured tiles");
  constexpr int BK = 128 / (int)sizeof(T), ACROSS = (int)XMC + (int)WMC;
  constexpr bool SMALL = TILE == 64, WIDE = sizeof(T) == 4;
  const double lat = WIDE    ? (SMALL ? 0.53 : 1.9)
                     : SMALL ? (ACROSS ? 0.4 : 0.25) + (aligned ? 0.0 : 0.5 + 0.3 * ACROSS)
                             : 0.6 + 0.25 * ACROSS + (aligned ? 0.0 : 0.8 + 0.6 * ACROSS);
  const double thr = WIDE ? (SMALL ? 0.48 : 1.8) : SMALL ? 0.2 + 0.04 * ACROSS + (aligned ? 0.0 : 0.1) : 0.47 + 0.03 * ACROSS;
  LinPlan p{(M + TILE - 1) / TILE, (N + TILE - 1) / TILE, 1};
  const long long tiles = (long long)p.tm * p.tn, kt = (K + BK - 1) / BK;
  auto cost = [&](long long s) {
    const long long a_cu = (tiles * s + LIN_CUS - 1) / LIN_CUS, rounds = (a_cu + resident - 1) / resident;
    const double step = std::max(lat * (double)rounds, thr * (double)a_cu);
    return (double)((kt + s - 1) / s) * step + 3.0 * (double)rounds + (s > 1 ? 6.0 + (double)s * M * N * 8 / 8e6 : 0.0);
  };
  best = cost(1);
  if (!split) return p;
  auto offer = [&](long long s) {
    if (s < 2 || s > kt || tiles * s > (long long)LIN_CUS * resident) return;
    const double c = cost(s);
    if (c < best) {
      best = c;
      p.splits = (int)s;
    }
  };
  for (int c = 1; c <= resident; ++c) offer(LIN_CUS * c / tiles);
  for (int s = 2; s <= 8; ++s) offer(s);
  return p;
}

template <typename T, bool XMC, bool WMC, int BM, int BN, int WM, int WN, int OCC, int RB, int SLOTS, bool ASYNC, bool SPLIT>
static int lin_launch(const LinOp<T>& x, const LinOp<T>& w, LinEpi<T> ep, const LinPlan& p, float* part, hipStream_t s) {
  constexpr int bytes = SLOTS * (BM + BN) * RB;
  ep.part = p.splits > 1 ? part : nullptr;
  const unsigned grid = (unsigned)(p.tm * p.tn * p.splits);
  auto launch = [&](auto part_, auto act) {
    auto* fn = lin_tile_k<T, XMC, WMC, BM, BN, WM, WN, OCC, RB, SLOTS, ASYNC, part_(), act()>;
    lds_attr((const void*)fn, bytes);
    fn<<<grid, 64 * WM * WN, bytes, s>>>(x, w, ep, p.tm, p.tn, p.splits);
    return 0;
  };
  const std::integral_constant<int, LIN_NONE> none;
  if constexpr (SPLIT) {
    if (p.splits > 1) {
      launch(std::true_type(), none);
      const size_t chunks = (size_t)x.O * ((w.O + 3) / 4);
      lin_with_act(ep.act, [&](auto act) {
        auto join = [&](auto sg) {
          const size_t blocks = (chunks * sg() + 255) / 256;
          lin_join_k<T, act(), sg()><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(ep, p.splits, x.O, w.O);
        };
        if (p.splits >= 32 && chunks < 256 * 64) join(std::integral_constant<int, 16>());
        else if (p.splits >= 8 && chunks < 256 * 1024) join(std::integral_constant<int, 4>());
        else join(std::integral_constant<int, 1>());
        return 0;
      });
      return fail_launch("linear");
    }
  }
  if constexpr (XMC || WMC)                                // gradients have no activation of their own
    launch(std::false_type(), none);
  else
    lin_with_act(ep.act, [&](auto act) { return launch(std::false_type(), act); });
  return fail_launch("linear");
}

// What the loads that go straight into LDS take: chunks at 4-byte boundaries (all of fp32; bf16 of an even pitch and start)
// and a tile's rows within 31 bits of bytes.  An operand that is read across fills a chunk in every row.
template <typename T>
static bool lin_dwords(const T* p, long long ld) {
  return (((uintptr_t)p | (uintptr_t)ld * sizeof(T)) & 3) == 0;
}
constexpr long long LIN_LD = 1 << 20;
template <typename T, bool MC>
static bool lin_aligned(const LinOp<T>& op) {
  return lin_dwords(op.p, op.ld) && (!MC || op.O >= LinT<T>::VE) && op.ld < LIN_LD;
}

// Which tiles a bf16 product takes.  Both measured with their contraction's length (one box, microseconds): a round of 256
// tiles of 256 x 256 (one a CU, 8 waves) takes 1.6 per 64 contraction values and 9 to start and to store; a round of 512
// tiles of 128 x 128 (two a CU, 4 waves each) 0.95 and 2.1: 8192^3 819 against 970, 16 384 x 2048 x 8192 483 against 518,
// but 92 160 x 256 x 1024 101 against 65 (forward), 23 040 x 1024 x 256 33 against 28.
template <typename T>
static bool lin_big(int M, int N, int K) {
  if (sizeof(T) != 2) return false;
  const long long t256 = (long long)((M + 255) / 256) * ((N + 255) / 256), t128 = (long long)((M + 127) / 128) * ((N + 127) / 128);
  const double kt = K / 64.0;
  const double big = (double)((t256 + LIN_CUS - 1) / LIN_CUS) * (1.6 * kt + 9.0);
  const double half_rounds = (double)((t128 + LIN_CUS - 1) / LIN_CUS);
  return t256 * 2 > LIN_CUS && big < (half_rounds < 2 ? 2 : half_rounds) * 0.5 * (0.95 * kt + 2.1);
}

// 128 x 128 tiles through three 64-byte slots, three blocks a CU, where a block is short (its loads, products and stores
// then overlap another's), or through two 128-byte slots, two blocks a CU.  Measured (microseconds, short / long slots):
// forward 92 160 x 256 x 64 bf16 18 / 22, 23 040 x 256 x 1024 fp32 107 / 114, but 8192 x 2048 x 2048 fp32 588 / 486; data
// gradient at a contraction of 256 97 / 117, of 1024 29 / 24; weight gradient (both operands read across) 95 / 76.
template <bool XMC>
static bool lin_short(int K) {
  return !XMC && K <= 512;
}

// fp32 products are bound by the matrix cores alone: 64-row tiles where 128-row ones leave the last round emptier (by more
// than the tenth that the smaller tiles cost)
template <typename T>
static bool lin_flat(int M, int N) {
  if (sizeof(T) != 4) return false;
  const long long tn = (N + 127) / 128, half = ((M + 63) / 64 * tn + LIN_CUS - 1) / LIN_CUS, full = ((M + 127) / 128 * tn + LIN_CUS - 1) / LIN_CUS;
  return full > 1 && half * 11 <= full * 20;
}

enum LinForm { LIN_F_BIG, LIN_F_FLAT, LIN_F_SHORT, LIN_F_LONG, LIN_F_SMALL };
struct LinChoice {
  LinForm form;
  LinPlan plan;
};
template <typename T, bool XMC, bool WMC>
static LinChoice lin_choose(int M, int N, int K, bool aligned) {
  if (aligned && lin_big<T>(M, N, K)) return {LIN_F_BIG, LinPlan{(M + 255) / 256, (N + 255) / 256, 1}};
  if (aligned && lin_flat<T>(M, N)) return {LIN_F_FLAT, LinPlan{(M + 63) / 64, (N + 127) / 128, 1}};
  constexpr int SMALL_RESIDENT = 3;                        // of three 16 KB slots each (two slots, four blocks: 1000 x 2048 x 1000 17.8 us, 11.3)
  double small_us, us;
  const LinPlan small = lin_plan<T, XMC, WMC, 64>(M, N, K, SMALL_RESIDENT, aligned, true, small_us);
  const bool brief = lin_short<XMC>(K);
  const LinPlan large = lin_plan<T, XMC, WMC, 128>(M, N, K, brief ? 3 : 2, aligned, !brief, us);      // (a short contraction is split in small tiles)
  if (small_us < us && (long long)small.tm * small.tn < (1 << 24)) return {LIN_F_SMALL, small};
  return {brief ? LIN_F_SHORT : LIN_F_LONG, large};
}

template <typename T, bool XMC, bool WMC, bool ASYNC>
static int lin_sized(const LinOp<T>& x, const LinOp<T>& w, const LinEpi<T>& ep, float* part, hipStream_t s) {
  const LinChoice c = lin_choose<T, XMC, WMC>(x.O, w.O, x.K, ASYNC);
  if constexpr (ASYNC) {
    if constexpr (sizeof(T) == 2)
      if (c.form == LIN_F_BIG) return lin_launch<T, XMC, WMC, 256, 256, 2, 4, 2, 128, 2, ASYNC, false>(x, w, ep, c.plan, part, s);
    if constexpr (sizeof(T) == 4)
      if (c.form == LIN_F_FLAT) return lin_launch<T, XMC, WMC, 64, 128, 2, 2, 3, 128, 2, ASYNC, false>(x, w, ep, c.plan, part, s);
  }
  if (c.form == LIN_F_SMALL) return lin_launch<T, XMC, WMC, 64, 64, 2, 2, 3, 128, 3, ASYNC, true>(x, w, ep, c.plan, part, s);
  if constexpr (!XMC)
    if (c.form == LIN_F_SHORT) return lin_launch<T, XMC, WMC, 128, 128, 2, 2, 3, 64, 3, ASYNC, false>(x, w, ep, c.plan, part, s);
  return lin_launch<T, XMC, WMC, 128, 128, 2, 2, 2, 128, 2, ASYNC, true>(x, w, ep, c.plan, part, s);
}

template <typename T, bool XMC, bool WMC>
static int lin_product(const LinOp<T>& x, const LinOp<T>& w, const LinEpi<T>& ep, float* part, hipStream_t s) {
  if (lin_aligned<T, XMC>(x) && lin_aligned<T, WMC>(w)) return lin_sized<T, XMC, WMC, true>(x, w, ep, part, s);
  return lin_sized<T, XMC, WMC, false>(x, w, ep, part, s);
}

// Of whichever of the two forms (by alignment, which a descriptor does not say) needs more
template <typename T, bool XMC, bool WMC>
static size_t lin_part_bytes(int M, int N, int K) {
  const int a = lin_choose<T, XMC, WMC>(M, N, K, true).plan.splits, b = lin_choose<T, XMC, WMC>(M, N, K, false).plan.splits;
  const int splits = a > b ? a : b;
  return splits > 1 ? (size_t)splits * M * N * sizeof(float) : 0;
}

// Row blocks of lin_act_bwd_k, 1024 blocks in all.  Without an activation (g read, its blocks' sums written; the launch that
// adds them, 4 to 5 us, is not counted): 92 160 x 256 bf16 13.1 us, 15.9 with 2048 and 21.2 with 4096; 16 384 x 8192 48.3, 51
// and 55; 23 040 x 1024 fp32 18.4, 19.1 and 19.7.
static int lin_strips(int M, int N, int V) {
  const int cb = (N + 64 * V - 1) / (64 * V), most = 1024 / cb > 0 ? 1024 / cb : 1, need = (M + 15) / 16;
  return need < most ? need : most;
}

// (a launch holds under 2^32 threads)
static bool lin_is_thin(const vfd_linear_desc* d) { return d->rows <= LIN_THIN && d->n <= (1 << 26); }

template <typename T>
static size_t lin_fwd_ws(const vfd_linear_desc* d) {
  return lin_is_thin(d) ? 0 : lin_part_bytes<T, false, false>(d->rows, d->n, d->k);
}

// The backward's workspace: gz (where an activation makes one for a product, or g cannot be streamed), copies of W and x where those
// cannot, and one scratch for the steps' partial sums, which follow each other on one stream.
struct LinBwdPlan {
  long long ldg, ldw, ldx;       // pitches of the operands that the products read
  bool gz, w, x;                 // whether each is a copy in the workspace
  size_t at_gz, at_w, at_x, at_part, bytes;
};
template <typename T>
static LinBwdPlan lin_bwd_plan(const vfd_linear_desc* d, const void* g, const void* w, const void* x, bool dx, bool dw) {
  // whole cache lines where that adds at most a sixteenth (12 345 x 1001 x 1367: 62.8 and 81.0 us, 66.4 and 85.2 without;
  // 60 001 x 333 x 777, where it would add a sixth: 104 and 131 us, 108 and 120 without)
  auto pitch = [](long long n) { return (n + 63) / 64 * 64 * 16 <= n * 17 ? (n + 63) / 64 * 64 : (n + 7) / 8 * 8; };
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  LinBwdPlan p;
  // A copy is made for a product whose operands can both be streamed with it (lin_aligned), for a whole tile of contraction at
  // least: never for one of fewer than VE values a row, or of a contraction that ends inside its first tile (both gradients
  // of 2 000 000 x 255 x 3 809 us and 1 MB of workspace, 2015 us and 1.06 GB with copies that nothing streamed).
  // A product of few terms is not worth copies of its operands (both gradients, with and without: 20 001 x 255 x 257 60 and
  // 50 us, 2000 x 1001 x 1003 51 and 58).
  constexpr int VE = LinT<T>::VE, TILE = 64 / (int)sizeof(T);
  const bool pack = (double)d->rows * d->k * d->n > 1.5e9;
  const bool bad_g = !lin_dwords((const T*)g, d->n), bad_w = !lin_dwords((const T*)w, d->k), bad_x = !lin_dwords((const T*)x, d->ldx);
  const long long ldg = d->act != LIN_NONE || bad_g ? pitch(d->n) : d->n, ldw = bad_w ? pitch(d->k) : d->k,
                  ldx = bad_x ? pitch(d->k) : d->ldx;
  const bool for_dx = pack && dx && d->n >= TILE && d->k >= VE && ldg < LIN_LD && ldw < LIN_LD;
  const bool for_dw = pack && dw && d->rows >= TILE && d->n >= VE && d->k >= VE && ldg < LIN_LD && ldx < LIN_LD;
  p.gz = (d->act != LIN_NONE && (dx || dw)) || (bad_g && (for_dx || for_dw));
  p.w = bad_w && for_dx;
  p.x = bad_x && for_dw;
  p.ldg = p.gz ? ldg : d->n;
  p.ldw = p.w ? ldw : d->k;
  p.ldx = p.x ? ldx : d->ldx;
  p.at_gz = 0;
  p.at_w = p.at_gz + up(p.gz ? (size_t)d->rows * p.ldg * sizeof(T) : 0);
  p.at_x = p.at_w + up(p.w ? (size_t)d->n * p.ldw * sizeof(T) : 0);
  p.at_part = p.at_x + up(p.x ? (size_t)d->rows * p.ldx * sizeof(T) : 0);
  const size_t act = (size_t)lin_strips(d->rows, d->n, LinT<T>::VE) * d->n * sizeof(float);
  const size_t sx = dx ? lin_part_bytes<T, false, true>(d->rows, d->k, d->n) : 0;
  const size_t sw = dw ? lin_part_bytes<T, true, true>(d->n, d->k, d->rows) : 0;
  p.bytes = p.at_part + std::max(act, std::max(sx, sw));
  return p;
}

static int lin_check(const char* what, const vfd_linear_desc* d) {
  VFD_REQUIRE(d && d->rows >= 0 && d->k >= 1 && d->n >= 1 && d->rows <= VFD_LINEAR_MAX && d->k <= VFD_LINEAR_MAX &&
                  d->n <= VFD_LINEAR_MAX && d->ldx >= d->k && d->act >= 0 && d->act < LIN_ACTS && (d->dtype == 0 || d->dtype == 1),
              "%s: bad descriptor", what);
  const long long T = 128;                                 // (a launch holds under 2^32 threads)
  VFD_REQUIRE(((long long)d->rows / T + 1) * (d->n / T + 1) < (1 << 24) && ((long long)d->rows / T + 1) * (d->k / T + 1) < (1 << 24) &&
                  ((long long)d->n / T + 1) * (d->k / T + 1) < (1 << 24),
              "%s: too many tiles", what);
  return VFD_OK;
}

template <typename T>
static int lin_fwd_run(const vfd_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y,
                       void* z, float* part, hipStream_t s) {
  const LinOp<T> ox{(const T*)x, d->ldx, d->rows, d->k}, ow{(const T*)w, d->k, d->n, d->k};
  const LinEpi<T> ep{(const T*)bias, (const T*)res, (T*)z, (T*)y, nullptr, d->act};
  if (lin_is_thin(d)) {
    lin_with_act(d->act, [&](auto act) {
      const unsigned grid = (unsigned)((d->n + 15) / 16);
      if (d->rows <= 16) lin_thin_k<T, 1, act()><<<grid, 512, 0, s>>>(ox, ow, ep);
      else if (d->rows <= 32) lin_thin_k<T, 2, act()><<<grid, 512, 0, s>>>(ox, ow, ep);
      else lin_thin_k<T, 4, act()><<<grid, 512, 0, s>>>(ox, ow, ep);
      return 0;
    });
    return fail_launch("linear_fwd");
  }
  return lin_product<T, false, false>(ox, ow, ep, part, s);
}

template <typename T>
static void lin_pack(const T* src, long long lds, T* dst, long long ldd, int rows, int cols, hipStream_t s) {
  const size_t chunks = (size_t)rows * ((cols + 7) / 8), blocks = (chunks + 255) / 256;
  lin_pack_k<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>(src, lds, dst, ldd, rows, cols);
}

template <typename T>
static int lin_bwd_run(const vfd_linear_desc* d, const T* g, const T* z, const T* w, const T* x, T* dx, T* dw, T* db, char* ws,
                       hipStream_t s) {
  const LinBwdPlan p = lin_bwd_plan<T>(d, g, w, x, dx != nullptr, dw != nullptr);
  float* part = (float*)(ws + p.at_part);
  const LinEpi<T> plain{nullptr, nullptr, nullptr, nullptr, nullptr, LIN_NONE};
  if (p.gz || db) {
    T* gz = p.gz ? (T*)(ws + p.at_gz) : nullptr;
    const int strips = lin_strips(d->rows, d->n, LinT<T>::VE);
    const dim3 grid(cdiv(d->n, 64 * LinT<T>::VE), strips);
    lin_with_act(d->act, [&](auto act) {
      lin_act_bwd_k<T, act()><<<grid, 256, 0, s>>>(g, z, gz, p.ldg, db ? part : nullptr, d->rows, d->n);
      return 0;
    });
    if (db) col_sums_k<T><<<col_sums_grid(d->n), 1024, 0, s>>>(part, strips, d->n, d->n, db, nullptr);
    if (int e = fail_launch("linear_bwd activation")) return e;
    if (gz) g = gz;
  }
  if (dx) {
    if (p.w) {
      T* c = (T*)(ws + p.at_w);
      lin_pack(w, d->k, c, p.ldw, d->n, d->k, s);
      w = c;
    }
    LinEpi<T> ep = plain;
    ep.y = dx;
    const LinOp<T> og{g, p.ldg, d->rows, d->n}, ow{w, p.ldw, d->k, d->n};
    if (int e = lin_product<T, false, true>(og, ow, ep, part, s)) return e;
  }
  if (dw) {
    if (p.x) {
      T* c = (T*)(ws + p.at_x);
      lin_pack(x, d->ldx, c, p.ldx, d->rows, d->k, s);
      x = c;
    }
    LinEpi<T> ep = plain;
    ep.y = dw;
    const LinOp<T> og{g, p.ldg, d->n, d->rows}, ox{x, p.ldx, d->k, d->rows};
    if (int e = lin_product<T, true, true>(og, ox, ep, part, s)) return e;
  }
  return VFD_OK;
}

}  // namespace vfd

using namespace vfd;

extern "C" {

size_t vfd_linear_fwd_workspace(const vfd_linear_desc* d) {
  if (lin_check("linear", d) != VFD_OK || d->rows == 0) return 0;
  return d->dtype ? lin_fwd_ws<__bf16>(d) : lin_fwd_ws<float>(d);
}

int vfd_linear_fwd(const vfd_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z,
                   void* workspace, size_t ws_bytes, void* stream) {
  if (int e = lin_check("linear_fwd", d)) return e;
  if (d->rows == 0) return VFD_OK;
  VFD_REQUIRE(y && x && w, "linear_fwd: null tensor");
  const size_t need = vfd_linear_fwd_workspace(d);
  VFD_REQUIRE(need == 0 || (workspace && ws_bytes >= need), "linear_fwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_LINEAR_FWD, s);
  return (d->dtype ? lin_fwd_run<__bf16> : lin_fwd_run<float>)(d, x, w, bias, res, y, z, (float*)workspace, s);
}

size_t vfd_linear_bwd_workspace(const vfd_linear_desc* d, const void* g, const void* w, const void* x, int dx, int dw) {
  if (lin_check("linear", d) != VFD_OK || d->rows == 0) return 0;
  return (d->dtype ? lin_bwd_plan<__bf16> : lin_bwd_plan<float>)(d, g, w, x, dx != 0, dw != 0).bytes;
}

int vfd_linear_bwd(const vfd_linear_desc* d, const void* g, const void* z, const void* w, const void* x, void* dx, void* dw,
                   void* db, void* workspace, size_t ws_bytes, void* stream) {
  if (int e = lin_check("linear_bwd", d)) return e;
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof(K_LINEAR_BWD, s);
  const size_t es = d->dtype ? 2 : 4;
  if (d->rows == 0) {
    if (dw) zero_async(dw, (size_t)d->n * d->k * es, s);
    if (db) zero_async(db, (size_t)d->n * es, s);
    return fail_launch("linear_bwd");
  }
  if (!dx && !dw && !db) return VFD_OK;
  VFD_REQUIRE(g && (d->act == LIN_NONE || z) && (!dx || w) && (!dw || x), "linear_bwd: null tensor");
  VFD_REQUIRE(workspace && ws_bytes >= vfd_linear_bwd_workspace(d, g, w, x, dx != nullptr, dw != nullptr),
              "linear_bwd: workspace too small");
  if (d->dtype)
    return lin_bwd_run<__bf16>(d, (const __bf16*)g, (const __bf16*)z, (const __bf16*)w, (const __bf16*)x, (__bf16*)dx, (__bf16*)dw,
                               (__bf16*)db, (char*)workspace, s);
  return lin_bwd_run<float>(d, (const float*)g, (const float*)z, (const float*)w, (const float*)x, (float*)dx, (float*)dw, (float*)db,
                            (char*)workspace, s);
}

}  // extern "C"
