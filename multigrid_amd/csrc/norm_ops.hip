// Layer norm with its gradients, and clipping by the global gradient norm (include/mgrid_norm.h): the normalisation of the
// PPO trainer's policies and of their gradients.  Both are bound by HBM traffic; every element is moved 16 bytes per lane.
// Rows and gradients may start at any element: gfx950 loads and stores 16 bytes at any address of an element's alignment,
// so a row of odd length takes the same path as an even one: its last vector ends at its end and overlaps the one before.
// Rows shorter than one vector move element by element, and so does the last, shorter vector of a gradient.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "mgrid_norm.h"

namespace {

constexpr int kWave = 64;

// ---- element types: 16 bytes of T as floats and back (round to nearest even) ----
template <typename T>
struct Pack {
  static constexpr int V = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(V)));
  typedef Vec VecAny __attribute__((aligned(sizeof(T))));
  static __device__ __forceinline__ Vec load(const T* p) { return *reinterpret_cast<const VecAny*>(p); }
  static __device__ __forceinline__ void store(T* p, Vec v) { *reinterpret_cast<VecAny*>(p) = v; }
  static __device__ __forceinline__ void store_past_caches(T* p, Vec v) { __builtin_nontemporal_store(v, reinterpret_cast<VecAny*>(p)); }
};

// the vector at element `col` of a row of C elements; elements past the end (and whole vectors past it) are 0
template <typename T>
__device__ __forceinline__ typename Pack<T>::Vec load_part(const T* row, int col, int C) {
  constexpr int V = Pack<T>::V;
  if (col + V <= C) return Pack<T>::load(row + col);
  typename Pack<T>::Vec v;
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = col + k < C ? row[col + k] : (T)0.f;
  return v;
}

template <typename T>
__device__ __forceinline__ void store_part(T* row, int col, int C, typename Pack<T>::Vec v) {
  constexpr int V = Pack<T>::V;
  if (col + V <= C) {
    Pack<T>::store(row + col, v);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (col + k < C) row[col + k] = v[k];
  }
}

__device__ __forceinline__ void store_from_float(void* p, int type, int64_t i, float v) {
  if (type == MGNN_F32) static_cast<float*>(p)[i] = v;
  else if (type == MGNN_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// Sum over aligned groups of L lanes, in every lane of the group (all 64 lanes take part), on the vector units alone: lane
// permutations within 16 lanes, then whole rows of 16 and halves of the wave swapped between two registers.  float or double.
template <int CTRL, typename F>
__device__ __forceinline__ F dpp_add(F v) {
  if constexpr (sizeof(F) == 4) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
  } else {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
    return v + __hiloint2double(hi, lo);
  }
}
template <bool HALVES, typename F>      // + the other half of the wave, or the other 16 lanes of a half
__device__ __forceinline__ F swap_add(F v) {
  auto both = [](unsigned u) {
    if constexpr (HALVES) return __builtin_amdgcn_permlane32_swap(u, u, false, false);
    else return __builtin_amdgcn_permlane16_swap(u, u, false, false);
  };
  if constexpr (sizeof(F) == 4) {
    const auto r = both(__float_as_uint(v));
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const auto lo = both((unsigned)__double2loint(v)), hi = both((unsigned)__double2hiint(v));
    return __hiloint2double((int)hi[0], (int)lo[0]) + __hiloint2double((int)hi[1], (int)lo[1]);
  }
}
template <int L, typename F>
__device__ __forceinline__ F lanes_sum(F v) {
  if constexpr (L >= 2) v = dpp_add<0xB1>(v);       // lane ^ 1
  if constexpr (L >= 4) v = dpp_add<0x4E>(v);       // lane ^ 2
  if constexpr (L >= 8) v = dpp_add<0x141>(v);      // mirrored within 8: the other four lanes
  if constexpr (L >= 16) v = dpp_add<0x140>(v);     // mirrored within 16: the other eight
  if constexpr (L >= 32) v = swap_add<false>(v);
  if constexpr (L >= 64) v = swap_add<true>(v);
  return v;
}

// ---- layer norm ----
// TPR threads share a row, thread t holding the vectors t, t + TPR, ... (NV of them) in registers, so a row is read once;
// a workgroup works on SLOTS rows at a time.  Rows of up to 64 * NV vectors belong to part of a wave or a whole one and need
// no barrier; longer ones to several waves.
template <int TPR>
struct Shape {
  static constexpr int BLOCK = TPR > 256 ? TPR : 256;
  static constexpr int SLOTS = BLOCK / TPR;
  static constexpr int WAVES = BLOCK / kWave;
  static constexpr int L = TPR < kWave ? TPR : kWave;              // lanes of a wave that share a row
  static constexpr int ROW_WAVES = TPR > kWave ? TPR / kWave : 1;
};

// Where a thread's vectors lie in a row of C elements.  FULL: the row is exactly TPR * NV vectors.  Else the last vector of
// a row whose length is no multiple of V ends at the row's end and overlaps the one before by `dup` elements, which it
// loads and stores like the rest (both threads compute the same values) but leaves out of sums; rows shorter than one
// vector are moved element by element.  With several vectors per thread the row is longer than half of TPR * NV vectors
// (row_split), so the first half of them lies inside it.
template <typename T, int TPR, int NV, bool FULL>
struct Cols {
  static constexpr int V = Pack<T>::V;
  int at[NV], dup[NV];      // first column, leading elements that another thread counts (V: no vector)
  int C;
  __device__ __forceinline__ Cols(int lane, int C_) : C(C_) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (lane + i * TPR) * V;
      at[i] = inside(i) ? col : max(min(col, C - V), 0);
      dup[i] = inside(i) ? 0 : min(col - at[i], V);
    }
  }
  static __device__ __forceinline__ constexpr bool inside(int i) { return FULL || i < NV / 2; }
  // whether element k of vector i counts (a vector that ends past C starts at column 0 of a row shorter than itself)
  __device__ __forceinline__ bool counts(int i, int k) const { return inside(i) || (k >= dup[i] && (NV > 1 || k < C)); }
  __device__ __forceinline__ int count() const {
    if (FULL) return NV * V;
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) n += max(min(V, C) - dup[i], 0);
    return n;
  }
  __device__ __forceinline__ void load(const T* row, bool live, typename Pack<T>::Vec (&v)[NV]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = {};
      if (live && (inside(i) || dup[i] < V)) {
        if (NV > 1 || FULL || C >= V) {
          v[i] = Pack<T>::load(row + at[i]);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k < C) v[i][k] = row[k];
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int i, typename Pack<T>::Vec v) const {
    if (!inside(i) && dup[i] >= V) return;
    if (NV > 1 || FULL || C >= V) {
      Pack<T>::store(row + at[i], v);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k < C) row[k] = v[k];
    }
  }
  // a weight or bias row (NULL: `other`)
  __device__ __forceinline__ void load_weight(const void* p, int type, int64_t row, float other, float (&w)[NV * V]) const {
#pragma unroll
    for (int k = 0; k < NV * V; ++k) w[k] = other;
    if (!p) return;
    if (type == MGNN_F32) {
      const float* f = static_cast<const float*>(p) + row * C;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!inside(i) && dup[i] >= V) continue;
        if (NV > 1 || FULL || C >= V) {
#pragma unroll
          for (int j = 0; j < V; j += 4) {
            const auto q = Pack<float>::load(f + at[i] + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[i * V + j + k] = q[k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k < C) w[i * V + k] = f[k];
        }
      }
    } else {      // x's own 16-bit type
      typename Pack<T>::Vec v[NV];
      load(static_cast<const T*>(p) + row * C, true, v);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) w[i * V + k] = (float)v[i][k];
    }
  }
};

// sum / n for the sum of n values, with the rounding of inv_n = fl(1 / n) taken out again: exact where the quotient is a float
__device__ __forceinline__ float divide(float sum, float n, float inv_n) {
  const float q = sum * inv_n;
  return __builtin_fmaf(__builtin_fmaf(-q, n, sum), inv_n, q);
}

// Mean and sum of squared deviations of a row in the registers of TPR threads: passes over the registers, so no digits cancel.
// The mean is origin + shift, `origin` being a first mean that all of the row's threads share (so that two of them that hold the
// same element agree about it), and a deviation is (x - origin) - shift.
// Where a row's elements lie close together, far from 0, the first mean's roundings are large beside their deviations (and all
// there is of them in a row of equal values).  In 16 bits such elements add up exactly in fp32, a wave's 1024 at most, and the
// quotient is rounded once.  In 32 bits the deviations from the first mean, which are exact there, are added up once more:
// 3 x 4096 rows of 128 4.27 -> 4.43 us, 509 of 16381 15.4 -> 15.9, 3 x 409600 of 128 as before (226); 16-bit rows 0 to 2 %.
// n, inv_n: the wave's elements of the row.  Rows over several waves: each wave's own mean m_w and deviations M_w, combined as
// M = sum of M_w + n_w (m_w - m)^2, which takes one barrier instead of two; `origin` is the first wave's first mean.
template <typename T, int TPR, int NV, bool FULL>
__device__ __forceinline__ void row_stats(const float (&v)[NV * Pack<T>::V], const Cols<T, TPR, NV, FULL>& cols, float n, float inv_n,
                                          float inv_c, float4 (*red)[Shape<TPR>::WAVES], int parity, float& origin, float& shift, float& m2) {
  constexpr int V = Pack<T>::V, L = Shape<TPR>::L;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV * V; ++k) s += cols.counts(k / V, k % V) ? v[k] : 0.f;
  origin = divide(lanes_sum<L>(s), n, inv_n);
  shift = 0.f;
  if constexpr (sizeof(T) == 4) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < NV * V; ++k) s += cols.counts(k / V, k % V) ? v[k] - origin : 0.f;
    shift = divide(lanes_sum<L>(s), n, inv_n);
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NV * V; ++k) {
    const float d = cols.counts(k / V, k % V) ? (v[k] - origin) - shift : 0.f;
    q = __builtin_fmaf(d, d, q);
  }
  m2 = lanes_sum<L>(q);
  if constexpr (TPR > kWave) {
    constexpr int W = Shape<TPR>::ROW_WAVES;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) red[parity][wave] = make_float4(origin, shift, m2, n);
    __syncthreads();
    const float4 r = red[parity][wave / W * W + threadIdx.x % W];      // each lane one wave's, then a sum over lanes
    origin = red[parity][wave / W * W].x;
    const float at = (r.x - origin) + r.y;
    shift = divide(lanes_sum<W>(r.w * at), (float)cols.C, inv_c);
    const float d = at - shift;
    m2 = lanes_sum<W>(r.w > 0.f ? __builtin_fmaf(r.w * d, d, r.z) : 0.f);
  }
}

// y = (x - m) s w + b.  Bound by HBM, each element read once and written once: 3 x 409600 rows of 128 fp32 222 us (5.7 TB/s),
// 16384 of 4096 bf16 46 us (5.8); at 3 x 4096 rows of 128 fp32 4.2 us, a launch and one trip to memory.
template <typename T, int TPR, int NV, bool FULL>
__global__ __launch_bounds__(Shape<TPR>::BLOCK) void ln_fwd_kernel(const T* x, int64_t ld, const void* weight, const void* bias,
                                                                   int wtype, T* y, float2* stats, int64_t rows, int C, float eps) {
  constexpr int V = Pack<T>::V, NE = NV * V, SLOTS = Shape<TPR>::SLOTS, L = Shape<TPR>::L;
  __shared__ float4 red[2][Shape<TPR>::WAVES];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t g = blockIdx.y, step = (int64_t)gridDim.x * SLOTS;
  const Cols<T, TPR, NV, FULL> cols(lane, C);
  const float n = lanes_sum<L>((float)cols.count()), inv_n = n > 0.f ? 1.f / n : 0.f, inv_c = 1.f / (float)C;
  x += g * rows * ld;
  y += g * rows * C;
  int64_t base = (int64_t)blockIdx.x * SLOTS, row = base + slot;
  typename Pack<T>::Vec next[NV];
  cols.load(x + row * ld, row < rows, next);
  float w[NE], b[NE];
  cols.load_weight(weight, wtype, g, 1.f, w);
  cols.load_weight(bias, wtype, g, 0.f, b);
  int parity = 0;
  for (; base < rows; base += step, row += step, parity ^= 1) {
    float v[NE];
#pragma unroll
    for (int k = 0; k < NE; ++k) v[k] = (float)next[k / V][k % V];
    cols.load(x + (row + step) * ld, row + step < rows, next);      // under the sums of this row
    float origin, shift, m2;
    row_stats<T, TPR, NV, FULL>(v, cols, n, inv_n, inv_c, red, parity, origin, shift, m2);
    const float rstd = rsqrtf(__builtin_fmaf(m2, inv_c, eps));
    if (row < rows) {
      if (stats && lane == 0) stats[g * rows + row] = make_float2(origin + shift, rstd);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        typename Pack<T>::Vec p;
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] = (T)__builtin_fmaf(((v[i * V + k] - origin) - shift) * rstd, w[i * V + k], b[i * V + k]);
        cols.store(y + row * C, i, p);
      }
    }
  }
}

// Sum over the rows that a workgroup's slots hold of one value per column, in slot 0 (threads below TPR): over the lanes of
// a wave that hold the same columns, then over the waves, halving.  Every thread of the workgroup takes part.
template <int TPR, int NE>
__device__ __forceinline__ void slots_sum(float (&acc)[NE], float* lds) {
  constexpr int WAVES = Shape<TPR>::WAVES;
  if constexpr (TPR < kWave) {
#pragma unroll
    for (int k = 0; k < NE; ++k)
#pragma unroll
      for (int s = TPR; s < kWave; s <<= 1) acc[k] += __shfl_xor(acc[k], s);
  }
  constexpr int SETS = TPR < kWave ? WAVES : Shape<TPR>::SLOTS;      // waves or groups of waves that hold the same columns
  constexpr int WIDTH = TPR < kWave ? kWave : TPR;
  const int set = threadIdx.x / WIDTH, at = threadIdx.x % WIDTH;
#pragma unroll
  for (int half = SETS / 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (set >= half && set < 2 * half) {
#pragma unroll
      for (int k = 0; k < NE; ++k) lds[((set - half) * NE + k) * WIDTH + at] = acc[k];
    }
    __syncthreads();
    if (set < half) {
#pragma unroll
      for (int k = 0; k < NE; ++k) acc[k] += lds[(set * NE + k) * WIDTH + at];
    }
  }
}

// dx = s (e - mean(e) - h mean(e h)) with e = dy w, and the sums of dy h and dy over this workgroup's rows.  Bound by HBM, x
// and dy read once, dx written once: 3 x 409600 rows of 128 fp32 370 us (5.1 TB/s), 16384 of 4096 bf16 86 us (4.7); 509 rows
// of 16381 fp32, four to each of 128 workgroups, 31 us (3.8 TB/s), a seventh of the traffic shares.
// partial: [groups][blocks][2][C] floats (this workgroup's shares of dweight and dbias), or NULL with one block per group:
// then dweight / dbias are written here
template <typename T, int TPR, int NV, bool FULL>
__global__ __launch_bounds__(Shape<TPR>::BLOCK) void ln_bwd_kernel(const T* x, int64_t ld, const T* dy, const void* weight,
                                                                   int wtype, const float2* stats, T* dx, float* partial,
                                                                   void* dweight, void* dbias, int64_t rows, int C) {
  constexpr int V = Pack<T>::V, NE = NV * V, SLOTS = Shape<TPR>::SLOTS, WAVES = Shape<TPR>::WAVES, L = Shape<TPR>::L;
  constexpr int SETS = TPR < kWave ? WAVES : SLOTS, WIDTH = TPR < kWave ? kWave : TPR;
  // 16 elements a thread in workgroups of 1024: the running sums take 128 KB of LDS, so that the next row fits the registers
  constexpr bool SUMS_IN_LDS = TPR == 1024 && NE >= 16;
  __shared__ float2 red[2][WAVES];
  __shared__ float fold[SUMS_IN_LDS ? 2 * NE * TPR : SETS > 1 ? SETS / 2 * NE * WIDTH : 1];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t g = blockIdx.y, step = (int64_t)gridDim.x * SLOTS;
  const Cols<T, TPR, NV, FULL> cols(lane, C);
  const float inv_c = 1.f / (float)C;
  x += g * rows * ld;
  dy += g * rows * C;
  stats += g * rows;
  int64_t base = (int64_t)blockIdx.x * SLOTS, row = base + slot;
  typename Pack<T>::Vec next_x[NV], next_d[NV];
  float2 next_st = row < rows ? stats[row] : make_float2(0.f, 0.f);
  cols.load(x + row * ld, row < rows, next_x);
  cols.load(dy + row * C, row < rows, next_d);
  float w[NE], aw[NE], ab[NE];
  cols.load_weight(weight, wtype, g, 1.f, w);
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    aw[k] = ab[k] = 0.f;
    if constexpr (SUMS_IN_LDS) fold[k * TPR + lane] = fold[(NE + k) * TPR + lane] = 0.f;
  }
  int parity = 0;
  for (; base < rows; base += step, row += step, parity ^= 1) {
    const float2 st = next_st;
    float h[NE], e[NE];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      const float d = (float)next_d[j / V][j % V];      // 0 past the row's end and past the last row
      h[j] = ((float)next_x[j / V][j % V] - st.x) * st.y;
      e[j] = d * w[j];
      s1 += cols.counts(j / V, j % V) ? e[j] : 0.f;
      s2 += cols.counts(j / V, j % V) ? e[j] * h[j] : 0.f;
      if constexpr (SUMS_IN_LDS) {
        fold[j * TPR + lane] = __builtin_fmaf(d, h[j], fold[j * TPR + lane]);
        fold[(NE + j) * TPR + lane] += d;
      } else {
        aw[j] = __builtin_fmaf(d, h[j], aw[j]);
        ab[j] += d;
      }
    }
    const bool more = row + step < rows;
    next_st = more ? stats[row + step] : make_float2(0.f, 0.f);
    cols.load(x + (row + step) * ld, more, next_x);
    cols.load(dy + (row + step) * C, more, next_d);
    if (dx) {
      s1 = lanes_sum<L>(s1);
      s2 = lanes_sum<L>(s2);
      if constexpr (TPR > kWave) {
        constexpr int W = Shape<TPR>::ROW_WAVES;
        const int wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0) red[parity][wave] = make_float2(s1, s2);
        __syncthreads();
        const float2 r = red[parity][wave / W * W + threadIdx.x % W];
        s1 = lanes_sum<W>(r.x);
        s2 = lanes_sum<W>(r.y);
      }
      s1 *= inv_c;
      s2 *= inv_c;
      if (row < rows) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          typename Pack<T>::Vec p;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int j = i * V + k;
            p[k] = (T)(st.y * (e[j] - __builtin_fmaf(h[j], s2, s1)));
          }
          cols.store(dx + (g * rows + row) * C, i, p);
        }
      }
    }
  }
  if (!dweight && !dbias) return;
  if constexpr (SUMS_IN_LDS) {
#pragma unroll
    for (int k = 0; k < NE; ++k) aw[k] = fold[k * TPR + lane], ab[k] = fold[(NE + k) * TPR + lane];
  } else {
    slots_sum<TPR, NE>(aw, fold);
    slots_sum<TPR, NE>(ab, fold);
  }
  if (threadIdx.x >= TPR) return;
  float* share = partial ? partial + (g * gridDim.x + blockIdx.x) * 2 * C : nullptr;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    if (!cols.counts(j / V, j % V)) continue;
    const int col = cols.at[j / V] + j % V;
    if (share) {
      share[col] = aw[j];
      share[C + col] = ab[j];
    } else {
      if (dweight) store_from_float(dweight, wtype, g * C + col, aw[j]);
      if (dbias) store_from_float(dbias, wtype, g * C + col, ab[j]);
    }
  }
}

// dweight / dbias of group blockIdx.y from the workgroups' shares, in a fixed order: 32 columns x 32 slices of the blocks,
// sixteen loads in flight a thread.  4.5 to 5 us at up to 1024 shares of a few thousand columns, most of it a launch and two
// trips to memory; 8.3 us for 128 shares of 2 x 16381 (2.0 TB/s): each thread's four loads are in flight at once, and then none.
constexpr int kJoinCols = 32, kJoinSlices = 32;
static_assert(kJoinCols == kJoinSlices);      // the transposed read
__global__ __launch_bounds__(kJoinCols* kJoinSlices) void ln_join_kernel(const float* partial, int blocks, int C, void* dweight,
                                                                         void* dbias, int wtype) {
  __shared__ float red[kJoinSlices][kJoinCols + 1];
  const int64_t g = blockIdx.y;
  const int c = threadIdx.x % kJoinCols, s = threadIdx.x / kJoinCols;
  const int64_t col = (int64_t)blockIdx.x * kJoinCols + c;
  float acc = 0.f;
  if (col < 2 * C) {
    const float* p = partial + g * blocks * 2 * C + col;
#pragma unroll 16
    for (int k = s; k < blocks; k += kJoinSlices) acc += p[(int64_t)k * 2 * C];
  }
  red[s][c] = acc;
  __syncthreads();
  // now 32 lanes of a wave hold a column's slices
  const float sum = lanes_sum<kJoinSlices>(red[c][s]);
  const int64_t out_col = (int64_t)blockIdx.x * kJoinCols + s;
  if (c == 0 && out_col < 2 * C) {
    void* out = out_col < C ? dweight : dbias;
    if (out) store_from_float(out, wtype, g * C + (out_col < C ? out_col : out_col - C), sum);
  }
}

// Enqueues a kernel.  The status is the launch's own: the thread's last error may be an older one, of another call.
template <typename T>
struct Same { using type = T; };
template <typename... P>
int launch(void (*kernel)(P...), dim3 grid, int block, hipStream_t stream, const typename Same<P>::type&... args) {
  void* list[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  if (hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(block), list, 0, stream) == hipSuccess) return MGNN_OK;
  (void)hipGetLastError();      // reported here
  return MGNN_ERR_LAUNCH;
}

int elem_bytes(int type) { return type == MGNN_F32 ? 4 : type == MGNN_BF16 || type == MGNN_F16 ? 2 : 0; }

// Threads per row (a power of two) and vectors per thread of a row of C elements.  Rows that fit 64 vectors: one per lane,
// the fewest lanes.  Longer ones: two per thread, which beat one (half the waves meet at the barrier) and four (registers)
// in the backward pass and lose nothing in the forward one: bf16 4096 columns x 16384 rows, 256 x 2 / 512 x 1 / 128 x 4:
// forward 50.3 / 50.4 / 49.0 us, backward 83 / 85 / 94; fp32 1024 columns, 128 x 2 / 256 x 1 / 64 x 4: backward 41.4 / 44.8 / 41.6.
struct RowSplit {
  int tpr, nv;
};
RowSplit row_split(int C, int type) {
  const int V = 16 / elem_bytes(type), vecs = (C + V - 1) / V;
  const int nv = vecs <= kWave ? 1 : vecs <= 2048 ? 2 : 4;
  int tpr = 1;
  while (tpr * nv < vecs) tpr <<= 1;
  return {tpr, nv};
}
int block_of(const RowSplit& s) { return s.tpr > 256 ? s.tpr : 256; }

// Workgroups per group for `want` workgroup-steps of rows each, at most about `most` workgroups in all groups: every one
// takes the same number of steps, the last one apart.
int64_t even_blocks(int64_t want, int64_t groups, int64_t most) {
  const int64_t cap = std::max<int64_t>(1, most / groups), steps = (want + cap - 1) / cap;
  return steps ? (want + steps - 1) / steps : 1;
}

// How many workgroups carry a stream of rows is a matter of bytes in flight: half-empty vectors (a row of 35 floats takes 9
// of 16 lanes) want twice as many.  `base` full ones, at most what the registers let stand on the card at once.
int64_t by_bytes(const RowSplit& s, int C, int type, int64_t base, int64_t resident) {
  const int64_t lanes = (int64_t)s.tpr * s.nv * (16 / elem_bytes(type));
  return std::min(resident, base * lanes / C);
}

// Forward: workgroups stay, keep their weight rows in registers and load the next row under the sums of this one.  Of 256
// threads: four per CU for fp32 (3 x 409600 rows of 128, 512 / 1024 / 2048 workgroups: 294 / 229 / 249 us; 958698 of 35, 1024 /
// 2048: 65 / 54), six for 16-bit rows within a wave, which have twice the arithmetic per byte (3 x 409600 of 64, 1024 / 1536 /
// 2048: 73 / 61 / 62 us; 958698 of 35: 39 / 33 / 40).  Work that does not fill the card once over goes out one step each.
int64_t forward_blocks(int64_t groups, int64_t rows, int C, int type) {
  const RowSplit s = row_split(C, type);
  const int64_t block = block_of(s), slots = block / s.tpr, want = (rows + slots - 1) / slots;
  const int64_t most = block > 256 ? 262144 / block : type == MGNN_F32 ? by_bytes(s, C, type, 1024, 2048)
                                                    : s.nv == 1        ? 1536 : by_bytes(s, C, type, 1024, 1280);
  return want * groups <= 2048 * 256 / block ? want : even_blocks(want, groups, most);
}

// Backward: each workgroup leaves one row of shares of dweight and dbias to be added up, so there are fewer, the more so the longer
// the rows.  fp32 3 x 409600 x 128, 512 / 768 / 1536 workgroups: 355 / 350 / 383 us; bf16 3 x 409600 x 64: 97 / 92 / 96, and 704 / 768
// 93.4 / 93.2, 409600 x 512 235 / 240; 16384 x 4096, 512 / 768 / 1536: 83 / 93 / 107; 8192 columns (512 threads), 256 / 512: 56 / 67;
// half-empty fp32 958698 x 35, 512 / 1024 / 1280: 129 / 86 / 81.
// Each takes at least four steps, even where that leaves CUs idle: fewer shares are worth more.  With and without that minimum,
// the join included: 509 x 16381 fp32 128 / 255 workgroups 43.4 / 47.8 us, 512 x 4096 bf16 128 / 512: 14.6 / 24.5, 256 x 8192 bf16
// 64 / 256: 19.2 / 22.7, 2000 x 512 bf16 125 / 500: 8.4 / 11.6, 1024 x 1024 fp32 128 / 512: 9.8 / 10.2.  A pass for dx alone, which leaves
// no shares, takes the same workgroups, and there the minimum costs: 27.9 / 24.6, 5.9 / 3.7, 6.9 / 3.7, 4.1 / 2.8, 4.9 / 3.2.
int64_t backward_blocks(int64_t groups, int64_t rows, int C, int type) {
  const RowSplit s = row_split(C, type);
  const int64_t block = block_of(s), slots = block / s.tpr, want = (rows + slots - 1) / slots;
  const bool half = type != MGNN_F32;      // twice the elements and registers per vector
  const int64_t resident = s.nv == 1 ? half ? 1024 : 2048 : half ? 768 : 1280;
  const int64_t most = block > 256 ? 256 : by_bytes(s, C, type, half && s.nv == 1 ? 704 : 512, resident);
  return std::max<int64_t>(1, std::min((want + 3) / 4, even_blocks(want, groups, most)));
}

int check_ln(int64_t ld, int64_t groups, int64_t rows, int C, int type, int wtype) {
  if (!elem_bytes(type) || (wtype != type && wtype != MGNN_F32)) return MGNN_ERR_TYPE;
  if (C < 1 || C > MGNN_LN_MAX_C || ld < C || groups < 0 || groups > MGNN_MAX_GROUPS || rows < 0) return MGNN_ERR_SHAPE;
  // every offset below is computed in 64 bits of elements
  if (groups > 0 && rows > INT64_MAX / 8 / groups / ld) return MGNN_ERR_SHAPE;
  return MGNN_OK;
}

// calls f.template operator()<TPR, NV, FULL>() for the split of rows of C elements
template <typename T, typename F>
int with_split(const RowSplit& s, int C, F f) {
  const bool full = C == s.tpr * s.nv * Pack<T>::V;
  switch (s.tpr * 8 + s.nv) {
    case 1 * 8 + 1: return full ? f.template operator()<1, 1, true>() : f.template operator()<1, 1, false>();
    case 2 * 8 + 1: return full ? f.template operator()<2, 1, true>() : f.template operator()<2, 1, false>();
    case 4 * 8 + 1: return full ? f.template operator()<4, 1, true>() : f.template operator()<4, 1, false>();
    case 8 * 8 + 1: return full ? f.template operator()<8, 1, true>() : f.template operator()<8, 1, false>();
    case 16 * 8 + 1: return full ? f.template operator()<16, 1, true>() : f.template operator()<16, 1, false>();
    case 32 * 8 + 1: return full ? f.template operator()<32, 1, true>() : f.template operator()<32, 1, false>();
    case 64 * 8 + 1: return full ? f.template operator()<64, 1, true>() : f.template operator()<64, 1, false>();
    case 64 * 8 + 2: return full ? f.template operator()<64, 2, true>() : f.template operator()<64, 2, false>();
    case 128 * 8 + 2: return full ? f.template operator()<128, 2, true>() : f.template operator()<128, 2, false>();
    case 256 * 8 + 2: return full ? f.template operator()<256, 2, true>() : f.template operator()<256, 2, false>();
    case 512 * 8 + 2: return full ? f.template operator()<512, 2, true>() : f.template operator()<512, 2, false>();
    case 1024 * 8 + 2: return full ? f.template operator()<1024, 2, true>() : f.template operator()<1024, 2, false>();
    case 1024 * 8 + 4:      // fp32 rows of more than 8192
      if constexpr (std::is_same_v<T, float>) return full ? f.template operator()<1024, 4, true>() : f.template operator()<1024, 4, false>();
  }
  return MGNN_ERR_SHAPE;      // row_split gives no other
}

template <typename T>
struct LnFwd {
  const T* x; int64_t ld; const void *weight, *bias; int wtype; T* y; float2* stats; int64_t groups, rows, blocks; int C; float eps;
  hipStream_t stream;
  template <int TPR, int NV, bool FULL>
  int operator()() {
    return launch(ln_fwd_kernel<T, TPR, NV, FULL>, dim3((unsigned)blocks, (unsigned)groups), Shape<TPR>::BLOCK, stream, x, ld, weight, bias,
                  wtype, y, stats, rows, C, eps);
  }
};

template <typename T>
struct LnBwd {
  const T* x; int64_t ld; const T* dy; const void* weight; int wtype; const float2* stats; T* dx; float* partial;
  void *dweight, *dbias; int64_t groups, rows, blocks; int C; hipStream_t stream;
  template <int TPR, int NV, bool FULL>
  int operator()() {
    return launch(ln_bwd_kernel<T, TPR, NV, FULL>, dim3((unsigned)blocks, (unsigned)groups), Shape<TPR>::BLOCK, stream, x, ld, dy, weight, wtype,
                  stats, dx, partial, dweight, dbias, rows, C);
  }
};

// ---- the global gradient norm ----
// The list travels in the kernel arguments (so a captured launch holds it), up to kTensors tensors per launch; longer
// lists take several launches, each with its own rows of partial sums.  A tensor is cut into chunks of 16 KB per group.
constexpr int kTensors = 112;
constexpr int64_t kMaxChunks = 1 << 30;      // of a table: a workgroup's next chunk stays an int
constexpr int kBlock = 256;
constexpr int kChunkBytes = kBlock * 16 * 4;
struct GradTable {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t n_type[kTensors];      // elements per group << 2 | type (a scalar load takes words)
  int32_t end[kTensors];         // chunks of a group up to and with this tensor
  int32_t count;
  __host__ __device__ int64_t n(int i) const { return n_type[i] >> 2; }
  __host__ __device__ int type(int i) const { return (int)(n_type[i] & 3); }
};
static_assert(sizeof(GradTable) <= 3800, "kernel arguments hold 4 KB");

template <int BLOCK>
__device__ __forceinline__ double block_sum(double v, double* lds) {      // in every thread of the first wave
  v = lanes_sum<kWave>(v);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  return threadIdx.x < kWave ? lanes_sum<BLOCK / kWave>(lds[threadIdx.x % (BLOCK / kWave)]) : 0.0;
}

// The tensor of a chunk: the number of tensors that end at or before it, counted by a wave's lanes in one go
struct Finder {
  int low, high;      // this lane's two ends
  __device__ __forceinline__ explicit Finder(const GradTable& t) {
    const int lane = threadIdx.x % kWave;
    low = lane < t.count ? t.end[lane] : INT32_MAX;
    high = lane + kWave < t.count ? t.end[lane + kWave] : INT32_MAX;
  }
  __device__ __forceinline__ int operator()(int chunk) const {
    return __popcll(__ballot(low <= chunk)) + __popcll(__ballot(high <= chunk));
  }
};
static_assert(kTensors <= 2 * kWave);

// Squares are exact in fp64, and no fp32 value overflows there; the conversions hide under the loads: 2.1 GB of fp32 in
// 335 us (6.4 TB/s), which is all that bounds it.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n) {      // n elements from p on, one chunk at most
  constexpr int V = Pack<T>::V;
  double acc = 0.0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = (u * kBlock + threadIdx.x) * V;
    if (at < n) {
      const typename Pack<T>::Vec v = load_part(p, at, (int)min(n, (int64_t)kChunkBytes));
#pragma unroll
      for (int k = 0; k < V; ++k) acc = __builtin_fma((double)(float)v[k], (double)(float)v[k], acc);
    }
  }
  return acc;
}

__global__ __launch_bounds__(kBlock, 8) void grad_squares_kernel(GradTable t, double* partial, int row, int rows_of_group) {
  __shared__ double lds[kBlock / kWave];
  const int64_t g = blockIdx.y;
  const Finder find(t);
  const int chunks = t.end[t.count - 1];
  double acc = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = __builtin_amdgcn_readfirstlane(find(c));
    const int64_t at = (int64_t)(c - (i ? t.end[i - 1] : 0)) * (kChunkBytes / (t.type(i) == MGNN_F32 ? 4 : 2));
    const int64_t off = g * t.n(i) + at, n = t.n(i) - at;
    if (t.type(i) == MGNN_F32) acc += chunk_squares(static_cast<const float*>(t.src[i]) + off, n);
    else if (t.type(i) == MGNN_BF16) acc += chunk_squares(static_cast<const __bf16*>(t.src[i]) + off, n);
    else acc += chunk_squares(static_cast<const _Float16*>(t.src[i]) + off, n);
  }
  acc = block_sum<kBlock>(acc, lds);
  if (threadIdx.x == 0) partial[g * rows_of_group + row + blockIdx.x] = acc;
}

// Group g's norm from the partial sums, in every thread of the first wave
__device__ __forceinline__ double group_norm(const double* partial, int64_t g, int rows_of_group, double* lds) {
  double acc = 0.0;
  for (int k = threadIdx.x; k < rows_of_group; k += kBlock) acc += partial[g * rows_of_group + k];
  const double sum = block_sum<kBlock>(acc, lds);
  return threadIdx.x < kWave ? sqrt(sum) : 0.0;
}

// min(1, max_norm / (norm + 1e-6)), where NaN stays NaN; norm is the first wave's, which alone does the fp64 division
__device__ __forceinline__ float clip_factor(double norm, double max_norm, float* lds) {
  if (threadIdx.x < kWave) {
    const float f = (float)(max_norm / (norm + 1e-6));
    if (threadIdx.x == 0) *lds = f > 1.f ? 1.f : f;
  }
  __syncthreads();
  return *lds;
}

// Lists of many launches leave more partial sums than every workgroup should add up by itself: each group's become one
constexpr int kMostRows = 16384;      // 128 KB from the caches, 2 us of a scaling launch
__global__ __launch_bounds__(1024) void grad_sum_kernel(const double* partial, int rows_of_group, double* sums) {
  __shared__ double lds[1024 / kWave];
  double acc = 0.0;
#pragma unroll 8
  for (int k = threadIdx.x; k < rows_of_group; k += 1024) acc += partial[(int64_t)blockIdx.x * rows_of_group + k];
  acc = block_sum<1024>(acc, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = acc;
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double* partial, int rows_of_group, float* norms) {
  __shared__ double lds[kBlock / kWave];
  const double norm = group_norm(partial, blockIdx.x, rows_of_group, lds);
  if (threadIdx.x == 0) norms[blockIdx.x] = (float)norm;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* q, int64_t n, float f, bool past_caches) {
  constexpr int V = Pack<T>::V;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = (u * kBlock + threadIdx.x) * V, end = (int)min(n, (int64_t)kChunkBytes);
    if (at < n) {
      typename Pack<T>::Vec v = load_part(p, at, end);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (T)((float)v[k] * f);
      if (past_caches && at + V <= end) Pack<T>::store_past_caches(q + at, v);
      else store_part(q, at, end, v);
    }
  }
}

// Every workgroup adds up the partial sums itself (16 KB a table of the list, 128 KB at most, from the caches) rather than waiting for a launch between.
// 2.1 GB of fp32 read and written in 767 us (5.6 TB/s), bound by HBM.
__global__ __launch_bounds__(kBlock, 8) void grad_scale_kernel(GradTable t, const double* partial, int rows_of_group, double max_norm,
                                                            float* norms, bool past_caches) {
  __shared__ double lds[kBlock / kWave];
  __shared__ float factor;
  const int64_t g = blockIdx.y;
  const Finder find(t);
  const double norm = group_norm(partial, g, rows_of_group, lds);
  const float f = clip_factor(norm, max_norm, &factor);
  if (norms && blockIdx.x == 0 && threadIdx.x == 0) norms[g] = (float)norm;
  // from the end on, which was read last: what the caches still hold of it is not read from memory again
  for (int c = t.end[t.count - 1] - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const int i = __builtin_amdgcn_readfirstlane(find(c));
    if (f == 1.f && t.src[i] == t.dst[i]) continue;      // a factor of 1 in place: nothing changes
    const int64_t at = (int64_t)(c - (i ? t.end[i - 1] : 0)) * (kChunkBytes / (t.type(i) == MGNN_F32 ? 4 : 2));
    const int64_t off = g * t.n(i) + at, n = t.n(i) - at;
    if (t.type(i) == MGNN_F32) chunk_scale(static_cast<const float*>(t.src[i]) + off, static_cast<float*>(t.dst[i]) + off, n, f, past_caches);
    else if (t.type(i) == MGNN_BF16)
      chunk_scale(static_cast<const __bf16*>(t.src[i]) + off, static_cast<__bf16*>(t.dst[i]) + off, n, f, past_caches);
    else chunk_scale(static_cast<const _Float16*>(t.src[i]) + off, static_cast<_Float16*>(t.dst[i]) + off, n, f, past_caches);
  }
}

// Norms and clipping of gradients that one workgroup per group holds in its registers, SLOTS vectors of 16 bytes a thread:
// one launch, and every element is read once.  The list's vectors are numbered through (t.end: vectors up to and with a
// tensor); a tensor's last vector ends at its end and overlaps the one before, which counts the common elements; both
// write the same values.  37544 fp32 in 13 tensors take 8.1 us, all on one CU: the table and each vector's tensor 0.9, loading
// 1.5, fp64 squares 1.9, the norm 0.6, scaling and storing 2.7.
// The limit is what the registers hold, and not where two launches over many CUs begin to win.  Called from the host, for which the
// second launch is the dearer one, that is near it, written in place, one launch and two: 37544 fp32 8.5 and 11 us a call, 50544 in 16
// tensors 10.7 and 11.8, 64800 12.7 and 11.1.  In a replayed graph it is at about 27000: 15996 4.8 and 6.2 us, 30000 6.8 and 6.6, 50544
// 10.6 and 7.1, 129996 bf16 18.4 and 7.1.  FLOATS: all of the
// list is fp32.  max_norm < 0: the norms alone.
constexpr int kSmallBlock = 1024;
constexpr int kSmallSlots = 16;      // at most: 64 of the 128 registers a thread of 1024 has
struct SmallTable : GradTable {
  uint8_t first[kSmallSlots * kSmallBlock / kWave];      // the tensor of every wave's first vector; count past the last one
};
static_assert(sizeof(SmallTable) <= 3800 && kTensors < 256 && kTensors < kSmallBlock);
template <typename T>
__device__ __forceinline__ double raw_squares(uint4 raw, int skip, int n) {      // elements skip .. n-1 of the vector
  constexpr int V = Pack<T>::V;
  typename Pack<T>::Vec v = __builtin_bit_cast(typename Pack<T>::Vec, raw);
  if (skip > 0 || n < V) {      // a tensor's last vector
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k >= skip && k < n ? v[k] : (T)0.f;
  }
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < V; ++k) acc = __builtin_fma((double)(float)v[k], (double)(float)v[k], acc);
  return acc;
}
template <typename T>
__device__ __forceinline__ uint4 raw_load(const T* p, int n) {
  constexpr int V = Pack<T>::V;
  typename Pack<T>::Vec v = {};
  if (n >= V) {
    v = Pack<T>::load(p);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) v[k] = p[k];
  }
  return __builtin_bit_cast(uint4, v);
}
template <typename T>
__device__ __forceinline__ void raw_scale(T* p, uint4 raw, int n, float f) {
  constexpr int V = Pack<T>::V;
  typename Pack<T>::Vec v = __builtin_bit_cast(typename Pack<T>::Vec, raw);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = (T)((float)v[k] * f);
  if (n >= V) {
    Pack<T>::store(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) p[k] = v[k];
  }
}

template <int SLOTS, bool FLOATS>
__global__ __launch_bounds__(kSmallBlock) void grad_small_kernel(SmallTable t, double max_norm, float* norms) {
  __shared__ double lds[kSmallBlock / kWave];
  __shared__ int32_t end[kTensors + 1];
  __shared__ const char* from[kTensors];
  __shared__ char* to[kTensors];
  __shared__ int32_t len[kTensors];
  __shared__ uint8_t type[kTensors];
  __shared__ float factor;
  const auto type_of = [&](int i) { return FLOATS ? MGNN_F32 : (int)type[i]; };
  const int64_t g = blockIdx.x;
  int which[SLOTS], stop[SLOTS];      // each vector's tensor, and where that ends
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) which[k] = t.first[k * (kSmallBlock / kWave) + threadIdx.x / kWave];
  if (threadIdx.x <= t.count) {
    const int i = threadIdx.x;
    end[i] = i < t.count ? t.end[i] : INT32_MAX;
    if (i < t.count) {
      const int64_t off = g * t.n(i) * (t.type(i) == MGNN_F32 ? 4 : 2);
      from[i] = static_cast<const char*>(t.src[i]) + off;
      to[i] = t.dst[i] ? static_cast<char*>(t.dst[i]) + off : nullptr;
      len[i] = (int32_t)t.n(i);
      type[i] = t.type(i);
    }
  }
  __syncthreads();
  const int vectors = end[t.count - 1];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) stop[k] = end[which[k]];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k)
    while (k * kSmallBlock + (int)threadIdx.x >= stop[k]) stop[k] = end[++which[k]];      // end[count], at the latest, is past them all
  uint4 raw[SLOTS];
  int place[SLOTS];      // tensor << 20 | first element; -1: no vector
  static_assert(kSmallSlots * kSmallBlock * 8 <= 1 << 20 && kTensors < 1 << 11);
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    const int v = k * kSmallBlock + threadIdx.x, i = which[k];
    place[k] = -1;
    if (v < vectors) {
      const int V = type_of(i) == MGNN_F32 ? 4 : 8;
      const int at = max(min((v - (i ? end[i - 1] : 0)) * V, len[i] - V), 0);
      place[k] = i << 20 | at;
      raw[k] = type_of(i) == MGNN_F32 ? raw_load(reinterpret_cast<const float*>(from[i]) + at, len[i])
                                   : raw_load(reinterpret_cast<const _Float16*>(from[i]) + at, len[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    if (place[k] < 0) continue;
    const int i = place[k] >> 20, ty = type_of(i), V = ty == MGNN_F32 ? 4 : 8;
    const int skip = (k * kSmallBlock + (int)threadIdx.x - (i ? end[i - 1] : 0)) * V - (place[k] & 0xfffff);
    acc += ty == MGNN_F32 ? raw_squares<float>(raw[k], skip, len[i])
                          : ty == MGNN_BF16 ? raw_squares<__bf16>(raw[k], skip, len[i]) : raw_squares<_Float16>(raw[k], skip, len[i]);
  }
  const double sum = block_sum<kSmallBlock>(acc, lds);
  const double norm = threadIdx.x < kWave ? sqrt(sum) : 0.0;
  if (threadIdx.x == 0) norms[g] = (float)norm;
  if (max_norm < 0.0) return;
  const float f = clip_factor(norm, max_norm, &factor);
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    if (place[k] < 0) continue;
    const int i = place[k] >> 20, at = place[k] & 0xfffff, ty = type_of(i);
    if (f == 1.f && from[i] == to[i]) continue;      // a factor of 1 in place: nothing changes
    if (ty == MGNN_F32) raw_scale(reinterpret_cast<float*>(to[i]) + at, raw[k], len[i], f);
    else if (ty == MGNN_BF16) raw_scale(reinterpret_cast<__bf16*>(to[i]) + at, raw[k], len[i], f);
    else raw_scale(reinterpret_cast<_Float16*>(to[i]) + at, raw[k], len[i], f);
  }
}

// no gradients at all: norms of 0
__global__ void zero_norms_kernel(float* norms, int groups) {
  for (int g = threadIdx.x; g < groups; g += blockDim.x) norms[g] = 0.f;
}

// The launches of a list: tables of at most kTensors non-empty tensors, and each one's workgroups per group.
struct GradPlan {
  std::vector<GradTable> tables;
  std::vector<int> blocks;
  int rows = 0;      // partial sums per group; 0 with a table: one workgroup per group does it all
  int slots = 0;     // then its vectors per thread
  int64_t workspace(int64_t groups) const { return (rows + (rows > kMostRows)) * groups * (int64_t)sizeof(double); }
};

// chunks a tensor is cut into; -1: not a tensor that the list may hold
int64_t chunks_of(int64_t n, int type) {
  const int bytes = elem_bytes(type);
  if (!bytes || n < 0) return -1;
  const int64_t per = kChunkBytes / bytes;
  return n / per + (n % per != 0);
}

int grad_plan(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count, int64_t groups,
              GradPlan& plan) {
  if (groups < 1 || groups > MGNN_MAX_GROUPS) return MGNN_ERR_SHAPE;
  if (count < 0 || (count > 0 && (!n || !type))) return MGNN_ERR_VALUE;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!elem_bytes(type[i])) return MGNN_ERR_TYPE;
    if (n[i] < 0 || n[i] > INT64_MAX / 8 / groups) return MGNN_ERR_SHAPE;
    if (n[i] == 0) continue;
    if (src && (!src[i] || (dst && !dst[i]))) return MGNN_ERR_VALUE;
    const int64_t c = chunks_of(n[i], type[i]);
    if (plan.tables.empty() || plan.tables.back().count == kTensors || chunks + c > kMaxChunks) {
      if (c > kMaxChunks) return MGNN_ERR_SHAPE;
      plan.tables.emplace_back();
      plan.tables.back().count = 0;
      chunks = 0;
    }
    GradTable& t = plan.tables.back();
    chunks += c;
    t.src[t.count] = src ? src[i] : nullptr;
    t.dst[t.count] = dst ? dst[i] : nullptr;
    t.n_type[t.count] = n[i] << 2 | type[i];
    t.end[t.count++] = (int32_t)chunks;
  }
  if (plan.tables.size() == 1) {
    GradTable& t = plan.tables[0];
    int64_t vectors = 0;
    for (int i = 0; i < t.count; ++i) {
      const int V = t.type(i) == MGNN_F32 ? 4 : 8;
      vectors += t.n(i) / V + (t.n(i) % V != 0);
      if (vectors > kSmallSlots * kSmallBlock) break;
    }
    if (vectors <= kSmallSlots * kSmallBlock) {
      for (int i = 0, v = 0; i < t.count; ++i) {
        const int V = t.type(i) == MGNN_F32 ? 4 : 8;
        t.end[i] = v += (int)((t.n(i) + V - 1) / V);
      }
      plan.slots = (int)((vectors + 4 * kSmallBlock - 1) / (4 * kSmallBlock)) * 4;
      return MGNN_OK;
    }
  }
  for (const GradTable& t : plan.tables) {
    // as many workgroups as stand on the card at once, eight per CU, so that none starts late (2.1 GB of fp32, at 80 registers
    // and 1536 / 2048 workgroups: 1131 / 1277 us, at 64 registers: 1130 / 1113)
    const int64_t cap = std::max<int64_t>(1, 2048 / groups);
    plan.blocks.push_back((int)std::min<int64_t>(t.end[t.count - 1], cap));
    plan.rows += plan.blocks.back();
  }
  return MGNN_OK;
}

// whether memory that is written (every dst) overlaps anything else of the list
bool overlaps(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count, int64_t groups) {
  struct Range {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Range> r;
  r.reserve(2 * count);
  for (int64_t i = 0; i < count; ++i) {
    if (!n[i]) continue;
    const uintptr_t bytes = (uintptr_t)n[i] * groups * elem_bytes(type[i]);
    const uintptr_t d = (uintptr_t)dst[i], s = (uintptr_t)src[i];
    r.push_back({d, d + bytes, true});
    if (s != d) r.push_back({s, s + bytes, false});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  uintptr_t any = 0, written = 0;      // furthest end seen
  for (const Range& a : r) {
    if (a.from < written || (a.written && a.from < any)) return true;
    any = std::max(any, a.to);
    if (a.written) written = std::max(written, a.to);
  }
  return false;
}

int clip(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count, int64_t groups,
         double max_norm, float* norms, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  GradPlan plan;
  if (int rc = grad_plan(src, dst, n, type, count, groups, plan)) return rc;
  if (!norms || (count > 0 && (!src || (max_norm >= 0 && !dst)))) return MGNN_ERR_VALUE;
  if (plan.tables.empty()) {
    return launch(zero_norms_kernel, dim3(1), 256, stream, norms, (int)groups);
  }
  if (dst && overlaps(src, dst, n, type, count, groups)) return MGNN_ERR_OVERLAP;
  if (plan.slots) {
    SmallTable t;
    static_cast<GradTable&>(t) = plan.tables[0];
    for (int wave = 0, i = 0; wave < plan.slots * kSmallBlock / kWave; ++wave) {
      while (i < t.count && t.end[i] <= wave * kWave) ++i;
      t.first[wave] = (uint8_t)i;
    }
    const bool floats = std::all_of(t.n_type, t.n_type + t.count, [](int64_t nt) { return (nt & 3) == MGNN_F32; });
    const auto pick = [&](auto all) {
      constexpr bool F = decltype(all)::value;
      return plan.slots == 4 ? grad_small_kernel<4, F> : plan.slots == 8 ? grad_small_kernel<8, F>
             : plan.slots == 12 ? grad_small_kernel<12, F> : grad_small_kernel<kSmallSlots, F>;
    };
    const auto kernel = floats ? pick(std::true_type()) : pick(std::false_type());
    return launch(kernel, dim3((unsigned)groups), kSmallBlock, stream, t, dst ? max_norm : -1.0, norms);
  }
  if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < plan.workspace(groups)) return MGNN_ERR_WORKSPACE;
  double* partial = static_cast<double*>(workspace);
  int row = 0;
  for (size_t k = 0; k < plan.tables.size(); ++k) {
    if (int rc = launch(grad_squares_kernel, dim3(plan.blocks[k], (unsigned)groups), kBlock, stream, plan.tables[k], partial, row, plan.rows))
      return rc;
    row += plan.blocks[k];
  }
  int rows = plan.rows;
  if (rows > kMostRows) {
    double* sums = partial + rows * groups;
    if (int rc = launch(grad_sum_kernel, dim3((unsigned)groups), 1024, stream, partial, rows, sums)) return rc;
    partial = sums;
    rows = 1;
  }
  if (!dst) return launch(grad_norm_kernel, dim3((unsigned)groups), kBlock, stream, partial, rows, norms);
  // Results of more than the 256 MB of the memory-side cache go past it: they would push out the gradients that are still
  // to be read, and the next reader would not find them there either (256 MB of bf16 apart: 153 -> 131 us, with a copy of
  // the results behind it 350 -> 348).
  int64_t bytes = 0;
  for (int64_t i = 0; i < count; ++i) bytes += n[i] * groups * elem_bytes(type[i]);
  const bool past_caches = bytes >= (int64_t)256 << 20;
  for (size_t k = plan.tables.size(); k-- > 0;)
    if (int rc = launch(grad_scale_kernel, dim3(plan.blocks[k], (unsigned)groups), kBlock, stream, plan.tables[k], partial, rows, max_norm,
                        k == 0 ? norms : nullptr, past_caches))
      return rc;
  return MGNN_OK;
}

}  // namespace

extern "C" {

int mgnn_layer_norm(const void* x, int64_t ld, const void* weight, const void* bias, void* y, float* stats, int64_t groups,
                    int64_t rows, int C, double eps, int type, int wtype, void* stream) {
  if (int rc = check_ln(ld, groups, rows, C, type, wtype)) return rc;
  if (!(eps >= 0.0)) return MGNN_ERR_VALUE;
  if (groups == 0 || rows == 0) return MGNN_OK;
  if (!x || !y) return MGNN_ERR_VALUE;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    return with_split<T>(row_split(C, type), C, LnFwd<T>{static_cast<const T*>(x), ld, weight, bias, wtype, static_cast<T*>(y),
                                                         reinterpret_cast<float2*>(stats), groups, rows, forward_blocks(groups, rows, C, type), C,
                                                         (float)eps, (hipStream_t)stream});
  };
  return type == MGNN_F32 ? go(0.f) : type == MGNN_BF16 ? go((__bf16)0.f) : go((_Float16)0.f);
}

int64_t mgnn_layer_norm_workspace(int64_t groups, int64_t rows, int C, int type) {
  if (check_ln(C, groups, rows, C, type, type)) return -1;
  if (groups == 0) return 0;
  const int64_t blocks = backward_blocks(groups, rows, C, type);
  return blocks == 1 ? 0 : groups * blocks * 2 * C * (int64_t)sizeof(float);
}

int mgnn_layer_norm_backward(const void* x, int64_t ld, const void* dy, const void* weight, const float* stats, void* dx,
                             void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, int64_t groups, int64_t rows,
                             int C, int type, int wtype, void* stream) {
  if (int rc = check_ln(ld, groups, rows, C, type, wtype)) return rc;
  if (groups == 0 || (!dx && !dweight && !dbias)) return MGNN_OK;
  if (rows == 0 && !dweight && !dbias) return MGNN_OK;
  if (rows > 0 && (!x || !dy || !stats)) return MGNN_ERR_VALUE;
  const int64_t blocks = backward_blocks(groups, rows, C, type);
  const bool join = blocks > 1 && (dweight || dbias);
  if (join && (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < mgnn_layer_norm_workspace(groups, rows, C, type)))
    return MGNN_ERR_WORKSPACE;
  float* partial = join ? static_cast<float*>(workspace) : nullptr;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    return with_split<T>(row_split(C, type), C, LnBwd<T>{static_cast<const T*>(x), ld, static_cast<const T*>(dy), weight, wtype,
                                                         reinterpret_cast<const float2*>(stats), static_cast<T*>(dx), partial, dweight, dbias,
                                                         groups, rows, blocks, C, (hipStream_t)stream});
  };
  const int rc = type == MGNN_F32 ? go(0.f) : type == MGNN_BF16 ? go((__bf16)0.f) : go((_Float16)0.f);
  if (rc || !join) return rc;
  return launch(ln_join_kernel, dim3((unsigned)((2 * (int64_t)C + kJoinCols - 1) / kJoinCols), (unsigned)groups), kJoinCols * kJoinSlices,
                (hipStream_t)stream, partial, (int)blocks, C, dweight, dbias, wtype);
}

int64_t mgnn_grad_norm_workspace(const int64_t* n, const int32_t* type, int64_t count, int64_t groups) try {
  GradPlan plan;
  if (grad_plan(nullptr, nullptr, n, type, count, groups, plan)) return -1;
  return plan.workspace(groups);
} catch (...) {
  return -1;
}

int mgnn_grad_norm(const void* const* src, const int64_t* n, const int32_t* type, int64_t count, int64_t groups, float* norms,
                   void* workspace, int64_t workspace_bytes, void* stream) try {
  return clip(src, nullptr, n, type, count, groups, -1.0, norms, workspace, workspace_bytes, (hipStream_t)stream);
} catch (...) {
  return MGNN_ERR_MEMORY;
}

int mgnn_clip_grads(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count,
                    int64_t groups, double max_norm, float* norms, void* workspace, int64_t workspace_bytes, void* stream) try {
  if (!(max_norm >= 0.0)) return MGNN_ERR_VALUE;
  return clip(src, dst, n, type, count, groups, max_norm, norms, workspace, workspace_bytes, (hipStream_t)stream);
} catch (...) {
  return MGNN_ERR_MEMORY;
}

}  // extern "C"
