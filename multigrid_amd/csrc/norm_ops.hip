// Layer norm with its gradients, and clipping by the global gradient norm (include/mgrid_norm.h): the normalisation of the
// PPO trainer's policies and of their gradients.  Both are bound by HBM traffic; every element is moved 16 bytes per lane.
// Rows and gradients may start at any element: gfx950 loads and stores 16 bytes at any address of an element's alignment,
// so a row of odd length takes the same path as an even one, with its last, shorter vector element by element.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
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

__device__ __forceinline__ float load_as_float(const void* p, int type, int64_t i) {
  if (type == MGNN_F32) return static_cast<const float*>(p)[i];
  if (type == MGNN_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}

__device__ __forceinline__ void store_from_float(void* p, int type, int64_t i, float v) {
  if (type == MGNN_F32) static_cast<float*>(p)[i] = v;
  else if (type == MGNN_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// sum over aligned groups of L lanes, in every lane of the group (all 64 lanes take part)
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v += __shfl_xor(v, s);
  return v;
}

// ---- layer norm ----
// TPR threads share a row, thread t holding the vectors t, t + TPR, ... (NV of them) in registers, so a row is read once;
// a workgroup works on SLOTS rows at a time.  Rows of up to 64 vectors belong to part of a wave or a whole one and need no
// barrier; longer ones to a whole workgroup.
template <int TPR>
struct Shape {
  static constexpr int BLOCK = TPR > 256 ? TPR : 256;
  static constexpr int SLOTS = BLOCK / TPR;
  static constexpr int WAVES = BLOCK / kWave;
  static constexpr int ROW_WAVES = TPR > kWave ? TPR / kWave : 1;
};

// Mean and sum of squared deviations of a row whose elements the TPR threads hold (those past C are not counted): two
// passes over the registers, so no digits cancel.  Rows over several waves: each wave's own mean and deviations, combined
// as M = sum M_w + n_w (m_w - m)^2, which takes one barrier instead of two.
template <int TPR, int NE, int V>
__device__ __forceinline__ void row_stats(const float (&v)[NE], int lane, int C, float2 (*red)[Shape<TPR>::WAVES], int parity,
                                          float& mean, float& m2) {
  constexpr int L = TPR < kWave ? TPR : kWave;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NE; ++k) s += v[k];
  s = lanes_sum<L>(s);
  int n = 0;      // this wave's elements of the row
#pragma unroll
  for (int i = 0; i < NE / V; ++i) {
    const int first = ((TPR <= kWave ? 0 : (lane & ~(kWave - 1))) + i * TPR) * V;
    n += min(max(C - first, 0), L * V);
  }
  mean = n > 0 ? s / (float)n : 0.f;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int col = (lane + (k / V) * TPR) * V + k % V;
    const float d = v[k] - mean;
    q += col < C ? d * d : 0.f;
  }
  m2 = lanes_sum<L>(q);
  if constexpr (TPR > kWave) {
    constexpr int W = Shape<TPR>::ROW_WAVES;
    const int wave = threadIdx.x / kWave, first = wave / W * W;
    if (threadIdx.x % kWave == 0) red[parity][wave] = make_float2(mean, m2);
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      int nw = 0;
#pragma unroll
      for (int i = 0; i < NE / V; ++i) nw += min(max(C - (w * kWave + i * TPR) * V, 0), kWave * V);
      total += red[parity][first + w].x * (float)nw;
    }
    mean = total / (float)C;
    m2 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      int nw = 0;
#pragma unroll
      for (int i = 0; i < NE / V; ++i) nw += min(max(C - (w * kWave + i * TPR) * V, 0), kWave * V);
      const float2 r = red[parity][first + w];
      const float d = r.x - mean;
      m2 += nw > 0 ? r.y + (float)nw * (d * d) : 0.f;
    }
  }
}

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(Shape<TPR>::BLOCK) void ln_fwd_kernel(const T* x, int64_t ld, const void* weight, const void* bias,
                                                                   int wtype, T* y, float2* stats, int64_t rows, int C, float eps) {
  constexpr int V = Pack<T>::V, NE = NV * V, SLOTS = Shape<TPR>::SLOTS;
  __shared__ float2 red[2][Shape<TPR>::WAVES];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t g = blockIdx.y;
  float w[NE], b[NE];
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int col = (lane + (k / V) * TPR) * V + k % V;
    w[k] = weight && col < C ? load_as_float(weight, wtype, g * C + col) : 1.f;
    b[k] = bias && col < C ? load_as_float(bias, wtype, g * C + col) : 0.f;
  }
  int parity = 0;
  for (int64_t base = (int64_t)blockIdx.x * SLOTS; base < rows; base += (int64_t)gridDim.x * SLOTS, parity ^= 1) {
    const int64_t row = g * rows + base + slot;
    const bool live = base + slot < rows;
    float v[NE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (lane + i * TPR) * V;
      typename Pack<T>::Vec p = {};
      if (live && col < C) p = load_part(x + row * ld, col, C);
#pragma unroll
      for (int k = 0; k < V; ++k) v[i * V + k] = (float)p[k];
    }
    float mean, m2;
    row_stats<TPR, NE, V>(v, lane, C, red, parity, mean, m2);
    const float rstd = 1.f / sqrtf(m2 / (float)C + eps);
    if (live) {
      if (stats && lane == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (lane + i * TPR) * V;
        typename Pack<T>::Vec p;
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] = (T)__builtin_fmaf((v[i * V + k] - mean) * rstd, w[i * V + k], b[i * V + k]);
        if (col < C) store_part(y + row * C, col, C, p);
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

// partial: [groups][blocks][2][C] floats (this workgroup's shares of dweight and dbias), or NULL with one block per group:
// then dweight / dbias are written here
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(Shape<TPR>::BLOCK) void ln_bwd_kernel(const T* x, int64_t ld, const T* dy, const void* weight,
                                                                   int wtype, const float2* stats, T* dx, float* partial,
                                                                   void* dweight, void* dbias, int64_t rows, int C) {
  constexpr int V = Pack<T>::V, NE = NV * V, SLOTS = Shape<TPR>::SLOTS, WAVES = Shape<TPR>::WAVES;
  constexpr int L = TPR < kWave ? TPR : kWave;
  constexpr int SETS = TPR < kWave ? WAVES : SLOTS, WIDTH = TPR < kWave ? kWave : TPR;
  __shared__ float2 red[2][WAVES];
  __shared__ float fold[SETS > 1 ? SETS / 2 * NE * WIDTH : 1];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t g = blockIdx.y;
  const float inv_c = 1.f / (float)C;
  float w[NE], aw[NE], ab[NE];
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int col = (lane + (k / V) * TPR) * V + k % V;
    w[k] = weight && col < C ? load_as_float(weight, wtype, g * C + col) : 1.f;
    aw[k] = ab[k] = 0.f;
  }
  int parity = 0;
  for (int64_t base = (int64_t)blockIdx.x * SLOTS; base < rows; base += (int64_t)gridDim.x * SLOTS, parity ^= 1) {
    const int64_t row = g * rows + base + slot;
    const bool live = base + slot < rows;
    const float2 st = live ? stats[row] : make_float2(0.f, 0.f);
    float h[NE], e[NE];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (lane + i * TPR) * V;
      typename Pack<T>::Vec px = {}, pd = {};
      if (live && col < C) {
        px = load_part(x + row * ld, col, C);
        pd = load_part(dy + row * C, col, C);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int j = i * V + k;
        const float d = (float)pd[k];
        h[j] = ((float)px[k] - st.x) * st.y;
        if (col + k >= C) h[j] = 0.f;      // past the end x is 0, which is no element of the row
        e[j] = d * w[j];
        s1 += e[j];
        s2 = __builtin_fmaf(e[j], h[j], s2);
        aw[j] = __builtin_fmaf(d, h[j], aw[j]);
        ab[j] += d;
      }
    }
    if (dx) {
      s1 = lanes_sum<L>(s1);
      s2 = lanes_sum<L>(s2);
      if constexpr (TPR > kWave) {
        constexpr int W = Shape<TPR>::ROW_WAVES;
        const int wave = threadIdx.x / kWave, first = wave / W * W;
        if (threadIdx.x % kWave == 0) red[parity][wave] = make_float2(s1, s2);
        __syncthreads();
        s1 = s2 = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float2 r = red[parity][first + k];
          s1 += r.x;
          s2 += r.y;
        }
      }
      s1 *= inv_c;
      s2 *= inv_c;
      if (live) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (lane + i * TPR) * V;
          typename Pack<T>::Vec p;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int j = i * V + k;
            p[k] = (T)(st.y * (e[j] - __builtin_fmaf(h[j], s2, s1)));
          }
          if (col < C) store_part(dx + row * C, col, C, p);
        }
      }
    }
  }
  if (!dweight && !dbias) return;
  slots_sum<TPR, NE>(aw, fold);
  slots_sum<TPR, NE>(ab, fold);
  if (threadIdx.x >= TPR) return;
  float* share = partial ? partial + (g * gridDim.x + blockIdx.x) * 2 * C : nullptr;
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int col = (lane + (k / V) * TPR) * V + k % V;
    if (col >= C) continue;
    if (share) {
      share[col] = aw[k];
      share[C + col] = ab[k];
    } else {
      if (dweight) store_from_float(dweight, wtype, g * C + col, aw[k]);
      if (dbias) store_from_float(dbias, wtype, g * C + col, ab[k]);
    }
  }
}

// dweight / dbias of group blockIdx.y from the workgroups' shares, in a fixed order: 32 columns x 32 slices of the blocks
constexpr int kJoinCols = 32, kJoinSlices = 32;
__global__ __launch_bounds__(kJoinCols* kJoinSlices) void ln_join_kernel(const float* partial, int blocks, int C, void* dweight,
                                                                         void* dbias, int wtype) {
  __shared__ float red[kJoinSlices][kJoinCols + 1];
  const int64_t g = blockIdx.y;
  const int c = threadIdx.x % kJoinCols, s = threadIdx.x / kJoinCols;
  const int64_t col = (int64_t)blockIdx.x * kJoinCols + c;
  float acc = 0.f;
  if (col < 2 * C) {
#pragma unroll 8
    for (int k = s; k < blocks; k += kJoinSlices) acc += partial[(g * blocks + k) * 2 * C + col];
  }
  red[s][c] = acc;
  __syncthreads();
  for (int half = kJoinSlices / 2; half >= 1; half >>= 1) {
    if (s < half) red[s][c] += red[s + half][c];
    __syncthreads();
  }
  if (s == 0 && col < 2 * C) {
    void* out = col < C ? dweight : dbias;
    if (out) store_from_float(out, wtype, g * C + (col < C ? col : col - C), red[0][c]);
  }
}

int launched() { return hipGetLastError() == hipSuccess ? MGNN_OK : MGNN_ERR_LAUNCH; }

int elem_bytes(int type) { return type == MGNN_F32 ? 4 : type == MGNN_BF16 || type == MGNN_F16 ? 2 : 0; }

// threads per row (a power of two) and vectors per thread of a row of C elements
struct RowSplit {
  int tpr, nv;
};
RowSplit row_split(int C, int type) {
  const int V = 16 / elem_bytes(type), vecs = (C + V - 1) / V;
  int tpr = 1;
  while (tpr < vecs && tpr < 1024) tpr <<= 1;
  int nv = 1;
  while (tpr * nv < vecs) nv <<= 1;
  return {tpr, nv};
}
int slots_of(const RowSplit& s) { return s.tpr > 256 ? 1 : 256 / s.tpr; }

// workgroups per group of the backward pass: each leaves one row of shares to be added up
int64_t backward_blocks(int64_t groups, int64_t rows, int C, int type) {
  const RowSplit s = row_split(C, type);
  const int64_t slots = slots_of(s), want = (rows + 4 * slots - 1) / (4 * slots);
  const int64_t cap = std::max<int64_t>(1, (s.tpr > 256 ? 262144 / s.tpr : 1024) / groups);
  return std::max<int64_t>(1, std::min(want, cap));
}

int check_ln(int64_t ld, int64_t groups, int64_t rows, int C, int type, int wtype) {
  if (!elem_bytes(type) || (wtype != type && wtype != MGNN_F32)) return MGNN_ERR_TYPE;
  if (C < 1 || C > MGNN_LN_MAX_C || ld < C || groups < 0 || groups > MGNN_MAX_GROUPS || rows < 0) return MGNN_ERR_SHAPE;
  // every offset below is computed in 64 bits of elements
  if (groups > 0 && rows > INT64_MAX / 8 / groups / ld) return MGNN_ERR_SHAPE;
  return MGNN_OK;
}

// calls f.template operator()<TPR, NV>() for the split
template <typename F>
void with_split(const RowSplit& s, F f) {
  switch (s.tpr * 8 + s.nv) {
    case 1 * 8 + 1: return f.template operator()<1, 1>();
    case 2 * 8 + 1: return f.template operator()<2, 1>();
    case 4 * 8 + 1: return f.template operator()<4, 1>();
    case 8 * 8 + 1: return f.template operator()<8, 1>();
    case 16 * 8 + 1: return f.template operator()<16, 1>();
    case 32 * 8 + 1: return f.template operator()<32, 1>();
    case 64 * 8 + 1: return f.template operator()<64, 1>();
    case 128 * 8 + 1: return f.template operator()<128, 1>();
    case 256 * 8 + 1: return f.template operator()<256, 1>();
    case 512 * 8 + 1: return f.template operator()<512, 1>();
    case 1024 * 8 + 1: return f.template operator()<1024, 1>();
    case 1024 * 8 + 2: return f.template operator()<1024, 2>();
    case 1024 * 8 + 4: return f.template operator()<1024, 4>();
  }
}

template <typename T>
struct LnFwd {
  const T* x; int64_t ld; const void *weight, *bias; int wtype; T* y; float2* stats; int64_t groups, rows; int C; float eps;
  hipStream_t stream;
  template <int TPR, int NV>
  void operator()() {
    const int64_t slots = Shape<TPR>::SLOTS, want = (rows + slots - 1) / slots;
    const int64_t cap = std::max<int64_t>(1, 16384 / groups);
    hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV>), dim3((unsigned)std::min(want, cap), (unsigned)groups), dim3(Shape<TPR>::BLOCK), 0,
                       stream, x, ld, weight, bias, wtype, y, stats, rows, C, eps);
  }
};

template <typename T>
struct LnBwd {
  const T* x; int64_t ld; const T* dy; const void* weight; int wtype; const float2* stats; T* dx; float* partial;
  void *dweight, *dbias; int64_t groups, rows, blocks; int C; hipStream_t stream;
  template <int TPR, int NV>
  void operator()() {
    hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV>), dim3((unsigned)blocks, (unsigned)groups), dim3(Shape<TPR>::BLOCK), 0, stream, x,
                       ld, dy, weight, wtype, stats, dx, partial, dweight, dbias, rows, C);
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
  int64_t n[kTensors];     // elements per group
  int32_t end[kTensors];   // chunks of a group up to and with this tensor
  uint8_t type[kTensors];
  int32_t count;
};
static_assert(sizeof(GradTable) <= 3800, "kernel arguments hold 4 KB");

__device__ __forceinline__ double block_sum(double v, double* lds) {      // in every thread
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) v += __shfl_xor(v, s);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int k = 0; k < kBlock / kWave; ++k) t += lds[k];
  __syncthreads();
  return t;
}

__device__ __forceinline__ int find_tensor(const GradTable& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (chunk < t.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

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

__global__ __launch_bounds__(kBlock) void grad_squares_kernel(GradTable t, double* partial, int row, int rows_of_group) {
  __shared__ double lds[kBlock / kWave];
  const int64_t g = blockIdx.y;
  const int chunks = t.end[t.count - 1];
  double acc = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find_tensor(t, c);
    const int64_t at = (int64_t)(c - (i ? t.end[i - 1] : 0)) * (kChunkBytes / (t.type[i] == MGNN_F32 ? 4 : 2));
    const int64_t off = g * t.n[i] + at, n = t.n[i] - at;
    if (t.type[i] == MGNN_F32) acc += chunk_squares(static_cast<const float*>(t.src[i]) + off, n);
    else if (t.type[i] == MGNN_BF16) acc += chunk_squares(static_cast<const __bf16*>(t.src[i]) + off, n);
    else acc += chunk_squares(static_cast<const _Float16*>(t.src[i]) + off, n);
  }
  acc = block_sum(acc, lds);
  if (threadIdx.x == 0) partial[g * rows_of_group + row + blockIdx.x] = acc;
}

__device__ __forceinline__ double group_norm(const double* partial, int64_t g, int rows_of_group, double* lds) {
  double acc = 0.0;
  for (int k = threadIdx.x; k < rows_of_group; k += kBlock) acc += partial[g * rows_of_group + k];
  return sqrt(block_sum(acc, lds));
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
  const float f = (float)(max_norm / (norm + 1e-6));
  return f > 1.f ? 1.f : f;
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double* partial, int rows_of_group, float* norms) {
  __shared__ double lds[kBlock / kWave];
  const double norm = group_norm(partial, blockIdx.x, rows_of_group, lds);
  if (threadIdx.x == 0) norms[blockIdx.x] = (float)norm;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* q, int64_t n, float f) {
  constexpr int V = Pack<T>::V;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = (u * kBlock + threadIdx.x) * V;
    if (at < n) {
      typename Pack<T>::Vec v = load_part(p, at, (int)min(n, (int64_t)kChunkBytes));
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (T)((float)v[k] * f);
      store_part(q, at, (int)min(n, (int64_t)kChunkBytes), v);
    }
  }
}

__global__ __launch_bounds__(kBlock) void grad_scale_kernel(GradTable t, const double* partial, int rows_of_group, double max_norm,
                                                            float* norms) {
  __shared__ double lds[kBlock / kWave];
  const int64_t g = blockIdx.y;
  const double norm = group_norm(partial, g, rows_of_group, lds);
  const float f = clip_factor(norm, max_norm);
  if (norms && blockIdx.x == 0 && threadIdx.x == 0) norms[g] = (float)norm;
  const int chunks = t.end[t.count - 1];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find_tensor(t, c);
    if (f == 1.f && t.src[i] == t.dst[i]) continue;      // a factor of 1 in place: nothing changes
    const int64_t at = (int64_t)(c - (i ? t.end[i - 1] : 0)) * (kChunkBytes / (t.type[i] == MGNN_F32 ? 4 : 2));
    const int64_t off = g * t.n[i] + at, n = t.n[i] - at;
    if (t.type[i] == MGNN_F32) chunk_scale(static_cast<const float*>(t.src[i]) + off, static_cast<float*>(t.dst[i]) + off, n, f);
    else if (t.type[i] == MGNN_BF16) chunk_scale(static_cast<const __bf16*>(t.src[i]) + off, static_cast<__bf16*>(t.dst[i]) + off, n, f);
    else chunk_scale(static_cast<const _Float16*>(t.src[i]) + off, static_cast<_Float16*>(t.dst[i]) + off, n, f);
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
  int rows = 0;      // partial sums per group
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
    t.n[t.count] = n[i];
    t.type[t.count] = (uint8_t)type[i];
    t.end[t.count++] = (int32_t)chunks;
  }
  for (const GradTable& t : plan.tables) {
    const int64_t cap = std::max<int64_t>(1, 1024 / groups);
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
    hipLaunchKernelGGL(zero_norms_kernel, dim3(1), dim3(256), 0, stream, norms, (int)groups);
    return launched();
  }
  if (dst && overlaps(src, dst, n, type, count, groups)) return MGNN_ERR_OVERLAP;
  if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < plan.rows * groups * (int64_t)sizeof(double)) return MGNN_ERR_WORKSPACE;
  double* partial = static_cast<double*>(workspace);
  int row = 0;
  for (size_t k = 0; k < plan.tables.size(); ++k) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(plan.blocks[k], (unsigned)groups), dim3(kBlock), 0, stream, plan.tables[k], partial, row,
                       plan.rows);
    row += plan.blocks[k];
  }
  if (!dst) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)groups), dim3(kBlock), 0, stream, partial, plan.rows, norms);
    return launched();
  }
  for (size_t k = 0; k < plan.tables.size(); ++k)
    hipLaunchKernelGGL(grad_scale_kernel, dim3(plan.blocks[k], (unsigned)groups), dim3(kBlock), 0, stream, plan.tables[k], partial,
                       plan.rows, max_norm, k == 0 ? norms : nullptr);
  return launched();
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
    with_split(row_split(C, type), LnFwd<T>{static_cast<const T*>(x), ld, weight, bias, wtype, static_cast<T*>(y), reinterpret_cast<float2*>(stats),
                                            groups, rows, C, (float)eps, (hipStream_t)stream});
  };
  if (type == MGNN_F32) go(0.f);
  else if (type == MGNN_BF16) go((__bf16)0.f);
  else go((_Float16)0.f);
  return launched();
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
    with_split(row_split(C, type), LnBwd<T>{static_cast<const T*>(x), ld, static_cast<const T*>(dy), weight, wtype,
                                            reinterpret_cast<const float2*>(stats), static_cast<T*>(dx), partial, dweight, dbias, groups,
                                            rows, blocks, C, (hipStream_t)stream});
  };
  if (type == MGNN_F32) go(0.f);
  else if (type == MGNN_BF16) go((__bf16)0.f);
  else go((_Float16)0.f);
  if (join)
    hipLaunchKernelGGL(ln_join_kernel, dim3((unsigned)((2 * (int64_t)C + kJoinCols - 1) / kJoinCols), (unsigned)groups),
                       dim3(kJoinCols * kJoinSlices), 0, (hipStream_t)stream, partial, (int)blocks, C, dweight, dbias, wtype);
  return launched();
}

int64_t mgnn_grad_norm_workspace(const int64_t* n, const int32_t* type, int64_t count, int64_t groups) try {
  GradPlan plan;
  if (grad_plan(nullptr, nullptr, n, type, count, groups, plan)) return -1;
  return plan.rows * groups * (int64_t)sizeof(double);
} catch (...) {
  return -1;
}

int mgnn_grad_norm(const void* const* src, const int64_t* n, const int32_t* type, int64_t count, int64_t groups, float* norms,
                   void* workspace, int64_t workspace_bytes, void* stream) try {
  return clip(src, nullptr, n, type, count, groups, -1.0, norms, workspace, workspace_bytes, (hipStream_t)stream);
} catch (...) {
  return MGNN_ERR_VALUE;
}

int mgnn_clip_grads(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count,
                    int64_t groups, double max_norm, float* norms, void* workspace, int64_t workspace_bytes, void* stream) try {
  if (!(max_norm >= 0.0)) return MGNN_ERR_VALUE;
  return clip(src, dst, n, type, count, groups, max_norm, norms, workspace, workspace_bytes, (hipStream_t)stream);
} catch (...) {
  return MGNN_ERR_VALUE;
}

}  // extern "C"
