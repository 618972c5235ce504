// psx_bias.hip — a learned relative position bias whose buckets are rows of a table, and its
// gradient.  With r = k - q - begin (key position minus query position):
//   bias[h][q][k] = W[bucket(r)][h]
//   grad[j][h]    = gain * sum over b, q, k with bucket(r) = j of d[b][h][q][k]
// bucket(r): both directions: half = buckets / 2, n = |r|, plus half where r > 0; one
// direction: half = buckets, n = max(-r, 0).  n < exact = half / 2 has a bucket of its own;
// behind that, bucket exact + i starts at border[i - 1], the least n with
// (n / exact)^(half - exact) >= (distance / exact)^i (whole numbers, computed by the host).
#include <hip/hip_runtime.h>
#include <cstdint>
#include "psx_operators.hpp"

namespace psx {

typedef uint32_t b32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t b32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

namespace {

template <int T> constexpr int kVec = T == PSX_ACT_F32 ? 4 : 8;   // values of a 16-byte vector
template <int T> constexpr int kEs = T == PSX_ACT_F32 ? 4 : 2;

// The bucket of r; `border` in LDS.
__device__ __forceinline__ int bucket_of(const BiasMap &m, const int *border, int64_t r) {
  const int64_t n64 = r < 0 ? -r : m.both ? r : 0;
  const int n = (int)min(n64, (int64_t)0x7fffffff);
  int b = n;
  if (n >= m.exact) {
    int lo = 0, hi = m.nborder;   // borders at or below n
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (border[mid] <= n) lo = mid + 1;
      else hi = mid;
    }
    b = m.exact + lo;
  }
  return b + (m.both && r > 0 ? m.half : 0);
}

template <int T>
__device__ __forceinline__ uint32_t bias_bits(float f) {
  if constexpr (T == PSX_ACT_F16) return __builtin_bit_cast(uint16_t, (_Float16)f);
  if constexpr (T == PSX_ACT_BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  return __builtin_bit_cast(uint32_t, f);
}

// Both kernels walk a window of distances e = k - q, [e0, e0 + w), for `rows` queries from q0
// on, in V phases of queries q0 + phase + V i: there a thread's V distances lie at a multiple of
// V keys in every row, so a row's vector is the one before it, V keys further, and neither
// kernel looks anything up in its inner loop.
struct Window {
  int64_t q0, q1, e0;
};
__device__ __forceinline__ Window window_of(const BiasTiles &t, int64_t q, int block) {
  Window w;
  w.q0 = (int64_t)(block / t.windows) * t.rows;
  w.q1 = min(q, w.q0 + t.rows);
  w.e0 = (int64_t)(block % t.windows) * t.width - (w.q0 + t.rows - 1) - 7;
  return w;
}
// The phase of query q: the least shift that puts e0 + shift + q at a multiple of V.
template <int V>
__device__ __forceinline__ int shift_of(int64_t e0, int64_t q) { return (int)(((-(e0 + q)) % V + V) % V); }

// One block: one window, one head.  The window's values are laid in LDS once; a thread takes its
// V of them a phase and stores them in every row of the phase.  Bound by the stores (HBM).
template <int T>
__global__ void bias_kernel(BiasArgs a) {
  constexpr int V = kVec<T>, es = kEs<T>;
  extern __shared__ uint32_t line[];   // [width + 8]
  __shared__ float w[kMaxBuckets];
  __shared__ int border[kMaxBuckets];
  const Window win = window_of(a.tiles, a.q, blockIdx.x);
  const int h = blockIdx.y;
  if (win.e0 + win.q0 >= a.k) return;   // past the last key of the first query
  for (int i = threadIdx.x; i < a.map.buckets; i += blockDim.x) {
    w[i] = a.w[(int64_t)i * a.heads + h];
    border[i] = i < a.map.nborder ? a.map.border[i] : 0;
  }
  __syncthreads();
  const int need = (int)min((int64_t)a.tiles.width + 8, a.k - win.q0 - win.e0);
  for (int i = threadIdx.x; i < a.tiles.width + 8; i += blockDim.x)
    line[i] = i < need ? bias_bits<T>(w[bucket_of(a.map, border, win.e0 + i - a.begin)]) : 0;
  __syncthreads();
  if ((int)threadIdx.x * V >= a.tiles.width) return;
  uint8_t *out = a.out + (int64_t)h * a.head_ld * es;
  for (int ph = 0; ph < V && win.q0 + ph < win.q1; ++ph) {
    const int at = shift_of<V>(win.e0, win.q0 + ph) + (int)threadIdx.x * V;
    b32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = T == PSX_ACT_F32 ? line[at + i] : line[at + 2 * i] | line[at + 2 * i + 1] << 16;
    const int64_t e = win.e0 + at;
    // keys e + q in [0, k): queries of this phase from `q` on
    int64_t q = win.q0 + ph;
    if (e + q < 0) q += (-(e + q) + V - 1) / V * V;
    const int64_t end = min(win.q1, a.k - e);
    uint8_t *o = out + (q * a.q_ld + e + q) * es;
    const int64_t step = (a.q_ld + 1) * V * es;
    for (; q < end && e + q + V <= a.k; q += V, o += step) *reinterpret_cast<b32x4_a1 *>(o) = x;
    if (q < end) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e + q + i < a.k) {
          if constexpr (T == PSX_ACT_F32) reinterpret_cast<uint32_t *>(o)[i] = x[i];
          else reinterpret_cast<uint16_t *>(o)[i] = (uint16_t)(x[i / 2] >> (i % 2 * 16));
        }
    }
  }
}

// ---- gradient ---------------------------------------------------------------------------------

template <int T, int V>
__device__ __forceinline__ void add_vec(const b32x4 &d, float (&acc)[V]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = d[i];   // a copy: the builtin below casts a vector's element as its first
    if constexpr (T == PSX_ACT_F32) acc[i] += __builtin_bit_cast(float, w);
    if constexpr (T == PSX_ACT_F16) {
      acc[2 * i] += (float)__builtin_bit_cast(_Float16, (uint16_t)w);
      acc[2 * i + 1] += (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
    }
    if constexpr (T == PSX_ACT_BF16) {
      acc[2 * i] += __builtin_bit_cast(float, w << 16);
      acc[2 * i + 1] += __builtin_bit_cast(float, w & 0xffff0000u);
    }
  }
}
template <int T>
__device__ __forceinline__ float one_value(const uint8_t *p) {
  if constexpr (T == PSX_ACT_F32) return *reinterpret_cast<const float *>(p);
  const uint16_t h = *reinterpret_cast<const uint16_t *>(p);
  return T == PSX_ACT_F16 ? (float)__builtin_bit_cast(_Float16, h) : __builtin_bit_cast(float, (uint32_t)h << 16);
}

// One block: one window of one (batch, head).  A thread adds whole vectors of its phase's rows,
// eight loads at a time, into V registers and those to the window's sums in LDS; short windows
// have `groups` threads a vector, which take the phases among them and add in turn (the order of
// every sum is fixed).  Then a wave sums each bucket's interval.  Bound by the loads (HBM).
template <int T>
__global__ void __launch_bounds__(1024) bias_grad_kernel(BiasGradArgs a) {
  constexpr int V = kVec<T>, es = kEs<T>, U = 8;
  extern __shared__ float sums[];   // [width + 8]
  const int h = blockIdx.y, b = blockIdx.z;
  const Window win = window_of(a.tiles, a.q, blockIdx.x);
  const int width = a.tiles.width, across = a.tiles.threads, group = threadIdx.x / across, vec = threadIdx.x % across;
  const uint8_t *d = a.d + ((int64_t)b * a.batch_ld + (int64_t)h * a.head_ld) * es;
  for (int i = threadIdx.x; i < width + 8; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  for (int p0 = 0; p0 < V; p0 += a.tiles.groups) {
    const int ph = p0 + group;
    const int at = shift_of<V>(win.e0, win.q0 + ph) + vec * V;
    const int64_t e = win.e0 + at;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    if (vec * V < width) {
      int64_t q = win.q0 + ph;
      if (e + q < 0) q += (-(e + q) + V - 1) / V * V;
      const int64_t end = min(win.q1, a.k - e);
      const int64_t whole = min(end, a.k - e - V + 1);   // rows below have the vector's V keys
      const uint8_t *p = d + (q * a.q_ld + e + q) * es;
      const int64_t step = (a.q_ld + 1) * V * es;
      int n = whole > q ? (int)((whole - q + V - 1) / V) : 0;
      q += (int64_t)n * V;
      for (; n >= U; n -= U) {
        b32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const b32x4_a1 *>(p + u * step);
        __builtin_amdgcn_sched_barrier(0);
        p += U * step;
#pragma unroll
        for (int u = 0; u < U; ++u) add_vec<T, V>(x[u], acc);
      }
      if (n > 0) {
        b32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const b32x4_a1 *>(p + min(u, n - 1) * step);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < n) add_vec<T, V>(x[u], acc);
        p += n * step;
      }
      if (q < end) {   // the one row whose vector the last key cuts
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (e + q + i < a.k) acc[i] += one_value<T>(p + i * es);
      }
    }
    for (int g = 0; g < a.tiles.groups; ++g) {
      if (g == group && vec * V < width) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[at + i] += acc[i];
      }
      __syncthreads();
    }
  }
  // bucket j's distances r are an interval; the window's entry i is r = e0 + i - begin
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  float *out = a.partial + (((int64_t)h * a.batch + b) * gridDim.x + blockIdx.x) * a.map.buckets;
  for (int j = wave; j < a.map.buckets; j += waves) {
    const bool after = a.map.both && j >= a.map.half;
    const int jj = after ? j - a.map.half : j, far = jj - a.map.exact;
    const int64_t n0 = jj <= a.map.exact ? jj : a.map.border[far - 1];
    const int64_t n1 = jj < a.map.exact ? jj + 1 : far < a.map.nborder ? a.map.border[far] : (int64_t)1 << 62;
    int64_t r0, r1;   // [r0, r1)
    if (after) {
      r0 = n0 > 0 ? n0 : 1;
      r1 = n1;
    } else {
      r0 = -n1 + 1;
      r1 = -n0 + 1;
      if (!a.map.both && jj == 0) r1 = (int64_t)1 << 62;
    }
    const int64_t i0 = max((int64_t)0, r0 + a.begin - win.e0), i1 = min((int64_t)width + 8, r1 + a.begin - win.e0);
    float s = 0.f;
    for (int64_t i = i0 + lane; i < i1; i += 64) s += sums[i];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    if (lane == 0) out[j] = s;
  }
}

// One wave a (bucket, head): the blocks' sums in double, in a fixed order.
__global__ void __launch_bounds__(64) bias_grad_sum_kernel(BiasGradArgs a) {
  const int j = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int64_t n = (int64_t)a.batch * a.tiles.blocks;
  const float *p = a.partial + (int64_t)h * n * a.map.buckets + j;
  double s = 0;
  for (int64_t i = lane; i < n; i += 64) s += (double)p[i * a.map.buckets];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if (lane == 0) a.grad[(int64_t)j * a.heads + h] = (float)(s * (double)a.gain);
}

}  // namespace

// Windows of at most `most` vectors: distances from -(rows - 1) - 7 above q0 to k - 1 - q0, and
// V - 1 more for the shift.
static BiasTiles tiles_of(int64_t q, int64_t k, int rows, int v, int most) {
  BiasTiles t{};
  t.rows = rows;
  const int64_t all = k + rows + 7 + v;
  t.windows = (int32_t)((all + (int64_t)most * v - 1) / ((int64_t)most * v));
  t.width = (int32_t)(((all + t.windows - 1) / t.windows + v - 1) / v * v);
  t.threads = (t.width / v + 63) / 64 * 64;
  t.groups = 1;
  t.blocks = (int32_t)((q + rows - 1) / rows * t.windows);
  return t;
}

hipError_t launch_bias(const BiasArgs &in, hipStream_t st) {
  if (in.q <= 0 || in.k <= 0) return hipSuccess;
  BiasArgs a = in;
  const int v = a.type == PSX_ACT_F32 ? 4 : 8;
  // 64 queries share a window's values; for a few queries (decode) small windows fill the chip
  a.tiles = tiles_of(a.q, a.k, a.q < 64 ? (int)a.q : 64, v, a.q < 64 ? 128 : 512);
  const dim3 g((unsigned)a.tiles.blocks, (unsigned)a.heads), t((unsigned)a.tiles.threads);
  const size_t lds = (size_t)(a.tiles.width + 8) * 4;
  if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F32>, g, t, lds, st, a);
  else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F16>, g, t, lds, st, a);
  else hipLaunchKernelGGL(bias_kernel<PSX_ACT_BF16>, g, t, lds, st, a);
  return hipGetLastError();
}

// 256 queries a block where that leaves 1024 blocks, 32 at least; windows of 128 vectors (537 MB
// of scores, 2048 x 2048: 95 us; 256 vectors 102, 512 vectors 124 — fewer, longer blocks leave
// the chip uneven).
BiasTiles bias_grad_tiles(int64_t batch, int64_t heads, int64_t q, int64_t k, int32_t type) {
  const int v = type == PSX_ACT_F32 ? 4 : 8;
  int rows = 256;
  while (rows > 32 && (q + rows - 1) / rows * batch * heads < 1024) rows /= 2;
  BiasTiles t = tiles_of(q, k, rows, v, 128);
  while (t.groups < v && t.threads * t.groups * 2 <= 512) t.groups *= 2;
  return t;
}

hipError_t launch_bias_grad(const BiasGradArgs &a, hipStream_t st) {
  if (a.batch > 0 && a.q > 0 && a.k > 0) {
    const dim3 g((unsigned)a.tiles.blocks, (unsigned)a.heads, (unsigned)a.batch), t((unsigned)(a.tiles.threads * a.tiles.groups));
    const size_t lds = (size_t)(a.tiles.width + 8) * 4;
    if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_F32>, g, t, lds, st, a);
    else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_F16>, g, t, lds, st, a);
    else hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_BF16>, g, t, lds, st, a);
  }
  hipLaunchKernelGGL(bias_grad_sum_kernel, dim3((unsigned)a.map.buckets, (unsigned)a.heads), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace psx
