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
template <int ES> struct BitsOf { typedef uint32_t type; };
template <> struct BitsOf<2> { typedef uint16_t type; };

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

// One block: `rows` queries x `keys` keys of one head.  The values of the block's distances are
// laid in LDS once, V times, the p-th time p distances on: a query's vectors of V keys then are
// aligned vectors of one of the copies, and the stores run through the rows, whole lines each.
// Bound by the stores (HBM).  268 MB (32 heads, 2048 x 2048, bf16), one call after another:
// 55 us, 4.9 TB/s; a plain fill of as much takes 40.
template <int T>
__global__ void __launch_bounds__(256) bias_kernel(BiasArgs a) {
  constexpr int V = kVec<T>, es = kEs<T>;
  typedef typename BitsOf<es>::type U;
  extern __shared__ b32x4 copies[];   // [phases][pitch]
  __shared__ float w[kMaxBuckets];
  __shared__ int border[kMaxBuckets];
  const int across = (int)((a.k + a.keys - 1) / a.keys), h = blockIdx.y;
  const int64_t k0 = (int64_t)(blockIdx.x % across) * a.keys, q0 = (int64_t)(blockIdx.x / across) * a.rows;
  for (int i = threadIdx.x; i < a.map.buckets; i += 256) {
    w[i] = a.w[(int64_t)i * a.heads + h];
    border[i] = i < a.map.nborder ? a.map.border[i] : 0;
  }
  __syncthreads();
  // distance i is key k0 + i - (rows - 1) against query q0: the block's least is 0
  const int all = a.keys + a.rows + V, pitch = all / V + 1, phases = a.rows < V ? a.rows : V;
  U *c = reinterpret_cast<U *>(copies);
  for (int i = threadIdx.x; i < all; i += 256) {
    const U x = (U)bias_bits<T>(w[bucket_of(a.map, border, k0 + i - (q0 + a.rows - 1) - a.begin)]);
    for (int p = 0; p < phases; ++p)
      if (i >= p) c[p * pitch * V + i - p] = x;
  }
  __syncthreads();
  const int rows = (int)min((int64_t)a.rows, a.q - q0);
  for (int kk = (int)threadIdx.x * V; kk < a.keys && k0 + kk < a.k; kk += 256 * V) {
    const int n = (int)min((int64_t)V, a.k - k0 - kk);
    uint8_t *o = a.out + ((int64_t)h * a.head_ld + q0 * a.q_ld + k0 + kk) * es;
#pragma unroll 4
    for (int r = 0; r < rows; ++r, o += a.q_ld * es) {
      const int at = kk + a.rows - 1 - r, p = at % V;
      const b32x4 x = copies[p * pitch + at / V];
      if (n == V) {
        *reinterpret_cast<b32x4_a1 *>(o) = x;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < n) {
            if constexpr (T == PSX_ACT_F32) reinterpret_cast<uint32_t *>(o)[i] = x[i];
            else reinterpret_cast<uint16_t *>(o)[i] = (uint16_t)(x[i / 2] >> (i % 2 * 16));
          }
      }
    }
  }
}

// The gradient walks a window of distances e = k - q, [e0, e0 + width), for `rows` queries from
// q0 on, in V phases of queries q0 + phase + V i: there a thread's V distances lie at a multiple
// of V keys in every row, so a row's vector is the one before it, V keys further, and nothing is
// looked up in the inner loop.
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
  t.windows = (int32_t)((all + (int64_t)most * v - 1) / ((int64_t)most * v));   // lengths end at 2^24
  t.width = (int32_t)(((all + t.windows - 1) / t.windows + v - 1) / v * v);
  t.threads = (t.width / v + 63) / 64 * 64;
  t.groups = 1;
  t.blocks = (q + rows - 1) / rows * t.windows;
  return t;
}

int64_t bias_blocks(BiasArgs &a) {
  if (a.q <= 0 || a.k <= 0) return 0;
  // 64 queries share a block's values, or as many as there are (decode)
  a.rows = a.q < 64 ? (int32_t)a.q : 64;
  a.keys = a.q < 16 ? 1024 : a.type == PSX_ACT_F32 ? 1024 : 2048;
  return (a.k + a.keys - 1) / a.keys * ((a.q + a.rows - 1) / a.rows);
}

hipError_t launch_bias(const BiasArgs &in, hipStream_t st) {
  BiasArgs a = in;
  const int64_t blocks = bias_blocks(a);
  if (blocks == 0) return hipSuccess;
  const int v = a.type == PSX_ACT_F32 ? 4 : 8;
  const int phases = a.rows < v ? a.rows : v, pitch = (a.keys + a.rows + v) / v + 1;
  const dim3 g((unsigned)blocks, (unsigned)a.heads);
  const size_t lds = (size_t)phases * pitch * 16;
  if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F32>, g, dim3(256), lds, st, a);
  else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F16>, g, dim3(256), lds, st, a);
  else hipLaunchKernelGGL(bias_kernel<PSX_ACT_BF16>, g, dim3(256), lds, st, a);
  return hipGetLastError();
}

// 256 queries a block where that leaves 1024 blocks, 32 at least; windows of 128 vectors (537 MB
// of scores, 2048 x 2048: 95 us; 256 vectors 102, 512 vectors 124 — fewer, longer blocks leave
// the chip uneven).
BiasTiles bias_grad_tiles(int64_t batch, int64_t heads, int64_t q, int64_t k, int32_t type) {
  if (batch == 0 || q == 0 || k == 0) return BiasTiles{};   // no partial sums at all
  const int v = type == PSX_ACT_F32 ? 4 : 8;
  int rows = 256;
  while (rows > 32 && (q + rows - 1) / rows * batch * heads < 1024) rows /= 2;
  BiasTiles t = tiles_of(q, k, rows, v, 128);
  while (t.groups < v && t.threads * t.groups * 2 <= 512) t.groups *= 2;
  return t;
}

hipError_t launch_bias_grad(const BiasGradArgs &a, hipStream_t st) {
  if (a.tiles.blocks > 0) {
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
