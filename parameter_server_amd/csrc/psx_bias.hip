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

__device__ __forceinline__ int bucket_of(const BiasMap &m, int64_t r) {
  const int64_t n64 = m.both ? (r < 0 ? -r : r) : (r < 0 ? -r : 0);
  const int n = (int)min(n64, (int64_t)0x7fffffff);
  int b = n;
  if (n >= m.exact) {
    b = m.exact;
    for (int i = 0; i < m.nborder; ++i) b += n >= m.border[i];
  }
  return b + (m.both && r > 0 ? m.half : 0);
}

template <int T>
__device__ __forceinline__ uint32_t bias_bits(float f) {
  if constexpr (T == PSX_ACT_F16) return __builtin_bit_cast(uint16_t, (_Float16)f);
  if constexpr (T == PSX_ACT_BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  return __builtin_bit_cast(uint32_t, f);
}

constexpr int kBiasK = 2048, kBiasQ = 16;   // one block's keys and queries

// One block: kBiasQ queries x kBiasK keys of one head.  The values of the distances that occur
// are laid in LDS once (a query's row is that line, shifted); each thread stores 16 bytes.
template <int T>
__global__ void __launch_bounds__(256) bias_kernel(BiasArgs a) {
  constexpr int V = T == PSX_ACT_F32 ? 4 : 8, es = T == PSX_ACT_F32 ? 4 : 2;
  __shared__ float w[kMaxBuckets];
  __shared__ uint32_t line[kBiasK + kBiasQ + 8];
  const int across = (int)((a.k + kBiasK - 1) / kBiasK), h = blockIdx.y;
  const int64_t k0 = (int64_t)(blockIdx.x % across) * kBiasK, q0 = (int64_t)(blockIdx.x / across) * kBiasQ;
  for (int i = threadIdx.x; i < a.map.buckets; i += 256) w[i] = a.w[(int64_t)i * a.heads + h];
  __syncthreads();
  // line[i]: r = k0 + i - (q0 + kBiasQ - 1) - begin
  for (int i = threadIdx.x; i < kBiasK + kBiasQ; i += 256)
    line[i] = bias_bits<T>(w[bucket_of(a.map, k0 + i - (q0 + kBiasQ - 1) - a.begin)]);
  __syncthreads();
  for (int v = threadIdx.x; v < kBiasQ * kBiasK / V; v += 256) {
    const int qi = v / (kBiasK / V), ki = v % (kBiasK / V) * V;
    const int64_t q = q0 + qi, k = k0 + ki;
    if (q >= a.q || k >= a.k) continue;
    const uint32_t *s = line + ki + kBiasQ - 1 - qi;
    uint8_t *o = a.out + ((int64_t)h * a.head_ld + q * a.q_ld + k) * es;
    if (k + V <= a.k) {
      b32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = T == PSX_ACT_F32 ? s[i] : s[2 * i] | s[2 * i + 1] << 16;
      *reinterpret_cast<b32x4_a1 *>(o) = x;
    } else {
      for (int i = 0; i < V; ++i)
        if (k + i < a.k) {
          if constexpr (T == PSX_ACT_F32) reinterpret_cast<uint32_t *>(o)[i] = s[i];
          else reinterpret_cast<uint16_t *>(o)[i] = (uint16_t)s[i];
        }
    }
  }
}

// ---- gradient ---------------------------------------------------------------------------------
constexpr int kGradQ = 256, kGradE = 2048;   // one block's queries and distances

template <int T, int V>
__device__ __forceinline__ void add_vec(const uint8_t *p, float (&acc)[V]) {
  const b32x4 d = *reinterpret_cast<const b32x4_a1 *>(p);
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

// One block: kGradQ queries of one (batch, head), distances e = k - q in a window of
// V * 256.  The queries are taken in V phases, q = q0 + phase + V i: there a thread's V
// distances lie at the same key offset modulo V in every row, so it adds whole 16-byte
// vectors into V registers, and adds those to the window's sums in LDS (own entries, a
// barrier between phases: the order of every sum is fixed).  Then a wave sums each bucket's
// interval of the window.
template <int T>
__global__ void __launch_bounds__(256) bias_grad_kernel(BiasGradArgs a) {
  constexpr int V = T == PSX_ACT_F32 ? 4 : 8, es = T == PSX_ACT_F32 ? 4 : 2, W = kGradE;
  constexpr int passes = W / (256 * V);
  __shared__ float sums[W + 8];
  const int qt = blockIdx.x / a.ktiles, kt = blockIdx.x % a.ktiles, h = blockIdx.y, b = blockIdx.z;
  const int64_t q0 = (int64_t)qt * kGradQ, q1 = min(a.q, q0 + kGradQ);
  const int64_t e0 = (int64_t)kt * W - (q0 + kGradQ - 1) - 7;   // the window's least distance
  const uint8_t *d = a.d + ((int64_t)b * a.batch_ld + (int64_t)h * a.head_ld) * es;
  for (int i = threadIdx.x; i < W + 8; i += 256) sums[i] = 0.f;
  __syncthreads();
  for (int ph = 0; ph < V; ++ph) {
    const int64_t qa = q0 + ph;
    const int adj = (int)(((-(e0 + qa)) % V + V) % V);   // e0 + adj + qa is a multiple of V
#pragma unroll
    for (int s = 0; s < passes; ++s) {
      const int at = adj + (s * 256 + (int)threadIdx.x) * V;   // the thread's first distance is e0 + at
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      // keys e0 + at + q in [0, k): the queries of this phase that have them
      const int64_t lo = max(qa, -(e0 + at)), hi = min(q1, a.k - (e0 + at));
      int64_t q = lo <= qa ? qa : qa + (lo - qa + V - 1) / V * V;
      for (; q < hi; q += V) {
        const int64_t k = e0 + at + q;
        const uint8_t *p = d + (q * a.q_ld + k) * es;
        if (k + V <= a.k) add_vec<T, V>(p, acc);
        else
          for (int i = 0; i < V; ++i)
            if (k + i < a.k) acc[i] += one_value<T>(p + i * es);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sums[at + i] += acc[i];
    }
    __syncthreads();
  }
  // bucket j's distances r are an interval; the window's entry i is r = e0 + i - begin
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *out = a.partial + (((int64_t)h * a.batch + b) * a.qtiles * a.ktiles + blockIdx.x) * a.map.buckets;
  for (int j = wave; j < a.map.buckets; j += 4) {
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
    const int64_t i0 = max((int64_t)0, r0 + a.begin - e0), i1 = min((int64_t)W + 8, r1 + a.begin - e0);
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
  const int64_t n = (int64_t)a.batch * a.qtiles * a.ktiles;
  const float *p = a.partial + (int64_t)h * n * a.map.buckets + j;
  double s = 0;
  for (int64_t i = lane; i < n; i += 64) s += (double)p[i * a.map.buckets];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  if (lane == 0) a.grad[(int64_t)j * a.heads + h] = (float)(s * (double)a.gain);
}

}  // namespace

hipError_t launch_bias(const BiasArgs &a, hipStream_t st) {
  if (a.q <= 0 || a.k <= 0) return hipSuccess;
  const dim3 g((unsigned)((a.k + kBiasK - 1) / kBiasK * ((a.q + kBiasQ - 1) / kBiasQ)), (unsigned)a.heads);
  if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F32>, g, dim3(256), 0, st, a);
  else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(bias_kernel<PSX_ACT_F16>, g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(bias_kernel<PSX_ACT_BF16>, g, dim3(256), 0, st, a);
  return hipGetLastError();
}

// Windows of distances: e from -(kGradQ - 1) - 7 above q0 to k - 1.
void bias_grad_tiles(int64_t q, int64_t k, int32_t *qtiles, int32_t *ktiles) {
  *qtiles = (int32_t)((q + kGradQ - 1) / kGradQ);
  *ktiles = (int32_t)((k + kGradQ - 1 + 7 + kGradE - 1) / kGradE);
}

hipError_t launch_bias_grad(const BiasGradArgs &a, hipStream_t st) {
  if (a.batch > 0 && a.qtiles > 0 && a.ktiles > 0 && a.q > 0 && a.k > 0) {
    const dim3 g((unsigned)(a.qtiles * a.ktiles), (unsigned)a.heads, (unsigned)a.batch);
    if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_F32>, g, dim3(256), 0, st, a);
    else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_F16>, g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(bias_grad_kernel<PSX_ACT_BF16>, g, dim3(256), 0, st, a);
  }
  hipLaunchKernelGGL(bias_grad_sum_kernel, dim3((unsigned)a.map.buckets, (unsigned)a.heads), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace psx
