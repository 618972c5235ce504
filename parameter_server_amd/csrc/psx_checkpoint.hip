// psx_checkpoint.hip — an activation kept in 8 bits between the forward and the backward pass.
//
// Every 32 values of a row share a power of two: e is the least integer with
// max |x| <= 127 * 2^e (kept in [-126, 122]), a value is stored as q = x / 2^e rounded to the
// nearest integer, ties to even, and reads back as q * 2^e: off by at most 2^(e - 1).  The
// scale is a power of two so that the division and the product are exact, and so that q * 2^e
// (7 significant bits) is a bf16 value: a matrix product takes it without another rounding.
// int8 and not e4m3: the same byte, 7 significant bits against 4.
//   codes[rows][groups * 32] int8, zero behind a row's last value; exps[rows][groups] = e + 127.
// A group that holds an Inf or a NaN is marked (255) and reads back as NaN.
// Bound by HBM: one pass, 8 values a lane, the group's maximum over four lanes.  The activation
// is read and written past the caches' keeping (16384 x 8192 bf16: store 86 -> 68 us, load 65 ->
// 58 us, 6.0 and 7.0 TB/s).
#include <hip/hip_runtime.h>
#include <cstdint>
#include "psx_operators.hpp"

namespace psx {

typedef uint32_t c32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t c32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t c32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

namespace {

__device__ __forceinline__ float f_of(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t u_of(float f) { return __builtin_bit_cast(uint32_t, f); }

template <int T>
__device__ __forceinline__ void act_load8(const uint8_t *p, int n, float (&f)[8]) {
  constexpr int es = T == PSX_ACT_F32 ? 4 : 2;
  if (n >= 8) {
#pragma unroll
    for (int w = 0; w < es / 2; ++w) {
      const c32x4 d = __builtin_nontemporal_load(reinterpret_cast<const c32x4_a1 *>(p + 16 * w));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (T == PSX_ACT_F32) f[4 * w + i] = f_of(d[i]);
        if constexpr (T == PSX_ACT_F16) {
          f[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)d[i]);
          f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(d[i] >> 16));
        }
        if constexpr (T == PSX_ACT_BF16) {
          f[2 * i] = f_of(d[i] << 16);
          f[2 * i + 1] = f_of(d[i] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = 0.f;
      if (i < n) {
        if constexpr (T == PSX_ACT_F32) f[i] = reinterpret_cast<const float *>(p)[i];
        else {
          const uint16_t h = reinterpret_cast<const uint16_t *>(p)[i];
          f[i] = T == PSX_ACT_F16 ? (float)__builtin_bit_cast(_Float16, h) : f_of((uint32_t)h << 16);
        }
      }
    }
  }
}

template <int T>
__device__ __forceinline__ uint32_t act_bits(float f) {
  if constexpr (T == PSX_ACT_F16) {
    // 64 * 2^10 can stand for the largest binary16 values: finite values stay finite
    if (__builtin_fabsf(f) > 65504.f && __builtin_fabsf(f) < __builtin_inff()) f = __builtin_copysignf(65504.f, f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
  if constexpr (T == PSX_ACT_BF16) return u_of(f) >> 16;   // exact
  return u_of(f);
}

// Lanes take 8 values each: `lanes` of them (a power of two, at most 256) a row.
struct Place {
  int64_t row, step, col;
};
__device__ __forceinline__ Place place_of(int lanes) {
  const int per = 256 / lanes, r = threadIdx.x / lanes, l = threadIdx.x % lanes;
  return {(int64_t)blockIdx.y * per + r, (int64_t)gridDim.y * per, ((int64_t)blockIdx.x * lanes + l) * 8};
}

template <int T>
__global__ void __launch_bounds__(256) checkpoint_store_kernel(CkArgs a, int lanes) {
  constexpr int es = T == PSX_ACT_F32 ? 4 : 2;
  const Place w = place_of(lanes);
  const int64_t pitch = a.groups * kCkGroup;
  if (w.col >= pitch) return;   // whole groups of four lanes
  const int n = (int)min((int64_t)8, max((int64_t)0, a.cols - w.col));
  for (int64_t r = w.row; r < a.rows; r += w.step) {
    float f[8];
    act_load8<T>(a.p + (r * a.ld + w.col) * es, n, f);
    uint32_t top = 0;   // the magnitudes' bits order as the magnitudes do, Inf and NaN above all
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, u_of(f[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    // 127 = 2^6 * 1.984375
    int e = (int)(top >> 23) - 127 - ((top & 0x7fffffu) <= 0x7e0000u ? 6 : 5);
    e = min(max(e, -126), 122);
    const bool bad = top >= 0x7f800000u;
    const float down = f_of((uint32_t)(127 - e) << 23);
    const float most = e == 122 ? 63.f : 127.f;   // 64 * 2^122 is past the largest f32
    c32x2 q{0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = __builtin_rintf(f[i] * down);
      s = bad ? 0.f : __builtin_fminf(__builtin_fmaxf(s, -most), most);
      q[i / 4] |= ((uint32_t)(int)s & 0xffu) << (i % 4 * 8);
    }
    *reinterpret_cast<c32x2 *>(a.codes + r * pitch + w.col) = q;
    if ((threadIdx.x & 3) == 0) a.exps[r * a.groups + w.col / kCkGroup] = bad ? 255 : (uint8_t)(e + 127);
  }
}

template <int T>
__global__ void __launch_bounds__(256) checkpoint_load_kernel(CkArgs a, int lanes) {
  constexpr int es = T == PSX_ACT_F32 ? 4 : 2;
  const Place w = place_of(lanes);
  const int64_t pitch = a.groups * kCkGroup;
  const int n = (int)min((int64_t)8, max((int64_t)0, a.cols - w.col));
  if (n <= 0) return;
  for (int64_t r = w.row; r < a.rows; r += w.step) {
    const c32x2 q = *reinterpret_cast<const c32x2 *>(a.codes + r * pitch + w.col);
    const uint32_t e = a.exps[r * a.groups + w.col / kCkGroup];
    const float up = f_of(e == 255 ? 0x7fc00000u : e << 23);
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = act_bits<T>((float)(int8_t)(q[i / 4] >> (i % 4 * 8)) * up);
    uint8_t *p = a.p + (r * a.ld + w.col) * es;
    if (n == 8) {
      if constexpr (T == PSX_ACT_F32) {
        __builtin_nontemporal_store(c32x4{o[0], o[1], o[2], o[3]}, reinterpret_cast<c32x4_a1 *>(p));
        __builtin_nontemporal_store(c32x4{o[4], o[5], o[6], o[7]}, reinterpret_cast<c32x4_a1 *>(p + 16));
      } else {
        __builtin_nontemporal_store(c32x4{o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16},
                                    reinterpret_cast<c32x4_a1 *>(p));
      }
    } else {
      for (int i = 0; i < 8; ++i)
        if (i < n) {
          if constexpr (T == PSX_ACT_F32) reinterpret_cast<uint32_t *>(p)[i] = o[i];
          else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)o[i];
        }
    }
  }
}

int ck_lanes(const CkArgs &a) {
  int lanes = 4;
  while (lanes < 256 && lanes < a.groups * 4) lanes *= 2;
  return lanes;
}
dim3 ck_grid(const CkArgs &a, int lanes) {
  const int64_t across = (a.groups * 4 + lanes - 1) / lanes, per = 256 / lanes;
  int64_t down = (a.rows + per - 1) / per;
  if (down > 4096) down = 4096;   // further rows by a loop
  return dim3((unsigned)across, (unsigned)down, 1);
}

}  // namespace

hipError_t launch_checkpoint_store(const CkArgs &a, hipStream_t st) {
  if (a.rows <= 0 || a.cols <= 0) return hipSuccess;
  const int lanes = ck_lanes(a);
  const dim3 g = ck_grid(a, lanes);
  if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(checkpoint_store_kernel<PSX_ACT_F32>, g, dim3(256), 0, st, a, lanes);
  else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(checkpoint_store_kernel<PSX_ACT_F16>, g, dim3(256), 0, st, a, lanes);
  else hipLaunchKernelGGL(checkpoint_store_kernel<PSX_ACT_BF16>, g, dim3(256), 0, st, a, lanes);
  return hipGetLastError();
}

hipError_t launch_checkpoint_load(const CkArgs &a, hipStream_t st) {
  if (a.rows <= 0 || a.cols <= 0) return hipSuccess;
  const int lanes = ck_lanes(a);
  const dim3 g = ck_grid(a, lanes);
  if (a.type == PSX_ACT_F32) hipLaunchKernelGGL(checkpoint_load_kernel<PSX_ACT_F32>, g, dim3(256), 0, st, a, lanes);
  else if (a.type == PSX_ACT_F16) hipLaunchKernelGGL(checkpoint_load_kernel<PSX_ACT_F16>, g, dim3(256), 0, st, a, lanes);
  else hipLaunchKernelGGL(checkpoint_load_kernel<PSX_ACT_BF16>, g, dim3(256), 0, st, a, lanes);
  return hipGetLastError();
}

}  // namespace psx
