// psx_adapter.hip — low-rank adapters whose rank rows are rows of two tables, for a batch of
// requests: request n owns tokens [begin[n], begin[n + 1]) and one adapter (or none).
//
//   shrink   v[t][r]   = sum_k x[t][k] W[slot + r][k]            (x, table A; dy, table B)
//   expand   out[t][j] = base[t][j] + s sum_r v[t][r] W[slot + r][j]
//   grad     g[r][j]   = gain s sum_t v[t][r] x[t][j]            (partial sums, then their sum)
//
// Arithmetic.  The tables are f32 and a server adds increments far below a bf16 step to them,
// so an f32 operand is cut into bf16 parts by truncation: 8 + 8 + 8 significant bits, each
// remainder exact, so three parts are the f32 value itself.  A product of parts is exact in
// f32, and v_mfma_f32_16x16x32_bf16 adds in f32: the products (i, j) with i + j <= 2 leave out
// less than 2^-23 of a product.  A bf16 activation is one part, binary16 two, f32 three, an
// 8-bit checkpoint (7 significant bits and a power of two) one.  16-bit outputs are rounded
// once; expand takes two parts a factor for them (2^-16 against their 2^-9 or 2^-12).
// A factor that is not finite makes the products that it meets NaN.
//
// Operand layout of the 16x16x32 product: lane l holds row (or column) l % 16 and 8 values of
// k; both operands number k alike, so any order of k will do.  The result: column l % 16,
// rows (l / 16) * 4 + i.
#include <hip/hip_runtime.h>
#include <cstdint>
#include "psx_operators.hpp"

namespace psx {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// rows of odd widths start at any multiple of their element: the vector loads and stores of
// global memory take any address
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

enum { kF32 = PSX_ACT_F32, kF16 = PSX_ACT_F16, kBF16 = PSX_ACT_BF16 };

template <int XT> struct ActInfo;
template <> struct ActInfo<kF32> { static constexpr int parts = 3, size = 4; };
template <> struct ActInfo<kF16> { static constexpr int parts = 2, size = 2; };
template <> struct ActInfo<kBF16> { static constexpr int parts = 1, size = 2; };
template <> struct ActInfo<kAct8> { static constexpr int parts = 1, size = 1; };

__device__ __forceinline__ float as_f(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_u(float f) { return __builtin_bit_cast(uint32_t, f); }
// the top halves of two words: a's below, b's above
__device__ __forceinline__ uint32_t tops(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t bottoms(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ float half_at(uint32_t w, int hi) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
}

// Eight f32 values as P bf16 fragments.
template <int P>
__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&o)[P]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    float a = v[2 * d], b = v[2 * d + 1];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      o[p][d] = tops(as_u(a), as_u(b));
      if (p + 1 < P) {
        a -= as_f(as_u(a) & 0xffff0000u);
        b -= as_f(as_u(b) & 0xffff0000u);
      }
    }
  }
}

template <int PA, int PB>
__device__ __forceinline__ void products(f32x4 &acc, const u32x4 (&a)[PA], const u32x4 (&b)[PB]) {
  constexpr int deep = PA > PB ? PA : PB;
#pragma unroll
  for (int i = 0; i < PA; ++i)
#pragma unroll
    for (int j = 0; j < PB; ++j)
      if (i + j < deep)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[j]),
                                                      acc, 0, 0, 0);
}

// 2^e of a checkpoint's exponent byte e + 127; 255 marks a group that held an Inf or a NaN.
__device__ __forceinline__ float ck_scale(uint32_t e) { return as_f(e == 255 ? 0x7fc00000u : e << 23); }

// ---- the batch ------------------------------------------------------------------------------

__device__ __forceinline__ int begin_of(const BatchView &b, int n) { return min(max(b.begin[n], 0), b.tokens); }

// Work item `item` of tiles of M tokens: tile c of request n has the number c + n, which rises
// strictly along the requests, so that ceil(tokens / M) + requests numbers hold every
// (tile, request) that meet.  Every lane of the wave calls it.  False: nothing to do.
struct Item {
  int n, t0, t1;
};
__device__ __forceinline__ bool find_item(const BatchView &b, int M, int item, int lane, Item *out) {
  int lo = 0, hi = b.requests;
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64, j = lo + lane * step;
    const bool p = j < hi && begin_of(b, j) / M + j <= item;
    const int c = __builtin_popcountll(__ballot(p));
    if (c == 0) return false;
    lo += (c - 1) * step;
    hi = min(hi, lo + step);
  }
  const int j = lo + lane;
  const bool p = j < hi && begin_of(b, j) / M + j <= item;
  const int c = __builtin_popcountll(__ballot(p));
  if (lo + c == 0) return false;
  const int n = lo + c - 1;
  const int64_t tile = (int64_t)(item - n) * M;
  const int64_t t0 = max((int64_t)begin_of(b, n), tile), t1 = min((int64_t)begin_of(b, n + 1), tile + M);
  if (t0 >= t1) return false;
  *out = {n, (int)t0, (int)t1};
  return true;
}

__device__ __forceinline__ int adapter_of(const BatchView &b, int n) {
  const int a = b.which[n];
  return a >= 0 && a < b.adapters ? a : -1;
}

__device__ __forceinline__ void check_batch(const BatchView &b) {
  uint32_t bad = 0;
  for (int n = threadIdx.x; n < b.requests; n += blockDim.x) {
    const int t0 = b.begin[n], t1 = b.begin[n + 1], a = b.which[n];
    if (t0 < 0 || t0 > t1 || t1 > b.tokens) bad |= kOpRequests;
    if (a < -1 || a >= b.adapters) bad |= kOpAdapter;
  }
  if (bad) atomicOr(b.status, bad);
}

// ---- shrink -----------------------------------------------------------------------------------

// Sixteen consecutive values of a row, as they lie in memory.
template <int XT> struct Raw16 {
  static constexpr int words = ActInfo<XT>::size;   // 16-byte words
  u32x4 d[words];
  __device__ __forceinline__ void load(const uint8_t *p) {
#pragma unroll
    for (int i = 0; i < words; ++i) d[i] = *reinterpret_cast<const u32x4_a1 *>(p + 16 * i);
  }
  // the first n values, zeros behind them
  __device__ __forceinline__ void load_tail(const uint8_t *p, int n) {
#pragma unroll
    for (int i = 0; i < words; ++i) d[i] = u32x4{0, 0, 0, 0};
    if constexpr (XT == kF32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n) d[i / 4][i % 4] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n) d[i / 8][i / 2 % 4] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (i % 2 * 16);
    }
  }
  // values [8 h, 8 h + 8) as bf16 fragments
  __device__ __forceinline__ void parts(int h, u32x4 (&o)[ActInfo<XT>::parts]) const {
    if constexpr (XT == kBF16) {
      o[0] = d[h];
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (XT == kF32) f[i] = as_f(d[2 * h + i / 4][i % 4]);
        if constexpr (XT == kF16) f[i] = half_at(d[h][i / 2], i % 2);
      }
      split8<ActInfo<XT>::parts>(f, o);
    }
  }
};

// One block: one item (up to 16 MT tokens of one request) and one part of k; its four waves
// take chunks of 64 k in turn and add their sums in LDS.  A wave reads each token's row and
// each rank row in pieces of 128 bytes or more (16 consecutive values a lane), once.
template <int XT, int MT, int NR>
__global__ void __launch_bounds__(256) adapter_shrink_kernel(ShrinkArgs a) {
  constexpr int PX = ActInfo<XT>::parts, es = ActInfo<XT>::size;
  __shared__ f32x4 red[3][MT * NR][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_batch(a.b);
  Item it;
  if (!find_item(a.b, 16 * MT, blockIdx.x, lane, &it)) return;
  const int id = adapter_of(a.b, it.n);
  if (id < 0) return;
  const AdapterDev ad = a.b.ads[id];
  const int r0 = blockIdx.z * 16 * NR;
  if (r0 >= ad.rank) return;
  const int row = lane & 15, quad = lane >> 4;
  // tokens and rows past the last are read as the last again; what they give is not used
  const uint8_t *xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = min(it.t0 + m * 16 + row, it.t1 - 1);
    xp[m] = a.x.p + (t * a.x.ld + quad * 16) * es;
  }
  const float *wp[NR];
#pragma unroll
  for (int j = 0; j < NR; ++j)
    wp[j] = a.w + (int64_t)((a.use_b ? ad.slot_b : ad.slot_a) + min(r0 + j * 16 + row, ad.rank - 1)) * a.d + quad * 16;
  const int nr = min(NR, (ad.rank - r0 + 15) / 16), mt = (it.t1 - it.t0 + 15) / 16;
  f32x4 acc[MT][NR];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NR; ++j) acc[m][j] = f32x4{0, 0, 0, 0};

  auto multiply = [&](const Raw16<XT> (&x)[MT], const f32x4 (&w)[NR][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 wf[NR][3];
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = w[j][2 * h + i / 4][i % 4];
        split8<3>(f, wf[j]);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m < mt) {
          u32x4 xf[PX];
          x[m].parts(h, xf);
#pragma unroll
          for (int j = 0; j < NR; ++j)
            if (j < nr) products<3, PX>(acc[m][j], wf[j], xf);
        }
      }
    }
  };

  const int chunks = (int)((a.d + 63) / 64), full = (int)(a.d / 64);
  const int per = (chunks + a.splits - 1) / a.splits;
  const int c0 = blockIdx.y * per, c1 = min(chunks, c0 + per);
  for (int c = c0 + wave; c < min(c1, full); c += 4) {
    const int64_t k = (int64_t)c * 64;
    Raw16<XT> x[MT];
    f32x4 w[NR][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < mt) x[m].load(xp[m] + k * es);
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j < nr) w[j][i] = *reinterpret_cast<const f32x4_a4 *>(wp[j] + k + 4 * i);
    multiply(x, w);
  }
  if (c1 > full && c0 <= full && (full - c0) % 4 == wave) {   // the last, short chunk
    const int64_t k = (int64_t)full * 64;
    const int n = (int)min((int64_t)16, max((int64_t)0, a.d - k - quad * 16));
    Raw16<XT> x[MT];
    f32x4 w[NR][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m].load_tail(xp[m] + k * es, n);
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) w[j][i / 4][i % 4] = i < n ? wp[j][k + i] : 0.f;
    multiply(x, w);
  }

  if (wave) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NR; ++j) red[wave - 1][m * NR + j][lane] = acc[m][j];
  }
  __syncthreads();
  if (wave) return;
  float *v = a.v + blockIdx.y * a.part;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = it.t0 + m * 16 + row;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      if (t >= it.t1 || j >= nr) continue;
      f32x4 s = acc[m][j];
#pragma unroll
      for (int w = 0; w < 3; ++w) s += red[w][m * NR + j][lane];
      *reinterpret_cast<f32x4 *>(v + t * a.rl + r0 + j * 16 + quad * 4) = s;
    }
  }
}

// Tokens a shrink block takes.  Sixteen while the batch is short (decode steps, where each
// request has one token), 64 above, where a rank row read once should serve more tokens.
int adapter_tile(int64_t tokens) { return tokens <= 1024 ? 16 : 64; }
// Parts that k is cut into, so that a short batch still fills the chip.
int adapter_splits(int64_t tokens, int64_t d) {
  const int64_t items = (tokens + adapter_tile(tokens) - 1) / adapter_tile(tokens);
  const int64_t want = items > 0 ? 512 / items : 1, most = (d + 255) / 256;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

template <int XT, int MT>
static void shrink_nr(const ShrinkArgs &a, dim3 g, hipStream_t st) {
  if (a.max_rank <= 16) hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 1>), g, dim3(256), 0, st, a);
  else if (a.max_rank <= 32) hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 2>), g, dim3(256), 0, st, a);
  else {
    g.z = (a.max_rank + 63) / 64;
    hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 4>), g, dim3(256), 0, st, a);
  }
}

template <int XT>
static void shrink_mt(const ShrinkArgs &a, hipStream_t st) {
  const int M = adapter_tile(a.b.tokens);
  const dim3 g((unsigned)((a.b.tokens + M - 1) / M + a.b.requests), (unsigned)a.splits, 1);
  if (M == 16) shrink_nr<XT, 1>(a, g, st);
  else shrink_nr<XT, 4>(a, g, st);
}

hipError_t launch_adapter_shrink(const ShrinkArgs &a, hipStream_t st) {
  if (a.x.type == kF32) shrink_mt<kF32>(a, st);
  else if (a.x.type == kF16) shrink_mt<kF16>(a, st);
  else shrink_mt<kBF16>(a, st);
  return hipGetLastError();
}

// ---- expand -------------------------------------------------------------------------------------

// v[t][r0 .. r0 + 8) over its parts; zero at and behind `rank`.
__device__ __forceinline__ void v_load8(const float *v, int64_t part, int splits, int r0, int rank, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  if (r0 < rank) {   // rows of v end at a multiple of 16: all eight lie inside
    for (int s = 0; s < splits; ++s) {
      const f32x4 lo = *reinterpret_cast<const f32x4 *>(v + s * part + r0);
      const f32x4 hi = *reinterpret_cast<const f32x4 *>(v + s * part + r0 + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] += lo[i];
        f[i + 4] += hi[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r0 + i >= rank) f[i] = 0.f;
  }
}

template <int YT>
__device__ __forceinline__ float out_value(const uint8_t *p, int i) {
  if constexpr (YT == kF32) return reinterpret_cast<const float *>(p)[i];
  if constexpr (YT == kF16) return half_at(reinterpret_cast<const uint16_t *>(p)[i], 0);
  return as_f((uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << 16);
}
template <int YT>
__device__ __forceinline__ uint32_t out_bits(float f) {
  if constexpr (YT == kF32) return as_u(f);
  if constexpr (YT == kF16) return __builtin_bit_cast(uint16_t, (_Float16)f);
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}

// Sixteen consecutive outputs of a row, n of them real.
template <int YT>
__device__ __forceinline__ void out_load16(const uint8_t *p, int n, float (&f)[16]) {
  constexpr int es = ActInfo<YT>::size;
  if (n >= 16) {
#pragma unroll
    for (int w = 0; w < es; ++w) {
      const u32x4 d = *reinterpret_cast<const u32x4_a1 *>(p + 16 * w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (YT == kF32) f[4 * w + i] = as_f(d[i]);
        if constexpr (YT == kF16) {
          f[8 * w + 2 * i] = half_at(d[i], 0);
          f[8 * w + 2 * i + 1] = half_at(d[i], 1);
        }
        if constexpr (YT == kBF16) {
          f[8 * w + 2 * i] = as_f(d[i] << 16);
          f[8 * w + 2 * i + 1] = as_f(d[i] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = i < n ? out_value<YT>(p, i) : 0.f;
  }
}
template <int YT>
__device__ __forceinline__ void out_store16(uint8_t *p, int n, const float (&f)[16]) {
  constexpr int es = ActInfo<YT>::size;
  if (n >= 16) {
#pragma unroll
    for (int w = 0; w < es; ++w) {
      u32x4 d;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (YT == kF32) d[i] = as_u(f[4 * w + i]);
        else d[i] = out_bits<YT>(f[8 * w + 2 * i]) | out_bits<YT>(f[8 * w + 2 * i + 1]) << 16;
      }
      *reinterpret_cast<u32x4_a1 *>(p + 16 * w) = d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) {
        if constexpr (YT == kF32) reinterpret_cast<uint32_t *>(p)[i] = out_bits<YT>(f[i]);
        else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)out_bits<YT>(f[i]);
      }
  }
}

// One wave: 64 columns of one item's tokens.  Row m of product q is column 4 m + q, so that a
// lane loads four columns of a rank row at once and ends with 16 consecutive outputs of one
// token.  Up to 32 KS ranks the rank rows stay in registers over the item's tokens.
template <int YT, int KS>
__global__ void __launch_bounds__(256) adapter_expand_kernel(ExpandArgs a) {
  constexpr int P = YT == kF32 ? 3 : 2, es = ActInfo<YT>::size;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Item it;
  if (!find_item(a.b, a.tile, blockIdx.x, lane, &it)) return;
  const int row = lane & 15, quad = lane >> 4;
  const int64_t j0 = (int64_t)blockIdx.y * 256 + wave * 64, c0 = j0 + quad * 16;
  if (j0 >= a.d) return;
  const int nc = (int)min((int64_t)16, max((int64_t)0, a.d - c0));
  const int id = adapter_of(a.b, it.n);
  AdapterDev ad{};
  if (id >= 0) ad = a.b.ads[id];
  else if (a.base == a.out) return;
  const float *w = a.w + (int64_t)(a.use_b ? ad.slot_b : ad.slot_a) * a.d;

  u32x4 wf[KS][4][P];
  auto load_rows = [&](int g0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float f[4][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = g0 + s * 32 + quad * 8 + i;
        const int64_t j = j0 + 4 * row;
        const float *p = w + (int64_t)r * a.d + j;
        f32x4 x{0, 0, 0, 0};
        if (r < ad.rank) {
          if (j + 4 <= a.d) x = *reinterpret_cast<const f32x4_a4 *>(p);
          else
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (j + q < a.d) x[q] = p[q];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) f[q][i] = x[q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) split8<P>(f[q], wf[s][q]);
    }
  };
  const bool resident = ad.rank <= 32 * KS;
  if (resident) load_rows(0);
  for (int tt = it.t0; tt < it.t1; tt += 16) {
    const int64_t t = min(tt + row, it.t1 - 1);
    float b[16];
    if (a.base) out_load16<YT>(a.base + (t * a.base_ld + c0) * es, nc, b);
    else
#pragma unroll
      for (int i = 0; i < 16; ++i) b[i] = 0.f;
    f32x4 acc[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = f32x4{0, 0, 0, 0};
    for (int g0 = 0; g0 < ad.rank; g0 += 32 * KS) {
      if (!resident) load_rows(g0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float f[8];
        v_load8(a.v + t * a.rl, a.part, a.splits, g0 + s * 32 + quad * 8, ad.rank, f);
        u32x4 vf[P];
        split8<P>(f, vf);
#pragma unroll
        for (int q = 0; q < 4; ++q) products<P, P>(acc[q], wf[s][q], vf);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = __builtin_fmaf(ad.scale, acc[i % 4][i / 4], b[i]);
    if (tt + row < it.t1) out_store16<YT>(a.out + (t * a.out_ld + c0) * es, nc, b);
  }
}

template <int YT>
static void expand_ks(const ExpandArgs &a, dim3 g, hipStream_t st) {
  if (a.max_rank <= 32) hipLaunchKernelGGL((adapter_expand_kernel<YT, 1>), g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_expand_kernel<YT, 2>), g, dim3(256), 0, st, a);
}

hipError_t launch_adapter_expand(const ExpandArgs &a, hipStream_t st) {
  const dim3 g((unsigned)((a.b.tokens + a.tile - 1) / a.tile + a.b.requests), (unsigned)((a.d + 255) / 256), 1);
  if (a.type == kF32) expand_ks<kF32>(a, g, st);
  else if (a.type == kF16) expand_ks<kF16>(a, g, st);
  else expand_ks<kBF16>(a, g, st);
  return hipGetLastError();
}

// ---- grad -----------------------------------------------------------------------------------------

// Q consecutive values of a row as they lie in memory.
template <int XT, int Q> struct RawQ {
  static constexpr int words = ActInfo<XT>::size * Q / 4;
  uint32_t d[words];
  float scale;
  __device__ __forceinline__ void load(const uint8_t *p, const uint8_t *e, int n) {
    if (XT == kAct8 || n >= Q) {   // a checkpoint's rows are padded
      if constexpr (words == 2) {
        const u32x2 v = *reinterpret_cast<const u32x2_a1 *>(p);
        d[0] = v[0];
        d[1] = v[1];
      } else {
        const u32x4 v = *reinterpret_cast<const u32x4_a1 *>(p);
        d[0] = v[0];
        d[1] = v[1];
        d[2] = v[2];
        d[3] = v[3];
      }
      if constexpr (XT == kAct8) scale = ck_scale(*e);
    } else {
#pragma unroll
      for (int i = 0; i < words; ++i) d[i] = 0;
#pragma unroll
      for (int i = 0; i < Q; ++i)
        if (i < n) {
          if constexpr (XT == kF32) d[i] = reinterpret_cast<const uint32_t *>(p)[i];
          else d[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (i % 2 * 16);
        }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < words; ++i) d[i] = 0;
    scale = 0.f;
  }
  __device__ __forceinline__ float value(int q) const {
    if constexpr (XT == kF32) return as_f(d[q]);
    if constexpr (XT == kF16) return half_at(d[q / 2], q % 2);
    return (float)(int8_t)(d[q / 4] >> (q % 4 * 8)) * scale;
  }
};

// Eight tokens' values of column q as fragments: pairs of tokens from two words by one byte
// permutation, so the transposition costs no LDS.
template <int XT, int Q>
__device__ __forceinline__ void column_parts(const RawQ<XT, Q> (&x)[8], int q, u32x4 (&o)[ActInfo<XT>::parts]) {
  if constexpr (XT == kBF16) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
      o[0][d] = q % 2 ? tops(x[2 * d].d[q / 2], x[2 * d + 1].d[q / 2]) : bottoms(x[2 * d].d[q / 2], x[2 * d + 1].d[q / 2]);
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = x[i].value(q);
    split8<ActInfo<XT>::parts>(f, o);
  }
}

// Items of one gradient: adapter i's tokens, all its requests one after another, in chunks;
// start[i] = the first item of adapter i.  The items of an adapter that has two or more leave
// partial sums in slots from start[adapters + 1 + i] on.  Computed by every block (LDS counts
// are whole numbers: their order does not matter).
__device__ __forceinline__ void grad_items(const BatchView &b, int chunk, int32_t *start) {
  int32_t *slot = start + b.adapters + 1;
  for (int i = threadIdx.x; i <= b.adapters; i += blockDim.x) start[i] = 0;
  if (threadIdx.x == 0) slot[0] = 0;
  __syncthreads();
  for (int n = threadIdx.x; n < b.requests; n += blockDim.x) {
    const int id = adapter_of(b, n), len = begin_of(b, n + 1) - begin_of(b, n);
    if (id >= 0 && len > 0) atomicAdd(&start[id + 1], len);
  }
  __syncthreads();
  if (threadIdx.x < 64) {   // prefix sums, 64 adapters at a time
    int carry = 0, carry2 = 0;
    for (int i0 = 0; i0 < b.adapters; i0 += 64) {
      const int i = i0 + (int)threadIdx.x;
      int s = i < b.adapters ? (int)(((int64_t)start[i + 1] + chunk - 1) / chunk) : 0, s2 = s > 1 ? s : 0;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int u = __shfl_up(s, m, 64), u2 = __shfl_up(s2, m, 64);
        if ((int)threadIdx.x >= m) {
          s += u;
          s2 += u2;
        }
      }
      if (i < b.adapters) {
        start[i + 1] = carry + s;
        slot[i + 1] = carry2 + s2;
      }
      carry += __shfl(s, 63, 64);
      carry2 += __shfl(s2, 63, 64);
    }
  }
  __syncthreads();
}

// The tokens [from, to) of adapter `id`, counted over its requests, in steps of up to 32 of one
// request.  Every wave of a block walks the same steps.
struct Steps {
  const BatchView &b;
  int id, lane;
  int64_t from, to, at = 0;
  int n0 = -64, b0 = 0, b1 = 0, tt = 0, t1 = 0;
  uint64_t todo = 0;
  __device__ __forceinline__ Steps(const BatchView &b_, int id_, int lane_, int64_t from_, int64_t to_)
      : b(b_), id(id_), lane(lane_), from(from_), to(to_) {}
  __device__ __forceinline__ bool next(int *t, int *end) {
    while (tt >= t1) {
      if (at >= to) return false;
      while (!todo) {
        n0 += 64;
        if (n0 >= b.requests) return false;
        const int n = n0 + lane;
        b0 = b1 = 0;
        if (n < b.requests && adapter_of(b, n) == id) {
          b0 = begin_of(b, n);
          b1 = begin_of(b, n + 1);
        }
        todo = __ballot(b1 > b0);
      }
      const int src = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int s0 = __builtin_amdgcn_readlane(b0, src), s1 = __builtin_amdgcn_readlane(b1, src);
      tt = (int)min((int64_t)s1, s0 + max((int64_t)0, from - at));
      t1 = (int)min((int64_t)s1, s0 + to - at);
      at += s1 - s0;
    }
    *t = tt;
    *end = t1;
    tt += 32;
    return true;
  }
};

// Columns a lane takes: 16 bytes of a row for few ranks, 8 where the sums of more ranks fill the
// registers; a checkpoint's values are a byte.
template <int XT, int NR> struct GradCols { static constexpr int value = XT == kAct8 || (NR == 1 && XT != kF32) ? 8 : 4; };

// One block: 64 Q columns (its four waves side by side) and one item.  A step is 32 tokens: a
// wave loads Q columns of 8 tokens a lane (the next step's before this step's products), turns
// them into fragments in registers, and takes v's fragments from LDS, where one wave a rank
// tile has cut them into parts.  Both sums over tokens are f32 in the matrix unit.
template <int XT, int NR>
__device__ __forceinline__ void grad_block(const GradArgs &a, int block, int32_t *start, u32x4 (*frag)[NR][3][64]) {
  constexpr int PX = ActInfo<XT>::parts, es = ActInfo<XT>::size, Q = GradCols<XT, NR>::value;
  grad_items(a.b, a.chunk, start);
  if (block == 0 && blockIdx.z == 0)
    for (int i = threadIdx.x; i < a.b.adapters; i += blockDim.x)
      a.items[i] = int2{start[a.b.adapters + 1 + i], start[i + 1] - start[i]};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int across = (int)((a.d + 64 * Q - 1) / (64 * Q)), item = block / across;
  if (item >= start[a.b.adapters]) return;
  int lo = 0, hi = a.b.adapters;   // the adapter with start[lo] <= item < start[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (start[mid] <= item) lo = mid;
    else hi = mid;
  }
  const int id = lo;
  const AdapterDev ad = a.b.ads[id];
  const int r0 = blockIdx.z * 16 * NR;
  if (r0 >= ad.rank) return;
  const int nr = min(NR, (ad.rank - r0 + 15) / 16);
  const int row = lane & 15, quad = lane >> 4;
  const int64_t j0 = ((int64_t)(block % across) * 4 + wave) * 16 * Q, j = j0 + Q * row;
  const int nc = (int)min((int64_t)Q, max((int64_t)0, a.d - j));
  const bool whole_cols = j0 + 16 * Q <= a.d;
  const int64_t from = (int64_t)(item - start[id]) * a.chunk;
  Steps steps(a.b, id, lane, from, from + a.chunk);
  const uint8_t *xp = a.x.p + j * es;
  const uint8_t *ep = XT == kAct8 ? a.x.exps + j / kCkGroup : nullptr;
  const int64_t ex_ld = a.x.ld / kCkGroup;
  const float *vp = a.v + r0 + wave * 16 + row;   // wave w cuts rank tile w
  const bool cuts = wave < nr;

  f32x4 acc[Q][NR];
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int r = 0; r < NR; ++r) acc[q][r] = f32x4{0, 0, 0, 0};

  auto load_x = [&](RawQ<XT, Q> (&x)[8], int t0, int end) {
    if (whole_cols && t0 + 32 <= end) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t t = t0 + quad * 8 + i;
        x[i].load(xp + t * a.x.ld * es, XT == kAct8 ? ep + t * ex_ld : nullptr, Q);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t t = t0 + quad * 8 + i;
        if (t < end && nc > 0) x[i].load(xp + t * a.x.ld * es, XT == kAct8 ? ep + t * ex_ld : nullptr, nc);
        else x[i].clear();
      }
    }
  };
  auto load_v = [&](float (&f)[8], int t0, int end) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float *p = vp + s * a.part;
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = p[min(t0 + quad * 8 + i, end - 1) * (int64_t)a.rl];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += t0 + quad * 8 + i < end ? g[i] : 0.f;
    }
  };
  auto put_v = [&](const float (&f)[8], int buf) {
    u32x4 o[3];
    split8<3>(f, o);
#pragma unroll
    for (int p = 0; p < 3; ++p) frag[buf][wave][p][lane] = o[p];
  };
  auto stage = [&](const RawQ<XT, Q> (&x)[8], RawQ<XT, Q> (&ahead)[8], int buf) {
    int t, end;
    const bool more = steps.next(&t, &end);
    float f[8];
    if (more) {
      load_x(ahead, t, end);
      if (cuts) load_v(f, t, end);
    }
    u32x4 xf[Q][PX];
#pragma unroll
    for (int q = 0; q < Q; ++q) column_parts<XT, Q>(x, q, xf[q]);
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r < nr) {
        u32x4 vf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) vf[p] = frag[buf][r][p][lane];
#pragma unroll
        for (int q = 0; q < Q; ++q) products<PX, 3>(acc[q][r], xf[q], vf);
      }
    if (more && cuts) put_v(f, buf ^ 1);
    __syncthreads();
    return more;
  };
  RawQ<XT, Q> xa[8], xb[8];
  int t, end;
  if (steps.next(&t, &end)) {
    load_x(xa, t, end);
    if (cuts) {
      float f[8];
      load_v(f, t, end);
      put_v(f, 0);
    }
    __syncthreads();
    while (stage(xa, xb, 0) && stage(xb, xa, 1)) {
    }
  }
  // row r0 + 16 r + lane % 16, columns j0 + Q (4 quad + i) + q: 4 Q consecutive values a lane
  const bool whole = start[id + 1] - start[id] == 1;
  const int slot = start[a.b.adapters + 1 + id] + item - start[id];
  if (!whole && (uint32_t)slot >= (uint32_t)a.slots) return;   // requests that overlap, reported by check_batch
  const float gain = a.gain * ad.scale;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int k = r0 + 16 * r + row;
    if (k >= ad.rank) continue;
    float *g = whole ? a.grad + (int64_t)(ad.out_row + k) * a.d : a.partial + ((int64_t)slot * a.max_rank + k) * a.d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < Q; q += 4) {
        const int64_t c = j0 + Q * (4 * quad + i) + q;
        f32x4 s{acc[q][r][i], acc[q + 1][r][i], acc[q + 2][r][i], acc[q + 3][r][i]};
        if (whole) s *= gain;
        if (c + 4 <= a.d) *reinterpret_cast<f32x4_a4 *>(g + c) = s;
        else
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (c + u < a.d) g[c + u] = s[u];
      }
  }
}

// Both gradients of a call in one launch: the first blocks0 blocks are table A's.
template <int XA, int XB, int NR>
__global__ void __launch_bounds__(256) adapter_grad_kernel(GradArgs ga, GradArgs gb, int blocks0) {
  extern __shared__ int32_t start[];
  __shared__ u32x4 frag[2][NR][3][64];
  const int block = blockIdx.x;
  if constexpr (XA == XB) {
    grad_block<XA, NR>(block < blocks0 ? ga : gb, block < blocks0 ? block : block - blocks0, start, frag);
  } else {
    if (block < blocks0) grad_block<XA, NR>(ga, block, start, frag);
    else grad_block<XB, NR>(gb, block - blocks0, start, frag);
  }
}

// The items' partial sums of one gradient row, in item order; zero for an adapter without tokens.
__global__ void __launch_bounds__(256) adapter_grad_sum_kernel(GradArgs ga, GradArgs gb, int blocks0) {
  const GradArgs &a = (int)blockIdx.x < blocks0 ? ga : gb;
  const int id = blockIdx.y, block = (int)blockIdx.x < blocks0 ? blockIdx.x : blockIdx.x - blocks0;
  const AdapterDev ad = a.b.ads[id];
  if ((int)blockIdx.z >= ad.rank) return;
  int i0 = 0, i1 = 0;
  if (a.b.requests > 0 && a.b.tokens > 0) {
    const int2 items = a.items[id];
    if (items.y == 1) return;   // written whole
    i0 = max(items.x, 0);
    i1 = min(items.x + items.y, a.slots);
  }
  const float gain = a.gain * ad.scale;
  const int64_t c = ((int64_t)block * 256 + threadIdx.x) * 4;
  if (c >= a.d) return;
  const int n = (int)min((int64_t)4, a.d - c);
  float *g = a.grad + (int64_t)(ad.out_row + blockIdx.z) * a.d + c;
  const float *p = a.partial + (int64_t)blockIdx.z * a.d + c;
  const int64_t step = (int64_t)a.max_rank * a.d;
  f32x4 s{0, 0, 0, 0};
  if (n == 4) {
#pragma unroll 4
    for (int i = i0; i < i1; ++i) s += *reinterpret_cast<const f32x4_a4 *>(p + i * step);
    *reinterpret_cast<f32x4_a4 *>(g) = s * gain;
  } else {
    for (int i = i0; i < i1; ++i)
      for (int u = 0; u < n; ++u) s[u] += p[i * step + u];
    for (int u = 0; u < n; ++u) g[u] = s[u] * gain;
  }
}

// Tokens of one item: enough items for three blocks a CU, but 128 tokens or more for each rank
// tile, so that an item's partial sums (written and read once) stay small beside what it reads.
int adapter_grad_chunk(int64_t tokens, int64_t d, int max_rank) {
  const int tiles = max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : 4;
  const int64_t across = (d + (tiles == 1 ? 511 : 255)) / (tiles == 1 ? 512 : 256);
  const int64_t items = 768 / across < 1 ? 1 : 768 / across;
  int64_t c = ((tokens + items - 1) / items + 31) / 32 * 32;
  if (c < 128 * tiles) c = 128 * tiles;
  return (int)(c > 4096 ? 4096 : c);
}

template <int XT, int NR>
static int grad_blocks(const GradArgs &a) {
  const int cols = 64 * GradCols<XT, NR>::value;
  const int64_t items = (a.b.tokens + a.chunk - 1) / a.chunk + (a.b.requests < a.b.adapters ? a.b.requests : a.b.adapters);
  return (int)((a.d + cols - 1) / cols * items);
}

template <int XA, int XB, int NR>
static void grad_launch(const GradArgs &a, const GradArgs &b, hipStream_t st) {
  const int blocks0 = grad_blocks<XA, NR>(a);
  const dim3 g((unsigned)(blocks0 + grad_blocks<XB, NR>(b)), 1, (unsigned)(NR == 4 ? (a.max_rank + 63) / 64 : 1));
  hipLaunchKernelGGL((adapter_grad_kernel<XA, XB, NR>), g, dim3(256), sizeof(int32_t) * 2 * (a.b.adapters + 1), st, a, b,
                     blocks0);
}

template <int XA, int XB>
static void grad_nr(const GradArgs &a, const GradArgs &b, hipStream_t st) {
  if (a.max_rank <= 16) grad_launch<XA, XB, 1>(a, b, st);
  else if (a.max_rank <= 32) grad_launch<XA, XB, 2>(a, b, st);
  else grad_launch<XA, XB, 4>(a, b, st);
}

hipError_t launch_adapter_grad(const GradArgs &a, const GradArgs &b, hipStream_t st) {
  if (a.x.type == kAct8) {
    if (b.x.type == kF32) grad_nr<kAct8, kF32>(a, b, st);
    else if (b.x.type == kF16) grad_nr<kAct8, kF16>(a, b, st);
    else grad_nr<kAct8, kBF16>(a, b, st);
  } else if (a.x.type == kF32) grad_nr<kF32, kF32>(a, b, st);
  else if (a.x.type == kF16) grad_nr<kF16, kF16>(a, b, st);
  else grad_nr<kBF16, kBF16>(a, b, st);
  return hipGetLastError();
}

hipError_t launch_adapter_grad_sum(const GradArgs &a, const GradArgs &b, hipStream_t st) {
  const int64_t blocks0 = (a.d + 1023) / 1024, blocks = blocks0 + (b.d + 1023) / 1024;
  hipLaunchKernelGGL(adapter_grad_sum_kernel, dim3((unsigned)blocks, (unsigned)a.b.adapters, (unsigned)a.max_rank),
                     dim3(256), 0, st, a, b, (int)blocks0);
  return hipGetLastError();
}

}  // namespace psx
