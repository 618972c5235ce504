// psx_adapter.hip — low-rank adapters whose rank rows are rows of two tables, for a batch of
// requests: request n owns tokens [begin[n], begin[n + 1]) and one adapter (or none).
//
//   shrink   v[t][r]   = sum_k x[t][k] W[slot + r][k]            (x, table A; dy, table B)
//   expand   out[t][j] = base[t][j] + s sum_r v[t][r] W[slot + r][j]
//   grad     g[r][j]   = gain s sum_t v[t][r] x[t][j]            (partial sums, then their sum)
//
// Arithmetic.  The tables are f32 and a server adds increments far below a bf16 step to them,
// so an f32 operand is cut into bf16 parts, each the nearest to what is left: 2^-8 of the value at
// most behind one part, 2^-17 behind two, and nothing behind three (8 + 9 + 7 bits), as every
// remainder is exact.  A product of parts is exact in f32, and v_mfma_f32_16x16x32_bf16 adds in
// f32.  Three parts a factor: the six products (i, j) with i + j <= 2 leave out 2^-24 of a product
// (times 1 + 2^-10) at most, either sign.  A bf16 activation is one part, binary16 two, f32 three, an
// 8-bit checkpoint (7 significant bits and a power of two) one.  16-bit outputs are rounded once;
// expand takes two parts a factor for them, three products, which leave out 2^-15 of a product at
// most and 2^-17.8 in the root mean square, either sign, where half a step of the output is 2^-9
// to 2^-8 (bf16) or 2^-12 to 2^-11 of it (three parts: 16384 tokens x 4096 bf16, rank 16, 94 -> 98 us
// a forward call; rank 64 from a checkpoint, whose registers they overfill, 300 -> 441 us backward).
// A factor that is not finite makes the sums that it enters NaN or Inf.
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
typedef uint32_t u32_a1 __attribute__((aligned(1)));
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

// Addresses are a base that the wave shares plus a lane's 32-bit offset (rows lie at most 64 MiB
// apart): the base moves in scalar registers and the loads take both.
__device__ __forceinline__ const uint8_t *at(const uint8_t *base, uint32_t lane_offset) { return base + lane_offset; }

// Two values rounded to nearest, packed.
template <int YT> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (YT == PSX_ACT_F16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)lo, (__bf16)hi});
  }
}

// A value whose nearest bf16 is finite: past the largest bf16 the next part takes what is left, and
// an Inf or a NaN comes out of that difference.
__device__ __forceinline__ float in_bf16(float f) {
  constexpr float most = 0x1.fep127f;
  return __builtin_amdgcn_fmed3f(f, -most, most);
}
// A pair of values as P bf16 parts, each the nearest to what the parts before it left.  Wide: any
// f32 values; the others (binary16, one part) have no first part past the largest bf16.
template <int P, bool Wide>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&o)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    o[p] = Wide && p == 0 ? pack2<PSX_ACT_BF16>(in_bf16(a), in_bf16(b)) : pack2<PSX_ACT_BF16>(a, b);
    if (p + 1 < P) {
      // byte permutations: of a shift and a mask the compiler makes a second conversion each
      a -= as_f(__builtin_amdgcn_perm(o[p], 0u, 0x05040c0cu));
      b -= as_f(__builtin_amdgcn_perm(o[p], 0u, 0x07060c0cu));
    }
  }
}

// Eight values as P bf16 fragments.
template <bool Wide, int P>
__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&o)[P]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    uint32_t w[P];
    split2<P, Wide>(v[2 * d], v[2 * d + 1], w);
#pragma unroll
    for (int p = 0; p < P; ++p) o[p][d] = w[p];
  }
}

// The smallest products first: the first part of a value may lie past it, and the parts behind it
// bring it back.
template <int PA, int PB>
__device__ __forceinline__ void products(f32x4 &acc, const u32x4 (&a)[PA], const u32x4 (&b)[PB]) {
  constexpr int deep = PA > PB ? PA : PB;
#pragma unroll
  for (int order = deep - 1; order >= 0; --order)
#pragma unroll
    for (int i = 0; i < PA; ++i)
#pragma unroll
      for (int j = 0; j < PB; ++j)
        if (i + j == order)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[j]),
                                                        acc, 0, 0, 0);
}

// 2^e of a checkpoint's exponent byte e + 127; 255 marks a group that held an Inf or a NaN.
__device__ __forceinline__ float ck_scale(uint32_t e) { return as_f(e == 255 ? 0x7fc00000u : e << 23); }

// Loads of the next step stay in front of this step's products: the compiler would sink them
// behind, and wait for them at once.
__device__ __forceinline__ void issue_first() { __builtin_amdgcn_sched_barrier(0); }

// ---- the batch ------------------------------------------------------------------------------

__device__ __forceinline__ int begin_of(const BatchView &b, int n) { return min(max(b.begin[n], 0), b.tokens); }

__device__ __forceinline__ int adapter_of(const BatchView &b, int n) {
  const int a = b.which[n];
  return a >= 0 && a < b.adapters ? a : -1;
}

// Work item `item` of tiles of M tokens: tile c of request n has the number c + n, which rises
// strictly along the requests, so that ceil(tokens / M) + requests numbers hold every
// (tile, request) that meet.  Every lane of the wave calls it.  False: nothing to do.  Up to 64
// requests take one round of loads.
struct Item {
  int id, t0, t1;   // adapter (-1: none), tokens
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
  const int j = min(lo + lane, b.requests - 1);
  const int b0 = begin_of(b, j), b1 = begin_of(b, j + 1), id = adapter_of(b, j);
  const int c = __builtin_popcountll(__ballot(lo + lane < hi && b0 / M + j <= item));
  if (c == 0) return false;
  const int64_t tile = (int64_t)(item - (lo + c - 1)) * M;
  const int64_t t0 = max((int64_t)__builtin_amdgcn_readlane(b0, c - 1), tile);
  const int64_t t1 = min((int64_t)__builtin_amdgcn_readlane(b1, c - 1), tile + M);
  if (t0 >= t1) return false;
  *out = {__builtin_amdgcn_readlane(id, c - 1), (int)t0, (int)t1};
  return true;
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

// A tile of 16 rows x 32 k, 16 bytes of it a lane and load.  Memory wants adjacent lanes in one
// row (a load whose lanes are 16 rows apart takes the address unit four times as long), the
// product wants lane l to hold row l % 16: the tile turns in LDS, which belongs to the wave
// alone.  16-byte places are exchanged within a row so that no two lanes of a quarter wave meet
// in a bank, neither writing nor reading.
template <int XT> struct Tile {
  static constexpr int es = ActInfo<XT>::size, loads = es / 2, bytes = 512 * es;   // 1 or 2 loads
  static constexpr int vals = 16 / es;   // values a lane and load
  u32x4 d[loads];
  static __device__ __forceinline__ int row(int lane, int i) { return loads == 1 ? lane >> 2 : i * 8 + (lane >> 3); }
  static __device__ __forceinline__ int piece(int lane) { return loads == 1 ? lane & 3 : lane & 7; }
  static __device__ __forceinline__ int place(int row, int piece) {
    return loads == 1 ? row * 4 + (piece ^ (row >> 2 & 3)) : row * 8 + (piece ^ (row >> 1 & 7));
  }
  __device__ __forceinline__ void load(int i, const uint8_t *p) { d[i] = *reinterpret_cast<const u32x4_a1 *>(p); }
  // the first n values, zeros behind them
  __device__ __forceinline__ void load_tail(int i, const uint8_t *p, int n) {
    d[i] = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < vals; ++k)
      if (k < n) {
        if constexpr (XT == kF32) d[i][k] = reinterpret_cast<const uint32_t *>(p)[k];
        else d[i][k / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[k] << (k % 2 * 16);
      }
  }
  __device__ __forceinline__ void put(u32x4 *lds, int lane) const {
#pragma unroll
    for (int i = 0; i < loads; ++i) lds[place(row(lane, i), piece(lane))] = d[i];
  }
  // row lane % 16, k (lane / 16) * 8 .. + 8
  static __device__ __forceinline__ void get(const u32x4 *lds, int lane, u32x4 (&o)[loads]) {
#pragma unroll
    for (int i = 0; i < loads; ++i) o[i] = lds[place(lane & 15, (lane >> 4) * loads + i)];
  }
  static __device__ __forceinline__ void parts(const u32x4 *lds, int lane, u32x4 (&o)[ActInfo<XT>::parts]) {
    u32x4 w[loads];
    get(lds, lane, w);
    if constexpr (XT == kBF16) {
      o[0] = w[0];
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (XT == kF32) f[i] = as_f(w[i / 4][i % 4]);
        else f[i] = half_at(w[0][i / 2], i % 2);
      }
      split8<XT == kF32>(f, o);
    }
  }
};

// Waves of a block: more for items of few tokens, whose blocks hold less each (4 and 8 waves: 22.1
// and 18.1 us for 4096 tokens x 4096 bf16, rank 32; 32.3 and 41.6 us for 16384 tokens, rank 16).
template <int MT> struct ShrinkWaves { static constexpr int value = MT <= 2 ? 8 : 4; };
// Tiles of k that a step holds: two where the registers and the LDS allow it (16384 x 4096 bf16,
// rank 16: 33.9 -> 32.3 us).
template <int XT, int MT, int NR> struct ShrinkHalves {
  static constexpr int value = NR == 1 && XT != kF32 ? 2 : 1;
};
template <int XT, int MT, int NR> struct ShrinkLds {   // 16-byte places of one wave
  static constexpr int step = ShrinkHalves<XT, MT, NR>::value * (MT * Tile<XT>::bytes + NR * Tile<kF32>::bytes) / 16;
  static constexpr int value = step > MT * NR * 64 ? step : MT * NR * 64;   // the sums of the waves, too
};

template <int XT, int MT, int NR, int WV>
__device__ __forceinline__ void shrink_block(const ShrinkArgs &a, const Item &it, const AdapterDev &ad, int r0, int lane,
                                             int wave, int per_wave, u32x4 *lds) {
  constexpr int PX = ActInfo<XT>::parts, es = ActInfo<XT>::size, H = ShrinkHalves<XT, MT, NR>::value, K = 32 * H;
  typedef Tile<XT> TX;
  typedef Tile<kF32> TW;
  u32x4 *xl = lds + wave * per_wave, *wl = xl + H * MT * (TX::bytes / 16);
  // tokens and rows past the last are read as the last again; what they give is not used
  const uint8_t *xb = a.x.p + it.t0 * a.x.ld * es;
  const uint8_t *wb = reinterpret_cast<const uint8_t *>(a.w + (int64_t)((a.use_b ? ad.slot_b : ad.slot_a) + r0) * a.d);
  uint32_t xo[MT][TX::loads], wo[NR][TW::loads];
  const int kx = TX::piece(lane) * TX::vals, kw = TW::piece(lane) * TW::vals;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < TX::loads; ++i)
      xo[m][i] = ((uint32_t)min(m * 16 + TX::row(lane, i), it.t1 - it.t0 - 1) * (uint32_t)a.x.ld + kx) * es;
#pragma unroll
  for (int j = 0; j < NR; ++j)
#pragma unroll
    for (int i = 0; i < TW::loads; ++i)
      wo[j][i] = ((uint32_t)min(j * 16 + TW::row(lane, i), ad.rank - r0 - 1) * (uint32_t)a.d + kw) * 4;
  f32x4 acc[MT][NR];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NR; ++j) acc[m][j] = f32x4{0, 0, 0, 0};

  TX x[H][MT];
  TW w[H][NR];
  auto load = [&](int c) {
    const int64_t k = (int64_t)c * K;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < TX::loads; ++i) x[h][m].load(i, at(xb + (k + 32 * h) * es, xo[m][i]));
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int i = 0; i < TW::loads; ++i) w[h][j].load(i, at(wb + (k + 32 * h) * 4, wo[j][i]));
    }
  };
  // the step in registers goes to LDS, the next one's loads go out, then the products
  auto multiply = [&](int next, bool more) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int m = 0; m < MT; ++m) x[h][m].put(xl + (h * MT + m) * (TX::bytes / 16), lane);
#pragma unroll
      for (int j = 0; j < NR; ++j) w[h][j].put(wl + (h * NR + j) * (TW::bytes / 16), lane);
    }
    if (more) load(next);
    issue_first();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int h = 0; h < H; ++h) {
      u32x4 xf[MT][PX];
#pragma unroll
      for (int m = 0; m < MT; ++m) TX::parts(xl + (h * MT + m) * (TX::bytes / 16), lane, xf[m]);
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        u32x4 wf[3];
        TW::parts(wl + (h * NR + j) * (TW::bytes / 16), lane, wf);
#pragma unroll
        for (int m = 0; m < MT; ++m) products<3, PX>(acc[m][j], wf, xf[m]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  const int chunks = (int)((a.d + K - 1) / K), full = (int)(a.d / K);
  const int per = (chunks + a.splits - 1) / a.splits;
  const int c0 = blockIdx.y * per, c1 = min(full, c0 + per);
  int c = c0 + wave;
  if (c < c1) {
    load(c);
    for (; c + WV < c1; c += WV) multiply(c + WV, true);
    multiply(0, false);
  }
  if (full < chunks && full >= c0 && full < c0 + per && (full - c0) % WV == wave) {   // the last, short step
    const int64_t k = (int64_t)full * K;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int nx = (int)min((int64_t)TX::vals, max((int64_t)0, a.d - k - 32 * h - kx));
      const int nw = (int)min((int64_t)TW::vals, max((int64_t)0, a.d - k - 32 * h - kw));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < TX::loads; ++i) x[h][m].load_tail(i, at(xb + (k + 32 * h) * es, xo[m][i]), nx);
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int i = 0; i < TW::loads; ++i) w[h][j].load_tail(i, at(wb + (k + 32 * h) * 4, wo[j][i]), nw);
    }
    multiply(0, false);
  }

  // wave w adds wave w + half's sums; the LDS is now the block's
  f32x4 *red = reinterpret_cast<f32x4 *>(lds);
  __syncthreads();
#pragma unroll
  for (int half = WV / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NR; ++j) red[((wave - half) * MT * NR + m * NR + j) * 64 + lane] = acc[m][j];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[m][j] += red[(wave * MT * NR + m * NR + j) * 64 + lane];
    }
    __syncthreads();
  }
  if (wave) return;
  float *v = a.v + blockIdx.y * a.part;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = it.t0 + m * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < NR; ++j)   // a row of v ends at the last rank tile of the set's largest rank
      if (t < it.t1 && r0 + j * 16 < ad.rank)
        *reinterpret_cast<f32x4 *>(v + t * a.rl + r0 + j * 16 + (lane >> 4) * 4) = acc[m][j];
  }
}

// One block: one item (up to 16 MT tokens of one request) and one part of k.  Its waves take
// steps of k in turn, each loading the next step before it multiplies, and add their sums in
// LDS.  Every token value is read once, and by one wave; a rank row's is cut into parts once for
// the block's tokens.  Items of few tokens or few ranks take the narrower code.  Bound by x's
// bytes for few ranks (16384 x 4096 bf16, rank 16: 32 us, 4.1 TB/s); past 32 ranks by the chain from
// load over LDS to product, with two waves a SIMD to hide it (16384 x 8192, rank 64: 95 us, 2.8
// TB/s; out of idle 102, there without x's loads 86, with a third of the products 90).
template <int XT, int MT, int NR>
__global__ void __launch_bounds__(64 * ShrinkWaves<MT>::value, 2) adapter_shrink_kernel(ShrinkArgs a) {
  constexpr int WV = ShrinkWaves<MT>::value;
  constexpr int n0 = ShrinkLds<XT, MT, NR>::value, n1 = ShrinkLds<XT, MT, (NR > 2 ? 2 : NR)>::value;
  constexpr int n2 = ShrinkLds<XT, MT, 1>::value, n3 = ShrinkLds<XT, 1, NR>::value;
  constexpr int n01 = n0 > n1 ? n0 : n1, n23 = n2 > n3 ? n2 : n3, per_wave = n01 > n23 ? n01 : n23;
  __shared__ u32x4 lds[WV * per_wave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_batch(a.b);
  Item it;
  if (!find_item(a.b, 16 * MT, blockIdx.x, lane, &it)) return;
  if (it.id < 0) return;
  const AdapterDev ad = a.b.ads[it.id];
  const int r0 = blockIdx.z * 16 * NR;
  if (r0 >= ad.rank) return;
  if (MT > 1 && it.t1 - it.t0 <= 16) {
    if (NR > 1 && ad.rank - r0 <= 16) shrink_block<XT, 1, 1, WV>(a, it, ad, r0, lane, wave, per_wave, lds);
    else shrink_block<XT, 1, NR, WV>(a, it, ad, r0, lane, wave, per_wave, lds);
  } else {
    if (NR > 1 && ad.rank - r0 <= 16) shrink_block<XT, MT, 1, WV>(a, it, ad, r0, lane, wave, per_wave, lds);
    else if (NR > 2 && ad.rank - r0 <= 32) shrink_block<XT, MT, 2, WV>(a, it, ad, r0, lane, wave, per_wave, lds);
    else shrink_block<XT, MT, NR, WV>(a, it, ad, r0, lane, wave, per_wave, lds);
  }
}

// Tokens a shrink block takes: enough blocks for the chip first (16 tokens; decode steps, where
// each request has one, need no more), then more tokens for each rank row read.  4096 tokens x
// 4096 bf16, rank 32: 16, 32, 64 tokens 23.5, 18.1, 24.4 us; 16384 x 4096, rank 16: 32, 64 tokens
// 36.7, 32.3 us; 16384 x 8192, rank 64: 155, 102 us; 1531 x 2047 binary16, ranks to 64: 16, 32
// tokens 17.4, 20.5 us.
static int adapter_tile(int64_t tokens) { return tokens <= kFewTokens ? 16 : tokens <= 8192 ? 32 : 64; }
// Parts that k is cut into: for a few tokens, so that they still fill the chip (expand adds the
// parts, and leaves their sum behind them for the gradients: 1531 x 2047, ranks to 64, shrink and
// expand together 43.3 -> 40.8 us; 200 x 4096 bf16, rank 16, 14.2 -> 11.6 us); for a long batch,
// whose blocks are few more than the chip's places, so that the last ones do not take a second
// round alone (adapter_join adds them into the first: 16384 x 4096, rank 16, 41.7 -> 32.3 + 4.8 us;
// 16384 x 8192, rank 64, 138 -> 102 + 6 us).  Between them they are one, as
// a join costs about what the parts save where this was tuned (4096 x 4096, rank 32: 15.9 us, against
// 15.6 + 4.5).  It is not the best everywhere: the blocks there are fewer than the chip's places, so
// a block's walk over the width sets the time, whatever the tokens (2048, 2049, 4096, 8192 tokens x 4096:
// 10.6, 15.6, 15.9, 18.1 us for rank 32; x 8192: 13.9, 27.0, 27.5, 34.2, for rank 64 22.9, 48.3, 47.1, 52.8).
int adapter_splits(int64_t tokens, int64_t d) {
  if (tokens > kFewTokens && tokens <= 8192) return 1;
  const int64_t s = (d + 511) / 512;
  return (int)(s < 1 ? 1 : s > kMostParts ? kMostParts : s);
}
bool adapter_joins(int64_t tokens, int64_t d) { return tokens > kFewTokens && adapter_splits(tokens, d) > 1; }

// v's parts added to the first, in order.
__global__ void __launch_bounds__(256) adapter_join_kernel(float *v, int64_t part, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;   // a part is whole rows of 16 values
  if (i >= part) return;
  f32x4 s = *reinterpret_cast<const f32x4 *>(v + i);
  f32x4 g[kMostParts - 1];
#pragma unroll
  for (int k = 1; k < kMostParts; ++k)
    if (k < splits) g[k - 1] = *reinterpret_cast<const f32x4 *>(v + k * part + i);
#pragma unroll
  for (int k = 1; k < kMostParts; ++k)
    if (k < splits) s += g[k - 1];
  *reinterpret_cast<f32x4 *>(v + i) = s;
}

hipError_t launch_adapter_join(const ShrinkArgs &a, hipStream_t st) {
  hipLaunchKernelGGL(adapter_join_kernel, dim3((unsigned)((a.part / 4 + 255) / 256)), dim3(256), 0, st, a.v, a.part,
                     a.splits);
  return hipGetLastError();
}

template <int XT, int MT>
static void shrink_nr(const ShrinkArgs &a, hipStream_t st) {
  dim3 g((unsigned)(((int64_t)a.b.tokens + 16 * MT - 1) / (16 * MT) + a.b.requests), (unsigned)a.splits, 1);
  const dim3 b(64 * ShrinkWaves<MT>::value);
  if (a.max_rank <= 16) hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 1>), g, b, 0, st, a);
  else if (a.max_rank <= 32) hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 2>), g, b, 0, st, a);
  else {
    g.z = (a.max_rank + 63) / 64;
    hipLaunchKernelGGL((adapter_shrink_kernel<XT, MT, 4>), g, b, 0, st, a);
  }
}

template <int XT>
static void shrink_mt(const ShrinkArgs &a, hipStream_t st) {
  const int M = adapter_tile(a.b.tokens);
  if (M == 16) shrink_nr<XT, 1>(a, st);
  else if (M == 32) shrink_nr<XT, 2>(a, st);
  else shrink_nr<XT, 4>(a, st);
}

hipError_t launch_adapter_shrink(const ShrinkArgs &a, hipStream_t st) {
  if (a.x.type == kF32) shrink_mt<kF32>(a, st);
  else if (a.x.type == kF16) shrink_mt<kF16>(a, st);
  else shrink_mt<kBF16>(a, st);
  if (adapter_joins(a.b.tokens, a.d)) return launch_adapter_join(a, st);
  return hipGetLastError();
}

// ---- expand -------------------------------------------------------------------------------------

// Q consecutive values of a row, n of them real, as they lie in memory.
template <int YT, int Q> struct RawOut {
  static constexpr int words = ActInfo<YT>::size * Q / 4;
  uint32_t d[words];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < words; ++i) d[i] = 0;
  }
  // `once`: past the caches' keeping
  __device__ __forceinline__ void load(const uint8_t *p, int n, bool once) {
    if (n >= Q) {
      if constexpr (words == 2) {
        const u32x2_a1 *u = reinterpret_cast<const u32x2_a1 *>(p);
        const u32x2 v = once ? __builtin_nontemporal_load(u) : *u;
        d[0] = v[0];
        d[1] = v[1];
      } else {
        const u32x4_a1 *u = reinterpret_cast<const u32x4_a1 *>(p);
        const u32x4 v = once ? __builtin_nontemporal_load(u) : *u;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = v[i];
      }
    } else {
      clear();
#pragma unroll
      for (int i = 0; i < Q; ++i)
        if (i < n) {
          if constexpr (YT == kF32) d[i] = reinterpret_cast<const uint32_t *>(p)[i];
          else d[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (i % 2 * 16);
        }
    }
  }
  __device__ __forceinline__ void store(uint8_t *p, int n) const {
    if (n >= Q) {
      // past the caches' keeping: written lines that stay would be written back under the next
      // kernel's reads (16384 tokens x 4096: 109 -> 103 us for shrink and expand together)
      if constexpr (words == 2) __builtin_nontemporal_store(u32x2{d[0], d[1]}, reinterpret_cast<u32x2_a1 *>(p));
      else __builtin_nontemporal_store(u32x4{d[0], d[1], d[2], d[3]}, reinterpret_cast<u32x4_a1 *>(p));
    } else {
#pragma unroll
      for (int i = 0; i < Q; ++i)
        if (i < n) {
          if constexpr (YT == kF32) reinterpret_cast<uint32_t *>(p)[i] = d[i];
          else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(d[i / 2] >> (i % 2 * 16));
        }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (YT == kF32) return as_f(d[i]);
    if constexpr (YT == kF16) return half_at(d[i / 2], i % 2);
    return as_f(i % 2 ? d[i / 2] & 0xffff0000u : d[i / 2] << 16);
  }
  __device__ __forceinline__ void set2(int i, float lo, float hi) {   // i even
    if constexpr (YT == kF32) {
      d[i] = as_u(lo);
      d[i + 1] = as_u(hi);
    } else {
      d[i / 2] = pack2<YT>(lo, hi);
    }
  }
};

template <int YT, int KS> struct ExpandCols { static constexpr int value = YT == kF32 || KS > 1 ? 4 : 8; };

// 16-byte places of a token's ranks in LDS: an odd number, so that 16 rows meet no bank twice.
__host__ __device__ inline int expand_pitch(int max_rank) { return (max_rank + 31) / 32 * 4 + 1; }

// One block: one item and 64 Q columns, 16 Q a wave.  Columns are the product's second operand,
// column Q n + q in product q: a lane loads Q columns of a rank row at once, and holds Q
// consecutive outputs of four tokens, so that 16 lanes read and write a row through.  The item's
// rows of v lie in LDS (their parts of k added, zeros behind the adapter's rank); up to 32 KS
// ranks the rank rows stay in registers.  The next 16 tokens' base is loaded before these are
// multiplied.  Bound by base and out (16384 x 4096 bf16, rank 16: 60 us, 4.5 TB/s) and by what a wave
// has in flight: more than 32 ranks are held to the registers
// of three waves a SIMD (16384 tokens x 4096 of 16 bits, rank 64: 94 -> 77 us; the narrower code
// would spill there, 60 -> 104 us).
template <int YT, int KS>
__global__ void __launch_bounds__(256, KS > 1 && YT != kF32 ? 3 : 1) adapter_expand_kernel(ExpandArgs a) {
  constexpr int P = YT == kF32 ? 3 : 2, es = ActInfo<YT>::size, Q = ExpandCols<YT, KS>::value;
  extern __shared__ u32x4 vl[];   // [P][tokens of the tile][pitch]: v's parts
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int across = (int)((a.d + 64 * Q - 1) / (64 * Q));
  Item it;
  if (!find_item(a.b, a.tile, blockIdx.x / across, lane, &it)) return;
  const int row = lane & 15, quad = lane >> 4;
  const int64_t j0 = ((int64_t)(blockIdx.x % across) * 4 + wave) * 16 * Q, c0 = j0 + Q * row;
  const int nc = (int)min((int64_t)Q, max((int64_t)0, a.d - c0));
  AdapterDev ad{};
  if (it.id >= 0) ad = a.b.ads[it.id];
  else if (a.base == a.out) return;
  const float *w = a.w + (int64_t)(a.use_b ? ad.slot_b : ad.slot_a) * a.d;
  const int ranks = (ad.rank + 31) / 32 * 32, pitch = expand_pitch(a.max_rank), plane = a.tile * pitch;

  u32x4 wf[KS][Q][P];
  auto load_rows = [&](int g0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8][Q];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = g0 + s * 32 + quad * 8 + i;
        const float *p = w + (int64_t)r * a.d + c0;
#pragma unroll
        for (int q = 0; q < Q; ++q) x[i][q] = 0.f;
        if (r < ad.rank) {
          if (nc == Q) {
#pragma unroll
            for (int q = 0; q < Q; q += 4) {
              const f32x4 y = *reinterpret_cast<const f32x4_a4 *>(p + q);
#pragma unroll
              for (int u = 0; u < 4; ++u) x[i][q + u] = y[u];
            }
          } else {
#pragma unroll
            for (int q = 0; q < Q; ++q)
              if (q < nc) x[i][q] = p[q];
          }
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = x[i][q];
        split8<true>(f, wf[s][q]);
      }
    }
  };
  typedef RawOut<YT, Q> Raw;
  Raw base[4];
  // rows that start in the middle of a line share it with their neighbours' blocks: those are kept
  const bool once = a.base_ld * es % 128 == 0 && (uintptr_t)a.base % 128 == 0;
  const bool whole = j0 + 16 * Q <= a.d;
  const int64_t b_ld = a.base_ld * es, o_ld = a.out_ld * es;
  const uint32_t b_off = quad * 4 * (uint32_t)b_ld + (uint32_t)c0 * es, o_off = quad * 4 * (uint32_t)o_ld + (uint32_t)c0 * es;
  auto load_base = [&](int tt) {
    if (!a.base) {
#pragma unroll
      for (int i = 0; i < 4; ++i) base[i].clear();
    } else if (whole && tt + 16 <= it.t1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) base[i].load(at(a.base + (tt + i) * b_ld, b_off), Q, once);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tt + quad * 4 + i < it.t1) base[i].load(at(a.base + (tt + i) * b_ld, b_off), nc, once);
        else base[i].clear();
      }
    }
  };
  const bool resident = ad.rank <= 32 * KS, first_cols = blockIdx.x % across == 0;
  load_base(it.t0);
  // v's rows cut into parts, four values a thread and step
  const int pieces = ranks / 4, n = (it.t1 - it.t0) * pieces;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int t = i / pieces, r = i % pieces * 4;
    f32x4 s{0, 0, 0, 0};
    if (r < a.rl) {
      const float *p = a.v + (it.t0 + t) * (int64_t)a.rl + r;
      s = *reinterpret_cast<const f32x4 *>(p);
      for (int k = 1; k < a.splits; ++k) s += *reinterpret_cast<const f32x4 *>(p + k * a.part);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (r + u >= ad.rank) s[u] = 0.f;
    if (a.sum && first_cols && r < a.rl) *reinterpret_cast<f32x4 *>(a.sum + (it.t0 + t) * (int64_t)a.rl + r) = s;
    uint32_t lo[P], hi[P];
    split2<P, true>(s[0], s[1], lo);
    split2<P, true>(s[2], s[3], hi);
#pragma unroll
    for (int p = 0; p < P; ++p) reinterpret_cast<u32x2 *>(vl + p * plane + t * pitch)[r / 4] = u32x2{lo[p], hi[p]};
  }
  if (resident) load_rows(0);
  __syncthreads();
  for (int tt = it.t0; tt < it.t1; tt += 16) {
    Raw now[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i] = base[i];
    if (tt + 16 < it.t1) load_base(tt + 16);
    issue_first();
    f32x4 acc[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) acc[q] = f32x4{0, 0, 0, 0};
    for (int g0 = 0; g0 < ad.rank; g0 += 32 * KS) {
      if (!resident) load_rows(g0);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (g0 + s * 32 < ad.rank) {
          u32x4 vf[P];
#pragma unroll
          for (int p = 0; p < P; ++p) vf[p] = vl[p * plane + (tt - it.t0 + row) * pitch + (g0 + s * 32) / 8 + quad];
#pragma unroll
          for (int q = 0; q < Q; ++q) products<P, P>(acc[q], vf, wf[s][q]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < Q; q += 2)
        now[i].set2(q, __builtin_fmaf(ad.scale, acc[q][i], now[i].get(q)),
                    __builtin_fmaf(ad.scale, acc[q + 1][i], now[i].get(q + 1)));
    if (whole && tt + 16 <= it.t1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) now[i].store(a.out + (tt + i) * o_ld + o_off, Q);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tt + quad * 4 + i < it.t1) now[i].store(a.out + (tt + i) * o_ld + o_off, nc);
    }
  }
}

static int expand_row_bytes(int max_rank, int parts) { return expand_pitch(max_rank) * 16 * parts; }

// Tokens an expand block takes: rank rows loaded once serve more of them in longer batches, as
// long as v's rows leave the LDS room for four blocks a CU.  16384 tokens, rank 64: 64 of them 106
// us, 128 94; 1531 tokens, ranks to 64: 32 of them 26 us, 64 28.
int adapter_expand_tile(int64_t tokens, int max_rank, int parts) {
  int tile = tokens <= 256 ? 16 : tokens <= 2048 ? 32 : tokens <= 8192 ? 64 : 128;
  while (tile > 16 && tile * expand_row_bytes(max_rank, parts) > 40 * 1024) tile /= 2;
  return tile;
}

template <int YT, int KS>
static void expand_launch(const ExpandArgs &in, hipStream_t st) {
  constexpr int cols = 64 * ExpandCols<YT, KS>::value, P = YT == kF32 ? 3 : 2;
  ExpandArgs a = in;
  a.tile = adapter_expand_tile(a.b.tokens, a.max_rank, P);
  // columns fastest: blocks that run together read rows through
  const dim3 g((unsigned)((((int64_t)a.b.tokens + a.tile - 1) / a.tile + a.b.requests) * ((a.d + cols - 1) / cols)), 1, 1);
  hipLaunchKernelGGL((adapter_expand_kernel<YT, KS>), g, dim3(256), (size_t)a.tile * expand_row_bytes(a.max_rank, P), st, a);
}

template <int YT>
static void expand_ks(const ExpandArgs &a, hipStream_t st) {
  if (a.max_rank <= 32) expand_launch<YT, 1>(a, st);
  else expand_launch<YT, 2>(a, st);
}

hipError_t launch_adapter_expand(const ExpandArgs &a, hipStream_t st) {
  if (a.type == kF32) expand_ks<kF32>(a, st);
  else if (a.type == kF16) expand_ks<kF16>(a, st);
  else expand_ks<kBF16>(a, st);
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
      if constexpr (words == 1) {
        d[0] = *reinterpret_cast<const u32_a1 *>(p);
      } else if constexpr (words == 2) {
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
    split8<XT == kF32>(f, o);
  }
}

// Items of one gradient: adapter i's tokens, all its requests one after another, in chunks;
// start[i] = the first item of adapter i.  The items of an adapter that has two or more leave
// partial sums in slots from start[adapters + 1 + i] on.  Computed by every block (LDS counts
// are whole numbers: their order does not matter).  Where all tokens fit a chunk (`whole`), item i
// is adapter i, with tokens or without, and adapter_grad_sum does not run (77 tokens, 513 and 1025
// wide, f32: 11.6 + 3.1 -> 10.1 us).
__device__ __forceinline__ void grad_items(const GradArgs &a, int32_t *start) {
  const BatchView &b = a.b;
  int32_t *slot = start + b.adapters + 1;
  if (a.whole) {
    for (int i = threadIdx.x; i <= b.adapters; i += blockDim.x) {
      start[i] = i;
      slot[i] = 0;
    }
    __syncthreads();
    return;
  }
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
      int s = i < b.adapters ? (int)(((int64_t)start[i + 1] + a.chunk - 1) / a.chunk) : 0, s2 = s > 1 ? s : 0;
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

// Columns a lane takes: 8 to 16 bytes of a row, of a checkpoint 8, or 4 where the sums of more ranks
// fill the registers (16384 x 4096 from a checkpoint, rank 32: 8 columns 71.8 us, 4 76.5 us).
template <int XT, int NR> struct GradCols { static constexpr int value = XT == kAct8 && NR < 4 ? 8 : 4; };

// One block: 64 Q columns (its four waves side by side) and one item.  A step is 32 tokens: a
// wave loads Q columns of 8 tokens a lane (the next step's before this step's products), turns
// them into fragments in registers, and takes v's fragments from LDS, where one wave a rank
// tile has cut them into parts.  Both sums over tokens are f32 in the matrix unit.  Bound by the
// wait for a step's rows: four waves that meet at every step, three blocks a CU (4096 x 4096 and
// 4096 bf16, rank 32: 25 us, 2.7 TB/s; 16384 x 4096 from a checkpoint and 8192, rank 64: 116 us,
// 2.9 TB/s, of the products' 59; out of idle 136).
template <int XT, int NR>
__device__ __forceinline__ void grad_block(const GradArgs &a, int block, int32_t *start, u32x4 (*frag)[NR][3][64]) {
  constexpr int PX = ActInfo<XT>::parts, es = ActInfo<XT>::size, Q = GradCols<XT, NR>::value;
  grad_items(a, start);
  if (block == 0 && blockIdx.z == 0)
    for (int i = threadIdx.x; i < a.b.adapters; i += blockDim.x)
      a.items[i] = int2{start[a.b.adapters + 1 + i], start[i + 1] - start[i]};
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  // a lane's first row of a step: its offset from the step's first token
  const int64_t x_ld = a.x.ld * es, e_ld = a.x.ld / kCkGroup, v_ld = a.rl * 4;
  const uint32_t x_off = quad * 8 * (uint32_t)x_ld + (uint32_t)j * es, e_off = quad * 8 * (uint32_t)e_ld + (uint32_t)(j / kCkGroup);
  const uint32_t v_off = quad * 8 * (uint32_t)v_ld + (r0 + wave * 16 + row) * 4;   // wave w cuts rank tile w
  const bool cuts = wave < nr;

  f32x4 acc[Q][NR];
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int r = 0; r < NR; ++r) acc[q][r] = f32x4{0, 0, 0, 0};

  auto load_x = [&](RawQ<XT, Q> (&x)[8], int t0, int end) {
    const uint8_t *p = a.x.p + t0 * x_ld, *e = XT == kAct8 ? a.x.exps + t0 * e_ld : nullptr;
    if (whole_cols && t0 + 32 <= end) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i].load(at(p + i * x_ld, x_off), XT == kAct8 ? at(e + i * e_ld, e_off) : nullptr, Q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (t0 + quad * 8 + i < end && nc > 0)
          x[i].load(at(p + i * x_ld, x_off), XT == kAct8 ? at(e + i * e_ld, e_off) : nullptr, nc);
        else x[i].clear();
      }
    }
  };
  auto load_v = [&](float (&f)[8], int t0, int end) {
    const uint8_t *p = reinterpret_cast<const uint8_t *>(a.v) + t0 * v_ld;
    if (t0 + 32 <= end) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float *>(at(p + i * v_ld, v_off));
    } else {   // a token behind the request's last counts as nothing, whatever v holds there
#pragma unroll
      for (int i = 0; i < 8; ++i)
        f[i] = t0 + quad * 8 + i < end ? *reinterpret_cast<const float *>(at(p + i * v_ld, v_off)) : 0.f;
    }
  };
  auto put_v = [&](const float (&f)[8], int buf) {
    u32x4 o[3];
    split8<true>(f, o);
#pragma unroll
    for (int p = 0; p < 3; ++p) frag[buf][wave][p][lane] = o[p];
  };
  RawQ<XT, Q> x[8];
  float f[8];
  u32x4 xf[Q][PX];
  auto multiply = [&](int buf) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r < nr) {
        u32x4 vf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) vf[p] = frag[buf][r][p][lane];
#pragma unroll
        for (int q = 0; q < Q; ++q) products<PX, 3>(acc[q][r], xf[q], vf);
      }
  };
  int t, end;
  if (steps.next(&t, &end)) {
    load_x(x, t, end);
    if (cuts) {
      load_v(f, t, end);
      put_v(f, 0);
    }
    __syncthreads();
    int buf = 0;
    for (;;) {
      const bool more = steps.next(&t, &end);
#pragma unroll
      for (int q = 0; q < Q; ++q) column_parts<XT, Q>(x, q, xf[q]);
      if (!more) break;
      load_x(x, t, end);
      if (cuts) load_v(f, t, end);
      issue_first();
      multiply(buf);
      buf ^= 1;
      if (cuts) put_v(f, buf);
      __syncthreads();
    }
    multiply(buf);
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
__global__ void __launch_bounds__(256, 2) adapter_grad_kernel(GradArgs ga, GradArgs gb, int blocks0) {
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
// tile (1024 for more than two), so that an item's partial sums (written and read once) stay small
// beside what it reads.  4096 x 4096 bf16, rank 32: 128, 256, 512 tokens 30.2 + 8.4, 25.9 + 5.9,
// 30.2 + 4.6 us with the sum; rank 16: 64, 128, 256 tokens 27.4 + 8.6, 21.9 + 5.9, 21.9 + 4.8; 16384
// x 4096 and 8192 from a checkpoint, rank 64: 512, 1024, 1536 tokens 147 + 19, 136 + 13, 156 + 11.
constexpr int kMostChunk = 4096;
static int least_chunk(int max_rank) { return max_rank <= 16 ? 128 : max_rank <= 32 ? 256 : 1024; }
static int64_t wanted_items(int64_t d, int max_rank) {
  const int64_t cols = max_rank <= 16 ? 512 : 256, n = 768 / ((d + cols - 1) / cols);
  return n < 1 ? 1 : n;
}
int adapter_grad_chunk(int64_t tokens, int64_t d, int max_rank) {
  const int64_t items = wanted_items(d, max_rank);
  int64_t c = ((tokens + items - 1) / items + 31) / 32 * 32;
  if (c < least_chunk(max_rank)) c = least_chunk(max_rank);
  return (int)(c > kMostChunk ? kMostChunk : c);
}
// The most chunks that `tokens` or any fewer tokens are cut into.
int64_t adapter_grad_most_chunks(int64_t tokens, int64_t d, int max_rank) {
  const int64_t least = (tokens + least_chunk(max_rank) - 1) / least_chunk(max_rank), items = wanted_items(d, max_rank);
  const int64_t most = (tokens + kMostChunk - 1) / kMostChunk, n = least < items ? least : items;
  return n > most ? n : most;
}

template <int XT, int NR>
static int grad_blocks(const GradArgs &a) {
  const int cols = 64 * GradCols<XT, NR>::value;
  const int64_t items = a.whole ? a.b.adapters
                                : ((int64_t)a.b.tokens + a.chunk - 1) / a.chunk +
                                      (a.b.requests < a.b.adapters ? a.b.requests : a.b.adapters);
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
