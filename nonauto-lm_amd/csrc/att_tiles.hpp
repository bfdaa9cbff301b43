// Tile machinery of the biased attention kernels (biased_attention.hip, token_attention.hip): operand fragments, the staged
// LDS tiles and the score arithmetic, for bf16 and fp32 operands on the same 32 x 32 accumulator layout.
//
// A fragment is 8 consecutive contraction elements per lane, lane = (hh, r32), elements 8 hh .. 8 hh + 7 of a 16-wide
// slice.  bf16: one v_mfma_f32_32x32x16_bf16.  fp32: eight v_mfma_f32_32x32x2_f32, the j-th taking element j of both
// half-waves; a contraction does not care which k an instruction handles as long as A and B agree, so both types share
// every index below.
#pragma once
#include "common.hpp"

namespace mivae {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 att_bf16x4 __attribute__((__vector_size__(4 * sizeof(__bf16))));

constexpr int kChunk = 64;                          // rows of the streamed operands staged per pass
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNoCode = -2;                         // query code that equals no key code

// Kernel arguments; the C struct of include/mivae.h after the host's checks.  Strides are in elements (batch, row, head).
struct BiasedArgs {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  void* out;                    // (B, Sq, heads, d) contiguous
  unsigned short* out_lo;       // bf16: what the rounding of out leaves, or null
  // (2, B, heads, Sq), or null: m, then 1 / l, with p = 2^(score - m) / l; m = +inf and 0 for a row that sees no key.  (One
  // m + log2 l instead is off by half its last place, 1e-6 at 20, in every p of the row alike: that much of an fp32 gradient.)
  float* lse;
  const void* dout;             // (B, Sq, heads, d) contiguous
  float* delta;                 // (B, heads, Sq): sum_d dout * out
  void *dq, *dk, *dv;           // contiguous, may be null
  float* dtab;                  // bucket partials (heads, B * q blocks, nb), or null
  // visibility codes, or null: a pair is seen iff the codes are equal.  Keys: document id (0 without documents), -1 where
  // hidden.  Queries: document id, kNoCode where it is negative.  tiles: {lowest, highest visible code, visible rows} per 64
  const int *kcodes, *qcodes;
  const i32x4 *ktiles, *qtiles;
  const i32x4* sighted;         // backward: the queries' summaries with only the rows that see a key, or null: all do
  const int *prefix, *q_starts;
  const float* slopes;          // (heads), or null
  const float* table;           // (nb, heads), or null
  const int* buckets;           // (2 R + 1)
  int B, Sq, Sk, heads, kv, group, d, q_start, causal, nb, R, kpad, qpad, makes_delta;
  float scale, cap;             // cap = 0: no cap
};

__device__ __forceinline__ int acc_row(int reg) { return (reg & 3) + 8 * (reg >> 2); }    // + 4 hh

template <typename T>
struct Frag;
template <>
struct Frag<unsigned short> { typedef bf16x8 type; };
template <>
struct Frag<float> { typedef f32x8 type; };

__device__ __forceinline__ f32x16 mma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// accumulator registers 8 s .. 8 s + 7 as a fragment (rows 16 s + 4 hh + (j & 3) + 8 (j >> 2))
__device__ __forceinline__ void pack8(bf16x8& f, const f32x16& x, int s) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (bf16_t)x[8 * s + j];
}
__device__ __forceinline__ void pack8(f32x8& f, const f32x16& x, int s) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = x[8 * s + j];
}

// what the rounding of x to fragments f0, f1 left, as fragments
template <typename F>
__device__ __forceinline__ void pack_rest(F& f0, F& f1, f32x16& x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] -= (float)f0[j];
    x[8 + j] -= (float)f1[j];
  }
  pack8(f0, x, 0);
  pack8(f1, x, 1);
}

__device__ __forceinline__ float to_f32(unsigned short u) { return bf16_to_f32(u); }
__device__ __forceinline__ float to_f32(float f) { return f; }

// LDS tile of rows of 32 NDB elements, without padding for bf16: the 16-byte granule index is XORed with bits of the row so
// that both the 16-byte row reads (16 rows, one granule) and the transposing reads (4 rows, 4 granules) touch all 64 banks
// once.  4 or 12 granules per row: bits 2-3 of the row; 8: rows of one parity share the banks, bit 1 picks the half;
// 16: bits 0-1 pick the quarter.  fp32: an odd number of granules per row.
template <typename T, int NDB>
struct Tile;

template <int NDB>
struct Tile<unsigned short, NDB> {
  static constexpr int W = 32 * NDB;
  static constexpr int PITCH = W;
  static constexpr int GE = 8, GPR = W / GE;
  static __device__ __forceinline__ int swizzle(int r) {
    return NDB == 4 ? (r & 3) << 2 | ((r >> 2) & 3) : NDB == 2 ? (r & 2) << 1 | ((r >> 2) & 3) : (r >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * PITCH + ((c ^ swizzle(r)) << 3); }
  // f[j] = tile[r][16 s + 8 hh + j]
  static __device__ __forceinline__ bf16x8 row(const unsigned short* t, int r, int s, int hh) {
    return *reinterpret_cast<const bf16x8*>(t + at(r, 2 * s + hh));
  }
  // f[j] = tile[row0 + 4 hh + (j & 3) + 8 (j >> 2)][32 db + r32].  EXEC must be all ones.
  static __device__ __forceinline__ bf16x8 col(const unsigned short* t, int row0, int db, int lane) {
    const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
    const int r0 = row0 + 4 * (g >> 1) + q, r1 = r0 + 8;
    const int c = 4 * db + 2 * (g & 1) + (p >> 1), e = 4 * (p & 1);
    typedef __attribute__((address_space(3))) att_bf16x4* lds_ptr;
    const att_bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr)(t + at(r0, c) + e));
    const att_bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr)(t + at(r1, c) + e));
    return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <int NDB>
struct Tile<float, NDB> {
  static constexpr int W = 32 * NDB;
  static constexpr int PITCH = W + 4;
  static constexpr int GE = 4, GPR = W / GE;
  static __device__ __forceinline__ int at(int r, int c) { return r * PITCH + 4 * c; }
  static __device__ __forceinline__ f32x8 row(const float* t, int r, int s, int hh) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(t + at(r, 4 * s + 2 * hh));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(t + at(r, 4 * s + 2 * hh + 1));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ f32x8 col(const float* t, int row0, int db, int lane) {
    const float* p = t + (row0 + 4 * (lane >> 5)) * PITCH + 32 * db + (lane & 31);
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p[((j & 3) + 8 * (j >> 2)) * PITCH];
    return f;
  }
};

// row `row` of a head from global memory as the NS = 2 NDB fragments of an operand; zero where !ok and beyond d
template <typename T, int NDB>
__device__ __forceinline__ void load_row(typename Frag<T>::type (&f)[2 * NDB], const T* p, bool ok, int d, int hh) {
#pragma unroll
  for (int s = 0; s < 2 * NDB; ++s) {
    const int c = 16 * s + 8 * hh;
    constexpr int NV = sizeof(typename Frag<T>::type) / 16;
    i32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = i32x4{0, 0, 0, 0};
      if (ok && c < d) v[i] = reinterpret_cast<const i32x4*>(p + c)[i];
    }
    f[s] = __builtin_bit_cast(typename Frag<T>::type, v);
  }
}

// kChunk rows of one head on their way into an LDS tile, by 64 NW threads.  Rows whose bit of `rows` is 0 (beyond the end, or
// hidden keys: whatever they hold must not meet a product, 0 * NaN is NaN) and columns beyond d arrive as zeros.
//   bf16: global_load_lds, 16 bytes per lane into 64 consecutive granules of the tile.  The swizzle is on the global side (the
//         lane at position `pos` of row r fetches granule pos ^ x(r)), a zero granule is fetched from kZero16, no registers
//         are held while the loads travel.  land() waits for them; a barrier has to follow.
//   fp32: through registers (the padded tile is not linear); land() needs the tile consumed by everybody.
static __device__ const i32x4 kZero16[1] = {{0, 0, 0, 0}};

__device__ __forceinline__ uint64_t low_rows(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

template <typename T, int NDB, int NW>
struct Stage;

template <int NDB, int NW>
struct Stage<unsigned short, NDB, NW> {
  using L = Tile<unsigned short, NDB>;
  static constexpr int NBUF = 2, N = L::GPR / NW;
  static_assert(L::GPR % NW == 0, "whole waves of granules");
  __device__ __forceinline__ void issue(unsigned short* tile, const unsigned short* src, int64_t sr, int row0, uint64_t rows, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int first = (i * NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 64, g = first + (threadIdx.x & 63);
      const int row = g / L::GPR, c = (g % L::GPR) ^ L::swizzle(row);
      const bool ok = ((rows >> row) & 1) && c * L::GE < d;
      const void* p = ok ? (const void*)(src + (int64_t)(row0 + row) * sr + c * L::GE) : (const void*)kZero16;
      const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned short*)(tile + first * L::GE);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "memory", "m0");
    }
  }
  __device__ __forceinline__ void land(unsigned short*) { __builtin_amdgcn_s_waitcnt(0x0f70); }       // vmcnt(0)
};

template <int NDB, int NW>
struct Stage<float, NDB, NW> {
  using L = Tile<float, NDB>;
  static constexpr int NBUF = 1, N = kChunk * L::GPR / (64 * NW);
  i32x4 r[N];
  __device__ __forceinline__ void issue(float*, const float* src, int64_t sr, int row0, uint64_t rows, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = threadIdx.x + i * 64 * NW, row = idx / L::GPR, c = idx % L::GPR;
      r[i] = i32x4{0, 0, 0, 0};
      if (((rows >> row) & 1) && c * L::GE < d) r[i] = *reinterpret_cast<const i32x4*>(src + (int64_t)(row0 + row) * sr + c * L::GE);
    }
  }
  __device__ __forceinline__ void land(float* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = threadIdx.x + i * 64 * NW, row = idx / L::GPR, c = idx % L::GPR;
      *reinterpret_cast<i32x4*>(tile + L::at(row, c)) = r[i];
    }
  }
};

__device__ __forceinline__ void store_lse(const BiasedArgs& a, int64_t at, float m, float l) {
  a.lse[at] = l == 0.f ? INFINITY : m;
  a.lse[(int64_t)a.B * a.heads * a.Sq + at] = l == 0.f ? 0.f : 1.f / l;
}

// rows d = 32 db + 8 a + 4 hh .. + 3 of the transposed accumulators -> one row of a contiguous (.., d) tensor
__device__ __forceinline__ void store4(unsigned short* p, float a, float b, float c, float e) {
  const u16x4 o = {f32_to_bf16(a), f32_to_bf16(b), f32_to_bf16(c), f32_to_bf16(e)};
  *reinterpret_cast<u16x4*>(p) = o;
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float e) {
  const f32x4 o = {a, b, c, e};
  *reinterpret_cast<f32x4*>(p) = o;
}
// four values of the output, and with `lo` what their rounding leaves
__device__ __forceinline__ void store_out(unsigned short* out, unsigned short* lo, int64_t at, float a, float b, float c, float e) {
  const u16x4 o = {f32_to_bf16(a), f32_to_bf16(b), f32_to_bf16(c), f32_to_bf16(e)};
  *reinterpret_cast<u16x4*>(out + at) = o;
  if (lo != nullptr) store4(lo + at, a - bf16_to_f32(o[0]), b - bf16_to_f32(o[1]), c - bf16_to_f32(o[2]), e - bf16_to_f32(o[3]));
}
__device__ __forceinline__ void store_out(float* out, unsigned short*, int64_t at, float a, float b, float c, float e) {
  store4(out + at, a, b, c, e);
}
template <typename T, int NDB>
__device__ __forceinline__ void store_row(T* dst, const f32x16 (&x)[NDB], float mul, int d, int hh) {
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) {
      const int c = 32 * db + 8 * a4 + 4 * hh;
      if (c < d)
        store4(dst + c, x[db][4 * a4] * mul, x[db][4 * a4 + 1] * mul, x[db][4 * a4 + 2] * mul, x[db][4 * a4 + 3] * mul);
    }
}

// Scores of a block.  The raw product x of a pair becomes u = x, or with a cap u = tanh(scale x / cap); the score is then
// A u, A >= 0, plus the bias.  bf16: in base-2 exponent units, log2 e inside A and the bias, so that where the bias is constant
// over a tile everything folds into the exponential's one fma.  fp32: in natural units, and log2 e in that fma: a rounded
// A log2 e would err by up to 6e-8 of every score, alike over the row (log2 e itself: 1.3e-8).
template <typename T>
constexpr float kUnit = sizeof(T) == 4 ? 1.f : kLog2e;
template <typename T>
constexpr float kPost = sizeof(T) == 4 ? kLog2e : 1.f;

struct Score {
  float A, k;         // k = scale / cap
  float slope;
  bool cap, slopes, tab;
};

template <typename T>
__device__ __forceinline__ Score score_of(const BiasedArgs& a, int head) {
  Score p;
  p.cap = a.cap > 0.f;
  p.A = (p.cap ? a.cap : a.scale) * kUnit<T>;
  p.k = p.cap ? a.scale / a.cap : 0.f;
  p.slopes = a.slopes != nullptr;
  p.slope = p.slopes ? a.slopes[head] * kUnit<T> : 0.f;
  p.tab = a.table != nullptr;
  return p;
}

// u <- tanh(k u).  |y| <= 3/4, the usual case, takes y P(y^2), P of degree 5 with the smallest largest relative error (fitted on
// Chebyshev nodes; 1.5e-7 evaluated in fp32): 8 plain instructions an element, where 1 - 2 / (1 + e^2y) takes two
// transcendental ones and is off by 2e-7 absolutely, i.e. by cap * 2e-7 in every score.  Larger |y| take the latter, whose relative
// error is as small there.  Each element by itself: next to a score near a large cap, small ones keep their places.
//   kCapRough: always the latter, in one basic block with the products around it (bf16 without gradients and caps up to kRoughCap,
//              where an error of 1e-4 in the exponent stands against the 2e-3 of a probability's rounding; 8191 queries of 128:
//              515 us, 540 with kCapAhead)
//   kCapTile:  a tile whose |y| are all small leaves the transcendental instructions out (4 x 16 x 4096 documents, bf16: dq 139 us,
//              dk and dv 187; with a larger one in every tile 162 and 207)
//   kCapAhead: as kCapTile with the polynomial before that branch, where it overlaps the products (bf16 training forward: 115
//              instead of 130 us at the same size, 126 with a larger one in every tile; in dq and dk / dv it
//              makes no difference and costs registers)
enum Cap { kCapRough, kCapTile, kCapAhead };
constexpr float kRoughCap = 512.f;
__device__ __forceinline__ float tanh_near(float y) {
  const float t = y * y;
  float q = fmaf(t, -0.00471625663f, 0.0195829067f);
  q = fmaf(t, q, -0.0533444285f);
  q = fmaf(t, q, 0.133254066f);
  q = fmaf(t, q, -0.333329588f);
  return fmaf(t * y, q, y);
}
__device__ __forceinline__ float tanh_far(float y2) {      // of y2 / (2 log2 e)
  return fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y2)), 1.f);
}
template <Cap KIND>
__device__ __forceinline__ void cap_tile(f32x16& u, const Score& p) {
  const float k2 = 2.f * kLog2e * p.k;
  if (KIND == kCapRough) {
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = tanh_far(k2 * u[r]);
    return;
  }
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(u[r]));
  const bool far = __builtin_amdgcn_ballot_w64(most * p.k > 0.75f) != 0;
  f32x16 near = u;
  if (KIND == kCapAhead) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      near[r] = tanh_near(p.k * u[r]);
      asm volatile("" : "+v"(near[r]));          // here, not in the branch below
    }
  }
  if (far) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float y = p.k * u[r], n = KIND == kCapAhead ? near[r] : tanh_near(y);
      u[r] = fabsf(y) <= 0.75f ? n : tanh_far(k2 * u[r]);
    }
  } else if (KIND == kCapTile) {
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = tanh_near(p.k * u[r]);
  } else {
    u = near;
  }
}
__device__ __forceinline__ float cap_slope(float u) { return fmaf(-u, u, 1.f); }

__device__ __forceinline__ void scale_tile(f32x16& u, const Score& p) {
#pragma unroll
  for (int r = 0; r < 16; ++r) u[r] *= p.A;
}

// Element-wise part: u <- A u + bias.  Register r's relative distance key - query is rel + SIGN * acc_row(r) (SIGN = 1: the
// lane is a query, -1: the lane is a key); rel0 is that of the wave's first lane's row to the tile's first.
template <int SIGN>
__device__ __forceinline__ void bias_tile(f32x16& u, const Score& p, const float* tab, int R, int rel, int rel0) {
  const bool inside = rel0 - 31 >= -R && rel0 + 31 <= R;        // wave-uniform
  scale_tile(u, p);
  if (p.slopes) {                       // one rounding, of the score itself: forward and backward agree on it
    const float from = (float)rel;
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = fmaf(-p.slope, fabsf(from + (float)(SIGN * acc_row(r))), u[r]);
  }
  if (p.tab) {
    const float* t = tab + R + rel;
    if (inside) {
#pragma unroll
      for (int r = 0; r < 16; ++r) u[r] += t[SIGN * acc_row(r)];
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) u[r] += tab[min(max(rel + SIGN * acc_row(r), -R), R) + R];
    }
  }
}

// the bias by relative distance of one head: tab[R + rel], rel = -R .. R
template <typename T>
__device__ __forceinline__ void stage_table(float* tab, const BiasedArgs& a, int head, int nthreads) {
  for (int i = threadIdx.x; i <= 2 * a.R; i += nthreads) {
    const int b = min(max(a.buckets[i], 0), a.nb - 1);
    tab[i] = a.table[(int64_t)b * a.heads + head] * kUnit<T>;
  }
}

__device__ __forceinline__ int clamp_start(int s) { return min(max(s, -(1 << 30)), 1 << 30); }

// ---- visibility ---------------------------------------------------------------------------------------------------------
// Causal mask and prefix are one limit per query, non-decreasing in the row: it sees the keys below limit(i).
struct View {
  int start, prefix, Sk;
  bool causal, codes, docs;
  __device__ __forceinline__ int limit(int row) const { return causal ? min(Sk, max(start + row + 1, prefix)) : Sk; }
  // first query row that sees key j
  __device__ __forceinline__ int first_row(int key) const { return !causal || key < prefix ? 0 : max(0, key - start); }
};

__device__ __forceinline__ View view_of(const BiasedArgs& a, int64_t b) {
  View v;
  v.start = clamp_start(a.q_starts ? a.q_starts[b] : a.q_start);
  v.prefix = a.prefix ? a.prefix[b] : 0;
  v.Sk = a.Sk;
  v.causal = a.causal != 0;
  v.codes = a.kcodes != nullptr;
  v.docs = a.qcodes != nullptr;
  return v;
}

// lowest / highest value of `code` over the wave's lanes with code >= 0
__device__ __forceinline__ void wave_range(int code, int& lo, int& hi) {
  lo = code >= 0 ? code : INT32_MAX;
  hi = code >= 0 ? code : -1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off, 64));
    hi = max(hi, __shfl_xor(hi, off, 64));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
}

__device__ __forceinline__ i32x4 merge(const i32x4& a, const i32x4& b) {
  return i32x4{min(a[0], b[0]), max(a[1], b[1]), 0, 0};
}
__device__ __forceinline__ uint64_t rows_of(const i32x4& t) { return (uint64_t)(unsigned)t[3] << 32 | (unsigned)t[2]; }

// the other half-wave's value, without a trip through LDS
__device__ __forceinline__ float max_halves(float x) {
  const unsigned b = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);        // {both low halves, both high halves}
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Issue order for a run of N bf16 products whose A operands take DS LDS reads each: the reads stay two products ahead of the
// matrix core.  (The compiler's own order waits for the LDS before most products.)  A no-op for fp32.
template <typename T, int N, int DS>
__device__ __forceinline__ void reads_ahead() {
  if (sizeof(T) == 2 && N > 2) {
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * DS, 0);
#pragma unroll
    for (int i = 0; i < N - 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, DS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace mivae
