// Root-mean-square norm of every query and key head, learned scale and position rotation in one pass, forward and backward.
//
//   r = (mean_d x^2 + eps)^-1/2;  n = x r w;  a pair (a, b) of n at angle t: (a cos t - b sin t, a sin t + b cos t)
//   dn = R(-t) dy;  dw = sum over rows of dn x r;  dx = r (dn w - x r mean_d(dn w x r))
//
// Bound by HBM: reads x and writes y once (backward: reads x and dy, writes dx).  (2 x 8191 tokens, 16 + 4 heads of 96, fp32,
// half rotated: 55 us and 76 us, 4.7 and 5.0 TB/s; 64 x 512, 4 + 4 heads of 128, bf16: 32 and 59 us, 4.2 and 3.4 TB/s, where
// the VALU issues in 78 % and 65 % of the cycles.)  A lane holds one or more chunks of VEC
// pairs of a head row, so the two halves of a pair meet in its registers whatever the pairing, and a row is a power of two
// of neighbouring lanes.  The angles of a token are shared by all its heads: a block takes a few whole tokens and puts
// their cosines and sines into LDS once.  t = 2 pi frac(position f) is reduced in 64 bits, where positions of 2^31 keep
// 22 bits behind the point, and only then rounded: an fp32 product would be off by whole turns at far positions.
#include "common.hpp"
#include "mivae.h"

using namespace mivae;

namespace {

struct RotArgs {
  const void *q, *k, *dyq, *dyk;        // dy*: backward, contiguous
  void *oq, *ok;                        // outputs (forward) or input gradients (backward), contiguous
  const float *qw, *kw;                 // (d), or null: 1
  float* part;                          // backward: (blocks, 2, d) weight-gradient partials, or null
  const double* freq;                   // (rot / 2) turns per position, or null: no rotation
  const int64_t* pos;                   // element (b, s) at pos[b * pos_b + s * pos_s], or null: start + s
  int64_t qs[3], ks[3], pos_b, pos_s, start;
  unsigned tokens, S, rows_magic, half_magic;       // x / (H + G) = umulhi(x, rows_magic) and x / half likewise, x < 2^16
  int H, G, d, half, rest, lpr, tpb, inter;         // half = rot / 2, rest = (d - rot) / 2; lpr lanes per row, tpb tokens at a time
  float eps;
};

// (batch row, position) of token t behind token (b0, s0)
__device__ __forceinline__ void token_at(unsigned S, unsigned b0, unsigned s0, unsigned t, int64_t& b, int64_t& s) {
  unsigned x = s0 + t, y = b0;
  while (x >= S) {
    x -= S;
    ++y;
  }
  b = y;
  s = x;
}

constexpr int kThreads = 256;

// where pair chunk c of VEC pairs keeps its two vectors.  Pairs: (i, half + i) or, interleaved, (2 i, 2 i + 1) in the
// rotated part; the rest is cut into two halves likewise, only to be read and written.
template <int VEC>
__device__ __forceinline__ void chunk_at(const RotArgs& a, int c, int& ia, int& ib) {
  const int i = c * VEC;
  if (a.inter) {
    ia = 2 * i;
    ib = ia + VEC;
  } else if (i < a.half) {
    ia = i;
    ib = a.half + i;
  } else {
    ia = a.half + i;                    // 2 half + (i - half)
    ib = ia + a.rest;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void load2(const T* p, int ia, int ib, float (&u)[VEC], float (&w)[VEC]) {
  RowIO<T, VEC>::load(p + ia, u);
  RowIO<T, VEC>::load(p + ib, w);
}

// (first, second) elements of the chunk's pairs <-> the two vectors
template <int VEC>
__device__ __forceinline__ void split_pairs(bool inter, const float (&u)[VEC], const float (&w)[VEC], float (&a)[VEC], float (&b)[VEC]) {
  if (!inter) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { a[i] = u[i]; b[i] = w[i]; }
  } else if (VEC == 1) {
    a[0] = u[0]; b[0] = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = 2 * i < VEC ? u[(2 * i) % VEC] : w[(2 * i) % VEC];
      b[i] = 2 * i < VEC ? u[(2 * i + 1) % VEC] : w[(2 * i + 1) % VEC];
    }
  }
}
template <int VEC>
__device__ __forceinline__ void join_pairs(bool inter, const float (&a)[VEC], const float (&b)[VEC], float (&u)[VEC], float (&w)[VEC]) {
  if (!inter || VEC == 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { u[i] = a[i]; w[i] = b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      u[i] = i % 2 ? b[i / 2] : a[i / 2];
      w[i] = i % 2 ? b[(VEC + i) / 2] : a[(VEC + i) / 2];
    }
  }
}

// cosines and sines of ntok tokens from (b0, s0) on: cs[token][pair] = {cos, sin}
__device__ __forceinline__ void stage_angles(float2* cs, const RotArgs& a, unsigned b0, unsigned s0, int ntok) {
  for (int i = threadIdx.x; i < ntok * a.half; i += kThreads) {
    const unsigned t = a.half == 1 ? i : __umulhi(i, a.half_magic);
    int64_t b, s;
    token_at(a.S, b0, s0, t, b, s);
    const int64_t p = a.pos ? a.pos[b * a.pos_b + s * a.pos_s] : a.start + s;
    const double turns = (double)p * a.freq[i - t * a.half];
    float sn, cn;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
    cs[i] = make_float2(cn, sn);
  }
}

// CPL: chunks per lane (1 but for the scalar form of rows of more than 64 pairs)
template <typename T, int VEC, int CPL, bool NORM, bool BWD>
__global__ __launch_bounds__(kThreads) void k_qk(RotArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2* cs = reinterpret_cast<float2*>(smem);       // [2][tpb][half]: written for the next tokens while these are read
  const int HG = a.H + a.G, lane_c = threadIdx.x % a.lpr, slot = threadIdx.x / a.lpr, slots = kThreads / a.lpr;
  const int chunks = (a.half + a.rest) / VEC;
  const float inv_d = 1.f / (float)a.d;
  int ia[CPL], ib[CPL];
  bool on[CPL];
  float wq[CPL][2][VEC], wk[CPL][2][VEC], gq[CPL][2][VEC], gk[CPL][2][VEC];      // scales, and their gradients' sums
#pragma unroll
  for (int n = 0; n < CPL; ++n) {
    const int c = lane_c + n * a.lpr;
    on[n] = c < chunks;
    chunk_at<VEC>(a, on[n] ? c : 0, ia[n], ib[n]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      gq[n][0][i] = gq[n][1][i] = gk[n][0][i] = gk[n][1][i] = 0.f;
      if (NORM) {
        // element index of the pair's first and second member
        const int ea = a.inter ? ia[n] + 2 * i : ia[n] + i, eb = a.inter ? ia[n] + 2 * i + 1 : ib[n] + i;
        wq[n][0][i] = a.qw && on[n] ? a.qw[ea] : 1.f;
        wq[n][1][i] = a.qw && on[n] ? a.qw[eb] : 1.f;
        wk[n][0][i] = a.kw && on[n] ? a.kw[ea] : 1.f;
        wk[n][1][i] = a.kw && on[n] ? a.kw[eb] : 1.f;
      }
    }
  }
  unsigned odd = 0;
  for (unsigned tok0 = blockIdx.x * a.tpb; tok0 < a.tokens; tok0 += gridDim.x * a.tpb, odd ^= 1) {
    const int ntok = (int)min((unsigned)a.tpb, a.tokens - tok0);
    const unsigned b0 = tok0 / a.S, s0 = tok0 % a.S;
    const float2* now = cs + odd * a.tpb * a.half;
    if (a.freq) {
      stage_angles(cs + odd * a.tpb * a.half, a, b0, s0, ntok);
      __syncthreads();
    }
    const int rows = ntok * HG;
    // every lane of the block takes the same number of turns: the row sums are shuffles
    for (int r0 = 0; r0 < rows; r0 += slots) {
      const int r = r0 + slot;
      const bool live = r < rows;
      const int t = live ? (int)__umulhi(r, a.rows_magic) : 0, hd = live ? r - t * HG : 0;
      const bool isq = hd < a.H;
      const int64_t tok = (int64_t)tok0 + t;
      int64_t b, s;
      token_at(a.S, b0, s0, t, b, s);
      const T* x = isq ? static_cast<const T*>(a.q) + b * a.qs[0] + s * a.qs[1] + hd * a.qs[2]
                       : static_cast<const T*>(a.k) + b * a.ks[0] + s * a.ks[1] + (hd - a.H) * a.ks[2];
      const int64_t o = isq ? (tok * a.H + hd) * a.d : (tok * a.G + hd - a.H) * a.d;
      T* y = (isq ? static_cast<T*>(a.oq) : static_cast<T*>(a.ok)) + o;
      const T* dy = BWD ? (isq ? static_cast<const T*>(a.dyq) : static_cast<const T*>(a.dyk)) + o : nullptr;
      float xa[CPL][VEC], xb[CPL][VEC], da[CPL][VEC], db[CPL][VEC];
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < CPL; ++n) {
        float u[VEC], w[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) { u[i] = w[i] = 0.f; xa[n][i] = xb[n][i] = 0.f; }
        if (NORM || !BWD) {
          if (live && on[n]) load2<T, VEC>(x, ia[n], ib[n], u, w);
          split_pairs<VEC>(a.inter, u, w, xa[n], xb[n]);
        }
        if (BWD) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) u[i] = w[i] = 0.f;
          if (live && on[n]) load2<T, VEC>(dy, ia[n], ib[n], u, w);
          split_pairs<VEC>(a.inter, u, w, da[n], db[n]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum = fmaf(xa[n][i], xa[n][i], fmaf(xb[n][i], xb[n][i], sum));
      }
      float inv = 1.f;
      if (NORM) inv = 1.f / sqrtf(fmaf(group_sum(sum, a.lpr), inv_d, a.eps));
      const float2* c0 = now + t * a.half;
      float dot = 0.f;
#pragma unroll
      for (int n = 0; n < CPL; ++n) {
        const int p0 = (lane_c + n * a.lpr) * VEC;
        const bool turn = a.freq && on[n] && p0 < a.half;       // a chunk is rotated as a whole or not at all
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 c = turn ? c0[p0 + i] : make_float2(1.f, 0.f);
          if (!BWD) {
            float va = xa[n][i], vb = xb[n][i];
            if (NORM) {
              va *= inv * (isq ? wq[n][0][i] : wk[n][0][i]);
              vb *= inv * (isq ? wq[n][1][i] : wk[n][1][i]);
            }
            xa[n][i] = va * c.x - vb * c.y;
            xb[n][i] = fmaf(va, c.y, vb * c.x);
          } else {
            const float ga = fmaf(da[n][i], c.x, db[n][i] * c.y), gb = db[n][i] * c.x - da[n][i] * c.y;
            if (NORM) {
              xa[n][i] *= inv;
              xb[n][i] *= inv;
              const float ta = ga * xa[n][i], tb = gb * xb[n][i];
              gq[n][0][i] += isq ? ta : 0.f;
              gq[n][1][i] += isq ? tb : 0.f;
              gk[n][0][i] += isq ? 0.f : ta;
              gk[n][1][i] += isq ? 0.f : tb;
              da[n][i] = ga * (isq ? wq[n][0][i] : wk[n][0][i]);
              db[n][i] = gb * (isq ? wq[n][1][i] : wk[n][1][i]);
              dot = fmaf(da[n][i], xa[n][i], fmaf(db[n][i], xb[n][i], dot));
            } else {
              xa[n][i] = ga;
              xb[n][i] = gb;
            }
          }
        }
      }
      if (BWD && NORM) {
        const float mean = group_sum(dot, a.lpr) * inv_d;
#pragma unroll
        for (int n = 0; n < CPL; ++n)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            xa[n][i] = inv * (da[n][i] - xa[n][i] * mean);
            xb[n][i] = inv * (db[n][i] - xb[n][i] * mean);
          }
      }
#pragma unroll
      for (int n = 0; n < CPL; ++n) {
        float u[VEC], w[VEC];
        join_pairs<VEC>(a.inter, xa[n], xb[n], u, w);
        if (live && on[n] && y != nullptr) {
          RowIO<T, VEC>::store(y + ia[n], u);
          RowIO<T, VEC>::store(y + ib[n], w);
        }
      }
    }
  }
  if (BWD && NORM && a.part) {          // sum over the block's rows: slots of a wave by shuffles, then the waves in order
    float* red = reinterpret_cast<float*>(smem);                // [4 waves][2 d]
    __syncthreads();
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int n = 0; n < CPL; ++n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float v[4] = {gq[n][0][i], gq[n][1][i], gk[n][0][i], gk[n][1][i]};
        for (int off = 32; off >= a.lpr; off >>= 1)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], off, 64);
        const int ea = a.inter ? ia[n] + 2 * i : ia[n] + i, eb = a.inter ? ia[n] + 2 * i + 1 : ib[n] + i;
        if ((threadIdx.x & 63) < a.lpr && on[n]) {
          red[wave * 2 * a.d + ea] = v[0];
          red[wave * 2 * a.d + eb] = v[1];
          red[wave * 2 * a.d + a.d + ea] = v[2];
          red[wave * 2 * a.d + a.d + eb] = v[3];
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) s += red[w * 2 * a.d + i];
      a.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
    }
  }
}

// dqw / dkw = the blocks' partials summed in a fixed order: 16 columns per block, 64 rows at a time
__global__ __launch_bounds__(1024) void k_qk_dw(const float* part, float* dqw, float* dkw, int blocks, int d) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  float s = 0.f;
  if (e < 2 * d)
    for (int i = g; i < blocks; i += 64) s += part[(int64_t)i * 2 * d + e];
  red[g][c] = s;
  for (int n = 32; n > 0; n >>= 1) {
    __syncthreads();
    if (g < n) red[g][c] += red[g + n][c];
  }
  float* dst = e < d ? dqw : dkw;
  if (g == 0 && e < 2 * d && dst) dst[e < d ? e : e - d] = red[0][c];
}

// Four blocks per CU; the backward leaves a row of partials for each.  Forward, backward, fold: 32 + 60 + 7 us at 64 x 512 tokens, 4 + 4
// heads of 128, bf16, and 59 + 79 + 7 at 2 x 8191, 16 + 4 heads of 96, fp32.  With two per CU 38 + 56 + 4 and 86 + 110 + 4, with
// eight 35 + 59 + 12 and 59 + 80 + 12.
constexpr int kMaxBlocks = 1024;

struct Geometry {
  bool vec;
  int tpb, blocks, lpr;
};
Geometry geometry(const mivae_rotary_args* x) {
  Geometry g;
  const int V = x->dtype == MIVAE_F32 ? 4 : 8;
  const int64_t half = x->freq ? x->rotary_dim / 2 : 0, rest = x->head_size / 2 - half;
  // 16-byte accesses: whole chunks of 16 bytes in both members of the pairs and 16-byte aligned rows; otherwise scalars
  g.vec = half % V == 0 && rest % V == 0 && aligned16(x->q) && aligned16(x->k) && aligned16(x->q_out) && aligned16(x->k_out) &&
          aligned16(x->dq_out) && aligned16(x->dk_out);
  for (int i = 0; i < 3; ++i) g.vec = g.vec && x->q_stride[i] % V == 0 && x->k_stride[i] % V == 0;
  const int64_t chunks = (half + rest) / (g.vec ? V : 1);
  g.lpr = 1;
  while (g.lpr < chunks && g.lpr < 64) g.lpr <<= 1;
  // Whole tokens at a time: enough rows for two turns of a block's lanes, up to 16 tokens (64 x 512 tokens with 1 + 1 heads of 32, bf16:
  // 11 + 22 us forward and backward, 14 + 29 with 8, 21 + 43 with 4), while there are two blocks for every CU (8 x 1024 tokens, 1 + 1
  // heads of 16: 5 + 11 us, 8 + 21 if eight are asked for; half a block per CU: no difference)
  const int64_t HG = x->heads + x->kv_heads, tokens = x->batch * x->len, slots = kThreads / g.lpr;
  int64_t tpb = (2 * slots + HG - 1) / HG;
  if (tpb > 16) tpb = 16;
  while (tpb > 1 && (tokens + tpb - 1) / tpb < 512) tpb >>= 1;
  g.tpb = (int)tpb;
  const int64_t need = (tokens + tpb - 1) / tpb;
  g.blocks = (int)(need < kMaxBlocks ? need : kMaxBlocks);
  return g;
}

template <typename T, int V>
void launch(const RotArgs& a, const Geometry& g, int64_t blocks, size_t lds, bool norm, bool bwd, hipStream_t st) {
  const bool two = (a.half + a.rest) > 64;
  void (*fn)(RotArgs);
#define MIVAE_QK(VEC, CPL) \
  (norm ? (bwd ? k_qk<T, VEC, CPL, true, true> : k_qk<T, VEC, CPL, true, false>) : (bwd ? k_qk<T, VEC, CPL, false, true> : k_qk<T, VEC, CPL, false, false>))
  if (g.vec) fn = MIVAE_QK(V, 1);
  else if (two) fn = MIVAE_QK(1, 2);
  else fn = MIVAE_QK(1, 1);
#undef MIVAE_QK
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(kThreads), lds, st, a);
}

int run(const mivae_rotary_args* x, bool bwd, const char* name, void* stream) {
  MIVAE_REQUIRE(x != nullptr, "%s: null arguments", name);
  MIVAE_REQUIRE(x->dtype == MIVAE_F32 || x->dtype == MIVAE_BF16, "%s: dtype %d is neither float32 nor bfloat16", name, x->dtype);
  MIVAE_REQUIRE(x->batch >= 1 && x->len >= 1 && x->heads >= 1 && x->kv_heads >= 1 && x->heads + x->kv_heads <= 4095 &&
                    x->batch < (1ll << 31) && x->len < (1ll << 31) && x->batch * x->len < (1ll << 31) - (1 << 16),
                "%s: batch %lld, length %lld, heads %lld + %lld out of range", name, (long long)x->batch, (long long)x->len,
                (long long)x->heads, (long long)x->kv_heads);
  MIVAE_REQUIRE(x->head_size >= 2 && x->head_size <= 256 && x->head_size % 2 == 0, "%s: head size %lld is not an even number in 2 .. 256",
                name, (long long)x->head_size);
  MIVAE_REQUIRE(!x->freq || (x->rotary_dim >= 2 && x->rotary_dim % 2 == 0 && x->rotary_dim <= x->head_size),
                "%s: rotary size %lld is not an even number up to the head size", name, (long long)x->rotary_dim);
  MIVAE_REQUIRE(x->norm || x->freq, "%s: neither a norm nor a rotation", name);
  MIVAE_REQUIRE(x->norm || !(x->q_weight || x->k_weight), "%s: weights without a norm", name);
  MIVAE_REQUIRE(!x->norm || (x->eps >= 0.f && x->eps < 1e30f), "%s: eps out of range", name);
  MIVAE_REQUIRE(x->q_out && x->k_out, "%s: null output", name);
  MIVAE_REQUIRE((x->q && x->k) || (bwd && !x->norm), "%s: null operand", name);
  MIVAE_REQUIRE(!bwd || (x->dq_out && x->dk_out), "%s: null gradient", name);
  MIVAE_REQUIRE(!(x->dq_weight || x->dk_weight) || (bwd && x->norm && x->scratch), "%s: weight gradients need a norm and the scratch buffer", name);
  RotArgs a = {};
  a.q = x->q; a.k = x->k; a.dyq = x->dq_out; a.dyk = x->dk_out; a.oq = x->q_out; a.ok = x->k_out;
  a.qw = x->q_weight; a.kw = x->k_weight;
  a.freq = x->freq; a.pos = x->positions;
  for (int i = 0; i < 3; ++i) { a.qs[i] = x->q_stride[i]; a.ks[i] = x->k_stride[i]; }
  a.pos_b = x->position_stride[0]; a.pos_s = x->position_stride[1]; a.start = x->start;
  a.tokens = (unsigned)(x->batch * x->len);
  a.S = (unsigned)x->len; a.H = (int)x->heads; a.G = (int)x->kv_heads; a.d = (int)x->head_size;
  a.half = x->freq ? (int)x->rotary_dim / 2 : 0;
  a.rest = a.d / 2 - a.half;
  a.inter = x->interleaved ? 1 : 0;
  a.eps = x->eps;
  const Geometry g = geometry(x);
  a.lpr = g.lpr; a.tpb = g.tpb;
  const bool dw = x->dq_weight || x->dk_weight;
  a.part = dw ? x->scratch : nullptr;
  size_t lds = (size_t)2 * a.tpb * a.half * sizeof(float2);
  if (dw && lds < (size_t)kThreads / 64 * 2 * a.d * 4) lds = (size_t)kThreads / 64 * 2 * a.d * 4;
  const int64_t blocks = g.blocks;
  a.rows_magic = (unsigned)(((1ull << 32) + a.H + a.G - 1) / (a.H + a.G));
  a.half_magic = a.half > 1 ? (unsigned)(((1ull << 32) + a.half - 1) / a.half) : 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (x->dtype == MIVAE_F32) launch<float, 4>(a, g, blocks, lds, x->norm != 0, bwd, st);
  else launch<unsigned short, 8>(a, g, blocks, lds, x->norm != 0, bwd, st);
  MIVAE_CHECK_LAUNCH(name);
  if (dw) {
    hipLaunchKernelGGL(k_qk_dw, dim3((unsigned)((2 * a.d + 15) / 16)), dim3(1024), 0, st, x->scratch, x->dq_weight, x->dk_weight, (int)blocks, a.d);
    MIVAE_CHECK_LAUNCH(name);
  }
  return MIVAE_OK;
}

}  // namespace

extern "C" {

int64_t mivae_qk_norm_rotary_scratch_floats(int64_t head_size) { return (int64_t)kMaxBlocks * 2 * head_size; }

int mivae_qk_norm_rotary_fwd(const mivae_rotary_args* args, void* stream) {
  return run(args, false, "mivae_qk_norm_rotary_fwd", stream);
}

int mivae_qk_norm_rotary_bwd(const mivae_rotary_args* args, void* stream) {
  return run(args, true, "mivae_qk_norm_rotary_bwd", stream);
}

}  // extern "C"
