// Attention whose scores are capped by a tanh, biased by distance (slopes per head, or a learned table by buckets) and
// limited by key masks, documents and a prefix; shared key heads; any lengths; bf16 and fp32; forward and backward.
//
//   s = scale q.k;  s = cap tanh(s / cap);  s += -slope_h |i - j|  or  table[bucket(j - i), h];  p = softmax over the seen j
//   o = sum_j p v_j;  a row that sees no key gives 0 and passes no gradient
//   ds = p (do.v - delta), delta = do.o;  dtable[bucket, h] = sum ds;  ds' = scale (1 - tanh^2) ds
//   dq = ds' k;  dk = ds'^T q;  dv = p^T do, the latter two summed over the query heads of a key head
//
// 32 x 32 score tiles on the matrix cores; per product the operand order is chosen so that the accumulator layout is the
// next product's B operand and no score passes through LDS:
//   forward / dq: a wave owns 32 queries, S^T = K Q^T, so softmax statistics are per lane, then O^T = V^T P^T
//   dk / dv:      a wave owns 32 keys, S = Q K^T, then dV^T = dO^T P, dK^T = Q^T dS
// The backward recomputes the scores in both kernels (7 products, not 5): every output is written once, without atomics.
// Softmax statistics, sums and all score arithmetic are fp32; P and dS are rounded to the operands' type for the second
// products, which is what lets them run on the bf16 matrix instruction.
#include "att_tiles.hpp"
#include "mivae.h"

using namespace mivae;

namespace {

static inline hipStream_t S_(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr float kSlack = 8.f;       // exponent slack before the accumulators are rescaled
constexpr int kWaves = 4, kRows = 32 * kWaves;      // rows (queries or keys) of a block
constexpr int kMaxDistance = 1024, kMaxBuckets = 256;

// ---- visibility codes ------------------------------------------------------------------------------------------------
// One wave per 64 keys (or queries): code per row and {lowest, highest visible code, any hidden} per 64 rows.
__global__ __launch_bounds__(256) void k_ba_codes(const int64_t* mask, const int* documents, const int* q_starts, int q_start,
                                                  int B, int Sq, int Sk, int kpad, int qpad, int* kcodes, int* qcodes,
                                                  i32x4* ktiles, i32x4* qtiles) {
  const int nkt = kpad / 64, nqt = documents ? qpad / 64 : 0, lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)B * (nkt + nqt)) return;
  const int64_t b = w / (nkt + nqt);
  const int t = (int)(w % (nkt + nqt));
  const bool keys = t < nkt;
  int code;
  bool seen;
  if (keys) {
    const int j = t * 64 + lane;
    code = j < Sk ? (documents ? documents[b * Sk + j] : 0) : -1;
    if (j < Sk && mask && mask[b * Sk + j] == 0) code = -1;
    code = max(code, -1);
    seen = code >= 0;
    kcodes[b * kpad + j] = code;
  } else {
    const int i = (t - nkt) * 64 + lane;
    const int64_t pos = (int64_t)clamp_start(q_starts ? q_starts[b] : q_start) + i;
    code = i < Sq && pos >= 0 && pos < Sk ? documents[b * Sk + pos] : kNoCode;
    if (code < 0) code = kNoCode;
    seen = code >= 0;
    qcodes[b * qpad + i] = code;
  }
  int lo = seen ? code : INT32_MAX, hi = seen ? code : -1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off, 64));
    hi = max(hi, __shfl_xor(hi, off, 64));
  }
  const bool hidden = __builtin_amdgcn_ballot_w64(!seen) != 0;
  if (lane == 0) {
    const i32x4 s = {lo, hi, hidden ? 1 : 0, 0};
    if (keys) ktiles[b * nkt + t] = s;
    else qtiles[b * nqt + (t - nkt)] = s;
  }
}

// ---- delta = sum_d dout * out: 16 lanes per (b, i, head) row -----------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_ba_delta(const T* dout, const T* out, float* delta, int64_t rows, int Sq, int heads, int d) {
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  float s = 0.f;
  if (r < rows)
    for (int c = l * 4; c < d; c += 64) {
      float x[4], y[4];
      RowIO<T, 4>::load(dout + r * d + c, x);
      RowIO<T, 4>::load(out + r * d + c, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fmaf(x[i], y[i], s);
    }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (r < rows && l == 0) {                       // r = (b * Sq + i) * heads + head
    const int head = (int)(r % heads);
    const int64_t bi = r / heads;
    delta[((bi / Sq) * heads + head) * Sq + bi % Sq] = s;
  }
}

// What a block of 32 NW rows knows about visibility
struct View {
  int start, prefix;      // position of query 0, length of the beginning that everybody sees
  bool causal, codes, docs;
};

__device__ __forceinline__ View view_of(const BiasedArgs& a, int64_t b) {
  View v;
  v.start = clamp_start(a.q_starts ? a.q_starts[b] : a.q_start);
  v.prefix = a.prefix ? a.prefix[b] : 0;
  v.causal = a.causal != 0;
  v.codes = a.kcodes != nullptr;
  v.docs = a.qcodes != nullptr;
  return v;
}

// lowest / highest value of `code` over the wave, over lanes with code >= 0
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
  return i32x4{min(a[0], b[0]), max(a[1], b[1]), a[2] | b[2], 0};
}

// The walk of a block of queries over the keys in chunks of kChunk, shared by the forward and the dq kernel.
struct KeyWalk {
  int end;                // no query of the block sees a key at or beyond it
  int lo, hi;             // range of the block's query codes
  const i32x4* tiles;     // of this batch row, or null
  __device__ __forceinline__ int next(int kc) const {
    if (tiles != nullptr)
      while (kc < end) {
        const i32x4 t = tiles[kc / kChunk];
        if (t[1] >= lo && t[0] <= hi) break;
        kc += kChunk;
      }
    return kc;
  }
};

__device__ __forceinline__ KeyWalk key_walk(const BiasedArgs& a, const View& v, int64_t b, int row0) {
  KeyWalk w;
  w.end = a.Sk;
  if (v.causal) w.end = min(a.Sk, max(v.start + min(row0 + kRows, a.Sq), v.prefix));
  w.lo = w.hi = 0;
  w.tiles = v.codes ? a.ktiles + b * (a.kpad / 64) : nullptr;
  if (v.docs) {
    const i32x4* t = a.qtiles + b * (a.qpad / 64);
    i32x4 r = t[row0 / 64];
    if (row0 + 64 < a.Sq) r = merge(r, t[row0 / 64 + 1]);
    w.lo = r[0];
    w.hi = r[1];
  }
  return w;
}

// A tile of 32 queries (the lanes) x 32 keys (the registers): -inf where a pair is not seen
__device__ __forceinline__ void hide_keys(f32x16& sc, const View& v, int key, int rel, int Sk, const int* kc, int qcode) {
#pragma unroll
  for (int a4 = 0; a4 < 4; ++a4) {
    const i32x4 code = v.codes ? *reinterpret_cast<const i32x4*>(kc + 8 * a4) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = 8 * a4 + i;
      bool see = key + o < Sk;
      if (v.causal) see = see && (rel + o <= 0 || key + o < v.prefix);
      if (v.codes) see = see && code[i] == qcode;
      if (!see) sc[4 * a4 + i] = -INFINITY;
    }
  }
}

struct Ids {
  int64_t b;
  int head, blk;
};
// block id -> (batch row, head, block of rows).  Blocks of one head follow one another; with a causal mask the long ones
// (many keys to walk) come first.
__device__ __forceinline__ Ids ids_of(int heads, int nblk, bool last_first) {
  Ids r;
  const int64_t id = blockIdx.x;
  r.blk = (int)(id % nblk);
  if (last_first) r.blk = nblk - 1 - r.blk;
  const int64_t bh = id / nblk;
  r.head = (int)(bh % heads);
  r.b = bh / heads;
  return r;
}

// ---- forward ---------------------------------------------------------------------------------------------------------
template <typename T, int NDB>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 ? 1 : 2) void k_ba_fwd(BiasedArgs a) {
  using L = Tile<T, NDB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* kt = reinterpret_cast<T*>(smem);
  T* vt = kt + kChunk * L::PITCH;
  int* kc_lds = reinterpret_cast<int*>(vt + kChunk * L::PITCH);
  float* tab = reinterpret_cast<float*>(kc_lds + kChunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, hh = lane >> 5;
  const int nblk = (a.Sq + kRows - 1) / kRows;
  const Ids id = ids_of(a.heads, nblk, a.causal);
  const int64_t b = id.b;
  const int head = id.head, kvh = head / a.group, row0 = id.blk * kRows, q0 = row0 + 32 * wave, row = q0 + r32;
  const View v = view_of(a, b);
  const KeyWalk walk = key_walk(a, v, b, row0);
  const ScoreParams sp = score_params(a, head);
  if (sp.tab) stage_table(tab, a, head, 64 * kWaves);
  const int qpos = v.start + row;
  const int qcode = !v.docs ? 0 : row < a.qpad ? a.qcodes[b * a.qpad + row] : kNoCode;
  int qlo = 0, qhi = 0;
  bool qneg = false;                    // some row of the wave sees nothing
  if (v.docs) {
    wave_range(qcode, qlo, qhi);
    qneg = __builtin_amdgcn_ballot_w64(qcode < 0) != 0;
  }
  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const int* codes = v.codes ? a.kcodes + b * a.kpad : nullptr;
  typename Frag<T>::type qf[2 * NDB];
  load_row<T, NDB>(qf, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)row * a.qs[1] + head * a.qs[2], row < a.Sq, a.d, hh);
  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -__FLT_MAX__, l = 0.f;
  Stage<T, NDB, kWaves> sk, sv;
  int pc = 0;
  auto load = [&](int kc) {
    sk.load(kbase, a.ks[1], kc, a.Sk, a.d, codes);
    sv.load(vbase, a.vs[1], kc, a.Sk, a.d, codes);
    if (v.codes && threadIdx.x < kChunk) pc = codes[kc + threadIdx.x];
  };
  int kc = walk.next(0);
  if (kc < walk.end) load(kc);
  while (kc < walk.end) {
    __syncthreads();                    // the previous chunk has been consumed
    sk.store(kt);
    sv.store(vt);
    if (v.codes && threadIdx.x < kChunk) kc_lds[threadIdx.x] = pc;
    __syncthreads();
    const int kn = walk.next(kc + kChunk);
    if (kn < walk.end) load(kn);        // travels while this chunk is multiplied
    if (q0 < a.Sq) {                    // wave-uniform, like every branch below
#pragma unroll
      for (int t = 0; t < kChunk / 32; ++t) {
        const int key0 = kc + 32 * t;
        if (key0 >= walk.end) break;
        const int rel0 = key0 - (v.start + q0);                       // query 0 of the wave to key 0 of the tile
        const bool beyond = v.causal && rel0 > 31 && key0 >= v.prefix;
        bool clean = key0 + 32 <= a.Sk && (!v.causal || rel0 + 31 <= 0 || key0 + 32 <= v.prefix);
        bool other = false;
        if (v.codes) {
          const i32x4 ts = walk.tiles[kc / kChunk];
          other = ts[1] < qlo || ts[0] > qhi;
          clean = clean && !ts[2] && ts[0] == ts[1] && !qneg && qlo == qhi && ts[0] == qlo;
        }
        if (beyond || other) continue;
        f32x16 sc, tt;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
        for (int s = 0; s < 2 * NDB; ++s) sc = mma(L::row(kt, 32 * t + r32, s, hh), qf[s], sc);
        score_tile<T, 1, false>(sc, tt, sp, tab, key0 + 4 * hh - qpos, rel0 - 31, rel0 + 31);
        if (!clean) hide_keys(sc, v, key0 + 4 * hh, key0 + 4 * hh - qpos, a.Sk, kc_lds + 32 * t + 4 * hh, qcode);
        float tmax = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, sc[r]);
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
        // m follows the running maximum only when that has grown by more than 2^kSlack: most tiles skip the rescaling
        if (__builtin_amdgcn_ballot_w64(tmax > m + kSlack) != 0) {
          const float mn = tmax > m + kSlack ? tmax : m;
          const float alpha = __builtin_amdgcn_exp2f(m - mn);
          l *= alpha;
          m = mn;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        }
        float ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sc[r] = __builtin_amdgcn_exp2f(sc[r] - m);
          ps += sc[r];
        }
        l += ps;
        typename Frag<T>::type p0, p1;
        pack8(p0, sc, 0);
        pack8(p1, sc, 1);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          o[db] = mma(L::col(vt, 32 * t, db, lane), p0, o[db]);
          o[db] = mma(L::col(vt, 32 * t + 16, db, lane), p1, o[db]);
        }
      }
    }
    kc = kn;
  }
  l += __shfl_xor(l, 32, 64);           // the half-waves hold disjoint keys of the same query
  if (row < a.Sq) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ((b * a.Sq + row) * a.heads + head) * a.d;
    store_row<T, NDB>(static_cast<T*>(a.out) + at, o, inv, a.d, hh);
    if (a.lse && hh == 0)
      a.lse[(b * a.heads + head) * a.Sq + row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
}

// ---- backward: dq and the table's gradient ---------------------------------------------------------------------------
// The table's gradient sums ds along diagonals.  Every wave has two LDS arrays by relative distance, one per half-wave, and
// adds with ds_add_f32: the lanes of a half-wave hold 32 queries, so within one instruction they hit 32 different
// distances, and a wave's LDS instructions keep their order -- the sums have one order, from run to run.  Distances at or
// beyond R go to two registers instead.  The block then folds its eight arrays by bucket into one partial row.
//
// DELTA: the first half of the same walk, delta_i = sum_j p_ij (do_i . v_j), instead of dout . out.  Needed by the table's
// gradient on bf16 operands: the o of the forward carries the rounding of P (2^-9 of it, as does its own), which averages
// out in dq and dk but enters the few values of an fp32 dtable in full (4e-4 of their norm).
template <typename T, int NDB, bool DELTA>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 ? 1 : 2) void k_ba_dq(BiasedArgs a) {
  using L = Tile<T, NDB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* kt = reinterpret_cast<T*>(smem);
  T* vt = kt + kChunk * L::PITCH;
  int* kc_lds = reinterpret_cast<int*>(vt + kChunk * L::PITCH);
  float* tab = reinterpret_cast<float*>(kc_lds + kChunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, hh = lane >> 5;
  const int nblk = (a.Sq + kRows - 1) / kRows;
  const Ids id = ids_of(a.heads, nblk, a.causal);
  const int64_t b = id.b;
  const int head = id.head, kvh = head / a.group, row0 = id.blk * kRows, q0 = row0 + 32 * wave, row = q0 + r32;
  const View v = view_of(a, b);
  const KeyWalk walk = key_walk(a, v, b, row0);
  const ScoreParams sp = score_params(a, head);
  const int TW = 2 * a.R + 1;
  float* hist = tab + TW;                            // [2 kWaves][TW]
  float* mine = hist + (2 * wave + hh) * TW;
  const bool grad_tab = !DELTA && a.dtab != nullptr;
  if (sp.tab) stage_table(tab, a, head, 64 * kWaves);
  if (grad_tab)
    for (int i = threadIdx.x; i < 2 * kWaves * TW; i += 64 * kWaves) hist[i] = 0.f;
  const int qpos = v.start + row;
  const int qcode = !v.docs ? 0 : row < a.qpad ? a.qcodes[b * a.qpad + row] : kNoCode;
  int qlo = 0, qhi = 0;
  bool qneg = false;                    // some row of the wave sees nothing
  if (v.docs) {
    wave_range(qcode, qlo, qhi);
    qneg = __builtin_amdgcn_ballot_w64(qcode < 0) != 0;
  }
  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const int* codes = v.codes ? a.kcodes + b * a.kpad : nullptr;
  const int64_t at = ((b * a.Sq + row) * a.heads + head) * a.d, at1 = (b * a.heads + head) * a.Sq + row;
  typename Frag<T>::type qf[2 * NDB], dof[2 * NDB];
  load_row<T, NDB>(qf, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)row * a.qs[1] + head * a.qs[2], row < a.Sq, a.d, hh);
  load_row<T, NDB>(dof, static_cast<const T*>(a.dout) + at, row < a.Sq, a.d, hh);
  const float lse = row < a.Sq ? a.lse[at1] : INFINITY, delta = !DELTA && row < a.Sq ? a.delta[at1] : 0.f;
  float dsum = 0.f;
  f32x16 dq[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[db][r] = 0.f;
  float far_lo = 0.f, far_hi = 0.f;
  Stage<T, NDB, kWaves> sk, sv;
  int pc = 0;
  auto load = [&](int kc) {
    sk.load(kbase, a.ks[1], kc, a.Sk, a.d, codes);
    sv.load(vbase, a.vs[1], kc, a.Sk, a.d, codes);
    if (v.codes && threadIdx.x < kChunk) pc = codes[kc + threadIdx.x];
  };
  int kc = walk.next(0);
  if (kc < walk.end) load(kc);
  while (kc < walk.end) {
    __syncthreads();
    sk.store(kt);
    sv.store(vt);
    if (v.codes && threadIdx.x < kChunk) kc_lds[threadIdx.x] = pc;
    __syncthreads();
    const int kn = walk.next(kc + kChunk);
    if (kn < walk.end) load(kn);
    if (q0 < a.Sq) {
#pragma unroll
      for (int t = 0; t < kChunk / 32; ++t) {
        const int key0 = kc + 32 * t;
        if (key0 >= walk.end) break;
        const int rel0 = key0 - (v.start + q0);
        const bool beyond = v.causal && rel0 > 31 && key0 >= v.prefix;
        bool clean = key0 + 32 <= a.Sk && (!v.causal || rel0 + 31 <= 0 || key0 + 32 <= v.prefix);
        bool other = false;
        if (v.codes) {
          const i32x4 ts = walk.tiles[kc / kChunk];
          other = ts[1] < qlo || ts[0] > qhi;
          clean = clean && !ts[2] && ts[0] == ts[1] && !qneg && qlo == qhi && ts[0] == qlo;
        }
        if (beyond || other) continue;
        f32x16 sc, dp, tt;
#pragma unroll
        for (int r = 0; r < 16; ++r) { sc[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int s = 0; s < 2 * NDB; ++s) {
          sc = mma(L::row(kt, 32 * t + r32, s, hh), qf[s], sc);
          dp = mma(L::row(vt, 32 * t + r32, s, hh), dof[s], dp);
        }
        const int rel = key0 + 4 * hh - qpos;
        score_tile<T, 1, !DELTA>(sc, tt, sp, tab, rel, rel0 - 31, rel0 + 31);
        if (!clean) hide_keys(sc, v, key0 + 4 * hh, rel, a.Sk, kc_lds + 32 * t + 4 * hh, qcode);
        if (DELTA) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dsum = fmaf(__builtin_amdgcn_exp2f(sc[r] - lse), dp[r], dsum);
          continue;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = __builtin_amdgcn_exp2f(sc[r] - lse) * (dp[r] - delta);     // ds
        if (grad_tab) {
          const int lo = rel0 - 31, hi = rel0 + 31;
          if (hi <= -a.R || lo >= a.R) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) s += sc[r];
            if (hi <= -a.R) far_lo += s;
            else far_hi += s;
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int x = rel + acc_row(r);
              if (x <= -a.R) far_lo += sc[r];
              else if (x >= a.R) far_hi += sc[r];
              else __builtin_amdgcn_ds_faddf((__attribute__((address_space(3))) float*)(mine + x + a.R), sc[r], 0, 0, false);
            }
          }
        }
        if (sp.cap) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[r] *= 1.f - tt[r] * tt[r];
        }
        typename Frag<T>::type d0, d1;
        pack8(d0, sc, 0);
        pack8(d1, sc, 1);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dq[db] = mma(L::col(kt, 32 * t, db, lane), d0, dq[db]);
          dq[db] = mma(L::col(kt, 32 * t + 16, db, lane), d1, dq[db]);
        }
      }
    }
    kc = kn;
  }
  if (DELTA) {
    dsum += __shfl_xor(dsum, 32, 64);
    if (row < a.Sq && hh == 0) a.delta[at1] = dsum;
    return;
  }
  if (row < a.Sq && a.dq) store_row<T, NDB>(static_cast<T*>(a.dq) + at, dq, a.scale, a.d, hh);
  if (grad_tab) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      far_lo += __shfl_xor(far_lo, off, 64);
      far_hi += __shfl_xor(far_hi, off, 64);
    }
    __syncthreads();          // the arrays are zeroed also where no chunk was walked
    if (r32 == 0) {
      mine[0] = far_lo;
      mine[2 * a.R] = far_hi;
    }
    __syncthreads();
    int* ids = reinterpret_cast<int*>(tab);
    for (int i = threadIdx.x; i < TW; i += 64 * kWaves) {
      float s = 0.f;
      for (int w = 0; w < 2 * kWaves; ++w) s += hist[w * TW + i];
      hist[i] = s;
      ids[i] = min(max(a.buckets[i], 0), a.nb - 1);
    }
    __syncthreads();
    for (int n = threadIdx.x; n < a.nb; n += 64 * kWaves) {
      float s = 0.f;
      for (int i = 0; i < TW; ++i) s += ids[i] == n ? hist[i] : 0.f;
      a.dtab[((int64_t)head * a.B * nblk + b * nblk + id.blk) * a.nb + n] = s;
    }
  }
}

// dtable[n][head] = sum of the partials of head, in a fixed order; one wave per (head, bucket)
__global__ __launch_bounds__(64) void k_ba_dtable(const float* part, float* dtable, int64_t blocks, int nb, int heads) {
  const int head = blockIdx.x % heads, n = blockIdx.x / heads;
  double s = 0.0;             // up to 2^20 partials of either sign
  for (int64_t i = threadIdx.x; i < blocks; i += 64) s += (double)part[(head * blocks + i) * nb + n];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (threadIdx.x == 0) dtable[(int64_t)n * heads + head] = (float)s;
}

// ---- backward: dk and dv ---------------------------------------------------------------------------------------------
template <typename T, int NDB>
__global__ __launch_bounds__(64 * kWaves, NDB >= 3 || sizeof(T) == 4 ? 1 : 2) void k_ba_dkv(BiasedArgs a) {
  using L = Tile<T, NDB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* qt = reinterpret_cast<T*>(smem);
  T* dt = qt + kChunk * L::PITCH;
  float* lses = reinterpret_cast<float*>(dt + kChunk * L::PITCH);
  float* dels = lses + kChunk;
  int* qc_lds = reinterpret_cast<int*>(dels + kChunk);
  float* tab = reinterpret_cast<float*>(qc_lds + kChunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, hh = lane >> 5;
  const int nblk = (a.Sk + kRows - 1) / kRows;
  const Ids id = ids_of(a.kv, nblk, false);
  const int64_t b = id.b;
  const int kvh = id.head, row0 = id.blk * kRows, k0 = row0 + 32 * wave, key = k0 + r32;
  const View v = view_of(a, b);
  const bool ok = key < a.Sk;
  const int kcode = !ok ? -1 : v.codes ? a.kcodes[b * a.kpad + key] : 0;
  int klo = 0, khi = 0;
  bool khid = k0 + 32 > a.Sk;
  if (v.codes) {
    wave_range(kcode, klo, khi);
    khid = __builtin_amdgcn_ballot_w64(kcode < 0) != 0;
  }
  // the block's first query chunk and range of key codes
  int qfirst = 0;
  if (v.causal && row0 >= v.prefix) qfirst = max(0, row0 - v.start) / kChunk * kChunk;
  i32x4 br = {0, 0, 0, 0};
  if (v.codes) {
    const i32x4* t = a.ktiles + b * (a.kpad / 64);
    br = t[row0 / 64];
    if (row0 + 64 < a.Sk) br = merge(br, t[row0 / 64 + 1]);
  }
  const i32x4* qtiles = v.docs ? a.qtiles + b * (a.qpad / 64) : nullptr;
  auto next = [&](int qc) {
    if (v.codes && !v.docs && br[1] < 0) return a.Sq;              // every key of the block is hidden
    if (qtiles != nullptr)
      while (qc < a.Sq) {
        const i32x4 t = qtiles[qc / kChunk];
        if (t[1] >= br[0] && t[0] <= br[1]) break;
        qc += kChunk;
      }
    return qc;
  };
  typename Frag<T>::type kf[2 * NDB], vf[2 * NDB];
  load_row<T, NDB>(kf, static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)key * a.ks[1] + kvh * a.ks[2], kcode >= 0, a.d, hh);
  load_row<T, NDB>(vf, static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)key * a.vs[1] + kvh * a.vs[2], kcode >= 0, a.d, hh);
  f32x16 dk[NDB], dv[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[db][r] = 0.f; dv[db][r] = 0.f; }
  Stage<T, NDB, kWaves> sq, sd;
  float pl = 0.f, pd = 0.f;
  int pq = 0;
  auto load = [&](int head, int qc) {
    sq.load(static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[2], a.qs[1], qc, a.Sq, a.d, nullptr);
    sd.load(static_cast<const T*>(a.dout) + (b * a.Sq * a.heads + head) * a.d, (int64_t)a.heads * a.d, qc, a.Sq, a.d, nullptr);
    const int i = qc + (int)threadIdx.x;
    const bool in = threadIdx.x < kChunk && i < a.Sq;
    pl = in ? a.lse[(b * a.heads + head) * a.Sq + i] : INFINITY;    // rows beyond Sq: p = exp2(. - inf) = 0
    pd = in ? a.delta[(b * a.heads + head) * a.Sq + i] : 0.f;
    if (v.docs && threadIdx.x < kChunk) pq = a.qcodes[b * a.qpad + i];
  };
  for (int g = 0; g < a.group; ++g) {
    const int head = kvh * a.group + g;
    const ScoreParams sp = score_params(a, head);
    __syncthreads();                    // the last chunk of the previous head has been consumed
    if (sp.tab) stage_table(tab, a, head, 64 * kWaves);
    int qc = next(qfirst);
    if (qc < a.Sq) load(head, qc);
    while (qc < a.Sq) {
      __syncthreads();
      sq.store(qt);
      sd.store(dt);
      if (threadIdx.x < kChunk) {
        lses[threadIdx.x] = pl;
        dels[threadIdx.x] = pd;
        qc_lds[threadIdx.x] = pq;
      }
      __syncthreads();
      const int qn = next(qc + kChunk);
      if (qn < a.Sq) load(head, qn);
      if (k0 < a.Sk) {
#pragma unroll
        for (int t = 0; t < kChunk / 32; ++t) {
          const int q0 = qc + 32 * t;
          if (q0 >= a.Sq) break;
          const int rel0 = k0 - (v.start + q0);             // query 0 of the tile to key 0 of the wave
          const bool beyond = v.causal && rel0 > 31 && k0 >= v.prefix;
          bool clean = !khid && (!v.causal || rel0 + 31 <= 0 || k0 + 32 <= v.prefix);
          bool other = v.codes && khi < 0;
          if (v.docs) {
            const i32x4 ts = qtiles[qc / kChunk];
            other = ts[1] < klo || ts[0] > khi;
            clean = clean && !ts[2] && ts[0] == ts[1] && klo == khi && ts[0] == klo;
          } else if (v.codes) {
            clean = clean && klo == khi;
          }
          if (beyond || other) continue;
          f32x16 sc, dp, tt;
#pragma unroll
          for (int r = 0; r < 16; ++r) { sc[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
          for (int s = 0; s < 2 * NDB; ++s) {
            sc = mma(L::row(qt, 32 * t + r32, s, hh), kf[s], sc);
            dp = mma(L::row(dt, 32 * t + r32, s, hh), vf[s], dp);
          }
          const int rel = key - (v.start + q0 + 4 * hh);    // register r: rel - acc_row(r)
          score_tile<T, -1, true>(sc, tt, sp, tab, rel, rel0 - 31, rel0 + 31);
          if (!clean) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              bool see = kcode >= 0;
              if (v.causal) see = see && (rel - acc_row(r) <= 0 || key < v.prefix);
              if (v.docs) see = see && qc_lds[32 * t + 4 * hh + acc_row(r)] == kcode;
              if (!see) sc[r] = -INFINITY;
            }
          }
#pragma unroll
          for (int a4 = 0; a4 < 4; ++a4) {
            const f32x4 ls = *reinterpret_cast<const f32x4*>(lses + 32 * t + 8 * a4 + 4 * hh);
            const f32x4 de = *reinterpret_cast<const f32x4*>(dels + 32 * t + 8 * a4 + 4 * hh);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 4 * a4 + i;
              sc[r] = __builtin_amdgcn_exp2f(sc[r] - ls[i]);
              dp[r] = sc[r] * (dp[r] - de[i]);
              if (sp.cap) dp[r] *= 1.f - tt[r] * tt[r];
            }
          }
          typename Frag<T>::type p0, p1, d0, d1;
          pack8(p0, sc, 0);
          pack8(p1, sc, 1);
          pack8(d0, dp, 0);
          pack8(d1, dp, 1);
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            dv[db] = mma(L::col(dt, 32 * t, db, lane), p0, dv[db]);
            dv[db] = mma(L::col(dt, 32 * t + 16, db, lane), p1, dv[db]);
            dk[db] = mma(L::col(qt, 32 * t, db, lane), d0, dk[db]);
            dk[db] = mma(L::col(qt, 32 * t + 16, db, lane), d1, dk[db]);
          }
        }
      }
      qc = qn;
    }
  }
  if (ok) {
    const int64_t at = ((b * a.Sk + key) * a.kv + kvh) * a.d;
    store_row<T, NDB>(static_cast<T*>(a.dk) + at, dk, a.scale, a.d, hh);
    store_row<T, NDB>(static_cast<T*>(a.dv) + at, dv, 1.f, a.d, hh);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int64_t pad64(int64_t n) { return (n + 63) / 64 * 64; }
size_t tile_bytes(int es, int ndb) {
  const int pitch = es == 4 ? 32 * ndb + 4 : (ndb == 1 || ndb == 3 ? 32 * ndb : 32 * ndb + 32);
  return (size_t)2 * kChunk * pitch * es;
}

enum Which { kFwd, kDelta, kDq, kDkv };

template <typename T, int NDB>
void launch(Which which, const BiasedArgs& a, dim3 grid, size_t lds, hipStream_t st) {
  void (*fn)(BiasedArgs) = which == kFwd   ? k_ba_fwd<T, NDB>
                           : which == kDq  ? k_ba_dq<T, NDB, false>
                           : which == kDkv ? k_ba_dkv<T, NDB>
                                           : k_ba_dq<unsigned short, NDB, true>;
  if (lds > 64 * 1024)        // at most 141 KiB: fp32 heads of 128, a table gradient over 2049 distances
    (void)hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL(fn, grid, dim3(64 * kWaves), lds, st, a);
}

void dispatch(Which which, int dtype, const BiasedArgs& a, dim3 grid, size_t lds, hipStream_t st) {
  const int ndb = (a.d + 31) / 32;
  if (dtype == MIVAE_F32) switch (ndb) {
      case 1: return launch<float, 1>(which, a, grid, lds, st);
      case 2: return launch<float, 2>(which, a, grid, lds, st);
      case 3: return launch<float, 3>(which, a, grid, lds, st);
      default: return launch<float, 4>(which, a, grid, lds, st);
    }
  switch (ndb) {
    case 1: return launch<unsigned short, 1>(which, a, grid, lds, st);
    case 2: return launch<unsigned short, 2>(which, a, grid, lds, st);
    case 3: return launch<unsigned short, 3>(which, a, grid, lds, st);
    default: return launch<unsigned short, 4>(which, a, grid, lds, st);
  }
}

int set_args(BiasedArgs& a, const mivae_attention_args* x, const char* name) {
  MIVAE_REQUIRE(x != nullptr, "%s: null arguments", name);
  MIVAE_REQUIRE(x->dtype == MIVAE_F32 || x->dtype == MIVAE_BF16, "%s: dtype %d is neither float32 nor bfloat16", name, x->dtype);
  MIVAE_REQUIRE(x->batch >= 1 && x->q_len >= 1 && x->k_len >= 1 && x->q_len <= (1 << 24) && x->k_len <= (1 << 24),
                "%s: batch %lld, lengths %lld and %lld: at least 1, lengths at most 2^24", name, (long long)x->batch,
                (long long)x->q_len, (long long)x->k_len);
  MIVAE_REQUIRE(x->heads >= 1 && x->kv_heads >= 1 && x->heads % x->kv_heads == 0 && x->heads <= 65535,
                "%s: %lld heads over %lld key heads", name, (long long)x->heads, (long long)x->kv_heads);
  MIVAE_REQUIRE(x->head_size >= 8 && x->head_size <= 128 && x->head_size % 8 == 0,
                "%s: head size %lld is not a multiple of 8 in 8 .. 128", name, (long long)x->head_size);
  const int64_t per16 = x->dtype == MIVAE_F32 ? 4 : 8;
  const int64_t* st[3] = {x->q_stride, x->k_stride, x->v_stride};
  for (int t = 0; t < 3; ++t)
    for (int i = 0; i < 3; ++i)
      MIVAE_REQUIRE(st[t][i] >= 0 && st[t][i] % per16 == 0 && st[t][i] < (1ll << 40),
                    "%s: stride %lld is negative or does not keep rows 16-byte aligned", name, (long long)st[t][i]);
  MIVAE_REQUIRE(x->q && x->k && x->v, "%s: null operand", name);
  MIVAE_REQUIRE(aligned16(x->q) && aligned16(x->k) && aligned16(x->v), "%s: q / k / v must be 16-byte aligned", name);
  MIVAE_REQUIRE(!(x->prefix && !x->causal), "%s: a prefix needs the causal mask", name);
  MIVAE_REQUIRE(x->softcap >= 0.f && x->softcap < 1e30f && x->scale > -1e30f && x->scale < 1e30f,
                "%s: softcap or scale out of range", name);
  MIVAE_REQUIRE(!(x->slopes && x->table), "%s: slopes and a table are alternatives", name);
  if (x->table)
    MIVAE_REQUIRE(x->buckets && x->num_buckets >= 1 && x->num_buckets <= kMaxBuckets && x->distance >= 1 && x->distance <= kMaxDistance,
                  "%s: %lld buckets up to distance %lld: 1 .. %d buckets, distance 1 .. %d", name, (long long)x->num_buckets,
                  (long long)x->distance, kMaxBuckets, kMaxDistance);
  MIVAE_REQUIRE(x->q_starts || (x->q_start >= 0 && x->q_start <= (1 << 24)), "%s: q_start %lld out of range", name, (long long)x->q_start);
  MIVAE_REQUIRE(!(x->mask || x->documents) || (x->codes && aligned16(x->codes)), "%s: a mask or documents need the codes buffer", name);
  a.q = x->q; a.k = x->k; a.v = x->v;
  for (int i = 0; i < 3; ++i) { a.qs[i] = x->q_stride[i]; a.ks[i] = x->k_stride[i]; a.vs[i] = x->v_stride[i]; }
  a.out = x->out; a.lse = x->lse;
  a.B = (int)x->batch; a.Sq = (int)x->q_len; a.Sk = (int)x->k_len; a.heads = (int)x->heads; a.kv = (int)x->kv_heads;
  a.group = a.heads / a.kv; a.d = (int)x->head_size;
  a.q_start = (int)x->q_start; a.q_starts = x->q_starts; a.prefix = x->prefix; a.causal = x->causal ? 1 : 0;
  a.slopes = x->slopes; a.table = x->table; a.buckets = x->buckets;
  a.nb = (int)x->num_buckets; a.R = x->table ? (int)x->distance : 0;
  a.scale = x->scale; a.cap = x->softcap;
  a.kpad = (int)pad64(a.Sk); a.qpad = (int)pad64(a.Sq);
  const int64_t nq = (x->batch * x->heads) * ((a.Sq + kRows - 1) / kRows), nk = (x->batch * x->kv_heads) * ((a.Sk + kRows - 1) / kRows);
  MIVAE_REQUIRE(x->batch <= (1 << 24) && nq < (1ll << 31) && nk < (1ll << 31) && x->batch * (a.kpad + a.qpad) / 256 < (1ll << 31),
                "%s: too many blocks", name);
  if (x->mask || x->documents) {          // [codes][key tiles], and with documents the same of the queries
    int* p = static_cast<int*>(x->codes);
    a.kcodes = p;
    p += x->batch * a.kpad;
    a.ktiles = reinterpret_cast<const i32x4*>(p);
    p += x->batch * a.kpad / 16;
    if (x->documents) {
      a.qcodes = p;
      p += x->batch * a.qpad;
      a.qtiles = reinterpret_cast<const i32x4*>(p);
    }
  }
  return MIVAE_OK;
}

}  // namespace

extern "C" {

int64_t mivae_biased_attention_codes_ints(int64_t batch, int64_t q_len, int64_t k_len, int documents) {
  return batch * (pad64(k_len) + (documents ? pad64(q_len) : 0)) / 16 * 17;
}

int64_t mivae_biased_attention_bwd_floats(int64_t batch, int64_t q_len, int64_t heads, int64_t num_buckets) {
  const int64_t nblk = (q_len + kRows - 1) / kRows;
  return batch * heads * q_len + batch * heads * nblk * num_buckets;
}

int mivae_biased_attention_fwd(const mivae_attention_args* x, void* stream) {
  BiasedArgs a = {};
  const int rc = set_args(a, x, "mivae_biased_attention_fwd");
  if (rc != MIVAE_OK) return rc;
  MIVAE_REQUIRE(x->out && aligned16(x->out), "mivae_biased_attention_fwd: out must be a 16-byte aligned buffer");
  if (a.kcodes) {
    const int64_t waves = (int64_t)a.B * (a.kpad + (x->documents ? a.qpad : 0)) / 64;
    hipLaunchKernelGGL(k_ba_codes, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, S_(stream), x->mask, x->documents,
                       a.q_starts, a.q_start, a.B, a.Sq, a.Sk, a.kpad, a.qpad, const_cast<int*>(a.kcodes),
                       const_cast<int*>(a.qcodes), const_cast<i32x4*>(a.ktiles), const_cast<i32x4*>(a.qtiles));
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_fwd (codes)");
  }
  const int ndb = (a.d + 31) / 32, es = x->dtype == MIVAE_F32 ? 4 : 2;
  const size_t lds = tile_bytes(es, ndb) + kChunk * 4 + (a.table ? (2 * a.R + 1) * 4 : 0);
  const dim3 grid((unsigned)((int64_t)a.B * a.heads * ((a.Sq + kRows - 1) / kRows)));
  dispatch(kFwd, x->dtype, a, grid, lds, S_(stream));
  MIVAE_CHECK_LAUNCH("mivae_biased_attention_fwd");
  return MIVAE_OK;
}

int mivae_biased_attention_bwd(const mivae_attention_args* x, void* stream) {
  BiasedArgs a = {};
  const int rc = set_args(a, x, "mivae_biased_attention_bwd");
  if (rc != MIVAE_OK) return rc;
  MIVAE_REQUIRE(x->out && x->dout && x->lse && x->scratch, "mivae_biased_attention_bwd: null operand");
  MIVAE_REQUIRE((x->dk == nullptr) == (x->dv == nullptr), "mivae_biased_attention_bwd: dk and dv are written together");
  MIVAE_REQUIRE(!x->dtable || x->table, "mivae_biased_attention_bwd: dtable without a table");
  MIVAE_REQUIRE(aligned16(x->out) && aligned16(x->dout) && aligned16(x->dq) && aligned16(x->dk) && aligned16(x->dv),
                "mivae_biased_attention_bwd: out / dout / dq / dk / dv must be 16-byte aligned");
  const int64_t rows = (int64_t)a.B * a.Sq * a.heads;
  MIVAE_REQUIRE(rows / 16 < (1ll << 31), "mivae_biased_attention_bwd: too many rows");
  a.dout = x->dout;
  a.dq = x->dq; a.dk = x->dk; a.dv = x->dv;
  a.delta = x->scratch;
  a.dtab = x->dtable ? x->scratch + rows : nullptr;
  hipStream_t st = S_(stream);
  const int ndb = (a.d + 31) / 32, es = x->dtype == MIVAE_F32 ? 4 : 2;
  const size_t tiles = tile_bytes(es, ndb), tw = a.table ? 2 * a.R + 1 : 0;
  const int nblk = (a.Sq + kRows - 1) / kRows;
  const dim3 grid((unsigned)((int64_t)a.B * a.heads * nblk)), dgrid((unsigned)((rows + 15) / 16));
  if (es == 4)
    hipLaunchKernelGGL((k_ba_delta<float>), dgrid, dim3(256), 0, st, static_cast<const float*>(x->dout),
                       static_cast<const float*>(x->out), a.delta, rows, a.Sq, a.heads, a.d);
  else if (!a.dtab)
    hipLaunchKernelGGL((k_ba_delta<unsigned short>), dgrid, dim3(256), 0, st, static_cast<const unsigned short*>(x->dout),
                       static_cast<const unsigned short*>(x->out), a.delta, rows, a.Sq, a.heads, a.d);
  else
    dispatch(kDelta, x->dtype, a, grid, tiles + (kChunk + tw) * 4, st);
  MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (delta)");
  if (a.dq || a.dtab) {
    const size_t lds = tiles + kChunk * 4 + (tw + (a.dtab ? 2 * kWaves * tw : 0)) * 4;
    dispatch(kDq, x->dtype, a, grid, lds, st);
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dq)");
    if (a.dtab) {
      hipLaunchKernelGGL(k_ba_dtable, dim3((unsigned)(a.heads * a.nb)), dim3(64), 0, st, a.dtab, x->dtable, (int64_t)a.B * nblk,
                         a.nb, a.heads);
      MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dtable)");
    }
  }
  if (a.dk) {
    const size_t lds = tiles + 3 * kChunk * 4 + tw * 4;
    const dim3 grid((unsigned)((int64_t)a.B * a.kv * ((a.Sk + kRows - 1) / kRows)));
    dispatch(kDkv, x->dtype, a, grid, lds, st);
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dk, dv)");
  }
  return MIVAE_OK;
}

}  // extern "C"
