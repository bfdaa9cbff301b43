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
// products, which is what lets them run on the bf16 matrix instruction.  That is one rounding more than the result's own: errors
// relative to the norm 2.3e-3 (outputs without gradients, or with the table's) and 2.35e-3 (gradients) where the result's alone
// leaves 1.66e-3.  Second bf16 values for what they leave reach 1.66e-3 everywhere and were measured: for P in the forward
// 535 us instead of 470 (8191 queries of 128), for P and dS in all products 460 instead of 420 (documents), 549 instead of 439
// (64 x 512, table), 1482 instead of 1220 (4 x 4096, table).  They are kept where the error grows or stays for good: P where few
// keys carry a row (k_ba_fwd), the output for delta (out_lo), delta of the table's gradient (kDelta), dS of up to 16 columns.
//
// Bound: fp32 by its matrix instructions (55 - 64 % busy), the bf16 forward by the VALU (a score costs an exponential, with a cap
// a tanh, and two conversions: issued in 75 - 84 % of the cycles of long walks).  The bf16 backward fills neither (long walks: dq VALU
// 59 - 62 %, dk and dv 45 - 48 %, matrix cores 11 - 26 %): at 177 - 256 registers two waves share a SIMD and wait together.
//   8191 causal queries of 16 + 4 heads of 128 with a cap, no gradient: 470 us, 585 TFLOP/s
//   4 x 4096, 16 + 4 heads of 64, causal, a table and its gradient: forward 212 us, delta 202, dq 354, dk and dv 440
//   4 x 4096 in documents of 600, 16 heads of 64, a cap: forward 106 us, dq 129, dk and dv 174
//   4 x 1001, 8 + 2 heads of 80, fp32, a prefix and slopes: forward 109 us, dq 134, dk and dv 183, joining the parts 29
#include <type_traits>

#include "att_tiles.hpp"
#include "mivae.h"
#include "token_attention.hpp"

using namespace mivae;

namespace {

static inline hipStream_t S_(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr float kSlack = 8.f;       // exponent slack before the accumulators are rescaled
constexpr int kWaves = 4, kRows = 32 * kWaves;      // rows (queries or keys) of a block
constexpr int kMaxDistance = 1024, kMaxBuckets = 256;

// ---- visibility codes ------------------------------------------------------------------------------------------------
// One wave per 64 keys (or queries): code per row and {lowest, highest visible code, visible rows as 64 bits} per 64 rows.
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
  const uint64_t rows = __builtin_amdgcn_ballot_w64(seen);
  if (lane == 0) {
    const i32x4 s = {lo, hi, (int)(unsigned)rows, (int)(unsigned)(rows >> 32)};
    if (keys) ktiles[b * nkt + t] = s;
    else qtiles[b * nqt + (t - nkt)] = s;
  }
}

// Backward: the summaries of the queries anew, with only the rows that see a key, i.e. whose maximum is finite for some head.  dk and dv stage no others: whatever a blind row and its gradient hold must not meet a product, 0 * NaN is NaN.
__global__ __launch_bounds__(256) void k_ba_sighted(const float* lse, const int* qcodes, int B, int Sq, int qpad, int heads, i32x4* tiles) {
  const int n = qpad / 64, lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)B * n) return;
  const int64_t b = w / n;
  const int i = (int)(w % n) * 64 + lane;
  bool sees = false;
  if (i < Sq)
    for (int h = 0; h < heads; ++h) sees |= !(lse[(b * heads + h) * Sq + i] == INFINITY);
  int lo, hi;
  wave_range(!sees ? -1 : qcodes ? qcodes[b * qpad + i] : 0, lo, hi);
  const uint64_t rows = __builtin_amdgcn_ballot_w64(sees);
  if (lane == 0) tiles[w] = i32x4{lo, hi, (int)(unsigned)rows, (int)(unsigned)(rows >> 32)};
}

// ---- delta = sum_d dout * out where dk and dv alone are asked for (else the dq kernel forms it): 16 lanes per (b, i, head) row -----------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void k_ba_delta(const T* dout, const T* out, const unsigned short* lo, float* delta, int64_t rows, int Sq, int heads, int d) {
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
      if (lo != nullptr) {
        RowIO<unsigned short, 4>::load(lo + r * d + c, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(x[i], y[i], s);
      }
    }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (r < rows && l == 0) {                       // r = (b * Sq + i) * heads + head
    const int head = (int)(r % heads);
    const int64_t bi = r / heads;
    delta[((bi / Sq) * heads + head) * Sq + bi % Sq] = s;
  }
}

// ---- what a block knows about visibility -------------------------------------------------------------------------------
// The chunks of kChunk rows of a batch row that a block has to walk: all of them, or with codes those whose range of codes meets
// the block's.  A wave looks at the summaries of 64 chunks at once, one per lane, and keeps them: one load per 4096 rows (chunk
// after chunk, a block far down a row of packed documents waited for up to 60 loads in a row before its first product).
struct Walk {
  const i32x4* tiles;     // summaries of this batch row, or null
  int end;                // the limit of the walk
  int lo, hi;             // range of the block's codes
  int base;
  i32x4 mine;
  uint64_t meets;
  __device__ __forceinline__ void init(const i32x4* t, int limit, int low, int high) {
    tiles = t; end = limit; lo = low; hi = high;
    base = -64;
    meets = 0;
    mine = i32x4{0, 0, 0, 0};
  }
  // keeps part i of n equal ones (in chunks) of the walk; its first row
  __device__ __forceinline__ int take(int i, int n) {
    const int chunks = (end + kChunk - 1) / kChunk, from = chunks * i / n * kChunk;
    end = min(end, chunks * (i + 1) / n * kChunk);
    return from;
  }
  // first chunk at or behind row c that counts, or something >= end; its summary, with only the rows before `end`: what keys
  // behind every query's limit hold (the rest of a cache) must not meet a product.  All lanes of the wave have to be active.
  __device__ __forceinline__ int next(int c, i32x4& info) {
    if (tiles == nullptr) {
      const uint64_t rows = low_rows(end - c);
      info = i32x4{0, 0, (int)(unsigned)rows, (int)(unsigned)(rows >> 32)};
      return c;
    }
    while (c < end) {
      const int t = c / kChunk;
      if (t >= base + 64 || t < base) {
        base = t & ~63;
        const int at = base + (int)(threadIdx.x & 63);
        const bool in = at * kChunk < end;
        mine = in ? tiles[at] : i32x4{INT32_MAX, -1, 0, 0};
        meets = __builtin_amdgcn_ballot_w64(in && mine[1] >= lo && mine[0] <= hi);
      }
      const uint64_t left = meets >> (t - base);
      if (left != 0) {
        const int at = t - base + __builtin_ctzll(left);
#pragma unroll
        for (int i = 0; i < 4; ++i) info[i] = __builtin_amdgcn_readlane(mine[i], at);
        c = (base + at) * kChunk;
        const uint64_t rows = low_rows(end - c);
        info[2] &= (int)(unsigned)rows;
        info[3] &= (int)(unsigned)(rows >> 32);
        return c;
      }
      c = (base + 64) * kChunk;
    }
    return c;
  }
};

// codes of the block's rows [row0, row0 + kRows), from the summaries of n rows
__device__ __forceinline__ void block_range(const i32x4* tiles, int row0, int n, int& lo, int& hi) {
  i32x4 r = tiles[row0 / 64];
  if (row0 + 64 < n) {
    const i32x4 t = tiles[row0 / 64 + 1];
    r[0] = min(r[0], t[0]);
    r[1] = max(r[1], t[1]);
  }
  lo = r[0];
  hi = r[1];
}

__device__ __forceinline__ Walk key_walk(const BiasedArgs& a, const View& v, int64_t b, int row0) {
  Walk w;
  int lo = 0, hi = 0;
  if (v.docs) block_range(a.qtiles + b * (a.qpad / 64), row0, a.Sq, lo, hi);
  w.init(v.codes ? a.ktiles + b * (a.kpad / 64) : nullptr, v.limit(min(row0 + kRows, a.Sq) - 1), lo, hi);
  return w;
}

// What a wave of 32 queries (one per lane, both half-waves the same) sees of a chunk
struct QueryWave {
  int row, limit;               // the lane's query
  int first, last;              // limits of the wave's first and last query
  int code, lo, hi;             // the lane's code and the wave's range
  bool none, codes;             // some lane's query sees nothing; pairs are compared by codes
  // 0: nothing of the chunk, 1: its pairs below the limit, 2: those of equal codes too, 3: all of them
  __device__ __forceinline__ int sees(int kc, const i32x4& t) const {
    if (kc >= last || t[1] < lo || t[0] > hi) return 0;
    if (rows_of(t) != ~0ull || none || lo != hi || t[0] != lo || t[1] != lo) return codes ? 2 : 1;
    return kc + kChunk <= first ? 3 : 1;
  }
};

__device__ __forceinline__ QueryWave query_wave(const BiasedArgs& a, const View& v, int64_t b, int q0, int r32) {
  QueryWave w;
  w.row = q0 + r32;
  w.limit = v.limit(w.row);
  w.first = v.limit(q0);
  w.last = q0 < a.Sq ? v.limit(min(q0 + 32, a.Sq) - 1) : 0;
  w.code = w.lo = w.hi = 0;
  w.none = false;
  w.codes = v.codes;
  if (v.docs) {
    w.code = w.row < a.qpad ? a.qcodes[b * a.qpad + w.row] : kNoCode;
    wave_range(w.code, w.lo, w.hi);
    w.none = __builtin_amdgcn_ballot_w64(w.code < 0) != 0;
  }
  return w;
}

// lane: query, registers: keys key0 + 4 hh + acc_row(r)
__device__ __forceinline__ void hide_keys(f32x16& u, const QueryWave& w, bool codes, int key, const int* kc) {
  const int lim = w.limit - key;
  if (!codes) {
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = acc_row(r) < lim ? u[r] : -INFINITY;
  } else {
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) {
      const i32x4 code = *reinterpret_cast<const i32x4*>(kc + 8 * a4);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[4 * a4 + i] = 8 * a4 + i < lim && code[i] == w.code ? u[4 * a4 + i] : -INFINITY;
    }
  }
}

struct Ids {
  int64_t b;
  int head, blk;
  bool none;
};
// Block id -> (batch row, head, block of rows).  Blocks go round the eight XCDs, each with an L2 of its own.
//   From 32 (batch row, head) pairs, or a multiple of 8, on: an XCD takes a contiguous run of pairs, so that the blocks of a
//   pair (and the heads of a group) read their keys through one L2.  The grid is rounded up to a multiple of 8; ids beyond
//   the last pair do nothing.  (64 x 512 tokens, 4 heads of 128: 69 instead of 133 us forward.)
//   Fewer pairs, or a causal mask over pairs that do not divide by 8: the position is the slow index, which spreads every
//   pair over the XCDs.
// A causal mask makes the blocks' walks unequal: the longest (last queries, first keys) start first, over as many pairs at a
// time as keep an XCD's 32 CUs busy four times over, and the short ones fill the end.  (4 x 16 x 4096 queries: 263
// instead of 317 us forward with pair after pair.)
__host__ __device__ __forceinline__ bool by_xcd(int64_t pairs, bool causal) { return pairs % 8 == 0 || (!causal && pairs >= 32); }
int64_t grid_of(int64_t pairs, int64_t nblk, bool causal) { return by_xcd(pairs, causal) ? (pairs * nblk + 7) / 8 * 8 : pairs * nblk; }

__device__ __forceinline__ Ids ids_of(int B, int heads, int nblk, bool causal, bool last_first) {
  Ids r;
  const unsigned pairs = (unsigned)B * (unsigned)heads, n = (unsigned)nblk;
  unsigned bh;
  r.none = false;
  if (by_xcd(pairs, causal)) {
    const unsigned x = blockIdx.x & 7, i = blockIdx.x >> 3, each = gridDim.x >> 3;
    if (causal) {
      const unsigned mine = pairs / 8, most = min(mine, (255 + n) / n), g = i / (most * n), j = i % (most * n);
      const unsigned size = min(most, mine - g * most);
      bh = x * mine + g * most + j % size;
      r.blk = (int)(j / size);
    } else {
      const unsigned w = x * each + i;
      bh = w / n;
      r.blk = (int)(w % n);
      r.none = bh >= pairs;
    }
  } else {
    r.blk = (int)(blockIdx.x / pairs);
    bh = blockIdx.x % pairs;
  }
  if (last_first) r.blk = nblk - 1 - r.blk;
  r.head = (int)(bh % (unsigned)heads);
  r.b = bh / (unsigned)heads;
  return r;
}

// ---- forward ---------------------------------------------------------------------------------------------------------
// kInfer: no lse, bf16 with the rough tanh (a cap above kRoughCap takes kTrain, which then leaves no lse).  kTrain: lse.
// kTrainRest (bf16): also the rounding's rest of large probabilities and the output's residue, for delta = dout . out.
// (Modes, not branches: a branch between the products and the exponentials of a chunk keeps them from overlapping, 7 % at
// 8191 queries of 128.)
enum Mode { kInfer, kTrain, kTrainRest };

// slices > 1: a block takes one of that many equal parts of its rows' walk and leaves (O, max, sum) in `part`, laid out for
// token_attention_join.
template <typename T, int NDB, Mode MODE>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 ? 1 : 2) void k_ba_fwd(BiasedArgs a, int slices, float* part) {
  using L = Tile<T, NDB>;
  constexpr int TW = kChunk / 32, TILE = kChunk * L::PITCH, NBUF = Stage<T, NDB, kWaves>::NBUF;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* tiles = reinterpret_cast<T*>(smem);                                  // [NBUF][K, V]
  int* kc_lds = reinterpret_cast<int*>(tiles + 2 * NBUF * TILE);          // [NBUF][kChunk]
  float* tab = reinterpret_cast<float*>(kc_lds + NBUF * kChunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, hh = lane >> 5;
  const Ids id = ids_of(a.B, a.heads * slices, (a.Sq + kRows - 1) / kRows, a.causal != 0, true);
  if (id.none) return;
  const int64_t b = id.b;
  const int head = id.head / slices, slice = id.head % slices, kvh = head / a.group, row0 = id.blk * kRows, q0 = row0 + 32 * wave;
  const View v = view_of(a, b);
  Walk walk = key_walk(a, v, b, row0);
  const int begin = walk.take(slice, slices);
  const QueryWave qw = query_wave(a, v, b, q0, r32);
  const Score sp = score_of<T>(a, head);
  if (sp.tab) stage_table<T>(tab, a, head, 64 * kWaves);
  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const int* codes = v.codes ? a.kcodes + b * a.kpad : nullptr;
  const bool live = qw.row < a.Sq;
  typename Frag<T>::type qf[2 * NDB];
  load_row<T, NDB>(qf, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)qw.row * a.qs[1] + head * a.qs[2], live, a.d, hh);
  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -__FLT_MAX__, l = 0.f;
  // Two LDS buffers with bf16: the next chunk is on its way while one is multiplied, one barrier per chunk.
  Stage<T, NDB, kWaves> sk, sv;
  int pc = 0, buf = 0;
  i32x4 info = {0, 0, 0, 0};             // of the chunk on its way
  auto issue = [&](int n, int kc) {
    const uint64_t rows = rows_of(info);
    sk.issue(tiles + 2 * n * TILE, kbase, a.ks[1], kc, rows, a.d);
    sv.issue(tiles + (2 * n + 1) * TILE, vbase, a.vs[1], kc, rows, a.d);
    if (v.codes && threadIdx.x < kChunk) pc = codes[kc + threadIdx.x];
  };
  int kc = walk.next(begin, info);
  if (kc < walk.end) issue(0, kc);
  for (; kc < walk.end; buf ^= NBUF - 1) {
    if (NBUF == 1) __syncthreads();     // the previous chunk has been consumed
    sk.land(tiles + 2 * buf * TILE);
    sv.land(tiles + (2 * buf + 1) * TILE);
    if (v.codes && threadIdx.x < kChunk) kc_lds[buf * kChunk + threadIdx.x] = pc;
    __syncthreads();
    const int at = kc;
    const i32x4 seen = info;
    kc = walk.next(kc + kChunk, info);
    if (kc < walk.end) issue(buf ^ (NBUF - 1), kc);
    const int sees = qw.sees(at, seen); // wave-uniform, like every branch below
    if (sees == 0) continue;
    const T *kt = tiles + 2 * buf * TILE, *vt = kt + TILE;
    const int rel0 = at - (v.start + q0);                       // the wave's first query to the chunk's first key
    f32x16 u[TW];
#pragma unroll
    for (int t = 0; t < TW; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) u[t][r] = 0.f;
#pragma unroll
      for (int s = 0; s < 2 * NDB; ++s) u[t] = mma(L::row(kt, 32 * t + r32, s, hh), qf[s], u[t]);
    }
    if (sp.cap) {
#pragma unroll
      for (int t = 0; t < TW; ++t) cap_tile<sizeof(T) == 4 ? kCapTile : MODE == kInfer ? kCapRough : kCapAhead>(u[t], sp);
    }
    float A = sp.A, C = 0.f;
    const bool near = sp.tab && rel0 + kChunk - 1 > -a.R && rel0 - 31 < a.R;
    if (sees < 3 || sp.slopes || near) {
#pragma unroll
      for (int t = 0; t < TW; ++t) {
        const int key = at + 32 * t + 4 * hh;
        bias_tile<1>(u[t], sp, tab, a.R, key - (v.start + qw.row), rel0 + 32 * t);
        if (sees < 3) hide_keys(u[t], qw, sees == 2, key, kc_lds + buf * kChunk + 32 * t + 4 * hh);
      }
      A = kPost<T>;
    } else {
      if (sizeof(T) == 4) {
#pragma unroll
        for (int t = 0; t < TW; ++t) scale_tile(u[t], sp);
        A = kPost<T>;
      }
      if (sp.tab) C = tab[rel0 < 0 ? 0 : 2 * a.R] * kPost<T>;
    }
    float top = u[0][0];
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, u[t][r]);
    top = fmaf(A, max_halves(top), C);
    // m follows the running maximum only when that has grown by more than 2^kSlack: most chunks skip the rescaling
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) {
      const float mn = top > m + kSlack ? top : m;
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
      m = mn;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    }
    // P is rounded to bf16 for its product, an error of 2^-9 that o passes on to delta, where it counts as soon as few keys
    // carry a row.  Chunks with a p of more than about 1/8 of its row so far (l is half a row's) also multiply what the
    // rounding leaves; eight p of 1/8 without it add a sixteenth to the two roundings' error of dq and dk.
    const bool rest = MODE == kTrainRest && __builtin_amdgcn_ballot_w64(4.f * __builtin_amdgcn_exp2f(top - m) > l) != 0;
    const float cm = C - m;
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < TW; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        u[t][r] = __builtin_amdgcn_exp2f(fmaf(A, u[t][r], cm));
        ps[r & 3] += u[t][r];
      }
      typename Frag<T>::type p0, p1;
      pack8(p0, u[t], 0);
      pack8(p1, u[t], 1);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        o[db] = mma(L::col(vt, 32 * t, db, lane), p0, o[db]);
        o[db] = mma(L::col(vt, 32 * t + 16, db, lane), p1, o[db]);
      }
      if (rest) {
        pack_rest(p0, p1, u[t]);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          o[db] = mma(L::col(vt, 32 * t, db, lane), p0, o[db]);
          o[db] = mma(L::col(vt, 32 * t + 16, db, lane), p1, o[db]);
        }
      }
    }
    l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  }
  l += __shfl_xor(l, 32, 64);           // the half-waves hold disjoint keys of the same query
  if (live && part != nullptr) {
    float* p = part + (((b * a.heads + head) * a.Sq + qw.row) * slices + slice) * (a.d + 4);
    store_row<float, NDB>(p, o, 1.f, a.d, hh);
    if (hh == 0) {
      p[a.d] = m;
      p[a.d + 1] = l;
    }
  } else if (live) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ((b * a.Sq + qw.row) * a.heads + head) * a.d;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4) {
        const int c = 32 * db + 8 * a4 + 4 * hh;
        if (c < a.d)
          store_out(static_cast<T*>(a.out), MODE == kTrainRest ? a.out_lo : nullptr, at + c, o[db][4 * a4] * inv, o[db][4 * a4 + 1] * inv, o[db][4 * a4 + 2] * inv,
                    o[db][4 * a4 + 3] * inv);
      }
    if (MODE != kInfer && a.lse != nullptr && hh == 0) store_lse(a, (b * a.heads + head) * a.Sq + qw.row, m, l);
  }
}

// ---- backward: dq and the table's gradient ---------------------------------------------------------------------------
// Sums of a tile's diagonals: lane c returns the sum over key - query = c - 31 (c = 63: 0).  Lane (hh, q), register r holds the value
// of query q and key 4 hh + acc_row(r).  For one register, sending lane (hh, q) to lane 31 - q + acc_row(r) + 32 hh (mod 64) is
// a permutation of the wave: half 0 lands on its columns acc_row(r) .. acc_row(r) + 31, half 1 everywhere else, 28 to the right
// (mod 64) of its own.  Two running sums take the two, and one more permutation brings the second home.
__device__ __forceinline__ float diagonal_sums(const f32x16& u, int lane) {
  asm volatile("" : "+v"(lane));        // the 16 lane masks are formed here: kept over the walk they push scalars out of registers
  const int base = 4 * (31 - (lane & 31) + (lane & 32));
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int to = (base + 4 * acc_row(r)) & 255;
    const float x = __int_as_float(__builtin_amdgcn_ds_permute(to, __float_as_int(u[r])));
    const bool first = (unsigned)(lane - acc_row(r)) < 32u;
    s0 += first ? x : 0.f;
    s1 += first ? 0.f : x;
  }
  return s0 + __int_as_float(__builtin_amdgcn_ds_permute(4 * ((lane + 36) & 63), __float_as_int(s1)));
}

// sum_d dout out of the lane's row, whose dout it holds (both half-waves)
template <typename T, int NDB>
__device__ __forceinline__ float row_delta(const typename Frag<T>::type (&dof)[2 * NDB], const BiasedArgs& a, int64_t at, bool live, int hh) {
  float sum = 0.f;
  typename Frag<T>::type o[2 * NDB];
  load_row<T, NDB>(o, static_cast<const T*>(a.out) + at, live, a.d, hh);
#pragma unroll
  for (int s = 0; s < 2 * NDB; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf((float)dof[s][j], (float)o[s][j], sum);
  if (sizeof(T) == 2 && a.out_lo != nullptr) {
    load_row<T, NDB>(o, reinterpret_cast<const T*>(a.out_lo) + at, live, a.d, hh);
#pragma unroll
    for (int s = 0; s < 2 * NDB; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf((float)dof[s][j], (float)o[s][j], sum);
  }
  return sum + __shfl_xor(sum, 32, 64);
}

// bf16, d <= 16: dS enters its products as the sum of two bf16 values.  Its rows sum to zero, so its sums over k and q cancel, the
// more the fewer the columns, and the rounding of dS shows: dq of 2978 keys of 16 2.55e-3 of its norm off with one value, 1.7e-3
// (the output's own rounding) with two, for 127 us instead of 105 in dq and 174 instead of 156 in dk and dv (4 x 12 x 2048).
template <typename T, int NDB>
__device__ __forceinline__ bool ds_in_halves(int d) { return sizeof(T) == 2 && NDB == 1 && d <= 16; }

// dq, and the table's gradient: ds summed along the diagonals of the tiles (diagonal_sums), a lane's diagonal at a time into the
// wave's array by relative distance, so that every sum has one order, from run to run.  Tiles at or beyond distance R go to two
// registers instead.  The block then folds its four arrays by bucket into one partial row.  (LDS float atomics, 16 per tile,
// took 190 cycles each: 686 us instead of 370 at 4 x 16 x 4096^2 causal; skewing the tile in LDS costs 8 KiB a wave, which at
// d = 128 leaves one block per CU: 163 us instead of 112 at 64 x 512 tokens, 4 heads.)
//   kTable: with the table's gradient.  kDelta: the first half of the same walk, delta_i = sum_j p_ij (do_i . v_j), instead of
// dout . out.  Needed by the table's gradient on bf16 operands: the o of the forward carries what is left of the rounding of P,
// which averages out in dq and dk but enters the few values of an fp32 dtable in full (4e-4 of their norm with a once rounded P).
//   slices > 1: as in the forward; dq (or delta) then goes to `part` [slice][..] in fp32 and k_ba_fold sums the slices in order.
enum DqKind { kPlain, kTable, kDelta };

template <typename T, int NDB, DqKind KIND>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 ? 1 : 2) void k_ba_dq(BiasedArgs a, int slices, float* part) {
  constexpr bool DELTA = KIND == kDelta, grad_tab = KIND == kTable;
  using L = Tile<T, NDB>;
  constexpr int TILE = kChunk * L::PITCH, NBUF = Stage<T, NDB, kWaves>::NBUF;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* tiles = reinterpret_cast<T*>(smem);                                  // [NBUF][K, V]
  int* kc_lds = reinterpret_cast<int*>(tiles + 2 * NBUF * TILE);          // [NBUF][kChunk]
  float* tab = reinterpret_cast<float*>(kc_lds + NBUF * kChunk);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, hh = lane >> 5;
  const int nblk = (a.Sq + kRows - 1) / kRows;
  const Ids id = ids_of(a.B, a.heads * slices, nblk, a.causal != 0, true);
  if (id.none) return;
  const int64_t b = id.b;
  const int head = id.head / slices, slice = id.head % slices, kvh = head / a.group, row0 = id.blk * kRows, q0 = row0 + 32 * wave;
  const View v = view_of(a, b);
  Walk walk = key_walk(a, v, b, row0);
  const int begin = walk.take(slice, slices);
  const QueryWave qw = query_wave(a, v, b, q0, r32);
  const Score sp = score_of<T>(a, head);
  const int TW = 2 * a.R + 1;
  float* hist = tab + TW;                                                 // [kWaves][TW]
  float* mine = hist + wave * TW;
  if (sp.tab) stage_table<T>(tab, a, head, 64 * kWaves);
  if (grad_tab)
    for (int i = threadIdx.x; i < kWaves * TW; i += 64 * kWaves) hist[i] = 0.f;
  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const int* codes = v.codes ? a.kcodes + b * a.kpad : nullptr;
  const bool live = qw.row < a.Sq;
  const int64_t at_q = ((b * a.Sq + qw.row) * a.heads + head) * a.d, at_l = (b * a.heads + head) * a.Sq + qw.row;
  typename Frag<T>::type qf[2 * NDB], dof[2 * NDB];
  load_row<T, NDB>(qf, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)qw.row * a.qs[1] + head * a.qs[2], live, a.d, hh);
  load_row<T, NDB>(dof, static_cast<const T*>(a.dout) + at_q, live, a.d, hh);
  const float lse = live ? a.lse[at_l] : INFINITY, inv = live ? a.lse[(int64_t)a.B * a.heads * a.Sq + at_l] : 0.f;
  const bool sighted = lse != INFINITY; // a row that sees no key passes no gradient, whatever it and its gradient hold
#pragma unroll
  for (int s = 0; s < 2 * NDB; ++s) {
    qf[s] = sighted ? qf[s] : typename Frag<T>::type{};
    dof[s] = sighted ? dof[s] : typename Frag<T>::type{};
  }
  float delta = 0.f;
  if (!DELTA && a.makes_delta) {
    delta = row_delta<T, NDB>(dof, a, at_q, live, hh);
    if (live && hh == 0 && slice == 0) a.delta[at_l] = delta;
  } else if (!DELTA && sighted) {
    delta = a.delta[at_l];
  }
  const float di = delta * inv;
  float dsum = 0.f;
  f32x16 dq[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[db][r] = 0.f;
  float far_lo = 0.f, far_hi = 0.f;
  Stage<T, NDB, kWaves> sk, sv;
  int pc = 0, buf = 0;
  i32x4 info = {0, 0, 0, 0};             // of the chunk on its way
  auto issue = [&](int n, int kc) {
    const uint64_t rows = rows_of(info);
    sk.issue(tiles + 2 * n * TILE, kbase, a.ks[1], kc, rows, a.d);
    sv.issue(tiles + (2 * n + 1) * TILE, vbase, a.vs[1], kc, rows, a.d);
    if (v.codes && threadIdx.x < kChunk) pc = codes[kc + threadIdx.x];
  };
  int kc = walk.next(begin, info);
  if (kc < walk.end) issue(0, kc);
  for (; kc < walk.end; buf ^= NBUF - 1) {
    if (NBUF == 1) __syncthreads();     // the previous chunk has been consumed
    sk.land(tiles + 2 * buf * TILE);
    sv.land(tiles + (2 * buf + 1) * TILE);
    if (v.codes && threadIdx.x < kChunk) kc_lds[buf * kChunk + threadIdx.x] = pc;
    __syncthreads();
    const int at = kc;
    const i32x4 seen = info;
    kc = walk.next(kc + kChunk, info);
    if (kc < walk.end) issue(buf ^ (NBUF - 1), kc);
    const int sees = qw.sees(at, seen);
    if (sees == 0) continue;
    const T *kt = tiles + 2 * buf * TILE, *vt = kt + TILE;
#pragma unroll
    for (int t = 0; t < kChunk / 32; ++t) {
      const int key0 = at + 32 * t, rel0 = key0 - (v.start + q0);
      if (key0 >= qw.last) break;
      f32x16 u, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { u[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
      for (int s = 0; s < 2 * NDB; ++s) {
        u = mma(L::row(kt, 32 * t + r32, s, hh), qf[s], u);
        dp = mma(L::row(vt, 32 * t + r32, s, hh), dof[s], dp);
      }
      reads_ahead<T, 4 * NDB, 1>();
      f32x16 g;                          // the cap's slope
      if (sp.cap) {
        cap_tile<kCapTile>(u, sp);
        if (!DELTA)
#pragma unroll
          for (int r = 0; r < 16; ++r) g[r] = cap_slope(u[r]);
      }
      float A = sp.A, C = 0.f;
      const int rel = key0 + 4 * hh - (v.start + qw.row);
      const bool far = sp.tab && (rel0 + 31 <= -a.R || rel0 - 31 >= a.R);
      if (sees < 3 || sp.slopes || (sp.tab && !far)) {
        bias_tile<1>(u, sp, tab, a.R, rel, rel0);
        if (sees < 3) hide_keys(u, qw, sees == 2, key0 + 4 * hh, kc_lds + buf * kChunk + 32 * t + 4 * hh);
        A = kPost<T>;
      } else {
        if (sizeof(T) == 4) {
          scale_tile(u, sp);
          A = kPost<T>;
        }
        if (sp.tab) C = tab[rel0 < 0 ? 0 : 2 * a.R] * kPost<T>;
      }
      const float cm = C - lse;
      if (DELTA) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dsum = fmaf(__builtin_amdgcn_exp2f(fmaf(A, u[r], cm)), dp[r], dsum);
        continue;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) u[r] = __builtin_amdgcn_exp2f(fmaf(A, u[r], cm)) * fmaf(dp[r], inv, -di);     // ds
      if (grad_tab) {
        if (far) {
          float s = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) s += u[r];
          if (rel0 < 0) far_lo += s;
          else far_hi += s;
        } else {
          const float sum = diagonal_sums(u, lane);
          const int x = rel0 - 31 + lane;
          if (x <= -a.R) far_lo += sum;
          else if (x >= a.R) far_hi += sum;
          else mine[x + a.R] += sum;
        }
      }
      if (sp.cap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] *= g[r];
      }
      typename Frag<T>::type d0, d1;
      pack8(d0, u, 0);
      pack8(d1, u, 1);
      if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        dq[db] = mma(L::col(kt, 32 * t, db, lane), d0, dq[db]);
        dq[db] = mma(L::col(kt, 32 * t + 16, db, lane), d1, dq[db]);
      }
      if (ds_in_halves<T, NDB>(a.d)) {
        pack_rest(d0, d1, u);
        dq[0] = mma(L::col(kt, 32 * t, 0, lane), d0, dq[0]);
        dq[0] = mma(L::col(kt, 32 * t + 16, 0, lane), d1, dq[0]);
      }
      reads_ahead<T, 2 * NDB, 2>();
    }
  }
  if (DELTA) {
    dsum = (dsum + __shfl_xor(dsum, 32, 64)) * inv;
    if (live && hh == 0) (part != nullptr ? part + slice * (((int64_t)a.B * a.heads * a.Sq + 3) / 4 * 4) : a.delta)[at_l] = dsum;
    return;
  }
  if (live && a.dq) {
    if (part != nullptr) store_row<float, NDB>(part + (int64_t)slice * a.B * a.Sq * a.heads * a.d + at_q, dq, a.scale, a.d, hh);
    else store_row<T, NDB>(static_cast<T*>(a.dq) + at_q, dq, a.scale, a.d, hh);
  }
  if (grad_tab) {
    far_lo = group_sum(far_lo, 64);
    far_hi = group_sum(far_hi, 64);
    __syncthreads();          // the arrays are zeroed also where no chunk was walked
    if (lane == 0) {
      mine[0] = far_lo;
      mine[2 * a.R] = far_hi;
    }
    __syncthreads();
    int* ids = reinterpret_cast<int*>(tab);
    for (int i = threadIdx.x; i < TW; i += 64 * kWaves) {
      float s = 0.f;
      for (int w = 0; w < kWaves; ++w) s += hist[w * TW + i];
      hist[i] = s;
      ids[i] = min(max(a.buckets[i], 0), a.nb - 1);
    }
    __syncthreads();
    int lanes = 64;                      // lanes per bucket, a power of two
    while (lanes > 1 && lanes * a.nb > 64 * kWaves) lanes >>= 1;
    for (int n0 = 0; n0 < a.nb; n0 += 64 * kWaves / lanes) {
      const int n = n0 + (int)threadIdx.x / lanes;
      float s = 0.f;
      for (int i = threadIdx.x % lanes; i < TW; i += lanes) s += ids[i] == n ? hist[i] : 0.f;
      s = group_sum(s, lanes);
      if (threadIdx.x % lanes == 0 && n < a.nb)
        a.dtab[(((int64_t)head * a.B * nblk + b * nblk + id.blk) * slices + slice) * a.nb + n] = s;
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
// A block's walk over the queries of all heads of a group.  Where there are few blocks, `split` blocks share a group's heads and
// each share's queries are cut into `cuts` equal parts; they leave fp32 partials that k_ba_fold sums in order.
//
// Roles (bf16, d > 64): dk and dv of 32 keys, their operands and the scores do not fit the 256 registers of two waves per SIMD.
// Eight waves a block then, wave w forming dv and wave w + 4 dk of the same keys: 5 products and two exponentials instead of 4
// and one, but two waves to fill each other's waits (64 x 512 tokens, 4 heads of 128: 200 us instead of 214; one kernel squeezed
// into 256 registers spills 304 bytes a lane, 238 us).
template <typename T, int NDB>
constexpr bool by_roles() { return sizeof(T) == 2 && NDB >= 3; }

template <typename T, int NDB>
__global__ __launch_bounds__(64 * kWaves * (by_roles<T, NDB>() ? 2 : 1), sizeof(T) == 4 ? 1 : 2) void k_ba_dkv(BiasedArgs a, int split, int cuts, float* part) {
  using L = Tile<T, NDB>;
  constexpr int TILE = kChunk * L::PITCH, NBUF = Stage<T, NDB, kWaves>::NBUF;
  constexpr bool ROLES = by_roles<T, NDB>();
  constexpr int NT = 64 * kWaves * (ROLES ? 2 : 1);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* tiles = reinterpret_cast<T*>(smem);                                  // [NBUF][Q, dO]
  float* lses = reinterpret_cast<float*>(tiles + 2 * NBUF * TILE);        // [NBUF][kChunk] each
  float* dels = lses + NBUF * kChunk;
  float* invs = dels + NBUF * kChunk;                                     // fp32 alone
  int* qc_lds = reinterpret_cast<int*>(sizeof(T) == 4 ? invs + NBUF * kChunk : invs);
  float* tab = reinterpret_cast<float*>(qc_lds + NBUF * kChunk);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, hh = lane >> 5;
  const Ids id = ids_of(a.B, a.kv * split * cuts, (a.Sk + kRows - 1) / kRows, a.causal != 0, false);
  if (id.none) return;
  const int64_t b = id.b;
  const int kvh = id.head / (split * cuts), piece = id.head % (split * cuts), share = piece / cuts, row0 = id.blk * kRows, k0 = row0 + 32 * (wave % kWaves), key = k0 + r32;
  const bool does_v = !ROLES || wave < kWaves, does_k = !ROLES || wave >= kWaves;
  const View v = view_of(a, b);
  const bool ok = key < a.Sk;
  const int kcode = !ok ? -1 : v.codes ? a.kcodes[b * a.kpad + key] : 0;
  int klo = 0, khi = 0;
  bool khid = k0 + 32 > a.Sk;
  if (v.codes) {
    wave_range(kcode, klo, khi);
    khid = __builtin_amdgcn_ballot_w64(kcode < 0) != 0;
  }
  const int first = v.first_row(key);                                     // the lane's key is seen from this row on
  const int wfirst = v.first_row(k0), wall = v.first_row(min(k0 + 31, a.Sk - 1));        // some / every key of the wave
  // the queries from the first that sees a key of the block on, cut into equal parts of whole chunks
  const int first_chunk = v.first_row(row0) / kChunk, chunks = max(0, (a.Sq + kChunk - 1) / kChunk - first_chunk);
  const int qfirst = (first_chunk + chunks * (piece % cuts) / cuts) * kChunk;
  const int qend = min(a.Sq, (first_chunk + chunks * (piece % cuts + 1) / cuts) * kChunk);
  int blo = 0, bhi = 0;
  if (v.codes) block_range(a.ktiles + b * (a.kpad / 64), row0, a.Sk, blo, bhi);
  Walk walk;
  walk.init(a.sighted ? a.sighted + b * (a.qpad / 64) : nullptr, qend, blo, bhi);
  // next chunk of queries of the group's heads that the block's keys may be seen from
  const int glast = bhi < 0 ? 0 : (share + 1) * a.group / split;          // (every key of the block hidden: none)
  struct Pos { int g, qc; };
  i32x4 info = {0, 0, 0, 0};             // of the chunk on its way
  auto settle = [&](Pos p) {
    while (p.g < glast) {
      p.qc = walk.next(p.qc, info);
      if (p.qc < qend) break;
      p.g += 1;
      p.qc = qfirst;
    }
    return p;
  };
  typename Frag<T>::type kf[2 * NDB], vf[2 * NDB];
  load_row<T, NDB>(kf, static_cast<const T*>(a.k) + b * a.ks[0] + (int64_t)key * a.ks[1] + kvh * a.ks[2], kcode >= 0 && first < a.Sq, a.d, hh);
  load_row<T, NDB>(vf, static_cast<const T*>(a.v) + b * a.vs[0] + (int64_t)key * a.vs[1] + kvh * a.vs[2], does_k && kcode >= 0 && first < a.Sq, a.d, hh);
  constexpr int NV = ROLES ? 1 : NDB;
  f32x16 dk[NDB], dv[NV];                // with roles, dk holds what the wave forms
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dk[db][r] = 0.f;
      dv[db % NV][r] = 0.f;
    }
  Stage<T, NDB, kWaves> sq, sd;
  float pl = 0.f, pd = 0.f, pi = 0.f;
  int pq = 0, buf = 0;
  auto issue = [&](int n, Pos p) {
    const int head = kvh * a.group + p.g;
    const uint64_t rows = rows_of(info);          // (rows that see no key arrive as zeros)
    if (!ROLES || wave < kWaves) {
      sq.issue(tiles + 2 * n * TILE, static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[2], a.qs[1], p.qc, rows, a.d);
      sd.issue(tiles + (2 * n + 1) * TILE, static_cast<const T*>(a.dout) + (b * a.Sq * a.heads + head) * a.d,
               (int64_t)a.heads * a.d, p.qc, rows, a.d);
    }
    const int i = p.qc + (int)threadIdx.x;
    const bool in = threadIdx.x < kChunk && i < a.Sq;
    pl = in ? a.lse[(b * a.heads + head) * a.Sq + i] : INFINITY;    // rows beyond Sq: p = exp2(. - inf) = 0
    pi = in ? a.lse[(b + a.B) * a.heads * a.Sq + (int64_t)head * a.Sq + i] : 0.f;
    pd = in ? a.delta[(b * a.heads + head) * a.Sq + i] : 0.f;
    if (v.docs && threadIdx.x < kChunk) pq = a.qcodes[b * a.qpad + i];
  };
  Pos p = settle(Pos{share * a.group / split, qfirst});
  if (p.g < glast) issue(0, p);
  int tab_head = -1;
  Score sp = score_of<T>(a, kvh * a.group);
  for (; p.g < glast; buf ^= NBUF - 1) {
    const Pos at = p;
    const int head = kvh * a.group + at.g;
    const bool other_head = head != tab_head;                             // block-uniform: another head's bias
    if (NBUF == 1 || (other_head && sp.tab)) __syncthreads();             // the previous chunk has been consumed
    sq.land(tiles + 2 * buf * TILE);
    sd.land(tiles + (2 * buf + 1) * TILE);
    if (threadIdx.x < kChunk) {
      // bf16: m + log2 l, whose rounding is far below that of p to the operands' type
      lses[buf * kChunk + threadIdx.x] = sizeof(T) == 4 || pl == INFINITY ? pl : pl - __builtin_amdgcn_logf(pi);
      if (sizeof(T) == 4) invs[buf * kChunk + threadIdx.x] = pi;
      dels[buf * kChunk + threadIdx.x] = pl == INFINITY ? 0.f : pd;       // such a row's dout may hold anything
      qc_lds[buf * kChunk + threadIdx.x] = pq;
    }
    if (other_head) {
      sp = score_of<T>(a, head);
      tab_head = head;
      if (sp.tab) stage_table<T>(tab, a, head, NT);
    }
    __syncthreads();
    const i32x4 seen = info;
    p = settle(Pos{p.g, p.qc + kChunk});
    if (p.g < glast) issue(buf ^ (NBUF - 1), p);
    if (k0 >= a.Sk || at.qc + kChunk <= wfirst) continue;
    bool clean = !khid && at.qc >= wall;
    bool codes = false;                 // pairs have to be compared by codes
    if (v.codes) {
      if (khi < 0 || seen[1] < klo || seen[0] > khi) continue;
      codes = v.docs && (rows_of(seen) != ~0ull || seen[0] != seen[1] || klo != khi || seen[0] != klo);
      clean = clean && !codes && klo == khi;
    }
    const T *qt = tiles + 2 * buf * TILE, *dt = qt + TILE;
    const float *ls = lses + buf * kChunk, *de = dels + buf * kChunk;
    const int* qcs = qc_lds + buf * kChunk;
#pragma unroll
    for (int t = 0; t < kChunk / 32; ++t) {
      const int q0 = at.qc + 32 * t;
      if (q0 >= a.Sq) break;
      if (q0 + 32 <= wfirst) continue;
      f32x16 u, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { u[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
      for (int s = 0; s < 2 * NDB; ++s) {
        u = mma(L::row(qt, 32 * t + r32, s, hh), kf[s], u);
        if (!ROLES) dp = mma(L::row(dt, 32 * t + r32, s, hh), vf[s], dp);
      }
      if (ROLES && does_k)
#pragma unroll
        for (int s = 0; s < 2 * NDB; ++s) dp = mma(L::row(dt, 32 * t + r32, s, hh), vf[s], dp);
      f32x16 g;
      if (sp.cap) {
        cap_tile<kCapTile>(u, sp);
#pragma unroll
        for (int r = 0; r < 16; ++r) g[r] = cap_slope(u[r]);
      }
      float A = sp.A, C = 0.f;
      const int rel0 = k0 - (v.start + q0), rel = key - (v.start + q0 + 4 * hh);        // register r: rel - acc_row(r)
      const bool near = sp.tab && rel0 + 31 > -a.R && rel0 - 31 < a.R;
      if (!clean || sp.slopes || near) {
        bias_tile<-1>(u, sp, tab, a.R, rel, rel0);
        if (!clean) {
          const int from = kcode >= 0 ? first - (q0 + 4 * hh) : INT32_MAX;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            bool see = acc_row(r) >= from;
            if (codes) see = see && qcs[32 * t + 4 * hh + acc_row(r)] == kcode;
            u[r] = see ? u[r] : -INFINITY;
          }
        }
        A = kPost<T>;
      } else {
        if (sizeof(T) == 4) {
          scale_tile(u, sp);
          A = kPost<T>;
        }
        if (sp.tab) C = tab[rel0 < 0 ? 0 : 2 * a.R] * kPost<T>;
      }
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(ls + 32 * t + 8 * a4 + 4 * hh);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[4 * a4 + i] = __builtin_amdgcn_exp2f(fmaf(A, u[4 * a4 + i], C - l4[i]));
        if (sizeof(T) == 4) {
          const f32x4 i4 = *reinterpret_cast<const f32x4*>(invs + buf * kChunk + 32 * t + 8 * a4 + 4 * hh);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[4 * a4 + i] *= i4[i];
        }
      }
      typename Frag<T>::type x0, x1;
      if (does_v) {
        pack8(x0, u, 0);
        pack8(x1, u, 1);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          f32x16& acc = ROLES ? dk[db] : dv[db % NV];
          acc = mma(L::col(dt, 32 * t, db, lane), x0, acc);
          acc = mma(L::col(dt, 32 * t + 16, db, lane), x1, acc);
        }
      }
      if (does_k) {
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(de + 32 * t + 8 * a4 + 4 * hh);
#pragma unroll
          for (int i = 0; i < 4; ++i) dp[4 * a4 + i] = u[4 * a4 + i] * (dp[4 * a4 + i] - d4[i]);
        }
        if (sp.cap) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= g[r];
        }
        pack8(x0, dp, 0);
        pack8(x1, dp, 1);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dk[db] = mma(L::col(qt, 32 * t, db, lane), x0, dk[db]);
          dk[db] = mma(L::col(qt, 32 * t + 16, db, lane), x1, dk[db]);
        }
        if (ds_in_halves<T, NDB>(a.d)) {
          pack_rest(x0, x1, dp);
          dk[0] = mma(L::col(qt, 32 * t, 0, lane), x0, dk[0]);
          dk[0] = mma(L::col(qt, 32 * t + 16, 0, lane), x1, dk[0]);
        }
      }
    }
  }
  if (!ok) return;
  const int64_t at = ((b * a.Sk + key) * a.kv + kvh) * a.d;
  const int64_t n = (int64_t)a.B * a.Sk * a.kv * a.d;                     // with parts: [piece][dk, dv][(B, Sk, kv, d)]
  auto put = [&](const auto& x, void* out, int64_t which, float mul) {
    if (part == nullptr) store_row<T, NDB>(static_cast<T*>(out) + at, x, mul, a.d, hh);
    else store_row<float, NDB>(part + which * n + at, x, mul, a.d, hh);
  };
  if constexpr (ROLES) {
    if (does_v) put(dk, a.dv, 2 * piece + 1, 1.f);
    else put(dk, a.dk, 2 * piece, a.scale);
  } else {
    put(dk, a.dk, 2 * piece, a.scale);
    put(dv, a.dv, 2 * piece + 1, 1.f);
  }
}

// out0 (and out1) = n pieces' partials in order: [piece][out0, out1][4 n4 values]
template <typename T>
__global__ __launch_bounds__(256) void k_ba_fold(const float* part, T* out0, T* out1, int64_t n4, int n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int outs = out1 != nullptr ? 2 : 1;
  if (i >= outs * n4) return;
  const bool second = i >= n4;
  const int64_t e = 4 * (second ? i - n4 : i);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < n; ++k) s += *reinterpret_cast<const f32x4*>(part + (outs * k + (second ? 1 : 0)) * 4 * n4 + e);
  store4((second ? out1 : out0) + e, s[0], s[1], s[2], s[3]);
}

// ---- host --------------------------------------------------------------------------------------------------------------
// Few queries take the split form, which packs (position, head of the group) into tiles of 32 rows.  8 rows of 32 + 8 heads of 128
// over 8192 keys, bf16: 51 us instead of 172 for one query, 93 instead of 176 for 16; 157 against 177 for 17, 164 against 181 for
// 32, and 300 against 210 for 64, whose 8 tiles a key head read the keys 8 times.  4 rows of 8 + 2 heads of 80 over 2000
// keys, fp32: 19 instead of 43 for 16.
bool few_queries(int64_t Sq) { return Sq <= 16; }

// Parts of a walk that blocks of their own take: until the chip's 1024 SIMDs have two waves each to choose from, and of two
// chunks at least.  A wave's walk is serial: with one wave per SIMD the longest one is waited for (4 x 8 heads x 1001
// fp32 causal queries are 1024 waves of 1 .. 16 chunks).  1 x 4 heads x 4096 causal bf16 queries, training: 178 us; 406 us
// without parts, 204 us with parts up to 4096 waves.
int parts_of(int64_t waves, int64_t chunks) {
  int64_t n = (2048 + waves - 1) / waves;
  if (n > chunks / 2) n = chunks / 2;
  if (n > 16) n = 16;
  return (int)(n < 1 ? 1 : n);
}
int key_slices(int64_t B, int64_t heads, int64_t Sq, int64_t Sk) {
  return parts_of(B * heads * ((Sq + 31) / 32), (Sk + kChunk - 1) / kChunk);
}
struct Pieces {
  int split, cuts;
};
// dk and dv: heads of a group first, until there are four blocks per CU, then their queries.  (4 x 4096, 16 + 4 heads of 64, training:
// 1224 us; 1495 with two blocks per CU, 1237 with eight)
Pieces query_pieces(int64_t B, int64_t Sq, int64_t Sk, int64_t kv, int64_t group) {
  const int64_t blocks = B * kv * ((Sk + kRows - 1) / kRows);
  Pieces p = {1, 1};
  for (int64_t s = 1; s <= group; ++s)
    if (group % s == 0) {
      p.split = (int)s;
      if (blocks * s >= 1024) break;
    }
  p.cuts = parts_of(B * kv * p.split * ((Sk + 31) / 32), (Sq + kChunk - 1) / kChunk);
  return p;
}
int64_t pad4(int64_t n) { return (n + 3) / 4 * 4; }

int64_t pad64(int64_t n) { return (n + 63) / 64 * 64; }
// LDS of the buffers (two with bf16, one with fp32): two tiles and `words` 4-byte values per row of a chunk
size_t tile_bytes(int dtype, int d, int words) {
  const int ndb = (d + 31) / 32, w = 32 * ndb;
  const int row = dtype == MIVAE_F32 ? (w + 4) * 4 : w * 2;
  return (size_t)(dtype == MIVAE_F32 ? 1 : 2) * kChunk * (2 * row + 4 * words);
}

template <typename... A>
void start(void (*fn)(A...), dim3 grid, size_t lds, hipStream_t st, A... args) {
  if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL(fn, grid, dim3(64 * kWaves), lds, st, args...);
}
template <typename T, int NDB>
void start_dkv(dim3 grid, size_t lds, hipStream_t st, const BiasedArgs& a, const Pieces& p, float* part) {
  if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)k_ba_dkv<T, NDB>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((k_ba_dkv<T, NDB>), grid, dim3(64 * kWaves * (by_roles<T, NDB>() ? 2 : 1)), lds, st, a, p.split, p.cuts, part);
}

// f(type tag, std::integral_constant NDB)
template <typename F>
void by_shape(int dtype, int d, F f) {
  using std::integral_constant;
  const int ndb = (d + 31) / 32;
  auto by_width = [&](auto tag) {
    switch (ndb) {
      case 1: return f(tag, integral_constant<int, 1>());
      case 2: return f(tag, integral_constant<int, 2>());
      case 3: return f(tag, integral_constant<int, 3>());
      default: return f(tag, integral_constant<int, 4>());
    }
  };
  if (dtype == MIVAE_F32) by_width(float());
  else by_width((unsigned short)0);
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
  MIVAE_REQUIRE(x->softcap >= 0.f && x->softcap < 1e30f && x->scale >= 0.f && x->scale < 1e30f,
                "%s: softcap or scale out of range", name);
  MIVAE_REQUIRE(x->softcap == 0.f || x->scale / x->softcap < 1e30f, "%s: softcap %g is too small for the scale", name, (double)x->softcap);
  MIVAE_REQUIRE(!(x->slopes && x->table), "%s: slopes and a table are alternatives", name);
  if (x->table)
    MIVAE_REQUIRE(x->buckets && x->num_buckets >= 1 && x->num_buckets <= kMaxBuckets && x->distance >= 1 && x->distance <= kMaxDistance,
                  "%s: %lld buckets up to distance %lld: 1 .. %d buckets, distance 1 .. %d", name, (long long)x->num_buckets,
                  (long long)x->distance, kMaxBuckets, kMaxDistance);
  MIVAE_REQUIRE(x->q_starts || (x->q_start >= 0 && x->q_start <= (1 << 24)), "%s: q_start %lld out of range", name, (long long)x->q_start);
  MIVAE_REQUIRE(aligned16(x->out_lo) && !(x->out_lo && !x->lse), "%s: out_lo must be 16-byte aligned and needs lse", name);
  MIVAE_REQUIRE(!(x->mask || x->documents) || (x->codes && aligned16(x->codes)), "%s: a mask or documents need the codes buffer", name);
  a.q = x->q; a.k = x->k; a.v = x->v;
  for (int i = 0; i < 3; ++i) { a.qs[i] = x->q_stride[i]; a.ks[i] = x->k_stride[i]; a.vs[i] = x->v_stride[i]; }
  a.out = x->out; a.lse = x->lse;
  a.out_lo = x->dtype == MIVAE_BF16 ? static_cast<unsigned short*>(x->out_lo) : nullptr;
  a.B = (int)x->batch; a.Sq = (int)x->q_len; a.Sk = (int)x->k_len; a.heads = (int)x->heads; a.kv = (int)x->kv_heads;
  a.group = a.heads / a.kv; a.d = (int)x->head_size;
  a.q_start = (int)x->q_start; a.q_starts = x->q_starts; a.prefix = x->prefix; a.causal = x->causal ? 1 : 0;
  a.slopes = x->slopes; a.table = x->table; a.buckets = x->buckets;
  a.nb = (int)x->num_buckets; a.R = x->table ? (int)x->distance : 0;
  a.scale = x->scale; a.cap = x->softcap;
  a.kpad = (int)pad64(a.Sk); a.qpad = (int)pad64(a.Sq);
  const int64_t nq = (x->batch * x->heads) * ((a.Sq + kRows - 1) / kRows), nk = (x->batch * x->heads) * ((a.Sk + kRows - 1) / kRows);        // parts only where there are few
  MIVAE_REQUIRE(x->batch <= (1 << 24) && nq < (1ll << 31) - 8 && nk < (1ll << 31) - 8 && x->batch * (a.kpad + a.qpad) / 256 < (1ll << 31),
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

int64_t mivae_biased_attention_fwd_floats(int64_t batch, int64_t q_len, int64_t k_len, int64_t heads, int64_t kv_heads,
                                          int64_t head_size) {
  if (few_queries(q_len)) return token_attention_floats(batch, q_len, k_len, heads, kv_heads, head_size);
  const int n = key_slices(batch, heads, q_len, k_len);
  return n > 1 ? batch * heads * q_len * n * (head_size + 4) : 0;
}

// [delta][the queries' summaries][table gradient's partials][the parts' delta, dq or dk and dv, one after another in the same place]
int64_t mivae_biased_attention_bwd_floats(int64_t batch, int64_t q_len, int64_t k_len, int64_t heads, int64_t kv_heads,
                                          int64_t head_size, int64_t num_buckets) {
  const int64_t nblk = (q_len + kRows - 1) / kRows, n = key_slices(batch, heads, q_len, k_len);
  const Pieces p = query_pieces(batch, q_len, k_len, kv_heads, heads / kv_heads);
  const int64_t rows = batch * heads * q_len, dq = n > 1 ? n * pad4(rows * head_size) : 0;
  const int64_t dkv = p.split * p.cuts > 1 ? 2 * p.split * p.cuts * batch * k_len * kv_heads * head_size : 0;
  return pad4(rows) + batch * pad64(q_len) / 16 + pad4(batch * heads * nblk * n * num_buckets) + (dq > dkv ? dq : dkv);
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
  if (few_queries(a.Sq)) {
    const int64_t need = token_attention_floats(a.B, a.Sq, a.Sk, a.heads, a.kv, a.d);
    MIVAE_REQUIRE(need == 0 || (x->scratch && aligned16(x->scratch)), "mivae_biased_attention_fwd: the keys are split and need the scratch buffer");
    token_attention(a, x->scratch, x->dtype, stream);
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_fwd (few queries)");
    return MIVAE_OK;
  }
  const int slices = key_slices(a.B, a.heads, a.Sq, a.Sk);
  MIVAE_REQUIRE(slices == 1 || (x->scratch && aligned16(x->scratch)), "mivae_biased_attention_fwd: the keys are split and need the scratch buffer");
  float* part = slices > 1 ? x->scratch : nullptr;
  const size_t lds = tile_bytes(x->dtype, a.d, 1) + (a.table ? (2 * a.R + 1) * 4 : 0);
  const dim3 grid((unsigned)grid_of((int64_t)a.B * a.heads * slices, (a.Sq + kRows - 1) / kRows, a.causal));
  by_shape(x->dtype, a.d, [&](auto t, auto n) {
    if (a.out_lo) start(k_ba_fwd<unsigned short, n(), kTrainRest>, grid, lds, S_(stream), a, slices, part);     // bf16 alone has it
    else if (a.lse || a.cap > kRoughCap) start(k_ba_fwd<decltype(t), n(), kTrain>, grid, lds, S_(stream), a, slices, part);
    else start(k_ba_fwd<decltype(t), n(), kInfer>, grid, lds, S_(stream), a, slices, part);
  });
  MIVAE_CHECK_LAUNCH("mivae_biased_attention_fwd");
  if (part) {
    token_attention_join(a, part, slices, x->dtype, stream);
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_fwd (join)");
  }
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
  MIVAE_REQUIRE(aligned16(x->scratch), "mivae_biased_attention_bwd: scratch must be 16-byte aligned");
  const int nblk = (a.Sq + kRows - 1) / kRows;
  a.delta = x->scratch;
  i32x4* sighted = reinterpret_cast<i32x4*>(x->scratch + pad4(rows));
  float* dtab = x->scratch + pad4(rows) + (int64_t)a.B * a.qpad / 16;
  a.dtab = x->dtable ? dtab : nullptr;
  const int slices = key_slices(a.B, a.heads, a.Sq, a.Sk);
  float* parts = dtab + (x->dtable ? pad4((int64_t)a.B * a.heads * nblk * slices * a.nb) : 0);
  float* part = slices > 1 ? parts : nullptr;
  hipStream_t st = S_(stream);
  const size_t tw = a.table ? 2 * a.R + 1 : 0, lds = tile_bytes(x->dtype, a.d, 1) + tw * 4;
  const dim3 grid((unsigned)grid_of((int64_t)a.B * a.heads * slices, nblk, a.causal)), dgrid((unsigned)((rows + 15) / 16));
  auto fold = [&](auto* out0, auto* out1, int64_t values, int n) {
    const int64_t n4 = (values + 3) / 4;
    hipLaunchKernelGGL((k_ba_fold<std::remove_pointer_t<decltype(out0)>>), dim3((unsigned)(((out1 ? 2 : 1) * n4 + 255) / 256)), dim3(256), 0,
                       st, parts, out0, out1, n4, n);
  };
  const bool exact = a.dtab && x->dtype == MIVAE_BF16;        // delta from a walk of its own
  a.makes_delta = !exact && (a.dq || a.dtab);                 // by the dq kernel, on its way
  if (a.makes_delta) {
  } else if (x->dtype == MIVAE_F32)
    hipLaunchKernelGGL((k_ba_delta<float>), dgrid, dim3(256), 0, st, static_cast<const float*>(x->dout),
                       static_cast<const float*>(x->out), nullptr, a.delta, rows, a.Sq, a.heads, a.d);
  else if (!exact)
    hipLaunchKernelGGL((k_ba_delta<unsigned short>), dgrid, dim3(256), 0, st, static_cast<const unsigned short*>(x->dout),
                       static_cast<const unsigned short*>(x->out), a.out_lo, a.delta, rows, a.Sq, a.heads, a.d);
  else {
    by_shape(MIVAE_BF16, a.d, [&](auto, auto n) { start(k_ba_dq<unsigned short, n(), kDelta>, grid, lds, st, a, slices, part); });
    if (part) fold(a.delta, (float*)nullptr, rows, slices);
  }
  MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (delta)");
  if (a.dq || a.dtab) {
    const size_t more = a.dtab ? kWaves * tw * 4 : 0;
    by_shape(x->dtype, a.d, [&](auto t, auto n) {
      if (a.dtab) start(k_ba_dq<decltype(t), n(), kTable>, grid, lds + more, st, a, slices, part);
      else start(k_ba_dq<decltype(t), n(), kPlain>, grid, lds, st, a, slices, part);
    });
    if (part && a.dq) {
      if (x->dtype == MIVAE_F32) fold(static_cast<float*>(a.dq), (float*)nullptr, rows * a.d, slices);
      else fold(static_cast<unsigned short*>(a.dq), (unsigned short*)nullptr, rows * a.d, slices);
    }
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dq)");
    if (a.dtab) {
      hipLaunchKernelGGL(k_ba_dtable, dim3((unsigned)(a.heads * a.nb)), dim3(64), 0, st, a.dtab, x->dtable,
                         (int64_t)a.B * nblk * slices, a.nb, a.heads);
      MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dtable)");
    }
  }
  if (a.dk) {
    if (a.kcodes || a.q_starts) {         // otherwise every query sees a key
      const int64_t waves = (int64_t)a.B * a.qpad / 64;
      hipLaunchKernelGGL(k_ba_sighted, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a.lse, a.qcodes, a.B, a.Sq, a.qpad, a.heads, sighted);
      a.sighted = sighted;
    }
    const Pieces p = query_pieces(a.B, a.Sq, a.Sk, a.kv, a.group);
    const int pieces = p.split * p.cuts;
    const dim3 kgrid((unsigned)grid_of((int64_t)a.B * a.kv * pieces, (a.Sk + kRows - 1) / kRows, a.causal));
    by_shape(x->dtype, a.d, [&](auto t, auto n) {
      start_dkv<decltype(t), n()>(kgrid, tile_bytes(x->dtype, a.d, x->dtype == MIVAE_F32 ? 4 : 3) + tw * 4, st, a, p, pieces > 1 ? parts : nullptr);
    });
    if (pieces > 1) {
      const int64_t values = (int64_t)a.B * a.Sk * a.kv * a.d;
      if (x->dtype == MIVAE_F32) fold(static_cast<float*>(a.dk), static_cast<float*>(a.dv), values, pieces);
      else fold(static_cast<unsigned short*>(a.dk), static_cast<unsigned short*>(a.dv), values, pieces);
    }
    MIVAE_CHECK_LAUNCH("mivae_biased_attention_bwd (dk, dv)");
  }
  return MIVAE_OK;
}

}  // extern "C"
