// The biased attention (biased_attention.hip) for a few new queries over long keys: bound by reading the keys and values once
// (one query for each of 32 rows of up to 8192 keys, 8 key heads of 128, bf16: 160 to 168 us by card, 4.8 to 5.0 TB/s, as
// fast as a large copy).
//
// The queries of a batch row that share a key head, (position, head of the group), are packed into tiles of up to 32 rows, so
// that one read of the keys serves all of them.  The keys are split over blocks and, inside a block, over two waves that
// work by themselves: a wave brings 32 keys and values at a time into its own part of LDS (bf16: two buffers, direct loads,
// two tiles of 16 KiB a wave on their way at d = 128, 128 KiB a CU), takes S^T = K Q^T, the softmax step and O^T += V^T P^T,
// and no wave waits for another until its walk ends.  Then the block joins its waves' (max, sum, O), and with more than one
// split a second kernel joins the blocks' in order.
//
// bf16: P enters its product as the sum of two bf16 values, P and what its rounding leaves.  The extra products are free
// here, and the output has one rounding instead of two.
#include "att_tiles.hpp"
#include "mivae.h"
#include "token_attention.hpp"

using namespace mivae;

namespace {

constexpr int kWaves = 2, kKeys = 32;          // keys of a tile
constexpr int kSpan = kWaves * kKeys;          // keys of a block's turn

// 32 rows of a head on their way into a wave's own tile; rows whose bit is 0 and columns beyond d arrive as zeros
template <typename T, int NDB>
struct WaveStage;

template <int NDB>
struct WaveStage<unsigned short, NDB> {
  using L = Tile<unsigned short, NDB>;
  static constexpr int NBUF = 2, N = L::GPR / 2;        // loads of a tile
  __device__ __forceinline__ void issue(unsigned short* tile, const unsigned short* src, int64_t sr, int row0, unsigned rows, int d) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i * 64 + lane, row = g / L::GPR, c = (g % L::GPR) ^ L::swizzle(row);
      const bool ok = ((rows >> row) & 1) && c * L::GE < d;
      const void* p = ok ? (const void*)(src + (int64_t)(row0 + row) * sr + c * L::GE) : (const void*)kZero16;
      const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned short*)(tile + i * 64 * L::GE));
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "memory", "m0");
    }
  }
  __device__ __forceinline__ void land(unsigned short*) {}
};

template <int NDB>
struct WaveStage<float, NDB> {
  using L = Tile<float, NDB>;
  static constexpr int NBUF = 1, N = L::GPR / 2;
  i32x4 r[N];
  __device__ __forceinline__ void issue(float*, const float* src, int64_t sr, int row0, unsigned rows, int d) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i * 64 + lane, row = g / L::GPR, c = g % L::GPR;
      r[i] = i32x4{0, 0, 0, 0};
      if (((rows >> row) & 1) && c * L::GE < d) r[i] = *reinterpret_cast<const i32x4*>(src + (int64_t)(row0 + row) * sr + c * L::GE);
    }
  }
  __device__ __forceinline__ void land(float* tile) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i * 64 + lane;
      *reinterpret_cast<i32x4*>(tile + L::at(g / L::GPR, g % L::GPR)) = r[i];
    }
  }
};

// No read or write of memory is moved across it by the compiler.  A wave's tile is written by other lanes than read it (and with
// bf16 by loads that the compiler does not know), with no barrier in between: the LDS serves a wave's own accesses in order.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }

// wait until at most `newer` of the wave's vector loads are outstanding
template <int NEWER>
__device__ __forceinline__ void wait_loads() {
  static_assert(NEWER < 64, "six bits");
  keep_order();
  __builtin_amdgcn_s_waitcnt(0x0f70 | (NEWER & 15) | (NEWER >> 4) << 14);
  keep_order();
}

struct TokenArgs {
  BiasedArgs a;
  float* part;          // [pair of (b, key head)][row tile][split][rows][d + 2]: O, max, sum; or null: one split
  int rows, tiles, splits, span;      // packed rows of a pair, tiles of 32 of them, splits of `span` keys
};

template <typename T, int NDB>
__global__ __launch_bounds__(64 * kWaves, 1) void k_token(TokenArgs t) {
  using L = Tile<T, NDB>;
  using S = WaveStage<T, NDB>;
  constexpr int TILE = kKeys * L::PITCH, NBUF = S::NBUF, W = 32 * NDB;
  const BiasedArgs& a = t.a;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, hh = lane >> 5;
  T* tiles = reinterpret_cast<T*>(smem) + wave * 2 * NBUF * TILE;         // [NBUF][K, V]
  const unsigned id = blockIdx.x;
  // the key heads of a row are neighbours in memory and in the grid
  const int kvh = (int)(id % (unsigned)a.kv), split = (int)(id / (unsigned)a.kv % (unsigned)t.splits);
  const unsigned rest = id / (unsigned)(a.kv * t.splits);
  const int rt = (int)(rest % (unsigned)t.tiles);
  const int64_t b = rest / (unsigned)t.tiles, pair = b * a.kv + kvh;
  const View v = view_of(a, b);
  // the lane's row
  const int row = rt * 32 + r32, pos = row / a.group, head = kvh * a.group + row % a.group;
  const bool live = row < t.rows;
  const int qpos = v.start + pos, limit = live ? v.limit(pos) : 0;
  const int first_pos = rt * 32 / a.group, last_pos = (min(rt * 32 + 32, t.rows) - 1) / a.group;
  const int code = !v.docs ? 0 : live ? a.qcodes[b * a.qpad + pos] : kNoCode;
  int lo = 0, hi = 0;
  if (v.docs) wave_range(code, lo, hi);
  const bool same = !v.docs || (lo == hi && __builtin_amdgcn_ballot_w64(code < 0) == 0);
  const int begin = split * t.span, end = min(min(begin + t.span, a.Sk), v.limit(last_pos));
  const int clean_end = v.limit(first_pos);                               // every row sees the keys below
  const Score sp = score_of<T>(a, kvh * a.group);
  const float slope = sp.slopes ? a.slopes[live ? head : 0] * kUnit<T> : 0.f;
  float far[2] = {0.f, 0.f};
  auto bias_at = [&](int rel) {
    const int n = min(max(a.buckets[min(max(rel, -a.R), a.R) + a.R], 0), a.nb - 1);
    return a.table[(int64_t)n * a.heads + (live ? head : 0)] * kUnit<T>;
  };
  if (sp.tab) {
    far[0] = bias_at(-a.R);
    far[1] = bias_at(a.R);
  }
  typename Frag<T>::type qf[2 * NDB];
  load_row<T, NDB>(qf, static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)pos * a.qs[1] + head * a.qs[2], live, a.d, hh);
  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m = -__FLT_MAX__, l = 0.f;
  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const int* codes = v.codes ? a.kcodes + b * a.kpad : nullptr;
  const i32x4* ktiles = v.codes ? a.ktiles + b * (a.kpad / 64) : nullptr;
  auto rows_at = [&](int key) -> unsigned {
    uint64_t all = low_rows(end - key / 64 * 64);       // what keys behind every query's limit hold must not meet a product
    if (ktiles) all &= rows_of(ktiles[key / 64]);
    return (unsigned)(all >> (key & 32));
  };
  S sk, sv;
  auto issue = [&](int n, int key) {
    const unsigned rows = rows_at(key);
    sk.issue(tiles + 2 * n * TILE, kbase, a.ks[1], key, rows, a.d);
    sv.issue(tiles + (2 * n + 1) * TILE, vbase, a.vs[1], key, rows, a.d);
  };
  int key0 = begin + kKeys * wave, buf = 0;
  wait_loads<0>();                      // from here on the only vector loads in flight are the tiles'
  if (key0 < end) issue(0, key0);
  for (; key0 < end; key0 += kSpan, buf ^= NBUF - 1) {
    const int next = key0 + kSpan;
    keep_order();
    __builtin_amdgcn_s_waitcnt(0xc07f);                 // lgkmcnt(0): the other buffer has been read to its end
    keep_order();
    if (NBUF == 2) {
      if (next < end) {
        issue(buf ^ 1, next);
        wait_loads<2 * S::N>();         // this tile is here, the next one may be on its way
      } else {
        wait_loads<0>();
      }
    }
    T* kt = tiles + 2 * buf * TILE;
    T* vt = kt + TILE;
    sk.land(kt);
    sv.land(vt);
    keep_order();
    if (NBUF == 1 && next < end) issue(0, next);
    bool clean = key0 + kKeys <= clean_end;
    if (ktiles != nullptr) {
      const i32x4 s = ktiles[key0 / 64];
      if (s[1] < lo || s[0] > hi) continue;
      clean = clean && rows_of(s) == ~0ull && same && s[0] == s[1] && s[0] == lo;
    }
    f32x16 u;
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * NDB; ++s) u = mma(L::row(kt, r32, s, hh), qf[s], u);
    if (sp.cap) {
      if (sizeof(T) == 2 && a.lse == nullptr && a.cap <= kRoughCap) cap_tile<kCapRough>(u, sp);
      else cap_tile<kCapTile>(u, sp);
    }
    const int key = key0 + 4 * hh, rel = key - qpos;
#pragma unroll
    for (int r = 0; r < 16; ++r) u[r] *= sp.A;
    if (sp.slopes) {
#pragma unroll
      for (int r = 0; r < 16; ++r) u[r] = fmaf(-slope, fabsf((float)rel + (float)acc_row(r)), u[r]);
    }
    if (sp.tab) {
      const int rel_lo = key0 - (v.start + last_pos), rel_hi = key0 + 31 - (v.start + first_pos);
      if (rel_hi <= -a.R || rel_lo >= a.R) {
        const float f = rel_hi <= -a.R ? far[0] : far[1];
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] += f;
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] += bias_at(rel + acc_row(r));
        wait_loads<0>();                // keeps the count of the tiles' loads: none of these is left
      }
    }
    if (!clean) {
      const int lim = limit - key;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        bool see = acc_row(r) < lim;
        if (codes != nullptr) see = see && codes[key + acc_row(r)] == code;
        u[r] = see ? u[r] : -INFINITY;
      }
      if (codes != nullptr) wait_loads<0>();
    }
    float top = u[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, u[r]);
    top = max_halves(top) * kPost<T>;
    const float mn = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - mn);
    if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      l *= alpha;
      m = mn;
    }
    float ps = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      u[r] = __builtin_amdgcn_exp2f(fmaf(kPost<T>, u[r], -m));
      ps += u[r];
    }
    l += ps;
    typename Frag<T>::type p0, p1;
    pack8(p0, u, 0);
    pack8(p1, u, 1);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      o[db] = mma(L::col(vt, 0, db, lane), p0, o[db]);
      o[db] = mma(L::col(vt, 16, db, lane), p1, o[db]);
    }
    if (sizeof(T) == 2) {
      pack_rest(p0, p1, u);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        o[db] = mma(L::col(vt, 0, db, lane), p0, o[db]);
        o[db] = mma(L::col(vt, 16, db, lane), p1, o[db]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  // join the waves: [wave][row][W + 4] floats of O, max, sum (the pitch keeps 16-byte stores aligned)
  constexpr int P = W + 4;
  float* join = reinterpret_cast<float*>(smem);
  __syncthreads();
  {
    float* mine = join + (wave * 32 + r32) * P;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4)
        store4(mine + 32 * db + 8 * a4 + 4 * hh, o[db][4 * a4], o[db][4 * a4 + 1], o[db][4 * a4 + 2], o[db][4 * a4 + 3]);
    if (hh == 0) {
      mine[W] = m;
      mine[W + 1] = l;
    }
  }
  __syncthreads();
  const int rows = min(32, t.rows - rt * 32);
  for (int i = threadIdx.x; i < rows * (a.d / 4); i += 64 * kWaves) {
    const int r = i / (a.d / 4), c = i % (a.d / 4) * 4;
    float top = -__FLT_MAX__;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, join[(w * 32 + r) * P + W]);
    float sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float* p = join + (w * 32 + r) * P;
      const float f = __builtin_amdgcn_exp2f(p[W] - top);
      sum = fmaf(f, p[W + 1], sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = fmaf(f, p[c + j], x[j]);
    }
    const int pr = rt * 32 + r;
    if (t.part == nullptr) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t i1 = pr / a.group, h1 = kvh * a.group + pr % a.group;
      store_out(static_cast<T*>(a.out), a.out_lo, ((b * a.Sq + i1) * a.heads + h1) * a.d + c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      if (a.lse && c == 0) store_lse(a, (b * a.heads + h1) * a.Sq + i1, top, sum);
    } else {
      float* p = t.part + (((int64_t)pair * t.rows + pr) * t.splits + split) * (a.d + 4);
      store4(p + c, x[0], x[1], x[2], x[3]);
      if (c == 0) {
        p[a.d] = top;
        p[a.d + 1] = sum;
      }
    }
  }
}

// out = the splits' partials joined in order, one wave per packed row: lanes take splits for the maximum and the sum, then
// stripes of splits for groups of four columns
template <typename T>
__global__ __launch_bounds__(64) void k_token_join(TokenArgs t) {
  const BiasedArgs& a = t.a;
  const int64_t pr = blockIdx.x;         // a row per block: below 2^31
  const int lane = threadIdx.x, pitch = a.d + 4;
  const float* p = t.part + pr * t.splits * pitch;
  int lpg = 1;                           // lanes per row of d / 4 groups, a power of two
  while (lpg < a.d / 4) lpg <<= 1;
  const int c = (lane % lpg) * 4, stripes = 64 / lpg, first = lane / lpg;
  const bool on = c < a.d && first < t.splits;
  // the first loads of all three parts go out together: with few splits they are all there are
  float m0 = -__FLT_MAX__, l0 = 0.f, mx = 0.f;
  f32x4 y0 = {0.f, 0.f, 0.f, 0.f};
  if (lane < t.splits) {
    m0 = p[lane * pitch + a.d];
    l0 = p[lane * pitch + a.d + 1];
  }
  if (on) {
    y0 = *reinterpret_cast<const f32x4*>(p + first * pitch + c);
    mx = p[first * pitch + a.d];
  }
  float top = m0;
  for (int s = lane + 64; s < t.splits; s += 64) top = fmaxf(top, p[s * pitch + a.d]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  float sum = __builtin_amdgcn_exp2f(m0 - top) * l0;
  for (int s = lane + 64; s < t.splits; s += 64) sum = fmaf(__builtin_amdgcn_exp2f(p[s * pitch + a.d] - top), p[s * pitch + a.d + 1], sum);
  sum = group_sum(sum, 64);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    x = y0 * __builtin_amdgcn_exp2f(mx - top);
#pragma unroll 4
    for (int s = first + stripes; s < t.splits; s += stripes) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + s * pitch + c);
      const float f = __builtin_amdgcn_exp2f(p[s * pitch + a.d] - top);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = fmaf(f, y[j], x[j]);
    }
  }
  for (int off = 32; off >= lpg; off >>= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += __shfl_xor(x[j], off, 64);
  const unsigned pair = blockIdx.x / (unsigned)t.rows, row = blockIdx.x % (unsigned)t.rows, kvh = pair % (unsigned)a.kv;
  const int64_t b = pair / (unsigned)a.kv, pos = row / (unsigned)a.group, head = kvh * a.group + row % (unsigned)a.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane < lpg && c < a.d)
    store_out(static_cast<T*>(a.out), a.out_lo, ((b * a.Sq + pos) * a.heads + head) * a.d + c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  if (a.lse && lane == 0) store_lse(a, (b * a.heads + head) * a.Sq + pos, top, sum);
}

template <typename T, int NDB>
void start(const TokenArgs& t, unsigned grid, hipStream_t st) {
  constexpr int pitch = Tile<T, NDB>::PITCH * (int)sizeof(T), join = (32 * NDB + 4) * 4;
  constexpr size_t loop = (size_t)kWaves * 2 * WaveStage<T, NDB>::NBUF * kKeys * pitch, end = (size_t)kWaves * 32 * join;
  constexpr size_t lds = loop > end ? loop : end;
  if (lds > 64 * 1024)
    (void)hipFuncSetAttribute((const void*)k_token<T, NDB>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((k_token<T, NDB>), dim3(grid), dim3(64 * kWaves), lds, st, t);
}

void join(const TokenArgs& t, int dtype, hipStream_t st) {
  const dim3 rows((unsigned)((int64_t)t.a.B * t.a.kv * t.rows));
  if (dtype == MIVAE_F32) hipLaunchKernelGGL((k_token_join<float>), rows, dim3(64), 0, st, t);
  else hipLaunchKernelGGL((k_token_join<unsigned short>), rows, dim3(64), 0, st, t);
}

// Splits: 1024 blocks, two turns of two blocks per CU, each of at least one turn of its waves (64 keys).  More pay for more
// starts and partials (2048: 178 us at the size above), fewer wait for the longest row (512: 165 us there, 56 % to 100 % full).
int splits_of(int64_t blocks, int64_t Sk) {
  int64_t s = (1024 + blocks - 1) / blocks;
  const int64_t most = (Sk + kSpan - 1) / kSpan;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

}  // namespace

namespace mivae {

int64_t token_attention_floats(int64_t B, int64_t Sq, int64_t Sk, int64_t heads, int64_t kv, int64_t d) {
  const int64_t rows = Sq * (heads / kv), tiles = (rows + 31) / 32;
  const int s = splits_of(B * kv * tiles, Sk);
  return s > 1 ? B * kv * rows * s * (d + 4) : 0;
}

void token_attention(const BiasedArgs& a, float* scratch, int dtype, void* stream) {
  TokenArgs t = {};
  t.a = a;
  t.rows = a.Sq * a.group;
  t.tiles = (t.rows + 31) / 32;
  t.splits = splits_of((int64_t)a.B * a.kv * t.tiles, a.Sk);
  t.span = (int)(((int64_t)(a.Sk + t.splits - 1) / t.splits + kSpan - 1) / kSpan * kSpan);
  t.part = t.splits > 1 ? scratch : nullptr;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)((int64_t)a.B * a.kv * t.tiles * t.splits);
  const int ndb = (a.d + 31) / 32;
  if (dtype == MIVAE_F32) {
    if (ndb == 1) start<float, 1>(t, grid, st);
    else if (ndb == 2) start<float, 2>(t, grid, st);
    else if (ndb == 3) start<float, 3>(t, grid, st);
    else start<float, 4>(t, grid, st);
  } else {
    if (ndb == 1) start<unsigned short, 1>(t, grid, st);
    else if (ndb == 2) start<unsigned short, 2>(t, grid, st);
    else if (ndb == 3) start<unsigned short, 3>(t, grid, st);
    else start<unsigned short, 4>(t, grid, st);
  }
  if (t.part) join(t, dtype, st);
}

void token_attention_join(const BiasedArgs& a, float* part, int splits, int dtype, void* stream) {
  TokenArgs t = {};
  t.a = a;
  t.a.kv = a.heads;
  t.a.group = 1;
  t.part = part;
  t.rows = a.Sq;
  t.splits = splits;
  join(t, dtype, reinterpret_cast<hipStream_t>(stream));
}

}  // namespace mivae
