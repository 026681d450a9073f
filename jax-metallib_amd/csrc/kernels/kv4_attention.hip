// Attention of the newest tokens of each sequence over the paged 4-bit cache
// (kv4.h), for gfx950.
//
//   out[b, i, hq] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max)
//
// over the keys j < lens[b] - (L - 1 - i) of sequence b that lie in a page the
// cache has, query head hq reading key head hq / (Hq / Hkv).  No key: zeros.
//
// The L Hq / Hkv query rows of a sequence and key head (row r: token r / group,
// head r % group) are the columns of the matrix products, 16 to an item.  The
// 64-key tiles of all items, one item after the other, are cut into equal runs
// for the 2048 waves that the card holds (2 per SIMD), whatever the lengths
// and without the host knowing them: each wave finds its run from the lengths,
// and keeps a running maximum, sum and output per item.  An item within one
// wave's run is finished there; the others' partial results, joined first in
// LDS where a workgroup's 4 waves share one item, are added up in order by a
// second kernel.  (Against parts of each sequence chosen by the batch size, and
// with what that made possible: 64 sequences of 4096 .. 16129 keys 195 -> 160
// us, 16 of 1 .. 2048 30.9 -> 21.3 us.)
//   K, V, scales and zero points of a tile (64 x 140 bytes at D = 128) come by
//   LDS DMA into the wave's own two stages, one tile ahead; nothing in the
//   loop waits for another wave.
//   The numbers n of 4 bits go to the matrix cores as the bf16 128 + n, made
//   two at a time by (x >> 4i) & 0x000f000f | 0x43004300; this pairs the
//   dimensions (or keys) i and i + 4 of 8, and the other operand is laid out to
//   match.
//   S = K Q^T per group of 64 dimensions: the accumulator starts at
//     -128 sum(q), so it ends at sum(n q); score = sum over groups of
//     s (sum(n q) - z sum(q)).  Tile row 4g + e of block tt is key 16g + 4tt + e,
//     so lane (g, query) ends with 16 keys in a row.
//   O += V^T P^T: V is read transposed (ds_read_b64_tr_b4: 16 keys of one
//     dimension), P' = p s per group rounded to bf16, and a second product with
//     the rows -(128 + z) takes the offset off again right away, so what
//     accumulates is sum(P' (n - z)) and the rounding of P' (2^-8) is the only
//     one to fewer than 32 bits: P' takes the range of the scales, which 16 bits
//     with more digits do not have without a common factor for each tile.  Against
//     64 bits the results are off by 0.0016 .. 0.0023 of their size, where rounding
//     the result alone gives 0.0015 .. 0.0017.
// Bound by HBM when the cache is long: 726 MB in 157 us, 4.6 TB/s where a copy
// reaches 4.95.  711 vector (counted, with the start and end of each run) and 48
// matrix instructions a tile of 64 keys; both grow with the keys and heads of the
// cache and with every 16 query rows of a key head, whose blocks read and unpack
// the tile again.  28 % of the LDS cycles in use are lost to banks (counted).
// Short batches are bound by latency: lengths, page ids, the tile, its chain of
// products, the second kernel (10 us for one row of 2049 keys).
#include "kv4.h"
#include "wave.h"

#include <math.h>

namespace mk {

struct Kv4AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_strides[3], out_strides[3];  // sequence, token, head; elements
  Kv4View c;
  const int32_t* table;
  const int32_t* lens;
  float* part;     // [wave, 2][prow][D] f32 and, behind them all,
  float* part_ml;  // [wave, 2][prow] (maximum, sum)
  int64_t width;   // block table columns
  uint64_t page_magic;  // ceil(2^32 / (page / 16))
  int B, L, Hq, group;
  int blocks;  // of 16 rows, per sequence and key head
  int prow;    // rows of a partial result
  float scale_log2;
};

constexpr int kKaTile = 64;  // keys per tile
constexpr float kKaSlack = 8.f;  // log2 units
// p is held below 2^-5, so that the offsets (128 + z <= 143 steps of a scale,
// where the largest value of a group has 7 or more) cannot pass the f32 range
// before the sum of p times those largest values does.
constexpr float kKaLift = kKaSlack + 5.f;
constexpr int kKaWaves = 4;  // per workgroup
constexpr int kKaLog = 11;   // log2 of the waves that share the work

typedef int ka_i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) ka_i32x2* ka_lds_i32x2;

// Keys of sequence b; table rows hold 2^28 at most.
__device__ __forceinline__ int ka_len(const Kv4AttnArgs& a, int b) {
  const int len = a.lens[b], top = (int)(a.width * a.c.page);
  return len < 0 ? 0 : len > top ? top : len;
}

// Tiles of a sequence in the shared list: at least one, which writes the zeros
// of an empty sequence.
__device__ __forceinline__ int ka_tiles(int len) { return len > 0 ? (len + kKaTile - 1) / kKaTile : 1; }

// The lengths of a batch as one wave holds them: the first 64 in its lanes,
// the rest read as they are needed.
struct KaLens {
  int len, tiles, upto;  // of sequence `lane`: keys, tiles, tiles up to and with it
  int all;               // tiles of all sequences

  __device__ __forceinline__ KaLens(const Kv4AttnArgs& a, int lane) {
    len = lane < a.B ? ka_len(a, lane) : 0;
    tiles = lane < a.B ? ka_tiles(len) : 0;
    upto = wave_scan(tiles);
    all = __builtin_amdgcn_readlane(upto, 63);
    if (a.B > 64) {
      int v = 0;
      for (int c = 64 + lane; c < a.B; c += 64) v += ka_tiles(ka_len(a, c));
      all += wave_sum(v);
    }
  }
  __device__ __forceinline__ int keys(const Kv4AttnArgs& a, int b) const {
    return b < 64 ? __builtin_amdgcn_readlane(len, b) : __builtin_amdgcn_readfirstlane(ka_len(a, b));
  }
  // The tiles before sequence b.
  __device__ __forceinline__ int before(const Kv4AttnArgs& a, int b, int lane) const {
    if (b < 64) return __builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(tiles, b);
    int v = 0;
    for (int c = 64 + lane; c < b; c += 64) v += ka_tiles(ka_len(a, c));
    return __builtin_amdgcn_readlane(upto, 63) + wave_sum(v);
  }
  // The sequence that the y-th tile belongs to, and the tiles before it.
  __device__ __forceinline__ int find(const Kv4AttnArgs& a, int y, int lane, int* before) const {
    int run = 0, mine = tiles, sum = upto;
    for (int c = 0;; c += 64) {
      const uint64_t past = __ballot(run + sum > y);
      if (past || c + 64 >= a.B) {
        const int at = past ? __ffsll((unsigned long long)past) - 1 : 0;
        *before = run + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(mine, at);
        return c + at;
      }
      run += __builtin_amdgcn_readlane(sum, 63);
      mine = c + 64 + lane < a.B ? ka_tiles(ka_len(a, c + 64 + lane)) : 0;
      sum = wave_scan(mine);
    }
  }
};

// The list has `all` tiles (below 2^31); wave W of 2^kKaLog takes those from
// ka_start(W) to ka_start(W + 1), one each while there are fewer than waves.
__device__ __forceinline__ int ka_start(int64_t W, int all) {
  if (all >> kKaLog) return (int)((W * all) >> kKaLog);
  return W < all ? (int)W : all;
}
// The wave that takes tile x.
__device__ __forceinline__ int ka_wave_of(int x, int all) {
  if (all >> kKaLog) return (int)(((((uint64_t)x + 1) << kKaLog) - 1) / (uint32_t)all);
  return x;
}

// Whether one of the first `lim` keys of sequence b lies in a page the cache
// has.
__device__ __forceinline__ bool ka_sees(const Kv4AttnArgs& a, int b, int lim) {
  const int32_t* table = a.table + (int64_t)b * a.width;
  for (int c = 0; (int64_t)c * a.c.page < lim; ++c)
    if (table[c] >= 0 && table[c] < a.c.pages) return true;
  return false;
}

// What a row of the sum `sum` is multiplied with at the end: no key seen gives
// zeros, only scores of -infinity NaN.
__device__ __forceinline__ float ka_inverse(const Kv4AttnArgs& a, float sum, int b, int lim) {
  return sum == 0.f && !ka_sees(a, b, lim) ? 0.f : 1.0f / sum;
}

// 8 numbers of 4 bits as the bf16 128 + n, in the order 0 4 1 5 2 6 3 7.  The
// mask M = 0x000f000f comes in a vector register: v_and_or_b32 takes one
// constant only.
__device__ __forceinline__ u32x4 ka_numbers(uint32_t x, uint32_t M) {
  constexpr uint32_t C = 0x43004300u;
  return u32x4{(x & M) | C, ((x >> 4) & M) | C, ((x >> 8) & M) | C, ((x >> 12) & M) | C};
}

// 8 bf16 in that order.
__device__ __forceinline__ u32x4 ka_order(const u32x4& x) {
  return u32x4{perm(x.z, x.x, 0x05040100u), perm(x.z, x.x, 0x07060302u), perm(x.w, x.y, 0x05040100u),
               perm(x.w, x.y, 0x07060302u)};
}

template <int D>
__global__ __launch_bounds__(256, 2) void attention_kv4_kernel(Kv4AttnArgs a) {
  constexpr int GP = D / kKv4Group, NB = D / 16, ROWB = D / 2;
  constexpr int HALF = kKaTile * ROWB, STAGE = 2 * HALF + 1024;  // K, V, scales and zero points
  constexpr int NDMA = 2 * HALF / 1024 + 1;
  constexpr int OROW = D + 4;  // floats per output row in LDS
  extern __shared__ __attribute__((aligned(16))) unsigned char ka_smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int HB = a.c.heads * a.blocks;
  const int W = (int)blockIdx.x * kKaWaves + w;
  const KaLens lens(a, lane);
  const int all = lens.all * HB;
  const int x0 = ka_start(W, all), x1 = ka_start(W + 1, all);
  // The workgroup's run; if it lies within one item, its waves join in LDS (a
  // wave without tiles too, which looks at the run's last item).
  const int64_t first = (int64_t)blockIdx.x * kKaWaves;
  const int g0 = ka_start(first, all), g1 = ka_start(first + kKaWaves, all);
  if (g0 >= g1) return;
  int before = 0, b = lens.find(a, (x0 < g1 ? x0 : g1 - 1) / HB, lane, &before);
  const int rows = a.L * a.group;
  bool joined, whole;
  int left, block, h;  // of the item at hand: rows in use, row block, key head
  {
    const int nt = ka_tiles(lens.keys(a, b)), hb = ((x0 < g1 ? x0 : g1 - 1) - before * HB) / nt;
    const int s0 = before * HB + hb * nt;
    block = hb % a.blocks;
    h = hb / a.blocks;
    left = rows - 16 * block < 16 ? rows - 16 * block : 16;
    joined = g0 >= s0 && g1 <= s0 + nt;  // the same for all four waves
    whole = g0 == s0 && g1 == s0 + nt;
  }
  const int jb = b;
  uint32_t mask = 0x000f000fu;
  asm("" : "+v"(mask));
  unsigned char* mine = ka_smem + w * 2 * STAGE;
  const uint32_t sbase = lds_addr(mine);
  f32x4 o[NB];
  float m = -INFINITY, lsum = 0.f;
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int x = x0; x < x1;) {
    const int len = lens.keys(a, b), nt = ka_tiles(len);
    const int hb = (x - before * HB) / nt;
    const int s0 = before * HB + hb * nt, s1 = s0 + nt;  // the item's tiles
    const int xe = x1 < s1 ? x1 : s1;                    // this wave's end of them
    const int ta = x - s0, tb = xe - s0;
    block = hb % a.blocks;
    h = hb / a.blocks;
    if (!joined) whole = x == s0 && xe == s1;
    left = rows - 16 * block < 16 ? rows - 16 * block : 16;
    const int r = 16 * block + (l16 < left ? l16 : left - 1);
    const int qi = r / a.group, qh = h * a.group + r % a.group;
    const int lim = len - (a.L - 1 - qi);                     // keys the row sees
    const int lim0 = len - (a.L - 1 - 16 * block / a.group);  // the block's first row

    // The page ids of the 16-key runs 64 c .. 64 c + 63, a lane each: 16 tiles.
    const int32_t* table = a.table + (int64_t)b * a.width;
    auto pages_of = [&](int c) {
      const uint32_t run = (uint32_t)c * 64 + lane, idx = (uint32_t)(((uint64_t)run * a.page_magic) >> 32);
      return run * 16 < (uint32_t)len ? table[idx] : -1;
    };
    int pids = pages_of(ta >> 4);
    // Q: dimensions 64 G + 16 g + 8 x .. +7 of row l16.
    const uint16_t* q = a.q + b * a.q_strides[0] + qi * a.q_strides[1] + qh * a.q_strides[2];
    u32x4 qf[GP][2];
#pragma unroll
    for (int G = 0; G < GP; ++G)
#pragma unroll
      for (int i = 0; i < 2; ++i) qf[G][i] = *reinterpret_cast<const u32x4*>(q + 64 * G + 16 * g + 8 * i);

    // Issues tile t into a stage; the bits of the result say which of its four
    // runs of 16 keys lie in a page the cache has.  Runs that do not, and those
    // behind the sequence, read page 0.
    auto issue = [&](int t, int slot) {
      const uint32_t st = sbase + (uint32_t)(slot * STAGE);
      uint32_t ok = 0;
      int64_t at[4];  // (page id * heads + h) * page
      int off[4];     // place in the page
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t run = (uint32_t)t * 4 + j, idx = (uint32_t)(((uint64_t)run * a.page_magic) >> 32);
        const int pid = __builtin_amdgcn_readlane(pids, (int)(run & 63));
        const bool good = pid >= 0 && pid < a.c.pages;
        ok |= (good ? 1u : 0u) << j;
        off[j] = good ? (int)(run - idx * (uint32_t)(a.c.page / 16)) * 16 : 0;
        at[j] = ((int64_t)(good ? pid : 0) * a.c.heads + h) * a.c.page;
      }
#pragma unroll
      for (int i = 0; i < HALF / 1024; ++i) {
        if constexpr (D == 128) {
          const int tau = lane >> 2, c = lane & 3;
          const int64_t row = (at[i] + off[i] + tau) * ROWB;
          dma16_asm(a.c.k.rows + row + 16 * (c ^ i), st + (uint32_t)(i * 1024));
          dma16_asm(a.c.v.rows + row + 16 * (c ^ (tau >> 2)), st + (uint32_t)(HALF + i * 1024));
        } else {
          const bool up = lane >= 32;
          const int tau = (lane & 31) >> 1, c = lane & 1;
          const int64_t row = ((up ? at[2 * i + 1] + off[2 * i + 1] : at[2 * i] + off[2 * i]) + tau) * ROWB;
          dma16_asm(a.c.k.rows + row + 16 * (c ^ (up ? 1 : 0)), st + (uint32_t)(i * 1024));
          dma16_asm(a.c.v.rows + row + 16 * (c ^ (tau >> 3)), st + (uint32_t)(HALF + i * 1024));
        }
      }
      // Scales of K, of V (bf16 [GP][64] each), zero points of K, of V (bytes
      // [GP][64]): 24 GP lanes, the rest copies of the last.
      const int x = lane < 24 * GP ? lane : 24 * GP - 1;
      const bool zero = x >= 16 * GP;
      const int y = zero ? x - 16 * GP : x, half = zero ? 4 * GP : 8 * GP;
      const bool ofv = y >= half;
      const int z = ofv ? y - half : y;
      const int G = zero ? z >> 2 : z >> 3, j = zero ? z & 3 : (z >> 1) & 3, tok = zero ? 0 : 8 * (z & 1);
      const int64_t aj = j == 0 ? at[0] : j == 1 ? at[1] : j == 2 ? at[2] : at[3];
      const int oj = j == 0 ? off[0] : j == 1 ? off[1] : j == 2 ? off[2] : off[3];
      const int64_t el = aj * GP + (int64_t)G * a.c.page + oj + tok;
      const unsigned char* base =
          zero ? (ofv ? a.c.v.zero : a.c.k.zero)
               : reinterpret_cast<const unsigned char*>(ofv ? a.c.v.scale : a.c.k.scale);
      dma16_asm(base + (zero ? el : 2 * el), st + (uint32_t)(2 * HALF));
      return ok;
    };

#pragma unroll
    for (int n = 0; n < NB; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    lsum = 0.f;
    uint32_t ok = 0, ok_next = 0;
    int slot = 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    ok_next = issue(ta, 0);
    // The sums of Q per group; then its order is that of the numbers.
    float sq[GP];
#pragma unroll
    for (int G = 0; G < GP; ++G) {
      sq[G] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sq[G] += bf16_to_f32(qf[G][i][e] & 0xffffu) + bf16_to_f32(qf[G][i][e] >> 16);
        qf[G][i] = ka_order(qf[G][i]);
      }
      sq[G] = quad_sum(sq[G]);
    }
    for (int t = ta; t < tb; ++t) {
      ok = ok_next;
      if (t + 1 < tb) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other stage's reads are done
        if (((t + 1) & 15) == 0) pids = pages_of((t + 1) >> 4);
        ok_next = issue(t + 1, slot ^ 1);
        vm_wait(NDMA);
      } else {
        vm_wait(0);
      }
      const unsigned char* Ks = mine + slot * STAGE;
      const unsigned char* Vs = Ks + HALF;
      const unsigned char* Ps = Vs + HALF;
      const int kv0 = t * kKaTile;

      // All of the tile's LDS reads up front: their latency is paid once.
      uint32_t kw[4][2 * GP];
      u32x4 kz[GP], ks0[GP], ks1[GP], vz[GP], vs0[GP], vs1[GP];
      ka_i32x2 vw[NB];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const int j = l16 >> 2, tau = 4 * tt + (l16 & 3);
        if constexpr (D == 128) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(Ks + j * 1024 + tau * ROWB + 16 * (g ^ j));
#pragma unroll
          for (int i = 0; i < 4; ++i) kw[tt][i] = v[i];
        } else {
          const u32x2 v =
              *reinterpret_cast<const u32x2*>(Ks + (16 * j + tau) * ROWB + 16 * ((g >> 1) ^ (j & 1)) + 8 * (g & 1));
          kw[tt][0] = v.x;
          kw[tt][1] = v.y;
        }
      }
#pragma unroll
      for (int G = 0; G < GP; ++G) {
        kz[G] = *reinterpret_cast<const u32x4*>(Ps + 256 * GP + 64 * G + 16 * g);
        ks0[G] = *reinterpret_cast<const u32x4*>(Ps + 128 * G + 32 * g);
        ks1[G] = *reinterpret_cast<const u32x4*>(Ps + 128 * G + 32 * g + 16);
      }
#pragma unroll
      for (int G = 0; G < GP; ++G) {
        vz[G] = *reinterpret_cast<const u32x4*>(Ps + 320 * GP + 64 * G + 16 * g);
        vs0[G] = *reinterpret_cast<const u32x4*>(Ps + 128 * GP + 128 * G + 32 * g);
        vs1[G] = *reinterpret_cast<const u32x4*>(Ps + 128 * GP + 128 * G + 32 * g + 16);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const unsigned char* v = D == 128 ? Vs + 1024 * g + 64 * l16 + 16 * ((n >> 1) ^ (l16 >> 2)) + 8 * (n & 1)
                                          : Vs + 512 * g + 32 * l16 + 16 * ((n >> 1) ^ (l16 >> 3)) + 8 * (n & 1);
        vw[n] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((ka_lds_i32x2)v);
      }

      // Scores of the keys 16 g + 4 tt + e.
      f32x4 s[4];
      {
        f32x4 acc[GP][4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int G = 0; G < GP; ++G) {
            const float c = -128.f * sq[G];
            acc[G][tt] = f32x4{c, c, c, c};
#pragma unroll
            for (int x = 0; x < 2; ++x)
              acc[G][tt] = mfma16x16x32(ka_numbers(kw[tt][2 * G + x], mask), qf[G][x], acc[G][tt]);
          }
#pragma unroll
        for (int G = 0; G < GP; ++G) {
          const u32x4 z = kz[G], s0 = ks0[G], s1 = ks1[G];
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t sw = tt < 2 ? s0[2 * tt + e / 2] : s1[2 * (tt - 2) + e / 2];
              const float sc = __uint_as_float(e & 1 ? sw & 0xffff0000u : sw << 16);
              const float zf = (float)((z[tt] >> (8 * e)) & 0xffu);
              const float v = __builtin_fmaf(-zf, sq[G], acc[G][tt][e]);
              s[tt][e] = G == 0 ? sc * v : __builtin_fmaf(sc, v, s[tt][e]);
            }
        }
      }
      // Some key of the tile is masked for some row; the lane's row sees the
      // first `after` of its 16 keys.
      const bool edge = __builtin_amdgcn_readfirstlane(kv0 + kKaTile > lim0 || ok != 15u);
      const int after = (ok >> g) & 1 ? lim - kv0 - 16 * g : 0;
      if (edge) {
        asm volatile("");  // a branch, not 16 selects
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * tt + e >= after) s[tt][e] = -INFINITY;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[tt][e]);
      mt = quad_max(mt);
      // m follows the maximum only when some row has passed it by kKaSlack, and
      // p counts from m + kKaLift, so it stays below 2^-5 and most tiles rescale
      // nothing.
      const float mn = fmaxf(m, mt * a.scale_log2);  // the scale is positive
      if (!__all(mn <= m + kKaSlack)) {
        const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        lsum *= alpha;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[n] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m + kKaLift;
      float ps = 0.f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[tt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][e], a.scale_log2, -ref));
          ps += s[tt][e];
        }
      lsum += ps;
#pragma unroll
      for (int G = 0; G < GP; ++G) {
        const u32x4 z = vz[G], s0 = vs0[G], s1 = vs1[G];
        f32x4 pv[4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t sw = tt < 2 ? s0[2 * tt + e / 2] : s1[2 * (tt - 2) + e / 2];
            pv[tt][e] = s[tt][e] * __uint_as_float(e & 1 ? sw & 0xffff0000u : sw << 16);
          }
        if (edge) {  // the scale of a masked key may be anything
          asm volatile("");
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (4 * tt + e >= after) pv[tt][e] = 0.f;
        }
        u32x4 pf[2], zf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            pf[u][i] = pack_bf16x2(pv[2 * u][i], pv[2 * u + 1][i]);
            zf[u][i] = perm(z[2 * u + 1], z[2 * u], 0x0c000c00u | (uint32_t)i | (uint32_t)(4 + i) << 16) | 0xc300c300u;
          }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int n = 4 * G + x;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            o[n] = mfma16x16x32(zf[u], pf[u], o[n]);
            o[n] = mfma16x16x32(ka_numbers((uint32_t)vw[n][u], mask), pf[u], o[n]);
          }
        }
      }
      slot ^= 1;
    }

    lsum = quad_sum(lsum);
    // The end of an item that this wave has to itself, or a part of one.
    if (!joined && l16 < left) {
      if (whole) {
        const float inv = ka_inverse(a, lsum, b, lim);
        uint16_t* out = a.out + b * a.out_strides[0] + qi * a.out_strides[1] + qh * a.out_strides[2] + 4 * g;
#pragma unroll
        for (int n = 0; n < NB; ++n)
          *reinterpret_cast<u32x2*>(out + 16 * n) =
              u32x2{pack_bf16x2(o[n].x * inv, o[n].y * inv), pack_bf16x2(o[n].z * inv, o[n].w * inv)};
      } else {
        const int64_t at = ((int64_t)W * 2 + (x == x0 ? 0 : 1)) * a.prow + l16;
#pragma unroll
        for (int n = 0; n < NB; ++n) *reinterpret_cast<f32x4*>(a.part + at * D + 16 * n + 4 * g) = o[n];
        if (g == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{m, lsum};
      }
    }
    x = xe;
    if (x == before * HB + HB * nt) {
      before += nt;
      ++b;
    }
  }
  if (!joined) return;  // the same for all four waves
  const int jlen = lens.keys(a, jb);

  // Join the waves: each leaves its rows in its own stages.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* orow = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int n = 0; n < NB; ++n) *reinterpret_cast<f32x4*>(orow + l16 * OROW + 16 * n + 4 * g) = o[n];
  if (g == 0) {
    orow[16 * OROW + 2 * l16] = m;
    orow[16 * OROW + 2 * l16 + 1] = lsum;
  }
  __syncthreads();
  constexpr int PT = D / 16;  // floats per thread: 16 threads a row
  const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PT;
  if (row >= left) return;
  float top = -INFINITY, sum = 0.f, y[PT];
#pragma unroll
  for (int e = 0; e < PT; ++e) y[e] = 0.f;
  const float* parts = reinterpret_cast<const float*>(ka_smem);
  constexpr int WS = 2 * STAGE / 4;
#pragma unroll
  for (int x = 0; x < kKaWaves; ++x) top = fmaxf(top, parts[x * WS + 16 * OROW + 2 * row]);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int x = 0; x < kKaWaves; ++x) {
    const float f = __builtin_amdgcn_exp2f(parts[x * WS + 16 * OROW + 2 * row] - ref);
    sum += parts[x * WS + 16 * OROW + 2 * row + 1] * f;
#pragma unroll
    for (int e = 0; e < PT; ++e) y[e] += parts[x * WS + row * OROW + d0 + e] * f;
  }
  if (whole) {
    const int rr = 16 * block + row;
    const float inv = ka_inverse(a, sum, jb, jlen - (a.L - 1 - rr / a.group));
    uint16_t* out = a.out + jb * a.out_strides[0] + (int64_t)(rr / a.group) * a.out_strides[1] +
                    (int64_t)(h * a.group + rr % a.group) * a.out_strides[2] + d0;
#pragma unroll
    for (int e = 0; e < PT; e += 4)
      *reinterpret_cast<u32x2*>(out + e) =
          u32x2{pack_bf16x2(y[e] * inv, y[e + 1] * inv), pack_bf16x2(y[e + 2] * inv, y[e + 3] * inv)};
  } else {
    const int64_t at = (int64_t)blockIdx.x * kKaWaves * 2 * a.prow + row;
#pragma unroll
    for (int e = 0; e < PT; e += 4)
      *reinterpret_cast<f32x4*>(a.part + at * D + d0 + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
    if (d0 == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{top, sum};
  }
}

// Adds up the partial results of each query row, in the order of the waves
// that left them: NW waves a row (of the 4 of a workgroup) that take the parts
// in turn, D / 64 dimensions a lane.
template <int D, int NW>
__global__ __launch_bounds__(256) void attention_kv4_join_kernel(Kv4AttnArgs a) {
  constexpr int PER = D / 64;
  typedef float vec __attribute__((ext_vector_type(PER)));
  __shared__ float red[NW][D];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wv % NW;
  // B L Hq < 2^24: the row number fits 32 bits.
  const uint32_t row = blockIdx.x * (4 / NW) + wv / NW;
  if (row >= (uint32_t)a.B * a.L * a.Hq) return;
  const uint32_t rest = row / (uint32_t)a.Hq;
  const int hq = (int)(row - rest * (uint32_t)a.Hq), b = (int)(rest / (uint32_t)a.L);
  const int i = (int)(rest - (uint32_t)b * (uint32_t)a.L);
  const int HB = a.c.heads * a.blocks, h = hq / a.group, r = i * a.group + hq % a.group;
  const KaLens lens(a, lane);
  const int len = lens.keys(a, b), nt = ka_tiles(len);
  const int s0 = lens.before(a, b, lane) * HB + (h * a.blocks + r / 16) * nt, s1 = s0 + nt;
  const int all = lens.all * HB;
  const int W0 = ka_wave_of(s0, all), W1 = ka_wave_of(s1 - 1, all);
  // In place already: one wave's, or exactly one workgroup's.
  if (W0 == W1) return;
  if (W0 % kKaWaves == 0 && ka_start(W0, all) == s0 && ka_start(W0 + kKaWaves, all) == s1) return;

  // Which of the waves W from `first` on left a part (a lane each), and where.
  auto part_of = [&](int first, int64_t* at) {
    const int W = first + lane, i0 = W / kKaWaves * kKaWaves;
    const bool one = ka_start(i0, all) >= s0 && ka_start(i0 + kKaWaves, all) <= s1;  // joined in LDS
    *at = ((int64_t)W * 2 + (ka_start(W, all) < s0 ? 1 : 0)) * a.prow + r % 16;
    return W <= W1 && (!one || W == i0);
  };
  float top = -INFINITY;
  for (int first = W0; first <= W1; first += 64) {
    int64_t at;
    if (part_of(first, &at)) top = fmaxf(top, a.part_ml[at * 2]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  vec y = 0.f;
  for (int first = W0; first <= W1; first += 64) {
    int64_t at;
    const bool in = part_of(first, &at);
    f32x2_t ml = f32x2_t{-INFINITY, 0.f};
    if (in) ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + at * 2);
    const float f = __builtin_amdgcn_exp2f(ml.x - ref);
    sum += ml.y * f;
    // This wave's share of the parts, eight loads at a time.
    uint64_t left = __ballot(in);
    for (int skip = 0; skip < w; ++skip) left &= left - 1;
    while (left) {
      float fs[8];
      vec v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at_lane = left ? __ffsll((unsigned long long)left) - 1 : 0;
        fs[j] = left ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), at_lane)) : 0.f;
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at, at_lane);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)at >> 32), at_lane);
        v[j] = vec(0.f);
        if (left) v[j] = *reinterpret_cast<const vec*>(a.part + (int64_t)((uint64_t)hi << 32 | lo) * D + lane * PER);
#pragma unroll
        for (int skip = 0; skip < NW; ++skip) left &= left - 1;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) y += v[j] * fs[j];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if constexpr (NW > 1) {
    *reinterpret_cast<vec*>(&red[w][lane * PER]) = y;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int x = 1; x < NW; ++x) y += *reinterpret_cast<const vec*>(&red[x][lane * PER]);
  }
  const float inv = ka_inverse(a, sum, b, len - (a.L - 1 - i));
  uint16_t* out = a.out + b * a.out_strides[0] + (int64_t)i * a.out_strides[1] + (int64_t)hq * a.out_strides[2];
#pragma unroll
  for (int e = 0; e < PER; ++e) out[lane * PER + e] = (uint16_t)f32_to_bf16(y[e] * inv);
}

}  // namespace mk

// ---------------------------------------------------------------------------
// Host launcher
// ---------------------------------------------------------------------------
#include "launch.h"

#include <cmath>

namespace {

// Tiles of all items if every sequence filled its table row.
int64_t kv4_most_tiles(int64_t B, int64_t L, int64_t Hq, int64_t Hkv, int64_t width, int64_t page) {
  const int64_t items = B * Hkv * ((L * (Hq / Hkv) + 15) / 16), tiles = (width * page + mk::kKaTile - 1) / mk::kKaTile;
  return items * (tiles > 0 ? tiles : 1);
}

// Sizes both entry points take (those of the cache as kv4_view has them).
bool kv4_sizes_ok(int64_t B, int64_t L, int64_t Hq, int64_t Hkv, int64_t width, int64_t page) {
  return B >= 0 && B <= 65536 && L > 0 && L <= (1 << 20) && Hq > 0 && Hq <= 65536 && Hkv > 0 && Hkv <= 65535 &&
         Hq % Hkv == 0 && B * L <= (int64_t)1 << 30 && B * L * Hq < (int64_t)1 << 24 && width >= 0 &&
         width <= (int64_t)1 << 28 && page > 0 && page % 16 == 0 && page <= 1024 &&
         width * page <= (int64_t)1 << 28 && kv4_most_tiles(B, L, Hq, Hkv, width, page) < (int64_t)1 << 31;
}

// Workgroups that take a share of at most `most` tiles.
int64_t kv4_groups(int64_t most) {
  const int64_t full = ((int64_t)1 << mk::kKaLog) / mk::kKaWaves, need = (most + mk::kKaWaves - 1) / mk::kKaWaves;
  return need < full ? need : full;
}

int64_t kv4_part_rows(int64_t L, int64_t group) { return L * group < 16 ? L * group : 16; }

}  // namespace

extern "C" int64_t mk_attention_kv4_workspace_bytes(int64_t B, int64_t L, int64_t Hq, int64_t Hkv, int64_t D,
                                                    int64_t width, int64_t page) {
  if (!kv4_sizes_ok(B, L, Hq, Hkv, width, page) || (D != 64 && D != 128)) return -1;
  const int64_t waves = kv4_groups(kv4_most_tiles(B, L, Hq, Hkv, width, page)) * mk::kKaWaves;
  return waves * 2 * kv4_part_rows(L, Hq / Hkv) * (D + 2) * (int64_t)sizeof(float);
}

extern "C" int mk_attention_kv4_bf16(const void* q, const mk_kv4_cache* cache, const int32_t* block_table,
                                     const int32_t* lens, void* out, const int64_t* strides, int64_t B, int64_t L,
                                     int64_t Hq, int64_t width, float scale, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  mkc::clear_error();
  const char* fn = "mk_attention_kv4_bf16";
  mk::Kv4AttnArgs a;
  const int rc = mkc::kv4_view(cache, &a.c, fn);
  if (rc != MK_OK) return rc;
  if (!kv4_sizes_ok(B, L, Hq, a.c.heads, width, a.c.page))
    return mkc::fail(MK_EINVAL, "%s: bad sizes (B %lld, L %lld, %lld query heads for %d key heads, table width %lld)",
                     fn, (long long)B, (long long)L, (long long)Hq, a.c.heads, (long long)width);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return mkc::fail(MK_EINVAL, "%s: scale must be positive and finite (got %g)", fn, (double)scale);
  if (B == 0) return MK_OK;
  if (!q || !out || !lens || !strides || (width && !block_table)) return mkc::fail(MK_EINVAL, "%s: null pointer", fn);
  const int64_t dims[3] = {B, L, Hq};
  for (int i = 0; i < 6; ++i) {
    const int64_t st = mkc::stride_of(strides[i], dims[i % 3]);
    if (st < 0 || st > (int64_t)1 << 40 || st % 8)
      return mkc::fail(MK_EINVAL, "%s: stride %d (multiples of 8 elements)", fn, i);
    (i < 3 ? a.q_strides : a.out_strides)[i % 3] = st;
  }
  if (((uintptr_t)q | (uintptr_t)out) % 16) return mkc::fail(MK_EINVAL, "%s: q and out must be 16-byte aligned", fn);
  if (!mkc::runs_apart(dims, a.out_strides, cache->dim))
    return mkc::fail(MK_EINVAL, "%s: the heads of out share memory", fn);
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.table = block_table;
  a.lens = lens;
  a.width = width;
  a.B = (int)B;
  a.L = (int)L;
  a.Hq = (int)Hq;
  a.group = (int)(Hq / a.c.heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  if (!std::isfinite(a.scale_log2)) return mkc::fail(MK_EINVAL, "%s: scale %g is too large", fn, (double)scale);
  a.blocks = (int)((L * a.group + 15) / 16);
  a.page_magic = (((uint64_t)1 << 32) + a.c.page / 16 - 1) / (uint64_t)(a.c.page / 16);
  const int64_t need = mk_attention_kv4_workspace_bytes(B, L, Hq, a.c.heads, cache->dim, width, a.c.page);
  if (!workspace || workspace_bytes < need)
    return mkc::fail(MK_EWORKSPACE, "%s: needs %lld bytes of workspace, got %lld", fn, (long long)need,
                     (long long)(workspace ? workspace_bytes : 0));
  if ((uintptr_t)workspace % 16) return mkc::fail(MK_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  const int64_t groups = kv4_groups(kv4_most_tiles(B, L, Hq, a.c.heads, width, a.c.page));
  a.prow = (int)kv4_part_rows(L, a.group);
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + groups * mk::kKaWaves * 2 * a.prow * cache->dim;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)groups);
  // Four waves a row where rows are few and their parts may be many, one
  // where the rows alone fill the card (64 rows x 32 heads: 6.5 us against 11.1 with four).
  const bool wide = B * L * Hq < 1024;
  const dim3 join((unsigned)(wide ? B * L * Hq : (B * L * Hq + 3) / 4));
  const int lds = mk::kKaWaves * 2 * (2 * mk::kKaTile * (int)cache->dim / 2 + 1024);
  static std::atomic<uint64_t> done[2];
  const void* kernels[2] = {(const void*)mk::attention_kv4_kernel<64>, (const void*)mk::attention_kv4_kernel<128>};
  const int ra = mkc::lds_opt_in(kernels[cache->dim == 128], lds, done[cache->dim == 128], fn);
  if (ra != MK_OK) return ra;
  if (cache->dim == 128) {
    hipLaunchKernelGGL(mk::attention_kv4_kernel<128>, grid, dim3(256), lds, st, a);
    if (wide) hipLaunchKernelGGL((mk::attention_kv4_join_kernel<128, 4>), join, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mk::attention_kv4_join_kernel<128, 1>), join, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(mk::attention_kv4_kernel<64>, grid, dim3(256), lds, st, a);
    if (wide) hipLaunchKernelGGL((mk::attention_kv4_join_kernel<64, 4>), join, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mk::attention_kv4_join_kernel<64, 1>), join, dim3(256), 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mkc::fail(MK_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return MK_OK;
}
