// Attention over whole prompts of different lengths packed one after the
// other, with grouped heads, for gfx950.
//
// Sequence b has the query rows cu_q[b] .. cu_q[b+1] and the key rows
// cu_k[b] .. cu_k[b+1].  Query i of nq sees the keys 0 .. i + nk - nq (causal:
// the last query sees the last key), or all nk; a query that sees none gives
// zeros.  Rows from cu_q[B] on are left as they were.
//
// The Hq / Hkv query heads of a key head are packed into the rows of one
// matrix, row r being query r / group of head r % group, so that a key tile is
// read once for all of them and the rows of a tile see nearly the same keys.
// A workgroup has 256 or 128 rows of one sequence and key head, 32 a wave, and
// loops over tiles of 64 keys up to the last one that its rows see; the
// running maximum and sum of the softmax and the output stay in registers.
//   S = K Q^T: first operand K rows (lane: key 16t + l%16, 8 dimensions from
//     an XOR-swizzled LDS tile), second the wave's Q rows (registers): a lane
//     holds row l%16 and the keys 4(l/16) .. +3 of each 16.
//   O += V^T P^T: second operand P straight from those registers, rounded to
//     bf16 (the sum l takes the unrounded p); the V fragment is read transposed
//     from the rows of the same keys.  Both operands of a matrix instruction have
//     one type, and v needs the range of bf16; p in two parts would keep its
//     bits at twice the products of this half.  The rounding is half a step,
//     2^-8 of each term: against 64 bits the results are off by 0.0019 .. 0.0023
//     of their size, where rounding the result alone gives 0.0015 .. 0.0017.
// Matrix and vector work must overlap, which the two waves of a SIMD do for each
// other:
//   8 waves: two groups of 4, one wave of each on every SIMD.  A tile is two
//     phases, M(t): P V of tile t-1 and Q K of tile t, and E(t): mask, maximum,
//     exponentials and the rescale of O; the groups run them in turn, a barrier
//     between.  K and V come by LDS DMA into a ring of four stages, two tiles
//     ahead.
//   4 waves: two workgroups per CU, which drift apart by themselves (the
//     softmax at raised priority); two stages, one tile ahead.  Each one's
//     start and end lie under the other's work.
// Bound by the matrix cores and the exponentials together, one exponential for
// 4 D operations: 6097 queries of 32 heads over 24385 keys of 8 take 1.14 ms (in
// a graph), 1.05 PFLOP/s where a large product reaches 1.2.  Short prompts pay for
// the queries' loads, the first tiles and the stores around few tiles; few queries
// behind long keys for a workgroup's walk over all of them (64 of 32 heads behind
// 8192: 249 us).  With D = 128 the second pass spills 8 (4 waves: 12) registers;
// the first, which all rows take, none.
#include "wave.h"

#include <math.h>

#include <type_traits>

namespace mk {

struct PackedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, out_tok, out_head;  // strides, elements
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t Tq, Tk;
  int B, Hq, group;
  int causal;
  float scale_log2;
};

// Bound b of sequences over T rows: whatever the array holds, bounds are taken
// in 0 .. T.
__device__ __forceinline__ int packed_bound(const int32_t* cu, int b, int64_t T) {
  const int c = cu[b];
  return c < 0 ? 0 : c > T ? (int)T : c;
}

constexpr int kPaKV = 64;          // keys per tile
constexpr float kPaSlack = 8.f;    // log2 units

typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pa_s16x4* pa_lds_s16x4;

// Chunk swizzles of the LDS tiles (16-byte chunk position = chunk ^ swizzle of
// the row): the 16 rows that one K read touches, and the 16 of one transposed
// V read, spread over all banks.
template <int D>
__device__ __forceinline__ int pa_kswz(int r) {
  return D == 128 ? r & 15 : (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int pa_vswz(int r) {
  return D == 128 ? (2 * (r & 3)) | (8 * ((r >> 2) & 1)) : 2 * ((r >> 1) & 3);
}

// The first tile (of kPaRows rows) of sequence b in a grid that gives every
// sequence rows / kPaRows + 1 places without knowing the others' lengths: at
// least the tiles it has, and at most one too many.
template <int kPaRows>
__device__ __forceinline__ int64_t pa_first_tile(const PackedArgs& a, int b) {
  return (int64_t)packed_bound(a.cu_q, b, a.Tq) * a.group / kPaRows + b;
}

// A workgroup's rows: the bounds of their sequence, and the first of them.
struct PaPlace {
  int q0, nq, k0, nk, r0;
};

// Batches of up to 64 sequences (one per lane): the rank-th tile by falling
// number of key tiles, so that the longest start first and the last to start
// are short (together with maxima over lanes without LDS, built in the same step:
// 8 ragged prompts 181 -> 165 us, 6097 queries over 24385 keys 1242 -> 1153; not
// measured apart).  With n rows a tile, tile i of a sequence ends at row min(rows, n (i + 1))
// - 1, so it has c key tiles or more from i = floor(X group / n) on, X = 64 (c - 1)
// - (nk - nq) the first query that sees key 64 (c - 1); the c of the rank-th is
// found by halving.  False: there are fewer tiles.
template <int kPaRows>
__device__ __forceinline__ bool pa_by_cost(const PackedArgs& a, int rank, int lane, PaPlace* out) {
  int q0 = 0, k0 = 0, nq = 0, nk = 0;
  if (lane < a.B) {
    q0 = packed_bound(a.cu_q, lane, a.Tq);
    nq = packed_bound(a.cu_q, lane + 1, a.Tq) - q0;
    k0 = packed_bound(a.cu_k, lane, a.Tk);
    nk = packed_bound(a.cu_k, lane + 1, a.Tk) - k0;
    nq = nq > 0 ? nq : 0;
    nk = nk > 0 ? nk : 0;
  }
  const int tiles = (nq * a.group + kPaRows - 1) / kPaRows;  // nq group <= 2^30
  // Tiles of the lane's sequence with c key tiles or more.
  auto many = [&](int c) {
    if (!a.causal) return c <= (nk + kPaKV - 1) / kPaKV ? tiles : 0;
    const int X = kPaKV * (c - 1) - (nk - nq);
    return c == 0 || X <= 0 ? tiles : X < nq ? tiles - X * a.group / kPaRows : 0;
  };
  if (wave_sum(tiles) <= rank) return false;
  int lo = 0, hi = (int)((a.Tk + kPaKV - 1) / kPaKV) + 1;  // many(lo) > rank >= many(hi), summed
  int above = 0;                                           // the sum of many(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, n = wave_sum(many(mid));
    if (n > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = n;
    }
  }
  const int from = many(lo), here = from - many(lo + 1), upto = wave_scan(here), want = rank - above;
  const int at = __ffsll((unsigned long long)__ballot(upto > want)) - 1;
  out->q0 = __builtin_amdgcn_readlane(q0, at);
  out->nq = __builtin_amdgcn_readlane(nq, at);
  out->k0 = __builtin_amdgcn_readlane(k0, at);
  out->nk = __builtin_amdgcn_readlane(nk, at);
  out->r0 = kPaRows * __builtin_amdgcn_readlane(tiles - from + want - (upto - here), at);
  return true;
}

// Any number of sequences: the tiles in the order of the sequences, their last
// rows first.
template <int kPaRows>
__device__ __forceinline__ bool pa_by_order(const PackedArgs& a, int64_t tile, int lane, PaPlace* out) {
  int lo = 0, hi = a.B;  // the last sequence whose first tile is at or before this one
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, probe = lo + step * lane;
    const int n = __popcll(__ballot(probe < hi && pa_first_tile<kPaRows>(a, probe) <= tile));
    const int nlo = lo + step * (n > 0 ? n - 1 : 0);
    hi = nlo + step < hi ? nlo + step : hi;
    lo = nlo;
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  out->q0 = packed_bound(a.cu_q, b, a.Tq);
  out->nq = packed_bound(a.cu_q, b + 1, a.Tq) - out->q0;
  out->k0 = packed_bound(a.cu_k, b, a.Tk);
  out->nk = packed_bound(a.cu_k, b + 1, a.Tk) - out->k0;
  if (out->nk < 0) out->nk = 0;
  const int64_t r0 = (tile - pa_first_tile<kPaRows>(a, b)) * kPaRows;
  if (r0 < 0 || r0 >= (int64_t)out->nq * a.group) return false;
  out->r0 = (int)r0;
  return true;
}

// O += P V of one tile with the non-finite numbers of v taken as 0; rows that
// see one (in the key order of the fragments: 8 per lane from key0 and key0 +
// 16 of each 32) get NaN in its dimension.
template <int D, typename F>
__device__ __forceinline__ void pa_careful(f32x4 (&o)[2][D / 16], const u32x4 (&pf)[2][2], const int (&lim)[2],
                                           int key0, F vfrag) {
#pragma unroll 1
  for (int u = 0; u < 2; ++u) {
    u32x4 sees[2], p[2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      p[rb] = u ? pf[rb][1] : pf[rb][0];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 32 * u + (i < 2 ? 2 * i : 16 + 2 * i - 4);
        sees[rb][i] = (key <= lim[rb] ? 0x3f80u : 0u) | (key + 1 <= lim[rb] ? 0x3f800000u : 0u);
      }
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      u32x4 vf = vfrag(n, u), odd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (vf[i] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
        const uint32_t hi = (vf[i] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
        odd[i] = 0x3f803f80u & (lo | hi);
        vf[i] &= ~(lo | hi);
      }
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        o[rb][n] = mfma16x16x32(vf, p[rb], o[rb][n]);
        const f32x4 hit = mfma16x16x32(odd, sees[rb], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (hit[e] != 0.f) o[rb][n][e] = __builtin_nanf("");
      }
      __builtin_amdgcn_sched_barrier(0);  // one block's fragments at a time: registers
    }
  }
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attention_packed_kernel(PackedArgs a, int hkv) {
  constexpr int RB = 2, NS = D / 32, NB = D / 16;  // row blocks, d chunks, d blocks
  constexpr int ROWB = D * 2, CH = D / 8;          // bytes, 16-byte chunks per K / V row
  constexpr int RPI = 64 / CH;                     // rows per DMA instruction
  constexpr int PER = kPaKV / RPI / NW;            // DMA instructions per wave for a K (or V) tile
  constexpr int TILE = kPaKV * ROWB, STAGE = 2 * TILE, R = NW / 2;
  constexpr int kPaRows = 32 * NW;
  extern __shared__ __attribute__((aligned(16))) unsigned char pa_smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int h = (int)(blockIdx.x % hkv);
  PaPlace at;
  const bool any = a.B <= 64 ? pa_by_cost<kPaRows>(a, (int)(blockIdx.x / hkv), lane, &at)
                             : pa_by_order<kPaRows>(a, (int64_t)(gridDim.x / hkv) - 1 - blockIdx.x / hkv, lane, &at);
  if (!any) return;
  const int q0 = at.q0, nq = at.nq, k0 = at.k0, nk = at.nk, r0 = at.r0;
  const int rows = nq * a.group;  // <= 2^30

  // Rows of this lane (one per row block): clamped to the last, which is
  // computed again and not stored.
  const uint16_t* qrow[RB];
  int lim[RB];  // the last key the row sees
  const int wr0 = r0 / a.group, rbase = r0 - wr0 * a.group;
  const int left = rows - r0 < kPaRows ? rows - r0 : kPaRows;  // rows of this workgroup
  const int shift = a.causal ? nk - nq : 0;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    int r = 32 * w + 16 * rb + l16;
    r = rbase + (r < left ? r : left - 1);
    const int i = wr0 + r / a.group;
    lim[rb] = a.causal ? i + shift : nk - 1;
    qrow[rb] = a.q + (int64_t)(q0 + i) * a.q_tok + (int64_t)(h * a.group + r % a.group) * a.q_head;
  }
  // First and last row of the wave and the last of the workgroup.
  const int wlast = 32 * w + 31 < left ? 32 * w + 31 : left - 1;
  const bool idle = 32 * w >= left;  // no rows at all
  const int wmin = a.causal ? wr0 + (rbase + 32 * w) / a.group + shift : nk - 1;
  const int wmax = idle ? -1 : a.causal ? wr0 + (rbase + wlast) / a.group + shift : nk - 1;
  const int gmax = a.causal ? wr0 + (rbase + left - 1) / a.group + shift : nk - 1;
  const int nt = gmax < 0 ? 0 : gmax / kPaKV + 1;

  u32x4 qf[RB][NS];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[rb][s] = *reinterpret_cast<const u32x4*>(qrow[rb] + 8 * (4 * s + g));

  const uint32_t sbase = lds_addr(pa_smem);
  const uint16_t* kb = a.k + (int64_t)k0 * a.k_tok + (int64_t)h * a.k_head;
  const uint16_t* vb = a.v + (int64_t)k0 * a.v_tok + (int64_t)h * a.v_head;
  // DMA instruction I = PER w + u of a tile fills rows RPI I .. of K, then of
  // V; the source chunk is the one that the swizzle puts in the lane's place.
  // Rows behind the last key are copies of it (their scores are masked).
  auto issue = [&](int t) {
    const uint32_t st = sbase + (uint32_t)((t % R) * STAGE);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int row = RPI * (PER * w + u) + lane / CH, p = lane % CH;
      const int j = t * kPaKV + row < nk ? t * kPaKV + row : nk - 1;
      dma16_asm(kb + j * a.k_tok + 8 * (p ^ pa_kswz<D>(row)), st + (uint32_t)((PER * w + u) * 1024));
      dma16_asm(vb + j * a.v_tok + 8 * (p ^ pa_vswz<D>(row)), st + (uint32_t)(TILE + (PER * w + u) * 1024));
    }
  };

  f32x4 o[RB][NB], sacc[RB][4];
  u32x4 pf[RB][2];
  float m[RB], lsum[RB];
  const int vr_r = l16 >> 2, vr_q = l16 & 3;
  // The V fragment of d block n and 32 keys u.
  auto vfrag = [&](const unsigned char* Vs, int n, int u) {
    const int c = 2 * n + (vr_q >> 1), hb = 8 * (vr_q & 1);
    const int ra = 32 * u + 4 * g + vr_r, rz = ra + 16;
    const pa_s16x4 va = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (pa_lds_s16x4)(Vs + ra * ROWB + 16 * (c ^ pa_vswz<D>(ra)) + hb));
    const pa_s16x4 vz = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (pa_lds_s16x4)(Vs + rz * ROWB + 16 * (c ^ pa_vswz<D>(rz)) + hb));
    const u32x2 x = __builtin_bit_cast(u32x2, va), y = __builtin_bit_cast(u32x2, vz);
    return u32x4{x.x, x.y, y.x, y.y};
  };
  // Phase boundaries, the same for every wave.  Before phase 2u the wave's
  // part of tile u has landed (tile u+1 may be in flight), and behind the
  // barrier everyone's; everyone is then done with M(u-1), the last reader of
  // tile u-2, whose stage takes tile u+2.
  int phase = 0;
  auto boundary = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if ((phase & 1) == 0) {
      const int u = phase >> 1;
      if (u + 1 < nt) vm_wait(2 * PER);
      else vm_wait(0);
      asm volatile("s_barrier" ::: "memory");
      if (u + 2 < nt) issue(u + 2);
    } else {
      asm volatile("s_barrier" ::: "memory");
    }
    ++phase;
    __builtin_amdgcn_sched_barrier(0);
  };

  // In a tile that some rows see only in part, a NaN or an infinity of v
  // would reach all of them through the products with p = 0.  The first pass
  // takes no notice; if it leaves a NaN in any row, the second computes such
  // tiles again with v's non-finite numbers taken as 0, and marks the outputs
  // of the rows that see one.
  auto pass = [&](auto careful_t) {
    constexpr bool careful = decltype(careful_t)::value;
    // S = K Q^T of tile t.
    auto scores = [&](int t) {
      if (t * kPaKV > wmax) return;  // no row of the wave sees any of it
      const unsigned char* Ks = pa_smem + (t % R) * STAGE;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) sacc[rb][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int j = 16 * tt + l16;
          const u32x4 kf = *reinterpret_cast<const u32x4*>(Ks + j * ROWB + 16 * ((4 * s + g) ^ pa_kswz<D>(j)));
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sacc[rb][tt] = mfma16x16x32(kf, qf[rb][s], sacc[rb][tt]);
        }
    };
    // Mask, maximum, exponentials, P, and the rescale of O.
    auto softmax = [&](int t) {
      const int kv0 = t * kPaKV;
      if (kv0 > wmax) return;
      if (kv0 + kPaKV - 1 > wmin) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (kv0 + 16 * tt + 4 * g + e > lim[rb]) sacc[rb][tt][e] = -INFINITY;
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        // The scale (log2 units) is positive, so the maximum of the scaled
        // scores is the scaled maximum.
        float mt = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e) mt = fmaxf(mt, sacc[rb][tt][e]);
        mt = quad_max(mt);
        // m follows the maximum only when some row of the block has passed it
        // by kPaSlack, and p counts from m + kPaSlack, so it stays below 1 and
        // most tiles rescale nothing (long prompts 1149 -> 1137 us).
        const float mn = fmaxf(m[rb], mt * a.scale_log2);
        if (!__all(mn <= m[rb] + kPaSlack)) {
          const float alpha = __builtin_amdgcn_exp2f(m[rb] - (mn == -INFINITY ? 0.f : mn));
          m[rb] = mn;
          lsum[rb] *= alpha;
#pragma unroll
          for (int n = 0; n < NB; ++n) o[rb][n] *= alpha;
        }
        const float ref = m[rb] == -INFINITY ? 0.f : m[rb] + kPaSlack;  // (a row that has seen nothing yet)
        float ps = 0.f;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[rb][tt][e], a.scale_log2, -ref));
            sacc[rb][tt][e] = p;
            ps += p;
          }
        lsum[rb] += ps;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          pf[rb][u] = u32x4{pack_bf16x2(sacc[rb][2 * u][0], sacc[rb][2 * u][1]),
                            pack_bf16x2(sacc[rb][2 * u][2], sacc[rb][2 * u][3]),
                            pack_bf16x2(sacc[rb][2 * u + 1][0], sacc[rb][2 * u + 1][1]),
                            pack_bf16x2(sacc[rb][2 * u + 1][2], sacc[rb][2 * u + 1][3])};
      }
    };
    // O += P V of tile t.
    auto values = [&](int t) {
      if (t * kPaKV > wmax) return;
      const unsigned char* Vs = pa_smem + (t % R) * STAGE + TILE;
      if (!careful || t * kPaKV + kPaKV - 1 <= wmin) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u32x4 vf = vfrag(Vs, n, u);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) o[rb][n] = mfma16x16x32(vf, pf[rb][u], o[rb][n]);
          }
      } else {
        pa_careful<D>(o, pf, lim, t * kPaKV + 4 * g, [&](int n, int u) { return vfrag(Vs, n, u); });
      }
    };
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      lsum[rb] = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n) o[rb][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (nt > 0) issue(0);
    if constexpr (NW == 8) {
      phase = 0;
      if (nt > 1) issue(1);
      if (w >= 4) boundary();
      for (int t = 0; t <= nt; ++t) {
        boundary();
        if (t > 0) values(t - 1);
        if (t == nt) break;
        scores(t);
        boundary();
        softmax(t);
      }
      if (w < 4) boundary();
    } else {
      for (int t = 0; t < nt; ++t) {
        // This wave's part of tile t has landed and behind the barrier
        // everyone's; the other stage has been read.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < nt) issue(t + 1);
        scores(t);
        __builtin_amdgcn_s_setprio(1);
        softmax(t);
        __builtin_amdgcn_s_setprio(0);
        values(t);
      }
    }
  };

  pass(std::false_type{});
  if (a.causal) {
    bool nan = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) nan = nan || o[rb][n][e] != o[rb][n][e];
    if (__syncthreads_or(nan)) pass(std::true_type{});
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    // No key seen: zeros; only scores of -infinity: NaN.
    const float l = quad_sum(lsum[rb]);
    const float inv = l == 0.f && lim[rb] < 0 ? 0.f : 1.0f / l;
    const int r = 32 * w + 16 * rb + l16;
    if (r >= left) continue;
    const int rr = rbase + r;
    uint16_t* out = a.out + (int64_t)(q0 + wr0 + rr / a.group) * a.out_tok +
                    (int64_t)(h * a.group + rr % a.group) * a.out_head + 4 * g;
#pragma unroll
    for (int n = 0; n < NB; ++n)
      *reinterpret_cast<u32x2*>(out + 16 * n) = u32x2{pack_bf16x2(o[rb][n].x * inv, o[rb][n].y * inv),
                                                      pack_bf16x2(o[rb][n].z * inv, o[rb][n].w * inv)};
  }
}

}  // namespace mk

// ---------------------------------------------------------------------------
// Host launcher
// ---------------------------------------------------------------------------
#include "launch.h"

#include <cmath>

namespace {

template <int D, int NW>
int packed_launch(const mk::PackedArgs& a, unsigned grid, int hkv, hipStream_t st, const char* fn) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = NW / 2 * 2 * mk::kPaKV * D * 2;
  const int rc = mkc::lds_opt_in((const void*)mk::attention_packed_kernel<D, NW>, lds, done, fn);
  if (rc != MK_OK) return rc;
  hipLaunchKernelGGL((mk::attention_packed_kernel<D, NW>), dim3(grid), dim3(64 * NW), lds, st, a, hkv);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mkc::fail(MK_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return MK_OK;
}

}  // namespace

extern "C" int mk_attention_packed_bf16(const void* q, const void* k, const void* v, void* out, const int64_t* strides,
                                        const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int64_t B,
                                        int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hkv, int64_t D, int causal,
                                        float scale, void* stream) {
  mkc::clear_error();
  const char* fn = "mk_attention_packed_bf16";
  if (B < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return mkc::fail(MK_EINVAL, "%s: bad sizes", fn);
  if (D != 64 && D != 128) return mkc::fail(MK_EUNSUPPORTED, "%s: head dim %lld (64 or 128)", fn, (long long)D);
  if (Hq % Hkv)
    return mkc::fail(MK_EINVAL, "%s: %lld query heads for %lld key heads", fn, (long long)Hq, (long long)Hkv);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return mkc::fail(MK_EINVAL, "%s: scale must be positive and finite (got %g)", fn, (double)scale);
  if (B > (1 << 24) || Hq > 65536 || Hkv > 65536 || Tq > (1 << 28) || Tk > (1 << 28) || Tq * Hq > (int64_t)1 << 30)
    return mkc::fail(MK_EINVAL, "%s: shape too large", fn);
  if (B == 0 || Tq == 0) return MK_OK;
  if (!q || !out || !strides || !cu_seqlens_q || !cu_seqlens_k || (Tk && (!k || !v)))
    return mkc::fail(MK_EINVAL, "%s: null pointer", fn);
  int64_t st8[8];
  for (int i = 0; i < 8; ++i) {
    const bool of_q = i < 2 || i > 5;
    st8[i] = mkc::stride_of(strides[i], i & 1 ? (of_q ? Hq : Hkv) : of_q ? Tq : Tk);
    if (st8[i] < 0 || st8[i] > (int64_t)1 << 40 || st8[i] % 8)
      return mkc::fail(MK_EINVAL, "%s: stride %d (multiples of 8 elements)", fn, i);
  }
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16)
    return mkc::fail(MK_EINVAL, "%s: q, k, v and out must be 16-byte aligned", fn);
  if (!mkc::runs_apart({Tq, Hq, 1}, {st8[6], st8[7], 0}, D))
    return mkc::fail(MK_EINVAL, "%s: the heads of out share memory", fn);
  mk::PackedArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.q_tok = st8[0]; a.q_head = st8[1];
  a.k_tok = st8[2]; a.k_head = st8[3];
  a.v_tok = st8[4]; a.v_head = st8[5];
  a.out_tok = st8[6]; a.out_head = st8[7];
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.Tq = Tq;
  a.Tk = Tk;
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.group = (int)(Hq / Hkv);
  a.causal = causal ? 1 : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  if (!std::isfinite(a.scale_log2)) return mkc::fail(MK_EINVAL, "%s: scale %g is too large", fn, (double)scale);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // 8 waves and phases where sequences are long (one of 8192 keys: 568 against
  // 585 us with 4 waves, 6097 queries over 24385 keys 1177 / 1230), 4 waves and
  // two workgroups per CU elsewhere (16 of 1024: 219 / 231 us, 8 ragged ones of
  // 64 .. 2100: 157 / 166, 4 of 1 .. 300: 13.1 / 17.7; even at 4096).  The rule
  // takes the mean length, keys behind the last sequence included.  With few
  // queries behind long keys either can win (8192 keys, 8 / 4 waves: 1 query 189
  // / 217 us, 64 249 / 222, 1024 252 / 224, 64 in each of 8 sequences 264 / 275),
  // and one long prompt among short ones has 4 (8192 and seven of 1: 561 / 575).
  const bool big = Tk / B >= 4096;
  const int64_t tiles = Tq * a.group / (big ? 256 : 128) + B;
  if (!mkc::grid_fits(tiles * Hkv, big ? 512 : 256)) return mkc::fail(MK_EINVAL, "%s: shape too large", fn);
  const unsigned grid = (unsigned)(tiles * Hkv);
  const int kv = (int)Hkv;
  if (D == 128) return big ? packed_launch<128, 8>(a, grid, kv, st, fn) : packed_launch<128, 4>(a, grid, kv, st, fn);
  return big ? packed_launch<64, 8>(a, grid, kv, st, fn) : packed_launch<64, 4>(a, grid, kv, st, fn);
}
