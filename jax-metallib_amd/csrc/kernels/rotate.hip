// Norms of queries and keys for each head, with the rotary positions in the
// same pass, for gfx950.
//
//   y = rot(x * rsqrt(mean(x^2) + eps) * g)     (x alone without a gain)
//
// over the D dimensions of one token and head; rot turns the pairs of the
// first R dimensions by the angles of the token's position,
//   (a, b) -> (a c - b s, b c + a s),  c, s = row `position` of the tables,
// pair i being dimensions (i, i + R/2) (half) or (2i, 2i + 1) (interleaved);
// the dimensions from R on are only normalised.  Everything between the load
// and the one rounding at the store is f32.
//
// Layout: a lane holds 8 dimensions that are 4 pairs: runs of 4 at 4c and
// R/2 + 4c (half, 8 bytes a load), or one run of 8 at 8c (interleaved, and the
// part that is not turned), so a pair never leaves its lane and both layouts
// read tables entries 4c .. 4c + 3.  A row takes D/8 lanes, a wave 64 / (lanes
// per row) heads of one token at a time, and the norm is a sum over those
// lanes by row shifts.  A workgroup is 4 waves of one token, each with U
// groups of heads whose loads are all in flight before the first is used.
// Bound by HBM with many tokens (8191 of 40 heads, 169 MB: 38.5 us, 4.4 TB/s),
// by launch and two dependent loads (position, then table row) with few.
#include "wave.h"

namespace mk {

struct RotateArgs {
  const void* in[2];     // q, k
  void* out[2];
  const void* gain[2];   // null: no norm
  int64_t in_tok[2], in_head[2], out_tok[2], out_head[2];  // strides, elements
  const int32_t* pos;
  const float* cosb;
  const float* sinb;
  int64_t table_len;
  int64_t T;
  int Hq, H;     // query heads, query and key heads
  int D, R;
  float eps;
  bool clear[2];  // padding rows are zeros, else left as they were
};

// 4 elements of a lane as they are in memory.
template <typename E>
struct RotRun;
template <>
struct RotRun<float> {
  f32x4 v;
  __device__ __forceinline__ float at(int i) const { return v[i]; }
};
template <>
struct RotRun<uint16_t> {
  u32x2 v;
  __device__ __forceinline__ float at(int i) const {
    return i & 1 ? __uint_as_float(v[i >> 1] & 0xffff0000u) : __uint_as_float(v[i >> 1] << 16);
  }
};

// The outputs are not read here again: stored past the L2's lines in use (8191
// tokens of 40 heads: 38.7 us, against 43.7 with plain stores).  What reads them
// next loses by it what this gains, no more: rotation in place, cache and packed
// attention of 8191 tokens take 169.5 us either way, of 500 29.9.
__device__ __forceinline__ void rot_store(float* p, const float (&f)[8], int i) {
  __builtin_nontemporal_store(f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]}, reinterpret_cast<f32x4*>(p));
}
__device__ __forceinline__ void rot_store(uint16_t* p, const float (&f)[8], int i) {
  __builtin_nontemporal_store(u32x2{pack_bf16x2(f[i], f[i + 1]), pack_bf16x2(f[i + 2], f[i + 3])},
                              reinterpret_cast<u32x2*>(p));
}

template <int CTRL>
__device__ __forceinline__ float rot_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// The sum over LPR neighbouring lanes, in each of them.
template <int LPR>
__device__ __forceinline__ float rot_sum(float v) {
  v += rot_dpp<0xb1>(v);   // quad_perm 1 0 3 2
  v += rot_dpp<0x4e>(v);   // quad_perm 2 3 0 1
  v += rot_dpp<0x141>(v);  // row_half_mirror
  if constexpr (LPR > 8) v += rot_dpp<0x140>(v);  // row_mirror
  if constexpr (LPR > 16) {
    const wave_u2 x = swap16(v);
    v = __uint_as_float(x.x) + __uint_as_float(x.y);
  }
  if constexpr (LPR > 32) {
    const wave_u2 x = swap32(v);
    v = __uint_as_float(x.x) + __uint_as_float(x.y);
  }
  return v;
}

// LPR lanes per row (a power of two >= D/8).  Workgroup (t, y): token t, head
// groups 4 U y .. 4 U y + 4 U - 1, wave w those at w, w + 4, ..
template <typename E, int LPR, bool INTER, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RotateArgs a) {
  constexpr int HPW = 64 / LPR;
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 63, c = lane % LPR;
  const int first = ((int)blockIdx.y * 4 * U + (int)(threadIdx.x >> 6)) * HPW + lane / LPR;
  const int pos = a.pos[t];
  const bool turn = 8 * c < a.R;
  const int off0 = !INTER && turn ? 4 * c : 8 * c;
  const int off1 = !INTER && turn ? a.R / 2 + 4 * c : 8 * c + 4;
  RotRun<E> lo[U], hi[U];
  bool mine[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = first + 4 * i * HPW;
    mine[i] = 8 * c < a.D && h < a.H;
    lo[i].v = hi[i].v = 0;
    if (mine[i]) {
      const int part = h < a.Hq ? 0 : 1;
      const E* src = static_cast<const E*>(a.in[part]) + t * a.in_tok[part] + (h - (part ? a.Hq : 0)) * a.in_head[part];
      lo[i] = *reinterpret_cast<const RotRun<E>*>(src + off0);
      hi[i] = *reinterpret_cast<const RotRun<E>*>(src + off1);
    }
  }
  if (pos < 0) {  // padding
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = first + 4 * i * HPW, part = h < a.Hq ? 0 : 1;
      if (!mine[i] || !a.clear[part]) continue;
      const float zeros[8] = {};
      E* dst = static_cast<E*>(a.out[part]) + t * a.out_tok[part] + (h - (part ? a.Hq : 0)) * a.out_head[part];
      rot_store(dst + off0, zeros, 0);
      rot_store(dst + off1, zeros, 4);
    }
    return;
  }
  const bool known = pos < a.table_len;
  f32x4 cv = {1.f, 1.f, 1.f, 1.f}, sv = {0.f, 0.f, 0.f, 0.f};
  if (turn && known) {
    cv = *reinterpret_cast<const f32x4*>(a.cosb + (int64_t)pos * (a.R / 2) + 4 * c);
    sv = *reinterpret_cast<const f32x4*>(a.sinb + (int64_t)pos * (a.R / 2) + 4 * c);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = first + 4 * i * HPW;
    float y[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = lo[i].at(e);
      y[4 + e] = hi[i].at(e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += y[e] * y[e];
    sum = rot_sum<LPR>(sum);
    if (!mine[i]) continue;
    const int part = h < a.Hq ? 0 : 1;
    const E* g = static_cast<const E*>(a.gain[part]);
    if (g) {
      const float r = 1.0f / sqrtf(sum / (float)a.D + a.eps);
      const RotRun<E> g0 = *reinterpret_cast<const RotRun<E>*>(g + off0);
      const RotRun<E> g1 = *reinterpret_cast<const RotRun<E>*>(g + off1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = y[e] * r * g0.at(e);
        y[4 + e] = y[4 + e] * r * g1.at(e);
      }
    }
    if (turn) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = INTER ? 2 * e : e, q = INTER ? 2 * e + 1 : 4 + e;
        const float u = y[p], v = y[q];
        y[p] = u * cv[e] - v * sv[e];
        y[q] = v * cv[e] + u * sv[e];
      }
    }
    if (!known) {  // a position the tables do not hold
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __builtin_nanf("");
    }
    E* dst = static_cast<E*>(a.out[part]) + t * a.out_tok[part] + (h - (part ? a.Hq : 0)) * a.out_head[part];
    rot_store(dst + off0, y, 0);
    rot_store(dst + off1, y, 4);
  }
}

}  // namespace mk

// ---------------------------------------------------------------------------
// Host launcher
// ---------------------------------------------------------------------------
#include "launch.h"

#include <algorithm>
#include <cmath>

namespace {

template <typename E, int LPR, bool INTER>
void rotate_launch_u(const mk::RotateArgs& a, int u, dim3 grid, hipStream_t st) {
  if (u == 1) hipLaunchKernelGGL((mk::qk_norm_rope_kernel<E, LPR, INTER, 1>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mk::qk_norm_rope_kernel<E, LPR, INTER, 3>), grid, dim3(256), 0, st, a);
}

template <typename E, int LPR>
void rotate_launch_l(const mk::RotateArgs& a, int layout, int u, dim3 grid, hipStream_t st) {
  if (layout == MK_ROPE_INTERLEAVED) rotate_launch_u<E, LPR, true>(a, u, grid, st);
  else rotate_launch_u<E, LPR, false>(a, u, grid, st);
}

template <typename E>
void rotate_launch(const mk::RotateArgs& a, int lpr, int layout, int u, dim3 grid, hipStream_t st) {
  switch (lpr) {
    case 8: rotate_launch_l<E, 8>(a, layout, u, grid, st); break;
    case 16: rotate_launch_l<E, 16>(a, layout, u, grid, st); break;
    case 32: rotate_launch_l<E, 32>(a, layout, u, grid, st); break;
    default: rotate_launch_l<E, 64>(a, layout, u, grid, st); break;
  }
}

}  // namespace

extern "C" int mk_qk_norm_rope(int dtype, const void* q, const void* k, void* q_out, void* k_out,
                               const int64_t* strides, const int32_t* positions, const float* cos_table,
                               const float* sin_table, int64_t table_len, const void* g_q, const void* g_k, float eps,
                               int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t R, int layout, void* stream) {
  mkc::clear_error();
  const char* fn = "mk_qk_norm_rope";
  if (dtype != MK_DT_F32 && dtype != MK_DT_BF16) return mkc::fail(MK_EUNSUPPORTED, "%s: dtype %d", fn, dtype);
  const int flags = layout & (MK_ROPE_CLEAR_Q | MK_ROPE_CLEAR_K);
  layout -= flags;
  if (layout != MK_ROPE_HALF && layout != MK_ROPE_INTERLEAVED)
    return mkc::fail(MK_EINVAL, "%s: layout %d", fn, layout);
  if (T < 0 || Hq < 0 || Hkv < 0 || Hq + Hkv <= 0 || D <= 0 || R < 0 || table_len < 0)
    return mkc::fail(MK_EINVAL, "%s: bad sizes", fn);
  if (D % 8 || D > 512) return mkc::fail(MK_EUNSUPPORTED, "%s: head dim %lld (a multiple of 8, at most 512)", fn,
                                         (long long)D);
  if (R % 8 || R > D) return mkc::fail(MK_EUNSUPPORTED, "%s: rotary dim %lld (a multiple of 8, at most the head dim)",
                                       fn, (long long)R);
  if (!mkc::grid_fits(T, 256) || Hq > 65536 || Hkv > 65536 || table_len > (int64_t)1 << 31)
    return mkc::fail(MK_EINVAL, "%s: shape too large", fn);
  if (T == 0) return MK_OK;
  if (!strides || !positions || (Hq && (!q || !q_out)) || (Hkv && (!k || !k_out)) ||
      (R && (!cos_table || !sin_table)))
    return mkc::fail(MK_EINVAL, "%s: null pointer", fn);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return mkc::fail(MK_EINVAL, "%s: eps must be finite and >= 0", fn);
  const uintptr_t step = dtype == MK_DT_F32 ? 16 : 8;  // bytes of a lane's run of 4 elements
  uintptr_t bits = 0;
  if (Hq) bits |= (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)g_q;
  if (Hkv) bits |= (uintptr_t)k | (uintptr_t)k_out | (uintptr_t)g_k;
  int64_t odd = 0, sd[8];
  for (int i = 0; i < 8; ++i) {
    sd[i] = mkc::stride_of(strides[i], i & 1 ? (i & 2 ? Hkv : Hq) : i & 2 && !Hkv ? 0 : !(i & 2) && !Hq ? 0 : T);
    if (sd[i] < 0 || sd[i] > (int64_t)1 << 40) return mkc::fail(MK_EINVAL, "%s: stride %d", fn, i);
    odd |= sd[i];
  }
  if (bits % step || odd % 4 || ((uintptr_t)cos_table | (uintptr_t)sin_table) % 16)
    return mkc::fail(MK_EINVAL, "%s: heads must start at multiples of 4 elements, tables at 16 bytes", fn);
  if (!mkc::runs_apart({T, Hq, 1}, {sd[4], sd[5], 0}, D) || !mkc::runs_apart({T, Hkv, 1}, {sd[6], sd[7], 0}, D))
    return mkc::fail(MK_EINVAL, "%s: an output's heads share memory", fn);
  mk::RotateArgs a;
  a.in[0] = q; a.in[1] = k;
  a.out[0] = q_out; a.out[1] = k_out;
  a.gain[0] = g_q; a.gain[1] = g_k;
  a.in_tok[0] = sd[0]; a.in_head[0] = sd[1];
  a.in_tok[1] = sd[2]; a.in_head[1] = sd[3];
  a.out_tok[0] = sd[4]; a.out_head[0] = sd[5];
  a.out_tok[1] = sd[6]; a.out_head[1] = sd[7];
  a.pos = positions;
  a.cosb = cos_table;
  a.sinb = sin_table;
  a.table_len = table_len;
  a.T = T;
  a.Hq = (int)Hq;
  a.H = (int)(Hq + Hkv);
  a.D = (int)D;
  a.R = (int)R;
  a.eps = eps;
  a.clear[0] = flags & MK_ROPE_CLEAR_Q;
  a.clear[1] = flags & MK_ROPE_CLEAR_K;
  int lpr = 8;
  while (8 * lpr < D) lpr *= 2;
  const int groups = (a.H * lpr + 63) / 64;
  // Three head groups a wave once the tokens alone are enough workgroups (8191
  // tokens of 40 heads: 38.6 us against 41.9 with one; 16 tokens: 2.1 us with one
  // against 2.8 with two).
  const int u = T >= 1024 && groups > 4 ? 3 : 1;
  const dim3 grid((unsigned)T, (unsigned)((groups + 4 * u - 1) / (4 * u)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MK_DT_F32) rotate_launch<float>(a, lpr, layout, u, grid, st);
  else rotate_launch<uint16_t>(a, lpr, layout, u, grid, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mkc::fail(MK_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return MK_OK;
}
