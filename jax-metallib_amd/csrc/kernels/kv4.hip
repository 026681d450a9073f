// Quantising keys and values to 4 bits as they enter the paged cache, and
// reading them back, for gfx950 (the format: kv4.h).
//
// Of the 64 values x of one group, with t = max(x, 0) and l = min(x, 0),
//   s = bf16((t - l) / 15),  z = clamp(round(-l / s)),
//   n = clamp(round(x / s) + z)     (halves to even, clamped to 0 .. 15).
// x is divided by the scale that is kept, so the quotients of two numbers of
// 8 significant bits decide the rounding: the correctly rounded f32 quotient
// rounds to the same whole number as the exact one, and n is determined by x
// alone.  s is off by at most 2^-8 of itself, so a value read back is within
// s (1/2 + 15 2^-8) of the one written.  A group without a step to count in
// (s below the smallest normal f32) is kept as zeros; one that holds a NaN or
// an infinity reads back as NaN.
//
// Layout: a lane holds 8 dimensions (16 bytes in, one dword out) of the key and
// of the value, a group is 8 lanes.  Both directions are one pass.  8000 tokens
// of 8 heads of 128 (in a graph): in 11.3 us (3.7 TB/s), bound by its 374 vector
// instructions a wave, 4 keys and values (counted: 9.7 us of issue); back to bf16
// in 7.8 (5.4 TB/s, partly from the cache), to f32 in 37 (2.0 TB/s; each lane's
// 32 bytes go out in two stores).
#include "kv4.h"

namespace mk {

struct Kv4Rows {
  const uint16_t* in[2];  // k, v of the tokens (append)
  void* out[2];           // (read)
  int64_t tok[2], head[2];  // their strides, elements
  const int64_t* slots;
  int64_t T;
  uint64_t page_magic;  // ceil(2^32 / (page / 16))
  int64_t near;         // slots below it are divided by the magic number
  Kv4View c;
};

template <int CTRL>
__device__ __forceinline__ uint32_t kv4_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}

// The page and the place in it of a slot of the cache; a multiplication
// for slots below `near`.
__device__ __forceinline__ void kv4_place(const Kv4Rows& a, int64_t slot, int64_t* page, int* place) {
  if (slot < a.near) {
    const uint32_t pg = (uint32_t)((((uint64_t)slot >> 4) * a.page_magic) >> 32);
    *page = pg;
    *place = (int)((uint32_t)slot - pg * (uint32_t)a.c.page);
  } else {
    *page = slot / a.c.page;
    *place = (int)(slot - *page * a.c.page);
  }
}

// x / 15, correctly rounded: one correction of x (1/15) by its exact remainder
// (a quotient by 15 is no nearer than 1/30 of a unit to the middle of two).
__device__ __forceinline__ float kv4_15th(float x) {
  constexpr float r = 1.f / 15.f;
  const float q = x * r;
  return __builtin_fmaf(__builtin_fmaf(-15.f, q, x), r, q);
}

// Scale, zero point and the lane's 8 numbers of a group of 64 values, 8 to a
// lane; the 8 lanes are neighbours and all active.
__device__ __forceinline__ uint32_t kv4_quantise(const u32x4& xw, uint32_t* scale, uint32_t* zero) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(xw[i] << 16);
    x[2 * i + 1] = __uint_as_float(xw[i] & 0xffff0000u);
  }
  float top = 0.f, low = 0.f;
  uint32_t mag = 0;  // the largest magnitude's bits: NaN and infinity from 0x7f800000
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = fmaxf(top, x[i]);
    low = fminf(low, x[i]);
    const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
    mag = mag > b ? mag : b;
  }
#define MK_KV4_STEP(CTRL)                                                             \
  {                                                                                   \
    top = fmaxf(top, __uint_as_float(kv4_dpp<CTRL>(__float_as_uint(top))));           \
    low = fminf(low, __uint_as_float(kv4_dpp<CTRL>(__float_as_uint(low))));           \
    const uint32_t o = kv4_dpp<CTRL>(mag);                                            \
    mag = mag > o ? mag : o;                                                          \
  }
  MK_KV4_STEP(0xb1)   // quad_perm 1 0 3 2
  MK_KV4_STEP(0x4e)   // quad_perm 2 3 0 1
  MK_KV4_STEP(0x141)  // row_half_mirror
#undef MK_KV4_STEP
  // (top - low) / 15; halved where the difference of two large numbers would
  // pass the f32 range.
  const float span = top - low;
  const float s = bf16_to_f32(f32_to_bf16(span < INFINITY ? kv4_15th(span) : 2.f * kv4_15th(0.5f * top - 0.5f * low)));
  *zero = 0;
  *scale = 0;
  if (mag >= 0x7f800000u) {
    *scale = 0x7fc0;
    return 0;
  }
  if (s < 0x1p-126f) return 0;
  *scale = f32_to_bf16(s);
  float n[8], z;
  if (s >= 0x1p-60f) {
    // x / s as x r and one correction by its exact remainder.  What is rounded
    // next is a quotient of two numbers of 8 significant bits below 16: it is
    // either a half exactly, and then the correction hits it, or 2^-11 away
    // from any, far beyond the error of x r.
    const float r0 = __builtin_amdgcn_rcpf(s);
    const float r = __builtin_fmaf(__builtin_fmaf(-s, r0, 1.f), r0, r0);
    auto quotient = [&](float v) {
      const float q = v * r;
      return __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
    };
    z = rintf(quotient(-low));
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = rintf(quotient(x[i]));
  } else {  // remainders near the smallest numbers are not exact
    z = rintf(-low / s);
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = rintf(x[i] / s);
  }
  z = fminf(z, 15.f);
  *zero = (uint32_t)z;
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = __builtin_amdgcn_fmed3f(n[i] + z, 0.f, 15.f);
  // Four numbers at a time as one exact f32 below 2^16.
  uint32_t half[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    half[i] = (uint32_t)__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(n[4 * i + 3], 16.f, n[4 * i + 2]), 16.f,
                                                      n[4 * i + 1]), 16.f, n[4 * i]);
  return half[0] | half[1] << 16;
}

// The row (token, head) of a thread: D / 8 threads a row, a workgroup 16 tokens
// of one head (two of 64 dimensions), so that neighbouring rows are neighbours
// in a page and their scales and zero points share lines (8000 tokens of 8
// heads in and out, when this was chosen: 20.8 us, against 21.6 with the heads of
// a token one after the other; 18.6 since places and scales are multiplications).
template <int D>
__device__ __forceinline__ bool kv4_row(const Kv4Rows& a, uint32_t* t, uint32_t* h) {
  const uint32_t row = threadIdx.x / (D / 8);
  *t = 16 * blockIdx.x + (row & 15);
  *h = blockIdx.y * (128 / D) + (row >> 4);
  return *t < (uint32_t)a.T && *h < (uint32_t)a.c.heads;
}

template <int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Rows a) {
  constexpr int GP = D / kKv4Group;
  const int w = threadIdx.x % (D / 8);
  uint32_t t, h;
  if (!kv4_row<D>(a, &t, &h)) return;  // whole rows, and a group's lanes are of one row
  const int64_t slot = a.slots[t];
  u32x4 x[2];
#pragma unroll
  for (int part = 0; part < 2; ++part)
    x[part] = *reinterpret_cast<const u32x4*>(a.in[part] + t * a.tok[part] + h * a.head[part] + 8 * w);
  if (slot < 0 || slot >= a.c.pages * a.c.page) return;
  int64_t pg;
  int place;
  kv4_place(a, slot, &pg, &place);
  const int64_t ph = pg * a.c.heads + h;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t scale, zero;
    const uint32_t word = kv4_quantise(x[part], &scale, &zero);
    const Kv4Half c = part ? a.c.v : a.c.k;
    uint32_t* dst = reinterpret_cast<uint32_t*>(c.rows + (ph * a.c.page + place) * (D / 2));
    dst[part ? w : kv4_word<D>(w)] = word;
    if ((w & 7) == 0) {
      const int64_t at = (ph * GP + (w >> 3)) * a.c.page + place;
      c.scale[at] = (uint16_t)scale;
      c.zero[at] = (uint8_t)zero;
    }
  }
}

template <int D, typename E>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Rows a) {
  constexpr int GP = D / kKv4Group;
  const int w = threadIdx.x % (D / 8);
  uint32_t t, h, word[2] = {0, 0}, scale[2] = {0, 0}, zero[2] = {0, 0};
  if (!kv4_row<D>(a, &t, &h)) return;
  const int64_t slot = a.slots[t];
  if (slot >= 0 && slot < a.c.pages * a.c.page) {  // else zeros
    int64_t pg;
    int place;
    kv4_place(a, slot, &pg, &place);
    const int64_t ph = pg * a.c.heads + h, at = (ph * GP + (w >> 3)) * a.c.page + place;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const Kv4Half c = part ? a.c.v : a.c.k;
      word[part] =
          reinterpret_cast<const uint32_t*>(c.rows + (ph * a.c.page + place) * (D / 2))[part ? w : kv4_word<D>(w)];
      scale[part] = c.scale[at];
      zero[part] = c.zero[at];
    }
  }
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const float s = bf16_to_f32(scale[part]), z = (float)(zero[part] & 15);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = ((float)((word[part] >> (4 * i)) & 15u) - z) * s;
    E* dst = static_cast<E*>(a.out[part]) + t * a.tok[part] + h * a.head[part] + 8 * w;
    if constexpr (sizeof(E) == 4) {
      __builtin_nontemporal_store(f32x4{y[0], y[1], y[2], y[3]}, reinterpret_cast<f32x4*>(dst));
      __builtin_nontemporal_store(f32x4{y[4], y[5], y[6], y[7]}, reinterpret_cast<f32x4*>(dst + 4));
    } else {
      __builtin_nontemporal_store(u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                        pack_bf16x2(y[6], y[7])},
                                  reinterpret_cast<u32x4*>(dst));
    }
  }
}

}  // namespace mk

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
#include "launch.h"

namespace mkc {

int kv4_view(const mk_kv4_cache* c, mk::Kv4View* out, const char* fn) {
  if (!c || !c->k || !c->k_scale || !c->k_zero || !c->v || !c->v_scale || !c->v_zero)
    return fail(MK_EINVAL, "%s: null pointer", fn);
  if (c->pages <= 0 || c->heads <= 0 || c->page <= 0 || c->dim <= 0)
    return fail(MK_EINVAL, "%s: cache sizes must be positive", fn);
  if (c->dim != 64 && c->dim != 128)
    return fail(MK_EUNSUPPORTED, "%s: head dim %lld (64 or 128)", fn, (long long)c->dim);
  if (c->page % 16 || c->page > 1024)
    return fail(MK_EUNSUPPORTED, "%s: pages of %lld (a multiple of 16, at most 1024)", fn, (long long)c->page);
  if (c->heads > 65535 || c->pages > 0x7fffffff) return fail(MK_EINVAL, "%s: cache too large", fn);
  const uintptr_t bits = (uintptr_t)c->k | (uintptr_t)c->k_scale | (uintptr_t)c->k_zero | (uintptr_t)c->v |
                         (uintptr_t)c->v_scale | (uintptr_t)c->v_zero;
  if (bits % 16) return fail(MK_EINVAL, "%s: the cache's arrays must be 16-byte aligned", fn);
  out->k = {static_cast<uint8_t*>(c->k), static_cast<uint16_t*>(c->k_scale), static_cast<uint8_t*>(c->k_zero)};
  out->v = {static_cast<uint8_t*>(c->v), static_cast<uint16_t*>(c->v_scale), static_cast<uint8_t*>(c->v_zero)};
  out->pages = c->pages;
  out->heads = (int)c->heads;
  out->page = (int)c->page;
  return MK_OK;
}

}  // namespace mkc

namespace {

// The checks and arguments that both directions share; the number of blocks
// or -1.
int rows_args(mk::Kv4Rows* a, const mk_kv4_cache* cache, const void* k, const void* v, const int64_t* strides,
              const int64_t* slots, int64_t T, size_t elem, const char* fn) {
  const int rc = mkc::kv4_view(cache, &a->c, fn);
  if (rc != MK_OK) return rc;
  if (T < 0 || !mkc::grid_fits(T / 16 + 1, 256)) return mkc::fail(MK_EINVAL, "%s: %lld tokens", fn, (long long)T);
  if (T == 0) return MK_OK;
  if (!k || !v || !strides || !slots) return mkc::fail(MK_EINVAL, "%s: null pointer", fn);
  for (int i = 0; i < 4; ++i) {
    const int64_t st = mkc::stride_of(strides[i], i & 1 ? a->c.heads : T);
    if (st < 0 || st > (int64_t)1 << 40 || st * elem % 16)
      return mkc::fail(MK_EINVAL, "%s: stride %d (16-byte multiples)", fn, i);
    (i & 1 ? a->head : a->tok)[i >> 1] = st;
  }
  if (((uintptr_t)k | (uintptr_t)v) % 16) return mkc::fail(MK_EINVAL, "%s: k and v must be 16-byte aligned", fn);
  a->slots = slots;
  a->T = T;
  // (slot / 16) (page / 16) below 2^32 makes the product's error less than one
  // part of the page; the slot itself stays below 2^32 too.
  const int64_t d = a->c.page / 16;
  a->page_magic = (((uint64_t)1 << 32) + d - 1) / d;
  a->near = (((int64_t)1 << 32) / d < (int64_t)1 << 28 ? ((int64_t)1 << 32) / d : (int64_t)1 << 28) * 16;
  return MK_OK;
}

// A workgroup per 16 tokens and head (two heads of 64 dimensions).
dim3 rows_grid(const mk::Kv4Rows& a, int64_t dim) {
  return dim3((unsigned)((a.T + 15) / 16), (unsigned)((a.c.heads * dim + 127) / 128));
}

}  // namespace

extern "C" int mk_kv4_append(const mk_kv4_cache* cache, const void* k, const void* v, const int64_t* strides,
                             const int64_t* slots, int64_t T, void* stream) {
  mkc::clear_error();
  const char* fn = "mk_kv4_append";
  mk::Kv4Rows a;
  const int rc = rows_args(&a, cache, k, v, strides, slots, T, 2, fn);
  if (rc != MK_OK) return rc;
  if (T == 0) return MK_OK;
  a.in[0] = static_cast<const uint16_t*>(k);
  a.in[1] = static_cast<const uint16_t*>(v);
  a.out[0] = a.out[1] = nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid = rows_grid(a, cache->dim);
  if (cache->dim == 128) hipLaunchKernelGGL(mk::kv4_append_kernel<128>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(mk::kv4_append_kernel<64>, grid, dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mkc::fail(MK_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return MK_OK;
}

extern "C" int mk_kv4_read(const mk_kv4_cache* cache, int dtype, void* k, void* v, const int64_t* strides,
                           const int64_t* slots, int64_t T, void* stream) {
  mkc::clear_error();
  const char* fn = "mk_kv4_read";
  if (dtype != MK_DT_F32 && dtype != MK_DT_BF16) return mkc::fail(MK_EUNSUPPORTED, "%s: dtype %d", fn, dtype);
  mk::Kv4Rows a;
  const int rc = rows_args(&a, cache, k, v, strides, slots, T, dtype == MK_DT_F32 ? 4 : 2, fn);
  if (rc != MK_OK) return rc;
  if (T == 0) return MK_OK;
  for (int i = 0; i < 2; ++i)
    if (!mkc::runs_apart({T, a.c.heads, 1}, {a.tok[i], a.head[i], 0}, cache->dim))
      return mkc::fail(MK_EINVAL, "%s: an output's heads share memory", fn);
  a.in[0] = a.in[1] = nullptr;
  a.out[0] = k;
  a.out[1] = v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid = rows_grid(a, cache->dim);
  if (cache->dim == 128) {
    if (dtype == MK_DT_F32) hipLaunchKernelGGL((mk::kv4_read_kernel<128, float>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mk::kv4_read_kernel<128, uint16_t>), grid, dim3(256), 0, st, a);
  } else {
    if (dtype == MK_DT_F32) hipLaunchKernelGGL((mk::kv4_read_kernel<64, float>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((mk::kv4_read_kernel<64, uint16_t>), grid, dim3(256), 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mkc::fail(MK_ELAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return MK_OK;
}
