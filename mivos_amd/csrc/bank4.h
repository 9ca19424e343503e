// The 4-bit memory bank (mivos_bank4) seen from device code: a row of D channels is D/32 blocks of 32 codes (sign, two exponent bits,
// one mantissa bit; two to a byte, the even channel in the low half) and one scale byte each, value = code * 2^(byte - 127).
// Every such value has at most two significant bits, so it is exact in bf16 for all the scales the bank writes (bytes 7..252).
#pragma once
#include "common.h"

namespace mivos {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kBank4NanScale = 255;   // the block held an infinity or a NaN

// scale byte -> the fp32 power of two the conversion instructions take (255 -> NaN: they answer NaN for every code)
__device__ __forceinline__ float bank4_scale(uint32_t byte) {
  return __uint_as_float((byte << 23) | (byte == kBank4NanScale ? 0x400000u : 0u));
}

// 8 codes of one block (low half of the first byte first) -> 8 bf16 values, exactly
__device__ __forceinline__ bf16x8 bank4_unpack8(uint32_t codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  const bf16x4 lo = __builtin_shufflevector(a, b, 0, 1, 2, 3), hi = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The same in fp16: exact where bank4_fits_f16 says so.
__device__ __forceinline__ f16x8 bank4_unpack8_f16(uint32_t codes, float scale) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
  const f16x4 lo = __builtin_shufflevector(a, b, 0, 1, 2, 3), hi = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// 0.5 * 2^(byte - 127) >= 2^-24 and 6 * 2^(byte - 127) <= 6 * 2^13, or a block of zeros (under kBank4NanScale too: the conversion answers NaN)
constexpr uint32_t kBank4F16Least = 104, kBank4F16Most = 140;
__device__ __forceinline__ bool bank4_zeros(u32x4 codes) { return ((codes[0] | codes[1] | codes[2] | codes[3]) & 0x77777777u) == 0; }
// (most: a smaller limit of the caller's)
__device__ __forceinline__ bool bank4_fits_f16(uint32_t byte, u32x4 codes, uint32_t most = kBank4F16Most) {
  return (byte >= kBank4F16Least && byte <= most) || bank4_zeros(codes);
}

// 8 consecutive elements of a row as fp32; `vec`: the address is a multiple of 16 bytes
template <typename T>
__device__ __forceinline__ f32x8 load8(const T *p, bool vec) {
  f32x8 r;
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
      r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      typedef T Tx8 __attribute__((ext_vector_type(8)));
      const Tx8 a = *reinterpret_cast<const Tx8 *>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = (float)a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (float)p[i];
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T *p, f32x8 v) {   // 16-byte aligned
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4 *>(p)[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    reinterpret_cast<f32x4 *>(p)[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  } else {
    typedef T Tx8 __attribute__((ext_vector_type(8)));
    Tx8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
    *reinterpret_cast<Tx8 *>(p) = a;
  }
}

inline bool dtype_ok(int dtype) { return dtype == MIVOS_F32 || dtype == MIVOS_F16 || dtype == MIVOS_BF16; }
inline int dtype_bytes(int dtype) { return dtype == MIVOS_F32 ? 4 : 2; }

// host-side checks shared by the bank entry points
inline int bank4_check(const mivos_bank4 *k, const char *what) {
  if (!k || !k->key_codes || !k->key_scales || !k->value_codes || !k->value_scales || !k->weight || !k->lens || !k->status)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: null bank pointer", what);
  if (k->batch < 1 || k->heads < 1 || k->slots < 1 || k->slots > (1ll << 30) || (int64_t)k->batch * k->heads > 65535)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: bank of %d x %d heads x %lld slots", what, k->batch, k->heads, (long long)k->slots);
  if (k->key_dim < 32 || k->key_dim > 1024 || k->key_dim % 32 || k->value_dim < 32 || k->value_dim > 1024 || k->value_dim % 32)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: key / value rows of %d / %d channels (multiples of 32 up to 1024)", what, k->key_dim, k->value_dim);
  if (((uintptr_t)k->key_codes | (uintptr_t)k->key_scales | (uintptr_t)k->value_codes | (uintptr_t)k->value_scales) & 15)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: codes and scales must be 16-byte aligned", what);
  return MIVOS_OK;
}

struct Span {
  uintptr_t first, end;
  Span(const void *p, int64_t bytes) : first((uintptr_t)p), end((uintptr_t)p + bytes) {}
  bool meets(const Span &o) const { return first < o.end && o.first < end; }
};
// whether a buffer of the one bank shares memory with a buffer of the other
inline bool bank4_meet(const mivos_bank4 &x, const mivos_bank4 &y) {
  auto spans = [](const mivos_bank4 &k, auto &&use) {
    const int64_t rows = (int64_t)k.batch * k.heads * k.slots;
    return use(Span(k.key_codes, rows * k.key_dim / 2)) || use(Span(k.key_scales, rows * k.key_dim / 32)) || use(Span(k.value_codes, rows * k.value_dim / 2)) ||
           use(Span(k.value_scales, rows * k.value_dim / 32)) || use(Span(k.weight, rows * 4)) || use(Span(k.lens, (int64_t)k.batch * 4)) ||
           use(Span(k.status, (int64_t)(1 + k.batch) * 4));
  };
  return spans(x, [&](const Span &a) { return spans(y, [&](const Span &b) { return a.meets(b); }); });
}

}  // namespace mivos
