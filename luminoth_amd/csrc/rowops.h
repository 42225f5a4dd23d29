// Building blocks of the row-wise kernels (lnorm.hip, logprobs.hip): 16-byte loads of fp32 / f16 / bf16 rows at any
// element alignment, and sums over 16, 64, 256 or 1024 threads in a fixed order (gfx950).
#pragma once
#include "lmh_common.h"

#ifdef __HIPCC__
enum { LMH_F32 = LMH_DTYPE_F32, LMH_F16 = LMH_DTYPE_F16, LMH_BF16 = LMH_DTYPE_BF16 };

struct f32_t { float v; };
struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };

template <typename T> struct row_type;
template <> struct row_type<f32_t> { static constexpr int VEC = 4; };
template <> struct row_type<f16_t> { static constexpr int VEC = 8; };
template <> struct row_type<bf16_t> { static constexpr int VEC = 8; };

// 16 bytes of a row as they lie in memory.  The hardware takes a 16-byte access at any element's address (the compiler emits
// ONE global_load_dwordx4 for this type), so rows of odd length or of a wider buffer need no scalar path: only the last,
// partial vector of a row is read element by element.
typedef uint32_t raw16 __attribute__((ext_vector_type(4)));
typedef uint32_t raw16_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t raw16_a2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T> __device__ __forceinline__ raw16 load16(const T* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const raw16_a4*>(p);
  else return *reinterpret_cast<const raw16_a2*>(p);
}
template <typename T> __device__ __forceinline__ void store16(T* p, raw16 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<raw16_a4*>(p) = v;
  else *reinterpret_cast<raw16_a2*>(p) = v;
}
template <typename T> __device__ __forceinline__ float elem(const raw16& r, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(r[e]);
  } else {
    const uint16_t h = (uint16_t)(r[e >> 1] >> (16 * (e & 1)));
    if constexpr (__is_same(T, f16_t)) return (float)__builtin_bit_cast(_Float16, h);
    else return __uint_as_float((e & 1) ? (r[e >> 1] & 0xffff0000u) : (r[e >> 1] << 16));
  }
}
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v.v; }
template <typename T> __device__ __forceinline__ T from_f32(float f) {      // round to nearest even
  T t;
  if constexpr (sizeof(T) == 4) t.v = f;
  else if constexpr (__is_same(T, f16_t)) t.v = (_Float16)f;
  else t.v = (__bf16)f;
  return t;
}
template <typename T> __device__ __forceinline__ raw16 pack16(const float* f) {
  raw16 r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = __builtin_bit_cast(uint16_t, from_f32<T>(f[2 * e])), hi = __builtin_bit_cast(uint16_t, from_f32<T>(f[2 * e + 1]));
      r[e] = lo | (hi << 16);
    }
  }
  return r;
}
// The last vector of a row, `rem` < VEC values (the same for every lane: a row's length modulo VEC): 8, 4 and 2 bytes at a time, as
// its bits say, so at most three accesses instead of seven.
typedef uint32_t raw8_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t raw8_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t raw4_a2 __attribute__((aligned(2)));
template <typename T> __device__ __forceinline__ raw16 load_tail(const T* p, int rem, uint32_t fill) {
  raw16 r = {fill, fill, fill, fill};
  if constexpr (sizeof(T) == 4) {
    if (rem & 2) {
      const raw8_a4 v = *reinterpret_cast<const raw8_a4*>(p);
      r[0] = v[0];
      r[1] = v[1];
      if (rem & 1) r[2] = *reinterpret_cast<const uint32_t*>(p + 2);
    } else {
      r[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  } else {
    auto one = [&](int i) { return (fill & 0xffff0000u) | *reinterpret_cast<const uint16_t*>(p + i); };
    if (rem & 4) {
      const raw8_a2 v = *reinterpret_cast<const raw8_a2*>(p);
      r[0] = v[0];
      r[1] = v[1];
      if (rem & 2) {
        r[2] = *reinterpret_cast<const raw4_a2*>(p + 4);
        if (rem & 1) r[3] = one(6);
      } else if (rem & 1) {
        r[2] = one(4);
      }
    } else if (rem & 2) {
      r[0] = *reinterpret_cast<const raw4_a2*>(p);
      if (rem & 1) r[1] = one(2);
    } else {
      r[0] = one(0);
    }
  }
  return r;
}
template <typename T> __device__ __forceinline__ void store_tail(T* p, int rem, raw16 r) {
  if constexpr (sizeof(T) == 4) {
    if (rem & 2) {
      *reinterpret_cast<raw8_a4*>(p) = raw8_a4{r[0], r[1]};
      if (rem & 1) *reinterpret_cast<uint32_t*>(p + 2) = r[2];
    } else {
      *reinterpret_cast<uint32_t*>(p) = r[0];
    }
  } else {
    auto one = [&](int i, uint32_t v) { *reinterpret_cast<uint16_t*>(p + i) = (uint16_t)v; };
    if (rem & 4) {
      *reinterpret_cast<raw8_a2*>(p) = raw8_a2{r[0], r[1]};
      if (rem & 2) {
        *reinterpret_cast<raw4_a2*>(p + 4) = r[2];
        if (rem & 1) one(6, r[3]);
      } else if (rem & 1) {
        one(4, r[2]);
      }
    } else if (rem & 2) {
      *reinterpret_cast<raw4_a2*>(p) = r[0];
      if (rem & 1) one(2, r[1]);
    } else {
      one(0, r[0]);
    }
  }
}
// Columns [col, col + VEC) of a row of D, col a multiple of VEC; `fill` (two 16-bit values or one of 32) behind its end.
template <typename T> __device__ __forceinline__ raw16 load_cols(const T* row, int col, int D, uint32_t fill = 0) {
  constexpr int VEC = row_type<T>::VEC;
  raw16 r = {fill, fill, fill, fill};
  if (col + VEC <= D) r = load16(row + col);
  else if (col < D) r = load_tail(row + col, D & (VEC - 1), fill);
  return r;
}
template <typename T> __device__ __forceinline__ void store_cols(T* row, int col, int D, const float* f) {
  constexpr int VEC = row_type<T>::VEC;
  if (col + VEC <= D) store16(row + col, pack16<T>(f));
  else if (col < D) store_tail(row + col, D & (VEC - 1), pack16<T>(f));
}

// N parameters from column `col` on, `fill` where there are none.
template <int N, typename P> __device__ __forceinline__ void load_params(float* out, const P* p, int col, int D, float fill) {
  constexpr int VEC = row_type<P>::VEC < N ? row_type<P>::VEC : N;
#pragma unroll
  for (int i = 0; i < N; i += VEC) {
    raw16 r = {0, 0, 0, 0};
    if (p && VEC == row_type<P>::VEC) r = load_cols(p, col + i, D);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      out[i + e] = fill;
      if (p && col + i + e < D) out[i + e] = VEC == row_type<P>::VEC ? elem<P>(r, e) : to_f32(p[col + i + e]);
    }
  }
}

// ---- sums and maxima over lanes -------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp_mov(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
struct op_add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct op_max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// Every lane of a 16-lane row gets the row's result: quads (two permutations), halves and the row mirrored.
template <typename OP> __device__ __forceinline__ float reduce16(float v, OP op) {
  v = op(v, dpp_mov<0xB1>(v));      // lane ^ 1
  v = op(v, dpp_mov<0x4E>(v));      // lane ^ 2
  v = op(v, dpp_mov<0x141>(v));     // mirrored inside 8
  return op(v, dpp_mov<0x140>(v));  // mirrored inside 16
}
template <typename OP> __device__ __forceinline__ float reduce64(float v, OP op) {
  v = reduce16(v, op);
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
// Over the TPR threads that share a row.  TPR > 64: `red` (TPR / 64 floats of LDS per group, one group a block there) is
// written before ONE barrier and read behind it: a caller that loops alternates between two arrays.
template <int TPR, typename OP> __device__ __forceinline__ float reduce_row(float v, OP op, float* red) {
  if constexpr (TPR == 16) {
    return reduce16(v, op);
  } else {
    v = reduce64(v, op);
    if constexpr (TPR > 64) {
      if ((threadIdx.x & 63) == 0) red[(threadIdx.x & (TPR - 1)) >> 6] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int i = 1; i < TPR / 64; ++i) v = op(v, red[i]);
    }
    return v;
  }
}
#endif  // __HIPCC__
