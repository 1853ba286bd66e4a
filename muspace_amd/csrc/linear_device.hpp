// Building blocks of the dense-layer kernels (linear_kernels.hpp): 16-byte
// pieces of a row ("chunks"), their layouts in LDS and the matrix instructions.
//
// A chunk is 16 bytes of a row: 8 values of a 16-bit type or 4 float32 values.
// The matrix cores multiply 16-bit values sixteen times as fast as float32 ones,
// so float32 operands are multiplied as sums of three bfloat16 numbers, x = x1 +
// x2 + x3 (split_chunk): each takes the next 8 bits of x, rounded, which leaves
// |x2| <= 2^-8 |x| and |x3| <= 2^-16 |x|, and x3 what is left of 24 bits exactly.
// Of the nine products those of planes i + j <= 4 are taken, six; the rest is
// under 2^-23 |x y| for a product x y, the size of float32's own two roundings, and
// of random sign. bfloat16's smallest number is 2^-133, so float32 values keep an
// absolute 2^-134: those under 2^-109 keep fewer than 24 bits. Infinities, NaN and
// numbers that round to an infinity in bfloat16 make such a sum an infinity or NaN: a
// tile with one in it is multiplied again in float32.
//
// A tile of an operand (of one plane) is staged in LDS in one of two layouts, by
// how the operand lies in memory against the product's summed index k:
//
//   along    k is the contiguous index (x and W of x W^T). LDS holds a row of
//            128 bytes (a plane of float32: 64) per tile row, the step's values of
//            k. A chunk sits in its slot XOR a key of the row, so that 16 rows of
//            one chunk column, what an access serves at a time, touch each of the
//            64 banks once.
//   across   k is the row index (both operands of dz^T x, W of dz W). LDS holds a
//            row per k. 16-bit values are read with the transposing LDS read
//            (four rows of 16 values per 16 lanes): 32-byte pieces are moved by XOR
//            with a key of k, so that the four rows' two neighbouring pieces, what
//            32 lanes read at a time, lie in different banks. float32 values are
//            read a dword a lane, 32 consecutive ones a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "msda_device.hpp"

namespace dense {

using msda::bf16_t;
using msda::from_float;
using msda::to_float;

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kRowBytes = 128;  // of k per row of an operand and step

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// values per chunk, and k per step
template <typename T>
struct Piece {
  static constexpr int kValues = 16 / static_cast<int>(sizeof(T));
  static constexpr int kStep = kRowBytes / static_cast<int>(sizeof(T));
};

// A chunk at any alignment of its type: global_load_dwordx4 takes byte
// addresses, the packed type tells the compiler so.
struct __attribute__((packed, aligned(2))) Loose16 {
  u32x4 v;
};

template <typename T>
__device__ __forceinline__ void unpack(const u32x4 &v, float (&o)[Piece<T>::kValues]);
template <>
__device__ __forceinline__ void unpack<float>(const u32x4 &v, float (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(v[i]);
}
template <>
__device__ __forceinline__ void unpack<bf16_t>(const u32x4 &v, float (&o)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = __uint_as_float(v[i] << 16);
    o[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const u32x4 &v, float (&o)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = __half2float(__ushort_as_half(static_cast<unsigned short>(v[i] & 0xffffu)));
    o[2 * i + 1] = __half2float(__ushort_as_half(static_cast<unsigned short>(v[i] >> 16)));
  }
}

template <typename T>
__device__ __forceinline__ uint32_t bits_of(T v);
template <>
__device__ __forceinline__ uint32_t bits_of<float>(float v) {
  return __float_as_uint(v);
}
template <>
__device__ __forceinline__ uint32_t bits_of<bf16_t>(bf16_t v) {
  return v.bits;
}
template <>
__device__ __forceinline__ uint32_t bits_of<__half>(__half v) {
  return __half_as_ushort(v);
}

// Two values, rounded to nearest even by one conversion instruction (gfx950's; NaN
// stays NaN).
__device__ __forceinline__ uint32_t pack_pair_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ uint32_t pack_pair_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// round to nearest even, once: the results' only rounding below 32 bits
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&v)[Piece<T>::kValues]);
template <>
__device__ __forceinline__ u32x4 pack<float>(const float (&v)[4]) {
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
               __float_as_uint(v[3])};
}
template <>
__device__ __forceinline__ u32x4 pack<__half>(const float (&v)[8]) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = pack_pair_f16(v[2 * i], v[2 * i + 1]);
  }
  return o;
}
template <>
__device__ __forceinline__ u32x4 pack<bf16_t>(const float (&v)[8]) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_pair_bf16(v[2 * i], v[2 * i + 1]);
  return o;
}

// ------------------------------------------------------------ row loads ---

// Loads of one operand's chunks. kTight: every chunk starts on a 16-byte
// boundary and a row's length is a whole number of chunks; the loads are then
// unconditional buffer loads, whose range check returns zeros past the operand.
// Otherwise rows start anywhere: every chunk is one load at its own alignment, a row's
// last as the row's last 16 bytes, whose values drop_front moves to the front; only
// rows shorter than a chunk are read value by value (loose_load).
struct Source {
  const char *base;   // first byte of the step's window (uniform)
  uint32_t bytes;     // of the window: what lies beyond reads as zero
};

__device__ __forceinline__ u32x4 tight_load(const Source &s, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.base), 0, s.bytes, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
#else
  return u32x4{};
#endif
}

__device__ __forceinline__ uint32_t tight_load_byte(const Source &s, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.base), 0, s.bytes, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b8(r, offset, 0, 0);
#else
  return 0;
#endif
}

__device__ __forceinline__ u32x2 tight_load8(const Source &s, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.base), 0, s.bytes, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0);
#else
  return u32x2{};
#endif
}

__device__ __forceinline__ uint32_t tight_load4(const Source &s, uint32_t offset) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.base), 0, s.bytes, 0x00020000);
  return __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
#else
  return 0;
#endif
}

constexpr uint32_t kPast = 0x80000000u;  // an offset past every window

// `left` values of a row from `p` on (at most a chunk of them; none when <= 0)
template <typename T>
__device__ __forceinline__ u32x4 loose_load(const T *p, int left) {
  if (left >= Piece<T>::kValues) return reinterpret_cast<const Loose16 *>(p)->v;
  u32x4 o = {0, 0, 0, 0};
  if (left > 0) {
#pragma unroll
    for (int i = 0; i < Piece<T>::kValues; ++i) {
      if (i < left) {
        const uint32_t b = bits_of(p[i]);
        if constexpr (sizeof(T) == 4) {
          o[i] = b;
        } else {
          o[i / 2] |= b << (16 * (i & 1));
        }
      }
    }
  }
  return o;
}

// A chunk whose first `skip` values are another's: the rest, moved to the front,
// zeros behind (skip at or over a chunk's values: zeros).
template <typename T>
__device__ __forceinline__ u32x4 drop_front(const u32x4 &v, int skip) {
  const int bits = skip * 8 * static_cast<int>(sizeof(T));
  const uint64_t lo = v[0] | static_cast<uint64_t>(v[1]) << 32;
  const uint64_t hi = v[2] | static_cast<uint64_t>(v[3]) << 32;
  const int b = bits & 63;
  const uint64_t hi_down = hi >> b;
  const uint64_t lo_down = b == 0 ? lo : (lo >> b | hi << (64 - b));
  const uint64_t o_lo = bits < 64 ? lo_down : (bits < 128 ? hi_down : 0);
  const uint64_t o_hi = bits < 64 ? hi_down : 0;
  return u32x4{static_cast<uint32_t>(o_lo), static_cast<uint32_t>(o_lo >> 32),
               static_cast<uint32_t>(o_hi), static_cast<uint32_t>(o_hi >> 32)};
}

template <typename T>
__device__ __forceinline__ void loose_store(T *p, const u32x4 &v, int left) {
  if (left >= Piece<T>::kValues) {
    reinterpret_cast<Loose16 *>(p)->v = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < Piece<T>::kValues; ++i) {
    if (i < left) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<uint32_t *>(p)[i] = v[i];
      } else {
        reinterpret_cast<uint16_t *>(p)[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
      }
    }
  }
}

// ------------------------------------------------- masks and 8-bit codes ---

// Keep the values whose bit is set (the others become zero, whatever they are).
template <typename T>
__device__ __forceinline__ u32x4 keep_bits(u32x4 v, uint32_t bits) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      o[i] = v[i] & static_cast<uint32_t>(-static_cast<int>((bits >> i) & 1u));
    } else {
      const uint32_t lo = static_cast<uint32_t>(-static_cast<int>((bits >> (2 * i)) & 1u));
      const uint32_t hi = static_cast<uint32_t>(-static_cast<int>((bits >> (2 * i + 1)) & 1u));
      o[i] = v[i] & ((lo & 0xffffu) | (hi & 0xffff0000u));
    }
  }
  return o;
}

// The value of a scale byte: 2^(s - 127); 255 stands for a block that held an
// infinity or NaN and reads back as NaN.
__device__ __forceinline__ float scale_value(uint32_t s) {
  // s is at least 1 by construction (the writer clamps), so 2^(s - 127) is normal
  return __uint_as_float(s == 255u ? 0x7fc00000u : s << 23);
}

// Values of a chunk from its codes. code * 2^e needs 7 bits and is exact in every
// type (the writer keeps e within the type's range).
template <typename T>
__device__ __forceinline__ u32x4 decode(const uint32_t (&w)[Piece<T>::kValues / 4], float scale) {
  float v[Piece<T>::kValues];
#pragma unroll
  for (int i = 0; i < Piece<T>::kValues; ++i) {
    const int code = static_cast<int>(w[i / 4] << (24 - 8 * (i & 3))) >> 24;
    v[i] = static_cast<float>(code) * scale;
  }
  return pack<T>(v);
}

// lane l's value from lane l ^ kDistance, where the lanes of each aligned group of
// kDistance hold the same (1 and 2: any values)
template <int kDistance>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
  // lanes 1 0 3 2; 2 3 0 1; a mirrored half row of 8
  constexpr int kMove = kDistance == 1 ? 0xB1 : kDistance == 2 ? 0x4E : 0x141;
  return __builtin_amdgcn_mov_dpp(static_cast<int>(v), kMove, 0xf, 0xf, true);
#else
  return v;
#endif
}

// A chunk's codes and its block's scale byte. The 32 / kV neighbouring lanes that hold a
// block's chunks call it together. A block shares 2^e, the smallest power of two with 127 *
// 2^e >= its largest magnitude; a code is the nearest integer to x / 2^e (ties to even).
// The byte is e + 127, or 255 for a block with an infinity or NaN. e stays where 2^e is a
// normal number (and, for float16, a float16 number), and codes end at 63 where 64 * 2^e is
// past the type's range, so that every code * 2^e is a number of the type.
template <typename T>
__device__ __forceinline__ uint32_t encode(const float (&v)[Piece<T>::kValues],
                                           uint32_t (&w)[Piece<T>::kValues / 4]) {
  constexpr int kV = Piece<T>::kValues;
  constexpr bool kHalf = std::is_same_v<T, __half>;
  constexpr int kLow = kHalf ? 127 - 24 : 1, kHigh = kHalf ? 127 + 10 : 127 + 122;
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = max(top, from_lane<1>(top));
  top = max(top, from_lane<2>(top));
  if constexpr (kV == 4) top = max(top, from_lane<4>(top));
  const bool finite = top < 0x7f800000u;
  // 127 * 2^e reaches top = 1.f * 2^E from E - 6 on, one later if 1.f > 127 / 64
  const int s = max(kLow, static_cast<int>(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u));
  const float inverse = __uint_as_float(static_cast<uint32_t>(254 - s) << 23);
  const float limit = s >= kHigh ? 63.0f : 127.0f;
#pragma unroll
  for (int i = 0; i < kV / 4; ++i) w[i] = 0;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    float q = rintf(v[e] * inverse);
    q = finite ? fminf(fmaxf(q, -limit), limit) : 1.0f;  // 1 * NaN reads back as NaN
    w[e / 4] |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xffu) << (8 * (e & 3));
  }
  return finite ? static_cast<uint32_t>(s) : 255u;
}

// The chunk at `col` of a row's checkpoint: codes [rows][padded], scales [rows][padded / 32].
template <typename T>
__device__ __forceinline__ void keep_codes(uint8_t *codes, uint8_t *scales, int64_t row, int col,
                                           int padded,
                                           const uint32_t (&w)[Piece<T>::kValues / 4],
                                           uint32_t scale) {
  uint8_t *to = codes + row * padded + col;
  if constexpr (Piece<T>::kValues == 8) {
    *reinterpret_cast<u32x2 *>(to) = u32x2{w[0], w[1]};
  } else {
    *reinterpret_cast<uint32_t *>(to) = w[0];
  }
  if (col % 32 == 0) scales[row * (padded / 32) + col / 32] = static_cast<uint8_t>(scale);
}

// ---------------------------------------------------------- gelu's slope ---

// What gelu's backward needs of a pre-activation is the derivative there, and it lies in
// [-0.129, 1.129]: sixteen bits hold it closer than they hold z. From 2^-5 on a code counts
// steps of 2^-15 (an error of 2^-16 at most; rounding z would cost up to 2^-9.6 in bfloat16,
// 2^-12.6 in float16), below that it is the float16 number, which keeps the relative
// accuracy of the tails. float32 keeps the derivative itself.
constexpr uint32_t kTailCodes = 0x2800u;               // float16 numbers under 2^-5
constexpr uint32_t kZeroStep = 2 * kTailCodes + 4230u;  // code of step 0; steps from -4229 on
constexpr uint32_t kSlopeNan = 0xffffu;

__device__ __forceinline__ uint32_t slope_code(float s) {
  const uint32_t tail = __half_as_ushort(__float2half(fabsf(s)));
  const uint32_t step = kZeroStep + static_cast<uint32_t>(static_cast<int>(rintf(s * 32768.0f)));
  const uint32_t code = tail < kTailCodes ? tail + (s < 0.0f ? kTailCodes : 0u) : step;
  return s == s ? code : kSlopeNan;
}

__device__ __forceinline__ float slope_value(uint32_t code) {
  const bool below = code >= kTailCodes;
  const float tail = __half2float(__ushort_as_half(
      static_cast<unsigned short>(below ? code - kTailCodes : code)));
  const float step = static_cast<float>(static_cast<int>(code) - static_cast<int>(kZeroStep)) *
                     0x1p-15f;
  const float s = code >= 2 * kTailCodes ? step : below ? -tail : tail;
  return code == kSlopeNan ? __uint_as_float(0x7fc00000u) : s;
}

// A chunk of derivatives as it is kept.
template <typename T>
__device__ __forceinline__ u32x4 pack_slopes(const float (&s)[Piece<T>::kValues]) {
  if constexpr (sizeof(T) == 4) {
    return pack<T>(s);
  } else {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = slope_code(s[2 * i]) | slope_code(s[2 * i + 1]) << 16;
    return o;
  }
}
template <typename T>
__device__ __forceinline__ void unpack_slopes(const u32x4 &v, float (&s)[Piece<T>::kValues]) {
  if constexpr (sizeof(T) == 4) {
    unpack<T>(v, s);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[2 * i] = slope_value(v[i] & 0xffffu);
      s[2 * i + 1] = slope_value(v[i] >> 16);
    }
  }
}

// ----------------------------------------------------------- three planes ---

// Four float32 values as kPlanes bfloat16 numbers each, the largest first.
template <int kPlanes>
__device__ __forceinline__ void split_chunk(const u32x4 &v, u32x2 (&o)[kPlanes]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float a = __uint_as_float(v[2 * half]), b = __uint_as_float(v[2 * half + 1]);
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) {
      const uint32_t w = pack_pair_bf16(a, b);
      o[i][half] = w;
      a -= __uint_as_float(w << 16);  // exact
      b -= __uint_as_float(w & 0xffff0000u);
    }
  }
}

// ------------------------------------------------------------ LDS layouts ---

// chunk `c` of row `row` of an along tile with rows of kRow bytes
template <int kRow>
__device__ __forceinline__ uint32_t along_offset(int row, int c) {
  const int key = kRow == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
  return row * kRow + ((c ^ key) << 4);
}

// chunk `c` of row `k` of an across tile of R 16-bit values a row
template <int R>
__device__ __forceinline__ uint32_t across_offset(int k, int c) {
  // rows of 256 bytes (R = 128): pieces 2 k apart; of 128 bytes: two rows fill the
  // banks, every second pair is moved; of 64 bytes: the four rows fill them
  static_assert(R == 32 || R == 64 || R == 128, "a row's pieces are 2, 4 or 8");
  const int key = R == 128 ? (k & 3) << 1 : R == 64 ? k & 2 : 0;
  return k * (R * 2) + ((((c >> 1) ^ key) << 1 | (c & 1)) << 4);
}

// A lane's part of 32 rows by 16 of k, 16-bit values: lane l holds row l % 32 and,
// with h = l / 32, the eight k of the step's chunk 2 s + h.
template <bool kAlong, int R, int kRow>
__device__ __forceinline__ u32x4 read_fragment(const char *tile, int row0, int s, int lane) {
  if constexpr (kAlong) {
    return *reinterpret_cast<const u32x4 *>(
        tile + along_offset<kRow>(row0 + (lane & 31), 2 * s + (lane >> 5)));
  } else {
    // a group of 16 lanes hands in four k rows of 16 values (lane i: row i / 4,
    // values 4 (i % 4) on) and gets back, lane i, the four k of value i
#if defined(__HIP_DEVICE_COMPILE__)
    const int group = lane >> 4, i = lane & 15;
    const int k = (2 * s + (group >> 1)) * 8 + (i >> 2);
    const int c = (row0 + (group & 1) * 16) / 8 + ((i & 3) >> 1);
    typedef __attribute__((address_space(3))) i16x4 *lds_ptr;
    const uint32_t o0 = across_offset<R>(k, c) + (i & 1) * 8;
    const uint32_t o1 = across_offset<R>(k + 4, c) + (i & 1) * 8;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_ptr)const_cast<char *>(tile + o0));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_ptr)const_cast<char *>(tile + o1));
    const i16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(u32x4, v);
#else
    return u32x4{};
#endif
  }
}

// The same of float32 values: 32 rows by 8 of k, four k a lane.
template <bool kAlong, int R>
__device__ __forceinline__ u32x4 read_fragment_f32(const char *tile, int row0, int s, int lane) {
  if constexpr (kAlong) {
    return *reinterpret_cast<const u32x4 *>(
        tile + along_offset<128>(row0 + (lane & 31), 2 * s + (lane >> 5)));
  } else {
    u32x4 o;
    const int k = (2 * s + (lane >> 5)) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = *reinterpret_cast<const uint32_t *>(tile + ((k + i) * R + row0 + (lane & 31)) * 4);
    }
    return o;
  }
}

// acc[i][j] += sum over the fragments' k of a[i] b[j], i and j in 0..31. Lane l
// holds column j = l % 32 of acc, register r row 8 (r / 4) + 4 (l / 32) + r % 4.
template <typename T>
__device__ __forceinline__ f32x16 multiply(const u32x4 &a, const u32x4 &b, f32x16 acc) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]),
                                                 acc, 0, 0, 0);
    }
    return acc;
  } else if constexpr (std::is_same_v<T, bf16_t>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
#else
  return acc;
#endif
}

// v plus the value of the lane at XOR kDistance, given that the lanes of each
// aligned group of kDistance hold the same: moves within the vector unit, where a
// shuffle would go through LDS and wait.
template <int kDistance>
__device__ __forceinline__ float add_across(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int i = __float_as_int(v);
  if constexpr (kDistance <= 8) {
    // lanes 1 0 3 2, 2 3 0 1, mirrored halves of a row of 16, mirrored row
    constexpr int kMove = kDistance == 1 ? 0xB1 : kDistance == 2 ? 0x4E
                          : kDistance == 4 ? 0x141 : 0x140;
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(i, kMove, 0xf, 0xf, true));
  } else if constexpr (kDistance == 16) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(i, i, false, false));
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(i, i, false, false));
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#else
  return v;
#endif
}

// LDS that only one wavefront touches: its accesses run in order, the compiler
// must not reorder them.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace dense
