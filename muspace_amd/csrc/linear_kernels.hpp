// Kernels of the dense layer (include/muspace_layer.h):
//
//   y  = act(x W^T + b) + r          linear_product<Job::kForward>, linear_few or
//                                    linear_vector
//   dz = g * act'(x W^T + b)         on the fly from a bit mask (relu), or
//                                    linear_gelu_grad (gelu, from the kept derivative)
//   dx = dz W                        linear_product<Job::kInput> or linear_few
//   dW = dz^T x, db = sum of dz      linear_product<Job::kWeight> + linear_weight_sum
//   x in 8 bits                      written by the forward as it reads x (Kind::kKept), or
//                                    linear_checkpoint; read back by kWeight's loader
//
// The gated layer, W = [Wg; Wu], a = x Wg^T + bg, u = x Wu^T + bu:
//
//   y  = act(a) u                    the same three kernels, Job::kGated
//   da = g u act'(a), du = g act(a)  Job::kGatedGrad: a and u multiplied again
//   dx = [da du] W, dW = [da du]^T x as above, from [da du] in memory
//   db = sums of da and du           as they are made, a row of sums a wavefront, and
//                                    gated_bias_sum
//
// A tile's rows of W are half Wg's and half Wu's, of the same results, 16 or 32 of each in
// turn, so that a wavefront holds a and u of a result and neither is ever written.
//
// linear_product: a workgroup of four wavefronts makes a BM x BN tile of the
// result, each wavefront a quarter. Both operands go through LDS in steps of 128
// bytes of k; the chunks of step i + 1 are in registers on their way while step i
// is multiplied. One LDS buffer, not two: a second workgroup more on a CU hides
// more of the loads than the second buffer did (369900 x 256 -> 256 bf16 114 ->
// 94 us, 44446 x 256 -> 1024 float32 217 -> 208). The matrix cores multiply 16-bit
// values (32x32x16), float32 ones as three bfloat16 planes (linear_device.hpp).
// The wavefront multiplies with the result's columns as the matrix instruction's
// rows, so that a lane holds runs of four columns of a row and the tile goes
// through LDS in 16-byte pieces into whole 128-byte row segments, where bias,
// activation, residual and mask are applied once per value.
//
// All sums are in float32 and in a fixed order: results do not change from run to
// run. Results are rounded once, to the tensors' type.
#pragma once

#include <type_traits>

#include "linear_device.hpp"

namespace dense {

enum class Job { kForward, kInput, kWeight, kGated, kGatedGrad };
// (silu and sigmoid: the gated layer's alone)
enum Activation : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3, kSigmoid = 4 };

constexpr bool gated(Job job) { return job == Job::kGated || job == Job::kGatedGrad; }

struct Product {
  const void *p;         // rows of the result: x, dz or dz^T
  const void *p_rest;    // what rounding left of p (gelu's dz in 16 bits)
  const void *q;         // columns: W, W^T or x
  int64_t ldp, ldq;      // values per row in memory
  int m, n, k;           // result rows, columns; summed index
  const uint8_t *mask;   // relu's bits for p (0: none), [blocks of 64 columns][rows][8]
  int64_t mask_ld;       // bytes of a block of columns: 8 a row
  const uint8_t *scales;  // kWeight with codes: q are codes, a scale byte per 32
  int64_t scale_ld;
  int tiles_n, tiles;    // tiles along n; all tiles of the result
  int splits, k_split;   // kWeight: parts of k, steps' values in each
  // forward
  const void *bias, *residual;
  void *out, *slope_out;  // slope_out: kept derivative (gelu under training)
  uint8_t *mask_out;     // kept sign bits (relu under training), as mask
  int act;
  uint8_t *codes, *code_scales;  // Kind::kKept: the checkpoint of x
  // kGatedGrad: g [m, n]; out is [m, ldz], da, du and zeros up to whole chunks; sums of da
  // and du over rows, before they are rounded, [parts of the rows][2 n] (0: none)
  const void *grad;
  int64_t ldz;
  float *row_sums;
  // kWeight
  float *partial, *bias_partial;  // [splits][m][pad8(n)], [splits][m]
  void *bias_out;                 // splits == 1: db (0: none)
};

// Workgroups go to the eight XCDs in turn. Give each XCD a contiguous run of the
// tile order, so that the tiles of one row strip (or one part of k) share an L2.
__device__ __forceinline__ int xcd_order(int id, int count) {
  const int xcd = id & 7, per = count >> 3, rest = count & 7;
  return xcd * per + (xcd < rest ? xcd : rest) + (id >> 3);
}

// --------------------------------------------------------- operand loader ---

// One operand's R rows (of the result) by a step of k: kCount chunks for each of kTeam
// threads, fetched into registers, then put into LDS. Loads are unconditional, so that all of
// a step's are in flight together. Rows off every alignment (!kTight): a chunk that
// passes the end of its memory row is read as the row's last 16 bytes and its values
// are moved to the front when it is used; rows past the operand read its last one,
// which only marks results that are not stored (past k: zeros). Memory rows shorter
// than a chunk are read value by value.
// What an operand is besides its values in memory: relu's bits go with it (masked), or a
// second tensor holds what rounding to 16 bits left of each value (pair: gelu's dz), or
// its 8-bit checkpoint is written as it is read (kept: the forward's x), or it is the gated
// layer's weight, half of its R rows from either half (`rows` is the rows of one).
enum class Kind { kPlain, kMasked, kPair, kKept, kGated };

template <typename T, bool kAlong, int R, bool kTight, Kind kKind, bool kCodes,
          int kTeam = kThreads>
struct Loader {
  static constexpr bool kMask = kKind == Kind::kMasked;
  static constexpr int kLoads = kKind == Kind::kPair ? 2 : 1;
  static_assert(kKind != Kind::kPair || (sizeof(T) == 2 && kTight), "the pair's rows are whole");
  static constexpr int kV = Piece<T>::kValues;
  static constexpr int kStep = Piece<T>::kStep;
  static constexpr int kCount = R * 8 / kTeam;
  static constexpr int kDown = kTeam / 8;          // rows between a thread's chunks (along)
  static constexpr int kAcross = R / kV;           // chunks per k row (across)
  static constexpr int kStride = kTeam / kAcross;  // k rows between a thread's chunks
  static constexpr bool kGated = kKind == Kind::kGated;
  static_assert(!kGated || kAlong, "the gated weight is read along k");

  // of chunk i (along): its row, counted from row0, of the operand or of its half; the
  // tile's row that it is put into
  __device__ __forceinline__ int line(int i) const { return r + kDown * (kGated ? i >> 1 : i); }
  __device__ __forceinline__ int slot(int i) const {
    if constexpr (!kGated) return line(i);
    constexpr int kRun = R == 128 ? 32 : 16;  // half a wavefront's columns
    return line(i) / kRun * 2 * kRun + (i & 1) * kRun + line(i) % kRun;
  }
  // rows of memory before chunk i's half
  __device__ __forceinline__ int64_t half(int i) const { return kGated && (i & 1) ? rows : 0; }

  const T *ptr, *rest;    // rest: the pair's second tensor
  const uint8_t *bytes;   // mask or scales
  int64_t ld, bytes_ld;
  int row0, rows, k_end;  // first result row, their number in all, end of k
  int r, c;               // thread's first row (along) or k row (across); its chunk
  int skip;               // !kTight: values of the read chunk that are not its own
  bool moved, past;       // !kTight, uniform: some chunk has skip > 0, k past its end
  int k_at;
  u32x4 v[kLoads][kCount];
  uint32_t side[kCount];  // mask byte or scale byte

  __device__ __forceinline__ void init(const void *src, const void *rest_, int64_t ld_,
                                       const uint8_t *b, int64_t b_ld, int row0_, int rows_,
                                       int k_end_) {
    ptr = static_cast<const T *>(src);
    rest = static_cast<const T *>(rest_);
    bytes = b;
    ld = ld_;
    bytes_ld = b_ld;
    row0 = row0_;
    rows = rows_;
    k_end = k_end_;
    const int t = threadIdx.x % kTeam;
    if constexpr (kAlong) {
      r = t >> 3;
      c = t & 7;
    } else {
      r = t / kAcross;
      c = t % kAcross;
    }
  }

  static __device__ __forceinline__ uint32_t window(int64_t bytes_left) {
    return bytes_left > 0x7fffffff ? 0x7fffffffu
                                   : (bytes_left < 0 ? 0u : static_cast<uint32_t>(bytes_left));
  }

  // memory rows from `first` on, columns from `col` on, of `count` rows in all
  template <typename U>
  static __device__ __forceinline__ Source view(const U *p, int64_t ld_, int64_t first, int col,
                                                int64_t count) {
    Source s;
    s.base = reinterpret_cast<const char *>(p + first * ld_ + col);
    s.bytes = window(((count - first) * ld_ - col) * static_cast<int64_t>(sizeof(U)));
    return s;
  }

  __device__ __forceinline__ void fetch(int k0) {
    if constexpr (kAlong) {
      const bool inside = k0 + c * kV < k_end;
      if constexpr (kTight) {
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          const Source s = view(e == 0 ? ptr : rest, ld, row0, k0, rows);
          const Source up = kGated ? view(ptr + rows * ld, ld, row0, k0, rows) : s;
#pragma unroll
          for (int i = 0; i < kCount; ++i) {
            const uint32_t off = static_cast<uint32_t>(line(i) * ld + c * kV) *
                                 static_cast<uint32_t>(sizeof(T));
            v[e][i] = tight_load(kGated && (i & 1) ? up : s, inside ? off : kPast);
          }
        }
      } else if (k_end >= kV) {
        const int col = min(k0 + c * kV, k_end - kV);
        skip = k0 + c * kV - col;
        moved = k0 + kStep > k_end;
        past = false;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          const int64_t row = min(row0 + line(i), rows - 1) + half(i);
          v[0][i] = reinterpret_cast<const Loose16 *>(ptr + row * ld + col)->v;
        }
      } else {
        moved = past = false;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          const int64_t row = row0 + line(i);
          v[0][i] = loose_load<T>(ptr + (row + half(i)) * ld + k0 + c * kV,
                                  row < rows ? k_end - (k0 + c * kV) : 0);
        }
      }
      if constexpr (kMask) {
        const int col = min(k0 + c * kV, k_end - 1);
        const uint8_t *b = bytes + (col >> 6) * bytes_ld + ((col >> 3) & 7);
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          side[i] = b[static_cast<int64_t>(min(row0 + r + kDown * i, rows - 1)) * 8];
        }
      }
    } else {
      const bool inside = row0 + c * kV < rows;
      if constexpr (kCodes) {
        const uint8_t *codes = reinterpret_cast<const uint8_t *>(ptr);
        const Source s = view(codes, ld, k0, row0, k_end);
        const Source f = view(bytes, bytes_ld, k0, row0 / 32, k_end);
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          const uint32_t kr = r + i * kStride;
          const uint32_t off = kr * static_cast<uint32_t>(ld) + c * kV;
          if constexpr (kV == 8) {
            const u32x2 w = tight_load8(s, inside ? off : kPast);
            v[0][i][0] = w[0];
            v[0][i][1] = w[1];
          } else {
            v[0][i][0] = tight_load4(s, inside ? off : kPast);
          }
          side[i] = tight_load_byte(
              f, inside ? kr * static_cast<uint32_t>(bytes_ld) + (c * kV) / 32 : kPast);
        }
      } else if constexpr (kTight) {
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          const Source s = view(e == 0 ? ptr : rest, ld, k0, row0, k_end);
#pragma unroll
          for (int i = 0; i < kCount; ++i) {
            const uint32_t off = static_cast<uint32_t>((r + i * kStride) * ld + c * kV) *
                                 static_cast<uint32_t>(sizeof(T));
            v[e][i] = tight_load(s, inside ? off : kPast);
          }
        }
      } else if (rows >= kV) {
        const int col = min(row0 + c * kV, rows - kV);
        skip = row0 + c * kV - col;
        moved = row0 + R > rows;
        past = k0 + kStep > k_end;
        k_at = k0;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          const int64_t kr = min(k0 + r + i * kStride, k_end - 1);
          v[0][i] = reinterpret_cast<const Loose16 *>(ptr + kr * ld + col)->v;
        }
      } else {
        moved = past = false;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          const int64_t kr = k0 + r + i * kStride;
          v[0][i] = loose_load<T>(ptr + kr * ld + row0 + c * kV,
                                  kr < k_end ? rows - (row0 + c * kV) : 0);
        }
      }
      if constexpr (kMask) {
        const int col = min(row0 + c * kV, rows - 1);
        const uint8_t *b = bytes + (col >> 6) * bytes_ld + ((col >> 3) & 7);
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
          side[i] = b[static_cast<int64_t>(min(k0 + r + i * kStride, k_end - 1)) * 8];
        }
      }
    }
  }

  // the fetched chunk as the product reads it (`e`: of the pair's second tensor)
  __device__ __forceinline__ u32x4 chunk(int i, int e = 0) const {
    if constexpr (kCodes) {
      uint32_t w[kV / 4];
      w[0] = v[0][i][0];
      if constexpr (kV == 8) w[1] = v[0][i][1];
      return decode<T>(w, scale_value(side[i]));
    } else {
      u32x4 o = v[e][i];
      if constexpr (!kTight) {
        if (moved) o = drop_front<T>(o, skip);
        if (!kAlong && past && k_at + r + i * kStride >= k_end) o = u32x4{0, 0, 0, 0};
      }
      if constexpr (kMask) o = keep_bits<T>(o, side[i] >> ((c * kV) & 7));
      return o;
    }
  }

  // LDS bytes of one plane's tile
  static constexpr int kRow = sizeof(T) == 4 ? 64 : 128;
  static constexpr int kPlaneBytes = R * kRow;
  // 8-bit codes need one plane: 7 bits
  static constexpr int kPlanes = sizeof(T) == 4 ? (kCodes ? 1 : 3) : kLoads;

  __device__ __forceinline__ void put(char *tile, int i, const u32x4 &value) const {
    if constexpr (sizeof(T) == 4) {
      u32x2 part[kPlanes];
      split_chunk<kPlanes>(value, part);
      const uint32_t at = (kAlong ? along_offset<64>(slot(i), c >> 1)
                                  : across_offset<R>(r + i * kStride, c >> 1)) +
                          (c & 1) * 8;
#pragma unroll
      for (int e = 0; e < kPlanes; ++e) {
        *reinterpret_cast<u32x2 *>(tile + e * kPlaneBytes + at) = part[e];
      }
    } else {
      const uint32_t at = kAlong ? along_offset<128>(slot(i), c)
                                 : across_offset<R>(r + i * kStride, c);
      *reinterpret_cast<u32x4 *>(tile + at) = value;
    }
  }

  // the checkpoint of a fetched chunk (along): every lane of a row's takes part
  __device__ __forceinline__ void keep(uint8_t *codes, uint8_t *scales, int k0, int i,
                                       const u32x4 &value) const {
    float f[kV];
    unpack<T>(value, f);
    uint32_t w[kV / 4];
    const uint32_t scale = encode<T>(f, w);
    const int row = row0 + r + kDown * i, col = k0 + c * kV, padded = (k_end + 31) & ~31;
    if (row < rows && col < padded) keep_codes<T>(codes, scales, row, col, padded, w, scale);
  }

  // float32 as it is, for the tiles that hold more than bfloat16's range
  __device__ __forceinline__ void put_f32(char *tile, int i, const u32x4 &value) const {
    const uint32_t at = kAlong ? along_offset<128>(slot(i), c)
                               : static_cast<uint32_t>(((r + i * kStride) * R + c * 4) * 4);
    *reinterpret_cast<u32x4 *>(tile + at) = value;
  }
};

// ---------------------------------------------------------------- epilogue ---

// Phi(z), the normal distribution function, and exp(-z^2 / 2). With t = 1 / (1 +
// 0.35 |z|), the upper tail is exp(-z^2 / 2) t P(t); P, of degree 8, is a least
// squares fit, reweighted until its relative error was level, 3.2e-8 over |z| <= 14
// (past that the tail is under float32's normal numbers). The tail is computed
// itself, without a difference from one, so that negative z keep most of their relative
// accuracy: the exponent's roundings grow with z^2 and leave the tail's relative error at
// 4e-7 near zero, 2e-6 for z in [-6, -4] and 8e-6 in [-13, -9]. The library's error function
// costs two to three times the instructions: gelu was a third of the time of the products
// it ends.
__device__ __forceinline__ float normal_cdf(float z, float &density) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(z), 1.0f));
  float p = -0.029145927f;
  p = fmaf(p, t, 0.14397168f);
  p = fmaf(p, t, -0.25571422f);
  p = fmaf(p, t, 0.15917413f);
  p = fmaf(p, t, -0.023109811f);
  p = fmaf(p, t, 0.10550799f);
  p = fmaf(p, t, 0.11983287f);
  p = fmaf(p, t, 0.13986187f);
  p = fmaf(p, t, 0.13962140f);
  density = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  const float tail = t * p * density;
  return z < 0.0f ? tail : 1.0f - tail;
}

// gelu and its derivative. z where the other factor is zero must be finite: infinite
// pre-activations have the limits' value and slope. NaN stays, in the cdf.
__device__ __forceinline__ float gelu(float z, float &slope) {
  float density;
  const float cdf = normal_cdf(z, density);
  const float low = fmaxf(z, -64.0f);
  slope = fmaf(fminf(low, 64.0f) * 0.39894228f, density, cdf);
  return low * cdf;
}

// `left` values of bias from `p` on
template <typename T>
__device__ __forceinline__ void load_bias(const T *p, int left, float (&b)[Piece<T>::kValues]) {
  const u32x4 v = loose_load<T>(p, left);
  unpack<T>(v, b);
}

// A chunk of the forward's result: z holds x W^T + b. `half`: the lane holds the
// upper four columns of a mask byte (float32).
template <typename T>
__device__ __forceinline__ void finish_forward(const Product &a, int64_t row, int col, int left,
                                               float (&z)[Piece<T>::kValues]) {
  constexpr int kV = Piece<T>::kValues;
  const int64_t at = row * a.n + col;
  if (a.act == kRelu) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const bool keep = !(z[i] <= 0.0f);  // NaN stays NaN
      bits |= (keep ? 1u : 0u) << i;
      z[i] = keep ? z[i] : 0.0f;
    }
    if (a.mask_out != nullptr) {
      uint8_t *mask = a.mask_out + (col >> 6) * a.mask_ld + row * 8 + ((col >> 3) & 7);
      if constexpr (kV == 4) {
        // lanes l and l ^ 1 hold the two halves of a byte
        const uint32_t other = from_lane<1>(bits);
        if ((col & 4) == 0 && left > 0) {
          *mask = static_cast<uint8_t>(bits | other << 4);
        }
      } else if (left > 0) {
        *mask = static_cast<uint8_t>(bits);
      }
    }
  } else if (a.act == kGelu) {
    float slope[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) z[i] = gelu(z[i], slope[i]);
    if (a.slope_out != nullptr && left > 0) {
      loose_store(static_cast<T *>(a.slope_out) + at, pack_slopes<T>(slope), left);
    }
  }
  if (left <= 0) return;
  if (a.residual != nullptr) {
    float r[kV];
    unpack<T>(loose_load<T>(static_cast<const T *>(a.residual) + at, left), r);
#pragma unroll
    for (int i = 0; i < kV; ++i) z[i] += r[i];
  }
  loose_store(static_cast<T *>(a.out) + at, pack<T>(z), left);
}

// The logistic function and one less it, from exp(-|z|), which has no overflow: both
// keep their relative accuracy, 6e-7 (the exponent's product is carried to twice
// float32's bits, rcp rounds to one step), down to 2^-126, and steps of 2^-149 below, which
// silu multiplies into normal numbers: exp2 has no such results, its square has.
__device__ __forceinline__ float logistic(float z, float &other) {
  // (past 128 exp is zero; an infinity would be subtracted from itself, NaN stays)
  const float m = fabsf(z) > 128.0f ? -128.0f : -fabsf(z), p = m * 1.44269504f;
  const float rest = fmaf(m, 1.44269504f, -p) + m * 1.92596300e-8f;
  const float root = __builtin_amdgcn_exp2f(0.5f * p), power = root * root;
  const float e = fmaf(power * rest, 0.69314718f, power);
  const float large = __builtin_amdgcn_rcpf(1.0f + e), small = e * large;
  // (!(z < 0): NaN stays in both)
  other = z < 0.0f ? large : small;
  return z < 0.0f ? small : large;
}

// The gate's activation and its derivative; infinities have the limits' values. kShort:
// for results of 16 bits, the logistic function in seven instructions where the other takes
// seventeen. The exponent's product is rounded once, which with log2(e)'s own rounding is relative
// 2^-24 (1.3 |z| + 30) of either factor at the most, a hundredth of float16's own rounding.
// Either is a product with the reciprocal r of 1 + exp(-z), and for silu of 2^-32 (1 + exp(-z)):
// rcp has no results under 2^-126, but silu is a normal number down to z = -92. (40000 x 256 -> 2 x
// 512 bf16 36.8 us; 36.6 with 1 - s for the other factor, which loses a saturated sigmoid's
// derivative; 3 more with the float32 form.)
template <bool kShort>
__device__ __forceinline__ float gate_of(int act, float z, float &slope) {
  if (act == kSilu || act == kSigmoid) {
    float s, other;
    if constexpr (kShort) {
      const float shift = act == kSilu ? 32.0f : 0.0f, one = act == kSilu ? 0x1p-32f : 1.0f;
      const float e = __builtin_amdgcn_exp2f(fmaf(z, -1.44269504f, -shift));
      const float r = __builtin_amdgcn_rcpf(one + e);
      s = one * r;
      other = fminf(e, 0x1.fffffep127f) * r;  // (no infinity times zero)
    } else {
      s = logistic(z, other);
    }
    if (act == kSigmoid) {
      slope = s * other;
      return s;
    }
    const float low = fmaxf(z, -128.0f);  // past it the other factor is zero
    slope = s * fmaf(fminf(low, 128.0f), other, 1.0f);
    return low * s;
  }
  if (act == kGelu) return gelu(z, slope);
  if (act == kRelu) {
    const bool keep = !(z <= 0.0f);  // NaN stays NaN
    slope = keep ? 1.0f : 0.0f;
    return keep ? z : 0.0f;
  }
  slope = 1.0f;
  return z;
}

// The biases of a chunk's a, then of its u.
template <typename T>
__device__ __forceinline__ void load_biases(const Product &a, int col, int left,
                                            float (&bias)[2][Piece<T>::kValues]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (a.bias != nullptr) {
      load_bias<T>(static_cast<const T *>(a.bias) + (h == 0 ? col : a.n + col), left, bias[h]);
    } else {
#pragma unroll
      for (int i = 0; i < Piece<T>::kValues; ++i) bias[h][i] = 0.0f;
    }
  }
}
template <typename T>
__device__ __forceinline__ u32x4 load_grad(const Product &a, int64_t row, int col, int left) {
  return loose_load<T>(static_cast<const T *>(a.grad) + row * a.n + col, left);
}

// A chunk of the gated layer's result, or of da and du: z and u hold the products
// without their biases, `grad` the chunk of g (kGrad). da and du are rounded to the
// tensors' type, once, as gradients that leave an operator are: their errors, independent,
// are as large as the gradients' own rounding, 1.41 times it together. In two numbers each,
// as gelu's dz below, they would cost twice the products and twice the bytes: 40000 x 256
// -> 2 x 512 bf16 moves 246 MB of da and du as it is.
// `sums` gathers a lane's da and du as they are, for db: of few columns, sums of the rounded
// ones erred by up to 1.6 times their own rounding, and these cost 5 of 155 us there.
template <typename T, bool kGrad>
__device__ __forceinline__ void finish_gated(const Product &a, int64_t row, int col, int left,
                                             float (&z)[Piece<T>::kValues],
                                             float (&u)[Piece<T>::kValues],
                                             const float (&bias)[2][Piece<T>::kValues],
                                             const u32x4 &grad,
                                             float (&sums)[2][Piece<T>::kValues]) {
  constexpr int kV = Piece<T>::kValues;
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < kV; ++i) {
    z[i] += bias[0][i];
    u[i] += bias[1][i];
  }
  float slope[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) z[i] = gate_of<sizeof(T) == 2>(a.act, z[i], slope[i]);
  if constexpr (!kGrad) {
#pragma unroll
    for (int i = 0; i < kV; ++i) z[i] *= u[i];
    loose_store(static_cast<T *>(a.out) + row * a.n + col, pack<T>(z), left);
  } else {
    float g[kV];
    unpack<T>(grad, g);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      slope[i] *= g[i] * u[i];
      z[i] *= g[i];
      sums[0][i] += slope[i];
      sums[1][i] += z[i];
    }
    T *to = static_cast<T *>(a.out) + row * a.ldz + col;
    loose_store(to, pack<T>(slope), left);
    loose_store(to + a.n, pack<T>(z), left);
    if (left <= kV) {  // the row's last chunk: zeros up to whole chunks
      for (int64_t i = 2 * static_cast<int64_t>(a.n) - col; i < a.ldz - col; ++i) {
        to[i] = from_float<T>(0.0f);
      }
    }
  }
}

// The sums of a wavefront's rows: its lanes l, l + kLanes, l + 2 kLanes ... hold rows of the
// same columns, and the first kLanes leave their sum as row `part` of row_sums.
template <typename T, int kLanes>
__device__ __forceinline__ void leave_sums(const Product &a, int part, int lane, int col, int left,
                                           float (&sums)[2][Piece<T>::kValues]) {
  constexpr int kV = Piece<T>::kValues;
  if (a.row_sums == nullptr) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      float v = sums[h][e];
#if defined(__HIP_DEVICE_COMPILE__)
      // rows of 16 lanes turned by 2, 4 and 8
      if constexpr (kLanes <= 2) {
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, true));
      }
      if constexpr (kLanes <= 4) {
        v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true));
      }
      v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true));
#endif
      static_assert(kLanes == 2 || kLanes == 4 || kLanes == 8, "a row's lanes");
      v = add_across<32>(add_across<16>(v));
      if (lane < kLanes && e < left) {
        a.row_sums[(static_cast<int64_t>(part) * 2 + h) * a.n + col + e] = v;
      }
    }
  }
}

// ------------------------------------------------------------- tile kernel ---

// Three workgroups a CU where the registers allow it (168 of them): the loads and
// stores of one hide behind the products of the others. 16-bit products need 136 to
// 168 by themselves; float32 ones are held to it where rows are whole chunks (44446 x
// 256 -> 1024, input gradient: 158 us at two, 144 at three; the masked gradient
// spills four registers, the forward that keeps its input eight).
// Four, at 128 registers, spill; the chunks of two steps in registers cost the third
// workgroup (369900 x 256 -> 256 bf16 94 -> 113 us); tiles of 64 x 128 and 128 x 64
// read more per product (114 and 104 us).
template <typename T, Job kJob, int BM, int BN, bool kTight, Kind kKind, bool kCodes>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && kTight) ? 3 : 2) void linear_product(const Product a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kStep = Piece<T>::kStep;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr bool kPAlong = kJob != Job::kWeight;
  constexpr bool kQAlong = kJob == Job::kForward || gated(kJob);
  constexpr int WM = BM / 2, WN = BN / 2;  // a wavefront's quarter
  constexpr int kColumns = gated(kJob) ? BN / 2 : BN;  // of the result
  constexpr int kI = WM / 32, kJ = WN / 32;
  // (the pair is this library's own tensor, its rows padded to whole chunks)
  using P = Loader<T, kPAlong, BM, kTight || kKind == Kind::kPair, kKind, false>;
  using Q = Loader<T, kQAlong, BN, kTight, gated(kJob) ? Kind::kGated : Kind::kPlain, kCodes>;
  constexpr int kStageLd = WN + 4;  // floats; the pad spreads rows over the banks
  constexpr int kTiles = P::kPlanes * P::kPlaneBytes + Q::kPlanes * Q::kPlaneBytes;
  constexpr int kTilesF32 = kF32 ? (BM + BN) * kRowBytes : 0;
  constexpr int kStage = 4 * 32 * kStageLd * 4;
  constexpr int kLds = kStage > kTiles ? (kStage > kTilesF32 ? kStage : kTilesF32)
                                       : (kTiles > kTilesF32 ? kTiles : kTilesF32);
  __shared__ __attribute__((aligned(16))) char lds[kLds];

  int tile = xcd_order(blockIdx.x, gridDim.x);
  int split = 0;
  if constexpr (kJob == Job::kWeight) {
    split = tile / a.tiles;
    tile -= split * a.tiles;
  }
  const int row0 = tile / a.tiles_n * BM, col0 = tile % a.tiles_n * kColumns;
  const int k_begin = split * a.k_split;
  const int k_end = kJob == Job::kWeight && a.k - k_begin > a.k_split ? k_begin + a.k_split : a.k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * WM, wc = (wave & 1) * WN;

  P p;
  Q q;
  p.init(a.p, a.p_rest, a.ldp, a.mask, a.mask_ld, row0, a.m, k_end);
  q.init(a.q, nullptr, a.ldq, a.scales, a.scale_ld, col0, a.n, k_end);

  f32x16 acc[kI][kJ];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < kI; ++i) {
#pragma unroll
      for (int j = 0; j < kJ; ++j) acc[i][j] = f32x16{};
    }
  };
  clear();
  // kWeight's first tile column also sums dz over its rows: a thread's chunks all
  // lie in one column of chunks
  float sums[kV] = {};
  const bool sum_p = kJob == Job::kWeight && col0 == 0;

  // The checkpoint's rows are shared out among the first columns of tiles. 40000 x 256 -> 512
  // bf16: a launch of its own and the plain forward 7.7 + 23.7 us, all rows with the first
  // column 32.8, shared 26.5; 1800 x 1024 -> 256 float32: 4.2 + 15.3 us, shared 18.1.
  const int keepers = min(a.tiles_n, static_cast<int>(P::kCount)), keeper = tile % a.tiles_n;

  char *const tile_p = lds, *const tile_q = lds + P::kPlanes * P::kPlaneBytes;
  if (k_begin < k_end) {
    p.fetch(k_begin);
    q.fetch(k_begin);
  }
  for (int k0 = k_begin; k0 < k_end; k0 += kStep) {
#pragma unroll
    for (int i = 0; i < P::kCount; ++i) {
#pragma unroll
      for (int l = 0; l < P::kLoads; ++l) {
        const u32x4 v = p.chunk(i, l);
        if constexpr (kJob == Job::kWeight) {
          if (sum_p) {
            float f[kV];
            unpack<T>(v, f);
#pragma unroll
            for (int e = 0; e < kV; ++e) sums[e] += f[e];
          }
        }
        if constexpr (kKind == Kind::kKept) {
          if (i % keepers == keeper) p.keep(a.codes, a.code_scales, k0, i, v);
        }
        p.put(tile_p + l * P::kPlaneBytes, i, v);
      }
    }
#pragma unroll
    for (int i = 0; i < Q::kCount; ++i) q.put(tile_q, i, q.chunk(i));
    __syncthreads();
    if (k0 + kStep < k_end) {
      p.fetch(k0 + kStep);
      q.fetch(k0 + kStep);
    }
#pragma unroll
    for (int s = 0; s < P::kRow / 32; ++s) {
      u32x4 fp[P::kPlanes][kI], fq[Q::kPlanes][kJ];
#pragma unroll
      for (int e = 0; e < P::kPlanes; ++e) {
#pragma unroll
        for (int i = 0; i < kI; ++i) {
          fp[e][i] = read_fragment<kPAlong, BM, P::kRow>(tile_p + e * P::kPlaneBytes, wr + 32 * i,
                                                         s, lane);
        }
      }
#pragma unroll
      for (int e = 0; e < Q::kPlanes; ++e) {
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          fq[e][j] = read_fragment<kQAlong, BN, P::kRow>(tile_q + e * Q::kPlaneBytes, wc + 32 * j,
                                                         s, lane);
        }
      }
#pragma unroll
      for (int x = 0; x < P::kPlanes; ++x) {
#pragma unroll
        for (int y = 0; y < Q::kPlanes; ++y) {
          if (x + y > 2) continue;
#pragma unroll
          for (int i = 0; i < kI; ++i) {
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              acc[i][j] = multiply<std::conditional_t<kF32, bf16_t, T>>(fq[y][j], fp[x][i],
                                                                       acc[i][j]);
            }
          }
        }
      }
    }
    __syncthreads();
  }

  if constexpr (kF32) {
    // a sum that is not finite: an infinity, NaN or a number past bfloat16's range
    // among its values, or an overflow. Then the tile again, in float32.
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < kI; ++i) {
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
#pragma unroll
        for (int e = 0; e < 16; ++e) zero = fmaf(acc[i][j][e], 0.0f, zero);
      }
    }
    if (__syncthreads_or(!(zero == 0.0f))) {
      clear();
      char *const wide_q = lds + BM * kRowBytes;
      for (int k0 = k_begin; k0 < k_end; k0 += kStep) {
        p.fetch(k0);
        q.fetch(k0);
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) p.put_f32(lds, i, p.chunk(i));
#pragma unroll
        for (int i = 0; i < Q::kCount; ++i) q.put_f32(wide_q, i, q.chunk(i));
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
          for (int i = 0; i < kI; ++i) {
            const u32x4 fp = read_fragment_f32<kPAlong, BM>(lds, wr + 32 * i, s, lane);
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              const u32x4 fq = read_fragment_f32<kQAlong, BN>(wide_q, wc + 32 * j, s, lane);
              acc[i][j] = multiply<float>(fq, fp, acc[i][j]);
            }
          }
        }
        __syncthreads();
      }
    }
  }

  // the bias gradient: threads of one chunk column add their sums, in thread order
  if constexpr (kJob == Job::kWeight) {
    if (sum_p && (a.bias_partial != nullptr || a.bias_out != nullptr)) {
      constexpr int kGroups = kThreads / (BM / kV);
      float *s = reinterpret_cast<float *>(lds);
      const int c = threadIdx.x % (BM / kV), g = threadIdx.x / (BM / kV);
#pragma unroll
      for (int e = 0; e < kV; ++e) s[g * BM + c * kV + e] = sums[e];
      __syncthreads();
      const int row = row0 + threadIdx.x;
      if (threadIdx.x < BM && row < a.m) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) total += s[i * BM + threadIdx.x];
        if (a.bias_partial != nullptr) {
          a.bias_partial[static_cast<int64_t>(split) * a.m + row] = total;
        } else {
          static_cast<T *>(a.bias_out)[row] = from_float<T>(total);
        }
      }
      __syncthreads();
    }
  }

  // the tile, 32 rows of a wavefront at a time, through the wavefront's own LDS
  float *stage = reinterpret_cast<float *>(lds) + wave * 32 * kStageLd;
  constexpr int kOut = gated(kJob) ? WN / 2 : WN;  // a wavefront's columns of the result
  constexpr int kLanes = kOut / kV;       // lanes per row
  constexpr int kRows = kWave / kLanes;   // rows at a time
  const int chunk = lane % kLanes;
  const int col = col0 + (gated(kJob) ? wc / 2 : wc) + chunk * kV, left = a.n - col;
  float bias[kV] = {}, biases[2][kV];
  if constexpr (kJob == Job::kForward) {
    if (a.bias != nullptr) load_bias<T>(static_cast<const T *>(a.bias) + col, left, bias);
  }
  float row_sums[2][kV] = {};
  if constexpr (gated(kJob)) load_biases<T>(a, col, left, biases);
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    u32x4 grads[32 / kRows] = {};
    if constexpr (kJob == Job::kGatedGrad) {
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += kRows) {
        const int64_t row = row0 + wr + 32 * i + r0 + lane / kLanes;
        grads[r0 / kRows] = load_grad<T>(a, row, col, row < a.m ? left : 0);
      }
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
        *reinterpret_cast<f32x4 *>(stage + (lane & 31) * kStageLd + 32 * j + 8 * g +
                                   4 * (lane >> 5)) = v;
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int64_t row = row0 + wr + 32 * i + r;
      const float *src = stage + r * kStageLd + chunk * kV;
      float z[kV];
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(src + e);
#pragma unroll
        for (int x = 0; x < 4; ++x) z[e + x] = v[x];
      }
      const int here = row < a.m ? left : 0;
      if constexpr (gated(kJob)) {
        float u[kV];
#pragma unroll
        for (int e = 0; e < kV; e += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4 *>(src + kOut + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) u[e + x] = v[x];
        }
        finish_gated<T, kJob == Job::kGatedGrad>(a, row, col, here, z, u, biases,
                                                 grads[r0 / kRows], row_sums);
      } else if constexpr (kJob == Job::kForward) {
#pragma unroll
        for (int e = 0; e < kV; ++e) z[e] += bias[e];
        finish_forward<T>(a, row, col, here, z);
      } else {
        if (here > 0) {
          if (kJob == Job::kWeight && a.partial != nullptr) {
            const int64_t ld = (a.n + 7) & ~7;
            float *to = a.partial + (static_cast<int64_t>(split) * a.m + row) * ld + col;
#pragma unroll
            for (int e = 0; e < kV; e += 4) {
              f32x4 v = {z[e], z[e + 1], z[e + 2], z[e + 3]};
              *reinterpret_cast<f32x4 *>(to + e) = v;
            }
          } else {
            loose_store(static_cast<T *>(a.out) + row * a.n + col, pack<T>(z), here);
          }
        }
      }
    }
    wave_lds_sync();
  }
  if constexpr (kJob == Job::kGatedGrad) {
    leave_sums<T, kLanes>(a, row0 / BM * 2 + (wave >> 1), lane, col, left, row_sums);
  }
}

// ------------------------------------------------------------ few results ---

// kForward, kInput and the gated jobs where the tiles would leave most CUs idle: a workgroup
// makes 32 x 32 results (gated: 32 x 16) and its kWaves wavefronts take turns at the steps
// of k, each with its own tiles in LDS, so that none waits for another until the sums are
// joined, in wavefront order. float32 is multiplied as it is: the time is that of the loads.
template <typename T, Job kJob, int kWaves, bool kTight, Kind kKind>
__global__ __launch_bounds__(kWaves *kWave) void linear_few(const Product a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kStep = Piece<T>::kStep;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr bool kQAlong = kJob == Job::kForward || gated(kJob);
  constexpr int kColumns = gated(kJob) ? 16 : 32;
  using P = Loader<T, true, 32, kTight || kKind == Kind::kPair, kKind, false, kWave>;
  using Q = Loader<T, kQAlong, 32, kTight, gated(kJob) ? Kind::kGated : Kind::kPlain, false, kWave>;
  constexpr int kTile = 32 * kRowBytes;
  constexpr int kTiles = (P::kLoads + 1) * kTile;  // of a wavefront
  constexpr int kLd = 36;
  static_assert(32 * kLd * 4 <= kTiles, "a wavefront's sums exceed its tiles");
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kTiles];
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int row0 = tile / a.tiles_n * 32, col0 = tile % a.tiles_n * kColumns;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char *const tile_p = lds + wave * kTiles, *const tile_q = tile_p + P::kLoads * kTile;
  P p;
  Q q;
  p.init(a.p, a.p_rest, a.ldp, a.mask, a.mask_ld, row0, a.m, a.k);
  q.init(a.q, nullptr, a.ldq, nullptr, 0, col0, a.n, a.k);
  const int keepers = min(a.tiles_n, static_cast<int>(P::kCount)), keeper = tile % a.tiles_n;
  f32x16 acc = {};
  int k0 = wave * kStep;
  if (k0 < a.k) {
    p.fetch(k0);
    q.fetch(k0);
  }
  for (; k0 < a.k; k0 += kWaves * kStep) {
#pragma unroll
    for (int i = 0; i < P::kCount; ++i) {
      if constexpr (kKind == Kind::kKept) {
        if (i % keepers == keeper) p.keep(a.codes, a.code_scales, k0, i, p.chunk(i));
      }
      if constexpr (kF32) {
        p.put_f32(tile_p, i, p.chunk(i));
      } else {
#pragma unroll
        for (int l = 0; l < P::kLoads; ++l) p.put(tile_p + l * kTile, i, p.chunk(i, l));
      }
    }
#pragma unroll
    for (int i = 0; i < Q::kCount; ++i) {
      if constexpr (kF32) {
        q.put_f32(tile_q, i, q.chunk(i));
      } else {
        q.put(tile_q, i, q.chunk(i));
      }
    }
    wave_lds_sync();
    if (k0 + kWaves * kStep < a.k) {
      p.fetch(k0 + kWaves * kStep);
      q.fetch(k0 + kWaves * kStep);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if constexpr (kF32) {
        acc = multiply<T>(read_fragment_f32<kQAlong, 32>(tile_q, 0, s, lane),
                          read_fragment_f32<true, 32>(tile_p, 0, s, lane), acc);
      } else {
        const u32x4 fq = read_fragment<kQAlong, 32, 128>(tile_q, 0, s, lane);
#pragma unroll
        for (int l = 0; l < P::kLoads; ++l) {
          acc = multiply<T>(fq, read_fragment<true, 32, 128>(tile_p + l * kTile, 0, s, lane), acc);
        }
      }
    }
    wave_lds_sync();
  }
  float *const sums = reinterpret_cast<float *>(tile_p);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    *reinterpret_cast<f32x4 *>(sums + (lane & 31) * kLd + 8 * g + 4 * (lane >> 5)) = v;
  }
  __syncthreads();
  constexpr int kLanes = kColumns / kV;
  // whole wavefronts take part (the mask's halves are exchanged between lanes)
  for (int i = threadIdx.x; i < 32 * kLanes; i += kWaves * kWave) {
    const int chunk = i % kLanes, r = i / kLanes;
    const int col = col0 + chunk * kV;
    const int64_t row = row0 + r;
    const int left = row < a.m ? a.n - col : 0;
    float z[kV] = {};
#pragma unroll
    for (int u = 0; u < kWaves; ++u) {
      const float *src = reinterpret_cast<const float *>(lds + u * kTiles) + r * kLd + chunk * kV;
#pragma unroll
      for (int e = 0; e < kV; ++e) z[e] += src[e];
    }
    if constexpr (gated(kJob)) {
      float up[kV] = {};
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const float *src =
            reinterpret_cast<const float *>(lds + u * kTiles) + r * kLd + kColumns + chunk * kV;
#pragma unroll
        for (int e = 0; e < kV; ++e) up[e] += src[e];
      }
      float biases[2][kV];
      load_biases<T>(a, col, left, biases);
      const u32x4 grad = kJob == Job::kGatedGrad ? load_grad<T>(a, row, col, left) : u32x4{};
      float row_sums[2][kV] = {};
      finish_gated<T, kJob == Job::kGatedGrad>(a, row, col, left, z, up, biases, grad, row_sums);
      if constexpr (kJob == Job::kGatedGrad) {
        // (a wavefront's lanes are 16 rows of float32, or 32 of 16 bits)
        constexpr int kParts = 32 * kLanes / kWave;
        leave_sums<T, kLanes>(a, row0 / 32 * kParts + wave, lane, col, a.n - col, row_sums);
      }
    } else if constexpr (kJob == Job::kForward) {
      if (a.bias != nullptr) {
        float b[kV];
        load_bias<T>(static_cast<const T *>(a.bias) + col, a.n - col, b);
#pragma unroll
        for (int e = 0; e < kV; ++e) z[e] += b[e];
      }
      finish_forward<T>(a, row, col, left, z);
    } else {
      loose_store(static_cast<T *>(a.out) + row * a.n + col, pack<T>(z), left);
    }
  }
}

// --------------------------------------------------------- a row or a few ---

// The forward of up to kRows rows: reading W is all of it, and it takes many loads in
// flight on many CUs, not matrix cores that would multiply 32 rows. A wavefront takes
// kCols rows of W whole, its lanes 16 bytes of each at a time, multiplies them with the
// rows of x (in the caches after the first wavefront) on the vector unit and sums over its
// lanes. A workgroup makes eight columns, a byte of the mask. Gated: kCols rows of either
// half of W.
template <typename T, Job kJob, int kRows, int kCols>
__global__ __launch_bounds__(8 / kCols *kWave) void linear_vector(const Product a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kAhead = 4;  // of a lane's chunks, in flight together
  constexpr int kSpan = kWave * kV;
  constexpr int kLanes = 8 / kV;  // of a result row, at the end
  constexpr int kHalves = gated(kJob) ? 2 : 1;
  constexpr int kW = kCols * kHalves;  // rows of W
  static_assert(kRows * kLanes <= kWave && kRows * kW <= kWave, "one wavefront ends it");
  __shared__ __attribute__((aligned(16))) float lds[kHalves][kRows * 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.x * 8, col0 = first + wave * kCols;
  const T *w[kW], *x[kRows];
#pragma unroll
  for (int c = 0; c < kW; ++c) {
    const int64_t row = min(col0 + c % kCols, a.n - 1) + (c < kCols ? 0 : a.n);
    w[c] = static_cast<const T *>(a.q) + row * a.ldq;
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m) x[m] = static_cast<const T *>(a.p) + min(m, a.m - 1) * a.ldp;
  const int col = first + lane % kLanes * kV, row = lane / kLanes;
  float bias[kV] = {};
  if (!gated(kJob) && wave == 0 && a.bias != nullptr) {
    load_bias<T>(static_cast<const T *>(a.bias) + col, a.n - col, bias);
  }
  float sum[kRows][kW] = {};
  // the products of one chunk each, but for the first `drop` values
  auto add = [&](const u32x4(&wv)[kW], const u32x4(&xv)[kRows], int drop) {
    float f[kW][kV];
#pragma unroll
    for (int c = 0; c < kW; ++c) {
      unpack<T>(wv[c], f[c]);
#pragma unroll
      for (int e = 0; e < kV; ++e) f[c][e] = e < drop ? 0.0f : f[c][e];
    }
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      float g[kV];
      unpack<T>(xv[m], g);
#pragma unroll
      for (int e = 0; e < kV; ++e) g[e] = e < drop ? 0.0f : g[e];
#pragma unroll
      for (int c = 0; c < kW; ++c) {
#pragma unroll
        for (int e = 0; e < kV; ++e) sum[m][c] = fmaf(g[e], f[c][e], sum[m][c]);
      }
    }
  };
  int k0 = lane * kV;
  // `kCount` whole spans
  auto spans = [&](auto count) {
    constexpr int kCount = decltype(count)::value;
    u32x4 wv[kCount][kW], xv[kCount][kRows];
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int k = k0 + i * kSpan;
#pragma unroll
      for (int c = 0; c < kW; ++c) wv[i][c] = reinterpret_cast<const Loose16 *>(w[c] + k)->v;
#pragma unroll
      for (int m = 0; m < kRows; ++m) xv[i][m] = reinterpret_cast<const Loose16 *>(x[m] + k)->v;
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) add(wv[i], xv[i], 0);
    k0 += kCount * kSpan;
  };
  while (k0 - lane * kV + kAhead * kSpan <= a.k) spans(std::integral_constant<int, kAhead>{});
  // (a row of two spans would take them one after the other: gated, 1024 -> 2 x 4096 bf16 6.2 us,
  // so 5.9)
  if (k0 - lane * kV + 2 * kSpan <= a.k) spans(std::integral_constant<int, 2>{});
  for (; k0 < a.k; k0 += kSpan) {
    u32x4 wv[kW], xv[kRows];
    if (a.k >= kV) {
      // a chunk that passes the end: the rows' last 16 bytes, less what came before
      const int k = min(k0, a.k - kV);
#pragma unroll
      for (int c = 0; c < kW; ++c) wv[c] = reinterpret_cast<const Loose16 *>(w[c] + k)->v;
#pragma unroll
      for (int m = 0; m < kRows; ++m) xv[m] = reinterpret_cast<const Loose16 *>(x[m] + k)->v;
      add(wv, xv, k0 - k);
    } else {
#pragma unroll
      for (int c = 0; c < kW; ++c) wv[c] = loose_load<T>(w[c], a.k);
#pragma unroll
      for (int m = 0; m < kRows; ++m) xv[m] = loose_load<T>(x[m], a.k);
      add(wv, xv, 0);
    }
  }
  float mine = 0.0f;
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
#pragma unroll
    for (int c = 0; c < kW; ++c) {
      float v = sum[m][c];
      v = add_across<8>(add_across<4>(add_across<2>(add_across<1>(v))));
      v = add_across<32>(add_across<16>(v));
      if (lane == m * kW + c && col0 + c % kCols < a.n) mine = v;
    }
  }
  if (lane < kRows * kW) {
    lds[lane % kW / kCols][lane / kW * 8 + wave * kCols + lane % kCols] = mine;
  }
  __syncthreads();
  if (wave != 0) return;
  float z[kV];
  const int at = min(row, kRows - 1) * 8 + col - first;
#pragma unroll
  for (int e = 0; e < kV; ++e) z[e] = lds[0][at + e] + bias[e];
  const int left = row < min(kRows, a.m) ? a.n - col : 0;
  if constexpr (gated(kJob)) {
    float u[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) u[e] = lds[kHalves - 1][at + e];
    float biases[2][kV];
    load_biases<T>(a, col, left, biases);
    const u32x4 grad = kJob == Job::kGatedGrad ? load_grad<T>(a, row, col, left) : u32x4{};
    float row_sums[2][kV] = {};
    finish_gated<T, kJob == Job::kGatedGrad>(a, row, col, left, z, u, biases, grad, row_sums);
    if (kJob == Job::kGatedGrad && a.row_sums != nullptr && left > 0) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        if (e < left) {
          a.row_sums[static_cast<int64_t>(row) * 2 * a.n + col + e] = row_sums[0][e];
          a.row_sums[static_cast<int64_t>(row) * 2 * a.n + a.n + col + e] = row_sums[1][e];
        }
      }
    }
    return;
  }
  // the whole wavefront: the mask's halves are exchanged between lanes
  finish_forward<T>(a, row, col, left, z);
}

// ----------------------------------------------------- gradient's last step ---

// dW and db from the parts of k: a workgroup takes 32 pieces of four columns (or 32
// rows of db) with eight threads each, which add every eighth part in order and join
// in LDS, in order. Reading is all of it: one thread a piece kept too little in
// flight (512 x 256 in 63 parts 16.6 us, 33 MB).
constexpr int kSumPieces = 32;

template <typename T>
__global__ __launch_bounds__(kThreads) void linear_weight_sum(const float *partial,
                                                              const float *bias_partial, T *dw,
                                                              T *db, int m, int n, int splits) {
  constexpr int kRuns = kThreads / kSumPieces;
  __shared__ __attribute__((aligned(16))) f32x4 lds[kRuns][kSumPieces];
  const int ld = (n + 7) & ~7, per_row = ld / 4;
  const int x = threadIdx.x % kSumPieces, y = threadIdx.x / kSumPieces;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kSumPieces + x;
  const int64_t count = static_cast<int64_t>(m) * per_row;
  const bool weight = i < count, bias = !weight && db != nullptr && i - count < m;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (weight) {
    const float *src = partial + i * 4;
    const int64_t stride = static_cast<int64_t>(m) * ld;
    int u = y;
    for (; u + 3 * kRuns < splits; u += 4 * kRuns) {
      f32x4 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = *reinterpret_cast<const f32x4 *>(src + (u + e * kRuns) * stride);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s += v[e];
    }
    for (; u < splits; u += kRuns) s += *reinterpret_cast<const f32x4 *>(src + u * stride);
  } else if (bias) {
    for (int u = y; u < splits; u += kRuns) {
      s[0] += bias_partial[static_cast<int64_t>(u) * m + (i - count)];
    }
  }
  lds[y][x] = s;
  __syncthreads();
  if (y != 0) return;
#pragma unroll
  for (int u = 1; u < kRuns; ++u) s += lds[u][x];
  if (weight) {
    const int64_t row = i / per_row;
    const int col = static_cast<int>(i - row * per_row) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (col + e < n) dw[row * n + col + e] = from_float<T>(s[e]);
    }
  } else if (bias) {
    db[i - count] = from_float<T>(s[0]);
  }
}

// db of the gated layer from its rows of sums.
template <typename T>
__global__ __launch_bounds__(kThreads) void gated_bias_sum(const float *rows, int parts,
                                                           int columns, T *db) {
  static_assert(kThreads == 256, "add_rows");
  const int col = blockIdx.x * 16 + (threadIdx.x & 15);
  const float total = add_rows(rows + col, col < columns ? parts : 0, columns);
  if (threadIdx.x < 16 && col < columns) db[col] = from_float<T>(total);
}

// ------------------------------------------------------------- elementwise ---

// i / d and i % d, with the short division where it holds
__device__ __forceinline__ int64_t divide(int64_t i, int d, int &rest) {
  if (i < (int64_t{1} << 32)) {
    const uint32_t n = static_cast<uint32_t>(i), q = n / static_cast<uint32_t>(d);
    rest = static_cast<int>(n - q * static_cast<uint32_t>(d));
    return q;
  }
  const int64_t q = i / d;
  rest = static_cast<int>(i - q * d);
  return q;
}

// dz = g * gelu'(z), the derivative as the forward kept it. dz is an operand of two matrix products;
// in a 16-bit type it is written as two numbers, itself rounded and what the rounding
// left, which the products add: rounded once, dz would cost the gradients as much
// precision again as their own rounding does. A dz past the type's range becomes its
// largest number and the rest. Rows are padded with zeros to whole chunks, which the
// products then read as if they were aligned, whatever the number of columns.
template <typename T>
__global__ __launch_bounds__(kThreads) void linear_gelu_grad(const T *g, const T *slope, T *dz,
                                                             T *rest, int64_t rows, int cols) {
  constexpr int kV = Piece<T>::kValues;
  constexpr float kLargest = std::is_same_v<T, __half> ? 65504.0f : 3.38953139e38f;
  const int per_row = (cols + kV - 1) / kV;
  const int64_t chunks = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < chunks;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    int chunk;
    const int64_t row = divide(i, per_row, chunk);
    const int col = chunk * kV;
    float a[kV], b[kV];
    unpack<T>(loose_load<T>(g + row * cols + col, cols - col), a);
    unpack_slopes<T>(loose_load<T>(slope + row * cols + col, cols - col), b);
#pragma unroll
    for (int e = 0; e < kV; ++e) a[e] *= b[e];
    u32x4 *const to = reinterpret_cast<u32x4 *>(dz) + i;
    if constexpr (sizeof(T) == 2) {
      float h[kV];
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        // infinities and NaN stay what they are
        h[e] = fabsf(a[e]) < INFINITY ? fminf(fmaxf(a[e], -kLargest), kLargest) : a[e];
      }
      const u32x4 w = pack<T>(h);
      *to = w;
      unpack<T>(w, h);
#pragma unroll
      for (int e = 0; e < kV; ++e) a[e] = fabsf(a[e]) < INFINITY ? a[e] - h[e] : 0.0f;
      reinterpret_cast<u32x4 *>(rest)[i] = pack<T>(a);
    } else {
      *to = pack<T>(a);
    }
  }
}

// x in 8 bits: codes [rows][pad32(cols)], zero past cols, and scales (encode).
template <typename T>
__global__ __launch_bounds__(kThreads) void linear_checkpoint(const T *x, uint8_t *codes,
                                                              uint8_t *scales, int64_t rows,
                                                              int cols) {
  constexpr int kV = Piece<T>::kValues;
  const int padded = (cols + 31) & ~31, per_row = padded / kV;
  const int64_t chunks = rows * per_row;
  // per_row and the launch's stride are multiples of a block's lanes: they stay together
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < chunks;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    int chunk;
    const int64_t row = divide(i, per_row, chunk);
    const int col = chunk * kV;
    float v[kV];
    unpack<T>(loose_load<T>(x + row * cols + col, cols - col), v);
    uint32_t w[kV / 4];
    const uint32_t scale = encode<T>(v, w);
    keep_codes<T>(codes, scales, row, col, padded, w, scale);
  }
}

}  // namespace dense
