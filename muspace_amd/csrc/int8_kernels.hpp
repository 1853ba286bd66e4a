// The linear layer in 8-bit integers (include/muspace_layer.h):
//
//   s_r = max(max |x_r| / 127, 2^-126), q_rk = rint(x_rk / s_r)     rows of x, and of W before
//   y = act(s_r t_o sum of q_rk w_ok + b_o) + residual              w codes, t scales of W
//
// Sums are exact, in int32 (in_features up to 2^17). The row's quotients are float32
// divisions, so that codes are the same on any machine.
//
// int8_rows quantises, or, of few rows or many short ones, the product's own kernel;
// int8_product is linear_product (linear_kernels.hpp) with 128 codes a step in the same 128
// bytes: the same LDS layout serves, a lane's 16 bytes of a row are 16 codes, and v_mfma_i32_32x32x32_i8 takes 32 of k a time, at twice the 16-bit types' rate.
// Rows of x's codes are padded with zeros to whole chunks, so what a weight's chunk holds
// past the row's end (the next row's first codes) counts for nothing.
#pragma once

#include "linear_kernels.hpp"

namespace dense {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kCodeStep = kRowBytes;  // of k

struct __attribute__((packed, aligned(1))) Bytes16 {
  u32x4 v;
};
struct __attribute__((packed, aligned(1))) Bytes8 {
  u32x2 v;
};
struct __attribute__((packed, aligned(1))) Bytes4 {
  uint32_t v;
};

// ---------------------------------------------------------------- quantise ---

constexpr int kQuantThreads = 512;

struct Quantise {
  const void *x;
  int8_t *codes;
  float *scales;
  int64_t rows, ld;  // codes of a row in memory; zeros past cols
  int cols;
};

// the largest magnitude of kLanes lanes (as bits), the same on all of them
template <int kLanes>
__device__ __forceinline__ uint32_t team_top(uint32_t v, uint32_t *lds) {
  v = max(v, from_lane<1>(v));
  v = max(v, from_lane<2>(v));
  v = max(v, from_lane<4>(v));
#pragma unroll
  for (int d = 8; d < kWave && d < kLanes; d *= 2) {
    v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)));
  }
  if constexpr (kLanes > kWave) {
    const int wave = threadIdx.x / kWave, first = threadIdx.x / kLanes * (kLanes / kWave);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[wave] = v;
    __syncthreads();
    v = lds[first];
#pragma unroll
    for (int u = 1; u < kLanes / kWave; ++u) v = max(v, lds[first + u]);
  }
  return v;
}

// A row's scale from its largest magnitude; NaN for a row with an infinity or NaN.
__device__ __forceinline__ float row_scale(uint32_t top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
}

// A piece's codes, four a word. The quotient's nearest integer is that of the product with
// the reciprocal, which errs by 3 * 2^-24 * 127 < 2^-15 at the most, but where that falls
// as near as this to the middle of two: only then values are divided (a division takes ten
// instructions: 40000 x 256 bf16 10.9 us with it, 10.3 without).
// Codes of a row without a scale are 1: times NaN.
template <int kV>
__device__ __forceinline__ void encode_row(const float (&v)[kV], float scale, float inverse,
                                           uint32_t (&w)[kV / 4]) {
  float q[kV], far = 0.0f;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    const float product = v[e] * inverse;
    q[e] = rintf(product);
    far = fmaxf(far, fabsf(product - q[e]));
  }
  if (far > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int e = 0; e < kV; ++e) q[e] = rintf(v[e] / scale);
  }
#pragma unroll
  for (int i = 0; i < kV / 4; ++i) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = static_cast<uint32_t>(static_cast<int>(q[4 * i + e])) & 0xffu;
    }
    w[i] = scale == scale ? (c[0] | c[1] << 8) | (c[2] | c[3] << 8) << 16 : 0x01010101u;
  }
}

// `left` codes of a row in memory from `to` on
template <int kV>
__device__ __forceinline__ void store_codes(int8_t *to, const uint32_t (&w)[kV / 4], int64_t left) {
  if (left >= kV) {
    if constexpr (kV == 8) {
      reinterpret_cast<Bytes8 *>(to)->v = u32x2{w[0], w[1]};
    } else {
      reinterpret_cast<Bytes4 *>(to)->v = w[0];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    if (e < left) to[e] = static_cast<int8_t>(w[e / 4] >> (8 * (e & 3)));
  }
}

// Rows of up to kLanes pieces, a piece a lane; a wavefront holds several short rows. 40000 x 256
// bf16 9.3 us of 6.0 for its bytes, 16384 x 2048 24.9 of 19.5: a row's loads, its largest value and
// its codes follow one another, between barriers where a row takes several wavefronts, and no
// next row is on its way (with one, 40000 x 256 took 10.9 for 10.2: more registers, fewer wavefronts).
template <typename T, int kLanes>
__global__ __launch_bounds__(kQuantThreads) void int8_rows(const Quantise a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kGroups = kQuantThreads / kLanes;
  __shared__ uint32_t lds[kQuantThreads / kWave];
  const int lane = threadIdx.x % kLanes, col = lane * kV, left = a.cols - col;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows;
       base += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = base + threadIdx.x / kLanes;
    const bool any = row < a.rows;
    float v[kV];
    unpack<T>(loose_load<T>(static_cast<const T *>(a.x) + row * a.cols + col, any ? left : 0), v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    const float scale = row_scale(team_top<kLanes>(top, lds));
    if (!any) continue;
    uint32_t w[kV / 4];
    encode_row<kV>(v, scale, 1.0f / scale, w);
    store_codes<kV>(a.codes + row * a.ld + col, w, a.ld - col);
    if (lane == 0) a.scales[row] = scale;
  }
}

// Rows of any length: a workgroup a row, read twice, from the caches the second time.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void int8_rows_long(const Quantise a) {
  constexpr int kV = Piece<T>::kValues;
  __shared__ uint32_t lds[kQuantThreads / kWave];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.cols;
    uint32_t top = 0;
    for (int col = threadIdx.x * kV; col < a.cols; col += kQuantThreads * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, a.cols - col), v);
#pragma unroll
      for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    const float scale = row_scale(team_top<kQuantThreads>(top, lds));
    for (int64_t col = threadIdx.x * kV; col < a.ld; col += kQuantThreads * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, static_cast<int>(a.cols - col)), v);
      uint32_t w[kV / 4];
      encode_row<kV>(v, scale, 1.0f / scale, w);
      store_codes<kV>(a.codes + row * a.ld + col, w, a.ld - col);
    }
    if (threadIdx.x == 0) a.scales[row] = scale;
  }
}

// ----------------------------------------------------------------- product ---

struct Codes {
  const int8_t *x, *weight;             // x [m][ldx], weight [n][k]
  const float *x_scales, *weight_scales;
  int64_t ldx;
  Product p;                            // m, n, k, tiles and the epilogue; p.p: x itself
};

// R rows by a step of codes, 16 bytes a chunk (see Loader). !kTight: rows of any length,
// read at their own addresses; a chunk that would pass the end of the whole operand is
// read as its last 16 bytes, moved to the front.
template <int R, bool kTight, int kTeam = kThreads>
struct CodeLoader {
  static constexpr int kCount = R * 8 / kTeam;
  static constexpr int kDown = kTeam / 8;
  const int8_t *ptr;
  int64_t ld, end;  // end: bytes of the operand
  int row0, rows, r, c;
  u32x4 v[kCount];

  __device__ __forceinline__ void init(const int8_t *src, int64_t ld_, int row0_, int rows_) {
    ptr = src;
    ld = ld_;
    row0 = row0_;
    rows = rows_;
    end = ld_ * rows_;
    const int t = threadIdx.x % kTeam;
    r = t >> 3;
    c = t & 7;
  }

  __device__ __forceinline__ void fetch(int k0) {
    if constexpr (kTight) {
      Source s;
      s.base = reinterpret_cast<const char *>(ptr + row0 * ld + k0);
      const int64_t left = end - row0 * ld - k0;
      s.bytes = left > 0x7fffffff ? 0x7fffffffu : static_cast<uint32_t>(left);
      const bool inside = k0 + c * 16 < ld;
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const uint32_t off = static_cast<uint32_t>((r + kDown * i) * ld + c * 16);
        v[i] = tight_load(s, inside ? off : kPast);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const int64_t row = min(row0 + r + kDown * i, rows - 1);
        const int64_t off = row * ld + k0 + c * 16;
        if (end >= 16) {
          const int64_t at = min(off, end - 16);
          v[i] = reinterpret_cast<const Bytes16 *>(ptr + at)->v;
          const int64_t skip = off - at;
          if (skip > 0) v[i] = drop_front<int8_t>(v[i], skip > 16 ? 16 : static_cast<int>(skip));
        } else {
          u32x4 o = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (off + e < end) {
              o[e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(ptr[off + e])) << (8 * (e & 3));
            }
          }
          v[i] = o;
        }
      }
    }
  }

  __device__ __forceinline__ void put(char *tile) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      *reinterpret_cast<u32x4 *>(tile + along_offset<128>(r + kDown * i, c)) = v[i];
    }
  }
};

__device__ __forceinline__ i32x16 multiply_codes(const u32x4 &a, const u32x4 &b, i32x16 acc) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a),
                                               __builtin_bit_cast(i32x4, b), acc, 0, 0, 0);
#else
  return acc;
#endif
}

// A chunk of the result from its integer sums, of a row with scale `s`. (A sum past 2^24 is
// rounded to float32, relative 2^-24, as the two products with the scales are.)
template <typename T>
__device__ __forceinline__ void finish_codes(const Codes &a, float s, int64_t row, int col,
                                             int left, const int (&sum)[Piece<T>::kValues],
                                             const float (&scale)[Piece<T>::kValues],
                                             const float (&bias)[Piece<T>::kValues]) {
  constexpr int kV = Piece<T>::kValues;
  float z[kV];
#pragma unroll
  for (int e = 0; e < kV; ++e) z[e] = static_cast<float>(sum[e]) * s * scale[e] + bias[e];
  finish_forward<T>(a.p, row, col, left, z);
}

// the weight's scales and the bias of a chunk of columns
template <typename T>
__device__ __forceinline__ void load_columns(const Codes &a, int col, int left,
                                             float (&scale)[Piece<T>::kValues],
                                             float (&bias)[Piece<T>::kValues]) {
  constexpr int kV = Piece<T>::kValues;
#pragma unroll
  for (int e = 0; e < kV; e += 4) {
    float f[4];
    unpack<float>(loose_load<float>(a.weight_scales + col + e, left - e), f);
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[e + i] = f[i];
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) bias[e] = 0.0f;
  if (a.p.bias != nullptr) load_bias<T>(static_cast<const T *>(a.p.bias) + col, left, bias);
}

template <typename T, int BM, int BN, bool kTight>
__global__ __launch_bounds__(kThreads, 3) void int8_product(const Codes a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int WM = BM / 2, WN = BN / 2;  // a wavefront's quarter
  constexpr int kI = WM / 32, kJ = WN / 32;
  constexpr int kStageLd = WN + 4;  // ints; the pad spreads rows over the banks
  constexpr int kStage = 4 * 32 * kStageLd * 4, kTiles = (BM + BN) * kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[kStage > kTiles ? kStage : kTiles];
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int row0 = tile / a.p.tiles_n * BM, col0 = tile % a.p.tiles_n * BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * WM, wc = (wave & 1) * WN;
  CodeLoader<BM, true> p;
  CodeLoader<BN, kTight> q;
  p.init(a.x, a.ldx, row0, a.p.m);
  q.init(a.weight, a.p.k, col0, a.p.n);
  char *const tile_p = lds, *const tile_q = lds + BM * kRowBytes;
  i32x16 acc[kI][kJ] = {};
  if (a.p.k > 0) {
    p.fetch(0);
    q.fetch(0);
  }
  for (int k0 = 0; k0 < a.p.k; k0 += kCodeStep) {
    p.put(tile_p);
    q.put(tile_q);
    __syncthreads();
    if (k0 + kCodeStep < a.p.k) {
      p.fetch(k0 + kCodeStep);
      q.fetch(k0 + kCodeStep);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4 fp[kI], fq[kJ];
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        fp[i] = read_fragment<true, BM, 128>(tile_p, wr + 32 * i, s, lane);
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        fq[j] = read_fragment<true, BN, 128>(tile_q, wc + 32 * j, s, lane);
      }
#pragma unroll
      for (int i = 0; i < kI; ++i) {
#pragma unroll
        for (int j = 0; j < kJ; ++j) acc[i][j] = multiply_codes(fq[j], fp[i], acc[i][j]);
      }
    }
    __syncthreads();
  }
  // the tile, 32 rows of a wavefront at a time, through the wavefront's own LDS
  int *stage = reinterpret_cast<int *>(lds) + wave * 32 * kStageLd;
  constexpr int kLanes = WN / kV, kRows = kWave / kLanes;
  const int chunk = lane % kLanes;
  const int col = col0 + wc + chunk * kV, left = a.p.n - col;
  float scale[kV], bias[kV];
  load_columns<T>(a, col, left, scale, bias);
#pragma unroll
  for (int i = 0; i < kI; ++i) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        i32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
        *reinterpret_cast<i32x4 *>(stage + (lane & 31) * kStageLd + 32 * j + 8 * g +
                                   4 * (lane >> 5)) = v;
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int64_t row = row0 + wr + 32 * i + r;
      int sum[kV];
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const i32x4 v = *reinterpret_cast<const i32x4 *>(stage + r * kStageLd + chunk * kV + e);
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[e + x] = v[x];
      }
      finish_codes<T>(a, row < a.p.m && left > 0 ? a.x_scales[row] : 0.0f, row, col,
                      row < a.p.m ? left : 0, sum, scale, bias);
    }
    wave_lds_sync();
  }
}

// Where the tiles would leave most CUs idle (see linear_few): 32 x 32 results a workgroup,
// whose wavefronts take turns at the steps of k. kFused: the workgroup quantises its 32 rows
// itself, into LDS, while the weight's first steps are on their way, in place of a launch
// before (300 x 256 -> 256 float16: 3.1 + 4.0 us in two, 5.5 in one).
constexpr int kFusedIn = 2048;  // of k at the most: 64 KB of codes

template <typename T, int kWaves, bool kTight, bool kFused>
__global__ __launch_bounds__(kWaves *kWave) void int8_few(const Codes a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kTile = 32 * kRowBytes;
  constexpr int kLd = 36;
  constexpr int kOwn = kFused ? kTile : 2 * kTile;  // of a wavefront
  static_assert(32 * kLd * 4 <= 2 * kTile, "a wavefront's sums exceed its tiles");
  // fused: 16 tiles of the rows' codes, then the wavefronts' tiles of the weight; the sums
  // take the place of both
  __shared__ __attribute__((aligned(16))) char
      lds[kFused ? kFusedIn / kCodeStep * kTile + kWaves * kTile : kWaves * 2 * kTile];
  __shared__ float row_scales[32];
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int row0 = tile / a.p.tiles_n * 32, col0 = tile % a.p.tiles_n * 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char *const codes = lds;  // fused: of all steps
  char *const tile_q =
      kFused ? lds + kFusedIn / kCodeStep * kTile + wave * kOwn : lds + wave * kOwn + kTile;
  CodeLoader<32, true, kWave> p;
  CodeLoader<32, kTight, kWave> q;
  p.init(a.x, a.ldx, row0, a.p.m);
  q.init(a.weight, a.p.k, col0, a.p.n);
  i32x16 acc = {};
  int k0 = wave * kCodeStep;
  if (k0 < a.p.k) {
    if constexpr (!kFused) p.fetch(k0);
    q.fetch(k0);
  }
  if constexpr (kFused) {
    // 16 threads a row: its largest magnitude, then its codes (read again, from the caches)
    static_assert(kWaves * kWave == 32 * 16, "a row's threads are a row of lanes");
    const int r = threadIdx.x / 16, t = threadIdx.x % 16;
    const bool any = row0 + r < a.p.m;
    const T *x = static_cast<const T *>(a.p.p) + static_cast<int64_t>(row0 + r) * a.p.k;
    uint32_t top = 0;
    for (int col = t * kV; col < a.p.k; col += 16 * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, any ? a.p.k - col : 0), v);
#pragma unroll
      for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    const float scale = row_scale(team_top<16>(top, nullptr)), inverse = 1.0f / scale;
    if (t == 0) row_scales[r] = scale;
    // zeros up to whole steps
    const int steps_end = (a.p.k + kCodeStep - 1) / kCodeStep * kCodeStep;
    for (int col = t * kV; col < steps_end; col += 16 * kV) {
      float v[kV];
      uint32_t w[kV / 4];
      unpack<T>(loose_load<T>(x + col, any ? a.p.k - col : 0), v);
      encode_row<kV>(v, scale, inverse, w);
      char *to = codes + col / kCodeStep * kTile +
                 along_offset<128>(r, col % kCodeStep / 16) + col % 16;
      if constexpr (kV == 8) {
        *reinterpret_cast<u32x2 *>(to) = u32x2{w[0], w[1]};
      } else {
        *reinterpret_cast<uint32_t *>(to) = w[0];
      }
    }
    __syncthreads();
  }
  for (; k0 < a.p.k; k0 += kWaves * kCodeStep) {
    const char *const tile_p = kFused ? codes + k0 / kCodeStep * kTile : lds + wave * kOwn;
    if constexpr (!kFused) p.put(lds + wave * kOwn);
    q.put(tile_q);
    wave_lds_sync();
    if (k0 + kWaves * kCodeStep < a.p.k) {
      if constexpr (!kFused) p.fetch(k0 + kWaves * kCodeStep);
      q.fetch(k0 + kWaves * kCodeStep);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      acc = multiply_codes(read_fragment<true, 32, 128>(tile_q, 0, s, lane),
                           read_fragment<true, 32, 128>(tile_p, 0, s, lane), acc);
    }
    wave_lds_sync();
  }
  if constexpr (kFused) __syncthreads();  // the codes are every wavefront's
  constexpr int kSumBytes = 2 * kTile;
  int *const sums = reinterpret_cast<int *>(lds + wave * kSumBytes);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const i32x4 v = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    *reinterpret_cast<i32x4 *>(sums + (lane & 31) * kLd + 8 * g + 4 * (lane >> 5)) = v;
  }
  __syncthreads();
  constexpr int kLanes = 32 / kV;
  for (int i = threadIdx.x; i < 32 * kLanes; i += kWaves * kWave) {
    const int chunk = i % kLanes, r = i / kLanes;
    const int col = col0 + chunk * kV;
    const int64_t row = row0 + r;
    const int left = row < a.p.m ? a.p.n - col : 0;
    int sum[kV] = {};
#pragma unroll
    for (int u = 0; u < kWaves; ++u) {
      const int *src = reinterpret_cast<const int *>(lds + u * kSumBytes) + r * kLd + chunk * kV;
#pragma unroll
      for (int e = 0; e < kV; ++e) sum[e] += src[e];
    }
    float scale[kV], bias[kV];
    load_columns<T>(a, col, a.p.n - col, scale, bias);
    finish_codes<T>(a, kFused ? row_scales[r] : left > 0 ? a.x_scales[row] : 0.0f, row, col, left,
                    sum, scale, bias);
  }
}

// Many short rows: a workgroup quantises 64 rows into LDS, where their codes stay, and makes all
// their results, 128 columns at a time, the weight's next step on its way over the ends of
// results. x is read once, and nothing but results is written. 40000 x 256 -> 512 bf16 26.5 us,
// 12 of them the bytes': a workgroup's steps wait for each other at barriers. With the weight's
// fragments straight from the caches into registers none did, and it took 32.
constexpr int kBlockRows = 64;
constexpr int kBlockIn = 256;  // of k at the most: 16 KB of codes

template <typename T, bool kTight>
__global__ __launch_bounds__(kThreads, 3) void int8_row_block(const Codes a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int BN = 128, WN = BN / 2, kJ = WN / 32;  // a wavefront's part: 32 x 64
  constexpr int kTile = kBlockRows * kRowBytes;
  constexpr int kStageLd = WN + 4, kStage = 4 * 32 * kStageLd * 4;
  static_assert(BN * kRowBytes <= kStage, "the weight's tile and the results take turns");
  __shared__ __attribute__((aligned(16))) char codes[kBlockIn / kCodeStep * kTile], lds[kStage];
  __shared__ float row_scales[kBlockRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * 32, wc = (wave & 1) * WN;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kBlockRows;
  CodeLoader<BN, kTight> q;
  q.init(a.weight, a.p.k, 0, a.p.n);
  if (a.p.k > 0) q.fetch(0);
  {
    // 16 threads a row, 16 rows at a time
    constexpr int kTimes = kBlockRows / 16, kPieces = kBlockIn / (16 * kV);
    const int r = threadIdx.x / 16, t = threadIdx.x % 16;
    u32x4 piece[kTimes][kPieces];
#pragma unroll
    for (int u = 0; u < kTimes; ++u) {
      const int64_t row = row0 + 16 * u + r;
      const T *x = static_cast<const T *>(a.p.p) + row * a.p.k;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int col = (t + 16 * i) * kV;
        piece[u][i] = loose_load<T>(x + col, row < a.p.m ? a.p.k - col : 0);
      }
    }
#pragma unroll
    for (int u = 0; u < kTimes; ++u) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        float v[kV];
        unpack<T>(piece[u][i], v);
#pragma unroll
        for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
      }
      const float scale = row_scale(team_top<16>(top, nullptr)), inverse = 1.0f / scale;
      if (t == 0) row_scales[16 * u + r] = scale;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int col = (t + 16 * i) * kV;
        float v[kV];
        uint32_t w[kV / 4];
        unpack<T>(piece[u][i], v);
        encode_row<kV>(v, scale, inverse, w);
        char *to = codes + col / kCodeStep * kTile +
                   along_offset<128>(16 * u + r, col % kCodeStep / 16) + col % 16;
        if constexpr (kV == 8) {
          *reinterpret_cast<u32x2 *>(to) = u32x2{w[0], w[1]};
        } else {
          *reinterpret_cast<uint32_t *>(to) = w[0];
        }
      }
    }
  }
  __syncthreads();
  int *stage = reinterpret_cast<int *>(lds) + wave * 32 * kStageLd;
  constexpr int kLanes = WN / kV, kRows = kWave / kLanes;
  const int chunk = lane % kLanes;
  for (int col0 = 0; col0 < a.p.n; col0 += BN) {
    i32x16 acc[kJ] = {};
    for (int k0 = 0; k0 < a.p.k; k0 += kCodeStep) {
      q.put(lds);
      __syncthreads();
      if (k0 + kCodeStep < a.p.k) {
        q.fetch(k0 + kCodeStep);
      } else if (col0 + BN < a.p.n) {
        q.row0 = col0 + BN;
        q.fetch(0);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4 fp =
            read_fragment<true, kBlockRows, 128>(codes + k0 / kCodeStep * kTile, wr, s, lane);
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          acc[j] = multiply_codes(read_fragment<true, BN, 128>(lds, wc + 32 * j, s, lane), fp,
                                  acc[j]);
        }
      }
      __syncthreads();
    }
    const int col = col0 + wc + chunk * kV, left = a.p.n - col;
    float scale[kV], bias[kV];
    load_columns<T>(a, col, left, scale, bias);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        i32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[j][4 * g + e];
        *reinterpret_cast<i32x4 *>(stage + (lane & 31) * kStageLd + 32 * j + 8 * g +
                                   4 * (lane >> 5)) = v;
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int64_t row = row0 + wr + r;
      int sum[kV];
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const i32x4 v = *reinterpret_cast<const i32x4 *>(stage + r * kStageLd + chunk * kV + e);
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[e + x] = v[x];
      }
      finish_codes<T>(a, row_scales[wr + r], row, col, row < a.p.m ? left : 0, sum, scale, bias);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------ a row or a few ---

// Lane l's sum over the wavefront's lanes (as add_across).
__device__ __forceinline__ int sum_lanes(int v) {
#if defined(__HIP_DEVICE_COMPILE__)
  v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true);
  u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(v, v, false, false));
  v = static_cast<int>(r[0] + r[1]);
  r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
  v = static_cast<int>(r[0] + r[1]);
#endif
  return v;
}

__device__ __forceinline__ int dot_codes(const u32x4 &a, const u32x4 &b, int sum) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = __builtin_amdgcn_sdot4(static_cast<int>(a[i]), static_cast<int>(b[i]), sum, false);
  }
#endif
  return sum;
}

// Up to kRows rows: reading the weight is all of it, as in linear_vector. A workgroup of
// eight wavefronts makes 16 columns, two a wavefront; it quantises the rows itself while the
// weight's first chunks are on their way. bf16, one row: 4096 -> 16384 16.7 us (4.0 TB/s of the
// weight), 4096 -> 4096 7.6, one round of loads and the call; four rows 28 and 12.
constexpr int kVectorCodes = 48 << 10;  // of the rows, in LDS, at the most

template <typename T, int kRows>
__global__ __launch_bounds__(kQuantThreads) void int8_vector(const Codes a) {
  constexpr int kV = Piece<T>::kValues;
  constexpr int kCols = 2, kAcross = 16;
  constexpr int kAhead = 4;                // of a lane's chunks, in flight together
  constexpr int kSpan = kWave * 16;        // of k, a chunk a lane
  constexpr int kLanes = kAcross / kV;     // of a result row, at the end
  static_assert(kRows * kLanes <= kWave, "one wavefront ends it");
  extern __shared__ __attribute__((aligned(16))) char codes[];  // [kRows][pad16(k)]
  __shared__ uint32_t tops[kQuantThreads / kWave];
  __shared__ int sums[kRows][kAcross];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.x * kAcross, col0 = first + wave * kCols;
  const int k = a.p.k, padded = (k + 15) & ~15;
  const int8_t *w[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    w[c] = a.weight + static_cast<int64_t>(min(col0 + c, a.p.n - 1)) * k;
  }
  // the lane's chunk at `at`; one that passes the end as the row's last 16 bytes, moved
  auto load = [&](int at, u32x4(&v)[kCols]) {
    if (k >= 16) {
      const int from = min(at, k - 16), skip = at - from;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        v[c] = reinterpret_cast<const Bytes16 *>(w[c] + from)->v;
        if (skip > 0) v[c] = drop_front<int8_t>(v[c], min(skip, 16));
      }
    } else {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        v[c] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (at + e < k) {
            v[c][e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(w[c][at + e])) << (8 * (e & 3));
          }
        }
      }
    }
  };
  u32x4 wv[kAhead][kCols];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (i * kSpan < k) load(i * kSpan + lane * 16, wv[i]);
  }
  float scales[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    const T *x = static_cast<const T *>(a.p.p) + static_cast<int64_t>(min(m, a.p.m - 1)) * k;
    uint32_t top = 0;
    for (int col = threadIdx.x * kV; col < k; col += kQuantThreads * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, k - col), v);
#pragma unroll
      for (int e = 0; e < kV; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    const float scale = row_scale(team_top<kQuantThreads>(top, tops)), inverse = 1.0f / scale;
    scales[m] = scale;
    for (int col = threadIdx.x * kV; col < padded; col += kQuantThreads * kV) {
      float v[kV];
      uint32_t c[kV / 4];
      unpack<T>(loose_load<T>(x + col, k - col), v);
      encode_row<kV>(v, scale, inverse, c);
      char *to = codes + m * padded + col;
      if constexpr (kV == 8) {
        *reinterpret_cast<u32x2 *>(to) = u32x2{c[0], c[1]};
      } else {
        *reinterpret_cast<uint32_t *>(to) = c[0];
      }
    }
  }
  __syncthreads();
  int sum[kRows][kCols] = {};
  for (int k0 = 0; k0 < k; k0 += kAhead * kSpan) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = k0 + i * kSpan + lane * 16;
      if (at < k) {
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
          const u32x4 x = *reinterpret_cast<const u32x4 *>(codes + m * padded + at);
#pragma unroll
          for (int c = 0; c < kCols; ++c) sum[m][c] = dot_codes(wv[i][c], x, sum[m][c]);
        }
      }
    }
    if (k0 + kAhead * kSpan < k) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load(k0 + (kAhead + i) * kSpan + lane * 16, wv[i]);
    }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int v = sum_lanes(sum[m][c]);
      if (lane == 0) sums[m][wave * kCols + c] = v;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  const int row = lane / kLanes, chunk = lane % kLanes, col = first + chunk * kV;
  const int left = row < min(kRows, a.p.m) ? a.p.n - col : 0;
  int mine[kV];
  float s = scales[0];
#pragma unroll
  for (int m = 1; m < kRows; ++m) s = row == m ? scales[m] : s;
#pragma unroll
  for (int e = 0; e < kV; ++e) mine[e] = sums[min(row, kRows - 1)][chunk * kV + e];
  float scale[kV], bias[kV];
  load_columns<T>(a, col, a.p.n - col, scale, bias);
  finish_codes<T>(a, s, row, col, left, mine, scale, bias);
}

}  // namespace dense
