// Large products of the gated layer and of linear on integers (linear_kernels.hpp,
// int8_kernels.hpp): the results of linear_product and int8_product, in the same order of
// sums.
//
// A workgroup of eight wavefronts makes 256 x 256 products, a wavefront 128 x 64 of them:
// per step of 128 bytes of k it reads 24 KB of LDS for 32 matrix instructions, where a
// wavefront of a 128 x 128 tile reads 16 KB for 16, which is what bounds that one. Tiles go from
// memory into LDS without passing registers (buffer loads to LDS), a step ahead. Such a
// load writes 16 bytes a lane in lane order, so the layout of linear_device.hpp, which
// moves chunks within their rows, is made by permuting which chunk of memory a lane
// reads. Loads have no conditions: what lies beyond an operand, or k, reads as zeros.
//
// 16384 x 1024 -> 2 x 4096 bf16 274 us (0.99 PFLOP/s; in tiles of 128 331), 2048 x 2048 ->
// 2 x 4096 62 (87): a step takes 1.5 us, at 1.4 PFLOP/s, and the rest of a workgroup, 11 us, what
// ends its results above all, which nothing on the CU hides. Tiles of 256 x 128 at two
// workgroups a CU hid it and read more of LDS and memory (290), as did 128 x 128 at four, loaded
// like here (332).
#pragma once

#include "int8_kernels.hpp"

namespace dense {

constexpr int kWide = 256;  // rows and columns of a tile
constexpr int kWideThreads = 512;
constexpr int kWideTile = kWide * kRowBytes, kWideStage = 2 * kWideTile;  // bytes of LDS
constexpr int kWidePasses = 4;  // loads of a thread, operand and step: 64 rows of the tile each

// An operand's tile by steps of k. Rows in memory are whole chunks on 16-byte boundaries.
// kHalves: the gated weight, whose rows in LDS are 32 of either half in turn; a
// wavefront's are of one half.
template <typename T, bool kHalves>
struct Stream {
  static constexpr int kV = 16 / static_cast<int>(sizeof(T));
  const T *ptr;
  int64_t ld;
  int row0, rows, k_end, c;  // c: the thread's chunk of memory, in its row
  uint32_t offset, stride;   // of the thread's first row in the window; between its rows

  __device__ __forceinline__ void init(const void *src, int64_t ld_, int row0_, int rows_,
                                       int k_end_) {
    ptr = static_cast<const T *>(src);
    ld = ld_;
    row0 = row0_;
    rows = rows_;
    k_end = k_end_;
    int r = threadIdx.x / 8;
    c = threadIdx.x % 8 ^ (r >> 1 & 7);  // (as along_offset)
    stride = static_cast<uint32_t>(64 * ld * sizeof(T));
    if constexpr (kHalves) {
      if (r >= 32) ptr += rows * ld;
      r &= 31;
      stride /= 2;
    }
    offset = static_cast<uint32_t>((r * ld + c * kV) * sizeof(T));
  }

  // the step's tile into LDS: there once the wavefronts' loads are done and all have met
  __device__ __forceinline__ void issue(char *tile, int k0) const {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void *lds_ptr;
    const int64_t left =
        ((static_cast<int64_t>(rows) - row0) * ld - k0) * static_cast<int64_t>(sizeof(T));
    // (the halves' pointers differ between wavefronts, not within one)
    const uint64_t at = reinterpret_cast<uint64_t>(ptr + row0 * ld + k0);
    const uint64_t base =
        static_cast<uint64_t>(static_cast<uint32_t>(
            __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32)))) << 32 |
        static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<char *>(base), 0,
        left > 0x7fffffff ? 0x7fffffffu : (left < 0 ? 0u : static_cast<uint32_t>(left)),
        0x00020000);
    const bool inside = k0 + c * kV < k_end;
    char *const to = tile + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int i = 0; i < kWidePasses; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(to + i * 64 * kRowBytes), 16,
                                               inside ? offset + i * stride : kPast, 0, 0, 0);
    }
#endif
  }
};

// Until at most `kLeft` of the wavefront's loads are under way.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
#if defined(__HIP_DEVICE_COMPILE__)
  static_assert(kLeft < 64, "the counter has six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kLeft & 15) | (kLeft >> 4) << 14);
#endif
}

// T: the operands' type (int8_t: codes, Job::kForward); Out: the result's
template <typename T, typename Out, Job kJob>
__global__ __launch_bounds__(kWideThreads, 2) void wide_product(const Codes a) {
  constexpr bool kInt = std::is_same_v<T, int8_t>;
  static_assert(kInt ? kJob == Job::kForward : gated(kJob), "both operands lie along k");
  constexpr int kV = Piece<Out>::kValues;
  constexpr int kStep = kRowBytes / static_cast<int>(sizeof(T));
  constexpr int WM = 128, WN = 64, kI = WM / 32, kJ = WN / 32;  // a wavefront's part
  constexpr int kColumns = gated(kJob) ? kWide / 2 : kWide;     // of the result
  constexpr int kStageLd = WN + 4;
  using Acc = std::conditional_t<kInt, i32x16, f32x16>;
  using Word4 = std::conditional_t<kInt, i32x4, f32x4>;
  using Word = std::conditional_t<kInt, int, float>;
  __shared__ __attribute__((aligned(16))) char lds[2 * kWideStage];
  static_assert(8 * 32 * kStageLd * 4 <= sizeof(lds), "results' rows go through the tiles");

  const int tile = xcd_order(blockIdx.x, gridDim.x);
  // four rows of tiles at a time, column by column: what the CUs of an XCD work on together
  // then shares rows of both operands in its L2
  const int rows_of_tiles = a.p.tiles / a.p.tiles_n, group = tile / (4 * a.p.tiles_n);
  const int within = tile - group * 4 * a.p.tiles_n, high = min(4, rows_of_tiles - 4 * group);
  const int row0 = (4 * group + within % high) * kWide, col0 = within / high * kColumns;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = wave / 4 * WM, wc = wave % 4 * WN;

  Stream<T, false> p;
  Stream<T, gated(kJob)> q;
  // (rows of codes are padded to whole chunks, in which k may end)
  p.init(kInt ? static_cast<const void *>(a.x) : a.p.p, kInt ? a.ldx : a.p.ldp, row0, a.p.m, a.p.k);
  q.init(kInt ? static_cast<const void *>(a.weight) : a.p.q, kInt ? a.p.k : a.p.ldq, col0, a.p.n,
         a.p.k);
  auto issue = [&](char *stage, int k0) {
    p.issue(stage, k0);
    q.issue(stage + kWideTile, k0);
  };

  // A step's quarters of 16 values (32 codes) of k: the next quarter's fragments are on their
  // way while one is multiplied. Before the last quarter the wavefronts meet: what they read of
  // the step is in registers, and the next step's tiles are there. (Steps past k are zeros;
  // their loads keep the count of those under way the same.)
  u32x4 fp[2][kI], fq[2][kJ];
  auto read = [&](const char *stage, int part) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      fq[part & 1][j] =
          read_fragment<true, kWide, kRowBytes>(stage + kWideTile, wc + 32 * j, part, lane);
    }
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      fp[part & 1][i] = read_fragment<true, kWide, kRowBytes>(stage, wr + 32 * i, part, lane);
    }
  };
  Acc acc[kI][kJ] = {};
  issue(lds, 0);
  issue(lds + kWideStage, kStep);
  wait_loads<2 * kWidePasses>();
  __syncthreads();
  read(lds, 0);
  int at = 0;  // the step's place in LDS
  for (int k0 = 0; k0 < a.p.k; k0 += kStep, at ^= kWideStage) {
#pragma unroll
    for (int part = 0; part < 4; ++part) {
      if (part < 3) {
        read(lds + at, part + 1);
      } else {
        wait_loads<0>();
        __syncthreads();
        issue(lds + at, k0 + 2 * kStep);
        read(lds + (at ^ kWideStage), 0);
      }
#pragma unroll
      for (int i = 0; i < kI; ++i) {
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          if constexpr (kInt) {
            acc[i][j] = multiply_codes(fq[part & 1][j], fp[part & 1][i], acc[i][j]);
          } else {
            acc[i][j] = multiply<T>(fq[part & 1][j], fp[part & 1][i], acc[i][j]);
          }
        }
      }
    }
  }
  wait_loads<0>();  // none may write into the results' rows
  __syncthreads();

  // the tile, 32 rows of a wavefront at a time, through the wavefront's own LDS
  Word *stage = reinterpret_cast<Word *>(lds) + wave * 32 * kStageLd;
  constexpr int kOut = gated(kJob) ? WN / 2 : WN;  // a wavefront's columns of the result
  constexpr int kLanes = kOut / kV;                // lanes per row
  constexpr int kRows = kWave / kLanes;            // rows at a time
  const int chunk = lane % kLanes;
  const int col = col0 + (gated(kJob) ? wc / 2 : wc) + chunk * kV, left = a.p.n - col;
  float scale[kV], bias[kV], biases[2][kV];
  if constexpr (kInt) load_columns<Out>(a, col, left, scale, bias);
  float row_sums[2][kV] = {};
  if constexpr (gated(kJob)) load_biases<Out>(a.p, col, left, biases);
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    u32x4 grads[32 / kRows] = {};
    if constexpr (kJob == Job::kGatedGrad) {
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += kRows) {
        const int64_t row = row0 + wr + 32 * i + r0 + lane / kLanes;
        grads[r0 / kRows] = load_grad<Out>(a.p, row, col, row < a.p.m ? left : 0);
      }
    }
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        Word4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
        *reinterpret_cast<Word4 *>(stage + (lane & 31) * kStageLd + 32 * j + 8 * g +
                                   4 * (lane >> 5)) = v;
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int64_t row = row0 + wr + 32 * i + r;
      const Word *src = stage + r * kStageLd + chunk * kV;
      const int here = row < a.p.m ? left : 0;
      Word z[kV];
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const Word4 v = *reinterpret_cast<const Word4 *>(src + e);
#pragma unroll
        for (int x = 0; x < 4; ++x) z[e + x] = v[x];
      }
      if constexpr (kInt) {
        finish_codes<Out>(a, here > 0 ? a.x_scales[row] : 0.0f, row, col, here, z, scale, bias);
      } else {
        float u[kV];
#pragma unroll
        for (int e = 0; e < kV; e += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4 *>(src + kOut + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) u[e + x] = v[x];
        }
        finish_gated<Out, kJob == Job::kGatedGrad>(a.p, row, col, here, z, u, biases,
                                                   grads[r0 / kRows], row_sums);
      }
    }
    wave_lds_sync();
  }
  if constexpr (kJob == Job::kGatedGrad) {
    leave_sums<Out, kLanes>(a.p, row0 / kWide * 2 + wave / 4, lane, col, left, row_sums);
  }
}

// Whether m x n products of k values of `size` bytes are made in these tiles: k long against the
// 11 us that are not its, and the workgroups, one a CU, filling their rounds over the 256 CUs by
// 85%, or 70% of rows of 4096 bytes. us, in tiles of 128 and in these, gated forward bf16: 8192 x
// 1024 -> 2 x 2048 (512 tiles, 100%) 83 and 70 us, 16384 x 1024 -> 2 x 1664 (832, 81%) 129 and
// 130, 11000 x 1024 -> 2 x 1664 (559, 73%) 98 and 102, 11000 x 2048 -> 2 x 1664 194 and 172, 40000
// x 256 -> 2 x 512 (628) 38 and 46, 20000 x 512 -> 2 x 1024 (632) 54 and 60; integers: 16384 x
// 1024 -> 8192 (100%) 227 and 195, 16384 x 1024 -> 3328 (81%) 95 and 103, x 4096 325 and 291.
// And where whole tiles are under a third more rows, and columns, than tiles of 128: 5 x 1024 -> 2 x
// 28672 24 and 32, 128 rows 28 and 35, 160 rows 49 and 35, 288 rows 67 and 62, 288 x 2048 -> 2 x
// 24576 103 and 111, 448 rows 122 and 113; 60000 x 1024 -> 2 x 64 23 and 32, 2 x 72 38 and 33, 2 x
// 160 56 and 60; integers: 128 x 1024 -> 57344 22 and 28, 160 rows 35 and 29, 288 rows 48 and 49, 60000
// x 1024 -> 128 57 and 64, 144 columns 65 and 65 (70 and 67 in another session), 320 76 and 85.
inline int64_t whole(int64_t n, int tile) { return (n + tile - 1) / tile * tile; }
inline bool wide_tiles(int64_t m, int64_t n, int64_t k, int size) {
  const int64_t tiles = whole(m, kWide) / kWide * (whole(n, kWide) / kWide);
  const int64_t rounds = (tiles + 255) / 256;
  return k >= 1024 && whole(m, kWide) * 3 < whole(m, 128) * 4 &&
         whole(n, kWide) * 3 < whole(n, 128) * 4 &&
         tiles * 100 >= rounds * 256 * (k * size >= 4096 ? 70 : 85);
}

}  // namespace dense
