// Layer norm over the last dimension and its gradients (include/muspace_layer.h).
//
//   c = x - mean(x), s = 1 / sqrt(mean(c^2) + eps), y = c s w + b
//   dx = s (u - mean(u) - h mean(u h)),  u = g w, h = c s
//   dw = sum of g h, db = sum of g over rows
//
// Memory-bound: every value of x (and g) is read once, held in registers over the
// reductions, and the result written once. kLanes lanes share a row, each with
// kChunks 16-byte pieces at a stride of kLanes; a wavefront holds several short
// rows. Wavefronts walk the rows with the next row's pieces on their way.
//
// The mean is held as an offset from a base, the row's first value x0 or zero, the
// nearer of the two: c = (x - base) - offset. Rows far from zero, where float32 has
// few bits for a mean, are then as exact as the differences of their values, a
// constant row gives c = 0 exactly, and a first value far from the others (a channel
// of large activation) does not set the size at which they are rounded. A first
// reduction sums x - x0, which finds base and offset to a few roundings of the row's
// reach; the second sums c and c^2 together, and the mean of c corrects the offset (and
// the variance). Kept for the backward: the offset, and s, negative where the base
// is zero.
//
// The backward keeps each column's sums in registers over its rows; workgroups
// leave one row of sums each, and norm_sum_columns adds them in workgroup order.
#pragma once

#include "linear_device.hpp"

namespace dense {

constexpr int kNormThreads = 512;

// kLanes lanes' sums, the same on all of them
template <int kLanes, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = add_across<8>(add_across<4>(add_across<2>(add_across<1>(v[i]))));
    if constexpr (kLanes >= 32) v[i] = add_across<16>(v[i]);
    if constexpr (kLanes >= 64) v[i] = add_across<32>(v[i]);
  }
  if constexpr (kLanes > kWave) {
    // one row per workgroup: wavefront sums through LDS
    constexpr int kWaves = kLanes / kWave;
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < kWaves; ++u) v[i] += lds[u * N + i];
    }
  }
}

// a piece of weight or bias: kW32 says that they are float32 next to a 16-bit type
template <typename T, bool kW32>
__device__ __forceinline__ void load_weight(const void *p, int col, int left,
                                            float (&w)[Piece<T>::kValues], float none) {
  constexpr int kV = Piece<T>::kValues;
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < kV; ++e) w[e] = none;
  } else if constexpr (kW32) {
    float lo[4], hi[4];
    const float *f = static_cast<const float *>(p) + col;
    unpack<float>(loose_load<float>(f, left), lo);
    unpack<float>(loose_load<float>(f + 4, left - 4), hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = lo[e];
      w[(e + 4) % kV] = hi[e];
    }
  } else {
    unpack<T>(loose_load<T>(static_cast<const T *>(p) + col, left), w);
  }
}

struct Norm {
  const void *x, *weight, *bias, *grad;
  void *out;
  float *stats;        // [rows][2]: offset, s or -s (keep_centre)
  float *partial;      // [workgroups][2][cols]
  int64_t rows;
  int cols;
  float eps;
};

// What is subtracted from a row's values: the base, then the offset.
struct Centre {
  float base, offset;
};

// from the first sum; an infinity or NaN ends in the offset, and with it in every value
__device__ __forceinline__ Centre find_centre(float x0, float mean_from_x0) {
  const float mean = x0 + mean_from_x0;
  return fabsf(mean_from_x0) < fabsf(mean) ? Centre{x0, mean_from_x0} : Centre{0.0f, mean};
}

// s from the second sums, of c and c^2, whose mean goes to the offset. (fma: an infinite
// sum of squares stays one, whatever the mean's square.)
__device__ __forceinline__ float correct_centre(Centre &centre, const float (&sums)[2], float inv,
                                                float eps) {
  const float rest = sums[0] * inv;
  centre.offset += rest;
  return 1.0f / sqrtf(fmaxf(fmaf(-rest, rest, sums[1] * inv), 0.0f) + eps);
}

__device__ __forceinline__ void keep_centre(float *stats, float x0, const Centre &centre, float s) {
  stats[0] = centre.offset;
  stats[1] = centre.base == x0 ? s : -s;
}

__device__ __forceinline__ Centre kept_centre(float x0, float offset, float s) {
  return Centre{__float_as_uint(s) >> 31 ? 0.0f : x0, offset};
}

template <int kLanes>
struct NormShape {
  static constexpr int kThreads = kLanes > kWave ? kLanes : kNormThreads;
  static constexpr int kGroups = kThreads / kLanes;  // rows at a time
};

// A lane's pieces of a row. All loads are unconditional, so that a row's are in
// flight together: a piece that passes the row's end is read as the row's last 16
// bytes and its values are moved to the front when it is used, rows past the last
// read the last and count as zeros. kFull: the pieces end with the row. Rows shorter
// than a piece are read value by value.
template <typename T, int kLanes, int kChunks, bool kFull>
struct RowPieces {
  static constexpr int kV = Piece<T>::kValues;
  u32x4 v[kChunks];

  static __device__ __forceinline__ int left(int cols, int lane, int i) {
    return kFull ? kV : cols - (lane + i * kLanes) * kV;
  }
  __device__ __forceinline__ void load(const T *x, int64_t row, int64_t rows, int cols, int lane) {
    const T *p = x + min(row, rows - 1) * cols;
    if (kFull || cols >= kV) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = (lane + i * kLanes) * kV;
        v[i] = reinterpret_cast<const Loose16 *>(p + (kFull ? col : min(col, cols - kV)))->v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) v[i] = loose_load<T>(p, i == 0 && lane == 0 ? cols : 0);
    }
  }
  // the piece's values, zeros past the row (and of no row: `any` false)
  __device__ __forceinline__ void values(int i, int cols, int lane, bool any, float (&o)[kV]) const {
    u32x4 w = v[i];
    if (!kFull && cols >= kV) {
      w = drop_front<T>(w, max((lane + i * kLanes + 1) * kV - cols, 0));
    }
    if (!any) w = u32x4{0, 0, 0, 0};
    unpack<T>(w, o);
  }
};

template <typename T, bool kW32, int kLanes, int kChunks, bool kFull>
__global__ __launch_bounds__(NormShape<kLanes>::kThreads) void norm_forward(const Norm a) {
  using Shape = NormShape<kLanes>;
  constexpr int kV = Piece<T>::kValues;
  constexpr bool kHold = kChunks <= 3;  // weight and bias stay in registers
  __shared__ float lds[16];
  using Pieces = RowPieces<T, kLanes, kChunks, kFull>;
  const int lane = threadIdx.x % kLanes;
  const T *x = static_cast<const T *>(a.x);
  T *out = static_cast<T *>(a.out);
  const float inv = 1.0f / static_cast<float>(a.cols);
  float w[kChunks][kV], b[kChunks][kV];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (lane + i * kLanes) * kV;
      load_weight<T, kW32>(a.weight, col, a.cols - col, w[i], 1.0f);
      load_weight<T, kW32>(a.bias, col, a.cols - col, b[i], 0.0f);
    }
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * Shape::kGroups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * Shape::kGroups + threadIdx.x / kLanes;
  Pieces next;
  next.load(x, row, a.rows, a.cols, lane);
  // groups of one wavefront walk together: lanes past the last row take part in the
  // sums with zeros
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * Shape::kGroups; base < a.rows;
       base += step, row += step) {
    float v[kChunks][kV];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) next.values(i, a.cols, lane, row < a.rows, v[i]);
    const bool any = row < a.rows;
    float x0;
    if constexpr (kLanes > kWave) {
      x0 = to_float(x[row * a.cols]);
    } else {
      x0 = __shfl(v[0][0], 0, kLanes);
    }
    next.load(x, row + step, a.rows, a.cols, lane);
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        sum[0] += kFull || e < Pieces::left(a.cols, lane, i) ? v[i][e] - x0 : 0.0f;
      }
    }
    group_sum<kLanes, 1>(sum, lds);
    Centre centre = find_centre(x0, sum[0] * inv);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        v[i][e] -= centre.base;
        const float c =
            kFull || e < Pieces::left(a.cols, lane, i) ? v[i][e] - centre.offset : 0.0f;
        sums[0] += c;
        sums[1] += c * c;
      }
    }
    group_sum<kLanes, 2>(sums, lds);
    const float s = correct_centre(centre, sums, inv, a.eps);
    if (a.stats != nullptr && any && lane == 0) keep_centre(a.stats + 2 * row, x0, centre, s);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (lane + i * kLanes) * kV;
      if constexpr (!kHold) {
        load_weight<T, kW32>(a.weight, col, a.cols - col, w[i], 1.0f);
        load_weight<T, kW32>(a.bias, col, a.cols - col, b[i], 0.0f);
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        v[i][e] = (v[i][e] - centre.offset) * s * w[i][e] + b[i][e];
      }
      loose_store(out + row * a.cols + col, pack<T>(v[i]),
                  any ? Pieces::left(a.cols, lane, i) : 0);
    }
  }
}

template <typename T, bool kW32, int kLanes, int kChunks, bool kFull>
__global__ __launch_bounds__(NormShape<kLanes>::kThreads) void norm_backward(const Norm a) {
  using Shape = NormShape<kLanes>;
  constexpr int kV = Piece<T>::kValues;
  constexpr bool kHold = kChunks <= 3;
  constexpr int kCols = kLanes * kChunks * kV;
  using Pieces = RowPieces<T, kLanes, kChunks, kFull>;
  __shared__ float lds[Shape::kGroups > 1 ? Shape::kGroups * kCols : 16];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const T *x = static_cast<const T *>(a.x), *g = static_cast<const T *>(a.grad);
  T *dx = static_cast<T *>(a.out);
  const float inv = 1.0f / static_cast<float>(a.cols);
  float w[kChunks][kV];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = (lane + i * kLanes) * kV;
      load_weight<T, kW32>(a.weight, col, a.cols - col, w[i], 1.0f);
    }
  }
  float dw[kChunks][kV] = {}, db[kChunks][kV] = {};
  const int64_t step = static_cast<int64_t>(gridDim.x) * Shape::kGroups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * Shape::kGroups + group;
  Pieces nx, ng;
  float n_offset = 0.0f, n_s = 0.0f;
  auto fetch = [&](int64_t r) {
    nx.load(x, r, a.rows, a.cols, lane);
    ng.load(g, r, a.rows, a.cols, lane);
    const f32x2 stats = reinterpret_cast<const f32x2 *>(a.stats)[min(r, a.rows - 1)];
    n_offset = stats[0];
    n_s = stats[1];
  };
  fetch(row);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * Shape::kGroups; base < a.rows;
       base += step, row += step) {
    float h[kChunks][kV], u[kChunks][kV];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      nx.values(i, a.cols, lane, row < a.rows, h[i]);
      ng.values(i, a.cols, lane, row < a.rows, u[i]);
    }
    const bool any = row < a.rows;
    const float s = fabsf(n_s);
    float x0;
    if constexpr (kLanes > kWave) {
      x0 = to_float(x[row * a.cols]);
    } else {
      x0 = __shfl(h[0][0], 0, kLanes);
    }
    const Centre centre = kept_centre(x0, n_offset, n_s);
    fetch(row + step);
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if constexpr (!kHold) {
        const int col = (lane + i * kLanes) * kV;
        load_weight<T, kW32>(a.weight, col, a.cols - col, w[i], 1.0f);
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        // the operations of the forward, so that h is the forward's own
        h[i][e] = kFull || e < Pieces::left(a.cols, lane, i)
                      ? (h[i][e] - centre.base - centre.offset) * s
                      : 0.0f;
        dw[i][e] += u[i][e] * h[i][e];
        db[i][e] += u[i][e];
        u[i][e] *= w[i][e];
        sum[0] += u[i][e];
        sum[1] += u[i][e] * h[i][e];
      }
    }
    if (a.out != nullptr) {
      group_sum<kLanes, 2>(sum, lds);
      const float mu = sum[0] * inv, mh = sum[1] * inv;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
#pragma unroll
        for (int e = 0; e < kV; ++e) u[i][e] = s * (u[i][e] - mu - h[i][e] * mh);
        loose_store(dx + row * a.cols + (lane + i * kLanes) * kV, pack<T>(u[i]),
                    any ? Pieces::left(a.cols, lane, i) : 0);
      }
    }
  }
  if (a.partial == nullptr) return;
  float *to = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
  if constexpr (Shape::kGroups == 1) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        const int col = (lane + i * kLanes) * kV + e;
        if (col < a.cols) {
          to[col] = dw[i][e];
          to[a.cols + col] = db[i][e];
        }
      }
    }
  } else {
    auto join = [&](const float(&d)[kChunks][kV], float *dst) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
#pragma unroll
        for (int e = 0; e < kV; e += 4) {
          const f32x4 v = {d[i][e], d[i][e + 1], d[i][e + 2], d[i][e + 3]};
          *reinterpret_cast<f32x4 *>(lds + group * kCols + (lane + i * kLanes) * kV + e) = v;
        }
      }
      __syncthreads();
      for (int col = threadIdx.x; col < a.cols; col += Shape::kThreads) {
        float total = 0.0f;
#pragma unroll
        for (int q = 0; q < Shape::kGroups; ++q) total += lds[q * kCols + col];
        dst[col] = total;
      }
    };
    join(dw, to);
    join(db, to + a.cols);
  }
}

// --------------------------------------------------- rows of any length ---

// A workgroup per row, three passes over it (the second and third from the caches).
template <typename T, bool kW32>
__global__ __launch_bounds__(256) void norm_forward_long(const Norm a) {
  constexpr int kV = Piece<T>::kValues;
  __shared__ float lds[16];
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.cols;
    T *out = static_cast<T *>(a.out) + row * a.cols;
    const float x0 = to_float(x[0]);
    float sum[1] = {0.0f};
    for (int col = threadIdx.x * kV; col < a.cols; col += 256 * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, a.cols - col), v);
#pragma unroll
      for (int e = 0; e < kV; ++e) sum[0] += col + e < a.cols ? v[e] - x0 : 0.0f;
    }
    group_sum<256, 1>(sum, lds);
    Centre centre = find_centre(x0, sum[0] * inv);
    float sums[2] = {0.0f, 0.0f};
    for (int col = threadIdx.x * kV; col < a.cols; col += 256 * kV) {
      float v[kV];
      unpack<T>(loose_load<T>(x + col, a.cols - col), v);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        const float c = col + e < a.cols ? v[e] - centre.base - centre.offset : 0.0f;
        sums[0] += c;
        sums[1] += c * c;
      }
    }
    group_sum<256, 2>(sums, lds);
    const float s = correct_centre(centre, sums, inv, a.eps);
    if (a.stats != nullptr && threadIdx.x == 0) keep_centre(a.stats + 2 * row, x0, centre, s);
    for (int col = threadIdx.x * kV; col < a.cols; col += 256 * kV) {
      float v[kV], w[kV], b[kV];
      unpack<T>(loose_load<T>(x + col, a.cols - col), v);
      load_weight<T, kW32>(a.weight, col, a.cols - col, w, 1.0f);
      load_weight<T, kW32>(a.bias, col, a.cols - col, b, 0.0f);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        v[e] = (v[e] - centre.base - centre.offset) * s * w[e] + b[e];
      }
      loose_store(out + col, pack<T>(v), a.cols - col);
    }
  }
}

template <typename T, bool kW32>
__global__ __launch_bounds__(256) void norm_backward_long(const Norm a) {
  constexpr int kV = Piece<T>::kValues;
  __shared__ float lds[16];
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.cols;
    const T *g = static_cast<const T *>(a.grad) + row * a.cols;
    T *dx = static_cast<T *>(a.out) + row * a.cols;
    const float kept_s = a.stats[2 * row + 1], s = fabsf(kept_s);
    const Centre centre = kept_centre(to_float(x[0]), a.stats[2 * row], kept_s);
    float sum[2] = {0.0f, 0.0f};
    for (int pass = 0; pass < 2; ++pass) {
      for (int col = threadIdx.x * kV; col < a.cols; col += 256 * kV) {
        float h[kV], u[kV], w[kV];
        unpack<T>(loose_load<T>(x + col, a.cols - col), h);
        unpack<T>(loose_load<T>(g + col, a.cols - col), u);
        load_weight<T, kW32>(a.weight, col, a.cols - col, w, 1.0f);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          h[e] = (h[e] - centre.base - centre.offset) * s;
          u[e] *= w[e];
          if (pass == 0) {
            sum[0] += col + e < a.cols ? u[e] : 0.0f;
            sum[1] += col + e < a.cols ? u[e] * h[e] : 0.0f;
          } else {
            u[e] = s * (u[e] - sum[0] - h[e] * sum[1]);
          }
        }
        if (pass == 1) loose_store(dx + col, pack<T>(u), a.cols - col);
      }
      if (pass == 0) {
        group_sum<256, 2>(sum, lds);
        sum[0] *= inv;
        sum[1] *= inv;
      }
    }
  }
}

// Column sums of long rows: a thread per piece of columns, blockIdx.y a run of rows.
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_long(const Norm a) {
  constexpr int kV = Piece<T>::kValues;
  const int col = (blockIdx.x * 256 + threadIdx.x) * kV;
  if (col >= a.cols) return;
  const int left = a.cols - col;
  float dw[kV] = {}, db[kV] = {};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T *x = static_cast<const T *>(a.x) + row * a.cols;
    const T *g = static_cast<const T *>(a.grad) + row * a.cols;
    const float kept_s = a.stats[2 * row + 1], s = fabsf(kept_s);
    const Centre centre = kept_centre(to_float(x[0]), a.stats[2 * row], kept_s);
    float h[kV], u[kV];
    unpack<T>(loose_load<T>(x + col, left), h);
    unpack<T>(loose_load<T>(g + col, left), u);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      dw[e] += u[e] * ((h[e] - centre.base - centre.offset) * s);
      db[e] += u[e];
    }
  }
  float *to = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    if (e < left) {
      to[col + e] = dw[e];
      to[a.cols + col + e] = db[e];
    }
  }
}

// The workgroups' rows of sums, added in order: 16 columns by 16 runs of rows a
// workgroup, runs joined in LDS.
template <typename W>
__global__ __launch_bounds__(256) void norm_sum_columns(const float *partial, int parts, int cols,
                                                        W *dw, W *db) {
  __shared__ float lds[16][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + x;
  float total = 0.0f;
  if (col < 2 * cols) {
    const float *src = partial + col;
    const int64_t ld = 2 * static_cast<int64_t>(cols);
    int p = y;
    for (; p + 7 * 16 < parts; p += 8 * 16) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = src[(p + 16 * e) * ld];
#pragma unroll
      for (int e = 0; e < 8; ++e) total += v[e];
    }
    for (; p < parts; p += 16) total += src[p * ld];
  }
  lds[y][x] = total;
  __syncthreads();
  if (y == 0 && col < 2 * cols) {
    total = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) total += lds[e][x];
    if (col < cols) {
      if (dw != nullptr) dw[col] = from_float<W>(total);
    } else if (db != nullptr) {
      db[col - cols] = from_float<W>(total);
    }
  }
}

}  // namespace dense
