// The end of a block of an encoder or decoder layer and the start of the next
// (include/muspace_layer.h):
//
//   y      = post_norm(block), or the block's output itself
//   stream = residual_scale residual + gate dropout(y)
//   output = norm(stream)
//
// and its gradients: with h = norm's unit row, s its factor and g = d output,
//   u  = g w;  ds = d stream + s (u - mean(u) - h mean(u h))
//   d residual = residual_scale ds;  dw = sum of g h, db = sum of g
//   dt = ds kept / (1 - p);  d gate = sum of dt y;  dy = dt gate
//   d block = dy, or the post norm's s' (v - mean(v) - h' mean(v h')), v = dy w'
// The rms norm is the same without means. Memory-bound: each tensor is read and written
// once, rows in registers over the reductions as in layer norm (layer_norm_kernels.hpp,
// whose statistics these are); the dropout's mask is computed in both directions
// (dropout_device.hpp).
//
// `output` is the norm of the sum in float32, before it is rounded into the stream. In
// 16-bit types the backward therefore sums the block and the residual again, rather than
// read the stream: from the stored stream, h would carry its rounding, and the norm's
// output and the weight's gradient would err by 1.3 to 1.66 times their own rounding. float32
// reads the stream, which is the sum. Kept per norm and row: what is subtracted, in two
// parts (Centre), and s.
#pragma once

#include "dropout_device.hpp"
#include "layer_norm_kernels.hpp"

namespace dense {

enum Norms : int { kNoNorm = -1, kLayerNorm = 0, kRmsNorm = 1 };

constexpr int kSums = 5;  // dw, db, d gate, d post weight, d post bias

struct Residual {
  const void *block, *residual, *weight, *bias, *gate, *post_weight, *post_bias;
  const void *grad_out, *grad_stream;
  const void *stream_in;           // float32's backward
  void *out, *stream;              // forward
  void *d_block, *d_residual;      // backward
  float *stats, *post_stats;       // [rows][4] each: base, offset, s, 0
  float *partial;                  // [workgroups][sums][cols]
  float *row_sums;                 // rows of any length: [rows][2], means of u and u h
  int slot[kSums];                 // a column sum's place in `partial` (-1: not wanted)
  int sums;                        // of them
  int64_t rows;
  int cols;
  float eps, scale;                // residual_scale
  int w32, norm, post;             // weights are float32; Norms
  Drop drop;
};

// a piece of a weight, `none` without one
template <typename T>
__device__ __forceinline__ void load_vector(const void *p, int w32, int col, int left,
                                            float (&w)[Piece<T>::kValues], float none) {
  if (w32) {
    load_weight<T, sizeof(T) == 2>(p, col, left, w, none);
  } else {
    load_weight<T, false>(p, col, left, w, none);
  }
}

// 0 beyond a row's values, so that sums may take whole pieces
template <bool kFull>
__device__ __forceinline__ float inside(float v, int e, int left) {
  return kFull || e < left ? v : 0.0f;
}

// kLanes threads a row, a 16-byte piece each: rows of up to 512 pieces. Short rows share a
// wavefront, long ones take several and join their sums in LDS. A workgroup has 256
// threads, or a row's 512: with 512 for all rows more wavefronts wait at a barrier (20000 x
// 1024 bf16 with a post norm, forward 44 -> 38 us, 20000 x 611 float16 51 -> 40).
constexpr int kMaxLanes = 512;
constexpr int kTeamLds = 2 * (kMaxLanes / kWave);  // floats of a Meeting's turn
constexpr int row_threads(int lanes) { return lanes > 256 ? lanes : 256; }

// Where wavefronts that share rows meet: two turns of LDS, taken one after the other, so
// that a turn's readers are done when its next writers have passed the barrier between, and
// one barrier a meeting is enough.
struct Meeting {
  float *lds;
  int turn;

  __device__ __forceinline__ float *next() {
    turn ^= kTeamLds;
    return lds + turn;
  }
};

// kLanes lanes' sums, the same on all of them (every thread of the workgroup calls it)
template <int kLanes, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], Meeting &meet) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = add_across<8>(add_across<4>(add_across<2>(add_across<1>(v[i]))));
    if constexpr (kLanes >= 32) v[i] = add_across<16>(v[i]);
    if constexpr (kLanes >= 64) v[i] = add_across<32>(v[i]);
  }
  if constexpr (kLanes > kWave) {
    const int wave = threadIdx.x / kWave, first = threadIdx.x / kLanes * (kLanes / kWave);
    float *lds = meet.next();
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < kLanes / kWave; ++u) v[i] += lds[(first + u) * N + i];
    }
  }
}

// a row's first value, on all of its lanes
template <int kLanes>
__device__ __forceinline__ float first_value(float v, Meeting &meet) {
  if constexpr (kLanes <= kWave) {
    return __shfl(v, 0, kLanes);
  } else {
    float *lds = meet.next();
    if (threadIdx.x % kLanes == 0) lds[threadIdx.x / kLanes] = v;
    __syncthreads();
    return lds[threadIdx.x / kLanes];
  }
}

__device__ __forceinline__ void keep_statistics(float *stats, int64_t row, const Centre &c,
                                                float s) {
  reinterpret_cast<f32x4 *>(stats)[row] = f32x4{c.base, c.offset, s, 0.0f};
}

// x without its row's centre, times s; the forward's and the backward's
__device__ __forceinline__ float unit_of(float x, const f32x4 &stats) {
  return (x - stats[0] - stats[1]) * stats[2];
}

// Centre and factor of a row in registers. `v` keeps its values.
template <int kLanes, bool kFull, int kV>
__device__ __forceinline__ float row_statistics(const float (&v)[kV], int cols, int lane, int norm,
                                                float inv, float eps, Meeting &meet,
                                                Centre &centre) {
  float sums[2] = {0.0f, 0.0f};
  centre = Centre{0.0f, 0.0f};
  if (norm == kLayerNorm) {
    const float x0 = first_value<kLanes>(v[0], meet);
    float sum[1] = {0.0f};
    const int left = cols - lane * kV;
#pragma unroll
    for (int e = 0; e < kV; ++e) sum[0] += inside<kFull>(v[e] - x0, e, left);
    team_sum<kLanes, 1>(sum, meet);
    centre = find_centre(x0, sum[0] * inv);
  }
  const int left = cols - lane * kV;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    const float c = inside<kFull>(v[e] - centre.base - centre.offset, e, left);
    sums[0] += c;
    sums[1] += c * c;
  }
  team_sum<kLanes, 2>(sums, meet);
  if (norm == kRmsNorm) return 1.0f / sqrtf(sums[1] * inv + eps);
  return correct_centre(centre, sums, inv, eps);
}

template <typename T, int kLanes, bool kFull, bool kPost>
__global__ __launch_bounds__(row_threads(kLanes)) void residual_forward(const Residual a) {
  constexpr int kGroups = row_threads(kLanes) / kLanes;  // rows at a time
  constexpr int kV = Piece<T>::kValues;
  using Pieces = RowPieces<T, kLanes, 1, kFull>;
  __shared__ float lds[2 * kTeamLds];
  Meeting meet = {lds, 0};
  const int lane = threadIdx.x % kLanes;
  const T *block = static_cast<const T *>(a.block), *residual = static_cast<const T *>(a.residual);
  const float inv = 1.0f / static_cast<float>(a.cols);
  const uint64_t seed = seed_of(a.drop);
  float w[kV], b[kV], gate[kV], pw[kV], pb[kV];
  const int col = lane * kV, left = Pieces::left(a.cols, lane, 0);
  load_vector<T>(a.weight, a.w32, col, left, w, 1.0f);
  load_vector<T>(a.bias, a.w32, col, left, b, 0.0f);
  load_vector<T>(a.gate, a.w32, col, left, gate, 1.0f);
  if constexpr (kPost) {
    load_vector<T>(a.post_weight, a.w32, col, left, pw, 1.0f);
    load_vector<T>(a.post_bias, a.w32, col, left, pb, 0.0f);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kLanes;
  Pieces next_y, next_r;
  next_y.load(block, row, a.rows, a.cols, lane);
  next_r.load(residual, row, a.rows, a.cols, lane);
  // groups of one workgroup walk together: past the last row they sum zeros
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows;
       base += step, row += step) {
    const bool any = row < a.rows;
    float y[kV], v[kV];
    next_y.values(0, a.cols, lane, any, y);
    next_r.values(0, a.cols, lane, any, v);
    next_y.load(block, row + step, a.rows, a.cols, lane);
    next_r.load(residual, row + step, a.rows, a.cols, lane);
    Centre centre;
    if constexpr (kPost) {
      const float s =
          row_statistics<kLanes, kFull>(y, a.cols, lane, a.post, inv, a.eps, meet, centre);
      if (a.post_stats != nullptr && any && lane == 0) {
        keep_statistics(a.post_stats, row, centre, s);
      }
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        y[e] = (y[e] - centre.base - centre.offset) * s * pw[e] + pb[e];
      }
    }
    if (a.drop.on) {
      const uint32_t bits = kept_bits<kV>(a.drop, seed, row * a.cols + col);
#pragma unroll
      for (int e = 0; e < kV; ++e) y[e] = (bits >> e) & 1u ? y[e] * a.drop.scale : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = fmaf(a.scale, v[e], gate[e] * y[e]);
    if (a.stream != nullptr) {
      loose_store(static_cast<T *>(a.stream) + row * a.cols + col, pack<T>(v), any ? left : 0);
    }
    const float s =
        row_statistics<kLanes, kFull>(v, a.cols, lane, a.norm, inv, a.eps, meet, centre);
    if (a.stats != nullptr && any && lane == 0) keep_statistics(a.stats, row, centre, s);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      v[e] = (v[e] - centre.base - centre.offset) * s * w[e] + b[e];
    }
    loose_store(static_cast<T *>(a.out) + row * a.cols + col, pack<T>(v), any ? left : 0);
  }
}

// kBlock: for a post norm or the gate's gradient (float32 reads the block's output for
// these alone).
template <typename T, int kLanes, bool kFull, bool kBlock>
__global__ __launch_bounds__(row_threads(kLanes)) void residual_backward(const Residual a) {
  constexpr int kGroups = row_threads(kLanes) / kLanes;  // rows at a time
  constexpr int kV = Piece<T>::kValues;
  constexpr int kCols = kLanes * kV;
  constexpr int kMine = kBlock ? kSums : 2;
  constexpr bool kSum = sizeof(T) == 2;  // the stream is summed again
  using Pieces = RowPieces<T, kLanes, 1, kFull>;
  constexpr int kJoin = kGroups * kCols, kMeet = 2 * kTeamLds;
  __shared__ float lds[kGroups > 1 && kJoin > kMeet ? kJoin : kMeet];
  Meeting meet = {lds, 0};
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const T *stream = static_cast<const T *>(kSum ? a.residual : a.stream_in);
  const T *block = static_cast<const T *>(a.block);
  const T *go = static_cast<const T *>(a.grad_out), *gs = static_cast<const T *>(a.grad_stream);
  const float inv = 1.0f / static_cast<float>(a.cols);
  const uint64_t seed = seed_of(a.drop);
  float w[kV], gate[kV], pw[kV], pb[kV];
  const int col = lane * kV, left = Pieces::left(a.cols, lane, 0);
  load_vector<T>(a.weight, a.w32, col, left, w, 1.0f);
  load_vector<T>(a.gate, a.w32, col, left, gate, 1.0f);
  if constexpr (kBlock) {
    load_vector<T>(a.post_weight, a.w32, col, left, pw, 1.0f);
    load_vector<T>(a.post_bias, a.w32, col, left, pb, 0.0f);
  }
  float sum[kMine][kV] = {};
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  Pieces n_stream, n_go = {}, n_gs = {}, n_block;
  f32x4 n_stats, n_post = {0.0f, 0.0f, 1.0f, 0.0f};  // without a post norm: the block's output
  auto fetch = [&](int64_t r) {
    const int64_t at = min(r, a.rows - 1);
    n_stream.load(stream, r, a.rows, a.cols, lane);
    if (go != nullptr) n_go.load(go, r, a.rows, a.cols, lane);
    if (gs != nullptr) n_gs.load(gs, r, a.rows, a.cols, lane);
    n_stats = reinterpret_cast<const f32x4 *>(a.stats)[at];
    if constexpr (kBlock || kSum) n_block.load(block, r, a.rows, a.cols, lane);
    if constexpr (kBlock) {
      if (a.post != kNoNorm) n_post = reinterpret_cast<const f32x4 *>(a.post_stats)[at];
    }
  };
  fetch(row);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < a.rows;
       base += step, row += step) {
    const bool any = row < a.rows;
    const int64_t at = row * a.cols + col;
    float h[kV], u[kV], ds[kV], unit[kV];
    n_stream.values(0, a.cols, lane, any, h);
    n_go.values(0, a.cols, lane, any && go != nullptr, u);
    n_gs.values(0, a.cols, lane, any && gs != nullptr, ds);
    if constexpr (kBlock || kSum) n_block.values(0, a.cols, lane, any, unit);
    const f32x4 stats = n_stats, post = n_post;
    fetch(row + step);
    // (no bits past the last row)
    const uint32_t bits = !any ? 0u : a.drop.on ? kept_bits<kV>(a.drop, seed, at) : ~0u;
    float along[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      if constexpr (kBlock) unit[e] = inside<kFull>(unit_of(unit[e], post), e, left);
      if constexpr (kSum) {
        // the operations of the forward
        float y = unit[e];
        if constexpr (kBlock) y = y * pw[e] + pb[e];
        y = (bits >> e) & 1u ? y * a.drop.scale : 0.0f;
        h[e] = fmaf(a.scale, h[e], gate[e] * y);
      }
      h[e] = inside<kFull>(unit_of(h[e], stats), e, left);
      sum[0][e] += u[e] * h[e];
      sum[1][e] += u[e];
      u[e] *= w[e];
      along[0] += u[e];
      along[1] += u[e] * h[e];
    }
    // (without a gradient of the output both are zero, and rows that have no statistics
    // to speak of, of infinities, do not reach the stream's gradient)
    if (go != nullptr) {
      team_sum<kLanes, 2>(along, meet);
      const float mu = a.norm == kLayerNorm ? along[0] * inv : 0.0f, mh = along[1] * inv;
#pragma unroll
      for (int e = 0; e < kV; ++e) ds[e] += stats[2] * (u[e] - mu - h[e] * mh);
    }
    if (a.d_residual != nullptr) {
      float r[kV];
#pragma unroll
      for (int e = 0; e < kV; ++e) r[e] = a.scale * ds[e];
      loose_store(static_cast<T *>(a.d_residual) + at, pack<T>(r), any ? left : 0);
    }
    float across[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const bool kept = (bits >> e) & 1u;
      const float dt = kept ? ds[e] * a.drop.scale : 0.0f;
      float dy = kept ? dt * gate[e] : 0.0f;
      if constexpr (kBlock) {
        dy = inside<kFull>(dy, e, left);
        const float y = unit[e] * pw[e] + pb[e];
        sum[2][e] += kept && (kFull || e < left) ? dt * y : 0.0f;
        sum[3][e] += dy * unit[e];
        sum[4][e] += dy;
        dy *= pw[e];
        across[0] += dy;
        across[1] += dy * unit[e];
      }
      ds[e] = dy;
    }
    if (a.d_block == nullptr) continue;
    if constexpr (kBlock) {
      if (a.post != kNoNorm) {
        team_sum<kLanes, 2>(across, meet);
        const float mv = a.post == kLayerNorm ? across[0] * inv : 0.0f, mh = across[1] * inv;
#pragma unroll
        for (int e = 0; e < kV; ++e) ds[e] = post[2] * (ds[e] - mv - unit[e] * mh);
      }
    }
    loose_store(static_cast<T *>(a.d_block) + at, pack<T>(ds), any ? left : 0);
  }
  if (a.partial == nullptr) return;
  float *to = a.partial + static_cast<int64_t>(blockIdx.x) * a.sums * a.cols;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    if (a.slot[k] < 0) continue;
    float *dst = to + static_cast<int64_t>(a.slot[k]) * a.cols;
    if constexpr (kGroups == 1) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        if (col + e < a.cols) dst[col + e] = sum[k][e];
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const f32x4 v = {sum[k][e], sum[k][e + 1], sum[k][e + 2], sum[k][e + 3]};
        *reinterpret_cast<f32x4 *>(lds + group * kCols + col + e) = v;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += row_threads(kLanes)) {
        float total = 0.0f;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) total += lds[q * kCols + c];
        dst[c] = total;
      }
    }
  }
}

// --------------------------------------------------- rows of any length ---

// A workgroup per row, its values computed from memory in every pass over it, the dropout's mask
// among them: forward two passes (rms one) for the statistics and one that writes, as many as the
// first again for a post norm; backward two, three with a post norm, and one for the columns' sums.
// Layer norm, dropout, us of a forward and of a backward: 16384 x 4096 bf16, the longest rows in
// registers, 108 and 171 (4.9 and 4.7 TB/s), 16384 x 5120 374 and 956, x 8192 508 and 1140; float32 x
// 2048 100 and 138, x 5120 431 and 560, x 8192 679 and 786. The 16-bit backward is the slowest: it
// sums block and residual again in each pass.
constexpr int kLongThreads = 256;

template <typename T, typename F>
__device__ __forceinline__ void over_row(int cols, F &&f) {
  constexpr int kV = Piece<T>::kValues;
  for (int col = threadIdx.x * kV; col < cols; col += kLongThreads * kV) f(col, cols - col);
}

// Centre and factor of a row whose pieces `values(col, left, v)` gives.
template <typename T, typename F>
__device__ __forceinline__ float long_statistics(int cols, float x0, int norm, float inv, float eps,
                                                 Meeting &meet, Centre &centre, F &&values) {
  constexpr int kV = Piece<T>::kValues;
  float sums[2] = {0.0f, 0.0f};
  centre = Centre{0.0f, 0.0f};
  if (norm == kLayerNorm) {
    float sum[1] = {0.0f};
    over_row<T>(cols, [&](int col, int left) {
      float v[kV];
      values(col, left, v);
#pragma unroll
      for (int e = 0; e < kV; ++e) sum[0] += e < left ? v[e] - x0 : 0.0f;
    });
    team_sum<kLongThreads, 1>(sum, meet);
    centre = find_centre(x0, sum[0] * inv);
  }
  over_row<T>(cols, [&](int col, int left) {
    float v[kV];
    values(col, left, v);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const float c = e < left ? v[e] - centre.base - centre.offset : 0.0f;
      sums[0] += c;
      sums[1] += c * c;
    }
  });
  team_sum<kLongThreads, 2>(sums, meet);
  if (norm == kRmsNorm) return 1.0f / sqrtf(sums[1] * inv + eps);
  return correct_centre(centre, sums, inv, eps);
}

// A row's pieces, forward and backward.
template <typename T>
struct LongRow {
  static constexpr int kV = Piece<T>::kValues;
  f32x4 stats, post;  // without a post norm: the block's output is its own unit row

  // the post norm's unit row, and what the dropout is taken of
  __device__ __forceinline__ void block(const Residual &a, int64_t row, int col, int left,
                                        float (&unit)[kV], float (&y)[kV]) const {
    unpack<T>(loose_load<T>(static_cast<const T *>(a.block) + row * a.cols + col,
                            a.block != nullptr ? left : 0), unit);
    float pw[kV], pb[kV];
    load_vector<T>(a.post_weight, a.w32, col, left, pw, 1.0f);
    load_vector<T>(a.post_bias, a.w32, col, left, pb, 0.0f);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      unit[e] = e < left ? unit_of(unit[e], post) : 0.0f;
      y[e] = unit[e] * pw[e] + pb[e];
    }
  }
  // the stream, summed
  __device__ __forceinline__ void stream(const Residual &a, uint64_t seed, int64_t row, int col,
                                         int left, float (&v)[kV]) const {
    const int64_t at = row * a.cols + col;
    float unit[kV], y[kV], gate[kV];
    block(a, row, col, left, unit, y);
    unpack<T>(loose_load<T>(static_cast<const T *>(a.residual) + at, left), v);
    load_vector<T>(a.gate, a.w32, col, left, gate, 1.0f);
    const uint32_t bits = a.drop.on ? kept_bits<kV>(a.drop, seed, at) : ~0u;
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      y[e] = (bits >> e) & 1u ? y[e] * a.drop.scale : 0.0f;
      v[e] = fmaf(a.scale, v[e], gate[e] * y[e]);
    }
  }
  // backward: the statistics of a row
  __device__ __forceinline__ void open(const Residual &a, int64_t row) {
    stats = reinterpret_cast<const f32x4 *>(a.stats)[row];
    post = f32x4{0.0f, 0.0f, 1.0f, 0.0f};
    if (a.post != kNoNorm) post = reinterpret_cast<const f32x4 *>(a.post_stats)[row];
  }
  // h and g of the norm
  __device__ __forceinline__ void unit(const Residual &a, uint64_t seed, int64_t row, int col,
                                       int left, float (&h)[kV], float (&g)[kV]) const {
    const int64_t at = row * a.cols + col;
    if constexpr (sizeof(T) == 2) {
      stream(a, seed, row, col, left, h);
    } else {
      unpack<T>(loose_load<T>(static_cast<const T *>(a.stream_in) + at, left), h);
    }
    unpack<T>(loose_load<T>(static_cast<const T *>(a.grad_out) + at,
                            a.grad_out != nullptr ? left : 0), g);
#pragma unroll
    for (int e = 0; e < kV; ++e) h[e] = e < left ? unit_of(h[e], stats) : 0.0f;
  }
  // the stream's gradient, given the means of u and u h
  __device__ __forceinline__ void stream_grad(const Residual &a, int64_t row, int col, int left,
                                              float mu, float mh, const float (&h)[kV],
                                              const float (&g)[kV], float (&ds)[kV]) const {
    const int64_t at = row * a.cols + col;
    unpack<T>(loose_load<T>(static_cast<const T *>(a.grad_stream) + at,
                            a.grad_stream != nullptr ? left : 0), ds);
    if (a.grad_out == nullptr) return;
    float w[kV];
    load_vector<T>(a.weight, a.w32, col, left, w, 1.0f);
#pragma unroll
    for (int e = 0; e < kV; ++e) ds[e] += stats[2] * (g[e] * w[e] - mu - h[e] * mh);
  }
  // from ds: dy, the post norm's unit row (or the block's output) and the gate's term
  __device__ __forceinline__ void block_grad(const Residual &a, uint64_t seed, int64_t row, int col,
                                             int left, const float (&ds)[kV], float (&dy)[kV],
                                             float (&unit)[kV], float (&gated)[kV]) const {
    const uint32_t bits = a.drop.on ? kept_bits<kV>(a.drop, seed, row * a.cols + col) : ~0u;
    float gate[kV], y[kV];
    load_vector<T>(a.gate, a.w32, col, left, gate, 1.0f);
    block(a, row, col, left, unit, y);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const bool kept = ((bits >> e) & 1u) && e < left;
      const float dt = kept ? ds[e] * a.drop.scale : 0.0f;
      dy[e] = kept ? dt * gate[e] : 0.0f;
      gated[e] = kept ? dt * y[e] : 0.0f;
    }
  }
};

template <typename T>
__global__ __launch_bounds__(kLongThreads) void residual_forward_long(const Residual a) {
  constexpr int kV = Piece<T>::kValues;
  __shared__ float lds[2 * kTeamLds];
  Meeting meet = {lds, 0};
  const float inv = 1.0f / static_cast<float>(a.cols);
  const uint64_t seed = seed_of(a.drop);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *block = static_cast<const T *>(a.block) + row * a.cols;
    LongRow<T> r;
    r.post = f32x4{0.0f, 0.0f, 1.0f, 0.0f};
    Centre centre;
    if (a.post != kNoNorm) {
      const float s = long_statistics<T>(a.cols, to_float(block[0]), a.post, inv, a.eps, meet,
                                         centre, [&](int col, int left, float(&v)[kV]) {
                                           unpack<T>(loose_load<T>(block + col, left), v);
                                         });
      r.post = f32x4{centre.base, centre.offset, s, 0.0f};
      if (a.post_stats != nullptr && threadIdx.x == 0) {
        keep_statistics(a.post_stats, row, centre, s);
      }
    }
    auto stream = [&](int col, int left, float(&v)[kV]) { r.stream(a, seed, row, col, left, v); };
    float v0[kV] = {};
    if (threadIdx.x == 0) stream(0, a.cols, v0);
    const float x0 = first_value<kLongThreads>(v0[0], meet);
    const float s = long_statistics<T>(a.cols, x0, a.norm, inv, a.eps, meet, centre, stream);
    if (a.stats != nullptr && threadIdx.x == 0) keep_statistics(a.stats, row, centre, s);
    over_row<T>(a.cols, [&](int col, int left) {
      float v[kV], w[kV], b[kV];
      stream(col, left, v);
      if (a.stream != nullptr) {
        loose_store(static_cast<T *>(a.stream) + row * a.cols + col, pack<T>(v), left);
      }
      load_vector<T>(a.weight, a.w32, col, left, w, 1.0f);
      load_vector<T>(a.bias, a.w32, col, left, b, 0.0f);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        v[e] = (v[e] - centre.base - centre.offset) * s * w[e] + b[e];
      }
      loose_store(static_cast<T *>(a.out) + row * a.cols + col, pack<T>(v), left);
    });
  }
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void residual_backward_long(const Residual a) {
  constexpr int kV = Piece<T>::kValues;
  __shared__ float lds[2 * kTeamLds];
  Meeting meet = {lds, 0};
  const float inv = 1.0f / static_cast<float>(a.cols);
  const uint64_t seed = seed_of(a.drop);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    LongRow<T> r;
    r.open(a, row);
    float mean[2] = {0.0f, 0.0f}, mean_p[2] = {0.0f, 0.0f};
    if (a.grad_out != nullptr) {
      over_row<T>(a.cols, [&](int col, int left) {
        float h[kV], g[kV], w[kV];
        r.unit(a, seed, row, col, left, h, g);
        load_vector<T>(a.weight, a.w32, col, left, w, 1.0f);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          mean[0] += g[e] * w[e];
          mean[1] += g[e] * w[e] * h[e];
        }
      });
      team_sum<kLongThreads, 2>(mean, meet);
      mean[0] = a.norm == kLayerNorm ? mean[0] * inv : 0.0f;
      mean[1] *= inv;
    }
    if (a.row_sums != nullptr && threadIdx.x == 0) {
      a.row_sums[2 * row] = mean[0];
      a.row_sums[2 * row + 1] = mean[1];
    }
    auto block_grad = [&](int col, int left, float(&ds)[kV], float(&dy)[kV], float(&unit)[kV]) {
      float h[kV], g[kV], gated[kV];
      r.unit(a, seed, row, col, left, h, g);
      r.stream_grad(a, row, col, left, mean[0], mean[1], h, g, ds);
      r.block_grad(a, seed, row, col, left, ds, dy, unit, gated);
      if (a.post != kNoNorm) {
        float pw[kV];
        load_vector<T>(a.post_weight, a.w32, col, left, pw, 1.0f);
#pragma unroll
        for (int e = 0; e < kV; ++e) dy[e] *= pw[e];
      }
    };
    if (a.post != kNoNorm && a.d_block != nullptr) {
      over_row<T>(a.cols, [&](int col, int left) {
        float ds[kV], dy[kV], unit[kV];
        block_grad(col, left, ds, dy, unit);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          mean_p[0] += dy[e];
          mean_p[1] += dy[e] * unit[e];
        }
      });
      team_sum<kLongThreads, 2>(mean_p, meet);
      mean_p[0] = a.post == kLayerNorm ? mean_p[0] * inv : 0.0f;
      mean_p[1] *= inv;
    }
    over_row<T>(a.cols, [&](int col, int left) {
      float ds[kV], dy[kV], unit[kV];
      block_grad(col, left, ds, dy, unit);
      const int64_t at = row * a.cols + col;
      if (a.d_block != nullptr) {
        if (a.post != kNoNorm) {
#pragma unroll
          for (int e = 0; e < kV; ++e) dy[e] = r.post[2] * (dy[e] - mean_p[0] - unit[e] * mean_p[1]);
        }
        loose_store(static_cast<T *>(a.d_block) + at, pack<T>(dy), left);
      }
      if (a.d_residual != nullptr) {
#pragma unroll
        for (int e = 0; e < kV; ++e) ds[e] *= a.scale;
        loose_store(static_cast<T *>(a.d_residual) + at, pack<T>(ds), left);
      }
    });
  }
}

// Column sums of long rows, after residual_backward_long: a thread per piece of columns,
// blockIdx.y a run of rows.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void residual_columns_long(const Residual a) {
  constexpr int kV = Piece<T>::kValues;
  const int col = (blockIdx.x * kLongThreads + threadIdx.x) * kV;
  if (col >= a.cols) return;
  const int left = a.cols - col;
  const uint64_t seed = seed_of(a.drop);
  float sum[kSums][kV] = {};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    LongRow<T> r;
    r.open(a, row);
    float h[kV], g[kV];
    r.unit(a, seed, row, col, left, h, g);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      sum[0][e] += g[e] * h[e];
      sum[1][e] += g[e];
    }
    if (a.slot[2] < 0 && a.slot[3] < 0 && a.slot[4] < 0) continue;
    float ds[kV], dy[kV], unit[kV], gated[kV];
    r.stream_grad(a, row, col, left, a.row_sums[2 * row], a.row_sums[2 * row + 1], h, g, ds);
    r.block_grad(a, seed, row, col, left, ds, dy, unit, gated);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      sum[2][e] += gated[e];
      sum[3][e] += dy[e] * unit[e];
      sum[4][e] += dy[e];
    }
  }
  float *to = a.partial + static_cast<int64_t>(blockIdx.y) * a.sums * a.cols;
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    if (a.slot[k] < 0) continue;
    float *dst = to + static_cast<int64_t>(a.slot[k]) * a.cols + col;
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      if (e < left) dst[e] = sum[k][e];
    }
  }
}

struct SumTargets {
  void *to[kSums];  // by place in `partial`
};

// The workgroups' rows of sums, added in order.
template <typename W>
__global__ __launch_bounds__(256) void residual_sum_columns(const float *partial, int parts,
                                                            int cols, int sums, SumTargets out) {
  const int64_t ld = static_cast<int64_t>(sums) * cols;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x & 15);
  const float total = add_rows(partial + col, col < ld ? parts : 0, ld);
  if (threadIdx.x >= 16 || col >= ld) return;
  const int k = static_cast<int>(col / cols);
  static_cast<W *>(out.to[k])[col - static_cast<int64_t>(k) * cols] = from_float<W>(total);
}

}  // namespace dense
