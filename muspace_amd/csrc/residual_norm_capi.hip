// C-ABI entry points of dropout and the residual norm (declared in
// include/muspace_layer.h). Plans are functions of sizes and types only.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/muspace_layer.h"
#include "capi_errors.hpp"
#include "residual_norm_kernels.hpp"

namespace {

using capi::check_launch;
using capi::fail;
using capi::ok;
using dense::Drop;
using dense::Residual;

constexpr int64_t kMaxCols = 1 << 20;
constexpr int64_t kMaxRows = INT_MAX - 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename F>
void by_type(int dtype, F &&f) {
  if (dtype == 0) {
    f(float{});
  } else if (dtype == 1) {
    f(__half{});
  } else {
    f(dense::bf16_t{});
  }
}

// A probability's border: words below p 2^32, to the nearest, are dropped. (p under
// 2^-33 drops nothing.)
Drop drop_of(double p, uint64_t seed, const int64_t *device_seed, uint64_t offset) {
  Drop d = {};
  const double border = std::nearbyint(p * 4294967296.0);
  d.seed = seed;
  d.device_seed = device_seed;
  d.offset = offset;
  d.on = border > 0.0;
  d.last = d.on ? static_cast<uint32_t>(static_cast<uint64_t>(border) - 1) : 0;
  d.scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f;
  return d;
}

int validate_p(const char *fn, double p, const int64_t *device_seed) {
  if (!(p >= 0.0 && p <= 1.0)) {
    return fail(MUSPACE_EINVAL, "%s: the probability must be in [0, 1], got %g", fn, p);
  }
  if (reinterpret_cast<uintptr_t>(device_seed) % 8 != 0) {
    return fail(MUSPACE_EINVAL, "%s: the seed must be 8-byte aligned", fn);
  }
  return MUSPACE_OK;
}

int validate(const char *fn, int dtype, int weight_dtype, int64_t rows, int64_t cols, int norm,
             int post_norm) {
  if (dtype < 0 || dtype > 2) {
    return fail(MUSPACE_EINVAL, "%s: tensors must be float32, float16 or bfloat16", fn);
  }
  if (weight_dtype != dtype && weight_dtype != 0) {
    return fail(MUSPACE_EINVAL, "%s: weights must be float32 or of the tensors' type", fn);
  }
  if (rows < 0 || cols < 0) {
    return fail(MUSPACE_EINVAL, "%s: invalid dims rows=%lld cols=%lld", fn, (long long)rows,
                (long long)cols);
  }
  if (norm != dense::kLayerNorm && norm != dense::kRmsNorm) {
    return fail(MUSPACE_EINVAL, "%s: norm must be 0 (layer) or 1 (rms), got %d", fn, norm);
  }
  if (post_norm < dense::kNoNorm || post_norm > dense::kRmsNorm) {
    return fail(MUSPACE_EINVAL, "%s: post_norm must be -1 (none), 0 (layer) or 1 (rms), got %d", fn,
                post_norm);
  }
  if (rows > kMaxRows || cols > kMaxCols) {
    return fail(MUSPACE_ERANGE, "%s: dims exceed the kernels' 32-bit indexing", fn);
  }
  return ok();
}

// Lanes that share a row, a 16-byte piece each: the least that hold it; 0: longer rows.
int plan_lanes(int dtype, int64_t cols) {
  const int64_t n = ceil_div(cols, dtype == 0 ? 4 : 8);
  for (int lanes = 16; lanes <= dense::kMaxLanes; lanes *= 2) {
    if (n <= lanes) return lanes;
  }
  return 0;
}

int forward_blocks(int lanes, int64_t rows) {
  const int64_t want = ceil_div(rows, lanes == 0 ? 1 : dense::row_threads(lanes) / lanes);
  return static_cast<int>(want < 4096 ? want : 4096);
}

// Workgroups of the backward; each leaves a row of every column sum.
int backward_blocks(int lanes, int64_t rows) {
  if (lanes == 0) return static_cast<int>(rows < 64 ? rows : 64);
  const int64_t want = ceil_div(rows, dense::row_threads(lanes) / lanes);
  return static_cast<int>(want < 512 ? want : 512);
}

// the means of long rows, for the column sums
size_t row_bytes(int lanes, int64_t rows) {
  return lanes == 0 ? (static_cast<size_t>(rows) * 8 + 15) & ~size_t{15} : 0;
}

template <typename T, int kLanes, bool kFull, bool kBackward>
void launch_rows(const Residual &a, int blocks, bool block, hipStream_t st) {
  constexpr int kThreads = dense::row_threads(kLanes);
  if constexpr (kBackward) {
    if (block) {
      dense::residual_backward<T, kLanes, kFull, true><<<blocks, kThreads, 0, st>>>(a);
    } else {
      dense::residual_backward<T, kLanes, kFull, false><<<blocks, kThreads, 0, st>>>(a);
    }
  } else if (block) {
    dense::residual_forward<T, kLanes, kFull, true><<<blocks, kThreads, 0, st>>>(a);
  } else {
    dense::residual_forward<T, kLanes, kFull, false><<<blocks, kThreads, 0, st>>>(a);
  }
}

// `block`: forward: a post norm; backward: or the gate's gradient
template <typename T, bool kBackward, int kLanes = 16>
void launch(int lanes, const Residual &a, int blocks, bool block, hipStream_t st) {
  if (lanes != kLanes) {
    if constexpr (kLanes < dense::kMaxLanes) {
      launch<T, kBackward, kLanes * 2>(lanes, a, blocks, block, st);
    }
  } else if (a.cols == kLanes * dense::Piece<T>::kValues) {
    launch_rows<T, kLanes, true, kBackward>(a, blocks, block, st);
  } else {
    launch_rows<T, kLanes, false, kBackward>(a, blocks, block, st);
  }
}

}  // namespace

extern "C" {

int dropout_forward(const void *x, int dtype, const void *residual, void *output, int64_t count,
                    double p, uint64_t seed, const int64_t *device_seed, uint64_t offset,
                    void *stream) {
  const char *fn = "dropout_forward";
  if (dtype < 0 || dtype > 2) {
    return fail(MUSPACE_EINVAL, "%s: tensors must be float32, float16 or bfloat16", fn);
  }
  const int rc = validate_p(fn, p, device_seed);
  if (rc != MUSPACE_OK) return rc;
  if (count < 0) return fail(MUSPACE_EINVAL, "%s: invalid count %lld", fn, (long long)count);
  if (count == 0) return ok();
  if (x == nullptr || output == nullptr) return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  const Drop d = drop_of(p, seed, device_seed, offset);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t want = ceil_div(ceil_div(count, dense::Piece<T>::kValues), dense::kThreads);
    dense::dropout_elements<T>
        <<<static_cast<int>(want < 2048 ? want : 2048), dense::kThreads, 0, st>>>(
            static_cast<const T *>(x), static_cast<const T *>(residual), static_cast<T *>(output),
            count, d);
  });
  return check_launch(fn);
}

int residual_norm_forward(const void *block, int dtype, const void *residual, const void *weight,
                          const void *bias, const void *gate, const void *post_weight,
                          const void *post_bias, int weight_dtype, void *output,
                          void *stream_values, float *statistics, float *post_statistics,
                          int64_t rows, int64_t cols, int norm, int post_norm, float eps,
                          float residual_scale, double p, uint64_t seed,
                          const int64_t *device_seed, uint64_t offset, void *stream) {
  const char *fn = "residual_norm_forward";
  int rc = validate(fn, dtype, weight_dtype, rows, cols, norm, post_norm);
  if (rc == MUSPACE_OK) rc = validate_p(fn, p, device_seed);
  if (rc != MUSPACE_OK) return rc;
  if (rows == 0 || cols == 0) return ok();
  if (block == nullptr || residual == nullptr || output == nullptr) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  if (!aligned16(statistics) || !aligned16(post_statistics)) {
    return fail(MUSPACE_EINVAL, "%s: statistics must be 16-byte aligned", fn);
  }
  Residual a = {};
  a.block = block;
  a.residual = residual;
  a.weight = weight;
  a.bias = bias;
  a.gate = gate;
  a.post_weight = post_weight;
  a.post_bias = post_bias;
  a.out = output;
  a.stream = stream_values;
  a.stats = statistics;
  a.post_stats = post_statistics;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.eps = eps;
  a.scale = residual_scale;
  a.w32 = weight_dtype == 0;
  a.norm = norm;
  a.post = post_norm;
  a.drop = drop_of(p, seed, device_seed, offset);
  const int lanes = plan_lanes(dtype, cols);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (lanes == 0) {
      dense::residual_forward_long<T>
          <<<static_cast<int>(rows < 2048 ? rows : 2048), dense::kLongThreads, 0, st>>>(a);
    } else {
      launch<T, false>(lanes, a, forward_blocks(lanes, rows), post_norm != dense::kNoNorm, st);
    }
  });
  return check_launch(fn);
}

size_t residual_norm_backward_workspace_size(int dtype, int64_t rows, int64_t cols, int sums) {
  if (validate("residual_norm_backward_workspace_size", dtype, dtype, rows, cols, 0, 0) !=
          MUSPACE_OK ||
      sums <= 0) {
    return 0;
  }
  const int lanes = plan_lanes(dtype, cols);
  return static_cast<size_t>(backward_blocks(lanes, rows)) * sums * cols * 4 +
         row_bytes(lanes, rows);
}

int residual_norm_backward(const void *grad_output, const void *grad_stream, int dtype,
                           const void *block, const void *residual, const void *stream_values,
                           const void *weight, const void *gate, const void *post_weight,
                           const void *post_bias, int weight_dtype, const float *statistics, const float *post_statistics,
                           void *grad_block, void *grad_residual, void *grad_weight,
                           void *grad_bias, void *grad_gate, void *grad_post_weight,
                           void *grad_post_bias, int64_t rows, int64_t cols, int norm,
                           int post_norm, float residual_scale, double p, uint64_t seed,
                           const int64_t *device_seed, uint64_t offset, void *workspace,
                           size_t workspace_bytes, void *stream) {
  const char *fn = "residual_norm_backward";
  int rc = validate(fn, dtype, weight_dtype, rows, cols, norm, post_norm);
  if (rc == MUSPACE_OK) rc = validate_p(fn, p, device_seed);
  if (rc != MUSPACE_OK) return rc;
  Residual a = {};
  void *const wanted[dense::kSums] = {grad_weight, grad_bias, grad_gate, grad_post_weight,
                                      grad_post_bias};
  dense::SumTargets targets = {};
  for (int k = 0; k < dense::kSums; ++k) {
    a.slot[k] = wanted[k] != nullptr ? a.sums : -1;
    if (wanted[k] != nullptr) targets.to[a.sums++] = wanted[k];
  }
  if (cols == 0 || (grad_block == nullptr && grad_residual == nullptr && a.sums == 0)) return ok();
  if (post_norm == dense::kNoNorm && (grad_post_weight != nullptr || grad_post_bias != nullptr)) {
    return fail(MUSPACE_EINVAL, "%s: gradients of a post norm without one", fn);
  }
  // 16-bit types sum block and residual again; float32 reads the stream, and the block's
  // output for the post norm and the gate's gradient
  const bool of_block = post_norm != dense::kNoNorm || grad_gate != nullptr;
  const bool reads_block = of_block || dtype != 0;
  if (rows > 0 &&
      ((dtype == 0 ? stream_values : residual) == nullptr || statistics == nullptr ||
       (reads_block && block == nullptr) ||
       (post_norm != dense::kNoNorm && post_statistics == nullptr))) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  if (!aligned16(statistics) || !aligned16(post_statistics)) {
    return fail(MUSPACE_EINVAL, "%s: statistics must be 16-byte aligned", fn);
  }
  const size_t need =
      a.sums > 0 ? residual_norm_backward_workspace_size(dtype, rows, cols, a.sums) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
    return fail(MUSPACE_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", fn,
                need, workspace == nullptr ? size_t{0} : workspace_bytes);
  }
  const int lanes = plan_lanes(dtype, cols);
  a.block = reads_block ? block : nullptr;
  a.residual = residual;
  a.stream_in = stream_values;
  a.grad_out = grad_output;
  a.grad_stream = grad_stream;
  a.weight = weight;
  a.gate = gate;
  a.post_weight = post_weight;
  a.post_bias = post_bias;
  a.d_block = grad_block;
  a.d_residual = grad_residual;
  a.stats = const_cast<float *>(statistics);
  a.post_stats = const_cast<float *>(post_statistics);
  if (a.sums > 0) {
    if (lanes == 0) a.row_sums = static_cast<float *>(workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + row_bytes(lanes, rows));
  }
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.scale = residual_scale;
  a.w32 = weight_dtype == 0;
  a.norm = norm;
  a.post = post_norm;
  a.drop = drop_of(p, seed, device_seed, offset);
  const int blocks = backward_blocks(lanes, rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (rows > 0) {
      if (lanes != 0) {
        launch<T, true>(lanes, a, blocks, of_block, st);
      } else {
        dense::residual_backward_long<T>
            <<<static_cast<int>(rows < 2048 ? rows : 2048), dense::kLongThreads, 0, st>>>(a);
        if (a.sums > 0) {
          const int across =
              static_cast<int>(ceil_div(cols, dense::kLongThreads * dense::Piece<T>::kValues));
          dense::residual_columns_long<T>
              <<<dim3(across, blocks), dense::kLongThreads, 0, st>>>(a);
        }
      }
    }
    if (a.sums > 0) {
      const int sum_blocks = static_cast<int>(ceil_div(a.sums * cols, 16));
      if (weight_dtype == 0) {
        dense::residual_sum_columns<float>
            <<<sum_blocks, 256, 0, st>>>(a.partial, blocks, a.cols, a.sums, targets);
      } else {
        dense::residual_sum_columns<T>
            <<<sum_blocks, 256, 0, st>>>(a.partial, blocks, a.cols, a.sums, targets);
      }
    }
  });
  return check_launch(fn);
}

}  // extern "C"
