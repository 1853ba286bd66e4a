// C-ABI entry points of layer norm (declared in include/muspace_layer.h).
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "../../include/muspace_layer.h"
#include "capi_errors.hpp"
#include "layer_norm_kernels.hpp"

namespace {

using capi::check_launch;
using capi::fail;
using capi::ok;
using dense::Norm;

constexpr int64_t kMaxCols = 1 << 20;
constexpr int64_t kMaxRows = INT_MAX - 256;

int validate(const char *fn, int dtype, int weight_dtype, int64_t rows, int64_t cols) {
  if (dtype < 0 || dtype > 2) {
    return fail(MUSPACE_EINVAL, "%s: tensors must be float32, float16 or bfloat16", fn);
  }
  if (weight_dtype != dtype && weight_dtype != 0) {
    return fail(MUSPACE_EINVAL, "%s: weight and bias must be float32 or of the tensors' type", fn);
  }
  if (rows < 0 || cols < 0) {
    return fail(MUSPACE_EINVAL, "%s: invalid dims rows=%lld cols=%lld", fn, (long long)rows,
                (long long)cols);
  }
  if (rows > kMaxRows || cols > kMaxCols) {
    return fail(MUSPACE_ERANGE, "%s: dims exceed the kernels' 32-bit indexing", fn);
  }
  return ok();
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Lanes that share a row and pieces per lane; lanes 0: rows of any length.
struct RowPlan {
  int lanes, chunks;
};

// The least lanes and pieces that hold a row, two rows to a wavefront from 65 to 96
// pieces (77 pieces as 64 lanes by 2 leave 40% of the slots empty).
RowPlan plan_row(int dtype, int64_t cols) {
  const int64_t n = ceil_div(cols, dtype == 0 ? 4 : 8);
  for (const RowPlan p : {RowPlan{16, 1}, RowPlan{32, 1}, RowPlan{64, 1}, RowPlan{32, 3},
                          RowPlan{64, 2}, RowPlan{64, 3}, RowPlan{64, 4}, RowPlan{256, 2},
                          RowPlan{256, 4}, RowPlan{256, 8}}) {
    if (n <= p.lanes * p.chunks) return p;
  }
  return {0, 0};
}

int rows_at_once(const RowPlan &p) {
  return p.lanes > 64 ? 1 : dense::kNormThreads / p.lanes;
}

int forward_blocks(const RowPlan &p, int64_t rows) {
  const int64_t most = p.lanes > 64 ? 2048 : 1024, want = ceil_div(rows, rows_at_once(p));
  return static_cast<int>(want < most ? want : most);
}

// Workgroups of the backward; each leaves a row of column sums, so wide rows take
// fewer: at 256 and 512, 20000 x 1024 bf16 28.6 and 31.5 us, 30021 x 611 float16 37.5
// and 41.1, but 180000 x 256 bf16 59.1 and 58.0; a workgroup a row, at 512 and 1024,
// 8000 x 4096 bf16 57 and 71.
int backward_blocks(const RowPlan &p, int64_t rows) {
  if (p.lanes == 0) return static_cast<int>(rows < 64 ? rows : 64);
  const int64_t most = p.lanes <= 64 && p.chunks > 1 ? 256 : 512;
  const int64_t want = ceil_div(rows, rows_at_once(p));
  return static_cast<int>(want < most ? want : most);
}

template <typename F>
void by_type(int dtype, int weight_dtype, F &&f) {
  if (dtype == 0) {
    f(float{}, std::false_type{}, float{});
  } else if (dtype == 1) {
    if (weight_dtype == 0) {
      f(__half{}, std::true_type{}, float{});
    } else {
      f(__half{}, std::false_type{}, __half{});
    }
  } else if (weight_dtype == 0) {
    f(dense::bf16_t{}, std::true_type{}, float{});
  } else {
    f(dense::bf16_t{}, std::false_type{}, dense::bf16_t{});
  }
}

template <typename T, bool kW32, bool kBackward, int kLanes, int kChunks, bool kFull>
void launch_rows(const Norm &a, int blocks, hipStream_t st) {
  constexpr int kThreads = dense::NormShape<kLanes>::kThreads;
  if constexpr (kBackward) {
    dense::norm_backward<T, kW32, kLanes, kChunks, kFull><<<blocks, kThreads, 0, st>>>(a);
  } else {
    dense::norm_forward<T, kW32, kLanes, kChunks, kFull><<<blocks, kThreads, 0, st>>>(a);
  }
}

template <typename T, bool kW32, bool kBackward, int kLanes, int kChunks>
void launch_full(const Norm &a, int blocks, hipStream_t st) {
  if (a.cols == kLanes * kChunks * dense::Piece<T>::kValues) {
    launch_rows<T, kW32, kBackward, kLanes, kChunks, true>(a, blocks, st);
  } else {
    launch_rows<T, kW32, kBackward, kLanes, kChunks, false>(a, blocks, st);
  }
}

template <typename T, bool kW32, bool kBackward>
void launch(const RowPlan &p, const Norm &a, int blocks, hipStream_t st) {
  if (p.lanes == 16) {
    launch_full<T, kW32, kBackward, 16, 1>(a, blocks, st);
  } else if (p.lanes == 32 && p.chunks == 1) {
    launch_full<T, kW32, kBackward, 32, 1>(a, blocks, st);
  } else if (p.lanes == 32) {
    launch_full<T, kW32, kBackward, 32, 3>(a, blocks, st);
  } else if (p.lanes == 64 && p.chunks == 1) {
    launch_full<T, kW32, kBackward, 64, 1>(a, blocks, st);
  } else if (p.lanes == 64 && p.chunks == 2) {
    launch_full<T, kW32, kBackward, 64, 2>(a, blocks, st);
  } else if (p.lanes == 64 && p.chunks == 3) {
    launch_full<T, kW32, kBackward, 64, 3>(a, blocks, st);
  } else if (p.lanes == 64) {
    launch_full<T, kW32, kBackward, 64, 4>(a, blocks, st);
  } else if (p.chunks == 2) {
    launch_rows<T, kW32, kBackward, 256, 2, false>(a, blocks, st);
  } else if (p.chunks == 4) {
    launch_rows<T, kW32, kBackward, 256, 4, false>(a, blocks, st);
  } else {
    launch_rows<T, kW32, kBackward, 256, 8, false>(a, blocks, st);
  }
}

}  // namespace

extern "C" {

int layer_norm_forward(const void *x, int dtype, const void *weight, const void *bias,
                       int weight_dtype, void *output, float *statistics, int64_t rows,
                       int64_t cols, float eps, void *stream) {
  const char *fn = "layer_norm_forward";
  int rc = validate(fn, dtype, weight_dtype, rows, cols);
  if (rc != MUSPACE_OK) return rc;
  if (rows == 0 || cols == 0) return ok();
  if (x == nullptr || output == nullptr) return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  Norm a = {};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.out = output;
  a.stats = statistics;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.eps = eps;
  const RowPlan plan = plan_row(dtype, cols);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, weight_dtype, [&](auto t, auto w32, auto) {
    using T = decltype(t);
    constexpr bool kW32 = decltype(w32)::value;
    if (plan.lanes == 0) {
      const int blocks = static_cast<int>(rows < 2048 ? rows : 2048);
      dense::norm_forward_long<T, kW32><<<blocks, 256, 0, st>>>(a);
    } else {
      launch<T, kW32, false>(plan, a, forward_blocks(plan, rows), st);
    }
  });
  return check_launch(fn);
}

size_t layer_norm_backward_workspace_size(int dtype, int64_t rows, int64_t cols) {
  if (validate("layer_norm_backward_workspace_size", dtype, 0, rows, cols) != MUSPACE_OK) return 0;
  return static_cast<size_t>(backward_blocks(plan_row(dtype, cols), rows)) * 2 * cols * 4;
}

int layer_norm_backward(const void *grad_output, int dtype, const void *x, const void *weight,
                        int weight_dtype, const float *statistics, void *grad_input,
                        void *grad_weight, void *grad_bias, int64_t rows, int64_t cols,
                        void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "layer_norm_backward";
  int rc = validate(fn, dtype, weight_dtype, rows, cols);
  if (rc != MUSPACE_OK) return rc;
  const bool columns = grad_weight != nullptr || grad_bias != nullptr;
  if (cols == 0 || (grad_input == nullptr && !columns)) return ok();
  if (rows > 0 && (grad_output == nullptr || x == nullptr || statistics == nullptr)) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  const size_t need = columns ? layer_norm_backward_workspace_size(dtype, rows, cols) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
    return fail(MUSPACE_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", fn,
                need, workspace == nullptr ? size_t{0} : workspace_bytes);
  }
  Norm a = {};
  a.x = x;
  a.weight = weight;
  a.grad = grad_output;
  a.out = rows > 0 ? grad_input : nullptr;
  a.stats = const_cast<float *>(statistics);
  a.partial = columns ? static_cast<float *>(workspace) : nullptr;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  const RowPlan plan = plan_row(dtype, cols);
  const int blocks = backward_blocks(plan, rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, weight_dtype, [&](auto t, auto w32, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr bool kW32 = decltype(w32)::value;
    if (rows > 0) {
      if (plan.lanes != 0) {
        launch<T, kW32, true>(plan, a, blocks, st);
      } else {
        if (a.out != nullptr) {
          dense::norm_backward_long<T, kW32>
              <<<static_cast<int>(rows < 2048 ? rows : 2048), 256, 0, st>>>(a);
        }
        if (columns) {
          const int across = static_cast<int>(ceil_div(cols, 256 * dense::Piece<T>::kValues));
          dense::norm_columns_long<T><<<dim3(across, blocks), 256, 0, st>>>(a);
        }
      }
    }
    if (columns) {
      dense::norm_sum_columns<W><<<static_cast<int>(ceil_div(2 * cols, 16)), 256, 0, st>>>(
          a.partial, blocks, a.cols, static_cast<W *>(grad_weight), static_cast<W *>(grad_bias));
    }
  });
  return check_launch(fn);
}

}  // extern "C"
