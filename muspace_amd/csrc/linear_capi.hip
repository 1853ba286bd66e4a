// C-ABI entry points of the linear layer (declared in include/muspace_layer.h).
// Plans (tile sizes, parts of k) are functions of sizes, type and alignment only.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "../../include/muspace_layer.h"
#include "capi_errors.hpp"
#include "linear_kernels.hpp"

namespace {

using capi::check_launch;
using capi::fail;
using capi::ok;
using dense::Job;
using dense::Kind;
using dense::Product;

constexpr int64_t kMaxRows = INT_MAX - 256;
constexpr int64_t kMaxFeatures = 1 << 20;
constexpr int kCus = 256;

int validate(const char *fn, int dtype, int64_t rows, int64_t in, int64_t out, int act) {
  if (dtype < 0 || dtype > 2) {
    return fail(MUSPACE_EINVAL, "%s: tensors must be float32, float16 or bfloat16", fn);
  }
  if (rows < 0 || in < 0 || out < 0) {
    return fail(MUSPACE_EINVAL, "%s: invalid dims rows=%lld in_features=%lld out_features=%lld",
                fn, (long long)rows, (long long)in, (long long)out);
  }
  if (act < dense::kNone || act > dense::kGelu) {
    return fail(MUSPACE_EINVAL, "%s: activation must be 0 (none), 1 (relu) or 2 (gelu), got %d",
                fn, act);
  }
  // a launch holds fewer than 2^32 threads: 2^24 tiles of 128 x 128
  const int64_t r = rows / 128 + 1, i = in / 128 + 1, o = out / 128 + 1;
  constexpr int64_t kTiles = 1 << 24;
  if (rows > kMaxRows || in > kMaxFeatures || out > kMaxFeatures || r * i > kTiles ||
      r * o > kTiles || i * o > kTiles) {
    return fail(MUSPACE_ERANGE, "%s: dims exceed the kernels' 32-bit indexing", fn);
  }
  return ok();
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int value_bytes(int dtype) { return dtype == 0 ? 4 : 2; }
int chunk_values(int dtype) { return 16 / value_bytes(dtype); }
int step_values(int dtype) { return dense::kRowBytes / value_bytes(dtype); }
size_t pad256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// gelu's dz in the workspace: rows of whole chunks, and a second tensor for what
// rounding to 16 bits left
int dz_tensors(int dtype) { return dtype == 0 ? 1 : 2; }
int64_t dz_chunks(int dtype, int64_t out) { return ceil_div(out, chunk_values(dtype)); }
size_t dz_bytes(int dtype, int64_t rows, int64_t out) {
  return pad256(static_cast<size_t>(rows) * dz_chunks(dtype, out) * 16);
}

// Tiles of 128 x 128 where they give every two CUs three, else 64 x 64. Forward, 64 and
// 128: 10000 x 512 -> 256 (158 tiles of 128) bf16 8.7 and 10.7 us, 12000 x 256 -> 512
// (376) 9.8 and 10.4, float32 26.0 and 26.8; 16000 x 256 -> 512 (500) 11.9 and 11.4,
// float32 33.4 and 29.1; 24000 x 1024 -> 512 (752) 46 and 35, float32 161 and 137.
bool large_tiles(int64_t m, int64_t n) {
  return ceil_div(m, 128) * ceil_div(n, 128) * 2 >= 3 * kCus;
}

// So few tiles of 64 x 64 that workgroups for 32 x 32 results, whose wavefronts share k,
// are done sooner. With them and in tiles, forward: 300 x 256 -> 256 (20 tiles) bf16 3.4
// and 3.8 us, float32 4.3 and 8.5; 1800 x 256 -> 256 (116) 4.0 and 4.0, float32 5.9 and
// 8.8; 2400 x 256 -> 256 (152) 5.7 and 4.0, float32 8.4 and 8.8; 3000 x 1024 -> 256 (188)
// 8.7 and 10.5, float32 21 and 26; 4000 x 1024 -> 256 (252) 10.6 and 11.2, float32 26.7
// and 25.9; 1500 x 1024 -> 1024 (384) 15 and 11.5.
template <typename T>
bool few_results(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = ceil_div(m, 64) * ceil_div(n, 64);
  if (sizeof(T) == 4) return tiles < 208;
  return tiles < (k >= 1024 ? 256 : 120);
}

struct WeightPlan {
  bool large;
  int splits, k_split;  // parts of the rows, rows in each
};

// dz^T x has few tiles and a long sum: the sum is cut into parts until there are
// about two workgroups a CU, each of at least four steps. At one, two, three and four
// workgroups a CU: 80000 x 512 -> 256 bf16 52, 47, 52 and 59 us, 44446 x 256 -> 1024
// float32 202, 154, 169 and 165, 40000 x 256 -> 512 bf16 35, 36, 40 and 49; more parts
// are more partial sums to write and read.
WeightPlan plan_weight(int dtype, int64_t rows, int64_t in, int64_t out) {
  WeightPlan p;
  p.large = in > 64 && out > 64;
  const int b = p.large ? 128 : 64;
  const int64_t tiles = ceil_div(out, b) * (in > 0 ? ceil_div(in, b) : 1);
  const int64_t steps = ceil_div(rows, step_values(dtype));
  int64_t splits = tiles > 0 ? 2 * kCus / tiles : 1;
  if (splits > steps / 4) splits = steps / 4;
  if (splits < 1) splits = 1;
  const int64_t per = ceil_div(steps, splits);
  p.k_split = static_cast<int>((per > 0 ? per : 1) * step_values(dtype));
  p.splits = static_cast<int>(rows > 0 ? ceil_div(rows, p.k_split) : 1);
  return p;
}

// gradients that are asked for and have values
struct Wanted {
  bool input, weight, bias;
  Wanted(bool input_, bool weight_, bool bias_, int64_t rows, int64_t in, int64_t out)
      : input(input_ && rows > 0 && in > 0), weight(weight_ && in > 0 && out > 0),
        bias(bias_ && out > 0) {}
  bool any() const { return input || weight || bias; }
};

// The parts' sums: the weight's, then the bias's.
size_t weight_partial_bytes(const WeightPlan &p, const Wanted &want, int64_t in, int64_t out) {
  if (p.splits == 1 || !want.weight) return 0;
  const size_t ld = static_cast<size_t>((in + 7) & ~int64_t{7});
  return pad256(static_cast<size_t>(p.splits) * out * ld * 4);
}
size_t bias_partial_bytes(const WeightPlan &p, const Wanted &want, int64_t out) {
  return p.splits == 1 || !want.bias ? 0 : pad256(static_cast<size_t>(p.splits) * out * 4);
}

size_t workspace_bytes_of(int dtype, const Wanted &want, int64_t rows, int64_t in, int64_t out,
                          int activation) {
  const WeightPlan plan = plan_weight(dtype, rows, in, out);
  size_t bytes = weight_partial_bytes(plan, want, in, out) + bias_partial_bytes(plan, want, out);
  if (activation == dense::kGelu && want.any()) bytes += dz_tensors(dtype) * dz_bytes(dtype, rows, out);
  return bytes;
}

template <typename T, Job kJob, int B, Kind kKind, bool kCodes>
void launch_tight(const Product &a, int blocks, bool tight, hipStream_t st) {
  if (tight) {
    dense::linear_product<T, kJob, B, B, true, kKind, kCodes>
        <<<blocks, dense::kThreads, 0, st>>>(a);
  } else {
    dense::linear_product<T, kJob, B, B, false, kKind, kCodes>
        <<<blocks, dense::kThreads, 0, st>>>(a);
  }
}

template <typename T, Job kJob, Kind kKind, bool kCodes>
void launch_product(Product a, bool large, bool tight, hipStream_t st) {
  const int b = large ? 128 : 64;
  a.tiles_n = static_cast<int>(ceil_div(a.n > 0 ? a.n : 1, b));
  a.tiles = static_cast<int>(ceil_div(a.m, b)) * a.tiles_n;
  const int blocks = a.tiles * a.splits;
  if (blocks == 0) return;
  if (large) {
    launch_tight<T, kJob, 128, kKind, kCodes>(a, blocks, tight, st);
  } else {
    launch_tight<T, kJob, 64, kKind, kCodes>(a, blocks, tight, st);
  }
}

template <typename T, Job kJob, Kind kKind>
void launch_few(Product a, bool tight, hipStream_t st) {
  // four and eight: 64 x 2048 -> 2048 bf16 8.7 and 6.6 us, 300 x 256 -> 256 3.3 and 3.4
  constexpr int kWaves = 8;
  a.tiles_n = static_cast<int>(ceil_div(a.n, 32));
  a.tiles = static_cast<int>(ceil_div(a.m, 32)) * a.tiles_n;
  if (tight) {
    dense::linear_few<T, kJob, kWaves, true, kKind><<<a.tiles, kWaves * 64, 0, st>>>(a);
  } else {
    dense::linear_few<T, kJob, kWaves, false, kKind><<<a.tiles, kWaves * 64, 0, st>>>(a);
  }
}

template <typename T, Job kJob, Kind kKind>
void run_rows(const Product &a, bool tight, hipStream_t st) {
  if (few_results<T>(a.m, a.n, a.k)) {
    launch_few<T, kJob, kKind>(a, tight, st);
  } else {
    launch_product<T, kJob, kKind, false>(a, large_tiles(a.m, a.n), tight, st);
  }
}

// Rows that the vector unit multiplies while W is read. linear_few and linear_vector, us,
// at one row, and at the most here (8 of float32, 4 of 16 bits):
//   float32   256 -> 256    4.1  2.1    4.2  3.1      bfloat16    3.3  2.3    3.3  2.9
//            2048 -> 2048  15.1  4.3   15.2  6.9                  6.0  2.7    6.0  3.7
//            4096 -> 16384  117   47    117   79                 54.7 23.9   54.8 32.7
//             203 -> 611    4.5  2.2    4.6  3.2                  3.6  2.4    3.8  3.0
// Eight 16-bit rows were no gain (256 -> 256 3.3 3.5, 2048 -> 2048 6.0 5.5).
template <typename T>
bool few_rows(int64_t rows) {
  return rows <= (sizeof(T) == 4 ? 8 : 4);
}

template <typename T, int kRows, int kCols>
void launch_vector(const Product &a, hipStream_t st) {
  dense::linear_vector<T, kRows, kCols>
      <<<static_cast<int>(ceil_div(a.n, 8)), 8 / kCols * 64, 0, st>>>(a);
}

template <typename T>
void run_vector(const Product &a, hipStream_t st) {
  if (a.m == 1) {
    launch_vector<T, 1, 1>(a, st);
  } else if (a.m == 2) {
    launch_vector<T, 2, 1>(a, st);
  } else if (a.m <= 4) {
    launch_vector<T, 4, 2>(a, st);
  } else if constexpr (sizeof(T) == 4) {
    launch_vector<T, 8, 2>(a, st);
  }
}

int grid_for(int64_t work) {
  const int64_t b = ceil_div(work, dense::kThreads);
  return static_cast<int>(b > 65536 ? 65536 : (b < 1 ? 1 : b));
}

template <typename T>
void run_checkpoint(const void *x, uint8_t *codes, uint8_t *scales, int64_t rows,
                    int64_t in_features, hipStream_t st) {
  const int64_t work = rows * (((in_features + 31) & ~int64_t{31}) / dense::Piece<T>::kValues);
  dense::linear_checkpoint<T><<<grid_for(work), dense::kThreads, 0, st>>>(
      static_cast<const T *>(x), codes, scales, rows, static_cast<int>(in_features));
}

// f(the kind of dz that `a` holds, as a type)
template <typename T, typename F>
void by_kind(const Product &a, F &&f) {
  if (a.mask != nullptr) {
    f(std::integral_constant<Kind, Kind::kMasked>{});
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (a.p_rest != nullptr) {
      f(std::integral_constant<Kind, Kind::kPair>{});
      return;
    }
  }
  f(std::integral_constant<Kind, Kind::kPlain>{});
}

template <typename T>
void run_weight(const Product &a, const WeightPlan &plan, bool tight, bool codes, void *dw, void *db,
                hipStream_t st) {
  by_kind<T>(a, [&](auto kind) {
    constexpr Kind kKind = decltype(kind)::value;
    if (codes) {
      launch_product<T, Job::kWeight, kKind, true>(a, plan.large, tight, st);
    } else {
      launch_product<T, Job::kWeight, kKind, false>(a, plan.large, tight, st);
    }
  });
  if (plan.splits > 1) {
    const int64_t work = static_cast<int64_t>(a.m) * ((a.n + 7) / 8 * 2) + a.m;
    dense::linear_weight_sum<T>
        <<<static_cast<unsigned>(ceil_div(work, dense::kSumPieces)), dense::kThreads, 0, st>>>(
            a.partial, a.bias_partial, static_cast<T *>(dw), static_cast<T *>(db), a.m, a.n,
            plan.splits);
  }
}

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

}  // namespace

extern "C" {

int linear_forward(const void *x, int dtype, const void *weight, const void *bias,
                   const void *residual, void *output, uint8_t *relu_mask, void *pre_activation,
                   int8_t *codes, uint8_t *scales, int64_t rows, int64_t in_features,
                   int64_t out_features, int activation, void *stream) {
  int rc = validate("linear_forward", dtype, rows, in_features, out_features, activation);
  if (rc != MUSPACE_OK) return rc;
  if (rows == 0 || out_features == 0) return ok();
  if (output == nullptr || (in_features > 0 && (x == nullptr || weight == nullptr))) {
    return fail(MUSPACE_EINVAL, "linear_forward: null tensor pointer");
  }
  if ((codes == nullptr) != (scales == nullptr)) {
    return fail(MUSPACE_EINVAL, "linear_forward: codes and scales come together");
  }
  if (reinterpret_cast<uintptr_t>(codes) % 8 != 0) {
    return fail(MUSPACE_EINVAL, "linear_forward: codes must be 8-byte aligned");
  }
  Product a = {};
  a.p = x;
  a.q = weight;
  a.ldp = a.ldq = in_features;
  a.m = static_cast<int>(rows);
  a.n = static_cast<int>(out_features);
  a.k = static_cast<int>(in_features);
  a.splits = 1;
  a.bias = bias;
  a.residual = residual;
  a.out = output;
  a.slope_out = activation == dense::kGelu ? pre_activation : nullptr;
  a.mask_out = activation == dense::kRelu ? relu_mask : nullptr;
  a.mask_ld = rows * 8;
  a.act = activation;
  a.codes = reinterpret_cast<uint8_t *>(codes);
  a.code_scales = scales;
  const bool tight =
      in_features % chunk_values(dtype) == 0 && aligned16(x) && aligned16(weight);
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (few_rows<T>(a.m)) {
      if (codes != nullptr && a.k > 0) run_checkpoint<T>(x, a.codes, scales, rows, a.k, st);
      run_vector<T>(a, st);
      return;
    }
    if (codes != nullptr) {
      run_rows<T, Job::kForward, Kind::kKept>(a, tight, st);
    } else {
      run_rows<T, Job::kForward, Kind::kPlain>(a, tight, st);
    }
  });
  return check_launch("linear_forward");
}

int linear_checkpoint(const void *x, int dtype, int8_t *codes, uint8_t *scales, int64_t rows,
                      int64_t in_features, void *stream) {
  int rc = validate("linear_checkpoint", dtype, rows, in_features, 0, 0);
  if (rc != MUSPACE_OK) return rc;
  if (rows == 0 || in_features == 0) return ok();
  if (x == nullptr || codes == nullptr || scales == nullptr) {
    return fail(MUSPACE_EINVAL, "linear_checkpoint: null tensor pointer");
  }
  if (reinterpret_cast<uintptr_t>(codes) % 8 != 0) {
    return fail(MUSPACE_EINVAL, "linear_checkpoint: codes must be 8-byte aligned");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    run_checkpoint<decltype(t)>(x, reinterpret_cast<uint8_t *>(codes), scales, rows,
                                in_features, st);
  });
  return check_launch("linear_checkpoint");
}

size_t linear_backward_workspace_size_for(int dtype, int64_t rows, int64_t in_features,
                                          int64_t out_features, int activation, int want_input,
                                          int want_weight, int want_bias) {
  if (validate("linear_backward_workspace_size", dtype, rows, in_features, out_features,
               activation) != MUSPACE_OK) {
    return 0;
  }
  const Wanted want(want_input != 0, want_weight != 0, want_bias != 0, rows, in_features,
                    out_features);
  return workspace_bytes_of(dtype, want, rows, in_features, out_features, activation);
}

size_t linear_backward_workspace_size(int dtype, int64_t rows, int64_t in_features,
                                      int64_t out_features, int activation) {
  return linear_backward_workspace_size_for(dtype, rows, in_features, out_features, activation, 1,
                                            1, 1);
}

int linear_backward(const void *grad_output, int dtype, const void *x, const int8_t *codes,
                    const uint8_t *scales, const void *weight, const uint8_t *relu_mask,
                    const void *pre_activation, void *grad_input, void *grad_weight,
                    void *grad_bias, int64_t rows, int64_t in_features, int64_t out_features,
                    int activation, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "linear_backward";
  int rc = validate(fn, dtype, rows, in_features, out_features, activation);
  if (rc != MUSPACE_OK) return rc;
  const Wanted want(grad_input != nullptr, grad_weight != nullptr, grad_bias != nullptr, rows,
                    in_features, out_features);
  if (!want.any()) return ok();
  const bool summed = rows > 0 && out_features > 0;  // dz has values
  if ((codes == nullptr) != (scales == nullptr)) {
    return fail(MUSPACE_EINVAL, "%s: codes and scales come together", fn);
  }
  if (reinterpret_cast<uintptr_t>(codes) % 8 != 0) {
    return fail(MUSPACE_EINVAL, "%s: codes must be 8-byte aligned", fn);
  }
  if (summed &&
      (grad_output == nullptr || (want.input && weight == nullptr) ||
       (want.weight && x == nullptr && codes == nullptr) ||
       (activation == dense::kRelu && relu_mask == nullptr) ||
       (activation == dense::kGelu && pre_activation == nullptr))) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  const size_t need =
      workspace_bytes_of(dtype, want, rows, in_features, out_features, activation);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 256 != 0)) {
    return fail(MUSPACE_EINVAL, "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu", fn,
                need, workspace == nullptr ? size_t{0} : workspace_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  const void *dz = grad_output, *dz_rest = nullptr;
  const int v = chunk_values(dtype);
  int64_t dz_ld = out_features;
  if (activation == dense::kGelu && summed) {
    const size_t bytes = dz_bytes(dtype, rows, out_features);
    if (dz_tensors(dtype) == 2) dz_rest = ws + bytes;
    dz_ld = dz_chunks(dtype, out_features) * v;
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      dense::linear_gelu_grad<T>
          <<<grid_for(rows * dz_chunks(dtype, out_features)), dense::kThreads, 0, st>>>(
              static_cast<const T *>(grad_output), static_cast<const T *>(pre_activation),
              reinterpret_cast<T *>(ws), static_cast<T *>(const_cast<void *>(dz_rest)), rows,
              static_cast<int>(out_features));
    });
    dz = ws;
    ws += dz_tensors(dtype) * bytes;
  }
  const bool whole_out = dz_ld % v == 0 && aligned16(dz);
  const uint8_t *mask = activation == dense::kRelu && summed ? relu_mask : nullptr;

  if (want.input) {
    Product a = {};
    a.p = dz;
    a.p_rest = dz_rest;
    a.q = weight;
    a.ldp = dz_ld;
    a.ldq = in_features;
    a.m = static_cast<int>(rows);
    a.n = static_cast<int>(in_features);
    a.k = static_cast<int>(out_features);
    a.mask = mask;
    a.mask_ld = rows * 8;
    a.splits = 1;
    a.out = grad_input;
    const bool tight = whole_out && in_features % v == 0 && aligned16(weight);
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      by_kind<T>(a, [&](auto kind) {
        run_rows<T, Job::kInput, decltype(kind)::value>(a, tight, st);
      });
    });
  }
  if (want.weight || want.bias) {
    const WeightPlan plan = plan_weight(dtype, rows, in_features, out_features);
    Product a = {};
    a.p = dz;
    a.p_rest = dz_rest;
    a.ldp = dz_ld;
    a.m = static_cast<int>(out_features);
    // without a weight gradient: no columns, the first column of tiles sums dz
    a.n = want.weight ? static_cast<int>(in_features) : 0;
    a.k = static_cast<int>(rows);
    const bool coded = want.weight && codes != nullptr;
    a.q = coded ? static_cast<const void *>(codes) : x;
    a.ldq = coded ? (in_features + 31) & ~int64_t{31} : in_features;
    a.scales = coded ? scales : nullptr;
    a.scale_ld = a.ldq / 32;
    a.mask = mask;
    a.mask_ld = rows * 8;
    a.splits = plan.splits;
    a.k_split = plan.k_split;
    a.out = grad_weight;
    if (plan.splits > 1) {
      a.partial = reinterpret_cast<float *>(ws);  // (without a weight gradient: not written)
      if (want.bias) {
        a.bias_partial = reinterpret_cast<float *>(
            ws + weight_partial_bytes(plan, want, in_features, out_features));
      }
    } else if (want.bias) {
      a.bias_out = grad_bias;
    }
    const bool tight =
        whole_out && (!want.weight || coded || (in_features % v == 0 && aligned16(x)));
    by_type(dtype, [&](auto t) {
      run_weight<decltype(t)>(a, plan, tight, coded, grad_weight, want.bias ? grad_bias : nullptr,
                              st);
    });
  }
  return check_launch(fn);
}

}  // extern "C"
