// C-ABI entry points of the linear layer in 8-bit integers (declared in
// include/muspace_layer.h). Plans are functions of sizes, types and alignment only.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "../../include/muspace_layer.h"
#include "capi_errors.hpp"
#include "wide_kernels.hpp"

namespace {

using capi::check_launch;
using capi::fail;
using capi::ok;
using dense::Codes;

constexpr int64_t kMaxRows = INT_MAX - 256;
constexpr int64_t kMaxOut = 1 << 20;
constexpr int64_t kMaxIn = 1 << 17;  // 2^17 * 128 * 127 < 2^31: a sum is an int32 number
constexpr int kCus = 256;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t pad256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
int64_t padded(int64_t in) { return (in + 15) & ~int64_t{15}; }

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

int validate(const char *fn, int dtype, int64_t rows, int64_t in, int64_t out) {
  if (dtype < 0 || dtype > 2) {
    return fail(MUSPACE_EINVAL, "%s: tensors must be float32, float16 or bfloat16", fn);
  }
  if (rows < 0 || in < 0 || out < 0) {
    return fail(MUSPACE_EINVAL, "%s: invalid dims rows=%lld in_features=%lld out_features=%lld",
                fn, (long long)rows, (long long)in, (long long)out);
  }
  // a launch holds fewer than 2^32 threads: 2^24 tiles of 128 x 128
  if (rows > kMaxRows || in > kMaxIn || out > kMaxOut ||
      (rows / 128 + 1) * (out / 128 + 1) > (1 << 24)) {
    return fail(MUSPACE_ERANGE, "%s: dims exceed the kernels' 32-bit indexing and sums", fn);
  }
  return ok();
}

template <typename T, int kLanes = 16>
void launch_rows(int64_t pieces, const dense::Quantise &a, hipStream_t st) {
  if constexpr (kLanes > dense::kQuantThreads) {
    dense::int8_rows_long<T>
        <<<static_cast<int>(a.rows < 4096 ? a.rows : 4096), dense::kQuantThreads, 0, st>>>(a);
  } else if (pieces > kLanes) {
    launch_rows<T, kLanes * 2>(pieces, a, st);
  } else {
    const int64_t want = ceil_div(a.rows, dense::kQuantThreads / kLanes);
    dense::int8_rows<T, kLanes>
        <<<static_cast<int>(want < 4096 ? want : 4096), dense::kQuantThreads, 0, st>>>(a);
  }
}

void quantise(const void *x, int dtype, int8_t *codes, float *scales, int64_t rows, int64_t cols,
              int64_t ld, hipStream_t st) {
  const dense::Quantise a = {x, codes, scales, rows, ld, static_cast<int>(cols)};
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    launch_rows<T>(ceil_div(ld, dense::Piece<T>::kValues), a, st);
  });
}

template <typename T, int B>
void launch_product(Codes a, bool tight, hipStream_t st) {
  a.p.tiles_n = static_cast<int>(ceil_div(a.p.n, B));
  a.p.tiles = static_cast<int>(ceil_div(a.p.m, B)) * a.p.tiles_n;
  if (tight) {
    dense::int8_product<T, B, B, true><<<a.p.tiles, dense::kThreads, 0, st>>>(a);
  } else {
    dense::int8_product<T, B, B, false><<<a.p.tiles, dense::kThreads, 0, st>>>(a);
  }
}

// So few results that workgroups of 32 x 32 are done sooner (see linear_capi's few_results).
bool few_results(int64_t m, int64_t n) { return ceil_div(m, 64) * ceil_div(n, 64) < 120; }

// Whether the product's own kernel quantises x: codes and scales are not written.
bool few_rows(int64_t m, int64_t k) {
  return m <= 4 && (m <= 2 ? m : 4) * padded(k) <= dense::kVectorCodes;
}
// Rows that workgroups quantise and multiply with all of the weight: many, so that one and a
// half workgroups and more share a CU, and short ones; of a long weight 64 rows a time read too
// much. In two kernels and in this one, us, bf16: 180000 x 256 -> 256 65.6 and 57.1, 40000 x 256
// -> 512 32.2 and 29.7, 25000 x 256 -> 256 19.0 and 16.3, 100000 x 128 -> 128 25.4 and 22.7; 17000
// x 256 -> 256 13.0 and 14.9, 33000 x 256 -> 1024 52 and 62; between, 40000 x 256 -> 640 33.4 and
// 30.6, -> 768 34.5 and 33.6. With codes of 512 values in LDS, two workgroups a CU: 40000 x 320 ->
// 512 35.9 and 40.9, x 512 39.1 and 47.7. Unaligned rows of the weight, which every workgroup reads
// anew: 40000 x 100 -> 512 24.5 and 31.2, 180000 x 3 -> 256 44.5 and 57.3. Few products for a row:
// 40000 x 32 -> 32 9.5 and 10.5, float32 9.0 and 10.7, x 64 -> 64 10.1 and 11.3; 40000 x 64 -> 256
// float32 18.0 and 16.2, x 128 -> 64 13.4 and 11.7. (A launch holds fewer than 2^32 threads;
// tiles are of twice as many rows.)
bool row_blocks(int64_t m, int64_t n, int64_t k) {
  const int64_t blocks = ceil_div(m, dense::kBlockRows);
  return k <= dense::kBlockIn && k % 16 == 0 && (k > 64 || n > 128) && n <= 512 &&
         blocks * 2 >= 3 * kCus && blocks * dense::kThreads < int64_t{1} << 32;
}
bool fused(int64_t m, int64_t n, int64_t k) {
  return few_rows(m, k) || (few_results(m, n) ? k <= dense::kFusedIn : row_blocks(m, n, k));
}

template <typename T, int kRows>
void launch_vector(const Codes &a, hipStream_t st) {
  dense::int8_vector<T, kRows><<<static_cast<int>(ceil_div(a.p.n, 16)), dense::kQuantThreads,
                                 kRows * padded(a.p.k), st>>>(a);
}

template <typename T, bool kFused>
void launch_few(Codes a, bool tight, hipStream_t st) {
  constexpr int kWaves = 8;
  a.p.tiles_n = static_cast<int>(ceil_div(a.p.n, 32));
  a.p.tiles = static_cast<int>(ceil_div(a.p.m, 32)) * a.p.tiles_n;
  if (tight) {
    dense::int8_few<T, kWaves, true, kFused><<<a.p.tiles, kWaves * 64, 0, st>>>(a);
  } else {
    dense::int8_few<T, kWaves, false, kFused><<<a.p.tiles, kWaves * 64, 0, st>>>(a);
  }
}

template <typename T>
void run(Codes a, bool tight, hipStream_t st) {
  if (few_rows(a.p.m, a.p.k)) {
    if (a.p.m == 1) {
      launch_vector<T, 1>(a, st);
    } else if (a.p.m == 2) {
      launch_vector<T, 2>(a, st);
    } else {
      launch_vector<T, 4>(a, st);
    }
  } else if (few_results(a.p.m, a.p.n)) {
    if (a.p.k <= dense::kFusedIn) {
      launch_few<T, true>(a, tight, st);
    } else {
      launch_few<T, false>(a, tight, st);
    }
  } else if (row_blocks(a.p.m, a.p.n, a.p.k)) {
    const int blocks = static_cast<int>(ceil_div(a.p.m, dense::kBlockRows));
    if (tight) {
      dense::int8_row_block<T, true><<<blocks, dense::kThreads, 0, st>>>(a);
    } else {
      dense::int8_row_block<T, false><<<blocks, dense::kThreads, 0, st>>>(a);
    }
  } else if (tight && dense::wide_tiles(a.p.m, a.p.n, a.p.k, 1)) {
    a.p.tiles_n = static_cast<int>(ceil_div(a.p.n, dense::kWide));
    a.p.tiles = static_cast<int>(ceil_div(a.p.m, dense::kWide)) * a.p.tiles_n;
    dense::wide_product<int8_t, T, dense::Job::kForward>
        <<<a.p.tiles, dense::kWideThreads, 0, st>>>(a);
  } else if (ceil_div(a.p.m, 128) * ceil_div(a.p.n, 128) * 2 >= 3 * kCus) {
    launch_product<T, 128>(a, tight, st);
  } else {
    launch_product<T, 64>(a, tight, st);
  }
}

}  // namespace

extern "C" {

int quantize_int8(const void *x, int dtype, int8_t *codes, float *scales, int64_t rows,
                  int64_t cols, void *stream) {
  const char *fn = "quantize_int8";
  const int rc = validate(fn, dtype, rows, 0, 0);
  if (rc != MUSPACE_OK) return rc;
  if (cols < 0 || cols > kMaxOut) {
    return fail(cols < 0 ? MUSPACE_EINVAL : MUSPACE_ERANGE, "%s: invalid dims cols=%lld", fn,
                (long long)cols);
  }
  if (rows == 0) return ok();
  if (scales == nullptr || (cols > 0 && (x == nullptr || codes == nullptr))) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  quantise(x, dtype, codes, scales, rows, cols, cols, static_cast<hipStream_t>(stream));
  return check_launch(fn);
}

size_t linear_int8_workspace_size(int dtype, int64_t rows, int64_t in_features,
                                  int64_t out_features) {
  if (validate("linear_int8_workspace_size", dtype, rows, in_features, out_features) !=
          MUSPACE_OK ||
      rows == 0 || out_features == 0 || fused(rows, out_features, in_features)) {
    return 0;
  }
  return pad256(static_cast<size_t>(rows) * padded(in_features)) +
         pad256(static_cast<size_t>(rows) * 4);
}

int linear_int8_forward(const void *x, int dtype, const int8_t *weight, const float *weight_scales,
                        const void *bias, const void *residual, void *output, int64_t rows,
                        int64_t in_features, int64_t out_features, int activation,
                        void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "linear_int8_forward";
  const int rc = validate(fn, dtype, rows, in_features, out_features);
  if (rc != MUSPACE_OK) return rc;
  if (activation < dense::kNone || activation > dense::kGelu) {
    return fail(MUSPACE_EINVAL, "%s: activation must be 0 (none), 1 (relu) or 2 (gelu), got %d",
                fn, activation);
  }
  if (rows == 0 || out_features == 0) return ok();
  if (output == nullptr || weight_scales == nullptr ||
      (in_features > 0 && (x == nullptr || weight == nullptr))) {
    return fail(MUSPACE_EINVAL, "%s: null tensor pointer", fn);
  }
  const size_t need = linear_int8_workspace_size(dtype, rows, in_features, out_features);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 256 != 0)) {
    return fail(MUSPACE_EINVAL, "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu", fn,
                need, workspace == nullptr ? size_t{0} : workspace_bytes);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t ld = padded(in_features);
  Codes a = {};
  if (need > 0) {
    int8_t *codes = static_cast<int8_t *>(workspace);
    float *scales = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                              pad256(static_cast<size_t>(rows) * ld));
    quantise(x, dtype, codes, scales, rows, in_features, ld, st);
    a.x = codes;
    a.x_scales = scales;
  }
  a.weight = weight;
  a.weight_scales = weight_scales;
  a.ldx = ld;
  a.p.p = x;
  a.p.m = static_cast<int>(rows);
  a.p.n = static_cast<int>(out_features);
  a.p.k = static_cast<int>(in_features);
  a.p.bias = bias;
  a.p.residual = residual;
  a.p.out = output;
  a.p.act = activation;
  const bool tight = in_features % 16 == 0 && aligned16(weight);
  by_type(dtype, [&](auto t) { run<decltype(t)>(a, tight, st); });
  return check_launch(fn);
}

}  // extern "C"
