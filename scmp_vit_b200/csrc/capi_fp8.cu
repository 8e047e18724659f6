// C ABI of the 8-bit linear and its parts (declared in include/scmp_b200.h):
// argument checks, layouts and launches.
#include "capi_check.cuh"
#include "fp8_common.cuh"

namespace scmp {
namespace {

int check_operand(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || rows > kMaxRows || K > kMaxRows)
    return fail(SCMP_EINVAL, "bad operand shape [%lld, %lld]", (long long)rows, (long long)K);
  return SCMP_OK;
}

int quantize(const Fp8Quantize &q, cudaStream_t s) {
  const cudaError_t e = launch_fp8_quantize(q, s);
  if (e != cudaSuccess) return cuda_fail(e, "fp8_quantize launch");
  add_launches(1);
  return SCMP_OK;
}

// Quantised operands on the tensor cores, or few rows in one launch.
int multiply(const Fp8Product &p, bool may_be_thin, cudaStream_t s) {
  cudaError_t e;
  if (may_be_thin && fp8_thin(p.M, p.N, p.K)) {
    e = launch_fp8_thin(p, nullptr, 0, 0, s);
    if (e == cudaSuccess) add_launches(1);
  } else {
    unsigned int *err = device_error_word();
    if (!err) return fail(SCMP_ECUDA, "cannot resolve the engine error word");
    e = launch_fp8_matmul(p, err, s);
  }
  return e == cudaSuccess ? SCMP_OK : cuda_fail(e, "fp8_matmul launch");
}

// A product's arguments; `codes`: A's buffers are needed.
int check_product(const scmp_fp8_matmul_args *args, bool codes, Fp8Product &p) {
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_fp8_matmul_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  int rc;
  if ((rc = check_operand(x.M, x.K)) != SCMP_OK || (rc = check_operand(x.N, x.K)) != SCMP_OK)
    return rc;
  if (!known_dtype(x.out_dtype) || (x.bias && !known_dtype(x.bias_dtype)))
    return fail(SCMP_EINVAL, "unknown dtype (out %d, bias %d)", x.out_dtype, x.bias_dtype);
  if (x.M > 0 && x.N > 0) {
    if ((codes && (!x.a || !x.a_scales)) || !x.b || !x.b_scales || !x.out)
      return fail(SCMP_EINVAL, "a, b, their scales and out must be non-NULL");
    if (!aligned({x.a, x.a_scales, x.b, x.b_scales}, 16))
      return fail(SCMP_EINVAL, "a, b and their scales must be 16-byte aligned");
    if ((rc = check_elements({x.out}, x.out_dtype)) != SCMP_OK ||
        (x.bias && (rc = check_elements({x.bias}, x.bias_dtype)) != SCMP_OK))
      return rc;
  }
  p.a = static_cast<const uint8_t *>(x.a);
  p.a_scales = static_cast<const uint8_t *>(x.a_scales);
  p.b = static_cast<const uint8_t *>(x.b);
  p.b_scales = static_cast<const uint8_t *>(x.b_scales);
  p.M = x.M;
  p.N = x.N;
  p.K = x.K;
  p.bias = x.bias;
  p.bias_dtype = x.bias_dtype;
  p.out = x.out;
  p.out_dtype = x.out_dtype;
  return SCMP_OK;
}

// Codes and scales of one operand, one behind the other, each on 256 bytes.
struct Operand {
  uint8_t *data, *scales;
};
size_t on_256(int64_t n) { return ((size_t)n + 255) & ~(size_t)255; }
size_t operand_bytes(int64_t rows, int64_t K) {
  const Fp8Layout l = fp8_layout(rows, K);
  return on_256(l.data_bytes()) + on_256(l.scale_bytes());
}
Operand carve(uint8_t *&at, int64_t rows, int64_t K) {
  const Fp8Layout l = fp8_layout(rows, K);
  Operand o{at, at + on_256(l.data_bytes())};
  at = o.scales + on_256(l.scale_bytes());
  return o;
}
size_t sums_bytes(int64_t M, int64_t N) { return on_256((M + 127) / 128 * N * 4); }

}  // namespace
}  // namespace scmp

using namespace scmp;

extern "C" {

size_t scmp_fp8_data_size(int64_t rows, int64_t K) {
  return check_operand(rows, K) != SCMP_OK ? 0 : (size_t)fp8_layout(rows, K).data_bytes();
}
size_t scmp_fp8_scale_size(int64_t rows, int64_t K) {
  return check_operand(rows, K) != SCMP_OK ? 0 : (size_t)fp8_layout(rows, K).scale_bytes();
}

int scmp_fp8_quantize(const scmp_fp8_quantize_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_fp8_quantize_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  int rc = check_operand(x.rows, x.K);
  if (rc != SCMP_OK) return rc;
  if (!known_dtype(x.dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", x.dtype);
  if (x.ld < x.K)
    return fail(SCMP_EINVAL, "ld=%lld below K=%lld", (long long)x.ld, (long long)x.K);
  if (x.rows == 0) return SCMP_OK;
  if (!x.x || !x.data != !x.scales || !x.t_data != !x.t_scales || (!x.data && !x.t_data))
    return fail(SCMP_EINVAL, "x, and codes and scales of one order at least, must be non-NULL");
  if (!aligned({x.data, x.scales, x.t_data, x.t_scales}, 16))
    return fail(SCMP_EINVAL, "codes and scales must be 16-byte aligned");
  if ((rc = check_elements({x.x}, x.dtype)) != SCMP_OK) return rc;
  Fp8Quantize q{};
  q.x = x.x;
  q.dtype = x.dtype;
  q.rows = x.rows;
  q.K = x.K;
  q.ld = x.ld;
  q.square = x.square != 0;
  q.data = static_cast<uint8_t *>(x.data);
  q.scales = static_cast<uint8_t *>(x.scales);
  q.t_data = static_cast<uint8_t *>(x.t_data);
  q.t_scales = static_cast<uint8_t *>(x.t_scales);
  return quantize(q, static_cast<cudaStream_t>(stream));
}

int scmp_fp8_dequantize(const void *data, const void *scales, int64_t rows, int64_t K, void *out,
                        int dtype, void *stream) {
  set_last_error("");
  int rc = check_operand(rows, K);
  if (rc != SCMP_OK) return rc;
  if (!known_dtype(dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", dtype);
  if (rows == 0) return SCMP_OK;
  if (!out || !data || !scales) return fail(SCMP_EINVAL, "data, scales and out must be non-NULL");
  if (!aligned({data, scales}, 16))
    return fail(SCMP_EINVAL, "data and scales must be 16-byte aligned");
  if ((rc = check_elements({out}, dtype)) != SCMP_OK) return rc;
  const cudaError_t e = launch_fp8_dequantize(
      static_cast<const uint8_t *>(data), static_cast<const uint8_t *>(scales),
      fp8_layout(rows, K), out, dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "fp8_dequantize launch");
  add_launches(1);
  return SCMP_OK;
}

int scmp_fp8_matmul(const scmp_fp8_matmul_args *args, void *stream) {
  set_last_error("");
  Fp8Product p{};
  const int rc = check_product(args, true, p);
  if (rc != SCMP_OK || p.M == 0 || p.N == 0) return rc;
  return multiply(p, true, static_cast<cudaStream_t>(stream));
}

int scmp_fp8_linear(const void *x, int x_dtype, int64_t ld, const scmp_fp8_matmul_args *args,
                    void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const bool thin =
      args->a ? fp8_thin(args->M, args->N, args->K) : fp8_thin_fits(args->M, args->K);
  Fp8Product p{};
  int rc = check_product(args, !thin, p);
  if (rc != SCMP_OK) return rc;
  if (!known_dtype(x_dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", x_dtype);
  if (ld < p.K) return fail(SCMP_EINVAL, "ld=%lld below K=%lld", (long long)ld, (long long)p.K);
  if (p.M == 0 || p.N == 0) return SCMP_OK;
  if (!x) return fail(SCMP_EINVAL, "x must be non-NULL");
  if ((rc = check_elements({x}, x_dtype)) != SCMP_OK) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (thin) {
    const cudaError_t e = launch_fp8_thin(p, x, x_dtype, ld, s);
    if (e != cudaSuccess) return cuda_fail(e, "fp8_linear launch");
    add_launches(1);
    return SCMP_OK;
  }
  Fp8Quantize q{};
  q.x = x;
  q.dtype = x_dtype;
  q.rows = p.M;
  q.K = p.K;
  q.ld = ld;
  q.data = const_cast<uint8_t *>(p.a);
  q.scales = const_cast<uint8_t *>(p.a_scales);
  rc = quantize(q, s);
  return rc != SCMP_OK ? rc : multiply(p, false, s);
}

size_t scmp_fp8_train_saved_size(int64_t rows, int64_t K) {
  return check_operand(rows, K) != SCMP_OK || rows == 0 ? 0 : operand_bytes(K, rows);
}
size_t scmp_fp8_train_workspace(int64_t M, int64_t N, int64_t K, int backward) {
  if (M <= 0 || check_operand(M, K) != SCMP_OK || N <= 0 || check_operand(N, K) != SCMP_OK)
    return 0;
  return backward ? operand_bytes(M, N) + operand_bytes(N, M) + sums_bytes(M, N)
                  : operand_bytes(M, K) + operand_bytes(N, K);
}

int scmp_fp8_train_forward(const scmp_fp8_train_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_fp8_train_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  int rc;
  if (!known_dtype(x.dtype) || !known_dtype(x.weight_dtype) ||
      (x.bias && !known_dtype(x.bias_dtype)))
    return fail(SCMP_EINVAL, "unknown dtype (x %d, weight %d, bias %d)", x.dtype, x.weight_dtype,
                x.bias_dtype);
  if (x.M <= 0 || x.N <= 0 || (rc = check_operand(x.M, x.K)) != SCMP_OK ||
      (rc = check_operand(x.N, x.K)) != SCMP_OK)
    return fail(SCMP_EINVAL, "bad shape M=%lld N=%lld K=%lld", (long long)x.M, (long long)x.N,
                (long long)x.K);
  if (x.ld < x.K || x.weight_ld < x.K)
    return fail(SCMP_EINVAL, "ld=%lld or weight_ld=%lld below K=%lld", (long long)x.ld,
                (long long)x.weight_ld, (long long)x.K);
  if (!x.x || !x.weight || !x.y) return fail(SCMP_EINVAL, "x, weight and y must be non-NULL");
  if ((rc = check_elements({x.x, x.y}, x.dtype)) != SCMP_OK ||
      (rc = check_elements({x.weight}, x.weight_dtype)) != SCMP_OK ||
      (x.bias && (rc = check_elements({x.bias}, x.bias_dtype)) != SCMP_OK))
    return rc;
  const size_t need = scmp_fp8_train_workspace(x.M, x.N, x.K, 0);
  if (!x.workspace || x.workspace_bytes < need)
    return fail(SCMP_EWORKSPACE, "workspace needs %zu bytes, got %zu", need,
                x.workspace ? x.workspace_bytes : (size_t)0);
  if (!aligned({x.workspace, x.saved_x, x.saved_weight}, 16))
    return fail(SCMP_EINVAL, "workspace and saved codes must be 16-byte aligned");
  auto s = static_cast<cudaStream_t>(stream);
  uint8_t *at = static_cast<uint8_t *>(x.workspace);
  const Operand qx = carve(at, x.M, x.K), qw = carve(at, x.N, x.K);
  Fp8Quantize q{};
  q.x = x.x;
  q.dtype = x.dtype;
  q.rows = x.M;
  q.K = x.K;
  q.ld = x.ld;
  q.data = qx.data;
  q.scales = qx.scales;
  if (x.saved_x) {
    at = static_cast<uint8_t *>(x.saved_x);
    const Operand t = carve(at, x.K, x.M);
    q.t_data = t.data;
    q.t_scales = t.scales;
  }
  if ((rc = quantize(q, s)) != SCMP_OK) return rc;
  q = Fp8Quantize{};
  q.x = x.weight;
  q.dtype = x.weight_dtype;
  q.rows = x.N;
  q.K = x.K;
  q.ld = x.weight_ld;
  q.square = true;
  q.data = qw.data;
  q.scales = qw.scales;
  if (x.saved_weight) {
    at = static_cast<uint8_t *>(x.saved_weight);
    const Operand t = carve(at, x.K, x.N);
    q.t_data = t.data;
    q.t_scales = t.scales;
  }
  if ((rc = quantize(q, s)) != SCMP_OK) return rc;
  Fp8Product p{qx.data, qx.scales, qw.data, qw.scales, x.M, x.N, x.K,
               x.bias, x.bias_dtype, x.y, x.dtype};
  return multiply(p, false, s);
}

int scmp_fp8_train_backward(const scmp_fp8_train_bwd_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_fp8_train_bwd_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  int rc;
  if (!known_dtype(x.dtype) || (x.dweight && !known_dtype(x.weight_dtype)) ||
      (x.dbias && !known_dtype(x.bias_dtype)))
    return fail(SCMP_EINVAL, "unknown dtype (dy %d, weight %d, bias %d)", x.dtype, x.weight_dtype,
                x.bias_dtype);
  if (x.M <= 0 || x.N <= 0 || (rc = check_operand(x.M, x.K)) != SCMP_OK ||
      (rc = check_operand(x.N, x.K)) != SCMP_OK)
    return fail(SCMP_EINVAL, "bad shape M=%lld N=%lld K=%lld", (long long)x.M, (long long)x.N,
                (long long)x.K);
  if (x.ld < x.N) return fail(SCMP_EINVAL, "ld=%lld below N=%lld", (long long)x.ld, (long long)x.N);
  if (!x.dy || (!x.dx && !x.dweight && !x.dbias) || (x.dx && !x.saved_weight) ||
      (x.dweight && !x.saved_x))
    return fail(SCMP_EINVAL, "dy, an output, and what it is made of, must be non-NULL");
  if ((rc = check_elements({x.dy, x.dx}, x.dtype)) != SCMP_OK ||
      (x.dweight && (rc = check_elements({x.dweight}, x.weight_dtype)) != SCMP_OK) ||
      (x.dbias && (rc = check_elements({x.dbias}, x.bias_dtype)) != SCMP_OK))
    return rc;
  const size_t need = scmp_fp8_train_workspace(x.M, x.N, x.K, 1);
  if (!x.workspace || x.workspace_bytes < need)
    return fail(SCMP_EWORKSPACE, "workspace needs %zu bytes, got %zu", need,
                x.workspace ? x.workspace_bytes : (size_t)0);
  if (!aligned({x.workspace, x.saved_x, x.saved_weight}, 16))
    return fail(SCMP_EINVAL, "workspace and saved codes must be 16-byte aligned");
  auto s = static_cast<cudaStream_t>(stream);
  uint8_t *at = static_cast<uint8_t *>(x.workspace);
  const Operand rows = carve(at, x.M, x.N), cols = carve(at, x.N, x.M);
  float *sums = reinterpret_cast<float *>(at);
  Fp8Quantize q{};
  q.x = x.dy;
  q.dtype = x.dtype;
  q.rows = x.M;
  q.K = x.N;
  q.ld = x.ld;
  if (x.dx) {
    q.data = rows.data;
    q.scales = rows.scales;
  }
  if (x.dweight) {
    q.t_data = cols.data;
    q.t_scales = cols.scales;
  }
  q.column_sums = x.dbias ? sums : nullptr;
  if ((rc = quantize(q, s)) != SCMP_OK) return rc;
  if (x.dbias) {
    const cudaError_t e =
        launch_fp8_sum_columns(sums, (x.M + 127) / 128, x.N, x.dbias, x.bias_dtype, s);
    if (e != cudaSuccess) return cuda_fail(e, "fp8_sum_columns launch");
    add_launches(1);
  }
  if (x.dx) {
    uint8_t *w = static_cast<uint8_t *>(const_cast<void *>(x.saved_weight));
    const Operand wt = carve(w, x.K, x.N);
    const Fp8Product p{rows.data, rows.scales, wt.data, wt.scales, x.M, x.K, x.N,
                       nullptr, 0, x.dx, x.dtype};
    if ((rc = multiply(p, false, s)) != SCMP_OK) return rc;
  }
  if (x.dweight) {
    uint8_t *v = static_cast<uint8_t *>(const_cast<void *>(x.saved_x));
    const Operand xt = carve(v, x.K, x.M);
    const Fp8Product p{cols.data, cols.scales, xt.data, xt.scales, x.N, x.K, x.M,
                       nullptr, 0, x.dweight, x.weight_dtype};
    if ((rc = multiply(p, false, s)) != SCMP_OK) return rc;
  }
  return SCMP_OK;
}

int scmp_debug_fp8_plan(int64_t M, int64_t N, int64_t K, int pairs, int32_t *plan) {
  set_last_error("");
  int rc;
  if ((rc = check_operand(M, K)) != SCMP_OK || (rc = check_operand(N, K)) != SCMP_OK) return rc;
  if (M == 0 || N == 0 || pairs < 1 || !plan)
    return fail(SCMP_EINVAL, "fp8_plan takes a product with outputs, pairs >= 1 and a plan");
  const Fp8TilePlan tiles = fp8_tile_plan(M, N, K, pairs);
  plan[0] = fp8_thin(M, N, K) ? 1 : 0;
  plan[1] = tiles.w[0];
  plan[2] = tiles.w[1];
  plan[3] = (int32_t)tiles.units;
  return SCMP_OK;
}

}  // extern "C"
