// C ABI of the 4-bit block operators (declared in include/scmp_b200.h):
// argument checks, layouts and launches.
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "mx_common.cuh"
#include "norm.cuh"
#include "rotary.cuh"
#include "sc_common.cuh"

namespace scmp {
namespace {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}
int cuda_fail(cudaError_t e, const char *what) {
  return fail(SCMP_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr int64_t kMaxRows = INT32_MAX - 1023;  // a tile's coordinates stay 32-bit
constexpr int kMaxScaleExp = 120;        // 2^+-e and its reciprocal are normal fp32 numbers

bool known_dtype(int d) { return d >= SCMP_F32 && d <= SCMP_F16; }
int64_t dtype_bytes(int d) { return d == SCMP_F32 ? 4 : 2; }
bool aligned(std::initializer_list<const void *> ptrs, int64_t to) {
  uintptr_t a = 0;
  for (const void *p : ptrs) a |= reinterpret_cast<uintptr_t>(p);
  return (a & (uintptr_t)(to - 1)) == 0;
}
int check_elements(std::initializer_list<const void *> ptrs, int dtype) {
  if (!aligned(ptrs, dtype_bytes(dtype)))
    return fail(SCMP_EINVAL, "a pointer is not aligned to its elements of %lld bytes",
                (long long)dtype_bytes(dtype));
  return SCMP_OK;
}

int check_mx(int64_t rows, int64_t K, int fmt) {
  if (fmt != SCMP_MXFP4 && fmt != SCMP_NVFP4) return fail(SCMP_EINVAL, "unknown 4-bit format %d", fmt);
  if (rows < 0 || K <= 0 || rows > kMaxRows || K > kMaxRows)
    return fail(SCMP_EINVAL, "bad operand shape [%lld, %lld]", (long long)rows, (long long)K);
  return SCMP_OK;
}
int check_exp(int fmt, int e, int limit) {
  if (fmt == SCMP_MXFP4 ? e != 0 : (e < -limit || e > limit))
    return fail(SCMP_EINVAL, "scale_exp %d: 0 for mxfp4, within +-%d for nvfp4", e, limit);
  return SCMP_OK;
}

// A product's arguments; `codes`: A's buffers are needed.
int check_product(const scmp_mx_matmul_args *args, bool codes, MxProduct &p) {
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_mx_matmul_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  int rc;
  if ((rc = check_mx(x.M, x.K, x.fmt)) != SCMP_OK || (rc = check_mx(x.N, x.K, x.fmt)) != SCMP_OK ||
      (rc = check_exp(x.fmt, x.scale_exp, kMaxScaleExp)) != SCMP_OK)
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
  p.fmt = x.fmt;
  p.alpha = ldexpf(1.0f, x.scale_exp);
  p.bias = x.bias;
  p.bias_dtype = x.bias_dtype;
  p.out = x.out;
  p.out_dtype = x.out_dtype;
  return SCMP_OK;
}

}  // namespace
}  // namespace scmp

using namespace scmp;

extern "C" {

size_t scmp_mx_data_size(int64_t rows, int64_t K, int fmt) {
  if (check_mx(rows, K, fmt) != SCMP_OK) return 0;
  return (size_t)mx_layout(rows, K, fmt).data_bytes();
}
size_t scmp_mx_scale_size(int64_t rows, int64_t K, int fmt) {
  if (check_mx(rows, K, fmt) != SCMP_OK) return 0;
  return (size_t)mx_layout(rows, K, fmt).scale_bytes();
}

int scmp_mx_quantize(const void *x, int dtype, int64_t rows, int64_t K, int64_t ld, int fmt,
                     int scale_exp, void *data, void *scales, void *stream) {
  set_last_error("");
  int rc = check_mx(rows, K, fmt);
  if (rc != SCMP_OK || (rc = check_exp(fmt, scale_exp, kMaxScaleExp)) != SCMP_OK) return rc;
  if (!known_dtype(dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", dtype);
  if (ld < K) return fail(SCMP_EINVAL, "ld=%lld below K=%lld", (long long)ld, (long long)K);
  if (rows == 0) return SCMP_OK;
  if (!x || !data || !scales) return fail(SCMP_EINVAL, "x, data and scales must be non-NULL");
  if (!aligned({data, scales}, 16))
    return fail(SCMP_EINVAL, "data and scales must be 16-byte aligned");
  if ((rc = check_elements({x}, dtype)) != SCMP_OK) return rc;
  const cudaError_t e = launch_mx_quantize(
      x, dtype, ld, mx_layout(rows, K, fmt), fmt, scale_exp, static_cast<uint8_t *>(data),
      static_cast<uint8_t *>(scales), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "mx_quantize launch");
  add_launches(1);
  return SCMP_OK;
}

int scmp_mx_dequantize(const void *data, const void *scales, int64_t rows, int64_t K, int fmt,
                       int scale_exp, void *out, int dtype, void *stream) {
  set_last_error("");
  int rc = check_mx(rows, K, fmt);
  if (rc != SCMP_OK || (rc = check_exp(fmt, scale_exp, kMaxScaleExp)) != SCMP_OK) return rc;
  if (!known_dtype(dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", dtype);
  if (rows == 0) return SCMP_OK;
  if (!out || !data || !scales) return fail(SCMP_EINVAL, "data, scales and out must be non-NULL");
  if (!aligned({data, scales}, 16))
    return fail(SCMP_EINVAL, "data and scales must be 16-byte aligned");
  if ((rc = check_elements({out}, dtype)) != SCMP_OK) return rc;
  const cudaError_t e = launch_mx_dequantize(
      static_cast<const uint8_t *>(data), static_cast<const uint8_t *>(scales),
      mx_layout(rows, K, fmt), fmt, scale_exp, out, dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "mx_dequantize launch");
  add_launches(1);
  return SCMP_OK;
}

int scmp_mx_matmul(const scmp_mx_matmul_args *args, void *stream) {
  set_last_error("");
  MxProduct p{};
  const int rc = check_product(args, true, p);
  if (rc != SCMP_OK || p.M == 0 || p.N == 0) return rc;
  auto s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (mx_thin(p.M, p.N, p.K)) {
    e = launch_mx_thin(p, nullptr, 0, 0, s);
  } else {
    unsigned int *err = device_error_word();
    if (!err) return fail(SCMP_ECUDA, "cannot resolve the engine error word");
    e = launch_mx_matmul(p, err, s);
  }
  if (e != cudaSuccess) return cuda_fail(e, "mx_matmul launch");
  add_launches(1);
  return SCMP_OK;
}

int scmp_mx_linear(const void *x, int x_dtype, int64_t ld, const scmp_mx_matmul_args *args,
                   void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const bool thin = args->a ? mx_thin(args->M, args->N, args->K) : mx_thin_fits(args->M, args->K);
  MxProduct p{};
  int rc = check_product(args, !thin, p);
  if (rc != SCMP_OK) return rc;
  if (!known_dtype(x_dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", x_dtype);
  if (ld < p.K) return fail(SCMP_EINVAL, "ld=%lld below K=%lld", (long long)ld, (long long)p.K);
  if (p.M == 0 || p.N == 0) return SCMP_OK;
  if (!x) return fail(SCMP_EINVAL, "x must be non-NULL");
  if ((rc = check_elements({x}, x_dtype)) != SCMP_OK) return rc;
  if (thin) {
    const cudaError_t e = launch_mx_thin(p, x, x_dtype, ld, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "mx_linear launch");
    add_launches(1);
    return SCMP_OK;
  }
  rc = scmp_mx_quantize(x, x_dtype, p.M, p.K, ld, p.fmt, 0, const_cast<uint8_t *>(p.a),
                        const_cast<uint8_t *>(p.a_scales), stream);
  return rc != SCMP_OK ? rc : scmp_mx_matmul(args, stream);
}

int scmp_debug_mx_plan(int64_t M, int64_t N, int64_t K, int pairs, int32_t *plan) {
  set_last_error("");
  int rc;
  if ((rc = check_mx(M, K, SCMP_MXFP4)) != SCMP_OK || (rc = check_mx(N, K, SCMP_MXFP4)) != SCMP_OK)
    return rc;
  if (M == 0 || N == 0 || pairs < 1 || !plan)
    return fail(SCMP_EINVAL, "mx_plan takes a product with outputs, pairs >= 1 and a plan");
  const MxTilePlan tiles = mx_tile_plan(M, N, pairs);
  plan[0] = mx_thin(M, N, K) ? 1 : 0;
  plan[1] = tiles.nt;
  plan[2] = (int32_t)tiles.tiles;
  return SCMP_OK;
}

int scmp_residual_norm(const scmp_norm_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_norm_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  if (!known_dtype(x.dtype) || (x.param_dtype != x.dtype && x.param_dtype != SCMP_F32))
    return fail(SCMP_EINVAL, "dtype %d with parameters of dtype %d", x.dtype, x.param_dtype);
  if (x.rows < 0 || x.C <= 0 || x.rows > kMaxRows)
    return fail(SCMP_EINVAL, "bad shape rows=%lld C=%lld", (long long)x.rows, (long long)x.C);
  if (x.C > kNormMaxC)
    return fail(SCMP_EUNSUPPORTED, "residual_norm takes rows of up to %lld values, got %lld",
                (long long)kNormMaxC, (long long)x.C);
  if (!(x.eps >= 0.0f)) return fail(SCMP_EINVAL, "eps must be >= 0");
  if (x.rows == 0) return SCMP_OK;
  if (!x.x || !x.weight || (x.y && !x.r) || (!x.h && !x.mx_data))
    return fail(SCMP_EINVAL, "x, weight, an output and, with y, r must be non-NULL");
  if (!x.y && (x.gamma || x.gate || x.post_weight))
    return fail(SCMP_EINVAL, "gamma, gate and post_weight scale y, which is NULL");
  if (x.post_bias && !x.post_weight) return fail(SCMP_EINVAL, "post_bias without post_weight");
  if (x.gate && (x.rows_per_gate <= 0 || x.rows % x.rows_per_gate != 0))
    return fail(SCMP_EINVAL, "rows=%lld is not a multiple of rows_per_gate=%lld",
                (long long)x.rows, (long long)x.rows_per_gate);
  if (!x.mx_data != !x.mx_scales)
    return fail(SCMP_EINVAL, "mx_data and mx_scales go together");
  int rc;
  if ((rc = check_elements({x.x, x.y, x.r}, x.dtype)) != SCMP_OK ||
      (rc = check_elements({x.h}, x.h_f32 ? SCMP_F32 : x.dtype)) != SCMP_OK ||
      (rc = check_elements({x.weight, x.bias, x.gamma, x.gate, x.post_weight, x.post_bias},
                           x.param_dtype)) != SCMP_OK)
    return rc;
  NormParams p{};
  p.x = x.x;
  p.y = x.y;
  p.weight = x.weight;
  p.bias = x.bias;
  p.gamma = x.gamma;
  p.gate = x.gate;
  p.post_weight = x.post_weight;
  p.post_bias = x.post_bias;
  p.r = x.r;
  p.h = x.h;
  p.stats = reinterpret_cast<float2 *>(x.stats);
  p.rows = x.rows;
  p.rows_per_gate = x.gate ? x.rows_per_gate : x.rows;
  p.C = (int)x.C;
  p.eps = x.eps;
  p.rms = x.rms != 0;
  p.h_f32 = x.h_f32 != 0 || x.dtype == SCMP_F32;
  const bool vec = x.C * dtype_bytes(x.dtype) % 16 == 0 &&
                   aligned({x.x, x.y, x.weight, x.bias, x.gamma, x.gate, x.post_weight,
                            x.post_bias, x.r, x.h}, 16);
  if (x.mx_data) {
    if (x.mx_fmt != SCMP_MXFP4 && x.mx_fmt != SCMP_NVFP4)
      return fail(SCMP_EINVAL, "unknown 4-bit format %d", x.mx_fmt);
    if (!vec || !aligned({x.mx_data, x.mx_scales}, 16))
      return fail(SCMP_EUNSUPPORTED,
                  "4-bit output takes rows of whole 16-byte pieces and 16-byte aligned pointers");
    const MxLayout l = mx_layout(x.rows, x.C, x.mx_fmt);
    p.mx_data = static_cast<uint8_t *>(x.mx_data);
    p.mx_scales = static_cast<uint8_t *>(x.mx_scales);
    p.kp = l.kp;
    p.groups = l.groups;
    p.fmt = x.mx_fmt;
  }
  if (!aligned({x.stats}, 8)) return fail(SCMP_EINVAL, "stats must be 8-byte aligned");
  const cudaError_t e =
      launch_residual_norm(p, x.dtype, x.param_dtype, vec, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "residual_norm launch");
  add_launches(1);
  return SCMP_OK;
}

size_t scmp_residual_norm_bwd_workspace(int64_t rows, int64_t C, int64_t rows_per_gate) {
  if (rows <= 0 || C <= 0 || C > kNormMaxC || rows_per_gate <= 0 || rows % rows_per_gate != 0)
    return 0;
  return (size_t)norm_bwd_floats(rows, rows / rows_per_gate, C) * sizeof(float);
}

int scmp_residual_norm_bwd(const scmp_norm_bwd_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_norm_bwd_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  if (!known_dtype(x.dtype) || (x.param_dtype != x.dtype && x.param_dtype != SCMP_F32))
    return fail(SCMP_EINVAL, "dtype %d with parameters of dtype %d", x.dtype, x.param_dtype);
  if (x.rows <= 0 || x.C <= 0 || x.rows > kMaxRows)
    return fail(SCMP_EINVAL, "bad shape rows=%lld C=%lld", (long long)x.rows, (long long)x.C);
  if (x.C > kNormMaxC)
    return fail(SCMP_EUNSUPPORTED, "residual_norm takes rows of up to %lld values, got %lld",
                (long long)kNormMaxC, (long long)x.C);
  if (!x.r || !x.weight || !x.stats)
    return fail(SCMP_EINVAL, "r, weight and stats must be non-NULL");
  if (!x.y && (x.gamma || x.gate || x.post_weight || x.dy || x.dgamma || x.dgate))
    return fail(SCMP_EINVAL, "gamma, gate and post_weight scale y, which is NULL");
  if ((x.post_bias || x.dpost_weight || x.dpost_bias) && !x.post_weight)
    return fail(SCMP_EINVAL, "post_bias without post_weight");
  if (x.dgate && !x.gate) return fail(SCMP_EINVAL, "dgate without gate");
  if (x.gate && (x.rows_per_gate <= 0 || x.rows % x.rows_per_gate != 0))
    return fail(SCMP_EINVAL, "rows=%lld is not a multiple of rows_per_gate=%lld",
                (long long)x.rows, (long long)x.rows_per_gate);
  int rc;
  if ((rc = check_elements({x.r, x.y, x.dr, x.dh, x.dx, x.dy}, x.dtype)) != SCMP_OK ||
      (rc = check_elements({x.weight, x.gamma, x.gate, x.post_weight, x.post_bias, x.dweight,
                            x.dbias, x.dgamma, x.dgate, x.dpost_weight, x.dpost_bias},
                           x.param_dtype)) != SCMP_OK)
    return rc;
  NormBwdParams p{};
  p.r = x.r;
  p.y = x.y;
  p.dr = x.dr;
  p.dh = x.dh;
  p.weight = x.weight;
  p.gamma = x.gamma;
  p.gate = x.gate;
  p.post_weight = x.post_weight;
  p.post_bias = x.post_bias;
  p.stats = reinterpret_cast<const float2 *>(x.stats);
  p.dx = x.dx;
  p.dy = x.dy;
  p.dweight = x.dweight;
  p.dbias = x.dbias;
  p.dgamma = x.dgamma;
  p.dgate = x.dgate;
  p.dpost_weight = x.dpost_weight;
  p.dpost_bias = x.dpost_bias;
  p.rows = x.rows;
  p.groups = x.gate ? x.rows / x.rows_per_gate : 1;
  p.C = (int)x.C;
  p.rms = x.rms != 0;
  if (x.dweight || x.dbias || x.dgamma || x.dgate || x.dpost_weight || x.dpost_bias) {
    const size_t need = (size_t)norm_bwd_floats(p.rows, p.groups, p.C) * sizeof(float);
    if (!x.workspace || x.workspace_bytes < need)
      return fail(SCMP_EWORKSPACE, "workspace needs %zu bytes, got %zu", need,
                  x.workspace ? x.workspace_bytes : (size_t)0);
    p.part = static_cast<float *>(x.workspace);
  }
  if (!aligned({x.stats, x.workspace}, 8))
    return fail(SCMP_EINVAL, "stats and workspace must be 8-byte aligned");
  const bool vec = x.C * dtype_bytes(x.dtype) % 16 == 0 &&
                   aligned({x.r, x.y, x.dr, x.dh, x.weight, x.gamma, x.gate, x.post_weight, x.dx,
                            x.dy}, 16);
  int launches = 0;
  const cudaError_t e = launch_residual_norm_bwd(p, x.dtype, x.param_dtype, vec,
                                                 static_cast<cudaStream_t>(stream), &launches);
  if (e != cudaSuccess) return cuda_fail(e, "residual_norm_bwd launch");
  add_launches((uint64_t)launches);
  return SCMP_OK;
}

int scmp_split_qkv_rotary(const scmp_rotary_args *args, void *stream) {
  set_last_error("");
  if (!args) return fail(SCMP_EINVAL, "args is NULL");
  const scmp_rotary_args &x = *args;
  if (x.abi_version != SCMP_ABI_VERSION)
    return fail(SCMP_EINVAL, "abi_version %d != %d", x.abi_version, SCMP_ABI_VERSION);
  if (!known_dtype(x.dtype)) return fail(SCMP_EINVAL, "unknown dtype %d", x.dtype);
  if (x.B < 0 || x.N < 0 || x.H < 1 || x.Hk < 1 || x.D < 1 || x.H > 65535 || x.Hk > 65535)
    return fail(SCMP_EINVAL, "bad shape B=%lld N=%lld H=%lld Hk=%lld D=%lld", (long long)x.B,
                (long long)x.N, (long long)x.H, (long long)x.Hk, (long long)x.D);
  if (x.H % x.Hk != 0) return fail(SCMP_EINVAL, "H must be a multiple of Hk");
  if (x.D > 256 || x.D % 2 != 0)
    return fail(SCMP_EUNSUPPORTED, "split_qkv_rotary takes even head sizes up to 256, got %lld",
                (long long)x.D);
  if (x.axes < 1 || x.axes > SCMP_MAX_AXES)
    return fail(SCMP_EINVAL, "axes must be 1 to %d, got %d", SCMP_MAX_AXES, x.axes);
  RotaryParams p{};
  int64_t at = 0, turned = 0;
  for (int a = 0; a < x.axes; ++a) {
    if (x.dims[a] < 2 || x.dims[a] > x.D || x.dims[a] % 2 != 0 || x.sizes[a] < 1)
      return fail(SCMP_EINVAL, "axis %d: dims %d (even, >= 2), size %d (>= 1)", a, x.dims[a],
                  x.sizes[a]);
    p.dims[a] = x.dims[a];
    p.sizes[a] = x.sizes[a];
    p.table_at[a] = at;
    turned += x.dims[a];
    at += (int64_t)x.sizes[a] * (x.dims[a] / 2);
  }
  if (turned > x.D) return fail(SCMP_EINVAL, "the axes' dims exceed the head size");
  if (x.B == 0 || x.N == 0) return SCMP_OK;
  // pieces of a head row are counted in 32 bits
  if (x.N > UINT32_MAX / x.D || x.B > UINT32_MAX / x.D / x.N)
    return fail(SCMP_EUNSUPPORTED, "split_qkv_rotary takes up to 2^32 - 1 elements per head, got "
                "B=%lld N=%lld D=%lld tokens", (long long)x.B, (long long)x.N, (long long)x.D);
  if (!x.qkv || !x.q || !x.k || !x.v || !x.table || !x.pos)
    return fail(SCMP_EINVAL, "qkv, q, k, v, table and pos must be non-NULL");
  if (!aligned({x.table}, 8) || !aligned({x.pos}, 4))
    return fail(SCMP_EINVAL, "table must be 8-byte and pos 4-byte aligned");
  const int rc = check_elements({x.qkv, x.q, x.k, x.v}, x.dtype);
  if (rc != SCMP_OK) return rc;
  p.qkv = x.qkv;
  p.q = x.q;
  p.k = x.k;
  p.v = x.v;
  p.table = reinterpret_cast<const float2 *>(x.table);
  p.pos = x.pos;
  p.B = x.B;
  p.N = x.N;
  p.H = x.H;
  p.Hk = x.Hk;
  p.D = (int)x.D;
  p.axes = x.axes;
  p.pos_batched = x.pos_batched != 0;
  p.interleaved = x.interleaved != 0;
  p.v_transposed = x.v_transposed != 0;
  p.inverse = x.inverse != 0;
  const cudaError_t e = launch_rotary(p, x.dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "split_qkv_rotary launch");
  add_launches(1);
  return SCMP_OK;
}

}  // extern "C"
