"""Microscaled 4-bit floating point: quantisation byte for byte against a
search over the representable values in 64 bits, the product against the
64-bit product of the dequantised operands, and the refusals."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

from scmp_vit_b200 import _lib, mx

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([i * 2.0 ** -9 for i in range(8)]
                + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)])[:127]
FMTS = ("mxfp4", "nvfp4")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def nearest(v, grid):
    """Index of the nearest grid entry (ascending), the even one between two."""
    hi = np.searchsorted((grid[1:] + grid[:-1]) / 2, v, side="right")
    lo = np.searchsorted((grid[1:] + grid[:-1]) / 2, v, side="left")
    return np.where((lo != hi) & (lo % 2 == 1), hi, lo)


def quantize_ref(x, fmt, scale_exp=0):
    """(element codes [rows, kp], scale codes [rows, kp / block], values [rows, K])."""
    x = np.asarray(x, dtype=np.float64)
    rows, K = x.shape
    block = _lib.MX_BLOCK[fmt]
    kp = -(-K // 32) * 32
    v = np.zeros((rows, kp))
    v[:, :K] = x
    v = v.reshape(rows, -1, block)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(v).all(-1)
        v = np.where(bad[..., None], 0.0, v)
        amax = np.abs(v).max(-1)
    if fmt == "mxfp4":
        _, e = np.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
        e = np.maximum(np.where(amax > 0, e - 3, -127), -127)
        scale, step = e + 127, 2.0 ** e.astype(np.float64)
    else:
        # a sixth in fp32: the scale is a choice, and this product is its definition
        with np.errstate(over="ignore"):
            sixth = (amax / 2.0 ** scale_exp).astype(np.float32) * np.float32(1 / 6)
        scale = nearest(np.minimum(sixth.astype(np.float64), 448.0), E4M3)
        step = E4M3[scale] * 2.0 ** scale_exp
    mag = np.where(step[..., None] > 0, np.abs(v) / np.where(step > 0, step, 1)[..., None], 0)
    code = nearest(mag, E2M1)
    value = E2M1[code] * step[..., None] * np.where(np.signbit(v), -1, 1)
    value[bad] = np.nan
    code = code + 8 * np.signbit(v)
    code[bad] = 0
    scale = np.where(bad, 0xFF if fmt == "mxfp4" else 0x7F, scale)
    return code.reshape(rows, kp), scale, value.reshape(rows, kp)[:, :K]


def pack_ref(code, scale):
    """The bytes of the documented layout."""
    rows, nb = scale.shape
    data = (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)
    groups = -(-nb // 4)
    out = np.zeros((-(-rows // 128), groups, 512), dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scale
    return data.reshape(-1), out.reshape(-1)


# ------------------------------------------------------------ CPU: refusals

def test_sizes():
    lib = _lib.load()
    for fmt, code in _lib.MX_FORMAT.items():
        for rows, K in ((0, 5), (1, 1), (128, 32), (129, 33), (257, 1024)):
            kp = -(-K // 32) * 32
            assert lib.scmp_mx_data_size(rows, K, code) == rows * kp // 2
            groups = -(-kp // (4 * _lib.MX_BLOCK[fmt]))
            assert lib.scmp_mx_scale_size(rows, K, code) == -(-rows // 128) * groups * 512
    for rows, K, code in ((-1, 4, 0), (4, 0, 0), (4, 4, 2), (1 << 31, 4, 0), (4, 1 << 31, 1),
                          ((1 << 31) - 1, 4, 0)):
        assert lib.scmp_mx_data_size(rows, K, code) == 0
        assert lib.scmp_mx_scale_size(rows, K, code) == 0


@pytest.mark.parametrize("pack,cls", [
    (_lib.PACK_MX_MATMUL, _lib.MxMatmulArgs), (_lib.PACK_NORM, _lib.NormArgs),
    (_lib.PACK_NORM_BWD, _lib.NormBwdArgs), (_lib.PACK_ROTARY, _lib.RotaryArgs)])
def test_packed_arguments_are_the_structs(pack, cls):
    a, values, n = cls(), [], 0
    for name, kind in cls._fields_:
        for i in range(getattr(kind, "_length_", 0) or 1):
            n += 1
            v = n / 4 if kind is ctypes.c_float else n
            values.append(v)
            if hasattr(kind, "_length_"):
                getattr(a, name)[i] = v
            else:
                setattr(a, name, v)
    assert pack.pack(*values) == bytes(a)


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_lib.MxMatmulArgs) == 8 + 32 + 24 + 8 + 16 + 8
    assert ctypes.sizeof(_lib.NormArgs) == 16 + 13 * 8 + 24 + 16
    assert ctypes.sizeof(_lib.NormBwdArgs) == 16 + 19 * 8 + 8 + 24
    assert ctypes.sizeof(_lib.RotaryArgs) == 8 + 48 + 40 + 4 + 32 + 16 + 12


@pytest.mark.parametrize("args,msg", [
    (dict(fmt=7), "format"),
    (dict(rows=-1), "shape"),
    (dict(K=0), "shape"),
    (dict(dtype=3), "dtype"),
    (dict(ld=7), "ld"),
    (dict(fmt=0, scale_exp=1), "scale_exp"),
    (dict(fmt=1, scale_exp=121), "scale_exp"),
    (dict(x=0), "non-NULL"),
    (dict(data=0), "non-NULL"),
    (dict(data=24), "aligned"),
    (dict(scales=8), "aligned"),
    (dict(x=18), "aligned to its elements"),
    (dict(x=17, dtype=1), "aligned to its elements"),
])
def test_quantize_refusals(args, msg):
    a = dict(x=16, dtype=0, rows=4, K=8, ld=8, fmt=0, scale_exp=0, data=16, scales=16)
    a.update(args)
    lib = _lib.load()
    assert lib.scmp_mx_quantize(a["x"], a["dtype"], a["rows"], a["K"], a["ld"], a["fmt"],
                                a["scale_exp"], a["data"], a["scales"], None) == -1
    assert msg in _lib.last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(x_dtype=3), "dtype"),
    (dict(ld=31), "ld"),
    (dict(x=None), "non-NULL"),
    (dict(M=5, a=None), "non-NULL"),       # past the rows that need no buffers
    (dict(K=6400, ld=6400, a=None), "non-NULL"),
    (dict(fmt=1, scale_exp=200), "scale_exp"),
    (dict(x=18), "aligned to its elements"),
])
def test_linear_refusals(args, msg):
    a = _lib.MxMatmulArgs()
    a.abi_version, a.M, a.N, a.K = _lib.ABI_VERSION, 4, 4, 32
    a.a = a.a_scales = a.b = a.b_scales = a.out = 16
    call = dict(x=16, x_dtype=0, ld=32)
    for k, v in args.items():
        if k in call:
            call[k] = v
        else:
            setattr(a, k, v)
    assert _lib.load().scmp_mx_linear(call["x"], call["x_dtype"], call["ld"], ctypes.byref(a),
                                      None) == -1
    assert msg in _lib.last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(abi_version=9), "abi_version"),
    (dict(fmt=2), "format"),
    (dict(M=-1), "shape"),
    (dict(K=0), "shape"),
    (dict(scale_exp=3), "scale_exp"),
    (dict(out_dtype=5), "dtype"),
    (dict(bias=16, bias_dtype=4), "dtype"),
    (dict(a=None), "non-NULL"),
    (dict(out=None), "non-NULL"),
    (dict(b_scales=8), "aligned"),
    (dict(out=18), "aligned to its elements"),
    (dict(bias=17, bias_dtype=2), "aligned to its elements"),
])
def test_matmul_refusals(args, msg):
    a = _lib.MxMatmulArgs()
    a.abi_version, a.M, a.N, a.K = _lib.ABI_VERSION, 4, 4, 32
    a.a = a.a_scales = a.b = a.b_scales = a.out = 16
    for k, v in args.items():
        setattr(a, k, v)
    assert _lib.load().scmp_mx_matmul(ctypes.byref(a), None) == -1
    assert msg in _lib.last_error()


def test_copies_are_tensors_of_their_own():
    """A copied or loaded MXTensor points at its own bytes, not at the first one's."""
    q = mx.mx_empty(torch.Size((5, 40)), "nvfp4", torch.device("cpu"), torch.bfloat16, 3)
    q.data.copy_(torch.arange(q.data.numel()) % 251)
    q.scales.copy_(torch.arange(q.scales.numel()) % 127)
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert c.data_ptr == c.data.data_ptr() and c.scales_ptr == c.scales.data_ptr()
        assert c.data_ptr != q.data_ptr and c.scales_ptr != q.scales_ptr
        assert torch.equal(c.data, q.data) and torch.equal(c.scales, q.scales)
        assert (c.shape, c.rows, c.fmt, c.scale_exp, c.dtype) == ((5, 40), 5, "nvfp4", 3,
                                                                   torch.bfloat16)
    assert copy.copy(q).data_ptr == q.data_ptr


def test_python_refusals_on_cpu():
    with pytest.raises(RuntimeError, match="no CPU path"):
        mx.mx_quantize(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="format"):
        mx.mx_quantize(torch.zeros(4, 32), "fp4")
    with pytest.raises(ValueError, match="scale_exp"):
        mx.MXTensor(torch.zeros(64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8),
                    (4, 32), "nvfp4", 1 << 32)
    with pytest.raises(TypeError, match="float32"):
        mx.mx_quantize(torch.zeros(4, 32, dtype=torch.int32))
    with pytest.raises(TypeError, match="MXTensor"):
        mx.mx_matmul(torch.zeros(4, 32), torch.zeros(4, 32))
    with pytest.raises(ValueError, match="contiguous bytes"):
        mx.MXTensor(torch.zeros(3, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8),
                    (4, 32), "mxfp4")


# ------------------------------------------------------------ GPU: quantise

def special_rows(K):
    """Rows that borders, ends of ranges and odd values decide."""
    g = torch.Generator().manual_seed(K)
    rows = [torch.zeros(K), torch.full((K,), -0.0), torch.full((K,), 1e-45),
            torch.full((K,), 3.0e38), torch.randn(K, generator=g) * 1e-40,
            torch.randn(K, generator=g) * 2.0 ** -125, torch.randn(K, generator=g) * 1e37]
    ties = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75,
                         -2.5, -3.5, -5.0, 0.5])
    for s in (1.0, 1.125, 0.8125, 2.0 ** -9, 448.0, 7.0):  # e4m3 steps; 7 makes mxfp4 saturate
        rows.append((ties.repeat(K // 16 + 1) * s)[:K])
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.randn(K, generator=g)
        r[K // 2] = bad
        rows.append(r)
    return torch.stack(rows)


def check_quantize(x, fmt, scale_exp=0):
    q = mx.mx_quantize(x, fmt, scale_exp=scale_exp)
    values = q.dequantize(torch.float32)
    torch.cuda.synchronize()
    x2 = x.detach().cpu().reshape(-1, x.shape[-1])
    code, scale, value = quantize_ref(x2.double().numpy(), fmt, scale_exp)
    data, scales = pack_ref(code, scale)
    assert np.array_equal(q.data.cpu().numpy(), data)
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    got = values.cpu().double().numpy().reshape(value.shape)
    assert np.array_equal(got, value, equal_nan=True)
    return q


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (2, 31), (3, 33), (130, 64), (5, 257),
                                    (129, 100), (257, 1024), (4, 4104), (33, 520)])
def test_quantize_bytes(cuda_device, fmt, rows, K):
    g = torch.Generator().manual_seed(rows * 1000 + K)
    for dtype in DTYPES:
        x = torch.randn(rows, K, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
        check_quantize(x.to(dtype).to(cuda_device), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,scale_exp", [("mxfp4", 0), ("nvfp4", 0), ("nvfp4", -11),
                                           ("nvfp4", 5), ("nvfp4", 120), ("nvfp4", -120)])
@pytest.mark.parametrize("K", [16, 47, 256])
def test_quantize_special_values(cuda_device, fmt, scale_exp, K):
    x = special_rows(K).to(cuda_device)
    check_quantize(x, fmt, scale_exp)
    check_quantize(x.to(torch.bfloat16), fmt, scale_exp)
    check_quantize(x.to(torch.float16), fmt, scale_exp)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_strides_and_shapes(cuda_device, fmt):
    x = torch.randn(6, 40, 96, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    check_quantize(x, fmt)
    check_quantize(x[:, ::3, 1:65], fmt)               # strided rows at an odd offset
    check_quantize(x[:, :, ::2], fmt)                  # strided elements
    check_quantize(x.transpose(0, 2), fmt)
    check_quantize(x[0, :1].expand(5, 96), fmt)        # one row five times
    check_quantize(x[2, 3], fmt)                       # one dimension
    empty = mx.mx_quantize(x[:0], fmt)
    assert empty.shape == (0, 40, 96) and empty.dequantize().shape == (0, 40, 96)
    r = mx.mx_quantize(x, fmt).reshape(-1, 96)
    assert r.shape == (240, 96)
    assert torch.equal(r.dequantize(), mx.mx_quantize(x, fmt).dequantize().reshape(240, 96))
    with pytest.raises(ValueError, match="last dimension"):
        r.reshape(96, 240)


@pytest.mark.gpu
def test_values_fit_the_types_they_came_from(cuda_device):
    """Two significant bits (mxfp4) or six (nvfp4): exact in 16-bit types."""
    for fmt in FMTS:
        for dtype in DTYPES:
            x = torch.randn(64, 96, generator=torch.Generator().manual_seed(2)).to(dtype)
            q = mx.mx_quantize(x.to(cuda_device), fmt)
            assert torch.equal(q.dequantize().float(), q.dequantize(torch.float32))


# ------------------------------------------------------------- GPU: product

def product_bound(a, b, y, out_dtype):
    """|error| allowed for fp32 sums of exact products in any order, each
    addition off by at most one unit in the last place (2^-23 of the running
    magnitude, itself at most sum |a||b|), plus the final rounding."""
    K = a.shape[-1]
    return (K + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t() + y.abs()) + \
        torch.finfo(out_dtype).eps / 2 * y.abs()


def check_product(a, w, fmt, dtype, bias=None, w_exp=0):
    qa = mx.mx_quantize(a, fmt)
    qw = mx.mx_quantize(w, fmt, scale_exp=w_exp)
    y = mx.mx_matmul(a, qw, bias=bias, out_dtype=dtype)
    y2 = mx.mx_matmul(qa, qw, bias=bias, out_dtype=dtype)
    torch.cuda.synchronize()
    assert _lib.engine_status() == 0
    va = qa.dequantize(torch.float32).double().reshape(-1, a.shape[-1])
    vw = qw.dequantize(torch.float32).double()
    ref = va @ vw.t()
    if bias is not None:
        ref = ref + bias.double()
    bound = product_bound(va, vw, ref, dtype)
    if dtype == torch.float16:
        ref = ref.clamp(-65504, 65504)
    for got in (y, y2):
        assert got.dtype == dtype and got.shape == (*a.shape[:-1], w.shape[0])
        err = (got.double().reshape(ref.shape) - ref).abs()
        assert bool((err <= bound).all()), (err / bound).max()
    return y


SHAPES = [(1, 1, 1), (1, 48, 32), (3, 5, 7), (2, 130, 96), (1, 300, 6144), (2, 9, 6145),
          (4, 1030, 1025), (5, 64, 96), (7, 64, 4104), (16, 40, 64), (32, 40, 64), (17, 200, 64),
          (33, 257, 100), (127, 128, 128), (129, 257, 260), (257, 1024, 1024), (200, 511, 352),
          (193, 264, 544), (385, 520, 2080), (64, 4096, 1024), (600, 96, 40), (1500, 300, 288)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul(cuda_device, fmt, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    a = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g)))
    w = torch.randn(N, K, generator=g) * 0.05
    bias = torch.randn(N, generator=g)
    exp = -12 if fmt == "nvfp4" else 0
    for dtype in DTYPES:
        check_product(a.to(dtype).to(cuda_device), w.to(cuda_device), fmt, dtype,
                      bias.to(dtype).to(cuda_device), exp)
    check_product(a.to(cuda_device), w.to(cuda_device), fmt, torch.float32, None, exp)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 96, 96), (5, 40, 200), (300, 256, 160)])
def test_matmul_not_finite(cuda_device, fmt, M, N, K):
    """A block that is not finite makes its own row (column) NaN and leaves
    every other output as it is."""
    g = torch.Generator().manual_seed(9)
    a, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    clean = mx.mx_matmul(a.to(cuda_device), mx.mx_quantize(w.to(cuda_device), fmt))
    a[M // 2, K - 1] = float("inf")
    w[3, 0] = float("nan")
    got = mx.mx_matmul(a.to(cuda_device), mx.mx_quantize(w.to(cuda_device), fmt))
    assert bool(got[M // 2].isnan().all()) and bool(got[:, 3].isnan().all())
    keep_m = torch.arange(M) != M // 2
    keep_n = torch.arange(N) != 3
    assert torch.equal(got[keep_m][:, keep_n], clean[keep_m][:, keep_n])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_matmul_wide_scales(cuda_device, M):
    """Blocks of one row many powers of two apart: the largest decides."""
    g = torch.Generator().manual_seed(5)
    a, w = torch.randn(M, 256, generator=g), torch.randn(80, 256, generator=g)
    a[:, :32] *= 2.0 ** 40
    w[:, 32:64] *= 2.0 ** -60
    check_product(a.to(cuda_device), w.to(cuda_device), "mxfp4", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 16390, 1024), (2, 4104, 2048), (4, 4096, 1024)])
def test_few_rows_long_weight(cuda_device, fmt, M, N, K):
    """Few rows of a long weight go through the tensor-core tiles; without
    buffers for their codes the one launch takes them all the same."""
    g = torch.Generator().manual_seed(10)
    a, w = torch.randn(M, K, generator=g).to(cuda_device), torch.randn(N, K, generator=g)
    w = w.to(cuda_device)
    y = check_product(a, w, fmt, torch.float32)
    q, qa = mx.mx_quantize(w, fmt), mx.mx_quantize(a, fmt)
    launches = _lib.kernel_launches()
    mx.mx_matmul(a, q)
    assert _lib.kernel_launches() - launches == 2
    out = torch.empty(M, N, device=cuda_device)
    args = _lib.MxMatmulArgs(_lib.ABI_VERSION, _lib.MX_FORMAT[fmt], None, None, q.data_ptr,
                             q.scales_ptr, M, N, K, 0, 0, None, out.data_ptr(), 0, 0)
    launches = _lib.kernel_launches()
    _lib.check(_lib.load().scmp_mx_linear(
        a.data_ptr(), 0, K, ctypes.byref(args),
        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert _lib.kernel_launches() - launches == 1
    va, vw = (t.dequantize().double() for t in (qa, q))
    ref = va @ vw.t()
    for got in (y, out):
        assert bool(((got.double() - ref).abs() <= product_bound(va, vw, ref, got.dtype)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 4, 40, 300])
@pytest.mark.parametrize("big,small", [(2.0 ** 120, 2.0 ** -110), (2.0 ** -110, 2.0 ** 120)])
def test_matmul_scales_that_meet(cuda_device, M, big, small):
    """Scales near both ends of fp32 whose products are ordinary numbers: no step
    on the way overflows."""
    g = torch.Generator().manual_seed(8)
    a, w = torch.randn(M, 256, generator=g) * big, torch.randn(80, 256, generator=g) * small
    check_product(a.to(cuda_device), w.to(cuda_device), "mxfp4", torch.float32)


@pytest.mark.gpu
def test_matmul_out_counts_as_a_write(cuda_device):
    """autograd notices that a tensor it saved was written, and out that shares
    memory with an input is refused."""
    w = mx.mx_quantize(torch.randn(64, 64, device=cuda_device))
    leaf = torch.randn(3, 64, device=cuda_device, requires_grad=True)
    out = torch.randn(3, 64, device=cuda_device)
    y = (leaf * out).sum()
    with torch.no_grad():
        mx.mx_matmul(leaf, w, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    buf = torch.randn(7, 64, device=cuda_device)
    with pytest.raises(ValueError, match="shares memory"):
        mx.mx_matmul(buf[:3], w, out=buf[:3])
    with pytest.raises(ValueError, match="shares memory"):
        mx.mx_matmul(buf[:3], w, out=buf[2:5])
    with pytest.raises(ValueError, match="shares memory"):
        mx.mx_matmul(buf[:3], w, out=buf[4:7], bias=buf[6])
    assert torch.equal(mx.mx_matmul(buf[:3], w, out=buf[3:6]), mx.mx_matmul(buf[:3], w))


@pytest.mark.gpu
def test_matmul_empty_and_out(cuda_device):
    w = mx.mx_quantize(torch.randn(24, 64, device=cuda_device))
    x = torch.randn(3, 5, 64, device=cuda_device)
    assert mx.mx_matmul(x[:0], w).shape == (0, 5, 24)
    none = mx.mx_quantize(torch.zeros(0, 64, device=cuda_device))
    assert mx.mx_matmul(x, none).shape == (3, 5, 0)
    # an output one element off 16-byte alignment, with guards on both sides
    buf = torch.full((3 * 5 * 24 + 2,), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = buf[1:-1].view(3, 5, 24)
    assert mx.mx_matmul(x, w, out=out) is out
    ref = mx.mx_matmul(x, w, out_dtype=torch.bfloat16)
    assert torch.equal(out, ref) and buf[0] == 7 and buf[-1] == 7


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,K", [(1, 130), (3, 200), (4, 4100), (70, 130)])
def test_matmul_strided_rows(cuda_device, fmt, M, K):
    """Rows a distance apart, at offsets off every alignment; a transposed bias."""
    g = torch.Generator().manual_seed(6)
    big = torch.randn(M, K + 37, generator=g).to(cuda_device)
    w = mx.mx_quantize(torch.randn(48, K, generator=g).to(cuda_device), fmt)
    bias = torch.randn(48, 2, generator=g).to(cuda_device)[:, 1]
    for dtype in DTYPES:
        for at in (0, 1, 8):
            a = big.to(dtype)[:, at:at + K]
            assert torch.equal(mx.mx_matmul(a, w, bias=bias),
                               mx.mx_matmul(a.clone(), w, bias=bias.clone()))


@pytest.mark.gpu
def test_matmul_repeats_bit_for_bit(cuda_device):
    """A call made again gives the same bits."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(700, 512, generator=g).to(cuda_device)
    w = mx.mx_quantize(torch.randn(384, 512, generator=g).to(cuda_device))
    full = mx.mx_matmul(x, w)
    assert torch.equal(full, mx.mx_matmul(x, w))


@pytest.mark.gpu
def test_python_refusals(cuda_device):
    w = mx.mx_quantize(torch.randn(24, 64, device=cuda_device))
    x = torch.randn(4, 64, device=cuda_device)
    with pytest.raises(ValueError, match="inner-dim"):
        mx.mx_matmul(x[:, :32], w)
    with pytest.raises(ValueError, match="formats"):
        mx.mx_matmul(mx.mx_quantize(x, "nvfp4"), w)
    with pytest.raises(ValueError, match="bias"):
        mx.mx_matmul(x, w, bias=torch.zeros(23, device=cuda_device))
    with pytest.raises(TypeError, match="bias"):
        mx.mx_matmul(x, w, bias=torch.zeros(24, device=cuda_device, dtype=torch.float64))
    with pytest.raises(TypeError, match="out"):
        mx.mx_matmul(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="out must"):
        mx.mx_matmul(x, w, out=torch.empty(4, 23, device=cuda_device))
    with pytest.raises(ValueError, match="devices"):
        mx.mx_matmul(x.cpu(), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.mx_matmul(x.clone().requires_grad_(), w)
    with torch.no_grad():
        mx.mx_matmul(x.clone().requires_grad_(), w)
    with pytest.raises(_lib.EngineError, match="scale_exp"):
        mx.mx_quantize(x, "mxfp4", scale_exp=2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_linear(cuda_device, fmt):
    lin = torch.nn.Linear(96, 72).to(cuda_device)
    m = mx.MXLinear(lin, fmt)
    x = torch.randn(2, 11, 96, device=cuda_device)
    ref = mx.mx_matmul(x, mx.mx_quantize(lin.weight.detach(), fmt, scale_exp=m.scale_exp),
                       bias=lin.bias.detach())
    assert torch.equal(m(x), ref)
    assert torch.equal(m(mx.mx_quantize(x, fmt)), ref)
    again = mx.MXLinear(torch.nn.Linear(96, 72).to(cuda_device), fmt)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), ref)
    other = mx.MXLinear(torch.nn.Linear(96, 72).to(cuda_device), FMTS[1 - FMTS.index(fmt)])
    with pytest.raises((ValueError, RuntimeError)):
        other.load_state_dict(m.state_dict())


@pytest.mark.gpu
def test_streams_and_graph(cuda_device):
    """A call on a side stream, and one captured and replayed on new inputs."""
    g = torch.Generator().manual_seed(4)
    w = mx.mx_quantize(torch.randn(160, 128, generator=g).to(cuda_device))
    xs = [torch.randn(m, 128, generator=g).to(cuda_device) for m in (1, 300)]
    for x in xs:
        ref = mx.mx_matmul(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = mx.mx_matmul(x, w)
        side.synchronize()
        assert torch.equal(got, ref)
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mx.mx_matmul(static, w)
        static.copy_(x * 2 + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mx.mx_matmul(x * 2 + 1, w))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_matmul_bounded_wait_gives_up_and_recovers(cuda_device, fmt):
    """With the loaders held on a flag that nothing sets, every wait runs out
    after its (shortened) limit, the launch returns and says so, and the next
    call on the same context is right."""
    g = torch.Generator().manual_seed(8)
    a, w = torch.randn(300, 320, generator=g), torch.randn(300, 320, generator=g)
    a, w = a.to(cuda_device), w.to(cuda_device)
    qa, qw = mx.mx_quantize(a, fmt), mx.mx_quantize(w, fmt)
    torch.cuda.synchronize()
    _lib.engine_status(reset=True)
    _lib.set_wait_limit(20_000_000)
    _lib.hold_producers(True)
    try:
        mx.mx_matmul(qa, qw)
        torch.cuda.synchronize()
        status = _lib.engine_status(reset=True)
    finally:
        _lib.hold_producers(False)
        _lib.set_wait_limit(2_000_000_000)
    assert status & 1
    check_product(a, w, fmt, torch.float32)


# --------------------------------------------------- CPU: tensors and modules

@pytest.mark.parametrize("shape", [(4, 0), (0, 0), (0,), (), (-4, 32), (2, -2, 32), (4, -32)])
def test_tensor_refuses_shapes_without_columns(shape):
    """A product would divide by the last dimension."""
    data, scales = torch.zeros(0, dtype=torch.uint8), torch.zeros(0, dtype=torch.uint8)
    with pytest.raises(ValueError, match="last dimension"):
        mx.MXTensor(data, scales, shape, "mxfp4")
    assert mx.MXTensor(data, scales, (0, 32), "mxfp4").rows == 0


def linear_on_cpu(monkeypatch, fmt="mxfp4"):
    monkeypatch.setattr(mx, "mx_quantize", lambda w, fmt, scale_exp: mx.mx_empty(
        w.shape, fmt, w.device, w.dtype, scale_exp))
    return mx.MXLinear(torch.nn.Linear(96, 72), fmt)


@pytest.mark.parametrize("name", ["data", "scales"])
@pytest.mark.parametrize("change", [
    lambda t: t.float(), lambda t: torch.zeros(1, dtype=torch.uint8).expand(t.shape),
    lambda t: torch.cat([t, t])[::2],
])
def test_linear_refuses_buffers_of_another_kind(monkeypatch, name, change):
    """``load_state_dict(assign=True)`` takes the given tensors themselves, of any
    type and stride; the kernels would read them as the packed layout."""
    m = linear_on_cpu(monkeypatch)
    state = m.state_dict()
    state[name] = change(state[name])
    m.load_state_dict(state, assign=True)
    with pytest.raises(ValueError, match="contiguous bytes"):
        m.quantized_weight()
    m.load_state_dict(linear_on_cpu(monkeypatch).state_dict(), assign=True)
    assert m.quantized_weight().shape == (72, 96)
    setattr(m, name, getattr(m, name)[:-16])
    with pytest.raises(ValueError, match="contiguous bytes"):
        m.quantized_weight()


def test_out_shares_no_memory_with_codes(monkeypatch):
    """Outputs written while codes are still read; refused before any launch."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    launched = []
    monkeypatch.setattr(mx, "call", lambda *a: launched.append(a))
    cpu = torch.device("cpu")
    a = mx.mx_empty(torch.Size((256, 64)), "nvfp4", cpu, torch.bfloat16)
    b = mx.mx_empty(torch.Size((16, 64)), "nvfp4", cpu, torch.bfloat16)
    few = mx.mx_empty(torch.Size((16, 64)), "nvfp4", cpu, torch.bfloat16)
    for x, q in ((a, a), (few, b)):
        size = 2 * x.rows * 16
        for part in (q.data, q.scales):
            memory = torch.empty(0, dtype=torch.uint8).set_(part.untyped_storage())
            at = min(part.storage_offset(), memory.numel() - size)
            out = memory[at:at + size].view(torch.bfloat16).view(x.rows, 16)
            with pytest.raises(ValueError, match="shares memory"):
                mx.mx_matmul(x, b, out=out)
    with pytest.raises(ValueError, match="shares memory"):
        mx.mx_matmul(torch.zeros(16, 64).bfloat16(), b, out=out)
    assert launched == []
    out = torch.empty(256, 16, dtype=torch.bfloat16)
    assert mx.mx_matmul(a, b, out=out) is out and len(launched) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("scale_exp", [120, 119, 0, -120])
def test_dequantize_ends_of_the_range(cuda_device, scale_exp):
    """Every scale code under the largest and smallest tensor scales: the values
    that fp32 holds are exact, zero codes are zero whatever their scale."""
    code = np.tile(np.arange(16), (128, 2))                # a row: two blocks of all codes
    scale = np.stack([np.arange(128), np.arange(128)[::-1]], 1)  # 0x7F is NaN
    data, scales = pack_ref(code, scale)
    q = mx.MXTensor(torch.from_numpy(data).to(cuda_device),
                    torch.from_numpy(scales).to(cuda_device), (128, 32), "nvfp4", scale_exp)
    value = np.append(E4M3, np.nan)[scale] * 2.0 ** scale_exp
    ref = np.repeat(value, 16, 1) * E2M1[code % 8] * np.where(code < 8, 1, -1)
    ref = torch.from_numpy(ref)
    for dtype in DTYPES:
        got = q.dequantize(dtype).cpu()
        want = ref.to(torch.float32).to(dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0, posinf=None, neginf=None),
                           want.nan_to_num(nan=0.0, posinf=None, neginf=None))
        assert torch.equal(got.isinf(), want.isinf())


# ------------------------------------- the variants that large calls take
# Tiles: a pair of CTAs that goes from tile to tile uses its second accumulator,
# hands accumulators back and carries the ring's phases on; 128 and 192 rows a
# tile read scales of two row groups and store a second and a third piece.

# M, N, K, rows per tile and tiles per pair (at least) on 74 pairs
MANY_TILES = [(16448, 1040, 288, 192, 5),   # rows of whole 16-byte pieces: TMA stores
              (20000, 1030, 96, 192, 7),    # two features a store
              (12000, 2049, 544, 192, 7),   # one feature a store
              (30000, 1040, 40, 192, 10),   # one stage a tile, mostly past K
              (3000, 8200, 64, 192, 7),
              (2000, 2056, 1100, 128, 1.9),
              (1800, 4102, 64, 128, 3),
              (1700, 4099, 2600, 128, 3),   # eleven stages a tile: the ring wraps inside it
              (3500, 1000, 2600, 64, 2.9),
              (800, 4101, 160, 64, 2.9),
              (1300, 4100, 1024, 192, 1.6)]


def test_many_tiles_are_many():
    for M, N, K, nt, each in MANY_TILES:
        few, rows, tiles = _lib.mx_plan(M, N, K)
        assert not few and rows == nt and tiles >= 74 * each, (M, N, K, rows, tiles)


def test_few_rows_rule():
    """``mx._thin`` (no buffers asked for) is the engine's own rule."""
    sizes = [*range(1, 200, 13), *range(200, 20000, 331), *(1024 * i for i in range(1, 40))]
    for K in (1, 31, 32, 1000, 1024, 2048, 4096, 5000, 6143, 6144, 6145, 8192):
        for M in range(1, 7):
            for N in sizes:
                assert mx._thin(M, N, K) == _lib.mx_plan(M, N, K)[0], (M, N, K)


@pytest.mark.parametrize("M,N,K,pairs", [(0, 4, 4, 74), (4, 0, 4, 74), (4, 4, 0, 74),
                                         (4, 4, 4, 0), (-1, 4, 4, 74)])
def test_plan_refusals(M, N, K, pairs):
    with pytest.raises(_lib.EngineError):
        _lib.mx_plan(M, N, K, pairs)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [s[:3] for s in MANY_TILES])
def test_matmul_many_tiles(cuda_device, fmt, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    a = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    w = (torch.randn(N, K, generator=g) * 0.05).to(cuda_device)
    bias = torch.randn(N, generator=g).to(cuda_device)
    exp = -12 if fmt == "nvfp4" else 0
    for dtype in DTYPES:
        x = a.to(dtype).to(cuda_device)
        y = check_product(x, w, fmt, dtype, bias.to(dtype), exp)
        # a row's result does not depend on the rows around it, nor on its tile
        q = mx.mx_quantize(w, fmt, scale_exp=exp)
        for at in (0, M // 2 + 1, M - 70):
            assert torch.equal(mx.mx_matmul(x[at:at + 70], q, bias=bias.to(dtype)), y[at:at + 70])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_many_tiles_repeat_and_keep_to_their_rows(cuda_device, fmt):
    """The same bits again, and guards around an output whose last tile is cut."""
    M, N, K = 16449, 1040, 288
    x = torch.randn(M, K, device=cuda_device).bfloat16()
    w = mx.mx_quantize(torch.randn(N, K, device=cuda_device), fmt)
    first = mx.mx_matmul(x, w)
    for dtype, pad in ((torch.bfloat16, 64), (torch.bfloat16, 1), (torch.float32, 3)):
        buf = torch.full((M * N + 2 * pad,), 7.0, dtype=dtype, device=cuda_device)
        out = buf[pad:-pad].view(M, N)
        mx.mx_matmul(x, w, out=out)
        assert torch.equal(out.bfloat16(), first)
        assert bool((buf[:pad] == 7).all()) and bool((buf[-pad:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,K,dtypes", [
    (1300, 1056, DTYPES), (1300, 1057, DTYPES),   # four chunks a warp, whole and odd rows
    (2600, 4104, DTYPES[1:2]),                    # several units a row
    (19500, 520, DTYPES[:1]),                     # more units than warps
])
def test_quantize_bytes_many_rows(cuda_device, fmt, rows, K, dtypes):
    g = torch.Generator().manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    for dtype in dtypes:
        q = check_quantize(x.to(dtype).to(cuda_device), fmt)
        values = q.dequantize(torch.float32)      # (compared with the reference above)
        for to in DTYPES[1:]:
            # (fp16 inputs past their range are infinities: blocks of NaN)
            assert torch.allclose(q.dequantize(to), values.to(to), rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
def test_captured_product_behind_two_streams(cuda_device):
    """A captured product whose operands come from two streams, with a copy
    between them: it waits for all of them in every replay."""
    g = torch.Generator().manual_seed(11)
    a, w = (torch.randn(n, 256, generator=g).to(cuda_device) for n in (3000, 520))
    src, wsrc, out = a.clone(), w.clone(), torch.empty(3000, 520, device=cuda_device)
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            w.copy_(wsrc)
            qw = mx.mx_quantize(w)
        a.copy_(src)
        qa = mx.mx_quantize(a)
        main.wait_stream(side)
        y = mx.mx_matmul(qa, qw, out=out)
        out.mul_(2)
        return mx.mx_matmul(qa, qw), y

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plain, doubled = step()
    for i in range(3):
        src.copy_(torch.randn(3000, 256, generator=g))
        wsrc.copy_(torch.randn(520, 256, generator=g))
        graph.replay()
        want = mx.mx_matmul(src, mx.mx_quantize(wsrc))
        assert torch.equal(plain, want) and torch.equal(doubled, 2 * want)
