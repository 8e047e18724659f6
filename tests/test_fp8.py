"""8-bit floating point with a scale per block of 128: quantisation byte for byte
against a search over the representable values in 64 bits, the products and the
gradients against 64-bit products of the dequantised operands, and the refusals."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

from scmp_vit_b200 import _lib, fp8

E4M3 = np.array([i * 2.0 ** -9 for i in range(8)]
                + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)])[:127]
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def nearest(v, grid):
    """Index of the nearest grid entry (ascending), the even one between two."""
    hi = np.searchsorted((grid[1:] + grid[:-1]) / 2, v, side="right")
    lo = np.searchsorted((grid[1:] + grid[:-1]) / 2, v, side="left")
    return np.where((lo != hi) & (lo % 2 == 1), hi, lo)


def quantize_ref(x, blocks="row"):
    """(codes [rows, kp], scale codes [rows, blocks], values [rows, K])."""
    x = np.asarray(x, dtype=np.float64)
    rows, K = x.shape
    height = 128 if blocks == "square" else 1
    nb, nr = -(-K // 128), -(-rows // height)
    v = np.zeros((nr * height, nb * 128))
    v[:rows, :K] = x
    v = v.reshape(nr, height, nb, 128)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(v).all((1, 3), keepdims=True)
        v = np.where(bad, 0.0, v)
    amax = np.abs(v).max((1, 3), keepdims=True)
    e = np.full(amax.shape, -127)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):  # the smallest e with amax <= 448 2^e
        e = np.where(amax > 448 * 2.0 ** (e + step - 1.0), e + step, e)
    code = nearest(np.abs(v) / 2.0 ** e.astype(np.float64), E4M3)
    value = E4M3[code] * 2.0 ** e.astype(np.float64) * np.where(np.signbit(v), -1, 1)
    value = np.where(bad, np.nan, value)
    code = code + 128 * np.signbit(v)
    scale = np.broadcast_to(np.where(bad, 0xFF, e + 127), v.shape)[:, :, :, 0]
    flat = (nr * height, nb * 128)
    kp = nb * 128
    return (code.reshape(flat)[:rows, :kp], scale.reshape(-1, nb)[:rows],
            value.reshape(flat)[:rows, :K])


def pack_scales(scale):
    rows, nb = scale.shape
    out = np.zeros((-(-rows // 128), -(-nb // 4), 512), dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scale
    return out.reshape(-1)


# ------------------------------------------------------------ CPU: refusals

def test_sizes():
    lib = _lib.load()
    for rows, K in ((0, 5), (1, 1), (128, 32), (129, 513), (257, 1024)):
        data, scales = fp8._sizes(rows, K)
        assert lib.scmp_fp8_data_size(rows, K) == data == rows * (-(-K // 128) * 128)
        assert lib.scmp_fp8_scale_size(rows, K) == scales == -(-rows // 128) * -(-K // 512) * 512
    for rows, K in ((-1, 4), (4, 0), (1 << 31, 4), (4, 1 << 31)):
        assert lib.scmp_fp8_data_size(rows, K) == lib.scmp_fp8_scale_size(rows, K) == 0


@pytest.mark.parametrize("pack,cls", [
    (_lib.PACK_FP8_QUANTIZE, _lib.Fp8QuantizeArgs), (_lib.PACK_FP8_MATMUL, _lib.Fp8MatmulArgs),
    (_lib.PACK_FP8_TRAIN, _lib.Fp8TrainArgs), (_lib.PACK_FP8_TRAIN_BWD, _lib.Fp8TrainBwdArgs)])
def test_packed_arguments_are_the_structs(pack, cls):
    a, values = cls(), []
    for n, (name, _) in enumerate(cls._fields_, 1):
        values.append(n)
        setattr(a, name, n)
    assert pack.pack(*values) == bytes(a)


@pytest.mark.parametrize("args,msg", [
    (dict(abi_version=9), "abi_version"),
    (dict(rows=-1), "shape"),
    (dict(K=0), "shape"),
    (dict(dtype=3), "dtype"),
    (dict(ld=7), "ld"),
    (dict(x=0), "non-NULL"),
    (dict(data=0), "non-NULL"),
    (dict(t_data=16), "non-NULL"),
    (dict(data=0, scales=0), "non-NULL"),
    (dict(data=24), "aligned"),
    (dict(t_data=16, t_scales=8), "aligned"),
    (dict(x=18), "aligned to its elements"),
])
def test_quantize_refusals(args, msg):
    a = _lib.Fp8QuantizeArgs()
    for k, v in dict(dict(abi_version=_lib.ABI_VERSION, x=16, dtype=0, rows=4, K=8, ld=8, data=16,
                          scales=16), **args).items():
        setattr(a, k, v)
    assert _lib.load().scmp_fp8_quantize(ctypes.byref(a), None) == -1
    assert msg in _lib.last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(abi_version=9), "abi_version"),
    (dict(M=-1), "shape"),
    (dict(K=0), "shape"),
    (dict(out_dtype=5), "dtype"),
    (dict(bias=16, bias_dtype=4), "dtype"),
    (dict(a=None), "non-NULL"),
    (dict(out=None), "non-NULL"),
    (dict(b_scales=8), "aligned"),
    (dict(out=18), "aligned to its elements"),
    (dict(bias=17, bias_dtype=2), "aligned to its elements"),
])
def test_matmul_refusals(args, msg):
    a = _lib.Fp8MatmulArgs()
    a.abi_version, a.M, a.N, a.K = _lib.ABI_VERSION, 4, 4, 32
    a.a = a.a_scales = a.b = a.b_scales = a.out = 16
    for k, v in args.items():
        setattr(a, k, v)
    assert _lib.load().scmp_fp8_matmul(ctypes.byref(a), None) == -1
    assert msg in _lib.last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(x_dtype=3), "dtype"),
    (dict(ld=31), "ld"),
    (dict(x=None), "non-NULL"),
    (dict(M=5, a=None), "non-NULL"),       # past the rows that need no buffers
    (dict(K=6400, ld=6400, a=None), "non-NULL"),
    (dict(x=18), "aligned to its elements"),
])
def test_linear_refusals(args, msg):
    a = _lib.Fp8MatmulArgs()
    a.abi_version, a.M, a.N, a.K = _lib.ABI_VERSION, 4, 4, 32
    a.a = a.a_scales = a.b = a.b_scales = a.out = 16
    call = dict(x=16, x_dtype=0, ld=32)
    for k, v in args.items():
        if k in call:
            call[k] = v
        else:
            setattr(a, k, v)
    assert _lib.load().scmp_fp8_linear(call["x"], call["x_dtype"], call["ld"], ctypes.byref(a),
                                       None) == -1
    assert msg in _lib.last_error()


def train_args(cls, names, **kw):
    a = cls()
    a.abi_version, a.M, a.N, a.K, a.ld = _lib.ABI_VERSION, 4, 8, 32, 32
    if hasattr(a, "weight_ld"):
        a.weight_ld = 32
    for n in names:
        setattr(a, n, 16)
    a.workspace_bytes = 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=2), -1, "abi_version"),
    (dict(dtype=3), -1, "dtype"),
    (dict(weight_dtype=-1), -1, "dtype"),
    (dict(bias_dtype=7), -1, "dtype"),
    (dict(M=0), -1, "shape"),
    (dict(K=0), -1, "shape"),
    (dict(ld=31), -1, "ld"),
    (dict(weight_ld=31), -1, "ld"),
    (dict(y=None), -1, "non-NULL"),
    (dict(weight=18), -1, "aligned to its elements"),
    (dict(workspace_bytes=100), -3, "workspace"),
    (dict(saved_x=24), -1, "16-byte"),
])
def test_train_forward_refusals(kw, code, msg):
    a = train_args(_lib.Fp8TrainArgs, ("x", "weight", "bias", "y", "saved_x", "saved_weight",
                                       "workspace"), **kw)
    assert _lib.load().scmp_fp8_train_forward(ctypes.byref(a), None) == code
    assert msg in _lib.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(abi_version=2), -1, "abi_version"),
    (dict(dtype=3), -1, "dtype"),
    (dict(weight_dtype=3), -1, "dtype"),
    (dict(bias_dtype=3), -1, "dtype"),
    (dict(N=0), -1, "shape"),
    (dict(ld=7), -1, "ld"),
    (dict(dy=None), -1, "non-NULL"),
    (dict(saved_x=None), -1, "non-NULL"),
    (dict(saved_weight=None), -1, "non-NULL"),
    (dict(dx=None, dweight=None, dbias=None), -1, "non-NULL"),
    (dict(dbias=18), -1, "aligned to its elements"),
    (dict(workspace=None), -3, "workspace"),
])
def test_train_backward_refusals(kw, code, msg):
    a = train_args(_lib.Fp8TrainBwdArgs, ("dy", "saved_x", "saved_weight", "dx", "dweight",
                                          "dbias", "workspace"), **kw)
    assert _lib.load().scmp_fp8_train_backward(ctypes.byref(a), None) == code
    assert msg in _lib.last_error()


def test_python_refusals_on_cpu():
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp8.fp8_quantize(x)
    with pytest.raises(ValueError, match="blocks"):
        fp8.fp8_quantize(x, "column")
    with pytest.raises(TypeError, match="float32"):
        fp8.fp8_quantize(x.double())
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp8.fp8_linear(x, torch.zeros(8, 32))
    q = fp8.fp8_empty((8, 32), torch.device("cpu"), torch.float32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fp8.fp8_matmul(x, q)
    with pytest.raises(RuntimeError, match="no CPU path"):
        q.dequantize()
    with pytest.raises(TypeError, match="2-D"):
        fp8.fp8_matmul(x, x)
    with pytest.raises(ValueError, match="last dimension"):
        fp8.FP8Tensor(q.data, q.scales, (32, 8, 0))
    with pytest.raises(ValueError, match="contiguous bytes"):
        fp8.FP8Tensor(q.data[:-16], q.scales, (8, 32))
    with pytest.raises(ValueError, match="contiguous bytes"):
        fp8.FP8Tensor(q.data.float(), q.scales, (8, 32))
    with pytest.raises(ValueError, match="keeps its last"):
        q.reshape(32, 8)
    assert q.reshape(2, 4, 32).rows == 8


def test_copies_are_tensors_of_their_own():
    q = fp8.fp8_empty((5, 40), torch.device("cpu"), torch.bfloat16, "square")
    q.data.copy_(torch.arange(q.data.numel()) % 251)
    q.scales.copy_(torch.arange(q.scales.numel()) % 127)
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert c.data_ptr == c.data.data_ptr() != q.data_ptr
        assert c.scales_ptr == c.scales.data_ptr() != q.scales_ptr
        assert torch.equal(c.data, q.data) and torch.equal(c.scales, q.scales)
        assert (c.shape, c.rows, c.blocks, c.dtype) == ((5, 40), 5, "square", torch.bfloat16)


@pytest.fixture
def no_launch(monkeypatch):
    """CPU tensors in the place of CUDA ones, launches recorded."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    launched = []
    monkeypatch.setattr(fp8, "call", lambda *a: launched.append(a))
    return launched


def test_few_rows_rule_in_both_places():
    """The Python side allocates no buffers where the engine needs none."""
    for M in (1, 2, 3, 4, 5):
        for N in (1, 300, 1024, 4096, 16384):
            for K in (1, 700, 1024, 4096, 6144, 6145):
                assert _lib.fp8_plan(M, N, K)[0] == fp8._thin(M, N, K)


def test_shapes_and_types_are_checked(no_launch):
    x, w = torch.zeros(6, 32), torch.zeros(8, 32)
    q = fp8.fp8_empty((8, 32), x.device, x.dtype)
    for bad, match in ((lambda: fp8.fp8_quantize(x[None], "square"), "matrices"),
                       (lambda: fp8.fp8_quantize(x[None], transpose=True), "matrices"),
                       (lambda: fp8.fp8_quantize(x[:0], transpose=True), "no rows"),
                       (lambda: fp8.fp8_quantize(x[:, :0]), "last dimension"),
                       (lambda: fp8.fp8_matmul(x[:, :16], q), "inner-dim"),
                       (lambda: fp8.fp8_matmul(x, q, bias=torch.zeros(7)), "bias"),
                       (lambda: fp8.fp8_matmul(x, q, out=torch.zeros(6, 9)), "out must"),
                       (lambda: fp8.fp8_linear(x, w[:, :16]), "inner-dim"),
                       (lambda: fp8.fp8_linear(x, w[None]), "weight"),
                       (lambda: fp8.fp8_linear(x, w, torch.zeros(9)), "bias")):
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(TypeError, match="weight"):
        fp8.fp8_linear(x, w.double())
    with pytest.raises(TypeError, match="bias"):
        fp8.fp8_linear(x, w, torch.zeros(8).double())
    for f in (lambda t: fp8.fp8_quantize(t), lambda t: fp8.fp8_matmul(t, q)):
        with pytest.raises(RuntimeError, match="no gradient"):
            f(x.clone().requires_grad_())
    out = x.view(-1)[:48].view(6, 8)
    with pytest.raises(ValueError, match="shares memory"):
        fp8.fp8_matmul(x, q, out=out)
    assert no_launch == []
    import torch.autograd.forward_ad as fwAD
    for grad in (True, False):
        with fwAD.dual_level(), torch.set_grad_enabled(grad):
            d = fwAD.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="jvp"):
                fp8.fp8_linear(d, w)
            with pytest.raises(RuntimeError, match="no gradient"):
                fp8.fp8_matmul(d, q)


def test_linear_refuses_buffers_of_another_kind(monkeypatch):
    """``load_state_dict(assign=True)`` takes the given tensors themselves; the
    kernels would read them as the packed layout."""
    monkeypatch.setattr(fp8, "fp8_quantize", lambda w, blocks: fp8.fp8_empty(
        w.shape, w.device, w.dtype, blocks))
    m = fp8.FP8Linear(torch.nn.Linear(96, 72))
    for name in ("data", "scales"):
        state = m.state_dict()
        state[name] = state[name].float()
        m.load_state_dict(state, assign=True)
        with pytest.raises(ValueError, match="contiguous bytes"):
            m.quantized_weight()
        m = fp8.FP8Linear(torch.nn.Linear(96, 72))
    assert m.quantized_weight().shape == (72, 96)
    t = fp8.FP8Linear(torch.nn.Linear(96, 72), train=True)
    assert sorted(n for n, _ in t.named_parameters()) == ["bias", "weight"]


# ------------------------------------------------------------ GPU: quantise

def special_rows(K):
    """Rows that borders, ends of ranges and odd values decide."""
    g = torch.Generator().manual_seed(K)
    rows = [torch.zeros(K), torch.full((K,), -0.0), torch.full((K,), 1e-45),
            torch.full((K,), 3.0e38), torch.randn(K, generator=g) * 1e-40,
            torch.randn(K, generator=g) * 2.0 ** -118, torch.randn(K, generator=g) * 1e37,
            torch.exp(12 * torch.randn(K, generator=g))]
    ties = torch.tensor([1.0625, -1.1875, 1.9375, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -0.0, 15.5])
    for s in (1.0, 448.0, 28.0, 1.75 * 2.0 ** 5, 1.7500002 * 2.0 ** 5, 2.0 ** -9, 2.0 ** -100):
        r = (ties.repeat(K // 8 + 1) * s)[:K]
        r[K // 3] = s * 16
        rows.append(r)
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.randn(K, generator=g)
        r[K // 2] = bad
        rows.append(r)
    return torch.stack(rows)


def check_tensor(q, x, blocks):
    values = q.dequantize(torch.float32)
    torch.cuda.synchronize()
    x2 = x.detach().cpu().reshape(-1, x.shape[-1])
    code, scale, value = quantize_ref(x2.double().numpy(), blocks)
    got = q.data.cpu().numpy().reshape(code.shape)
    fine = np.repeat(scale != 0xFF, 128, 1)[:, :code.shape[1]]  # (codes of a NaN block: any)
    assert np.array_equal(got[fine], code[fine].astype(np.uint8))
    assert np.array_equal(q.scales.cpu().numpy(), pack_scales(scale))
    with np.errstate(over="ignore"):
        value = value.astype(np.float32)
    assert np.array_equal(values.cpu().numpy().reshape(value.shape), value, equal_nan=True)


def check_quantize(x, blocks="row"):
    q = fp8.fp8_quantize(x, blocks)
    assert (q.shape, q.blocks, q.dtype) == (x.shape, blocks, x.dtype)
    check_tensor(q, x, blocks)
    if x.dim() == 2 and x.shape[0]:
        p, t = fp8.fp8_quantize(x, blocks, transpose=True)
        check_tensor(p, x, blocks)
        check_tensor(t, x.t(), blocks)
        fine = ~torch.isnan(q.dequantize(torch.float32))
        assert torch.equal(p.dequantize(torch.float32)[fine], q.dequantize(torch.float32)[fine])


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", fp8.BLOCKS)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 128), (2, 127), (3, 129), (130, 64), (5, 257),
                                    (129, 513), (257, 1024), (4, 4104), (33, 520), (640, 1040)])
def test_quantize_bytes(cuda_device, blocks, rows, K):
    g = torch.Generator().manual_seed(rows * 1000 + K)
    for dtype in DTYPES:
        x = torch.randn(rows, K, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
        check_quantize(x.to(dtype).to(cuda_device), blocks)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [16, 47, 256, 300])
def test_quantize_special_values(cuda_device, K):
    for dtype in DTYPES:
        x = special_rows(K).to(dtype).to(cuda_device)
        check_quantize(x)
        for r in range(x.shape[0]):
            check_quantize(x[r:r + 1], "square")


@pytest.mark.gpu
def test_quantize_strides_and_shapes(cuda_device):
    x = torch.randn(6, 40, 96, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    check_quantize(x)
    check_quantize(x[:, ::3, 1:65])               # strided rows at an odd offset
    check_quantize(x[:, :, ::2])                  # strided elements
    check_quantize(x.transpose(0, 2))
    check_quantize(x[0, :1].expand(5, 96))        # one row five times
    check_quantize(x[2, 3])                       # one dimension
    check_quantize(x.reshape(240, 96)[3:, 1:90], "square")
    check_quantize(x.reshape(240, 96).t(), "square")
    empty = fp8.fp8_quantize(x[:0])
    assert empty.shape == (0, 40, 96) and empty.dequantize().shape == (0, 40, 96)
    r = fp8.fp8_quantize(x).reshape(-1, 96)
    assert torch.equal(r.dequantize(), fp8.fp8_quantize(x).dequantize().reshape(240, 96))


@pytest.mark.gpu
def test_quantize_walks(cuda_device):
    """More units than warps: every form of the row kernel, and many tiles."""
    g = torch.Generator().manual_seed(3)
    for rows, K in ((40000, 130), (5000, 2050), (5003, 2056)):
        x = torch.randn(rows, K, generator=g).to(torch.bfloat16).to(cuda_device)
        check_quantize(x)


# ------------------------------------------------------------- GPU: product

def product_bound(a, b, y, out_dtype):
    """|error| allowed for fp32 sums of exact products in any order, each
    addition off by at most one unit in the last place (2^-23 of the running
    magnitude, itself at most sum |a||b|), plus the final rounding: half a step,
    relative to y or, below the type's smallest normal number, where numbers are a
    fixed distance apart, to that one."""
    K, out = a.shape[-1], torch.finfo(out_dtype)
    return (K + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t() + y.abs()) + \
        out.eps / 2 * y.abs().clamp(min=out.tiny)


def close(got, a, b, bias=None):
    """got against a b^T (+ bias) of 64-bit operands."""
    ref = a @ b.t()
    if bias is not None:
        ref = ref + bias.double()
    bound = product_bound(a, b, ref, got.dtype)
    if got.dtype == torch.float16:
        ref = ref.clamp(-65504, 65504)
    err = (got.double().reshape(ref.shape) - ref).abs()
    assert bool((err <= bound).all()), (err / bound).max()


def values(q):
    return q.dequantize(torch.float32).double().reshape(-1, q.shape[-1])


def check_product(a, w, dtype, bias=None):
    qa, qw = fp8.fp8_quantize(a), fp8.fp8_quantize(w, "square")
    y = fp8.fp8_matmul(a, qw, bias=bias, out_dtype=dtype)
    y2 = fp8.fp8_matmul(qa, qw, bias=bias, out_dtype=dtype)
    torch.cuda.synchronize()
    assert _lib.engine_status() == 0
    for got in (y, y2):
        assert got.dtype == dtype and got.shape == (*a.shape[:-1], w.shape[0])
        close(got, values(qa), values(qw), bias)
    return y


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 4096, 1024), (2, 77, 200), (3, 300, 6144), (4, 1024, 1030),
          (5, 40, 128), (16, 257, 129), (17, 256, 640), (33, 1000, 333), (64, 130, 96),
          (129, 512, 512), (257, 1024, 1024), (300, 100, 4096), (1000, 1300, 260)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(cuda_device, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    for i, dtype in enumerate(DTYPES):
        a = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
        w = torch.randn(N, K, generator=g) * 0.05
        bias = torch.randn(N, generator=g).to(DTYPES[(i + 1) % 3]).to(cuda_device)
        check_product(a.to(dtype).to(cuda_device), w.to(cuda_device), dtype, bias)
        check_product(a.to(dtype).to(cuda_device), w.to(cuda_device), DTYPES[(i + 1) % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 300])
def test_product_is_exact_where_sums_are(cuda_device, rows):
    """Small whole numbers: every partial sum is exact in fp32, so the product's
    layout, scales and order of blocks are seen bit for bit."""
    g = torch.Generator().manual_seed(rows)
    a = torch.randint(-8, 9, (rows, 1300), generator=g).float()
    w = torch.randint(-8, 9, (520, 1300), generator=g).float()
    for b in range(11):  # blocks of different scales
        a[:, b * 128:(b + 1) * 128] *= 2.0 ** (b % 5 - 2)
        w[:, b * 128:(b + 1) * 128] *= 2.0 ** (b % 3 - 1)
    a, w = a.to(cuda_device), w.to(cuda_device)
    qa, qw = fp8.fp8_quantize(a), fp8.fp8_quantize(w, "square")
    assert torch.equal(qa.dequantize(), a) and torch.equal(qw.dequantize(), w)
    ref = (a.double() @ w.double().t()).float()
    assert torch.equal(fp8.fp8_matmul(a, qw), ref)
    assert torch.equal(fp8.fp8_matmul(qa, qw), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 40])
def test_product_ranges_and_nan(cuda_device, M):
    """Blocks at the ends of the scales' range, and NaN blocks."""
    g = torch.Generator().manual_seed(M)
    for ea, ew in ((2.0 ** 100, 2.0 ** -100), (2.0 ** -60, 2.0 ** -60), (2.0 ** 50, 2.0 ** 50)):
        a = (torch.randn(M, 300, generator=g) * ea).to(cuda_device)
        w = (torch.randn(70, 300, generator=g) * ew).to(cuda_device)
        check_product(a, w, torch.float32)
    a, w = torch.randn(M, 300, generator=g), torch.randn(70, 300, generator=g)
    a[0, 200] = float("nan")
    w[5, 10] = float("inf")  # one square of 70 rows
    y = fp8.fp8_matmul(a.to(cuda_device), fp8.fp8_quantize(w.to(cuda_device), "square"))
    assert bool(torch.isnan(y).all())
    y = fp8.fp8_matmul(a.to(cuda_device), fp8.fp8_quantize(w.to(cuda_device)))
    nan = torch.isnan(y).cpu()
    assert bool(nan[0].all()) and bool(nan[:, 5].all())
    nan[0] = False
    nan[:, 5] = False
    assert not bool(nan.any())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,widths,units", [
    (16135, 952, 640, (256, 192), 148), (7299, 1817, 1100, (256, 192), 136),
    (9000, 1152, 1024, (192, 0), 235), (16697, 80, 71, (128, 0), 131),
    (788, 333, 1000, (64, 0), 26), (1024, 4096, 4300, (256, 0), 64),
    (1500, 4100, 6200, (192, 0), 136)])
def test_product_many_tiles(cuda_device, M, N, K, widths, units):
    """Every choice of tile widths, several units per pair where it has them, ragged
    ends, and (the last) a weight that is walked in groups of its rows."""
    assert _lib.fp8_plan(M, N, K)[1:] == (widths, units)
    g = torch.Generator().manual_seed(M)
    a = torch.randn(M, K, generator=g).to(torch.bfloat16).to(cuda_device)
    w = (torch.randn(N, K, generator=g) * 0.05).to(cuda_device)
    bias = torch.randn(N, generator=g).to(cuda_device)
    qa, qw = fp8.fp8_quantize(a), fp8.fp8_quantize(w, "square")
    for dtype in (torch.float32, torch.bfloat16):
        close(fp8.fp8_matmul(qa, qw, bias=bias, out_dtype=dtype), values(qa), values(qw), bias)


@pytest.mark.gpu
def test_long_sums(cuda_device):
    """fp32 outputs of long sums go in pieces that are rounded, not cut off: with
    2^-24 per 4096 values and piece at most 8 of them (the tensor core's 128 adds of
    32 products each cut at most 2^-23 of the running sum, and a quarter of that on
    average is far from reached), against a root mean square over the outputs."""
    g = torch.Generator().manual_seed(2)
    a = torch.randn(300, 16500, generator=g).to(cuda_device)
    w = torch.randn(520, 16500, generator=g).to(cuda_device)
    bias = torch.randn(520, generator=g).to(cuda_device)
    qa, qw = fp8.fp8_quantize(a), fp8.fp8_quantize(w)
    before = _lib.kernel_launches()
    y = fp8.fp8_matmul(qa, qw, bias=bias)
    assert _lib.kernel_launches() - before == 5
    ref = values(qa) @ values(qw).t() + bias.double()
    assert float((y.double() - ref).norm() / ref.norm()) < 16 * 2.0 ** -24
    close(y, values(qa), values(qw), bias)


def one_sign(rows, K, g, device):
    """Positive values of many magnitudes, rows of different size, whose products sum
    to a few units: every addition to a long sum has bits below the sum's last one."""
    x = torch.exp(2 * torch.randn(rows, K, generator=g, device=device) - 2)
    return x.mul_((1 + torch.rand(rows, 1, generator=g, device=device)) / K ** 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,M,N,K", [
    (torch.float16, 300, 296, 16384), (torch.float16, 300, 300, 16385),
    (torch.float16, 40, 299, 70000),
    (torch.float16, 5, 4100, 20000), (torch.float16, 17, 520, 300000),
    (torch.float16, 500, 296, 524288), (torch.bfloat16, 300, 296, 131072),
    (torch.bfloat16, 300, 296, 131073), (torch.bfloat16, 260, 299, 1048576),
    (torch.float32, 300, 296, 16500)])
def test_long_sums_of_one_sign(cuda_device, dtype, M, N, K):
    """Sums of positive products, where cut-off bits all point one way.  An addition
    of 32 products to a sum cuts each product off at 2^-25 of the sum's power of two and
    the new sum at 2^-23: at most 32 * 2^-25 + 2^-23 = 9 * 2^-23 of the sum.  Up to 16384
    values (fp16 outputs) and 131072 (bf16) are one sum, fp32 outputs add up launches of
    at most 4096; longer 16-bit ones go in pieces of 1024 (32 additions), which are added
    up rounded (2^-24 each, the bias 2^-24)."""
    g = torch.Generator(device=cuda_device).manual_seed(K)
    qa, qw = (fp8.fp8_quantize(one_sign(rows, K, g, cuda_device)) for rows in (M, N))
    bias = torch.rand(N, generator=g, device=cuda_device)
    y = fp8.fp8_matmul(qa, qw, bias=bias, out_dtype=dtype)
    torch.cuda.synchronize()
    assert _lib.engine_status() == 0
    ref = torch.zeros(M, N, dtype=torch.float64, device=cuda_device)
    a, w = (q.dequantize(torch.float32) for q in (qa, qw))
    for k in range(0, K, 65536):
        ref += a[:, k:k + 65536].double() @ w[:, k:k + 65536].double().t()
    ref += bias.double()
    whole, piece = {torch.float16: (16384, 1024), torch.bfloat16: (131072, 1024),
                    torch.float32: (4096, 4096)}[dtype]
    pieces = 1 if K <= whole else -(-K // piece)
    cut = (K if K <= whole else piece) / 32 * 9 * 2.0 ** -23
    half = torch.finfo(dtype).eps / 2
    err = ((y.double() - ref) / ref).abs()
    assert float(err.max()) <= (cut + (pieces + 2) * 2.0 ** -24) * (1 + half) + half
    assert torch.equal(y, fp8.fp8_matmul(qa, qw, bias=bias, out_dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(16, 264), (40, 257), (300, 130), (1500, 2100)])
def test_long_sums_are_exact_where_sums_are(cuda_device, M, N):
    """Sums in pieces of whole numbers, both signs: every partial sum is exact, so each
    piece, and what the last one leaves, counts once; several tiles per pair."""
    g = torch.Generator().manual_seed(M)
    K = 20 * 4096 + 300
    a = torch.randint(-2, 3, (M, K), generator=g, dtype=torch.int8).to(cuda_device).half()
    w = torch.randint(-2, 3, (N, K), generator=g, dtype=torch.int8).to(cuda_device).half()
    bias = torch.randint(-500, 501, (N,), generator=g).float().to(cuda_device)
    ref = a.double() @ w.double().t() + bias.double()
    y = fp8.fp8_matmul(fp8.fp8_quantize(a), fp8.fp8_quantize(w), bias=bias)
    assert y.dtype == torch.float16 and torch.equal(y, ref.to(torch.float16))


@pytest.mark.gpu
def test_long_sums_give_up_and_recover(cuda_device):
    """A sum in pieces whose loaders are held: every wait runs out, the next call is right."""
    g = torch.Generator(device=cuda_device).manual_seed(8)
    qa, qw = (fp8.fp8_quantize(one_sign(300, 20000, g, cuda_device)) for _ in range(2))
    want = fp8.fp8_matmul(qa, qw, out_dtype=torch.float16)
    torch.cuda.synchronize()
    _lib.engine_status(reset=True)
    _lib.set_wait_limit(20_000_000)
    _lib.hold_producers(True)
    try:
        fp8.fp8_matmul(qa, qw, out_dtype=torch.float16)
        torch.cuda.synchronize()
        status = _lib.engine_status(reset=True)
    finally:
        _lib.hold_producers(False)
        _lib.set_wait_limit(2_000_000_000)
    assert status & 1
    assert torch.equal(fp8.fp8_matmul(qa, qw, out_dtype=torch.float16), want)


@pytest.mark.gpu
def test_training_over_many_tokens(cuda_device):
    """A weight gradient that is a sum in pieces, in fp16."""
    g = torch.Generator().manual_seed(17)
    x, dy = (torch.randn(17000, n, generator=g).half().to(cuda_device) for n in (40, 72))
    w = (torch.randn(72, 40, generator=g) * 0.05).half().to(cuda_device)
    check_training(x, w, None, dy * 0.1)


@pytest.mark.gpu
def test_out_and_its_refusals(cuda_device):
    a = torch.randn(30, 64, device=cuda_device)
    qw = fp8.fp8_quantize(torch.randn(40, 64, device=cuda_device))
    out = torch.empty(30, 40, device=cuda_device)
    version = out._version
    assert fp8.fp8_matmul(a, qw, out=out) is out and out._version > version
    assert torch.equal(out, fp8.fp8_matmul(a, qw))
    with pytest.raises(ValueError, match="devices"):
        fp8.fp8_matmul(a.cpu(), qw)
    with pytest.raises(ValueError, match="devices"):
        fp8.fp8_linear(a, torch.randn(40, 64))
    assert fp8.fp8_matmul(a[:0], qw).shape == (0, 40)
    assert fp8.fp8_matmul(a[0], qw).shape == (40,)
    assert fp8.fp8_matmul(a.reshape(5, 6, 64), qw).shape == (5, 6, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 300])
def test_streams_graphs_and_repeats(cuda_device, M):
    """A side stream, a captured call replayed on new inputs, the same bits from
    every call."""
    g = torch.Generator().manual_seed(4)
    w = fp8.fp8_quantize(torch.randn(160, 128, generator=g).to(cuda_device), "square")
    x = torch.randn(M, 128, generator=g).to(cuda_device)
    ref = fp8.fp8_matmul(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp8.fp8_matmul(x, w)
    side.synchronize()
    assert torch.equal(got, ref)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8.fp8_matmul(static, w)
    static.copy_(x * 2 + 1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, fp8.fp8_matmul(x * 2 + 1, w))


@pytest.mark.gpu
def test_bounded_wait_gives_up_and_recovers(cuda_device):
    """With the loaders held on a flag that nothing sets, every wait runs out
    after its (shortened) limit, the launch returns and says so, and the next
    call on the same context is right."""
    g = torch.Generator().manual_seed(8)
    a, w = torch.randn(300, 320, generator=g), torch.randn(300, 320, generator=g)
    a, w = a.to(cuda_device), w.to(cuda_device)
    qa, qw = fp8.fp8_quantize(a), fp8.fp8_quantize(w)
    torch.cuda.synchronize()
    _lib.engine_status(reset=True)
    _lib.set_wait_limit(20_000_000)
    _lib.hold_producers(True)
    try:
        fp8.fp8_matmul(qa, qw)
        torch.cuda.synchronize()
        status = _lib.engine_status(reset=True)
    finally:
        _lib.hold_producers(False)
        _lib.set_wait_limit(2_000_000_000)
    assert status & 1
    check_product(a, w, torch.float32)


# ------------------------------------------------------------ GPU: training

def check_training(x, w, b, dy):
    """y and every gradient against the formula in 64 bits on the definition's
    values (``quantize_ref``, not the kernels)."""
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    y = fp8.fp8_linear(x, w, b)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], w.shape[0])
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.synchronize()
    assert _lib.engine_status() == 0

    def q(t, blocks="row"):
        v = quantize_ref(t.detach().double().cpu().numpy(), blocks)[2]
        return torch.from_numpy(np.ascontiguousarray(v)).to(x.device)
    x2, dy2 = x.detach().reshape(-1, x.shape[-1]), dy.reshape(-1, w.shape[0])
    qw = q(w, "square")
    close(y, q(x2), qw, None if b is None else b.detach())
    close(grads[0], q(dy2), qw.t())
    close(grads[1], q(dy2.t()), q(x2.t()))
    for t, gr in zip(leaves, grads):
        assert gr.dtype == t.dtype and gr.shape == t.shape
    if b is not None:
        close(grads[2], torch.ones(1, dy2.shape[0], device=x.device, dtype=torch.float64),
              dy2.double().t())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 40, 64), (3, 257, 130), (128, 128, 128),
                                   (129, 100, 1000), (788, 333, 1000), (1028, 1024, 520)])
def test_training(cuda_device, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g).to(dtype).to(cuda_device)
    for i, dtype in enumerate(DTYPES):
        other = DTYPES[(i + 1) % 3]
        check_training(randn(M, K, dtype=dtype), randn(N, K, dtype=dtype) * 0.05,
                       randn(N, dtype=dtype), randn(M, N, dtype=dtype) * 0.1)
        check_training(randn(M, K, dtype=dtype), randn(N, K, dtype=other) * 0.05,
                       randn(N, dtype=other) if i else None, randn(M, N, dtype=dtype) * 0.1)


@pytest.mark.gpu
def test_training_strides(cuda_device):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 50, 200, generator=g).to(cuda_device)
    w = torch.randn(96, 200, generator=g).to(cuda_device)
    dy = torch.randn(3, 50, 192, generator=g).to(cuda_device)
    check_training(x, w, None, dy[..., :96])
    check_training(x[:, ::2], w, w[:, 3], dy[:, ::2, 96:])
    check_training(x.transpose(0, 1), w[:, 1:].repeat(1, 2)[:, :200], None,
                   dy[..., ::2].transpose(0, 1))
    check_training(x[..., :96], w.t()[:96, :96], None, dy[..., :1].expand(3, 50, 96))
    check_training(x[0, 0], w, w[:, 0].contiguous(), dy[0, 0, :96])


@pytest.mark.gpu
def test_training_wants(cuda_device):
    """Any subset of gradients gives the same ones; no rows give zeros."""
    g = torch.Generator().manual_seed(6)
    x, w, b = (torch.randn(*s, generator=g).to(cuda_device) for s in ((70, 130), (60, 130), (60,)))
    dy = torch.randn(70, 60, generator=g).to(cuda_device)
    full = None
    for wants in range(7, 0, -1):
        t = [v.clone().requires_grad_(bool(wants >> i & 1)) for i, v in enumerate((x, w, b))]
        y = fp8.fp8_linear(*t)
        got = torch.autograd.grad(y, [v for v in t if v.requires_grad], dy)
        full = full or got
        for i, gr in zip([i for i in range(3) if wants >> i & 1], got):
            assert torch.equal(gr, full[i])
    with torch.no_grad():
        assert torch.equal(fp8.fp8_linear(x, w, b), y)
    t = [v.clone().requires_grad_() for v in (x[:0], w, b)]
    y = fp8.fp8_linear(*t)
    assert y.shape == (0, 60)
    grads = torch.autograd.grad(y, t, dy[:0])
    assert grads[0].shape == (0, 130) and not grads[1].any() and not grads[2].any()
    x.requires_grad_()
    y = fp8.fp8_linear(x, w)
    (gr,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gr.sum(), x)


@pytest.mark.gpu
def test_gradients_by_differences(cuda_device):
    """Where codes are exact (small whole numbers, a difference of one code), the
    product is the linear itself: gradients are its differences, bit for bit."""
    g = torch.Generator().manual_seed(7)
    x = torch.randint(-4, 5, (40, 150), generator=g).float().to(cuda_device)
    w = torch.randint(-4, 5, (30, 150), generator=g).float().to(cuda_device)
    dy = torch.randint(-2, 3, (40, 30), generator=g).float().to(cuda_device)
    x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(fp8.fp8_linear(x, w), (x, w), dy)
    with torch.no_grad():
        for t, gr, at in ((x, gx, (3, 140)), (x, gx, (39, 0)), (w, gw, (29, 149)), (w, gw, (0, 7))):
            f = []
            for step in (1.0, -1.0):
                t[at] += step
                f.append((fp8.fp8_linear(x, w) * dy).double().sum())
                t[at] -= step
            assert float(gr[at]) == float((f[0] - f[1]) / 2)


@pytest.mark.gpu
def test_training_captured(cuda_device):
    """A captured step replayed on new inputs gives the eager step's bits."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(200, 160, generator=g).to(cuda_device)
    w = torch.randn(96, 160, generator=g).to(cuda_device)
    b, dy = torch.randn(96, generator=g).to(cuda_device), torch.randn(200, 96, generator=g).to(
        cuda_device)

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = fp8.fp8_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    static.copy_(x * 3 - 1)
    graph.replay()
    torch.cuda.synchronize()
    for a, r in zip(out, step(x * 3 - 1)):
        assert torch.equal(a, r)


@pytest.mark.gpu
def test_module(cuda_device):
    lin = torch.nn.Linear(96, 72).to(cuda_device)
    m = fp8.FP8Linear(lin)
    x = torch.randn(2, 11, 96, device=cuda_device)
    ref = fp8.fp8_matmul(x, fp8.fp8_quantize(lin.weight.detach(), "square"),
                         bias=lin.bias.detach())
    assert torch.equal(m(x), ref)
    assert torch.equal(m(fp8.fp8_quantize(x)), ref)
    again = fp8.FP8Linear(torch.nn.Linear(96, 72).to(cuda_device))
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), ref)
    t = fp8.FP8Linear(lin, train=True)
    assert t.weight is lin.weight
    assert torch.equal(t(x), ref)
    t(x).sum().backward()
    assert lin.weight.grad is not None and lin.bias.grad is not None
    assert torch.equal(t.quantized_weight().dequantize(), m.quantized_weight().dequantize())
