"""``vit.dropout`` bit for bit against Philox4x32-10 in integers, its gradient, its
modules in a block, and the refusals."""
import copy
import ctypes
import datetime
import io
import math
import os
import pickle
import socket
import sys
import threading

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from scmp_vit_b200 import _lib, vit

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
M32 = (1 << 32) - 1


def philox(counter, key):
    """One block of Philox4x32-10, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [b >> 32 ^ c[1] ^ k[0], b & M32, a >> 32 ^ c[3] ^ k[1], a & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def words(n, seed, offset, start=0):
    """Words start .. start + n of the generator, as numpy uint64."""
    seed &= (1 << 64) - 1
    first = start // 4
    i = np.arange(first, (start + n + 3) // 4, dtype=np.uint64)
    m = np.uint64(M32)
    c = [i & m, i >> np.uint64(32), np.full_like(i, offset & M32), np.full_like(i, offset >> 32)]
    k = [seed & M32, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return np.stack(c, -1).reshape(-1)[start - 4 * first:][:n]


def keep_of(shape, p, seed, offset, per):
    draws = {"element": shape, "row": (*shape[:-1], 1),
             "sample": (shape[0], *[1] * (len(shape) - 1))}[per]
    u = words(math.prod(draws), seed, offset)
    return torch.from_numpy(u >= np.uint64(round(p * 2 ** 32))).reshape(draws).expand(shape)


def expect(x, p, seed, offset, per, residual=None):
    """The definition in the kernel's steps: one fp32 product, one fp32 sum, one
    rounding (so equality, not a tolerance)."""
    keep = keep_of(tuple(x.shape), p, seed, offset, per).to(x.device)
    scale = torch.tensor(1 / (1 - p) if p < 1 else 0.0, dtype=torch.float32, device=x.device)
    y = torch.where(keep, x.float() * scale, torch.zeros((), device=x.device))
    return (y if residual is None else residual.float() + y).to(x.dtype)


# ------------------------------------------------------------ CPU

def test_generator_known_answers():
    """The published vectors of Philox4x32-10."""
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([M32] * 4, [M32] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344],
                  [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    seed, offset = 0x299F31D0A4093822, 0x0370734413198A2E
    got = words(9, seed, offset, 4 * 5 + 2)
    want = [w for i in (5, 6, 7) for w in philox([i, 0, offset & M32, offset >> 32],
                                                 [seed & M32, seed >> 32])][2:11]
    assert got.tolist() == want


@pytest.mark.parametrize("kw,msg", [
    (dict(abi_version=2), "abi_version"),
    (dict(dtype=3), "dtype"),
    (dict(n=-1), "sizes"),
    (dict(span=0), "sizes"),
    (dict(p=-0.1), "p must"),
    (dict(p=1.5), "p must"),
    (dict(p=math.nan), "p must"),
    (dict(x=None), "non-NULL"),
    (dict(y=None), "non-NULL"),
    (dict(residual=18), "aligned to its elements"),
    (dict(state=20), "8-byte"),
])
def test_refusals(kw, msg):
    a = _lib.DropoutArgs()
    for k, v in dict(dict(abi_version=_lib.ABI_VERSION, x=16, y=16, n=4, span=1, p=0.5),
                     **kw).items():
        setattr(a, k, v)
    assert _lib.load().scmp_dropout(ctypes.byref(a), None) == -1
    assert msg in _lib.last_error()


def test_packed_arguments_are_the_struct():
    a, values = _lib.DropoutArgs(), []
    for name, _ in a._fields_:
        values.append(len(values) + 1)
        setattr(a, name, values[-1])
    assert _lib.PACK_DROPOUT.pack(*values) == bytes(a)


def test_python_refusals(monkeypatch):
    x = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        vit.dropout(x, 0.1, 1)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    launched = []
    monkeypatch.setattr(vit, "call", lambda *a: launched.append(a))
    for kw, match in ((dict(per="column"), "per"), (dict(p=1.1), "p must"),
                      (dict(p=math.nan), "p must"), (dict(residual=x[:2]), "residual"),
                      (dict(residual=x.half()), "residual"), (dict(seed=1 << 64), "64-bit"),
                      (dict(offset=-1), "64-bit"), (dict(offset=1 << 64), "64-bit"),
                      (dict(seed=torch.zeros(2)), "seed tensor"),
                      (dict(seed=torch.zeros(3, dtype=torch.int64)), "seed tensor"),
                      (dict(seed=torch.zeros(4, dtype=torch.int64)[::2]), "seed tensor"),
                      (dict(x=x[0, 0], per="row"), "dimensions")):
        with pytest.raises(ValueError, match=match):
            vit.dropout(**dict(dict(x=x, p=0.1, seed=1), **kw))
    with pytest.raises(TypeError, match="float32"):
        vit.dropout(x.double(), 0.1, 1)
    assert launched == []
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), torch.no_grad():
        d = fwAD.make_dual(x, torch.ones_like(x))
        for t in ((d, None), (x, d)):
            with pytest.raises(NotImplementedError, match="jvp"):
                vit.dropout(t[0], 0.1, 1, residual=t[1])


def test_modules_on_cpu():
    for kw, match in ((dict(p=-1.0), "p must"), (dict(p=0.1, per="x"), "per"),
                      (dict(p=0.1, index=1 << 16), "index"), (dict(p=0.1, seed=1 << 64), "seed")):
        with pytest.raises(ValueError, match=match):
            vit.Dropout(**kw)
    x = torch.randn(2, 3)
    for m in (vit.Dropout(0.5).eval(), vit.Dropout(0.0)):
        assert m(x) is x and torch.equal(m(x, x), x + x) and m.calls == 0
    assert vit.Dropout(0.1, seed=(1 << 64) - 2).seed == vit.Dropout(0.1, seed=-2).state[0] == -2
    m = vit.vit_l14(dim=64, depth=3, heads=1, hidden=64, img=28)
    names = set(m.state_dict())
    with pytest.raises(ValueError, match="rates"):
        vit.set_dropout(m, drop_path=[0.1])
    vit.set_dropout(m, 0.1, [0.0, 0.1, 0.2], seed=7)
    b = m.backbone.blocks
    assert b[0].drop_path is None and b[2].drop_path.p == 0.2 and b[1].drop_path.per == "sample"
    assert not b[0].attn.proj_drop.active and type(b[1].mlp.drop) is vit.Dropout
    index = [d.index for d in m.modules() if type(d) is vit.Dropout]
    assert len(set(index)) == len(index) == 8
    assert set(m.state_dict()) == names  # (checkpoints load either way)
    m.train()
    assert b[0].attn.proj_drop.active
    assert copy.deepcopy(b[2]).drop_path.seed == 7
    vit.set_dropout(m)
    assert not any(type(d) is vit.Dropout for d in m.modules())


def test_module_refused_inside_a_backward_pass():
    """A recomputation would draw the next mask, not the first call's."""
    m = vit.Dropout(0.5)
    message = []

    class Recomputed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 1

        @staticmethod
        def backward(ctx, dy):
            with pytest.raises(RuntimeError, match="inside a backward pass") as e:
                m(dy)
            message.append(e.value)
            return m.eval()(dy)  # (what drops nothing may be called)

    x = torch.ones(3, requires_grad=True)
    Recomputed.apply(x).sum().backward()
    assert message and m.calls == 0 and torch.equal(x.grad, torch.ones(3))


def test_module_refused_where_torch_does_not_tell(monkeypatch):
    """Without the query a recomputation would draw another mask in silence."""
    from scmp_vit_b200 import _call
    monkeypatch.setattr(_call, "_graph_task", None)
    m, x = vit.Dropout(0.5), torch.ones(3)
    with pytest.raises(RuntimeError, match="does not tell"):
        m(x)
    assert m.calls == 0 and m.eval()(x) is x


@pytest.fixture
def offsets(monkeypatch):
    """Dropout modules record the offsets of their calls instead of launching."""
    seen = []
    monkeypatch.setattr(vit, "dropout", lambda x, p, seed, offset, **kw: (seen.append(offset), x)[1])
    return seen


def test_threads_take_a_mask_each(offsets):
    """No two calls of a shared module draw the same mask."""
    m, x = vit.Dropout(0.5, index=1), torch.ones(2)
    old, go = sys.getswitchinterval(), threading.Barrier(8)

    def run():
        go.wait()
        for _ in range(1500):
            m(x)
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=run) for _ in range(8)]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sys.setswitchinterval(old)
    assert sorted(offsets) == [(1 << 48) + i for i in range(12000)] and m.calls == 12000


def test_data_parallel_replicas_draw_on(offsets, monkeypatch):
    """Replicas live for one call: what they count stays with the module, on each
    device a sequence of its own."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: int(t[0]))
    m = vit.Dropout(0.5, index=2)
    for step in range(2):
        for device in (1, 0):
            m._replicate_for_data_parallel()(torch.tensor([float(device)]))
    assert offsets == [(2 << 48) + (d + 1 << 40) + i for i in range(2) for d in (1, 0)]
    m(torch.ones(1))
    assert offsets[4:] == [2 << 48] and m.calls == 2
    for c in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        c(torch.ones(1))
        assert offsets[-1] == (2 << 48) + 2 and c.calls == 3 and m.calls == 2
    m.calls = 7
    m(torch.ones(1))
    m._replicate_for_data_parallel()(torch.zeros(1))
    assert offsets[-2:] == [(2 << 48) + 7, (2 << 48) + (1 << 40) + 7] and m.calls == 8

def saved(module):
    """Its state dict, written to a file and read again."""
    f = io.BytesIO()
    torch.save(module.state_dict(), f)
    f.seek(0)
    return torch.load(f, weights_only=True)


def test_a_resumed_run_draws_on(offsets):
    """Counts go with the state dict, whose keys stay; models with and without dropout
    load each other's."""
    def model():
        m = torch.nn.Sequential(torch.nn.Linear(2, 2), vit.Dropout(0.5, index=1),
                                torch.nn.Sequential(vit.Dropout(0.5, index=2)))
        return m.train()
    m, x = model(), torch.ones(1, 2)
    for _ in range(3):
        m(x)
    m[1](x)
    state = saved(m)
    assert set(state) == {"0.weight", "0.bias"}
    again = model()
    again.load_state_dict(state)
    del offsets[:]
    again(x)
    assert offsets == [(1 << 48) + 4, (2 << 48) + 3]
    assert (m[1].calls, m[2][0].calls) == (4, 3)
    plain = torch.nn.Sequential(torch.nn.Linear(2, 2), torch.nn.Identity(), torch.nn.Identity())
    plain.load_state_dict(state)
    again.load_state_dict(saved(plain))
    again.load_state_dict(dict(state))  # (no metadata: the counts stay)
    assert (again[1].calls, again[2][0].calls) == (5, 4)
    with torch.no_grad():  # captured calls count in `state`
        m[1].state[1], m[1]._captured = 9, True
    again.load_state_dict(saved(m))
    assert int(again[1].state[1]) == 9 and int(again[2][0].state[1]) == 0
    assert saved(again)._metadata["1"]["captured"] == 9



def test_modules_saved_whole_before_replicas_counted():
    m = vit.Dropout(0.5)
    state = m.__dict__.copy()
    del state["_calls"]
    old = vit.Dropout.__new__(vit.Dropout)
    old.__setstate__(dict(state, calls=5))
    assert old.calls == 5 and old._calls.take() == 5 and old.calls == 6


def _rank(rank, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2,
                            timeout=datetime.timedelta(seconds=60))
    m = torch.nn.Sequential(torch.nn.Linear(2, 2), vit.Dropout(0.5, seed=10 + rank)).eval()
    wrapped = torch.nn.parallel.DistributedDataParallel(m)
    wrapped(torch.ones(1, 2)).sum().backward()
    q.put((rank, m[1].state.tolist()))
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_keep_their_seeds():
    """What a data-parallel wrapper makes alike on all ranks leaves the seeds apart."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ranks = [ctx.Process(target=_rank, args=(r, port, q)) for r in range(2)]
    [r.start() for r in ranks]
    got = dict(q.get(timeout=120) for _ in ranks)
    [r.join(60) for r in ranks]
    assert got == {0: [10, 0], 1: [11, 0]} and all(r.exitcode == 0 for r in ranks)


def test_the_captured_state_moves_with_its_module():
    m = torch.nn.Sequential(vit.Dropout(0.5, seed=-4))
    assert not list(m.buffers()) and m.half()[0].state.tolist() == [-4, 0]
    m[0].state[1] = 3
    assert copy.deepcopy(m)[0].state.tolist() == [-4, 3]
    assert m.to_empty(device="cpu")[0].state.tolist() == [-4, 3]
    assert m.to("meta")[0].state.is_meta
    assert m.to_empty(device="cpu")[0].state.tolist() == [-4, 0]
    d = vit.Dropout(0.5, seed=5)  # (the module itself, which passes `recurse` on)
    assert d.to_empty(device="meta", recurse=False).state.is_meta
    assert d.to_empty(device="cpu").state.tolist() == [5, 0]
    old = vit.Dropout(0.5, seed=6)  # as earlier versions kept it
    state = dict(old.__dict__, _buffers={"state": old.state}, _non_persistent_buffers_set={"state"})
    del state["state"]
    new = vit.Dropout.__new__(vit.Dropout)
    new.__setstate__(state)
    assert new.state.tolist() == [6, 0] and not list(new.buffers())


# ------------------------------------------------------------ GPU

@pytest.mark.gpu
@pytest.mark.parametrize("per", vit.PER)
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 8), (3, 5, 9), (2, 257, 64), (4, 1, 1000),
                                   (5, 3, 2, 24), (130, 2), (2, 3001)])
def test_values_and_gradients(cuda_device, shape, per):
    g = torch.Generator().manual_seed(sum(shape))
    for i, dtype in enumerate(DTYPES):
        for p, seed, offset in ((0.1, 12345, 0), (0.5, -3, (1 << 63) + 17), (0.0, 9, 1),
                                (1.0, 1, 2), (0.9, (1 << 64) - 1, (1 << 32) - 1)):
            x, r, dy = (torch.randn(*shape, generator=g).to(dtype).to(cuda_device)
                        for _ in range(3))
            x.requires_grad_(), r.requires_grad_()
            y = vit.dropout(x, p, seed, offset, per=per)
            assert torch.equal(y, expect(x, p, seed, offset, per))
            (dx,) = torch.autograd.grad(y, x, dy)
            assert torch.equal(dx, expect(dy, p, seed, offset, per))
            y = vit.dropout(x, p, seed, offset, per=per, residual=r)
            assert torch.equal(y, expect(x, p, seed, offset, per, r))
            dx2, dr = torch.autograd.grad(y, (x, r), dy)
            assert torch.equal(dx2, dx) and torch.equal(dr, dy)


@pytest.mark.gpu
def test_large_strided_and_unaligned(cuda_device):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3000, 2100, generator=g).bfloat16().to(cuda_device)
    for per in vit.PER:
        assert torch.equal(vit.dropout(x, 0.3, 5, 6, per=per), expect(x, 0.3, 5, 6, per))
    y = vit.dropout(x, 0.5, 5, 6)
    assert abs(float((y == 0).float().mean()) - 0.5) < 5 * 0.5 / math.sqrt(x.numel())
    for t in (x[:40, 1:], x[:40, ::2], x[:40].t(), x.reshape(-1)[1:8001], x[:1].expand(7, 2100)):
        for per in vit.PER:
            assert torch.equal(vit.dropout(t, 0.3, 5, 6, per=per, residual=t),
                               expect(t, 0.3, 5, 6, per, t))
    assert vit.dropout(x[:0], 0.3, 5, per="sample").shape == (0, 2100)
    assert vit.dropout(x[:, :0], 0.3, 5, per="row").shape == (3000, 0)
    assert vit.dropout(x[0, 0], 0.0, 5).shape == ()


@pytest.mark.gpu
def test_gradient_by_differences(cuda_device):
    """Linear in x: with whole numbers and p = 1/2, differences are exact."""
    x = torch.arange(40.0, device=cuda_device).reshape(4, 10).requires_grad_()
    dy = torch.arange(40.0, device=cuda_device).reshape(4, 10) - 20
    (dx,) = torch.autograd.grad(vit.dropout(x, 0.5, 3), x, dy)
    with torch.no_grad():
        for at in ((0, 0), (1, 7), (3, 9), (2, 2)):
            f = []
            for step in (1.0, -1.0):
                x[at] += step
                f.append((vit.dropout(x, 0.5, 3) * dy).sum())
                x[at] -= step
            assert float(dx[at]) == float(f[0] - f[1]) / 2


@pytest.mark.gpu
def test_dropped_values_leave_nothing(cuda_device):
    """A NaN or an infinity in a dropped place is 0, in both directions."""
    for bad in (math.nan, math.inf):
        x = torch.full((64, 32), bad, device=cuda_device)
        keep = keep_of((64, 32), 0.5, 1, 0, "element").to(cuda_device)
        y = vit.dropout(x, 0.5, 1)
        assert bool((y[~keep] == 0).all()) and not bool(y[keep].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("per", vit.PER)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_dropped_values_leave_nothing_either_way(cuda_device, dtype, bad, per):
    """The same of gradients, for every draw and type: what comes in at a dropped place
    is 0 in x's gradient and comes through in the residual's, whose value is y's there."""
    shape = (33, 7, 24)
    keep = keep_of(shape, 0.5, 1, 2, per).to(cuda_device)
    g = torch.Generator().manual_seed(7)
    x, r, dy = (torch.randn(*shape, generator=g).to(dtype).to(cuda_device) for _ in range(3))
    x[~keep] = bad
    dy[~keep] = bad
    leaves = [x.requires_grad_(), r.requires_grad_()]
    y = vit.dropout(x, 0.5, 1, 2, per=per, residual=r)
    assert torch.equal(y[~keep], r[~keep]) and bool(y.isfinite().all())
    dx, dr = torch.autograd.grad(y, leaves, dy)
    assert not dx[~keep].any() and torch.equal(dx[keep], 2 * dy[keep])
    assert torch.equal(dr.nan_to_num(7.0), dy.nan_to_num(7.0))
    y = vit.dropout(x, 0.5, 1, 2, per=per)
    (dx2,) = torch.autograd.grad(y, x, dy)
    assert not y[~keep].any() and torch.equal(dx2, dx)


@pytest.mark.gpu
def test_in_place_at_the_c_entry(cuda_device):
    """y may be x or residual."""
    x = torch.randn(1000, device=cuda_device)
    r = torch.randn(1000, device=cuda_device)
    want = vit.dropout(x, 0.3, 1, 2, residual=r)
    for y in (x.clone(), r.clone()):
        a = x.clone() if not torch.equal(y, x) else y
        b = r.clone() if not torch.equal(y, r) else y
        args = _lib.PACK_DROPOUT.pack(_lib.ABI_VERSION, 0, a.data_ptr(), b.data_ptr(),
                                      y.data_ptr(), 0, 1000, 1, 1, 2, 0.3)
        vit.call(_lib.load().scmp_dropout, 0, args)
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_seed_tensor_streams_and_graph(cuda_device):
    dev = cuda_device
    x = torch.randn(300, 70, device=dev)
    state = torch.tensor([-77, 1000], device=dev)
    assert torch.equal(vit.dropout(x, 0.4, state, 5), expect(x, 0.4, -77, 1005, "element"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = vit.dropout(x, 0.4, 8)
    side.synchronize()
    assert torch.equal(y, vit.dropout(x, 0.4, 8))
    leaf = x.clone().requires_grad_()
    y = vit.dropout(leaf, 0.4, state)
    state[1] += 1  # a seed tensor that moved on is noticed, not used
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()

    def step():
        leaf = x.detach().requires_grad_()
        y = vit.dropout(leaf, 0.4, state)
        return y.detach(), torch.autograd.grad(y, leaf, x)[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for more in (3, 4):
        state.copy_(torch.tensor([5, more]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expect(x, 0.4, 5, more, "element"))
        assert torch.equal(dx, expect(x, 0.4, 5, more, "element"))


@pytest.mark.gpu
def test_module_masks(cuda_device):
    """Every call its own mask, the same from the same seed; a captured call's
    replays too, none of them an eager call's."""
    x = torch.randn(64, 96, device=cuda_device)
    m = vit.Dropout(0.5, seed=3, index=2).to(cuda_device)
    a, b = m(x), m(x)
    assert not torch.equal(a, b)
    assert torch.equal(a, expect(x, 0.5, 3, 2 << 48, "element"))
    assert torch.equal(b, expect(x, 0.5, 3, (2 << 48) + 1, "element"))
    m.calls = 0
    assert torch.equal(m(x), a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
        z = m(x)
    seen = []
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for j, t in enumerate((y, z)):
            seen.append(t.clone())
            assert torch.equal(t, expect(x, 0.5, 3, (2 << 48) + (1 << 47) + 2 * i + j, "element"))
    assert all(not torch.equal(s, t) for i, s in enumerate(seen) for t in seen[:i])


@pytest.mark.gpu
def test_captured_masks_of_a_resumed_run(cuda_device):
    x = torch.randn(64, 96, device=cuda_device)
    m = vit.Dropout(0.5, seed=3, index=2).to(cuda_device)

    def captured(m):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x)
        return graph, y
    graph, y = captured(m)
    for _ in range(3):
        graph.replay()
    state = saved(m)
    for loaded_first in (True, False):
        n = vit.Dropout(0.5, seed=3, index=2).to(cuda_device)
        if loaded_first:
            n.load_state_dict(state)
        graph, y = captured(n)
        if not loaded_first:
            n.load_state_dict(state)
        for i in (3, 4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, expect(x, 0.5, 3, (2 << 48) + (1 << 47) + i, "element"))


def small(dev, **kw):
    m = vit.vit_l14(seed=0, dim=128, depth=2, heads=2, hidden=256, img=56, **kw).to(dev)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith("gamma"):
                p.add_(0.2)
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_in_the_blocks(cuda_device, fused):
    """A block's forward is the calls one by one; evaluation is untouched; without
    gradients (the fused glue's case) training mode still drops.  Fused norms sum
    in another order: fp32 sums of at most 256 terms, whose magnitudes add up to less
    than 6 here, are off by at most 256 2^-24 6 = 1e-4."""
    m = small(cuda_device)
    images = torch.randn(3, 3, 56, 56, device=cuda_device)
    ref = m(images)
    vit.set_dropout(m, 0.2, 0.5, seed=11)
    vit.set_fused_norm(fused)
    try:
        vit.set_fused_norm(False)
        assert torch.equal(m(images), ref)  # (m is in evaluation mode)
        vit.set_fused_norm(fused)
        m.train()
        x = torch.randn(3, 17, 128, device=cuda_device)
        blk = m.backbone.blocks[1]
        for grad in (True, False):
            for d in m.modules():
                if type(d) is vit.Dropout:
                    d.calls = 0
            with torch.set_grad_enabled(grad):
                got = blk(x)
                a = blk.attn
                a.proj_drop.calls = blk.mlp.drop.calls = 0
                y = a(blk.norm1(x))
                assert torch.equal(y == 0, expect(torch.ones_like(y), 0.2, 11, 3 << 48,
                                                  "element") == 0)
                y = vit.dropout(blk.ls1(y), 0.5, 11, 5 << 48, per="sample", residual=x)
                u = blk.mlp(blk.norm2(y))
                want = vit.dropout(blk.ls2(u), 0.5, 11, (5 << 48) + 1, per="sample", residual=y)
            torch.testing.assert_close(got, want, rtol=0, atol=1e-4 if fused else 0)
        m.zero_grad()
        m(images).square().sum().backward()
        assert all(p.grad is None or bool(p.grad.isfinite().all()) for p in m.parameters())
    finally:
        vit.set_fused_norm(False)


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_module_is_refused(cuda_device, reentrant):
    """With an offset of the caller's own a checkpoint repeats the mask."""
    from torch.utils.checkpoint import checkpoint

    x = torch.randn(5, 40, device=cuda_device, requires_grad=True)
    m = vit.Dropout(0.5)
    with pytest.raises(RuntimeError, match="inside a backward pass"):
        checkpoint(lambda t: m(t).square(), x, use_reentrant=reentrant).sum().backward()

    def f(t):
        return vit.dropout(t, 0.5, 3, 4).square().sum()

    checkpoint(f, x, use_reentrant=reentrant).backward()
    want = x.detach().clone().requires_grad_()
    f(want).backward()
    assert torch.equal(x.grad, want.grad)


@pytest.mark.gpu
def test_more_elements_than_32_bits(cuda_device):
    """Past 2^31 elements counters are 64 bits wide; the ends and the middle."""
    n = (1 << 31) + 40
    if torch.cuda.mem_get_info()[0] < 6 * n:
        pytest.skip("needs 13 GB of device memory")
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda_device)
    y = vit.dropout(x, 0.5, 21, 22)
    z = vit.dropout(x.view(8, n // 8), 0.5, 21, 22, per="sample")
    row = words(8, 21, 22)
    for at in (0, 1 << 30, (1 << 31) - 20, n - 36):
        keep = torch.from_numpy(words(36, 21, 22, at) >= np.uint64(1 << 31))
        assert torch.equal(y[at:at + 36].cpu() != 0, keep)
        assert torch.equal(z.view(-1)[at:at + 36].cpu() != 0, torch.from_numpy(
            row[np.arange(at, at + 36) // (n // 8)] >= np.uint64(1 << 31)))
