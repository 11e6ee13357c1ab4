"""Microscaled 4-bit operands without a GPU: the oracle against the GGUF container's own decoder,
operand checks, and the refusals of the C entry points (perm_b200/mx4.py)."""
import copy
import ctypes
import io
import pickle

import numpy as np
import pytest
import torch

import mx4_oracle as mo
from perm_b200 import _native as nat
from perm_b200 import mx4


def test_oracle_container_decodes_as_gguf_does():
    import gguf
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((5, 256)) * np.exp(rng.standard_normal((5, 1)))).astype(np.float32)
    codes, byte = mo.quantize(x, "MXFP4")
    got = gguf.dequantize(mo.container(codes, byte), gguf.GGMLQuantizationType.MXFP4)
    assert np.array_equal(got.astype(np.float64), mo.values(codes, byte, "MXFP4"))


def test_oracle_pack_round_trips():
    rng = np.random.default_rng(1)
    for fmt in mo.BLOCK:
        for rows, n in ((1, 5), (130, 300), (257, 512)):
            codes, byte = mo.quantize(rng.standard_normal((rows, n)), fmt)
            c, s = mo.pack(codes, byte, fmt, n)
            c2, b2 = mo.unpack(c, s, fmt, rows, n)
            assert np.array_equal(c2[:, :codes.shape[1]], codes) and np.array_equal(b2[:, :byte.shape[1]], byte)
            assert c.size == nat.lib().cp_mx4_codes_bytes(rows, n)
            assert s.size == nat.lib().cp_mx4_scales_bytes(nat.MX4_ID[fmt], rows, n)


def test_operand_checks():
    def make(rows=3, n=300, fmt="MXFP4", g=1.0, codes=None, scales=None):
        c = torch.zeros((3, 256), dtype=torch.uint8) if codes is None else codes
        s = torch.zeros((1, 4, 32, 4, 4), dtype=torch.uint8) if scales is None else scales
        return mx4.Mx4Tensor(c, s, fmt, rows, n, g)
    q = make()
    assert q.shape == (3, 300) and "MXFP4" in repr(q)
    for kw in (dict(fmt="MXFP8"), dict(rows=4), dict(n=0), dict(n=600), dict(fmt="NVFP4"), dict(g=0.0), dict(g=-1.0),
               dict(g=float("nan")), dict(g=float("inf")), dict(codes=torch.zeros((3, 256))),
               dict(codes=torch.zeros((3, 512), dtype=torch.uint8)[:, ::2]),
               dict(scales=torch.zeros((2, 4, 32, 4, 4), dtype=torch.uint8))):
        with pytest.raises(ValueError):
            make(**kw)


def _saved(q):
    f = io.BytesIO()
    torch.save({"w": q}, f)
    f.seek(0)
    return torch.load(f, weights_only=False)["w"]


@pytest.mark.parametrize("rows", [0, 3, 130])
@pytest.mark.parametrize("fmt", mo.BLOCK)
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)), _saved],
                         ids=["copy", "deepcopy", "pickle", "save"])
def test_copies_of_an_operand_point_to_their_own_tensors(how, fmt, rows):
    """The addresses that the kernels get are those of the copy's codes and scales, for operands of two
    tensors and of one buffer."""
    c = torch.randint(0, 256, (rows, 256), dtype=torch.uint8)
    s = torch.randint(0, 256, ((rows + 127) // 128, 512 // (4 * mo.BLOCK[fmt]), 32, 4, 4), dtype=torch.uint8)
    g = 0.5 if fmt == "NVFP4" else 1.0
    two = mx4.Mx4Tensor(c.clone(), s.clone(), fmt, rows, 300, g)
    one = mx4.Mx4Tensor._new(torch.empty(0), fmt, rows, 300, g)
    one.codes.copy_(c)
    one.scales.copy_(s)
    for q in (two, one):
        k = how(q)
        assert k._cp == k.codes.data_ptr() and k._sp == k.scales.data_ptr() and k.dev == q.dev
        assert torch.equal(k.codes, c) and torch.equal(k.scales, s)
        assert (k.fmt, k.shape, k.tensor_scale) == (fmt, (rows, 300), g)
        if how is not copy.copy:
            q.codes.fill_(0x11)                       # a copy has storage of its own
            q.scales.fill_(0x11)
            assert torch.equal(k.codes, c) and torch.equal(k.scales, s)


def test_host_tensors_are_refused():
    q = mx4.Mx4Tensor(torch.zeros((3, 128), dtype=torch.uint8), torch.zeros((1, 2, 32, 4, 4), dtype=torch.uint8), "MXFP4", 3, 64)
    x = torch.zeros(2, 64)
    for call in (lambda: mx4.quantize(x, "MXFP4"), lambda: mx4.dequantize(q), lambda: mx4.matmul(q, q),
                 lambda: mx4.linear(x, q), lambda: mx4.linear_grad(torch.zeros(2, 3), q),
                 lambda: mx4.from_gguf(torch.zeros((1, 34), dtype=torch.uint8), 64)):
        with pytest.raises(nat.CudaPathError):
            call()


def test_argument_checks_need_no_gpu():
    q = mx4.Mx4Tensor(torch.zeros((3, 128), dtype=torch.uint8), torch.zeros((1, 2, 32, 4, 4), dtype=torch.uint8), "MXFP4", 3, 64)
    r = mx4.Mx4Tensor(torch.zeros((3, 128), dtype=torch.uint8), torch.zeros((1, 2, 32, 4, 4), dtype=torch.uint8), "MXFP4", 3, 65)
    with pytest.raises(ValueError):
        mx4.matmul(q, r)
    with pytest.raises(ValueError):
        mx4.matmul(q, q, torch.float64)
    with pytest.raises(ValueError):
        mx4.dequantize(q, torch.int8)
    with pytest.raises(ValueError):
        mx4.linear(torch.zeros(2, 65), q)
    with pytest.raises(ValueError):
        mx4.linear(torch.zeros(2, 64, dtype=torch.float64), q)
    with pytest.raises(ValueError):
        mx4.linear_grad(torch.zeros(2, 64), q)
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(2, 64), "FP4")


def test_c_entry_points_refuse():
    L = nat.lib()
    buf = ctypes.create_string_buffer(4096 + 64)
    p = (ctypes.addressof(buf) + 63) // 64 * 64        # never dereferenced: every call below is refused first
    MX, NV, BF = nat.MX4_ID["MXFP4"], nat.MX4_ID["NVFP4"], nat.CP_MX4_BF16
    quant = lambda f=MX, d=BF, x=p, rows=2, n=64, ld=64, g=1.0, c=p, s=p: L.cp_mx4_quantize(f, d, x, rows, n, ld, None, g, c, s, None)  # noqa: E731
    assert quant(f=41) == nat.CP_ERR_TYPE and quant(d=7) == nat.CP_ERR_TYPE
    assert quant(rows=-1) == nat.CP_ERR_SHAPE and quant(n=0) == nat.CP_ERR_SHAPE and quant(ld=63) == nat.CP_ERR_SHAPE
    assert quant(rows=1 << 40) == nat.CP_ERR_SHAPE
    assert quant(g=2.0) == nat.CP_ERR_ARG                       # MXFP4 has no tensor scale
    for g in (3.0, 0.0, -1.0, float("nan"), float("inf"), 2.0 ** 110):
        assert quant(f=NV, g=g) == nat.CP_ERR_ARG
    assert quant(x=None) == nat.CP_ERR_ARG and quant(c=p + 8) == nat.CP_ERR_ARG and quant(x=p + 1) == nat.CP_ERR_ARG
    assert quant(rows=0) == nat.CP_OK
    deq = lambda f=MX, d=BF, c=p, n=64, o=p: L.cp_mx4_dequantize(f, c, p, 2, n, 1.0, d, o, None)  # noqa: E731
    assert deq(f=8) == nat.CP_ERR_TYPE and deq(d=-1) == nat.CP_ERR_TYPE and deq(n=-4) == nat.CP_ERR_SHAPE
    assert deq(c=None) == nat.CP_ERR_ARG and deq(o=p + 1) == nat.CP_ERR_ARG
    assert L.cp_mx4_from_gguf(p, 2, 48, p, p, None) == nat.CP_ERR_SHAPE
    assert L.cp_mx4_from_gguf(None, 2, 64, p, p, None) == nat.CP_ERR_ARG
    mm = lambda f=MX, a=p, n=64, d=BF, y=p, t=2: L.cp_mx4_matmul(f, a, p, t, p, p, 3, n, 1.0, d, y, None)  # noqa: E731
    assert mm(f=2) == nat.CP_ERR_TYPE and mm(d=3) == nat.CP_ERR_TYPE and mm(n=0) == nat.CP_ERR_SHAPE
    assert mm(a=p + 4) == nat.CP_ERR_ARG and mm(y=None) == nat.CP_ERR_ARG and mm(t=0) == nat.CP_OK
    lin = lambda f=MX, d=BF, x=p, T=2, ld=64, tr=0, y=p, ws=None, wsb=0: L.cp_mx4_linear(  # noqa: E731
        f, d, x, T, ld, p, p, 64, 64, 1.0, tr, y, ws, wsb, None)
    assert lin(f=0) == nat.CP_ERR_TYPE and lin(d=9) == nat.CP_ERR_TYPE and lin(T=-1) == nat.CP_ERR_SHAPE
    assert lin(ld=60) == nat.CP_ERR_SHAPE and lin(x=None) == nat.CP_ERR_ARG and lin(y=p + 1) == nat.CP_ERR_ARG
    assert lin(T=0) == nat.CP_OK
    big = L.cp_mx4_linear_workspace_bytes(nat.CP_MX4_F32, p, 4096, 64, 64, 64, 0)
    if big:
        assert lin(d=nat.CP_MX4_F32, T=4096) == nat.CP_ERR_WORKSPACE
    # the container's entry points
    assert L.cp_kquant_encode(MX, p, 2, 48, None, p, None) == nat.CP_ERR_SHAPE
    assert L.cp_kquant_decode(MX, p + 1, 2, 64, p, None) == nat.CP_ERR_ARG
    assert L.cp_kquant_encode(NV, p, 2, 64, None, p, None) == nat.CP_ERR_TYPE
    assert L.cp_grid_params(MX, p, 2, 256, p, p, None) == nat.CP_ERR_TYPE
    assert L.cp_block_bytes(MX) == 17


@pytest.mark.parametrize("tt", ["MXFP4", "Q8_0", "Q2_K"])
def test_codec_refuses_buffers_that_are_too_small(tt):
    """Fewer container bytes than the rows take, and column weights of another length, would be read past their end."""
    from perm_b200 import kquant as kq
    per = kq.row_bytes(tt, 512)
    for raw in (torch.zeros((3, per - 1), dtype=torch.uint8), torch.zeros(3 * per, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            kq.dequantize_dev(tt, raw, 512)
    for qw in (torch.ones(511), torch.ones(1), torch.ones(1024)):
        with pytest.raises(ValueError):
            kq.quantize_dev(tt, torch.zeros(3, 512), qw)


def _module(fmt, g, seed):
    rng = np.random.default_rng(seed)
    c, s = mo.pack(*mo.quantize(rng.standard_normal((5, 70)), fmt, g), fmt, 70)
    return mx4.Linear(mx4.Mx4Tensor(torch.from_numpy(c), torch.from_numpy(s), fmt, 5, 70, g), torch.full((5,), float(seed)))


def test_a_saved_module_keeps_its_tensor_scale():
    a, b = _module("NVFP4", 0.25, 1), _module("NVFP4", 1.0, 2)
    f = io.BytesIO()
    torch.save(a.state_dict(), f)
    f.seek(0)
    assert not any(b.load_state_dict(torch.load(f))), "all keys match"
    assert b.tensor_scale == 0.25 and b.weight4.tensor_scale == 0.25
    assert torch.equal(b.codes, a.codes) and torch.equal(b.scales, a.scales) and torch.equal(b.bias, a.bias)
    nested = torch.nn.Sequential(_module("NVFP4", 2.0, 3))
    nested.load_state_dict(torch.nn.Sequential(a).state_dict())
    assert nested[0].tensor_scale == 0.25
    assert copy.deepcopy(a).tensor_scale == 0.25 and pickle.loads(pickle.dumps(a)).weight4.tensor_scale == 0.25


def test_a_saved_module_of_another_format_or_without_its_scale_is_refused():
    a = _module("NVFP4", 0.25, 1)
    with pytest.raises((ValueError, RuntimeError)):
        _module("MXFP4", 1.0, 2).load_state_dict(a.state_dict())
    part = {k: v for k, v in a.state_dict().items() if "extra" not in k}
    with pytest.raises(RuntimeError):
        _module("NVFP4", 1.0, 2).load_state_dict(part)
    one = _module("MXFP4", 1.0, 2)
    with pytest.raises(ValueError):
        one.set_extra_state(a.get_extra_state())


def test_forward_mode_derivatives(monkeypatch):
    """linear's tangent, the tangent of its gradient (forward over reverse), and differences, with a plain
    product in the place of the kernels'."""
    import torch.autograd.forward_ad as fw
    W = torch.randn(5, 7, dtype=torch.float64)
    monkeypatch.setattr(mx4, "_product", lambda x, w, t, what: x.detach() @ (W if t else W.T))
    q = mx4.Mx4Tensor._new(torch.empty(0), "MXFP4", 5, 7, 1.0)
    x, t = torch.randn(3, 7, dtype=torch.float64), torch.randn(3, 7, dtype=torch.float64)
    v, u = torch.randn(3, 5, dtype=torch.float64), torch.randn(3, 5, dtype=torch.float64)
    with fw.dual_level():
        assert torch.equal(fw.unpack_dual(mx4.linear(fw.make_dual(x, t), q)).tangent, t @ W.T)
        assert torch.equal(fw.unpack_dual(mx4.linear_grad(fw.make_dual(v, u), q)).tangent, u @ W)
        assert fw.unpack_dual(mx4.linear(x, q)).tangent is None
        d = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(mx4.linear(d, q), d, fw.make_dual(v, u))
        assert torch.equal(fw.unpack_dual(g).tangent, u @ W)
    leaf = x.clone().requires_grad_(True)
    assert torch.autograd.gradcheck(lambda z: mx4.linear(z, q), (leaf,), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(lambda z: mx4.linear(z, q), (leaf,), check_fwd_over_rev=True)
    for f in (lambda: torch.func.jvp(lambda z: mx4.linear(z, q), (x,), (t,)),
              lambda: torch.func.grad(lambda z: mx4.linear(z, q).sum())(x)):
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("buffer", [False, True])
def test_weights_written_between_forward_and_backward(monkeypatch, buffer):
    """They are saved tensors: a write in place is noticed, hooks see them and what a hook gives back is used."""
    seen = []
    monkeypatch.setattr(mx4, "_product", lambda x, w, t, what: seen.append(w) or x.new_zeros(x.shape[0], w.n if t else w.rows))
    q = mx4.Mx4Tensor._new(torch.empty(0), "MXFP4", 5, 7, 1.0)
    q.codes.zero_(), q.scales.zero_()
    if not buffer:
        q = copy.copy(q)
    x = torch.zeros(3, 7, requires_grad=True)
    mx4.linear(x, q).sum().backward()
    assert seen[-1] is q
    y = mx4.linear(x, q)
    q.codes.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.clone()) or packed[-1], lambda t: t):
        y = mx4.linear(x, q)
        assert sum(p.numel() for p in packed) >= q.codes.numel() + q.scales.numel()
        y.sum().backward()
    w = seen[-1]
    assert w is not q and w._cp == w.codes.data_ptr() != q._cp and torch.equal(w.codes, q.codes) and torch.equal(w.scales, q.scales)
    with torch.inference_mode():
        r = mx4.Mx4Tensor._new(torch.empty(0), "MXFP4", 5, 7, 1.0)
    mx4.linear(x, r).sum().backward()
    assert seen[-1] is r


def test_tensor_scales_outside_float32_are_refused():
    """The kernels take the scale of a result as one float32 number: beyond its range all of a result was infinite,
    NaN or zero."""
    def make(g):
        return mx4.Mx4Tensor(torch.zeros((3, 128), dtype=torch.uint8), torch.zeros((1, 4, 32, 4, 4), dtype=torch.uint8), "NVFP4", 3, 64, g)
    for g in (1e300, 2.0 ** 128, 2.0 ** -127, 1e-300):
        with pytest.raises(ValueError):
            make(g)
    for a, b in ((2.0 ** 99, 2.0 ** 29), (2.0 ** -100, 2.0 ** -27), (2.0 ** 99, 2.0 ** 99)):
        with pytest.raises(ValueError, match="product of the tensor scales"):
            mx4.matmul(make(a), make(b))
    for a, b in ((2.0 ** 99, 2.0 ** 28), (2.0 ** -100, 2.0 ** -26), (2.0 ** 99, 2.0 ** -99)):
        with pytest.raises(nat.CudaPathError):   # host operands: all that is wrong with these
            mx4.matmul(make(a), make(b))


def test_status_of_a_device_without_a_number_is_the_current_devices(monkeypatch):
    asked = []
    monkeypatch.setattr(nat, "torch_cuda", lambda: torch)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(mx4, "_call", lambda idx, fn, what: asked.append(idx))
    for dev in (None, "cuda", torch.device("cuda"), "cuda:1", torch.device("cuda", 0)):
        mx4.status(dev)
    assert asked == [3, 3, 3, 1, 0]


def test_inject_stall_checks_its_arguments():
    L = nat.lib()
    for skip, wait in ((-1, 5_000_000), (0, 10), (0, 999_999), (0, 2_000_000_001)):
        assert L.cp_mx4_inject_stall(skip, wait) == nat.CP_ERR_ARG
