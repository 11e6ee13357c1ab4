"""Microscaled 4-bit operators on the GPU against their definition in float64 (tests/mx4_oracle.py):
perm_b200.mx4, and MXFP4 in perm_b200.kquant."""
import numpy as np
import pytest
import torch

import mx4_oracle as mo
from perm_b200 import _native as nat
from perm_b200 import kquant as kq
from perm_b200 import mx4

pytestmark = pytest.mark.gpu

FMTS = ("MXFP4", "NVFP4")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half a step of each type, relative to the value
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def make_x(rows, n, seed, dtype=torch.float32, spread=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, n)) * np.exp(spread * rng.standard_normal((1, n)))
    return torch.from_numpy(x).to(dtype).cuda()


def operand(rows, n, fmt, seed, g=None):
    """A random operand and its values [rows, n] in float64."""
    rng = np.random.default_rng(seed)
    g = (2.0 ** -12 if fmt == "NVFP4" else 1.0) if g is None else g
    codes, byte = mo.quantize(0.05 * rng.standard_normal((rows, n)), fmt, g if fmt == "NVFP4" else 1.0)
    c, s = mo.pack(codes, byte, fmt, n)
    q = mx4.Mx4Tensor(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), fmt, rows, n, g)
    return q, mo.values(codes, byte, fmt, g, n)


def check_operand(q, x, g=1.0, qw=None):
    """codes and scale bytes of q are the oracle's for x, and the padding is zero."""
    codes, byte = mo.quantize(f64(x), q.fmt, g, None if qw is None else f64(qw))
    got_c, got_b = mo.unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), q.fmt, q.rows, q.n)
    nb = byte.shape[1]
    assert np.array_equal(got_b[:, :nb], byte)
    assert not got_b[:, nb:].any() and not got_c[:, nb:].any()
    # a zero's sign is free
    a, b = got_c[:, :nb], codes
    assert np.array_equal(np.where(a == 8, 0, a), np.where(b == 8, 0, b))


# ------------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 16), (3, 33), (33, 100), (128, 256), (130, 1000), (257, 264), (2, 4096)])
def test_quantize_matches_the_definition(fmt, dtype, rows, n):
    x = make_x(rows, n, rows * 1000 + n, DTYPES[dtype])
    g = 2.0 ** -5 if fmt == "NVFP4" else 1.0
    q = mx4.quantize(x, fmt, tensor_scale=g)
    check_operand(q, x, g)
    codes, byte = mo.quantize(f64(x), fmt, g)
    want = mo.values(codes, byte, fmt, g, n)
    for dt in DTYPES.values():
        got = mx4.dequantize(q, dt)
        # every value has at most six bits, so it is exact in each type unless it is below f16's range
        assert np.abs(f64(got) - want).max() <= (2.0 ** -25 if dt == torch.float16 else 0.0)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_and_borders(fmt):
    """Values on and one unit beside every border between two codes, for many block scales."""
    rng = np.random.default_rng(5)
    b = mo.BLOCK[fmt]
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    tops = np.concatenate([rng.uniform(0.01, 8, 200), mo.E4M3[8:120] * 6, 2.0 ** np.arange(-8, 9), 2.0 ** np.arange(-8, 9) * 1.75])
    x = np.zeros((len(tops), b), np.float32)
    x[:, 0] = tops
    s = mo.scale_value(mo.first_scale(np.abs(x.astype(np.float64)).max(1), fmt), fmt)
    for i in range(b - 1):
        v = (borders[i % 7] * s * (-1) ** i).astype(np.float32)
        v = v if i % 3 == 0 else np.nextafter(v, np.float32(100 if i % 3 == 1 else -100))
        x[:, i + 1] = np.where(np.abs(v) < tops, v, 0)
    xt = torch.from_numpy(x).cuda()
    check_operand(mx4.quantize(xt, fmt), xt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_scale_borders(fmt):
    """Block maxima on and beside the borders of the scale's own rounding."""
    mid = (mo.E4M3[1:] + mo.E4M3[:-1]) * 3.0                 # 6 x the midpoints: exact in float32
    v = np.concatenate([mid, mo.E4M3 * 6, [2688.0, 2700.0, 1e30, 3e38, 1e-30, 1e-38, 1e-45, 0.0]]).astype(np.float32)
    v = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(0))])
    v = v[np.isfinite(v)]
    x = np.zeros((len(v), mo.BLOCK[fmt]), np.float32)
    x[:, 3] = v
    xt = torch.from_numpy(x).cuda()
    check_operand(mx4.quantize(xt, fmt), xt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,n", [(1, 16), (5, 70), (140, 512), (40, 2000)])
def test_quantize_importance(fmt, rows, n):
    x = make_x(rows, n, 7 * rows + n) * 0.02
    qw = torch.exp(1.5 * torch.from_numpy(np.random.default_rng(n).standard_normal(n))).float().cuda()
    g = 2.0 ** -14 if fmt == "NVFP4" else 1.0
    check_operand(mx4.quantize(x, fmt, qw, g), x, g, qw)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_importance_ties(fmt):
    """Weights of zero, blocks that 4 bits hold exactly, and equal errors: the first candidate stays."""
    rng = np.random.default_rng(3)
    x = np.zeros((8, 256), np.float32)
    x[1] = mo.LEVELS[rng.integers(0, 8, 256)]                  # exact
    x[2] = rng.integers(-6, 7, 256)                            # ties (5 lies between 4 and 6)
    x[3:6] = rng.standard_normal((3, 256))
    x[6] = 5.0
    x[7, ::2] = 1e-20
    xt = torch.from_numpy(x).cuda()
    for qw in (np.zeros(256), np.ones(256), np.where(np.arange(256) % 64 < 32, 0.0, 1.0), np.full(256, 1e-35), np.full(256, 1e30)):
        qt = torch.from_numpy(qw.astype(np.float32)).cuda()
        check_operand(mx4.quantize(xt, fmt, qt), xt, 1.0, qt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_non_finite_blocks(fmt):
    x = make_x(4, 256, 11)
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 255] = float("-inf")
    for qw in (None, torch.ones(256, device="cuda")):
        q = mx4.quantize(x, fmt, qw)
        check_operand(q, x, 1.0, qw)
        v = f64(mx4.dequantize(q))
        b = mo.BLOCK[fmt]
        bad = ~np.isfinite(f64(x)).reshape(4, -1, b).all(2)
        assert np.array_equal(np.isnan(v).reshape(4, -1, b).all(2), bad) and np.isnan(v).sum() == bad.sum() * b


def test_quantize_strides():
    base = make_x(70, 600, 13, torch.bfloat16)
    for x in (base[:, :300], base[::2, 8:508], base[3:, 1:258], base.t()[:300], base[:1].expand(5, 600)):
        check_operand(mx4.quantize(x, "MXFP4"), x)
    assert mx4.quantize(base[:0], "NVFP4").shape == (0, 600)
    assert mx4.dequantize(mx4.quantize(base[:0], "NVFP4")).shape == (0, 600)


def test_tensor_scale_for():
    for m in (1e-6, 0.1, 2688.0, 2689.0, 1e20):
        x = torch.tensor([[m, -m / 3]], device="cuda")
        g = mx4.tensor_scale_for(x)
        assert float(x[0, 0]) <= 2688.0 * g < 2.000001 * float(x[0, 0])
        assert not torch.isnan(mx4.dequantize(mx4.quantize(x, "NVFP4", tensor_scale=g))).any()
    assert mx4.tensor_scale_for(torch.zeros(3, 3, device="cuda")) == 1.0


# ------------------------------------------------------------------------------- container

@pytest.mark.parametrize("rows,n", [(1, 32), (3, 96), (65, 512), (7, 4096)])
@pytest.mark.parametrize("weighted", [False, True])
def test_container_matches_the_definition(rows, n, weighted):
    import gguf
    x = f64(make_x(rows, n, rows + n)).astype(np.float32) * np.float32(0.02)
    qw = np.exp(np.random.default_rng(n).standard_normal(n)).astype(np.float32) if weighted else None
    codes, byte = mo.quantize(x, "MXFP4", 1.0, qw)
    raw = kq.QUANTIZE["MXFP4"](x, qw)
    want = mo.container(np.where(codes == 8, 0, codes), byte)
    got_c = raw.reshape(rows, -1, 17)
    assert np.array_equal(got_c[..., 0], byte)
    assert np.array_equal(kq.DEQUANTIZE["MXFP4"](raw, n).astype(np.float64), mo.values(codes, byte, "MXFP4"))
    assert np.array_equal(gguf.dequantize(raw, gguf.GGMLQuantizationType.MXFP4), kq.DEQUANTIZE["MXFP4"](want, n))
    assert np.array_equal(kq.roundtrip(x, "MXFP4", qw), kq.DEQUANTIZE["MXFP4"](raw, n))
    q = mx4.from_gguf(torch.from_numpy(raw).cuda(), n)
    assert np.array_equal(f64(mx4.dequantize(q)), mo.values(codes, byte, "MXFP4"))
    same = mx4.quantize(torch.from_numpy(x).cuda(), "MXFP4", None if qw is None else torch.from_numpy(qw).cuda())
    assert torch.equal(q.codes, same.codes)


def test_container_checks():
    assert kq.QUANTIZE["MXFP4"](np.zeros((0, 64), np.float32), None).shape == (0, 34)
    with pytest.raises(ValueError):
        kq.QUANTIZE["MXFP4"](np.zeros((2, 40), np.float32), None)
    with pytest.raises(ValueError):
        mx4.from_gguf(torch.zeros((2, 17), dtype=torch.uint8, device="cuda"), 64)


def test_container_weighted_error_and_objective():
    from perm_b200 import objective
    x = f64(make_x(37, 512, 2)).astype(np.float32)
    qw = np.exp(np.random.default_rng(4).standard_normal(512)).astype(np.float32)
    codes, byte = mo.quantize(x, "MXFP4", 1.0, qw)
    want = float(((mo.values(codes, byte, "MXFP4") - x) ** 2 * qw.astype(np.float64)).sum())
    assert abs(objective.tensor_err(x, "MXFP4", qw) - want) <= 1e-12 * want
    raw = torch.from_numpy(kq.QUANTIZE["MXFP4"](x, qw)).cuda()
    err = torch.full((1,), 3.0, dtype=torch.float64, device="cuda")
    xt, qt = torch.from_numpy(x).cuda(), torch.from_numpy(qw).cuda()
    nat.check(nat.lib().cp_weighted_err(39, nat.ptr(raw), nat.ptr(xt), nat.ptr(qt), 37, 512, nat.ptr(err),
                                        nat.stream_ptr(torch)))
    assert abs(err.item() - want) <= 1e-12 * want


def test_encode_gguf_with_an_mxfp4_target(tmp_path):
    """A target whose tensors are MXFP4 and Q4_K: MXFP4 ones are fitted with the imatrix."""
    import gguf
    import gguf_fixtures as fx
    from perm_b200 import ef, gguf_io
    rng = np.random.default_rng(9)
    names = {"blk.0.attn_q.weight": "MXFP4", "blk.0.ffn_up.weight": "Q4_K"}
    w = {k: (rng.standard_normal((64, 256)) * 0.02).astype(np.float16) for k in names}
    src, tgt, out, im = (str(tmp_path / f) for f in ("src.gguf", "tgt.gguf", "out.gguf", "im.gguf"))
    ws = gguf.GGUFWriter(src, "qwen3")
    wt = gguf.GGUFWriter(tgt, "qwen3")
    for k, tt in names.items():
        ws.add_tensor(k, w[k])
        raw = kq.QUANTIZE[tt](w[k].astype(np.float32), None)
        wt.add_tensor(k, raw, raw_dtype=getattr(gguf.GGMLQuantizationType, tt))
    for g in (ws, wt):
        g.write_header_to_file(); g.write_kv_data_to_file(); g.write_tensors_to_file(); g.close()
    fx.write_imatrix(im, [(k, 256) for k in names])
    # the MXFP4 tensor has a Hessian too: error feedback covers the k-quants only, so it is fitted
    gguf_io.save_hessians({"blk.0.attn_q.weight": {"H": np.eye(256, dtype=np.float32), "n": 1}}, str(tmp_path / "h"))
    st = ef.encode_gguf(src, tgt, str(tmp_path / "h"), out, imatrix_path=im, log=lambda *_: None)
    assert st["blk.0.attn_q.weight"]["type"] == "MXFP4" and st["blk.0.attn_q.weight"]["mode"] == "wRTN"
    means = gguf_io.imatrix_means(im)
    for t in gguf.GGUFReader(out).tensors:
        want = kq.QUANTIZE[names[t.name]](w[t.name].astype(np.float32), means[t.name])
        assert np.array_equal(np.asarray(t.data).reshape(want.shape), want)


# ------------------------------------------------------------------------------- products

def chain(K):
    """Error of a float32 accumulation of K products, in units of sum |x w|: tensor cores add groups of
    at least 16 products with a relative error below 2^-22 a step, and partial sums are joined in a
    few more."""
    return (K / 16 + 32) * 2.0 ** -22


def check_product(got, x, w, out_dtype, extra=0.0):
    want, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = HALF[out_dtype] * np.abs(want) + chain(x.shape[1]) * mag * (1 + HALF[out_dtype]) + extra
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -25
    bad = np.abs(f64(got) - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(f64(got) - want).max(), int(bad.sum()))


SHAPES = [(1, 1, 1), (1, 64, 32), (2, 100, 33), (7, 130, 257), (16, 300, 512), (17, 128, 256), (33, 520, 1000), (65, 257, 264),
          (128, 256, 256), (129, 64, 2050), (300, 384, 768), (5, 4096, 512), (260, 1300, 130)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,out,n", SHAPES)
def test_matmul(fmt, dtype, T, out, n):
    a, av = operand(T, n, fmt, T + n, 2.0 ** -10 if fmt == "NVFP4" else 1.0)
    w, wv = operand(out, n, fmt, out + n)
    check_product(mx4.matmul(a, w, DTYPES[dtype]), av, wv, DTYPES[dtype])
    mx4.status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,out,n", SHAPES)
def test_linear_and_its_gradient(fmt, dtype, T, out, n):
    dt = DTYPES[dtype]
    w, wv = operand(out, n, fmt, out + n)
    x = make_x(T, n, T + out, dt, 0.5).requires_grad_(True)
    y = mx4.linear(x, w)
    assert y.shape == (T, out) and y.dtype == dt
    check_product(y, f64(x), wv, dt)
    dy = make_x(T, out, T * 3 + out, dt, 0.5)
    dx, = torch.autograd.grad(y, x, dy)
    assert dx.shape == (T, n) and dx.dtype == dt
    check_product(dx, f64(dy), wv.T, dt)
    mx4.status()


# every launch variant: few tokens with x converted ahead, SM pairs, and weights decoded first
VARIANTS = [(16, 8200, 2048), (3, 14400, 4100), (130, 14336, 256), (512, 14340, 200), (600, 300, 200), (545, 1030, 530)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,out,n", VARIANTS)
def test_products_in_every_variant(fmt, dtype, T, out, n):
    dt = DTYPES[dtype]
    w, wv = operand(out, n, fmt, out + n)
    x = make_x(T, n, T + out, dt, 0.5)
    check_product(mx4.linear(x, w), f64(x), wv, dt)
    dy = make_x(T, out, T * 3 + out, dt, 0.5)
    check_product(mx4.linear_grad(dy, w), f64(dy), wv.T, dt)
    a, av = operand(T, n, fmt, T + n, 2.0 ** -10 if fmt == "NVFP4" else 1.0)
    check_product(mx4.matmul(a, w, dt), av, wv, dt)
    mx4.status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out,n", [(2050, 12300), (12800, 2048)])
def test_many_tokens_with_weights_too_large_to_decode_first(fmt, dtype, out, n):
    dt, T = DTYPES[dtype], 560
    w, wv = operand(out, n, fmt, out + n)
    x = make_x(T, n, T + out, dt, 0.5)
    check_product(mx4.linear(x, w), f64(x), wv, dt)
    dy = make_x(T, out, T * 3 + out, dt, 0.5)
    check_product(mx4.linear_grad(dy, w), f64(dy), wv.T, dt)
    mx4.status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 300, 700])
def test_captured_forward_and_backward(dtype, T):
    dt = DTYPES[dtype]
    w, wv = operand(520, 320, "MXFP4", T)
    x, dy = make_x(T, 320, T, dt, 0.5), make_x(T, 520, T + 1, dt, 0.5)

    def step():
        leaf = x.detach().requires_grad_(True)
        y = mx4.linear(leaf, w)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y, dx = step()
    for rep in range(2):
        x.copy_(make_x(T, 320, 40 + rep, dt, 0.5))
        dy.copy_(make_x(T, 520, 50 + rep, dt, 0.5))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_product(y, f64(x), wv, dt)
        check_product(dx, f64(dy), wv.T, dt)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_variants_in_a_graph_on_another_stream(dtype):
    dt = DTYPES[dtype]
    w, wv = operand(8200, 2048, "MXFP4", 3)
    xs = [make_x(T, 2048, T, dt, 0.5) for T in (16, 130, 600)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            mx4.linear_grad(mx4.linear(x, w), w)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ys = [mx4.linear(x, w) for x in xs]
            zs = [mx4.linear_grad(y, w) for y in ys]
    side.synchronize()
    for rep in range(2):
        for x in xs:
            x.copy_(make_x(x.shape[0], 2048, 70 + rep, dt, 0.5))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
            g.replay()
        side.synchronize()
        for x, y, z in zip(xs, ys, zs):
            check_product(y, f64(x), wv, dt)
            check_product(z, f64(y), wv.T, dt)


def test_gradient_from_a_thread_without_a_context():
    """The first CUDA call of a thread that has made no context current is a product's launch."""
    import threading
    w, wv = operand(600, 256, "MXFP4", 4)
    x = make_x(600, 256, 1, torch.bfloat16)
    out = []
    torch.cuda.synchronize()
    t = threading.Thread(target=lambda: out.extend([mx4.linear(x[:40], w), mx4.linear(x, w), mx4.matmul(w, w, torch.float32)]))
    t.start()
    t.join()
    torch.cuda.synchronize()
    check_product(out[0], f64(x[:40]), wv, torch.bfloat16)
    check_product(out[1], f64(x), wv, torch.bfloat16)
    check_product(out[2], wv, wv, torch.float32)


@pytest.mark.parametrize("T", [40, 600])
def test_undefined_scales_of_padding_rows(T):
    """The scale bytes of rows past the last may hold anything: they reach no result."""
    w, wv = operand(130, 200, "NVFP4", 5)
    s = w.scales.clone()
    rows = torch.arange(256, device="cuda").view(2, 4, 32).permute(0, 2, 1).view(2, 1, 32, 4, 1).expand_as(s)
    s = torch.where(rows >= 130, torch.full_like(s, 0x7F), s).contiguous()
    w2 = mx4.Mx4Tensor(w.codes, s, "NVFP4", 130, 200, w.tensor_scale)
    x, dy = make_x(T, 200, 1, torch.bfloat16), make_x(T, 130, 2, torch.bfloat16)
    check_product(mx4.linear(x, w2), f64(x), wv, torch.bfloat16)
    check_product(mx4.linear_grad(dy, w2), f64(dy), wv.T, torch.bfloat16)
    check_product(mx4.matmul(mx4.Mx4Tensor(w.codes, s, "NVFP4", 130, 200, w.tensor_scale), w2, torch.float32), wv, wv, torch.float32)
    assert np.array_equal(f64(mx4.dequantize(w2)), wv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 150])
def test_linear_strides_and_shapes(dtype, T):
    dt = DTYPES[dtype]
    w, wv = operand(130, 200, "MXFP4", 1)
    base = make_x(2 * T + 2, 512, 5, dt, 0.5)
    for x in (base[:T, :200], base[::2, 8:208][:T], base[1:T + 1, 3:203], base.t()[:200, :T].t(), base[:1, :200].expand(T, 200)):
        check_product(mx4.linear(x, w), f64(x), wv, dt)
    x3 = base[:T * 2].view(2, T, 512)[..., :200]
    y3 = mx4.linear(x3, w)
    assert y3.shape == (2, T, 130)
    check_product(y3.reshape(-1, 130), f64(x3).reshape(-1, 200), wv, dt)
    check_product(mx4.linear(base[0, :200], w).view(1, -1), f64(base[:1, :200]), wv, dt)


def test_empty_products():
    w, _ = operand(10, 64, "NVFP4", 1)
    none = mx4.quantize(torch.zeros((0, 64), device="cuda"), "NVFP4")
    assert mx4.linear(torch.zeros((0, 64), device="cuda"), w).shape == (0, 10)
    assert mx4.linear(torch.zeros((2, 0, 64), device="cuda"), w).shape == (2, 0, 10)
    assert mx4.matmul(none, w).shape == (0, 10) and mx4.matmul(w, none).shape == (10, 0)
    assert mx4.linear(torch.zeros((3, 64), device="cuda"), none).shape == (3, 0)
    g = mx4.linear_grad(torch.zeros((3, 0), device="cuda"), none)
    assert g.shape == (3, 64) and not g.any()


def test_gradient_of_broadcast_and_second_order():
    w, wv = operand(96, 160, "MXFP4", 2)
    x = make_x(5, 160, 1).requires_grad_(True)
    mx4.linear(x, w).sum().backward()                         # dy is an expanded scalar
    check_product(x.grad, np.ones((5, 96)), wv.T, torch.float32)
    v = make_x(5, 96, 3).requires_grad_(True)
    g, = torch.autograd.grad(mx4.linear(x, w), x, v, create_graph=True)
    u = make_x(5, 160, 4)
    gg, = torch.autograd.grad(g, v, u)                        # d <u, v w> / dv = u w^T
    check_product(gg, f64(u), wv, torch.float32)
    row = make_x(1, 160, 6).requires_grad_(True)              # one row shared by many
    mx4.linear(row.expand(7, 160), w).backward(v[:1].detach().expand(7, 96))
    want = 7 * (f64(v[:1]) @ wv)
    assert np.abs(f64(row.grad) - want).max() <= 8 * chain(96) * np.abs(f64(v[:1])).dot(np.abs(wv)).max() * 7


@pytest.mark.parametrize("T", [4, 200])
def test_gradient_against_differences(T):
    """linear is linear, so a central difference in float32 equals the directional derivative up to the
    accumulation's rounding of the two values."""
    w, wv = operand(72, 96, "NVFP4", 3)
    x, d, c = make_x(T, 96, 1), make_x(T, 96, 2), make_x(T, 72, 3)
    xg = x.clone().requires_grad_(True)
    (mx4.linear(xg, w) * c).sum().backward()
    got = float((xg.grad.double() * d.double()).sum())
    diff = float(((mx4.linear(x + d, w).double() - mx4.linear(x - d, w).double()) * c.double()).sum()) / 2
    mag = float((np.abs(f64(c)) * ((np.abs(f64(x)) + np.abs(f64(d))) @ np.abs(wv).T)).sum())
    assert abs(got - diff) <= (2 * chain(96) + 4 * 2.0 ** -24) * mag


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T", [1, 40, 300])
def test_nan_stays_where_it_belongs(fmt, T):
    """A NaN block of the weights reaches its output row only; a NaN of x its own row only."""
    w, wv = operand(200, 512, fmt, 4)
    W = torch.from_numpy(wv).float().cuda()
    W[77, 300] = float("nan")
    w = mx4.quantize(W, fmt, tensor_scale=w.tensor_scale)
    x = make_x(T, 512, 1, torch.bfloat16)
    nan = torch.isnan(mx4.linear(x, w))
    assert nan[:, 77].all() and int(nan.sum()) == T
    nan = torch.isnan(mx4.matmul(mx4.quantize(x, fmt), w))
    assert nan[:, 77].all() and int(nan.sum()) == T
    b = mo.BLOCK[fmt]
    nan = torch.isnan(mx4.linear_grad(make_x(T, 200, 2, torch.bfloat16), w))
    assert nan[:, 300 // b * b:300 // b * b + b].all() and int(nan.sum()) == T * b
    x[T - 1, 3] = float("nan")
    w, _ = operand(200, 512, fmt, 4)
    nan = torch.isnan(mx4.linear(x, w))
    assert nan[T - 1].all() and int(nan.sum()) == 200


@pytest.mark.parametrize("T", [2, 200])
def test_infinities_in_x(T):
    w, wv = operand(64, 256, "MXFP4", 5)
    for dt in DTYPES.values():
        x = make_x(T, 256, 1, dt)
        x[0, 7] = float("inf")
        y = f64(mx4.linear(x, w))
        col = wv[:, 7]
        assert (y[0][col > 0] == np.inf).all() and (y[0][col < 0] == -np.inf).all() and np.isnan(y[0][col == 0]).all()
        assert np.isfinite(y[1:]).all()


@pytest.mark.parametrize("T", [1, 9, 200])
def test_extreme_scales(T):
    """Block scales over the whole range of e8m0, and activations far from 1."""
    rng = np.random.default_rng(6)
    for top, xs in ((100, 2.0 ** -90), (-60, 2.0 ** 40), (3, 1.0)):
        byte = np.clip(rng.integers(-8, 9, (64, 8)) + 127 + top, 1, 253)
        codes = rng.integers(0, 16, (64, 8, 32))
        c, s = mo.pack(codes, byte, "MXFP4", 256)
        w = mx4.Mx4Tensor(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), "MXFP4", 64, 256)
        wv = mo.values(codes, byte, "MXFP4")
        x = (make_x(T, 256, 2).double() * xs).float()
        for dt in (torch.bfloat16, torch.float32):
            check_product(mx4.linear(x.to(dt), w), f64(x.to(dt)), wv, dt)
            check_product(mx4.linear_grad((make_x(T, 64, 3).double() * xs).to(dt), w),
                          f64((make_x(T, 64, 3).double() * xs).to(dt)), wv.T, dt)


def test_small_values_beside_large_ones():
    """A large activation does not cost the small ones of its row their bits."""
    w, wv = operand(64, 256, "MXFP4", 7)
    for T in (1, 200):
        for dt in DTYPES.values():
            x = make_x(T, 256, 3, dt) * 2.0 ** -6
            x[:, 100] = 1000.0
            wz = wv.copy()
            check_product(mx4.linear(x, w), f64(x), wz, dt)


# ------------------------------------------------------------------------------- streams, graphs, devices

def test_other_stream_and_reuse():
    w, wv = operand(300, 512, "MXFP4", 1)
    s = torch.cuda.Stream()
    xs = [make_x(T, 512, T, torch.float16) for T in (1, 20, 200)]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        ys = [mx4.linear(x, w) for x in xs for _ in range(3)]
        zs = [mx4.matmul(mx4.quantize(x, "MXFP4"), w, torch.float32) for x in xs]
    s.synchronize()
    for i, x in enumerate(xs):
        for k in range(3):
            check_product(ys[3 * i + k], f64(x), wv, torch.float16)
        codes, byte = mo.quantize(f64(x), "MXFP4")
        check_product(zs[i], mo.values(codes, byte, "MXFP4", 1.0, 512), wv, torch.float32)


def test_two_graphs_and_replay():
    """Two captured graphs of the same operands, replayed in turn and on two streams at once."""
    w, wv = operand(500, 1024, "NVFP4", 2)
    xs = [make_x(T, 1024, T, torch.float32, 0.5) for T in (1, 96)]
    mx4.linear(xs[0], w), mx4.linear(xs[1], w), mx4.linear_grad(make_x(96, 500, 1), w)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = mx4.linear(x, w)
            z = mx4.linear_grad(y, w)
            q = mx4.matmul(mx4.quantize(x, "NVFP4", tensor_scale=2.0 ** -5), w, torch.float32)
        graphs.append(g)
        outs.append((y, z, q))
    for rep in range(3):
        for i, x in enumerate(xs):
            x.copy_(make_x(x.shape[0], 1024, 50 + rep, torch.float32, 0.5))
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for x, (y, z, q) in zip(xs, outs):
            check_product(y, f64(x), wv, torch.float32)
            check_product(z, f64(y), wv.T, torch.float32)
            codes, byte = mo.quantize(f64(x), "NVFP4", 2.0 ** -5)
            check_product(q, mo.values(codes, byte, "NVFP4", 2.0 ** -5, 1024), wv, torch.float32)
    mx4.status()


def test_repeated_calls_give_the_same_bits():
    w, _ = operand(700, 2048, "MXFP4", 8)
    for T in (1, 30, 400):
        x = make_x(T, 2048, T)
        a = mx4.quantize(x, "MXFP4")
        y, z, q = mx4.linear(x, w), mx4.linear_grad(make_x(T, 700, 1), w), mx4.matmul(a, w, torch.float32)
        for _ in range(3):
            assert torch.equal(y, mx4.linear(x, w))
            assert torch.equal(z, mx4.linear_grad(make_x(T, 700, 1), w))
            assert torch.equal(q, mx4.matmul(a, w, torch.float32))


def test_gpu_refusals():
    w, _ = operand(10, 64, "NVFP4", 1)
    x = torch.zeros((2, 64), device="cuda")
    with pytest.raises(ValueError):
        mx4.matmul(mx4.quantize(x, "MXFP4"), w)
    with pytest.raises(ValueError):
        mx4.linear(x.cpu(), w)
    with pytest.raises(ValueError):
        mx4.quantize(x.int(), "MXFP4")
    with pytest.raises(ValueError):
        mx4.quantize(x, "MXFP4", torch.ones(63, device="cuda"))
    with pytest.raises(ValueError):
        mx4.quantize(x, "MXFP4", torch.ones(64))
    with pytest.raises(nat.CudaPathError):
        mx4.quantize(x, "NVFP4", tensor_scale=3.0)


# ------------------------------------------------------------------------------- together

def test_encoded_model_trains_its_input_and_yields_hessians():
    """Encode a model's linears with importance weights, collect the Hessians of the encoded model's
    activations, encode the next layer with them, and take a gradient through all of it."""
    import gguf  # noqa: F401
    from transformers import Qwen3Config, Qwen3ForCausalLM
    from perm_b200 import hessians
    torch.manual_seed(0)
    cfg = Qwen3Config(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, vocab_size=128, tie_word_embeddings=False)
    model = Qwen3ForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    ids = [torch.randint(0, 128, (1, 48)) for _ in range(2)]
    ne0 = {}
    for i in range(2):
        for k in ("attn_q", "attn_k", "attn_v", "ffn_gate", "ffn_up"):
            ne0[f"blk.{i}.{k}.weight"] = 256
        ne0[f"blk.{i}.attn_output.weight"] = 256
        ne0[f"blk.{i}.ffn_down.weight"] = 512
    H, _ = hessians.collect_hessians(model, ids, ne0, "qwen3", 2, log=lambda *_: None)
    mlp = model.model.layers[0].mlp
    for name, key in (("gate_proj", "ffn_gate"), ("up_proj", "ffn_up"), ("down_proj", "ffn_down")):
        lin = getattr(mlp, name)
        qw = torch.from_numpy(np.ascontiguousarray(np.diag(H[f"blk.0.{key}.weight"]["H"]))).cuda()
        setattr(mlp, name, mx4.Linear.from_linear(lin, "MXFP4" if name != "down_proj" else "NVFP4", qw))
    H2, _ = hessians.collect_hessians(model, ids, ne0, "qwen3", 2, log=lambda *_: None)
    assert set(H2) == set(H)
    assert np.array_equal(H2["blk.0.ffn_up.weight"]["H"], H["blk.0.ffn_up.weight"]["H"])       # the same input
    assert not np.array_equal(H2["blk.0.ffn_down.weight"]["H"], H["blk.0.ffn_down.weight"]["H"])   # encoded upstream
    # the gradient of the encoded mlp's input against the same mlp with dequantised weights in float64
    x = make_x(20, 256, 1, torch.float32, 0.3).requires_grad_(True)
    m32 = mlp.float()
    m32(x).square().sum().backward()
    ref = [f64(mx4.dequantize(getattr(mlp, k).weight4)) for k in ("gate_proj", "up_proj", "down_proj")]
    xd = x.detach().double().cpu().requires_grad_(True)
    g, u, d = (torch.from_numpy(r) for r in ref)
    ((torch.nn.functional.silu(xd @ g.T) * (xd @ u.T)) @ d.T).square().sum().backward()
    rel = (x.grad.double().cpu() - xd.grad).norm() / xd.grad.norm()
    assert rel <= 2.0 ** -16, rel     # some ten float32 steps of at most chain(512) each
    mx4.status()
