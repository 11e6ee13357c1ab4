"""Microscaled 4-bit operators where they can go wrong: alignment, ranges, padding, derivatives other than the
plain gradient, saved state.  Values against the definition in float64 (tests/mx4_oracle.py)."""
import numpy as np
import pytest
import torch

import mx4_oracle as mo
from perm_b200 import _native as nat
from perm_b200 import mx4
from test_mx4_gpu import DTYPES, FMTS, HALF, chain, check_operand, check_product, f64, make_x, operand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 8, 16])
def test_few_tokens_at_every_alignment_of_x(fmt, dtype, T):
    """x starts anywhere its type may, and its rows end inside a group of 256 columns: the asynchronous copies
    take 16-byte sources only."""
    dt = DTYPES[dtype]
    for n in (200, 248, 520):
        w, wv = operand(130, n, fmt, n)
        base = make_x(T + 1, n + 9, n, dt, 0.5).reshape(-1)
        for at in range(1, 9):
            x = base[at:at + T * n].view(T, n)
            check_product(mx4.linear(x, w), f64(x), wv, dt)
            x = base[at:at + T * (n + 3)].view(T, n + 3)[:, :n]
            check_product(mx4.linear(x, w), f64(x), wv, dt)
    mx4.status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,n", [(1, 40), (5, 256), (33, 300), (127, 64), (130, 1000)])
def test_padding_is_written_and_nothing_behind_it(fmt, rows, n):
    """Every byte of an operand is defined, whatever its memory held: codes and scales past n and the scales of
    rows past the last are zero.  Bytes behind the arrays stay."""
    L, s = nat.lib(), nat.stream_ptr(torch)
    nc, ns = L.cp_mx4_codes_bytes(rows, n), L.cp_mx4_scales_bytes(nat.MX4_ID[fmt], rows, n)

    def run(call):
        codes = torch.full((nc + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        scales = torch.full((ns + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        nat.check(call(codes.data_ptr(), scales.data_ptr()))
        assert (codes[nc:] == 0xA5).all() and (scales[ns:] == 0xA5).all()
        return codes[:nc].view(rows, -1).cpu().numpy(), scales[:ns].view(-1, nc // rows // (2 * mo.BLOCK[fmt]), 32, 4, 4).cpu().numpy()

    for dt, kind in ((torch.bfloat16, nat.CP_MX4_BF16), (torch.float32, nat.CP_MX4_F32)):
        x = make_x(rows, n, rows + n, dt)
        for qw in (None, torch.linspace(0.5, 2.0, n, device="cuda")):
            codes, byte = mo.quantize(f64(x), fmt, 1.0, None if qw is None else f64(qw))
            want = mo.pack(np.where(codes == 8, 0, codes), byte, fmt, n)
            got = run(lambda c, p: L.cp_mx4_quantize(nat.MX4_ID[fmt], kind, x.data_ptr(), rows, n, n,
                                                     None if qw is None else qw.data_ptr(), 1.0, c, p, s))
            assert np.array_equal(got[1], want[1])
            gc, _ = mo.unpack(got[0], got[1], fmt, rows, n)
            wc, _ = mo.unpack(want[0], want[1], fmt, rows, n)
            assert np.array_equal(np.where(gc == 8, 0, gc), wc)
    if fmt == "MXFP4" and n % 32 == 0:
        x = f64(make_x(rows, n, 1))
        codes, byte = mo.quantize(x, fmt)
        raw = torch.from_numpy(mo.container(codes, byte)).cuda()
        got = run(lambda c, p: L.cp_mx4_from_gguf(raw.data_ptr(), rows, n, c, p, s))
        want = mo.pack(codes, byte, fmt, n)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2, 40])
def test_forward_mode(dtype, T):
    import torch.autograd.forward_ad as fw
    dt = DTYPES[dtype]
    w, wv = operand(96, 200, "MXFP4", 3)
    x, t = make_x(T, 200, 1, dt, 0.5), make_x(T, 200, 2, dt, 0.5)
    dy, u = make_x(T, 96, 3, dt, 0.5), make_x(T, 96, 4, dt, 0.5)
    with fw.dual_level():
        y = fw.unpack_dual(mx4.linear(fw.make_dual(x, t), w))
        check_product(y.primal, f64(x), wv, dt)
        check_product(y.tangent, f64(t), wv, dt)
        leaf = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(mx4.linear(leaf, w), leaf, fw.make_dual(dy, u))
        g = fw.unpack_dual(g)
        check_product(g.primal, f64(dy), wv.T, dt)
        check_product(g.tangent, f64(u), wv.T, dt)
    x3 = x.view(1, T, 200)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda z: mx4.linear(z, w))(x3)


@pytest.mark.parametrize("n", [32, 96, 4096])
def test_container_rows_sliced_on_the_device(n):
    from perm_b200 import kquant as kq
    x = make_x(9, n, n)
    raw = kq.QUANTIZE["MXFP4"](x)
    want = kq.DEQUANTIZE["MXFP4"](raw, n)
    for r0 in range(9):
        assert torch.equal(kq.DEQUANTIZE["MXFP4"](raw[r0:], n), want[r0:])
        assert torch.equal(mx4.dequantize(mx4.from_gguf(raw[r0:], n)), want[r0:])


def test_collected_hessians_ask_for_the_products_status(monkeypatch):
    """A product whose wait ran out is incomplete, and so is what later layers saw: collection ends with the error."""
    from perm_b200 import hessians

    class Mlp(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.up_proj, self.down_proj = torch.nn.Linear(64, 96), torch.nn.Linear(96, 64)

        def forward(self, x):
            return self.down_proj(self.up_proj(x))

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.model = torch.nn.Module()
            self.model.embed_tokens = torch.nn.Embedding(16, 64)
            self.model.layers = torch.nn.ModuleList([torch.nn.Module()])
            self.model.layers[0].mlp = Mlp()

        def forward(self, ids):
            return self.model.layers[0].mlp(self.model.embed_tokens(ids))

    net = Net().cuda().to(torch.bfloat16)
    mlp = net.model.layers[0].mlp
    mlp.up_proj = mx4.Linear.from_linear(mlp.up_proj)
    ne0 = {"blk.0.ffn_up.weight": 64, "blk.0.ffn_down.weight": 96}
    collect = lambda: hessians.collect_hessians(net, [torch.arange(16)], ne0, "qwen3", 1, log=lambda *_: None)  # noqa: E731
    asked = []
    real = mx4.status
    monkeypatch.setattr(mx4, "status", lambda dev=None: asked.append(dev) or real(dev))
    H, _ = collect()
    assert set(H) == set(ne0) and asked == [torch.device("cuda", 0)]

    def ran_out(dev=None):
        raise nat.CudaPathError("a bounded wait ran out")
    monkeypatch.setattr(mx4, "status", ran_out)
    with pytest.raises(nat.CudaPathError):
        collect()


@pytest.mark.parametrize("g", [2.0 ** -100, 2.0 ** -30, 1.0, 4.0, 2.0 ** 40, 2.0 ** 99])
def test_weighted_blocks_far_from_the_tensor_scale(g):
    """Blocks of zeros, far below and far above what the tensor scale's e4m3 scales reach: codes as without weights."""
    rng = np.random.default_rng(7)
    x = np.zeros((12, 64))
    for r, e in enumerate((0, 20, -8, -12, -40, -120, 60, 90, 104, 127)):
        x[r] = rng.standard_normal(64) * np.exp2(np.clip(np.log2(g) + e, -140, 126))
    x[10, :16] = 1.5 * g
    xt = torch.from_numpy(x).float().cuda()
    assert torch.isfinite(xt).all()
    check_operand(mx4.quantize(xt, "NVFP4", tensor_scale=g), xt, g)
    for qw in (torch.ones(64, device="cuda"), torch.exp(torch.linspace(-3, 3, 64, device="cuda"))):
        check_operand(mx4.quantize(xt, "NVFP4", qw, g), xt, g, qw)


# ------------------------------------------------------------------------------- activations at their own precision

def picker(out, n, fmt, code, byte):
    """Weights of one code in every row, each in another column, and zero elsewhere; the columns."""
    b = mo.BLOCK[fmt]
    nb = -(-n // b)
    codes, col = np.zeros((out, nb, b), np.int64), np.random.default_rng(out + n).permutation(n)[np.arange(out) % n]
    codes[np.arange(out), col // b, col % b] = code
    c, s = mo.pack(codes, np.full((out, nb), byte), fmt, n)
    return mx4.Mx4Tensor(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), fmt, out, n), torch.from_numpy(col).cuda()


def wide(T, n, dtype, seed, span):
    """Values of random significands with exponents spread over 2^-span .. 2^span."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-span, span + 1, (T, n), generator=g)
    return (torch.randn(T, n, generator=g).double() * torch.exp2(e.double())).to(dtype).cuda()


ONE = {"MXFP4": 127, "NVFP4": 0x38}     # the scale byte of 1


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,out,n", [(1, 300, 520), (2, 300, 520), (8, 300, 520), (16, 300, 520), (17, 300, 520), (130, 300, 520),
                                     (600, 300, 520), (16, 8200, 2048), (3, 15000, 4096), (12, 130, 12000)])
def test_every_value_of_x_counts(fmt, dtype, T, out, n):
    """Each result is one value of x times one: what a row's large values take from its small ones, or a part of
    a value that is left out, shows at once.  float32 rows of a narrow range with up to 16 tokens may be off
    by a unit in the last place, 2^-23; all else is exact."""
    dt = DTYPES[dtype]
    w, col = picker(out, n, fmt, 2, ONE[fmt])
    wide_span, narrow_span = (8, 3) if dt == torch.float16 else (55, 5)
    x, z = wide(T, n, dt, T, wide_span), wide(T, n, dt, T + 1, narrow_span)
    z = torch.where(z.abs() < 2.0 ** -7, torch.ones_like(z), z)      # narrow: 2^-7 to about 2^8
    assert torch.equal(mx4.linear(x, w), x[:, col])
    for scale in (1.0, 2.0 ** -60, 2.0 ** -90, 2.0 ** -110, 2.0 ** 50, 2.0 ** 90) if dt != torch.float16 else (1.0,):
        if dt == torch.float32 and T > 16 and scale < 2.0 ** -100:
            continue                                    # of three parts, the last below 2^-133
        y, want = mx4.linear(z * scale, w), z[:, col] * scale
        if dt == torch.float32 and T <= 16 and scale < 2.0 ** 60:
            assert ((y.double() - want.double()).abs() <= 2.0 ** -23 * want.double().abs()).all()
        else:
            assert torch.equal(y, want)
    if T > 1:                                                          # one wide row among narrow ones
        m = z.clone()
        m[T - 1] = x[T - 1]
        assert torch.equal(mx4.linear(m, w)[T - 1], x[T - 1, col])
    if out <= n:
        dy = wide(T, out, dt, T + 2, wide_span)
        want = torch.zeros((T, n), dtype=dt, device="cuda").index_copy(1, col, dy)
        assert torch.equal(mx4.linear_grad(dy, w), want)
    mx4.status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 16, 17, 600])
def test_products_near_the_end_of_float32(fmt, dtype, T):
    """x at float32's end times a small weight is finite, for any number of tokens."""
    dt = DTYPES[dtype]
    w, col = picker(64, 256, fmt, 7, 127 - 6 if fmt == "MXFP4" else 8)           # 6 x 2^-6
    x = torch.full((T, 256), 3e38, device="cuda").to(dt)
    want = f64(x[:, :1]) * 6 * 2.0 ** -6
    for v in (x, -x, x * 2.0 ** -245):
        got = f64(mx4.linear(v, w))
        want = f64(v[:, :1]) * 6 * 2.0 ** -6
        # one rounding to the type; float32 values of one significand are as in the test above
        assert (np.abs(got - want) <= (HALF[dt] + 2.0 ** -22) * np.abs(want)).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,out,n", [(1, 130, 600), (5, 130, 600), (16, 130, 600), (16, 8200, 2048)])
def test_wide_rows_against_dense_weights(fmt, dtype, T, out, n):
    """Rows that their units do not hold, with every weight set; a NaN and infinities among them."""
    dt = DTYPES[dtype]
    w, wv = operand(out, n, fmt, 11)
    x = wide(T, n, dt, T, 40)
    check_product(mx4.linear(x, w), f64(x), wv, dt)
    x[0, 5] = float("inf")
    y = f64(mx4.linear(x, w))
    c = wv[:, 5]
    assert (y[0][c > 0] == np.inf).all() and (y[0][c < 0] == -np.inf).all() and np.isnan(y[0][c == 0]).all()
    check_product(mx4.linear(x, w)[1:], f64(x[1:]), wv, dt)
    x[T - 1, 7] = float("nan")
    assert torch.isnan(mx4.linear(x, w)[T - 1]).all()


@pytest.mark.parametrize("T", [1, 16, 200])
def test_small_values_beside_a_large_one_that_has_no_weight(T):
    """The large value's column is zero in every row of the weights, so the tolerance knows the small ones only."""
    for fmt in FMTS:
        codes, byte = mo.quantize(0.05 * np.random.default_rng(7).standard_normal((64, 256)), fmt, 2.0 ** -12 if fmt == "NVFP4" else 1.0)
        b = mo.BLOCK[fmt]
        codes[:, 100 // b, 100 % b] = 0
        c, s = mo.pack(codes, byte, fmt, 256)
        w = mx4.Mx4Tensor(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), fmt, 64, 256)
        for dt in DTYPES.values():
            for big in (1e3, 6e4) if dt == torch.float16 else (1e3, 1e13, 1e30):
                x = make_x(T, 256, 3, dt) * 2.0 ** -6
                x[:, 100] = big
                check_product(mx4.linear(x, w), f64(x), mo.values(codes, byte, fmt, 1.0, 256), dt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T", [1, 16, 40, 300, 600])
def test_float32_sums_keep_their_size(fmt, T):
    """Sums of positive products: truncation, which the tensor core's accumulation does, does not cancel here.  A chain
    ends with at most 16 MMAs of x's largest part, each of which takes half a unit (2^-24) of a sum that is on
    average half grown; chains are added with rounding.  16 2^-25 = 2^-21."""
    rng = np.random.default_rng(T)
    b, n, out = mo.BLOCK[fmt], 1024, 256
    codes = rng.integers(1, 8, (out, n // b, b))
    byte = rng.integers(125, 130, (out, n // b)) if fmt == "MXFP4" else rng.integers(0x30, 0x48, (out, n // b))
    c, s = mo.pack(codes, byte, fmt, n)
    w = mx4.Mx4Tensor(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), fmt, out, n)
    wv = mo.values(codes, byte, fmt)
    x = torch.from_numpy(0.5 + rng.random((T, n))).float().cuda()
    dy = torch.from_numpy(0.5 + rng.random((T, out))).float().cuda()
    for got, want in ((mx4.linear(x, w), f64(x) @ wv.T), (mx4.linear_grad(dy, w), f64(dy) @ wv)):
        assert abs((f64(got) / want - 1).mean()) <= 2.0 ** -21


# ------------------------------------------------------------------------------- waits that run out

STALLS = [("matmul", "MXFP4", "bf16", 5, 300, 2048, 0), ("matmul", "NVFP4", "f32", 100, 300, 2048, 0),
          ("matmul", "NVFP4", "bf16", 600, 4000, 4096, 11),
          ("linear", "MXFP4", "bf16", 1, 300, 2048, 0), ("linear", "NVFP4", "f32", 16, 8200, 2048, 1), ("linear", "MXFP4", "f16", 9, 130, 512, 0),
          ("linear", "MXFP4", "bf16", 40, 520, 2048, 0), ("linear", "NVFP4", "f32", 40, 520, 2048, 1),
          ("linear", "MXFP4", "bf16", 512, 14340, 1024, 7), ("linear", "NVFP4", "f16", 512, 14340, 1024, 0),
          ("linear", "MXFP4", "bf16", 600, 1030, 2048, 9), ("linear", "NVFP4", "f32", 600, 1030, 2048, 0),
          ("grad", "MXFP4", "bf16", 3, 520, 2048, 0), ("grad", "NVFP4", "bf16", 200, 2048, 520, 1), ("grad", "MXFP4", "bf16", 600, 1030, 2048, 8)]


@pytest.mark.parametrize("call,fmt,dtype,T,out,n,skip", STALLS)
def test_a_wait_that_runs_out_is_reported(call, fmt, dtype, T, out, n, skip):
    """The failure paths of the products' bounded waits, made on the host: the next call leaves out one step of its
    loads and every wait gives up after 5 ms.  The kernel stops, status() says so once, and the next call is right."""
    dt = DTYPES[dtype]
    w, wv = operand(out, n, fmt, out + n)
    if call == "matmul":
        a, av = operand(T, n, fmt, T + n, 2.0 ** -10 if fmt == "NVFP4" else 1.0)
        run, x, m = (lambda: mx4.matmul(a, w, dt)), av, wv
    else:
        xt = make_x(T, n if call == "linear" else out, T + out, dt, 0.5)
        run, x, m = (lambda: (mx4.linear if call == "linear" else mx4.linear_grad)(xt, w)), f64(xt), wv if call == "linear" else wv.T
    check_product(run(), x, m, dt)
    mx4.status()
    assert nat.lib().cp_mx4_inject_stall(skip, 5_000_000) == nat.CP_OK
    run()
    with pytest.raises(nat.CudaPathError, match="ran out"):
        mx4.status()
    check_product(run(), x, m, dt)
    mx4.status()
