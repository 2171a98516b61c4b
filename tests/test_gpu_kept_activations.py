"""GPU: activations kept in 8 bits and the weight gradient that reads them, against plain 64-bit forms (tests/token_oracle.py)."""
import math

import pytest
import torch
from torch.autograd import forward_ad as fwAD

import token_oracle as O
from torchrl_amd.objectives.value import CheckpointedLinear, QuantizedActivation, checkpointed_linear, functional as F, quantize_activation

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(N, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, D, generator=g) * torch.exp(torch.randn(N, 1, generator=g) * 3) * (1 + 30 * (torch.rand(D, generator=g) < 0.02))
    return x.clamp(-6e4, 6e4).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(1, 1), (3, 7), (2, 31), (2, 32), (5, 33), (1, 64), (37, 100), (130, 257), (3, 2080)])
def test_format(dtype, N, D):
    x = inputs(N, D, dtype, seed=N * D)
    codes, exps, values = O.kept(x)
    q = quantize_activation(x.cuda())
    assert F.last_kernel() == "act_quantize" and q.shape == x.shape and q.dtype == dtype
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.exponents.cpu(), exps)
    for dt in {dtype, torch.bfloat16, torch.float32}:
        back = q.dequantize(dt)
        assert back.dtype == dt and torch.equal(back.cpu().double(), values)  # exact
    # within half a step, below the clamp
    step = torch.ldexp(torch.ones((), dtype=torch.float64), exps.int() - 127).repeat_interleave(32, -1)[:, :D]
    off = (x.double() - values).abs()
    assert (off <= torch.where(x.double().abs() <= 127.5 * step, 0.5, 1.0) * step).all()


def test_edges_of_the_format():
    tiny = torch.finfo(torch.float32).tiny
    x = torch.zeros(9, 64)
    x[0, :3] = torch.tensor([127.0, 127.5, -127.99])  # clamped at the top
    x[1, :4] = torch.tensor([64.0, 0.5, 1.5, 2.5])  # ties to even
    x[2, 0] = math.nan
    x[3, 40] = math.inf
    x[4, 33] = -math.inf
    x[5, :2] = torch.tensor([tiny, tiny / 4])
    x[6, :2] = torch.tensor([2.0 ** -149, 0.0])
    x[7, :2] = torch.tensor([torch.finfo(torch.float32).max, 1.0])
    x[8, 1] = -0.0
    codes, exps, values = O.kept(x)
    q = quantize_activation(x.cuda())
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.exponents.cpu(), exps)
    got = q.dequantize().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(values)) and torch.equal(got.nan_to_num(0), values.nan_to_num(0))
    h = torch.tensor([[65504.0, 65280.0, 6.0e-8, -65504.0]], dtype=torch.float16)  # the codes' clamp keeps the largest finite
    assert torch.isfinite(quantize_activation(h.cuda()).dequantize()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_batch_dims(dtype):
    x = inputs(24, 80, dtype)
    wide = torch.full((24, 100), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:83] = x.cuda()
    want = quantize_activation(x.cuda())
    got = quantize_activation(wide[:, 3:83])
    assert torch.equal(got.codes, want.codes) and torch.equal(got.exponents, want.exponents)
    got = quantize_activation(x.cuda().view(2, 3, 4, 80).transpose(0, 1))
    assert torch.equal(got.dequantize(), want.dequantize().view(2, 3, 4, 80).transpose(0, 1))
    assert quantize_activation(torch.zeros(0, 5, device="cuda")).dequantize().shape == (0, 5)


def bound(dy, x):
    """Sums of N exact products in 32 bits: N roundings, each of at most half a step of the sum of magnitudes."""
    return (dy.shape[0] + 1) * O.U * (dy.abs().T @ x.abs())


def weight_grad(x, dy, bias):
    N, D = x.shape
    w = torch.zeros(dy.shape[1], D, dtype=x.dtype, device="cuda", requires_grad=True)
    b = torch.zeros(dy.shape[1], dtype=x.dtype, device="cuda", requires_grad=True) if bias else None
    y = checkpointed_linear(x.cuda(), w, b)
    return torch.autograd.grad(y, (w, b) if bias else (w,), dy.cuda())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,O_", [(1, 1, 1), (3, 5, 2), (64, 64, 64), (65, 33, 31), (200, 129, 130), (130, 257, 65), (1000, 40, 1), (700, 300, 3),
                                    (257, 32, 300), (31, 500, 17), (2100, 96, 33)])
def test_weight_gradient(dtype, N, D, O_):
    x = inputs(N, D, dtype, seed=N + D).clamp(-100, 100)
    dy = torch.randn(N, O_, generator=torch.Generator().manual_seed(O_)).to(dtype)
    dw, db = weight_grad(x, dy, True)
    kept = O.kept(x)[2]
    O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "dw")
    O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")
    (dw2,) = weight_grad(x, dy, False)
    assert torch.equal(dw2, dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradient_over_a_long_batch(dtype):
    """Many tokens and few outputs: the sum is split and joined; twice the same bits."""
    N, D, O_ = 30011, 72, 5
    x = inputs(N, D, dtype, seed=1).clamp(-100, 100)
    dy = torch.randn(N, O_, generator=torch.Generator().manual_seed(2)).to(dtype)
    dw, db = weight_grad(x, dy, True)
    xc = x.cuda()
    kept = quantize_activation(xc).dequantize().cpu().double()  # checked by test_format
    O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "dw")
    O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")
    again = weight_grad(x, dy, True)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_and_small_values_reach_the_gradient(dtype):
    x = torch.randn(70, 96, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[5, 40] = math.inf  # the block of features 32-63 of token 5
    dy = torch.randn(70, 40, generator=torch.Generator().manual_seed(4)).to(dtype)
    dw, _ = weight_grad(x, dy, True)
    assert torch.isnan(dw[:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()
    x = (torch.randn(40, 64, generator=torch.Generator().manual_seed(5)) * 2.0 ** -14).to(dtype)
    dy = (torch.randn(40, 33, generator=torch.Generator().manual_seed(6)) * 2.0 ** -10).to(dtype)
    dw, db = weight_grad(x, dy, True)
    kept = O.kept(x)[2]
    O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "small dw")
    big = torch.full((3, 40), 3e4).to(dtype)
    dw, _ = weight_grad(big, torch.full((3, 8), 2.0 ** -12).to(dtype), True)
    kept = O.kept(big)[2]
    O.assert_close(dw, torch.full((8, 3), 2.0 ** -12, dtype=torch.float64) @ kept, bound(torch.full((3, 8), 2.0 ** -12, dtype=torch.float64), kept), "large dw")


@pytest.mark.parametrize("form", ["expanded", "transposed", "row stride", "sum"])
def test_incoming_gradients_of_any_layout(form):
    N, D, O_ = 90, 70, 40
    x = inputs(N, D, torch.bfloat16, seed=9).clamp(-50, 50)
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(N, O_, generator=g).bfloat16()
    if form == "expanded":
        dy = dy[:1].expand(N, O_)
        d = dy[:1].cuda().expand(N, O_)
    elif form == "transposed":
        d = dy.t().contiguous().cuda().t()
    elif form == "row stride":
        d = torch.cat([dy, dy], 1).cuda()[:, :O_]
    else:
        dy = torch.ones(N, O_).bfloat16()
        d = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(N, O_)
    w = torch.zeros(O_, D, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    b = torch.zeros(O_, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(checkpointed_linear(x.cuda(), w, b), (w, b), d)
    kept = O.kept(x)[2]
    O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "dw")
    O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")


@pytest.mark.parametrize("need", ["x", "weight", "bias", "x weight", "weight bias", "x weight bias"])
def test_output_and_the_gradients_asked_for(need):
    x = inputs(3 * 11, 50, torch.float32, seed=2).clamp(-20, 20).view(3, 11, 50).cuda()
    layer = CheckpointedLinear(50, 20, device="cuda")
    x.requires_grad_("x" in need.split())
    layer.weight.requires_grad_("weight" in need)
    layer.bias.requires_grad_("bias" in need)
    y = layer(x)
    assert torch.equal(y, torch.nn.functional.linear(x, layer.weight, layer.bias))
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).cuda()
    y.backward(dy)
    d = dy.reshape(33, 20).cpu().double()
    xs = x.detach().reshape(33, 50).cpu()
    if "x" in need.split():
        w = layer.weight.detach().cpu().double()
        O.assert_close(x.grad, d @ w, 21 * O.U * (d.abs() @ w.abs()), "dx")
    assert (layer.weight.grad is not None) == ("weight" in need) and (layer.bias.grad is not None) == ("bias" in need)
    if "weight" in need:
        kept = O.kept(xs)[2]
        O.assert_close(layer.weight.grad, d.T @ kept, bound(d, kept), "dw")
    if "bias" in need:
        O.assert_close(layer.bias.grad, d.sum(0), 34 * O.U * d.abs().sum(0), "db")


def test_what_is_kept():
    """Half of a bfloat16 activation's bytes (and one more every 32) until the backward pass."""
    x = torch.randn(4096, 1024, device="cuda").bfloat16()
    w = torch.randn(8, 1024, device="cuda").bfloat16().requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = checkpointed_linear(x, w)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert 4096 * 1024 * (1 + 1 / 32) <= kept <= 4096 * 1024 * (1 + 1 / 32) + 4096
    with torch.no_grad():
        before = torch.cuda.memory_allocated()
        z = checkpointed_linear(x, w)
        assert torch.cuda.memory_allocated() - before <= z.numel() * 2 + 512


def test_autocast():
    x = torch.randn(20, 64, device="cuda")
    layer = CheckpointedLinear(64, 8, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    kept = O.kept(x.cpu().bfloat16())[2]
    d = torch.ones(20, 8, dtype=torch.float64)
    want = d.T @ kept
    half = torch.finfo(torch.bfloat16).eps / 2  # the gradient is rounded to bfloat16 before it reaches the float32 weight
    O.assert_close(layer.weight.grad, want, bound(d, kept) + half * (want.abs() + bound(d, kept)), "dw")


def test_captured_and_replayed():
    x = torch.randn(300, 96, device="cuda").bfloat16()
    dy = torch.randn(300, 40, device="cuda").bfloat16()
    w0, b0 = torch.randn(40, 96, device="cuda").bfloat16(), torch.randn(40, device="cuda").bfloat16()

    def step(x, w, b):
        y = checkpointed_linear(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w0.clone().requires_grad_(), b0.clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    w, b = w0.clone().requires_grad_(), b0.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, w, b)
    for k in range(4):
        x.copy_(torch.roll(x, 1, 0) * 1.5)
        graph.replay()
        eager = step(x, w0.clone().requires_grad_(), b0.clone().requires_grad_())
        torch.cuda.synchronize()
        for a, e in zip(outs, eager):
            assert torch.equal(a, e)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_the_host_module(dtype, monkeypatch):
    """The python route (a tree without lib/_trl_host.so) makes the same calls: the same bits."""
    x = inputs(140, 75, dtype, seed=3).clamp(-50, 50).cuda().view(2, 70, 75)
    w, b = (torch.randn(s, generator=torch.Generator().manual_seed(4)).to(dtype).cuda() for s in ((33, 75), (33,)))
    dy = torch.randn(2, 70, 33, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()

    def everything():
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = checkpointed_linear(*leaves)
        q = quantize_activation(x)
        only_b = b.clone().requires_grad_()
        return (y.detach(), *torch.autograd.grad(y, leaves, dy), q.codes, q.exponents, q.dequantize(), q.dequantize(torch.float32),
                *torch.autograd.grad(checkpointed_linear(x, w, only_b), only_b, dy))

    assert F.host_fast_path()
    fast = everything()
    monkeypatch.setattr(F, "_HOST", None)
    for got, want in zip(everything(), fast):
        assert got.dtype == want.dtype and torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,O_", [(1, 1), (37, 300), (5000, 7), (40000, 513)])
def test_bias_gradient_alone(dtype, N, O_):
    x = torch.zeros(N, 8, dtype=dtype, device="cuda")
    dy = torch.randn(N, O_, generator=torch.Generator().manual_seed(N)).to(dtype)
    w, b = torch.zeros(O_, 8, dtype=dtype, device="cuda"), torch.zeros(O_, dtype=dtype, device="cuda", requires_grad=True)
    (db,) = torch.autograd.grad(checkpointed_linear(x, w, b), b, dy.cuda())
    O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")


def test_no_tokens():
    w, b = torch.zeros(3, 40, device="cuda", requires_grad=True), torch.zeros(3, device="cuda", requires_grad=True)
    y = checkpointed_linear(torch.zeros(0, 40, device="cuda"), w, b)
    assert y.shape == (0, 3)
    y.sum().backward()
    assert (w.grad == 0).all() and (b.grad == 0).all()


def test_a_kept_activation_is_checked_before_it_is_read():
    x = inputs(6, 70, torch.float32, seed=9).clamp(-50, 50).cuda()
    q = quantize_activation(x)
    want = q.dequantize()
    apart = QuantizedActivation(q.codes.t().contiguous().t(), q.exponents.t().contiguous().t(), q.shape, q.dtype)  # another layout
    assert torch.equal(apart.dequantize(), want)
    for codes, exponents, shape in [(q.codes[:, :64], q.exponents, q.shape), (q.codes, q.exponents[:, :2], q.shape), (q.codes[:4], q.exponents[:4], q.shape),
                                    (q.codes, q.exponents, torch.Size((6, 97))), (q.codes.int(), q.exponents, q.shape), (q.codes, q.exponents.int(), q.shape)]:
        with pytest.raises(RuntimeError, match="do not hold"):
            QuantizedActivation(codes, exponents, shape, q.dtype).dequantize()


def test_function_transforms_and_forward_mode_are_refused():
    """Their derivatives are not there: an error, not a result without them."""
    x, w = torch.randn(5, 40, device="cuda"), torch.randn(3, 40, device="cuda")
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: checkpointed_linear(x, w).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda w: checkpointed_linear(x, w).sum())(w)
    with fwAD.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        checkpointed_linear(fwAD.make_dual(x, torch.ones_like(x)), w.clone().requires_grad_())


def test_offsets_past_32_bits():
    """Rows behind 2^31 elements and 2^32 bytes: the bits of the same rows alone."""
    N, D = 40000, 65600
    x = torch.randn(100, D, device="cuda", dtype=torch.bfloat16).repeat(N // 100, 1)
    x[-3:] *= torch.rand(3, D, device="cuda").to(x.dtype)
    q, few = quantize_activation(x), quantize_activation(x[-3:].clone())
    assert torch.equal(q.codes[-3:], few.codes) and torch.equal(q.exponents[-3:], few.exponents)
    back = q.dequantize()
    assert torch.equal(back[-3:], few.dequantize()) and torch.equal(back[:100], back[100:200])
    del back, q
    w = torch.zeros(2, D, device="cuda", dtype=x.dtype, requires_grad=True)
    dy = torch.zeros(N, 2, device="cuda", dtype=x.dtype)
    dy[-3] = torch.tensor([1.0, -2.0], device="cuda")  # one row alone: the sum has one term
    (dw,) = torch.autograd.grad(checkpointed_linear(x, w), w, dy)
    assert torch.equal(dw, dy[-3].unsqueeze(1) * few.dequantize()[0])


@pytest.mark.parametrize("route", ["host", "python"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(1, 1), (1, 700), (3, 5), (67, 64), (130, 511), (129, 513), (1000, 1000), (300, 4099), (2049, 1536), (5000, 40), (2, 65537)])
def test_one_output(route, dtype, N, D, monkeypatch):
    """A value head: one pass over x forward, one over what is kept backward."""
    if route == "python":
        assert F.host_fast_path()
        monkeypatch.setattr(F, "_HOST", None)
    g = torch.Generator().manual_seed(N + D)
    x = inputs(N, D, dtype, seed=N + D).clamp(-100, 100)
    w, b, dy = (torch.randn(s, generator=g).to(dtype) for s in ((1, D), (1,), (N, 1)))
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = checkpointed_linear(*leaves)
    if D <= 65536:
        assert F.last_kernel() == "act_head"
    # fp32 sums: a lane adds 8 products of every 512, then 7 additions over the lanes and the bias; the library's own sum above that width
    terms = (8 * -(-D // 512) if D <= 65536 else D) + 8
    X, W = x.double(), w.double()
    largest = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)  # half a step above the last number a rounding is infinite (fp16's 65520)
    want = X @ W.T + b.double()
    want = torch.where(want.abs() < largest, want, want * math.inf)
    O.assert_close(y.detach(), want, terms * O.U * (X.abs() @ W.abs().T + b.double().abs()), "y")
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    assert torch.equal(dx.cpu(), (dy.float() * w.float()).to(dtype))  # one product, one rounding
    kept = O.kept(x)[2]
    O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "dw")
    O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")
    x2, w2 = leaves[0].detach(), w.cuda().requires_grad_()
    y2 = checkpointed_linear(x2, w2, leaves[2].detach())
    (dw2,) = torch.autograd.grad(y2, w2, dy.cuda())
    assert torch.equal(y2, y) and torch.equal(dw2, dw)
    x3 = leaves[0].detach().clone().requires_grad_()
    (dx3,) = torch.autograd.grad(checkpointed_linear(x3, w.cuda()), x3, dy.cuda())  # the weight is frozen
    O.assert_close(dx3, dy.double() @ W, 0.0, "dx alone")


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_output_layouts_and_non_finite(dtype):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(4, 9, 2 * 133, generator=g).to(dtype).cuda()
    x, w = big[..., 1:134], torch.randn(133, 2, generator=g).to(dtype).cuda()[:, 0].unsqueeze(0).requires_grad_()  # rows at odd places, a strided weight
    b = torch.zeros(1, dtype=dtype, device="cuda", requires_grad=True)
    leaf = x.detach().requires_grad_()
    y = checkpointed_linear(leaf, w, b)
    dy = torch.ones(1, 1, 1, dtype=dtype, device="cuda").expand(4, 9, 1)
    got = torch.autograd.grad(y, (leaf, w, b), dy)
    plain = x.contiguous().requires_grad_()
    dense = w.detach().contiguous().requires_grad_()
    y2 = checkpointed_linear(plain, dense, b)
    assert torch.equal(y, y2) and y.shape == (4, 9, 1)
    for a, e in zip(got, torch.autograd.grad(y2, (plain, dense, b), dy.contiguous())):
        assert torch.equal(a, e)
    bad = x.clone()
    bad[0, 0, 40], bad[1, 2, 3] = math.nan, math.inf
    y3 = checkpointed_linear(bad, dense)
    assert y3[0, 0, 0].isnan() and not y3[1, 2, 0].isfinite() and torch.isfinite(y3).sum() == 34
    (dw,) = torch.autograd.grad(y3, dense, dy)
    assert dw[0, 32:64].isnan().all() and dw[0, :32].isnan().all() and torch.isfinite(dw[0, 64:]).all()  # whole blocks stand for NaN


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,O_", [(2048, 1500, 1101), (700, 1003, 1001), (1000, 300, 77), (999, 129, 257), (4096, 70, 500), (331, 513, 9), (5000, 40, 6)])
def test_weight_gradient_at_the_edges_of_tiles(dtype, N, D, O_):
    """Tiles that reach over the last output: the gradients lie in a buffer whose gaps between the rows hold NaN, which must not come in."""
    x = inputs(N, D, dtype, seed=N).clamp(-50, 50)
    wide = torch.full((N, O_ + 11), math.nan, dtype=dtype)
    wide[:, :O_] = torch.randn(N, O_, generator=torch.Generator().manual_seed(O_)).to(dtype)
    dy = wide[:, :O_]
    kept = O.kept(x)[2]
    for there in (wide.cuda()[:, :O_], dy.contiguous().cuda()):
        w, b = torch.zeros(O_, D, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(O_, dtype=dtype, device="cuda", requires_grad=True)
        dw, db = torch.autograd.grad(checkpointed_linear(x.cuda(), w, b), (w, b), there)
        O.assert_close(dw, dy.double().T @ kept, bound(dy.double(), kept), "dw")
        O.assert_close(db, dy.double().sum(0), (N + 1) * O.U * dy.double().abs().sum(0), "db")


def test_one_output_captured_and_replayed():
    N, D = 700, 520
    x, dy = inputs(N, D, torch.bfloat16, seed=21).clamp(-50, 50).cuda(), torch.randn(N, 1, dtype=torch.bfloat16, device="cuda")
    w0, b0 = torch.randn(1, D, dtype=torch.bfloat16, device="cuda"), torch.randn(1, dtype=torch.bfloat16, device="cuda")

    def step(x, w, b):
        leaf = x.detach().requires_grad_()
        y = checkpointed_linear(leaf, w, b)
        return (y.detach(), *torch.autograd.grad(y, (leaf, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w0.clone().requires_grad_(), b0.clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    w, b = w0.clone().requires_grad_(), b0.clone().requires_grad_()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x, w, b)
        graphs.append((graph, outs))
    for _ in range(4):
        x.copy_(torch.roll(x, 1, 0) * 1.25)
        for graph, _ in graphs:
            graph.replay()
        eager = step(x, w0.clone().requires_grad_(), b0.clone().requires_grad_())
        torch.cuda.synchronize()
        for _, outs in graphs:
            for got, want in zip(outs, eager):
                assert torch.equal(got, want)


def test_one_output_past_32_bits():
    """Rows behind 2^31 elements: the bits of the same rows alone."""
    N, D = 40000, 60000
    x = torch.randn(100, D, device="cuda", dtype=torch.bfloat16).repeat(N // 100, 1)
    w = torch.randn(1, D, device="cuda", dtype=x.dtype, requires_grad=True)
    x[-3:] *= torch.rand(3, D, device="cuda").to(x.dtype)
    dy = torch.zeros(N, 1, device="cuda", dtype=x.dtype)
    dy[-3:] = torch.tensor([[1.5], [0.0], [0.0]], device="cuda")
    few = x[-3:].clone()
    leaf = x.requires_grad_()
    y = checkpointed_linear(leaf, w)
    assert torch.equal(y[-3:], checkpointed_linear(few, w)) and torch.equal(y[:100], y[100:200])
    dx, dw = torch.autograd.grad(y, (leaf, w), dy)
    assert torch.equal(dx[-3:], dy[-3:] * w) and not dx[:-3].any()
    assert torch.equal(dw, (1.5 * quantize_activation(few).dequantize()[:1].float()).to(x.dtype))  # one term


@pytest.mark.parametrize("route", ["host", "python", "compiled"])
@pytest.mark.parametrize("shape", [(6, 40), (2, 3, 40), (2, 2, 3, 40), (40,)])
@pytest.mark.parametrize("bias", [True, False])
def test_outputs_may_be_written_in_place(shape, bias, route, monkeypatch):
    """As torch.nn.Linear's: an activation or a residual in place, with and without a gradient to the weight, and behind a no_grad block."""
    if route == "python":
        monkeypatch.setattr(F, "_HOST", None)
    torch._dynamo.reset()
    torch.manual_seed(0)
    for out in (20, 1):
        layer = CheckpointedLinear(40, out, bias=bias, device="cuda")
        x = torch.randn(shape, device="cuda")
        r = torch.randn(shape[:-1] + (out,), device="cuda", requires_grad=True)

        def step(leaf):
            y = layer(leaf)
            y += r
            return y.relu_()

        f = torch.compile(step, fullgraph=True) if route == "compiled" else step
        for frozen in (False, True):
            layer.weight.requires_grad_(not frozen)
            leaf = x.clone().requires_grad_()
            y = f(leaf)
            want = torch.relu(layer(leaf) + r)
            torch.testing.assert_close(y, want, rtol=1e-6, atol=1e-6)  # sums of 40 products of this size, in two orders at most
            (dx,), (dx2,) = (torch.autograd.grad(t.sum(), leaf) for t in (y, want))
            torch.testing.assert_close(dx, dx2, rtol=1e-6, atol=1e-6)
        with torch.no_grad():
            y = layer(x)
        y += r
        assert torch.equal(torch.autograd.grad(y.sum(), r)[0], torch.ones_like(r))


@pytest.mark.parametrize("route", ["host", "python"])
@pytest.mark.parametrize("need", ["x", "weight", "x weight", "x weight bias"])
def test_the_gradient_is_not_differentiable_again(need, route, monkeypatch):
    if route == "python":
        monkeypatch.setattr(F, "_HOST", None)
    leaves = {"x": torch.randn(2, 5, 40, device="cuda"), "weight": torch.randn(3, 40, device="cuda"), "bias": torch.randn(3, device="cuda")}
    for k in need.split():
        leaves[k].requires_grad_()
    dy = torch.randn(2, 5, 3, device="cuda", requires_grad=True)
    y = checkpointed_linear(leaves["x"], leaves["weight"], leaves["bias"])
    grads = torch.autograd.grad(y, [leaves[k] for k in need.split()], dy, create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward(retain_graph=True)


@pytest.mark.parametrize("route", ["host", "python"])
@pytest.mark.parametrize("out", [1, 20])
def test_what_a_saved_tensor_hook_hands_back_is_checked(out, route, monkeypatch):
    """The kernels read what the kept sizes say: another layout is taken, another type, shape or device refused."""
    if route == "python":
        monkeypatch.setattr(F, "_HOST", None)
    g = torch.Generator().manual_seed(1)
    x, w, dy = (torch.randn(s, generator=g).cuda() for s in ((6, 70), (out, 70), (6, out)))

    def gradients(k, change):
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        count = []

        def pack(t):
            count.append(t)
            return len(count) - 1, t.detach().clone()

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda it: change(it[1]) if it[0] == k else it[1]):
            y = checkpointed_linear(*leaves)
        assert len(count) == 3  # codes, exponents, weight
        return torch.autograd.grad(y, leaves, dy)

    want = gradients(-1, None)
    for k in range(3):
        for a, b in zip(gradients(k, lambda t: t.t().contiguous().t()), want):
            if k < 2 or out == 1:
                assert torch.equal(a, b)
            else:  # the library's product of another layout: sums of 20 in another order
                torch.testing.assert_close(a, b, rtol=0, atol=40 * 2.0 ** -24 * 20 * 10)
        for change in (lambda t: t.to(torch.int16), lambda t: t[:, :-1], lambda t: t.cpu()):
            with pytest.raises(RuntimeError):
                gradients(k, change)


def test_more_rows_than_a_launch_takes():
    """2^26 rows of a value head and 2^35 elements of an activation are several launches: the bits of the same rows alone."""
    few, N, D = 1 << 10, (1 << 26) + 37, 32
    x, w, dy = (torch.randn(s, device="cuda").bfloat16() for s in ((few, D), (1, D), (few, 1)))
    want_y = checkpointed_linear(x, w.requires_grad_())
    kept = quantize_activation(x)
    (want_dx,) = torch.autograd.grad(checkpointed_linear(x.requires_grad_(), w), x, dy)
    leaf = x.detach().repeat(N // few + 1, 1)[:N].requires_grad_()
    y = checkpointed_linear(leaf, w)
    dx, dw = torch.autograd.grad(y, (leaf, w), dy.repeat(N // few + 1, 1)[:N])
    for got, want in ((y.detach(), want_y.detach()), (dx, want_dx)):
        whole = got[:N // few * few].view(-1, few, got.shape[-1])
        assert torch.equal(whole.amin(0), whole.amax(0)) and torch.equal(got[:few], want) and torch.equal(got[-(N % few):], want[:N % few])
    # sums of one wave's every 8th row of 256 splits, 32769 roundings, then 8 waves and 256 splits: under 34000 of the sum of magnitudes
    parts = dy.double().T @ kept.dequantize().double()
    size = dy.double().abs().T @ kept.dequantize().double().abs()
    times = N / few
    rest = dy.double()[:N % few].T @ kept.dequantize().double()[:N % few]
    whole_sum = parts * (N // few) + rest
    O.assert_close(dw, whole_sum.cpu(), (34000 * O.U * size * (times + 1)).cpu(), "dw")
    del leaf, y, dx, dw, got, whole
    row = torch.randn(1, 512, device="cuda").bfloat16()
    q = quantize_activation(row.expand(N, 512))  # 2^35 elements and some
    one = quantize_activation(row)
    back = q.dequantize()
    values = one.dequantize()
    for i in range(0, N, 1 << 23):
        assert torch.equal(q.codes[i:i + (1 << 23)], one.codes.expand(min(1 << 23, N - i), -1))
        assert torch.equal(back[i:i + (1 << 23)], values.expand(min(1 << 23, N - i), -1))
    assert torch.equal(q.exponents, one.exponents.expand(N, -1))
    del q, back
    torch.cuda.empty_cache()


@pytest.mark.parametrize("route", ["host", "python", "compiled"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", [1, 3])
def test_the_same_output_in_training_and_evaluation(out, dtype, route, monkeypatch):
    if route == "python":
        monkeypatch.setattr(F, "_HOST", None)
    torch._dynamo.reset()
    x = inputs(300, 1100, dtype, seed=5).clamp(-30, 30).cuda().view(3, 100, 1100)
    layer = CheckpointedLinear(1100, out, device="cuda", dtype=dtype)
    f = torch.compile(layer, fullgraph=True) if route == "compiled" else layer
    want = layer(x).detach()  # the weight wants a gradient
    assert torch.equal(f(x).detach(), want)
    with torch.no_grad():
        assert torch.equal(f(x), want)
    with torch.inference_mode():
        assert torch.equal(f(x), want)
    layer.weight.requires_grad_(False)
    assert torch.equal(f(x.clone().requires_grad_()).detach(), want)
    layer.bias.requires_grad_(False)
    y = f(x)
    assert torch.equal(y, want) and not y.requires_grad
    if out == 1:
        assert F.last_kernel() == "act_head"


def test_the_python_route_keeps_nothing_without_a_gradient(monkeypatch):
    monkeypatch.setattr(F, "_HOST", None)
    x, layer = torch.randn(4096, 1024, device="cuda"), CheckpointedLinear(1024, 1, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        y = layer(x)
    assert torch.cuda.max_memory_allocated() - before <= y.numel() * 4 + 4096
