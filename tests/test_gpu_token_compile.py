"""GPU: torch.compile(fullgraph=True) over the token-policy operators and the 8-bit activations: the eager calls' results, gradients included."""
import pytest
import torch

from torchrl_amd.objectives.value import CheckpointedLinear, process_logits, quantize_activation, token_log_prob

pytestmark = pytest.mark.gpu


def test_a_policy_gradient_step_compiles_fullgraph():
    torch.manual_seed(0)
    B, T, D, V, P = 2, 6, 40, 130, 3
    dev = "cuda"
    x = torch.randn(B, T, D, device=dev)
    tokens = torch.randint(0, V, (B, P + T), device=dev)
    lengths = (P + torch.arange(T, device=dev)).expand(B, T).contiguous()
    mask = torch.rand(B, T, V, device=dev) < 0.8
    temperature = torch.rand(B, device=dev) + 0.5
    adv = torch.randn(B, T, device=dev)
    head = CheckpointedLinear(D, V, device=dev)

    def step(x):
        z = head(x)
        kw = dict(tokens=tokens, lengths=lengths, repetition_penalty=1.2, frequency_penalty=0.1, mask=mask, temperature=temperature)
        lp, H = token_log_prob(z, tokens[:, P:], entropy=True, **kw)
        out = process_logits(z, **kw)
        return lp, H, out, -(lp.clamp(min=-20) * adv).mean() - 0.01 * H.mean() + 0.001 * out.clamp(min=-20).mean()

    def run(fn):
        leaf = x.clone().requires_grad_()
        head.zero_grad()
        lp, H, out, loss = fn(leaf)
        loss.backward()
        return lp.detach(), H.detach(), out.detach(), leaf.grad, head.weight.grad.clone(), head.bias.grad.clone()

    for a, b in zip(run(step), run(torch.compile(step, fullgraph=True))):
        # the ops are the same kernels; the sums around them are fused: a few roundings of values of this size
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_refusals_under_compile():
    z = torch.randn(2, 3, 20, device="cuda", requires_grad=True)
    bias = torch.zeros(20, device="cuda", requires_grad=True)
    with pytest.raises(Exception, match="bias"):
        torch.compile(lambda z: process_logits(z, bias=bias), fullgraph=True)(z)


def test_kept_activations_compile_fullgraph():
    x = torch.randn(3, 5, 70, device="cuda", dtype=torch.bfloat16)

    def there_and_back(x):
        q = quantize_activation(x)
        return q.codes, q.exponents, q.dequantize(), q.dequantize(torch.float32)

    for a, b in zip(there_and_back(x), torch.compile(there_and_back, fullgraph=True)(x)):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_a_value_head_compiles_fullgraph():
    torch.manual_seed(0)
    x, dy = torch.randn(3, 50, 200, device="cuda"), torch.randn(3, 50, 1, device="cuda")
    head = CheckpointedLinear(200, 1, device="cuda")

    def run(fn):
        leaf = x.clone().requires_grad_()
        head.zero_grad()
        y = fn(leaf)
        y.backward(dy)
        return y.detach(), leaf.grad, head.weight.grad.clone(), head.bias.grad.clone()

    for a, b in zip(run(head), run(torch.compile(head, fullgraph=True))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("out", [1, 24])
@pytest.mark.parametrize("form", ["no_grad", "frozen weight", "bias alone", "all"])
def test_a_compiled_layer_keeps_what_the_eager_one_keeps(form, out):
    """No quantization and no weight gradient where the weight wants none; the same results."""
    torch._dynamo.reset()
    torch.manual_seed(0)
    x, dy = torch.randn(5, 64, 512, device="cuda"), torch.randn(5, 64, out, device="cuda")
    layer = CheckpointedLinear(512, out, device="cuda")
    layer.weight.requires_grad_(form in ("no_grad", "all"))
    graphs = []

    def backend(graph, example_inputs):
        from torch._dynamo.backends.common import aot_autograd

        def seen(g, _):
            graphs.append([str(n.target) for n in g.graph.nodes])
            return g

        return aot_autograd(fw_compiler=seen, bw_compiler=seen)(graph, example_inputs)

    def run(f):
        leaf = x.clone().requires_grad_(form != "bias alone")
        layer.zero_grad()
        if form == "no_grad":
            with torch.no_grad():
                return (f(leaf),)
        y = f(leaf)
        y.backward(dy)
        return y.detach(), leaf.grad, layer.weight.grad, None if layer.bias.grad is None else layer.bias.grad.clone()

    for a, b in zip(run(layer), run(torch.compile(layer, fullgraph=True, backend=backend))):
        if a is None:
            assert b is None
        else:  # the bias's gradient is a sum of 320 numbers in two orders
            torch.testing.assert_close(a, b, rtol=0, atol=320 * 2.0 ** -24 * 320 ** 0.5 * 4 if a.shape == (out,) and a.ndim == 1 else 0)
    ops = [n for g in graphs for n in g]
    kept = any("checkpointed_linear" in n or "weight_grad" in n or "head_grad" in n for n in ops)
    assert ops and kept == (form == "all")


def test_refused_layers_under_compile():
    layer = CheckpointedLinear(40, 8)
    with torch.no_grad(), pytest.raises(Exception, match="HIP"):
        torch.compile(layer, fullgraph=True)(torch.zeros(3, 40))
