"""CPU: what the token-policy operators and the 8-bit activations refuse (nothing is launched), and the oracle's own known answers."""
import ctypes
import math

import pytest
import torch

import token_oracle as O
from torchrl_amd import _extension
from torchrl_amd.objectives.value import CheckpointedLinear, TokenActor, checkpointed_linear, process_logits, quantize_activation, token_log_prob

Z = torch.zeros(2, 3, 40)
TOK = torch.zeros(2, 9, dtype=torch.long)
LEN = torch.zeros(2, 3, dtype=torch.long)
ACT = torch.zeros(2, 3, dtype=torch.long)
PEN = dict(tokens=TOK, lengths=LEN, repetition_penalty=1.1)


@pytest.mark.parametrize("logits,kwargs,error,match", [
    (Z, {}, RuntimeError, "HIP"),  # a good call, but for the device
    (Z, PEN, RuntimeError, "HIP"),
    (Z.double(), {}, NotImplementedError, "float32, bfloat16 and float16"),
    (torch.zeros(2, 0), {}, RuntimeError, "vocabulary"),
    (torch.zeros(()), {}, RuntimeError, "vocabulary"),
    (Z, dict(repetition_penalty=1.1), ValueError, "penalties need the tokens"),
    (Z, dict(lengths=LEN), ValueError, "go with tokens"),
    (Z, dict(tokens=TOK), ValueError, "need lengths"),
    (Z, dict(tokens=TOK.float(), lengths=LEN), RuntimeError, "int32 or int64"),
    (Z, dict(tokens=torch.zeros(3, 9, dtype=torch.long), lengths=LEN), RuntimeError, "do not belong"),
    (Z, dict(tokens=torch.zeros(9, dtype=torch.long), lengths=LEN), RuntimeError, r"\[\*B, L\]"),
    (Z, dict(tokens=TOK, lengths=LEN[:, :2]), RuntimeError, "lengths must have shape"),
    (Z, dict(tokens=TOK, lengths=LEN.float()), RuntimeError, "lengths must be"),
    (Z, dict(PEN, prompt_lengths=LEN), RuntimeError, "prompt_lengths must have shape"),
    (Z, dict(PEN, repetition_penalty=0.0), ValueError, "positive"),
    (Z, dict(PEN, presence_penalty=math.inf), ValueError, "finite"),
    (Z, dict(temperature=0.0), ValueError, "positive"),
    (Z, dict(temperature=-1.0), ValueError, "positive"),
    (Z, dict(temperature=math.nan), ValueError, "positive"),
    (Z, dict(temperature=1e-39), ValueError, "positive"),
    (Z, dict(PEN, frequency_penalty=1e39), ValueError, "finite"),
    (Z, dict(temperature=torch.ones(3)), RuntimeError, "does not broadcast to the sequences"),
    (Z, dict(temperature=torch.ones(2, dtype=torch.long)), RuntimeError, "floating-point"),
    (Z, dict(temperature=torch.ones(2, requires_grad=True)), NotImplementedError, "temperature"),
    (Z, dict(bias=torch.zeros(39)), RuntimeError, "40 entries"),
    (Z, dict(bias=torch.zeros(40, dtype=torch.float64)), RuntimeError, "bias must be"),
    (Z, dict(bias=torch.zeros(40, requires_grad=True)), NotImplementedError, "bias"),
    (Z, dict(bias=torch.zeros(3, 3, 40)), RuntimeError, "broadcast"),
    (Z, dict(mask=torch.ones(2, 3, 39, dtype=torch.bool)), RuntimeError, "40 entries"),
    (Z, dict(mask=torch.ones(2, 3, 40, dtype=torch.int32)), RuntimeError, "2 entries"),
    (Z, dict(mask=torch.ones(2, 3, 40, dtype=torch.uint8)), RuntimeError, "bool tensor"),
    (Z, dict(mask=torch.ones(4, 2, 3, 40, dtype=torch.bool)), RuntimeError, "broadcast"),
])
def test_refused_processing(logits, kwargs, error, match):
    with pytest.raises(error, match=match):
        process_logits(logits, **kwargs)
    if logits.ndim and logits.numel():
        with pytest.raises(error, match=match):
            token_log_prob(logits, ACT, **kwargs)


@pytest.mark.parametrize("action", [ACT[:, :2], ACT.float(), ACT.bool(), None])
def test_refused_actions(action):
    with pytest.raises(RuntimeError, match="action must"):
        token_log_prob(Z, action)


def test_refused_linear():
    x, w, b = torch.zeros(4, 6), torch.zeros(5, 6), torch.zeros(5)
    for args, error, match in [((x, w, b), RuntimeError, "HIP"), ((x, w[:, :5], b), RuntimeError, "do not fit"), ((x, w[0], b), RuntimeError, "do not fit"),
                               ((x, w, b[:4]), RuntimeError, "bias must have shape"), ((x, w.bfloat16(), b), RuntimeError, "weight is"),
                               ((x, w, b.half()), RuntimeError, "bias is"), ((x.double(), w, b), NotImplementedError, "float32"),
                               ((x, w[:0], None), RuntimeError, "do not fit"), ((None, w, b), TypeError, "x must be")]:
        with pytest.raises(error, match=match):
            checkpointed_linear(*args)
    with pytest.raises(RuntimeError, match="HIP"):
        CheckpointedLinear(6, 5)(x)
    for bad, error, match in [(x, RuntimeError, "HIP"), (x.long(), NotImplementedError, "float32"), (torch.zeros(3, 0), RuntimeError, "feature dim")]:
        with pytest.raises(error, match=match):
            quantize_activation(bad)


def test_actor_hands_everything_over():
    class Data(dict):
        pass

    actor = TokenActor(lambda d: Z, tokens_key="tokens", lengths_key="lengths", temperature=0.5, repetition_penalty=1.5)
    logits, kwargs = actor._inputs(Data(tokens=TOK, lengths=LEN))
    assert logits is Z and kwargs["tokens"] is TOK and kwargs["lengths"] is LEN and kwargs["temperature"] == 0.5
    assert kwargs["repetition_penalty"] == 1.5 and kwargs["bias"] is None and "mask" not in kwargs
    with pytest.raises(RuntimeError, match="HIP"):
        actor(Data(tokens=TOK, lengths=LEN, action=ACT))


# ---- the C entry points (bad arguments come back before anything is launched) --------------------------------------------------
def token_args(**kw):
    # what the pointers point to is never read: every call below is refused
    a = dict(dtype=0, B=2, T=3, V=40, L=0, rep=1.0, temp=1.0, logits=64, out=64, logits_sb=120, logits_st=40, action=64, log_prob=64, stats=64,
             g_log_prob=64, grad_out=64)
    a.update(kw)
    return _extension.TokenArgs(**a)


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=1), 1), (dict(dtype=9), 1), (dict(B=-1), 1), (dict(V=0), 1), (dict(V=2 ** 31), 1), (dict(L=-1), 1), (dict(mask_kind=1), 1),
    (dict(mask_kind=7, mask=64), 1), (dict(bias_kind=1), 1), (dict(bias_kind=2, bias=64), 1), (dict(rep=0.0), 1), (dict(temp=math.nan), 1),
    (dict(logits=None), 1), (dict(B=2 ** 40, T=2 ** 20), 1),
])
@pytest.mark.parametrize("name", ["trl_process_logits_fwd", "trl_token_log_prob_fwd", "trl_token_log_prob_bwd"])
def test_c_entry_points_refuse(name, bad, code):
    lib = _extension.get_lib()
    more = (64, 1 << 40) if name == "trl_token_log_prob_fwd" else ()
    assert getattr(lib, name)(None, token_args(**bad), *more) == code
    assert name.encode() in lib.trl_last_error()


def test_c_entry_points_refuse_more():
    lib = _extension.get_lib()
    need = lib.trl_token_workspace_bytes(2, 3, 40)
    assert need == 2 * 3 * (16 + 4) and lib.trl_token_workspace_bytes(0, 3, 40) == 0
    assert lib.trl_token_log_prob_fwd(None, token_args(), 64, need - 1) == 3  # too small
    assert lib.trl_token_log_prob_fwd(None, token_args(), 72, need) == 3  # not aligned
    assert lib.trl_token_log_prob_fwd(None, token_args(), None, need) == 3
    for missing in ("action", "log_prob"):
        assert lib.trl_token_log_prob_fwd(None, token_args(**{missing: None}), 64, need) == 1
    for missing in ("action", "stats", "out", "g_log_prob"):
        assert lib.trl_token_log_prob_bwd(None, token_args(**{missing: None})) == 1
    assert lib.trl_token_log_prob_bwd(None, token_args(g_entropy=64)) == 1  # the entropy itself is missing
    assert lib.trl_process_logits_bwd(None, token_args(grad_out=None)) == 1
    assert lib.trl_process_logits_bwd(None, token_args(logits=None, tokens=64, rep=1.5)) == 1  # the sign of the logits is needed
    assert lib.trl_process_logits_fwd(None, token_args(B=0, logits=None, out=None)) == 0  # no rows: nothing to do
    assert lib.trl_process_logits_fwd(None, None) == 1
    assert lib.trl_act_quantize(None, 1, 64, 8, 4, 8, 64, 64) == 1 and lib.trl_act_quantize(None, 0, None, 8, 4, 8, 64, 64) == 1
    assert lib.trl_act_quantize(None, 0, 64, 8, -1, 8, 64, 64) == 1 and lib.trl_act_quantize(None, 0, 64, 8, 4, 8, 72, 64) == 1
    assert lib.trl_act_quantize(None, 0, 64, 8, 2 ** 30, 2 ** 20, 64, 64) == 2
    assert lib.trl_act_quantize(None, 0, None, 8, 0, 8, None, None) == 0
    assert lib.trl_act_dequantize(None, 0, 64, 64, 4, 0, 64) == 1 and lib.trl_act_dequantize(None, 3, 64, None, 4, 8, 64) == 1
    assert lib.trl_act_weight_grad(None, 2, None, 8, 64, 64, 4, 8, 8, 64, None, 64, 1 << 30) == 1
    assert lib.trl_act_weight_grad(None, 2, 64, 8, 64, 64, 4, 0, 8, 64, None, 64, 1 << 30) == 1
    need = lib.trl_act_weight_grad_workspace_bytes(2, 100000, 4, 32)
    if need:
        assert lib.trl_act_weight_grad(None, 2, 64, 8, 64, 64, 100000, 4, 32, 64, None, 64, need - 1) == 3
    assert lib.trl_act_head_fwd(None, 0, None, 8, 4, 8, 64, None, 64, 64, 64) == 1 and lib.trl_act_head_fwd(None, 0, 64, 8, 4, 8, 64, None, 72, 64, 64) == 1
    assert lib.trl_act_head_fwd(None, 1, 64, 8, 4, 8, 64, None, 64, 64, 64) == 1 and lib.trl_act_head_fwd(None, 0, None, 8, 0, 8, None, None, None, None, None) == 0
    assert lib.trl_act_head_bwd(None, 0, 64, 1, 64, 64, 4, 8, None, 64, None, 64, 64, 1 << 30) == 1  # dx without w
    assert lib.trl_act_head_bwd(None, 0, 64, 1, 64, 64, 4, 8, 64, None, None, 64, 64, 1 << 30) == 1  # no dw
    need = lib.trl_act_weight_grad_workspace_bytes(0, 100000, 1, 32)
    assert need and lib.trl_act_head_bwd(None, 0, 64, 1, 64, 64, 100000, 32, 64, 64, None, 64, 64, need - 1) == 3


# ---- the oracle's known answers -----------------------------------------------------------------------------------------------
def test_oracle_by_hand():
    z = torch.tensor([[[2.0, -1.0, 0.0, 4.0]]])
    r = O.token_policy(z, tokens=torch.tensor([[0, 1, 1, 7, -1, 3]]), lengths=torch.tensor([[5]]), prompt=torch.tensor([1]), rep=2.0, pres=0.5, freq=0.25,
                       bias=torch.tensor([0.0, 0.0, 1.0, 0.0]), temp=0.5, mask=torch.tensor([True, True, True, False]), action=torch.tensor([[2]]))
    # token 0 in the prompt only, token 1 twice behind it, 3 not yet
    assert r.out.flatten().tolist() == [2.0, (-2.0 - 0.5 - 0.5) * 2, 2.0, -math.inf]
    assert float(r.log_prob) == pytest.approx(2.0 - math.log(2 * math.exp(2.0) + math.exp(-6.0)), abs=1e-12)
    words = O.bool_to_bits(torch.tensor([True] * 31 + [True, False, True]))
    assert words.tolist() == [-1, 2] and O.bits_to_bool(words, 34).tolist() == [True] * 32 + [False, True]


def test_oracle_gradient_is_autograds():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(2, 3, 11, generator=g, dtype=torch.float64).requires_grad_()
    action, a, b = torch.randint(0, 11, (2, 3), generator=g), torch.randn(2, 3, generator=g), torch.randn(2, 3, generator=g)
    lp = torch.log_softmax(z / 0.7, -1)
    loss = (lp.gather(-1, action.unsqueeze(-1)).squeeze(-1) * a).sum() - ((lp.exp() * lp).sum(-1) * b).sum()
    (want,) = torch.autograd.grad(loss, z)
    got = O.token_policy(z.detach(), temp=0.7, action=action, g_lp=a, g_H=b).d_logits
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)


def processing(logits, **tensors):
    from torchrl_amd.objectives.value import tokens as K

    B, V = logits.shape
    p = K._Processing(B, 1, V, logits.unsqueeze(1), None, None, None, 1.0, 0.0, 0.0, 1.0, *[None] * 6)
    return p._replace(**tensors)


def test_out_shares_no_memory_with_the_inputs_but_the_logits():
    from torchrl_amd.objectives.value.tokens import _out_rows

    z, refused = torch.zeros(4, 40), "share no memory"
    shared = z[:1].expand(4, 40).unsqueeze(1)  # a bias read by all rows, and written with the first
    with pytest.raises(RuntimeError, match=refused):
        _out_rows(processing(z, bias=shared), z, z)
    with pytest.raises(RuntimeError, match=refused):
        _out_rows(processing(z, mask=z.view(torch.bool)[:, :40].unsqueeze(1)), z, z)
    with pytest.raises(RuntimeError, match=refused):
        _out_rows(processing(z[:, :20], bias=z[:, 10:30].unsqueeze(1)), z[:, :20], z[:, :20])  # columns that overlap
    with pytest.raises(RuntimeError, match=refused):
        _out_rows(processing(z[1:], bias=None), z[1:], z[:3])  # the logits, a row further on
    with pytest.raises(RuntimeError, match=refused):
        _out_rows(processing(z, temp_t=z.view(-1)[100:104]), z, z)
    # beside each other in one buffer
    assert _out_rows(processing(z, bias=torch.zeros(40).expand(4, 1, 40)), z, z).shape == (4, 1, 40)
    assert _out_rows(processing(z[:, :20], bias=z[:, 20:].unsqueeze(1)), z[:, :20], z[:, :20]).data_ptr() == z.data_ptr()
    assert _out_rows(processing(z[:, 20:], bias=z[2, :20].expand(4, 1, 20)), z[:, 20:], z[:, 20:]).shape == (4, 1, 20)
    assert _out_rows(processing(z[:2], bias=z[2:].unsqueeze(1)), z[:2], z[:2]).shape == (2, 1, 40)
    assert _out_rows(processing(z[:, :20]), z[:, :20], z[:, 20:]).shape == (4, 1, 20)
    with pytest.raises(RuntimeError, match="do not overlap"):
        _out_rows(processing(z), z, torch.zeros(1, 40).expand(4, 40))
    with pytest.raises(RuntimeError, match="shape, dtype"):
        _out_rows(processing(z), z, z.half())


def test_more_rows_of_a_sequence_than_a_launch_takes():
    """2^32 threads and more: refused before anything is launched (sequences beyond that go in several launches)."""
    lib = _extension.get_lib()
    long = dict(B=1, T=1 << 33, V=4)
    assert lib.trl_process_logits_fwd(None, token_args(**long)) == 2 and b"more rows" in lib.trl_last_error()
    assert lib.trl_process_logits_bwd(None, token_args(**long)) == 2 and lib.trl_token_log_prob_bwd(None, token_args(**long)) == 2
    assert lib.trl_token_log_prob_fwd(None, token_args(**long), 64, 1 << 60) == 2
    assert lib.trl_token_log_prob_fwd(None, token_args(B=1, T=1 << 27, V=20000), 64, 1 << 60) == 2  # the rows' kernel would fit, joining would not


def test_a_value_head_without_keeping():
    lib = _extension.get_lib()
    assert lib.trl_act_head_fwd(None, 0, 64, 8, 4, 8, 64, None, None, 64, 64) == 1 and lib.trl_act_head_fwd(None, 0, 64, 8, 4, 8, 64, None, 64, None, 64) == 1


def test_an_actors_tensors_move_with_it():
    temperature = torch.tensor([0.7, 0.9])
    actor = TokenActor(torch.nn.Linear(3, 4), temperature=temperature, presence_penalty=0.5, bias=torch.zeros(4))
    keys = set(actor.state_dict())
    assert actor.to("meta") is actor
    assert actor.settings["temperature"].device.type == "meta" and actor.bias.device.type == "meta" and actor.settings["presence_penalty"] == 0.5
    actor = TokenActor(torch.nn.Linear(3, 4), temperature=temperature, bias=torch.zeros(4)).to(torch.bfloat16)
    assert torch.equal(actor.settings["temperature"], temperature) and actor.settings["temperature"].dtype == torch.float32
    assert set(actor.state_dict()) == keys == {"bias", "network.weight", "network.bias"}


@pytest.mark.parametrize("name", ["temperature", "presence_penalty"])
def test_numbers_that_round_to_infinity_are_refused(name):
    largest = torch.finfo(torch.float32).max
    kw = {} if name == "temperature" else dict(tokens=TOK, lengths=LEN)
    with pytest.raises(RuntimeError, match="HIP"):
        process_logits(Z, **{name: largest}, **kw)
    with pytest.raises(ValueError, match="finite"):
        process_logits(Z, **{name: math.nextafter(2.0 ** 128, 0.0)}, **kw)
