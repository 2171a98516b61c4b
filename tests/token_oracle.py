"""Plain 64-bit forms, on the CPU, of the token-policy operators and of the 8-bit activation format, with error bounds of the kernels'
32-bit arithmetic (include/trl_value.h has the formulas)."""
import math

import torch

U = 2.0 ** -24  # half a step of float32


def as_rows(x, B, T, n):
    """Any broadcastable tensor as (B, T, n)."""
    return x.expand(B, T, n) if x.ndim == 3 else x.reshape(1, 1, n).expand(B, T, n)


def bits_to_bool(words, V):
    b = (words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32)) & 1
    return b.bool().flatten(-2)[..., :V]


def bool_to_bits(mask):
    V = mask.shape[-1]
    pad = torch.nn.functional.pad(mask, (0, -V % 32)).unflatten(-1, (-1, 32)).long()
    w = (pad << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def counts(tokens, lengths, prompt, V):
    """(seen, generated) counts (B, T, V) of (B, L) tokens, (B, T) lengths, (B,) prompt lengths."""
    B, T = lengths.shape
    L = tokens.shape[1]
    seen, new = torch.zeros(B, T, V, dtype=torch.float64), torch.zeros(B, T, V, dtype=torch.float64)
    for b in range(B):
        for t in range(T):
            n = min(max(int(lengths[b, t]), 0), L)
            for lo, out in ((0, seen), (min(max(int(prompt[b]), 0), n), new)):
                ids = tokens[b, lo:n].long()
                out[b, t] = torch.bincount(ids[(ids >= 0) & (ids < V)], minlength=V).double()
    return seen, new


class Result:
    pass


def token_policy(z, tokens=None, lengths=None, prompt=None, rep=1.0, pres=0.0, freq=0.0, bias=None, mask=None, temp=1.0, action=None,
                 g_lp=None, g_H=None, g_out=None):
    """z (B, T, V) and CPU tensors of the kernels' inputs; penalties and temperature: numbers or (B,) tensors.  Returns the processed logits,
    log-probabilities, entropies, gradients, and bounds (`*_tol`) of what 32-bit arithmetic may be off by, final rounding not included."""
    r = Result()
    B, T, V = z.shape
    col = lambda x: x.double().reshape(B, 1, 1) if isinstance(x, torch.Tensor) else float(x)  # noqa: E731
    rep, pres, freq, temp = col(rep), col(pres), col(freq), col(temp)
    z = z.double()
    size = z.abs()
    slope = torch.ones_like(z)
    if tokens is not None:
        seen, new = counts(tokens, lengths, prompt if prompt is not None else torch.zeros(B), V)
        f = torch.where(seen > 0, torch.where(z > 0, 1.0 / rep + 0 * z, rep + 0 * z), 1.0)
        pen = freq * new + pres * (new > 0)
        z, slope, size = torch.where(f == 1.0, z, z * f) - pen, slope * f, size * f + torch.as_tensor(abs(freq) * new + abs(pres) * (new > 0))
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    z, slope, size = z / temp, slope / temp, size / temp
    ok = torch.ones(B, T, V, dtype=torch.bool) if mask is None else mask.expand(B, T, V)
    z = torch.where(ok, z, -math.inf)
    slope = torch.where(ok, slope, 0.0)
    size = torch.where(ok & torch.isfinite(size), size, 0.0)
    # parameters rounded to 32 bits and their reciprocals (4), the products and sums (5), rounded up
    r.out, r.out_tol, r.ok = z, 12 * U * size, ok
    if g_out is not None:
        r.d_process = torch.where(ok, g_out.double() * slope, 0.0)
        r.d_process_tol = 8 * U * r.d_process.abs()
    if action is None:
        return r
    real = action >= 0
    inside = real & (action < V)
    top = z.amax(-1, keepdim=True)
    empty = top == -math.inf
    d = torch.where(empty, -math.inf, z - torch.where(empty, 0.0, top))
    s = torch.exp(d).sum(-1, keepdim=True)
    log_p = torch.where(empty, -math.inf, d - torch.log(torch.where(empty, 1.0, s)))
    p = torch.exp(log_p)
    plogp = torch.where(p > 0, p * torch.where(p > 0, log_p, 0.0), 0.0)
    H = -plogp.sum(-1)
    at = torch.where(inside, action, 0).unsqueeze(-1)
    lp = log_p.gather(-1, at).squeeze(-1)
    r.log_prob = torch.where(real, torch.where(inside, lp, math.nan), 0.0)
    r.entropy = torch.where(real, H, 0.0)
    # the logits' own error moves log p by at most twice its largest; d and its constant round, and so do the sums (32 a lane, the
    # butterflies, the join: 64 steps are more than enough), the logarithm and the last difference
    big = 12 * size.amax(-1)
    fin = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
    r.log_prob_tol = U * (2 * big + 4 * fin + 2 * math.log(max(V, 2)) + 80)
    r.entropy_tol = U * (2 * big * (H + 1) + 160 * (H + math.log(max(V, 2)) + 1))
    if g_lp is not None or g_H is not None:
        g_lp = torch.zeros(B, T) if g_lp is None else g_lp
        g_H = torch.zeros(B, T) if g_H is None else g_H
        live = (real & ~empty.squeeze(-1)).unsqueeze(-1)
        a, b = g_lp.double().unsqueeze(-1), g_H.double().unsqueeze(-1)
        safe = torch.where(p > 0, log_p, 0.0)
        dz = -p * (a + b * (safe + H.unsqueeze(-1)))
        onehot = torch.zeros_like(z).scatter(-1, at, 1.0) * inside.unsqueeze(-1)
        dz = dz + onehot * a
        dz = torch.where((action >= V).unsqueeze(-1) & live, math.nan, dz)
        r.d_logits = torch.where(live & ok, dz * slope, 0.0)
        rel = U * (2 * big.unsqueeze(-1) + 4 * safe.abs() + 2 * math.log(max(V, 2)) + 100)  # of p
        inner = a.abs() + b.abs() * (safe.abs() + H.unsqueeze(-1) + 1)
        r.d_logits_tol = torch.where(live & ok, slope * (p * inner * (2 * rel + 8 * U) + p * b.abs() * (rel + r.entropy_tol.unsqueeze(-1))
                                                         + onehot * a.abs() * 4 * U), 0.0)
    return r


def assert_close(got, want, tol, what, floor=0.0):
    """|got - want| <= tol + half a step of got's type; infinities and NaN have to be where they belong.  floor: half a subnormal step."""
    got, dt = got.detach().cpu(), got.dtype
    half = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    g = got.double()
    want = want.reshape(g.shape)
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape) if not isinstance(tol, torch.Tensor) else tol.reshape(g.shape)
    bad_kind = (torch.isnan(g) != torch.isnan(want)) | (torch.isinf(g) != torch.isinf(want))
    assert not bad_kind.any(), f"{what}: NaN or infinity at {bad_kind.nonzero()[:4].tolist()}: {g[bad_kind][:4]} for {want[bad_kind][:4]}"
    same = torch.isinf(want) & (g == want) | torch.isnan(want)
    off = torch.where(same, 0.0, (g - torch.where(same, 0.0, want)).abs())
    limit = torch.where(same, 0.0, tol + half * (torch.where(same, 0.0, want).abs() + tol) + tiny + floor)
    worst = off - limit
    assert (worst <= 0).all(), f"{what}: off by {off[worst > 0][:4].tolist()}, allowed {limit[worst > 0][:4].tolist()} at {(worst > 0).nonzero()[:4].tolist()}"


# ---- 8-bit activations -----------------------------------------------------------------------------------------------------
def kept(x):
    """(codes, exponents, values in 64 bits) of a finite or non-finite (N, D) tensor: loops over blocks, python's frexp."""
    x = x.double()
    N, D = x.shape
    blocks = (D + 31) // 32
    codes, exps, values = torch.zeros(N, blocks * 32, dtype=torch.int8), torch.zeros(N, blocks, dtype=torch.uint8), torch.zeros(N, D, dtype=torch.float64)
    for n in range(N):
        for k in range(blocks):
            part = x[n, 32 * k:32 * k + 32]
            if not torch.isfinite(part).all():
                exps[n, k] = 255
                values[n, 32 * k:32 * k + 32] = math.nan
                continue
            top = float(part.abs().max())
            e = max((math.frexp(top)[1] - 1 - 6) if top > 0 else -126, -126)
            q = torch.round(part / 2.0 ** e).clamp(-127, 127)
            codes[n, 32 * k:32 * k + len(part)] = q.to(torch.int8)
            exps[n, k] = e + 127
            values[n, 32 * k:32 * k + 32] = q * 2.0 ** e
    return codes, exps, values
