"""TEST INFRASTRUCTURE ONLY -- Python front-end of the CPU oracle.

Only tests/, ``__graft_entry__.smoke()`` and ``bench.py``'s ``cpu_baseline`` leg may
import this module; the product package ``torchrl_amd`` never does.

The arithmetic lives in ``value_oracle.c`` / ``value_oracle_impl.h`` (plain C restatement of
the reference's sequential loops, reference: torchrl/objectives/value/functional.py:121-182,
783-889, 1270-1350).  This file only (i) reshapes ``[*B, T, *F]`` inputs to the canonical
contiguous ``(O, T, I)`` view (the effect of the reference's ``_transpose_time`` decorator,
functional.py:49-113), and (ii) reproduces the dtype the reference's coefficient tensors get
(``gamma * int_mask`` rounds python floats to the default dtype) by running
the same torch expression on a one-element int32 tensor.

Parity pin: tests/test_oracle_golden.py checks every function against the golden fixtures in
tests/golden/ (generated by tools/gen_golden.py from the imported reference) and, when
/root/reference is present, against the reference itself.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "_build", "libvalue_oracle.so")
_lib = None

_c_f = {torch.float32: ctypes.c_float, torch.float64: ctypes.c_double}
_sfx = {
    (torch.float32, torch.float32): "f32",
    (torch.float64, torch.float64): "f64",
    (torch.float64, torch.float32): "f64g32",
    (torch.float32, torch.float64): "f32g64",
}


def build(force: bool = False) -> str:
    """Compile the C oracle with gcc (idempotent)."""
    src = [os.path.join(_HERE, f) for f in ("value_oracle.c", "value_oracle_impl.h")]
    if (
        force
        or not os.path.exists(_LIB_PATH)
        or any(os.path.getmtime(s) > os.path.getmtime(_LIB_PATH) for s in src)
    ):
        subprocess.check_call(["make", "-C", _HERE, "-B", "-s"])
    return _LIB_PATH


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            build()
        _lib = ctypes.CDLL(_LIB_PATH)
    return _lib


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _canon_dims(shape, time_dim):
    nd = len(shape)
    td = time_dim if time_dim < 0 else time_dim - nd
    if nd == 1 and td == -1:
        return 1, shape[0], 1
    if nd < 2 or td < -nd or td >= 0:
        raise RuntimeError(f"The tensor shape and the time dimension are not compatible: got {shape} and time_dim={td}.")
    td += nd
    O = int(np.prod(shape[:td], dtype=np.int64))
    I = int(np.prod(shape[td + 1 :], dtype=np.int64))
    return O, int(shape[td]), I


def _c(t, dtype=None):
    t = t.detach()
    if dtype is not None:
        t = t.to(dtype)
    return t.contiguous()


def _mask(m, shape):
    return m.expand(shape).to(torch.uint8).contiguous()


_ONE = None


def _int_one():
    return torch.ones(1, dtype=torch.int32)


def _coef(x, shape):
    """Return (tensor_or_None, scalar_value, dtype) for ``x * int_mask``."""
    y = x * _int_one()
    if not y.dtype.is_floating_point:
        y = y.to(torch.get_default_dtype())
    if y.numel() > 1:
        return y.expand(shape).contiguous(), 0.0, y.dtype
    return None, float(y.reshape(()).item()), y.dtype


def gae(gamma, lmbda, state_value, next_state_value, reward, done, terminated=None, *, time_dim=-2):
    """functional.py:121-182 -- returns (advantage, value_target)."""
    if terminated is None:
        terminated = done
    shape = next_state_value.shape
    O, T, I = _canon_dims(shape, time_dim)
    ts = next_state_value.dtype
    g_t, g_s, g_dt = _coef(gamma, shape)
    lg_t, lg_s, lg_dt = _coef(lmbda * gamma, shape)
    tg = torch.promote_types(g_dt, lg_dt)
    if g_t is not None:
        g_t = g_t.to(tg)
    if lg_t is not None:
        lg_t = lg_t.to(tg)
    if (g_t is None) != (lg_t is None):
        # one full tensor, one scalar: materialise the scalar one
        if g_t is None:
            g_t = torch.full(shape, g_s, dtype=tg)
        else:
            lg_t = torch.full(shape, lg_s, dtype=tg)
    r, v, nv = _c(reward, ts), _c(state_value, ts), _c(next_state_value, ts)
    d, tm = _mask(done, shape), _mask(terminated, shape)
    adv = torch.empty(shape, dtype=ts)
    vt = torch.empty(shape, dtype=ts)
    fn = getattr(lib(), "oracle_gae_" + _sfx[(ts, tg)])
    fn.restype = None
    fn(_ptr(r), _ptr(v), _ptr(nv), _ptr(d), _ptr(tm), _ptr(g_t), _ptr(lg_t),
       ctypes.c_double(g_s), ctypes.c_double(lg_s),
       ctypes.c_long(O), ctypes.c_long(T), ctypes.c_long(I), _ptr(adv), _ptr(vt))
    return adv, vt


def td_lambda(gamma, lmbda, next_state_value, reward, done, terminated=None, rolling_gamma=None, *, time_dim=-2):
    """functional.py:783-889 -- returns the TD(lambda) return."""
    if terminated is None:
        terminated = done
    shape = next_state_value.shape
    O, T, I = _canon_dims(shape, time_dim)
    ts = next_state_value.dtype

    def full_or_scalar(x):
        if isinstance(x, torch.Tensor) and x.shape == done.shape:
            return x.detach().contiguous(), 0.0, x.dtype
        # torch.full_like(next_state_value, x): value rounded to the storage dtype
        val = torch.full((1,), x.item() if isinstance(x, torch.Tensor) else x, dtype=ts)
        return None, float(val.item()), ts

    g_t, g_s, g_dt = full_or_scalar(gamma)
    l_t, l_s, l_dt = full_or_scalar(lmbda)
    single = g_t is None and l_t is None
    if rolling_gamma is None:
        rolling_gamma = True
    elif not rolling_gamma and single:
        raise RuntimeError("rolling_gamma=False is expected only with time-sensitive gamma or lambda values")
    tg = torch.promote_types(g_dt, l_dt)
    if g_t is None and l_t is not None:
        g_t = torch.full(shape, g_s, dtype=tg)
    if l_t is None and g_t is not None:
        l_t = torch.full(shape, l_s, dtype=tg)
    if g_t is not None:
        g_t, l_t = g_t.to(tg).contiguous(), l_t.to(tg).contiguous()
    r, nv = _c(reward, ts), _c(next_state_value, ts)
    d, tm = _mask(done, shape), _mask(terminated, shape)
    out = torch.empty(shape, dtype=ts)
    fn = getattr(lib(), "oracle_td_lambda_" + _sfx[(ts, tg)])
    fn.restype = None
    fn(_ptr(r), _ptr(nv), _ptr(d), _ptr(tm), _ptr(g_t), _ptr(l_t),
       ctypes.c_double(g_s), ctypes.c_double(l_s), ctypes.c_int(1 if rolling_gamma else 0),
       ctypes.c_long(O), ctypes.c_long(T), ctypes.c_long(I), _ptr(out))
    return out


def td1(gamma, next_state_value, reward, done, terminated=None, rolling_gamma=None, *, time_dim=-2):
    """functional.py:464-562 -- returns the TD(1) return (rolling and rolling_gamma=False loops)."""
    if terminated is None:
        terminated = done
    shape = next_state_value.shape
    O, T, I = _canon_dims(shape, time_dim)
    ts = next_state_value.dtype
    if isinstance(gamma, torch.Tensor) and gamma.shape == done.shape:
        g_t, g_s, tg = gamma.detach().contiguous(), 0.0, gamma.dtype
    else:  # torch.full_like(next_state_value, gamma)
        val = torch.full((1,), gamma.item() if isinstance(gamma, torch.Tensor) else gamma, dtype=ts)
        g_t, g_s, tg = None, float(val.item()), ts
    if rolling_gamma is None:
        rolling_gamma = True
    elif not rolling_gamma and g_t is None:
        raise RuntimeError("rolling_gamma=False is expected only with time-sensitive gamma values")
    r, nv = _c(reward, ts), _c(next_state_value, ts)
    d, tm = _mask(done, shape), _mask(terminated, shape)
    out = torch.empty(shape, dtype=ts)
    fn = getattr(lib(), "oracle_td1_" + _sfx[(ts, tg)])
    fn.restype = None
    fn(_ptr(r), _ptr(nv), _ptr(d), _ptr(tm), _ptr(g_t), ctypes.c_double(g_s), ctypes.c_int(1 if rolling_gamma else 0),
       ctypes.c_long(O), ctypes.c_long(T), ctypes.c_long(I), _ptr(out))
    return out


def td0(gamma, next_state_value, reward, terminated):
    """functional.py:418-456 -- reward + gamma * not_terminated * next_state_value, op for op in numpy
    (``gamma * int_mask`` first: a python-float gamma is rounded to the default dtype)."""
    nt = (~terminated).to(torch.int32)
    coef = gamma * nt
    if not coef.dtype.is_floating_point:
        coef = coef.to(torch.get_default_dtype())
    c = coef.numpy()
    nv, r = next_state_value.detach().numpy(), reward.detach().numpy()
    return torch.from_numpy(np.asarray(r + c * nv))


def reward2go(reward, done, gamma, *, time_dim=-2):
    """functional.py:1358-1432 -- discounted cumulative reward per trajectory; trailing dims after the time dim are
    independent rows.  Sequential double loop in the reward's dtype (the reference's own arithmetic goes through a
    cumsum of discounted rewards divided by the discounts: it agrees with this loop to rounding, not bit for bit)."""
    shape = reward.shape
    O, T, I = _canon_dims(shape, time_dim)
    nd = len(shape)
    td = (time_dim if time_dim >= 0 else nd + time_dim) if nd > 1 else 0
    r = reward.detach().movedim(td, -1).reshape(-1, T) if nd > 1 else reward.detach().reshape(1, T)
    d = done.movedim(td, -1).reshape(-1, T) if nd > 1 else done.reshape(1, T)
    out = torch.zeros_like(r)
    g = float(gamma)
    rn, dn, on = r.numpy(), d.numpy(), out.numpy()
    for row in range(rn.shape[0]):
        acc = rn.dtype.type(0)
        for t in range(T - 1, -1, -1):
            if dn[row, t]:
                acc = rn.dtype.type(0)
            acc = rn.dtype.type(rn[row, t] + rn.dtype.type(g) * acc)
            on[row, t] = acc
    if nd > 1:
        lead = [shape[k] for k in range(nd) if k != td]
        return out.reshape(*lead, T).movedim(-1, td)
    return out.reshape(shape)


def vtrace(gamma, log_pi, log_mu, state_value, next_state_value, reward, done, terminated=None,
           rho_thresh=1.0, c_thresh=1.0, *, time_dim=-2):
    """functional.py:1270-1350 -- returns (advantage, vs)."""
    if terminated is None:
        terminated = done
    shape = next_state_value.shape
    O, T, I = _canon_dims(shape, time_dim)
    ts = next_state_value.dtype
    g_t, g_s, tg = _coef(gamma, shape)
    tc = torch.promote_types(ts, tg)

    def thr(x):
        """(scalar, per-element tensor or None): a threshold tensor with more than one element broadcasts against the
        inputs after the reference's time transposition (functional.py:64-91, 1326-1330)."""
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(x)
        if x.numel() == 1:
            return float(x.reshape(()).item()), None
        nd = len(shape)
        td = time_dim if time_dim < 0 else time_dim - nd
        if tuple(x.shape) != tuple(shape) and td != -2 and nd >= 2:
            xtd = time_dim if time_dim < 0 else time_dim - x.ndim
            tshape = list(shape)
            tshape[td], tshape[-2] = tshape[-2], tshape[td]
            x = x.transpose(xtd, -2).expand(tshape).transpose(td, -2)
        return 0.0, _c(x.expand(shape), ts)

    lp, lm = _c(log_pi.expand(shape), ts), _c(log_mu.expand(shape), ts)
    r, v, nv = _c(reward, ts), _c(state_value, ts), _c(next_state_value, ts)
    d, tm = _mask(done, shape), _mask(terminated, shape)
    adv = torch.empty(shape, dtype=tc)
    vs = torch.empty(shape, dtype=tc)
    fn = getattr(lib(), "oracle_vtrace_" + _sfx[(ts, tg)])
    fn.restype = None
    rho_s, rho_t = thr(rho_thresh)
    c_s, c_t = thr(c_thresh)
    fn(_ptr(lp), _ptr(lm), _ptr(v), _ptr(nv), _ptr(r), _ptr(d), _ptr(tm), _ptr(g_t),
       ctypes.c_double(g_s), ctypes.c_double(rho_s), ctypes.c_double(c_s), _ptr(rho_t), _ptr(c_t),
       ctypes.c_long(O), ctypes.c_long(T), ctypes.c_long(I), _ptr(adv), _ptr(vs))
    return adv, vs


def gae_normalize_mt(gamma, lmbda, state_value, next_state_value, reward, done, terminated, eps, threads=None):
    """All-cores CPU baseline of the benchmark: fp32 GAE with scalar gamma / lmbda on [O, T, 1] inputs followed by the
    normalisation, env dimension split over OpenMP threads (oracle_gae_normalize_mt_f32).  Returns
    (normalised advantage, value_target, threads used)."""
    O, T, I = _canon_dims(next_state_value.shape, -2)
    assert I == 1 and next_state_value.dtype == torch.float32
    _, g_s, _ = _coef(gamma, next_state_value.shape)
    _, lg_s, _ = _coef(lmbda * gamma, next_state_value.shape)
    r, v, nv = _c(reward), _c(state_value), _c(next_state_value)
    d, tm = _mask(done, r.shape), _mask(terminated, r.shape)
    adv, vt = torch.empty_like(r), torch.empty_like(r)
    L = lib()
    if threads:
        import os
        os.environ["OMP_NUM_THREADS"] = str(threads)
    fn = L.oracle_gae_normalize_mt_f32
    fn.restype = ctypes.c_int
    used = fn(_ptr(r), _ptr(v), _ptr(nv), _ptr(d), _ptr(tm), ctypes.c_double(g_s), ctypes.c_double(lg_s),
              ctypes.c_long(O), ctypes.c_long(T), ctypes.c_double(eps), _ptr(adv), _ptr(vt), ctypes.c_void_p(0))
    return adv, vt, used


def normalize(x, eps, return_stats=False):
    """advantages.py:1459-1463 -- (x - mean) / std.clamp_min(eps), unbiased std over all elements."""
    xc = _c(x)
    out = torch.empty_like(xc)
    stats = torch.zeros(3, dtype=torch.float64)
    fn = getattr(lib(), "oracle_normalize_" + _sfx[(xc.dtype, xc.dtype)])
    fn.restype = None
    fn(_ptr(xc), ctypes.c_long(xc.numel()), ctypes.c_double(eps), _ptr(out), _ptr(stats))
    return (out, stats) if return_stats else out


def standardize(x, exclude_dims=(), eps=None):
    """torchrl/_utils.py:875-936 (_standardize with mean = std = None): per index of the excluded dims,
    mean and unbiased std over the remaining dims, then (x - mean) / std.clamp_min(eps).  numpy
    restatement: statistics in fp64 ({M, sum, sumsq} as the HIP path carries them), mean / std rounded
    to x's dtype, the scale in x's dtype.  torch's own mean / std reduce in the storage dtype with an
    internal order, so goldens agree to ~1e-6 relative (fp32), not bit for bit."""
    import numpy as np

    if eps is None:
        eps = 1e-6  # torch.finfo(torch.float).resolution
    a = x.detach().cpu().numpy()
    nd = a.ndim
    ex = sorted(d if d >= 0 else d + nd for d in exclude_dims)
    if len(ex) == nd:
        return x
    incl = tuple(d for d in range(nd) if d not in ex)
    a64 = a.astype(np.float64)
    m = 1
    for d in incl:
        m *= a.shape[d]
    s = a64.sum(axis=incl, keepdims=True)
    ss = (a64 * a64).sum(axis=incl, keepdims=True)
    mean = s / m
    with np.errstate(invalid="ignore", divide="ignore"):
        var = (ss - m * mean * mean) / (m - 1.0) if m > 1 else np.full_like(mean, np.nan)
    var = np.where(var < 0.0, 0.0, var)
    mean_s = mean.astype(a.dtype)
    std_s = np.sqrt(var).astype(a.dtype)
    eps_s = a.dtype.type(eps)
    std_s = np.where(std_s < eps_s, eps_s, std_s)  # NaN kept (comparison false)
    out = (a - mean_s) / std_s
    return torch.from_numpy(out.astype(a.dtype))
