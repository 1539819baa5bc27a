"""CPU: the oracle of the map's optimiser against brute force, and what gs_localization_amd.map_optimizer refuses before any GPU is touched."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gs_localization_amd import _lib, map_optimizer as MO
from oracle import map_optimizer_oracle as O


# ---- the oracle --------------------------------------------------------------------------------------------------------------------

def test_oracle_adamw_is_torchs():
    rng = np.random.default_rng(0)
    p = torch.tensor(rng.normal(size=37), dtype=torch.float64, requires_grad=True)
    opt = torch.optim.AdamW([p], lr=0.01, betas=(0.8, 0.95), eps=1e-9, weight_decay=0.1)
    q, m, v = p.detach().numpy().copy(), np.zeros(37), np.zeros(37)
    for t in range(1, 6):
        g = rng.normal(size=37)
        p.grad = torch.tensor(g)
        opt.step()
        q, m, v, _ = O.adamw(q, g, m, v, t, 0.01, (0.8, 0.95), 1e-9, 0.1)
    assert np.abs(q - p.detach().numpy()).max() < 1e-13


def test_oracle_norm_is_torchs():
    rng = np.random.default_rng(1)
    gs = [rng.normal(size=s) for s in (5, 17, 1)]
    ps = [torch.zeros(g.shape, dtype=torch.float64) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = torch.tensor(g)
    n = torch.nn.utils.clip_grad_norm_(ps, 0.7)
    got = O.norm(gs, 0.7)
    assert abs(got[0] - float(n)) < 1e-12 and abs(got[1] * gs[0][2] - float(ps[0].grad[2])) < 1e-12


def test_the_ratio_bound_holds_and_is_reached():
    """|m| / sqrt(v) <= span for any gradients; the extremal ones g_k ~ (b1 / b2)^k reach it."""
    rng = np.random.default_rng(2)
    for b1, b2 in ((0.9, 0.999), (0.5, 0.9), (0.0, 0.99)):
        m = v = np.zeros(1000)
        for k in range(200):
            g = rng.standard_cauchy(1000)
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            assert (np.abs(m) <= O.span(b1, b2) * np.sqrt(v) * (1 + 1e-12)).all()
        m = v = 0.0
        for k in range(3000, -1, -1):          # oldest first
            g = (b1 / b2) ** k
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        assert 0.999 < m / math.sqrt(v) / O.span(b1, b2) <= 1 + 1e-12


def test_grid_is_the_upper_bits_of_a_float():
    bits = np.arange(0, 255 << 4, dtype=np.uint32) << 19
    x = bits.view(np.float32).astype(np.float64)
    assert (O.grid_value(bits >> 19) == x).all()
    assert (O.grid_place(x) == (bits >> 19)).all()
    y = (bits + np.uint32(1 << 18)).view(np.float32).astype(np.float64)          # half-way between two
    assert (O.grid_place(y) == (bits >> 19) + 0.5).all()


def test_random_bits_are_spread():
    """Mean and variance of both parts over 2^20 elements, neighbours uncorrelated: five standard errors."""
    n = 1 << 20
    for t in (1, 2, 1000):
        du, dr = O.dither(np.arange(n), 7, 0, t)
        for x, top in ((du, 1 << 19), (dr, 1 << 13)):
            x = (x + 0.5) / top - 0.5
            assert abs(x.mean()) < 5 * math.sqrt(1 / 12 / n)
            assert abs(x.var() - 1 / 12) < 5 * math.sqrt(1 / 180 / n)
            for lag in (1, 2, 3, 4, 64, 256):
                assert abs((x[lag:] * x[:-lag]).mean()) < 5 / 12 / math.sqrt(n - lag)
        assert abs(((du / 2.0 ** 19 - 0.5) * (dr / 8192.0 - 0.5)).mean()) < 5 / 12 / math.sqrt(n)


def test_oracle_evict_by_brute_force():
    rng = np.random.default_rng(3)
    for _ in range(50):
        P = int(rng.integers(1, 12))
        s = rng.choice([0.0, -0.0, 1.0, 2.0, np.nan, -np.inf, np.inf], P).astype(np.float32)
        keep = int(rng.integers(0, P + 1))
        recent = int(rng.integers(0, keep + 1))
        alive = list(range(P))
        key = lambda i: (-math.inf if math.isnan(s[i]) else s[i], -i)                         # noqa: E731
        while len(alive) > keep:
            alive.remove(min((i for i in alive if i < P - recent), key=key))
        kept, _ = O.evict(s, keep, recent)
        assert kept.tolist() == alive


# ---- refusals ----------------------------------------------------------------------------------------------------------------------

def test_no_cpu_path():
    z, f = torch.zeros(4), torch.zeros(2)
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.grad_norm([z])
    clock = torch.zeros(4, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.adamw_step([z], [z], [z], [z], [clock], lr=0.1)
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.adamw_step_8bit([z], [z], [z.byte()], [z.char()], [z[:1].byte()], [clock], lr=0.1)
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.moments_8bit([z.byte()], [z.char()], [z[:1].byte()])
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.evict_rows(z, 2, [z])
    p = torch.nn.Parameter(z)
    p.grad = z.clone()
    with pytest.raises(RuntimeError, match="HIP tensors"):
        MO.AdamW([p]).step()


def test_python_refusals():
    z = torch.zeros(4)
    with pytest.raises(ValueError, match="no gradients"):
        MO.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        MO.grad_norm([z], -1.0)
    with pytest.raises(ValueError, match="different lengths"):
        MO.adamw_step([z], [], [], [], [], lr=0.1)
    with pytest.raises(ValueError, match="lr"):
        MO.adamw_step([z], [z], [z], [z], [z], lr=[0.1, 0.2])
    for keep, recent in ((5, 0), (-1, 0), (2, 3), (2, -1)):
        with pytest.raises(ValueError, match="recent <= keep <= P"):
            MO.evict_rows(z, keep, [], recent=recent)
    with pytest.raises(ValueError, match="scores"):
        MO.evict_rows(z.double(), 2, [])
    with pytest.raises(ValueError, match="weights"):
        MO.evict_rows(z, 2, [], weights=torch.zeros(2, 3))
    p = torch.nn.Parameter(z)
    for kw, what in ((dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "beta"), (dict(eps=-1.0), "eps"), (dict(weight_decay=-1.0), "weight_decay"),
                     (dict(state_bits=16), "state_bits"), (dict(state_bits=8, betas=(0.99, 0.9)), "beta1"), (dict(max_norm=-1.0), "max_norm")):
        with pytest.raises(ValueError, match=what):
            MO.AdamW([p], **kw)


def _adamw(lib, **kw):
    """gsr_adamw_step on made-up addresses: every refusal below comes before a pointer is used."""
    base = dict(param=0x1000, grad=0x20000, state0=0x30000, state1=0x40000, window=0x50000, clock=0x60000, lr_device=0, lr=0.1, decay=0.0, n=64, pt=0, gt=0)
    tensors = kw.pop("tensors", [{}])
    buf = bytearray(MO._OPT.size * len(tensors))
    for i, t in enumerate(tensors):
        d = dict(base, **t)
        MO._OPT.pack_into(buf, i * MO._OPT.size, *d.values())
    a = dict(n_tensors=len(tensors), state_bits=32, tensors=MO._address(buf), beta1=0.9, beta2=0.999, eps=1e-8, clip=None, seed=0, stream=None)
    a.update(kw)
    return lib.gsr_adamw_step(C.byref(_lib.AdamwArgs(*a.values()))), lib.gsr_last_error().decode()


@pytest.mark.parametrize("kw, what", [
    (dict(state_bits=16), "32 or 8"), (dict(beta1=1.0), "beta"), (dict(beta2=float("nan")), "beta"), (dict(eps=-1e-8), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(state_bits=8, beta1=0.99, beta2=0.9), "beta1"), (dict(n_tensors=-1), "NULL"), (dict(tensors=[dict(n=-1)]), "size"),
    (dict(tensors=[dict(n=1 << 41)]), "size"), (dict(tensors=[dict(pt=3)]), "type"), (dict(tensors=[dict(gt=-1)]), "type"), (dict(tensors=[dict(param=0)]), "NULL"),
    (dict(tensors=[dict(clock=0)]), "NULL"), (dict(state_bits=8, tensors=[dict(window=0)]), "NULL"), (dict(tensors=[dict(param=0x1002)]), "aligned"),
    (dict(tensors=[dict(grad=0x20001, gt=1)]), "aligned"), (dict(tensors=[dict(state1=0x40002)]), "aligned"), (dict(tensors=[dict(clock=0x60004)]), "aligned"),
    (dict(tensors=[{}, {}]), "overlaps"),                                        # the same tensor twice
    (dict(tensors=[dict(grad=0x10fc)]), "overlaps"),                             # the gradient's first element is the parameter's last
    (dict(tensors=[dict(state1=0x30080)]), "overlaps"), (dict(tensors=[dict(clock=0x300f8)]), "overlaps"), (dict(clip=0x60010), "overlaps"),
    (dict(tensors=[{}, dict(param=0x101000, state0=0x130000, state1=0x140000)]), "overlaps"),       # two tensors, one clock
])
def test_adamw_c_refusals(kw, what):
    rc, said = _adamw(_lib.load(), **kw)
    assert rc == -1 and what in said, (rc, said)


def test_shared_gradient_is_only_read():
    """two parameters may share a gradient (and a rate): only what is written must be apart (this call gets as far as looking for its device)"""
    rc, said = _adamw(_lib.load(), tensors=[dict(lr_device=0x70000), dict(lr_device=0x70000, param=0x101000, state0=0x130000, state1=0x140000, clock=0x160000)])
    assert rc == -4, (rc, said)


def test_norm_and_moments_c_refusals():
    lib = _lib.load()
    one, size, t = (C.c_void_p * 1)(0x1000), (C.c_longlong * 1)(4), (C.c_int * 1)(0)
    fn, call = _lib.fixed_buffer_fn(), lambda g, s, ty, mx=1.0, out=0x2000: lib.gsr_grad_norm(1, g, s, ty, mx, out, fn, None, None)       # noqa: E731
    assert call(one, (C.c_longlong * 1)(-1), t) == -1 and call(one, size, (C.c_int * 1)(3)) == -1 and call(one, size, t, -1.0) == -1
    assert call(one, size, t, float("nan")) == -1 and call(one, size, t, 1.0, None) == -1 and call((C.c_void_p * 1)(0x1002), size, t) == -1
    assert lib.gsr_adamw_moments(-1, None, 0.9, 0.999, 0, None) == -1 and lib.gsr_adamw_moments(0, None, 0.9, 0.999, 7, None) == -1
    assert lib.gsr_adamw_moments(0, None, 0.9, 0.8, 0, None) == -1 and lib.gsr_adamw_moments(0, None, 0.9, 0.999, 0, None) == 0
    buf = bytearray(MO._MOMENT.pack(0x1000, 0x2000, 0x3000, 0x4000, 0x4010, 64))
    assert lib.gsr_adamw_moments(1, MO._address(buf), 0.9, 0.999, 0, None) == -1 and b"overlaps" in lib.gsr_last_error()
    assert lib.gsr_adamw_step(None) == -1 and lib.gsr_evict_rows(None) == -1


def test_evict_c_refusals():
    lib = _lib.load()

    def call(row=(0x10000, 0x20000, 0, 0, 12), **kw):
        buf = bytearray(MO._ROW.pack(*row))
        a = dict(P=8, n_views=0, keep=4, recent=0, scores=0x1000, weights=None, decay=1.0, kept=0x2000, scores_out=0x3000, n_tensors=1,
                 tensors=MO._address(buf), workspace=_lib.fixed_buffer_fn(), ctx=None, stream=None)
        a.update(kw)
        return lib.gsr_evict_rows(C.byref(_lib.EvictArgs(*a.values()))), lib.gsr_last_error().decode()
    for kw, what in ((dict(P=-1, keep=0), "negative"), (dict(keep=9), "recent <= keep <= P"), (dict(recent=5), "recent <= keep <= P"), (dict(n_views=-1), "negative"),
                     (dict(n_views=1), "NULL"), (dict(scores=None), "NULL"), (dict(kept=None), "NULL"), (dict(tensors=None), "NULL"),
                     (dict(row=(0, 0x20000, 0, 0, 12)), "NULL"), (dict(row=(0x10000, 0x20000, 0x30000, 0, 12)), "NULL"), (dict(row=(0x10000, 0x20000, 0, 0, -1)), "row size"), (dict(row=(0x10000, 0x20000, 0, 0, 1 << 31)), "row size"), (dict(P=1 << 30, row=(0x10000, 0x20000, 0, 0, 1 << 10)), "row size"),
                     (dict(row=(0x10000, 0x10020, 0, 0, 12)), "overlaps"), (dict(scores_out=0x2010), "overlaps"), (dict(kept=0x1008), "overlaps")):
        rc, said = call(**kw)
        assert rc == -1 and what in said, (kw, rc, said)
    assert call(keep=0, scores=None)[0] == 0
