"""-m gpu : gs_localization_amd.map_optimizer where values, options and calls meet that tests/test_gpu_map_optimizer.py takes apart: roots that
overflow, betas that change, several groups, layouts that torch has not resolved yet, codes that an eviction raises."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

from oracle import map_optimizer_oracle as O
from tests.test_gpu_map_optimizer import DEV, E, HALF, MO, SIZES, Guarded, bound32, check8, clocks, n64, random_codes, small_map

pytestmark = pytest.mark.gpu


def codes(n):
    return torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros((n + 255) // 256, dtype=torch.uint8, device=DEV)


# ---- 8-bit moments: values at the ends ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("beside", [0.0, 1e-5, 1.0])
def test_overflowed_root_keeps_the_momentums_sign(dtype, shift, beside):
    """One gradient per block of 256 whose square is no float: its root's code is 255 and |exp_avg| is more than the span times what that code
    stands for (1e19 and more against 2 roots of the largest neighbour), so its ratio is 127 with the gradient's sign.  The
    neighbours round as if it were not there, and the next step does not go up the gradient."""
    bad = [3e38, -3e38, 1e30, -1e30, 1e20, -1e20, float("inf"), -float("inf"), 2e38]
    n = 2048 + 100          # eight blocks of whole waves, one of a partial wave
    gen = torch.Generator(device=DEV).manual_seed(50)
    g = torch.randn(n, generator=gen, device=DEV) * beside
    at = torch.arange(len(bad), device=DEV) * 256 + 17
    out = []
    for values in (bad, [0.0] * len(bad)):
        gg = g.clone()
        gg[at] = torch.tensor(values, device=DEV)
        p, gg = Guarded(torch.ones(n, device=DEV), shift), Guarded(gg.to(dtype), shift)
        rms, ratio, window = (Guarded(x, shift) for x in codes(n))
        ck = clocks(1, 0, (0.9, 0.999))
        step = lambda: MO().adamw_step_8bit([p.t], [gg.t], [rms.t], [ratio.t], [window.t], ck, lr=0.1, seed=3)          # noqa: E731
        step()
        out.append([x.t.clone() for x in (p, rms, ratio, window)])
    (p1, rms1, ratio1, window1), (p0, rms0, ratio0, window0) = out
    sign = torch.tensor([math.copysign(1.0, x) for x in bad], device=DEV)
    assert ratio1[at].tolist() == (127 * sign).tolist()
    assert (rms1[at] == 255).all()
    finite = torch.tensor([math.isfinite(x) for x in bad], device=DEV)
    assert (p1[at][finite] == 1.0).all() and p1[at][~finite].isnan().all()          # (finite / infinite is nothing, infinite / infinite is NaN)
    others = torch.ones(n, dtype=torch.bool, device=DEV)
    others[at] = False
    for x, y in ((p1, p0), (rms1, rms0), (ratio1, ratio0)):
        assert torch.equal(x[others], y[others])
    assert torch.equal(window1, window0)
    q = torch.ones(n, device=DEV)
    MO().adamw_step_8bit([q], [torch.zeros(n, device=DEV)], [rms1], [ratio1], [window1], clocks(1, 1, (0.9, 0.999)), lr=0.1, seed=3)
    assert ((q[at] - 1.0) * sign <= 0).all()


@pytest.mark.parametrize("eps", [1e30, 2.0 ** 100, 1e35, 2.0 ** 127, 3e38, math.inf])
def test_first_8_bit_step_with_a_large_eps(eps):
    """The same bits as with 32-bit moments (nothing has been rounded to a byte yet), whatever eps is added to the root."""
    n = 4096
    gen = torch.Generator(device=DEV).manual_seed(51)
    g = torch.randn(n, generator=gen, device=DEV) * torch.exp2(torch.randint(-55, 60, (n,), generator=gen, device=DEV).float())
    p = torch.randn(n, generator=gen, device=DEV)
    q = p.clone()
    a = codes(n)
    MO().adamw_step([p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)], clocks(1, 0, (0.9, 0.999)), lr=1e25, eps=eps)
    MO().adamw_step_8bit([q], [g], [a[0]], [a[1]], [a[2]], clocks(1, 0, (0.9, 0.999)), lr=1e25, eps=eps)
    assert bool(p.isfinite().all()) and torch.equal(p.view(torch.int32), q.view(torch.int32))


# ---- 8-bit moments: which random bits ------------------------------------------------------------------------------------------------

class Held:
    def __init__(self, t):
        self.t = t


def test_groups_round_by_bits_of_their_own():
    """A parameter rounds by the random bits of its place among all of the optimiser's parameters: equal tensors in groups of other options (another
    call each) get other bits, and one that has no gradient this time leaves the others'."""
    n = 6000
    gen = torch.Generator(device=DEV).manual_seed(52)
    g = torch.randn(n, generator=gen, device=DEV) * 1e-3
    eps = [1e-15, 1e-8, 1e-15, 1e-15]
    ps = [torch.nn.Parameter(torch.ones(n, device=DEV)) for _ in eps]
    opt = MO().AdamW([{"params": [p], "eps": e} for p, e in zip(ps, eps)], lr=0.01, state_bits=8, seed=11)
    for t, stepped in ((1, (0, 1, 2, 3)), (2, (0, 1, 3)), (3, (2, 3))):
        for k, p in enumerate(ps):
            p.grad = g.clone() if k in stepped else None
        before = {}
        for k in stepped:
            st = opt.state[ps[k]] if ps[k] in opt.state else dict(zip(("rms", "ratio", "window"), codes(n)), step=clocks(1, 0, (0.9, 0.999))[0])
            before[k] = ([x.detach().clone() for x in (ps[k], g, st["rms"], st["ratio"], st["window"])], int(st["step"][2]) + 1)
        opt.step()
        for k in stepped:
            st = opt.state[ps[k]]
            after = [Held(x) for x in (ps[k], g, st["rms"], st["ratio"], st["window"])]
            check8(before[k][0], after, k, before[k][1], 0.01, (0.9, 0.999), eps[k], 0.0, 1.0, 11, torch.float32)
        if t == 1:
            a, b = (opt.state[p]["rms"] for p in ps[:2])
            # from the same roots two independent roundings differ in 2 f (1 - f) of the elements, f uniform: a third
            assert 0.25 < float((a != b).float().mean()) < 0.42


# ---- betas that change -----------------------------------------------------------------------------------------------------------------

def check8_from(before, after, t, lr, betas, was, eps, place, seed):
    """One 8-bit step whose ratios were stored with the betas `was`: the parameter by the roundings of a step, the moments within a step of their codes."""
    p, g, rms, ratio, window = before
    p1, m1, u1, at, dr, scale = O.adamw8(n64(p), n64(g), rms.cpu().numpy(), ratio.cpu().numpy(), window.cpu().numpy(), t, lr, betas, eps, 0.0, 1.0, seed, place, was)
    assert (np.abs(n64(after[0]) - p1) <= bound32(p1, m1, None, scale * 1.2, lr, 0.0, torch.float32)).all()
    codes_, window_ = after[2].cpu().numpy().reshape(-1), after[4].cpu().numpy()
    u = O.decode(codes_, window_)
    low = O.decode(np.ones_like(codes_), window_)
    assert (np.abs(u - u1) <= np.maximum(u1 / 16 * (1 + 64 * E), low)).all() and ((u > 0) == (u1 > 0)).all()
    unit = O.span(*betas) / 127 * u
    m = n64(after[3]) * unit          # (a floor of a value with random bits added: under one step off; past 127 steps, 127)
    size = np.abs(n64(ratio)) / 127 * O.span(*was) * O.decode(rms.cpu().numpy(), window.cpu().numpy()) + np.abs(n64(g))
    assert (np.abs(m - np.clip(m1, -127 * unit, 127 * unit)) <= unit * (1 + 1e-6) + 20 * E * size).all()


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.8, 0.95), (0.95, 0.999), (0.0, 0.5), (0.5, 0.3)])
@pytest.mark.parametrize("was", [None, (0.95, 0.999), (0.85, 0.999), (0.3, 0.9)])
def test_8_bit_step_of_other_betas(betas, was):
    n = 5001
    gen = torch.Generator(device=DEV).manual_seed(53)
    rms, ratio, window = (x.t for x in random_codes(n, gen, 0, 95, 105))
    p, g = torch.randn(n, generator=gen, device=DEV), torch.randn(n, generator=gen, device=DEV) * 1e-3 * (torch.rand(n, generator=gen, device=DEV) < 0.7)
    (avg,), (root,) = MO().moments_8bit([rms], [ratio], [window], betas=was or betas)
    m = n64(ratio) / 127 * O.span(*(was or betas)) * n64(root)
    assert (np.abs(n64(avg) - m) <= 3 * E * np.abs(m)).all()
    ck = clocks(1, 4, betas)
    first = was or betas
    for t in (5, 6):
        before = [x.clone() for x in (p, g, rms, ratio, window)]
        MO().adamw_step_8bit([p], [g], [rms], [ratio], [window], ck, lr=0.01, betas=betas, eps=1e-12, seed=5, **({} if first == betas else dict(state_betas=first)))
        check8_from(before, (p, g, rms, ratio, window), t, 0.01, betas, first, 1e-12, 0, 5)
        first = betas
    assert abs(float(ck[0][0]) - betas[0] ** 6) < 1e-15 and float(ck[0][2]) == 6


def test_state_betas_are_checked():
    p, a = torch.ones(4, device=DEV), codes(4)
    ck = clocks(1, 0, (0.9, 0.999))
    for bad in ((0.99, 0.9), (1.0, 0.999), (-0.1, 0.9), (0.9, 1.0), (float("nan"), 0.9)):
        with pytest.raises(RuntimeError, match="beta"):
            MO().adamw_step_8bit([p], [p.clone()], [a[0]], [a[1]], [a[2]], ck, lr=0.1, state_betas=bad)
    with pytest.raises(ValueError, match="state_betas"):
        MO().adamw_step_8bit([p], [p.clone()], [a[0]], [a[1]], [a[2]], ck, lr=0.1, state_betas=[(0.9, 0.999)] * 2)
    assert float(ck[0][2]) == 0.0 and bool((p == 1).all())


def cycled(opt, steps):
    return torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=[0.01 * (i + 1) for i in range(len(opt.param_groups))], total_steps=steps)


def test_scheduler_that_cycles_beta1():
    """torch.optim.lr_scheduler.OneCycleLR sets beta1 anew for every step (0.95 to 0.85 and back): as torch.optim.Adam, whose bias corrections are 1 - beta^t of
    the betas of the step.  An update's size is under 4 lr: with weights of at most 0.15 the momentum of t gradients is at most 0.15 t of their root mean
    square (Cauchy-Schwarz), over 1 - 0.95^t that is 3.8 at t = 10.  Its roundings are 40 e of it a step, fed on over 1 / (1 - beta1) <= 20 steps."""
    gen = torch.Generator(device=DEV).manual_seed(54)
    ps, opt = small_map(500, gen, 32)
    qs = [torch.nn.Parameter(p.detach().double().cpu()) for p in ps.values()]
    ref = torch.optim.Adam([{"params": [q], "lr": 0.01 * (i + 1)} for i, q in enumerate(qs)], lr=0.0, eps=1e-15)
    sa, sb = cycled(opt, 12), cycled(ref, 12)
    for t in range(1, 11):
        for p, q in zip(ps.values(), qs):
            p.grad = torch.randn(p.shape, generator=gen, device=DEV)
            q.grad = p.grad.double().cpu()
        opt.step(); ref.step()
        b = opt.param_groups[0]["betas"]
        assert b[0] != 0.9
        for p in ps.values():
            c = opt.state[p]["step"].tolist()
            assert c[0] == pytest.approx(b[0] ** t, rel=1e-14) and c[1] == pytest.approx(b[1] ** t, rel=1e-14) and c[2:] == [t, 0.0]
        sa.step(); sb.step()
    for i, (p, q) in enumerate(zip(ps.values(), qs)):
        assert (np.abs(n64(p) - n64(q)) <= E * (10 * 40 * 4 * 20 * 0.01 * (i + 1) + 30 * np.abs(n64(q)))).all()


def step_checked8(opt, gen, missing=()):
    """One step of an 8-bit optimiser with new gradients, each parameter against the oracle that knows the betas its ratios were stored with."""
    params = [p for g in opt.param_groups for p in g["params"]]
    before = []
    for p in params:
        st = opt.state.get(p) or {}
        fresh = codes(p.numel())
        before.append([p.detach().clone()] + [st[k].clone() if k in st else z for k, z in zip(("rms", "ratio", "window"), fresh)] + [float(st["step"][2]) if st else 0.0])
        p.grad = None if id(p) in missing else torch.randn(p.shape, generator=gen, device=DEV) * 1e-2
    opt.step()
    place = 0
    for g in opt.param_groups:
        for p in g["params"]:
            b, st = before[place], opt.state.get(p)
            if p.grad is not None:
                t = int(b[4]) + 1
                check8_from((b[0], p.grad, b[1], b[2], b[3]), (p, p.grad, st["rms"], st["ratio"], st["window"]), t, g["lr"], g["betas"], p.was if t > 1 else g["betas"], g["eps"], place, opt.seed)
                assert st["step"].tolist()[0] == pytest.approx(g["betas"][0] ** t, rel=1e-14)
                p.was = g["betas"]
            place += 1


def test_8_bit_optimizer_under_cycled_betas():
    """... through steps that leave a parameter out (its ratios keep the betas they were stored with), an eviction, copies, pickles and a state dict"""
    gen = torch.Generator(device=DEV).manual_seed(55)
    ps, opt = small_map(300, gen, 8, seed=9)
    sched = cycled(opt, 40)
    left_out = ps["opacity"]
    for t in range(1, 6):
        step_checked8(opt, gen, (id(left_out),) if t in (2, 3) else ())
        sched.step()

    def follow(other, params):
        for p, q in zip([p for g in opt.param_groups for p in g["params"]], params):
            q.was = p.was
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        follow(other, [q for g in other.param_groups for q in g["params"]])
        step_checked8(other, gen)
    saved = opt.state_dict()
    saved = dict(saved, state={i: {k: v.cpu().clone() if torch.is_tensor(v) else v for k, v in s.items()} for i, s in saved["state"].items()})
    qs, other = small_map(300, gen, 8, seed=9)
    with torch.no_grad():
        for p, q in zip(ps.values(), qs.values()):
            q.copy_(p)
    other.load_state_dict(saved)
    follow(other, qs.values())
    for g in other.param_groups:
        g["betas"] = (0.7, 0.99)
    step_checked8(other, gen)
    was = [p.was for g in opt.param_groups for p in g["params"]]
    opt.evict(torch.rand(300, generator=gen, device=DEV), 200)
    for p, w in zip((p for g in opt.param_groups for p in g["params"]), was):
        p.was = w
    sched.step()
    step_checked8(opt, gen)


def test_changed_betas_are_not_captured_with_8_bits():
    """a replay would decode with the betas from before again and again"""
    p = torch.nn.Parameter(torch.ones(500, device=DEV))
    p.grad = torch.ones_like(p)
    opt = MO().AdamW([p], lr=0.1, state_bits=8)
    opt.step()
    opt.param_groups[0]["betas"] = (0.8, 0.99)
    before = [x.clone() for x in (p.detach(), *(opt.state[p][k] for k in ("rms", "ratio", "window", "step")))]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    for x, y in zip(before, (p.detach(), *(opt.state[p][k] for k in ("rms", "ratio", "window", "step")))):
        assert torch.equal(x, y)
    opt.step()          # eagerly, and from then on captured
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    other = copy.deepcopy(opt)
    q = other.param_groups[0]["params"][0]
    for _ in range(3):
        graph.replay()
        q.grad = torch.ones_like(q)
        other.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and torch.equal(opt.state[p]["ratio"], other.state[q]["ratio"])


def test_changed_betas_captured_with_32_bits():
    """every replay forms its corrections from the count and the betas of the capture, as an eager step that follows one with the same betas: the
    powers agree to a few 2^-53, the parameters to the roundings of four steps (40 e of an update of the rate's size each)"""
    p = torch.nn.Parameter(torch.linspace(-1, 1, 500, device=DEV))
    p.grad = torch.linspace(-2, 1, 500, device=DEV)
    opt = MO().AdamW([p], lr=0.1)
    opt.step()
    opt.param_groups[0]["betas"] = (0.8, 0.99)
    torch.cuda.synchronize()
    other = copy.deepcopy(opt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    q = other.param_groups[0]["params"][0]
    q.grad = p.grad.clone()
    for t in range(2, 6):
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        a, b = opt.state[p]["step"].tolist(), other.state[q]["step"].tolist()
        assert a[2:] == b[2:] == [t, 0.0] and a[:2] == pytest.approx([0.8 ** t, 0.99 ** t], rel=1e-14) and b[:2] == pytest.approx(a[:2], rel=1e-14)
        assert float((p - q).detach().abs().max()) <= E * (4 * 40 * 0.2 + 4 * 2)


# ---- refused as a whole ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("what", ["type", "betas", "overlap", "size"])
def test_a_refused_step_has_stepped_nothing(bits, what):
    gen = torch.Generator(device=DEV).manual_seed(56)
    ps = [torch.nn.Parameter(torch.randn(500, generator=gen, device=DEV)) for _ in range(3)]
    opt = MO().AdamW([{"params": ps[:1]}, {"params": ps[1:2], "eps": 1e-3}, {"params": ps[2:], "eps": 1e-4}], lr=0.1, state_bits=bits, max_norm=1.0)
    for p in ps:
        p.grad = torch.randn(500, generator=gen, device=DEV)
    opt.step()
    st, k = opt.state[ps[1]], "exp_avg" if bits == 32 else "ratio"
    good, betas = dict(st), opt.param_groups[1]["betas"]
    if what == "type":
        st[k] = st[k].bfloat16()
    elif what == "betas":
        opt.param_groups[1]["betas"] = (1.0, 0.999)
    elif what == "overlap":
        st["step"] = ps[1].detach()[2:10].view(torch.float64)          # (its own, and yet in the parameter)
    else:
        st[k] = st[k][:400]
    watched = [x for p in ps for x in (p.detach(), *(y for y in opt.state[p].values() if torch.is_tensor(y)))]
    before = [x.clone() for x in watched]
    with pytest.raises((RuntimeError, TypeError, ValueError)):
        opt.step()
    torch.cuda.synchronize()
    for x, y in zip(watched, before):
        assert torch.equal(x, y)
    opt.param_groups[1]["betas"] = betas
    opt.state[ps[1]] = good
    opt.step()
    assert [float(opt.state[p]["step"][2]) for p in ps] == [2.0] * 3


# ---- layouts that torch has not resolved -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("P", [1, 3000])
def test_lazy_conjugates_and_negatives(P):
    """conj() and the imaginary part of a conjugate are marks on the same memory until something resolves them; one row of the latter is contiguous"""
    gen = torch.Generator(device=DEV).manual_seed(57)
    z = torch.randn(P, 2, generator=gen, device=DEV, dtype=torch.complex64)
    neg = z.conj()[:, :1].imag
    assert z.conj().is_conj() and z.conj().is_contiguous() and neg.is_neg()
    s = torch.rand(P, generator=gen, device=DEV)
    marked = torch.complex(s, -s).conj().imag
    keep = (P + 2) // 3
    kept, scores, rows, _ = MO().evict_rows(marked, keep, [z.conj(), neg, neg.t().contiguous().t()], weights=marked)
    want, ws = O.evict(s.cpu().numpy(), keep, 0, s.cpu().numpy()[None])
    assert np.array_equal(kept.cpu().numpy(), want) and np.array_equal(scores.cpu().numpy(), ws)
    assert torch.equal(rows[0], z.conj().resolve_conj()[kept]) and torch.equal(rows[1], -z[:, :1].imag[kept]) and torch.equal(rows[2], rows[1])
    out = []
    for grad in (s, marked):
        p, m, v = torch.ones(P, device=DEV), torch.zeros(P, device=DEV), torch.zeros(P, device=DEV)
        MO().adamw_step([p], [grad], [m], [v], clocks(1, 0, (0.9, 0.999)), lr=0.1)
        out.append((p, m, v, MO().grad_norm([grad], 1.0)))
    for x, y in zip(*out):
        assert torch.equal(x, y)
    if P == 1:
        m, v, ck = torch.zeros(P, device=DEV), torch.zeros(P, device=DEV), clocks(1, 0, (0.9, 0.999))
        with pytest.raises(ValueError, match="negative"):
            MO().adamw_step([marked], [s], [m], [v], ck, lr=0.1)
        assert float(ck[0][2]) == 0.0 and not bool(m.any())


# ---- codes that an eviction raises -------------------------------------------------------------------------------------------------------

def test_step_after_an_eviction_that_raises_roots():
    """Rows of roots 2^-30 of their new neighbours': a code becomes its new window's lowest, the ratio stays as it was.  What the bytes stand for is then
    exp_avg = ratio x span / 127 x the raised root, and the next update is the one that the row would have got without the eviction
    (its ratio's; never more than the span allows): here by a gradient of zero, to the roundings of two steps and eps."""
    P = 1024
    gen = torch.Generator(device=DEV).manual_seed(58)
    small = torch.arange(P, device=DEV) < 256
    p = torch.nn.Parameter(torch.zeros(P, 1, device=DEV))
    opt = MO().AdamW([p], lr=0.1, eps=1e-30, state_bits=8, seed=2)
    for _ in range(3):
        p.grad = torch.randn(P, 1, generator=gen, device=DEV).abs() + 0.5
        p.grad[small] *= 2.0 ** -30
        opt.step()
    whole = copy.deepcopy(opt)
    (w,) = whole.param_groups[0]["params"]
    kept, _, _ = opt.evict(torch.arange(P, device=DEV).float(), 824)
    assert kept[0] == 200
    (q,) = opt.param_groups[0]["params"]
    raised = small[kept]
    a, b = opt.state[q], whole.state[w]
    assert torch.equal(a["ratio"], b["ratio"][kept]) and bool((a["rms"][raised] == 1).all())
    (m,), (u,) = MO().moments_8bit([a["rms"]], [a["ratio"]], [a["window"]])
    (m0,), (u0,) = MO().moments_8bit([b["rms"]], [b["ratio"]], [b["window"]])
    assert bool((u[raised] > 1000 * u0[kept][raised]).all()) and torch.equal(u[~raised], u0[kept][~raised])
    # the same ratio: m / u is the same in 32 bits but for two roundings each
    assert float(((m / u) / (m0 / u0)[kept] - 1).abs().max()) <= 8 * E
    q0, w0 = q.detach().clone(), w.detach().clone()
    q.grad, w.grad = torch.zeros_like(q), torch.zeros_like(w)
    opt.step(); whole.step()
    x, y = n64(q.detach() - q0), n64(w.detach() - w0)[kept.cpu().numpy()]
    assert (np.abs(x - y) <= 60 * E * np.abs(y) + 4 * E * np.abs(n64(q0))).all()


# ---- what the calls leave alone, and the types they give ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
def test_grad_norm_writes_nothing(dtype, shift):
    gen = torch.Generator(device=DEV).manual_seed(59)
    gs = [Guarded((torch.randn(n, generator=gen, device=DEV) * 3).to(dtype), shift) for n in SIZES]
    before = [g.t.clone() for g in gs]
    for k in (1, len(gs)):
        MO().grad_norm([g.t for g in gs[:k]], 1.0)
    for g, b in zip(gs, before):
        assert torch.equal(g.t, b)
        g.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1])
def test_moments_of_each_type(dtype, shift):
    """The values that the codes stand for, computed in 32 bits (the unit's rounding and two products: 3 e) and rounded once: the roots' five bits are exact
    in every type that has their exponents (float16: in windows 112 and 113, 2^-15 to 4, where its spacing is 2^-24 or finer than five bits)."""
    gen = torch.Generator(device=DEV).manual_seed(60)
    low, high = (112, 114) if dtype is torch.float16 else (60, 120)
    ts = [random_codes(n, gen, shift, low, high) for n in SIZES]
    before = [[x.t.clone() for x in q] for q in ts]
    avg, root = MO().moments_8bit([q[0].t for q in ts], [q[1].t for q in ts], [q[2].t for q in ts], dtype=dtype)
    for q, b, a, r in zip(ts, before, avg, root):
        u = O.decode(q[0].t.cpu().numpy(), q[2].t.cpu().numpy())
        m = n64(q[1].t) / 127 * O.span(0.9, 0.999) * u
        assert a.dtype == r.dtype == dtype and a.shape == r.shape == q[0].t.shape
        assert (n64(r) == u).all()
        assert (np.abs(n64(a) - m) <= (3 * E + HALF[dtype] * (1 + 4 * E)) * np.abs(m) + (2.0 ** -25 if dtype is torch.float16 else 2.0 ** -149)).all()
        for x, y in zip(q, b):
            assert torch.equal(x.t, y)
            x.check()


def test_spread_of_the_8_bit_root():
    """What a byte for the root costs: after many steps of normal gradients it lies about the 32-bit moment's by a tenth.  A step moves a root by about 0.0005 x
    0.968 of itself (E|g^2 - 1| = 0.968), which the rounding to steps of 1/32 to 1/16 of it turns into that times the step in variance; deviations
    decay by 0.001 a step; so the variance settles between 0.968 x 0.0005 / 0.002 times 1/32 and 1/16: a deviation of 0.087 to 0.123, five standard
    errors of 1 / sqrt(2 n) more.  It is unbiased, but its square is larger by the variance."""
    n = 16384
    gen = torch.Generator(device=DEV).manual_seed(61)
    p, q, m, v = (torch.zeros(n, device=DEV) for _ in range(4))
    rms, ratio, window = codes(n)
    ca, cb = clocks(1, 0, (0.9, 0.999)), clocks(1, 0, (0.9, 0.999))
    for _ in range(3000):
        g = torch.randn(n, generator=gen, device=DEV) * 1e-4
        MO().adamw_step([p], [g], [m], [v], ca, lr=0.0)
        MO().adamw_step_8bit([q], [g], [rms], [ratio], [window], cb, lr=0.0, seed=6)
    _, (u,) = MO().moments_8bit([rms], [ratio], [window])
    r = u.double() / v.double().sqrt()
    more = 5 / math.sqrt(2 * n)
    assert 0.087 * (1 - more) < float(r.std()) < 0.123 * (1 + more)
    assert abs(float(r.mean()) - 1) < 0.123 ** 2 / 2 + 5 * 0.123 / math.sqrt(n)          # (curvature of the root: under half the variance)
    assert 0.087 ** 2 / 2 < float((r * r).mean()) - 1 < 0.123 ** 2 * 2
