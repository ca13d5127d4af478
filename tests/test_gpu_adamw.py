"""AdamW over many tensors: 32-bit moments against a plain fp64 implementation, 8-bit moments against the same arithmetic step by step.

Tolerances, 32 bits: u = 2^-24.  One step rounds a moment three times (two products, one sum: the sum's terms have one sign in v; in m they may cancel, so the bound
is on |b1 m| + |(1 - b1) g|); p is rounded three times (u each) and its update carries about 8 roundings of its factors.  Over n steps the
bounds add: v, m: 3 n u of their terms' sums; p: n (3 u |p| + 10 u |update| + what m and v are off) with |update| <= lr (1 + wd |p|) / (1 - b1)."""
import copy
import io
import math
import warnings

import pytest
import torch

from asyrp_official_amd import AdamW, AsyrpDeviceError

U = 2.0 ** -24



def tensors(shapes, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(dtype) for s in shapes]


def params_of(ts):
    return [t.clone().cuda().requires_grad_() for t in ts]


class Plain:
    """The step in fp64; None as a gradient leaves a parameter and its count alone."""

    def __init__(self, ps, lr, betas, eps, wd, max_norm=None):
        self.p = [p.double() for p in ps]
        self.m, self.v, self.t = [torch.zeros_like(p) for p in self.p], [torch.zeros_like(p) for p in self.p], [0] * len(ps)
        self.lr, self.b, self.eps, self.wd, self.max_norm = lr, betas, eps, wd, max_norm

    def step(self, gs):
        gs = [None if g is None else g.double() for g in gs]
        self.norm = math.sqrt(sum(float((g * g).sum()) for g in gs if g is not None))
        f = 1.0 if self.max_norm is None else min(1.0, self.max_norm / (self.norm + 1e-6))
        for i, g in enumerate(gs):
            if g is None:
                continue
            self.t[i] += 1
            g, (b1, b2) = g * f, self.b
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            mh, vh = self.m[i] / (1 - b1 ** self.t[i]), self.v[i] / (1 - b2 ** self.t[i])
            self.p[i] = self.p[i] * (1 - self.lr * self.wd) - self.lr * mh / (vh.sqrt() + self.eps)


SHAPES = {
    "one": [(1,)], "odd": [(3,), (255,), (256,), (257,), (1023, 3)], "chunks": [(4096,), (4097,), (8191,), (12288,)],
    "delta": [(512, 64, 1, 1), (512,), (64, 512), (64,)], "many": [(k % 7 + 1, 5) for k in range(230)], "empty": [(0,), (5,), (0, 4)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [None, 0.5], ids=["free", "clipped"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_32_bit_steps_follow_fp64(name, max_norm):
    shapes, n, hyper = SHAPES[name], 4, dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    init = tensors(shapes)
    ps = params_of(init)
    opt, plain = AdamW(ps, **hyper, max_norm=max_norm), Plain(init, 1e-2, (0.9, 0.999), 1e-8, 0.1, max_norm)
    for k in range(n):
        gs = tensors(shapes, seed=10 + k, std=10.0 ** (k - 2))
        for p, g in zip(ps, gs):
            p.grad = g.cuda()
        opt.step()
        plain.step(gs)
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - plain.norm) <= 2 * U * plain.norm
    for i, p in enumerate(ps):
        st = opt.state[p]
        assert int(st["step"]) == n
        big = 10.0 ** (n - 3) * 6            # no gradient is over six standard deviations
        assert ((st["exp_avg"].double().cpu() - plain.m[i]).abs() <= 4 * n * U * (plain.m[i].abs() + 0.1 * big)).all()
        assert ((st["exp_avg_sq"].double().cpu() - plain.v[i]).abs() <= 4 * n * U * plain.v[i] + 1e-30).all()
        # m cancels between steps: its error over sqrt(v) is at most 4 n u 0.1 big / sqrt(v); v holds the largest step's square
        noise = 4 * n * U * (0.1 * big) / (plain.v[i] / (1 - 0.999 ** n)).sqrt().clamp(min=1e-12)
        assert ((p.detach().double().cpu() - plain.p[i]).abs() <= n * (3 * U * (plain.p[i].abs() + 0.1) + 1e-2 * (10 * U * 10 + 10 * noise))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)], ids=["bf16", "f16"])
def test_16_bit_parameters_are_rounded_once(dtype, half):
    init, grads = tensors([(300,), (17, 31)], dtype), tensors([(300,), (17, 31)], dtype, seed=1)
    ps = params_of(init)
    opt, plain = AdamW(ps, lr=1e-1), Plain(init, 1e-1, (0.9, 0.999), 1e-8, 1e-2)
    for p, g in zip(ps, grads):
        p.grad = g.cuda()
    opt.step()
    plain.step(grads)
    for p, want in zip(ps, plain.p):       # half a step of the result, and the fp32 arithmetic's error (1 % of it at most)
        assert ((p.detach().double().cpu() - want).abs() <= 1.01 * half * want.abs() + 1e-7).all()


# ---- 8 bits: the codes' arithmetic written apart, value by value --------------------------------------------------------------------------
def keep8(t, coin, exponents):
    """What one block keeps of values t >= 0 (fp32 list) under random bits `coin` (20 each)."""
    import numpy as np
    t = np.asarray(t, np.float32)
    top = float(t.max())
    if top == 0:
        return [0.0] * len(t)
    mant, e = math.frexp(top)                  # top = mant 2^e, mant in [0.5, 1)
    e -= 1                                     # top = (2 mant) 2^e
    if 2 * mant > 1.875:
        e += 1                                 # rounding up may not leave the codes
    e = max(e, exponents + 2 - 127)
    low, out = e - (exponents - 2), []
    for v, c in zip(t.astype(np.float64), coin):
        k = math.frexp(v)[1] - 1 if v else None
        if v and k >= low:
            step = 2.0 ** (k - 3)
            out.append(math.floor(v / step + c / 2.0 ** 20) * step)
        else:
            unit = 2.0 ** (low - 3)
            out.append(float(int(np.float32(np.float32(v / unit) + np.float32(c / 2.0 ** 20)))) * unit)
    return out, 2.0 ** (low - 3)


def coins(i, seed, step):
    M = 0xFFFFFFFF
    x = (i & M) ^ (((seed * 0x9E3779B1) ^ (step * 0x85EBCA77)) & M) ^ (((i >> 32) * 0xC2B2AE3D) & M)
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & M
    x = ((x ^ (x >> 15)) * 0x846CA68B) & M
    x ^= x >> 16
    return x & 0xFFFFF, ((x * 0x9E3779B1) & M) >> 12


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 255, 256, 700])
def test_8_bit_moments_are_the_codes_values(n):
    import numpy as np
    init = tensors([(7,), (n,)])
    ps = params_of(init)
    opt = AdamW(ps, lr=1e-2, state_bits=8, seed=1234)
    m, v = np.zeros(n, np.float32), np.zeros(n, np.float32)
    p = init[1].numpy().copy()
    f = np.float32
    for k in range(1, 4):
        g = tensors([(n,)], seed=k)[0] * 10.0 ** torch.linspace(-9, 1, n)        # ten powers of ten within a block: both kinds of codes
        if k == 2:
            g[::3] = 0
        ps[0].grad, ps[1].grad = torch.ones(7, device="cuda"), g.cuda()
        opt.step()
        g = g.numpy()
        m = m * f(0.9) + g * f(1 - 0.9)
        v = v * f(0.999) + (g * g) * f(1 - 0.999)
        up = (m.astype(np.float64) / (1 - 0.9 ** k)) / (np.sqrt(v.astype(np.float64) / (1 - 0.999 ** k)) + 1e-8)
        p = p * (1 - 1e-2 * 1e-2) - 1e-2 * up
        assert np.all(np.abs(ps[1].detach().double().cpu().numpy() - p) <= k * (4 * U * (np.abs(p) + 1) + 1e-2 * 20 * U * np.abs(up) * 10))
        for b in range(0, n, 256):
            at = range(b, min(n, b + 256))
            c = [coins(256 + i, 1234, k) for i in at]                             # the second parameter's values start at 256
            km, _ = keep8(np.abs(m[b:b + 256]), [x[0] for x in c], 16)
            kv, unit = keep8(v[b:b + 256], [x[1] for x in c], 32)
            m[b:b + 256] = np.where(m[b:b + 256] < 0, -np.array(km), km).astype(f)
            v[b:b + 256] = np.maximum(kv, unit).astype(f)
        gm, gv = (t[256:256 + n].cpu().numpy() for t in opt.moments()[0])
        assert np.array_equal(gm, m) and np.array_equal(gv, v)
        assert not opt.moments()[0][0][256 + n:].any() and not opt.moments()[0][1][256 + n:].any()


def same_run(opt_a, ps_a, opt_b, ps_b, steps=2, seed=50):
    """Both take the same gradients; their parameters and moments are equal to the bit afterwards."""
    for k in range(steps):
        for p, q, g in zip(ps_a, ps_b, tensors([p.shape for p in ps_a], seed=seed + k)):
            p.grad = g.cuda().to(p.dtype)
            q.grad = p.grad.clone()
        opt_a.step()
        opt_b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps_a, ps_b))
    for (m, v), (m2, v2) in zip(opt_a.moments(), opt_b.moments()):
        assert torch.equal(m, m2) and torch.equal(v, v2)


def trained(bits=32, shapes=((300,), (5, 7), (256,)), dtype=torch.float32, steps=3, **kw):
    ps = params_of(tensors(shapes, dtype))
    opt = AdamW(ps, lr=1e-2, state_bits=bits, seed=9, **kw)
    for k in range(steps):
        for p, g in zip(ps, tensors(shapes, dtype, seed=20 + k)):
            p.grad = g.cuda()
        opt.step()
    return opt, ps


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_travels_through_files_copies_and_pickles(bits):
    opt, ps = trained(bits)
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf)
    buf.seek(0)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = AdamW(qs, lr=5.0, state_bits=bits, seed=9)
    other.load_state_dict(torch.load(buf, weights_only=True))
    assert other.param_groups[0]["lr"] == 1e-2 and int(other.state[qs[0]]["step"]) == 3
    same_run(opt, ps, other, qs)
    opt, ps = trained(bits)
    twin = copy.deepcopy({"opt": opt, "ps": ps})
    same_run(opt, ps, twin["opt"], twin["ps"])
    started, qs = trained(bits, steps=5)                        # into an optimiser that has moments of its own
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    started.load_state_dict(opt.state_dict())
    same_run(opt, ps, started, qs)
    with pytest.raises(ValueError):
        AdamW(qs, state_bits=40 - bits).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        AdamW(qs[:2], state_bits=bits).load_state_dict(opt.state_dict())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_without_a_gradient_stands_still(bits):
    init = tensors([(300,), (40,), (7,)])
    ps = params_of(init)
    opt, plain = AdamW(ps, lr=1e-2, state_bits=bits), Plain(init, 1e-2, (0.9, 0.999), 1e-8, 1e-2)
    for k in range(3):
        gs = tensors([p.shape for p in init], seed=k)
        gs[1] = None if k < 2 else gs[1]
        for p, g in zip(ps, gs):
            p.grad = None if g is None else g.cuda()
        opt.step()
        plain.step(gs)
        assert (k == 2) != torch.equal(ps[1].detach().cpu(), init[1])
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 1, 3]
    # its first step is corrected as a first one: the whole rate, not a third of it.  (1 - lr wd), its product with p and the difference are rounded
    # (u |p| each), and the update of at most lr in about ten places
    assert ((ps[1].detach().double().cpu() - plain.p[1]).abs() <= 3 * U * plain.p[1].abs() + 10 * U * 1e-2).all()
    before = [p.detach().clone() for p in ps]
    opt.zero_grad()
    opt.step()                                                  # no gradient at all
    assert all(torch.equal(p, b) for p, b in zip(ps, before))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_skips_the_step(bits, bad):
    opt, ps = trained(bits, max_norm=1.0)
    before = [p.detach().clone() for p in ps], [t.clone() for pair in opt.moments() for t in pair]
    ps[2].grad[17] = bad
    opt.step()
    assert not math.isfinite(float(opt.grad_norm))
    assert all(torch.equal(p, b) for p, b in zip(ps, before[0])) and all(torch.equal(t, b) for t, b in zip([t for pair in opt.moments() for t in pair], before[1]))
    assert int(opt.state[ps[0]]["step"]) == 3


@pytest.mark.gpu
def test_without_a_norm_it_goes_its_way():
    for bits in (32, 8):
        opt, ps = trained(bits)
        ps[0].grad[3] = math.nan
        opt.step()
        assert ps[0][3].isnan() and torch.isfinite(ps[1]).all() and int(ps[0].isnan().sum()) == 1
        m, v = opt.moments()[0]
        assert m[3].isnan() and v[3].isnan()
        if bits == 8:                                           # the block that held it, and nothing else
            assert m[:256].isnan().all() and torch.isfinite(m[256:]).all() and torch.isfinite(v[256:]).all()


@pytest.mark.gpu
def test_groups_types_and_layouts_of_one_step():
    """Two groups with rates of their own, three types, gradients laid out otherwise, odd addresses: like one optimiser each."""
    shapes = [(6, 4, 3, 3), (300,), (129,), (64, 2)]
    types = [torch.float32, torch.bfloat16, torch.float16, torch.float32]
    init = [t.to(d) for t, d in zip(tensors(shapes), types)]
    ps = params_of(init)
    flat = torch.zeros(129 + 3, device="cuda", dtype=torch.float16)
    ps[2] = flat[3:].copy_(ps[2].detach()).requires_grad_()     # an address that no wide load may take
    opt = AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.5, "betas": (0.5, 0.9)}], lr=1e-3, max_norm=0.1)
    alone = [AdamW([p.detach().clone().requires_grad_()], lr=lr, weight_decay=wd, betas=b) for p, lr, wd, b in
             zip(ps, (1e-2, 1e-2, 1e-3, 1e-3), (1e-2, 1e-2, 0.5, 0.5), ((0.9, 0.999),) * 2 + ((0.5, 0.9),) * 2)]
    for k in range(2):
        gs = [t.to(d).cuda() for t, d in zip(tensors(shapes, seed=k), types)]
        ps[0].grad = gs[0].to(memory_format=torch.channels_last)
        ps[1].grad, ps[2].grad, ps[3].grad = gs[1], gs[2], gs[3].t().contiguous().t()
        opt.step()
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
        assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        for o, g in zip(alone, gs):
            (q,) = o.param_groups[0]["params"]
            q.grad = g
            o.max_norm = None
            q.grad = (g.float() * torch.tensor(min(1.0, 0.1 / (norm + 1e-6)), dtype=torch.float64).float().cuda()).to(torch.float32) if q.dtype == torch.float32 else g
        for o, p in list(zip(alone, ps))[:1] + list(zip(alone, ps))[3:]:
            o.step()
            assert torch.equal(o.param_groups[0]["params"][0], p)
    assert all(torch.isfinite(p).all() and not torch.equal(p.detach().cpu(), t) for p, t in zip(ps, init))
    assert not flat[:3].any()


@pytest.mark.gpu
def test_a_captured_step_counts_and_follows_a_rate_on_the_device():
    shapes = [(1000,), (33, 5)]
    init = tensors(shapes)
    for bits in (32, 8):
        ps, qs = params_of(init), params_of(init)
        lr = torch.tensor(1e-2, device="cuda")
        opt = AdamW(ps, lr=lr, state_bits=bits, max_norm=2.0, seed=3)
        eager = AdamW(qs, lr=1e-2, state_bits=bits, max_norm=2.0, seed=3)
        for p, g in zip(ps, tensors(shapes, seed=1)):
            p.grad = g.cuda()
        opt.prepare()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        for k in range(4):
            rate = float(torch.tensor(1e-2 / (k + 1)))          # what a float32 holds of it
            lr.fill_(rate)
            for p, q, g in zip(ps, qs, tensors(shapes, seed=10 + k)):
                p.grad.copy_(g)
                q.grad = g.cuda()
            eager.param_groups[0]["lr"] = rate
            graph.replay()
            eager.step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(ps, qs)), (bits, k)
            assert float(opt.grad_norm) == float(eager.grad_norm)
        assert int(opt.state[ps[0]]["step"]) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on_with_loaded_moments(bits):
    shapes = [(1000,), (33, 5)]
    init, grads = tensors(shapes), [tensors(shapes, seed=20 + k) for k in range(5)]
    lr = torch.tensor(1e-2, device="cuda")
    ps, qs = params_of(init), params_of(init)
    opt, eager = AdamW(ps, lr=lr, state_bits=bits, max_norm=2.0, seed=3), AdamW(qs, lr=2.0 ** -9, state_bits=bits, max_norm=2.0, seed=3)
    for p, g in zip(ps, grads[0]):
        p.grad = g.cuda()
    opt.prepare()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    for k in (1, 2):                            # the eager one's steps, which the captured one takes over
        for q, g in zip(qs, grads[k]):
            q.grad = g.cuda()
        eager.step()
    opt.load_state_dict(copy.deepcopy(eager.state_dict()))
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 2.0 ** -9
    with torch.no_grad():
        for p, q in zip(ps, qs):
            p.copy_(q)
    for k in (3, 4):
        for p, q, g in zip(ps, qs, grads[k]):
            p.grad.copy_(g)
            q.grad = g.cuda()
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
        assert float(opt.grad_norm) == float(eager.grad_norm)
    assert int(opt.state[ps[1]]["step"]) == 4
    opt.load_state_dict(AdamW(params_of(init), state_bits=bits).state_dict())        # of one that has not stepped
    assert not any(m.any() or v.any() for m, v in opt.moments()) and int(opt.state[ps[0]]["step"]) == 0


def test_a_parameter_twice_is_refused():
    p = torch.zeros(8, requires_grad=True)
    with pytest.raises(ValueError), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        AdamW([p, p])


@pytest.mark.gpu
def test_a_first_step_is_not_captured():
    ps = params_of(tensors([(100,)]))
    ps[0].grad = torch.ones_like(ps[0])
    opt = AdamW(ps)
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)                       # a graph of nothing is a warning
        with pytest.raises(RuntimeError):
            opt.step()
    assert torch.equal(ps[0].detach().cpu(), tensors([(100,)])[0])
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 1


@pytest.mark.gpu
def test_another_stream_and_two_optimisers_at_once():
    a, pa = trained(8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, pb = trained(8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))
    c, pc = trained(8)
    assert all(torch.equal(p, q) for p, q in zip(pa, pc))        # one seed, one result
    # another seed rounds otherwise
    d = AdamW(params_of(tensors([(300,)])), state_bits=8, seed=1)
    e = AdamW(params_of(tensors([(300,)])), state_bits=8, seed=2)
    for o in (d, e):
        (p,) = o.param_groups[0]["params"]
        p.grad = tensors([(300,)], seed=5)[0].cuda()
        o.step()
    assert not torch.equal(d.moments()[0][0], e.moments()[0][0])


@pytest.mark.gpu
def test_8_bit_rounding_keeps_the_mean():
    """20000 values of one size, each block with a larger one beside them: the mean of what is kept is theirs within five standard errors (a code's
    step is at most 1/8 of a value, so one rounding's deviation is at most 1/16)."""
    n = 256 * 80
    g = torch.full((n,), 0.731)
    g[::256] = 100.0
    p = torch.zeros(n, device="cuda", requires_grad=True)
    opt = AdamW([p], state_bits=8, seed=77)
    p.grad = g.cuda()
    opt.step()
    m, v = (t.double().cpu() for t in opt.moments()[0])
    some = torch.ones(n, dtype=torch.bool)
    some[::256] = False
    for kept, want in ((m[some], 0.1 * 0.731), (v[some], 0.001 * 0.731 ** 2)):
        assert abs(float(kept.mean()) / want - 1) <= 5 * (1 / 16) / math.sqrt(int(some.sum()))
        assert float((kept / want - 1).abs().max()) <= 1 / 8


@pytest.mark.gpu
def test_the_deltablock_is_uploaded_again_behind_a_step():
    """The engine keeps a copy of the DeltaBlock's weights and takes what a step changed."""
    import os
    import sys
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from oracle import sampler as osamp
    from oracle.weights import SMALL, hash_normal
    from util_models import hip_model, synthetic
    from asyrp_official_amd import denoising_step
    model = hip_model(SMALL, synthetic(SMALL, 1, seed=11), 1, max_batch=1)
    for p in model.parameters():
        p.requires_grad_(False)
    for p in model.layer_0.parameters():
        p.requires_grad_(True)
    b = osamp.beta_schedule().cuda()
    x, tgt = (hash_normal(f"adamw.{k}", (1, 3, SMALL.resolution, SMALL.resolution)).cuda() for k in "xt")
    one = torch.ones(1, device="cuda")
    kw = dict(models=model, logvars=None, b=b, sampling_type="ddim", eta=0.0, index=0, t_edit=500, hs_coeff=(1.0, 1.0))
    step = lambda: denoising_step(x, t=one * 768.0, t_next=one * 743.0, **kw)[1]  # noqa: E731
    opt = AdamW(model.layer_0.parameters(), lr=1e-2, state_bits=8, max_norm=1.0)
    seen = []
    for _ in range(3):
        opt.zero_grad()
        x0 = step()
        seen.append(x0.detach().clone())
        torch.nn.functional.l1_loss(x0, tgt).backward()
        opt.step()
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    # a model that is given the stepped weights as new ones computes the same
    fresh = hip_model(SMALL, {k: v.detach().cpu() for k, v in model.state_dict().items()}, 1, max_batch=1)
    with torch.no_grad():
        a = step()
        kw["models"] = fresh
        assert torch.equal(a, step())


@pytest.mark.gpu
def test_refusals():
    p = torch.zeros(8, device="cuda", requires_grad=True)
    for kw in (dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=math.inf), dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1),
               dict(lr=torch.ones(2))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError):
        AdamW([torch.zeros(3, device="cuda", dtype=torch.float64, requires_grad=True)])
    cpu = torch.zeros(3, requires_grad=True)
    cpu.grad = torch.ones(3)
    with pytest.raises(AsyrpDeviceError):
        AdamW([cpu]).step()
    bad = torch.zeros(4, 6, device="cuda").t().requires_grad_()
    bad.grad = torch.ones_like(bad)
    with pytest.raises(ValueError):
        AdamW([bad]).step()
    opt = AdamW([p], lr=torch.tensor(1e-3, device="cuda", dtype=torch.float64))
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError):
        opt.step()
    opt = AdamW([p])
    opt.step()
    p.data = torch.zeros(4, device="cuda")                       # the moments are of eight values
    p.grad = None
    p.grad = torch.ones(4, device="cuda")
    with pytest.raises(ValueError):
        opt.step()


def test_library_refuses_what_its_kernels_do_not_take():
    import struct
    from asyrp_official_amd import _lib
    lib = _lib.load()

    def call(numel=8, at=0, index=0, p=4096, g=4096, n=1, dtype=_lib.F32, lr=1e-3, b1=0.9, eps=1e-8, wd=0.0, steps=4096, sumsq=0, max_norm=0.0, count=0, m=4096, v=4096, me=4096,
             bits=32, scratch=4096):
        spec = _lib.ADAMW.pack(lr, b1, 0.999, eps, wd, 0, steps, sumsq, max_norm, 0, m, v, me, me, count, bits, 0)
        return lib.asyrp_adamw_step(0, spec, struct.pack("5q", p, g, numel, at, index), n, dtype, scratch, None)

    for bad in (dict(numel=-1), dict(at=100), dict(at=-256), dict(index=-1), dict(p=0), dict(g=0), dict(p=4098), dict(g=4097), dict(n=-1), dict(dtype=3), dict(lr=math.nan), dict(b1=1.0),
                dict(b1=-0.1), dict(eps=-1.0), dict(eps=math.nan), dict(wd=math.inf), dict(steps=0), dict(sumsq=4096), dict(sumsq=4096, max_norm=1.0, count=-1), dict(m=0), dict(v=4104),
                dict(me=0, bits=8), dict(bits=16), dict(scratch=None), dict(scratch=4100)):
        assert call(**bad) == -1, bad
        assert b"AdamW" in lib.asyrp_last_error()
    one = struct.pack("5q", 4096, 4096, 8, 0, 0)
    assert lib.asyrp_adamw_step(0, None, one, 1, 0, 4096, None) == -1
    assert lib.asyrp_grad_sumsq(0, one, 1, 0, None, None) == -1 and lib.asyrp_grad_sumsq(0, None, 1, 0, 4096, None) == -1
    assert lib.asyrp_adamw_moments(0, 4096, 4096, 4096, 4096, 100, 4096, 4096, None) == -1
    assert lib.asyrp_adamw_moments(0, None, 4096, 4096, 4096, 256, 4096, 4096, None) == -1
    assert lib.asyrp_adamw_moments(0, None, None, None, None, 0, None, None, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("stepped", [False, True], ids=["fresh", "stepped"])
def test_hooks_of_a_load_see_the_state(bits, stepped):
    """A hook in front may edit or replace what is loaded, one behind sees what was; both come off again."""
    src, _ = trained(bits)
    dst, ps = trained(bits, steps=5) if stepped else trained(bits, steps=0)
    seen = []

    def front(opt, sd):
        assert opt is dst and set(sd["state"]) == {0, 1, 2}
        return {**sd, "state": {i: {**st, "step": torch.full_like(st["step"], 7)} for i, st in sd["state"].items() if i != 1}}

    front_handle = dst.register_load_state_dict_pre_hook(front)
    behind = dst.register_load_state_dict_post_hook(lambda opt: seen.append([int(opt.state[p]["step"]) if opt.state.get(p) else 0 for p in ps]))
    dst.load_state_dict(src.state_dict())
    assert seen == [[7, 0, 7]]
    for (a, b), (c, d) in zip(dst.moments(), src.moments()):
        keep = torch.ones_like(a, dtype=torch.bool)
        keep[512:768] = False                                          # the second of three parameters of 300, 35 and 256 values: its moments were left out
        assert torch.equal(a[keep], c[keep]) and torch.equal(b[keep], d[keep]) and not a[~keep].any() and not b[~keep].any()
    front_handle.remove()
    behind.remove()
    dst.load_state_dict(src.state_dict())
    assert len(seen) == 1 and [int(dst.state[p]["step"]) for p in ps] == [3, 3, 3]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_load_that_is_refused_changes_nothing(bits):
    src, _ = trained(bits)
    opt, ps = trained(bits, steps=5)
    opt.param_groups[0]["lr"] = 0.25
    want = [t.clone() for pair in opt.moments() for t in pair]
    good = src.state_dict()
    for key in ("exp_avg", "exp_avg_sq", "step") + (("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ()):
        bad = {**good, "state": {i: {**st, key: torch.zeros(3, device="cuda", dtype=st[key].dtype)} if i == 2 else st for i, st in good["state"].items()}}
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert all(torch.equal(a, b) for a, b in zip(want, [t for pair in opt.moments() for t in pair])), key
        assert opt.param_groups[0]["lr"] == 0.25 and [int(opt.state[p]["step"]) for p in ps] == [5, 5, 5]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_is_refused_changes_nothing(bits):
    """A value of the second group that the step does not take is found before the first group has moved."""
    for key, bad in (("lr", math.nan), ("lr", torch.tensor(1e-3, device="cuda", dtype=torch.float64)), ("lr", torch.tensor(math.inf)), ("betas", (0.9, 1.0)), ("betas", (math.nan, 0.9)), ("eps", -1.0),
                     ("weight_decay", math.inf)):
        ps = params_of(tensors([(40,), (50,)]))
        opt = AdamW([{"params": ps[:1]}, {"params": ps[1:]}], state_bits=bits, max_norm=1.0)
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        want = [p.detach().clone() for p in ps] + [t.clone() for pair in opt.moments() for t in pair]
        opt.param_groups[1][key] = bad
        with pytest.raises(ValueError):
            opt.step()
        assert all(torch.equal(a, b) for a, b in zip(want, [p.detach() for p in ps] + [t for pair in opt.moments() for t in pair])), (key, bad)
        assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_of_nothing_but_empty_parameters_steps(bits):
    e = torch.zeros(0, 3, device="cuda", requires_grad=True)
    p = torch.ones(5, device="cuda", requires_grad=True)
    opt = AdamW([{"params": [e]}, {"params": [p]}], state_bits=bits, max_norm=1.0)
    e.grad, p.grad = torch.zeros_like(e), torch.ones_like(p)
    opt.step()
    assert int(opt.state[e]["step"]) == 1 and int(opt.state[p]["step"]) == 1 and not torch.equal(p.detach(), torch.ones_like(p))
    alone = AdamW([e], state_bits=bits)
    alone.step()
    assert int(alone.state[e]["step"]) == 1 and [t.numel() for t in alone.moments()[0]] == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)], ids=["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 255, 700, 4500])
def test_8_bit_moments_of_16_bit_parameters(n, dtype, half):
    """The moments are those of the gradients' values, code for code; a parameter is off by half a step of its type from the fp64 step that starts at what it held."""
    import numpy as np
    f, lr = np.float32, 1e-2
    (p,) = params_of(tensors([(n,)], dtype))
    opt = AdamW([p], lr=lr, state_bits=8, seed=77)
    m, v = np.zeros(n, f), np.zeros(n, f)
    for k in range(1, 4):
        g = (tensors([(n,)], seed=k)[0] * 10.0 ** torch.linspace(-3, 1, n)).to(dtype)
        if k == 2:
            g[::3] = 0
        p.grad, before = g.cuda(), p.detach().double().cpu().numpy()
        opt.step()
        g = g.float().numpy()
        m = m * f(0.9) + g * f(1 - 0.9)
        v = v * f(0.999) + (g * g) * f(1 - 0.999)
        up = (m.astype(np.float64) / (1 - 0.9 ** k)) / (np.sqrt(v.astype(np.float64) / (1 - 0.999 ** k)) + 1e-8)
        want = before * (1 - lr * 1e-2) - lr * up
        # half a step of the stored value (where it is under the type's normal range: of 2^-24 or less), and fp32 arithmetic as in the test above
        assert np.all(np.abs(p.detach().double().cpu().numpy() - want) <= half * np.abs(want) + 2.0 ** -25 + 4 * U * (np.abs(want) + 1) + lr * 200 * U * np.abs(up))
        for b in range(0, n, 256):
            c = [coins(i, 77, k) for i in range(b, min(n, b + 256))]
            km, _ = keep8(np.abs(m[b:b + 256]), [x[0] for x in c], 16)
            kv, unit = keep8(v[b:b + 256], [x[1] for x in c], 32)
            m[b:b + 256] = np.where(m[b:b + 256] < 0, -np.array(km), km).astype(f)
            v[b:b + 256] = np.maximum(kv, unit).astype(f)
        gm, gv = (t[:n].cpu().numpy() for t in opt.moments()[0])
        assert np.array_equal(gm, m) and np.array_equal(gv, v)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_addresses_that_no_wide_load_may_take(dtype, bits):
    """A parameter, its gradient or both one value behind a wide address: equal to the bit to the aligned run, and nothing beside them moves."""
    n = 2 * 4096 + 809
    init, grads = tensors([(n,)], dtype)[0], [tensors([(n,)], dtype, seed=60 + k)[0] for k in range(3)]

    def go(shift_p, shift_g):
        pads = [torch.full((n + 9,), 3.0, device="cuda", dtype=dtype) for _ in range(2)]
        p, g = (t[s:s + n] for t, s in zip(pads, (shift_p, shift_g)))
        p = p.copy_(init).requires_grad_()
        opt = AdamW([p], lr=1e-2, state_bits=bits, seed=5, max_norm=20.0)
        for src in grads:
            g.copy_(src)
            p.grad = g
            opt.step()
        for t, s in zip(pads, (shift_p, shift_g)):
            assert (t[:s] == 3.0).all() and (t[s + n:] == 3.0).all()
        assert torch.equal(g.cpu(), grads[-1])
        return [p.detach().clone(), opt.grad_norm.clone(), *opt.moments()[0]]

    want = go(0, 0)
    assert not torch.equal(want[0].cpu(), init)
    for shifts in ((1, 0), (0, 1), (1, 1), (3, 2)):
        assert all(torch.equal(a, b) for a, b in zip(go(*shifts), want)), shifts


@pytest.mark.gpu
def test_every_parameter_of_two_groups_and_three_types_follows_fp64():
    shapes, types = [(6, 4, 3, 3), (300,), (129,), (64, 2)], [torch.float32, torch.bfloat16, torch.float16, torch.float32]
    hyper = [dict(lr=1e-2, betas=(0.9, 0.999), weight_decay=1e-2)] * 2 + [dict(lr=1e-3, betas=(0.5, 0.9), weight_decay=0.5)] * 2
    ps = params_of([t.to(d) for t, d in zip(tensors(shapes), types)])
    flat = torch.zeros(129 + 3, device="cuda", dtype=torch.float16)
    ps[2] = flat[3:].copy_(ps[2].detach()).requires_grad_()
    opt = AdamW([{"params": ps[:2], **hyper[0]}, {"params": ps[2:], **hyper[2]}], max_norm=0.1)
    m, v = [0.0] * 4, [0.0] * 4
    for k in range(1, 4):
        gs, before = [t.to(d) for t, d in zip(tensors(shapes, seed=k), types)], [p.detach().double().cpu() for p in ps]
        for p, g in zip(ps, gs):
            p.grad = g.cuda()
        opt.step()
        f = min(1.0, 0.1 / (math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs)) + 1e-6))
        for i, (p, g, h) in enumerate(zip(ps, gs, hyper)):
            (b1, b2), g = h["betas"], g.double() * f
            m[i], v[i] = b1 * m[i] + (1 - b1) * g, b2 * v[i] + (1 - b2) * g * g
            up = (m[i] / (1 - b1 ** k)) / ((v[i] / (1 - b2 ** k)).sqrt() + 1e-8)
            want = before[i] * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * up
            half = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[p.dtype]
            # half a step of its type; three roundings of p; the update's ten, and what the moments are off: 4 u of terms that reach 6 f (the largest gradient) over sqrt(v)
            noise = 4 * k * U * 6 * f / (v[i] / (1 - b2 ** k)).sqrt().clamp(min=1e-12)
            off = (p.detach().double().cpu() - want).abs()
            assert (off <= half * want.abs() + (2.0 ** -25 if half else 0.0) + 3 * U * (before[i].abs() + 0.1) + h["lr"] * (10 * U * (1 + up.abs()) + noise)).all(), (k, i)
