"""gated_residual_norm against fp64: forward and gradients over kinds, types, widths, gates and absent parts.

Tolerances.  u = 2^-24, half = half a step of the stored type.  Beside its one store (half |value|) every result passes through at most about 20 fp32 roundings, and its
row sums through at most 4 + 6 + 16 additions one behind another, its column sums through at most rows / workgroup (<= 16 here) + 4 + 64 + 16; each is off by at most u times
the sum of its terms' magnitudes.  `bounds` evaluates those sums with every term by its magnitude (differences t - mean as |t| + |mean|), in fp64; K = 128 covers the longest chain."""
import math

import pytest
import torch

from asyrp_official_amd import gated_residual_norm

U, K = 2.0 ** -24, 128
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
f32, f16, bf16 = torch.float32, torch.float16, torch.bfloat16


def oracle(x, y, gate, after, before, kind, a, eps, dh, dn):
    """fp64 results and the magnitudes that bound what fp32 is off, by name.  gate [G, C] or None; after / before None or (w, b)."""
    N, C = x.shape
    r, A = {}, {}

    def norm(t, At):
        mean = t.mean(1, keepdim=True) if kind == "layer" else torch.zeros(N, 1, dtype=t.dtype)
        rstd = ((t - mean).pow(2).mean(1, keepdim=True) + eps).rsqrt()
        big = (At + At.mean(1, keepdim=True)) * rstd
        return (t - mean) * rstd, rstd, big + big.mean(1, keepdim=True)

    def back(d, Ad, hat, big, rstd):
        g = d - hat * (d * hat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0)
        return rstd * g, rstd * (Ad + big * (Ad * big).mean(1, keepdim=True) + Ad.mean(1, keepdim=True))

    one = torch.ones(C, dtype=x.dtype)
    pick = lambda wb: (one if wb is None or wb[0] is None else wb[0], 0 * one if wb is None or wb[1] is None else wb[1])  # noqa: E731
    (w1, b1), (w2, b2) = pick(after), pick(before)
    u, Au = y, y.abs()
    if after is not None:
        yhat, r1, yb = norm(y, y.abs())
        u, Au = yhat * w1 + b1, yb * w1.abs() + b1.abs()
    g = one.expand(N, C) if gate is None else gate.repeat_interleave(N // gate.shape[0], 0)
    h, Ah = a * x + g * u, (a * x).abs() + g.abs() * Au
    r["h"], A["h"] = h, Ah
    if before is not None:
        hat, r2, hb = norm(h, Ah)
        r["n"], A["n"] = hat * w2 + b2, hb * w2.abs() + b2.abs()
    if dh is None:
        dh = torch.zeros_like(x)
    D, AD = dh, dh.abs()
    if before is not None and dn is not None:
        e, Ae = back(dn * w2, (dn * w2).abs(), hat, hb, r2)
        D, AD = D + e, AD + Ae
        r["w2"], A["w2"] = (dn * hat).sum(0), (dn.abs() * hb).sum(0)
        r["b2"], A["b2"] = dn.sum(0), dn.abs().sum(0)
    r["x"], A["x"] = a * D, abs(a) * AD
    if gate is not None:
        fold = lambda t: t.reshape(gate.shape[0], -1, C).sum(1)  # noqa: E731
        r["gate"], A["gate"] = fold(D * u), fold(AD * Au)
    d, Ad = D * g, AD * g.abs()
    if after is not None:
        r["w1"], A["w1"] = (d * yhat).sum(0), (Ad * yb).sum(0)
        r["b1"], A["b1"] = d.sum(0), Ad.sum(0)
        d, Ad = back(d * w1, Ad * w1.abs(), yhat, yb, r1)
    r["y"], A["y"] = d, Ad
    return r, A


def case(N, C, kind="layer", X=f32, Y=f32, gates=0, after="wb", before="wb", P=f32, a=0.75, eps=1e-5, seed=0, grads="hn"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, dt=f32, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dt)  # noqa: E731
    wb = lambda k: None if k is None else (n(C, dt=P, std=0.3, mean=1.0) if "w" in k else None, n(C, dt=P, std=0.3) if "b" in k else None)  # noqa: E731
    return dict(x=n(N, C, dt=X, std=2.0, mean=0.3), y=n(N, C, dt=Y, std=1.5, mean=-0.5), gate=n(gates, C, dt=P, std=0.5, mean=0.4) if gates else None,
                after=wb(after), before=wb(before), kind=kind, a=a, eps=eps, dh=n(N, C, dt=X) if "h" in grads else None, dn=n(N, C, dt=Y) if "n" in grads and before else None)


def run(c):
    """Kernel results by the oracle's names."""
    leaf = lambda t: None if t is None else t.cuda().requires_grad_()  # noqa: E731
    x, y, gate = leaf(c["x"]), leaf(c["y"]), leaf(c["gate"])
    after, before = (None if wb is None else tuple(leaf(t) for t in wb) for wb in (c["after"], c["before"]))
    h, n = gated_residual_norm(x, y, gate=gate, residual_scale=c["a"], kind=c["kind"], after=after, before=before, eps=c["eps"])
    got = {"h": h.detach()}
    outs, ups = [], []
    if n is not None:
        got["n"] = n.detach()
    for o, d in ((h, c["dh"]), (n, c["dn"])):
        if d is not None:
            outs.append(o)
            ups.append(d.cuda())
    leaves = {"x": x, "y": y, "gate": gate, "w1": after and after[0], "b1": after and after[1], "w2": before and before[0], "b2": before and before[1]}
    leaves = {k: t for k, t in leaves.items() if t is not None}
    got.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups, allow_unused=True)))
    return got


def compare(c, got):
    d = lambda t: None if t is None else t.double()  # noqa: E731
    pair = lambda wb: None if wb is None else tuple(d(t) for t in wb)  # noqa: E731
    want, mag = oracle(d(c["x"]), d(c["y"]), d(c["gate"]), pair(c["after"]), pair(c["before"]), c["kind"], c["a"], c["eps"], d(c["dh"]), d(c["dn"]))
    for name, g in got.items():
        if name not in want:
            assert name in ("w2", "b2") and not g.any(), name      # n takes no gradient: its norm's parameters get zeros
            continue
        err = (g.double().cpu() - want[name]).abs()
        bad = err > HALF[g.dtype] * want[name].abs() + K * U * mag[name] + 2.0 ** -25
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / (HALF[g.dtype] * want[name].abs() + U * mag[name] + 1e-30)).max()):.1f}"


CASES = {
    "one": case(1, 1, eps=0.1), "row": case(1, 777), "column": case(300, 1, kind="rms", eps=0.1), "pair": case(2, 8), "rms": case(33, 512, "rms", after="w", before="w"),
    "odd_16": case(67, 131, X=bf16, Y=bf16, gates=1), "odd_mixed": case(40, 1003, X=f32, Y=f16, gates=4), "f16": case(64, 768, X=f16, Y=f16, gates=32, after=None),
    "rows_gate": case(36, 264, "rms", gates=36, after="w"), "many_gates": case(5000, 40, gates=2500, Y=bf16), "bare": case(50, 96, after="", before=""),
    "no_norms": case(50, 100, after=None, before=None, gates=5, grads="h"), "only_after": case(21, 1024, before=None, gates=3, grads="h"), "bias_only": case(9, 2056, after="b", before="b"),
    "wide": case(19, 4096, "rms", X=bf16, Y=bf16, gates=19, after="w"), "widest": case(11, 8192, X=f32, Y=bf16, gates=1), "widest_odd": case(5, 8191, X=f32, Y=f32),
    "half_params": case(48, 384, X=bf16, Y=bf16, gates=2, P=bf16), "grad_h": case(30, 520, gates=3, grads="h"), "grad_n": case(30, 520, gates=3, grads="n"),
    "long": case(3001, 256, "rms", X=f16, Y=f16, gates=1, after="w"), "negative_scale": case(17, 200, a=-1.5), "zero_scale": case(17, 200, a=0.0), "steps_2": case(4, 2040, Y=f16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_forward_and_gradients(name):
    compare(CASES[name], run(CASES[name]))


def test_oracle_formulas_against_autograd_and_differences():
    """The oracle itself, in fp64 on the CPU: its gradients are those of automatic differentiation, and of differences along a random direction."""
    c = case(12, 20, gates=3, seed=3)
    t = {k: c[k].double().requires_grad_() for k in ("x", "y", "gate")}
    p = {f"{n}{i}": w.double().requires_grad_() for i, k in ((1, "after"), (2, "before")) for n, w in zip("wb", c[k])}

    def f(x, y, gate, w1, b1, w2, b2, kind):
        r, _ = oracle(x, y, gate, (w1, b1), (w2, b2), kind, c["a"], c["eps"], None, None)
        return (r["h"] * c["dh"].double()).sum() + (r["n"] * c["dn"].double()).sum()

    for kind in ("layer", "rms"):
        args = [t["x"], t["y"], t["gate"], p["w1"], p["b1"], p["w2"], p["b2"]]
        grads = torch.autograd.grad(f(*args, kind), args)
        with torch.no_grad():
            r, _ = oracle(*args[:3], tuple(args[3:5]), tuple(args[5:]), kind, c["a"], c["eps"], c["dh"].double(), c["dn"].double())
            for name, g in zip(("x", "y", "gate", "w1", "b1", "w2", "b2"), grads):
                assert (r[name] - g).abs().max() <= 1e-12 * (1 + g.abs().max())
            for i, a in enumerate(args):
                d = torch.randn(a.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
                up, down = [b + 1e-6 * d if j == i else b for j, b in enumerate(args)], [b - 1e-6 * d if j == i else b for j, b in enumerate(args)]
                slope = (f(*up, kind) - f(*down, kind)) / 2e-6
                assert abs(float(slope - (grads[i] * d).sum())) <= 1e-6 * (1 + abs(float(slope)))
