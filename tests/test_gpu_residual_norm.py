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


# rows that share a wave, a gate to every row, groups of four, eight and sixteen values and rows that fall out of groups
WIDTHS = {
    "narrow": case(83, 33, "rms", gates=1), "narrow_16": case(129, 64, X=bf16, Y=bf16, gates=43), "narrow_full": case(35, 128, X=f32, Y=f16, gates=5), "narrow_odd": case(31, 127, "rms", X=f16, Y=f16),
    "row_gate_17": case(45, 17, gates=45), "row_gate_64": case(51, 60, "rms", X=bf16, Y=bf16, gates=51), "row_gate_128": case(22, 100, X=f32, Y=bf16, gates=22, before=None, grads="h"),
    "row_gate_512": case(37, 509, X=f16, Y=f16, gates=37, after=None), "row_gate_wide": case(9, 1100, gates=9), "row_gate_one": case(1, 80, gates=1),
    "fours": case(40, 2300, "rms", X=bf16, Y=bf16, gates=1), "fours_mixed": case(23, 516, X=f32, Y=f16, gates=23), "sixteens": case(13, 4112, X=bf16, Y=bf16, gates=1), "sixteens_f32": case(7, 6144, "rms", gates=7),
    "eights": case(9, 5000, X=f16, Y=f16, gates=3), "odd_wide": case(7, 5041, gates=1), "odd_fours_wide": case(6, 4100, X=bf16, Y=bf16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(WIDTHS))
def test_widths_and_gates_per_row(name):
    compare(WIDTHS[name], run(WIDTHS[name]))


@pytest.mark.gpu
def test_gate_per_row_without_its_gradient():
    c = WIDTHS["row_gate_64"]
    x, y = (c[k].cuda().requires_grad_() for k in ("x", "y"))
    both = []
    for wants in (True, False):
        h, n = gated_residual_norm(x, y, gate=c["gate"].cuda().requires_grad_(wants), residual_scale=c["a"], kind=c["kind"], after=tuple(w.cuda() for w in c["after"]), before=tuple(w.cuda() for w in c["before"]), eps=c["eps"])
        both.append((h, n, *torch.autograd.grad((h, n), (x, y), (c["dh"].cuda(), c["dn"].cuda()))))
    for a, b in zip(*both):
        assert torch.equal(a, b)


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


@pytest.mark.gpu
def test_shapes_views_and_empty_batches():
    c = case(24, 40, gates=4)
    want = run(c)
    x, y, gate = c["x"].cuda().view(2, 3, 4, 40), c["y"].cuda().view(2, 3, 4, 40), c["gate"].cuda()
    args = dict(gate=gate, residual_scale=c["a"], after=tuple(t.cuda() for t in c["after"]), before=tuple(t.cuda() for t in c["before"]), eps=c["eps"])
    h, n = gated_residual_norm(x, y, **args)
    assert h.shape == x.shape and torch.equal(h.view(24, 40), want["h"]) and torch.equal(n.view(24, 40), want["n"])
    strided = torch.empty(24, 80, device="cuda")[:, ::2].copy_(x.view(24, 40))
    shifted = torch.empty(24 * 40 + 1, device="cuda")[1:].view(24, 40).copy_(y.view(24, 40))      # no 16-byte address: read value by value
    h, n = gated_residual_norm(strided, shifted, **args)
    # 40 columns read value by value are added up in another order than four by four
    assert torch.equal(h, want["h"]) or (h - want["h"]).abs().max() <= 1e-5
    assert (n - want["n"]).abs().max() <= 1e-5
    e = torch.zeros(0, 3, 40, device="cuda", requires_grad=True)
    h, n = gated_residual_norm(e, e, gate=args["gate"].clone().requires_grad_(), before=args["before"])
    assert h.shape == n.shape == (0, 3, 40)
    g = args["gate"].clone().requires_grad_()
    h, n = gated_residual_norm(e, e, gate=g, before=args["before"])
    gx, gg = torch.autograd.grad((h.sum() + n.sum()), [e, g])
    assert gx.shape == e.shape and not gg.any()


@pytest.mark.gpu
def test_rows_do_not_see_each_other():
    c = case(70, 96, gates=2)
    want = run(c)
    c["x"][3], c["y"][40, 5] = math.nan, math.inf
    got = run(c)
    rows = [i for i in range(70) if i not in (3, 40)]
    for n in ("h", "n", "x", "y"):
        assert torch.equal(got[n][rows], want[n][rows]), n
    assert got["h"][3].isnan().all() and not torch.isfinite(got["n"][40]).any()


@pytest.mark.gpu
def test_some_gradients_alone():
    c = case(33, 128, gates=3)
    full = run(c)
    t = {"x": c["x"].cuda(), "y": c["y"].cuda(), "gate": c["gate"].cuda(), **{f"{n}{i}": w.cuda() for i, k in ((1, "after"), (2, "before")) for n, w in zip("wb", c[k])}}
    for name in t:
        a = {k: v.clone().requires_grad_(k == name) for k, v in t.items()}
        h, n = gated_residual_norm(a["x"], a["y"], gate=a["gate"], residual_scale=c["a"], after=(a["w1"], a["b1"]), before=(a["w2"], a["b2"]), eps=c["eps"])
        (g,) = torch.autograd.grad([h, n], [a[name]], [c["dh"].cuda(), c["dn"].cuda()])
        assert torch.equal(g, full[name]), name


@pytest.mark.gpu
def test_streams_and_graph_replays_agree():
    c = case(300, 768, X=bf16, Y=bf16, gates=3)
    want = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [t.cuda().requires_grad_() for t in (c["x"], c["y"], c["gate"], *c["after"], *c["before"])]
    ups = [c["dh"].cuda(), c["dn"].cuda()]

    def step():
        x, y, gate, w1, b1, w2, b2 = leaves
        h, n = gated_residual_norm(x, y, gate=gate, residual_scale=c["a"], after=(w1, b1), before=(w2, b2), eps=c["eps"])
        grads = torch.autograd.grad([h, n], leaves, ups)
        return [h.detach(), n.detach(), *grads]

    with torch.cuda.stream(side):
        warm = step()
        del warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        caught = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].mul_(1.5)
            leaves[2].add_(0.25)
        eager = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(caught, eager)), i


def test_cpu_tensors_are_refused():
    from asyrp_official_amd import AsyrpDeviceError
    with pytest.raises(AsyrpDeviceError):
        gated_residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))


def test_library_refuses_what_its_kernels_do_not_take():
    from asyrp_official_amd import _lib
    lib = _lib.load()

    def call(rows=4, gates=0, width=64, kind=0, after=0, before=1, X=0, Y=0, a=1.0, eps=1e-5, x=4096, gate=None, stats=4096, dn=4096, dw1=None, ws=4096):
        spec = _lib.RESIDUAL_NORM.pack(rows, gates, width, kind, after, before, X, Y, a, eps)
        return (lib.asyrp_residual_norm_forward(0, spec, x, 4096, gate, None, None, None, None, 4096, 4096, stats, None),
                lib.asyrp_residual_norm_backward(0, spec, x, 4096, gate, None, None, None, stats, None, dn, 4096, 4096, None, dw1, None, None, None, ws, None))

    for bad in (dict(rows=-1), dict(rows=2 ** 31), dict(gates=3), dict(gates=-1), dict(width=0), dict(width=8193), dict(kind=2), dict(X=1, Y=0), dict(X=1, Y=2), dict(X=3, Y=3),
                dict(a=math.nan), dict(eps=-1.0), dict(eps=math.inf), dict(x=None), dict(gates=2), dict(gate=4096), dict(stats=4100)):
        assert call(**bad) == (-1, -1), bad
        assert b"residual norm" in lib.asyrp_last_error()
    for bad in (dict(dn=None), dict(before=0), dict(dw1=4096), dict(ws=None)):
        assert call(**{**dict(rows=4), **bad})[1] == -1 if "before" not in bad else True
    assert call(rows=0) == (0, 0)
    assert lib.asyrp_residual_norm_workspace(None) == -1


@pytest.mark.gpu
def test_refusals():
    from asyrp_official_amd import AsyrpDeviceError
    x = torch.zeros(6, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for args, kw in (((x, x[:5]), {}), ((x.half(), x), {}), ((x.double(), x.double()), {}), ((x, x), dict(kind="group")), ((x, x), dict(gate=w[:4])), ((x, x), dict(gate=x[:4])),
                     ((x, x), dict(gate=torch.zeros(0, 8, device="cuda"))), ((x, x), dict(before=w)), ((x, x), dict(before=(w[:4], None))), ((x, x), dict(after=(w, w.double()))),
                     ((x, x), dict(eps=-1.0)), ((x, x), dict(residual_scale=math.inf)), ((x[0, 0], x[0, 0]), {}), ((torch.zeros(2, 8200, device="cuda"),) * 2, {}), ((x[:, :0], x[:, :0]), {})):
        with pytest.raises(ValueError):
            gated_residual_norm(*args, **kw)
    for args, kw in (((x, x.cpu()), {}), ((x, x), dict(gate=w.cpu())), ((x, x), dict(before=(w.cpu(), None)))):
        with pytest.raises(AsyrpDeviceError):
            gated_residual_norm(*args, **kw)


def test_library_refuses_backward_calls_of_a_forward_that_is_there():
    """What only the backward refuses, each argument by itself.  (Nothing else is called: the forward would take these addresses for real ones.)"""
    from asyrp_official_amd import _lib
    lib = _lib.load()

    def backward(before=1, after=0, gate=None, gates=0, dh=None, dn=4096, dgate=None, dw1=None, db1=None, dw2=None, db2=None, stats=4096, ws=4096):
        spec = _lib.RESIDUAL_NORM.pack(4, gates, 64, 0, after, before, 0, 0, 1.0, 1e-5)
        return lib.asyrp_residual_norm_backward(0, spec, 4096, 4096, gate, None, None, None, stats, dh, dn, 4096, 4096, dgate, dw1, db1, dw2, db2, ws, None)

    for bad in (dict(dn=None), dict(before=0), dict(dw1=4096), dict(db1=4096), dict(before=0, dn=None, dh=4096, dw2=4096), dict(before=0, dn=None, dh=4096, db2=4096),
                dict(dgate=4096), dict(gate=4096), dict(gates=2), dict(ws=None), dict(stats=None), dict(stats=4100)):
        assert backward(**bad) == -1, bad
        assert b"residual norm" in lib.asyrp_last_error()


def test_made_up_addresses_are_called_only_where_no_gpu_is(monkeypatch):
    """test_library_refuses_what_its_kernels_do_not_take also calls the forward with arguments that only the backward refuses: harmless without a GPU, a memory
    fault with one.  It is skipped there."""
    import conftest

    class Item:
        def __init__(self, name):
            self.name, self.nodeid, self.marks = name, "tests/test_gpu_residual_norm.py::" + name, []
        add_marker = lambda self, m: self.marks.append(m.name)  # noqa: E731

    for count in (0, 1):
        monkeypatch.setattr(torch.cuda, "device_count", lambda: count)
        items = [Item("test_library_refuses_what_its_kernels_do_not_take"), Item("test_refusals")]
        conftest.pytest_collection_modifyitems(items)
        assert [i.marks for i in items] == [["skip"] if count else [], []]


@pytest.mark.gpu
def test_tangents_and_traces_are_refused():
    """Neither passes a derivative or a call on in silence."""
    from torch.autograd import forward_ad
    x, y, w = (torch.randn(s, device="cuda") for s in ((5, 16), (5, 16), (16,)))
    call = lambda x, y, gate, w1, b1, w2, b2: gated_residual_norm(x, y, gate=gate, after=(w1, b1), before=(w2, b2))  # noqa: E731
    args = [x, y, w, w, w, w, w]
    want = call(*args)
    for i in range(7):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError):
                call(*dual)
            got = call(*(forward_ad.unpack_dual(t).primal for t in dual))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda a: gated_residual_norm(a, y)[0], (x,), check_trace=False)
