"""packed_attention against a plain fp64 implementation: forward and gradients, at the sizes and layouts where it can go wrong.

Tolerances.  eps = half a step of the operands' type (fp16 2^-11, bf16 2^-8).  Of an output o = sum p v, the store rounds by eps |o|, each
probability by eps p, so eps sum p |v| <= eps max |v|; the exact result is taken from the same rounded inputs, and fp32 sums of the lengths used here add less than eps / 4.
A gradient rounds P or dS once more per term: |d dv| <= eps (|dv| + sum P |do|), |d dq| <= eps (|dq| + scale sum |dS| |k|) and the same for dk, plus what o's
rounding in delta moves dS by: P eps sum |do o|.  The bounds are evaluated element by element from the fp64 values, times 1.5 for the fp32 sums and exp2."""
import math

import pytest
import torch

from asyrp_official_amd import AsyrpDeviceError, packed_attention

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def offsets(lens, device="cuda"):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(device)


def reference(q, k, v, lens, causal, scale, do):
    """fp64 on the CPU: outputs and their bounds (in units of eps)."""
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    G = q.shape[1] // k.shape[1]
    got = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in got.items()}
    at = 0
    for n in lens:
        r = slice(at, at + n)
        at += n
        if not n:
            continue
        for h in range(q.shape[1]):
            Q, K, V, D = q[r, h], k[r, h // G], v[r, h // G], do[r, h]
            s = scale * Q @ K.T
            if causal:
                s = s.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
            p = torch.softmax(s, 1)
            o = p @ V
            # o is an operand of the backward as stored: delta is taken from what the forward rounded
            ds = p * (D @ V.T - (D * o).sum(1, keepdim=True))
            eds = ds.abs() + p * (D * o).abs().sum(1, keepdim=True)
            got["o"][r, h], tol["o"][r, h] = o, o.abs() + p @ V.abs()
            got["dq"][r, h] = scale * ds @ K
            tol["dq"][r, h] = (scale * ds @ K).abs() + abs(scale) * eds @ K.abs()
            got["dk"][r, h // G] += scale * ds.T @ Q
            tol["dk"][r, h // G] += abs(scale) * eds.T @ Q.abs()
            got["dv"][r, h // G] += p.T @ D
            tol["dv"][r, h // G] += p.T @ D.abs()
    for n in ("dk", "dv"):
        tol[n] += got[n].abs()
    return got, tol


def check(name, got, want, tol, eps):
    err = (got.double().cpu() - want).abs()
    # 2^-24: fp16 results under its smallest normal value are rounded to its fixed smallest step
    bad = err > 1.5 * eps * tol + 2.0 ** -24
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / (eps * tol + 1e-30)).max()):.2f} half steps"


def make(T, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hk, Hk, Hq)]


def run(q, k, v, do, cu, causal, scale=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = packed_attention(q, k, v, cu, causal=causal, scale=scale)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, [q, k, v], do))))


CASES = [  # lens, Hq, Hk, D, causal
    ([1], 1, 1, 8, True), ([1, 1, 1], 2, 1, 64, False), ([31], 2, 2, 32, True), ([33, 0, 64, 65], 4, 2, 64, True), ([127, 128, 129], 2, 1, 40, False),
    ([0, 0, 77, 0], 8, 8, 64, True), ([300], 3, 1, 96, True), ([257, 3, 130], 6, 2, 128, True), ([200, 191], 2, 2, 128, False), ([197] * 3, 4, 4, 72, False),
    ([513, 1, 0, 2], 4, 1, 88, True), ([5] * 70, 1, 1, 24, False), ([640], 16, 2, 16, True), ([1100], 1, 1, 64, False), ([64, 128, 192], 2, 2, 120, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=[f"{'-'.join(map(str, c[0][:4]))}_{c[1]}x{c[2]}x{c[3]}{'c' if c[4] else ''}" for c in CASES])
def test_forward_and_gradients(case, dtype):
    lens, Hq, Hk, D, causal = case
    q, k, v, do = make(sum(lens), Hq, Hk, D, dtype)
    got = run(q, k, v, do, offsets(lens), causal)
    want, tol = reference(q, k, v, lens, causal, 1 / math.sqrt(D), do)
    for n in got:
        check(n, got[n], want[n], tol[n], HALF[dtype])
