"""The operators together, as a training step uses them: the blocks of a transformer encoder over packed sequences (attention, gated residual seams, plain matrix
products of PyTorch between them), its backward pass and AdamW's step.

Tolerance of the gradients.  The branch is f16.  From an input to an output and back a value is rounded at most about 24 times on its way (six stores per block and direction, two blocks),
by 2^-11 of its size at most each; norms and the softmax pass relative errors on without growth beyond about 2 at these widths.  24 * 2 * 2^-11 = 2.3 %
of a gradient's 2-norm bounds what that adds up to, and every gradient is compared in its 2-norm."""
import math

import pytest
import torch

from asyrp_official_amd import AdamW, gated_residual_norm, packed_attention

LENS, WIDTH, HEADS, KV = [77, 5, 0, 130, 1], 256, 4, 2
D = WIDTH // HEADS


def weights(blocks, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0, mean=0.0: torch.randn(*s, generator=g) * std + mean  # noqa: E731
    one = lambda: {"qkv": n((HEADS + 2 * KV) * D, WIDTH, std=WIDTH ** -0.5), "out": n(WIDTH, WIDTH, std=WIDTH ** -0.5), "up": n(2 * WIDTH, WIDTH, std=WIDTH ** -0.5),  # noqa: E731
                   "down": n(WIDTH, 2 * WIDTH, std=(2 * WIDTH) ** -0.5), "gate1": n(WIDTH, std=0.2, mean=0.6), "gate2": n(WIDTH, std=0.2, mean=0.6),
                   **{f"{k}{i}": n(WIDTH, std=0.1, mean=float(k == "w")) for i in (1, 2) for k in "wb"}}
    return [one() for _ in range(blocks)]


def encoder(x, blocks, cu):
    """The residual stream in float32, the branches in f16; the first seam only norms."""
    half = lambda t, w: torch.nn.functional.linear(t, w.half())  # noqa: E731
    h, n = gated_residual_norm(x, torch.zeros_like(x, dtype=torch.float16), before=(blocks[0]["w1"], blocks[0]["b1"]))
    for i, b in enumerate(blocks):
        qkv = half(n, b["qkv"])
        q, k, v = (t.view(len(x), -1, D) for t in qkv.split([HEADS * D, KV * D, KV * D], 1))
        y = half(packed_attention(q, k, v, cu, causal=True).flatten(1), b["out"])
        h, n = gated_residual_norm(h, y, gate=b["gate1"], before=(b["w2"], b["b2"]))
        y = half(torch.nn.functional.gelu(half(n, b["up"])), b["down"])
        last = i + 1 == len(blocks)
        after = blocks[i + 1] if not last else None
        h, n = gated_residual_norm(h, y, gate=b["gate2"], before=None if last else (after["w1"], after["b1"]))
    return h


def plain(x, blocks, lens):
    """The same in fp64 with PyTorch's own operations."""
    F = torch.nn.functional
    h = x
    for b in blocks:
        n = F.layer_norm(h, (WIDTH,), b["w1"], b["b1"])
        q, k, v = (t.view(len(x), -1, D).transpose(0, 1) for t in F.linear(n, b["qkv"]).split([HEADS * D, KV * D, KV * D], 1))
        k, v = k.repeat_interleave(HEADS // KV, 0), v.repeat_interleave(HEADS // KV, 0)
        o, at = [], 0
        for m in lens:
            s = q[:, at:at + m] @ k[:, at:at + m].transpose(1, 2) / math.sqrt(D)
            o.append(torch.softmax(s.masked_fill(torch.ones(m, m).triu(1).bool(), -math.inf), -1) @ v[:, at:at + m])
            at += m
        h = h + b["gate1"] * F.linear(torch.cat(o, 1).transpose(0, 1).flatten(1), b["out"])
        n = F.layer_norm(h, (WIDTH,), b["w2"], b["b2"])
        h = h + b["gate2"] * F.linear(F.gelu(F.linear(n, b["up"])), b["down"])
    return h


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_an_encoder(bits):
    blocks = weights(2)
    g = torch.Generator().manual_seed(1)
    x, target = torch.randn(sum(LENS), WIDTH, generator=g), torch.randn(sum(LENS), WIDTH, generator=g)
    ref = [{k: t.double().requires_grad_() for k, t in b.items()} for b in blocks]
    xr = x.double().requires_grad_()
    loss = ((plain(xr, ref, LENS) - target) ** 2).mean()
    loss.backward()
    own = [{k: t.cuda().requires_grad_() for k, t in b.items()} for b in blocks]
    xo = x.cuda().requires_grad_()
    cu = torch.tensor([0] + LENS).cumsum(0).to(torch.int32).cuda()
    flat = [t for b in own for t in b.values()]
    opt = AdamW(flat, lr=1e-3, state_bits=bits, max_norm=0.5)
    got = ((encoder(xo, own, cu) - target.cuda()) ** 2).mean()
    got.backward()
    assert abs(float(got.detach()) / float(loss.detach()) - 1) <= 0.023
    for a, b, name in [(xo, xr, "x")] + [(a[k], b[k], k) for a, b in zip(own, ref) for k in a]:
        rel = float((a.grad.double().cpu() - b.grad).norm() / b.grad.norm())
        assert rel <= 0.023, f"{name}: {rel:.4f}"
    # the step itself, from the gradients that it was given
    grads, before = [t.grad.double() for t in flat], [t.detach().double() for t in flat]
    opt.step()
    norm = math.sqrt(sum(float((t * t).sum()) for t in grads))
    f = min(1.0, 0.5 / (norm + 1e-6))
    assert abs(float(opt.grad_norm) / norm - 1) <= 2.0 ** -22
    for t, g0, p0 in zip(flat, grads, before):
        want = p0 * (1 - 1e-3 * 1e-2) - 1e-3 * (f * g0) / ((f * g0).abs() + 1e-8)      # the first step: m^ = g, sqrt(v^) = |g|
        # p's three roundings, and the quotient's about ten of a value that is at most 1
        assert ((t.detach().double() - want).abs() <= 2.0 ** -24 * (3 * want.abs() + 1e-3 * 10 * 2)).all()
    # and the next passes run on what it left
    for _ in range(2):
        opt.zero_grad()
        ((encoder(xo, own, cu) - target.cuda()) ** 2).mean().backward()
        opt.step()
    assert all(torch.isfinite(t).all() for t in flat)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_deltablock_step_encoder_loss_and_adamw_in_one_chain(bits):
    """The training loop's shape: one denoising step through the frozen UNet, its x0 as patches through the encoder, a loss against an embedding, back into the DeltaBlock, and AdamW on it."""
    import os
    import sys
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from oracle import sampler as osamp
    from oracle.weights import SMALL, hash_normal
    from util_models import hip_model, synthetic
    from asyrp_official_amd import denoising_step
    B, side, patch = 2, SMALL.resolution, 4
    model = hip_model(SMALL, synthetic(SMALL, 1, seed=11), 1, max_batch=B)
    for p in model.parameters():
        p.requires_grad_(False)
    delta = list(model.layer_0.parameters())
    for p in delta:
        p.requires_grad_(True)
    b, one = osamp.beta_schedule().cuda(), torch.ones(B, device="cuda")
    x = hash_normal("chain.x", (B, 3, side, side)).cuda()
    kw = dict(models=model, logvars=None, b=b, sampling_type="ddim", eta=0.0, index=0, t_edit=500, hs_coeff=(1.0, 1.0))
    lens = [(side // patch) ** 2] * B
    blocks, g = weights(2, seed=3), torch.Generator().manual_seed(4)
    embed, target = torch.randn(WIDTH, 3 * patch * patch, generator=g) * (3 * patch * patch) ** -0.5, torch.randn(B, WIDTH, generator=g)
    own, cu = [{k: t.cuda() for k, t in blk.items()} for blk in blocks], torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()

    def loss_of(x0, embed, blocks, target, run):
        rows = torch.nn.functional.unfold(x0, patch, stride=patch).transpose(1, 2).reshape(-1, 3 * patch * patch)
        h = run(torch.nn.functional.linear(rows, embed), blocks)
        return ((h.view(B, -1, WIDTH).mean(1) - target) ** 2).mean()

    opt = AdamW(delta, lr=1e-2, state_bits=bits, max_norm=1.0)
    for k in range(3):
        opt.zero_grad()
        x0 = denoising_step(x, t=one * 768.0, t_next=one * 743.0, **kw)[1]
        leaf = x0.detach().clone().requires_grad_()
        loss = loss_of(leaf, embed.cuda(), own, target.cuda(), lambda t, w: encoder(t, w, cu))
        (up,) = torch.autograd.grad(loss, leaf)
        ref = x0.detach().double().cpu().requires_grad_()
        want = loss_of(ref, embed.double(), [{n: t.double() for n, t in blk.items()} for blk in blocks], target.double(), lambda t, w: plain(t, w, lens))
        (exact,) = torch.autograd.grad(want, ref)
        assert abs(float(loss.detach()) / float(want.detach()) - 1) <= 0.023
        assert float((up.double().cpu() - exact).norm() / exact.norm()) <= 0.023
        # the chain in one piece gives the DeltaBlock what its pieces give
        pieces = torch.autograd.grad(x0, delta, up)
        x0 = denoising_step(x, t=one * 768.0, t_next=one * 743.0, **kw)[1]
        loss_of(x0, embed.cuda(), own, target.cuda(), lambda t, w: encoder(t, w, cu)).backward()
        assert all(torch.equal(p.grad, q) for p, q in zip(delta, pieces)) and any(q.any() for q in pieces)
        before = [p.detach().clone() for p in delta]
        opt.step()
        norm = math.sqrt(sum(float((q.double() ** 2).sum()) for q in pieces))
        assert abs(float(opt.grad_norm) / norm - 1) <= 2.0 ** -22
        if k == 0:
            f = min(1.0, 1.0 / (norm + 1e-6))
            for p, p0, q in zip(delta, before, pieces):
                p0, q = p0.double(), f * q.double()
                step = p0 * (1 - 1e-2 * 1e-2) - 1e-2 * q / (q.abs() + 1e-8)
                assert ((p.detach().double() - step).abs() <= 2.0 ** -24 * (3 * step.abs() + 1e-2 * 10 * 2)).all()
        assert all(torch.isfinite(p).all() for p in delta)
