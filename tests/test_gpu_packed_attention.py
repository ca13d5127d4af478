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


# ---- two parts of the queries per key tile, more than 64 sequences, other layouts -----------------------------------------------------------
LONG = [([1500], 4, 1, 128, True), ([2600], 1, 1, 64, True), ([0, 2300, 31], 2, 1, 128, False), ([1100, 700], 8, 1, 96, False), ([3] * 80 + [90], 2, 1, 64, True), ([1, 0] * 50, 2, 2, 32, True), ([130] * 66, 1, 1, 128, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LONG, ids=[f"{len(c[0])}x{c[0][0]}_{c[1]}x{c[2]}x{c[3]}" for c in LONG])
def test_long_and_many(case):
    lens, Hq, Hk, D, causal = case
    q, k, v, do = make(sum(lens), Hq, Hk, D, torch.bfloat16, seed=1)
    got = run(q, k, v, do, offsets(lens), causal)
    want, tol = reference(q, k, v, lens, causal, 1 / math.sqrt(D), do)
    for n in got:
        check(n, got[n], want[n], tol[n], HALF[torch.bfloat16])


@pytest.mark.gpu
def test_long_causal_sequences_dealt_out_beyond_the_cus():
    """Over 256 workgroups of 128 rows in sequences of a mean length over 2560: the keys of a query tile go to two of them."""
    lens = [2700, 2500]
    q, k, v, do = make(sum(lens), 7, 1, 32, torch.float16, seed=2)
    got = run(q, k, v, do, offsets(lens), True)
    want, tol = reference(q, k, v, lens, True, 1 / math.sqrt(32), do)
    for n in got:
        check(n, got[n], want[n], tol[n], HALF[torch.float16])


@pytest.mark.gpu
def test_views_of_a_fused_projection_and_odd_layouts_read_the_same():
    lens, H, K, D = [60, 1, 131], 4, 2, 64
    T = sum(lens)
    q, k, v, do = make(T, H, K, D, torch.float16, seed=2)
    want = run(q, k, v, do, offsets(lens), True)
    qkv = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    views = [t.view(T, -1, D) for t in qkv.split([H * D, K * D, K * D], 1)]                    # rows 512 values apart, read in place
    apart = [torch.empty(t.shape[1], T, D, device="cuda", dtype=t.dtype).transpose(0, 1).copy_(t) for t in (q, k, v)]    # heads outside
    shifted = [torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:].view_as(t).copy_(t) for t in (q, k, v)]      # address of 2 mod 16
    last = [torch.empty(*t.shape, 2, device="cuda", dtype=t.dtype)[..., 0].copy_(t) for t in (q, k, v)]                  # last axis strided
    for other in (views, apart, shifted, last):
        got = run(*other, do.transpose(0, 1).contiguous().transpose(0, 1), offsets(lens), True)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    one = run(q[:1, :1].expand(1, 1, D), k[:1, :1], v[:1, :1], do[:1, :1], offsets([1]), True)  # axes of one
    assert torch.equal(one["o"][0, 0], v[0, 0])


@pytest.mark.gpu
def test_rows_of_no_sequence_stay_zero_or_untouched():
    q, k, v, do = make(700, 2, 1, 64, torch.bfloat16, seed=3)
    for t in (q, k, v, do):
        t[300:] = math.nan                                             # nothing of these rows may be seen
    got = run(q, k, v, do, offsets([100, 0, 200]), True)
    # (how the work is dealt out goes by the number of rows, so the bits may differ from those of the 300 rows alone; the values' bounds do not)
    want, tol = reference(q[:300], k[:300], v[:300], [100, 0, 200], True, 1 / 8, do[:300])
    for n in got:
        check(n, got[n][:300], want[n], tol[n], HALF[torch.bfloat16])
        assert not got[n][300:].any()
    out = torch.full_like(q, 7.0)
    with torch.no_grad():
        assert packed_attention(q, k, v, offsets([100, 0, 200]), causal=True, out=out) is out
    assert torch.equal(out[:300], got["o"][:300]) and (out[300:] == 7.0).all()
    none = run(q, k, v, do, offsets([0, 0]), False)                    # no rows in any sequence
    assert not any(t.any() for t in none.values())
    assert packed_attention(q[:0], k[:0], v[:0], offsets([0])).shape == (0, 2, 64)
    nothing = run(q[:0], k[:0], v[:0], do[:0], offsets([0]), True)
    assert all(t.shape[0] == 0 for t in nothing.values())


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_sequence():
    lens = [65, 64, 130]
    q, k, v, do = make(sum(lens), 2, 2, 64, torch.float16, seed=4)
    want = run(q, k, v, do, offsets(lens), True)
    v[100], k[70] = math.inf, math.nan                                 # in the second sequence
    got = run(q, k, v, do, offsets(lens), True)
    for n in want:
        assert torch.equal(got[n][:65], want[n][:65]) and torch.equal(got[n][129:], want[n][129:])
    # keys of minus infinity in a whole tile take no part
    q, k, v, do = make(200, 1, 1, 64, torch.float16, seed=5)
    q[..., 0], k[:150, 0, 0] = 1.0, -math.inf
    with torch.no_grad():
        o = packed_attention(q, k, v, offsets([200]))
        assert torch.allclose(o, packed_attention(q, k[150:].repeat(4, 1, 1), v[150:].repeat(4, 1, 1), offsets([200])), rtol=2e-3, atol=2e-3)


@pytest.mark.gpu
def test_offsets_that_fall_or_pass_the_end_touch_nothing_outside():
    pad = 64
    big = [torch.zeros(300 + 2 * pad, 2, 64, device="cuda", dtype=torch.float16) for _ in range(4)]
    for t, s in zip(big, make(300, 2, 2, 64, torch.float16, seed=6)):
        t[pad:-pad] = s
    out = torch.full((300 + 2 * pad, 2, 64), 5.0, device="cuda", dtype=torch.float16)
    for cu in ([0, 1000], [-5, 300], [200, 100, 300], [0, 2 ** 31 - 1, -2 ** 31]):
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        with torch.no_grad():
            packed_attention(*(t[pad:-pad] for t in big[:3]), cu, out=out[pad:-pad])
        run(*(t[pad:-pad] for t in big), cu, True)
        assert (out[:pad] == 5.0).all() and (out[-pad:] == 5.0).all()


@pytest.mark.gpu
def test_streams_repeats_and_graph_replays_agree():
    lens = [257, 1, 600]
    q, k, v, do = make(sum(lens), 8, 2, 128, torch.bfloat16, seed=7)
    cu = offsets(lens)
    want = run(q, k, v, do, cu, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, do, cu, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g = run(*leaves, do, cu, True)                                 # warm up on the stream of the capture
        del g
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        o = packed_attention(*leaves, cu, causal=True)
        caught = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
        del o
    for i in range(3):
        with torch.no_grad():
            for t, s in zip(leaves, (q, k, v)):
                t.copy_(s * (1 + i))
        eager = run(*(s * (1 + i) for s in (q, k, v)), do, cu, True)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(caught[n], eager[n]) for n in eager), i


@pytest.mark.gpu
def test_offsets_over_32_bits():
    """Rows 2^23 values apart: the last ones lie behind 4 G values, read in place."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 30 GB")
    T, D = 520, 32
    base = torch.empty((T - 1) * 2 ** 23 + D, device="cuda", dtype=torch.float16)
    wide = base.as_strided((T, 1, D), (2 ** 23, D, 1))
    q, k, v, do = make(T, 1, 1, D, torch.float16, seed=8)
    wide.copy_(k)
    with torch.no_grad():
        want = packed_attention(q, k, v, offsets([3, 517]), causal=True)
        assert torch.equal(packed_attention(q, wide, v, offsets([3, 517]), causal=True), want)
        assert torch.equal(packed_attention(wide, k, v, offsets([3, 517])), packed_attention(k, k, v, offsets([3, 517])))
        packed_attention(q, k, v, offsets([3, 517]), causal=True, out=wide)
        assert torch.equal(wide, want)


# ---- refusals (no GPU work) ---------------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 1, 8, dtype=torch.float16)
    with pytest.raises(AsyrpDeviceError):
        packed_attention(t, t, t, torch.tensor([0, 4], dtype=torch.int32))


def test_library_refuses_what_its_kernels_do_not_take():
    from asyrp_official_amd import _lib
    lib = _lib.load()

    def call(T=4, n=1, H=2, K=1, D=64, dtype=_lib.F16, scale=1.0, sq=(128, 64), ptr=4096):
        spec = _lib.PACKED_ATTENTION.pack(T, n, H, K, D, 0, dtype, scale, *sq, 64, 64, 64, 64, 128, 64, 128, 64)
        f = lib.asyrp_packed_attention_forward(0, spec, ptr, ptr, ptr, 4096, ptr, None, None, 4096, 1, None)
        b = lib.asyrp_packed_attention_backward(0, spec, ptr, ptr, ptr, 4096, ptr, 4096, None, ptr, 4096, ptr, ptr, ptr, None)
        assert f == b
        return f

    for bad in (dict(D=4), dict(D=60), dict(D=136), dict(K=3), dict(H=0), dict(n=0), dict(T=-1), dict(T=2 ** 31), dict(dtype=_lib.F32), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=math.nan), dict(scale=math.inf), dict(sq=(100, 64)), dict(sq=(2 ** 24, 64)), dict(sq=(-128, 64)), dict(ptr=4098), dict(ptr=None)):
        assert call(**bad) == -1, bad
        assert b"packed attention" in lib.asyrp_last_error()
    assert call(n=2 ** 23, H=2) == -1 and call(n=2 ** 22, H=8, K=2) == -1       # more workgroups than a launch takes
    assert call(T=0) == 0                                              # nothing to do, nothing launched
    assert lib.asyrp_packed_attention_forward(0, None, 4096, 4096, 4096, 4096, 4096, None, None, 4096, 1, None) == -1
    assert lib.asyrp_packed_attention_workspace(None, 0) == -1


@pytest.mark.gpu
def test_refusals():
    q, k, v, _ = make(8, 4, 2, 16, torch.float16)
    cu = offsets([8])
    ok = lambda **kw: packed_attention(**{**dict(q=q, k=k, v=v, cu_seqlens=cu), **kw})  # noqa: E731
    assert ok().shape == q.shape
    for kw in (dict(q=q.float()), dict(k=k.bfloat16()), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:1]), dict(cu_seqlens=cu[None]), dict(q=q[0]), dict(k=k[:7]), dict(v=v[:, :1]),
               dict(k=k[:, :0], v=v[:, :0]), dict(q=q[:, :3]), dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
               dict(out=q[:4]), dict(out=q.float()), dict(out=torch.empty(16, 4, 8, device="cuda", dtype=q.dtype).transpose(0, 2)),
               dict(q=q.clone().requires_grad_(), out=torch.empty_like(q))):
        with pytest.raises(ValueError):
            ok(**kw)
    for kw in (dict(q=q.cpu()), dict(cu_seqlens=cu.cpu()), dict(out=q.cpu())):
        with pytest.raises(AsyrpDeviceError):
            ok(**kw)


@pytest.mark.gpu
def test_out_beside_and_over_its_inputs():
    T, H, D = 70, 4, 16
    q, k, v, _ = make(T, H, 2, D, torch.float16)
    cu = offsets([30, 40])
    want = packed_attention(q, k, v, cu, causal=True)
    fused = torch.cat([q, k, v, torch.zeros_like(q)], 1)                  # [T, 4 + 2 + 2 + 4, D]
    qf, kf, vf, of = fused.split([4, 2, 2, 4], 1)
    assert packed_attention(qf, kf, vf, cu, causal=True, out=of) is of and torch.equal(of, want)
    planes = torch.stack([q, q]).transpose(1, 2).contiguous().transpose(1, 2)        # heads in front of rows, q behind out
    assert torch.equal(packed_attention(planes[1], kf, vf, cu, causal=True, out=planes[0]), want)
    blocks = torch.cat([q, q]).transpose(0, 1).contiguous().transpose(0, 1)          # a head's block holds the rows of q, then of out
    assert torch.equal(packed_attention(blocks[:T], kf, vf, cu, causal=True, out=blocks[T:]), want)
    long = torch.cat([q, q])
    twice = torch.empty(T * H * D, device="cuda", dtype=q.dtype).as_strided((T, H, D), (D, D, 1))
    for kw in (dict(q=qf, out=qf), dict(q=long[:T], out=long[1:T + 1]), dict(q=long[1:T + 1], out=long[:T]), dict(q=q, k=fused[:, :2], out=fused[:, 1:5]),
               dict(q=q, k=fused[:, 4:6], out=fused[:, 1:5]), dict(q=q, out=twice), dict(q=q, v=of[:, 2:], out=of)):
        with pytest.raises(ValueError, match="overlap"):
            packed_attention(**{**dict(k=k, v=v, cu_seqlens=cu), **kw})


def test_reference_gradients_against_differences():
    """The reference itself, in fp64 on the CPU."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(9, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    lens = [5, 0, 4]
    for causal in (True, False):
        f = lambda *a: float((reference(*a, lens, causal, 0.3, do)[0]["o"] * do).sum())  # noqa: E731
        got, _ = reference(q, k, v, lens, causal, 0.3, do)
        for i, n in enumerate(("dq", "dk", "dv")):
            d = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)
            up, down = ([t + s * 1e-6 * d if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
            slope = (f(*up) - f(*down)) / 2e-6
            assert abs(slope - float((got[n] * d).sum())) <= 1e-7 * (1 + abs(slope))


@pytest.mark.gpu
def test_autograd_sees_that_out_was_written():
    q, k, v, _ = make(40, 2, 1, 16, torch.float16)
    cu, w = offsets([40]), torch.ones(40, 2, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    base = torch.zeros(40, 4, 16, device="cuda", dtype=torch.float16)
    for buf in (torch.zeros_like(q), base[:, 1:3]):                    # a buffer, and a part of one
        packed_attention(q, k, v, cu, out=buf)
        loss, before = (buf * w).sum(), buf._version                   # keeps buf for its backward
        with torch.no_grad():
            packed_attention(q, k, v, cu, causal=True, out=buf)
        assert buf._version == before + 1
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    leaf = torch.zeros_like(q).requires_grad_()
    with pytest.raises(ValueError, match="graph"):
        packed_attention(q, k, v, cu, out=leaf)
    with pytest.raises(ValueError, match="graph"):
        packed_attention(q, k, v, cu, out=leaf * 1)
    want = packed_attention(q, k, v, cu)
    with torch.no_grad():                                              # as other operations may write to a leaf there
        before = leaf._version
        assert torch.equal(packed_attention(q, k, v, cu, out=leaf), want) and leaf._version == before + 1
    with torch.inference_mode():                                       # tensors made here have no version
        buf = torch.empty_like(q)
        assert torch.equal(packed_attention(q, k, v, cu, out=buf), want)


@pytest.mark.gpu
def test_tangents_and_traces_are_refused():
    from torch.autograd import forward_ad
    q, k, v, _ = make(12, 2, 2, 16, torch.float16)
    cu = offsets([12])
    for i in range(3):
        with forward_ad.dual_level():
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((q, k, v))]
            with pytest.raises(RuntimeError):
                packed_attention(*args, cu)
            with torch.no_grad(), pytest.raises(RuntimeError):
                packed_attention(*args, cu, out=torch.empty_like(q))
            assert torch.equal(packed_attention(*(forward_ad.unpack_dual(t).primal for t in args), cu), packed_attention(q, k, v, cu))
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda a: packed_attention(a, k, v, cu), (q,), check_trace=False)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("size", [1e4, 1e5, 1e6, 2e7, 1e8])
def test_large_scores_of_equal_keys(size, dtype, D):
    """Rows that see one key, or several equal ones: probabilities are 1 / n whatever the scores, in the backward pass too.  (Score sums of the same numbers in the same order are equal to the bit.)"""
    lens = [1] * 20 + [2, 4] * 6 + [130]
    q, k, v, do = make(sum(lens), 2, 1, D, dtype, seed=3)
    c = (size / math.log2(math.e) / math.sqrt(D)) ** 0.5
    at = 0
    for n in lens:
        k[at:at + n] = k[at:at + 1].sign() * (c * (1 + k[at:at + 1].abs() / 8)).to(dtype)
        q[at:at + n] = (k[at:at + n].expand(n, 2, D).float() * (1 + torch.arange(n, device="cuda")[:, None, None] / 256)).to(dtype)
        at += n
    for causal in (True, False):
        got = run(q, k, v, do, offsets(lens), causal)
        want, tol = reference(q, k, v, lens, causal, 1 / math.sqrt(D), do)
        for m in got:
            check(m, got[m], want[m], tol[m], HALF[dtype])


# ---- other sizes of scores and gradients -------------------------------------------------------------------------------------------------------
def exact(q, k, v, causal, scale, do, eps):
    """One sequence in fp64: results, bounds on each element's error, and what rounding one by one adds up to as a root of a sum of squares.

    As above, with the fp32 scores' own errors: a score is a sum of D products, off by at most D 2^-24 of the sum A of their sizes, scale and its product with
    the score add 4 roundings, and numerator and denominator of a probability both have it: P is off by rho = 2 (D + 4) 2^-24 max A of its value."""
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    n, G, D = q.shape[0], q.shape[1] // k.shape[1], q.shape[2]
    got = {m: torch.zeros_like(t) for m, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    tol, sq = ({m: torch.zeros_like(t) for m, t in got.items()} for _ in range(2))
    for h in range(q.shape[1]):
        Q, K, V, g, j = q[:, h], k[:, h // G], v[:, h // G], do[:, h], h // G
        s, A = scale * Q @ K.T, scale * Q.abs() @ K.abs().T
        if causal:
            late = torch.ones(n, n).triu(1).bool()
            s, A = s.masked_fill(late, -math.inf), A.masked_fill(late, 0.0)
        rho = 2 * (D + 4) * 2.0 ** -24 * A.amax(1, keepdim=True)
        p = torch.softmax(s, 1)
        o, dp = p @ V, g @ V.T
        ds = p * (dp - (g * o).sum(1, keepdim=True))
        eds = eps * (ds.abs() + p * (g * o).abs().sum(1, keepdim=True)) + rho * (ds.abs() + p * (p * dp.abs()).sum(1, keepdim=True))
        got["o"][:, h], tol["o"][:, h] = o, eps * o.abs() + (eps + rho) * (p @ V.abs())
        got["dq"][:, h], tol["dq"][:, h], sq["dq"][:, h] = scale * ds @ K, scale * (eds @ K.abs()), scale ** 2 * eps ** 2 * (ds ** 2 @ K ** 2)
        got["dk"][:, j] += scale * ds.T @ Q
        tol["dk"][:, j] += scale * (eds.T @ Q.abs())
        sq["dk"][:, j] += scale ** 2 * eps ** 2 * (ds.T ** 2 @ Q ** 2)
        got["dv"][:, j] += p.T @ g
        tol["dv"][:, j] += ((eps + rho) * p).T @ g.abs()
        sq["dv"][:, j] += eps ** 2 * (p.T ** 2 @ g ** 2)
    for m in ("dq", "dk", "dv"):
        tol[m] += eps * got[m].abs()
    return got, tol, sq


RAMPS = [(400, 2, 1, 64, True, 0.125), (400, 2, 2, 64, False, 0.125), (300, 2, 1, 128, True, 0.25), (257, 3, 3, 96, False, 0.05), (333, 2, 1, 40, True, 1.5), (2600, 1, 1, 64, True, 0.125),
         (2600, 1, 1, 64, False, 0.125), (2100, 2, 1, 128, True, 0.125), (2100, 1, 1, 128, False, 0.125)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", RAMPS, ids=[f"{c[0]}_{c[1]}x{c[2]}x{c[3]}{'c' if c[4] else ''}" for c in RAMPS])
def test_scores_that_climb_and_fall_along_the_keys(case, dtype):
    """Scores from -60 to 60 and beyond: every second query's climb from key to key, so that its maximum moves tile after tile (and, where the keys are dealt out, lies in
    the last part), the others' fall, so that it lies in the first.  Scales other than the default."""
    n, H, K, D, causal, scale = case
    q, k, v, do = make(n, H, K, D, torch.float32, seed=n)
    q, k = 0.3 * q, 0.3 * k
    q[..., 0] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 8.0, -8.0)[:, None]
    k[..., 0] = torch.linspace(-60, 60, n, device="cuda")[:, None] / (8 * scale)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    got = run(q, k, v, do, offsets([n]), causal, scale)
    want, tol, _ = exact(q, k, v, causal, scale, do, HALF[dtype])
    for m in got:
        check(m, got[m], want[m], tol[m], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, "mixed"])
def test_small_gradients_of_long_sequences_in_f16(size, D, causal):
    """Gradients of a mean loss.  Every term of a sum is rounded by itself, by at most half a step of f16 relative to it, and the stored result once more, or by half its smallest step
    (2^-25): of independent errors the squares add up, and 1.5 times the root bounds the 2-norm of all of them (an error is uniform up to its bound, so its root mean square is 1 / sqrt(3) of it)."""
    n, eps = 3000, 2.0 ** -11
    q, k, v, do = make(n, 1, 1, D, torch.float16, seed=4)
    sizes = 10.0 ** (-6 * torch.rand(n, 1, 1, generator=torch.Generator().manual_seed(0))).cuda() if size == "mixed" else size
    do = (do.float() * sizes).half()
    got = run(q, k, v, do, offsets([n]), causal)
    want, _, sq = exact(q, k, v, causal, 1 / math.sqrt(D), do, eps)
    for m in ("dq", "dk", "dv"):
        bound = (sq[m] + (eps * want[m]) ** 2 + 2.0 ** -50).sum().sqrt()
        err = (got[m].double().cpu() - want[m]).norm()
        assert err <= 1.5 * bound, f"{m}: {float(err / bound):.2f} of the bound, {float(err / want[m].norm()):.2e} of the gradient"


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_whose_inner_values_pass_f16(D):
    """dS is over 65504 here, dq and dk are not; sizes grow along the rows of the first sequence, so that what went before is small beside what follows."""
    lens = [200] + [4] * 16
    q, k, v, do = make(sum(lens), 2, 1, D, torch.float32, seed=5)
    grow = torch.cat([torch.logspace(-2, 1, 200), torch.full((64,), 10.0)]).cuda()[:, None, None]
    q, k, v, do = (t.half() for t in (0.02 * q, 0.02 * k, 0.8 * v * grow, 800 * do * grow))
    dp = do[-4:, 0].double() @ v[-4:, 0].double().T                    # of the last sequence, whose probabilities are all close to 1 / 4
    assert ((dp - dp.mean(1, keepdim=True)) / 4).abs().max() > 70000
    for causal in (True, False):
        got = run(q, k, v, do, offsets(lens), causal)
        want, tol = reference(q, k, v, lens, causal, 1 / math.sqrt(D), do)
        assert max(float(want[m].abs().max()) for m in want) < 60000
        for m in got:
            check(m, got[m], want[m], tol[m], HALF[torch.float16])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_outputs_among_the_smallest_of_f16(D):
    """Outputs of about 1e-6 (f16 has steps of 6e-8 there), keys of about 40: rowsum(do * o) is to be that of the unrounded output here too."""
    q, k, v, do = make(400, 2, 1, D, torch.float32, seed=12)
    q, k, v, do = (t.half() for t in (0.02 * q, 40 + k, 1e-5 * v, do))
    for causal in (True, False):
        got = run(q, k, v, do, offsets([400]), causal)
        want, tol, _ = exact(q, k, v, causal, 1 / math.sqrt(D), do, HALF[torch.float16])
        for m in got:
            check(m, got[m], want[m], tol[m], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [500, 3000])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_a_heavy_key_whose_value_is_nothing(n, causal):
    """The first key takes all but 1.3e-6 per key of every query and has a value of zero: outputs are sums of what the others get, all of one size, so that roundings do not average out."""
    q, k, v, do = make(n, 1, 1, 64, torch.float16, seed=11)
    q.zero_()
    k.zero_()
    q[..., 0], k[0, 0, 0] = 8.0, 13.55
    v = v.abs()
    v[0] = 0
    got = run(q, k, v, do, offsets([n]), causal)
    want, tol, _ = exact(q, k, v, causal, 0.125, do, HALF[torch.float16])
    for m in got:
        check(m, got[m], want[m], tol[m], 1.0)


def test_launch_limits_are_those_of_each_direction():
    """The workspace query launches nothing.  2^32 - 1 threads are one launch's most: 256 a workgroup of 128 rows and query head (forward, dq), or of a key / value head (dk and dv of heads up to 64),
    512 of one of wider heads; every sequence may need a workgroup of its own."""
    from asyrp_official_amd import _lib
    lib = _lib.load()
    most = 2 ** 24 - 1                                                  # workgroups of 256 threads, one of which the launch keeps for itself

    def words(n, H, K, D, backward):
        return lib.asyrp_packed_attention_workspace(_lib.PACKED_ATTENTION.pack(0, n, H, K, D, 0, _lib.F16, 1.0, *([H * D, D] * 5)), backward)

    for D, H, K, backward, n in ((64, 1, 1, 0, most - 1), (128, 1, 1, 0, most - 1), (64, 1, 1, 1, most - 1), (128, 1, 1, 1, 2 ** 23 - 2), (64, 4, 4, 0, 2 ** 22 - 2), (128, 4, 1, 1, 2 ** 22 - 2),
                                 (128, 4, 4, 1, 2 ** 21 - 2), (128, 2, 1, 1, 2 ** 23 - 2)):
        assert words(n, H, K, D, backward) >= 0, (D, H, K, backward)
        assert words(n + 1, H, K, D, backward) == -1, (D, H, K, backward)
        assert b"too many for one launch" in lib.asyrp_last_error()
    assert words(2 ** 31 - 1, 2 ** 31 - 1, 1, 8, 0) == -1


@pytest.mark.gpu
def test_bad_offsets_touch_nothing_around_the_gradients_and_the_workspace():
    """The C entries with every output in the middle of a larger buffer."""
    from asyrp_official_amd import _lib
    lib, T, H, K, pad = _lib.load(), 1500, 2, 1, 4096
    for D, nseq in ((64, 1), (128, 1), (64, 70), (128, 2)):
        q, k, v, do = make(T, H, K, D, torch.float16, seed=9)
        spec = _lib.PACKED_ATTENTION.pack(T, nseq, H, K, D, 1, _lib.F16, 0.125, *(H * D, D), *(K * D, D), *(K * D, D), *(H * D, D), *(H * D, D))
        words = [lib.asyrp_packed_attention_workspace(spec, b) for b in (0, 1)]
        assert min(words) >= 0

        def room(numel, dtype):
            t = torch.full((numel + 2 * pad,), 5.0, device="cuda", dtype=dtype)
            return t, t[pad:pad + numel].data_ptr()

        outs = {m: room(T * h * D, torch.float16) for m, h in (("out", H), ("rest", H), ("dq", H), ("dk", K), ("dv", K))}
        stats, ws = room(2 * H * T, torch.float32), [room(max(4, w), torch.float32) for w in words]
        for cu in ([0] * nseq + [2000], [-5] + [1500] * nseq, [900, 100] + [1400] * nseq, [0, 2 ** 31 - 1] + [-2 ** 31] * nseq, [1450] + [10] * nseq, [-2 ** 31] * (nseq + 1)):
            cu = torch.tensor(cu[:nseq + 1], dtype=torch.int32, device="cuda")
            stream = torch.cuda.current_stream().cuda_stream
            for fill in (0, 1):
                assert lib.asyrp_packed_attention_forward(0, spec, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), outs["out"][1], stats[1], outs["rest"][1], ws[0][1], fill, stream) == 0
            assert lib.asyrp_packed_attention_backward(0, spec, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), outs["out"][1], stats[1], outs["rest"][1], do.data_ptr(), ws[1][1],
                                                       outs["dq"][1], outs["dk"][1], outs["dv"][1], stream) == 0
            torch.cuda.synchronize()
            for t in [t for t, _ in outs.values()] + [stats[0]] + [t for t, _ in ws]:
                assert (t[:pad] == 5.0).all() and (t[-pad:] == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("D", [32, 128])
def test_thousands_of_sequences_read_as_in_small_batches(D, causal):
    """Every sequence by itself gives the same bits: in calls of up to 50 sequences and in one of 5000, empty ones, rows in front of the first and behind the last among them."""
    g = torch.Generator().manual_seed(0)
    lens = torch.tensor([0, 1, 1, 2, 3, 7, 64, 127, 128, 129, 200])[torch.randint(0, 11, (5000,), generator=g)].tolist()
    lens[:3], lens[70:140], lens[-2:] = [0, 130, 0], [0] * 70, [1, 0]
    ahead, T = 300, sum(lens)
    q, k, v, do = make(ahead + T + 500, 2, 1, D, torch.float16, seed=1)
    got = run(q, k, v, do, offsets(lens) + ahead, causal)
    at = 0
    for i in range(0, len(lens), 50):
        part = lens[i:i + 50]
        r = slice(ahead + at, ahead + at + sum(part))
        at += sum(part)
        want = run(q[r], k[r], v[r], do[r], offsets(part), causal)
        for m in got:
            assert torch.equal(got[m][r], want[m]), (m, i)
    for m in got:
        assert not got[m][:ahead].any() and not got[m][ahead + T:].any()


@pytest.mark.gpu
def test_the_time_of_many_sequences_goes_with_their_number():
    """200000 sequences of one row, both directions: some milliseconds, where every workgroup reading all offsets up to its own took 200 in the forward alone."""
    n = 200_000
    q, k, v, do = make(n, 1, 1, 64, torch.float16)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    got = run(q, k, v, do, cu, True)
    assert torch.equal(got["o"], v) and torch.equal(got["dv"], do)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    run(q, k, v, do, cu, True)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 50
