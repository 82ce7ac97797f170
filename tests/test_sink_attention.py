"""Attention with a sliding window and sinks (ops.attention_packed(window=, sinks=)): query q sees key k iff k <= q and
(q - k < window or k < sinks).  Forward and backward against the definition in 64 bits.

Tolerances (bf16 tensors, half a step = 2^-8 relative; 32-bit sums and exponentials: 2^-12 of the summed magnitudes):
  o    every p is rounded once, the output once:             2^-8 (sum p |v| + |o|)
  dS   = p (dP - delta), delta granted a rounded output:     p sum |do| tol_o, and the rounding of dS 2^-8 |dS|
       (the kernels keep 8 more bits of it, which has tests of its own below)
  dQ, dK  scale sum tol_dS |k|, |q|, the output's rounding 2^-8
  dV   2^-8 (sum p |do| + |dV|)"""
import math

import pytest
import torch

from finetune_controller_amd import ops
from finetune_controller_amd.ops.attention import RopeGrad

BF, H8, SL = torch.bfloat16, 2.0 ** -8, 2.0 ** -12


def _seen(S, window, sinks):
    i = torch.arange(S)
    d = i[:, None] - i[None, :]
    return (d >= 0) & ((d < window) | (i[None, :] < sinks))


def _definition(qkv, do, B, S, H, KV, D, window, sinks, scale):
    """64-bit o and dqkv with their tolerances: (o, tol_o, g, tol_g), [B*S, ...]."""
    x = qkv.detach().cpu().double()[:, :(H + 2 * KV) * D].view(B, S, H + 2 * KV, D)
    dO = do.detach().cpu().double().view(B, S, H, D)
    seen = _seen(S, window, sinks)
    o, to = torch.zeros_like(dO), torch.zeros_like(dO)
    g, tg = torch.zeros_like(x), torch.zeros_like(x)
    for b in range(B):
        for h in range(H):
            kh, vh = H + h // (H // KV), H + KV + h // (H // KV)
            q, k, v, d = x[b, :, h], x[b, :, kh], x[b, :, vh], dO[b, :, h]
            p = torch.softmax((q @ k.T * scale).masked_fill(~seen, -math.inf), 1)
            oh, pv = p @ v, p @ v.abs()
            tol_o = H8 * (pv + oh.abs()) + SL * pv
            dP = d @ v.T
            delta = (d * oh).sum(1, keepdim=True)
            dS = p * (dP - delta)
            tS = p * ((d.abs() * tol_o).sum(1, keepdim=True) + SL * (d.abs() @ v.abs().T + delta.abs())) + H8 * dS.abs()
            o[b, :, h], to[b, :, h] = oh, tol_o
            g[b, :, h], tg[b, :, h] = scale * dS @ k, scale * tS @ k.abs()
            g[b, :, kh] += scale * dS.T @ q
            tg[b, :, kh] += scale * tS.T @ q.abs()
            g[b, :, vh] += p.T @ d
            tg[b, :, vh] += (H8 + SL) * p.T @ d.abs()
    tg += H8 * g.abs()
    return o.view(B * S, -1), to.view(B * S, -1), g.view(B * S, -1), tg.view(B * S, -1)


def _inputs(B, S, H, KV, D, seed=0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B * S, (H + 2 * KV) * D, generator=g)
    qkv[:, :(H + KV) * D] *= 1.3
    return qkv.to(dtype), torch.randn(B * S, H * D, generator=g).to(dtype)


def _close(got, want, tol):
    err = (got.detach().double().cpu() - want).abs()
    assert err.isfinite().all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())


# ---------------------------------------------------------------- torch path
@pytest.mark.parametrize("S,window,sinks", [(1, 1, 1), (9, 3, 2), (20, 1, 4), (20, 7, 30), (17, 40, 3), (16, 5, 0)])
def test_torch_path_matches_the_definition(S, window, sinks):
    B, H, KV, D = 2, 4, 2, 8
    qkv, do = _inputs(B, S, H, KV, D, dtype=torch.float64)
    qkv.requires_grad_()
    o = ops.attention_packed(qkv, B, S, H, KV, D, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, qkv, do)
    wo, _, wg, _ = _definition(qkv, do, B, S, H, KV, D, window, sinks, D ** -0.5)
    torch.testing.assert_close(o.detach(), wo, atol=1e-12, rtol=1e-12)
    torch.testing.assert_close(g, wg, atol=1e-12, rtol=1e-12)
    torch.testing.assert_close(ops.attention_reference(qkv.detach(), B, S, H, KV, D, window=window, sinks=sinks).double(), wo,
                               atol=1e-5, rtol=1e-5)


def test_gradient_against_differences():
    B, S, H, KV, D = 1, 7, 2, 1, 4
    qkv, _ = _inputs(B, S, H, KV, D, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda x: ops.attention_packed(x, B, S, H, KV, D, window=2, sinks=1), qkv.requires_grad_())


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(dev):
    qkv = torch.zeros(8, 4 * 64, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="negative"):
        ops.attention_packed(qkv, 1, 8, 2, 1, 64, window=4, sinks=-1)
    with pytest.raises(ValueError, match="causal"):
        ops.attention_packed(qkv, 1, 8, 2, 1, 64, False, window=4, sinks=1)
    docs = ops.segments_from_eos(torch.zeros(1, 8, dtype=torch.long, device=dev), 5)
    with pytest.raises(ValueError, match="one document"):
        ops.attention_packed(qkv, 1, 8, 2, 1, 64, window=4, sinks=1, docs=docs)
    if dev == "cuda":
        with pytest.raises(ValueError, match="head_dim"):
            ops.attention_packed(torch.zeros(8, 4 * 136, dtype=BF, device=dev), 1, 8, 2, 1, 136, window=4, sinks=1)
    for scale in (0.0, -0.1, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            ops.attention_packed(qkv, 1, 8, 2, 1, 64, window=4, sinks=1, scale=scale)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("B,S", [(0, 4), (2, 0)])
def test_nothing_to_attend_to(dev, B, S):
    x = torch.zeros(B * S, 4 * 64, dtype=BF, device=dev, requires_grad=True)
    o = ops.attention_packed(x, B, S, 2, 1, 64, window=3, sinks=1)
    (g,) = torch.autograd.grad(o.sum(), x)
    assert o.shape == (0, 128) and g.shape == x.shape


# ---------------------------------------------------------------- kernels
SHAPES = [  # B, S, H, KV, D, window, sinks
    (1, 1, 1, 1, 128, 1, 1),
    (2, 33, 2, 1, 64, 5, 1),
    (1, 64, 2, 2, 128, 64, 7),
    (1, 129, 4, 1, 64, 1, 64),
    (2, 257, 2, 1, 128, 17, 4),
    (1, 300, 3, 3, 64, 100, 65),
    (1, 511, 4, 2, 128, 128, 3),
    (3, 640, 2, 1, 64, 33, 33),
    (1, 1025, 2, 1, 128, 300, 300),
    (1, 1300, 2, 2, 128, 40, 260),
    (1, 600, 6, 3, 80, 50, 5),
    (2, 77, 2, 1, 32, 9, 2),
    (1, 700, 8, 1, 128, 200, 40),  # few key blocks: swept in parts
    (2, 530, 4, 2, 64, 530, 3),
    (16, 260, 32, 16, 64, 100, 5),  # many: each by one workgroup
    (5, 260, 20, 4, 128, 150, 5),  # query blocks past one a compute unit
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,KV,D,window,sinks", SHAPES)
def test_kernels(B, S, H, KV, D, window, sinks):
    qkv, do = _inputs(B, S, H, KV, D, seed=S)
    x = qkv.cuda().requires_grad_()
    scale = 0.7 / math.sqrt(D)
    o = ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks, scale=scale)
    (g,) = torch.autograd.grad(o, x, do.cuda())
    wo, to, wg, tg = _definition(qkv, do, B, S, H, KV, D, window, sinks, scale)
    assert o.dtype == BF and g.dtype == BF and o.shape == (B * S, H * D) and g.shape == qkv.shape
    _close(o, wo, to)
    _close(g, wg, tg)
    # against differences of the 64-bit function, along one direction
    d = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(1)).double()
    e, xd = 1e-6, qkv.double()
    up, dn = (_definition(xd + t * e * d, do, B, S, H, KV, D, window, sinks, scale)[0] for t in (1, -1))
    diff = float(((up - dn) * do.double()).sum() / (2 * e))
    assert abs(float((g.double().cpu() * d).sum()) - diff) <= float((tg * d.abs()).sum()) + 1e-5 * abs(diff) + 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,KV,D,window,sinks", [(1, 333, 4, 2, 128, 100, 4), (30, 333, 6, 3, 128, 100, 70),
                                                     (2, 150, 4, 4, 80, 31, 3), (1, 1, 2, 1, 64, 5, 1)])
def test_without_gradients(B, S, H, KV, D, window, sinks):
    """The forward alone, from a wider projection into a padded output: the same values whether a backward may follow."""
    qkv, do = _inputs(B, S, H, KV, D, seed=2)
    wide = torch.cat([qkv, torch.full((B * S, 8), math.nan, dtype=BF)], 1).cuda()[:, :qkv.shape[1]]
    wo, to, _, _ = _definition(qkv, do, B, S, H, KV, D, window, sinks, D ** -0.5)
    with torch.no_grad():
        o = ops.attention_packed(wide, B, S, H, KV, D, window=window, sinks=sinks, out_pad=8)
    assert o.shape == (B * S, H * D) and o.stride(0) == H * D + 8 and not o.requires_grad
    _close(o, wo, to)
    assert torch.equal(o, ops.attention_packed(wide.requires_grad_(), B, S, H, KV, D, window=window, sinks=sinks).detach())


@pytest.mark.gpu
@pytest.mark.parametrize("S,window", [(512, 100), (300, 512)])
def test_views_and_padded_buffers(S, window):
    """A row-padded projection, padded output and gradient buffers, an output gradient with odd strides."""
    B, H, KV, D, sinks = 1, 4, 2, 128, 4
    W = (H + 2 * KV) * D
    qkv, do = _inputs(B, S, H, KV, D, seed=3)
    wo, to, wg, tg = _definition(qkv, do, B, S, H, KV, D, window, sinks, D ** -0.5)
    buf = torch.full((B * S, W + 24), math.nan, dtype=BF, device="cuda")
    buf[:, :W] = qkv.cuda()
    leaf = buf.requires_grad_()
    o = ops.attention_packed(leaf[:, :W], B, S, H, KV, D, window=window, sinks=sinks, out_pad=64, grad_pad=64)
    assert o.stride(0) == H * D + 64
    odd = torch.empty(B * S, H * D + 3, dtype=BF, device="cuda")[:, 1:H * D + 1]
    odd.copy_(do.cuda())
    (g,) = torch.autograd.grad(o, leaf, odd)
    _close(o, wo, to)
    _close(g[:, :W], wg, tg)
    x = torch.empty(B * S * W + 1, dtype=BF, device="cuda")[1:].view(B * S, W).copy_(qkv.cuda()).requires_grad_()  # off 16 bytes
    (g2,) = torch.autograd.grad(ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks), x, do.cuda())
    assert torch.equal(g2, g[:, :W])
    wide = leaf.detach().requires_grad_()  # more columns than heads: their gradient is zero
    (g3,) = torch.autograd.grad(ops.attention_packed(wide, B, S, H, KV, D, window=window, sinks=sinks), wide, do.cuda())
    assert torch.equal(g3[:, :W], g2) and (g3[:, W:] == 0).all()


@pytest.mark.gpu
def test_expanded_and_single_row_gradients():
    """Output gradients as autograd makes them: one row expanded over all, a single row with an odd row stride."""
    H, KV, D, window, sinks = 2, 1, 64, 7, 2
    for S in (40, 1):
        qkv, do = _inputs(1, S, H, KV, D, seed=8)
        do = do[:1].expand(S, -1)
        _, _, wg, tg = _definition(qkv, do.contiguous(), 1, S, H, KV, D, window, sinks, D ** -0.5)
        odd = torch.empty(S, H * D + 5, dtype=BF, device="cuda")[:, :H * D]
        odd.copy_(do.cuda())
        for g_out in (do[:1].cuda().expand(S, -1), odd):
            x = qkv.cuda().requires_grad_()
            o = ops.attention_packed(x, 1, S, H, KV, D, window=window, sinks=sinks)
            (g,) = torch.autograd.grad(o, x, g_out)
            _close(g, wg, tg)


@pytest.mark.gpu
def test_projections_past_32_bit_offsets():
    """4.8 GB of rows: the last sequence's last rows are those of a short sequence of what they see."""
    B, S, D, window, sinks, tail = 3, 2 ** 22, 64, 64, 4, 100
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B * S, 3 * D, generator=g, device="cuda", dtype=BF)
    do = torch.randn(B * S, D, generator=g, device="cuda", dtype=BF)
    assert x.numel() * 2 > 2 ** 32
    near = torch.cat([torch.arange(sinks), torch.arange(S - tail - window, S)]) + (B - 1) * S
    wo, to, wg, tg = _definition(x[near.cuda()].cpu(), do[near.cuda()].cpu(), 1, near.numel(), 1, 1, D, window, sinks, D ** -0.5)
    x.requires_grad_()
    o = ops.attention_packed(x, B, S, 1, 1, D, window=window, sinks=sinks)
    (gx,) = torch.autograd.grad(o, x, do)
    _close(o[-tail:], wo[-tail:], to[-tail:])
    _close(gx[-tail:], wg[-tail:], tg[-tail:])
    # and the first sequence's rows before any window is left
    wo, to, _, _ = _definition(x.detach()[:window].cpu(), do[:window].cpu(), 1, window, 1, 1, D, window, sinks, D ** -0.5)
    _close(o[:window], wo, to)


@pytest.mark.gpu
def test_rope_handoff():
    """The backward takes RoPE's inverse rotation into its epilogues (rows past a tile, positions given)."""
    B, S, H, KV, D, window, sinks = 2, 290, 2, 1, 128, 64, 4
    qkv, do = _inputs(B, S, H, KV, D, seed=9)
    table = ops.RotaryTable(D, 512)
    cos, sin = table.get("cuda")
    pos = (torch.arange(S) + 11).repeat(B).to(torch.int32).cuda()
    for p in (None, pos):
        rg = RopeGrad(cos, sin, p)
        x = qkv.cuda().requires_grad_()
        o = ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks, rope_grad=rg)
        assert rg.taken
        (g,) = torch.autograd.grad(o, x, do.cuda())
        _, _, wg, tg = _definition(qkv, do, B, S, H, KV, D, window, sinks, D ** -0.5)
        idx = (torch.arange(S).repeat(B) if p is None else p.cpu()).long()
        c, s = cos.cpu().double()[idx][:, None], sin.cpu().double()[idx][:, None]
        n = H + KV
        a, t = (z[:, :n * D].reshape(B * S, n, D) for z in (wg, tg))
        rot = torch.cat([a[..., :64] * c + a[..., 64:] * s, a[..., 64:] * c - a[..., :64] * s], -1)
        tr = t[..., :64] + t[..., 64:]
        _close(g[:, :n * D], rot.reshape(B * S, -1), torch.cat([tr, tr], -1).reshape(B * S, -1))
        _close(g[:, n * D:], wg[:, n * D:], tg[:, n * D:])


@pytest.mark.gpu
def test_reproducible_on_a_side_stream_and_in_a_graph():
    B, S, H, KV, D, window, sinks = 1, 700, 4, 1, 128, 90, 5
    qkv, do = (t.cuda() for t in _inputs(B, S, H, KV, D, seed=4))

    def step(x, d):
        x = x.detach().requires_grad_()
        o = ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks)
        return o.detach(), torch.autograd.grad(o, x, d)[0]

    want = [step(qkv * s, do) for s in (1.0, 0.5, 2.0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(qkv, do)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    xin = qkv.clone()
    with torch.cuda.stream(side):
        step(xin, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xin, do)
    for s, w in zip((1.0, 0.5, 2.0), want):
        xin.copy_(qkv * s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w)), s


@pytest.mark.gpu
def test_everything_in_the_window_equals_causal_attention():
    B, S, H, KV, D = 1, 512, 4, 2, 128
    qkv, do = (t.cuda() for t in _inputs(B, S, H, KV, D, seed=6))
    wo, to, wg, tg = _definition(qkv, do, B, S, H, KV, D, S, 0, D ** -0.5)
    for window, sinks in ((S, 4), (3, S), (10 ** 9, 10 ** 9)):
        x = qkv.detach().requires_grad_()
        o = ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks)
        (g,) = torch.autograd.grad(o, x, do)
        _close(o, wo, to)
        _close(g, wg, tg)


# ---------------------------------------------------------------- derivatives that the kernels do not have
class _StubKernels:
    """The extension's forward without a GPU: an output and no derivative, as a kernel gives it."""

    def sink_fwd(self, qkv, B, S, H, KV, D, scale, window, sinks, out_pad, grad):
        return qkv.new_zeros(B * S, H * D), None, None


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("D", [64, 48])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, D, grad, monkeypatch):
    """A tensor that carries a tangent is refused: it never comes back as an output without one."""
    from torch.autograd import forward_ad

    from finetune_controller_amd.ops import attention

    if dev == "cpu":
        monkeypatch.setattr(attention, "use_hip", lambda t: True)
        monkeypatch.setattr(attention, "ext", _StubKernels)
    x = torch.randn(6, 4 * D, dtype=BF, device=dev).requires_grad_(grad)
    for mode in (torch.enable_grad, torch.no_grad):
        with forward_ad.dual_level(), mode(), pytest.raises(NotImplementedError):
            ops.attention_packed(forward_ad.make_dual(x, torch.ones_like(x)), 1, 6, 2, 1, D, window=3, sinks=1)
        with forward_ad.dual_level(), torch.no_grad():  # the level alone refuses nothing
            assert ops.attention_packed(x, 1, 6, 2, 1, D, window=3, sinks=1).shape == (6, 2 * D)


def _odd_rows(x, extra):
    """``x`` in rows of ``extra`` more columns, contiguous: with an odd number of them most start off 16 bytes."""
    return torch.cat([x, torch.full((x.shape[0], extra), math.nan, dtype=x.dtype, device=x.device)], 1)


@pytest.mark.parametrize("extra", [0, 3, 8])
def test_copied_rows_can_be_read_16_bytes_at_a_time(extra):
    from finetune_controller_amd.ops.attention import _rows16

    x = torch.randn(5, 256).to(BF)
    for t in (_odd_rows(x, extra), _odd_rows(x, extra)[:, :256], _odd_rows(x, extra).t().contiguous().t()):
        y = _rows16(t, 256)
        assert torch.equal(y, x) and y.stride(1) == 1 and y.stride(0) % 8 == 0 and y.stride(0) >= 256


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [3, 8])
@pytest.mark.parametrize("D", [64, 48])
def test_more_columns_than_heads(extra, D):
    B, S, H, KV, window, sinks = 1, 70, 2, 1, 9, 2
    qkv, do = _inputs(B, S, H, KV, D, seed=10)
    wo, to, wg, tg = _definition(qkv, do, B, S, H, KV, D, window, sinks, D ** -0.5)
    x = _odd_rows(qkv, extra).cuda()
    with torch.no_grad():
        _close(ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks), wo, to)
    o = ops.attention_packed(x.requires_grad_(), B, S, H, KV, D, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, x, do.cuda())
    _close(o, wo, to)
    _close(g[:, :qkv.shape[1]], wg, tg)
    assert g.shape == x.shape and (g[:, qkv.shape[1]:] == 0).all()


# ---------------------------------------------------------------- the output's bits below bf16
def _uniform(B, S, H, KV, D, seed):
    """Queries of zero: every visible key has the same weight, exactly, so that no weight is rounded.  Values and keys of a
    large common part: dP and delta cancel, and delta's error goes to dQ undamped."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B * S, H + 2 * KV, D, generator=g)
    x[:, :H] = 0
    x[:, H:H + KV] = x[:1, H:H + KV]
    x[:, H + KV:] += 3.0 + torch.rand(D, generator=g)
    return x.flatten(1).to(BF), torch.randn(B * S, H * D, generator=g).to(BF)


LOW = [(1, 200, 2, 1, 128, 64, 2), (1, 200, 2, 1, 64, 64, 2), (16, 260, 6, 2, 128, 90, 70), (16, 260, 6, 2, 64, 90, 70)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,KV,D,window,sinks", LOW)
def test_low_byte_of_the_output(B, S, H, KV, D, window, sinks):
    """o and its low byte make 16 significant bits: the byte counts 2^-8 of a bf16 step (2^-7 of the value's power of two),
    rounded down, and stops at 127 where half a step is 128 -- an error under 2 * 2^-15 relative; 2^-20 of the mean
    magnitude for the 32-bit sums.  Half a bf16 step is up to 2^-8."""
    from finetune_controller_amd.ops._backend import ext

    qkv, _ = _uniform(B, S, H, KV, D, seed=D + B)
    o, low, _ = ext().sink_fwd(qkv.cuda(), B, S, H, KV, D, D ** -0.5, window, sinks, 0, True)
    v = qkv.double().view(B, S, H + 2 * KV, D)[:, :, H + KV:].repeat_interleave(H // KV, 2)
    seen = _seen(S, window, sinks).double()
    want = (torch.einsum("qk,bkhd->bqhd", seen, v) / seen.sum(1)[:, None, None]).reshape(B * S, H * D)
    bits = o.cpu().view(torch.int16).int() << 16

    def err(byte):
        return ((bits + (byte.int() << 8)).view(torch.float32).double() - want).abs()

    tol = (2.0 ** -14 + 2.0 ** -20) * want.abs()
    got = low.cpu().view(torch.int8)
    assert (err(got) <= tol).all()
    # the tolerance tells the byte from none, from one of the wrong sign and from a neighbour's
    for wrong in (torch.zeros_like(got), ~got, got.roll(1, 1), got.view(-1, 2).flip(1).view(got.shape)):
        assert (err(wrong) > tol).double().mean() > 0.8


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,KV,D,window,sinks", LOW)
def test_the_backward_reads_the_low_byte(B, S, H, KV, D, window, sinks):
    """With equal keys k, dQ = scale k sum dS is zero but for errors, and delta's is the largest of them if it is formed from
    the rounded output: over the rows the kernels' dQ has to be less than half of what that alone gives."""
    qkv, do = _uniform(B, S, H, KV, D, seed=2 * D + B)
    x = qkv.cuda().requires_grad_()
    (g,) = torch.autograd.grad(ops.attention_packed(x, B, S, H, KV, D, window=window, sinks=sinks), x, do.cuda())
    v = qkv.double().view(B, S, H + 2 * KV, D)[:, :, H + KV:].repeat_interleave(H // KV, 2)
    k = qkv.double().view(B, S, H + 2 * KV, D)[:, :, H:H + KV].repeat_interleave(H // KV, 2)
    seen = _seen(S, window, sinks).double()
    o = torch.einsum("qk,bkhd->bqhd", seen, v) / seen.sum(1)[:, None, None]
    off = ((o.to(BF).double() - o) * do.double().view(B, S, H, D)).sum(-1, keepdim=True)  # delta's error, from bf16 o
    rounded = (D ** -0.5 * off * k).flatten()
    got = g[:, :H * D].double().cpu().flatten()
    assert got.norm() < 0.5 * rounded.norm(), float(got.norm() / rounded.norm())


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launchers' own checks, called without tensors")
def test_launchers_refuse_rows_off_16_bytes():
    """The kernels load and store 16 bytes at a time: any row stride that is no multiple of 8 is refused before a launch."""
    import ctypes

    from finetune_controller_amd.ops._backend import load_ext

    lib = ctypes.CDLL(load_ext().__file__)
    null, i, ll, f = ctypes.c_void_p(), ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    for odd in range(3):
        rs = [ll(256 + (4 if j == odd else 0)) for j in range(3)]
        assert lib.ftc_sink_fwd(*[null] * 6, i(1), i(8), i(2), i(1), i(64), *rs, f(0.1), i(4), i(1), null) == -1
    for odd in range(6):
        rs = [ll(256 + (4 if j == odd else 0)) for j in range(6)]
        assert lib.ftc_sink_bwd(*[null] * 11, i(1), i(8), i(2), i(1), i(64), *rs, f(0.1), i(4), i(1), *[null] * 4) == -1
