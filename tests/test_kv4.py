"""The 4-bit KV cache (ops.kv4): rows quantised as they are written, read back, decode attention over it.

Oracles: the definition in exact arithmetic (``fractions``) for codes, 64-bit attention over the held values.
Tolerance of the attention (bf16 output): every weight p * s is rounded to bf16 once (relative 2^-8 at most)
and so is the output, so |error| <= 2^-8 (sum p |v| + |o|); 2^-12 sum p |v| covers the 32-bit sums
(relative 2^-24 each over scores below 2^6 and products against codes offset by 24)."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from finetune_controller_amd import ops
from finetune_controller_amd.ops import kv4

BF = torch.bfloat16


def _exact_codes(row):
    """(s, codes) of one group of 32 bf16 values by the definition, in exact arithmetic."""
    x = [Fraction(float(v)) for v in row]
    e = max(x, key=lambda v: (abs(v), v))
    if abs(e) < Fraction(1, 2 ** 100):
        return Fraction(0), [0] * 32
    s = -e / 8
    return s, [max(-8, min(7, round(v / s))) for v in x]  # Fraction rounds half to even


def _rows(*shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(BF)


def _codes_of(x):
    """Values that x [..., D] is held as, fp64."""
    c, s = kv4.quantize_reference(x)
    return kv4._held(c, s).double()


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("kind", ["normal", "ties", "wide", "tiny", "both_signs"])
def test_quantisation_matches_the_exact_definition(kind):
    x = _rows(24, 64, seed=3)
    if kind == "ties":  # half integers of the scale everywhere: e = 8, s = -1
        x = (torch.arange(24 * 64).reshape(24, 64) % 33 - 16).float().div(2).to(BF)
    elif kind == "wide":
        x = (x.float() * torch.exp2(torch.randint(-60, 60, x.shape, generator=torch.Generator().manual_seed(1)).float())).to(BF)
    elif kind == "tiny":
        x = (x.float() * 2.0 ** torch.arange(-104, -80)[:, None]).to(BF)
    elif kind == "both_signs":
        x[:, 5], x[:, 9], x[:, 40], x[:, 50] = -4.0, 4.0, 4.0, -4.0
    codes, s = kv4.quantize_reference(x)
    for i in range(x.shape[0]):
        for g in range(2):
            es, ec = _exact_codes(x[i, 32 * g:32 * g + 32])
            assert Fraction(float(s[i, g])) == es
            assert (codes[i, 32 * g:32 * g + 32].int() - 8).tolist() == ec


def test_kernel_rounding_is_exact_for_every_pair_of_significands():
    """The kernel forms x / s as a product with the rounded reciprocal, snaps it to multiples of 2^-11 (the sum
    with 6144) and rounds the sum with 1.5 * 2^23 + 8 (kv4.h kv4_code).  The same arithmetic in numpy against exact integers, for every significand of
    x and s at every exponent distance that gives |x / s| <= 8."""
    f32 = np.float32
    X = np.arange(128, 256, dtype=np.int64)[:, None]
    S = np.arange(128, 256, dtype=np.int64)[None, :]
    for k in range(-12, 4):  # x / s = X / S * 2^k
        x = (X * 2.0 ** k).astype(f32)
        rinv = f32(1.0) / S.astype(f32)
        for fused in (False, True):  # the compiler may contract the product into the add
            prod = x.astype(np.float64) * rinv.astype(np.float64)
            t = (prod + 6144.0).astype(f32) if fused else (prod.astype(f32) + f32(6144.0))
            n = (t + f32(12576776.0)).astype(f32).view(np.int32) - 0x4B400000
            num, den = X * (1 << (k + 12)), S * (1 << 12)
            q, r = num // den, num % den
            want = q + ((2 * r > den) | ((2 * r == den) & (q % 2 == 1)))
            ok = (num <= 8 * den)
            assert np.array_equal(np.broadcast_to(n, ok.shape)[ok], (want + 8)[ok]), k


def test_non_finite_groups_read_back_as_nan():
    x = torch.ones(1, 2, 64, dtype=BF)
    x[0, 0, 3], x[0, 1, 40] = math.inf, math.nan
    data = ops.kv4_alloc(1, 32, 1, 64)
    ops.kv4_store(data, x, x, torch.zeros(1, dtype=torch.int32))
    k, _ = ops.kv4_load(data, torch.zeros(1, dtype=torch.int32), 2, 64)
    assert k[0, 0, :32].isnan().all() and (k[0, 0, 32:] == 1).all()
    assert k[0, 1, 32:].isnan().all() and (k[0, 1, :32] == 1).all()


# ---------------------------------------------------------------- layout, writes
@pytest.mark.parametrize("D", [64, 128])
def test_layout_covers_the_record_once(D):
    kb, kd, ks, vb, vd, vs = kv4._maps(D)
    seen = torch.cat([kb.reshape(-1), vb.reshape(-1)] + [t.reshape(-1) + z for t in (ks, vs) for z in (0, 1)])
    assert torch.equal(seen.sort().values, torch.arange(kv4._record(D)))
    for d in (kd, vd):
        assert torch.equal(d.reshape(-1).sort().values, torch.arange(D))


@pytest.mark.parametrize("D,KV", [(64, 3), (128, 2)])
@pytest.mark.parametrize("n,start", [(1, (0, 31, 64)), (33, (0, 7, 95)), (70, (5, -20, 100)), (4, (126, 128, -9))])
def test_store_and_load(D, KV, n, start):
    """Rows come back as the values they are held as; rows outside the cache are dropped, all else stays."""
    cap, B = 128, 3
    data = ops.kv4_alloc(B, cap - 3, KV, D)
    old_k, old_v = _rows(B, cap, KV * D, seed=1), _rows(B, cap, KV * D, seed=2)
    zero = torch.zeros(B, dtype=torch.int32)
    ops.kv4_store(data, old_k, old_v, zero)
    k, v = _rows(B, n, KV * D, seed=4), _rows(B, n, KV * D, seed=5)
    st = torch.tensor(start, dtype=torch.int32)
    count = torch.tensor([n, max(0, n - 2), n + 5], dtype=torch.int32)
    ops.kv4_store(data, k, v, st, count)
    got = ops.kv4_load(data, zero, cap, D, dtype=torch.float64)
    for new, old, g in ((k, old_k, got[0]), (v, old_v, got[1])):
        want = _codes_of(old.unflatten(-1, (KV, D))).flatten(-2)
        held = _codes_of(new.unflatten(-1, (KV, D))).flatten(-2)
        for b in range(B):
            for i in range(min(n, int(count[b]))):
                if 0 <= start[b] + i < cap:
                    want[b, start[b] + i] = held[b, i]
        assert torch.equal(g, want)
    part = ops.kv4_load(data, torch.tensor([-3, 100, 126], dtype=torch.int32), 40, D, dtype=torch.float64)
    assert (part[0][0, :3] == 0).all() and torch.equal(part[0][0, 3:], got[0][0, :37])
    assert torch.equal(part[1][1, :28], got[1][1, 100:]) and (part[1][1, 28:] == 0).all()
    assert torch.equal(part[1][2, :2], got[1][2, 126:]) and (part[1][2, 2:] == 0).all()


# ---------------------------------------------------------------- attention
def _attend64(q, K, V, seen, H, KV, D, scale):
    """One sequence in 64 bits: q [H*D], K / V [L, KV*D] -> (o [H*D], sum p |v| [H*D])."""
    G = H // KV
    o, pv = torch.zeros(H, D, dtype=torch.float64), torch.zeros(H, D, dtype=torch.float64)
    idx = seen.nonzero().flatten()
    if idx.numel() == 0:
        return o.flatten(), pv.flatten()
    for h in range(H):
        c = slice((h // G) * D, (h // G + 1) * D)
        p = torch.softmax(K[idx, c] @ q[h * D:(h + 1) * D].double() * scale, 0)
        o[h], pv[h] = p @ V[idx, c], p @ V[idx, c].abs()
    return o.flatten(), pv.flatten()


def _decode_case(B, H, KV, D, lens, cap, seed=0, qscale=1.0):
    qkv = _rows(B, (H + 2 * KV) * D, seed=seed, scale=1.0)
    qkv[:, :H * D] *= qscale
    return qkv, _rows(B, cap, KV * D, seed=seed + 1), _rows(B, cap, KV * D, seed=seed + 2)


def _expected(qkv, k, v, lens, H, KV, D, scale, window, sinks):
    out = []
    for b, n in enumerate(lens):
        K, V = (_codes_of(t[b].cpu().unflatten(-1, (KV, D))).flatten(-2) for t in (k, v))
        x = qkv[b].cpu()
        if n > 0:
            K[n - 1] = _codes_of(x[H * D:(H + KV) * D].view(KV, D)).flatten()
            V[n - 1] = _codes_of(x[(H + KV) * D:(H + 2 * KV) * D].view(KV, D)).flatten()
        t = torch.arange(K.shape[0])
        seen = (t < n) & ((t >= n - window) | (t < sinks) if window > 0 else True)
        out.append(_attend64(x, K, V, seen, H, KV, D, scale))
    return torch.stack([o for o, _ in out]), torch.stack([p for _, p in out])


def _check(got, want, pv, extra=0.0):
    err = (got.double().cpu() - want).abs()
    tol = 2.0 ** -8 * (pv + want.abs()) + (2.0 ** -12 + extra) * pv
    assert (err <= tol).all(), (err / tol.clamp_min(1e-30)).max()


CASES = [  # B, H, KV, D, lens, window, sinks
    (1, 8, 2, 128, (1,), 0, 0),
    (3, 4, 4, 64, (0, 31, 96), 0, 0),
    (4, 8, 2, 64, (5, 32, 33, 160), 40, 3),
    (3, 8, 1, 128, (160, 159, 64), 1, 0),
    (2, 14, 2, 128, (129, 160), 17, 40),
    (3, 3, 1, 64, (100, 2, 160), 64, 200),
    (2, 24, 1, 128, (97, 160), 0, 0),
    (2, 40, 2, 64, (97, 160), 33, 5),
]


@pytest.mark.parametrize("B,H,KV,D,lens,window,sinks", CASES)
def test_decode_reference(B, H, KV, D, lens, window, sinks):
    cap, scale = 160, 1.0 / math.sqrt(D)
    qkv, k, v = _decode_case(B, H, KV, D, lens, cap)
    data = ops.kv4_alloc(B, cap, KV, D)
    ops.kv4_store(data, k, v, torch.zeros(B, dtype=torch.int32))
    got = ops.decode_attention_kv4(qkv, data, torch.tensor(lens, dtype=torch.int32), cap, H, KV, D, window=window,
                                   sinks=sinks)
    _check(got, *_expected(qkv, k, v, lens, H, KV, D, scale, window, sinks))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(dev):
    """The same calls are refused on both paths, before anything is launched or written."""
    i32 = dict(dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv4_alloc(1, 32, 1, 96)
    with pytest.raises(ValueError, match="positive"):
        ops.kv4_alloc(1, 0, 1, 64)
    data = ops.kv4_alloc(2, 64, 2, 64, device=dev)
    k, z = torch.zeros(2, 3, 128, dtype=BF, device=dev), torch.zeros(2, **i32)
    for bad in (dict(k=k[:, :, :127]), dict(k=k[:1]), dict(start=z.long()), dict(start=z[:1]),
                dict(count=torch.zeros(3, **i32)), dict(data=data.float()), dict(data=data[:, :, ::2]), dict(data=data[0])):
        a = {**dict(data=data, k=k, start=z, count=None), **bad}
        with pytest.raises(ValueError):
            ops.kv4_store(a["data"], a["k"], a["k"], a["start"], a["count"])
    with pytest.raises(ValueError, match="of one dtype"):
        ops.kv4_store(data, k, k.float(), z)
    with pytest.raises(ValueError, match="negative"):
        ops.kv4_load(data, z, -1, 64)
    q, n = torch.zeros(2, 8 * 64, dtype=BF, device=dev), torch.ones(2, **i32)
    for args in ((q, n, 65, 4, 2), (q, n, 0, 4, 2), (q, n, 64, 5, 2), (q, n, 64, 4, 1), (q[:, :400], n, 64, 4, 2),
                 (q[:1], n, 64, 4, 2), (q, n.long(), 64, 4, 2)):
        with pytest.raises(ValueError):
            ops.decode_attention_kv4(args[0], data, args[1], args[2], args[3], args[4], 64)
    with pytest.raises(ValueError, match="sinks"):
        ops.decode_attention_kv4(q, data, n, 64, 4, 2, 64, window=4, sinks=-1)
    for scale in (0.0, -0.1, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            ops.decode_attention_kv4(q, data, n, 64, 4, 2, 64, scale=scale)
    for bad in (dict(data=data.cpu()), dict(start=z.cpu()), dict(v=k.cpu())):
        if dev == "cuda":  # tensors of another device
            a = {**dict(data=data, v=k, start=z), **bad}
            with pytest.raises(ValueError):
                ops.kv4_store(a["data"], k, a["v"], a["start"])
    ops.kv4_store(data, k[:, :0], k[:, :0], z)
    assert ops.kv4_load(data, z, 0, 64)[0].shape == (2, 0, 128)
    assert int(data.sum()) == 0  # nothing was written


# ---------------------------------------------------------------- kernels
@pytest.mark.gpu
@pytest.mark.parametrize("D,KV", [(64, 1), (128, 3)])
@pytest.mark.parametrize("n,start", [(1, (0, 31, 64)), (33, (0, 7, 95)), (70, (5, -20, 100)), (128, (0, 0, 32)),
                                     (4, (126, 128, -9)), (300, (-40, -128, 1))])
def test_store_kernel_writes_the_reference_bytes(D, KV, n, start):
    cap, B = 128, 3
    pad = 8 * ((n + D) % 3)  # row-padded column views, as a projection's
    buf = _rows(B, n, 2 * KV * D + pad, seed=n)
    if n >= 33:
        buf[0, 1, 5], buf[0, 2, 9], buf[0, 3] = math.inf, math.nan, 0.0
        buf[1, 0] *= 2.0 ** -101
    k, v = buf[..., :KV * D], buf[..., KV * D:2 * KV * D]
    st, count = torch.tensor(start, dtype=torch.int32), torch.tensor([n, max(0, n - 2), n + 5], dtype=torch.int32)
    old = torch.randint(0, 256, (B, KV, cap // 32, kv4._record(D)), generator=torch.Generator().manual_seed(9)).to(torch.uint8)
    for cnt in (None, count):
        want = old.clone()
        ops.kv4_store(want, k, v, st, cnt)
        got = old.cuda()
        g = buf.cuda()
        ops.kv4_store(got, g[..., :KV * D], g[..., KV * D:2 * KV * D], st.cuda(), cnt.cuda() if cnt is not None else None)
        kb, _, ks, vb, _, vs = kv4._maps(D)
        # groups of a NaN scale: the scale alone says what they hold
        assert _same_held(got.cpu(), want, D)
        if n < 33:
            assert torch.equal(got.cpu(), want)
    none, got = torch.zeros(B, dtype=torch.int32), old.cuda()  # no rows of a padded batch, or fewer than none
    for cnt in (none, none - 7):
        ops.kv4_store(got, g[..., :KV * D], g[..., KV * D:2 * KV * D], st.cuda(), cnt.cuda())
    assert torch.equal(got.cpu(), old)
    off = g.flatten()[1:1 + B * n * KV * D].view(B, n, KV * D)  # rows that start off a 16-byte boundary
    want, got = old.clone(), old.cuda()
    ops.kv4_store(want, off.cpu(), off.cpu(), st)
    ops.kv4_store(got, off, off, st.cuda())
    assert _same_held(got.cpu(), want, D)


def _same_held(a, b, D):
    return all(torch.equal(torch.nan_to_num(kv4._get(a, w, D), nan=7e37), torch.nan_to_num(kv4._get(b, w, D), nan=7e37))
               for w in (0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("D,KV", [(64, 3), (128, 2)])
@pytest.mark.parametrize("n,start", [(1, (0, 127)), (5, (-3, 126)), (64, (32, 0)), (77, (-31, 100)), (200, (-64, 1000))])
def test_load_kernel(D, KV, n, start):
    data = torch.randint(0, 256, (2, KV, 4, kv4._record(D)), generator=torch.Generator().manual_seed(2)).to(torch.uint8)
    ops.kv4_store(data, _rows(2, 90, KV * D), _rows(2, 90, KV * D, seed=1), torch.tensor([3, 3], dtype=torch.int32))
    st = torch.tensor(start, dtype=torch.int32)
    for a, b in zip(ops.kv4_load(data.cuda(), st.cuda(), n, D), ops.kv4_load(data, st, n, D)):
        assert a.dtype == BF and torch.equal(torch.nan_to_num(a.cpu()), torch.nan_to_num(b))


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,KV,D,lens,window,sinks", CASES)
def test_decode_kernel(B, H, KV, D, lens, window, sinks):
    """Ragged lengths, window and sinks; the tokens behind a sequence hold NaN and infinities."""
    cap, scale = 160, 0.11
    qkv, k, v = _decode_case(B, H, KV, D, lens, cap, seed=7, qscale=2.0)
    data = ops.kv4_alloc(B, cap, KV, D, device="cuda")
    bk, bv = k.clone(), v.clone()
    for b, n in enumerate(lens):
        bk[b, n:], bv[b, n:] = math.nan, math.inf
    ops.kv4_store(data, bk.cuda(), bv.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"))
    before = data.clone()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = torch.cat([qkv, qkv[:, :8]], 1).cuda()  # row-padded projection
    got = ops.decode_attention_kv4(wide, data, ln, cap, H, KV, D, scale=scale, window=window, sinks=sinks)
    _check(got, *_expected(qkv, k, v, lens, H, KV, D, scale, window, sinks))
    # exactly one token a sequence was written
    new = qkv[:, None, H * D:]
    ops.kv4_store(before, new[..., :KV * D].cuda(), new[..., KV * D:].cuda(), ln - 1)
    assert torch.equal(before, data)


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KV", [(128, 32, 8), (64, 16, 2)])
def test_decode_kernel_long(D, H, KV):
    """Lengths that split over many workgroups, with a max_len far above some of them."""
    lens, cap = (9000, 4097, 1, 8191), 9001
    qkv, k, v = _decode_case(4, H, KV, D, lens, cap, seed=11)
    data = ops.kv4_alloc(4, cap, KV, D, device="cuda")
    ops.kv4_store(data, k.cuda(), v.cuda(), torch.zeros(4, dtype=torch.int32, device="cuda"))
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (4096, 4), (100, 33)):
        got = ops.decode_attention_kv4(qkv.cuda(), data, ln, 9000, H, KV, D, window=window, sinks=sinks)
        _check(got, *_expected(qkv, k, v, lens, H, KV, D, D ** -0.5, window, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("D,H", [(128, 3), (128, 8), (128, 11), (64, 1), (64, 8), (64, 16)])
def test_decode_kernel_many_short_sequences(D, H):
    """More short sequences than workgroups of a round, every number of query heads a set of columns can hold."""
    B, cap = 300, 96
    lens = tuple((37 * b) % 91 for b in range(B))
    qkv, k, v = _decode_case(B, H, 1, D, lens, cap, seed=31)
    data = ops.kv4_alloc(B, cap, 1, D, device="cuda")
    ops.kv4_store(data, k.cuda(), v.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"))
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = ops.decode_attention_kv4(qkv.cuda(), data, ln, cap, H, 1, D)
    _check(got, *_expected(qkv, k, v, lens, H, 1, D, D ** -0.5, 0, 0))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("max_len", [64, 120])
def test_lengths_outside_the_bound(dev, max_len):
    """Zero and negative lengths give zero rows; longer than max_len: its first max_len tokens, nothing written."""
    B, H, KV, D, cap = 5, 4, 2, 64, 128
    lens = (0, -3, max_len, max_len + 1, 2 ** 31 - 1)
    qkv, k, v = _decode_case(B, H, KV, D, lens, cap, seed=21)
    data = ops.kv4_alloc(B, cap, KV, D, device=dev)
    ops.kv4_store(data, k.to(dev), v.to(dev), torch.zeros(B, dtype=torch.int32, device=dev))
    before = data.clone()
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = ops.decode_attention_kv4(qkv.to(dev), data, ln, max_len, H, KV, D).cpu()
    assert (got[:2] == 0).all()
    ops.kv4_store(before[2:3], qkv[2:3, None, H * D:(H + KV) * D].to(dev), qkv[2:3, None, (H + KV) * D:].to(dev), ln[2:3] - 1)
    assert torch.equal(before, data)
    want, pv = _expected(qkv[2:3], k[2:3], v[2:3], (max_len,), H, KV, D, D ** -0.5, 0, 0)
    _check(got[2:3], want, pv)
    for b in (3, 4):
        K, V = (_codes_of(t[b].unflatten(-1, (KV, D))).flatten(-2) for t in (k, v))
        o, p = _attend64(qkv[b], K, V, torch.arange(cap) < max_len, H, KV, D, D ** -0.5)
        _check(got[b], o, p)


@pytest.mark.gpu
def test_a_cache_past_32_bit_offsets():
    """4.8 GB, 2^21 tokens: the far ends are written, read back and attended to as the same tokens in a small cache are."""
    B, H, KV, D, cap, small = 2, 16, 8, 128, 2 ** 21, 320
    window, sinks, tail = 100, 8, 150
    lens, short = (cap, cap - 52), (small, small - 52)
    qkv, k, v = _decode_case(B, H, KV, D, None, small, seed=41)
    dev = dict(dtype=torch.int32, device="cuda")
    data = ops.kv4_alloc(B, cap, KV, D, device="cuda")
    assert data.numel() > 2 ** 32
    i = torch.stack([torch.arange(n - tail, n) for n in short])  # the small cache's last rows, put at the end
    far = [torch.stack([t[b, i[b]] for b in range(B)]).cuda() for t in (k, v)]
    at = torch.tensor([n - tail for n in lens], **dev)
    ops.kv4_store(data, *far, at)
    for g, w in zip(ops.kv4_load(data, at, tail, D), far):
        # (read back as bf16: the held values, 12 significant bits, rounded once)
        assert torch.equal(g.cpu(), _codes_of(w.cpu().unflatten(-1, (KV, D))).flatten(-2).to(BF))
    ops.kv4_store(data, k[:, :sinks].cuda(), v[:, :sinks].cuda(), torch.zeros(B, **dev))
    got = ops.decode_attention_kv4(qkv.cuda(), data, torch.tensor(lens, **dev), cap, H, KV, D, window=window, sinks=sinks)
    _check(got, *_expected(qkv, k, v, short, H, KV, D, D ** -0.5, window, sinks))
    # the whole length: keys of zero weigh alike, and only the last rows' values are not zero
    data.zero_()
    ops.kv4_store(data, torch.zeros_like(far[0]), far[1], at)
    flat = qkv.clone()
    flat[:, H * D:(H + KV) * D] = 0
    got = ops.decode_attention_kv4(flat.cuda(), data, torch.tensor(lens, **dev), cap, H, KV, D)
    V = _codes_of(far[1].cpu().unflatten(-1, (KV, D)))  # [B, tail, KV, D]
    V[:, -1] = _codes_of(flat[:, (H + KV) * D:].view(B, KV, D))
    n = torch.tensor(lens, dtype=torch.float64)[:, None, None]
    want, pv = V.sum(1) / n, V.abs().sum(1) / n
    _check(got, *(t.repeat_interleave(H // KV, 1).flatten(1) for t in (want, pv)))


@pytest.mark.gpu
def test_decode_step_on_a_stream_and_in_a_graph():
    """The same step eagerly, on a side stream and replayed from a graph with growing lengths."""
    B, H, KV, D, cap = 3, 8, 2, 128, 200
    qkv, k, v = _decode_case(B, H, KV, D, None, cap, seed=5)
    ln0 = torch.tensor([50, 1, 150], dtype=torch.int32, device="cuda")

    def fresh():
        data = ops.kv4_alloc(B, cap, KV, D, device="cuda")
        ops.kv4_store(data, k.cuda(), v.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"))
        return data

    x = qkv.cuda()
    eager, want, lens = fresh(), [], ln0.clone()
    for i in range(4):
        want.append(ops.decode_attention_kv4(x * (1 + i), eager, lens, cap, H, KV, D).clone())
        lens += 1
    side, data, lens = torch.cuda.Stream(), fresh(), ln0.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = ops.decode_attention_kv4(x, data, lens, cap, H, KV, D)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, want[0])
    data, lens, xin = fresh(), ln0.clone(), x.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.decode_attention_kv4(xin, data, lens, cap, H, KV, D)
    for i in range(4):
        xin.copy_(x * (1 + i))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        lens += 1
    assert torch.equal(data, eager)


class _StubKernels:
    """The extension's decode attention without a GPU: an output and no derivative, as a kernel gives it."""

    def decode_attention_kv4(self, qkv, data, lens, max_len, H, KV, D, scale, window, sinks):
        return qkv.detach().new_zeros(qkv.shape[0], H * D)


@pytest.mark.parametrize("dev", ["cpu", "kernels without a gpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_decode_attention_has_no_derivative(dev, monkeypatch):
    """Both paths alike: an output that requires no grad, and a tensor with a tangent is refused."""
    from torch.autograd import forward_ad

    if dev == "kernels without a gpu":
        monkeypatch.setattr(kv4, "use_hip", lambda t: True)
        monkeypatch.setattr(kv4, "ext", _StubKernels)
        dev = "cpu"
    data = ops.kv4_alloc(2, 32, 1, 64, device=dev)
    lens = torch.tensor([1, 5], dtype=torch.int32, device=dev)
    x = _rows(2, 4 * 64).to(dev).requires_grad_()
    assert not ops.decode_attention_kv4(x, data, lens, 32, 2, 1, 64).requires_grad
    before = data.clone()
    for y in (x, x.detach()):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="derivative"):
            ops.decode_attention_kv4(forward_ad.make_dual(y, torch.ones_like(y)) * 2, data, lens, 32, 2, 1, 64)
    assert torch.equal(before, data)


def test_the_torch_path_waits_for_nothing():
    """Decode steps may be captured into a graph: no operation of theirs reads a tensor on the host."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class NoHostRead(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            assert func._overloadpacket not in (torch.ops.aten.nonzero, torch.ops.aten._local_scalar_dense,
                                                torch.ops.aten.is_nonzero, torch.ops.aten.masked_select), func
            return func(*args, **(kwargs or {}))

    data = ops.kv4_alloc(3, 64, 2, 64)
    qkv, lens = _rows(3, 8 * 64), torch.tensor([0, 5, 70], dtype=torch.int32)
    k = _rows(3, 7, 2 * 64)
    with NoHostRead():
        ops.kv4_store(data, k, k, lens - 3, lens)
        ops.kv4_load(data, lens, 4, 64)
        ops.decode_attention_kv4(qkv, data, lens, 64, 4, 2, 64, window=9, sinks=2)


@pytest.mark.gpu
def test_decode_kernel_on_rows_of_odd_width():
    """A contiguous projection of three more columns than the heads': its rows start off 16 bytes and are copied."""
    B, H, KV, D, lens, cap = 3, 8, 2, 128, (40, 1, 64), 64
    qkv, k, v = _decode_case(B, H, KV, D, lens, cap, seed=51)
    data = ops.kv4_alloc(B, cap, KV, D, device="cuda")
    ops.kv4_store(data, k.cuda(), v.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"))
    wide = torch.cat([qkv, torch.full((B, 3), math.nan, dtype=BF)], 1).cuda()
    got = ops.decode_attention_kv4(wide, data, torch.tensor(lens, dtype=torch.int32, device="cuda"), cap, H, KV, D)
    _check(got, *_expected(qkv, k, v, lens, H, KV, D, D ** -0.5, 0, 0))
