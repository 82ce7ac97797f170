"""KV cache held in 4 bits: rows quantised as they are written, read back, and attended to in place.

A cache is one uint8 tensor ``[B, KV, tiles, record]`` (``kv4_alloc``; per layer in ``KV4Cache``).
Values are quantised in groups of 32 along the head dimension with one bf16 scale each: with ``e`` the
group's element of largest magnitude (the positive one where both signs have it),

    s = -e / 8,    c = clamp(round_half_even(x / s), -8, 7),    held value = s * c

so ``e`` itself is held exactly and one group takes 32 x 4 + 16 bits: 4.5 bits a value, 3.56x less
than bf16.  A group whose largest magnitude is under 2^-100 is held as zeros; a group with an infinity
or NaN reads back as NaN.

The record of 32 tokens (4608 bytes at head_dim 128, 2304 at 64) is laid out for the matrix
instructions of ``csrc/kernels/kv4_attn.hip``: K codes, K scales, V codes, V scales, each 16-byte
chunk being what one lane feeds to them (``csrc/kernels/kv4.h``; ``_maps`` below is the same layout as
index tables).  Every byte holds two values of the same token, so tokens are written independently.

GPU: ``csrc/kernels/kv4.hip`` and ``kv4_attn.hip``.  CPU / ``FTC_KERNELS=torch``: the torch forms
below, which are also the numerics oracle.
"""
from __future__ import annotations

import functools
import math

import torch

from ._backend import ext, has_tangent, use_hip
from .decode import KVCache, visible_keys

KV4_TILE = 32   # tokens per record
KV4_GROUP = 32  # values per scale
_TINY = 2.0 ** -100


def _record(D: int) -> int:
    if D not in (64, 128):
        raise ValueError(f"4-bit KV cache: head_dim must be 64 or 128, got {D}")
    return 2 * KV4_TILE * (D // 2 + D // KV4_GROUP * 2)


def kv4_alloc(B: int, max_len: int, KV: int, D: int, device=None, layers: int | None = None) -> torch.Tensor:
    """A zeroed cache for ``B`` sequences of up to ``max_len`` tokens (rounded up to whole records of 32):
    uint8 ``[B, KV, tiles, record]``, with a leading ``layers`` dimension if given."""
    rec = _record(D)
    if B < 1 or KV < 1 or max_len < 1:
        raise ValueError(f"4-bit KV cache: B, KV and max_len must be positive, got {B}, {KV}, {max_len}")
    shape = (B, KV, -(-max_len // KV4_TILE), rec)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=None)
def _maps(D: int):
    """Byte offsets within a record and the value of each nibble: ``(kb, kd, ks, vb, vd, vs)``; ``kb[t]``
    [D/2] offsets of token t's K bytes, ``kd`` [D/2, 2] the d of their low and high nibbles, ``ks[t]``
    [D/32] offsets of its (2-byte) K scales; the same for V."""
    NG, t = D // KV4_GROUP, torch.arange(KV4_TILE)
    blk, i = t // 8, t % 8
    # K: 16-byte chunk of lane (r, q): word j = values 32 j + 8 q + 0..7; bytes of a word: d 0|2, 4|6, 1|3, 5|7
    half, r = i // 4, 4 * blk + i % 4
    kb, kd = [], []
    for j in range(NG):
        for q in range(4):
            off = (half * 1024 + q * 256 + r * 16 + j * 4) if D == 128 else (q * 256 + r * 16 + half * 8 + j * 4)
            for b, (lo, hi) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
                kb.append(off + b)
                kd.append((32 * j + 8 * q + lo, 32 * j + 8 * q + hi))
    codes, scales = KV4_TILE * D // 2, KV4_TILE * NG * 2
    g = torch.arange(NG)
    ks = codes + (blk[:, None] * NG + g) * 16 + i[:, None] * 2
    # V: 16-byte chunk of lane (r, block): word p = tokens 2p | 2p + 1 (halves), values 64 c + 4 r + 0..3 each
    vb, vd = [], []
    for c in range(D // 64):
        for rr in range(16):
            off = c * 1024 + blk * 256 + rr * 16 + (i // 2) * 4 + (i % 2) * 2
            for b in range(2):
                vb.append(codes + scales + off + b)
                d0 = 64 * c + 4 * rr + 2 * b
                vd.append((d0, d0 + 1))
    vs = ks + codes + scales
    return (torch.stack(kb, 1), torch.tensor(kd), ks, torch.stack(vb, 1), torch.tensor(vd), vs)


@functools.lru_cache(maxsize=None)
def _maps_on(D: int, device: torch.device):
    """``_maps`` on a device, copied there once: a captured step may copy nothing from the host."""
    return tuple(z.to(device) for z in _maps(D))


def quantize_reference(x: torch.Tensor):
    """``[..., D]`` -> (codes + 8 as uint8 ``[..., D]``, bf16 scales ``[..., D/32]``)."""
    g = x.float().unflatten(-1, (-1, KV4_GROUP))
    hi, lo = g.amax(-1), g.amin(-1)
    s = torch.where(hi >= -lo, hi, lo) * -0.125
    s = torch.where(s.abs() * 8.0 < _TINY, torch.zeros_like(s), s).to(torch.bfloat16)
    s = torch.where(torch.isfinite(g).all(-1) & torch.isfinite(s), s, torch.full_like(s, math.nan))
    live = torch.isfinite(s) & (s != 0)
    c = torch.round(g / torch.where(live, s, torch.ones_like(s)).float()[..., None])
    c = torch.where(live[..., None], c.clamp(-8, 7), torch.zeros_like(c))
    return (c + 8).to(torch.uint8).flatten(-2), s


def _held(codes: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """fp32 values of codes + 8 ``[..., D]`` with scales ``[..., D/32]``."""
    return ((codes.float() - 8.0).unflatten(-1, (-1, KV4_GROUP)) * s.float()[..., None]).flatten(-2)


def _put(data: torch.Tensor, which: int, b, t, x: torch.Tensor, D: int, live):
    """Quantise rows ``x`` [N, KV, D] into tokens (sequence b[i], position t[i]); where ``live`` is false the token's bytes
    are written back as they were."""
    m = _maps_on(D, data.device)
    by, d, sc = m[3 * which], m[3 * which + 1], m[3 * which + 2]
    codes, s = quantize_reference(x)
    bytes_ = codes[..., d[:, 0]] | (codes[..., d[:, 1]] << 4)
    sb = s.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
    tile, tt = t // KV4_TILE, t % KV4_TILE
    kv = torch.arange(x.shape[1], device=data.device)
    bi, ki, ti, live = b[:, None, None], kv[None, :, None], tile[:, None, None], live[:, None, None]
    at = (bi, ki, ti, by[tt][:, None])
    data.index_put_(at, torch.where(live, bytes_, data[at]))
    for z in range(2):
        at = (bi, ki, ti, sc[tt][:, None] + z)
        data.index_put_(at, torch.where(live, sb[..., z], data[at]))


def _get(data: torch.Tensor, which: int, D: int) -> torch.Tensor:
    """fp32 values [B, KV, L, D] of a whole cache (L = its capacity)."""
    m = _maps_on(D, data.device)
    by, d, sc = m[3 * which], m[3 * which + 1], m[3 * which + 2]
    B, KV, tiles, _ = data.shape
    raw = data[..., by.reshape(-1)].view(B, KV, tiles * KV4_TILE, -1)
    codes = torch.empty(B, KV, tiles * KV4_TILE, D, dtype=torch.uint8, device=data.device)
    codes[..., d[:, 0]], codes[..., d[:, 1]] = raw & 15, raw >> 4
    s = torch.stack([data[..., sc.reshape(-1) + z] for z in range(2)], -1).contiguous().view(torch.bfloat16)
    return _held(codes, s.view(B, KV, tiles * KV4_TILE, D // KV4_GROUP))


def _check_cache(data: torch.Tensor, D: int) -> tuple[int, int, int]:
    rec = _record(D)
    if data.dtype != torch.uint8 or data.dim() != 4 or data.shape[3] != rec or not data.is_contiguous():
        raise ValueError(f"4-bit KV cache: expected a contiguous uint8 [B, KV, tiles, {rec}] tensor (kv4_alloc), "
                         f"got {data.dtype} {tuple(data.shape)}")
    return data.shape[0], data.shape[1], data.shape[2] * KV4_TILE


def _check_index(name: str, t: torch.Tensor, data: torch.Tensor, B: int):
    if t.dtype != torch.int32 or t.shape != (B,) or t.device != data.device or not t.is_contiguous():
        raise ValueError(f"{name}: int32 [{B}] on the cache's device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def kv4_store(data: torch.Tensor, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
              count: torch.Tensor | None = None) -> None:
    """Write rows ``k`` / ``v`` [B, n, KV*D] (views with unit column stride) to positions ``start[b] + i``.

    ``start`` int32 [B].  ``count`` (int32 [B], optional): only the first ``count[b]`` rows of sequence b are
    written (a padded batch).  Rows that fall outside the cache are not written; nothing else of the cache
    changes."""
    if use_hip(k) and k.dtype == torch.bfloat16:
        ext().kv4_store_(data, k, v, start, count)
        return
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.device != data.device:
        raise ValueError(f"kv4_store: k and v must be [B, n, KV*D] of one dtype on the cache's device, got "
                         f"{k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    KV = data.shape[1] if data.dim() == 4 else 0
    if KV == 0 or k.shape[2] % KV:
        raise ValueError(f"kv4_store: {k.shape[2]} columns for a cache of {KV} kv heads")
    D = k.shape[2] // KV
    B, KV, cap = _check_cache(data, D)
    if k.shape[0] != B:
        raise ValueError(f"kv4_store: {k.shape[0]} sequences for a cache of {B}")
    _check_index("kv4_store: start", start, data, B)
    if count is not None:
        _check_index("kv4_store: count", count, data, B)
    n = k.shape[1]
    if n == 0:
        return
    # rows lo..hi - 1 of a sequence are written; the others are its nearest one of those once more (the same bytes again),
    # so that nothing is read on the host
    i, first = torch.arange(n, device=data.device), start.long()[:, None]
    lo, hi = (-first).clamp(min=0), (cap - first).clamp(max=n)
    if count is not None:
        hi = torch.minimum(hi, count.long()[:, None])
    live = hi > lo
    r = torch.where(live, torch.minimum(torch.maximum(i, lo), hi - 1), torch.zeros_like(i))
    t = (first + r).clamp(0, cap - 1).flatten()
    b = torch.arange(B, device=data.device)[:, None].expand(B, n)
    for which, x in ((0, k), (1, v)):
        _put(data, which, b.flatten(), t, x[b, r].flatten(0, 1).unflatten(-1, (KV, D)), D, live.expand(B, n).flatten())


def kv4_load(data: torch.Tensor, start: torch.Tensor, n: int, D: int,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of positions ``start[b] + 0 .. n - 1``: K and V rows [B, n, KV*D] in ``dtype`` (positions
    outside the cache give zero rows)."""
    if use_hip(data) and dtype == torch.bfloat16:
        return ext().kv4_load(data, start, n, D)
    B, KV, cap = _check_cache(data, D)
    _check_index("kv4_load: start", start, data, B)
    if n < 0:
        raise ValueError(f"kv4_load: n must not be negative, got {n}")
    pos = start.long()[:, None] + torch.arange(n, device=data.device)
    ok = (pos >= 0) & (pos < cap)
    out = []
    for which in range(2):
        x = _get(data, which, D).gather(2, pos.clamp(0, cap - 1)[:, None, :, None].expand(B, KV, n, D))
        x = torch.where(ok[:, None, :, None], x, torch.zeros_like(x))
        out.append(x.transpose(1, 2).reshape(B, n, KV * D).to(dtype))
    return out[0], out[1]


def decode_attention_kv4_reference(q, data, lens, H: int, KV: int, D: int, scale: float, window: int = 0,
                                   sinks: int = 0) -> torch.Tensor:
    """q [B, >=H*D] against the first ``lens`` tokens of the cache -> [B, H*D] (fp32 math).  A sequence with
    no visible token gives a zero row."""
    B, cap = data.shape[0], data.shape[2] * KV4_TILE
    qf = q[:, :H * D].float().reshape(B, KV, H // KV, D)
    n = lens.long().clamp(max=cap)
    ok = visible_keys(n, cap, window, sinks)[:, None, None]
    s = (qf @ _get(data, 0, D).transpose(2, 3).contiguous()) * scale
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    v = torch.where(ok[:, :, 0, :, None], _get(data, 1, D), torch.zeros((), device=data.device))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = torch.where(ok, p, torch.zeros_like(p))
    o = (p @ v) / p.sum(-1, keepdim=True)
    return torch.where(n.view(B, 1, 1, 1) > 0, o, torch.zeros_like(o)).reshape(B, H * D).to(q.dtype)


def decode_attention_kv4(qkv: torch.Tensor, data: torch.Tensor, lens: torch.Tensor, max_len: int, H: int, KV: int,
                         D: int, scale: float | None = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """One query token per sequence against its 4-bit cache -> [B, H*D].

    ``qkv`` [B, (H+2KV)*D]: the current token's packed projection; its K / V rows are written at position
    ``lens - 1`` and attended to as they are held.  ``lens`` int32 [B] counts the current token; ``max_len``
    (host int) bounds it (a longer sequence is attended to over its first ``max_len`` tokens and not written).
    ``window`` > 0: the last ``window`` tokens and the first ``sinks`` are seen.  A sequence of length 0 writes
    nothing and gives a zero row.  ``scale`` must be positive (1 / sqrt(D) by default).  For inference: the output has
    no gradient, and a ``qkv`` with a forward-mode tangent is refused."""
    if has_tangent(qkv):
        raise NotImplementedError("decode_attention_kv4 has no derivative")
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if use_hip(qkv) and qkv.dtype == torch.bfloat16:
        return ext().decode_attention_kv4(qkv, data, lens, max_len, H, KV, D, scale, window or 0, sinks)
    qkv = qkv.detach()
    B, nkv, cap = _check_cache(data, D)
    if nkv != KV or KV < 1 or H < KV or H % KV:
        raise ValueError(f"decode_attention_kv4: {H} query / {KV} kv heads on a cache of {nkv}")
    if qkv.dim() != 2 or qkv.shape[0] != B or qkv.shape[1] < (H + 2 * KV) * D or qkv.device != data.device:
        raise ValueError(f"decode_attention_kv4: qkv must be [{B}, >={(H + 2 * KV) * D}] on the cache's device, got "
                         f"{tuple(qkv.shape)} on {qkv.device}")
    _check_index("decode_attention_kv4: lens", lens, data, B)
    if not 1 <= max_len <= cap:
        raise ValueError(f"decode_attention_kv4: max_len {max_len} outside the cache's 1..{cap}")
    if sinks < 0:
        raise ValueError(f"decode_attention_kv4: sinks must not be negative, got {sinks}")
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError(f"decode_attention_kv4: scale must be positive and finite, got {scale}")
    window = max(0, int(window or 0))
    new = qkv[:, H * D:(H + 2 * KV) * D].unflatten(1, (2, KV * D))
    kv4_store(data, new[:, None, 0], new[:, None, 1], torch.where(lens <= max_len, lens - 1, lens - lens - 1))
    return decode_attention_kv4_reference(qkv, data, lens.clamp(max=max_len), H, KV, D, scale, window, sinks)


class KV4Cache(KVCache):
    """``KVCache`` with its rows held in 4 bits: ``data`` [n_layers, B, KV, tiles, record].  Prefill attends over the
    prompt's own rows and stores them quantised; decode steps attend over the quantised cache."""

    def __init__(self, n_layers: int, B: int, max_len: int, KV: int, D: int, device):
        self._init_lens(B, max_len, KV, D, device)
        self.data = kv4_alloc(B, max_len, KV, D, device, layers=n_layers)
        self._zero = torch.zeros(1, dtype=torch.int32, device=device)

    def store(self, layer: int, qkv: torch.Tensor, H: int, S: int):
        k0, v0 = H * self.D, (H + self.KV) * self.D
        rows = qkv[None, :S]
        kv4_store(self.data[layer, self.row:self.row + 1], rows[..., k0:v0], rows[..., v0:v0 + self.KV * self.D], self._zero)

    def attend(self, layer: int, qkv: torch.Tensor, H: int, window: int = 0, sinks: int = 0) -> torch.Tensor:
        return decode_attention_kv4(qkv, self.data[layer], self.lens_next, self.attend_len(), H, self.KV, self.D,
                                    window=window, sinks=sinks)
