"""Plain 64-bit implementations of the language-model operators, on the CPU,
and the input builders their tests share."""

from __future__ import annotations

import math

import torch

INF = math.inf


def rotate(x, positions, frequencies, axes=None, interleaved=False):
    """x [tokens, heads, dim]; positions [rows, tokens]."""
    x = x.double().clone()
    half = frequencies.numel()
    axis = torch.zeros(half, dtype=torch.long) if axes is None else axes.long()
    ok = (axis >= 0) & (axis < positions.shape[0])
    p = positions.double()[axis.clamp(0, positions.shape[0] - 1)].t() * ok  # [tokens, half]
    t = (p * frequencies.double())[:, None]
    c, s = t.cos(), t.sin()
    lo = torch.arange(half) * 2 if interleaved else torch.arange(half)
    hi = lo + 1 if interleaved else lo + half
    a, b = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo], x[..., hi] = a * c - b * s, b * c + a * s
    return x


def rope_append(q, k, v, positions, frequencies, slots, key_cache, value_cache, axes=None,
                interleaved=False):
    """Returns (q_out, k_out, key_cache, value_cache) in 64 bits."""
    if positions.dim() == 1:
        positions = positions[None]
    qo = rotate(q, positions, frequencies, axes, interleaved)
    ko = rotate(k, positions, frequencies, axes, interleaved)
    kc, vc = key_cache.double().clone(), value_cache.double().clone()
    page = kc.shape[2]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < kc.shape[0] * page:
            kc[s // page, :, s % page] = ko[t]
            vc[s // page, :, s % page] = v[t].double()
    return qo, ko, kc, vc


def _rows(q, k, v, visible, distance, scale, softcap, slope):
    """q [n, d], k and v [m, d]: only visible keys and values are touched."""
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    for i in range(q.shape[0]):
        seen = visible[i].nonzero()[:, 0]
        if not len(seen):
            continue
        s = (k[seen].double() * q[i].double()).sum(-1) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slope is not None:
            s = s - float(slope) * distance[i, seen].double()
        p = torch.softmax(s, 0)
        out[i] = (p[:, None] * v[seen].double()).sum(0)
    return out


def paged_attention(q, key_cache, value_cache, page_table, lengths, scale=None, window=0,
                    softcap=0.0, slopes=None):
    batch, heads, dim = q.shape
    pages, kv_heads, page = key_cache.shape[:3]
    scale = scale or 1.0 / math.sqrt(dim)
    out = torch.zeros(batch, heads, dim, dtype=torch.float64)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), page_table.shape[1] * page)
        at = [j for j in range(max(0, n - window) if window else 0, n)
              if 0 <= int(page_table[b, j // page]) < pages]
        if not at:
            continue
        rows = torch.tensor([int(page_table[b, j // page]) for j in at])
        off = torch.tensor([j % page for j in at])
        distance = (n - 1 - torch.tensor(at))[None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            out[b, h] = _rows(q[b, h][None], key_cache[rows, g, off], value_cache[rows, g, off],
                              torch.ones(1, len(at), dtype=torch.bool), distance, scale, softcap,
                              None if slopes is None else slopes[h])[0]
    return out


def visible_keys(seq, b, causal, window, documents, prefixes):
    i = torch.arange(seq)
    distance = i[:, None] - i
    seen = distance >= 0 if causal else torch.ones(seq, seq, dtype=torch.bool)
    if window:
        seen = seen & (distance.abs() < window)
    if prefixes is not None:
        seen = seen | (i < int(prefixes[b]))
    if documents is not None:
        ids = documents[b]
        seen = seen & (ids[:, None] == ids) & (ids >= 0)[:, None]
    return seen, distance.abs()


def masked_attention(q, k, v, causal=False, window=0, softcap=0.0, slopes=None, documents=None,
                     prefixes=None, scale=None):
    batch, heads, seq, dim = q.shape
    scale = scale or 1.0 / math.sqrt(dim)
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        seen, distance = visible_keys(seq, b, causal, window, documents, prefixes)
        for h in range(heads):
            g = h // (heads // k.shape[1])
            kh, vh = k[b, g].double(), v[b, g].double()
            if torch.isfinite(kh).all() and torch.isfinite(vh).all():
                s = (q[b, h].double() @ kh.t()) * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - float(slopes[h]) * distance.double()
                s = s.masked_fill(~seen, -INF)
                m = s.amax(-1, keepdim=True)
                p = (s - m.masked_fill(m == -INF, 0.0)).exp()
                out[b, h] = (p @ vh) / p.sum(-1, keepdim=True).clamp_min(1e-300)
            else:  # non-finite values: only what a row sees
                out[b, h] = _rows(q[b, h], kh, vh, seen, distance, scale, softcap,
                                  None if slopes is None else slopes[h])
    return out


# Shapes that reach every instance of masked_attention: (dtype, head_dim,
# (groups, wavefronts, tile keys), batch, heads, sequence, causal, window).
_WIDE_F16 = [((4, 1, 32), 1, 2, 150, True, 0), ((1, 2, 32), 9, 16, 150, True, 0), ((4, 2, 32), 1, 24, 500, False, 0),
             ((2, 2, 32), 1, 20, 1000, True, 0), ((2, 4, 64), 1, 20, 1000, False, 0),
             ((2, 4, 64), 1, 20, 1600, True, 0), ((1, 4, 64), 1, 40, 1000, False, 90)]
_NARROW_F16 = [((4, 1, 32), 1, 2, 150, True, 0), ((1, 2, 32), 9, 16, 150, False, 0), ((2, 2, 64), 1, 20, 1000, False, 0),
               ((2, 4, 64), 1, 20, 1600, True, 0), ((1, 4, 64), 1, 40, 1000, True, 0)]
_WIDE_F32 = [((2, 2, 32), 1, 2, 150, True, 0), ((2, 2, 32), 1, 20, 1000, True, 0), ((1, 2, 32), 1, 40, 1000, True, 0),
             ((1, 4, 32), 1, 40, 1000, False, 0)]
_NARROW_F32 = [((4, 1, 32), 1, 2, 150, True, 0), ((2, 2, 32), 1, 20, 500, False, 0), ((1, 2, 32), 1, 40, 1000, False, 0),
               ((1, 4, 32), 1, 64, 1000, False, 90)]
MASKED_ROUTES = ([("f16", d, *r) for d in (128, 80) for r in _WIDE_F16] + [("f16", 64, *r) for r in _NARROW_F16]
                 + [("f32", d, *r) for d in (128, 80) for r in _WIDE_F32] + [("f32", 64, *r) for r in _NARROW_F32])
