"""The language-model operators on the GPU against plain 64-bit
implementations (tests/lm_reference.py), at the sizes, layouts and masks where
they can go wrong.

Tolerances, derived:
* rope: the angle's fraction of a turn is rounded once to fp32 (2^-26 of a
  turn, 9.4e-8 radians), cos and sin are off by 2 ulp (1.2e-7), two products
  and a sum add 3 x 2^-24: 4e-7 (|a| + |b|); fp16 adds half a step, 2^-11.
* attention, fp16: the probabilities and the output are each rounded once, at
  most half a step of 2^-11 relative: 2^-10 of the values' size in all (the
  fp32 scores and sums are below a tenth of that). fp32: scores are sums of
  head_dim products and the output a sum of at most 4096, in fp32:
  2^-24 sqrt(terms) each as rounding errors add at random, times the score's
  size (up to 30) in the exponent: 1e-5 of the values' size.
"""

from __future__ import annotations

import math

import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def dev(t):
    return None if t is None else t.to("cuda")


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


# ------------------------------------------------------------------- rope_append

def rope_inputs(seed, dtype, tokens, heads, kv_heads, dim, rotary, page, axes=1, far=1 << 17):
    g = gen(seed)
    dt = DT[dtype]
    pages = (tokens + page - 1) // page + 2
    qkv = normal(g, tokens, (heads + 2 * kv_heads) * dim, dtype=dt)
    positions = torch.randint(0, far, (axes, tokens), generator=g).to(torch.int32)
    half = rotary // 2
    freq = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    caches = [normal(g, pages, kv_heads, page, dim, dtype=dt) for _ in range(2)]
    return qkv, positions, freq, slots, caches


def split(qkv, heads, kv_heads, dim):
    t = qkv.shape[0]
    return (qkv[:, :heads * dim].view(t, heads, dim),
            qkv[:, heads * dim:(heads + kv_heads) * dim].view(t, kv_heads, dim),
            qkv[:, (heads + kv_heads) * dim:].view(t, kv_heads, dim))


def check_rope(got, want, size, dtype):
    """`size`: |a| + |b| is at most twice the largest input."""
    err = (got.cpu().double() - want).abs()
    tol = 4e-7 * 2 * size + (2.0 ** -11 * want.abs() + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * want.abs())
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,page,axes", [
    (1, 32, 8, 128, 128, 16, 1),     # one token
    (64, 32, 8, 128, 128, 16, 1),
    (7, 12, 12, 64, 32, 24, 1),      # partial rotation, pages of 24
    (33, 6, 2, 80, 48, 5, 3),        # three axes
    (19, 3, 1, 80, 40, 16, 1),       # half a rotary width of 20: element accesses
    (5, 2, 2, 63, 42, 3, 2),         # odd head_dim
    (3, 1, 1, 1, 0, 1, 1),           # nothing rotates, one dim, pages of one token
    (300, 4, 4, 64, 64, 16, 1),
    (2, 1, 1, 2048, 2048, 2, 1),     # wider than the angle table
])
def test_rope_append(ops, dtype, interleaved, tokens, heads, kv_heads, dim, rotary, page, axes):
    qkv, positions, freq, slots, (kc, vc) = rope_inputs(
        tokens * 7 + dim, dtype, tokens, heads, kv_heads, dim, rotary, page, axes)
    axis = (torch.arange(rotary // 2, dtype=torch.int32) % axes).contiguous() if axes > 1 else None
    q, k, v = split(qkv, heads, kv_heads, dim)
    want = ref.rope_append(q, k, v, positions, freq, slots, kc, vc, axis, interleaved)
    dq, dk, dv = split(dev(qkv), heads, kv_heads, dim)
    dkc, dvc = dev(kc), dev(vc)
    qo, ko = ops.rope_append(dq, dk, dv, dev(positions), dev(freq), dev(slots), dkc, dvc,
                             axes=dev(axis), interleaved=interleaved, return_keys=True)
    size = float(qkv.abs().max())
    check_rope(qo, want[0], size, dtype)
    check_rope(ko, want[1], size, dtype)
    check_rope(dkc, want[2], size, dtype)
    assert torch.equal(dvc.cpu().double(), want[3])
    # the rows that no token was stored in are the old ones, bit for bit
    kept = torch.ones(kc.shape[0] * page, dtype=torch.bool)
    kept[slots.long()] = False
    rows = lambda c: c.cpu().transpose(1, 2).reshape(-1, kv_heads, dim)[kept]
    assert torch.equal(rows(dkc), rows(kc)) and torch.equal(rows(dvc), rows(vc))
    # the stored keys are the returned ones; without return_keys nothing else changes
    flat = dkc.transpose(1, 2).reshape(-1, kv_heads, dim)
    assert torch.equal(flat[dev(slots).long()], ko)
    kc2, vc2 = dev(kc), dev(vc)
    qo2, none = ops.rope_append(dq, dk, dv, dev(positions), dev(freq), dev(slots), kc2, vc2,
                                axes=dev(axis), interleaved=interleaved)
    assert none is None and torch.equal(qo2, qo)
    assert torch.equal(kc2, dkc) and torch.equal(vc2, dvc)


def test_rope_append_far_positions(ops):
    """Angles of positions up to 2^31 - 1 and below zero, frequency 1."""
    heads, dim = 2, 64
    positions = i32([2 ** 31 - 1, -2 ** 31, 1 << 24, 131071, -1, 0])
    g = gen(3)
    q, k, v = (normal(g, 6, heads, dim) for _ in range(3))
    freq = torch.ones(32)
    kc, vc = torch.zeros(1, heads, 8, dim), torch.zeros(1, heads, 8, dim)
    want = ref.rope_append(q, k, v, positions, freq, torch.arange(6), kc, vc)
    qo, _ = ops.rope_append(dev(q), dev(k), dev(v), dev(positions), dev(freq),
                            dev(i32(list(range(6)))), dev(kc), dev(vc))
    # 2^31 radians in 64 bits: the product with 1 / (2 pi) is off by 2^-53 of
    # 3.4e8 turns, 2.4e-7 radians, on either side
    err = (qo.cpu().double() - want[0]).abs().max()
    assert err <= (4e-7 + 5e-7) * 2 * float(q.abs().max()), float(err)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rope_append_skips_bad_slots_and_axes(ops, dtype):
    tokens, heads, kv_heads, dim, page = 6, 4, 2, 64, 4
    qkv, positions, freq, _, (kc, vc) = rope_inputs(5, dtype, tokens, heads, kv_heads, dim, 64, page)
    slots = i32([-1, 3, kc.shape[0] * page, 2 ** 31 - 1, -2 ** 31, 0])
    axis = torch.zeros(32, dtype=torch.int32)
    axis[5], axis[9] = -1, 1  # no such rows of positions: those pairs do not rotate
    q, k, v = split(qkv, heads, kv_heads, dim)
    want = ref.rope_append(q, k, v, positions, freq, slots, kc, vc, axis)
    dq, dk, dv = split(dev(qkv), heads, kv_heads, dim)
    dkc, dvc = dev(kc), dev(vc)
    qo, ko = ops.rope_append(dq, dk, dv, dev(positions), dev(freq), dev(slots), dkc, dvc,
                             axes=dev(axis), return_keys=True)
    size = float(qkv.abs().max())
    for got, exp in ((qo, want[0]), (ko, want[1]), (dkc, want[2])):
        check_rope(got, exp, size, dtype)
    assert torch.equal(dvc.cpu().double(), want[3])
    assert torch.equal(ko[:, :, [5, 9, 37, 41]], dk[:, :, [5, 9, 37, 41]])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rope_append_unaligned(ops, dtype):
    """Parts of a projection that start off a 16-byte border."""
    tokens, heads, kv_heads, dim = 9, 3, 3, 64
    g = gen(8)
    wide = normal(g, tokens, 3 * heads * dim + 1, dtype=DT[dtype])
    q, k, v = split(wide[:, 1:], heads, kv_heads, dim)
    _, positions, freq, slots, (kc, vc) = rope_inputs(8, dtype, tokens, heads, kv_heads, dim, 64, 16)
    want = ref.rope_append(q, k, v, positions, freq, slots, kc, vc)
    dq, dk, dv = split(dev(wide)[:, 1:], heads, kv_heads, dim)
    dkc, dvc = dev(kc), dev(vc)
    qo, _ = ops.rope_append(dq, dk, dv, dev(positions), dev(freq), dev(slots), dkc, dvc)
    check_rope(qo, want[0], float(wide.abs().max()), dtype)
    check_rope(dkc, want[2], float(wide.abs().max()), dtype)
    assert torch.equal(dvc.cpu().double(), want[3])


# --------------------------------------------------------------- paged_attention

def paged_inputs(seed, dtype, lengths, heads, kv_heads, dim, page, extra=3, fill=None):
    """A cache whose unused rows hold `fill` (NaN by default)."""
    g = gen(seed)
    dt = DT[dtype]
    used = [(max(n, 0) + page - 1) // page for n in lengths]
    width = max(max(used), 1)
    pages = sum(used) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)  # never read past a length
    kc = torch.full((pages, kv_heads, page, dim), math.nan if fill is None else fill, dtype=dt)
    vc = kc.clone()
    for b, n in enumerate(lengths):
        for p in range(used[b]):
            at = order.pop()
            table[b, p] = at
            m = min(page, n - p * page)
            kc[at, :, :m] = normal(g, kv_heads, m, dim, dtype=dt)
            vc[at, :, :m] = normal(g, kv_heads, m, dim, dtype=dt)
    q = normal(g, len(lengths), heads, dim, dtype=dt)
    return q, kc, vc, table, i32(lengths)


def check_attention(got, want, dtype):
    err = got.cpu().double() - want
    far, norm = float(err.norm()), float(want.norm())
    if dtype == "f16":
        assert far <= 2.0 ** -10 * norm + 1e-7, (far, norm)
        worst = float(err.abs().max())
        assert worst <= 2.0 ** -10 * max(float(want.abs().max()), 4.0), worst
    else:
        assert far <= 1e-5 * norm + 1e-12, (far, norm)


def run_paged(ops, t, **kw):
    kw = {n: dev(v) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    return ops.paged_attention(*(dev(x) for x in t), **kw)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [
    ([1], 1, 1, 64, 16),
    ([1, 2, 15, 16, 17], 32, 8, 128, 16),
    ([0, 5, 0, 31, 32, 33], 4, 4, 64, 16),
    ([127, 128, 129, 255, 256, 257], 8, 2, 128, 16),
    ([1000], 32, 8, 128, 16),
    ([700, 3, 1500, 0, 64], 12, 12, 64, 24),    # pages of 24: rows looked up one by one
    ([100, 37], 6, 2, 80, 1),                   # pages of one token
    ([333, 21], 4, 1, 96, 7),
    ([513], 16, 1, 128, 64),
    ([300, 40], 24, 1, 64, 128),                # 24 heads on a key head
    ([200, 129], 71, 1, 64, 16),                # three tiles of heads
    ([90, 200], 40, 1, 128, 5),
    ([4000], 2, 2, 128, 48),
    ([50], 3, 3, 8, 16),
])
def test_paged_attention(ops, dtype, lengths, heads, kv_heads, dim, page):
    t = paged_inputs(sum(lengths) + dim, dtype, lengths, heads, kv_heads, dim, page)
    check_attention(run_paged(ops, t), ref.paged_attention(*t), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("window,softcap,bias", [(1, 0.0, False), (17, 0.0, True), (64, 5.0, False),
                                                 (1000, 30.0, True), (2 ** 31 - 1, 0.0, False)])
def test_paged_attention_rules(ops, dtype, page, window, softcap, bias):
    lengths = [1, 16, 17, 400, 0, 1100]
    t = paged_inputs(11, dtype, lengths, 8, 2, 64, page)
    slopes = 2.0 ** -torch.arange(1.0, 9.0) if bias else None
    kw = dict(window=window, softcap=softcap, scale=0.5)
    want = ref.paged_attention(*t, slopes=slopes, **kw)
    check_attention(run_paged(ops, t, slopes=slopes, **kw), want, dtype)


# Small caps, both sides of the one past which fp16 takes the precise form, and caps
# that no score comes near.
CAPS = [2.0 ** -40, 0.02, 1024.0, 1025.0, 30000.0, 1e6, 2.0 ** 80]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("bias", [False, True])
def test_paged_attention_caps(ops, dtype, softcap, bias):
    t = paged_inputs(21, dtype, [1, 40, 300], 8, 2, 64, 16)
    kw = dict(softcap=softcap, slopes=2.0 ** -torch.arange(1.0, 9.0) if bias else None)
    check_attention(run_paged(ops, t, **kw), ref.paged_attention(*t, **kw), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("bias", [False, True])
def test_masked_attention_caps(ops, dtype, softcap, bias):
    t = masked_inputs(22, dtype, 2, 8, 2, 200, 64)
    kw = dict(causal=True, softcap=softcap, slopes=2.0 ** -torch.arange(1.0, 9.0) if bias else None)
    check_attention(run_masked(ops, t, **kw), ref.masked_attention(*t, **kw), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("scale", [2.0 ** -100, 1e-6])
def test_attention_small_scales(ops, dtype, scale):
    """Every visible key weighs the same."""
    t = paged_inputs(23, dtype, [1, 40, 300], 8, 2, 64, 16)
    check_attention(run_paged(ops, t, scale=scale), ref.paged_attention(*t, scale=scale), dtype)
    t = masked_inputs(24, dtype, 2, 8, 2, 200, 64)
    check_attention(run_masked(ops, t, causal=True, scale=scale),
                    ref.masked_attention(*t, causal=True, scale=scale), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_paged_attention_many_sequences(ops, dtype):
    """More sequences than a workgroup has threads, most of them short."""
    g = gen(4)
    lengths = torch.randint(0, 40, (600,), generator=g).tolist()
    lengths[17], lengths[599] = 900, 333
    t = paged_inputs(12, dtype, lengths, 2, 1, 64, 16)
    check_attention(run_paged(ops, t), ref.paged_attention(*t), dtype)


@pytest.mark.parametrize("page", [16, 12])
def test_paged_attention_bad_pages_and_lengths(ops, page):
    """Pages outside the cache are left out; lengths are cut to the table."""
    t = list(paged_inputs(13, "f16", [200, 90, 64], 4, 2, 64, page, fill=0.0))
    t[3][0, 1], t[3][0, 3], t[3][1, 0] = -1, t[1].shape[0], 2 ** 31 - 1
    t[3][2] = -1  # every page of the last sequence
    want = ref.paged_attention(*t)
    assert (want[2] == 0).all()
    check_attention(run_paged(ops, t), want, "f16")
    t[3] = t[3].clamp(0, t[1].shape[0] - 1)
    t[4] = i32([10 ** 9, -5, 64])
    check_attention(run_paged(ops, t), ref.paged_attention(*t), "f16")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("page", [16, 10])
def test_paged_attention_ignores_what_hidden_rows_hold(ops, dtype, page):
    """Infinities, NaN and the type's lowest value behind a length and before a window."""
    lengths, window = [45, 130, 257], 33
    t = paged_inputs(14, dtype, lengths, 4, 2, 64, page)
    want = ref.paged_attention(*t, window=window)
    q, kc, vc, table, _ = t
    bad = [math.inf, -math.inf, math.nan, torch.finfo(DT[dtype]).min]
    for b, n in enumerate(lengths):
        for j in range(n - window):
            at, off = int(table[b, j // page]), j % page
            kc[at, :, off], vc[at, :, off] = bad[j % 4], bad[(j + 1) % 4]
    check_attention(run_paged(ops, t, window=window), want, dtype)


def test_paged_attention_propagates_visible_nan(ops):
    t = paged_inputs(15, "f16", [40, 40], 2, 2, 64, 16)
    t[2][int(t[3][1, 0]), 1, 3, 7] = math.nan
    out = run_paged(ops, t).cpu()
    assert torch.isnan(out[1, 1, 7]) and int(torch.isnan(out).sum()) == 1


def test_paged_attention_low_probabilities(ops):
    """One key far above 8000 others: their share survives the rounding to fp16."""
    n, dim = 8001, 64
    q = torch.zeros(1, 1, dim, dtype=torch.float16)
    q[..., 0] = 8.0
    kc, vc = torch.zeros(1, 1, n, dim, dtype=torch.float16), torch.zeros(1, 1, n, dim, dtype=torch.float16)
    kc[0, 0, 4000, 0] = 12.0  # score 12 against 0: the others are 2^-17.3 each, 0.05 in all
    vc[0, 0, 4000, 0], vc[0, 0, :, 1] = 1.0, 1.0
    t = (q, kc, vc, i32([[0]]), i32([n]))
    check_attention(run_paged(ops, t), ref.paged_attention(*t), "f16")


def test_paged_attention_strided_inputs(ops):
    """q in a fused projection's output, a page table that is part of a wider one."""
    t = paged_inputs(16, "f16", [70, 33, 128], 4, 2, 64, 16)
    wide = torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda")
    wide[:, 2:6] = dev(t[0])
    table = torch.full((3, t[3].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    table[:, :t[3].shape[1]] = dev(t[3])
    got = ops.paged_attention(wide[:, 2:6], dev(t[1]), dev(t[2]), table[:, :t[3].shape[1]], dev(t[4]))
    assert torch.equal(got, run_paged(ops, t))


# -------------------------------------------------------------- masked_attention

def masked_inputs(seed, dtype, batch, heads, kv_heads, seq, dim, token_major=True):
    g = gen(seed)
    dt = DT[dtype]
    if token_major:
        return [normal(g, batch, seq, h, dim, dtype=dt).transpose(1, 2) for h in (heads, kv_heads, kv_heads)]
    return [normal(g, batch, h, seq, dim, dtype=dt) for h in (heads, kv_heads, kv_heads)]


def run_masked(ops, t, **kw):
    kw = {n: dev(v) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    return ops.masked_attention(*(dev(x) for x in t), **kw)


SIZES = [  # batch, heads, kv_heads, seq, dim
    (1, 1, 1, 1, 64), (2, 4, 2, 17, 64), (1, 3, 1, 64, 128), (2, 2, 2, 131, 80),
    (1, 8, 2, 257, 128), (1, 2, 1, 500, 96), (3, 40, 8, 130, 64), (2, 48, 12, 129, 128),
    (1, 1, 1, 33, 8),
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_masked_attention_plain(ops, dtype, causal, size):
    t = masked_inputs(size[3], dtype, *size)
    out = run_masked(ops, t, causal=causal)
    assert out.shape == t[0].shape and out.dtype == DT[dtype]
    check_attention(out, ref.masked_attention(*t, causal=causal), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [(2, 4, 2, 200, 64), (2, 40, 20, 330, 128)])
@pytest.mark.parametrize("window,softcap,bias,prefix", [
    (0, 20.0, False, None), (0, 0.0, True, None), (1, 0.0, False, None), (50, 0.0, False, None),
    (50, 5.0, True, [3, 150]), (0, 0.0, False, [0, 190]), (129, 0.0, False, [10 ** 6, -4]),
    (2 ** 31 - 1, 0.0, False, None),
])
def test_masked_attention_rules(ops, dtype, causal, size, window, softcap, bias, prefix):
    t = masked_inputs(window % 1000 + size[3], dtype, *size)
    kw = dict(causal=causal, window=window, softcap=softcap, scale=0.3,
              slopes=2.0 ** (-8 * torch.arange(1.0, size[1] + 1) / size[1]) if bias else None,
              prefixes=i32(prefix) if prefix else None)
    check_attention(run_masked(ops, t, **kw), ref.masked_attention(*t, **kw), dtype)


def documents_of(kind, batch, seq):
    if kind == "packed":
        row = [i // 37 for i in range(seq)]
    elif kind == "padded":  # padding in front, in the middle, behind
        row = [-1 if i < 5 or 70 <= i < 140 or i >= seq - 9 else 3 + i // 90 for i in range(seq)]
    elif kind == "long":
        row = [0 if i < seq // 2 else 1 for i in range(seq)]
    elif kind == "mixed":   # ids in no order
        row = [(i * 7919) % 5 - 1 for i in range(seq)]
    elif kind == "one":
        row = [2 ** 31 - 1] * seq
    else:
        row = [-3] * seq
    rows = [row] + [list(reversed(row)) for _ in range(batch - 1)]
    return i32(rows)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [(2, 2, 1, 300, 64), (2, 40, 20, 333, 128)])
@pytest.mark.parametrize("kind", ["packed", "padded", "long", "mixed", "one", "none"])
def test_masked_attention_documents(ops, dtype, causal, size, kind):
    t = masked_inputs(21, dtype, *size)
    docs = documents_of(kind, size[0], size[3])
    prefixes = i32([40, 0])
    for kw in (dict(), dict(window=60, prefixes=prefixes)):
        got = run_masked(ops, t, causal=causal, documents=docs, **kw)
        check_attention(got, ref.masked_attention(*t, causal=causal, documents=docs, **kw), dtype)
    assert (got.cpu()[:, :, docs[0] < 0][0] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [(1, 2, 1, 150, 64), (1, 48, 24, 200, 128), (1, 2, 2, 150, 128)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, "lowest"])
def test_masked_attention_ignores_what_masked_rows_hold(ops, dtype, size, bad):
    """Padding tokens, and tokens later than a query, with anything in them."""
    t = masked_inputs(22, dtype, *size)
    seq = size[3]
    docs = torch.zeros(1, seq, dtype=torch.int32)
    docs[:, 20:30], docs[:, 100:] = -1, 1
    docs[:, seq - 3:] = -1
    value = torch.finfo(DT[dtype]).min if bad == "lowest" else bad
    want = ref.masked_attention(*t, causal=True, documents=docs)
    hidden = docs[0] < 0
    for x in t:
        x[:, :, hidden] = value
    check_attention(run_masked(ops, t, causal=True, documents=docs), want, dtype)
    # causal: a bad last token changes its own row only
    t = masked_inputs(23, dtype, *size)
    want = ref.masked_attention(*t, causal=True)
    for x in t[1:]:
        x[:, :, -1] = value
    got = run_masked(ops, t, causal=True).cpu()
    check_attention(got[:, :, :-1], want[:, :, :-1], dtype)
    if bad != "lowest":
        assert not torch.isfinite(got[:, :, -1]).any()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [(1, 2, 1, 150, 64), (1, 48, 24, 200, 128)])
def test_masked_attention_visible_infinity(ops, dtype, size):
    """An infinite value reaches the rows that see it, with its sign, and no others."""
    t = masked_inputs(24, dtype, *size)
    t[2][0, 0, 70, 3], t[2][0, 0, 90, 5] = math.inf, math.nan
    got = run_masked(ops, t, causal=True, window=40).cpu().double()
    want = ref.masked_attention(*t, causal=True, window=40)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and (got[torch.isinf(got)] > 0).all()
    fine = torch.isfinite(want)
    check_attention(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), dtype)


def test_masked_attention_layouts(ops):
    """Head-major, token-major, parts of a fused projection and shared heads give the same bits."""
    b, h, hk, s, d = 2, 6, 2, 90, 64
    t = masked_inputs(25, "f16", b, h, hk, s, d, token_major=False)
    want = run_masked(ops, t, causal=True)
    assert want.is_contiguous()
    major = [dev(x).transpose(1, 2).contiguous().transpose(1, 2) for x in t]
    got = ops.masked_attention(*major, causal=True)
    assert got.transpose(1, 2).is_contiguous() and torch.equal(got, want)
    fused = torch.cat([dev(x).transpose(1, 2).reshape(b, s, -1) for x in t], dim=-1)
    q, k, v = (p.view(b, s, -1, d).transpose(1, 2) for p in fused.split([h * d, hk * d, hk * d], dim=-1))
    assert torch.equal(ops.masked_attention(q, k, v, causal=True), want)
    one = ops.masked_attention(dev(t[0]), dev(t[1])[:, :1].expand(b, 2, s, d), dev(t[2])[:, :1].expand(b, 2, s, d))
    many = ops.masked_attention(dev(t[0]), dev(t[1])[:, :1], dev(t[2])[:, :1])
    assert torch.equal(one, many)
    single = ops.masked_attention(dev(t[0])[:, :, :1], dev(t[1])[:, :, :1], dev(t[2])[:, :, :1])
    assert torch.equal(single, dev(t[2])[:, :, :1].repeat_interleave(h // hk, 1))


# ------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("softcap,bias,window", [(0.0, False, 0), (20.0, False, 100), (0.0, True, 0)])
def test_prompt_then_decode(ops, dtype, softcap, bias, window):
    """A prompt stored and attended to, then tokens one by one: each new token's
    attention over the cache is the last row of a prompt that ends with it."""
    g = gen(31)
    dt, h, hk, d, page, total, prompt = DT[dtype], 8, 2, 64, 16, 150, 140
    qkv = normal(g, total, (h + 2 * hk) * d, dtype=dt).cuda()
    freq = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    slopes = (2.0 ** -torch.arange(1.0, h + 1)).cuda() if bias else None
    pages = (total + page - 1) // page
    table = torch.randperm(pages + 2, generator=g)[:pages].to(torch.int32).cuda()
    slots = (table[:, None] * page + torch.arange(page, dtype=torch.int32).cuda()).reshape(-1)[:total].contiguous()
    kc, vc = (torch.full((pages + 2, hk, page, d), math.nan, dtype=dt, device="cuda") for _ in range(2))
    positions = torch.arange(total, dtype=torch.int32).cuda()
    rules = dict(softcap=softcap, slopes=slopes, window=window)

    def step(a, b):
        q, k, v = split(qkv[a:b], h, hk, d)
        qo, ko = ops.rope_append(q, k, v, positions[a:b], freq, slots[a:b], kc, vc, return_keys=True)
        return qo, ko, v

    qs, ks, vs = [], [], []
    for a, b in [(0, prompt)] + [(i, i + 1) for i in range(prompt, total)]:
        q, k, v = step(a, b)
        qs.append(q), ks.append(k), vs.append(v)
        qh, kh, vh = (torch.cat(x).transpose(0, 1)[None] for x in (qs, ks, vs))
        whole = ops.masked_attention(qh, kh, vh, causal=True, **rules)[0].transpose(0, 1)
        one = ops.paged_attention(q[-1:], kc, vc, table[None], i32([b]).cuda(), **rules)
        want = ref.masked_attention(qh.cpu(), kh.cpu(), vh.cpu(), causal=True, softcap=softcap, window=window,
                                    slopes=None if slopes is None else slopes.cpu())[0].transpose(0, 1)
        check_attention(whole, want, dtype)
        check_attention(one, want[-1:], dtype)


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (40, 2)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 24])
def test_paged_attention_wide_cap_instances(ops, heads, kv_heads, dim, page):
    """Caps past kSigmaCap have instances of their own; also of a cache that is streamed."""
    t = paged_inputs(25, "f16", [70, 600], heads, kv_heads, dim, page)
    check_attention(run_paged(ops, t, softcap=1e5), ref.paged_attention(*t, softcap=1e5), "f16")
    q, kc, vc, table, lengths = (dev(x) for x in t)
    wide = (200 << 20) // (2 * kv_heads * page * dim * 2) + 1   # pages of 200 MiB
    kw, vw = (torch.zeros(wide, *kc.shape[1:], dtype=kc.dtype, device="cuda") for _ in range(2))
    kw[-kc.shape[0]:], vw[-kc.shape[0]:] = kc, vc
    reach = torch.zeros(2, wide, dtype=torch.int32, device="cuda")
    reach[:, :table.shape[1]] = table + (wide - kc.shape[0])
    got = ops.paged_attention(q, kw, vw, reach, lengths, softcap=1e5)
    check_attention(got, ref.paged_attention(*t, softcap=1e5), "f16")


@pytest.mark.parametrize("route", [r for r in ref.MASKED_ROUTES if r[0] == "f16"],
                         ids=lambda r: "-".join(map(str, r)).replace(" ", ""))
def test_masked_attention_wide_cap_is_no_cap(ops, route):
    """Every launch shape, without slopes: 1e6 tanh(s / 1e6) differs from s by s^3 / 3e12."""
    _, dim, _, batch, heads, seq, causal, window = route
    g = torch.Generator(device="cuda").manual_seed(seq)
    q, k, v = (torch.randn(batch, h, seq, dim, generator=g, device="cuda").half() for h in (heads, heads // 2, heads // 2))
    got = ops.masked_attention(q, k, v, causal=causal, window=window, softcap=1e6)
    check_attention(got, ops.masked_attention(q, k, v, causal=causal, window=window).double().cpu(), "f16")
