"""Every compiled variant of the language-model operators on the GPU, and the
calls that their documentation allows beyond the plain ones: the C ABI's plain
and workspace forms, streams, threads, captured and replayed graphs, caches past
32-bit offsets, long sequences, wide strides, shared pages, repeated slots.
Tolerances as in tests/test_lm_ops.py; references in 64 bits."""

from __future__ import annotations

import ctypes
import math
import threading

import pytest
import torch

import lm_reference as ref
import operatorlib
from gpu_util import ptr, stream_handle
from test_lm_ops import DT, check_attention, dev, gen, i32, normal, paged_inputs, run_paged, split

pytestmark = pytest.mark.gpu


def on_gpu(q, k, v, causal, window, softcap, slopes, documents, prefixes=None):
    """masked_attention in 64 bits on the GPU, a head at a time."""
    b, h, s, d = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        seen, distance = ref.visible_keys(s, i, causal, window, None if documents is None else documents.cpu(),
                                          None if prefixes is None else prefixes.cpu())
        seen, distance = seen.cuda(), distance.cuda().double()
        for j in range(h):
            g = j // (h // k.shape[1])
            x = torch.mm(q[i, j].double(), k[i, g].double().t().contiguous()) / math.sqrt(d)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - slopes[j].double() * distance
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(-1, keepdim=True)
            p = (x - m.masked_fill(m == -math.inf, 0.0)).exp()
            out[i, j] = torch.mm(p, v[i, g].double()) / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return out


def packed(batch, seq):
    """Documents of 3 to 211 tokens; padding in the middle and at the end."""
    row, n, i = [], 3, 0
    while len(row) < seq:
        row += [i if i % 5 != 4 else -1] * n
        n, i = (n * 7) % 211 + 3, i + 1
    row = row[:seq - 2] + [-1] * min(2, seq)
    return i32([row[:seq]] * batch)


@pytest.mark.parametrize("route", ref.MASKED_ROUTES, ids=lambda r: "-".join(map(str, r)).replace(" ", ""))
@pytest.mark.parametrize("capped", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_masked_attention_instance(ops, route, capped, biased):
    dtype, dim, _, batch, heads, seq, causal, window = route
    g = torch.Generator(device="cuda").manual_seed(seq + heads)
    q, k, v = (torch.randn(batch, seq, h, dim, generator=g, device="cuda").to(DT[dtype]).transpose(1, 2)
               for h in (heads, heads // 2, heads // 2))
    slopes = 2.0 ** (-8 * torch.arange(1.0, heads + 1, device="cuda") / heads) if biased else None
    softcap = 8.0 if capped else 0.0
    got = ops.masked_attention(q, k, v, causal=causal, window=window, softcap=softcap, slopes=slopes)
    check_attention(got, on_gpu(q, k, v, causal, window, softcap, slopes, None).cpu(), dtype)
    # with documents, and anything at all in the padding
    docs = packed(batch, seq)
    want = on_gpu(q, k, v, causal, window, softcap, slopes, docs)
    hidden = (docs[0] < 0).cuda()
    for x in (q, k, v):
        x[:, :, hidden] = math.nan
    got = ops.masked_attention(q, k, v, causal=causal, window=window, softcap=softcap, slopes=slopes, documents=docs.cuda())
    check_attention(got, want.cpu(), dtype)


def test_masked_attention_past_the_marks(ops):
    """Documents of more than 2^18 keys, the largest sequence: the tiles behind the
    marks are all visited; rows checked here and there."""
    for seq in (2 ** 18 + 1000, 2 ** 20):
        g = torch.Generator(device="cuda").manual_seed(1)
        q, k, v = (torch.randn(1, 1, seq, 16, generator=g, device="cuda").half() for _ in range(3))
        docs = (torch.arange(seq, device="cuda") // 5000).to(torch.int32)
        docs[2 ** 18 + 100:2 ** 18 + 300] = -1
        got = ops.masked_attention(q, k, v, causal=True, window=3000, documents=docs[None])
        for i in (0, 4999, 5000, 2 ** 18 - 1, 2 ** 18, 2 ** 18 + 99, 2 ** 18 + 150, 2 ** 18 + 305, seq - 1):
            seen = [j for j in range(max(0, i - 2999), i + 1) if docs[j] == docs[i] and docs[i] >= 0] if i != 2 ** 18 + 150 else []
            if not seen:
                assert (got[0, 0, i] == 0).all()
                continue
            x = (k[0, 0, seen].double() * q[0, 0, i].double()).sum(-1) / 4.0
            want = torch.softmax(x, 0) @ v[0, 0, seen].double()
            check_attention(got[0, 0, i], want.cpu(), "f16")


def test_masked_attention_wide_strides(ops):
    """Tokens a megabyte apart: offsets within a head up to 2^31 bytes."""
    seq, stride = 1000, 1_000_000
    wide = torch.zeros(seq * stride, dtype=torch.float16, device="cuda")
    view = wide.as_strided((1, 1, seq, 64), (0, 0, stride, 1))
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(1, 1, seq, 64, generator=g, device="cuda").half() for _ in range(3))
    view.copy_(k)
    assert torch.equal(ops.masked_attention(q, view, v, causal=True), ops.masked_attention(q, k, v, causal=True))
    view.copy_(v)
    assert torch.equal(ops.masked_attention(q, k, view), ops.masked_attention(q, k, v))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_masked_attention_c_abi(dtype, device):
    lib = operatorlib.lm_clib()
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(2, h, 100, 64, generator=g, device="cuda").to(DT[dtype]) for h in (4, 2, 2))
    out = torch.full_like(q, math.nan)
    s = lambda h: operatorlib.Strides(h * 6400, 6400, 64)
    fn = getattr(lib, f"operatorlib_masked_attention_{dtype}")
    assert fn(ptr(q), s(4), ptr(k), s(2), ptr(v), s(2), None, None, None, ptr(out), s(4), 2, 4, 2, 100, 64,
              0.125, 1, 0, 0.0, stream_handle()) == 0
    torch.cuda.synchronize()
    check_attention(out, ref.masked_attention(q.cpu(), k.cpu(), v.cpu(), causal=True), dtype)


# ------------------------------------------------------------- paged attention

def c_args(t, out, dim, heads, kv, page):
    q, kc, vc, table, lengths = t
    return [ptr(q), heads * dim, ptr(kc), ptr(vc), ptr(table), table.shape[1], ptr(lengths), None, ptr(out),
            q.shape[0], heads, kv, dim, kc.shape[0], page, table.shape[1], 1.0 / math.sqrt(dim), 0, 0.0]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lengths", [[900, 3], [300] * 90 + [2000], [5000]])
def test_paged_attention_forms_agree(ops, dtype, lengths):
    """The arena, a workspace of exactly the queried bytes and the torch operator: the same bits."""
    lib = operatorlib.lm_clib()
    heads, kv, dim, page = 8, 2, 128, 16
    t = [dev(x) for x in paged_inputs(41, dtype, lengths, heads, kv, dim, page, fill=0.0)]
    want = ops.paged_attention(*t)
    out = torch.full_like(want, math.nan)
    args = c_args(t, out, dim, heads, kv, page)
    assert getattr(lib, f"operatorlib_paged_attention_{dtype}")(*args, stream_handle()) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    need = getattr(lib, f"operatorlib_paged_attention_{dtype}_workspace_size")(
        len(lengths), heads, kv, dim, page, t[3].shape[1])
    assert need > 0
    ws = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    out.fill_(math.nan)
    fn = getattr(lib, f"operatorlib_paged_attention_{dtype}_ws")
    assert fn(*args, ptr(ws), need, stream_handle()) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert (ws[need:] == 0xAB).all()  # nothing behind the queried bytes
    assert fn(*args, ptr(ws), need - 1, stream_handle()) == 1


def test_paged_attention_past_32_bits(ops):
    """A cache of 9.4 GB per tensor: pages and slots whose elements lie past 2^32."""
    pages, kv, page, dim, heads = 36000, 8, 128, 128, 16
    kc, vc = (torch.zeros(pages, kv, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 32
    g = gen(5)
    n = 300
    table = i32([[35999, 33000, 2]])
    slots = torch.cat([table[0, j // page] * page + torch.arange(j, min(j + page, n)) % page for j in range(0, n, page)])
    qkv = normal(g, n, (heads + 2 * kv) * dim, dtype=torch.float16)
    q, k, v = split(qkv, heads, kv, dim)
    freq = torch.full((64,), 0.01)
    positions = torch.arange(n, dtype=torch.int32)
    dq, dk, dv = split(dev(qkv), heads, kv, dim)
    qo, ko = ops.rope_append(dq, dk, dv, dev(positions), dev(freq), dev(slots.to(torch.int32)), kc, vc, return_keys=True)
    assert torch.equal(kc[35999, :, 5], ko[5]) and torch.equal(vc[33000, :, 7], dv[128 + 7])
    assert torch.equal(kc[2, :, 43], ko[299]) and int((kc != 0).any(-1).any(-1).any(-1).sum()) == 3
    got = ops.paged_attention(qo[-1:], kc, vc, dev(table), dev(i32([n])))
    small = i32([[2, 1, 0]])
    order = torch.tensor([2, 33000, 35999]).cuda()
    assert torch.equal(got, ops.paged_attention(qo[-1:], kc[order].contiguous(), vc[order].contiguous(), dev(small), dev(i32([n]))))
    want = ref.paged_attention(qo[-1:].cpu(), kc[order].cpu(), vc[order].cpu(), small, i32([n]))
    check_attention(got, want, "f16")


@pytest.mark.parametrize("page", [16, 24])
def test_paged_attention_streamed_cache(ops, page):
    """A cache large enough for the non-temporal reads: the same results as a small one."""
    t = paged_inputs(17, "f16", [500, 70, 1300], 8, 8, 128, page, fill=0.0)
    want = ref.paged_attention(*t)
    q, kc, vc, table, lengths = (dev(x) for x in t)
    pages = 2 * 10 ** 8 // (8 * page * 128 * 4) + kc.shape[0]
    big = [torch.zeros(pages, *kc.shape[1:], dtype=torch.float16, device="cuda") for _ in range(2)]
    for b, c in zip(big, (kc, vc)):
        b[-kc.shape[0]:] = c
    wide = torch.full((3, 30000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table + (pages - kc.shape[0])
    check_attention(ops.paged_attention(q, *big, wide, lengths), want, "f16")


def test_paged_attention_shared_pages(ops):
    """Sequences that begin with the same pages."""
    t = list(paged_inputs(18, "f16", [200, 200, 200], 4, 2, 64, 16, fill=0.0))
    t[3][1, :8] = t[3][0, :8]
    t[3][2] = t[3][0]
    check_attention(run_paged(ops, t), ref.paged_attention(*t), "f16")


def test_rope_append_repeated_slots(ops):
    """Of two tokens with one slot every element keeps one or the other's."""
    g = gen(6)
    qkv = normal(g, 8, 3 * 2 * 64).cuda()
    q, k, v = split(qkv, 2, 2, 64)
    kc, vc = torch.zeros(2, 2, 4, 64, device="cuda"), torch.zeros(2, 2, 4, 64, device="cuda")
    slots = i32([5, 5, 5, 5, 1, 1, 2, 2]).cuda()
    _, ko = ops.rope_append(q, k, v, torch.arange(8, dtype=torch.int32).cuda(), torch.ones(32, device="cuda"), slots,
                            kc, vc, return_keys=True)
    for slot, tokens in ((5, range(4)), (1, (4, 5)), (2, (6, 7))):
        for cache, rows in ((kc, ko), (vc, v)):
            kept = cache[slot // 4, :, slot % 4]
            assert torch.stack([kept == rows[t] for t in tokens]).any(0).all()
    assert (kc[0, :, [0, 3]] == 0).all() and (kc[1, :, [0, 2, 3]] == 0).all()


# ------------------------------------------------ streams, threads and graphs

class Decoder:
    """The operators as a program runs them: a prompt, then steps over a batch."""

    def __init__(self, ops, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ops, self.h, self.hk, self.d, self.page, self.b = ops, 8, 2, 64, 16, 5
        n = 40
        self.kc, self.vc = (torch.zeros(self.b * n, self.hk, self.page, self.d, device="cuda", dtype=DT[dtype]) for _ in range(2))
        self.table = torch.randperm(self.b * n, generator=g, device="cuda").to(torch.int32).view(self.b, n)
        self.freq = (100.0 ** (-torch.arange(32, device="cuda") / 32.0)).float()
        self.lengths = i32([1, 200, 17, 0, 513]).cuda()
        for c in (self.kc, self.vc):
            c.copy_(torch.randn(c.shape, generator=g, device="cuda"))
        self.x = torch.randn(self.b, (self.h + 2 * self.hk) * self.d, generator=g, device="cuda").to(DT[dtype])
        self.positions = self.lengths.clone()
        self.slots = torch.zeros_like(self.lengths)
        self.place()
        self.prompt = [torch.randn(1, 300, h, self.d, generator=g, device="cuda").to(DT[dtype]).transpose(1, 2) for h in (8, 2, 2)]
        self.docs = (torch.arange(300, device="cuda") // 70).to(torch.int32)[None]

    def place(self):
        """Room for one more token in every sequence (in place)."""
        at = self.lengths.long()
        page = self.table.gather(1, (at // self.page)[:, None])[:, 0]
        self.slots.copy_(page * self.page + at % self.page)
        self.positions.copy_(self.lengths)
        self.lengths.add_(1)

    def step(self):
        q, k, v = split(self.x, self.h, self.hk, self.d)
        qo, _ = self.ops.rope_append(q, k, v, self.positions, self.freq, self.slots, self.kc, self.vc)
        out = self.ops.paged_attention(qo, self.kc, self.vc, self.table, self.lengths, softcap=20.0)
        prompt = self.ops.masked_attention(*self.prompt, causal=True, documents=self.docs)
        return out, prompt


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_graph_replays_follow_the_state(ops, dtype):
    """A captured decode step, replayed as the sequences grow, with eager work between."""
    eager, replayed = Decoder(ops, dtype, 1), Decoder(ops, dtype, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        warm = Decoder(ops, dtype, 2)
        warm.step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = replayed.step()
    # (the capture ran nothing: both caches are the same until here)
    for i in range(5):
        want = eager.step()
        for y in outs:
            y.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
        assert torch.equal(eager.kc, replayed.kc) and torch.equal(eager.vc, replayed.vc)
        for d in (eager, replayed):
            d.place()
            d.x.mul_(-1.1)
        ops.softmax(torch.ones(3, 50001, device="cuda"))
    # ended sequences: lengths of zero, slots of padding
    for d in (eager, replayed):
        d.lengths[2:4], d.slots[2:4] = 0, -1
    want = eager.step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and (outs[0][2:4] == 0).all()


def test_two_graphs_at_once(ops):
    """Two captured steps replayed on two streams at the same time."""
    steps, graphs, outs, wants = [], [], [], []
    for i in range(2):
        d = Decoder(ops, "f16", 7 + i)
        wants.append([y.clone() for y in d.step()])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(d.step())
        steps.append(d), graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, wants):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_two_threads_two_streams(ops):
    wants = [[y.clone() for y in Decoder(ops, "f16", i).step()] for i in (3, 4)]
    torch.cuda.synchronize()
    results, errors = {}, []

    def worker(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                d = Decoder(ops, "f16", 3 + i)
                for _ in range(10):
                    out = d.step()
            s.synchronize()
            results[i] = [y.clone() for y in out]
        except Exception as exc:  # reported below
            errors.append(repr(exc))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    for i, want in enumerate(wants):
        assert all(torch.equal(a, b) for a, b in zip(results[i], want))


def test_arena_users_on_two_streams(ops, lib):
    """The plain form's partial results and a split GEMM's share the arena, on two streams."""
    lm = operatorlib.lm_clib()
    t = [dev(x) for x in paged_inputs(42, "f16", [3000, 2500], 8, 2, 128, 16, fill=0.0)]
    want = ops.paged_attention(*t)
    a, b = torch.randn(1, 4096, device="cuda").half(), torch.randn(4096, 1024, device="cuda").half()
    product = ops.gemm(a, b)
    out, c = torch.empty_like(want), torch.empty_like(product)
    args = c_args(t, out, 128, 8, 2, 16)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        assert lm.operatorlib_paged_attention_f16(*args, stream_handle(s1)) == 0
        assert lib.operatorlib_gemm_f16(ptr(a), ptr(b), ptr(c), 1, 1024, 4096, stream_handle(s2)) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(c, product)


# ------------------------------------------------------------------- refusals

def raises(fn, text):
    with pytest.raises(RuntimeError) as err:
        fn()
    assert text in str(err.value), str(err.value)


def test_torch_refusals(ops):
    cuda = dict(device="cuda")
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, **cuda)
    n = lambda *s: torch.zeros(*s, dtype=torch.int32, **cuda)
    q, kc, vc, table, lengths = h(2, 4, 64), h(5, 2, 16, 64), h(5, 2, 16, 64), n(2, 3), n(2)
    paged = lambda a=q, b=kc, c=vc, d=table, e=lengths, **kw: lambda: ops.paged_attention(a, b, c, d, e, **kw)
    raises(paged(a=q.float()), "dtype")
    raises(paged(a=h(2, 3, 64)), "multiple")
    raises(paged(a=h(2, 4, 128)), "head dimension")
    raises(paged(a=h(2, 4, 128)[..., ::2]), "contiguous")
    raises(paged(a=h(2 * 4 * 64 + 1)[1:].view(2, 4, 64)), "16-byte")
    raises(paged(c=h(5, 2, 16, 32)), "same shape")
    raises(paged(b=h(5, 16, 2, 64).transpose(1, 2), c=h(5, 16, 2, 64).transpose(1, 2)), "contiguous")
    raises(paged(d=table.long()), "int32")
    raises(paged(d=n(3, 3)), "page_table")
    raises(paged(e=n(3)), "lengths")
    raises(paged(d=table.cpu()), "must be on")
    raises(paged(window=-1), "window")
    raises(paged(softcap=-1.0), "softcap")
    raises(paged(scale=0.0), "scale")
    raises(paged(slopes=torch.zeros(3, **cuda)), "slopes")
    raises(paged(a=h(2, 4, 136), b=h(5, 2, 16, 136), c=h(5, 2, 16, 136)), "at most 128")
    raises(paged(a=h(0, 4, 64), d=n(0, 3), e=n(0)), "positive int32")
    k = h(1, 2, 30, 64)
    masked = lambda a=h(1, 4, 30, 64), b=k, c=k, **kw: lambda: ops.masked_attention(a, b, c, **kw)
    raises(masked(a=h(1, 4, 31, 64)), "same shape")
    raises(masked(c=h(1, 2, 30, 32)), "same shape")
    raises(masked(b=h(1, 3, 30, 64), c=h(1, 3, 30, 64)), "multiple")
    raises(masked(b=h(1, 2, 64, 30).transpose(2, 3), c=h(1, 2, 64, 30).transpose(2, 3)), "contiguous")
    raises(masked(documents=n(1, 31)), "documents")
    raises(masked(documents=torch.zeros(1, 30, dtype=torch.int64, **cuda)), "documents")
    raises(masked(prefixes=n(2)), "prefixes")
    raises(masked(a=h(1, 4, 30, 60), b=h(1, 2, 30, 60), c=h(1, 2, 30, 60)), "multiple of 8")
    raises(masked(b=h(1, 2, 1, 64).expand(1, 2, 30, 64)), "overlap")
    x = h(3, 2, 64)
    rope = lambda a=h(3, 4, 64), b=x, c=x, p=n(3), f=torch.ones(32, **cuda), s=n(3), kc=kc, vc=vc, **kw: (
        lambda: ops.rope_append(a, b, c, p, f, s, kc, vc, **kw))
    raises(rope(s=n(4)), "slots")
    raises(rope(s=n(3).long()), "slots")
    raises(rope(p=n(2, 4)), "positions")
    raises(rope(f=torch.ones(33, **cuda)), "frequencies")
    raises(rope(f=torch.ones(32, dtype=torch.float64, **cuda)), "frequencies")
    raises(rope(axes=n(31)), "axes")
    raises(rope(vc=kc), "different tensors")
    raises(rope(b=h(3, 3, 64), c=h(3, 3, 64)), "do not agree")
    raises(rope(c=h(3, 2, 32)), "same shape")
    raises(rope(a=h(3, 64, 4).transpose(1, 2)), "contiguous")


def test_most_workgroups(ops):
    """As many tokens and blocks as a launch takes."""
    tokens = 2 ** 24 - 8
    q, k, v = (torch.arange(tokens, device="cuda").remainder(n).half().view(tokens, 1, 1) for n in (1999, 2003, 2011))
    nothing = torch.zeros(0, device="cuda")
    slots = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device="cuda")
    caches = [torch.zeros(tokens // 8, 1, 8, 1, dtype=torch.float16, device="cuda") for _ in range(2)]
    qo, ko = ops.rope_append(q, k, v, slots, nothing, slots, *caches, return_keys=True)
    assert torch.equal(qo, q) and torch.equal(ko, k)
    assert torch.equal(caches[0].flatten(), k.flatten().flip(0)) and torch.equal(caches[1].flatten(), v.flatten().flip(0))
    for dtype in (torch.float16, torch.float32):
        q = torch.ones(8, 2 ** 21 - 1, 1, 8, dtype=dtype, device="cuda")
        v = torch.arange(q.numel(), device="cuda").remainder(2039).to(dtype).view(q.shape)
        assert torch.equal(ops.masked_attention(q, q, v), v)  # of one key
