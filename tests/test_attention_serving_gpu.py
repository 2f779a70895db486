"""norm_rope_axes, cache_write, cache_read, attention_prefill and attention_decode as a serving layer
uses them: one after the other over requests' lives on one cache, captured in graphs, on several
streams, and on buffers past 2^32 bytes.  Values are held against the definitions in 64 bits
(oracle/attention.py), each call from the cache that the calls ahead of it left; replays and concurrent
runs against eager results, bit for bit."""

from __future__ import annotations

import pytest
import torch

from lightdelta_amd import ops
from oracle import attention as oracle
from tests.test_attention_gpu import (
    CACHE,
    EPS,
    SCALE,
    announce,
    attend,
    case_of,
    check_attention,
    check_axes,
    check_read,
    check_write,
)

pytestmark = pytest.mark.gpu

DIM = 128
HQ, HKV, PAGE = 6, 2, 32


def ints(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Layer:
    """One attention layer's parameters and cache, a pool of pages and seeded activations; each
    step's calls, each checked."""

    def __init__(self, device, pages=40, width=12):
        self.gen = torch.Generator(device=device).manual_seed(5)
        self.device, self.width = device, width
        self.cache = dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"),
                              ops.attention_cache(pages, HKV, PAGE, device)))
        self.free = list(range(1, pages))
        self.tables, self.lengths = {}, {}
        self.weights = [1 + 0.1 * torch.randn(DIM, generator=self.gen, device=device)
                        for _ in range(2)]
        self.axes = torch.arange(32, device=device, dtype=torch.int32) % 3
        self.inv_freq = 10000.0 ** (-torch.arange(0, 64, 2, device=device) / 64)

    def release(self, request):
        self.free += self.tables.pop(request)
        del self.lengths[request]

    def step(self, new, width=None, before=None):
        """`new`: tokens of each request, in order; `before`: requests whose last tokens were
        rejected, with the lengths that they have left."""
        self.lengths.update(before or {})
        requests = list(new)
        for r in requests:
            self.lengths[r] = self.lengths.get(r, 0) + new[r]
            table = self.tables.setdefault(r, [])
            while len(table) * PAGE < self.lengths[r]:
                table.append(self.free.pop(len(self.free) // 2))
        counts = [new[r] for r in requests]
        tokens = sum(counts)
        rows = torch.randn(tokens, (2 * HQ + 2 * HKV) * DIM, generator=self.gen,
                           device=self.device).bfloat16()
        position = torch.cat([torch.arange(self.lengths[r] - new[r], self.lengths[r])
                              for r in requests]).to(self.device)
        check_axes(dict(qkv=rows, q_weight=self.weights[0], k_weight=self.weights[1],
                        positions=torch.stack([position, position // 7, position % 7]),
                        axes=self.axes, inv_freq=self.inv_freq, q_heads=HQ, k_heads=HKV), False)
        q, k, v, gate = (x.view(tokens, -1, DIM) for x in
                         rows.split([n * DIM for n in (HQ, HKV, HKV, HQ)], 1))
        table = [self.tables[r] + [0] * (self.width - len(self.tables[r])) for r in requests]
        case = dict(
            pages=ints(self.device, table),
            cu=ints(self.device, [sum(counts[:i]) for i in range(len(counts) + 1)]),
            lengths=ints(self.device, [self.lengths[r] for r in requests]), **self.cache, q=q, k=k,
            v=v, gate=gate,
            out=torch.full((tokens, HQ, DIM), 7.0, dtype=torch.bfloat16, device=self.device))
        check_write(case)
        check_attention(case, width)
        return case


def test_requests_from_prompt_to_release(gpu):
    """Three prompts, single tokens, a verify step of up to four tokens of which some are rejected and
    written over, a prompt that goes on, a release whose pages a new prompt takes, and a request's
    whole context read back."""
    announce(test="attention_lifecycle")
    layer = Layer(gpu)
    layer.step({"a": 70, "b": 130, "c": 5})
    for _ in range(3):
        layer.step({"a": 1, "b": 1, "c": 1}, width=1)
    layer.step({"a": 4, "b": 3, "c": 1}, width=4)
    kept = {r: layer.lengths[r] - n for r, n in (("a", 3), ("b", 1))}
    layer.step({"a": 2, "b": 1, "c": 4}, width=4, before=kept)
    layer.step({"c": 90, "b": 33})
    layer.release("a")
    layer.step({"d": 100, "b": 1})
    case = layer.step({"b": 1, "c": 1, "d": 1}, width=1)
    lengths = case["lengths"].tolist()
    case["cu"] = ints(gpu, [0] + [sum(lengths[:i + 1]) for i in range(3)])
    case["k"] = case["v"] = torch.empty(sum(lengths), HKV, DIM, dtype=torch.bfloat16, device=gpu)
    check_read(case)


def test_what_was_written_is_attended(gpu):
    """Attention over the cache is attention over the rows that went in, but for e4m3: a prompt
    written in parts and read in one."""
    announce(test="attention_of_rows")
    new = [40, 41, 3, 16, 1]
    case = case_of([sum(new)], [sum(new)], 16, (2, 1), seed=3, device=gpu)
    rows, at = {x: case[x].clone() for x in "kv"}, 0
    for n in new:
        part = dict(case, lengths=ints(gpu, [at + n]), cu=ints(gpu, [0, n]),
                    **{x: rows[x][at:at + n] for x in "kv"})
        check_write(part)
        at += n
    check_attention(case)
    q, k, v = (x.double().cpu() for x in (case["q"], rows["k"], rows["v"]))
    s = SCALE * torch.einsum("qhd,kd->hqk", q, k[:, 0])
    s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool).triu(1), -float("inf"))
    want = torch.einsum("hqk,kd->qhd", s.softmax(-1), v[:, 0])
    # e4m3 rounds keys and values by 2^-4 of themselves at the most; on average a third of it
    error = (case["out"].double().cpu() - want).norm() / want.norm()
    assert error < 2.0**-4


def padded(case, requests):
    """The case in a batch of `requests`, padded by requests without rows, tokens and pages."""
    more = requests - case["lengths"].numel()
    device = case["cu"].device
    return dict(case, cu=torch.cat([case["cu"], case["cu"][-1:].expand(more)]),
                lengths=torch.cat([case["lengths"], ints(device, [0] * more)]),
                pages=torch.cat([case["pages"], torch.zeros_like(case["pages"][:1]).expand(more, -1)]))


@pytest.mark.parametrize("requests", [8, 70, 200])
def test_padded_batches(gpu, requests):
    announce(test="attention_padded", requests=requests)
    case = padded(case_of([90, 5, 300], [1, 3, 2], 32, (4, 2), seed=2, device=gpu), requests)
    check_write(case)
    check_read(case)
    check_attention(case, width=4)
    check_attention(case)


def test_nothing_to_do(gpu):
    """No requests, no rows, no pages, tables without columns: rows that a request has get zeros,
    nothing else changes."""
    announce(test="attention_nothing")
    case = case_of([40, 20], [3, 2], 16, (4, 2), seed=1, device=gpu)
    for change in (dict(cu=case["cu"][:1], lengths=case["lengths"][:0], pages=case["pages"][:0]),
                   dict(pages=case["pages"][:, :0]),
                   {x: case[x][:0] for x in CACHE[3:]}, {x: case[x][:1] for x in CACHE[3:]}):
        now = dict(case, **change, out=torch.full_like(case["out"], 7.0))
        check_write(now)
        check_read(now)
        check_attention(now, width=4)
        check_attention(dict(now, out=torch.full_like(case["out"], 7.0)))
    none = dict(case, cu=ints(gpu, [0, 0, 0]), **{x: case[x][:0] for x in ("q", "k", "v", "out")})
    check_write(none)
    check_attention(none)


# ---- graphs and streams --------------------------------------------------------------------


def capture(call):
    """A graph of `call`, warmed up on a stream of its own."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def layer_step(case, rope, width):
    """The layer's calls on fresh activations: rotation in place, the write, attention."""
    rope["qkv"].copy_(rope["source"])
    torch.ops.lightdelta.norm_rope_axes(*[rope[x] for x in (
        "qkv", "q_weight", "k_weight", "positions", "axes", "inv_freq")], HQ, HKV, EPS, False)
    torch.ops.lightdelta.cache_write(case["k"], case["v"], *(case[x] for x in CACHE))
    attend(case, width)


def graph_case(device, lengths, new, seed):
    case = case_of(lengths, new, PAGE, (HQ, HKV), seed=seed, device=device, gated=True)
    tokens = sum(new)
    rows = torch.randn(tokens, (HQ + 2 * HKV) * DIM, device=device).bfloat16()
    q, k, v = (x.view(tokens, -1, DIM) for x in
               rows.split([n * DIM for n in (HQ, HKV, HKV)], 1))
    case.update(q=q, k=k, v=v)
    rope = dict(source=rows.clone(), qkv=rows, q_weight=torch.ones(DIM, device=device),
                k_weight=torch.ones(DIM, device=device),
                positions=torch.randint(0, 1000, (3, tokens), device=device),
                axes=torch.arange(32, dtype=torch.int32, device=device) % 3,
                inv_freq=torch.rand(32, device=device))
    return case, rope


STATE = ("k_cache", "v_cache", "k_scale", "v_scale", "out")


def copied(case, rope):
    """A copy whose activations are views of a buffer of its own."""
    rope = {k: v.clone() for k, v in rope.items()}
    tokens = rope["qkv"].shape[0]
    q, k, v = (x.view(tokens, -1, DIM) for x in
               rope["qkv"].split([n * DIM for n in (HQ, HKV, HKV)], 1))
    return dict({x: y.clone() for x, y in case.items()}, q=q, k=k, v=v), rope


def same(a, b):
    return torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a,
                       b.view(torch.uint8) if b.element_size() == 1 else b)


@pytest.mark.parametrize("width", [None, 3])
def test_graph_replays(gpu, width):
    """Replays with new activations, lengths and tables, eager work between them."""
    announce(test="attention_graph", width=width)
    new = [50, 30, 20] if width is None else [3, 2, 1]
    case, rope = graph_case(gpu, [2000, 90, 300], new, 1)
    graph = capture(lambda: layer_step(case, rope, width))
    most = case["pages"].shape[1] * PAGE
    rows = sum(new)
    for i, lengths in enumerate([[2000, 90, 300], [60, 1500, 33], [most, most, most], [0, 40, 55],
                                 [51, 31, 2100]]):
        rope["source"].normal_()
        rope["positions"].random_(0, 10**6)
        case["lengths"].copy_(ints(gpu, lengths))
        case["pages"].copy_(case["pages"].roll(1, 0))
        # (each page to one request: the rows of a shared one would be undefined)
        if i % 2:
            case["cu"].copy_(ints(gpu, [0, 1, rows - 1, rows] if width is None else [0, 1, 4, 6]))
        case["out"].fill_(7.0)
        eager, eager_rope = copied(case, rope)
        layer_step(eager, eager_rope, width)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in STATE:
            assert same(case[name], eager[name]), (i, name)


def attention_cases(device):
    """A decode and a prompt whose sums go by way of a workspace."""
    return [(case_of([3000, 40, 700], [1, 2, 1], 64, (8, 2), seed=1, device=device), 2),
            (case_of([5000, 300], [40, 30], 16, (8, 2), seed=2, device=device), None),
            (case_of([900, 4000], [1, 1], 16, (8, 2), seed=3, device=device), 1)]


def test_graphs_on_streams(gpu):
    """Each graph's workspace is its own: replays that run at once give what each gives alone."""
    announce(test="attention_graphs")
    cases = attention_cases(gpu)
    graphs = [capture(lambda c=c, w=w: attend(c, w)) for c, w in cases]
    alone = []
    for (c, _), graph in zip(cases, graphs):
        graph.replay()
        torch.cuda.synchronize()
        alone.append(c["out"].clone())
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for c, _ in cases:
            c["out"].zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (c, _), out in zip(cases, alone):
            assert torch.equal(c["out"], out)


def test_eager_calls_on_streams(gpu):
    """Calls at once on several streams, each several times: the same bits every time."""
    announce(test="attention_streams")
    cases = attention_cases(gpu)
    want = []
    for c, w in cases:
        attend(c, w)
        torch.cuda.synchronize()
        want.append(c["out"].clone())
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for stream, (c, w) in zip(streams, cases):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                c["out"].zero_()
                attend(c, w)
        torch.cuda.synchronize()
        for (c, _), out in zip(cases, want):
            assert torch.equal(c["out"], out)


# ---- strides and offsets past 2^32 bytes ----------------------------------------------------


def test_one_pool_of_keys_and_values(gpu):
    """Keys and values of a page together in one allocation, scales as columns of one buffer, tables
    as part of wider ones, rows at odd elements."""
    announce(test="attention_strides")
    case = case_of([90, 200], [33, 4], 32, (4, 2), seed=4, device=gpu, gated=True)
    count, page = case["k_cache"].shape[0], 32
    pool = torch.zeros(count, 4, 2 * page * DIM, dtype=torch.uint8, device=gpu)
    for i, x in enumerate(("k_cache", "v_cache")):
        place = pool[:, i].view(torch.float8_e4m3fn).view(case[x].shape)
        place.view(torch.uint8).copy_(case[x].view(torch.uint8))
        case[x] = place
    scales = torch.zeros(count, 9, dtype=torch.uint8, device=gpu)
    for x, at in (("k_scale", 1), ("v_scale", 6)):
        scales[:, at:at + 2].copy_(case[x].view(torch.uint8))
        case[x] = scales[:, at:at + 2].view(torch.float8_e8m0fnu)
    wide = torch.full((2, case["pages"].shape[1] + 9), -1, dtype=torch.int32, device=gpu)
    wide[:, 3:-6].copy_(case["pages"])
    case["pages"] = wide[:, 3:-6]
    for x in ("q", "k", "v", "gate"):
        n, h = case[x].shape[:2]
        odd = torch.zeros(n, h * DIM + 5, dtype=torch.bfloat16, device=gpu)[:, 3:-2]
        odd.copy_(case[x].reshape(n, -1))
        case[x] = odd.view(n, h, DIM)
    check_write(case)
    check_read(case)
    check_attention(case)
    check_attention(case, width=4)


def test_far_pages(gpu):
    """Pages 512 MiB apart: the last starts 5 GiB into the cache."""
    announce(test="attention_far_pages")
    case = case_of([70, 100], [9, 2], 16, (4, 2), seed=5, device=gpu)
    apart, count = 2**29, 11
    flat = torch.zeros(count * apart, dtype=torch.uint8, device=gpu)
    codes = torch.randint(0, 120, (count, 2 * 16 * DIM), dtype=torch.uint8, device=gpu)
    for x, shape, at in (("k_cache", (8, 16, 16), 0), ("v_cache", (1, DIM, 16), 2**20)):
        place = flat[at:].as_strided((count, 2, *shape),
                                     (apart, 2048, shape[1] * shape[2], shape[2], 1))
        place.copy_(codes.view(count, 2, *shape))
        case[x] = place.view(torch.float8_e4m3fn)
    for x in ("k_scale", "v_scale"):
        case[x] = torch.full((count, 2), 125, dtype=torch.uint8, device=gpu).view(
            torch.float8_e8m0fnu)
    case["pages"] = ints(gpu, [[10, 3, 9, 1, 8, 0, 0, 0], [2, 4, 5, 6, 7, 0, 0, 0]])
    case["lengths"] = ints(gpu, [70, 75])
    check_write(case)
    check_read(case)
    check_attention(case)
    check_attention(dict(case, cu=ints(gpu, [0, 4, 6])), width=4)


def test_far_rows(gpu):
    """Activation rows 256 MiB apart: the last start past 4 GiB."""
    announce(test="attention_far_rows")
    tokens, apart = 21, 2**27
    flat = torch.zeros((tokens - 1) * apart + 8 * DIM, dtype=torch.bfloat16, device=gpu)
    case = case_of([60, 12], [17, 4], 16, (2, 1), seed=6, device=gpu, gated=True)
    for x, at, h in (("q", 0, 2), ("k", 2, 1), ("v", 3, 1), ("gate", 4, 2)):
        place = flat[at * DIM:].as_strided((tokens, h, DIM), (apart, DIM, 1))
        place.copy_(case[x])
        case[x] = place
    check_write(case)
    check_attention(case)
    check_attention(dict(case, cu=ints(gpu, [17, 17, 21])), width=4)
    want = oracle.expected_read(*(case[x] for x in CACHE), case["k"], case["v"])
    torch.ops.lightdelta.cache_read(*(case[x] for x in CACHE), case["k"], case["v"])
    torch.cuda.synchronize()
    for got, expected in zip((case["k"], case["v"]), want):
        assert torch.equal(got.double().cpu(), expected)
