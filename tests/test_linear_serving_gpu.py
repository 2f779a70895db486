"""norm_rope, linear_prefill and linear_decode as a serving layer uses them: one after the other
on one pool, captured in graphs, on several streams, and on buffers past 2^32 bytes.  Values are
held against the definitions in 64 bits (oracle/linear.py), each call from the state that the
calls ahead of it left; replays and concurrent runs against eager results, bit for bit."""

from __future__ import annotations

import pytest
import torch

from lightdelta_amd.workloads import HEAD_DIM as DIM
from oracle.linear import expected_linear_decode, expected_linear_prefill, expected_norm_rope
from tests.test_linear_gpu import (
    DECODE,
    EPS,
    PREFILL,
    SCALE,
    announce,
    check_decode,
    check_prefill,
    check_rope,
    decode_case,
    prefill_case,
    rope_case,
    run_decode,
    run_prefill,
    within,
)

pytestmark = pytest.mark.gpu

H, HV = 2, 4


def ints(device, values):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Layer:
    """One layer's parameters, pool and stream of seeded activations; its calls, each checked."""

    def __init__(self, device, slots=12, rows=400):
        gen = torch.Generator(device=device).manual_seed(31)
        self.device = device
        cols = (2 * H + HV) * DIM
        self.rows = torch.randn(rows, cols + HV * DIM, generator=gen, device=device).bfloat16()
        self.decays = -0.2 * torch.rand(rows, HV, generator=gen, device=device)
        self.weights = [1 + 0.1 * torch.randn(DIM, generator=gen, device=device) for _ in range(3)]
        self.inv_freq = 10000.0 ** (-torch.arange(0, 64, 2, device=device) / 64)
        self.pool = torch.randn(slots, HV, DIM, DIM, generator=gen, device=device)
        self.next = 0

    def tokens(self, positions):
        """Activations for these positions, their q and k normalised and rotated."""
        n = len(positions)
        rows = self.rows[self.next:self.next + n]
        decays = self.decays[self.next:self.next + n]
        self.next += n
        qkv, gate = rows[:, :-HV * DIM], rows[:, -HV * DIM:].view(n, HV, DIM)
        args = (qkv, self.weights[0], self.weights[1], ints(self.device, positions),
                self.inv_freq, H, H, EPS, False)
        want, bound = expected_norm_rope(*args)
        torch.ops.lightdelta.norm_rope(*args)
        torch.cuda.synchronize()
        within(qkv, want, bound, "norm_rope")
        return dict(qkv=qkv, log_decay=decays, gate=gate, weight=self.weights[2], pool=self.pool,
                    out=torch.full((n, HV, DIM), 7.0, dtype=torch.bfloat16, device=self.device))

    def prefill(self, lengths, slots, has_initial, starts):
        case = self.tokens([s + i for s, n in zip(starts, lengths) for i in range(n)])
        case.update(cu=ints(self.device, [sum(lengths[:i]) for i in range(len(lengths) + 1)]),
                    slots=ints(self.device, slots),
                    has_initial=torch.tensor(has_initial, device=self.device))
        check_prefill(case)

    def decode(self, indices, accepted, starts, lengths):
        case = self.tokens([s + i for s, n in zip(starts, lengths) for i in range(n)])
        case.update(cu=ints(self.device, [sum(lengths[:i]) for i in range(len(lengths) + 1)]),
                    indices=ints(self.device, indices), accepted=ints(self.device, accepted))
        check_decode(case)


def test_requests_from_prompt_to_release(gpu):
    """Three prompts, single tokens, a verify step of 4, 3 and 1 draft tokens, the step that reads
    the accepted states, a fork of one request, the release of another's slot to a new prompt in
    two parts."""
    announce(test="linear_lifecycle")
    layer = Layer(gpu)
    at = [70, 130, 5]
    layer.prefill(at, [3, 7, 1], [False] * 3, [0, 0, 0])
    for _ in range(2):
        layer.decode([[3], [7], [1]], [1, 1, 1], at, [1, 1, 1])
        at = [p + 1 for p in at]
    rows = [[3, 4, 5, 6], [7, 8, 9, 10], [1, 2, 11, 0]]
    layer.decode(rows, [1, 1, 1], at, [4, 3, 1])
    accepted = [3, 1, 1]
    at = [p + n for p, n in zip(at, accepted)]
    # the next tokens read column accepted - 1 and write the home slots
    layer.decode(rows, accepted, at, [1, 1, 1])
    torch.ops.lightdelta.copy_state(layer.pool, ints(gpu, [3]), ints(gpu, [4]))
    assert torch.equal(layer.pool[3], layer.pool[4])
    layer.decode([[3], [4]], [1, 1], [at[0] + 1] * 2, [1, 1])
    assert not torch.equal(layer.pool[3], layer.pool[4])
    torch.ops.lightdelta.zero_slots(layer.pool, ints(gpu, [7]))
    layer.prefill([20], [7], [True], [0])    # from a slot of zeros, as from no state
    layer.prefill([33, 0], [7, 1], [True, True], [20, at[2] + 1])


def padded(case, requests):
    """The decode case in a batch of `requests`, padded by requests of slot 0 over no rows."""
    n, width = case["indices"].shape
    more = requests - n
    device = case["pool"].device
    return dict(case, indices=torch.cat([case["indices"], ints(device, [[0] * width] * more)]),
                cu=torch.cat([case["cu"], case["cu"][-1:].expand(more)]),
                accepted=torch.cat([case["accepted"], ints(device, [1] * more)]))


def test_padded_batches(gpu):
    announce(test="linear_padded")
    for width in (1, 3):
        check_decode(padded(decode_case(3, width, H, HV, seed=2, device=gpu), 8))
    case = prefill_case([40, 600], 1, 2, seed=3, device=gpu)
    case["slots"] = torch.cat([case["slots"], ints(gpu, [0, 0, 0])])
    case["cu"] = torch.cat([case["cu"], case["cu"][-1:].expand(3)])
    case["has_initial"] = torch.cat([case["has_initial"], torch.ones(3, dtype=torch.bool, device=gpu)])
    check_prefill(case)


def test_no_tokens(gpu):
    """Sequences of no rows at all: states without an initial one become zeros."""
    announce(test="linear_prefill_no_tokens")
    case = prefill_case([0, 0, 0], H, HV, seed=5, device=gpu)
    check_prefill(case)


def snapshot(case):
    return {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in case.items()}


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


def steps(source, rope, prompt, step):
    """One captured run: fresh activations, norm_rope, a prompt of several segments, a decode."""
    rope["qkv"].copy_(source)
    torch.ops.lightdelta.norm_rope(*rope.values(), EPS, False)
    run_prefill(prompt)
    run_decode(step)


def graph_case(device, seed):
    """A prefill whose activations norm_rope prepares in place, and a decode on the same pool."""
    prompt = prefill_case([700, 90], 1, 2, seed=seed, device=device)
    source = prompt["qkv"].clone()
    rope = rope_case(790, 1, 1, 64, seed=seed, device=device)
    rope["qkv"] = prompt["qkv"] = source.clone()
    step = decode_case(2, 1, 1, 2, seed=seed, device=device)
    step.update(pool=prompt["pool"], indices=prompt["slots"][:, None].contiguous())
    return source, rope, prompt, step


def test_graph_replays(gpu):
    """Replays with new activations, lengths and slots, eager work between them."""
    announce(test="linear_graph")
    source, rope, prompt, step = graph_case(gpu, 1)
    graph = capture(lambda: steps(source, rope, prompt, step))
    for i, (lengths, slots) in enumerate([([700, 90], [1, 2]), ([90, 700], [3, 1]),
                                          ([395, 395], [2, 3]), ([790, 0], [0, 1]),
                                          ([10, 20], [1, 3])]):
        source.normal_()
        prompt["log_decay"].uniform_(-0.1, 0.0)
        prompt["cu"].copy_(ints(gpu, [0, lengths[0], sum(lengths)]))
        prompt["slots"].copy_(ints(gpu, slots))
        step["indices"].copy_(ints(gpu, slots)[:, None])
        for case in (prompt, step):
            case["out"].fill_(7.0)
        # the eager run, on copies
        eager_prompt, eager_step = snapshot(prompt), snapshot(step)
        eager_rope = snapshot(rope)
        eager_rope["qkv"] = eager_prompt["qkv"]
        eager_step["pool"] = eager_prompt["pool"]
        steps(source, eager_rope, eager_prompt, eager_step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("qkv", "out", "pool"):
            assert torch.equal(prompt[name], eager_prompt[name]), (i, name)
        assert torch.equal(step["out"], eager_step["out"]), i


def test_two_graphs_on_two_streams(gpu):
    """Each graph's workspace is its own: replays that run at once give what each gives alone."""
    announce(test="linear_two_graphs")
    cases = [prefill_case([1500, 30], 1, 2, seed=s, device=gpu) for s in (1, 2)]
    starts = [c["pool"].clone() for c in cases]
    graphs = [capture(lambda c=c: run_prefill(c)) for c in cases]
    alone = []
    for c, start, graph in zip(cases, starts, graphs):
        c["pool"].copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        alone.append((c["out"].clone(), c["pool"].clone()))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for c, start in zip(cases, starts):
            c["pool"].copy_(start)
            c["out"].zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c, (out, pool) in zip(cases, alone):
            assert torch.equal(c["out"], out) and torch.equal(c["pool"], pool)


def test_eager_calls_on_two_streams(gpu):
    """Calls at once on two streams, each several times: the same bits every time."""
    announce(test="linear_streams")
    cases = [prefill_case([900, 300], 1, 2, seed=s, device=gpu) for s in (3, 4)]
    starts = [c["pool"].clone() for c in cases]
    want = []
    for c, start in zip(cases, starts):
        run_prefill(c)
        torch.cuda.synchronize()
        want.append((c["out"].clone(), c["pool"].clone()))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for stream, c, start in zip(streams, cases, starts):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                c["pool"].copy_(start)
                c["out"].zero_()
                run_prefill(c)
        torch.cuda.synchronize()
        for c, (out, pool) in zip(cases, want):
            assert torch.equal(c["out"], out) and torch.equal(c["pool"], pool)


# ---- offsets past 2^32 bytes ---------------------------------------------------------------


def test_far_slots(gpu):
    """Slots 1 GiB apart: the last starts 5 GiB into the pool."""
    announce(test="linear_far_slots")
    flat = torch.zeros(5 * 2**28 + 2 * DIM * DIM, device=gpu)
    pool = flat.as_strided((6, 2, DIM, DIM), (2**28, DIM * DIM, DIM, 1))
    case = decode_case(2, 2, 1, 2, seed=1, device=gpu)
    pool.copy_(torch.randn(6, 2, DIM, DIM, device=gpu))
    case.update(pool=pool, indices=ints(gpu, [[5, 1], [4, 2]]), accepted=ints(gpu, [1, 1]))
    check_decode(case)
    prompt = prefill_case([600, 20], 1, 2, seed=2, device=gpu)
    prompt.update(pool=pool, slots=ints(gpu, [4, 5]))
    check_prefill(prompt)


def test_far_rows(gpu):
    """Activation rows 2^23 elements apart (16 MiB): the last tokens' start past 4 GiB."""
    announce(test="linear_far_rows")
    tokens, apart = 290, 2**23
    flat = torch.zeros((tokens - 1) * apart + 6 * DIM, dtype=torch.bfloat16, device=gpu)
    case = prefill_case([20, 270], 1, 2, seed=4, device=gpu)
    far = flat.as_strided((tokens, 4 * DIM), (apart, 1))
    gate = flat[4 * DIM:].as_strided((tokens, 2, DIM), (apart, DIM, 1))
    far.copy_(case["qkv"])
    gate.copy_(case["gate"])
    case.update(qkv=far, gate=gate)
    check_prefill(case)
    step = decode_case(1, 1, 1, 2, seed=5, device=gpu)
    step.update(qkv=far, gate=gate, log_decay=case["log_decay"], cu=ints(gpu, [289, 290]),
                out=case["out"])
    check_decode(step)
    rope = rope_case(tokens, 1, 1, 64, seed=6, device=gpu)
    rope["qkv"] = far
    check_rope(rope, False)


# ---- segments ------------------------------------------------------------------------------


@pytest.mark.parametrize("lengths,heads", [([513], (1, 1)), ([767, 768, 769], (1, 2)),
                                           ([1023, 256, 1025, 257], (1, 1)), ([9000], (2, 8)),
                                           ([2300, 700, 2], (4, 16)),
                                           ([3] * 250 + [300] * 8 + [2] * 20 + [520], (1, 1)),
                                           ([200, 312], (1, 2)), ([512], (1, 2)),
                                           ([8000, 450], (1, 1)), ([4352], (1, 1)),
                                           ([4353], (1, 1))])
def test_prefill_segments(gpu, lengths, heads):
    """Sequences cut into segments of equal whole chunks: a token to either side of a further
    segment, more heads than leave a segment at its least, long sequences among many short ones,
    segments that sum the states ahead of them by themselves and ones that find them joined."""
    announce(test="linear_prefill_segments", lengths=lengths[-3:], heads=heads)
    check_prefill(prefill_case(lengths, *heads, seed=11, device=gpu, decay=0.05))
