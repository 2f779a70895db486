"""The softmax-attention operators without a GPU: the oracle against closed forms, the ops' checks
of arguments (on the meta device), and the C ABI's declarations and refusals."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from lightdelta_amd import _lib, ops
from oracle import attention as oracle

DIM = 128
HEADER = Path(__file__).resolve().parents[1] / "include" / "lightdelta_attention_hip.h"


# ---- the oracle ----------------------------------------------------------------------------


def test_oracle_codes_are_the_types():
    """The 256 values are torch's, and rounding is torch's for every bf16 within the range."""
    codes = torch.arange(256, dtype=torch.uint8)
    torch.testing.assert_close(oracle.e4m3_values(), codes.view(torch.float8_e4m3fn).double(),
                               rtol=0, atol=0, equal_nan=True)
    x = torch.arange(-(2**15), 2**15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x[x.float().abs() <= 448]
    want = x.to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(oracle.round_e4m3(x.double()), want)
    far = torch.tensor([449.0, 1e9, -1e9], dtype=torch.float64)
    assert oracle.round_e4m3(far).tolist() == [0x7E, 0x7E, 0xFE]


def test_oracle_scale_is_the_least():
    for bits in range(1, 0x7F80, 37):
        x = torch.tensor(bits, dtype=torch.int16).view(torch.bfloat16).double().item()
        e = oracle.scale_exponent(x)
        assert e == oracle.HIGH or x <= 448 * 2.0**e
        assert e == oracle.LOW or x > 448 * 2.0 ** (e - 1)


def request(lengths, new, page, kv_heads, seed, device="cpu", extra=2, heads=None):
    """A filled cache, tables and metadata of requests with `lengths` tokens, `new` of them the
    call's."""
    gen = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    count = sum(held) + 1 + extra
    ids = (torch.randperm(count - 1, generator=gen) + 1).tolist()
    table = torch.zeros(len(lengths), max(held, default=0) + 1, dtype=torch.int32)
    for r, n in enumerate(held):
        table[r, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    def codes(*shape):
        return (torch.randn(count, kv_heads, *shape, generator=gen) * 40).clamp(-448, 448).to(
            torch.float8_e4m3fn).to(device)

    scales = (127 - 6 + torch.randint(0, 3, (2, count, kv_heads), generator=gen)).to(torch.uint8)
    k_scale, v_scale = scales.to(device).view(torch.float8_e8m0fnu).unbind(0)
    tokens = int(cu[-1])

    def rows(h):
        return torch.randn(tokens, h, DIM, generator=gen).bfloat16().to(device)

    cache = dict(pages=table.to(device), cu=cu.to(device),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=device),
                 k_cache=codes(8, page, 16), v_cache=codes(page // 16, DIM, 16), k_scale=k_scale,
                 v_scale=v_scale)
    return cache, rows


def test_oracle_attention_is_the_closed_form():
    """Against a dense softmax over what cache_read's oracle gives back."""
    lengths, new = [37, 5], [3, 5]
    cache, rows = request(lengths, new, 16, 2, 0)
    q, out = rows(4), torch.zeros(8, 4, DIM, dtype=torch.bfloat16)
    got, bound = oracle.expected_attention(q, *cache.values(), None, out, 0.1)
    for r, n in enumerate(lengths):
        whole = dict(cache, pages=cache["pages"][r:r + 1], lengths=cache["lengths"][r:r + 1],
                     cu=torch.tensor([0, n]))
        empty = torch.zeros(n, 2, DIM, dtype=torch.bfloat16)
        k, v = oracle.expected_read(*whole.values(), empty, empty)
        at = slice(int(cache["cu"][r]), int(cache["cu"][r + 1]))
        x = q[at].double().transpose(0, 1)
        k, v = (y.repeat_interleave(2, 1).transpose(0, 1) for y in (k, v))
        mask = torch.ones(new[r], n, dtype=torch.bool).tril(n - new[r])
        p = (0.1 * x @ k.transpose(1, 2)).masked_fill(~mask, -float("inf")).softmax(-1)
        torch.testing.assert_close(got[at], (p @ v).transpose(0, 1), rtol=1e-12, atol=1e-12)
    assert (bound < 0.05 * got.abs().amax()).all()


def test_oracle_write_and_read():
    """Rows come back within half a step of their page's scale, pages begun in the call hold the
    least scale that carries them, and nothing else changes."""
    lengths, new = [40, 20, 33], [9, 20, 1]
    cache, rows = request(lengths, new, 16, 2, 1)
    k, v = rows(2), 3 * rows(2)
    kc, vc, ks, vs = oracle.expected_write(k, v, *cache.values())
    changed = dict(cache, k_cache=kc.view(torch.float8_e4m3fn), v_cache=vc.view(torch.float8_e4m3fn),
                   k_scale=ks.view(torch.float8_e8m0fnu), v_scale=vs.view(torch.float8_e8m0fnu))
    back = oracle.expected_read(*changed.values(), torch.zeros_like(k), torch.zeros_like(v))
    for x, y, scale in zip((k, v), back, (ks, vs)):
        largest = 2.0 ** (scale.max().item() - 127)
        step = torch.maximum(x.double().abs() * 2.0**-4, torch.tensor(2.0**-10 * largest))
        assert ((x.double() - y).abs() <= step).all()
    touched = {int(cache["pages"][0, 1]), int(cache["pages"][0, 2]), int(cache["pages"][1, 0]),
               int(cache["pages"][1, 1]), int(cache["pages"][2, 2])}
    for page in range(len(kc)):
        if page not in touched:
            assert torch.equal(kc[page], cache["k_cache"].view(torch.uint8)[page])
            assert torch.equal(vs[page], cache["v_scale"].view(torch.uint8)[page])


# ---- argument checks -----------------------------------------------------------------------


@pytest.fixture
def meta(monkeypatch):
    monkeypatch.setattr(ops, "_is_gpu", lambda t: t.device.type == "meta")
    return torch.device("meta")


def t(device, *shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=device)


def i32(device, *shape):
    return t(device, *shape, dtype=torch.int32)


def e4m3(device, *shape):
    return t(device, *shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def e8m0(device, *shape):
    return t(device, *shape, dtype=torch.uint8).view(torch.float8_e8m0fnu)


def cache_args(device):
    return dict(pages=i32(device, 3, 5), cu=i32(device, 4), lengths=i32(device, 3),
                k_cache=e4m3(device, 7, 2, 8, 32, 16), v_cache=e4m3(device, 7, 2, 2, DIM, 16),
                k_scale=e8m0(device, 7, 2), v_scale=e8m0(device, 7, 2))


def rows_args(device):
    return dict(cache_args(device), k=t(device, 6, 2, DIM), v=t(device, 6, 2, DIM))


def attention_args(device):
    return dict(cache_args(device), q=t(device, 6, 4, DIM), gate=t(device, 6, 4, DIM),
                out=t(device, 6, 4, DIM), scale=0.1)


def decode_args(device):
    return dict(attention_args(device), width=2)


def rope_args(device):
    return dict(qkv=t(device, 5, 7 * DIM), q_weight=t(device, DIM), k_weight=t(device, DIM),
                positions=t(device, 3, 5, dtype=torch.int64), axes=i32(device, 32),
                inv_freq=t(device, 32, dtype=torch.float32), q_heads=4, k_heads=2, eps=1e-6,
                interleaved=False)


CACHE = [
    (dict(k_cache=lambda m: t(m, 7, 2, 8, 32, 16, dtype=torch.uint8)), "caches must be"),
    (dict(v_cache=lambda m: e4m3(m, 7, 2, 2, DIM, 32)[..., :16]), "caches must be"),
    (dict(k_cache=lambda m: e4m3(m, 7, 8200).as_strided((7, 2, 8, 32, 16), (8200, 4096, 512, 16, 1))),
     "caches must be"),
    (dict(k_cache=lambda m: e4m3(m, 7, 2, 8, 48, 16)), "k_cache must be"),
    (dict(k_cache=lambda m: e4m3(m, 7, 2, 8, 256, 16)), "k_cache must be"),
    (dict(k_cache=lambda m: e4m3(m, 7, 2, 4, 32, 16)), "k_cache must be"),
    (dict(v_cache=lambda m: e4m3(m, 7, 2, 4, DIM, 16)), "v_cache must be"),
    (dict(v_cache=lambda m: e4m3(m, 6, 2, 2, DIM, 16)), "v_cache must be"),
    (dict(k_scale=lambda m: t(m, 7, 2, dtype=torch.float32)), "scales must be"),
    (dict(v_scale=lambda m: e8m0(m, 2, 7)), "scales must be"),
    (dict(v_scale=lambda m: e8m0(m, 1, 2).expand(7, 2)), "scales must be"),
    (dict(pages=lambda m: t(m, 3, 5, dtype=torch.int64)), "metadata must be"),
    (dict(pages=lambda m: i32(m, 3, 10)[:, ::2]), "invalid request metadata"),
    (dict(pages=lambda m: i32(m, 4, 5)), "invalid request metadata"),
    (dict(cu=lambda m: i32(m, 3)), "invalid request metadata"),
    (dict(lengths=lambda m: i32(m, 6)[::2]), "invalid request metadata"),
    (dict(lengths=lambda m: torch.zeros(3, dtype=torch.int32)), "metadata must be"),
    (dict(k_cache=lambda m: torch.zeros(7, 2, 8, 32, 16, dtype=torch.uint8)
          .view(torch.float8_e4m3fn)), "caches must be"),
]
ROWS = [
    (dict(k=lambda m: t(m, 6, 2, DIM, dtype=torch.float32)), "k and v must be"),
    (dict(v=lambda m: t(m, 6, 2, 64)), "k and v must be"),
    (dict(v=lambda m: t(m, 5, 2, DIM)), "k and v must be"),
    (dict(k=lambda m: t(m, 6, DIM, 2).transpose(1, 2)), "k and v must be"),
]
READ = [(dict(v=lambda m: t(m, 1, 2, DIM).expand(6, 2, DIM)), "must not overlap")]
ATTENTION = [
    (dict(q=lambda m: t(m, 6, 4, DIM, dtype=torch.float16)), "q must be CUDA BF16"),
    (dict(q=lambda m: t(m, 6, 4, 64)), "q must be CUDA BF16"),
    (dict(q=lambda m: t(m, 6, 8, DIM)[:, ::2]), "q must be CUDA BF16"),
    (dict(q=lambda m: t(m, 6, 3, DIM)), "multiple of kv_heads"),
    (dict(q=lambda m: t(m, 6, 0, DIM)), "multiple of kv_heads"),
    (dict(gate=lambda m: t(m, 6, 2, DIM)), "gate must be"),
    (dict(gate=lambda m: t(m, 6, 4, DIM, dtype=torch.float32)), "gate must be"),
    (dict(out=lambda m: t(m, 6, 8, DIM)[:, :4]), "out must be contiguous"),
    (dict(out=lambda m: t(m, 7, 4, DIM)), "out must be contiguous"),
    (dict(out=lambda m: torch.zeros(6, 4, DIM, dtype=torch.bfloat16)), "out must be contiguous"),
    (dict(scale=lambda m: 0.0), "scale must be positive"),
    (dict(scale=lambda m: -1.0), "scale must be positive"),
    (dict(scale=lambda m: float("nan")), "scale must be positive"),
    (dict(scale=lambda m: 1e39), "scale must be positive"),
]
WIDTH = [(dict(width=lambda m: 0), "1 through 4 tokens"),
         (dict(width=lambda m: 5), "1 through 4 tokens")]
ROPE = [
    (dict(qkv=lambda m: t(m, 5, 5 * DIM)), r"qkv must be \[tokens"),
    (dict(positions=lambda m: t(m, 5, dtype=torch.int64)), "positions must be"),
    (dict(positions=lambda m: t(m, 3, 4, dtype=torch.int64)), "positions must be"),
    (dict(positions=lambda m: t(m, 0, 5, dtype=torch.int64)), "positions must be"),
    (dict(positions=lambda m: t(m, 5, 3, dtype=torch.int32).t()), "positions must be"),
    (dict(positions=lambda m: t(m, 3, 5, dtype=torch.float32)), "positions must be"),
    (dict(axes=lambda m: i32(m, 31)), "axes must be"),
    (dict(axes=lambda m: t(m, 32, dtype=torch.int64)), "axes must be"),
    (dict(axes=lambda m: torch.zeros(32, dtype=torch.int32)), "axes must be"),
    (dict(inv_freq=lambda m: t(m, 65, dtype=torch.float32)), "inv_freq must be"),
    (dict(eps=lambda m: 0.0), "epsilon must be positive"),
]
KINDS = {
    "cache_write": (rows_args, ops.check_cache_write, CACHE + ROWS),
    "cache_read": (rows_args, ops.check_cache_read, CACHE + ROWS + READ),
    "attention_decode": (decode_args, ops.check_attention_decode, CACHE + ATTENTION + WIDTH),
    "attention_prefill": (attention_args, ops.check_attention_prefill, CACHE + ATTENTION),
    "norm_rope_axes": (rope_args, ops.check_norm_rope_axes, ROPE),
}
CASES = [(name, i) for name, (_, _, cases) in KINDS.items() for i in range(len(cases))]


@pytest.mark.parametrize("name", KINDS)
def test_accepts(meta, name):
    make, check, _ = KINDS[name]
    args = make(meta)
    check(**args)
    if name == "norm_rope_axes":
        check(**dict(args, positions=i32(meta, 3, 9)[:, 2:7]))
        check(**dict(args, inv_freq=t(meta, 0, dtype=torch.float32), axes=i32(meta, 0)))
        return
    # one pool for keys and values, wider tables, rows as column slices
    pool = e4m3(meta, 7, 2 * 8192).as_strided((7, 2, 8, 32, 16), (16384, 4096, 512, 16, 1))
    check(**dict(args, k_cache=pool, pages=i32(meta, 3, 9)[:, :4]))
    if name.startswith("cache"):
        check(**dict(args, k=t(meta, 6, 8 * DIM)[:, 2 * DIM:4 * DIM].view(6, 2, DIM)))
    else:
        check(**dict(args, gate=None, q=t(meta, 6, 8 * DIM)[:, :4 * DIM].view(6, 4, DIM)))


@pytest.mark.parametrize("name,i", CASES)
def test_refusals(meta, name, i):
    make, check, cases = KINDS[name]
    change, message = cases[i]
    with pytest.raises(RuntimeError, match=message):
        check(**dict(make(meta), **{k: f(meta) for k, f in change.items()}))


def zeroed(x):
    if not isinstance(x, torch.Tensor) or 0 in x.stride():
        return x
    (x.view(torch.uint8) if x.element_size() == 1 else x).zero_()
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("name,i", CASES)
def test_kernel_refusals(gpu, name, i):
    """The same by the ops' own kernels; zeros as metadata, so that nothing is launched that
    reads or writes a cache."""
    make, _, cases = KINDS[name]
    change, message = cases[i]
    args = {k: zeroed(v) for k, v in make(gpu).items()}
    args.update({k: zeroed(f(gpu)) for k, f in change.items()})
    order = re.findall(r"(\w+)[,)]", ops.SCHEMAS[name])
    with pytest.raises(RuntimeError, match=message):
        getattr(torch.ops.lightdelta, name)(*[args[k] for k in order])


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_cache(page):
    cache = ops.attention_cache(9, 3, page, device="cpu")
    assert [tuple(x.shape) for x in cache] == [(9, 3, 8, page, 16), (9, 3, page // 16, DIM, 16),
                                              (9, 3), (9, 3)]
    assert all(float(x.float().abs().max()) == want for x, want in zip(cache, (0, 0, 1, 1)))
    with pytest.raises(RuntimeError, match="page size"):
        ops.attention_cache(9, 3, 24, device="cpu")


# ---- the C ABI -----------------------------------------------------------------------------


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(ld_\w+)\s*\(", text, flags=re.M))
    assert declared == set(_lib.ATTENTION_SIGNATURES)
    for struct, mirror in (("ld_paged_cache", _lib.PagedCache), ("ld_cache_rows", _lib.CacheRows),
                           ("ld_attention_args", _lib.AttentionArgs),
                           ("ld_rope_axes", _lib.RopeAxes)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\}", text, flags=re.S).group(1)
        assert re.findall(r"(\w+);", body) == [name for name, _ in mirror._fields_]


def refused(message, call, *args):
    assert call(*[None if x is None else ctypes.byref(x) for x in args], None) == 1
    assert message in _lib.load().ld_last_error().decode()


GOOD = dict(k=16, v=16, k_scale=16, v_scale=16, pages=16, cu=16, lengths=16, num_tokens=4,
            table_width=1, num_pages=2, page_size=16, num_kv_heads=2, num_requests=1)


@pytest.mark.parametrize("change,message", [
    (dict(num_requests=-1), ">= 0"), (dict(num_tokens=-1), ">= 0"), (dict(num_pages=-1), ">= 0"),
    (dict(table_width=-1), ">= 0"), (dict(num_kv_heads=0), "num_kv_heads"),
    (dict(num_kv_heads=2**16 + 1), "num_kv_heads"), (dict(page_size=0), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=256), "page_size"),
    (dict(num_tokens=2**31), "too many tokens"), (dict(k=None), "NULL tensor pointer"),
    (dict(cu=None), "NULL tensor pointer"), (dict(pages=None), "NULL tensor pointer"),
    (dict(v=8), "16-byte aligned"), (dict(k_page_stride=8), "16-byte aligned"),
])
def test_c_abi_refuses_a_cache(change, message):
    lib = _lib.load()
    cache = _lib.PagedCache(**dict(GOOD, **change))
    rows = _lib.CacheRows(k=16, v=16, k_row_stride=256, v_row_stride=256)
    args = _lib.AttentionArgs(q=16, out=16, num_q_heads=4, width=1, scale=0.1)
    for call, what in ((lib.ld_cache_write, rows), (lib.ld_cache_read, rows),
                       (lib.ld_attention_decode, args), (lib.ld_attention_prefill, args)):
        refused(message, call, cache, what)


def test_c_abi_refuses_without_launching():
    lib = _lib.load()
    good = _lib.PagedCache(**GOOD)
    for call in (lib.ld_cache_write, lib.ld_cache_read):
        refused("cache is NULL", call, None, None)
        refused("rows is NULL", call, good, None)
        refused("NULL tensor pointer", call, good, _lib.CacheRows(k=16))
    refused("must not overlap", lib.ld_cache_read, good,
            _lib.CacheRows(k=16, v=16, k_row_stride=256, v_row_stride=255))
    for call in (lib.ld_attention_decode, lib.ld_attention_prefill):
        refused("cache is NULL", call, None, None)
        refused("args is NULL", call, good, None)
        args = dict(q=16, out=16, num_q_heads=4, width=1, scale=0.1)
        for change, message in [(dict(num_q_heads=3), "multiple of num_kv_heads"),
                                (dict(num_q_heads=0), "multiple of num_kv_heads"),
                                (dict(num_q_heads=2**17), "at most 2^16"),
                                (dict(scale=0.0), "positive"), (dict(scale=-1.0), "positive"),
                                (dict(scale=float("nan")), "positive"),
                                (dict(scale=float("inf")), "positive"),
                                (dict(q=None), "NULL tensor pointer")]:
            refused(message, call, good, _lib.AttentionArgs(**dict(args, **change)))
    for width in (0, 5):
        refused("1 through 4 tokens", lib.ld_attention_decode, good,
                _lib.AttentionArgs(q=16, out=16, num_q_heads=4, width=width, scale=0.1))
    rope = _lib.NormRopeArgs(num_tokens=1, q_heads=1, k_heads=1, eps=1e-6, rotary=32)
    refused("axes is NULL", lib.ld_norm_rope_axes, rope, None)
    refused("num_axes", lib.ld_norm_rope_axes, rope, _lib.RopeAxes(num_axes=0))
    refused("NULL tensor pointer", lib.ld_norm_rope_axes, rope, _lib.RopeAxes(num_axes=3))
    refused("args is NULL", lib.ld_norm_rope_axes, None, _lib.RopeAxes(num_axes=3, axes=16))


def test_c_abi_empty_work_is_a_no_op():
    lib = _lib.load()
    rows, args = _lib.CacheRows(), _lib.AttentionArgs(num_q_heads=4, width=1, scale=0.1)
    for empty in (dict(num_requests=0), dict(num_tokens=0)):
        cache = _lib.PagedCache(**dict(GOOD, k=None, pages=None, **empty))
        for call, what in ((lib.ld_cache_write, rows), (lib.ld_cache_read, rows),
                           (lib.ld_attention_decode, args), (lib.ld_attention_prefill, args)):
            assert call(ctypes.byref(cache), ctypes.byref(what), None) == 0
        for call in (lib.ld_attention_decode_workspace_bytes,
                     lib.ld_attention_prefill_workspace_bytes):
            assert call(ctypes.byref(cache), ctypes.byref(args)) == 0
    none = _lib.PagedCache(**dict(GOOD, table_width=0, pages=None))
    assert lib.ld_cache_write(ctypes.byref(none), ctypes.byref(_lib.CacheRows(k=16, v=16)), None) == 0
