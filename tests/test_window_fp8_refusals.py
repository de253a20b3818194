"""Refusals of the windowed attention and 8-bit cache entry points, on the CPU:
every bad argument is reported before any launch."""
import ctypes

import pytest
import torch

from grout_b200 import attn, build

P = 0x10000  # aligned, never dereferenced
ODD = 0x10008


@pytest.fixture(scope="module")
def L():
    build.build()
    return attn.lib()


def _dims(hq=64, hkv=8, hd=128, ms=4096):
    return attn.AttnDims(hq, hkv, hd, ms, 1e-6, 0.0, 0)


def _refused(L, status, message, st):
    assert st == status, (st, L.grout_attn_last_error())
    assert message in L.grout_attn_last_error().decode(), L.grout_attn_last_error()


def _pages(k=P, v=P, ks=P, vs=P, n=64, ps=64):
    return attn.Fp8Pages(k, v, ks, vs, n, ps)


DECODE_BAD = [
    ({"q": None}, 1, "null"), ({"q": ODD}, 1, "aligned"), ({"out": None}, 1, "null"), ({"out": ODD}, 1, "aligned"),
    ({"pos": None}, 1, "null"), ({"batch": -1}, 1, "batch"), ({"batch": 70000}, 2, "65535"),
    ({"max_kv_len": 0}, 1, "max_kv_len"), ({"max_kv_len": 4097}, 1, "max_kv_len"), ({"window": -1}, 1, "window"),
    ({"sinks": -1}, 1, "sinks"), ({"splits": -1}, 1, "num_splits"), ({"splits": 1025}, 1, "num_splits"),
    ({"splits": 40}, 1, "workspace"), ({"splits": 40, "ws": P, "ws_bytes": 100}, 1, "workspace"),
    ({"splits": 40, "ws": ODD, "ws_bytes": 1 << 40}, 1, "workspace"),
    ({"dims": _dims(hd=64)}, 2, "head_dim"), ({"dims": _dims(hq=64, hkv=4)}, 2, "group"), ({"dims": _dims(hq=63)}, 1, "multiple"),
    ({"dims": _dims(ms=0)}, 1, "max_seq"), ({"dims": None}, 1, "dims"),
]


def _decode(L, kind, **bad):
    a = dict(q=P, out=P, pos=P, batch=2, max_kv_len=100, window=10, sinks=2, splits=1, ws=None, ws_bytes=0, dims=_dims(), cache=P, bs=8 * 4096 * 128,
             hs=4096 * 128, table=P, stride=64, n=64, ps=64, pages=_pages())
    a.update(bad)
    tail = (a["pos"], a["out"], a["batch"], a["max_kv_len"], a["window"], a["sinks"], a["splits"], a["dims"], a["ws"], a["ws_bytes"], None)
    if kind == "contiguous":
        return L.grout_attn_decode_window(a["q"], a["cache"], a["cache"], a["bs"], a["hs"], *tail)
    if kind == "paged":
        return L.grout_attn_decode_paged_window(a["q"], a["cache"], a["cache"], a["n"], a["ps"], a["table"], a["stride"], *tail)
    return L.grout_attn_decode_paged_fp8(a["q"], a["pages"], a["table"], a["stride"], *tail)


@pytest.mark.parametrize("kind", ["contiguous", "paged", "fp8"])
@pytest.mark.parametrize("bad,status,message", DECODE_BAD)
def test_decode_refusals(L, kind, bad, status, message):
    _refused(L, status, message, _decode(L, kind, **bad))


def test_decode_cache_refusals(L):
    for kind in ("contiguous", "paged"):
        _refused(L, 1, "window", _decode(L, kind, window=0))
        _refused(L, 1, "null", _decode(L, kind, cache=None))
        _refused(L, 1, "aligned", _decode(L, kind, cache=ODD))
    _refused(L, 1, "cache_head_stride", _decode(L, "contiguous", hs=4095 * 128))
    _refused(L, 1, "cache_batch_stride", _decode(L, "contiguous", bs=4096 * 128))
    _refused(L, 1, "window", _decode(L, "fp8", window=0, sinks=3))
    _refused(L, 1, "pages is null", _decode(L, "fp8", pages=None))
    for bad, message in (({"k": None}, "null"), ({"v": ODD}, "aligned"), ({"ks": None}, "null"), ({"vs": ODD}, "aligned"), ({"n": 0}, "num_pages"),
                         ({"ps": 96}, "page_size"), ({"ps": 32}, "page_size"), ({"ps": 8192}, "page_size")):
        _refused(L, 1, message, _decode(L, "fp8", pages=_pages(**bad)))
    for kind in ("paged", "fp8"):
        _refused(L, 1, "table_stride", _decode(L, kind, stride=63))
        _refused(L, 1, "null", _decode(L, kind, table=None))
    for kind in ("contiguous", "paged", "fp8"):
        assert _decode(L, kind, batch=0, q=None, cache=None, table=None, pages=None) == 0


def test_write_refusals(L):
    def decode(**bad):
        a = dict(qkv=P, w=P, rope=P, out=P, pages=_pages(), table=P, stride=64, pos=P, batch=2, dims=_dims())
        a.update(bad)
        return L.grout_qk_norm_rope_kv_decode_paged_fp8(a["qkv"], a["w"], a["w"], a["rope"], a["out"], a["pages"], a["table"], a["stride"], a["pos"], a["batch"], a["dims"], None)

    def prefill(**bad):
        a = dict(q=P, k=P, w=P, rope=P, out=P, pages=_pages(), table=P, qs=64 * 128, kvs=8 * 128, start=0, S=16, dims=_dims())
        a.update(bad)
        return L.grout_qk_norm_rope_kv_prefill_paged_fp8(a["q"], a["k"], a["k"], a["qs"], a["kvs"], a["w"], a["w"], a["rope"], a["out"], a["pages"], a["table"], a["start"], a["S"], a["dims"], None)

    for call in (decode, prefill):
        for name in ("w", "rope", "out"):
            _refused(L, 1, "null", call(**{name: None}))
            _refused(L, 1, "aligned", call(**{name: ODD}))
        _refused(L, 1, "null", call(table=None))
        _refused(L, 1, "pages is null", call(pages=None))
        _refused(L, 1, "page_size", call(pages=_pages(ps=65)))
        _refused(L, 1, "null", call(pages=_pages(ks=None)))
        _refused(L, 2, "head_dim", call(dims=_dims(hd=64)))
    _refused(L, 1, "null", decode(pos=None))
    _refused(L, 1, "batch", decode(batch=-1))
    _refused(L, 1, "table_stride", decode(stride=63))
    assert decode(batch=0, qkv=None) == 0
    _refused(L, 1, "exceeds max_seq", prefill(start=4090))
    _refused(L, 1, "exceeds max_seq", prefill(start=2 ** 31 - 1))
    _refused(L, 1, "position_start", prefill(start=-1))
    _refused(L, 1, "q_row_stride", prefill(qs=63 * 128))
    _refused(L, 1, "kv_row_stride", prefill(kvs=8 * 128 + 4))
    assert prefill(S=0, q=None) == 0


def test_read_refusals(L):
    def read(**bad):
        a = dict(pages=_pages(), table=P, stride=64, cu=P, start=None, batch=2, rows=100, k=P, v=P, rs=8 * 128, dims=_dims())
        a.update(bad)
        return L.grout_kv_read_paged_fp8(a["pages"], a["table"], a["stride"], a["cu"], a["start"], a["batch"], a["rows"], a["k"], a["v"], a["rs"], a["dims"], None)

    for bad, status, message in (({"cu": None}, 1, "null"), ({"k": None}, 1, "null"), ({"v": ODD}, 1, "aligned"), ({"rs": 8 * 128 - 8}, 1, "out_row_stride"),
                                 ({"rs": 8 * 128 + 4}, 1, "out_row_stride"), ({"batch": -1}, 1, "batch"), ({"rows": -1}, 1, "rows"),
                                 ({"rows": 2 ** 40}, 1, "rows"), ({"pages": None}, 1, "pages"), ({"stride": 10}, 1, "table_stride"),
                                 ({"dims": _dims(hd=96)}, 2, "head_dim")):
        _refused(L, status, message, read(**bad))
    assert read(batch=0, cu=None) == 0 and read(rows=0, k=None) == 0


def test_prefill_refusals(L):
    def varlen(window=10, sinks=2, dims=None, splits=1, ws=None, ws_bytes=0, **bad):
        a = attn.PrefillVarlenArgs(P, P, 64 * 128, 100, P, P, 0, 128, 4096 * 128, 4096, P, None, None, 2, 100)
        for k, v in bad.items():
            setattr(a, k, v)
        return L.grout_attn_prefill_varlen_window(a, window, sinks, splits, dims or _dims(), ws, ws_bytes, None)

    def paged(window=10, sinks=2, dims=None, splits=1, ws=None, ws_bytes=0, **bad):
        a = attn.PrefillPagedArgs(P, P, 64 * 128, 100, P, P, 64, 64, P, 64, P, None, 2, 100)
        for k, v in bad.items():
            setattr(a, k, v)
        return L.grout_attn_prefill_paged_window(a, window, sinks, splits, dims or _dims(), ws, ws_bytes, None)

    for call in (varlen, paged):
        _refused(L, 1, "window", call(window=0))
        _refused(L, 1, "window", call(window=-5))
        _refused(L, 1, "sinks", call(sinks=-1))
        _refused(L, 1, "cu_seqlens_q", call(cu_seqlens_q=None))
        _refused(L, 1, "q_rows", call(cu_seqlens_q=None, batch=1, q_rows=99))
        _refused(L, 1, "null", call(q=None))
        _refused(L, 1, "aligned", call(out=ODD))
        _refused(L, 1, "q_row_stride", call(q_row_stride=63 * 128))
        _refused(L, 1, "batch", call(batch=-1))
        _refused(L, 2, "head_dim", call(dims=_dims(hd=64)))
        _refused(L, 1, "num_splits", call(splits=-1))
        _refused(L, 1, "num_splits", call(splits=33))
        _refused(L, 1, "num_splits", call(splits=2, batch=65536, ws=P, ws_bytes=1 << 40))
        _refused(L, 1, "workspace", call(splits=2))
        _refused(L, 1, "workspace", call(splits=3, ws=P, ws_bytes=100 * 64 * 3 * 129 * 4 - 1))
        _refused(L, 1, "workspace", call(splits=0, ws=ODD, ws_bytes=1 << 40))
        assert call(batch=0) == 0 and call(max_q_len=0) == 0
    _refused(L, 1, "null", varlen(k=None))
    _refused(L, 1, "kv strides", varlen(kv_row_stride=0))
    _refused(L, 1, "kv strides", varlen(kv_head_stride=12))
    _refused(L, 1, "page_size", paged(page_size=100))
    _refused(L, 1, "table_stride", paged(table_stride=63))
    assert L.grout_attn_prefill_varlen_window(None, 1, 0, 1, _dims(), None, 0, None) == 1
    assert L.grout_attn_prefill_paged_window(None, 1, 0, 1, _dims(), None, 0, None) == 1


def test_prefill_split_counts(L):
    """One where there are items enough or the window is short, at most 32, and
    no more than an item for each SM."""
    count = L.grout_attn_prefill_window_splits
    d = _dims()
    assert count(1, 5, 1 << 20, 300, 4, d) == 1
    assert count(1, 8192, 1 << 20, 1 << 20, 0, d) == 1
    assert count(32, 5, 1 << 20, 1 << 20, 0, d) == 1
    assert count(1, 5, 64, 1 << 20, 0, d) == 1
    for bad in ((0, 5, 100, 10, 0), (1, 0, 100, 10, 0), (1, 5, 0, 10, 0), (1, 5, 100, 0, 0), (1, 5, 100, 10, -1), (65536, 1, 1 << 20, 1 << 20, 0)):
        assert count(*bad, d) == 1
    for B in (1, 2, 7):
        for S in (1, 16, 17, 100, 2 ** 31 - 1):
            for n in (1, 2000, 40000, 2 ** 31 - 1, 2 ** 62):
                for w, sinks in ((1, 0), (2000, 4), (2 ** 31 - 1, 2 ** 31 - 1)):
                    k = count(B, S, n, w, sinks, d)
                    assert 1 <= k <= 32
                    if k > 1:
                        assert k * B * 8 * -(-S // 32) <= 148 and n >= 10 * 64
    ws = L.grout_attn_prefill_window_workspace_bytes
    assert ws(5, 1, d) == 0 and ws(5, 4, d) == 5 * 64 * 4 * 129 * 4


def test_window_split_counts(L):
    """A window bounds what a split count is chosen for, whatever the context;
    a cluster's splits need no workspace."""
    d = _dims(ms=1 << 20)
    count = L.grout_attn_decode_window_splits
    for fp8 in (0, 1):
        a = [count(1, n, 1024, 4, fp8, d) for n in (2048, 32768, 1 << 20)]
        assert a[0] == a[1] == a[2] >= 1
        assert count(1, 2 ** 20, 2 ** 31 - 1, 2 ** 31 - 1, fp8, d) >= 1
        for hq, hkv in ((64, 8), (8, 1), (8, 8)):
            d2 = _dims(hq=hq, hkv=hkv, ms=1 << 20)
            for B in (1, 2, 3, 5, 8, 17, 40, 300):
                for n in (1, 64, 1000, 5000, 40000, 1 << 20):
                    s = count(B, n, 0, 0, fp8, d2)
                    assert 1 <= s <= max(1, -(-n // 64)) and s <= 64
                    need = L.grout_attn_decode_window_workspace_bytes(B, n, 0, 0, 0, fp8, d2)
                    assert need == (0 if s <= 16 else B * hq * s * 129 * 4)
    assert count(64, 32768, 4096, 4, 0, d) == 1
    assert L.grout_attn_decode_window_workspace_bytes(2, 4096, 1024, 4, 16, 0, d) == 0
    assert L.grout_attn_decode_window_workspace_bytes(2, 4096, 1024, 4, 17, 0, d) == 2 * 64 * 17 * 129 * 4


def test_python_refuses_what_is_not_on_the_gpu():
    """Tensors are checked before anything else is read."""
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    f8 = torch.zeros(2, 1, 64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc, tab, pos = torch.zeros(2, 1, 64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = h(1, 8, 128)
    calls = [
        lambda: attn.attention_decode_window(q, h(1, 1, 64, 128), h(1, 1, 64, 128), pos, q, 64, 10),
        lambda: attn.attention_decode_paged_window(q, h(2, 1, 64, 128), h(2, 1, 64, 128), tab, pos, q, 64, 10),
        lambda: attn.attention_decode_paged_fp8(q, f8, f8, sc, sc, tab, pos, q, 64),
        lambda: attn.kv_read_paged_fp8(f8, f8, sc, sc, tab, h(4, 1, 128), h(4, 1, 128), pos),
        lambda: attn.attention_prefill_varlen_window(q, h(1, 1, 64, 128), h(1, 1, 64, 128), q, None, 1, 1, 128, 64 * 128, 10),
        lambda: attn.attention_prefill_paged_window(q, h(2, 1, 64, 128), h(2, 1, 64, 128), tab, q, 10),
        lambda: attn.qk_norm_rope_kv_decode_paged_fp8(h(1, 10 * 128), h(128), h(128), sc, q, f8, f8, sc, sc, tab, pos, 8, 1, 1e-6),
        lambda: attn.qk_norm_rope_kv_prefill_paged_fp8(q, h(1, 1, 128), h(1, 1, 128), h(128), h(128), sc, q, f8, f8, sc, sc, tab[0], 0, 1e-6),
    ]
    for call in calls:
        with pytest.raises(attn.GroutError, match="CUDA tensor"):
            call()


def test_counts_past_32_bits(L):
    """As large (or as bad) as the largest that fits, not wrapped."""
    dims = (64, 8, 4096)
    assert attn.decode_window_splits(1, 4096, 2 ** 40 + 1, 0, *dims) == attn.decode_window_splits(1, 4096, 4096, 0, *dims)
    assert attn._span(-(2 ** 40)) < 0 and attn._span(17) == 17 and attn._span(2 ** 32) == 2 ** 31 - 1


def test_binding_takes_its_arguments_only():
    """Too few, too many or no arguments, and values that are no tensors."""
    b = attn._load_bind()
    names = ("write_decode", "write_prefill", "kv_read", "decode_window", "decode_paged_window", "decode_paged_fp8",
             "prefill_varlen", "prefill_paged")
    for name in names:
        for n in (0, 1, 40):
            with pytest.raises(TypeError, match="arguments"):
                getattr(b, name)(*[None] * n)
    for name, n in zip(names, (15, 15, 10, 12, 14, 16, 18, 14)):
        with pytest.raises(attn.GroutError, match="CUDA tensor"):
            getattr(b, name)(*[None] * n)
    for bad in ((), (attn.GroutError,), (attn.GroutError, (1, 2)), (attn.GroutError, (0,) * 12)):
        with pytest.raises((TypeError, ValueError)):
            b.use(*bad)
    attn._load_bind()
