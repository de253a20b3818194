"""GPU checks of the binding of the window attention and 8-bit cache calls: every
tensor that does not fit is refused before anything is launched, numbers count
by their value at the call, and calls from several threads at once are right."""
import threading

import pytest
import torch

from window_ref import D, SCALE_F16, attention64, check, fp8_cache, normal

pytestmark = pytest.mark.gpu

HQ, HKV, PS, B = 8, 2, 64, 2


def _f16(*shape):
    return torch.zeros(*shape, dtype=torch.float16, device="cuda")


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _args():
    """A fitting set of arguments of each call."""
    codes = lambda: torch.zeros(6, HKV, PS, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    pools = dict(k_pages=codes(), v_pages=codes(), k_scales=torch.zeros(6, HKV, PS, device="cuda"), v_scales=torch.zeros(6, HKV, PS, device="cuda"))
    pages = dict(k_pages=_f16(6, HKV, PS, D), v_pages=_f16(6, HKV, PS, D))
    table = _i32(*range(6)).view(B, 3)
    rope = torch.zeros(3 * PS, D, device="cuda")
    norms = dict(q_norm_w=_f16(D), k_norm_w=_f16(D), rope_table=rope)
    one = dict(q=_f16(B, HQ, D), position=_i32(5, 100), out=_f16(B, HQ, D), max_kv_len=3 * PS, window=10)
    rows = dict(q=_f16(9, HQ, D), out=_f16(9, HQ, D), window=10, cu_seqlens_q=_i32(0, 4, 9), max_q_len=5)
    return {
        "qk_norm_rope_kv_decode_paged_fp8": dict(qkv=_f16(B, (HQ + 2 * HKV) * D), q_out=_f16(B, HQ, D), page_table=table, position=_i32(5, 100),
                                                 num_q_heads=HQ, num_kv_heads=HKV, eps=1e-6, **norms, **pools),
        "qk_norm_rope_kv_prefill_paged_fp8": dict(q=_f16(9, HQ, D), k=_f16(9, HKV, D), v=_f16(9, HKV, D), q_out=_f16(9, HQ, D), page_table_row=table[0],
                                                  position_start=3, eps=1e-6, **norms, **pools),
        "kv_read_paged_fp8": dict(page_table=table, k_out=_f16(9, HKV, D), v_out=_f16(9, HKV, D), cu_seqlens=_i32(0, 4, 9), position_start=_i32(0, 1), **pools),
        "attention_decode_window": dict(k_cache=_f16(B, HKV, 3 * PS, D), v_cache=_f16(B, HKV, 3 * PS, D), **one),
        "attention_decode_paged_window": dict(page_table=table, **pages, **one),
        "attention_decode_paged_fp8": dict(page_table=table, **pools, **one),
        "attention_prefill_varlen_window": dict(k=_f16(20, HKV, D), v=_f16(20, HKV, D), num_kv_heads=HKV, kv_row_stride=HKV * D, kv_head_stride=D,
                                                kv_start=_i32(0, 5), position_start=_i32(0, 1), **rows),
        "attention_prefill_paged_window": dict(page_table=table, position_start=_i32(0, 1), **pages, **rows),
    }


NAMES = ["qk_norm_rope_kv_decode_paged_fp8", "qk_norm_rope_kv_prefill_paged_fp8", "kv_read_paged_fp8", "attention_decode_window",
         "attention_decode_paged_window", "attention_decode_paged_fp8", "attention_prefill_varlen_window", "attention_prefill_paged_window"]


@pytest.mark.parametrize("name", NAMES)
def test_refuses_tensors_that_do_not_fit(grout, name):
    fn, good = getattr(grout, name), _args()[name]
    fn(**good)
    torch.cuda.synchronize()
    grout.check_device_error()
    for key, t in good.items():
        if not isinstance(t, torch.Tensor):
            continue
        other = torch.int32 if t.dtype is not torch.int32 else torch.float32
        bad = [t.cpu(), t.to(other) if t.dtype is not torch.float8_e4m3fn else t.view(torch.uint8), "no tensor", 3]
        if t.numel() > 2:  # every second element: not contiguous
            bad.append(torch.empty(t.numel() * 2, device="cuda").to(t.dtype)[::2].view(*t.shape[:-1], -1) if t.dim() == 1 else t.transpose(0, -1))
        if key not in ("q", "k", "v", "rope_table", "page_table_row", "cu_seqlens", "cu_seqlens_q"):  # (a shorter one of these is another call)
            bad.append(t[:-1])
        if t.dim() > 1 and key != "page_table" and not (key in "kv" and "kv_start" in good):
            bad.append(t[..., : t.shape[-1] // 2].contiguous())
        for x in bad:
            with pytest.raises(grout.GroutError):
                fn(**{**good, key: x})
    for key in ("max_kv_len", "num_q_heads", "num_kv_heads", "max_q_len", "position_start"):
        if isinstance(good.get(key), int):
            for x in (-1, 2 ** 31, 2 ** 70, -(2 ** 70)):
                with pytest.raises(grout.GroutError):
                    fn(**{**good, key: x})
            for x in (None, 1.5, "3"):
                with pytest.raises((TypeError, grout.GroutError)):
                    fn(**{**good, key: x})
    if "window" in good:
        for extra in ({"window": -1}, {"window": -(2 ** 70)}, {"sinks": -1}, {"sinks": -(2 ** 33)}):
            with pytest.raises(grout.GroutError):
                fn(**{**good, **extra})
        fn(**{**good, "window": 2 ** 70, "sinks": 2 ** 70})
    fn(**good)
    torch.cuda.synchronize()
    grout.check_device_error()


def test_refuses_rows_that_k_and_v_do_not_hold(grout):
    good = _args()["attention_prefill_varlen_window"]
    for extra in ({"kv_rows": 21}, {"kv_rows": 0}, {"kv_rows": -1}, {"kv_batch_stride": 10 * HKV * D, "kv_rows": 11}, {"kv_head_stride": 20 * HKV * D},
                  {"kv_row_stride": 2 ** 62}, {"kv_batch_stride": 2 ** 62}, {"kv_head_stride": 2 ** 62}, {"num_kv_heads": 3}):
        if extra.get("kv_row_stride") == 2 ** 62:  # one row is all that fits, and the sequences need more
            grout.attention_prefill_varlen_window(**{**good, "kv_row_stride": 20 * HKV * D})
            with pytest.raises(grout.GroutError, match="0x200"):
                grout.check_device_error()
        with pytest.raises(grout.GroutError):
            grout.attention_prefill_varlen_window(**{**good, **extra})


def test_numbers_count_by_their_value(grout):
    q, k, v = normal(1, 1, HQ, D).half(), normal(2, 1, HKV, 100, D).half(), normal(3, 1, HKV, 100, D).half()
    out, pos = torch.empty_like(q), _i32(99)
    scale = torch.tensor(0.25)
    for _ in range(2):
        grout.attention_decode_window(q, k, v, pos, out, 100, 40, qk_scale=scale, scale_f16=False)
        check(out, *attention64(q, k[0].transpose(0, 1), v[0].transpose(0, 1), pos.long(), 40, 0, float(scale)))
        scale.mul_(0.25)


def test_calls_from_several_threads(grout):
    """Eight threads, a stream each, decode calls that take their own workspace."""
    n = 4096
    (kc, ks), (vc, vs) = (fp8_cache(s, n // PS, 1, PS, D) for s in (10, 20))
    table = torch.arange(n // PS, dtype=torch.int32, device="cuda").view(1, -1)
    pos = _i32(n - 1)
    q = normal(30, 8, 1, HQ, D).half()
    want = [grout.attention_decode_paged_fp8(q[i], kc, vc, ks, vs, table, pos, torch.empty_like(q[i]), n, num_splits=20) for i in range(8)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    out = torch.empty_like(q[i])
                    grout.attention_decode_paged_fp8(q[i], kc, vc, ks, vs, table, pos, out, n, num_splits=20)
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(out, want[i])
                    with pytest.raises(grout.GroutError, match="max_kv_len"):
                        grout.attention_decode_paged_fp8(q[i], kc, vc, ks, vs, table, pos, out, 0)
        except BaseException as e:  # noqa: BLE001 (reported by the test below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    grout.check_device_error()


def test_empty_calls_and_unsigned_positions(grout):
    """No sequences, no rows: nothing is launched, nothing is refused; positions
    may be uint32."""
    a = _args()
    none = dict(q=_f16(0, HQ, D), out=_f16(0, HQ, D), position=_i32())
    for name in NAMES[3:6]:
        good = dict(a[name])
        getattr(grout, name)(**{**good, **none})
        getattr(grout, name)(**{**good, "position": good["position"].view(torch.uint32)})
    grout.qk_norm_rope_kv_decode_paged_fp8(**{**a[NAMES[0]], "qkv": _f16(0, (HQ + 2 * HKV) * D), "q_out": _f16(0, HQ, D), "position": _i32()})
    rows = lambda h: _f16(0, h, D)  # noqa: E731
    grout.qk_norm_rope_kv_prefill_paged_fp8(**{**a[NAMES[1]], "q": rows(HQ), "k": rows(HKV), "v": rows(HKV), "q_out": rows(HQ)})
    grout.kv_read_paged_fp8(**{**a[NAMES[2]], "k_out": rows(HKV), "v_out": rows(HKV), "cu_seqlens": _i32(0), "position_start": None})
    for name in NAMES[6:]:
        good = {k: v for k, v in a[name].items() if k not in ("position_start", "kv_start")}
        getattr(grout, name)(**{**good, "q": rows(HQ), "out": rows(HQ), "cu_seqlens_q": None, "max_q_len": None})
        getattr(grout, name)(**{**good, "cu_seqlens_q": _i32(0), "max_q_len": 0})
        getattr(grout, name)(**{**good, "cu_seqlens_q": _i32(0, 0, 0), "max_q_len": 7})
    torch.cuda.synchronize()
    grout.check_device_error()


def test_captured_calls_take_their_workspace_from_the_graph(grout):
    """Two graphs and eager calls, each with a workspace of its own, in turn."""
    n = 6000
    q, k, v = normal(40, 1, HQ, D).half(), normal(41, 1, 1, n, D).half(), normal(42, 1, 1, n, D).half()
    pos = _i32(0)
    outs, graphs = [torch.empty_like(q) for _ in range(3)], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for out, splits in zip(outs, (20, 33)):
            grout.attention_decode_window(q, k, v, pos, out, n, 5000, 4, num_splits=splits)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                grout.attention_decode_window(q, k, v, pos, out, n, 5000, 4, num_splits=splits)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    for p in (5999, 10, 3000):
        pos.fill_(p)
        for g in graphs:
            g.replay()
        grout.attention_decode_window(q, k, v, pos, outs[2], n, 5000, 4, num_splits=40)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        grout.check_device_error()
        for out in outs:
            check(out, *attention64(q, k[0].transpose(0, 1), v[0].transpose(0, 1), pos.long(), 5000, 4, SCALE_F16))
