"""More GPU checks of the window attention and 8-bit cache calls: scales that
are NaN, counts and workspaces that are refused, positions next to 2^31, runs
of many key tiles in one CTA."""
import pytest
import torch

from window_ref import D, SCALE_F16, attention64, check, fp8_cache, free_pages, normal, page_pool, values

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("splits", [1, 3, 20])
@pytest.mark.parametrize("row", [0, 100, 299])
def test_a_nan_value_scale_reaches_the_rows_that_see_it(grout, splits, row):
    """A cache row stands for code * scale: with a NaN scale every element of a
    value row is NaN, in attention as in the read-back.  Out of the window it
    is not seen."""
    hq, hkv, n, ps = 8, 2, 320, 64
    (kc, ks), (vc, vs) = (fp8_cache(s, n // ps, hkv, ps, D) for s in (10, 20))
    table = torch.arange(n // ps, dtype=torch.int32, device="cuda").view(1, -1)
    pos = _i32(299)
    q = normal(30, 1, hq, D).half()
    vs[row // ps, 1, row % ps] = NAN
    out = torch.empty_like(q)
    grout.attention_decode_paged_fp8(q, kc, vc, ks, vs, table, pos, out, n, num_splits=splits)
    ko, vo = (torch.empty(300, hkv, D, dtype=torch.float16, device="cuda") for _ in "kv")
    grout.kv_read_paged_fp8(kc, vc, ks, vs, table, ko, vo, _i32(0, 300))
    torch.cuda.synchronize()
    grout.check_device_error()
    assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all()
    assert torch.isnan(vo[row, 1]).all() and torch.isfinite(vo[row, 0]).all()
    if row == 100:
        grout.attention_decode_paged_fp8(q, kc, vc, ks, vs, table, pos, out, n, 199, 100, num_splits=splits)  # keys 101..299 and 0..99
        k, v = (values(c, s).transpose(1, 2).reshape(n, hkv, D)[:300] for c, s in ((kc, ks), (vc, vs)))
        v[row, 1] = 0.0
        check(out, *attention64(q, k, v, pos.long(), 199, 100, SCALE_F16))


def _calls(grout, B=2, hq=8, hkv=2):
    """name -> (call with extra keywords, most splits)"""
    f16 = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    q, out, kv = f16(B, hq, D), f16(B, hq, D), f16(B, hkv, 128, D)
    codes = torch.zeros(B, hkv, 128, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(B, hkv, 128, device="cuda")
    table, pos = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1), torch.full((B,), 127, dtype=torch.int32, device="cuda")
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    return {
        "decode": (lambda **x: grout.attention_decode_window(q, kv, kv, pos, out, 128, 100, 3, **x), 1024),
        "paged": (lambda **x: grout.attention_decode_paged_window(q, kv, kv, table, pos, out, 128, 100, 3, **x), 1024),
        "fp8": (lambda **x: grout.attention_decode_paged_fp8(q, codes, codes, scales, scales, table, pos, out, 128, **x), 1024),
        "varlen": (lambda **x: grout.attention_prefill_varlen_window(q, kv, kv, out, cu, 1, hkv, D, 128 * D, 100, 3, kv_rows=128,
                                                                     kv_batch_stride=hkv * 128 * D, position_start=pos, **x), 32),
        "chunk": (lambda **x: grout.attention_prefill_paged_window(q, kv, kv, table, out, 100, 3, cu_seqlens_q=cu, position_start=pos, max_q_len=1, **x), 32),
    }


@pytest.mark.parametrize("name", ["decode", "paged", "fp8", "varlen", "chunk"])
def test_split_counts_are_refused_before_a_workspace_is_made(grout, name):
    call, most = _calls(grout)[name]
    for n in (1, most, 0, None):
        call(num_splits=n)
    torch.cuda.synchronize()
    grout.check_device_error()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    for n in (-1, most + 1, 10 ** 5, 2 ** 31 - 1, -(2 ** 31)):
        with pytest.raises(grout.GroutError, match="num_splits"):
            call(num_splits=n)
    assert torch.cuda.max_memory_allocated() == held
    call()
    torch.cuda.synchronize()
    grout.check_device_error()


def test_a_split_prefill_of_too_many_sequences_is_refused_before_a_workspace_is_made(grout):
    B = 65536
    q, out, kv = (torch.zeros(n, h, D, dtype=torch.float16, device="cuda") for n, h in ((B, 2), (B, 2), (1, 1)))
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    with pytest.raises(grout.GroutError, match="batch"):
        grout.attention_prefill_varlen_window(q, kv, kv, out, cu, 1, 1, D, D, 100, num_splits=4)
    assert torch.cuda.max_memory_allocated() == held
    grout.attention_prefill_varlen_window(q, kv, kv, out, cu, 1, 1, D, D, 100)
    torch.cuda.synchronize()
    grout.check_device_error()


@pytest.mark.parametrize("name", ["decode", "paged", "fp8", "varlen", "chunk"])
def test_a_workspace_that_cannot_be_had_is_out_of_memory(grout, name):
    """As PyTorch reports it, so that a caller can make the batch smaller and try
    again: here PyTorch itself is told to hold no more than it does."""
    calls = _calls(grout, B=4096, hq=64, hkv=8) if name in ("varlen", "chunk") else _calls(grout, B=64, hq=64, hkv=8)
    call, most = calls[name]
    call(num_splits=1)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + 2 ** 28) / torch.cuda.get_device_properties(0).total_memory)
        with pytest.raises(torch.OutOfMemoryError):
            call(num_splits=most)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    call(num_splits=most)
    torch.cuda.synchronize()
    grout.check_device_error()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("position", [2 ** 31 - 2, 2 ** 31 - 65, 2 ** 31 - 1025])
@pytest.mark.parametrize("window,sinks", [(1, 0), (70, 5), (2500, 200)])
def test_decode_next_to_the_last_position(grout, fp8, position, window, sinks):
    """Tables of 2^31 positions whose pages are freed but for the sinks' and the
    window's: the counts of tiles and keys stay in 32 bits."""
    hq, hkv, ps = 8, 2, 1024
    table = torch.full((1, 2 ** 31 // ps), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 3
    table[0, -4:] = _i32(2, 5, 0, 4)
    q = normal(40, 1, hq, D, scale=1.5).half()
    out = torch.full_like(q, NAN)
    pos = _i32(position)
    if fp8:
        (kc, ks), (vc, vs) = (fp8_cache(s, 6, hkv, ps, D) for s in (50, 60))
        k, v = values(kc, ks), values(vc, vs)
        call = lambda n: grout.attention_decode_paged_fp8(q, kc, vc, ks, vs, table, pos, out, 2 ** 31 - 1, window, sinks, max_seq=2 ** 31 - 1, num_splits=n)  # noqa: E731
    else:
        k, v = (normal(s, 6, hkv, ps, D).half() for s in (50, 60))
        call = lambda n: grout.attention_decode_paged_window(q, k, v, table, pos, out, 2 ** 31 - 1, window, sinks, max_seq=2 ** 31 - 1, num_splits=n)  # noqa: E731
    keys = torch.cat([torch.arange(sinks), torch.arange(position - window + 1, position + 1)]).cuda()
    rows = [x[table[0, keys // ps].long(), :, keys % ps] for x in (k, v)]
    for n in (None, 1, 3, 20):
        out.fill_(NAN)
        call(n)
        torch.cuda.synchronize()
        grout.check_device_error()
        check(out, *attention64(q, *rows, torch.tensor([len(keys) - 1], device="cuda"), 0, 0, SCALE_F16))


def test_plain_decode_next_to_the_last_position(grout):
    """2^31 - 1 keys, every page but the last one the same: the last tile is
    attended to and the one key behind the position is not.  Key 1000 of the
    last page outscores all others by more than 100 (weights below e^-100), the
    unseen key 1023 would outscore it."""
    hq, hkv, ps = 8, 1, 1024
    table = torch.zeros(1, 2 ** 31 // ps, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    k, v = (normal(s, 2, hkv, ps, D, scale=0.01).half() for s in (70, 71))
    q = torch.full((1, hq, D), 4.0, dtype=torch.float16, device="cuda")
    k[1, 0, 1000], k[1, 0, 1023] = 4.0, 8.0  # scores 4 * 4 * 128 * scale = 181 and 362; the others are within 10
    out = torch.full_like(q, NAN)
    grout.attention_decode_paged(q, k, v, table, _i32(2 ** 31 - 2), out, 2 ** 31 - 1, max_seq=2 ** 31 - 1)
    torch.cuda.synchronize()
    grout.check_device_error()
    assert torch.equal(out, v[1, :, 1000].expand_as(out))


def _hidden(cache, first, last, window, sinks):
    """A cache [1, Hkv, n, ...] whose rows that no query of positions first .. last sees are NaN (8-bit codes: 0x7F)."""
    c = cache.clone()
    low = max(0, first - window + 1)
    fill = 0x7F if c.dtype is torch.uint8 else NAN
    c[:, :, last + 1:] = fill
    if low > sinks:
        c[:, :, sinks:low] = fill
    return c


@pytest.mark.parametrize("page_size", [0, 64, 192])
@pytest.mark.parametrize("position,window,sinks", [(5200, 4900, 130), (6100, 9000, 0), (6100, 4160, 64)])
@pytest.mark.parametrize("splits", [1, 2])
def test_decode_of_many_tiles_per_cta(grout, page_size, position, window, sinks, splits):
    """More than 64 tiles of 64 keys in a split (pages are looked up 32 tiles at
    a time), sinks and window from shuffled pages with freed ones between."""
    hq, hkv, n = 8, 1, 6200
    q = normal(80, 1, hq, D, scale=1.5).half()
    k, v = (_hidden(normal(s, 1, hkv, n, D).half(), position, position, window, sinks) for s in (81, 82))
    out, pos = torch.full_like(q, NAN), _i32(position)
    if page_size:
        (kp, vp), table = page_pool([k, v], page_size, 9)
        table = free_pages(table, page_size, [position - window + 1], sinks)
        grout.attention_decode_paged_window(q, kp, vp, table, pos, out, n, window, sinks, num_splits=splits)
    else:
        grout.attention_decode_window(q, k, v, pos, out, n, window, sinks, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    check(out, *attention64(q, k[0].transpose(0, 1), v[0].transpose(0, 1), pos.long(), window, sinks, SCALE_F16))


@pytest.mark.parametrize("page_size", [64, 192])
@pytest.mark.parametrize("position,window,sinks", [(5200, 4900, 130), (6100, 0, 0), (6100, 4160, 64)])
@pytest.mark.parametrize("splits", [1, 2])
def test_8_bit_decode_of_many_tiles_per_cta(grout, page_size, position, window, sinks, splits):
    hq, hkv, n = 8, 1, 6200
    q = normal(90, 1, hq, D, scale=1.5).half()
    (kc, ks), (vc, vs) = (fp8_cache(s, 1, hkv, n, D) for s in (91, 93))
    parts = [_hidden(x, position, position, window or n, sinks) for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    pools, table = page_pool(parts, page_size, 9, fill=0x7F)
    table = free_pages(table, page_size, [position - (window or n) + 1], sinks)
    pools = [p.view(torch.float8_e4m3fn) for p in pools[:2]] + pools[2:]
    out, pos = torch.full_like(q, NAN), _i32(position)
    grout.attention_decode_paged_fp8(q, *pools, table, pos, out, n, window, sinks, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    check(out, *attention64(q, values(kc, ks)[0].transpose(0, 1), values(vc, vs)[0].transpose(0, 1), pos.long(), window, sinks, SCALE_F16))


@pytest.mark.parametrize("page_size", [0, 64, 192])
@pytest.mark.parametrize("tokens", [5, 45])
@pytest.mark.parametrize("position,window,sinks", [(5000, 4500, 130), (5000, 9000, 0), (9000, 4160, 64)])
@pytest.mark.parametrize("splits", [1, 2])
def test_prefill_of_many_tiles_per_item(grout, page_size, tokens, position, window, sinks, splits):
    """More than 32 tiles of 128 keys for a block of rows (pages are looked up 16
    tiles at a time), by both chains on one query tile and by two query tiles."""
    hq, hkv, n = 8, 1, position + tokens
    q = normal(100, tokens, hq, D, scale=1.5).half()
    k, v = (_hidden(normal(s, 1, hkv, n, D).half(), position, n - 1, window, sinks) for s in (101, 102))
    out, first = torch.full_like(q, NAN), _i32(position)
    if page_size:
        (kp, vp), table = page_pool([k, v], page_size, 9)
        table = free_pages(table, page_size, [position - window + 1], sinks)
        grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, position_start=first, num_splits=splits)
    else:
        grout.attention_prefill_varlen_window(q, k, v, out, None, tokens, hkv, D, n * D, window, sinks, kv_rows=n, position_start=first, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    pos = position + torch.arange(tokens, device="cuda")
    check(out, *attention64(q, k[0].transpose(0, 1), v[0].transpose(0, 1), pos, window, sinks))


def test_chunk_over_the_8_bit_cache_with_sinks_and_freed_pages(grout):
    """The sinks and the window of each sequence read back as two neighbouring
    runs (two rows of the page table each); positions count the joined rows.
    Sequences before and past their windows, freed pages between the runs."""
    hq, hkv, ps, window, sinks, n = 8, 2, 64, 300, 70, 2000
    firsts, lens = [1500, 0, 369, 1900, 200], [40, 33, 1, 100, 260]
    B = len(lens)
    (kc, ks), (vc, vs) = (fp8_cache(s, B, hkv, n, D) for s in (110, 112))
    parts = [x.clone() for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    for x in parts:  # what nobody sees
        for b in range(B):
            x[b, :, firsts[b] + lens[b]:] = 0x7F if x.dtype is torch.uint8 else NAN
            if firsts[b] - window + 1 > sinks:
                x[b, :, sinks:firsts[b] - window + 1] = 0x7F if x.dtype is torch.uint8 else NAN
    pools, table = page_pool(parts, ps, 11, fill=0x7F)
    pools = [p.view(torch.float8_e4m3fn) for p in pools[:2]] + pools[2:]
    table = free_pages(table, ps, [p - window + 1 for p in firsts], sinks)
    assert (table == -1).any()
    runs, starts, at = [], [], []
    for p, m in zip(firsts, lens):
        low = p - window + 1
        if low <= sinks:
            low, held = 0, 0
        else:
            held = sinks
        runs += [held, p + m - low]
        starts += [0, low]
        at.append(held + p - low)
    ends = torch.tensor([0] + runs).cumsum(0)
    ko, vo = (torch.empty(int(ends[-1]), hkv, D, dtype=torch.float16, device="cuda") for _ in "kv")
    grout.kv_read_paged_fp8(*pools, table.repeat_interleave(2, 0), ko, vo, ends.int().cuda(), position_start=_i32(*starts))
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(120, cu[-1], hq, D, scale=1.5).half()
    out = torch.full_like(q, NAN)
    grout.attention_prefill_varlen_window(q, ko, vo, out, _i32(*cu), max(lens), hkv, hkv * D, D, window, sinks, position_start=_i32(*at),
                                          kv_start=ends[:-1:2].int().cuda())
    torch.cuda.synchronize()
    grout.check_device_error()
    for b in range(B):
        rows = slice(cu[b], cu[b + 1])
        k, v = ((c[b].float() * s[b, ..., None]).half().transpose(0, 1) for c, s in ((kc, ks), (vc, vs)))  # the read-back's roundings
        pos = firsts[b] + torch.arange(lens[b], device="cuda")
        check(out[rows], *attention64(q[rows], k, v, pos, window, sinks))


@pytest.mark.parametrize("splits", [1, 2])
def test_infinite_scores(grout, splits):
    """+infinity (or NaN) among the visible scores: NaN; -infinity: no weight; nothing but -infinity: zero."""
    hq, hkv, n, p = 8, 2, 192, 150
    q = normal(130, 1, hq, D).abs().half() + 1
    k, v = (normal(s, 1, hkv, n, D).half() for s in (131, 132))
    pos = _i32(p)
    for bad, window, want in ((float("-inf"), 1, "zero"), (float("inf"), 1, "nan"), (float("-inf"), 2, "other"), (float("inf"), 100, "nan"), (NAN, 100, "nan")):
        kb = k.clone()
        kb[0, 0, p, 3] = bad
        a, b = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
        grout.attention_decode_window(q, kb, v, pos, a, n, window, 0, num_splits=splits)
        grout.attention_prefill_varlen_window(q, kb, v, b, None, 1, hkv, D, n * D, window, 0, kv_rows=n, position_start=pos, num_splits=splits)
        torch.cuda.synchronize()
        grout.check_device_error()
        for o in (a, b):
            if want == "nan":
                assert torch.isnan(o[0, :4]).all()
            elif want == "zero":
                assert (o[0, :4] == 0).all()
            else:
                assert torch.equal(o[0, :4], v[0, :1, p - 1].expand(4, D))
            assert torch.isfinite(o[0, 4:]).all() and (o[0, 4:] != 7.0).any()
