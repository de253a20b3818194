"""GPU checks of sliding-window attention with sinks: single tokens
(contiguous and paged caches) and prompt chunks (varlen and paged) against a
plain 64-bit implementation, at the lengths, windows and layouts where tile
lists, masks and page lookups can go wrong; rows that nobody sees hold NaN and
freed pages have no table entry."""
import pytest
import torch

from window_ref import D, SCALE_F16, attention64, check, free_pages, normal, page_pool

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _caches(B, hkv, n, seed):
    return (normal(seed + k, B, hkv, n, D).half() for k in (1, 2))


def _hide(cache, lens, window, sinks, first_query=None):
    """Sets the rows that no query sees to NaN (queries from first_query[b] on)."""
    c = cache.clone()
    for b, n in enumerate(lens):
        p = n - 1 if first_query is None else first_query[b]
        low = max(0, p - window + 1)
        c[b, :, n:] = NAN
        if low > sinks:
            c[b, :, sinks:low] = NAN
    return c


LENGTHS = [1, 2, 63, 64, 65, 129, 640, 700]


@pytest.mark.parametrize("hq,hkv", [(8, 8), (10, 2), (8, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 0), (64, 4), (65, 64), (100, 65), (128, 200), (700, 3), (5000, 0)])
@pytest.mark.parametrize("splits", [None, 1, 3])
def test_decode_contiguous(grout, hq, hkv, window, sinks, splits):
    B, n = len(LENGTHS), 704
    q = normal(5, B, hq, D, scale=1.5).half()
    k, v = _caches(B, hkv, n, 10)
    k, v = _hide(k, LENGTHS, window, sinks), _hide(v, LENGTHS, window, sinks)
    pos = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda") - 1
    out = torch.full_like(q, NAN)
    grout.attention_decode_window(q, k, v, pos, out, n, window, sinks, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    for b in range(B):
        ref, bound = attention64(q[b:b + 1], k[b].transpose(0, 1), v[b].transpose(0, 1), pos[b:b + 1].long(), window, sinks, SCALE_F16)
        check(out[b:b + 1], ref, bound)


@pytest.mark.parametrize("page_size", [64, 192, 256])
@pytest.mark.parametrize("window,sinks,splits", [(1, 0, None), (70, 4, 2), (200, 130, 16), (333, 1, 40), (4000, 7, None)])
def test_decode_paged(grout, page_size, window, sinks, splits):
    hq, hkv, n = 16, 2, 1500
    lens = [1, 64, 255, 800, 1500]
    B = len(lens)
    q = normal(6, B, hq, D, scale=1.5).half()
    k, v = _caches(B, hkv, n, 20)
    k, v = _hide(k, lens, window, sinks), _hide(v, lens, window, sinks)
    (kp, vp), table = page_pool([k, v], page_size, 3)
    table = free_pages(table, page_size, [m - window for m in lens], sinks)
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
    out = torch.full_like(q, NAN)
    grout.attention_decode_paged_window(q, kp, vp, table, pos, out, n, window, sinks, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    for b in range(B):
        ref, bound = attention64(q[b:b + 1], k[b].transpose(0, 1), v[b].transpose(0, 1), pos[b:b + 1].long(), window, sinks, SCALE_F16)
        check(out[b:b + 1], ref, bound)


def test_decode_of_a_full_window_agrees_with_plain_decode(grout):
    """A window at least as long as the context sees every key: both kernels
    (which sum in different orders) are within the bound of the same result."""
    B, hq, hkv, n = 3, 32, 8, 900
    q = normal(7, B, hq, D).half()
    k, v = _caches(B, hkv, n, 30)
    pos = torch.tensor([899, 0, 450], dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    grout.attention_decode(q, k, v, pos, a, n, num_splits=2)
    grout.attention_decode_window(q, k, v, pos, b, n, 900, 0, num_splits=2)
    torch.cuda.synchronize()
    grout.check_device_error()
    for i in range(B):
        ref, bound = attention64(q[i:i + 1], k[i].transpose(0, 1), v[i].transpose(0, 1), pos[i:i + 1].long(), 0, 0, SCALE_F16)
        check(a[i:i + 1], ref, bound)
        check(b[i:i + 1], ref, bound)


def test_decode_errors_on_the_device(grout):
    """A position past the cache: zero row and 0x200; a bad page that holds a
    visible key: 0x201, its tile left out; one that holds none: no error."""
    hq, hkv, ps = 8, 2, 64
    q = normal(8, 2, hq, D).half()
    kp, vp = (normal(40 + i, 8, hkv, ps, D).half() for i in (0, 1))
    table = torch.tensor([[0, 99, 2, 3], [4, -1, 6, 7]], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, NAN)
    pos = torch.tensor([255, 400], dtype=torch.int32, device="cuda")
    grout.attention_decode_paged_window(q, kp, vp, table, pos, out, 256, 100, 4)  # keys 156..255 and 0..3
    with pytest.raises(grout.GroutError, match="0x200"):
        grout.check_device_error()
    assert (out[1] == 0).all()
    keep = torch.cat([torch.arange(4), torch.arange(156, 256)]).cuda()
    ks, vs = (torch.cat([c[0], c[0], c[2], c[3]], 1).transpose(0, 1)[keep] for c in (kp, vp))
    ref, bound = attention64(q[:1], ks, vs, torch.tensor([255], device="cuda"), 0, 0, SCALE_F16)
    check(out[:1], ref, bound)
    pos = torch.tensor([255, 100], dtype=torch.int32, device="cuda")
    grout.attention_decode_paged_window(q, kp, vp, table, pos, out, 256, 100, 4)  # row 1: keys 1..100, page 1 is bad
    with pytest.raises(grout.GroutError, match="0x201"):
        grout.check_device_error()
    ks, vs = (c[4].transpose(0, 1) for c in (kp, vp))
    ref, bound = attention64(q[1:], ks, vs, torch.tensor([63], device="cuda"), 63 + 1, 4, SCALE_F16)
    check(out[1:], ref, bound)
    # every visible key in a bad page: nothing is left, the row is zero
    table[1] = -1
    for splits in (1, 2):
        grout.attention_decode_paged_window(q, kp, vp, table, pos, out, 256, 100, 4, num_splits=splits)
        with pytest.raises(grout.GroutError, match="0x201"):
            grout.check_device_error()
        assert (out[1] == 0).all()


def test_decode_graph_replay_and_streams(grout):
    """Recorded once on a side stream, replayed while positions grow; two
    recordings with their own workspaces interleave."""
    hq, hkv, n, window, sinks = 8, 1, 4096, 3000, 4
    q = normal(9, 1, hq, D).half()
    k, v = _caches(1, hkv, n, 50)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs, graphs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for splits in (24, 9):  # a workspace merge and a cluster merge
            out = torch.empty_like(q)
            need = grout.decode_window_workspace_bytes(1, n, window, sinks, hq, hkv, n, splits)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            grout.attention_decode_window(q, k, v, pos, out, n, window, sinks, num_splits=splits, workspace=ws)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                grout.attention_decode_window(q, k, v, pos, out, n, window, sinks, num_splits=splits, workspace=ws)
            outs.append((out, ws))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    for p in (0, 100, 2999, 3000, 4095):
        pos.fill_(p)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        grout.check_device_error()
        ref, bound = attention64(q, k[0].transpose(0, 1), v[0].transpose(0, 1), pos.long(), window, sinks, SCALE_F16)
        for out, _ in outs:
            check(out, ref, bound)


def _prefill_ref(q, k, v, cu, firsts, window, sinks):
    """Rows of all sequences in order; k, v [B, Hkv, n, D]."""
    refs, bounds = [], []
    for b in range(len(cu) - 1):
        m = cu[b + 1] - cu[b]
        if m == 0:
            continue
        pos = firsts[b] + torch.arange(m, device="cuda")
        n = firsts[b] + m
        r, e = attention64(q[cu[b]:cu[b + 1]], k[b, :, :n].transpose(0, 1), v[b, :, :n].transpose(0, 1), pos, window, sinks)
        refs.append(r)
        bounds.append(e)
    return torch.cat(refs), torch.cat(bounds)


CHUNKS = [  # (lengths, first positions): one token to several tiles, an empty sequence, odd offsets
    ([1], [0]),
    ([1], [777]),
    ([300], [0]),
    ([513], [1001]),
    ([5, 0, 130, 257, 1], [640, 3, 0, 383, 1023]),
]


@pytest.mark.parametrize("lens,firsts", CHUNKS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (64, 4), (129, 0), (256, 130), (1000, 64), (9000, 5)])
@pytest.mark.parametrize("page_size", [0, 64, 192])
def test_prefill(grout, lens, firsts, window, sinks, page_size):
    hq, hkv = 10, 2
    B, n = len(lens), max(a + b for a, b in zip(lens, firsts))
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    rows = cu[-1]
    q = torch.full((rows + 3, hq, D), NAN, device="cuda").half()
    q[:rows] = normal(11, rows, hq, D, scale=1.5).half()
    k, v = _caches(B, hkv, n, 60)
    ends = [a + b for a, b in zip(lens, firsts)]
    k, v = (_hide(c, ends, window, sinks, firsts) for c in (k, v))
    out = torch.full_like(q, 7.0)
    dcu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    first = torch.tensor(firsts, dtype=torch.int32, device="cuda")
    if page_size:
        (kp, vp), table = page_pool([k, v], page_size, 4)
        table = free_pages(table, page_size, [max(0, p - window + 1) for p in firsts], sinks)
        for b in range(B):
            table[b, -(-max(1, ends[b]) // page_size):] = -1
        grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, cu_seqlens_q=dcu, position_start=first, max_q_len=max(lens))
    else:
        grout.attention_prefill_varlen_window(q, k, v, out, dcu, max(lens), hkv, D, n * D, window, sinks, kv_batch_stride=hkv * n * D, kv_rows=n,
                                              position_start=first)
    torch.cuda.synchronize()
    grout.check_device_error()
    assert (out[rows:] == 7.0).all()  # rows behind the last sequence
    ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
    check(out[:rows], ref, bound)


@pytest.mark.parametrize("batch,hq,hkv", [(3, 64, 8), (40, 8, 1)])
def test_prefill_many_items(grout, batch, hq, hkv):
    """More work items than SMs, in the plain and in the compacted order."""
    window, sinks = 200, 4
    lens = [1 + (37 * i) % 600 for i in range(batch)]
    firsts = [(91 * i) % 500 for i in range(batch)]
    n = max(a + b for a, b in zip(lens, firsts))
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(12, cu[-1], hq, D).half()
    k, v = _caches(batch, hkv, n, 70)
    out = torch.empty_like(q)
    grout.attention_prefill_varlen_window(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device="cuda"), max(lens), hkv, D, n * D, window, sinks,
                                          kv_batch_stride=hkv * n * D, kv_rows=n,
                                          position_start=torch.tensor(firsts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    grout.check_device_error()
    ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
    check(out, ref, bound)


def test_prefill_of_a_full_window_agrees_with_plain_prefill(grout):
    """A window as long as the context: both kernels (which take keys in
    different blocks) are within the bound of the same result."""
    S, hq, hkv, n, p = 400, 16, 4, 900, 300
    q = normal(13, S, hq, D).half()
    k, v = _caches(1, hkv, n, 80)
    a, b = torch.empty_like(q), torch.empty_like(q)
    grout.attention_prefill(q, k[0], v[0], a, p)
    grout.attention_prefill_varlen_window(q, k[0], v[0], b, None, S, hkv, D, n * D, 900, 0,
                                          position_start=torch.tensor([p], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    grout.check_device_error()
    ref, bound = _prefill_ref(q, k, v, [0, S], [p], 0, 0)
    check(a, ref, bound)
    check(b, ref, bound)


def test_prefill_packed_keys(grout):
    """Packed K/V rows of several sequences addressed by kv_start."""
    hq, hkv, window, sinks = 4, 2, 90, 3
    lens = [100, 1, 333]
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(14, cu[-1], hq, D).half()
    k, v = (normal(90 + i, cu[-1], hkv, D).half() for i in (0, 1))
    out = torch.empty_like(q)
    dcu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    grout.attention_prefill_varlen_window(q, k, v, out, dcu, max(lens), hkv, hkv * D, D, window, sinks, kv_start=dcu)
    torch.cuda.synchronize()
    grout.check_device_error()
    for b in range(3):
        at = slice(cu[b], cu[b + 1])
        ref, bound = attention64(q[at], k[at], v[at], torch.arange(lens[b], device="cuda"), window, sinks)
        check(out[at], ref, bound)


def test_prefill_bad_page_is_reported(grout):
    hq, hkv, ps = 4, 2, 64
    q = normal(15, 70, hq, D).half()
    kp, vp = (normal(100 + i, 4, hkv, ps, D).half() for i in (0, 1))
    out = torch.empty_like(q)
    start = torch.tensor([100], dtype=torch.int32, device="cuda")
    table = torch.tensor([[-1, 1, 2]], dtype=torch.int32, device="cuda")
    grout.attention_prefill_paged_window(q, kp, vp, table, out, 30, 0, position_start=start)  # keys 71..169
    torch.cuda.synchronize()
    grout.check_device_error()
    for bad in (-7, 4, 2 ** 31 - 1):
        table[0, 2] = bad
        grout.attention_prefill_paged_window(q, kp, vp, table, out, 30, 0, position_start=start)
        with pytest.raises(grout.GroutError, match="0x201"):
            grout.check_device_error()


def test_graph_of_a_prefill_chunk(grout):
    """A chunk recorded once and replayed at other positions and chunk lengths."""
    hq, hkv, ps, window, sinks = 8, 2, 64, 150, 4
    n = 1024
    q = normal(16, 200, hq, D).half()
    k, v = _caches(1, hkv, n, 110)
    (kp, vp), table = page_pool([k, v], ps, 5)
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    first = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    call = lambda: grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, cu_seqlens_q=cu, position_start=first, max_q_len=200)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
    torch.cuda.current_stream().wait_stream(s)
    for p, m in ((0, 200), (500, 129), (823, 1), (700, 200)):
        first.fill_(p)
        cu[1] = m
        g.replay()
        torch.cuda.synchronize()
        grout.check_device_error()
        ref, bound = _prefill_ref(q, k, v, [0, m], [p], window, sinks)
        check(out[:m], ref, bound)


@pytest.mark.parametrize("hq,hkv", [(3, 3), (6, 2), (7, 1), (33, 3), (100, 1), (128, 1)])
def test_prefill_of_any_group(grout, hq, hkv):
    """Groups that leave rows of the query tile unused, up to one token a tile."""
    lens, firsts, n = [70, 0, 3], [500, 0, 17], 576
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(17, cu[-1], hq, D, scale=1.5).half()
    k, v = _caches(3, hkv, n, 120)
    out = torch.full_like(q, NAN)
    for window, sinks in ((9, 2), (300, 0)):
        grout.attention_prefill_varlen_window(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device="cuda"), 70, hkv, D, n * D, window, sinks,
                                              kv_batch_stride=hkv * n * D, kv_rows=n,
                                              position_start=torch.tensor(firsts, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        grout.check_device_error()
        ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
        check(out, ref, bound)


@pytest.mark.parametrize("hq,hkv", [(8, 2), (8, 1), (4, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 4), (500, 130), (2 ** 31 - 1, 0), (2 ** 40, 2 ** 40)])
def test_prefill_of_short_chunks(grout, hq, hkv, window, sinks):
    """More sequences than a warp looks at together, empty ones among them, no
    chunk longer than a query tile, contexts from one key to many tiles."""
    B, ps, most = 75, 64, 13
    lens = [(5 * i + 3) % (most + 1) if i % 9 else 0 for i in range(B)]
    firsts = [(i * 83) % 1200 if i % 5 else 0 for i in range(B)]
    ends = [a + b for a, b in zip(lens, firsts)]
    n = max(ends)
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(18, cu[-1], hq, D, scale=1.5).half()
    k, v = _caches(B, hkv, n, 130)
    k, v = (_hide(c, ends, window, sinks, firsts) for c in (k, v))
    (kp, vp), table = page_pool([k, v], ps, 6)
    out = torch.full_like(q, NAN)
    grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, max_q_len=most,
                                         cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                         position_start=torch.tensor(firsts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    grout.check_device_error()
    ref, bound = _prefill_ref(q, k, v, cu, firsts, min(window, 2 ** 30), min(sinks, 2 ** 30))
    check(out, ref, bound)


def test_prefill_takes_lengths_from_the_device(grout):
    """max_q_len only sizes the launch: sequences may be longer."""
    hq, hkv, window, sinks = 8, 2, 90, 3
    lens, firsts = [260, 5, 100], [0, 300, 7]
    n = 320
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    q = normal(19, cu[-1], hq, D).half()
    k, v = _caches(3, hkv, n, 140)
    for most in (1, 32, 33, 260, 4000):
        out = torch.full_like(q, NAN)
        grout.attention_prefill_varlen_window(q, k, v, out, torch.tensor(cu, dtype=torch.int32, device="cuda"), most, hkv, D, n * D, window, sinks,
                                              kv_batch_stride=hkv * n * D, kv_rows=n,
                                              position_start=torch.tensor(firsts, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        grout.check_device_error()
        ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
        check(out, ref, bound)


@pytest.mark.parametrize("bad", ["position", "negative", "past_rows", "decreasing"])
@pytest.mark.parametrize("most", [4, 100])
def test_prefill_leaves_out_what_does_not_fit(grout, bad, most):
    """A sequence past the cache or the query rows has no items: its rows stay
    as they were, 0x200 is recorded, the others are right."""
    hq, hkv, ps, window, sinks = 8, 2, 64, 60, 2
    lens, firsts, n = [4, 3, 4], [40, 100, 252], 256
    cu = [0, 4, 7, 11]
    q = normal(20, 11, hq, D).half()
    k, v = _caches(3, hkv, n, 150)
    (kp, vp), table = page_pool([k, v], ps, 7)
    given_cu, given_first, left = list(cu), list(firsts), [1]
    if bad == "position":
        given_first[1] = 254
    elif bad == "negative":
        given_first[1] = -5
    elif bad == "past_rows":
        given_cu[3], left = 12, [2]
    else:
        given_cu[1:3], left = [7, 4], [0, 1, 2]  # rows 0..6 and 4..10 (past the cache at 252): none is checked
    out = torch.full_like(q, 7.0)
    grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, max_q_len=most,
                                         cu_seqlens_q=torch.tensor(given_cu, dtype=torch.int32, device="cuda"),
                                         position_start=torch.tensor(given_first, dtype=torch.int32, device="cuda"))
    with pytest.raises(grout.GroutError, match="0x200"):
        grout.check_device_error()
    ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
    for b in range(3):
        at = slice(cu[b], cu[b + 1])
        if b not in left:
            check(out[at], ref[at], bound[at])
        elif bad != "decreasing":
            assert (out[at] == 7.0).all()


def test_offsets_past_32_bits(grout):
    """f16 pools of more than 2^32 bytes and more than 2^31 elements: only the
    pages at the far end are used."""
    hq, hkv, ps, window, sinks = 8, 1, 1024, 500, 70
    pages = 2 ** 31 // (hkv * ps * D) + 4
    k, v = (normal(160 + i, 1, hkv, 2 * ps, D).half() for i in (0, 1))
    kp, vp = (torch.empty(pages, hkv, ps, D, dtype=torch.float16, device="cuda") for _ in "kv")
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    for pool, c in ((kp, k), (vp, v)):
        pool[pages - 1], pool[pages - 3] = c[0, :, :ps], c[0, :, ps:]
    q = normal(21, 40, hq, D).half()
    out = torch.empty_like(q)
    grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, position_start=torch.tensor([1300], dtype=torch.int32, device="cuda"))
    one = torch.empty_like(q[:1])
    pos = torch.tensor([1339], dtype=torch.int32, device="cuda")
    grout.attention_decode_paged_window(q[39:], kp, vp, table, pos, one, 2 * ps, window, sinks)
    torch.cuda.synchronize()
    grout.check_device_error()
    ref, bound = _prefill_ref(q, k, v, [0, 40], [1300], window, sinks)
    check(out, ref, bound)
    ref, bound = attention64(q[39:], k[0].transpose(0, 1), v[0].transpose(0, 1), pos.long(), window, sinks, SCALE_F16)
    check(one, ref, bound)


def test_calls_on_two_streams_at_once(grout):
    """Decode with its own workspace and a chunk, on two streams, many times:
    the results are those of the calls alone, bit for bit."""
    hq, hkv, n, window, sinks = 8, 1, 8192, 6000, 4
    q = normal(22, 2, 64, hq, D).half()
    k, v = _caches(1, hkv, n, 170)
    pos = torch.tensor([8000], dtype=torch.int32, device="cuda")
    first = torch.tensor([5000], dtype=torch.int32, device="cuda")

    def run(i):
        a, b = torch.full_like(q[i, :1], NAN), torch.full_like(q[i], NAN)
        grout.attention_decode_window(q[i, :1], k, v, pos, a, n, window, sinks, num_splits=30)
        grout.attention_prefill_varlen_window(q[i], k, v, b, None, 64, hkv, D, n * D, window, sinks, kv_rows=n, position_start=first)
        return a, b

    want = [run(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    grout.check_device_error()
    for i in (0, 1):
        for pair in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(pair, want[i]))


@pytest.mark.parametrize("lens,firsts", CHUNKS + [([3] * 9, [10, 700, 0, 129, 64, 2000, 1, 1500, 333])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (129, 70), (1000, 64), (9000, 5)])
@pytest.mark.parametrize("page_size", [0, 192])
@pytest.mark.parametrize("splits", [2, 5, 32])
def test_prefill_splits(grout, lens, firsts, window, sinks, page_size, splits):
    """Keys cut into runs, more of them than tiles among the counts: same results,
    rows behind the last sequence left alone, whatever the workspace held."""
    hq, hkv = 10, 2
    B, n = len(lens), max(a + b for a, b in zip(lens, firsts))
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    rows = cu[-1]
    q = torch.full((rows + 3, hq, D), NAN, device="cuda").half()
    q[:rows] = normal(31, rows, hq, D, scale=1.5).half()
    k, v = _caches(B, hkv, n, 180)
    ends = [a + b for a, b in zip(lens, firsts)]
    k, v = (_hide(c, ends, window, sinks, firsts) for c in (k, v))
    out = torch.full_like(q, 7.0)
    dcu, first = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, firsts))
    need = grout.prefill_window_workspace_bytes(rows + 3, splits, hq, hkv)
    ws = torch.full((need // 4,), NAN, device="cuda")
    if page_size:
        (kp, vp), table = page_pool([k, v], page_size, 4)
        table = free_pages(table, page_size, [max(0, p - window + 1) for p in firsts], sinks)
        grout.attention_prefill_paged_window(q, kp, vp, table, out, window, sinks, cu_seqlens_q=dcu, position_start=first, max_q_len=max(lens),
                                             workspace=ws, num_splits=splits)
    else:
        grout.attention_prefill_varlen_window(q, k, v, out, dcu, max(lens), hkv, D, n * D, window, sinks, kv_batch_stride=hkv * n * D, kv_rows=n,
                                              position_start=first, workspace=ws, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    assert (out[rows:] == 7.0).all()
    ref, bound = _prefill_ref(q, k, v, cu, firsts, window, sinks)
    check(out[:rows], ref, bound)


def test_prefill_of_few_rows_over_a_long_context(grout):
    """The automatic count splits; a NaN in a seen key makes its rows NaN, a
    sequence that does not fit is left out."""
    hq, hkv, n, S = 16, 2, 20000, 6
    assert grout.prefill_window_splits(1, S, n, n, 0, hq, hkv) > 8
    q = normal(32, S, hq, D).half()
    k, v = _caches(1, hkv, n, 190)
    out = torch.full_like(q, NAN)
    call = lambda p, w: grout.attention_prefill_varlen_window(q, k, v, out, None, S, hkv, D, n * D, w, 3, kv_rows=n,  # noqa: E731
                                                              position_start=torch.tensor([p], dtype=torch.int32, device="cuda"))
    for p in (n - S, 5000, 40, 0):
        for w in (n, 10000):
            call(p, w)
            torch.cuda.synchronize()
            grout.check_device_error()
            ref, bound = _prefill_ref(q, k, v, [0, S], [p], w, 3)
            check(out, ref, bound)
    k[0, 1, 7777, 5] = NAN
    call(15000, n)
    assert torch.isnan(out[:, hq // 2:]).all() and torch.isfinite(out[:, : hq // 2]).all()
    out.fill_(7.0)
    call(n - 3, n)
    with pytest.raises(grout.GroutError, match="0x200"):
        grout.check_device_error()
    assert (out == 7.0).all()


def test_split_prefill_in_a_graph_and_with_spare_rows(grout):
    """The automatic split recorded once and replayed at other positions, lengths
    and beside eager calls; a q of many spare rows is not split beyond its
    workspace."""
    hq, hkv, n, ps = 8, 2, 6000, 64
    q = normal(33, 12, hq, D).half()
    k, v = _caches(2, hkv, n, 200)
    (kp, vp), table = page_pool([k, v], ps, 8)
    cu, first = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    assert grout.prefill_window_splits(2, 7, table.shape[1] * ps, 3500, 4, hq, hkv) > 4
    outs = [torch.full_like(q, 7.0) for _ in range(2)]
    call = lambda x, o: grout.attention_prefill_paged_window(x, kp, vp, table, o, 3500, 4, cu_seqlens_q=cu, position_start=first, max_q_len=7)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(q, outs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(q, outs[0])
    torch.cuda.current_stream().wait_stream(s)
    spare = torch.zeros(30000, hq, D, dtype=torch.float16, device="cuda")
    spare[:12] = q
    wide = torch.full_like(spare, 7.0)
    for lens, at in (([5, 7], [5000, 100]), ([1, 2], [0, 5900]), ([0, 7], [9, 4000])):
        cu.copy_(torch.tensor([0, lens[0], sum(lens)]))
        first.copy_(torch.tensor(at))
        for o in outs + [wide]:
            o.fill_(7.0)
        g.replay()
        call(q, outs[1])
        g.replay()
        call(spare, wide)
        torch.cuda.synchronize()
        grout.check_device_error()
        m = sum(lens)
        ref, bound = _prefill_ref(q, k, v, [0, lens[0], m], at, 3500, 4)
        for o in outs + [wide]:
            check(o[:m], ref, bound)
            assert (o[m:] == 7.0).all()
