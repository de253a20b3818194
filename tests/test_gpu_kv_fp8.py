"""GPU checks of the 8-bit paged KV cache: the fused write (codes and scales
bit for bit against the same f32 arithmetic on the CPU, and against 64 bits),
the read-back, decode attention over it, and a serving run of all of them."""
import math

import numpy as np
import pytest
import torch

import oracle
from grout_b200 import synth
from window_ref import D, SCALE_F16, attention64, check, fp8_cache, free_pages, normal, page_pool, quantise64, values

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1.0e6
NAN = float("nan")


def _norm_rope32(x, w, tab, pos):
    """numpy f32, every operation rounded once, the squares in the kernel's
    order: [rows, heads, D] f16 -> f32."""
    x = x.astype(np.float32)
    lo, hi = x[..., :64], x[..., 64:]
    t = (lo * lo + hi * hi).reshape(*x.shape[:-1], 8, 8)
    s = ((t[..., 0] + t[..., 1]) + (t[..., 2] + t[..., 3])) + ((t[..., 4] + t[..., 5]) + (t[..., 6] + t[..., 7]))
    for half in (4, 2, 1):
        s = s[..., :half] + s[..., half:]
    inv = np.float32(1) / np.sqrt(s * np.float32(0.0078125) + np.float32(EPS))
    n = x * inv * w.astype(np.float32)
    lo, hi = n[..., :64], n[..., 64:]
    cos, sin = tab[pos][:, 0][:, None], tab[pos][:, 1][:, None]
    return np.concatenate([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _quantise32(y, exact):
    """f32 rows -> (code bytes, scales); exact (V): the quotient rounded to f32
    once, else (K) y times the factor 448 (1 / max), each step rounded."""
    top = np.abs(y).max(-1)
    zero = top <= 2.0 ** -25
    with np.errstate(divide="ignore", invalid="ignore"):
        x = y * np.float32(448) / top[..., None] if exact else y * (np.float32(448) * (np.float32(1) / top))[..., None]
        x = np.where(zero[..., None], y * np.float32(0), x).astype(np.float32)
    code = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return code, np.where(zero, np.float32(0), top / np.float32(448)).astype(np.float32)


def _pools(pages, hkv, ps):
    """Pools with a recognisable filling."""
    codes = [torch.full((pages, hkv, ps, D), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    return codes + [torch.full((pages, hkv, ps), -3.0, device="cuda") for _ in range(2)]


def _expect(pools, table, rows, ks, vs, ps):
    """Checks that exactly the rows (sequence, position) were written, bit for bit."""
    want = [p.clone() for p in _pools(*pools[0].shape[:3])]
    codes = [w.view(torch.uint8).cpu().numpy() for w in want[:2]]
    scales = [w.cpu().numpy() for w in want[2:]]
    for y, code, scale in ((ks, codes[0], scales[0]), (vs, codes[1], scales[1])):
        c, s = _quantise32(y, y is vs)
        for i, (b, p) in enumerate(rows):
            page = int(table[b, p // ps])
            code[page, :, p % ps] = c[i]
            scale[page, :, p % ps] = s[i]
    for got, w in zip(pools[:2], codes):
        assert np.array_equal(got.view(torch.uint8).cpu().numpy(), w)
    for got, w in zip(pools[2:], scales):
        assert np.array_equal(got.cpu().numpy().view(np.uint32), w.view(np.uint32))


T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731


@pytest.mark.parametrize("B,hq,hkv,ps", [(1, 64, 8, 64), (5, 10, 2, 192), (300, 8, 1, 64)])
def test_decode_write(grout, B, hq, hkv, ps):
    per = 3
    ms = per * ps
    qkv = (synth.normal(11, B * (hq + 2 * hkv) * D).reshape(B, -1).astype(np.float32) * np.exp(synth.normal(12, B).astype(np.float32))[:, None]).astype(np.float16)
    qw, kw = synth.norm_weight(4, D), synth.norm_weight(5, D)
    tab = oracle.rope_table(oracle.inv_freq(THETA, D), ms)
    pos = (np.arange(B) * 97 + 63) % ms
    table = torch.randperm(B * per + 2, generator=torch.Generator().manual_seed(1))[: B * per].view(B, per).int()
    pools = _pools(B * per + 2, hkv, ps)
    q_out = torch.empty(B, hq, D, dtype=torch.float16, device="cuda")
    grout.qk_norm_rope_kv_decode_paged_fp8(T(qkv), T(qw), T(kw), grout.rope_table(THETA, ms), q_out, *pools, table.cuda(), T(pos.astype(np.int32)), hq, hkv, EPS)
    torch.cuda.synchronize()
    grout.check_device_error()
    x = qkv.reshape(B, hq + 2 * hkv, D)
    q = _norm_rope32(x[:, :hq], qw, tab, pos).astype(np.float16)
    assert np.array_equal(q_out.cpu().numpy().view(np.uint16), q.view(np.uint16))
    _expect(pools, table, list(enumerate(pos.tolist())), _norm_rope32(x[:, hq:hq + hkv], kw, tab, pos), x[:, hq + hkv:].astype(np.float32), ps)


@pytest.mark.parametrize("S,pos0,hq,hkv,ps", [(1, 0, 8, 8, 64), (300, 100, 10, 2, 192), (700, 65, 64, 8, 64), (2000, 0, 2, 1, 1024)])
def test_prefill_write(grout, S, pos0, hq, hkv, ps):
    ms = -(-(pos0 + S) // ps) * ps
    q, k, v = (synth.normal(20 + i, S * h * D).reshape(S, h, D) for i, h in enumerate((hq, hkv, hkv)))
    qw, kw = synth.norm_weight(4, D), synth.norm_weight(5, D)
    tab = oracle.rope_table(oracle.inv_freq(THETA, D), ms)
    table = torch.randperm(ms // ps + 2, generator=torch.Generator().manual_seed(2))[: ms // ps].view(1, -1).int()
    pools = _pools(ms // ps + 2, hkv, ps)
    q_out = torch.empty(S, hq, D, dtype=torch.float16, device="cuda")
    grout.qk_norm_rope_kv_prefill_paged_fp8(T(q), T(k), T(v), T(qw), T(kw), grout.rope_table(THETA, ms), q_out, *pools, table[0].cuda(), pos0, EPS)
    torch.cuda.synchronize()
    grout.check_device_error()
    pos = pos0 + np.arange(S)
    assert np.array_equal(q_out.cpu().numpy().view(np.uint16), _norm_rope32(q, qw, tab, pos).astype(np.float16).view(np.uint16))
    _expect(pools, table, [(0, p) for p in pos.tolist()], _norm_rope32(k, kw, tab, pos), v.astype(np.float32), ps)
    # in 64 bits: half a step of e4m3 relative to the value (2^-4), or of its subnormal step (2^-10)
    # relative to the row's scale; f32 rounding of scale, reciprocal and product adds 3 * 2^-24
    got = values(pools[1].view(torch.uint8)[table[0].cuda().long()[T(pos // ps)], :, T(pos % ps)].view(torch.float8_e4m3fn),
                 pools[3][table[0].cuda().long()[T(pos // ps)], :, T(pos % ps)])
    y = T(v).double()
    step = torch.maximum(y.abs() * 2.0 ** -4, y.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10)
    assert ((got - y).abs() <= step * (1 + 2.0 ** -10)).all()


def test_write_of_unusual_rows(grout):
    """Zero rows, the smallest and largest f16 values, NaN and infinities."""
    hq, hkv, ps = 1, 1, 64
    v = torch.zeros(8, hkv, D, dtype=torch.float16)
    v[1, 0, 5] = 2.0 ** -24           # f16's smallest value: the row's only one
    v[2, 0] = 65504.0
    v[3, 0, :3] = torch.tensor([65504.0, 1.0, -2.0 ** -24])
    v[4, 0] = torch.linspace(-1, 1, D)
    v[4, 0, 7] = NAN
    v[5, 0] = torch.linspace(-1, 1, D)
    v[5, 0, 0] = math.inf
    v[6, 0] = -0.0
    v[7, 0] = torch.linspace(-448, 448, D)
    q = torch.zeros(8, hq, D, dtype=torch.float16, device="cuda")
    pools = _pools(1, hkv, ps)
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    grout.qk_norm_rope_kv_prefill_paged_fp8(q, torch.zeros(8, hkv, D, dtype=torch.float16, device="cuda"), v.cuda(), w, w, grout.rope_table(THETA, ps), torch.empty_like(q),
                                            *pools, torch.zeros(1, dtype=torch.int32, device="cuda"), 0, EPS)
    torch.cuda.synchronize()
    grout.check_device_error()
    ko, vo = (torch.full((8, hkv, D), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    grout.kv_read_paged_fp8(*pools, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), ko, vo, cu)
    torch.cuda.synchronize()
    grout.check_device_error()
    assert (ko == 0).all() and (pools[2][0, 0, :8] == 0).all()
    vo = vo.cpu()
    assert (vo[0] == 0).all() and (vo[6] == 0).all()
    assert vo[1, 0, 5] == 2.0 ** -24 and vo[1].count_nonzero() == 1
    assert (vo[2] == 65504.0).all()
    assert vo[3, 0, 0] == 65504.0 and vo[3, 0, 2] == 0
    assert torch.isnan(vo[4, 0, 7]) and torch.isfinite(vo[4, 0, 8:]).all() and vo[4, 0, -1] == 1.0
    assert torch.isnan(vo[5]).all()
    assert ((vo[7] - v[7]).abs() <= v[7].abs() * 2.0 ** -4 + 2.0 ** -10).all()


def test_write_errors_on_the_device(grout):
    hq, hkv, ps = 8, 2, 64
    qkv = normal(30, 3, (hq + 2 * hkv) * D).half()
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    table = torch.tensor([[0, 9], [1, -1], [2, 3]], dtype=torch.int32, device="cuda")
    pools = _pools(4, hkv, ps)
    rope = grout.rope_table(THETA, 128)
    q_out = torch.empty(3, hq, D, dtype=torch.float16, device="cuda")
    for pos, code in (([64, 127, 1], "0x201"), ([0, 128, 127], "0x200")):
        want = [p.clone() for p in pools]
        pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
        grout.qk_norm_rope_kv_decode_paged_fp8(qkv, w, w, rope, q_out, *pools, table, pos, hq, hkv, EPS)
        with pytest.raises(grout.GroutError, match=code):
            grout.check_device_error()
        wrote = [int((a.view(torch.int32) != b.view(torch.int32)).any((-1, -2)).any(-1).sum()) if a.dim() == 4 else 0 for a, b in zip(pools, want)]
        assert wrote[0] == wrote[1] == (1 if code == "0x201" else 2)


@pytest.mark.parametrize("hkv,ps", [(1, 64), (3, 192), (8, 1024)])
def test_read(grout, hkv, ps):
    lens, firsts = [0, 5, 130, 0, 1, 777, 0], [9, 0, 100, 0, 1023, 3, 0]
    B, n, rows = len(lens), 1024, sum(lens)
    (kc, ks), (vc, vs) = (fp8_cache(40 + 2 * i, B, hkv, n, D) for i in range(2))
    (kp, vp, ksp, vsp), table = page_pool([kc.view(torch.uint8), vc.view(torch.uint8), ks, vs], ps, 6, fill=0)
    kp, vp = (x.view(torch.float8_e4m3fn) for x in (kp, vp))
    cu = torch.tensor([0] + lens).cumsum(0).tolist()
    ko, vo = (torch.full((rows + 4, hkv, D), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    grout.kv_read_paged_fp8(kp, vp, ksp, vsp, table, ko, vo, ints(cu), ints(firsts))
    torch.cuda.synchronize()
    grout.check_device_error()
    for got, c, s in ((ko, kc, ks), (vo, vc, vs)):
        assert (got[rows:] == 5.0).all()
        for b in range(B):
            at = slice(firsts[b], firsts[b] + lens[b])
            want = (c.float()[b, :, at] * s[b, :, at, None]).half().transpose(0, 1)
            assert torch.equal(got[cu[b]:cu[b + 1]].view(torch.int16), want.contiguous().view(torch.int16))
    # a position past the cache and a bad page read as zeros
    table[1, 0] = 10 ** 6
    grout.kv_read_paged_fp8(kp, vp, ksp, vsp, table, ko, vo, ints(cu), ints(firsts))
    with pytest.raises(grout.GroutError, match="0x201"):
        grout.check_device_error()
    assert (ko[:5] == 0).all() and (ko[5:rows] != 0).any()
    table[1, 0] = 0
    firsts[4] = table.shape[1] * ps
    grout.kv_read_paged_fp8(kp, vp, ksp, vsp, table, ko, vo, ints(cu), ints(firsts))
    with pytest.raises(grout.GroutError, match="0x200"):
        grout.check_device_error()
    assert (ko[cu[4]] == 0).all() and (vo[cu[4]] == 0).all()


def _fp8_pools(lens, hkv, n, ps, window, sinks, seed):
    """Caches [B, Hkv, n, D] with NaN in every row nobody sees, and their pools."""
    B = len(lens)
    (kc, ks), (vc, vs) = (fp8_cache(seed + 2 * i, B, hkv, n, D) for i in range(2))
    for c, s in ((kc, ks), (vc, vs)):
        for b, m in enumerate(lens):
            hide = torch.zeros(n, dtype=torch.bool, device="cuda")
            hide[m:] = True
            if window:
                hide[sinks:max(sinks, m - window)] = True
            c.view(torch.uint8)[b, :, hide] = 0x7F
            s[b, :, hide] = NAN
    pools, table = page_pool([kc.view(torch.uint8), vc.view(torch.uint8), ks, vs], ps, seed, fill=0x7F)
    pools = [p.view(torch.float8_e4m3fn) for p in pools[:2]] + pools[2:]
    if window:
        table = free_pages(table, ps, [m - window for m in lens], sinks)
    for b, m in enumerate(lens):
        table[b, -(-m // ps):] = -1
    return pools, table, values(kc, ks), values(vc, vs)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (10, 2), (8, 1), (7, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (65, 4), (128, 64), (200, 130), (3000, 5)])
@pytest.mark.parametrize("splits", [None, 1, 5, 33])
def test_decode(grout, hq, hkv, window, sinks, splits):
    lens = [1, 2, 63, 64, 65, 128, 129, 191, 640, 1001]
    B, n, ps = len(lens), 1001, 64 if hkv == 2 else 192
    pools, table, k, v = _fp8_pools(lens, hkv, n, ps, window, sinks, 50)
    q = normal(7, B, hq, D, scale=1.5).half()
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
    out = torch.full_like(q, NAN)
    grout.attention_decode_paged_fp8(q, *pools, table, pos, out, n, window, sinks, num_splits=splits)
    torch.cuda.synchronize()
    grout.check_device_error()
    for b in range(B):
        m = lens[b]
        ref, bound = attention64(q[b:b + 1], k[b, :, :m].transpose(0, 1), v[b, :, :m].transpose(0, 1), pos[b:b + 1].long(), window, sinks, SCALE_F16)
        check(out[b:b + 1], ref, bound)


def test_decode_scales_far_apart(grout):
    """Value rows whose scales span f16's whole range, zero rows among them."""
    hq, hkv, n, ps = 8, 1, 512, 64
    pools, table, _, _ = _fp8_pools([n], hkv, n, ps, 0, 0, 70)
    flat = torch.exp2(torch.linspace(-33, 7, n, device="cuda"))[torch.randperm(n, generator=torch.Generator().manual_seed(3)).cuda()]
    flat[::7] = 0.0
    pools[3][table[0].long()] = flat.view(n // ps, 1, ps)
    codes = pools[1].view(torch.uint8)
    for i in range(0, n, 7):
        codes[int(table[0, i // ps]), 0, i % ps] = 0
    k, v = (values(c, s)[table[0].long()].transpose(0, 1).reshape(hkv, n, D) for c, s in ((pools[0], pools[2]), (pools[1], pools[3])))
    for size in (0.01, 3.0):
        q = normal(8, 1, hq, D, scale=size).half()
        out = torch.empty_like(q)
        for splits in (1, 4):
            grout.attention_decode_paged_fp8(q, *pools, table, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), out, n, num_splits=splits)
            torch.cuda.synchronize()
            grout.check_device_error()
            # rounding the folded weights keeps each term's relative error; the 2^-25 floor is relative to the
            # largest term |p v|, which the bound's own floor (largest |v|) covers
            check(out, *attention64(q, k.transpose(0, 1), v.transpose(0, 1), torch.tensor([n - 1], device="cuda"), 0, 0, SCALE_F16))
    pools[3].zero_()  # every value row zero: the output is zero, not NaN
    pools[1].view(torch.uint8).zero_()
    grout.attention_decode_paged_fp8(q, *pools, table, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), out, n)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_decode_nan_is_seen_only_where_visible(grout):
    hq, hkv, n, ps = 8, 2, 300, 64
    pools, table, k, v = _fp8_pools([n], hkv, n, ps, 0, 0, 80)
    q = normal(9, 1, hq, D).half()
    out = torch.empty_like(q)
    pos = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    page, row = int(table[0, 100 // ps]), 100 % ps
    pools[1].view(torch.uint8)[page, 1, row, 17] = 0x7F
    for splits in (1, 3, 20):
        grout.attention_decode_paged_fp8(q, *pools, table, pos, out, n, num_splits=splits)
        assert torch.isnan(out[0, 4:, 17]).all() and torch.isfinite(out[0, :4]).all()
        assert torch.isfinite(out[0, 4:, :17]).all()
    pools[2][page, 1, row] = NAN  # a key: every output of its head
    for splits in (1, 3, 20):
        grout.attention_decode_paged_fp8(q, *pools, table, pos, out, n, num_splits=splits)
        assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all()


def test_serving_run(grout):
    """A prompt in two chunks and then tokens over one 8-bit pool: write, read
    back, windowed attention of the chunk, fused decode write, decode
    attention; the steps recorded in a graph and replayed across pages.  Every
    attention output against 64 bits over the values that the pool stands for."""
    hq, hkv, ps, window, sinks = 16, 2, 64, 200, 4
    per, chunks = 10, [257, 130]
    ms = per * ps
    rope = grout.rope_table(THETA, ms)
    qw, kw = (torch.from_numpy(synth.norm_weight(s, D)).cuda() for s in (4, 5))
    table = torch.randperm(per + 3, generator=torch.Generator().manual_seed(7))[:per].view(1, per).int().cuda()
    pools = _pools(per + 3, hkv, ps)

    def cache(n):
        rows = torch.arange(n, device="cuda")
        at = table[0].long()[rows // ps]
        return [values(c.view(torch.uint8)[at, :, rows % ps].view(torch.float8_e4m3fn), s[at, :, rows % ps]) for c, s in ((pools[0], pools[2]), (pools[1], pools[3]))]

    done = 0
    for i, S in enumerate(chunks):
        q, k, v = (normal(200 + 10 * i + j, S, h, D).half() for j, h in enumerate((hq, hkv, hkv)))
        q_out, out = torch.empty_like(q), torch.empty_like(q)
        grout.qk_norm_rope_kv_prefill_paged_fp8(q, k, v, qw, kw, rope, q_out, *pools, table[0], done, EPS)
        n = done + S
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        ko, vo = (torch.empty(n, hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
        grout.kv_read_paged_fp8(*pools, table, ko, vo, cu)
        grout.attention_prefill_varlen_window(q_out, ko, vo, out, None, S, hkv, hkv * D, D, window, sinks,
                                              position_start=torch.tensor([done], dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        grout.check_device_error()
        ck, cv = cache(n)
        # the rows are read back to f16: half a step relative to each value on both sides
        assert ((ko.double() - ck).abs() <= ck.abs() * 2.0 ** -11 + 2.0 ** -25).all()
        ref, bound = attention64(q_out, ko, vo, done + torch.arange(S, device="cuda"), window, sinks)
        check(out, ref, bound)
        done = n

    qkv = torch.empty(1, (hq + 2 * hkv) * D, dtype=torch.float16, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out, out, full = (torch.empty(1, hq, D, dtype=torch.float16, device="cuda") for _ in range(3))

    def step():
        grout.qk_norm_rope_kv_decode_paged_fp8(qkv, qw, kw, rope, q_out, *pools, table, pos, hq, hkv, EPS)
        grout.attention_decode_paged_fp8(q_out, *pools, table, pos, out, ms, window, sinks)
        grout.attention_decode_paged_fp8(q_out, *pools, table, pos, full, ms)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qkv.copy_(normal(300, *qkv.shape))
        pos.fill_(done)
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(70):  # across a page's end
        qkv.copy_(normal(300 + i, *qkv.shape))
        pos.fill_(done + i)
        g.replay()
        if i % 23 and i != 60:
            continue
        torch.cuda.synchronize()
        grout.check_device_error()
        ck, cv = cache(done + i + 1)
        for o, w, sk in ((out, window, sinks), (full, 0, 0)):
            check(o, *attention64(q_out, ck, cv, pos.long(), w, sk, SCALE_F16))


def test_offsets_past_32_bits(grout):
    """Pools of more than 2^32 bytes of codes: pages at the far end are written (the query rows in place), read back and attended to."""
    hq, hkv, ps, S = 8, 1, 1024, 1500
    pages = 2 ** 32 // (hkv * ps * D) + 4
    pools = [torch.empty(pages, hkv, ps, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv"]
    pools += [torch.empty(pages, hkv, ps, device="cuda") for _ in "kv"]
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    q, k, v = (normal(400 + j, S, h, D).half() for j, h in enumerate((hq, hkv, hkv)))
    w = torch.ones(D, dtype=torch.float16, device="cuda")
    rope = grout.rope_table(THETA, 2 * ps)
    near = [torch.zeros(2, hkv, ps, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv"]
    near += [torch.zeros(2, hkv, ps, device="cuda") for _ in "kv"]
    q_near = torch.empty_like(q)
    grout.qk_norm_rope_kv_prefill_paged_fp8(q, k, v, w, w, rope, q_near, *near, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 0, EPS)
    grout.qk_norm_rope_kv_prefill_paged_fp8(q, k, v, w, w, rope, q, *pools, table[0], 0, EPS)
    cu = torch.tensor([0, S], dtype=torch.int32, device="cuda")
    ko, vo = (torch.empty(S, hkv, D, dtype=torch.float16, device="cuda") for _ in "kv")
    grout.kv_read_paged_fp8(*pools, table, ko, vo, cu)
    out = torch.empty(1, hq, D, dtype=torch.float16, device="cuda")
    pos = torch.tensor([S - 1], dtype=torch.int32, device="cuda")
    grout.attention_decode_paged_fp8(q[-1:], *pools, table, pos, out, S)
    torch.cuda.synchronize()
    grout.check_device_error()
    assert torch.equal(q, q_near)
    ck, cv = (values(c, s).transpose(1, 2).reshape(2 * ps, hkv, D)[:S] for c, s in ((near[0], near[2]), (near[1], near[3])))
    for got, want in ((ko, ck), (vo, cv)):  # f16(code * scale): the product and the result are rounded
        assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all()
    check(out, *attention64(q[-1:], ck, cv, pos.long(), 0, 0, SCALE_F16))


def test_codes_are_those_of_the_formula(grout):
    """V's codes against y * 448 / max|y| in 64 bits, bit for bit: rows that are
    full of ties (the quotient midway between two codes), f16's whole range of
    largest values, signed zeros."""
    hkv, ps, S = 2, 1024, 1024
    g = torch.Generator().manual_seed(9)
    y = torch.randint(-2047, 2048, (S, hkv, D), generator=g).double()
    top = torch.randint(1, 293, (S, hkv, 1), generator=g).double() * 7  # max = 7 t: y = 64 max (odd / 2^n) / 448 = t odd / 2^n is a tie
    odd = torch.randint(1, 32, (S, hkv, D), generator=g).double() * 2 - 1
    tie = odd * (top / 7) / 2.0 ** torch.randint(0, 3, (S, hkv, D), generator=g)
    y = torch.where((torch.arange(S) % 2 == 0)[:, None, None] & (tie.abs() < top) & (tie.half().double() == tie), tie * torch.sign(y + 0.5), y.clamp(-top, top))
    y[:, :, 3] = top[:, :, 0]
    y[5, 0], y[6, 1, ::2] = -0.0, -0.0
    v = (y * 2.0 ** torch.randint(-20, 5, (S, hkv, 1), generator=g)).half().cuda()
    q, w = torch.zeros(S, 1 * hkv, D, dtype=torch.float16, device="cuda"), torch.ones(D, dtype=torch.float16, device="cuda")
    pools, table = _pools(1, hkv, ps), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    grout.qk_norm_rope_kv_prefill_paged_fp8(q, torch.zeros_like(v), v, w, w, grout.rope_table(THETA, ps), torch.empty_like(q), *pools, table[0], 0, EPS)
    torch.cuda.synchronize()
    grout.check_device_error()
    x = v.double()
    m = x.abs().amax(-1, keepdim=True)
    x = torch.where(m <= 2.0 ** -25, x * 0, x * 448 / m)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    ties = ((x / step).abs() % 1 == 0.5).sum().item()
    assert ties > 1000, ties
    want = (torch.round(x / step) * step).float().to(torch.float8_e4m3fn).view(torch.uint8)
    got = pools[1].view(torch.uint8)[0].transpose(0, 1)
    differ = (got != want) & ~((got & 0x7F == 0) & (want & 0x7F == 0))  # (the sign of a code that rounds to zero is torch.round's)
    assert not differ.any(), differ.sum().item()
    assert (got[5, 0] & 0x7F == 0).all() and (got[6, 1, ::2] == 0x80).all()
