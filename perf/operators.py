"""The serving operators next to the paged attention path: an 8-bit KV cache
(quantised as it is written, read back, attended to by single tokens) and
attention with a sliding window and a few first tokens that stay visible
(single tokens and prompt chunks).

`listed()` gives the cases, `run()` one pass of an operator: the plain form in
elementary torch operations, or, with `own` set, this package's kernels.

Definitions (f16 activations, head_dim 128, D = 128):

  write   y = rope(rmsnorm(k) * w) in f32; per cache row (token, KV head)
          scale = max|y| / 448, code = e4m3(y * (448 / max|y|)); V the same
          without norm and rotation; q_out = f16(rope(rmsnorm(q) * w)).
  read    f16(code * scale) of rows position_start[b] .. of each sequence.
  decode  softmax(q . k * qk_scale) v over the keys a query at position p
          sees: n <= p, and with a window also n > p - window or n < sinks.
  prefill the same for every row of a chunk of new tokens.
"""
import math
import random

import torch

own = False

D = 128
EPS = 1e-6
E4M3_MAX = 448.0


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a single user: launch latency
        {"name": "write_step_b1", "op": "write", "batch": 1, "seq": 0, "start": 8191, "hq": 64, "hkv": 8, "page": 64},
        # a 4096-token prompt chunk behind 1001 cached tokens, the Qwen3-32B layer's heads
        {"name": "write_chunk_s4096", "op": "write", "batch": 0, "seq": 4096, "start": 1001, "hq": 64, "hkv": 8, "page": 64},
        # a short history of one KV head (a tensor-parallel shard) read back
        {"name": "read_shard", "op": "read", "batch": 1, "length": 517, "skip": 0, "hkv": 1, "page": 64},
        # sixteen ragged histories read back before a chunk's attention
        {"name": "read_ragged_16", "op": "read", "batch": 16, "length": 8192, "skip": 37, "hkv": 8, "page": 128},
        # one user, long context: the whole 8-bit cache for one token
        {"name": "decode_fp8_b1_l32768", "op": "decode_fp8", "batch": 1, "length": 32768, "window": 0, "sinks": 0, "hq": 64, "hkv": 8, "page": 256},
        # a serving batch of ragged lengths
        {"name": "decode_fp8_b64_l8192", "op": "decode_fp8", "batch": 64, "length": 8192, "window": 0, "sinks": 0, "hq": 32, "hkv": 8, "page": 64},
        # a KV-head shard with a window of odd size over the 8-bit cache
        {"name": "decode_fp8_window_shard", "op": "decode_fp8", "batch": 8, "length": 16384, "window": 2000, "sinks": 4, "hq": 8, "hkv": 1, "page": 64},
        # one user, window of 1024 behind 4 sinks, contiguous cache
        {"name": "decode_window_b1", "op": "decode_window", "batch": 1, "length": 8448, "window": 1024, "sinks": 4, "hq": 64, "hkv": 8, "page": 0},
        # a serving batch, window of 4096, pages outside it already freed
        {"name": "decode_window_b64", "op": "decode_window", "batch": 64, "length": 32768, "window": 4096, "sinks": 64, "hq": 64, "hkv": 8, "page": 128},
        # a whole 8192-token prompt, contiguous cache
        {"name": "prefill_window_s8192", "op": "prefill_window", "batch": 1, "seq": 8192, "start": 0, "window": 1024, "sinks": 4, "hq": 32, "hkv": 8, "page": 0},
        # ragged chunks of several prompts far into their contexts, paged
        {"name": "prefill_window_chunks", "op": "prefill_window", "batch": 6, "seq": 700, "start": 9000, "window": 4096, "sinks": 16, "hq": 64, "hkv": 8, "page": 64},
        # a few tokens each of many sequences (drafted tokens to be verified)
        {"name": "prefill_window_drafts", "op": "prefill_window", "batch": 32, "seq": 5, "start": 4000, "window": 1024, "sinks": 4, "hq": 32, "hkv": 8, "page": 64},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hkv = rng.choice([(64, 8), (32, 8), (16, 8), (8, 1), (16, 2), (6, 2), (5, 1), (8, 8)])
    op = rng.choice(["write", "read", "decode_fp8", "decode_window", "prefill_window"])
    page = rng.choice([64, 128, 192, 256, 1024])
    most = {c["op"]: 0.0 for c in listed()}
    for c in listed():
        most[c["op"]] = max(most[c["op"]], _cost(c))
    while True:
        c = {"op": op, "hq": hq, "hkv": hkv, "page": page}
        if op == "write":
            step = rng.random() < 0.5
            c.update(batch=_log(rng, 1, 256) if step else 0, seq=0 if step else _log(rng, 1, 4096), start=_log(rng, 1, 16384) - 1)
        elif op == "read":
            c.update(batch=_log(rng, 1, 24), length=_log(rng, 1, 8192), skip=rng.choice([0, rng.randrange(500)]))
            c.pop("hq")
        elif op == "decode_fp8":
            w = rng.choice([0, _log(rng, 1, 6000)])
            c.update(batch=_log(rng, 1, 64), length=_log(rng, 1, 32768), window=w, sinks=rng.choice([0, 1, 4, 77]) if w else 0)
        elif op == "decode_window":
            c.update(batch=_log(rng, 1, 64), length=_log(rng, 1, 32768), window=_log(rng, 1, 6000), sinks=rng.choice([0, 1, 4, 64, 130]))
            c["page"] = rng.choice([0, page])
        else:
            c.update(batch=_log(rng, 1, 32), seq=_log(rng, 1, 4096), start=_log(rng, 1, 12000) - 1, window=_log(rng, 1, 6000), sinks=rng.choice([0, 1, 4, 64, 130]))
            c["page"] = rng.choice([0, page])
            if c["batch"] * hq * c["seq"] * (c["start"] + c["seq"]) > 2.2e9:  # the plain form's score matrix
                continue
        if c.get("length", 0) * c.get("batch", 1) * hkv > 64 * 32768 * 2:  # the cache itself
            continue
        if _cost(c) <= most[op]:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


def _lens(case):
    """Context lengths of a batch: the first the longest, the others spread over its upper two thirds, odd ones among them."""
    n, b = case["length"], case["batch"]
    return [max(1, n - (i * 2 * n) // (3 * b)) for i in range(b)]


def _chunks(case):
    """(new tokens, position of the first one) of each sequence of a prefill case."""
    s, p, b = case["seq"], case["start"], case["batch"]
    return [(max(1, s - (i * s) // (2 * b)), p - (i * p) // (3 * b)) for i in range(b)]


def _positions(case):
    """Positions of a decode write's new tokens."""
    return [case["start"] - (i * case["start"]) // (2 * case["batch"]) for i in range(case["batch"])]


# ---------------------------------------------------------------- the work

def _seen(p, window, sinks):
    """How many keys a query at position p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    op = case["op"]
    hkv = case["hkv"]
    if op == "write":
        rows = case["seq"] or case["batch"]
        per = (case["hq"] + 2 * hkv) * D * 2 + case["hq"] * D * 2 + 2 * hkv * (D + 4) + D * 4 + 4
        return {"bytes": rows * per + 4 * D, "flops": rows * (case["hq"] + 2 * hkv) * D * 8}
    if op == "read":
        rows = sum(_lens(case))
        return {"bytes": rows * 2 * hkv * (D + 4 + 2 * D), "flops": rows * 2 * hkv * D}
    hq = case["hq"]
    if op in ("decode_fp8", "decode_window"):
        keys = sum(_seen(n - 1, case["window"], case["sinks"]) for n in _lens(case))
        per = 2 * (D + 4) if op == "decode_fp8" else 4 * D
        return {"bytes": keys * hkv * per + 2 * case["batch"] * hq * D * 2, "flops": 4 * D * hq * keys}
    pairs = keys = rows = 0
    for s, p in _chunks(case):
        w = case["window"]
        pairs += sum(_seen(p + i, w, case["sinks"]) for i in range(s))
        first = max(0, p - w + 1)
        keys += p + s - first + min(case["sinks"], first)
        rows += s
    return {"bytes": 2 * rows * hq * D * 2 + keys * hkv * 4 * D, "flops": 4 * D * hq * pairs}


# -------------------------------------------------------------- the inputs

def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * scale


def _rope_table(n):
    """cos and sin of f32(position) * inv_freq, one f32 row [cos | sin] a position."""
    inv = (1.0 / (1.0e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))).float().cuda()
    angle = (torch.arange(n, device="cuda").float()[:, None] * inv[None]).double()
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _table(g, firsts, lens, page, live=None):
    """A page table over a shuffled pool: sequence b holds the pages of positions 0 .. lens[b]-1, those that `live` drops
    freed (-1).  Returns (table, pages in the pool)."""
    width = -(-max(lens) // page)
    at = torch.arange(width, device="cuda")[None]
    held = at < torch.tensor([-(-n // page) for n in lens], device="cuda")[:, None]
    if live is not None:
        window, sinks = live
        low = torch.tensor([max(0, f - window + 1) for f in firsts], device="cuda")[:, None]
        held &= ((at + 1) * page > low) | (at * page < sinks)
    n = int(held.sum())
    table = torch.full(held.shape, -1, dtype=torch.int32, device="cuda")
    table[held] = torch.randperm(n, device="cuda", generator=g).int()
    return table, n


def _codes(g, pages, hkv, page):
    """A pool of 8-bit rows with their scales, as a model's keys or values leave them: rows of unlike size."""
    y = _normal(g, pages, hkv, page, D) * torch.exp(_normal(g, pages, hkv, page, 1, scale=0.3))
    top = y.abs().amax(-1, keepdim=True)
    return (y * (E4M3_MAX / top)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), (top / E4M3_MAX)[..., 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    op, hkv, page = case["op"], case["hkv"], case["page"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if op == "write":
        hq = case["hq"]
        last = max(_positions(case)) if case["batch"] else case["start"] + case["seq"] - 1
        st["rope"] = _rope_table(page * (last // page + 1))
        rows = case["batch"] or case["seq"]
        lens = [p + 1 for p in _positions(case)] if case["batch"] else [last + 1]
        # of the pages a sequence holds only those that this call writes are kept in the pool
        st["table"], n = _table(g, [p for p in _positions(case)] if case["batch"] else [case["start"]], lens, page, live=(1, 0))
        for name in ("k", "v"):
            st[name + "_pages"] = torch.zeros(n, hkv, page, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
            st[name + "_scales"] = torch.zeros(n, hkv, page, device="cuda")
        st["qw"], st["kw"] = ((1 + _normal(g, D, scale=0.1)).half() for _ in range(2))
        size = torch.exp(_normal(g, rows, 1, 1, scale=0.5))  # tokens differ in size
        q, k, v = ((_normal(g, rows, h, D) * size).half() for h in (hq, hkv, hkv))
        st["q_out"] = torch.empty(rows, hq, D, dtype=torch.float16, device="cuda")
        if case["batch"]:
            st["qkv"] = torch.cat([q, k, v], 1).reshape(rows, -1).contiguous()
            st["position"] = ints(_positions(case))
        else:
            st["q"], st["k"], st["v"] = q, k, v
        return st
    if op == "read":
        lens = [n + case["skip"] for n in _lens(case)]
        st["table"], n = _table(g, lens, lens, page)
        st["k_pages"], st["k_scales"] = _codes(g, n, hkv, page)
        st["v_pages"], st["v_scales"] = _codes(g, n, hkv, page)
        st["cu"] = ints([0] + torch.tensor(_lens(case)).cumsum(0).tolist())
        st["first"] = ints([case["skip"]] * case["batch"])
        st["rows"] = sum(_lens(case))
        st["k_out"], st["v_out"] = (torch.empty(st["rows"], hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
        return st
    hq = case["hq"]
    if op == "prefill_window":
        chunks = _chunks(case)
        lens, firsts = [s + p for s, p in chunks], [p for _, p in chunks]
        rows = sum(s for s, _ in chunks)
        st["q"] = _normal(g, rows, hq, D, scale=1.5).half()
        st["cu"] = ints([0] + torch.tensor([s for s, _ in chunks]).cumsum(0).tolist())
        st["start_at"] = ints(firsts)
        st["most"] = max(s for s, _ in chunks)
    else:
        lens = _lens(case)
        firsts = [n - 1 for n in lens]
        st["q"] = _normal(g, case["batch"], hq, D, scale=1.5).half()
        st["position"] = ints(firsts)
    st["longest"] = max(lens)
    st["out"] = torch.empty_like(st["q"])
    if page:
        live = (case["window"], case["sinks"]) if case["window"] else None
        st["table"], n = _table(g, firsts, lens, page, live)
        if op == "decode_fp8":
            st["k_pages"], st["k_scales"] = _codes(g, n, hkv, page)
            st["v_pages"], st["v_scales"] = _codes(g, n, hkv, page)
        else:
            st["k_pages"], st["v_pages"] = (_normal(g, n, hkv, page, D).half() for _ in range(2))
    else:
        st["k_cache"], st["v_cache"] = (_normal(g, case["batch"], hkv, st["longest"], D).half() for _ in range(2))
    return st


# ------------------------------------------------------------------ the pass

def run(st):
    if own:
        return _own(st)
    return {"write": _plain_write, "read": _plain_read, "decode_fp8": _plain_decode, "decode_window": _plain_decode, "prefill_window": _plain_prefill}[st["op"]](st)


def _own(st):
    import grout_b200 as g
    op = st["op"]
    if op == "write":
        if st["batch"]:
            g.qk_norm_rope_kv_decode_paged_fp8(st["qkv"], st["qw"], st["kw"], st["rope"], st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"],
                                               st["v_scales"], st["table"], st["position"], st["hq"], st["hkv"], EPS)
        else:
            g.qk_norm_rope_kv_prefill_paged_fp8(st["q"], st["k"], st["v"], st["qw"], st["kw"], st["rope"], st["q_out"], st["k_pages"], st["v_pages"],
                                                st["k_scales"], st["v_scales"], st["table"][0], st["start"], EPS)
        return [st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]]
    if op == "read":
        g.kv_read_paged_fp8(st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"], st["table"], st["k_out"], st["v_out"], st["cu"],
                            position_start=st["first"])
        return [st["k_out"], st["v_out"]]
    w, s = st["window"], st["sinks"]
    if op == "decode_fp8":
        g.attention_decode_paged_fp8(st["q"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"], st["table"], st["position"], st["out"],
                                     st["longest"], window=w, sinks=s)
    elif op == "decode_window" and st["page"]:
        g.attention_decode_paged_window(st["q"], st["k_pages"], st["v_pages"], st["table"], st["position"], st["out"], st["longest"], w, s)
    elif op == "decode_window":
        g.attention_decode_window(st["q"], st["k_cache"], st["v_cache"], st["position"], st["out"], st["longest"], w, s)
    elif st["page"]:
        g.attention_prefill_paged_window(st["q"], st["k_pages"], st["v_pages"], st["table"], st["out"], w, s, cu_seqlens_q=st["cu"],
                                         position_start=st["start_at"], max_q_len=st["most"])
    else:
        n, hkv = st["longest"], st["hkv"]
        g.attention_prefill_varlen_window(st["q"], st["k_cache"], st["v_cache"], st["out"], st["cu"], st["most"], hkv, D, n * D, w, s,
                                          kv_batch_stride=hkv * n * D, kv_rows=n, position_start=st["start_at"])
    return st["out"]


def _plain_norm_rope(x, w, rope):
    """[rows, heads, 128] f16 -> f32: RMS norm (the squares summed in the cache's order, so that values next to a border fall on
    the same side), weight, rotation by the table's rows."""
    x = x.float()
    lo, hi = x[..., :64], x[..., 64:]
    t = (lo * lo + hi * hi).reshape(*x.shape[:-1], 8, 8)
    s = ((t[..., 0] + t[..., 1]) + (t[..., 2] + t[..., 3])) + ((t[..., 4] + t[..., 5]) + (t[..., 6] + t[..., 7]))
    s = s[..., :4] + s[..., 4:]
    s = s[..., :2] + s[..., 2:]
    s = s[..., :1] + s[..., 1:]
    inv = 1.0 / torch.sqrt(s * 0.0078125 + EPS)
    n = (x * inv) * w.float()
    lo, hi = n[..., :64], n[..., 64:]
    cos, sin = rope[:, None, :64], rope[:, None, 64:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_write(st):
    hq, hkv = st["hq"], st["hkv"]
    if st["batch"]:
        x = st["qkv"].view(st["batch"], hq + 2 * hkv, D)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        pos = st["position"].long()
        pages = torch.gather(st["table"], 1, (pos // st["page"])[:, None])[:, 0].long()
    else:
        q, k, v = st["q"], st["k"], st["v"]
        pos = st["start"] + torch.arange(st["seq"], device="cuda")
        pages = st["table"][0][pos // st["page"]].long()
    rope = st["rope"][pos]
    st["q_out"].copy_(_plain_norm_rope(q, st["qw"], rope))
    at = pos % st["page"]
    for name, y in (("k", _plain_norm_rope(k, st["kw"], rope)), ("v", v.float())):
        top = y.abs().amax(-1, keepdim=True)
        code = (y * (E4M3_MAX / top)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        st[name + "_pages"].view(torch.uint8)[pages, :, at] = code.view(torch.uint8)
        st[name + "_scales"][pages, :, at] = (top / E4M3_MAX)[..., 0]
    return [st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]]


def _rows_of(st, name, pages, at):
    """f32 cache rows [..., hkv, 128] at (page, row in page)."""
    if st["op"] == "decode_window" or st["op"] == "prefill_window":
        return st[name + "_pages"][pages, :, at].float()
    return st[name + "_pages"].view(torch.uint8)[pages, :, at].view(torch.float8_e4m3fn).float() * st[name + "_scales"][pages, :, at][..., None]


def _plain_read(st):
    row = torch.arange(st["rows"], device="cuda")
    b = torch.searchsorted(st["cu"].long(), row, right=True) - 1
    pos = st["first"].long()[b] + row - st["cu"].long()[b]
    pages = st["table"][b, pos // st["page"]].long()
    for name in ("k", "v"):
        st[name + "_out"].copy_(_rows_of(st, name, pages, pos % st["page"]))
    return [st["k_out"], st["v_out"]]


def _cache(st, pos):
    """f32 keys and values [batch, n, hkv, 128] at positions pos [batch, n]."""
    if st["page"]:
        pages = torch.gather(st["table"], 1, pos // st["page"]).clamp(min=0).long()
        return tuple(_rows_of(st, name, pages, pos % st["page"]) for name in ("k", "v"))
    at = pos[:, None, :, None].expand(-1, st["hkv"], -1, D)
    return tuple(torch.gather(st[name + "_cache"], 2, at).float().transpose(1, 2) for name in ("k", "v"))


def _plain_decode(st):
    B, hq, hkv = st["batch"], st["hq"], st["hkv"]
    n = st["position"].long()[:, None] + 1
    if st["window"]:  # the sinks, then the window: each key once
        first = torch.arange(st["sinks"], device="cuda")[None].expand(B, -1)
        last = n - st["window"] + torch.arange(st["window"], device="cuda")[None]
        pos = torch.cat([first, last], 1)
        seen = torch.cat([first < n, last >= st["sinks"]], 1) & (pos >= 0)
    else:
        pos = torch.arange(st["longest"], device="cuda")[None].expand(B, -1)
        seen = pos < n
    k, v = _cache(st, pos.clamp(min=0, max=st["longest"] - 1))
    scale = torch.tensor(1.0 / math.sqrt(D)).half().float().item()  # the decode path's softmax scale is an f16 value
    s = torch.einsum("bhgd,bnhd->bhgn", st["q"].float().view(B, hkv, hq // hkv, D), k) * scale
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.einsum("bhgn,bnhd->bhgd", p, v) / p.sum(-1, keepdim=True)
    st["out"].copy_(o.reshape(B, hq, D))
    return st["out"]


def _plain_prefill(st):
    B, hq, hkv, most = st["batch"], st["hq"], st["hkv"], st["most"]
    cu, start = st["cu"].long(), st["start_at"].long()
    row = cu[:-1, None] + torch.arange(most, device="cuda")[None]
    there = row < cu[1:, None]
    q = st["q"][row.clamp(max=st["q"].shape[0] - 1)].float().view(B, most, hkv, hq // hkv, D)
    # the keys that the batch's rows see: the sinks, then from the first window's first key on
    low = (start - st["window"] + 1).clamp(min=0)
    span = int(st["longest"]) if st["window"] >= st["longest"] else min(st["longest"], st["window"] - 1 + most)
    pos = torch.cat([torch.arange(st["sinks"], device="cuda")[None].expand(B, -1), low[:, None] + torch.arange(span, device="cuda")[None]], 1)
    once = torch.arange(pos.shape[1], device="cuda")[None] >= st["sinks"]
    once = (pos >= st["sinks"]) == once  # each key once
    k, v = _cache(st, pos.clamp(max=st["longest"] - 1))
    at = (start[:, None] + torch.arange(most, device="cuda")[None])[:, :, None]
    key = pos[:, None]
    seen = (key <= at) & ((key > at - st["window"]) | (key < st["sinks"])) & once[:, None]
    s = torch.einsum("bmhgd,bnhd->bhgmn", q, k) * (1.0 / math.sqrt(D))
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.einsum("bhgmn,bnhd->bmhgd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    st["out"][row[there]] = o.reshape(B, most, hq, D)[there].half()
    return st["out"]


# --------------------------------------------------- the definition in 64 bits

def _exact_code(y):
    """y [..., 128] in 64 bits -> (e4m3 value of y * 448 / max|y|, max|y| / 448)."""
    top = y.abs().max(-1).values
    x = y * (E4M3_MAX / top)[..., None]
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return torch.round(x / step) * step, top / E4M3_MAX


def _exact_attention(q, k, v, pos, window, sinks, scale):
    """q [m, hq, 128], keys k, v [n, hkv, 128] of positions 0 .., query rows at pos [m]."""
    key = torch.arange(k.shape[0], device="cuda")
    seen = key[None] <= pos[:, None]
    if window:
        seen &= (key[None] > pos[:, None] - window) | (key[None] < sinks)
    outs = []
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ k[:, h // group].double().T) * scale
        s[~seen] = -math.inf
        outs.append(torch.softmax(s, -1) @ v[:, h // group].double())
    return torch.stack(outs, 1)


def exact(case, seed):
    st = prepare(case, seed)
    op, page = case["op"], case["page"]
    if op == "write":
        hq, hkv = case["hq"], case["hkv"]
        if case["batch"]:
            q, k, v = st["qkv"].double().view(-1, hq + 2 * hkv, D).split([hq, hkv, hkv], 1)
            where = [(b, p) for b, p in enumerate(_positions(case))]
        else:
            q, k, v = (st[x].double() for x in "qkv")
            where = [(0, case["start"] + i) for i in range(case["seq"])]
        angles = st["rope"].double()[torch.tensor([p for _, p in where], device="cuda")]
        turn = torch.complex(angles[:, :64], angles[:, 64:])[:, None]

        def rotate(x, w):
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        table = st["table"].cpu()
        page_at = torch.tensor([int(table[b, p // page]) for b, p in where], device="cuda")
        row_at = torch.tensor([p % page for _, p in where], device="cuda")
        outs = [rotate(q, st["qw"])]
        pools, scales = [], []
        for y in (rotate(k, st["kw"]), v):
            code, scale = _exact_code(y)
            pool = torch.zeros(st["k_pages"].shape, dtype=torch.float64, device="cuda")
            pool[page_at, :, row_at] = code
            pools.append(pool)
            scales.append(torch.zeros(pool.shape[:3], dtype=torch.float64, device="cuda"))
            scales[-1][page_at, :, row_at] = scale
        return outs + pools + scales
    if op == "read":
        outs = {"k": [], "v": []}
        for b, n in enumerate(_lens(case)):
            for name, to in outs.items():
                got = _exact_pages(st, name, b, case["skip"] + n)
                to.append(got[case["skip"]:])
        return [torch.cat(outs["k"]), torch.cat(outs["v"])]
    outs = []
    scale = 1.0 / math.sqrt(D)
    if op == "prefill_window":
        row = 0
        for b, (m, p) in enumerate(_chunks(case)):
            k, v = (_exact_pages(st, name, b, p + m) for name in ("k", "v"))
            outs.append(_exact_attention(st["q"][row:row + m], k, v, p + torch.arange(m, device="cuda"), case["window"], case["sinks"], scale))
            row += m
        return torch.cat(outs)
    scale = float(torch.tensor(scale).half())
    for b, n in enumerate(_lens(case)):
        k, v = (_exact_pages(st, name, b, n) for name in ("k", "v"))
        outs.append(_exact_attention(st["q"][b:b + 1], k, v, torch.tensor([n - 1], device="cuda"), case["window"], case["sinks"], scale))
    return torch.cat(outs)


def _exact_pages(st, name, b, n):
    """Rows 0 .. n-1 of a sequence's cache in 64 bits, [n, hkv, 128]; zeros where a page was freed."""
    if not st["page"]:
        return st[name + "_cache"][b, :, :n].transpose(0, 1).double()
    rows = []
    for i, at in enumerate(st["table"][b, :-(-n // st["page"])].tolist()):
        if at < 0:
            rows.append(torch.zeros(st["page"], st["hkv"], D, dtype=torch.float64, device="cuda"))
            continue
        x = st[name + "_pages"][at].to(torch.float64) if st["op"] not in ("read", "decode_fp8") else st[name + "_pages"][at].float().double() * st[name + "_scales"][at].double()[..., None]
        rows.append(x.transpose(0, 1))
    return torch.cat(rows)[:n]


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
