"""What is measured of the paged key/value cache in 8 bits and the attention over it.

Three operators of the library (include/vnpu_b200.h): PAGED_KV_APPEND rotates the new tokens'
queries and keys and appends keys and values to the cache, PAGED_KV_READ gives cached tokens back
as values, PAGED_ATTENTION attends to the cache.  The cache holds int8 codes with one f32 scale
for each page of tokens and head, [pages][heads][page_size][head_dim] and [pages][heads].

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or, where
`own` is true, through the library's command stream.
"""
import ctypes
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def _case(name, op, dtype, batch, q_heads, kv_heads, head_dim, page, new, length, ragged=False,
          causal=True, window=0, interleaved=False):
    """new: the longest run of new tokens of a sequence; length: its longest cache after them."""
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "new": new,
            "length": length, "ragged": ragged, "causal": causal, "window": window,
            "interleaved": interleaved}


def listed():
    return [
        # One user's next token in the decoder block's shape (32 heads of 128, f32 activations):
        # latency is all there is.
        _case("append_one_f32", "append", "f32", 1, 32, 32, 128, 64, 1, 513),
        # A serving step's next tokens, one for each of 64 users, grouped heads.
        _case("append_decode64_bf16", "append", "bf16", 64, 32, 8, 128, 64, 1, 4096, ragged=True),
        # Prompts of uneven lengths entering the cache together.
        _case("append_prompts_bf16", "append", "bf16", 16, 32, 8, 128, 64, 1024, 1024, ragged=True),
        # A cached prefix of the block's prefill length taken out in f32 for ATTENTION_F32.
        _case("read_prefix_f32", "read", "f32", 1, 32, 32, 128, 64, 512, 512),
        # Many users' caches moved out together, heads of 64, small pages.
        _case("read_ragged_f16", "read", "f16", 24, 16, 8, 64, 16, 2000, 2000, ragged=True),
        # One user's decode step in the block's shape: 640 slots, all heads their own keys.
        _case("attend_one_f32", "attend", "f32", 1, 32, 32, 128, 64, 1, 640),
        # A serving step: 64 users, one token each, caches of uneven lengths.
        _case("attend_decode64_bf16", "attend", "bf16", 64, 32, 8, 128, 64, 1, 4096, ragged=True),
        # Two users with very long caches: few rows, the work has to be split over the keys.
        _case("attend_long_bf16", "attend", "bf16", 2, 32, 8, 128, 64, 1, 131072),
        # Verification of five drafted tokens at once for 16 users, small pages, a window.
        _case("attend_verify_f16", "attend", "f16", 16, 32, 8, 64, 16, 5, 2047, ragged=True,
              window=1024),
        # The block's prefill: 512 tokens, 32 heads, f32 in and out.
        _case("attend_prefill_f32", "attend", "f32", 1, 32, 32, 128, 64, 512, 512),
        # Prompts of uneven lengths, some with a cached prefix before them.
        _case("attend_prompts_bf16", "attend", "bf16", 8, 32, 8, 128, 64, 1500, 2500, ragged=True),
        # A chunk of a long prompt over what is cached already: the largest.
        _case("attend_chunk_bf16", "attend", "bf16", 1, 32, 8, 128, 128, 2048, 32768),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; its cost is held below the largest listed one's."""
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    head_dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    group = rng.choice([g for g in (1, 2, 4, 4, 5, 8) if g * kv_heads <= 64])
    batch = _log(rng, 1, 96)
    length = _log(rng, 1, 65536)
    # what the plain form gathers in 32 bits, and the cache itself, stay below 2 GB
    length = max(1, min(length, 4_000_000 * 128 // (batch * kv_heads * head_dim)))
    new = 1 if op != "read" and rng.random() < 0.5 else _log(rng, 1, 4096)
    new = min(new, length)
    if op == "attend":  # scores of at most 8 GB, and half the largest listed case's products
        new = max(1, min(new, 2_000_000_000 // (batch * kv_heads * group * length),
                         300_000_000_000 // (batch * kv_heads * group * length * head_dim)))
    else:  # at most 256 MB of rows in 32 bits
        new = max(1, min(new, 64_000_000 // (batch * (group + 2) * kv_heads * head_dim)))
    return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "batch": batch,
            "q_heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": rng.choice([16, 32, 64, 64, 128]), "new": new, "length": length,
            "ragged": rng.random() < 0.7, "causal": op != "attend" or rng.random() < 0.8,
            "window": _log(rng, 16, 4096) if op == "attend" and rng.random() < 0.2 else 0,
            "interleaved": op == "append" and rng.random() < 0.3}


def _spans(case):
    """(new tokens, cache length after them) of each sequence: the case's own, whatever the seed."""
    spans = []
    for b in range(case["batch"]):
        if not case["ragged"] or b == 0:
            spans.append((case["new"], case["length"]))
            continue
        length = max(1, round(case["length"] * (0.1 + 0.9 * (b * 0.6180339887 % 1))))
        new = max(1, round(case["new"] * (0.1 + 0.9 * (b * 0.7548776662 % 1))))
        spans.append((min(new, length), length))
    return spans


def _first_read(case, new, length):
    """Where an append's read-back starts: the first slot of the first page that it writes to."""
    return (length - new) // case["page"] * case["page"]


def work(case):
    wide = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    hq, hk, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    spans = _spans(case)
    tokens = sum(n for n, _ in spans)
    pages = sum(-(-length // ps) for _, length in spans)
    if case["op"] == "append":
        touched = sum(-(-length // ps) - (length - n) // ps for n, length in spans)
        values = sum(length - _first_read(case, n, length) for n, length in spans)
        # q, k, v in; q out; codes and scales written; the written pages' values out in 16 bits
        nbytes = tokens * (2 * hq + 2 * hk) * d * wide + 2 * tokens * hk * d
        nbytes += 2 * 2 * touched * hk * 4 + 2 * values * hk * d * 2 + 4 * touched
        return {"bytes": nbytes, "flops": tokens * (hq + hk) * d * 3 + 4 * tokens * hk * d}
    if case["op"] == "read":
        return {"bytes": 2 * tokens * hk * d * (1 + wide) + 2 * pages * hk * 4 + 4 * pages,
                "flops": 2 * tokens * hk * d}
    pairs, keys = 0, 0
    for n, length in spans:
        first = length - n  # position of the first query
        low = 0 if not case["window"] else max(0, first - case["window"] + 1)
        keys += length - low
        if not case["causal"] and not case["window"]:
            pairs += n * length
            continue
        for pos in range(first, length):
            hi = pos + 1 if case["causal"] else length
            lo = max(0, pos - case["window"] + 1) if case["window"] else 0
            pairs += hi - lo
    return {"bytes": 2 * tokens * hq * d * wide + 2 * keys * hk * d +
            2 * 4 * hk * -(-keys // ps) + 4 * -(-keys // ps),
            "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    spans = _spans(case)
    tokens = sum(n for n, _ in spans)
    per_seq = [-(-length // ps) for _, length in spans]
    pages = sum(per_seq) + 3  # a pool has pages of others, too
    # pages of a sequence lie anywhere in the pool
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((case["batch"], max(per_seq)), -1, dtype=torch.int32, device=dev)
    width = torch.tensor(per_seq, device=dev)[:, None]
    used = torch.arange(max(per_seq), device=dev)[None, :] < width
    table[used] = order[: sum(per_seq)]
    cu, cu_read = [0], [0]
    for n, length in spans:
        cu.append(cu[-1] + n)
        cu_read.append(cu_read[-1] + length - _first_read(case, n, length))
    # keys and values of unit size, as norms before the projections give them: the largest of a
    # page's codes is near 127, so the scales are near 1/40, uneven from page to page
    def codes():
        c = torch.empty((pages, hk, ps, d), dtype=torch.int8, device=dev)
        step = max(1, (1 << 27) // (hk * ps * d))
        for i in range(0, pages, step):
            part = c[i:i + step]
            part.copy_(torch.randn(part.shape, generator=g, device=dev).mul_(38).round_().clamp_(-127, 127))
        return c

    def scales():
        return torch.rand((pages, hk), generator=g, device=dev).mul_(0.02).add_(0.015)

    s = {"case": case, "tokens": tokens, "k": codes(), "v": codes(), "ks": scales(), "vs": scales(),
         "table": table, "lens": torch.tensor([x for _, x in spans], dtype=torch.int32, device=dev),
         "cu": torch.tensor(cu, dtype=torch.int32, device=dev),
         "max_new": max(n for n, _ in spans), "max_len": max(x for _, x in spans)}
    if case["op"] == "attend":
        s["q"] = torch.randn((tokens, hq, d), generator=g, device=dev).to(dt)
    elif case["op"] == "append":
        # one projection's output, its rows [Q | K | V]: the operator reads the parts in place
        s["qkv"] = torch.randn((tokens, (hq + 2 * hk) * d), generator=g, device=dev).to(dt)
        s["cu_read"] = torch.tensor(cu_read, dtype=torch.int32, device=dev)
        s["read_tokens"] = cu_read[-1]
        s["max_read"] = max(cu_read[i + 1] - cu_read[i] for i in range(case["batch"]))
    return s


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------
def _places(s, cu, tokens):
    """Each row's sequence and position, and the page and slot of that position."""
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = s["lens"][seq] - cu[1:][seq] + t
    ps = s["case"]["page"]
    return seq, pos.long(), s["table"][seq, (pos // ps).long()].long(), (pos % ps).long()


def _turns(pos, d):
    """cos and sin of the positions' angles, [rows][d / 2].  An angle is a whole number of 2^-64
    turns times the position, modulo 2^64, so it is as exact at position 100000 as at 1."""
    turn = [int(10000.0 ** (-2.0 * j / d) / (2 * math.pi) * 2.0 ** 64) for j in range(d // 2)]
    turn = torch.tensor([x - (1 << 64) if x >= 1 << 63 else x for x in turn], device="cuda")
    angle = (pos[:, None] * turn[None, :]).float() * (2.0 * math.pi / 2.0 ** 64)
    return torch.cos(angle), torch.sin(angle)


def _rotate(x, cos, sin, interleaved):
    """x: [rows][heads][d] in 32 bits."""
    cos, sin = cos[:, None, :], sin[:, None, :]
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y = torch.empty_like(x)
    ya, yb = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :half], y[..., half:])
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    return y


def _plain_append(s):
    c = s["case"]
    hq, hk, d, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    _, pos, page, slot = _places(s, s["cu"], s["tokens"])
    x = s["qkv"].float().view(s["tokens"], hq + 2 * hk, d)
    cos, sin = _turns(pos, d)
    q = _rotate(x[:, :hq], cos, sin, c["interleaved"])
    new = {"k": _rotate(x[:, hq:hq + hk], cos, sin, c["interleaved"]), "v": x[:, hq + hk:]}
    # the first slot that the new tokens take in a page: tokens before it stay
    first = torch.full((s["k"].shape[0],), ps, device="cuda").scatter_reduce(0, page, slot, "amin")
    head_page = s["table"][torch.arange(c["batch"], device="cuda"),
                           ((s["lens"] - s["cu"].diff()) // ps).long()].long()
    stays = torch.arange(ps, device="cuda")[None, :] < first[head_page][:, None]

    def put(x, codes, scale):
        most = torch.zeros_like(scale).scatter_reduce(
            0, page[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
        old = torch.where(first[:, None] > 0, scale, torch.zeros_like(scale))
        now = torch.where(first[:, None] < ps, torch.maximum(old, most / 127.0), scale)
        ratio = torch.where(now > 0, old / now, torch.zeros_like(now))[head_page]
        held = codes[head_page].float()
        held = torch.where(stays[:, None, :, None], torch.round(held * ratio[:, :, None, None]), held)
        codes[head_page] = held.to(torch.int8)
        per = now[page][:, :, None]
        code = torch.where(per > 0, torch.round(x / per), torch.zeros_like(x)).clamp(-127, 127)
        codes[page, :, slot] = code.to(torch.int8)
        scale.copy_(now)

    put(new["k"], s["k"], s["ks"])
    put(new["v"], s["v"], s["vs"])
    k, v = _plain_read(s, s["cu_read"], s["read_tokens"], _value_type(c))
    return {"q": q.to(DTYPES[c["dtype"]]), "k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}


def _value_type(case):
    """What an append's written pages are read back in: 16 bits hold 8-bit values well."""
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _plain_read(s, cu, tokens, dt):
    _, _, page, slot = _places(s, cu, tokens)
    return [(codes[page, :, slot].float() * scale[page][:, :, None]).to(dt)
            for codes, scale in ((s["k"], s["ks"]), (s["v"], s["vs"]))]


def _plain_attend(s):
    c = s["case"]
    hq, hk, d, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    n, length, batch = s["max_new"], s["max_len"], c["batch"]
    at = torch.arange(length, device="cuda")
    page = s["table"][:, at // ps].long().clamp(min=0)  # [batch][length]
    k = s["k"][page, :, (at % ps)[None, :]].float() * s["ks"][page][..., None]
    k = k.permute(0, 2, 3, 1)  # [batch][kv_heads][d][length]
    row = torch.arange(n, device="cuda")
    count = s["cu"].diff()
    real = row[None, :] < count[:, None]
    where = (s["cu"][:-1, None] + row[None, :]).clamp(max=s["tokens"] - 1).long()
    pos = s["lens"][:, None] - count[:, None] + row[None, :]  # [batch][n]
    q = s["q"].float()[where].view(batch, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, hk, -1, d)  # rows: head of the group, token
    score = torch.matmul(q, k).view(batch, hk, hq // hk, n, length)
    del k
    score.mul_(1.0 / math.sqrt(d))
    seen = at[None, None, :] < s["lens"][:, None, None]
    if c["causal"]:
        seen = seen & (at[None, None, :] <= pos[:, :, None])
    if c["window"]:
        seen = seen & (at[None, None, :] > pos[:, :, None] - c["window"])
    score.masked_fill_(~seen.expand(batch, n, length)[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    most = torch.where(torch.isinf(most), torch.zeros_like(most), most)
    p = score.sub_(most).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v"][page, :, (at % ps)[None, :]].float() * s["vs"][page][..., None]
    o = torch.matmul(p.view(batch, hk, -1, length), v.permute(0, 2, 1, 3))
    o = o.view(batch, hk, hq // hk, n, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, n, hq, d)
    return o[real].to(DTYPES[c["dtype"]])


# ---------------------------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------------------------
_device = None


def _library():
    global _device
    if _device is None:
        path = os.path.join(os.getcwd(), "npuxl-improved_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import vnpu

        _device = (vnpu, vnpu.Device(vnpu.Lib(vnpu.LIB_PATH)))
    return _device


def _own_plan(s):
    """The command packets of a state and its output buffers, as a serving loop keeps them: what
    changes between its steps (lengths, pages, rows) is in device memory."""
    vnpu, dev = _library()
    c = s["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    kind = {"f32": vnpu.DTYPE_F32, "f16": vnpu.DTYPE_F16, "bf16": vnpu.DTYPE_BF16}
    cache = vnpu.paged_cache(s["k"], s["v"], s["ks"], s["vs"])
    batch = vnpu.paged_batch(s["table"], s["cu"], s["lens"], s["tokens"], s["max_new"])
    rows = lambda n, heads, dt: torch.empty((n, heads, d), dtype=dt, device="cuda")  # noqa: E731
    if c["op"] == "append":
        parts = s["qkv"].split([hq * d, hk * d, hk * d], dim=1)
        q = rows(s["tokens"], hq, DTYPES[c["dtype"]])
        dt = _value_type(c)
        k, v = rows(s["read_tokens"], hk, dt), rows(s["read_tokens"], hk, dt)
        back = vnpu.paged_batch(s["table"], s["cu_read"], s["lens"], s["read_tokens"], s["max_read"])
        cmds = [vnpu.paged_kv_append_cmd(cache, batch, *parts, q, q_heads=hq,
                                         interleaved=c["interleaved"]),
                vnpu.paged_kv_read_cmd(cache, back, k, v)]
        out = {"q": q, "k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}
    elif c["op"] == "read":
        k, v = rows(s["tokens"], hk, DTYPES[c["dtype"]]), rows(s["tokens"], hk, DTYPES[c["dtype"]])
        cmds = [vnpu.paged_kv_read_cmd(cache, batch, k, v)]
        out = [k, v]
    else:
        out = rows(s["tokens"], hq, DTYPES[c["dtype"]])
        cmds = [vnpu.paged_attention_cmd(cache, batch, s["q"], out, causal=c["causal"],
                                         window=c["window"], max_length=s["max_len"])]
    return (vnpu.Command * len(cmds))(*cmds), out


def _own_run(s):
    if "plan" not in s:
        s["plan"] = _own_plan(s)
    _, dev = _library()
    cmds, out = s["plan"]
    dev.lib.check(dev.lib.stream_submit(dev.stream, cmds, len(cmds), None), "stream_submit")
    return out


def run(state):
    if own:
        return _own_run(state)
    c = state["case"]
    if c["op"] == "append":
        return _plain_append(state)
    if c["op"] == "read":
        return _plain_read(state, state["cu"], state["tokens"], DTYPES[c["dtype"]])
    return _plain_attend(state)


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _cached(s, which, b, upto):
    """A sequence's codes [tokens][heads][d] and their scales [tokens][heads] in 64 bits."""
    ps = s["case"]["page"]
    pages = s["table"][b, : -(-upto // ps)].long()
    codes = s[which][pages].double().transpose(1, 2).flatten(0, 1)[:upto]
    return codes, s[which + "s"][pages].double().repeat_interleave(ps, 0)[:upto]


def exact(case, seed):
    s = prepare(case, seed)
    hq, hk, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    spans = _spans(case)
    if case["op"] == "read":
        out = []
        for which in ("k", "v"):
            parts = []
            for b, (n, length) in enumerate(spans):
                codes, scale = _cached(s, which, b, length)
                parts.append((codes * scale[:, :, None])[length - n:])
            out.append(torch.cat(parts))
        return out
    if case["op"] == "attend":
        out, row = [], 0
        for b, (n, length) in enumerate(spans):
            k, ks = _cached(s, "k", b, length)
            v, vs = _cached(s, "v", b, length)
            at = torch.arange(length, device="cuda")
            o = torch.empty((n, hq, d), dtype=torch.float64, device="cuda")
            for h in range(hq):
                kv = h // (hq // hk)
                for i in range(0, n, 1024):
                    pos = torch.arange(length - n + i, length - n + min(n, i + 1024), device="cuda")[:, None]
                    q = s["q"][row + i:row + i + len(pos), h].double()
                    x = (q @ (k[:, kv] * ks[:, kv, None]).T) / math.sqrt(d)
                    if case["causal"]:
                        x[at[None, :] > pos] = -math.inf
                    if case["window"]:
                        x[at[None, :] <= pos - case["window"]] = -math.inf
                    w = torch.softmax(x, -1)
                    o[i:i + len(pos), h] = w @ (v[:, kv] * vs[:, kv, None])
            out.append(o)
            row += n
        return torch.cat(out)
    out = {"q": [], "k": [], "v": []}
    scales = {"k": s["ks"].double(), "v": s["vs"].double()}
    freq = 10000.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64, device="cuda") / d)

    def turned(x, pos):
        angle = pos.double()[:, None, None] * freq
        if case["interleaved"]:
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], d // 2, 2).contiguous())
        else:
            z = torch.complex(x[..., : d // 2].contiguous(), x[..., d // 2:].contiguous())
        z = z * torch.polar(torch.ones_like(angle), angle)
        if case["interleaved"]:
            return torch.view_as_real(z).flatten(-2)
        return torch.cat([z.real, z.imag], -1)

    row = 0
    for b, (n, length) in enumerate(spans):
        pos = torch.arange(length - n, length, device="cuda")
        x = s["qkv"][row:row + n].double().view(n, hq + 2 * hk, d)
        row += n
        out["q"].append(turned(x[:, :hq], pos))
        start = _first_read(case, n, length)
        for which, fresh in (("k", turned(x[:, hq:hq + hk], pos)), ("v", x[:, hq + hk:])):
            for p0 in range(start, length, ps):  # one page after the other
                page = int(s["table"][b, p0 // ps])
                lo, hi = max(p0, length - n), min(p0 + ps, length)
                mine = fresh[lo - (length - n):hi - (length - n)]
                old = scales[which][page] if lo > p0 else torch.zeros(hk, dtype=torch.float64, device="cuda")
                now = torch.maximum(old, mine.abs().amax((0, 2)) / 127)
                kept = s[which][page].double()[:, :lo - p0] * (old / now)[:, None, None]
                whole = torch.cat([kept, mine.transpose(0, 1) / now[:, None, None]], 1).round()
                out[which].append((whole * now[:, None, None]).transpose(0, 1))
                scales[which][page] = now
    return {"q": torch.cat(out["q"]), "k": torch.cat(out["k"]), "v": torch.cat(out["v"]),
            "k_scale": scales["k"], "v_scale": scales["v"]}
