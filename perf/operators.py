"""The operators around the 4-bit key-value cache, as they are timed and checked: the tables of a step built on the GPU, the rotary
embedding that quantises into the cache (with the rows read back), and paged attention over it, whole contexts and sliding windows.

  maps     block tables, slots, positions and row offsets of a step from its requests' lengths
  write    rotary positions, quantisation and the scatter into the pages; then the written rows back in 16 bits
  attn     attention of a flattened batch (decode rows first, then prompt chunks) over the pages; `window` > 0 keeps the last `window`
           keys of a query and the first `first` ones

A row (one token, one kv head) of the cache holds codes c of 4 bits, a scale s and a low end m in the model's 16-bit type, and stands for
m + s c.  Sixteen tokens of a kv head lie together: key codes, value codes, (s, m) of the keys, (s, m) of the values.  Within 8 codes the
even dimensions are the low half of a 32-bit word, the odd ones the high half; key rows lie in the order KEY_ORDER; in value rows of
128 dimensions the two halves of every second pair of tokens are exchanged.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
KEY_ORDER = [0, 4, 1, 5, 2, 6, 3, 7, 8, 12, 9, 13, 10, 14, 11, 15]      # the token at each place of a group's key codes
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]                                      # the dimension at each nibble of a word


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    write = dict(kind="write", dtype="bf16", heads=32, kv=8, hd=128, block=64, pad=0)
    attn = dict(kind="attn", dtype="bf16", heads=32, kv=8, hd=128, block=64, window=0, first=0, prompts=0, chunk=0, prior=0)
    return [
        # a decode step of 64 requests at 2k-in / 256-out: one token each
        dict(kind="maps", name="maps-decode-64", reqs=64, ctx_lo=2048, ctx_hi=2304, prompts=0, chunk=0, block=64, rows=64),
        # a full step: 500 decode requests and prompt chunks in a token budget of 8192, with blocks of 16
        dict(kind="maps", name="maps-mixed-512", reqs=500, ctx_lo=1, ctx_hi=4000, prompts=12, chunk=700, block=16, rows=8192),
        # the 8B model's decode step of 64 requests: one layer's keys and values
        dict(write, name="write-8b-64", rows=64),
        # the same in a full prompt step
        dict(write, name="write-8b-8192", rows=8192),
        # an odd number of prompt tokens of the 1B model in float16, padded rows behind them
        dict(write, name="write-fp16-1339", dtype="fp16", hd=64, block=16, rows=1339, pad=5),
        # 32 short chats on the 1B model with blocks of 16 tokens: little work for the whole chip
        dict(attn, name="attn-decode-1b", hd=64, block=16, reqs=32, ctx_lo=96, ctx_hi=256),
        # 64 concurrent requests of the 8B model generate at 2k-in / 256-out
        dict(attn, name="attn-decode-8b", reqs=64, ctx_lo=2048, ctx_hi=2304),
        # one request with a very long document: few rows, a long axis
        dict(attn, name="attn-decode-long", reqs=1, ctx_lo=131001, ctx_hi=131001),
        # a prompt step: four whole 2k prompts fill the token budget of 8192
        dict(attn, name="attn-prefill-8b", reqs=0, ctx_lo=0, ctx_hi=0, prompts=4, chunk=2048),
        # a mixed step in float16: decode rows beside odd chunks of prompts whose beginnings are already cached
        dict(attn, name="attn-mixed-fp16", dtype="fp16", block=16, reqs=6, ctx_lo=50, ctx_hi=3000, prompts=2, chunk=1011, prior=1777),
        # decode under a sliding window of 1024 keys with four kept first tokens
        dict(attn, name="window-decode-8b", reqs=64, ctx_lo=500, ctx_hi=6000, window=1024, first=4),
        # a long prompt under the same window, in odd chunks behind cached keys
        dict(attn, name="window-prefill-8b", reqs=0, ctx_lo=0, ctx_hi=0, prompts=2, chunk=1931, prior=999, window=1024, first=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["maps", "write", "write", "attn", "attn", "attn", "window", "window"])
    if kind == "maps":
        prompts = rng.choice([0, _log(rng, 1, 16)])
        reqs, chunk = _log(rng, 1, 512), _log(rng, 1, 500)
        hi = _log(rng, 2, 8000)
        return dict(kind=kind, reqs=reqs, ctx_lo=rng.randint(1, hi), ctx_hi=hi, prompts=prompts, chunk=chunk if prompts else 0, block=rng.choice([16, 32, 64]),
                    rows=max(1, reqs + prompts * chunk + rng.choice([-3, 0, 5, 100])))
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    hd, block, kv = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 3, 4, 4, 8])
    c = dict(kind=kind if kind == "write" else "attn", dtype=dtype, heads=heads, kv=kv, hd=hd, block=block)
    if kind == "write":
        c.update(rows=_log(rng, 1, 6000 if heads <= 32 else 3500), pad=rng.choice([0, 0, rng.randint(1, 40)]))
        return c
    c.update(window=0, first=0, prompts=0, chunk=0, prior=0)
    if kind == "window":
        c.update(window=_log(rng, 1, 4096), first=rng.choice([0, 1, 4, 64, _log(rng, 2, 300)]))
    mode = rng.choice(["decode", "decode", "long", "prefill", "mixed"])
    if mode == "long":
        hi = _log(rng, 8000, 131000)
        c.update(reqs=rng.choice([1, 1, 2]) if hi < 65000 else 1, ctx_lo=hi // 2, ctx_hi=hi)
    elif mode == "decode":
        hi = _log(rng, 16, 4096)
        c.update(reqs=min(_log(rng, 1, 150), 140_000_000 // (hi * kv * hd)), ctx_lo=max(1, hi // rng.choice([1, 2, 20])), ctx_hi=hi)
    else:
        prompts, prior, hi = _log(rng, 1, 6), rng.choice([0, 0, _log(rng, 10, 2500)]), _log(rng, 16, 2500)
        c.update(reqs=_log(rng, 1, 12) if mode == "mixed" else 0, ctx_lo=max(1, hi // 3) if mode == "mixed" else 0, ctx_hi=hi if mode == "mixed" else 0)
        n, longest = c["reqs"] + prompts, max(hi if mode == "mixed" else 0, 1900 + prior)
        c.update(prompts=prompts, prior=prior, chunk=_log(rng, 2, max(3, min(1900, 500_000_000 // (n * heads * longest)))))
    return c


# ----------------------------------------------------------------------------------------------------- inputs, shared

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 + seed)


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _lengths(case, seed):
    """Cached and new tokens of the flattened batch: decode requests first, then prompt chunks."""
    r = np.random.default_rng(seed + 17)
    cached = (r.integers(case["ctx_lo"], case["ctx_hi"] + 1, case["reqs"]) - 1).tolist() if case["reqs"] else []
    new = [1] * len(cached)
    for i in range(case["prompts"]):
        new.append(max(1, case["chunk"] - i * 7 % 5 if case.get("prior") or case["kind"] == "maps" else case["chunk"]))
        cached.append(case["prior"] + 131 * i if case.get("prior") else 0)
    return cached, new


def _tables(g, cached, new, bs):
    """Each request's blocks, in random order of the pool; block 0 is the null block."""
    per = [-(-(c + n) // bs) for c, n in zip(cached, new)]
    blocks = sum(per) + 1
    order = torch.randperm(blocks - 1, generator=g, device="cuda").add_(1).to(torch.int32)
    table = torch.zeros(len(per), max(per), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, blocks


def _round_up(x, dt):
    """Numbers that are not negative, rounded up to a 16-bit type."""
    r = x.to(dt)
    return torch.where(r.float() < x, (r.view(torch.int16) + 1).view(dt), r)


def _quantise(x):
    """16-bit rows [..., hd] -> codes (uint8), scale and low end (16 bits)."""
    f = x.float()
    low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    s = _round_up((high - low) / torch.full_like(low, 15.0), x.dtype)      # (a division; by a number it would be a product with 1 / 15)
    code = torch.where(s > 0, torch.round((f - low) / s.float()), torch.zeros_like(f))
    bad = ~torch.isfinite(high - low)
    nan = torch.full_like(s, math.nan)
    return torch.where(bad, 0.0, code).to(torch.uint8), torch.where(bad, nan, s), torch.where(bad, nan, low.to(x.dtype))


def _pack(code):
    """Codes [..., hd] -> bytes [..., hd / 2]."""
    w = code.unflatten(-1, (-1, 8))[..., NIBBLES].unflatten(-1, (4, 2))
    return (w[..., 0] + w[..., 1] * 16).flatten(-2)


def _unpack(b):
    """Bytes [..., hd / 2] -> codes [..., hd]."""
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))
    return n[..., [NIBBLES.index(d) for d in range(8)]].flatten(-2)


def _value_bytes(hd, device):
    """[16, hd / 2]: where the bytes of each token's value row lie in the row."""
    at = torch.arange(hd // 2, device=device)[None, :].expand(16, -1)
    return at ^ ((torch.arange(16, device=device)[:, None] >> 1 & 1) * 32) if hd == 128 else at


def _groups(k, v, bs):
    """16-bit rows [blocks, KV, bs, hd] of keys and values -> the cache's bytes [blocks, KV, bs / 16, 16 (hd + 8)]."""
    hd, parts, params = k.shape[-1], [], []
    for x, keys in ((k, True), (v, False)):
        code, s, low = _quantise(x)
        b = _pack(code).unflatten(2, (-1, 16))
        b = b[:, :, :, KEY_ORDER] if keys else torch.gather(b, -1, _value_bytes(hd, b.device).expand_as(b))
        parts.append(b.flatten(-2))
        params.append(torch.cat([s, low], -1).contiguous().view(torch.uint8).unflatten(2, (-1, 16)).flatten(-2))
    return torch.cat(parts + params, -1)


def _rows(groups, hd, dt):
    """The cache's bytes [..., 16 (hd + 8)] -> numbers [..., 16, hd] of keys and of values, in 32 bits."""
    n, out = 8 * hd, []
    for keys in (True, False):
        b = groups[..., :n] if keys else groups[..., n:2 * n]
        b = b.unflatten(-1, (16, hd // 2))
        b = b[..., [KEY_ORDER.index(t) for t in range(16)], :] if keys else torch.gather(b, -1, _value_bytes(hd, b.device).expand_as(b))
        p = groups[..., 2 * n + (0 if keys else 64):2 * n + (64 if keys else 128)].contiguous().view(dt).unflatten(-1, (16, 2)).float()
        out.append(p[..., 1:] + p[..., :1] * _unpack(b).float())
    return out


def _lib(st):
    """The framework's library, and the stream of the pass."""
    if "lib" not in st:
        from kge_loader import load
        st["kge"] = load()
        st["lib"] = st["kge"].lib()
    return st["lib"]


def _call(st, name, *args):
    """One entry point of the C ABI on torch's current stream; tensors are passed by their device pointer."""
    lib = _lib(st)
    rc = getattr(lib, name)(*[a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args], torch.cuda.current_stream().cuda_stream)
    if rc < 0:
        st["kge"].check(rc, name)


def _name(case, name):
    return name + ("_f16" if case["dtype"] == "fp16" else "")


# --------------------------------------------------------------------------------------------------------------- maps

def _maps_prepare(case, seed):
    g = _gen(seed)
    cached, new = _lengths(case, seed)
    bs, B = case["block"], len(cached)
    held = [-(-c // bs) for c in cached]
    need = sum(-(-(c + n) // bs) for c, n in zip(cached, new)) - sum(held)
    free = need + 40 if seed % 4 else max(1, need - 3)                       # now and then the pool is short of blocks
    ids = torch.randperm(sum(held) + free + 7, generator=g, device="cuda").add_(1).to(torch.int32)
    most = max(-(-case["ctx_hi"] // bs), -(-case["chunk"] // bs)) + 1
    table = torch.zeros(B, most, dtype=torch.int32, device="cuda")
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    i32 = dict(dtype=torch.int32, device="cuda")
    T = case["rows"]
    return dict(case=case, B=B, T=T, most=most, table=table, cached=torch.tensor(cached, **i32), new=torch.tensor(new, **i32), free=ids[at:].contiguous(),
                nfree=7 + free, first=torch.full((1,), 7, **i32), lens=torch.zeros(B, **i32), qsl=torch.zeros(B + 1, **i32), pos=torch.zeros(T, **i32),
                slots=torch.zeros(T, dtype=torch.int64, device="cuda"), counts=torch.zeros(4, **i32))


def _excl(x):
    return x.cumsum(0) - x


def _maps_plain(st):
    bs, T, M, dev = st["case"]["block"], st["T"], st["most"], "cuda"
    c = st["cached"].long().clamp(0, M * bs)
    asked = st["new"].long().clamp(min=0)
    n = torch.minimum(asked, M * bs - c)
    n = torch.minimum(n, (T - _excl(n)).clamp(min=0))
    held = (c + bs - 1) // bs
    need = (c + n + bs - 1) // bs - held
    first = st["first"].long().clamp(0, st["nfree"])
    pos = first + _excl(need)
    got = torch.minimum(need, (st["nfree"] - pos).clamp(min=0))
    n = torch.where(got < need, torch.minimum(n, (held + got) * bs - c), n)
    at = torch.arange(M, device=dev)[None, :] - held[:, None]
    fresh = (at >= 0) & (at < got[:, None])
    st["table"].copy_(torch.where(fresh, st["free"][(pos[:, None] + at).clamp(0, st["free"].numel() - 1)], st["table"]))
    st["lens"].copy_(c + n)
    end = n.cumsum(0)
    st["qsl"][1:] = end
    row = torch.arange(T, device=dev)
    b = torch.searchsorted(end, row, right=True).clamp(max=st["B"] - 1)
    there = row < end[-1]
    p = torch.where(there, c[b] + row - (end - n)[b], 0)
    st["pos"].copy_(p)
    st["slots"].copy_(torch.where(there, st["table"][b, (p // bs).clamp(max=M - 1)].long() * bs + p % bs, -1))
    st["counts"].copy_(torch.cat([end[-1:], asked.sum()[None], first + got.sum(), (need - got).sum()[None]]))


def _maps_run(st):
    if own:
        _call(st, "kge_step_maps", st["table"], st["most"], st["lens"], st["qsl"], st["pos"], st["slots"], st["counts"], st["cached"], st["new"], st["free"],
              st["nfree"], st["first"], st["B"], st["T"], st["case"]["block"])
    else:
        _maps_plain(st)
    return {k: st[k] for k in ("table", "lens", "qsl", "pos", "slots", "counts")}


def _maps_exact(case, seed):
    st = _maps_prepare(case, seed)
    bs, T, M = case["block"], st["T"], st["most"]
    table, free = st["table"].cpu().numpy().copy(), st["free"].cpu().numpy()
    cached, new = st["cached"].tolist(), st["new"].tolist()
    rows, lack, at, lens, qsl, pos, slots = T, 0, 7, [], [0], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        n = min(n, M * bs - c, rows)
        rows -= n
        held = -(-c // bs)
        need = -(-(c + n) // bs) - held
        got = min(need, st["nfree"] - at)
        table[b, held:held + got] = free[at:at + got]
        at, lack = at + got, lack + need - got
        n = min(n, (held + got) * bs - c)
        lens.append(c + n)
        qsl.append(qsl[-1] + n)
        pos += list(range(c, c + n))
        slots += [int(table[b, p // bs]) * bs + p % bs for p in range(c, c + n)]
    end = [0] * (T - len(pos))
    return {"table": torch.tensor(table), "lens": torch.tensor(lens, dtype=torch.int32), "qsl": torch.tensor(qsl, dtype=torch.int32),
            "pos": torch.tensor(pos + end, dtype=torch.int32), "slots": torch.tensor(slots + [-1] * len(end)),
            "counts": torch.tensor([qsl[-1], sum(new), at, lack], dtype=torch.int32)}


def _maps_work(case):
    n = case["reqs"] + case["prompts"]
    return {"bytes": 24.0 * n + 12.0 * case["rows"], "flops": 0.0}


# -------------------------------------------------------------------------------------------------------------- write

def _write_inputs(case, seed):
    g, dt, T, hd, bs = _gen(seed), DT[case["dtype"]], case["rows"], case["hd"], case["block"]
    n = case["heads"] + 2 * case["kv"]
    qkv = _randn(g, (T, n * hd), dt)
    ang = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)[None, :]
    cs = torch.cat([ang.cos(), ang.sin()], -1).to(dt)
    pos = torch.randint(0, 8192, (T,), generator=g, device="cuda", dtype=torch.int32)
    blocks = (T + bs - 1) // bs + 3
    # runs of tokens in order, as prompts have them, over blocks in random order; padded rows at the end
    page = torch.randperm(blocks - 1, generator=g, device="cuda") + 1
    t = torch.arange(T, device="cuda")
    slots = page[t // bs] * bs + t % bs
    slots[max(0, T - case["pad"]):] = -1
    return dict(qkv=qkv, cs=cs, pos=pos, slots=slots, blocks=blocks)


def _write_prepare(case, seed):
    st = dict(_write_inputs(case, seed), case=case)
    T, hd, bs, kv, dt = case["rows"], case["hd"], case["block"], case["kv"], DT[case["dtype"]]
    st["cache"] = torch.zeros(st["blocks"], kv, bs // 16, 16 * (hd + 8), dtype=torch.uint8, device="cuda")
    st["q"] = torch.empty(T, case["heads"] * hd, dtype=dt, device="cuda")
    st["k"], st["v"] = (torch.empty(T, kv, hd, dtype=dt, device="cuda") for _ in range(2))
    return st


def _rotate(x, cs):
    """Rows [T, heads, hd] turned by the pairs (i, i + hd / 2), in the type of the tables."""
    cos, sin = cs[:, None, :].chunk(2, -1)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _write_plain(st):
    c = st["case"]
    H, KV, hd, bs, dt = c["heads"], c["kv"], c["hd"], c["block"], DT[c["dtype"]]
    x = st["qkv"].view(-1, H + 2 * KV, hd)
    turned = _rotate(x[:, :H + KV].float(), st["cs"][st["pos"].long()].float()).to(dt)
    st["q"].copy_(turned[:, :H].flatten(1))
    there = st["slots"] >= 0
    slot = st["slots"][there]
    blk, grp, tok = slot // bs, slot % bs // 16, slot % 16
    head = torch.arange(KV, device="cuda")
    at = blk[:, None, None], head[None, :, None], grp[:, None, None]
    half = torch.arange(hd // 2, device="cuda")
    place = torch.tensor([KEY_ORDER.index(t) for t in range(16)], device="cuda")[tok]
    for n, rows in enumerate((turned[:, H:][there], x[:, H + KV:][there])):
        code, s, low = _quantise(rows)
        off = (place[:, None] * (hd // 2) + half) if n == 0 else 8 * hd + tok[:, None] * (hd // 2) + _value_bytes(hd, "cuda")[tok]
        st["cache"][at + (off[:, None, :],)] = _pack(code)
        off = 16 * hd + 64 * n + 4 * tok[:, None] + torch.arange(4, device="cuda")
        st["cache"][at + (off[:, None, :],)] = torch.cat([s, low], -1).contiguous().view(torch.uint8)
    # the rows again, from the cache
    slot = st["slots"].clamp(min=0)
    k, v = _rows(st["cache"][slot // bs, :, slot % bs // 16], hd, dt)
    at = (slot % 16)[:, None, None, None].expand(-1, KV, 1, hd)
    for name, rows in (("k", k), ("v", v)):
        st[name].copy_(torch.where(there[:, None, None], torch.gather(rows, 2, at)[:, :, 0], 0.0))


def _write_run(st):
    c = st["case"]
    T, H, KV, hd, bs = c["rows"], c["heads"], c["kv"], c["hd"], c["block"]
    if own:
        _call(st, _name(c, "kge_rope_kv4write"), st["q"], H * hd, st["cache"], st["qkv"], st["cs"], st["pos"], st["slots"], T, H, KV, hd, bs)
        _call(st, _name(c, "kge_kv4_read"), st["k"], st["v"], st["cache"], st["slots"], T, KV, hd, bs)
    else:
        _write_plain(st)
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def _write_exact(case, seed):
    i = _write_inputs(case, seed)
    H, KV, hd, dt = case["heads"], case["kv"], case["hd"], DT[case["dtype"]]
    x = i["qkv"].double().view(-1, H + 2 * KV, hd)
    turned = _rotate(x[:, :H + KV], i["cs"].double()[i["pos"].long()])
    out = {"q": turned[:, :H].flatten(1)}
    for name, rows in (("k", turned[:, H:].float().to(dt).double()), ("v", x[:, H + KV:])):      # what is quantised has 16 bits
        low, high = rows.amin(-1, keepdim=True), rows.amax(-1, keepdim=True)
        s = _round_up(((high - low) / 15.0).float(), dt).double()
        y = low + s * torch.round((rows - low) / s)
        out[name] = torch.where((i["slots"] >= 0)[:, None, None], y, 0.0)
    return out


def _write_work(case):
    T, H, KV, hd = case["rows"], case["heads"], case["kv"], case["hd"]
    rows = T - min(T, case["pad"])
    # qkv in, q out, a row of the tables, the cache's rows out and (to be read back) in, keys and values out
    return {"bytes": 2.0 * T * hd * (2 * H + 2 * KV) + T * (2.0 * hd + 12) + 2.0 * rows * KV * (hd + 8) + 4.0 * T * KV * hd, "flops": 3.0 * T * (H + KV) * hd}


# ---------------------------------------------------------------------------------------------------------- attention

def _attn_inputs(case, seed):
    g, dt = _gen(seed), DT[case["dtype"]]
    cached, new = _lengths(case, seed)
    KV, hd, bs = case["kv"], case["hd"], case["block"]
    table, blocks = _tables(g, cached, new, bs)
    q = _randn(g, (sum(new), case["heads"] * hd), dt)
    cache = torch.empty(blocks, KV, bs // 16, 16 * (hd + 8), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 24) // (KV * bs * hd))
    for at in range(0, blocks, step):                                        # a part of the pool at a time
        n = min(step, blocks - at)
        cache[at:at + n] = _groups(_randn(g, (n, KV, bs, hd), dt), _randn(g, (n, KV, bs, hd), dt), bs)
    return dict(cached=cached, new=new, table=table, q=q, cache=cache)


def _attn_prepare(case, seed):
    st = dict(_attn_inputs(case, seed), case=case)
    cached, new = st["cached"], st["new"]
    i32 = dict(dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor([c + n for c, n in zip(cached, new)], **i32)
    st["qsl"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]).tolist(), **i32)
    st["B"], st["T"], st["maxq"], st["maxc"] = len(new), sum(new), max(new), max(c + n for c, n in zip(cached, new))
    st["out"] = torch.empty_like(st["q"])
    st["ws"] = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")
    return st


def _attn_plain(st):
    c = st["case"]
    H, KV, hd, bs, B, T, maxq = c["heads"], c["kv"], c["hd"], c["block"], st["B"], st["T"], st["maxq"]
    G = H // KV
    k, v = _rows(st["cache"][st["table"].long()], hd, DT[c["dtype"]])                      # [B, pages, KV, bs / 16, 16, hd]
    k, v = (x.permute(0, 2, 1, 3, 4, 5).reshape(B, KV, -1, hd) for x in (k, v))
    lens, start = st["lens"].long(), st["qsl"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(maxq, device="cuda")
    q = st["q"].float().view(T, KV, G, hd)[(start[:-1, None] + i).clamp(max=T - 1)]        # [B, maxq, KV, G, hd]
    q = q.permute(0, 2, 3, 1, 4).reshape(B, KV, G * maxq, hd)
    s = (q @ k.transpose(-1, -2)).view(B, KV, G, maxq, -1) * hd ** -0.5
    at = (lens - n)[:, None, None] + i[None, :, None] - torch.arange(k.shape[2], device="cuda")     # how far a key lies behind its query
    seen = (at >= 0) & (i[None, :, None] < n[:, None, None])
    if c["window"]:
        seen &= (at < c["window"]) | (torch.arange(k.shape[2], device="cuda") < c["first"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    del s
    o = (p.view(B, KV, G * maxq, -1) @ v).view(B, KV, G, maxq, hd) / p.sum(-1, keepdim=True).clamp(min=1e-37)
    row = torch.arange(T, device="cuda")
    b = torch.searchsorted(start[1:], row, right=True)
    st["out"].copy_(o.permute(0, 3, 1, 2, 4)[b, row - start[b]].reshape(T, H * hd))


def _attn_run(st):
    c = st["case"]
    if own:
        _call(st, _name(c, "kge_paged_attn_kv4"), st["out"], st["q"], st["q"].shape[1], st["cache"], st["table"], st["table"].shape[1], st["lens"], st["qsl"], st["B"],
              st["T"], st["maxq"], st["maxc"], c["heads"], c["kv"], c["hd"], c["block"], c["hd"] ** -0.5, c["window"], c["first"], st["ws"], st["ws"].numel())
    else:
        _attn_plain(st)
    return st["out"]


def _attn_exact(case, seed):
    i = _attn_inputs(case, seed)
    H, KV, hd, bs, dt = case["heads"], case["kv"], case["hd"], case["block"], DT[case["dtype"]]
    G, outs, at = H // KV, [], 0
    for b, (c, n) in enumerate(zip(i["cached"], i["new"])):
        ctx = c + n
        rows = i["cache"][i["table"][b, :-(-ctx // bs)].long()]                             # [pages, KV, groups, bytes]
        q = i["q"][at:at + n].double().view(n, KV, G, hd)
        key = torch.arange(ctx, device="cuda")
        back = c + torch.arange(n, device="cuda")[:, None] - key[None, :]
        hidden = back < 0
        if case["window"]:
            hidden |= (back >= case["window"]) & (key[None, :] >= case["first"])
        o = torch.empty(n, KV, G, hd, dtype=torch.float64, device="cuda")
        for h in range(KV):
            k, v = (x.reshape(-1, hd)[:ctx].double() for x in _rows64(rows[:, h], hd, dt))
            s = torch.einsum("ngd,kd->gnk", q[:, h], k) * hd ** -0.5
            s.masked_fill_(hidden, -math.inf)
            o[:, h] = torch.einsum("gnk,kd->ngd", torch.softmax(s, -1), v)
        outs.append(o.reshape(n, H * hd))
        at += n
    return torch.cat(outs)


def _rows64(groups, hd, dt):
    """Numbers of keys and values in 64 bits, nibble by nibble from the words."""
    words = groups[..., :16 * hd].contiguous().view(torch.int32).view(*groups.shape[:-1], 2, 16, hd // 8)
    code = torch.stack([words >> (4 * (d // 2 + 4 * (d % 2))) & 15 for d in range(8)], -1).double()      # [..., 2, 16, hd / 8, 8]
    p = groups[..., 16 * hd:].contiguous().view(dt).view(*groups.shape[:-1], 2, 16, 2).double()
    for n in range(2):
        c = torch.empty_like(code[..., 0, :, :, :])
        for t in range(16):
            turn = n == 1 and hd == 128 and t & 2
            src = code[..., n, KEY_ORDER.index(t) if n == 0 else t, :, :]
            c[..., t, :, :] = src.roll(hd // 16, -2) if turn else src
        yield p[..., n, :, 1:] + p[..., n, :, :1] * c.flatten(-2)


def _attn_work(case, seed=0):
    cached, new = _lengths(case, seed)
    H, KV, hd, w, f = case["heads"], case["kv"], case["hd"], case["window"], case["first"]
    keys = pairs = 0
    for c, n in zip(cached, new):
        if not w:
            keys, pairs = keys + c + n, pairs + n * c + n * (n + 1) // 2
            continue
        low = max(0, c + 1 - w)                                                # the first query's oldest window key
        keys += c + n - low + min(f, low)
        i = np.arange(c, c + n)
        out = np.maximum(0, i + 1 - w)                                         # keys that have left the window
        pairs += int((i + 1 - out + np.minimum(out, f)).sum())
    return {"bytes": float(keys * KV * (hd + 8) + sum(new) * H * hd * 4), "flops": 4.0 * H * hd * pairs}


# ----------------------------------------------------------------------------------------------------------- the calls

_KINDS = {"maps": (_maps_prepare, _maps_run, _maps_exact, _maps_work), "write": (_write_prepare, _write_run, _write_exact, _write_work),
          "attn": (_attn_prepare, _attn_run, _attn_exact, _attn_work)}


def prepare(case, seed):
    return _KINDS[case["kind"]][0](case, seed)


def run(st):
    return _KINDS[st["case"]["kind"]][1](st)


def exact(case, seed):
    return _KINDS[case["kind"]][2](case, seed)


def work(case):
    return _KINDS[case["kind"]][3](case)
