"""The 4-bit key-value cache restated on the CPU, row by row from its definition: quantisation, where a group's bytes lie, attention and
the tables of a step.  Test infrastructure only."""
import numpy as np
import torch

KEY_ROWS = [0, 4, 1, 5, 2, 6, 3, 7, 8, 12, 9, 13, 10, 14, 11, 15]       # the token whose key codes lie in each row of a group
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def quantise(x):
    """16-bit rows [n, hd] -> codes (int64), scale and low end (16 bits, [n])."""
    f = x.float()
    low, high = f.amin(1) + 0.0, f.amax(1)                          # (no negative zero)
    want = (high - low) / torch.full_like(low, 15.0)
    s = want.to(x.dtype)
    s = torch.where(s.float() < want, (s.view(torch.int16) + 1).view(x.dtype), s)
    top = (low.double() + 15 * s.double()).float().to(x.dtype).float()
    s = torch.where(torch.isfinite(top), s, (s.view(torch.int16) - 1).view(x.dtype))
    fine = torch.isfinite(f).all(1) & torch.isfinite(high - low)
    code = torch.round((f - low[:, None]) / s.float()[:, None]).clamp(max=15)
    code = torch.where(fine[:, None] & (s > 0)[:, None], code, 0.0)
    nan = torch.full_like(s, float("nan"))
    return code.long(), torch.where(fine, s, nan), torch.where(fine, low.to(x.dtype), nan)


def pack_words(code):
    """Codes [hd] -> hd / 8 words."""
    out = []
    for j in range(0, len(code), 8):
        w = 0
        for d in range(8):
            w |= int(code[j + d]) << (4 * (d // 2) + 16 * (d % 2))
        out.append(w)
    return out


class Cache:
    """Codes, scales and low ends by slot; `data` is the buffer that the kernels see."""

    def __init__(self, blocks, KV, hd, bs, dt, fill=None):
        self.blocks, self.KV, self.hd, self.bs, self.dt = blocks, KV, hd, bs, dt
        self.group = 16 * (hd + 8)
        self.data = np.zeros((blocks, KV, bs // 16, self.group), dtype=np.uint8)
        if fill is not None:
            self.data[:] = fill

    def put(self, k, v, slots):
        """16-bit rows [T, KV, hd] at their slots."""
        hd = self.hd
        for h in range(self.KV):
            for x, key in ((k[:, h], True), (v[:, h], False)):
                code, s, low = quantise(x)
                par = torch.stack([s, low], 1).contiguous().view(torch.int16).numpy().astype(np.uint16)
                nan = ~torch.isfinite(s)
                for i, slot in enumerate(slots):
                    if slot < 0:
                        continue
                    g = self.data[slot // self.bs, h, slot % self.bs // 16]
                    tok = slot % 16
                    words = pack_words(code[i])
                    if key:
                        at = KEY_ROWS.index(tok) * hd // 2
                    else:
                        at = 8 * hd + tok * hd // 2
                        if hd == 128 and tok & 2:
                            words = words[8:] + words[:8]
                    g[at:at + hd // 2] = np.frombuffer(np.array(words, dtype=np.uint32).tobytes(), dtype=np.uint8)
                    pair = np.array([0x7fff, 0x7fff], dtype=np.uint16) if nan[i] else par[i]
                    at = 16 * hd + (0 if key else 64) + 4 * tok
                    g[at:at + 4] = np.frombuffer(pair.tobytes(), dtype=np.uint8)

    def put_all(self, k, v, slots):
        """put() for many rows, all of them at once; slots from 0 on."""
        hd, slots = self.hd, np.asarray(slots, dtype=np.int64)
        at, tok = (slots // self.bs, slice(None), slots % self.bs // 16), slots % 16
        g = self.data[at]                                           # [n, KV, group]
        n = np.arange(len(slots))
        for x, key in ((k, True), (v, False)):
            code, s, low = (y.reshape(x.shape[:2] + y.shape[1:]) for y in quantise(x.reshape(-1, hd)))
            c = code.numpy().astype(np.uint32).reshape(*x.shape[:2], hd // 8, 8)
            words = sum(c[..., d] << np.uint32(4 * (d // 2) + 16 * (d % 2)) for d in range(8))
            if not key and hd == 128:
                words = np.where((tok & 2)[:, None, None] > 0, np.roll(words, 8, 2), words)
            row = np.array([KEY_ROWS.index(t) for t in range(16)])[tok] if key else tok
            part = slice(0, 8 * hd) if key else slice(8 * hd, 16 * hd)
            rows = g[:, :, part].reshape(len(slots), self.KV, 16, hd // 2)
            rows[n, :, row] = np.ascontiguousarray(words).view(np.uint8)
            g[:, :, part] = rows.reshape(len(slots), self.KV, 8 * hd)
            pair = torch.stack([s, low], -1).contiguous().view(torch.int16).numpy().astype(np.uint16)
            pair[torch.isnan(s).numpy()] = 0x7fff
            part = slice(16 * hd, 16 * hd + 64) if key else slice(16 * hd + 64, 16 * hd + 128)
            rows = g[:, :, part].reshape(len(slots), self.KV, 16, 4)
            rows[n, :, tok] = np.ascontiguousarray(pair).view(np.uint8)
            g[:, :, part] = rows.reshape(len(slots), self.KV, 64)
        for t in range(16):                                         # (tokens of one group one after the other)
            i = np.nonzero(tok == t)[0]
            old = self.data[at[0][i], :, at[2][i]]
            for key in (True, False):
                r = (KEY_ROWS.index(t) if key else 16 + t) * (hd // 2)
                old[:, :, r:r + hd // 2] = g[i][:, :, r:r + hd // 2]
                r = 16 * hd + 4 * t + (0 if key else 64)
                old[:, :, r:r + 4] = g[i][:, :, r:r + 4]
            self.data[at[0][i], :, at[2][i]] = old

    def parts(self, slots, h):
        """(codes, scales, low ends) of keys and of values at `slots`, in 64 bits: low + scale code is get()."""
        hd, out = self.hd, []
        slots = np.asarray(slots, dtype=np.int64)
        g, tok, n = self.data[slots // self.bs, h, slots % self.bs // 16], slots % 16, np.arange(len(slots))
        for key, vals in zip((True, False), self.get(slots, h)):
            at = 16 * hd + (0 if key else 64)
            par = torch.from_numpy(np.ascontiguousarray(g[:, at:at + 64].reshape(len(slots), 16, 4)[n, tok])).view(self.dt).double()
            s, low = par[:, :1], par[:, 1:]
            out.append((torch.where(s > 0, torch.round((vals - low) / torch.where(s > 0, s, 1.0)), 0.0), s, low))
        return out

    def get(self, slots, h):
        """Keys and values [n, hd] in 64 bits at `slots`."""
        hd, out = self.hd, []
        slots = np.asarray(slots, dtype=np.int64)
        g = self.data[slots // self.bs, h, slots % self.bs // 16]
        tok = slots % 16
        n = np.arange(len(slots))
        for key in (True, False):
            row = np.array([KEY_ROWS.index(t) for t in range(16)])[tok] if key else tok
            rows = g[:, (0 if key else 8 * hd):(8 * hd if key else 16 * hd)].reshape(len(slots), 16, hd // 2)[n, row]
            words = np.ascontiguousarray(rows).view(np.uint32)
            if not key and hd == 128:
                words = np.where((tok & 2)[:, None] > 0, np.roll(words, 8, 1), words)
            code = np.stack([words >> (4 * (d // 2) + 16 * (d % 2)) & 15 for d in range(8)], -1).reshape(len(slots), hd)
            at = 16 * hd + (0 if key else 64)
            par = torch.from_numpy(np.ascontiguousarray(g[:, at:at + 64].reshape(len(slots), 16, 4)[n, tok])).view(self.dt).double()
            out.append(par[:, 1:] + par[:, :1] * torch.from_numpy(code.astype(np.float64)))
        return out

    def tensor(self):
        return torch.from_numpy(self.data).cuda()


def attention(cache, q, table, lens, qsl, H, scale, window=0, first=0):
    """q [T, H, hd]; returns (out, sum of p |v|, the largest of scale sum |q| |k|) in 64 bits; rows of no request are NaN."""
    T, KV, hd, bs = q.shape[0], cache.KV, cache.hd, cache.bs
    out = torch.full((T, H, hd), float("nan"), dtype=torch.float64)
    size, reach = torch.zeros(T, H, hd, dtype=torch.float64), torch.zeros(T, H, 1, dtype=torch.float64)
    G = H // KV
    for b, n in enumerate(lens):
        r0, r1 = qsl[b], qsl[b + 1]
        pos = torch.arange(n - (r1 - r0), n)
        if r1 == r0:
            continue
        slots = [int(table[b][j // bs]) * bs + j % bs for j in range(n)]
        j = torch.arange(n)
        seen = j[None, :] <= pos[:, None]
        if window:
            seen &= (pos[:, None] - j[None, :] < window) | (j[None, :] < first)
        for h in range(KV):
            if n:
                k, v = cache.get(slots, h)
            else:
                k = v = torch.zeros(0, hd, dtype=torch.float64)
            for g in range(G):
                x = q[r0:r1, h * G + g].double()
                s = x @ k.T * scale
                bad = torch.isnan(k).any(1) | torch.isnan(v).any(1)
                s = torch.where(seen, s, -torch.inf)
                top = s.nan_to_num(nan=-torch.inf).amax(1, keepdim=True) if n else torch.zeros(r1 - r0, 1)
                p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
                p = torch.where(seen, p, 0.0)
                l = p.sum(1, keepdim=True)
                clean = torch.where(bad[:, None], 0.0, v)
                o = torch.where(l == 0, 0.0, (p @ clean) / torch.where(l == 0, 1.0, l))
                o = torch.where((seen & bad[None, :]).any(1, keepdim=True), torch.nan, o)
                out[r0:r1, h * G + g] = o
                size[r0:r1, h * G + g] = (p @ clean.abs()) / torch.where(l == 0, 1.0, l)
                if n:
                    reach[r0:r1, h * G + g, 0] = (torch.where(seen, (x.abs() @ k.nan_to_num().abs().T) * scale, 0.0)).amax(1)
    return out, size, reach


def attention_terms(cache, q, table, lens, qsl, H, scale, window=0, first=0, device="cpu"):
    """attention() for finite rows, with what its errors are measured by: with z = low + 8 s of a row, a sum of 16-bit weights is off by their
    rounding times sum p s |code - 8|, sums in 32 bits by theirs times that and sum p |z|, and a score by theirs times reach, the largest visible
    scale (s sum |q| |code - 8| + |z| sum |q|).  most: the largest p s / sum p.  square: of p s |code - 8|, the root of the sum of
    squares.  whole: the visible rows' sum of |v|.  Returns (out, codes, rest, most, reach, keys, whole, square), [T, H, hd] or 1."""
    T, KV, hd, bs = q.shape[0], cache.KV, cache.hd, cache.bs
    G = H // KV
    out, codes, rest, whole, square = (torch.zeros(T, H, hd, dtype=torch.float64, device=device) for _ in range(5))
    most, reach, keys = (torch.zeros(T, H, 1, dtype=torch.float64, device=device) for _ in range(3))
    for b, n in enumerate(lens):
        r0, r1 = int(qsl[b]), int(qsl[b + 1])
        if r1 == r0 or n == 0:
            continue
        j, pos = torch.arange(n, device=device), torch.arange(n - (r1 - r0), n, device=device)
        back = pos[:, None] - j[None, :]
        seen = back >= 0
        if window:
            seen &= (back < window) | (j[None, :] < first)
        seen = seen[None]
        slots = table[b][np.arange(n) // bs].astype(np.int64) * bs + np.arange(n) % bs
        for h in range(KV):
            (kc, ks, kl), (vc, vs, vl) = ((x.to(device) for x in p) for p in cache.parts(slots, h))
            x = q[r0:r1, h * G:(h + 1) * G].double().to(device).transpose(0, 1)                      # [G, rows, hd]
            s = (x @ (kl + ks * kc).T * scale).masked_fill(~seen, -torch.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, 1.0, l)
            far = ((x.abs() @ ((kc - 8).abs() * ks).T + x.abs().sum(-1, keepdim=True) * (kl + 8 * ks).abs().T) * scale).masked_fill(~seen, 0.0)
            at = (slice(r0, r1), slice(h * G, (h + 1) * G))
            out[at] = (p @ (vl + vs * vc)).transpose(0, 1)
            codes[at] = ((p * vs.T) @ (vc - 8).abs()).transpose(0, 1)
            whole[at] = (seen[0].double() @ (vl + vs * vc).abs())[:, None].expand(-1, G, -1)
            square[at] = ((p * vs.T) ** 2 @ (vc - 8) ** 2).sqrt().transpose(0, 1)
            rest[at] = (p @ (vl + 8 * vs).abs()).expand(-1, -1, hd).transpose(0, 1)
            most[at] = (p * vs.T).amax(-1, keepdim=True).transpose(0, 1)
            reach[at] = far.amax(-1, keepdim=True).transpose(0, 1)
            keys[at] = seen.sum(-1, keepdim=True).double().expand(G, -1, -1).transpose(0, 1)
    return out, codes, rest, most, reach, keys, whole, square


def allowed(terms, dt):
    """How far a result may be from attention_terms(): its own rounding; weights rounded to float16, 2^-11 of each, or 2^-25 where they are smaller
    than its normal numbers (the largest is 2^0 or more, or the largest exponential is 2^90 or more, or there is a row 2^90 above the codes' steps);
    a score of hd + 8 roundings of 2^-23 of its reach, which stand in weights and in their sum; 2^-18 for sums, exponentials and the division in 32
    bits; what 16 and 32 bits hold no more, which for exponentials is 2^-126 of the largest."""
    out, codes, rest, most, reach, keys, whole, square = terms
    hd = out.shape[-1]
    fp32 = 2.0 ** -18 + 2 * (hd + 8) * 2.0 ** -23 * reach
    small = 8 * 2.0 ** -25 * keys * (most + 2.0 ** -90 + 2.0 ** -90 * rest)
    return half_step(dt) * out.abs() + 2.0 ** -11 * codes + fp32 * (codes + rest) + small + 2.0 ** -126 * whole + torch.finfo(dt).smallest_normal * half_step(dt) + 2.0 ** -126


def maps(table, cached, new, free, first, T, bs):
    """kge_step_maps, one request after the other."""
    table = table.copy()
    M = table.shape[1] * bs
    rows, at, lack, asked = T, min(max(first, 0), len(free)), 0, 0
    lens, qsl, pos, slots = [], [0], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = min(max(c, 0), M), max(n, 0)
        asked += n
        n = min(n, M - c, rows)
        rows -= n
        held, want = -(-c // bs), -(-(c + n) // bs)
        got = min(want - held, len(free) - at)
        table[b, held:held + got] = free[at:at + got]
        at, lack = at + got, lack + want - held - got
        n = min(n, (held + got) * bs - c)
        lens.append(c + n)
        qsl.append(qsl[-1] + n)
        pos += range(c, c + n)
        slots += [int(table[b, p // bs]) * bs + p % bs for p in range(c, c + n)]
    pad = T - len(pos)
    return table, lens, qsl, pos + [0] * pad, slots + [-1] * pad, [qsl[-1], min(asked, 2 ** 31 - 1), at, lack]
