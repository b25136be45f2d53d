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
