"""Attention over the 4-bit cache, row by row: what a query does not see changes none of its bits, rows of one context may lie as far apart as
their type allows, and errors are no larger than what is rounded (kv4_oracle.allowed); prompts that fill both query tiles of an item among them.

In the 2-norm a rounding to the nearest of relative step 2 u is 0.392 u of its number where the leading digits are spread evenly over their
logarithm (the mean of u^2 / 3 over that of x^2, x from 1 to 2); weights are rounded independently, which adds 0.392 2^-11 of their terms' root of
squares.  Held to 1.12 of both; weights in bfloat16 would be at 1.4, float16 rows of a float16 model at 1.2.
"""
import math

import numpy as np
import pytest
import torch

import kv4_oracle as ko
from test_kv4_gpu import I32, call, name, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(kge):
    kge.require_cuda()
    return kge.lib()


class Batch:
    """Requests over a cache whose rows the test sets; q, keys and values N(0, 1) to begin with."""

    def __init__(self, dtype, hd, H, KV, bs, lens, news, seed=0):
        self.dt, self.hd, self.H, self.KV, self.bs, self.lens = ko.DT[dtype], hd, H, KV, bs, list(lens)
        self.g = torch.Generator().manual_seed(77 + seed)
        per = [-(-n // bs) for n in lens]
        order = (torch.randperm(sum(per), generator=self.g) + 1).tolist()
        self.table, at = np.zeros((len(lens), max(per) + 1), dtype=np.int32), 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cache = ko.Cache(sum(per) + 1, KV, hd, bs, self.dt, fill=0xFF)
        self.k, self.v = ([randn(self.g, n, KV, hd) for n in lens] for _ in range(2))
        self.news, self.T = list(news), sum(news)
        self.q = randn(self.g, self.T, H, hd).to(self.dt)
        self.qsl = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)

    def fill(self):
        for b, n in enumerate(self.lens):
            j = np.arange(n)
            self.cache.put_all(self.k[b].to(self.dt), self.v[b].to(self.dt), self.table[b][j // self.bs].astype(np.int64) * self.bs + j % self.bs)
        return self

    def run(self, kge, window=0, first=0, scale=None):
        H, KV, hd = self.H, self.KV, self.hd
        out = torch.full((self.T, H, hd), 5.0, dtype=self.dt, device="cuda")
        ws = torch.full((max(16, kge.lib().kge_attn_kv4_workspace_bytes(H, KV, hd)),), 0xFF, dtype=torch.uint8, device="cuda")
        call(kge, name("kge_paged_attn_kv4", self.dt), out, self.q.cuda(), H * hd, self.cache.tensor(), torch.from_numpy(self.table).cuda(), self.table.shape[1],
             torch.tensor(self.lens, **I32), torch.from_numpy(self.qsl).cuda(), len(self.lens), self.T, max(self.news), max(self.lens), H, KV, hd, self.bs,
             scale or hd ** -0.5, window, first, ws, ws.numel())
        torch.cuda.synchronize()
        return out

    def terms(self, window=0, first=0, scale=None):
        return ko.attention_terms(self.cache, self.q, self.table, self.lens, self.qsl, self.H, scale or self.hd ** -0.5, window, first, device="cuda")

    def check(self, out, window=0, first=0, scale=None, norm=False):
        t = self.terms(window, first, scale)
        err, tol = (out.double() - t[0]).abs(), ko.allowed(t, self.dt)
        assert (err <= tol).all(), (float((err / tol).nan_to_num(torch.inf).max()), float(err.nan_to_num(torch.inf).max()))
        if norm:
            u = ko.half_step(self.dt)
            assert err.norm() <= 1.12 * 0.392 * math.hypot(u * float(t[0].norm()), 2.0 ** -11 * float(t[-1].norm())), float(err.norm() / t[0].norm() / u)


# ------------------------------------------------------------------------------------------- what a query does not see

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,H,KV,lens,news,window,first", [
    (128, 4, 1, [60, 200, 64], [60, 100, 33], 0, 0), (64, 8, 2, [60, 200, 64], [60, 100, 33], 0, 0), (128, 4, 1, [60, 400, 64], [60, 100, 33], 70, 3),
    (64, 40, 2, [90, 1, 50], [1, 1, 50], 0, 0), (128, 32, 8, [700] * 5, [500] * 5, 0, 0)])      # the last: two query tiles an item
@pytest.mark.parametrize("size", [1e3, 1e5, 1e30])
def test_later_rows_leave_earlier_queries_alone(kge, L, dtype, hd, H, KV, lens, news, window, first, size):
    """A key or a value behind a query, however large, changes no bit of its result, and what sees it stays as near to 64 bits as ever."""
    s = Batch(dtype, hd, H, KV, 16, lens, news).fill()
    before = s.run(kge, window, first)
    s.check(before, window, first)
    size = min(size, 6e3) if dtype == "fp16" else size              # (rows of up to 60000, with all the digits of their ends)
    at = {}
    for b, (n, new) in enumerate(zip(lens, news)):
        if new < 5:
            continue
        at[b] = n - new // 3                                         # in the same tile of 64 as queries before it
        s.k[b][at[b]] *= size ** (b % 2)
        s.v[b][at[b]] *= size
    after = s.fill().run(kge, window, first)
    for b, j in at.items():
        rows = slice(int(s.qsl[b]), int(s.qsl[b]) + j - (lens[b] - news[b]))
        assert torch.equal(after[rows], before[rows]), b
    s.check(after, window, first)


# ------------------------------------------------------------------------------------------------------ rows far apart

SINGLE = [(128, 4, 1, [150, 90, 64], [1, 1, 1]), (64, 12, 1, [900, 33], [1, 1]), (128, 16, 1, [70, 500], [1, 1]), (128, 32, 8, [1500, 700], [1, 1]),
          (128, 16, 1, [2000, 40], [1, 1]), (64, 10, 1, [1300], [1]), (128, 3, 1, [3100], [1])]      # the last three: shares of one group, many pieces
FAR = SINGLE + [(128, 4, 1, [150, 90, 64], [64, 90, 7]), (64, 40, 2, [150, 90, 64], [1, 90, 1]), (128, 32, 8, [300] * 6, [300] * 6)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
@pytest.mark.parametrize("window,first", [(0, 0), (40, 5)])
def test_values_of_all_sizes_in_one_tile(kge, L, dtype, hd, H, KV, lens, news, window, first):
    """Values from 10^-2 to 6 10^4 (float16) or 10^-14 to 10^14 (bfloat16), the larger ones under smaller weights; and keys likewise, under q
    that makes their scores ordinary."""
    s = Batch(dtype, hd, H, KV, 16, lens, news, seed=1)
    far = 2.0 if dtype == "fp16" else 14.0
    for b, n in enumerate(lens):
        e = torch.empty(n, 1, 1).uniform_(-far, far, generator=s.g)
        s.v[b] *= 10 ** (e + (1.5 if dtype == "fp16" else 0))
        s.k[b] = s.k[b] * 0.1
        s.k[b][..., 0] = -e[..., 0] * math.log(10) * 2 * hd ** 0.5 / 8       # weights fall as 10^(-2 e): exp(q k / hd^1/2) with q = 8
    s.q[..., 0] = 8
    s.check(s.fill().run(kge, window, first), window, first)


@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
def test_keys_of_all_sizes_in_one_tile(kge, L, hd, H, KV, lens, news):
    """Keys from 10^-9 to 10^3 of ordinary ones, so that scores run from none to steep ones."""
    s = Batch("bf16", hd, H, KV, 32, lens, news, seed=2)
    for b, n in enumerate(lens):
        s.k[b] *= 10 ** torch.empty(n, 1, 1).uniform_(-9, 3, generator=s.g)
    s.check(s.fill().run(kge))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
@pytest.mark.parametrize("steep", [43, 60, 75, 87])
@pytest.mark.parametrize("level", [0.0, 5.0, 1e20, 3e38])
def test_constant_values_under_steep_scores(kge, L, dtype, hd, H, KV, lens, news, steep, level):
    """Values whose rows have no range (s = 0), under weights of up to e^87 times those of all rows before: the weights' reference has to move for
    them too, since weight times s says nothing."""
    if dtype == "fp16":
        level = min(level, 6e4)
    s = Batch(dtype, hd, H, KV, 16, lens, news, seed=3)
    for b, n in enumerate(lens):
        s.k[b] *= 0.05
        s.k[b][..., 0] = 0
        s.v[b] *= 1e-3
        for j in (n - 1, 2 * n // 3, n // 2 + 1):
            s.k[b][j, :, 0] = steep * hd ** 0.5 / 8 * (1 if j == n - 1 else 0.97)
            s.v[b][j] = level
    s.q[..., 0] = 8
    out = s.fill().run(kge)
    assert torch.isfinite(out).all()
    s.check(out)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
@pytest.mark.parametrize("steep", [5, 30, 65, 87])
@pytest.mark.parametrize("small", [0.0, 1e-12, 1.0])
def test_small_values_under_steep_scores_behind_large_ones(kge, L, dtype, hd, H, KV, lens, news, steep, small):
    """The first third of a context has values of 10^30 (float16: 10^4), the rest small ones whose weights are up to e^87 times theirs: results from
    the one to the other, by scores alone."""
    s = Batch(dtype, hd, H, KV, 16, lens, news, seed=8)
    for b, n in enumerate(lens):
        s.k[b] *= 0.05
        s.k[b][..., 0] = 0
        s.k[b][n // 3:, :, 0] = steep * hd ** 0.5 / 8 * torch.linspace(0.2, 1, n - n // 3)[:, None]
        s.v[b][:n // 3] *= 1e4 if dtype == "fp16" else 1e30
        s.v[b][n // 3:] *= small
    s.q[..., 0] = 8
    out = s.fill().run(kge)
    assert torch.isfinite(out).all()
    s.check(out)


@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e18, 1e36])
def test_values_near_the_ends_of_their_type(kge, L, hd, H, KV, lens, news, size):
    s = Batch("bf16", hd, H, KV, 16, lens, news, seed=4)
    for b in range(len(lens)):
        s.v[b] *= size
    s.check(s.fill().run(kge))


@pytest.mark.parametrize("hd,H,KV,lens,news", SINGLE)
def test_heads_of_one_group_far_apart(kge, L, hd, H, KV, lens, news):
    """Single-token requests whose heads' q lie 10^12 apart: each is as exact as alone, and has the same bits."""
    s = Batch("bf16", hd, H, KV, 16, lens, news, seed=5).fill()
    s.q[:, 0] *= 1e12
    s.q[:, 2] *= 1e-12
    out = s.run(kge)
    s.check(out)
    s.q[:, 0] *= 1e-12
    again = s.run(kge)
    assert torch.equal(again[:, 1:], out[:, 1:])


@pytest.mark.parametrize("hd,H,KV,lens,news", FAR)
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e37])
@pytest.mark.parametrize("above", [8.2, 13.0])
def test_many_small_weights_beside_a_large_one(kge, L, hd, H, KV, lens, news, size, above):
    """One key lies e^8 or e^13 above all others, whose weights together still count, whatever the values' size."""
    s = Batch("bf16", hd, H, KV, 16, lens, news, seed=10)
    for b in range(len(lens)):
        s.k[b] *= 0.05
        s.k[b][..., 0] = 0
        s.k[b][min(3, lens[b] - 1), :, 0] = above * hd ** 0.5 / 8
        s.v[b] *= size
    s.q[..., 0] = 8
    s.check(s.fill().run(kge))


# ---------------------------------------------------------------------------------------------------- scores of any level

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,H,KV,lens,news", [
    (128, 4, 1, [1, 20, 64, 200], [1, 1, 1, 1]), (64, 12, 1, [900, 1], [1, 1]), (128, 16, 1, [3, 500], [1, 1]), (128, 32, 8, [1500], [1]), (64, 16, 2, [1300, 1], [1, 1]),
    (128, 4, 1, [5, 90, 64], [5, 90, 7]), (64, 40, 2, [1, 90], [1, 90]), (128, 32, 8, [300] * 6, [300] * 6)])
@pytest.mark.parametrize("level", [-1e6, -200, 200, 1e6])
def test_all_scores_far_from_zero(kge, L, dtype, hd, H, KV, lens, news, level):
    """Every score of a context lies about one level, far below or above zero: the first reference comes from there."""
    s = Batch(dtype, hd, H, KV, 16, lens, news, seed=9)
    for b in range(len(lens)):
        s.k[b] *= 0.05
        s.k[b][..., 0] = math.copysign(64, level)
    s.q[..., 0] = 8
    scale = abs(level) / 512                                         # the level is q k = 8 x 64 times that
    out = s.fill().run(kge, scale=scale)
    assert torch.isfinite(out).all()
    s.check(out, scale=scale)


# -------------------------------------------------------------------------------------------- two query tiles of an item

MANY = [  # dtype, hd, H, KV, block, lengths, rows
    ("bf16", 128, 32, 8, 64, [700, 333, 150, 900], [700, 201, 150, 650]), ("fp16", 128, 32, 8, 16, [515, 640, 300], [515, 500, 300]),
    ("bf16", 64, 64, 64, 32, [300, 299, 140], [300, 280, 129]), ("fp16", 64, 48, 16, 16, [411, 200, 390], [411, 200, 160]),
    ("bf16", 128, 80, 4, 16, [270, 150, 333], [270, 101, 150]), ("fp16", 128, 40, 10, 128, [333, 640, 250], [333, 401, 250])]


def tiles_of(H, KV, news):
    """(query tiles of an item, whether some item has tokens in its second one), as the launch decides for at most 300 x 128 rows."""
    TT, B, T = 128 // (H // KV), len(news), sum(news)
    tiles = -(-max(news) // (2 * TT))
    items = KV * (T // (2 * TT) + B) if tiles > 65535 or 2 * (T // (2 * TT) + B) < tiles * B else KV * B * tiles
    return (1 if items <= 74 or items <= 148 else 2), any(n % (2 * TT) > TT or n >= 2 * TT for n in news)


@pytest.mark.parametrize("dtype,hd,H,KV,bs,lens,news", MANY)
@pytest.mark.parametrize("window,first", [(0, 0), (100, 4), (64, 0), (7, 130), (400, 70)])
def test_prompts_of_two_query_tiles_an_item(kge, L, dtype, hd, H, KV, bs, lens, news, window, first):
    """Enough items that each has two query tiles, walks of unequal length, odd tails and several items a CTA."""
    assert tiles_of(H, KV, news) == (2, True)
    s = Batch(dtype, hd, H, KV, bs, lens, news, seed=6).fill()
    out = s.run(kge, window, first)
    s.check(out, window, first, norm=True)
    assert torch.equal(out, s.run(kge, window, first))               # the same bits again


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("news", [[1, 1, 1], [300, 100, 77]])
def test_errors_are_the_roundings_alone(kge, L, dtype, news):
    """In the 2-norm: the result's rounding and that of weights to float16, in either type."""
    s = Batch(dtype, 128, 32, 8, 16, [1500, 200, 900], news, seed=7).fill()
    s.check(s.run(kge), norm=True)
    s.check(s.run(kge, 130, 7), 130, 7, norm=True)
