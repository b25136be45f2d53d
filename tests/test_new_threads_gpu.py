"""An entry point may be the first thing that a new thread does with the GPU: what tensor maps need is there, as it is for launches.  Buffers are new in each test, so
that no map is remembered."""
import threading

import pytest
import torch

from test_fp8_gpu import call, quantised, workspace

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def product16(kge, T, N, K):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randn(n, K, generator=g, device="cuda").to(torch.bfloat16) for n in (T, N))
    return lambda: torch.zeros(T, N, dtype=torch.bfloat16, device="cuda"), "kge_gemm_bf16", lambda y: (y, x, w, None, T, N, K, 0, None, 0)


def product8(kge, T, N, K, groups):
    g = torch.Generator().manual_seed(2)
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N, K, 128)
    E = max(groups, 1)
    args = [x.cuda(), xs.t().contiguous().cuda(), T, torch.stack([w] * E).cuda(), torch.stack([ws] * E).cuda()]
    args += [torch.arange(E + 1, **I32) * (T // E), E] if groups else [None]
    work = workspace(kge.lib(), T)
    args += [T, N, K, work, work.numel()]
    return lambda: torch.zeros(T, N, dtype=torch.bfloat16, device="cuda"), "kge_gemm_fp8" + ("_grouped" if groups else ""), lambda y: (y, *args)


def prompt(kge, H, KV, hd, bs, T):
    g = torch.Generator(device="cuda").manual_seed(3)
    n = -(-T // bs)
    kc, vc = (torch.randn(n + 1, KV, bs, hd, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    qkv = torch.randn(T, (H + 2 * KV) * hd, generator=g, device="cuda").to(torch.bfloat16)
    table, lens, qsl = torch.arange(1, n + 1, **I32), torch.tensor([T], **I32), torch.tensor([0, T], **I32)
    return (lambda: torch.zeros(T, H * hd, dtype=torch.bfloat16, device="cuda"), "kge_paged_attn",
            lambda out: (out, qkv, qkv.shape[1], kc, vc, table, n, lens, qsl, 1, T, T, T, H, KV, hd, bs, hd ** -0.5, None, 0))


@pytest.mark.parametrize("make", [lambda k: product16(k, 128, 1024, 1024), lambda k: product16(k, 1024, 2048, 512), lambda k: product8(k, 16, 2048, 1024, 0), lambda k: product8(k, 700, 2048, 512, 0),
                                  lambda k: product8(k, 60, 512, 256, 3), lambda k: product8(k, 600, 512, 256, 3), lambda k: prompt(k, 32, 8, 128, 64, 600)],
                         ids=["16 bits", "16 bits, many rows", "8 bits", "8 bits, many rows", "8 bits, groups", "8 bits, large groups", "prompt"])
def test_first_call_of_a_thread(kge, make):
    kge.require_cuda()
    out, name, args = make(kge)
    one, two = out(), out()
    torch.cuda.synchronize()
    fn, failed = getattr(kge.lib(), name), []
    flat = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args(one)] + [None]

    def first():
        if fn(*flat) != 0:
            failed.append(kge.lib().kge_last_error().decode())
    t = threading.Thread(target=first)
    t.start()
    t.join()
    assert not failed, failed
    torch.cuda.synchronize()
    call(kge, name, *args(two))
    torch.cuda.synchronize()
    assert torch.equal(one, two) and one.abs().sum() > 0
