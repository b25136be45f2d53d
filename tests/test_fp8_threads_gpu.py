"""8-bit products from two threads of a program at once, each with a stream and a workspace of its own, whose kernels are one function with different amounts of
shared memory: no launch is refused and each has the results that it has alone."""
import threading

import pytest
import torch

from test_fp8_gpu import L, call, quantised, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


def job(kge, L, form, T, N, K, off):
    """A call with these sizes and its result's tensors; `off`: elements that y begins behind a 16-byte boundary."""
    g = torch.Generator().manual_seed(T)
    E = 1 if form == "gated" else 3
    x, xs, _ = quantised(g, T, K, 1)
    w, ws, _ = quantised(g, N * (2 if "gated" in form else 1), K, 128)
    w, ws = torch.stack([w] * E).cuda(), torch.stack([ws] * E).cuda()
    args = [x.cuda(), xs.t().contiguous().cuda(), T, w, ws]
    if E > 1:
        args += [torch.tensor([0, T // 2, T // 2, T], dtype=torch.int32, device="cuda"), E]
    work = workspace(L, T)
    args += [T, N, K, work, work.numel()]
    if "gated" in form:
        out = torch.zeros(T, N, dtype=torch.uint8, device="cuda"), torch.zeros(N // 128, T, device="cuda")
        return out, "kge_gemm_fp8_" + ("grouped_" if E > 1 else "") + "silu_gate", [*out, T, *args]
    y = torch.zeros(T * N + 8, dtype=torch.bfloat16, device="cuda")
    return (y,), "kge_gemm_fp8_grouped", [y[off:], *args]


@pytest.mark.parametrize("form,N,K,one,two", [("gated", 9600, 256, (32, 0), (64, 0)), ("grouped gated", 256, 400, (20, 0), (100, 0)), ("grouped", 200, 272, (96, 0), (96, 1)),
                                              ("grouped", 10000, 272, (96, 0), (30, 3))], ids=lambda v: str(v).replace(" ", "-"))
def test_two_threads(kge, L, form, N, K, one, two):
    jobs = [job(kge, L, form, T, N, K, off) for T, off in (one, two)]
    alone = []
    for out, fn, args in jobs:
        call(kge, fn, *args)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in out])
        for t in out:
            t.zero_()
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(2)

    def run(fn, args):
        torch.cuda.set_device(0)
        stream = torch.cuda.Stream()
        fn, args = getattr(kge.lib(), fn), [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args] + [stream.cuda_stream]
        start.wait()
        for _ in range(40):
            failed.extend(kge.lib().kge_last_error() for _ in range(150) if fn(*args) != 0)
            stream.synchronize()
    threads = [threading.Thread(target=run, args=j[1:]) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, (len(failed), failed[0])
    assert all(torch.equal(a, b) for (out, *_), want in zip(jobs, alone) for a, b in zip(out, want))


def test_weights_written_by_one_thread_and_read_by_another(kge, L):
    """A matrix is quantised anew on a stream, the same thread launches on another stream, and another thread makes the products on the first: each has this turn's weights."""
    T, N, K, turns = 64, 4096, 1024, 60
    g = torch.Generator().manual_seed(3)
    x, xs, _ = quantised(g, T, K, 1)
    x, xs = x.cuda(), xs.t().contiguous().cuda()
    mats = [(torch.randn(N, K, generator=g) * 0.03 * (i + 1)).to(torch.bfloat16).cuda() for i in range(3)]
    cw, sw, other = torch.zeros(N, K, dtype=torch.uint8, device="cuda"), torch.zeros(N // 128, K // 128, device="cuda"), [torch.zeros(T, K, dtype=torch.uint8, device="cuda"), torch.zeros(K // 128, T, device="cuda")]
    rows, work = torch.randn(T, K, generator=g).to(torch.bfloat16).cuda(), workspace(L, T)
    want = []
    for m in mats:
        y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
        call(kge, "kge_fp8_quant_weight", cw, sw, m, 1, N, K)
        torch.cuda.synchronize()
        call(kge, "kge_gemm_fp8", y, x, xs, T, cw, sw, None, T, N, K, work, work.numel())
        want.append(y)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    out = [torch.zeros(T, N, dtype=torch.bfloat16, device="cuda") for _ in range(turns)]
    torch.cuda.synchronize()
    for i in range(turns):
        call(kge, "kge_fp8_quant_weight", cw, sw, mats[i % 3], 1, N, K, stream=a)
        call(kge, "kge_fp8_quant", *other, T, rows, K, None, T, K, stream=b)
        t = threading.Thread(target=call, args=(kge, "kge_gemm_fp8", out[i], x, xs, T, cw, sw, None, T, N, K, work, work.numel()), kwargs=dict(stream=a))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(out))
