"""The operators of 8-bit floating point with a scale for each block of 128, as they are timed and checked: rows of activations and matrices
of weights quantised, the matrix product of the two, the same grouped by expert with ragged sizes, and both with a gated pair whose result is
quantised for the product behind it.

  quant    16-bit rows -> e4m3 codes and a scale for each row and 128 columns; rows may be gathered (tokens sorted by expert)
  weight   16-bit matrices -> e4m3 codes and a scale for each block of 128 x 128
  gemm     y = x w^T from codes and scales, with an optional bias, in 16 bits
  glu      h = silu(x w_gate^T) * (x w_up^T), quantised as `quant` quantises rows
  experts  either of the two with rows in groups: group e has rows offsets[e] .. offsets[e + 1] and its own matrix

A block of numbers with the largest magnitude m has the scale s = max(m / 448, 2^-126), held in fp32, and a number x of it the code that is
nearest to 448 x / m (to 2^126 x where m is below 448 2^-126) in e4m3, ties to even.  Scales of rows lie by columns, [ceil(K / 128), rows];
those of weights as [ceil(N / 128), ceil(K / 128)].
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
LEAST = 2.0 ** -126                      # the smallest scale


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    quant = dict(kind="quant", dtype="bf16", gather=0)
    gemm = dict(kind="gemm", dtype="bf16", bias=False)
    experts = dict(kind="experts", dtype="bf16", pad=0)
    return [
        # the normed rows of a decode step of 64 requests, 8B model
        dict(quant, name="quant-decode-64", rows=64, K=4096),
        # the tokens of a prompt step, each for the eight experts that it goes to: rows sorted by expert
        dict(quant, name="quant-sorted-16k", dtype="fp16", rows=16384, K=2048, gather=2048),
        # the 8B model's gate and up projections, when a 16-bit checkpoint is loaded
        dict(kind="weight", name="weight-8b-gate-up", dtype="bf16", E=1, N=28672, K=4096),
        # a few experts whose sizes are no multiples of 128
        dict(kind="weight", name="weight-odd-experts", dtype="fp16", E=6, N=1000, K=1424),
        # the 8B model's attention projections in a decode step of 64 requests
        dict(gemm, name="gemm-decode-64", T=64, N=6144, K=4096),
        # a single request's down projection
        dict(gemm, name="gemm-decode-1", dtype="fp16", T=1, N=4096, K=14336),
        # a chunk of a prompt beside decode rows, biased projections, no size a multiple of 128
        dict(gemm, name="gemm-odd-333", T=333, N=2504, K=2064, bias=True),
        # the down projection of a prompt step with a token budget of 8192
        dict(gemm, name="gemm-prompt-8192", T=8192, N=4096, K=14336),
        # gate and up projections of a decode step and of a prompt step
        dict(kind="glu", name="glu-decode-64", T=64, f=14336, K=4096),
        dict(kind="glu", name="glu-prompt-8192", T=8192, f=14336, K=4096),
        # a decode step of 64 tokens through a mixture of 128 experts, eight a token: few rows an expert
        dict(experts, name="experts-decode-64", glu=True, E=128, tokens=64, top=8, N=1536, K=2048),
        # the experts' second product in a prompt step, a few padded rows behind the last expert
        dict(experts, name="experts-prompt-2048", glu=False, E=64, tokens=2048, top=6, N=2048, K=1408, pad=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "quant", "weight", "gemm", "gemm", "gemm", "glu", "glu", "experts", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    K = rng.choice([16 * _log(rng, 16, 896), 128 * _log(rng, 2, 112)])
    if kind == "quant":
        rows = _log(rng, 1, min(16384, 60_000_000 // K))
        return dict(kind=kind, dtype=dtype, rows=rows, K=K, gather=rng.choice([0, 0, max(1, rows // rng.choice([2, 6, 8]))]))
    if kind == "weight":
        E = rng.choice([1, 1, _log(rng, 2, 32)])
        return dict(kind=kind, dtype=dtype, E=E, N=_log(rng, 64, max(65, min(28672, 110_000_000 // (E * K)))), K=K)
    if kind == "gemm":
        N = rng.choice([8 * _log(rng, 8, 3584), 128 * _log(rng, 1, 224), _log(rng, 64, 5000)])
        N = min(N, 110_000_000 // K)
        return dict(kind=kind, dtype=dtype, T=_log(rng, 1, max(2, min(8192, 450_000_000_000 // (N * K)))), N=N, K=K, bias=rng.random() < 0.3)
    if kind == "glu":
        f = 128 * _log(rng, 1, 112)
        K = min(K, 60_000_000 // f // 16 * 16)
        return dict(kind=kind, T=_log(rng, 1, max(2, min(8192, 220_000_000_000 // (f * K)))), f=f, K=K)
    E, glu = _log(rng, 4, 256), rng.random() < 0.5
    K = rng.choice([16 * _log(rng, 16, 256), 128 * _log(rng, 2, 32)])
    N = rng.choice([256 * _log(rng, 1, 16), 256 * _log(rng, 1, 16) if glu else _log(rng, 100, 4000)])
    while E * N * K > 420_000_000:
        E //= 2
    top = min(E, rng.choice([1, 2, 4, 6, 8]))
    tokens = _log(rng, 1, max(2, min(24576 // top, 100_000_000_000 // (top * N * K))))
    return dict(kind=kind, dtype=dtype, glu=glu, E=E, tokens=tokens, top=top, N=N, K=K, pad=rng.choice([0, 0, rng.randint(1, 40)]))


# ----------------------------------------------------------------------------------------------------- inputs, shared

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(2_000_003 + seed)


def _rows(g, rows, K, dt):
    """Activations: a few columns much larger than the others, rows of different size."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    col = torch.rand(K, generator=g, device="cuda")
    x *= torch.where(col < 0.01, 20.0, 1.0) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(dt)


def _weights(g, N, K, dt):
    w = torch.randn(N, K, generator=g, device="cuda")
    w *= K ** -0.5 * torch.exp(0.3 * torch.randn(N, 1, generator=g, device="cuda"))
    return w.to(dt)


def _blocks(x, rows):
    """[N, K] -> [ceil(N / rows), rows, ceil(K / 128), 128], with zeros behind the ends."""
    N, K = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -N % rows))
    return x.unflatten(-1, (-1, 128)).unflatten(-3, (-1, rows))


def _quantise(x, rows):
    """[..., N, K] -> codes (e4m3) and scales [..., ceil(N / rows), ceil(K / 128)]."""
    N, K = x.shape[-2:]
    b = _blocks(x.float(), rows)
    m = b.abs().amax((-3, -1), keepdim=True)
    s = torch.clamp(m / torch.full_like(m, 448.0), min=LEAST)
    code = (b.double() * 448.0 / m.double().clamp(min=448.0 * LEAST)).to(E4M3)            # (halves of a step are kept apart from what lies next to them)
    return code.flatten(-2).flatten(-3, -2)[..., :N, :K].contiguous(), s.squeeze(-1).squeeze(-2)


def _numbers(code, s, rows):
    """Codes [..., N, K] and scales [..., ceil(N / rows), ceil(K / 128)] -> the numbers that they stand for, in fp32."""
    N, K = code.shape[-2:]
    return code.float() * s.repeat_interleave(rows, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]


def _quantised_weights(g, E, N, K, dt):
    """[E, N, K] codes and [E, ceil(N / 128), ceil(K / 128)] scales, a matrix at a time."""
    code = torch.empty(E, N, K, dtype=E4M3, device="cuda")
    s = torch.empty(E, -(-N // 128), -(-K // 128), device="cuda")
    for e in range(E):
        code[e], s[e] = _quantise(_weights(g, N, K, dt), 128)
    return code, s


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


def _workspace():
    return torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")


def _nearest(v):
    """Numbers in 64 bits, at most 448 -> the nearest of e4m3, ties to even."""
    step = torch.exp2(torch.clamp(torch.frexp(v.abs()).exponent - 1, min=-6).double() - 3)
    return torch.round(v / step) * step


# -------------------------------------------------------------------------------------------------- quant and weight

def _quant_inputs(case, seed):
    g = _gen(seed)
    x = _rows(g, case["gather"] or case["rows"], case["K"], DT[case["dtype"]])
    at = torch.randint(0, case["gather"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32) if case["gather"] else None
    return dict(x=x, at=at)


def _quant_prepare(case, seed):
    st = dict(_quant_inputs(case, seed), case=case)
    st["codes"] = torch.zeros(case["rows"], case["K"], dtype=E4M3, device="cuda")
    st["scales"] = torch.zeros(-(-case["K"] // 128), case["rows"], device="cuda")
    return st


def _quant_run(st):
    c = st["case"]
    if own:
        _call(st, _name(c, "kge_fp8_quant"), st["codes"], st["scales"], c["rows"], st["x"], c["K"], st["at"], c["rows"], c["K"])
    else:
        code, s = _quantise(st["x"] if st["at"] is None else st["x"][st["at"].long()], 1)
        st["codes"].copy_(code)
        st["scales"].copy_(s.t())
    return {"codes": st["codes"], "scales": st["scales"]}


def _quant_exact(case, seed):
    i = _quant_inputs(case, seed)
    x = i["x"].double() if i["at"] is None else i["x"].double()[i["at"].long()]
    code, scales = torch.empty_like(x), []
    for k in range(0, case["K"], 128):
        part = x[:, k:k + 128]
        m = torch.clamp(part.abs().amax(1), min=448.0 * LEAST)
        code[:, k:k + 128] = _nearest(448.0 * part / m[:, None])
        scales.append(m / 448.0)
    return {"codes": code, "scales": torch.stack(scales)}


def _quant_work(case):
    T, K = case["rows"], case["K"]
    return {"bytes": 2.0 * (case["gather"] or T) * K + T * K + 4.0 * T * -(-K // 128) + (4.0 * T if case["gather"] else 0), "flops": 4.0 * T * K}


def _weight_inputs(case, seed):
    g = _gen(seed)
    return torch.stack([_weights(g, case["N"], case["K"], DT[case["dtype"]]) for _ in range(case["E"])])


def _weight_prepare(case, seed):
    E, N, K = case["E"], case["N"], case["K"]
    return dict(case=case, w=_weight_inputs(case, seed), codes=torch.zeros(E, N, K, dtype=E4M3, device="cuda"),
                scales=torch.zeros(E, -(-N // 128), -(-K // 128), device="cuda"))


def _weight_run(st):
    c = st["case"]
    if own:
        _call(st, _name(c, "kge_fp8_quant_weight"), st["codes"], st["scales"], st["w"], c["E"], c["N"], c["K"])
    else:
        code, s = _quantise(st["w"], 128)
        st["codes"].copy_(code)
        st["scales"].copy_(s)
    return {"codes": st["codes"], "scales": st["scales"]}


def _weight_exact(case, seed):
    w = _weight_inputs(case, seed).double()
    code, scales = torch.empty_like(w), torch.empty(case["E"], -(-case["N"] // 128), -(-case["K"] // 128), dtype=torch.float64, device="cuda")
    for n in range(0, case["N"], 128):
        for k in range(0, case["K"], 128):
            part = w[:, n:n + 128, k:k + 128]
            m = torch.clamp(part.abs().amax((1, 2)), min=448.0 * LEAST)
            code[:, n:n + 128, k:k + 128] = _nearest(448.0 * part / m[:, None, None])
            scales[:, n // 128, k // 128] = m / 448.0
    return {"codes": code, "scales": scales}


def _weight_work(case):
    E, N, K = case["E"], case["N"], case["K"]
    return {"bytes": 3.0 * E * N * K + 4.0 * E * -(-N // 128) * -(-K // 128), "flops": 4.0 * E * N * K}


# --------------------------------------------------------------------------------------------------------------- gemm

def _gemm_inputs(case, seed):
    """Activations and weights as the product finds them: codes and scales."""
    g, dt = _gen(seed), DT[case.get("dtype", "bf16")]
    N = 2 * case["f"] if case["kind"] == "glu" else case["N"]
    x, xs = _quantise(_rows(g, case["T"], case["K"], dt), 1)
    w, ws = _quantised_weights(g, 1, N, case["K"], dt)
    bias = torch.randn(N, generator=g, device="cuda").to(dt) if case.get("bias") else None
    return dict(x=x, xs=xs.t().contiguous(), w=w[0], ws=ws[0], bias=bias)


def _gemm_prepare(case, seed):
    st = dict(_gemm_inputs(case, seed), case=case, work=_workspace())
    T = case["T"]
    if case["kind"] == "glu":
        st["codes"] = torch.zeros(T, case["f"], dtype=E4M3, device="cuda")
        st["scales"] = torch.zeros(case["f"] // 128, T, device="cuda")
    else:
        st["y"] = torch.zeros(T, case["N"], dtype=DT[case["dtype"]], device="cuda")
    return st


def _gated(z):
    """[..., 2 f] -> silu(gate) * up."""
    a, b = z.chunk(2, -1)
    return a / (1 + torch.exp(-a)) * b


def _gemm_run(st):
    c = st["case"]
    T, K = c["T"], c["K"]
    if c["kind"] == "glu":
        if own:
            _call(st, "kge_gemm_fp8_silu_gate", st["codes"], st["scales"], T, st["x"], st["xs"], T, st["w"], st["ws"], T, c["f"], K, st["work"], st["work"].numel())
        else:
            code, s = _quantise(_gated(_numbers(st["x"], st["xs"].t(), 1) @ _numbers(st["w"], st["ws"], 128).t()), 1)
            st["codes"].copy_(code)
            st["scales"].copy_(s.t())
        return {"codes": st["codes"], "scales": st["scales"]}
    if own:
        _call(st, _name(c, "kge_gemm_fp8"), st["y"], st["x"], st["xs"], T, st["w"], st["ws"], st["bias"], T, c["N"], K, st["work"], st["work"].numel())
    else:
        z = _numbers(st["x"], st["xs"].t(), 1) @ _numbers(st["w"], st["ws"], 128).t()
        st["y"].copy_(z if st["bias"] is None else z + st["bias"].float())
    return st["y"]


def _product64(x, xs, w, ws):
    """x w^T in 64 bits, block of K by block of K: codes [T, K] and [N, K], scales [blocks of K, T] and [blocks of N, blocks of K]."""
    z = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    block = torch.arange(w.shape[0], device="cuda") // 128
    for b in range(xs.shape[0]):
        k = slice(128 * b, 128 * b + 128)
        z.addmm_(x[:, k].double() * xs[b].double()[:, None], (w[:, k].double() * ws.double()[block, b][:, None]).t())
    return z


def _quantised64(h):
    """Rows in 64 bits -> codes and scales [f / 128, T]."""
    part = h.unflatten(1, (-1, 128))
    m = torch.clamp(part.abs().amax(-1), min=448.0 * LEAST)
    return {"codes": _nearest(448.0 * part / m[..., None]).flatten(1), "scales": (m / 448.0).t().contiguous()}


def _gemm_exact(case, seed):
    i = _gemm_inputs(case, seed)
    z = _product64(i["x"], i["xs"], i["w"], i["ws"])
    if case["kind"] == "gemm":
        return z if i["bias"] is None else z + i["bias"].double()
    gate, up = z[:, :case["f"]], z[:, case["f"]:]
    return _quantised64(gate * torch.sigmoid(gate) * up)


def _gemm_work(case):
    T, K, glu = case["T"], case["K"], case["kind"] == "glu"
    N = 2 * case["f"] if glu else case["N"]
    kb = -(-K // 128)
    out = T * case["f"] * (1 + 4 / 128) if glu else 2.0 * T * N
    return {"bytes": 1.0 * T * K + 1.0 * N * K + 4.0 * kb * (T + -(-N // 128)) + out, "flops": 2.0 * T * N * K}


# ------------------------------------------------------------------------------------------------------------ experts

def _sizes(case, seed):
    """Rows of each expert: every token goes to `top` different ones, some of which are more popular than others."""
    r = np.random.default_rng(seed + 29)
    liking = r.normal(size=case["E"]) * 0.7 + r.gumbel(size=(case["tokens"], case["E"]))
    chosen = np.argsort(-liking, axis=1)[:, :case["top"]]
    return np.bincount(chosen.ravel(), minlength=case["E"])


def _experts_inputs(case, seed):
    g, dt = _gen(seed), DT[case["dtype"]]
    sizes = _sizes(case, seed)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")
    x, xs = _quantise(_rows(g, int(sizes.sum()) + case["pad"], case["K"], dt), 1)
    w, ws = _quantised_weights(g, case["E"], case["N"], case["K"], dt)
    return dict(x=x, xs=xs.t().contiguous(), w=w, ws=ws, offsets=offsets, sizes=sizes)


def _experts_prepare(case, seed):
    st = dict(_experts_inputs(case, seed), case=case, work=_workspace())
    st["T"], st["most"] = st["x"].shape[0], max(1, int(st["sizes"].max()))
    f = case["N"] // 2
    if case["glu"]:
        st["codes"] = torch.zeros(st["T"], f, dtype=E4M3, device="cuda")
        st["scales"] = torch.zeros(f // 128, st["T"], device="cuda")
    else:
        st["y"] = torch.zeros(st["T"], case["N"], dtype=DT[case["dtype"]], device="cuda")
    return st


def _experts_plain(st):
    """The experts' products as one batched product of rows padded to the longest group."""
    E, most, off = st["case"]["E"], st["most"], st["offsets"].long()
    n = int(st["sizes"].sum())
    row = torch.arange(n, device="cuda")
    e = torch.searchsorted(off[1:], row, right=True)
    at = e * most + row - off[e]
    x = torch.zeros(E * most, st["case"]["K"], device="cuda")
    x[at] = _numbers(st["x"][:n], st["xs"].t()[:n], 1)
    z = torch.bmm(x.view(E, most, -1), _numbers(st["w"], st["ws"], 128).transpose(1, 2)).flatten(0, 1)[at]
    if st["case"]["glu"]:
        code, s = _quantise(_gated(z), 1)
        st["codes"][:n] = code
        st["scales"][:, :n] = s.t()
    else:
        st["y"][:n] = z.to(st["y"].dtype)


def _experts_run(st):
    c, T = st["case"], st["T"]
    if own:
        sizes = (c["N"] // 2 if c["glu"] else c["N"]), c["K"]
        inputs = st["x"], st["xs"], T, st["w"], st["ws"], st["offsets"], c["E"], T, *sizes, st["work"], st["work"].numel()
        if c["glu"]:
            _call(st, "kge_gemm_fp8_grouped_silu_gate", st["codes"], st["scales"], T, *inputs)
        else:
            _call(st, _name(c, "kge_gemm_fp8_grouped"), st["y"], *inputs)
    else:
        _experts_plain(st)
    return {"codes": st["codes"], "scales": st["scales"]} if c["glu"] else st["y"]


def _experts_exact(case, seed):
    i = _experts_inputs(case, seed)
    T, f, at = i["x"].shape[0], case["N"] // 2, 0
    z = torch.zeros(T, f if case["glu"] else case["N"], dtype=torch.float64, device="cuda")
    s = torch.zeros(f // 128, T, dtype=torch.float64, device="cuda")
    for e, n in enumerate(i["sizes"].tolist()):
        rows = slice(at, at + n)
        at += n
        if not n:
            continue
        y = _product64(i["x"][rows], i["xs"][:, rows], i["w"][e], i["ws"][e])
        if case["glu"]:
            q = _quantised64(y[:, :f] * torch.sigmoid(y[:, :f]) * y[:, f:])
            y, s[:, rows] = q["codes"], q["scales"]
        z[rows] = y
    return {"codes": z, "scales": s} if case["glu"] else z


def _experts_work(case, seed=0):
    sizes = _sizes(case, seed)
    n, some, N, K = int(sizes.sum()), int((sizes > 0).sum()), case["N"], case["K"]
    kb = -(-K // 128)
    out = n * N / 2 * (1 + 4 / 128) if case["glu"] else 2.0 * n * N
    return {"bytes": 1.0 * n * K + some * (1.0 * N * K + 4.0 * kb * -(-N // 128)) + 4.0 * kb * n + out + 4.0 * case["E"], "flops": 2.0 * n * N * K}


# ----------------------------------------------------------------------------------------------------------- the calls

_KINDS = {"quant": (_quant_prepare, _quant_run, _quant_exact, _quant_work), "weight": (_weight_prepare, _weight_run, _weight_exact, _weight_work),
          "gemm": (_gemm_prepare, _gemm_run, _gemm_exact, _gemm_work), "glu": (_gemm_prepare, _gemm_run, _gemm_exact, _gemm_work),
          "experts": (_experts_prepare, _experts_run, _experts_exact, _experts_work)}


def prepare(case, seed):
    return _KINDS[case["kind"]][0](case, seed)


def run(st):
    return _KINDS[st["case"]["kind"]][1](st)


def exact(case, seed):
    return _KINDS[case["kind"]][2](case, seed)


def work(case):
    return _KINDS[case["kind"]][3](case)
