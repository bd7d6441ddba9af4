"""The 8-bit operators and the fused norm quantiser: cases, inputs and plain forms.

`run(state)` computes one pass: with `own` false in elementary torch operations, with `own` true by the
calls a program makes of mixedgemm_b200.  The kinds of cases:

  product       matmul_int8 on codes and scales that are already in hand
  quantise      quantize_int8 of rows (weights by channel, activations by token)
  linear        quantize_int8 of the activation, then matmul_int8: a projection without a norm in front
  norm          rms_norm_int8 with the residual's addition
  norm_linear   rms_norm_int8, then matmul_int8: a norm and the projections behind it
  mx_linear     rms_norm_reorder_quantize_x, then matmul: the same with MXFP4 / 6 / 8 codes

Codes of a case that ends with them are returned as the values they stand for.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TINY = 2.0 ** -100  # a row's largest magnitude counts as at least this much

# ------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one token through a 4096 x 4096 projection: latency of the product alone
        dict(name="product-1x4096x4096", kind="product", M=1, N=4096, K=4096, dtype="bf16", bias=False),
        # a decode batch through the gate projection: bound by the weights' bytes
        dict(name="product-64x14336x4096", kind="product", M=64, N=14336, K=4096, dtype="bf16", bias=False),
        # nothing a multiple of anything: a pruned layer with a bias, fp16 results
        dict(name="product-333x1537x1931", kind="product", M=333, N=1537, K=1931, dtype="fp16", bias=True),
        # the large square of this repository's sweep
        dict(name="product-8192x8192x8192", kind="product", M=8192, N=8192, K=8192, dtype="bf16", bias=False),
        # quantising the gate projection's weights by output channel
        dict(name="quantise-14336x4096", kind="quantise", M=14336, K=4096, dtype="bf16"),
        # a decode batch through the down projection
        dict(name="linear-16x4096x14336", kind="linear", M=16, N=4096, K=14336, dtype="bf16", bias=False),
        # a prefill through the output projection, fp16 model
        dict(name="linear-2048x4096x4096", kind="linear", M=2048, N=4096, K=4096, dtype="fp16", bias=True),
        # the norm of a long prefill at the larger hidden size
        dict(name="norm-8192x8192", kind="norm", M=8192, K=8192, dtype="bf16", residual=True),
        # one token: norm, then q, k and v as one product
        dict(name="norm-linear-1x6144x4096", kind="norm_linear", M=1, N=6144, K=4096, dtype="bf16", residual=True),
        # a prefill: norm, then gate and up as one product
        dict(name="norm-linear-2048x28672x4096", kind="norm_linear", M=2048, N=28672, K=4096, dtype="bf16",
             residual=True),
        # a decode batch of the MX path: norm, then q, k and v as one product
        dict(name="mx-linear-8x6144x4096", kind="mx_linear", M=8, N=6144, K=4096, dtype="bf16", residual=True),
        # a prefill of the MX path: norm, then the gate projection
        dict(name="mx-linear-2048x14336x4096", kind="mx_linear", M=2048, N=14336, K=4096, dtype="bf16", residual=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "quantise", "linear", "norm", "norm_linear", "mx_linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("quantise", "norm"):
        K = _spread(rng, 64, 16384)
        M = _spread(rng, 1, min(16384, 2 ** 26 // K))
        case = dict(kind=kind, M=M, K=K, dtype=dtype)
        if kind == "norm":
            case["residual"] = rng.random() < 0.7
        return case
    if kind == "mx_linear":
        K = 2048 * rng.randint(1, 7)
        M = _spread(rng, 1, 2048)
        N = 128 * _spread(rng, 1, 112)
        return dict(kind=kind, M=M, N=N, K=K, dtype="bf16", residual=rng.random() < 0.7)
    K = _spread(rng, 64, 16384)
    M = _spread(rng, 1, 8192)
    N = _spread(rng, 16, 16384)
    while M * N * K > 2 ** 38:
        M = max(1, M // 2)
    case = dict(kind=kind, M=M, N=N, K=K, dtype=dtype)
    if kind == "norm_linear":
        case["residual"] = rng.random() < 0.7
    else:
        case["bias"] = rng.random() < 0.4
    return case


def work(case):
    kind, M, K = case["kind"], case["M"], case["K"]
    e = SIZE[case["dtype"]]
    stream = M * K * e * (3 if case.get("residual") else 1)  # x; the residual in and out
    if kind == "quantise":
        return {"bytes": M * K * (e + 1) + 4 * M, "flops": 3 * M * K}
    if kind == "norm":
        return {"bytes": stream + K * e + M * K + 4 * M, "flops": 6 * M * K}
    N = case["N"]
    out = M * N * (2 if kind == "norm_linear" else e)
    product = 2.0 * M * N * K
    if kind == "mx_linear":  # 4-bit weights with a scale byte per 32
        return {"bytes": stream + 2 * K + 2 * K + N * K // 2 + N * K // 32 + out, "flops": product}
    weights = N * K + 4 * N + (4 * N if case.get("bias") else 0)
    if kind == "product":
        return {"bytes": M * K + 4 * M + weights + out, "flops": product}
    if kind == "linear":
        return {"bytes": M * K * e + weights + out, "flops": product}
    return {"bytes": stream + K * e + weights + out, "flops": product}


# ------------------------------------------------------------------------------------------ inputs


def _split(K):
    """62.5 / 34.375 / 3.125 % of the channels in 4, 6 and 8 bits."""
    KO = K // 32
    KN = K * 5 // 8
    return KN, K - KN - KO, KO


def _activation(M, K, dtype, g):
    """Tokens of different loudness; a few channels far above the others."""
    x = torch.randn(M, K, generator=g, device="cuda")
    loud = torch.randperm(K, generator=g, device="cuda")[:max(1, K // 32)]
    x[:, loud] *= 20
    x *= torch.exp2(torch.randn(M, 1, generator=g, device="cuda"))
    return x.to(dtype)


def _codes(rows, K, g):
    """int8 codes of normal values, rows 16-byte aligned, and a scale for each row."""
    q = (torch.randn(rows, K, generator=g, device="cuda") * 32).round_().clamp_(-127, 127)
    buf = torch.zeros(rows, (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    buf[:, :K] = q.to(torch.int8)
    scale = torch.exp2(torch.randn(rows, generator=g, device="cuda")) * 1e-3
    return buf[:, :K], scale


def _mx_weight(N, K, g):
    """MXFP4 weights as a program keeps them: nibbles (even element low) in rows padded to 128
    elements, one power-of-two scale byte for 32 elements in blocks of 128 rows x 4 scales."""
    code_of = torch.tensor([0, 2, 4, 5, 6, 6, 7], dtype=torch.uint8, device="cuda")  # of 0 1 2 3 4 4 6
    codes, scales = [], []
    for k in _split(K):
        v = (torch.randn(N, k, generator=g, device="cuda") * 2).round_().clamp_(-6, 6)
        c = code_of[v.abs().long()] | ((v < 0).to(torch.uint8) << 3)
        buf = torch.zeros(N, (k + 127) // 128 * 64, dtype=torch.uint8, device="cuda")
        buf[:, :k // 2] = c[:, 0::2] | (c[:, 1::2] << 4)
        codes.append(buf[:, :k // 2])
        nb, na = (N + 127) // 128, (k + 127) // 128
        s = torch.randint(119, 122, (nb * na * 512,), generator=g, device="cuda", dtype=torch.uint8)
        scales.append(s)
    return codes + scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, M, K = case["kind"], case["M"], case["K"]
    dtype = TYPES[case["dtype"]]
    s = dict(kind=kind, dtype=dtype, bias=None, residual=None)
    # an fp32 stream is quantised to the same 8 bits: what a norm's projections return is then bf16
    s["out"] = torch.bfloat16 if kind in ("norm", "norm_linear") and dtype == torch.float32 else dtype
    if kind == "product":
        s["a"], s["sa"] = _codes(M, K, g)
    elif kind == "quantise":
        s["x"] = (torch.randn(M, K, generator=g, device="cuda") * 0.02).to(dtype)
    else:
        s["x"] = _activation(M, K, dtype, g)
    if kind in ("norm", "norm_linear", "mx_linear"):
        s["norm"] = (1 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(dtype)
        if case.get("residual"):
            s["residual"] = _activation(M, K, dtype, g)
    if kind in ("product", "linear", "norm_linear"):
        s["b"], s["sb"] = _codes(case["N"], K, g)
        if case.get("bias"):
            s["bias"] = torch.randn(case["N"], generator=g, device="cuda")
    if kind == "mx_linear":
        s["w"] = _mx_weight(case["N"], K, g)
        s["split"] = _split(K)
        s["order"] = torch.randperm(K, generator=g, device="cuda").to(torch.int16)
    return s


# ------------------------------------------------------------------------- plain forms, in 32 bits


def _plain_quantise(v):
    """v fp32 [R, K] -> the codes as fp32 whole numbers, scale [R, 1]."""
    top = v.abs().amax(1, keepdim=True)
    fine = torch.isfinite(top)
    top = torch.where(fine, top, torch.ones_like(top)).clamp_min(TINY)
    full = torch.full_like(top, 127.0)
    q = torch.round(v * (full / top))
    nan = torch.full_like(top, float("nan"))
    return torch.where(fine, q, torch.zeros_like(q)), torch.where(fine, top / full, nan)


def _plain_norm(s):
    """The stream after the addition (in its own type) and the normalised values in fp32."""
    u = s["x"]
    if s["residual"] is not None:
        u = (u.float() + s["residual"].float()).to(u.dtype)
    f = u.float()
    r = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
    return u, f * r * s["norm"].float()


def _plain_product(a, sa, s):
    y = (a @ s["b"].float().t()) * sa * s["sb"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"])


def _to_grid(v, mantissa):
    """Whole numbers to the nearest value with `mantissa` bits after the leading one, ties to even."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1 - mantissa).float())
    return torch.round(v / step) * step


def _plain_mx_activation(h, split):
    """h [M, K], reordered -> the values that its 4-, 6- and 8-bit codes stand for."""
    parts = []
    at = 0
    for k, shift, border, mantissa in zip(split, (2, 4, 8), (1.5, 1.75, 1.75), (1, 2, 3)):
        v = h[:, at:at + k].reshape(h.shape[0], k // 32, 32)
        at += k
        top = v.abs().amax(2, keepdim=True)
        m, e = torch.frexp(top)
        e = e - 1 - shift + (2 * m > border).int()
        e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(-127, 127).float()
        t = v * torch.exp2(-e)
        n = torch.sign(t) * torch.floor(t.abs() + 0.5)
        if mantissa == 3:
            n = _to_grid(n, 7)
        parts.append((_to_grid(n, mantissa) * torch.exp2(e)).reshape(h.shape[0], k))
    return torch.cat(parts, 1)


def _plain_mx_weight(w, split):
    value_of = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    parts = []
    for k, c, sf in zip(split, w[:3], w[3:]):
        N = c.shape[0]
        v = value_of[torch.stack([c & 15, c >> 4], 2).long()].reshape(N, k // 32, 32)
        nb, na = (N + 127) // 128, (k + 127) // 128
        e = sf.view(nb, na, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(nb * 128, na * 4)[:N, :k // 32]
        parts.append((v * torch.exp2(e.float() - 127)[:, :, None]).reshape(N, k))
    return torch.cat(parts, 1)


def _plain(s):
    kind = s["kind"]
    if kind == "product":
        return {"y": _plain_product(s["a"].float(), s["sa"][:, None], s)}
    if kind == "quantise":
        q, scale = _plain_quantise(s["x"].float())
        return {"values": (q * scale).to(s["out"]), "scale": scale[:, 0]}
    if kind == "linear":
        q, scale = _plain_quantise(s["x"].float())
        return {"y": _plain_product(q, scale, s)}
    u, h = _plain_norm(s)
    got = {} if s["residual"] is None else {"residual": u}
    if kind == "norm":
        q, scale = _plain_quantise(h)
        return {"values": (q * scale).to(s["out"]), "scale": scale[:, 0], **got}
    if kind == "norm_linear":
        q, scale = _plain_quantise(h)
        return {"y": _plain_product(q, scale, s), **got}
    h = h.to(torch.bfloat16).float()[:, s["order"].long()]
    a = _plain_mx_activation(h, s["split"])
    return {"y": (a @ _plain_mx_weight(s["w"], s["split"]).t()).to(torch.bfloat16), **got}


# ------------------------------------------------------------------------------ the framework's calls


def _values(q, scale, dtype):
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    return torch.mul(q, scale[:, None], out=out)


def _own(s):
    import mixedgemm_b200 as mg
    kind = s["kind"]
    if kind == "product":
        return {"y": mg.matmul_int8(s["a"], s["b"], s["sa"], s["sb"], bias=s["bias"], out_dtype=s["out"])}
    if kind == "quantise":
        q, scale = mg.quantize_int8(s["x"])
        return {"values": _values(q, scale, s["out"]), "scale": scale}
    if kind == "linear":
        q, scale = mg.quantize_int8(s["x"])
        return {"y": mg.matmul_int8(q, s["b"], scale, s["sb"], bias=s["bias"], out_dtype=s["out"])}
    if kind == "mx_linear":
        got = mg.rms_norm_reorder_quantize_x(s["x"], s["norm"], s["order"], *s["split"], eps=EPS,
                                             residual=s["residual"])
        A, w = got[:6], s["w"]
        y = mg.matmul(A[0], w[0], A[1], w[1], A[2], w[2], A[3], w[3], A[4], w[4], A[5], w[5])
        return {"y": y} if s["residual"] is None else {"y": y, "residual": got[6]}
    q, scale, *u = mg.rms_norm_int8(s["x"], s["norm"], eps=EPS, residual=s["residual"])
    got = {} if s["residual"] is None else {"residual": u[0]}
    if kind == "norm":
        return {"values": _values(q, scale, s["out"]), "scale": scale, **got}
    return {"y": mg.matmul_int8(q, s["b"], scale, s["sb"], out_dtype=s["out"]), **got}


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------ in 64 bits


def _exact_rows(v):
    """Rows of float64 -> nearest multiples of (largest magnitude / 127), and that step."""
    top = torch.clamp(v.abs().max(dim=1).values, min=TINY)
    return torch.round(v * 127 / top[:, None]), top / 127


def _exact_round(v, bits):
    """Nearest value of `bits` significant bits, ties to even; 0 stays 0."""
    p = torch.floor(torch.log2(v.abs().clamp_min(1e-300)))
    p = p + (v.abs() >= 2 ** (p + 1)).double() - (v.abs() < 2 ** p).double()
    unit = 2 ** (p - bits + 1)
    return torch.round(v / unit) * unit


def _exact_mx_activation(h, split):
    out = torch.empty_like(h)
    at = 0
    for k, top, bits in zip(split, (6.0, 28.0, 448.0), (2, 3, 4)):
        v = h[:, at:at + k].unflatten(1, (-1, 32))
        peak = v.abs().max(dim=2, keepdim=True).values
        e = torch.ceil(torch.log2((peak / top).clamp_min(2.0 ** -127)))
        e = e - (top * 2 ** (e - 1) >= peak).double() + (top * 2 ** e < peak).double()
        e = e.clamp(-127, 127)
        n = v / 2 ** e
        n = torch.where(n < 0, -torch.floor(0.5 - n), torch.floor(n + 0.5))
        if bits == 4:
            n = _exact_round(n, 8)
        out[:, at:at + k] = (_exact_round(n, bits) * 2 ** e).flatten(1)
        at += k
    return out


def _exact_mx_weight(w, split):
    parts = []
    for k, c, sf in zip(split, w[:3], w[3:]):
        rows = torch.arange(c.shape[0], device=c.device)[:, None]
        col = torch.arange(k, device=c.device)[None, :]
        nibble = (c[rows, col // 2].int() >> (4 * (col % 2)).int()) & 15
        mag = nibble & 7
        value = torch.where(mag < 2, mag.double() / 2, (2 + (mag & 1)).double() * 2.0 ** ((mag >> 1).double() - 2))
        value = torch.where(nibble >= 8, -value, value)
        kb = col // 32
        at = (rows % 32) * 16 + rows // 32 % 4 * 4 + kb % 4 + kb // 4 * 512 + rows // 128 * 512 * ((k + 127) // 128)
        parts.append(value * 2.0 ** (sf[at].double() - 127))
    return torch.cat(parts, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]

    def product(a, sa):
        y = (a @ s["b"].double().t()) * sa[:, None] * s["sb"].double()[None, :]
        return y if s["bias"] is None else y + s["bias"].double()

    if kind == "product":
        return {"y": product(s["a"].double(), s["sa"].double())}
    x = s["x"].double()
    if kind in ("quantise", "linear"):
        q, step = _exact_rows(x)
        return {"values": q * step[:, None], "scale": step} if kind == "quantise" else {"y": product(q, step)}
    got = {}
    if s["residual"] is not None:
        x = x + s["residual"].double()
        got["residual"] = x
        x = x.to(s["dtype"]).double()  # the stream's own rounding is part of the definition
    h = x / torch.sqrt(x.pow(2).sum(dim=1, keepdim=True) / x.shape[1] + EPS) * s["norm"].double()
    if kind == "mx_linear":
        h = h.to(torch.bfloat16).double()[:, s["order"].long()]
        return {"y": _exact_mx_activation(h, s["split"]) @ _exact_mx_weight(s["w"], s["split"]).t(), **got}
    q, step = _exact_rows(h)
    if kind == "norm":
        return {"values": q * step[:, None], "scale": step, **got}
    return {"y": product(q, step), **got}
