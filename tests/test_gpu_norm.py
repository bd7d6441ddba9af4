"""RMS norm in front of the MX quantiser, and the modules that take a norm or 8-bit weights.

Tolerance of the norm, derived as for the 8-bit form (tests/test_gpu_int8.py): a row of K values is
shared by 32 lanes or more, so a thread adds at most 8 ceil(K / 256) squares one after the other; 13
roundings of the tree follow, half of all that counts after the square root, and rsqrtf and the
products add 14: EPS_H(K) = (8 ceil(K / 256) + 41) / 2 units of 2^-24.  h is then rounded to bf16, so it
equals the 64-bit value's rounding except where that value lies within EPS_H (relative) of the middle
between two bf16 numbers.  Codes and scales of a 32-group without such
an element have to be those of reorder_quantize_x of the 64-bit h, byte for byte.
"""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as orc
from tests import helpers as H

pytestmark = pytest.mark.gpu



def gen(seed):
    return torch.Generator().manual_seed(seed)


def exact_h(x, w, r, eps):
    """(u, h in 64 bits)"""
    u = x if r is None else (x.float() + r.float()).to(torch.bfloat16)
    f = u.double()
    return u, f / torch.sqrt(f.pow(2).mean(1, keepdim=True) + eps) * w.double()


def near_a_middle(h):
    """Elements whose bf16 rounding EPS_H could turn."""
    eps = (8 * -(-h.shape[1] // 256) + 41) / 2 * 2.0 ** -24
    return (h * (1 - eps)).to(torch.bfloat16) != (h * (1 + eps)).to(torch.bfloat16)


def compare_groups(got, want, near, idx, split):
    """Codes and scales, a 32-group at a time, where no element of the group is near a middle."""
    M, K = near.shape
    open_ = near[:, idx.long()].view(M, K // 32, 32).any(2)
    assert open_.numel() < 100 or float(open_.float().mean()) < 0.5  # something is left to compare
    at = 0
    for i, (k, nbytes) in enumerate(zip(split, (16, 24, 32))):
        g = k // 32
        if g == 0:
            continue
        ok = ~open_[:, at:at + g]
        at += g
        a, b = (t[i].cpu().contiguous().view(M, g, nbytes) for t in (got, want))
        assert torch.equal(a[ok], b[ok]), "codes of segment %d" % i
        rows, kb = torch.arange(M)[:, None], torch.arange(g)[None, :]
        off = rows % 32 * 16 + rows // 32 % 4 * 4 + kb % 4 + kb // 4 * 512 + rows // 128 * 512 * ((k + 127) // 128)
        assert torch.equal(got[3 + i].cpu()[off][ok], want[3 + i].cpu()[off][ok]), "scales of segment %d" % i


@pytest.mark.parametrize("split", [(0, 0, 32), (32, 0, 0), (64, 32, 32), (0, 96, 0), (640, 352, 32), (2560, 1408, 128),
                                   (8960, 4928, 448), (20448, 11264, 1024)])
def test_norm_then_split_against_64_bits(split):
    import mixedgemm_b200 as mg
    K = sum(split)
    for M, residual in ((1, True), (7, False), (150, True), (700 if K < 8192 else 310, True), (2500 if K <= 4096 else 5, False)):
        x = H.make_x(M, K, seed=M + K) if K >= 64 else torch.randn(M, K, generator=gen(M)).to(torch.bfloat16)
        r = torch.randn(M, K, generator=gen(M + 1)).to(torch.bfloat16) if residual else None
        w = (1 + 0.2 * torch.randn(K, generator=gen(2))).to(torch.bfloat16)
        idx = torch.randperm(K, generator=gen(3)).to(torch.int16)
        got = mg.rms_norm_reorder_quantize_x(x.cuda(), w.cuda(), idx.cuda(), *split, eps=1e-5,
                                             residual=r.cuda() if residual else None)
        u, h = exact_h(x, w, r, 1e-5)
        if residual:
            assert torch.equal(got[6].cpu(), u)
        want = mg.reorder_quantize_x(h.to(torch.bfloat16).cuda(), idx.cuda(), *split)
        assert len(got) == 6 + residual and all(a.shape == b.shape and a.stride() == b.stride() for a, b in zip(got, want))
        compare_groups(got, want, near_a_middle(h), idx, split)
    assert mg.device_status() == 0


@pytest.mark.parametrize("M", [1, 5, 300, 1300])
def test_same_bytes_as_the_quantiser_where_the_norm_is_exact(M):
    """Rows of +-2^j have the root-mean-square 2^j: h = +-w whatever the rounding of the statistics."""
    import mixedgemm_b200 as mg
    K, split = 4096, (2560, 1408, 128)
    g = gen(M)
    sign = torch.randint(0, 2, (M, K), generator=g) * 2 - 1
    x = (sign * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g).float())).to(torch.bfloat16)
    w = (torch.randn(K, generator=g) * 3).to(torch.bfloat16)
    idx = torch.randperm(K, generator=g).to(torch.int16).cuda()
    got = mg.rms_norm_reorder_quantize_x(x.cuda(), w.cuda(), idx, *split, eps=0.0)
    h = (sign * w.float()).to(torch.bfloat16)
    want = H.oracle_outputs(H.bits(h), idx.cpu().numpy(), *split)
    H.compare_quantised(got, want, M, split, "norm")


def test_rows_in_place_pitched_and_given_buffers():
    import mixedgemm_b200 as mg
    M, K, split = 70, 1024, (640, 256, 128)
    x, r = H.make_x(M, K, seed=1), H.make_x(M, K, seed=2)
    w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(torch.bfloat16).cuda()
    idx = torch.randperm(K, generator=gen(4)).to(torch.int16).cuda()
    ref = mg.rms_norm_reorder_quantize_x(x.cuda(), w, idx, *split, residual=r.cuda())
    buf = torch.full((2, M, K + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    xv, rv = buf[0, :, :K], buf[1, :, :K]
    xv.copy_(x), rv.copy_(r)
    out = mg.alloc_quantized_x(M, *split, "cuda", padded=False)
    got = mg.rms_norm_reorder_quantize_x(xv, w, idx, *split, residual=rv, residual_out=rv, out=out)
    assert got[6] is rv and torch.equal(rv, ref[6]) and torch.equal(xv.cpu(), x)
    for i in range(3):
        assert got[i] is out[i] and torch.equal(got[i], ref[i])
    assert bool((buf[:, :, K:] == 5).all())


def test_rows_that_are_not_finite_give_nan_products_and_spoil_no_other():
    import mixedgemm_b200 as mg
    M, N, K, split = 40, 256, 1024, (640, 256, 128)
    x = H.make_x(M, K, seed=1)
    x[3, 7], x[9, 1000], x[11] = float("nan"), float("inf"), 1e25
    x[12] = 0
    w = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    idx = torch.randperm(K, generator=gen(4)).to(torch.int16).cuda()
    B = mg.reorder_quantize_w(H.make_w(N, K).cuda(), idx, *split)
    y = []
    for rows in (x, x.clone().nan_to_num(0, 0, 0)):
        A = mg.rms_norm_reorder_quantize_x(rows.cuda(), w, idx, *split)
        y.append(mg.matmul(A[0], B[0], A[1], B[1], A[2], B[2], A[3], B[3], A[4], B[4], A[5], B[5]))
    bad = [3, 9, 11]
    assert bool(torch.isnan(y[0][bad]).all()) and bool((y[0][12] == 0).all())
    keep = [i for i in range(M) if i not in bad]
    assert torch.equal(y[0][keep], y[1][keep]) and bool(torch.isfinite(y[0][keep]).all())
    # a weight that overflows h has the same answer
    w[5] = 3e38
    x = torch.full((2, K), 1.0, dtype=torch.bfloat16)
    x[0, 5] = 30
    A = mg.rms_norm_reorder_quantize_x(x.cuda(), w, idx, *split)
    y = mg.matmul(A[0], B[0], A[1], B[1], A[2], B[2], A[3], B[3], A[4], B[4], A[5], B[5])
    assert bool(torch.isnan(y[0]).all()) and not bool(torch.isnan(y[1]).any())
    assert mg.device_status() == 0


def test_refusals():
    import mixedgemm_b200 as mg
    K, split = 256, (128, 64, 64)
    x, w = torch.zeros(4, K, dtype=torch.bfloat16, device="cuda"), torch.ones(K, dtype=torch.bfloat16, device="cuda")
    idx = torch.arange(K, dtype=torch.int16, device="cuda")
    f = mg.rms_norm_reorder_quantize_x
    odd = torch.zeros(4, K + 4, dtype=torch.bfloat16, device="cuda")
    good = mg.alloc_quantized_x(4, *split, "cuda")
    bad = [
        lambda: f(x.half(), w.half(), idx, *split), lambda: f(x, w, idx, 128, 64, 32), lambda: f(x, w, idx.int(), *split),
        lambda: f(x, w, idx[:200], *split), lambda: f(x, w, idx, 120, 72, 64), lambda: f(x, w, idx, *split, eps=-1.0),
        lambda: f(odd[:, :K], w, idx, *split), lambda: f(odd[:, 1:K + 1], w, idx, *split), lambda: f(x, w, idx, *split, residual=x[:3]),
        lambda: f(x, w, idx, *split, residual_out=x), lambda: f(x, w, idx, *split, residual=odd[:, :K]),
        lambda: f(x, w[:128], idx, *split), lambda: f(x, w, idx, *split, out=mg.alloc_quantized_x(3, *split, "cuda")),
        lambda: f(x, w, idx, *split, out=good[:3] + tuple(t[:100] for t in good[3:])), lambda: f(x.cpu(), w, idx, *split),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("case %d was not refused" % i)
    assert f(x[:0], w, idx, *split)[0].shape == (0, 64)


# ------------------------------------------------------------------------------------------ modules

def dense(N, K, seed):
    return H.make_w(N, K, seed=seed).cuda()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_mixed_linear_with_a_norm_is_its_operators_in_a_row(M):
    import mixedgemm_b200 as mg
    from mixedgemm_b200.linear import MixedLinear, QuantizedWeights
    K = 2048
    X = H.make_x(300, K, seed=3).cuda()
    r = torch.randn(M, K, generator=gen(8)).to(torch.bfloat16).cuda()
    w = (1 + 0.2 * torch.randn(K, generator=gen(9))).to(torch.bfloat16).cuda()
    idx = mg.reorder_index(X)
    Ws = [QuantizedWeights.from_dense(dense(N, K, 5 + N), idx) for N in (512, 256)]
    lin = MixedLinear(Ws, norm_weight=w, eps=1e-5)
    x = X[:M].contiguous()
    ys, stream = lin(x, residual=r)
    A = mg.rms_norm_reorder_quantize_x(x, w, idx, *lin.split, eps=1e-5, residual=r)
    assert torch.equal(stream, A[6]) and torch.equal(stream, (x.float() + r.float()).to(torch.bfloat16))
    for y, q in zip(ys, lin.weights):
        B = q.parts
        ref = mg.matmul(A[0], B[0], A[1], B[1], A[2], B[2], A[3], B[3], A[4], B[4], A[5], B[5])
        assert (y.float() - ref.float()).norm() <= 0.01 * ref.float().norm()  # another tile order may round otherwise
    again = lin(stream)  # without a residual: the outputs alone
    assert isinstance(again, list) and all((a.float() - y.float()).norm() <= 0.01 * y.float().norm() for a, y in zip(again, ys))
    with pytest.raises(ValueError):
        MixedLinear(Ws)(x, residual=r)
    with pytest.raises(ValueError):
        lin(x, residual=r[:, :8])
    assert mg.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lead", [(1,), (3, 50)])
def test_int8_linear(lead, dtype, tmp_path):
    import mixedgemm_b200 as mg
    from mixedgemm_b200.linear import Int8Linear, Int8Weights
    K, Ns = 1000, (384, 130)
    x = H.make_x(150, K, seed=3).to(dtype).cuda()[:int(np.prod(lead))].reshape(*lead, K)
    r = torch.randn(*lead, K, generator=gen(8)).to(dtype).cuda()
    Ws = [dense(N, K, N) for N in Ns]
    bias = torch.randn(Ns[1], generator=gen(1)).cuda()
    w = (1 + 0.2 * torch.randn(K, generator=gen(9))).to(dtype).cuda()
    plain, norm = Int8Linear.from_dense(Ws, bias=[None, bias]), Int8Linear.from_dense(Ws, norm_weight=w, eps=1e-5)
    ys = plain(x)
    for y, W, b in zip(ys, Ws, (0, bias)):
        assert y.shape == (*lead, W.shape[0]) and y.dtype == dtype
        ref = x.double() @ W.double().t() + b
        # x: half a step of amax / 127 per element; W likewise: a few per cent of a row's norm
        assert float((y.double() - ref).norm() / ref.norm()) < 0.1
    q, s = mg.quantize_int8(x.reshape(-1, K))
    f = plain.fused
    ref = mg.matmul_int8(q, f.codes, s, f.scale, bias=plain.bias, out_dtype=dtype)
    assert torch.equal(torch.cat(ys, -1).reshape(-1, sum(Ns)), ref)
    yn, stream = norm(x, residual=r)
    q, s, u = mg.rms_norm_int8(x.reshape(-1, K), w, eps=1e-5, residual=r.reshape(-1, K))
    assert torch.equal(stream, u.reshape(x.shape)) and torch.equal(
        torch.cat(yn, -1).reshape(-1, sum(Ns)), mg.matmul_int8(q, f.codes, s, f.scale, out_dtype=dtype))
    again = norm(stream)
    assert all(torch.equal(a, y) for a, y in zip(again, yn))
    # the container on disk
    plain.weights[1].save(str(tmp_path / "w.pt"))
    back = Int8Linear(Int8Weights.load(str(tmp_path / "w.pt")), bias=bias)
    assert torch.equal(back(x), ys[1])
    with pytest.raises(ValueError):
        plain(x, residual=r)
    with pytest.raises(ValueError):
        Int8Linear.from_dense(Ws, norm_weight=w[:10])


def test_a_block_of_both_kinds_in_a_graph():
    """norm -> 4-bit q/k/v, 8-bit o, norm -> 4-bit gate, 8-bit down: the operators as a layer uses
    them, eager and replayed with new inputs."""
    import mixedgemm_b200 as mg
    from mixedgemm_b200.linear import Int8Linear, MixedLinear, QuantizedWeights
    M, K, F = 20, 2048, 1024  # a split with KS and KO multiples of 64, as the product needs
    X = H.make_x(300, K, seed=3).cuda()
    idx = mg.reorder_index(X)
    w = [(1 + 0.2 * torch.randn(K, generator=gen(i))).to(torch.bfloat16).cuda() for i in range(2)]
    qkv = MixedLinear([QuantizedWeights.from_dense(dense(N, K, N), idx) for N in (2048, 256, 256)], norm_weight=w[0], max_tokens=M)
    o = Int8Linear.from_dense(dense(K, K, 11))
    gate = MixedLinear(QuantizedWeights.from_dense(dense(F, K, 12), idx), norm_weight=w[1], max_tokens=M)
    down = Int8Linear.from_dense(dense(K, F, 13))

    def block(x, stream):
        (q, _, _), stream = qkv(x, residual=stream)
        h, stream = gate(o(q), residual=stream)
        return down(torch.nn.functional.silu(h)), stream

    x, s = X[:M].contiguous(), X[M:2 * M].contiguous()
    want = block(x, s)
    x2, s2 = X[40:60].contiguous(), X[60:80].contiguous()
    want2 = block(x2, s2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xin, sin = x.clone(), s.clone()
    with torch.cuda.stream(side):
        got = block(xin, sin)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = block(xin, sin)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xin.copy_(x2), sin.copy_(s2)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want2))
    assert mg.device_status() == 0


def test_product_with_and_without_the_compiled_module(monkeypatch):
    """api.matmul through mixedgemm_ops and through ctypes: the same bytes, the same refusals."""
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import api
    for M, N, split in ((9, 256, (128, 64, 64)), (300, 512, (2560, 1408, 128)), (40, 128, (256, 0, 128))):
        K = sum(split)
        idx = torch.randperm(K, generator=gen(1)).to(torch.int16).cuda()
        A = mg.reorder_quantize_x(H.make_x(M, K, seed=2).cuda(), idx, *split)
        for padded in (True, False):  # (dense buffers of 64-tails need the workspace)
            B = mg.reorder_quantize_w(H.make_w(N, K).cuda(), idx, *split, out=api.alloc_quantized_w(N, *split, "cuda", padded=padded))
            ops = [t for pair in zip(A, B) for t in pair]
            C = torch.randn(M, N, generator=gen(3)).to(torch.bfloat16).cuda()
            calls = [dict(), dict(out_dtype=torch.float32), dict(C=C), dict(out=torch.empty(M, N, device="cuda"))]
            bad = [dict(out_dtype=torch.float16), dict(C=C.float()), dict(C=C[:, :-8]), dict(out=torch.empty(M, N + 8, dtype=torch.bfloat16, device="cuda"))]
            got = [mg.matmul(*ops, **kw).clone() for kw in calls]
            broken = [ops[:6] + [t[:100] for t in ops[6:]], [ops[0].cpu()] + ops[1:], ops[:2] + [ops[2][:, :-3] if split[1] else ops[2][1:]] + ops[3:], [ops[0][1:]] + ops[1:]]
            for module in (api._ops(), False):
                monkeypatch.setattr(api, "_ops_module", module)
                for kw in bad:
                    with pytest.raises(RuntimeError):
                        mg.matmul(*ops, **kw)
                for args in broken:
                    with pytest.raises(RuntimeError):
                        mg.matmul(*args)
            want = [mg.matmul(*ops, **kw) for kw in calls]  # ctypes
            monkeypatch.undo()
            assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))
    assert mg.device_status() == 0


@pytest.mark.parametrize("split", ((512, 256, 256), (1024, 0, 0), (576, 64, 384)))
@pytest.mark.parametrize("M", (1, 129))
def test_buffers_the_norm_makes_are_apart_from_one_another(M, split):
    import mixedgemm_b200 as mg
    g, K = gen(5), 1024
    x, w = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda(), torch.randn(K, generator=g).to(torch.bfloat16).cuda()
    order = torch.randperm(K, generator=g).to(torch.int16).cuda()
    got = mg.rms_norm_reorder_quantize_x(x, w, order, *split)
    given = mg.alloc_quantized_x(M, *split, x.device)
    for t, o in zip(got, given):
        assert t.dtype == torch.uint8 and t.shape == o.shape and t.stride() == o.stride() and t.data_ptr() % 128 == 0
        o.fill_(255)
    for i, t in enumerate(got):
        t.fill_(i + 1)
    for i, t in enumerate(got):
        assert (t == i + 1).all()
    for o in got:
        o.fill_(255)
    mg.rms_norm_reorder_quantize_x(x, w, order, *split, out=list(got))
    mg.rms_norm_reorder_quantize_x(x, w, order, *split, out=given)
    for t, o in zip(got, given):
        assert torch.equal(t, o)


@pytest.mark.parametrize("K", (32, 1024, 4096, 8192, 14336, 17408, 20480, 32736))
@pytest.mark.parametrize("M", (1, 150, 1333))
def test_rows_of_every_length(M, K):
    """Rows per stage and stages of x and of the residual depend on K: from eight rows in several stages to one row in
    a single one with the residual read from memory.  x + r = +-2^j, so h is exact and its bytes are the quantiser's."""
    import mixedgemm_b200 as mg
    g = gen(M + K)
    ko = K // 128 * 32
    split = (K - 2 * ko, ko, ko)
    sign = torch.randint(0, 2, (M, K), generator=g).cuda() * 2.0 - 1
    u = (sign * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g).float().cuda())).to(torch.bfloat16)
    r = (u.float() * -0.5).to(torch.bfloat16)
    w = (torch.randn(K, generator=g) * 3).to(torch.bfloat16).cuda()
    order = torch.randperm(K, generator=g).to(torch.int16).cuda()
    rows = mg.reorder_quantize_x((sign * w.float()).to(torch.bfloat16), order, *split)
    want = [t.clone() for t in rows]
    for x, res in ((u, None), ((u.float() * 1.5).to(torch.bfloat16), r)):
        got = mg.rms_norm_reorder_quantize_x(x, w, order, *split, eps=0.0, residual=res)
        if res is not None:
            assert torch.equal(got[6], u)
        for i in range(3):
            assert torch.equal(got[i], want[i])
        mg.rms_norm_reorder_quantize_x(x, w, order, *split, eps=0.0, residual=res, out=rows)
        for i in range(3, 6):  # scale bytes behind the last row are as they were
            assert torch.equal(rows[i], want[i])


def test_refusals_of_the_library_are_the_packages_error_on_every_route(monkeypatch):
    """What the C ABI refuses is MixedGemmError with its status, through the compiled module as through ctypes, and
    the same text from both."""
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import _capi, api
    SHAPE, ALIGN = 1, 3
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    w, q, s = x[0], torch.zeros(4, 256, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    idx = torch.arange(256, device="cuda").to(torch.int16)
    A = mg.alloc_quantized_x(4, 128, 64, 64, "cuda")
    narrow = [t for pair in zip(A, mg.alloc_quantized_w(100, 128, 64, 64, "cuda")) for t in pair]  # N % 128
    crooked = [t for pair in zip(A, mg.alloc_quantized_w(128, 128, 64, 64, "cuda")) for t in pair]
    crooked[0] = torch.zeros(4 * 64 + 4, dtype=torch.uint8, device="cuda")[4:].view(4, 64)
    for status, call in ((SHAPE, lambda: mg.quantize_int8(x[:, :0])), (SHAPE, lambda: mg.rms_norm_int8(x, w, eps=-1.0)),
                         (ALIGN, lambda: mg.matmul_int8(q[:, 1:33], q[:, :32], s, s)),
                         (SHAPE, lambda: mg.rms_norm_reorder_quantize_x(x, w, idx, 144, 80, 32)),
                         (ALIGN, lambda: mg.rms_norm_reorder_quantize_x(x[:, 1:129], w[:128], idx[:128], 64, 32, 32))):
        with pytest.raises(_capi.MixedGemmError) as e:
            call()
        assert e.value.status == status
    for status, args in ((SHAPE, narrow), (ALIGN, crooked)):
        seen = []
        for module in (api._ops(), False):
            monkeypatch.setattr(api, "_ops_module", module)
            with pytest.raises(_capi.MixedGemmError) as e:
                mg.matmul(*args)
            seen.append((type(e.value), e.value.status, str(e.value)))
            monkeypatch.undo()
        assert seen[0] == seen[1] and seen[0][1] == status


def test_mixed_linear_from_dense_takes_what_the_constructor_takes():
    import mixedgemm_b200 as mg
    from mixedgemm_b200.linear import MixedLinear, QuantizedWeights
    K = 2048  # (the product takes KS and KO that are multiples of 64: 1024 channels have 32 in 8 bits)
    X = H.make_x(300, K, seed=3).cuda()
    Ws = [dense(N, K, N) for N in (256, 128)]
    kw = dict(bias=[None, torch.randn(128, generator=gen(1)).cuda()], eps=1e-5,
              norm_weight=(1 + 0.2 * torch.randn(K, generator=gen(9))).to(torch.bfloat16).cuda())
    idx = mg.reorder_index(X)
    want = MixedLinear([QuantizedWeights.from_dense(W, idx) for W in Ws], **kw)
    for got, ref in zip(MixedLinear.from_dense(Ws, X, **kw)(X[:40]), want(X[:40])):
        assert torch.equal(got, ref)


def test_mx_norm_between_one_anothers_rows_and_over_one_another():
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import _capi
    M, split = 33, (64, 32, 32)
    x, r = H.make_x(M, 128, seed=1).cuda(), H.make_x(M, 128, seed=2).cuda()
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    idx = torch.randperm(128, generator=gen(4)).to(torch.int16).cuda()
    ref = mg.rms_norm_reorder_quantize_x(x, w, idx, *split, residual=r)
    whole = torch.zeros(M, 1024, dtype=torch.uint8, device="cuda")
    part = lambda b0, b1, t: whole[:, b0:b1].view(t)
    xv, rv, uv = part(0, 256, torch.bfloat16), part(256, 512, torch.bfloat16), part(512, 768, torch.bfloat16)
    xv.copy_(x), rv.copy_(r)
    out = [part(768, 800, torch.uint8), part(800, 824, torch.uint8), part(832, 864, torch.uint8)] + [torch.empty_like(t) for t in ref[3:6]]
    got = mg.rms_norm_reorder_quantize_x(xv, w, idx, *split, residual=rv, residual_out=uv, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got[:3] + got[6:], ref[:3] + ref[6:])) and torch.equal(xv, x) and torch.equal(rv, r)
    before = whole.clone()
    f = lambda **kw: mg.rms_norm_reorder_quantize_x(xv, w, idx, *split, residual=rv, **kw)
    bad = [lambda: f(residual_out=part(16, 272, torch.bfloat16)), lambda: f(residual_out=part(496, 752, torch.bfloat16)),
           lambda: f(residual_out=uv, out=[part(752, 784, torch.uint8)] + out[1:]), lambda: f(residual_out=uv, out=out[:1] + [part(784, 808, torch.uint8)] + out[2:]),
           lambda: f(out=out[:3] + [out[4], out[4], out[5]]), lambda: f(out=out[:2] + [part(0, 32, torch.uint8)] + out[3:])]
    for i, call in enumerate(bad):
        with pytest.raises(_capi.MixedGemmError) as e:
            call()
            pytest.fail("case %d was not refused" % i)
        assert e.value.status == 9, (i, str(e.value))
    assert torch.equal(whole, before)
