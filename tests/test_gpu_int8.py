"""8-bit operators on the GPU against their definitions in 64 bits.

Tolerances, derived:
  quantize_int8   every step is one correctly rounded fp32 operation, so codes and scales are equal to
                  the same steps done by numpy in fp32.
  rms_norm_int8   all terms of the sum of squares are positive; a thread adds at most 128 of them one
                  after the other and ten tree levels follow: 138 roundings of 2^-24, half of that
                  after the square root.  rsqrtf is off by 2^-22, and w u, v, 127/a, their products
                  and a/127 add at most ten roundings: 69 + 4 + 10 < 96 units of 2^-24 = EPS_NORM.
                  A code is then off by at most half a step plus twice 127 EPS_NORM; the scale by EPS_NORM.
                  u is one fp32 addition and one rounding: equal to the same done by torch.
  matmul_int8     the sum S is exact.  float(S), times sa, and the fused multiply-add with sb and the
                  bias are three roundings: 2^-24 (2 |S sa sb| + |y|) up to second-order terms, and
                  the result type adds eps / 2 |y|, or, below its smallest normal number, half of its
                  smallest step: fp16 has 2^-24 between all values under 2^-14, so 2^-25 there (a sum
                  that nearly cancels the bias lands in that range, where eps / 2 |y| is less than that).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS_NORM = 96 * 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = 2.0 ** -100


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tokens(M, K, dtype, seed=0):
    """Tokens of different loudness, a few loud channels; on the CPU."""
    g = gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randn(M, 1, generator=g))
    x[:, ::37] *= 20
    return x.to(dtype)


def pitched(t, pitch, fill):
    """A CUDA copy of t whose rows are `pitch` elements apart, `fill` in between; and the whole buffer."""
    buf = torch.full((t.shape[0], pitch), fill, dtype=t.dtype, device="cuda")
    buf[:, :t.shape[1]] = t.cuda()
    return buf[:, :t.shape[1]], buf


def want_codes(x):
    """The definition, every step one fp32 operation (numpy rounds as IEEE 754 asks)."""
    f = x.float().numpy()
    a = np.maximum(np.abs(f).max(1, keepdims=True), np.float32(TINY))
    q = np.rint(f * (np.float32(127) / a))
    return q.astype(np.int8), (a / np.float32(127))[:, 0]


# ------------------------------------------------------------------------------------- quantize_int8

# a warp's row, several warps' row, one row for a whole CTA, rows that are read twice; odd lengths
LENGTHS = [1, 2, 7, 8, 31, 64, 65, 500, 512, 1000, 1024, 1032, 1931, 4096, 8192, 14336, 16385, 32768, 40000, 131071]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", LENGTHS)
def test_quantise_equals_its_definition(K, dtype):
    import mixedgemm_b200 as mg
    for M in (1, 3, 300 if K <= 4096 else 5):
        x = tokens(M, K, dtype, seed=K + M)
        q, s = mg.quantize_int8(x.cuda())
        wq, ws = want_codes(x)
        assert q.shape == (M, K) and q.stride(0) % 16 == 0 and q.dtype == torch.int8
        assert np.array_equal(s.cpu().numpy(), ws)
        assert np.array_equal(q.cpu().numpy(), wq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K, pitch, lead", [(64, 72, 0), (64, 71, 0), (64, 80, 3), (1000, 1001, 1), (1032, 1040, 8), (4096, 4097, 5)])
def test_quantise_strided_rows_and_untouched_padding(K, pitch, lead, dtype):
    import mixedgemm_b200 as mg
    M = 9
    x = tokens(M, K, dtype, seed=K)
    flat = torch.full((lead + M * pitch,), float("nan"), dtype=dtype, device="cuda")  # padding must not be read
    view = flat[lead:].view(M, pitch)[:, :K]
    view.copy_(x.cuda())
    buf = torch.full((M, K + 5), 77, dtype=torch.int8, device="cuda")  # rows at odd addresses
    s = torch.empty(M, device="cuda")
    q, s2 = mg.quantize_int8(view, out=(buf[:, :K], s))
    wq, ws = want_codes(x)
    assert s2 is s and np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)
    assert bool((buf[:, K:] == 77).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [40, 65, 4096])
def test_quantise_rows_without_a_scale(K, dtype):
    """Zeros, values below the floor, NaN and infinities: only the row that holds them is affected."""
    import mixedgemm_b200 as mg
    x = tokens(7, K, dtype, seed=1)
    x[0] = 0
    x[1, K // 2] = float("nan")
    x[2, K - 1] = float("-inf")
    x[3, 0], x[3, 1] = float("inf"), float("nan")
    x[4] = torch.finfo(dtype).tiny if dtype != torch.float16 else 2.0 ** -24
    x[5] = -x[5].abs().amax()
    q, s = (t.cpu() for t in mg.quantize_int8(x.cuda()))
    good = [0, 4, 5, 6]
    wq, ws = want_codes(x[good])
    assert np.array_equal(q[good].numpy(), wq) and np.array_equal(s[good].numpy(), ws)
    assert (q[0] == 0).all() and s[0] == np.float32(TINY) / np.float32(127)
    assert (q[5] == -127).all()
    for r in (1, 2, 3):
        assert (q[r] == 0).all() and torch.isnan(s[r])


# ------------------------------------------------------------------------------------- rms_norm_int8

def check_norm(got, x, w, r, eps):
    q, s, u = [t.cpu() for t in got] + ([None] if r is None else [])
    f = x
    if r is not None:
        f = (x.float() + r.float()).to(x.dtype)
        assert torch.equal(u, f)
    f = f.double()
    h = f * w.double() / torch.sqrt(f.pow(2).mean(1, keepdim=True) + eps)
    a = h.abs().amax(1, keepdim=True).clamp_min(TINY)
    t = h * 127 / a
    assert ((s.double() - a[:, 0] / 127).abs() <= EPS_NORM * a[:, 0] / 127).all()
    assert float((q.double() - t).abs().max()) <= 0.5 + 2 * 127 * EPS_NORM


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", LENGTHS)
def test_norm_against_64_bits(K, dtype):
    import mixedgemm_b200 as mg
    for M, residual in ((1, True), (3, False), (200 if K <= 4096 else 4, True)):
        x, r = tokens(M, K, dtype, seed=K), tokens(M, K, dtype, seed=K + 1) if residual else None
        w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(dtype)
        got = mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5, residual=r.cuda() if residual else None)
        assert len(got) == 2 + residual
        check_norm(got, x, w, r, 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K, px, pr", [(64, 72, 80), (65, 67, 70), (1000, 1000, 1003), (1032, 1040, 1032), (4096, 4100, 4104)])
def test_norm_strided_and_in_place(K, px, pr, dtype):
    import mixedgemm_b200 as mg
    M = 11
    x, r = tokens(M, K, dtype, seed=5), tokens(M, K, dtype, seed=6)
    w = (1 + 0.2 * torch.randn(K, generator=gen(4))).to(dtype)
    xv, xb = pitched(x, px, float("nan"))
    rv, rb = pitched(r, pr, float("nan"))
    got = mg.rms_norm_int8(xv, w.cuda(), eps=1e-6, residual=rv, residual_out=rv)  # the stream in place
    assert got[2] is rv
    check_norm(got, x, w, r, 1e-6)
    assert bool(torch.isnan(rb[:, K:].float()).all()) and torch.equal(xv.cpu(), x)
    rv.copy_(r.cuda())
    got = mg.rms_norm_int8(xv, w.cuda(), eps=1e-6, residual=rv, residual_out=xv)  # or over x
    check_norm(got, x, w, r, 1e-6)
    assert torch.equal(rv.cpu(), r) and bool(torch.isnan(xb[:, K:].float()).all())


def test_norm_in_place_on_rows_that_are_read_twice():
    import mixedgemm_b200 as mg
    M, K = 2, 131071
    x, r = tokens(M, K, torch.bfloat16, seed=5), tokens(M, K, torch.bfloat16, seed=6)
    w = torch.ones(K, dtype=torch.bfloat16)
    rd = r.cuda()
    check_norm(mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-6, residual=rd, residual_out=rd), x, w, r, 1e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [40, 65, 4096])
def test_norm_rows_without_a_scale(K, dtype):
    import mixedgemm_b200 as mg
    x = tokens(6, K, dtype, seed=2)
    w = (1 + 0.2 * torch.randn(K, generator=gen(5))).to(dtype)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, K - 1] = float("inf")
    if dtype != torch.float16:
        x[3] = 1e20  # the sum of squares leaves fp32
    q, s = (t.cpu() for t in mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5))
    assert (q[0] == 0).all() and s[0] == np.float32(TINY) / np.float32(127)
    for row in (1, 2) + ((3,) if dtype != torch.float16 else ()):
        assert (q[row] == 0).all() and torch.isnan(s[row])
    check_norm((q[4:], s[4:]), x[4:], w, None, 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_faint_rows_under_weights_of_zero(dtype):
    """eps far below the squares and nothing left after the weight: codes 0 and the smallest scale, not NaN."""
    import mixedgemm_b200 as mg
    x = torch.full((3, 96), 2.0 ** -20, dtype=dtype)
    x[1, ::2] *= -1
    w = torch.zeros(96, dtype=dtype)
    for eps in (0.0, 1e-30):
        q, s = (t.cpu() for t in mg.rms_norm_int8(x.cuda(), w.cuda(), eps=eps))
        assert (q == 0).all() and (s == np.float32(TINY) / np.float32(127)).all()
    q, s = (t.cpu() for t in mg.rms_norm_int8(torch.zeros_like(x).cuda(), (w + 1).cuda(), eps=0.0))  # 0 / 0
    assert (q == 0).all() and torch.isnan(s).all()


# --------------------------------------------------------------------------------------- matmul_int8

def codes(rows, K, seed, lo=-128):
    q = torch.randint(lo, 128, (rows, K), generator=gen(seed), dtype=torch.int16).to(torch.int8)
    buf = torch.full((rows, (K + 15) // 16 * 16), 99, dtype=torch.int8, device="cuda")  # padding must not count
    buf[:, :K] = q.cuda()
    return q, buf[:, :K]


def check_product(y, a, b, sa, sb, bias):
    S = (a.double() @ b.double().t())  # whole numbers below 2^31: exact
    t = S * sa.double()[:, None] * sb.double()[None, :]
    want = t if bias is None else t + bias.double()
    y = y.cpu()
    tol = 2.0 ** -24 * (2 * t.abs() + want.abs()) * (1 + 2.0 ** -20)
    if y.dtype != torch.float32:
        half_step = torch.finfo(y.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10)
        tol = tol + half_step.clamp_min(torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps / 2)
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())


def run_product(M, N, K, dtype, with_bias, seed=0):
    import mixedgemm_b200 as mg
    a, av = codes(M, K, seed)
    b, bv = codes(N, K, seed + 1)
    g = gen(seed + 2)
    sa, sb = torch.rand(M, generator=g) * 0.01 + 1e-3, torch.rand(N, generator=g) * 0.01 + 1e-3
    bias = torch.randn(N, generator=g) if with_bias else None
    y = mg.matmul_int8(av, bv, sa.cuda(), sb.cuda(), bias=None if bias is None else bias.cuda(), out_dtype=dtype)
    assert y.shape == (M, N) and y.dtype == dtype
    check_product(y, a, b, sa, sb, bias)
    assert mg.device_status() == 0


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (3, 7, 16), (5, 129, 31), (32, 128, 129), (33, 300, 1000), (64, 256, 4096),
          (65, 127, 640), (127, 130, 2048), (128, 1024, 512), (129, 1, 257), (200, 333, 1931), (300, 513, 768),
          (513, 1000, 384), (777, 2049, 1200)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product_against_64_bits(M, N, K, dtype):
    run_product(M, N, K, dtype, with_bias=(M + N) % 2 == 0, seed=M + N + K)


@pytest.mark.parametrize("tile", [32, 64, 128])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
def test_product_of_every_tile_and_split(tile, split, mgopt):
    mgopt.set("INT8_FEW", 0)
    mgopt.set("INT8_PAIR", 0)
    mgopt.set("INT8_TOKENS", tile)
    mgopt.set("INT8_SPLIT", split)
    for M, N, K in ((1, 130, 1024), (37, 300, 1931), (140, 257, 4096), (300, 640, 128)):
        run_product(M, N, K, torch.float32, with_bias=True, seed=tile + split)


@pytest.mark.parametrize("dtype", TYPES)
def test_product_of_the_pair_form(dtype, mgopt):
    """No whole round of tiles or several (both accumulators), and what is left over whole, in halves and in
    quarters (74 pairs: 1, 9 and 6 = 80 - 74 tiles in quarters, 24 and 34 in halves, 40 whole, 74 nothing),
    parts beyond the last token, ragged edges, one slice of K."""
    mgopt.set("INT8_FEW", 0)
    mgopt.set("INT8_PAIR", 1)
    for M, N, K in ((1, 1, 1), (60, 200, 70), (200, 130, 1024), (140, 257, 1931), (513, 640, 128), (1000, 5000, 300), (2300, 3000, 128),
                    (700, 2000, 640), (1280, 2000, 1000), (500, 9472, 256), (4000, 4100, 256)):
        run_product(M, N, K, dtype, with_bias=True, seed=M)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4])
def test_product_of_single_tokens(M, dtype):
    """Whole rows to a warp and shared ones, odd channels, tails of K shorter than a vector."""
    for N, K in ((1, 1), (1, 15), (3, 16), (5, 17), (130, 511), (1000, 4096), (77, 14336), (5001, 1200), (2, 131071)):
        run_product(M, N, K, dtype, with_bias=N % 2 == 0, seed=M + N)


def test_product_does_not_depend_on_tile_or_split(mgopt):
    """The sum is exact, so every form gives the same bytes."""
    import mixedgemm_b200 as mg
    _, av = codes(100, 2000, 1)
    _, bv = codes(400, 2000, 2)
    sa, sb = torch.rand(100, device="cuda"), torch.rand(400, device="cuda")
    ref = mg.matmul_int8(av, bv, sa, sb)
    for tile in (32, 64, 128):
        for split in (1, 2, 4, 8):
            mgopt.set("INT8_TOKENS", tile)
            mgopt.set("INT8_SPLIT", split)
            assert torch.equal(mg.matmul_int8(av, bv, sa, sb), ref)
    mgopt.set("INT8_PAIR", 1)
    assert torch.equal(mg.matmul_int8(av, bv, sa, sb), ref)
    few = mg.matmul_int8(av[:2], bv, sa[:2], sb)
    mgopt.set("INT8_FEW", 0)
    assert torch.equal(few, mg.matmul_int8(av[:2], bv, sa[:2], sb)) and torch.equal(few, ref[:2])


def test_product_of_the_longest_row_does_not_overflow():
    import mixedgemm_b200 as mg
    K = 131071
    a, av = torch.full((3, K), -128, dtype=torch.int8), None
    a[1] = 127
    av, _ = pitched(a, 131072, 99)
    one = torch.ones(3, device="cuda")
    y = mg.matmul_int8(av, av, one, one, out_dtype=torch.float32)
    check_product(y, a, a, one.cpu(), one.cpu(), None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N", [(40, 130), (300, 257)])
def test_product_into_a_view_leaves_the_rest(M, N, dtype):
    import mixedgemm_b200 as mg
    K = 200
    a, av = codes(M, K, 1)
    b, bv = codes(N, K, 2)
    sa, sb = torch.rand(M) * 0.01, torch.rand(N) * 0.01
    flat = torch.full((1 + (M + 1) * (N + 3),), 7.0, dtype=dtype, device="cuda")  # odd base, odd pitch
    buf = flat[1:].view(M + 1, N + 3)
    out = buf[:M, :N]
    assert mg.matmul_int8(av, bv, sa.cuda(), sb.cuda(), out=out) is out
    check_product(out, a, b, sa, sb, None)
    assert bool((buf[:, N:] == 7).all()) and bool((buf[M:] == 7).all()) and flat[0] == 7


def test_product_of_nothing():
    import mixedgemm_b200 as mg
    q = lambda r: torch.zeros(r, 32, dtype=torch.int8, device="cuda")
    s = lambda r: torch.ones(r, device="cuda")
    assert mg.matmul_int8(q(0), q(5), s(0), s(5)).shape == (0, 5)
    assert mg.matmul_int8(q(4), q(0), s(4), s(0)).shape == (4, 0)
    assert mg.quantize_int8(torch.zeros(0, 32, device="cuda"))[0].shape == (0, 32)
    x = torch.zeros(0, 32, device="cuda")
    assert mg.rms_norm_int8(x, torch.ones(32, device="cuda"), residual=x)[2].shape == (0, 32)


def test_a_bad_token_spoils_its_own_row_only():
    import mixedgemm_b200 as mg
    x = tokens(40, 256, torch.bfloat16)
    x[17, 5] = float("nan")
    q, s = mg.quantize_int8(x.cuda())
    b, bv = codes(130, 256, 2)
    sb = torch.rand(130) * 0.01
    y = mg.matmul_int8(q, bv, s, sb.cuda())
    assert bool(torch.isnan(y[17]).all())
    keep = [i for i in range(40) if i != 17]
    check_product(y[keep], q[keep].cpu(), b, s[keep].cpu(), sb, None)


def test_refusals():
    import mixedgemm_b200 as mg
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w, q = torch.ones(64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(4, device="cuda")
    bad = [
        lambda: mg.quantize_int8(x.double()), lambda: mg.quantize_int8(x[0]), lambda: mg.quantize_int8(x.t()),
        lambda: mg.quantize_int8(x[:1].expand(4, 64)), lambda: mg.quantize_int8(x[:, ::2]),
        lambda: mg.quantize_int8(x, out=(q[:3], s)), lambda: mg.quantize_int8(x, out=(q, s[:3])),
        lambda: mg.quantize_int8(x, out=(q.int(), s)), lambda: mg.quantize_int8(torch.zeros(2, 0, device="cuda")),
        lambda: mg.rms_norm_int8(x, w.float()), lambda: mg.rms_norm_int8(x, w[:32]), lambda: mg.rms_norm_int8(x, w, eps=-1.0),
        lambda: mg.rms_norm_int8(x, w, residual=x[:2]), lambda: mg.rms_norm_int8(x, w, residual=x.float()),
        lambda: mg.rms_norm_int8(x, w, residual_out=x), lambda: mg.rms_norm_int8(x, w, residual=x, residual_out=x[:1].expand(4, 64)),
        lambda: mg.matmul_int8(q, q[:, :32], s, s), lambda: mg.matmul_int8(q, q, s[:3], s), lambda: mg.matmul_int8(q, q, s, s.half()),
        lambda: mg.matmul_int8(q, q, s, s, bias=s.bfloat16()), lambda: mg.matmul_int8(q.view(torch.uint8), q, s, s),
        lambda: mg.matmul_int8(q, q, s, s, out_dtype=torch.float64), lambda: mg.matmul_int8(q, q, s, s, out=x[:, :4].t()),
        lambda: mg.matmul_int8(q[:, :40].contiguous(), q[:, :40], s, s), lambda: mg.matmul_int8(q[:, 1:33], q[:, :32], s, s),
        lambda: mg.matmul_int8(q, q, s, s, out=x[:, :4], out_dtype=torch.float16),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("case %d was not refused" % i)
    torch.cuda.synchronize()


def test_norm_then_product_on_a_side_stream_and_in_two_graphs():
    """The operators as a layer runs them, on another stream, and captured twice on one stream and
    replayed at the same time on two: no call keeps anything from one to the next."""
    import mixedgemm_b200 as mg
    M, N, K = 24, 600, 4096
    w = (1 + 0.2 * torch.randn(K, generator=gen(4))).to(torch.bfloat16).cuda()
    bq, sb = mg.quantize_int8((torch.randn(N, K, generator=gen(5)) * 0.02).cuda())

    def layer(x, r):
        q, s, u = mg.rms_norm_int8(x, w, residual=r)
        return mg.matmul_int8(q, bq, s, sb), u

    xs = [tokens(M, K, torch.bfloat16, seed=i).cuda() for i in range(4)]
    want = [layer(xs[i], xs[3 - i]) for i in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(xs[0], xs[3])
    side.synchronize()
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    ins = [[xs[0].clone(), xs[3].clone()], [xs[1].clone(), xs[2].clone()]]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(*ins[i]))
        graphs.append(g)
    ins[0][0].copy_(xs[2]), ins[0][1].copy_(xs[1])
    ins[1][0].copy_(xs[3]), ins[1][1].copy_(xs[0])
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i][0], want[2 + i][0]) and torch.equal(outs[i][1], want[2 + i][1])
    assert mg.device_status() == 0


# ------------------------------------------------------------------------------ where calls go wrong

@pytest.mark.parametrize("opts, M", [(dict(INT8_PAIR=0, INT8_TOKENS=64, INT8_SPLIT=1), 40), (dict(INT8_PAIR=0, INT8_TOKENS=32, INT8_SPLIT=4), 20),
                                     (dict(INT8_PAIR=1), 700)])
def test_a_wait_that_runs_out_is_reported_and_the_context_survives(opts, M, mgopt):
    """Host-side fault injection: the first CTA withholds its second stage load.  With the wait limit at
    1 ms the kernel gives up, stores nothing of that tile and returns; the status word says so once."""
    import mixedgemm_b200 as mg
    for name, v in opts.items():
        mgopt.set(name, v)
    N, K = 900, 2048
    _, av = codes(M, K, 1)
    _, bv = codes(N, K, 2)
    sa, sb = torch.rand(M, device="cuda") + 1, torch.rand(N, device="cuda") + 1
    want = mg.matmul_int8(av, bv, sa, sb)
    torch.cuda.synchronize()
    mg.set_wait_limit_us(1000)
    mgopt.set("FAULT_SKIP_LOAD", 2)
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
    mg.matmul_int8(av, bv, sa, sb, out=out)
    torch.cuda.synchronize()
    assert mg.device_status() & (1 | 2 | 8)
    assert bool((out[:20, :128] == 7).all())  # the tile of the CTA that gave up
    mgopt.set("FAULT_SKIP_LOAD", 0)
    mg.set_wait_limit_us(0)
    assert mg.device_status() == 0
    assert torch.equal(mg.matmul_int8(av, bv, sa, sb), want)
    assert mg.device_status() == 0


def test_offsets_beyond_32_bits():
    import mixedgemm_b200 as mg
    M, K = 140001, 16384  # 2.3e9 elements, 4.6 GB
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    for r0 in range(0, M, 20000):
        x[r0:r0 + 20000].normal_()
    rows = [0, 1, 70000, 131071, 131072, M - 2, M - 1]
    q, s = mg.quantize_int8(x)
    part = x[rows].cpu()
    wq, ws = want_codes(part)
    assert np.array_equal(q[rows].cpu().numpy(), wq) and np.array_equal(s[rows].cpu().numpy(), ws)
    w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(torch.bfloat16)
    got = mg.rms_norm_int8(x, w.cuda(), eps=1e-5, residual=x, residual_out=x, out=(q, s))
    check_norm([t[rows] for t in got], part, w, part, 1e-5)
    # codes of 2.3 GB times a few channels, and a result of 2.6e9 elements
    b, bv = codes(40, K, 1)
    sb = torch.rand(40)
    y = mg.matmul_int8(q, bv, s, sb.cuda(), out_dtype=torch.float32)
    check_product(y[rows], q[rows].cpu(), b, s[rows].cpu(), sb, None)
    del x, y, got
    M, N, K = 65537, 40000, 48
    a, av = codes(M, K, 2)
    b, bv = codes(N, K, 3)
    sa, sb = torch.rand(M) * 0.01, torch.rand(N) * 0.01
    y = mg.matmul_int8(av, bv, sa.cuda(), sb.cuda())
    rows = [0, 53687, 53688, M - 1]
    check_product(y[rows], a[rows], b, sa[rows], sb, None)
    assert mg.device_status() == 0


def test_first_calls_inside_a_capture():
    """A fresh process whose first call of every form is made while a graph is being captured."""
    import os
    import subprocess
    import sys
    code = """
import torch
import mixedgemm_b200 as mg
torch.manual_seed(0)
shapes = [(1, 512, 1024), (20, 512, 4096), (60, 4096, 512), (100, 512, 1024), (700, 4096, 512), (150, 6000, 256)]
xs = [torch.randn(M, K, device="cuda", dtype=torch.bfloat16) for M, N, K in shapes]
ws = [torch.randn(N, K, device="cuda", dtype=torch.bfloat16) for M, N, K in shapes]
g1 = [torch.ones(K, device="cuda", dtype=torch.bfloat16) for M, N, K in shapes]
idx = [torch.arange(K, device="cuda").to(torch.int16) for M, N, K in shapes]
def run():
    outs = []
    for x, w, g, i in zip(xs, ws, g1, idx):
        q, s, u = mg.rms_norm_int8(x, g, residual=x)
        b, sb = mg.quantize_int8(w)
        K = x.shape[1]
        outs += [mg.matmul_int8(q, b, s, sb), u] + list(mg.rms_norm_reorder_quantize_x(x, g, i, K // 2, K // 4, K // 4)[:3])
    return outs
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
assert mg.device_status() == 0
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_two_host_threads_on_their_own_streams():
    import threading
    import mixedgemm_b200 as mg
    N, K = 600, 1024
    bq, sb = mg.quantize_int8((torch.randn(N, K, generator=gen(5)) * 0.02).cuda())
    w = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    xs = [tokens(M, K, torch.bfloat16, seed=M).cuda() for M in (1, 9, 70, 300)]

    def layer(x):
        q, s, u = mg.rms_norm_int8(x, w, residual=x)
        return mg.matmul_int8(q, bq, s, sb), u

    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(40):
                    j = (i + k) % len(xs)
                    got = layer(xs[j])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[j])):
                        bad.append((k, i))
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad, bad
    assert mg.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", (8193, 10477, 16380, 16383, 16384))
def test_long_rows_one_after_another(K, dtype):
    """More rows than CTAs, each kept in a CTA's registers (or read twice) while the next one is fetched."""
    import mixedgemm_b200 as mg
    M = 333
    x, r = tokens(M, K, dtype, seed=K), tokens(M, K, dtype, seed=K + 1)
    w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(dtype)
    q, s = mg.quantize_int8(x.cuda())
    wq, ws = want_codes(x)
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)
    check_norm(mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5), x, w, None, 1e-5)
    rd = r.cuda()
    check_norm(mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5, residual=rd, residual_out=rd), x, w, r, 1e-5)


def test_columns_of_one_tensor_are_apart_and_shared_bytes_are_refused():
    """x, the residual, the stream, the codes, the scales and a result between one another's rows are taken, and give
    what separate tensors give; a shared byte is refused, but for the stream over x or the residual."""
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import _capi
    M, K = 33, 64
    x, r = tokens(M, K, torch.bfloat16, seed=1).cuda(), tokens(M, K, torch.bfloat16, seed=2).cuda()
    w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(torch.bfloat16).cuda()
    q0, s0, u0 = mg.rms_norm_int8(x, w, residual=r)
    y0 = mg.matmul_int8(q0, q0, s0, s0)
    whole = torch.zeros(M, 1024, dtype=torch.int8, device="cuda")
    part = lambda b0, b1, t: whole[:, b0:b1].view(t)
    xv, rv, uv = part(0, 128, torch.bfloat16), part(128, 256, torch.bfloat16), part(256, 384, torch.bfloat16)
    qv, yv = part(384, 448, torch.int8), part(448, 448 + 2 * M, torch.bfloat16)
    xv.copy_(x), rv.copy_(r)
    q, s, u = mg.rms_norm_int8(xv, w, residual=rv, residual_out=uv, out=(qv, torch.empty_like(s0)))
    assert torch.equal(q, q0) and torch.equal(s, s0) and torch.equal(u, u0)
    assert torch.equal(mg.matmul_int8(qv, qv, s, s, out=yv), y0)
    assert torch.equal(xv, x) and torch.equal(rv, r) and torch.equal(qv, q0) and torch.equal(uv, u0)
    assert torch.equal(mg.quantize_int8(xv, out=(qv, s))[0], mg.quantize_int8(x)[0])
    before = whole.clone()
    fresh = lambda: (torch.empty_like(q0), torch.empty_like(s0))
    bad = [
        lambda: mg.quantize_int8(xv, out=(part(0, 64, torch.int8), s)), lambda: mg.quantize_int8(xv, out=(part(127, 191, torch.int8), s)),
        lambda: mg.quantize_int8(part(0, 256, torch.float32)[:1], out=(qv[:1], part(252, 256, torch.float32)[0])),
        lambda: mg.rms_norm_int8(xv, w, residual=rv, residual_out=part(2, 130, torch.bfloat16), out=fresh()),
        lambda: mg.rms_norm_int8(xv, w, residual=rv, residual_out=part(254, 382, torch.bfloat16), out=fresh()),
        lambda: mg.rms_norm_int8(xv[:-1], w, residual=rv[:-1], residual_out=xv[1:]), lambda: mg.rms_norm_int8(xv, xv[4], residual=rv, residual_out=xv),
        lambda: mg.rms_norm_int8(xv, w, residual=rv, residual_out=uv, out=(part(320, 384, torch.int8), s)),
        lambda: mg.matmul_int8(qv, qv, s, s, out=part(400, 400 + 2 * M, torch.bfloat16)),
        lambda: mg.matmul_int8(qv, q0, s, s, out=part(384 - 2 * M + 1 + 1, 386, torch.bfloat16)),
        lambda: mg.matmul_int8(q0[:1], q0, s[:1], s, out=s[None], out_dtype=torch.float32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_capi.MixedGemmError) as e:
            call()
            pytest.fail("case %d was not refused" % i)
        assert e.value.status == 9, (i, str(e.value))
    assert torch.equal(whole, before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K", [(20011, 31), (20011, 64), (20011, 500), (20011, 512), (296, 8192), (296, 4096), (296, 4093), (5003, 1931), (5003, 4096)])
def test_short_rows_one_after_another(M, K, dtype):
    """More rows than threads take at once, in every form for rows up to 8192: a warp to a row, one chunk a thread
    (8192 bf16 or fp16, 4096 fp32 and 4093 need 1024 threads, one CTA to an SM), four chunks a thread.  Each takes
    several rows, the next on its way while one is reduced."""
    import mixedgemm_b200 as mg
    x, r = tokens(M, K, dtype, seed=K), tokens(M, K, dtype, seed=K + 1)
    w = (1 + 0.2 * torch.randn(K, generator=gen(3))).to(dtype)
    q, s = mg.quantize_int8(x.cuda())
    wq, ws = want_codes(x)
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)
    check_norm(mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5), x, w, None, 1e-5)
    rd = r.cuda()
    check_norm(mg.rms_norm_int8(x.cuda(), w.cuda(), eps=1e-5, residual=rd, residual_out=rd), x, w, r, 1e-5)
