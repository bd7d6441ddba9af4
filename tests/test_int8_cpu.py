"""8-bit operators: what is refused, checked without a GPU (the C entry points answer shape, null and
alignment errors before any CUDA call; the Python layer refuses tensors that are not on a GPU)."""
import pytest
import torch

OK, SHAPE, NULL, ALIGN = 0, 1, 2, 3
P = 4096        # stands for an aligned device pointer: never dereferenced, the call is refused first
MAX_K = 131071


@pytest.fixture(scope="module")
def lib():
    from mixedgemm_b200 import build, _capi
    build.build_lib()
    return _capi.load()


def quantise(lib, X=P, dtype=0, M=4, K=64, ldx=64, Q=P, ldq=64, S=P):
    return lib.mg_quantize_int8(X, dtype, M, K, ldx, Q, ldq, S, None)


@pytest.mark.parametrize("want, args", [
    (OK, dict(M=0, X=None, Q=None, S=None)),
    (SHAPE, dict(M=-1)), (SHAPE, dict(K=0)), (SHAPE, dict(K=MAX_K + 1, ldx=1 << 20, ldq=1 << 20)),
    (SHAPE, dict(dtype=3)), (SHAPE, dict(dtype=-1)), (SHAPE, dict(ldx=63)), (SHAPE, dict(ldq=63)),
    (NULL, dict(X=None)), (NULL, dict(Q=None)), (NULL, dict(S=None)),
    (ALIGN, dict(X=P + 1)), (ALIGN, dict(dtype=2, X=P + 2)), (ALIGN, dict(S=P + 2)),
])
def test_quantise_refusals(lib, want, args):
    assert quantise(lib, **args) == want


def norm(lib, X=P, R=None, W=P, eps=1e-6, dtype=0, M=4, K=64, ldx=64, ldr=0, U=None, ldu=0, Q=P, ldq=64, S=P):
    return lib.mg_rms_norm_int8(X, R, W, eps, dtype, M, K, ldx, ldr, U, ldu, Q, ldq, S, None)


@pytest.mark.parametrize("want, args", [
    (OK, dict(M=0, X=None, W=None, Q=None, S=None)),
    (SHAPE, dict(M=-1)), (SHAPE, dict(K=0)), (SHAPE, dict(K=MAX_K + 1, ldx=1 << 20, ldq=1 << 20)), (SHAPE, dict(dtype=3)),
    (SHAPE, dict(eps=-1e-6)), (SHAPE, dict(eps=float("nan"))), (SHAPE, dict(eps=float("inf"))),
    (SHAPE, dict(R=P, U=P, ldr=63, ldu=64)), (SHAPE, dict(R=P, U=P, ldr=64, ldu=63)),
    (NULL, dict(W=None)), (NULL, dict(R=P, ldr=64, ldu=64)), (NULL, dict(U=P, ldu=64)),
    (ALIGN, dict(W=P + 1)), (ALIGN, dict(R=P + 1, U=P, ldr=64, ldu=64)), (ALIGN, dict(R=P, U=P + 1, ldr=64, ldu=64)),
])
def test_norm_refusals(lib, want, args):
    assert norm(lib, **args) == want


def product(lib, A=P, lda=64, B=P, ldb=64, sa=P, sb=P, bias=None, M=4, N=8, K=64, D=P, dtype=0, ldd=8):
    return lib.mg_matmul_int8(A, lda, B, ldb, sa, sb, bias, M, N, K, D, dtype, ldd, None)


@pytest.mark.parametrize("want, args", [
    (OK, dict(M=0, A=None, D=None)), (OK, dict(N=0, B=None, D=None)),
    (SHAPE, dict(M=-1)), (SHAPE, dict(N=-1)), (SHAPE, dict(K=0)), (SHAPE, dict(K=MAX_K + 1, lda=1 << 20, ldb=1 << 20)),
    (SHAPE, dict(dtype=3)), (SHAPE, dict(lda=48)), (SHAPE, dict(ldb=48)), (SHAPE, dict(ldd=7)),
    (SHAPE, dict(lda=1 << 40)), (SHAPE, dict(ldb=1 << 40)), (SHAPE, dict(M=0x7fffffff)), (SHAPE, dict(N=0x7fffffff, ldd=0x7fffffff)),
    (ALIGN, dict(lda=72)), (ALIGN, dict(ldb=65)), (ALIGN, dict(A=P + 8)), (ALIGN, dict(B=P + 1)), (ALIGN, dict(sa=P + 2)),
    (ALIGN, dict(sb=P + 1)), (ALIGN, dict(bias=P + 2)), (ALIGN, dict(D=P + 1)), (ALIGN, dict(D=P + 2, dtype=2)),
    (NULL, dict(A=None)), (NULL, dict(B=None)), (NULL, dict(sa=None)), (NULL, dict(sb=None)), (NULL, dict(D=None)),
])
def test_product_refusals(lib, want, args):
    assert product(lib, **args) == want


def test_python_layer_refuses_tensors_off_the_gpu():
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import build
    build.build_ext()
    x, q, s = torch.zeros(2, 32), torch.zeros(2, 32, dtype=torch.int8), torch.ones(2)
    for call in (lambda: mg.quantize_int8(x), lambda: mg.rms_norm_int8(x, torch.ones(32)),
                 lambda: mg.matmul_int8(q, q, s, s)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def mx_norm(lib, X=P, ldx=128, R=None, ldr=0, W=P, eps=1e-6, U=None, ldu=0, M=4, K=128, idx=P, split=(64, 32, 32), codes=P, scales=P):
    return lib.mg_rms_norm_reorder_quantize(X, ldx, R, ldr, W, eps, U, ldu, M, K, idx, *split, codes, codes, codes, None,
                                            scales, scales, scales, None)


@pytest.mark.parametrize("want, args", [
    (OK, dict(M=0, X=None, W=None, idx=None, codes=None, scales=None)),
    (SHAPE, dict(M=-1)), (SHAPE, dict(K=120)), (SHAPE, dict(split=(80, 16, 32))), (SHAPE, dict(eps=-1.0)), (SHAPE, dict(eps=float("nan"))),
    (SHAPE, dict(ldx=120)), (SHAPE, dict(R=P, U=P, ldr=120, ldu=128)), (SHAPE, dict(R=P, U=P, ldr=128, ldu=120)),
    (NULL, dict(X=None)), (NULL, dict(W=None)), (NULL, dict(idx=None)), (NULL, dict(codes=None)), (NULL, dict(scales=None)),
    (NULL, dict(R=P, ldr=128, ldu=128)), (NULL, dict(U=P, ldr=128, ldu=128)),
    (ALIGN, dict(X=P + 2)), (ALIGN, dict(W=P + 1)), (ALIGN, dict(ldx=132)), (ALIGN, dict(R=P + 2, U=P, ldr=128, ldu=128)),
    (ALIGN, dict(R=P, U=P, ldr=130, ldu=128)), (ALIGN, dict(R=P, U=P, ldr=128, ldu=129)), (ALIGN, dict(codes=P + 4)),
])
def test_mx_norm_refusals(lib, want, args):
    assert mx_norm(lib, **args) == want


def test_shapes_of_the_torch_operators():
    """What tracing sees: the operators' fake implementations return the shapes and types of the real ones."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    import mixedgemm_b200.linear  # noqa: F401
    ops = torch.ops.mixedgemm_b200
    with FakeTensorMode():
        x, w = torch.empty(7, 64, dtype=torch.float16), torch.empty(64, dtype=torch.float16)
        q, s = torch.empty(40, 64, dtype=torch.int8), torch.empty(40)
        y = ops.int8_linear(x, q, s, None)
        assert y.shape == (7, 40) and y.dtype == torch.float16
        y, u = ops.int8_norm_linear(x, x, w, 1e-6, q, s, None)
        assert y.shape == (7, 40) and u.shape == (7, 64) and u.dtype == torch.float16
        assert ops.int8_norm_linear(x, None, w, 1e-6, q, s, None)[1].shape == (1,)
        x, w = x.bfloat16(), w.bfloat16()
        parts = [torch.empty(256, n, dtype=torch.uint8) for n in (16, 8, 8)] + [torch.empty(4096, dtype=torch.uint8)] * 3
        idx = torch.empty(64, dtype=torch.int16)
        y, u = ops.mixed_norm_linear(x, x, w, 1e-6, idx, [32, 16, 16], parts, [])
        assert y.shape == (7, 256) and y.dtype == torch.bfloat16 and u.shape == (7, 64)
        a, b, u = ops.mixed_norm_linear(torch.empty(200, 64, dtype=torch.bfloat16), None, w, 1e-6, idx, [32, 16, 16], parts * 2, parts)
        assert a.shape == b.shape == (200, 256) and u.shape == (1,)


@pytest.mark.parametrize("state", [dict(version=2), dict()])
def test_int8_container_refuses_unknown_versions(state):
    from mixedgemm_b200.linear import Int8Weights
    with pytest.raises(RuntimeError, match="version"):
        Int8Weights.from_state(dict(codes=torch.zeros(2, 32, dtype=torch.int8), scale=torch.ones(2), **state), "cpu")


def test_int8_container_round_trip_on_the_cpu(tmp_path):
    """The file holds dense codes; loading pads the rows to 16 bytes again."""
    from mixedgemm_b200.linear import Int8Weights
    q = torch.arange(3 * 37, dtype=torch.int8).view(3, 37)
    w = Int8Weights(q, torch.tensor([1.0, 2.0, 3.0]))
    w.save(str(tmp_path / "w.pt"))
    back = Int8Weights.load(str(tmp_path / "w.pt"), "cpu")
    assert torch.equal(back.codes, q) and torch.equal(back.scale, w.scale) and back.codes.stride() == (48, 1)
    assert (back.out_features, back.in_features) == (3, 37)
    a, b = Int8Weights(q.clone(), w.scale.clone()), Int8Weights(q.clone() + 1, w.scale * 2)
    whole = Int8Weights.cat([a, b])
    assert torch.equal(whole.codes, torch.cat([q, q + 1])) and torch.equal(b.scale, w.scale * 2)
    assert b.codes.data_ptr() == whole.codes[3:].data_ptr()
    with pytest.raises(ValueError):
        Int8Weights.cat([a, Int8Weights(q[:, :20].contiguous(), w.scale)])


@pytest.mark.parametrize("there", [False, True])
def test_a_compiled_module_that_is_missing_or_does_not_load(there, monkeypatch, tmp_path):
    """matmul then takes the ctypes route (and says once that the file does not load); the operators that have no
    other route say why."""
    import warnings
    import mixedgemm_b200 as mg
    from mixedgemm_b200 import api, build
    path = tmp_path / "mixedgemm_ops.so"
    if there:
        path.write_bytes(b"not a shared object")
    monkeypatch.setattr(build, "ext_path", lambda name="mixedgemm": str(path))
    monkeypatch.setattr(api, "_ops_module", None)
    monkeypatch.setattr(api, "_ops_failure", None)
    codes, scale = torch.zeros(1, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        for _ in range(2):
            with pytest.raises(RuntimeError, match="code tensors must be"):  # the ctypes route's check
                mg.matmul(*[codes] * 6, *[scale] * 6)
    assert len(seen) == there and all("does not load" in str(w.message) for w in seen)
    with pytest.raises(ImportError, match="does not load" if there else "is not built"):
        mg.quantize_int8(torch.zeros(2, 32))


def _cpu_weights(K=64, N=128):
    """QuantizedWeights of nothing, for what a module does when it is made."""
    import mixedgemm_b200 as mg
    from mixedgemm_b200.linear import QuantizedWeights
    split = (K // 2, K // 4, K // 4)
    return QuantizedWeights(mg.alloc_quantized_w(N, *split, "cpu"), torch.arange(K, dtype=torch.int16), split, N)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_norm_weight_of_another_type_is_not_rounded_without_a_word(dtype):
    import warnings
    from mixedgemm_b200.linear import Int8Linear, Int8Weights, MixedLinear
    rough, fine = torch.full((64,), 1.25, dtype=dtype), torch.full((64,), 1 + 2.0 ** -9, dtype=dtype)
    with pytest.warns(UserWarning, match="rounded"):
        lin = MixedLinear(_cpu_weights(), norm_weight=fine)
    assert lin.norm_weight.dtype == torch.bfloat16 and torch.equal(lin.norm_weight, fine.bfloat16())
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert torch.equal(MixedLinear(_cpu_weights(), norm_weight=rough).norm_weight, rough.bfloat16())
        assert torch.equal(MixedLinear(_cpu_weights(), norm_weight=fine.bfloat16()).norm_weight, fine.bfloat16())
        w = Int8Weights(torch.zeros(128, 64, dtype=torch.int8), torch.ones(128))
        assert torch.equal(Int8Linear(w, norm_weight=fine).norm_weight, fine)


def test_a_module_with_a_norm_keeps_no_buffers_that_it_never_uses():
    from mixedgemm_b200.linear import MixedLinear
    assert MixedLinear(_cpu_weights(), max_tokens=40)._a is not None
    assert MixedLinear(_cpu_weights(), max_tokens=40, norm_weight=torch.ones(64).bfloat16())._a is None


# ------------------------------------------------------------------- outputs in the place of inputs

OVERLAP = 9


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    """overlap.h behind a C function of two spans (start, rows, bytes, pitch)."""
    import ctypes
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    d = tmp_path_factory.mktemp("overlap")
    (d / "o.cpp").write_text(
        '#include "overlap.h"\n'
        'extern "C" int f(const size_t* v) { return mg::overlap(mg::Span((void*)v[0], v[1], v[2], v[3]), '
        'mg::Span((void*)v[4], v[5], v[6], v[7])); }\n')
    subprocess.check_call(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(root, "mixedgemm_b200", "csrc"),
                           str(d / "o.cpp"), "-o", str(d / "o.so")])
    f = ctypes.CDLL(str(d / "o.so")).f
    return lambda a, b: bool(f((ctypes.c_size_t * 8)(*a, *b)))


def test_overlap_of_rows_is_what_their_bytes_say(overlap):
    import random
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(20000):
        spans = []
        for _ in range(2):
            size = rng.randint(0, 12)
            spans.append((rng.randint(1, 120), rng.randint(0, 6), size, size + rng.choice([0, 1, 5, 13, 20])))
        if rng.random() < 0.5:  # one pitch, as with columns of one tensor
            pitch = max(s[3] for s in spans)
            spans = [s[:3] + (pitch,) for s in spans]
        sets = [{p + r * pitch + i for r in range(rows) for i in range(size)} for p, rows, size, pitch in spans]
        want = bool(sets[0] & sets[1])
        seen[want] += 1
        assert overlap(*spans) == want, spans
    assert min(seen) > 3000


G = 1 << 40  # far from P


@pytest.mark.parametrize("args", [
    dict(Q=P), dict(Q=P + 4 * 64 * 2 - 1), dict(Q=P + 100, ldq=200), dict(Q=G, S=P + 3 * 128), dict(Q=G, S=G + 63 * 4),
    dict(Q=P + 127, ldx=100, ldq=200, K=64),
])
def test_quantise_refuses_outputs_over_its_input(lib, args):
    assert quantise(lib, **{**dict(S=2 * G), **args}) == OVERLAP


@pytest.mark.parametrize("args", [
    dict(Q=P), dict(S=P), dict(Q=2 * G), dict(S=2 * G + 64), dict(Q=3 * G), dict(Q=4 * G + 3), dict(S=4 * G),
    dict(U=P + 2), dict(U=P + 128), dict(U=P, ldu=72), dict(U=3 * G + 64), dict(U=2 * G), dict(U=2 * G + 126),
    dict(X=3 * G + 2, U=3 * G),
])
def test_norm_refuses_outputs_over_its_inputs(lib, args):
    base = dict(W=2 * G, R=3 * G, ldr=64, U=4 * G, ldu=64, Q=5 * G, S=6 * G)
    assert norm(lib, **{**base, **args}) == OVERLAP


@pytest.mark.parametrize("args", [
    dict(D=P), dict(D=G), dict(D=G + 7 * 64 + 62), dict(D=2 * G), dict(D=3 * G + 28), dict(D=4 * G - 2, ldd=1000), dict(D=4 * G + 28),
])
def test_product_refuses_a_result_over_its_operands(lib, args):
    base = dict(B=G, sa=2 * G, sb=3 * G, bias=4 * G)
    assert product(lib, **{**base, **args}) == OVERLAP


@pytest.mark.parametrize("args", [
    dict(codes=(P, G, 2 * G)), dict(codes=(G, G, 2 * G)), dict(codes=(G, G + 64, 2 * G)), dict(scales=(9 * G, 3 * G, 10 * G)),
    dict(scales=(4 * G, 9 * G, 10 * G)), dict(scales=(9 * G, 10 * G, 9 * G + 256)), dict(codes=(G, 5 * G, 2 * G)), dict(codes=(G, 2 * G, 6 * G)),
    dict(U=P + 16), dict(U=5 * G + 256), dict(U=3 * G), dict(U=4 * G), dict(U=P, ldu=136),
])
def test_mx_norm_refuses_outputs_over_its_inputs(lib, args):
    v = {**dict(codes=(G, 2 * G, 7 * G), scales=(8 * G, 9 * G, 10 * G), W=3 * G, idx=4 * G, R=5 * G, ldr=128, U=6 * G, ldu=128), **args}
    assert lib.mg_rms_norm_reorder_quantize(P, 128, v["R"], v["ldr"], v["W"], 1e-6, v["U"], v["ldu"], 4, 128, v["idx"], 64, 32, 32,
                                            *v["codes"], None, *v["scales"], None) == OVERLAP
