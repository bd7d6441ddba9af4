"""Launches that overlap: every kernel lets the next one start while it still writes, and the next one has to
read what was written all the same.  Every chain is run a few hundred times on new inputs through the same
buffers without a synchronisation in between, and has to give the bytes of a run with programmatic launches
off."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TURNS = 300


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same_without_overlap(mgopt, chain, outs):
    """chain(i) writes turn i's results into outs[k][i]."""
    mgopt.set("PDL", 1)
    for i in range(TURNS):
        chain(i)
    torch.cuda.synchronize()
    got = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    mgopt.set("PDL", 0)
    for i in range(TURNS):
        chain(i)
    torch.cuda.synchronize()
    for a, b in zip(got, outs):
        assert torch.equal(a, b)
    assert any(not torch.equal(got[0][0], got[0][i]) for i in range(1, TURNS))  # the inputs were new ones


@pytest.mark.parametrize("M", [1, 2, 3])
@pytest.mark.parametrize("K", [1024, 4096])
def test_tokens_quantised_right_before_their_product(M, K, mgopt):
    import mixedgemm_b200 as mg
    N = 1000
    xs = torch.randn(TURNS, M, K, generator=gen(1)).to(torch.bfloat16).cuda()
    w = (1 + 0.2 * torch.randn(K, generator=gen(2))).to(torch.bfloat16).cuda()
    bq, sb = mg.quantize_int8((torch.randn(N, K, generator=gen(3)) * 0.02).cuda())
    q, s = mg.quantize_int8(xs[0])  # the buffers of every turn
    y = torch.zeros(TURNS, M, N, device="cuda")

    def chain(i):
        mg.rms_norm_int8(xs[i], w, out=(q, s))
        mg.matmul_int8(q, bq, s, sb, out=y[i])

    same_without_overlap(mgopt, chain, [y])


@pytest.mark.parametrize("M", [1, 2, 3])
def test_weights_quantised_right_before_their_product(M, mgopt):
    import mixedgemm_b200 as mg
    N, K = 296, 2048
    ws = torch.randn(TURNS, N, K, generator=gen(4)).to(torch.bfloat16).cuda()
    q, s = mg.quantize_int8(torch.randn(M, K, generator=gen(5)).cuda())
    bq, sb = mg.quantize_int8(ws[0])
    y = torch.zeros(TURNS, M, N, device="cuda")

    def chain(i):
        mg.quantize_int8(ws[i], out=(bq, sb))
        mg.matmul_int8(q, bq, s, sb, out=y[i])

    same_without_overlap(mgopt, chain, [y])


def test_a_norm_whose_weight_a_product_has_just_written(mgopt):
    import mixedgemm_b200 as mg
    M, K = 40, 1024
    split = (640, 256, 128)
    a, sa = mg.quantize_int8(torch.randn(TURNS, 256, generator=gen(6)).cuda())
    b, sb = mg.quantize_int8(torch.randn(K, 256, generator=gen(7)).cuda())
    x = torch.randn(M, K, generator=gen(8)).to(torch.bfloat16).cuda()
    order = torch.randperm(K, generator=gen(9)).to(torch.int16).cuda()
    w = torch.empty(1, K, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(TURNS, M, K, dtype=torch.int8, device="cuda")
    s = torch.zeros(TURNS, M, device="cuda")
    mx = mg.alloc_quantized_x(M, *split, "cuda")
    kept = [torch.zeros(TURNS, *t.shape, dtype=torch.uint8, device="cuda") for t in mx[:3]]

    def chain(i):
        mg.matmul_int8(a[i:i + 1], b, sa[i:i + 1], sb, out=w)
        mg.rms_norm_int8(x, w[0], out=(q[i], s[i]))
        mg.matmul_int8(a[i:i + 1], b, sa[i:i + 1], sb, out=w)
        mg.rms_norm_reorder_quantize_x(x, w[0], order, *split, out=mx)
        for k, t in zip(kept, mx):
            k[i].copy_(t)

    same_without_overlap(mgopt, chain, [q, s] + kept)


def test_a_quantiser_whose_index_was_just_found(mgopt):
    import mixedgemm_b200 as mg
    M, K, split = 64, 1024, (640, 256, 128)
    xs = torch.randn(TURNS, M, K, generator=gen(10))
    xs *= torch.exp2(torch.randn(TURNS, 1, K, generator=gen(11)))
    xs = xs.to(torch.bfloat16).cuda()
    mx = mg.alloc_quantized_x(M, *split, "cuda")
    kept = [torch.zeros(TURNS, *t.shape, dtype=torch.uint8, device="cuda") for t in mx[:3]]
    order = torch.zeros(TURNS, K, dtype=torch.int16, device="cuda")

    def chain(i):
        idx = mg.reorder_index(xs[i])
        mg.reorder_quantize_x(xs[i], idx, *split, out=mx)
        order[i].copy_(idx)
        for k, t in zip(kept, mx):
            k[i].copy_(t)

    same_without_overlap(mgopt, chain, [order] + kept)
