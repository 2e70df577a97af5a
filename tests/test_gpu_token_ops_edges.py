"""-m gpu: edges of the token-side operators - beams that lie closer together than fp32 tells apart, narrow and wide tables, states
whose memory holds other values than they stand for, loss scales past fp32's range."""
import pytest
import torch

from gvd_amd import hip, ops, optim

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace('torch.', '')      # noqa: E731


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ beam_select
def select_want(logits, scores, W):
    """The definition in 64 bits: beams and words of the best W, and the least distance between neighbours of different beams among
    the best W + 1."""
    B, K = scores.shape
    x = logits.double().view(B, K, -1)
    V = x.shape[2]
    m = x.max(dim=2, keepdim=True)[0]
    cand = scores.double().unsqueeze(2) + (x - (m + (x - m).exp().sum(2, keepdim=True).log()))
    best, at = cand.view(B, K * V).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :W + 1], at[:, :W + 1]
    gap = torch.where(at[:, :W] // V != at[:, 1:] // V, best[:, :W] - best[:, 1:], torch.ones((), device='cuda', dtype=torch.float64))
    return at[:, :W] // V, at[:, :W] % V, gap.min(dim=1)[0]


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('V', [3, 50, 700, 5000, 70001])
def test_beam_select_orders_beams_that_are_close(V, dtype):
    """Every beam's score is set so that its best word comes out where the first beam's does, but for the score's rounding to fp32 (up
    to some 1e-7 between beams): the order is the definition's.  Both sides hold the log-sum-exp in fp64, to some 1e-14 (a relative
    error of a few 2^-53 in every term, all of one sign, and in the logarithm); pairs of beams closer than 1e-12 are left out, and
    there are hardly any."""
    B, K = 64, 4
    x = (torch.randn(B * K, V, generator=gen(V), device='cuda') * 3).to(dtype)
    lp = x.double().log_softmax(dim=1).max(dim=1)[0].view(B, K)
    scores = (lp[:, :1] - lp).float()
    for W in (K, 1):
        beam, word, gap = select_want(x, scores, W)
        _, parent, got, _ = ops.beam_select(x, scores, width=W)
        apart = gap > 1e-12
        assert int(apart.sum()) > 0.9 * B
        first = torch.arange(B, device='cuda').unsqueeze(1) * K
        assert torch.equal((parent - first)[apart], beam[apart]) and torch.equal(got[apart], word[apart])
        places = (parent * V + got).sort(dim=1)[0]
        assert bool((places[:, 1:] > places[:, :-1]).all())                       # no candidate twice


# -------------------------------------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize('n', [1, 5, 300, 4096])
@pytest.mark.parametrize('V,E', [(32768, 32), (32769, 32), (131072, 33), (1 << 20, 8), (1 << 21, 1), (200, 70001), (65, 1 << 17)])
def test_embedding_gradient_of_narrow_and_wide_tables(V, E, n):
    """Few tokens of tables on both sides of the rule that chooses the one-launch gradient.  The numbers are small multiples of a
    power of two, so that sums in any order are exact."""
    g = gen(n + V)
    tok = torch.randint(0, V, (n,), generator=g, device='cuda') * (torch.rand(n, generator=g, device='cuda') < 0.5)
    w = torch.randint(-4, 5, (V, E), generator=g, device='cuda').float().requires_grad_()
    dy = torch.randint(-8, 9, (n, E), generator=g, device='cuda').float()
    grad, = torch.autograd.grad(ops.embedding(tok, w, scale=0.5, act=1), w, dy)
    used = torch.unique(tok)
    want = torch.zeros(len(used), E, device='cuda').index_add_(0, torch.searchsorted(used, tok), dy) * 0.5 * (w.detach()[used] > 0)
    assert torch.equal(grad[used], want)
    grad[used] = 0
    assert not bool(grad.any())


# ----------------------------------------------------------------------------------------------------------- reorder_rows
def test_reorder_of_conjugated_and_negated_views():
    """Views whose values are not what their memory holds (lazy conjugation and negation) come out as index_select's."""
    p = torch.tensor([3, 0, 0, 2], device='cuda')
    z = torch.randn(2, 4, 5, generator=gen(1), device='cuda', dtype=torch.complex64)
    for x, d in ((z.conj(), 1), (z[0].conj(), 0), (z.conj().imag[:, :, 2], 1), (torch._neg_view(z.real.contiguous()), 1)):
        assert x.is_conj() or x.is_neg()
        got, = ops.reorder_rows([x], p, dim=d)
        want = x.index_select(d, p)
        assert torch.equal(got, want)
        out = torch.empty_like(want)
        ops.reorder_rows([x], p, dim=d, out=[out])
        assert torch.equal(out, want)
    for out in (torch.empty_like(z).conj(), torch._neg_view(torch.empty(2, 4, 5, device='cuda'))):
        with pytest.raises(hip.GvdHipError, match='conjugated or negated'):
            ops.reorder_rows([z if out.is_complex() else z.real], p, dim=1, out=[out])


# ------------------------------------------------------------------------------------------------------------------- clip
@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('inv', [1e30, 1e39, 1e100])
def test_clip_by_factors_over_the_range_of_fp32(inv, dtype):
    """A loss scale far under 1: the factor does not fit fp32, products that do come out, zeros stay zeros, the rest is infinite."""
    g = torch.tensor([0.0, -0.0, 2.0 ** -24, -2.0 ** -14, 1.0], device='cuda').to(dtype)
    out = torch.full((5,), 7.0, device='cuda')
    norm = optim.clip_grads([g], float('inf'), out=[out], inv_scale=inv)
    want = g.double() * inv
    big = want.abs() > torch.finfo(torch.float32).max
    assert torch.equal(torch.isinf(out), big) and torch.equal(torch.signbit(out), torch.signbit(want))
    # the factor, the product and a power of two: two roundings (values here are no subnormal numbers)
    assert bool(((out.double() - want).abs()[~big] <= want.abs()[~big] * 2.01 * 2.0 ** -24).all())
    assert float(norm) == float((g.double().square().sum().sqrt() * inv).float())
