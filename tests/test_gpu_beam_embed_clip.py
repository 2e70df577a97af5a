"""-m gpu: the token-side operators of training and search - embedding lookup with its gradient by sorted tokens, gradient norm
and clipping, beam selection, state reordering - against plain formulations in 64 bits.

Tolerances count roundings: u = half a step of a type relative to the value (fp32 2^-24, bf16 2^-8, fp16 2^-11; fp16 values under
2^-14 half a step of 2^-24 absolute).  A sum of m terms in fp32, in whatever order, is off by at most (m - 1) u32 times the
sum of the terms' magnitudes (to first order)."""
import math

import numpy as np
import pytest
import torch

from gvd_amd import hip, ops, optim

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace('torch.', '')      # noqa: E731


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def within(got, want64, bound64, what):
    """|got - want| <= bound, element by element."""
    off = (got.double() - want64).abs()
    bad = ~(off <= bound64)
    assert not bool(bad.any()), '%s: %d of %d off, worst %.3e against %.3e' % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound64.expand_as(off)[bad][off[bad].argmax()]))


# --------------------------------------------------------------------------------------------------------------- embedding
def words(kind, n, V, seed, dtype=torch.int64):
    g = gen(seed)
    if kind == 'uniform':
        t = torch.randint(0, V, (n,), generator=g, device='cuda')
    elif kind == 'one':
        t = torch.full((n,), V // 2, device='cuda')
    elif kind == 'half':                      # half of all is word 0, like padded captions
        t = torch.randint(0, V, (n,), generator=g, device='cuda') * (torch.rand(n, generator=g, device='cuda') < 0.5)
    elif kind == 'skew':
        t = (V * torch.rand(n, generator=g, device='cuda') ** 6).long().clamp_(max=V - 1)
    elif kind == 'down':                      # descending, every word as often
        t = (V - 1) - torch.arange(n, device='cuda') * V // n
    return t.to(dtype)


def embedding_want(tok, w, scale, act, dy, pad):
    """(out, gradient, sum of magnitudes per element of the gradient, terms per row) in 64 bits; tokens outside the table: NaN / nothing."""
    V = w.shape[0]
    inside = (tok >= 0) & (tok < V)
    rows = w.double() * scale
    if act:
        rows = torch.where(rows > 0, rows, torch.zeros_like(rows))
    t = torch.where(inside, tok, torch.zeros_like(tok)).long()
    out = torch.where(inside.unsqueeze(1), rows[t], torch.full((), float('nan'), device='cuda', dtype=torch.float64))
    use = inside if pad is None else inside & (tok != pad)
    d = torch.where(use.unsqueeze(1), dy.double(), torch.zeros((), device='cuda', dtype=torch.float64))
    k = scale * (w.double() * scale > 0) if act else torch.full((), scale, device='cuda', dtype=torch.float64)
    tc, dc = t.cpu(), d.cpu()
    add = lambda shape, x: torch.zeros(shape, dtype=torch.float64).index_add_(0, tc, x).cuda()      # noqa: E731
    return out, add(w.shape, dc) * k, add(w.shape, dc.abs()) * abs(scale), add((V,), use.double().cpu()).unsqueeze(1)


def check_embedding(tok, w, scale=1.0, act=0, pad=None, dy=None, what=''):
    w = w.detach().requires_grad_()
    n, E = tok.numel(), w.shape[1]
    out = ops.embedding(tok, w, scale, act, pad)
    assert out.shape == tok.shape + (E,) and out.dtype == w.dtype
    if dy is None:
        dy = torch.randn(tok.shape + (E,), generator=gen(n + E), device='cuda').to(w.dtype)
    grad, = torch.autograd.grad(out, w, dy)
    want, gw, mag, cnt = embedding_want(tok.reshape(-1), w.detach(), scale, act, dy.reshape(n, E), pad)
    got = out.detach().reshape(n, E)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    u = U[w.dtype]
    fine = ~torch.isnan(want)
    # the product in fp32, then the type: u32 + u of the value (an exact product: u alone)
    within(got[fine], want[fine], want[fine].abs() * ((1 + U[torch.float32]) * (1 + u) - 1) + TINY[w.dtype] / 2, what + ' out')
    # fp32 sums of cnt terms, the product with scale, the type
    assert grad.shape == w.shape and grad.dtype == w.dtype
    within(grad, gw, mag * (cnt + 1) * U[torch.float32] * 1.01 + gw.abs() * u * 1.01 + TINY[w.dtype], what + ' grad')
    return out, grad


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('n,V,E', [(1, 1, 1), (1, 5000, 512), (5, 3, 2), (63, 431, 300), (64, 432, 301), (65, 7, 64), (130, 2, 65),
                                   (1280, 5000, 512), (1281, 4999, 31), (4095, 300, 33), (4160, 64, 129), (8191, 1000, 257),
                                   (8192, 50, 1030), (8193, 50, 1030), (20011, 513, 40), (9000, 300000, 5)])
def test_embedding_sizes(n, V, E, dtype):
    tok = words('uniform', n, V, n + V)
    w = torch.randn(V, E, generator=gen(E), device='cuda').to(dtype)
    check_embedding(tok, w, 1.0, 0, what='plain')
    check_embedding(tok, w, math.sqrt(E), 1, what='scaled relu')


@pytest.mark.parametrize('kind', ['one', 'half', 'skew', 'down'])
@pytest.mark.parametrize('n,V,E', [(1280, 5000, 64), (3000, 17, 24), (4096, 900, 130), (4097, 900, 130), (7000, 40, 70), (20000, 5000, 96), (150001, 70000, 16), (140000, 400, 8)])
def test_embedding_repeated_tokens(kind, n, V, E):
    """Tokens that fill whole groups of 64 and of 4096 sorted positions, every sort path; int32 tokens; the same bits twice."""
    tok = words(kind, n, V, n, torch.int32)
    w = torch.randn(V, E, generator=gen(1), device='cuda')
    a = check_embedding(tok, w, 2.0, 1, what=kind)
    b = check_embedding(tok, w, 2.0, 1, what=kind)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('kind', ['uniform', 'one', 'half'])
@pytest.mark.parametrize('n', [1, 5, 31, 63, 64, 65, 1000, 1023, 1024, 1025, 4096])
def test_embedding_few_tokens_of_a_big_table(n, kind):
    """Tables that are sorted for, however few the tokens."""
    V, E = 70001, 129
    tok = words(kind, n, V, n)
    w = torch.randn(V, E, generator=gen(3), device='cuda')
    check_embedding(tok, w, 1.5, 1, what='%s %d' % (kind, n))


@pytest.mark.parametrize('n', [100, 9000])
def test_embedding_tokens_outside_and_padding(n):
    V, E = 37, 20
    tok = words('uniform', n, V, 3)
    tok[::7] = -1
    tok[3::11] = V
    tok[5::13] = 2 ** 40
    w = torch.randn(V, E, generator=gen(2), device='cuda')
    out, grad = check_embedding(tok, w, 0.5, 0, pad=4, what='outside')
    assert bool((grad[4] == 0).all()) and bool(torch.isnan(out[0]).all())
    a = ops.embedding(tok, w.requires_grad_(), padding_idx=-1)
    g, = torch.autograd.grad(a.nan_to_num().sum(), w)
    assert bool((g[V - 1] == 0).all()) and bool((g[0] != 0).any())


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
def test_embedding_strides(dtype):
    """A column block of a wider table, tokens in another order, gradients transposed and broadcast, 3-D tokens."""
    V, E = 50, 72
    wide = torch.randn(V, 200, generator=gen(5), device='cuda').to(dtype)
    tok = words('uniform', 60, V, 6).view(5, 12)
    for w in (wide[:, 3:3 + E], wide[::2][:25, 1:1 + E], torch.randn(E, V, generator=gen(7), device='cuda').to(dtype).t()):
        t = tok % w.shape[0]
        check_embedding(t, w, 1.5, 1, what='table')
        check_embedding(t.t(), w, 1.5, 0, what='tokens')
        check_embedding(t[:, ::3], w, 1.5, 0, what='tokens stepped')
        check_embedding(t.view(5, 3, 4), w, 1.5, 1, what='3-D')
        dy = torch.randn(E, generator=gen(8), device='cuda').to(dtype)
        check_embedding(t, w, 1.5, 1, dy=dy.expand(5, 12, E), what='one row for all')
        check_embedding(t, w, 1.5, 0, dy=dy[:1].expand(5, 12, E), what='one value for all')
        check_embedding(t, w, 1.5, 0, dy=torch.randn(E, 12, 5, generator=gen(9), device='cuda').to(dtype).permute(2, 1, 0), what='permuted')
    one = torch.randn(E, generator=gen(4), device='cuda').to(dtype)
    check_embedding(tok * 0, one.expand(1, E), 1.0, 0, what='one row')
    check_embedding(tok, one.expand(V, E), 1.0, 0, what='broadcast table')


def test_embedding_of_one_token():
    w = torch.randn(9, 6, device='cuda', requires_grad=True)
    for t in (torch.tensor(3, device='cuda'), torch.tensor([3], device='cuda', dtype=torch.int32)):
        out = ops.embedding(t, w, scale=2.0)
        assert out.shape == t.shape + (6,) and torch.equal(out.detach().view(-1), w.detach()[3] * 2)
        g, = torch.autograd.grad(out.sum(), w)
        assert float(g.sum()) == 12.0 and float(g[3].sum()) == 12.0


def test_embedding_of_nothing():
    w = torch.randn(9, 6, device='cuda', requires_grad=True)
    out = ops.embedding(torch.zeros(0, 4, dtype=torch.int64, device='cuda'), w)
    assert out.shape == (0, 4, 6)
    g, = torch.autograd.grad(out.sum(), w)
    assert torch.equal(g, torch.zeros_like(w))
    out = ops.embedding(torch.zeros(3, dtype=torch.int64, device='cuda'), torch.zeros(9, 0, device='cuda', requires_grad=True))
    assert out.shape == (3, 0)


def test_embedding_special_values():
    """NaN and infinities in the table go through; ReLU keeps a NaN and has slope 0 at 0 and below; rows not looked at do not matter."""
    w = torch.tensor([[1.0, -1.0, 0.0, -0.0], [float('nan'), float('inf'), float('-inf'), 2.0], [float('nan')] * 4], device='cuda',
                     requires_grad=True)
    tok = torch.tensor([0, 1, 0], device='cuda')
    out = ops.embedding(tok, w, act=1)
    assert torch.equal(out[0], torch.tensor([1.0, 0, 0, 0], device='cuda'))
    assert bool(torch.isnan(out[1, 0])) and out[1, 1:].tolist() == [float('inf'), 0.0, 2.0]
    dy = torch.ones_like(out)
    dy[1, 2] = float('nan')                       # under a slope of 0: not seen
    g, = torch.autograd.grad(out, w, dy)
    assert g.tolist() == [[2.0, 0, 0, 0], [0.0, 1.0, 0.0, 1.0], [0.0] * 4]


def test_embedding_gradient_against_differences():
    """The gradient of a loss against central differences; every number is a small multiple of a power of two, so they are exact."""
    V, E, n = 6, 5, 23
    tok = words('uniform', n, V, 11)
    w = (torch.randint(-8, 9, (V, E), generator=gen(12), device='cuda') * 2 + 1).float()       # odd: away from the kink at 0
    dy = torch.randint(-8, 9, (n, E), generator=gen(13), device='cuda').float()
    wr = w.clone().requires_grad_()
    grad, = torch.autograd.grad(ops.embedding(tok, wr, 0.5, 1), wr, dy)
    for v in range(V):
        for e in range(E):
            d = torch.zeros_like(w)
            d[v, e] = 0.25
            up, down = ((ops.embedding(tok, w + s * d, 0.5, 1) * dy).sum() for s in (1, -1))
            assert float(grad[v, e]) == float((up - down) / 0.5)


def test_embedding_past_32_bits():
    """A table, a result and a gradient of more than 2^32 bytes each (stores past the cache, nine tiles a sorting workgroup)."""
    V, E, n = 1100003, 2048, 1050007
    w = (torch.arange(V, device='cuda') % 61).to(torch.bfloat16).unsqueeze(1).expand(V, E).contiguous().requires_grad_()
    tok = torch.arange(n, device='cuda') * 7 % V
    tok[-5:] = V - 1
    out = ops.embedding(tok, w, scale=2.0)
    want = (tok % 61 * 2).to(torch.bfloat16)
    assert torch.equal(out.detach()[:, ::1023], want.unsqueeze(1).expand(n, 3)) and torch.equal(out.detach()[-1], want[-1].expand(E))
    dy = torch.randn(E, generator=gen(1), device='cuda').to(torch.bfloat16)
    grad, = torch.autograd.grad(out, w, dy.expand(n, E))
    times = torch.bincount(tok, minlength=V).float()
    assert float(times.max()) < 8                               # (times * 2 * dy: exact in fp32, rounded once)
    for cols in (slice(0, 3), slice(E - 2, E)):
        assert torch.equal(grad[:, cols], (times.unsqueeze(1) * 2.0 * dy[cols].float()).to(torch.bfloat16))
    assert torch.equal(grad[V - 1], (float(times[V - 1]) * 2.0 * dy.float()).to(torch.bfloat16))


def test_embedding_refuses_a_second_derivative_and_sees_changed_tables():
    w = torch.randn(5, 4, device='cuda', requires_grad=True)
    tok = torch.zeros(3, dtype=torch.int64, device='cuda')
    g, = torch.autograd.grad((ops.embedding(tok, w) ** 2).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    out = ops.embedding(tok, w, act=1)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


# ------------------------------------------------------------------------------------------------------------ clip / norm
def clip_want(grads, max_norm, inv):
    norm = math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads)) * inv
    factor = min(1.0, max_norm / (norm + 1e-6)) * inv
    return norm, factor


def check_clip(grads, got, norm, max_norm, inv, what):
    """got: the clipped tensors; grads: what they were."""
    want, factor = clip_want(grads, max_norm, inv)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= want * (U[torch.float32] + 1e-12), what                       # fp64 sums, one rounding
    for g, o in zip(grads, got):
        w = g.double() * factor
        # the factor and the product in fp32, then the type
        within(o, w, w.abs() * ((1 + U[torch.float32]) ** 2 * (1 + U[o.dtype]) - 1) * 1.001 + TINY[o.dtype] / 2, what)


def make_grads(sizes, types, seed, std=1.0):
    g = gen(seed)
    return [torch.randn(s, generator=g, device='cuda').mul_(std).to(t) for s, t in zip(sizes, types)]


@pytest.mark.parametrize('max_norm', [0.0, 0.1, 1e6, float('inf')])
@pytest.mark.parametrize('sizes', [[1], [3, 5, 8192, 8193, 1], [100003], [(7, 11, 13), (1,), (8191,), (64, 128)],
                                   [1 + (37 * i) % 301 for i in range(130)], [3, 0, 5]], ids=str)
def test_clip_in_place(sizes, max_norm):
    for types in ([torch.float32] * len(sizes), [TYPES[i % 3] for i in range(len(sizes))]):
        grads = make_grads(sizes, types, 1)
        was = [g.clone() for g in grads]
        n0 = optim.grad_norm(grads)
        norm = optim.clip_grads(grads, max_norm)
        assert torch.equal(n0, norm)
        check_clip(was, grads, norm, max_norm, 1.0, 'in place')
        if max_norm >= 1e6:
            assert all(torch.equal(a, b) for a, b in zip(was, grads))           # nothing to clip: the same bits
        again = [w.clone() for w in was]
        assert torch.equal(optim.clip_grads(again, max_norm), norm) and all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize('src', TYPES, ids=ids)
@pytest.mark.parametrize('dst', TYPES, ids=ids)
def test_clip_into_other_tensors(src, dst):
    """Into views of a flat buffer, at odd offsets; what lies between them is left alone; the gradients too."""
    sizes = [5, 8190, 1, 30001, 77]
    grads = make_grads(sizes, [src] * 5, 2, 3.0)
    was = [g.clone() for g in grads]
    flat = torch.full((sum(sizes) + 6,), 7.0, device='cuda', dtype=dst)
    out, at = [], 1
    for s in sizes:
        out.append(flat[at:at + s])
        at += s + 1
    for inv, mx in ((1.0, 1.0), (1.0 / 1024, 0.01), (0.3, 1e9)):
        norm = optim.clip_grads(grads, mx, out=out, inv_scale=inv)
        check_clip(was, out, norm, mx, inv, '%s %s' % (inv, mx))
        assert all(torch.equal(a, b) for a, b in zip(was, grads))
        gaps = flat.clone()
        at = 1
        for s in sizes:
            gaps[at:at + s] = 7.0
            at += s + 1
        assert bool((gaps == 7.0).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=ids)
def test_clip_more_than_the_cache_holds(dtype):
    """Results of over 256 MB take the stores past the cache; in place and into views at odd offsets."""
    sizes = [20000003, 8191, 60000001]
    grads = make_grads(sizes, [dtype] * 3, 12)
    flat = torch.zeros(sum(sizes) + 1, device='cuda')
    out = list(torch.split(flat[1:], sizes))
    norm = optim.clip_grads(grads, 100.0, out=out, inv_scale=0.5)
    check_clip(grads, out, norm, 100.0, 0.5, 'apart')
    was = [g.clone() for g in grads]
    norm = optim.clip_grads(grads, 100.0)
    check_clip(was, grads, norm, 100.0, 1.0, 'in place')


def test_clip_strides():
    """Transposed, permuted, stepped and offset gradients, in place and into results of other strides."""
    base = torch.randn(40, 60, generator=gen(3), device='cuda')
    grads = [base.t(), torch.randn(6, 5, 4, generator=gen(4), device='cuda').permute(2, 0, 1), torch.randn(33, 9, generator=gen(5), device='cuda')[::2, 1:8],
             torch.randn(1001, generator=gen(6), device='cuda', dtype=torch.bfloat16)[1:], torch.randn(1, 1, 7, generator=gen(7), device='cuda').expand(1, 1, 7)]
    was = [g.clone() for g in grads]
    rest = grads[2]._base.clone()
    norm = optim.clip_grads(grads, 0.5)
    check_clip(was, grads, norm, 0.5, 1.0, 'strided')
    rest[::2, 1:8] = grads[2]
    assert torch.equal(rest, grads[2]._base)                                    # what lies between stays
    grads = [w.clone(memory_format=torch.preserve_format) for w in was]
    out = [torch.empty(60, 40, device='cuda'), torch.empty(4, 6, 5, device='cuda').permute(0, 1, 2), torch.empty(7, 17, device='cuda').t(),
           torch.empty(2000, device='cuda')[::2], torch.empty(1, 1, 7, device='cuda', dtype=torch.float16)]
    norm = optim.clip_grads(grads, 0.5, out=out)
    check_clip(was, out, norm, 0.5, 1.0, 'other strides')


@pytest.mark.parametrize('value', [1e-30, 1e30, 3e38])
def test_clip_far_values(value):
    """Squares that fp32 cannot hold."""
    g = [torch.full((1000,), value, device='cuda')]
    was = [g[0].clone()]
    n = optim.grad_norm(g)
    want = float(was[0][0].double()) * math.sqrt(1000.0)
    if want < 3.4e38:
        assert abs(float(n) - want) <= want * 1.01 * U[torch.float32]
        check_clip(was, g, optim.clip_grads(g, 1.0), 1.0, 1.0, 'far')
    else:
        assert math.isinf(float(n))                                              # the norm itself is over fp32's range
        optim.clip_grads(g, 1.0)                                                 # ... but not the factor, held in fp64
        want = torch.full((1000,), 1000.0 ** -0.5, device='cuda', dtype=torch.float64)
        within(g[0], want, want * 4 * U[torch.float32], 'far')


def test_clip_not_finite():
    for bad, expect in ((float('nan'), 'nan'), (float('inf'), 'zero')):
        g = [torch.ones(10, device='cuda'), torch.ones(9000, device='cuda', dtype=torch.bfloat16)]
        g[1][8888] = bad
        was = [x.clone() for x in g]
        with pytest.raises(RuntimeError, match='not finite'):
            optim.clip_grads(g, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(g, was))
        norm = optim.clip_grads(g, 1.0)
        ref = [x.clone().requires_grad_() for x in was]
        for r, x in zip(ref, was):
            r.grad = x.clone()
        rn = torch.nn.utils.clip_grad_norm_(ref, 1.0)
        assert (math.isnan(float(norm)) and math.isnan(float(rn))) or float(norm) == float(rn)
        for a, b in zip(g, ref):
            assert torch.equal(torch.isnan(a), torch.isnan(b.grad)) and torch.equal(a.nan_to_num(), b.grad.nan_to_num())
    g = [torch.ones(10, device='cuda')]
    assert float(optim.clip_grads(g, 1.0, error_if_nonfinite=True)) == float(np.float32(math.sqrt(10.0)))


def test_clip_grad_norm_matches_torch():
    model = torch.nn.Sequential(torch.nn.Linear(300, 77), torch.nn.Linear(77, 5)).cuda()
    ref = torch.nn.Sequential(torch.nn.Linear(300, 77), torch.nn.Linear(77, 5)).cuda()
    ref.load_state_dict(model.state_dict())
    extra = torch.nn.Parameter(torch.zeros(3, device='cuda'))                   # no gradient: passed over
    x = torch.randn(50, 300, generator=gen(9), device='cuda')
    for m in (model, ref):
        m(x).square().sum().backward()
    a = optim.clip_grad_norm_(list(model.parameters()) + [extra], 0.1)
    b = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.1)
    assert abs(float(a) - float(b)) <= 1e-6 * float(b)
    for p, q in zip(model.parameters(), ref.parameters()):
        torch.testing.assert_close(p.grad, q.grad, rtol=2e-6, atol=0)
    version = model[0].weight.grad._version
    optim.clip_grad_norm_(model[0].weight, 0.05)
    assert model[0].weight.grad._version > version
    assert float(optim.clip_grad_norm_([extra], 1.0)) == 0.0


def test_clip_refuses_shared_memory():
    x = torch.randn(100, device='cuda')
    for grads, out in (([x, x], None), ([x[:60], x[50:]], None), ([x[:50], x[50:]], [x[1:51], x[50:]]), ([x[:50], x[50:]], [x[50:], x[:50]]),
                       ([x[:50], x[50:]], [torch.empty(100, device='cuda')[:50], torch.empty(50, device='cuda').expand(50)[:1].expand(50)]),
                       ([x.view(torch.bfloat16)[:100]], [x]), ([x[:1].expand(5)], None)):
        with pytest.raises(hip.GvdHipError):
            optim.clip_grads(grads, 1.0, out=out)
    assert float(optim.clip_grads([x[:50], x[50:]], 1e9)) > 0                   # neighbours are fine
    assert float(optim.clip_grads([x[:50], x[50:]], 1e9, out=[x[:50], x[50:]])) > 0
    assert float(optim.grad_norm([x, x])) > 0


# ------------------------------------------------------------------------------------------------------------ beam_select
def select_want(logits, scores, W, finished, eos):
    """The definition in 64 bits: (all candidates, the places of the best W)."""
    B, K = scores.shape
    x, s = logits.double().reshape(B, K, -1), scores.double()
    V = x.shape[2]
    m = x.max(dim=2, keepdim=True)[0]
    lse = m + (x - m).exp().sum(2, keepdim=True).log()
    cand = torch.full((B, K, V), float('-inf'), device='cuda', dtype=torch.float64)
    cand = torch.where((torch.isfinite(s).unsqueeze(2) & torch.isfinite(lse)), s.unsqueeze(2) + (x - lse), cand)
    if finished is not None:
        ended = torch.full_like(cand, float('-inf'))
        ended[:, :, eos] = torch.where(torch.isfinite(s), s, torch.full_like(s, float('-inf')))
        cand = torch.where(finished.bool().unsqueeze(2), ended, cand)
    flat = cand.reshape(B, K * V)
    return flat.cpu().numpy(), flat.sort(dim=1, descending=True, stable=True)[1][:, :W].cpu().numpy()


def check_select(logits, scores, W=None, finished=None, eos=None, what=''):
    B, K = scores.shape
    V = logits.shape[-1]
    got = ops.beam_select(logits, scores, width=W, finished=finished, eos=eos)
    W = W or K
    sc, parent, word, done = got
    assert sc.shape == parent.shape == word.shape == (B, W) and sc.dtype == torch.float32 and parent.dtype == word.dtype == torch.int64
    cand, order = select_want(logits, scores, W, finished, eos)
    beam = parent.cpu().numpy() - np.arange(B)[:, None] * K
    at = beam * V + word.cpu().numpy()
    assert ((beam >= 0) & (beam < K)).all() and ((word >= 0) & (word < V)).all(), what
    rows = np.arange(B)[:, None]
    best, have = cand[rows, order], cand[rows, at]
    # log-sum-exp: fp32 terms, each off by 2 u (the exponential, one unit in the last place) and by 2 |x - max| u (the difference
    # and the product that make its argument); weighted by the terms, |x - max| is log V on average at most.  They are added 32
    # at a time in fp32 (31 u), scaled from tile to tile and lane to lane (2 u and 2 |change of max| u, weighted likewise).  The
    # score is rounded once.
    tol = (2 + 31 + 2 + 4 * (math.log(V) + 1)) * U[torch.float32]
    fin = np.isfinite(best)
    assert (np.isfinite(sc.cpu().numpy()) == fin).all(), what
    assert (np.abs(sc.cpu().numpy()[fin].astype(np.float64) - have[fin]) <= tol + np.abs(have[fin]) * U[torch.float32]).all(), what
    # the same candidates, but for beams closer together than the log-sum-exp's error
    with np.errstate(invalid='ignore'):
        near = (at != order) & fin & (np.abs(have - best) <= 2 * tol) & (at // V != order // V)
    assert ((at == order) | near).all(), (what, at[at != order][:5], order[at != order][:5])
    if eos is None:
        assert done is None
    else:
        fw = word.cpu().numpy() == eos
        if finished is not None:
            fw = fw | finished.cpu().numpy().astype(bool)[rows, beam]
            assert done.dtype == finished.dtype
        assert (done.cpu().numpy().astype(bool) == fw).all(), what
    return got


def beams(B, K, V, seed, dtype=torch.float32, spread=3.0):
    g = gen(seed)
    return (torch.randn(B * K, V, generator=g, device='cuda') * spread).to(dtype), torch.randn(B, K, generator=g, device='cuda') * 2 - 10


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('B,K,V', [(1, 1, 1), (1, 1, 7), (3, 5, 5), (2, 2, 63), (1, 5, 5000), (7, 5, 5001), (2, 32, 1025), (3, 16, 4097), (64, 5, 5000),
                                   (1, 3, 8193), (2, 8, 32003), (5, 4, 70001), (60, 9, 9000), (1, 1, 600001)])
def test_beam_select_sizes(B, K, V, dtype):
    x, s = beams(B, K, V, B + K + V, dtype)
    check_select(x, s, what='plain')
    check_select(x, s, eos=V // 2, W=min(2 * K, 32, K * V), what='wider')
    check_select(x, s, W=1, what='one')
    f = torch.rand(B, K, generator=gen(V), device='cuda') < 0.4
    check_select(x, s, finished=f, eos=V - 1, W=min(K, V), what='ended')
    check_select(x.view(B, K, V), s, finished=f.to(torch.uint8), eos=0, W=min(32, K * V), what='ended, all')


def test_beam_select_first_step_and_dead_beams():
    """Only beam 0 in use; no beam in use; NaN and infinite scores: candidates of -inf come in the order of q * V + v."""
    x, _ = beams(4, 6, 300, 1)
    s = torch.full((4, 6), float('-inf'), device='cuda')
    s[0, 0] = 0.0
    s[1, 3] = -1.5
    s[2] = torch.tensor([float('nan'), float('inf'), float('-inf'), -2.0, float('nan'), -1.0], device='cuda')
    check_select(x, s, what='first')
    _, parent, word, _ = check_select(x, s, W=32, what='all')
    assert parent[3].tolist() == [18] * 32 and word[3].tolist() == list(range(32))
    f = torch.ones(4, 6, device='cuda', dtype=torch.uint8)
    check_select(x, s, W=32, finished=f, eos=5, what='all ended')
    check_select(x[:, :3], s[:, :], W=18, finished=f, eos=1, what='few words')


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
def test_beam_select_banned_words_and_broken_logits(dtype):
    x, s = beams(6, 4, 700, 2, dtype)
    x[:, torch.rand(700, generator=gen(3), device='cuda') < 0.97] = float('-inf')
    x[1] = float('-inf')                                   # all banned
    x[5, 17] = float('nan')
    x[9, 3] = float('inf')
    x[10] = float('nan')
    x[12:16] = float('-inf')
    x[13, 699] = 1.0                                       # one word in the sample
    x[16:20] = torch.finfo(dtype).min                      # the type's lowest value: equal words, not banned ones
    for W in (1, 4, 32):
        check_select(x, s, W=W, what='W %d' % W)
        check_select(x, s, W=W, finished=torch.tensor([[0, 1, 0, 0]] * 6, device='cuda', dtype=torch.uint8), eos=2, what='ended, W %d' % W)


@pytest.mark.parametrize('V', [5, 700, 5000, 40000])
def test_beam_select_equal_logits(V):
    """Ties go to the lower word, then the lower beam: all equal, a few values, -0 and +0."""
    s = torch.tensor([[-1.0, -1.0, -1.0], [-3.0, -2.0, -2.0]], device='cuda')
    for x in (torch.zeros(6, V, device='cuda'), torch.randint(0, 3, (6, V), generator=gen(V), device='cuda').float(),
              torch.where(torch.rand(6, V, generator=gen(V), device='cuda') < 0.5, 0.0, -0.0)):
        for t in TYPES:
            same = x[:1].expand(6, V).contiguous().to(t)
            for W in (1, 3, 15):
                check_select(same, s, W=W, what='same rows')
                check_select(x.to(t), s, W=W, what='rows')


def test_beam_select_strides():
    x = torch.randn(2, 5, 1000, generator=gen(5), device='cuda', dtype=torch.bfloat16) * 3
    s = torch.randn(3, 10, generator=gen(6), device='cuda')[1:, ::2] - 5
    f = (torch.rand(5, 2, generator=gen(7), device='cuda') < 0.5).t()
    for v in (x[:, :, 1:998], x[:, :, ::2], x.view(10, 1000)[:, 7:], x.transpose(0, 1).contiguous().transpose(0, 1)):
        check_select(v, s, finished=f, eos=3, what=str(tuple(v.shape)))


def test_beam_select_is_repeatable():
    x, s = beams(16, 8, 50000, 8, torch.bfloat16)
    a = ops.beam_select(x, s, eos=0)
    for _ in range(3):
        b = ops.beam_select(x, s, eos=0)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


# ----------------------------------------------------------------------------------------------------------------- reorder
STATES = [(torch.float32, (6,), 0), (torch.uint8, (6, 3), 0), (torch.bool, (2, 6), 1), (torch.float16, (6, 7), 0), (torch.bfloat16, (6, 8), 0),
          (torch.int64, (20, 6), 1), (torch.int32, (6, 3), 0), (torch.float32, (4, 6, 1024), 1), (torch.bfloat16, (6, 9001), 0),
          (torch.float64, (2, 3, 6, 5, 4), 2), (torch.uint8, (6, 17), 0), (torch.float16, (3, 6, 4099), 1), (torch.complex64, (6, 2), 0)]


def make_state(dtype, shape, seed):
    n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 2 if dtype == torch.bool else 120, (n,), generator=gen(seed), device='cuda', dtype=torch.uint8)
    return raw.view(dtype).view(shape)


@pytest.mark.parametrize('dtype,shape,dim', STATES, ids=str)
def test_reorder_rows(dtype, shape, dim):
    x = make_state(dtype, shape, 1)
    for p in (torch.tensor([5, 0, 0, 3, 5, 1], device='cuda'), torch.tensor([[2], [2]], device='cuda'), torch.arange(6, device='cuda'),
              torch.randint(0, 6, (30,), generator=gen(2), device='cuda')[::2]):
        y, = ops.reorder_rows([x], p, dim=dim)
        want = x.index_select(dim, p.reshape(-1))
        assert y.dtype == dtype and torch.equal(y, want)
        out = torch.zeros_like(want)
        got = ops.reorder_rows([x], p, dim=dim - x.dim(), out=[out])
        assert got[0] is out and torch.equal(out, want)


def test_reorder_many_states_in_one_call():
    xs = [make_state(t, s, i) for i, (t, s, d) in enumerate(STATES) if d == 0] * 4
    assert len(xs) > hip.REORDER_MAX_TENSORS
    p = torch.tensor([1, 1, 4, 0, 2, 5], device='cuda')
    for a, b in zip(ops.reorder_rows(xs, p), xs):
        assert torch.equal(a, b[p])


def test_reorder_strides_and_buffers():
    """Views of wider buffers, transposed states, results in a second set of buffers; what lies around the results stays."""
    p = torch.tensor([3, 3, 0], device='cuda')
    wide = make_state(torch.int64, (4, 5, 10), 3)
    for x, d in ((wide[:, :4, 2:9], 1), (wide[:, ::2, :], 0), (wide[1:, 1:, 3], 1), (wide.transpose(0, 2)[:, :4], 1), (wide.permute(1, 0, 2), 1),
                 (wide[:, :, ::3], 0), (wide[::2], 2), (wide[:1], 2)):
        assert torch.equal(ops.reorder_rows([x], p, dim=d)[0], x.index_select(d, p))
    buf = torch.full((4, 6, 11), -5, device='cuda')
    ops.reorder_rows([wide], p, dim=1, out=[buf[:, 2:5, 1:]])
    assert torch.equal(buf[:, 2:5, 1:], wide[:, p])
    buf[:, 2:5, 1:] = -5
    assert bool((buf == -5).all())
    turned = torch.empty(3, 4, 10, device='cuda', dtype=torch.int64)
    ops.reorder_rows([wide], p, dim=1, out=[turned.transpose(0, 1)])
    assert torch.equal(turned.transpose(0, 1), wide[:, p])


def test_reorder_refuses_shared_memory():
    x = torch.zeros(8, 16, device='cuda')
    p = torch.arange(8, device='cuda')
    o = torch.empty(8, 16, device='cuda')
    for states, out in (([x], [x]), ([x[:, :8].contiguous(), x], [x[:, 8:].contiguous().view(-1)[:64].view(8, 8), o.view(-1)[:128].view(8, 16)][:1] + [x]),
                        ([x, x], [o, o]), ([x], [x.view(-1).as_strided((8, 16), (16, 1))])):
        with pytest.raises(hip.GvdHipError):
            ops.reorder_rows(states, p, out=out)
    ops.reorder_rows([x, x], p, out=[o, torch.empty_like(o)])


def test_reorder_into_a_saved_tensor_is_seen_by_autograd():
    w = torch.ones(4, 3, device='cuda', requires_grad=True)
    buf = torch.ones(4, 3, device='cuda')
    y = (w * buf).sum()                           # saves buf
    ops.reorder_rows([torch.zeros(4, 3, device='cuda')], torch.arange(4, device='cuda'), out=[buf])
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_reorder_rows_outside_and_nothing():
    x = torch.ones(4, 5, device='cuda')
    h = torch.ones(3, 4, device='cuda', dtype=torch.int64)
    p = torch.tensor([1, -1, 4, 2 ** 40, 3], device='cuda')
    y, = ops.reorder_rows([x], p)
    assert torch.isnan(y[1:4]).all() and bool((y[[0, 4]] == 1).all())
    z, = ops.reorder_rows([h], p, dim=1)
    assert bool((z[:, 1:4] == -1).all()) and bool((z[:, [0, 4]] == 1).all())
    assert ops.reorder_rows([], p) == []
    assert ops.reorder_rows([x], p[:0])[0].shape == (0, 5)
    assert ops.reorder_rows([x[:, :0]], p)[0].shape == (5, 0)


def test_reorder_past_32_bits():
    """A cache of 5 GiB: rows that start behind 2^32 bytes, outer strides past 2^31 elements."""
    x = torch.zeros(2, 5, 1 << 29, device='cuda', dtype=torch.uint8)
    for o in range(2):
        for r in range(5):
            x[o, r, ::1 << 20] = 10 * o + r + 1
            x[o, r, -1] = 50 + 10 * o + r
    p = torch.tensor([4, 0, 3], device='cuda')
    y, = ops.reorder_rows([x], p, dim=1)
    for o in range(2):
        for i, r in enumerate(p.tolist()):
            assert bool((y[o, i, ::1 << 20] == 10 * o + r + 1).all()) and int(y[o, i, -1]) == 50 + 10 * o + r
            assert int(y[o, i].sum(dtype=torch.int64)) == 512 * (10 * o + r + 1) + 50 + 10 * o + r


# ------------------------------------------------------------------------------------------------- streams, graphs, together
def test_other_streams():
    """The launches go to the current stream: work queued there before is seen, and a second stream does not disturb it."""
    w0 = torch.randn(3000, 256, generator=gen(1), device='cuda')
    tok = words('half', 6000, 3000, 2)
    x, s = beams(32, 5, 20000, 3)
    want_e = ops.embedding(tok, w0 * 2, act=1)
    want_b = ops.beam_select(x * 2, s, eos=0)
    want_n = optim.grad_norm([w0 * 2, x * 2])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for st in (a, b, a):
        with torch.cuda.stream(st):
            w, y = w0 * 2, x * 2
            got.append((ops.embedding(tok, w, act=1), ops.beam_select(y, s, eos=0), optim.grad_norm([w, y])))
    torch.cuda.synchronize()
    for e, bs, n in got:
        assert torch.equal(e, want_e) and torch.equal(n, want_n) and all(torch.equal(u, v) for u, v in zip(bs, want_b))


def test_inference_mode_and_other_threads():
    """Tensors without versions; two host threads at once, each on a stream of its own."""
    import threading
    with torch.inference_mode():
        w = torch.randn(50, 16, generator=gen(1), device='cuda')
        assert torch.equal(ops.embedding(torch.arange(50, device='cuda'), w), w)
        g = torch.full((100,), 3.0, device='cuda')
        optim.clip_grads([g], 3.0)
        assert abs(float(g[0]) - 0.3) < 1e-6
        x, s = beams(2, 3, 40, 5)
        p = ops.beam_select(x, s)[1]
        assert torch.equal(ops.reorder_rows([x], p)[0], x[p.view(-1)])
    w = torch.randn(3000, 200, generator=gen(2), device='cuda')
    tok = words('half', 20000, 3000, 3)
    dy = torch.randn(20000, 200, generator=gen(4), device='cuda')
    wl = w.detach().clone().requires_grad_()
    want, = torch.autograd.grad(ops.embedding(tok, wl, act=1), wl, dy)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                v = wl.detach().clone().requires_grad_()
                got, = torch.autograd.grad(ops.embedding(tok, v, act=1), v, dy)
                if not torch.equal(got, want):
                    bad.append(1)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_captured_and_replayed():
    """Two captured graphs that live side by side, replayed several times with new inputs and eager work between the replays."""
    V, E, n, B, K, H = 700, 96, 9000, 4, 5, 32

    def inputs(seed):
        return (words('half', n, V, seed), torch.randn(V, E, generator=gen(seed), device='cuda'), torch.randn(n, E, generator=gen(seed + 1), device='cuda'),
                beams(B, K, V, seed + 2)[0], beams(B, K, V, seed + 2)[1], torch.randn(2, B * K, H, generator=gen(seed + 3), device='cuda'))

    def work(tok, w, dy, x, s, st):
        w = w.requires_grad_()
        out = ops.embedding(tok, w, 3.0, 1)
        grad, = torch.autograd.grad(out, w, dy)
        norm = optim.clip_grads([grad, dy], 1.0, out=[grad, torch.empty_like(dy)])
        sc, parent, word, done = ops.beam_select(x, s, eos=0)
        new, = ops.reorder_rows([st], parent, dim=1)
        return [out.detach(), grad, norm, sc, parent, word, done, new, ops.embedding(word, w.detach())]

    graphs = []
    for k in range(2):
        static = [t.clone() for t in inputs(100 + k)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*[t.detach() for t in static])
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = work(*[t.detach() for t in static])
        graphs.append((g, static, res))
    for rep in range(4):
        for k, (g, static, res) in enumerate(graphs):
            new = inputs(1000 + 10 * rep + k)
            for a, b in zip(static, new):
                a.copy_(b)
            g.replay()
            eager = work(*[t.clone() for t in new])
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(res, eager)):
                assert torch.equal(a, b), (rep, k, i)


def test_a_training_step_of_them_together():
    """Lookup -> loss -> gradient -> clipping in place, against the same step in 64 bits."""
    V, E, n = 300, 64, 2000
    tok = words('half', n, V, 5)
    w = (torch.randn(V, E, generator=gen(6), device='cuda')).requires_grad_()
    m = torch.randn(E, 10, generator=gen(7), device='cuda').div_(8).requires_grad_()
    h = ops.embedding(tok, w, 2.0, act=1)
    (h.matmul(m)).square().mean().backward()
    norm = optim.clip_grad_norm_([w, m], 0.01)
    w64, m64 = w.detach().double().requires_grad_(), m.detach().double().requires_grad_()
    (torch.relu(w64[tok] * 2.0).matmul(m64)).square().mean().backward()
    rn = torch.nn.utils.clip_grad_norm_([w64, m64], 0.01)
    assert abs(float(norm) - float(rn)) < 1e-5 * float(rn)
    for a, b in ((w, w64), (m, m64)):
        assert float((a.grad.double() - b.grad).norm()) < 1e-5 * float(b.grad.norm())


def test_a_search_of_them_together():
    """Lookup -> state -> logits -> selection -> reordering of state and histories over several steps, against the same search in
    64 bits; the histories are rebuilt from the parents."""
    B, K, V, E, L = 3, 4, 60, 16, 6
    table = torch.randn(V, E, generator=gen(1), device='cuda')
    head = torch.randn(E, V, generator=gen(2), device='cuda')

    def search(f64):
        c = (lambda t: t.double()) if f64 else (lambda t: t)
        state = torch.zeros(1, B * K, E, device='cuda', dtype=c(table).dtype)
        scores = torch.full((B, K), float('-inf'), device='cuda')
        scores[:, 0] = 0.0
        done = torch.zeros(B, K, device='cuda', dtype=torch.uint8)
        hist = torch.zeros(L, B * K, device='cuda', dtype=torch.int64)
        word = torch.arange(B, device='cuda').repeat_interleave(K) + 1
        for t in range(L):
            x = torch.relu(c(table)[word] * 0.5) if f64 else ops.embedding(word, table, 0.5, act=1)
            state = torch.tanh(state + x)
            logits = state[0].matmul(c(head))
            if f64:
                cand, order = select_want(logits, scores, K, done, 0)
                at = torch.from_numpy(order).cuda()
                scores = torch.from_numpy(np.take_along_axis(cand, order, 1)).cuda()
                parent, word = at // V + torch.arange(B, device='cuda')[:, None] * K, at % V
                done = (done.view(-1)[parent].bool() | (word == 0)).to(torch.uint8)
                state, hist = state[:, parent.view(-1)], hist[:, parent.view(-1)]
            else:
                scores, parent, word, done = ops.beam_select(logits, scores, finished=done, eos=0)
                state, = ops.reorder_rows([state], parent, dim=1)
                hist, = ops.reorder_rows([hist], parent, dim=1)
            word = word.reshape(-1)
            hist[t] = word
        return scores, hist, done
    a, b = search(False), search(True)
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    assert float((a[0].double() - b[0]).abs().max()) < 1e-4        # six steps of fp32 products and softmaxes
