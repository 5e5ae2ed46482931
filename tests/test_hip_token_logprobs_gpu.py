"""token_logprobs on the GPU against its definition in 64 bits (on the CPU): log probabilities, entropies, alternatives, gradients.

Tolerances, from the arithmetic (u = 2^-24; m the row's maximum, d_c = x_c - m): a term exp(d_c) is off by (2 |d_c| + 6) u relative (change of base,
exponential), a sum by its additions in a row, at most V / 64 + 32, in u; so log s by (V / 64 + 38 + 2 E|d|) u with E|d| = sum p |d|, a log probability by that
plus 4 u (|x_t - m| + |log s|), the entropy (log s - sum e d / s) by (V / 64 + 44 + 4 E|d|) u (1 + E|d| + |log s|) + the second moment's share
2 u E|d|^2.  A gradient element adds the relative error of p_c = exp(x_c - z) -- the error of z plus (4 |x_c - z| + 6) u -- and, at the end, half a
step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def reference(x, t, top, g=None):
    """x [R, V] (any type, CPU) -> logp, entropy, top_logp, ids, and with g = (g_logp, g_ent, g_top): the gradient; each with its error bound"""
    x = x.double()
    R, V = x.shape
    m = x.amax(1, keepdim=True)
    ls = torch.log((x - m).exp().sum(1))                 # (kept apart from m: next to 3e38 even 64 bits lose it)
    lp = (x - m) - ls[:, None]
    p = lp.exp()
    d = torch.where(p > 0, x - m, torch.zeros_like(x))
    Ed, Ed2 = (p * d.abs()).sum(1), (p * d * d).sum(1)
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    e_ls = (V / 64 + 38 + 2 * Ed) * U
    e_ent = (V / 64 + 44 + 4 * Ed) * U * (1 + Ed + ls.abs()) + 2 * U * Ed2
    ok = (t >= 0) & (t < V)
    tt = t.clamp(0, V - 1)
    xt = x.gather(1, tt[:, None])[:, 0]
    logp = torch.where(ok, (xt - m[:, 0]) - ls, torch.where(t < 0, torch.zeros_like(xt), torch.full_like(xt, float("nan"))))
    e_logp = e_ls + 4 * U * ((xt - m[:, 0]).abs().nan_to_num(posinf=0) + ls.abs())
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    best = lp.gather(1, ids)
    e_best = e_ls[:, None] + 4 * U * ((x.gather(1, ids) - m).abs().nan_to_num(posinf=0) + ls.abs()[:, None])
    if g is None:
        return (logp, e_logp), (ent, e_ent), (best, e_best), ids
    gl, gh, gt = (a.double() for a in g)
    gl = torch.where(ok, gl, torch.zeros_like(gl))
    gs = gl + gt.sum(1)
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    inner = gs[:, None] + gh[:, None] * (lp0 + ent[:, None])
    dx = -p * inner
    dx.scatter_add_(1, tt[:, None], gl[:, None])
    dx.scatter_add_(1, ids, gt)
    rel = e_ls[:, None] + (4 * (lp0.abs() + ls.abs()[:, None]) + 10) * U
    size = p * ((gl.abs() + gt.abs().sum(1))[:, None] + gh.abs()[:, None] * (lp0.abs() + ent[:, None]))
    e_dx = size * rel + p * gh.abs()[:, None] * (e_ent[:, None] + rel * 2) + (top + 4) * U * (dx.abs() + (gl.abs() + gt.abs().sum(1))[:, None] * (dx.abs() > 0))
    return (logp, e_logp), (ent, e_ent), (best, e_best), ids, (dx, e_dx)


def close(got, want, tol, what, dtype=F32):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want)), what
    f = torch.isfinite(want)
    half = torch.finfo(dtype).eps / 2
    err, tol = (got - want).abs()[f], (tol.expand_as(want)[f] * 1.01 + half * (want.abs() + tol.expand_as(want))[f] + 1e-36)
    assert bool((err <= tol).all()), (what, (err / tol).max())
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), what


def make(R, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, V, generator=g) * (0.3 + scale * torch.rand(R, 1, generator=g))).to(dtype)
    t = torch.randint(0, V, (R,), generator=g)
    t[::5] = -100
    return x, t, (torch.randn(R, generator=g), torch.randn(R, generator=g))


def check(x, t, top, xd=None, g=None, shape=None):
    from vilmedic_amd import ops
    R, V = x.shape
    gen = torch.Generator().manual_seed(77)
    g = g or (torch.randn(R, generator=gen), torch.randn(R, generator=gen))
    gt = torch.randn(R, top, generator=gen)
    xd = (x.to(dev()) if xd is None else xd).detach().requires_grad_(True)
    shape = (R,) if shape is None else shape
    out = ops.token_logprobs(xd, t.view(shape).to(dev()), top)
    assert out.logp.shape == shape and out.entropy.shape == shape and out.top_logp.shape == (*shape, top) and out.top_ids.shape == (*shape, top)
    assert out.logp.dtype == out.entropy.dtype == out.top_logp.dtype == F32 and out.top_ids.dtype == torch.int64
    (logp, e_l), (ent, e_h), (best, e_b), ids, (dx, e_dx) = reference(x, t, top, (*g, gt))
    assert torch.equal(out.top_ids.view(R, top).cpu(), ids)
    close(out.logp.detach().view(R), logp, e_l, "logp")
    close(out.entropy.detach().view(R), ent, e_h, "entropy")
    close(out.top_logp.detach().view(R, top), best, e_b, "top")
    outs, gs = [out.logp, out.entropy], [g[0].view(shape).to(dev()), g[1].view(shape).to(dev())]
    if top:
        outs, gs = outs + [out.top_logp], gs + [gt.view(*shape, top).to(dev())]
    grad = torch.autograd.grad(outs, xd, gs)[0]
    assert grad.shape == xd.shape and grad.dtype == x.dtype
    close(grad.reshape(R, V), dx, e_dx, "gradient", x.dtype)
    return out, grad


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V,top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 7), (4, 8, 0), (4, 9, 3), (6, 31, 31), (2, 64, 32), (7, 100, 5), (3, 255, 8), (3, 256, 16), (3, 257, 32), (2, 1024, 1), (9, 2047, 20),
    (64, 4000, 5), (5, 8832, 8), (70, 30522, 5), (600, 1000, 3), (1, 32768, 4), (3, 32769, 5), (2, 50001, 32), (2, 70003, 0), (1, 200000, 8)])
def test_values_and_gradients(dtype, R, V, top):
    x, t, g = make(R, V, dtype, seed=V)
    check(x, t, top, g=g)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [513, 2100])
def test_many_rows(dtype, rows):
    x, t, g = make(rows, 1003, dtype, seed=rows)
    check(x, t, 4, g=g)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,top", [(37, 32), (700, 5), (4100, 7)])
def test_many_rows_of_equal_and_missing_logits(dtype, V, top):
    x = torch.randint(0, 2, (2050, V), generator=torch.Generator().manual_seed(V)).to(dtype)
    x[::3] = 1.0
    x[1::7, top:] = -float("inf")
    x[2::9, 1:] = -float("inf")
    check(x, torch.zeros(2050, dtype=torch.int64), top)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,top", [(50, 32), (3000, 32), (30522, 32), (40000, 17)])
def test_equal_logits_are_ordered_by_column(dtype, V, top):
    g = torch.Generator().manual_seed(V)
    x = torch.stack([torch.zeros(V), torch.randint(0, 3, (V,), generator=g).float(), torch.cat([torch.full((V - 5,), 2.0), torch.full((5,), 3.0)]),
                     torch.where(torch.rand(V, generator=g) < 0.5, torch.tensor(-0.0), torch.tensor(0.0)), -torch.arange(V).div(7, rounding_mode="floor").float()]).to(dtype)
    check(x, torch.tensor([0, V - 1, 3, -1, 2]), top)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [40, 5000, 30522, 50001])
def test_banned_columns_and_empty_rows(dtype, V):
    x, _, _ = make(6, V, dtype, seed=3)
    inf = float("inf")
    x[0, :2] = -inf
    x[1] = -inf
    x[1, 9] = 1.5                                        # one column left
    x[2, :V - 3] = -inf                                  # fewer columns left than alternatives asked for: the others follow by column
    x[4, ::2] = -inf
    t = torch.tensor([5, 9, V - 1, 7, 1, -1])
    check(x, t, 5)
    from vilmedic_amd import ops
    x[3] = -inf                                          # nothing left
    x[5, 4] = -inf
    t[5] = 4                                             # a banned target
    xd = x.to(dev()).requires_grad_(True)
    out = ops.token_logprobs(xd, t.to(dev()), 3)
    assert out.logp[3].item() == -inf and out.entropy[3].item() == 0.0 and out.top_logp[3].tolist() == [-inf] * 3 and out.top_ids[3].tolist() == [0, 1, 2]
    assert out.logp[5].item() == -inf and torch.isfinite(out.entropy[5])
    grad = torch.autograd.grad(out.entropy.sum() + out.top_logp[:, 0].sum(), xd)[0]
    assert bool(torch.isfinite(grad).all()) and not bool(grad[3].any()) and not bool(grad[torch.isinf(xd)].any())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [30, 700, 40000])
def test_the_lowest_value_of_the_type_is_a_logit_like_any_other(dtype, V):
    """rows masked with finfo.min instead of -inf: uniform where nothing else is left, without weight next to ordinary logits"""
    x, _, _ = make(4, V, dtype, seed=5)
    low = torch.finfo(dtype).min
    x[0] = low
    x[1, ::2] = low
    x[2, 1:] = low
    x[3, :7] = low
    x[3, 7:] = -float("inf")
    g = (torch.tensor([1.0, -2.0, 0.5, 1.5]), torch.tensor([0.3, 0.2, -1.0, 0.7]))
    check(x, torch.tensor([3, 1, 0, 2]), 5, g=g)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [300, 40000])
def test_nan_inf_and_targets_outside(dtype, V):
    from vilmedic_amd import ops
    x, _, _ = make(5, V, dtype, seed=4)
    x[0, V // 2] = float("nan")
    x[1, 17] = float("inf")
    t = torch.tensor([1, 2, V, -3, V - 1])
    xd = x.to(dev()).requires_grad_(True)
    out = ops.token_logprobs(xd, t.to(dev()), 2)
    for r in (0, 1):                                     # as log_softmax has it: the whole row
        assert bool(torch.isnan(out.logp[r])) and bool(torch.isnan(out.entropy[r]))
    assert out.top_ids[0, 0].item() == V // 2 and out.top_ids[1, 0].item() == 17
    assert bool(torch.isnan(out.logp[2])) and out.logp[3].item() == 0.0 and bool(torch.isfinite(out.entropy[2:]).all())
    (logp, e_l), (ent, e_h), (best, e_b), ids = reference(x[2:], t[2:], 2)
    assert torch.equal(out.top_ids[2:].cpu(), ids)
    close(out.entropy[2:].detach(), ent, e_h, "entropy")
    close(out.top_logp[2:].detach(), best, e_b, "top")
    grad = torch.autograd.grad(out.entropy.sum(), xd)[0]
    assert bool(torch.isnan(grad[:2]).all()) and bool(torch.isfinite(grad[2:]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_and_shifted_logits(dtype):
    x, t, g = make(8, 999, dtype, seed=6)
    x = (x.float() * 30 + torch.tensor([0., 1e4, -1e4, 3e4, 0, 1e-3, 500, -500])[:, None]).to(dtype)
    check(x, t, 6, g=g)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,ld", [(30522, 30528), (1001, 1001), (1001, 1024), (77, 80)])
def test_a_shifted_slice_of_decoder_logits_is_read_in_place(dtype, V, ld):
    """logits[:, :-1] of a [B, L, padded V] buffer: outer strides of their own, odd row starts"""
    B, L = 3, 9
    buf = torch.randn(B, L, ld, generator=torch.Generator().manual_seed(V)).to(dtype)
    full = buf.to(dev())
    xd = full[:, :-1, :V]
    t = torch.randint(0, V, (B * (L - 1),), generator=torch.Generator().manual_seed(1))
    before = torch.cuda.memory_allocated()
    check(buf[:, :-1, :V].reshape(-1, V), t, 3, xd=xd, shape=(B, L - 1))
    assert torch.equal(full.cpu(), buf)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_other_layouts(dtype):
    x, t, g = make(12, 500, dtype, seed=8)
    check(x, t, 4, xd=x.to(dev()).t().contiguous().t(), g=g)                           # column-major: copied
    check(x, t, 4, xd=x.view(2, 3, 2, 500).to(dev()), g=g, shape=(2, 3, 2))            # four dimensions
    wide = torch.zeros(12, 511, dtype=dtype, device=dev())
    wide[:, 11:] = x.to(dev())
    check(x, t, 4, xd=wide[:, 11:], g=g)
    one = x[:1].to(dev()).expand(12, 500)                                              # one row for all targets
    check(x[:1].expand(12, 500), t, 4, xd=one, g=g)
    out, _ = check(x[:1], t[1:2], 4, xd=x[0].to(dev()), g=(g[0][:1], g[1][:1]), shape=())


def test_gradient_agrees_with_differences():
    from vilmedic_amd import ops
    x, t, _ = make(3, 40, F32, seed=9, scale=1.0)
    t[0] = 4
    w = torch.tensor([0.7, -1.3, 2.0])

    def f(a):
        lp = torch.log_softmax(a, 1)
        pick = torch.where(t >= 0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros(3, dtype=a.dtype))
        return (w * pick).sum() - 0.3 * (lp.exp() * lp).sum() + lp.topk(2, 1)[0][:, 1].sum()
    xd = x.to(dev()).requires_grad_(True)
    out = ops.token_logprobs(xd, t.to(dev()), 2)
    ((w.to(dev()) * out.logp).sum() + 0.3 * out.entropy.sum() + out.top_logp[:, 1].sum()).backward()
    h, xx = 1e-6, x.double()
    for r, c in [(0, 0), (0, 4), (1, 7), (1, int(x[1].argmax())), (2, 39), (2, int(x[2].topk(2)[1][1]))]:
        up, dn = xx.clone(), xx.clone()
        up[r, c] += h
        dn[r, c] -= h
        want = (f(up) - f(dn)) / (2 * h)                                               # difference error: h^2 times third derivatives, far below 1e-6
        assert abs(xd.grad[r, c].item() - want.item()) <= 1e-5 + 1e-5 * abs(want.item())


def test_second_derivatives_are_refused_and_in_place_changes_noticed():
    from vilmedic_amd import ops
    x = torch.randn(3, 50, device=dev(), requires_grad=True)
    t = torch.tensor([1, 2, 3], device=dev())
    g = torch.autograd.grad(ops.token_logprobs(x, t).logp.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
    y = x * 1.0
    out = ops.token_logprobs(y, t)
    out.logp.mul_(2.0)                                   # outputs are tensors of their own
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logp.sum().backward()


def test_each_gradient_alone_and_none():
    from vilmedic_amd import ops
    x, t, _ = make(6, 300, F32, seed=10)
    xd = x.to(dev()).requires_grad_(True)
    out = ops.token_logprobs(xd, t.to(dev()), 3)
    zero, ones = torch.zeros(6), torch.ones(6)
    for pick, g in ((0, (ones, zero, torch.zeros(6, 3))), (1, (zero, ones, torch.zeros(6, 3))), (2, (zero, zero, torch.ones(6, 3)))):
        grad = torch.autograd.grad(out[pick].sum(), xd, retain_graph=True)[0]
        dx, e = reference(x, t, 3, g)[4]
        close(grad, dx, e, pick)
    assert not out.top_ids.requires_grad
    with torch.no_grad():
        again = ops.token_logprobs(xd, t.to(dev()), 3)
    assert not again.logp.requires_grad and all(torch.equal(a, b) for a, b in zip(again, out))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_repeats_bit_for_bit_and_on_another_stream(dtype):
    from vilmedic_amd import ops
    x, t, _ = make(100, 30522, dtype, seed=11)
    xd, td = x.to(dev()), t.to(dev())
    want = ops.token_logprobs(xd, td, 8)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = [ops.token_logprobs(xd, td, 8) for _ in range(5)]
    again = [ops.token_logprobs(xd, td, 8) for _ in range(5)]
    torch.cuda.synchronize()
    for o in other + again:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_forward_and_backward_replayed_from_a_graph(dtype):
    from vilmedic_amd import ops
    x, t, _ = make(33, 5001, dtype, seed=12)
    xs, ts = x.to(dev()).requires_grad_(True), t.to(dev())
    g0, g1 = torch.randn(33, device=dev()), torch.randn(33, device=dev())

    def once(a):
        out = ops.token_logprobs(a, ts, 4)
        return (*[o.detach() for o in out], torch.autograd.grad([out.logp, out.entropy], a, [g0, g1])[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(xs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with ops.capture(graph):
        got = once(xs)
    for seed in range(4):
        new = make(33, 5001, dtype, seed=20 + seed)[0].to(dev())
        with torch.no_grad():
            xs.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = once(new.clone().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
