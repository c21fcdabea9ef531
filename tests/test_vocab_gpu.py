"""Embedding with scale and sorted gradient, distillation loss, and token sampling: the kernels against 64-bit definitions."""
import math

import pytest
import torch

import vocab_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _within(got, want, bound, what=""):
    got = got.detach().double().cpu()
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), "%s: %d of %d outside, first at %s: %r, wanted %r +- %r" % (
        what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), bound[bad][0].item())


# ---------------------------------------------------------------------------------------------- embedding
def _embed(idx, table, scale, pad, dout):
    from litetorch_b200.ops import functional as Fn
    table = table.detach().requires_grad_()
    out = Fn.token_embedding(idx, table, scale, pad)
    grad, = torch.autograd.grad(out, table, dout)
    return out.detach(), grad


def _check_embed(idx, V, D, dtype, scale, pad, seed, dout=None):
    g = _gen(seed)
    table = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    dout = torch.randn(*idx.shape, D, device="cuda", generator=g).to(dtype) if dout is None else dout
    out, grad = _embed(idx, table, scale, pad, dout)
    assert out.shape == (*idx.shape, D) and grad.shape == table.shape and out.dtype == grad.dtype == dtype
    want = ref.embedding(idx, table, scale)
    _within(out.reshape(-1, D), want, ref.rounding(want, dtype) + want.abs() * 2.0 ** -24, "rows")
    want, bound = ref.embedding_grad(idx, dout, V, scale, None if pad is None else pad % V)
    _within(grad, want, bound + ref.rounding(want, dtype) + bound * torch.finfo(dtype).eps, "gradient")
    again = _embed(idx, table, scale, pad, dout)
    assert torch.equal(out, again[0]) and torch.equal(grad, again[1])          # from run to run


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 5, 8), (3, 7, 17), (31, 11, 64), (32, 400, 72), (33, 513, 24), (64, 3, 40), (65, 512, 33), (1000, 50, 136),
                                   (2048, 70000, 16), (2500, 1000, 1027), (5000, 130, 2056), (4097, 262145, 8), (20000, 9, 24)])
def test_embedding(dtype, n, V, D):
    idx = torch.randint(0, V, (n,), device="cuda", generator=_gen(n))
    _check_embed(idx, V, D, dtype, 1.0, None, n + V)
    _check_embed(idx.int(), V, D, dtype, 22.627417, V // 2, n + D)


@pytest.mark.parametrize("n", [1, 33, 700, 9000, 40000])
def test_one_token_for_all_and_two_in_turn(n):
    _check_embed(torch.full((n,), 6, device="cuda"), 9, 48, torch.float32, 0.5, None, 1)
    _check_embed(torch.arange(n, device="cuda") % 2 * 8, 9, 48, torch.bfloat16, 0.5, None, 2)
    _check_embed(torch.full((n,), 6, device="cuda"), 9, 48, torch.bfloat16, 0.5, 6, 3)                  # padding alone


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 70000, 481), (33, 70000, 520), (700, 70000, 488), (2048, 40000, 856), (64, 17000, 2056)])
def test_few_tokens_of_a_large_table(dtype, n, V, D):
    """Gradients of more than 64 MB (of fp32 or 16-bit numbers): these are summed by sorted tokens however few there are."""
    idx = torch.randint(0, V, (n,), device="cuda", generator=_gen(n))
    idx[::3] = 7
    _check_embed(idx, V, D, dtype, 1.5, 11, n + D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(2048, 300, 64), (2049, 300, 64), (2048, 129, 1), (1500, 1000, 9), (2000, 17, 2048), (65, 3, 517), (2047, 128, 128), (256, 8192, 520)])
def test_one_launch_for_few_tokens(dtype, n, V, D):
    """Rows by a group of threads, and tokens with more than 64 places by all groups, beside tokens outside the table, padding, and none at all in most of it."""
    g = _gen(n + D)
    idx = torch.randint(-2, V + 2, (n,), device="cuda", generator=g)
    _check_embed(idx, V, D, dtype, 0.75, V - 1, n)
    idx[torch.rand(n, device="cuda", generator=g) < 0.6] = V // 2
    idx[torch.rand(n, device="cuda", generator=g) < 0.1] = 0
    _check_embed(idx.int(), V, D, dtype, 1.0, None, n + 1)
    idx.fill_(V - 1)
    idx[n // 2] = 0
    _check_embed(idx, V, D, dtype, 1.0, None, n + 2)
    _check_embed(idx, V, D, dtype, 1.0, V - 1, n + 3)


def test_tokens_outside_the_table():
    idx = torch.tensor([[3, -1, 7], [8, 1 << 40, -(1 << 40)], [0, 7, 100]], device="cuda")
    _check_embed(idx, 8, 24, torch.float32, 2.0, None, 5)
    _check_embed(idx, 8, 24, torch.float16, 2.0, -1, 6)
    _check_embed(torch.full((100,), -1, device="cuda"), 8, 24, torch.float32, 2.0, None, 7)
    _check_embed(torch.full((100,), (1 << 32) + 3, device="cuda"), 8, 24, torch.float32, 2.0, None, 8)  # 3 in its low 32 bits


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_and_tokens_that_do_not_lie_side_by_side(dtype):
    g = _gen(9)
    room = torch.randn(40, 3, 70, device="cuda", generator=g).to(dtype)
    idx = torch.randint(0, 11, (40, 6), device="cuda", generator=g)[:, 1::2]
    for dout in (room[:, :, 1:65], room[:, :, 3:67], room[:, 1:2, 6:].expand(40, 3, 64), room[0, 0, :64].expand(40, 3, 64), room[:, :, :1].expand(40, 3, 64),
                 room.transpose(0, 2)[:40, :, :].transpose(1, 2)[:, :40].transpose(0, 1)[:, :3, :1].expand(40, 3, 64)):
        _check_embed(idx, 11, 64, dtype, 1.5, 4, 10, dout)


def test_the_embedding_in_an_autograd_graph():
    """Both passes count as launches; the graph may be kept, checkpointed, hooked and run after what it read was freed, but not with tokens that changed since."""
    from torch.utils.checkpoint import checkpoint
    from litetorch_b200.ops import functional as Fn, kernels as K
    g = _gen(40)
    idx = torch.randint(0, 50, (6, 7), device="cuda", generator=g)
    table = torch.randn(50, 24, device="cuda", generator=g, requires_grad=True)
    dout = torch.randn(6, 7, 24, device="cuda", generator=g)
    want, bound = ref.embedding_grad(idx, dout, 50, 2.0)
    bound = bound + ref.rounding(want, torch.float32) + bound * 2.0 ** -23
    Fn.token_embedding(idx, table)
    K.reset_launch_count()
    out = Fn.token_embedding(idx, table, 2.0)
    seen = []
    out.register_hook(lambda d: seen.append(d.shape))
    first, = torch.autograd.grad(out, table, dout, retain_graph=True)
    assert K.launch_count() == 2 and seen == [(6, 7, 24)]
    keep = first.clone()
    first.zero_()
    again, = torch.autograd.grad(out, table, dout)
    assert torch.equal(again, keep)
    _within(again, want, bound)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, table, dout)
    checkpoint(lambda w: Fn.token_embedding(idx, w, 2.0), table, use_reentrant=False).backward(dout)
    assert torch.equal(table.grad, keep)
    (Fn.token_embedding(idx, table, 2.0) + Fn.token_embedding(idx, table, 2.0)).backward(dout)
    _within(table.grad, 3 * want, 4 * bound)
    out = Fn.token_embedding(idx, table, 2.0)
    del table.grad
    idx.copy_(49 - idx)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dout)
    with torch.no_grad():
        assert not Fn.token_embedding(idx, table).requires_grad
    assert not Fn.token_embedding(idx, table.detach()).requires_grad
    with torch.inference_mode():
        assert torch.equal(Fn.token_embedding(idx, table), table.detach()[idx])
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            Fn.token_embedding(idx, fwd.make_dual(table.detach(), torch.ones_like(table)))


def test_no_tokens_and_empty_rows():
    from litetorch_b200.ops import functional as Fn
    table = torch.randn(5, 8, device="cuda", requires_grad=True)
    out = Fn.token_embedding(torch.empty(2, 0, dtype=torch.int64, device="cuda"), table)
    assert out.shape == (2, 0, 8) and not torch.autograd.grad(out.sum(), table)[0].any()
    none = torch.randn(5, 0, device="cuda", requires_grad=True)
    out = Fn.token_embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), none)
    assert out.shape == (3, 0) and torch.autograd.grad(out.sum(), none)[0].shape == (5, 0)


# ---------------------------------------------------------------------------------------------- distillation
def _teacher(N, V, K, dtype, g, ragged=False):
    idx = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(min(N, 50))])
    idx = idx.repeat((N + len(idx) - 1) // len(idx), 1)[:N].contiguous()
    t = (torch.randn(N, K, device="cuda", generator=g) * 3 + 8).to(dtype)
    if ragged:
        idx[torch.arange(K, device="cuda") >= torch.randint(0, K + 1, (N, 1), device="cuda", generator=g)] = -1
        idx[0] = -1
    return t, idx


def _check_distill(z, t, idx, T, reduction, up=None):
    from litetorch_b200.ops import functional as Fn
    z = z.detach().requires_grad_()
    loss = Fn.distillation_loss(z, t, idx, T, reduction)
    grad, = torch.autograd.grad(loss, z, up)
    rows, lost, want, bound = ref.distillation(z, t, idx, T, reduction, up)
    assert loss.dtype == torch.float32 and grad.dtype == z.dtype and grad.shape == z.shape
    _within(loss.reshape(-1), rows.reshape(-1), lost.reshape(-1) + 1e-30, "loss")
    _within(grad, want, bound + ref.rounding(want, z.dtype) + bound * torch.finfo(z.dtype).eps, "gradient")
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (2, 3, 2), (5, 100, 7), (3, 4096, 64), (40, 1001, 20), (700, 514, 33), (9, 32000, 128), (2, 50257, 1024), (3, 128256, 5)])
def test_distillation(dtype, N, V, K):
    g = _gen(N + V)
    z = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
    t, idx = _teacher(N, V, K, dtype, g)
    _check_distill(z, t, idx, 1.0, "mean")
    _check_distill(z, t, idx.int(), 2.5, "sum")
    _check_distill(z, t.float(), idx, 0.7, "none", torch.rand(N, device="cuda", generator=g))
    _check_distill(z, t, idx, 1.3, "mean", torch.tensor(-3.0, device="cuda"))
    t, idx = _teacher(N, V, K, dtype, g, ragged=True)
    for reduction in ("mean", "sum"):
        _check_distill(z, t, idx, 1.5, reduction)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,V,pitch", [(0, 1000, 1000), (1, 1000, 1016), (3, 999, 1013), (5, 16, 33), (1, 3, 5), (8, 2048, 2064)])
def test_rows_of_a_wider_tensor(dtype, offset, V, pitch):
    g = _gen(V)
    room = (torch.randn(6, pitch, device="cuda", generator=g) * 3).to(dtype)
    t, idx = _teacher(6, V, 3, dtype, g)
    _check_distill(room[:, offset:offset + V], t, idx, 1.0, "mean")
    _check_distill(room[:, offset:offset + V], t, idx, 1.0, "none", torch.rand(6, device="cuda", generator=g))
    _check_distill(room[:, offset:offset + V].t().contiguous().t(), t, idx, 1.0, "sum")
    _check_distill(room[:1, offset:offset + V].expand(6, V), t, idx, 1.0, "sum")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,K", [(40, 4001, 257), (200, 2048, 301), (32, 32000, 301), (5, 50257, 256), (5, 50256, 257), (3, 40003, 1023), (290, 3001, 1023), (290, 9999, 511)])
def test_few_rows_with_more_than_255_entries(dtype, N, V, K):
    """Odd and even numbers of entries and classes, rows that one CTA or several hold, and classes that come again."""
    g = _gen(K + V)
    z = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
    t, cls = _teacher(N, V, K, dtype, g, ragged=True)
    cls[1, K // 2:] = cls[1, :K - K // 2].clone()
    cls[2] = V - 1
    for reduction in ("mean", "sum"):
        _check_distill(z, t, cls, 1.5, reduction)
    up = torch.rand(N, device="cuda", generator=g)
    a, b = (_check_distill(z, t, cls, 1.5, "none", up)[1] for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,N,V", [(torch.bfloat16, 400, 19197), (torch.float16, 400, 19197), (torch.bfloat16, 290, 40003), (torch.float32, 290, 20001),
                                       (torch.float32, 250, 12289), (torch.bfloat16, 700, 4093), (torch.float16, 290, 131)])
def test_rows_whose_last_vector_changes_its_owner(dtype, N, V):
    """CTAs, and clusters of them, that take several rows, which begin and end at other places within 16 bytes."""
    g = _gen(V)
    z = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
    t, cls = _teacher(N, V, 5, dtype, g, ragged=True)
    cls[1::2, 0], cls[1::2, 1] = V - 1, 0
    up = torch.rand(N, device="cuda", generator=g)
    _check_distill(z, t, cls, 1.0, "mean")
    _, want = _check_distill(z, t, cls, 0.8, "none", up)
    from litetorch_b200.ops import functional as Fn
    leaf = z.detach().requires_grad_()
    loss = Fn.distillation_loss(leaf, t, cls, 0.8, "none")
    for _ in range(20):
        grad, = torch.autograd.grad(loss, leaf, up, retain_graph=True)
        assert torch.equal(grad, want)


def test_classes_that_come_again_and_entries_that_are_not_there():
    g = _gen(3)
    z = torch.randn(5, 40, device="cuda", generator=g)
    t = torch.randn(5, 6, device="cuda", generator=g)
    idx = torch.tensor([[7, 7, 7, 7, 7, 7], [1, 2, 1, 2, 39, 0], [-1, 40, 5, 1 << 40, -7, 5], [-1] * 6, [3, 4, 5, 6, 7, 8]], device="cuda")
    t[4, 2] = t[1, 3] = -math.inf
    loss, _ = _check_distill(z, t, idx, 1.7, "none", torch.rand(5, device="cuda", generator=g))
    assert float(loss[3]) == 0.0
    _check_distill(z, t, idx, 1.0, "mean")
    t[4] = -math.inf                                              # logits all masked: as if there were no teacher
    _check_distill(z, t, idx, 1.0, "mean")
    idx.fill_(-1)
    loss, grad = _check_distill(z, t, idx, 1.0, "mean")           # nobody has one
    assert float(loss) == 0.0 and not grad.any()


def test_masked_student_logits():
    from litetorch_b200.ops import functional as Fn
    g = _gen(4)
    z = torch.randn(4, 3000, device="cuda", generator=g)
    z[:, 100:2000] = -math.inf
    z[1, :2990] = torch.finfo(torch.float32).min
    t, idx = torch.randn(4, 5, device="cuda", generator=g), torch.tensor([[1, 2, 3, 2995, 2999]] * 4, device="cuda")
    idx[1] = torch.tensor([2990, 2991, 2992, 2993, 2994], device="cuda")
    _check_distill(z, t, idx, 1.0, "mean")
    z[2, 3] = -math.inf                                           # the teacher wants what the student excludes: infinitely far, gradient finite
    z.requires_grad_()
    loss = Fn.distillation_loss(z, t, idx, 1.0, "none")
    grad, = torch.autograd.grad(loss.sum(), z)
    assert float(loss[2]) == math.inf and bool(torch.isfinite(loss[[0, 1, 3]]).all()) and bool(torch.isfinite(grad).all())
    with torch.no_grad():
        z[0] = -math.inf
        z[3, 7] = math.nan
    loss = Fn.distillation_loss(z, t, idx, 1.0, "none")
    assert bool(torch.isnan(loss[[0, 3]]).all()) and bool(torch.isfinite(loss[1]))


def test_backward_twice_in_parts_and_without_need():
    from litetorch_b200.ops import functional as Fn
    g = _gen(5)
    z = torch.randn(33, 777, device="cuda", generator=g).bfloat16().requires_grad_()
    t, idx = _teacher(33, 777, 9, torch.bfloat16, g)
    loss = Fn.distillation_loss(z, t, idx, 2.0)
    a, = torch.autograd.grad(loss, z, retain_graph=True)
    keep = a.clone()
    a.zero_()                                                     # what was handed out belongs to the caller
    b, = torch.autograd.grad(loss, z, retain_graph=True)
    c, = torch.autograd.grad(loss, z, torch.tensor(2.0, device="cuda"))
    assert torch.equal(b, keep) and not a.any()
    _, _, want, bound = ref.distillation(z, t, idx, 2.0, "mean", torch.tensor(2.0))
    _within(c, want, bound + ref.rounding(want, torch.bfloat16) + bound * 2.0 ** -7)
    with torch.no_grad():
        quiet = Fn.distillation_loss(z, t, idx, 2.0)
    assert torch.equal(quiet, loss) and not quiet.requires_grad
    (0.25 * loss.detach() + Fn.distillation_loss(z.view(3, 11, 777), t.view(3, 11, 9), idx.view(3, 11, 9), 2.0)).backward()
    assert torch.equal(z.grad, keep)
    frozen = Fn.distillation_loss(z.detach(), t, idx, 2.0)
    assert torch.equal(frozen, loss) and not frozen.requires_grad


def test_gradient_against_differences():
    from litetorch_b200.ops import functional as Fn
    g = _gen(6)
    z = torch.randn(3, 50, device="cuda", generator=g)
    t, idx = _teacher(3, 50, 4, torch.float32, g)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(Fn.distillation_loss(leaf, t, idx, 1.5, "sum"), leaf)
    h = 2.0 ** -5
    for r, j in [(0, int(idx[0, 0])), (1, 7), (2, int(idx[2, 3])), (2, 49)]:
        step = torch.zeros_like(z)
        step[r, j] = h
        up, down = (float(Fn.distillation_loss(z + s * step, t, idx, 1.5, "sum")) for s in (1, -1))
        # the loss (below 100) to 2^-17 each, over 2 h; the difference's own error h^2 / 6 times a third derivative, which is at most 1 / T
        assert abs((up - down) / (2 * h) - float(grad[r, j])) < 100 * 2.0 ** -17 / h + h * h


# ---------------------------------------------------------------------------------------------- sampling
def _check_sample(z, u, tau=1.0, k=0, p=1.0, low=0.0):
    from litetorch_b200.ops import functional as Fn
    tokens, logs = Fn.sample_tokens(z, u, tau, k, p, low)
    want, want_logs = ref.sample(z, u, tau, k, p, low)
    assert tokens.dtype == torch.int64 and logs.dtype == torch.float32
    assert torch.equal(tokens.cpu(), want), (tokens.cpu() != want).nonzero()[:5]
    finite = torch.isfinite(want_logs)
    assert torch.equal(torch.isfinite(logs.cpu()), finite)
    _within(logs[finite.cuda()], want_logs[finite], want_logs[finite].abs() * 2.0 ** -23 + 1e-9, "log probabilities")
    return tokens


def _peaked(rows, V, dtype, g):
    z = torch.randn(rows, V, device="cuda", generator=g) * 2
    z[:, ::max(1, V // 10)] += 8
    return z.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 17), (70, 255), (5, 2049), (200, 1000), (1, 32000), (2, 50257), (40, 8191), (3, 128256), (1, 262147), (1, 1 << 19)])
def test_sampling(dtype, rows, V):
    g = _gen(rows + V)
    z = _peaked(rows, V, dtype, g)
    u = torch.rand(rows, device="cuda", generator=g)
    _check_sample(z, u)
    _check_sample(z, u.double(), 0.7)
    for kw in (dict(k=1), dict(k=2), dict(k=50), dict(k=V), dict(k=V // 2 + 1), dict(p=0.9), dict(p=0.3), dict(p=0.0), dict(p=0.999999), dict(low=0.05), dict(low=1.0),
               dict(k=40, p=0.8), dict(k=40, p=0.9, low=0.1), dict(p=0.95, low=0.01), dict(k=7, low=0.5)):
        _check_sample(z, u, 0.8, **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_set_of_parameters_for_every_row(dtype):
    g = _gen(11)
    rows, V = 300, 4099
    z = _peaked(rows, V, dtype, g)
    tau = torch.rand(rows, device="cuda", generator=g) * 1.5
    tau[::9] = 0.0
    k = torch.randint(-2, 60, (rows,), device="cuda", generator=g)
    k[::7] = V + 5
    p = torch.rand(rows, device="cuda", generator=g) * 1.3
    low = (torch.rand(rows, device="cuda", generator=g) - 0.5).clamp(min=0)
    u = torch.rand(rows, device="cuda", generator=g)
    for order in (torch.arange(rows, device="cuda"), torch.randperm(rows, device="cuda", generator=g)):
        tokens = _check_sample(z[order], u[order], tau[order], k[order], p[order], low[order])
    alone = torch.cat([_check_sample(z[r:r + 1], u[r:r + 1], tau[r:r + 1], k[r:r + 1], p[r:r + 1], low[r:r + 1]) for r in order[:20].tolist()])
    assert torch.equal(alone, tokens[:20])                        # the choice does not depend on the batch


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_by_their_index(dtype):
    rows, V = 64, 5000
    z = torch.zeros(rows, V, device="cuda", dtype=dtype)
    z[:, 1::2] = -0.0
    u = (torch.arange(rows, device="cuda") + 0.5) / rows
    assert bool((_check_sample(z, u, k=8) < 8).all())
    assert bool((_check_sample(z, u, p=0.5) < 2500).all()) and int(_check_sample(z, u, p=0.5).max()) > 2400
    assert bool((_check_sample(z, u, k=10, p=0.5) < 5).all())
    _check_sample(z, u, low=1.0)
    z[:, 100:200] = 1.0
    for kw in (dict(k=30), dict(k=150), dict(p=0.02), dict(p=0.3), dict(k=150, p=0.9), dict(k=120, p=0.97), dict(low=0.9)):
        _check_sample(z, u, **kw)
    assert bool((_check_sample(z, u, 0.0) == 100).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_infinities_and_nan(dtype):
    g = _gen(12)
    V = 3001
    z = _peaked(9, V, dtype, g)
    z[0] = -math.inf
    z[1] = math.nan
    z[2, 1:] = -math.inf
    z[3] = torch.finfo(dtype).min
    z[4, 5] = z[4, 2000] = math.inf
    z[5, :V - 3] = -math.inf
    z[6, ::2] = math.nan
    z[7, 10] = torch.finfo(dtype).max
    z[8, :2900] = torch.finfo(dtype).min
    u = torch.rand(9, device="cuda", generator=g)
    for kw in (dict(), dict(k=2), dict(k=2999), dict(p=0.5), dict(low=0.2), dict(k=5, p=0.5, low=0.1), dict(tau=0.0), dict(tau=-1.0), dict(tau=1e-30), dict(tau=1e30, p=0.4)):
        tokens = _check_sample(z, u, **kw).tolist()
        assert tokens[0] == tokens[1] == -1 and tokens[2] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_parameters_of_rows_that_are_no_numbers(dtype):
    """NaN is a temperature of 0 or a limit that is off; an infinite temperature makes all finite logits alike."""
    g = _gen(41)
    nan = math.nan
    for V in (500, 50257):
        z = _peaked(4, V, dtype, g)
        z[3, ::3] = -math.inf
        u = torch.rand(4, device="cuda", generator=g)
        p, low = torch.tensor([0.5, nan, math.inf, -math.inf], device="cuda"), torch.tensor([nan, 0.1, -math.inf, math.inf], device="cuda")
        tau = torch.tensor([0.7, math.inf, nan, math.inf], device="cuda")
        p1, low1, tau1 = (torch.where(torch.isnan(a), b, a) for a, b in ((p, 1.0), (low, 0.0), (tau, 0.0)))
        from litetorch_b200.ops import functional as Fn
        for k in (0, 7, 400):
            for args, same in (((tau, k, 1.0, 0.0), (tau1, k, 1.0, 0.0)), ((0.8, k, p, 0.0), (0.8, k, p1, 0.0)), ((0.8, k, 1.0, low), (0.8, k, 1.0, low1)), ((tau, k, p, low), (tau1, k, p1, low1))):
                tokens, logs = Fn.sample_tokens(z, u, *args)
                want, want_logs = ref.sample(z, u, *same)
                assert torch.equal(tokens.cpu(), want)
                _within(logs, want_logs, want_logs.abs() * 2.0 ** -23 + 1e-9)


def test_random_numbers_at_and_outside_their_range():
    from litetorch_b200.ops import functional as Fn
    z = _peaked(7, 999, torch.float32, _gen(13))
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.inf, -math.inf], device="cuda")
    for kw in (dict(), dict(k=10), dict(p=0.7), dict(low=0.3)):
        _check_sample(z, u, **kw)
    tokens, _ = Fn.sample_tokens(z[:1], torch.full((1,), math.nan, device="cuda"))
    assert int(tokens) == int(Fn.sample_tokens(z[:1], torch.zeros(1, device="cuda"))[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,V,pitch", [(1, 1000, 1016), (3, 999, 1013), (5, 16, 33), (1, 1, 5), (7, 40001, 40010)])
def test_logits_of_a_wider_tensor(dtype, offset, V, pitch):
    g = _gen(V)
    room = _peaked(6, pitch, dtype, g)
    u = torch.rand(6, device="cuda", generator=g)
    for z in (room[:, offset:offset + V], room[:, offset:offset + V].t().contiguous().t(), room[:1, offset:offset + V].expand(6, V)):
        _check_sample(z, u, 0.9, 20, 0.9, 0.001)
        _check_sample(z, u, 0.9)


def test_draws_follow_the_distribution():
    from litetorch_b200.ops import functional as Fn
    z = torch.tensor([2.0, 1.0, 0.0, -1.0, 3.0], device="cuda").expand(1 << 14, 5)
    u = (torch.arange(1 << 14, device="cuda") + 0.5) / (1 << 14)
    tokens, logs = Fn.sample_tokens(z, u, 1.0)
    share = torch.bincount(tokens, minlength=5).double() / (1 << 14)
    assert float((share - torch.softmax(z[0].double(), 0)).abs().max()) < 2.0 ** -13            # a border falls between two of the even steps
    assert bool((tokens[1:] >= tokens[:-1]).all())


# ---------------------------------------------------------------------------------------------- all of them, as they are used
def test_streams_and_recorded_graphs():
    from litetorch_b200.ops import functional as Fn
    g = _gen(14)
    V, D, N = 1111, 40, 60
    idx = torch.randint(0, V, (N,), device="cuda", generator=g)
    table = torch.randn(V, D, device="cuda", generator=g)
    dout = torch.randn(N, D, device="cuda", generator=g)
    z = torch.randn(N, V, device="cuda", generator=g)
    t, cls = _teacher(N, V, 8, torch.float32, g)
    u = torch.rand(N, device="cuda", generator=g)
    up = torch.full((), 2.0, device="cuda")

    def work():
        w, s = table.detach().requires_grad_(), z.detach().requires_grad_()
        rows = Fn.token_embedding(idx, w, 3.0, 5)
        loss = Fn.distillation_loss(s, t, cls, 2.0)
        return [rows.detach(), torch.autograd.grad(rows, w, dout)[0], loss.detach(), torch.autograd.grad(loss, s, up)[0], *Fn.sample_tokens(z, u, 0.8, 50, 0.9, 0.01)]
    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = work()
    with torch.cuda.graph(other, stream=side):
        out2 = work()
    for seed in (20, 21):
        g = _gen(seed)
        for x in (table, dout, z):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        idx.copy_(torch.randint(0, V, (N,), device="cuda", generator=g))
        u.copy_(torch.rand(N, device="cuda", generator=g))
        up.fill_(1.0 if seed == 20 else 0.5)
        graph.replay()
        other.replay()
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(want, out)) and all(torch.equal(a, b) for a, b in zip(want, out2))


def test_backward_recorded_by_itself():
    """An eager forward pass whose backward is recorded and replayed: every replay gives the gradient of its upstream gradient, whatever was done to the last one."""
    from litetorch_b200.ops import functional as Fn
    g = _gen(15)
    z = torch.randn(20, 300, device="cuda", generator=g)
    t, cls = _teacher(20, 300, 8, torch.float32, g)
    up = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = z.clone().requires_grad_()
        loss = Fn.distillation_loss(leaf, t, cls, 2.0)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        graph.capture_begin()
        grad, = torch.autograd.grad(loss, leaf, up)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for value in (1.0, 3.0, 1.0):
        up.fill_(value)
        grad.fill_(7.0)
        graph.replay()
        _, _, want, bound = ref.distillation(z, t, cls, 2.0, "mean", torch.tensor(value))
        _within(grad, want, bound + ref.rounding(want, torch.float32) + bound * 2.0 ** -23)


def test_an_answer_is_drawn_read_and_learned_from():
    """On-policy distillation in small: a model of an embedding and a tied head draws its tokens, reads them again and is pulled to a teacher's top logits; both
    uses of the table meet in one gradient."""
    from litetorch_b200.ops import functional as Fn
    g = _gen(16)
    V, D, N, T = 500, 64, 48, 2.0
    table = (torch.randn(V, D, device="cuda", generator=g) * 0.3).requires_grad_()
    mix = torch.randn(D, D, device="cuda", generator=g) * 0.1
    idx = torch.randint(0, V, (N,), device="cuda", generator=g)
    with torch.no_grad():
        first = Fn.token_embedding(idx, table, 2.0) @ mix @ table.t()
    tokens = _check_sample(first, torch.rand(N, device="cuda", generator=g), 0.9, 40, 0.95)
    top = torch.randn(N, V, device="cuda", generator=g).topk(10)
    z = Fn.token_embedding(tokens, table, 2.0) @ mix @ table.t()
    Fn.distillation_loss(z, top.values, top.indices, T).backward()
    w = table.detach().double().requires_grad_()
    zz = (w[tokens] * 2.0) @ mix.double() @ w.t()
    log_p = torch.log_softmax(top.values.double() / T, 1)
    (T * T * (log_p.exp() * (log_p - torch.log_softmax(zz / T, 1).gather(1, top.indices))).sum(1).mean()).backward()
    # products over 64 and 500 numbers in 32 bits (torch's, without TF32): 500 roundings of 2^-24 of their sizes, which are within 8 of the largest gradient
    assert float((table.grad - w.grad).abs().max()) < 500 * 2.0 ** -24 * 8 * float(w.grad.abs().max()) + 1e-7


# ---------------------------------------------------------------------------------------------- the lowest value, losses of one's own, slices
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [7, 1000, 1 << 19])
def test_logits_of_the_lowest_value(dtype, V):
    """Masks of the type's lowest value: parts of a row, all but one, all of it (then the student knows nothing), and the highest value against them."""
    g = _gen(V)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z = torch.randn(6, V, device="cuda", generator=g).to(dtype)
    z[0, V // 2:] = low
    z[1] = low
    z[2] = low
    z[2, 3] = 0.5
    z[3, 5] = high
    z[4] = high
    z[5] = low
    z[5, ::2] = -math.inf
    t = torch.randn(6, 2, device="cuda", generator=g).to(dtype)
    idx = torch.tensor([[0, 1], [0, V - 1], [3, -1], [5, -1], [1, V - 2], [1, 5]], device="cuda")
    for T in (1.0, 0.3, 2.0, 2.0 ** 12, 2.0 ** -60):
        _check_distill(z, t, idx, T, "none", torch.rand(6, device="cuda", generator=g))
        _check_distill(z, t, idx, T, "mean")


def test_a_row_of_its_own_for_every_loss():
    from litetorch_b200.ops import functional as Fn
    g = _gen(31)
    z = torch.randn(4, 900, device="cuda", generator=g).requires_grad_()
    t, cls = _teacher(4, 900, 2, torch.float32, g)
    loss = Fn.distillation_loss(z, t, cls, reduction="none")
    loss *= torch.tensor([1.0, 0.0, 2.0, 0.0], device="cuda")
    loss.sum().backward()
    assert not z.grad[1::2].any() and bool(z.grad[::2].any(1).all())


def test_no_gradient_is_formed_that_nobody_asks_for(monkeypatch):
    from litetorch_b200.ops import functional as Fn
    z = torch.randn(4, 900, device="cuda", requires_grad=True)
    t, cls = _teacher(4, 900, 2, torch.float32, _gen(36))
    asked, real = [], Fn.K.distill_loss
    monkeypatch.setattr(Fn.K, "distill_loss", lambda *a: (asked.append(a[-1]), real(*a))[1])
    with torch.no_grad():
        Fn.distillation_loss(z, t, cls)
    Fn.distillation_loss(z.detach(), t, cls)
    Fn.distillation_loss(z, t, cls, reduction="none")
    Fn.distillation_loss(z, t, cls)
    assert asked == [False, False, False, True]


def test_the_gradient_of_a_slice_is_of_the_slices_size():
    """The last positions of long answers: neighbouring rows lie far apart, those of their gradient do not."""
    from litetorch_b200.ops import functional as Fn
    g = _gen(32)
    room = torch.randn(3, 500, 1003, device="cuda", generator=g).bfloat16()
    t, cls = _teacher(3, 1003, 2, torch.bfloat16, g)
    z = room[:, -1].requires_grad_()
    _check_distill(z, t, cls, 1.0, "mean")
    loss = Fn.distillation_loss(z, t, cls)
    before = torch.cuda.memory_allocated()
    grad, = torch.autograd.grad(loss, z)
    assert grad.untyped_storage().nbytes() < 3 * 1020 * 2 and torch.cuda.memory_allocated() - before < 1 << 16


def test_differentiable_once():
    from litetorch_b200.ops import functional as Fn
    z = torch.randn(4, 90, device="cuda", requires_grad=True)
    t, cls = _teacher(4, 90, 2, torch.float32, _gen(37))
    for out in (Fn.distillation_loss(z, t, cls), Fn.token_embedding(cls[:, 0], z).sum()):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out, z, create_graph=True)


def test_more_rows_than_the_gpu_holds_clusters():
    g = _gen(33)
    z = torch.randn(5000, 301, device="cuda", generator=g).half()
    t, cls = _teacher(5000, 301, 3, torch.float16, g, ragged=True)
    _check_distill(z, t, cls, 1.0, "mean")


@pytest.mark.parametrize("dtype", TYPES)
def test_longer_rows_than_a_cluster_holds(dtype):
    g = _gen(34)
    z = torch.randn(3, 300001, device="cuda", generator=g).to(dtype)
    z[1, 1000:] = -math.inf
    t, cls = _teacher(3, 300001, 9, dtype, g)
    cls[1] %= 1000
    cls[2, 5:] = cls[2, :4]
    _check_distill(z, t, cls, 1.3, "sum")
    _check_distill(z, t, cls, 1.3, "none", torch.rand(3, device="cuda", generator=g))


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 33001), (torch.float16, 33000), (torch.float32, 16601)])
def test_many_long_rows(dtype, V):
    """Rows that no CTA holds, more of them than there are places: of all kinds in turn."""
    g = _gen(V)
    N = 650
    z = (torch.randn(N, V, device="cuda", generator=g) * 3).to(dtype)
    t, cls = _teacher(N, V, 6, dtype, g, ragged=True)
    cls[5] = torch.tensor([0, V - 1, 7, 0, V - 1, 9], device="cuda")
    z[3] = torch.finfo(dtype).min
    z[4, 100:] = torch.finfo(dtype).min
    z[6, :V - 2] = -math.inf
    cls[6] = -1
    z[7, 11] = torch.finfo(dtype).max
    cls[7] = torch.tensor([11, -1, -1, -1, -1, -1], device="cuda")
    cls[4] = torch.tensor([1, 2, 3, -1, -1, -1], device="cuda")
    _check_distill(z, t, cls, 1.3, "mean")
    _check_distill(z, t, cls, 1.3, "none", torch.rand(N, device="cuda", generator=g))
    _check_distill(z[:, 1:-2], t, cls.where(cls < V - 3, -1).where(torch.arange(N, device="cuda")[:, None] != 7, -1), 0.9, "sum", torch.tensor(2.0, device="cuda"))


def test_many_entries_that_share_their_low_bits():
    """The entries of long rows are found by the low ten bits of their class: all in one bucket, and classes that come again."""
    g = _gen(38)
    N, V, K = 300, 40000, 1024
    z = torch.randn(N, V, device="cuda", generator=g).bfloat16()
    t = torch.randn(N, K, device="cuda", generator=g)
    idx = torch.randint(0, V, (N, K), device="cuda", generator=g)
    idx[::3] = 5 + 1024 * torch.randint(0, 39, (K,), device="cuda", generator=g)
    idx[1::3, 700:] = -1
    _check_distill(z, t, idx, 1.0, "mean")
    _check_distill(z, t, idx, 1.0, "none", torch.rand(N, device="cuda", generator=g))
    a, b = (_check_distill(z, t, idx, 1.0, "sum")[1] for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,K", [(515, 256), (4001, 1000)])
def test_many_short_rows_with_many_entries(dtype, V, K):
    g = _gen(V)
    z = (torch.randn(400, V, device="cuda", generator=g) * 3).to(dtype)
    t, cls = _teacher(400, V, K, dtype, g, ragged=True)
    cls[7] = cls[7, :1]
    _check_distill(z, t, cls, 1.5, "mean")
    _check_distill(z, t, cls, 1.5, "none", torch.rand(400, device="cuda", generator=g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,K", [(515, 255), (515, 224), (4001, 225), (20000, 255), (20001, 224)])
def test_many_rows_on_both_sides_of_many_entries(dtype, V, K):
    """Rows that a CTA could hold, with so many entries that they are taken as long ones, and with a few less."""
    g = _gen(V + K)
    z = (torch.randn(400, V, device="cuda", generator=g) * 3).to(dtype)
    t, cls = _teacher(400, V, K, dtype, g, ragged=True)
    cls[7] = cls[7, :1]
    _check_distill(z, t, cls, 1.5, "mean")
    _check_distill(z, t, cls, 1.5, "none", torch.rand(400, device="cuda", generator=g))


def test_two_streams_at_once():
    """Calls of the same kind on two streams have nothing in common."""
    from litetorch_b200.ops import functional as Fn
    g = _gen(35)
    V, N, D = 5003, 700, 96
    args = []
    for _ in range(2):
        t, cls = _teacher(N, V, 5, torch.float32, g)
        args.append((torch.randint(0, V, (N,), device="cuda", generator=g), torch.randn(V, D, device="cuda", generator=g), torch.randn(N, D, device="cuda", generator=g),
                     torch.randn(N, V, device="cuda", generator=g), t, cls, torch.rand(N, device="cuda", generator=g)))

    def work(idx, table, dout, z, t, cls, u):
        w, s = table.detach().requires_grad_(), z.detach().requires_grad_()
        loss = Fn.distillation_loss(s, t, cls, 2.0)
        return [torch.autograd.grad(Fn.token_embedding(idx, w), w, dout)[0], loss.detach(), torch.autograd.grad(loss, s)[0], *Fn.sample_tokens(z, u, 0.8, 0, 0.9)]
    want = [work(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = work(*args[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(want, got) for a, b in zip(x, y))


# ---------------------------------------------------------------------------------------------- served models
def _engine():
    from litetorch_b200.models.llama import LlamaConfig, LlamaEngine
    return LlamaEngine(LlamaConfig(vocab_size=512, n_layers=2, d_model=128, n_heads=4, n_kv_heads=2, head_dim=64, ffn=256, max_seq=256), "cuda", seed=2)


def test_recorded_steps_draw_anew():
    """A recorded decode step takes other random numbers at each replay, and its tokens are those of its own logits; another sampler records another step."""
    from litetorch_b200.models import registry
    from litetorch_b200.models.serving_base import TokenSampler
    model = registry.new_serving(_engine(), num_blocks=64, block_size=16, max_num_seqs=8)
    model.sampler = s = TokenSampler(30.0, 100, 0.98, 0.0, seed=7, device="cuda")
    first = [model.prefill_chunk(list(range(10 + i, 20 + i)), 0, [i], True) for i in range(4)]
    assert all(0 <= t < 512 for t in first)
    drawn = set()
    for _ in range(2):
        for rows in (4, 2, 4):                                    # graphs of two sizes in turn
            tokens = model.decode_batch(first[:rows], [10] * rows, [[i] for i in range(rows)])
            u = s._places[rows][0]
            want, logs = ref.sample(model.last_logits, u, 30.0, 100, 0.98, 0.0)
            assert tokens == want.tolist()
            _within(s.logprobs, logs, logs.abs() * 2.0 ** -23 + 1e-9)
            drawn.add(tuple(u.tolist()))
    assert len(drawn) == 6 and set(model._graphs) == {(4, 16), (2, 16)}
    model.sampler = TokenSampler(0.0)
    assert not model._graphs
    assert model.decode_batch(first, [10] * 4, [[i] for i in range(4)]) == model.last_logits.float().argmax(1).tolist()
    model.sampler = None
    assert model.decode_batch(first, [10] * 4, [[i] for i in range(4)]) == model.last_logits.float().argmax(1).tolist()


def test_parameters_on_the_device_are_read_at_every_replay():
    from litetorch_b200.models import registry
    from litetorch_b200.models.serving_base import TokenSampler
    model = registry.new_serving(_engine(), num_blocks=64, block_size=16, max_num_seqs=8)
    k = torch.ones((), dtype=torch.int32, device="cuda")
    model.sampler = s = TokenSampler(50.0, k, seed=7, device="cuda")
    first = model.prefill_chunk(list(range(10)), 0, [0], True)
    seen = set()
    for n in (1, 1, 200, 200, 200):
        k.fill_(n)
        token, = model.decode_batch([first], [10], [[0]])
        assert token == ref.sample(model.last_logits, s._places[1][0], 50.0, n, 1.0, 0.0)[0].item()
        seen.add(token)
    assert len(seen) > 1


def test_generate_is_seeded_and_greedy_at_its_limits():
    from litetorch_b200.models.llama_serving import generate
    engine = _engine()
    prompts = [[5, 6, 7], [9, 10, 11, 12, 13]]
    greedy = generate(engine, prompts, 12)
    a = [generate(engine, prompts, 12, temperature=20.0, top_k=100, seed=seed, sampler="kernel") for seed in (1, 1, 2)]
    assert a[0] == a[1] != a[2] and a[0] != greedy
    assert all(len(o) == 12 and all(0 <= t < 512 for t in o) for o in a[2])
