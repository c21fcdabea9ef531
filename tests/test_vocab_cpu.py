"""Embedding, distillation loss and token sampling on the CPU: the plain forms against 64-bit definitions, what is refused, and the calls that lead there."""
import ctypes
import math
import random

import pytest
import torch

import litetorch_b200 as lt
import vocab_ref as ref
from litetorch_b200.core import _unwrap
from litetorch_b200.ops import functional as Fn
from litetorch_b200.ops import kernels as K

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, bound):
    assert bool(((got.detach().double() - want).abs() <= bound).all())


# ---------------------------------------------------------------------------------------------- plain forms
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding(dtype):
    g = _gen(0)
    table = torch.randn(11, 6, generator=g).to(dtype).requires_grad_()
    idx = torch.tensor([[3, 3, -1], [10, 11, 3], [0, 1 << 40, 10]])
    dout = torch.randn(3, 3, 6, generator=g).to(dtype)
    out = Fn.token_embedding(idx, table, 1.5, -1)
    grad, = torch.autograd.grad(out, table, dout)
    want = ref.embedding(idx, table, 1.5)
    _within(out.reshape(-1, 6), want, ref.rounding(want, dtype) + want.abs() * 2.0 ** -24)
    want, bound = ref.embedding_grad(idx, dout, 11, 1.5, 10)
    # (the rows' gradients are cast to 32 bits exactly; the sum is rounded once)
    _within(grad, want, bound + ref.rounding(want, dtype) + bound * torch.finfo(dtype).eps)
    assert Fn.token_embedding(torch.empty(0, 2, dtype=torch.int32), table).shape == (0, 2, 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distillation(dtype, reduction):
    g = _gen(1)
    z = (torch.randn(5, 40, generator=g) * 3).to(dtype).requires_grad_()
    t = torch.randn(5, 6, generator=g).to(dtype)
    idx = torch.tensor([[7, 7, 7, 7, 7, 7], [1, 2, 1, 2, 39, 0], [-1, 40, 5, 1 << 40, -7, 5], [-1] * 6, [3, 4, 5, 6, 7, 8]])
    t[4, 2] = t[1, 3] = -math.inf
    with torch.no_grad():
        z[4, 10:] = torch.finfo(dtype).min
    up = torch.rand(5, generator=g) if reduction == "none" else None
    loss = Fn.distillation_loss(z, t, idx, 1.7, reduction)
    grad, = torch.autograd.grad(loss, z, up)
    rows, lost, want, bound = ref.distillation(z, t, idx, 1.7, reduction, up)
    _within(loss, rows, lost + 1e-30)
    _within(grad, want, bound + ref.rounding(want, dtype) + bound * torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_student_with_nothing_but_the_lowest_value_knows_nothing(dtype):
    z = torch.full((2, 10), torch.finfo(dtype).min, dtype=dtype).requires_grad_()
    loss = Fn.distillation_loss(z, torch.zeros(2, 1), torch.tensor([[3], [4]]), 0.5, "sum")
    grad, = torch.autograd.grad(loss, z)
    assert abs(float(loss) - 2 * 0.25 * math.log(10)) < 1e-5 and abs(float(grad[0, 3]) + 0.45) < 2.0 ** -8 and abs(float(grad[1, 0]) - 0.05) < 2.0 ** -8


def test_rows_without_a_teacher_have_no_gradient_whatever_the_student_says():
    z = torch.tensor([[-math.inf] * 4, [math.nan] * 4, [1.0, 2.0, 3.0, 4.0]]).requires_grad_()
    loss = Fn.distillation_loss(z, torch.zeros(3, 1), torch.tensor([[-1], [4], [0]]))
    loss.backward()
    assert bool(torch.isfinite(loss)) and not z.grad[:2].any() and bool(z.grad[2].all())


@pytest.mark.parametrize("dtype", TYPES)
def test_sampling(dtype):
    g = _gen(2)
    z = (torch.randn(60, 200, generator=g) * 3).to(dtype)
    z[3] = -math.inf
    z[4, 7] = math.nan
    u = torch.rand(60, generator=g)
    u[:3] = torch.tensor([0.0, 1.0, -2.0])
    for kw in (dict(), dict(tau=0.0), dict(tau=0.7, k=5), dict(p=0.8), dict(low=0.1), dict(tau=1.3, k=20, p=0.9, low=0.05)):
        args = kw.get("tau", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("low", 0.0)
        tokens, logs = Fn.sample_tokens(z, u, *args)
        want, want_logs = ref.sample(z, u, *args)
        assert torch.equal(tokens, want)
        finite = torch.isfinite(want_logs)
        assert torch.equal(torch.isfinite(logs), finite)
        _within(logs[finite], want_logs[finite], want_logs[finite].abs() * 2.0 ** -23 + 1e-9)
    k = torch.randint(0, 9, (60,), generator=g)
    assert torch.equal(Fn.sample_tokens(z, u, 1.0, k)[0], ref.sample(z, u, 1.0, k, 1.0, 0.0)[0])
    assert torch.equal(Fn.sample_tokens(z.view(3, 20, 200), u.view(3, 20), 1.0, k.view(3, 20))[0], Fn.sample_tokens(z, u, 1.0, k)[0].view(3, 20))
    assert Fn.sample_tokens(z[:0], u[:0])[0].shape == (0,)


# ---------------------------------------------------------------------------------------------- what is refused
def test_refusals_of_the_embedding():
    table, idx = torch.randn(5, 4), torch.tensor([1, 2])
    for bad in (lambda: Fn.token_embedding(idx.float(), table), lambda: Fn.token_embedding(idx.bool(), table), lambda: Fn.token_embedding(idx, table[0]),
                lambda: Fn.token_embedding(idx, table.long())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: Fn.token_embedding(idx, table, 1.0, 5), lambda: Fn.token_embedding(idx, table, 1.0, -6), lambda: Fn.token_embedding(idx, table[:0]),
                lambda: Fn.token_embedding(idx.to("meta"), table)):
        with pytest.raises(ValueError):
            bad()


def test_refusals_of_the_distillation_loss():
    z, t, idx = torch.randn(3, 8), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(TypeError):
        Fn.distillation_loss(z.long(), t, idx)
    with pytest.raises(TypeError):
        Fn.distillation_loss(z, t, idx.float())
    for args in ((z, t[:2], idx[:2]), (z, t, idx[:, :1]), (z, t[0], idx[0]), (z, t.to("meta"), idx), (z, t[:, :0], idx[:, :0]), (z[:, :0], t, idx),
                 (z, torch.zeros(3, 1025), torch.zeros(3, 1025, dtype=torch.int64)), (z, t, idx, 0.0), (z, t, idx, -1.0), (z, t, idx, math.nan), (z, t, idx, math.inf),
                 (z, t, idx, 1e-30), (z, t, idx, 1e30), (z, t, idx, 1.0, "average")):
        with pytest.raises(ValueError):
            Fn.distillation_loss(*args)


def test_refusals_of_sampling():
    z, u = torch.randn(3, 8), torch.rand(3)
    with pytest.raises(TypeError):
        Fn.sample_tokens(z.long(), u)
    with pytest.raises(TypeError):
        Fn.sample_tokens(z, u, top_k=2.5)
    with pytest.raises(TypeError):
        Fn.sample_tokens(z, u, top_k=torch.tensor([1.0, 2.0, 3.0]))
    for bad in (dict(uniform=u[:2]), dict(uniform=u.to("meta")), dict(uniform=u.long()), dict(uniform=0.5), dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=math.nan),
                dict(temperature=torch.ones(2)), dict(top_p=torch.ones(3, device="meta")), dict(logits=z[:, :0])):
        with pytest.raises(ValueError):
            Fn.sample_tokens(**{**dict(logits=z, uniform=u), **bad})
    with pytest.raises(ValueError):
        Fn.sample_tokens(torch.zeros(1, (1 << 19) + 1), u[:1])


def test_the_native_calls_refuse_what_they_cannot_take():
    """Every refusal comes before anything is launched; no pointer is read."""
    fn = K._fn
    embed = lambda type=0, n=4, D=8, V=9: fn("lt_token_embedding_fwd")(type, None, 0, None, None, n, D, V, 1.0, None)
    grad = lambda type=0, n=4, D=8, V=9, tile=8: fn("lt_token_embedding_bwd")(type, None, 0, None, 8, None, n, D, V, 1.0, -1, None, None, tile, None)
    for rc in (embed(type=3), embed(type=-1), embed(n=-1), embed(n=1 << 31), embed(D=-1), embed(D=(1 << 30) + 1), embed(V=0), grad(type=3), grad(n=-1), grad(n=(1 << 31) - 4096),
               grad(D=-1), grad(D=(1 << 30) + 1), grad(V=0), grad(V=(1 << 31) - 1), grad(tile=0), grad(tile=65)):
        assert rc < 0
    assert embed(n=0) == embed(D=0) == grad(D=0) == 0

    def distill(type=0, z=0, ldz=8, t_type=0, t=16, entries=0, N=2, V=8, K=1, T=1.0, stats=16, loss=16, out=None, grad=None, ldg=8, flags=None):
        return fn("lt_distill")(type, z, ldz, t_type, t, None, entries, N, V, K, T, flags, None, 0, 0, stats, 0, loss, out, grad, ldg, None)
    for bad in (dict(type=3), dict(t_type=-1), dict(N=-1), dict(N=1 << 30), dict(V=0), dict(V=1 << 30), dict(K=0), dict(K=1025), dict(T=0.0), dict(T=-1.0), dict(T=math.nan),
                dict(T=1e-30), dict(T=1e30), dict(entries=4), dict(flags=8), dict(out=16, loss=8), dict(stats=None), dict(t=None), dict(loss=None, out=16), dict(grad=4), dict(grad=16, ldg=9)):
        assert distill(**bad) < 0
    assert distill(N=0) == 0
    draw = lambda type=0, rows=2, V=8: fn("lt_sample_tokens")(type, None, 8, None, 0, None, None, None, None, 1.0, 0, 1.0, 0.0, rows, V, None, None, None)
    assert draw(type=3) < 0 and draw(rows=-1) < 0 and draw(V=0) < 0 and draw(V=(1 << 19) + 1) < 0 and draw(rows=0) == 0


def test_parts_of_the_distillation_kernels_shared_memory():
    """Every part lies where its widest access may go, whatever the number of entries, none reaches into the next, and all of it is there."""
    places = (ctypes.c_int * 5)()
    for threads in (32, 64, 128, 256, 512):
        for top in range(1, 1025):
            link, most = (1, 8) if top <= 255 else (2, 5)
            for vectors in range(1, most + 1):
                assert K._fn("lt_distill_places")(top, threads, vectors, places) == 0
                entries, pairs, chains, links, end = places
                # 16-byte vectors, 8-byte entries and pairs, the chains of a thread's eight vectors at once, links
                assert entries % 16 == 0 and pairs % 8 == 0 and chains % (8 * link) == 0 and links % link == 0, (top, threads, vectors)
                assert entries >= 3 * threads * vectors * 16 and pairs >= entries + 5 * 8 * top and chains >= pairs + 4 * 8 * 8 * (threads // 32)
                assert links >= chains + 4 * 8 * link * threads and end >= links + 4 * link * top and end <= 227 * 1024 - 1024
    assert K._fn("lt_distill_places")(1025, 512, 5, places) < 0 and K._fn("lt_distill_places")(0, 512, 5, places) < 0


def test_a_gradient_without_a_workspace_is_one_of_few_tokens():
    """One launch takes up to 2048 tokens; refused before anything is launched."""
    assert K._fn("lt_token_embedding_bwd")(0, None, 0, None, 8, None, 2049, 8, 9, 1.0, -1, None, None, 1, None) < 0


def test_the_autograd_node_refuses_what_its_kernels_cannot_take():
    """Checked before anything is launched; the public function makes dense tensors of what it is given."""
    idx, table = torch.tensor([1, 2]), torch.randn(5, 4)
    for args in ((idx, table), (idx, table.to("meta")), (idx, table.long()), (idx.float(), table), (idx, table[0])):
        with pytest.raises(RuntimeError, match="dense tokens and a dense table"):
            K.token_embedding(*args)
    assert K.launch_count() >= 0


class _Overrun(Exception):
    pass


def _rows_by_phases(rng, ctas, warps, rows, slow, heeded):
    """The warps of a cluster that go over rows as the distillation kernel's do, in any order of their steps: a warp sends its pair of a row to all CTAs and arrives at its
    own one's barrier for the row (four in turn), then waits for the barrier of the row before.  Waits that are not over run out with the probability `slow`;
    heeded: such a warp stops.  Returns whether a wait ran out; raises if something is counted into the phase of another row."""
    pending = [[[row, warps, ctas * warps] for row in range(4)] for _ in range(ctas)]             # row of the phase, arrivals and pairs that are missing

    def count(cta, row, what):
        p = pending[cta][row % 4]
        if p[0] != row:
            raise _Overrun
        p[what] -= 1
        if p[1] == 0 and p[2] == 0:
            p[0], p[1], p[2] = row + 4, warps, ctas * warps

    def warp(cta):
        for row in range(rows + 1):
            if row < rows:
                for to in rng.sample(range(ctas), ctas):
                    count(to, row, 2)
                    yield True
                count(cta, row, 1)
                yield True
            if row > 0:
                while pending[cta][(row - 1) % 4][0] == row - 1:
                    if rng.random() < slow:
                        out.append(row - 1)
                        if heeded:
                            return
                        break
                    yield True

    out = []
    running = [warp(c) for c in range(ctas) for _ in range(warps)]
    weights = [rng.choice((1, 1, 30)) for _ in running]
    for _ in range(200000):
        if not running:
            return bool(out)
        i = rng.choices(range(len(running)), weights)[0]
        if next(running[i], None) is None:
            del running[i], weights[i]
    assert heeded and out, "a wait that never ends"                # (here a wait without a limit, which others have left)
    return True


def test_no_row_is_counted_into_the_phase_of_another():
    """The protocol of the kernel that holds rows: phases stay apart whatever the order, and, if a wait runs out, because that warp stops."""
    assert not any(_rows_by_phases(random.Random(seed), 1 + seed % 3, 1 + seed % 4, 12, 0.0, True) for seed in range(60))
    ran_out = [_rows_by_phases(random.Random(seed), 1 + seed % 3, 2 + seed % 3, 12, 0.02, True) for seed in range(200)]
    assert sum(ran_out) > 100
    overruns = 0
    for seed in range(200):                                       # (what becomes of it otherwise)
        try:
            _rows_by_phases(random.Random(seed), 1 + seed % 3, 2 + seed % 3, 12, 0.02, False)
        except _Overrun:
            overruns += 1
    assert overruns > 0


# ---------------------------------------------------------------------------------------------- the calls that lead there
def test_operators_and_modules():
    g = _gen(3)
    table = lt.Tensor(torch.randn(9, 4, generator=g).requires_grad_())
    idx = torch.tensor([[1.0, 8.0], [3.0, 1.0]])                  # indices may be floats
    out = lt.Ops.embedding(lt.Tensor(idx), table, 2.0, 8)
    assert torch.equal(_unwrap(out), _unwrap(table)[idx.long()] * 2.0)
    lt.Ops.sum(out).backward()
    want = torch.zeros(9, 4)
    want[1], want[3] = 4.0, 2.0
    assert torch.equal(_unwrap(table).grad, want)
    plain, scaled = lt.nn.Embedding(9, 4), lt.nn.Embedding(9, 4, scale=0.5, padding_idx=1)
    assert not plain.sorted_grad and lt.nn.Embedding(9, 4, sorted_grad=True).sorted_grad
    with torch.no_grad():
        _unwrap(scaled.weight).copy_(_unwrap(plain.weight))
    a, b = plain(lt.Tensor(idx)), scaled(lt.Tensor(idx))
    assert torch.equal(_unwrap(a) * 0.5, _unwrap(b))
    lt.Ops.sum(b).backward()
    assert _unwrap(scaled.weight).grad.abs().sum(1).tolist() == [0, 0, 0, 2, 0, 0, 0, 0, 2]
    with pytest.raises(ValueError):
        lt.nn.Embedding(9, 4, padding_idx=9)(lt.Tensor(idx))

    z = lt.Tensor(torch.randn(2, 9, generator=g).requires_grad_())
    t, cls = torch.randn(2, 3, generator=g), torch.tensor([[0.0, 5.0, -1.0], [8.0, 2.0, 3.0]])
    loss = lt.nn.DistillationLoss(2.0, "sum")(z, lt.Tensor(t), lt.Tensor(cls))
    assert loss.shape == [1] and loss.item() == float(Fn.distillation_loss(_unwrap(z), t, cls.long(), 2.0, "sum"))
    loss.backward()
    assert torch.equal(_unwrap(z).grad, torch.autograd.grad(Fn.distillation_loss(_unwrap(z), t, cls.long(), 2.0, "sum"), _unwrap(z))[0])
    assert lt.Ops.distillation_loss(z, lt.Tensor(t), lt.Tensor(cls), reduction="none").shape == [2]

    u = torch.rand(2, generator=g)
    tokens, logs = lt.Ops.sample_tokens(lt.Tensor(_unwrap(z).detach()), lt.Tensor(u), lt.Tensor(torch.tensor([0.5, 2.0])), 4, 0.9)
    want = Fn.sample_tokens(_unwrap(z), u, torch.tensor([0.5, 2.0]), 4, 0.9)
    assert torch.equal(_unwrap(tokens), want[0]) and torch.equal(_unwrap(logs), want[1])


def test_a_row_of_its_own_for_every_loss():
    """The losses of reduction "none" may be changed in place before they are added up."""
    z = torch.randn(4, 9, generator=_gen(4)).requires_grad_()
    t, cls = torch.randn(4, 2, generator=_gen(5)), torch.tensor([[1, 2]] * 4)
    loss = Fn.distillation_loss(z, t, cls, reduction="none")
    loss *= torch.tensor([1.0, 0.0, 2.0, 0.0])
    loss.sum().backward()
    assert not z.grad[1::2].any() and bool(z.grad[::2].any(1).all())


def test_a_top_k_for_every_row_may_be_floats():
    """As indices of the other operators on framework tensors may."""
    g = _gen(8)
    z, u, k = torch.randn(4, 30, generator=g), torch.rand(4, generator=g), torch.tensor([1.0, 3.0, 0.0, 30.0])
    tokens, logs = lt.Ops.sample_tokens(lt.Tensor(z), lt.Tensor(u), 0.9, lt.Tensor(k))
    want = Fn.sample_tokens(z, u, 0.9, k.long())
    assert torch.equal(_unwrap(tokens), want[0]) and torch.equal(_unwrap(logs), want[1])
    with pytest.raises(TypeError):                                # (a number that is none of a count stays refused)
        lt.Ops.sample_tokens(lt.Tensor(z), lt.Tensor(u), 0.9, 2.5)


def test_nan_among_the_rows_parameters():
    """A temperature that is NaN is one of 0, a limit that is NaN is off; the other rows are as they were."""
    g = _gen(9)
    z, u = torch.randn(3, 200, generator=g) * 3, torch.rand(3, generator=g)
    nan = math.nan
    for kw, off in ((dict(temperature=torch.tensor([0.7, nan, 1.5])), dict(temperature=torch.tensor([0.7, 0.0, 1.5]))),
                    (dict(top_p=torch.tensor([0.5, nan, 0.9])), dict(top_p=torch.tensor([0.5, 1.0, 0.9]))),
                    (dict(min_p=torch.tensor([0.1, nan, 0.9])), dict(min_p=torch.tensor([0.1, 0.0, 0.9]))),
                    (dict(top_k=4, top_p=torch.tensor([0.5, nan, 0.9]), min_p=torch.tensor([nan, nan, 0.2])),
                     dict(top_k=4, top_p=torch.tensor([0.5, 1.0, 0.9]), min_p=torch.tensor([0.0, 0.0, 0.2])))):
        got, want = Fn.sample_tokens(z, u, **kw), Fn.sample_tokens(z, u, **off)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), kw


def _model(vocab=64):
    from litetorch_b200.models.llama import LlamaConfig, LlamaEngine
    cfg = LlamaConfig(vocab_size=vocab, n_layers=1, d_model=32, n_heads=2, n_kv_heads=1, head_dim=16, ffn=48, max_seq=64)
    return LlamaEngine(cfg, "cpu", seed=3)


def test_generate_draws_by_given_numbers():
    from litetorch_b200.models.llama_serving import generate
    engine = _model()
    prompts = [[5, 6, 7], [9, 10, 11, 12, 13]]
    greedy = generate(engine, prompts, 6)
    assert generate(engine, prompts, 6, temperature=0.7, top_k=1, sampler="kernel") == greedy
    a = generate(engine, prompts, 6, temperature=3.0, top_k=20, top_p=0.95, min_p=0.01, seed=5)
    assert a == generate(engine, prompts, 6, temperature=3.0, top_k=20, top_p=0.95, min_p=0.01, seed=5, sampler="kernel")
    assert a != generate(engine, prompts, 6, temperature=3.0, top_k=20, top_p=0.95, min_p=0.01, seed=6)
    assert generate(engine, prompts, 6, temperature=1.0, min_p=1.0) == greedy              # none but the likeliest
    with pytest.raises(ValueError):
        generate(engine, prompts, 6, sampler="dice")


def test_the_sampler_of_a_served_model():
    from litetorch_b200.models import registry
    from litetorch_b200.models.serving_base import TokenSampler
    model = registry.new_serving(_model(), num_blocks=16, block_size=8, max_num_seqs=4)
    model.sampler = s = TokenSampler(2.0, 10, 0.9, 0.0, seed=1)
    first = model.prefill_chunk([1, 2, 3], 0, [3], True)
    u = torch.rand(3, generator=torch.Generator().manual_seed(1))
    assert first == int(Fn.sample_tokens(model.last_logits, u[:1], 2.0, 10, 0.9)[0])
    tokens = model.decode_batch([first, 7], [3, 0], [[3], [4]])
    want, logs = Fn.sample_tokens(model.last_logits, u[1:], 2.0, 10, 0.9)
    assert tokens == want.tolist() and torch.equal(s.logprobs, logs)
    model._graphs["a recorded step"] = None
    model.sampler = s
    assert model._graphs
    model.sampler = None                                          # steps that were recorded with another sampler go
    assert not model._graphs
    for bad in (dict(temperature=torch.ones(2)), dict(top_k=torch.ones(1, dtype=torch.int32)), dict(min_p=torch.zeros(3))):
        with pytest.raises(ValueError):
            TokenSampler(**bad)


def test_the_server_takes_the_sampling_parameters(monkeypatch):
    from litetorch_b200 import server
    from litetorch_b200.models import registry
    from litetorch_b200.models.serving_base import TokenSampler
    seen = []

    class Stop(Exception):
        pass

    def loop(model, *a, **k):
        seen.append(model.sampler)
        raise Stop

    monkeypatch.setattr(registry, "load_engine", lambda *a: _model())
    monkeypatch.setattr(server, "EngineLoop", loop)
    for extra in ([], ["--temperature", "0.8", "--top-k", "40", "--top-p", "0.9", "--min-p", "0.02", "--seed", "4"]):
        with pytest.raises(Stop):
            server.main(["--model", "none", "--device", "cpu", "--bytes", "--kv-blocks", "8"] + extra)
    assert seen[0] is None and isinstance(seen[1], TokenSampler) and seen[1].params == (0.8, 40, 0.9, 0.02)
