"""Sampling and top logits through the model mirror: generate, the continuous-batch decoder, a teacher's top logits, and a
distillation step over them.  CPU: with the oracle as the cell (host logic).  GPU: the kernels."""
import types

import pytest
import torch

from oracle import vocab as V
from test_large_model import _continuous_case, _oracle_cell
from xlstm_b200.large_model import ContinuousDecoder, LargeConfig, LargeModel, Sampling, procedural_state_dict

CFG = LargeConfig(embedding_dim=128, num_heads=2, num_blocks=2, vocab_size=64)
SETTINGS = [Sampling(0.8, 20, 0.9, 0.0), Sampling(), Sampling(0.0), Sampling(1.2, 0, 1.0, 0.05), Sampling(1.0, 5), Sampling(0.7, 0, 0.8), Sampling(1.5, 1)]


def _model(device):
    kw = dict(cell_ops=_oracle_cell()) if device == "cpu" else {}
    return LargeModel(CFG, procedural_state_dict(CFG, 4), device, torch.float32, **kw)


def _alone(model, prompt, count, settings, numbers):
    """Token by token with given numbers."""
    last, state, out = prompt[None].to(model.device), None, []
    for u in numbers.reshape(count, 1):
        last, state = model.forward(last, state, sampling=settings, u=u)
        out.append(last[0, 0])
    return torch.stack(out).cpu()


def test_generate_draws_what_the_oracle_draws_on_cpu():
    model = _model("cpu")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1))
    s = Sampling(torch.tensor([0.9, 1.3, 0.0]), 12, 0.95, torch.tensor([0.0, 0.02, 0.0]))
    a, _ = model.generate(prompt, 6, sampling=s, generator=torch.Generator().manual_seed(5))
    b, _ = model.generate(prompt, 6, sampling=s, generator=torch.Generator().manual_seed(5))
    assert torch.equal(a, b)
    u = torch.rand(18, generator=torch.Generator().manual_seed(5)).reshape(6, 3)
    greedy, _ = model.generate(prompt, 6)
    assert torch.equal(a[2], greedy[2])                       # temperature 0
    last, state = prompt, None
    for i in range(6):
        logits, state = model.forward(last, state, last_only=True)
        raw = CFG.output_logit_soft_cap * torch.atanh(logits[:, -1].double() / CFG.output_logit_soft_cap)   # (fp32 logits: ties aside)
        for r in range(2):
            token, margin = V.sample_row(raw[r], CFG.output_logit_soft_cap, u[i, r], float(s.temperature[r]), 12, 0.95, float(s.min_p[r]))
            assert token == int(a[r, i]) or margin < 1e-5
        last = a[:, i:i + 1]


def test_decoder_draws_the_same_tokens_in_any_company_on_cpu():
    model = _model("cpu")
    prompts, counts = _continuous_case()
    runs = [ContinuousDecoder(model, 3, sampling=True).run(prompts, counts, sampling=SETTINGS, generator=torch.Generator().manual_seed(9)),
            ContinuousDecoder(model, 2, sampling=True).run(prompts, counts, quantum=2, sampling=SETTINGS, generator=torch.Generator().manual_seed(9)),
            ContinuousDecoder(model, 3, row_len=96, packed_admission=True, sampling=True).run(prompts, counts, sampling=SETTINGS,
                                                                                             generator=torch.Generator().manual_seed(9))]
    numbers = torch.rand(sum(counts), generator=torch.Generator().manual_seed(9)).split(counts)
    for d, (p, c) in enumerate(zip(prompts, counts)):
        want = _alone(model, p, c, SETTINGS[d], numbers[d])
        assert all(torch.equal(r[d], want) for r in runs), d
    for bad in (dict(sampling=SETTINGS[:3]), dict(sampling=Sampling(-1.0)), dict(sampling=Sampling(1.0, 0, 1.5)), dict(sampling=Sampling(torch.ones(3))), {}):
        with pytest.raises(ValueError):
            ContinuousDecoder(model, 3, sampling=True).run(prompts, counts, **bad)
    with pytest.raises(ValueError):
        ContinuousDecoder(model, 3).run(prompts, counts, sampling=Sampling())


def test_a_captured_step_serves_only_the_settings_it_was_captured_with():
    model = _model("cpu")
    for change in ("temperature", "top_k", "top_p", "min_p"):
        s = Sampling(0.9, 10)
        model._remember_sampling(s)
        assert model._captured_for(s) and model._captured_for(Sampling(0.9, 10)) and not model._captured_for(None)
        setattr(s, change, getattr(s, change) / 2 if change != "min_p" else 0.1)      # the same object, with other settings
        assert not model._captured_for(s)
    rows = Sampling(torch.tensor([0.9, 1.3]))
    model._remember_sampling(rows)
    assert model._captured_for(rows) and model._captured_for(Sampling(rows.temperature))   # (the step reads the tensor anew)
    assert not model._captured_for(Sampling(rows.temperature.clone()))
    rows.temperature = torch.tensor([0.9, 1.3])
    assert not model._captured_for(rows)
    model._remember_sampling(None)
    assert model._captured_for(None) and not model._captured_for(Sampling())


@pytest.mark.parametrize("top_k", [2.5, 2 ** 31, float("inf"), float("nan")])
def test_decoder_refuses_a_top_k_that_its_vector_cannot_hold(top_k):
    prompts, counts = _continuous_case()
    with pytest.raises(ValueError):
        ContinuousDecoder(_model("cpu"), 3, sampling=True).run(prompts, counts, sampling=Sampling(1.0, top_k))


def test_top_logits_on_cpu():
    model = _model("cpu")
    tokens = torch.randint(0, 64, (2, 21), generator=torch.Generator().manual_seed(2))
    values, ids, lse = model.top_logits(tokens, 7, 2.0)
    logits, _ = model.forward(tokens)
    assert values.shape == ids.shape == (2, 21, 7) and lse.shape == (2, 21)
    torch.testing.assert_close(values, logits.topk(7, dim=-1).values)
    torch.testing.assert_close(values, logits.gather(-1, ids.long()))
    torch.testing.assert_close(lse, torch.logsumexp(logits / 2.0, -1))


@pytest.mark.gpu
def test_generate_with_a_captured_step_draws_the_eager_tokens():
    model = _model("cuda")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1)).cuda()
    gen = lambda seed: torch.Generator(device="cuda").manual_seed(seed)   # noqa: E731
    per_row = Sampling(torch.tensor([0.9, 1.3, 0.0]).cuda(), 12, 0.95, torch.tensor([0.0, 0.02, 0.0]).cuda())
    for s in (Sampling(0.9, 10), Sampling(0.9, 10), Sampling(1.1, 0, 0.9), per_row, None, per_row):
        eager, _ = model.generate(prompt, 8, sampling=s, generator=gen(5))
        graphed, _ = model.generate(prompt, 8, use_cuda_graph=True, sampling=s, generator=gen(5))
        assert torch.equal(eager, graphed)
    other, _ = model.generate(prompt, 8, sampling=Sampling(2.0), generator=gen(6))
    assert not torch.equal(other, model.generate(prompt, 8)[0])
    model.release_graph()


@pytest.mark.gpu
def test_a_captured_step_follows_its_settings():
    model = _model("cuda")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1)).cuda()
    gen = lambda: torch.Generator(device="cuda").manual_seed(5)   # noqa: E731
    s = Sampling(2.0)
    for temperature in (2.0, 0.0, torch.tensor([0.0, 2.0, 0.0]).cuda(), 1.0):
        s.temperature = temperature
        eager, _ = model.generate(prompt, 8, sampling=s, generator=gen())
        assert torch.equal(eager, model.generate(prompt, 8, use_cuda_graph=True, sampling=s, generator=gen())[0])
    s.temperature = rows = torch.tensor([0.0, 2.0, 0.0]).cuda()
    for values in ([0.0, 2.0, 0.0], [2.0, 0.0, 1.0]):             # in place
        rows.copy_(torch.tensor(values))
        eager, _ = model.generate(prompt, 8, sampling=s, generator=gen())
        assert torch.equal(eager, model.generate(prompt, 8, use_cuda_graph=True, sampling=s, generator=gen())[0])
    model.release_graph()


@pytest.mark.gpu
def test_a_decoder_and_generate_on_one_model():
    model = _model("cuda")
    prompts, counts = _continuous_case()
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1)).cuda()
    gen = lambda: torch.Generator(device="cuda").manual_seed(5)   # noqa: E731
    want = model.generate(prompt, 8)[0]
    for kw in ({}, dict(sampling=True)):
        dec = ContinuousDecoder(model, 3, **kw)
        settings = dict(sampling=Sampling(0.9), generator=gen()) if kw else {}
        dec.run(prompts, counts, **settings)
        assert torch.equal(model.generate(prompt, 8, use_cuda_graph=True)[0], want)   # a step of its own: no slots
        with pytest.raises(RuntimeError):                                             # the decoder's step is gone
            dec.run(prompts, counts, **settings)
    model.release_graph()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [True, False])
def test_decoder_draws_the_same_tokens_in_any_company_on_gpu(packed):
    import xlstm_b200
    model = _model("cuda")
    prompts, counts = _continuous_case()
    gen = lambda: torch.Generator(device="cuda").manual_seed(9)   # noqa: E731
    dec = ContinuousDecoder(model, 3, packed_admission=packed, sampling=True)
    assert dec.graphed
    outs = dec.run(prompts, counts, sampling=SETTINGS, generator=gen())
    sliced = dec.run(prompts, counts, quantum=3, park_on_host=True, sampling=SETTINGS, generator=gen())
    assert dec.evictions > 0
    one = dec.run(prompts, counts, sampling=Sampling(0.0))
    xlstm_b200.check_device_status()
    model.release_graph()
    numbers = torch.rand(sum(counts), device="cuda", generator=gen()).split(counts)
    for d, (p, c) in enumerate(zip(prompts, counts)):
        want = _alone(model, p, c, SETTINGS[d], numbers[d])
        assert torch.equal(outs[d], want) and torch.equal(sliced[d], want)
        assert torch.equal(one[d], model.generate(p[None].cuda(), c)[0][0].cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_teacher_and_a_student_and_its_tokens(dtype):
    """The operators as they are used together: a teacher's top logits of a packed batch, a student (sLSTM cell and head) that
    is distilled from them -- in pieces with known weights, and through autograd --, and tokens drawn from its logits."""
    import xlstm_b200
    from xlstm_b200 import ops
    teacher = LargeModel(CFG, procedural_state_dict(CFG, 4), "cuda", dtype)
    g = torch.Generator().manual_seed(3)
    B, S, NH, DH, T = 2, 48, 2, 64, 2.0
    tokens = torch.randint(0, 64, (B, S), generator=g).cuda()
    values, ids, lse = teacher.top_logits(tokens, 8, T, cu_seqlens=[0, 20, 48, 96])
    alone = teacher.top_logits(tokens[1:], 8, T)
    assert torch.equal(ids[1:], alone[1]) or dtype is torch.bfloat16
    ids[0, 40:] = -1                                         # padding behind the first row's documents
    weight = torch.full((B, S), 1.0 / (B * S)).cuda()
    wx = (0.5 * torch.randn(B, S, 4 * NH * DH, generator=g)).bfloat16().cuda()
    R = (0.05 * torch.randn(NH, DH, 4, DH, generator=g)).bfloat16().cuda()
    bias = (0.1 * torch.randn(NH, 4, DH, generator=g)).cuda()
    head = (torch.randn(64, NH * DH, generator=g) / 8).to(dtype).cuda()

    def student(leaves):
        h, _ = ops.SlstmFunction.apply(leaves[0], leaves[1], bias, None)
        return h.transpose(1, 2).reshape(B, S, NH * DH).to(dtype) @ leaves[2].t()
    grads = []
    for way in ("autograd", "pieces", "plain"):
        leaves = [t.clone().requires_grad_() for t in (wx, R, head)]
        logits = student(leaves)
        if way == "autograd":
            (ops.distill_topk(logits, values, ids, 30.0, T, lse) * weight).sum().backward()
        elif way == "pieces":
            got = [ops.distill_topk_grad(logits[b].detach(), values[b], ids[b], weight[b], 30.0, T, lse[b])[1] for b in range(B)]
            logits.backward(torch.stack(got))
        else:
            d = V.distill_grad(logits.detach().double().cpu().reshape(B * S, 64), values.cpu().reshape(B * S, 8), ids.cpu().reshape(B * S, 8), 30.0, T,
                               lse.cpu().reshape(B * S))
            logits.backward((d.reshape(B, S, 64).cuda() * weight[..., None]).to(dtype))
        grads.append([t.grad.double() for t in leaves])
    xlstm_b200.check_device_status()
    # the kernels' gradient of the logits is the formula's rounded once (fp32: a few 2^-24 more); what follows is the same code
    tol = 2e-2 if dtype is torch.bfloat16 else 5e-3          # (bf16 roundings of dwx and R's gradient flip on last bits of dlogits: 2^-8 and a few)
    for a, b, c in zip(*grads):
        assert torch.isfinite(a).all()
        assert float((a - c).norm() / c.norm()) < tol and float((b - c).norm() / c.norm()) < tol
    assert torch.equal(grads[0][2] != 0, grads[2][2] != 0)
    drawn = xlstm_b200.softcap_sample(logits.detach(), 30.0, torch.rand(B, S, generator=g).cuda(), 0.8, 10, 0.9)
    kept = xlstm_b200.softcap_topk(logits.detach(), 30.0, 10)[1]
    assert bool((kept == drawn[..., None]).any(-1).all())    # every token is one of its row's ten largest


def test_sampling_off_the_gpu_is_the_operators_definition():
    """Masked, NaN and infinite logits, numbers outside [0, 1), settings per row: large_model._sample against the oracle."""
    import math

    from xlstm_b200 import large_model as L
    g = torch.Generator().manual_seed(12)
    x = 3 * torch.randn(11, 200, generator=g)
    x[0, ::2] = math.nan
    x[1, 5:] = -math.inf
    x[2] = math.nan
    x[3] = -math.inf
    x[4], x[4, ::3] = -math.inf, math.nan
    x[5, 7], x[5, 8], x[5, 9:40] = math.inf, math.nan, 500.0
    x[6, 100] = math.inf
    x[7, 199] = math.nan
    x[8] = 2.0
    u = torch.tensor([0.3, 0.9, 0.9, 0.9, 0.9, 0.9, 0.5, 0.999, 2.0, math.nan, -1.0])
    for kw in ({}, dict(T=0.5, k=20), dict(T=4.0, p=0.8), dict(mp=0.2), dict(T=3.0, k=150, p=0.9, mp=0.01)):
        s = Sampling(kw.get("T", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("mp", 0.0))
        got = L._sample(x, 30.0, u, s)
        assert got.shape == (11, 1)
        for r in range(11):
            assert int(got[r]) == V.sample_row(x[r], 30.0, u[r].nan_to_num(0.0), **kw)[0], (kw, r)
    greedy = L._sample(x, 30.0, u, Sampling(0.0))[:, 0]          # NaN is passed over, -inf stands at -cap
    assert greedy.tolist() == [int(torch.argmax((30.0 * torch.tanh(r / 30.0)).nan_to_num(-math.inf))) for r in x]


def test_top_logits_off_the_gpu_are_the_operators_definition():
    """NaN comes last, behind -inf; equal logits by index."""
    import math

    from xlstm_b200 import large_model as L
    g = torch.Generator().manual_seed(13)
    x = torch.randint(-3, 4, (6, 40), generator=g).float()
    x[0, ::2] = math.nan
    x[1], x[1, ::3] = -math.inf, math.nan
    x[2] = math.nan
    x[3, 5], x[3, 6], x[3, 7] = math.inf, -math.inf, math.nan
    x[4] = -math.inf
    for k in (1, 7, 40):
        values, ids, lse = L._top(x, 30.0, k, 2.0)
        for r in range(6):
            y, idx, l = V.topk_row(x[r], 30.0, k, 2.0)
            assert ids[r].tolist() == idx
            torch.testing.assert_close(values[r].double(), y, rtol=1e-6, atol=0, equal_nan=True)
            torch.testing.assert_close(lse[r].double(), l, rtol=1e-6, atol=1e-6, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 5])
def test_top_logits_leave_the_callers_state_as_it_was(dtype, S):
    """The states are not handed back, so the given ones stay those in front of the tokens (a decode step updates C in place)."""
    model = LargeModel(CFG, procedural_state_dict(CFG, 4), "cuda", dtype)
    g = torch.Generator().manual_seed(1)
    prompt, more = (torch.randint(0, 64, (3, n), generator=g).cuda() for n in (17, S))
    _, state = model.forward(prompt)
    before = {i: tuple(t.clone() for t in st) for i, st in state.items()}
    first = model.top_logits(more, 5, 1.0, state=state)
    for i, st in state.items():
        assert all(torch.equal(a, b) for a, b in zip(st, before[i]))
    again = model.top_logits(more, 5, 1.0, state=state)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    logits, _ = model.forward(more, state)
    # cap * tanh(x / cap): three roundings by half a step on either side (tanh in fp32 by two steps: 8 half steps in all, twice); in
    # bf16 on the side of the logits alone
    tol = 16 * 2.0 ** -24 if dtype is torch.float32 else 3.1 * 2.0 ** -8
    torch.testing.assert_close(first[0], logits.float().topk(5, dim=-1).values, rtol=tol, atol=0)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_drawing_does_not_depend_on_the_default_type(default):
    """Uniform numbers, the slots' settings and the captured step's buffers are float32 whatever torch's default is."""
    model = _model("cpu")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1))
    prompts, counts = _continuous_case()
    gen = lambda: torch.Generator().manual_seed(5)   # noqa: E731
    s = Sampling(0.9, 12, 0.95, 0.01)

    def draw():
        return [model._uniform(100, gen()), model.generate(prompt, 6, sampling=s, generator=gen())[0],
                *ContinuousDecoder(model, 3, sampling=True).run(prompts, counts, sampling=s, generator=gen())]
    want = draw()
    torch.set_default_dtype(default)
    try:
        got = draw()
    finally:
        torch.set_default_dtype(torch.float32)
    assert got[0].dtype == torch.float32
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_captured_draws_do_not_depend_on_the_default_type():
    model = _model("cuda")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1)).cuda()
    prompts, counts = _continuous_case()
    gen = lambda: torch.Generator(device="cuda").manual_seed(5)   # noqa: E731
    s = Sampling(0.9, 12, 0.95, 0.01)

    def draw():
        out = [model.generate(prompt, 6, use_cuda_graph=True, sampling=s, generator=gen())[0].cpu(),
               *ContinuousDecoder(model, 3, sampling=True).run(prompts, counts, sampling=s, generator=gen())]
        model.release_graph()
        return out
    want = draw()
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = draw()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("fails_at", [0, 2])      # in the first warm-up step, in the capture
def test_a_capture_that_fails_leaves_no_step_behind(fails_at):
    """The earlier step's buffers are gone by then: it must not be replayed for the settings that it was captured with."""
    model = _model("cuda")
    prompt = torch.randint(0, 64, (3, 17), generator=torch.Generator().manual_seed(1)).cuda()
    gen = lambda: torch.Generator(device="cuda").manual_seed(5)   # noqa: E731
    a, b = Sampling(0.9, 10), Sampling(1.1)
    want = model.generate(prompt, 8, sampling=a, generator=gen())[0]
    assert torch.equal(model.generate(prompt, 8, use_cuda_graph=True, sampling=a, generator=gen())[0], want)
    forward, calls = model.forward, [0]

    def failing(tokens, *args, **kw):
        if tokens.shape[1] == 1:
            calls[0] += 1
            if calls[0] > fails_at:
                raise MemoryError
        return forward(tokens, *args, **kw)
    model.forward = failing
    with pytest.raises(MemoryError):
        model.generate(prompt, 8, use_cuda_graph=True, sampling=b, generator=gen())
    del model.forward
    assert model._graph is None
    assert torch.equal(model.generate(prompt, 8, use_cuda_graph=True, sampling=a, generator=gen())[0], want)
    model.release_graph()
