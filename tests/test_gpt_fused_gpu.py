"""GPU: the GPT step with the vocabulary-sized operators (GPTConfig.fused_vocab):
against the step that keeps its logits, replayed from a CUDA graph, and with
distillation from a teacher."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def make(fused, params=None, **kw):
    from dreamcompiler_b200.gpt import GPT, GPTConfig
    cfg = GPTConfig(n_layer=2, d_model=128, n_head=4, seq_len=32, batch=8, vocab=kw.pop("vocab", 65), fused_vocab=fused,
                    **kw)
    return GPT(cfg, params=params, seed=3)


def batch(m, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = m.cfg
    tok, tgt = (torch.randint(0, c.vocab, (c.batch, c.seq_len), generator=g, dtype=torch.int32) for _ in range(2))
    m.set_batch(tok.cuda(), tgt.cuda())


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("vocab", [65, 1000])
def test_step_matches_the_one_with_logits(dgx, vocab):
    a, b = make(False, vocab=vocab), make(True, vocab=vocab)
    batch(a)
    batch(b)
    la, lb = a.forward_backward().item(), b.forward_backward().item()
    dgx.sync_check()
    # the same bf16 operands and fp32 accumulation: 64 terms a logit apart at most in order
    assert abs(la - lb) <= 1e-5 * abs(la)
    # each side rounds the logit gradient to bf16 once (2^-8 of it), so the head's gradients differ by at most
    # twice that in norm; the blocks below pass it on through bf16 operands of their own
    for name in ("Wout", "bout"):
        assert rel(b.g[name][:vocab], a.g[name][:vocab]) <= 2 * 2.0 ** -8, name
        assert not b.g[name][vocab:].any()
    for name in ("W_tok", "P", "Wqkv0", "W21"):
        assert rel(b.g[name], a.g[name]) <= 8 * 2.0 ** -8, name


def test_training_and_graph_replay(dgx):
    m, e = make(True), make(True)
    batch(m)
    batch(e)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            m.step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step()
    first = None
    for i in range(20):
        graph.replay()
        if first is None:
            first = m.loss.item()
    for _ in range(22):
        e.step()
    dgx.sync_check()
    assert m.loss.item() < first
    # eager and replayed steps agree but for the attention backward's summation order
    assert abs(m.loss.item() - e.loss.item()) <= 1e-3 * abs(e.loss.item())


def test_every_gradient_has_the_same_bits_on_every_run(dgx):
    dgx.flash_set_deterministic(True)
    try:
        got = []
        for _ in range(2):
            m = make(True)
            batch(m)
            m.forward_backward()
            torch.cuda.synchronize()
            got.append({k: v.clone() for k, v in m.g.items()})
        assert all(torch.equal(got[0][k], got[1][k]) for k in got[0])
    finally:
        dgx.flash_set_deterministic(False)


def test_embedding_scale(dgx):
    a = make(True)
    # half the table at twice the scale is the same model; its table gradient doubles
    params = {k: v.cpu().clone() for k, v in a.p.items()}
    params["W_tok"] = params["W_tok"] / 2
    params["Wout"], params["bout"] = params["Wout"][:65], params["bout"][:65]
    b = make(True, params=params, embed_scale=2.0)
    batch(a)
    batch(b)
    assert a.forward_backward().item() == b.forward_backward().item()
    assert rel(b.g["W_tok"], 2 * a.g["W_tok"]) <= 1e-3  # the attention backward's order of sums


def own_logits(m):
    from dreamcompiler_b200 import gemm
    V = m.cfg.vocab
    return gemm(m.h16[-1], m.w16["Wout"], transB=True, bias=m.p["bout"])[:, :V]


def test_a_teacher_equal_to_the_student_teaches_nothing(dgx):
    m = make(True, teacher_k=65, teacher_weight=1.0, temperature=2.0)
    batch(m)
    m.forward_backward()
    z = own_logits(m)
    top = z.topk(65, dim=1)
    m.set_teacher(top.indices.to(torch.int32), top.values)
    m.forward_backward()
    dgx.sync_check()
    assert abs(m.distill_loss.item()) <= 1e-5
    hard = make(True)
    batch(hard)
    hard.forward_backward()
    assert float(m.g["Wout"].norm()) <= 2.0 ** -7 * float(hard.g["Wout"].norm())


def test_distillation_pulls_the_student_to_the_teacher(dgx):
    teacher = make(True)
    teacher.p["Wout"].mul_(40.0)
    teacher._refresh_w16()
    batch(teacher)
    teacher.forward_backward()
    top = own_logits(teacher).topk(16, dim=1)
    m = make(True, teacher_k=16, teacher_weight=0.75, temperature=2.0, lr=3e-3)
    batch(m)
    m.set_teacher(top.indices.to(torch.int32), top.values)
    losses = []
    for _ in range(40):
        m.step()
        losses.append((m.distill_loss.item(), m.loss.item()))
    dgx.sync_check()
    assert losses[-1][0] < 0.5 * losses[0][0]


@pytest.mark.parametrize("weight", [0.0, 0.25, 0.75, 1.0])
def test_the_loss_returned_is_the_one_minimised(dgx, weight):
    """(1 - a) nll + a distillation, against its parts and against the gradient of the output bias, which the two
    losses and nothing else in the step depend on linearly."""
    m = make(True, teacher_k=6, teacher_weight=weight, temperature=2.0)
    batch(m)
    n = m.cfg.batch * m.cfg.seq_len
    g = torch.Generator().manual_seed(5)
    m.set_teacher(torch.randint(0, 20, (n, 6), generator=g).to(torch.int32), 4 * torch.randn(n, 6, generator=g))
    got = m.forward_backward()
    nll, distill, loss = m.nll_loss.item(), m.distill_loss.item(), got.item()
    assert got is m.loss and nll > 1.0 and distill > 1.0
    # two products and a sum in fp32
    assert abs(loss - ((1 - weight) * nll + weight * distill)) <= 3 * 2.0 ** -24 * max(nll, distill)
    # A step h along a direction of signs: the cubic term of a log-sum-exp along it is at most h^2 / 6 (its third
    # central moment over values of +-1 is below 1, T^2 / T^3 < 1); either end's loss is a mean of rows that are
    # 1e-5 off at most and the gradient sums n rows of fp32 probabilities (1e-5 of at most 2 per row).
    h, grad = 2.0 ** -5, m.g["bout"][:65].clone()
    sign = torch.where(grad < 0, -1.0, 1.0)
    ends = []
    for step in (h, -2 * h):
        m.p["bout"][:65] += step * sign
        ends.append(m.forward_backward().item())
    slope, along = (ends[0] - ends[1]) / (2 * h), float((grad * sign).sum())
    assert along > 0.1
    assert abs(slope - along) <= h * h / 6 + 1e-5 / h + 2e-5


def test_a_loss_of_weight_zero_does_not_touch_the_gradient(dgx):
    """A masked target makes the hard loss infinite; with all weight on the teacher the step stays finite."""
    m = make(True, teacher_k=3, teacher_weight=1.0)
    batch(m)
    n = m.cfg.batch * m.cfg.seq_len
    m.p["bout"][int(m.tgt[0])] = float("-inf")
    ids = (m.tgt[0].cpu() + 1 + torch.arange(3)).remainder(65).to(torch.int32).repeat(n, 1)
    m.set_teacher(ids, torch.zeros(n, 3))
    loss = m.forward_backward().item()
    assert m.nll_loss.item() == float("inf") and loss == m.distill_loss.item() and 0 < loss < float("inf")
    assert all(torch.isfinite(v).all() for v in m.g.values())


def test_options_need_the_fused_step(dgx):
    for kw in (dict(teacher_k=4), dict(embed_scale=2.0)):
        with pytest.raises(AssertionError):
            make(False, **kw)
