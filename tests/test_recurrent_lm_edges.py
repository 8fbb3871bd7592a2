"""The small language model around its operators, with stand-ins for them
where no GPU is needed: a row without a token, a batch that is all padding."""
import pytest
import torch
import torch.nn.functional as F

from bc_mamba_b200 import recurrent_lm as lm


class Model:
    """Logits from an embedding alone; the token of a row that has none must not index it."""

    def __init__(self):
        self.embed = torch.randn(7, 5, generator=torch.Generator().manual_seed(0))
        self.fed = []

    def logits(self, tokens):
        return F.embedding(tokens, self.embed), [torch.zeros(tokens.shape[0], 3)]

    def step_logits(self, tokens, states):
        self.fed.append(tokens.tolist())
        return F.embedding(tokens, self.embed)


def test_generate_after_a_row_without_a_token(monkeypatch):
    """sample_tokens gives -1 for a row whose logits are all NaN or -inf: it is returned, and never embedded."""
    given = iter([[3, -1], [-1, 2], [1, -1]])

    def sample_tokens(logits, u, **settings):
        t = torch.tensor(next(given))
        return t, torch.where(t < 0, -torch.inf, -1.0)

    monkeypatch.setattr(lm.itf, "sample_tokens", sample_tokens)
    model = Model()
    tokens, logps = lm.generate(model, torch.tensor([[1, 2], [3, 4]]), torch.rand(2, 3))
    assert tokens.tolist() == [[3, -1, 1], [-1, 2, -1]]
    assert (logps == -torch.inf).tolist() == [[False, True, False], [True, False, True]]
    assert model.fed == [[3, 0], [0, 2]]


@pytest.mark.gpu
def test_generate_from_a_model_that_went_astray():
    """Parameters of NaN: no token can be taken, at any step, and the device stays usable."""
    model = lm.RecurrentLM(50, 16, 24, 1, "cuda", torch.float32, seed=1)
    with torch.no_grad():
        model.head.fill_(torch.nan)
    tokens, logps = lm.generate(model, torch.tensor([[1, 2], [3, 4]], device="cuda"), torch.rand(2, 3, device="cuda"), top_k=5)
    assert (tokens == -1).all() and (logps == -torch.inf).all()


def test_a_batch_of_padding_has_weights_of_zero(monkeypatch):
    seen = []

    def with_grad(logits, teacher_logits, teacher_ids, weight, temperature):
        seen.append(weight)
        return weight * 1.0, torch.zeros_like(logits)

    class Student:
        w = torch.ones(4, requires_grad=True)

        def logits(self, tokens, cu_seqlens=None):
            return self.w.expand(3, 4) * 1.0, []

    monkeypatch.setattr(lm.itf, "distill_topk_with_grad", with_grad)
    student = Student()
    opt = torch.optim.SGD([student.w], lr=0.1)
    loss = lm.distill_step(student, opt, None, None, None, None, torch.zeros(3))
    assert seen[0].tolist() == [0.0, 0.0, 0.0] and loss == 0 and torch.isfinite(student.w).all()
    lm.distill_step(student, opt, None, None, None, None, torch.tensor([1.0, 0.0, 3.0]))
    assert seen[1].tolist() == [0.25, 0.0, 0.75]


@pytest.mark.gpu
def test_a_batch_of_padding_leaves_the_model_whole():
    model = lm.RecurrentLM(50, 16, 24, 1, "cuda", torch.float32, seed=1)
    before = [p.detach().clone() for p in model.parameters()]
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    ids = torch.arange(12, device="cuda").reshape(6, 2)
    loss = lm.distill_step(model, opt, torch.arange(6, device="cuda"), cu, torch.zeros(6, 2, device="cuda"), ids, torch.zeros(6, device="cuda"))
    assert loss == 0 and all(torch.equal(a, b) for a, b in zip(before, model.parameters()))
