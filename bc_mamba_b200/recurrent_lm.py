"""A small language model on the gated linear recurrence, trained by
distillation from a teacher's top logits and sampled token by token.

    python -m bc_mamba_b200.recurrent_lm            # needs a CUDA device

A layer maps the residual stream to values and two gates (one projection),
mixes over time with ``interface.gated_recurrence`` and adds the projected
output back.  ``distill_step`` is one training step on packed documents,
``generate`` a prefill of prompts of one length followed by decode steps whose
state is the recurrence's (batch, dim) per layer.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import interface as itf


class RecurrentLM:
    """Parameters and passes of the model; compute in `dtype`, decays in float32."""

    def __init__(self, vocab: int, d_model: int, dim: int, layers: int, device, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        rn = lambda *s, scale: (scale * torch.randn(*s, generator=g)).to(device=device, dtype=dtype).requires_grad_(True)
        self.embed = rn(vocab, d_model, scale=1.0)
        self.head = rn(vocab, d_model, scale=d_model ** -0.5)
        self.layers = []
        for _ in range(layers):
            # decays of 0.9 to 0.999 per token at a half-open gate
            decay = 0.9 + 0.099 * torch.rand(dim, generator=g)
            lam = torch.log(torch.expm1(-0.25 * torch.log(decay))).to(device).requires_grad_(True)
            self.layers.append(dict(w_in=rn(3 * dim, d_model, scale=d_model ** -0.5), lam=lam,
                                    w_out=rn(d_model, dim, scale=dim ** -0.5)))
        self.dim, self.device = dim, torch.device(device)

    def parameters(self):
        return [self.embed, self.head] + [p for layer in self.layers for p in layer.values()]

    def logits(self, tokens, cu_seqlens=None, states=None):
        """tokens (B, L), or packed (T,) with cu_seqlens -> (logits (.., vocab), one state (B, dim) per layer)."""
        v = F.embedding(tokens, self.embed)
        out = []
        for n, layer in enumerate(self.layers):
            x, r, i = F.linear(F.rms_norm(v, v.shape[-1:]), layer["w_in"]).split(self.dim, -1)
            y, h = itf.gated_recurrence(x, r, i, layer["lam"], h0=None if states is None else states[n], cu_seqlens=cu_seqlens)
            v = v + F.linear(y, layer["w_out"])
            out.append(h)
        return F.linear(F.rms_norm(v, v.shape[-1:]), self.head), out

    @torch.no_grad()
    def step_logits(self, tokens, states):
        """One token of every sequence: tokens (B,) -> logits (B, vocab); states are updated in place."""
        v = F.embedding(tokens, self.embed)
        for layer, h in zip(self.layers, states):
            x, r, i = F.linear(F.rms_norm(v, v.shape[-1:]), layer["w_in"]).split(self.dim, -1)
            v = v + F.linear(itf.gated_recurrence_step(x, r, i, layer["lam"], h), layer["w_out"])
        return F.linear(F.rms_norm(v, v.shape[-1:]), self.head)


def distill_step(model: RecurrentLM, optimizer, tokens, cu_seqlens, teacher_logits, teacher_ids, weight, temperature: float = 2.0):
    """One training step on packed documents (T,): the teacher's K top logits and ids per token, weight (T,) with 0
    for padding (all of it: loss and gradients are 0).  The head's gradient comes from the one-call form of the loss.
    Returns the mean loss (a tensor)."""
    logits, _ = model.logits(tokens, cu_seqlens=cu_seqlens)
    total = weight.sum()
    loss, dlogits = itf.distill_topk_with_grad(logits, teacher_logits, teacher_ids, weight=weight / torch.where(total == 0, 1.0, total),
                                               temperature=temperature)
    optimizer.zero_grad(set_to_none=True)
    logits.backward(dlogits)
    optimizer.step()
    return loss.sum()


@torch.no_grad()
def generate(model: RecurrentLM, prompts, u, **settings):
    """prompts (B, L), u (B, n) uniform numbers -> tokens (B, n), their log-probabilities (B, n).  A row whose logits
    are all NaN or -inf has token -1 there (log-probability -inf); its next step takes token 0."""
    logits, states = model.logits(prompts)
    logits = logits[:, -1]
    tokens, logps = [], []
    for k in range(u.shape[1]):
        if k:
            logits = model.step_logits(tokens[-1].clamp(min=0), states)
        token, logp = itf.sample_tokens(logits, u[:, k], **settings)
        tokens.append(token)
        logps.append(logp)
    return torch.stack(tokens, 1), torch.stack(logps, 1)


def main(steps: int = 60) -> None:
    """Distils a random teacher with the student's own architecture, then samples from the student."""
    dev, vocab, k = "cuda", 1000, 16
    teacher = RecurrentLM(vocab, 64, 128, 2, dev, torch.float32, seed=1)
    student = RecurrentLM(vocab, 64, 128, 2, dev, torch.float32, seed=2)
    opt = torch.optim.AdamW(student.parameters(), lr=3e-3)
    g = torch.Generator(device=dev).manual_seed(0)
    cu = torch.tensor([0, 300, 301, 301, 1024], dtype=torch.int32, device=dev)
    for n in range(steps):
        tokens = torch.randint(0, vocab, (1024,), generator=g, device=dev)
        with torch.no_grad():
            top, ids = teacher.logits(tokens, cu_seqlens=cu)[0].float().topk(k, -1)
        loss = distill_step(student, opt, tokens, cu, top, ids, torch.ones(1024, device=dev))
        if n % 10 == 0 or n == steps - 1:
            print(f"step {n}: distillation loss {loss.item():.4f}")
    tokens, logps = generate(student, torch.randint(0, vocab, (2, 20), generator=g, device=dev),
                             torch.rand(2, 12, generator=g, device=dev), temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)
    print("sampled", tokens.tolist(), "mean log-probability", round(logps.mean().item(), 3))


if __name__ == "__main__":
    main()
