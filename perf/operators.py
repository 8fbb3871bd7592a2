"""Timed cases of the language-model operators: the gated linear recurrence (training, prefill and one-token
decode), the distillation loss on a teacher's top logits, and sampling from given random numbers.

``run`` computes a case in plain torch (fp32 inside, rounded once at the end) or, with ``own`` set, through the
package's entry points.  ``exact`` computes the same outputs from the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ONE = float(2 ** 40)          # a token at the row's maximum weighs 2^40 in the sampler's integer sums


def listed():
    return [
        # one user's token through one narrow layer: nothing but latency
        dict(name="step_1x256_f32", op="step", B=1, D=256, dtype="f32"),
        # a serving batch's token through a wide layer
        dict(name="step_256x4096_bf16", op="step", B=256, D=4096, dtype="bf16"),
        # training on the sizes of the long-sequence configuration c1
        dict(name="train_32x2048x256_f32", op="train", B=32, L=2048, D=256, dtype="f32", packed=False),
        # training on the sizes of one block of the stack configuration c4
        dict(name="train_128x4000x256_f32", op="train", B=128, L=4000, D=256, dtype="f32", packed=False),
        # mixed-precision training on packed documents of uneven lengths, some empty, features no multiple of a warp
        dict(name="train_packed_30011x1000_bf16", op="train", B=37, L=30011, D=1000, dtype="bf16", packed=True),
        # prefill of one long prompt, continuing from a carried state
        dict(name="prefill_1x65536x2048_bf16", op="prefill", B=1, L=65536, D=2048, dtype="bf16", packed=False),
        # distillation of a short batch on full-precision logits, through autograd
        dict(name="distill_333x32000_f32", op="distill", T=333, V=32000, K=16, dtype="f32", fused=False),
        # an ordinary batch whose vocabulary leaves rows unaligned, with padding rows and short teacher lists
        dict(name="distill_4096x50257_bf16", op="distill", T=4096, V=50257, K=64, dtype="bf16", fused=False),
        # a large vocabulary: loss and gradient in one call
        dict(name="distill_8192x131072_bf16", op="distill", T=8192, V=131072, K=64, dtype="bf16", fused=True),
        # one user's token
        dict(name="sample_1x32000_f32", op="sample", B=1, V=32000, dtype="f32", masked=False),
        # a serving batch, each row with settings of its own, part of the vocabulary masked by a grammar
        dict(name="sample_64x50257_f16", op="sample", B=64, V=50257, dtype="f16", masked=True),
        # a large batch over a large vocabulary
        dict(name="sample_512x131072_bf16", op="sample", B=512, V=131072, dtype="bf16", masked=False),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    return n - 2 if n == 3 * 1024 else n


def draw(rng):
    op = rng.choice(["step", "train", "train", "prefill", "distill", "distill", "sample", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "step":
        return dict(op=op, B=_log_int(rng, 1, 256), D=_log_int(rng, 64, 4096), dtype=dtype)
    if op in ("train", "prefill"):
        d = _log_int(rng, 64, 4096)
        elements = _log_int(rng, 1 << 16, 120_000_000)
        tokens = max(1, elements // d)
        if op == "train" and rng.random() < 0.4:          # packed: L tokens in all, B documents
            tokens = min(tokens, 65536)
            return dict(op=op, B=_log_int(rng, 1, min(256, tokens + 1)), L=tokens, D=d, dtype=dtype, packed=True)
        length = _log_int(rng, 1, min(tokens, 65536))
        return dict(op=op, B=max(1, tokens // length), L=length, D=d, dtype=dtype, packed=False)
    if op == "distill":
        v = _log_int(rng, 1000, 160_000)
        t = _log_int(rng, 1, max(2, min(8192, (1_000_000_000 if dtype != "f32" else 500_000_000) // v)))
        return dict(op=op, T=t, V=v, K=_log_int(rng, 1, 128), dtype=dtype, fused=rng.random() < 0.5)
    v = _log_int(rng, 1000, 200_000)
    return dict(op=op, B=_log_int(rng, 1, min(512, 60_000_000 // v)), V=v, dtype=dtype, masked=rng.random() < 0.5)


def work(case):
    s = SIZE[case["dtype"]]
    op = case["op"]
    if op == "step":
        n = case["B"] * case["D"]
        return {"bytes": n * (4 * s + 8) + 4 * case["D"], "flops": 30 * n}
    if op in ("train", "prefill"):
        rows = case["L"] if case["packed"] else case["B"] * case["L"]
        n, states = rows * case["D"], case["B"] * case["D"]
        if op == "prefill":                               # three inputs, one output; the states in and out
            return {"bytes": 4 * s * n + 8 * states, "flops": 30 * n}
        # x, two gates and the upstream gradient in; y and three gradients out
        return {"bytes": 8 * s * n + 16 * states, "flops": 80 * n}
    if op == "distill":
        n = case["T"] * case["V"]
        return {"bytes": 2 * s * n + 12 * case["T"] * case["K"], "flops": 8 * n}
    return {"bytes": s * case["B"] * case["V"] + 40 * case["B"], "flops": 10 * case["B"] * case["V"]}


# ------------------------------------------------------------------ inputs ----
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    st = {"case": case}
    op = case["op"]
    if op in ("step", "train", "prefill"):
        d, b = case["D"], case["B"]
        # decays between 0.9 and 0.999 a step at a half-open gate: memories of ten to a thousand tokens
        sp = -2.0 / 8.0 * torch.log(0.9 + 0.099 * rand(d))
        st["lam"] = torch.log(torch.expm1(sp))
        if op == "step":
            for k in ("x", "r", "i"):
                st[k] = randn(b, d).to(dt)
            st["h"] = randn(b, d)
            return st
        shape = (case["L"], d) if case["packed"] else (b, case["L"], d)
        for k in ("x", "r", "i"):
            st[k] = randn(*shape).to(dt)
        st["h0"] = randn(b, d)
        st["cu"] = None
        if case["packed"]:                                # B documents in L tokens, cut at random; some are empty
            cuts = torch.sort(torch.randint(0, case["L"] + 1, (b - 1,), generator=g, device=DEV))[0]
            ends = torch.tensor([0, case["L"]], device=DEV)
            st["cu"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
        if op == "train":
            st["dy"] = randn(*shape).to(dt)
            st["dh"] = randn(b, d)
            for k in ("x", "r", "i", "lam", "h0"):
                st[k].requires_grad_(True)
        return st
    if op == "distill":
        t, v, k = case["T"], case["V"], case["K"]
        st["logits"] = (2.5 * randn(t, v)).to(dt)
        gap = v // k                                      # K distinct tokens a row: one in each K-th of the vocabulary
        ids = torch.arange(k, device=DEV) * gap + torch.randint(0, gap, (t, k), generator=g, device=DEV)
        st["teacher"] = 0.7 * torch.gather(st["logits"], 1, ids).float() + 1.5 * randn(t, k)
        short = torch.rand(t, 1, generator=g, device=DEV) < 0.1      # a tenth of the lists end early
        st["ids"] = torch.where(short & (torch.arange(k, device=DEV) >= (k + 1) // 2), -1, ids)
        scale = 8192.0 if dt == torch.float16 else 1.0               # half-precision training scales its loss
        st["weight"] = torch.where(rand(t) < 0.1, 0.0, scale / t)    # padding tokens weigh nothing
        if not case["fused"]:
            st["logits"].requires_grad_(True)
            st["dloss"] = 0.5 + rand(t)
        st["tau"] = 2.0
        return st
    b, v = case["B"], case["V"]
    x = 2.5 * randn(b, v)
    x.scatter_add_(1, torch.randint(0, v, (b, 8), generator=g, device=DEV), 3.0 + 6.0 * rand(b, 8))
    if case["masked"]:
        x.masked_fill_(rand(b, v) < 0.7, -math.inf)
    st["logits"] = x.to(dt)
    st["u"] = rand(b)
    st["temperature"] = torch.where(rand(b) < 0.1, 0.0, 0.6 + 0.6 * rand(b))
    st["top_k"] = torch.where(rand(b) < 0.5, 0, torch.randint(1, 200, (b,), generator=g, device=DEV)).to(torch.int32)
    st["top_p"] = torch.where(rand(b) < 0.25, 1.0, 0.8 + 0.2 * rand(b))
    st["min_p"] = torch.where(rand(b) < 0.5, 0.0, 0.1 * rand(b))
    return st


# ------------------------------------------------------------- plain forms ----
DECAY_SCALE = 8.0


def _gates(x, r, i, lam):
    """Decay, its logarithm, the gates, the input's factor and softplus(lam) of the recurrence, in fp32."""
    x, r, i = x.float(), r.float(), i.float()
    soft = torch.where(lam > 20, lam, torch.log1p(torch.exp(lam)))
    sr, si = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    u = -DECAY_SCALE * soft * sr
    a = torch.exp(u)
    m = torch.sqrt(-torch.expm1(2 * u))
    return x, sr, si, u, a, m


def _step_plain(st):
    x, sr, si, u, a, m = _gates(st["x"], st["r"], st["i"], st["lam"])
    h = a * st["h"] + m * si * x
    st["h"].copy_(h)
    return h.to(st["x"].dtype), st["h"]


def _scan(a, b):
    """h_t = a_t h_(t-1) + b_t along dim 1 by doubling: after step k every position holds the composition of the
    2^k positions up to it, so the loop has log2(L) turns."""
    k = 1
    while k < b.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _recurrence_plain(st, backward):
    packed = st["cu"] is not None
    x, r, i = (st[k].detach() for k in ("x", "r", "i"))
    lam, h0 = st["lam"].detach(), st["h0"].detach()
    if packed:
        x, r, i = x[None], r[None], i[None]
    n, d = x.shape[1], x.shape[2]
    xf, sr, si, u, a, m = _gates(x, r, i, lam)
    at = torch.arange(n, device=x.device)
    if packed:
        cu = st["cu"].long()
        doc = torch.searchsorted(cu[1:], at, right=True)            # the document of each token (empty ones have none)
        start = (at == cu[doc])[None, :, None]
        before = h0[doc][None]
        full = (cu[1:] > cu[:-1])[:, None]
        last = (cu[1:] - 1).clamp(min=0)
    else:
        start = (at == 0)[None, :, None]
        before = h0[:, None]
    a_in = torch.where(start, torch.zeros_like(a), a)               # nothing passes into a sequence's first token
    b = m * si * xf
    h = _scan(a_in, torch.where(start, b + a * before, b))
    y = h.to(x.dtype)
    h_last = torch.where(full, h[0][last], h0) if packed else h[:, -1]
    if not backward:
        return y, h_last
    dy, dh = st["dy"].float(), st["dh"]
    if packed:
        dy = dy[None].index_add(1, last, torch.where(full, dh, torch.zeros_like(dh))[None])
    else:
        dy = torch.cat([dy[:, :-1], dy[:, -1:] + dh[:, None]], 1)
    a_next = torch.cat([a_in[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(a_next.flip(1), dy.flip(1)).flip(1)
    h_prev = torch.where(start, before, torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1))
    dx = g * m * si
    di = dx * xf * (1 - si)
    slope = torch.where(m > 0, a * a / m, torch.zeros_like(m))
    du = g * (a * h_prev - slope * si * xf)
    dr = du * u * (1 - sr)
    dlam = -DECAY_SCALE * (du * sr).sum((0, 1)) / (1 + torch.exp(-lam))
    into = a * g
    if packed:
        dh0 = torch.where(full, into[0][cu[:-1].clamp(max=n - 1)], dh)
        y, dx, dr, di = y[0], dx[0], dr[0], di[0]
    else:
        dh0 = into[:, 0]
    return y, h_last, dx.to(x.dtype), dr.to(x.dtype), di.to(x.dtype), dlam, dh0


def _distill_plain(st):
    z, q, ids, w, tau = st["logits"].detach(), st["teacher"], st["ids"], st["weight"], st["tau"]
    up = st["dloss"] if "dloss" in st else torch.ones_like(w)
    there = (ids >= 0) & (ids < z.shape[1]) & (q > -math.inf)
    at = torch.where(there, ids, 0).long()
    qs = torch.where(there, q.float() / tau, -math.inf)
    top = qs.max(1, keepdim=True)[0]
    live = (top > -math.inf) & (w[:, None] != 0)
    e = torch.where(there & live, torch.exp(qs - torch.where(live, top, 0.0)), 0.0)
    total = torch.where(live, e.sum(1, keepdim=True), 1.0)
    p = e / total
    logp = qs - torch.where(live, top, 0.0) - torch.log(total)
    zs = z.float() / tau
    zmax = zs.max(1, keepdim=True)[0]
    ez = torch.exp(zs - zmax)
    zsum = ez.sum(1, keepdim=True)
    lse = zmax + torch.log(zsum)
    terms = torch.where(p > 0, p * (logp - torch.gather(zs, 1, at) + lse), 0.0)
    loss = torch.where(live[:, 0], w * tau * tau * terms.sum(1), 0.0)
    dz = (ez / zsum).scatter_add_(1, at, -p) * (up * w * tau)[:, None]
    dz = torch.where(live, dz, 0.0)
    return loss, dz.to(z.dtype)


def _sample_plain(st):
    x = st["logits"].float()
    v = x.shape[1]
    temp, k, p, least = st["temperature"], st["top_k"].long(), st["top_p"], st["min_p"]
    warm = temp > 0
    k = torch.where(warm, torch.where((k <= 0) | (k > v), v, k), 1)[:, None]      # temperature 0: the largest logit
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.max(1, keepdim=True)[0]
    s = torch.where(x == top, 0.0, (x - top) * torch.where(warm, 1 / temp, 1.0)[:, None])
    s = torch.where((x > -math.inf) & ~torch.isnan(s), s, -math.inf)
    e = torch.exp(s)
    w = (e * ONE).to(torch.int64)                                   # integer weights: sums that no order changes
    order = torch.sort(s, dim=1, descending=True, stable=True)[1]       # ties to the lowest index
    ws = torch.gather(w, 1, order)
    rank = torch.arange(v, device=x.device)[None]
    ws = torch.where(rank < k, ws, 0)
    before = torch.cumsum(ws, 1) - ws
    total = ws.sum(1, keepdim=True)
    most = torch.ceil(p.double()[:, None] * total.double()).to(torch.int64)
    keep = (rank < k) & ((before < most) | (rank == 0) | (p[:, None] >= 1))
    kept = torch.zeros_like(keep).scatter_(1, order, keep) & (e >= least[:, None].clamp(max=1.0))
    w = torch.where(kept, w, 0)
    run_up = torch.cumsum(w, 1)
    total = run_up[:, -1:]
    target = torch.minimum((st["u"].double()[:, None] * total.double()).floor().to(torch.int64), total - 1).clamp(min=0)
    token = (run_up <= target).sum(1)
    empty = total[:, 0] == 0
    token = torch.where(empty, 0, token)
    got = torch.gather(s, 1, token[:, None])[:, 0] - torch.log(total[:, 0].double() / ONE).float()
    return torch.where(empty, -1, token), torch.where(empty, -math.inf, got)


def run(state):
    op = state["case"]["op"]
    if own:
        from bc_mamba_b200 import interface as itf

        if op == "step":
            y = itf.gated_recurrence_step(state["x"], state["r"], state["i"], state["lam"], state["h"], decay_scale=DECAY_SCALE)
            return y, state["h"]
        if op in ("train", "prefill"):
            y, h_last = itf.gated_recurrence(state["x"], state["r"], state["i"], state["lam"], h0=state["h0"],
                                             cu_seqlens=state["cu"], decay_scale=DECAY_SCALE)
            if op == "prefill":
                return y, h_last
            grads = torch.autograd.grad((y, h_last), [state[k] for k in ("x", "r", "i", "lam", "h0")], (state["dy"], state["dh"]))
            return (y.detach(), h_last.detach(), *grads)
        if op == "distill":
            args = (state["logits"], state["teacher"], state["ids"])
            if state["case"]["fused"]:
                return itf.distill_topk_with_grad(*args, weight=state["weight"], temperature=state["tau"])
            loss = itf.distill_topk(*args, weight=state["weight"], temperature=state["tau"])
            return loss.detach(), torch.autograd.grad(loss, state["logits"], state["dloss"])[0]
        return itf.sample_tokens(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"])
    with torch.no_grad():
        if op == "step":
            return _step_plain(state)
        if op in ("train", "prefill"):
            return _recurrence_plain(state, op == "train")
        return _distill_plain(state) if op == "distill" else _sample_plain(state)


# ------------------------------------------------------- 64-bit definitions ----
def _exact_parts(st):
    x, r, i = (st[k].detach().double() for k in ("x", "r", "i"))
    soft = torch.nn.functional.softplus(st["lam"].detach().double())
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    u = -DECAY_SCALE * soft * sr
    return x, sr, si, u, torch.exp(u), torch.sqrt(-torch.expm1(2 * u))


def _exact_recurrence(st, backward):
    """Token by token, each sequence on its own; the gradient by the adjoint recurrence, token by token too."""
    x, sr, si, u, a, m = _exact_parts(st)
    h0 = st["h0"].detach().double()
    b = m * si * x
    cu = None if st["cu"] is None else st["cu"].tolist()
    h, h_last, prev = torch.empty_like(x), torch.empty_like(h0), torch.empty_like(x)
    if cu is None:
        now = h0
        for t in range(x.shape[1]):
            prev[:, t] = now
            now = torch.addcmul(b[:, t], a[:, t], now)
            h[:, t] = now
        h_last.copy_(now)
    else:
        for j in range(len(cu) - 1):
            now = h0[j]
            for t in range(cu[j], cu[j + 1]):
                prev[t] = now
                now = torch.addcmul(b[t], a[t], now)
                h[t] = now
            h_last[j] = now
    if not backward:
        return h, h_last
    dy, dh = st["dy"].double(), st["dh"].double()
    g, dh0 = torch.empty_like(x), torch.empty_like(h0)
    if cu is None:
        back = dh
        for t in range(x.shape[1] - 1, -1, -1):
            at = dy[:, t] + back
            g[:, t] = at
            back = a[:, t] * at
        dh0.copy_(back)
    else:
        for j in range(len(cu) - 1):
            back = dh[j]
            for t in range(cu[j + 1] - 1, cu[j] - 1, -1):
                at = dy[t] + back
                g[t] = at
                back = a[t] * at
            dh0[j] = back
    dx = g * m * si
    di = g * m * x * si * (1 - si)
    du = g * (a * prev - si * x * a.square() / m)
    dr = du * u * (1 - sr)
    dlam = (du * -DECAY_SCALE * sr).reshape(-1, x.shape[-1]).sum(0) * torch.sigmoid(st["lam"].detach().double())
    return h, h_last, dx, dr, di, dlam, dh0


def _exact_distill(st):
    """Row by row in blocks, with the library's log-softmax in float64."""
    z, tau = st["logits"].detach(), st["tau"]
    losses, grads = [], []
    for lo in range(0, z.shape[0], 1024):
        part = slice(lo, lo + 1024)
        logs = torch.log_softmax(z[part].double() / tau, 1)
        ids, w = st["ids"][part], st["weight"][part].double()
        q = st["teacher"][part].double().div(tau).masked_fill(ids < 0, -math.inf)
        logp = torch.log_softmax(q, 1)
        p = logp.exp()
        terms = p * (logp - torch.gather(logs, 1, ids.clamp(min=0)))
        losses.append(w * tau ** 2 * terms.masked_fill(ids < 0, 0).sum(1))
        up = st["dloss"][part].double() if "dloss" in st else 1.0
        soft = logs.exp_()
        soft.scatter_add_(1, ids.clamp(min=0), -p.masked_fill(ids < 0, 0))
        grads.append(soft.mul_((up * w * tau)[:, None]))
    return torch.cat(losses), torch.cat(grads)


def _exact_sample(st):
    """One row at a time: sort, cut, and walk the kept tokens in the order of their index."""
    found = []
    for x, u, t, k, p, least in zip(st["logits"].double().cpu(), st["u"].tolist(), st["temperature"].tolist(), st["top_k"].tolist(),
                                    st["top_p"].tolist(), st["min_p"].tolist()):
        if t <= 0:
            found.append(0.0)
            continue
        e = torch.exp((x - x.max()) / t)
        big, at = torch.sort(e, descending=True, stable=True)
        if k > 0:
            big, at = big[:k], at[:k]
        if p < 1:
            n = max(1, int((torch.cumsum(big, 0) - big < p * big.sum()).sum()))
            big, at = big[:n], at[:n]
        at = torch.sort(at[big >= least])[0]
        mass = torch.cumsum(e[at], 0)
        j = min(int((mass <= u * mass[-1]).sum()), len(at) - 1)
        found.append(float(torch.log(e[at[j]] / mass[-1])))
    return torch.tensor(found, dtype=torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "step":
            x, sr, si, u, a, m = _exact_parts(st)
            h = a * st["h"].double() + m * si * x
            return h, h
        if op in ("train", "prefill"):
            return _exact_recurrence(st, op == "train")
        if op == "distill":
            return _exact_distill(st)
        return None, _exact_sample(st)
