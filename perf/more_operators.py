"""Timed cases of the linear-attention block: linear attention with a decay for each head (training, prefill and the
one-token step), the norm of its output with the gate, and the residual addition with the norm of the next block.

``run`` computes a case in plain torch (fp32 inside, fp64 for the sums of the decays' logarithms, rounded once at the
end) or, with ``own`` set, through the package's entry points.  ``exact`` computes the same outputs from the
definitions in float64: the attention token by token, with the adjoint recurrence for its gradients.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # one user's token through one narrow layer whose heads share their queries and keys: nothing but latency
        dict(name="step_1x4x16x64_f32", op="step", B=1, H=4, Hk=1, N=16, P=64, dtype="f32", fixed=False),
        # a serving batch's token through a layer of 4096 features, the states of all its heads
        dict(name="step_256x64x64x64_bf16", op="step", B=256, H=64, Hk=8, N=64, P=64, dtype="bf16", fixed=False),
        # prompts of odd length and head sizes, with one constant decay for each head
        dict(name="prefill_3x1777_5x48x80_f16", op="prefill", B=3, L=1777, H=5, Hk=5, N=48, P=80, dtype="f16", packed=False,
             fixed=True),
        # prefill of one long prompt, continuing from a carried state
        dict(name="prefill_1x65536_32x64x64_bf16", op="prefill", B=1, L=65536, H=32, Hk=32, N=64, P=64, dtype="bf16",
             packed=False, fixed=False),
        # training on the sizes of the long-sequence configuration c1: 256 features, states of 16, shared queries and keys
        dict(name="train_32x2048_4x16x64_f32", op="train", B=32, L=2048, H=4, Hk=1, N=16, P=64, dtype="f32", packed=False,
             fixed=False),
        # mixed-precision training on the sizes of c2: 512 features over 4096 tokens
        dict(name="train_16x4096_8x64x64_bf16", op="train", B=16, L=4096, H=8, Hk=8, N=64, P=64, dtype="bf16", packed=False,
             fixed=False),
        # half-precision training on packed documents of uneven lengths, some empty, four heads to a query and key
        dict(name="train_packed_30011_12x128x64_f16", op="train", B=37, L=30011, H=12, Hk=3, N=128, P=64, dtype="f16",
             packed=True, fixed=False),
        # full-precision training of the gated output norm, heads of an odd size
        dict(name="gated_norm_333x1000_f32", op="gated_norm", T=333, D=1000, groups=8, dtype="f32", train=True),
        # the gated output norm on the tokens of one block of the stack configuration c4
        dict(name="gated_norm_512000x256_bf16", op="gated_norm", T=512000, D=256, groups=4, dtype="bf16", train=True),
        # the residual of a few users' tokens between two wide layers
        dict(name="add_norm_4x4096_bf16", op="add_norm", T=4, D=4096, dtype="bf16", wide=False, scaled=True, train=False),
        # half-precision training with the residual stream in full precision, rows off 16 bytes
        dict(name="add_norm_30011x1001_f16", op="add_norm", T=30011, D=1001, dtype="f16", wide=True, scaled=False, train=True),
        # mixed-precision training of a wide layer with a scale for each feature of the branch
        dict(name="add_norm_65536x2048_bf16", op="add_norm", T=65536, D=2048, dtype="bf16", wide=False, scaled=True, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "step", "prefill", "prefill", "train", "train", "train", "gated_norm", "gated_norm", "add_norm",
                     "add_norm"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("step", "prefill", "train"):
        hk = _log_int(rng, 1, 16)
        h = hk * rng.choice([1, 1, 2, 3, 4])
        n, p = _log_int(rng, 8, 128), _log_int(rng, 8, 128)
        case = dict(op=op, H=h, Hk=hk, N=n, P=p, dtype=dtype, fixed=rng.random() < 0.25)
        if op == "step":
            return dict(case, B=_log_int(rng, 1, max(2, min(256, 60_000_000 // (h * n * p)))))
        most = 250_000_000 if op == "prefill" else 60_000_000          # elements of q, k, v and y (h heads each)
        tokens = max(1, min(65536, _log_int(rng, 1 << 14, most) // (2 * h * (n + p))))
        if op == "train" and rng.random() < 0.4:                       # packed: L tokens in all, B documents
            return dict(case, B=_log_int(rng, 1, min(64, tokens + 1)), L=tokens, packed=True)
        length = _log_int(rng, 1, tokens)
        batch = max(1, min(tokens // length, 40_000_000 // (h * n * p)))
        return dict(case, B=batch, L=length, packed=False)
    wide = op == "add_norm" and rng.random() < 0.5
    d = _log_int(rng, 16, 8192)
    t = _log_int(rng, 1, max(2, min(600_000, (65_000_000 if wide or dtype == "f32" else 130_000_000) // d)))
    train = rng.random() < 0.7
    if op == "gated_norm":
        groups = rng.choice([1, 2, 4, 8])
        return dict(op=op, T=t, D=max(1, d // groups) * groups, groups=groups, dtype=dtype, train=train)
    return dict(op=op, T=t, D=d, dtype=dtype, wide=wide, scaled=rng.random() < 0.5, train=train)


def work(case):
    s = SIZE[case["dtype"]]
    op = case["op"]
    if op == "step":
        b, h, hk, n, p = (case[k] for k in ("B", "H", "Hk", "N", "P"))
        return {"bytes": b * (8 * h * n * p + s * (2 * hk * n + 2 * h * p) + 4 * h), "flops": 5 * b * h * n * p}
    if op in ("prefill", "train"):
        h, hk, n, p = (case[k] for k in ("H", "Hk", "N", "P"))
        rows = case["L"] if case["packed"] else case["B"] * case["L"]
        states = case["B"] * h * n * p
        decay = 4 * h * (1 if case["fixed"] else rows)
        # token by token: the state's decay and its outer product, its product with the query
        fwd = {"bytes": rows * s * (2 * hk * n + 2 * h * p) + decay + 8 * states, "flops": 5 * rows * h * n * p}
        if op == "prefill":
            return fwd
        # the backward reads q, k, v, dy, the decays, both states' ends and writes their gradients; five products
        return {"bytes": fwd["bytes"] + rows * s * (4 * hk * n + 3 * h * p) + 2 * decay + 12 * states,
                "flops": 18 * rows * h * n * p}
    n = case["T"] * case["D"]
    if op == "gated_norm":                                # x and gate in, out; then x, gate and dout in, dx and dgate out
        return {"bytes": n * s * (8 if case["train"] else 3) + 8 * case["D"], "flops": (30 if case["train"] else 10) * n}
    w = 4 if case["wide"] else s                          # the residual stream's own type
    fwd = n * (2 * w + 2 * s)
    if not case["train"]:
        return {"bytes": fwd, "flops": 6 * n}
    # residual, branch and both upstream gradients in; the gradients of residual and branch out
    return {"bytes": fwd + n * (3 * w + 3 * s), "flops": 20 * n}


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
    if op in ("step", "prefill", "train"):
        b, h, hk, n, p = (case[k] for k in ("B", "H", "Hk", "N", "P"))
        packed = op != "step" and case["packed"]
        shape = (b,) if op == "step" else (case["L"],) if packed else (b, case["L"])
        st["q"] = (randn(*shape, hk, n) * n ** -0.5).to(dt)
        st["k"] = randn(*shape, hk, n).to(dt)
        st["v"] = randn(*shape, h, p).to(dt)
        if case["fixed"]:                                 # memories of 32 to 512 tokens over the heads
            st["log_decay"] = -torch.exp(-math.log(32) - math.log(16) * rand(h))
        else:                                             # rates of 1 to 16, steps around 0.001 to 0.1 of the token's own
            rate = 1 + 15 * rand(h)
            bias = torch.log(torch.expm1(torch.exp(math.log(1e-3) + math.log(100) * rand(h))))
            st["log_decay"] = -rate * torch.nn.functional.softplus(randn(*shape, h) + bias)
        st["h"] = randn(b, h, n, p)
        if op == "step":
            return st
        st["cu"], st["longest"] = None, case["L"]
        if packed:                                        # B documents in L tokens, cut at random; some are empty
            cuts = torch.sort(torch.randint(0, case["L"] + 1, (b - 1,), generator=g, device=DEV))[0]
            ends = torch.tensor([0, case["L"]], device=DEV)
            st["cu"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
            st["longest"] = int((st["cu"][1:] - st["cu"][:-1]).max())      # the program that packed them knows it
        if op == "train":
            st["dy"] = randn(*shape, h, p).to(dt)
            st["dh"] = randn(b, h, n, p)
            for k in ("q", "k", "v", "log_decay", "h"):
                st[k].requires_grad_(True)
        return st
    t, d = case["T"], case["D"]
    st["weight"] = 1 + 0.2 * randn(d)
    if op == "gated_norm":
        st["x"], st["gate"] = randn(t, d).mul_(2).to(dt), randn(t, d).to(dt)
        leaves = ("x", "gate", "weight")
    else:
        st["residual"] = randn(t, d).mul_(3).to(torch.float32 if case["wide"] else dt)
        st["branch"] = randn(t, d).to(dt)
        st["scale"] = 0.5 + rand(d) if case["scaled"] else None
        leaves = ("residual", "branch", "weight") + (("scale",) if case["scaled"] else ())
        if case["train"]:
            st["dres"] = randn(t, d).to(st["residual"].dtype)
    st["leaves"] = leaves
    if case["train"]:
        st["dout"] = randn(t, d).to(dt)
        for k in leaves:
            st[k].requires_grad_(True)
    return st


# ------------------------------------------------------------- plain forms ----
def _shared(t, heads):
    """(.., Hk, N) -> (.., heads, N): head h reads query and key h // (heads / Hk)."""
    return t.repeat_interleave(heads // t.shape[-2], -2)


def _step_plain(st):
    h = st["h"].shape[1]
    q, k, v = _shared(st["q"].float(), h), _shared(st["k"].float(), h), st["v"].float()
    new = torch.exp(st["log_decay"])[..., None, None] * st["h"] + k[..., None] * v[..., None, :]
    st["h"].copy_(new)
    return (q[..., None] * new).sum(-2).to(st["v"].dtype), st["h"]


def _attention_plain(st, backward):
    """In chunks of up to 64 tokens: inside a chunk as masked products, between chunks through the states."""
    q, k, v, h0 = (st[x].detach() for x in ("q", "k", "v", "h"))
    total, heads, dt, longest = v.shape[0], v.shape[-2], v.dtype, st["longest"]
    size = max(1, min(64, longest))
    g = st["log_decay"].detach()
    fixed = g.dim() == 1
    g = g.expand(*v.shape[:-1])
    if st["cu"] is not None:                              # documents side by side, the short ones padded
        cu = st["cu"].long()
        at = cu[:-1, None] + torch.arange(longest, device=v.device)
        there = at < cu[1:, None]
        at = torch.where(there, at, 0)

        def rows(x):
            return torch.where(there.reshape(*there.shape, *[1] * (x.dim() - 1)), x[at], 0)
    else:
        def rows(x):
            return x
    nb = h0.shape[0]
    nc = max(1, -(-longest // size))

    def chunks(x):                                        # (B, L, heads, ..) -> (B, heads, chunks, size, ..)
        x = rows(x)
        x = torch.cat([x, x.new_zeros(nb, nc * size - x.shape[1], *x.shape[2:])], 1)
        return x.reshape(nb, nc, size, *x.shape[2:]).movedim(3, 1)

    def tokens(x):                                        # the way back
        x = x.movedim(1, 3).reshape(nb, nc * size, heads, *x.shape[4:])[:, :longest]
        if st["cu"] is None:
            return x
        return x.new_zeros(total, *x.shape[2:]).index_put_((at[there],), x[there])

    q, k, v = chunks(_shared(q.float(), heads)), chunks(_shared(k.float(), heads)), chunks(v.float())
    run = torch.cumsum(chunks(g.double()), -1)            # logarithms of the decay since the chunk's start
    tri = torch.ones(size, size, dtype=torch.bool, device=v.device).tril()
    between = torch.exp(torch.where(tri, run[..., :, None] - run[..., None, :], -math.inf).float())
    since, until, whole = torch.exp(run.float()), torch.exp((run[..., -1:] - run).float()), torch.exp(run[..., -1].float())
    into = (k * until[..., None]).transpose(-1, -2) @ v
    states, h = [], h0
    for c in range(nc):
        states.append(h)
        h = whole[:, :, c, None, None] * h + into[:, :, c]
    states = torch.stack(states, 2)
    scores = (q @ k.transpose(-1, -2)) * between
    y = tokens(scores @ v + since[..., None] * (q @ states)).to(dt)
    if not backward:
        return y, h
    dy, ds = chunks(st["dy"].float()), st["dh"]
    from_y = (q * since[..., None]).transpose(-1, -2) @ dy
    dstates = [None] * nc                                 # of the state after each chunk
    for c in range(nc - 1, -1, -1):
        dstates[c] = ds
        ds = whole[:, :, c, None, None] * ds + from_y[:, :, c]
    dstates = torch.stack(dstates, 2)
    dscores = dy @ v.transpose(-1, -2)
    pairs = scores * dscores                              # what the decays between token j and token i carry
    dscores = dscores * between
    far_q = since[..., None] * (dy @ states.transpose(-1, -2))
    far_k = until[..., None] * (v @ dstates.transpose(-1, -2))
    dq = dscores @ k + far_q
    dk = dscores.transpose(-1, -2) @ q + far_k
    dv = scores.transpose(-1, -2) @ dy + until[..., None] * (k @ dstates)
    # a token's decay acts on every pair that it lies between, on what enters the chunk and on what leaves it
    left = torch.cumsum(pairs, -1) - pairs
    dg = torch.where(tri, left, 0).sum(-2)
    dg = dg + (q * far_q).sum(-1).flip(-1).cumsum(-1).flip(-1)
    out = (k * far_k).sum(-1)
    dg = dg + torch.cumsum(out, -1) - out + (whole * (states * dstates).sum((-1, -2)))[..., None]
    dg = tokens(dg)
    if fixed:
        dg = dg.double().reshape(-1, heads).sum(0).float()

    def unshared(x, like):                                # gradients of shared queries and keys are summed
        return tokens(x).unflatten(-2, (like.shape[-2], -1)).sum(-2).to(dt)

    return y, h, unshared(dq, st["q"]), unshared(dk, st["k"]), tokens(dv).to(dt), dg, ds


def _rms(x):
    return torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _rms_backward(x, r, dn):
    """Gradient of x r(x) for the upstream gradient dn."""
    return r * (dn - x * (r * r * (dn * x).mean(-1, keepdim=True)))


def _gated_norm_plain(st):
    t, d = st["x"].shape
    dt, groups = st["x"].dtype, st["case"]["groups"]
    x, z, w = (st[k].detach().float().reshape(-1, groups, d // groups) for k in ("x", "gate", "weight"))
    r, sig = _rms(x), 1 / (1 + torch.exp(-z))
    n, gate = x * r, z * sig
    out = (n * w * gate).reshape(t, d).to(dt)
    if not st["case"]["train"]:
        return out
    dout = st["dout"].float().reshape(x.shape)
    dx = _rms_backward(x, r, dout * w * gate)
    dz = dout * n * w * (sig * (1 + z * (1 - sig)))
    dw = (dout * n * gate).sum(0)
    return out, dx.reshape(t, d).to(dt), dz.reshape(t, d).to(dt), dw.reshape(d)


def _add_norm_plain(st):
    w = st["weight"].detach()
    b = st["branch"].detach().float()
    s = 1.0 if st["scale"] is None else st["scale"].detach()
    v = st["residual"].detach().float() + s * b
    r = _rms(v)
    outs = v.to(st["residual"].dtype), (v * r * w).to(st["branch"].dtype)
    if not st["case"]["train"]:
        return outs
    dout = st["dout"].float()
    dv = st["dres"].float() + _rms_backward(v, r, dout * w)
    grads = dv.to(st["residual"].dtype), (s * dv).to(st["branch"].dtype), (dout * v * r).sum(0)
    return (*outs, *grads) if st["scale"] is None else (*outs, *grads, (dv * b).sum(0))


def run(state):
    op = state["case"]["op"]
    if own:
        from bc_mamba_b200 import interface as itf

        if op == "step":
            y = itf.decay_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["h"])
            return y, state["h"]
        if op in ("prefill", "train"):
            outs = itf.decay_attention(state["q"], state["k"], state["v"], state["log_decay"], h0=state["h"],
                                       cu_seqlens=state["cu"])
            if op == "prefill":
                return outs
            leaves, ups = ("q", "k", "v", "log_decay", "h"), (state["dy"], state["dh"])
        elif op == "gated_norm":
            outs = (itf.gated_norm(state["x"], state["gate"], state["weight"], groups=state["case"]["groups"], eps=EPS),)
            if not state["case"]["train"]:
                return outs[0]
            leaves, ups = state["leaves"], (state["dout"],)
        else:
            outs = itf.add_norm(state["residual"], state["branch"], state["weight"], scale=state["scale"], eps=EPS)
            if not state["case"]["train"]:
                return outs
            leaves, ups = state["leaves"], (state["dres"], state["dout"])
        grads = torch.autograd.grad(outs, [state[k] for k in leaves], ups)
        return (*(o.detach() for o in outs), *grads)
    with torch.no_grad():
        if op == "step":
            return _step_plain(state)
        if op in ("prefill", "train"):
            return _attention_plain(state, op == "train")
        return _gated_norm_plain(state) if op == "gated_norm" else _add_norm_plain(state)


# ------------------------------------------------------- 64-bit definitions ----
def _exact_sequence(q, k, v, g, state, dy=None, dstate=None):
    """(B, L, heads, ..) in float64, token by token; with dy also the adjoint recurrence, from states kept for every
    64th token.  -> y, state (B, heads, N, P), and dq, dk, dv, dg, dstate."""
    length = v.shape[1]
    a = torch.exp(g)[..., None, None]
    y, kept = torch.empty_like(v), []

    def step(t, s):
        return torch.addcmul(a[:, t] * s, k[:, t, ..., None], v[:, t, :, None])

    for t in range(length):
        if dy is not None and t % 64 == 0:
            kept.append(state)
        state = step(t, state)
        y[:, t] = torch.matmul(q[:, t, :, None], state)[..., 0, :]
    if dy is None:
        return y, state
    dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(g)
    for lo in range((length - 1) // 64 * 64, -1, -64):
        before = [kept.pop()]
        for t in range(lo, min(lo + 64, length)):
            before.append(step(t, before[-1]))
        for t in range(min(lo + 64, length) - 1, lo - 1, -1):
            after = before.pop()
            dstate = torch.addcmul(dstate, q[:, t, ..., None], dy[:, t, :, None])
            dq[:, t] = torch.matmul(after, dy[:, t, ..., None])[..., 0]
            dk[:, t] = torch.matmul(dstate, v[:, t, ..., None])[..., 0]
            dv[:, t] = torch.matmul(k[:, t, :, None], dstate)[..., 0, :]
            dstate = a[:, t] * dstate
            dg[:, t] = (dstate * before[-1]).sum((-1, -2))
    return y, state, dq, dk, dv, dg, dstate


def _exact_attention(st, backward):
    q, k, v, g, h = (st[x].detach().double() for x in ("q", "k", "v", "log_decay", "h"))
    heads, share = v.shape[-2], v.shape[-2] // q.shape[-2]
    fixed = g.dim() == 1
    g = g.expand(v.shape[:-1])
    q, k = (torch.stack([x] * share, -2).flatten(-3, -2) for x in (q, k))
    seqs = [q, k, v, g] + ([st["dy"].double()] if backward else [])
    if st["cu"] is None:
        parts = _exact_sequence(*seqs[:4], h, *((seqs[4], st["dh"].double()) if backward else ()))
    else:
        cu, parts = st["cu"].tolist(), [torch.zeros_like(x) for x in ((v, h, q, k, v, g, h) if backward else (v, h))]
        parts[1].copy_(h)
        if backward:
            parts[6].copy_(st["dh"])
        for j, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
            if lo == hi:
                continue
            one = [x[None, lo:hi] for x in seqs]
            got = _exact_sequence(*one[:4], h[j:j + 1], *((one[4], st["dh"][j:j + 1].double()) if backward else ()))
            for n, (x, r) in enumerate(zip(parts, got)):
                x[slice(j, j + 1) if n in (1, 6) else slice(lo, hi)] = r if n in (1, 6) else r[0]
    if not backward:
        return parts[0], parts[1]
    y, last, dq, dk, dv, dg, dh = parts
    dq, dk = (x.reshape(*x.shape[:-2], heads // share, share, -1).sum(-2) for x in (dq, dk))
    return y, last, dq, dk, dv, dg.flatten(0, -2).sum(0) if fixed else dg, dh


def _by_rows(parts, f, rows, whole):
    """f over blocks of rows (float64 copies of large inputs do not fit beside one another); outputs from `whole` on
    are sums over the rows."""
    outs = []
    for lo in range(0, rows, 65536):
        got = f(*(None if p is None else p[lo:lo + 65536].detach().double() for p in parts))
        outs.append(got if isinstance(got, tuple) else (got,))
    res = tuple(torch.stack(x).sum(0) if n >= whole else torch.cat(x) for n, x in enumerate(zip(*outs)))
    return res if len(res) > 1 else res[0]


def _exact_norm(case, st):
    w = st["weight"].detach().double()
    with torch.enable_grad():
        if case["op"] == "gated_norm":
            groups = case["groups"]

            def f(x, gate, dout):
                leaves = [v.requires_grad_(True) for v in (x, gate, w.clone())]
                n = x.unflatten(-1, (groups, -1))
                n = (n / (n.pow(2).mean(-1, keepdim=True) + EPS).sqrt()).flatten(-2)
                out = n * leaves[2] * torch.nn.functional.silu(gate)
                return out.detach() if dout is None else (out.detach(), *torch.autograd.grad(out, leaves, dout))

            return _by_rows([st["x"], st["gate"], st.get("dout")], f, case["T"], 3)

        def f(res, branch, dres, dout):
            leaves = [v.requires_grad_(True) for v in (res, branch, w.clone())]
            if st["scale"] is not None:
                leaves.append(st["scale"].detach().double().requires_grad_(True))
                branch = branch * leaves[3]
            v = res + branch
            out = v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * leaves[2]
            if dout is None:
                return v.detach(), out.detach()
            return (v.detach(), out.detach(), *torch.autograd.grad([v, out], leaves, [dres, dout]))

        return _by_rows([st["residual"], st["branch"], st.get("dres"), st.get("dout")], f, case["T"], 4)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "step":
            share = case["H"] // case["Hk"]
            q, k = (torch.stack([st[x].double()] * share, 2).flatten(1, 2) for x in ("q", "k"))
            h = torch.addcmul(torch.exp(st["log_decay"].double())[..., None, None] * st["h"].double(), k[..., None],
                              st["v"].double()[..., None, :])
            return torch.matmul(q[..., None, :], h)[..., 0, :], h
        if op in ("prefill", "train"):
            return _exact_attention(st, op == "train")
        return _exact_norm(case, st)
