"""GPU parity of token sampling against the float64 oracle.

Tokens are compared exactly.  The uniform numbers are the middles of the
oracle's intervals, and top-p lies in the middle between two of its cumulative
masses; the weights' relative error, 2^-22 + |s| 2^-24 + 2^-40, is far below
half an interval at the interval sizes that the tests take, so the expected
token is certain.  Log-probabilities within 1e-5."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_exact
from oracle import sample as orc

pytestmark = pytest.mark.gpu
dev = "cuda"


def _logits(B, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(B, V, generator=g)).to(dtype).to(dev)


def _clear_p(x, t, k, p):
    """A top-p near p that lies in the middle between two cumulative masses of row x."""
    at, pr = orc.kept(x, temperature=t, top_k=k)
    mass = np.cumsum(np.sort(pr)[::-1])
    j = int(np.searchsorted(mass, p))
    lo = mass[j - 1] if j > 0 else 0.0
    return float(np.float32((lo + mass[min(j, len(mass) - 1)]) / 2))


def _run(x, rows, seed=0, **settings):
    """Samples every row of x at several u, all at once; per-row settings as lists or numbers."""
    rng = np.random.default_rng(seed)
    xn = x.float().cpu().numpy()
    B = x.shape[0]
    per = [{k: (v[b] if isinstance(v, (list, np.ndarray)) else v) for k, v in settings.items()} for b in range(B)]
    us, want = np.zeros((rows, B), np.float32), np.zeros((rows, B), np.int64)
    lp = np.zeros((rows, B))
    for b in range(B):
        at, pr = orc.kept(xn[b], **per[b])
        cum = np.cumsum(pr)
        wide = np.flatnonzero(pr > 2e-6)
        js = np.concatenate([wide[[0, -1]], rng.choice(wide, rows)])[:rows]
        us[:, b] = cum[js] - pr[js] / 2
        want[:, b], lp[:, b] = at[js], np.log(pr[js])
    kind = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    args = {k: (torch.tensor(v, dtype=kind[k], device=dev) if isinstance(v, (list, np.ndarray)) else v) for k, v in settings.items()}
    for r in range(rows):
        tok, got = itf.sample_tokens(x, torch.tensor(us[r], device=dev), **args)
        assert tok.dtype == torch.int64 and got.dtype == torch.float32
        assert_exact(tok, want[r], "token")
        assert np.abs(got.double().cpu().numpy() - lp[r]).max() <= 1e-5


@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 31), (2, 33), (5, 1000), (2, 1025), (3, 32000), (2, 50257), (1, 131072), (2, 262147), (40, 4097)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_plain(B, V, dtype):
    _run(_logits(B, V, dtype, seed=B + V), 4)


@pytest.mark.parametrize("V", [50, 1000, 50257, 200001])
@pytest.mark.parametrize("k", [1, 2, 49, 50, 51, 999, 4000])
def test_top_k(V, k):
    _run(_logits(3, V, torch.float32, seed=V + k), 4, top_k=k, temperature=0.8)
    _run(_logits(3, V, torch.bfloat16, seed=V + k), 3, top_k=k)           # ties at the cut


@pytest.mark.parametrize("V", [3, 1000, 50257, 200001])
@pytest.mark.parametrize("p", [0.0, 0.05, 0.5, 0.9, 0.99])
def test_top_p(V, p):
    x = _logits(4, V, torch.float32, seed=V)
    ps = [_clear_p(x[b].cpu().numpy(), 0.9, 0, p) if p else 0.0 for b in range(4)]
    _run(x, 4, top_p=ps, temperature=0.9)
    _run(x, 4, top_p=[_clear_p(x[b].cpu().numpy(), 0.9, 40, p) if p else 0.0 for b in range(4)], temperature=0.9, top_k=40)


def test_top_p_with_ties():
    """Bf16 logits: hundreds of equal values at the cut, of which the lowest indices stay."""
    x = _logits(4, 20000, torch.bfloat16, seed=1, spread=1.0)
    ps = [_clear_p(x[b].float().cpu().numpy(), 1.0, 0, 0.7) for b in range(4)]
    _run(x, 6, top_p=ps)
    _run(x, 6, top_p=[_clear_p(x[b].float().cpu().numpy(), 1.0, 3000, 0.7) for b in range(4)], top_k=3000)


@pytest.mark.parametrize("V", [100, 30000, 140000])
def test_all_equal(V):
    """Every token in one place of the order: the first k of them, the first share p of them."""
    x = torch.full((2, V), 1.25, device=dev)
    _run(x, 4, top_k=37)
    p = float(np.float32((V // 3 + 0.5) / V))
    _run(x, 4, top_p=p, top_k=0) if V < 30001 else None
    u = torch.tensor([0.0, 0.9999999], device=dev)
    tok, _ = itf.sample_tokens(x, u, top_p=p)
    assert tok.tolist() == [0, V // 3]
    tok, _ = itf.sample_tokens(x, u, top_k=V // 2)
    assert tok.tolist() == [0, V // 2 - 1]


@pytest.mark.parametrize("V,spread,dtype", [(60000, 0.3, torch.float32), (60000, 1.0, torch.bfloat16), (150000, 0.05, torch.float16),
                                            (20000, 0.5, torch.float32)])
def test_cuts_among_many_close_tokens(V, spread, dtype):
    """More tokens around the cut than the list holds: flat rows, top-p alone, top-k in the thousands with and without top-p."""
    x = _logits(3, V, dtype, seed=V, spread=spread)
    xs = x.float().cpu().numpy()
    for k in (0, V // 3, V - 5):
        _run(x, 3, top_k=k, temperature=0.9)
        for p in (0.2, 0.97):
            _run(x, 3, top_p=[_clear_p(xs[b], 0.9, k, p) for b in range(3)], temperature=0.9, top_k=k, min_p=0.3 if k else 0.0)


@pytest.mark.parametrize("m", [0.01, 0.1, 0.5, 1.0, 3.0])
def test_min_p(m):
    x = _logits(3, 30000, torch.float32, seed=4)
    _run(x, 4, min_p=m)
    _run(x, 4, min_p=m, top_k=100, temperature=1.3)


def test_everything_per_row():
    B, V = 24, 33333
    rng = np.random.default_rng(3)
    x = _logits(B, V, torch.float32, seed=5, spread=3.0)
    t = np.where(rng.random(B) < 0.2, 0.0, rng.uniform(0.4, 1.5, B)).astype(np.float32)
    k = np.where(rng.random(B) < 0.4, 0, rng.integers(1, 3000, B)).astype(np.int32)
    xs = x.cpu().numpy()
    p = np.array([_clear_p(xs[b], t[b], int(k[b]), q) if t[b] > 0 and q < 0.98 else 1.0 for b, q in enumerate(rng.uniform(0.3, 1.2, B))])
    m = np.where(rng.random(B) < 0.5, 0.0, rng.uniform(0, 0.2, B)).astype(np.float32)
    _run(x, 5, temperature=t, top_k=k, top_p=p, min_p=m)


def test_greedy_and_its_ties():
    x = _logits(5, 70000, torch.bfloat16, seed=6)
    u = torch.rand(5, device=dev)
    want = x.float().cpu().numpy().argmax(1)
    for t in (0.0, -1.0, math.nan, 1e-42):
        tok, lp = itf.sample_tokens(x, u, temperature=t, top_k=5, top_p=0.3, min_p=0.1)
        assert_exact(tok, want, "greedy token")
        assert_exact(lp, np.zeros(5), "its log-probability")
    tok, _ = itf.sample_tokens(x, u, temperature=1e-30)
    assert (x.float().gather(1, tok[:, None])[:, 0] == x.float().max(1)[0]).all()


def test_masked_rows():
    """Masks of -inf, of the type's lowest value, NaN, +inf, and rows that leave one token or none."""
    V = 5000
    x = _logits(7, V, torch.float32, seed=7)
    x[0, 100:] = -math.inf
    x[1, ::2] = math.nan
    x[2] = -math.inf
    x[2, 4321] = -5.0
    x[3] = -math.inf
    x[4] = math.nan
    x[5, 100:] = torch.finfo(torch.float32).min
    x[6, [7, 9]] = math.inf
    _run(x[[0, 1, 2, 5]], 5, top_k=30)
    _run(x[[0, 1, 2, 5]], 5)
    _run(x[[0, 1, 2, 5]], 5, min_p=0.05)
    for settings in (dict(), dict(top_k=3), dict(top_p=0.5), dict(temperature=0.0), dict(min_p=0.5), dict(top_k=2, top_p=0.9, min_p=0.2)):
        tok, lp = itf.sample_tokens(x, torch.full((7,), 0.4, device=dev), **settings)
        assert tok[3] == -1 and tok[4] == -1 and lp[3] == -math.inf and lp[4] == -math.inf
        assert tok[2] == 4321 and tok[6] == 7 and 0 <= tok[5] < 100
    tok, lp = itf.sample_tokens(x[6:], torch.tensor([0.6], device=dev))
    assert tok[0] == 9 and abs(float(lp[0]) + math.log(2)) < 1e-6
    low = torch.full((1, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device=dev)
    tok, lp = itf.sample_tokens(low, torch.tensor([0.5], device=dev))
    assert tok[0] == 150


def test_ends_of_u():
    """u at and outside its range, and NaN."""
    x = _logits(1, 1000, torch.float32, seed=8).expand(6, 1000)
    at, pr = orc.kept(x[0].cpu().numpy(), top_k=20)
    tok, _ = itf.sample_tokens(x, torch.tensor([0.0, -1.0, math.nan, 1.0, 2.0, 0.99999994], device=dev), top_k=20)
    assert tok.tolist() == [at[0]] * 3 + [at[-1]] * 3


@pytest.mark.parametrize("off", [dict(top_p=math.nan), dict(top_p=1.0), dict(top_p=5.0), dict(min_p=math.nan), dict(min_p=-1.0),
                                 dict(top_k=-3), dict(top_k=10 ** 12)])
def test_settings_that_are_off(off):
    x, u = _logits(8, 3000, torch.float32, seed=9), torch.rand(8, device=dev)
    a, b = itf.sample_tokens(x, u), itf.sample_tokens(x, u, **off)
    per_row = {k: torch.full((8,), v, device=dev, dtype=torch.int64 if k == "top_k" else torch.float64) for k, v in off.items()}
    c = itf.sample_tokens(x, u, **per_row)
    for r in (b, c):
        assert_exact(r[0], a[0], "token")
        assert_exact(r[1], a[1], "log-probability")


def test_strides_offsets_and_batch_independence():
    """A row's token does not depend on its place, its alignment or its neighbours."""
    x, u = _logits(6, 33003, torch.float16, seed=10), torch.rand(6, device=dev)
    s = dict(temperature=0.7, top_k=500, top_p=0.95, min_p=0.01)
    want = itf.sample_tokens(x, u, **s)
    wide = torch.zeros(6, 40001, dtype=torch.float16, device=dev)
    wide[:, 3:33006] = x
    got = itf.sample_tokens(wide[:, 3:33006], u, **s)
    one = [itf.sample_tokens(x[b:b + 1], u[b:b + 1], **s) for b in range(6)]
    turned = itf.sample_tokens(x.t().contiguous().t(), u, **s)
    many = itf.sample_tokens(x.repeat(60, 1), u.repeat(60), **s)
    for t, l in (got, turned, (torch.cat([o[0] for o in one]), torch.cat([o[1] for o in one])), (many[0][-6:], many[1][-6:])):
        assert_exact(t, want[0], "token")
        assert_exact(l, want[1], "log-probability")
    gap = (1 << 30) + 5
    big = torch.empty(2 * gap + 33003, dtype=torch.float16, device=dev)
    far = torch.as_strided(big, (3, 33003), (gap, 1))
    far.copy_(x[:3])
    assert_exact(itf.sample_tokens(far, u[:3], **s)[0], want[0][:3], "far rows")


def test_distribution():
    """20 000 uniform numbers give the kept tokens their frequencies: chi-square of 20 cells below 60
    (its 1 - 1e-5 quantile at 19 degrees of freedom is 55)."""
    n = 20000
    x = _logits(1, 400, torch.float32, seed=11)
    at, pr = orc.kept(x[0].cpu().numpy(), top_k=20)
    u = torch.rand(n, device=dev, generator=torch.Generator(device=dev).manual_seed(5))
    tok, _ = itf.sample_tokens(x.expand(n, 400), u, top_k=20)
    counts = np.array([(tok == int(v)).sum().item() for v in at])
    assert counts.sum() == n and ((counts - n * pr) ** 2 / (n * pr)).sum() < 60


def test_empty_batch_and_stream():
    tok, lp = itf.sample_tokens(torch.zeros(0, 10, device=dev), torch.zeros(0, device=dev))
    assert tok.shape == (0,) and lp.shape == (0,)
    x, u = _logits(4, 60000, torch.float32, seed=12), torch.rand(4, device=dev)
    want = itf.sample_tokens(x, u, top_p=0.9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        got = itf.sample_tokens(late, u, top_p=0.9)
    s.synchronize()
    assert_exact(got[0], want[0], "token")


def test_refusals():
    x, u = torch.zeros(2, 50, device=dev), torch.zeros(2, device=dev)
    for args, kw, match in [((x.double(), u), {}, "float32, float16 or bfloat16"), ((x[0], u), {}, "\\(B, V\\)"), ((x, u[:1]), {}, "u has the wrong shape"),
                            ((x, u.half()), {}, "u must be"), ((x.cpu(), u), {}, "CUDA"), ((x, u), dict(top_p=u[:1]), "top_p has the wrong shape"),
                            ((x, u), dict(top_k=torch.zeros(3, dtype=torch.int32, device=dev)), "top_k"),
                            ((x, u), dict(temperature=torch.ones(2)), "temperature must be"), ((x[:, :0], u), {}, "empty vocabulary")]:
        with pytest.raises(RuntimeError, match=match):
            itf.sample_tokens(*args, **kw)
    with pytest.raises(RuntimeError, match="vocab must be"):
        itf.sample_tokens(torch.zeros(1, 4194305, device=dev, dtype=torch.float16), u[:1])
