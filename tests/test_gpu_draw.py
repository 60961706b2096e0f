"""rrnco_amd.ops.sample (csrc/rr_draw.hip) against the definition in 64 bits: choices have to be equal, log-probabilities within a rounding to float32.

Tolerance of logp: half a step of float32 of its value (2^-24 |logp|) plus 2^-40 for what the two 64-bit evaluations and the summation order differ by."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def _ops():
    from rrnco_amd import ops
    return ops


def reference_row(l, u, t, k, p, mp, allowed):
    """One row by sorting, numpy float64: (index, logp, kept indices)."""
    V = len(l)
    ok = allowed & ~np.isnan(l) & (l != -np.inf)
    if not ok.any():
        return 0, -math.inf, np.array([], int)
    ids = np.flatnonzero(ok)
    v = l[ids]
    top = v.max()
    if not t > 0:
        return int(ids[np.argmax(v)]), 0.0, ids[:0]
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(v == top, 0.0, (v - top) / t)
    w = np.exp(z)
    kept = np.ones(len(v), bool)
    if 0 < k < V and len(v) > k:
        kept &= v >= np.sort(v)[::-1][k - 1]
    if 0 < p < 1:
        order = np.argsort(-v[kept], kind="stable")
        vs, ws = v[kept][order], w[kept][order]
        lim = p * ws.sum()
        values, first = np.unique(-vs, return_index=True)                      # descending values, where each begins in the sorted row
        above = np.concatenate([[0.0], np.cumsum(ws)])[first]                  # the mass strictly above each
        thr = -values[above < lim].max()                                       # the smallest with less than lim strictly above it
        kept &= v >= thr
    if mp > 0:
        kept &= w >= min(mp, 1.0)
    w = np.where(kept, w, 0.0)
    cum = np.cumsum(w)
    u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    over = np.flatnonzero((cum > u * cum[-1]) & (w > 0))
    i = over[0] if len(over) else np.flatnonzero(w > 0)[-1]
    return int(ids[i]), float(z[i] - np.log(w.sum())), ids[kept]


def check(logits, u, mask=None, t=1.0, k=0, p=0.0, mp=0.0, rows=None):
    idx, lp = _ops().sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp, mask=mask)
    R, V = logits.shape
    x, un = logits.double().cpu().numpy(), u.double().cpu().numpy()
    m = np.ones((R, V), bool) if mask is None else mask.expand(R, V).cpu().numpy()
    at = lambda s, r: float(s.reshape(-1)[r]) if torch.is_tensor(s) else s         # noqa: E731
    idx, lp = idx.cpu(), lp.cpu()
    for r in rows if rows is not None else range(R):
        i, want, _ = reference_row(x[r], un[r], at(t, r), int(at(k, r)), at(p, r), at(mp, r), m[r])
        assert int(idx[r]) == i, (r, int(idx[r]), i)
        got = float(lp[r])
        assert got == want or abs(got - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -40, (r, got, want)
    return idx, lp


def make(dt, R, V, seed=0, spread=3.0, masked=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (spread * torch.randn(R, V, device="cuda", generator=g)).to(dt)
    u = torch.rand(R, device="cuda", generator=g)
    mask = None
    if masked:
        mask = torch.rand(R, V, device="cuda", generator=g) >= masked
        mask[0] = False                                                            # a row with nothing left
    return x, u, mask


SIZES = [1, 2, 20, 63, 64, 65, 100, 128, 129, 257, 512, 1000, 1024, 1025, 2048, 2049, 4097, 5003, 8192, 8200, 16384, 20001, 32768, 70000]
SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=5, t=1.3), dict(k=40), dict(p=0.9), dict(p=0.3, t=2.0), dict(mp=0.1), dict(k=40, p=0.9, mp=0.02, t=0.9), dict(t=0.0), dict(k=10 ** 6, p=1.0),
            dict(p=0.999, k=3000)]


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("V", SIZES)
def test_choices_and_log_probabilities(dt, V):
    R = 40 if V <= 1024 else 6
    for n, s in enumerate(SETTINGS):
        x, u, mask = make(dt, R, V, seed=V + n, masked=0.4 if n % 2 else 0.0)
        check(x, u, mask, **s)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [50, 700, 3000, 40000])
def test_ties_and_flat_rows(dt, V):
    """Rows of few distinct values (copies stay or go together), of one value, of two that a border separates exactly."""
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.randint(0, 4, (8, V), device="cuda", generator=g).to(dt)
    x[5], x[6], x[7] = 1.5, -2.0, 0.0
    x[6, V // 3], x[7, ::2] = 4.0, -0.0
    u = torch.rand(8, device="cuda", generator=g)
    for s in (dict(), dict(k=3), dict(k=V // 2), dict(p=0.5), dict(p=0.9, k=V - 1), dict(mp=0.3), dict(mp=1.0), dict(t=0.0)):
        check(x, u, **s)
    two = torch.zeros(4, 2, device="cuda", dtype=dt)
    check(two, torch.tensor([0.0, 0.4999, 0.5, 0.99], device="cuda"))
    check(two, torch.tensor([0.0, 0.4999, 0.5, 0.99], device="cuda"), p=0.5)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [30, 900, 2500, 30000])
def test_non_finite_logits_and_random_numbers_at_the_ends(dt, V):
    x, u, _ = make(dt, 8, V, seed=V)
    x[0, 3], x[1, 5:9], x[2] = float("nan"), -float("inf"), -float("inf")
    x[3, [4, 11]], x[4] = float("inf"), float("nan")
    x[5, : V // 2] = torch.finfo(dt).min
    x[6, 0] = -float("inf")
    u[0], u[1], u[5], u[6], u[7] = 0.0, 1.0 - 2.0 ** -24, 0.0, 0.0, float("nan")
    for s in (dict(), dict(k=4), dict(p=0.8), dict(mp=0.05), dict(t=0.0), dict(k=7, p=0.9, mp=0.01)):
        idx, lp = check(x, u, **s)
        assert int(idx[2]) == 0 and float(lp[2]) == -math.inf and int(idx[4]) == 0 and int(idx[3]) in (4, 11)
    over = torch.tensor([1.0, 5.0, -1.0, float("inf"), -float("inf"), 1.0, 1.0, 1.0], device="cuda")
    check(x, over, rows=[0, 1, 3, 5, 6, 7])


@pytest.mark.parametrize("V", [100, 1001, 12000])
def test_settings_of_each_row(V):
    R = 24 if V < 5000 else 12
    x, u, mask = make(torch.float32, R, V, seed=3, masked=0.3)
    g = torch.Generator("cuda").manual_seed(9)
    r = lambda: torch.rand(R, device="cuda", generator=g)                          # noqa: E731
    t = 0.3 + r()
    t[1], t[2], t[3] = 0.0, -1.0, float("nan")
    k = (r() * 60).int()
    k[4], k[5] = -3, 2 ** 30
    p, mp = r(), 0.2 * r()
    p[6], p[7], p[8], mp[9], mp[10] = 0.0, 1.0, 7.0, 3.0, -1.0
    check(x, u, mask, t=t, k=k, p=p, mp=mp)
    check(x, u, mask, t=t.double(), k=k.long(), p=0.8, mp=mp)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [1500, 6000, 16000, 40000, 131075])
def test_wide_kept_sets(dt, V):
    """Flat rows: the filters keep thousands of keys, the border lies in a crowded place."""
    for n, s in enumerate((dict(p=0.9), dict(p=0.5, mp=0.3), dict(p=0.99, t=0.5), dict(k=V // 3), dict(k=V // 2, p=0.7), dict(k=1500, p=0.9))):
        x, u, mask = make(dt, 4, V, seed=V + n, spread=0.7, masked=0.2)
        check(x, u, mask, **s)


def test_the_choices_follow_the_distribution():
    """2^18 draws from one row of 50 keys: every frequency within 6 standard deviations of its probability."""
    n = 1 << 18
    x = (2 * torch.randn(50, device="cuda", generator=torch.Generator("cuda").manual_seed(1))).expand(n, 50)
    u = torch.rand(n, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    idx, lp = _ops().sample(x, u, top_k=20)
    pr = torch.softmax(x[0].double().masked_fill(x[0] < x[0].topk(20).values[-1], -math.inf), 0)
    f = torch.bincount(idx, minlength=50).double() / n
    assert bool(((f - pr).abs() <= 6 * torch.sqrt(pr * (1 - pr) / n) + 1e-12).all()) and bool((f[pr == 0] == 0).all())
    assert bool(((lp.double() - torch.log(pr[idx])).abs() < 1e-6).all())


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_strides_masks_shapes_and_empty(dt):
    ops = _ops()
    for V in (90, 3001):
        x, u, _ = make(dt, 12, 2 * V + 5, seed=V)
        m = torch.rand(12, 2 * V + 5, device="cuda") < 0.6
        m[:, 7] = True
        for cut in (slice(3, 3 + V), slice(0, 2 * V, 2)):                          # rows of a wider tensor off the 16-byte grid; every second key
            check(x[:, cut], u, m[:, cut], k=30, p=0.95)
        check(x[:, :V], u, m[:1, :V], p=0.9)                                       # one mask for all rows
        check(x[:1, :V].expand(12, V), u, None, k=4)
    x = torch.randn(3, 4, 10, device="cuda").to(dt)
    u = torch.rand(3, 4, device="cuda")
    i, lp = ops.sample(x, u, mask=torch.ones(4, 10, dtype=torch.bool, device="cuda"))
    assert i.shape == lp.shape == (3, 4)
    i, lp = ops.sample(x[0, 0], u[0, 0])
    assert i.shape == ()
    i, lp = ops.sample(x[:0], u[:0])
    assert i.shape == lp.shape == (0, 4)


def test_same_choices_on_another_stream_and_in_a_graph():
    ops = _ops()

    def draw(x, u, m, long, ul):
        return [*ops.sample(x, u, top_k=30, top_p=0.9, mask=m), *ops.sample(long, ul, top_p=0.9), *ops.sample(long, ul, top_k=50)]
    x, u, m = make(torch.float32, 300, 500, seed=1, masked=0.5)
    long, ul, _ = make(torch.bfloat16, 5, 50000, seed=2)
    first = draw(x, u, m, long, ul)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(first, draw(x, u, m, long, ul)))
    torch.cuda.current_stream().wait_stream(side)
    held_in = [t.clone() for t in (x, u, m, long, ul)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = draw(*held_in)
    for i in range(4):
        nx, nu, nm = make(torch.float32, 300, 500, seed=40 + i, masked=0.5)
        nl, nul, _ = make(torch.bfloat16, 5, 50000, seed=60 + i)
        for a, b in zip(held_in, (nx, nu, nm, nl, nul)):
            a.copy_(b)
        graph.replay()
        eager = draw(nx, nu, nm, nl, nul)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), i


@pytest.mark.parametrize("R,V,s", [((1 << 25) + 5, 2, dict()), ((1 << 25) + 5, 2, dict(k=1)), ((1 << 21) + 5, 1040, dict(k=40, p=0.9))], ids=["narrow", "filtered", "wide"])
def test_more_rows_than_a_launch_holds(R, V, s):
    """Rows in front of, around and behind the border between two launches are the same as on their own, settings of each row among them."""
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.randn(R, V, device="cuda", generator=g, dtype=torch.bfloat16)
    u = torch.rand(R, device="cuda", generator=g)
    t = 0.5 + torch.rand(R, device="cuda", generator=g)
    mask = torch.rand(1, V, device="cuda", generator=g) < 0.9
    mask[0, 0] = True
    set_ = dict(top_k=s.get("k", 0), top_p=s.get("p", 0.0))
    idx, lp = _ops().sample(x, u, temperature=t, mask=mask, **set_)
    border = R & ~0xff
    for part in (slice(0, 64), slice(border - 100, R)):
        i1, l1 = _ops().sample(x[part], u[part], temperature=t[part], mask=mask, **set_)
        assert torch.equal(idx[part], i1) and torch.equal(lp[part], l1)
    tail = slice(R - 20, R)
    check(x[tail], u[tail], mask=mask, t=t[tail], **s)


def test_calls_on_two_streams_at_once():
    """Long rows (a workspace each) and short ones run against each other on two streams."""
    x, u, _ = make(torch.bfloat16, 9, 60000, seed=5)
    y, w, _ = make(torch.float32, 9, 40000, seed=6)
    ops = _ops()
    calls = [lambda: ops.sample(x, u, top_p=0.9, top_k=700), lambda: ops.sample(y, w, temperature=0.5, min_p=0.01)]
    alone = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(alone[i], r))


@pytest.mark.parametrize("R,V", [(300, 16400), (300, 32768), (513, 20001), (4100, 16500)])
def test_long_rows_in_every_number(R, V):
    """A workgroup a row and stretches of a row, and more rows than one pass over the stretches takes."""
    x, u, mask = make(torch.bfloat16, R, V, seed=V, masked=0.1)
    rows = [0, 1, 2, R // 2, R - 5, R - 4, R - 3, R - 1]
    for s in (dict(), dict(k=40, p=0.9, mp=0.01), dict(p=0.95, t=1.4)):
        check(x, u, mask=mask, rows=rows, **s)


def _wide_row(kind, V, dt, g):
    if kind == "equal":
        return torch.zeros(1, V, device="cuda", dtype=dt)
    if kind == "nearly flat":
        return (0.01 * torch.randn(1, V, device="cuda", generator=g)).to(dt)
    x = -1.0 - 19.0 * torch.rand(1, V, device="cuda", generator=g)                 # "two levels": most keys at 0, the others spread below, few to each bin
    return torch.where(torch.rand(1, V, device="cuda", generator=g) < 0.7, torch.zeros_like(x), x).to(dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1 << 19, (1 << 20) + 3, 1 << 24])
@pytest.mark.parametrize("kind,p", [("equal", 0.9), ("nearly flat", 0.9), ("two levels", 0.995)])
def test_weights_that_sum_past_half_a_million(kind, p, V, dt):
    """Flat rows so wide that their masses pass 64 bits in steps of 2^-45: top-p keeps what the definition keeps, alone and with top-k and min-p.
    A kept set that is off by n keys moves the log-probability by n / V, and the choice with it; the sums of both sides are exact to 2^-29."""
    g = torch.Generator("cuda").manual_seed(V)
    x = _wide_row(kind, V, dt, g)
    u = torch.rand(1, device="cuda", generator=g)
    check(x, u, p=p)
    if V <= 1 << 21:
        check(x, u, p=p, k=V // 2)
        check(x, 1 - u, p=p, mp=0.3, t=0.9)
        mask = torch.rand(1, V, device="cuda", generator=g) < 0.97
        check(torch.cat([x, -x]), torch.cat([u, 1 - u]), mask=mask, p=p, k=2500)
