"""rrnco_amd.ops.cross_attention (csrc/rr_xattn.hip) against the formulas in 64 bits.

Tolerances, elementwise, derived before the first run.  u = half a step of the type (fp32 2^-24, fp16 2^-11, bf16 2^-8), e = 2^-24.
  score      |ds| <= E = e (D + 8) scale sum|q k| + 4 e max|s|      (products of 16-bit inputs are exact, a sum of D terms in 32 bits, exp2's argument)
  weight     relative 2 E, rounded to the type for the product with v (u; fp16 below 2^-14: half a step 2^-25 of a largest weight of 1)
  out        sum p|v| (u16 + 2 E + e (Lk + 64)) + sub sum|v| + u |out|
  dv         sum p|do| (u16 + 2 E + e (R + 64)) + sub sum|do| + u |dv|
  ds         p (|dp - delta| 2 E + e (D + 8) sum|do v| + sum|do| T + e (D + 8) sum|do o|) + u16 |ds| + sub
             delta = sum do out is taken of the forward's stored out, which is off by up to T, the bound of `out` above (the rounding of the
             weights as much as that of the result): delta is off by sum|do| T
  dq, dk     scale sum |k| (its ds bound + e (n + 64) |ds|) + u |dq|
with u16 = u for the 16-bit types and 0 for fp32, sub = 2^-25 for fp16 and 0 otherwise, each bound doubled for second-order terms.
A stored result below 2^-14 in fp16 is rounded by up to half of that type's smallest step, 2^-25, whatever its size: + sub on every output."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E24 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _ops():
    from rrnco_amd import ops
    return ops


def _visible(B, H, Lq, Lk, mask, lens, dev):
    see = torch.ones(B, H, Lq, Lk, dtype=torch.bool, device=dev)
    if mask is not None:
        see = see & mask
    if lens is not None:
        see = see & (torch.arange(Lk, device=dev) < lens.clamp(0, Lk).view(-1, 1, 1, 1))
    return see


def reference(q, k, v, mask=None, lens=None, scale=None, do=None):
    """Formulas in float64 and the elementwise bounds above: {name: (value, tolerance)}."""
    dt, dev = q.dtype, q.device
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = H // Hk
    u, u16, sub = U[dt], (0.0 if dt == torch.float32 else U[dt]), (2.0 ** -25 if dt == torch.float16 else 0.0)
    scale = D ** -0.5 if scale is None else scale
    see = _visible(B, H, Lq, Lk, mask, lens, dev)
    qd, kd, vd = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    kd, vd = kd.repeat_interleave(G, 1), vd.repeat_interleave(G, 1)
    any_key = see.any(2, keepdim=True).transpose(2, 3)                        # keys that no query sees hold anything
    kd, vd = torch.where(any_key, kd, torch.zeros_like(kd)), torch.where(any_key, vd, torch.zeros_like(vd))
    qd = torch.where(see.any(3, keepdim=True), qd, torch.zeros_like(qd))
    s = qd @ kd.transpose(2, 3) * scale
    E = E24 * (D + 8) * scale * (qd.abs() @ kd.abs().transpose(2, 3)) + 4 * E24 * s.abs().amax().clamp(min=1.0)
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    lse = torch.where(z > 0, m + torch.log(z.clamp(min=1e-300)), torch.full_like(z, -math.inf))
    p = p / torch.where(z > 0, z, torch.ones_like(z))
    Em = E.amax(-1, keepdim=True)
    o = p @ vd
    seen_v = see.double() @ vd.abs()
    to = 2 * ((p @ vd.abs()) * (u16 + 2 * Em + E24 * (Lk + 64)) + sub * seen_v) + u * o.abs()
    out = {"out": (o, to),
           "lse": (lse.squeeze(-1), (2 * Em + 2.0 ** -22 * lse.abs().clamp(min=1.0)).squeeze(-1))}
    if do is not None:
        dod = torch.where(see.any(3, keepdim=True), do.double().transpose(1, 2), torch.zeros((), dtype=torch.float64, device=dev))
        dp = dod @ vd.transpose(2, 3)
        delta = (dod * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        eds = p * ((dp - delta).abs() * 2 * E + E24 * (D + 8) * (dod.abs() @ vd.abs().transpose(2, 3)) + (dod.abs() * (to + E24 * (D + 8) * o.abs())).sum(-1, keepdim=True)) + u16 * ds.abs() + sub * see
        grp = lambda x: x.unflatten(1, (Hk, G)).sum(2)                        # noqa: E731
        n = G * Lq
        dq, dk, dv = ds @ kd * scale, grp(ds.transpose(2, 3) @ qd) * scale, grp(p.transpose(2, 3) @ dod)
        tq = 2 * scale * ((eds + E24 * (Lk + 64) * ds.abs()) @ kd.abs()) + u * dq.abs()
        tk = 2 * scale * grp((eds + E24 * (n + 64) * ds.abs()).transpose(2, 3) @ qd.abs()) + u * dk.abs()
        tv = 2 * grp((p * (u16 + 2 * E + E24 * (n + 64)) + sub * see).transpose(2, 3) @ dod.abs()) + u * dv.abs()
        out.update(dq=(dq, tq), dk=(dk, tk), dv=(dv, tv))
    return {n: ((a, t) if n == "lse" else (a.transpose(1, 2), t.transpose(1, 2) + sub)) for n, (a, t) in out.items()}


def close(name, got, ref):
    want, tol = ref
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g = got.double()
    same_inf = torch.isinf(want) & (g == want)
    d = torch.where(same_inf, torch.zeros_like(want), (g - want).abs())
    tol = torch.where(same_inf, torch.ones_like(tol), tol + 1e-30)
    worst = (d / tol).max() if d.numel() else torch.zeros(())
    assert bool((d <= tol).all()), f"{name}: {float(worst):.3g} x the tolerance, |d| {float(d.max()):.3g}"


def make(dt, B, Lq, Lk, H, Hk, D, mask="none", seed=0, layout="plain"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)        # noqa: E731
    if layout == "policy":
        q = rn(Lq, B, H, D).permute(1, 0, 2, 3)
        c = rn(B, Lk, 3 * Hk * D)
        k, v = (c[..., i * Hk * D:(i + 1) * Hk * D].unflatten(-1, (Hk, D)) for i in (0, 1))
    elif layout == "heads_first":
        q, k, v = (rn(B, h, n, D).transpose(1, 2) for h, n in ((H, Lq), (Hk, Lk), (Hk, Lk)))
    elif layout == "odd_offset":                                              # bases off the 16-byte grid: copied by the wrapper
        q, k, v = (rn(B * n * h * D + 1)[1:].view(B, n, h, D) for h, n in ((H, Lq), (Hk, Lk), (Hk, Lk)))
    else:
        q, k, v = rn(B, Lq, H, D), rn(B, Lk, Hk, D), rn(B, Lk, Hk, D)
    m = lens = None
    r = lambda *s: torch.rand(*s, device="cuda", generator=g)                 # noqa: E731
    if mask == "rows":
        m = (r(B, Lq, Lk) < r(B, Lq, 1)) & (r(B, Lq, 1) > 0.1)
        m = m[:, None]
    elif mask == "keys":
        m = r(B, 1, 1, Lk) < 0.6
    elif mask == "heads":
        m = r(B, H, Lq, Lk) < 0.5
    elif mask == "query":                                                     # a mask of the queries alone: all keys or none
        m = r(B, 1, Lq, 1) < 0.7
    elif mask == "lens":
        lens = torch.randint(0, Lk + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        lens[0] = 0
    elif mask == "both":
        m = r(B, 1, Lq, Lk) < 0.5
        lens = torch.randint(-3, Lk + 4, (B,), device="cuda", generator=g, dtype=torch.int64)      # beyond the ends: the nearer end
    return q, k, v, m, lens, rn(B, Lq, H, D)


def run(q, k, v, m, lens, do, scale=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = _ops().cross_attention(q, k, v, mask=m, kv_lens=lens, scale=scale, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


CASES = [  # B, Lq, Lk, H, Hk, D, mask, layout
    (1, 1, 1, 1, 1, 8, "none", "plain"), (2, 1, 20, 8, 8, 16, "rows", "plain"), (3, 100, 100, 8, 8, 16, "rows", "policy"),
    (2, 101, 103, 8, 8, 16, "rows", "plain"), (1, 65, 63, 3, 3, 24, "none", "plain"), (2, 7, 129, 4, 2, 32, "lens", "plain"),
    (1, 64, 64, 2, 1, 40, "keys", "heads_first"), (2, 33, 200, 6, 2, 64, "both", "plain"), (1, 130, 257, 4, 1, 64, "heads", "policy"),
    (2, 17, 300, 2, 2, 96, "query", "plain"), (1, 200, 190, 4, 4, 128, "lens", "policy"), (2, 50, 65, 8, 1, 128, "rows", "odd_offset"),
    (1, 1, 5000, 16, 2, 128, "lens", "plain"), (3, 1, 2049, 4, 1, 64, "keys", "plain"), (2, 3, 3000, 2, 2, 16, "rows", "plain"),
    (1, 1500, 3, 2, 1, 32, "none", "plain"), (4, 300, 500, 16, 16, 64, "none", "plain"), (70, 130, 70, 4, 4, 32, "rows", "plain"),
]


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "-".join(map(str, c)))
def test_matches_the_formulas_in_64_bits(dt, c):
    B, Lq, Lk, H, Hk, D, mask, layout = c
    q, k, v, m, lens, do = make(dt, B, Lq, Lk, H, Hk, D, mask, layout=layout, seed=1 + B + Lq + Lk)
    ref = reference(q, k, v, m, lens, do=do)
    got = run(q, k, v, m, lens, do)
    for n in ("out", "lse", "dq", "dk", "dv"):
        close(n, got[n], ref[n])
    plain = _ops().cross_attention(q, k, v, mask=m, kv_lens=lens)                # without a graph: the same bits
    assert torch.equal(plain, got["out"])


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", [(2, 70, 150, 4, 2, 32), (1, 1, 1500, 4, 1, 64), (2, 5, 40, 2, 2, 128)], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_may_not_be_seen_never_shows(dt, c, bad):
    """Masked keys, keys behind kv_lens and queries that see nothing hold non-finite values: results and gradients are those without them."""
    B, Lq, Lk, H, Hk, D = c
    q, k, v, _, _, do = make(dt, B, Lq, Lk, H, Hk, D, seed=5)
    m = torch.rand(B, 1, Lq, Lk, device="cuda", generator=torch.Generator("cuda").manual_seed(3)) < 0.7
    hidden = torch.arange(Lk, device="cuda") % 7 == 3
    m = m & ~hidden
    if Lq > 1:
        m[:, :, 2] = False
    lens = torch.full((B,), Lk - 2, device="cuda", dtype=torch.int32)
    ref = reference(q, k, v, m, lens, do=do)
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    k2[:, hidden], v2[:, hidden, :, ::3] = bad, bad
    k2[:, Lk - 2:], v2[:, Lk - 2:] = bad, bad
    if Lq > 1:
        q2[:, 2], do2[:, 2, :, 1] = bad, bad
    got = run(q2, k2, v2, m, lens, do2)
    for n in ("out", "lse", "dq", "dk", "dv"):
        close(n, got[n], ref[n])


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
def test_a_visible_non_finite_value_shows_where_it_is_seen(dt):
    q, k, v, _, _, _ = make(dt, 1, 40, 90, 2, 2, 32, seed=8)
    m = torch.ones(1, 1, 40, 90, dtype=torch.bool, device="cuda")
    m[:, :, :20, 50] = False
    v = v.clone()
    clean = _ops().cross_attention(q, k, v, mask=m)
    v[0, 50, 1, 7] = float("inf")
    v[0, 50, 1, 20] = float("nan")
    got = _ops().cross_attention(q, k, v, mask=m)
    assert torch.equal(got[:, :20], clean[:, :20]) and torch.equal(got[:, :, 0], clean[:, :, 0])
    assert bool((got[0, 20:, 1, 7] == float("inf")).all()) and bool(torch.isnan(got[0, 20:, 1, 20]).all())
    rest = [d for d in range(32) if d not in (7, 20)]
    ref = reference(q, k, torch.nan_to_num(v, nan=0.0, posinf=0.0), m)["out"]
    close("rest", got[0, 20:, 1][:, rest], (ref[0][0, 20:, 1][:, rest], ref[1][0, 20:, 1][:, rest]))
    k = k.clone()
    k[0, 50, 0, 3] = float("nan")
    got = _ops().cross_attention(q, k, torch.nan_to_num(v, nan=0.0, posinf=0.0), mask=m)
    assert bool(torch.isnan(got[0, 20:, 0]).all()) and bool(torch.isfinite(got[0, :20]).all()) and bool(torch.isfinite(got[:, :, 1]).all())


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
def test_large_scores_stay_exact(dt):
    """Scores of hundreds, first rising then falling along the keys: the running maximum is carried, nothing overflows."""
    q, k, v, _, _, do = make(dt, 1, 20, 700, 2, 2, 32, seed=4)
    ramp = torch.linspace(-8, 8, 700, device="cuda").view(1, -1, 1, 1)
    for f in (ramp, -ramp):
        kk = (k.float() * 0.25 + f).to(dt)
        ref = reference(q, kk, v, do=do)
        got = run(q, kk, v, None, None, do)
        for n in ("out", "lse", "dq", "dk", "dv"):
            close(n, got[n], ref[n])


def test_empty_axes():
    ops = _ops()
    for dt in TYPES:
        z = lambda *s: torch.randn(*s, device="cuda").to(dt).requires_grad_()                      # noqa: E731
        for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
            q, k, v = z(B, Lq, 4, 16), z(B, Lk, 2, 16), z(B, Lk, 2, 16)
            out, lse = ops.cross_attention(q, k, v, return_lse=True)
            assert out.shape == (B, Lq, 4, 16) and not out.any() and lse.shape == (B, 4, Lq) and bool((lse == -math.inf).all())
            for g, t in zip(torch.autograd.grad(out.sum(), (q, k, v)), (q, k, v)):
                assert g.shape == t.shape and not g.any()


def test_gradient_against_differences():
    """Directional derivative of sum(out * do) in float32: central differences with step h have an error of h^2 f'''/6 plus 2^-24 |f| / h; with
    h = 2^-6, unit-variance inputs and sums of a few thousand terms of size one both stay under 1 % of the gradient's norm times the direction's."""
    q, k, v, m, _, do = make(torch.float32, 2, 30, 50, 4, 2, 16, "rows", seed=2)
    got = run(q, k, v, m, None, do)
    h = 2.0 ** -6
    for i, n in enumerate(("dq", "dk", "dv")):
        d = got[n] / got[n].norm()
        f = []
        for s in (h, -h):
            t = [q, k, v]
            t[i] = t[i] + s * d
            f.append((_ops().cross_attention(*t, mask=m).double() * do.double()).sum())
        diff, want = float((f[0] - f[1]) / (2 * h)), float(got[n].double().norm())
        assert abs(diff - want) < 0.01 * want, (n, diff, want)


def test_broadcast_states_and_shared_heads():
    """Encoder states expanded over the batch (stride 0): gradients of the one state are the sum over the batch."""
    q, k, v, _, _, do = make(torch.float32, 4, 20, 90, 4, 2, 16, seed=9)
    k1, v1 = k[:1].detach().requires_grad_(), v[:1].detach().requires_grad_()
    out = _ops().cross_attention(q, k1.expand(4, -1, -1, -1), v1.expand(4, -1, -1, -1))
    g1 = torch.autograd.grad(out, (k1, v1), do)
    ref = reference(q, k1.expand(4, -1, -1, -1), v1.expand(4, -1, -1, -1), do=do)
    close("out", out.detach(), ref["out"])
    for g, n in zip(g1, ("dk", "dv")):
        close(n, g, (ref[n][0].sum(0, keepdim=True), ref[n][1].sum(0, keepdim=True) * 1.5))
    s = q.detach().requires_grad_()
    _ops().cross_attention(s, k, v).sum().backward()                              # an expanded gradient
    ref = reference(q, k, v, do=torch.ones_like(do))
    close("dq", s.grad, ref["dq"])


def test_only_some_gradients_and_no_second_order():
    q, k, v, _, _, do = make(torch.float32, 1, 5, 9, 2, 1, 16, seed=3)
    full = run(q, k, v, None, None, do)
    k2 = k.detach().requires_grad_()
    (dk,) = torch.autograd.grad(_ops().cross_attention(q, k2, v), (k2,), do)
    assert torch.equal(dk, full["dk"])
    q2 = q.detach().requires_grad_()
    (dq,) = torch.autograd.grad(_ops().cross_attention(q2, k, v), (q2,), do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), (q2,))


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
def test_same_bits_every_time_on_any_stream_and_in_a_graph(dt):
    c = (2, 60, 1100, 4, 2, 64, "rows")
    q, k, v, m, lens, do = make(dt, *c, seed=6)
    first = run(q, k, v, m, lens, do)
    for _ in range(3):
        again = run(q, k, v, m, lens, do)
        assert all(torch.equal(first[n], again[n]) for n in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(q, k, v, m, lens, do)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first[n], other[n]) for n in first)
    # a captured forward and backward, replayed on changing inputs with eager work between the replays
    ql, kl, vl, dl = (t.clone() for t in (q, k, v, do))
    with torch.cuda.stream(side):
        run(ql, kl, vl, m, lens, dl)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(ql, kl, vl, m, lens, dl)
    for i in range(4):
        q2, k2, v2, _, _, do2 = make(dt, *c, seed=20 + i)
        for a, b in zip((ql, kl, vl, dl), (q2, k2, v2, do2)):
            a.copy_(b)
        graph.replay()
        eager = run(q2, k2, v2, m, lens, do2)
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], eager[n]) for n in held), i


def test_offsets_beyond_32_bits():
    """Keys of the last batch entry start behind 2^31 elements of one long cache (strides, no copy)."""
    Lk, rows = 300, 2 ** 25 + 7                                               # 2^25 rows x 64 elements x 2 bytes = 4 GB
    cache = torch.zeros(2, rows, 1, 64, device="cuda", dtype=torch.float16)
    g = torch.Generator("cuda").manual_seed(1)
    cache[:, :Lk] = torch.randn(2, Lk, 1, 64, device="cuda", generator=g).half()
    q = torch.randn(2, 3, 2, 64, device="cuda", generator=g).half()
    k = cache[:, :Lk]
    assert k.stride(0) > 2 ** 31 - 1
    got = _ops().cross_attention(q, k, k)
    close("out", got, reference(q, k, k)["out"])


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", [(2, 5, 1, 2, 2, 16, "rows"), (2, 70, 2, 4, 2, 32, "rows"), (3, 9, 3, 2, 1, 64, "heads"), (2, 40, 5, 2, 2, 128, "both"),
                               (2, 100, 64, 4, 4, 16, "both"), (3, 90, 128, 4, 2, 32, "both"), (2, 129, 192, 2, 2, 128, "both"),
                               (1, 1, 4096, 4, 2, 64, "both"), (2, 120, 60, 4, 2, 128, "rows")], ids=lambda c: "-".join(map(str, c)))
def test_masks_of_a_few_keys_and_of_whole_tiles(dt, c):
    q, k, v, m, lens, do = make(dt, *c, seed=11)
    got, ref = run(q, k, v, m, lens, do), reference(q, k, v, m, lens, do=do)
    for n in ("out", "lse", "dq", "dk", "dv"):
        close(n, got[n], ref[n])


def test_calls_on_two_streams_at_once():
    """Split forward and backward calls (workspaces of their own) run against each other, none waits for the other."""
    cases = [make(torch.bfloat16, 1, n, 6000, 4, 2, 64, "keys", seed=n) for n in (3, 70)]
    alone = [run(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(alone[i][n], r[n]) for n in r)


def test_one_tensor_in_every_place():
    """The same leaf as query, key and value: its gradient is the sum of the three."""
    x = torch.randn(2, 30, 4, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    do = torch.randn_like(x)
    parts = run(x, x, x, None, None, do)
    one = x.clone().requires_grad_()
    got, = torch.autograd.grad(_ops().cross_attention(one, one, one), (one,), do)
    want = parts["dq"].double() + parts["dk"].double() + parts["dv"].double()
    assert bool(((got.double() - want).abs() <= 2 * E24 * (parts["dq"].abs() + parts["dk"].abs() + parts["dv"].abs()).double()).all())      # two additions, each rounded once


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("B", [1, 600])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights_beside_a_large_one(dt, B, first):
    """20 000 keys of a weight of 1.47 2^-24 each beside one of weight 1 whose value is zero: the result is the small ones' sum, 1.75e-3.  One sequence: the keys are split over workgroups, 600: they are not.
    The scores are exact in the type; a weight is rounded by half a step, u, its exponent is off by 2^-24 (16 + 8 + 4) 16.25 < 3e-5, twice that in the weight, and the sums of
    20 000 equal terms in 32 bits by 2^-24 each, 1.2e-3 at the worst where all go one way, in numerator and quotient; the result is rounded by u again."""
    n = 20001
    q = torch.full((B, 1, 1, 16), 0.25, device="cuda", dtype=dt)
    k = torch.full((1, n, 1, 16), -4.0625, device="cuda", dtype=dt)              # scale 1: scores of -16.25
    v = torch.ones(1, n, 1, 16, device="cuda", dtype=dt)
    at = 0 if first else n - 1
    k[:, at], v[:, at] = 0, 0
    got = _ops().cross_attention(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), scale=1.0).double()
    w = 20000 * math.exp(-16.25)
    assert float((got / (w / (1 + w)) - 1).abs().max()) <= 2 * U[dt] + 6e-5 + 2.4e-3


def _by_norm(name, got, want, u):
    """|got - want| in the norm: the second operand's rounding and the result's, half a step u of each at the most and with no common sign, and half of the smallest step where the result lies
    below the type's normal numbers.  Everything else (sums in 32 bits, exponents) is under a hundredth of u."""
    floor = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    g = got.double()
    assert bool(torch.isfinite(g).all()), name
    err, lim = float((g - want).norm()), 2 * u * float(want.norm()) + floor * want.numel() ** 0.5
    assert err <= lim, f"{name}: {err / float(want.norm()):.3g} of its norm, {err / lim:.3g} x the tolerance"


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("lq,lk,d,fq,fk,fv,fd", [
    (64, 4099, 128, 2.0 ** -6, 16.0, 1.0, 1e-3), (300, 4099, 64, 16.0, 2.0 ** -6, 1.0, 1e-3), (40, 32768, 64, 2.0 ** -6, 16.0, 1.0, 1e-2), (64, 131072, 64, 1.0, 2.0 ** -6, 1.0, 8.0),
    (70, 300, 32, 1.0, 1.0, 1.0, 1e-4), (1, 5000, 64, 2.0 ** -6, 16.0, 1.0, 1e-3),
    (3, 2, 128, 0.25, 1.0, 8.0, 2000.0), (40, 60, 128, 0.25, 2.0, 8.0, 2000.0), (100, 500, 64, 0.25, 8.0, 8.0, 2000.0), (300, 1500, 128, 0.25, 8.0, 8.0, 2000.0), (90, 200, 16, 0.5, 2.0, 30.0, 3000.0),
])
def test_gradients_of_every_size(dt, lq, lk, d, fq, fk, fv, fd):
    """Small gradients on long states (weights and weight gradients among float16's subnormal numbers) and large ones on few (weight gradients beyond its largest, 65 504, though dq and dk fit)."""
    g = torch.Generator("cuda").manual_seed(lk)
    rn = lambda n, h, f: (f * torch.randn(1, n, h, d, device="cuda", generator=g)).to(dt)        # noqa: E731
    q, k, v, do = rn(lq, 2, fq), rn(lk, 1, fk), rn(lk, 1, fv), rn(lq, 2, fd)
    got = run(q, k, v, None, None, do)
    qd, kd, vd, dd = (t.double().transpose(1, 2) for t in (q, k, v, do))
    s = qd @ kd.transpose(2, 3).contiguous() / math.sqrt(d)
    p = torch.softmax(s, -1)
    dp = dd @ vd.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
    want = {"dq": (ds @ kd).transpose(1, 2), "dk": (ds.transpose(2, 3).contiguous() @ qd).sum(1, keepdim=True).transpose(1, 2), "dv": (p.transpose(2, 3).contiguous() @ dd).sum(1, keepdim=True).transpose(1, 2)}
    for n in ("dq", "dk", "dv"):
        if float(want[n].abs().max()) < 6e4 or dt != torch.float16:
            _by_norm(n, got[n], want[n], U[dt])


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("lk", [5, 64, 100])
def test_a_visible_key_of_weight_zero_with_an_infinite_entry(dt, lk):
    """Every query sees a key whose score is -inf (its first entry is infinite): its weight is zero, and out, lse and the other keys' dk and dv are those without the key."""
    q, k, v, _, _, do = make(dt, 1, 40, lk, 2, 1, 32, seed=lk)
    q[..., 0] = q[..., 0].abs() + 0.1
    m = torch.ones(1, 1, 40, lk, dtype=torch.bool, device="cuda")
    m[..., 3] = False
    ref = reference(q, k, v, m, do=do)
    k[0, 3, 0, 0] = -float("inf")
    got = run(q, k, v, None, None, do)
    for n in ("out", "lse", "dk", "dv"):
        close(n, got[n], ref[n])


def test_more_instances_than_a_launch_holds():
    """1 100 000 one-query instances of 8 heads (a launch holds 8 388 607 workgroups): those around the border between two launches and the last are the same as on their own."""
    B, H, D, Lk = 1_100_000, 8, 8, 2
    g = torch.Generator("cuda").manual_seed(7)
    rn = lambda n, h: torch.randn(B, n, h, D, device="cuda", generator=g, dtype=torch.float16)        # noqa: E731
    q, k, v, do = rn(1, H), rn(Lk, H), rn(Lk, H), rn(1, H)
    lens = torch.randint(0, Lk + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    m = torch.rand(B, H, 1, Lk, device="cuda", generator=g) < 0.8
    got = run(q, k, v, m, lens, do)
    border = 8388607 // H
    for part in (slice(0, 100), slice(border - 100, border + 100), slice(B - 100, B)):
        alone = run(q[part], k[part], v[part], m[part], lens[part], do[part])
        assert all(torch.equal(got[n][part], alone[n]) for n in got)
        ref = reference(q[part], k[part], v[part], m[part], lens[part], do=do[part])
        for n in ("out", "lse", "dq", "dk", "dv"):
            close(n, alone[n], ref[n])


@pytest.mark.parametrize("dt", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("lk", [5, 100])
def test_a_query_whose_scores_are_all_minus_infinity(dt, lk):
    """One query sees nothing but a key whose score is -inf: zeros, lse -inf and no part in any gradient, as one that sees no key."""
    q, k, v, _, _, do = make(dt, 1, 40, lk, 2, 1, 32, seed=lk)
    q[..., 0] = q[..., 0].abs() + 0.1
    m = torch.ones(1, 1, 40, lk, dtype=torch.bool, device="cuda")
    m[:, :, 7] = False
    without = m.clone()
    without[..., 3], m[:, :, 7, 3] = False, True
    ref = reference(q, k, v, without, do=do)
    k[0, 3, 0, 0] = -float("inf")
    got = run(q, k, v, m, None, do)
    for n in ("out", "lse", "dk", "dv"):
        close(n, got[n], ref[n])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("c", [(19, 304, 1716, 4, 4, 8, "none"), (2, 30, 213, 8, 8, 8, "none"), (12, 1, 100, 6, 2, 16, "none"), (13, 361, 348, 8, 8, 16, "rows"), (48, 3, 268, 16, 8, 40, "rows"),
                               (24, 52, 244, 16, 2, 64, "rows"), (37, 51, 1150, 4, 4, 96, "rows"), (2, 120, 60, 8, 8, 128, "none")], ids=lambda c: "-".join(map(str, c)))
def test_gradients_of_scores_lose_nothing_to_16_bits(dt, c):
    """dq and dk of 16-bit inputs are as far from 64 bits as their own rounding, and what delta costs: it is taken of the stored out, off by the roundings of the weights and of out.
    Both at the size that they have on average: a rounding is uniform in half a step, of a value anywhere in its binade, so its mean square is u^2 / 6 of the value's (the mean of 1 / m^2
    over m in 1 .. 2 is 1/2, a third of half of u^2).  With the gradients of the scores in one 16-bit piece a third such term, as large as the result's own, came in.
    Errors add in squares; 1.2 times the sum of the two covers sums of a few values (the mean of their mantissas)."""
    B, Lq, Lk, H, Hk, D, mask = c
    q, k, v, m, lens, do = make(dt, B, Lq, Lk, H, Hk, D, mask, seed=Lk)
    got = run(q, k, v, m, lens, do)
    G, scale = H // Hk, D ** -0.5
    qd, kd, vd, dd = (t.double().transpose(1, 2) for t in (q, k, v, do))
    kd, vd = kd.repeat_interleave(G, 1), vd.repeat_interleave(G, 1)
    see = _visible(B, H, Lq, Lk, m, lens, "cuda")
    p = torch.nan_to_num(torch.softmax((qd @ kd.transpose(2, 3).contiguous() * scale).masked_fill(~see, -math.inf), -1))
    dp, o = dd @ vd.transpose(2, 3).contiguous(), p @ vd
    ds = p * (dp - (dd * o).sum(-1, keepdim=True)) * scale
    back = lambda x: x.unflatten(1, (Hk, G)).sum(2)                               # noqa: E731
    want = {"dq": ds @ kd, "dk": back(ds.transpose(2, 3).contiguous() @ qd)}
    var = U[dt] ** 2 / 6
    ddelta = var * ((dd * o).square().sum(-1, keepdim=True) + (p * dp).square().sum(-1, keepdim=True))              # delta's mean square error
    of_delta = {"dq": ddelta * (p @ kd * scale).square().sum(-1, keepdim=True), "dk": back(p.square().transpose(2, 3).contiguous() @ (ddelta * (qd * scale).square()))}
    for n in want:
        err = float((got[n].double().transpose(1, 2) - want[n]).norm())
        lim = 1.2 * (var * float(want[n].square().sum()) + float(of_delta[n].sum())) ** 0.5
        assert err <= lim, f"{n}: {err / lim:.3g} x the tolerance, {err / float(want[n].norm()) / U[dt]:.3g} u"
