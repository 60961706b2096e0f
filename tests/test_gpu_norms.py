"""rrnco_amd.ops.add_rms_norm / add_rms_norm_fp8 (csrc/rr_norm.hip) against the formulas in 64 bits.

Tolerances, elementwise, derived before the first run: u = half a step of the type (fp32 2^-24, fp16 2^-11, bf16 2^-8), e = 2^-24, sub = 2^-25 for fp16 (half
of its smallest step), else 0.
  h     u |h| + e |h| + sub                                    (one 32-bit addition, one rounding)
  rstd  relative (E + 8) e                                     (a sum of E squares, a quotient, a root; the mean's error counts half)
  y     |y| ((E + 16) e + u) + e |s w| (|x| + |r|) + sub       (h cancels: its 32-bit error is e (|x| + |r|))
  dx    s (|g| + |n| mean|g n|) (3 E + 32) e + u |dx| + e |dh| + sub
  dw    sum|dy n| (E + rows + 32) e + u |dw| + sub
  scale relative (E + 20) e of the largest |y|; q: the quotient's rounding is half a step of e4m3 (2^-4 of the value, 2^-10 below 2^-6) of y / scale,
        and a quotient that is off by its own error may land on the neighbour: one more such half step is only reached on a border, counted once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E24 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def _ops():
    from rrnco_amd import ops
    return ops


def reference(x, r, w, eps, dy=None, dh=None):
    dt, E = x.dtype, x.shape[-1]
    u, sub = U[dt], (2.0 ** -25 if dt == torch.float16 else 0.0)
    xd = x.detach().double()
    rd = torch.zeros_like(xd) if r is None else r.detach().double()
    wd = torch.ones(E, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    h = xd + rd
    s = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    n, mag = h * s, xd.abs() + rd.abs()
    y = n * wd
    out = {"h": (h, (u + E24) * h.abs() + sub), "y": (y, y.abs() * ((E + 16) * E24 + u) + E24 * (s * wd).abs() * mag + sub)}
    if dy is not None:
        d = dy.double()
        g = d * wd
        dhd = torch.zeros_like(xd) if dh is None else dh.double()
        dx = dhd + s * (g - n * (g * n).mean(-1, keepdim=True))
        out["dx"] = (dx, s * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True) + s * mag * g.abs().amax(-1, keepdim=True)) * (3 * E + 32) * E24 + u * dx.abs() + E24 * dhd.abs() + sub)
        rows = x.numel() // E
        red = tuple(range(x.dim() - 1))
        dw = (d * n).sum(red)
        uw = u if w is None else U[w.dtype]
        out["dw"] = (dw, ((d * n).abs() + d.abs() * s * mag * 2).sum(red) * (E + rows + 32) * E24 + uw * dw.abs() + sub)
    return out


def close(name, got, ref):
    want, tol = ref
    assert got.shape == want.shape, (name, got.shape, want.shape)
    d = (got.double() - want).abs()
    assert bool((d <= tol + 1e-30).all()), f"{name}: {float((d / (tol + 1e-30)).max()):.3g} x the tolerance"


def make(dt, shape, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)               # noqa: E731
    return rn(*shape).to(dt), rn(*shape).to(dt), (1 + 0.3 * rn(shape[-1])), rn(*shape).to(dt), rn(*shape).to(dt)


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 16), (33, 64), (100, 128), (7, 130), (2, 3, 100), (9, 256), (6, 300), (5, 512), (3, 1000), (4, 1024), (3, 2048), (5, 4096), (2, 5000), (2, 8192),
          (3, 12001), (2, 16384), (2000, 128), (5000, 24), (1100, 520), (70, 4100)]


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formulas_in_64_bits(dt, shape):
    x, r, w, dy, dh = make(dt, shape, seed=len(shape) + shape[-1])
    w = w.to(dt)
    ref = reference(x, r, w, 1e-5, dy, dh)
    xg, rg, wg = (t.clone().requires_grad_() for t in (x, r, w))
    y, h = _ops().add_rms_norm(xg, rg, wg, eps=1e-5)
    close("y", y.detach(), ref["y"]), close("h", h.detach(), ref["h"])
    dx, dr, dw = torch.autograd.grad((y, h), (xg, rg, wg), (dy, dh))
    close("dx", dx, ref["dx"]), close("dw", dw, ref["dw"])
    assert torch.equal(dx, dr)
    y2, h2 = _ops().add_rms_norm(x, r, w, eps=1e-5)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(100, 128), (31, 77), (4, 2048)], ids=str)
def test_without_residual_or_weight_or_one_of_the_gradients(dt, shape):
    ops = _ops()
    x, r, w, dy, dh = make(dt, shape, seed=4)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()                 # a float32 weight beside 16-bit rows
    y, h = ops.add_rms_norm(xg, None, wg, eps=1e-6)
    assert h is xg
    ref = reference(x, None, w, 1e-6, dy)
    close("y", y.detach(), ref["y"])
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    close("dx", dx, ref["dx"]), close("dw", dw, ref["dw"])
    assert dw.dtype == torch.float32
    xg, rg = x.clone().requires_grad_(), r.clone().requires_grad_()
    y, h = ops.add_rms_norm(xg, rg)                                                # no weight
    ref = reference(x, r, None, 1e-5, dy, dh)
    close("y", y.detach(), ref["y"])
    (dr,) = torch.autograd.grad((y, h), (rg,), (dy, dh))
    close("dx", dr, ref["dx"])
    y, h = ops.add_rms_norm(xg, rg, w)
    (dx,) = torch.autograd.grad(h, (xg,), dh)                                      # only the sum is used
    assert torch.equal(dx, dh)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_strides_offsets_and_empty(dt):
    ops = _ops()
    x, r, w, dy, dh = make(dt, (40, 256), seed=6)
    w = w.to(dt)
    for cut in (slice(0, 128), slice(3, 131), slice(1, 256, 2)):                   # rows of a wider tensor, off the 16-byte grid, every second column
        ref = reference(x[:, cut], r[:, cut], w[cut], 1e-5)
        y, h = ops.add_rms_norm(x[:, cut], r[:, cut], w[cut])
        close("y", y, ref["y"]), close("h", h, ref["h"])
    one = r[:1].expand(40, 256)                                                    # one residual row for all
    ref = reference(x, one, w, 1e-5)
    close("y", ops.add_rms_norm(x, one, w)[0], ref["y"])
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, _ = ops.add_rms_norm(xg, r, wg)
    y.sum().backward()                                                             # an expanded gradient
    ref = reference(x, r, w, 1e-5, torch.ones_like(x))
    close("dx", xg.grad, ref["dx"]), close("dw", wg.grad, ref["dw"])
    e = torch.empty(0, 64, device="cuda", dtype=dt).requires_grad_()
    wg = w[:64].clone().requires_grad_()
    y, h = ops.add_rms_norm(e, e, wg)
    assert y.shape == (0, 64)
    assert not torch.autograd.grad(y.sum(), (wg,))[0].any()


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_rows_of_zeros_and_extreme_rows(dt):
    x = torch.zeros(6, 128, device="cuda", dtype=dt)
    x[1], x[2, 5], x[3] = 1e-4, float("nan"), 3e4
    w = torch.ones(128, device="cuda", dtype=dt)
    y, h = _ops().add_rms_norm(x, torch.zeros_like(x), w)
    assert not y[0].any() and bool(torch.isnan(y[2]).all()) and bool(torch.isfinite(y[[0, 1, 3, 4, 5]]).all())
    close("y", y[[0, 1, 3]], tuple(t[[0, 1, 3]] for t in reference(x, None, w, 1e-5)["y"]))


def test_gradient_against_differences():
    """Central differences along the gradient in float32, step 2^-6: truncation h^2 f'''/6 and rounding 2^-24 |f| / h both stay under 1 %."""
    x, r, w, dy, dh = make(torch.float32, (30, 96), seed=2)
    args = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = _ops().add_rms_norm(*args)
    grads = torch.autograd.grad((y, h), args, (dy, dh))
    step = 2.0 ** -6
    for i, g in enumerate(grads):
        f = []
        for s in (step, -step):
            t = [x, r, w]
            t[i] = t[i] + s * g / g.norm()
            a, b = _ops().add_rms_norm(*t)
            f.append((a.double() * dy.double()).sum() + (b.double() * dh.double()).sum())
        assert abs(float((f[0] - f[1]) / (2 * step)) - float(g.norm())) < 0.01 * float(g.norm())


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_same_bits_every_time_and_in_a_graph(dt):
    ops = _ops()

    def step(x, r, w, dy, dh):
        a = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = ops.add_rms_norm(*a)
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), a, (dy, dh)), *ops.add_rms_norm_fp8(x, r, w)]
    args = [t if t.dim() > 1 else t.to(dt) for t in make(dt, (3000, 136), seed=1)]
    first = step(*args)
    same = lambda p, q: all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(p, q))      # noqa: E731
    assert all(same(first, step(*args)) for _ in range(3))
    held_in = [t.clone() for t in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert same(first, step(*held_in))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*held_in)
    for i in range(4):
        new = [t if t.dim() > 1 else t.to(dt) for t in make(dt, (3000, 136), seed=30 + i)]
        for a, b in zip(held_in, new):
            a.copy_(b)
        graph.replay()
        eager = step(*new)
        torch.cuda.synchronize()
        assert same(held, eager), i


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (3, 64), (40, 128), (7, 129), (9, 300), (5, 512), (2, 3, 1000), (3, 4096), (2, 5003), (2, 16384)], ids=str)
def test_eight_bit_form(dt, shape):
    x, r, w, _, _ = make(dt, shape, seed=shape[-1])
    w = w.to(dt)
    x[..., : shape[-1] // 3] = 0 if shape[-1] >= 500 else x[..., : shape[-1] // 3]      # a group of zeros
    r[..., : shape[-1] // 3] = 0 if shape[-1] >= 500 else r[..., : shape[-1] // 3]
    q, scale, h = _ops().add_rms_norm_fp8(x, r, w)
    E, G = shape[-1], (shape[-1] + 127) // 128
    ref = reference(x, r, w, 1e-5)
    close("h", h, ref["h"])
    y, ty = ref["y"]
    ty = ty - U[dt] * y.abs()                                                           # y is not rounded to the type here
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (*shape[:-1], G) and scale.dtype == torch.float32
    for i in range(G):
        yi, si, qi, ti = (t[..., 128 * i:128 * (i + 1)] for t in (y, y, q.double(), ty))
        top = yi.abs().amax(-1)
        want = torch.where(top == 0, torch.ones_like(top), top / 448)
        assert bool(((scale[..., i].double() - want).abs() <= ti.amax(-1) / 448 + want * 4 * E24).all())
        z = yi / scale[..., i:i + 1].double()
        err = torch.maximum(z.abs() * 2.0 ** -4, torch.full_like(z, 2.0 ** -10)) * 2 + ti / scale[..., i:i + 1].double()
        assert bool(((qi - z).abs() <= err).all())
        half = torch.maximum(z.abs() * 2.0 ** -4, torch.full_like(z, 2.0 ** -10)) + ti / scale[..., i:i + 1].double()
        assert float(((qi - z).abs() <= half).float().mean()) > 0.999
    if E >= 500:
        assert not q.double()[..., :128].any() and bool((scale[..., 0] == 1).all())
    same_h = _ops().add_rms_norm(x, r, w)[1]
    assert torch.equal(h, same_h)


@pytest.mark.parametrize("E", [24, 128, 300, 5000])
@pytest.mark.parametrize("dt,big,eps", [(torch.float32, 1e25, 1e-5), (torch.bfloat16, 1e25, 1e-5), (torch.float32, 1e-25, 0.0), (torch.bfloat16, 1e-25, 0.0), (torch.float16, 6e4, 1e-5)])
def test_rows_whose_squares_leave_32_bits(dt, big, eps, E):
    """The elements' squares overflow, or vanish, in 32 bits; the norm does not.  Tolerances as above: the power of two that the sum is taken with is exact."""
    g = torch.Generator("cuda").manual_seed(E)
    x = (big * (0.5 + 0.5 * torch.rand(5, E, device="cuda", generator=g))).to(dt).requires_grad_()
    w = torch.randn(E, device="cuda", generator=g).to(dt).requires_grad_()
    dy = torch.randn(5, E, device="cuda", generator=g).to(dt)
    ref = reference(x, None, w, eps, dy)
    y, _ = _ops().add_rms_norm(x, None, w, eps)
    close("y", y.detach(), tuple(t.detach() for t in ref["y"]))
    dw, = torch.autograd.grad(y, (w,), dy)
    close("dw", dw, tuple(t.detach() for t in ref["dw"]))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_eight_bit_groups_of_tiny_values(dt):
    """y of 2^-131 .. 0 in a group: its 448th part has no finite reciprocal, the scale is 2^-126 and nothing becomes NaN.
    y / scale is sqrt(2) 2^-5 here: with three bits behind the leading one its step is 2^-8, half of it 2^-9 (the first bound written here took e4m3's smallest
    step, 2^-9, which holds below 2^-5 only); 2^-22 more for y's own error, a step of the subnormal numbers, 2^-149, over 2^-126."""
    x = torch.ones(3, 256, device="cuda", dtype=dt)
    x[:, ::2] = 0.0
    w = torch.full((256,), 2.0 ** -131, device="cuda", dtype=torch.float32)
    w[128:] = 1.0
    q, scale, _ = _ops().add_rms_norm_fp8(x, None, w)
    y = reference(x, None, w, 1e-5)["y"][0]
    assert bool((scale[:, 0] == 2.0 ** -126).all())
    z = y[:, :128] / 2.0 ** -126
    assert bool(((q.double()[:, :128] - z).abs() <= 2.0 ** -9 + 2.0 ** -22).all())
    assert not q.double()[:, ::2].any()


@pytest.mark.parametrize("rows,E", [((1 << 25) + 3, 2), ((1 << 21) + 5, 136)], ids=["narrow", "wide"])
def test_more_rows_than_a_launch_holds(rows, E):
    """Rows in front of, around and behind the border between two launches are the same as on their own."""
    g = torch.Generator("cuda").manual_seed(E)
    x = torch.randn(rows, E, device="cuda", generator=g, dtype=torch.bfloat16)
    w = torch.randn(E, device="cuda", generator=g)
    one = x[7:8].expand(rows, E)                                                  # (a residual of stride 0)
    y, h = _ops().add_rms_norm(x, one, w)
    q, scale, h8 = _ops().add_rms_norm_fp8(x, one, w)
    border = rows & ~0xff
    for part in (slice(0, 64), slice(border - 100, rows)):
        y1, h1 = _ops().add_rms_norm(x[part], one[part], w)
        q1, s1, _ = _ops().add_rms_norm_fp8(x[part], one[part], w)
        assert torch.equal(y[part], y1) and torch.equal(h[part], h1) and torch.equal(h8[part], h1)
        assert torch.equal(q[part].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(scale[part], s1)
    ref = reference(x[-50:], one[-50:], w, 1e-5)
    close("y", y[-50:], ref["y"])
    xg, wg = x[:rows].requires_grad_(), w.clone().requires_grad_()
    dx, = torch.autograd.grad(_ops().add_rms_norm(xg, one, wg)[0], (xg,), h)
    ref = reference(x[-50:], one[-50:], w, 1e-5, h[-50:])
    close("dx", dx[-50:], tuple(t.detach() for t in ref["dx"]))
