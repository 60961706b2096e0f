"""The decoder operators as they are used together: attention layers on an encoder's states, the residual stream's norm, logits, the draw; and the policy's
sampling from given random numbers."""
import math

import pytest
import torch

from tests import helpers as H

pytestmark = pytest.mark.gpu


def _layer(dt, E=64, heads=4, kv=2, kv_dim=48, seed=0):
    from rrnco_amd.models import CrossAttentionLayer
    torch.manual_seed(seed)
    m = CrossAttentionLayer(E, heads, kv, kv_dim).to("cuda", dt)
    with torch.no_grad():
        m.norm.weight.uniform_(0.5, 1.5)
    return m


def _plain_layer(m, y, h, states, mask, lens):
    """The layer in float64 from its definition."""
    a = m.attention
    d = lambda t: t.detach().double()                                             # noqa: E731
    q = (d(y) @ d(a.Wq.weight).t()).unflatten(-1, (a.num_heads, a.head_dim)).transpose(1, 2)
    k, v = ((d(states) @ d(a.Wkv.weight).t()).unflatten(-1, (2, a.num_kv_heads, a.head_dim)).unbind(2))
    k, v = (t.transpose(1, 2).repeat_interleave(a.num_heads // a.num_kv_heads, 1) for t in (k, v))
    s = q @ k.transpose(2, 3) / math.sqrt(a.head_dim)
    see = torch.ones_like(s, dtype=torch.bool)
    if mask is not None:
        see = see & mask.unsqueeze(1)
    if lens is not None:
        see = see & (torch.arange(k.shape[2], device=s.device) < lens.view(-1, 1, 1, 1))
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~see, -math.inf), -1))
    o = (p @ v).transpose(1, 2).flatten(2) @ d(a.out_proj.weight).t()
    h2 = d(h) + o
    return h2 / torch.sqrt(h2.square().mean(-1, keepdim=True) + m.eps) * d(m.norm.weight), h2


def _inputs(dt, B=3, Lq=7, Lk=40, E=64, kv_dim=48, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)             # noqa: E731
    mask = torch.rand(B, Lq, Lk, device="cuda", generator=g) < 0.6
    return r(B, Lq, E), r(B, Lk, kv_dim), mask, torch.tensor([Lk, Lk // 2, 1][:B], device="cuda")


# Each product of the layer sums E terms of its type's operands in 32 bits and rounds once; four roundings follow one another (q, k / v, attention, output), each half a
# step u of values of size one, and the norm divides by the stream's size: 16 u on values of size up to 8 covers them with room for E 2^-24
TOL = {torch.float32: 64 * 2.0 ** -24 * 8, torch.float16: 16 * 2.0 ** -11, torch.bfloat16: 16 * 2.0 ** -8}


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_layers_and_a_draw_match_their_definition(dt):
    from rrnco_amd import ops
    x, states, mask, lens = _inputs(dt)
    layers = [_layer(dt, seed=s) for s in (0, 1)]
    with torch.no_grad():
        y, h = layers[0].start(x)
        yd, hd = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5), x.double()
        for m in layers:
            yd, hd = _plain_layer(m, yd, hd, states, mask, lens)
            y, h = m(y, h, states, mask=mask, kv_lens=lens)
        assert float((y.double() - yd).abs().max()) <= TOL[dt] * 4 and float((h.double() - hd).abs().max()) <= TOL[dt] * 4
        logits = y @ torch.randn(64, 33, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dt)
        u = torch.rand(3, 7, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
        i, lp = ops.sample(logits, u, temperature=0.8, top_k=10, min_p=0.01)
        z = logits.double() / 0.8
        z = z.masked_fill(z < z.topk(10).values[..., -1:], -math.inf)
        p = torch.softmax(z, -1)
        p = torch.where(p >= 0.01 * p.amax(-1, keepdim=True), p, torch.zeros_like(p))
        c = (p / p.sum(-1, keepdim=True)).cumsum(-1)
        want = (c <= u.double().unsqueeze(-1)).sum(-1)
        assert torch.equal(i, want)
        assert float((lp.double() - torch.log(p / p.sum(-1, keepdim=True)).gather(-1, i.unsqueeze(-1)).squeeze(-1)).abs().max()) < 1e-5


def test_layer_gradients_match_autograd_of_the_definition():
    x, states, mask, lens = _inputs(torch.float32)
    m = _layer(torch.float32)
    leaves = [x.clone().requires_grad_(), states.clone().requires_grad_(), *m.parameters()]
    y, h = m.start(leaves[0])
    y, h = m(y, h, leaves[1], mask=mask, kv_lens=lens)
    gy, gh = torch.randn_like(y), torch.randn_like(h)
    got = torch.autograd.grad((y, h), leaves, (gy, gh))
    ref = [t.detach().double().requires_grad_() for t in leaves]
    import copy
    m2 = copy.deepcopy(m).double()
    for p, r in zip(m2.parameters(), ref[2:]):
        p.data = r.data
    xd, sd = ref[0], ref[1]
    a = m2.attention
    yd, hd = xd / torch.sqrt(xd.square().mean(-1, keepdim=True) + 1e-5), xd
    q = a.Wq(yd).unflatten(-1, (4, 16)).transpose(1, 2)
    k, v = (t.transpose(1, 2).repeat_interleave(2, 1) for t in a.Wkv(sd).unflatten(-1, (2, 2, 16)).unbind(2))
    s = (q @ k.transpose(2, 3) / 4.0).masked_fill(~(mask.unsqueeze(1) & (torch.arange(40, device="cuda") < lens.view(-1, 1, 1, 1))), -math.inf)
    dead = torch.isinf(s).all(-1, keepdim=True)
    p = torch.softmax(torch.where(dead, torch.zeros_like(s), s), -1) * ~dead
    h2 = hd + a.out_proj((p @ v).transpose(1, 2).flatten(2))
    y2 = h2 / torch.sqrt(h2.square().mean(-1, keepdim=True) + 1e-5) * m2.norm.weight
    want = torch.autograd.grad((y2, h2), [xd, sd, *m2.parameters()], (gy.double(), gh.double()))
    for g, w in zip(got, want):      # float32 sums of at most a few hundred terms along five products: 2^-24 x 512 of the gradient's norm
        assert float((g.double() - w).norm()) <= 512 * 2.0 ** -24 * float(w.norm()) + 1e-6


def test_one_token_steps_on_precomputed_states_equal_the_whole():
    """The serving form: keys and values once, one query at a time."""
    for dt, rel in ((torch.float32, 2e-6), (torch.bfloat16, 2.0 ** -7)):
        x, states, mask, lens = _inputs(dt, Lk=700)
        lens = torch.tensor([700, 350, 1], device="cuda")
        m = _layer(dt)
        with torch.no_grad():
            y, h = m.start(x)
            whole, _ = m(y, h, states, mask=mask, kv_lens=lens)
            cache = m.attention.precompute(states)
            steps = torch.cat([m(y[:, i:i + 1], h[:, i:i + 1], cache=cache, mask=mask[:, i:i + 1], kv_lens=lens)[0] for i in range(x.shape[1])], 1)
        # sums split differently over the states (2^-24 a term), then rounded to the type: one step of it
        assert float((whole.double() - steps.double()).abs().max()) <= rel * 2 * float(whole.double().abs().max())


@pytest.mark.parametrize("fixture", ["atsp_n20_b4_pomo", "rcvrp_n20_b4_pomo"])
def test_policy_samples_from_given_random_numbers(fixture):
    from rrnco_amd import TensorDict
    from rrnco_amd.envs import ATSPEnv, RCVRPEnv
    fx = H.load_fixture(fixture)
    atsp = fixture.startswith("atsp")
    if atsp:
        pol, env = H.make_policy(H.atsp_weights(fx), device="cuda:0"), ATSPEnv(generator_params=dict(num_loc=fx["N"]))
        inst = {k: fx[k] for k in ("locs", "distance_matrix")}
    else:
        pol, env = H.make_policy(H.rcvrp_weights(fx), env_name="rcvrp", device="cuda:0"), RCVRPEnv(generator_params=dict(num_loc=fx["N"]), check_solution=True)
        inst = H.rcvrp_instance(fx)
    inst["sample_idx"] = fx["sample_idx"]
    make = lambda: env.reset(TensorDict({k: v.cuda() for k, v in inst.items()}, batch_size=[fx["B"]]))        # noqa: E731
    S, R = fx["S"], fx["S"] * fx["B"]
    u = torch.rand(64, R, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    kw = dict(phase="test", decode_type="multistart_sampling", num_starts=S, return_actions=True, return_sum_log_likelihood=False)
    with torch.no_grad():
        a = pol(make(), env, uniforms=u, **kw)
        b = pol(make(), env, uniforms=u, **kw)
        c = pol(make(), env, uniforms=1 - u, **kw)
        assert torch.equal(a["actions"], b["actions"]) and not torch.equal(a["actions"], c["actions"])
        g = pol(make(), env, phase="test", decode_type="multistart_greedy", num_starts=S, return_actions=True)
        one = pol(make(), env, uniforms=u, min_p=1.0, **kw)                        # only the most probable node is left
        n = min(g["actions"].shape[1], one["actions"].shape[1])
        assert float((g["actions"][:, :n] == one["actions"][:, :n]).float().mean()) > 0.99
        s1 = pol(make(), env, min_p=0.05, seed=7, **kw)
        s2 = pol(make(), env, min_p=0.05, seed=7, **kw)
        assert torch.equal(s1["actions"], s2["actions"])
    with pytest.raises(ValueError):
        pol(make(), env, uniforms=u[:2], **kw)
    if atsp:                                                                      # every tour is a permutation
        assert torch.equal(a["actions"].sort(1).values, torch.arange(fx["N"], device="cuda").expand(R, -1))


def test_a_tangent_on_the_incoming_gradient_is_refused():
    import torch.autograd.forward_ad as fwAD
    from rrnco_amd import ops
    q = torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True)
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    for leaf, out in ((q, ops.cross_attention(q, q, q)), (x, ops.add_rms_norm(x)[0])):
        with fwAD.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, fwAD.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_layers_under_autocast(dt):
    """The usual mixed precision: float32 parameters and residual stream, products and attention in 16 bits.  Against the definition: beside the roundings that TOL counts, each
    of the three products rounds its two operands, ten half steps u in all, on values of size up to 4: 40 u, TOL times 4 is 64.  The parameters' gradients are
    those of the float32 layer to within the same on their norm."""
    x, states, mask, lens = _inputs(torch.float32)
    layers = [_layer(torch.float32, seed=s) for s in (0, 1)]
    gy, gh = torch.randn(3, 7, 64, device="cuda"), torch.randn(3, 7, 64, device="cuda")

    def step(cache=None):
        y, h = layers[0].start(x)
        for i, m in enumerate(layers):
            y, h = m(y, h, None if cache else states, mask=mask, kv_lens=lens, cache=cache[i] if cache else None)
        return y, h, torch.autograd.grad((y, h), [p for m in layers for p in m.parameters()], (gy, gh), allow_unused=True)
    with torch.autocast("cuda", dtype=dt):
        y, h, grads = step()
        with torch.no_grad():
            early = [m.attention.precompute(states) for m in layers]
    assert y.dtype == h.dtype == torch.float32 and all(g.dtype == torch.float32 for g in grads)
    yd, hd = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5), x.double()
    for m in layers:
        yd, hd = _plain_layer(m, yd, hd, states, mask, lens)
    assert float((y.double() - yd).abs().max()) <= TOL[dt] * 4 and float((h.double() - hd).abs().max()) <= TOL[dt] * 4
    for g, w in zip(grads, step()[2]):
        assert float((g - w).norm()) <= 64 * U16[dt] * float(w.norm())
    # keys and values made in one precision, used in the other
    with torch.no_grad():
        late = [m.attention.precompute(states) for m in layers]
        y1, h1 = layers[0](*layers[0].start(x), cache=early[0], mask=mask, kv_lens=lens)
        with torch.autocast("cuda", dtype=dt):
            y2, h2 = layers[0](*layers[0].start(x), cache=late[0], mask=mask, kv_lens=lens)
        yd, hd = _plain_layer(layers[0], x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5), x, states, mask, lens)
    for y, h in ((y1, h1), (y2, h2)):
        assert y.dtype == h.dtype == torch.float32
        assert float((y.double() - yd).abs().max()) <= TOL[dt] * 4 and float((h.double() - hd).abs().max()) <= TOL[dt] * 4


U16 = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
