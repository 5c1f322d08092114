"""SodAdamW (moments in 32 and in 8 bits) and grad_norm on the CPU: against
their definitions in 64 bits, torch's own AdamW, and what they refuse."""

import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from adamw_oracle import check, decode64, level, param_bound, step64
from sodkit.config import make_config
from sodkit.engine import Solver
from sodkit.ops import SodAdamW, SodSGD, grad_norm, reference
from sodkit.parallel import GradReducer

HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, wd=0.1)


def make(n, dtype=torch.float32, bits=32, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(n, generator=g).to(dtype))
    opt = SodAdamW([{"params": [p], "weight_decay": HYPER["wd"]}],
                   betas=HYPER["betas"], eps=HYPER["eps"], state_bits=bits,
                   seed=5, **kw)
    return p, opt, g


@pytest.mark.parametrize("n", [1, 3, 255, 256, 257, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_step_against_64_bits(n, dtype):
    p, opt, gen = make(n, dtype)
    st = opt.state[p]
    for t in range(1, 4):
        p.grad = (torch.randn(n, generator=gen) * 10.0 ** (t - 2)).to(dtype)
        w = st["master"] if "master" in st else p.detach()
        w1, m1, v1, em, ev, ew = step64(
            w.double(), p.grad.double(), st["exp_avg"].double(),
            st["exp_avg_sq"].double(), t, gs=0.25, **HYPER)
        opt.step(HYPER["lr"], 0.25)
        check(st["exp_avg"], m1, em, "m")
        check(st["exp_avg_sq"], v1, ev, "v")
        if "master" in st:
            check(st["master"], w1, ew, "master")
        check(p.detach(), w1, param_bound(w1, ew, dtype), "param")


def test_matches_torch_adamw():
    """Ten steps of torch.optim.AdamW: each may differ by the roundings of the
    weight (4 of 2^-24 relative) and of the update (24, of at most 1.2 lr)."""
    p, opt, gen = make(500)
    q = torch.nn.Parameter(p.detach().clone())
    ref = torch.optim.AdamW([q], lr=HYPER["lr"], betas=HYPER["betas"],
                            eps=HYPER["eps"], weight_decay=HYPER["wd"])
    for _ in range(10):
        p.grad = torch.randn(500, generator=gen)
        q.grad = p.grad.clone()
        opt.step(HYPER["lr"])
        ref.step()
    bound = 10 * 2.0 ** -24 * (4 * (q.abs() + 0.1) + 24 * 2 * HYPER["lr"])
    assert ((p - q).abs() <= bound).all()


LONG_RUNS = [((0.9, 0.999999), 1e-3, 12314), ((0.9, 0.999999), 1e-3, 155629),
             ((0.99999, 0.999), 1e-4, 20739), ((0.999999, 0.999), 1e-3, 5943),
             ((0.9, 0.999), 1e-3, 400000)]


@pytest.mark.parametrize("betas, lr, t", LONG_RUNS)
def test_late_steps_go_by_the_kernels_products(betas, lr, t):
    """b^t comes from squarings, rounded one by one, whose error at these steps
    decides a float32: the step is the one with the scalars that they give."""
    def power(b, k):
        out = 1.0
        for bit in reversed(bin(k)[2:]):
            out = out * b if bit == "1" else out
            b = b * b
        return out

    g = torch.Generator().manual_seed(0)
    p = torch.nn.Parameter(torch.zeros(4096))
    opt = SodAdamW([{"params": [p], "weight_decay": 0.0}], betas=betas)
    opt.exp_avg.copy_(torch.randn(4096, generator=g))
    opt.exp_avg_sq.copy_(torch.rand(4096, generator=g))
    opt.set_step(t - 1)
    p.grad = torch.zeros(4096)
    opt.step(lr)
    rate = torch.tensor(lr / (1 - power(betas[0], t)), dtype=torch.float32)
    rbc2 = torch.tensor(1 / math.sqrt(1 - power(betas[1], t)), dtype=torch.float32)
    r = opt.exp_avg_sq.double().sqrt().float()
    want = -(rate * (opt.exp_avg / (r * rbc2 + torch.tensor(1e-8))))
    assert torch.equal(p.detach(), want)


def test_groups_scale_and_skip():
    ps = [torch.nn.Parameter(torch.ones(5)) for _ in range(3)]
    opt = SodAdamW([{"params": ps[:1], "weight_decay": 0.5},
                    {"params": ps[1:]}], weight_decay=0.0)
    for p in ps[:2]:
        p.grad = torch.zeros(5)
    opt.step(0.1)                       # no gradient: decay alone, or nothing
    assert torch.equal(ps[0], torch.full((5,), 1.0) * (1 - 0.1 * 0.5))
    assert torch.equal(ps[1], torch.ones(5))
    assert [s["step"] for s in opt.state_dict()["param_state"]] == [1, 1, 0]
    ps[2].grad = torch.full((5,), 3.0)
    opt.step(0.1, scale_t=torch.tensor(0.0))
    assert [s["step"] for s in opt.state_dict()["param_state"]] == [1, 1, 0]
    assert torch.equal(ps[2], torch.ones(5))
    a = ps[2].detach().clone()
    opt.step(0.1, 0.5, scale_t=torch.tensor(0.25))
    want = step64(a.double(), torch.full((5,), 3.0).double(),
                  torch.zeros(5).double(), torch.zeros(5).double(), 1, 0.1,
                  (0.9, 0.999), 1e-8, 0.0, 0.125)
    check(ps[2].detach(), want[0], want[5], "scaled")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape", [(0,), (0, 3), (3, 0), (2, 0, 4)])
def test_empty_parameters(bits, shape):
    """Whatever their strides; their neighbours step as if alone."""
    p, alone = (torch.nn.Parameter(torch.ones(5)) for _ in range(2))
    e = torch.nn.Parameter(torch.empty(shape))
    opt = SodAdamW([{"params": [e, p]}], state_bits=bits)
    one = SodAdamW([{"params": [alone]}], state_bits=bits)
    for q in (e, p, alone):
        q.grad = torch.full_like(q, 0.5)
    opt.step(0.1)
    one.step(0.1)
    assert torch.equal(p, alone)
    again = SodAdamW([{"params": [e, p]}], state_bits=bits)
    again.load_state_dict(opt.state_dict())


def test_strided_parameters_and_gradients():
    """Parameters in another order than row by row, gradients in either."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5, 4, 3, generator=g)
    dense = torch.nn.Parameter(x.clone())
    last = torch.nn.Parameter(x.clone().contiguous(memory_format=torch.channels_last))
    for bits in (32, 8):
        opts = [SodAdamW([{"params": [p]}], state_bits=bits) for p in (dense, last)]
        assert opts[1].state[last].get("exp_avg", last).stride() == last.stride()
        for grad_last in (False, True):
            gr = torch.randn(6, 5, 4, 3, generator=g)
            if grad_last:
                gr = gr.contiguous(memory_format=torch.channels_last)
            dense.grad, last.grad = gr.clone(), gr.clone()
            for o in opts:
                o.step(0.01)
        if bits == 32:
            assert torch.equal(dense, last)


# ------------------------------------------------------------------ 8 bits

def test_codes_are_levels():
    """Every code is the value it stands for, to the bit."""
    c = torch.arange(256, dtype=torch.uint8)
    m, r = reference.adamw8_decode(c, c, torch.ones(1, 2))
    m64, r64 = decode64(c.int(), c.int(), torch.ones(1, 2))
    assert torch.equal(m.double(), m64) and torch.equal(r.double(), r64)
    assert m[127] == 1 and m[255] == -1 and r[255] == 1 and r[0] == 0
    assert (r[1:].diff() > 0).all()


def test_rounding_keeps_the_mean():
    """Over all 65536 noises a value's mean is itself, to the 16 bits of the noise:
    the bits below them (4 of m's 20 cut, 3 of r's 19) are lost, under one in
    65536 of a code step, 1/8 and 1/16 of the value at most."""
    noise = torch.arange(65536, dtype=torch.int64)
    for x in (1.0, 0.7301, 0.3, 0.0123, 1.7e-3, 4.4e-5):
        for which, steps in ((0, 8), (1, 16)):
            v = torch.full((65536, 256), x)
            v[:, 0] = 1.0                   # the block's largest
            n = (noise << 16 if which == 0 else noise).view(-1, 1).expand(-1, 256)
            args = (v, torch.zeros_like(v)) if which == 0 else (torch.zeros_like(v), v)
            got = torch.stack(reference.adamw8_decode(*reference.adamw8_encode(
                *(a.reshape(-1) for a in args), n.reshape(-1))))[which]
            mean = got.double().view(-1, 256)[:, 1].mean().item()
            want = float(torch.tensor(x).double())
            assert abs(mean - want) <= want / steps / 65536 * 1.001, (x, which)


def test_r_never_rounds_to_zero():
    r = torch.full((256,), 1e-30)
    r[0], r[1] = 1.0, 0.0
    for n in (0, 0xFFFFFFFF):
        _, code, _ = reference.adamw8_encode(torch.zeros(256), r,
                                             torch.full((256,), n, dtype=torch.int64))
        assert code[0] == 255 and code[1] == 0 and (code[2:] == 1).all()


@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step8_against_64_bits(n, dtype):
    """The weight goes by the moments before they are rounded; the codes lie
    within a step, 1/8 of m and 1/16 of r, of them."""
    p, opt, gen = make(n, dtype, bits=8)
    st = opt.state[p]
    for t in range(1, 4):
        p.grad = (torch.randn(n, generator=gen) * 10.0 ** (t - 2)).to(dtype)
        m0, r0 = decode64(st["code_m"].int(), st["code_r"].int(), st["scales"])
        w = st["master"] if "master" in st else p.detach()
        w1, m1, v1, em, ev, ew = step64(w.double(), p.grad.double(), m0[:n],
                                        r0[:n] ** 2, t, gs=1.0, **HYPER)
        # the old moments' own roundings: their scale's product, r's square
        ew = ew * 2
        opt.step(HYPER["lr"])
        check(p.detach(), w1, param_bound(w1, ew, dtype), "param")
        m, r = decode64(st["code_m"].int(), st["code_r"].int(), st["scales"])
        blk = torch.arange(n) // 256
        floor = st["scales"].double()[blk] * 2.0 ** -15
        check(m[:n], m1, m1.abs() / 8 + floor[:, 0] + em, "m")
        check(r[:n], v1.sqrt(), v1.sqrt() / 16 * (1 + 1e-5) + floor[:, 1], "r")
        assert (st["code_m"][n:] == 0).all() and (st["code_r"][n:] == 0).all()


def test_r_follows_a_change():
    """r of elements whose gradients grow a hundredfold follows them, though most
    steps move it by far less than half a code step: the rounding keeps the
    mean, and over 256 elements that each lie within a code step or two (6 % of
    r, 13 % of v) the mean is good to a few percent."""
    p, opt, _ = make(512, bits=8)
    small = torch.ones(512)
    small[::2] = 0.01                       # the other half sets the scales
    for _ in range(200):
        p.grad = small
        opt.step(0.0)
    p.grad = torch.ones(512)
    for _ in range(300):
        opt.step(0.0)
    _, v = opt.moments()
    want = 0.001 * sum(0.999 ** i * (1.0 if i < 300 else 1e-4) for i in range(500))
    got = v.float()[::2].mean().item()
    assert abs(got / want - 1) < 0.1, (got, want)


def test_non_finite_gradient_is_loud():
    p, opt, _ = make(512, bits=8)
    p.grad = torch.zeros(512)
    p.grad[300] = math.nan
    opt.step(0.1)
    s = opt.scales
    assert torch.isfinite(s[0]).all() and torch.isnan(s[1]).all()
    m, v = opt.moments()
    assert torch.isnan(m[256:512]).all() and torch.isfinite(m[:256]).all()
    p.grad[300] = math.inf
    opt2 = SodAdamW([{"params": [p]}], state_bits=8)
    opt2.step(0.1)
    assert not torch.isfinite(opt2.scales[1]).any()


@pytest.mark.parametrize("big", [2e21, 1e22, -3e38])
def test_square_past_float32_is_loud(big):
    """A finite gradient whose square is not (0.001 * g * g past 3.4e38) makes both
    moments of its block not finite, and of no other."""
    p, opt, gen = make(700, bits=8)
    p.grad = torch.randn(700, generator=gen)
    p.grad[300] = big
    opt.step(0.1)
    finite = torch.isfinite(opt.scales)
    assert finite[0].all() and finite[2].all() and not finite[1].any()
    for t in opt.moments():
        assert not torch.isfinite(t[256:512]).any()
        assert torch.isfinite(t[:256]).all() and torch.isfinite(t[512:]).all()


def test_noise_past_32_bits():
    """Elements 2^32 apart have other noise, tensors and steps too."""
    a = reference.adamw8_noise(4, 1, 1, 0)
    assert not torch.equal(a, reference.adamw8_noise(4, 1, 2, 0))
    assert not torch.equal(a, reference.adamw8_noise(4, 1, 1, 1))
    far = reference.adamw8_noise(4, 1, 1, 0, first=2 ** 32)
    assert not torch.equal(a, far)
    assert torch.equal(reference.adamw8_noise(6, 1, 1, 0, first=2 ** 32 - 2)[2:], far)


# ------------------------------------------------------------------ state

@pytest.mark.parametrize("bits", [32, 8])
def test_resume_is_bitwise(bits, tmp_path):
    p, opt, gen = make(700, torch.bfloat16, bits)
    for _ in range(3):
        p.grad = torch.randn(700, generator=gen).bfloat16()
        opt.step(0.01)
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    q = torch.nn.Parameter(p.detach().clone())
    other = SodAdamW([{"params": [q], "weight_decay": 0.0}], state_bits=bits, seed=77)
    other.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    for _ in range(2):
        p.grad = torch.randn(700, generator=gen).bfloat16()
        q.grad = p.grad.clone()
        opt.step(0.01)
        other.step(0.01)
    assert torch.equal(p, q) and torch.equal(opt.master, other.master)
    for a, b in zip(opt.moments(), other.moments()):
        assert torch.equal(a, b)


def test_resume_in_another_layout():
    """Moments in 32 bits follow their elements, codes lie in storage order."""
    x = torch.randn(4, 3, 2, 5)
    last = x.clone().contiguous(memory_format=torch.channels_last)
    for bits in (32, 8):
        p, q = torch.nn.Parameter(x.clone()), torch.nn.Parameter(last.clone())
        a, b = (SodAdamW([{"params": [t]}], state_bits=bits) for t in (p, q))
        p.grad = torch.randn(4, 3, 2, 5)
        a.step(0.01)
        if bits == 8:
            with pytest.raises(ValueError, match="layout"):
                b.load_state_dict(a.state_dict())
            continue
        q.data.copy_(p.data)
        b.load_state_dict(a.state_dict())
        q.grad = p.grad.clone()
        a.step(0.01)
        b.step(0.01)
        assert torch.equal(p, q)


def test_refusals():
    p = torch.nn.Parameter(torch.ones(4))
    ok = [{"params": [p]}]
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(-0.1, 0.9)), dict(eps=0.0),
               dict(state_bits=16)):
        with pytest.raises(ValueError):
            SodAdamW(ok, **kw)
    with pytest.raises(ValueError, match="twice"):
        SodAdamW([{"params": [p, p]}])
    with pytest.raises(ValueError, match="float"):
        SodAdamW([{"params": [torch.nn.Parameter(torch.ones(4).double())]}])
    with pytest.raises(ValueError, match="dense"):
        SodAdamW([{"params": [torch.nn.Parameter(torch.ones(8)[::2])]}])
    with pytest.raises(ValueError, match="dense"):
        SodAdamW([{"params": [torch.nn.Parameter(torch.ones(1).expand(4))]}])
    flat = torch.ones(6)
    with pytest.raises(ValueError, match="overlap"):
        SodAdamW([{"params": [torch.nn.Parameter(flat[:4]), torch.nn.Parameter(flat[3:])]}])
    opt = SodAdamW(ok)
    with pytest.raises(AttributeError):
        opt.code_m
    with pytest.raises(ValueError):
        opt.set_step(-1)
    opt.grad_src = {p: torch.ones(5)}
    with pytest.raises(RuntimeError, match="size"):
        opt.step(0.1)
    sgd = SodSGD(ok)
    with pytest.raises(ValueError, match="sgd"):
        opt.load_state_dict(sgd.state_dict())
    with pytest.raises(ValueError, match="32 bits"):
        SodAdamW(ok, state_bits=8).load_state_dict(opt.state_dict())
    two = SodAdamW([{"params": [p, torch.nn.Parameter(torch.ones(4))]}])
    with pytest.raises(ValueError, match="parameters"):
        two.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="fit"):
        SodAdamW([{"params": [torch.nn.Parameter(torch.ones(5))]}]).load_state_dict(
            opt.state_dict())
    q = torch.nn.Parameter(torch.ones(2, 3, 4, 5))
    opt = SodAdamW([{"params": [q]}])
    q.data = q.data.contiguous(memory_format=torch.channels_last)
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="layout"):
        opt.step(0.1)
    assert SodAdamW([]).step(0.1) is None


@pytest.mark.parametrize("eps", [1e-46, 7e-46, 0.0, -1e-8, math.nan])
def test_eps_that_float32_makes_zero(eps):
    """The step divides by root + eps in float32; moments that are zero have no
    root to save it."""
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="eps"):
        SodAdamW([{"params": [p]}], eps=eps)
    opt = SodAdamW([{"params": [p]}], eps=2e-45, weight_decay=0.0)  # a denormal is enough
    p.grad = torch.zeros(4)
    opt.step(0.1)
    assert torch.equal(p, torch.ones(4))
    sd = opt.state_dict()
    other = SodAdamW([{"params": [torch.nn.Parameter(torch.zeros(4))]}])
    with pytest.raises(ValueError, match="eps"):
        other.load_state_dict({**sd, "eps": eps})


def test_load_checks_before_it_writes():
    p = torch.nn.Parameter(torch.ones(4))
    opt = SodAdamW([{"params": [p]}])
    p.grad = torch.ones(4)
    opt.step(0.1)
    sd = opt.state_dict()
    other = SodAdamW([{"params": [torch.nn.Parameter(torch.ones(4))]}], betas=(0.8, 0.9))
    bad = [{**sd, "betas": b} for b in ((1.0, 0.9), (0.9, 1.5), (math.nan, 0.9))]
    bad += [{**sd, "param_state": [{**sd["param_state"][0], "step": t}]}
            for t in (-1, 2 ** 31 - 1)]
    for x in bad:
        with pytest.raises(ValueError):
            other.load_state_dict(x)
        assert other.betas == (0.8, 0.9) and not other.exp_avg.any()
        assert other.state_dict()["param_state"][0]["step"] == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_sgd_refuses_its_checkpoint(bits):
    """With a message that says why, and before it moves anything."""
    p = torch.nn.Parameter(torch.ones(4))
    sgd = SodSGD([{"params": [p]}], momentum=0.7)
    opt = SodAdamW([{"params": [p]}], state_bits=bits)
    with pytest.raises(ValueError, match="adamw"):
        sgd.load_state_dict(opt.state_dict())
    assert sgd.momentum == 0.7
    sgd.load_state_dict(sgd.state_dict())


def test_update_decay_hands_changes_over():
    """The device's copy is written when a group's decay changed, and if that
    fails it is not taken for written."""
    class Plan:
        calls, fail = [], False

        def set_decay(self, wd):
            if self.fail:
                raise RuntimeError("in a capture")
            self.calls.append(wd)

    opt = SodAdamW([{"params": [torch.nn.Parameter(torch.ones(2)) for _ in range(2)]},
                    {"params": [torch.nn.Parameter(torch.ones(2))], "weight_decay": 0.5}],
                   weight_decay=0.1)
    opt.update_decay()                          # nothing to do on the CPU
    opt._plan, opt._plan_wd = Plan(), [0.1, 0.5]
    opt.update_decay()
    assert Plan.calls == []
    opt.groups[1]["weight_decay"] = 0.0
    Plan.fail = True
    with pytest.raises(RuntimeError):
        opt.update_decay()
    Plan.fail = False
    opt.update_decay()
    opt.update_decay()
    assert Plan.calls == [[0.1, 0.1, 0.0]]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_of_another_type_is_refused(bits):
    """A float32 parameter is its own master: gone to 16 bits it would lose it."""
    for old, new in ((torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16),
                     (torch.bfloat16, torch.float32)):
        p = torch.nn.Parameter(torch.ones(5, dtype=old))
        opt = SodAdamW([{"params": [p]}], state_bits=bits)
        p.data = p.data.to(new)
        p.grad = torch.ones_like(p)
        with pytest.raises(RuntimeError, match="type"):
            opt.step(0.1)
        assert torch.equal(p, torch.ones(5, dtype=new))


@pytest.mark.parametrize("shape", [(4, 3, 1, 1), (1, 5, 2, 3), (2, 1, 3, 4)])
def test_strides_of_single_elements_do_not_count(shape):
    """The same order in storage under other strides is no change of layout."""
    x = torch.arange(math.prod(shape)).float()
    last = x.view(shape).clone().contiguous(memory_format=torch.channels_last)
    p, q = torch.nn.Parameter(last.clone()), torch.nn.Parameter(last.clone())
    opts = [SodAdamW([{"params": [t]}]) for t in (p, q)]
    strides = [st if n > 1 else 17 for st, n in zip(q.stride(), shape)]
    q.data = q.data.as_strided(shape, strides)
    for t, o in zip((p, q), opts):
        t.grad = last * 0.1
        o.step(0.1)
    assert torch.equal(p, q) and not torch.equal(p, last)


@pytest.mark.parametrize("shape", [(0,), (2,), (3, 1)])
def test_scalars_that_are_none(shape):
    """An empty one is not taken for one that was not given."""
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones_like(p)
    opt = SodAdamW([{"params": [p]}])
    t, one = torch.ones(shape), torch.ones(())
    with pytest.raises(RuntimeError, match="lr must be"):
        opt.step(t)
    with pytest.raises(RuntimeError, match="scale_t must be"):
        opt.step(0.1, scale_t=t)
    for kw in (dict(loss_scale=t), dict(loss_scale=one, good_steps=t, skips=one),
               dict(loss_scale=one, good_steps=one, skips=t)):
        with pytest.raises(ValueError, match="must be a scalar"):
            grad_norm([p.grad], **kw)
    assert (p == 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_come_to_overlap(bits):
    """Weights that move are looked at again; apart again, they step."""
    flat = torch.ones(600)
    ps = [torch.nn.Parameter(flat[:300]), torch.nn.Parameter(flat[300:])]
    opt = SodAdamW([{"params": ps}], state_bits=bits)
    opt.grad_src = {p: torch.ones(300) for p in ps}
    opt.step(0.1)
    for tied in (flat[:300], flat[299:599]):
        before = flat.clone()
        ps[1].data = tied
        with pytest.raises(RuntimeError, match="overlap"):
            opt.step(0.1)
        assert torch.equal(flat, before)
        ps[1].data = flat[300:]
        opt.step(0.1)
        assert not torch.equal(flat, before)


def test_grad_src_is_what_was_given():
    """Neither path goes by what becomes of the dict later, and the optimizer's own
    cannot be written."""
    p = torch.nn.Parameter(torch.zeros(3))
    opt = SodAdamW([{"params": [p]}])
    views = {p: torch.ones(3)}
    opt.grad_src = views
    views[p] = -views[p]
    opt.step(0.1)
    assert (p < 0).all()
    with pytest.raises(TypeError):
        opt.grad_src[p] = views[p]
    opt.grad_src = {**opt.grad_src, p: views[p]}
    for _ in range(3):
        opt.step(0.1)
    assert (p > 0).all()


def test_native_refusals():
    """The extension's own checks, which a GPU call would reach."""
    from sodkit import _C
    none = torch.Tensor()
    with pytest.raises(RuntimeError, match="no gradients"):
        _C.grad_norm([], 1.0, 0.0, none, none, none, 500.0)
    with pytest.raises(RuntimeError, match="GPU"):
        _C.grad_norm([torch.ones(3)], 1.0, 0.0, none, none, none, 500.0)
    with pytest.raises(RuntimeError):
        _C.AdamWPlan([torch.ones(3)], [0.0], [0], [-1], none, [none, none])
    with pytest.raises(RuntimeError):
        _C.adamw8_decode(torch.zeros(256, dtype=torch.uint8),
                         torch.zeros(256, dtype=torch.uint8), torch.zeros(1, 2))


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_grad_norm(dtype):
    """The sum is in 64 bits, so only the two results' own roundings count."""
    g = torch.Generator().manual_seed(0)
    grads = [torch.randn(n, generator=g).to(dtype) for n in (0, 1, 7, 1000)]
    grads.append(torch.randn(33, 9, generator=g).t())
    n64 = math.sqrt(sum((x.double() ** 2).sum().item() for x in grads)) * 0.5
    norm, mult = grad_norm(grads, prescale=0.5)
    assert abs(norm.item() - n64) <= 2.0 ** -23 * n64 and mult.item() == 1.0
    norm, mult = grad_norm(grads, prescale=0.5, max_norm=0.1)
    assert abs(mult.item() - 0.1 / (n64 + 1e-6)) <= 2.0 ** -22 * mult.item()
    _, mult = grad_norm(grads, max_norm=1e9, loss_scale=torch.tensor(4.0))
    assert mult.item() == 0.25


def test_grad_norm_range():
    """Squares past float32's range are no overflow, and a tiny multiplier is
    no skip."""
    norm, mult = grad_norm([torch.full((4,), 1e38)], max_norm=1e-6)
    assert abs(norm.item() / 2e38 - 1) < 1e-6 and mult.item() > 0
    for bad in (math.inf, -math.inf, math.nan):
        norm, mult = grad_norm([torch.tensor([1.0, bad])], max_norm=1.0)
        assert not math.isfinite(norm.item()) and mult.item() == 0.0
    norm, mult = grad_norm([torch.zeros(0)], max_norm=1.0)
    assert norm.item() == 0.0 and mult.item() == 1.0


def test_grad_norm_scaler():
    scale, good, skips = torch.tensor(64.0), torch.tensor(0.0), torch.tensor(0.0)
    kw = dict(loss_scale=scale, good_steps=good, skips=skips, growth_interval=2)
    fine, bad = [torch.ones(3)], [torch.tensor([math.inf])]
    assert grad_norm(fine, **kw)[1].item() == 1 / 64
    assert (scale.item(), good.item()) == (64.0, 1.0)
    assert grad_norm(fine, **kw)[1].item() == 1 / 64     # by the scale before
    assert (scale.item(), good.item()) == (128.0, 0.0)
    assert grad_norm(bad, **kw)[1].item() == 0.0
    assert (scale.item(), good.item(), skips.item()) == (64.0, 0.0, 1.0)
    scale.fill_(1.0)
    grad_norm(bad, **kw)
    assert scale.item() == 1.0 and skips.item() == 2.0
    scale.fill_(65536.0)
    good.fill_(1.0)
    grad_norm(fine, **kw)
    assert scale.item() == 65536.0


def test_grad_norm_refusals():
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(ValueError):
        grad_norm([torch.ones(3).double()])
    with pytest.raises(ValueError):
        grad_norm([torch.ones(3)], good_steps=torch.tensor(0.0))
    with pytest.raises(ValueError):
        grad_norm([torch.ones(3)], good_steps=torch.tensor(0.0),
                  skips=torch.tensor(0.0))
    with pytest.raises(ValueError):
        grad_norm([torch.ones(3)], growth_interval=0)


# ------------------------------------------------------------------ ranks

def _net():
    torch.manual_seed(7)
    return torch.nn.Sequential(torch.nn.Linear(8, 50), torch.nn.ReLU(),
                               torch.nn.Linear(50, 4))


def _grads(m, rank, i):
    """The gradients of a rank's data in step i."""
    x = torch.full((2, 8), 0.1 * (rank + 1) * (i + 1)) + torch.arange(8) * 0.01
    return torch.autograd.grad(m(x).square().sum(), list(m.parameters()))


def _ranks_worker(rank, store, bits, q):
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=2,
                            init_method=f"file://{store}")
    m = _net()
    red = GradReducer(m, bucket_mb=1)
    opt = SodAdamW([{"params": list(m.parameters())}], state_bits=bits, seed=3)
    opt.grad_src = red.grad_views
    for i in range(3):
        red.zero_grad()
        x = torch.full((2, 8), 0.1 * (rank + 1) * (i + 1)) + torch.arange(8) * 0.01
        m(x).square().sum().backward()
        red.finalize()
        _, mult = grad_norm([b.flat for b in red.buckets],
                            prescale=red.grad_scale, max_norm=0.1)
        opt.step(1e-2, red.grad_scale, scale_t=mult)
    q.put((rank, [p.detach().numpy() for p in m.parameters()]))  # by value
    dist.destroy_process_group()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("bits", [32, 8])
def test_ranks_agree(bits, tmp_path):
    """Two ranks end with the same bits, those of one process that adds up both
    ranks' gradients."""
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    procs = [ctx.Process(target=_ranks_worker, args=(r, str(tmp_path / "s"), bits, q))
             for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get() for _ in range(2))
    for p in procs:
        p.join()
    assert all(p.exitcode == 0 for p in procs)
    m = _net()
    opt = SodAdamW([{"params": list(m.parameters())}], state_bits=bits, seed=3)
    for i in range(3):
        for p, a, b in zip(m.parameters(), _grads(m, 0, i), _grads(m, 1, i)):
            p.grad = a + b
        # the buckets' order: from the last parameter
        _, mult = grad_norm([p.grad for p in reversed(list(m.parameters()))],
                            prescale=0.5, max_norm=0.1)
        opt.step(1e-2, 0.5, scale_t=mult)
    for a, b, p in zip(got[0], got[1], m.parameters()):
        a, b = torch.from_numpy(a), torch.from_numpy(b)
        assert torch.equal(a, b)
        # (the norm's sum is grouped otherwise, in 64 bits: its float32 is the same)
        assert torch.equal(a, p)


# ------------------------------------------------------------------ the solver

def _solver(tmp_path, **kw):
    return Solver(make_config("cpu_plumbing", output_root=str(tmp_path), size=48,
                              train_samples=4, val_samples=2, epoch_num=1,
                              num_workers=0, log_interval=1, optimizer="adamw",
                              lr=1e-3, **kw))


@pytest.mark.parametrize("bits", [32, 8])
def test_solver_trains_and_resumes(tmp_path, bits):
    s = _solver(tmp_path, adam_state_bits=bits, grad_clip=1.0)
    assert isinstance(s.optimizer, SodAdamW) and s.optimizer.state_bits == bits
    before = [p.detach().clone() for p in s.model.parameters()]
    s.train()
    assert any(not torch.equal(a, b) for a, b in zip(before, s.model.parameters()))
    r = _solver(tmp_path, adam_state_bits=bits, resume=True)
    r.train()                                   # loads; no epoch is left
    for a, b in zip(s.optimizer.state_dict()["param_state"],
                    r.optimizer.state_dict()["param_state"]):
        assert a["step"] == b["step"] == 2
        for k in a:
            assert k in ("step", "order") or torch.equal(a[k], b[k])
    with pytest.raises(ValueError, match="checkpoint"):
        _solver(tmp_path, adam_state_bits=40 - bits, resume=True).train()


def test_solver_device_scaler_state(tmp_path):
    """The device scaler with adamw moves as the one with sgd does."""
    s = _solver(tmp_path)
    s.dynamic_scale = s._use_device_scaler = True
    s._growth_interval = 2
    s._scale_t, s._good_t, s._skips_t = torch.tensor(64.0), torch.zeros(()), torch.zeros(())
    for b in s.reducer.buckets:
        b.flat.fill_(1.0)
    assert s._device_clip_and_scale().item() == 1 / 64
    assert s._device_clip_and_scale().item() == 1 / 64
    assert s._scale_t.item() == 128.0
    s.reducer.buckets[0].flat[0] = float("inf")
    assert s._device_clip_and_scale().item() == 0.0
    assert (s._scale_t.item(), s._skips_t.item()) == (64.0, 1.0)


def test_solver_says_when_the_rate_is_sgds(tmp_path):
    """AdamW with a rate that was left as it is for SGD says so, any other is quiet."""
    for k, (kw, said) in enumerate(((dict(optimizer="adamw"), True),
                                    (dict(optimizer="adamw", lr=1e-3), False),
                                    (dict(), False))):
        s = Solver(make_config("cpu_plumbing", output_root=str(tmp_path),
                               exp_name=f"e{k}", **kw))
        with open(s.paths["log"]) as f:
            assert ("a rate for SGD" in f.read()) == said


def test_unknown_optimizer(tmp_path):
    with pytest.raises(ValueError, match="optimizer"):
        Solver(make_config("cpu_plumbing", output_root=str(tmp_path), optimizer="adam"))
