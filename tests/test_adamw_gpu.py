"""SodAdamW and grad_norm on the GPU: the bits of the CPU path, the definitions
in 64 bits, layouts, streams, captured steps and refusals."""

import math

import pytest
import torch

from adamw_oracle import check, param_bound, step64
from sodkit import ops
from sodkit.ops import SodAdamW, grad_norm, reference

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [1, 2, 3, 5, 64, 255, 256, 257, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 70001]


def pair(shapes, dtype, bits, grad_dtype=None, device="cuda", seed=0, odd=False):
    """The same parameters on the CPU and on the GPU, gradients given apart; odd:
    at any element of one storage."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(math.prod(s) for s in shapes) + 1
    flat = torch.randn(total, generator=gen).to(dtype)
    gflat = torch.randn(total, generator=gen).to(grad_dtype or dtype)
    sides = []
    for dev in ("cpu", device):
        f, g = flat.to(dev, copy=True), gflat.to(dev, copy=True)
        ps, src, at = [], {}, 1 if odd else 0
        for s in shapes:
            n = math.prod(s)
            p = f[at:at + n].view(s) if odd else f[at:at + n].view(s).clone()
            p = torch.nn.Parameter(p)
            src[p] = g[at:at + n].view(s) if odd else g[at:at + n].view(s).clone()
            ps.append(p)
            at += n
        k = len(ps) // 2
        opt = SodAdamW([{"params": ps[:k], "weight_decay": 0.1},
                        {"params": ps[k:], "weight_decay": 0.0}],
                       state_bits=bits, seed=11)
        opt.grad_src = src
        sides.append((ps, src, opt))
    return sides


def differ(a, b):
    """How many elements are not the same."""
    return int((a.detach().cpu() != b.detach().cpu()).sum())


def same(a, b):
    (ps, _, oa), (qs, _, ob) = a, b
    for k, (p, q) in enumerate(zip(ps, qs)):
        n = differ(p, q)
        assert n == 0, (k, tuple(p.shape))
    sa, sb = oa.state_dict()["param_state"], ob.state_dict()["param_state"]
    for k, (x, y) in enumerate(zip(sa, sb)):
        assert x["step"] == y["step"]
        for n in x:
            assert n in ("step", "order") or differ(x[n], y[n]) == 0, (k, n)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grad_dtype", TYPES)
@pytest.mark.parametrize("odd", [False, True])
def test_bits_of_the_cpu(bits, dtype, grad_dtype, odd):
    cpu, gpu = pair([(n,) for n in SIZES] + [(0,), (7, 3, 3, 5)], dtype, bits,
                    grad_dtype, odd=odd)
    for i in range(3):
        lr = torch.tensor(1e-3 * (i + 1), device="cuda") if i == 1 else 1e-3 * (i + 1)
        mult = torch.tensor(0.75) if i == 2 else None
        cpu[2].step(lr, 0.5, scale_t=mult)
        gpu[2].step(lr, 0.5, scale_t=None if mult is None else mult.cuda())
        same(cpu, gpu)


@pytest.mark.parametrize("dtype", TYPES)
def test_against_64_bits(dtype):
    _, (ps, src, opt) = pair([(70001,), (33,)], dtype, 32)
    opt.set_step(9)
    opt.exp_avg.normal_()
    opt.exp_avg_sq.uniform_()
    for p, wd in zip(ps, (0.1, 0.0)):
        st = opt.state[p]
        w = (st["master"] if "master" in st else p.detach()).double()
        st["want"] = step64(w, src[p].double(), st["exp_avg"].double(),
                            st["exp_avg_sq"].double(), 10, 1e-2, opt.betas,
                            opt.eps, wd, 0.5)
    opt.step(1e-2, 0.5)
    for p in ps:
        st = opt.state[p]
        w1, m1, v1, em, ev, ew = st.pop("want")
        check(st["exp_avg"], m1, em, "m")
        check(st["exp_avg_sq"], v1, ev, "v")
        check(p.detach(), w1, param_bound(w1, ew, dtype), "param")
        if "master" in st:
            check(st["master"], w1, ew, "master")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas, lr, t", [
    ((0.9, 0.999999), 1e-3, 12314), ((0.9, 0.999999), 1e-3, 155629),
    ((0.99999, 0.999), 1e-4, 20739), ((0.999999, 0.999), 1e-3, 5943),
    ((0.9, 0.999), 1e-3, 400000), ((0.9, 0.99999), 3e-4, 2 ** 31 - 2)])
def test_bits_late_in_a_run(bits, betas, lr, t):
    """At step counts and betas where the power's error decides a float32."""
    cpu, gpu = pair([(4096,), (33,)], torch.float32, bits)
    for _, _, opt in (cpu, gpu):
        opt.betas = betas
        opt.set_step(t - 1)
        opt.step(lr)
    same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than one launch's arguments hold."""
    cpu, gpu = pair([(i % 37 + 1,) for i in range(500)], torch.bfloat16, bits)
    for _ in range(2):
        cpu[2].step(1e-2)
        gpu[2].step(1e-2)
    same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_empty_parameters(bits):
    cpu, gpu = pair([(3, 0), (5,), (2, 0, 4), (300,), (0, 3)], torch.bfloat16, bits)
    for _ in range(2):
        cpu[2].step(1e-2)
        gpu[2].step(1e-2)
    same(cpu, gpu)
    only = SodAdamW([{"params": [torch.nn.Parameter(torch.empty(3, 0, device="cuda"))]}],
                    state_bits=bits)
    only.step(1e-2)


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_and_no_gradient(bits):
    ps = [torch.nn.Parameter(torch.randn(300, device="cuda").to(t)) for t in TYPES]
    qs = [torch.nn.Parameter(p.detach().cpu()) for p in ps]
    opts = [SodAdamW([{"params": x}], state_bits=bits) for x in (ps, qs)]
    for leave in (1, 0, None):
        for k, (p, q) in enumerate(zip(ps, qs)):
            p.grad = None if k == leave else torch.randn_like(p)
            q.grad = None if k == leave else p.grad.cpu()
        for o in opts:
            o.step(1e-2)
    same((qs, None, opts[1]), (ps, None, opts[0]))
    assert [s["step"] for s in opts[0].state_dict()["param_state"]] == [2, 2, 3]


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    x = torch.randn(6, 5, 4, 3)
    last = torch.channels_last
    for grad_last in (False, True):
        ps = [torch.nn.Parameter(x.to(d, copy=True).contiguous(memory_format=last))
              for d in ("cpu", "cuda")]
        gr = torch.randn(6, 5, 4, 3)
        opts = []
        for p in ps:
            p.grad = gr.to(p.device).contiguous(memory_format=last) if grad_last \
                else gr.to(p.device)
            opts.append(SodAdamW([{"params": [p]}], state_bits=bits))
            opts[-1].step(1e-2)
            p.grad = gr.to(p.device)[:, :, :, torch.arange(3)].expand_as(p)
            opts[-1].step(1e-2)
        same(([ps[0]], None, opts[0]), ([ps[1]], None, opts[1]))


@pytest.mark.parametrize("shape", [(4, 3, 1, 1), (1, 5, 2, 3), (2, 1, 3, 4)])
def test_strides_of_single_elements_do_not_count(shape):
    """The same order in storage under other strides is no change of layout."""
    x = torch.arange(math.prod(shape), device="cuda").float()
    last = x.view(shape).clone().contiguous(memory_format=torch.channels_last)
    p, q = torch.nn.Parameter(last.clone()), torch.nn.Parameter(last.clone())
    opts = [SodAdamW([{"params": [t]}]) for t in (p, q)]
    strides = [st if n > 1 else 17 for st, n in zip(q.stride(), shape)]
    q.data = q.data.as_strided(shape, strides)
    for t, o in zip((p, q), opts):
        t.grad = last * 0.1
        o.step(0.1)
    assert torch.equal(p, q) and not torch.equal(p, last)


def test_another_size_in_the_same_strides_is_refused():
    p = torch.nn.Parameter(torch.ones(6, 4, device="cuda").t())
    opt = SodAdamW([{"params": [p]}])
    wide = torch.ones(31, device="cuda")
    for shape, strides in (((3, 8), (1, 4)), ((24,), (1,)), ((2, 3, 4), (1, 2, 6))):
        p.data = wide.as_strided(shape, strides)
        p.grad = None
        opt.grad_src = {p: torch.ones(shape, device="cuda")}
        with pytest.raises(RuntimeError, match="changed"):
            opt.step(0.1)
    assert (wide == 1).all()


def test_no_memory_is_refused():
    """Storage that was given back, or never there, is not read."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = SodAdamW([{"params": [p]}])
    for gone in (torch.ones(300, device="cuda"), torch.ones(400, device="cuda")[50:350],
                 torch.ones(600, device="cuda")[::2]):
        gone.untyped_storage().resize_(0)
        opt.grad_src = {p: gone}
        with pytest.raises(RuntimeError, match="no memory"):
            opt.step(0.1)
        with pytest.raises(RuntimeError, match="no memory"):
            grad_norm([gone])
    part = torch.ones(300, device="cuda")
    part.untyped_storage().resize_(299 * 4)
    opt.grad_src = {p: part}
    with pytest.raises(RuntimeError, match="no memory"):
        opt.step(0.1)
    with pytest.raises(RuntimeError, match="no memory"):
        grad_norm([torch.ones(5, device="cuda"), part])
    opt.grad_src = {p: torch.ones(300, device="cuda")}
    p.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="no memory"):
        opt.step(0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_negated_views(bits):
    """A view that stands for the negation of its memory counts with its sign."""
    x = torch.randn(300)
    c = torch.complex(torch.zeros(1), torch.ones(1))
    for n, view in ((300, lambda d: torch._neg_view(x.to(d))),
                    (1, lambda d: c.to(d).conj().imag)):
        sides = []
        for d in ("cpu", "cuda"):
            p = torch.nn.Parameter(torch.ones(n, device=d))
            opt = SodAdamW([{"params": [p]}], state_bits=bits)
            g = view(d)
            assert g.is_neg() and g.is_contiguous()
            opt.grad_src = {p: g}
            opt.step(1e-2)
            sides.append(([p], None, opt))
        same(*sides)
    p.data = torch._neg_view(p.data)
    with pytest.raises(RuntimeError, match="negated"):
        opt.step(1e-2)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_come_to_overlap(bits):
    """Weights that move are looked at again; apart again, they step."""
    flat = torch.ones(600, device="cuda")
    ps = [torch.nn.Parameter(flat[:300]), torch.nn.Parameter(flat[300:])]
    opt = SodAdamW([{"params": ps}], state_bits=bits)
    opt.grad_src = {p: torch.ones(300, device="cuda") for p in ps}
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
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    opt = SodAdamW([{"params": [p]}])
    views = {p: torch.ones(3, device="cuda")}
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


def test_decay_that_changes():
    cpu, gpu = pair([(500,), (33,)], torch.float32, 32)
    for wd in (0.1, 0.4):
        for _, _, o in (cpu, gpu):
            o.groups[0]["weight_decay"] = wd
            o.step(1e-2)
        same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_skip(bits):
    _, (ps, src, opt) = pair([(5000,), (3,)], torch.bfloat16, bits)
    opt.step(1e-2)
    before = [t.clone() for t in [*ps, opt.master, *opt.moments()]]
    for g in src.values():
        g.fill_(math.nan)
    opt.step(1e-2, scale_t=torch.zeros((), device="cuda"))
    for a, b in zip(before, [*ps, opt.master, *opt.moments()]):
        assert differ(a, b) == 0
    assert [s["step"] for s in opt.state_dict()["param_state"]] == [1, 1]


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_in_8_bits(bad):
    cpu, gpu = pair([(1000,)], torch.float32, 8)
    for ps, src, opt in (cpu, gpu):
        src[ps[0]][300] = bad
        opt.step(1e-2)
    s, t = cpu[2].scales, gpu[2].scales.cpu()
    assert torch.equal(torch.isfinite(s), torch.isfinite(t))
    assert not torch.isfinite(t[1]).any() and torch.isfinite(t[0]).all()
    for m in gpu[2].moments():
        m = m.cpu()
        assert torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()


@pytest.mark.parametrize("big", [2e21, -3e38])
def test_square_past_float32_in_8_bits(big):
    """The CPU and the GPU agree on the block that such a gradient takes away."""
    cpu, gpu = pair([(1000,)], torch.float32, 8)
    for ps, src, opt in (cpu, gpu):
        src[ps[0]][300] = big
        opt.step(1e-2)
        opt.step(1e-2)
        finite = torch.isfinite(opt.scales)
        assert finite[[0, 2, 3]].all() and not finite[1].any()
        for t in opt.moments():
            assert not torch.isfinite(t[256:512]).any()
            assert torch.isfinite(t[:256]).all() and torch.isfinite(t[512:]).all()
    keep = torch.ones(1000, dtype=torch.bool)
    keep[256:512] = False
    assert differ(cpu[0][0][keep], gpu[0][0].cpu()[keep]) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_move(bits):
    """A new gradient each step, as autograd makes them, and weights that move."""
    p = torch.nn.Parameter(torch.randn(3000, device="cuda"))
    q = torch.nn.Parameter(p.detach().cpu())
    opts = [SodAdamW([{"params": [x]}], state_bits=bits) for x in (p, q)]
    keep = []
    for i in range(4):
        keep.append(torch.randn(3000, device="cuda"))
        p.grad, q.grad = keep[-1], keep[-1].cpu()
        if i == 2:
            p.data = p.detach().clone()
        for o in opts:
            o.step(1e-2)
    same(([q], None, opts[1]), ([p], None, opts[0]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eager_first", [False, True])
def test_captured_step(bits, eager_first):
    """norm -> step in a graph, replayed with eager steps between the replays; the
    graph's gradients lie elsewhere than the eager ones.  A second graph of the
    same optimizer follows."""
    cpu, gpu = pair([(5000,), (77,), (4096,)], torch.bfloat16, bits)
    (ps, src, opt), (qs, gsrc, gopt) = cpu, gpu
    lr_t = torch.tensor(1e-2, device="cuda")
    inside = {q: g.clone() for q, g in gsrc.items()}
    other = {q: (g * 3).clone() for q, g in gsrc.items()}

    def both(lr, which):
        _, mult = grad_norm([which[q].cpu() for q in qs], max_norm=1.0)
        opt.grad_src = {p: which[q].cpu() for p, q in zip(ps, qs)}
        opt.step(lr, scale_t=mult)

    def gpu_step(which, lr):
        gopt.grad_src = which
        _, mult = grad_norm([which[q] for q in qs], max_norm=1.0)
        gopt.step(lr, scale_t=mult)

    if eager_first:
        gpu_step(gsrc, 1e-2)
        both(1e-2, gsrc)
    graphs = []
    for which in (inside, other):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu_step(which, lr_t)
        graphs.append((graph, which))
    for i in range(4):
        for graph, which in graphs:
            lr = 1e-2 / (i + 1)
            lr_t.fill_(lr)
            for g in which.values():
                g.mul_(0.5)
            graph.replay()
            torch.cuda.synchronize()
            both(float(lr_t), which)
            same(cpu, gpu)
        gpu_step(gsrc, 1e-3)
        both(1e-3, gsrc)
        torch.cuda.synchronize()
        same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_decay_that_changes_under_replays(bits):
    cpu, gpu = pair([(5000,), (33,)], torch.bfloat16, bits)
    (_, _, opt), (_, _, gopt) = cpu, gpu
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gopt.step(1e-2)
    for wd in (0.1, 0.4, 0.4, 0.0):
        for o in (opt, gopt):
            o.groups[0]["weight_decay"] = wd
            o.update_decay()
        graph.replay()
        opt.step(1e-2)
        same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_decay_that_changed_before_a_capture(bits):
    """Refused, with nothing moved; after update_decay the capture has it."""
    cpu, gpu = pair([(5000,), (33,)], torch.bfloat16, bits)
    (_, _, opt), (_, _, gopt) = cpu, gpu
    for o in (opt, gopt):
        o.step(1e-2)
        o.groups[0]["weight_decay"] = 0.4
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="update_decay"):
            gopt.step(1e-2)
        with pytest.raises(RuntimeError, match="capture"):
            gopt.set_step(3)
        with pytest.raises(RuntimeError, match="capture"):
            gopt.state_dict()
        torch.zeros(1, device="cuda")           # a graph that is not empty
    assert [s["step"] for s in gopt.state_dict()["param_state"]] == [1, 1]
    same(cpu, gpu)
    gopt.update_decay()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gopt.step(1e-2)
    for _ in range(3):
        graph.replay()
        opt.step(1e-2)
        same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_other_stream(bits):
    cpu, gpu = pair([(70001,), (5,)], torch.bfloat16, bits)
    side = torch.cuda.Stream()
    for i in range(4):
        cpu[2].step(1e-2)
        if i % 2:
            gpu[2].step(1e-2)
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                gpu[2].step(1e-2)
            torch.cuda.current_stream().wait_stream(side)
    same(cpu, gpu)


@pytest.mark.parametrize("bits", [32, 8])
def test_two_at_once(bits):
    """Two optimizers and norms on two streams."""
    cpu, gpu = pair([(300001,), (5,)], torch.bfloat16, bits)
    _, other = pair([(300001,), (5,)], torch.bfloat16, bits)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(5):
        for (ps, src, opt), st in zip((gpu, other), streams):
            with torch.cuda.stream(st):
                _, mult = grad_norm(list(src.values()), max_norm=1.0)
                opt.step(1e-2, scale_t=mult)
        _, mult = grad_norm(list(cpu[1].values()), max_norm=1.0)
        cpu[2].step(1e-2, scale_t=mult)
    torch.cuda.synchronize()
    same(cpu, gpu)
    same(cpu, other)


def test_resume_on_gpu():
    for bits in (32, 8):
        _, (ps, src, opt) = pair([(5000,), (33,)], torch.bfloat16, bits)
        opt.step(1e-2)
        _, (qs, qsrc, other) = pair([(5000,), (33,)], torch.bfloat16, bits)
        for p, q in zip(ps, qs):
            q.data.copy_(p)
        other.load_state_dict(opt.state_dict())
        for o in (opt, other):
            o.step(1e-3)
        for p, q in zip(ps, qs):
            assert differ(p, q) == 0
        assert other.state_dict()["param_state"][1]["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_load_under_a_captured_step(bits):
    """A state loaded after the capture is what the replays go on from."""
    cpu, gpu = pair([(5000,), (33,)], torch.bfloat16, bits)
    (ps, src, opt), (qs, gsrc, gopt) = cpu, gpu
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gopt.step(1e-2)
    for o in (opt, gopt):
        saved = SodAdamW([{"params": list(g["params"]), "weight_decay": 0.3}
                          for g in o.groups], state_bits=bits, seed=11)
        saved.grad_src = o.grad_src
        before = [p.detach().clone() for p in saved.params()]
        saved.step(1e-3)
        saved.step(1e-3)
        sd = {k: v for k, v in saved.state_dict().items()}
        for p, b in zip(saved.params(), before):
            p.data.copy_(b)
        o.load_state_dict(sd)
        del saved
    for i in range(3):
        graph.replay()
        opt.step(1e-2)
        same(cpu, gpu)
    assert opt.state_dict()["group_wd"] == [0.3, 0.3]


@pytest.mark.parametrize("bits", [32, 8])
def test_wide_range(bits):
    """Gradients from denormal squares to roots past 2^31, zeros among them."""
    gen = torch.Generator().manual_seed(2)
    n = 40000
    g = torch.randn(n, generator=gen) * 10.0 ** (torch.rand(n, generator=gen) * 46 - 28)
    g[::7] = 0.0
    g[:2048] *= 1e-22
    sides = []
    for d in ("cpu", "cuda"):
        p = torch.nn.Parameter(torch.linspace(-1, 1, n).to(d))
        p.grad = g.to(d, copy=True)
        opt = SodAdamW([{"params": [p]}], state_bits=bits, seed=1)
        for _ in range(2):
            opt.step(1e-2)
            p.grad *= 0.3
        sides.append(([p], None, opt))
    same(*sides)


def test_past_32_bits():
    """An element's place passes 2^32: the last elements move as the CPU's do."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    n = 2 ** 32 + 300
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    opt = SodAdamW([{"params": [p], "weight_decay": 0.1}], state_bits=8, seed=3)
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(300).bfloat16()
    g[-300:] = tail.cuda()
    p.grad = g
    opt.step(1e-2)
    cm, cr, sc = (torch.zeros(512, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8),
                  torch.zeros(2, 2))
    w, out = torch.zeros(300), torch.zeros(300, dtype=torch.bfloat16)
    m, v = reference._adamw_moments(torch.nn.functional.pad(tail.float(), (0, 212)),
                                    torch.zeros(512), torch.zeros(512), opt.betas,
                                    torch.tensor(1.0))
    reference._adamw_weight(out, w, m[:300], reference._root(v)[:300], 1e-2, 1, opt.betas,
                            opt.eps, 0.1)
    noise = reference.adamw8_noise(512, 3, 1, 0, first=2 ** 32)
    cm, cr, sc = reference.adamw8_encode(m, reference._root(v), noise)
    assert differ(p[-300:], out) == 0 and differ(opt.scales[-2:], sc) == 0
    assert differ(opt.code_m[-512:], cm) == 0 and differ(opt.code_r[-512:], cr) == 0
    assert not opt.code_m[:-512].any() and not opt.scales[:-2].any()
    norm, _ = grad_norm([g])
    want = tail.double().square().sum().sqrt().item()
    assert abs(norm.item() - want) <= 2.0 ** -23 * want


def test_past_32_bits_with_32_bit_moments():
    """The same with moments in 32 bits."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    n = 2 ** 32 + 300
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    opt = SodAdamW([{"params": [p], "weight_decay": 0.1}])
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    head, tail = torch.randn(300).bfloat16(), torch.randn(300).bfloat16()
    g[:300], g[-300:] = head.cuda(), tail.cuda()
    p.grad = g
    opt.step(1e-2)
    for part, grad in ((slice(0, 300), head), (slice(n - 300, n), tail)):
        q = torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16))
        q.grad = grad
        one = SodAdamW([{"params": [q], "weight_decay": 0.1}])
        one.step(1e-2)
        assert differ(p[part], q) == 0
        for a, b in ((opt.master, one.master), (opt.exp_avg, one.exp_avg),
                     (opt.exp_avg_sq, one.exp_avg_sq)):
            assert differ(a[part], b[:300]) == 0
    assert not opt.exp_avg[300:n - 300].any() and not p[300:n - 300].any()


def test_refusals():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    opt = SodAdamW([{"params": [p]}])
    with pytest.raises(RuntimeError, match="scale_t"):
        p.grad = torch.ones_like(p)
        opt.step(0.1, scale_t=torch.ones(()))
    with pytest.raises(RuntimeError, match="lr"):
        opt.step(torch.ones((), dtype=torch.float64, device="cuda"))
    opt.grad_src = {p: torch.ones(4)}
    with pytest.raises(RuntimeError, match="device"):
        opt.step(0.1)
    opt.grad_src = {p: torch.ones(5, device="cuda")}
    with pytest.raises(RuntimeError, match="size"):
        opt.step(0.1)
    opt.grad_src = {p: torch.ones(4, device="cuda").double()}
    with pytest.raises(RuntimeError, match="float32"):
        opt.step(0.1)
    opt.grad_src = None
    p.data = p.data.bfloat16()
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="changed"):
        opt.step(0.1)
    q = torch.nn.Parameter(torch.ones(2, 3, 4, 5, device="cuda"))
    opt = SodAdamW([{"params": [q]}])
    q.data = q.data.contiguous(memory_format=torch.channels_last)
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="changed"):
        opt.step(0.1)
    with pytest.raises(RuntimeError, match="loss_scale"):
        grad_norm([p.grad], loss_scale=torch.ones(()))
    with pytest.raises(RuntimeError, match="one device"):
        grad_norm([p.grad, torch.ones(3)])
    with pytest.raises(RuntimeError, match="float32"):
        grad_norm([p.grad.double()])
    with pytest.raises(ValueError, match="one device"):
        SodAdamW([{"params": [p, torch.nn.Parameter(torch.ones(3))]}])


@pytest.mark.parametrize("shape", [(0,), (2,), (3, 1)])
def test_scalars_that_are_none(shape):
    """An empty one is not taken for one that was not given."""
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = SodAdamW([{"params": [p]}])
    t, one = torch.ones(shape, device="cuda"), torch.ones((), device="cuda")
    with pytest.raises(RuntimeError, match="lr must be"):
        opt.step(t)
    with pytest.raises(RuntimeError, match="scale_t must be"):
        opt.step(0.1, scale_t=t)
    for kw in (dict(loss_scale=t), dict(loss_scale=one, good_steps=t, skips=one),
               dict(loss_scale=one, good_steps=one, skips=t)):
        with pytest.raises(ValueError, match="must be a scalar"):
            grad_norm([p.grad], **kw)
    assert (p == 1).all()


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [0, 3], [8191, 8192, 8193], [1] * 700,
                                   [64, 7, 0, 300000, 16384] * 40, [20_000_003]])
def test_grad_norm(dtype, sizes):
    """Its sum is in 64 bits: only the results' own roundings count.  Views start
    at odd elements; a repeated call has the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(sum(sizes) + 1, generator=gen, device="cuda").to(dtype)
    grads = list(flat[1:].split(sizes))
    want = flat[1:].double().square().sum().sqrt().item() / 8
    norm, mult = grad_norm(grads, prescale=0.125, max_norm=want / 3)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    m = want / 3 / (want + 1e-6)
    assert abs(mult.item() - m) <= 2.0 ** -22 * m
    again = grad_norm(grads, prescale=0.125, max_norm=want / 3)
    assert differ(norm, again[0]) == 0 and differ(mult, again[1]) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [8192 * 2048 + 300, 8192 * 4096 + 1, 8192 * 2048 * 3 + 4097,
                               8192 * 33000 + 300])
def test_grad_norm_ends(dtype, n):
    """Every piece counts: alone, the first elements and the last, as the first,
    second and later piece of a workgroup."""
    x = torch.zeros(n, dtype=dtype, device="cuda")
    for part in (x[:300], x[-300:], x[-8193:-8192], x[n // 2:n // 2 + 1]):
        part.fill_(2.0)
        norm = grad_norm([x])[0].item()
        want = 2.0 * math.sqrt(part.numel())
        assert abs(norm - want) <= 2.0 ** -23 * want
        part.zero_()


def apart(sizes, dtypes, fill=None):
    """Gradients with a NaN between them, so that no two are neighbours and
    nothing beside them may be read, of the types in turn."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    ends = [0] * len(dtypes)
    places = []
    for k, n in enumerate(sizes):
        places.append(ends[k % len(dtypes)] + 1)
        ends[k % len(dtypes)] += n + 1
    flats = [torch.full((e + 1,), math.nan, dtype=t, device="cuda")
             for e, t in zip(ends, dtypes)]
    out = []
    for k, n in enumerate(sizes):
        g = flats[k % len(dtypes)][places[k]:places[k] + n]
        g.copy_(torch.randint(-3, 4, (n,), device="cuda", generator=gen)
                if fill is None else torch.full((n,), fill, device="cuda"))
        out.append(g)
    return out


def merged(grads):
    """How many stretches of memory they are."""
    return 1 + sum(a.dtype != b.dtype or a.data_ptr() + a.numel() * a.element_size()
                   != b.data_ptr() for a, b in zip(grads, grads[1:]))


@pytest.mark.parametrize("count", [1, 5, 64, 159, 160, 161, 320, 321, 700])
@pytest.mark.parametrize("size", [1, 23, 103, 8192, 8193, 20000])
@pytest.mark.parametrize("dtypes", [TYPES[:1], TYPES[1:2], TYPES])
def test_grad_norm_apart(count, size, dtypes):
    """Tensors that lie apart, below and past what one launch takes, in total and in
    number.  Whole numbers: the sum in 64 bits is exact, whatever its order, and
    the root is rounded once to 64 and once to 32 bits."""
    sizes = [max(1, size - 3 * (k % 7)) for k in range(count)]
    grads = apart(sizes, dtypes)
    assert merged(grads) == count
    total = sum(int(g.double().square().sum().item()) for g in grads)
    norm, mult = grad_norm(grads, max_norm=1.0)
    assert norm.item() == torch.tensor(math.sqrt(total)).float().item()
    again = grad_norm(grads, max_norm=1.0)
    assert norm.item() == again[0].item() and mult.item() == again[1].item()


@pytest.mark.parametrize("count, size", [(5, 7), (160, 100), (160, 9000), (161, 3), (700, 8200)])
def test_grad_norm_apart_ends(count, size):
    """The first and the last element of every tensor that ends or starts a launch's
    share count, alone."""
    grads = apart([size] * count, TYPES, fill=0.0)
    for k in sorted({0, 1, count // 2, count - 1, *(k for k in (63, 64, 159, 160, 319, 320, 639)
                                                    if k < count)}):
        for i in (0, size - 1):
            grads[k][i] = 2.0
            assert grad_norm(grads)[0].item() == 2.0, (k, i)
            grads[k][i] = 0.0


def test_grad_norm_wherever_the_allocator_puts_it():
    """Two tensors beside each other and the same two apart: the same bits.  The sum
    of squares is 2^46 + 2^23 + 1/4, whose root lies half way between two float32,
    and 15 squares of 2^-8 that decide it unless each is added to 2^46 by itself."""
    flat = torch.zeros(8192, device="cuda")
    flat[0], flat[4096], flat[4097], flat[4098] = 2.0 ** 23, 2.0 ** 11, 2.0 ** 11, 0.5
    flat[256:4096:256] = 2.0 ** -4
    rest = torch.zeros(20000, device="cuda")    # more than one workgroup's
    near = [torch.from_dlpack(flat[:4096]), torch.from_dlpack(flat[4096:])]
    assert near[0].data_ptr() + 4096 * 4 == near[1].data_ptr()
    gap = torch.zeros(3, 4096, device="cuda")
    far = [gap[0].copy_(flat[:4096]), gap[2].copy_(flat[4096:])]
    assert [grad_norm(x + [rest])[0].item() for x in (near, far)] == [2.0 ** 23] * 2
    # one stretch of one storage: grouped otherwise
    assert grad_norm([*flat.split(4096), rest])[0].item() == 2.0 ** 23 + 1


def test_grad_norm_apart_captured():
    """Several launches and the scaler in a graph, eager work between the replays."""
    grads = apart([8193, 5, 300] * 150, TYPES)
    scale, good, skips = (torch.tensor(v, device="cuda") for v in (8.0, 0.0, 0.0))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, mult = grad_norm(grads, max_norm=1.0, loss_scale=scale,
                               good_steps=good, skips=skips, growth_interval=2)
    for i in range(4):
        for g in grads[::40]:
            g.fill_(i)
        before = scale.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = grad_norm(grads, max_norm=1.0, loss_scale=before)
        assert differ(norm, want[0]) == 0 and differ(mult, want[1]) == 0
        assert math.isfinite(norm.item()) and scale.item() == 8.0 * 2 ** ((i + 1) // 2)


def test_grad_norm_views_and_range():
    x = torch.randn(40, 30, device="cuda")
    mixed = [x.t(), x[::2, ::3], x[:1].expand(5, 30), x.bfloat16(), x.half()]
    want = math.sqrt(sum(t.double().square().sum().item() for t in mixed))
    assert abs(grad_norm(mixed)[0].item() - want) <= 2.0 ** -23 * want
    big = torch.full((4096,), 1e38, device="cuda").bfloat16()
    norm, mult = grad_norm([big], max_norm=1e-6)
    want = big.double().square().sum().sqrt().item()
    assert want > 3.4e38 and math.isinf(norm.item()) and mult.item() == 0.0
    norm, mult = grad_norm([big], prescale=1e-3, max_norm=1e-6)
    assert abs(norm.item() - want * 1e-3) <= 2.0 ** -23 * want * 1e-3 and mult.item() > 0
    for bad in (math.inf, -math.inf, math.nan):
        norm, mult = grad_norm([torch.ones(9, device="cuda"),
                                torch.full((1,), bad, device="cuda").half()], max_norm=1.0)
        assert not math.isfinite(norm.item()) and mult.item() == 0.0
    norm, mult = grad_norm([torch.zeros(0, device="cuda")], max_norm=1.0)
    assert norm.item() == 0.0 and mult.item() == 1.0


def test_grad_norm_scaler_like_the_cpu():
    gen = torch.Generator().manual_seed(0)
    sides = [[torch.tensor(v, device=d) for v in (64.0, 0.0, 0.0)] for d in ("cpu", "cuda")]
    for i in range(30):
        g = torch.randn(1000, generator=gen)
        if i % 7 == 5:
            g[17] = math.inf
        out = [grad_norm([g.to(s[0].device)], max_norm=1.0, loss_scale=s[0],
                         good_steps=s[1], skips=s[2], growth_interval=3) for s in sides]
        assert [t.item() for t in sides[0]] == [t.item() for t in sides[1]]
        a, b = (o[1].item() for o in out)
        assert abs(a - b) <= 2.0 ** -22 * a


def test_grad_norm_captured():
    x = torch.randn(300_000, device="cuda").bfloat16()
    scale, good, skips = (torch.tensor(v, device="cuda") for v in (8.0, 0.0, 0.0))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, mult = grad_norm([x, x[:7]], max_norm=1.0, loss_scale=scale,
                               good_steps=good, skips=skips, growth_interval=2)
    for i in range(4):
        x.normal_()
        before = scale.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = grad_norm([x, x[:7]], max_norm=1.0, loss_scale=before)
        assert differ(norm, want[0]) == 0 and differ(mult, want[1]) == 0
        assert scale.item() == 8.0 * 2 ** ((i + 1) // 2)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("graph", [False, True])
def test_solver_steps(tmp_path, bits, dtype, graph):
    """Whole steps of a network, eager and replayed: an optimizer of its own on
    copies of the weights, given each step's gradients, follows to the bit.  (Two
    runs of the network itself need not agree: its loss adds with atomics.)"""
    from sodkit.config import make_config
    from sodkit.engine import Solver
    cfg = make_config("minet_r50_352", batch_size=2, size=64, num_workers=0,
                      output_root=str(tmp_path), dtype=dtype,
                      loss_scale=2.0 ** 16 if dtype == "fp16" else 1.0, grad_clip=1.0,
                      optimizer="adamw", adam_state_bits=bits, lr=1e-4,
                      weight_decay=0.05, hip_graph=graph)
    s = Solver(cfg)
    s.total_iters = 100
    copies = {p: torch.nn.Parameter(p.detach().clone()) for p in s.optimizer.params()}
    opt = SodAdamW([{"params": [copies[p] for p in g["params"]],
                     "weight_decay": g["weight_decay"]} for g in s.optimizer.groups],
                   state_bits=bits, seed=cfg.seed)
    opt.grad_src = {copies[p]: v for p, v in s.reducer.grad_views.items()}
    kw = dict(loss_scale=s._scale_t.clone())
    if s.dynamic_scale:
        kw |= dict(good_steps=s._good_t.clone(), skips=s._skips_t.clone())
    g = torch.Generator().manual_seed(0)
    x = s._to_device(torch.rand(2, 3, 64, 64, generator=g), cast=True)
    t = (torch.rand(2, 1, 64, 64, generator=g) > 0.5).float().cuda()
    for i in range(6):
        lr = torch.tensor(s._lr_at(i), device="cuda") if graph and i >= 2 else s._lr_at(i)
        assert math.isfinite(s.step(x, t).item())
        _, mult = grad_norm([b.flat for b in s.reducer.buckets], max_norm=1.0, **kw)
        opt.step(lr, scale_t=mult)
        for p, q in copies.items():
            assert differ(p, q) == 0, i
        for k, v in kw.items():
            mine = {"loss_scale": s._scale_t, "good_steps": s._good_t, "skips": s._skips_t}
            assert differ(v, mine[k]) == 0, k
    assert (s._graph is not None) == graph
    for a, b in zip([s.optimizer.master, *s.optimizer.moments()],
                    [opt.master, *opt.moments()]):
        assert differ(a, b) == 0
    steps = {st["step"] for st in s.optimizer.state_dict()["param_state"]}
    assert steps == {6 - s._scaler_state()[1]} and isinstance(s.optimizer, ops.SodAdamW)
